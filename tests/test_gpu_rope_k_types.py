"""b200attn_rope_k from Python: each of its types, and the tensors that it would misread."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("half", [False, True], ids=["interleaved", "half"])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_rope_k_in_16_bits_is_the_fp32_rotation_rounded_once(pkg, cuda, dtype, half):
    import torch
    td = getattr(torch, dtype)
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    x = torch.randn(2, 3, 77, 96, generator=g, device="cuda").to(td)
    pairing = pkg.PE_ROPE_HALF if half else pkg.PE_ROPE_INTERLEAVED
    want, got = pkg.rope_k(x.float(), pairing=pairing, pos0=3).double(), pkg.rope_k(x, pairing=pairing, pos0=3)
    assert got.dtype is td
    # x cos - y sin: two products and a sum in fp32 on either side, then half a step of the type (2^-25 below fp16's normal range)
    size = 2 * float(x.double().abs().max())
    bound = torch.finfo(td).eps / 2 * want.abs() + 6 * 2.0 ** -24 * size + 2.0 ** -25
    assert bool(((got.double() - want).abs() <= bound).all())


def test_rope_k_refuses(pkg, cuda):
    import torch
    x = torch.zeros(1, 2, 5, 8, device="cuda")
    c = torch.zeros(5, 8, device="cuda")
    for call in (lambda: pkg.rope_k(x.transpose(1, 2)), lambda: pkg.rope_k(x, out=x.half()), lambda: pkg.rope_k(x, out=x[:, :, :4]), lambda: pkg.rope_k(x.double()),
                 lambda: pkg.rope_k(x.cpu()), lambda: pkg.rope_k(x, cos_cache=c[:4], sin_cache=c), lambda: pkg.rope_k(x, cos_cache=c, sin_cache=c.half()),
                 lambda: pkg.rope_k(x, pos0=1, cos_cache=c, sin_cache=c)):
        with pytest.raises(pkg.B200AttnError):
            call()
    pkg.rope_k(x, cos_cache=c, sin_cache=c)
