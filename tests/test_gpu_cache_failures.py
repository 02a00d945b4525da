"""Failure detection in the tensor-core kernels of the cache calls, without faulting anything: their first key tile is made to wait, with a short limit, for an
arrival that never comes.  Every role gives up by itself, the call reports B200ATTN_ERR_KERNEL, and the next call on the same context is right again."""
import math

import pytest

from test_gpu_cache import Problem, check_attend

pytestmark = pytest.mark.gpu
ERR_KERNEL = 4
LIMIT = 2000


def lost(pkg, call):
    """`call` with lost arrivals: refused with the kernel's error, also where an asynchronous call left it for the next one to report."""
    import torch
    pkg.lib().b200attn_debug_lost_arrival(1, LIMIT)
    try:
        with pytest.raises(pkg.B200AttnError) as e:
            call(0)
        assert e.value.status == ERR_KERNEL and "0x" in str(e.value)
        call(pkg.FLAG_ASYNC)
        torch.cuda.synchronize()
        with pytest.raises(pkg.B200AttnError) as e:
            call(0)
        assert e.value.status == ERR_KERNEL and "earlier asynchronous call" in str(e.value)
    finally:
        pkg.lib().b200attn_debug_lost_arrival(0, 0)


def poisoned(nbytes):
    """Memory that torch's allocator hands out next holds numbers that are no addresses of anything."""
    import torch
    del_me = [torch.full((max(nbytes // 4, 1),), 0x7F7F7F7F, dtype=torch.int32, device="cuda") for _ in range(3)]
    torch.cuda.synchronize()
    del del_me


ATTEND = [
    ("cache_narrow", (1, 8, 2, 3, 5000, (5000,), 128, "tree")),              # few units, each cut over many CTAs: an entry per unit
    ("cache_narrow", (90, 4, 2, 2, 1500, (1500, 3, 0, 900), 64, "chain")),   # more units than CTAs: several a CTA, an entry per CTA
    ("cache_narrow", (70, 8, 2, 1, 1500, (1500, 1400), 128, "chain")),       # one unit a CTA or two: an entry per unit
    ("cache_tc", (1, 16, 2, 64, 3000, (3000,), 128, "tree")),                # two row tiles a unit
    ("cache_tc", (2, 4, 4, 200, 700, (700, 90), 64, "none")),                # ... the last one without a second tile
    ("cache_tc", (70, 16, 2, 16, 900, (900, 0, 5), 64, "tree")),             # one row tile a unit
    ("cache_tc", (3, 16, 2, 30, 500, (500, 31), 256, "chain")),              # tiles of 64 keys
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("path,shape", ATTEND, ids=lambda s: s if isinstance(s, str) else "-".join(map(str, s[:5])))
def test_attend_gives_up(pkg, cuda, path, shape, dtype):
    p = Problem(dtype, *shape, seed=40)
    pkg.cache_attend(*p.args())
    assert pkg.last_path() == path
    for n in {v for v in pkg._attend_ws.values() if v}:
        poisoned(n)
    lost(pkg, lambda flags: pkg.cache_attend(*p.args(), flags=flags))
    check_attend(pkg, p)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("A", [0, 5], ids=["by-tma", "gathered"])
def test_weights_gives_up(pkg, cuda, dtype, A):
    import torch
    p = Problem(dtype, 9, 8, 2, 24, 700, (700, 333, 1), 128, "none", token=True, seed=41)
    lse = torch.full((9, 8, 24), math.log(700.0), device="cuda")
    accepted = torch.arange(A, dtype=torch.int32, device="cuda").repeat(9, 1) if A else None
    w = torch.zeros(9, 2, 700, device="cuda")
    want = pkg.cache_weights(p.Q, p.K, p.length, lse, w.clone(), accepted)
    assert pkg.last_path() == "cache_tc"
    lost(pkg, lambda flags: pkg.cache_weights(p.Q, p.K, p.length, lse, w.clone(), accepted, flags=flags))
    assert torch.equal(pkg.cache_weights(p.Q, p.K, p.length, lse, w.clone(), accepted), want)
