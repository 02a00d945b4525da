"""The cache calls at the ends of the types' ranges: scores as large as fp32 holds, and cached values that are not finite, on every path of cache_attend."""
import math

import pytest

from test_gpu_cache import DT

pytestmark = pytest.mark.gpu
E = 2.0 ** -24

PATHS = [
    # path, B, Hq, Hkv, T, D
    ("cache_narrow", 2, 4, 2, 3, 64), ("cache_narrow", 1, 8, 1, 5, 128), ("cache_narrow", 1, 6, 2, 16, 192),
    ("cache_tc", 2, 4, 2, 40, 64), ("cache_tc", 1, 4, 1, 70, 128), ("cache_tc", 1, 4, 2, 40, 256),
    ("cache_generic", 2, 4, 2, 3, 64), ("cache_generic", 1, 4, 2, 9, 128), ("cache_generic", 1, 4, 4, 17, 100),
]
CASES = [(p, d) for p in PATHS for d in ("bf16", "f16", "f32") if d != "f32" or p[0] == "cache_generic"]
IDS = [f"{p[0]}-{'-'.join(map(str, p[1:]))}-{d}" for p, d in CASES]


def one_score(pkg, path, dtype, a, scale, S, lengths):
    """Every query is a e_0; cached keys are in turn e_0 and (1 - 2^-7) e_0, the new ones e_0 ((1 - 2^-7) e_0 where a < 0): the larger of the two scores,
    s = a scale or a scale (1 - 2^-7), takes all the weight (they differ by 2^-7 |s|, thousands and more), evenly: the result is a mean over the keys that have it."""
    import torch
    name, B, Hq, Hkv, T, D = path
    td = getattr(torch, DT[dtype])
    g = torch.Generator(device="cuda")
    g.manual_seed(50)
    low = 1.0 - 2.0 ** -7
    z = lambda h, rows: torch.zeros(B, h, rows, D, dtype=td, device="cuda")
    Q, K, Kd = z(Hq, T), z(Hkv, S), z(Hkv, T)
    Q[..., 0] = a
    K[:, :, ::2, 0], K[:, :, 1::2, 0], Kd[..., 0] = 1.0, low, 1.0 if a > 0 else low
    V, Vd = (torch.randn(B, Hkv, n, D, generator=g, device="cuda").to(td) for n in (S, T))
    length = torch.tensor([lengths[b % len(lengths)] for b in range(B)], dtype=torch.int32, device="cuda")
    out, lse = pkg.cache_attend(Q, K, V, length, Kd, Vd, scale=scale, flags=pkg.FLAG_FORCE_GENERIC if name == "cache_generic" else 0)
    assert pkg.last_path() == name
    u = torch.finfo(td).eps / 2
    s = a * scale * (1.0 if a > 0 else low)
    for b, n in enumerate(length.tolist()):
        for h in range(Hq):
            v = V[b, h // (Hq // Hkv), (0 if a > 0 else 1): n: 2].double()
            vd = Vd[b, h // (Hq // Hkv)].double()
            many = v.shape[0] + torch.arange(1, T + 1, device="cuda", dtype=torch.float64)
            want = (v.sum(0) + vd.cumsum(0)) / many[:, None]
            size = (v.abs().sum(0) + vd.abs().cumsum(0)) / many[:, None]
            # equal weights, rounded alike: u once for them and once for the result; the sums of at most `many` terms
            bound = u * (size + want.abs()) + (many[:, None] + 16) * 2 * E * size + (2.0 ** -25 if td is torch.float16 else 0.0)
            assert bool(((out[b, h].double() - want).abs() <= bound).all()), (b, h, float((out[b, h].double() - want).abs().max()))
            # the constants log2 e and ln 2, the scale's product and the three operations behind: 6 roundings relative to s, and those of the logarithm
            assert bool(((lse[b, h].double() - (s + many.log())).abs() <= 6.5 * E * abs(s) + 100 * E).all())


@pytest.mark.parametrize("S,lengths", [(300, (300, 129)), (5000, (5000, 2))], ids=["short", "long"])
@pytest.mark.parametrize("s", [2.0 ** 20, 2.0 ** 25, 2.0 ** 34, 1e30, 2.2e38])
@pytest.mark.parametrize("path,dtype", CASES, ids=IDS)
def test_attend_with_large_scores(pkg, cuda, path, dtype, s, S, lengths):
    """Scores whose rounding is more than an exponential takes, up to the end of fp32's range over log2 e (2.35e38)."""
    for sign in (1.0, -1.0):
        one_score(pkg, path, dtype, 1.25 * sign, s / 1.25, S, lengths)


@pytest.mark.parametrize("path,dtype", [c for c in CASES if c[1] != "f16"], ids=[i for i, c in zip(IDS, CASES) if c[1] != "f16"])
def test_attend_with_large_products(pkg, cuda, path, dtype):
    """The same from large products of the tensors' own values."""
    for a in (2.0 ** 126, -2.0 ** 126):
        one_score(pkg, path, dtype, a, 1.0, 700, (700, 300))


def with_low_keys(dtype, shape, drafts, low, seed):
    """A problem whose queries share a direction, and cached and new keys far down it (by e^-40: nothing in fp16; by e^-300: nothing in fp32), whose values are not finite."""
    import torch
    from test_gpu_cache import Problem
    _, B, Hq, Hkv, T, D = shape
    S, lengths = (300, (300, 129)) if seed % 2 else (5000, (5000, 2))
    p = Problem(dtype, B, Hq, Hkv, T, S, lengths, D, drafts, seed=seed)
    p.Q[..., 0], p.K[..., 0] = 8.0, 0.0
    if drafts != "none":
        p.Kd[..., 0] = 0.0
        p.Kd[:, :, T // 2] = math.nan
    down = -low * math.sqrt(D) / 8.0
    g = torch.Generator().manual_seed(seed)
    for b, n in enumerate(p.length.tolist()):
        for at, value, column, h in ((0, math.inf, 0, 0), (n // 3, -math.inf, 1, 0), (n // 2, math.nan, 2, Hkv - 1), (n - 1, math.inf, D - 1, Hkv - 1), (n // 4, math.inf, 1, 0),
                                     (n // 5, math.inf, D // 2, 0), (n // 6, math.inf, D // 2, 0)):
            p.V[b, h, at, column] = value
            p.K[b, h, at, 0] = down
    # every value of a column, and one that weighs what others do
    p.V[0, 0, : int(p.length[0]), 5], p.V[B - 1, 0, 1, 6] = math.inf, -math.inf
    if drafts != "none" and T > 2:
        p.Vd[0, 0, 0, 3], p.Vd[0, 0, 1, 4], p.Vd[0, Hkv - 1, 0, 0] = math.inf, -math.inf, -math.inf
        p.Kd[0, :, :2, 0] = down
    return p


@pytest.mark.parametrize("drafts", ["none", "tree"])
@pytest.mark.parametrize("low", [0.0, 40.0, 300.0])
@pytest.mark.parametrize("path,dtype", CASES, ids=IDS)
def test_attend_with_cached_values_that_are_not_finite(pkg, cuda, path, dtype, low, drafts):
    """A cached value that is infinite is so in the result, NaN where another of the other sign is seen, whatever it weighs."""
    import cache_ref as ref
    for seed in (60, 61):
        p = with_low_keys(dtype, path, drafts, low, seed)
        out, lse = pkg.cache_attend(*p.args(), flags=pkg.FLAG_FORCE_GENERIC if path[0] == "cache_generic" else 0)
        assert pkg.last_path() == path[0]
        want, want_lse, b_out, b_lse = ref.attend(*p.args())
        ok, worst = ref.close(lse, want_lse, b_lse)
        assert ok, ("lse", worst)
        ok, worst = ref.close(out, want, b_out)
        assert ok, ("out", worst)


@pytest.mark.parametrize("dtype,path,T,G", [("bf16", "cache_narrow", 1, 4), ("f16", "cache_tc", 40, 2), ("f32", "cache_generic", 1, 1)])
def test_a_cache_of_nothing_finite(pkg, cuda, dtype, path, T, G):
    """Long caches that are NaN throughout, or infinite throughout a column: an answer, in time."""
    import torch
    td = getattr(torch, DT[dtype])
    B, Hkv, S, D = 74, 2, 60000, 128
    Q, K = torch.randn(B, Hkv * G, T, D, device="cuda").to(td), torch.zeros(B, Hkv, S, D, dtype=td, device="cuda")
    K[:, :, : S // 2] = -1000.0
    V = torch.zeros(B, Hkv, S, D, dtype=td, device="cuda")
    V[0], V[1:, :, :, 7] = math.nan, -math.inf
    n = torch.full((B,), S, dtype=torch.int32, device="cuda")
    out, _ = pkg.cache_attend(Q, K, V, n)
    assert pkg.last_path() == path
    want = torch.zeros(B, Hkv * G, T, D, device="cuda")
    want[0], want[1:, :, :, 7] = math.nan, -math.inf
    assert torch.equal(out.float().nan_to_num(1.0, 2.0, 3.0), want.nan_to_num(1.0, 2.0, 3.0))
