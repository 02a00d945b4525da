"""The cache operators on the GPU against their definitions in 64 bits (cache_ref.py, where the bounds are derived): every type and path, lengths around the tile
sizes, empty rows, masked and unused places that hold NaN, views, lists that end early, captures, streams and threads, and a run of them together."""
import math
import threading

import pytest

import cache_ref as ref

pytestmark = pytest.mark.gpu
DT = {"f32": "float32", "bf16": "bfloat16", "f16": "float16"}


class Problem:
    """Inputs of one attention call.  `token`: Q, Kd, Vd are views of [B, T, heads, D]; every place that no token may see holds NaN."""

    def __init__(self, dtype, B, Hq, Hkv, T, S, lengths, D, drafts, token=False, seed=0, mask=None, cache_rows_first=False):
        import torch
        g = torch.Generator(device="cuda")
        g.manual_seed(1000 + seed)
        td = getattr(torch, DT[dtype])
        def make(heads, rows, tok, spread=1.0):
            t = torch.randn((B, rows, heads, D) if tok else (B, heads, rows, D), generator=g, device="cuda").mul_(spread).to(td)
            return t.transpose(1, 2) if tok else t
        self.Q, self.K, self.V = make(Hq, T, token, 1.5), make(Hkv, S, cache_rows_first), make(Hkv, S, cache_rows_first)
        self.length = torch.tensor([lengths[b % len(lengths)] for b in range(B)], dtype=torch.int32, device="cuda")
        for b, n in enumerate(self.length.tolist()):
            self.K[b, :, max(n, 0):], self.V[b, :, max(n, 0):] = math.nan, math.nan
        self.Kd = self.Vd = self.mask = None
        if drafts != "none":
            self.Kd, self.Vd = make(Hkv, T, token), make(Hkv, T, token)
        if drafts in ("tree", "shared"):
            m = torch.rand(1 if drafts == "shared" else B, T, T, generator=g, device="cuda") < 0.4
            m |= torch.eye(T, dtype=torch.bool, device="cuda")
            m[:, T // 3] = False              # a padded token: it sees none of the new ones
            m[:, :, T // 2] = False           # and one that nobody sees
            self.Kd[:, :, T // 2], self.Vd[:, :, T // 2] = math.nan, math.nan
            self.mask = m.to(torch.uint8)

    def args(self):
        return (self.Q, self.K, self.V, self.length, self.Kd, self.Vd, self.mask)


def check_attend(pkg, p, scale=0.0, flags=0):
    out, lse = pkg.cache_attend(*p.args(), scale=scale, flags=flags)
    want, want_lse, b_out, b_lse = ref.attend(*p.args(), scale=scale)
    ok, worst = ref.close(lse, want_lse, b_lse)
    assert ok, ("lse", worst)
    ok, worst = ref.close(out, want, b_out)
    assert ok, ("out", worst)
    return out, lse


SHAPES = [
    # B, Hq, Hkv, T, S, lengths, D, drafts
    (1, 1, 1, 1, 1, (0,), 64, "chain"),            # nothing cached: the new token alone
    (1, 1, 1, 1, 1, (1,), 64, "none"),
    (2, 4, 2, 1, 300, (0, 300), 64, "none"),       # a sequence without states: rows of zeros
    (3, 8, 2, 1, 260, (1, 64, 129), 128, "chain"),
    (4, 8, 1, 5, 200, (63, 65, 127, 128), 128, "tree"),
    (3, 6, 2, 17, 400, (0, 255, 400), 64, "tree"),
    (2, 5, 5, 33, 150, (149, 2), 128, "shared"),
    (1, 16, 2, 64, 1000, (999,), 128, "tree"),
    (2, 4, 4, 150, 260, (257, 130), 128, "chain"),  # more tokens than a tile, behind a cache
    (2, 6, 2, 130, 40, (0, 33), 64, "tree"),
    (1, 3, 3, 300, 130, (0,), 128, "chain"),        # a prompt from nothing
    (2, 4, 4, 200, 333, (333, 90), 64, "none"),     # cross attention
    (2, 4, 2, 3, 150, (150, 77), 256, "tree"),
    (1, 4, 2, 140, 300, (290,), 256, "chain"),
    (2, 2, 1, 3, 150, (129, 77), 192, "chain"),
    (2, 4, 2, 5, 150, (140, 3), 80, "tree"),
    (2, 4, 2, 5, 150, (140, 3), 96, "tree"),
    (2, 4, 2, 3, 140, (131, 1), 8, "tree"),
    (2, 4, 2, 3, 140, (131, 1), 100, "tree"),       # no whole 16 bytes a row in 16 bits
    (1, 2, 1, 3, 70, (66,), 33, "chain"),
    (1, 2, 1, 2, 70, (66,), 1, "chain"),
    (1, 14, 2, 19, 300, (290,), 128, "tree"),       # 7 query heads a key head
    (1, 40, 1, 4, 300, (290,), 64, "tree"),         # 40
    (1, 200, 1, 2, 100, (90,), 64, "tree"),         # more than a tile of rows for one token
    (40, 2, 1, 1, 100, tuple(range(0, 100, 7)), 64, "chain"),
    (1, 16, 1, 4, 300, (299,), 256, "tree"),        # 64 rows a key head at the widest head
    (2, 10, 1, 6, 300, (120, 299), 192, "chain"),
    (1, 9, 1, 7, 200, (190,), 64, "tree"),          # 63 rows
    (2, 8, 1, 12, 300, (300, 127), 128, "tree"),    # one tile of 96 rows
    (3, 16, 2, 16, 300, (300, 0, 5), 64, "tree"),   # one of 128
    (2, 100, 1, 1, 300, (300, 11), 128, "chain"),   # one token of 100 heads
    (1, 126, 1, 3, 90, (77,), 80, "tree"),
    (40, 16, 2, 16, 100, tuple(range(0, 100, 7)), 128, "tree"),   # many short sequences: several units a CTA
    (37, 8, 2, 70, 50, tuple(range(0, 50, 3)), 128, "tree"),      # ... of two tiles, some of them without rows
    (9, 5, 5, 300, 60, tuple(range(0, 60, 7)), 64, "chain"),
    (30, 8, 4, 9, 200, tuple(range(0, 200, 13)), 256, "tree"),
]
PATHS = ("cache_narrow", "cache_tc", "cache_generic")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s[:5])) + f"-{s[6]}-{s[7]}")
def test_attend(pkg, cuda, shape, dtype):
    check_attend(pkg, Problem(dtype, *shape, seed=len(str(shape))))
    B, Hq, Hkv, T, _, _, D, _ = shape
    generic = dtype == "f32" or D % 8 or Hq // Hkv > 128
    assert pkg.last_path() == PATHS[2 if generic else 0 if Hq // Hkv * T <= 64 else 1]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", [SHAPES[4], SHAPES[5], SHAPES[8], SHAPES[13], SHAPES[24]], ids=lambda s: "-".join(map(str, s[:5])))
def test_attend_without_the_tensor_cores(pkg, cuda, shape, dtype):
    check_attend(pkg, Problem(dtype, *shape, seed=3), flags=pkg.FLAG_FORCE_GENERIC)
    assert pkg.last_path() == "cache_generic"


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape", [SHAPES[4], SHAPES[8], SHAPES[12], SHAPES[15]], ids=lambda s: "-".join(map(str, s[:5])))
def test_attend_on_views(pkg, cuda, shape, dtype):
    p = Problem(dtype, *shape, token=True, cache_rows_first=True, seed=5)
    out, _ = check_attend(pkg, p, scale=0.3)
    # the same numbers densely, and an output with strides of its own
    import torch
    B, Hq, T, D = p.Q.shape
    wide = torch.full((B, T, Hq + 1, D), 7.0, dtype=p.Q.dtype, device="cuda")
    view = wide[:, :, :Hq].transpose(1, 2)
    dense = [t.contiguous() if t is not None else None for t in p.args()]
    pkg.cache_attend(*dense, scale=0.3, out=view)
    assert torch.equal(view, out)
    assert bool((wide[:, :, Hq] == 7.0).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attend_on_unaligned_views(pkg, cuda, dtype):
    """Rows that do not begin on 16 bytes: another kernel, the same answer."""
    import torch
    p = Problem(dtype, *SHAPES[4], seed=6)
    out, lse = check_attend(pkg, p)
    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        v = flat[1:].view(t.shape)
        v.copy_(t)
        return v
    p.Q, p.K, p.V, p.Kd, p.Vd = (shifted(t) for t in (p.Q, p.K, p.V, p.Kd, p.Vd))
    check_attend(pkg, p)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attend_with_values_that_are_not_finite(pkg, cuda, dtype, D):
    """A new token's key or value that is NaN or infinite reaches the tokens that see it, and no other."""
    import torch
    p = Problem(dtype, 2, 4, 2, 9, 140, (131, 0), D, "tree", seed=7)
    p.mask[:, :, 6] = 0
    p.mask[:, 6, 6] = 1
    p.Vd[0, 0, 6, 3], p.Vd[0, 1, 6, 5], p.Vd[1, 0, 6, 1] = math.inf, math.nan, -math.inf
    p.mask[:, :, 7] = 0
    p.mask[:, 7, 7] = 1
    p.Kd[0, 0, 7] = math.nan
    p.Kd[0, 1, 7] = math.inf
    check_attend(pkg, p)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_attend_grows_and_falls_back_from_large_scores(pkg, cuda, dtype):
    """Maxima that rise from tile to tile by more and by less than an accumulator's reference takes, and a range of scores that exp has to survive."""
    import torch
    p = Problem(dtype, 1, 4, 2, 6, 700, (700,), 64, "tree", seed=8)
    steps = torch.tensor([0.2, 8.0, 1.0, 14.0, 3.0, 25.0, 0.1, 2.0, 30.0, 5.0, 0.5], device="cuda").repeat_interleave(64)[:700]
    p.K = (p.K.float() * steps[None, None, :, None]).to(p.K.dtype)
    check_attend(pkg, p)
    p.Q = (p.Q.float() * -1).to(p.Q.dtype)
    check_attend(pkg, p)


def test_attend_lengths_out_of_range_count_as_the_nearest(pkg, cuda):
    import torch
    p = Problem("bf16", 3, 4, 2, 3, 130, (130, 0, 130), 64, "chain", seed=9)
    want = pkg.cache_attend(*p.args())
    p.length = torch.tensor([1 << 30, -5, 131], dtype=torch.int32, device="cuda")
    got = pkg.cache_attend(*p.args())
    assert ref.same(got[0], want[0]) and ref.same(got[1], want[1])


def test_attend_repeats_to_the_bit_and_shares_the_work_of_a_batch(pkg, cuda):
    """The share-out goes by all sequences' lengths: a sequence's answer stays within the bounds, and equal calls agree to the bit."""
    p = Problem("bf16", 24, 8, 2, 3, 900, tuple(range(0, 900, 61)), 128, "tree", seed=10)
    a, b = check_attend(pkg, p), pkg.cache_attend(*p.args())
    assert ref.same(a[0], b[0]) and ref.same(a[1], b[1])


def test_attend_behind_32_bits(pkg, cuda):
    """A cache of more than 2^32 elements: the last sequence's rows lie behind offsets that a 32-bit number holds."""
    import torch
    B, H, S, D, n = 3, 8, 524288, 256, 1000
    K, V = (torch.zeros(B, H, S, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    p = Problem("bf16", B, 2 * H, H, 2, n, (n, 0, n - 1), D, "chain", seed=11)
    K[:, :, :n], V[:, :, :n] = p.K, p.V
    want, want_lse, b_out, b_lse = ref.attend(*p.args())
    out, lse = pkg.cache_attend(p.Q, K, V, p.length, p.Kd, p.Vd)   # (shared out differently from the same rows in a shorter cache: the bounds, not the bits)
    assert ref.close(out, want, b_out)[0] and ref.close(lse, want_lse, b_lse)[0]
    # and rows at the far end of a long sequence
    m = S - 3
    K[2, :, m - 2: m], V[2, :, m - 2: m] = 3.0, 2.0
    p.length = torch.tensor([1, 1, m], dtype=torch.int32, device="cuda")
    K[2, :, :n], V[2, :, :n] = 0, 0
    out, lse = pkg.cache_attend(p.Q, K, V, p.length)
    q = p.Q[2].double().sum(-1) * 3.0 / 16
    total = torch.log((m - 2) + 2 * torch.exp(q))
    assert bool(((lse[2].double() - total).abs() < 1e-3).all())
    value = 4 * torch.exp(q - total)
    assert bool(((out[2].double() - value[..., None]).abs() <= 2 ** -7 * value[..., None] + 1e-6).all())


def test_attend_takes_the_library_s_workspace(pkg, cuda):
    """The C call without a workspace, asynchronous, behind a call of another stream."""
    import ctypes as C
    import torch
    p = Problem("bf16", 3, 8, 2, 5, 600, (600, 31, 0), 128, "tree", seed=12)
    want = pkg.cache_attend(*p.args())
    keep = pkg._pack_attend
    seen = []
    def without(*values):
        values = list(values)
        n = len(values)
        values[n - 4], values[n - 3] = 0, 0
        seen.append(1)
        return keep(*values)
    other = torch.cuda.Stream()
    pkg._pack_attend = without
    try:
        got = pkg.cache_attend(*p.args(), flags=pkg.FLAG_ASYNC)
        with torch.cuda.stream(other):
            other.wait_stream(torch.cuda.default_stream())
            again = pkg.cache_attend(*p.args(), flags=pkg.FLAG_ASYNC)
    finally:
        pkg._pack_attend = keep
    torch.cuda.synchronize()
    assert seen and all(ref.same(x, y) for g in (got, again) for x, y in zip(g, want))
    pkg.lib().b200attn_release_workspace()


# ---- commit --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D,token", [(64, False), (128, True), (100, False), (33, True), (1024, False)])
def test_commit(pkg, cuda, dtype, D, token):
    import torch
    B, H, T, S = 5, 3, 40, 100
    p = Problem(dtype, B, H, H, T, S, (0, 61, 100, 97, 30), D, "chain", token=token, seed=13)
    lists = torch.full((B, 35), -1, dtype=torch.int32, device="cuda")
    lists[0, :3] = torch.tensor([5, 5, 0], dtype=torch.int32)          # the same token twice
    lists[1] = torch.arange(34, -1, -1, dtype=torch.int32)             # backwards
    lists[2, :2] = 1                                                   # no room at all
    lists[3, :35] = 7                                                  # room for three
    lists[4, :6] = torch.tensor([1, 2, T, 3, -7, 4], dtype=torch.int32)   # ends at an index that names no token
    for accepted in (lists, None):
        for with_pos in (True, False):
            state = [p.K.clone(), p.V.clone(), torch.rand(B, H, S, device="cuda"), torch.zeros(B, H, S, dtype=torch.int32, device="cuda")]
            mine = [t.clone() for t in state]
            nxt = p.length + 1000 if with_pos else None
            W, P = (2, 3) if with_pos else (None, None)
            want = ref.commit(state[0], state[1], p.length, p.Kd, p.Vd, accepted, state[2] if with_pos else None, state[3] if with_pos else None, nxt)
            got = pkg.cache_commit(mine[0], mine[1], p.length, p.Kd, p.Vd, accepted, mine[2] if with_pos else None, mine[3] if with_pos else None, nxt)
            assert got.tolist() == want.tolist() and all(ref.same(x, y) for x, y in zip(mine, state))


# ---- weights ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", [
    # B, Hq, Hkv, T, S, lengths (behind the commit), D, A
    (1, 1, 1, 1, 1, (1,), 64, 0), (3, 8, 2, 7, 300, (300, 5, 0), 128, 4), (2, 6, 2, 20, 260, (129, 64), 64, 20), (2, 4, 4, 150, 400, (400, 150), 128, 0),
    (1, 14, 2, 9, 200, (199,), 256, 5), (2, 4, 2, 5, 130, (128, 3), 96, 3), (2, 4, 2, 5, 130, (128, 3), 100, 5), (1, 64, 1, 30, 140, (135,), 64, 9),
    (1, 200, 1, 3, 140, (135,), 64, 2), (1, 2, 1, 3, 70, (66,), 33, 2), (2, 8, 1, 200, 300, (270, 290), 128, 0),
    (1, 16, 2, 330, 700, (700,), 128, 0),        # 2640 rows a key head: in chunks, by TMA
    (1, 12, 1, 150, 300, (290,), 256, 150),      # 1800, gathered
    (1, 7, 1, 100, 300, (290,), 64, 0), (1, 40, 1, 30, 140, (135,), 64, 0), (2, 66, 2, 9, 140, (135, 9), 128, 0),
    (30, 8, 2, 6, 260, tuple(range(1, 260, 17)), 128, 6),   # short pairs: several a CTA
], ids=lambda s: "-".join(map(str, s[:5])) + f"-{s[6]}-{s[7]}")
def test_weights(pkg, cuda, shape, dtype):
    import torch
    B, Hq, Hkv, T, S, lengths, D, A = shape
    p = Problem(dtype, B, Hq, Hkv, T, S, lengths, D, "none", token=True, seed=14)
    lse = torch.rand(B, Hq, T, device="cuda") * 2 + math.log(S + 1)
    lse[:, 0, T // 2] = -math.inf
    accepted = None
    if A:
        accepted = torch.stack([torch.randperm(T, device="cuda")[:A] for _ in range(B)]).to(torch.int32)
        accepted[B - 1, A - 1] = -1
        if B > 4:
            accepted[2::5, 0] = -1     # sequences that have accepted nothing
    w = torch.rand(B, Hkv, S, device="cuda")
    w[0, 0, S - 1] = math.nan if lengths[0] < S else 0.5     # behind the last row: stays as it is
    want, bound = ref.weights(p.Q, p.K, p.length, lse, w, accepted)
    before = w.clone()
    got = pkg.cache_weights(p.Q, p.K, p.length, lse, w, accepted)
    assert got is w
    ok, worst = ref.close(w, want, bound)
    assert ok, worst
    again = pkg.cache_weights(p.Q, p.K, p.length, lse, before, accepted)
    assert ref.same(again, w)
    for b, n in enumerate(p.length.tolist()):
        assert ref.same(w[b, :, n:], before[b, :, n:])


# ---- evict -------------------------------------------------------------------------------------------------------------------
def eviction(B, H, S, D, dtype, seed, kind):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    K, V = (torch.randn(B, H, S, D, generator=g, device="cuda").to(getattr(torch, DT[dtype])) for _ in range(2))
    w = torch.rand(B, H, S, generator=g, device="cuda")
    if kind == "ties":
        w = (w * 4).floor() / 4
    elif kind == "zeros":
        w = torch.where(w < 0.7, torch.zeros_like(w), w)
        w[:, :, ::3] *= -0.0
    elif kind == "odd":
        w = (w - 0.5) * 10 ** ((w * 60).floor() - 30)
        w[:, :, 1::7], w[:, :, 2::11], w[:, :, 3::13], w[:, :, 4::17] = math.nan, math.inf, -math.inf, 1e-42
    pos = torch.rand(B, H, S, generator=g, device="cuda").argsort(dim=2).to(torch.int32)
    return K, V, w, pos


@pytest.mark.parametrize("into", [False, True], ids=["in-place", "into"])
@pytest.mark.parametrize("S,lengths,keep,sink,recent,D,dtype,kind", [
    (1, (1, 0), 1, 0, 0, 64, "bf16", "plain"), (40, (40, 33, 31, 7), 33, 2, 8, 64, "f32", "plain"), (100, (100, 50, 64, 65), 64, 0, 64, 100, "bf16", "ties"),
    (1500, (1500, 1025, 1024, 0), 1024, 4, 100, 8, "f16", "zeros"), (1100, (1100, 1099, 700), 32, 32, 0, 33, "bf16", "odd"), (2300, (2300, 2049), 2047, 1, 0, 64, "bf16", "ties"),
    (70, (70, 60), 80, 4, 8, 64, "bf16", "plain"), (5000, (4999, 4097), 1, 0, 0, 16, "bf16", "plain"), (40000, (39999, 12345), 20000, 4, 512, 8, "bf16", "zeros"),
])
def test_evict(pkg, cuda, S, lengths, keep, sink, recent, D, dtype, kind, into):
    import torch
    B, H = len(lengths), 2
    K, V, w, pos = eviction(B, H, S, D, dtype, S + keep, kind)
    length = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for with_pos in (True, False):
        nxt = torch.full_like(length, S) if with_pos else None
        room = min(keep, S) + 3
        def state():
            t = [K.clone(), V.clone(), w.clone(), pos.clone() if with_pos else None]
            o = None
            if into:
                o = (torch.full((B, H, room, D), 9.0, dtype=K.dtype, device="cuda"), torch.full((B, H, room, D), 9.0, dtype=K.dtype, device="cuda"),
                     torch.full((B, H, room), 9.0, device="cuda"), torch.full((B, H, room), 9, dtype=torch.int32, device="cuda") if with_pos else None)
            return t, o
        (a, ao), (b, bo) = state(), state()
        want, want_n = ref.evict(a[0], a[1], length, a[2], keep, sink, recent, a[3], nxt, ao)
        got, got_n = pkg.cache_evict(b[0], b[1], length, b[2], keep, sink, recent, b[3], nxt, bo)
        assert torch.equal(got.cpu(), want) and got_n.tolist() == want_n.tolist()
        for x, y in zip(list(a) + list(ao or []), list(b) + list(bo or [])):
            assert x is None or ref.same(x, y)


def test_evict_the_longest_capacity(pkg, cuda):
    import torch
    S = 524288
    K, V, w, pos = eviction(1, 1, S, 1, "bf16", 3, "zeros")
    n = torch.tensor([S - 1], dtype=torch.int32, device="cuda")
    for keep in (4000, S - 10):
        a, b = [t.clone() for t in (K, V, w, pos)], [t.clone() for t in (K, V, w, pos)]
        want, _ = ref.evict(a[0], a[1], n, a[2], keep, 4, 300, a[3], n)
        got, _ = pkg.cache_evict(b[0], b[1], n, b[2], keep, 4, 300, b[3], n)
        assert torch.equal(got.cpu(), want) and all(ref.same(x, y) for x, y in zip(a, b))


# ---- together ------------------------------------------------------------------------------------------------------------------
class Decoder:
    """A program that drafts trees: attend, accept, commit, accumulate, evict; `step` makes the package's calls, `check` follows in 64 bits."""

    def __init__(self, dtype, layers=2):
        import torch
        self.B, self.Hq, self.Hkv, self.T, self.S, self.D, self.A, self.keep, self.layers = 3, 6, 2, 12, 120, 64, 4, 96, layers
        self.td = getattr(torch, DT[dtype])
        z = lambda *s, d=None: torch.zeros(*s, dtype=d or self.td, device="cuda")
        self.cache = [(z(self.B, self.Hkv, self.S, self.D), z(self.B, self.Hkv, self.S, self.D), z(self.B, self.Hkv, self.S, d=torch.float32),
                       z(self.B, self.Hkv, self.S, d=torch.int32)) for _ in range(layers)]
        self.length, self.next_pos = z(self.B, d=torch.int32), z(self.B, d=torch.int32)
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(77)

    def inputs(self):
        import torch
        r = lambda h: torch.randn(self.B, self.T, h, self.D, generator=self.gen, device="cuda").to(self.td).transpose(1, 2)
        mask = torch.rand(self.B, self.T, self.T, generator=self.gen, device="cuda").lt(0.3).tril() | torch.eye(self.T, dtype=torch.bool, device="cuda")
        # the accepted path has to be a path: token 0 <- 1 <- .. as far as it goes
        acc = torch.full((self.B, self.A), -1, dtype=torch.int32, device="cuda")
        for b in range(self.B):
            n = int(torch.randint(0, self.A + 1, (1,), generator=self.gen, device="cuda"))
            acc[b, :n] = torch.arange(n, dtype=torch.int32)
            mask[b, : self.A, : self.A] = torch.ones(self.A, self.A, dtype=torch.bool, device="cuda").tril()
        return [(r(self.Hq), r(self.Hkv), r(self.Hkv)) for _ in range(self.layers)], mask.to(torch.uint8), acc

    def step(self, pkg, qkv, mask, acc, flags):
        outs = []
        for (K, V, W, P), (Q, Kd, Vd) in zip(self.cache, qkv):
            out, lse = pkg.cache_attend(Q, K, V, self.length, Kd, Vd, mask=mask, flags=flags)
            n = pkg.cache_commit(K, V, self.length, Kd, Vd, accepted=acc, weights=W, pos=P, next_pos=self.next_pos, flags=flags)
            nxt = self.next_pos + (n - self.length)
            pkg.cache_weights(Q, K, n, lse, W, accepted=acc, flags=flags)
            added = W.clone()
            kept, m = pkg.cache_evict(K, V, n, W, self.keep, sink=2, recent=10, pos=P, next_pos=nxt, flags=flags)
            outs.append((out, lse, added, kept))
        self.length.copy_(m)
        self.next_pos.copy_(nxt)
        return outs


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_the_operators_together(pkg, cuda, dtype):
    import torch
    d = Decoder(dtype)
    evicted = 0
    for _ in range(60):
        qkv, mask, acc = d.inputs()
        before = [tuple(t.clone() for t in c) for c in d.cache]
        length, nxt = d.length.clone(), d.next_pos.clone()
        outs = d.step(pkg, qkv, mask, acc, pkg.FLAG_ASYNC)
        torch.cuda.synchronize()
        for (K, V, W, P), (Q, Kd, Vd), (out, lse, added, kept), now in zip(before, qkv, outs, d.cache):
            want, want_lse, b_out, b_lse = ref.attend(Q, K, V, length, Kd, Vd, mask)
            assert ref.close(out, want, b_out)[0] and ref.close(lse, want_lse, b_lse)[0]
            n = ref.commit(K, V, length, Kd, Vd, acc, W, P, nxt).cuda()
            w, bound = ref.weights(Q, K, n, lse, W, acc)
            assert ref.close(added, w, bound)[0]
            W.copy_(added)            # the choice is exact on the numbers that it was made from
            want_kept, m = ref.evict(K, V, n, W, d.keep, 2, 10, P, nxt + (n - length))
            assert torch.equal(kept.cpu(), want_kept) and m.tolist() == d.length.tolist()
            for x, y in zip((K, V, W, P), now):
                for b in range(d.B):
                    assert ref.same(x[b], y[b])
            evicted += int((n > d.keep).sum())
            # every head holds each protected token exactly once
            for b in range(d.B):
                held = now[3][b, :, : int(m[b])].tolist()
                for row in held:
                    assert len(set(row)) == len(row) and set(range(min(2, int(m[b])))) <= set(row)
    assert evicted > 0


def test_captured_steps_replay_beside_eager_ones(pkg, cuda):
    """Two captured steps of different decoders replay on two streams at once, with eager calls of a third between: each has scratch of its own."""
    import torch
    decoders = [Decoder("bf16"), Decoder("bf16"), Decoder("bf16")]
    twins = [Decoder("bf16") for _ in decoders]
    steps = [d.inputs() for d in decoders]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs = [], []
    for d, s, (qkv, mask, acc) in zip(decoders, streams, steps):
        warm = Decoder("bf16")
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            warm.step(pkg, qkv, mask, acc, pkg.FLAG_ASYNC)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(d.step(pkg, qkv, mask, acc, pkg.FLAG_ASYNC))
        graphs.append(g)
    for i in range(40):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        last = decoders[2].step(pkg, *steps[2], pkg.FLAG_ASYNC)
    torch.cuda.synchronize()
    outs.append(last)
    for t, (qkv, mask, acc), got, d in zip(twins, steps, outs, decoders):
        for i in range(40):
            want = t.step(pkg, qkv, mask, acc, 0)
        assert all(ref.same(x, y) for w, o in zip(want, got) for x, y in zip(w, o))
        assert all(ref.same(x, y) for a, b in zip(t.cache, d.cache) for x, y in zip(a, b)) and t.length.tolist() == d.length.tolist()


def test_calls_from_threads_with_streams_of_their_own(pkg, cuda):
    import torch
    problems = [Problem("bf16", 4, 8, 2, 5 + i, 500, (500, 1, 0, 321), 128, "tree", seed=20 + i) for i in range(4)]
    want = [pkg.cache_attend(*p.args()) for p in problems]
    bad = []
    def work(i):
        s = torch.cuda.Stream()
        for _ in range(30):
            with torch.cuda.stream(s):
                got = pkg.cache_attend(*problems[i].args(), flags=pkg.FLAG_ASYNC)
            s.synchronize()
            if not all(ref.same(x, y) for x, y in zip(got, want[i])):
                bad.append(i)
    torch.cuda.synchronize()
    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad


def test_the_stream_argument(pkg, cuda):
    import torch
    s = torch.cuda.Stream()
    p = Problem("bf16", 2, 8, 2, 5, 300, (300, 41), 128, "tree", seed=30)
    want = pkg.cache_attend(*p.args())
    torch.cuda.synchronize()
    got = pkg.cache_attend(*p.args(), stream=s.cuda_stream, flags=pkg.FLAG_ASYNC)
    s.synchronize()
    assert ref.same(got[0], want[0]) and ref.same(got[1], want[1])


def test_wrappers_refuse(pkg, cuda):
    import torch
    p = Problem("bf16", 2, 8, 2, 5, 300, (300, 41), 128, "tree", seed=31)
    Q, K, V, n, Kd, Vd, m = p.args()
    w = torch.zeros(2, 2, 300, device="cuda")
    lse = torch.zeros(2, 8, 5, device="cuda")
    bad = [lambda: pkg.cache_attend(Q.float(), K, V, n), lambda: pkg.cache_attend(Q, K, V[:, :, :-1], n), lambda: pkg.cache_attend(Q, K, V, n.long()),
           lambda: pkg.cache_attend(Q, K, V, n[:1]), lambda: pkg.cache_attend(Q, K, V, n, Kd), lambda: pkg.cache_attend(Q, K, V, n, Kd, Vd, mask=m[:, :-1]),
           lambda: pkg.cache_attend(Q, K, V, n, Kd, Vd, mask=m.float()), lambda: pkg.cache_attend(Q, K, V, n, mask=m), lambda: pkg.cache_attend(Q[:, :7], K, V, n),
           lambda: pkg.cache_attend(Q, K, V, n, out=Q), lambda: pkg.cache_attend(Q.transpose(2, 3), K, V, n), lambda: pkg.cache_attend(Q, K, V, n.cpu()),
           lambda: pkg.cache_attend(Q, K, V, None), lambda: pkg.cache_attend(Q[:, :, :0], K, V, n),
           lambda: pkg.cache_commit(K, V, n, Kd, Vd, accepted=torch.zeros(2, 3, device="cuda")), lambda: pkg.cache_commit(K, V, n, K, V),
           lambda: pkg.cache_commit(K, V, n, Kd[:1], Vd), lambda: pkg.cache_commit(K, V, n, Kd, Vd, weights=w[:, :, :-1]),
           lambda: pkg.cache_weights(Q, K, n, lse[:, :, :-1], w), lambda: pkg.cache_weights(Q, K, n, lse, None),
           lambda: pkg.cache_evict(K, V, n, w, 0), lambda: pkg.cache_evict(K, V, n, w, 10, sink=4, recent=7), lambda: pkg.cache_evict(K, V, n, w, 10, into=(K, V, w, None)),
           lambda: pkg.cache_evict(K, V, n, w, 10, pos=n)]
    for call in bad:
        with pytest.raises(pkg.B200AttnError):
            call()
    torch.cuda.synchronize()
    check_attend(pkg, p)
