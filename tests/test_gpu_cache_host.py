"""Host side of the cache calls on the GPU: the share-out's size, which kernel took a call."""
import ctypes as C
import math

import pytest

import cache_ref as ref
from test_cache import attend_args
from test_gpu_cache import DT, Problem, check_attend, eviction

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 100, 124, 125, 128, 200, 256])
def test_the_work_on_the_cuda_cores_is_shared_out_over_ctas_that_run_at_once(pkg, cuda, D):
    """The workspace holds two slots a CTA, from which their number follows; that many fit the SMs' shared memory (16 rows of Q, 64 of K and of V, 64 x 20 weights)."""
    import torch
    sm = torch.cuda.get_device_properties(0)
    need = pkg.lib().b200attn_cache_attend_workspace(bytes(attend_args(pkg, head_d=D, dtype=pkg.F32, num_heads=1, num_kv_heads=1, batch_sz=1, Kd=0, Vd=0, mask=0)))
    slot = (16 * (D + 2) + 3) // 4 * 4
    ctas = (need - 32) // (2 * slot * 4)    # (and one entry of 8 words)
    assert ctas % sm.multi_processor_count == 0 and ctas > 0
    pitch = ((D + 3) // 4 | 1) * 4
    smem = ((16 + 128) * pitch + 64 * 20) * 4
    assert ctas // sm.multi_processor_count * (smem + 1024) <= sm.shared_memory_per_multiprocessor - 1024


@pytest.mark.parametrize("kind", ["ties", "zeros", "odd", "plain"])
@pytest.mark.parametrize("S,keep,lengths,sink,recent", [
    (4102, 4096, (4102, 4101, 4097, 4096), 4, 256),       # a step: rows of many threads, several of each
    (1500, 1468, (1500, 1499, 1469, 3), 2, 100),          # as many as are picked one by one
    (1500, 1469, (1500, 1470), 0, 1469),                  # all but a few are protected
    (33, 1, (33, 32, 2), 0, 0), (32, 1, (32, 31), 1, 0), (512, 511, (512,), 0, 0), (513, 512, (513,), 0, 512), (2048, 2016, (2048, 2047), 2000, 16),
])
def test_evict_picks_a_step_s_few_rows(pkg, cuda, S, keep, lengths, sink, recent, kind):
    """In place, up to 32 rows leaving: the least of several rows of a thread, the last of equal ones, NaN and infinities, a second row of the thread that lost one."""
    import torch
    B, H = len(lengths), 3
    K, V, w, pos = eviction(B, H, S, 16, "bf16", S + keep, kind)
    if kind == "plain":      # the rows that leave: all of one thread of 512, or neighbours
        w += 10.0
        w[:, 0, 7::512], w[:, 1, S // 2: S // 2 + 40] = 1.0, 2.0
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for with_pos in (True, False):
        nxt = torch.full_like(n, S) if with_pos else None
        a, b = ([K.clone(), V.clone(), w.clone(), pos.clone() if with_pos else None] for _ in range(2))
        before = pkg.launch_count()
        got, got_n = pkg.cache_evict(b[0], b[1], n, b[2], keep, sink, recent, b[3], nxt)
        assert pkg.launch_count() == before + 1
        want, want_n = ref.evict(a[0], a[1], n, a[2], keep, sink, recent, a[3], nxt)
        assert torch.equal(got.cpu(), want) and got_n.tolist() == want_n.tolist()
        assert all(x is None or ref.same(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("flags", [0, 2], ids=["any", "generic"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("B,Hq,Hkv,T,S,lengths,D,A", [
    (3, 8, 2, 7, 300, (300, 5, 0), 128, 4), (2, 4, 4, 150, 400, (400, 150), 128, 0), (1, 14, 2, 9, 200, (199,), 256, 5), (2, 4, 2, 5, 130, (128, 3), 100, 5),
    (1, 16, 2, 330, 700, (700,), 128, 0), (1, 12, 1, 150, 300, (290,), 256, 150), (2, 66, 2, 9, 140, (135, 9), 128, 0), (2, 8, 8, 30, 500, (500, 31), 192, 0),
])
def test_weights_by_either_kernel(pkg, cuda, B, Hq, Hkv, T, S, lengths, D, A, dtype, flags):
    """The kernel that a call names is the one that is meant to take it: 16 bits and whole 16 bytes a row on the tensor cores, all else, or on demand, on the CUDA cores."""
    import torch
    p = Problem(dtype, B, Hq, Hkv, T, S, lengths, D, "none", token=True, seed=70)
    lse = torch.rand(B, Hq, T, device="cuda") * 2 + math.log(S + 1)
    accepted = torch.stack([torch.randperm(T, device="cuda")[:A] for _ in range(B)]).to(torch.int32) if A else None
    w = torch.rand(B, Hkv, S, device="cuda")
    want, bound = ref.weights(p.Q, p.K, p.length, lse, w, accepted)
    pkg.cache_weights(p.Q, p.K, p.length, lse, w, accepted, flags=flags)
    assert pkg.last_path() == ("cache_generic" if dtype == "f32" or D % 8 or flags else "cache_tc")
    ok, worst = ref.close(w, want, bound)
    assert ok, worst


@pytest.mark.parametrize("what", ["Q", "K"])
def test_weights_of_unaligned_rows(pkg, cuda, what):
    import torch
    p = Problem("bf16", 2, 8, 2, 7, 300, (300, 5), 128, "none", seed=71)
    lse, w = torch.full((2, 8, 7), 6.0, device="cuda"), torch.zeros(2, 2, 300, device="cuda")
    t = getattr(p, what)
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
    flat[1:].view(t.shape).copy_(t)
    setattr(p, what, flat[1:].view(t.shape))
    want, bound = ref.weights(p.Q, p.K, p.length, lse, w)
    pkg.cache_weights(p.Q, p.K, p.length, lse, w)
    assert pkg.last_path() == "cache_generic" and ref.close(w, want, bound)[0]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("over", ["sequences", "heads", "rows"])
def test_keys_expanded_by_a_stride_of_0(pkg, cuda, dtype, over):
    """One sequence's states for all beams, one head's for all heads, one row for all rows: read as they are, on the CUDA cores."""
    import torch
    p = Problem(dtype, 3, 4, 2, 6, 200, (200, 130, 7), 64, "chain", seed=72)
    one = {"sequences": (slice(0, 1),), "heads": (slice(None), slice(0, 1)), "rows": (slice(None), slice(None), slice(0, 1))}[over]
    p.K, p.V = (t[one].expand(3, 2, 200, 64) for t in (p.K, p.V))
    check_attend(pkg, p)
    assert pkg.last_path() == "cache_generic"
    lse, w = torch.full((3, 4, 6), 6.0, device="cuda"), torch.zeros(3, 2, 200, device="cuda")
    want, bound = ref.weights(p.Q, p.K, p.length, lse, w)
    pkg.cache_weights(p.Q, p.K, p.length, lse, w)
    assert pkg.last_path() == "cache_generic" and ref.close(w, want, bound)[0]


def test_unaligned_views_go_to_the_cuda_cores(pkg, cuda):
    import torch
    p = Problem("bf16", 2, 8, 2, 5, 300, (300, 41), 128, "tree", seed=73)
    flat = torch.empty(p.V.numel() + 1, dtype=p.V.dtype, device="cuda")
    flat[1:].view(p.V.shape).copy_(p.V)
    p.V = flat[1:].view(p.V.shape)
    check_attend(pkg, p)
    assert pkg.last_path() == "cache_generic"


def test_a_list_without_entries_is_refused(pkg, cuda):
    """Not taken for no list, which accepts every token."""
    import torch
    p = Problem("bf16", 2, 8, 2, 5, 300, (100, 41), 128, "chain", seed=74)
    w, lse = torch.zeros(2, 2, 300, device="cuda"), torch.zeros(2, 8, 5, device="cuda")
    none = torch.empty(2, 0, dtype=torch.int32, device="cuda")
    K = p.K.clone()
    for call in (lambda: pkg.cache_commit(p.K, p.V, p.length, p.Kd, p.Vd, accepted=none, weights=w), lambda: pkg.cache_weights(p.Q, p.K, p.length, lse, w, accepted=none)):
        with pytest.raises(pkg.B200AttnError):
            call()
    assert ref.same(p.K, K) and float(w.abs().sum()) == 0


def test_a_cache_without_rows_to_evict_into_is_refused(pkg, cuda):
    """Not taken for no other cache, which evicts in place."""
    import torch
    K, V, w, pos = eviction(2, 2, 300, 64, "bf16", 75, "plain")
    before = [t.clone() for t in (K, V, w, pos)]
    n = torch.tensor([300, 120], dtype=torch.int32, device="cuda")
    for at, nxt in ((pos, n), (None, None)):
        into = (K[:, :, :0], V[:, :, :0], w[:, :, :0].contiguous(), pos[:, :, :0].contiguous() if at is not None else None)
        with pytest.raises(pkg.B200AttnError):
            pkg.cache_evict(K, V, n, w, 100, pos=at, next_pos=nxt, into=into)
    assert all(ref.same(x, y) for x, y in zip((K, V, w, pos), before))
