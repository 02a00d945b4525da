"""CPU tests of the cache entry points: the structures match the header, and what the host can refuse is refused before a device is looked at."""
import ctypes as C

import pytest

P = 1 << 20   # addresses that are never read


def view(name, ptr, B, H, L, D):
    return {name: ptr, name + "_b": H * L * D, name + "_h": L * D, name + "_l": D}


def attend_args(pkg, **over):
    B, Hq, Hkv, T, S, D = 2, 8, 4, 3, 40, 64
    f = {**view("Q", P, B, Hq, T, D), **view("K", 2 * P, B, Hkv, S, D), **view("V", 3 * P, B, Hkv, S, D), **view("Kd", 4 * P, B, Hkv, T, D),
         **view("Vd", 5 * P, B, Hkv, T, D), **view("out", 6 * P, B, Hq, T, D), "length": 7 * P, "lse": 8 * P, "mask": 9 * P, "mask_stride_b": T * T,
         "batch_sz": B, "num_heads": Hq, "num_kv_heads": Hkv, "len_new": T, "capacity": S, "head_d": D, "dtype": pkg.BF16}
    return fill(pkg.AttendArgs, f, over)


def commit_args(pkg, **over):
    B, H, T, S, D = 2, 4, 3, 40, 64
    f = {**view("K", 2 * P, B, H, S, D), **view("V", 3 * P, B, H, S, D), **view("Kd", 4 * P, B, H, T, D), **view("Vd", 5 * P, B, H, T, D), "length": 7 * P,
         "length_out": 8 * P, "accepted": 9 * P, "max_accepted": 2, "batch_sz": B, "num_kv_heads": H, "len_new": T, "capacity": S, "head_d": D, "dtype": pkg.F32}
    return fill(pkg.CommitArgs, f, over)


def weights_args(pkg, **over):
    B, Hq, Hkv, T, S, D = 2, 8, 4, 3, 40, 64
    f = {**view("Q", P, B, Hq, T, D), **view("K", 2 * P, B, Hkv, S, D), "length": 7 * P, "lse": 8 * P, "weights": 9 * P, "batch_sz": B, "num_heads": Hq,
         "num_kv_heads": Hkv, "len_new": T, "capacity": S, "head_d": D, "dtype": pkg.F16}
    return fill(pkg.WeightsArgs, f, over)


def evict_args(pkg, **over):
    B, H, S, D, So = 2, 4, 40, 64, 32
    f = {**view("K", 2 * P, B, H, S, D), **view("V", 3 * P, B, H, S, D), **view("K_out", 4 * P, B, H, So, D), **view("V_out", 5 * P, B, H, So, D), "weights": 6 * P,
         "pos": 7 * P, "length": 8 * P, "length_out": 9 * P, "kept": 10 * P, "keep": 30, "sink": 2, "recent": 8, "weights_out": 11 * P, "pos_out": 12 * P,
         "capacity_out": So, "batch_sz": B, "num_kv_heads": H, "capacity": S, "head_d": D, "dtype": pkg.BF16}
    return fill(pkg.EvictArgs, f, over)


def fill(cls, fields, over):
    a = cls(struct_size=C.sizeof(cls))
    for k, v in {**fields, **over}.items():
        setattr(a, k, v)
    return a


def status(pkg, name, a):
    return getattr(pkg.lib(), "b200attn_cache_" + name)(bytes(a)), pkg.lib().b200attn_last_error()


def test_structures_have_the_header_s_sizes(pkg):
    assert C.sizeof(pkg.AttendArgs) == 8 + 6 * 32 + 4 * 8 + 7 * 4 + 4 + 3 * 8 + 8
    assert C.sizeof(pkg.CommitArgs) == 8 + 4 * 32 + 3 * 8 + 8 + 3 * 8 + 6 * 4 + 8 + 8
    assert C.sizeof(pkg.WeightsArgs) == 8 + 2 * 32 + 3 * 8 + 8 + 8 + 7 * 4 + 4 + 8 + 8
    assert C.sizeof(pkg.EvictArgs) == 8 + 2 * 32 + 6 * 8 + 3 * 4 + 4 + 2 * 32 + 2 * 8 + 6 * 4 + 8 + 8
    for cls, pack in ((pkg.AttendArgs, pkg._pack_attend), (pkg.CommitArgs, pkg._pack_commit), (pkg.WeightsArgs, pkg._pack_weights), (pkg.EvictArgs, pkg._pack_evict)):
        a = cls.from_buffer_copy(pack(*range(1, len(cls._fields_))))
        assert [getattr(a, n) for n, _ in cls._fields_] == [C.sizeof(cls)] + list(range(1, len(cls._fields_)))


@pytest.mark.parametrize("over,word", [
    ({"struct_size": 8}, b"struct_size"), ({"Q": 0}, b"Q must be non-NULL"), ({"V": 0}, b"V must be"), ({"out": 0}, b"out must be"), ({"Kd": 0}, b"together"),
    ({"Kd": 0, "Vd": 0}, b"mask needs"), ({"length": 0}, b"length"), ({"length": P + 2}, b"aligned"), ({"lse": P + 1}, b"aligned"), ({"K": P + 1}, b"aligned"),
    ({"len_new": 0}, b"positive"), ({"capacity": 0}, b"positive"), ({"batch_sz": -1}, b"positive"), ({"num_heads": 6}, b"multiple"), ({"head_d": 257}, b"head_d"),
    ({"dtype": 7}, b"dtype"), ({"scale": -1.0}, b"scale"), ({"scale": float("nan")}, b"scale"), ({"scale": float("inf")}, b"scale"), ({"mask_stride_b": 4}, b"mask_stride_b"),
    ({"K_l": -64}, b"negative"), ({"out_l": 32}, b"overlap each other"), ({"out_h": 0}, b"overlap each other"), ({"out": P + 2}, b"overlap an input"), ({"out": 5 * P}, b"overlap an input"),
    ({"len_new": 1 << 30}, b"2^30"), ({"capacity": (1 << 30) + 1}, b"2^30"),
])
def test_attend_refuses(pkg, over, word):
    rc, msg = status(pkg, "attend", attend_args(pkg, **over))
    assert rc in (1, 5) and word in msg, msg


def test_attend_workspace_refuses(pkg):
    assert pkg.lib().b200attn_cache_attend_workspace(bytes(attend_args(pkg, head_d=0))) == 0
    assert b"positive" in pkg.lib().b200attn_last_error()


@pytest.mark.parametrize("over,word", [
    ({"struct_size": 8}, b"struct_size"), ({"K": 0}, b"K must be"), ({"Vd": 0}, b"Vd must be"), ({"length": 0}, b"length"), ({"length_out": 7 * P}, b"length_out"),
    ({"next_pos": 8 * P}, b"length_out"), ({"max_accepted": 0}, b"max_accepted"), ({"accepted": P + 2}, b"aligned"), ({"pos": P + 2}, b"aligned"), ({"dtype": -1}, b"dtype"),
    ({"batch_sz": 70000}, b"65535"), ({"head_d": 0}, b"positive"), ({"K_h": 64}, b"overlap each other"), ({"Kd": 3 * P}, b"must not overlap the cache"), ({"V": 3 * P + 2}, b"aligned"),
])
def test_commit_refuses(pkg, over, word):
    rc, msg = status(pkg, "commit", commit_args(pkg, **over))
    assert rc in (1, 5) and word in msg, msg


@pytest.mark.parametrize("over,word", [
    ({"struct_size": 8}, b"struct_size"), ({"Q": 0}, b"Q must be"), ({"lse": 0}, b"lse"), ({"weights": 0}, b"weights"), ({"weights": P + 1}, b"aligned"), ({"num_heads": 7}, b"multiple"),
    ({"head_d": 264}, b"head_d"), ({"accepted": P, "max_accepted": -1}, b"max_accepted"), ({"scale": -0.5}, b"scale"), ({"num_kv_heads": 0}, b"positive"),
    ({"num_heads": 140000, "num_kv_heads": 70000}, b"65535"),
])
def test_weights_refuses(pkg, over, word):
    rc, msg = status(pkg, "weights", weights_args(pkg, **over))
    assert rc in (1, 5) and word in msg, msg


@pytest.mark.parametrize("over,word", [
    ({"struct_size": 8}, b"struct_size"), ({"V": 0}, b"V must be"), ({"kept": 0}, b"kept"), ({"weights": 0}, b"weights"), ({"keep": 0}, b"keep"), ({"keep": 9}, b"keep"),
    ({"sink": -1}, b"keep"), ({"V_out": 0}, b"together"), ({"pos_out": 0}, b"together"), ({"K_out": 0, "V_out": 0, "weights_out": 0}, b"together"), ({"pos": 0}, b"together"),
    ({"capacity_out": 29}, b"capacity_out"), ({"K_out": 2 * P + 128}, b"must not overlap"), ({"weights_out": 6 * P}, b"must not overlap"), ({"length_out": 8 * P}, b"length_out"),
    ({"capacity": 1 << 20}, b"rows"), ({"kept": P + 2}, b"aligned"), ({"head_d": -1}, b"positive"),
])
def test_evict_refuses(pkg, over, word):
    rc, msg = status(pkg, "evict", evict_args(pkg, **over))
    assert rc in (1, 5) and word in msg, msg


def test_null_arguments_are_refused(pkg):
    for name in ("attend", "commit", "weights", "evict"):
        assert getattr(pkg.lib(), "b200attn_cache_" + name)(None) == 1 and b"NULL" in pkg.lib().b200attn_last_error()


def test_python_wrappers_refuse_cpu_tensors(pkg):
    import torch
    K = torch.zeros(1, 1, 4, 8)
    n = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: pkg.cache_attend(K, K, K, n), lambda: pkg.cache_commit(K, K, n, K, K), lambda: pkg.cache_weights(K, K, n, n, n), lambda: pkg.cache_evict(K, K, n, n, 1)):
        with pytest.raises(pkg.B200AttnError):
            call()
