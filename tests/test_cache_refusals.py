"""CPU tests of what the cache entry points refuse, beside test_cache.py."""
import pytest

from test_cache import attend_args, status, weights_args


@pytest.mark.parametrize("name,args", [("attend", attend_args), ("weights", weights_args)])
def test_a_scale_that_overflows_in_units_of_log2_e_is_refused(pkg, name, args):
    rc, msg = status(pkg, name, args(pkg, scale=2.4e38))   # times log2 e: beyond fp32
    assert rc == 1 and b"scale" in msg, msg


def test_rope_k_refuses_what_it_would_misread(pkg):
    import torch
    for X in (torch.zeros(1, 2, 3, 8), torch.zeros(2, 3, 8), torch.zeros(1, 2, 3, 8, dtype=torch.float64), torch.zeros(1, 3, 2, 8).transpose(1, 2)):
        with pytest.raises(pkg.B200AttnError):
            pkg.rope_k(X)


@pytest.mark.parametrize("cls,pack,field,value", [("AttendArgs", "_pack_attend", "capacity", 1 << 31), ("EvictArgs", "_pack_evict", "keep", 1 << 31), ("WeightsArgs", "_pack_weights", "flags", -1),
                                                  ("CommitArgs", "_pack_commit", "max_accepted", 0.5)])
def test_numbers_that_a_field_does_not_hold_are_refused(pkg, cls, pack, field, value):
    names = [n for n, _ in getattr(pkg, cls)._fields_][1:]
    with pytest.raises(pkg.B200AttnError):
        getattr(pkg, pack)(*(value if n == field else 0 for n in names))


def test_a_scale_beyond_fp32_arrives_as_infinity_and_is_refused(pkg):
    names = [n for n, _ in pkg.AttendArgs._fields_][1:]
    a = attend_args(pkg)
    packed = pkg._pack_attend(*((1e39 if n == "scale" else getattr(a, n) or 0) for n in names))
    assert pkg.lib().b200attn_cache_attend(packed) == 1 and b"scale" in pkg.lib().b200attn_last_error()
