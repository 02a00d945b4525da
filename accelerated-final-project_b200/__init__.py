"""b200attn: thin ctypes binding of lib/libb200attn.so (the C ABI of include/b200attn.h).

This module is host-side convenience for the tests and the benchmark: it passes torch device
pointers to the C entry points.  All arithmetic is in the CUDA library; there is no fallback, and
loading fails when the shared library has not been built.
"""
import ctypes as C
import os
import struct

_HERE = os.path.dirname(os.path.abspath(__file__))
# B200ATTN_LIB names another build of the same library (a profiling build, an older build to compare with)
LIB_PATH = os.environ.get("B200ATTN_LIB") or os.path.join(_HERE, "lib", "libb200attn.so")

F32, BF16, F16 = 0, 1, 2
PE_NONE, PE_ROPE_INTERLEAVED, PE_ROPE_HALF, PE_SINUSOIDAL, PE_ROPE_Q_ONLY, PE_ROPE_HALF_Q_ONLY = 0, 1, 2, 3, 4, 5
FLAG_ASYNC, FLAG_FORCE_GENERIC, FLAG_FORCE_TWO_PASS, FLAG_PREFER_ONE_KERNEL, FLAG_NO_OVERLAP, FLAG_TWO_KERNELS = 1, 2, 4, 8, 16, 32
OPT_SCORE_SCRATCH_MB, OPT_SPIN_LIMIT = 1, 2
OK = 0

# every symbol include/b200attn.h declares (checked by the CPU test-suite against the header)
DROP_IN_SYMBOLS = (
    "attention_forward_optimized", "attention_forward_bf16", "attention_forward_rope_fused_v2",
    "attention_forward_rope_fused", "attention_forward_rope_fused_v7_hybrid", "attention_forward_rope_bf16",
    "attention_forward_rope_bf16_v7", "attention_forward_sinusoidal_fused", "attention_forward_sinusoidal_bf16",
)


class Args(C.Structure):
    _fields_ = [
        ("struct_size", C.c_size_t),
        ("Q", C.c_void_p), ("K", C.c_void_p), ("V", C.c_void_p), ("out", C.c_void_p),
        ("batch_sz", C.c_int), ("num_heads", C.c_int), ("len_q", C.c_int), ("len_k", C.c_int), ("head_d", C.c_int),
        ("dtype", C.c_int), ("pe", C.c_int), ("rotary_dim", C.c_int), ("rope_base", C.c_float),
        ("cos_cache", C.c_void_p), ("sin_cache", C.c_void_p),
        ("stream", C.c_void_p), ("flags", C.c_uint),
    ]


_ARGS_SIZE = C.sizeof(Args)


def _with_views(*fields):
    """Field list of a b200attn_*_args: a bare name is a b200attn_view (pointer and strides of sequence, head and row)."""
    out = [("struct_size", C.c_size_t)]
    for f in fields:
        out += [(f, C.c_void_p), (f + "_b", C.c_longlong), (f + "_h", C.c_longlong), (f + "_l", C.c_longlong)] if isinstance(f, str) else [f]
    return out


class AttendArgs(C.Structure):
    _fields_ = _with_views("Q", "K", "V", "Kd", "Vd", "out", ("lse", C.c_void_p), ("length", C.c_void_p), ("mask", C.c_void_p),
                           ("mask_stride_b", C.c_longlong), ("batch_sz", C.c_int), ("num_heads", C.c_int), ("num_kv_heads", C.c_int),
                           ("len_new", C.c_int), ("capacity", C.c_int), ("head_d", C.c_int), ("dtype", C.c_int), ("scale", C.c_float),
                           ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t), ("stream", C.c_void_p), ("flags", C.c_uint))


class CommitArgs(C.Structure):
    _fields_ = _with_views("K", "V", "Kd", "Vd", ("length", C.c_void_p), ("length_out", C.c_void_p), ("accepted", C.c_void_p),
                           ("max_accepted", C.c_int), ("weights", C.c_void_p), ("pos", C.c_void_p), ("next_pos", C.c_void_p),
                           ("batch_sz", C.c_int), ("num_kv_heads", C.c_int), ("len_new", C.c_int), ("capacity", C.c_int), ("head_d", C.c_int),
                           ("dtype", C.c_int), ("stream", C.c_void_p), ("flags", C.c_uint))


class WeightsArgs(C.Structure):
    _fields_ = _with_views("Q", "K", ("length", C.c_void_p), ("lse", C.c_void_p), ("accepted", C.c_void_p), ("max_accepted", C.c_int),
                           ("weights", C.c_void_p), ("batch_sz", C.c_int), ("num_heads", C.c_int), ("num_kv_heads", C.c_int),
                           ("len_new", C.c_int), ("capacity", C.c_int), ("head_d", C.c_int), ("dtype", C.c_int), ("scale", C.c_float),
                           ("stream", C.c_void_p), ("flags", C.c_uint))


class EvictArgs(C.Structure):
    _fields_ = _with_views("K", "V", ("weights", C.c_void_p), ("pos", C.c_void_p), ("length", C.c_void_p), ("next_pos", C.c_void_p),
                           ("length_out", C.c_void_p), ("kept", C.c_void_p), ("keep", C.c_int), ("sink", C.c_int), ("recent", C.c_int),
                           "K_out", "V_out", ("weights_out", C.c_void_p), ("pos_out", C.c_void_p), ("capacity_out", C.c_int),
                           ("batch_sz", C.c_int), ("num_kv_heads", C.c_int), ("capacity", C.c_int), ("head_d", C.c_int), ("dtype", C.c_int),
                           ("stream", C.c_void_p), ("flags", C.c_uint))


def _packer(cls):
    """Fills a `cls` from values in the order of its fields, as bytes (a tenth of the time that ctypes takes to fill the structure)."""
    code = {C.c_size_t: "N", C.c_void_p: "P", C.c_longlong: "q", C.c_int: "i", C.c_float: "f", C.c_uint: "I"}
    packed = struct.Struct("@" + "".join(code[t] for _, t in cls._fields_))
    size = C.sizeof(cls)
    tail = bytes(size - packed.size)   # the structure's own alignment

    def pack(*values):
        try:
            return packed.pack(size, *values) + tail
        except (struct.error, OverflowError) as e:   # a number that its field does not hold
            _refuse(f"{cls.__name__}: {e}")
    return pack


_pack_attend, _pack_commit, _pack_weights, _pack_evict = (_packer(c) for c in (AttendArgs, CommitArgs, WeightsArgs, EvictArgs))


class B200AttnError(RuntimeError):
    def __init__(self, status, message):
        super().__init__(f"b200attn status {status}: {message}")
        self.status = status


_lib = None


def lib():
    """The loaded shared library (raises if it has not been built: there is no CPU path)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise FileNotFoundError(f"{LIB_PATH} is missing: run `python accelerated-final-project_b200/build.py`")
        L = C.CDLL(LIB_PATH)
        five = [C.c_int] * 5
        for name in ("attention_forward_optimized", "attention_forward_bf16", "attention_forward_rope_fused_v2",
                     "attention_forward_rope_bf16", "attention_forward_sinusoidal_fused", "attention_forward_sinusoidal_bf16"):
            getattr(L, name).argtypes = [C.c_void_p] * 4 + five
            getattr(L, name).restype = None
        L.attention_forward_rope_fused.argtypes = [C.c_void_p] * 6 + five
        L.attention_forward_rope_fused.restype = None
        for name in ("attention_forward_rope_fused_v7_hybrid", "attention_forward_rope_bf16_v7"):
            getattr(L, name).argtypes = [C.c_void_p] * 4 + five + [C.c_int]
            getattr(L, name).restype = None
        L.b200attn_forward_ex.argtypes = [C.POINTER(Args)]
        L.b200attn_forward_ex.restype = C.c_int
        L.b200attn_forward_many.argtypes = [C.POINTER(Args), C.c_int]
        L.b200attn_forward_many.restype = C.c_int
        L.b200attn_forward_host.argtypes = [C.POINTER(Args)]
        L.b200attn_forward_host.restype = C.c_int
        L.b200attn_forward_sharded.argtypes = [C.POINTER(Args), C.c_int, C.POINTER(C.c_int)] + \
            [C.POINTER(C.c_void_p)] * 4 + [C.POINTER(C.c_int)]
        L.b200attn_forward_sharded.restype = C.c_int
        L.b200attn_shard_ranges.argtypes = [C.c_longlong, C.c_int, C.POINTER(C.c_longlong), C.POINTER(C.c_longlong)]
        L.b200attn_shard_ranges.restype = None
        L.b200attn_last_error.restype = C.c_char_p
        L.b200attn_last_path.restype = C.c_char_p
        L.b200attn_launch_count.restype = C.c_ulonglong
        L.b200attn_version.restype = C.c_char_p
        L.b200attn_release_workspace.restype = None
        L.b200attn_forward_static.argtypes = [C.c_void_p] * 4 + [C.c_int] * 5 + [C.c_void_p]
        L.b200attn_forward_static.restype = C.c_int
        L.b200attn_static_last_error.restype = C.c_char_p
        L.b200attn_synth_fill.argtypes = [C.c_void_p, C.c_longlong, C.c_ulonglong, C.c_ulonglong, C.c_longlong,
                                          C.c_int, C.c_int, C.c_void_p]
        L.b200attn_synth_fill.restype = C.c_int
        L.b200attn_rope_k.argtypes = [C.c_void_p, C.c_void_p] + [C.c_int] * 7 + [C.c_float, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p]
        L.b200attn_rope_k.restype = C.c_int
        for name in ("attend", "commit", "weights", "evict"):
            getattr(L, "b200attn_cache_" + name).argtypes = [C.c_char_p]   # a filled structure's bytes
            getattr(L, "b200attn_cache_" + name).restype = C.c_int
        L.b200attn_cache_attend_workspace.argtypes = [C.c_char_p]
        L.b200attn_cache_attend_workspace.restype = C.c_size_t
        L.b200attn_set_option.argtypes = [C.c_int, C.c_longlong]
        L.b200attn_set_option.restype = C.c_int
        L.b200attn_debug_kernel_times.argtypes = [C.c_int, C.POINTER(C.c_double)]
        L.b200attn_debug_kernel_times.restype = C.c_int
        L.b200attn_debug_lost_arrival.argtypes = [C.c_uint, C.c_uint]
        L.b200attn_debug_lost_arrival.restype = None
        _lib = L
    return _lib


def make_args(Q, K, V, out, B, H, Lq, Lk, D, dtype, pe=PE_NONE, rotary_dim=0, rope_base=0.0,
              cos_cache=None, sin_cache=None, stream=None, flags=0):
    """Q, K, V, out, cos_cache, sin_cache are raw addresses (ints)."""
    return Args(C.sizeof(Args), Q, K, V, out, B, H, Lq, Lk, D, dtype, pe, rotary_dim, rope_base,
                cos_cache, sin_cache, stream, flags)


_torch = _DTYPES = None


def _with_torch():
    """torch, imported on first use (the binding itself does not need it)."""
    global _torch, _DTYPES
    if _torch is None:
        import torch
        _DTYPES = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}
        _torch = torch
    return _torch


def dtype_of(t):
    _with_torch()
    return _DTYPES[t.dtype]


def check(status):
    if status != OK:
        raise B200AttnError(status, lib().b200attn_last_error().decode())


_INVALID_ARG = 1


def _refuse(message):
    raise B200AttnError(_INVALID_ARG, message)


def forward(Q, K, V, out=None, pe=PE_NONE, rotary_dim=0, rope_base=0.0, cos_cache=None, sin_cache=None,
            stream=None, flags=0):
    """Attention forward on torch CUDA tensors Q [B,H,Lq,D], K/V [B,H,Lk,D] (float32 or bfloat16,
    contiguous) through b200attn_forward_ex.  Returns `out`."""
    # (a short call is bound by this function: 10.5 us of interpreter per call, against 10 us of GPU, with a torch.cuda.device block
    # around every call, a Stream object made to read its handle and the imports and tables set up again; 4 x 64 x 64, head_d 512)
    torch = _torch or _with_torch()
    assert Q.is_cuda and K.is_cuda and V.is_cuda and Q.is_contiguous() and K.is_contiguous() and V.is_contiguous()
    B, H, Lq, D = Q.shape
    dtype = _DTYPES[Q.dtype]
    if out is None:
        out = torch.empty_like(Q)
    dev = Q.get_device()
    if stream is None:
        stream = torch._C._cuda_getCurrentRawStream(dev)
    a = Args(_ARGS_SIZE, Q.data_ptr(), K.data_ptr(), V.data_ptr(), out.data_ptr(), B, H, Lq, K.shape[2], D, dtype, pe, rotary_dim,
             rope_base, cos_cache.data_ptr() if cos_cache is not None else None,
             sin_cache.data_ptr() if sin_cache is not None else None, stream, flags)
    fn = (_lib or lib()).b200attn_forward_ex
    if dev == torch.cuda.current_device():
        status = fn(C.byref(a))
    else:
        with torch.cuda.device(dev):
            status = fn(C.byref(a))
    if status != OK:
        check(status)
    return out


def args_for(Q, K, V, out, pe=PE_NONE, rotary_dim=0, rope_base=0.0, stream=None, flags=0):
    """A filled b200attn_args for torch CUDA tensors (for forward_many)."""
    import torch
    B, H, Lq, D = Q.shape
    if stream is None:
        stream = torch.cuda.current_stream(Q.device).cuda_stream
    return make_args(Q.data_ptr(), K.data_ptr(), V.data_ptr(), out.data_ptr(), B, H, Lq, K.shape[2], D,
                     dtype_of(Q), pe, rotary_dim, rope_base, None, None, stream, flags)


def kernel_times(enable, collect=False):
    """Per-kernel timing of the two-kernel bf16 path (b200attn_debug_kernel_times).  With collect,
    returns {"scores_encode": (ms, launches), "scores": (...), "pv": (...)} for the launches recorded
    since the last collection."""
    out = (C.c_double * 6)() if collect else None
    check(lib().b200attn_debug_kernel_times(1 if enable else 0, out))
    if not collect:
        return None
    return {k: (out[i], int(out[3 + i])) for i, k in enumerate(("scores_encode", "scores", "pv"))}


def forward_many(arg_list):
    """Enqueues a list of b200attn_args through one b200attn_forward_many call."""
    arr = (Args * len(arg_list))(*arg_list)
    check(lib().b200attn_forward_many(arr, len(arg_list)))


def forward_host(Q, K, V, out, pe=PE_NONE, rotary_dim=0, rope_base=0.0, flags=0):
    """Same through b200attn_forward_host: Q, K, V, out are HOST torch tensors (pinned or pageable)."""
    import torch
    B, H, Lq, D = Q.shape
    Lk = K.shape[2]
    dtype = dtype_of(Q)
    a = make_args(Q.data_ptr(), K.data_ptr(), V.data_ptr(), out.data_ptr(), B, H, Lq, Lk, D, dtype, pe, rotary_dim,
                  rope_base, None, None, None, flags)
    check(lib().b200attn_forward_host(C.byref(a)))
    return out


def rope_k(X, out=None, pairing=PE_ROPE_INTERLEAVED, rotary_dim=0, rope_base=0.0, pos0=0, cos_cache=None, sin_cache=None, stream=None):
    """RoPE(X) for a torch CUDA tensor [B,H,L,D] (float32, bfloat16 or float16, contiguous) through b200attn_rope_k.  Returns `out`."""
    torch = _torch or _with_torch()
    if X.dim() != 4 or X.dtype not in _DTYPES or not X.is_cuda or not X.is_contiguous():
        _refuse("X must be a contiguous 4-dimensional float32, bfloat16 or float16 CUDA tensor [B, heads, rows, D]")
    B, H, L, D = X.shape
    if out is None:
        out = torch.empty_like(X)
    elif out.shape != X.shape or out.dtype is not X.dtype or out.device != X.device or not out.is_contiguous():
        _refuse(f"out must be a contiguous {X.dtype} tensor of shape {tuple(X.shape)} on {X.device}")
    for c in (cos_cache, sin_cache):
        if c is not None and (c.dtype is not torch.float32 or c.device != X.device or not c.is_contiguous() or c.numel() < (pos0 + L) * (rotary_dim or D)):
            _refuse(f"cos_cache and sin_cache must be contiguous float32 tensors [{pos0 + L}, {rotary_dim or D}] on {X.device}")
    if stream is None:
        stream = torch.cuda.current_stream(X.device).cuda_stream
    with torch.cuda.device(X.device):
        check(lib().b200attn_rope_k(X.data_ptr(), out.data_ptr(), B, H, L, D, _DTYPES[X.dtype], pairing, rotary_dim,
                                    rope_base, pos0, cos_cache.data_ptr() if cos_cache is not None else None,
                                    sin_cache.data_ptr() if sin_cache is not None else None, stream))
    return out


# ---- a key/value cache ----------------------------------------------------------------------------------------------

# (a short call is bound by these functions, as above: 22 us of which the two launches take 5, one token over 777 cached rows, with the checks
# spread over more attribute look-ups; shapes are compared as tuples, and what a function has allocated itself is not checked)
def _view(t, name, shape, dtype, dev):
    """(address, strides of sequence, head and row) of a [B, heads, rows, D] tensor, after its checks."""
    if t.dtype is dtype and t.get_device() == dev and t.shape == shape:
        s = t.stride()
        if s[3] == 1 or shape[3] == 1:
            return t.data_ptr(), s[0], s[1], s[2]
        _refuse(f"the last dimension of {name} must be contiguous")
    _refuse(f"{name} must be a {dtype} tensor of shape {tuple(shape)} on device {dev}, got {t.dtype}, {tuple(t.shape)} on {t.device}")


def _dense(t, name, shape, dtype, dev):
    """Address of a dense tensor (0 for None), after its checks."""
    if t is None:
        return 0
    if t.dtype is dtype and t.get_device() == dev and t.shape == shape and t.is_contiguous():
        return t.data_ptr()
    _refuse(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on device {dev}, got {t.dtype}, {tuple(t.shape)} on {t.device}")


def _cache_shape(K):
    torch = _torch or _with_torch()
    shape, dev = K.shape, K.get_device()
    if dev < 0 or len(shape) != 4 or K.dtype not in _DTYPES:
        _refuse("the cache must be a 4-dimensional float32, bfloat16 or float16 CUDA tensor [B, heads, rows, D]")
    return torch, dev, shape


def _call_on(dev, fn, packed):
    if dev == _torch._C._cuda_getDevice():
        status = fn(packed)
    else:
        with _torch.cuda.device(dev):
            status = fn(packed)
    if status != OK:
        check(status)


def _elsewhere(stream, dev):
    """The stream to allocate on and to enter where `stream` is given and is not the current one, else None: memory that torch hands out belongs to
    the stream that was current then, and may be handed out again as soon as that stream is done with it."""
    torch = _torch
    if stream is None or stream == torch._C._cuda_getCurrentRawStream(dev):
        return None
    return torch.cuda.ExternalStream(stream, device=dev) if stream else torch.cuda.default_stream(dev)


_attend_ws = {}   # bytes of workspace by the sizes they depend on
_NO_VIEWS = (0,) * 8


def cache_attend(Q, K, V, length, Kd=None, Vd=None, mask=None, scale=0.0, out=None, lse=None, stream=None, flags=0):
    """Attention of T new tokens, Q [B, Hq, T, D], over the first length[b] rows of a cache K, V [B, Hkv, S, D] and over the new tokens' own Kd, Vd
    [B, Hkv, T, D] where mask [B or 1, T, T] (uint8 or bool) is not 0; without a mask token t sees the tokens u <= t; without Kd and Vd the cache alone
    (an encoder's states).  Tensors may be views whose last dimension is contiguous.  Returns (out [B, Hq, T, D], lse [B, Hq, T] float32)
    (b200attn_cache_attend).  The workspace comes from torch's allocator: calls on different streams do not share it."""
    torch, dev, k_shape = _cache_shape(K)
    if stream is not None and (at := _elsewhere(stream, dev)) is not None:
        with torch.cuda.stream(at):
            return cache_attend(Q, K, V, length, Kd, Vd, mask, scale, out, lse, None, flags)
    q_shape, dtype = Q.shape, K.dtype
    if len(q_shape) != 4:
        _refuse("Q must be a 4-dimensional tensor [B, heads, new tokens, D]")
    B, Hkv, S, D = k_shape
    _, Hq, T, _ = q_shape
    q = _view(Q, "Q", (B, Hq, T, D), dtype, dev)
    if out is None:
        out = torch.empty_like(Q)
        s = out.stride()
        o = out.data_ptr(), s[0], s[1], s[2]
    else:
        o = _view(out, "out", q_shape, dtype, dev)
    if lse is None:
        lse = Q.new_empty((B, Hq, T), dtype=torch.float32)
        lse_at = lse.data_ptr()
    else:
        lse_at = _dense(lse, "lse", (B, Hq, T), torch.float32, dev)
    if Kd is not None and Vd is not None:
        d_shape = (B, Hkv, T, D)
        d = *_view(Kd, "Kd", d_shape, dtype, dev), *_view(Vd, "Vd", d_shape, dtype, dev)
    elif Kd is not None or Vd is not None:
        _refuse("Kd and Vd must be given together")
    else:
        d = _NO_VIEWS
    mask_at = mask_b = 0
    if mask is not None:
        m_shape = mask.shape
        if mask.dtype not in (torch.uint8, torch.bool) or mask.get_device() != dev or not mask.is_contiguous() or \
                m_shape not in ((B, T, T), (1, T, T), (T, T)):
            _refuse(f"mask must be a contiguous uint8 or bool tensor of shape {(B, T, T)}, {(1, T, T)} or {(T, T)} on device {dev}")
        mask_at, mask_b = mask.data_ptr(), T * T if len(m_shape) == 3 and m_shape[0] == B else 0
    L = _lib or lib()
    filled = *q, *_view(K, "K", k_shape, dtype, dev), *_view(V, "V", k_shape, dtype, dev), *d, *o, lse_at, _dense(length, "length", (B,), torch.int32, dev), \
        mask_at, mask_b, B, Hq, Hkv, T, S, D, _DTYPES[dtype], scale
    # the size goes by the shapes and the device: kept per combination of them, it costs no second call
    key = dev, dtype, q_shape, k_shape, Kd is None, mask is None, flags
    need = _attend_ws.get(key)
    if need is None:
        with torch.cuda.device(dev):
            need = L.b200attn_cache_attend_workspace(_pack_attend(*filled, 0, 0, 0, flags))
        if need == 0 and (message := L.b200attn_last_error().decode()):
            _refuse(message)
        if len(_attend_ws) >= 4096:
            _attend_ws.clear()
        _attend_ws[key] = need
    ws = Q.new_empty((need + 1) // 2) if need else None   # (elements of 2 bytes at least)
    _call_on(dev, L.b200attn_cache_attend, _pack_attend(*filled, ws.data_ptr() if need else 0, need, torch._C._cuda_getCurrentRawStream(dev), flags))
    return out, lse


def cache_commit(K, V, length, Kd, Vd, accepted=None, weights=None, pos=None, next_pos=None, stream=None, flags=0):
    """The accepted ones of T new tokens (accepted [B, A] int32, padded with -1; None: all) become rows of the cache from row length[b] on:
    K, V [B, Hkv, S, D] are written from Kd, Vd [B, Hkv, T, D], weights [B, Hkv, S] with 0, pos [B, Hkv, S] with next_pos[b] + i.  Returns the new
    lengths [B] (int32); `length` stays (b200attn_cache_commit).  Tokens that the cache has no room for are dropped: see the new lengths."""
    torch, dev, k_shape = _cache_shape(K)
    B, Hkv, S, D = k_shape
    if stream is not None and (at := _elsewhere(stream, dev)) is not None:
        with torch.cuda.stream(at):
            return cache_commit(K, V, length, Kd, Vd, accepted, weights, pos, next_pos, None, flags)
    if Kd.dim() != 4 or (accepted is not None and accepted.dim() != 2):
        _refuse("Kd must be [B, heads, new tokens, D] and accepted [B, most accepted tokens]")
    T, dtype, i32 = Kd.shape[2], K.dtype, torch.int32
    A = 0 if accepted is None else accepted.shape[1]
    if accepted is not None and A == 0:   # (its address would be that of no list)
        _refuse("accepted must have room for one token of a sequence at least; -1 names none")
    n = _dense(length, "length", (B,), i32, dev)
    if n == 0:
        _refuse("length must be given")
    out = torch.empty_like(length)   # (half of the time of torch.empty)
    stream = torch._C._cuda_getCurrentRawStream(dev)
    d_shape = (B, Hkv, T, D)
    packed = _pack_commit(*_view(K, "K", k_shape, dtype, dev), *_view(V, "V", k_shape, dtype, dev), *_view(Kd, "Kd", d_shape, dtype, dev),
                          *_view(Vd, "Vd", d_shape, dtype, dev), n, out.data_ptr(),
                          _dense(accepted, "accepted", (B, A), i32, dev), A, _dense(weights, "weights", (B, Hkv, S), torch.float32, dev),
                          _dense(pos, "pos", (B, Hkv, S), i32, dev), _dense(next_pos, "next_pos", (B,), i32, dev), B, Hkv, T, S, D, _DTYPES[dtype],
                          stream, flags)
    _call_on(dev, (_lib or lib()).b200attn_cache_commit, packed)
    return out


def cache_weights(Q, K, length, lse, weights, accepted=None, scale=0.0, stream=None, flags=0):
    """Adds to weights [B, Hkv, S] the attention weight that each cached row had from the accepted tokens, which are the cache's last rows by now:
    Q [B, Hq, T, D] and lse [B, Hq, T] are those of the cache_attend call, `length` and `accepted` those after and of cache_commit (where that had no
    room for all, a list that ends in front of those it dropped).  Returns `weights` (b200attn_cache_weights)."""
    torch, dev, k_shape = _cache_shape(K)
    B, Hkv, S, D = k_shape
    if stream is not None and (at := _elsewhere(stream, dev)) is not None:
        with torch.cuda.stream(at):
            return cache_weights(Q, K, length, lse, weights, accepted, scale, None, flags)
    if Q.dim() != 4 or (accepted is not None and accepted.dim() != 2):
        _refuse("Q must be [B, heads, new tokens, D] and accepted [B, most accepted tokens]")
    Hq, T, dtype = Q.shape[1], Q.shape[2], K.dtype
    A = 0 if accepted is None else accepted.shape[1]
    if accepted is not None and A == 0:   # (its address would be that of no list)
        _refuse("accepted must have room for one token of a sequence at least; -1 names none")
    stream = torch._C._cuda_getCurrentRawStream(dev)
    if length is None or lse is None or weights is None:
        _refuse("length, lse and weights must be given")
    packed = _pack_weights(*_view(Q, "Q", (B, Hq, T, D), dtype, dev), *_view(K, "K", k_shape, dtype, dev), _dense(length, "length", (B,), torch.int32, dev),
                           _dense(lse, "lse", (B, Hq, T), torch.float32, dev), _dense(accepted, "accepted", (B, A), torch.int32, dev), A,
                           _dense(weights, "weights", (B, Hkv, S), torch.float32, dev), B, Hq, Hkv, T, S, D, _DTYPES[dtype], scale, stream, flags)
    _call_on(dev, (_lib or lib()).b200attn_cache_weights, packed)
    return weights


def cache_evict(K, V, length, weights, keep, sink=0, recent=0, pos=None, next_pos=None, into=None, kept=None, stream=None, flags=0):
    """Leaves at most `keep` rows in each head of the cache: the tokens of the first `sink` and the last `recent` positions, then the rows of largest
    weight.  In place, or into another cache (K, V, weights, pos; pos None where `pos` is None).  Returns (kept [B, Hkv, keep] int32: the former index
    of each row or -1, the new lengths [B]); `length` stays (b200attn_cache_evict)."""
    torch, dev, k_shape = _cache_shape(K)
    B, Hkv, S, D = k_shape
    if stream is not None and (at := _elsewhere(stream, dev)) is not None:
        with torch.cuda.stream(at):
            return cache_evict(K, V, length, weights, keep, sink, recent, pos, next_pos, into, kept, None, flags)
    dtype, i32, f32 = K.dtype, torch.int32, torch.float32
    if length is None or weights is None:
        _refuse("length and weights must be given")
    n = _dense(length, "length", (B,), i32, dev)
    if kept is None:
        kept = length.new_empty((B, Hkv, max(keep, 0)))
        kept_at = kept.data_ptr()
    else:
        kept_at = _dense(kept, "kept", (B, Hkv, max(keep, 0)), i32, dev)
    out = torch.empty_like(length)
    stream = torch._C._cuda_getCurrentRawStream(dev)
    target, So = (0,) * 10, 0
    if into is not None:
        Ko, Vo, Wo, Po = into
        if Ko.dim() != 4 or Wo is None or (Po is None) != (pos is None):
            _refuse("`into` must be (K, V, weights, pos), with pos where this cache has one")
        So = Ko.shape[2]
        if So == 0:   # (its addresses would be those of no other cache)
            _refuse("`into` must have rows")
        o_shape = (B, Hkv, So, D)
        target = _view(Ko, "K of `into`", o_shape, dtype, dev) + _view(Vo, "V of `into`", o_shape, dtype, dev) + (
            _dense(Wo, "weights of `into`", (B, Hkv, So), f32, dev), _dense(Po, "pos of `into`", (B, Hkv, So), i32, dev))
    packed = _pack_evict(*_view(K, "K", k_shape, dtype, dev), *_view(V, "V", k_shape, dtype, dev), _dense(weights, "weights", (B, Hkv, S), f32, dev),
                         _dense(pos, "pos", (B, Hkv, S), i32, dev), n, _dense(next_pos, "next_pos", (B,), i32, dev),
                         out.data_ptr(), kept_at, keep, sink, recent, *target, So, B, Hkv, S, D,
                         _DTYPES[dtype], stream, flags)
    _call_on(dev, (_lib or lib()).b200attn_cache_evict, packed)
    return kept, out


def set_option(option, value):
    check(lib().b200attn_set_option(option, value))


def shard_ranges(total_bh, n_parts):
    begin = (C.c_longlong * n_parts)()
    count = (C.c_longlong * n_parts)()
    lib().b200attn_shard_ranges(total_bh, n_parts, begin, count)
    return list(begin), list(count)


def synth_fill(t, seed, tensor_id, dist="uniform", index0=0, stream=None):
    """Fills a torch CUDA tensor (float32 / bfloat16) with the library's synthetic inputs."""
    import torch
    dtype = F32 if t.dtype == torch.float32 else BF16
    if stream is None:
        stream = torch.cuda.current_stream(t.device).cuda_stream
    with torch.cuda.device(t.device):
        check(lib().b200attn_synth_fill(t.data_ptr(), t.numel(), seed, tensor_id, index0,
                                        0 if dist == "uniform" else 1, dtype, stream))
    return t


def last_path():
    return lib().b200attn_last_path().decode()


def launch_count():
    return int(lib().b200attn_launch_count())
