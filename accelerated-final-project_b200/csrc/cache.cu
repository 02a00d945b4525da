// Entry points of the key/value cache (include/b200attn.h, "A key/value cache"): checks of the arguments, choice of the kernel, launches.
#include <atomic>
#include <cmath>
#include <cstring>

#include "host.h"
#include "cache_narrow.cuh"
#include "cache_weights.cuh"

namespace b200attn {
namespace {

#define CU_TRY(expr)                                                                                  \
    do {                                                                                              \
        cudaError_t e_ = (expr);                                                                      \
        if (e_ != cudaSuccess)                                                                        \
            return fail(B200ATTN_ERR_CUDA, "CUDA error %d (%s) at %s:%d: %s", (int)e_,                \
                        cudaGetErrorString(e_), __FILE__, __LINE__, #expr);                           \
    } while (0)

size_t esize(int dtype) { return dtype == B200ATTN_F32 ? 4 : 2; }

int check_dtype(int dtype) {
    if (dtype != B200ATTN_F32 && dtype != B200ATTN_BF16 && dtype != B200ATTN_F16) return fail(B200ATTN_ERR_INVALID_ARG, "unknown dtype %d", dtype);
    return B200ATTN_OK;
}

int check_capacity(int capacity) {
    if (capacity > (1 << 30)) return fail(B200ATTN_ERR_TOO_LARGE, "capacity must be at most 2^30 rows (got %d)", capacity);
    return B200ATTN_OK;
}

int check_scale(float scale) {   // (the kernels take it times log2 e)
    if (!(scale >= 0.0f) || std::isinf(scale * 1.4426950408889634f))
        return fail(B200ATTN_ERR_INVALID_ARG, "scale must be positive and finite, also times log2 e, or 0 for 1/sqrt(head_d)");
    return B200ATTN_OK;
}

int check_view(const char *name, const b200attn_view &v, int dtype) {
    if (v.ptr == nullptr) return fail(B200ATTN_ERR_INVALID_ARG, "%s must be non-NULL", name);
    if ((uintptr_t)v.ptr & (esize(dtype) - 1)) return fail(B200ATTN_ERR_INVALID_ARG, "%s must be aligned to the element size", name);
    if (v.stride_b < 0 || v.stride_h < 0 || v.stride_l < 0) return fail(B200ATTN_ERR_INVALID_ARG, "strides of %s must not be negative", name);
    return B200ATTN_OK;
}

// The bytes from a view's first element to behind its last.
size_t extent(const b200attn_view &v, long long B, long long H, long long L, long long D, int dtype) {
    return (size_t)((B - 1) * v.stride_b + (H - 1) * v.stride_h + (L - 1) * v.stride_l + D) * esize(dtype);
}
bool meet(const void *a, size_t na, const void *b, size_t nb) { return (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na; }

// What is written: rows of a view must not share elements (the dimensions, sorted by stride, each have to clear what is inside them).
int check_written(const char *name, const b200attn_view &v, long long B, long long H, long long L, long long D) {
    long long n[3] = {B, H, L}, s[3] = {v.stride_b, v.stride_h, v.stride_l}, inside = D;
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 3; ++j)
            if (s[j] < s[i]) { long long t = s[i]; s[i] = s[j]; s[j] = t; t = n[i]; n[i] = n[j]; n[j] = t; }
    for (int i = 0; i < 3; ++i) {
        if (n[i] == 1) continue;
        if (s[i] < inside) return fail(B200ATTN_ERR_INVALID_ARG, "rows of %s, which is written, overlap each other", name);
        inside = s[i] * (n[i] - 1) + inside;
    }
    return B200ATTN_OK;
}

CaView strides(const b200attn_view &v, long long unit = 1) { return CaView{v.stride_b * unit, v.stride_h * unit, v.stride_l * unit}; }
bool aligned16(const b200attn_view &v, int dtype) {
    const long long e = (long long)esize(dtype);
    return (((uintptr_t)v.ptr | (uintptr_t)(v.stride_b * e) | (uintptr_t)(v.stride_h * e) | (uintptr_t)(v.stride_l * e)) & 15) == 0;
}

// What tensor maps and 16-byte accesses take: rows on 16 bytes, strides that are not 0 (a dimension of size 1 has none to speak of).
bool strides_fit(b200attn_view v, int dtype, int B, int H, int L) {
    if (B == 1) v.stride_b = 8;
    if (H == 1) v.stride_h = 8;
    if (L == 1) v.stride_l = 8;
    return aligned16(v, dtype) && v.stride_b > 0 && v.stride_h > 0 && v.stride_l > 0;
}

// Lets a kernel have all the shared memory there is, once per device (asking each time costs a short call half a microsecond).
template <auto Kern>
int raise_smem(const HostCall &c) {
    static std::atomic<unsigned long long> done{0};
    const unsigned long long bit = 1ull << (c.dev & 63);
    if (done.load(std::memory_order_acquire) & bit) return B200ATTN_OK;
    cudaFuncAttributes fa;
    CU_TRY(cudaFuncGetAttributes(&fa, Kern));
    CU_TRY(cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(c.max_smem - fa.sharedSizeBytes)));
    done.fetch_or(bit, std::memory_order_release);
    return B200ATTN_OK;
}

// ---- attention ---------------------------------------------------------------------------------------------------------
int validate(const b200attn_attend_args *a, bool pointers) {
    if (a == nullptr) return fail(B200ATTN_ERR_INVALID_ARG, "args is NULL");
    if (a->struct_size != sizeof *a) return fail(B200ATTN_ERR_INVALID_ARG, "args->struct_size is %zu, expected %zu", a->struct_size, sizeof *a);
    if (a->batch_sz <= 0 || a->num_heads <= 0 || a->num_kv_heads <= 0 || a->len_new <= 0 || a->capacity <= 0 || a->head_d <= 0)
        return fail(B200ATTN_ERR_INVALID_ARG, "batch_sz, num_heads, num_kv_heads, len_new, capacity, head_d must be positive (got %d,%d,%d,%d,%d,%d)", a->batch_sz,
                    a->num_heads, a->num_kv_heads, a->len_new, a->capacity, a->head_d);
    int rc = check_dtype(a->dtype);
    if (rc) return rc;
    if (a->num_heads % a->num_kv_heads) return fail(B200ATTN_ERR_INVALID_ARG, "num_heads (%d) must be a multiple of num_kv_heads (%d)", a->num_heads, a->num_kv_heads);
    if (a->head_d > CA_MAX_D) return fail(B200ATTN_ERR_INVALID_ARG, "head_d must be at most %d (got %d)", CA_MAX_D, a->head_d);
    if ((rc = check_capacity(a->capacity))) return rc;
    if ((long long)a->len_new * (a->num_heads / a->num_kv_heads) > (1ll << 30))
        return fail(B200ATTN_ERR_TOO_LARGE, "len_new times the query heads of a key head is %lld, at most 2^30 are taken", (long long)a->len_new * (a->num_heads / a->num_kv_heads));
    if ((rc = check_scale(a->scale))) return rc;
    if ((a->Kd.ptr == nullptr) != (a->Vd.ptr == nullptr)) return fail(B200ATTN_ERR_INVALID_ARG, "Kd and Vd must be given together");
    if (a->mask && a->Kd.ptr == nullptr) return fail(B200ATTN_ERR_INVALID_ARG, "a mask needs Kd and Vd");
    if (a->mask && a->mask_stride_b != 0 && a->mask_stride_b != (long long)a->len_new * a->len_new)
        return fail(B200ATTN_ERR_INVALID_ARG, "mask_stride_b must be 0 or len_new * len_new");
    if (!pointers) return B200ATTN_OK;
    if ((rc = check_view("Q", a->Q, a->dtype)) || (rc = check_view("K", a->K, a->dtype)) || (rc = check_view("V", a->V, a->dtype)) || (rc = check_view("out", a->out, a->dtype)))
        return rc;
    if (a->Kd.ptr && ((rc = check_view("Kd", a->Kd, a->dtype)) || (rc = check_view("Vd", a->Vd, a->dtype)))) return rc;
    const long long B = a->batch_sz, Hq = a->num_heads, Hkv = a->num_kv_heads, T = a->len_new, S = a->capacity, D = a->head_d;
    if ((rc = check_written("out", a->out, B, Hq, T, D))) return rc;
    if (!a->length) return fail(B200ATTN_ERR_INVALID_ARG, "length must be non-NULL");
    if (((uintptr_t)a->length | (uintptr_t)a->lse) & 3) return fail(B200ATTN_ERR_INVALID_ARG, "length and lse must be aligned to 4 bytes");
    const size_t no = extent(a->out, B, Hq, T, D, a->dtype);
    if (meet(a->out.ptr, no, a->Q.ptr, extent(a->Q, B, Hq, T, D, a->dtype)) || meet(a->out.ptr, no, a->K.ptr, extent(a->K, B, Hkv, S, D, a->dtype)) ||
        meet(a->out.ptr, no, a->V.ptr, extent(a->V, B, Hkv, S, D, a->dtype)) ||
        (a->Kd.ptr && (meet(a->out.ptr, no, a->Kd.ptr, extent(a->Kd, B, Hkv, T, D, a->dtype)) || meet(a->out.ptr, no, a->Vd.ptr, extent(a->Vd, B, Hkv, T, D, a->dtype)))))
        return fail(B200ATTN_ERR_INVALID_ARG, "out must not overlap an input");
    return B200ATTN_OK;
}

// Workspace: the slots of cut units, then the entries.
long long units(const CaParams &p) { return (long long)p.B * p.Hkv * p.nrt; }
size_t entries_bytes(const CaParams &p) { return (size_t)(p.by_cta ? p.grid : units(p)) * 8 * sizeof(int); }
size_t attend_bytes(const CaParams &p) { return p.uncut ? 0 : ((size_t)p.grid * 2 * ca_slot_floats(p.RT, p.D) + 3) / 4 * 16 + entries_bytes(p); }

void share_out(CaParams &p, int RT, int TK, int OH, int grid) {
    p.RT = RT; p.TK = TK; p.OH = OH; p.grid = grid;
    p.nrt = (p.R + RT - 1) / RT;
    // few units are cut into many parts each, which a block's warps share out: then a block has as many rows as it can take at once
    p.by_cta = units(p) > grid;
    const long long parts = grid / units(p) + 1;
    p.join_rows = p.by_cta ? 16 : parts <= 4 ? 8 : parts <= 8 ? 4 : parts <= 16 ? 2 : 1;
}
// Of the kernel that runs: the tiles of new keys of a key head's units.
void count_drafts(CaParams &p) {
    p.DT = 0;
    if (!p.drafts) return;
    if (p.mask) p.DT = (long long)p.nrt * ca_draft_tiles(0, p.R, p.RT, p.G, p.T, p.TK, false);
    else
        for (int rt = 0; rt < p.nrt; ++rt) p.DT += ca_draft_tiles(rt, p.R, p.RT, p.G, p.T, p.TK, true);
}

void fill(CaParams &p, const b200attn_attend_args &a) {
    p.Q = a.Q.ptr; p.K = a.K.ptr; p.V = a.V.ptr; p.Kd = a.Kd.ptr; p.Vd = a.Vd.ptr; p.O = a.out.ptr;
    p.q = strides(a.Q); p.k = strides(a.K); p.v = strides(a.V); p.kd = strides(a.Kd); p.vd = strides(a.Vd); p.o = strides(a.out);
    p.lse = a.lse; p.len = a.length; p.mask = a.mask; p.mask_b = a.mask_stride_b;
    p.B = a.batch_sz; p.Hq = a.num_heads; p.Hkv = a.num_kv_heads; p.G = a.num_heads / a.num_kv_heads;
    p.T = a.len_new; p.S = a.capacity; p.D = a.head_d;
    p.R = p.T * p.G;
    p.drafts = a.Kd.ptr != nullptr;
    p.scale_log2 = (a.scale == 0.0f ? 1.0f / sqrtf((float)a.head_d) : a.scale) * 1.4426950408889634f;
}

template <typename T>
int launch_combine(const CaParams &p, cudaStream_t st) {
    if (p.uncut) {
        count_launches(1);
        return B200ATTN_OK;
    }
    const dim3 grid((unsigned)(p.by_cta ? p.grid : units(p)), (unsigned)(((p.RT < p.R ? p.RT : p.R) + p.join_rows - 1) / p.join_rows));
    CU_TRY(p.D <= 64 ? launch_dependent(ca_combine_kernel<T, 2>, grid, CB_THREADS, 0, 1, st, p)
                     : p.D <= 128 ? launch_dependent(ca_combine_kernel<T, 4>, grid, CB_THREADS, 0, 1, st, p) : launch_dependent(ca_combine_kernel<T, 8>, grid, CB_THREADS, 0, 1, st, p));
    count_launches(2);   // with the kernel whose parts these are
    return B200ATTN_OK;
}
// CTAs of ca_generic_kernel that share the work out: as many as run at once, so that equal shares end together.  Four, three or one an SM by the registers that its
// three widths take, and no more than fit its shared memory (two at head_d 117 to 128; three of 117 to 124 would fill it to the byte, and do not run at once).
//   fp32, 8 x 8 heads, 4 tokens, 4096 rows, head_d 128 / 124: 97 / 115 us with two an SM, 128 / 131 with three; 2 x 16 heads of 333 tokens over 1500 rows, 128: 690, 908
int generic_grid(const CaParams &p, const HostCall &c) {
    const int most = p.D <= 64 ? 4 : p.D <= 128 ? 3 : 1;
    const size_t cta = (cg_smem_bytes(p.D) + CG_STATIC_SMEM + 127) / 128 * 128 + 1024;   // (the system keeps 1 KB per CTA)
    const int fit = (int)(c.max_smem / cta);
    return c.sm_count * (fit < most ? fit : most);
}
template <typename T, int DB, bool FAST>
int launch_generic(const CaParams &p, const HostCall &c, cudaStream_t st) {
    const size_t smem = cg_smem_bytes(p.D);
    int rc = raise_smem<ca_generic_kernel<T, DB, FAST>>(c);
    if (rc) return rc;
    CU_TRY(launch_dependent(ca_generic_kernel<T, DB, FAST>, dim3((unsigned)p.grid), CG_THREADS, smem, 1, st, p));
    return B200ATTN_OK;
}
template <typename T, bool FAST>
int launch_attend(const CaParams &p, const HostCall &c, cudaStream_t st) {
    int rc = p.D <= 64 ? launch_generic<T, 64, FAST>(p, c, st) : p.D <= 128 ? launch_generic<T, 128, FAST>(p, c, st) : launch_generic<T, 256, FAST>(p, c, st);
    if (rc) return rc;
    return launch_combine<T>(p, st);
}

// The tensor-core kernel for these sizes: rows of a tile, tiles of a unit, ring.
bool tc_shape(const b200attn_attend_args *a, const HostCall &c, CaParams p, CtParams *out) {
    if (a->dtype == B200ATTN_F32 || p.D % 8 != 0 || p.G > 128 || (a->flags & B200ATTN_FLAG_FORCE_GENERIC)) return false;
    CtParams ct{};
    ct.tpt = 128 / p.G;
    ct.box_t = p.T < ct.tpt ? p.T : ct.tpt;
    ct.ng = (p.D + 63) / 64;
    const int NT = p.D <= 128 && p.T > ct.tpt ? 2 : 1;
    ct.rows8 = NT == 2 ? 128 : (p.G * ct.box_t + 7) & ~7;
    const int TK = p.D <= 128 ? 128 : 64;
    const size_t room = c.max_smem - 2048 - 1024, stage = (size_t)ct.ng * TK * 128;
    // one row tile: the next unit's Q and the next key tile's P beside the present ones' where four stages remain
    const int buffers[4][2] = {{2, 2}, {1, 2}, {2, 1}, {1, 1}};
    for (int i = NT == 1 ? 0 : 3; i < 4; ++i) {
        ct.nq = buffers[i][0]; ct.np = buffers[i][1];
        const size_t front = ct_front_bytes(NT, ct.nq, ct.np, ct.ng, ct.rows8, TK);
        ct.nst = front < room ? (int)((room - front) / stage) : 0;
        if (ct.nst > CT_MAX_STAGES) ct.nst = CT_MAX_STAGES;
        if (ct.nst >= (i < 3 ? 4 : 3)) break;
    }
    if (ct.nst < 3) return false;
    share_out(p, NT * ct.tpt * p.G, TK, CT_OH, c.sm_count);
    ct.a = p;
    *out = ct;
    return true;
}
// The kernel for up to 64 rows a key head.
bool narrow_shape(const b200attn_attend_args *a, const HostCall &c, CaParams p, CnParams *out) {
    if (a->dtype == B200ATTN_F32 || p.D % 8 != 0 || p.R > 64 || (a->flags & B200ATTN_FLAG_FORCE_GENERIC)) return false;
    CnParams cn{};
    cn.ng = (p.D + 63) / 64;
    cn.nh = (cn.ng + 1) / 2;
    cn.gp = cn.ng < 2 ? 1 : 2;
    const int N = p.R <= 16 ? 16 : p.R <= 32 ? 32 : 64, cols = 2 * N + 2 * cn.nh * N;
    for (cn.tmem_cols = 32; cn.tmem_cols < cols; cn.tmem_cols *= 2) {}
    const size_t room = c.max_smem - 4096 - 1024, front = cn_front_bytes(N, cn.ng);
    cn.nst = (int)((room - front) / ((size_t)cn.gp * CN_GROUP));
    if (cn.nst > CT_MAX_STAGES) cn.nst = CT_MAX_STAGES;
    share_out(p, p.R, CN_TK, CN_OH, c.sm_count);
    // a short cache's units are not cut: nothing is joined then, by a second launch
    p.uncut = (p.S + CN_TK - 1) / CN_TK + (p.drafts ? (p.T + CN_TK - 1) / CN_TK : 0) <= (units(p) * 4 >= c.sm_count * 3 ? CN_UNCUT_MANY : CN_UNCUT_FEW);
    cn.a = p;
    *out = cn;
    return true;
}
bool tc_aligned(const b200attn_attend_args *a) {
    auto fine = [&](const b200attn_view &v, int h, int l) { return strides_fit(v, a->dtype, a->batch_sz, h, l); };
    return fine(a->Q, a->num_heads, a->len_new) && fine(a->K, a->num_kv_heads, a->capacity) && fine(a->V, a->num_kv_heads, a->capacity) && fine(a->out, a->num_heads, a->len_new) &&
           (a->Kd.ptr == nullptr || (fine(a->Kd, a->num_kv_heads, a->len_new) && fine(a->Vd, a->num_kv_heads, a->len_new)));
}

template <int NT, int TK, bool F16>
int launch_tc(const CtParams &ct, const HostCall &c, const CUtensorMap (&m)[5], cudaStream_t st) {
    const size_t smem = ct_front_bytes(NT, ct.nq, ct.np, ct.ng, ct.rows8, TK) + (size_t)ct.nst * ct.ng * TK * 128 + 1024;
    int rc = raise_smem<ca_tc_kernel<NT, TK, F16>>(c);
    if (rc) return rc;
    CU_TRY(launch_dependent(ca_tc_kernel<NT, TK, F16>, dim3((unsigned)ct.a.grid), ct_threads(NT), smem, 1, st, m[0], m[1], m[2], m[3], m[4], ct));
    return B200ATTN_OK;
}
template <bool F16>
int launch_attend_tc(const CtParams &ct, const HostCall &c, const CUtensorMap (&m)[5], cudaStream_t st) {
    const CaParams &p = ct.a;
    int rc = p.TK == 64 ? launch_tc<1, 64, F16>(ct, c, m, st) : p.RT > ct.tpt * p.G ? launch_tc<2, 128, F16>(ct, c, m, st) : launch_tc<1, 128, F16>(ct, c, m, st);
    if (rc) return rc;
    return launch_combine<typename CtType<F16>::T>(p, st);
}

template <int N, bool F16>
int launch_narrow(const CnParams &cn, const HostCall &c, const CUtensorMap (&m)[5], cudaStream_t st) {
    const size_t smem = cn_front_bytes(N, cn.ng) + (size_t)cn.nst * cn.gp * CN_GROUP + 1024;
    int rc = raise_smem<ca_narrow_kernel<N, F16>>(c);
    if (rc) return rc;
    CU_TRY(launch_dependent(ca_narrow_kernel<N, F16>, dim3((unsigned)cn.a.grid), CN_THREADS, smem, 1, st, m[0], m[1], m[2], m[3], m[4], cn));
    return B200ATTN_OK;
}
template <bool F16>
int launch_attend_narrow(const CnParams &cn, const HostCall &c, const CUtensorMap (&m)[5], cudaStream_t st) {
    const CaParams &p = cn.a;
    int rc = p.R <= 16 ? launch_narrow<16, F16>(cn, c, m, st) : p.R <= 32 ? launch_narrow<32, F16>(cn, c, m, st) : launch_narrow<64, F16>(cn, c, m, st);
    if (rc) return rc;
    return launch_combine<typename CtType<F16>::T>(p, st);
}

int attend(const b200attn_attend_args *a, size_t *need) {
    int rc = validate(a, need == nullptr);
    if (rc) return rc;
    HostCall c;
    if ((rc = host_begin(&c))) return rc;
    cudaStream_t st = (cudaStream_t)a->stream;
    CaParams p{};
    fill(p, *a);
    p.err = c.err_dev; p.err_sys = c.err_sys; p.spin_limit = c.spin_limit; p.wait_extra = c.wait_extra;
    CtParams ct;
    CnParams cn;
    bool narrow = narrow_shape(a, c, p, &cn), tc = !narrow && tc_shape(a, c, p, &ct);
    share_out(p, CG_ROWS, CG_KEYS, CG_OH, generic_grid(p, c));
    p.uncut = narrow && cn.a.uncut;
    // the larger of the two kernels' needs: which one runs goes by the tensors' alignment, too
    size_t bytes = attend_bytes(p);
    const size_t other = narrow ? attend_bytes(cn.a) : tc ? attend_bytes(ct.a) : 0;
    if (other > bytes) bytes = other;
    if (need) { *need = bytes; return B200ATTN_OK; }
    CUtensorMap m[5];
    if (narrow || tc) {
        const CaParams &q = narrow ? cn.a : ct.a;
        memset(m, 0, sizeof m);
        const bool maps = tc_aligned(a) && ct_map_q(&m[0], q.Q, q.q, q.B, q.Hkv, q.G, q.T, q.D, narrow ? q.T : ct.box_t) &&
                          ct_map_rows(&m[1], q.K, q.k, q.B, q.Hkv, q.S, q.D, q.TK) && ct_map_rows(&m[2], q.V, q.v, q.B, q.Hkv, q.S, q.D, q.TK) &&
                          (!q.drafts || (ct_map_rows(&m[3], q.Kd, q.kd, q.B, q.Hkv, q.T, q.D, q.TK) && ct_map_rows(&m[4], q.Vd, q.vd, q.B, q.Hkv, q.T, q.D, q.TK)));
        narrow = narrow && maps;
        tc = tc && maps;
    }
    void *ws = bytes ? a->workspace : nullptr;
    if (ws) {
        if (a->workspace_bytes < bytes) return fail(B200ATTN_ERR_INVALID_ARG, "workspace_bytes is %zu, this call needs %zu", a->workspace_bytes, bytes);
        if ((uintptr_t)ws & 15) return fail(B200ATTN_ERR_INVALID_ARG, "workspace must be aligned to 16 bytes");
    } else if (bytes && (rc = host_workspace(&c, bytes, st, &ws))) {
        return rc;
    }
    CaParams &q = narrow ? cn.a : tc ? ct.a : p;
    count_drafts(q);
    q.part = (float *)ws;
    if (ws) q.entries = (int *)((char *)ws + attend_bytes(q) - entries_bytes(q));
    if (narrow) rc = a->dtype == B200ATTN_F16 ? launch_attend_narrow<true>(cn, c, m, st) : launch_attend_narrow<false>(cn, c, m, st);
    else if (tc) rc = a->dtype == B200ATTN_F16 ? launch_attend_tc<true>(ct, c, m, st) : launch_attend_tc<false>(ct, c, m, st);
    else if (a->dtype == B200ATTN_F32) rc = p.D % 4 == 0 && tc_aligned(a) ? launch_attend<float, true>(p, c, st) : launch_attend<float, false>(p, c, st);
    else rc = a->dtype == B200ATTN_F16 ? launch_attend<__half, false>(p, c, st) : launch_attend<__nv_bfloat16, false>(p, c, st);
    if (rc) return rc;
    set_last_path(narrow ? "cache_narrow" : tc ? "cache_tc" : "cache_generic");
    return host_end(&c, st, a->flags & B200ATTN_FLAG_ASYNC);
}

// ---- lists of accepted tokens ------------------------------------------------------------------------------------------
int check_accepted(const int *accepted, int max_accepted) {
    if (accepted && max_accepted <= 0) return fail(B200ATTN_ERR_INVALID_ARG, "max_accepted must be positive (got %d)", max_accepted);
    if ((uintptr_t)accepted & 3) return fail(B200ATTN_ERR_INVALID_ARG, "accepted must be aligned to 4 bytes");
    return B200ATTN_OK;
}
int check_grid(int B, int Hkv) {
    if (B > 65535 || Hkv > 65535) return fail(B200ATTN_ERR_TOO_LARGE, "batch_sz and num_kv_heads must be at most 65535 (got %d, %d)", B, Hkv);
    return B200ATTN_OK;
}

int commit(const b200attn_commit_args *a) {
    if (a == nullptr) return fail(B200ATTN_ERR_INVALID_ARG, "args is NULL");
    if (a->struct_size != sizeof *a) return fail(B200ATTN_ERR_INVALID_ARG, "args->struct_size is %zu, expected %zu", a->struct_size, sizeof *a);
    if (a->batch_sz <= 0 || a->num_kv_heads <= 0 || a->len_new <= 0 || a->capacity <= 0 || a->head_d <= 0)
        return fail(B200ATTN_ERR_INVALID_ARG, "batch_sz, num_kv_heads, len_new, capacity, head_d must be positive (got %d,%d,%d,%d,%d)", a->batch_sz, a->num_kv_heads,
                    a->len_new, a->capacity, a->head_d);
    int rc = check_dtype(a->dtype);
    if (rc || (rc = check_grid(a->batch_sz, a->num_kv_heads))) return rc;
    if (a->head_d > (1 << 20)) return fail(B200ATTN_ERR_TOO_LARGE, "head_d must be at most 2^20 (got %d)", a->head_d);
    if ((rc = check_capacity(a->capacity))) return rc;
    const long long B = a->batch_sz, H = a->num_kv_heads, T = a->len_new, S = a->capacity, D = a->head_d;
    if ((rc = check_view("K", a->K, a->dtype)) || (rc = check_view("V", a->V, a->dtype)) || (rc = check_view("Kd", a->Kd, a->dtype)) || (rc = check_view("Vd", a->Vd, a->dtype)) ||
        (rc = check_written("K", a->K, B, H, S, D)) || (rc = check_written("V", a->V, B, H, S, D)) || (rc = check_accepted(a->accepted, a->max_accepted)))
        return rc;
    if (!a->length) return fail(B200ATTN_ERR_INVALID_ARG, "length must be non-NULL");
    if (((uintptr_t)a->length | (uintptr_t)a->length_out | (uintptr_t)a->weights | (uintptr_t)a->pos | (uintptr_t)a->next_pos) & 3)
        return fail(B200ATTN_ERR_INVALID_ARG, "length, length_out, weights, pos and next_pos must be aligned to 4 bytes");
    if (a->length_out && (meet(a->length_out, 4 * B, a->length, 4 * B) || (a->next_pos && meet(a->length_out, 4 * B, a->next_pos, 4 * B))))
        return fail(B200ATTN_ERR_INVALID_ARG, "length_out must not overlap length or next_pos");
    const size_t nk = extent(a->K, B, H, S, D, a->dtype), nv = extent(a->V, B, H, S, D, a->dtype), nkd = extent(a->Kd, B, H, T, D, a->dtype), nvd = extent(a->Vd, B, H, T, D, a->dtype);
    if (meet(a->K.ptr, nk, a->Kd.ptr, nkd) || meet(a->K.ptr, nk, a->Vd.ptr, nvd) || meet(a->V.ptr, nv, a->Kd.ptr, nkd) || meet(a->V.ptr, nv, a->Vd.ptr, nvd))
        return fail(B200ATTN_ERR_INVALID_ARG, "Kd and Vd must not overlap the cache");
    HostCall c;
    if ((rc = host_begin(&c))) return rc;
    cudaStream_t st = (cudaStream_t)a->stream;
    const long long e = (long long)esize(a->dtype);
    CcParams p{};
    p.K = a->K.ptr; p.V = a->V.ptr; p.Kd = a->Kd.ptr; p.Vd = a->Vd.ptr;
    p.k = strides(a->K, e); p.v = strides(a->V, e); p.kd = strides(a->Kd, e); p.vd = strides(a->Vd, e);
    p.len = a->length; p.accepted = a->accepted; p.next_pos = a->next_pos; p.len_out = a->length_out; p.pos = a->pos; p.weights = a->weights;
    p.A = a->accepted ? a->max_accepted : a->len_new;
    p.B = a->batch_sz; p.Hkv = a->num_kv_heads; p.T = a->len_new; p.S = a->capacity; p.row_bytes = (int)(D * e);
    const bool wide = aligned16(a->K, a->dtype) && aligned16(a->V, a->dtype) && aligned16(a->Kd, a->dtype) && aligned16(a->Vd, a->dtype) && p.row_bytes % 16 == 0;
    p.groups = (p.A + CC_ROWS - 1) / CC_ROWS;
    const long long blocks = ((long long)p.groups * p.Hkv + CC_THREADS / 32 - 1) / (CC_THREADS / 32);
    if (blocks > 0x7fffffffll) return fail(B200ATTN_ERR_TOO_LARGE, "%lld rows to commit in a sequence are too many", (long long)p.A * p.Hkv);
    const dim3 grid((unsigned)blocks, (unsigned)p.B);
    CU_TRY(wide ? launch_dependent(cc_commit_kernel<uint4>, grid, CC_THREADS, 0, 1, st, p)
                : e == 4 ? launch_dependent(cc_commit_kernel<uint32_t>, grid, CC_THREADS, 0, 1, st, p) : launch_dependent(cc_commit_kernel<uint16_t>, grid, CC_THREADS, 0, 1, st, p));
    count_launches(1);
    return host_end(&c, st, a->flags & B200ATTN_FLAG_ASYNC);
}

template <typename T, bool FAST>
int launch_weights(const CwParams &p, const HostCall &c, cudaStream_t st) {
    const size_t smem = cw_smem_bytes(p.D, FAST);
    int rc = raise_smem<cw_generic_kernel<T, FAST>>(c);
    if (rc) return rc;
    CU_TRY(launch_dependent(cw_generic_kernel<T, FAST>, dim3((unsigned)((p.S + CG_KEYS - 1) / CG_KEYS), (unsigned)p.Hkv, (unsigned)p.B), CG_THREADS, smem, 1, st, p));
    count_launches(1);
    return B200ATTN_OK;
}

// The tensor-core kernel where it takes the call: -1 where it does not.
template <bool F16>
int launch_weights_tc(const CxParams &cx, const HostCall &c, const CUtensorMap (&m)[2], size_t smem, cudaStream_t st) {
    int rc = raise_smem<cw_tc_kernel<F16>>(c);
    if (rc) return rc;
    CU_TRY(launch_dependent(cw_tc_kernel<F16>, dim3((unsigned)cx.grid), CX_THREADS, smem, 1, st, m[0], m[1], cx));
    count_launches(1);
    return B200ATTN_OK;
}
int weights_tc(const b200attn_weights_args *a, const CwParams &p, const HostCall &c, cudaStream_t st) {
    if (a->dtype == B200ATTN_F32 || p.D % 8 != 0 || (a->flags & B200ATTN_FLAG_FORCE_GENERIC)) return -1;
    if (!strides_fit(a->Q, a->dtype, a->batch_sz, a->num_heads, a->len_new) || !strides_fit(a->K, a->dtype, a->batch_sz, a->num_kv_heads, a->capacity)) return -1;
    CxParams cx{};
    cx.a = p;
    cx.ng = (p.D + 63) / 64;
    cx.grid = c.sm_count;
    cx.oh = cx_overhead((long long)p.A * p.G);
    const long long room = (long long)c.max_smem - 2048 - 1024, stage = (long long)cx.ng * CX_TK * 128, row = cx.ng * 128 + 8, all = (long long)p.A * p.G;
    // all tokens accepted: boxes of whole groups of 8 rows, up to 64 rows or one such group of them
    int unit = CX_NB;   // a chunk is a multiple of this
    if (!p.accepted && p.G <= 32) {
        int t = 8;
        while (t > 1 && p.G * (t / 2) % 8 == 0) t /= 2;
        cx.box_t = p.G * t < CX_NB ? CX_NB / (p.G * t) * t : t;
        unit = p.G * cx.box_t;
    }
    for (cx.nq = 2; cx.nq > 0; --cx.nq) {   // two buffers for Q where that leaves four stages; else what two stages, the least that overlaps loads and products, leave
        const long long most = (room - (cx.nq == 2 ? 4 : 2) * stage) / (cx.nq * row) / CX_NB * CX_NB;   // rows of a buffer
        const long long fits = most < unit ? 0 : most / unit * unit, rows = (all + unit - 1) / unit * unit;
        if (cx.nq == 2 && rows > fits) continue;
        if (fits == 0) return -1;
        cx.chunk = (int)(rows < fits ? rows : fits);
        break;
    }
    const long long pitch = (cx.chunk + CX_NB - 1) / CX_NB * CX_NB;
    cx.nst = (int)((room - cx.nq * pitch * row) / stage);
    if (cx.nst > CT_MAX_STAGES) cx.nst = CT_MAX_STAGES;
    CUtensorMap m[2];
    memset(m, 0, sizeof m);
    if (!ct_map_rows(&m[1], p.K, p.k, p.B, p.Hkv, p.S, p.D, CX_TK) || (cx.box_t && !ct_map_q(&m[0], p.Q, p.q, p.B, p.Hkv, p.G, p.T, p.D, cx.box_t))) return -1;
    const size_t smem = (size_t)(cx.nq * pitch * row + cx.nst * stage + 1024);
    return a->dtype == B200ATTN_F16 ? launch_weights_tc<true>(cx, c, m, smem, st) : launch_weights_tc<false>(cx, c, m, smem, st);
}

int weights(const b200attn_weights_args *a) {
    if (a == nullptr) return fail(B200ATTN_ERR_INVALID_ARG, "args is NULL");
    if (a->struct_size != sizeof *a) return fail(B200ATTN_ERR_INVALID_ARG, "args->struct_size is %zu, expected %zu", a->struct_size, sizeof *a);
    if (a->batch_sz <= 0 || a->num_heads <= 0 || a->num_kv_heads <= 0 || a->len_new <= 0 || a->capacity <= 0 || a->head_d <= 0)
        return fail(B200ATTN_ERR_INVALID_ARG, "batch_sz, num_heads, num_kv_heads, len_new, capacity, head_d must be positive (got %d,%d,%d,%d,%d,%d)", a->batch_sz,
                    a->num_heads, a->num_kv_heads, a->len_new, a->capacity, a->head_d);
    int rc = check_dtype(a->dtype);
    if (rc || (rc = check_grid(a->batch_sz, a->num_kv_heads))) return rc;
    if (a->num_heads % a->num_kv_heads) return fail(B200ATTN_ERR_INVALID_ARG, "num_heads (%d) must be a multiple of num_kv_heads (%d)", a->num_heads, a->num_kv_heads);
    if (a->head_d > CA_MAX_D) return fail(B200ATTN_ERR_INVALID_ARG, "head_d must be at most %d (got %d)", CA_MAX_D, a->head_d);
    if ((rc = check_capacity(a->capacity))) return rc;
    const int A = a->accepted ? a->max_accepted : a->len_new, G = a->num_heads / a->num_kv_heads;
    if ((long long)A * G > (1ll << 30)) return fail(B200ATTN_ERR_TOO_LARGE, "accepted tokens times the query heads of a key head are %lld, at most 2^30 are taken", (long long)A * G);
    if ((rc = check_scale(a->scale))) return rc;
    if ((rc = check_view("Q", a->Q, a->dtype)) || (rc = check_view("K", a->K, a->dtype)) || (rc = check_accepted(a->accepted, a->max_accepted))) return rc;
    if (!a->length || !a->lse || !a->weights) return fail(B200ATTN_ERR_INVALID_ARG, "length, lse and weights must be non-NULL");
    if (((uintptr_t)a->length | (uintptr_t)a->lse | (uintptr_t)a->weights) & 3) return fail(B200ATTN_ERR_INVALID_ARG, "length, lse and weights must be aligned to 4 bytes");
    HostCall c;
    if ((rc = host_begin(&c))) return rc;
    cudaStream_t st = (cudaStream_t)a->stream;
    CwParams p{};
    p.Q = a->Q.ptr; p.K = a->K.ptr; p.q = strides(a->Q); p.k = strides(a->K);
    p.len = a->length; p.accepted = a->accepted; p.lse = a->lse; p.weights = a->weights;
    p.A = A; p.B = a->batch_sz; p.Hq = a->num_heads; p.Hkv = a->num_kv_heads; p.G = G; p.T = a->len_new; p.S = a->capacity; p.D = a->head_d;
    p.scale_log2 = (a->scale == 0.0f ? 1.0f / sqrtf((float)a->head_d) : a->scale) * 1.4426950408889634f;
    p.err = c.err_dev; p.err_sys = c.err_sys; p.spin_limit = c.spin_limit; p.wait_extra = c.wait_extra;
    rc = weights_tc(a, p, c, st);
    if (rc == B200ATTN_OK) {
        set_last_path("cache_tc");
        return host_end(&c, st, a->flags & B200ATTN_FLAG_ASYNC);
    }
    if (rc != -1) return rc;
    if (a->dtype == B200ATTN_F32) rc = p.D % 4 == 0 && strides_fit(a->K, a->dtype, p.B, p.Hkv, p.S) && strides_fit(a->Q, a->dtype, p.B, p.Hq, p.T) ? launch_weights<float, true>(p, c, st) : launch_weights<float, false>(p, c, st);
    else rc = a->dtype == B200ATTN_F16 ? launch_weights<__half, false>(p, c, st) : launch_weights<__nv_bfloat16, false>(p, c, st);
    if (rc) return rc;
    set_last_path("cache_generic");
    return host_end(&c, st, a->flags & B200ATTN_FLAG_ASYNC);
}

template <typename P, int THREADS>
int launch_select(const CeParams &p, const HostCall &c, int cl, cudaStream_t st) {
    int rc = raise_smem<ce_select_kernel<P, THREADS>>(c);
    if (rc) return rc;
    CU_TRY(launch_dependent(ce_select_kernel<P, THREADS>, dim3((unsigned)(p.Hkv * cl), (unsigned)p.B), THREADS, ce_smem_bytes(p.chunk_most, p.cached), cl, st, p));
    return B200ATTN_OK;
}
template <typename P>
int launch_evict(const CeParams &p, const HostCall &c, int cl, cudaStream_t st) {
    int rc = cl > 1 ? launch_select<P, 1024>(p, c, cl, st) : launch_select<P, 512>(p, c, cl, st);
    if (rc) return rc;
    count_launches(1);
    if (!p.K_out && p.S - p.keep <= CE_FEW) return B200ATTN_OK;
    const int most = p.keep < p.S ? p.keep : p.S;
    CU_TRY(launch_dependent(ce_move_kernel<P>, dim3((unsigned)((most + CC_THREADS - 1) / CC_THREADS), (unsigned)p.Hkv, (unsigned)p.B), CC_THREADS, 0, 1, st, p));
    count_launches(1);
    return B200ATTN_OK;
}

int evict(const b200attn_evict_args *a) {
    if (a == nullptr) return fail(B200ATTN_ERR_INVALID_ARG, "args is NULL");
    if (a->struct_size != sizeof *a) return fail(B200ATTN_ERR_INVALID_ARG, "args->struct_size is %zu, expected %zu", a->struct_size, sizeof *a);
    if (a->batch_sz <= 0 || a->num_kv_heads <= 0 || a->capacity <= 0 || a->head_d <= 0)
        return fail(B200ATTN_ERR_INVALID_ARG, "batch_sz, num_kv_heads, capacity, head_d must be positive (got %d,%d,%d,%d)", a->batch_sz, a->num_kv_heads, a->capacity, a->head_d);
    int rc = check_dtype(a->dtype);
    if (rc || (rc = check_grid(a->batch_sz, a->num_kv_heads))) return rc;
    if (a->head_d > (1 << 20)) return fail(B200ATTN_ERR_TOO_LARGE, "head_d must be at most 2^20 (got %d)", a->head_d);
    if (a->capacity > B200ATTN_EVICT_MAX_ROWS) return fail(B200ATTN_ERR_TOO_LARGE, "capacity must be at most %d rows (got %d)", B200ATTN_EVICT_MAX_ROWS, a->capacity);
    if (a->keep < 1 || a->sink < 0 || a->recent < 0 || (long long)a->sink + a->recent > a->keep)
        return fail(B200ATTN_ERR_INVALID_ARG, "keep must be at least 1 and at least sink + recent, both not negative (got %d, %d, %d)", a->keep, a->sink, a->recent);
    const bool into = a->K_out.ptr != nullptr;
    if (into != (a->V_out.ptr != nullptr) || into != (a->weights_out != nullptr) || (a->pos_out != nullptr) != (into && a->pos != nullptr))
        return fail(B200ATTN_ERR_INVALID_ARG, "K_out, V_out, weights_out and, with pos, pos_out must be given together");
    if (into && a->capacity_out < (a->keep < a->capacity ? a->keep : a->capacity)) return fail(B200ATTN_ERR_INVALID_ARG, "capacity_out (%d) must be at least keep (%d)", a->capacity_out, a->keep);
    const long long B = a->batch_sz, H = a->num_kv_heads, S = a->capacity, D = a->head_d, So = a->capacity_out;
    if ((rc = check_view("K", a->K, a->dtype)) || (rc = check_view("V", a->V, a->dtype)) || (rc = check_written("K", a->K, B, H, S, D)) || (rc = check_written("V", a->V, B, H, S, D)))
        return rc;
    if (into && ((rc = check_view("K_out", a->K_out, a->dtype)) || (rc = check_view("V_out", a->V_out, a->dtype)) || (rc = check_written("K_out", a->K_out, B, H, So, D)) ||
                 (rc = check_written("V_out", a->V_out, B, H, So, D))))
        return rc;
    if (!a->length || !a->weights || !a->kept) return fail(B200ATTN_ERR_INVALID_ARG, "length, weights and kept must be non-NULL");
    if (((uintptr_t)a->length | (uintptr_t)a->length_out | (uintptr_t)a->weights | (uintptr_t)a->pos | (uintptr_t)a->next_pos | (uintptr_t)a->kept | (uintptr_t)a->weights_out |
         (uintptr_t)a->pos_out) & 3)
        return fail(B200ATTN_ERR_INVALID_ARG, "length, length_out, weights, pos, next_pos, kept and their counterparts must be aligned to 4 bytes");
    if (a->length_out && (meet(a->length_out, 4 * B, a->length, 4 * B) || (a->next_pos && meet(a->length_out, 4 * B, a->next_pos, 4 * B))))
        return fail(B200ATTN_ERR_INVALID_ARG, "length_out must not overlap length or next_pos");
    if (into) {
        const size_t nk = extent(a->K, B, H, S, D, a->dtype), nv = extent(a->V, B, H, S, D, a->dtype), nko = extent(a->K_out, B, H, So, D, a->dtype), nvo = extent(a->V_out, B, H, So, D, a->dtype);
        const size_t nw = (size_t)(4 * B * H * S), nwo = (size_t)(4 * B * H * So);
        if (meet(a->K.ptr, nk, a->K_out.ptr, nko) || meet(a->K.ptr, nk, a->V_out.ptr, nvo) || meet(a->V.ptr, nv, a->K_out.ptr, nko) || meet(a->V.ptr, nv, a->V_out.ptr, nvo) ||
            meet(a->weights, nw, a->weights_out, nwo) || (a->pos && meet(a->pos, nw, a->pos_out, nwo)))
            return fail(B200ATTN_ERR_INVALID_ARG, "the cache that the kept rows go into must not overlap this one");
    }
    HostCall c;
    if ((rc = host_begin(&c))) return rc;
    cudaStream_t st = (cudaStream_t)a->stream;
    const long long e = (long long)esize(a->dtype);
    CeParams p{};
    p.K = a->K.ptr; p.V = a->V.ptr; p.K_out = a->K_out.ptr; p.V_out = a->V_out.ptr;
    p.k = strides(a->K, e); p.v = strides(a->V, e); p.ko = strides(a->K_out, e); p.vo = strides(a->V_out, e);
    p.weights = a->weights; p.weights_out = a->weights_out; p.pos = a->pos; p.pos_out = a->pos_out;
    p.len = a->length; p.next_pos = a->next_pos; p.len_out = a->length_out; p.kept = a->kept;
    p.keep = a->keep; p.sink = a->sink; p.recent = a->recent;
    p.B = a->batch_sz; p.Hkv = a->num_kv_heads; p.S = a->capacity; p.S_out = a->capacity_out; p.row_bytes = (int)(D * e);
    const bool wide = aligned16(a->K, a->dtype) && aligned16(a->V, a->dtype) && p.row_bytes % 16 == 0 &&
                      (!into || (aligned16(a->K_out, a->dtype) && aligned16(a->V_out, a->dtype)));
    // CTAs that share a head's rows: a cluster of up to 8, as many as fill the SMs, of 4096 rows each at least (its barriers cost what 4096 rows do); one
    // CTA where a step's few rows leave.  The ranks stay in shared memory where they fit.
    int cl = 1;
    const bool step = !into && p.S - p.keep <= CE_PICK && ce_smem_bytes((p.S + 31) & ~31, true) <= c.max_smem - 24 * 1024;
    while (!step && cl < 8 && (cl * 49152 < p.S || (2ll * cl * p.B * p.Hkv <= c.sm_count && cl * 4096 < p.S))) cl *= 2;
    p.chunk_most = ((p.S + cl - 1) / cl + 31) & ~31;
    p.cached = ce_smem_bytes(p.chunk_most, true) <= (c.max_smem - 24 * 1024) / (p.chunk_most <= 8192 ? 2 : 1);
    rc = wide ? launch_evict<uint4>(p, c, cl, st) : e == 4 ? launch_evict<uint32_t>(p, c, cl, st) : launch_evict<uint16_t>(p, c, cl, st);
    if (rc) return rc;
    return host_end(&c, st, a->flags & B200ATTN_FLAG_ASYNC);
}

}  // namespace
}  // namespace b200attn

using namespace b200attn;

extern "C" {

int b200attn_cache_attend(const b200attn_attend_args *args) { return attend(args, nullptr); }
size_t b200attn_cache_attend_workspace(const b200attn_attend_args *args) {
    size_t need = 0;
    return attend(args, &need) == B200ATTN_OK ? (fail(B200ATTN_OK, "%s", ""), need) : 0;
}
int b200attn_cache_commit(const b200attn_commit_args *args) { return commit(args); }
int b200attn_cache_weights(const b200attn_weights_args *args) { return weights(args); }
int b200attn_cache_evict(const b200attn_evict_args *args) { return evict(args); }

}  // extern "C"
