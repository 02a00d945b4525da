// A key/value cache: attention of new tokens over it and its upkeep (include/b200attn.h, "A key/value cache").  This file has the
// share-out of the attention's work, the kernels that join its parts, the CUDA-core kernels that take every shape, and commit and eviction.
//
// Attention, for the rows r = t G + g of a key head (G query heads share it), visible keys j:
//     s_rj = scale q_r . k_j,   lse_r = log sum_j exp(s_rj),   out_r = sum_j exp(s_rj - lse_r) v_j.
// One pass over the keys with a running maximum m and sum l: when m grows to m', l and the accumulator are multiplied by exp(m - m').
// Parts over different keys join by the same rule.  Exponents are differences of scores, times scale log2 e; where one is taken as s c - m with m = s' c rounded
// (one multiply-add), m has to be below CA_EXACT: from there on its rounding alone is more than an exponential takes.
//
// Sharing out: a unit is (sequence, key head, tile of RT rows); its items are the tiles of TK cached keys, then those of the new tokens' keys.  In front of
// them stand OH items without work: what a unit's beginning and end cost a CTA, in tiles (short sequences would be taken for cheap otherwise).
// The lengths are in device memory and differ, so no split can be chosen on the host: the items of all units, one after the other, are cut
// into equal contiguous ranges, one per CTA, by each CTA for itself (a scan over the lengths).  A unit inside one range is finished there; one
// that is cut leaves (accumulator, m, l) per row in the CTA's two slots of the workspace - only the first and the last unit of a range can be
// cut - and ca_combine_kernel joins the parts in the order of their CTAs: no atomics, the same result every time.
#pragma once

#include <type_traits>

#include "tc_common.cuh"

namespace b200attn {

constexpr int CA_MAX_D = 256;
constexpr float CA_EXACT = 16777216.0f;   // 2^24: rounded by half at the most

// the reference m (log2 units) of a row is one that the differences of scores have to be taken from first; not that of a row that has seen nothing (-inf)
__device__ __forceinline__ bool ca_large(float m) { return fabsf(m) >= CA_EXACT && fabsf(m) < INFINITY; }

struct CaView { long long b, h, l; };   // strides in elements

struct CaParams {
    const void *Q, *K, *V, *Kd, *Vd;
    void *O;
    CaView q, k, v, kd, vd, o;
    float *lse;
    const int *len;
    const unsigned char *mask;
    long long mask_b;
    int B, Hq, Hkv, G, T, S, D;
    int R;               // rows of a key head: T * G
    int RT, nrt, TK;     // rows of a unit, units of a key head, keys of a tile
    int OH;              // items in front of a unit's tiles
    int uncut;           // a unit belongs as a whole to the range that its first item is in: nothing to join
    long long DT;        // tiles of new keys, summed over the units of a key head
    int drafts;          // new keys are given
    int grid;            // CTAs that share the items out
    float scale_log2;    // scale * log2(e)
    float *part;         // [grid][2] slots of [RT][D] accumulators and [RT][2] (m in log2 units, l)
    int *entries;        // [8] words each: cut units (ca_entry_of_unit, ca_entry_of_cta)
    int by_cta;          // ... per CTA, else per unit
    int join_rows;       // rows that a block of ca_combine_kernel joins
    unsigned *err, *err_sys;
    unsigned spin_limit, wait_extra;   // wait_extra: test hook
};

__host__ __device__ inline size_t ca_slot_floats(int RT, int D) { return ((size_t)RT * (D + 2) + 3) & ~(size_t)3; }

// rows cached for a sequence
__device__ __forceinline__ int ca_len(const int *len, int b, int S) { return min(max(__ldg(len + b), 0), S); }
// tiles of cached keys (a call without new keys has one at least, so that every unit has a tile)
__device__ __forceinline__ int ca_tiles(const CaParams &p, int n) {
    const int ct = (n + p.TK - 1) / p.TK;
    return p.drafts ? ct : max(ct, 1);
}
// tiles of new keys of unit rt: the last row of a chain sees its own token last
__host__ __device__ inline int ca_draft_tiles(int rt, int R, int RT, int G, int T, int TK, bool chain) {
    const long long end = (long long)(rt + 1) * RT;
    const int t = chain ? (int)(((end < R ? end : R) - 1) / G) + 1 : T;
    return (t + TK - 1) / TK;
}
__device__ __forceinline__ int ca_draft_tiles(const CaParams &p, int rt) {
    return p.drafts ? ca_draft_tiles(rt, p.R, p.RT, p.G, p.T, p.TK, p.mask == nullptr) : 0;
}

struct CaStart { long long total; int b; int grid; long long rem; };   // all items; where a CTA's range begins: sequence, item within it; CTAs with work

__device__ __forceinline__ long long ca_range(long long total, int grid, int c) { return total * c / grid; }
__device__ __forceinline__ int ca_cta_of(long long total, int grid, long long i) { return (int)(((i + 1) * grid - 1) / total); }

// By one whole warp: where the range of CTA `c` begins.
__device__ __forceinline__ CaStart ca_locate(const CaParams &p, int c) {
    const int lane = threadIdx.x & 31;
    long long total = 0;
    for (int b0 = 0; b0 < p.B; b0 += 32) {
        long long x = b0 + lane < p.B ? (long long)p.Hkv * ((long long)p.nrt * (p.OH + ca_tiles(p, ca_len(p.len, b0 + lane, p.S))) + p.DT) : 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        total += x;
    }
    CaStart s{total, 0, (int)min((long long)p.grid, total), 0};
    if (c >= s.grid) return s;
    const long long i0 = ca_range(total, s.grid, c);
    long long before = 0;
    for (int b0 = 0; b0 < p.B; b0 += 32) {
        const long long x = b0 + lane < p.B ? (long long)p.Hkv * ((long long)p.nrt * (p.OH + ca_tiles(p, ca_len(p.len, b0 + lane, p.S))) + p.DT) : 0;
        long long incl = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        const unsigned past = __ballot_sync(0xffffffffu, before + incl > i0);
        if (past) {
            const int at = __ffs(past) - 1;
            s.b = b0 + at;
            s.rem = i0 - before - __shfl_sync(0xffffffffu, incl - x, at);
            return s;
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
    }
    return s;   // (not reached: i0 < total)
}

// The units of a CTA's range, one after the other.
struct CaWalk {
    long long left, u0;   // items left of the range; first item of the unit, counted over all
    int b, h, rt, n;      // the unit; rows cached
    int at, ct, nt;       // first item of this CTA in the unit; tiles of cached keys; all tiles
    __device__ __forceinline__ void unit(const CaParams &p) { nt = ct + ca_draft_tiles(p, rt); }
    __device__ __forceinline__ int tile(const CaParams &p) const { return max(at - p.OH, 0); }
    __device__ __forceinline__ int end(const CaParams &p) const { return p.uncut ? nt : (int)min((long long)nt, at + left - p.OH); }
    __device__ __forceinline__ bool whole(const CaParams &p) const { return p.uncut || (at <= p.OH && at + left >= p.OH + nt); }
    __device__ __forceinline__ void settle(const CaParams &p) {   // a range that ends before a unit's first tile has no part in it
        if (!p.uncut && at + left <= p.OH) left = 0;
    }
    __device__ __forceinline__ void start(const CaParams &p, const CaStart &s, int c) {
        const long long i0 = ca_range(s.total, s.grid, c);
        left = c < s.grid ? ca_range(s.total, s.grid, c + 1) - i0 : 0;
        if (left == 0) return;
        b = s.b;
        n = ca_len(p.len, b, p.S);
        ct = ca_tiles(p, n);
        const long long per = (long long)p.nrt * (p.OH + ct) + p.DT;
        h = (int)(s.rem / per);
        long long rem = s.rem % per;
        for (rt = 0;; ++rt) {
            unit(p);
            if (rem < p.OH + nt) break;
            rem -= p.OH + nt;
        }
        at = (int)rem;
        u0 = i0 - rem;
        if (p.uncut && at > 0) next(p);   // (another range's unit)
        settle(p);
    }
    __device__ __forceinline__ void next(const CaParams &p) {
        left -= min(left, (long long)p.OH + nt - at);
        if (left == 0) return;
        u0 += p.OH + nt;
        at = 0;
        if (++rt == p.nrt) {
            rt = 0;
            if (++h == p.Hkv) {
                h = 0;
                ++b;
                n = ca_len(p.len, b, p.S);
                ct = ca_tiles(p, n);
            }
        }
        unit(p);
        settle(p);
    }
};

// What ca_combine_kernel goes by, {first CTA of a cut unit or -1, its slot, last CTA, b, h, rt}; every other part is in slot 0 of its CTA.  Kept per unit where
// there are no more units than CTAs: written by the CTA with the unit's first tile, which calls this for each of its units ...
__device__ __forceinline__ void ca_entry_of_unit(const CaParams &p, const CaStart &s, const CaWalk &w, int c, bool first_of_range) {
    if (p.uncut || p.by_cta || w.tile(p) != 0) return;
    int *e = p.entries + (((size_t)w.b * p.Hkv + w.h) * p.nrt + w.rt) * 8;
    e[1] = first_of_range ? 0 : 1;
    e[2] = ca_cta_of(s.total, s.grid, w.u0 + p.OH + w.nt - 1);
    e[3] = w.b; e[4] = w.h; e[5] = w.rt;
    e[0] = w.whole(p) ? -1 : c;
}
// By a CTA that gives up in the unit `w` is at: the entries that it has not written yet.  The joining launch comes all the same, and takes addresses from them.
__device__ __forceinline__ void ca_entries_left(const CaParams &p, const CaStart &s, CaWalk &w, int c, int seg) {
    for (; w.left > 0; ++seg, w.next(p)) ca_entry_of_unit(p, s, w, c, seg == 0);
}
// ... else per CTA: by each CTA for the first unit of its range, which is listed where it was cut by this range's beginning and by none before it.
__device__ __forceinline__ void ca_entry_of_cta(const CaParams &p, const CaStart &s, const CaWalk &w, int c) {
    if (p.uncut || !p.by_cta) return;
    int *e = p.entries + (size_t)c * 8;
    e[0] = -1;
    if (w.left == 0 || w.at <= p.OH) return;
    const int first = ca_cta_of(s.total, s.grid, w.u0 + p.OH);
    if (ca_cta_of(s.total, s.grid, w.u0 + w.at - 1) != first) return;
    e[1] = ca_range(s.total, s.grid, first) >= w.u0 ? 0 : 1;
    e[2] = ca_cta_of(s.total, s.grid, w.u0 + p.OH + w.nt - 1);
    e[3] = w.b; e[4] = w.h; e[5] = w.rt;
    e[0] = first;
}

template <typename T>
__device__ __forceinline__ T *ca_row(void *base, const CaView &v, int b, int h, long long l) {
    return reinterpret_cast<T *>(base) + b * v.b + h * v.h + l * v.l;
}
template <typename T>
__device__ __forceinline__ const T *ca_row(const void *base, const CaView &v, int b, int h, long long l) {
    return reinterpret_cast<const T *>(base) + b * v.b + h * v.h + l * v.l;
}

// ---- values that are not finite -----------------------------------------------------------------------------------------
// A weight is above 0, but may be rounded to 0, and 0 times an infinite value is NaN.  So a result that is NaN, though no score of its row was, is looked at
// again where it was written: the values that the row sees in that column decide, whatever they weigh.
constexpr unsigned CA_POS = 1, CA_NEG = 2, CA_NAN = 4;
__device__ __forceinline__ unsigned ca_kind(float v) { return fabsf(v) < INFINITY ? 0u : v != v ? CA_NAN : v > 0.0f ? CA_POS : CA_NEG; }
// a sum of values of these kinds: an infinity where all that are not finite have one sign
template <typename T>
__device__ __forceinline__ void ca_settle(T *sum, unsigned kinds) {
    const float x = to_f32(*sum);
    if (x != x && (kinds == CA_POS || kinds == CA_NEG)) *sum = OutCvt<T>::one(kinds == CA_POS ? INFINITY : -INFINITY);
}
// By one thread: the kinds of column d of the new tokens [j0, j1) that token t sees.
template <typename T>
__device__ unsigned ca_new_kinds(const CaParams &p, int b, int h, int j0, int j1, int t, int d) {
    unsigned kinds = 0;
    for (int j = j0; j < j1; ++j)
        if (p.mask ? p.mask[b * p.mask_b + (long long)t * p.T + j] != 0 : j <= t) kinds |= ca_kind(to_f32(ca_row<T>(p.Vd, p.vd, b, h, j)[d]));
    return kinds;
}

// ---- joining the parts of cut units ---------------------------------------------------------------------------------
// Block (c, y): rows join_rows y .. of the unit that entry c lists.  A row is taken by `per` warps that share its parts out, so that a row cut over the whole
// chip (one sequence, one key head) does not wait for one part after the other; a warp asks for its first four parts' accumulators before it knows their
// weights, which it takes from all parts' (m, l), a part per lane.
//   16 units x 7 rows in some 40 parts each: 40 us with 16 rows a block, one after the other; 8 x 4 rows in 7 parts: 11 us with a chain through the parts
constexpr int CB_THREADS = 256;

template <typename T, int NI>   // NI: columns of a lane
__global__ void __launch_bounds__(CB_THREADS)
ca_combine_kernel(const CaParams p) {
    __shared__ float s_acc[8][NI * 32];
    grid_launch_dependents();
    grid_dependency_wait();
    const int4 e0 = *reinterpret_cast<const int4 *>(p.entries + (size_t)blockIdx.x * 8);
    const int2 e1 = *reinterpret_cast<const int2 *>(p.entries + (size_t)blockIdx.x * 8 + 4);
    const int first = e0.x;
    if (first < 0) return;
    const int slot0 = e0.y, parts = e0.z - first + 1, b = e0.w, h = e1.x, rt = e1.y;
    const int row0 = blockIdx.y * p.join_rows, rows = min(min(p.RT, p.R - rt * p.RT), row0 + p.join_rows);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per = parts <= 4 ? 1 : parts <= 8 ? 2 : parts <= 16 ? 4 : 8;   // warps of a row
    const size_t slot = ca_slot_floats(p.RT, p.D), ml = (size_t)p.RT * p.D;
    auto part = [&](int c) { return p.part + ((size_t)(first + c) * 2 + (c == 0 ? slot0 : 0)) * slot; };
    for (int r0 = row0; r0 < rows; r0 += 8 / per) {
        const int row = min(r0 + warp / per, rows - 1), w0 = warp % per;
        const bool mine = r0 + warp / per < rows;
        float acc[NI], o[4][NI], m = -INFINITY, l = 0.0f;
        auto ask = [&](int k0) {   // parts k0, k0 + per, ..
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float *from = part(min(k0 + u * per, parts - 1)) + (size_t)row * p.D;
#pragma unroll
                for (int i = 0; i < NI; ++i) o[u][i] = lane + 32 * i < p.D ? from[lane + 32 * i] : 0.0f;
            }
        };
        ask(w0);
#pragma unroll
        for (int i = 0; i < NI; ++i) acc[i] = 0.0f;
        float2 x = make_float2(-INFINITY, 0.0f);   // of part `lane`
        if (lane < parts) x = *reinterpret_cast<const float2 *>(part(lane) + ml + 2 * row);
        m = x.x;
        for (int c = lane + 32; c < parts; c += 32) m = fmaxf(m, part(c)[ml + 2 * row]);
        m = warp_max(m);
        for (int c0 = 0; c0 < parts; c0 += 32) {
            if (c0 > 0) {
                x = make_float2(-INFINITY, 0.0f);
                if (c0 + lane < parts) x = *reinterpret_cast<const float2 *>(part(c0 + lane) + ml + 2 * row);
            }
            const float w = x.x == -INFINITY ? 0.0f : exp2f(x.x - m);
            l += w * x.y;
            for (int k0 = c0 + w0; k0 < min(c0 + 32, parts); k0 += 4 * per) {   // (32 is a multiple of 4 per)
                if (k0 != w0) ask(k0);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int k = k0 + u * per;
                    const float wk = __shfl_sync(0xffffffffu, w, (k - c0) & 31);
                    if (k < parts) {
#pragma unroll
                        for (int i = 0; i < NI; ++i) acc[i] = fmaf(o[u][i], wk, acc[i]);
                    }
                }
            }
        }
        l = warp_sum(l);
        if (per > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NI; ++i) s_acc[warp][lane + 32 * i] = acc[i];
            __syncthreads();
            if (w0 != 0) continue;
            for (int w = warp + 1; w < warp + per; ++w)
#pragma unroll
                for (int i = 0; i < NI; ++i) acc[i] += s_acc[w][lane + 32 * i];
        }
        if (!mine) continue;
        bool odd = false;
#pragma unroll
        for (int i = 0; i < NI; ++i) odd |= acc[i] != acc[i];
        if (odd && l == l) {   // (a part's weight may be rounded to 0, too)
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                unsigned kinds = 0;
                for (int k = 0; k < parts && acc[i] != acc[i]; ++k) kinds |= ca_kind(part(k)[(size_t)row * p.D + lane + 32 * i]);
                ca_settle(&acc[i], kinds);
            }
        }
        const int r = rt * p.RT + row, t = r / p.G, hq = h * p.G + r % p.G;
        T *out = ca_row<T>(p.O, p.o, b, hq, t);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int i = 0; i < NI; ++i)
            if (lane + 32 * i < p.D) out[lane + 32 * i] = OutCvt<T>::one(acc[i] * inv);
        if (p.lse && lane == 0) p.lse[((long long)b * p.Hq + hq) * p.T + t] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
    }
}

// ---- attention on the CUDA cores: every type, width and stride ---------------------------------------------------------
// Units of 16 rows, tiles of 64 keys, 128 threads.  K and V pass through shared memory in fp32: with FAST (fp32 rows on 16 bytes) by asynchronous copies, the
// next tile's K under this one's softmax and products with V, its V under the next scores; else through registers.  A thread computes the scores of one
// key with eight rows, then owns 16 outputs (8 rows of one column up to head_d 64, else 16 rows) per 128 columns.  Bound by shared-memory reads: nine of 16 bytes
// per 32 multiply-adds of a score.
//   2 x 8 heads, 7 tokens, 1501 and 2999 rows cached, head_d 64, fp32 (18.5 MB): 40 us with element-wise loads, one after the other
constexpr int CG_ROWS = 16, CG_KEYS = 64, CG_THREADS = 128;
constexpr int CG_OH = 0;   // items in front of a unit's tiles (1: 72 us instead of 58, before the copies were asynchronous)
__host__ __device__ constexpr int cg_pitch(int D) { return (((D + 3) >> 2) | 1) << 2; }   // floats: whole 16 bytes, an odd number of them
constexpr size_t CG_STATIC_SMEM = 256;   // of a kernel below, at the most
inline size_t cg_smem_bytes(int D) { return ((size_t)(CG_ROWS + 2 * CG_KEYS) * cg_pitch(D) + CG_KEYS * (CG_ROWS + 4)) * sizeof(float); }

__device__ __forceinline__ void cg_copy16(float *dst, const void *src, bool there) {   // zeros where there is nothing to copy
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cg_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cg_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// 64 rows of a head from row j0 on into `dst`, those from n on as zeros; the columns behind head_d are zero already where FAST.
template <typename T, bool FAST>
__device__ __forceinline__ void cg_load(float *dst, const void *base, const CaView &v, int b, int h, int j0, int n, int D, int S) {
    const int pitch = cg_pitch(D), tid = threadIdx.x;
    const T *rows = ca_row<T>(base, v, b, h, 0);
    if (FAST) {
        const int pieces = D >> 2;
        for (int i = tid; i < CG_KEYS * pieces; i += CG_THREADS) {
            const int j = i / pieces, c = i - j * pieces;
            cg_copy16(dst + j * pitch + 4 * c, rows + min(j0 + j, S - 1) * v.l + 4 * c, j < n);
        }
        cg_commit();
    } else {
        for (int i0 = tid; i0 < CG_KEYS * pitch; i0 += 8 * CG_THREADS) {   // eight elements' requests in flight
            float x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int i = i0 + k * CG_THREADS, j = i / pitch, d = i - j * pitch;
                x[k] = i < CG_KEYS * pitch && j < n && d < D ? to_f32(rows[(j0 + j) * v.l + d]) : 0.0f;
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (i0 + k * CG_THREADS < CG_KEYS * pitch) dst[i0 + k * CG_THREADS] = x[k];
        }
    }
}
// Scores of a key's row with the first M of eight rows, four running sums each.
template <int M>
__device__ __forceinline__ void cg_scores(const float *q, const float *k, int pitch, float (&s)[8]) {
    float4 a[M];
#pragma unroll
    for (int r = 0; r < M; ++r) a[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int d = 0; d < pitch - 3; d += 4) {
        const float4 k4 = *reinterpret_cast<const float4 *>(k + d);
#pragma unroll
        for (int r = 0; r < M; ++r) {
            const float4 q4 = *reinterpret_cast<const float4 *>(q + r * pitch + d);
            a[r].x = fmaf(q4.x, k4.x, a[r].x); a[r].y = fmaf(q4.y, k4.y, a[r].y);
            a[r].z = fmaf(q4.z, k4.z, a[r].z); a[r].w = fmaf(q4.w, k4.w, a[r].w);
        }
    }
#pragma unroll
    for (int r = 0; r < M; ++r) s[r] = (a[r].x + a[r].y) + (a[r].z + a[r].w);
}
__device__ __forceinline__ void cg_scores(const float *q, const float *k, int pitch, float (&s)[8], int rows) {   // (rows: the same for a warp)
#pragma unroll
    for (int r = 0; r < 8; ++r) s[r] = 0.0f;
    if (rows <= 2) cg_scores<2>(q, k, pitch, s);
    else if (rows <= 4) cg_scores<4>(q, k, pitch, s);
    else cg_scores<8>(q, k, pitch, s);
}

// By one thread: column d of `n` rows, the first of them row r0 of the key head, whose sums over cached rows [j0, j1) and new tokens [u0, u1) were written to the
// output or, as parts, from `part` on.  `l`: the rows' sums of weights (NaN: a score was NaN).
template <typename T>
__device__ __noinline__ void cg_settle(const CaParams &p, int b, int h, int r0, int n, int j0, int j1, int u0, int u1, int d, const float *l, float *part) {
    const T *v = ca_row<T>(p.V, p.v, b, h, 0) + d;
    unsigned cached = 0;
#pragma unroll 8
    for (int j = j0; j < j1; ++j) cached |= ca_kind(to_f32(v[j * p.v.l]));
    for (int r = 0; r < n; ++r) {
        if (l[r] != l[r]) continue;
        const int t = (r0 + r) / p.G;
        const unsigned kinds = cached | ca_new_kinds<T>(p, b, h, u0, u1, t, d);
        if (part) ca_settle(part + (size_t)r * p.D + d, kinds);
        else ca_settle(ca_row<T>(p.O, p.o, b, h * p.G + (r0 + r) % p.G, t) + d, kinds);
    }
}

template <typename T, int DB, bool FAST>   // DB: columns rounded up to 64, 128 or 256
__global__ void __launch_bounds__(CG_THREADS)
ca_generic_kernel(const __grid_constant__ CaParams p) {
    extern __shared__ __align__(16) float cg_smem[];
    __shared__ CaStart s_start;
    __shared__ float s_m[CG_ROWS], s_l[CG_ROWS], s_f[CG_ROWS];
    const int pitch = cg_pitch(p.D), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    float *qs = cg_smem, *ks = qs + CG_ROWS * pitch, *vs = ks + CG_KEYS * pitch, *ps = vs + CG_KEYS * pitch;   // ps [64 keys][16 rows + 4]
    constexpr int PP = CG_ROWS + 4;
    constexpr int NC = DB <= 128 ? 1 : 2, NR = DB <= 64 ? 8 : 16;
    if (FAST)   // the columns behind head_d, once
        for (int i = tid; i < 2 * CG_KEYS * (pitch - p.D); i += CG_THREADS) ks[i / (pitch - p.D) * pitch + p.D + i % (pitch - p.D)] = 0.0f;
    grid_launch_dependents();
    grid_dependency_wait();
    if (warp == 0) {
        const CaStart s = ca_locate(p, blockIdx.x);
        if (lane == 0) s_start = s;
    }
    __syncthreads();
    CaWalk w;
    w.start(p, s_start, blockIdx.x);
    if (tid == 0) ca_entry_of_cta(p, s_start, w, blockIdx.x);
    const int col = DB <= 64 ? (tid & 63) : tid, rbase = DB <= 64 ? (tid >> 6) * 8 : 0;
    for (bool first = true; w.left > 0; first = false) {
        const int row0 = w.rt * p.RT, rows = min(p.RT, p.R - row0), end = w.end(p);
        if (tid == 0) ca_entry_of_unit(p, s_start, w, blockIdx.x, first);
        auto keys = [&](int tile) { return min(CG_KEYS, tile >= w.ct ? p.T - (tile - w.ct) * CG_KEYS : w.n - tile * CG_KEYS); };   // (0: an empty cache)
        auto load = [&](float *dst, bool v, int tile) {
            const bool draft = tile >= w.ct;
            cg_load<T, FAST>(dst, draft ? (v ? p.Vd : p.Kd) : (v ? p.V : p.K), draft ? (v ? p.vd : p.kd) : (v ? p.v : p.k), w.b, w.h, (draft ? tile - w.ct : tile) * CG_KEYS,
                             keys(tile), p.D, draft ? p.T : p.S);
        };
        __syncthreads();
        load(ks, false, w.tile(p));
        load(vs, true, w.tile(p));
        for (int i0 = tid; i0 < CG_ROWS * pitch; i0 += 4 * CG_THREADS) {
            float x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = i0 + k * CG_THREADS, r = i / pitch, d = i - r * pitch;
                x[k] = r < rows && d < p.D ? to_f32(ca_row<T>(p.Q, p.q, w.b, w.h * p.G + (row0 + r) % p.G, (row0 + r) / p.G)[d]) : 0.0f;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i0 + k * CG_THREADS < CG_ROWS * pitch) qs[i0 + k * CG_THREADS] = x[k];
        }
        if (tid < CG_ROWS) { s_m[tid] = -INFINITY; s_l[tid] = 0.0f; }
        float acc[NC][NR];
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int r = 0; r < NR; ++r) acc[c][r] = 0.0f;
        for (int tile = w.tile(p); tile < end; ++tile) {
            const bool draft = tile >= w.ct;
            const int j0 = (draft ? tile - w.ct : tile) * CG_KEYS, nk = keys(tile);
            cg_wait<1>();   // K; V may still be on its way
            __syncthreads();
            {   // scores of key j with rows rb .. rb + 7; what a row does not see is -inf
                const int j = tid & 63, rb = (tid >> 6) * 8;
                if (rb < rows) {   // (the same for a warp)
                    float s[8];
                    cg_scores(qs + rb * pitch, ks + j * pitch, pitch, s, rows - rb);
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        bool see = j < nk && rb + r < rows;
                        if (see && draft) {
                            const int t = (row0 + rb + r) / p.G;
                            see = p.mask ? p.mask[w.b * p.mask_b + (long long)t * p.T + j0 + j] != 0 : j0 + j <= t;
                        }
                        ps[j * PP + rb + r] = see ? s[r] : -INFINITY;
                    }
                }
            }
            __syncthreads();
            if (tile + 1 < end) load(ks, false, tile + 1);
            else if (FAST) cg_commit();   // (an empty group: the counts below stay the same)
            for (int r = warp; r < rows; r += CG_THREADS / 32) {
                const float a = ps[lane * PP + r], b = ps[(lane + 32) * PP + r], mo = s_m[r];   // (maxima of q . k, not yet scaled)
                const float mn = fmaxf(mo, warp_max(fmaxf(a, b)));
                const float ea = a == -INFINITY ? -0.0f : exp2f((a - mn) * p.scale_log2), eb = b == -INFINITY ? -0.0f : exp2f((b - mn) * p.scale_log2);
                const float sum = warp_sum(ea + eb);
                ps[lane * PP + r] = ea;
                ps[(lane + 32) * PP + r] = eb;
                if (lane == 0) {
                    const float f = mn == -INFINITY ? 0.0f : exp2f((mo - mn) * p.scale_log2);
                    s_f[r] = f;
                    s_l[r] = s_l[r] * f + sum;
                    s_m[r] = mn;
                }
            }
            cg_wait<1>();   // V; the next K may still be on its way
            __syncthreads();
            if (rbase < rows) {
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int c = 0; c < NC; ++c) acc[c][r] *= s_f[rbase + r];
                // four rows at a time, as many as there are (all 16 for 4 rows: 53 us a call of 4 x 2 heads, 4 tokens, 5153 to 9476 rows, head_d 96, fp32)
#pragma unroll
                for (int r = 0; r < NR; r += 4) {
                    if (rbase + r >= rows) break;
                    const float *es = ps + rbase + r;
                    auto products = [&](auto masked) {
#pragma unroll 8
                        for (int j = 0; j < nk; ++j) {
                            const float4 e4 = *reinterpret_cast<const float4 *>(es + j * PP);
                            const float e[4] = {e4.x, e4.y, e4.z, e4.w};
#pragma unroll
                            for (int c = 0; c < NC; ++c) {
                                const float v = col + 128 * c < pitch ? vs[j * pitch + col + 128 * c] : 0.0f;
#pragma unroll
                                for (int k = 0; k < 4; ++k)
                                    // a key that the row does not see weighs -0; its value may be NaN
                                    acc[c][r + k] = decltype(masked)::value && __float_as_uint(e[k]) == 0x80000000u ? acc[c][r + k] : fmaf(e[k], v, acc[c][r + k]);
                            }
                        }
                    };
                    if (draft) products(std::true_type{});
                    else products(std::false_type{});
                }
            }
            __syncthreads();
            if (tile + 1 < end) load(vs, true, tile + 1);
            else if (FAST) cg_commit();
        }
        const bool whole = w.whole(p);
        float *part = p.part + ((size_t)blockIdx.x * 2 + (first ? 0 : 1)) * ca_slot_floats(p.RT, p.D);
        bool odd[NC] = {};
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const int rr = rbase + r;
            if (rr >= rows) continue;
            const float l = s_l[rr], inv = l == 0.0f ? 0.0f : 1.0f / l;
            T *o = whole ? ca_row<T>(p.O, p.o, w.b, w.h * p.G + (row0 + rr) % p.G, (row0 + rr) / p.G) : nullptr;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int d = col + 128 * c;
                if (d >= p.D) continue;
                odd[c] |= acc[c][r] != acc[c][r];
                if (whole) o[d] = OutCvt<T>::one(acc[c][r] * inv);
                else part[(size_t)rr * p.D + d] = acc[c][r];
            }
        }
#pragma unroll
        for (int c = 0; c < NC; ++c)
            if (odd[c])
                cg_settle<T>(p, w.b, w.h, row0 + rbase, min(NR, rows - rbase), w.tile(p) * CG_KEYS, min(w.n, min(end, w.ct) * CG_KEYS), max(w.tile(p) - w.ct, 0) * CG_KEYS,
                             min(p.T, (end - w.ct) * CG_KEYS), col + 128 * c, s_l + rbase, whole ? nullptr : part + (size_t)rbase * p.D);
        if (tid < rows) {
            const float m = s_m[tid] * p.scale_log2, l = s_l[tid];
            if (!whole) {
                part[(size_t)p.RT * p.D + 2 * tid] = m;
                part[(size_t)p.RT * p.D + 2 * tid + 1] = l;
            } else if (p.lse) {
                const int r = row0 + tid;
                p.lse[((long long)w.b * p.Hq + w.h * p.G + r % p.G) * p.T + r / p.G] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
            }
        }
        w.next(p);
    }
}

// ---- lists of accepted tokens ------------------------------------------------------------------------------------------
// By one whole warp: entries of the list in front of the first that names no token, `most` at the most.
__device__ __forceinline__ int ca_count(const int *accepted, int b, int A, int T, int most) {
    const int lane = threadIdx.x & 31;
    if (accepted == nullptr) return min(T, most);
    for (int i0 = 0; i0 < min(A, most); i0 += 32) {
        const int i = i0 + lane;
        const bool ends = i >= A || (unsigned)__ldg(accepted + (long long)b * A + i) >= (unsigned)T;
        const unsigned any = __ballot_sync(0xffffffffu, ends);
        if (any) return min(i0 + __ffs(any) - 1, most);
    }
    return min(A, most);
}

// ---- accumulated weights on the CUDA cores -------------------------------------------------------------------------------
struct CwParams {
    const void *Q, *K;
    CaView q, k;
    const int *len, *accepted;
    const float *lse;
    float *weights;
    int A;               // entries of a list; T without lists
    int B, Hq, Hkv, G, T, S, D;
    float scale_log2;
    unsigned *err, *err_sys;
    unsigned spin_limit, wait_extra;
};

constexpr size_t cw_smem_bytes(int D, bool fast) { return (size_t)(CG_KEYS + (fast ? 2 : 1) * CG_ROWS) * cg_pitch(D) * sizeof(float); }

// Block: 64 keys of a head; thread = key (two threads share a key's rows).  A key's sum is taken by its threads in the order of the rows; the next 16 rows
// are on their way under the present ones' products (8 heads, 142 tokens, up to 303 rows, head_d 80, fp32: 44 us with each load waited for).
template <typename T, bool FAST>
__global__ void __launch_bounds__(CG_THREADS)
cw_generic_kernel(const CwParams p) {
    extern __shared__ __align__(16) float cg_smem[];
    __shared__ float s_lse[2][CG_ROWS], s_half[CG_KEYS];
    __shared__ int s_i[2][CG_ROWS];
    const int pitch = cg_pitch(p.D), tid = threadIdx.x;
    float *ks = cg_smem, *qs = ks + CG_KEYS * pitch;   // qs: two buffers where FAST
    grid_launch_dependents();
    grid_dependency_wait();
    const int b = blockIdx.z, h = blockIdx.y, j0 = blockIdx.x * CG_KEYS;
    const int n = ca_len(p.len, b, p.S);
    if (j0 >= n) return;
    const int count = ca_count(p.accepted, b, p.A, p.T, n);
    if (count == 0) return;
    if (FAST)   // the columns behind head_d, once
        for (int i = tid; i < (CG_KEYS + 2 * CG_ROWS) * (pitch - p.D); i += CG_THREADS) ks[i / (pitch - p.D) * pitch + p.D + i % (pitch - p.D)] = 0.0f;
    cg_load<T, FAST>(ks, p.K, p.k, b, h, j0, min(CG_KEYS, n - j0), p.D, p.S);
    const int j = tid & 63, rb = (tid >> 6) * 8, rows = count * p.G;
    const int *list = p.accepted ? p.accepted + (long long)b * p.A : nullptr;
    // 16 rows from r0 on into buffer `u`; where FAST they are on their way when this returns
    auto load = [&](int r0, int u) {
        float *dst = qs + u * CG_ROWS * pitch;
        if (tid < CG_ROWS) {
            const int r = r0 + tid, i = r / p.G;
            float x = -INFINITY;
            if (r < rows) x = p.lse[((long long)b * p.Hq + h * p.G + r - i * p.G) * p.T + (list ? list[i] : i)];
            s_i[u][tid] = x == -INFINITY ? -1 : i;   // a token that saw nothing gave no weight
            s_lse[u][tid] = x;
        }
        if (FAST) {
            const int pieces = p.D >> 2;
            for (int k = tid; k < CG_ROWS * pieces; k += CG_THREADS) {
                const int q = k / pieces, c = k - q * pieces, r = min(r0 + q, rows - 1), i = r / p.G;
                cg_copy16(dst + q * pitch + 4 * c, ca_row<T>(p.Q, p.q, b, h * p.G + r - i * p.G, list ? list[i] : i) + 4 * c, r0 + q < rows);
            }
            cg_commit();
        } else {
            for (int i0 = tid; i0 < CG_ROWS * pitch; i0 += 4 * CG_THREADS) {
                float x[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int at = i0 + k * CG_THREADS, q = at / pitch, d = at - q * pitch, r = r0 + q, i = r / p.G;
                    x[k] = q < CG_ROWS && r < rows && d < p.D ? to_f32(ca_row<T>(p.Q, p.q, b, h * p.G + r - i * p.G, list ? list[i] : i)[d]) : 0.0f;
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (i0 + k * CG_THREADS < CG_ROWS * pitch) dst[i0 + k * CG_THREADS] = x[k];
            }
        }
    };
    float sum = 0.0f;
    // rows of tokens in front of the first that sees any of these keys are left out
    const long long none = (long long)(j0 - (n - count)) * p.G;
    const int first = none <= 0 ? 0 : (int)(none / CG_ROWS * CG_ROWS);
    if (FAST) load(first, 0);
    for (int r0 = first, u = 0; r0 < rows; r0 += CG_ROWS, u ^= FAST ? 1 : 0) {
        if (!FAST) {
            __syncthreads();
            load(r0, 0);
        }
        cg_wait<0>();
        __syncthreads();   // (and everybody is done with the other buffer)
        if (FAST && r0 + CG_ROWS < rows) load(r0 + CG_ROWS, u ^ 1);
        if (r0 + rb >= rows) continue;   // (the same for a warp)
        float s[8];
        cg_scores(qs + (u * CG_ROWS + rb) * pitch, ks + j * pitch, pitch, s, rows - r0 - rb);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const int i = s_i[u][rb + r];
            if (i >= 0 && j0 + j <= n - count + i) sum += exp2f(fmaf(s[r], p.scale_log2, -1.4426950408889634f * s_lse[u][rb + r]));
        }
    }
    if (tid >= 64) s_half[j] = sum;
    __syncthreads();
    if (tid < 64 && j0 + j < n) p.weights[((long long)b * p.Hkv + h) * p.S + j0 + j] += sum + s_half[j];
}

// ---- rows from one place to another ------------------------------------------------------------------------------------
// A warp copies `n` pairs of rows (of K and of V) of `bytes` bytes in pieces of type P (16 bytes, or an element where rows are not that aligned):
// lanes share a row out as far as it has pieces, and four passes' pieces are in flight at once.  `at(i, ks, kd, vs, vd)` says where row i is and goes.
template <typename P, typename At>
__device__ __forceinline__ void ca_copy_rows(int n, int bytes, int lane, At at) {
    const int pieces = bytes / (int)sizeof(P);
    int L = 32;                       // lanes of a row
    while (L > 1 && L / 2 >= pieces) L >>= 1;
    const int per = 32 / L, sub = lane / L;
    for (int i0 = 0; i0 < n; i0 += 4 * per) {
        const P *ks[4], *vs[4];
        P *kd[4], *vd[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = i0 + u * per + sub;
            if (i < n) at(i, ks[u], kd[u], vs[u], vd[u]);
        }
        for (int c = lane % L; c < pieces; c += L) {
            P k[4], v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i0 + u * per + sub < n) { k[u] = ks[u][c]; v[u] = vs[u][c]; }
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i0 + u * per + sub < n) { kd[u][c] = k[u]; vd[u][c] = v[u]; }
        }
    }
}

struct CcParams {
    void *K, *V;
    const void *Kd, *Vd;
    CaView k, v, kd, vd;   // strides in bytes
    const int *len, *accepted, *next_pos;
    int *len_out, *pos;
    float *weights;
    int A, B, Hkv, T, S, row_bytes;
    int groups;            // of CC_ROWS entries of a list
};
constexpr int CC_THREADS = 256, CC_ROWS = 16;

// A warp per (head, 16 accepted tokens), sequences along y: bound by memory where a prompt enters, else by the launch.
//   4 x 8 heads, 2000 tokens, fp32, head_d 64 (66 MB): 22 us with a warp per row
template <typename P>
__global__ void __launch_bounds__(CC_THREADS)
cc_commit_kernel(const CcParams p) {
    grid_launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, b = blockIdx.y;
    const int n = ca_len(p.len, b, p.S);
    const long long wid = (long long)blockIdx.x * (CC_THREADS / 32) + (threadIdx.x >> 5);
    if (wid == 0 && p.len_out) {
        const int count = ca_count(p.accepted, b, p.A, p.T, p.S - n);
        if (lane == 0) p.len_out[b] = n + count;
    }
    if (wid >= (long long)p.groups * p.Hkv) return;
    const int h = (int)(wid / p.groups), first = (int)(wid % p.groups) * CC_ROWS;
    const int rows = ca_count(p.accepted, b, p.A, p.T, min(first + CC_ROWS, p.S - n)) - first;
    if (rows <= 0) return;
    const int *list = p.accepted ? p.accepted + (long long)b * p.A : nullptr;
    char *K = (char *)p.K + b * p.k.b + h * p.k.h + (long long)(n + first) * p.k.l, *V = (char *)p.V + b * p.v.b + h * p.v.h + (long long)(n + first) * p.v.l;
    const char *Kd = (const char *)p.Kd + b * p.kd.b + h * p.kd.h, *Vd = (const char *)p.Vd + b * p.vd.b + h * p.vd.h;
    ca_copy_rows<P>(rows, p.row_bytes, lane, [&](int i, const P *&ks, P *&kd, const P *&vs, P *&vd) {
        const long long t = list ? __ldg(list + first + i) : first + i;
        ks = (const P *)(Kd + t * p.kd.l); kd = (P *)(K + i * p.k.l);
        vs = (const P *)(Vd + t * p.vd.l); vd = (P *)(V + i * p.v.l);
    });
    if (lane < rows) {
        const long long at = ((long long)b * p.Hkv + h) * p.S + n + first + lane;
        if (p.weights) p.weights[at] = 0.0f;
        if (p.pos) p.pos[at] = (p.next_pos ? __ldg(p.next_pos + b) : n) + first + lane;
    }
}

// ---- eviction ------------------------------------------------------------------------------------------------------------
struct CeParams {
    void *K, *V, *K_out, *V_out;     // K_out == nullptr: in place
    CaView k, v, ko, vo;             // strides in bytes
    float *weights, *weights_out;
    int *pos, *pos_out;
    const int *len, *next_pos;
    int *len_out, *kept;
    int keep, sink, recent;
    int B, Hkv, S, S_out, row_bytes;
    int chunk_most, cached;          // rows of a CTA at the most; their ranks are kept in shared memory
};

// Weights as whole numbers of the same order: NaN lowest, -0 and 0 equal; protected rows are above all of them.
__device__ __forceinline__ unsigned ce_rank(float w, bool held) {
    if (held) return 0xffffffffu;
    if (w != w) return 0u;
    const unsigned u = __float_as_uint(w == 0.0f ? 0.0f : w);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int CE_BITS = 11, CE_BINS = 1 << CE_BITS;
constexpr int CE_COPIES = 4;   // of the first histogram: most weights share a few of its digits, and additions to one word wait for each other
constexpr size_t CE_HISTS = (size_t)(CE_COPIES + 2) * CE_BINS * 4;
// the histograms; per word of 32 rows: the mask of rows that stay, that of equal rank, a number; 16 bits a row (the list of kept rows that move); the ranks
inline size_t ce_smem_bytes(int chunk, bool cached) { return CE_HISTS + (size_t)(chunk / 32) * 12 + (size_t)chunk * 2 + (cached ? (size_t)chunk * 4 : 0); }
// In place, up to this many rows a head move with ce_select_kernel itself; ce_move_kernel is not launched where the capacity allows no more.
constexpr int CE_FEW = 128;
constexpr int CE_PICK = 32;   // up to so many rows that leave are picked one by one

// Exclusive scan of one value per thread of the block, and its total.
template <int CE_THREADS>
__device__ __forceinline__ int ce_scan(int x, int *s_warp, int *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    __syncthreads();
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < CE_THREADS / 32; ++w) {
        const int v = s_warp[w];
        if (w < warp) before += v;
        all += v;
    }
    *total = all;
    return before + incl - x;
}
__device__ __forceinline__ int ce_remote(const void *p, uint32_t rank) {   // a 32-bit word of the same variable in another CTA of the cluster
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(map_to_rank(smem_u32(p), rank)) : "memory");
    return v;
}
__device__ __forceinline__ int2 ce_remote2(const void *p, uint32_t rank) {
    int2 v;
    asm volatile("ld.shared::cluster.v2.s32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(map_to_rank(smem_u32(p), rank)));
    return v;
}
__device__ __forceinline__ int ce_remote_u16(const void *p, uint32_t rank) {
    unsigned short v;
    asm volatile("ld.shared::cluster.u16 %0, [%1];" : "=h"(v) : "r"(map_to_rank(smem_u32(p), rank)) : "memory");
    return v;
}
__device__ __forceinline__ void ce_cluster_sync(uint32_t cl) {
    if (cl > 1) { cluster_arrive(); cluster_wait(); } else __syncthreads();
}

// By one whole warp: `n` rows of a head move, pairs[2 i] to pairs[2 i + 1] (in shared memory).  In place the sources are rows >= m and the targets
// rows < m, so that no move reads what another writes.
template <typename P>
__device__ __forceinline__ void ce_move_rows(const CeParams &p, int b, int h, int n, const int *pairs) {
    const int lane = threadIdx.x & 31;
    const long long unit = (long long)b * p.Hkv + h;
    const CaView ko = p.K_out ? p.ko : p.k, vo = p.K_out ? p.vo : p.v;
    char *Ko = (char *)(p.K_out ? p.K_out : p.K) + b * ko.b + h * ko.h, *Vo = (char *)(p.K_out ? p.V_out : p.V) + b * vo.b + h * vo.h;
    const char *K = (const char *)p.K + b * p.k.b + h * p.k.h, *V = (const char *)p.V + b * p.v.b + h * p.v.h;
    ca_copy_rows<P>(n, p.row_bytes, lane, [&](int i, const P *&ks, P *&kd, const P *&vs, P *&vd) {
        const long long from = pairs[2 * i], to = pairs[2 * i + 1];
        ks = (const P *)(K + from * p.k.l); kd = (P *)(Ko + to * ko.l);
        vs = (const P *)(V + from * p.v.l); vd = (P *)(Vo + to * vo.l);
    });
    float *wo = p.K_out ? p.weights_out + unit * p.S_out : p.weights + unit * p.S;
    int *po = p.K_out ? p.pos_out + unit * p.S_out : p.pos + unit * p.S;
    for (int i = lane; i < n; i += 32) {
        wo[pairs[2 * i + 1]] = p.weights[unit * p.S + pairs[2 * i]];
        if (p.pos) po[pairs[2 * i + 1]] = p.pos[unit * p.S + pairs[2 * i]];
    }
}

// A cluster per (sequence, head), each CTA a piece of its rows, finds the rows that stay and writes `kept`:
//   the m-th largest rank by its digits from the top: three histograms over the rows that share the prefix found so far, added up over the cluster;
//   bit masks over the rows - above that rank, equal to it; of the equal rows the first that there is room for stay;
//   into another cache: the numbers of the rows that stay are their new places.  In place: the kept rows from m on are listed by their number, and the i-th
//   freed row below m takes the i-th of them, from the list of the CTA that has it.
// Where few rows leave, in place, they are picked one after the other instead: a reduction over the block each.
// Bound by latency: three passes over shared memory and some ten barriers; so a cluster's CTAs have 1024 threads (512: 48 us instead of 37 for 4 x 8 heads, up to 32768 rows), one on its
// own 512, of which two share an SM up to some 10000 rows.  Beyond 24896 rows a CTA's ranks are not kept but read anew in each pass.
//   32 sequences x 8 heads, up to 4102 rows: 22 us with 1024 threads that read weights and positions anew in each pass, 19 with the ranks in shared memory, 23
//   with two bits a round by counting; 4 x 8 heads, up to 32768 rows: 91, 33
template <typename P, int CE_THREADS>
__global__ void __launch_bounds__(CE_THREADS, 1024 / CE_THREADS)
ce_select_kernel(const CeParams p) {
    extern __shared__ __align__(16) unsigned ce_smem[];
    __shared__ int s_warp[CE_THREADS / 32], s_count[4], s_pairs[CE_FEW * 2];
    __shared__ int s_digit, s_above;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.y;
    uint32_t cl;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(cl));
    const uint32_t rank = cluster_ctarank();
    const int h = blockIdx.x / cl;
    grid_launch_dependents();
    grid_dependency_wait();
    const int n = ca_len(p.len, b, p.S), m = min(n, p.keep);
    const long long unit = (long long)b * p.Hkv + h;
    int *kept = p.kept + unit * p.keep;
    if (h == 0 && rank == 0 && tid == 0 && p.len_out) p.len_out[b] = m;
    for (int i = m + rank * CE_THREADS + tid; i < p.keep; i += cl * CE_THREADS) kept[i] = -1;
    if (n <= p.keep) {   // (the same for the whole cluster)
        for (int i = rank * CE_THREADS + tid; i < m; i += cl * CE_THREADS) kept[i] = i;
        return;
    }
    const int chunk = min((int)(((n + cl - 1) / cl + 31) & ~31), p.chunk_most);   // rows of a CTA: whole words
    const int lo = min((int)rank * chunk, n), rows = min(chunk, n - lo), words = (rows + 31) / 32;
    int *hists = (int *)ce_smem;
    unsigned *stays = ce_smem + CE_HISTS / 4, *equal = stays + p.chunk_most / 32;
    int *number = (int *)(equal + p.chunk_most / 32);
    unsigned short *list = (unsigned short *)(number + p.chunk_most / 32);
    unsigned *ranks = (unsigned *)(list + p.chunk_most);
    const float *w = p.weights + unit * p.S + lo;
    const int *pos = p.pos ? p.pos + unit * p.S + lo : nullptr;
    const int recent = (int)max((long long)(p.next_pos ? p.next_pos[b] : n) - p.recent, -0x80000000ll);
    auto rank_of = [&](int r) {   // of row lo + r
        const int at = pos ? pos[r] : lo + r;
        return ce_rank(w[r], at < p.sink || at >= recent);
    };
    const bool pick = cl == 1 && p.cached && !p.K_out && n - m <= CE_PICK;
    if (pick)
        for (int i = tid; i < m; i += CE_THREADS) kept[i] = i;   // (freed rows are put right below)
    else
        for (int i = tid; i < (CE_COPIES + 2) * CE_BINS / 4; i += CE_THREADS) reinterpret_cast<int4 *>(hists)[i] = make_int4(0, 0, 0, 0);
    if (p.cached) {
        for (int r0 = tid; r0 < rows; r0 += 8 * CE_THREADS) {   // eight rows' requests in flight
            float x[8];
            int at[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int r = min(r0 + k * CE_THREADS, rows - 1);
                x[k] = w[r];
                at[k] = pos ? pos[r] : lo + r;
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (r0 + k * CE_THREADS < rows) ranks[r0 + k * CE_THREADS] = ce_rank(x[k], at[k] < p.sink || at[k] >= recent);
        }
    }
    auto rank_at = [&](int r) { return p.cached ? ranks[r] : rank_of(r); };   // (a thread asks for the rows that it has written itself)
    unsigned prefix = 0;
    int need = m;   // rows to take from those that share the prefix
    if (pick) {
        // ---- a step's eviction: the row of least rank (of those, the last) leaves, n - m times ----
        unsigned *gone = stays, least;
        int *left = number, last;   // the rows that leave
        for (int i = tid; i < words; i += CE_THREADS) gone[i] = 0;
        __syncthreads();
        auto look = [&]() {   // at this thread's rows
            least = 0xffffffffu;
            last = -1;
            for (int r = tid; r < rows; r += CE_THREADS)
                if (ranks[r] <= least && !(gone[r >> 5] >> (r & 31) & 1u)) { least = ranks[r]; last = r; }
        };
        look();
        uint2 *s_round = reinterpret_cast<uint2 *>(hists);   // [2][warps]
        const int k = n - m;
        for (int i = 0; i < k; ++i) {
            const unsigned x = __reduce_min_sync(0xffffffffu, least);
            const int r = __reduce_max_sync(0xffffffffu, least == x ? last : -1);
            uint2 *at = s_round + (i & 1) * (CE_THREADS / 32);
            if (lane == 0) at[warp] = make_uint2(x, (unsigned)r);
            __syncthreads();
            const uint2 v = at[lane % (CE_THREADS / 32)];
            const unsigned y = __reduce_min_sync(0xffffffffu, v.x);
            const int out = __reduce_max_sync(0xffffffffu, v.x == y ? (int)v.y : -1);
            if (out % CE_THREADS == tid) {
                atomicOr(&gone[out >> 5], 1u << (out & 31));
                left[i] = out;
                look();
            }
        }
        __syncthreads();
        int holes = 0;
        if (warp == 0) {
            const int e = lane < k ? left[lane] : n;
            int before = 0;
            bool moves = lane < k;   // row m + lane stays, and moves
            for (int j = 0; j < k; ++j) {
                const int o = __shfl_sync(0xffffffffu, e, j);
                if (o < e) ++before;
                if (o == m + lane) moves = false;
            }
            const unsigned who = __ballot_sync(0xffffffffu, moves);
            if (e < m) s_pairs[2 * before + 1] = e;
            if (moves) s_pairs[2 * __popc(who & ((1u << lane) - 1u))] = m + lane;
            if (lane == 0) s_count[0] = __popc(who);
        }
        __syncthreads();
        holes = s_count[0];
        if (tid < holes) kept[s_pairs[2 * tid + 1]] = s_pairs[2 * tid];
        const int each = (holes + CE_THREADS / 32 - 1) / (CE_THREADS / 32), k0 = warp * each, k1 = min(k0 + each, holes);
        if (k0 < k1) ce_move_rows<P>(p, b, h, k1 - k0, s_pairs + 2 * k0);
        return;
    }
    __syncthreads();
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        const int bits = pass < 2 ? CE_BITS : 32 - 2 * CE_BITS, shift = pass < 2 ? 32 - (pass + 1) * CE_BITS : 0;
        int *hist = hists + (pass == 0 ? 0 : CE_COPIES + pass - 1) * CE_BINS, *copy = hist + (pass == 0 ? (warp % CE_COPIES) * CE_BINS : 0);
        for (int r0 = 0; r0 < rows; r0 += 4 * CE_THREADS) {
            unsigned x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = r0 + k * CE_THREADS + tid < rows ? rank_at(r0 + k * CE_THREADS + tid) : 0u;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const bool in = r0 + k * CE_THREADS + tid < rows && (pass == 0 || ((x[k] ^ prefix) >> (shift + bits)) == 0);
                const unsigned d = (x[k] >> shift) & ((1u << bits) - 1);
                // equal digits are common (weights of 0): those equal to the first lane's are added at once
                const unsigned who = __ballot_sync(0xffffffffu, in);
                if (who == 0) continue;
                const int leader = __ffs(who) - 1;
                const unsigned d0 = __shfl_sync(0xffffffffu, d, leader), same = __ballot_sync(0xffffffffu, in && d == d0);
                if (lane == leader) atomicAdd(&copy[d0], __popc(same));
                if (in && d != d0) atomicAdd(&copy[d], 1);
            }
        }
        // thread i has the digits CE_BINS - 1 - CE_PER i downwards, in pairs
        constexpr int CE_PER = CE_BINS / CE_THREADS, pairs = CE_PER / 2;
        int2 *mine2 = reinterpret_cast<int2 *>(hist) + (CE_THREADS - 1 - tid) * pairs;
        if (pass == 0) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < pairs; ++i) {
                int2 q = mine2[i];
#pragma unroll
                for (int k = 1; k < CE_COPIES; ++k) { q.x += mine2[k * CE_BINS / 2 + i].x; q.y += mine2[k * CE_BINS / 2 + i].y; }
                mine2[i] = q;
            }
        }
        ce_cluster_sync(cl);
        int c[CE_PER], sum = 0;
#pragma unroll
        for (int i = 0; i < pairs; ++i) {
            int2 q = mine2[i];
#pragma unroll
            for (uint32_t o = 1; o < 8; ++o) {
                if (o >= cl) break;
                const int2 v = ce_remote2(mine2 + i, (rank + o) % cl);
                q.x += v.x; q.y += v.y;
            }
            c[CE_PER - 1 - 2 * i] = q.x;
            c[CE_PER - 2 - 2 * i] = q.y;
            sum += q.x + q.y;
        }
        int all;
        int before = ce_scan<CE_THREADS>(sum, s_warp, &all);
        if (before < need && before + sum >= need) {
#pragma unroll
            for (int k = 0; k < CE_PER; ++k) {
                if (before < need && before + c[k] >= need) { s_digit = CE_BINS - 1 - CE_PER * tid - k; s_above = before; }
                before += c[k];
            }
        }
        __syncthreads();
        prefix |= (unsigned)s_digit << shift;
        need -= s_above;
    }
    int equals = 0;
#pragma unroll 4
    for (int i = warp; i < words; i += CE_THREADS / 32) {
        const int r = 32 * i + lane;
        // (with the ranks in shared memory this reads what other threads wrote: they have met since)
        const unsigned x = r < rows ? rank_at(r) : 0u;
        const unsigned gt = __ballot_sync(0xffffffffu, r < rows && x > prefix), eq = __ballot_sync(0xffffffffu, r < rows && x == prefix);
        if (lane == 0) { stays[i] = gt; equal[i] = eq; }
    }
    __syncthreads();
    const int per = (words + CE_THREADS - 1) / CE_THREADS, w0 = min(tid * per, words), w1 = min(w0 + per, words);   // words of this thread, in a row
    for (int i = w0; i < w1; ++i) equals += __popc(equal[i]);
    int all;
    int mine = ce_scan<CE_THREADS>(equals, s_warp, &all);
    // numbers over the CTAs in front of this one: `slot` of s_count in each, which the caller's total goes into
    auto in_front = [&](int total, int slot) {
        if (tid == 0) s_count[slot] = total;
        ce_cluster_sync(cl);
        int before = 0;
        for (uint32_t o = 0; o < rank; ++o) before += ce_remote(&s_count[slot], o);
        return before;
    };
    int room = need - in_front(all, 0) - mine;
    for (int i = w0; i < w1; ++i) {
        unsigned eq = equal[i];
        if (__popc(eq) <= room) {
            stays[i] |= eq;
            room -= __popc(eq);
        } else {
            for (; room > 0; --room) {
                stays[i] |= eq & -eq;
                eq &= eq - 1;
            }
        }
    }
    __syncthreads();
    // rows of word i below m
    auto front = [&](int i) {
        const int left = m - (lo + 32 * i);
        return left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
    };
    const bool into = p.K_out != nullptr;
    // the rows that are numbered: all that stay, or those of them from m on
    int count = 0;
    for (int i = w0; i < w1; ++i) count += __popc(into ? stays[i] : stays[i] & ~front(i));
    mine = ce_scan<CE_THREADS>(count, s_warp, &all);
    for (int i = w0; i < w1; ++i) {
        number[i] = mine;
        mine += __popc(into ? stays[i] : stays[i] & ~front(i));
    }
    const int base = in_front(all, 1);   // (a barrier: the numbers are there)
    __syncthreads();
#pragma unroll 4
    for (int i = warp; i < words; i += CE_THREADS / 32) {
        const unsigned bits = into ? stays[i] : stays[i] & ~front(i);
        if (bits >> lane & 1u) {
            const int at = number[i] + __popc(bits & ((1u << lane) - 1u));
            if (into) kept[base + at] = lo + 32 * i + lane;
            else list[at] = (unsigned short)(32 * i + lane);
        }
    }
    if (into) {
        ce_cluster_sync(cl);   // (nobody leaves while its counts are being read)
        return;
    }
    __syncthreads();
    // freed rows: numbered, too
    count = 0;
    for (int i = w0; i < w1; ++i) count += __popc(~stays[i] & front(i));
    mine = ce_scan<CE_THREADS>(count, s_warp, &all);
    for (int i = w0; i < w1; ++i) {
        number[i] = mine;
        mine += __popc(~stays[i] & front(i));
    }
    const int holes = in_front(all, 2);   // (a barrier: all lists are there)
    __syncthreads();
    for (int i = warp; i < words; i += CE_THREADS / 32) {
        const unsigned f = front(i), free = ~stays[i] & f;
        if (f == 0) break;
        int from = -1;
        if (f >> lane & 1u) {
            from = lo + 32 * i + lane;
            if (free >> lane & 1u) {
                int at = holes + number[i] + __popc(free & ((1u << lane) - 1u));
                uint32_t o = 0;
                for (;; ++o) {   // the CTA that has the at-th row that moves
                    const int v = cl > 1 ? ce_remote(&s_count[1], o) : s_count[1];
                    if (at < v || o + 1 == cl) break;
                    at -= v;
                }
                from = (int)o * chunk + (cl > 1 ? ce_remote_u16(&list[at], o) : list[at]);
            }
            kept[lo + 32 * i + lane] = from;
        }
        if (n - m <= CE_FEW && (free >> lane & 1u)) {
            const int k = number[i] + __popc(free & ((1u << lane) - 1u));
            s_pairs[2 * k] = from;
            s_pairs[2 * k + 1] = lo + 32 * i + lane;
        }
    }
    ce_cluster_sync(cl);   // (nobody leaves while its list is being read; the pairs are there)
    if (n - m <= CE_FEW) {
        const int each = (all + CE_THREADS / 32 - 1) / (CE_THREADS / 32), k0 = warp * each, k1 = min(k0 + each, all);
        if (k0 < k1) ce_move_rows<P>(p, b, h, k1 - k0, s_pairs + 2 * k0);
    }
}

// Moves what `kept` says: a warp per 32 rows.
template <typename P>
__global__ void __launch_bounds__(CC_THREADS)
ce_move_kernel(const CeParams p) {
    __shared__ int s_pairs[CC_THREADS * 2];
    grid_launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = blockIdx.z, h = blockIdx.y;
    const int n = ca_len(p.len, b, p.S), m = min(n, p.keep), to = (blockIdx.x * (CC_THREADS / 32) + warp) * 32 + lane;
    if (!p.K_out && n - m <= CE_FEW) return;   // (few rows have moved already)
    const int from = to < m ? p.kept[((long long)b * p.Hkv + h) * p.keep + to] : -1;
    const bool moves = from >= 0 && (p.K_out || from != to);
    const unsigned todo = __ballot_sync(0xffffffffu, moves);
    if (todo == 0) return;
    int *pairs = s_pairs + warp * 64;
    if (moves) {
        const int i = __popc(todo & ((1u << lane) - 1u));
        pairs[2 * i] = from;
        pairs[2 * i + 1] = to;
    }
    __syncwarp();
    ce_move_rows<P>(p, b, h, __popc(todo), pairs);
}

}  // namespace b200attn
