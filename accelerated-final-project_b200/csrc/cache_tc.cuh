// Attention of new tokens over a cache on the 5th-generation tensor cores: bf16 / fp16, head_d a multiple of 8, at most 256, up to 128 query
// heads a key head, 16-byte aligned rows.  The formulas and the sharing-out are those of cache.cuh.
//
// Rows (token t, query head g of the group: row t G + g) are the lanes of tensor memory, so the query heads that share a key head and the tokens of a
// tree share every key tile: a tile of K and V is read once for up to 128 rows (ca_tc_kernel<1, ..>) or 256 (<2, ..>).  The MMAs compute 128 rows whether
// they exist or not, which takes time and power where few do: up to 64 rows a key head go to cache_narrow.cuh, with keys as the lanes.
//   warp 0        one thread requests Q, K and V tiles by TMA through a ring of stages, in the order K_0 | K_1 V_0 | K_2 V_1 | ...
//   warps 1, 2    one thread per row tile issues the MMAs: S = Q K^T, then O += P V once P is there
//   warp 3        sees every V tile before the MMAs do: rows behind the cache's last are set to 0 (0 weight times NaN would be NaN); in a tile of
//                 new tokens, which some rows see and others do not, values that are not finite are set to 0 and remembered
//   warpgroups    a thread per row: scores into registers, the row's mask, running maximum and sum, P as 16-bit values to shared memory; at the end of a
//                 unit O / l to the output or (O, m, l) to the workspace.  Values that warp 3 took out are added for the rows that see them, and sums that an
//                 infinite cached value times a weight rounded to 0 made NaN are settled (the look for them costs the last call below 1.8 us).
// The accumulator O stays in tensor memory; it is rescaled only where a row's maximum has grown by more than 2^8 over the reference that its exponents are
// taken against (m is that reference, so the result is exact; weights up to 2^8 stay inside fp16).  Rounding: P to the tensors' type, since the MMA takes both
// operands in one 16-bit type and two products of P's halves would double its time; its error is of the size of the result's own rounding.  All else is fp32.
// Warps of rows that do not exist only keep the hand-offs in step.  Every wait is bounded; one that expires sets the error word.
// Bound by the row threads' chain per tile - scores from tensor memory, maximum, 128 exponentials, weights to shared memory: 4.0 thousand clocks where the MMAs of two
// row tiles take 2.0:  8 sequences of 48 drafts, 32 / 8 heads of 128, 1000 to 32768 rows, bf16 157 us (185 back to back, power cap); 1000 tokens behind 2000
// and 7001 rows 195 us, 0.84 PFLOP/s; 333 tokens over 100 to 1500 rows, 8 x 16 heads of 64, fp16 54 us.
#pragma once

#include <type_traits>

#include "cache.cuh"

namespace b200attn {

constexpr int CT_MAX_STAGES = 8;
// A unit's beginning and end (Q, the first tile without another under it, the epilogue), in tiles.  0 / 4 / 6: 8 sequences of 48 drafts, 1000 to 32768 rows,
// 218 / 168 / 167 us; cross attention of 333 tokens to 100 to 1500 rows 87 / 60 / 63; 1000 tokens behind 2000 and 7001 rows 235 / 224 / 227.  With tiles of 64 keys, 2 /
// 4 / 8, head_d 256, 16 / 4 heads: 8 x 48 drafts, 1000 to 16384 rows 102 / 101 / 100 us; 1000 tokens behind 2000 and 7001 rows 205 / 203 / 199; 8 x 333 tokens, 16
// heads, to 100 to 1500 rows 78 / 78 / 79; the drafts at head_d 192 86 / 83 / 83.
constexpr int CT_OH = 4;
constexpr float CT_RESCALE_LOG2 = 8.0f;

struct CtParams {
    CaParams a;
    int tpt, box_t;      // tokens of a row tile; tokens that a Q box has
    int rows8;           // rows of a Q or P buffer: those of a box in whole groups of 8; 128 where a unit has two tiles
    int ng;              // groups of 64 columns
    int nst, nq, np;     // ring stages, Q buffers, P buffers per row tile
};

constexpr int CT_SLOTS = 8;   // units of a CTA's range that its roles can be at: the ring lets the loading thread be four ahead

struct CtSeg {           // a unit, or the part of it that is in this CTA's range
    int b, h, rt, n;     // (n: rows cached)
    int tile, end, ct;   // first and behind the last tile; tiles of cached keys
    int whole;           // the whole unit; -1: no more units
};

struct CtBars {
    uint64_t kv_full[CT_MAX_STAGES], kv_empty[CT_MAX_STAGES], ready[CT_MAX_STAGES];
    uint64_t seg[CT_SLOTS];
    uint64_t q_full[2], q_empty[2];
    // per row tile, alternating from key tile to key tile: a wait by parity tells a phase from the one before it only
    uint64_t s_full[2][2], s_read[2][2];   // scores are there / in registers
    uint64_t p_full[2][2][2];              // each 64 keys of P
    uint64_t o_done[2][2];                 // the MMAs over P have completed
    uint64_t o_empty[2];
};

__device__ __forceinline__ void tma_load_5d(void *smem_dst, const CUtensorMap *tmap, int x, int y, int z, int w, int v, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(
            smem_u32(smem_dst)),
        "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ bool ct_any(bool x) {   // over the 128 threads of warps 4-7 (barrier 1)
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbarrier.cta.red.or.pred p, 1, 128, q;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(any) : "r"((uint32_t)x) : "memory");
    return any != 0;
}
__device__ __forceinline__ void ct_sync() { asm volatile("barrier.cta.sync 1, 128;" ::: "memory"); }

__device__ __forceinline__ void ct_st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Two fp32 operations in one instruction, and the largest of three values.
__device__ __forceinline__ uint64_t ct_pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void ct_unpair(uint64_t x, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ uint64_t ct_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t ct_add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float ct_max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// NaN where one of the three is NaN, else the largest of them.
__device__ __forceinline__ float ct_max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// A pair of 16-bit values with those that are not finite set to 0.
template <bool F16>
__device__ __forceinline__ uint32_t ct_finite(uint32_t w) {
    constexpr uint32_t lo = F16 ? 0x00007c00u : 0x00007f80u, hi = lo << 16;
    if ((w & lo) == lo) w &= 0xffff0000u;
    if ((w & hi) == hi) w &= 0x0000ffffu;
    return w;
}
template <bool F16> struct CtType { using T = __nv_bfloat16; };
template <> struct CtType<true> { using T = __half; };

// Bytes of shared memory in front of the ring: Q buffers, then P buffers.
__host__ __device__ inline size_t ct_front_bytes(int NT, int nq, int np, int ng, int rows8, int TK) { return (size_t)NT * ((size_t)nq * ng + (size_t)np * (TK / 64)) * rows8 * 128; }

// By one warp, on a V tile in shared memory ([groups][rows of 128 B]): rows from `first` on are set to 0 ...
__device__ __forceinline__ void ct_clear_rows(unsigned char *tile, int groups, int rows, int first, int lane) {
    const int per = (rows - first) * 8;   // 16-byte pieces of a group
    for (int g = 0; g < groups; ++g)
        for (int x = lane; x < per; x += 32) *reinterpret_cast<uint4 *>(tile + (size_t)g * rows * 128 + first * 128 + x * 16) = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
}
// ... and values that are not finite among the first `n` rows are set to 0.  True where there were any.  The look at all of them is a multiply-add
// with 0 per pair, whose sum stays 0 unless one is not finite (11 thousand clocks a tile of 128 x 128 became 1 thousand against comparing each).
template <bool F16>
__device__ __forceinline__ bool ct_take_out(unsigned char *tile, int groups, int rows, int n, int lane) {
    using T2 = typename std::conditional<F16, __half2, __nv_bfloat162>::type;
    const int per = n * 8;
    uint32_t zero = 0;
    T2 acc[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] = *reinterpret_cast<T2 *>(&zero);
    const T2 z = acc[0];
    for (int g = 0; g < groups; ++g) {
        const unsigned char *base = tile + (size_t)g * rows * 128;
        for (int x0 = lane; x0 < per; x0 += 256) {
            uint4 a[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) a[k] = x0 + 32 * k < per ? *reinterpret_cast<const uint4 *>(base + (x0 + 32 * k) * 16) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                acc[0] = __hfma2(*reinterpret_cast<T2 *>(&a[k].x), z, acc[0]);
                acc[1] = __hfma2(*reinterpret_cast<T2 *>(&a[k].y), z, acc[1]);
                acc[2] = __hfma2(*reinterpret_cast<T2 *>(&a[k].z), z, acc[2]);
                acc[3] = __hfma2(*reinterpret_cast<T2 *>(&a[k].w), z, acc[3]);
            }
        }
    }
    const T2 sum = __hadd2(__hadd2(acc[0], acc[1]), __hadd2(acc[2], acc[3]));
    const float2 f = F16 ? __half22float2(*reinterpret_cast<const __half2 *>(&sum)) : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&sum));
    if (!__any_sync(0xffffffffu, !(f.x + f.y == 0.0f))) return false;
    for (int g = 0; g < groups; ++g)
        for (int x = lane; x < per; x += 32) {
            uint4 *at = reinterpret_cast<uint4 *>(tile + (size_t)g * rows * 128 + x * 16);
            const uint4 a = *at;
            *at = make_uint4(ct_finite<F16>(a.x), ct_finite<F16>(a.y), ct_finite<F16>(a.z), ct_finite<F16>(a.w));
        }
    fence_proxy_async_smem();
    return true;
}

// By one whole warp, each lane with 128 bytes of a row, `at`: 4 x 4 blocks of 32-byte pieces are transposed among groups of four neighbouring lanes, then lane j of
// a group stores piece j of each of the group's rows.  Only the first `rows` of a group's rows, and `bytes` of the 128, exist.
__device__ __forceinline__ void ct_store_rows(unsigned char *at, uint32_t (&w)[32], int lane, int rows, int bytes) {
    const int j = lane & 3;
#pragma unroll
    for (int M = 2; M >= 1; M >>= 1) {
        const bool up = (j & M) != 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (k & M) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t send = up ? w[8 * k + e] : w[8 * (k | M) + e];
                const uint32_t recv = __shfl_xor_sync(0xffffffffu, send, M);
                if (up) w[8 * k + e] = recv; else w[8 * (k | M) + e] = recv;
            }
        }
    }
#pragma unroll
    for (int m = 0; m < 4; ++m) {   // the row of lane (group + m)
        unsigned char *row = reinterpret_cast<unsigned char *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(at), (lane & ~3) + m));
        if (m < rows && j * 32 < bytes) *reinterpret_cast<uint4 *>(row + j * 32) = make_uint4(w[8 * m], w[8 * m + 1], w[8 * m + 2], w[8 * m + 3]);
        if (m < rows && j * 32 + 16 < bytes) *reinterpret_cast<uint4 *>(row + j * 32 + 16) = make_uint4(w[8 * m + 4], w[8 * m + 5], w[8 * m + 6], w[8 * m + 7]);
    }
}

// By one whole warp: which of up to 32 rows, `row` those of the lanes, hold a value that is not finite.
template <bool F16>
__device__ __forceinline__ unsigned ct_odd_rows(const void *row, bool there, int D) {
    bool odd = false;
    if (there)
        for (int d = 0; d < D; d += 8) {   // (rows are on 16 bytes, head_d is a multiple of 8)
            const uint4 a = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(row) + d);
            odd |= ct_finite<F16>(a.x) != a.x || ct_finite<F16>(a.y) != a.y || ct_finite<F16>(a.z) != a.z || ct_finite<F16>(a.w) != a.w;
        }
    return __ballot_sync(0xffffffffu, odd);
}
// By one whole warp: the kinds of the cached values of rows [j0, j1) in the lane's column d.
template <bool F16>
__device__ unsigned ct_cached_kinds(const CaParams &p, int b, int h, int j0, int j1, int d) {
    using T = typename CtType<F16>::T;
    const int lane = threadIdx.x & 31;
    const T *v = ca_row<T>(p.V, p.v, b, h, 0);
    unsigned kinds = 0;
    for (int j = j0; j < j1; j += 32) {
        if (ct_odd_rows<F16>(v + min(j + lane, j1 - 1) * p.v.l, j + lane < j1, p.D) == 0) continue;
#pragma unroll 8
        for (int k = 0; k < 32; ++k)
            if (j + k < j1 && d < p.D) kinds |= ca_kind(to_f32(v[(j + k) * p.v.l + d]));
        if (__all_sync(0xffffffffu, d >= p.D || kinds > CA_NEG)) break;   // (NaN in every column: more rows change nothing)
    }
    return kinds;
}

// By one whole warp, behind the stores of a unit, or of this CTA's part of it: what values that are not finite leave in the lane's row, token `tok` (-1: no row), which
// is at `o` of the output or `part` of a part.  `settle`: a sum of the row is NaN, and no score was; `fresh`: some of the new tokens' values, taken out of
// the products, are not finite - they are added for the rows that see them.
template <bool F16>
__device__ __noinline__ void ct_odd_values(const CaParams &p, const CtSeg &w, int TK, int tok, bool settle, bool fresh, typename CtType<F16>::T *o, float *part) {
    using T = typename CtType<F16>::T;
    const int lane = threadIdx.x & 31;
    __syncwarp();   // (the warp's lanes have written each other's rows)
    if (__any_sync(0xffffffffu, settle)) {
        for (int c = 0; c < p.D; c += 32) {
            const unsigned kinds = ct_cached_kinds<F16>(p, w.b, w.h, w.tile * TK, min(w.n, min(w.end, w.ct) * TK), c + lane);
            for (int k = 0; k < min(32, p.D - c); ++k) {
                const unsigned of = __shfl_sync(0xffffffffu, kinds, k);
                if (settle && o) ca_settle(o + c + k, of);
                else if (settle) ca_settle(part + c + k, of);
            }
        }
    }
    if (!fresh) return;
    const T *vd = ca_row<T>(p.Vd, p.vd, w.b, w.h, 0);
    const int j1 = min(p.T, (w.end - w.ct) * TK);
    for (int j0 = max(w.tile - w.ct, 0) * TK; j0 < j1; j0 += 32) {
        unsigned odd = ct_odd_rows<F16>(vd + min(j0 + lane, j1 - 1) * p.vd.l, j0 + lane < j1, p.D);
        for (; odd; odd &= odd - 1) {
            const int j = j0 + __ffs(odd) - 1;
            if (tok < 0 || (p.mask ? p.mask[w.b * p.mask_b + (long long)tok * p.T + j] == 0 : j > tok)) continue;
            for (int d = 0; d < p.D; ++d) {
                const float x = to_f32(vd[j * p.vd.l + d]);
                if (fabsf(x) < INFINITY) continue;
                if (o) o[d] = OutCvt<T>::one(to_f32(o[d]) + x);
                else part[d] += x;
            }
        }
    }
}

// A lane whose wait has run out stays with its warp, which has barriers and collective instructions in front of it: it waits no more, computes on what there
// is, in bounds as ever, and the warp leaves together at the unit's end.  (It costs the waits nothing; a vote at each would.)
#define CT_WAIT_AT(site, wait)                                                                          \
    if (!failed && !(wait)) {                                                                           \
        report_kernel_error(p.err, p.err_sys, (unsigned)KERR_MBAR_TIMEOUT | (1u << (16 + (site))));     \
        failed = true;                                                                                  \
    }

constexpr int ct_threads(int NT) { return 128 + NT * 128; }
constexpr int CT_REGS_SMALL = 80, CT_REGS_LARGE = 208;   // NT = 2: 128 * 80 + 256 * 208 <= 384 * 168

// NT: row tiles of 128 lanes per unit; TK: keys of a tile (64 where head_d is above 128, for stages of 32 KB).
// Tensor memory: NT = 1: two score buffers at columns 0 and 128, O at 256; NT = 2: S_t at 128 t, O_t at 256 + 128 t.
template <int NT, int TK, bool F16>
__global__ void __launch_bounds__(ct_threads(NT), 1)
ca_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
             const __grid_constant__ CUtensorMap tmKd, const __grid_constant__ CUtensorMap tmVd, const __grid_constant__ CtParams ct) {
    using T = typename CtType<F16>::T;
    extern __shared__ unsigned char ct_smem_raw[];
    __shared__ CtBars bars;
    __shared__ CaStart s_start;
    __shared__ CtSeg s_seg[CT_SLOTS];
    __shared__ uint32_t tmem_slot;
    __shared__ int s_bad[CT_SLOTS];     // warp 3: [unit of this CTA & 7] = that unit + 1 where its new values were not all finite
    const CaParams &p = ct.a;
    constexpr int NH = TK / 64;
    const uint32_t raw_addr = smem_u32(ct_smem_raw);
    unsigned char *smem = ct_smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ng = ct.ng, nst = ct.nst, nq = ct.nq;
    const uint32_t slab = (uint32_t)ct.rows8 * 128u;        // 64 columns of a Q buffer, 64 keys of a P tile
    const uint32_t stage = (uint32_t)ng * TK * 128u;        // a K or V tile: [ng groups][TK keys][128 B]
    unsigned char *q_smem = smem;                           // [nq][NT][ng] slabs
    unsigned char *p_smem = q_smem + (size_t)nq * NT * ng * slab;   // [NT][np][NH] slabs
    // an MMA reads 128 rows from a slab's beginning on: behind the box's rows that is whatever follows, and only rows that nobody looks at depend on it
    unsigned char *ring = p_smem + (size_t)NT * ct.np * NH * slab;
    const uint32_t lim = p.spin_limit;

    if (threadIdx.x == 0) {
        for (int i = 0; i < CT_MAX_STAGES; ++i) { mbar_init(&bars.kv_full[i], 1 + p.wait_extra); mbar_init(&bars.kv_empty[i], NT + 1); mbar_init(&bars.ready[i], 1); }
        for (int i = 0; i < CT_SLOTS; ++i) { mbar_init(&bars.seg[i], 1); s_bad[i] = 0; }
        for (int i = 0; i < 2; ++i) { mbar_init(&bars.q_full[i], 1); mbar_init(&bars.q_empty[i], NT); }
        for (int t = 0; t < 2; ++t) {
            for (int b = 0; b < 2; ++b) {
                mbar_init(&bars.s_full[t][b], 1); mbar_init(&bars.s_read[t][b], 4); mbar_init(&bars.o_done[t][b], 1);
                for (int h = 0; h < 2; ++h) mbar_init(&bars.p_full[t][b][h], 4);
            }
            mbar_init(&bars.o_empty[t], 4);
        }
        mbar_fence_init();
        tma_prefetch_desc(&tmQ); tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV);
        if (p.drafts) { tma_prefetch_desc(&tmKd); tma_prefetch_desc(&tmVd); }
    }
    if (warp == 1) tmem_alloc(&tmem_slot, 512);
    grid_dependency_wait();
    if (warp == 2) {
        const CaStart s = ca_locate(p, blockIdx.x);
        if (lane == 0) s_start = s;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    grid_launch_dependents();   // (not before the allocation: a dependent on this SM could take the columns and wait for this CTA to end)
    const uint32_t tmem = tmem_slot;
    bool failed = false;

    if (warp < 4) {
        if (NT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(CT_REGS_SMALL));
        if (warp == 0) {
            if (elect_one()) {
                CaWalk w;
                w.start(p, s_start, blockIdx.x);
                ca_entry_of_cta(p, s_start, w, blockIdx.x);
                int s = 0;
                uint32_t ph = 0;
                bool ok = true;
                auto load = [&](bool v, int i) {   // tile i of the unit
                    ok = ok && mbar_wait(&bars.kv_empty[s], ph ^ 1u, lim);
                    if (!ok) return;
                    mbar_expect_tx(&bars.kv_full[s], stage);
                    const bool draft = i >= w.ct;
                    const CUtensorMap *tm = draft ? (v ? &tmVd : &tmKd) : (v ? &tmV : &tmK);
                    const int row = (draft ? i - w.ct : i) * TK;
                    for (int g = 0; g < ng; ++g) tma_load_4d(ring + (size_t)s * stage + (size_t)g * (TK * 128), tm, g * 64, row, w.h, w.b, &bars.kv_full[s]);
                    if (++s == nst) { s = 0; ph ^= 1u; }
                };
                int seg = 0;
                for (; w.left > 0 && ok; ++seg, w.next(p)) {
                    const int first = w.tile(p), end = w.end(p);
                    // (the slot's last unit is eight back: the ring has been handed back since by everybody who read it)
                    s_seg[seg & (CT_SLOTS - 1)] = CtSeg{w.b, w.h, w.rt, w.n, first, end, w.ct, w.whole(p) ? 1 : 0};
                    mbar_arrive(&bars.seg[seg & (CT_SLOTS - 1)]);
                    ca_entry_of_unit(p, s_start, w, blockIdx.x, seg == 0);
                    const int qi = nq == 2 ? seg & 1 : 0;
                    ok = mbar_wait(&bars.q_empty[qi], (uint32_t)((nq == 2 ? seg >> 1 : seg) & 1) ^ 1u, lim);
                    if (!ok) break;
                    const int tok0 = w.rt * NT * ct.tpt, nt = NT == 2 && tok0 + ct.tpt < p.T ? 2 : 1;
                    mbar_expect_tx(&bars.q_full[qi], (uint32_t)(nt * ng * p.G * ct.box_t) * 128u);
                    for (int t = 0; t < nt; ++t)
                        for (int g = 0; g < ng; ++g)
                            tma_load_5d(q_smem + (size_t)((qi * NT + t) * ng + g) * slab, &tmQ, g * 64, 0, tok0 + t * ct.tpt, w.h, w.b, &bars.q_full[qi]);
                    load(false, first);
                    for (int i = first; i < end && ok; ++i) {
                        if (i + 1 < end) load(false, i + 1);
                        load(true, i);
                    }
                }
                if (ok) {
                    s_seg[seg & (CT_SLOTS - 1)].whole = -1;
                    mbar_arrive(&bars.seg[seg & (CT_SLOTS - 1)]);
                } else {
                    report_kernel_error(p.err, p.err_sys, (unsigned)KERR_MBAR_TIMEOUT | (1u << 16));
                    failed = true;
                    ca_entries_left(p, s_start, w, blockIdx.x, seg);
                }
            }
        } else if (warp == 3) {
            // ---- every V tile before the MMAs see it ----
            int s = 0;
            uint32_t ph = 0;
            bool ok = true;
            auto pass = [&](bool v, int i, int seg, int n, int nct) {
                ok = ok && mbar_wait(&bars.kv_full[s], ph, lim);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) return;
                const bool draft = i >= nct;
                unsigned char *tile = ring + (size_t)s * stage;
                if (v && !draft && n - i * TK < TK) ct_clear_rows(tile, ng, TK, max(n - i * TK, 0), lane);
                if (v && draft && ct_take_out<F16>(tile, ng, TK, min(TK, p.T - (i - nct) * TK), lane) && lane == 0) s_bad[seg & (CT_SLOTS - 1)] = seg + 1;
                __syncwarp();
                if (lane == 0) { mbar_arrive(&bars.ready[s]); mbar_arrive(&bars.kv_empty[s]); }
                if (++s == nst) { s = 0; ph ^= 1u; }
            };
            for (int seg = 0; ok; ++seg) {
                ok = mbar_wait(&bars.seg[seg & (CT_SLOTS - 1)], (uint32_t)(seg / CT_SLOTS) & 1u, lim);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const CtSeg w = s_seg[seg & (CT_SLOTS - 1)];
                if (w.whole < 0) break;
                pass(false, w.tile, seg, w.n, w.ct);
                for (int i = w.tile; i < w.end && ok; ++i) {
                    if (i + 1 < w.end) pass(false, i + 1, seg, w.n, w.ct);
                    pass(true, i, seg, w.n, w.ct);
                }
            }
            if (!ok) { report_kernel_error(p.err, p.err_sys, (unsigned)KERR_MBAR_TIMEOUT | (1u << 17)); failed = true; }
        } else if (warp <= NT) {
            if (elect_one()) {
                const int t = warp - 1;
                const int ks = (p.D + 15) >> 4;   // MMA steps of a score
                const uint32_t id_qk = umma_idesc_16(128, TK, 0, 0, F16 ? 1 : 0), id_pv = umma_idesc_16(128, ks << 4, 0, 1, F16 ? 1 : 0);
                const uint32_t pa = smem_u32(p_smem + (size_t)t * ct.np * NH * slab);
                const uint32_t t_o = tmem + 256 + (NT == 2 ? t * 128 : 0);
                int s = 0;
                uint32_t ph = 0, gq = 0, gp = 0;   // key tiles so far: scores, products with V
                int lu = 0;                        // units
                bool ok = true;
                uint32_t qa = 0;
                int qi = 0;
                auto qk = [&](bool last) {
                    ok = ok && mbar_wait(&bars.kv_full[s], ph, lim);
                    const uint32_t back = gq - (NT == 1 ? 2 : 1);   // the tile whose scores were where these go
                    if (ok && gq >= (NT == 1 ? 2u : 1u)) ok = mbar_wait(&bars.s_read[t][back & 1], (back >> 1) & 1u, lim);
                    if (!ok) return;
                    tc_fence_after();
                    const uint32_t ka = smem_u32(ring + (size_t)s * stage), t_s = tmem + (NT == 1 ? (gq & 1) : t) * 128;
                    for (int g = 0; g < ng; ++g) {
                        const uint64_t dq = umma_desc_k_sw128(qa + g * slab), dk = umma_desc_k_sw128(ka + g * (TK * 128));
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (4 * g + k < ks) umma_bf16(t_s, dq + 2 * k, dk + 2 * k, id_qk, (g | k) != 0);
                    }
                    umma_commit(&bars.s_full[t][gq & 1]);
                    umma_commit(&bars.kv_empty[s]);
                    if (last) umma_commit(&bars.q_empty[qi]);
                    ++gq;
                    if (++s == nst) { s = 0; ph ^= 1u; }
                };
                for (int seg = 0; ok; ++seg) {
                    ok = mbar_wait(&bars.seg[seg & (CT_SLOTS - 1)], (uint32_t)(seg / CT_SLOTS) & 1u, lim);
                    if (!ok) break;
                    const CtSeg &w = s_seg[seg & (CT_SLOTS - 1)];
                    if (w.whole < 0) break;
                    const int first = w.tile, end = w.end;
                    qi = nq == 2 ? seg & 1 : 0;
                    ok = mbar_wait(&bars.q_full[qi], (uint32_t)((nq == 2 ? seg >> 1 : seg) & 1), lim);
                    if (!ok) break;
                    tc_fence_after();
                    if (NT == 2 && (w.rt * NT + t) * ct.tpt >= p.T) {
                        // no rows: the ring and the Q buffer are handed back in step with the other issuer, and the row threads are kept in step by a
                        // tile's hand-offs without a tile
                        mbar_arrive(&bars.q_empty[qi]);
                        ok = mbar_wait(&bars.o_empty[t], (uint32_t)(lu & 1) ^ 1u, lim);
                        if (ok && gq > 0) ok = mbar_wait(&bars.s_read[t][(gq - 1) & 1], ((gq - 1) >> 1) & 1u, lim);
                        if (!ok) break;
                        mbar_arrive(&bars.s_full[t][gq & 1]);
                        for (int h = 0; h < NH; ++h) ok = ok && mbar_wait(&bars.p_full[t][gp & 1][h], (gp >> 1) & 1u, lim);
                        if (!ok) break;
                        mbar_arrive(&bars.o_done[t][gp & 1]);
                        ++gq; ++gp; ++lu;
                        for (int i = 0; i < 2 * (end - first) && ok; ++i) {
                            ok = mbar_wait(&bars.kv_full[s], ph, lim);
                            if (!ok) break;
                            mbar_arrive(&bars.kv_empty[s]);
                            if (++s == nst) { s = 0; ph ^= 1u; }
                        }
                        continue;
                    }
                    qa = smem_u32(q_smem + (size_t)(qi * NT + t) * ng * slab);
                    qk(first + 1 == end);
                    for (int i = first; i < end && ok; ++i, ++gp) {
                        if (i + 1 < end) qk(i + 2 == end);
                        ok = ok && mbar_wait(&bars.ready[s], ph, lim);   // V_i
                        if (ok && i == first) ok = mbar_wait(&bars.o_empty[t], (uint32_t)(lu & 1) ^ 1u, lim);
                        const uint32_t va = smem_u32(ring + (size_t)s * stage), pb = pa + (ct.np == 2 ? (gp & 1) * NH * slab : 0u);
#pragma unroll
                        for (int h = 0; h < NH; ++h) {
                            ok = ok && mbar_wait(&bars.p_full[t][gp & 1][h], (gp >> 1) & 1u, lim);
                            if (!ok) break;
                            tc_fence_after();
                            const uint64_t dp = umma_desc_k_sw128(pb + h * slab);
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                umma_bf16(t_o, dp + 2 * k, umma_desc_mn_sw128(va + (4 * h + k) * 2048, TK * 128), id_pv, (i > first || h != 0 || k != 0) ? 1u : 0u);
                        }
                        if (!ok) break;
                        umma_commit(&bars.o_done[t][gp & 1]);
                        umma_commit(&bars.kv_empty[s]);
                        if (++s == nst) { s = 0; ph ^= 1u; }
                    }
                    ++lu;
                }
                if (!ok) { report_kernel_error(p.err, p.err_sys, (unsigned)KERR_MBAR_TIMEOUT | (1u << 18)); failed = true; }
            }
        }
    } else {
        if (NT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(CT_REGS_LARGE));
        // ---- softmax and epilogue of row tile t; thread = row (tensor-memory lane) ----
        const int t = (warp - 4) >> 2, q = warp & 3, row = 32 * q + lane;
        const uint32_t tl = tmem + ((uint32_t)(32 * q) << 16);
        const uint32_t to = tl + 256u + (NT == 2 ? t * 128u : 0u);
        const uint32_t prow = smem_u32(p_smem + (size_t)t * ct.np * NH * slab) + (uint32_t)row * 128u, sw = (uint32_t)(row & 7);
        const float sl2 = p.scale_log2;
        uint32_t g = 0;   // key tiles so far
        uint32_t r[TK / 32][32];
        auto pv_done = [&](uint32_t x) { return mbar_wait(&bars.o_done[t][x & 1], (x >> 1) & 1u, lim); };
        for (int seg = 0;; ++seg) {
            CT_WAIT_AT(7, mbar_wait(&bars.seg[seg & (CT_SLOTS - 1)], (uint32_t)(seg / CT_SLOTS) & 1u, lim));
            if (__any_sync(0xffffffffu, failed)) { failed = true; break; }
            const CtSeg &w = s_seg[seg & (CT_SLOTS - 1)];
            if (w.whole < 0) break;
            const int tok0 = (w.rt * NT + t) * ct.tpt, rows = min(ct.tpt, p.T - tok0) * p.G;
            if (NT == 2 && rows <= 0) {   // a tile's hand-offs (above)
                CT_WAIT_AT(3, mbar_wait(&bars.s_full[t][g & 1], (g >> 1) & 1u, lim));
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&bars.s_read[t][g & 1]);
                    for (int h = 0; h < NH; ++h) mbar_arrive(&bars.p_full[t][g & 1][h]);
                }
                CT_WAIT_AT(6, pv_done(g));
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.o_empty[t]);
                ++g;
                continue;
            }
            const bool act = 32 * q < rows;       // the same for a warp
            const bool mine = row < rows;
            const int tok = min(tok0 + row / p.G, p.T - 1);
            float x_ref = -INFINITY, l = 0.0f;   // the reference is x_ref sl2
            const int first = w.tile, end = w.end, nct = w.ct;
            for (int i = first; i < end; ++i, ++g) {
                const bool draft = i >= nct;
                const int j0 = (draft ? i - nct : i) * TK;
                const bool part = draft || i + 1 == nct;   // (the same for every thread) keys that may not be there, or not be seen
                if (!act) {   // a warp without rows keeps the hand-offs in step
                    CT_WAIT_AT(3, mbar_wait(&bars.s_full[t][g & 1], (g >> 1) & 1u, lim));
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars.s_read[t][g & 1]);
                    if (g >= (uint32_t)ct.np) CT_WAIT_AT(5, pv_done(g - ct.np));
                    __syncwarp();
                    if (lane == 0)
                        for (int h = 0; h < NH; ++h) mbar_arrive(&bars.p_full[t][g & 1][h]);
                    continue;
                }
                uint32_t see[TK / 32];
                if (part) {
                    const int valid = !draft ? w.n - j0 : p.mask ? 0 : tok - j0 + 1;
#pragma unroll
                    for (int x = 0; x < TK / 32; ++x) see[x] = valid >= 32 * (x + 1) ? 0xffffffffu : valid <= 32 * x ? 0u : (1u << (valid - 32 * x)) - 1u;
                    if (draft && p.mask && mine) {
                        const unsigned char *mrow = p.mask + w.b * p.mask_b + (long long)tok * p.T + j0;
                        const int n = min(TK, p.T - j0);
#pragma unroll
                        for (int x = 0; x < TK / 32; ++x) {
                            uint32_t bits = 0;
#pragma unroll 8
                            for (int k = 0; k < 32; ++k)
                                if (32 * x + k < n) bits |= (__ldg(mrow + 32 * x + k) != 0 ? 1u : 0u) << k;
                            see[x] = bits;
                        }
                    }
                }
                CT_WAIT_AT(3, mbar_wait(&bars.s_full[t][g & 1], (g >> 1) & 1u, lim));
                tc_fence_after();
                const uint32_t ts = tl + (NT == 1 ? (g & 1) : t) * 128u;
#pragma unroll
                for (int x = 0; x < TK / 32; ++x) tmem_ld32(ts + 32 * x, r[x]);
                tmem_ld_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.s_read[t][g & 1]);   // these scores may be overwritten
                if (part) {
#pragma unroll
                    for (int x = 0; x < TK / 32; ++x)
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (!(see[x] >> k & 1u)) r[x][k] = 0xff800000u;
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int k = 0; k < 32; k += 4)
#pragma unroll
                    for (int x = 0; x < TK / 32; ++x) {
                        float &a = mx[2 * (x & 1)], &b = mx[2 * (x & 1) + 1];
                        a = ct_max3(a, __uint_as_float(r[x][k]), __uint_as_float(r[x][k + 1]));
                        b = ct_max3(b, __uint_as_float(r[x][k + 2]), __uint_as_float(r[x][k + 3]));
                    }
                const float topx = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                bool taken = false;   // the scores are differences from x_ref already
                const bool need = i > first && mine && topx * sl2 > x_ref * sl2 + CT_RESCALE_LOG2;
                if (i == first) x_ref = topx;
                if (__any_sync(0xffffffffu, need || (mine && ca_large(x_ref * sl2)))) {
                    if (__any_sync(0xffffffffu, need)) {
                        CT_WAIT_AT(4, pv_done(g - 1));
                        tc_fence_after();
                        const float f = need ? fast_exp2(x_ref * sl2 - topx * sl2) : 1.0f;   // (0 where the row had seen nothing)
                        uint32_t o[16];
                        for (int c = 0; c < p.D; c += 16) {
                            tmem_ld16(to + c, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                            tmem_st16(to + c, o);
                        }
                        tmem_st_wait();
                        l *= f;
                        if (need) x_ref = topx;
                    }
                    if (__any_sync(0xffffffffu, mine && ca_large(x_ref * sl2))) {   // differences first, then the scale
                        const float x0 = x_ref == -INFINITY ? 0.0f : x_ref;
#pragma unroll
                        for (int x = 0; x < TK / 32; ++x)
#pragma unroll
                            for (int k = 0; k < 32; ++k) r[x][k] = __float_as_uint(__uint_as_float(r[x][k]) - x0);
                        taken = true;
                    }
                }
                const float neg = taken || x_ref == -INFINITY ? 0.0f : -x_ref * sl2;   // a row that has seen nothing: every score is -inf
                if (g >= (uint32_t)ct.np) CT_WAIT_AT(5, pv_done(g - ct.np));   // the MMAs have read what was in this P buffer
                const uint32_t pw = prow + (ct.np == 2 ? (g & 1) * NH * slab : 0u);
                const uint64_t sl2_2 = ct_pair(sl2, sl2), neg_2 = ct_pair(neg, neg);
                uint64_t sum = 0;   // a pair of sums
#pragma unroll
                for (int h = 0; h < NH; ++h) {
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        uint32_t pk[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int e = 8 * (c & 3) + 2 * k;
                            const uint32_t (&rr)[32] = r[2 * h + (c >> 2)];
                            float e0, e1;
                            ct_unpair(ct_fma2(ct_pair(__uint_as_float(rr[e]), __uint_as_float(rr[e + 1])), sl2_2, neg_2), e0, e1);
                            e0 = fast_exp2(e0); e1 = fast_exp2(e1);
                            sum = ct_add2(sum, ct_pair(e0, e1));
                            pk[k] = pack_16x2(e0, e1, F16);
                        }
                        if (NT == 2 || row < ct.rows8) ct_st_shared_v4(pw + h * slab + ((((uint32_t)c) ^ sw) << 4), pk[0], pk[1], pk[2], pk[3]);
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars.p_full[t][g & 1][h]);
                }
                float sum0, sum1;
                ct_unpair(sum, sum0, sum1);
                l += sum0 + sum1;
            }
            // ---- epilogue of the unit ----
            CT_WAIT_AT(6, pv_done(g - 1));
            tc_fence_after();
            if (act) {
                const bool whole = w.whole != 0, bad = s_bad[seg & (CT_SLOTS - 1)] == seg + 1;
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                const int hq = w.h * p.G + row % p.G;
                float *prt = p.part + ((size_t)blockIdx.x * 2 + (seg == 0 ? 0 : 1)) * ca_slot_floats(p.RT, p.D);
                const int urow = t * ct.tpt * p.G + row;   // row of the unit
                T *o = ca_row<T>(p.O, p.o, w.b, hq, tok);
                // 32 columns of a row: as fp32, 128 bytes of a part; two of them, as 16-bit values, 128 bytes of the output.  Lanes trade pieces so that a
                // store covers whole lines of eight rows, not 16 bytes of 32 (7 us a unit of 128 columns).
                uint32_t v[32];
                float nan[2] = {0.0f, 0.0f};   // NaN where a sum is (what lies behind head_d may be anything)
                auto columns = [&](int c) {   // c to c + 31 of the accumulator
                    tmem_ld32(to + c, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int k = 0; k < 32; k += 4)
#pragma unroll
                        for (int x = 0; x < 2; ++x) nan[x] = ct_max3_nan(nan[x], __uint_as_float(v[k + 2 * x]), __uint_as_float(v[k + 2 * x + 1]));
                };
                if (whole) {
                    uint32_t out[32];
                    for (int c = 0; c < p.D; c += 64) {
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            columns(c + 32 * x);
#pragma unroll
                            for (int k = 0; k < 16; ++k) out[16 * x + k] = pack_16x2(__uint_as_float(v[2 * k]) * inv, __uint_as_float(v[2 * k + 1]) * inv, F16);
                        }
                        ct_store_rows(reinterpret_cast<unsigned char *>(o + c), out, lane, rows - (row & ~3), (p.D - c) * 2);
                    }
                } else {
                    for (int c = 0; c < p.D; c += 32) {
                        columns(c);
                        ct_store_rows(reinterpret_cast<unsigned char *>(prt + (size_t)urow * p.D + c), v, lane, rows - (row & ~3), (p.D - c) * 4);
                    }
                }
                const bool settle = mine && l == l && (nan[0] != nan[0] || nan[1] != nan[1]);
                if (bad || __any_sync(0xffffffffu, settle))
                    ct_odd_values<F16>(p, w, TK, mine ? tok : -1, settle, bad, whole ? o : nullptr, whole ? nullptr : prt + (size_t)urow * p.D);
                if (mine) {
                    const float m_ref = x_ref * sl2;
                    if (!whole) {
                        prt[(size_t)p.RT * p.D + 2 * urow] = m_ref;
                        prt[(size_t)p.RT * p.D + 2 * urow + 1] = l;
                    } else if (p.lse) {
                        p.lse[((long long)w.b * p.Hq + hq) * p.T + tok] = l == 0.0f ? -INFINITY : (m_ref + log2f(l)) * 0.69314718055994531f;
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.o_empty[t]);
        }
    }

    if (failed) for (int i = 0; i < 2000; ++i) __nanosleep(1000);   // let copies and MMAs in flight drain
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, 512);
}
#undef CT_WAIT_AT

// ---- host: tensor maps ----------------------------------------------------------------------------------------------------
// [B, heads, rows, D] as {D, rows, heads, B}, boxes of 64 columns x `box_rows`; what lies outside reads as 0.  A dimension of size 1 has no stride to speak of.
inline bool ct_map_rows(CUtensorMap *m, const void *base, const CaView &v, int B, int H, long long L, int D, int box_rows) {
    PFN_tmapEncodeTiled enc = tmap_encode_fn();
    if (!enc) return false;
    cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)L, (cuuint64_t)H, (cuuint64_t)B};
    cuuint64_t st[3] = {(cuuint64_t)(L == 1 ? 512 : v.l * 2), (cuuint64_t)(H == 1 ? 512 : v.h * 2), (cuuint64_t)(B == 1 ? 512 : v.b * 2)};
    cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1}, es[4] = {1, 1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(base), dims, st, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Q [B, Hkv * G, T, D] as {D, G, T, Hkv, B}: a box of G x box_t rows is a row tile, row t G + g.
inline bool ct_map_q(CUtensorMap *m, const void *base, const CaView &v, int B, int Hkv, int G, int T, int D, int box_t) {
    PFN_tmapEncodeTiled enc = tmap_encode_fn();
    if (!enc) return false;
    cuuint64_t dims[5] = {(cuuint64_t)D, (cuuint64_t)G, (cuuint64_t)T, (cuuint64_t)Hkv, (cuuint64_t)B};
    cuuint64_t st[4] = {(cuuint64_t)(G == 1 ? 512 : v.h * 2), (cuuint64_t)(T == 1 ? 512 : v.l * 2), (cuuint64_t)(Hkv == 1 ? 512 : v.h * G * 2),
                        (cuuint64_t)(B == 1 ? 512 : v.b * 2)};
    cuuint32_t box[5] = {64, (cuuint32_t)G, (cuuint32_t)box_t, 1, 1}, es[5] = {1, 1, 1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void *>(base), dims, st, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace b200attn
