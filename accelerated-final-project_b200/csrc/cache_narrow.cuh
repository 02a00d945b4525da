// Attention of new tokens over a cache where a key head has few rows (tokens times query heads of the group: up to 64): one token, small trees.
// The call is bound by reading K and V once, so everything else has to be small: here the KEYS are the lanes of tensor memory,
//     S^T [128 keys x N rows] = K Q^T,      O^T [head_d x N rows] += V^T P^T,      N = 16, 32 or 64,
// so that the MMAs compute the rows that there are (with the rows as lanes, cache_tc.cuh, four rows cost what 128 do: 1.9 thousand clocks a tile for the
// exponentials of one warp, and so much power in the MMAs that the card lowered its clock), and the four softmax warps share a tile's exponentials.
//   warp 0       one thread requests pieces of 128 keys x 128 columns by TMA in the order K_0 | K_1 V_0 | K_2 V_1 | ...
//   warp 1       one thread issues the MMAs
//   warp 3       V pieces before the MMAs see them, as in cache_tc.cuh
//   warps 4-7    a thread per key: exp2 of its scores against a reference per row, P^T rows to shared memory, sums of its own keys; at a unit's end a
//                thread per output column.
// A row's reference only has to be within 2^8 of its maximum (the exponents stay exact in fp32, weights below 2^8 in fp16): per tile the threads
// only vote whether some score is beyond that - one barrier - and reduce maxima, set new references and rescale where it is, which is at a
// unit's first tile and hardly ever again.  Roundings as in cache_tc.cuh.
//   64 sequences, one token, 32 / 8 heads of 128, 0 to 8192 rows cached, bf16 (1.07 GB): 180 us, 6.0 TB/s, 0.91 of the copy rate; rows as lanes 250 us (1.63 GHz
//   under the power cap).  SMs get rates that differ by 12 % either way, and shares are equal.
#pragma once

#include "cache_tc.cuh"

namespace b200attn {

struct CnParams {
    CaParams a;
    int ng, nh, gp;      // groups of 64 columns; pieces of a tile: 128 columns each; groups of a stage
    int nst;             // ring stages
    int tmem_cols;
};
constexpr int CN_THREADS = 256, CN_TK = 128;
// Tiles that a cache's capacity and the new tokens may have for its units not to be cut, so that nothing is joined by a second launch: more where the units fill the
// SMs by themselves.  Cut / not, one token, 32 / 8 heads of 128: one sequence of 2, 4, 7 tiles 10.5 / 9.8, 10.6 / 11.8, 10.8 / 14.8 us (and 4 us of the host's time
// less); 16 sequences of 4, 9, 16 tiles 17 / 13, 22 / 18, 32 / 29; 64 of 4, 7, 9, 12 tiles 45 / 39, 53 / 52, 60 / 61, 72 / 76.  The second line is where many units
// an SM break even; 16 sequences, a unit an SM, would gain beyond it.  It goes by the capacity, as the lengths are not known on the host.
constexpr int CN_UNCUT_FEW = 4, CN_UNCUT_MANY = 8;
constexpr int CN_OH = 1;   // a unit's beginning and end, in tiles (0 / 1 / 3: 184.4 / 182.9 / 186.4 us for the call above)
constexpr uint32_t CN_GROUP = CN_TK * 128u;   // 128 keys x 64 columns

struct CnBars {
    uint64_t kv_full[CT_MAX_STAGES], kv_empty[CT_MAX_STAGES], ready[CT_MAX_STAGES];
    uint64_t seg[CT_SLOTS];
    uint64_t q_full[2], q_empty[2];
    uint64_t s_full[2], s_read[2], p_full[2], o_done[2];   // alternating from tile to tile
    uint64_t o_empty[2];                                   // alternating from unit to unit
};

__host__ __device__ inline size_t cn_front_bytes(int N, int ng) { return (size_t)2 * N * 128 * (ng + 2); }   // two Q buffers, two P buffers

__device__ __forceinline__ float cn_warp_max(float x) {
    float m;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(x));
    return m;
}
__device__ __forceinline__ void ct_st_shared_u16(uint32_t addr, uint16_t x) { asm volatile("st.shared.u16 [%0], %1;" ::"r"(addr), "h"(x) : "memory"); }

constexpr float CN_UNSET = 3.402823466e38f;   // minus the reference of a row that has seen nothing: any finite score is beyond it

#define CN_FAIL_AT(site, cond)                                                                          \
    if (cond) {                                                                                         \
        report_kernel_error(p.err, p.err_sys, (unsigned)KERR_MBAR_TIMEOUT | (1u << (16 + (site))));     \
        failed = true;                                                                                  \
    }

template <int N, bool F16>
__global__ void __launch_bounds__(CN_THREADS, 1)
ca_narrow_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                 const __grid_constant__ CUtensorMap tmKd, const __grid_constant__ CUtensorMap tmVd, const __grid_constant__ CnParams cn) {
    using T = typename CtType<F16>::T;
    extern __shared__ unsigned char ct_smem_raw[];
    __shared__ CnBars bars;
    __shared__ CaStart s_start;
    __shared__ CtSeg s_seg[CT_SLOTS];
    __shared__ uint32_t tmem_slot;
    __shared__ int s_bad[CT_SLOTS];
    __shared__ __align__(16) float s_neg[N], s_f[N], s_inv[N], s_red[4][N];   // minus the reference (log2 units), factor of a change, 1 / l, per-warp values
    __shared__ __align__(16) float s_x[N], s_zero[N];   // the reference before its scaling, 0 where there is none; zeros
    __shared__ int s_large;                             // some reference is large (ca_large)
    const CaParams &p = cn.a;
    const uint32_t raw_addr = smem_u32(ct_smem_raw);
    unsigned char *smem = ct_smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ng = cn.ng, nh = cn.nh, nst = cn.nst;
    constexpr uint32_t slab = N * 128u;
    const uint32_t stage = (uint32_t)cn.gp * CN_GROUP;
    unsigned char *q_smem = smem;                        // [2][ng] slabs of N rows x 64 columns
    unsigned char *p_smem = q_smem + (size_t)2 * ng * slab;   // [2][2] slabs of N rows x 64 keys
    unsigned char *ring = p_smem + 4 * slab;
    const uint32_t lim = p.spin_limit;

    if (threadIdx.x == 0) {
        for (int i = 0; i < CT_MAX_STAGES; ++i) { mbar_init(&bars.kv_full[i], 1 + p.wait_extra); mbar_init(&bars.kv_empty[i], 2); mbar_init(&bars.ready[i], 1); }
        for (int i = 0; i < CT_SLOTS; ++i) { mbar_init(&bars.seg[i], 1); s_bad[i] = 0; }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars.q_full[i], 1); mbar_init(&bars.q_empty[i], 1);
            mbar_init(&bars.s_full[i], 1); mbar_init(&bars.s_read[i], 4); mbar_init(&bars.p_full[i], 4); mbar_init(&bars.o_done[i], 1); mbar_init(&bars.o_empty[i], 4);
        }
        mbar_fence_init();
        tma_prefetch_desc(&tmQ); tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV);
        if (p.drafts) { tma_prefetch_desc(&tmKd); tma_prefetch_desc(&tmVd); }
    }
    if (threadIdx.x < N) { s_neg[threadIdx.x] = CN_UNSET; s_x[threadIdx.x] = s_zero[threadIdx.x] = 0.0f; }
    if (threadIdx.x == 0) s_large = 0;
    if (warp == 1) tmem_alloc(&tmem_slot, (uint32_t)cn.tmem_cols);
    grid_dependency_wait();
    if (warp == 2) {
        const CaStart s = ca_locate(p, blockIdx.x);
        if (lane == 0) s_start = s;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    grid_launch_dependents();   // (not before the allocation: a dependent on this SM could take the columns and wait for this CTA to end)
    const uint32_t tmem = tmem_slot;        // S^T buffers at columns 0 and N; O^T of unit parity u, piece c at 2 N + (u nh + c) N
    bool failed = false;

    if (warp == 0) {
        if (elect_one()) {
            CaWalk w;
            w.start(p, s_start, blockIdx.x);
            ca_entry_of_cta(p, s_start, w, blockIdx.x);
            int s = 0;
            uint32_t ph = 0;
            bool ok = true;
            auto load = [&](bool v, int i) {   // tile i of the unit
                const bool draft = i >= w.ct;
                const CUtensorMap *tm = draft ? (v ? &tmVd : &tmKd) : (v ? &tmV : &tmK);
                const int row = (draft ? i - w.ct : i) * CN_TK;
                for (int c = 0; c < nh; ++c) {
                    ok = ok && mbar_wait(&bars.kv_empty[s], ph ^ 1u, lim);
                    if (!ok) return;
                    const int n = min(2, ng - 2 * c);
                    mbar_expect_tx(&bars.kv_full[s], (uint32_t)n * CN_GROUP);
                    for (int g = 0; g < n; ++g) tma_load_4d(ring + (size_t)s * stage + (size_t)g * CN_GROUP, tm, (2 * c + g) * 64, row, w.h, w.b, &bars.kv_full[s]);
                    if (++s == nst) { s = 0; ph ^= 1u; }
                }
            };
            int seg = 0;
            for (; w.left > 0 && ok; ++seg, w.next(p)) {
                const int first = w.tile(p), end = w.end(p), qi = seg & 1;
                s_seg[seg & (CT_SLOTS - 1)] = CtSeg{w.b, w.h, w.rt, w.n, first, end, w.ct, w.whole(p) ? 1 : 0};
                mbar_arrive(&bars.seg[seg & (CT_SLOTS - 1)]);
                ca_entry_of_unit(p, s_start, w, blockIdx.x, seg == 0);
                ok = mbar_wait(&bars.q_empty[qi], (uint32_t)(seg >> 1 & 1) ^ 1u, lim);
                if (!ok) break;
                mbar_expect_tx(&bars.q_full[qi], (uint32_t)(ng * p.R) * 128u);
                for (int g = 0; g < ng; ++g) tma_load_5d(q_smem + (size_t)(qi * ng + g) * slab, &tmQ, g * 64, 0, 0, w.h, w.b, &bars.q_full[qi]);
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
                CN_FAIL_AT(0, true)
                ca_entries_left(p, s_start, w, blockIdx.x, seg);
            }
        }
    } else if (warp == 3) {
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        auto pass = [&](bool v, int i, int seg, int n, int nct) {
            for (int c = 0; c < nh; ++c) {
                ok = ok && mbar_wait(&bars.kv_full[s], ph, lim);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) return;
                if (v) {
                    const bool draft = i >= nct;
                    const int valid = draft ? p.T - (i - nct) * CN_TK : n - i * CN_TK;
                    if (!draft && valid < CN_TK) ct_clear_rows(ring + (size_t)s * stage, min(2, ng - 2 * c), CN_TK, max(valid, 0), lane);
                    if (draft && ct_take_out<F16>(ring + (size_t)s * stage, min(2, ng - 2 * c), CN_TK, min(valid, CN_TK), lane) && lane == 0) s_bad[seg & (CT_SLOTS - 1)] = seg + 1;
                }
                __syncwarp();
                if (lane == 0) { mbar_arrive(&bars.ready[s]); mbar_arrive(&bars.kv_empty[s]); }
                if (++s == nst) { s = 0; ph ^= 1u; }
            }
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
        if (!ok) CN_FAIL_AT(1, true)
    } else if (warp == 1) {
        if (elect_one()) {
            const int ks = (p.D + 15) >> 4;   // MMA steps of a score
            const uint32_t id_s = umma_idesc_16(128, N, 0, 0, F16 ? 1 : 0), id_o = umma_idesc_16(p.D <= 64 ? 64 : 128, N, 1, 0, F16 ? 1 : 0);
            const uint32_t pa = smem_u32(p_smem);
            int s = 0;
            uint32_t ph = 0, gq = 0, gp = 0;   // key tiles so far: scores, products with V
            bool ok = true;
            uint32_t qa = 0;
            int qi = 0;
            auto qk = [&](bool last) {
                if (gq >= 2) ok = ok && mbar_wait(&bars.s_read[gq & 1], ((gq - 2) >> 1) & 1u, lim);
                for (int c = 0; c < nh; ++c) {
                    ok = ok && mbar_wait(&bars.kv_full[s], ph, lim);
                    if (!ok) return;
                    tc_fence_after();
                    const uint32_t ka = smem_u32(ring + (size_t)s * stage);
                    for (int g = 0; g < min(2, ng - 2 * c); ++g) {
                        const uint64_t dk = umma_desc_k_sw128(ka + g * CN_GROUP), dq = umma_desc_k_sw128(qa + (2 * c + g) * slab);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (4 * (2 * c + g) + k < ks) umma_bf16(tmem + (gq & 1) * N, dk + 2 * k, dq + 2 * k, id_s, (c | g | k) != 0);
                    }
                    umma_commit(&bars.kv_empty[s]);
                    if (++s == nst) { s = 0; ph ^= 1u; }
                }
                umma_commit(&bars.s_full[gq & 1]);
                if (last) umma_commit(&bars.q_empty[qi]);
                ++gq;
            };
            for (int seg = 0; ok; ++seg) {
                ok = mbar_wait(&bars.seg[seg & (CT_SLOTS - 1)], (uint32_t)(seg / CT_SLOTS) & 1u, lim);
                if (!ok) break;
                const CtSeg &w = s_seg[seg & (CT_SLOTS - 1)];
                if (w.whole < 0) break;
                const int first = w.tile, end = w.end;
                qi = seg & 1;
                ok = mbar_wait(&bars.q_full[qi], (uint32_t)(seg >> 1 & 1), lim);
                if (!ok) break;
                tc_fence_after();
                qa = smem_u32(q_smem + (size_t)qi * ng * slab);
                qk(first + 1 == end);
                for (int i = first; i < end && ok; ++i, ++gp) {
                    if (i + 1 < end) qk(i + 2 == end);
                    if (i == first) ok = ok && mbar_wait(&bars.o_empty[seg & 1], (uint32_t)(seg >> 1 & 1) ^ 1u, lim);   // the epilogue two units back has read O
                    ok = ok && mbar_wait(&bars.p_full[gp & 1], (gp >> 1) & 1u, lim);
                    for (int c = 0; c < nh; ++c) {
                        ok = ok && mbar_wait(&bars.ready[s], ph, lim);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t va = smem_u32(ring + (size_t)s * stage), t_o = tmem + 2 * N + ((seg & 1) * nh + c) * N;
                        const uint64_t dp = umma_desc_k_sw128(pa + (gp & 1) * 2 * slab);
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            umma_bf16(t_o, umma_desc_mn_sw128(va + k * 2048, CN_GROUP), dp + (k >> 2) * (slab >> 4) + 2 * (k & 3), id_o, (i > first || k != 0) ? 1u : 0u);
                        umma_commit(&bars.kv_empty[s]);
                        if (++s == nst) { s = 0; ph ^= 1u; }
                    }
                    if (!ok) break;
                    umma_commit(&bars.o_done[gp & 1]);
                }
            }
            if (!ok) CN_FAIL_AT(2, true)
        }
    } else if (warp >= 4) {
        // ---- softmax: thread = key of the tile; epilogue: thread = output column ----
        // (a thread whose wait has run out goes on through the barriers of the four warps until they all leave together, so that none waits for it there)
        const int q = warp & 3, tid = threadIdx.x & 127;
        const uint32_t tl = tmem + ((uint32_t)(32 * q) << 16);
        const uint32_t pw = smem_u32(p_smem) + (uint32_t)(tid >> 6) * slab + (uint32_t)(tid & 7) * 2;
        const uint32_t chunk = (uint32_t)(tid & 63) >> 3;
        const float sl2 = p.scale_log2;
        const int R = p.R;
        uint32_t g = 0;   // key tiles so far
        auto pv_done = [&](uint32_t x) { return mbar_wait(&bars.o_done[x & 1], (x >> 1) & 1u, lim); };
        for (int seg = 0;; ++seg) {
            CN_FAIL_AT(7, !mbar_wait(&bars.seg[seg & (CT_SLOTS - 1)], (uint32_t)(seg / CT_SLOTS) & 1u, lim));
            if (ct_any(failed)) break;
            const CtSeg &w = s_seg[seg & (CT_SLOTS - 1)];
            if (w.whole < 0) break;
            const int first = w.tile, end = w.end, nct = w.ct;
            const uint32_t t_o = 2 * N + (seg & 1) * nh * N;
            float l[N];
#pragma unroll
            for (int r = 0; r < N; ++r) l[r] = 0.0f;
            bool stop = false;
            for (int i = first; i < end; ++i, ++g) {
                const bool draft = i >= nct;
                const int j = (draft ? i - nct : i) * CN_TK + tid;   // this thread's key
                const bool there = j < (draft ? p.T : w.n);
                CN_FAIL_AT(3, !mbar_wait(&bars.s_full[g & 1], (g >> 1) & 1u, lim));
                tc_fence_after();
                float x[N];
                {
                    uint32_t raw[16];
#pragma unroll
                    for (int c = 0; c < N; c += 16) {
                        if (c < R) {
                            tmem_ld16(tl + (g & 1) * N + c, raw);
                            tmem_ld_wait();
                        }
#pragma unroll
                        for (int r = 0; r < 16; ++r) x[c + r] = there && c + r < R ? __uint_as_float(raw[r]) : -INFINITY;
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.s_read[g & 1]);   // these scores may be overwritten
                if (draft) {   // rows t G .. t G + G - 1 are token t's
                    unsigned long long hidden;
                    if (p.mask == nullptr) {   // a chain: this key is seen from its own token on
                        const int first_row = min(j * p.G, 64);
                        hidden = first_row == 64 ? ~0ull : (1ull << first_row) - 1ull;
                    } else {
                        const unsigned long long token = p.G == 64 ? ~0ull : (1ull << p.G) - 1ull;
                        const unsigned char *col = p.mask + w.b * p.mask_b + min(j, p.T - 1);
                        hidden = 0;
                        for (int t0 = 0; t0 < p.T; t0 += 8) {
                            unsigned char see[8];
#pragma unroll
                            for (int k = 0; k < 8; ++k) see[k] = t0 + k < p.T ? __ldg(col + (long long)(t0 + k) * p.T) : 1;
#pragma unroll
                            for (int k = 0; k < 8; ++k)
                                if (see[k] == 0) hidden |= token << ((t0 + k) * p.G);
                        }
                    }
#pragma unroll
                    for (int r = 0; r < N; ++r)
                        if (hidden >> r & 1ull) x[r] = -INFINITY;
                }
                float top = -INFINITY;   // the largest score over its row's reference
#pragma unroll
                for (int r0 = 0; r0 < N; r0 += 16) {   // (16 rows without a branch)
                    if (r0 >= R) break;
#pragma unroll
                    for (int r = r0; r < r0 + 16; r += 4) {
                        const float4 n4 = *reinterpret_cast<const float4 *>(s_neg + r);
                        top = ct_max3(top, fmaf(x[r], sl2, n4.x), fmaf(x[r + 1], sl2, n4.y));
                        top = ct_max3(top, fmaf(x[r + 2], sl2, n4.z), fmaf(x[r + 3], sl2, n4.w));
                    }
                }
                if (ct_any(top > CT_RESCALE_LOG2 || failed)) {
                    if (ct_any(failed)) { stop = true; break; }
                    // ---- new references where a row's maximum is beyond its own; what has been added up so far is rescaled ----
#pragma unroll
                    for (int r0 = 0; r0 < N; r0 += 16) {
                        if (r0 >= R) break;
                        float m[16];
#pragma unroll
                        for (int r = 0; r < 16; ++r) m[r] = cn_warp_max(x[r0 + r]);
#pragma unroll
                        for (int r = 0; r < 16; r += 4)
                            if (lane == 0) *reinterpret_cast<float4 *>(&s_red[q][r0 + r]) = make_float4(m[r], m[r + 1], m[r + 2], m[r + 3]);
                    }
                    ct_sync();
                    if (tid < R) {
                        const float mx = fmaxf(fmaxf(s_red[0][tid], s_red[1][tid]), fmaxf(s_red[2][tid], s_red[3][tid])), m = mx * sl2, old = s_neg[tid];
                        float f = 1.0f;
                        if (m + old > CT_RESCALE_LOG2) {
                            f = old == CN_UNSET ? 0.0f : fast_exp2(-old - m);
                            s_neg[tid] = -m;
                            s_x[tid] = mx;
                            if (ca_large(m)) s_large = 1;
                        }
                        s_f[tid] = f;
                    }
                    ct_sync();
#pragma unroll
                    for (int r = 0; r < N; ++r)
                        if (r < R) l[r] *= s_f[r];
                    if (i > first) {
                        CN_FAIL_AT(4, !pv_done(g - 1));
                        tc_fence_after();
                        for (int c = 0; c < nh; ++c)
#pragma unroll
                            for (int r0 = 0; r0 < N; r0 += 16) {
                                if (r0 >= R) break;
                                uint32_t o[16];
                                tmem_ld16(tl + t_o + c * N + r0, o);
                                tmem_ld_wait();
#pragma unroll
                                for (int r = 0; r < 16; ++r) o[r] = __float_as_uint(__uint_as_float(o[r]) * (r0 + r < R ? s_f[r0 + r] : 1.0f));
                                tmem_st16(tl + t_o + c * N + r0, o);
                            }
                        tmem_st_wait();
                    }
                }
                if (g >= 2) CN_FAIL_AT(5, !pv_done(g - 2));   // the MMAs have read what was in this P buffer
                const uint32_t pb = pw + (g & 1) * 2 * slab;
                const float *refs = s_neg;
                if (s_large) {   // (the same for all four warps)
                    refs = s_zero;
#pragma unroll
                    for (int r = 0; r < N; ++r)
                        if (r < R) x[r] -= s_x[r];
                }
#pragma unroll
                for (int r0 = 0; r0 < N; r0 += 8) {   // (8 rows without a branch)
                    if (r0 >= R) break;
                    const float4 na = *reinterpret_cast<const float4 *>(refs + r0), nb = *reinterpret_cast<const float4 *>(refs + r0 + 4);
                    const float nn[8] = {na.x, na.y, na.z, na.w, nb.x, nb.y, nb.z, nb.w};
                    float e[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) e[k] = fast_exp2(fmaf(x[r0 + k], sl2, nn[k]));
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        l[r0 + k] += e[k];
                        ct_st_shared_u16(pb + (r0 + k) * 128 + ((chunk ^ k) << 4), pack_16(e[k], F16));
                    }
                }
                fence_proxy_async_smem();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.p_full[g & 1]);
            }
            if (stop || ct_any(failed)) break;
            // ---- the unit's sums, then its outputs ----
#pragma unroll
            for (int r0 = 0; r0 < N; r0 += 16) {   // (16 reductions side by side: one after the other they cost 32 rows 2 us)
                if (r0 >= R) break;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1)
#pragma unroll
                    for (int r = 0; r < 16; ++r) l[r0 + r] += __shfl_xor_sync(0xffffffffu, l[r0 + r], o);
#pragma unroll
                for (int r = 0; r < 16; r += 4)
                    if (lane == 0) *reinterpret_cast<float4 *>(&s_red[q][r0 + r]) = make_float4(l[r0 + r], l[r0 + r + 1], l[r0 + r + 2], l[r0 + r + 3]);
            }
            ct_sync();
            const bool whole = w.whole != 0, bad = s_bad[seg & (CT_SLOTS - 1)] == seg + 1;
            float *prt = p.part + ((size_t)blockIdx.x * 2 + (seg == 0 ? 0 : 1)) * ca_slot_floats(p.RT, p.D);
            const int b = w.b, h = w.h;
            if (tid < R) {
                const float sum = s_red[0][tid] + s_red[1][tid] + s_red[2][tid] + s_red[3][tid], neg = s_neg[tid], m = neg == CN_UNSET ? -INFINITY : -neg;
                if (!whole) {
                    prt[(size_t)p.RT * p.D + 2 * tid] = m;
                    prt[(size_t)p.RT * p.D + 2 * tid + 1] = sum;
                } else if (p.lse) {
                    p.lse[((long long)b * p.Hq + h * p.G + tid % p.G) * p.T + tid / p.G] = sum == 0.0f ? -INFINITY : (m + log2f(sum)) * 0.69314718055994531f;
                }
                s_inv[tid] = sum == 0.0f ? 0.0f : 1.0f / sum;
                s_neg[tid] = CN_UNSET;
                s_x[tid] = 0.0f;
                if (tid == 0) s_large = 0;
            }
            CN_FAIL_AT(6, !pv_done(g - 1));
            tc_fence_after();
            ct_sync();
            bool odd = false;   // a sum is NaN
            for (int c = 0; c < nh; ++c) {
                // lane -> column: with 64 rows in the MMA, row d of the accumulator is in lane 32 (d / 16) + d % 16
                const int d = p.D <= 64 ? (lane < 16 ? 16 * q + lane : p.D) : 128 * c + tid;
#pragma unroll
                for (int r0 = 0; r0 < N; r0 += 16) {
                    if (r0 >= R) break;
                    uint32_t o[16];
                    tmem_ld16(tl + t_o + c * N + r0, o);
                    tmem_ld_wait();
                    if (bad && d < p.D) {   // values of new tokens that are not finite, for the rows that see them
                        for (int j = max(first - nct, 0) * CN_TK; j < min(p.T, (end - nct) * CN_TK); ++j) {
                            const float v = to_f32(ca_row<T>(p.Vd, p.vd, b, h, j)[d]);
                            if (fabsf(v) < INFINITY) continue;
#pragma unroll
                            for (int r = 0; r < 16; ++r) {
                                const int t = (r0 + r) / p.G;
                                if (r0 + r < R && (p.mask ? p.mask[b * p.mask_b + (long long)t * p.T + j] != 0 : j <= t)) o[r] = __float_as_uint(__uint_as_float(o[r]) + v);
                            }
                        }
                    }
                    int t = r0 / p.G, hg = r0 % p.G;
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        if (r0 + r < R && d < p.D) {
                            const float v = __uint_as_float(o[r]);
                            odd |= v != v;
                            if (whole) {
                                const uint16_t y = pack_16(v * s_inv[r0 + r], F16);
                                *reinterpret_cast<uint16_t *>(ca_row<T>(p.O, p.o, b, h * p.G + hg, t) + d) = y;
                            } else {
                                prt[(size_t)(r0 + r) * p.D + d] = v;
                            }
                        }
                        if (++hg == p.G) { hg = 0; ++t; }
                    }
                    __syncwarp();
                }
            }
            if (__any_sync(0xffffffffu, odd)) {
                for (int c = 0; c < nh; ++c) {
                    const int d = p.D <= 64 ? (lane < 16 ? 16 * q + lane : p.D) : 128 * c + tid;
                    const unsigned cached = ct_cached_kinds<F16>(p, b, h, first * CN_TK, min(w.n, min(end, nct) * CN_TK), d);
                    for (int r = 0; d < p.D && r < R; ++r) {
                        if (s_inv[r] != s_inv[r]) continue;   // (a score was NaN)
                        const int t = r / p.G;
                        const unsigned kinds = cached | ca_new_kinds<T>(p, b, h, max(first - nct, 0) * CN_TK, min(p.T, (end - nct) * CN_TK), t, d);
                        if (whole) ca_settle(ca_row<T>(p.O, p.o, b, h * p.G + r % p.G, t) + d, kinds);
                        else ca_settle(prt + (size_t)r * p.D + d, kinds);
                    }
                    __syncwarp();
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.o_empty[seg & 1]);
        }
    }

    if (failed) for (int i = 0; i < 2000; ++i) __nanosleep(1000);   // let copies and MMAs in flight drain
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, (uint32_t)cn.tmem_cols);
}
#undef CN_FAIL_AT

}  // namespace b200attn
