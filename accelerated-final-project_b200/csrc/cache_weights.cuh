// Accumulated attention weights on the 5th-generation tensor cores: bf16 / fp16, head_d a multiple of 8, at most 256, 16-byte aligned rows.
//     weights_j += sum over the accepted rows r that see key j of exp(s_rj - lse_r)
// lse is known, so there is no softmax to run: keys are the lanes of tensor memory, S^T [128 keys x rows] = K Q^T, and the thread of a key adds its
// rows up in registers, in the order of the rows, and to the array once: no atomics, no exchange between threads.
// The tiles of 128 keys of all (sequence, key head) pairs with accepted tokens are shared out evenly and contiguously over the CTAs (as in cache.cuh; a
// tile needs no joining).  Per pair the accepted rows of Q are brought into shared memory once: by TMA where all new tokens are accepted, else gathered
// (the list names tokens anywhere).  More rows than fit are taken in chunks, each over the CTA's tiles of the pair again.  Blocks of rows that see nothing
// of a tile are left out.
//   32 sequences, up to 6 tokens, 32 / 8 heads of 128, 100 to 8000 rows, bf16 (244 MB read): 47 us, 5.2 TB/s; 700 tokens, 16 heads of 64, up to 2501 rows: 28 us,
//   bound by the exponentials of 11 blocks a tile.
//   warp 0       the walk over the tiles; one thread requests K tiles (and Q) by TMA
//   warp 1       one thread issues the MMAs, 64 rows at a time, into two buffers per summing warpgroup
//   warps 2, 3   gather the next rows of Q beside the present ones (61 us a call of 32 sequences, up to 6 tokens, 100 to 8000 rows, where the
//                summing warps did it between two pairs; 49 so)
//   warps 4-11   two warpgroups take the tiles in turn; a thread per key: its exponentials and their sum (bound by the latency of that chain: one
//                warpgroup was as fast with 24 rows, and 30 against 28 us with 700)
#pragma once

#include "cache_tc.cuh"

namespace b200attn {

constexpr int CX_THREADS = 384, CX_TK = 128, CX_NB = 64;   // (64 rows a block)
constexpr int CX_BUFS = 4;
// What a pair's beginning and end cost a CTA, in tiles, as in cache.cuh: two tiles of a block of rows (none: a CTA with 20 short sequences took 62 us
// where the others took 40; two also where a tile has eleven blocks: 34 us instead of 28).
__host__ __device__ inline int cx_overhead(long long rows) { return rows <= CX_NB ? 2 : rows <= 2 * CX_NB ? 1 : 0; }
constexpr int CX_SLOTS = 16;   // pairs that the roles can be at: one per ring stage (up to 8) and score buffer, and two

struct CxParams {
    CwParams a;
    int ng, nst;       // groups of 64 columns, ring stages
    int chunk, nq;     // rows of Q that a buffer holds: a multiple of 64; buffers
    int box_t;         // tokens of a Q box, a chunk is whole boxes of whole groups of 8 rows; 0: rows are gathered
    int grid, oh;      // CTAs; items in front of a pair's tiles
    // first row of a chunk [r0, ..) that sees something of tile t, down to whole blocks
    __device__ __forceinline__ int first_row(int t, int seen_by_all, int r0) const {
        const long long r = (long long)(t * CX_TK - seen_by_all) * a.G - r0;
        return r <= 0 ? 0 : (int)(r / CX_NB * CX_NB);
    }
};
struct CxSeg { int b, h, n, tile, end, count; };   // count -1: no more
struct CxBars {
    uint64_t k_full[CT_MAX_STAGES], k_empty[CT_MAX_STAGES];
    uint64_t seg[CX_SLOTS];
    uint64_t q_full[2], q_empty[2];
    uint64_t s_full[CX_BUFS], s_read[CX_BUFS];
};

// rows cached for a sequence, 0 where it has accepted nothing
__device__ __forceinline__ int cx_len(const CwParams &p, int b) {
    if (p.accepted && (unsigned)__ldg(p.accepted + (long long)b * p.A) >= (unsigned)p.T) return 0;
    return ca_len(p.len, b, p.S);
}

template <bool F16>
__global__ void __launch_bounds__(CX_THREADS, 1)
cw_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CxParams cx) {
    using T = typename CtType<F16>::T;
    extern __shared__ unsigned char ct_smem_raw[];
    __shared__ CxBars bars;
    __shared__ CxSeg s_seg[CX_SLOTS];
    __shared__ uint32_t tmem_slot;
    const CwParams &p = cx.a;
    const uint32_t raw_addr = smem_u32(ct_smem_raw);
    unsigned char *smem = ct_smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ng = cx.ng, nst = cx.nst, chunk = cx.chunk;
    const int pitch = (chunk + CX_NB - 1) / CX_NB * CX_NB;                // rows of a Q buffer: whole blocks
    const uint32_t stage = (uint32_t)ng * CX_TK * 128u, slab = (uint32_t)pitch * 128u;
    unsigned char *q_smem = smem;                                        // [nq][ng][pitch rows][128 B]
    unsigned char *ring = q_smem + (size_t)cx.nq * ng * slab;            // [nst][ng][128 keys][128 B]
    float *s_nl = reinterpret_cast<float *>(ring + (size_t)nst * stage); // [nq][pitch]: minus lse, log2 units
    int *s_i = reinterpret_cast<int *>(s_nl + cx.nq * pitch);            // [nq][pitch]: which accepted token; -1: one that saw nothing
    __shared__ int s_skip[2];                                            // some row of the buffer saw nothing
    const uint32_t lim = p.spin_limit;

    if (threadIdx.x == 0) {
        for (int i = 0; i < CT_MAX_STAGES; ++i) { mbar_init(&bars.k_full[i], 1 + p.wait_extra); mbar_init(&bars.k_empty[i], 1); }
        for (int i = 0; i < CX_SLOTS; ++i) mbar_init(&bars.seg[i], 1);
        for (int i = 0; i < 2; ++i) { mbar_init(&bars.q_full[i], cx.box_t ? 3 : 2); mbar_init(&bars.q_empty[i], 8); s_skip[i] = 0; }
        for (int i = 0; i < CX_BUFS; ++i) { mbar_init(&bars.s_full[i], 1); mbar_init(&bars.s_read[i], 4); }
        mbar_fence_init();
        tma_prefetch_desc(&tmK);
        if (cx.box_t) tma_prefetch_desc(&tmQ);
    }
    if (warp == 1) tmem_alloc(&tmem_slot, CX_BUFS * CX_NB);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    grid_launch_dependents();
    grid_dependency_wait();
    const uint32_t tmem = tmem_slot;
    bool failed = false;

    if (warp == 0) {
        // ---- the walk: this CTA's range [i0, i1) of the tiles of all pairs ----
        long long total = 0;
        auto items = [&](int b) {
            const int ct = b < p.B ? (cx_len(p, b) + CX_TK - 1) / CX_TK : 0;
            return ct > 0 ? (long long)p.Hkv * (cx.oh + ct) : 0ll;
        };
        for (int b0 = 0; b0 < p.B; b0 += 32) {
            long long x = items(b0 + lane);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
            total += x;
        }
        long long at = total * blockIdx.x / cx.grid;
        const long long i1 = total * (blockIdx.x + 1) / cx.grid;
        int b = 0;
        long long before = 0;   // items of the sequences before b
        for (int b0 = 0; b0 < p.B && at < i1; b0 += 32) {
            const long long x = items(b0 + lane);
            long long incl = x;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long y = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += y;
            }
            const unsigned past = __ballot_sync(0xffffffffu, before + incl > at);
            if (past) {
                const int k = __ffs(past) - 1;
                b = b0 + k;
                before += __shfl_sync(0xffffffffu, incl - x, k);
                break;
            }
            before += __shfl_sync(0xffffffffu, incl, 31);
        }
        int s = 0, seg = 0;
        uint32_t ph = 0, qn = 0;
        bool ok = true;
        while (at < i1 && ok) {
            const int n = cx_len(p, b), ct = (n + CX_TK - 1) / CX_TK, per = ct > 0 ? cx.oh + ct : 0;
            if ((long long)p.Hkv * per <= at - before) { before += (long long)p.Hkv * per; ++b; continue; }
            const int h = (int)((at - before) / per), from = (int)((at - before) % per), to = (int)min((long long)per, from + (i1 - at));
            const int tile = max(from - cx.oh, 0), end = to - cx.oh;
            at += to - from;
            if (end <= tile) continue;   // (a range that ends in front of a pair's tiles)
            const int count = ca_count(p.accepted, b, p.A, p.T, n);
            const int chunks = (count * p.G + chunk - 1) / chunk;
            if (lane == 0) {
                s_seg[seg & (CX_SLOTS - 1)] = CxSeg{b, h, n, tile, end, count};
                mbar_arrive(&bars.seg[seg & (CX_SLOTS - 1)]);
            }
            __syncwarp();
            if (elect_one()) {
                for (int c = 0; c < chunks && ok; ++c, ++qn) {
                    if (cx.box_t) {
                        const uint32_t qb = cx.nq == 2 ? qn & 1 : 0;
                        ok = mbar_wait(&bars.q_empty[qb], ((cx.nq == 2 ? qn >> 1 : qn) & 1u) ^ 1u, lim);
                        if (!ok) break;
                        const int boxes = (min(chunk, count * p.G - c * chunk) + p.G * cx.box_t - 1) / (p.G * cx.box_t);
                        mbar_expect_tx(&bars.q_full[qb], (uint32_t)(boxes * ng * p.G * cx.box_t) * 128u);
                        for (int k = 0; k < boxes; ++k)
                            for (int g = 0; g < ng; ++g)
                                tma_load_5d(q_smem + (size_t)(qb * ng + g) * slab + (size_t)k * p.G * cx.box_t * 128, &tmQ, g * 64, 0, c * (chunk / p.G) + k * cx.box_t, h, b, &bars.q_full[qb]);
                    }
                    for (int i = tile; i < end && ok; ++i) {
                        ok = mbar_wait(&bars.k_empty[s], ph ^ 1u, lim);
                        if (!ok) break;
                        mbar_expect_tx(&bars.k_full[s], stage);
                        for (int g = 0; g < ng; ++g) tma_load_4d(ring + (size_t)s * stage + (size_t)g * (CX_TK * 128), &tmK, g * 64, i * CX_TK, h, b, &bars.k_full[s]);
                        if (++s == nst) { s = 0; ph ^= 1u; }
                    }
                }
            }
            __syncwarp();
            ok = __all_sync(0xffffffffu, ok);
            ++seg;
        }
        if (ok) {
            if (lane == 0) {
                s_seg[seg & (CX_SLOTS - 1)].count = -1;
                mbar_arrive(&bars.seg[seg & (CX_SLOTS - 1)]);
            }
        } else {
            if (lane == 0) report_kernel_error(p.err, p.err_sys, (unsigned)KERR_MBAR_TIMEOUT | (1u << 16));
            failed = true;
        }
    } else if (warp == 1) {
        if (elect_one()) {
            const int ks = (p.D + 15) >> 4;
            int s = 0;
            uint32_t ph = 0, qn = 0, tn = 0;   // ring; chunks, tiles so far
            uint32_t blocks[2] = {0, 0};       // blocks of 64 rows so far, per summing warpgroup
            bool ok = true;
            for (int seg = 0; ok; ++seg) {
                ok = mbar_wait(&bars.seg[seg & (CX_SLOTS - 1)], (uint32_t)(seg / CX_SLOTS) & 1u, lim);
                if (!ok) break;
                const CxSeg w = s_seg[seg & (CX_SLOTS - 1)];
                if (w.count < 0) break;
                for (int r0 = 0; r0 < w.count * p.G && ok; r0 += chunk, ++qn) {
                    const int rows = min(chunk, w.count * p.G - r0);
                    const uint32_t qb = cx.nq == 2 ? qn & 1 : 0;
                    ok = mbar_wait(&bars.q_full[qb], (cx.nq == 2 ? qn >> 1 : qn) & 1u, lim);
                    for (int i = w.tile; i < w.end && ok; ++i, ++tn) {
                        uint32_t blk = tn & 1 ? blocks[1] : blocks[0];
                        ok = mbar_wait(&bars.k_full[s], ph, lim);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t ka = smem_u32(ring + (size_t)s * stage);
                        for (int n0 = cx.first_row(i, w.n - w.count, r0); n0 < rows; n0 += CX_NB, ++blk) {
                            const uint32_t u = 2 * (tn & 1) + (blk & 1);
                            ok = mbar_wait(&bars.s_read[u], (blk >> 1 & 1u) ^ 1u, lim);
                            if (!ok) break;
                            tc_fence_after();
                            const uint32_t id = umma_idesc_16(128, min(CX_NB, (rows - n0 + 15) & ~15), 0, 0, F16 ? 1 : 0);
                            const uint32_t qa = smem_u32(q_smem) + qb * ng * slab + (uint32_t)n0 * 128u;
                            for (int g = 0; g < ng; ++g) {
                                const uint64_t dk = umma_desc_k_sw128(ka + g * (CX_TK * 128)), dq = umma_desc_k_sw128(qa + g * slab);
#pragma unroll
                                for (int k = 0; k < 4; ++k)
                                    if (4 * g + k < ks) umma_bf16(tmem + u * CX_NB, dk + 2 * k, dq + 2 * k, id, (g | k) != 0);
                            }
                            umma_commit(&bars.s_full[u]);
                        }
                        if (!ok) break;
                        if (tn & 1) blocks[1] = blk; else blocks[0] = blk;
                        umma_commit(&bars.k_empty[s]);
                        if (++s == nst) { s = 0; ph ^= 1u; }
                    }
                }
            }
            if (!ok) { report_kernel_error(p.err, p.err_sys, (unsigned)KERR_MBAR_TIMEOUT | (1u << 17)); failed = true; }
        }
    } else if (warp < 4) {
        // ---- gather: rows of Q as the MMAs read them, 16-byte pieces, eight requests in flight per thread ----
        const int tid = threadIdx.x - 64;
        uint32_t qn = 0;
        bool ok = true;
        const int pieces = ng * 8;
        for (int seg = 0; ok; ++seg) {
            ok = __all_sync(0xffffffffu, mbar_wait(&bars.seg[seg & (CX_SLOTS - 1)], (uint32_t)(seg / CX_SLOTS) & 1u, lim));
            if (!ok) break;
            const CxSeg w = s_seg[seg & (CX_SLOTS - 1)];
            if (w.count < 0) break;
            const int *list = p.accepted ? p.accepted + (long long)w.b * p.A : nullptr;
            for (int r0 = 0; r0 < w.count * p.G; r0 += chunk, ++qn) {
                const uint32_t qb = cx.nq == 2 ? qn & 1 : 0;
                ok = __all_sync(0xffffffffu, mbar_wait(&bars.q_empty[qb], ((cx.nq == 2 ? qn >> 1 : qn) & 1u) ^ 1u, lim));
                if (!ok) break;
                unsigned char *dst = q_smem + (size_t)qb * ng * slab;
                const int rows = min(chunk, w.count * p.G - r0), todo = cx.box_t ? 0 : ((rows + 15) & ~15) * pieces;   // (rows of zeros up to whole MMA columns)
                for (int x0 = tid; x0 < todo; x0 += 64 * 8) {
                    uint4 v[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int x = x0 + 64 * k, r = x / pieces, c = x - r * pieces, rr = r0 + r, i = rr / p.G;
                        v[k] = make_uint4(0, 0, 0, 0);
                        if (r < rows && c * 8 < p.D)
                            v[k] = *reinterpret_cast<const uint4 *>(ca_row<T>(p.Q, p.q, w.b, w.h * p.G + rr - i * p.G, list ? __ldg(list + i) : i) + c * 8);
                    }
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int x = x0 + 64 * k, r = x / pieces, c = x - r * pieces;
                        if (x < todo) *reinterpret_cast<uint4 *>(dst + (size_t)(c >> 3) * slab + (size_t)r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v[k];
                    }
                }
                const int padded = (rows + 31) & ~31;   // rows that do not exist see nothing
                for (int x0 = tid; x0 < padded; x0 += 64 * 8) {
                    float x[8];
                    int at[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int rr = r0 + x0 + 64 * k;
                        at[k] = rr / p.G;
                        x[k] = x0 + 64 * k < rows ? p.lse[((long long)w.b * p.Hq + w.h * p.G + rr - at[k] * p.G) * p.T + (list ? __ldg(list + at[k]) : at[k])] : 0.0f;
                    }
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int r = x0 + 64 * k;
                        if (r < padded) {
                            s_nl[qb * pitch + r] = -1.4426950408889634f * x[k];
                            s_i[qb * pitch + r] = x[k] == -INFINITY || r >= rows ? -1 : at[k];
                            if (x[k] == -INFINITY) s_skip[qb] = (int)qn + 1;
                        }
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.q_full[qb]);
            }
        }
        if (!ok) { if (lane == 0) report_kernel_error(p.err, p.err_sys, (unsigned)KERR_MBAR_TIMEOUT | (1u << 19)); failed = true; }
    } else {
        const int q = warp & 3, tid = threadIdx.x & 127;
        const uint32_t tl = tmem + ((uint32_t)(32 * q) << 16);
        const float sl2 = p.scale_log2;
        const uint64_t sl2_2 = ct_pair(sl2, sl2);
        const uint32_t wg = (warp - 4) >> 2;
        uint32_t blk = 0, qn = 0, tn = 0;   // this warpgroup's blocks so far; chunks, tiles so far
        bool ok = true;
        for (int seg = 0; ok; ++seg) {
            ok = __all_sync(0xffffffffu, mbar_wait(&bars.seg[seg & (CX_SLOTS - 1)], (uint32_t)(seg / CX_SLOTS) & 1u, lim));
            if (!ok) break;
            const CxSeg w = s_seg[seg & (CX_SLOTS - 1)];
            if (w.count < 0) break;
            float *wrow = p.weights + ((long long)w.b * p.Hkv + w.h) * p.S;
            for (int r0 = 0; r0 < w.count * p.G && ok; r0 += chunk, ++qn) {
                const int rows = min(chunk, w.count * p.G - r0);
                const uint32_t qb = cx.nq == 2 ? qn & 1 : 0;
                ok = __all_sync(0xffffffffu, mbar_wait(&bars.q_full[qb], (cx.nq == 2 ? qn >> 1 : qn) & 1u, lim));
                if (!ok) break;
                const float *nl = s_nl + qb * pitch;
                const int *si = s_i + qb * pitch;
                const bool skip = s_skip[qb] == (int)qn + 1;
                const int mine = w.tile + ((tn ^ wg) & 1);   // this warpgroup's first tile
                tn += w.end - w.tile;
                float next = mine < w.end && mine * CX_TK + tid < w.n ? wrow[mine * CX_TK + tid] : 0.0f;   // (asked for a tile ahead)
                for (int t = mine; t < w.end && ok; t += 2) {
                    const int j = t * CX_TK + tid, first = max(j - (w.n - w.count), 0);   // the first accepted token that sees this key
                    const int n_first = cx.first_row(t, w.n - w.count, r0);
                    const bool there = j < w.n && n_first < rows;
                    const float old = next;
                    if (t + 2 < w.end) next = j + 2 * CX_TK < w.n ? wrow[j + 2 * CX_TK] : 0.0f;
                    const bool plain = !skip && (t + 1) * CX_TK <= w.n - w.count;         // every row sees every key of the tile
                    uint64_t sum[2] = {0, 0};
                    for (int n0 = n_first; n0 < rows && ok; n0 += CX_NB, ++blk) {
                        const uint32_t u = 2 * wg + (blk & 1);
                        ok = __all_sync(0xffffffffu, mbar_wait(&bars.s_full[u], blk >> 1 & 1u, lim));
                        if (!ok) break;
                        tc_fence_after();
                        uint32_t raw[CX_NB / 32][32];
#pragma unroll
                        for (int x = 0; x < CX_NB / 32; ++x)
                            if (n0 + 32 * x < rows) tmem_ld32(tl + u * CX_NB + 32 * x, raw[x]);
                        tmem_ld_wait();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&bars.s_read[u]);
#pragma unroll
                        for (int x = 0; x < CX_NB / 32; ++x) {   // (32 rows without a branch: one every 8 rows cost 27 clocks a row)
                            if (n0 + 32 * x >= rows) break;
                            const float4 *n4 = reinterpret_cast<const float4 *>(nl + n0 + 32 * x);
                            float e[32];
#pragma unroll
                            for (int k = 0; k < 32; k += 4) {
                                const float4 v = n4[k / 4];
                                ct_unpair(ct_fma2(ct_pair(__uint_as_float(raw[x][k]), __uint_as_float(raw[x][k + 1])), sl2_2, ct_pair(v.x, v.y)), e[k], e[k + 1]);
                                ct_unpair(ct_fma2(ct_pair(__uint_as_float(raw[x][k + 2]), __uint_as_float(raw[x][k + 3])), sl2_2, ct_pair(v.z, v.w)), e[k + 2], e[k + 3]);
                            }
#pragma unroll
                            for (int k = 0; k < 32; ++k) e[k] = fast_exp2(e[k]);
                            if (!plain || n0 + 32 * x + 32 > rows) {   // (the same for every thread)
                                const int4 *i4 = reinterpret_cast<const int4 *>(si + n0 + 32 * x);
#pragma unroll
                                for (int k = 0; k < 32; k += 4) {
                                    const int4 v = i4[k / 4];
                                    e[k] = v.x < first ? 0.0f : e[k];
                                    e[k + 1] = v.y < first ? 0.0f : e[k + 1];
                                    e[k + 2] = v.z < first ? 0.0f : e[k + 2];
                                    e[k + 3] = v.w < first ? 0.0f : e[k + 3];
                                }
                            }
#pragma unroll
                            for (int k = 0; k < 32; k += 8) {
                                sum[0] = ct_add2(sum[0], ct_add2(ct_pair(e[k], e[k + 1]), ct_pair(e[k + 2], e[k + 3])));
                                sum[1] = ct_add2(sum[1], ct_add2(ct_pair(e[k + 4], e[k + 5]), ct_pair(e[k + 6], e[k + 7])));
                            }
                        }
                    }
                    float a, c;
                    ct_unpair(ct_add2(sum[0], sum[1]), a, c);
                    if (there && ok) wrow[j] = old + (a + c);
                }
                if (!ok) break;
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.q_empty[qb]);
            }
        }
        if (!ok) { if (lane == 0) report_kernel_error(p.err, p.err_sys, (unsigned)KERR_MBAR_TIMEOUT | (1u << 18)); failed = true; }
    }

    if (failed) for (int i = 0; i < 2000; ++i) __nanosleep(1000);   // let copies and MMAs in flight drain
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, CX_BUFS * CX_NB);
}

}  // namespace b200attn
