// Accumulated attention weights on the 5th-generation tensor cores: bf16 / fp16, head_d a multiple of 8, at most 256, 16-byte aligned rows.
//     weights_j += sum over the accepted rows r that see key j of exp(s_rj - lse_r)
// lse is known, so there is no softmax to run: keys are the lanes of tensor memory, S^T [128 keys x rows] = K Q^T, and the thread of a key adds its
// rows up in registers, in the order of the rows, and to the array once: no atomics, no exchange between threads.
// The tiles of 128 keys of all (sequence, key head) pairs with accepted tokens are shared out evenly and contiguously over the CTAs (as in cache.cuh; a
// tile needs no joining).  Per pair the accepted rows of Q are gathered once into shared memory (the list names tokens anywhere); more rows than fit
// are taken in chunks, each over the CTA's tiles of the pair again.
//   warp 0       the walk over the tiles; one thread requests K tiles by TMA
//   warp 1       one thread issues the MMAs, 64 rows at a time into four buffers
//   warps 4-7    gather Q, then a thread per key
#pragma once

#include "cache_tc.cuh"

namespace b200attn {

constexpr int CX_THREADS = 256, CX_TK = 128, CX_NB = 64;
constexpr int CX_BUFS = 4;
constexpr int CX_SLOTS = 16;   // pairs that the roles can be at: one per ring stage (up to 8) and score buffer, and two

struct CxParams {
    CwParams a;
    int ng, nst;       // groups of 64 columns, ring stages
    int chunk;         // rows of Q that shared memory holds: a multiple of 64
    int grid;
};
struct CxSeg { int b, h, n, tile, end, count; };   // count -1: no more
struct CxBars {
    uint64_t k_full[CT_MAX_STAGES], k_empty[CT_MAX_STAGES];
    uint64_t seg[CX_SLOTS];
    uint64_t q_ready;
    uint64_t s_full[CX_BUFS], s_read[CX_BUFS];
};

// rows cached for a sequence, 0 where it has accepted nothing
__device__ __forceinline__ int cx_len(const CwParams &p, int b) {
    if (p.accepted && (unsigned)__ldg(p.accepted + (long long)b * p.A) >= (unsigned)p.T) return 0;
    return ca_len(p.len, b, p.S);
}

template <bool F16>
__global__ void __launch_bounds__(CX_THREADS, 1)
cw_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CxParams cx) {
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
    const uint32_t stage = (uint32_t)ng * CX_TK * 128u, slab = (uint32_t)chunk * 128u;
    unsigned char *q_smem = smem;                                        // [ng][chunk rows][128 B]
    unsigned char *ring = q_smem + (size_t)ng * slab;                    // [nst][ng][128 keys][128 B]
    float *s_nl = reinterpret_cast<float *>(ring + (size_t)nst * stage); // [chunk]: minus lse, log2 units
    int *s_i = reinterpret_cast<int *>(s_nl + chunk);                    // [chunk]: which accepted token
    const uint32_t lim = p.spin_limit;

    if (threadIdx.x == 0) {
        for (int i = 0; i < CT_MAX_STAGES; ++i) { mbar_init(&bars.k_full[i], 1); mbar_init(&bars.k_empty[i], 1); }
        for (int i = 0; i < CX_SLOTS; ++i) mbar_init(&bars.seg[i], 1);
        mbar_init(&bars.q_ready, 4);
        for (int i = 0; i < CX_BUFS; ++i) { mbar_init(&bars.s_full[i], 1); mbar_init(&bars.s_read[i], 4); }
        mbar_fence_init();
        tma_prefetch_desc(&tmK);
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
        auto items = [&](int b) { return b < p.B ? (long long)p.Hkv * ((cx_len(p, b) + CX_TK - 1) / CX_TK) : 0ll; };
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
        uint32_t ph = 0;
        bool ok = true;
        while (at < i1 && ok) {
            const int n = cx_len(p, b), ct = (n + CX_TK - 1) / CX_TK;
            if ((long long)p.Hkv * ct <= at - before) { before += (long long)p.Hkv * ct; ++b; continue; }
            const int h = (int)((at - before) / ct), tile = (int)((at - before) % ct), end = (int)min((long long)ct, tile + (i1 - at));
            const int count = ca_count(p.accepted, b, p.A, p.T, n);
            const int chunks = (count * p.G + chunk - 1) / chunk;
            if (lane == 0) {
                s_seg[seg & (CX_SLOTS - 1)] = CxSeg{b, h, n, tile, end, count};
                mbar_arrive(&bars.seg[seg & (CX_SLOTS - 1)]);
            }
            __syncwarp();
            if (elect_one()) {
                for (int c = 0; c < chunks && ok; ++c)
                    for (int i = tile; i < end && ok; ++i) {
                        ok = mbar_wait(&bars.k_empty[s], ph ^ 1u, lim);
                        if (!ok) break;
                        mbar_expect_tx(&bars.k_full[s], stage);
                        for (int g = 0; g < ng; ++g) tma_load_4d(ring + (size_t)s * stage + (size_t)g * (CX_TK * 128), &tmK, g * 64, i * CX_TK, h, b, &bars.k_full[s]);
                        if (++s == nst) { s = 0; ph ^= 1u; }
                    }
            }
            __syncwarp();
            ok = __all_sync(0xffffffffu, ok);
            at += end - tile;
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
            uint32_t ph = 0, blk = 0, qn = 0;   // ring, blocks of 64 rows so far, gathered chunks so far
            bool ok = true;
            for (int seg = 0; ok; ++seg) {
                ok = mbar_wait(&bars.seg[seg & (CX_SLOTS - 1)], (uint32_t)(seg / CX_SLOTS) & 1u, lim);
                if (!ok) break;
                const CxSeg w = s_seg[seg & (CX_SLOTS - 1)];
                if (w.count < 0) break;
                for (int r0 = 0; r0 < w.count * p.G && ok; r0 += chunk, ++qn) {
                    const int rows = min(chunk, w.count * p.G - r0);
                    ok = mbar_wait(&bars.q_ready, qn & 1u, lim);
                    for (int i = w.tile; i < w.end && ok; ++i) {
                        ok = mbar_wait(&bars.k_full[s], ph, lim);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t ka = smem_u32(ring + (size_t)s * stage);
                        for (int n0 = 0; n0 < rows; n0 += CX_NB, ++blk) {
                            const uint32_t u = blk & (CX_BUFS - 1);
                            ok = mbar_wait(&bars.s_read[u], (uint32_t)(blk / CX_BUFS & 1) ^ 1u, lim);
                            if (!ok) break;
                            tc_fence_after();
                            const uint32_t id = umma_idesc_16(128, min(CX_NB, (rows - n0 + 15) & ~15), 0, 0, F16 ? 1 : 0);
                            const uint32_t qa = smem_u32(q_smem) + (uint32_t)n0 * 128u;
                            for (int g = 0; g < ng; ++g) {
                                const uint64_t dk = umma_desc_k_sw128(ka + g * (CX_TK * 128)), dq = umma_desc_k_sw128(qa + g * slab);
#pragma unroll
                                for (int k = 0; k < 4; ++k)
                                    if (4 * g + k < ks) umma_bf16(tmem + u * CX_NB, dk + 2 * k, dq + 2 * k, id, (g | k) != 0);
                            }
                            umma_commit(&bars.s_full[u]);
                        }
                        if (!ok) break;
                        umma_commit(&bars.k_empty[s]);
                        if (++s == nst) { s = 0; ph ^= 1u; }
                    }
                }
            }
            if (!ok) { report_kernel_error(p.err, p.err_sys, (unsigned)KERR_MBAR_TIMEOUT | (1u << 17)); failed = true; }
        }
    } else if (warp >= 4) {
        const int q = warp & 3, tid = threadIdx.x & 127;
        const uint32_t tl = tmem + ((uint32_t)(32 * q) << 16);
        const float sl2 = p.scale_log2;
        uint32_t blk = 0;
        bool ok = true;
        // (a thread whose wait has run out goes on through the barriers of the four warps until they all leave together, so that none waits for it there)
        for (int seg = 0;; ++seg) {
            ok = ok && mbar_wait(&bars.seg[seg & (CX_SLOTS - 1)], (uint32_t)(seg / CX_SLOTS) & 1u, lim);
            if (ct_any(!ok)) { ok = false; break; }
            const CxSeg w = s_seg[seg & (CX_SLOTS - 1)];
            if (w.count < 0) break;
            float *wrow = p.weights + ((long long)w.b * p.Hkv + w.h) * p.S;
            for (int r0 = 0; r0 < w.count * p.G; r0 += chunk) {
                const int rows = min(chunk, w.count * p.G - r0);
                // ---- gather: the MMAs that read the rows before these have completed (their scores have been taken by every thread) ----
                if (ct_any(!ok)) { ok = false; break; }
                const int padded = (rows + 15) & ~15, pieces = ng * 8;   // rows of zeros up to whole MMA columns; 16-byte pieces of a row
                for (int x = tid; x < padded * pieces; x += 128) {
                    const int r = x / pieces, c = x % pieces, rr = r0 + r, i = rr / p.G;
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (r < rows && c * 8 < p.D) {
                        const int t = p.accepted ? __ldg(p.accepted + (long long)w.b * p.A + i) : i;
                        v = *reinterpret_cast<const uint4 *>(ca_row<T>(p.Q, p.q, w.b, w.h * p.G + rr % p.G, t) + c * 8);
                    }
                    *reinterpret_cast<uint4 *>(q_smem + (size_t)(c >> 3) * slab + (size_t)r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v;
                }
                for (int r = tid; r < rows; r += 128) {
                    const int rr = r0 + r, i = rr / p.G, t = p.accepted ? __ldg(p.accepted + (long long)w.b * p.A + i) : i;
                    const float x = p.lse[((long long)w.b * p.Hq + w.h * p.G + rr % p.G) * p.T + t];
                    s_nl[r] = -1.4426950408889634f * x;
                    s_i[r] = x == -INFINITY ? -1 : i;   // a token that saw nothing gave no weight
                }
                fence_proxy_async_smem();
                ct_sync();
                if (lane == 0) mbar_arrive(&bars.q_ready);
                for (int t = w.tile; t < w.end; ++t) {
                    const int j = t * CX_TK + tid, first = j - (w.n - w.count);   // the first accepted token that sees this key (<= 0: all do)
                    const bool there = j < w.n;
                    // rows of tokens that saw nothing, and keys behind the first accepted token, are looked at one by one
                    const float old = there ? wrow[j] : 0.0f;
                    const bool all = (t + 1) * CX_TK <= w.n - w.count;
                    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    for (int n0 = 0; n0 < rows; n0 += CX_NB, ++blk) {
                        const uint32_t u = blk & (CX_BUFS - 1);
                        ok = ok && mbar_wait(&bars.s_full[u], (uint32_t)(blk / CX_BUFS) & 1u, lim);
                        ok = __all_sync(0xffffffffu, ok);
                        tc_fence_after();
#pragma unroll
                        for (int c = 0; c < CX_NB; c += 16) {
                            if (n0 + c >= rows) break;
                            uint32_t raw[16];
                            tmem_ld16(tl + u * CX_NB + c, raw);
                            tmem_ld_wait();
                            const float4 *nl = reinterpret_cast<const float4 *>(s_nl + n0 + c);
                            const int4 *si = reinterpret_cast<const int4 *>(s_i + n0 + c);
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const float4 l4 = nl[k];
                                const int4 i4 = si[k];
                                const int left = rows - (n0 + c + 4 * k), f = all ? 0 : max(first, 0);
                                const float e0 = fast_exp2(fmaf(__uint_as_float(raw[4 * k]), sl2, l4.x)), e1 = fast_exp2(fmaf(__uint_as_float(raw[4 * k + 1]), sl2, l4.y));
                                const float e2 = fast_exp2(fmaf(__uint_as_float(raw[4 * k + 2]), sl2, l4.z)), e3 = fast_exp2(fmaf(__uint_as_float(raw[4 * k + 3]), sl2, l4.w));
                                if (0 < left && i4.x >= f) sum[0] += e0;
                                if (1 < left && i4.y >= f) sum[1] += e1;
                                if (2 < left && i4.z >= f) sum[2] += e2;
                                if (3 < left && i4.w >= f) sum[3] += e3;
                            }
                        }
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&bars.s_read[u]);
                    }
                    if (there && ok) wrow[j] = old + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
                }
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
