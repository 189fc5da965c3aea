// sampling.cuh — from a step's logits to accepted tokens: probabilities at a
// temperature (qraf_cuda_token_probs) and the verification of drafted tokens
// against the target's probabilities (qraf_cuda_verify_drafts).
//
// The reference samples on the CPU after every forward (src/sampling/sampler.cpp)
// and verifies drafts token by token (src/runtime/speculative.cpp); here a batch's
// rows are one launch each.
#pragma once

#include <cooperative_groups.h>

#include "common.cuh"
#include "kv_cache.cuh"   // load4 / store4

namespace qraf_dev {

constexpr uint32_t kProbThreads = 512;
constexpr uint32_t kProbMaxCluster = 8;
constexpr uint32_t kProbSlice = 16384;       // values of a row that a CTA keeps in shared memory, at most,
                                             // while the cluster can grow: three CTAs an SM
constexpr uint32_t kProbSliceMax = 49152;    // with the largest cluster: one CTA an SM

struct ProbParams {
    const float* x;      // [rows] rows of vocab, x_ld apart
    float* out;          // the same, out_ld apart
    uint64_t x_ld, out_ld;
    uint32_t vocab, slice;   // values of a row per CTA of its cluster, a multiple of 4
    float scale;         // log2(e) / temperature
    uint32_t cached;     // the slice fits shared memory; else the row is read again
};

__device__ __forceinline__ float ex2_probs(float x) {   // 2^x, within 2 ulp; 0 at -inf
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Max or sum of v over the CTA's threads, to all of them.  s_red: one float a warp.
template <bool MAX>
__device__ __forceinline__ float block_reduce(float v, float* s_red) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float y = __shfl_xor_sync(0xFFFFFFFFu, v, o);
        v = MAX ? fmaxf(v, y) : __fadd_rn(v, y);
    }
    if (lane == 0u) s_red[warp] = v;
    __syncthreads();
    v = s_red[lane % (kProbThreads / 32u)];
#pragma unroll
    for (uint32_t o = kProbThreads / 64u; o > 0u; o >>= 1) {
        const float y = __shfl_xor_sync(0xFFFFFFFFu, v, o);
        v = MAX ? fmaxf(v, y) : __fadd_rn(v, y);
    }
    return v;
}

// out = exp((x - max) / T) / sum over each row; a row of nothing but -inf gives
// zeros.  A cluster has a row and each of its CTAs a slice that stays in shared
// memory, so the row is read once and written once.  A CTA takes its slice's own
// maximum and sum, and the cluster exchanges both at once: out = e 2^(own - all) / l.
// Measured on a B200: 320 rows of 32003 25 us, 3.3 TB/s read and written (640 CTAs on
// 444 places, each loading before it stores); 5 rows of 151936 7.2 us, latency.
__global__ void __launch_bounds__(kProbThreads) token_probs_kernel(const __grid_constant__ ProbParams p) {
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) float prob_smem[];
    __shared__ float s_max[kProbThreads / 32u], s_sum[kProbThreads / 32u];
    __shared__ float2 s_ml;
    const cg::cluster_group cl = cg::this_cluster();
    const uint32_t tid = threadIdx.x, rank = cl.block_rank(), blocks = cl.num_blocks();
    const uint64_t row = blockIdx.x / blocks;
    const uint32_t i0 = min(p.vocab, rank * p.slice), n = min(p.vocab, i0 + p.slice) - i0;
    const float* x = p.x + row * p.x_ld + i0;
    float* out = p.out + row * p.out_ld + i0;
    // values up to the first 16-byte boundary one by one, then by four
    const uint32_t hx = min(n, static_cast<uint32_t>((16u - (reinterpret_cast<uintptr_t>(x) & 15u)) & 15u) / 4u);
    const uint32_t qx = (n - hx) / 4u;
    float m = -INFINITY;
    auto each = [&](auto&& f1, auto&& f4) {
        if (tid < hx) f1(tid);
#pragma unroll 4
        for (uint32_t j = tid; j < qx; j += kProbThreads) f4(hx + 4u * j);
        const uint32_t rest = hx + 4u * qx;
        if (rest + tid < n) f1(rest + tid);
    };
    float* keep = prob_smem + 4u - hx;   // value i of the slice, its quads aligned
    each(
        [&](uint32_t i) {
            const float v = x[i];
            m = fmaxf(m, v);
            if (p.cached) keep[i] = v;
        },
        [&](uint32_t i) {
            const float4 v = *reinterpret_cast<const float4*>(x + i);
            m = fmaxf(m, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)));
            if (p.cached) *reinterpret_cast<float4*>(keep + i) = v;
        });
    m = block_reduce<true>(m, s_max);
    const float mu = m == -INFINITY ? 0.0f : m;
    float l = 0.0f;
    auto e = [&](float v) { return ex2_probs(__fmul_rn(__fsub_rn(v, mu), p.scale)); };
    each(
        [&](uint32_t i) {
            const float v = e(p.cached ? keep[i] : x[i]);
            l = __fadd_rn(l, v);
            if (p.cached) keep[i] = v;
        },
        [&](uint32_t i) {
            float4 v = *reinterpret_cast<const float4*>(p.cached ? keep + i : x + i);
            v = make_float4(e(v.x), e(v.y), e(v.z), e(v.w));
            l = __fadd_rn(l, __fadd_rn(__fadd_rn(v.x, v.y), __fadd_rn(v.z, v.w)));
            if (p.cached) *reinterpret_cast<float4*>(keep + i) = v;
        });
    l = block_reduce<false>(l, s_sum);
    float f;   // what this slice's values are multiplied by
    if (blocks > 1u) {
        if (tid == 0u) s_ml = make_float2(m, l);
        cl.sync();
        float m_all = -INFINITY, l_all = 0.0f;
        for (uint32_t r = 0; r < blocks; ++r) m_all = fmaxf(m_all, cl.map_shared_rank(&s_ml, r)->x);
        for (uint32_t r = 0; r < blocks; ++r) {
            const float2 o = *cl.map_shared_rank(&s_ml, r);
            if (o.x > -INFINITY || isnan(o.y)) l_all = fmaf(o.y, ex2_probs(__fmul_rn(__fsub_rn(o.x, m_all), p.scale)), l_all);
        }
        cl.barrier_arrive();   // no CTA leaves while another reads its pair
        f = l_all == 0.0f ? 0.0f : __fdiv_rn(m > -INFINITY ? ex2_probs(__fmul_rn(__fsub_rn(m, m_all), p.scale)) : 0.0f, l_all);
        if (isnan(l_all)) f = l_all;
    } else {
        f = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
    }
    const bool wide = ((reinterpret_cast<uintptr_t>(out + hx)) & 15u) == 0u;
    each(
        [&](uint32_t i) { out[i] = __fmul_rn(p.cached ? keep[i] : e(x[i]), f); },
        [&](uint32_t i) {
            float4 v = *reinterpret_cast<const float4*>(p.cached ? keep + i : x + i);
            if (!p.cached) v = make_float4(e(v.x), e(v.y), e(v.z), e(v.w));
            store4(out + i, make_float4(__fmul_rn(v.x, f), __fmul_rn(v.y, f), __fmul_rn(v.z, f), __fmul_rn(v.w, f)), wide);
        });
    if (blocks > 1u) cl.barrier_wait();
}

// ── verification of drafts ───────────────────────────────────────────────────
constexpr uint32_t kVerThreads = 256;   // by registers four CTAs an SM: 64 sequences are one round of clusters
constexpr uint32_t kVerWarps = kVerThreads / 32u;
constexpr uint32_t kVerMaxCluster = 8;
constexpr uint32_t kVerMaxDrafts = 256;

struct VerifyParams {
    const float* target;     // [B][K + 1] rows of vocab
    const float* draft;      // [B][K] rows of vocab
    uint64_t t_seq, t_row, d_seq, d_row;   // elements from sequence to sequence and row to row
    const int32_t* tokens;   // [B][K]
    const float* u;          // [B][K]
    const float* u_last;     // [B]
    const int32_t* counts;   // [B] drafts of each sequence (-1: skip it), or nullptr: K
    int32_t* out;            // [B][K + 1]
    int32_t* accepted;       // [B]
    uint32_t drafts, vocab, slice;   // slice: values per CTA of the cluster, a multiple of 4 * kVerWarps
};

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// Draft i stands while u_i q_i(x_i) < p_i(x_i): with probability min(1, p / q),
// without a division.  The first that falls is replaced by a draw from
// max(p - q, 0) of its row (from p where that is zero everywhere); when all stand,
// one more token is drawn from the next row of p.  A draw is the smallest token
// whose running sum of weights exceeds u_last times their total.  Products,
// differences and sums are taken in 64 bits, so that the answer does not depend on
// how the sums are split (their rounding is 2^-53).
//
// A cluster has a sequence: each CTA sums a slice of the row (each warp a part of
// the slice), the sums meet in distributed shared memory, and the CTA whose part
// holds the crossing reads that part again (from L2) to find the token.  Bound by
// reading the two rows once: measured on a B200, 64 sequences of 6 drafts over 151936
// tokens 22 us, 3.5 TB/s; one sequence 7.2 us, latency.
__global__ void __launch_bounds__(kVerThreads, 4) verify_drafts_kernel(const __grid_constant__ VerifyParams p) {
    namespace cg = cooperative_groups;
    __shared__ double s_sum[kVerWarps];   // the weights of this CTA's parts
    __shared__ double s_scan[kVerWarps], s_from, s_goal;
    __shared__ uint32_t s_fall;
    __shared__ int32_t s_found, s_last, s_pick;
    const cg::cluster_group cl = cg::this_cluster();
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, rank = cl.block_rank(), blocks = cl.num_blocks();
    const uint32_t seq = blockIdx.x / blocks, K = p.drafts;
    const int32_t given = p.counts ? p.counts[seq] : static_cast<int32_t>(K);
    if (given < 0) {   // the whole cluster
        if (given != -1 && rank == 0u && tid == 0u) raise_error(kErrBadLaunch);
        return;
    }
    const uint32_t count = min(static_cast<uint32_t>(given), K);
    if (tid == 0u) {
        s_fall = count;
        s_found = -1;
        s_last = -1;
        if (static_cast<uint32_t>(given) > K && rank == 0u) raise_error(kErrBadLaunch);
    }
    __syncthreads();
    const float* target = p.target + seq * p.t_seq;
    const float* draft = p.draft + seq * p.d_seq;
    if (tid < count) {
        const int32_t tok = p.tokens[static_cast<uint64_t>(seq) * K + tid];
        const bool in = tok >= 0 && static_cast<uint32_t>(tok) < p.vocab;
        if (!in && rank == 0u) raise_error(kErrBadLaunch);
        bool ok = false;
        if (in) {
            const double pt = target[tid * p.t_row + tok], qt = draft[tid * p.d_row + tok];
            ok = static_cast<double>(p.u[static_cast<uint64_t>(seq) * K + tid]) * qt < pt;
        }
        if (!ok) atomicMin(&s_fall, tid);
    }
    __syncthreads();
    const uint32_t at = s_fall;
    const bool all = at == count;
    const float* pr = target + at * p.t_row;
    const float* qr = all ? nullptr : draft + at * p.d_row;

    // ── sums of this warp's part ──
    const uint32_t part = p.slice / kVerWarps;   // a multiple of 4
    const uint32_t a0 = min(p.vocab, rank * p.slice + warp * part), a1 = min(p.vocab, a0 + part);
    auto weigh = [](float pv, float qv) { return pv > qv ? static_cast<double>(pv) - static_cast<double>(qv) : 0.0; };
    auto own = [](float pv) { return pv > 0.0f ? static_cast<double>(pv) : 0.0; };
    const bool wide = ((reinterpret_cast<uintptr_t>(pr) | reinterpret_cast<uintptr_t>(qr)) & 15u) == 0u;
    auto sum_part = [&](bool use_rest) {
        double sum = 0.0;
        uint32_t i = a0;
        if (wide) {
            const uint32_t quads = (a1 - a0) / 4u;
            const float4* x4 = reinterpret_cast<const float4*>(pr + a0);
            const float4* y4 = reinterpret_cast<const float4*>(qr + a0);
            if (use_rest) {
#pragma unroll 4
                for (uint32_t j = lane; j < quads; j += 32u) {
                    const float4 x = __ldg(x4 + j), y = __ldg(y4 + j);
                    sum += (weigh(x.x, y.x) + weigh(x.y, y.y)) + (weigh(x.z, y.z) + weigh(x.w, y.w));
                }
            } else {
#pragma unroll 4
                for (uint32_t j = lane; j < quads; j += 32u) {
                    const float4 x = __ldg(x4 + j);
                    sum += (own(x.x) + own(x.y)) + (own(x.z) + own(x.w));
                }
            }
            i = a0 + 4u * quads;
        }
#pragma unroll 4
        for (uint32_t j = i + lane; j < a1; j += 32u) sum += use_rest ? weigh(__ldg(pr + j), __ldg(qr + j)) : own(__ldg(pr + j));
        sum = warp_sum_f64(sum);
        if (lane == 0u) s_sum[warp] = sum;
    };

    // ── which part holds the crossing: the first warp of every CTA finds the same ──
    const uint32_t parts = blocks * kVerWarps;
    constexpr uint32_t PPL = kVerMaxCluster * kVerWarps / 32u;   // parts a lane, at most
    bool use_rest = !all;
    for (;;) {
        sum_part(use_rest);
        cl.sync();
        if (warp == 0u) {
            double mine[PPL], lane_sum = 0.0;
#pragma unroll
            for (uint32_t k = 0; k < PPL; ++k) {
                const uint32_t j = lane * PPL + k;
                mine[k] = j < parts ? cl.map_shared_rank(s_sum, j / kVerWarps)[j % kVerWarps] : 0.0;
                lane_sum += mine[k];
            }
            double run = lane_sum;   // inclusive scan of the lanes' sums
#pragma unroll
            for (uint32_t o = 1u; o < 32u; o <<= 1) {
                const double y = __shfl_up_sync(0xFFFFFFFFu, run, o);
                if (lane >= o) run += y;
            }
            double acc = __shfl_up_sync(0xFFFFFFFFu, run, 1);
            if (lane == 0u) acc = 0.0;
            const double goal = static_cast<double>(p.u_last[seq]) * __shfl_sync(0xFFFFFFFFu, run, 31);
            // the first part whose running sum exceeds the goal; without one (u_last of 1 or
            // more), the last part with any weight
            int32_t hit = -1, tail = -1;
            double hit_start = 0.0, tail_start = 0.0;
#pragma unroll
            for (uint32_t k = 0; k < PPL; ++k) {
                if (mine[k] > 0.0) {
                    tail = static_cast<int32_t>(lane * PPL + k);
                    tail_start = acc;
                    if (hit < 0 && acc + mine[k] > goal) {
                        hit = tail;
                        hit_start = acc;
                    }
                }
                acc += mine[k];
            }
            const uint32_t hits = __ballot_sync(0xFFFFFFFFu, hit >= 0), tails = __ballot_sync(0xFFFFFFFFu, tail >= 0);
            const int src = hits ? __ffs(static_cast<int>(hits)) - 1 : tails ? 31 - __clz(static_cast<int>(tails)) : 0;
            const int32_t pick = __shfl_sync(0xFFFFFFFFu, hits ? hit : tail, src);
            const double from = __shfl_sync(0xFFFFFFFFu, hits ? hit_start : tail_start, src);
            if (lane == 0u) {
                s_pick = pick;   // -1: no weight at all
                s_from = from;
                s_goal = goal;
            }
        }
        cl.sync();   // the sums have been read, the answer is there
        if (s_pick >= 0 || !use_rest) break;
        use_rest = false;   // p <= q everywhere: draw from p
    }
    if (s_pick < 0) {   // nothing can be drawn
        if (rank == 0u && tid == 0u) {
            raise_error(kErrBadLaunch);
            for (uint32_t k = 0; k <= K; ++k)
                p.out[static_cast<uint64_t>(seq) * (K + 1u) + k] =
                    k < at ? p.tokens[static_cast<uint64_t>(seq) * K + k] : -1;
            p.accepted[seq] = static_cast<int32_t>(at);
        }
        return;
    }
    const int32_t pick = s_pick;
    const double from = s_from, goal = s_goal;
    if (static_cast<uint32_t>(pick) / kVerWarps != rank) return;

    // ── the token within the part, by this CTA: a stretch of it per thread ──
    const uint32_t b0 = min(p.vocab, rank * p.slice + (static_cast<uint32_t>(pick) % kVerWarps) * part);
    const uint32_t b1 = min(p.vocab, b0 + part), per = (b1 - b0 + kVerThreads - 1u) / kVerThreads;
    const uint32_t c0 = min(b1, b0 + tid * per), c1 = min(b1, c0 + per);
    auto weight = [&](uint32_t j) {
        const float pv = __ldg(pr + j);
        return use_rest ? weigh(pv, __ldg(qr + j)) : own(pv);
    };
    double sum = 0.0;
    for (uint32_t j = c0; j < c1; ++j) sum += weight(j);
    double scan = sum;
#pragma unroll
    for (uint32_t o = 1u; o < 32u; o <<= 1) {
        const double y = __shfl_up_sync(0xFFFFFFFFu, scan, o);
        if (lane >= o) scan += y;
    }
    if (lane == 31u) s_scan[warp] = scan;
    __syncthreads();
    double base = from;
    for (uint32_t k = 0; k < warp; ++k) base += s_scan[k];
    double low = __shfl_up_sync(0xFFFFFFFFu, scan, 1);
    low = lane == 0u ? base : base + low;
    int32_t found = INT32_MAX, last = -1;
    for (uint32_t j = c0; j < c1; ++j) {
        const double w = weight(j);
        low += w;
        if (w > 0.0) {
            last = static_cast<int32_t>(j);
            if (found == INT32_MAX && low > goal) found = static_cast<int32_t>(j);
        }
    }
    // the lowest crossing of all threads, else (rounding, or u_last >= 1) the last weight
    if (tid == 0u) s_found = INT32_MAX;
    __syncthreads();
    if (found != INT32_MAX) atomicMin(&s_found, found);
    if (last >= 0) atomicMax(&s_last, last);
    __syncthreads();
    for (uint32_t k = tid; k <= K; k += kVerThreads)
        p.out[static_cast<uint64_t>(seq) * (K + 1u) + k] =
            k < at ? p.tokens[static_cast<uint64_t>(seq) * K + k]
                   : (k == at ? (s_found != INT32_MAX ? s_found : s_last) : -1);
    if (tid == 0u) p.accepted[seq] = static_cast<int32_t>(at);
}

}  // namespace qraf_dev
