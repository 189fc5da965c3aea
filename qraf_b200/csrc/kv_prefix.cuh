// kv_prefix.cuh — the shared prefix's part of kv_attention (kv_attention.cuh) on
// the 5th-generation tensor cores, for batches with enough query rows to fill
// their tiles.
//
// A CTA works on 128 rows of one KV head (the MMA's M, one TMEM lane each) and a
// stretch of the prefix in tiles of 128 keys:
//     S = Q K^T  (tcgen05, Q and K in shared memory)  ->  P = weights of S
//     O += P V   (tcgen05, P in TMEM, V in shared memory)
// The codes become fp16 exactly; Q and P are split into hi + lo of two fp16, each
// part an MMA of its own into the same fp32 accumulator.  The queries of 16-bit
// activations are exact in one part.  The weights take two whatever the type: in one
// they are off by 2^-12 of themselves, which moved a tenth of the outputs of bf16 calls
// (8 sequences behind 65536 rows) to a neighbouring number.
//
// Two softmax warpgroups take the tiles in turn.  S becomes P in place (a thread owns
// a row, so it overwrites only what it has read) in one of three TMEM buffers, so
// that the scores of the tile after next are there when a warpgroup is done.  The
// maximum that a row's weights refer to passes from tile to tile through shared
// memory; it moves only when a tile exceeds it by 2^8 (then the O row is scaled in
// TMEM, after the PV before), so weights stay below 2^15 and O has one accumulator.
// Eight warps turn the codes into the MMA's shared-memory layout (K as it lies, V
// transposed, both K-major with the 128-byte swizzle), the next tiles' codes in flight
// (cp.async) behind them.
//
// The (128 rows, KV head) units times their key tiles are dealt out evenly, one
// contiguous range a CTA and one CTA an SM; each stretch of one unit leaves a
// record per row (output, maximum, sum) for the joining kernel.
//
// Measured on a B200: the MMAs of one tile take about 8 x 80 cycles a part for S and
// 8 x 73 for O (N = 128, K = 16 each), in two parts about 2400; a tile takes some 4400,
// bound by the warps that turn codes into fp16.  512 rows of 8 KV heads of 128 behind
// 8192 keys, f32, with the join: 58 us, 300 TFLOP/s of the formula's.
#pragma once

#include "common.cuh"
#include "kv_attention.cuh"
#include "matmul_tc.cuh"

namespace qraf_dev {

constexpr uint32_t kPreThreads = 544;   // two softmax warpgroups, eight transform warps, one MMA warp
constexpr uint32_t kPreWarpXf = 8, kPreWarpMma = 16, kPreXfThreads = 256;
// log2 of how far a row may exceed the maximum it refers to.  With 4 the first half dozen
// tiles still had a row to scale in nearly every warp, each waiting for the PV before; 8
// makes that rare, and still leaves a weight's lower part 2^-31 of the largest.
constexpr float kPreLag = 8.0f;
constexpr int32_t kPreUp = 7;           // weights of p = 1 are below 2^7

// Parts of the queries (16-bit ones are exact in one) and of the weights.
template <typename Q>
constexpr uint32_t pre_q_parts() { return sizeof(Q) == 4u ? 2u : 1u; }
constexpr uint32_t kPreParts = 2;

template <uint32_t HDP, uint32_t QP>
struct PreShape {
    static constexpr uint32_t kAtoms = HDP / 64u;                      // 64-element (128-byte) column blocks of Q and K
    static constexpr uint32_t kQPart = kPreRows * HDP * 2u;            // one part of Q
    static constexpr uint32_t kKTile = kPreKeys * HDP * 2u;            // one K or V tile in fp16
    static constexpr uint32_t kRaw = kPreKeys * HDP;                   // one K or V tile in codes
    static constexpr uint32_t kQ = 0, kK = kQ + QP * kQPart, kV = kK + kKTile;      // one K tile, two V tiles
    static constexpr uint32_t kRawK = kV + 2u * kKTile, kRawV = kRawK + kRaw, kEnd = kRawV + 2u * kRaw;
    static constexpr uint32_t kScales = kEnd;                          // [3][2][128] floats: K and V scales of a buffer's tile
    static constexpr uint32_t kRf = kScales + 3u * 1024u;              // [128] row factors
    static constexpr uint32_t kM = kRf + 512u;                         // [2][128] the maxima referred to, after a tile
    static constexpr uint32_t kMl = kM + 1024u;                        // [2][2][128]: each warpgroup's sums and their maxima
    static constexpr uint32_t kBars = kMl + 2048u;
    static constexpr uint32_t kSmem = kBars + 256u + 1024u;            // + alignment of the tiles
    static constexpr uint32_t kJoinLd = HDP + 4u;                      // floats per row where the two outputs meet (over K and V)
    static_assert(kPreRows * kJoinLd * 4u <= 3u * kKTile, "the joined output must fit over the K and V tiles");
};

__device__ __forceinline__ void pre_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&v)[32]) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const float (&v)[32]) {
    const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

// warp_wait for two barriers at once: with both phases complete, as they mostly are, one
// vote instead of two.
__device__ __forceinline__ bool warp_wait2(uint64_t* a, uint32_t pa, uint64_t* b, uint32_t pb) {
    const bool fa = mbar_try_wait(a, pa), fb = mbar_try_wait(b, pb);
    if (__all_sync(0xFFFFFFFFu, fa && fb)) return true;
    return warp_wait(a, pa) && warp_wait(b, pb);
}

// A row's (thread's) largest scaled score of a tile: S at TMEM column s_col, ks the K
// scales.  MASK: keys from `valid` on are not there.  The loops here and below stay
// rolled: five kinds of code share the instruction caches, and unrolled (1500
// instructions a tile) fetching them took a quarter of the issue slots' waits.
template <bool MASK>
__device__ __forceinline__ float pre_max(uint32_t s_col, const float* ks, uint32_t valid) {
    float ymax = -INFINITY;
#pragma unroll 1
    for (uint32_t c = 0; c < 4u; ++c) {
        float v[32];
        tmem_ld32(s_col + 32u * c, v);
        tmem_wait_ld();
#pragma unroll
        for (uint32_t j = 0; j < 32u; j += 4u) {
            const float4 k4 = *reinterpret_cast<const float4*>(ks + 32u * c + j);
            float2 y = f2_mul(make_float2(v[j], v[j + 1u]), make_float2(k4.x, k4.y));
            float2 z = f2_mul(make_float2(v[j + 2u], v[j + 3u]), make_float2(k4.z, k4.w));
            if constexpr (MASK) {
                if (32u * c + j >= valid) y.x = -INFINITY;
                if (32u * c + j + 1u >= valid) y.y = -INFINITY;
                if (32u * c + j + 2u >= valid) z.x = -INFINITY;
                if (32u * c + j + 3u >= valid) z.y = -INFINITY;
            }
            ymax = fmaxf(fmaxf(ymax, fmaxf(y.x, y.y)), fmaxf(z.x, z.y));
        }
    }
    return ymax;
}

// The row's weights, relative to the maximum m, in the place of its scores (the hi
// parts of 32 keys, then their lo parts); returns the sum of exp(s - m).
template <bool MASK>
__device__ __forceinline__ float pre_weights(uint32_t s_col, const float* ks, const float* vs, uint32_t valid, float rf, float m) {
    const float2 rf2 = make_float2(rf, rf), m2 = make_float2(-m, -m), neg = make_float2(-1.0f, -1.0f);
    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll 1
    for (uint32_t c = 0; c < 4u; ++c) {
        float v[32];
        tmem_ld32(s_col + 32u * c, v);
        tmem_wait_ld();
        uint32_t hi[16], lo[16];
#pragma unroll
        for (uint32_t j = 0; j < 32u; j += 4u) {
            const float4 k4 = *reinterpret_cast<const float4*>(ks + 32u * c + j);
            const float4 v4 = *reinterpret_cast<const float4*>(vs + 32u * c + j);
#pragma unroll
            for (uint32_t i = 0; i < 4u; i += 2u) {
                const float2 kk = i ? make_float2(k4.z, k4.w) : make_float2(k4.x, k4.y);
                const float2 vv = i ? make_float2(v4.z, v4.w) : make_float2(v4.x, v4.y);
                float2 x = f2_fma(f2_mul(make_float2(v[j + i], v[j + i + 1u]), kk), rf2, m2);
                if constexpr (MASK) {
                    if (32u * c + j + i >= valid) x.x = -INFINITY;
                    if (32u * c + j + i + 1u >= valid) x.y = -INFINITY;
                }
                const float2 p = make_float2(ex2(x.x), ex2(x.y));
                sum = f2_add(sum, p);
                const float2 w = f2_mul(p, vv);
                const __half2 h = __floats2half2_rn(w.x, w.y);
                hi[(j + i) / 2u] = *reinterpret_cast<const uint32_t*>(&h);
                const float2 d = f2_fma(__half22float2(h), neg, w);
                const __half2 r = __floats2half2_rn(d.x, d.y);
                lo[(j + i) / 2u] = *reinterpret_cast<const uint32_t*>(&r);
            }
        }
        tmem_st16(s_col + 32u * c, hi);
        tmem_st16(s_col + 32u * c + 16u, lo);
    }
    tmem_wait_st();
    return __fadd_rn(sum.x, sum.y);
}

// The tensor cores' fp32 accumulator truncates: every accumulation may lose a last bit, and
// always toward zero (measured on a B200: evenly weighted keys lose 1.0e-7 of the sum a tile
// and part, 8 accumulations).  So the lower parts' products go first (into small sums), and O
// starts anew every kPreTerm tiles: its sum so far is added, rounded to nearest, to the CTA's
// own sums (p.pre_sum), which stay in L2.  512 rows of 8 KV heads behind 8192 keys (16 tiles a
// CTA), off the 64-bit answer and time of the kernels: 4 tiles 1.1e-6, 64 us; 8 tiles 1.8e-6,
// 59 us; 16 tiles 3.4e-6, 59 us.  Plain fp32 is off by 1.8e-6.

// o times alpha plus v times unit (a power of two).
__device__ __forceinline__ float4 pre_add4(float4 o, float alpha, const float* v, float unit) {
    return make_float4(fmaf(o.x, alpha, __fmul_rn(v[0], unit)), fmaf(o.y, alpha, __fmul_rn(v[1], unit)),
                       fmaf(o.z, alpha, __fmul_rn(v[2], unit)), fmaf(o.w, alpha, __fmul_rn(v[3], unit)));
}

// Where a CTA's sums have columns c .. c + 4 of row r: a warp's rows next to each other.
__device__ __forceinline__ float4* pre_sum_at(float4* sums, uint32_t c, uint32_t r) { return sums + (c / 4u) * kPreRows + r; }

// The row's output so far, in numbers, added to its sums times alpha (FIRST: to nothing).
template <uint32_t HDP, bool FIRST>
__device__ __forceinline__ void pre_add_row(uint32_t o_col, float4* sums, uint32_t r, uint32_t hd, float unit, float alpha) {
#pragma unroll 1
    for (uint32_t c = 0; c < HDP; c += 32u) {
        float v[32];
        tmem_ld32(o_col + c, v);
        tmem_wait_ld();
        float4 old[8];
#pragma unroll
        for (uint32_t j = 0; j < 8u; ++j)
            old[j] = FIRST || c + 4u * j >= hd ? make_float4(0.f, 0.f, 0.f, 0.f) : __ldcg(pre_sum_at(sums, c + 4u * j, r));
#pragma unroll
        for (uint32_t j = 0; j < 8u; ++j)
            if (c + 4u * j < hd) __stcg(pre_sum_at(sums, c + 4u * j, r), pre_add4(old[j], alpha, v + 4u * j, unit));
    }
}

// The row's output so far times alpha.
template <uint32_t HDP>
__device__ __forceinline__ void pre_scale_row(uint32_t o_col, float alpha) {
#pragma unroll 1
    for (uint32_t c = 0; c < HDP; c += 32u) {
        float v[32];
        tmem_ld32(o_col + c, v);
        tmem_wait_ld();
#pragma unroll
        for (uint32_t j = 0; j < 32u; j += 2u) {
            const float2 y = f2_mul(make_float2(v[j], v[j + 1u]), make_float2(alpha, alpha));
            v[j] = y.x;
            v[j + 1u] = y.y;
        }
        tmem_st32(o_col + c, v);
    }
    tmem_wait_st();
}

// One row of n floats (a multiple of 4, both ends 16-byte aligned) from shared to
// global memory, in the executing thread's bulk group.
__device__ __forceinline__ void bulk_s2g(float* dst, const float* src, uint32_t n) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(src)), "r"(4u * n) : "memory");
}

// Q: the type of q and out.
template <uint32_t HDP, typename Q>
__global__ void __launch_bounds__(kPreThreads, 1) kv_prefix_kernel(const __grid_constant__ KvAttnParams p) {
    constexpr uint32_t QP = pre_q_parts<Q>();
    using S = PreShape<HDP, QP>;
    extern __shared__ uint8_t pre_smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pre_smem_raw) + 1023u) & ~uintptr_t(1023));
    __shared__ uint32_t s_tmem, s_fail, s_unit[8];
    float* s_scales = reinterpret_cast<float*>(smem + S::kScales);
    float* s_rf = reinterpret_cast<float*>(smem + S::kRf);
    float* s_ml = reinterpret_cast<float*>(smem + S::kMl);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
    float* s_m = reinterpret_cast<float*>(smem + S::kM);
    // by S buffer (three): the K tile and the scales are there, S is, P is; by tile parity:
    // the V tile is there, O has it, a warp's rows have their maxima; by stretch: the query
    // rows are there, O has all of its tiles
    uint64_t *k_ready = bars, *s_ready = bars + 3, *p_ready = bars + 6, *v_ready = bars + 9, *pv_done = bars + 11,
             *m_ready = bars + 13 /* [2][4] */, *q_ready = bars + 21, *o_ready = bars + 22, *drain = bars + 23;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t hd = p.kv.hd, H = p.kv.kv_heads, G = p.group;
    const uint32_t rows = p.runs.n * G;
    const uint64_t stride = static_cast<uint64_t>(H) * hd;

    pdl_launch_dependents();
    if (tid == 0) {
        for (uint32_t i = 0; i < 3u; ++i) {
            mbar_init(&k_ready[i], 4);
            mbar_init(&s_ready[i], 1);
            mbar_init(&p_ready[i], 4);
        }
        for (uint32_t i = 0; i < 2u; ++i) {
            mbar_init(&v_ready[i], 4);
            mbar_init(&pv_done[i], 1);
            for (uint32_t j = 0; j < 4u; ++j) mbar_init(&m_ready[4u * i + j], 1);
        }
        mbar_init(q_ready, 8);
        mbar_init(o_ready, 1);
        mbar_init(drain, 1);
        fence_mbar_init();
        s_fail = 0u;
    }
    if (warp == kPreWarpMma) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;   // columns: the S buffers [0, 384), O [384, 384 + HDP)

    const uint32_t T = (p.prefix_len + kPreKeys - 1u) / kPreKeys;
    const uint32_t w1 = pre_start(p.pre_base, p.pre_extra, blockIdx.x + 1u);
    uint32_t x0 = 0u;   // tiles of the CTA's stretches before this one: tile t is the CTA's tile x0 + t
    uint32_t q_phase = 0u;
    bool ok = true;
    float4* sums = reinterpret_cast<float4*>(p.pre_sum) + static_cast<uint64_t>(blockIdx.x) * (kPreRows * HDP / 4u);
    for (uint32_t w = pre_start(p.pre_base, p.pre_extra, blockIdx.x); w < w1;) {
        const uint32_t unit = w / T, tile0 = w - unit * T, n = min(T - tile0, w1 - w);
        const uint32_t h = unit / p.row_tiles, row0 = (unit - h * p.row_tiles) * kPreRows;
        const uint32_t key0 = tile0 * kPreKeys, key1 = min(p.prefix_len, (tile0 + n) * kPreKeys);
        float m = -INFINITY, l = 0.0f;       // of a softmax thread: its sum, and the maximum that it refers to
        const uint32_t wg = warp >> 2;       // softmax warpgroup: tiles of this parity (of the stretch)
        float m_sum = -INFINITY;             // and of its row's sums of earlier terms
        const uint32_t rec_at = blockIdx.x - pre_owner(p.pre_base, p.pre_extra, unit * T);
        auto record = [&](uint32_t r) -> float* {   // of the tile's row r; nullptr past the last row
            const uint32_t row = row0 + r, t = row / G, head = h * G + (row - t * G);
            return row < rows ? p.part + ((static_cast<uint64_t>(t) * p.heads + head) * (p.p_chunks + p.splits) + rec_at) * (hd + 4u)
                              : nullptr;
        };
        auto unit_factor = [&]() {   // O to numbers
            uint32_t most = 14u;
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) most = max(most, s_unit[i]);
            return pow2_bits(static_cast<int32_t>(most) - kPreUp + 1);
        };
        auto rescale = [](float from, float to) { return from == to ? 1.0f : ex2(__fsub_rn(from, to)); };   // from <= to, -inf too

        if (warp < kPreWarpXf) {
            // ── the query rows: 16 a warp, all of its loads in flight ──
            {
                constexpr uint32_t LPR = HDP / 4u, RPA = 32u / LPR, A = 16u / RPA;   // lanes a row, rows an access, accesses
                const uint32_t ql = lane % LPR, r0 = warp * 16u + lane / LPR;
                auto src = [&](uint32_t i) {
                    const uint32_t row = row0 + r0 + i * RPA, t = row / G;
                    return static_cast<const Q*>(p.q) + static_cast<uint64_t>(t) * p.q_ld +
                           static_cast<uint64_t>(h * G + (row - t * G)) * hd + 4u * ql;
                };
                auto in = [&](uint32_t i) { return row0 + r0 + i * RPA < rows && 4u * ql < hd; };
                float4 x[A];
                if (p.q_wide) {
#pragma unroll
                    for (uint32_t i = 0; i < A; ++i) x[i] = in(i) ? load4(src(i), true) : make_float4(0.f, 0.f, 0.f, 0.f);
                } else {
#pragma unroll
                    for (uint32_t i = 0; i < A; ++i) x[i] = in(i) ? load4(src(i), false) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
                const float sign = p.scale_log2 < 0.0f ? -1.0f : 1.0f;
#pragma unroll
                for (uint32_t i = 0; i < A; ++i) {
                    const uint32_t r = r0 + i * RPA;
                    float mx = absmax4(x[i], 0.0f);
#pragma unroll
                    for (uint32_t o = LPR / 2u; o > 0u; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
                    // the largest becomes 2^10 .. 2^11, as in kva_item
                    const int32_t e = max(exponent_bits(mx), 11);
                    const float up = __fmul_rn(pow2_bits(264 - e), sign);
                    if (ql == 0u) s_rf[r] = __fmul_rn(pow2_bits(e - 10), fabsf(p.scale_log2));
                    uint32_t hi[2], lo[2];
                    split_f16(__fmul_rn(x[i].x, up), __fmul_rn(x[i].y, up), hi[0], lo[0]);
                    split_f16(__fmul_rn(x[i].z, up), __fmul_rn(x[i].w, up), hi[1], lo[1]);
                    const uint32_t off = (ql >> 4) * (kPreRows * 128u) + tc_sw128_off(r, (ql & 15u) >> 1) + 8u * (ql & 1u);
                    *reinterpret_cast<uint2*>(smem + S::kQ + off) = make_uint2(hi[0], hi[1]);
                    if constexpr (QP == 2u) *reinterpret_cast<uint2*>(smem + S::kQ + S::kQPart + off) = make_uint2(lo[0], lo[1]);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0u) mbar_arrive(q_ready);
            asm volatile("bar.sync 2, 256;" ::: "memory");   // the row factors, across warps

            // ── softmax ──
            const uint32_t lane_row = (warp & 3u) * 32u, r = lane_row + lane;   // TMEM lanes of this warp; this thread's row
            const uint32_t o_col = tmem + (lane_row << 16) + 384u;
            const float rf = s_rf[r];
            for (uint32_t t = wg; ok && t < n; t += 2u) {
                const uint32_t x = x0 + t, b = x % 3u, ph = x / 3u & 1u;
                const uint32_t s_col = tmem + (lane_row << 16) + 128u * b;
                const float* ks = s_scales + b * 256u;
                ok = warp_wait2(&k_ready[b], ph, &s_ready[b], ph);
                if (!ok) break;
                tc_fence_after();
                const uint32_t valid = key1 - (key0 + t * kPreKeys);
                const float ymax = valid >= kPreKeys ? pre_max<false>(s_col, ks, kPreKeys) : pre_max<true>(s_col, ks, valid);
                const float mt = __fmul_rn(ymax, rf);
                // the maximum that the row refers to from this tile on (-inf while every score was)
                float m_now = mt > -INFINITY ? mt : -INFINITY, alpha = 1.0f, before = -INFINITY;
                if (t > 0u) {
                    const uint32_t px = x - 1u;
                    ok = warp_wait(&m_ready[4u * (px & 1u) + (warp & 3u)], px >> 1 & 1u);
                    if (!ok) break;
                    before = s_m[(px & 1u) * 128u + r];
                    // never a lower one: the sum of weights runs on over the stretch's terms, and one
                    // scaled up by 2^128 would overflow
                    if (t % kPreTerm == 0u) {   // O starts anew
                        m_now = fmaxf(before, mt);
                    } else if (mt > __fadd_rn(before, kPreLag)) {
                        alpha = ex2(__fsub_rn(before, mt));
                    } else {
                        m_now = before;
                    }
                }
                s_m[(x & 1u) * 128u + r] = m_now;
                __syncwarp();
                if (lane == 0u) mbar_arrive(&m_ready[4u * (x & 1u) + (warp & 3u)]);
                if (__any_sync(0xFFFFFFFFu, alpha != 1.0f)) {   // O has the term's tiles before this one, and no other yet
                    ok = warp_wait(&pv_done[(x - 1u) & 1u], (x - 1u) >> 1 & 1u);
                    if (!ok) break;
                    tc_fence_after();
                    pre_scale_row<HDP>(o_col, alpha);
                }
                if (m_now != m) l = __fmul_rn(l, ex2(__fsub_rn(m, m_now)));
                m = m_now;
                const float m_use = m > -INFINITY ? m : 0.0f;   // nothing seen yet: every weight 2^-inf = 0
                l = __fadd_rn(l, valid >= kPreKeys ? pre_weights<false>(s_col, ks, ks + 128, kPreKeys, rf, m_use)
                                                   : pre_weights<true>(s_col, ks, ks + 128, valid, rf, m_use));
                if (t > 0u && t % kPreTerm == 0u) {   // the term before leaves O
                    ok = warp_wait(&pv_done[(x - 1u) & 1u], (x - 1u) >> 1 & 1u);
                    if (!ok) break;
                    tc_fence_after();
                    if (t == kPreTerm) pre_add_row<HDP, true>(o_col, sums, r, hd, unit_factor(), 0.0f);
                    else pre_add_row<HDP, false>(o_col, sums, r, hd, unit_factor(), rescale(m_sum, before));
                    m_sum = before;
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0u) mbar_arrive(&p_ready[b]);
            }
        } else if (warp < kPreWarpMma) {
            // ── codes -> fp16 tiles ──
            // The MMAs run ... PV(t) S(t+3) PV(t+1) S(t+4) ...: K(t+3) is made while PV(t) runs
            // and V(t+2) from then on, so K has one fp16 tile and V two, behind one and two
            // tiles of codes in flight (cp.async).  Four warps make K, four V.
            const uint32_t xw = warp & 3u, xt = tid & 127u;
            const bool for_k = warp < kPreWarpXf + 4u;
            constexpr uint32_t U = HDP / 16u;            // 16-byte units of a row
            constexpr uint32_t KL = kPreKeys * U / 128u; // units of a tile a thread
            constexpr uint32_t VB = HDP / 32u;           // 32-dim blocks of V
            const int8_t* src_codes = (for_k ? p.pk : p.pv) + static_cast<uint64_t>(h) * hd;
            const uint32_t last = key1 - 1u;
            // K: lane (unit of 16 codes, key), so that eight consecutive lanes load from and
            // store to eight different 16-byte columns; a thread loads what it converts.
            // Access i is key k_key + KI i of the tile, at raw offset k_src + i KI HDP.
            constexpr uint32_t KI = 32u / U;   // keys per access
            const uint32_t k_kk = HDP == 128u ? ((lane >> 2) & 1u) + 2u * (lane >> 4) : lane >> 2;
            const uint32_t k_u = HDP == 128u ? (lane & 3u) + 4u * ((lane >> 3) & 1u) : lane & 3u;
            const uint32_t k_key = xw * 32u + k_kk;
            const uint32_t k_src = k_key * HDP + 16u * (HDP == 128u ? k_u ^ (4u * (k_kk & 1u)) : k_u);
            // fp16 row of key 32 xw + i KI + k_kk: 8-row atom 4 xw + (i KI) / 8, row (i KI & 7) + k_kk
            const uint32_t k_dst = (k_u >> 2) * (kPreKeys * 128u) + xw * 4096u + k_kk * 128u;
            const uint32_t k_col = (2u * (k_u & 3u)) ^ k_kk;   // its 16-byte column, ^ (i KI & 7), ^ 1 for the second eight codes
            const bool k_in = 16u * k_u < hd;
            // V: unit u of key k lies at unit u ^ 2 (k / 8) so that a lane's four-byte reads of
            // four octets of keys meet four groups of banks
            const uint32_t vf_u = xt % U, vf_key = xt / U;   // fetch: unit, first key; keys 128 / U apart
            const bool vf_in = 16u * vf_u < hd;
            // conversion: lane (4 dims dq, octet of keys ko) of 32 keys x 32 dims
            const uint32_t dq = (lane & 1u) + 2u * (lane >> 3), ko = (lane >> 1) & 3u;
            const uint32_t v_src = (32u * xw + 8u * ko) * HDP + 4u * dq;   // + i HDP + 32 (block ^ ko)
            // transposed row 32 block + 4 dq + j, 64 keys per 128-byte row: 16-byte column = octet of keys
            const uint32_t v_dst = (xw >> 1) * (HDP * 128u) + (dq >> 1) * 1024u + (dq & 1u) * 512u;
            const uint32_t v_col = (4u * (xw & 1u) + ko) ^ (4u * (dq & 1u));   // ^ j
            auto fetch_k = [&](uint32_t t) {
                if (t < n && k_in) {
                    uint8_t* dst = smem + S::kRawK + k_src;
                    const uint32_t k0 = key0 + t * kPreKeys + k_key;
#pragma unroll 2
                    for (uint32_t i = 0; i < KL; ++i)
                        cp_async16(dst + i * KI * HDP, src_codes + static_cast<uint64_t>(min(k0 + i * KI, last)) * stride + 16u * k_u);
                }
                cp_async_commit();
            };
            auto fetch_v = [&](uint32_t t) {
                if (t < n && vf_in) {
                    uint8_t* dst = smem + S::kRawV + (t & 1u) * S::kRaw;
                    const uint32_t k0 = key0 + t * kPreKeys;
#pragma unroll 2
                    for (uint32_t i = 0; i < KL; ++i) {
                        const uint32_t key = vf_key + i * (128u / U);
                        cp_async16(dst + key * HDP + 16u * (vf_u ^ (2u * ((key >> 3) & (U / 2u - 1u)))),
                                   src_codes + static_cast<uint64_t>(min(k0 + key, last)) * stride + 16u * vf_u);
                    }
                }
                cp_async_commit();
            };
            // a barrier of V's warps that tells whether all of them are fine, so that they
            // give up together when a wait runs out
            auto all_v = [](bool fine) {
                uint32_t r;
                asm volatile(
                    "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
                    "bar.red.and.pred q, 3, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                    : "=r"(r)
                    : "r"(fine ? 1u : 0u)
                    : "memory");
                return r != 0u;
            };
            // the unit of the weights: every V scale of the stretch is below 2^(eb - 126)
            // (an infinity or NaN has no say); before the tiles' copies, which would hold its loads up
            uint32_t most = 0u;
            for (uint32_t key = key0 + tid - kPreWarpXf * 32u; key < key1; key += 4u * kPreXfThreads) {
                float v[4];
#pragma unroll
                for (uint32_t i = 0; i < 4u; ++i)
                    v[i] = __ldg(p.pvs + h + static_cast<uint64_t>(min(key + i * kPreXfThreads, last)) * H);
#pragma unroll
                for (uint32_t i = 0; i < 4u; ++i) {
                    const uint32_t e = static_cast<uint32_t>(exponent_bits(v[i]));
                    if (e < 255u) most = max(most, e);
                }
            }
            if (for_k) {   // a group a tile, even past the last
                fetch_k(0);
            } else {
                fetch_v(0);
                fetch_v(1);
            }
            most = __reduce_max_sync(0xFFFFFFFFu, most);
            if (lane == 0u) s_unit[warp - kPreWarpXf] = most;
            asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) most = max(most, s_unit[i]);
            const float up = pow2_bits(kPreUp + 253 - max(static_cast<int32_t>(most), 14));
            float ksc = 0.0f, vsc = 0.0f;   // the scales of key xt of the next K tile
            auto fetch_scale = [&](uint32_t t) {
                const uint32_t key = key0 + t * kPreKeys + xt;
                const bool in = t < n && key < key1;
                ksc = in ? __ldg(p.pks + h + static_cast<uint64_t>(key) * H) : 0.0f;
                vsc = in ? __ldg(p.pvs + h + static_cast<uint64_t>(key) * H) : 0.0f;
            };
            auto make_k = [&](uint32_t t) {
                const uint32_t x = x0 + t, b = x % 3u;
                cp_async_wait<0>();
                const uint8_t* raw = smem + S::kRawK + k_src;
                // the K tile is free once the previous tile's S is there, and the buffer's
                // scales once its previous P is written
                if (x > 0u && !warp_wait(&s_ready[(x - 1u) % 3u], (x - 1u) / 3u & 1u)) return false;
                if (x > 2u && !warp_wait(&p_ready[b], (x / 3u - 1u) & 1u)) return false;
                uint8_t* dst = smem + S::kK + k_dst;
#pragma unroll 2
                for (uint32_t i = 0; i < KL; ++i) {
                    const uint4 c = k_in ? *reinterpret_cast<const uint4*>(raw + i * KI * HDP) : make_uint4(0u, 0u, 0u, 0u);
                    uint8_t* row = dst + (i * KI >> 3) * 1024u + (i * KI & 7u) * 128u;
                    const uint32_t col = k_col ^ (i * KI & 7u);
                    const uint32_t a0 = c.x ^ 0x80808080u, a1 = c.y ^ 0x80808080u, a2 = c.z ^ 0x80808080u, a3 = c.w ^ 0x80808080u;
                    *reinterpret_cast<uint4*>(row + (col << 4)) =
                        make_uint4(codes_f16<0x4140u>(a0), codes_f16<0x4342u>(a0), codes_f16<0x4140u>(a1), codes_f16<0x4342u>(a1));
                    *reinterpret_cast<uint4*>(row + ((col ^ 1u) << 4)) =
                        make_uint4(codes_f16<0x4140u>(a2), codes_f16<0x4342u>(a2), codes_f16<0x4140u>(a3), codes_f16<0x4342u>(a3));
                }
                s_scales[b * 256u + xt] = ksc;
                s_scales[b * 256u + 128u + xt] = __fmul_rn(vsc, up);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0u) mbar_arrive(&k_ready[b]);
                fetch_k(t + 1u);
                fetch_scale(t + 1u);
                return true;
            };
            auto make_v = [&](uint32_t t, bool fine) {
                const uint32_t x = x0 + t, sl = x & 1u;
                cp_async_wait<1>();
                if (!all_v(fine)) return false;   // the other threads' pieces have come too
                const uint8_t* raw = smem + S::kRawV + (t & 1u) * S::kRaw + v_src;
                // the V tile is free once the O of the tile before the previous one is done
                if (x > 1u) fine = warp_wait(&pv_done[sl], (x / 2u - 1u) & 1u);
#pragma unroll 1
                for (uint32_t b = 0; b < VB; ++b) {
                    if (!fine) break;
                    const bool in = 32u * b + 4u * dq < hd;
                    const uint8_t* src = raw + 32u * (b ^ (ko & (U / 2u - 1u)));
                    uint32_t x[8];
#pragma unroll
                    for (uint32_t i = 0; i < 8u; ++i) x[i] = in ? *reinterpret_cast<const uint32_t*>(src + i * HDP) ^ 0x80808080u : 0x80808080u;
                    uint8_t* dst = smem + S::kV + sl * S::kKTile + v_dst + b * 4096u;
                    uint32_t c01[4], c23[4];   // keys 2 i and 2 i + 1, byte-interleaved: dims 0-1 and 2-3
#pragma unroll
                    for (uint32_t i = 0; i < 4u; ++i) {
                        c01[i] = __byte_perm(x[2u * i], x[2u * i + 1u], 0x5140u);
                        c23[i] = __byte_perm(x[2u * i], x[2u * i + 1u], 0x7362u);
                    }
                    *reinterpret_cast<uint4*>(dst + (v_col << 4)) =
                        make_uint4(codes_f16<0x4140u>(c01[0]), codes_f16<0x4140u>(c01[1]), codes_f16<0x4140u>(c01[2]), codes_f16<0x4140u>(c01[3]));
                    *reinterpret_cast<uint4*>(dst + 128u + ((v_col ^ 1u) << 4)) =
                        make_uint4(codes_f16<0x4342u>(c01[0]), codes_f16<0x4342u>(c01[1]), codes_f16<0x4342u>(c01[2]), codes_f16<0x4342u>(c01[3]));
                    *reinterpret_cast<uint4*>(dst + 256u + ((v_col ^ 2u) << 4)) =
                        make_uint4(codes_f16<0x4140u>(c23[0]), codes_f16<0x4140u>(c23[1]), codes_f16<0x4140u>(c23[2]), codes_f16<0x4140u>(c23[3]));
                    *reinterpret_cast<uint4*>(dst + 384u + ((v_col ^ 3u) << 4)) =
                        make_uint4(codes_f16<0x4342u>(c23[0]), codes_f16<0x4342u>(c23[1]), codes_f16<0x4342u>(c23[2]), codes_f16<0x4342u>(c23[3]));
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0u && fine) mbar_arrive(&v_ready[sl]);
                if (!all_v(fine)) return false;   // every piece of the stage has been read
                fetch_v(t + 2u);
                return true;
            };
            if (for_k) {
                fetch_scale(0);
                for (uint32_t t = 0; ok && t < n; ++t) ok = make_k(t);
            } else {
                for (uint32_t t = 0; ok && t < n; ++t) ok = make_v(t, ok);
            }
            cp_async_wait<0>();
        } else {
            // ── MMA issue ──
            const uint32_t base = smem_u32(smem);
            const uint32_t idesc_s = (1u << 4) | ((kPreKeys >> 3) << 17) | ((kPreRows >> 4) << 24);
            const uint32_t idesc_o = (1u << 4) | ((HDP >> 3) << 17) | ((kPreRows >> 4) << 24);
            // S of tile t into buffer x % 3, once `other` (with its parity) is complete too
            auto scores = [&](uint32_t t, uint64_t* other, uint32_t parity) {
                const uint32_t x = x0 + t, b = x % 3u;
                if (!warp_wait2(&k_ready[b], x / 3u & 1u, other, parity)) return false;
                tc_fence_after();
                if (tc_elect_one()) {
#pragma unroll 1
                    for (uint32_t part = 0; part < QP; ++part)
#pragma unroll 4
                        for (uint32_t k = 0; k < HDP / 16u; ++k)
                            tc_mma_f16(tmem + b * 128u,
                                       tc_smem_desc(base + S::kQ + (QP - 1u - part) * S::kQPart + (k >> 2) * (kPreRows * 128u) + (k & 3u) * 32u),
                                       tc_smem_desc(base + S::kK + (k >> 2) * (kPreKeys * 128u) + (k & 3u) * 32u),
                                       idesc_s, part + k > 0u);
                    tc_commit(&s_ready[b]);
                }
                __syncwarp();
                return true;
            };
            for (uint32_t t = 0; ok && t < 3u && t < n; ++t) ok = scores(t, q_ready, q_phase);
            for (uint32_t t = 0; ok && t < n; ++t) {
                const uint32_t x = x0 + t, b = x % 3u, sl = x & 1u;
                ok = warp_wait2(&p_ready[b], x / 3u & 1u, &v_ready[sl], x >> 1 & 1u);
                if (!ok) break;
                tc_fence_after();
                if (tc_elect_one()) {
#pragma unroll 1
                    for (uint32_t part = 0; part < kPreParts; ++part)
#pragma unroll 4
                        for (uint32_t k = 0; k < kPreKeys / 16u; ++k)
                            pre_mma_ts(tmem + 384u, tmem + b * 128u + 32u * (k >> 1) + 16u * (kPreParts - 1u - part) + 8u * (k & 1u),
                                       tc_smem_desc(base + S::kV + sl * S::kKTile + (k >> 2) * (HDP * 128u) + (k & 3u) * 32u), idesc_o,
                                       t % kPreTerm + part + k > 0u);
                    tc_commit(&pv_done[sl]);
                    if (t + 1u == n) tc_commit(o_ready);
                }
                __syncwarp();
                // the next S of this buffer overwrites the P that has just been used
                if (t + 3u < n) ok = scores(t + 3u, &pv_done[sl], x >> 1 & 1u);
            }
        }
        x0 += n;
        // ── the rows leave as records, by way of shared memory (over K and V) ──
        if (warp < kPreWarpXf && ok) {
            // not pv_done of the last tile: a warp here knows only that the tile three before its own
            // last is in O, so that one's parity may be that of the tile two before the last
            ok = warp_wait(o_ready, q_phase);
            tc_fence_after();
            const uint32_t r = (warp & 3u) * 32u + lane;
            s_ml[wg * 256u + r] = m;   // -inf and 0 where the warpgroup had no tile
            s_ml[wg * 256u + 128u + r] = l;
            if (wg == 0u) s_m[(x0 & 1u) * 128u + r] = m_sum;   // the slot of the tile before the last: that has been read
        }
        q_phase ^= 1u;
        if (!ok) s_fail = 1u;
        __syncthreads();
        if (s_fail) {   // a wait ran out (the status is raised): let the MMAs in flight end, then leave
            if (warp == kPreWarpMma) {
                if (tc_elect_one()) tc_commit(drain);
                __syncwarp();
                warp_wait(drain, 0u);
            }
            break;
        }
        float* jo = reinterpret_cast<float*>(smem + S::kK);   // [128][HDP + 4]
        if (warp < kPreWarpXf) {   // each warpgroup has half of the columns
            const uint32_t r = (warp & 3u) * 32u + lane;
            const float unit_f = unit_factor();
            const float m_end = s_m[((x0 - 1u) & 1u) * 128u + r], alpha = rescale(s_m[(x0 & 1u) * 128u + r], m_end);
            const uint32_t o_col = tmem + (((warp & 3u) * 32u) << 16) + 384u;
            float* dst = jo + r * S::kJoinLd;
#pragma unroll 1
            for (uint32_t c = wg * (HDP / 2u); c < (wg + 1u) * (HDP / 2u); c += 32u) {
                float v[32];
                tmem_ld32(o_col + c, v);
                tmem_wait_ld();
                float4 old[8];
#pragma unroll
                for (uint32_t k = 0; k < 8u; ++k)
                    old[k] = n > kPreTerm && c + 4u * k < hd ? __ldcg(pre_sum_at(sums, c + 4u * k, r)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (uint32_t k = 0; k < 8u; ++k)
                    if (c + 4u * k < hd) *reinterpret_cast<float4*>(dst + c + 4u * k) = pre_add4(old[k], alpha, v + 4u * k, unit_f);
            }
            if (wg == 0u) {
                float sum = 0.0f;
#pragma unroll
                for (uint32_t i = 0; i < 2u; ++i) {
                    sum = fmaf(s_ml[i * 256u + 128u + r], rescale(s_ml[i * 256u + r], m_end), sum);
                }
                *reinterpret_cast<float4*>(dst + hd) = make_float4(m_end, sum, 0.0f, 0.0f);
            }
            tc_fence_before();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the copies below read what was written here
        }
        __syncthreads();
        if (warp < 4u) {   // one bulk copy a row
            if (float* rec = record(tid)) bulk_s2g(rec, jo + tid * S::kJoinLd, hd + 4u);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");   // written: K and V tiles may come, the CTA may end
        }
        w += n;
        if (w < w1) {
            tc_fence_after();
            __syncthreads();   // the records have left: K and V tiles may come
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kPreWarpMma) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

}  // namespace qraf_dev
