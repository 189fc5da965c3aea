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
// activations are exact in one part; for bf16 the weights take one part too: their
// rounding, 2^-12 of themselves, is an eighth of the output's own.
//
// Two softmax warpgroups take the tiles in turn, each with accumulators S and O of
// its own, so that the tensor cores work on one while the other's S becomes P (in
// place: a thread owns a row, so it overwrites only what it has read).  The maximum
// that weights refer to moves only when a row exceeds it by 2^4 (then the O row is
// scaled in TMEM); weights stay below 2^15.  Four warps turn the codes into the
// MMA's shared-memory layout (K as it lies, V transposed, both K-major with the
// 128-byte swizzle), with the next tile's loads in flight.
//
// The (128 rows, KV head) units times their key tiles are dealt out evenly, one
// contiguous range a CTA and one CTA an SM; each stretch of one unit leaves a
// record per row (output, maximum, sum) for the joining kernel.
//
// Measured on a B200: the MMAs of one tile take about 8 x 80 cycles a part for S and
// 8 x 73 for O (N = 128, K = 16 each).
#pragma once

#include "common.cuh"
#include "kv_attention.cuh"
#include "matmul_tc.cuh"

namespace qraf_dev {

constexpr uint32_t kPreThreads = 416;   // two softmax warpgroups, four transform warps, one MMA warp
constexpr uint32_t kPreWarpXf = 8, kPreWarpMma = 12;
constexpr float kPreLag = 4.0f;         // log2 of how far a row may exceed the maximum it refers to
constexpr int32_t kPreUp = 11;          // weights of p = 1 are below 2^11

template <uint32_t HDP, uint32_t QP>
struct PreShape {
    static constexpr uint32_t kAtoms = HDP / 64u;                      // 64-element (128-byte) column blocks of Q and K
    static constexpr uint32_t kQPart = kPreRows * HDP * 2u;            // one part of Q
    static constexpr uint32_t kKTile = kPreKeys * HDP * 2u;            // one K or V tile in fp16
    static constexpr uint32_t kQ = 0, kK = kQ + QP * kQPart, kV = kK + 2u * kKTile, kEnd = kV + 2u * kKTile;
    static constexpr uint32_t kScales = kEnd;                          // [2][2][128] floats: K and V scales of a slot's tile
    static constexpr uint32_t kRf = kScales + 2048u;                   // [128] row factors
    static constexpr uint32_t kMl = kRf + 512u;                        // [2][2][128]: max and sum of each warpgroup's rows
    static constexpr uint32_t kBars = kMl + 2048u;
    static constexpr uint32_t kSmem = kBars + 128u + 1024u;            // + alignment of the tiles
    static constexpr uint32_t kJoinLd = HDP + 4u;                      // floats per row where the two outputs meet (over K and V)
    static_assert(kPreRows * kJoinLd * 4u <= 4u * kKTile, "the joined output must fit over the K and V tiles");
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

// 32 scores of a row starting at key `c0` of the tile -> weights.  MASK: keys from
// `valid` on are not there.
template <bool MASK>
__device__ __forceinline__ float2 pre_scaled(const float* v, uint32_t j, const float* ks, uint32_t c0, uint32_t valid) {
    float2 y = f2_mul(make_float2(v[j], v[j + 1u]), *reinterpret_cast<const float2*>(ks + c0 + j));
    if constexpr (MASK) {
        if (c0 + j >= valid) y.x = -INFINITY;
        if (c0 + j + 1u >= valid) y.y = -INFINITY;
    }
    return y;
}

// One tile's softmax for one row (thread): S at TMEM column s_col becomes P in
// place, the row's maximum and sum move on, O at o_col is scaled where the maximum
// moved.  `first`: the warpgroup's first tile of the stretch (O is written anew).
template <uint32_t HDP, uint32_t PP, bool MASK>
__device__ __forceinline__ void pre_softmax(uint32_t s_col, uint32_t o_col, const float* ks, const float* vs, uint32_t valid,
                                            float rf, bool first, float& m, float& l) {
    float v[32];
    float ymax = -INFINITY;
#pragma unroll
    for (uint32_t c = 0; c < 4u; ++c) {
        tmem_ld32(s_col + 32u * c, v);
        tmem_wait_ld();
#pragma unroll
        for (uint32_t j = 0; j < 32u; j += 2u) {
            const float2 y = pre_scaled<MASK>(v, j, ks, 32u * c, valid);
            ymax = fmaxf(ymax, fmaxf(y.x, y.y));
        }
    }
    const float mt = __fmul_rn(ymax, rf);
    float alpha = 1.0f;
    if (first) {
        m = mt > -INFINITY ? mt : 0.0f;
    } else if (mt > __fadd_rn(m, kPreLag)) {
        alpha = ex2(__fsub_rn(m, mt));
        m = mt;
    }
    if (__any_sync(0xFFFFFFFFu, alpha != 1.0f)) {
        l = __fmul_rn(l, alpha);
#pragma unroll 1
        for (uint32_t c = 0; c < HDP; c += 32u) {
            tmem_ld32(o_col + c, v);
            tmem_wait_ld();
#pragma unroll
            for (uint32_t j = 0; j < 32u; ++j) v[j] = __fmul_rn(v[j], alpha);
            tmem_st32(o_col + c, v);
        }
    }
    const float2 rf2 = make_float2(rf, rf), m2 = make_float2(-m, -m), neg = make_float2(-1.0f, -1.0f);
    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
    for (uint32_t c = 0; c < 4u; ++c) {
        tmem_ld32(s_col + 32u * c, v);
        tmem_wait_ld();
        uint32_t hi[16], lo[16];
#pragma unroll
        for (uint32_t j = 0; j < 32u; j += 2u) {
            float2 x = f2_fma(pre_scaled<false>(v, j, ks, 32u * c, valid), rf2, m2);
            if constexpr (MASK) {
                if (32u * c + j >= valid) x.x = -INFINITY;
                if (32u * c + j + 1u >= valid) x.y = -INFINITY;
            }
            const float2 p = make_float2(ex2(x.x), ex2(x.y));
            sum = f2_add(sum, p);
            const float2 w = f2_mul(p, *reinterpret_cast<const float2*>(vs + 32u * c + j));
            const __half2 h = __floats2half2_rn(w.x, w.y);
            hi[j / 2u] = *reinterpret_cast<const uint32_t*>(&h);
            if constexpr (PP == 2u) {
                const float2 d = f2_fma(__half22float2(h), neg, w);
                const __half2 r = __floats2half2_rn(d.x, d.y);
                lo[j / 2u] = *reinterpret_cast<const uint32_t*>(&r);
            }
        }
        tmem_st16(s_col + 32u * c, hi);   // the chunk's hi parts, then its lo parts
        if constexpr (PP == 2u) tmem_st16(s_col + 32u * c + 16u, lo);
    }
    l = __fadd_rn(l, __fadd_rn(sum.x, sum.y));
    tmem_wait_st();
}

template <uint32_t HDP, uint32_t QP, uint32_t PP>
__global__ void __launch_bounds__(kPreThreads, 1) kv_prefix_kernel(const __grid_constant__ KvAttnParams p) {
    using S = PreShape<HDP, QP>;
    extern __shared__ uint8_t pre_smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pre_smem_raw) + 1023u) & ~uintptr_t(1023));
    __shared__ uint32_t s_tmem, s_unit, s_fail;
    float* s_scales = reinterpret_cast<float*>(smem + S::kScales);
    float* s_rf = reinterpret_cast<float*>(smem + S::kRf);
    float* s_ml = reinterpret_cast<float*>(smem + S::kMl);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
    uint64_t *k_ready = bars, *v_ready = bars + 2, *s_ready = bars + 4, *p_ready = bars + 6, *pv_done = bars + 8, *drain = bars + 10;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t hd = p.kv.hd, H = p.kv.kv_heads, G = p.group;
    const uint32_t rows = p.runs.n * G;
    const uint64_t stride = static_cast<uint64_t>(H) * hd;

    pdl_launch_dependents();
    if (tid == 0) {
        for (uint32_t i = 0; i < 2u; ++i) {
            mbar_init(&k_ready[i], 4);
            mbar_init(&v_ready[i], 4);
            mbar_init(&s_ready[i], 1);
            mbar_init(&p_ready[i], 4);
            mbar_init(&pv_done[i], 1);
        }
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
    const uint32_t tmem = s_tmem;   // columns: S of slots 0 and 1 [0, 256), O of slots 0 and 1 [256, 512)

    const uint32_t T = (p.prefix_len + kPreKeys - 1u) / kPreKeys;
    const uint64_t work = static_cast<uint64_t>(p.row_tiles) * H * T;
    const uint64_t w1 = pre_start(work, blockIdx.x + 1u, gridDim.x);
    uint32_t used[2] = {0u, 0u};   // tiles that each slot has had, over the CTA's stretches
    bool ok = true;
    for (uint64_t w = pre_start(work, blockIdx.x, gridDim.x); w < w1;) {
        const uint32_t unit = static_cast<uint32_t>(w / T), tile0 = static_cast<uint32_t>(w - static_cast<uint64_t>(unit) * T);
        const uint32_t n = static_cast<uint32_t>(min(static_cast<uint64_t>(T - tile0), w1 - w));
        const uint32_t h = unit / p.row_tiles, row0 = (unit - h * p.row_tiles) * kPreRows;
        const uint32_t key0 = tile0 * kPreKeys, key1 = min(p.prefix_len, (tile0 + n) * kPreKeys);
        const int8_t* pk = p.pk + static_cast<uint64_t>(h) * hd;
        const int8_t* pv = p.pv + static_cast<uint64_t>(h) * hd;
        const float* pks = p.pks + h;
        const float* pvs = p.pvs + h;

        // ── the query rows (softmax warps) and the unit of the V scales (transform warps) ──
        if (tid == 0) s_unit = 0u;
        __syncthreads();
        if (warp < kPreWarpXf) {
            const float sign = p.scale_log2 < 0.0f ? -1.0f : 1.0f;
            constexpr uint32_t LPR = HDP / 4u, RPW = 32u / LPR;   // lanes per row, rows per warp access
            const uint32_t l = lane % LPR;
#pragma unroll 4
            for (uint32_t i = 0; i < 16u / RPW; ++i) {
                const uint32_t r = warp * 16u + i * RPW + lane / LPR, row = row0 + r;
                float x[4] = {0.f, 0.f, 0.f, 0.f};
                if (row < rows && 4u * l < hd) {
                    const uint32_t t = row / G;
                    const uint64_t at = static_cast<uint64_t>(t) * p.q_ld + static_cast<uint64_t>(h * G + (row - t * G)) * hd + 4u * l;
#pragma unroll
                    for (uint32_t k = 0; k < 4u; ++k) x[k] = __fmul_rn(load_any(p.q, p.type, at + k), sign);
                }
                float m = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
#pragma unroll
                for (uint32_t o = LPR / 2u; o > 0u; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
                // the largest becomes 2^10 .. 2^11, as in kva_item
                const int32_t e = max(exponent_bits(m), 11);
                const float up = pow2_bits(264 - e);
                if (l == 0u) s_rf[r] = __fmul_rn(pow2_bits(e - 10), fabsf(p.scale_log2));
                uint32_t hi[2], lo[2];
                split_f16(__fmul_rn(x[0], up), __fmul_rn(x[1], up), hi[0], lo[0]);
                split_f16(__fmul_rn(x[2], up), __fmul_rn(x[3], up), hi[1], lo[1]);
                const uint32_t off = (l >> 4) * (kPreRows * 128u) + tc_sw128_off(r, (l & 15u) >> 1) + 8u * (l & 1u);
                *reinterpret_cast<uint2*>(smem + S::kQ + off) = make_uint2(hi[0], hi[1]);
                if constexpr (QP == 2u) *reinterpret_cast<uint2*>(smem + S::kQ + S::kQPart + off) = make_uint2(lo[0], lo[1]);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        } else if (warp < kPreWarpMma) {
            uint32_t most = 0u;
            for (uint32_t key = key0 + tid - kPreWarpXf * 32u; key < key1; key += 128u) {
                const uint32_t e = static_cast<uint32_t>(exponent_bits(__ldg(pvs + static_cast<uint64_t>(key) * H)));
                if (e < 255u) most = max(most, e);
            }
            most = __reduce_max_sync(0xFFFFFFFFu, most);
            if (lane == 0u) atomicMax(&s_unit, most);
        }
        __syncthreads();
        // every V scale is below 2^(eb - 126); scaled by 2^(kPreUp + 126 - eb) they are below 2^kPreUp
        const int32_t eb = max(static_cast<int32_t>(s_unit), 14);
        float m = -INFINITY, l = 0.0f;
        const uint32_t slot = warp >> 2;   // of a softmax warp

        if (warp < kPreWarpXf) {
            // ── softmax ──
            const uint32_t lane_row = (warp & 3u) * 32u;   // TMEM lanes of this warp
            const uint32_t s_col = tmem + (lane_row << 16) + slot * 128u, o_col = tmem + (lane_row << 16) + 256u + slot * 128u;
            const float rf = s_rf[lane_row + lane];
            const float* ks = s_scales + slot * 256u;
            for (uint32_t t = slot, j = used[slot]; ok && t < n; t += 2u, ++j) {
                ok = warp_wait(&k_ready[slot], j & 1u) && warp_wait(&s_ready[slot], j & 1u);
                if (!ok) break;
                tc_fence_after();
                const uint32_t valid = key1 - (key0 + t * kPreKeys);
                if (valid >= kPreKeys) pre_softmax<HDP, PP, false>(s_col, o_col, ks, ks + 128, kPreKeys, rf, t == slot, m, l);
                else pre_softmax<HDP, PP, true>(s_col, o_col, ks, ks + 128, valid, rf, t == slot, m, l);
                tc_fence_before();
                __syncwarp();
                if (lane == 0u) mbar_arrive(&p_ready[slot]);
            }
        } else if (warp < kPreWarpMma) {
            // ── codes -> fp16 tiles ──
            const uint32_t xw = warp - kPreWarpXf, xt = tid - kPreWarpXf * 32u;
            const float vup = pow2_bits(kPreUp + 253 - eb);
            constexpr uint32_t KL = HDP / 16u;    // 16-byte loads of K a thread
            constexpr uint32_t VB = HDP / 32u;    // 32-dim blocks of V
            uint4 kr[KL];
            uint32_t vr[VB][8];
            float ksc = 0.0f, vsc = 0.0f;
            // K: lane (unit a of 16 codes, key) so that eight consecutive lanes store to
            // eight different 16-byte columns of the swizzled rows
            const uint32_t ka = lane & 3u;
            auto k_place = [&](uint32_t i, uint32_t& key, uint32_t& u) {   // key of the tile, 16-code unit of its row
                if constexpr (HDP == 128u) {
                    key = xw * 32u + i * 4u + ((lane >> 2) & 1u) + 2u * (lane >> 4);
                    u = ka + 4u * ((lane >> 3) & 1u);
                } else {
                    key = xw * 32u + i * 8u + (lane >> 2);
                    u = ka;
                }
            };
            // V: lane (4 dims, octet of keys), likewise
            const uint32_t dq = (lane & 1u) + 2u * (lane >> 3), ko = (lane >> 1) & 3u;
            auto load = [&](uint32_t t) {
                const uint32_t k0 = key0 + t * kPreKeys, last = key1 - 1u;
#pragma unroll
                for (uint32_t i = 0; i < KL; ++i) {
                    uint32_t key, u;
                    k_place(i, key, u);
                    kr[i] = 16u * u < hd ? __ldg(reinterpret_cast<const uint4*>(
                                               pk + static_cast<uint64_t>(min(k0 + key, last)) * stride + 16u * u))
                                         : make_uint4(0u, 0u, 0u, 0u);
                }
#pragma unroll
                for (uint32_t b = 0; b < VB; ++b)
#pragma unroll
                    for (uint32_t i = 0; i < 8u; ++i) {
                        const uint32_t d = 32u * b + 4u * dq;
                        vr[b][i] = d < hd ? __ldg(reinterpret_cast<const uint32_t*>(
                                                pv + static_cast<uint64_t>(min(k0 + 32u * xw + 8u * ko + i, last)) * stride + d))
                                          : 0u;
                    }
                const uint32_t key = k0 + xt;
                ksc = key < key1 ? __ldg(pks + static_cast<uint64_t>(key) * H) : 0.0f;
                vsc = key < key1 ? __fmul_rn(__ldg(pvs + static_cast<uint64_t>(key) * H), vup) : 0.0f;
            };
            load(0);
            for (uint32_t t = 0; ok && t < n; ++t) {
                const uint32_t sl = t & 1u, j = used[sl] + (t >> 1);
                // the slot's K tile, scales and V tile are free once its previous tile's
                // S is there, its P is written and its O is done
                if (j > 0u) ok = warp_wait(&s_ready[sl], (j - 1u) & 1u) && warp_wait(&p_ready[sl], (j - 1u) & 1u);
                if (!ok) break;
                uint8_t* kt = smem + S::kK + sl * S::kKTile;
#pragma unroll
                for (uint32_t i = 0; i < KL; ++i) {
                    uint32_t key, u;
                    k_place(i, key, u);
                    uint8_t* atom = kt + (u >> 2) * (kPreKeys * 128u);
                    const uint32_t a0 = kr[i].x ^ 0x80808080u, a1 = kr[i].y ^ 0x80808080u, a2 = kr[i].z ^ 0x80808080u,
                                   a3 = kr[i].w ^ 0x80808080u;
                    *reinterpret_cast<uint4*>(atom + tc_sw128_off(key, 2u * (u & 3u))) =
                        make_uint4(codes_f16<0x4140u>(a0), codes_f16<0x4342u>(a0), codes_f16<0x4140u>(a1), codes_f16<0x4342u>(a1));
                    *reinterpret_cast<uint4*>(atom + tc_sw128_off(key, 2u * (u & 3u) + 1u)) =
                        make_uint4(codes_f16<0x4140u>(a2), codes_f16<0x4342u>(a2), codes_f16<0x4140u>(a3), codes_f16<0x4342u>(a3));
                }
                s_scales[sl * 256u + xt] = ksc;
                s_scales[sl * 256u + 128u + xt] = vsc;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0u) mbar_arrive(&k_ready[sl]);
                if (j > 0u) ok = warp_wait(&pv_done[sl], (j - 1u) & 1u);
                if (!ok) break;
                // V transposed: row = dim, 64 keys per 128-byte row; eight keys are one 16-byte column
                uint8_t* vt = smem + S::kV + sl * S::kKTile + (xw >> 1) * (HDP * 128u);
                const uint32_t chunk = 4u * (xw & 1u) + ko;
#pragma unroll
                for (uint32_t b = 0; b < VB; ++b) {
                    uint32_t x[8];
#pragma unroll
                    for (uint32_t i = 0; i < 8u; ++i) x[i] = vr[b][i] ^ 0x80808080u;
                    uint32_t c01[4], c23[4];   // keys 2 i and 2 i + 1, byte-interleaved: dims 0-1 and 2-3
#pragma unroll
                    for (uint32_t i = 0; i < 4u; ++i) {
                        c01[i] = __byte_perm(x[2u * i], x[2u * i + 1u], 0x5140u);
                        c23[i] = __byte_perm(x[2u * i], x[2u * i + 1u], 0x7362u);
                    }
                    const uint32_t d = 32u * b + 4u * dq;
                    *reinterpret_cast<uint4*>(vt + tc_sw128_off(d, chunk)) =
                        make_uint4(codes_f16<0x4140u>(c01[0]), codes_f16<0x4140u>(c01[1]), codes_f16<0x4140u>(c01[2]), codes_f16<0x4140u>(c01[3]));
                    *reinterpret_cast<uint4*>(vt + tc_sw128_off(d + 1u, chunk)) =
                        make_uint4(codes_f16<0x4342u>(c01[0]), codes_f16<0x4342u>(c01[1]), codes_f16<0x4342u>(c01[2]), codes_f16<0x4342u>(c01[3]));
                    *reinterpret_cast<uint4*>(vt + tc_sw128_off(d + 2u, chunk)) =
                        make_uint4(codes_f16<0x4140u>(c23[0]), codes_f16<0x4140u>(c23[1]), codes_f16<0x4140u>(c23[2]), codes_f16<0x4140u>(c23[3]));
                    *reinterpret_cast<uint4*>(vt + tc_sw128_off(d + 3u, chunk)) =
                        make_uint4(codes_f16<0x4342u>(c23[0]), codes_f16<0x4342u>(c23[1]), codes_f16<0x4342u>(c23[2]), codes_f16<0x4342u>(c23[3]));
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0u) mbar_arrive(&v_ready[sl]);
                if (t + 1u < n) load(t + 1u);
            }
        } else {
            // ── MMA issue ──
            const uint32_t base = smem_u32(smem);
            const uint32_t idesc_s = (1u << 4) | ((kPreKeys >> 3) << 17) | ((kPreRows >> 4) << 24);
            const uint32_t idesc_o = (1u << 4) | ((HDP >> 3) << 17) | ((kPreRows >> 4) << 24);
            auto scores = [&](uint32_t t) {
                const uint32_t sl = t & 1u, j = used[sl] + (t >> 1);
                if (!warp_wait(&k_ready[sl], j & 1u)) return false;
                tc_fence_after();
                if (tc_elect_one()) {
#pragma unroll
                    for (uint32_t part = 0; part < QP; ++part)
#pragma unroll
                        for (uint32_t k = 0; k < HDP / 16u; ++k)
                            tc_mma_f16(tmem + sl * 128u,
                                       tc_smem_desc(base + S::kQ + part * S::kQPart + (k >> 2) * (kPreRows * 128u) + (k & 3u) * 32u),
                                       tc_smem_desc(base + S::kK + sl * S::kKTile + (k >> 2) * (kPreKeys * 128u) + (k & 3u) * 32u),
                                       idesc_s, part + k > 0u);
                    tc_commit(&s_ready[sl]);
                }
                __syncwarp();
                return true;
            };
            ok = scores(0);
            if (ok && n > 1u) ok = scores(1);
            for (uint32_t t = 0; ok && t < n; ++t) {
                const uint32_t sl = t & 1u, j = used[sl] + (t >> 1);
                ok = warp_wait(&p_ready[sl], j & 1u) && warp_wait(&v_ready[sl], j & 1u);
                if (!ok) break;
                tc_fence_after();
                if (tc_elect_one()) {
#pragma unroll
                    for (uint32_t part = 0; part < PP; ++part)
#pragma unroll
                        for (uint32_t k = 0; k < kPreKeys / 16u; ++k)
                            pre_mma_ts(tmem + 256u + sl * 128u, tmem + sl * 128u + 32u * (k >> 1) + 16u * part + 8u * (k & 1u),
                                       tc_smem_desc(base + S::kV + sl * S::kKTile + (k >> 2) * (HDP * 128u) + (k & 3u) * 32u), idesc_o,
                                       t >= 2u || part + k > 0u);
                    tc_commit(&pv_done[sl]);
                }
                __syncwarp();
                // the next S overwrites this P
                if (t + 2u < n) ok = warp_wait(&pv_done[sl], j & 1u) && scores(t + 2u);
            }
        }
        used[0] += (n + 1u) / 2u;
        used[1] += n / 2u;
        // ── both outputs of a row meet in shared memory (over K and V) and leave as one record ──
        if (warp < kPreWarpXf && ok && slot < n) {
            ok = warp_wait(&pv_done[slot], (used[slot] - 1u) & 1u);
            tc_fence_after();
            const uint32_t r = (warp & 3u) * 32u + lane;
            s_ml[slot * 256u + r] = m;
            s_ml[slot * 256u + 128u + r] = l;
        }
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
        const float unit_f = pow2_bits(eb - kPreUp + 1);
        const bool both = n > 1u;
        for (uint32_t turn = both ? 1u : 0u;; --turn) {   // slot 1 stores, slot 0 adds
            if (warp < kPreWarpXf && slot == turn) {
                const uint32_t r = (warp & 3u) * 32u + lane;
                const float m_all = both ? fmaxf(s_ml[r], s_ml[256u + r]) : m;
                const float f = __fmul_rn(ex2(__fsub_rn(m, m_all)), unit_f);
                const uint32_t o_col = tmem + (((warp & 3u) * 32u) << 16) + 256u + slot * 128u;
                float* dst = jo + r * S::kJoinLd;
#pragma unroll 1
                for (uint32_t c = 0; c < HDP; c += 32u) {
                    float v[32];
                    tmem_ld32(o_col + c, v);
                    tmem_wait_ld();
#pragma unroll
                    for (uint32_t k = 0; k < 32u; k += 4u) {
                        float4 y = make_float4(__fmul_rn(v[k], f), __fmul_rn(v[k + 1u], f), __fmul_rn(v[k + 2u], f),
                                               __fmul_rn(v[k + 3u], f));
                        float4* at = reinterpret_cast<float4*>(dst + c + k);
                        if (both && turn == 0u) {
                            const float4 z = *at;
                            y = make_float4(__fadd_rn(y.x, z.x), __fadd_rn(y.y, z.y), __fadd_rn(y.z, z.z), __fadd_rn(y.w, z.w));
                        }
                        *at = y;
                    }
                }
                if (turn == 0u) {
                    float l_all = l;
                    if (both)
                        l_all = __fadd_rn(__fmul_rn(l, ex2(__fsub_rn(m, m_all))),
                                          __fmul_rn(s_ml[256u + 128u + r], ex2(__fsub_rn(s_ml[256u + r], m_all))));
                    dst[HDP] = m_all;
                    dst[HDP + 1u] = l_all;
                }
            }
            tc_fence_before();
            __syncthreads();
            if (turn == 0u) break;
        }
        const uint32_t chunk = blockIdx.x - pre_owner(work, static_cast<uint64_t>(unit) * T, gridDim.x);
        for (uint32_t r = warp; r < kPreRows; r += kPreThreads / 32u) {
            const uint32_t row = row0 + r;
            if (row >= rows) break;
            const uint32_t t = row / G, head = h * G + (row - t * G);
            float* rec = p.part + ((static_cast<uint64_t>(t) * p.heads + head) * (p.p_chunks + p.splits) + chunk) * (hd + 4u);
            const float* src = jo + r * S::kJoinLd;
            if (4u * lane < hd) *reinterpret_cast<float4*>(rec + 4u * lane) = *reinterpret_cast<const float4*>(src + 4u * lane);
            if (lane == 0u) *reinterpret_cast<float2*>(rec + hd) = *reinterpret_cast<const float2*>(src + HDP);
        }
        w += n;
        if (w < w1) {
            tc_fence_after();
            __syncthreads();   // the record has been read: K and V tiles may come
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
