// kv_attention.cuh — attention over the int8 KV cache for a batch whose sequences
// may share a prefix (qraf_cuda_kv_attention).
//
// For a query row q (one head of one new token), over the prefix's rows and the
// visible rows of the sequence's own slot,
//     s_t = scale * ks_t * <q, kc_t>,   p_t = exp(s_t - max s),
//     out = sum_t p_t vs_t vc_t / sum_t p_t
// with int8 codes kc, vc and fp32 scales ks, vs per (row, KV head).  Token i of a
// run of n new tokens sees the slot's rows below len - n + 1 + i.  A row that sees
// nothing gets zeros.
//
// Arithmetic.  The codes are integers that fp16 holds exactly, so the products run
// on the tensor cores at fp32 accuracy by splitting only the other operand: a
// query row is scaled by a power of two and written as hi + lo of two fp16 (22
// bits), and each weight p_t vs_t likewise, relative to the largest vs met.  The
// four products accumulate in fp32; maxima, sums and the running output are fp32.
//
// Work.  The rows of a work item (up to 16 of one KV head) meet one chunk of keys:
// a chunk of the prefix, with rows of any sequences, so the prefix is read once
// for every 16 rows; or a chunk of one sequence's own rows.  The four warps of a
// CTA take steps of 32 keys in turn and keep maximum, sum and output of their
// own; they are joined in shared memory, and the chunks of a row by a second
// kernel (in a fixed order: results do not depend on timing).  A call with one
// chunk a row writes its output at once.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"
#include "kv_cache.cuh"

namespace qraf_dev {

constexpr uint32_t kKvaThreads = 128;
constexpr uint32_t kKvaWarps = kKvaThreads / 32u;
constexpr uint32_t kKvaMinChunk = 128;      // keys per chunk, at least: one step of each warp
constexpr uint32_t kKvaMaxHeadDim = 256;
constexpr uint32_t kKvaMaxChunks = 512;     // chunks of one row, prefix and own rows together

constexpr uint32_t kPreRows = 128;          // kv_prefix.cuh: query rows of a tile = MMA M
constexpr uint32_t kPreKeys = 128;          // and keys of a tile

// kv_prefix_kernel's (unit, key tile) pairs, unit-major, are dealt out in contiguous
// ranges of `base` pairs a CTA, one more for the first `extra`: the first pair of CTA c,
__host__ __device__ __forceinline__ uint32_t pre_start(uint32_t base, uint32_t extra, uint32_t c) {
    return c * base + (c < extra ? c : extra);
}
// and the CTA that has pair x.
__host__ __device__ __forceinline__ uint32_t pre_owner(uint32_t base, uint32_t extra, uint32_t x) {
    const uint32_t split = extra * (base + 1u);
    return x < split ? x / (base + 1u) : extra + (x - split) / base;
}

struct KvAttnParams {
    KvView kv;
    KvRuns runs;             // firsts = visible rows of each slot
    const int8_t* pk;        // the prefix: row 0, head 0 of its slot
    const int8_t* pv;
    const float* pks;
    const float* pvs;
    uint32_t prefix_len;
    const void* q;           // [n][heads * hd], rows q_ld elements apart
    void* out;               // [n][heads * hd], rows out_ld elements apart
    uint64_t q_ld, out_ld;
    uint32_t type, wide;     // element type of q and out; every four elements of out aligned for one store
    uint32_t q_wide;         // and of q for one load
    uint32_t group, heads;   // query heads per KV head; all query heads
    float scale_log2;        // scale * log2(e)
    uint32_t max_len;        // the longest visible length allowed
    uint32_t row_tiles;      // prefix: tiles of 16 rows (pre_ctas: of 128) of a KV head
    uint32_t p_chunks, p_chunk;   // its chunks (pre_ctas: records of a row at most) and keys in one
    uint32_t pre_ctas;       // CTAs of kv_prefix_kernel, which has the prefix then; 0: kv_attention_kernel has it
    uint32_t pre_base, pre_extra;   // its ranges
    uint32_t chained;        // kv_attention_kernel was launched as kv_prefix_kernel's dependent
    uint32_t own_tiles, splits;              // own rows: row tiles over all runs (at most), chunks of each (at most)
    uint32_t own_wide;       // own rows in tiles of 16 rows, else 8
    float* part;             // [n * heads][p_chunks + splits][hd + 4]: output, max (log2), sum; nullptr: one chunk a row
};

// (a chunk's keys, how many) of `len` own rows in at most `splits` chunks.
__device__ __forceinline__ uint32_t own_chunk(uint32_t len, uint32_t splits, uint32_t* count) {
    if (len == 0u) {
        *count = 0u;
        return 32u;
    }
    const uint32_t s0 = min(splits, (len + kKvaMinChunk - 1u) / kKvaMinChunk);
    const uint32_t chunk = ((len + s0 - 1u) / s0 + 31u) & ~31u;
    *count = (len + chunk - 1u) / chunk;
    return chunk;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two codes (bytes SEL of w, already with the sign bit flipped: code + 128) as
// fp16: 0x6400 | u is 1024 + u, and subtracting 1152 leaves the code, exactly.
template <uint32_t SEL>
__device__ __forceinline__ uint32_t codes_f16(uint32_t w) {
    const uint32_t h = __byte_perm(w, 0x64646464u, SEL);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ float ex2(float x) {   // 2^x, within 2 ulp; 0 at -inf
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float load_any(const void* p, uint32_t type, uint64_t i) {
    if (type == QRAF_TYPE_F32) return static_cast<const float*>(p)[i];
    if (type == QRAF_TYPE_F16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ float4 load4_any(const void* p, uint32_t type, uint64_t i, bool wide) {
    if (type == QRAF_TYPE_F32) return load4(static_cast<const float*>(p) + i, wide);
    if (type == QRAF_TYPE_F16) return load4(static_cast<const __half*>(p) + i, wide);
    return load4(static_cast<const __nv_bfloat16*>(p) + i, wide);
}
__device__ __forceinline__ void store4_any(void* p, uint32_t type, uint64_t i, float4 x, bool wide) {
    if (type == QRAF_TYPE_F32) store4(static_cast<float*>(p) + i, x, wide);
    else if (type == QRAF_TYPE_F16) store4(static_cast<__half*>(p) + i, x, wide);
    else store4(static_cast<__nv_bfloat16*>(p) + i, x, wide);
}

// hi + lo of two values as packed fp16 pairs.
__device__ __forceinline__ void split_f16(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(__fsub_rn(a, f.x), __fsub_rn(b, f.y));
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

__device__ __forceinline__ float pow2_bits(int32_t biased) {   // 2^(biased - 127), 0 below the normal range
    return biased > 0 ? __int_as_float(min(biased, 254) << 23) : 0.0f;
}
__device__ __forceinline__ int32_t exponent_bits(float x) { return static_cast<int32_t>(__float_as_uint(x) >> 23) & 0xFF; }

// What one CTA works on.
struct KvaItem {
    const int8_t* k;      // key 0 of this KV head
    const int8_t* v;
    const float* ks;
    const float* vs;
    uint64_t stride;      // elements from key to key
    uint32_t sstride;     // scales from key to key
    uint32_t key0, key1;  // the chunk
    uint32_t row0, rows;  // rows [row0, rows) of the group; row r is token t0 + r / group, head h * group + r % group
    int32_t t0;
    uint32_t h;
    int32_t seen0;        // keys that row 0's token sees (grows by one a token); INT_MAX: all of the chunk
    uint32_t chunk;       // index of the chunk in the row's partials
};

// A run's slot and visible length; false (and the status raised for all but
// padding runs) when they are out of range.
__device__ __forceinline__ bool run_ok(const KvAttnParams& p, uint32_t b, uint32_t* slot, uint32_t* len) {
    const int32_t s = p.runs.slots[b], m = p.runs.firsts[b];
    if (s == -1) return false;
    if (s < 0 || static_cast<uint32_t>(s) >= p.kv.slots || m < 0 || static_cast<uint32_t>(m) > p.max_len) {
        if ((threadIdx.x & 31u) == 0u) raise_error(kErrBadLaunch);
        return false;
    }
    *slot = static_cast<uint32_t>(s);
    *len = static_cast<uint32_t>(m);
    return true;
}

template <uint32_t HDP, bool WIDE>
struct KvaShape {
    static constexpr uint32_t kKeys = HDP == 256u ? 16u : 32u;   // keys a step (registers)
    static constexpr uint32_t kTiles = kKeys / 8u;               // 8-key score tiles
    static constexpr uint32_t kSteps = HDP / 16u;                // 16-element steps of the score product
    static constexpr uint32_t kWords = HDP / 32u;                // 4-code words a thread reads of one V row
    static constexpr uint32_t kOut = HDP / 8u;                   // 8-column output tiles
    static constexpr uint32_t kRows = WIDE ? 16u : 8u;
    static constexpr uint32_t kQBytes = kSteps * 32u * 16u * (WIDE ? 2u : 1u);
    static constexpr uint32_t kJoinBytes = kKvaWarps * kRows * (HDP + 4u) * 4u;
    static constexpr uint32_t kSmem = kQBytes > kJoinBytes ? kQBytes : kJoinBytes;
};

// One work item.  WIDE: 16 rows, hi and lo parts as two products into one
// accumulator; else 8 rows, the tensor-core tile's rows 0-7 their hi parts and
// rows 8-15 their lo parts, whose two results meet in one thread.
//
// Lane (g = lane / 4, c = lane % 4).  The codes' order in the products is free as
// long as both operands agree, and is chosen so that every fragment comes from wide
// loads without going through shared memory: of a K row a lane reads 16 bytes
// (dims 64 j + 16 c ..), each of its four words one step's fragment; of V it reads
// its columns (16 g ..) of the four keys that its score accumulators belong to, and
// pairs their bytes.
template <uint32_t HDP, bool WIDE>
__device__ __forceinline__ void kva_item(const KvAttnParams& p, const KvaItem& it, uint8_t* smem, float* s_rf) {
    using S = KvaShape<HDP, WIDE>;
    constexpr uint32_t R = S::kRows, RT = WIDE ? 2u : 1u;   // RT: score rows of a thread
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, g = lane >> 2, c = lane & 3u;
    const uint32_t hd = p.kv.hd, G = p.group;
    const uint32_t nrows = min(R, it.rows - it.row0);

    // ── the query rows: powers of two, then the fragments in shared memory ──
    auto q_at = [&](uint32_t r) {
        const uint32_t row = it.row0 + r, i = row / G;
        return static_cast<uint64_t>(it.t0 + static_cast<int32_t>(i)) * p.q_ld +
               static_cast<uint64_t>(it.h * G + (row - i * G)) * hd;
    };
    for (uint32_t r = warp; r < R; r += kKvaWarps) {
        float m = 0.0f;
        if (r < nrows) {
            const uint64_t at = q_at(r);
            for (uint32_t d = lane; d < hd; d += 32u) m = fmaxf(m, fabsf(__fmul_rn(load_any(p.q, p.type, at + d), p.scale_log2)));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        // the largest becomes 2^10 .. 2^11: hi up to 2048, lo's last bit 2^-24
        if (lane == 0) s_rf[r] = pow2_bits(max(exponent_bits(m), 11) - 10);
    }
    __syncthreads();
    for (uint32_t j = tid; j < S::kSteps * 32u; j += kKvaThreads) {
        const uint32_t l = j & 31u, st = j >> 5;
        const uint32_t d = 64u * (st >> 2) + 16u * (l & 3u) + 4u * (st & 3u);
        uint32_t hi[2][2] = {}, lo[2][2] = {};
#pragma unroll
        for (uint32_t e = 0; e < RT; ++e) {
            const uint32_t r = (l >> 2) + 8u * e;
            if (r < nrows && d < hd) {
                const uint64_t at = q_at(r) + d;
                const float up = pow2_bits(254 - exponent_bits(s_rf[r]));
                float x[4];
#pragma unroll
                for (uint32_t k = 0; k < 4u; ++k)
                    x[k] = __fmul_rn(__fmul_rn(load_any(p.q, p.type, at + k), p.scale_log2), up);
                split_f16(x[0], x[1], hi[e][0], lo[e][0]);
                split_f16(x[2], x[3], hi[e][1], lo[e][1]);
            }
        }
        uint4* dst = reinterpret_cast<uint4*>(smem);
        if constexpr (WIDE) {
            dst[j] = make_uint4(hi[0][0], hi[1][0], hi[0][1], hi[1][1]);
            dst[S::kSteps * 32u + j] = make_uint4(lo[0][0], lo[1][0], lo[0][1], lo[1][1]);
        } else {
            dst[j] = make_uint4(hi[0][0], lo[0][0], hi[0][1], lo[0][1]);
        }
    }
    __syncthreads();

    float rf[RT];
    int32_t seen[RT];
#pragma unroll
    for (uint32_t e = 0; e < RT; ++e) {
        const uint32_t r = g + 8u * e, row = it.row0 + r;
        rf[e] = s_rf[r];
        seen[e] = it.seen0 == INT32_MAX ? INT32_MAX : it.seen0 + static_cast<int32_t>(row / G);
        if (r >= nrows) seen[e] = 0;
    }
    float o[S::kOut][4];
#pragma unroll
    for (uint32_t i = 0; i < S::kOut; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    float run_m[RT], run_l[RT];
#pragma unroll
    for (uint32_t e = 0; e < RT; ++e) {
        run_m[e] = -INFINITY;
        run_l[e] = 0.0f;
    }
    int32_t vref[RT];   // the output's unit is 2^(vref - 140), every V scale seen is below 2^(vref - 126)
#pragma unroll
    for (uint32_t e = 0; e < RT; ++e) vref[e] = 14;

    uint4 kr[S::kTiles][HDP / 64u];
    float sk = 0.0f, sv = 0.0f;   // K and V scale of key (lane) of the step
    const uint32_t last = it.key1 - 1u;
    auto load_k = [&](uint32_t k0) {
#pragma unroll
        for (uint32_t t = 0; t < S::kTiles; ++t) {
            const int8_t* row = it.k + static_cast<uint64_t>(min(k0 + 8u * t + g, last)) * it.stride;
#pragma unroll
            for (uint32_t j = 0; j < HDP / 64u; ++j)
                kr[t][j] = 64u * j + 16u * c < hd ? __ldg(reinterpret_cast<const uint4*>(row + 64u * j + 16u * c))
                                                  : make_uint4(0u, 0u, 0u, 0u);
        }
        const uint32_t key = k0 + lane;
        const bool in = lane < S::kKeys && key < it.key1;
        sk = in ? __ldg(it.ks + static_cast<uint64_t>(key) * it.sstride) : 0.0f;
        sv = in ? __ldg(it.vs + static_cast<uint64_t>(key) * it.sstride) : 0.0f;
    };
    const uint32_t step = S::kKeys * kKvaWarps;
    uint32_t k0 = it.key0 + warp * S::kKeys;
    if (k0 < it.key1) load_k(k0);
    for (; k0 < it.key1; k0 += step) {
        // V of this step: in flight through the score product and the softmax
        uint32_t vw[S::kKeys / 16u][4][S::kWords];
#pragma unroll
        for (uint32_t u = 0; u < S::kKeys / 16u; ++u) {
#pragma unroll
            for (uint32_t r = 0; r < 4u; ++r) {
                const uint32_t key = min(k0 + 16u * u + 2u * c + (r & 1u) + 8u * (r >> 1), last);
                const int8_t* row = it.v + static_cast<uint64_t>(key) * it.stride;
                if constexpr (HDP == 64u) {
                    const uint2 w = 8u * g < hd ? __ldg(reinterpret_cast<const uint2*>(row + 8u * g)) : make_uint2(0u, 0u);
                    vw[u][r][0] = w.x;
                    vw[u][r][1] = w.y;
                } else {
#pragma unroll
                    for (uint32_t h = 0; h < HDP / 128u; ++h) {
                        const uint4 w = 128u * h + 16u * g < hd
                                            ? __ldg(reinterpret_cast<const uint4*>(row + 128u * h + 16u * g))
                                            : make_uint4(0u, 0u, 0u, 0u);
                        vw[u][r][4u * h] = w.x;
                        vw[u][r][4u * h + 1u] = w.y;
                        vw[u][r][4u * h + 2u] = w.z;
                        vw[u][r][4u * h + 3u] = w.w;
                    }
                }
            }
        }
        // ── scores ──
        float s[S::kTiles][4];
#pragma unroll
        for (uint32_t t = 0; t < S::kTiles; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.0f;
#pragma unroll
        for (uint32_t st = 0; st < S::kSteps; ++st) {
            const uint4 qa = reinterpret_cast<const uint4*>(smem)[st * 32u + lane];
            const uint32_t a[4] = {qa.x, qa.y, qa.z, qa.w};
            uint32_t al[4];
            if constexpr (WIDE) {
                const uint4 ql = reinterpret_cast<const uint4*>(smem)[(S::kSteps + st) * 32u + lane];
                al[0] = ql.x;
                al[1] = ql.y;
                al[2] = ql.z;
                al[3] = ql.w;
            }
#pragma unroll
            for (uint32_t t = 0; t < S::kTiles; ++t) {
                const uint4 kk = kr[t][st >> 2];
                const uint32_t w = ((st & 3u) == 0u ? kk.x : (st & 3u) == 1u ? kk.y : (st & 3u) == 2u ? kk.z : kk.w) ^ 0x80808080u;
                const uint32_t b0 = codes_f16<0x4140u>(w), b1 = codes_f16<0x4342u>(w);
                mma_f16(s[t], a, b0, b1);
                if constexpr (WIDE) mma_f16(s[t], al, b0, b1);
            }
        }
        const float sk_now = sk, sv_now = sv;
        const uint32_t k_now = k0;
        if (k0 + step < it.key1) load_k(k0 + step);   // in flight through the rest of this step

        // ── softmax ──
        float x[RT][2u * S::kTiles], vsc[2u * S::kTiles];
        float mt[RT];
        int32_t ev[RT];   // the largest exponent of the V scales that the row sees (not of an infinity or NaN)
#pragma unroll
        for (uint32_t e = 0; e < RT; ++e) {
            mt[e] = -INFINITY;
            ev[e] = 0;
        }
#pragma unroll
        for (uint32_t t = 0; t < S::kTiles; ++t) {
#pragma unroll
            for (uint32_t b = 0; b < 2u; ++b) {
                const uint32_t in = 8u * t + 2u * c + b, key = k_now + in;
                const float ks = __shfl_sync(0xFFFFFFFFu, sk_now, in);
                vsc[2u * t + b] = __shfl_sync(0xFFFFFFFFu, sv_now, in);
                const int32_t eb = exponent_bits(vsc[2u * t + b]);
#pragma unroll
                for (uint32_t e = 0; e < RT; ++e) {
                    const float dot = WIDE ? s[t][2u * e + b] : __fadd_rn(s[t][b], s[t][2u + b]);
                    const bool on = key < it.key1 && static_cast<int64_t>(key) < static_cast<int64_t>(seen[e]);
                    const float v = on ? __fmul_rn(dot, __fmul_rn(ks, rf[e])) : -INFINITY;
                    x[e][2u * t + b] = v;
                    mt[e] = fmaxf(mt[e], v);
                    if (on && eb < 255) ev[e] = max(ev[e], eb);
                }
            }
        }
        float alpha[RT], down[RT], m_use[RT], vup[RT];
        bool moved = false;
#pragma unroll
        for (uint32_t e = 0; e < RT; ++e) {
            mt[e] = fmaxf(mt[e], __shfl_xor_sync(0xFFFFFFFFu, mt[e], 1));
            mt[e] = fmaxf(mt[e], __shfl_xor_sync(0xFFFFFFFFu, mt[e], 2));
            ev[e] = max(ev[e], __shfl_xor_sync(0xFFFFFFFFu, ev[e], 1));
            ev[e] = max(ev[e], __shfl_xor_sync(0xFFFFFFFFu, ev[e], 2));
            const float m_new = fmaxf(run_m[e], mt[e]);
            alpha[e] = m_new == run_m[e] ? 1.0f : ex2(__fsub_rn(run_m[e], m_new));   // 0 at the first keys
            run_m[e] = m_new;
            m_use[e] = m_new == -INFINITY ? 0.0f : m_new;   // nothing seen yet: every weight exp(-inf) = 0
            run_l[e] = __fmul_rn(run_l[e], alpha[e]);
            const int32_t vnew = max(vref[e], ev[e]);
            down[e] = __fmul_rn(alpha[e], pow2_bits(127 + vref[e] - vnew));
            vref[e] = vnew;
            vup[e] = pow2_bits(267 - vnew);   // 2^14 over the unit: weights below 2^14
            moved |= down[e] != 1.0f;
        }
        if (__any_sync(0xFFFFFFFFu, moved)) {
#pragma unroll
            for (uint32_t i = 0; i < S::kOut; ++i) {
                o[i][0] = __fmul_rn(o[i][0], down[0]);
                o[i][1] = __fmul_rn(o[i][1], down[0]);
                o[i][2] = __fmul_rn(o[i][2], down[RT - 1u]);
                o[i][3] = __fmul_rn(o[i][3], down[RT - 1u]);
            }
        }
        uint32_t ph[RT][S::kTiles], pl[RT][S::kTiles];
#pragma unroll
        for (uint32_t t = 0; t < S::kTiles; ++t) {
#pragma unroll
            for (uint32_t e = 0; e < RT; ++e) {
                const float p0 = ex2(__fsub_rn(x[e][2u * t], m_use[e])), p1 = ex2(__fsub_rn(x[e][2u * t + 1u], m_use[e]));
                run_l[e] = __fadd_rn(run_l[e], __fadd_rn(p0, p1));
                // a key that this row does not see has weight 0 whatever its scale
                const float w0 = x[e][2u * t] == -INFINITY ? 0.0f : __fmul_rn(p0, __fmul_rn(vsc[2u * t], vup[e]));
                const float w1 = x[e][2u * t + 1u] == -INFINITY ? 0.0f : __fmul_rn(p1, __fmul_rn(vsc[2u * t + 1u], vup[e]));
                split_f16(w0, w1, ph[e][t], pl[e][t]);
            }
        }
        // ── weighted sum of V ──
#pragma unroll
        for (uint32_t u = 0; u < S::kKeys / 16u; ++u) {
            uint32_t a[4], al[4];
            if constexpr (WIDE) {
                a[0] = ph[0][2u * u];
                a[1] = ph[1][2u * u];
                a[2] = ph[0][2u * u + 1u];
                a[3] = ph[1][2u * u + 1u];
                al[0] = pl[0][2u * u];
                al[1] = pl[1][2u * u];
                al[2] = pl[0][2u * u + 1u];
                al[3] = pl[1][2u * u + 1u];
            } else {
                a[0] = ph[0][2u * u];
                a[1] = pl[0][2u * u];
                a[2] = ph[0][2u * u + 1u];
                a[3] = pl[0][2u * u + 1u];
            }
#pragma unroll
            for (uint32_t w = 0; w < S::kWords; ++w) {
                const uint32_t v0 = vw[u][0][w] ^ 0x80808080u, v1 = vw[u][1][w] ^ 0x80808080u;
                const uint32_t v2 = vw[u][2][w] ^ 0x80808080u, v3 = vw[u][3][w] ^ 0x80808080u;
                const uint32_t a01 = __byte_perm(v0, v1, 0x5140u), a23 = __byte_perm(v0, v1, 0x7362u);
                const uint32_t b01 = __byte_perm(v2, v3, 0x5140u), b23 = __byte_perm(v2, v3, 0x7362u);
                const uint32_t b[4][2] = {{codes_f16<0x4140u>(a01), codes_f16<0x4140u>(b01)},
                                          {codes_f16<0x4342u>(a01), codes_f16<0x4342u>(b01)},
                                          {codes_f16<0x4140u>(a23), codes_f16<0x4140u>(b23)},
                                          {codes_f16<0x4342u>(a23), codes_f16<0x4342u>(b23)}};
#pragma unroll
                for (uint32_t j = 0; j < 4u; ++j) {
                    mma_f16(o[4u * w + j], a, b[j][0], b[j][1]);
                    if constexpr (WIDE) mma_f16(o[4u * w + j], al, b[j][0], b[j][1]);
                }
            }
        }
    }

    // ── join the warps ──
#pragma unroll
    for (uint32_t e = 0; e < RT; ++e) {
        run_l[e] = __fadd_rn(run_l[e], __shfl_xor_sync(0xFFFFFFFFu, run_l[e], 1));
        run_l[e] = __fadd_rn(run_l[e], __shfl_xor_sync(0xFFFFFFFFu, run_l[e], 2));
    }
    __syncthreads();   // the query fragments have been read
    float* jo = reinterpret_cast<float*>(smem);   // [warp][row][HDP + 4]: output, max, sum
    constexpr uint32_t LD = HDP + 4u;
#pragma unroll
    for (uint32_t e = 0; e < RT; ++e) {
        float* row = jo + (warp * R + g + 8u * e) * LD;
        const float unit = pow2_bits(vref[e] - 13);
#pragma unroll
        for (uint32_t b = 0; b < 2u; ++b) {
            const uint32_t n = 2u * c + b;   // column within an output tile
#pragma unroll
            for (uint32_t w = 0; w < S::kWords; ++w) {
                const uint32_t d = HDP == 64u ? 8u * n + 4u * w : 128u * (w >> 2) + 16u * n + 4u * (w & 3u);
                float y[4];
#pragma unroll
                for (uint32_t j = 0; j < 4u; ++j) {
                    const float* a = o[4u * w + j];
                    y[j] = __fmul_rn(WIDE ? a[2u * e + b] : __fadd_rn(a[b], a[2u + b]), unit);
                }
                *reinterpret_cast<float4*>(row + d) = make_float4(y[0], y[1], y[2], y[3]);
            }
        }
        if (c == 0u) {
            row[HDP] = run_m[e];
            row[HDP + 1u] = run_l[e];
        }
    }
    __syncthreads();
    for (uint32_t r = warp; r < nrows; r += kKvaWarps) {
        const uint32_t row = it.row0 + r, i = row / G, head = it.h * G + (row - i * G);
        const int32_t t = it.t0 + static_cast<int32_t>(i);
        float m = -INFINITY, l = 0.0f, f[kKvaWarps];
#pragma unroll
        for (uint32_t w = 0; w < kKvaWarps; ++w) m = fmaxf(m, jo[(w * R + r) * LD + HDP]);
#pragma unroll
        for (uint32_t w = 0; w < kKvaWarps; ++w) {
            const float mw = jo[(w * R + r) * LD + HDP];
            f[w] = mw == -INFINITY ? 0.0f : ex2(__fsub_rn(mw, m));
            l = fmaf(f[w], jo[(w * R + r) * LD + HDP + 1u], l);
        }
        float* rec = p.part ? p.part + ((static_cast<uint64_t>(t) * p.heads + head) * (p.p_chunks + p.splits) + it.chunk) *
                                           (hd + 4u)
                            : nullptr;
        bool live = true;
        if (!rec) {   // the only chunk: this is the row's output, unless its run is padding
            const int32_t b = find_run(p.runs, t);
            uint32_t slot, len;
            live = b >= 0 && run_ok(p, static_cast<uint32_t>(b), &slot, &len);
        }
        const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
        for (uint32_t d = 4u * lane; d < hd; d += 128u) {
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (uint32_t w = 0; w < kKvaWarps; ++w) {
                if (f[w] == 0.0f) continue;
                const float4 a = *reinterpret_cast<const float4*>(jo + (w * R + r) * LD + d);
                y.x = fmaf(f[w], a.x, y.x);
                y.y = fmaf(f[w], a.y, y.y);
                y.z = fmaf(f[w], a.z, y.z);
                y.w = fmaf(f[w], a.w, y.w);
            }
            if (rec) {
                *reinterpret_cast<float4*>(rec + d) = y;
            } else if (live) {
                store4_any(p.out, p.type, static_cast<uint64_t>(t) * p.out_ld + static_cast<uint64_t>(head) * hd + d,
                           make_float4(__fmul_rn(y.x, inv), __fmul_rn(y.y, inv), __fmul_rn(y.z, inv), __fmul_rn(y.w, inv)),
                           p.wide);
            }
        }
        if (rec && lane == 0u) {
            rec[hd] = m;
            rec[hd + 1u] = l;
        }
    }
}

// Run and row tile of own-row tile `idx`: runs in order, ceil(rows / R) tiles each.
__device__ __forceinline__ bool find_tile(const KvAttnParams& p, uint32_t idx, uint32_t R, uint32_t* b, uint32_t* tile) {
    const KvRuns& r = p.runs;
    if (!r.cu) {
        const uint32_t per = (p.group + R - 1u) / R;
        *b = idx / per;
        *tile = idx - *b * per;
        return *b < r.count;
    }
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t before = 0;
    for (uint32_t i0 = 0; i0 < r.count; i0 += 32u) {
        const uint32_t i = i0 + lane;
        uint32_t mine = 0;
        if (i < r.count) {
            const int32_t n = min(r.cu[i + 1u], static_cast<int32_t>(r.n)) - max(r.cu[i], 0);
            if (n > 0) mine = (static_cast<uint32_t>(n) * p.group + R - 1u) / R;
        }
        uint32_t sum = mine;
#pragma unroll
        for (uint32_t o = 1u; o < 32u; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, sum, o);
            if (lane >= o) sum += y;
        }
        const uint32_t hit = __ballot_sync(0xFFFFFFFFu, idx >= before + sum - mine && idx < before + sum);
        if (hit) {
            const uint32_t l = static_cast<uint32_t>(__ffs(static_cast<int>(hit)) - 1);
            *b = i0 + l;
            *tile = idx - (before + __shfl_sync(0xFFFFFFFFu, sum - mine, l));
            return true;
        }
        before += __shfl_sync(0xFFFFFFFFu, sum, 31);
    }
    return false;
}

template <uint32_t HDP>
__device__ __forceinline__ void kva_cta(const KvAttnParams& p, uint8_t* kva_smem, float* s_rf) {
    const uint32_t H = p.kv.kv_heads;
    KvaItem it;
    it.sstride = H;
    it.stride = static_cast<uint64_t>(H) * p.kv.hd;
    uint32_t idx = blockIdx.x;
    const uint32_t p_items = p.pre_ctas ? 0u : p.row_tiles * H * p.p_chunks;
    if (idx < p_items) {
        const uint32_t q = idx / p.row_tiles, rt = idx - q * p.row_tiles;
        it.chunk = q / H;
        it.h = q - it.chunk * H;
        it.key0 = it.chunk * p.p_chunk;
        it.key1 = min(p.prefix_len, it.key0 + p.p_chunk);
        it.k = p.pk + static_cast<uint64_t>(it.h) * p.kv.hd;
        it.v = p.pv + static_cast<uint64_t>(it.h) * p.kv.hd;
        it.ks = p.pks + it.h;
        it.vs = p.pvs + it.h;
        it.row0 = rt * 16u;
        it.rows = p.runs.n * p.group;
        it.t0 = 0;
        it.seen0 = INT32_MAX;
        kva_item<HDP, true>(p, it, kva_smem, s_rf);
        return;
    }
    idx -= p_items;
    const uint32_t R = p.own_wide ? 16u : 8u;
    const uint32_t q = idx / p.splits, s = idx - q * p.splits;
    const uint32_t tile_idx = q / H;
    it.h = q - tile_idx * H;
    uint32_t b, tile, slot, len;
    if (!find_tile(p, tile_idx, R, &b, &tile) || !run_ok(p, b, &slot, &len)) return;
    const int32_t t0 = max(run_begin(p.runs, b), 0);
    const int32_t t1 = p.runs.cu ? min(p.runs.cu[b + 1u], static_cast<int32_t>(p.runs.n)) : t0 + 1;
    const uint32_t n = static_cast<uint32_t>(t1 - t0);
    uint32_t count;
    const uint32_t chunk = own_chunk(len, p.splits, &count);
    if (s >= max(count, p.part ? 0u : 1u)) return;   // with one chunk a row, an empty slot's rows still get their zeros
    it.key0 = s * chunk;
    it.key1 = min(len, it.key0 + chunk);
    const uint64_t base = static_cast<uint64_t>(slot) * p.kv.slot_rows * H + it.h;
    it.k = p.kv.k + base * p.kv.hd;
    it.v = p.kv.v + base * p.kv.hd;
    it.ks = p.kv.ks + base;
    it.vs = p.kv.vs + base;
    it.row0 = tile * R;
    it.rows = n * p.group;
    it.t0 = t0;
    it.seen0 = static_cast<int32_t>(len) - static_cast<int32_t>(n) + 1;
    it.chunk = p.p_chunks + s;
    if (p.own_wide) kva_item<HDP, true>(p, it, kva_smem, s_rf);
    else kva_item<HDP, false>(p, it, kva_smem, s_rf);
}

template <uint32_t HDP>
__global__ void __launch_bounds__(kKvaThreads, 2) kv_attention_kernel(const __grid_constant__ KvAttnParams p) {
    extern __shared__ __align__(16) uint8_t kva_smem[];
    __shared__ float s_rf[16];
    pdl_launch_dependents();
    kva_cta<HDP>(p, kva_smem, s_rf);
    // not to end before the prefix's kernel has: the joining kernel waits for this one alone
    if (p.chained && blockIdx.x == 0u) pdl_wait();
}

// out = sum_c w_c o_c / sum_c w_c l_c with w_c = 2^(m_c - max m) over a row's chunks,
// in chunk order.  WPR warps a row: one where a row has few chunks (then a CTA
// joins four rows), else four, each with every fourth chunk.
template <uint32_t WPR>
__global__ void __launch_bounds__(kKvaThreads) kv_attention_join_kernel(const __grid_constant__ KvAttnParams p) {
    __shared__ float s_w[kKvaWarps / WPR][kKvaMaxChunks];
    __shared__ float s_o[kKvaWarps][kKvaMaxHeadDim];
    __shared__ float s_l[kKvaWarps];
    pdl_wait();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, hd = p.kv.hd;
    const uint64_t row = static_cast<uint64_t>(blockIdx.x) * (kKvaWarps / WPR) + warp / WPR;
    const uint32_t sub = warp % WPR;
    bool live = row < static_cast<uint64_t>(p.runs.n) * p.heads;
    const uint32_t t = live ? static_cast<uint32_t>(row / p.heads) : 0u, head = static_cast<uint32_t>(row - static_cast<uint64_t>(t) * p.heads);
    uint32_t own = 0;
    if (live) {
        const int32_t b = find_run(p.runs, static_cast<int32_t>(t));
        uint32_t slot, len;
        live = b >= 0 && run_ok(p, static_cast<uint32_t>(b), &slot, &len);
        if (live && p.splits) own_chunk(len, p.splits, &own);
    }
    uint32_t pre = p.p_chunks;
    if (p.pre_ctas) {   // the CTAs whose ranges meet this row's unit
        const uint32_t T = (p.prefix_len + kPreKeys - 1u) / kPreKeys, h = head / p.group;
        const uint32_t unit = h * p.row_tiles + (t * p.group + head - h * p.group) / kPreRows;
        pre = pre_owner(p.pre_base, p.pre_extra, unit * T + T - 1u) - pre_owner(p.pre_base, p.pre_extra, unit * T) + 1u;
    }
    const uint32_t chunks = live ? pre + own : 0u;
    auto at = [&](uint32_t i) { return i < pre ? i : p.p_chunks + (i - pre); };   // record of chunk i
    const uint64_t ld = hd + 4u;
    const float* rec = p.part + row * (p.p_chunks + p.splits) * ld;
    float* w = s_w[warp / WPR];
    float m = -INFINITY;
    for (uint32_t i = lane; i < chunks; i += 32u) m = fmaxf(m, __ldcg(rec + at(i) * ld + hd));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    float l = 0.0f;
    for (uint32_t i = sub + WPR * lane; i < chunks; i += 32u * WPR) {
        const float mi = __ldcg(rec + at(i) * ld + hd);
        const float wi = mi == -INFINITY ? 0.0f : ex2(__fsub_rn(mi, m));
        w[i] = wi;
        l = fmaf(wi, __ldcg(rec + at(i) * ld + hd + 1u), l);
    }
    l = warp_sum(l);
    __syncwarp();
    float4 y[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll 4
    for (uint32_t i = sub; i < chunks; i += WPR) {
        const float wi = w[i];
#pragma unroll
        for (uint32_t j = 0; j < 2u; ++j) {
            const uint32_t d = 4u * lane + 128u * j;
            if (d >= hd) continue;
            const float4 a = __ldcg(reinterpret_cast<const float4*>(rec + at(i) * ld + d));
            if (wi == 0.0f) continue;
            y[j].x = fmaf(wi, a.x, y[j].x);
            y[j].y = fmaf(wi, a.y, y[j].y);
            y[j].z = fmaf(wi, a.z, y[j].z);
            y[j].w = fmaf(wi, a.w, y[j].w);
        }
    }
    if constexpr (WPR > 1u) {
#pragma unroll
        for (uint32_t j = 0; j < 2u; ++j) {
            const uint32_t d = 4u * lane + 128u * j;
            if (d < hd) *reinterpret_cast<float4*>(&s_o[warp][d]) = y[j];
        }
        if (lane == 0u) s_l[warp] = l;
        __syncthreads();
        if (sub != 0u) return;
        for (uint32_t k = 1; k < WPR; ++k) {
            l = __fadd_rn(l, s_l[warp + k]);
#pragma unroll
            for (uint32_t j = 0; j < 2u; ++j) {
                const uint32_t d = 4u * lane + 128u * j;
                if (d >= hd) continue;
                const float4 a = *reinterpret_cast<const float4*>(&s_o[warp + k][d]);
                y[j] = make_float4(__fadd_rn(y[j].x, a.x), __fadd_rn(y[j].y, a.y), __fadd_rn(y[j].z, a.z),
                                   __fadd_rn(y[j].w, a.w));
            }
        }
    }
    if (!live) return;
    const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
#pragma unroll
    for (uint32_t j = 0; j < 2u; ++j) {
        const uint32_t d = 4u * lane + 128u * j;
        if (d < hd)
            store4_any(p.out, p.type, static_cast<uint64_t>(t) * p.out_ld + static_cast<uint64_t>(head) * hd + d,
                       make_float4(__fmul_rn(y[j].x, inv), __fmul_rn(y[j].y, inv), __fmul_rn(y[j].z, inv),
                                   __fmul_rn(y[j].w, inv)),
                       p.wide);
    }
}

}  // namespace qraf_dev
