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
// four products accumulate in fp32; maxima, sums and the running output are fp32.  The
// tensor cores' accumulator truncates toward zero, so it takes the products of 16 keys,
// or of 64 dimensions of a score, and the running output and the scores are added to
// outside of it, rounded to nearest: left in it, 4096 evenly weighted keys came out
// 1.8e-5 short, 16384 9.2e-5 (measured on a B200).
//
// Work.  The rows of a work item (up to 16 of one KV head) meet one chunk of keys:
// a chunk of the prefix, with rows of any sequences, so the prefix is read once
// for every 16 rows (kv_prefix.cuh has it instead where there are rows enough for
// the 5th-generation tensor cores); or a chunk of one sequence's own rows.  One
// warp has an item and is a CTA of its own: it takes steps of 32 keys, keeps
// maximum, sum and output in registers and leaves them as the chunk's record; a
// second kernel joins the chunks of a row, in their order, so results do not
// depend on timing.  A call with one chunk a row writes its output at once, and a
// small call joins its chunks within a thread-block cluster (one launch).
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "common.cuh"
#include "kv_cache.cuh"

namespace qraf_dev {

constexpr uint32_t kKvaStages = 2;          // steps of codes that a warp has in shared memory
constexpr uint32_t kJoinThreads = 256, kJoinWarps = kJoinThreads / 32u;
constexpr uint32_t kKvaMinChunk = 64;       // keys per chunk, at least: two steps
constexpr uint32_t kKvaMaxHeadDim = 256;
constexpr uint32_t kKvaMaxChunks = 512;     // chunks of one row, prefix and own rows together

constexpr uint32_t kPreRows = 128;          // kv_prefix.cuh: query rows of a tile = MMA M
constexpr uint32_t kPreKeys = 128;          // and keys of a tile
constexpr uint32_t kPreTerm = 8;            // tiles of one sum on the tensor cores
static_assert(kPreTerm % 2u == 0u, "the same warpgroup begins every sum");

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
    float* pre_sum;          // its CTAs' sums of finished terms, [128][64 or 128] each; nullptr: no stretch has two
    uint32_t chained;        // kv_attention_kernel was launched as kv_prefix_kernel's dependent
    uint32_t own_tiles, splits;              // own rows: row tiles over all runs (at most), chunks of each (at most)
    uint32_t own_wide;       // the kernel with tiles of 16 rows, else 8
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

// The same product alone.
__device__ __forceinline__ void mma_f16_new(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
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

// A span of keys of one KV head.
struct KvaKeys {
    const int8_t* k;      // key 0
    const int8_t* v;
    const float* ks;
    const float* vs;
    uint32_t key0, key1;
    int32_t seen0;        // keys that row 0's token sees (grows by one a token); INT32_MAX: all of the span
};

// What one warp works on.
struct KvaItem {
    KvaKeys a, b;         // one span or two
    uint32_t spans;
    uint64_t stride;      // elements from key to key
    uint32_t sstride;     // scales from key to key
    uint32_t row0, rows;  // rows [row0, rows) of the group; row r is token t0 + r / group, head h * group + r % group
    int32_t t0;
    uint32_t h;
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
    static constexpr uint32_t kStage = 2u * kKeys * HDP + 2u * kKeys * 4u;   // a step's codes of K and V, their scales
    static constexpr uint32_t kSmem = kQBytes + kKvaStages * kStage;
};

// One work item, one warp.  WIDE: 16 rows, hi and lo parts as two products into one
// accumulator; else 8 rows, the tensor-core tile's rows 0-7 their hi parts and
// rows 8-15 their lo parts, whose two results meet in one thread.
//
// Lane (g = lane / 4, c = lane % 4).  The codes' order in the products is free as
// long as both operands agree, and is chosen so that every fragment comes from wide
// reads: of a K row a lane reads 16 bytes (dims 64 j + 16 c ..), each of its four
// words one step's fragment; of V it reads its columns (16 g ..) of the four keys
// that its score accumulators belong to, and pairs their bytes.  The codes come to
// shared memory by cp.async, one step ahead; the rows' 16-byte units are exchanged
// so that both reads meet no bank twice.
//
// SHARED: the record goes to the start of the warp's ring ([row][head_dim + 4]).
template <uint32_t HDP, bool WIDE, bool SHARED>
__device__ __forceinline__ void kva_item(const KvAttnParams& p, const KvaItem& it, uint8_t* smem) {
    using S = KvaShape<HDP, WIDE>;
    constexpr uint32_t R = S::kRows, RT = WIDE ? 2u : 1u;   // RT: score rows of a thread
    constexpr uint32_t U = HDP / 16u;                       // 16-byte units of a row
    const uint32_t lane = threadIdx.x & 31u, g = lane >> 2, c = lane & 3u;
    const uint32_t hd = p.kv.hd, G = p.group;
    const uint32_t nrows = min(R, it.rows - it.row0);

    // ── the first step's codes and scales ──
    uint8_t* ring = smem + S::kQBytes;
    KvaKeys span = it.a;
    constexpr uint32_t KPA = 32u / U;   // keys per copy
    const uint32_t cu = lane % U, ck = lane / U;
    const uint32_t k_at = ck * HDP, k_sw = 4u & (U - 1u), v_sw = 6u & (U - 1u);
    auto fetch = [&](uint32_t k0, uint32_t stage) {   // the step from key k0, a group even past the end
        if (k0 < span.key1) {
            const uint32_t last = span.key1 - 1u;
            uint8_t* dst = ring + stage * S::kStage;
            if (16u * cu < hd) {
#pragma unroll
                for (uint32_t i = 0; i < S::kKeys / KPA; ++i) {
                    const uint32_t k = ck + i * KPA;
                    const uint64_t off = static_cast<uint64_t>(min(k0 + k, last)) * it.stride + 16u * cu;
                    cp_async16(dst + k_at + i * KPA * HDP + 16u * (cu ^ ((k & 1u) * k_sw)), span.k + off);
                    cp_async16(dst + S::kKeys * HDP + k_at + i * KPA * HDP + 16u * (cu ^ (k & v_sw)), span.v + off);
                }
            }
            if (lane < S::kKeys) {
                const uint64_t off = static_cast<uint64_t>(min(k0 + lane, last)) * it.sstride;
                cp_async4(dst + 2u * S::kKeys * HDP + 4u * lane, span.ks + off);
                cp_async4(dst + 2u * S::kKeys * HDP + 4u * (S::kKeys + lane), span.vs + off);
            }
        }
        cp_async_commit();
    };
    if (it.spans) fetch(span.key0, 0);

    // ── the query rows: powers of two, then the fragments in shared memory ──
    float rf[RT];
    {
        constexpr uint32_t TPR = 32u / R, QN = HDP / 4u / TPR;   // lanes a row, quads (4 dims) a lane
        constexpr uint32_t QB = QN > 16u ? 16u : QN;             // in flight at a time
        const uint32_t r = lane / TPR, j0 = lane % TPR, row = it.row0 + r, i = row / G;
        const uint64_t at = static_cast<uint64_t>(it.t0 + static_cast<int32_t>(i)) * p.q_ld +
                            static_cast<uint64_t>(it.h * G + (row - i * G)) * hd;
        float4 x[QB];
        auto load = [&](uint32_t q0) {
            auto typed = [&](const auto* q) {
#pragma unroll
                for (uint32_t j = 0; j < QB; ++j) {
                    const uint32_t d = 4u * (j0 + (q0 + j) * TPR);
                    x[j] = r < nrows && d < hd ? load4(q + at + d, p.q_wide) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
            };
            if (p.type == QRAF_TYPE_F32) typed(static_cast<const float*>(p.q));
            else if (p.type == QRAF_TYPE_F16) typed(static_cast<const __half*>(p.q));
            else typed(static_cast<const __nv_bfloat16*>(p.q));
#pragma unroll
            for (uint32_t j = 0; j < QB; ++j)
                x[j] = make_float4(__fmul_rn(x[j].x, p.scale_log2), __fmul_rn(x[j].y, p.scale_log2),
                                   __fmul_rn(x[j].z, p.scale_log2), __fmul_rn(x[j].w, p.scale_log2));
        };
        float m = 0.0f;
#pragma unroll 1
        for (uint32_t q0 = 0; q0 < QN; q0 += QB) {
            load(q0);
#pragma unroll
            for (uint32_t j = 0; j < QB; ++j) m = absmax4(x[j], m);
        }
#pragma unroll
        for (uint32_t o = TPR / 2u; o > 0u; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        // the largest becomes 2^10 .. 2^11: hi up to 2048, lo's last bit 2^-24
        const int32_t e = max(exponent_bits(m), 11);
        const float up = pow2_bits(264 - e);
#pragma unroll
        for (uint32_t n = 0; n < RT; ++n) rf[n] = __shfl_sync(0xFFFFFFFFu, pow2_bits(e - 10), (g + 8u * n) * TPR);
        uint32_t* frag = reinterpret_cast<uint32_t*>(smem);
#pragma unroll 1
        for (uint32_t q0 = 0; q0 < QN; q0 += QB) {
            if (QN > QB) load(q0);
#pragma unroll
            for (uint32_t j = 0; j < QB; ++j) {
                const uint32_t d = 4u * (j0 + (q0 + j) * TPR);
                uint32_t hi[2], lo[2];
                split_f16(__fmul_rn(x[j].x, up), __fmul_rn(x[j].y, up), hi[0], lo[0]);
                split_f16(__fmul_rn(x[j].z, up), __fmul_rn(x[j].w, up), hi[1], lo[1]);
                const uint32_t st = 4u * (d >> 6) + ((d >> 2) & 3u), l = 4u * (r & 7u) + ((d >> 4) & 3u);
                uint32_t* f = frag + 4u * (st * 32u + l);
                if constexpr (WIDE) {
                    f += r >> 3;
                    f[0] = hi[0];
                    f[2] = hi[1];
                    f += 4u * S::kSteps * 32u;
                    f[0] = lo[0];
                    f[2] = lo[1];
                } else {
                    *reinterpret_cast<uint4*>(f) = make_uint4(hi[0], lo[0], hi[1], lo[1]);
                }
            }
        }
    }

    // the output: per tile two columns of the lane's RT rows
    float2 o[S::kOut][RT];
#pragma unroll
    for (uint32_t i = 0; i < S::kOut; ++i)
#pragma unroll
        for (uint32_t e = 0; e < RT; ++e) o[i][e] = make_float2(0.0f, 0.0f);
    float run_m[RT], run_l[RT];
    int32_t vref[RT];   // the output's unit is 2^(vref - 140), every V scale seen is below 2^(vref - 126)
#pragma unroll
    for (uint32_t e = 0; e < RT; ++e) {
        run_m[e] = -INFINITY;
        run_l[e] = 0.0f;
        vref[e] = 14;
    }

#pragma unroll 1
    for (uint32_t n_span = 0; n_span < it.spans; ++n_span) {
        if (n_span) {
            span = it.b;
            fetch(span.key0, 0);
        }
        uint32_t seen[RT];   // keys below this one are visible to the row
#pragma unroll
        for (uint32_t e = 0; e < RT; ++e) {
            const uint32_t r = g + 8u * e, row = it.row0 + r;
            seen[e] = span.key1;
            if (span.seen0 != INT32_MAX && r < nrows) {
                const int32_t n = span.seen0 + static_cast<int32_t>(row / G);
                seen[e] = min(span.key1, static_cast<uint32_t>(max(n, 0)));
            }
        }   // rows past the tile's last are zeros that see every key; they are not written
        const uint32_t all_see = __reduce_min_sync(0xFFFFFFFFu, RT == 2u ? min(seen[0], seen[RT - 1u]) : seen[0]);
        uint32_t stage = 0;
#pragma unroll 1
        for (uint32_t k0 = span.key0; k0 < span.key1; k0 += S::kKeys, stage ^= 1u) {
            fetch(k0 + S::kKeys, stage ^ 1u);   // that stage's step was read before the last __syncwarp
            cp_async_wait<1>();
            __syncwarp();   // the other lanes' copies (and, at first, the query fragments)
            const uint8_t* kc = ring + stage * S::kStage;
            const uint8_t* vc = kc + S::kKeys * HDP;
            const float* scales = reinterpret_cast<const float*>(vc + S::kKeys * HDP);
            // ── scores ──
            float2 s[S::kTiles][RT];   // two keys of the lane's RT rows; 64 dims at a time in the accumulator
#pragma unroll
            for (uint32_t j = 0; j < HDP / 64u; ++j) {
                uint4 kr[S::kTiles];
                float acc[S::kTiles][4];
                const bool in = 64u * j + 16u * c < hd;
#pragma unroll
                for (uint32_t t = 0; t < S::kTiles; ++t)
                    kr[t] = in ? *reinterpret_cast<const uint4*>(kc + (8u * t + g) * HDP + 16u * ((4u * j + c) ^ ((g & 1u) * k_sw)))
                               : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                for (uint32_t i = 0; i < 4u; ++i) {
                    const uint4 qa = reinterpret_cast<const uint4*>(smem)[(4u * j + i) * 32u + lane];
                    const uint32_t a[4] = {qa.x, qa.y, qa.z, qa.w};
                    uint32_t al[4];
                    if constexpr (WIDE) {
                        const uint4 ql = reinterpret_cast<const uint4*>(smem)[(S::kSteps + 4u * j + i) * 32u + lane];
                        al[0] = ql.x;
                        al[1] = ql.y;
                        al[2] = ql.z;
                        al[3] = ql.w;
                    }
#pragma unroll
                    for (uint32_t t = 0; t < S::kTiles; ++t) {
                        const uint32_t w = (i == 0u ? kr[t].x : i == 1u ? kr[t].y : i == 2u ? kr[t].z : kr[t].w) ^ 0x80808080u;
                        const uint32_t b0 = codes_f16<0x4140u>(w), b1 = codes_f16<0x4342u>(w);
                        if constexpr (WIDE) {
                            if (i == 0u) mma_f16_new(acc[t], al, b0, b1);
                            else mma_f16(acc[t], al, b0, b1);
                            mma_f16(acc[t], a, b0, b1);
                        } else {
                            if (i == 0u) mma_f16_new(acc[t], a, b0, b1);
                            else mma_f16(acc[t], a, b0, b1);
                        }
                    }
                }
#pragma unroll
                for (uint32_t t = 0; t < S::kTiles; ++t) {
                    const float2 d0 = make_float2(acc[t][0], acc[t][1]), d1 = make_float2(acc[t][2], acc[t][3]);
                    const float2 y = WIDE ? d0 : f2_add(d0, d1);
                    s[t][0] = j ? f2_add(s[t][0], y) : y;
                    if constexpr (WIDE) s[t][RT - 1u] = j ? f2_add(s[t][RT - 1u], d1) : d1;
                }
            }

            // ── softmax ──
            float x[RT][2u * S::kTiles], vs[RT][2u * S::kTiles];   // scores, and the V scales as the row sees them
            float mt[RT];
            int32_t ev[RT];   // the largest exponent of those scales (not of an infinity or NaN)
            {
                const int32_t e = lane < S::kKeys && k0 + lane < span.key1 ? exponent_bits(scales[S::kKeys + lane]) : 0;
                const int32_t most = static_cast<int32_t>(__reduce_max_sync(0xFFFFFFFFu, static_cast<uint32_t>(e == 255 ? 0 : e)));
#pragma unroll
                for (uint32_t n = 0; n < RT; ++n) {
                    mt[n] = -INFINITY;
                    ev[n] = most;
                }
            }
#pragma unroll
            for (uint32_t t = 0; t < S::kTiles; ++t) {
                const float2 ks = *reinterpret_cast<const float2*>(scales + 8u * t + 2u * c);
                const float2 vv = *reinterpret_cast<const float2*>(scales + S::kKeys + 8u * t + 2u * c);
#pragma unroll
                for (uint32_t e = 0; e < RT; ++e) {
                    const float2 v = f2_mul(s[t][e], f2_mul(ks, make_float2(rf[e], rf[e])));
                    x[e][2u * t] = v.x;
                    x[e][2u * t + 1u] = v.y;
                    vs[e][2u * t] = vv.x;
                    vs[e][2u * t + 1u] = vv.y;
                }
            }
            if (k0 + S::kKeys > all_see) {   // the step has keys that some row does not see: weight 0 whatever they hold
#pragma unroll
                for (uint32_t e = 0; e < RT; ++e) {
                    ev[e] = 0;
#pragma unroll
                    for (uint32_t i = 0; i < 2u * S::kTiles; ++i) {
                        const int32_t eb = exponent_bits(vs[e][i]);
                        if (k0 + 8u * (i >> 1) + 2u * c + (i & 1u) >= seen[e]) {
                            x[e][i] = -INFINITY;
                            vs[e][i] = 0.0f;
                        } else if (eb < 255) {
                            ev[e] = max(ev[e], eb);
                        }
                    }
                    ev[e] = max(ev[e], __shfl_xor_sync(0xFFFFFFFFu, ev[e], 1));
                    ev[e] = max(ev[e], __shfl_xor_sync(0xFFFFFFFFu, ev[e], 2));
                }
            }
            float down[RT], m_use[RT], vup[RT];
            bool moved = false;
#pragma unroll
            for (uint32_t e = 0; e < RT; ++e) {
#pragma unroll
                for (uint32_t i = 0; i < 2u * S::kTiles; ++i) mt[e] = fmaxf(mt[e], x[e][i]);
                mt[e] = fmaxf(mt[e], __shfl_xor_sync(0xFFFFFFFFu, mt[e], 1));
                mt[e] = fmaxf(mt[e], __shfl_xor_sync(0xFFFFFFFFu, mt[e], 2));
                const float m_new = fmaxf(run_m[e], mt[e]);
                const float alpha = m_new == run_m[e] ? 1.0f : ex2(__fsub_rn(run_m[e], m_new));   // 0 at the first keys
                run_m[e] = m_new;
                m_use[e] = m_new == -INFINITY ? 0.0f : m_new;   // nothing seen yet: every weight exp(-inf) = 0
                run_l[e] = __fmul_rn(run_l[e], alpha);
                const int32_t vnew = max(vref[e], ev[e]);
                down[e] = __fmul_rn(alpha, pow2_bits(127 + vref[e] - vnew));
                vref[e] = vnew;
                vup[e] = pow2_bits(267 - vnew);   // 2^14 over the unit: weights below 2^14
                moved |= down[e] != 1.0f;
            }
            if (__any_sync(0xFFFFFFFFu, moved)) {
#pragma unroll
                for (uint32_t i = 0; i < S::kOut; ++i)
#pragma unroll
                    for (uint32_t e = 0; e < RT; ++e) o[i][e] = f2_mul(o[i][e], make_float2(down[e], down[e]));
            }
            uint32_t ph[RT][S::kTiles], pl[RT][S::kTiles];
#pragma unroll
            for (uint32_t t = 0; t < S::kTiles; ++t) {
#pragma unroll
                for (uint32_t e = 0; e < RT; ++e) {
                    const float2 w = make_float2(ex2(__fsub_rn(x[e][2u * t], m_use[e])), ex2(__fsub_rn(x[e][2u * t + 1u], m_use[e])));
                    run_l[e] = __fadd_rn(run_l[e], __fadd_rn(w.x, w.y));
                    const float2 y = f2_mul(w, f2_mul(make_float2(vs[e][2u * t], vs[e][2u * t + 1u]), make_float2(vup[e], vup[e])));
                    split_f16(y.x, y.y, ph[e][t], pl[e][t]);
                }
            }
            // ── weighted sum of V ──
#pragma unroll
            for (uint32_t u = 0; u < S::kKeys / 16u; ++u) {
                uint32_t vw[4][S::kWords];   // this lane's columns of keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9
#pragma unroll
                for (uint32_t r = 0; r < 4u; ++r) {
                    const uint32_t k = 16u * u + 2u * c + (r & 1u) + 8u * (r >> 1);   // k & 6 = 2 c
                    const uint8_t* row = vc + k * HDP;
                    if constexpr (HDP == 64u) {
                        const uint2 w = 8u * g < hd ? *reinterpret_cast<const uint2*>(row + 16u * ((g >> 1) ^ (2u * c & v_sw)) + 8u * (g & 1u))
                                                    : make_uint2(0u, 0u);
                        vw[r][0] = w.x;
                        vw[r][1] = w.y;
                    } else {
#pragma unroll
                        for (uint32_t h = 0; h < HDP / 128u; ++h) {
                            const uint4 w = 128u * h + 16u * g < hd
                                                ? *reinterpret_cast<const uint4*>(row + 16u * ((8u * h + g) ^ (2u * c & v_sw)))
                                                : make_uint4(0u, 0u, 0u, 0u);
                            vw[r][4u * h] = w.x;
                            vw[r][4u * h + 1u] = w.y;
                            vw[r][4u * h + 2u] = w.z;
                            vw[r][4u * h + 3u] = w.w;
                        }
                    }
                }
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
                    const uint32_t v0 = vw[0][w] ^ 0x80808080u, v1 = vw[1][w] ^ 0x80808080u;
                    const uint32_t v2 = vw[2][w] ^ 0x80808080u, v3 = vw[3][w] ^ 0x80808080u;
                    const uint32_t a01 = __byte_perm(v0, v1, 0x5140u), a23 = __byte_perm(v0, v1, 0x7362u);
                    const uint32_t b01 = __byte_perm(v2, v3, 0x5140u), b23 = __byte_perm(v2, v3, 0x7362u);
                    const uint32_t b[4][2] = {{codes_f16<0x4140u>(a01), codes_f16<0x4140u>(b01)},
                                              {codes_f16<0x4342u>(a01), codes_f16<0x4342u>(b01)},
                                              {codes_f16<0x4140u>(a23), codes_f16<0x4140u>(b23)},
                                              {codes_f16<0x4342u>(a23), codes_f16<0x4342u>(b23)}};
#pragma unroll
                    for (uint32_t j = 0; j < 4u; ++j) {
                        float d[4];
                        float2(&y)[RT] = o[4u * w + j];
                        if constexpr (WIDE) {
                            mma_f16_new(d, al, b[j][0], b[j][1]);
                            mma_f16(d, a, b[j][0], b[j][1]);
                            y[0] = f2_add(y[0], make_float2(d[0], d[1]));
                            y[RT - 1u] = f2_add(y[RT - 1u], make_float2(d[2], d[3]));
                        } else {
                            mma_f16_new(d, a, b[j][0], b[j][1]);
                            y[0] = f2_add(y[0], f2_add(make_float2(d[0], d[1]), make_float2(d[2], d[3])));
                        }
                    }
                }
            }
            __syncwarp();   // the stage has been read
        }
        cp_async_wait<0>();
    }
    __syncwarp();

    // ── the record, or with one chunk a row the output itself ──
#pragma unroll
    for (uint32_t e = 0; e < RT; ++e) {
        run_l[e] = __fadd_rn(run_l[e], __shfl_xor_sync(0xFFFFFFFFu, run_l[e], 1));
        run_l[e] = __fadd_rn(run_l[e], __shfl_xor_sync(0xFFFFFFFFu, run_l[e], 2));
        const uint32_t r = g + 8u * e, row = it.row0 + r, i = row / G, head = it.h * G + (row - i * G);
        const int32_t t = it.t0 + static_cast<int32_t>(i);
        float* rec = SHARED ? reinterpret_cast<float*>(ring) + r * (hd + 4u)
                     : p.part ? p.part + ((static_cast<uint64_t>(t) * p.heads + head) * (p.p_chunks + p.splits) + it.chunk) * (hd + 4u)
                            : nullptr;
        float f = pow2_bits(vref[e] - 13);   // to numbers
        bool live = r < nrows;
        if (!rec) {   // the row's output, unless its run is padding
            uint32_t slot, len;
            for (uint32_t q = 0; q < 8u; ++q) {   // find_run takes the whole warp: one row at a time
                const int32_t tq = __shfl_sync(0xFFFFFFFFu, t, 4u * q);
                const bool lq = __shfl_sync(0xFFFFFFFFu, live, 4u * q);
                bool ok = false;
                if (lq) {
                    const int32_t b = find_run(p.runs, tq);
                    ok = b >= 0 && run_ok(p, static_cast<uint32_t>(b), &slot, &len);
                }
                if (g == q) live = ok;
            }
            f = run_l[e] == 0.0f ? 0.0f : __fmul_rn(f, __fdiv_rn(1.0f, run_l[e]));
        }
        if (!live) continue;
#pragma unroll
        for (uint32_t b = 0; b < 2u; ++b) {
            const uint32_t n = 2u * c + b;   // column within an output tile
#pragma unroll
            for (uint32_t w = 0; w < S::kWords; ++w) {
                const uint32_t d = HDP == 64u ? 8u * n + 4u * w : 128u * (w >> 2) + 16u * n + 4u * (w & 3u);
                if (d >= hd) continue;
                float y[4];
#pragma unroll
                for (uint32_t j = 0; j < 4u; ++j) {
                    const float2 a = o[4u * w + j][e];
                    y[j] = __fmul_rn(b ? a.y : a.x, f);
                }
                const float4 v = make_float4(y[0], y[1], y[2], y[3]);
                if (rec) *reinterpret_cast<float4*>(rec + d) = v;
                else store4_any(p.out, p.type, static_cast<uint64_t>(t) * p.out_ld + static_cast<uint64_t>(head) * hd + d, v, p.wide);
            }
        }
        if (rec && c == 0u) *reinterpret_cast<float2*>(rec + hd) = make_float2(run_m[e], run_l[e]);
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

// The keys of a KV head: of the prefix, and of a run's slot.
__device__ __forceinline__ KvaKeys prefix_keys(const KvAttnParams& p, uint32_t h) {
    KvaKeys k;
    k.k = p.pk + static_cast<uint64_t>(h) * p.kv.hd;
    k.v = p.pv + static_cast<uint64_t>(h) * p.kv.hd;
    k.ks = p.pks + h;
    k.vs = p.pvs + h;
    k.seen0 = INT32_MAX;
    return k;
}
__device__ __forceinline__ KvaKeys slot_keys(const KvAttnParams& p, uint32_t h, uint32_t slot, uint32_t len, uint32_t n) {
    const uint64_t base = static_cast<uint64_t>(slot) * p.kv.slot_rows * p.kv.kv_heads + h;
    KvaKeys k;
    k.k = p.kv.k + base * p.kv.hd;
    k.v = p.kv.v + base * p.kv.hd;
    k.ks = p.kv.ks + base;
    k.vs = p.kv.vs + base;
    k.seen0 = static_cast<int32_t>(len) - static_cast<int32_t>(n) + 1;
    return k;
}

// Own-row tile `idx` of R rows into the item; false where there is none, or its run
// is padding or out of range.  *seen: rows of the slot that the tile's last token sees.
__device__ __forceinline__ bool own_item(const KvAttnParams& p, uint32_t idx, uint32_t R, KvaItem& it, uint32_t* slot,
                                         uint32_t* len, uint32_t* n, uint32_t* seen) {
    uint32_t b, tile;
    if (!find_tile(p, idx, R, &b, &tile) || !run_ok(p, b, slot, len)) return false;
    const int32_t t0 = max(run_begin(p.runs, b), 0);
    const int32_t t1 = p.runs.cu ? min(p.runs.cu[b + 1u], static_cast<int32_t>(p.runs.n)) : t0 + 1;
    *n = static_cast<uint32_t>(t1 - t0);
    it.row0 = tile * R;
    it.rows = *n * p.group;
    it.t0 = t0;
    const int32_t last = static_cast<int32_t>((min(it.rows, it.row0 + R) - 1u) / p.group);
    *seen = min(*len, static_cast<uint32_t>(max(static_cast<int32_t>(*len) - static_cast<int32_t>(*n) + 1 + last, 0)));
    return true;
}

// WIDE: prefix items and own rows in tiles of 16 rows, else own rows in tiles of 8.
//
// Measured on a B200 (64 sequences, 8 KV heads of 128, 8 query heads each, with the joining
// kernel): up to 1024 rows a sequence 37.5 us, up to 4096 106 us, 3.6 TB/s of codes and
// scales.  The loads alone take 76 us there: what bounds it is issuing some 950 instructions
// a step of 32 keys, most of them turning codes into fp16 fragments (64 are the additions to
// the output: left in the tensor cores' accumulator it was 101 us, and short).  Registers for
// eight CTAs an SM at least: for eleven it took a tenth longer.
template <uint32_t HDP, bool WIDE>
__device__ __forceinline__ void kva_cta(const KvAttnParams& p, uint8_t* kva_smem) {
    const uint32_t H = p.kv.kv_heads;
    KvaItem it;
    it.sstride = H;
    it.stride = static_cast<uint64_t>(H) * p.kv.hd;
    it.spans = 1u;
    uint32_t idx = blockIdx.x;
    const uint32_t p_items = !WIDE || p.pre_ctas ? 0u : p.row_tiles * H * p.p_chunks;
    if (WIDE && idx < p_items) {
        const uint32_t q = idx / p.row_tiles, rt = idx - q * p.row_tiles;
        it.chunk = q / H;
        it.h = q - it.chunk * H;
        it.a = prefix_keys(p, it.h);
        it.a.key0 = it.chunk * p.p_chunk;
        it.a.key1 = min(p.prefix_len, it.a.key0 + p.p_chunk);
        it.row0 = rt * 16u;
        it.rows = p.runs.n * p.group;
        it.t0 = 0;
    } else {
        idx -= p_items;
        const uint32_t q = idx / p.splits, s = idx - q * p.splits, tile_idx = q / H;
        it.h = q - tile_idx * H;
        uint32_t slot, len, n, seen, count;
        if (!own_item(p, tile_idx, WIDE ? 16u : 8u, it, &slot, &len, &n, &seen)) return;
        const uint32_t chunk = own_chunk(len, p.splits, &count);
        if (s >= max(count, p.part ? 0u : 1u)) return;   // with one chunk a row, an empty slot's rows still get their zeros
        it.a = slot_keys(p, it.h, slot, len, n);
        it.a.key0 = s * chunk;
        it.a.key1 = min(seen, it.a.key0 + chunk);   // not past key0: a record of nothing
        it.chunk = p.p_chunks + s;
    }
    kva_item<HDP, WIDE, false>(p, it, kva_smem);
}

template <uint32_t HDP, bool WIDE>
__global__ void __launch_bounds__(32, 8) kv_attention_kernel(const __grid_constant__ KvAttnParams p) {
    extern __shared__ __align__(16) uint8_t kva_smem[];
    pdl_launch_dependents();
    kva_cta<HDP, WIDE>(p, kva_smem);
    // not to end before the prefix's kernel has: the joining kernel waits for this one alone
    if (p.chained && blockIdx.x == 0u) pdl_wait();
}

// Small calls, where latency counts: one launch, no workspace.  A cluster has a row
// tile of one sequence and one KV head; its up to 32 warps take the steps of prefix
// and own rows in equal shares, and join their records through distributed shared
// memory.  The prefix is read once for every tile here, from L2.  Bound by latency: 9.5
// us on a B200 for 4 sequences of 16 / 2 heads behind 777 rows, 24 with the kernels below.
constexpr uint32_t kKvaClusterWarps = 4;   // a CTA

template <uint32_t HDP, bool WIDE>
__global__ void __launch_bounds__(32 * kKvaClusterWarps) kv_attention_cluster_kernel(const __grid_constant__ KvAttnParams p) {
    namespace cg = cooperative_groups;
    using S = KvaShape<HDP, WIDE>;
    extern __shared__ __align__(16) uint8_t kva_smem[];
    const cg::cluster_group cl = cg::this_cluster();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, H = p.kv.kv_heads, hd = p.kv.hd;
    const uint32_t ctas = cl.num_blocks(), rank = cl.block_rank(), W = ctas * kKvaClusterWarps, me = rank * kKvaClusterWarps + warp;
    const uint32_t idx = blockIdx.x / ctas, tile_idx = idx / H;
    KvaItem it;
    it.sstride = H;
    it.stride = static_cast<uint64_t>(H) * hd;
    it.chunk = 0u;
    it.h = idx - tile_idx * H;
    uint32_t slot, len, n, seen;
    if (!own_item(p, tile_idx, S::kRows, it, &slot, &len, &n, &seen)) return;   // the whole cluster
    const uint32_t pre = (p.prefix_len + S::kKeys - 1u) / S::kKeys, own = (seen + S::kKeys - 1u) / S::kKeys;
    const uint32_t s0 = (pre + own) * me / W, s1 = (pre + own) * (me + 1u) / W;   // steps of this warp
    it.spans = 0u;
    if (s0 < min(s1, pre)) {
        it.a = prefix_keys(p, it.h);
        it.a.key0 = s0 * S::kKeys;
        it.a.key1 = min(p.prefix_len, min(s1, pre) * S::kKeys);
        it.spans = 1u;
    }
    if (s1 > max(s0, pre)) {
        KvaKeys k = slot_keys(p, it.h, slot, len, n);
        k.key0 = (max(s0, pre) - pre) * S::kKeys;
        k.key1 = min(seen, (s1 - pre) * S::kKeys);
        if (it.spans) it.b = k;
        else it.a = k;
        ++it.spans;
    }
    kva_item<HDP, WIDE, true>(p, it, kva_smem + warp * S::kSmem);
    cl.sync();
    const uint32_t ld = hd + 4u, nrows = min(S::kRows, it.rows - it.row0);
    auto record = [&](uint32_t w, uint32_t r) {   // row r of warp w of the cluster
        return reinterpret_cast<const float*>(cl.map_shared_rank(kva_smem, w / kKvaClusterWarps) +
                                              (w % kKvaClusterWarps) * S::kSmem + S::kQBytes) + r * ld;
    };
    for (uint32_t r = rank + ctas * warp; r < nrows; r += W) {
        const float2 ml = lane < W ? *reinterpret_cast<const float2*>(record(lane, r) + hd) : make_float2(-INFINITY, 0.0f);
        float m = ml.x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        const float w = ml.x == -INFINITY ? 0.0f : ex2(__fsub_rn(ml.x, m));
        const float l = warp_sum(__fmul_rn(w, ml.y));
        const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
        const uint32_t row = it.row0 + r, i = row / p.group, head = it.h * p.group + (row - i * p.group);
        const uint64_t out = static_cast<uint64_t>(it.t0 + static_cast<int32_t>(i)) * p.out_ld + static_cast<uint64_t>(head) * hd;
#pragma unroll 1
        for (uint32_t d0 = 0; d0 < hd; d0 += 128u) {
            const uint32_t d = d0 + 4u * lane;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
            for (uint32_t c = 0; c < W; ++c) {
                const float f = __shfl_sync(0xFFFFFFFFu, w, c);
                const float4 a = d < hd ? *reinterpret_cast<const float4*>(record(c, r) + d) : make_float4(0.f, 0.f, 0.f, 0.f);
                if (f == 0.0f) continue;
                y.x = fmaf(f, a.x, y.x);
                y.y = fmaf(f, a.y, y.y);
                y.z = fmaf(f, a.z, y.z);
                y.w = fmaf(f, a.w, y.w);
            }
            if (d < hd)
                store4_any(p.out, p.type, out + d,
                           make_float4(__fmul_rn(y.x, inv), __fmul_rn(y.y, inv), __fmul_rn(y.z, inv), __fmul_rn(y.w, inv)), p.wide);
        }
    }
    cl.sync();   // no CTA leaves while another reads its records
}

// out = sum_c w_c o_c / sum_c w_c l_c with w_c = 2^(m_c - max m) over a row's chunks,
// in chunk order.  WPR warps a row: one where a row has up to 16 chunks (then a CTA
// joins eight rows), else eight, each with every eighth chunk; eight records are in
// flight at a time.  The runs are looked up before the dependency wait: nothing that
// they say is written by the kernels before.  Bound by latency and by reading the
// records, from L2: with this order, 8 sequences behind 65536 rows went from 48 to 42 us.
constexpr uint32_t kJoinFew = 16;

template <uint32_t WPR>
__global__ void __launch_bounds__(kJoinThreads) kv_attention_join_kernel(const __grid_constant__ KvAttnParams p) {
    constexpr uint32_t kMine = WPR == 1u ? 1u : kKvaMaxChunks / (32u * WPR);   // records a lane has the weights of
    __shared__ float s_m[kJoinWarps], s_l[kJoinWarps];
    __shared__ float s_o[WPR == 1u ? 1u : kJoinWarps][kKvaMaxHeadDim];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, hd = p.kv.hd;
    const uint64_t row = static_cast<uint64_t>(blockIdx.x) * (kJoinWarps / WPR) + warp / WPR;
    const uint32_t sub = warp % WPR;
    bool live = row < static_cast<uint64_t>(p.runs.n) * p.heads;
    const uint32_t t = live ? static_cast<uint32_t>(row) / p.heads : 0u, head = static_cast<uint32_t>(row) - t * p.heads;
    uint32_t own = 0;
    if (live) {
        const int32_t b = find_run(p.runs, static_cast<int32_t>(t));
        uint32_t slot, len;
        live = b >= 0 && run_ok(p, static_cast<uint32_t>(b), &slot, &len);
        if (live && p.splits) own_chunk(len, p.splits, &own);
    }
    uint32_t pre = p.p_chunks;
    if (p.pre_ctas) {   // the CTAs whose ranges meet this row's unit leave a record each
        const uint32_t T = (p.prefix_len + kPreKeys - 1u) / kPreKeys, h = head / p.group;
        const uint32_t tile0 = (h * p.row_tiles + (t * p.group + head - h * p.group) / kPreRows) * T;
        pre = pre_owner(p.pre_base, p.pre_extra, tile0 + T - 1u) - pre_owner(p.pre_base, p.pre_extra, tile0) + 1u;
    }
    const uint32_t chunks = live ? pre + own : 0u;
    auto at = [&](uint32_t i) { return i < pre ? i : p.p_chunks + (i - pre); };   // record of chunk i
    const uint64_t ld = hd + 4u;
    const float* rec = p.part + row * (p.p_chunks + p.splits) * ld;
    // this warp's records are sub, sub + WPR, ...; lane i of it has the weights of its (i + 32 k)th
    pdl_wait();
    float2 ml[kMine];
    float m = -INFINITY;
#pragma unroll
    for (uint32_t k = 0; k < kMine; ++k) {
        const uint32_t i = sub + WPR * (lane + 32u * k);
        ml[k] = i < chunks ? __ldcg(reinterpret_cast<const float2*>(rec + at(i) * ld + hd)) : make_float2(-INFINITY, 0.0f);
        m = fmaxf(m, ml[k].x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    if constexpr (WPR > 1u) {
        if (lane == 0u) s_m[warp] = m;
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < kJoinWarps; ++k) m = fmaxf(m, s_m[k]);
    }
    float l = 0.0f;
    float4 y[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll
    for (uint32_t k = 0; k < kMine; ++k) {
        const float w = ml[k].x == -INFINITY ? 0.0f : ex2(__fsub_rn(ml[k].x, m));
        l = fmaf(w, ml[k].y, l);
        const uint32_t i0 = sub + WPR * 32u * k;
        const uint32_t n = i0 < chunks ? min(32u, (chunks - i0 + WPR - 1u) / WPR) : 0u;   // of this warp's, in this round
#pragma unroll 1
        for (uint32_t j0 = 0; j0 < n; j0 += 8u) {
#pragma unroll
            for (uint32_t half = 0; half < 2u; ++half) {
                const uint32_t d = 4u * lane + 128u * half;
                if (128u * half >= hd) break;
                float4 a[8];
                float f[8];
#pragma unroll
                for (uint32_t j = 0; j < 8u; ++j) {
                    f[j] = __shfl_sync(0xFFFFFFFFu, w, j0 + j);
                    a[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (j0 + j < n && f[j] != 0.0f && d < hd)
                        a[j] = __ldcg(reinterpret_cast<const float4*>(rec + at(i0 + WPR * (j0 + j)) * ld + d));
                }
#pragma unroll
                for (uint32_t j = 0; j < 8u; ++j) {
                    y[half].x = fmaf(f[j], a[j].x, y[half].x);
                    y[half].y = fmaf(f[j], a[j].y, y[half].y);
                    y[half].z = fmaf(f[j], a[j].z, y[half].z);
                    y[half].w = fmaf(f[j], a[j].w, y[half].w);
                }
            }
        }
    }
    l = warp_sum(l);
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
