// kv_cache.cuh — the int8 KV cache as an operator of its own: rows of K and V are
// quantised as they are written (qraf_cuda_kv_store) and read back as numbers
// (qraf_cuda_kv_load).  The codes and scales are those of the reference's
// QuantizedKVCache (include/nn/kv_cache_quant.h:61-94) and of the decoder's int8
// cache: per (row, KV head) scale = max |x| / 127, code = clamp(round(x / scale)).
//
// New rows come in runs: rows cu[b] .. cu[b + 1] of the input belong to
// consecutive cache rows starts[b], starts[b] + 1, ... of slot slots[b], so that
// one call takes one token of every sequence, a prompt, or drafts of uneven
// lengths.  Both directions are bound by memory: nothing is read twice.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace qraf_dev {

// One layer's cache in a kernel: row (slot, r) of head h starts at element
// ((slot * slot_rows + r) * kv_heads + h) * hd of the codes, its scale at the
// same index without hd.
struct KvView {
    int8_t* k;
    int8_t* v;
    float* ks;
    float* vs;
    uint64_t slot_rows;
    uint32_t slots, rows, kv_heads, hd;
};

// The runs of new rows: count of them over n rows; cu == nullptr is one row each.
struct KvRuns {
    const int32_t* slots;
    const int32_t* firsts;   // store / load: the run's first cache row; attention: the slot's visible rows
    const int32_t* cu;       // [count + 1] or nullptr
    uint32_t count, n;
};

__device__ __forceinline__ int32_t run_begin(const KvRuns& r, uint32_t b) {
    return r.cu ? r.cu[b] : static_cast<int32_t>(b);
}

// The last run b with cu[b] <= t (-1: none), by the whole warp: 32 samples of the
// remaining range a step, so two steps up to 1023 runs.  An unsorted cu gives
// some run in range.
__device__ __forceinline__ int32_t find_run(const KvRuns& r, int32_t t) {
    if (!r.cu) return t < static_cast<int32_t>(r.count) ? t : -1;
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t lo = 0, hi = r.count + 1u;
    bool first = true;
    while (first || hi - lo > 1u) {
        const uint32_t step = (hi - lo + 31u) / 32u, i = lo + lane * step;
        const uint32_t found = __popc(__ballot_sync(0xFFFFFFFFu, i < hi && r.cu[i] <= t));
        if (found == 0u) return -1;
        lo += (found - 1u) * step;
        hi = min(hi, lo + step);
        first = false;
    }
    return lo < r.count ? static_cast<int32_t>(lo) : -1;
}

__device__ __forceinline__ float4 load4(const float* p, bool wide) {
    if (wide) return *reinterpret_cast<const float4*>(p);
    return make_float4(p[0], p[1], p[2], p[3]);
}
__device__ __forceinline__ float4 load4(const __half* p, bool wide) {
    if (!wide) return make_float4(__half2float(p[0]), __half2float(p[1]), __half2float(p[2]), __half2float(p[3]));
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p, bool wide) {
    if (!wide)
        return make_float4(__bfloat162float(p[0]), __bfloat162float(p[1]), __bfloat162float(p[2]),
                           __bfloat162float(p[3]));
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u), __uint_as_float(w.y << 16),
                       __uint_as_float(w.y & 0xFFFF0000u));
}
// Stores round to nearest even once, from the fp32 value.
__device__ __forceinline__ void store4(float* p, float4 x, bool wide) {
    if (wide) {
        *reinterpret_cast<float4*>(p) = x;
    } else {
        p[0] = x.x;
        p[1] = x.y;
        p[2] = x.z;
        p[3] = x.w;
    }
}
__device__ __forceinline__ void store4(__half* p, float4 x, bool wide) {
    const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);
    if (wide) {
        *reinterpret_cast<uint2*>(p) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
        p[0] = a.x;
        p[1] = a.y;
        p[2] = b.x;
        p[3] = b.y;
    }
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, float4 x, bool wide) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
    if (wide) {
        *reinterpret_cast<uint2*>(p) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
        p[0] = a.x;
        p[1] = a.y;
        p[2] = b.x;
        p[3] = b.y;
    }
}

// QuantizedKVCache::store for one value (include/nn/kv_cache_quant.h:61-94):
// clamp(round(x * inv), -127, 127), inv = 1 / (max |x| / 127) (0 when the max is 0).
__device__ __forceinline__ int8_t kvq_code(float x, float inv) {
    return static_cast<int8_t>(fmaxf(-127.0f, fminf(127.0f, roundf(__fmul_rn(x, inv)))));
}
// The same for four values, packed.  Without conversions: with truncating adds
// (|y| + 0.5) + 2^23 leaves round-half-away(|y|) in the low bits, exactly (a truncated
// sum does not reach the next integer); the bytes of negative values are negated
// together.  A NaN (sign clear: the product's) gives 127, as the clamp of kvq_code does.
__device__ __forceinline__ uint32_t kvq_code4(float4 x, float inv) {
    const float y[4] = {__fmul_rn(x.x, inv), __fmul_rn(x.y, inv), __fmul_rn(x.z, inv), __fmul_rn(x.w, inv)};
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        u[i] = __float_as_uint(__fadd_rz(__fadd_rz(fminf(127.0f, fabsf(y[i])), 0.5f), 8388608.0f));
    const uint32_t v = __byte_perm(__byte_perm(u[0], u[1], 0x0040u), __byte_perm(u[2], u[3], 0x0040u), 0x5410u);
    // 0xFF where the value is negative (the top bytes' sign bits, replicated)
    auto sign = [](float a, float b) {
        uint32_t r;
        asm("prmt.b32 %0, %1, %2, 0x00fb;" : "=r"(r) : "r"(__float_as_uint(a)), "r"(__float_as_uint(b)));
        return r;
    };
    const uint32_t m = __byte_perm(sign(y[0], y[1]), sign(y[2], y[3]), 0x5410u);
    const uint32_t n = v ^ m;   // per byte n - m, no borrow between bytes: v is at most 127
    return ((n | 0x80808080u) - (m & 0x7F7F7F7Fu)) ^ ((n ^ ~m) & 0x80808080u);
}
__device__ __forceinline__ float4 i8x4_to_f4(uint32_t w) {
    return make_float4(static_cast<float>(static_cast<int8_t>(w)), static_cast<float>(static_cast<int8_t>(w >> 8)),
                       static_cast<float>(static_cast<int8_t>(w >> 16)), static_cast<float>(static_cast<int8_t>(w >> 24)));
}
// max |x|, a NaN never the max (fmaxf returns the other operand), as std::max skips it.
__device__ __forceinline__ float absmax4(float4 x, float m) {
    return fmaxf(fmaxf(fmaxf(fmaxf(m, fabsf(x.x)), fabsf(x.y)), fabsf(x.z)), fabsf(x.w));
}

struct KvIoParams {
    KvView kv;
    KvRuns runs;
    const void* k_in;    // store: [n][kv_heads * hd], rows ld elements apart
    const void* v_in;
    void* k_out;         // load: the same, written
    void* v_out;
    uint64_t ld_k, ld_v;
    uint32_t wide;       // every row of four elements is aligned for one vector access
};

constexpr uint32_t kKvIoThreads = 256;

// Cache row of the runs' row t, by the whole warp; *slot its slot.  -1: none (padding,
// behind the last run, outside the slot, or, for a store, written by a later run too:
// the last run wins, as if the runs were stored one after another).
template <bool STORE>
__device__ __forceinline__ int64_t place_row(const KvRuns& r, const KvView& kv, int32_t t, uint32_t* slot) {
    const uint32_t lane = threadIdx.x & 31u;
    const int32_t b = find_run(r, t);
    if (b < 0) return -1;
    const int32_t lo = run_begin(r, b), hi = r.cu ? r.cu[b + 1] : lo + 1, s = r.slots[b], first = r.firsts[b];
    if (s == -1 || t < lo || t >= hi) return -1;   // padding, or an unsorted cu
    const int64_t at = static_cast<int64_t>(first) + (t - lo);
    if (s < 0 || static_cast<uint32_t>(s) >= kv.slots || first < 0 || at >= static_cast<int64_t>(kv.rows)) {
        if (lane == 0u) raise_error(kErrBadLaunch);
        return -1;
    }
    if constexpr (STORE) {
        bool hit = false;
        for (uint32_t j = static_cast<uint32_t>(b) + 1u + lane; j < r.count; j += 32u) {
            if (r.slots[j] != s) continue;
            const int64_t f = r.firsts[j], len = r.cu ? static_cast<int64_t>(r.cu[j + 1]) - r.cu[j] : 1;
            hit |= f >= 0 && at >= f && at < f + len;
        }
        if (__any_sync(0xFFFFFFFFu, hit)) return -1;
    }
    *slot = static_cast<uint32_t>(s);
    return at;
}

// A warp has one row's next kKvIoHeads x HPW heads (blockIdx.y: which): a group of
// LPH lanes has one head, QUADS times four elements a lane.  A store's values are
// loaded before its row is looked up, so that the two latencies overlap; there is no
// loop around it: enough warps are resident to keep some 100 KB an SM in flight.
// Measured on a B200: 8 runs of about 1500 rows, 8 heads of 128, f32, stored and
// loaded: 49.7 us, 4.84 TB/s of reads and writes together; one row a sequence, 32
// sequences: 5.3 us, the latency of two launches.
constexpr uint32_t kKvIoHeads = 4;

template <typename T, bool STORE, uint32_t LPH, uint32_t QUADS>
__global__ void __launch_bounds__(kKvIoThreads) kv_io_kernel(const __grid_constant__ KvIoParams p) {
    constexpr uint32_t HPW = 32u / LPH, N = QUADS == 1u ? kKvIoHeads : kKvIoHeads / 2u;
    const KvView& kv = p.kv;
    const uint32_t lane = threadIdx.x & 31u, hd = kv.hd, l = lane % LPH;
    const uint32_t t = blockIdx.x * (kKvIoThreads / 32u) + (threadIdx.x >> 5);
    if (t >= p.runs.n) return;
    const uint32_t h0 = blockIdx.y * (N * HPW) + lane / LPH;   // this lane's first head; HPW apart
    const uint64_t io_k = static_cast<uint64_t>(t) * p.ld_k, io_v = static_cast<uint64_t>(t) * p.ld_v;
    uint32_t slot = 0;
    if constexpr (STORE) {
        float4 x[2][N][QUADS];
        auto load = [&](bool wide) {
#pragma unroll
            for (uint32_t n = 0; n < N; ++n)
#pragma unroll
                for (uint32_t i = 0; i < QUADS; ++i) {
                    const uint32_t h = h0 + n * HPW, d = 4u * (l + i * LPH);
                    const bool in = h < kv.kv_heads && d < hd;
                    const uint64_t at = static_cast<uint64_t>(h) * hd + d;
                    x[0][n][i] = in ? load4(static_cast<const T*>(p.k_in) + io_k + at, wide) : make_float4(0.f, 0.f, 0.f, 0.f);
                    x[1][n][i] = in ? load4(static_cast<const T*>(p.v_in) + io_v + at, wide) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
        };
        if (p.wide) load(true);
        else load(false);
        const int64_t at = place_row<true>(p.runs, kv, static_cast<int32_t>(t), &slot);
        if (at < 0) return;
        const uint64_t idx0 = (static_cast<uint64_t>(slot) * kv.slot_rows + static_cast<uint64_t>(at)) * kv.kv_heads;
        // the largest of each of the 2 N rows of this lane's group; one lane a row divides
        float most[2u * N], mine = 0.0f;
#pragma unroll
        for (uint32_t k = 0; k < 2u * N; ++k) {
            float m = 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < QUADS; ++i) m = absmax4(x[k & 1u][k >> 1][i], m);
            if constexpr (LPH == 32u) {
                m = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(m)));
            } else {
#pragma unroll
                for (uint32_t o = LPH / 2u; o > 0u; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
            }
            most[k] = m;
            if (l == k % LPH) mine = m;
        }
        constexpr bool kShare = LPH >= 2u * N;   // lanes enough for one row each
        const float my_scale = kShare ? __fdiv_rn(mine, 127.0f) : 0.0f;
        const float my_inv = kShare && my_scale > 0.0f ? __fdiv_rn(1.0f, my_scale) : 0.0f;
#pragma unroll
        for (uint32_t k = 0; k < 2u * N; ++k) {
            const uint32_t h = h0 + (k >> 1) * HPW;
            float scale, inv;
            if constexpr (kShare) {
                scale = __shfl_sync(0xFFFFFFFFu, my_scale, (lane - l) + k);
                inv = __shfl_sync(0xFFFFFFFFu, my_inv, (lane - l) + k);
            } else {
                scale = __fdiv_rn(most[k], 127.0f);
                inv = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
            }
            if (h >= kv.kv_heads) continue;
            int8_t* codes = ((k & 1u) ? kv.v : kv.k) + (idx0 + h) * hd;
#pragma unroll
            for (uint32_t i = 0; i < QUADS; ++i) {
                const uint32_t d = 4u * (l + i * LPH);
                if (d < hd) *reinterpret_cast<uint32_t*>(codes + d) = kvq_code4(x[k & 1u][k >> 1][i], inv);
            }
            if (l == 0u) ((k & 1u) ? kv.vs : kv.ks)[idx0 + h] = scale;
        }
    } else {
        const int64_t at = place_row<false>(p.runs, kv, static_cast<int32_t>(t), &slot);
        if (at < 0) return;
        const uint64_t idx0 = (static_cast<uint64_t>(slot) * kv.slot_rows + static_cast<uint64_t>(at)) * kv.kv_heads;
        uint32_t w[2][N][QUADS];
        float sc[2][N];
#pragma unroll
        for (uint32_t n = 0; n < N; ++n) {
            const uint32_t h = h0 + n * HPW;
            const bool on = h < kv.kv_heads;
            sc[0][n] = on ? kv.ks[idx0 + h] : 0.0f;
            sc[1][n] = on ? kv.vs[idx0 + h] : 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < QUADS; ++i) {
                const uint32_t d = 4u * (l + i * LPH);
                w[0][n][i] = on && d < hd ? *reinterpret_cast<const uint32_t*>(kv.k + (idx0 + h) * hd + d) : 0u;
                w[1][n][i] = on && d < hd ? *reinterpret_cast<const uint32_t*>(kv.v + (idx0 + h) * hd + d) : 0u;
            }
        }
#pragma unroll
        for (uint32_t n = 0; n < N; ++n) {
            const uint32_t h = h0 + n * HPW;
#pragma unroll
            for (uint32_t s = 0; s < 2u; ++s)
#pragma unroll
                for (uint32_t i = 0; i < QUADS; ++i) {
                    const uint32_t d = 4u * (l + i * LPH);
                    if (h >= kv.kv_heads || d >= hd) continue;
                    const float4 c = i8x4_to_f4(w[s][n][i]);
                    const float f = sc[s][n];
                    T* dst = static_cast<T*>(s ? p.v_out : p.k_out) + (s ? io_v : io_k) + static_cast<uint64_t>(h) * hd + d;
                    store4(dst, make_float4(__fmul_rn(c.x, f), __fmul_rn(c.y, f), __fmul_rn(c.z, f), __fmul_rn(c.w, f)), p.wide);
                }
        }
    }
}

}  // namespace qraf_dev
