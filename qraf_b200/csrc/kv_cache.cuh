// kv_cache.cuh — the int8 KV cache as an operator of its own: rows of K and V are
// quantised as they are written (qraf_cuda_kv_store) and read back as numbers
// (qraf_cuda_kv_load).  The codes and scales are those of the reference's
// QuantizedKVCache (include/nn/kv_cache_quant.h:61-94) and of the decoder's int8
// cache: per (row, KV head) scale = max |x| / 127, code = clamp(round(x / scale)).
//
// New rows come in runs: rows cu[b] .. cu[b + 1] of the input belong to
// consecutive cache rows starts[b], starts[b] + 1, ... of slot slots[b], so that
// one call takes one token of every sequence, a prompt, or drafts of uneven
// lengths.  Both directions are bound by memory: nothing is read twice, and a
// warp has two to four 512-byte rows in flight.
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
__device__ __forceinline__ uint32_t kvq_code4(float4 x, float inv) {
    return static_cast<uint32_t>(static_cast<uint8_t>(kvq_code(x.x, inv))) |
           static_cast<uint32_t>(static_cast<uint8_t>(kvq_code(x.y, inv))) << 8 |
           static_cast<uint32_t>(static_cast<uint8_t>(kvq_code(x.z, inv))) << 16 |
           static_cast<uint32_t>(static_cast<uint8_t>(kvq_code(x.w, inv))) << 24;
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

// Where row t of the runs lives, kept from row to row of one warp.
struct RunCursor {
    int32_t b = -1, lo = 0, hi = 0;   // the run that covers [lo, hi), or none there (b = -1)
    int32_t slot = -1, first = 0;
    bool bad = false, shared = false;   // shared: a later run writes rows of the same slot

    // The whole warp calls with one t.
    __device__ __forceinline__ void seek(const KvRuns& r, const KvView& kv, int32_t t, bool stores) {
        if (t >= lo && t < hi) return;
        b = find_run(r, t);
        slot = -1;
        bad = shared = false;
        if (b < 0) {
            lo = t;
            hi = t + 1;
            return;
        }
        lo = run_begin(r, b);
        hi = r.cu ? r.cu[b + 1] : lo + 1;
        if (t >= hi) {   // an unsorted cu
            lo = t;
            hi = t + 1;
            b = -1;
            return;
        }
        first = r.firsts[b];
        const int32_t s = r.slots[b];
        if (s == -1) return;   // a padding run
        // the rows past the slot's end are left out one by one; a run that starts outside is bad
        bad = s < 0 || static_cast<uint32_t>(s) >= kv.slots || first < 0 || static_cast<uint32_t>(first) >= kv.rows ||
              static_cast<int64_t>(first) + (hi - lo) > static_cast<int64_t>(kv.rows);
        if (s < 0 || static_cast<uint32_t>(s) >= kv.slots || first < 0) return;
        slot = s;
        if (stores) {
            bool hit = false;
            for (uint32_t j = b + 1u + (threadIdx.x & 31u); j < r.count; j += 32u) hit |= r.slots[j] == s;
            shared = __any_sync(0xFFFFFFFFu, hit);
        }
    }
    // Cache row of row t, or -1: outside the slot, or written by a later run (the
    // last run wins, as if the runs were stored one after another).
    __device__ __forceinline__ int64_t row(const KvRuns& r, const KvView& kv, int32_t t) const {
        if (slot < 0) return -1;
        const int64_t at = static_cast<int64_t>(first) + (t - lo);
        if (at >= static_cast<int64_t>(kv.rows)) return -1;
        if (shared) {
            bool hit = false;
            for (uint32_t j = static_cast<uint32_t>(b) + 1u + (threadIdx.x & 31u); j < r.count; j += 32u) {
                if (r.slots[j] != slot) continue;
                const int64_t f = r.firsts[j], len = r.cu ? static_cast<int64_t>(r.cu[j + 1]) - r.cu[j] : 1;
                hit |= f >= 0 && at >= f && at < f + len;
            }
            if (__any_sync(0xFFFFFFFFu, hit)) return -1;
        }
        return at;
    }
};

// Warp tasks are (row, group of HPW heads); a group of LPH lanes has one head,
// QUADS times four elements a lane.  Consecutive tasks go to one warp, so that a
// warp looks its run up once.
template <typename T, bool STORE, uint32_t LPH, uint32_t QUADS>
__global__ void __launch_bounds__(kKvIoThreads) kv_io_kernel(const KvIoParams p) {
    constexpr uint32_t HPW = 32u / LPH;
    const KvView& kv = p.kv;
    const uint32_t lane = threadIdx.x & 31u, hd = kv.hd;
    const uint32_t groups = (kv.kv_heads + HPW - 1u) / HPW;
    const uint64_t tasks = static_cast<uint64_t>(p.runs.n) * groups;
    const uint64_t warps = static_cast<uint64_t>(gridDim.x) * (kKvIoThreads / 32u);
    const uint64_t w = static_cast<uint64_t>(blockIdx.x) * (kKvIoThreads / 32u) + (threadIdx.x >> 5);
    const uint64_t per = (tasks + warps - 1u) / warps;
    const uint64_t t0 = w * per, t1 = min(tasks, t0 + per);
    RunCursor cur;
    for (uint64_t task = t0; task < t1; ++task) {
        const int32_t t = static_cast<int32_t>(task / groups);
        const uint32_t g = static_cast<uint32_t>(task - static_cast<uint64_t>(t) * groups);
        cur.seek(p.runs, kv, t, STORE);
        if (cur.bad && lane == 0u) raise_error(kErrBadLaunch);
        const int64_t at = cur.row(p.runs, kv, t);
        if (at < 0) continue;
        const uint32_t h = g * HPW + lane / LPH, l = lane % LPH;
        const bool on = h < kv.kv_heads;
        const uint64_t idx = (static_cast<uint64_t>(cur.slot) * kv.slot_rows + static_cast<uint64_t>(at)) * kv.kv_heads + h;
        const uint64_t io_k = static_cast<uint64_t>(t) * p.ld_k + static_cast<uint64_t>(h) * hd;
        const uint64_t io_v = static_cast<uint64_t>(t) * p.ld_v + static_cast<uint64_t>(h) * hd;
        if constexpr (STORE) {
            float4 x[2][QUADS];
            float m[2] = {0.0f, 0.0f};
#pragma unroll
            for (uint32_t i = 0; i < QUADS; ++i) {
                const uint32_t d = 4u * (l + i * LPH);
                const bool in = on && d < hd;
                x[0][i] = in ? load4(static_cast<const T*>(p.k_in) + io_k + d, p.wide) : make_float4(0.f, 0.f, 0.f, 0.f);
                x[1][i] = in ? load4(static_cast<const T*>(p.v_in) + io_v + d, p.wide) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (uint32_t s = 0; s < 2u; ++s) {
#pragma unroll
                for (uint32_t i = 0; i < QUADS; ++i) m[s] = absmax4(x[s][i], m[s]);
#pragma unroll
                for (uint32_t o = LPH / 2u; o > 0u; o >>= 1) m[s] = fmaxf(m[s], __shfl_xor_sync(0xFFFFFFFFu, m[s], o));
                const float scale = __fdiv_rn(m[s], 127.0f);
                const float inv = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
                int8_t* codes = (s ? kv.v : kv.k) + idx * hd;
                if (on) {
#pragma unroll
                    for (uint32_t i = 0; i < QUADS; ++i) {
                        const uint32_t d = 4u * (l + i * LPH);
                        if (d < hd) *reinterpret_cast<uint32_t*>(codes + d) = kvq_code4(x[s][i], inv);
                    }
                    if (l == 0u) (s ? kv.vs : kv.ks)[idx] = scale;
                }
            }
        } else if (on) {
            const float ks = kv.ks[idx], vs = kv.vs[idx];
            uint32_t w4[2][QUADS];
#pragma unroll
            for (uint32_t i = 0; i < QUADS; ++i) {
                const uint32_t d = 4u * (l + i * LPH);
                w4[0][i] = d < hd ? *reinterpret_cast<const uint32_t*>(kv.k + idx * hd + d) : 0u;
                w4[1][i] = d < hd ? *reinterpret_cast<const uint32_t*>(kv.v + idx * hd + d) : 0u;
            }
#pragma unroll
            for (uint32_t i = 0; i < QUADS; ++i) {
                const uint32_t d = 4u * (l + i * LPH);
                if (d >= hd) continue;
                const float4 a = i8x4_to_f4(w4[0][i]), b = i8x4_to_f4(w4[1][i]);
                store4(static_cast<T*>(p.k_out) + io_k + d,
                       make_float4(__fmul_rn(a.x, ks), __fmul_rn(a.y, ks), __fmul_rn(a.z, ks), __fmul_rn(a.w, ks)), p.wide);
                store4(static_cast<T*>(p.v_out) + io_v + d,
                       make_float4(__fmul_rn(b.x, vs), __fmul_rn(b.y, vs), __fmul_rn(b.z, vs), __fmul_rn(b.w, vs)), p.wide);
            }
        }
    }
}

}  // namespace qraf_dev
