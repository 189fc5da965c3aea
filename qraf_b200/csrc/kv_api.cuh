// kv_api.cuh — the C entries of the KV-cache operators (kv_cache.cuh,
// kv_attention.cuh) and of the sampling operators (sampling.cuh): argument checks,
// launch plans, launches.  Included once, near the end of capi.cu.
#pragma once

namespace {

int check_kv(const qraf_kv_t* kv, const char* what, int cur) {
    if (!kv) return fail(QRAF_ERR_INVALID, "%s is NULL", what);
    if (!kv->k || !kv->v || !kv->k_scale || !kv->v_scale || kv->slots == 0 || kv->rows == 0 || kv->kv_heads == 0 ||
        kv->head_dim == 0)
        return fail(QRAF_ERR_INVALID, "%s is not a cache made by qraf_cuda_kv_wrap", what);
    if (kv->device != cur)
        return fail(QRAF_ERR_INVALID, "%s lives on device %d, the current device is %d", what, kv->device, cur);
    return QRAF_OK;
}

KvView view_of(const qraf_kv_t& kv) {
    KvView v;
    v.k = kv.k;
    v.v = kv.v;
    v.ks = kv.k_scale;
    v.vs = kv.v_scale;
    v.slot_rows = kv.slot_rows;
    v.slots = kv.slots;
    v.rows = kv.rows;
    v.kv_heads = kv.kv_heads;
    v.hd = kv.head_dim;
    return v;
}

uint32_t type_bytes(uint32_t type) { return type == QRAF_TYPE_F32 ? 4u : 2u; }
bool known_type(uint32_t type) { return type == QRAF_TYPE_F32 || type == QRAF_TYPE_F16 || type == QRAF_TYPE_BF16; }

// Whether every four elements of rows `ld` elements apart can be one access.
bool wide_rows(const void* p, uint64_t ld, uint32_t type) {
    const uint64_t quad = 4u * type_bytes(type);
    return reinterpret_cast<uintptr_t>(p) % quad == 0 && ld % 4u == 0;
}
bool element_aligned(const void* p, uint32_t type) { return reinterpret_cast<uintptr_t>(p) % type_bytes(type) == 0; }

int check_runs(const int32_t* slots, const int32_t* firsts, uint32_t count, uint32_t n, const int32_t* cu) {
    if (!slots || !firsts) return fail(QRAF_ERR_INVALID, "slots or starts / lens is NULL");
    if (!cu && count != n) return fail(QRAF_ERR_INVALID, "%u runs and %u rows without cu: one row a run", count, n);
    if (n > 0x7FFFFFFFu || count > 0x7FFFFFFEu) return fail(QRAF_ERR_UNSUPPORTED, "more than 2^31 - 1 rows or runs");
    return QRAF_OK;
}

template <typename T, bool STORE>
void (*kv_io_pick(uint32_t hd))(const KvIoParams) {
    // lanes per head: the quads of a head rounded up to a power of two
    if (hd <= 16u) return kv_io_kernel<T, STORE, 4, 1>;
    if (hd <= 32u) return kv_io_kernel<T, STORE, 8, 1>;
    if (hd <= 64u) return kv_io_kernel<T, STORE, 16, 1>;
    if (hd <= 128u) return kv_io_kernel<T, STORE, 32, 1>;
    return kv_io_kernel<T, STORE, 32, 2>;
}
template <bool STORE>
void (*kv_io_pick(uint32_t type, uint32_t hd))(const KvIoParams) {
    if (type == QRAF_TYPE_F32) return kv_io_pick<float, STORE>(hd);
    if (type == QRAF_TYPE_F16) return kv_io_pick<__half, STORE>(hd);
    return kv_io_pick<__nv_bfloat16, STORE>(hd);
}

int kv_io(const qraf_kv_t* kv, const void* k, const void* v, uint32_t type, uint64_t ld_k, uint64_t ld_v, uint32_t n,
          const int32_t* slots, const int32_t* starts, const int32_t* cu, uint32_t count, bool store, cudaStream_t st) {
    DeviceInfo* dev = nullptr;
    int cur = 0;
    if (!known_type(type)) return fail(QRAF_ERR_UNSUPPORTED, "type %u is not F32 (0), F16 (1) or BF16 (2)", type);
    if (n == 0 || count == 0) return QRAF_OK;
    int rc = check_runs(slots, starts, count, n, cu);
    if (rc) return rc;
    if (!k || !v) return fail(QRAF_ERR_INVALID, "k or v is NULL");
    if (!element_aligned(k, type) || !element_aligned(v, type))
        return fail(QRAF_ERR_INVALID, "k or v is not aligned to its element type");
    if (!kv) return fail(QRAF_ERR_INVALID, "the cache is NULL");
    const uint64_t row = static_cast<uint64_t>(kv->kv_heads) * kv->head_dim;
    if (n > 1 && (ld_k < row || ld_v < row))
        return fail(QRAF_ERR_INVALID, "rows of %llu elements do not fit row strides of %llu and %llu",
                    static_cast<unsigned long long>(row), static_cast<unsigned long long>(ld_k),
                    static_cast<unsigned long long>(ld_v));
    rc = ensure_device(&cur, &dev);
    if (rc) return rc;
    rc = check_kv(kv, "the cache", cur);
    if (rc) return rc;
    KvIoParams p{};
    p.kv = view_of(*kv);
    p.runs = {slots, starts, cu, count, n};
    p.k_in = k;
    p.v_in = v;
    p.k_out = const_cast<void*>(k);
    p.v_out = const_cast<void*>(v);
    p.ld_k = ld_k;
    p.ld_v = ld_v;
    p.wide = wide_rows(k, ld_k, type) && wide_rows(v, ld_v, type);
    const uint32_t hd = kv->head_dim;
    const uint32_t hpw = hd <= 16u ? 8u : hd <= 32u ? 4u : hd <= 64u ? 2u : 1u;
    const uint32_t heads = hpw * (hd > 128u ? kKvIoHeads / 2u : kKvIoHeads);   // of one row a warp
    const dim3 grid((n + kKvIoThreads / 32u - 1u) / (kKvIoThreads / 32u), (kv->kv_heads + heads - 1u) / heads);
    void (*kernel)(const KvIoParams) = store ? kv_io_pick<true>(type, hd) : kv_io_pick<false>(type, hd);
    (kernel<<<grid, kKvIoThreads, 0, st>>>(p), count_launch());
    QRAF_CUDA_TRY(cudaGetLastError());
    return QRAF_OK;
}

// Whether the prefix goes to kv_prefix_kernel's tiles of 128 rows x 128 keys, or to
// kv_attention_kernel's of 16 rows.  Measured on a B200 (us a call, tiles / by 16; heads of
// 128, 64 own rows): 2 KV heads, 8 rows, 8192 keys 19 / 25; 64 rows, 32768 keys 36 / 49; 8 KV
// heads, 64 rows, 8192 keys 35 / 40; but 8 KV heads, 32 rows, 8192 keys 34 / 27, where most of
// a tile's rows are empty and there are many tiles.
bool prefix_on_tiles(uint64_t rows, uint64_t kv_heads, uint32_t hd, uint64_t prefix_len, int sm_count) {
    const uint64_t tiles = (rows + kPreRows - 1u) / kPreRows * kv_heads * ((prefix_len + kPreKeys - 1u) / kPreKeys);
    return hd <= 128u && prefix_len >= kPreKeys && tiles < (1ull << 31) &&
           (rows >= 48u || tiles <= 3ull * static_cast<uint64_t>(sm_count));
}

struct KvaPlan {
    uint32_t row_tiles = 0, p_chunks = 0, p_chunk = 0, own_tiles = 0, splits = 0, own_wide = 0, pre_ctas = 0;
    uint32_t pre_base = 0, pre_extra = 0;
    uint32_t cluster = 0;   // CTAs of a cluster: kv_attention_cluster_kernel has the call
    uint64_t items = 0, part_bytes = 0;   // part_bytes: the workspace, records and
    uint64_t sum_at = 0;                  // from this byte of it kv_prefix_kernel's sums (0: none)
};

// How a call's rows and keys are cut.  Items of a few hundred keys keep the warps that run
// at once evenly busy; every chunk more costs each row one record of (head_dim + 4) floats,
// written and read once.
int plan_kva(uint32_t n, uint32_t heads, uint32_t kv_heads, uint32_t hd, uint32_t prefix_len, uint32_t count, bool ragged,
             uint32_t max_len, int sm_count, KvaPlan* pl) {
    const uint64_t G = heads / kv_heads, rows = static_cast<uint64_t>(n) * G;
    if (rows > 0x7FFFFFFFull / 16u || static_cast<uint64_t>(n) * heads > 0x7FFFFFFFull)
        return fail(QRAF_ERR_UNSUPPORTED, "%u new rows of %u heads are too many for one call", n, heads);
    {   // kv_attention_cluster_kernel
        const bool wide = ragged ? rows > 8ull * std::min(count, n) : G > 8u;
        const uint64_t R = wide ? 16u : 8u, keys = hd > 128u ? 16u : 32u;
        const uint64_t tiles = ragged ? (rows + static_cast<uint64_t>(std::min(count, n)) * (R - 1u)) / R
                                      : static_cast<uint64_t>(count) * ((G + R - 1u) / R);
        const uint64_t equal = ragged ? std::max<uint64_t>({1, rows / R, std::min(count, n)}) : tiles;   // for runs of equal lengths
        const uint64_t steps = (prefix_len + keys - 1u) / keys + (max_len + keys - 1u) / keys;
        const uint64_t groups = equal * kv_heads, sms = static_cast<uint64_t>(sm_count);
        const uint64_t room = wide && hd > 128u ? sms : 2u * sms;   // CTAs that run at once: 132 KB of shared memory, or up to 100
        uint32_t cl = 1;
        while (cl < 8u && steps > 4u * cl && 2u * cl * groups <= room) cl *= 2;   // a step a warp
        // One launch where every cluster runs at once and the warps' shares are short.  A prefix is
        // read for every tile of rows here; own rows alone go on longer where the clusters leave
        // no SM empty.  Measured on a B200 (us a call, cluster / the other kernels; 8 query heads a
        // KV head of 128): behind a prefix, 2 KV heads, 64 sequences of 64 own rows behind 512
        // 12 / 19, behind 2048 24 / 24; 16 behind 8192 25 / 22.  Own rows alone, 2 KV heads, one
        // sequence of 512 8.0 / 8.8, of 1024 9.2 / 10.2, of 2048 11.0 / 8.9, of 131072 229 / 32; 4 runs
        // of 5 tokens (160 CTAs) of 8192 36 / 39, of 32768 104 / 95; 8 KV heads, 16 sequences (256
        // CTAs) of 2048 25.9 / 27.6, of 4096 44.4 / 42.8, of 131072 1140 / 965; 4 sequences (256 CTAs)
        // of 1024 10.9 / 11.4, of 8192 27.6 / 24.5 (of 1024 where 32768 are allowed 11.0 / 12.3).  Heads
        // of 256, 2 KV heads, 16 sequences (256 CTAs) of 1024 17.2 / 18.0, of 2048 22.1 / 19.6.
        const uint64_t a_warp = (steps + 4u * cl - 1u) / (4u * cl), share = a_warp * keys;
        const bool brief = prefix_len ? a_warp <= 8u : share <= (hd <= 128u && groups * cl >= sms ? 256u : 32u);
        if (groups * cl <= room && brief) {
            pl->own_wide = wide;
            pl->own_tiles = static_cast<uint32_t>(tiles);
            pl->cluster = cl;
            pl->items = tiles * kv_heads * cl;
            return QRAF_OK;
        }
    }
    const bool tiles = prefix_len && prefix_on_tiles(rows, kv_heads, hd, prefix_len, sm_count);
    // rows by 16: wherever the prefix is among the kernel's items (it is read once for every
    // tile of rows), or where a sequence's own rows do not fit 8
    pl->own_wide = (prefix_len && !tiles) || (ragged ? rows > 8ull * std::min(count, n) : G > 8u);
    const uint32_t R = pl->own_wide ? 16u : 8u;
    const uint64_t own_tiles = ragged ? (rows + static_cast<uint64_t>(std::min(count, n)) * (R - 1u)) / R
                                      : static_cast<uint64_t>(count) * ((G + R - 1u) / R);
    // Warps (CTAs) to fill: what the chunk counts below were measured with, not the kernels'
    // residency, which by registers and shared memory is 16 an SM (tiles of 16 rows: 12) for heads up
    // to 64, 10 (8) up to 128 and 8 (6) above.
    const uint64_t slots = (pl->own_wide || hd > 128u ? 8ull : 11ull) * static_cast<uint64_t>(sm_count);
    uint64_t items = 0;
    if (max_len) {
        // About one round of them, counting the tiles that runs of equal lengths would have:
        // the nearest whole number of chunks, or behind kv_prefix_kernel, whose SMs come free one
        // by one, the next larger.  Measured on a B200 (us a call, 3 / 4 chunks; 64 sequences, 8 KV
        // heads of 128): own rows up to 1024 37.5 / 39.9, up to 4096 106.3 / 108.5; up to 1024
        // behind a prefix of 8192 92.8 / 86.3.
        const uint64_t groups = std::max<uint64_t>({1, rows / R, std::min(count, n)}) * kv_heads;
        const uint64_t by_len = (max_len + kKvaMinChunk - 1ull) / kKvaMinChunk;
        const uint64_t round = tiles ? slots + groups - 1u : slots + groups / 2u;
        pl->splits = static_cast<uint32_t>(std::max<uint64_t>(1, std::min<uint64_t>({round / groups, by_len, kKvaMaxChunks / 2u})));
        items += own_tiles * kv_heads * pl->splits;
    }
    pl->own_tiles = static_cast<uint32_t>(own_tiles);
    if (tiles) {
        pl->row_tiles = static_cast<uint32_t>((rows + kPreRows - 1u) / kPreRows);
        const uint32_t T = (prefix_len + kPreKeys - 1u) / kPreKeys, work = pl->row_tiles * kv_heads * T;
        // One CTA an SM, each with two tiles at least (its two warpgroups).  Beginning and
        // ending a stretch of one unit takes about as long as 2.5 tiles, so ranges that
        // meet two units are worth it only where whole numbers of CTAs a unit would be
        // much longer.
        const uint32_t units = pl->row_tiles * kv_heads, sms = static_cast<uint32_t>(sm_count);
        pl->pre_ctas = std::min(std::max(1u, (work + 1u) / 2u), sms);
        if (units <= sms) {
            const uint32_t per = std::max(1u, std::min(sms / units, (T + 1u) / 2u));
            const uint32_t alone = 2u * ((T + per - 1u) / per) + 5u, shared = 2u * ((work + pl->pre_ctas - 1u) / pl->pre_ctas) + 10u;
            if (alone <= shared) pl->pre_ctas = units * per;
        }
        pl->pre_base = work / pl->pre_ctas;
        pl->pre_extra = work % pl->pre_ctas;
        // a unit's T tiles may start inside one CTA's range and end inside another's
        pl->p_chunks = std::min({T, pl->pre_ctas, (T + pl->pre_base - 1u) / pl->pre_base + 1u});
        if (pl->p_chunks > kKvaMaxChunks / 2u) return fail(QRAF_ERR_UNSUPPORTED, "a GPU of %d SMs cuts the prefix too finely", sm_count);
    } else if (prefix_len) {
        pl->row_tiles = static_cast<uint32_t>((rows + 15u) / 16u);
        const uint64_t units = static_cast<uint64_t>(pl->row_tiles) * kv_heads;
        const uint64_t by_len = (prefix_len + kKvaMinChunk - 1ull) / kKvaMinChunk;
        uint64_t chunks = std::max<uint64_t>(
            1, std::min<uint64_t>({(slots + units - 1) / units, by_len, kKvaMaxChunks / 2u}));
        pl->p_chunk = static_cast<uint32_t>(((prefix_len + chunks - 1) / chunks + 31u) & ~31ull);
        pl->p_chunks = (prefix_len + pl->p_chunk - 1u) / pl->p_chunk;
        items += units * pl->p_chunks;
    }
    if (items > 0x7FFFFFFFull) return fail(QRAF_ERR_UNSUPPORTED, "the call has too many work items");
    if (items == 0 && !pl->pre_ctas) {
        pl->splits = 1;   // no keys at all: one item a row tile writes the zeros
        items = own_tiles * kv_heads;
    }
    pl->items = items;
    if (pl->p_chunks + pl->splits > 1u || pl->pre_ctas)
        pl->part_bytes = static_cast<uint64_t>(n) * heads * (pl->p_chunks + pl->splits) * (hd + 4u) * sizeof(float);
    if (pl->pre_ctas && pl->pre_base + (pl->pre_extra ? 1u : 0u) > kPreTerm) {
        pl->sum_at = pl->part_bytes;
        pl->part_bytes += static_cast<uint64_t>(pl->pre_ctas) * kPreRows * (hd <= 64u ? 64u : 128u) * sizeof(float);
    }
    return QRAF_OK;
}

template <typename K>
cudaError_t launch_kv(K kernel, uint64_t grid, uint32_t threads, uint32_t smem, bool dependent, const KvAttnParams& p,
                      cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent ? 1 : 0;
    return counted(cudaLaunchKernelEx(&cfg, kernel, p));
}

template <uint32_t HDP, bool WIDE>
cudaError_t launch_cluster(const KvAttnParams& p, uint64_t items, uint32_t cl, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(items));
    cfg.blockDim = dim3(32u * kKvaClusterWarps);
    cfg.dynamicSmemBytes = kKvaClusterWarps * KvaShape<HDP, WIDE>::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cl;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return counted(cudaLaunchKernelEx(&cfg, kv_attention_cluster_kernel<HDP, WIDE>, p));
}
template <uint32_t HDP>
cudaError_t launch_cluster(const KvAttnParams& p, uint64_t items, uint32_t cl, cudaStream_t st) {
    return p.own_wide ? launch_cluster<HDP, true>(p, items, cl, st) : launch_cluster<HDP, false>(p, items, cl, st);
}

template <uint32_t HDP>
cudaError_t launch_kva(const KvAttnParams& p, uint64_t items, cudaStream_t st) {
    return p.own_wide
               ? launch_kv(kv_attention_kernel<HDP, true>, items, 32u, KvaShape<HDP, true>::kSmem, p.chained != 0u, p, st)
               : launch_kv(kv_attention_kernel<HDP, false>, items, 32u, KvaShape<HDP, false>::kSmem, p.chained != 0u, p, st);
}

template <uint32_t HDP>
cudaError_t launch_prefix(const KvAttnParams& p, cudaStream_t st) {
    constexpr uint32_t one = PreShape<HDP, 1>::kSmem, two = PreShape<HDP, 2>::kSmem;
    if (p.type == QRAF_TYPE_F32) return launch_kv(kv_prefix_kernel<HDP, float>, p.pre_ctas, kPreThreads, two, false, p, st);
    if (p.type == QRAF_TYPE_F16) return launch_kv(kv_prefix_kernel<HDP, __half>, p.pre_ctas, kPreThreads, one, false, p, st);
    return launch_kv(kv_prefix_kernel<HDP, __nv_bfloat16>, p.pre_ctas, kPreThreads, one, false, p, st);
}

}  // namespace

extern "C" {

int qraf_cuda_kv_wrap(int8_t* k_dev, int8_t* v_dev, float* k_scale_dev, float* v_scale_dev, uint32_t slots, uint32_t rows,
                      uint64_t slot_rows, uint32_t kv_heads, uint32_t head_dim, qraf_kv_t* out) {
    if (!out) return fail(QRAF_ERR_INVALID, "out is NULL");
    std::memset(out, 0, sizeof(*out));
    if (!k_dev || !v_dev || !k_scale_dev || !v_scale_dev) return fail(QRAF_ERR_INVALID, "a pointer is NULL");
    if (slots == 0 || rows == 0 || kv_heads == 0) return fail(QRAF_ERR_INVALID, "slots, rows and kv_heads must be positive");
    if (head_dim == 0 || head_dim % 16u || head_dim > kKvaMaxHeadDim)
        return fail(QRAF_ERR_UNSUPPORTED, "head_dim %u: the int8 cache needs a multiple of 16, at most 256", head_dim);
    if (rows > 0x7FFFFFFFu || slots > 0x7FFFFFFFu || kv_heads > 65535u)
        return fail(QRAF_ERR_UNSUPPORTED, "more than 2^31 - 1 slots or rows, or more than 65535 KV heads");
    if (slot_rows < rows) return fail(QRAF_ERR_INVALID, "slots of %u rows overlap: %llu rows apart", rows,
                                      static_cast<unsigned long long>(slot_rows));
    if (!aligned16(k_dev) || !aligned16(v_dev) || reinterpret_cast<uintptr_t>(k_scale_dev) % 4u ||
        reinterpret_cast<uintptr_t>(v_scale_dev) % 4u)
        return fail(QRAF_ERR_INVALID, "codes must be 16-byte aligned and scales 4-byte aligned");
    cudaPointerAttributes a;
    QRAF_CUDA_TRY(cudaPointerGetAttributes(&a, k_dev));
    if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged)
        return fail(QRAF_ERR_INVALID, "the codes are not in device memory");
    out->k = k_dev;
    out->v = v_dev;
    out->k_scale = k_scale_dev;
    out->v_scale = v_scale_dev;
    out->slot_rows = slot_rows;
    out->slots = slots;
    out->rows = rows;
    out->kv_heads = kv_heads;
    out->head_dim = head_dim;
    out->device = a.device;
    return QRAF_OK;
}

int qraf_cuda_kv_store(const qraf_kv_t* kv, const void* k_dev, const void* v_dev, uint32_t type, uint64_t k_ld,
                       uint64_t v_ld, uint32_t n, const int32_t* slots_dev, const int32_t* starts_dev,
                       const int32_t* cu_dev, uint32_t count, void* stream) {
    return kv_io(kv, k_dev, v_dev, type, k_ld, v_ld, n, slots_dev, starts_dev, cu_dev, count, true,
                 static_cast<cudaStream_t>(stream));
}

int qraf_cuda_kv_load(const qraf_kv_t* kv, void* k_dev, void* v_dev, uint32_t type, uint64_t k_ld, uint64_t v_ld,
                      uint32_t n, const int32_t* slots_dev, const int32_t* starts_dev, const int32_t* cu_dev,
                      uint32_t count, void* stream) {
    return kv_io(kv, k_dev, v_dev, type, k_ld, v_ld, n, slots_dev, starts_dev, cu_dev, count, false,
                 static_cast<cudaStream_t>(stream));
}

static int kva_check(const qraf_kv_t* kv, uint32_t prefix_len, uint32_t heads, uint32_t max_len) {
    if (!kv) return fail(QRAF_ERR_INVALID, "the cache is NULL");
    if (kv->kv_heads == 0 || heads == 0 || heads % kv->kv_heads)
        return fail(QRAF_ERR_INVALID, "%u query heads are not a multiple of %u KV heads", heads, kv->kv_heads);
    if (max_len > kv->rows) return fail(QRAF_ERR_INVALID, "max_len %u exceeds the slots' %u rows", max_len, kv->rows);
    if (prefix_len > 0x7FFFFFFFu) return fail(QRAF_ERR_UNSUPPORTED, "a prefix of more than 2^31 - 1 rows");
    return QRAF_OK;
}

int qraf_cuda_kv_attention_workspace(const qraf_kv_t* kv, uint32_t prefix_len, uint32_t n, uint32_t heads, uint32_t count,
                                     int ragged, uint32_t max_len, uint64_t* bytes) {
    if (!bytes) return fail(QRAF_ERR_INVALID, "bytes is NULL");
    *bytes = 0;
    int rc = kva_check(kv, prefix_len, heads, max_len);
    if (rc || n == 0 || count == 0) return rc;
    DeviceInfo* dev = nullptr;
    rc = ensure_device(nullptr, &dev);
    if (rc) return rc;
    KvaPlan pl;
    rc = plan_kva(n, heads, kv->kv_heads, kv->head_dim, prefix_len, count, ragged != 0, max_len, dev->sm_count, &pl);
    *bytes = pl.part_bytes;
    return rc;
}

int qraf_cuda_kv_attention(const qraf_kv_t* kv, const qraf_kv_t* prefix, uint32_t prefix_slot, uint32_t prefix_len,
                           const void* q_dev, void* out_dev, uint32_t type, uint64_t q_ld, uint64_t out_ld, uint32_t n,
                           uint32_t heads, const int32_t* slots_dev, const int32_t* lens_dev, const int32_t* cu_dev,
                           uint32_t count, uint32_t max_len, float scale, void* workspace_dev, uint64_t workspace_bytes,
                           void* stream) {
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!known_type(type)) return fail(QRAF_ERR_UNSUPPORTED, "type %u is not F32 (0), F16 (1) or BF16 (2)", type);
    int rc = kva_check(kv, prefix_len, heads, max_len);
    if (rc) return rc;
    if (n == 0 || count == 0) return QRAF_OK;
    rc = check_runs(slots_dev, lens_dev, count, n, cu_dev);
    if (rc) return rc;
    if (!q_dev || !out_dev) return fail(QRAF_ERR_INVALID, "q or out is NULL");
    if (!std::isfinite(scale * 1.44269504088896340736f))
        return fail(QRAF_ERR_INVALID, "scale %g is not finite in units of log2(e)", static_cast<double>(scale));
    if (!element_aligned(q_dev, type) || !element_aligned(out_dev, type))
        return fail(QRAF_ERR_INVALID, "q or out is not aligned to its element type");
    const uint64_t row = static_cast<uint64_t>(heads) * kv->head_dim;
    if (n > 1 && (q_ld < row || out_ld < row))
        return fail(QRAF_ERR_INVALID, "rows of %llu elements do not fit row strides of %llu and %llu",
                    static_cast<unsigned long long>(row), static_cast<unsigned long long>(q_ld),
                    static_cast<unsigned long long>(out_ld));
    DeviceInfo* dev = nullptr;
    int cur = 0;
    rc = ensure_device(&cur, &dev);
    if (rc) return rc;
    rc = check_kv(kv, "the cache", cur);
    if (rc) return rc;
    KvAttnParams p{};
    p.kv = view_of(*kv);
    p.runs = {slots_dev, lens_dev, cu_dev, count, n};
    p.prefix_len = prefix_len;
    if (prefix_len) {
        rc = check_kv(prefix, "the prefix's cache", cur);
        if (rc) return rc;
        if (prefix->kv_heads != kv->kv_heads || prefix->head_dim != kv->head_dim)
            return fail(QRAF_ERR_INVALID, "the prefix has %u heads of %u, the cache %u of %u", prefix->kv_heads,
                        prefix->head_dim, kv->kv_heads, kv->head_dim);
        if (prefix_slot >= prefix->slots || prefix_len > prefix->rows)
            return fail(QRAF_ERR_INVALID, "prefix slot %u or length %u exceeds its cache (%u slots of %u rows)", prefix_slot,
                        prefix_len, prefix->slots, prefix->rows);
        const uint64_t base = static_cast<uint64_t>(prefix_slot) * prefix->slot_rows * prefix->kv_heads;
        p.pk = prefix->k + base * prefix->head_dim;
        p.pv = prefix->v + base * prefix->head_dim;
        p.pks = prefix->k_scale + base;
        p.pvs = prefix->v_scale + base;
    }
    KvaPlan pl;
    rc = plan_kva(n, heads, kv->kv_heads, kv->head_dim, prefix_len, count, cu_dev != nullptr, max_len, dev->sm_count, &pl);
    if (rc) return rc;
    if (pl.part_bytes && (!workspace_dev || workspace_bytes < pl.part_bytes || !aligned16(workspace_dev)))
        return fail(QRAF_ERR_INVALID, "the call needs a 16-byte-aligned workspace of %llu bytes, it was given %llu",
                    static_cast<unsigned long long>(pl.part_bytes),
                    static_cast<unsigned long long>(workspace_dev ? workspace_bytes : 0));
    p.q = q_dev;
    p.out = out_dev;
    p.q_ld = q_ld;
    p.out_ld = out_ld;
    p.type = type;
    p.wide = wide_rows(out_dev, out_ld, type);
    p.q_wide = wide_rows(q_dev, q_ld, type);
    p.group = heads / kv->kv_heads;
    p.heads = heads;
    p.scale_log2 = scale * 1.44269504088896340736f;
    p.max_len = max_len;
    p.row_tiles = pl.row_tiles;
    p.p_chunks = pl.p_chunks;
    p.p_chunk = pl.p_chunk;
    p.own_tiles = pl.own_tiles;
    p.splits = pl.splits;
    p.own_wide = pl.own_wide;
    p.pre_ctas = pl.pre_ctas;
    p.pre_base = pl.pre_base;
    p.pre_extra = pl.pre_extra;
    p.pre_sum = pl.sum_at ? reinterpret_cast<float*>(static_cast<uint8_t*>(workspace_dev) + pl.sum_at) : nullptr;
    p.chained = pl.pre_ctas ? 1u : 0u;
    p.part = pl.part_bytes ? static_cast<float*>(workspace_dev) : nullptr;
    const uint32_t hd = kv->head_dim;
    if (pl.cluster) {
        QRAF_CUDA_TRY(hd <= 64u ? launch_cluster<64>(p, pl.items, pl.cluster, st)
                                : hd <= 128u ? launch_cluster<128>(p, pl.items, pl.cluster, st)
                                             : launch_cluster<256>(p, pl.items, pl.cluster, st));
        return QRAF_OK;
    }
    if (p.pre_ctas) QRAF_CUDA_TRY(hd <= 64u ? launch_prefix<64>(p, st) : launch_prefix<128>(p, st));
    if (pl.items)
        QRAF_CUDA_TRY(hd <= 64u ? launch_kva<64>(p, pl.items, st)
                                : hd <= 128u ? launch_kva<128>(p, pl.items, st) : launch_kva<256>(p, pl.items, st));
    if (!p.part) return QRAF_OK;
    const uint64_t out_rows = static_cast<uint64_t>(n) * heads;
    const bool few = pl.p_chunks + pl.splits <= kJoinFew;
    QRAF_CUDA_TRY(few ? launch_kv(kv_attention_join_kernel<1>, (out_rows + kJoinWarps - 1) / kJoinWarps, kJoinThreads, 0, true, p, st)
                      : launch_kv(kv_attention_join_kernel<8>, out_rows, kJoinThreads, 0, true, p, st));
    return QRAF_OK;
}

int qraf_cuda_token_probs(const float* logits_dev, uint64_t logits_ld, float* probs_dev, uint64_t probs_ld, uint32_t rows,
                          uint32_t vocab, float temperature, void* stream) {
    if (!(temperature > 0.0f) || !std::isfinite(temperature) || !std::isfinite(1.44269504088896340736f / temperature))
        return fail(QRAF_ERR_INVALID, "temperature %g must be positive and finite", static_cast<double>(temperature));
    if (rows == 0 || vocab == 0) return QRAF_OK;
    if (!logits_dev || !probs_dev) return fail(QRAF_ERR_INVALID, "a pointer is NULL");
    if (!element_aligned(logits_dev, QRAF_TYPE_F32) || !element_aligned(probs_dev, QRAF_TYPE_F32))
        return fail(QRAF_ERR_INVALID, "logits or probs is not 4-byte aligned");
    if (vocab > 0x7FFFFFF0u) return fail(QRAF_ERR_UNSUPPORTED, "a vocabulary of more than 2^31 - 16");
    if (rows > 1 && (logits_ld < vocab || probs_ld < vocab))
        return fail(QRAF_ERR_INVALID, "rows of %u values do not fit the row strides", vocab);
    DeviceInfo* dev = nullptr;
    int rc = ensure_device(nullptr, &dev);
    if (rc) return rc;
    // CTAs per row: until a slice fits a third of an SM's shared memory, and further
    // while the SMs are not all busy and a CTA keeps 2048 values
    uint32_t cl = 1;
    auto slice_of = [&](uint32_t c) { return ((vocab + c - 1u) / c + 3u) & ~3u; };
    while (cl < kProbMaxCluster && (slice_of(cl) > kProbSlice || (static_cast<uint64_t>(rows) * cl * 2u <=
                                        static_cast<uint64_t>(dev->sm_count) && slice_of(cl) > 4096u)))
        cl *= 2;
    ProbParams p{};
    p.x = logits_dev;
    p.out = probs_dev;
    p.x_ld = logits_ld;
    p.out_ld = probs_ld;
    p.vocab = vocab;
    p.slice = slice_of(cl);
    p.scale = 1.44269504088896340736f / temperature;
    p.cached = p.slice <= kProbSliceMax;
    if (static_cast<uint64_t>(rows) * cl > 0x7FFFFFFFull) return fail(QRAF_ERR_UNSUPPORTED, "too many rows for one call");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(rows * cl);
    cfg.blockDim = dim3(kProbThreads);
    cfg.dynamicSmemBytes = p.cached ? (p.slice + 8u) * sizeof(float) : 0u;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cl;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    QRAF_CUDA_TRY(counted(cudaLaunchKernelEx(&cfg, token_probs_kernel, p)));
    return QRAF_OK;
}

int qraf_cuda_verify_drafts(const float* target_dev, uint64_t target_seq, uint64_t target_row, const float* draft_dev,
                            uint64_t draft_seq, uint64_t draft_row, const int32_t* tokens_dev, const float* u_dev,
                            const float* u_last_dev, const int32_t* counts_dev, uint32_t seqs, uint32_t drafts,
                            uint32_t vocab, int32_t* out_tokens_dev, int32_t* accepted_dev, void* stream) {
    if (drafts > kVerMaxDrafts) return fail(QRAF_ERR_UNSUPPORTED, "more than %u drafts a sequence", kVerMaxDrafts);
    if (seqs == 0) return QRAF_OK;
    if (vocab == 0) return fail(QRAF_ERR_INVALID, "the vocabulary is empty");
    if (vocab > 0x7FFF0000u) return fail(QRAF_ERR_UNSUPPORTED, "a vocabulary of more than 2^31 - 2^16");
    if (!target_dev || !u_last_dev || !out_tokens_dev || !accepted_dev || (drafts && (!draft_dev || !tokens_dev || !u_dev)))
        return fail(QRAF_ERR_INVALID, "a pointer is NULL");
    if (!element_aligned(target_dev, QRAF_TYPE_F32) || !element_aligned(draft_dev, QRAF_TYPE_F32))
        return fail(QRAF_ERR_INVALID, "target or draft is not 4-byte aligned");
    if ((drafts && target_row < vocab) || (drafts > 1 && draft_row < vocab) ||
        (seqs > 1 && (target_seq < vocab || (drafts && draft_seq < vocab))))
        return fail(QRAF_ERR_INVALID, "rows of %u values do not fit the strides", vocab);
    DeviceInfo* dev = nullptr;
    int rc = ensure_device(nullptr, &dev);
    if (rc) return rc;
    // CTAs per sequence: up to eight while there is more than 2048 values for each
    uint32_t cl = 1;
    while (cl < kVerMaxCluster && vocab > cl * 2048u) cl *= 2;
    if (static_cast<uint64_t>(seqs) * cl > 0x7FFFFFFFull) return fail(QRAF_ERR_UNSUPPORTED, "too many sequences for one call");
    VerifyParams p{};
    p.target = target_dev;
    p.draft = draft_dev;
    p.t_seq = target_seq;
    p.t_row = target_row;
    p.d_seq = draft_seq;
    p.d_row = draft_row;
    p.tokens = tokens_dev;
    p.u = u_dev;
    p.u_last = u_last_dev;
    p.counts = counts_dev;
    p.out = out_tokens_dev;
    p.accepted = accepted_dev;
    p.drafts = drafts;
    p.vocab = vocab;
    const uint32_t unit = 4u * kVerWarps;
    p.slice = ((vocab + cl - 1u) / cl + unit - 1u) / unit * unit;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(seqs * cl);
    cfg.blockDim = dim3(kVerThreads);
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cl;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    QRAF_CUDA_TRY(counted(cudaLaunchKernelEx(&cfg, verify_drafts_kernel, p)));
    return QRAF_OK;
}

}  // extern "C"
