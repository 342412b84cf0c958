// fds_window.cu - fds_window_attn_fwd: argument checks, tensor maps over
// strided q / k / v, the choice between the two kernels and of the split, and
// the launch.
#include <algorithm>

#include "capi_internal.h"
#include "window_kernel.cuh"

using namespace fds_detail;

namespace {

using fds::window::Params;

constexpr int kMaxLen = 1 << 28;

// Clusters of `split` CTAs along x, with programmatic stream serialization.
template <typename... KArgs, typename... Args>
cudaError_t launch_cluster(void (*kern)(KArgs...), dim3 grid, int block, size_t smem, int split, cudaStream_t stream,
                           Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(static_cast<unsigned>(block));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (split > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = static_cast<unsigned>(split);
        attr[n].val.clusterDim.y = 1;
        attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = static_cast<unsigned>(n);
    return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

// [batch, len, heads, 64] of any strides: boxes of `rows` rows x `pack` heads (the
// heads of a row next to each other), 128-byte swizzle, zero fill past the last row.
int make_heads_map(CUtensorMap* map, const void* base, int dtype, int heads, int len, int batch, const int64_t* stride,
                   int rows, int pack = 1) {
    EncodeTiledFn enc = encode_fn();
    if (enc == nullptr) return set_error(FDS_ERR_TENSOR_MAP, "cuTensorMapEncodeTiled unavailable from the driver");
    const cuuint64_t dims[4] = {64, static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(len),
                                static_cast<cuuint64_t>(batch)};
    // the stride of an extent of one is never used: any valid value
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(heads > 1 ? 2 * stride[2] : 128),
                                   static_cast<cuuint64_t>(len > 1 ? 2 * stride[1] : 128),
                                   static_cast<cuuint64_t>(batch > 1 ? 2 * stride[0] : 128)};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(pack), static_cast<cuuint32_t>(rows), 1};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUtensorMapDataType dt =
        dtype == FDS_DTYPE_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    CUresult r = enc(map, dt, 4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(FDS_ERR_TENSOR_MAP, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
    return FDS_OK;
}

// Keys a block of `rows` queries can see at most.
int64_t most_keys(const Params& p, int rows) {
    return std::min<int64_t>(p.k_len, static_cast<int64_t>(p.left) + p.right + rows + p.sinks);
}

// CTAs (1, 2, 4 or 8, a cluster) that a unit's tiles are dealt to: the split that
// should finish first, of those whose clusters are all resident at once. The constants
// are microseconds on a B200 (77 queries, 4 - 128 units, 2 - 24 tiles; within 10 % but
// for a few): a launch, more for a cluster's merge, and a tile of each CTA, dearer
// where CTAs share a pair of SMs, then one. E.g. 12 units: 3 tiles 8.1 us whole, 8.3
// in four; 8 tiles 13.0, 8.9 in four; 36 units: 4 tiles 9.7, 9.1 in two, 9.9 in four;
// 16 tiles 23.4, 15.5, 14.0. Eight CTAs a cluster fit up to four thirds of the SMs (36
// units of 4 tiles: 16.9 us, in two waves).
int choose_split(int64_t units, int64_t tiles, int64_t sms) {
    int best = 1;
    double best_cost = 1e30;
    for (int split = 1; split <= fds::window::kMaxSplit; split *= 2) {
        const int64_t ctas = units * split;
        if (split > 1 && ctas > (split == 8 ? sms * 4 / 3 : 2 * sms)) break;
        const int step = ctas <= sms / 2 ? 0 : (ctas <= sms ? 1 : 2);
        const double launch[] = {5.2, 5.9, 5.9}, merge[] = {1.8, 2.6, 2.8}, tile[] = {1.05, 1.43, 1.67};
        const double cost = launch[step] + (split > 1 ? merge[step] : 0.) + static_cast<double>((tiles + split - 1) / split) * tile[step];
        if (cost < best_cost) best_cost = cost, best = split;
    }
    return best;
}

template <typename T, bool kSplit>
int launch_units(const fds::window::Maps& maps, const Params& p, int batch, int split, cudaStream_t stream) {
    auto kern = fds::window::window_tile_kernel<T, kSplit>;
    constexpr int smem = fds::window::TileSmem<kSplit>::alloc;
    static std::atomic<uint64_t> smem_set{0};
    cudaError_t e = set_smem_once(kern, smem, smem_set);
    if (e != cudaSuccess) return set_error(FDS_ERR_CUDA, "cudaFuncSetAttribute(window): %s", cudaGetErrorString(e));
    const dim3 grid(static_cast<unsigned>(p.row_blocks * split), static_cast<unsigned>(p.heads / p.pack), static_cast<unsigned>(batch));
    e = launch_cluster(kern, grid, fds::window::kTileThreads, smem, split, stream, maps, p);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) return set_error(FDS_ERR_CUDA, "window attention launch: %s", cudaGetErrorString(e));
    return FDS_OK;
}

template <typename T>
int launch_tile(const FdsWindowArgs* a, Params& p, int sms, cudaStream_t stream) {
    // the heads of a key head share units, so that its keys are read once for them
    p.group = p.heads / p.kv_heads;
    p.pack = p.group <= fds::kBlockM ? p.group : 1;
    p.queries = fds::kBlockM / p.pack;
    fds::window::Maps maps;
    int rc;
    if ((rc = make_heads_map(&maps.q, a->q, a->dtype, p.heads, p.q_len, a->batch, p.q_stride, p.queries, p.pack)) != FDS_OK ||
        (rc = make_heads_map(&maps.k, a->k, a->dtype, p.kv_heads, p.k_len, a->batch, p.k_stride, fds::kBlockN)) != FDS_OK ||
        (rc = make_heads_map(&maps.v, a->v, a->dtype, p.kv_heads, p.k_len, a->batch, p.v_stride, fds::kBlockN)) != FDS_OK)
        return rc;
    // (a map costs the host a third of a microsecond: only those the launch reads)
    maps.k8 = maps.k, maps.v8 = maps.v, maps.out = maps.q;
    if (p.sinks > 0 &&
        ((rc = make_heads_map(&maps.k8, a->k, a->dtype, p.kv_heads, p.k_len, a->batch, p.k_stride, 8)) != FDS_OK ||
         (rc = make_heads_map(&maps.v8, a->v, a->dtype, p.kv_heads, p.k_len, a->batch, p.v_stride, 8)) != FDS_OK))
        return rc;
    p.row_blocks = (p.q_len + p.queries - 1) / p.queries;
    const int64_t units = static_cast<int64_t>(a->batch) * (p.heads / p.pack) * p.row_blocks;
    const int64_t tiles = (most_keys(p, p.queries) + fds::kBlockN - 1) / fds::kBlockN;
    const int split = choose_split(units, tiles, sms);
    // a warp's 32 output rows are whole queries: one box each (else a row per thread)
    p.out_boxes = split == 1 && 32 % p.pack == 0;
    if (p.out_boxes && (rc = make_heads_map(&maps.out, a->out, a->dtype, p.heads, p.q_len, a->batch, p.out_stride, 32 / p.pack, p.pack)) != FDS_OK)
        return rc;
    if (p.heads / p.pack > 65535) return set_error(FDS_ERR_INVALID_ARGUMENT, "more than 65535 heads");
    return split > 1 ? launch_units<T, true>(maps, p, a->batch, split, stream) : launch_units<T, false>(maps, p, a->batch, 1, stream);
}

template <typename T, int kHalves, bool kMulti>
int launch_step(const Params& p, int batch, int sms, cudaStream_t stream) {
    // The keys of a (window, key head) are dealt to the warps of a cluster while that
    // leaves most warps a block of 32 keys and at most 2 CTAs per SM (12 heads, 504 keys:
    // 3.75 us in four CTAs, 4.2 in two). A cluster has 8 CTAs at most, so few key heads
    // leave SMs idle however long the window: one window x 4 key heads, 4112 keys 6.2
    // us, 30000 keys 23.1 us or 1.3 TB/s, where 16 such windows read 4.6 TB/s.
    const int64_t units = static_cast<int64_t>(batch) * p.kv_heads, keys = most_keys(p, p.q_len);
    int split = 1;
    while (split < fds::window::kMaxSplit && units * split * 2 <= 2 * sms &&
           keys >= split * fds::window::kStepWarps * fds::window::kStepKeys)
        split *= 2;
    auto kern = fds::window::window_step_kernel<T, kHalves, kMulti>;
    static std::atomic<uint64_t> smem_set{0};
    cudaError_t e = set_smem_once(kern, fds::window::kStepSmem, smem_set);
    if (e != cudaSuccess) return set_error(FDS_ERR_CUDA, "cudaFuncSetAttribute(window step): %s", cudaGetErrorString(e));
    e = launch_cluster(kern, dim3(static_cast<unsigned>(split), static_cast<unsigned>(p.kv_heads), static_cast<unsigned>(batch)),
                       fds::window::kStepThreads, fds::window::kStepSmem, split, stream, p);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) return set_error(FDS_ERR_CUDA, "window attention launch: %s", cudaGetErrorString(e));
    return FDS_OK;
}

template <typename T>
int launch_step_rows(const Params& p, int batch, int sms, cudaStream_t s) {
    const int rows = p.q_len * (p.heads / p.kv_heads);
    if (p.q_len == 1) return rows <= 8 ? launch_step<T, 1, false>(p, batch, sms, s) : launch_step<T, 2, false>(p, batch, sms, s);
    return rows <= 8 ? launch_step<T, 1, true>(p, batch, sms, s) : launch_step<T, 2, true>(p, batch, sms, s);
}

bool strides_ok(const void* base, const int64_t* st, int batch, int len, int heads) {
    const int n[3] = {batch, len, heads};
    if (!aligned16(base)) return false;
    for (int i = 0; i < 3; ++i)
        if (n[i] > 1 && (st[i] < 64 || st[i] % 8 != 0)) return false;
    return true;
}

}  // namespace

extern "C" int fds_window_attn_fwd(const FdsWindowArgs* a, void* stream) {
    if (a == nullptr) return set_error(FDS_ERR_INVALID_ARGUMENT, "null args");
    if (a->q == nullptr || a->k == nullptr || a->v == nullptr || a->out == nullptr)
        return set_error(FDS_ERR_INVALID_ARGUMENT, "null q/k/v/out pointer");
    if (a->dtype != FDS_DTYPE_FP16 && a->dtype != FDS_DTYPE_BF16)
        return set_error(FDS_ERR_INVALID_ARGUMENT, "dtype must be FDS_DTYPE_FP16 or FDS_DTYPE_BF16 (got %d)", a->dtype);
    if (a->head_dim != 64) return set_error(FDS_ERR_INVALID_ARGUMENT, "head_dim must be 64 (got %d)", a->head_dim);
    if (a->batch < 1 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads != 0)
        return set_error(FDS_ERR_INVALID_ARGUMENT, "batch and heads must be >= 1, heads a multiple of kv_heads (got %d, %d, %d)",
                         a->batch, a->heads, a->kv_heads);
    if (a->batch > 65535 || a->kv_heads > 65535) return set_error(FDS_ERR_INVALID_ARGUMENT, "batch and kv_heads must be <= 65535");
    if (a->q_len < 0 || a->k_len < 0 || a->q_len > kMaxLen || a->k_len > kMaxLen)
        return set_error(FDS_ERR_INVALID_ARGUMENT, "q_len and k_len must be in [0, 2^28]");
    if (a->left < 0 || a->right < 0 || a->sinks < 0)
        return set_error(FDS_ERR_INVALID_ARGUMENT, "left, right and sinks must be >= 0 (got %d, %d, %d)", a->left, a->right,
                         a->sinks);
    if (!(a->scale > 0.f)) return set_error(FDS_ERR_INVALID_ARGUMENT, "scale must be > 0");
    if (!strides_ok(a->q, a->q_stride, a->batch, a->q_len, a->heads) ||
        !strides_ok(a->k, a->k_stride, a->batch, a->k_len, a->kv_heads) ||
        !strides_ok(a->v, a->v_stride, a->batch, a->k_len, a->kv_heads) ||
        !strides_ok(a->out, a->out_stride, a->batch, a->q_len, a->heads))
        return set_error(FDS_ERR_INVALID_ARGUMENT,
                         "q, k, v and out must be 16-byte aligned, their strides multiples of 8 elements and >= 64");
    if (a->q_len == 0) return set_ok();
    if (a->k_len == 0) return set_error(FDS_ERR_INVALID_ARGUMENT, "k_len must be >= 1 (an empty window is kv_len 0)");
    const int rc0 = check_device();
    if (rc0 != FDS_OK) return rc0;
    const int sms = sm_count();
    if (sms <= 0) return set_error(FDS_ERR_CUDA, "cannot query the SM count of the current device");

    Params p{};
    p.q = a->q, p.k = a->k, p.v = a->v, p.out = a->out;
    p.q_start = a->q_start, p.kv_len = a->kv_len;
    p.status = a->status, p.status_host = a->status_host, p.timeout_ns = a->timeout_ns, p.debug_flags = a->debug_flags;
    for (int i = 0; i < 3; ++i) {
        p.q_stride[i] = a->q_stride[i], p.k_stride[i] = a->k_stride[i];
        p.v_stride[i] = a->v_stride[i], p.out_stride[i] = a->out_stride[i];
    }
    p.heads = a->heads, p.kv_heads = a->kv_heads, p.q_len = a->q_len, p.k_len = a->k_len;
    p.left = std::min(a->left, kMaxLen), p.right = std::min(a->right, kMaxLen), p.sinks = std::min(a->sinks, a->k_len);
    p.scale_log2 = a->scale * 1.4426950408889634f;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int64_t rows = static_cast<int64_t>(a->q_len) * (a->heads / a->kv_heads);
    int rc;
    if (rows <= fds::window::kStepRows)
        rc = a->dtype == FDS_DTYPE_FP16 ? launch_step_rows<__half>(p, a->batch, sms, s)
                                        : launch_step_rows<__nv_bfloat16>(p, a->batch, sms, s);
    else
        rc = a->dtype == FDS_DTYPE_FP16 ? launch_tile<__half>(a, p, sms, s) : launch_tile<__nv_bfloat16>(a, p, sms, s);
    return rc == FDS_OK ? set_ok() : rc;
}
