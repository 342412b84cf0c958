// fds_int8.cu - fds_linear_int8_fwd: the linear layers of fds_linear_fwd over
// 8-bit integer operands with a scale per token and per output channel.
#include <algorithm>

#include "capi_internal.h"
#include "gemm_kernel.cuh"
#include "gemv_i8_kernel.cuh"

using namespace fds_detail;

namespace {

struct Maps {
    CUtensorMap a, b, out, cos, sin;
};

// 2-D row-major map with 128-byte swizzled boxes of `box_cols` x `box_rows`.
int make_map(CUtensorMap* map, CUtensorMapDataType type, int esize, const void* base, int64_t cols, int64_t rows,
             int64_t row_stride, int box_cols, int box_rows) {
    EncodeTiledFn enc = encode_fn();
    if (enc == nullptr) return set_error(FDS_ERR_TENSOR_MAP, "cuTensorMapEncodeTiled unavailable from the driver");
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(row_stride * esize)};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t estr[2] = {1, 1};
    CUresult r = enc(map, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(FDS_ERR_TENSOR_MAP, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
    return FDS_OK;
}

template <typename T, int BN, int kEpi, bool kPair, bool kCut = false>
int launch(const Maps& m, const fds::gemm::Params& p, int grid, cudaStream_t stream) {
    auto kern = fds::gemm::gemm_kernel<T, BN, kEpi, kPair, true, kCut>;
    constexpr int smem = fds::gemm::Smem<BN, kPair, kEpi == fds::gemm::kRope, true>::alloc;
    static std::atomic<uint64_t> smem_set{0};
    cudaError_t e = set_smem_once(kern, smem, smem_set);
    if (e != cudaSuccess) return set_error(FDS_ERR_CUDA, "cudaFuncSetAttribute(int8 gemm): %s", cudaGetErrorString(e));
    const dim3 g(static_cast<unsigned>(grid)), b(fds::gemm::kThreads);
    e = kPair ? launch_pair(kern, g, b, smem, stream, m.a, m.b, m.out, m.cos, m.sin, p)
              : launch_pdl(kern, g, b, smem, stream, m.a, m.b, m.out, m.cos, m.sin, p);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) return set_error(FDS_ERR_CUDA, "int8 linear launch: %s", cudaGetErrorString(e));
    return FDS_OK;
}

template <typename T, int BN, bool kPair>
int launch_epi(int epi, const Maps& m, const fds::gemm::Params& p, int grid, cudaStream_t s) {
    if constexpr (BN == 256) {
        if (p.cut > 0)
            return epi == FDS_EPILOGUE_STORE ? launch<T, BN, fds::gemm::kStore, kPair, true>(m, p, grid, s)
                                             : launch<T, BN, fds::gemm::kAccum, kPair, true>(m, p, grid, s);
    }
    switch (epi) {
        case FDS_EPILOGUE_STORE: return launch<T, BN, fds::gemm::kStore, kPair>(m, p, grid, s);
        case FDS_EPILOGUE_ROPE: return launch<T, BN, fds::gemm::kRope, kPair>(m, p, grid, s);
        default: return launch<T, BN, fds::gemm::kAccum, kPair>(m, p, grid, s);
    }
}

template <typename T>
int launch_shape(int bn, bool pair, int epi, const Maps& m, const fds::gemm::Params& p, int grid, cudaStream_t s) {
    if (pair) return bn == 256 ? launch_epi<T, 256, true>(epi, m, p, grid, s) : launch_epi<T, 128, true>(epi, m, p, grid, s);
    if (bn == 64) return launch_epi<T, 64, false>(epi, m, p, grid, s);
    return bn == 256 ? launch_epi<T, 256, false>(epi, m, p, grid, s) : launch_epi<T, 128, false>(epi, m, p, grid, s);
}

template <typename T, int M, int kEpi>
int launch_gemv(const fds::gemv::Params& p, cudaStream_t s) {
    const int per = 2 * fds::gemv::kWarps;
    cudaError_t e = launch_pdl(fds::gemv::gemv_i8_kernel<T, M, kEpi>, dim3(static_cast<unsigned>((p.n + per - 1) / per)),
                               dim3(32 * fds::gemv::kWarps), 0, s, p);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) return set_error(FDS_ERR_CUDA, "int8 linear launch: %s", cudaGetErrorString(e));
    return FDS_OK;
}

template <typename T, int kEpi>
int launch_gemv_rows(const fds::gemv::Params& p, cudaStream_t s) {
    if (p.m == 1) return launch_gemv<T, 1, kEpi>(p, s);
    if (p.m == 2) return launch_gemv<T, 2, kEpi>(p, s);
    if (p.m <= 4) return launch_gemv<T, 4, kEpi>(p, s);
    return launch_gemv<T, 8, kEpi>(p, s);
}

template <typename T>
int launch_gemv_epi(int epi, const fds::gemv::Params& p, cudaStream_t s) {
    switch (epi) {
        case FDS_EPILOGUE_STORE: return launch_gemv_rows<T, fds::gemm::kStore>(p, s);
        case FDS_EPILOGUE_ROPE: return launch_gemv_rows<T, fds::gemm::kRope>(p, s);
        default: return launch_gemv_rows<T, fds::gemm::kAccum>(p, s);
    }
}

// CTA pairs of the 256-column tile that can be resident at once (cached per
// device; 0 if it cannot be queried).
int max_pairs() {
    static std::atomic<int> cached[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    int n = cached[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        auto kern = fds::gemm::gemm_kernel<__half, 256, fds::gemm::kStore, true, true>;
        constexpr int smem = fds::gemm::Smem<256, true, false, true>::alloc;
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return 0;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2);
        cfg.blockDim = dim3(fds::gemm::kThreads);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
            cudaGetLastError();
            return 0;
        }
        cached[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

// Pieces (log2) that the tiles of the last wave are cut into, so that more SMs share
// them: as many as fit into one wave. Whole / cut, us: 4101 x 768 -> 2304 10.6 / 9.7,
// 10000 x 1024 -> 1024 15.3 / 13.6, 2500 x 768 -> 2304 10.1 / 7.9. Not with RoPE, whose
// pieces would read whole boxes of W (no map left): 2500 x 768 11.8 / 10.7, but 10000 x
// 1024 -> 3072 33.4 / 35.1.
int last_cut(int bn, int epilogue, int64_t tiles, int64_t units) {
    const int64_t rest = tiles % units;
    if (bn != 256 || epilogue == FDS_EPILOGUE_ROPE || rest == 0) return 0;
    return 4 * rest <= units ? 2 : (2 * rest <= units ? 1 : 0);
}

struct Tile {
    int bn;
    bool pair;
};

// Of the tilings, the one that should finish first: its launch, then as many
// waves of tiles as the SMs (pairs) need, each tile for as long as its products
// take (they grow with k) but at least as long as its epilogue. The constants are
// microseconds fitted to a sweep on a B200 (m 600 - 48000, n 1024 - 3072, k 256 - 4096,
// each within 10 %): at n = 3072, m = 6000 single 256-column tiles lead below k =
// 2048 (k = 256: 13.1 against 16.1 us, 1024: 19.5 against 20.7), pairs from there
// on (2048: 28.5 against 31.4, 4096: 50.4 against 55.2); narrow tiles lead where
// wide ones leave SMs idle (m = 1500, n = k = 1024: 128 columns 5.7 us, 256 6.7).
Tile choose_tile(int64_t m, int64_t n, int64_t k, int epilogue, int64_t sms, int64_t pairs, int want_bn, int want_pair) {
    struct Cost {
        int bn;
        bool pair;
        double launch, tile, per_k, epi16, epi32;  // per_k: of 1024
    };
    const Cost all[] = {{256, true, 4.0, 1.2, 2.70, 3.0, 5.2},
                        {128, true, 4.0, 0.8, 1.62, 1.9, 3.3},
                        {256, false, 3.0, 1.2, 2.90, 2.5, 5.0},
                        {128, false, 3.0, 0.5, 2.08, 1.35, 2.8},
                        {64, false, 3.0, 0.3, 1.85, 0.9, 1.6}};
    Tile best{128, false};
    double best_cost = 1e30;
    for (const Cost& c : all) {
        if (want_bn != 0 && c.bn != want_bn) continue;
        if (want_pair == FDS_GEMM_SINGLE && c.pair) continue;
        if (want_pair == FDS_GEMM_PAIR && !c.pair) continue;
        if (c.pair && (pairs < 1 || (m <= fds::gemm::kBM && want_pair != FDS_GEMM_PAIR))) continue;
        const int64_t units = c.pair ? pairs : sms;
        const int64_t tm = c.pair ? 2 * fds::gemm::kBM : fds::gemm::kBM;
        const int64_t tiles = (m + tm - 1) / tm * ((n + c.bn - 1) / c.bn);
        const int cut = last_cut(c.bn, epilogue, tiles, units);
        // a wave of halves or quarters costs 0.6 or 0.35 of a whole one
        const double waves = cut == 0 ? static_cast<double>((tiles + units - 1) / units)
                                      : static_cast<double>(tiles / units) + (cut == 1 ? 0.6 : 0.35);
        const double products = c.tile + c.per_k * static_cast<double>(k) / 1024.0;
        const double cost = c.launch + waves * std::max(products, epilogue == FDS_EPILOGUE_ACCUMULATE_F32 ? c.epi32 : c.epi16);
        if (cost < best_cost) best_cost = cost, best = Tile{c.bn, c.pair};
    }
    return best;
}

}  // namespace

extern "C" int fds_linear_int8_fwd(const FdsLinearInt8Args* a, void* stream) {
    if (a == nullptr) return set_error(FDS_ERR_INVALID_ARGUMENT, "null args");
    if (a->a == nullptr || a->w == nullptr || a->out == nullptr || a->a_scale == nullptr || a->w_scale == nullptr)
        return set_error(FDS_ERR_INVALID_ARGUMENT, "null a/w/scale/out pointer");
    if (a->dtype != FDS_DTYPE_FP16 && a->dtype != FDS_DTYPE_BF16)
        return set_error(FDS_ERR_INVALID_ARGUMENT, "dtype must be FDS_DTYPE_FP16 or FDS_DTYPE_BF16 (got %d)", a->dtype);
    if (a->epilogue < FDS_EPILOGUE_STORE || a->epilogue > FDS_EPILOGUE_ACCUMULATE_F32)
        return set_error(FDS_ERR_INVALID_ARGUMENT, "unknown epilogue %d", a->epilogue);
    if (a->m < 0 || a->n < 1 || a->k < 1) return set_error(FDS_ERR_INVALID_ARGUMENT, "m >= 0, n >= 1, k >= 1 required");
    if (a->k % 16 != 0 || a->k > 65536)
        return set_error(FDS_ERR_INVALID_ARGUMENT, "k must be a multiple of 16, at most 65536 (got %d)", a->k);
    if (a->n % 8 != 0) return set_error(FDS_ERR_INVALID_ARGUMENT, "n must be a multiple of 8 (got %d)", a->n);
    if (a->a_row_stride < a->k || a->a_row_stride % 16 != 0 || a->w_row_stride < a->k || a->w_row_stride % 16 != 0)
        return set_error(FDS_ERR_INVALID_ARGUMENT, "a / w row strides must be >= k and multiples of 16");
    const bool f32_out = a->epilogue == FDS_EPILOGUE_ACCUMULATE_F32;
    if (a->out_row_stride < a->n || a->out_row_stride % (f32_out ? 4 : 8) != 0)
        return set_error(FDS_ERR_INVALID_ARGUMENT, "out row stride must be >= n and keep rows 16-byte aligned");
    if (!aligned16(a->a) || !aligned16(a->w) || !aligned16(a->out) || !aligned16(a->bias) || !aligned16(a->w_scale) ||
        (reinterpret_cast<uintptr_t>(a->a_scale) & 3u) != 0)
        return set_error(FDS_ERR_INVALID_ARGUMENT,
                         "a, w, bias, w_scale and out must be 16-byte aligned, a_scale 4-byte aligned");
    if (a->epilogue == FDS_EPILOGUE_ROPE) {
        if (a->cos == nullptr || a->sin == nullptr || !aligned16(a->cos) || !aligned16(a->sin))
            return set_error(FDS_ERR_INVALID_ARGUMENT, "cos/sin must be 16-byte aligned fp32 [>= seq_len, 64] tables");
        if (a->seq_len < 1) return set_error(FDS_ERR_INVALID_ARGUMENT, "seq_len must be >= 1");
        if (a->n % 64 != 0 || a->rope_cols < 0 || a->rope_cols > a->n || a->rope_cols % 64 != 0)
            return set_error(FDS_ERR_INVALID_ARGUMENT, "n and rope_cols must be multiples of 64, rope_cols in [0, n]");
    }
    if (a->tile_n != 0 && a->tile_n != 64 && a->tile_n != 128 && a->tile_n != 256)
        return set_error(FDS_ERR_INVALID_ARGUMENT, "tile_n must be 0, 64, 128 or 256 (got %d)", a->tile_n);
    if (a->cta_pair < FDS_GEMM_AUTO || a->cta_pair > FDS_GEMM_PAIR || (a->cta_pair == FDS_GEMM_PAIR && a->tile_n == 64))
        return set_error(FDS_ERR_INVALID_ARGUMENT,
                         "cta_pair must be FDS_GEMM_AUTO, FDS_GEMM_SINGLE or FDS_GEMM_PAIR (tile_n 128 or 256)");
    if (a->m == 0) return set_ok();
    int rc = check_device();
    if (rc != FDS_OK) return rc;
    const int rope_cols = a->epilogue == FDS_EPILOGUE_ROPE ? a->rope_cols : 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);

    if (a->m <= fds::gemv::kMaxRows && a->tile_n == 0 && a->cta_pair == FDS_GEMM_AUTO) {
        fds::gemv::Params p{};
        p.a = static_cast<const int8_t*>(a->a), p.w = static_cast<const int8_t*>(a->w);
        p.a_scale = a->a_scale, p.w_scale = a->w_scale, p.bias = a->bias, p.out = a->out;
        p.cos_t = a->cos, p.sin_t = a->sin;
        p.a_stride = a->a_row_stride, p.w_stride = a->w_row_stride, p.out_stride = a->out_row_stride;
        p.m = a->m, p.n = a->n, p.k = a->k, p.seq_len = a->seq_len, p.rope_cols = rope_cols;
        rc = a->dtype == FDS_DTYPE_FP16 ? launch_gemv_epi<__half>(a->epilogue, p, s)
                                        : launch_gemv_epi<__nv_bfloat16>(a->epilogue, p, s);
        return rc == FDS_OK ? set_ok() : rc;
    }

    const int sms = sm_count();
    if (sms <= 0) return set_error(FDS_ERR_CUDA, "cannot query the SM count of the current device");
    const int64_t pairs = a->cta_pair == FDS_GEMM_SINGLE ? 0 : std::min<int64_t>(sms / 2, max_pairs());
    if (a->cta_pair == FDS_GEMM_PAIR && pairs < 1)
        return set_error(FDS_ERR_INVALID_ARGUMENT, "no CTA pair can be launched on this device");
    const Tile t = choose_tile(a->m, a->n, a->k, a->epilogue, sms, pairs, a->tile_n, a->cta_pair);
    const int tile_m = t.pair ? 2 * fds::gemm::kBM : fds::gemm::kBM;
    const int64_t tiles_n = (a->n + t.bn - 1) / t.bn;
    const int64_t tiles = (static_cast<int64_t>(a->m) + tile_m - 1) / tile_m * tiles_n;
    if (tiles > 0x7fffffffLL) return set_error(FDS_ERR_INVALID_ARGUMENT, "too many tiles");

    Maps maps;
    const auto u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
    if ((rc = make_map(&maps.a, u8, 1, a->a, a->k, a->m, a->a_row_stride, fds::gemm::kRowBytes, fds::gemm::kBM)) != FDS_OK ||
        (rc = make_map(&maps.b, u8, 1, a->w, a->k, a->n, a->w_row_stride, fds::gemm::kRowBytes, t.pair ? t.bn / 2 : t.bn)) != FDS_OK)
        return rc;
    const auto ot = f32_out ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                            : a->dtype == FDS_DTYPE_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                         : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const int os = f32_out ? 4 : 2;
    if ((rc = make_map(&maps.out, ot, os, a->out, a->n, a->m, a->out_row_stride, 128 / os, 32)) != FDS_OK) return rc;
    const int64_t units = t.pair ? pairs : sms;
    const int cut = last_cut(t.bn, a->epilogue, tiles, units);
    maps.cos = maps.sin = maps.out;
    // (the cut tiles' quarter boxes of W travel in the place of the cosines)
    if (cut > 0 && (rc = make_map(&maps.cos, u8, 1, a->w, a->k, a->n, a->w_row_stride, fds::gemm::kRowBytes, t.bn / (t.pair ? 8 : 4))) != FDS_OK)
        return rc;
    if (a->epilogue == FDS_EPILOGUE_ROPE &&
        ((rc = make_map(&maps.cos, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, a->cos, 64, a->seq_len, 64, 32, fds::gemm::kBM)) != FDS_OK ||
         (rc = make_map(&maps.sin, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, a->sin, 64, a->seq_len, 64, 32, fds::gemm::kBM)) != FDS_OK))
        return rc;
    fds::gemm::Params p{};
    p.bias = a->bias;
    p.cos_t = a->cos;
    p.sin_t = a->sin;
    p.a_scale = a->a_scale;
    p.w_scale = a->w_scale;
    p.status = a->status;
    p.status_host = a->status_host;
    p.timeout_ns = a->timeout_ns;
    p.m = a->m;
    p.n = a->n;
    p.k = a->k;
    p.seq_len = a->seq_len;
    p.rope_cols = rope_cols;
    p.tiles_n = static_cast<int32_t>(tiles_n);
    p.cut = cut;
    p.whole = static_cast<int32_t>(p.cut > 0 ? tiles - tiles % units : tiles);
    p.tiles = static_cast<int32_t>(p.whole + ((tiles - p.whole) << p.cut));
    const int grid = static_cast<int>(std::min<int64_t>(p.tiles, units) * (t.pair ? 2 : 1));
    rc = a->dtype == FDS_DTYPE_FP16 ? launch_shape<__half>(t.bn, t.pair, a->epilogue, maps, p, grid, s)
                                    : launch_shape<__nv_bfloat16>(t.bn, t.pair, a->epilogue, maps, p, grid, s);
    return rc == FDS_OK ? set_ok() : rc;
}
