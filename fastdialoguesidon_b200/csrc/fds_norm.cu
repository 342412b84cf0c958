// fds_norm.cu - fds_residual_norm_fwd: argument checks, the shape of the CTAs,
// and the launch.
#include <algorithm>

#include "capi_internal.h"
#include "norm_kernel.cuh"

using namespace fds_detail;

namespace {

using namespace fds::norm;

// CTAs of `warps` warps that an SM holds at once: 16 warps at 128 registers, and each
// CTA's ring, reduction slots and the 1 KB that every CTA takes in 228 KB.
template <int NCH, int R, int kMode, bool kXf32>
int resident(int warps) {
    const int bytes = Ring<NCH, kMode, kXf32>::bytes(32 * warps) + kReduceBytes<R> + 1024;
    return std::max(1, std::min(kMaxWarps / warps, 228 * 1024 / bytes));
}

template <typename T, int NCH, int R, int kMode, bool kXf32, bool kQuant>
int launch(Params& p, int warps, int sms, cudaStream_t stream) {
    using Rg = Ring<NCH, kMode, kXf32>;
    const int threads = 32 * warps, per_sm = resident<NCH, R, kMode, kXf32>(warps);
    const dim3 grid(static_cast<unsigned>(std::min(p.rows, sms * per_sm))), block(threads);
    auto kern = residual_norm_kernel<T, NCH, R, kMode, kXf32, kQuant>;
    static std::atomic<uint64_t> smem_set{0};
    cudaError_t e = set_smem_once(kern, Rg::bytes(32 * kMaxWarps), smem_set);
    if (e != cudaSuccess) return set_error(FDS_ERR_CUDA, "cudaFuncSetAttribute(norm): %s", cudaGetErrorString(e));
    e = launch_pdl(kern, grid, block, Rg::bytes(threads), stream, p);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) return set_error(FDS_ERR_CUDA, "residual norm launch: %s", cudaGetErrorString(e));
    return FDS_OK;
}

// A CTA as wide as the row: 8 columns a thread up to 4096, 16 or 32 beyond. The
// grid is what the SMs hold at once; four rows at a time once a CTA has two or more
// (3000 x 768 fp32 stream: 6.9 us against 8.3 us row by row, 6000 x 768: 13.9 against
// 16.9), single rows below, which are bound by one row's latency. (A grid of 16 CTAs
// an SM where shared memory holds 14 ran a second wave of whole CTAs: 8000 x 256 7.1
// us against 5.7, 100000 x 128 37.6 against 30.3.)
template <typename T, int kMode, bool kXf32, bool kQuant>
int launch_shape(Params& p, int sms, cudaStream_t s) {
    const int nch = p.c <= 4096 ? 1 : (p.c <= 8192 ? 2 : 4);
    const int warps = (p.c + 256 * nch - 1) / (256 * nch);
    if (nch == 4) return launch<T, 4, 1, kMode, kXf32, kQuant>(p, warps, sms, s);
    if (nch == 2) return launch<T, 2, 1, kMode, kXf32, kQuant>(p, warps, sms, s);
    if (p.rows >= 2 * sms * resident<1, 4, kMode, kXf32>(warps)) return launch<T, 1, 4, kMode, kXf32, kQuant>(p, warps, sms, s);
    return launch<T, 1, 1, kMode, kXf32, kQuant>(p, warps, sms, s);
}

template <typename T, int NCH, int kR>
int launch_quantise(const Params& p, cudaStream_t stream) {
    const dim3 grid(static_cast<unsigned>((p.rows - 1) / (kQuantWarps * kR) + 1)), block(32 * kQuantWarps);
    cudaError_t e = launch_pdl(quantise_rows_kernel<T, NCH, kR>, grid, block, 0, stream, p);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) return set_error(FDS_ERR_CUDA, "row quantiser launch: %s", cudaGetErrorString(e));
    return FDS_OK;
}

// By the row's width: the chunks a lane holds, and four or two rows a warp where
// one row would leave it less than 1 KB in flight.
template <typename T>
int launch_quantise_width(const Params& p, cudaStream_t s) {
    const int chunks = (p.c + 255) / 256;
    if (chunks <= 1) return launch_quantise<T, 1, 4>(p, s);
    if (chunks <= 2) return launch_quantise<T, 2, 2>(p, s);
    if (chunks <= 3) return launch_quantise<T, 3, 1>(p, s);
    if (chunks <= 4) return launch_quantise<T, 4, 1>(p, s);
    if (chunks <= 6) return launch_quantise<T, 6, 1>(p, s);
    if (chunks <= 8) return launch_quantise<T, 8, 1>(p, s);
    if (chunks <= 12) return launch_quantise<T, 12, 1>(p, s);
    if (chunks <= 16) return launch_quantise<T, 16, 1>(p, s);
    return launch_quantise<T, 32, 1>(p, s);
}
constexpr int kQuantWidth = 8192;  // columns a warp's registers hold; wider rows take the norm's kernel

template <typename T, bool kXf32>
int launch_mode(Params& p, int sms, cudaStream_t s) {
    const bool quant = p.h_scale != nullptr;
    if (p.y != nullptr)
        return quant ? launch_shape<T, kBoth, kXf32, true>(p, sms, s) : launch_shape<T, kBoth, kXf32, false>(p, sms, s);
    const bool plain = p.norm == kNone && p.w == nullptr && p.b == nullptr && p.scale == nullptr && p.shift == nullptr;
    if (quant && plain && !kXf32 && p.c <= kQuantWidth) return launch_quantise_width<T>(p, s);
    return quant ? launch_shape<T, kNormOnly, kXf32, true>(p, sms, s) : launch_shape<T, kNormOnly, kXf32, false>(p, sms, s);
}

template <typename T>
int launch_type(Params& p, int sms, cudaStream_t s) {
    return p.x_f32 ? launch_mode<T, true>(p, sms, s) : launch_mode<T, false>(p, sms, s);
}

constexpr int kMaxWidth = 16384;

bool rows_ok(const void* p, int64_t stride, int c, int esize) {
    return aligned16(p) && stride >= c && (stride * esize) % 16 == 0;
}

}  // namespace

extern "C" int fds_residual_norm_fwd(const FdsResidualNormArgs* a, void* stream) {
    if (a == nullptr) return set_error(FDS_ERR_INVALID_ARGUMENT, "null args");
    if (a->x == nullptr) return set_error(FDS_ERR_INVALID_ARGUMENT, "null x pointer");
    if (a->dtype != FDS_DTYPE_FP16 && a->dtype != FDS_DTYPE_BF16)
        return set_error(FDS_ERR_INVALID_ARGUMENT, "dtype must be FDS_DTYPE_FP16 or FDS_DTYPE_BF16 (got %d)", a->dtype);
    if (a->rows < 0 || a->length < 1) return set_error(FDS_ERR_INVALID_ARGUMENT, "rows >= 0 and length >= 1 required");
    if (a->c < 8 || a->c % 8 != 0 || a->c > kMaxWidth)
        return set_error(FDS_ERR_INVALID_ARGUMENT, "c must be a multiple of 8 in [8, %d] (got %d)", kMaxWidth, a->c);
    if (a->post < FDS_NORM_NONE || a->post > FDS_NORM_RMS || a->norm < FDS_NORM_NONE || a->norm > FDS_NORM_RMS)
        return set_error(FDS_ERR_INVALID_ARGUMENT, "post and norm must be FDS_NORM_NONE, FDS_NORM_LAYER or FDS_NORM_RMS");
    if (!(a->eps >= 0.f)) return set_error(FDS_ERR_INVALID_ARGUMENT, "eps must be >= 0");
    if (a->y == nullptr && (a->gate != nullptr || a->post_w != nullptr || a->post_b != nullptr || a->post != FDS_NORM_NONE))
        return set_error(FDS_ERR_INVALID_ARGUMENT, "gate and the norm after the block need y");
    if (a->y != nullptr && a->x_out == nullptr) return set_error(FDS_ERR_INVALID_ARGUMENT, "null x_out pointer");
    if (a->y == nullptr && a->x_out != nullptr) return set_error(FDS_ERR_INVALID_ARGUMENT, "x_out without y (x is not changed)");
    if (a->x_out == nullptr && a->h == nullptr) return set_error(FDS_ERR_INVALID_ARGUMENT, "neither x_out nor h is given");
    if (a->h_scale != nullptr && a->h == nullptr) return set_error(FDS_ERR_INVALID_ARGUMENT, "h_scale without h");
    const int xs = a->x_f32 ? 4 : 2, ps = a->param_f32 ? 4 : 2, hs = a->h_scale != nullptr ? 1 : 2;
    if (!rows_ok(a->x, a->x_stride, a->c, xs) || (a->y != nullptr && !rows_ok(a->y, a->y_stride, a->c, 2)) ||
        (a->x_out != nullptr && !rows_ok(a->x_out, a->x_out_stride, a->c, xs)))
        return set_error(FDS_ERR_INVALID_ARGUMENT, "x, y and x_out rows must be 16-byte aligned, strides >= c");
    if (a->h != nullptr && ((reinterpret_cast<uintptr_t>(a->h) & (hs == 1 ? 7u : 15u)) != 0 || a->h_stride < a->c ||
                            (a->h_stride * hs) % (hs == 1 ? 8 : 16) != 0))
        return set_error(FDS_ERR_INVALID_ARGUMENT, "h rows must be 16-byte (8-bit rows: 8-byte) aligned, stride >= c");
    const void* params[] = {a->gate, a->post_w, a->post_b, a->w, a->b, a->scale, a->shift};
    for (const void* q : params)
        if (!aligned16(q)) return set_error(FDS_ERR_INVALID_ARGUMENT, "parameter vectors must be 16-byte aligned");
    if (a->gate_stride < 0 || a->mod_stride < 0 || (a->gate_stride * ps) % 16 != 0 || (a->mod_stride * ps) % 16 != 0)
        return set_error(FDS_ERR_INVALID_ARGUMENT, "gate / mod strides must be >= 0 and keep rows 16-byte aligned");
    if (a->rows == 0) return set_ok();
    const int rc0 = check_device();
    if (rc0 != FDS_OK) return rc0;

    fds::norm::Params p{};
    p.x = a->x, p.y = a->y, p.x_out = a->x_out, p.h = a->h, p.h_scale = a->h_scale;
    p.gate = a->gate, p.post_w = a->post_w, p.post_b = a->post_b, p.w = a->w, p.b = a->b;
    p.scale = a->scale, p.shift = a->shift;
    p.x_stride = a->x_stride, p.y_stride = a->y_stride, p.x_out_stride = a->x_out_stride, p.h_stride = a->h_stride;
    p.gate_stride = a->gate_stride, p.mod_stride = a->mod_stride;
    p.rows = a->rows, p.c = a->c, p.length = a->length;
    p.x_f32 = a->x_f32, p.param_f32 = a->param_f32, p.post = a->post, p.norm = a->norm;
    p.alpha = a->alpha, p.eps = a->eps;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    p.x_out_wide = (reinterpret_cast<uintptr_t>(p.x_out) & 31u) == 0 && (p.rows <= 1 || p.x_out_stride % 8 == 0);
    const int sms = sm_count();
    if (sms <= 0) return set_error(FDS_ERR_CUDA, "cannot query the SM count of the current device");
    const int rc = a->dtype == FDS_DTYPE_FP16 ? launch_type<__half>(p, sms, s) : launch_type<__nv_bfloat16>(p, sms, s);
    return rc == FDS_OK ? set_ok() : rc;
}
