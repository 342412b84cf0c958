// fds_norm.cu - fds_residual_norm_fwd: argument checks, the choice of how many
// warps share a row, and the launch.
#include "capi_internal.h"
#include "norm_kernel.cuh"

using namespace fds_detail;

namespace {

template <typename T, int NCH, int WPR, bool kQuant>
int launch(const fds::norm::Params& p, cudaStream_t stream) {
    const int per = WPR == 1 ? fds::norm::kWarpRows : 1;
    const dim3 grid(static_cast<unsigned>((p.rows + per - 1) / per)), block(32 * (WPR == 1 ? per : WPR));
    cudaError_t e = launch_pdl(fds::norm::residual_norm_kernel<T, NCH, WPR, kQuant>, grid, block, 0, stream, p);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) return set_error(FDS_ERR_CUDA, "residual norm launch: %s", cudaGetErrorString(e));
    return FDS_OK;
}

// The fewest warps per row whose threads hold at most 4 chunks of 8 elements
// (5 and more would leave fewer warps per SM to cover the memory latency);
// past 4 warps x 4 chunks a row takes 8 warps and as many chunks as it needs.
template <typename T, bool kQuant>
int launch_shape(const fds::norm::Params& p, cudaStream_t s) {
    const int c = p.c;
    if (c <= 256) return launch<T, 1, 1, kQuant>(p, s);
    if (c <= 512) return launch<T, 2, 1, kQuant>(p, s);
    if (c <= 768) return launch<T, 3, 1, kQuant>(p, s);
    if (c <= 1024) return launch<T, 4, 1, kQuant>(p, s);
    if (c <= 1536) return launch<T, 3, 2, kQuant>(p, s);
    if (c <= 2048) return launch<T, 4, 2, kQuant>(p, s);
    if (c <= 3072) return launch<T, 3, 4, kQuant>(p, s);
    if (c <= 4096) return launch<T, 4, 4, kQuant>(p, s);
    if (c <= 8192) return launch<T, 4, 8, kQuant>(p, s);
    return launch<T, 8, 8, kQuant>(p, s);
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
    const bool quant = a->h_scale != nullptr;
    int rc;
    if (a->dtype == FDS_DTYPE_FP16)
        rc = quant ? launch_shape<__half, true>(p, s) : launch_shape<__half, false>(p, s);
    else
        rc = quant ? launch_shape<__nv_bfloat16, true>(p, s) : launch_shape<__nv_bfloat16, false>(p, s);
    return rc == FDS_OK ? set_ok() : rc;
}
