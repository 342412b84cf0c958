// norm_kernel.cuh - the step between two blocks of a pre- / post-norm layer, one
// pass over the rows:
//   z  = post(y) * post_w + post_b            post: none, LayerNorm or RMS norm
//   x' = alpha * x + gate * z                 the residual stream, rounded once when stored
//   h  = (norm(x') * w + b) * (1 + scale) + shift
// with norm: none, LayerNorm or RMS norm, h in the operand type or, quantised
// per row, in 8-bit integers: s = max|h| / 127, q = rint(h * (127 / max|h|)).
// With y absent x' = x (nothing is written back), so norm none + quantised
// output is the row quantiser of the 8-bit linear layers.
//
// LayerNorm(t) = (t - mean t) / sqrt(mean (t - mean t)^2 + eps), the variance
// from a second sweep over the registers (no cancellation); RMS(t) = t /
// sqrt(mean t^2 + eps). h uses the 32-bit x', not its stored rounding.
//
// Bound by memory: a row is read once (x, y), held in registers through up to
// five reductions, and written once (x', h): (2 * stream + 4) bytes per
// element against ~14 flops. A row belongs to WPR warps whose threads hold NCH
// chunks of 8 consecutive elements each; all of a row's loads are issued before
// the first reduction, so a warp has NCH * 256 elements in flight. The 16-byte
// parameter loads hit L1 / L2: a window's rows share them.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "fds_b200.h"
#include "fds_ptx.cuh"

namespace fds {
namespace norm {

enum Kind : int { kNone = 0, kLayer = 1, kRms = 2 };

struct Params {
    const void* x;        // residual stream in: fp32 (x_f32) or operand type
    const void* y;        // block output, operand type, or null
    void* x_out;          // residual stream out, x's type, or null
    void* h;              // operand type or int8 (h_scale given), or null
    float* h_scale;       // [rows] of a quantised h, or null
    const void* gate;     // [c], or one row of c per window; parameter type, or null
    const void* post_w;   // [c], or null
    const void* post_b;
    const void* w;
    const void* b;
    const void* scale;    // [c], or one row per window
    const void* shift;
    int64_t x_stride, y_stride, x_out_stride, h_stride;  // elements
    int64_t gate_stride, mod_stride;                     // elements between windows (0: shared)
    int32_t rows, c, length;  // rows per window
    int32_t x_f32, param_f32;
    int32_t post, norm;       // Kind
    float alpha, eps;
};

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
    return __half22float2(*reinterpret_cast<__half2*>(&v));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& r, float (&v)[8]) {
    const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2<T>(u[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

// 8 parameters from element `at` (a multiple of 8)
template <typename T>
__device__ __forceinline__ void param8(const void* p, bool f32, int64_t at, float (&v)[8]) {
    if (f32) {
        const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
        const float4 a = __ldg(q), b = __ldg(q + 1);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        unpack8<T>(__ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p) + at)), v);
    }
}

// Sum / maximum over the WPR warps of a row; `slot` differs between the
// reductions of one row, so one barrier each is enough.
template <int WPR>
__device__ __forceinline__ float row_sum(float v, float* red, int slot) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if constexpr (WPR > 1) {
        if ((threadIdx.x & 31) == 0) red[slot * WPR + (threadIdx.x >> 5)] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < WPR; ++i) v += red[slot * WPR + i];
    }
    return v;
}
template <int WPR>
__device__ __forceinline__ uint32_t row_max(uint32_t v, float* red, int slot) {
    v = __reduce_max_sync(0xffffffffu, v);
    if constexpr (WPR > 1) {
        if ((threadIdx.x & 31) == 0) red[slot * WPR + (threadIdx.x >> 5)] = __uint_as_float(v);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WPR; ++i) v = max(v, __float_as_uint(red[slot * WPR + i]));
    }
    return v;
}

// t <- LayerNorm / RMS norm of the row (elements past c stay 0 and count for nothing)
template <int NCH, int WPR>
__device__ __forceinline__ void normalise(float (&t)[NCH][8], int kind, int lane8, int c, float eps, float* red,
                                          int slot) {
    const float inv_c = 1.f / static_cast<float>(c);
    if (kind == kLayer) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) s += t[i][e];
        const float mean = row_sum<WPR>(s, red, slot) * inv_c;
#pragma unroll
        for (int i = 0; i < NCH; ++i)
            if (lane8 + i * WPR * 256 < c)
#pragma unroll
                for (int e = 0; e < 8; ++e) t[i][e] -= mean;
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(t[i][e], t[i][e], s);
    const float r = rsqrtf(row_sum<WPR>(s, red, slot + 1) * inv_c + eps);
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) t[i][e] *= r;
}

constexpr int kSlots = 5;
constexpr int kWarpRows = 4;  // rows per CTA when a warp holds a whole row

template <typename T, int NCH, int WPR, bool kQuant>
__global__ void __launch_bounds__(WPR == 1 ? 32 * kWarpRows : 32 * WPR) residual_norm_kernel(const Params p) {
    __shared__ float red[kSlots * WPR];
    grid_launch_dependents();
    grid_dependency_wait();
    const int row = WPR == 1 ? static_cast<int>(blockIdx.x) * kWarpRows + static_cast<int>(threadIdx.x >> 5)
                             : static_cast<int>(blockIdx.x);
    if (row >= p.rows) return;  // whole warps of a one-warp-per-row CTA only
    const int lane8 = 8 * static_cast<int>(WPR == 1 ? threadIdx.x & 31 : threadIdx.x);  // first element of chunk 0
    const int64_t window = row / p.length;
    const bool pf = p.param_f32 != 0;

    float x[NCH][8];
    {
        uint4 ry[NCH];
        if (p.y != nullptr) {
            const T* y = static_cast<const T*>(p.y) + row * p.y_stride;
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int at = lane8 + i * WPR * 256;
                ry[i] = at < p.c ? *reinterpret_cast<const uint4*>(y + at) : make_uint4(0, 0, 0, 0);
            }
        }
        if (p.x_f32) {
            const float* xr = static_cast<const float*>(p.x) + row * p.x_stride;
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int at = lane8 + i * WPR * 256;
                float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
                if (at < p.c) {
                    a = *reinterpret_cast<const float4*>(xr + at);
                    b = *reinterpret_cast<const float4*>(xr + at + 4);
                }
                x[i][0] = a.x, x[i][1] = a.y, x[i][2] = a.z, x[i][3] = a.w;
                x[i][4] = b.x, x[i][5] = b.y, x[i][6] = b.z, x[i][7] = b.w;
            }
        } else {
            const T* xr = static_cast<const T*>(p.x) + row * p.x_stride;
            uint4 rx[NCH];
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int at = lane8 + i * WPR * 256;
                rx[i] = at < p.c ? *reinterpret_cast<const uint4*>(xr + at) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < NCH; ++i) unpack8<T>(rx[i], x[i]);
        }
        if (p.y != nullptr) {
            float y[NCH][8];
#pragma unroll
            for (int i = 0; i < NCH; ++i) unpack8<T>(ry[i], y[i]);
            if (p.post != kNone) normalise<NCH, WPR>(y, p.post, lane8, p.c, p.eps, red, 0);
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int at = lane8 + i * WPR * 256;
                if (at >= p.c) continue;
                float v[8];
                if (p.post_w != nullptr) {
                    param8<T>(p.post_w, pf, at, v);
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[i][e] *= v[e];
                }
                if (p.post_b != nullptr) {
                    param8<T>(p.post_b, pf, at, v);
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[i][e] += v[e];
                }
                if (p.gate != nullptr) {
                    param8<T>(p.gate, pf, window * p.gate_stride + at, v);
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[i][e] *= v[e];
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) x[i][e] = fmaf(p.alpha, x[i][e], y[i][e]);
            }
        }
    }
    if (p.x_out != nullptr) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int at = lane8 + i * WPR * 256;
            if (at >= p.c) continue;
            const float(&v)[8] = x[i];
            if (p.x_f32) {
                float4* o = reinterpret_cast<float4*>(static_cast<float*>(p.x_out) + row * p.x_out_stride + at);
                o[0] = make_float4(v[0], v[1], v[2], v[3]);
                o[1] = make_float4(v[4], v[5], v[6], v[7]);
            } else {
                *reinterpret_cast<uint4*>(static_cast<T*>(p.x_out) + row * p.x_out_stride + at) =
                    make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
            }
        }
    }
    if (p.h == nullptr) return;

    if (p.norm != kNone) normalise<NCH, WPR>(x, p.norm, lane8, p.c, p.eps, red, 2);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int at = lane8 + i * WPR * 256;
        if (at >= p.c) continue;
        float v[8];
        if (p.w != nullptr) {
            param8<T>(p.w, pf, at, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[i][e] *= v[e];
        }
        if (p.b != nullptr) {
            param8<T>(p.b, pf, at, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[i][e] += v[e];
        }
        if (p.scale != nullptr) {
            param8<T>(p.scale, pf, window * p.mod_stride + at, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[i][e] = fmaf(x[i][e], v[e], x[i][e]);
        }
        if (p.shift != nullptr) {
            param8<T>(p.shift, pf, window * p.mod_stride + at, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[i][e] += v[e];
        }
        if constexpr (!kQuant)
            *reinterpret_cast<uint4*>(static_cast<T*>(p.h) + row * p.h_stride + at) =
                make_uint4(pack2<T>(x[i][0], x[i][1]), pack2<T>(x[i][2], x[i][3]), pack2<T>(x[i][4], x[i][5]),
                           pack2<T>(x[i][6], x[i][7]));
    }
    if constexpr (kQuant) {
        // max|h| as unsigned bits: orders the finite values, and infinities and
        // NaN above them all
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(fabsf(x[i][e])));
        m = row_max<WPR>(m, red, 4);
        const float big = __uint_as_float(m);
        // a row with an infinity or a NaN gets the scale NaN (its products say so);
        // one whose 127 / max could overflow is zero to every 16-bit reader
        const bool finite = m < 0x7f800000u, tiny = big < 7.888609e-31f;  // 2^-100
        const float inv = finite && !tiny ? __fdiv_rn(127.f, big) : 0.f;
        const float s = finite ? (tiny ? 0.f : __fdiv_rn(big, 127.f)) : __uint_as_float(0x7fffffffu);
        if (lane8 == 0) p.h_scale[row] = s;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int at = lane8 + i * WPR * 256;
            if (at >= p.c) continue;
            // rint(h * inv) from the 1.5 * 2^23 shifter: the low byte of the sum's
            // bits is the integer (|h * inv| <= 127; the product is rounded first, as
            // a separate multiply and rint would)
            uint32_t u[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] = __float_as_uint(__fadd_rn(__fmul_rn(x[i][e], inv), 12582912.f));
            const uint32_t lo = __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
            const uint32_t hi = __byte_perm(__byte_perm(u[4], u[5], 0x0040), __byte_perm(u[6], u[7], 0x0040), 0x5410);
            *reinterpret_cast<uint2*>(static_cast<int8_t*>(p.h) + row * p.h_stride + at) = make_uint2(lo, hi);
        }
    }
}

}  // namespace norm
}  // namespace fds
