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
// element against ~14 flops. A CTA is as wide as a row (a thread holds NCH
// chunks of 8 columns) and walks a contiguous range of rows, R at a time:
// * the vectors of a thread's columns are folded once per window into four fp32
//   coefficients a column that stay in registers,
//     x' = alpha * x + unit(y) * G + Gb    G = gate * post_w, Gb = gate * post_b
//     h  = unit(x') * W + Wb               W = w (1 + scale), Wb = b (1 + scale) + shift
//   (unit: the norm without its vectors);
// * R rows share each reduction's shuffles and barrier;
// * the next rows come through a ring of asynchronous copies in shared memory
//   that each warp fills and reads by itself (no CTA barrier), so that up to
//   192 KB per SM are in flight while the present rows pass through their
//   reductions.
// 29777 x 1160, 16-bit stream: 52.7 us, 5.2 TB/s (71 without the ring; issue slots
// 57 %, DRAM 55 % of its nominal rate); 6000 x 768, fp32 stream: 13.8 us; one row:
// 2.8 us, 1.9 of which an empty launch takes. A warp per row instead, its vectors
// read where they are used, is faster only while they stay in L1 and L2 (6000 x
// 768: 13.0 us with one vector for all, 19.5 with five that come from DRAM).
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
    int32_t x_out_wide;       // fp32 rows of x_out on 32-byte boundaries: 256-bit stores
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

// 8 parameters from element `at` (a multiple of 8), as they come from memory: a
// vector that is absent reads nothing. Loading and converting are separate, so
// that the loads of all vectors are in flight together.
struct Param8 {
    uint4 a, b;
};
__device__ __forceinline__ Param8 param_load(const void* p, bool f32, int64_t at) {
    Param8 r;
    r.a = r.b = make_uint4(0, 0, 0, 0);
    const uint4* q = reinterpret_cast<const uint4*>(static_cast<const char*>(p) + (f32 ? 4 : 2) * at);
    if (p != nullptr) r.a = __ldg(q);
    if (p != nullptr && f32) r.b = __ldg(q + 1);
    return r;
}
template <typename T>
__device__ __forceinline__ void param_value(const Param8& r, bool f32, bool present, float otherwise, float (&v)[8]) {
    if (f32) {
        const uint32_t u[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(u[e]);
    } else {
        unpack8<T>(r.a, v);
    }
    if (!present) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = otherwise;
    }
}

// Stores 8 fp32 values as one 256-bit access (32-byte aligned), or as two of 128 bits
__device__ __forceinline__ void store8(float* p, bool wide, const float (&v)[8]) {
    if (wide) {
        asm volatile("st.global.v8.f32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"f"(v[0]), "f"(v[1]), "f"(v[2]),
                     "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "l"(p)
                     : "memory");
    } else {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
}

struct Add {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
    static __device__ __forceinline__ float zero() { return 0.f; }
};
// the larger of two non-negative floats by their bits: infinities and, above them, NaN win
struct MaxBits {
    __device__ __forceinline__ float operator()(float a, float b) const {
        return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
    }
    static __device__ __forceinline__ float zero() { return 0.f; }
};

constexpr int kSlots = 5;       // reductions per group of rows at most
constexpr int kMaxWarps = 16;
template <int R>
constexpr int kReduceBytes = 2 * kSlots * kMaxWarps * R * 4;  // two sets of slots, used in turn

// Reduces v[r] (row r) over the CTA's threads, in place. Four rows share their
// shuffles: after two exchanging steps each 8-lane group holds one row. `red`
// is this reduction's own [kMaxWarps][R] block (slots alternate, so that one
// barrier separates its writes from the previous reads).
template <int R, typename Op>
__device__ __forceinline__ void reduce(float (&v)[R], float* red, Op op) {
    static_assert(R == 1 || R == 4, "one or four rows");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    float a = v[0];
    if constexpr (R == 4) {
        const bool hi = (lane & 16) != 0, odd = (lane & 8) != 0;
        a = op(hi ? v[2] : v[0], __shfl_xor_sync(0xffffffffu, hi ? v[0] : v[2], 16));
        const float b = op(hi ? v[3] : v[1], __shfl_xor_sync(0xffffffffu, hi ? v[1] : v[3], 16));
        a = op(odd ? b : a, __shfl_xor_sync(0xffffffffu, odd ? a : b, 8));
    } else {
        a = op(a, __shfl_xor_sync(0xffffffffu, a, 16));
        a = op(a, __shfl_xor_sync(0xffffffffu, a, 8));
    }
#pragma unroll
    for (int d = 4; d > 0; d >>= 1) a = op(a, __shfl_xor_sync(0xffffffffu, a, d));
    if (warps == 1) {
#pragma unroll
        for (int r = 0; r < R; ++r) v[r] = __shfl_sync(0xffffffffu, a, 8 * r);
        return;
    }
    if ((lane & 7) == 0 && (lane >> 3) < R) red[warp * R + (lane >> 3)] = a;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) v[r] = Op::zero();
    if (warps <= 4) {
        for (int w = 0; w < warps; ++w) {
            if constexpr (R == 4) {
                const float4 t = *reinterpret_cast<const float4*>(red + 4 * w);
                v[0] = op(v[0], t.x), v[1] = op(v[1], t.y), v[2] = op(v[2], t.z), v[3] = op(v[3], t.w);
            } else {
                v[0] = op(v[0], red[w]);
            }
        }
    } else if constexpr (R == 4) {
        // many warps: two lanes take a warp's four rows, two rows each
        float2 t = (lane >> 1) < warps ? *reinterpret_cast<const float2*>(red + 2 * lane) : make_float2(0.f, 0.f);
#pragma unroll
        for (int d = 2; d < 32; d <<= 1) {
            t.x = op(t.x, __shfl_xor_sync(0xffffffffu, t.x, d));
            t.y = op(t.y, __shfl_xor_sync(0xffffffffu, t.y, d));
        }
        const float ox = __shfl_xor_sync(0xffffffffu, t.x, 1), oy = __shfl_xor_sync(0xffffffffu, t.y, 1);
        const bool upper = (lane & 1) != 0;
        v[0] = upper ? ox : t.x, v[1] = upper ? oy : t.y, v[2] = upper ? t.x : ox, v[3] = upper ? t.y : oy;
    } else {
        float t = (lane & 15) < warps ? red[lane & 15] : 0.f;
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) t = op(t, __shfl_xor_sync(0xffffffffu, t, d));
        v[0] = t;
    }
}

// The largest magnitude of 8 values (packed pairs; a NaN anywhere gives NaN).
template <typename T>
__device__ __forceinline__ float largest(const uint4& r);
template <>
__device__ __forceinline__ float largest<__half>(const uint4& r) {
    const __half2* h = reinterpret_cast<const __half2*>(&r);
    const __half2 m = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
    return __half2float(__hmax_nan(__low2half(m), __high2half(m)));
}
template <>
__device__ __forceinline__ float largest<__nv_bfloat16>(const uint4& r) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
    return __bfloat162float(__hmax_nan(__low2bfloat16(m), __high2bfloat16(m)));
}

// The scale of a quantised row with largest magnitude `big`, and the factor of
// its values: a row with an infinity or a NaN gets the scale NaN (its products say
// so), one whose 127 / max could overflow is zero.
__device__ __forceinline__ float row_scale(float big, float& inv) {
    const bool finite = __float_as_uint(big) < 0x7f800000u, tiny = big < 7.888609e-31f;  // 2^-100
    inv = finite && !tiny ? __fdiv_rn(127.f, big) : 0.f;
    return finite ? (tiny ? 0.f : __fdiv_rn(big, 127.f)) : __uint_as_float(0x7fffffffu);
}

// rint(v * inv) of 8 values as bytes, from the 1.5 * 2^23 shifter: the low byte of
// the sum's bits is the integer (|v * inv| <= 127; the product is rounded first, as
// a separate multiply and rint would).
__device__ __forceinline__ uint2 quantise8(const float (&v)[8], float inv) {
    uint32_t u[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] = __float_as_uint(__fadd_rn(__fmul_rn(v[e], inv), 12582912.f));
    return make_uint2(__byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(u[4], u[5], 0x0040), __byte_perm(u[6], u[7], 0x0040), 0x5410));
}

// t <- LayerNorm / RMS norm of its rows without the vectors (columns past c hold
// 0 and count for nothing)
template <int NCH, int R>
__device__ __forceinline__ void unit(float (&t)[R][NCH][8], int kind, const bool (&in)[NCH], float inv_c, float eps,
                                     float* red, int slot) {
    float s[R];
    if (kind == kLayer) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            s[r] = 0.f;
#pragma unroll
            for (int i = 0; i < NCH; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) s[r] += t[r][i][e];
        }
        reduce<R>(s, red + slot * kMaxWarps * R, Add{});
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float mean = s[r] * inv_c;
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const float m = in[i] ? mean : 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) t[r][i][e] -= m;
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        s[r] = 0.f;
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) s[r] = fmaf(t[r][i][e], t[r][i][e], s[r]);
    }
    reduce<R>(s, red + (slot + 1) * kMaxWarps * R, Add{});
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float k = rsqrtf(s[r] * inv_c + eps);
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) t[r][i][e] *= k;
    }
}

// What a launch computes: the norm before a block alone, or both sides of a block
// (with y).
enum Mode : int { kNormOnly = 0, kBoth = 1 };

// Ring depth in rows, and the 16-byte pieces of a row's chunk (x, then y).
template <int NCH, int kMode, bool kXf32>
struct Ring {
    static constexpr int kPieces = (kXf32 ? 2 : 1) + (kMode == kBoth ? 1 : 0);
    static constexpr int kRows = 8 / NCH;  // at most 192 KB per SM
    static constexpr int bytes(int threads) { return kRows * NCH * kPieces * 16 * threads; }
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}
__device__ __forceinline__ uint4 ld_shared_u4(uint32_t addr) {
    const int4 v = ld_shared_v4(addr);
    return make_uint4(static_cast<uint32_t>(v.x), static_cast<uint32_t>(v.y), static_cast<uint32_t>(v.z),
                      static_cast<uint32_t>(v.w));
}

// G, Gb of chunk column `at` (1 and 0 where a vector is absent)
template <typename T>
__device__ __forceinline__ void block_coefficients(const Params& p, int64_t window, int at, float (&G)[8], float (&Gb)[8]) {
    const bool pf = p.param_f32 != 0;
    const Param8 w = param_load(p.post_w, pf, at), b = param_load(p.post_b, pf, at),
                 g = param_load(p.gate, pf, window * p.gate_stride + at);
    float v[8];
    param_value<T>(w, pf, p.post_w != nullptr, 1.f, G);
    param_value<T>(b, pf, p.post_b != nullptr, 0.f, Gb);
    param_value<T>(g, pf, p.gate != nullptr, 1.f, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) G[e] *= v[e], Gb[e] *= v[e];
}
// W, Wb likewise
template <typename T>
__device__ __forceinline__ void norm_coefficients(const Params& p, int64_t window, int at, float (&W)[8], float (&Wb)[8]) {
    const bool pf = p.param_f32 != 0;
    const Param8 w = param_load(p.w, pf, at), b = param_load(p.b, pf, at),
                 s = param_load(p.scale, pf, window * p.mod_stride + at), t = param_load(p.shift, pf, window * p.mod_stride + at);
    float v[8];
    param_value<T>(w, pf, p.w != nullptr, 1.f, W);
    param_value<T>(b, pf, p.b != nullptr, 0.f, Wb);
    param_value<T>(s, pf, p.scale != nullptr, 0.f, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) W[e] = fmaf(W[e], v[e], W[e]), Wb[e] = fmaf(Wb[e], v[e], Wb[e]);
    param_value<T>(t, pf, p.shift != nullptr, 0.f, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) Wb[e] += v[e];
}

template <typename T, int NCH, int R, int kMode, bool kXf32, bool kQuant>
__global__ void __launch_bounds__(32 * kMaxWarps, 1) residual_norm_kernel(const Params p) {
    using Rg = Ring<NCH, kMode, kXf32>;
    constexpr bool kKeep = NCH < 4;  // coefficients in registers; the widest rows read them again per group
    static_assert((Rg::kRows & (Rg::kRows - 1)) == 0 && Rg::kRows >= R, "ring rows");
    __shared__ __align__(16) float red_all[kReduceBytes<R> / 4];
    extern __shared__ __align__(16) uint8_t ring_raw[];
    grid_launch_dependents();
    grid_dependency_wait();
    const int row_begin = static_cast<int>(static_cast<int64_t>(p.rows) * blockIdx.x / gridDim.x);
    const int row_end = static_cast<int>(static_cast<int64_t>(p.rows) * (blockIdx.x + 1) / gridDim.x);
    const float inv_c = 1.f / static_cast<float>(p.c);
    int at[NCH];
    bool in[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        at[i] = 8 * static_cast<int>(threadIdx.x + i * blockDim.x);
        in[i] = at[i] < p.c;
    }
    // chunk i of ring row s: x's 16 or 32 bytes a thread, then y's 16. An fp32
    // chunk is copied in 16-byte pieces that are contiguous over the lanes (whole
    // sectors) and read as each thread's 32 bytes, so the lanes of a warp hand
    // pieces to one another.
    const uint32_t ring = smem_u32(ring_raw), step = 16u * blockDim.x;
    const auto chunk = [&](int s, int i) { return ring + ((s * NCH + i) * Rg::kPieces) * step; };
    const uint32_t unit0 = 2 * (threadIdx.x & ~31u) + (threadIdx.x & 31);  // fp32: this thread copies pieces unit0, unit0 + 32
    // the next row to fetch; this thread's addresses walk with it
    int next = row_begin;
    const char* fx = static_cast<const char*>(p.x) +
                     (static_cast<int64_t>(row_begin) * p.x_stride + (kXf32 ? 4 * unit0 : at[0])) * (kXf32 ? 4 : 2);
    const char* fy = static_cast<const char*>(p.y) + (static_cast<int64_t>(row_begin) * p.y_stride + at[0]) * 2;
    const int64_t fx_step = p.x_stride * (kXf32 ? 4 : 2), fy_step = p.y_stride * 2;
    const auto fetch = [&]() {  // one commit group per row, empty past the end
        if (next < row_end) {
            const int s = (next - row_begin) & (Rg::kRows - 1);
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int first = 8 * i * static_cast<int>(blockDim.x);  // the chunk's first column
                if constexpr (kXf32) {
                    const char* g = fx + static_cast<int64_t>(first) * 4;
                    const int col = first + 4 * static_cast<int>(unit0);
                    if (col < p.c) copy16(chunk(s, i) + 16u * unit0, g);
                    if (col + 128 < p.c) copy16(chunk(s, i) + 16u * (unit0 + 32), g + 512);
                } else if (in[i]) {
                    copy16(chunk(s, i) + 16u * threadIdx.x, fx + static_cast<int64_t>(first) * 2);
                }
                if constexpr (kMode == kBoth)
                    if (in[i])
                        copy16(chunk(s, i) + (Rg::kPieces - 1) * step + 16u * threadIdx.x, fy + static_cast<int64_t>(first) * 2);
            }
        }
        copy_commit();
        ++next;
        fx += fx_step;
        fy += fy_step;
    };
#pragma unroll
    for (int r = 0; r < Rg::kRows; ++r) fetch();

    char* ox = static_cast<char*>(p.x_out) + (static_cast<int64_t>(row_begin) * p.x_out_stride + at[0]) * (kXf32 ? 4 : 2);
    char* oh = static_cast<char*>(p.h) + (static_cast<int64_t>(row_begin) * p.h_stride + at[0]) * (kQuant ? 1 : 2);
    const int64_t ox_step = p.x_out_stride * (kXf32 ? 4 : 2), oh_step = p.h_stride * (kQuant ? 1 : 2);
    float G[kKeep ? NCH : 1][8], Gb[kKeep ? NCH : 1][8], W[kKeep ? NCH : 1][8], Wb[kKeep ? NCH : 1][8];
    int window = 0, window_end = 0, parity = 0;
    for (int this_row = row_begin; this_row < row_end;) {
        if (this_row >= window_end) {
            window = this_row / p.length;
            window_end = p.rows - window * p.length > p.length ? (window + 1) * p.length : p.rows;
            if constexpr (kKeep) {
#pragma unroll
                for (int i = 0; i < NCH; ++i) {
                    if (in[i]) {
                        if constexpr (kMode == kBoth) block_coefficients<T>(p, window, at[i], G[i], Gb[i]);
                        norm_coefficients<T>(p, window, at[i], W[i], Wb[i]);
                    } else {  // columns past c stay 0
#pragma unroll
                        for (int e = 0; e < 8; ++e) G[i][e] = Gb[i][e] = W[i][e] = Wb[i][e] = 0.f;
                    }
                }
            }
        }
        const int this_n = min(R, min(row_end, window_end) - this_row);  // a group's rows are of one window
        const int slot = this_row - row_begin;
        copy_wait<Rg::kRows - R>();
        __syncwarp();
        const auto load_x = [&](int r, int i, float (&v)[8]) {
            const bool on = in[i] && r < this_n;
            const int s = (slot + r) & (Rg::kRows - 1);
            const uint32_t from = chunk(s, i) + (kXf32 ? 32u : 16u) * threadIdx.x;
            const uint4 a = on ? ld_shared_u4(from) : make_uint4(0, 0, 0, 0);
            if constexpr (kXf32) {
                const uint4 b = on ? ld_shared_u4(from + 16) : make_uint4(0, 0, 0, 0);
                const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(u[e]);
            } else {
                unpack8<T>(a, v);
            }
        };
        float x[R][NCH][8];
        float* red = red_all + parity * kSlots * kMaxWarps * R;
        parity ^= 1;
        if constexpr (kMode == kBoth) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < NCH; ++i) {
                    const bool on = in[i] && r < this_n;
                    const uint32_t from =
                        chunk((slot + r) & (Rg::kRows - 1), i) + (Rg::kPieces - 1) * step + 16u * threadIdx.x;
                    unpack8<T>(on ? ld_shared_u4(from) : make_uint4(0, 0, 0, 0), x[r][i]);
                }
            if (p.post != kNone) unit<NCH, R>(x, p.post, in, inv_c, p.eps, red, 0);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < NCH; ++i) {
                    if constexpr (!kKeep) {
                        if (!in[i]) continue;
                        block_coefficients<T>(p, window, at[i], G[0], Gb[0]);
                    }
                    constexpr int kI = kKeep ? 1 : 0;
                    float v[8];
                    load_x(r, i, v);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        x[r][i][e] = fmaf(p.alpha, v[e], fmaf(x[r][i][e], G[kI * i][e], Gb[kI * i][e]));
                    if (!in[i] || r >= this_n) continue;
                    const float(&o)[8] = x[r][i];
                    char* to = ox + r * ox_step + static_cast<int64_t>(8 * i) * blockDim.x * (kXf32 ? 4 : 2);
                    if constexpr (kXf32)
                        store8(reinterpret_cast<float*>(to), p.x_out_wide != 0, o);
                    else
                        *reinterpret_cast<uint4*>(to) = make_uint4(pack2<T>(o[0], o[1]), pack2<T>(o[2], o[3]),
                                                                   pack2<T>(o[4], o[5]), pack2<T>(o[6], o[7]));
                }
            ox += this_n * ox_step;
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < NCH; ++i) load_x(r, i, x[r][i]);
        }
        __syncwarp();  // every lane has read its slots
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (r < this_n) fetch();  // into them
        if (p.h != nullptr) {
            if (p.norm != kNone) unit<NCH, R>(x, p.norm, in, inv_c, p.eps, red, 2);
            float big[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                big[r] = 0.f;
#pragma unroll
                for (int i = 0; i < NCH; ++i) {
                    constexpr int kI = kKeep ? 1 : 0;
                    if constexpr (!kKeep) {
                        if (!in[i]) continue;
                        norm_coefficients<T>(p, window, at[i], W[0], Wb[0]);
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        x[r][i][e] = fmaf(x[r][i][e], W[kI * i][e], Wb[kI * i][e]);
                        if constexpr (kQuant) big[r] = MaxBits{}(big[r], fabsf(x[r][i][e]));
                    }
                }
            }
            if constexpr (kQuant) reduce<R>(big, red + 4 * kMaxWarps * R, MaxBits{});
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (r >= this_n) continue;
                float inv = 0.f;
                if constexpr (kQuant) {
                    const float scale = row_scale(big[r], inv);
                    if (threadIdx.x == 0) p.h_scale[this_row + r] = scale;
                }
#pragma unroll
                for (int i = 0; i < NCH; ++i) {
                    if (!in[i]) continue;
                    const float(&v)[8] = x[r][i];
                    char* to = oh + r * oh_step + static_cast<int64_t>(8 * i) * blockDim.x * (kQuant ? 1 : 2);
                    if constexpr (kQuant) {
                        *reinterpret_cast<uint2*>(to) = quantise8(v, inv);
                    } else {
                        *reinterpret_cast<uint4*>(to) = make_uint4(
                            pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
                    }
                }
            }
        }
        oh += this_n * oh_step;
        this_row += this_n;
    }
}

// The quantiser alone: a warp per kR rows (NCH 16-byte chunks a lane each), the
// values packed in registers between the maximum and the rounding, so that many
// warps fit an SM and no row waits at a barrier for another. (The ring above
// with the same arithmetic: 48000 x 4096 at 109 us against 86 us here, 6000 x
// 1024 at 6.7 us against 3.1.)
constexpr int kQuantWarps = 4;

template <typename T, int NCH, int kR>
__global__ void __launch_bounds__(32 * kQuantWarps) quantise_rows_kernel(const Params p) {
    grid_launch_dependents();
    grid_dependency_wait();
    const int row0 = (static_cast<int>(blockIdx.x) * kQuantWarps + static_cast<int>(threadIdx.x >> 5)) * kR;
    const int at = 8 * static_cast<int>(threadIdx.x & 31);
    uint4 raw[kR][NCH];
    const T* x = static_cast<const T*>(p.x) + row0 * p.x_stride + at;
#pragma unroll
    for (int r = 0; r < kR; ++r)
#pragma unroll
        for (int i = 0; i < NCH; ++i)
            raw[r][i] = row0 + r < p.rows && at + 256 * i < p.c ? *reinterpret_cast<const uint4*>(x + r * p.x_stride + 256 * i)
                                                                : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < kR; ++r) {
        if (row0 + r >= p.rows) return;
        float big = 0.f;
#pragma unroll
        for (int i = 0; i < NCH; ++i) big = MaxBits{}(big, largest<T>(raw[r][i]));
        big = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(big)));
        float inv;
        const float scale = row_scale(big, inv);
        if (at == 0) p.h_scale[row0 + r] = scale;
        int8_t* h = static_cast<int8_t*>(p.h) + (row0 + r) * p.h_stride + at;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            if (at + 256 * i >= p.c) continue;
            float v[8];
            unpack8<T>(raw[r][i], v);
            *reinterpret_cast<uint2*>(h + 256 * i) = quantise8(v, inv);
        }
    }
}

}  // namespace norm
}  // namespace fds
