// gemv_i8_kernel.cuh - the 8-bit linear layer for a few tokens (one to eight
// rows of A): D[m, n] = (sum_k A[m, k] W[n, k]) * (a_scale[m] * w_scale[n]) (+ bias)
// with the epilogues of gemm_kernel.cuh.
//
// Bound by reading W once (n * k bytes) and, below a few MB, by latency: a
// 128-row tensor-core tile would leave most SMs without work at the usual n.
// One warp takes two rows of W -- the two columns of a rotation for the RoPE
// epilogue, neighbours otherwise -- and walks k in 16-byte chunks per lane,
// kUnroll chunks of each row in flight; A (a few rows) comes through L1. The
// products are summed in 32-bit integers (dp4a), exactly, so the result does
// not depend on the split of k over lanes. 768 -> 2304, one row: 1.95 us, as long as
// an empty launch; 4096 -> 4096 in us (this / the 64-column tiles of gemm_kernel):
// one row 4.3 / 13.4, eight rows 7.2 / 12.
#pragma once

#include <cstdint>

#include "fds_b200.h"
#include "fds_ptx.cuh"
#include "gemm_kernel.cuh"

namespace fds {
namespace gemv {

constexpr int kWarps = 4;
constexpr int kMaxRows = 8;

struct Params {
    const int8_t* a;
    const int8_t* w;
    const float* a_scale;
    const float* w_scale;
    const void* bias;
    void* out;
    const float* cos_t;
    const float* sin_t;
    int64_t a_stride, w_stride, out_stride;
    int32_t m, n, k;
    int32_t seq_len, rope_cols;
};

__device__ __forceinline__ uint4 ldg_stream(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

__device__ __forceinline__ int dot16(const uint4& a, const uint4& b, int acc) {
    acc = __dp4a(static_cast<int>(a.x), static_cast<int>(b.x), acc);
    acc = __dp4a(static_cast<int>(a.y), static_cast<int>(b.y), acc);
    acc = __dp4a(static_cast<int>(a.z), static_cast<int>(b.z), acc);
    return __dp4a(static_cast<int>(a.w), static_cast<int>(b.w), acc);
}

template <typename T, int M, int kEpi>
__global__ void __launch_bounds__(32 * kWarps) gemv_i8_kernel(const Params p) {
    constexpr int kUnroll = M <= 2 ? 4 : 2;
    grid_launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31;
    const int g = static_cast<int>(blockIdx.x) * kWarps + static_cast<int>(threadIdx.x >> 5);
    if (2 * g >= p.n) return;
    const int r0 = kEpi == gemm::kRope ? (g >> 5) * 64 + (g & 31) : 2 * g;
    const int r1 = kEpi == gemm::kRope ? r0 + 32 : r0 + 1;
    const int8_t* w0 = p.w + r0 * p.w_stride;
    const int8_t* w1 = p.w + r1 * p.w_stride;

    int acc0[M], acc1[M];
#pragma unroll
    for (int i = 0; i < M; ++i) acc0[i] = acc1[i] = 0;
    for (int base = 16 * lane; base < p.k; base += 512 * kUnroll) {
        uint4 x0[kUnroll], x1[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const bool in = base + 512 * u < p.k;
            x0[u] = in ? ldg_stream(w0 + base + 512 * u) : make_uint4(0, 0, 0, 0);
            x1[u] = in ? ldg_stream(w1 + base + 512 * u) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            if (base + 512 * u >= p.k) break;
#pragma unroll
            for (int i = 0; i < M; ++i) {
                // rows past m repeat the last one; they are not written
                const int8_t* ar = p.a + (i < p.m ? i : p.m - 1) * p.a_stride;
                const uint4 x = __ldg(reinterpret_cast<const uint4*>(ar + base + 512 * u));
                acc0[i] = dot16(x, x0[u], acc0[i]);
                acc1[i] = dot16(x, x1[u], acc1[i]);
            }
        }
    }
    int s0 = 0, s1 = 0;  // this lane's row (lane < M)
#pragma unroll
    for (int i = 0; i < M; ++i) {
        const int t0 = __reduce_add_sync(0xffffffffu, acc0[i]);
        const int t1 = __reduce_add_sync(0xffffffffu, acc1[i]);
        if (lane == i) s0 = t0, s1 = t1;
    }
    if (lane >= M || lane >= p.m) return;
    const float as = __ldg(p.a_scale + lane);
    const T* bias = static_cast<const T*>(p.bias);
    float y0 = fmaf(static_cast<float>(s0), as * __ldg(p.w_scale + r0), bias != nullptr ? gemm::to_f<T>(bias[r0]) : 0.f);
    float y1 = fmaf(static_cast<float>(s1), as * __ldg(p.w_scale + r1), bias != nullptr ? gemm::to_f<T>(bias[r1]) : 0.f);
    if constexpr (kEpi == gemm::kAccum) {
        float* o = static_cast<float*>(p.out) + lane * p.out_stride;
        o[r0] = __fadd_rn(o[r0], y0);
        o[r1] = __fadd_rn(o[r1], y1);
    } else {
        if (kEpi == gemm::kRope && r0 < p.rope_cols) {
            const int64_t at = static_cast<int64_t>(lane % p.seq_len) * 64 + (r0 & 63);
            gemm::rotate(y0, y1, __ldg(p.cos_t + at), __ldg(p.sin_t + at));
        }
        T* o = static_cast<T*>(p.out) + lane * p.out_stride;
        o[r0] = static_cast<T>(y0);
        o[r1] = static_cast<T>(y1);
    }
}

}  // namespace gemv
}  // namespace fds
