// window_kernel.cuh - attention over a sliding window of keys with a few first
// keys that stay visible (sinks), head width 64.
//
// Query i of window b sits at position p = q_start[b] + i of the key sequence
// and sees key j iff j < kv_len[b], j <= p + right and (j >= p - left or
// j < sinks); O_i = softmax_j(q_i . k_j * scale) V over the keys it sees, 0 if
// it sees none. Query head h reads key head h / (heads / kv_heads).
//
// Two kernels, chosen by the number of query rows that share a key head:
//
// * window_tile_kernel: tensor cores, one CTA per 128 query rows of a (window,
//   head), walking 128-column tiles over the union of the keys its rows see.
//   The columns are the sinks before the union's window part, rounded up to 8
//   (one swizzle atom), then the window part, packed: a tile may hold both, so
//   the sinks cost their own columns and not a tile of their own. The first
//   column of the window part is the first key that the CTA's first row sees
//   (TMA rows start anywhere), which leaves at most two partly seen tiles per
//   end. A tile that every row of a warp sees whole runs the mask-free step.
//   The step is the bidirectional attention's (attn_kernel.cuh RowSoftmax); a
//   CTA has one query tile and half an SM (128 + 128 threads, 256 TMEM
//   columns, 98 KB), because a window is a handful of tiles: the start and
//   the epilogue of one CTA run under the tiles of its neighbour, and a
//   128-row tile overlaps fewer keys that its rows do not see than a 256-row
//   unit. With few query tiles and many key tiles the column tiles of a unit
//   are dealt to a cluster of up to 8 CTAs, whose partial (O, max, sum) are
//   merged through distributed shared memory in rank order.
// * window_step_kernel: up to 8 query rows per key head (a decoding step):
//   bound by reading the keys and values once. 8 lanes hold a key's 64
//   values, 16 keys run abreast in a CTA, and the keys of a unit are dealt to a
//   cluster of up to 8 CTAs merged the same way.
//
// Keys and values that no row of a unit sees may hold anything (a cache's
// unwritten rows): their scores are replaced, and their value rows are zeroed
// in shared memory before the P V product reads them (0 times an infinity
// would not be 0). The tile kernel does multiply a value row that one row of
// the tile sees by the zero weights of the rows that do not.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "attn_kernel.cuh"
#include "norm_kernel.cuh"

namespace fds {
namespace window {

struct Params {
    const void* q;  // step kernel (the tile kernel reads through tensor maps)
    const void* k;
    const void* v;
    void* out;
    const int32_t* q_start;  // [batch] or null (0)
    const int32_t* kv_len;   // [batch] or null (k_len)
    int32_t* status;
    int32_t* status_host;
    int64_t timeout_ns;
    int64_t q_stride[3], k_stride[3], v_stride[3], out_stride[3];  // elements: batch, row, head
    int32_t heads, kv_heads, q_len, k_len;
    int32_t left, right, sinks;
    int32_t row_blocks;  // ceil(q_len / 128)
    float scale_log2;
};

// Positions stay within +-2^30 (the host bounds left, right, lengths by 2^28),
// so that sums of three fit 32 bits.
__device__ __forceinline__ int first_position(const Params& p, int b) {
    return p.q_start != nullptr ? min(max(p.q_start[b], -(1 << 30)), 1 << 30) : 0;
}
__device__ __forceinline__ int key_end(const Params& p, int b) {
    return p.kv_len != nullptr ? min(max(p.kv_len[b], 0), p.k_len) : p.k_len;
}

// The columns of a unit of query positions [p0, p1]: keys [0, n_sink), padded
// to s8 columns (a multiple of 8), then keys [begin, begin + n_win).
struct Columns {
    int p0, kv_end, n_sink, s8, begin, n_win;
    __device__ __forceinline__ Columns(const Params& p, int b, int row0, int rows) {
        p0 = first_position(p, b) + row0;
        kv_end = key_end(p, b);
        const int end = min(kv_end, p0 + rows - 1 + p.right + 1);
        begin = max(0, p0 - p.left);
        n_sink = min(p.sinks, kv_end);
        if (begin < n_sink) {  // the sinks touch the window part: one range from key 0
            begin = 0;
            n_sink = 0;
        }
        s8 = (n_sink + 7) & ~7;
        n_win = max(0, end - begin);
    }
    __device__ __forceinline__ int total() const { return s8 + n_win; }
};

// ---------------------------------------------------------------- tile kernel

constexpr int kTileThreads = 256;
constexpr int kTileRegs = 128;  // per thread at launch: 65536 / (2 CTAs x 256)
constexpr int kSoftmaxRegs = 208, kControlRegs = 48;
static_assert(128 * kSoftmaxRegs + 128 * kControlRegs <= kTileThreads * kTileRegs, "register split exceeds the launch pool");
constexpr int kKStages = 3, kVStages = 2;
constexpr int kMaxSplit = 8;

struct TileSmem {
    static constexpr int q = 0;
    static constexpr int k = q + kTileBytes;
    static constexpr int v = k + kKStages * kTileBytes;
    static constexpr int bars = v + kVStages * kTileBytes;
    static constexpr int kQ = 0;
    static constexpr int kKFull = 1;
    static constexpr int kVFull = kKFull + kKStages;
    static constexpr int kKEmpty = kVFull + kVStages;
    static constexpr int kVEmpty = kKEmpty + kKStages;
    static constexpr int kSFull = kVEmpty + kVStages;
    static constexpr int kSFree = kSFull + 1;
    static constexpr int kPHalf = kSFree + 1;
    static constexpr int kPFull = kPHalf + 1;
    static constexpr int kPvDone = kPFull + 1;
    static constexpr int kDrain = kPvDone + 1;
    static constexpr int kNumBars = kDrain + 1;
    static constexpr int misc = bars + kNumBars * 8;  // the bounded waits' block (attn_kernel.cuh Smem::misc)
    static constexpr int total = misc + 48;
    static constexpr int alloc = total + 1024;
    // a split unit's partial rows, [66][128] floats (64 of O, max, sum), over the K ring
    static constexpr int part = k;
    static_assert(66 * 128 * 4 <= kKStages * kTileBytes, "partial rows");
    static_assert(2 * (alloc + 1024) <= 228 * 1024, "two CTAs per SM");
};
constexpr int kTmemColsTile = 256;  // S [0, 128), P [128, 192), O [192, 256)
constexpr int kTP = 128, kTO = 192;

struct Maps {
    CUtensorMap q, k, v;    // boxes of 128 rows
    CUtensorMap k8, v8;     // boxes of 8 rows (tiles that hold sinks and window keys)
};

// Columns [x0, x0 + 128) of the unit's keys or values into `dst` (128 rows of
// 128 bytes, 16384 bytes in all; rows past the tensor read as zero).
__device__ __forceinline__ void load_columns(uint32_t dst, const CUtensorMap* map, const CUtensorMap* map8, uint32_t bar,
                                             const Columns& c, int x0, int head, int b) {
    mbar_arrive_expect_tx(bar, kTileBytes);
    if (x0 >= c.s8) {
        tma_load_4d(dst, map, bar, 0, head, c.begin + x0 - c.s8, b);
    } else if (x0 + kBlockN <= c.s8) {
        tma_load_4d(dst, map, bar, 0, head, x0, b);
    } else {
#pragma unroll 1
        for (int r = 0; r < kBlockN; r += 8) {
            const int x = x0 + r;
            tma_load_4d(dst + r * 128, map8, bar, 0, head, x < c.s8 ? x : c.begin + x - c.s8, b);
        }
    }
}

// Merge of a split unit: CTA `rank` of the cluster takes rows [128 rank / split,
// 128 (rank + 1) / split), `split` threads a row; parts are folded in rank
// order, so the result does not depend on their timing.
template <typename T>
__device__ __forceinline__ void merge_parts(uint32_t part, int split, int rank, int tid, int rows, T* out,
                                            int64_t out_stride) {
    const int row = rank * (kBlockM / split) + tid / split;
    const int width = kHeadDim / split, c0 = (tid % split) * width;  // this thread's columns: 32, 16 or 8
    float m = -INFINITY;
    for (int r = 0; r < split; ++r) m = fmaxf(m, ld_cluster_f32(map_to_rank(part + 512u * 64 + 4u * row, r)));
    float l = 0.f, f[kMaxSplit];
#pragma unroll
    for (int r = 0; r < kMaxSplit; ++r) {
        f[r] = 0.f;
        if (r >= split) continue;
        const uint32_t at = map_to_rank(part + 4u * row, r);
        const float mr = ld_cluster_f32(at + 512u * 64);
        f[r] = mr == -INFINITY ? 0.f : ex2_approx(mr - m);
        l = fmaf(ld_cluster_f32(at + 512u * 65), f[r], l);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
    for (int c = c0; c < c0 + width; c += 8) {
        float acc[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = 0.f;
#pragma unroll
        for (int r = 0; r < kMaxSplit; ++r) {
            if (r >= split) continue;
            const uint32_t at = map_to_rank(part + 4u * row, r);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = fmaf(ld_cluster_f32(at + 512u * (c + e)), f[r], acc[e]);
        }
        if (row < rows)
            *reinterpret_cast<uint4*>(out + row * out_stride + c) =
                make_uint4(norm::pack2<T>(acc[0] * inv, acc[1] * inv), norm::pack2<T>(acc[2] * inv, acc[3] * inv),
                           norm::pack2<T>(acc[4] * inv, acc[5] * inv), norm::pack2<T>(acc[6] * inv, acc[7] * inv));
    }
}

template <typename T>
__global__ void __launch_bounds__(kTileThreads, 2) window_tile_kernel(const __grid_constant__ Maps maps, const Params p) {
    using S = TileSmem;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    const uint32_t sbase = (raw_addr + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (sbase - raw_addr);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::bars);
    const WaitCtl ctl{sbase + S::misc};
    const auto bar = [&](int idx) { return sbase + S::bars + 8u * idx; };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t split = cluster_nctarank(), rank = cluster_ctarank();
    grid_launch_dependents();

    if (threadIdx.x == 0) {
        mbar_init(&bars[S::kQ], 1);
        for (int s = 0; s < kKStages; ++s) mbar_init(&bars[S::kKFull + s], 1), mbar_init(&bars[S::kKEmpty + s], 1);
        for (int s = 0; s < kVStages; ++s) mbar_init(&bars[S::kVFull + s], 1), mbar_init(&bars[S::kVEmpty + s], 1);
        mbar_init(&bars[S::kSFull], 1);
        mbar_init(&bars[S::kSFree], 4);  // one arrival per softmax warp
        mbar_init(&bars[S::kPHalf], 4);
        mbar_init(&bars[S::kPFull], 4);
        mbar_init(&bars[S::kPvDone], 1);
        mbar_init(&bars[S::kDrain], 1);
        st_shared_volatile_u32(ctl.misc + 4, 0);
        st_shared_u64(ctl.misc + 8, reinterpret_cast<uint64_t>(p.status));
        st_shared_u64(ctl.misc + 16, static_cast<uint64_t>(p.timeout_ns > 0 ? p.timeout_ns : kDefaultTimeoutNs));
        st_shared_u64(ctl.misc + 32, reinterpret_cast<uint64_t>(p.status_host));
        fence_barrier_init();
        fence_proxy_async_smem();
    }
    if (warp == 1 && lane == 0) {
        prefetch_tensormap(&maps.q);
        prefetch_tensormap(&maps.k);
        prefetch_tensormap(&maps.v);
    }
    if (warp == 2) {
        tmem_alloc(reinterpret_cast<uint32_t*>(smem + S::misc), kTmemColsTile);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    grid_dependency_wait();
    const uint32_t tmem = *reinterpret_cast<uint32_t*>(smem + S::misc);

    const int unit = static_cast<int>(blockIdx.x / split);
    const int rb = unit % p.row_blocks;
    const int bh = unit / p.row_blocks;
    const int h = bh % p.heads, b = bh / p.heads;
    const int hk = h / (p.heads / p.kv_heads);
    const int row0 = rb * kBlockM;
    const int rows = min(kBlockM, p.q_len - row0);
    const Columns cols(p, b, row0, rows);
    const int tiles = (cols.total() + kBlockN - 1) / kBlockN;
    const int per = (tiles + static_cast<int>(split) - 1) / static_cast<int>(split);
    const int t0 = min(tiles, static_cast<int>(rank) * per), t1 = min(tiles, t0 + per);  // this CTA's tiles

    if (warp >= 4) {
        setmaxnreg_inc<kSoftmaxRegs>();
        const int row = ((warp & 3) << 5) + lane;
        const uint32_t lane_addr = static_cast<uint32_t>((warp & 3) * 32) << 16;
        RowSoftmax<T, false> rs;
        rs.tS = tmem + lane_addr;
        rs.tP = tmem + lane_addr + kTP;
        rs.tO = tmem + lane_addr + kTO;
        rs.sl = p.scale_log2;
        rs.qrow = 0;
        rs.s_full = bar(S::kSFull);
        rs.s_free = bar(S::kSFree);
        rs.p_half = bar(S::kPHalf);
        rs.p_full = bar(S::kPFull);
        rs.pv_done = bar(S::kPvDone);
        rs.ctl = ctl;
        rs.lane = lane;
        rs.i = 0;
        rs.kv_end = 0;
        rs.t_begin = t0;
        rs.m_run = -INFINITY;
        rs.l_run = 0.f;
        rs.s_parity = 0;
        rs.pv_parity = 0;
        // this row's columns: the sinks (or, where they lie in the window part,
        // those of them up to p + right), and [lo, hi)
        const int pos = cols.p0 + row;
        const int hi = cols.s8 + min(pos + p.right + 1, cols.kv_end) - cols.begin;
        const int lo = cols.s8 + max(pos - p.left - cols.begin, 0);
        const int first = cols.n_sink > 0 ? cols.n_sink : min(p.sinks, hi);
        bool ok = true;
        for (int t = t0; ok && t < t1; ++t) {
            const int n0 = t * kBlockN;
            rs.w_first = first - n0;
            rs.w_lo = lo - n0;
            rs.w_hi = hi - n0;
            const bool whole = rs.w_first >= kBlockN || (rs.w_lo <= 0 && rs.w_hi >= kBlockN);
            ok = __all_sync(0xffffffffu, whole) ? rs.template step<false, kMaskNone>(t, 0.f)
                                                : rs.template step<false, kMaskWindow>(t, 0.f);
        }
        float o[64];
#pragma unroll
        for (int c = 0; c < 64; ++c) o[c] = 0.f;
        if (ok && t1 > t0) {
            ok = warp_wait(rs.pv_done, rs.pv_parity, ctl, FDS_STATUS_TIMEOUT_SOFTMAX);
            if (ok) {
                tc_fence_after();
                uint32_t ou[64];
                tmem_ld64(rs.tO, ou);
                tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < 64; ++c) o[c] = __uint_as_float(ou[c]);
            }
        }
        T* out = static_cast<T*>(p.out) + b * p.out_stride[0] + row0 * p.out_stride[1] + h * p.out_stride[2];
        if (split == 1) {
            if (ok && row < rows) {
                const bool none = rs.l_run == 0.f;  // no key seen
                if (none) {
#pragma unroll
                    for (int c = 0; c < 64; ++c) o[c] = 0.f;
                }
                store_row<T>(out + row * p.out_stride[1], o, none ? 1.f : 1.f / rs.l_run);
            }
        } else {
            const uint32_t part = sbase + S::part + 4u * row;
#pragma unroll
            for (int c = 0; c < 64; ++c) st_shared_f32(part + 512u * c, rs.l_run == 0.f ? 0.f : o[c]);
            st_shared_f32(part + 512u * 64, rs.m_run);
            st_shared_f32(part + 512u * 65, rs.l_run);
        }
        __syncwarp();
        tc_fence_before();
        named_barrier_sync(1, kTileThreads);
        if (split > 1) {
            cluster_sync_all();
            merge_parts<T>(sbase + S::part, static_cast<int>(split), static_cast<int>(rank),
                           static_cast<int>(threadIdx.x) - 128, rows, out, p.out_stride[1]);
            __syncwarp();
            cluster_sync_all();  // no CTA leaves while its parts are read
        }
    } else {
        setmaxnreg_dec<kControlRegs>();
        if (warp == 0 && t1 > t0) {
            // ------------------------------------------------ MMA issuer
            constexpr int fmt = DTypeTraits<T>::kFormat;
            constexpr uint32_t idesc_qk = idesc_f16(kBlockM, kBlockN, fmt, 0, 0);
            constexpr uint32_t idesc_pv = idesc_f16(kBlockM, kHeadDim, fmt, 0, 1);
            constexpr int err = FDS_STATUS_TIMEOUT_MMA;
            const auto issue_s = [&](int j) {
                if (elect_one()) {
                    const uint64_t dq = sw128_desc(sbase + S::q), dk = sw128_desc(sbase + S::k + (j % kKStages) * kTileBytes);
#pragma unroll
                    for (int k = 0; k < kHeadDim / 16; ++k) mma_ss(tmem, dq + 2 * k, dk + 2 * k, idesc_qk, k > 0);
                    mma_commit(bar(S::kSFull));
                    mma_commit(bar(S::kKEmpty + j % kKStages));
                }
                __syncwarp();
            };
            const auto issue_pv = [&](int j, int half) {
                if (elect_one()) {
                    const uint64_t dv = sw128_desc(sbase + S::v + (j % kVStages) * kTileBytes);
#pragma unroll
                    for (int k = 0; k < kBlockN / 32; ++k) {
                        const int kk = half * (kBlockN / 32) + k;
                        mma_ts(tmem + kTO, tmem + kTP + 8 * kk, dv + 128 * kk, idesc_pv, (j > 0 || kk > 0) ? 1u : 0u);
                    }
                    if (half == 1) {
                        mma_commit(bar(S::kPvDone));
                        mma_commit(bar(S::kVEmpty + j % kVStages));
                    }
                }
                __syncwarp();
            };
            const int n = t1 - t0;
            bool issued = false;
            bool ok = warp_wait(bar(S::kQ), 0, ctl, err) && warp_wait(bar(S::kKFull), 0, ctl, err);
            if (ok) {
                tc_fence_after();
                issue_s(0);
                issued = true;
            }
            for (int j = 0; ok && j < n; ++j) {
                if (j + 1 < n) {
                    ok = warp_wait(bar(S::kSFree), j & 1, ctl, err) &&
                         warp_wait(bar(S::kKFull + (j + 1) % kKStages), ((j + 1) / kKStages) & 1, ctl, err);
                    if (!ok) break;
                    tc_fence_after();
                    issue_s(j + 1);
                }
                ok = warp_wait(bar(S::kVFull + j % kVStages), (j / kVStages) & 1, ctl, err);
                if (!ok) break;
                // value rows of columns that no row sees: the sinks' padding and past the end
                const int x0 = (t0 + j) * kBlockN;
                const int z0 = max(cols.n_sink - x0, 0), z1 = min(cols.s8 - x0, kBlockN), z2 = max(cols.total() - x0, 0);
                if (z0 < z1 || z2 < kBlockN) {
                    const uint32_t vs = sbase + S::v + (j % kVStages) * kTileBytes;
                    for (int i = lane; i < kBlockN * 8; i += 32) {
                        const int r = i >> 3;
                        if ((r >= z0 && r < z1) || r >= z2) st_shared_v4(vs + 16u * i, make_int4(0, 0, 0, 0));
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                }
                ok = warp_wait(bar(S::kPHalf), j & 1, ctl, err);
                if (!ok) break;
                tc_fence_after();
                issue_pv(j, 0);
                ok = warp_wait(bar(S::kPFull), j & 1, ctl, err);
                if (!ok) break;
                tc_fence_after();
                issue_pv(j, 1);
            }
            if (issued) {  // every MMA issued completes before TMEM is released
                if (elect_one()) mma_commit(bar(S::kDrain));
                __syncwarp();
                wait_bounded(bar(S::kDrain), 0, ctl, FDS_STATUS_TIMEOUT_DRAIN, false);
                __syncwarp();
            }
        } else if (warp == 1 && t1 > t0) {
            // ------------------------------------------------ TMA producer
            constexpr int err = FDS_STATUS_TIMEOUT_LOAD;
            if (elect_one()) {
                mbar_arrive_expect_tx(bar(S::kQ), kTileBytes);
                tma_load_4d(sbase + S::q, &maps.q, bar(S::kQ), 0, h, row0, b);
            }
            __syncwarp();
            const int n = t1 - t0;
            int nk = 0, nv = 0;  // tiles issued
            bool ok = true;
            for (int j = 0; j < n; ++j) {
                const int sk = j % kKStages, sv = j % kVStages;
                if (j >= kKStages) ok = warp_wait(bar(S::kKEmpty + sk), (j / kKStages - 1) & 1, ctl, err);
                if (!ok) break;
                if (elect_one())
                    load_columns(sbase + S::k + sk * kTileBytes, &maps.k, &maps.k8, bar(S::kKFull + sk), cols,
                                 (t0 + j) * kBlockN, hk, b);
                __syncwarp();
                ++nk;
                if (j >= kVStages) ok = warp_wait(bar(S::kVEmpty + sv), (j / kVStages - 1) & 1, ctl, err);
                if (!ok) break;
                if (elect_one())
                    load_columns(sbase + S::v + sv * kTileBytes, &maps.v, &maps.v8, bar(S::kVFull + sv), cols,
                                 (t0 + j) * kBlockN, hk, b);
                __syncwarp();
                ++nv;
            }
            if (!ok) {
                // aborted: the copies already issued land before the CTA exits
                wait_bounded(bar(S::kQ), 0, ctl, FDS_STATUS_TIMEOUT_DRAIN, false);
                for (int s = 0; s < kKStages; ++s)
                    if (nk > s)
                        wait_bounded(bar(S::kKFull + s), ((nk - 1 - s) / kKStages) & 1, ctl, FDS_STATUS_TIMEOUT_DRAIN, false);
                for (int s = 0; s < kVStages; ++s)
                    if (nv > s)
                        wait_bounded(bar(S::kVFull + s), ((nv - 1 - s) / kVStages) & 1, ctl, FDS_STATUS_TIMEOUT_DRAIN, false);
                __syncwarp();
            }
        }
        __syncwarp();
        tc_fence_before();
        named_barrier_sync(1, kTileThreads);
        if (warp == 2) {
            tc_fence_after();
            tmem_dealloc(tmem, kTmemColsTile);
        }
        if (split > 1) {
            cluster_sync_all();
            cluster_sync_all();
        }
    }
}

// ---------------------------------------------------------------- step kernel

constexpr int kStepThreads = 128;
constexpr int kStepRows = 8;     // query rows per key head at most
constexpr int kStepUnroll = 4;   // keys per 8-lane group in flight

// R query rows (row r: query r / group, head hk * group + r % group), R a power
// of two >= the rows there are. kMulti: several queries, whose windows differ.
template <typename T, int R, bool kMulti>
__global__ void __launch_bounds__(kStepThreads) window_step_kernel(const Params p) {
    __shared__ float part[4][R][66];  // per warp: 64 of O, max, sum
    grid_launch_dependents();
    grid_dependency_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int sub = lane & 7;                                    // dims [8 sub, 8 sub + 8)
    const int grp = static_cast<int>(threadIdx.x >> 3);          // 16 groups
    const int split = static_cast<int>(gridDim.x), rank = static_cast<int>(blockIdx.x);
    const int hk = blockIdx.y, b = blockIdx.z;
    const int group = p.heads / p.kv_heads;
    const int n_rows = p.q_len * group;
    const Columns cols(p, b, 0, p.q_len);
    const int total = cols.n_sink + cols.n_win;  // no padding here
    const int per = (total + split - 1) / split;
    const int x_begin = min(total, rank * per), x_end = min(total, x_begin + per);

    float q[R][8];
    int lo[R], hi[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int rr = min(r, n_rows - 1), i = rr / group;
        const T* src = static_cast<const T*>(p.q) + b * p.q_stride[0] + i * p.q_stride[1] +
                       (hk * group + rr % group) * p.q_stride[2] + 8 * sub;
        norm::unpack8<T>(*reinterpret_cast<const uint4*>(src), q[r]);
#pragma unroll
        for (int e = 0; e < 8; ++e) q[r][e] *= p.scale_log2;
        lo[r] = cols.p0 + i - p.left;
        hi[r] = cols.p0 + i + p.right;
    }
    float m[R], l[R], acc[R][8];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[r][e] = 0.f;
    }
    const T* kb = static_cast<const T*>(p.k) + b * p.k_stride[0] + hk * p.k_stride[2] + 8 * sub;
    const T* vb = static_cast<const T*>(p.v) + b * p.v_stride[0] + hk * p.v_stride[2] + 8 * sub;
    for (int x0 = x_begin; x0 < x_end; x0 += 16 * kStepUnroll) {
        uint4 kr[kStepUnroll], vr[kStepUnroll];
        int key[kStepUnroll];
#pragma unroll
        for (int u = 0; u < kStepUnroll; ++u) {
            const int x = x0 + grp + 16 * u;
            key[u] = x < x_end ? (x < cols.n_sink ? x : cols.begin + x - cols.n_sink) : -1;
            kr[u] = vr[u] = make_uint4(0, 0, 0, 0);
            if (key[u] >= 0) {
                kr[u] = __ldg(reinterpret_cast<const uint4*>(kb + key[u] * p.k_stride[1]));
                vr[u] = __ldg(reinterpret_cast<const uint4*>(vb + key[u] * p.v_stride[1]));
            }
        }
        float s[R][kStepUnroll];
#pragma unroll
        for (int u = 0; u < kStepUnroll; ++u) {
            float kf[8];
            norm::unpack8<T>(kr[u], kf);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float d = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) d = fmaf(q[r][e], kf[e], d);
#pragma unroll
                for (int w = 4; w > 0; w >>= 1) d += __shfl_xor_sync(0xffffffffu, d, w);
                const bool seen = key[u] >= 0 &&
                                  (!kMulti || (key[u] <= hi[r] && (key[u] >= lo[r] || key[u] < p.sinks)));
                s[r][u] = seen ? d : -INFINITY;
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float mt = m[r];
#pragma unroll
            for (int u = 0; u < kStepUnroll; ++u) mt = fmaxf(mt, s[r][u]);
            const float base = mt == -INFINITY ? 0.f : mt;
            const float alpha = ex2_approx(m[r] - base);
            m[r] = mt;
            l[r] *= alpha;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[r][e] *= alpha;
#pragma unroll
            for (int u = 0; u < kStepUnroll; ++u) {
                s[r][u] = ex2_approx(s[r][u] - base);
                l[r] += s[r][u];
            }
        }
#pragma unroll
        for (int u = 0; u < kStepUnroll; ++u) {
            float vf[8];
            norm::unpack8<T>(vr[u], vf);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (kMulti && !(key[u] <= hi[r] && (key[u] >= lo[r] || key[u] < p.sinks))) continue;
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[r][e] = fmaf(s[r][u], vf[e], acc[r][e]);
            }
        }
    }
    // the four groups of a warp, then the warps, then the CTAs of the unit
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int w = 8; w < 32; w <<= 1) {
            const float mo = __shfl_xor_sync(0xffffffffu, m[r], w), lo_ = __shfl_xor_sync(0xffffffffu, l[r], w);
            const float mm = fmaxf(m[r], mo), base = mm == -INFINITY ? 0.f : mm;
            const float fa = ex2_approx(m[r] - base), fb = ex2_approx(mo - base);
            m[r] = mm;
            l[r] = l[r] * fa + lo_ * fb;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                acc[r][e] = acc[r][e] * fa + __shfl_xor_sync(0xffffffffu, acc[r][e], w) * fb;
        }
        if (lane < 8) {
#pragma unroll
            for (int e = 0; e < 8; ++e) part[warp][r][8 * lane + e] = acc[r][e];
            if (lane == 0) part[warp][r][64] = m[r], part[warp][r][65] = l[r];
        }
    }
    __syncthreads();
    // fold the warps into part[0] (each thread its own columns; max and sum last)
    for (int i = threadIdx.x; i < R * 64; i += kStepThreads) {
        const int r = i >> 6, c = i & 63;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) mm = fmaxf(mm, part[w][r][64]);
        const float base = mm == -INFINITY ? 0.f : mm;
        float o = 0.f, ll = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = ex2_approx(part[w][r][64] - base);
            o = fmaf(part[w][r][c], f, o);
            ll = fmaf(part[w][r][65], f, ll);
        }
        part[0][r][c] = o;
        if (split == 1) {
            if (r < n_rows) {
                T* out = static_cast<T*>(p.out) + b * p.out_stride[0] + (r / group) * p.out_stride[1] +
                         (hk * group + r % group) * p.out_stride[2];
                out[c] = static_cast<T>(ll == 0.f ? 0.f : o / ll);
            }
        }
    }
    if (split == 1) return;
    __syncthreads();
    if (threadIdx.x < R) {
        const int r = threadIdx.x;
        float mm = -INFINITY;
        for (int w = 0; w < 4; ++w) mm = fmaxf(mm, part[w][r][64]);
        const float base = mm == -INFINITY ? 0.f : mm;
        float ll = 0.f;
        for (int w = 0; w < 4; ++w) ll = fmaf(part[w][r][65], ex2_approx(part[w][r][64] - base), ll);
        part[0][r][64] = mm;
        part[0][r][65] = ll;
    }
    __syncthreads();
    cluster_sync_all();
    // merge in rank order; the CTAs of the cluster share the rows' columns
    for (int i = rank * kStepThreads + static_cast<int>(threadIdx.x); i < R * 64; i += split * kStepThreads) {
        const int r = i >> 6, c = i & 63;
        const uint32_t at = smem_u32(&part[0][r][0]);
        float mm = -INFINITY;
        for (int k = 0; k < split; ++k) mm = fmaxf(mm, ld_cluster_f32(map_to_rank(at + 4u * 64, k)));
        const float base = mm == -INFINITY ? 0.f : mm;
        float o = 0.f, ll = 0.f;
        for (int k = 0; k < split; ++k) {
            const uint32_t a = map_to_rank(at, k);
            const float f = ex2_approx(ld_cluster_f32(a + 4u * 64) - base);
            o = fmaf(ld_cluster_f32(a + 4u * c), f, o);
            ll = fmaf(ld_cluster_f32(a + 4u * 65), f, ll);
        }
        if (r < n_rows) {
            T* out = static_cast<T*>(p.out) + b * p.out_stride[0] + (r / group) * p.out_stride[1] +
                     (hk * group + r % group) * p.out_stride[2];
            out[c] = static_cast<T>(ll == 0.f ? 0.f : o / ll);
        }
    }
    __syncwarp();
    cluster_sync_all();
}

}  // namespace window
}  // namespace fds
