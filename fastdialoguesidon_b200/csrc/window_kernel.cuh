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
// * window_tile_kernel: tensor cores, a unit of 128 query rows of a (window,
//   head) at a time, walking 128-column tiles over the union of the keys its rows
//   see. The columns are the union's window part, from the first key its first
//   row sees on (TMA rows start anywhere), rounded up to 8 (one swizzle atom),
//   then the sinks before it, packed: a tile may hold both, so the sinks cost
//   their own columns and not a tile of their own, and at most one tile at the
//   left edge and two at the right are seen in part. The step is the
//   bidirectional attention's (attn_kernel.cuh RowSoftmax). A CTA has one query
//   tile and half an SM (128 + 128 threads, 256 TMEM columns, 98 KB): a window is
//   a handful of tiles, and a 128-row tile overlaps fewer keys that its rows do
//   not see than a 256-row unit. With few query tiles and many key tiles the
//   column tiles of a unit are dealt to a cluster of up to 8 CTAs, whose partial
//   (O, max, sum) are merged through distributed shared memory in rank order.
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
    int32_t units;       // batch * heads * row_blocks
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

// The columns of a unit of `rows` query rows: keys [begin, begin + n_win), padded
// to s0 columns (a multiple of 8, where sinks follow), then keys [0, n_sink).
struct Columns {
    int p0, kv_end, begin, n_win, s0, n_sink;
    Columns() = default;
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
        n_win = max(0, end - begin);
        s0 = n_sink > 0 ? (n_win + 7) & ~7 : n_win;
    }
    __device__ __forceinline__ int total() const { return s0 + n_sink; }
};

// ---------------------------------------------------------------- tile kernel

constexpr int kTileThreads = 256;
constexpr int kTileRegs = 128;  // per thread at launch: 65536 / (2 CTAs x 256)
constexpr int kSoftmaxRegs = 200, kControlRegs = 56;
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
    static constexpr int kQEmpty = kPvDone + 1;
    static constexpr int kDrain = kQEmpty + 1;
    static constexpr int kRecFull = kDrain + 1;     // [record] laid out
    static constexpr int kRecEmpty = kRecFull + 2;  // [record] read by every role
    static constexpr int kNext = kRecEmpty + 2;     // the next unit's launch-control answer landed
    static constexpr int kNumBars = kNext + 1;
    static constexpr int misc = bars + kNumBars * 8;  // the bounded waits' block (attn_kernel.cuh Smem::misc)
    static constexpr int records = (misc + 48 + 15) / 16 * 16;
    static constexpr int answer = records + 2 * 64;
    static constexpr int total = answer + 16;
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

// A unit (row block fastest, then head, then window) and this CTA's share of
// its tiles, [t0, t1).
struct Unit {
    int b, h, row0, rows, t0, t1;
    Columns c;
};

__device__ __forceinline__ Unit make_unit(const Params& p, int unit, int split, int rank) {
    const int bh = unit / p.row_blocks;
    Unit u;
    u.b = bh / p.heads;
    u.h = bh - u.b * p.heads;
    u.row0 = (unit - bh * p.row_blocks) * kBlockM;
    u.rows = min(kBlockM, p.q_len - u.row0);
    u.c = Columns(p, u.b, u.row0, u.rows);
    const int tiles = (u.c.total() + kBlockN - 1) / kBlockN;
    const int per = (tiles + split - 1) / split;
    u.t0 = min(tiles, rank * per);
    u.t1 = min(tiles, u.t0 + per);
    return u;
}

// The units of a CTA are laid out by warp 3 ahead of the roles that use them
// (divisions and the loads of q_start and kv_len stay off their paths), as 64-byte
// records in a ring: {b, h, row0, rows}, {t0, t1, p0, kv_end}, {begin, n_win, s0,
// n_sink}, {key head, tile with padding columns, tile with columns past the end,
// more} (tiles counted from t0, -1: none; more = 0 ends the list).
constexpr int kRecords = 2;
constexpr int kRecordReaders = 6;  // MMA, TMA, four softmax warps

__device__ __forceinline__ void store_record(uint32_t at, const Unit& u, int hk) {
    st_shared_v4(at, make_int4(u.b, u.h, u.row0, u.rows));
    st_shared_v4(at + 16, make_int4(u.t0, u.t1, u.c.p0, u.c.kv_end));
    st_shared_v4(at + 32, make_int4(u.c.begin, u.c.n_win, u.c.s0, u.c.n_sink));
    const int pad = u.c.s0 > u.c.n_win ? u.c.n_win / kBlockN - u.t0 : -1;
    const int end = u.c.total() % kBlockN != 0 ? u.c.total() / kBlockN - u.t0 : -1;
    st_shared_v4(at + 48, make_int4(hk, pad, end, 1));
}

// Columns [x0, x0 + 128), some of them sinks, of the keys or values of a unit
// (128 rows of 128 bytes, 16384 bytes in all; rows past the tensor read as zero).
inline __device__ __noinline__ void load_sink_columns(uint32_t dst, const CUtensorMap* map, const CUtensorMap* map8,
                                                      uint32_t bar, uint32_t rec, int x0) {
    const int4 c = ld_shared_v4(rec + 32);  // begin, n_win, s0, n_sink
    const int b = ld_shared_v4(rec).x, head = ld_shared_v4(rec + 48).x;
    if (x0 >= c.z) {
        tma_load_4d(dst, map, bar, 0, head, x0 - c.z, b);
        return;
    }
#pragma unroll 1
    for (int r = 0; r < kBlockN; r += 8) {
        const int x = x0 + r;
        tma_load_4d(dst + r * 128, map8, bar, 0, head, x < c.z ? c.x + x : x - c.z, b);
    }
}

// Zeroes the value rows of columns that no row of the unit sees -- the window
// part's padding and past the end -- before a product reads them (a whole warp).
inline __device__ __noinline__ void zero_unseen(uint32_t rec, int x0, uint32_t tile, int lane) {
    const int4 c = ld_shared_v4(rec + 32);
    const int z0 = c.y - x0, z1 = c.z - x0, z2 = c.z + c.w - x0;
#pragma unroll 1
    for (int i = lane; i < kBlockN * 8; i += 32) {
        const int r = i >> 3;
        if ((r >= z0 && r < z1) || r >= z2) st_shared_v4(tile + 16u * i, make_int4(0, 0, 0, 0));
    }
    fence_proxy_async_smem();
    __syncwarp();
}

// The grid has a CTA (or cluster) per unit; a CTA that finishes early takes over
// the units of CTAs that have not started, so that the next unit's copies and
// first scores run under the present one's last tiles and epilogue.
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
    const int split = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
    grid_launch_dependents();

    if (threadIdx.x == 0) {
        mbar_init(&bars[S::kQ], 1);
        mbar_init(&bars[S::kQEmpty], 1);
        for (int s = 0; s < kKStages; ++s) mbar_init(&bars[S::kKFull + s], 1), mbar_init(&bars[S::kKEmpty + s], 1);
        for (int s = 0; s < kVStages; ++s) mbar_init(&bars[S::kVFull + s], 1), mbar_init(&bars[S::kVEmpty + s], 1);
        mbar_init(&bars[S::kSFull], 1);
        mbar_init(&bars[S::kSFree], 4);  // one arrival per softmax warp
        mbar_init(&bars[S::kPHalf], 4);
        mbar_init(&bars[S::kPFull], 4);
        mbar_init(&bars[S::kPvDone], 1);
        mbar_init(&bars[S::kDrain], 1);
        for (int r = 0; r < kRecords; ++r) {
            mbar_init(&bars[S::kRecFull + r], 1);
            mbar_init(&bars[S::kRecEmpty + r], kRecordReaders);
        }
        mbar_init(&bars[S::kNext], 1);
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

    // record of this CTA's i-th unit; record_wait: it is laid out (0 on a timeout,
    // and at the end of the list); `release` hands its slot back
    const auto record = [&](int i) { return sbase + S::records + 64u * (i % kRecords); };
    const auto record_wait = [&](int i, int err) {
        return warp_wait(bar(S::kRecFull + i % kRecords), (i / kRecords) & 1, ctl, err) &&
               ld_shared_volatile_u32(record(i) + 60) != 0;
    };
    const auto record_release = [&](int i) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(S::kRecEmpty + i % kRecords));
    };

    // The two register classes never share code again (attn_kernel.cuh).
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
        rs.s_parity = 0;
        rs.pv_parity = 0;
        bool ok = true;
        for (int i = 0; ok && record_wait(i, FDS_STATUS_TIMEOUT_SOFTMAX); ++i) {
            const int4 un = ld_shared_v4(record(i) + 16);  // t0, t1, p0, kv_end
            const int t1 = un.y;
            rs.t_begin = un.x;
            rs.m_run = -INFINITY;
            rs.l_run = 0.f;
            // this row's columns: [lo, hi) of the window part and the sinks, [a, z) (where
            // they lie in the window part: those of them up to p + right)
            const int4 c = ld_shared_v4(record(i) + 32);  // begin, n_win, s0, n_sink
            const int pos = un.z + row;
            const int hi = min(pos + p.right + 1, un.w) - c.x;
            const int lo = max(pos - p.left - c.x, 0);
            const int a = c.w > 0 ? c.z : 0, z = c.w > 0 ? c.z + c.w : min(p.sinks, hi);
            for (int t = rs.t_begin; ok && t < t1; ++t) {
                const int n0 = t * kBlockN;
                rs.w_a = a - n0;
                rs.w_z = z - n0;
                rs.w_lo = lo - n0;
                rs.w_hi = hi - n0;
                rs.w_whole = __all_sync(0xffffffffu, (rs.w_lo <= 0 && rs.w_hi >= kBlockN) || (rs.w_a <= 0 && rs.w_z >= kBlockN));
                ok = rs.template step<false, kMaskWindow>(t, 0.f);
            }
            const bool none = rs.m_run == -INFINITY;  // no key seen
            float o[64];
            if (ok && t1 > rs.t_begin) {
                // (the next unit's first P V overwrites O only after this warpgroup's
                // next P store, which follows this read in program order)
                ok = warp_wait(rs.pv_done, rs.pv_parity, ctl, FDS_STATUS_TIMEOUT_SOFTMAX);
                rs.pv_parity ^= 1;
                tc_fence_after();
                uint32_t ou[64];
                tmem_ld64(rs.tO, ou);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 64; ++e) o[e] = none ? 0.f : __uint_as_float(ou[e]);
            } else {
#pragma unroll
                for (int e = 0; e < 64; ++e) o[e] = 0.f;
            }
            if (split == 1) {
                const int4 at = ld_shared_v4(record(i));  // b, h, row0, rows: not held in registers over the tiles
                if (ok && row < at.w)
                    store_row<T>(static_cast<T*>(p.out) + at.x * p.out_stride[0] + (at.z + row) * p.out_stride[1] +
                                     at.y * p.out_stride[2],
                                 o, none ? 1.f : 1.f / rs.l_run);
            } else {
                const uint32_t part = sbase + S::part + 4u * row;
#pragma unroll
                for (int e = 0; e < 64; ++e) st_shared_f32(part + 512u * e, o[e]);
                st_shared_f32(part + 512u * 64, rs.m_run);
                st_shared_f32(part + 512u * 65, none ? 0.f : rs.l_run);
            }
            if (split == 1) record_release(i);
        }
        __syncwarp();
        tc_fence_before();
        named_barrier_sync(1, kTileThreads);
        if (split > 1) {
            cluster_sync_all();
            const int4 at = ld_shared_v4(record(0));  // (the end of the list is in the other slot)
            merge_parts<T>(sbase + S::part, split, rank, static_cast<int>(threadIdx.x) - 128, at.w,
                           static_cast<T*>(p.out) + at.x * p.out_stride[0] + at.z * p.out_stride[1] + at.y * p.out_stride[2],
                           p.out_stride[1]);
            __syncwarp();
            cluster_sync_all();  // no CTA leaves while its parts are read
        }
    } else {
        setmaxnreg_dec<kControlRegs>();
        if (warp == 0) {
            // ------------------------------------------------ MMA issuer
            constexpr int fmt = DTypeTraits<T>::kFormat;
            constexpr uint32_t idesc_qk = idesc_f16(kBlockM, kBlockN, fmt, 0, 0);
            constexpr uint32_t idesc_pv = idesc_f16(kBlockM, kHeadDim, fmt, 0, 1);
            constexpr int err = FDS_STATUS_TIMEOUT_MMA;
            int g = 0, q = 0;  // tiles and units so far (ring stages and barrier phases run on)
            bool ok = true;
            // S columns <- Q K(tile g)^T, once the previous scores are read out; the unit's last also frees Q
            const auto scores = [&](int gt, bool last) {
                if (gt > 0) ok = warp_wait(bar(S::kSFree), (gt - 1) & 1, ctl, err);
                if (ok) ok = warp_wait(bar(S::kKFull + gt % kKStages), (gt / kKStages) & 1, ctl, err);
                if (!ok) return;
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t dq = sw128_desc(sbase + S::q), dk = sw128_desc(sbase + S::k + (gt % kKStages) * kTileBytes);
#pragma unroll
                    for (int k = 0; k < kHeadDim / 16; ++k) mma_ss(tmem, dq + 2 * k, dk + 2 * k, idesc_qk, k > 0);
                    mma_commit(bar(S::kSFull));
                    mma_commit(bar(S::kKEmpty + gt % kKStages));
                    if (last) mma_commit(bar(S::kQEmpty));
                }
                __syncwarp();
            };
            // O (+)= P V(tile g) over half of the tile's keys
            const auto values = [&](int gt, int half, bool accumulate) {
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t dv = sw128_desc(sbase + S::v + (gt % kVStages) * kTileBytes);
#pragma unroll
                    for (int k = 0; k < kBlockN / 32; ++k) {
                        const int kk = half * (kBlockN / 32) + k;
                        mma_ts(tmem + kTO, tmem + kTP + 8 * kk, dv + 128 * kk, idesc_pv, (accumulate || kk > 0) ? 1u : 0u);
                    }
                    if (half == 1) {
                        mma_commit(bar(S::kPvDone));
                        mma_commit(bar(S::kVEmpty + gt % kVStages));
                    }
                }
                __syncwarp();
            };
            for (int i = 0; ok && record_wait(i, err); ++i) {
                const uint32_t rec = record(i);
                const int4 tiles = ld_shared_v4(rec + 16), zero = ld_shared_v4(rec + 48);
                const int n = tiles.y - tiles.x;
                if (n <= 0) {
                    record_release(i);
                    continue;
                }
                ok = warp_wait(bar(S::kQ), q & 1, ctl, err);
                ++q;
                if (ok) scores(g, n == 1);
                for (int j = 0; ok && j < n; ++j, ++g) {
                    if (j + 1 < n) scores(g + 1, j + 2 == n);
                    if (ok) ok = warp_wait(bar(S::kVFull + g % kVStages), (g / kVStages) & 1, ctl, err);
                    if (!ok) break;
                    if (j == zero.y || j == zero.z)
                        zero_unseen(rec, (tiles.x + j) * kBlockN, sbase + S::v + (g % kVStages) * kTileBytes, lane);
                    ok = warp_wait(bar(S::kPHalf), g & 1, ctl, err);
                    if (!ok) break;
                    values(g, 0, j > 0);
                    ok = warp_wait(bar(S::kPFull), g & 1, ctl, err);
                    if (!ok) break;
                    values(g, 1, true);
                }
                record_release(i);
            }
            if (q > 0) {  // every MMA issued completes before TMEM is released
                if (elect_one()) mma_commit(bar(S::kDrain));
                __syncwarp();
                wait_bounded(bar(S::kDrain), 0, ctl, FDS_STATUS_TIMEOUT_DRAIN, false);
                __syncwarp();
            }
        } else if (warp == 1) {
            // ------------------------------------------------ TMA producer
            constexpr int err = FDS_STATUS_TIMEOUT_LOAD;
            int nk = 0, nv = 0, nq = 0;  // copies issued
            bool ok = true;
            for (int i = 0; ok && record_wait(i, err); ++i) {
                const uint32_t rec = record(i);
                const int4 at = ld_shared_v4(rec), tiles = ld_shared_v4(rec + 16), c = ld_shared_v4(rec + 32);  // begin, n_win, s0, n_sink
                const int hk = ld_shared_v4(rec + 48).x;
                if (tiles.y > tiles.x) {
                    if (nq > 0) ok = warp_wait(bar(S::kQEmpty), (nq - 1) & 1, ctl, err);
                    if (!ok) break;
                    if (elect_one()) {
                        mbar_arrive_expect_tx(bar(S::kQ), kTileBytes);
                        tma_load_4d(sbase + S::q, &maps.q, bar(S::kQ), 0, at.y, at.z, at.x);
                    }
                    __syncwarp();
                    ++nq;
                }
                for (int t = tiles.x; t < tiles.y; ++t) {
                    const int x0 = t * kBlockN, key = c.x + x0;
                    const bool plain = c.w == 0 || x0 + kBlockN <= c.z;  // no sinks in the tile: keys from `key` on
                    const int sk = nk % kKStages, sv = nv % kVStages;
                    if (nk >= kKStages) ok = warp_wait(bar(S::kKEmpty + sk), (nk / kKStages - 1) & 1, ctl, err);
                    if (!ok) break;
                    if (elect_one()) {
                        mbar_arrive_expect_tx(bar(S::kKFull + sk), kTileBytes);
                        if (plain)
                            tma_load_4d(sbase + S::k + sk * kTileBytes, &maps.k, bar(S::kKFull + sk), 0, hk, key, at.x);
                        else
                            load_sink_columns(sbase + S::k + sk * kTileBytes, &maps.k, &maps.k8, bar(S::kKFull + sk), rec, x0);
                    }
                    __syncwarp();
                    ++nk;
                    if (nv >= kVStages) ok = warp_wait(bar(S::kVEmpty + sv), (nv / kVStages - 1) & 1, ctl, err);
                    if (!ok) break;
                    if (elect_one()) {
                        mbar_arrive_expect_tx(bar(S::kVFull + sv), kTileBytes);
                        if (plain)
                            tma_load_4d(sbase + S::v + sv * kTileBytes, &maps.v, bar(S::kVFull + sv), 0, hk, key, at.x);
                        else
                            load_sink_columns(sbase + S::v + sv * kTileBytes, &maps.v, &maps.v8, bar(S::kVFull + sv), rec, x0);
                    }
                    __syncwarp();
                    ++nv;
                }
                record_release(i);
            }
            if (!ok) {
                // aborted: the copies already issued land before the CTA exits
                if (nq > 0) wait_bounded(bar(S::kQ), (nq - 1) & 1, ctl, FDS_STATUS_TIMEOUT_DRAIN, false);
                for (int s = 0; s < kKStages; ++s)
                    if (nk > s)
                        wait_bounded(bar(S::kKFull + s), ((nk - 1 - s) / kKStages) & 1, ctl, FDS_STATUS_TIMEOUT_DRAIN, false);
                for (int s = 0; s < kVStages; ++s)
                    if (nv > s)
                        wait_bounded(bar(S::kVFull + s), ((nv - 1 - s) / kVStages) & 1, ctl, FDS_STATUS_TIMEOUT_DRAIN, false);
                __syncwarp();
            }
        } else if (warp == 3) {
            // ------------------------------------------------ unit records
            // This CTA's own unit, then the units of CTAs that have not started:
            // launch control hands them out as they are asked for, so SMs of
            // different speeds share the units as if each had its own CTA.
            constexpr int err = FDS_STATUS_TIMEOUT_LOAD;
            int unit = static_cast<int>(blockIdx.x) / split;
            bool ok = true, more = true;
            for (int i = 0; ok; ++i) {
                if (i >= kRecords) ok = warp_wait(bar(S::kRecEmpty + i % kRecords), (i / kRecords - 1) & 1, ctl, err);
                if (!ok) break;
                if (more) {
                    const Unit un = make_unit(p, unit, split, rank);
                    if (lane == 0) store_record(record(i), un, un.h / (p.heads / p.kv_heads));
                } else if (lane == 0) {
                    st_shared_volatile_u32(record(i) + 60, 0);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(S::kRecFull + i % kRecords));
                if (!more) break;
                if (split > 1) {  // a cluster holds one unit
                    more = false;
                    continue;
                }
                if (lane == 0) {
                    mbar_arrive_expect_tx(bar(S::kNext), 16);
                    launch_control_ask(sbase + S::answer, bar(S::kNext));
                }
                __syncwarp();
                ok = warp_wait(bar(S::kNext), i & 1, ctl, err);
                if (!ok) {  // (the answer still lands before the CTA exits)
                    wait_bounded(bar(S::kNext), i & 1, ctl, FDS_STATUS_TIMEOUT_DRAIN, false);
                    __syncwarp();
                    break;
                }
                more = launch_control_answer(sbase + S::answer, unit);
                fence_proxy_async_smem();  // the answer is read before the next one is written
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
