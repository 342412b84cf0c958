// window_kernel.cuh - attention over a sliding window of keys with a few first
// keys that stay visible (sinks), head width 64.
//
// Query i of window b sits at position p = q_start[b] + i of the key sequence
// and sees key j iff j < kv_len[b], j <= p + right and (j >= p - left or
// j < sinks); O_i = softmax_j(q_i . k_j * scale) V over the keys it sees, 0 if
// it sees none. Query head h reads key head h / (heads / kv_heads).
//
// Two kernels, chosen by the number of query rows that share a key head, 16 at most
// for steps (steps / tiles, us: 16 windows x 16 heads x 1000 keys, one row 13.4 / 19.7,
// 16 rows 17.2 / 19.8; one window x 12 heads x 500 keys 3.6 / 7.5 and 6.3 / 8.0):
//
// * window_tile_kernel: tensor cores, a unit of 128 query rows of a window at a
//   time -- the queries of one head, or 128 / group queries of all the heads that
//   share a key head, interleaved (20 queries x 16 windows, 4 heads a key head: 14.0
//   us against 20.4 with a unit per head; 6000 queries 52.9 and 53.6) -- walking 128-column tiles over the union of the keys
//   its rows see. The columns are the union's window part, from the first key its
//   first row sees on (TMA rows start anywhere), rounded up to 8 (one swizzle
//   atom), then the sinks before it, packed: a tile may hold both, so the sinks cost
//   their own columns and not a tile of their own, and at most one tile at the
//   left edge and two at the right are seen in part. The step is the
//   bidirectional attention's (attn_kernel.cuh RowSoftmax). A CTA has one query
//   tile and half an SM (128 + 128 threads, 256 TMEM columns, 112 KB): a window is
//   a handful of tiles, and a 128-row tile overlaps fewer keys that its rows do
//   not see than a 256-row unit. With few query tiles and many key tiles the
//   column tiles of a unit are dealt to a cluster of up to 8 CTAs: each owns some
//   of the rows, whose partial O and log-sums the others store into its shared
//   memory, and merges them in rank order.
//   Bound by the latency of a softmax warp's own instructions, two warps a
//   scheduler: 12 heads x 6000 queries x 1000 keys 39.5 us (issue slots 43 %,
//   exponential units 30 %, DRAM 8 %), 16 x 30000 x 1000 207 us, 597 TFLOP/s over
//   the pairs seen at full clock (228 us once the power cap holds the SMs at 1.78
//   GHz). A tile of a CTA takes 2250 to 2650 cycles, one with masks 3000;
//   from a unit's last tile to the next one's scores another 2200.
// * window_step_kernel: up to 16 query rows per key head (a decoding step):
//   bound by reading the keys and values once. Each warp streams its share of the
//   keys through a shared-memory ring of its own and multiplies them with the
//   rows as warp-level 16 x 8 x 16 products (a 128-row tcgen05 tile would be
//   seven-eighths empty, and the products are not what bounds it); the shares --
//   4 warps of up to 8 CTAs of a cluster -- are merged the same way. 16 windows x
//   4 key heads x 4112 keys: 14.6 us, 4.6 TB/s; one window, 12 heads x 1004 keys:
//   3.7, 1.9 of which an empty launch takes.
//
// Scores, maxima, sums, O and the parts' merge are fp32. The weights are rounded to
// the operand type for the P V product, in both kernels: the tensor cores take P in
// V's type (fp32 weights would need V as tf32, at half the rate and twice the
// shared memory), and a rounding of u relative per weight averages out over the
// keys, below the output's own rounding. Sums are of the unrounded weights. Tiles
// take 3 in 10 exponentials from a polynomial within 7.5e-5 (attn_kernel.cuh
// poly_pair), below u / 6 in fp16. In all the error against 64 bits is 1.2 to 1.4
// times the output's rounding alone (fp16 2.6e-4 to 2.9e-4 against 2.1e-4, bf16
// 2.1e-3 to 2.3e-3 against 1.7e-3, relative, in the 2-norm).
//
// Keys and values that no row of a unit sees may hold anything (a cache's
// unwritten rows): their scores are replaced, and their value rows are zeroed
// in shared memory before the P V product reads them (0 times an infinity
// would not be 0), or not read at all. A value row that one row of the unit sees
// is multiplied by the zero weights of the rows that do not.
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
    int32_t debug_flags;
    int32_t heads, kv_heads, q_len, k_len;
    int32_t left, right, sinks;
    // tile kernel: `pack` heads of a unit (the `group` of one key head, or 1) and
    // `queries` = 128 / pack of each; row r of a unit is query r / pack, head r % pack
    int32_t group, pack, queries;
    int32_t row_blocks;  // ceil(q_len / queries)
    int32_t out_boxes;   // whole units, pack divides 32: a warp's output rows are a box of heads x queries
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
constexpr int kVStages = 2;
constexpr int kMaxSplit = 8;

// kSplit: units dealt to clusters. Such a CTA needs no staged output rows, and gives
// a key stage too for the parts of the rows it owns.
template <bool kSplit>
struct TileSmem {
    static constexpr int kKStages = kSplit ? 2 : 3;
    static constexpr int q = 0;
    static constexpr int v = q + kTileBytes;
    static constexpr int k = v + kVStages * kTileBytes;
    static constexpr int stage = k + 3 * kTileBytes;  // 4 KB per softmax warp: its output rows
    // kSplit: O of the parts, [source CTA][row this CTA owns][64] floats (16-byte piece
    // c of a row at c ^ (row & 15)), each divided by its sum
    static constexpr int part = k + kKStages * kTileBytes;
    static_assert(!kSplit || part + kBlockM * 256 == stage + kTileBytes, "parts fill the space");
    static constexpr int bars = stage + kTileBytes;
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
    static constexpr int kNever = kNext + 1;
    static constexpr int kNumBars = kNever + 1;
    static constexpr int misc = bars + kNumBars * 8;  // the bounded waits' block (attn_kernel.cuh Smem::misc)
    static constexpr int records = (misc + 48 + 15) / 16 * 16;
    static constexpr int answer = records + 2 * 64;
    static constexpr int lse = answer + 16;  // kSplit: log2 of the parts' sums, [source CTA][row]
    static constexpr int alloc = lse + (kSplit ? kBlockM * 4 : 0);
    static_assert(2 * (alloc + 1024) <= 228 * 1024, "two CTAs per SM");
};
constexpr int kTmemColsTile = 256;  // S [0, 128), P [128, 192), O [192, 256)
constexpr int kTP = 128, kTO = 192;
constexpr int kTmemDone = 128 + 2 * 32;  // the softmax warps, the MMA warp and the one that releases TMEM

struct Maps {
    CUtensorMap q, k, v;    // boxes of 128 rows
    CUtensorMap k8, v8;     // boxes of 8 rows (tiles that hold sinks and window keys)
    CUtensorMap out;        // boxes of 32 rows (out_boxes)
};

// Row `row` of a split unit from its parts in this CTA's shared memory, columns
// [c0, c0 + 64 / split) of it into `out` if it is a real row: sum_r w_r O_r / sum_r w_r
// with w_r = 2^(lse_r - max lse), in rank order, so the result does not depend on the
// parts' timing. (The log's rounding is one more of the size of the scores' own. The
// loops are rolled: this runs once, and fetching its instructions is most of it.)
template <typename T>
__device__ __forceinline__ void merge_parts(uint32_t part, uint32_t lse, int split, int row, int c0, bool real, T* out) {
    const int rows = kBlockM / split;
    float m = -INFINITY;
#pragma unroll 2
    for (int r = 0; r < split; ++r) m = fmaxf(m, ld_shared_f32(lse + 4 * (r * rows + row)));
    if (m == -INFINITY) m = 0.f;
#pragma unroll 1
    for (int c = c0; c < c0 + kHeadDim / split; c += 8) {
        float acc[8], l = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = 0.f;
#pragma unroll 2
        for (int r = 0; r < split; ++r) {
            const int at = r * rows + row;
            const float f = ex2_approx(ld_shared_f32(lse + 4 * at) - m);
            const float4 a = ld_shared_v4f32(part + 256 * at + 16 * ((c >> 2) ^ (at & 15)));
            const float4 b = ld_shared_v4f32(part + 256 * at + 16 * (((c >> 2) + 1) ^ (at & 15)));
            l += f;
            acc[0] = fmaf(a.x, f, acc[0]), acc[1] = fmaf(a.y, f, acc[1]), acc[2] = fmaf(a.z, f, acc[2]);
            acc[3] = fmaf(a.w, f, acc[3]), acc[4] = fmaf(b.x, f, acc[4]), acc[5] = fmaf(b.y, f, acc[5]);
            acc[6] = fmaf(b.z, f, acc[6]), acc[7] = fmaf(b.w, f, acc[7]);
        }
        const float inv = l == 0.f ? 0.f : __fdividef(1.f, l);  // l: 1 to 8 and the smaller weights
        if (real)
            *reinterpret_cast<uint4*>(out + c) =
                make_uint4(norm::pack2<T>(acc[0] * inv, acc[1] * inv), norm::pack2<T>(acc[2] * inv, acc[3] * inv),
                           norm::pack2<T>(acc[4] * inv, acc[5] * inv), norm::pack2<T>(acc[6] * inv, acc[7] * inv));
    }
}

// A unit, by its place in the grid (row block, head group, window): queries [row0,
// row0 + n) of heads [h, h + pack) of window b, which read key head hk, and this CTA's
// share of its tiles, [t0, t1).
struct Unit {
    int b, h, hk, row0, n, t0, t1;
    Columns c;
};

__device__ __forceinline__ Unit make_unit(const Params& p, int block, int group, int b, int split_log2, int rank) {
    Unit u;
    u.b = b;
    u.h = group * p.pack;
    u.hk = p.pack == p.group ? group : group / p.group;
    u.row0 = block * p.queries;
    u.n = min(p.queries, p.q_len - u.row0);
    u.c = Columns(p, u.b, u.row0, u.n);
    const int tiles = (u.c.total() + kBlockN - 1) / kBlockN;
    const int per = (tiles + (1 << split_log2) - 1) >> split_log2;
    u.t0 = min(tiles, rank * per);
    u.t1 = min(tiles, u.t0 + per);
    return u;
}

// The units of a CTA are laid out by warp 3 ahead of the roles that use them
// (divisions and the loads of q_start and kv_len stay off their paths), as 64-byte
// records in a ring: {b, h, row0, n}, {t0, t1, p0, kv_end}, {begin, n_win, s0,
// n_sink}, {key head, tile with padding columns, tile with columns past the end,
// more} (tiles counted from t0, -1: none; more = 0 ends the list).
constexpr int kRecords = 2;
constexpr int kRecordReaders = 6;  // MMA, TMA, four softmax warps

__device__ __forceinline__ void store_record(uint32_t at, const Unit& u) {
    st_shared_v4(at, make_int4(u.b, u.h, u.row0, u.n));
    st_shared_v4(at + 16, make_int4(u.t0, u.t1, u.c.p0, u.c.kv_end));
    st_shared_v4(at + 32, make_int4(u.c.begin, u.c.n_win, u.c.s0, u.c.n_sink));
    const int pad = u.c.s0 > u.c.n_win ? u.c.n_win / kBlockN - u.t0 : -1;
    const int end = u.c.total() % kBlockN != 0 ? u.c.total() / kBlockN - u.t0 : -1;
    st_shared_v4(at + 48, make_int4(u.hk, pad, end, 1));
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

// Thread `lane` of a warp has row `lane` of 32 output rows, 64 values in w. Rows
// [query0 ..] x [head .. head + pack) of window b as one box, through the warp's
// 4 KB of shared memory (16-byte piece c of a row at c ^ (row & 7)). An epilogue is
// one warp's dependent instructions, and takes 1000 cycles this way; 2250 with the
// addresses of 64-byte pieces worked out per lane (600 s of audio in 16 heads: 221
// us against 214), and rows written by their own threads in 32-byte stores, as few
// instructions, cost the steps beside them more (226 us).
__device__ __forceinline__ void store_box(uint32_t stage, const CUtensorMap* map, int lane, const uint32_t (&w)[32], int head,
                                          int query0, int b, bool any) {
    if (lane == 0) bulk_wait_read_all();  // the previous unit's rows are read out
    __syncwarp();
    const uint32_t mine = stage + 128u * lane;
#pragma unroll
    for (int c = 0; c < 8; ++c)
        st_shared_v4(mine + 16u * (c ^ (lane & 7)), make_int4(static_cast<int>(w[4 * c]), static_cast<int>(w[4 * c + 1]),
                                                              static_cast<int>(w[4 * c + 2]), static_cast<int>(w[4 * c + 3])));
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0 && any) {
        tma_store_4d(map, stage, 0, head, query0, b);
        bulk_commit_group();
    }
}

// The grid has a CTA (or cluster) per unit; a CTA that finishes early takes over
// the units of CTAs that have not started, so that the next unit's copies and
// first scores run under the present one's last tiles and epilogue.
template <typename T, bool kSplit>
__global__ void __launch_bounds__(kTileThreads, 2) window_tile_kernel(const __grid_constant__ Maps maps, const Params p) {
    using S = TileSmem<kSplit>;
    constexpr int kKStages = S::kKStages;
    extern __shared__ __align__(1024) uint8_t smem[];  // the tiles' swizzle repeats every 1024 bytes
    const uint32_t sbase = smem_u32(smem);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::bars);
    const WaitCtl ctl{sbase + S::misc};
    const auto bar = [&](int idx) { return sbase + S::bars + 8u * idx; };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = kSplit ? static_cast<int>(cluster_nctarank()) : 1, rank = kSplit ? static_cast<int>(cluster_ctarank()) : 0;
    const int split_log2 = kSplit ? 31 - __clz(split) : 0;
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
        mbar_init(&bars[S::kNever], 1);
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
        if (p.out_boxes) prefetch_tensormap(&maps.out);
    }
    if (warp == 2) {
        tmem_alloc(reinterpret_cast<uint32_t*>(smem + S::misc), kTmemColsTile);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if constexpr (kSplit) cluster_arrive();  // this CTA runs: its shared memory may be stored to (waited for before the first store)
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
        const int query = row / p.pack;  // of this row in its unit
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
        bool ok = true, all_run = !kSplit;
        for (int i = 0; ok && record_wait(i, FDS_STATUS_TIMEOUT_SOFTMAX); ++i) {
            const int4 un = ld_shared_v4(record(i) + 16);  // t0, t1, p0, kv_end
            const int t1 = un.y;
            rs.t_begin = un.x;
            rs.m_run = -INFINITY;
            rs.l_run = 0.f;
            // this row's columns: [lo, hi) of the window part and the sinks, [a, z) (where
            // they lie in the window part: those of them up to p + right)
            const int4 c = ld_shared_v4(record(i) + 32);  // begin, n_win, s0, n_sink
            const int pos = un.z + query;
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
            // (a score of plus infinity: every weight is NaN, whatever the exponentials made of it)
            const float inv = none ? 1.f : (rs.m_run < INFINITY ? 1.f / rs.l_run : __uint_as_float(0x7fffffffu));
            uint32_t o[64];
            if (ok && t1 > rs.t_begin) {
                // (the next unit's first P V overwrites O only after this warpgroup's
                // next P store, which follows this read in program order)
                ok = warp_wait(rs.pv_done, rs.pv_parity, ctl, FDS_STATUS_TIMEOUT_SOFTMAX);
                rs.pv_parity ^= 1;
                tc_fence_after();
                tmem_ld64(rs.tO, o);
                tmem_wait_ld();
                if (__any_sync(0xffffffffu, none)) {
#pragma unroll
                    for (int e = 0; e < 64; ++e) o[e] = none ? 0 : o[e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 64; ++e) o[e] = 0;
            }
            if constexpr (!kSplit) {
                const int4 at = ld_shared_v4(record(i));  // b, h, row0, n: not held in registers over the tiles
                uint32_t w[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    const float2 v = fmul2(make_float2(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1])), make_float2(inv, inv));
                    w[e] = DTypeTraits<T>::pack(v.x, v.y);
                }
                if (p.out_boxes) {
                    const int q0 = __shfl_sync(0xffffffffu, query, 0);
                    store_box(sbase + S::stage + 4096u * (warp & 3), &maps.out, lane, w, at.y, at.z + q0, at.x, ok && q0 < at.w);
                } else if (ok && query < at.w) {
                    T* to = static_cast<T*>(p.out) + at.x * p.out_stride[0] + (at.z + query) * p.out_stride[1] +
                            (at.y + row - query * p.pack) * p.out_stride[2];
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        *reinterpret_cast<uint4*>(to + 2 * e) = make_uint4(w[e], w[e + 1], w[e + 2], w[e + 3]);
                }
            } else {
                cluster_wait();
                all_run = true;
                // to the CTA that owns the row (its row of it: row % (128 / split))
                const int own = kBlockM >> split_log2, at = rank * own + (row & (own - 1)), owner = row >> (7 - split_log2);
                const uint32_t to = map_to_rank(sbase + S::part + 256 * at, owner);
#pragma unroll
                for (int c = 0; c < 16; ++c)
                    st_cluster_v4f32(to + 16 * (c ^ (at & 15)), __uint_as_float(o[4 * c]) * inv, __uint_as_float(o[4 * c + 1]) * inv,
                                     __uint_as_float(o[4 * c + 2]) * inv, __uint_as_float(o[4 * c + 3]) * inv);
                st_cluster_f32(map_to_rank(sbase + S::lse + 4 * at, owner), none ? -INFINITY : rs.m_run + __log2f(rs.l_run));
            }
            if constexpr (!kSplit) record_release(i);
        }
        if (lane == 0) bulk_wait_all();  // the output boxes are written
        __syncwarp();
        tc_fence_before();
        named_barrier_arrive(1, kTmemDone);
        if constexpr (kSplit) {
            if (!all_run) cluster_wait();  // (a timeout before the unit was known)
            cluster_arrive();
            const int4 at = ld_shared_v4(record(0));  // (the end of the list is in the other slot)
            const int own = kBlockM >> split_log2, tid = static_cast<int>(threadIdx.x) - 128;
            const int mine = tid & (own - 1), mrow = rank * own + mine, mq = mrow / p.pack;
            T* to = static_cast<T*>(p.out) + at.x * p.out_stride[0] + (at.z + mq) * p.out_stride[1] +
                    (at.y + mrow - mq * p.pack) * p.out_stride[2];
            cluster_wait();  // every part is in place
            merge_parts<T>(sbase + S::part, sbase + S::lse, split, mine, (tid >> (7 - split_log2)) * (kHeadDim >> split_log2),
                           ok && all_run && mq < at.w, to);
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
            // test hook: a wait on a barrier that nothing arrives on, to exercise the
            // bounded-wait error path without a real hang
            if (p.debug_flags & FDS_DEBUG_FORCE_TIMEOUT) ok = warp_wait(bar(S::kNever), 0, ctl, err);
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
                        mbar_arrive_expect_tx(bar(S::kQ), static_cast<uint32_t>(p.pack * p.queries) * 128u);
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
            int block[3] = {static_cast<int>(blockIdx.x) >> split_log2, static_cast<int>(blockIdx.y), static_cast<int>(blockIdx.z)};
            bool ok = true, more = true;
            for (int i = 0; ok; ++i) {
                if (i >= kRecords) ok = warp_wait(bar(S::kRecEmpty + i % kRecords), (i / kRecords - 1) & 1, ctl, err);
                if (!ok) break;
                if (more) {
                    const Unit un = make_unit(p, block[0], block[1], block[2], split_log2, rank);
                    if (lane == 0) store_record(record(i), un);
                } else if (lane == 0) {
                    st_shared_volatile_u32(record(i) + 60, 0);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(S::kRecFull + i % kRecords));
                if (!more) break;
                if constexpr (kSplit) {  // a cluster holds one unit
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
                more = launch_control_answer(sbase + S::answer, block);
                fence_proxy_async_smem();  // the answer is read before the next one is written
                __syncwarp();
            }
        }
        __syncwarp();
        tc_fence_before();
        if constexpr (kSplit) {
            cluster_wait();
            cluster_arrive();
        }
        // TMEM is released once the MMAs have completed and the softmax warps have read O
        if (warp == 0) named_barrier_arrive(1, kTmemDone);
        if (warp == 2) {
            named_barrier_sync(1, kTmemDone);
            tc_fence_after();
            tmem_dealloc(tmem, kTmemColsTile);
        }
        if constexpr (kSplit) cluster_wait();
    }
}

// ---------------------------------------------------------------- step kernel

constexpr int kStepWarps = 4;
constexpr int kStepThreads = 32 * kStepWarps;
constexpr int kStepRows = 16;     // query rows per key head at most: one m16 fragment
constexpr int kStepKeys = 32;     // keys of a block
constexpr int kStepStages = 3;    // blocks in a warp's ring
constexpr int kBlockBytes = kStepKeys * 128;                       // keys or values of a block
constexpr int kStepWarpBytes = kStepStages * 2 * kBlockBytes;
constexpr int kPartFloats = 66;   // a row's 64 of O, max, sum
constexpr int kStepRings = kStepWarps * kStepWarpBytes;
constexpr int kStepSmem = kStepRings + kStepRows * kPartFloats * 4;  // and a cluster's parts of the rows this CTA owns
static_assert(kStepWarps * kStepRows * kPartFloats * 4 <= kStepRings, "partial rows over the rings");

// 16 bytes, or zeros, asynchronously into shared memory.
__device__ __forceinline__ void copy16_or_zero(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}

template <bool kTrans>
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t addr) {
    if constexpr (kTrans)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(addr)
                     : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(addr)
                     : "memory");
}

// c += a (16 x 16, row major) * b (16 x 8, column major), fp32 accumulation
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Row r is query r / group of key head hk, head hk * group + r % group. kHalves:
// 1 with at most 8 rows (the fragments' rows 8..15 are zero and skipped), else 2.
// kMulti: several queries, whose windows differ. The keys of a unit go to
// 4 * cluster warps in contiguous shares of whole blocks.
template <typename T, int kHalves, bool kMulti>
__global__ void __launch_bounds__(kStepThreads) window_step_kernel(const Params p) {
    extern __shared__ __align__(128) uint8_t step_smem[];
    const int split = static_cast<int>(gridDim.x), rank = static_cast<int>(blockIdx.x);
    if (split > 1) cluster_arrive();  // this CTA runs: its shared memory may be stored to
    grid_launch_dependents();
    grid_dependency_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;  // fragment row (or key, or value column) and column pair
    const int hk = blockIdx.y, b = blockIdx.z;
    const int group = p.heads / p.kv_heads;
    const int n_rows = p.q_len * group;

    // the query rows as A fragments, straight from memory
    uint32_t q[4][4];
    const T* qb = static_cast<const T*>(p.q) + b * p.q_stride[0] + 2 * t;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = g + 8 * h;
        const bool on = h < kHalves && r < n_rows;
        const T* src = qb + (on ? (r / group) * p.q_stride[1] + (hk * group + r % group) * p.q_stride[2] : 0);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            q[k][h] = on ? __ldg(reinterpret_cast<const uint32_t*>(src + 16 * k)) : 0u;
            q[k][2 + h] = on ? __ldg(reinterpret_cast<const uint32_t*>(src + 16 * k + 8)) : 0u;
        }
    }

    const Columns cols(p, b, 0, p.q_len);
    const int total = cols.n_sink + cols.n_win;  // sinks first, unpadded
    const int blocks = (total + kStepKeys - 1) / kStepKeys;
    const int shares = split * kStepWarps, share = rank * kStepWarps + warp;
    const int b_begin = static_cast<int>(static_cast<int64_t>(blocks) * share / shares);
    const int b_end = static_cast<int>(static_cast<int64_t>(blocks) * (share + 1) / shares);

    const uint32_t ring = smem_u32(step_smem) + warp * kStepWarpBytes;
    const T* kb = static_cast<const T*>(p.k) + b * p.k_stride[0] + hk * p.k_stride[2] + 8 * (lane & 7);
    const T* vb = static_cast<const T*>(p.v) + b * p.v_stride[0] + hk * p.v_stride[2] + 8 * (lane & 7);
    const auto fetch = [&](int blk) {  // 8 lanes a key; 16-byte piece c of key r at c ^ (r & 7)
        if (blk < b_end) {
            const uint32_t dst = ring + ((blk - b_begin) % kStepStages) * 2 * kBlockBytes;
#pragma unroll
            for (int i = 0; i < kStepKeys / 4; ++i) {
                const int r = 4 * i + (lane >> 3), x = blk * kStepKeys + r;
                const bool on = x < total;
                const int64_t key = on ? (x < cols.n_sink ? x : cols.begin + x - cols.n_sink) : 0;
                const uint32_t to = dst + 128u * r + 16u * ((lane & 7) ^ (r & 7));
                copy16_or_zero(to, kb + key * p.k_stride[1], on);
                copy16_or_zero(to + kBlockBytes, vb + key * p.v_stride[1], on);
            }
        }
        norm::copy_commit();
    };
#pragma unroll
    for (int s = 0; s < kStepStages - 1; ++s) fetch(b_begin + s);

    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[8][4];
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.f;

    for (int blk = b_begin; blk < b_end; ++blk) {
        norm::copy_wait<kStepStages - 2>();
        __syncwarp();  // every lane's copies of this block have landed, and the slot read last is free
        fetch(blk + kStepStages - 1);
        const uint32_t ks = ring + ((blk - b_begin) % kStepStages) * 2 * kBlockBytes, vs = ks + kBlockBytes;

        float s[4][4];  // scores of 8-key columns n: rows g (0, 1) and g + 8 (2, 3), keys 8 n + 2 t, + 1
#pragma unroll
        for (int n = 0; n < 4; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2) {  // 32 dims: four 8 x 8 matrices, keys 8 n .. 8 n + 7
                uint32_t f[4];
                load_matrices<false>(f, ks + 128u * (8 * n + (lane & 7)) + 16u * ((4 * k2 + (lane >> 3)) ^ (lane & 7)));
                mma16816<T>(s[n], q[2 * k2], f[0], f[1]);
                mma16816<T>(s[n], q[2 * k2 + 1], f[2], f[3]);
            }
        }
        const int x0 = blk * kStepKeys;
        if (kMulti || x0 + kStepKeys > total) {
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int x = x0 + 8 * n + 2 * t + (e & 1);
                    bool seen = x < total;
                    if constexpr (kMulti) {
                        const int key = x < cols.n_sink ? x : cols.begin + x - cols.n_sink;
                        const int pos = cols.p0 + (g + 8 * (e >> 1)) / group;
                        seen = seen && key <= pos + p.right && (key >= pos - p.left || key < p.sinks);
                    }
                    if (!seen) s[n][e] = -INFINITY;
                }
        }
        uint32_t pa[2][4];  // the weights as A fragments over 16 keys each
#pragma unroll
        for (int i = 0; i < 2; ++i) pa[i][1] = pa[i][3] = 0;
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
            float mt = s[0][2 * h];
#pragma unroll
            for (int n = 0; n < 4; ++n) mt = fmaxf(mt, fmaxf(s[n][2 * h], s[n][2 * h + 1]));
            mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
            mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2)) * p.scale_log2;
            const float mn = fmaxf(m[h], mt), base = mn == -INFINITY ? 0.f : mn;
            const float alpha = ex2_approx(m[h] - base);
            m[h] = mn;
            l[h] *= alpha;
#pragma unroll
            for (int n = 0; n < 8; ++n) o[n][2 * h] *= alpha, o[n][2 * h + 1] *= alpha;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const float e0 = ex2_approx(fmaf(s[n][2 * h], p.scale_log2, -base));
                const float e1 = ex2_approx(fmaf(s[n][2 * h + 1], p.scale_log2, -base));
                l[h] += e0 + e1;
                pa[n >> 1][2 * (n & 1) + h] = norm::pack2<T>(e0, e1);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int n = 0; n < 8; n += 2) {  // keys 16 i .. + 15, value columns 8 n .. + 15
                uint32_t f[4];
                const int r = 16 * i + (lane & 15);
                load_matrices<true>(f, vs + 128u * r + 16u * ((n + (lane >> 4)) ^ (r & 7)));
                mma16816<T>(o[n], pa[i], f[0], f[1]);
                mma16816<T>(o[n + 1], pa[i], f[2], f[3]);
            }
    }

    // this warp's rows, over the rings once every warp is done with its own
    norm::copy_wait<0>();
    __syncthreads();
    float* part = reinterpret_cast<float*>(step_smem);  // [warp][row][66]
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        float* row = part + (warp * kStepRows + g + 8 * h) * kPartFloats;
#pragma unroll
        for (int n = 0; n < 8; ++n) *reinterpret_cast<float2*>(row + 8 * n + 2 * t) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
        if (t == 0) row[64] = m[h], row[65] = l[h];
    }
    __syncthreads();
    const auto store = [&](int r, int c, float acc, float sum) {
        T* out = static_cast<T*>(p.out) + b * p.out_stride[0] + (r / group) * p.out_stride[1] +
                 (hk * group + r % group) * p.out_stride[2];
        out[c] = static_cast<T>(sum == 0.f ? 0.f : acc / sum);
    };
    // the warps' shares in order, then (a cluster) the CTAs' by the one that owns the
    // row, row % split: the others store theirs into its shared memory
    if (split > 1) cluster_wait();
    float* owned = reinterpret_cast<float*>(step_smem + kStepRings);  // [row / split][source][66]
    for (int i = threadIdx.x; i < n_rows * 64; i += kStepThreads) {
        const int r = i >> 6, c = i & 63;
        const float* from = part + r * kPartFloats;
        float mm = -INFINITY, acc = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kStepWarps; ++w) mm = fmaxf(mm, from[w * kStepRows * kPartFloats + 64]);
        const float base = mm == -INFINITY ? 0.f : mm;
#pragma unroll
        for (int w = 0; w < kStepWarps; ++w) {
            const float* fw = from + w * kStepRows * kPartFloats;
            const float f = ex2_approx(fw[64] - base);
            acc = fmaf(fw[c], f, acc);
            sum = fmaf(fw[65], f, sum);
        }
        if (split == 1) {
            store(r, c, acc, sum);
        } else {
            const int own = r / split;
            const uint32_t to = map_to_rank(smem_u32(owned + (own * split + rank) * kPartFloats), r - own * split);
            st_cluster_f32(to + 4u * c, acc);
            if (c == 0) st_cluster_f32(to + 4u * 64, mm);
            if (c == 1) st_cluster_f32(to + 4u * 65, sum);
        }
    }
    if (split == 1) return;
    __syncwarp();
    cluster_sync_all();
    for (int i = threadIdx.x; i < n_rows * 64; i += kStepThreads) {
        const int own = i >> 6, r = own * split + rank, c = i & 63;
        if (r >= n_rows) break;
        const float* from = owned + own * split * kPartFloats;
        float mm = -INFINITY, acc = 0.f, sum = 0.f;
        for (int k = 0; k < split; ++k) mm = fmaxf(mm, from[k * kPartFloats + 64]);
        const float base = mm == -INFINITY ? 0.f : mm;
        for (int k = 0; k < split; ++k) {
            const float f = ex2_approx(from[k * kPartFloats + 64] - base);
            acc = fmaf(from[k * kPartFloats + c], f, acc);
            sum = fmaf(from[k * kPartFloats + 65], f, sum);
        }
        store(r, c, acc, sum);
    }
}

}  // namespace window
}  // namespace fds
