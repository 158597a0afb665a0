// attention_tree on tcgen05 for BF16/FP16 and dim up to 128 (attention_tree.cu has
// the operator's definition).
//
// The M = group * seq rows of a (sequence, kv head) are one operand of the tensor
// core, 128 to a tile, so a key is read from HBM once whatever the number of query
// heads and drafted tokens; the kernel is bound by that stream up to M = 256
// (256 FLOP per byte of a 16-bit cache). dim is padded to 64 or 128 by the TMA
// loads' zero fill.
//
// Work: an item is a (sequence, kv head, row block); its keys are tiles of 128. The
// tiles of all items form one list (lengths are read on the device), cut into equal
// ranges, one per CTA: sequences of any mix of lengths load every SM alike. A range
// is a run of segments, each a part of one item. A CTA writes the rows of an item
// that it has whole; of an item that it shares it writes the unnormalised sums with
// their maxima, and tree_join_tc joins them in range order.
//   warp 0     TMA: Q of each segment, then K and V tiles through one ring of stages
//              in the order in which the MMA warp takes them
//   warp 1     MMA: S = Q K^T, O += P V, two chains t = 0, 1 so that the tensor core
//              works for one while the other's softmax runs
//   warps 2-5, 6-9  softmax of chain 0 / 1, one thread per row: scores out of TMEM,
//              running maximum and sum in FP32, P rounded to the input type back into
//              TMEM (the sum is of unrounded weights), O rescaled only when a maximum
//              has grown by more than 2^8 (BF16) or 2^4 (FP16). Relative error 2^-9 / 2^-12
//              per weight; FP16 has no exponents below 2^-14, so there P is kept 2^11
//              times as large: full precision down to 2^-25 of the row's largest weight,
//              an absolute error of 2^-36 of it below
// M <= 128: the chains take alternate key tiles of the same rows and are joined at
// the segment's end, both sums being in the same TMEM lanes. M > 128: the chains are
// two row tiles that share each K and V tile. M <= 64: the tile holds two copies of the
// rows, M <= 32: four, and each copy takes a half or a quarter of a key tile's columns
// (its P is zero in the others), so that all four warps of a chain work and none forms
// more than 128 / copies weights per row and tile; the copies' sums are joined with the
// chains'.
// Measured on B200, 8 kv heads of 128: 16 sequences of 1,000 to 8,000 keys, one token of 4
// heads each (295 MB), 63 us with the join = 4.7 TB/s; 4 of 9,000 to 16,000, 128 rows, 56 us
// (28 more for the weights); one of 131,000 in FP16, 256 rows, 152 to 157 us = 900 TFLOP/s at
// 1965 MHz (175 to 180 under the power cap), 2.2 us per pair of row tiles and key tile: bound
// by the chain of S, its softmax and P V, not by HBM. Copies: 4 rows of 64 elements, 43.7 us
// with four copies and 49.3 with none.
//
// A tile that reaches beyond the committed slots is masked per row by the drafts'
// bits. Its V rows from lengths + seq on are zeroed in shared memory before the
// product; non-finite elements of drafted V rows are zeroed too and added to the
// rows that see them at the end, so that they reach no other row.
#include <climits>
#include <mutex>
#include <type_traits>

#include "attention_softmax.cuh"
#include "attention_tree.cuh"

namespace jade {
namespace {

constexpr int kThreads = 10 * 32, kTileKeys = 128, kTileRows = 128;
// P = 2^(score - m): m lies kHeadroom below the largest score when it is set, and is kept
// until the largest has grown by kRescaleThreshold more (log2 units), so P <= 2^15 in FP16.
// Without the headroom a key of weight 2^-25 beside one of weight 1 became 0, while the
// row's sum counted it.
template <uint32_t kFmt>
struct Exponents {
    static constexpr float kHeadroom = kFmt == 0 ? 11.0f : 0.0f, kRescaleThreshold = kFmt == 0 ? 4.0f : 8.0f;
};
// An item's end in tiles (see "work ranges"), more of them the more rows it writes.
// Measured on B200, 4 rows, 128 items of 9 to 63 tiles: 73.8 us with 0, 67.3 with 2,
// 65.7 with 4, 64.6 with 6, 64.5 with 8, 67.0 with 12; 128 rows, 32 items of 72 to 126
// tiles: 60.3 us with 6, 56.8 with 10, 55.8 with 12, 55.4 with 16. Two row tiles
// (twice the time per tile): 73.6 us with 6, 74.9 with 10. Row counts between (4 to 128,
// three mixes of lengths from 100 to 16,000 keys): within 5 % of the best of 4, 8, 12 and 16.
constexpr int boundary_tiles(int rows) { return rows > 128 ? 6 : 6 + rows / 20; }

template <int DP, bool kTwoTiles, int kCopies>
struct Layout {
    static constexpr uint32_t kChunk = 128 * 128;  // 128 rows x 64 elements, 128-byte swizzle
    static constexpr uint32_t kTile = (DP / 64) * kChunk;
    static constexpr uint32_t kRing = 2 * kTile;  // behind Q: two row tiles, or this segment's and the next one's
    static constexpr uint32_t kMergeChain = 16384;  // joining the copies: 32 columns of the rows of all copies but one
    static constexpr uint32_t kMergeBytes = kCopies > 1 ? 2 * kMergeChain : 0;
    static constexpr int kStages = (224 * 1024 - kRing - kMergeBytes) / kTile;  // 128 KB or more of K and V in flight per SM
    static constexpr uint32_t kMerge = kRing + kStages * kTile;
    static constexpr uint32_t kExchange = kMerge + kMergeBytes;  // (maximum, sum) of every lane and chain
    static constexpr uint32_t kBar = kExchange + 2 * 128 * 8;
    static constexpr uint32_t kBytes = kBar + 512;
    // dynamic shared memory starts on a 1024-byte boundary in practice (checked in
    // the kernel); the slack covers the alignment where the layout leaves room for it
    static constexpr uint32_t kSmem = kBytes + 1024 < 227 * 1024 ? kBytes + 1024 : 227 * 1024;
};

// Stats of an item: x of every row, p_j = 2^(s_j scale_log2 + x) (the row's sum folded
// into the exponent: one constant per column for the weights' pass to read), -inf for
// rows that see nothing or add no weight, and up to whole groups of 32 columns of that
// pass's MMA.
__host__ __device__ constexpr size_t stats_stride(int rows) { return ((size_t)rows + 31) / 32 * 32; }
__device__ __forceinline__ void store_stats(const TreeArgs &t, size_t item, int row, float m, float inv) {
    float *x = t.row_exponents + item * stats_stride(t.rows) + row;
    *x = adds_weight(t, (int)(item / t.kv_heads), row) ? log2f(inv) - (m == -INFINITY ? 0.0f : m) : -INFINITY;
    if (row == t.rows - 1)
        for (int r = t.rows; r < (int)stats_stride(t.rows); ++r) *++x = -INFINITY;
}

struct TcArgs {
    TreeArgs t;
    int row_blocks, ctas, boundary, slot_rows;  // slot_rows: rows of a partial result
};

// ------------------------------------------------------------------ work ranges
// An item counts as its tiles and `boundary` more, the time that a CTA loses at an
// item's end (epilogue, new Q, an emptied pipeline) in tiles, so that ranges with
// more ends hold fewer tiles.
__device__ __forceinline__ int length_of(const TreeArgs &t, int b) { return b < t.batch ? __ldg(t.lengths + b) : 0; }
__device__ __forceinline__ int tiles_of(const TreeArgs &t, int length) {
    if (length < 0 || length > t.capacity - t.seq) return 0;
    return (length + t.seq + kTileKeys - 1) / kTileKeys;
}
__device__ __forceinline__ int units_of(const TcArgs &a, int b) {
    const int tiles = tiles_of(a.t, length_of(a.t, b));
    return tiles ? tiles + a.boundary : 0;
}
// Units of a CTA's range; total: of all sequences' items.
__device__ __forceinline__ long long range_units(const TcArgs &a, long long total) { return max(1ll, (total + a.ctas - 1) / a.ctas); }

struct Segment {
    int b, hk, rb, first, last, tiles, length;  // key tiles [first, last) of the item's `tiles`
    __device__ __forceinline__ int count() const { return last - first; }
};

// The segments of a CTA's range, in order; every role walks the same sequence. The
// next sequence's length is read one sequence ahead: under the stream of K and V a
// load takes microseconds.
struct Segments {
    int b, sub, unit, length, next_length;
    long long left;
    __device__ __forceinline__ bool next(const TcArgs &a, Segment &s) {
        while (left > 0) {
            const int tiles = tiles_of(a.t, length), units = tiles ? tiles + a.boundary : 0;
            if (unit >= units) {
                unit = 0;
                if (tiles == 0 || ++sub >= a.t.kv_heads * a.row_blocks) {
                    sub = 0;
                    if (++b >= a.t.batch) return false;
                    length = next_length;
                    next_length = length_of(a.t, b + 1);
                }
                continue;
            }
            const int upto = (int)min((long long)units, unit + left);
            s.b = b, s.hk = sub / a.row_blocks, s.rb = sub - s.hk * a.row_blocks;
            s.first = min(unit, tiles), s.last = min(upto, tiles), s.tiles = tiles, s.length = length;
            left -= upto - unit;
            unit = upto;
            if (s.count() > 0) return true;
        }
        return false;
    }
};

// The CTA's range (whole block; also the barrier behind its set-up, TMEM allocation
// included). plan: 4 ints, scratch: a long long per warp.
__device__ __forceinline__ Segments open_range(const TcArgs &a, int *plan, long long *scratch) {
    const TreeArgs &t = a.t;
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    long long mine = 0;
    for (int i = threadIdx.x; i < t.batch; i += blockDim.x) {
        const int units = units_of(a, i);
        mine += units;
        if (blockIdx.x == 0 && units == 0) atomicCAS(t.err, 0, kErrCacheLength);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0) scratch[threadIdx.x >> 5] = mine;
    __syncthreads();
    const long long items = (long long)t.kv_heads * a.row_blocks;
    long long total = 0;
    for (int w = 0; w < warps; ++w) total += scratch[w];
    total *= items;
    const long long per = range_units(a, total), begin = per * blockIdx.x;
    if (threadIdx.x < 32) {  // the first sequence whose units reach beyond `begin`
        long long base = 0;
        for (int b0 = 0; b0 < t.batch && begin < total; b0 += 32) {
            const int units = b0 + lane < t.batch ? units_of(a, b0 + lane) : 0;
            long long upto = units * items;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += x;
            }
            const uint32_t beyond = __ballot_sync(0xffffffffu, base + upto > begin);
            if (beyond && lane == __ffs(beyond) - 1) {
                const long long into = begin - (base + upto - units * items);
                plan[0] = b0 + lane, plan[1] = (int)(into / units), plan[2] = (int)(into % units);
            }
            if (beyond) break;
            base += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (begin >= total) return Segments{0, 0, 0, 0, 0, 0};
    return Segments{plan[0], plan[1], plan[2], length_of(t, plan[0]), length_of(t, plan[0] + 1), min(per, total - begin)};
}

// ------------------------------------------------------------------ masks
// Bit c of the result: the row sees column c of the tile whose first key lies `off`
// slots before the first draft (off may be negative: the tile starts among the drafts).
__device__ __forceinline__ void column_mask(const uint32_t (&bits)[4], int off, uint32_t (&mask)[4]) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const int i0 = 32 * w - off;  // draft of column 32 w
        uint32_t m = 0;
        if (i0 <= -32) m = 0xffffffffu;
        else if (i0 < 0) m = (1u << -i0) - 1 | bits[0] << -i0;
        else if (i0 < 128) {
            const int q = i0 >> 5, r = i0 & 31;
            uint32_t lo = 0, hi = 0;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                if (x == q) lo = bits[x];
                if (x == q + 1) hi = bits[x];
            }
            m = __funnelshift_r(lo, hi, r);
        }
        mask[w] = m;
    }
}

template <typename T>
__device__ __forceinline__ uint32_t exponent_bits() { return std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u; }

// Zeroes V rows that hold no entry, and the non-finite elements of drafted rows
// (whose drafts are noted in `bad`). A row's 64 elements are 128 contiguous bytes
// (the swizzle permutes 16-byte units within them), so both are runs of memory that
// the chain's 128 threads take 16 bytes at a time.
template <int DP, typename T>
__device__ __forceinline__ void clean_v(uint8_t *v, int thread, int j0, int length, int seq, uint32_t *bad) {
    const int draft0 = j0 - length;  // draft of the tile's first row
    const int from = max(0, -draft0), upto = min(kTileKeys, seq - draft0);
#pragma unroll 1
    for (uint32_t at = 0; at < (DP / 64) * 128 * 128; at += 128 * 128) {
        for (int u = upto * 8 + thread; u < kTileKeys * 8; u += 128) *reinterpret_cast<uint4 *>(v + at + u * 16) = make_uint4(0, 0, 0, 0);
        for (int u = from * 8 + thread; u < upto * 8; u += 128) {
            uint4 x = *reinterpret_cast<uint4 *>(v + at + u * 16);
            uint32_t *w = reinterpret_cast<uint32_t *>(&x);
            const uint32_t e = exponent_bits<T>();
            bool hit = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if ((w[i] & e) == e) w[i] &= 0xffff0000u, hit = true;
                if ((w[i] >> 16 & e) == e) w[i] &= 0x0000ffffu, hit = true;
            }
            if (hit) {
                *reinterpret_cast<uint4 *>(v + at + u * 16) = x;
                const int draft = draft0 + (u >> 3);
                atomicOr(&bad[draft >> 5], 1u << (draft & 31));
            }
        }
    }
}

// The infinities and NaN in 32 columns of `keys` rows of V, as a bit per column: {+inf, -inf,
// NaN} (whole warp, a row a lane; the first `columns`, a multiple of 8, are the head's).
template <typename T>
__device__ __noinline__ uint3 non_finite_columns(const T *v, int keys, int dim, int columns) {
    const uint32_t e = exponent_bits<T>();
    uint32_t pos = 0, neg = 0, nan = 0;
    for (int j = threadIdx.x & 31; j < keys; j += 32)
#pragma unroll 1
        for (int c = 0; c < min(32, columns); c += 8) {
            const uint4 u = __ldg(reinterpret_cast<const uint4 *>(v + (size_t)j * dim + c));
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t x = w[i / 2] >> 16 * (i & 1) & 0xffffu;
                if ((x & e) == e) ((x & 0x7fffu) != e ? nan : x & 0x8000u ? neg : pos) |= 1u << (c + i);
            }
        }
    return make_uint3(__reduce_or_sync(0xffffffffu, pos), __reduce_or_sync(0xffffffffu, neg), __reduce_or_sync(0xffffffffu, nan));
}

// ------------------------------------------------------------------ kernel
template <int DP, typename T, bool kTwoTiles, int kCopies>
__global__ void __launch_bounds__(kThreads, 1)
    tree_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const TcArgs args) {
    using L = Layout<DP, kTwoTiles, kCopies>;
    constexpr int kCopyRows = 128 / kCopies, kCopyKeys = 128 / kCopies;  // rows of a copy, columns of a tile that it takes
    constexpr uint32_t kFmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    constexpr uint32_t kIdescS = idesc_f32acc(kFmt, kFmt, false, false, kTileRows, kTileKeys);
    constexpr uint32_t kIdescO = idesc_f32acc(kFmt, kFmt, false, true, kTileRows, DP);
    constexpr int kDChunks = DP / 64, kStages = L::kStages;

    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    if (smem + L::kBytes > smem_raw + L::kSmem) {
        if (threadIdx.x == 0) atomicCAS(args.t.err, 0, kErrBadLaunch);
        return;
    }
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kBar);
    uint64_t *q_full = bars, *q_empty = bars + 2, *s_full = bars + 4, *p_full = bars + 6, *o_full = bars + 8, *o_free = bars + 10;
    uint64_t *x_full = bars + 12, *x_empty = bars + 13, *mma_done = bars + 14;
    uint64_t *full = bars + 16, *empty = bars + 16 + kStages;  // ring stages
    uint64_t *g_full = bars + 44, *g_empty = bars + 46;  // joining the copies [chain]
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 48);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    uint32_t *bad = tmem_slot + 4;  // [4][4]: drafts with non-finite V, by segment number modulo 4
    int *plan = reinterpret_cast<int *>(tmem_slot + 20);  // the range's first b, sub, tile and (64 bits) length
    float2 *exchange = reinterpret_cast<float2 *>(smem + L::kExchange);  // [chain][row]
    static_assert(16 + 2 * kStages <= 44, "barriers");

    const TreeArgs &ta = args.t;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int *err = ta.err;
    int ring_loads = 0, q_loads = 0;  // issued by the producer (read on the abort path, after every role ended)

    if (threadIdx.x == 0) {
        for (int t = 0; t < 2; ++t) {
            mbar_init(&q_full[t], 1); mbar_init(&q_empty[t], 1);
            mbar_init(&s_full[t], 1); mbar_init(&p_full[t], 128);
            mbar_init(&o_full[t], 1); mbar_init(&o_free[t], kTwoTiles ? 128 : 256);
        }
        for (int t = 0; t < 2; ++t) mbar_init(&g_full[t], 128 - kCopyRows + (kCopies == 1)), mbar_init(&g_empty[t], kCopyRows);
        mbar_init(x_full, 256); mbar_init(x_empty, 256); mbar_init(mma_done, 1);
        for (int s = 0; s < kStages; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
        *abort_flag = 0;
        for (int i = 0; i < 16; ++i) bad[i] = 0;
        fence_barrier_init();
        fence_proxy_async();
    }
    if (warp == 0) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    Segments segments = open_range(args, plan, reinterpret_cast<long long *>(exchange));
    grid_dependency_trigger();
    const uint32_t tmem = *tmem_slot;
    const uint32_t tmem_s[2] = {tmem, tmem + 128};
    const uint32_t tmem_o[2] = {tmem + 256, tmem + 384};
    Segment s;

    if (warp == 0) {
        if (lane == 0) {  // ------------------------------------- TMA producer
            tma_prefetch_desc(&tmQ);
            tma_prefetch_desc(&tmK);
            tma_prefetch_desc(&tmV);
            bool ok = true;
            while (ok && segments.next(args, s)) {
                const int bh = s.b * ta.kv_heads + s.hk, n = s.count();
                auto load = [&](const CUtensorMap &map, int tile) {
                    const int st = ring_loads % kStages;
                    if (!(ok = ok && mbar_wait(&empty[st], (ring_loads / kStages & 1) ^ 1, abort_flag, err, kErrWaitSmemEmpty))) return;
                    mbar_arrive_expect_tx(&full[st], L::kTile);
                    for (int c = 0; c < kDChunks; ++c)
                        tma_load_3d(smem + L::kRing + st * L::kTile + c * L::kChunk, &map, &full[st], c * 64, (s.first + tile) * kTileKeys, bh);
                    ++ring_loads;
                };
                auto load_q = [&](int buffer, int tile, int use) {
                    if (!(ok = ok && mbar_wait(&q_empty[buffer], (use & 1) ^ 1, abort_flag, err, kErrWaitSmemEmpty))) return;
                    mbar_arrive_expect_tx(&q_full[buffer], L::kTile);
                    for (int c = 0; c < kDChunks; ++c)
                        for (int copy = 0; copy < kCopies; ++copy)
                            tma_load_3d(smem + buffer * L::kTile + c * L::kChunk + copy * kCopyRows * 128, &tmQ, &q_full[buffer], c * 64,
                                        tile * kTileRows, bh);
                };
                if constexpr (kTwoTiles) {  // row tiles 2 rb and 2 rb + 1 (which may lie beyond the rows: zeros)
                    load_q(0, 2 * s.rb, q_loads);
                    load_q(1, 2 * s.rb + 1, q_loads);
                    if (ok) ++q_loads;
                    load(tmK, 0);
                    for (int i = 0; i < n; ++i) {
                        load(tmV, i);
                        if (i + 1 < n) load(tmK, i + 1);
                    }
                } else {  // Q buffers alternate between segments
                    load_q(q_loads & 1, 0, q_loads >> 1);
                    if (ok) ++q_loads;
                    load(tmK, 0);
                    if (n > 1) load(tmK, 1);
                    for (int i = 0; i < n; ++i) {
                        load(tmV, i);
                        if (i + 2 < n) load(tmK, i + 2);
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------- MMA issuer (whole warp, one elected lane issues)
        auto wait = [&](uint64_t *bar, uint32_t parity, int code) {
            return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, err, code));
        };
        const uint64_t dq0 = sdesc_sw128(smem_u32(smem), 16, 1024);
        const uint64_t dk0 = sdesc_sw128(smem_u32(smem + L::kRing), 16, 1024);
        const uint64_t dv0 = sdesc_sw128(smem_u32(smem + L::kRing), L::kChunk, 1024);
        auto issue_s = [&](int t, int q_buffer, int stage) {
            uint64_t a[DP / 16], b[DP / 16];
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
                const uint32_t off = ((k >> 2) * L::kChunk + (k & 3) * 32) >> 4;
                a[k] = dq0 + ((q_buffer * L::kTile) >> 4) + off;
                b[k] = dk0 + ((stage * L::kTile) >> 4) + off;
            }
            umma_ss_group<DP / 16>(tmem_s[t], a, b, kIdescS, 0);
            umma_commit(&s_full[t]);
        };
        auto issue_pv = [&](int t, int stage, bool accumulate) {
            uint64_t b[kTileKeys / 16];
#pragma unroll
            for (int k = 0; k < kTileKeys / 16; ++k) b[k] = dv0 + ((stage * L::kTile) >> 4) + ((k * 16 * 128) >> 4);
            umma_ts_group8(tmem_o[t], tmem_s[t], b, kIdescO, accumulate);
        };
        // pos: ring loads consumed; qn: segments begun; cp: P tiles consumed; on: segments whose O_t was used
        int pos = 0, qn = 0, cp[2] = {0, 0}, on[2] = {0, 0};
        bool ok = true;
        auto ready = [&] {  // the ring's next stage has landed
            ok = ok && wait(&full[pos % kStages], pos / kStages & 1, kErrWaitTmaFull);
            return ok;
        };
        auto release = [&] { umma_commit(&empty[pos++ % kStages]); };
        auto p_ready = [&](int t, bool first) {  // P_t is written; for an item's first P V also: the last segment's O_t is read out
            ok = ok && wait(&p_full[t], cp[t]++ & 1, kErrWaitProb);
            if (first) {
                if (on[t] > 0) ok = ok && wait(&o_free[t], (on[t] - 1) & 1, kErrWaitAccEmpty);
                ++on[t];
            }
            return ok;
        };
        while (ok && segments.next(args, s)) {
            const int n = s.count();
            if constexpr (kTwoTiles) {
                ok = wait(&q_full[0], qn & 1, kErrWaitTmaFull) && wait(&q_full[1], qn & 1, kErrWaitTmaFull);
                ++qn;
                if (!ready()) break;
                tc_fence_after();
                for (int t = 0; t < 2; ++t) issue_s(t, t, pos % kStages);
                release();
                for (int i = 0; i < n && ready(); ++i) {
                    const int v = pos % kStages, k = (pos + 1) % kStages;
                    for (int t = 0; t < 2 && p_ready(t, i == 0); ++t) {
                        tc_fence_after();
                        issue_pv(t, v, i > 0);  // reads P_t(i) from TMEM: must precede S_t(i + 1)
                        if (i + 1 < n) {
                            if (t == 0 && !(ok = wait(&full[k], (pos + 1) / kStages & 1, kErrWaitTmaFull))) break;
                            tc_fence_after();
                            issue_s(t, t, k);
                        } else {
                            umma_commit(&o_full[t]);
                        }
                    }
                    if (!ok) break;
                    release();
                    if (i + 1 < n) release();
                }
                for (int t = 0; t < 2; ++t) umma_commit(&q_empty[t]);
            } else {
                const int q = qn & 1;
                ok = wait(&q_full[q], qn++ >> 1 & 1, kErrWaitTmaFull);
                for (int i = 0; i < 2 && i < n && ready(); ++i) {
                    tc_fence_after();
                    issue_s(i, q, pos % kStages);
                    release();
                }
                if (n <= 2) umma_commit(&q_empty[q]);
                for (int i = 0; i < n && ready() && p_ready(i & 1, i < 2); ++i) {
                    const int t = i & 1;
                    tc_fence_after();
                    issue_pv(t, pos % kStages, i >= 2);
                    release();
                    if (i + 2 < n) {
                        if (!ready()) break;
                        tc_fence_after();
                        issue_s(t, q, pos % kStages);
                        release();
                        if (i + 3 == n) umma_commit(&q_empty[q]);  // the segment's last S: Q may be replaced
                    } else {
                        umma_commit(&o_full[t]);
                    }
                }
            }
        }
        umma_commit(mma_done);
        mbar_wait_drain(mma_done, 0, err);
    } else {
        // ----------------------------------------------------- softmax (warps 2-5: chain 0, 6-9: chain 1)
        const int t = (warp - 2) >> 2, quarter = warp & 3, row = quarter * 32 + lane, copy = row / kCopyRows, copy_row = row % kCopyRows;
        const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
        const uint32_t ts = tmem_s[t] + lane_off, to = tmem_o[t] + lane_off;
        const float c = ta.scale_log2;
        // cs: S tiles consumed; on: segments with O_t; xn: exchanges; gn: columns joined; ring: loads before the segment; sn: segments
        int cs = 0, on[2] = {0, 0}, xn = 0, gn = 0, ring = 0, sn = 0;
        bool ok = true;
        for (; ok && segments.next(args, s); ++sn) {
            const int n = s.count(), bh = s.b * ta.kv_heads + s.hk;
            const int item_row = kTwoTiles ? s.rb * 256 + t * 128 + row : copy_row;  // row of the item's M
            const bool live = __any_sync(0xffffffffu, item_row < ta.rows);      // some row of this warp is one
            uint32_t bits[4] = {0, 0, 0, 0};
            // The next segment's notes are cleared here by chain 0. With two row tiles chain 1 may
            // still read those of segment sn - 2, as O_0 of a segment of one tile is ready without
            // chain 1's P; but not those of sn - 3: the MMA warp has seen o_free[1] of that segment
            // before its first P_1 V of sn - 2, and so before anything of sn - 1.
            uint32_t *bad_now = bad + (sn & 3) * 4;
            if (threadIdx.x == 64)
                for (int i = 0; i < 4; ++i) bad[((sn + 1) & 3) * 4 + i] = 0;
            if (item_row < ta.rows)
                for (int w = 0; w < 4; ++w)
                    if (w < ta.words) bits[w] = __ldg(ta.tree + ((size_t)s.b * ta.seq + item_row % ta.seq) * ta.words + w);
            float m_used = -INFINITY, l_run = 0.0f;
            const int step = kTwoTiles ? 1 : 2;
            bool first = true;
            for (int i = kTwoTiles ? 0 : t; i < n; i += step, first = false) {
                ok = __all_sync(0xffffffffu, mbar_wait(&s_full[t], cs++ & 1, abort_flag, err, kErrWaitScore));
                if (!ok) break;
                tc_fence_after();
                const int j0 = (s.first + i) * kTileKeys;
                const bool masked = j0 + kTileKeys > s.length;
                if (masked && (!kTwoTiles || t == 0)) {  // V(i) in place of what no row may multiply
                    const int at = ring + (kTwoTiles ? 1 + 2 * i : min(2, n) + i + max(0, min(i, n - 2)));
                    ok = __all_sync(0xffffffffu, mbar_wait(&full[at % kStages], at / kStages & 1, abort_flag, err, kErrWaitTmaFull));
                    if (!ok) break;
                    clean_v<DP, T>(smem + L::kRing + (at % kStages) * L::kTile, row, j0, s.length, ta.seq, bad_now);
                    fence_proxy_async();
                }
                if (live) {
                    float sv[kCopyKeys];
#pragma unroll
                    for (int k = 0; k < kCopyKeys; k += 32) tmem_ld32f(ts + copy * kCopyKeys + k, sv + k);
                    tmem_wait_ld();
                    if (masked) {
                        uint32_t seen[4], mask[4];
#pragma unroll
                        for (int w = 0; w < 4; ++w) seen[w] = bits[w] & draft_bits(w, ta.seq);
                        column_mask(seen, s.length - j0 - copy * kCopyKeys, mask);
#pragma unroll
                        for (int k = 0; k < kCopyKeys; ++k) sv[k] = mask[k >> 5] >> (k & 31) & 1 ? sv[k] : -INFINITY;
                    }
                    float mx[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) mx[e] = max3(sv[e], sv[e + 8], sv[e + 16]);
#pragma unroll
                    for (int k = 24; k < kCopyKeys - 8; k += 16)
#pragma unroll
                        for (int e = 0; e < 8; ++e) mx[e] = max3(mx[e], sv[k + e], sv[k + 8 + e]);
#pragma unroll
                    for (int e = 0; e < 8; ++e) mx[e] = fmaxf(mx[e], sv[kCopyKeys - 8 + e]);
                    using E = Exponents<kFmt>;
                    const float m_tile = max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7])) * c - E::kHeadroom;
                    float m_new = m_used, alpha = 1.0f;
                    if (first) m_new = m_tile;
                    else if (m_tile > m_used + E::kRescaleThreshold) {
                        m_new = m_tile;
                        alpha = mufu_exp2(m_used - m_new);
                    }
                    m_used = m_new;
                    // a row that has seen nothing yet, or only scores of -inf, has maximum -inf: its weights are e^-inf = 0
                    const uint32_t tp = ts + copy * (kCopyKeys / 2);
                    // Every exponential on the special-function units: the polynomial that the prompt kernel
                    // gives a share to clamps a NaN, so that a NaN key would drop out of its row, and
                    // gains nothing here (131,000 keys, 256 rows: 155 us with it and without).
                    const float psum = store_p<kFmt, false, kCopyKeys>(sv, c, m_used == -INFINITY ? 0.0f : m_used, tp);
                    if constexpr (kCopies > 1) {
                        const uint32_t zeros[8] = {};
#pragma unroll
                        for (int k = 0; k < 64; k += 8)
                            if (k / (kCopyKeys / 2) != copy) tmem_st8(ts + k, zeros);
                    }
                    if (!first && __any_sync(0xffffffffu, alpha != 1.0f)) {
#pragma unroll 1
                        for (int oc = 0; oc < DP; oc += 32) {
                            float ov[32];
                            tmem_ld32f(to + oc, ov);
                            tmem_wait_ld();
#pragma unroll
                            for (int k = 0; k < 32; ++k) ov[k] *= alpha;
                            tmem_st32f(to + oc, ov);
                        }
                    }
                    l_run = l_run * alpha + psum;
                    tmem_wait_st();
                }
                tc_fence_before();
                mbar_arrive(&p_full[t]);
            }
            ring += 2 * n;
            if (!ok) break;
            // ------------------------------------------------- the segment's rows
            const bool both = !kTwoTiles && n > 1;  // chain 1 has sums too
            float f0 = 1.0f, f1 = 0.0f;             // factors of the two chains' sums
            if constexpr (!kTwoTiles) {             // both chains' threads write half of the columns each
                ok = __all_sync(0xffffffffu, mbar_wait(x_empty, (xn & 1) ^ 1, abort_flag, err, kErrWaitAccEmpty));
                if (!ok) break;
                exchange[t * 128 + row] = make_float2(m_used, l_run);
                mbar_arrive(x_full);
                ok = __all_sync(0xffffffffu, mbar_wait(x_full, xn++ & 1, abort_flag, err, kErrWaitPv));
                if (!ok) break;
                float2 e[2][kCopies];
                m_used = -INFINITY;
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int y = 0; y < kCopies; ++y) e[x][y] = exchange[x * 128 + y * kCopyRows + copy_row], m_used = fmaxf(m_used, e[x][y].x);
                mbar_arrive(x_empty);
                const float shift = m_used == -INFINITY ? 0.0f : m_used;
                l_run = 0.0f;
#pragma unroll
                for (int y = 0; y < kCopies; ++y) {
                    const float g0 = mufu_exp2(e[0][y].x - shift), g1 = mufu_exp2(e[1][y].x - shift);
                    l_run += e[0][y].y * g0 + e[1][y].y * g1;
                    if (y == copy) f0 = g0, f1 = g1;
                }
            }
            const int o0 = kTwoTiles ? t : 0;
            ok = __all_sync(0xffffffffu, mbar_wait(&o_full[o0], on[o0]++ & 1, abort_flag, err, kErrWaitPv));
            if (ok && both) ok = __all_sync(0xffffffffu, mbar_wait(&o_full[1], on[1]++ & 1, abort_flag, err, kErrWaitPv));
            if (!ok) break;
            tc_fence_after();
            const bool whole = s.first == 0 && s.last == s.tiles, valid = item_row < ta.rows && copy == 0;
            const float inv = l_run > 0.0f || l_run != l_run ? 1.0f / l_run : 0.0f;
            if (whole) f0 *= inv, f1 *= inv;
            uint32_t extra[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) extra[w] = valid ? bad_now[w] & bits[w] & draft_bits(w, ta.seq) : 0;
            const size_t slot = (size_t)blockIdx.x * 2 + (s.first == 0);
            const int g = item_row / ta.seq, tok = item_row - g * ta.seq;
            T *out = static_cast<T *>(ta.out) + (((size_t)s.b * ta.seq + tok) * ta.kv_heads * ta.group + s.hk * ta.group + g) * ta.dim;
            const int slot_row = kTwoTiles ? t * 128 + row : row, slot_rows = args.slot_rows;
            float4 *part = reinterpret_cast<float4 *>(ta.part_o) + slot * (DP / 4) * slot_rows + slot_row;
            constexpr int kColumns = kTwoTiles ? DP : DP / 2;
            const int first_column = kTwoTiles ? 0 : t * kColumns;
            if (live) {
#pragma unroll 1
                for (int oc = first_column; oc < first_column + kColumns; oc += 32) {
                    float r[32];
                    tmem_ld32f(tmem_o[o0] + lane_off + oc, r);
                    tmem_wait_ld();
                    if (both) {
                        float x[32];
                        tmem_ld32f(tmem_o[1] + lane_off + oc, x);
                        tmem_wait_ld();
#pragma unroll
                        for (int k = 0; k < 32; ++k) r[k] = f0 * r[k] + f1 * x[k];
                    } else {
#pragma unroll
                        for (int k = 0; k < 32; ++k) r[k] *= f0;
                    }
                    if constexpr (kCopies > 1) {  // the first copy's threads add up the others' rows, 32 columns at a time
                        float *merge = reinterpret_cast<float *>(smem + L::kMerge + t * L::kMergeChain);
                        if (copy > 0) {
                            ok = ok && __all_sync(0xffffffffu, mbar_wait(&g_empty[t], (gn & 1) ^ 1, abort_flag, err, kErrWaitAccEmpty));
#pragma unroll
                            for (int k = 0; k < 32; ++k) merge[((copy - 1) * 32 + k) * kCopyRows + copy_row] = r[k];
                            mbar_arrive(&g_full[t]);
                        } else {
                            ok = ok && __all_sync(0xffffffffu, mbar_wait(&g_full[t], gn & 1, abort_flag, err, kErrWaitPv));
#pragma unroll
                            for (int y = 0; y < kCopies - 1; ++y)
#pragma unroll
                                for (int k = 0; k < 32; ++k) r[k] += merge[(y * 32 + k) * kCopyRows + copy_row];
                            mbar_arrive(&g_empty[t]);
                        }
                        ++gn;
                    }
                    // An infinity of a committed V row times a P of 0 (another copy's columns, a weight below
                    // the type's range) is NaN, where the row's value is that infinity: such a column is
                    // read again. Never taken by a finite cache.
                    bool odd = false;
#pragma unroll
                    for (int k = 0; k < 32; ++k) odd |= !isfinite(r[k]);
                    const int committed = min(s.last * kTileKeys, s.length) - s.first * kTileKeys;
                    if (__any_sync(0xffffffffu, odd && valid) && committed > 0) {
                        const uint3 at = non_finite_columns(static_cast<const T *>(ta.v) + ((size_t)bh * ta.capacity + (size_t)s.first * kTileKeys) * ta.dim + oc,
                                                            committed, ta.dim, ta.dim - oc);
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if ((at.x | at.y | at.z) >> k & 1) {
                                const float x = (at.z | (at.x & at.y)) >> k & 1 ? NAN : at.x >> k & 1 ? INFINITY : -INFINITY;
                                r[k] = whole ? x * inv : x;
                            }
                    }
                    if (extra[0] | extra[1] | extra[2] | extra[3]) {  // non-finite values that this row sees
#pragma unroll
                        for (int w = 0; w < 4; ++w)
#pragma unroll 1
                            for (uint32_t left = extra[w]; left; left &= left - 1) {
                                const int d = 32 * w + __ffs(left) - 1;
                                const T *v = static_cast<const T *>(ta.v) + ((size_t)bh * ta.capacity + s.length + d) * ta.dim + oc;
#pragma unroll
                                for (int k = 0; k < 32; ++k)
                                    if (oc + k < ta.dim) {
                                        const float x = to_f32<T>(v[k]);
                                        if (!isfinite(x)) r[k] += x;
                                    }
                            }
                    }
                    if (valid && whole) {
#pragma unroll
                        for (int k = 0; k < 32; k += 8)
                            if (oc + k < ta.dim)
                                *reinterpret_cast<uint4 *>(out + oc + k) = make_uint4(pack16<kFmt>(r[k], r[k + 1]), pack16<kFmt>(r[k + 2], r[k + 3]),
                                                                                      pack16<kFmt>(r[k + 4], r[k + 5]), pack16<kFmt>(r[k + 6], r[k + 7]));
                    } else if (valid) {  // [dim / 4][row] so that a warp's rows are one run of memory
#pragma unroll
                        for (int k = 0; k < 32; k += 4)
                            part[(size_t)((oc + k) / 4) * slot_rows] = make_float4(r[k], r[k + 1], r[k + 2], r[k + 3]);
                    }
                    __syncwarp();
                }
            }
            if (!ok) break;
            tc_fence_before();
            mbar_arrive(&o_free[o0]);
            if (both) mbar_arrive(&o_free[1]);
            if (valid && (kTwoTiles || t == 0)) {
                if (!whole) ta.part_ml[slot * slot_rows + slot_row] = make_float2(m_used, l_run);
                else if (ta.row_exponents) store_stats(ta, bh, item_row, m_used, inv);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        if (lane == 0 && *abort_flag) {  // TMA loads still in flight land before the CTA exits
            for (int i = max(0, ring_loads - kStages); i < ring_loads; ++i) mbar_wait_drain(&full[i % kStages], i / kStages & 1, err);
            for (int i = max(0, q_loads - (kTwoTiles ? 1 : 2)); i < q_loads; ++i) {
                if (kTwoTiles) mbar_wait_drain(&q_full[0], i & 1, err), mbar_wait_drain(&q_full[1], i & 1, err);
                else mbar_wait_drain(&q_full[i & 1], i >> 1 & 1, err);
            }
        }
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Joins the parts of items that several CTAs share, in range order. A thread takes
// one row and four columns: consecutive threads, consecutive memory of every part.
// kWays > 1: the parts are dealt to kWays threads each, whose sums are added in order:
// few items have many parts, and one thread would wait for them one after the other
// (one head of 90,000 keys: 29 us with eight, 69 with one; the rule is at the launch).
constexpr int kJoinThreads = 256;

template <int DP, typename T, int kWays>
__global__ void __launch_bounds__(kJoinThreads) tree_join_tc(const TcArgs a, int blocks) {
    constexpr int kEach = kJoinThreads / kWays;  // rows x columns / 4 of a block
    __shared__ long long counts[2];
    __shared__ float maxima[kWays][kEach];
    __shared__ float4 sums[kWays][kEach];
    __shared__ float totals[kWays][kEach];
    const TreeArgs &t = a.t;
    const int subs = t.kv_heads * a.row_blocks;
    const int item = blockIdx.x / blocks, b = item / subs, sub = item - b * subs, hk = sub / a.row_blocks, rb = sub - hk * a.row_blocks;
    grid_dependency_trigger();
    if (threadIdx.x < 32) {
        long long all = 0, before = 0;
        for (int i = threadIdx.x; i < t.batch; i += 32) {
            const int n = units_of(a, i);
            all += n;
            if (i < b) before += n;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o), before += __shfl_xor_sync(0xffffffffu, before, o);
        if (threadIdx.x == 0) counts[0] = all, counts[1] = before;
    }
    __syncthreads();
    const int way = threadIdx.x / kEach, lane = threadIdx.x % kEach;
    const int at = (blockIdx.x - item * blocks) * kEach + lane, col = at / a.slot_rows, slot_row = at - col * a.slot_rows;
    const int row = rb * a.slot_rows + slot_row;
    const int tiles = tiles_of(t, length_of(t, b));
    grid_dependency_wait();  // in every block: this grid's end stands for the one's before it
    const long long per = range_units(a, counts[0] * subs), begin = counts[1] * subs + (long long)sub * (tiles + a.boundary);
    const int c0 = (int)(begin / per), c1 = (int)((begin + tiles - 1) / per);
    if (tiles == 0 || c0 == c1) return;  // c0 == c1: written whole
    const bool on = row < t.rows && col * 4 < DP;
    auto slot = [&](int c) { return (size_t)c * 2 + (c == c0); };
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (on)
        for (int c = c0 + way; c <= c1; c += kWays) m = fmaxf(m, t.part_ml[slot(c) * a.slot_rows + slot_row].x);
    if constexpr (kWays > 1) {
        maxima[way][lane] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWays; ++w) m = fmaxf(m, maxima[w][lane]);
    }
    const float shift = m == -INFINITY ? 0.0f : m;
    if (on) {
        const float4 *part = reinterpret_cast<const float4 *>(t.part_o) + at;
#pragma unroll 4
        for (int c = c0 + way; c <= c1; c += kWays) {
            const float2 ml = t.part_ml[slot(c) * a.slot_rows + slot_row];
            const float4 x = part[slot(c) * (DP / 4) * a.slot_rows];
            const float w = exp2f(ml.x - shift);
            l = fmaf(ml.y, w, l);
            o.x = fmaf(w, x.x, o.x), o.y = fmaf(w, x.y, o.y), o.z = fmaf(w, x.z, o.z), o.w = fmaf(w, x.w, o.w);
        }
    }
    if constexpr (kWays > 1) {
        sums[way][lane] = o, totals[way][lane] = l;
        __syncthreads();
        if (way > 0) return;
#pragma unroll
        for (int w = 1; w < kWays; ++w) {
            const float4 x = sums[w][lane];
            o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
            l += totals[w][lane];
        }
    }
    if (!on) return;
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    if (col == 0 && t.row_exponents) store_stats(t, (size_t)b * t.kv_heads + hk, row, m, inv);
    if (col * 4 >= t.dim) return;
    constexpr uint32_t kFmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    const int g = row / t.seq, tok = row - g * t.seq;
    T *out = static_cast<T *>(t.out) + (((size_t)b * t.seq + tok) * t.kv_heads * t.group + hk * t.group + g) * t.dim + col * 4;
    *reinterpret_cast<uint2 *>(out) = make_uint2(pack16<kFmt>(o.x * inv, o.y * inv), pack16<kFmt>(o.z * inv, o.w * inv));
}

// ------------------------------------------------------------------ weights
// weights[j] += sum over the item's M rows of p_j = 2^(s_j c + x), x the rows' stats
// from the pass before. Transposed, S^T = K Q^T with 128 keys in the TMEM
// lanes and up to 256 rows of Q in the columns, so that a thread owns a key and adds
// its row of p in order: no sums between threads, no atomics. Ranges of key tiles per
// CTA as above; more than 256 rows take several passes over the segment's keys. Tiles
// go last to first: the pass before has left a range's last ones in L2.
// Bound by K's second read and by one exponential per (row, key): 32 heads of 9,000 to
// 16,000 keys, 128 rows, 28 us, where the exponentials alone take 11.
//   warp 0 TMA (Q rows and their stats per segment, K tiles through a ring),
//   warp 1 MMA into two or four buffers (four where 128 columns do, so that S of a
//   group's next tile is ready when it has finished one), warps 2-5 and 6-9 take the
//   tiles in turn.
constexpr int kWeightRows = 256, kWeightsBoundary = 2, kTreeBytes = 128 * 4 * 4;

template <int DP>
struct WeightsLayout {
    static constexpr uint32_t kRows64 = kWeightRows * 128;  // 64 elements of every row of Q
    static constexpr uint32_t kTile = (DP / 64) * 128 * 128;
    static constexpr int kStages = DP == 128 ? 4 : 8;
    static constexpr uint32_t kRing = (DP / 64) * kRows64;
    static constexpr uint32_t kStats = kRing + kStages * kTile;
    static constexpr uint32_t kTree = kStats + kWeightRows * 4;  // per consumer warp: the sequence's tree words
    static constexpr uint32_t kBar = kTree + 8 * kTreeBytes;
    static constexpr uint32_t kSmem = kBar + 512 + 1024;
};

template <int DP, typename T>
__global__ void __launch_bounds__(kThreads, 1)
    tree_weights_tc(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const TcArgs args) {
    using L = WeightsLayout<DP>;
    constexpr uint32_t kFmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    constexpr int kDChunks = DP / 64, kStages = L::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kBar);
    uint64_t *q_full = bars, *q_empty = bars + 2, *mma_done = bars + 4, *s_full = bars + 5, *s_empty = bars + 9;
    uint64_t *full = bars + 13, *empty = bars + 13 + kStages;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 30);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    int *plan = reinterpret_cast<int *>(tmem_slot + 2);
    long long *scratch = reinterpret_cast<long long *>(tmem_slot + 6);

    const TreeArgs &ta = args.t;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int *err = ta.err;
    int ring_loads = 0, q_loads = 0;
    if (threadIdx.x == 0) {
        mbar_init(mma_done, 1);
        for (int t = 0; t < 2; ++t) mbar_init(&q_full[t], 1), mbar_init(&q_empty[t], 1 + 256);
        for (int t = 0; t < 4; ++t) mbar_init(&s_full[t], 1), mbar_init(&s_empty[t], 128);
        for (int i = 0; i < kStages; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
        *abort_flag = 0;
        fence_barrier_init();
        fence_proxy_async();
    }
    if (warp == 0) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    Segments segments = open_range(args, plan, scratch);
    const uint32_t tmem = *tmem_slot;
    // Up to 128 rows: four S buffers, and Q of the next segment loads beside this one's
    // (128 rows each); else two buffers, one Q of up to 256 rows at a time.
    const bool narrow = ta.rows <= 128;
    const int buffers = narrow ? 4 : 2, buffer_columns = 512 / buffers;
    auto q_buffer = [&](int use) { return narrow ? use & 1 : 0; };
    auto q_phase = [&](int use) { return narrow ? use >> 1 & 1 : use & 1; };
    Segment s;

    if (warp == 0) {
        if (lane == 0) {
            tma_prefetch_desc(&tmQ);
            tma_prefetch_desc(&tmK);
            bool ok = true, waited = false;
            while (ok && segments.next(args, s)) {
                const int bh = s.b * ta.kv_heads + s.hk, n = s.count();
                const float *item = ta.row_exponents + (size_t)bh * stats_stride(ta.rows);
                for (int r0 = 0; ok && r0 < ta.rows; r0 += kWeightRows) {
                    const int qb = q_buffer(q_loads);
                    if (!(ok = mbar_wait(&q_empty[qb], q_phase(q_loads) ^ 1, abort_flag, err, kErrWaitSmemEmpty))) break;
                    const int boxes = min(2, (ta.rows - r0 + 127) / 128), padded = min(kWeightRows, (ta.rows - r0 + 31) & ~31);
                    mbar_arrive_expect_tx(&q_full[qb], boxes * L::kTile + padded * 4);
                    for (int t = 0; t < boxes; ++t)
                        for (int c = 0; c < kDChunks; ++c)
                            tma_load_3d(smem + c * L::kRows64 + (qb + t) * 128 * 128, &tmQ, &q_full[qb], c * 64, r0 + t * 128, bh);
                    ++q_loads;
                    auto load = [&](int i) {
                        const int st = ring_loads % kStages;
                        if (!(ok = mbar_wait(&empty[st], (ring_loads / kStages & 1) ^ 1, abort_flag, err, kErrWaitSmemEmpty))) return;
                        mbar_arrive_expect_tx(&full[st], L::kTile);
                        for (int c = 0; c < kDChunks; ++c)
                            tma_load_3d(smem + L::kRing + st * L::kTile + c * 128 * 128, &tmK, &full[st], c * 64, (s.last - 1 - i) * kTileKeys, bh);
                        ++ring_loads;
                    };
                    int i = 0;
                    if (!waited) {  // the first tiles are under way before the rows' stats are there
                        for (; i < min(n, kStages); ++i) load(i);
                        grid_dependency_wait();
                        waited = true;
                    }
                    bulk_load(smem + L::kStats + qb * 128 * 4, item + r0, padded * 4, &q_full[qb]);
                    for (; ok && i < n; ++i) load(i);
                }
            }
            if (!waited) grid_dependency_wait();  // in every block: this grid's end stands for the one's before it
        }
    } else if (warp == 1) {
        auto wait = [&](uint64_t *bar, uint32_t parity, int code) {
            return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, err, code));
        };
        const uint64_t dq0 = sdesc_sw128(smem_u32(smem), 16, 1024), dk0 = sdesc_sw128(smem_u32(smem + L::kRing), 16, 1024);
        int pos = 0, qn = 0;
        bool ok = true;
        while (ok && segments.next(args, s))
            for (int r0 = 0; ok && r0 < ta.rows; r0 += kWeightRows) {
                const uint32_t idesc = idesc_f32acc(kFmt, kFmt, false, false, kTileKeys, min(kWeightRows, (ta.rows - r0 + 31) & ~31));
                const int qb = q_buffer(qn);
                ok = wait(&q_full[qb], q_phase(qn++), kErrWaitTmaFull);
                for (int i = s.first; ok && i < s.last; ++i, ++pos) {
                    const int st = pos % kStages, t = pos % buffers;
                    ok = wait(&full[st], pos / kStages & 1, kErrWaitTmaFull) && wait(&s_empty[t], (pos / buffers & 1) ^ 1, kErrWaitAccEmpty);
                    if (!ok) break;
                    tc_fence_after();
                    uint64_t a[DP / 16], b[DP / 16];
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k) {
                        a[k] = dk0 + ((st * L::kTile + (k >> 2) * 128 * 128 + (k & 3) * 32) >> 4);
                        b[k] = dq0 + (((k >> 2) * L::kRows64 + qb * 128 * 128 + (k & 3) * 32) >> 4);
                    }
                    umma_ss_group<DP / 16>(tmem + t * buffer_columns, a, b, idesc, 0);
                    umma_commit(&s_full[t]);
                    umma_commit(&empty[st]);
                }
                umma_commit(&q_empty[qb]);
            }
        umma_commit(mma_done);
        mbar_wait_drain(mma_done, 0, err);
    } else {
        const int group = (warp - 2) >> 2, quarter = warp & 3, key = quarter * 32 + lane;
        const float c = ta.scale_log2;
        const uint64_t c2 = pack2f(c, c);
        uint32_t *tree = reinterpret_cast<uint32_t *>(smem + L::kTree + (warp - 2) * kTreeBytes);
        int pos = 0, qn = 0;
        bool ok = true;
        while (ok && segments.next(args, s)) {
            float *weights = ta.weights + ((size_t)s.b * ta.kv_heads + s.hk) * ta.capacity;
            for (int r0 = 0; ok && r0 < ta.rows; r0 += kWeightRows) {
                const int qb = q_buffer(qn);
                if (s.last * kTileKeys > s.length && r0 == 0) {  // the segment reaches the drafts
                    __syncwarp();
                    for (int i = lane; i < ta.seq * ta.words; i += 32) tree[i] = __ldg(ta.tree + (size_t)s.b * ta.seq * ta.words + i);
                    __syncwarp();
                }
                ok = __all_sync(0xffffffffu, mbar_wait(&q_full[qb], q_phase(qn++), abort_flag, err, kErrWaitTmaFull));
                const float *stats = reinterpret_cast<const float *>(smem + L::kStats) + qb * 128;
                const int count = min(kWeightRows, ta.rows - r0);
                for (int i = s.last - 1; ok && i >= s.first; --i, ++pos) {
                    if ((pos & 1) != group) continue;
                    const int t = pos % buffers, j = i * kTileKeys + key, draft = j - s.length;
                    const uint32_t ts = tmem + t * buffer_columns + ((uint32_t)(quarter * 32) << 16);
                    const float old = draft < ta.seq ? weights[j] : 0.0f;
                    ok = __all_sync(0xffffffffu, mbar_wait(&s_full[t], pos / buffers & 1, abort_flag, err, kErrWaitScore));
                    if (!ok) break;
                    tc_fence_after();
                    float sum = 0.0f;
                    if (i * kTileKeys + kTileKeys <= s.length) {
                        // columns beyond the rows: their exponent is -inf, and the score is a product
                        // with zeros, but NaN if the key is infinite
                        uint64_t sums[2] = {0, 0};
                        float sv[32];
                        tmem_ld32f(ts, sv);
#pragma unroll 1
                        for (int n = 0; n < count; n += 32) {
                            tmem_wait_ld();
                            reg_fence(sv);
                            float e[32];
#pragma unroll
                            for (int k = 0; k < 32; ++k) e[k] = sv[k];
                            if (n + 32 < count) tmem_ld32f(ts + n + 32, sv);
                            if (n + 32 > count) {
#pragma unroll
                                for (int k = 0; k < 32; ++k)
                                    if (n + k >= count) e[k] = 0.0f;
                            }
#pragma unroll
                            for (int k = 0; k < 32; k += 4) {
                                const ulonglong2 x = *reinterpret_cast<const ulonglong2 *>(stats + n + k);
                                float a0, a1, b0, b1;
                                unpack2f(fma2(pack2f(e[k], e[k + 1]), c2, x.x), a0, a1);
                                unpack2f(fma2(pack2f(e[k + 2], e[k + 3]), c2, x.y), b0, b1);
                                sums[0] = add2(pack2f(mufu_exp2(a0), mufu_exp2(a1)), sums[0]);
                                sums[1] = add2(pack2f(mufu_exp2(b0), mufu_exp2(b1)), sums[1]);
                            }
                        }
                        float a0, a1;
                        unpack2f(add2(sums[0], sums[1]), a0, a1);
                        sum = a0 + a1;
                    } else {
                        // selected without branches: lanes lie on both sides of the first draft
                        const uint32_t *word = tree + (min(max(draft, 0), ta.seq - 1) >> 5);
                        const uint32_t always = draft < 0, drafted = draft >= 0 && draft < ta.seq;
                        int tok = r0 % ta.seq;
#pragma unroll 1
                        for (int n = 0; n < count; n += 16) {
                            uint32_t raw[16];
                            tmem_ld16(ts + n, raw);
                            tmem_wait_ld();
#pragma unroll
                            for (int k = 0; k < 16; ++k) {
                                const uint32_t sees = always | (word[tok * ta.words] >> (draft & 31) & drafted);
                                const float p = mufu_exp2(fmaf(__uint_as_float(raw[k]), c, stats[n + k]));
                                sum += sees && n + k < count ? p : 0.0f;
                                tok = tok + 1 == ta.seq ? 0 : tok + 1;
                            }
                        }
                    }
                    tc_fence_before();
                    mbar_arrive(&s_empty[t]);
                    if (draft < ta.seq) weights[j] = old + sum;
                }
                mbar_arrive(&q_empty[qb]);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        if (lane == 0 && *abort_flag) {
            for (int i = max(0, ring_loads - kStages); i < ring_loads; ++i) mbar_wait_drain(&full[i % kStages], i / kStages & 1, err);
            for (int i = max(0, q_loads - (narrow ? 2 : 1)); i < q_loads; ++i) mbar_wait_drain(&q_full[q_buffer(i)], q_phase(i), err);
        }
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ------------------------------------------------------------------ host side
using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                              const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encoder() {
    static EncodeFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] { fn = reinterpret_cast<EncodeFn>(driver_entry("cuTensorMapEncodeTiled")); });
    return fn;
}

// [heads, rows, dim] tensor, box {64, box_rows, 1}, 128-byte swizzle; elements beyond dim or rows read as 0.
bool row_map(CUtensorMap *map, CUtensorMapDataType dt, const void *ptr, uint64_t heads, uint64_t rows, uint64_t dim, uint32_t box_rows = 128) {
    const cuuint64_t dims[3] = {dim, rows, heads};
    const cuuint64_t strides[2] = {dim * 2, rows * dim * 2};
    const cuuint32_t box[3] = {64, box_rows, 1};
    const cuuint32_t estr[3] = {1, 1, 1};
    return encoder()(map, dt, 3, const_cast<void *>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DP, typename T, bool kTwoTiles, int kCopies>
LaunchFn tc_launch(Context *ctx, const Spec &s) {
    using L = Layout<DP, kTwoTiles, kCopies>;
    auto kernel = tree_tc_kernel<DP, T, kTwoTiles, kCopies>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::kSmem) != cudaSuccess)
        throw IrError("cannot reserve shared memory for the tcgen05 attention_tree");
    constexpr int kSlotRows = kTwoTiles ? 256 : 128;
    TcArgs base{};
    base.t = tree_args(ctx, s);
    const uint64_t heads = (uint64_t)s.batch * s.kv_heads, capacity = s.capacity, dim = s.dim, rows = base.t.rows;
    base.row_blocks = (int)((rows + kSlotRows - 1) / kSlotRows);
    // one CTA per SM, none for which even full caches have no tile
    const unsigned __int128 most = (unsigned __int128)heads * base.row_blocks * ((capacity + kTileKeys - 1) / kTileKeys);
    base.ctas = most < (unsigned __int128)ctx->sm_count ? (int)most : ctx->sm_count;
    base.boundary = boundary_tiles((int)rows);
    base.slot_rows = rows >= (uint64_t)kSlotRows ? kSlotRows : (int)((rows + 7) / 8 * 8);
    // an item's parts: the CTAs over the items; from about 8 on a thread's are too many
    const bool spread = heads * base.row_blocks * 8 <= (uint64_t)base.ctas;
    constexpr int kWays = 8;
    const int each = spread ? kJoinThreads / kWays : kJoinThreads, item_blocks = (base.slot_rows * (DP / 4) + each - 1) / each;
    const long long join_blocks = (long long)heads * base.row_blocks * item_blocks;
    if (join_blocks > INT_MAX) throw IrError("attention_tree too large for one launch");
    const bool weights = s.weights;
    const size_t stats = (heads * stats_stride((int)rows) * sizeof(float) + 255) / 256 * 256, slots = (size_t)base.ctas * 2 * base.slot_rows;
    auto ws = kernel_workspace(stats + slots * (sizeof(float2) + DP * sizeof(float)), "attention_tree partial results");
    base.t.row_exponents = weights ? static_cast<float *>(ws.get()) : nullptr;
    base.t.part_o = reinterpret_cast<float *>(static_cast<char *>(ws.get()) + stats);
    base.t.part_ml = reinterpret_cast<float2 *>(base.t.part_o + slots * DP);
    const CUtensorMapDataType dt = std::is_same<T, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    auto weights_kernel = tree_weights_tc<DP, T>;
    using W = WeightsLayout<DP>;
    if (weights && cudaFuncSetAttribute(weights_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)W::kSmem) != cudaSuccess)
        throw IrError("cannot reserve shared memory for the tcgen05 attention_tree");
    return [=, keep = ws](cudaStream_t st, void **b) {
        TcArgs a = base;
        a.t = tree_bind(base.t, b, weights);
        CUtensorMap mq, mqw, mk, mv;  // mqw: Q for the weights' pass
        if (!row_map(&mq, dt, b[0], heads, rows, dim, 128 / kCopies) || !row_map(&mqw, dt, b[0], heads, rows, dim) || !row_map(&mk, dt, b[1], heads, capacity, dim) || !row_map(&mv, dt, b[2], heads, capacity, dim))
            return cudaErrorInvalidValue;
        kernel<<<a.ctas, kThreads, L::kSmem, st>>>(mq, mk, mv, a);
        cudaError_t e = launch_after(st, spread ? tree_join_tc<DP, T, kWays> : tree_join_tc<DP, T, 1>, (int)join_blocks, kJoinThreads, 0, a, item_blocks);
        if (weights && e == cudaSuccess) {
            TcArgs w = a;
            w.row_blocks = 1, w.boundary = kWeightsBoundary;
            e = launch_after(st, weights_kernel, a.ctas, kThreads, W::kSmem, mqw, mk, w);
        }
        return e == cudaSuccess ? cudaGetLastError() : e;
    };
}

}  // namespace

LaunchFn make_attention_tree_tc(Context *ctx, const Spec &s) {
    if (!encoder()) throw IrError("cuTensorMapEncodeTiled unavailable");
    const uint64_t rows = (uint64_t)s.heads / s.kv_heads * s.seq;
    auto shape = [&](auto type, auto width) -> LaunchFn {
        using T = decltype(type);
        constexpr int DP = decltype(width)::value;
        if (rows > kTileRows) return tc_launch<DP, T, true, 1>(ctx, s);
        return rows > 64 ? tc_launch<DP, T, false, 1>(ctx, s) : rows > 32 ? tc_launch<DP, T, false, 2>(ctx, s) : tc_launch<DP, T, false, 4>(ctx, s);
    };
    auto pick = [&](auto type) {
        return s.dim > 64 ? shape(type, std::integral_constant<int, 128>{}) : shape(type, std::integral_constant<int, 64>{});
    };
    return s.dtype == DType::BF16 ? pick(__nv_bfloat16{}) : pick(__half{});
}

}  // namespace jade
