// attention_tree: the newest tokens of each sequence (one, or a tree of drafted
// ones) attend to the sequence's cache.
//
//   q [batch, heads, seq, dim], k, v [batch, kv_heads, capacity, dim], heads =
//   group * kv_heads; token t of sequence b sees slots j < lengths[b] and, of the
//   drafted tokens in slots lengths[b] + i, those whose bit i of tree[b, t] is set.
//   out[b, t, h] = sum_j p_j v_j,  p = softmax_j(q k_j / sqrt(dim)) over what it sees
//   (0 where it sees nothing); weights[b, hk, j] += sum of p_j over the group's heads
//   and the tokens (with drafts_only: those that see a draft, as every token sees itself;
//   a place of a step that holds no token has no bits and leaves no weight).
//
// The group's heads and tokens of a (sequence, kv head) are M = group * seq rows of q
// that lie together and share its keys. Keys are split over blocks; each split keeps
// a running maximum m and sum l per row (FP32) and an unnormalised FP32 sum of
// e^(s - m) v, and the splits are joined by rescaling to the common maximum in split
// order, so results do not depend on timing. Entries that a row does not see are
// never multiplied (a NaN or infinity there cannot reach the row), nor is anything in slots
// from lengths[b] + seq on (the tcgen05 form's last tile loads what lies there and masks it).
// Entries that a row does see count as they are: a NaN, or a score of +inf, makes the row
// NaN, a score of -inf weighs nothing, an infinity in v reaches its column.
//
// This file: FP32, and 16-bit types with dim above 128, on FFMA; weights; dispatch.
// attention_tree_tc.cu: 16-bit types with dim up to 128, on tcgen05.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "attention_softmax.cuh"
#include "attention_tree.cuh"

namespace jade {
namespace {

constexpr int kMaxSplits = 64;
constexpr float kRescaleThreshold = 8.0f;  // log2 units

__device__ __forceinline__ bool sees(const TreeArgs &a, int b, int row, int j, int length) {
    if (j < length) return true;
    const int i = j - length;
    if (i >= a.seq || row >= a.rows) return false;
    return a.tree[((size_t)b * a.seq + row % a.seq) * a.words + (i >> 5)] >> (i & 31) & 1;
}

// A block of four warps: K and V tiles of a split's keys, each a contiguous run of the
// cache, come by bulk copies through a ring. Warps take row groups
// of four rows, in registers with their sums, and a group's warps share the tile's keys.
// kLanes lanes hold a key's elements (four at 4 lane + 4 kLanes i), so a warp works on
// 32 / kLanes keys at once and on kSets times twice as many an iteration (more of them hide
// more latency: 64 rows below 153 us with one set, 137 with two, 129 with four): a set's 4
// rows x 2 keys of scores per lane are summed by halving exchanges (7 shuffles, not 24) that leave each lane one
// score, whose exponential it forms alone and hands back to the others. Maxima and sums
// are per lane group and joined at the end; sums are rescaled only when a maximum grows
// by more than 2^8. K and V cross shared memory once per row group.
// Bound by HBM for a few rows, else by FFMA issue beside shuffles and shared-memory reads.
// Measured on B200, FP32, dim 128: 64 heads of 1,000 to 8,000 keys, 4 rows (295 MB), 62 us
// with the join = 4.8 TB/s; 32 heads of 1,000 to 4,000, 4 / 16 / 64 rows: 26 / 42 / 129 us;
// 16 heads of up to 4,000, 512 rows, 378 us = 27 TFLOP/s. No fifth warp for the copies: it
// would cap the others at 168 registers, and the spills cost more (16 rows, one set: 62 us
// for 49).
constexpr int kStreamWarps = 4, kStreamThreads = 32 * kStreamWarps, kStreamStages = 3, kGroupRows = 4;
constexpr int kStreamPad = 1024;  // behind the ring: the last V row is read up to the lanes' width

struct Four {  // four elements as packed FP32 pairs
    uint64_t lo, hi;
};
__device__ __forceinline__ Four four_of(const float *p) {
    const ulonglong2 u = *reinterpret_cast<const ulonglong2 *>(p);
    return {u.x, u.y};
}
__device__ __forceinline__ Four four_of(const __nv_bfloat16 *p) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    return {pack2f(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u)), pack2f(__uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u))};
}
__device__ __forceinline__ Four four_of(const __half *p) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&u.x)), y = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
    return {pack2f(x.x, x.y), pack2f(y.x, y.y)};
}

// The pieces of a head that a lane holds, four elements each. kAll: as they lie there,
// else zeros beyond the head.
template <bool kAll, int kLanes, int kPieces, typename T>
__device__ __forceinline__ void load_pieces(uint64_t (&x)[2 * kPieces], const T *p, int c, int dim) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        Four f{0, 0};
        if (kAll || 4 * (c + kLanes * i) < dim) f = four_of(p + 4 * (c + kLanes * i));
        x[2 * i] = f.lo, x[2 * i + 1] = f.hi;
    }
}
template <int kPairs>
__device__ __forceinline__ float dot(const uint64_t (&x)[kPairs], const uint64_t (&y)[kPairs]) {
    uint64_t s = mul2(x[0], y[0]);
#pragma unroll
    for (int i = 1; i < kPairs; ++i) s = fma2(x[i], y[i], s);
    float lo, hi;
    unpack2f(s, lo, hi);
    return lo + hi;
}
// Sums eight values over kLanes lanes; lane c gets the total of value c * 8 / kLanes.
template <int kLanes>
__device__ __forceinline__ float scattered_sum(float (&v)[8], int c) {
    int o = kLanes / 2;
#pragma unroll
    for (int n = 4; n > 0; n >>= 1, o >>= 1) {
        const bool up = c & o;
#pragma unroll
        for (int i = 0; i < n; ++i) v[i] = (up ? v[i + n] : v[i]) + __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + n], o);
    }
#pragma unroll
    for (; o > 0; o >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    return v[0];
}

// grid: (row blocks of `groups` row groups, splits, batch * kv_heads)
template <typename T, int kLanes, int kPieces, bool kWhole, int kSets>
__global__ void __launch_bounds__(kStreamThreads, 2) tree_stream_kernel(const TreeArgs a, int splits, int groups, int tile_keys) {
    constexpr int kKeys = 32 / kLanes, kSame = kLanes / 8;  // keys at once; lanes that get the same score
    extern __shared__ __align__(128) uint8_t ring_smem[];
    __shared__ uint64_t full[kStreamStages], empty[kStreamStages];
    __shared__ int aborted;
    volatile int *abort_flag = &aborted;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, bh = blockIdx.z, b = bh / a.kv_heads;
    const int length = a.lengths[b];
    if (length < 0 || length > a.capacity - a.seq) {
        if (threadIdx.x == 0) atomicCAS(a.err, 0, kErrCacheLength);
        return;
    }
    grid_dependency_trigger();
    const int key_warps = kStreamWarps / groups, active = key_warps * groups;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStreamStages; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], active);
        aborted = 0;
        fence_barrier_init();
        fence_proxy_async();
    }
    __syncthreads();
    const int n = length + a.seq, tiles = (n + tile_keys - 1) / tile_keys;
    const int t0 = (int)((long long)tiles * blockIdx.y / splits), t1 = (int)((long long)tiles * (blockIdx.y + 1) / splits);
    const size_t base = (size_t)bh * a.capacity * a.dim;
    const uint32_t tile = (uint32_t)tile_keys * a.dim;  // elements
    T *ring = reinterpret_cast<T *>(ring_smem);
    int loads = 0;

    const int g = lane / kLanes, c = lane % kLanes, group = warp % groups, kw = warp / groups;
    const int row0 = (blockIdx.x * groups + group) * kGroupRows;
    const int mine = c / kSame, my_row = row0 + (mine >> 1), my_key = (mine & 1) * kKeys + g;  // of this lane's score
    uint64_t o[kGroupRows][2 * kPieces];
    float m = -INFINITY, l = 0.0f;
    // Thread 0 issues the copies; a stage is refilled one tile after it was read, when the
    // other warps have read it too.
    auto load = [&] {
        const int st = loads % kStreamStages, j0 = (t0 + loads) * tile_keys;
        if (!mbar_wait(&empty[st], (loads / kStreamStages & 1) ^ 1, abort_flag, a.err, kErrWaitSmemEmpty)) return;
        const uint32_t bytes = (uint32_t)min(tile_keys, n - j0) * a.dim * sizeof(T);
        mbar_arrive_expect_tx(&full[st], 2 * bytes);
        bulk_load(ring + 2 * st * tile, static_cast<const T *>(a.k) + base + (size_t)j0 * a.dim, bytes, &full[st]);
        bulk_load(ring + (2 * st + 1) * tile, static_cast<const T *>(a.v) + base + (size_t)j0 * a.dim, bytes, &full[st]);
        ++loads;
    };
    if (threadIdx.x == 0)
        while (loads < min(kStreamStages, t1 - t0)) load();
    if (warp < active) {
        uint64_t q[kGroupRows][2 * kPieces];
#pragma unroll
        for (int r = 0; r < kGroupRows; ++r) {
#pragma unroll
            for (int i = 0; i < 2 * kPieces; ++i) q[r][i] = o[r][i] = 0;
            if (row0 + r < a.rows) load_pieces<kWhole, kLanes, kPieces>(q[r], static_cast<const T *>(a.q) + ((size_t)bh * a.rows + row0 + r) * a.dim, c, a.dim);
        }
        const float threshold = kRescaleThreshold / a.scale_log2;
        auto pass = [&](const T *k, const T *v, int j0, int count, auto careful) {
#pragma unroll 1
            for (int k0 = kw * 2 * kSets * kKeys; k0 < count; k0 += key_warps * 2 * kSets * kKeys) {
                float s8[kSets][8], p[kSets], top = -INFINITY;
#pragma unroll
                for (int u = 0; u < 2 * kSets; ++u) {
                    uint64_t x[2 * kPieces];
                    load_pieces<kWhole, kLanes, kPieces>(x, k + (k0 + u * kKeys + g) * a.dim, c, a.dim);
#pragma unroll
                    for (int r = 0; r < kGroupRows; ++r) s8[u / 2][2 * r + u % 2] = dot(q[r], x);
                }
#pragma unroll
                for (int h = 0; h < kSets; ++h) {
                    const int key = k0 + 2 * h * kKeys + my_key;
                    p[h] = scattered_sum<kLanes>(s8[h], c);
                    if (careful) p[h] = key < count && sees(a, b, my_row, j0 + key, length) ? p[h] : -INFINITY;
                    top = fmaxf(top, p[h]);
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, kSame));
                if (__any_sync(0xffffffffu, top > m + threshold)) {
                    const float m_new = fmaxf(m, top), alpha = exp2f((m - (m_new == -INFINITY ? 0.0f : m_new)) * a.scale_log2);
                    m = m_new;
                    l *= alpha;
#pragma unroll
                    for (int r = 0; r < kGroupRows; ++r) {
                        const float f = __shfl_sync(0xffffffffu, alpha, g * kLanes + 2 * r * kSame);
#pragma unroll
                        for (int i = 0; i < 2 * kPieces; ++i) o[r][i] = mul2(o[r][i], pack2f(f, f));
                    }
                }
#pragma unroll
                for (int h = 0; h < kSets; ++h) {
                    p[h] = exp2f((p[h] - (m == -INFINITY ? 0.0f : m)) * a.scale_log2);
                    l += p[h];
                }
#pragma unroll
                for (int u = 0; u < 2 * kSets; ++u) {
                    uint64_t x[2 * kPieces];
                    load_pieces<true, kLanes, kPieces>(x, v + (k0 + u * kKeys + g) * a.dim, c, a.dim);  // columns beyond the head are not written
#pragma unroll
                    for (int r = 0; r < kGroupRows; ++r) {
                        const float w = __shfl_sync(0xffffffffu, p[u / 2], g * kLanes + (2 * r + u % 2) * kSame);
                        if (!careful || w != 0.0f)  // drafts: no product with one that the row does not see
#pragma unroll
                            for (int i = 0; i < 2 * kPieces; ++i) o[r][i] = fma2(pack2f(w, w), x[i], o[r][i]);
                    }
                }
            }
        };
        for (int t = t0; t < t1; ++t) {
            const int i = t - t0, st = i % kStreamStages, j0 = t * tile_keys, count = min(tile_keys, n - j0);
            if (threadIdx.x == 0 && i > 0 && t0 + loads < t1) load();
            if (!mbar_wait_warp(&full[st], i / kStreamStages & 1, abort_flag, a.err, kErrWaitTmaFull)) break;
            const T *k = ring + 2 * st * tile, *v = k + tile;
            if (j0 + tile_keys <= length) pass(k, v, j0, count, std::false_type{});
            else pass(k, v, j0, count, std::true_type{});
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
        }
        // the lane groups' maxima and sums, then the scores' of the two keys
#pragma unroll
        for (int x = kLanes; x < 32; x <<= 1) {
            const float m_new = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x)), alpha = exp2f((m - (m_new == -INFINITY ? 0.0f : m_new)) * a.scale_log2);
            m = m_new;
            l *= alpha;
            l += __shfl_xor_sync(0xffffffffu, l, x);
#pragma unroll
            for (int r = 0; r < kGroupRows; ++r) {
                const float f = __shfl_sync(0xffffffffu, alpha, g * kLanes + 2 * r * kSame);
#pragma unroll
                for (int i = 0; i < 2 * kPieces; ++i) {
                    o[r][i] = mul2(o[r][i], pack2f(f, f));
                    o[r][i] = add2(o[r][i], __shfl_xor_sync(0xffffffffu, o[r][i], x));
                }
            }
        }
        l += __shfl_xor_sync(0xffffffffu, l, kSame);
    }
    __syncthreads();  // the ring has been read
    if (aborted) {
        if (threadIdx.x == 0)  // copies still in flight land before the block exits
            for (int i = max(0, loads - kStreamStages); i < loads; ++i) mbar_wait_drain(&full[i % kStreamStages], i / kStreamStages & 1, a.err);
        return;
    }
    // the key warps of a row group, in order: [warp][row][width] sums, [warp][row] maxima and sums
    constexpr int kWidth = 4 * kLanes * kPieces;
    float *sums = reinterpret_cast<float *>(ring_smem);
    float2 *stats = reinterpret_cast<float2 *>(sums + kStreamWarps * kGroupRows * kWidth);
    if (warp < active) {
#pragma unroll
        for (int r = 0; r < kGroupRows; ++r)
            if (g == r % kKeys) {
                if (c == 2 * r * kSame) stats[warp * kGroupRows + r] = make_float2(m, l);
#pragma unroll
                for (int i = 0; i < kPieces; ++i)
                    *reinterpret_cast<ulonglong2 *>(sums + (warp * kGroupRows + r) * kWidth + 4 * (c + kLanes * i)) = make_ulonglong2(o[r][2 * i], o[r][2 * i + 1]);
            }
    }
    __syncthreads();
    const int quads = a.dim / 4, block_rows = min(groups * kGroupRows, a.rows - (int)blockIdx.x * groups * kGroupRows);
    for (int i = threadIdx.x; i < block_rows * quads; i += kStreamThreads) {
        const int r = i / quads, d = 4 * (i - r * quads);
        float top = -INFINITY, sum = 0.0f;
        for (int w = 0; w < key_warps; ++w) top = fmaxf(top, stats[w * groups * kGroupRows + r].x);
        const float shift = top == -INFINITY ? 0.0f : top;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < key_warps; ++w) {
            const float2 st = stats[w * groups * kGroupRows + r];
            const float f = exp2f((st.x - shift) * a.scale_log2);
            const float4 y = *reinterpret_cast<const float4 *>(sums + (w * groups * kGroupRows + r) * kWidth + d);
            sum += st.y * f;
            x.x += y.x * f, x.y += y.y * f, x.z += y.z * f, x.w += y.w * f;
        }
        const size_t out = ((size_t)bh * a.rows + blockIdx.x * groups * kGroupRows + r) * splits + blockIdx.y;
        if (d == 0) a.part_ml[out] = make_float2(top, sum);
        *reinterpret_cast<float4 *>(a.part_o + out * a.dim + d) = x;
    }
}

// Joins the splits of one row: one warp a row.
template <typename T>
__device__ __forceinline__ void join_rows(const TreeArgs &a, int splits, int total_rows, int block) {
    const int row = block * (int)(blockDim.x >> 5) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row >= total_rows) return;
    const int bh = row / a.rows, rr = row - bh * a.rows, b = bh / a.kv_heads, hk = bh - b * a.kv_heads;
    if (a.lengths[b] < 0 || a.lengths[b] > a.capacity - a.seq) return;
    // lane s holds splits s and s + 32 (at most kMaxSplits)
    const float2 *ml = a.part_ml + (size_t)row * splits;
    const float2 none = make_float2(-INFINITY, 0.0f);
    const float2 u = lane < splits ? ml[lane] : none, v = lane + 32 < splits ? ml[lane + 32] : none;
    float m = fmaxf(u.x, v.x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float shift = m == -INFINITY ? 0.0f : m;
    const float wu = exp2f((u.x - shift) * a.scale_log2), wv = exp2f((v.x - shift) * a.scale_log2);
    float l = u.y * wu + v.y * wv;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    const int g = rr / a.seq, t = rr - g * a.seq;
    T *out = static_cast<T *>(a.out) + (((size_t)b * a.seq + t) * a.kv_heads * a.group + hk * a.group + g) * a.dim;
    for (int d0 = 0; d0 < a.dim; d0 += 128) {
        const int d = d0 + lane * 4;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int s = 0; s < splits; ++s) {
            const float w = __shfl_sync(0xffffffffu, s < 32 ? wu : wv, s & 31);
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
            if (d < a.dim) y = *reinterpret_cast<const float4 *>(a.part_o + ((size_t)row * splits + s) * a.dim + d);
            if (w != 0.0f) x.x = fmaf(w, y.x, x.x), x.y = fmaf(w, y.y, x.y), x.z = fmaf(w, y.z, x.z), x.w = fmaf(w, y.w, x.w);
        }
        if (d < a.dim)
            out[d] = from_f32<T>(x.x * inv), out[d + 1] = from_f32<T>(x.y * inv), out[d + 2] = from_f32<T>(x.z * inv), out[d + 3] = from_f32<T>(x.w * inv);
    }
}

// weights[j] += sum over all rows of p_j, p from the rows' joined maximum and sum. A block
// takes the rows 32 at a time from shared memory; a warp holds four keys a lane group in
// registers and adds their sums in row order.
constexpr int kWeightRows = 32;

template <typename T, int kLanes, int kPieces>
__device__ __forceinline__ void add_weights(const TreeArgs &a, int splits, int first, int step, int bh) {
    constexpr int kKeys = 32 / kLanes, kSame = kLanes / 8, kWidth = 4 * kLanes * kPieces, kUnit = 4 * kKeys;
    __shared__ __align__(16) float q[kWeightRows * kWidth];
    __shared__ float2 stats[kWeightRows];  // maximum (0 if the row sees nothing), 1 / sum
    const int b = bh / a.kv_heads, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane / kLanes, c = lane % kLanes, mine = c / kSame;
    const int length = a.lengths[b], n = length + a.seq;
    if (length < 0 || length > a.capacity - a.seq) return grid_dependency_wait();
    const T *k = static_cast<const T *>(a.k) + (size_t)bh * a.capacity * a.dim, *queries = static_cast<const T *>(a.q) + (size_t)bh * a.rows * a.dim;
    auto stage_rows = [&](int r0) {
        for (int i = threadIdx.x; i < kWeightRows * kWidth / 4; i += kStreamThreads) {
            const int r = i / (kWidth / 4), d = 4 * (i % (kWidth / 4));
            Four f{0, 0};
            if (r0 + r < a.rows && d < a.dim) f = four_of(queries + (size_t)(r0 + r) * a.dim + d);
            *reinterpret_cast<ulonglong2 *>(q + 4 * i) = make_ulonglong2(f.lo, f.hi);
        }
    };
    auto stage_stats = [&](int r0) {  // four threads a row
        const int row = min(r0 + (int)(threadIdx.x >> 2), a.rows - 1), part = threadIdx.x & 3;
        const float2 *ml = a.part_ml + ((size_t)bh * a.rows + row) * splits;
        float m = -INFINITY, l = 0.0f;
        for (int s = part; s < splits; s += 4) m = fmaxf(m, ml[s].x);
#pragma unroll
        for (int x = 1; x < 4; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
        const float shift = m == -INFINITY ? 0.0f : m;
        for (int s = part; s < splits; s += 4) l = fmaf(ml[s].y, exp2f((ml[s].x - shift) * a.scale_log2), l);
#pragma unroll
        for (int x = 1; x < 4; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
        if (part == 0) stats[threadIdx.x >> 2] = make_float2(shift, adds_weight(a, b, row) && (l > 0.0f || l != l) ? 1.0f / l : 0.0f);
    };
    uint64_t x[4][2 * kPieces];
    auto load_keys = [&](int block) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
            load_pieces<false, kLanes, kPieces>(x[u], k + (size_t)min((block * kStreamWarps + warp) * kUnit + u * kKeys + g, n - 1) * a.dim, c, a.dim);
    };
    // the first keys and rows do not depend on the splits
    load_keys(first);
    stage_rows(0);
    grid_dependency_wait();
    stage_stats(0);
    __syncthreads();
    bool staged = true;  // rows 0 ..
    for (int block = first; block * kStreamWarps * kUnit < n; block += step) {
        const int key0 = (block * kStreamWarps + warp) * kUnit + (mine & 1) * kKeys + g;  // of this lane's first score, the second 2 kKeys on
        if (block != first) load_keys(block);
        float acc[2] = {};
        for (int r0 = 0; r0 < a.rows; r0 += kWeightRows) {
            if (!staged) {
                __syncthreads();
                stage_rows(r0);
                stage_stats(r0);
                __syncthreads();
            }
            staged = a.rows <= kWeightRows;
            const int rows = min(kWeightRows, a.rows - r0);
#pragma unroll 1
            for (int r = 0; r < rows; r += kGroupRows) {
                float s8[2][8];
#pragma unroll
                for (int i = 0; i < kGroupRows; ++i) {
                    uint64_t y[2 * kPieces];
                    load_pieces<true, kLanes, kPieces>(y, q + (r + i) * kWidth, c, kWidth);
#pragma unroll
                    for (int u = 0; u < 4; ++u) s8[u >> 1][2 * i + (u & 1)] = dot(y, x[u]);
                }
                const int row = r + (mine >> 1);
                const float2 st = stats[row];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float s = scattered_sum<kLanes>(s8[h], c);
                    const int key = key0 + 2 * h * kKeys;
                    if (row < rows && key < n && sees(a, b, r0 + row, key, length)) acc[h] += exp2f((s - st.x) * a.scale_log2) * st.y;
                }
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            acc[h] += __shfl_xor_sync(0xffffffffu, acc[h], 2 * kSame);
            acc[h] += __shfl_xor_sync(0xffffffffu, acc[h], 4 * kSame);
            const int key = key0 + 2 * h * kKeys;
            if (mine < 2 && c % kSame == 0 && key < n) a.weights[(size_t)bh * a.capacity + key] += acc[h];
        }
    }
}

// Behind the splits: the first join_blocks blocks join rows, the others add weights
// (which read the splits' maxima and sums themselves, so neither waits for the other).
template <typename T, int kLanes, int kPieces>
__global__ void __launch_bounds__(kStreamThreads) tree_finish_kernel(const TreeArgs a, int splits, int total_rows, int join_blocks, int key_blocks) {
    if ((int)blockIdx.x < join_blocks) {
        grid_dependency_wait();
        return join_rows<T>(a, splits, total_rows, blockIdx.x);
    }
    const int i = blockIdx.x - join_blocks, bh = i / key_blocks;
    add_weights<T, kLanes, kPieces>(a, splits, i - bh * key_blocks, key_blocks, bh);
}

// The kernels of a head dimension (16-bit types come here above 128 only).
template <typename T, int kSets>
auto kernel_of(int dim) -> void (*)(TreeArgs, int, int, int) {
    if constexpr (std::is_same<T, float>::value) {
        if (dim <= 64) return dim == 64 ? tree_stream_kernel<T, 8, 2, true, kSets> : tree_stream_kernel<T, 8, 2, false, kSets>;
        if (dim <= 128) return dim == 128 ? tree_stream_kernel<T, 8, 4, true, kSets> : tree_stream_kernel<T, 8, 4, false, kSets>;
    }
    return dim == 256 ? tree_stream_kernel<T, 16, 4, true, kSets> : tree_stream_kernel<T, 16, 4, false, kSets>;
}
template <typename T>
auto finish_of(int dim) -> void (*)(TreeArgs, int, int, int, int) {
    if constexpr (std::is_same<T, float>::value)
        if (dim <= 128) return dim <= 64 ? tree_finish_kernel<T, 8, 2> : tree_finish_kernel<T, 8, 4>;
    return tree_finish_kernel<T, 16, 4>;
}

template <typename T>
LaunchFn simt_launch(Context *ctx, const Spec &s) {
    TreeArgs base = tree_args(ctx, s);
    const int heads = (int)(s.batch * s.kv_heads), rows = base.rows, total_rows = heads * rows;
    if (heads > 65535) throw IrError("attention_tree: batch * kv_heads must be at most 65535");
    // blocks of up to four row groups, dealt evenly; tiles of 32 KB of K and V
    const int row_groups = (rows + kGroupRows - 1) / kGroupRows, row_blocks = (row_groups + kStreamWarps - 1) / kStreamWarps;
    const int groups = (row_groups + row_blocks - 1) / row_blocks, tile_keys = s.dim * sizeof(T) <= 512 ? 32 : 16;
    // four blocks per SM at most, two whole waves. Fewer and longer ones leave mixed lengths
    // unbalanced (64 heads of 1,000 to 8,000 keys: 62 us with four per SM, 74 with two, 69
    // with six), more cost partial results.
    const long long items = (long long)heads * row_blocks;
    const int splits = (int)std::max<long long>(1, std::min<long long>({4ll * ctx->sm_count / items, ((long long)s.capacity + tile_keys - 1) / tile_keys, (long long)kMaxSplits}));
    const size_t parts = (size_t)total_rows * splits;
    auto ws = kernel_workspace(parts * (s.dim * sizeof(float) + sizeof(float2)), "attention_tree partial results");
    base.part_o = static_cast<float *>(ws.get());  // rows of a multiple of 32 bytes: read as 16-byte vectors
    base.part_ml = reinterpret_cast<float2 *>(base.part_o + parts * s.dim);
    const int width = s.dim <= 64 ? 64 : s.dim <= 128 ? 128 : 256;
    const size_t joined = kStreamWarps * kGroupRows * (width * sizeof(float) + sizeof(float2));
    const size_t smem = std::max(2 * kStreamStages * tile_keys * s.dim * sizeof(T) + kStreamPad, joined);
    // key sets of an iteration: as many as give each of a row group's warps keys of every tile
    const auto kernel = groups > 2 ? kernel_of<T, 4>(s.dim) : groups > 1 ? kernel_of<T, 2>(s.dim) : kernel_of<T, 1>(s.dim);
    const auto finish = finish_of<T>(s.dim);
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        throw IrError("cannot reserve shared memory for attention_tree");
    const bool weights = s.weights;
    const int unit = width > 128 ? 32 : 64;  // keys of a block of the weights' pass
    const int key_blocks = (int)std::min<long long>((s.capacity + unit - 1) / unit, std::max<long long>(1, 8ll * ctx->sm_count / heads));
    const int join_blocks = (total_rows + kStreamWarps - 1) / kStreamWarps;
    return [=, keep = ws](cudaStream_t st, void **b) {
        const TreeArgs a = tree_bind(base, b, weights);
        kernel<<<dim3(row_blocks, splits, heads), kStreamThreads, smem, st>>>(a, splits, groups, tile_keys);
        const cudaError_t e = launch_after(st, finish, dim3(join_blocks + (weights ? key_blocks * heads : 0)), kStreamThreads, 0, a, splits, total_rows,
                                           join_blocks, key_blocks);
        return e == cudaSuccess ? cudaGetLastError() : e;
    };
}

}  // namespace

LaunchFn make_attention_tree(Context *ctx, const Spec &s, std::string &impl, std::string &path) {
    if (s.dtype != DType::F32 && s.dim <= 128) {
        impl = std::string("attention_tree_tcgen05_d") + std::to_string(s.dim) + "_" + dtype_name(s.dtype);
        path = "tcgen05";
        return make_attention_tree_tc(ctx, s);
    }
    impl = std::string("attention_tree_simt_d") + std::to_string(s.dim) + "_" + dtype_name(s.dtype);
    path = "simt";
    if (s.dtype == DType::BF16) return simt_launch<__nv_bfloat16>(ctx, s);
    return s.dtype == DType::F16 ? simt_launch<__half>(ctx, s) : simt_launch<float>(ctx, s);
}

}  // namespace jade
