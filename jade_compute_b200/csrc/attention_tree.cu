// attention_tree: the newest tokens of each sequence (one, or a tree of drafted
// ones) attend to the sequence's cache.
//
//   q [batch, heads, seq, dim], k, v [batch, kv_heads, capacity, dim], heads =
//   group * kv_heads; token t of sequence b sees slots j < lengths[b] and, of the
//   drafted tokens in slots lengths[b] + i, those whose bit i of tree[b, t] is set.
//   out[b, t, h] = sum_j p_j v_j,  p = softmax_j(q k_j / sqrt(dim)) over what it sees
//   (0 where it sees nothing); weights[b, hk, j] += sum of p_j over the group's heads
//   and the tokens.
//
// The group's heads and tokens of a (sequence, kv head) are M = group * seq rows of q
// that lie together and share its keys. Keys are split over blocks; each split keeps
// a running maximum m and sum l per row (FP32) and an unnormalised FP32 sum of
// e^(s - m) v, and the splits are joined by rescaling to the common maximum in split
// order, so results do not depend on timing. Entries that a row does not see are
// never multiplied (a NaN or infinity there cannot reach the row), slots from
// lengths[b] + seq on are not read.
//
// This file: FP32, and 16-bit types with dim above 128, on FFMA; weights; dispatch.
// attention_tree_tc.cu: 16-bit types with dim up to 128, on tcgen05.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "attention_tree.cuh"

namespace jade {
namespace {

constexpr int kThreads = 128, kRows = 16, kKeys = 32;  // a block: 16 rows of q, tiles of 32 keys
constexpr int kMaxSplits = 64;

template <typename T>
__device__ __forceinline__ float4 load4(const T *p);
template <>
__device__ __forceinline__ float4 load4<float>(const float *p) { return __ldg(reinterpret_cast<const float4 *>(p)); }
template <>
__device__ __forceinline__ float4 load4<__nv_bfloat16>(const __nv_bfloat16 *p) {
    const uint2 u = __ldg(reinterpret_cast<const uint2 *>(p));
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&u.x)), b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&u.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
template <>
__device__ __forceinline__ float4 load4<__half>(const __half *p) {
    const uint2 u = __ldg(reinterpret_cast<const uint2 *>(p));
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&u.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
    return make_float4(a.x, a.y, b.x, b.y);
}

__host__ __device__ constexpr int q_stride(int dim) { return dim + 4; }  // rows 4 banks apart

// Rows of q or keys (zeros from `limit` on) as FP32 into shared memory: 8 threads a
// row, 16 rows at a time, the loads of all of a thread's rows under way together.
template <typename T, int kCount>
__device__ __forceinline__ void stage(float *dst, const T *src, int first, int limit, int dim) {
    const int r = threadIdx.x >> 3;
    for (int c = (threadIdx.x & 7) * 4; c < dim; c += 32) {
        float4 x[kCount / 16];
#pragma unroll
        for (int i = 0; i < kCount / 16; ++i) {
            x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (first + r + 16 * i < limit) x[i] = load4(src + (size_t)(first + r + 16 * i) * dim + c);
        }
#pragma unroll
        for (int i = 0; i < kCount / 16; ++i) *reinterpret_cast<float4 *>(dst + (r + 16 * i) * q_stride(dim) + c) = x[i];
    }
}

// Scores of row r with keys c, c + 8, c + 16, c + 24 of the tile.
__device__ __forceinline__ void tile_scores(const float *q, const float *k, int r, int c, int dim, float (&s)[4]) {
#pragma unroll
    for (int u = 0; u < 4; ++u) s[u] = 0.0f;
    for (int d = 0; d < dim; d += 4) {
        const float4 a = *reinterpret_cast<const float4 *>(q + r * q_stride(dim) + d);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float4 b = *reinterpret_cast<const float4 *>(k + (c + 8 * u) * q_stride(dim) + d);
            s[u] = fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, fmaf(a.w, b.w, s[u]))));
        }
    }
}

__device__ __forceinline__ bool sees(const TreeArgs &a, int b, int row, int j, int length) {
    if (j < length) return true;
    const int i = j - length;
    if (i >= a.seq || row >= a.rows) return false;
    return a.tree[((size_t)b * a.seq + row % a.seq) * a.words + (i >> 5)] >> (i & 31) & 1;
}

// grid: (row blocks, splits, batch * kv_heads); kCols: 32-element columns of a head
template <typename T, int kCols>
__global__ void __launch_bounds__(kThreads) tree_simt_kernel(const TreeArgs a, int splits) {
    extern __shared__ float smem[];
    float *q = smem, *k = q + kRows * q_stride(a.dim), *v = k + kKeys * q_stride(a.dim), *p = v + kKeys * q_stride(a.dim);
    const int bh = blockIdx.z, b = bh / a.kv_heads, r = threadIdx.x >> 3, c = threadIdx.x & 7, row = blockIdx.x * kRows + r;
    const int length = a.lengths[b];
    if (length < 0 || length > a.capacity - a.seq) {
        if (threadIdx.x == 0) atomicCAS(a.err, 0, kErrCacheLength);
        return;
    }
    grid_dependency_trigger();
    const int n = length + a.seq, tiles = (n + kKeys - 1) / kKeys;
    const int t0 = (int)((long long)tiles * blockIdx.y / splits), t1 = (int)((long long)tiles * (blockIdx.y + 1) / splits);
    const size_t base = (size_t)bh * a.capacity * a.dim;
    stage<T, kRows>(q, static_cast<const T *>(a.q) + (size_t)bh * a.rows * a.dim, blockIdx.x * kRows, a.rows, a.dim);
    float m = -INFINITY, l = 0.0f;
    float4 o[kCols];
#pragma unroll
    for (int i = 0; i < kCols; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int t = t0; t < t1; ++t) {
        const int j0 = t * kKeys;
        __syncthreads();
        stage<T, kKeys>(k, static_cast<const T *>(a.k) + base, j0, n, a.dim);
        stage<T, kKeys>(v, static_cast<const T *>(a.v) + base, j0, n, a.dim);
        __syncthreads();
        float s[4], top = -INFINITY;
        tile_scores(q, k, r, c, a.dim, s);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            s[u] = sees(a, b, row, j0 + c + 8 * u, length) ? s[u] : -INFINITY;
            top = fmaxf(top, s[u]);
        }
#pragma unroll
        for (int x = 1; x < 8; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float m_new = fmaxf(m, top), shift = m_new == -INFINITY ? 0.0f : m_new;
        const float alpha = exp2f((m - shift) * a.scale_log2);
        m = m_new;
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float e = exp2f((s[u] - shift) * a.scale_log2);
            p[r * (kKeys + 1) + c + 8 * u] = e;
            sum += e;
        }
        l = l * alpha + sum;  // this thread's keys
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kCols; ++i) o[i].x *= alpha, o[i].y *= alpha, o[i].z *= alpha, o[i].w *= alpha;
        auto add = [&](int j, float w) {
#pragma unroll
            for (int i = 0; i < kCols; ++i)
                if ((c + 8 * i) * 4 < a.dim) {
                    const float4 x = *reinterpret_cast<const float4 *>(v + j * q_stride(a.dim) + (c + 8 * i) * 4);
                    o[i].x = fmaf(w, x.x, o[i].x), o[i].y = fmaf(w, x.y, o[i].y), o[i].z = fmaf(w, x.z, o[i].z), o[i].w = fmaf(w, x.w, o[i].w);
                }
        };
        const float *mine = p + r * (kKeys + 1);
        if (j0 + kKeys <= length) {
#pragma unroll 4
            for (int j = 0; j < kKeys; ++j) add(j, mine[j]);
        } else {  // drafts: no product with one that the row does not see
            for (int j = 0; j < kKeys; ++j)
                if (mine[j] != 0.0f) add(j, mine[j]);
        }
    }
#pragma unroll
    for (int x = 1; x < 8; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
    if (row >= a.rows) return;
    const size_t at = ((size_t)bh * a.rows + row) * splits + blockIdx.y;
    if (c == 0) a.part_ml[at] = make_float2(m, l);
#pragma unroll
    for (int i = 0; i < kCols; ++i)
        if ((c + 8 * i) * 4 < a.dim) *reinterpret_cast<float4 *>(a.part_o + at * a.dim + (c + 8 * i) * 4) = o[i];
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

// weights[j] += sum over all rows of p_j, p from the rows' joined maximum and sum: a
// block owns 32 keys of a (sequence, head), walks over the rows 16 at a time and adds
// the 16 row slots in order.
template <typename T>
__device__ __forceinline__ void add_weights(const TreeArgs &a, int splits, int first_tile, int step, int bh, float *smem) {
    float *q = smem, *k = q + kRows * q_stride(a.dim), *sums = k + kKeys * q_stride(a.dim);
    const int b = bh / a.kv_heads, r = threadIdx.x >> 3, c = threadIdx.x & 7;
    const int length = a.lengths[b], n = length + a.seq;
    if (length < 0 || length > a.capacity - a.seq) return;
    for (int j0 = first_tile * kKeys; j0 < n; j0 += step * kKeys) {
        float acc[4] = {};
        __syncthreads();
        stage<T, kKeys>(k, static_cast<const T *>(a.k) + (size_t)bh * a.capacity * a.dim, j0, n, a.dim);
        for (int r0 = 0; r0 < a.rows; r0 += kRows) {
            __syncthreads();
            stage<T, kRows>(q, static_cast<const T *>(a.q) + (size_t)bh * a.rows * a.dim, r0, a.rows, a.dim);
            // the row's maximum and sum over its splits, by its 8 threads
            float m = -INFINITY, l = 0.0f;
            if (r0 + r < a.rows) {
                const float2 *ml = a.part_ml + ((size_t)bh * a.rows + r0 + r) * splits;
                for (int s = c; s < splits; s += 8) m = fmaxf(m, ml[s].x);
            }
#pragma unroll
            for (int x = 1; x < 8; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
            const float shift = m == -INFINITY ? 0.0f : m;
            if (r0 + r < a.rows) {
                const float2 *ml = a.part_ml + ((size_t)bh * a.rows + r0 + r) * splits;
                for (int s = c; s < splits; s += 8) l = fmaf(ml[s].y, exp2f((ml[s].x - shift) * a.scale_log2), l);
            }
#pragma unroll
            for (int x = 1; x < 8; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
            __syncthreads();
            if (r0 + r >= a.rows) continue;
            const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
            float s[4];
            tile_scores(q, k, r, c, a.dim, s);
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (sees(a, b, r0 + r, j0 + c + 8 * u, length)) acc[u] += exp2f((s[u] - shift) * a.scale_log2) * inv;
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 4; ++u) sums[r * kKeys + c + 8 * u] = acc[u];
        __syncthreads();
        if (threadIdx.x < kKeys && j0 + threadIdx.x < n) {
            float s = 0.0f;
            for (int i = 0; i < kRows; ++i) s += sums[i * kKeys + threadIdx.x];
            a.weights[(size_t)bh * a.capacity + j0 + threadIdx.x] += s;
        }
    }
}

// Behind the splits: the first join_blocks blocks join rows, the others add weights
// (which read the splits' maxima and sums themselves, so neither waits for the other).
template <typename T>
__global__ void __launch_bounds__(kThreads) tree_finish_kernel(const TreeArgs a, int splits, int total_rows, int join_blocks, int key_blocks) {
    extern __shared__ float smem[];
    grid_dependency_wait();
    if ((int)blockIdx.x < join_blocks) return join_rows<T>(a, splits, total_rows, blockIdx.x);
    const int i = blockIdx.x - join_blocks, bh = i / key_blocks;
    add_weights<T>(a, splits, i - bh * key_blocks, key_blocks, bh, smem);
}

// ------------------------------------------------------------------ many rows
// From kWideRows rows on (FP32, 32 sequences and heads of 1,000 to 4,000 keys of 128: 144 us
// here and 202 on 16-row blocks at 48 rows, 146 and 283 at 64, equal up to 32): 64 rows
// by 64 keys a block of 256 threads, 4 x 4 scores and 4 rows by kCols x 4 columns of the
// sums a thread, so that a 16-byte shared-memory read feeds 8 to 11 FFMAs (the 16-row
// blocks: 3). K and V share a buffer; V is loaded into registers while the scores are
// formed, the next K while the sums are. Bound by FFMA issue beside shared-memory reads:
// 512 rows of 128 in FP32 run at about 20 TFLOP/s.
constexpr int kWideThreads = 256, kWideTile = 64, kWideRows = 33;

template <typename T, int kCols>  // kCols: 64-element columns of a head
struct WideStage {  // a tile of rows on its way to shared memory: 8 threads a row, 32 rows at a time
    float4 x[2][2 * kCols];
    __device__ __forceinline__ void load(const T *src, int first, int limit, int dim) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = first + (threadIdx.x >> 3) + 32 * i;
#pragma unroll
            for (int u = 0; u < 2 * kCols; ++u) {
                const int c = (threadIdx.x & 7) * 4 + 32 * u;
                x[i][u] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (r < limit && c < dim) x[i][u] = load4(src + (size_t)r * dim + c);
            }
        }
    }
    __device__ __forceinline__ void store(float *dst, int dim) const {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int u = 0; u < 2 * kCols; ++u) {
                const int c = (threadIdx.x & 7) * 4 + 32 * u;
                if (c < dim) *reinterpret_cast<float4 *>(dst + ((threadIdx.x >> 3) + 32 * i) * q_stride(dim) + c) = x[i][u];
            }
    }
};

// s[i][u]: row 4 ty + i with key tx + 16 u.
__device__ __forceinline__ void wide_scores(const float *q, const float *k, int dim, float (&s)[4][4]) {
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u) s[i][u] = 0.0f;
#pragma unroll 2
    for (int d = 0; d < dim; d += 4) {
        float4 x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4 *>(q + (4 * ty + i) * q_stride(dim) + d);
#pragma unroll
        for (int u = 0; u < 4; ++u) y[u] = *reinterpret_cast<const float4 *>(k + (tx + 16 * u) * q_stride(dim) + d);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int u = 0; u < 4; ++u) s[i][u] = fmaf(x[i].x, y[u].x, fmaf(x[i].y, y[u].y, fmaf(x[i].z, y[u].z, fmaf(x[i].w, y[u].w, s[i][u]))));
    }
}

constexpr int kWideP = kWideTile + 4;  // floats of a row of weights

// grid: (row blocks, splits, batch * kv_heads)
template <typename T, int kCols>
__global__ void __launch_bounds__(kWideThreads, kCols == 4 ? 1 : 2) tree_wide_kernel(const TreeArgs a, int splits) {
    extern __shared__ float smem[];
    float *q = smem, *kv = q + kWideTile * q_stride(a.dim), *p = kv + kWideTile * q_stride(a.dim);
    const int bh = blockIdx.z, b = bh / a.kv_heads, ty = threadIdx.x >> 4, tx = threadIdx.x & 15, row0 = blockIdx.x * kWideTile + 4 * ty;
    const int length = a.lengths[b];
    if (length < 0 || length > a.capacity - a.seq) {
        if (threadIdx.x == 0) atomicCAS(a.err, 0, kErrCacheLength);
        return;
    }
    grid_dependency_trigger();
    const int n = length + a.seq, tiles = (n + kWideTile - 1) / kWideTile;
    const int t0 = (int)((long long)tiles * blockIdx.y / splits), t1 = (int)((long long)tiles * (blockIdx.y + 1) / splits);
    const T *k = static_cast<const T *>(a.k) + (size_t)bh * a.capacity * a.dim, *v = static_cast<const T *>(a.v) + (size_t)bh * a.capacity * a.dim;
    WideStage<T, kCols> stage;
    stage.load(static_cast<const T *>(a.q) + (size_t)bh * a.rows * a.dim, blockIdx.x * kWideTile, a.rows, a.dim);
    stage.store(q, a.dim);
    if (t0 < t1) stage.load(k, t0 * kWideTile, n, a.dim);
    float m[4], l[4];
    float4 o[4][kCols];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m[i] = -INFINITY, l[i] = 0.0f;
#pragma unroll
        for (int c = 0; c < kCols; ++c) o[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int t = t0; t < t1; ++t) {
        const int j0 = t * kWideTile;
        __syncthreads();
        stage.store(kv, a.dim);
        stage.load(v, j0, n, a.dim);
        __syncthreads();
        float s[4][4];
        wide_scores(q, kv, a.dim, s);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float top = -INFINITY;
            if (j0 + kWideTile > length)
#pragma unroll
                for (int u = 0; u < 4; ++u) s[i][u] = sees(a, b, row0 + i, j0 + tx + 16 * u, length) ? s[i][u] : -INFINITY;
#pragma unroll
            for (int u = 0; u < 4; ++u) top = fmaxf(top, s[i][u]);
#pragma unroll
            for (int x = 1; x < 16; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
            const float m_new = fmaxf(m[i], top), shift = m_new == -INFINITY ? 0.0f : m_new;
            const float alpha = exp2f((m[i] - shift) * a.scale_log2);
            m[i] = m_new;
            float sum = 0.0f;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float e = exp2f((s[i][u] - shift) * a.scale_log2);
                p[(4 * ty + i) * kWideP + tx + 16 * u] = e;
                sum += e;
            }
            l[i] = l[i] * alpha + sum;  // this thread's keys
#pragma unroll
            for (int c = 0; c < kCols; ++c) o[i][c].x *= alpha, o[i][c].y *= alpha, o[i][c].z *= alpha, o[i][c].w *= alpha;
        }
        __syncthreads();  // K has been read, P is written
        stage.store(kv, a.dim);
        if (t + 1 < t1) stage.load(k, j0 + kWideTile, n, a.dim);
        __syncthreads();
        auto add = [&](auto careful) {
#pragma unroll 1
            for (int j = 0; j < kWideTile; j += 4) {
                float w[4][4];
#pragma unroll
                for (int i = 0; i < 4; ++i) *reinterpret_cast<float4 *>(w[i]) = *reinterpret_cast<const float4 *>(p + (4 * ty + i) * kWideP + j);
#pragma unroll
                for (int jj = 0; jj < 4; ++jj)
#pragma unroll
                    for (int c = 0; c < kCols; ++c)
                        if (tx * 4 + 64 * c < a.dim) {
                            const float4 x = *reinterpret_cast<const float4 *>(kv + (j + jj) * q_stride(a.dim) + tx * 4 + 64 * c);
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (!careful || w[i][jj] != 0.0f) {
                                    o[i][c].x = fmaf(w[i][jj], x.x, o[i][c].x), o[i][c].y = fmaf(w[i][jj], x.y, o[i][c].y);
                                    o[i][c].z = fmaf(w[i][jj], x.z, o[i][c].z), o[i][c].w = fmaf(w[i][jj], x.w, o[i][c].w);
                                }
                        }
            }
        };
        if (j0 + kWideTile <= length) add(std::false_type{});
        else add(std::true_type{});  // drafts: no product with one that the row does not see
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int x = 1; x < 16; x <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
        if (row0 + i >= a.rows) continue;
        const size_t at = ((size_t)bh * a.rows + row0 + i) * splits + blockIdx.y;
        if (tx == 0) a.part_ml[at] = make_float2(m[i], l[i]);
#pragma unroll
        for (int c = 0; c < kCols; ++c)
            if (tx * 4 + 64 * c < a.dim) *reinterpret_cast<float4 *>(a.part_o + at * a.dim + tx * 4 + 64 * c) = o[i][c];
    }
}

// add_weights for many rows: 64 keys a block, 64 rows at a time.
template <typename T, int kCols>
__device__ __forceinline__ void add_weights_wide(const TreeArgs &a, int splits, int first_tile, int step, int bh, float *smem) {
    float *q = smem, *k = q + kWideTile * q_stride(a.dim), *sums = k + kWideTile * q_stride(a.dim);
    float2 *stats = reinterpret_cast<float2 *>(sums + 16 * kWideTile);
    const int b = bh / a.kv_heads, ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    const int length = a.lengths[b], n = length + a.seq;
    if (length < 0 || length > a.capacity - a.seq) return;
    for (int j0 = first_tile * kWideTile; j0 < n; j0 += step * kWideTile) {
        float acc[4] = {};
        WideStage<T, kCols> stage;
        stage.load(static_cast<const T *>(a.k) + (size_t)bh * a.capacity * a.dim, j0, n, a.dim);
        __syncthreads();
        stage.store(k, a.dim);
        for (int r0 = 0; r0 < a.rows; r0 += kWideTile) {
            stage.load(static_cast<const T *>(a.q) + (size_t)bh * a.rows * a.dim, r0, a.rows, a.dim);
            __syncthreads();
            stage.store(q, a.dim);
            {  // a row's maximum and 1 / sum over its splits, by four threads
                const int row = r0 + (threadIdx.x >> 2), part = threadIdx.x & 3;
                const float2 *ml = a.part_ml + ((size_t)bh * a.rows + min(row, a.rows - 1)) * splits;
                float m = -INFINITY, l = 0.0f;
                for (int s = part; s < splits; s += 4) m = fmaxf(m, ml[s].x);
#pragma unroll
                for (int x = 1; x < 4; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
                const float shift = m == -INFINITY ? 0.0f : m;
                for (int s = part; s < splits; s += 4) l = fmaf(ml[s].y, exp2f((ml[s].x - shift) * a.scale_log2), l);
#pragma unroll
                for (int x = 1; x < 4; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
                if (part == 0) stats[threadIdx.x >> 2] = make_float2(shift, row < a.rows && (l > 0.0f || l != l) ? 1.0f / l : 0.0f);
            }
            __syncthreads();
            float s[4][4];
            wide_scores(q, k, a.dim, s);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = r0 + 4 * ty + i;
                const float2 st = stats[4 * ty + i];
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (row < a.rows && sees(a, b, row, j0 + tx + 16 * u, length)) acc[u] += exp2f((s[i][u] - st.x) * a.scale_log2) * st.y;
            }
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 4; ++u) sums[ty * kWideTile + tx + 16 * u] = acc[u];
        __syncthreads();
        if (threadIdx.x < kWideTile && j0 + threadIdx.x < n) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) s += sums[i * kWideTile + threadIdx.x];
            a.weights[(size_t)bh * a.capacity + j0 + threadIdx.x] += s;
        }
    }
}

template <typename T, int kCols>
__global__ void __launch_bounds__(kWideThreads, kCols == 4 ? 1 : 2)
    tree_finish_wide_kernel(const TreeArgs a, int splits, int total_rows, int join_blocks, int key_blocks) {
    extern __shared__ float smem[];
    grid_dependency_wait();
    if ((int)blockIdx.x < join_blocks) return join_rows<T>(a, splits, total_rows, blockIdx.x);
    const int i = blockIdx.x - join_blocks, bh = i / key_blocks;
    add_weights_wide<T, kCols>(a, splits, i - bh * key_blocks, key_blocks, bh, smem);
}

template <typename T>
LaunchFn simt_launch(Context *ctx, const Spec &s) {
    TreeArgs base = tree_args(ctx, s);
    const int heads = (int)(s.batch * s.kv_heads), rows = base.rows, total_rows = heads * rows;
    if (heads > 65535) throw IrError("attention_tree: batch * kv_heads must be at most 65535");
    const bool wide = rows >= kWideRows;
    const int tile_rows = wide ? kWideTile : kRows, tile_keys = wide ? kWideTile : kKeys, threads = wide ? kWideThreads : kThreads;
    const int row_blocks = (rows + tile_rows - 1) / tile_rows;
    // about four blocks per SM
    const long long items = (long long)heads * row_blocks;
    const int splits = (int)std::max<long long>(1, std::min<long long>({(4ll * ctx->sm_count + items - 1) / items, ((long long)s.capacity + tile_keys - 1) / tile_keys,
                                                                        (long long)kMaxSplits}));
    const size_t parts = (size_t)total_rows * splits;
    auto ws = kernel_workspace(parts * (s.dim * sizeof(float) + sizeof(float2)), "attention_tree partial results");
    base.part_o = static_cast<float *>(ws.get());  // rows of a multiple of 32 bytes: read as 16-byte vectors
    base.part_ml = reinterpret_cast<float2 *>(base.part_o + parts * s.dim);
    const size_t row = (size_t)q_stride(s.dim) * 4;
    const size_t smem = wide ? 2 * kWideTile * row + kWideTile * kWideP * 4 : (kRows + 2 * kKeys) * row + kRows * (kKeys + 1) * 4;
    const size_t smem_w = !s.weights ? 0 : wide ? 2 * kWideTile * row + 16 * kWideTile * 4 + kWideTile * 8 : (kRows + kKeys) * row + kRows * kKeys * 4;
    void (*kernel)(TreeArgs, int);
    void (*finish)(TreeArgs, int, int, int, int);
    if (wide) {
        kernel = s.dim <= 64 ? tree_wide_kernel<T, 1> : s.dim <= 128 ? tree_wide_kernel<T, 2> : tree_wide_kernel<T, 4>;
        finish = s.dim <= 64 ? tree_finish_wide_kernel<T, 1> : s.dim <= 128 ? tree_finish_wide_kernel<T, 2> : tree_finish_wide_kernel<T, 4>;
    } else {
        kernel = s.dim <= 64 ? tree_simt_kernel<T, 2> : s.dim <= 128 ? tree_simt_kernel<T, 4> : tree_simt_kernel<T, 8>;
        finish = tree_finish_kernel<T>;
    }
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
        cudaFuncSetAttribute(finish, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_w) != cudaSuccess)
        throw IrError("cannot reserve shared memory for attention_tree");
    const bool weights = s.weights;
    const int key_blocks = (int)std::min<long long>((s.capacity + tile_keys - 1) / tile_keys, std::max<long long>(1, 8ll * ctx->sm_count / heads));
    const int join_blocks = (total_rows + threads / 32 - 1) / (threads / 32);
    return [=, keep = ws](cudaStream_t st, void **b) {
        const TreeArgs a = tree_bind(base, b, weights);
        kernel<<<dim3(row_blocks, splits, heads), threads, smem, st>>>(a, splits);
        const cudaError_t e = launch_after(st, finish, dim3(join_blocks + (weights ? key_blocks * heads : 0)), threads, smem_w, a, splits, total_rows,
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
