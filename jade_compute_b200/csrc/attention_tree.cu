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

#include "attention_tree.cuh"

namespace jade {
namespace {

constexpr int kThreads = 128, kRows = 16, kKeys = 32;  // a block: 16 rows of q, tiles of 32 keys

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

// Rows of q or keys (zeros from `limit` on) as FP32 into shared memory.
template <typename T>
__device__ __forceinline__ void stage(float *dst, const T *src, int first, int count, int limit, int dim) {
    const int vecs = dim / 4;
    for (int i = threadIdx.x; i < count * vecs; i += kThreads) {
        const int r = i / vecs, c = (i - r * vecs) * 4;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (first + r < limit) x = load4(src + (size_t)(first + r) * dim + c);
        *reinterpret_cast<float4 *>(dst + r * q_stride(dim) + c) = x;
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

// grid: (row blocks, splits, batch * kv_heads)
template <typename T>
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
    stage(q, static_cast<const T *>(a.q) + (size_t)bh * a.rows * a.dim, blockIdx.x * kRows, kRows, a.rows, a.dim);
    float m = -INFINITY, l = 0.0f;
    float4 o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int t = t0; t < t1; ++t) {
        const int j0 = t * kKeys;
        __syncthreads();
        stage(k, static_cast<const T *>(a.k) + base, j0, kKeys, n, a.dim);
        stage(v, static_cast<const T *>(a.v) + base, j0, kKeys, n, a.dim);
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
        for (int i = 0; i < 8; ++i) o[i].x *= alpha, o[i].y *= alpha, o[i].z *= alpha, o[i].w *= alpha;
        for (int j = 0; j < kKeys; ++j) {
            const float w = p[r * (kKeys + 1) + j];
            if (w == 0.0f) continue;  // not seen, or below FP32: no product
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if ((c + 8 * i) * 4 < a.dim) {
                    const float4 x = *reinterpret_cast<const float4 *>(v + j * q_stride(a.dim) + (c + 8 * i) * 4);
                    o[i].x = fmaf(w, x.x, o[i].x), o[i].y = fmaf(w, x.y, o[i].y), o[i].z = fmaf(w, x.z, o[i].z), o[i].w = fmaf(w, x.w, o[i].w);
                }
        }
    }
#pragma unroll
    for (int x = 1; x < 8; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
    if (row >= a.rows) return;
    const size_t at = ((size_t)bh * a.rows + row) * splits + blockIdx.y;
    if (c == 0) a.part_ml[at] = make_float2(m, l);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if ((c + 8 * i) * 4 < a.dim) *reinterpret_cast<float4 *>(a.part_o + at * a.dim + (c + 8 * i) * 4) = o[i];
}

// Joins the splits of one row: one warp a row.
template <typename T>
__global__ void __launch_bounds__(128) tree_join_kernel(const TreeArgs a, int splits, int total_rows) {
    const int row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    grid_dependency_trigger();
    grid_dependency_wait();
    if (row >= total_rows) return;
    const int bh = row / a.rows, rr = row - bh * a.rows, b = bh / a.kv_heads, hk = bh - b * a.kv_heads;
    if (a.lengths[b] < 0 || a.lengths[b] > a.capacity - a.seq) return;
    const float2 *ml = a.part_ml + (size_t)row * splits;
    float m = -INFINITY, l = 0.0f;
    for (int s = 0; s < splits; ++s) m = fmaxf(m, ml[s].x);
    const float shift = m == -INFINITY ? 0.0f : m;
    for (int s = 0; s < splits; ++s) l += ml[s].y * exp2f((ml[s].x - shift) * a.scale_log2);
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    if (lane == 0 && a.stats) a.stats[row] = make_float2(shift * a.scale_log2, inv);
    const int g = rr / a.seq, t = rr - g * a.seq;
    T *out = static_cast<T *>(a.out) + (((size_t)b * a.seq + t) * a.kv_heads * a.group + hk * a.group + g) * a.dim;
    for (int d = lane * 4; d < a.dim; d += 128) {
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s = 0; s < splits; ++s) {
            const float w = exp2f((ml[s].x - shift) * a.scale_log2);
            if (w == 0.0f) continue;
            const float4 y = *reinterpret_cast<const float4 *>(a.part_o + ((size_t)row * splits + s) * a.dim + d);
            x.x = fmaf(w, y.x, x.x), x.y = fmaf(w, y.y, x.y), x.z = fmaf(w, y.z, x.z), x.w = fmaf(w, y.w, x.w);
        }
        out[d] = from_f32<T>(x.x * inv), out[d + 1] = from_f32<T>(x.y * inv), out[d + 2] = from_f32<T>(x.z * inv), out[d + 3] = from_f32<T>(x.w * inv);
    }
}

// weights[j] += sum over all rows of p_j, p from the rows' final maximum and sum: a
// block owns 32 keys of a (sequence, head), walks over the rows 16 at a time and
// adds the 16 row slots in order. grid: (key tiles, batch * kv_heads)
template <typename T>
__global__ void __launch_bounds__(kThreads) tree_weights_simt_kernel(const TreeArgs a) {
    extern __shared__ float smem[];
    float *q = smem, *k = q + kRows * q_stride(a.dim), *sums = k + kKeys * q_stride(a.dim);
    const int bh = blockIdx.y, b = bh / a.kv_heads, r = threadIdx.x >> 3, c = threadIdx.x & 7;
    const int length = a.lengths[b], n = length + a.seq;
    grid_dependency_wait();  // the rows' stats
    if (length < 0 || length > a.capacity - a.seq) return;
    for (int j0 = blockIdx.x * kKeys; j0 < n; j0 += gridDim.x * kKeys) {
        float acc[4] = {};
        __syncthreads();
        stage(k, static_cast<const T *>(a.k) + (size_t)bh * a.capacity * a.dim, j0, kKeys, n, a.dim);
        for (int r0 = 0; r0 < a.rows; r0 += kRows) {
            __syncthreads();
            stage(q, static_cast<const T *>(a.q) + (size_t)bh * a.rows * a.dim, r0, kRows, a.rows, a.dim);
            __syncthreads();
            if (r0 + r >= a.rows) continue;
            float s[4];
            tile_scores(q, k, r, c, a.dim, s);
            const float2 st = a.stats[(size_t)bh * a.rows + r0 + r];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (sees(a, b, r0 + r, j0 + c + 8 * u, length)) acc[u] += exp2f(fmaf(s[u], a.scale_log2, -st.x)) * st.y;
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

template <typename T>
LaunchFn simt_launch(Context *ctx, const Spec &s) {
    TreeArgs base = tree_args(ctx, s);
    const int heads = (int)(s.batch * s.kv_heads), rows = base.rows, row_blocks = (rows + kRows - 1) / kRows, total_rows = heads * rows;
    if (heads > 65535) throw IrError("attention_tree: batch * kv_heads must be at most 65535");
    // about four blocks per SM
    const long long items = (long long)heads * row_blocks;
    const int splits = (int)std::max<long long>(1, std::min<long long>({(4ll * ctx->sm_count + items - 1) / items, ((long long)s.capacity + kKeys - 1) / kKeys, 64ll}));
    const size_t stats = (size_t)total_rows * sizeof(float2), ml = stats * splits;
    auto ws = kernel_workspace(stats + ml + (size_t)total_rows * splits * s.dim * 4, "attention_tree partial results");
    base.stats = static_cast<float2 *>(ws.get());
    base.part_ml = base.stats + total_rows;
    base.part_o = reinterpret_cast<float *>(base.part_ml + (size_t)total_rows * splits);
    const size_t row = (size_t)q_stride(s.dim) * 4;
    const size_t smem = (kRows + 2 * kKeys) * row + kRows * (kKeys + 1) * 4, smem_w = (kRows + kKeys) * row + kRows * kKeys * 4;
    if (cudaFuncSetAttribute(tree_simt_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
        cudaFuncSetAttribute(tree_weights_simt_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_w) != cudaSuccess)
        throw IrError("cannot reserve shared memory for attention_tree");
    const bool weights = s.weights;
    const int key_blocks = (int)std::min<long long>((s.capacity + kKeys - 1) / kKeys, std::max<long long>(1, 8ll * ctx->sm_count / heads));
    return [=, keep = ws](cudaStream_t st, void **b) {
        const TreeArgs a = tree_bind(base, b, weights);
        tree_simt_kernel<T><<<dim3(row_blocks, splits, heads), kThreads, smem, st>>>(a, splits);
        cudaError_t e = launch_after(st, tree_join_kernel<T>, dim3((total_rows + 3) / 4), 128, 0, a, splits, total_rows);
        if (weights && e == cudaSuccess) e = launch_after(st, tree_weights_simt_kernel<T>, dim3(key_blocks, heads), kThreads, smem_w, a);
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
