// cache_evict and cache_commit: which entries of a key/value cache stay, and
// moving them together. k, v are [batch, kv_heads, capacity, dim]; entry j of a
// sequence is slot j < length. Rows are moved as 16-byte vectors whatever their
// type (dim is a multiple of 8).
//
// cache_evict keeps, for every (sequence, head), the `recent` newest entries and
// of the others those of largest accumulated weight up to `keep` in all (equal
// weights: the lower slot; NaN counts as largest, -0 as 0), in slot order, and
// writes them to another cache from slot 0 on. kept: their old slots, then -1.
//
// cache_commit: after attention_tree over seq drafted tokens in slots length ..,
// moves the accepted ones, path[0 .. count) ascending, to slots length + 0, 1, ...
// in place; their accumulated weights too, the rest of the drafts' weights to 0.
#include <cooperative_groups.h>

#include <algorithm>
#include <climits>

#include "common.cuh"
#include "internal.hpp"

namespace jade {
namespace {

namespace cg = cooperative_groups;

// ------------------------------------------------------------------ cache_evict
struct EvictArgs {
    const uint4 *k, *v;
    const float *weights;
    const int *lengths;
    uint4 *k_out, *v_out;
    float *weights_out;
    int *kept, *lengths_out;
    int kv_heads, capacity, keep, recent, vecs;  // vecs: 16-byte vectors of a row
    int *err;
};

// Unsigned keys in the order of the weights.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w == 0.0f ? 0.0f : w);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelectThreads = 1024, kSelectEach = 8, kSelectTile = kSelectThreads * kSelectEach, kBins = 2048;

// Exclusive prefix sum of v over the block, in thread order, and its total.
__device__ __forceinline__ uint32_t block_prefix(uint32_t v, uint32_t *warp_sums, uint32_t &total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t sum = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t n = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += n;
    }
    __syncthreads();  // warp_sums may still be read
    if (lane == 31) warp_sums[warp] = sum;
    __syncthreads();
    uint32_t w = warp_sums[lane], upto = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t n = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += n;
    }
    total = __shfl_sync(0xffffffffu, upto, 31);
    return __shfl_sync(0xffffffffu, upto - w, warp) + sum - v;
}

// A cluster of blocks per (sequence, head), each with a run of its entries. The
// need-th largest key among the entries that may go is found digit by digit from the
// top (11, 11, 10 bits: with 8-bit digits the first holds little but the exponent, and
// its few bins serialise the counting): every block counts its run in shared memory and
// adds up the counts of all blocks, two bins a thread. Then the kept slots are written
// in order: 8 neighbouring entries a thread, one prefix sum over the block for entries
// above the threshold and entries equal to it together, behind the earlier blocks'
// totals. Weights come from memory once where a run has at most kSelectTile entries
// (their keys stay in shared memory), else once per pass. Bound by latency: block
// barriers and shared-memory atomics of the three passes; 64 heads of 4,096 to 8,192
// entries take about 15 us. evict_move is bound by HBM: 64 heads of 2,048
// kept rows of 128 in BF16 (134 MB moved) take about 21 us, 6.2 TB/s with its writes to L2.
template <bool kCluster>
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const EvictArgs a) {
    __shared__ uint32_t keys[kSelectTile + kSelectTile / 32], hist[kBins], warp_sums[32], chosen[2], totals[2];
    const cg::cluster_group cluster = cg::this_cluster();
    const int blocks = kCluster ? cluster.num_blocks() : 1, rank = kCluster ? cluster.block_rank() : 0;
    const int bh = blockIdx.x / blocks, b = bh / a.kv_heads, n = a.lengths[b], thread = threadIdx.x;
    grid_dependency_trigger();
    if (n < 0 || n > a.capacity) {  // the same for the whole cluster
        if (thread == 0) atomicCAS(a.err, 0, kErrCacheLength);
        return;
    }
    auto sync = [&] {  // all blocks of the cluster
        if constexpr (kCluster) cluster.sync();
        else __syncthreads();
    };
    int *kept = a.kept + (size_t)bh * a.keep;
    const float *w = a.weights + (size_t)bh * a.capacity;
    float *w_out = a.weights_out + (size_t)bh * a.capacity;
    const int count = min(n, a.keep), last = max(0, n - a.recent);
    const int run = (n + blocks - 1) / blocks, lo = min(n, rank * run), hi = min(n, lo + run);
    uint32_t need = count - (n - last);  // of the first `last` entries
    const bool all = need >= (uint32_t)last, single = run <= kSelectTile;
    auto at = [](int j) { return j + (j >> 5); };  // a thread's run of 8 without bank conflicts
    auto load_tile = [&](int j0) {
#pragma unroll
        for (int u = 0; u < kSelectEach; ++u) {
            const int j = u * kSelectThreads + thread;
            if (j0 + j < hi) keys[at(j)] = weight_key(w[j0 + j]);
        }
    };
    uint32_t threshold = 0;
    if (single) load_tile(lo);
    for (int pass = 0; pass < 3 && !all && need > 0; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, digit = pass < 2 ? 11 : 10;
        for (int i = thread; i < kBins; i += kSelectThreads) hist[i] = 0;
        __syncthreads();
        for (int j = lo + thread; j < min(hi, last); j += kSelectThreads) {
            const uint32_t key = single ? keys[at(j - lo)] : weight_key(w[j]);
            if (pass == 0 || key >> (shift + digit) == threshold) atomicAdd(&hist[key >> shift & ((1u << digit) - 1)], 1u);
        }
        sync();
        const int high = kBins - 1 - 2 * thread;  // two bins a thread, the largest first
        uint32_t c0 = 0, c1 = 0;
#pragma unroll 8
        for (int r = 0; r < blocks; ++r) {
            const uint2 c = *reinterpret_cast<const uint2 *>((kCluster ? cluster.map_shared_rank(hist, r) : hist) + high - 1);
            c0 += c.y, c1 += c.x;
        }
        uint32_t total;
        const uint32_t above = block_prefix(c0 + c1, warp_sums, total);
        if (above < need && need <= above + c0) chosen[0] = high, chosen[1] = need - above;
        else if (above + c0 < need && need <= above + c0 + c1) chosen[0] = high - 1, chosen[1] = need - above - c0;
        sync();  // and no block clears counts that another still reads
        threshold = threshold << digit | chosen[0];
        need = chosen[1];
    }
    // threshold: the smallest kept key; need: how many entries with exactly it are kept, the lowest slots
    auto sort_out = [&](int j0, uint32_t &mask, uint32_t &equal) {  // of the thread's 8 entries of the tile
        mask = equal = 0;
#pragma unroll
        for (int i = 0; i < kSelectEach; ++i) {
            const int j = j0 + thread * kSelectEach + i;
            if (j >= hi) break;
            const uint32_t key = keys[at(thread * kSelectEach + i)];
            if (all || j >= last || (need > 0 && key > threshold)) mask |= 1u << i;
            else if (need > 0 && key == threshold) equal |= 1u << i;
        }
    };
    uint32_t takes = 0, ties = 0, mask, equal, total;
    if constexpr (kCluster) {
        for (int j0 = lo; j0 < hi; j0 += kSelectTile) {
            if (!single) {
                __syncthreads();
                load_tile(j0);
            }
            __syncthreads();
            sort_out(j0, mask, equal);
            block_prefix(__popc(mask) | __popc(equal) << 16, warp_sums, total);
            takes += total & 0xffffu, ties += total >> 16;
        }
        if (thread == 0) totals[0] = takes, totals[1] = ties;
        sync();
        takes = ties = 0;
        for (int r = 0; r < rank; ++r) {
            const uint32_t *t = cluster.map_shared_rank(totals, r);
            takes += t[0], ties += t[1];
        }
        sync();  // no block leaves while another reads its totals
    }
    for (int j0 = lo; j0 < hi; j0 += kSelectTile) {
        if (!single) {
            __syncthreads();
            load_tile(j0);
        }
        __syncthreads();
        sort_out(j0, mask, equal);
        const uint32_t before = block_prefix(__popc(mask) | __popc(equal) << 16, warp_sums, total);
        uint32_t take = takes + (before & 0xffffu), tie = ties + (before >> 16);
#pragma unroll
        for (int i = 0; i < kSelectEach; ++i) {
            const bool is_tie = equal >> i & 1, on = (mask >> i & 1) || (is_tie && tie < need);
            if (on) {
                const int j = j0 + thread * kSelectEach + i;
                const uint32_t to = take + min(tie, need);
                kept[to] = j;
                w_out[to] = w[j];
            }
            take += mask >> i & 1;
            tie += is_tie;
        }
        takes += total & 0xffffu, ties += total >> 16;
    }
    const int first = rank * kSelectThreads + thread, step = blocks * kSelectThreads;
    for (int i = count + first; i < a.keep; i += step) kept[i] = -1;
    for (int i = count + first; i < a.capacity; i += step) w_out[i] = 0.0f;
    if (bh % a.kv_heads == 0 && first == 0) a.lengths_out[b] = count;
}

__global__ void __launch_bounds__(256) evict_move_kernel(const EvictArgs a) {
    const int bh = blockIdx.y, n = a.lengths[bh / a.kv_heads], count = min(n, a.keep);
    const int *kept = a.kept + (size_t)bh * a.keep;
    const size_t base = (size_t)bh * a.capacity;
    const long long total = (long long)count * a.vecs;
    grid_dependency_wait();  // kept; in every block: this grid's end stands for the one's before it
    if (n < 0 || n > a.capacity) return;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const int row = (int)(i / a.vecs), vec = (int)(i - (long long)row * a.vecs);
        const size_t from = (base + kept[row]) * a.vecs + vec, to = (base + row) * a.vecs + vec;
        a.k_out[to] = __ldg(a.k + from);
        a.v_out[to] = __ldg(a.v + from);
    }
}

// ------------------------------------------------------------------ cache_commit
struct CommitArgs {
    const int *path, *counts, *lengths;
    uint4 *k, *v;
    float *weights;
    int *lengths_out;
    int kv_heads, capacity, seq, vecs;
    int *err;
};

constexpr int kCommitThreads = 256, kCommitVecs = 4;

// Bound by latency (lengths, then paths, then rows): 32 sequences of 8 heads that move
// up to 8 rows of 128 take 4.8 us, one sequence 3.8.
// One block per (sequence, head). Paths ascend, so path[i] >= i: rows are moved in
// order, a block's worth at a time (all read before any is written), and no later
// row's source is overwritten.
__global__ void __launch_bounds__(kCommitThreads) commit_kernel(const CommitArgs a) {
    const int bh = blockIdx.x, b = bh / a.kv_heads, n = a.lengths[b], count = a.counts[b];
    const int *path = a.path + (size_t)b * a.seq;
    const int i = threadIdx.x;
    bool good = n >= 0 && n <= a.capacity - a.seq;
    if (!good && i == 0) atomicCAS(a.err, 0, kErrCacheLength);
    bool path_good = count >= 0 && count <= a.seq;
    if (path_good && i < count) path_good = path[i] >= 0 && path[i] < a.seq && (i == 0 || path[i] > path[i - 1]);
    path_good = __syncthreads_and(path_good);
    if (!path_good && i == 0) atomicCAS(a.err, 0, kErrCommitPath);
    if (!good || !path_good) return;
    const size_t base = (size_t)bh * a.capacity + n;
    if (bh % a.kv_heads == 0 && i == 0) a.lengths_out[b] = n + count;
    if (a.weights) {
        float moved = 0.0f;
        if (i < count) moved = a.weights[base + path[i]];
        __syncthreads();
        if (i < a.seq) a.weights[base + i] = moved;
    }
    const int total = count * a.vecs;
    for (int j0 = 0; j0 < total; j0 += kCommitThreads * kCommitVecs) {
        uint4 kr[kCommitVecs], vr[kCommitVecs];
#pragma unroll
        for (int u = 0; u < kCommitVecs; ++u) {
            const int j = j0 + u * kCommitThreads + i;
            if (j < total) {
                const size_t from = (base + path[j / a.vecs]) * a.vecs + j % a.vecs;
                kr[u] = a.k[from], vr[u] = a.v[from];
            }
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kCommitVecs; ++u) {
            const int j = j0 + u * kCommitThreads + i;
            if (j < total) a.k[base * a.vecs + j] = kr[u], a.v[base * a.vecs + j] = vr[u];
        }
        __syncthreads();
    }
}

}  // namespace

LaunchFn make_cache_op(Context *ctx, const Spec &s, std::string &impl) {
    impl = std::string(spec_name(s)) + "_" + dtype_name(s.dtype);
    const int heads = (int)(s.batch * s.kv_heads), vecs = (int)(s.dim * dtype_size(s.dtype) / 16);
    if (s.op == Op::CacheCommit) {
        CommitArgs base{};
        base.kv_heads = s.kv_heads, base.capacity = s.capacity, base.seq = s.seq, base.vecs = vecs, base.err = ctx->err_dev;
        const bool weights = s.weights;
        return [=](cudaStream_t st, void **b) {
            CommitArgs a = base;
            a.path = static_cast<const int *>(b[0]), a.counts = static_cast<const int *>(b[1]), a.lengths = static_cast<const int *>(b[2]);
            a.k = static_cast<uint4 *>(b[3]), a.v = static_cast<uint4 *>(b[4]);
            a.weights = weights ? static_cast<float *>(b[5]) : nullptr;
            a.lengths_out = static_cast<int *>(b[weights ? 6 : 5]);
            commit_kernel<<<heads, kCommitThreads, 0, st>>>(a);
            return cudaGetLastError();
        };
    }
    if (heads > 65535) throw IrError("cache_evict: batch * kv_heads must be at most 65535");
    EvictArgs base{};
    base.kv_heads = s.kv_heads, base.capacity = s.capacity, base.keep = s.keep, base.recent = s.recent, base.vecs = vecs;
    base.err = ctx->err_dev;
    const int blocks = (int)std::min<long long>(((long long)s.keep * vecs + 1023) / 1024, std::max(1, 16 * ctx->sm_count / heads));
    // Blocks per (sequence, head), up to 8: more while a block would have more than one
    // tile and there are SMs. A cluster's barriers and counts from the other blocks cost
    // about what a second tile does: 64 heads of 8192 entries take 37 us with one block
    // each and 39 with two; 8 of 60,000 took 171 us with one, 89 with eight.
    int cluster = 1;
    while (cluster < 8 && heads * cluster * 2 <= ctx->sm_count && s.capacity > (uint32_t)(kSelectTile * cluster)) cluster *= 2;
    return [=](cudaStream_t st, void **b) {
        EvictArgs a = base;
        a.k = static_cast<const uint4 *>(b[0]), a.v = static_cast<const uint4 *>(b[1]), a.weights = static_cast<const float *>(b[2]);
        a.lengths = static_cast<const int *>(b[3]), a.k_out = static_cast<uint4 *>(b[4]), a.v_out = static_cast<uint4 *>(b[5]);
        a.weights_out = static_cast<float *>(b[6]), a.kept = static_cast<int *>(b[7]), a.lengths_out = static_cast<int *>(b[8]);
        cudaLaunchAttribute shape{};
        shape.id = cudaLaunchAttributeClusterDimension;
        shape.val.clusterDim.x = cluster, shape.val.clusterDim.y = shape.val.clusterDim.z = 1;
        cudaLaunchConfig_t config{};
        config.gridDim = dim3(heads * cluster), config.blockDim = dim3(kSelectThreads), config.stream = st, config.attrs = &shape, config.numAttrs = cluster > 1;
        cudaError_t e = cudaLaunchKernelEx(&config, cluster > 1 ? evict_select_kernel<true> : evict_select_kernel<false>, a);
        if (e == cudaSuccess) e = launch_after(st, evict_move_kernel, dim3(blocks, heads), 256, 0, a);
        return e == cudaSuccess ? cudaGetLastError() : e;
    };
}

}  // namespace jade
