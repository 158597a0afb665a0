// Arguments shared by the attention_tree kernels (attention_tree.cu has the
// operator's definition).
#pragma once
#include <cmath>

#include "common.cuh"
#include "internal.hpp"

namespace jade {

struct TreeArgs {
    const void *q, *k, *v;
    const int *lengths;
    const uint32_t *tree;  // [batch, seq, words]
    void *out;
    float *weights;
    float *row_exponents;  // for the tcgen05 weights (attention_tree_tc.cu)
    float2 *part_ml;  // per row and split: maximum and sum
    float *part_o;    // per row and split: dim unnormalised sums
    int batch, kv_heads, group, seq, words, dim, capacity, rows;  // rows = group * seq
    float scale_log2;  // log2(e) / sqrt(dim): scores to exponents of 2
    bool drafts_only;  // rows that see no draft add no weight
    int *err;
};

// The bits of word w that stand for drafts: bits beyond them may be anything.
__device__ __forceinline__ uint32_t draft_bits(int w, int seq) {
    const int n = seq - 32 * w;
    return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1;
}
// Whether a row of sequence b adds weights.
__device__ __forceinline__ bool adds_weight(const TreeArgs &a, int b, int row) {
    if (!a.drafts_only) return true;
    const uint32_t *words = a.tree + ((size_t)b * a.seq + row % a.seq) * a.words;
    uint32_t any = 0;
    for (int w = 0; w < a.words; ++w) any |= __ldg(words + w) & draft_bits(w, a.seq);
    return any;
}

inline TreeArgs tree_args(Context *ctx, const Spec &s) {
    TreeArgs a{};
    a.batch = s.batch, a.kv_heads = s.kv_heads, a.group = s.heads / s.kv_heads, a.seq = s.seq, a.words = (s.seq + 31) / 32;
    a.dim = s.dim, a.capacity = s.capacity, a.rows = a.group * a.seq;
    a.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)s.dim));
    a.drafts_only = s.drafts_only;
    a.err = ctx->err_dev;
    return a;
}
// the spec's bindings: q, k, v, lengths, tree, out, weights
inline TreeArgs tree_bind(TreeArgs a, void **b, bool weights) {
    a.q = b[0], a.k = b[1], a.v = b[2], a.lengths = static_cast<const int *>(b[3]), a.tree = static_cast<const uint32_t *>(b[4]);
    a.out = b[5];
    a.weights = weights ? static_cast<float *>(b[6]) : nullptr;
    return a;
}

LaunchFn make_attention_tree_tc(Context *ctx, const Spec &s);  // 16-bit types, dim up to 128

}  // namespace jade
