// qk_norm_rope and its gradient: per-head RMS norm of queries and keys, rotary
// positions, and the layout change from a projection's packed rows to the
// attention's operands, in one pass over the data.
//
//   x = qkv[b, t, head, :],  r = 1 / sqrt(mean(x^2) + eps),  y = P(pos) (x r w)
//
// P turns element pairs (a, b) by the angle pos * theta_i: (a cos - b sin,
// a sin + b cos), i = 0 .. rotary/2 - 1, for the halves (i, i + rotary/2) or the
// neighbours (2i, 2i + 1); the rest of the head passes. theta_i = base^(-2i/rotary),
// scaled for longer contexts by `linear` (theta / factor), `ntk` (base *
// factor^(rotary / (rotary - 2))) or `yarn` (Peng et al. 2023: theta / factor for
// pairs that turn less than once within the original context, theta for those that
// turn more than 32 times, a linear mix between; cos and sin times 0.1 ln(factor) + 1).
// Queries go to [batch, heads, seq, dim], keys and values to rows start .. of
// [batch, kv_heads, capacity, dim]; values are copied.
//
// Gradient, with g = P^T dy: dw = sum g x r, u = g w, dx = r (u - x r mean(u x r)).
//
// All arithmetic is FP32, one rounding to the output type. The angle is formed as
// a fraction of a turn in 64-bit fixed point (theta / 2 pi as a 0.64 fraction, times
// the position, modulo 2^64): exact reduction at every position, where an FP32
// product is off by 0.004 rad at position 100,000.
#include <cmath>
#include <vector>

#include "common.cuh"
#include "internal.hpp"

namespace jade {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;

struct RopeArgs {
    const void *qkv, *q_weight, *k_weight;
    const int *positions, *starts;
    const uint64_t *turns;  // theta / 2 pi as 0.64 fractions, rotary / 2 of them
    void *q, *k, *v;        // outputs (gradient: dq, dk, dv, inputs)
    void *dqkv;
    float *partial;         // gradient: [block][2][dim] sums of the norm weights' gradients
    int batch, seq, heads, kv_heads, dim, rotary, interleaved, norm, rows;  // rows: of k and v per head
    float epsilon, gain;
    int *err;
};

// 8 consecutive elements: 16 bytes of a 16-bit type, 32 of FP32.
__device__ __forceinline__ void load8(const float *p, float (&x)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&x)[8]) {
    const uint4 u = __ldg(reinterpret_cast<const uint4 *>(p));
    const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __bfloat1622float2(h[i]);
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void load8(const __half *p, float (&x)[8]) {
    const uint4 u = __ldg(reinterpret_cast<const uint4 *>(p));
    const __half2 *h = reinterpret_cast<const __half2 *>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(h[i]);
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void store8(float *p, const float (&x)[8]) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16 *p, const float (&x)[8]) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}
__device__ __forceinline__ void store8(__half *p, const float (&x)[8]) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(pack_f16(x[0], x[1]), pack_f16(x[2], x[3]), pack_f16(x[4], x[5]), pack_f16(x[6], x[7]));
}

// A warp holds 32 / kLanes head rows, kLanes lanes each, 8 elements a lane.
template <int kLanes>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Turns the lane's 8 elements (first: index of the first) by the token's angles;
// sign -1 turns back. The halves' partners are fetched through the warp's rows in
// shared memory.
template <int kLanes>
__device__ __forceinline__ void turn8(const RopeArgs &a, const float2 *cs, float *warp_rows, int row, int first, float sign, float (&x)[8]) {
    if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 8; i += 2)
            if (first + i < a.rotary) {
                const float2 t = cs[(first + i) >> 1];
                const float u = x[i] * t.x - sign * (x[i + 1] * t.y), w = sign * (x[i] * t.y) + x[i + 1] * t.x;
                x[i] = u, x[i + 1] = w;
            }
        return;
    }
    float *mine = warp_rows + row * (kLanes * 8);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) mine[first + i] = x[i];
    __syncwarp();
    const int half = a.rotary >> 1;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int e = first + i;
        if (e < half) {
            const float2 t = cs[e];
            x[i] = x[i] * t.x - sign * (mine[e + half] * t.y);
        } else if (e < a.rotary) {
            const float2 t = cs[e - half];
            x[i] = x[i] * t.x + sign * (mine[e - half] * t.y);
        }
    }
}

__device__ __forceinline__ void token_angles(const RopeArgs &a, int position, float2 *cs) {
    for (int i = threadIdx.x; i < a.rotary / 2; i += kThreads) {
        const uint64_t turn = (uint64_t)(int64_t)position * a.turns[i];
        float s, c;
        sincospif((float)(int32_t)(turn >> 32) * 0x1p-31f, &s, &c);
        cs[i] = make_float2(c * a.gain, s * a.gain);
    }
}

template <typename T, int kLanes>
__global__ void __launch_bounds__(kThreads) rope_kernel(const RopeArgs a) {
    __shared__ float2 cs[128];
    __shared__ float rows[kWarps][256];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int sub = lane / kLanes, first = (lane % kLanes) * 8;
    const bool live = first < a.dim;
    const int total = a.heads + 2 * a.kv_heads;
    float wq[8], wk[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) wq[i] = wk[i] = 1.0f;
    if (a.norm && live) {
        load8(static_cast<const T *>(a.q_weight) + first, wq);
        load8(static_cast<const T *>(a.k_weight) + first, wk);
    }
    for (int token = blockIdx.x; token < a.batch * a.seq; token += gridDim.x) {
        const int b = token / a.seq, t = token - b * a.seq;
        const int start = a.starts ? a.starts[b] : 0;
        if (start < 0 || start > a.rows - a.seq) {
            if (threadIdx.x == 0) atomicCAS(a.err, 0, kErrCacheLength);
            continue;
        }
        __syncthreads();
        token_angles(a, a.positions[token], cs);
        __syncthreads();
        for (int h0 = warp * (32 / kLanes); h0 < total; h0 += kWarps * (32 / kLanes)) {
            const int h = h0 + sub;
            const bool on = live && h < total;
            float x[8] = {};
            if (on) load8(static_cast<const T *>(a.qkv) + ((size_t)token * total + h) * a.dim + first, x);
            if (h0 < a.heads + a.kv_heads) {  // some row of the warp is a query or a key
                float y[8], scale = 1.0f;
                if (a.norm) {
                    float ss = 0.0f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
                    scale = rsqrtf(row_sum<kLanes>(ss) / (float)a.dim + a.epsilon);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = x[i] * scale * (h < a.heads ? wq[i] : wk[i]);
                turn8<kLanes>(a, cs, rows[warp], sub, first, 1.0f, y);
                if (h < a.heads + a.kv_heads)
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = y[i];
            }
            if (!on) continue;
            T *out;
            if (h < a.heads) out = static_cast<T *>(a.q) + (((size_t)b * a.heads + h) * a.seq + t) * a.dim;
            else {
                const bool key = h < a.heads + a.kv_heads;
                const int hk = h - a.heads - (key ? 0 : a.kv_heads);
                out = static_cast<T *>(key ? a.k : a.v) + (((size_t)b * a.kv_heads + hk) * a.rows + start + t) * a.dim;
            }
            store8(out + first, x);
        }
    }
}

template <typename T, int kLanes>
__global__ void __launch_bounds__(kThreads) rope_grad_kernel(const RopeArgs a) {
    __shared__ float2 cs[128];
    __shared__ float rows[kWarps][256];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int sub = lane / kLanes, first = (lane % kLanes) * 8;
    const bool live = first < a.dim;
    const int total = a.heads + 2 * a.kv_heads;
    float wq[8], wk[8], dwq[8] = {}, dwk[8] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i) wq[i] = wk[i] = 1.0f;
    if (a.norm && live) {
        load8(static_cast<const T *>(a.q_weight) + first, wq);
        load8(static_cast<const T *>(a.k_weight) + first, wk);
    }
    for (int token = blockIdx.x; token < a.batch * a.seq; token += gridDim.x) {
        const int b = token / a.seq, t = token - b * a.seq;
        __syncthreads();
        token_angles(a, a.positions[token], cs);
        __syncthreads();
        for (int h0 = warp * (32 / kLanes); h0 < total; h0 += kWarps * (32 / kLanes)) {
            const int h = h0 + sub;
            const bool on = live && h < total, query = h < a.heads, value = h >= a.heads + a.kv_heads;
            const size_t at = ((size_t)token * total + h) * a.dim + first;
            float g[8] = {};
            if (on) {
                const void *from = query ? a.q : value ? a.v : a.k;
                const int heads = query ? a.heads : a.kv_heads, index = query ? h : h - a.heads - (value ? a.kv_heads : 0);
                load8(static_cast<const T *>(from) + (((size_t)b * heads + index) * a.seq + t) * a.dim + first, g);
            }
            if (h0 < a.heads + a.kv_heads) {
                float d[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] = g[i];
                turn8<kLanes>(a, cs, rows[warp], sub, first, -1.0f, d);
                if (a.norm) {
                    float x[8] = {}, ss = 0.0f, ux = 0.0f;
                    if (on && !value) load8(static_cast<const T *>(a.qkv) + at, x);
#pragma unroll
                    for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
                    const float scale = rsqrtf(row_sum<kLanes>(ss) / (float)a.dim + a.epsilon);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        x[i] *= scale;
                        if (on && query) dwq[i] = fmaf(d[i], x[i], dwq[i]);
                        if (on && !query && !value) dwk[i] = fmaf(d[i], x[i], dwk[i]);
                        d[i] *= query ? wq[i] : wk[i];
                        ux = fmaf(d[i], x[i], ux);
                    }
                    const float mean = row_sum<kLanes>(ux) / (float)a.dim;
#pragma unroll
                    for (int i = 0; i < 8; ++i) d[i] = scale * (d[i] - x[i] * mean);
                }
                if (!value)
#pragma unroll
                    for (int i = 0; i < 8; ++i) g[i] = d[i];
            }
            if (on) store8(static_cast<T *>(a.dqkv) + at, g);
        }
    }
    if (!a.norm) return;
    // the block's sums, rows of the warp first, then warps, each in a fixed order
    for (int which = 0; which < 2; ++which) {
        float(&dw)[8] = which ? dwk : dwq;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
            for (int o = kLanes; o < 32; o <<= 1) dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
            if (sub == 0 && live) rows[warp][first + i] = dw[i];
        }
        __syncthreads();
        for (int e = threadIdx.x; e < a.dim; e += kThreads) {
            float s = 0.0f;
            for (int w = 0; w < kWarps; ++w) s += rows[w][e];
            a.partial[((size_t)blockIdx.x * 2 + which) * a.dim + e] = s;
        }
    }
}

// Sums the blocks' partial weight gradients: 32 columns of [blocks][2 dim] a block,
// its 32 warps striding over the blocks, then over the warps' sums in order.
__global__ void __launch_bounds__(1024) rope_weight_grad_kernel(const float *partial, int blocks, int dim, float *dq, float *dk) {
    __shared__ float sums[32][33];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (col < 2 * dim)
        for (int i = warp; i < blocks; i += 32) s += partial[(size_t)i * 2 * dim + col];
    sums[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && col < 2 * dim) {
        s = 0.0f;
        for (int i = 0; i < 32; ++i) s += sums[i][lane];
        (col < dim ? dq : dk)[col < dim ? col : col - dim] = s;
    }
}

// theta_i / 2 pi as 0.64 fixed-point fractions of a turn.
std::vector<uint64_t> turn_fractions(const Spec &s) {
    const double pi = 3.14159265358979323846, factor = s.factor;
    double base = s.base;
    if (s.scaling == "ntk") base *= std::pow(factor, (double)s.rotary / (s.rotary - 2.0));
    std::vector<uint64_t> out(s.rotary / 2);
    for (size_t i = 0; i < out.size(); ++i) {
        double theta = std::pow(base, -2.0 * (double)i / s.rotary);
        if (s.scaling == "linear") theta /= factor;
        if (s.scaling == "yarn") {
            const double turns = s.original * theta / (2.0 * pi);
            const double kept = std::min(1.0, std::max(0.0, (turns - 1.0) / 31.0));
            theta = kept * theta + (1.0 - kept) * theta / factor;
        }
        out[i] = (uint64_t)std::ldexp(theta / (2.0 * pi), 64);
    }
    return out;
}

template <typename T, int kLanes>
LaunchFn rope_launch(Context *ctx, const Spec &s) {
    RopeArgs base{};
    base.batch = s.batch, base.seq = s.seq, base.heads = s.heads, base.kv_heads = s.kv_heads, base.dim = s.dim, base.rotary = s.rotary;
    base.interleaved = s.interleaved, base.norm = s.norm, base.rows = s.capacity ? s.capacity : s.seq;
    base.epsilon = s.epsilon;
    base.gain = s.scaling == "yarn" ? (float)(0.1 * std::log((double)s.factor) + 1.0) : 1.0f;
    base.err = ctx->err_dev;
    const bool grad = s.op == Op::QkNormRopeGrad, norm = s.norm, cached = s.capacity != 0;
    const int blocks = std::min<int>(s.batch * s.seq, ctx->sm_count * (grad ? 4 : 8)), dim = s.dim;
    // the frequencies, and behind them the gradient's partial sums
    const std::vector<uint64_t> turns = turn_fractions(s);
    const size_t table = (turns.size() * 8 + 255) / 256 * 256;
    auto ws = kernel_workspace(table + 256 + (grad ? (size_t)blocks * 2 * dim * 4 : 0), "rotation table and partial sums");
    if (!turns.empty() && cudaMemcpy(ws.get(), turns.data(), turns.size() * 8, cudaMemcpyHostToDevice) != cudaSuccess)
        throw IrError("cannot upload the rotation table");
    base.turns = static_cast<const uint64_t *>(ws.get());
    base.partial = reinterpret_cast<float *>(static_cast<char *>(ws.get()) + table);
    return [=, keep = ws](cudaStream_t st, void **b) {
        RopeArgs a = base;
        size_t i = 0;
        a.qkv = b[i++];
        if (norm) a.q_weight = b[i], a.k_weight = b[i + 1], i += 2;
        a.positions = static_cast<const int *>(b[i++]);
        if (cached) a.starts = static_cast<const int *>(b[i++]);
        a.q = b[i++], a.k = b[i++], a.v = b[i++];
        if (!grad) {
            rope_kernel<T, kLanes><<<blocks, kThreads, 0, st>>>(a);
            return cudaGetLastError();
        }
        a.dqkv = b[i++];
        rope_grad_kernel<T, kLanes><<<blocks, kThreads, 0, st>>>(a);
        if (norm)
            rope_weight_grad_kernel<<<(2 * dim + 31) / 32, 1024, 0, st>>>(a.partial, blocks, dim, static_cast<float *>(b[i]), static_cast<float *>(b[i + 1]));
        return cudaGetLastError();
    };
}

template <typename T>
LaunchFn rope_pick(Context *ctx, const Spec &s) {
    if (s.dim <= 64) return rope_launch<T, 8>(ctx, s);
    return s.dim <= 128 ? rope_launch<T, 16>(ctx, s) : rope_launch<T, 32>(ctx, s);
}

}  // namespace

LaunchFn make_qk_norm_rope(Context *ctx, const Spec &s, std::string &impl) {
    impl = std::string(spec_name(s)) + "_d" + std::to_string(s.dim) + "_" + dtype_name(s.dtype);
    if (s.dtype == DType::BF16) return rope_pick<__nv_bfloat16>(ctx, s);
    return s.dtype == DType::F16 ? rope_pick<__half>(ctx, s) : rope_pick<float>(ctx, s);
}

}  // namespace jade
