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
//
// Both kernels are bound by HBM (each row read and written once). A warp takes
// heads of one token, 32 / kLanes rows at a time, 8 elements a lane, and forms the
// token's sines and cosines once in registers for all of them; no block barrier, no
// shared memory in the loop. Rows of several rounds are loaded before the first is
// worked on, so that enough bytes are in flight.
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
    int batch, seq, heads, kv_heads, dim, rotary, norm, rows;  // rows: of k and v per head
    int parts;              // warps that share a token's heads
    float epsilon, gain;
    int *err;
};

// How a lane's 8 elements lie in the head and find their partners.
//   kHalves      rotated lanes hold 4 of the first half and their 4 partners of the
//                second, two pieces rotary / 2 apart (rotary a multiple of 8); the
//                others 8 in a row
//   kNeighbours  8 in a row, partners beside each other
//   kGeneral     8 in a row, partners through the warp's rows in shared memory
//                (halves of any length)
enum Pairing { kHalves, kNeighbours, kGeneral };

template <typename T>
struct Vec4;  // 4 elements as loaded
template <>
struct Vec4<float> { using type = float4; };
template <>
struct Vec4<__nv_bfloat16> { using type = uint2; };
template <>
struct Vec4<__half> { using type = uint2; };

__device__ __forceinline__ void widen(const float4 &u, float *x, float) { x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w; }
__device__ __forceinline__ void widen(const uint2 &u, float *x, __nv_bfloat16) {
    x[0] = __uint_as_float(u.x << 16), x[1] = __uint_as_float(u.x & 0xffff0000u);
    x[2] = __uint_as_float(u.y << 16), x[3] = __uint_as_float(u.y & 0xffff0000u);
}
__device__ __forceinline__ void widen(const uint2 &u, float *x, __half) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&u.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}
__device__ __forceinline__ float4 narrow(const float *x, float) { return make_float4(x[0], x[1], x[2], x[3]); }
__device__ __forceinline__ uint2 narrow(const float *x, __nv_bfloat16) { return make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])); }
__device__ __forceinline__ uint2 narrow(const float *x, __half) { return make_uint2(pack_f16(x[0], x[1]), pack_f16(x[2], x[3])); }

// A lane's elements of a row: 4 from offset a, 4 from offset b.
template <typename T>
struct Row8 {
    typename Vec4<T>::type lo, hi;
};
struct Place {
    int a, b;
    bool live;
};
template <typename T, Pairing kPair>
__device__ __forceinline__ Row8<T> load_row(const T *p, Place at) {
    using V = typename Vec4<T>::type;
    Row8<T> r{};
    if (!at.live) return r;
    if constexpr (kPair != kHalves && sizeof(T) == 2) {
        const uint4 u = __ldcs(reinterpret_cast<const uint4 *>(p + at.a));
        r.lo = make_uint2(u.x, u.y), r.hi = make_uint2(u.z, u.w);
    } else {
        r.lo = __ldcs(reinterpret_cast<const V *>(p + at.a)), r.hi = __ldcs(reinterpret_cast<const V *>(p + at.b));
    }
    return r;
}
template <typename T, Pairing kPair>
__device__ __forceinline__ void store_row(T *p, Place at, const Row8<T> &r) {
    using V = typename Vec4<T>::type;
    if (!at.live) return;
    if constexpr (kPair != kHalves && sizeof(T) == 2) {
        *reinterpret_cast<uint4 *>(p + at.a) = make_uint4(r.lo.x, r.lo.y, r.hi.x, r.hi.y);
    } else {
        *reinterpret_cast<V *>(p + at.a) = r.lo;
        *reinterpret_cast<V *>(p + at.b) = r.hi;
    }
}
template <typename T>
__device__ __forceinline__ void widen8(const Row8<T> &r, float (&x)[8]) {
    widen(r.lo, x, T{});
    widen(r.hi, x + 4, T{});
}
template <typename T>
__device__ __forceinline__ Row8<T> narrow8(const float (&x)[8]) {
    return Row8<T>{narrow(x, T{}), narrow(x + 4, T{})};
}

template <Pairing kPair>
__device__ __forceinline__ Place lane_place(int chunk, int dim, int rotary) {
    Place at{8 * chunk, 8 * chunk + 4, 8 * chunk < dim};
    if (kPair == kHalves && 8 * chunk < rotary) at.a = 4 * chunk, at.b = 4 * chunk + rotary / 2;
    return at;
}

// Cosines and sines of the lane's pairs at a position; passed elements turn by 0.
// kGeneral: for each of its 8 elements, y = x c + partner s.
template <Pairing kPair>
struct Angles {
    static constexpr int kCount = kPair == kGeneral ? 8 : 4;
    float c[kCount], s[kCount];
    __device__ __forceinline__ void set(const RopeArgs &a, int chunk, int position, float sign) {
        const int half = a.rotary / 2;
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            const int e = kCount * chunk + i;  // pair, or element
            const int pair = kPair == kGeneral && e >= half ? e - half : e;
            c[i] = 1.0f, s[i] = 0.0f;
            if (pair < half) {
                const uint64_t turn = (uint64_t)(int64_t)position * __ldg(a.turns + pair);
                sincospif((float)(int32_t)(turn >> 32) * 0x1p-31f, &s[i], &c[i]);
                c[i] *= a.gain, s[i] *= kPair == kGeneral && e < half ? -sign * a.gain : sign * a.gain;
            }
        }
    }
    // x: the lane's elements; row: the warp row's elements in shared memory (kGeneral)
    __device__ __forceinline__ void turn(float (&x)[8], float *row, int chunk, int half) const {
        if constexpr (kPair == kHalves) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float u = x[i] * c[i] - x[4 + i] * s[i];
                x[4 + i] = x[i] * s[i] + x[4 + i] * c[i];
                x[i] = u;
            }
        } else if constexpr (kPair == kNeighbours) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float u = x[2 * i] * c[i] - x[2 * i + 1] * s[i];
                x[2 * i + 1] = x[2 * i] * s[i] + x[2 * i + 1] * c[i];
                x[2 * i] = u;
            }
        } else {
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) row[8 * chunk + i] = x[i];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = 8 * chunk + i;
                if (e < 2 * half) x[i] = x[i] * c[i] + row[e < half ? e + half : e - half] * s[i];
            }
        }
    }
};

// Sum over the kLanes lanes of a row.
template <int kLanes>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The rounds of a warp: a token's heads in the order queries, keys, values, 32 /
// kLanes heads of one kind a round, the rounds of a token dealt evenly to its `parts`
// warps.
template <int kLanes>
struct Rounds {
    int q, k, total;  // rounds of queries, of queries and keys, of all
    __device__ __forceinline__ Rounds(const RopeArgs &a) {
        constexpr int per = 32 / kLanes;
        q = (a.heads + per - 1) / per;
        k = q + (a.kv_heads + per - 1) / per;
        total = k + k - q;
    }
};

template <typename T, int kLanes, Pairing kPair>
__global__ void __launch_bounds__(kThreads, 4) rope_kernel(const RopeArgs a) {
    constexpr int kPer = 32 / kLanes, kAhead = 4;  // rounds loaded at a time
    __shared__ float shared_rows[kPair == kGeneral ? kWarps : 1][256];
    const int lane = threadIdx.x & 31, sub = lane / kLanes, chunk = lane % kLanes;
    const Place at = lane_place<kPair>(chunk, a.dim, a.rotary);
    const Rounds<kLanes> rounds(a);
    const int total_heads = a.heads + 2 * a.kv_heads;
    float *row = shared_rows[kPair == kGeneral ? threadIdx.x >> 5 : 0] + sub * (kLanes * 8);
    const long long items = (long long)a.batch * a.seq * a.parts;
    for (long long item = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5); item < items; item += (long long)gridDim.x * kWarps) {
        const int token = (int)(item / a.parts), part = (int)(item - (long long)token * a.parts);
        const int b = token / a.seq, t = token - b * a.seq;
        const int r0 = (int)((long long)rounds.total * part / a.parts), r1 = (int)((long long)rounds.total * (part + 1) / a.parts);
        const int start = a.starts ? __ldg(a.starts + b) : 0, position = __ldg(a.positions + token);
        if (start < 0 || start > a.rows - a.seq) {
            if (lane == 0) atomicCAS(a.err, 0, kErrCacheLength);
            continue;
        }
        const T *in = static_cast<const T *>(a.qkv) + (size_t)token * total_heads * a.dim;
        // head of the packed row and its destination in round r; -1 where the round has no head for this lane
        auto head_of = [&](int r, T *&out) {
            int h;
            if (r < rounds.q) {
                h = r * kPer + sub;
                out = static_cast<T *>(a.q) + (((size_t)b * a.heads + h) * a.seq + t) * a.dim;
                return h < a.heads ? h : -1;
            }
            const bool key = r < rounds.k;
            h = (r - (key ? rounds.q : rounds.k)) * kPer + sub;
            out = static_cast<T *>(key ? a.k : a.v) + (((size_t)b * a.kv_heads + h) * a.rows + start + t) * a.dim;
            return h < a.kv_heads ? a.heads + (key ? 0 : a.kv_heads) + h : -1;
        };
        Angles<kPair> angles;
        float w[8];
        int weights = -1;  // whose weights w holds: 0 queries, 1 keys
        for (int r = r0; r < r1; r += kAhead) {
            Row8<T> x[kAhead];
            T *out[kAhead];
            bool on[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int h = head_of(min(r + u, r1 - 1), out[u]);
                on[u] = h >= 0 && r + u < r1;
                x[u] = load_row<T, kPair>(in + (size_t)max(h, 0) * a.dim, Place{at.a, at.b, at.live && on[u]});
            }
            if (r == r0 && r < rounds.k) angles.set(a, chunk, position, 1.0f);
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (r + u >= r1) break;
                if (r + u < rounds.k) {  // a query or a key
                    const int kind = r + u < rounds.q ? 0 : 1;
                    if (a.norm && kind != weights) {
                        weights = kind;
                        widen8(load_row<T, kPair>(static_cast<const T *>(kind ? a.k_weight : a.q_weight), at), w);
                    }
                    float y[8];
                    widen8(x[u], y);
                    if (a.norm) {
                        float ss = 0.0f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) ss = fmaf(y[i], y[i], ss);
                        const float scale = rsqrtf(row_sum<kLanes>(ss) / (float)a.dim + a.epsilon);
#pragma unroll
                        for (int i = 0; i < 8; ++i) y[i] *= scale * w[i];
                    }
                    angles.turn(y, row, chunk, a.rotary / 2);
                    x[u] = narrow8<T>(y);
                }
                store_row<T, kPair>(out[u], Place{at.a, at.b, at.live && on[u]}, x[u]);
            }
        }
    }
}

template <typename T, int kLanes, Pairing kPair>
__global__ void __launch_bounds__(kThreads, 2) rope_grad_kernel(const RopeArgs a) {
    constexpr int kPer = 32 / kLanes, kAhead = 4;
    __shared__ float shared_rows[kWarps][256];
    const int lane = threadIdx.x & 31, sub = lane / kLanes, chunk = lane % kLanes;
    const Place at = lane_place<kPair>(chunk, a.dim, a.rotary);
    const Rounds<kLanes> rounds(a);
    const int total_heads = a.heads + 2 * a.kv_heads;
    float *row = shared_rows[threadIdx.x >> 5] + sub * (kLanes * 8);
    float wq[8], wk[8], dwq[8] = {}, dwk[8] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i) wq[i] = wk[i] = 1.0f;
    if (a.norm) {
        widen8(load_row<T, kPair>(static_cast<const T *>(a.q_weight), at), wq);
        widen8(load_row<T, kPair>(static_cast<const T *>(a.k_weight), at), wk);
    }
    const long long items = (long long)a.batch * a.seq * a.parts;
    for (long long item = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5); item < items; item += (long long)gridDim.x * kWarps) {
        const int token = (int)(item / a.parts), part = (int)(item - (long long)token * a.parts);
        const int b = token / a.seq, t = token - b * a.seq;
        const int r0 = (int)((long long)rounds.total * part / a.parts), r1 = (int)((long long)rounds.total * (part + 1) / a.parts);
        const int position = __ldg(a.positions + token);
        const size_t packed = (size_t)token * total_heads * a.dim;
        Angles<kPair> angles;
        for (int r = r0; r < r1; r += kAhead) {
            Row8<T> g[kAhead], x[kAhead];
            size_t to[kAhead];
            bool on[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int rr = min(r + u, r1 - 1), kind = rr < rounds.q ? 0 : rr < rounds.k ? 1 : 2;
                const int h = (rr - (kind == 0 ? 0 : kind == 1 ? rounds.q : rounds.k)) * kPer + sub, heads = kind ? a.kv_heads : a.heads;
                on[u] = h < heads && r + u < r1;
                const Place here{at.a, at.b, at.live && on[u]};
                const T *from = static_cast<const T *>(kind == 0 ? a.q : kind == 1 ? a.k : a.v);
                to[u] = packed + (size_t)(h + (kind == 0 ? 0 : kind == 1 ? a.heads : a.heads + a.kv_heads)) * a.dim;
                g[u] = load_row<T, kPair>(from + (((size_t)b * heads + h) * a.seq + t) * a.dim, here);
                if (a.norm && kind < 2) x[u] = load_row<T, kPair>(static_cast<const T *>(a.qkv) + to[u], here);
            }
            if (r == r0 && r < rounds.k) angles.set(a, chunk, position, -1.0f);
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (r + u >= r1) break;
                if (r + u < rounds.k) {
                    const bool query = r + u < rounds.q;
                    float d[8];
                    widen8(g[u], d);
                    angles.turn(d, row, chunk, a.rotary / 2);
                    if (a.norm) {
                        float y[8], ss = 0.0f, ux = 0.0f;
                        widen8(x[u], y);
#pragma unroll
                        for (int i = 0; i < 8; ++i) ss = fmaf(y[i], y[i], ss);
                        const float scale = rsqrtf(row_sum<kLanes>(ss) / (float)a.dim + a.epsilon);
                        if (query) {  // lanes without a row hold zeros
#pragma unroll
                            for (int i = 0; i < 8; ++i) y[i] *= scale, dwq[i] = fmaf(d[i], y[i], dwq[i]), d[i] *= wq[i], ux = fmaf(d[i], y[i], ux);
                        } else {
#pragma unroll
                            for (int i = 0; i < 8; ++i) y[i] *= scale, dwk[i] = fmaf(d[i], y[i], dwk[i]), d[i] *= wk[i], ux = fmaf(d[i], y[i], ux);
                        }
                        const float mean = row_sum<kLanes>(ux) / (float)a.dim;
#pragma unroll
                        for (int i = 0; i < 8; ++i) d[i] = scale * (d[i] - y[i] * mean);
                    }
                    g[u] = narrow8<T>(d);
                }
                store_row<T, kPair>(static_cast<T *>(a.dqkv) + to[u], Place{at.a, at.b, at.live && on[u]}, g[u]);
            }
        }
    }
    if (!a.norm) return;
    // the block's sums: rows of the warp first, then the warps, each in a fixed order
    for (int which = 0; which < 2; ++which) {
        float(&dw)[8] = which ? dwk : dwq;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
            for (int o = kLanes; o < 32; o <<= 1) dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
            if (sub == 0 && at.live) shared_rows[threadIdx.x >> 5][(i < 4 ? at.a : at.b) + (i & 3)] = dw[i];
        }
        __syncthreads();
        for (int e = threadIdx.x; e < a.dim; e += kThreads) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) s += shared_rows[w][e];
            a.partial[((size_t)blockIdx.x * 2 + which) * a.dim + e] = s;
        }
    }
}

// Sums the blocks' partial weight gradients: 32 columns of [blocks][2 dim] a block,
// its 32 warps striding over the blocks, then over the warps' sums in order.
__global__ void __launch_bounds__(1024) rope_weight_grad_kernel(const float *partial, int blocks, int dim, float *dq, float *dk) {
    __shared__ float sums[32][33];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = blockIdx.x * 32 + lane;
    grid_dependency_wait();
    float s = 0.0f;
    if (col < 2 * dim) {
#pragma unroll 8
        for (int i = warp; i < blocks; i += 32) s += partial[(size_t)i * 2 * dim + col];
    }
    sums[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && col < 2 * dim) {
        s = 0.0f;
#pragma unroll
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

template <typename T, int kLanes, Pairing kPair>
LaunchFn rope_launch(Context *ctx, const Spec &s) {
    RopeArgs base{};
    base.batch = s.batch, base.seq = s.seq, base.heads = s.heads, base.kv_heads = s.kv_heads, base.dim = s.dim, base.rotary = s.rotary;
    base.norm = s.norm, base.rows = s.capacity ? s.capacity : s.seq;
    base.epsilon = s.epsilon;
    base.gain = s.scaling == "yarn" ? (float)(0.1 * std::log((double)s.factor) + 1.0) : 1.0f;
    base.err = ctx->err_dev;
    const bool grad = s.op == Op::QkNormRopeGrad, norm = s.norm, cached = s.capacity != 0;
    // Resident warps get one token each where there are as many; fewer tokens share
    // theirs among warps, down to one round of rows a warp.
    const long long tokens = (long long)s.batch * s.seq, resident = (long long)ctx->sm_count * kWarps * (grad ? 2 : 4);
    const int per = 32 / kLanes, rounds = (int)((s.heads + per - 1) / per + 2 * ((s.kv_heads + per - 1) / per));
    base.parts = (int)std::max(1ll, std::min<long long>(rounds, resident / tokens));
    const int blocks = (int)std::min((tokens * base.parts + kWarps - 1) / kWarps, grad ? resident / kWarps : 1ll << 30), dim = s.dim;
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
            rope_kernel<T, kLanes, kPair><<<blocks, kThreads, 0, st>>>(a);
            return cudaGetLastError();
        }
        a.dqkv = b[i++];
        rope_grad_kernel<T, kLanes, kPair><<<blocks, kThreads, 0, st>>>(a);
        if (!norm) return cudaGetLastError();
        const cudaError_t e = launch_after(st, rope_weight_grad_kernel, (2 * dim + 31) / 32, 1024, 0, static_cast<const float *>(a.partial), blocks,
                                           dim, static_cast<float *>(b[i]), static_cast<float *>(b[i + 1]));
        return e == cudaSuccess ? cudaGetLastError() : e;
    };
}

template <typename T, Pairing kPair>
LaunchFn rope_lanes(Context *ctx, const Spec &s) {
    if (s.dim <= 64) return rope_launch<T, 8, kPair>(ctx, s);
    return s.dim <= 128 ? rope_launch<T, 16, kPair>(ctx, s) : rope_launch<T, 32, kPair>(ctx, s);
}
template <typename T>
LaunchFn rope_pick(Context *ctx, const Spec &s) {
    if (s.interleaved) return rope_lanes<T, kNeighbours>(ctx, s);
    return s.rotary % 8 == 0 ? rope_lanes<T, kHalves>(ctx, s) : rope_lanes<T, kGeneral>(ctx, s);
}

}  // namespace

LaunchFn make_qk_norm_rope(Context *ctx, const Spec &s, std::string &impl) {
    impl = std::string(spec_name(s)) + "_d" + std::to_string(s.dim) + "_" + dtype_name(s.dtype);
    if (s.dtype == DType::BF16) return rope_pick<__nv_bfloat16>(ctx, s);
    return s.dtype == DType::F16 ? rope_pick<__half>(ctx, s) : rope_pick<float>(ctx, s);
}

}  // namespace jade
