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
// Both kernels are bound by HBM (each row read and written once), with the issue rate
// close behind: 16 elements a lane, 32 / kLanes rows a warp (a round), packed FP32x2
// arithmetic. A persistent warp walks over items, a token's heads or a part of them, and
// forms the token's sines and cosines once, a few a lane, in shared memory. While it works
// on a step of rounds, the next step's rows, of the next item where this one ends, come by
// asynchronous copies. Angles and norm weights are read from shared memory for every
// round: registers hold one round's rows only, so that enough warps are resident. No block
// barrier per token, so that warps drift apart and memory stays busy. Measured on B200, BF16, 4 x 2048 tokens of 16 + 2 x 16
// heads of 128 (201 MB moved; a plain copy of them takes 36 us): 41 us = 4.9 TB/s with
// halves, 41 with neighbours, 52 with a rotary that is no multiple of 16; the gradient (268
// MB) 59, 60 and 67 us = 4.6 TB/s. With rows loaded to registers: 43, 45 and 51, 64, 71 and
// 83. One token: 4.4 us.
#include <climits>
#include <cmath>
#include <type_traits>
#include <vector>

#include "attention_softmax.cuh"
#include "common.cuh"
#include "internal.hpp"

namespace jade {
namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;

struct RopeArgs {
    const void *qkv, *q_weight, *k_weight;
    const int *positions, *starts;
    const uint64_t *turns;  // theta / 2 pi as 0.64 fractions, rotary / 2 of them
    void *q, *k, *v;        // outputs (gradient: dq, dk, dv, inputs)
    void *dqkv;
    float *partial;         // gradient: [block][2][dim] sums of the norm weights' gradients
    int batch, seq, heads, kv_heads, dim, rotary, norm, rows;  // rows: of k and v per head
    int parts;              // warps that share a token's heads
    float epsilon, gain, inv_dim;
    int *err;
};

// How a lane's 16 elements, two pieces of 8, lie in the head and find their partners.
//   kHalves      rotated lanes hold 8 of the first half and their 8 partners of the
//                second, rotary / 2 apart (rotary a multiple of 16); the others the
//                same of the rest
//   kNeighbours  16 in a row, partners beside each other
//   kGeneral     16 in a row, partners through the warp's rows in shared memory
//                (halves of any length)
enum Pairing { kHalves, kNeighbours, kGeneral };

struct Place {
    int lo, hi;            // offsets of the pieces in the head
    bool has_lo, has_hi;   // the head has them
};
template <Pairing kPair>
__device__ __forceinline__ Place lane_place(int chunk, int dim, int rotary) {
    Place at{16 * chunk, 16 * chunk + 8, 16 * chunk < dim, 16 * chunk + 8 < dim};
    if (kPair == kHalves) {
        const bool turns = 16 * chunk < rotary;
        const int i = turns ? chunk : chunk - rotary / 16, lanes = turns ? rotary / 16 : ((dim - rotary) / 8 + 1) / 2;
        at.lo = (turns ? 0 : rotary) + 8 * i, at.hi = at.lo + 8 * lanes;
        at.has_lo = i < lanes, at.has_hi = at.has_lo && at.hi < dim;
    }
    return at;
}

// Pieces as they are loaded and stored, and as four pairs of FP32 each.
template <typename T>
struct Piece { uint4 u; };
template <>
struct Piece<float> { float4 a, b; };

__device__ __forceinline__ void store_piece(float *p, const Piece<float> &x) {
    reinterpret_cast<float4 *>(p)[0] = x.a;
    reinterpret_cast<float4 *>(p)[1] = x.b;
}
template <typename T>
__device__ __forceinline__ void store_piece(T *p, const Piece<T> &x) { *reinterpret_cast<uint4 *>(p) = x.u; }

__device__ __forceinline__ void widen(const Piece<float> &x, uint64_t *v) {
    v[0] = pack2f(x.a.x, x.a.y), v[1] = pack2f(x.a.z, x.a.w), v[2] = pack2f(x.b.x, x.b.y), v[3] = pack2f(x.b.z, x.b.w);
}
__device__ __forceinline__ void widen(const Piece<__nv_bfloat16> &x, uint64_t *v) {
    const uint32_t w[4] = {x.u.x, x.u.y, x.u.z, x.u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = pack2f(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
__device__ __forceinline__ void widen(const Piece<__half> &x, uint64_t *v) {
    const uint32_t w[4] = {x.u.x, x.u.y, x.u.z, x.u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        v[i] = pack2f(f.x, f.y);
    }
}
__device__ __forceinline__ void narrow(Piece<float> &x, const uint64_t *v) {
    unpack2f(v[0], x.a.x, x.a.y), unpack2f(v[1], x.a.z, x.a.w), unpack2f(v[2], x.b.x, x.b.y), unpack2f(v[3], x.b.z, x.b.w);
}
template <typename T>
__device__ __forceinline__ void narrow(Piece<T> &x, const uint64_t *v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a, b;
        unpack2f(v[i], a, b);
        w[i] = std::is_same<T, __nv_bfloat16>::value ? pack_bf16(a, b) : pack_f16(a, b);
    }
    x.u = make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T>
struct Row {  // a lane's share of a head
    Piece<T> lo, hi;
    __device__ __forceinline__ void store(T *p, const Place &at, bool on) const {
        if (on && at.has_lo) store_piece(p + at.lo, lo);
        if (on && at.has_hi) store_piece(p + at.hi, hi);
    }
};

// A round's rows on their way through shared memory, in units of 16 bytes that leave
// memory in whole sectors. A piece of kHalves in 16 bits is a unit whose neighbours lie
// beside it: every lane copies its own. Else the lanes of a row copy its units in turn;
// unit n is kept at n ^ (n / 8 mod kUnits), clear of bank conflicts.
template <typename T, int kLanes, Pairing kPair>
struct Staged {
    static constexpr int kUnits = 2 * sizeof(Piece<T>) / 16, kEach = 16 / sizeof(T);
    static constexpr bool kOwn = kPair == kHalves && sizeof(T) == 2;
    static __device__ __forceinline__ int slot(int lane, int n) { return lane / kLanes * (kLanes * kUnits) + (n ^ (n >> 3 & (kUnits - 1))); }
    static __device__ __forceinline__ void copy(uint4 *to, const T *p, const Place &at, bool on, int lane, int dim) {
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const int n = lane % kLanes + kLanes * i;
            const bool has = on && (kOwn ? (i ? at.has_hi : at.has_lo) : n * kEach < dim);
            const int from = kOwn ? (i ? at.hi : at.lo) : n * kEach;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to + (kOwn ? 32 * i + lane : slot(lane, n)))),
                         "l"(p + (has ? from : 0)), "r"(has ? 16 : 0)
                         : "memory");
        }
    }
    // zeros where the lane has no piece
    static __device__ __forceinline__ Row<T> take(const uint4 *from, const Place &at, int lane) {
        uint4 x[kUnits];
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const bool hi = i >= kUnits / 2;
            if (kOwn) x[i] = from[32 * i + lane];
            else {
                x[i] = make_uint4(0, 0, 0, 0);
                if (hi ? at.has_hi : at.has_lo) x[i] = from[slot(lane, (hi ? at.hi : at.lo) / kEach + i % (kUnits / 2))];
            }
        }
        return {*reinterpret_cast<const Piece<T> *>(&x[0]), *reinterpret_cast<const Piece<T> *>(&x[kUnits / 2])};
    }
    // other lanes' copies have landed; the stage has been read by all
    static __device__ __forceinline__ void meet() {
        if (!kOwn) __syncwarp();
    }
};
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_wait_but_one() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }

__device__ __forceinline__ uint64_t both(float x) { return pack2f(x, x); }

// FP32 tables in shared memory without bank conflicts: entry e lies at table_at(e). Lanes
// read 8 in a row (kHalves: two 16-byte loads) or 16 (four).
constexpr int kTable = 256;
template <Pairing kPair>
__device__ __forceinline__ int table_at(int e) {
    return kPair == kHalves ? (e >> 2 & 1) * (kTable / 2) + (e >> 3) * 4 + (e & 3) : (e >> 2 & 3) * (kTable / 4) + (e >> 4) * 4 + (e & 3);
}
template <Pairing kPair>
__device__ __forceinline__ void table8(const float *table, int first, uint64_t *v) {
    const ulonglong2 a = *reinterpret_cast<const ulonglong2 *>(table + table_at<kPair>(first)), b = *reinterpret_cast<const ulonglong2 *>(table + table_at<kPair>(first + 4));
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
}

// A row's elements in shared memory (kGeneral): lanes write and read 16 in a row each,
// 17 words apart, so that no two meet in a bank (all rows of 16 words apart would: a
// forward pass of 201 MB took 88 us so).
__device__ __forceinline__ int row_at(int e) { return e + (e >> 4); }
constexpr int kZeroAt = 16;  // between two lanes' elements: 0

struct Elements {
    uint64_t v[8];
    template <typename T>
    __device__ __forceinline__ void from(const Row<T> &r) { widen(r.lo, v), widen(r.hi, v + 4); }
    template <typename T>
    __device__ __forceinline__ void to(Row<T> &r) const { narrow(r.lo, v), narrow(r.hi, v + 4); }
    // sum of the products with another row's elements
    __device__ __forceinline__ float dot(const Elements &o) const {
        uint64_t s[2] = {mul2(v[0], o.v[0]), mul2(v[1], o.v[1])};
#pragma unroll
        for (int i = 2; i < 8; ++i) s[i & 1] = fma2(v[i], o.v[i], s[i & 1]);
        float x, y;
        unpack2f(add2(s[0], s[1]), x, y);
        return x + y;
    }
};

// The token's cosines and sines, formed by the warp in its shared memory as the
// pairing multiplies them; kBack turns back.
//   kHalves  a = c, b = s, n = -s of each pair
//   else     x' = x a + (x with its pairs swapped) b, of each element: a = c, b = -s or s
template <int kLanes, Pairing kPair, bool kBack>
struct Turn {
    float *a, *b, *n;
    __device__ __forceinline__ explicit Turn(float *tables) : a(tables), b(tables + kTable), n(tables + 2 * kTable) {}
    static constexpr int kFloats = (kPair == kHalves ? 3 : 2) * kTable;
    __device__ __forceinline__ void form(const RopeArgs &args, int position, int lane) {
        __syncwarp();  // the last token's have been read
        for (int i = lane; i < 8 * kLanes; i += 32) {
            float c = 1.0f, s = 0.0f;  // passed elements, and beyond the head: lanes read whole pieces
            if (i < args.rotary / 2) {
                const uint64_t turn = (uint64_t)(int64_t)position * __ldg(args.turns + i);
                sincospif((float)(int32_t)(turn >> 32) * 0x1p-31f, &s, &c);
                c *= args.gain, s *= kBack ? -args.gain : args.gain;
            }
            if constexpr (kPair == kNeighbours) {
                *reinterpret_cast<float2 *>(a + table_at<kPair>(2 * i)) = make_float2(c, c);
                *reinterpret_cast<float2 *>(b + table_at<kPair>(2 * i)) = make_float2(-s, s);
            } else if constexpr (kPair == kHalves) {
                a[table_at<kPair>(i)] = c, b[table_at<kPair>(i)] = s, n[table_at<kPair>(i)] = -s;
            } else {  // i beyond the pairs: two of the elements that pass
                const int half = args.rotary / 2, e = i < half ? i : 2 * i, pair = i < half ? i + half : 2 * i + 1;
                a[table_at<kPair>(e)] = c, b[table_at<kPair>(e)] = -s, a[table_at<kPair>(pair)] = c, b[table_at<kPair>(pair)] = s;
            }
        }
        __syncwarp();
    }
    // row, partners (kGeneral): the row's elements in shared memory, and where each
    // element's partner lies there. Elements that pass are not touched: a partner's
    // infinity times 0 would reach them.
    __device__ __forceinline__ void apply(Elements &x, float *row, const int *partners, int chunk, int rotary) const {
        if constexpr (kPair == kHalves) {
            if (16 * chunk >= rotary) return;
            uint64_t c[4], s[4], m[4];
            table8<kPair>(a, 8 * chunk, c), table8<kPair>(b, 8 * chunk, s), table8<kPair>(n, 8 * chunk, m);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint64_t lo = x.v[i], hi = x.v[4 + i];
                x.v[i] = fma2(lo, c[i], mul2(hi, m[i]));
                x.v[4 + i] = fma2(hi, c[i], mul2(lo, s[i]));
            }
        } else if constexpr (kPair == kNeighbours) {
            uint64_t c[8], s[8];
            table8<kPair>(a, 16 * chunk, c), table8<kPair>(a, 16 * chunk + 8, c + 4), table8<kPair>(b, 16 * chunk, s), table8<kPair>(b, 16 * chunk + 8, s + 4);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float p, q;
                unpack2f(x.v[i], p, q);
                if (16 * chunk + 2 * i < rotary) x.v[i] = fma2(x.v[i], c[i], mul2(pack2f(q, p), s[i]));
            }
        } else {
            float y[16];
#pragma unroll
            for (int i = 0; i < 8; ++i) unpack2f(x.v[i], y[2 * i], y[2 * i + 1]);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 16; ++i) row[row_at(16 * chunk) + i] = y[i];
            __syncwarp();
            uint64_t c[8], s[8];
            table8<kPair>(a, 16 * chunk, c), table8<kPair>(a, 16 * chunk + 8, c + 4), table8<kPair>(b, 16 * chunk, s), table8<kPair>(b, 16 * chunk + 8, s + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int4 at = *reinterpret_cast<const int4 *>(partners + table_at<kPair>(16 * chunk + 4 * i));
                x.v[2 * i] = fma2(x.v[2 * i], c[2 * i], mul2(pack2f(row[at.x], row[at.y]), s[2 * i]));
                x.v[2 * i + 1] = fma2(x.v[2 * i + 1], c[2 * i + 1], mul2(pack2f(row[at.z], row[at.w]), s[2 * i + 1]));
            }
        }
    }
};

// Where each element's partner lies in a row; a zero for those that pass (whole block; a
// barrier is due before its use).
template <Pairing kPair>
__device__ __forceinline__ void partner_table(const RopeArgs &a, int *partners) {
    for (int e = threadIdx.x; e < kTable; e += kThreads) {
        const int half = a.rotary / 2;
        partners[table_at<kPair>(e)] = e < 2 * half ? row_at(e < half ? e + half : e - half) : kZeroAt;
    }
}

// The norm weights of queries and keys as tables (whole block; a barrier is due before their use).
template <typename T, Pairing kPair>
__device__ __forceinline__ void weight_tables(const RopeArgs &a, float (*w)[kTable]) {
    if (!a.norm) return;
    for (int e = threadIdx.x; e < kTable; e += kThreads) {  // 0 beyond the head: lanes read whole pieces
        w[0][table_at<kPair>(e)] = e < a.dim ? to_f32<T>(static_cast<const T *>(a.q_weight)[e]) : 0.0f;
        w[1][table_at<kPair>(e)] = e < a.dim ? to_f32<T>(static_cast<const T *>(a.k_weight)[e]) : 0.0f;
    }
}
template <Pairing kPair>
__device__ __forceinline__ void load_weights(Elements &w, const float *table, const Place &at) {
    table8<kPair>(table, at.lo, w.v);
    table8<kPair>(table, at.hi & (kTable - 1), w.v + 4);  // a piece that the head lacks is not stored
}

// Sum over the kLanes lanes of a row.
template <int kLanes>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Rounds of a token: its heads in the order queries, keys, values, 32 / kLanes heads
// of one kind a round; dealt evenly to the token's `parts` warps.
__host__ __device__ constexpr int rounds_of(int heads, int per) { return (heads + per - 1) / per; }
template <int kLanes>
struct Rounds {
    static constexpr int kPer = 32 / kLanes;
    int q, k, total;  // rounds of queries, of queries and keys, of all
    __device__ __forceinline__ Rounds(const RopeArgs &a) {
        q = rounds_of(a.heads, kPer), k = q + rounds_of(a.kv_heads, kPer);
        total = k + k - q;
    }
    // kind (0 queries, 1 keys, 2 values) of round r and the lane's head of it; false: it has none
    __device__ __forceinline__ bool at(const RopeArgs &a, int r, int sub, int &kind, int &h) const {
        kind = r < q ? 0 : r < k ? 1 : 2;
        h = (r - (kind == 0 ? 0 : kind == 1 ? q : k)) * kPer + sub;
        return h < (kind ? a.kv_heads : a.heads);
    }
};

// 16-byte pieces of a lane and step: two rounds in 16 bits (four: 42.7 us for 41.0), one in 32
constexpr int kForwardUnits = 4;
constexpr int kForwardStaged = kWarps * 2 * kForwardUnits * 32 * 16;

template <typename T, int kLanes, Pairing kPair>
__global__ void __launch_bounds__(kThreads, 5) rope_kernel(const RopeArgs a) {
    using Stage = Staged<T, kLanes, kPair>;
    constexpr int kUnits = Stage::kUnits, kStep = kForwardUnits / kUnits;  // rounds of a step
    extern __shared__ uint4 staged[];
    __shared__ __align__(16) float tables[kWarps][Turn<kLanes, kPair, false>::kFloats];
    __shared__ __align__(16) float weights[2][kTable];
    __shared__ float shared_rows[kPair == kGeneral ? kWarps : 1][32 * 17];
    __shared__ __align__(16) int partners[kPair == kGeneral ? kTable : 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / kLanes, chunk = lane % kLanes;
    const Place at = lane_place<kPair>(chunk, a.dim, a.rotary);
    const Rounds<kLanes> rounds(a);
    float *row = shared_rows[kPair == kGeneral ? warp : 0] + sub * (kLanes * 17);
    Turn<kLanes, kPair, false> turn(tables[warp]);
    weight_tables<T, kPair>(a, weights);
    if constexpr (kPair == kGeneral) {
        partner_table<kPair>(a, partners);
        if (chunk == 0) row[kZeroAt] = 0.0f;
    }
    __syncthreads();
    const int q_step = a.seq * a.dim, items = a.batch * a.seq * a.parts;
    const long long kv_step = (long long)a.rows * a.dim;
    // the next step: its item, rounds r .. of r1, and the rows of its token
    int item = blockIdx.x * kWarps + warp, r = 0, r1 = 0, position = 0, start = 0, token = 0, stage = 0;
    auto open = [&] {
        token = item / a.parts;
        const int part = item - token * a.parts;
        r = rounds.total * part / a.parts, r1 = rounds.total * (part + 1) / a.parts;
        position = __ldg(a.positions + token);
        start = a.starts ? __ldg(a.starts + token / a.seq) : 0;
    };
    auto pieces = [&](int stage, int u) { return staged + ((warp * 2 + stage) * kForwardUnits + kUnits * u) * 32; };
    auto copy = [&](int stage) {
        const T *in = static_cast<const T *>(a.qkv) + (size_t)token * (a.heads + 2 * a.kv_heads) * a.dim;
#pragma unroll
        for (int u = 0; u < kStep; ++u) {
            int kind, h;
            const bool on = rounds.at(a, r + u, sub, kind, h) && r + u < r1;
            Stage::copy(pieces(stage, u), in + (on ? ((kind == 0 ? 0 : kind == 1 ? a.heads : a.heads + a.kv_heads) + h) * a.dim : 0), at, on, lane, a.dim);
        }
        copies_commit();
    };
    bool more = item < items, fresh = true;
    if (more) open(), copy(0);
    while (more) {
        const int now = r, end = r1, angle = position, slot0 = start, b = token / a.seq, t = token - b * a.seq;
        const bool first = fresh;
        r += kStep, fresh = r >= r1;
        if (fresh) {
            item += gridDim.x * kWarps, more = item < items;
            if (more) open();
        }
        if (more) copy(stage ^ 1);
        else copies_commit();
        const bool fits = slot0 >= 0 && slot0 <= a.rows - a.seq;
        if (!fits && lane == 0) atomicCAS(a.err, 0, kErrCacheLength);
        if (first && now < rounds.k) turn.form(a, angle, lane);
        T *q = static_cast<T *>(a.q) + ((size_t)b * a.heads * a.seq + t) * a.dim;
        const size_t slot = ((size_t)b * a.kv_heads * a.rows + slot0 + t) * a.dim;
        copies_wait_but_one();
        Stage::meet();
#pragma unroll
        for (int u = 0; u < kStep; ++u) {
            if (now + u >= end) break;
            int kind, h;
            const bool on = rounds.at(a, now + u, sub, kind, h) && fits;
            Row<T> x = Stage::take(pieces(stage, u), at, lane);
            if (kind < 2) {
                Elements y;
                y.from(x);
                if (a.norm) {
                    Elements w;
                    load_weights<kPair>(w, weights[kind], at);
                    const uint64_t scale = both(rsqrtf(fmaf(row_sum<kLanes>(y.dot(y)), a.inv_dim, a.epsilon)));
#pragma unroll
                    for (int i = 0; i < 8; ++i) y.v[i] = mul2(mul2(y.v[i], scale), w.v[i]);
                }
                turn.apply(y, row, partners, chunk, a.rotary);
                y.to(x);
            }
            x.store(kind == 0 ? q + h * q_step : static_cast<T *>(kind == 1 ? a.k : a.v) + slot + h * kv_step, at, on);
        }
        stage ^= 1;
        Stage::meet();
    }
}

// As rope_kernel; a warp keeps its sums of the weights' gradients over all its items.
constexpr int kStepUnits = 8;  // 16-byte pieces of a lane and step
constexpr int kGradStaged = kWarps * 2 * kStepUnits * 32 * 16;

template <typename T, int kLanes, Pairing kPair>
__global__ void __launch_bounds__(kThreads, 4) rope_grad_kernel(const RopeArgs a) {
    using Stage = Staged<T, kLanes, kPair>;
    constexpr int kUnits = Stage::kUnits, kStep = kStepUnits / (2 * kUnits);  // rounds of a step
    extern __shared__ uint4 staged[];
    __shared__ __align__(16) float tables[kWarps][Turn<kLanes, kPair, true>::kFloats];
    __shared__ __align__(16) float weights[2][kTable];
    __shared__ float shared_rows[kWarps][kPair == kGeneral ? 32 * 17 : kTable];
    __shared__ __align__(16) int partners[kPair == kGeneral ? kTable : 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / kLanes, chunk = lane % kLanes;
    const Place at = lane_place<kPair>(chunk, a.dim, a.rotary);
    const Rounds<kLanes> rounds(a);
    float *row = shared_rows[warp] + (kPair == kGeneral ? sub * (kLanes * 17) : 0);
    const int q_step = a.seq * a.dim;
    Turn<kLanes, kPair, true> turn(tables[warp]);
    weight_tables<T, kPair>(a, weights);
    if constexpr (kPair == kGeneral) {
        partner_table<kPair>(a, partners);
        if (chunk == 0) row[kZeroAt] = 0.0f;
    }
    __syncthreads();
    Elements dwq, dwk;
#pragma unroll
    for (int i = 0; i < 8; ++i) dwq.v[i] = dwk.v[i] = 0;
    const int items = a.batch * a.seq * a.parts;
    // the next step: its item, rounds r .. of r1, and the rows of its token
    int item = blockIdx.x * kWarps + warp, r = 0, r1 = 0, position = 0, stage = 0;
    size_t packed = 0, query = 0, slot = 0;
    auto open = [&] {
        const int token = item / a.parts, part = item - token * a.parts, b = token / a.seq, t = token - b * a.seq;
        r = rounds.total * part / a.parts, r1 = rounds.total * (part + 1) / a.parts;
        position = __ldg(a.positions + token);
        packed = (size_t)token * (a.heads + 2 * a.kv_heads) * a.dim;
        query = ((size_t)b * a.heads * a.seq + t) * a.dim, slot = ((size_t)b * a.kv_heads * a.seq + t) * a.dim;
    };
    auto pieces = [&](int stage, int u) { return staged + ((warp * 2 + stage) * kStepUnits + 2 * kUnits * u) * 32; };
    auto offset = [&](int kind, int h) { return ((kind == 0 ? 0 : kind == 1 ? a.heads : a.heads + a.kv_heads) + h) * a.dim; };
    auto copy = [&](int stage) {
#pragma unroll
        for (int u = 0; u < kStep; ++u) {
            int kind, h;
            const bool on = rounds.at(a, r + u, sub, kind, h) && r + u < r1;
            if (!on) h = 0;
            Stage::copy(pieces(stage, u), static_cast<const T *>(kind == 0 ? a.q : kind == 1 ? a.k : a.v) + (kind == 0 ? query : slot) + h * q_step, at, on, lane, a.dim);
            Stage::copy(pieces(stage, u) + 32 * kUnits, static_cast<const T *>(a.qkv) + packed + offset(kind, h), at, on && a.norm && kind < 2, lane, a.dim);
        }
        copies_commit();
    };
    bool more = item < items, fresh = true;
    if (more) open(), copy(0);
    while (more) {
        const int now = r, end = r1, angle = position;
        const bool first = fresh;
        T *out = static_cast<T *>(a.dqkv) + packed;
        r += kStep, fresh = r >= r1;
        if (fresh) {
            item += gridDim.x * kWarps, more = item < items;
            if (more) open();
        }
        if (more) copy(stage ^ 1);
        else copies_commit();
        if (first && now < rounds.k) turn.form(a, angle, lane);
        copies_wait_but_one();
        Stage::meet();
#pragma unroll
        for (int u = 0; u < kStep; ++u) {
            if (now + u >= end) break;
            int kind, h;
            const bool on = rounds.at(a, now + u, sub, kind, h);
            Row<T> g = Stage::take(pieces(stage, u), at, lane);
            if (kind < 2) {
                Elements d;
                d.from(g);
                turn.apply(d, row, partners, chunk, a.rotary);
                if (a.norm) {
                    Elements y;
                    y.from(Stage::take(pieces(stage, u) + 32 * kUnits, at, lane));
                    const float scale = rsqrtf(fmaf(row_sum<kLanes>(y.dot(y)), a.inv_dim, a.epsilon));
#pragma unroll
                    for (int i = 0; i < 8; ++i) y.v[i] = mul2(y.v[i], both(scale));
                    // lanes without a row hold zeros
                    if (kind == 0) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) dwq.v[i] = fma2(d.v[i], y.v[i], dwq.v[i]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) dwk.v[i] = fma2(d.v[i], y.v[i], dwk.v[i]);
                    }
                    Elements w;
                    load_weights<kPair>(w, weights[kind], at);
#pragma unroll
                    for (int i = 0; i < 8; ++i) d.v[i] = mul2(d.v[i], w.v[i]);
                    const float mean = -row_sum<kLanes>(d.dot(y)) * a.inv_dim;
#pragma unroll
                    for (int i = 0; i < 8; ++i) d.v[i] = mul2(both(scale), fma2(y.v[i], both(mean), d.v[i]));
                }
                d.to(g);
            }
            g.store(out + offset(kind, on ? h : 0), at, on);
        }
        stage ^= 1;
        Stage::meet();
    }
    grid_dependency_trigger();
    if (!a.norm) return;
    // the block's sums: rows of the warp first, then the warps, each in a fixed order
    for (int which = 0; which < 2; ++which) {
        const Elements &sums = which ? dwk : dwq;
        float dw[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) unpack2f(sums.v[i], dw[2 * i], dw[2 * i + 1]);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
#pragma unroll
            for (int o = kLanes; o < 32; o <<= 1) dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
            if (sub == 0 && (i < 8 ? at.has_lo : at.has_hi)) shared_rows[warp][(i < 8 ? at.lo : at.hi) + (i & 7)] = dw[i];
        }
        __syncthreads();
        for (int e = threadIdx.x; e < a.dim; e += kThreads) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < kWarps; ++i) s += shared_rows[i][e];
            a.partial[((size_t)blockIdx.x * 2 + which) * a.dim + e] = s;
        }
    }
}

// Sums the blocks' partial weight gradients (592 blocks of 2 x 128: about 3 us behind the
// rows, bound by the latency of a few dependent loads): 32 columns of [blocks][2 dim] a block,
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

// Warps that share a token's heads: the number for which the resident warps take fewest
// rounds in a row, an item's angles counted as one more (they cost about that). Against
// one warp a token, of 48 heads of 128: 700 tokens 8.4 us for 12, 3,000 tokens 17.5 for 20.6.
// From two items a warp on their ends fall apart by themselves (gradient of 8,192 tokens:
// 59 us with one warp a token, 63 with two; neighbours forward 41 and 45).
int parts_of(long long tokens, int rounds, long long resident) {
    if (tokens >= 2 * resident) return 1;
    int best = 1;
    long long least = LLONG_MAX;
    for (int parts = 1; parts <= rounds; ++parts) {
        const long long cost = (tokens * parts + resident - 1) / resident * ((rounds + parts - 1) / parts + 1);
        if (cost < least) best = parts, least = cost;
    }
    return best;
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
    base.inv_dim = 1.0f / (float)s.dim;
    const int per = 32 / kLanes, rounds = rounds_of((int)s.heads, per) + 2 * rounds_of((int)s.kv_heads, per), dim = s.dim;
    int per_sm = 0;
    const int staged = grad ? kGradStaged : kForwardStaged;
    const void *kernel = grad ? reinterpret_cast<const void *>(rope_grad_kernel<T, kLanes, kPair>) : reinterpret_cast<const void *>(rope_kernel<T, kLanes, kPair>);
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, staged) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kThreads, staged) != cudaSuccess || per_sm < 1)
        throw IrError("the rotation kernel does not fit on an SM");
    const long long tokens = (long long)s.batch * s.seq, resident = (long long)per_sm * ctx->sm_count * kWarps;
    base.parts = parts_of(tokens, rounds, resident);
    if (tokens * base.parts > INT_MAX / 2) throw IrError("too many tokens for one launch");
    const int blocks = (int)std::min((tokens * base.parts + kWarps - 1) / kWarps, resident / kWarps);
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
            rope_kernel<T, kLanes, kPair><<<blocks, kThreads, staged, st>>>(a);
            return cudaGetLastError();
        }
        a.dqkv = b[i++];
        rope_grad_kernel<T, kLanes, kPair><<<blocks, kThreads, staged, st>>>(a);
        if (!norm) return cudaGetLastError();
        const cudaError_t e = launch_after(st, rope_weight_grad_kernel, (2 * dim + 31) / 32, 1024, 0, static_cast<const float *>(a.partial), blocks,
                                           dim, static_cast<float *>(b[i]), static_cast<float *>(b[i + 1]));
        return e == cudaSuccess ? cudaGetLastError() : e;
    };
}

template <typename T, Pairing kPair>
LaunchFn rope_lanes(Context *ctx, const Spec &s) {
    if (s.dim <= 64) return rope_launch<T, 4, kPair>(ctx, s);
    return s.dim <= 128 ? rope_launch<T, 8, kPair>(ctx, s) : rope_launch<T, 16, kPair>(ctx, s);
}
template <typename T>
LaunchFn rope_pick(Context *ctx, const Spec &s) {
    if (s.interleaved) return rope_lanes<T, kNeighbours>(ctx, s);
    return s.rotary % 16 == 0 ? rope_lanes<T, kHalves>(ctx, s) : rope_lanes<T, kGeneral>(ctx, s);
}

}  // namespace

LaunchFn make_qk_norm_rope(Context *ctx, const Spec &s, std::string &impl) {
    impl = std::string(spec_name(s)) + "_d" + std::to_string(s.dim) + "_" + dtype_name(s.dtype);
    if (s.dtype == DType::BF16) return rope_pick<__nv_bfloat16>(ctx, s);
    return s.dtype == DType::F16 ? rope_pick<__half>(ctx, s) : rope_pick<float>(ctx, s);
}

}  // namespace jade
