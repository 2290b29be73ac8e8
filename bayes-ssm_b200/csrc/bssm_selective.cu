// bssm_selective.cu -- selective state space scan: per channel, a state of N
// values that decays by its own rate at a step size chosen token by token.
//
//   d_t = softplus(s_t + bias)            (or s_t + bias)
//   h_t = exp(d_t A) h_{t-1} + d_t x_t k_t     h, A, k, q in R^N
//   y_t = (q_t . h_t + skip x_t) silu(z_t)
//
// keys k and queries q are shared by the channels of a group.  Backward, with
// the adjoint g of h running from the last token to the first:
//
//   dr_t = dy_t silu(z_t),  dz_t = dy_t r_t silu'(z_t),  r = q.h + skip x
//   g_t  = q_t dr_t + exp(d_{t+1} A) g_{t+1}
//   dq_t = sum_c dr h,  dk_t = sum_c g d x,  dx = skip dr + d (g.k)
//   dd   = sum_n g (A a h_{t-1} + x k),  dA = sum_t g d a h_{t-1},  a = exp(d A)
//
// Work split.  A lane holds 4 states of a channel and LPC = ceil(N / 4) lanes
// (a power of two, 1..16) hold the channel, so the sums over N take log2(LPC)
// exchanges and a warp advances 32 / LPC channels; tokens are walked in order.
// A CTA of 8 warps holds CH adjacent channels of one group and one sequence.
// Its threads first turn a tile of tokens into d, d x (and dr) in shared
// memory, coalesced along the channels and once per element rather than once
// per lane; then every warp scans the tile; then the threads finish their own
// elements (skip, gate) and store them.  Sums and states are float32.
//
// Bounds: one exp per state and token in the forward (16 a clock and SM: 3.6
// ps per channel-token at N = 16 against 1.2 ps for its bytes) and two in the
// backward, beside about 7 and 15 other float32 operations.
#include <cuda_runtime.h>

#include <cstdint>

#include "bayes_ssm_b200.h"
#include "bssm_internal.h"
#include "bssm_io.cuh"

namespace bssm {
namespace {

constexpr int kThreads = 256, kWarps = 8;
constexpr int kSegment = 16;  // tokens between the states a forward saves for its backward
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct ScanArgs {
    const void *values, *steps, *keys, *queries, *gate;
    const float *rates, *skip, *step_bias, *state0;
    long value_stride, step_stride, key_stride, query_stride, gate_stride;
    Sequences seq;
    int channels, states, groups, softplus;
    int tiles, tiles_per_group, group_channels;
    void *out;
    float *state1, *saved;
    // a sequence's chunks of `chunk` tokens (the last to its end), each its own CTA
    int chunks;
    long chunk;
    float *carry;  // [sequences][chunks][channels][states]
    float *span;   // [sequences][chunks][channels]: sum of d
    // backward
    const void *grad_out;
    const float *grad_state1;
    void *grad_values, *grad_steps, *grad_gate;
    float *grad_state0, *key_part, *rate_part, *channel_part;
};

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }

// exp(d A) of two states with rate = A log2 e, by the multifunction unit's exp2 (relative error below 2^-22;
// subnormal results are zero).  The unit cuts its argument's low bits off: measured over d A in [-0.35, -1e-4],
// where a state remembers many tokens and a bias adds up, its results were 0.10 to 0.37 of 2^-24 low on average,
// and within -0.11 to 0.16 with 3 * 2^-27 added to the argument, which the multiplication takes along as an FMA.
__device__ __forceinline__ float exp2_unit(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float2 decay_of(float d, float2 rate) {
    const float2 e = fma2(both(d), rate, both(3.f / 134217728.f));
    return make_float2(exp2_unit(e.x), exp2_unit(e.y));
}

// log(1 + exp(x)) = max(x, 0) + log1p(exp(-|x|)), and log1p(e) = 2 atanh(e / (2 + e)) = 2 v P(v^2) with
// v = e / (2 + e) in (0, 1/3]; P is atanh(v) / v fitted for the least relative error over v^2 in (0, 1/9], 2^-27.9
// (iterated weighted least squares).  A step's error is one of the decay's exponent, so expf, which keeps the bits
// that rounding x log2 e would lose.
__device__ __forceinline__ float softplus_f(float x) {
    const float e = expf(-fabsf(x));
    const float v = __fdividef(e, 2.f + e), w = v * v;
    float p = 0.14089173f;
    p = fmaf(p, w, 0.13980305f);
    p = fmaf(p, w, 0.20012454f);
    p = fmaf(p, w, 0.33333157f);
    p = fmaf(p, w, 1.f);
    return fmaf(2.f * v, p, fmaxf(x, 0.f));
}

template <int LPC> struct Geometry {
    static constexpr int kStates = 4 * LPC;           // states a channel's lanes hold (N padded)
    static constexpr int kChannels = kWarps * 32 / LPC;
    static constexpr int kPerWarp = 32 / LPC;         // channels per warp
    static constexpr int kBatch = LPC < 4 ? 4 : LPC;  // tokens whose sums over the lanes are taken together
    static constexpr int kTile = LPC <= 2 ? 8 * LPC : 32;                     // forward tile, tokens
    static constexpr int kElems = kTile * kChannels / kThreads;
    static constexpr int kRows = kThreads / kChannels;                        // token rows a pass of the CTA covers
    static constexpr int kPairs = (kTile * kStates + kThreads - 1) / kThreads;
    // row pitch of the sums: a batch's tokens fall into different banks
    static constexpr int kPitch = LPC == 16 ? 34 : LPC == 1 ? 256 : LPC == 2 ? 136 : kChannels + kPerWarp;
};

// Sums over a channel's LPC lanes of v[0 .. COUNT), each lane keeping COUNT /
// LPC of them (all, when LPC is 1): lane `sub` ends with v[i] the sum of entry
// sub * (COUNT / LPC) + i.  Halves are exchanged, so it takes COUNT - COUNT /
// LPC shuffles rather than COUNT log2(LPC).
template <int COUNT, int LPC> __device__ __forceinline__ void lane_sums(float (&v)[COUNT], int sub) {
    int half = COUNT / 2;
#pragma unroll
    for (int off = LPC / 2; off >= 1; off /= 2) {
        const bool upper = (sub & off) != 0;
#pragma unroll
        for (int i = 0; i < COUNT / 2; ++i) {
            if (i < half) {
                const float send = upper ? v[i] : v[i + half];
                const float keep = upper ? v[i + half] : v[i];
                v[i] = keep + __shfl_xor_sync(0xffffffffu, send, off);
            }
        }
        half /= 2;
    }
}

struct Place {  // what a CTA works on
    int group, c0, width;       // group, first channel (of all channels), channels that exist
    long s, first, tokens;      // sequence, its first row, its tokens
    long begin, end;            // the chunk's tokens of it
};

template <int LPC> __device__ __forceinline__ Place place_of(const ScanArgs &a, int chunk) {
    Place p;
    const int tile = static_cast<int>(blockIdx.x % a.tiles);
    p.s = blockIdx.x / a.tiles;
    p.group = tile / a.tiles_per_group;
    const int in_group = (tile - p.group * a.tiles_per_group) * Geometry<LPC>::kChannels;
    p.c0 = p.group * a.group_channels + in_group;
    p.width = min(Geometry<LPC>::kChannels, a.group_channels - in_group);
    p.first = a.seq.begin(p.s);
    p.tokens = max(0L, a.seq.end(p.s) - p.first);
    p.begin = min(p.tokens, chunk * a.chunk);
    p.end = chunk == a.chunks - 1 ? p.tokens : min(p.tokens, p.begin + a.chunk);
    return p;
}

// The four states n0 .. n0 + 3 of a lane in the order n0 + (j ^ m); those past N are zero.
__device__ __forceinline__ void load_states(const float *p, int n0, int m, int states, float2 (&o)[2]) {
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = p != nullptr && n0 + (j ^ m) < states ? p[j ^ m] : 0.f;
    o[0] = make_float2(v[0], v[1]);
    o[1] = make_float2(v[2], v[3]);
}
__device__ __forceinline__ void store_states(float *p, int n0, int m, int states, const float2 (&o)[2]) {
    const float v[4] = {o[0].x, o[0].y, o[1].x, o[1].y};
    if ((states & 3) == 0 && m == 0) {
        if (n0 < states) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (n0 + (j ^ m) < states) p[j ^ m] = v[j];
}

// Row of `saved` for token t (a multiple of kSegment) of a sequence: segments
// of different sequences never share one.
__device__ __forceinline__ long segment_row(const Sequences &q, long s, long first, long t) {
    return (q.offsets == nullptr ? s * ((q.length + kSegment - 1) / kSegment) : first / kSegment + s) + t / kSegment;
}

// A tile's rows on their way from global to shared memory.
template <typename T, int LPC> struct TileRows {
    using G = Geometry<LPC>;
    T x[G::kElems], s[G::kElems], z[G::kElems], k[G::kPairs], q[G::kPairs];

    __device__ __forceinline__ void load(const ScanArgs &a, const Place &p, long t0, int ec, int er) {
        const int count = static_cast<int>(min(static_cast<long>(G::kTile), p.end - t0));
        const long row0 = p.first + t0;
        const long cc = p.c0 + ec;
#pragma unroll
        for (int i = 0; i < G::kElems; ++i) {
            const int t = er + i * G::kRows;
            x[i] = s[i] = z[i] = from_float<T>(0.f);
            if (ec < p.width && t < count) {
                s[i] = static_cast<const T *>(a.steps)[(row0 + t) * a.step_stride + cc];
                x[i] = static_cast<const T *>(a.values)[(row0 + t) * a.value_stride + cc];
                if (a.gate != nullptr) z[i] = static_cast<const T *>(a.gate)[(row0 + t) * a.gate_stride + cc];
            }
        }
#pragma unroll
        for (int i = 0; i < G::kPairs; ++i) {
            const int e = threadIdx.x + i * kThreads, t = e / G::kStates, n = e % G::kStates;
            k[i] = q[i] = from_float<T>(0.f);
            if (t < count && n < a.states) {
                const long col = static_cast<long>(p.group) * a.states + n;
                k[i] = static_cast<const T *>(a.keys)[(row0 + t) * a.key_stride + col];
                q[i] = static_cast<const T *>(a.queries)[(row0 + t) * a.query_stride + col];
            }
        }
    }
};

// The next tile's rows are loaded while this one is scanned.
template <typename T, int LPC> __global__ void __launch_bounds__(kThreads, 2) scan_forward(const ScanArgs a) {
    using G = Geometry<LPC>;
    __shared__ float2 in_s[G::kTile][G::kChannels];  // (d, d x)
    __shared__ float sum_s[G::kTile * G::kPitch];
    __shared__ __align__(16) float k_s[G::kTile][G::kStates], q_s[G::kTile][G::kStates];
    const int chunk = static_cast<int>(blockIdx.y);
    const Place p = place_of<LPC>(a, chunk);
    if (chunk > 0 && p.begin >= p.end) return;  // past the end
    const int tid = threadIdx.x, lane = tid & 31;
    // elements: channel ec, token rows er + i * kRows
    const int ec = tid % G::kChannels, er = tid / G::kChannels;
    const bool own = ec < p.width;
    const long cc = p.c0 + ec;
    const float bias = own && a.step_bias != nullptr ? a.step_bias[cc] : 0.f;
    const float skip = own && a.skip != nullptr ? a.skip[cc] : 0.f;
    // scan: channel c, states n0 .. n0 + 3
    const int sub = lane % LPC, c = tid / 32 * G::kPerWarp + lane / LPC, n0 = 4 * sub;
    const bool live = c < p.width && n0 < a.states;
    const long row = static_cast<long>(a.channels) * a.states, at = static_cast<long>(p.c0 + c) * a.states + n0;
    float2 rate[2], h[2];
    load_states(live ? a.rates + at : nullptr, n0, 0, a.states, rate);
#pragma unroll
    for (int j = 0; j < 2; ++j) rate[j] = mul2(rate[j], both(kLog2e));
    const float *start = chunk > 0 ? a.carry + (p.s * a.chunks + chunk - 1) * row
                         : a.state0 != nullptr ? a.state0 + p.s * row : nullptr;
    load_states(live && start != nullptr ? start + at : nullptr, n0, 0, a.states, h);

    TileRows<T, LPC> next;
    next.load(a, p, p.begin, ec, er);
    for (long t0 = p.begin; t0 < p.end; t0 += G::kTile) {
        const int count = static_cast<int>(min(static_cast<long>(G::kTile), p.end - t0));
        T x[G::kElems], z[G::kElems];
#pragma unroll
        for (int i = 0; i < G::kElems; ++i) {
            const int t = er + i * G::kRows;
            x[i] = next.x[i];
            z[i] = next.z[i];
            float d = to_float(next.s[i]) + bias;
            if (a.softplus) d = softplus_f(d);
            if (!own || t >= count) d = 0.f;
            in_s[t][ec] = make_float2(d, d * to_float(x[i]));
        }
#pragma unroll
        for (int i = 0; i < G::kPairs; ++i) {
            const int e = tid + i * kThreads;
            if (G::kTile * G::kStates % kThreads == 0 || e < G::kTile * G::kStates) {
                (&k_s[0][0])[e] = to_float(next.k[i]);
                (&q_s[0][0])[e] = to_float(next.q[i]);
            }
        }
        __syncthreads();
        if (t0 + G::kTile < p.end) next.load(a, p, t0 + G::kTile, ec, er);
        for (int tb = 0; tb < count; tb += G::kBatch) {
            if (a.saved != nullptr && (t0 + tb) % kSegment == 0 && live)
                store_states(a.saved + segment_row(a.seq, p.s, p.first, t0 + tb) * row + at, n0, 0, a.states, h);
            float sum[G::kBatch];
#pragma unroll
            for (int u = 0; u < G::kBatch; ++u) {
                const float2 in = in_s[tb + u][c];
                const float4 k = *reinterpret_cast<const float4 *>(&k_s[tb + u][n0]);
                const float4 q = *reinterpret_cast<const float4 *>(&q_s[tb + u][n0]);
                h[0] = fma2(decay_of(in.x, rate[0]), h[0], mul2(both(in.y), make_float2(k.x, k.y)));
                h[1] = fma2(decay_of(in.x, rate[1]), h[1], mul2(both(in.y), make_float2(k.z, k.w)));
                const float2 y = fma2(make_float2(q.z, q.w), h[1], mul2(make_float2(q.x, q.y), h[0]));
                sum[u] = y.x + y.y;
            }
            lane_sums<G::kBatch, LPC>(sum, sub);
#pragma unroll
            for (int i = 0; i < G::kBatch / LPC; ++i)
                sum_s[(tb + sub * (G::kBatch / LPC) + i) * G::kPitch + c] = sum[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < G::kElems; ++i) {
            const int t = er + i * G::kRows;
            if (own && t < count) {
                float y = fmaf(skip, to_float(x[i]), sum_s[t * G::kPitch + ec]);
                if (a.gate != nullptr) y *= to_float(z[i]) * sigmoid_f(to_float(z[i]));
                static_cast<T *>(a.out)[(p.first + t0 + t) * a.channels + cc] = from_float<T>(y);
            }
        }
        // no barrier here: the next tile's in_s, k_s and q_s were last read before the one above, and its
        // sum_s is written after the next one
    }
    if (live && a.state1 != nullptr && p.end == p.tokens) store_states(a.state1 + p.s * row + at, n0, 0, a.states, h);
}

// What a chunk does to the state that enters it, h -> exp(A D) h + local: the
// scan from a state of zero, its outputs left out, and the sum D of its steps.
// BACKWARD: the same of the adjoint, which enters at the chunk's end:
// g -> exp(A D) g + local with g_{t-1} = a_t (q_t dr_t + g_t).
template <typename T, int LPC, bool BACKWARD>
__global__ void __launch_bounds__(kThreads, 3) scan_local(const ScanArgs a) {
    using G = Geometry<LPC>;
    __shared__ float2 in_s[G::kTile][G::kChannels];  // (d, d x) or (d, dr)
    __shared__ __align__(16) float k_s[G::kTile][G::kStates];
    const int chunk = static_cast<int>(blockIdx.y) + (BACKWARD ? 1 : 0);
    const Place p = place_of<LPC>(a, chunk);
    const int tid = threadIdx.x, lane = tid & 31;
    const int ec = tid % G::kChannels, er = tid / G::kChannels;
    const bool own = ec < p.width;
    const long cc = p.c0 + ec;
    const float bias = own && a.step_bias != nullptr ? a.step_bias[cc] : 0.f;
    const int sub = lane % LPC, c = tid / 32 * G::kPerWarp + lane / LPC, n0 = 4 * sub;
    const bool live = c < p.width && n0 < a.states;
    const long row = static_cast<long>(a.channels) * a.states, at = static_cast<long>(p.c0 + c) * a.states + n0;
    float2 rate[2], h[2] = {both(0.f), both(0.f)};
    load_states(live ? a.rates + at : nullptr, n0, 0, a.states, rate);
#pragma unroll
    for (int j = 0; j < 2; ++j) rate[j] = mul2(rate[j], both(kLog2e));
    float span = 0.f;

    const T *steps = static_cast<const T *>(a.steps), *gate = static_cast<const T *>(a.gate);
    const T *in = static_cast<const T *>(BACKWARD ? a.grad_out : a.values);
    const T *keys = static_cast<const T *>(BACKWARD ? a.queries : a.keys);
    const long in_stride = BACKWARD ? a.channels : a.value_stride;
    const long key_stride = BACKWARD ? a.query_stride : a.key_stride;
    const long tiles = (p.end - p.begin + G::kTile - 1) / G::kTile;
    T x[G::kElems], s[G::kElems], z[G::kElems], k[G::kPairs];
    auto load = [&](long tile) {
        const long t0 = p.begin + (BACKWARD ? tiles - 1 - tile : tile) * G::kTile;
        const int count = static_cast<int>(min(static_cast<long>(G::kTile), p.end - t0));
#pragma unroll
        for (int i = 0; i < G::kElems; ++i) {
            const int t = er + i * G::kRows;
            x[i] = s[i] = z[i] = from_float<T>(0.f);
            if (own && t < count) {
                s[i] = steps[(p.first + t0 + t) * a.step_stride + cc];
                if (in != nullptr) x[i] = in[(p.first + t0 + t) * in_stride + cc];
                if (BACKWARD && gate != nullptr) z[i] = gate[(p.first + t0 + t) * a.gate_stride + cc];
            }
        }
#pragma unroll
        for (int i = 0; i < G::kPairs; ++i) {
            const int e = tid + i * kThreads, t = e / G::kStates, n = e % G::kStates;
            k[i] = t < count && n < a.states
                       ? keys[(p.first + t0 + t) * key_stride + static_cast<long>(p.group) * a.states + n]
                       : from_float<T>(0.f);
        }
        return count;
    };
    int count = tiles > 0 ? load(0) : 0;
    for (long tile = 0; tile < tiles; ++tile) {
#pragma unroll
        for (int i = 0; i < G::kElems; ++i) {
            const int t = er + i * G::kRows;
            float d = to_float(s[i]) + bias, v = to_float(x[i]);
            if (a.softplus) d = softplus_f(d);
            if (!own || t >= count) d = 0.f;
            if (BACKWARD && gate != nullptr) v *= to_float(z[i]) * sigmoid_f(to_float(z[i]));
            span += d;
            in_s[t][ec] = make_float2(d, BACKWARD ? v : d * v);
        }
#pragma unroll
        for (int i = 0; i < G::kPairs; ++i) {
            const int e = tid + i * kThreads;
            if (G::kTile * G::kStates % kThreads == 0 || e < G::kTile * G::kStates) (&k_s[0][0])[e] = to_float(k[i]);
        }
        __syncthreads();
        if (tile + 1 < tiles) count = load(tile + 1);
#pragma unroll 4
        for (int i = 0; i < G::kTile; ++i) {
            const int t = BACKWARD ? G::kTile - 1 - i : i;
            const float2 v = in_s[t][c];
            const float4 kk = *reinterpret_cast<const float4 *>(&k_s[t][n0]);
            const float2 a0 = decay_of(v.x, rate[0]), a1 = decay_of(v.x, rate[1]);
            if (BACKWARD) {
                h[0] = mul2(a0, fma2(both(v.y), make_float2(kk.x, kk.y), h[0]));
                h[1] = mul2(a1, fma2(both(v.y), make_float2(kk.z, kk.w), h[1]));
            } else {
                h[0] = fma2(a0, h[0], mul2(both(v.y), make_float2(kk.x, kk.y)));
                h[1] = fma2(a1, h[1], mul2(both(v.y), make_float2(kk.z, kk.w)));
            }
        }
        __syncthreads();
    }
    const long entry = p.s * a.chunks + chunk;
    if (live) store_states(a.carry + entry * row + at, n0, 0, a.states, h);
    float *spans = reinterpret_cast<float *>(&in_s[0][0]);  // [kRows][kChannels]
    spans[er * G::kChannels + ec] = span;
    __syncthreads();
    if (er == 0 && own) {
        float v = 0.f;
        for (int i = 0; i < G::kRows; ++i) v += spans[i * G::kChannels + ec];
        a.span[entry * a.channels + cc] = v;
    }
}

// The chunks of a sequence joined, in place: entry i of `carry` becomes the
// state after chunk i (backward: the adjoint before chunk i), which the chunk
// after (before) it starts from.  A thread per state; the chain is short.
template <bool BACKWARD> __global__ void __launch_bounds__(kThreads) scan_join(const ScanArgs a) {
    const long row = static_cast<long>(a.channels) * a.states;
    const long i = static_cast<long>(blockIdx.x) * kThreads + threadIdx.x;
    if (i >= a.seq.count * row) return;
    const long s = i / row, at = i % row, c = at / a.states;
    const float rate = a.rates[at] * kLog2e;
    const float *start = BACKWARD ? a.grad_state1 : a.state0;
    float h = start != nullptr ? start[i] : 0.f;
    for (int k = 0; k + 1 < a.chunks; ++k) {
        const long entry = s * a.chunks + (BACKWARD ? a.chunks - 1 - k : k);
        h = fmaf(exp2f(a.span[entry * a.channels + c] * rate), h, a.carry[entry * row + at]);
        a.carry[entry * row + at] = h;
    }
}

template <int LPC> struct BackwardShared {
    using G = Geometry<LPC>;
    static constexpr int kCopies = G::kPerWarp >= 4 ? 4 : 2;
    float4 in[kSegment][G::kChannels];     // d, d x, dr, x
    float2 slopes[kSegment][G::kChannels]; // d's slope in the step, dy silu'(z)
    float gk[kSegment * G::kPitch], ga[kSegment * G::kPitch], r[kSegment * G::kPitch];
    // keys and queries, once for every order n ^ m of a lane's four states
    alignas(16) float k[kSegment][kCopies][G::kStates];
    alignas(16) float q[kSegment][kCopies][G::kStates];
    float part[kWarps][kSegment][2 * G::kStates];
};

// One CTA walks a chunk's segments of kSegment tokens from the last to the
// first: each is replayed from the state the forward saved at its start, its 16
// states kept in registers, then the adjoint runs back over them.  Keys' and
// queries' gradients are summed over the warp's channels by exchanges, over the
// CTA's warps in shared memory and written as one row per channel tile of
// key_part [tiles][tokens][2][N]; rates', skip's and step bias's as one row per
// chunk.  All are added up afterwards in a fixed order.
//
// A lane holds its four states in the order j ^ m, m from two of the bits that
// tell the warp's channels apart.  The two halves of an exchange over such a
// bit then are the same registers in every lane, so summing four states over
// four channels needs no selects (of 7 exchanges a token, 1 has them).
template <typename T, int LPC> __global__ void __launch_bounds__(kThreads, LPC < 2 ? 1 : 2)
scan_backward(const ScanArgs a) {
    using G = Geometry<LPC>;
    using S = BackwardShared<LPC>;
    constexpr int kElems = kSegment * G::kChannels / kThreads;
    extern __shared__ __align__(16) unsigned char raw[];
    S &sh = *reinterpret_cast<S *>(raw);
    const long tile = blockIdx.x % a.tiles;
    const int chunk = static_cast<int>(blockIdx.y);
    const Place p = place_of<LPC>(a, chunk);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32;
    const int ec = tid % G::kChannels, er = tid / G::kChannels;
    const bool own = ec < p.width;
    const long cc = p.c0 + ec;
    const float bias = own && a.step_bias != nullptr ? a.step_bias[cc] : 0.f;
    const float skip = own && a.skip != nullptr ? a.skip[cc] : 0.f;
    const int sub = lane % LPC, in_warp = lane / LPC, c = warp * G::kPerWarp + in_warp, n0 = 4 * sub;
    const int m = (in_warp & 1) * 2 + (G::kPerWarp >= 4 ? (in_warp >> 1) & 1 : 0);
    const int copy = G::kPerWarp >= 4 ? m : m / 2;
    const bool live = c < p.width && n0 < a.states;
    const long row = static_cast<long>(a.channels) * a.states, at = static_cast<long>(p.c0 + c) * a.states + n0;
    float2 rate[2], g[2], grate[2] = {both(0.f), both(0.f)};
    load_states(live ? a.rates + at : nullptr, n0, m, a.states, rate);
#pragma unroll
    for (int j = 0; j < 2; ++j) rate[j] = mul2(rate[j], both(kLog2e));
    const float *start = chunk < a.chunks - 1 ? a.carry + (p.s * a.chunks + chunk + 1) * row
                         : a.grad_state1 != nullptr ? a.grad_state1 + p.s * row : nullptr;
    load_states(live && start != nullptr ? start + at : nullptr, n0, m, a.states, g);
    float gskip = 0.f, gbias = 0.f;

    const T *values = static_cast<const T *>(a.values), *steps = static_cast<const T *>(a.steps);
    const T *keys = static_cast<const T *>(a.keys), *queries = static_cast<const T *>(a.queries);
    const T *gate = static_cast<const T *>(a.gate), *gy = static_cast<const T *>(a.grad_out);
    const long segments = (p.end - p.begin + kSegment - 1) / kSegment;
    for (long seg = segments - 1; seg >= 0; --seg) {
        const long t0 = p.begin + seg * kSegment;
        const int count = static_cast<int>(min(static_cast<long>(kSegment), p.end - t0));
#pragma unroll
        for (int i = 0; i < kElems; ++i) {
            const int t = er + i * G::kRows;
            float x = 0.f, d = 0.f, slope = 0.f, dr = 0.f, gz = 0.f;
            if (own && t < count) {
                const long r = p.first + t0 + t;
                d = to_float(steps[r * a.step_stride + cc]) + bias;
                x = to_float(values[r * a.value_stride + cc]);
                dr = gy == nullptr ? 0.f : to_float(gy[r * a.channels + cc]);
                slope = 1.f;
                if (a.softplus) {
                    slope = sigmoid_f(d);
                    d = softplus_f(d);
                }
                if (gate != nullptr) {
                    const float z = to_float(gate[r * a.gate_stride + cc]), sg = sigmoid_f(z);
                    gz = dr * sg * fmaf(z, 1.f - sg, 1.f);
                    dr *= z * sg;
                }
            }
            sh.in[t][ec] = make_float4(d, d * x, dr, x);
            sh.slopes[t][ec] = make_float2(slope, gz);  // read back by this thread only
        }
        for (int i = tid; i < kSegment * G::kStates; i += kThreads) {
            const int t = i / G::kStates, n = i % G::kStates;
            const bool ok = t < count && n < a.states;
            const long r = p.first + t0 + t, col = static_cast<long>(p.group) * a.states + n;
            const float k = ok ? to_float(keys[r * a.key_stride + col]) : 0.f;
            const float q = ok ? to_float(queries[r * a.query_stride + col]) : 0.f;
#pragma unroll
            for (int o = 0; o < S::kCopies; ++o) {
                const int order = S::kCopies == 4 ? o : 2 * o;
                sh.k[t][o][n ^ order] = k;
                sh.q[t][o][n ^ order] = q;
            }
        }
        __syncthreads();
        float2 h[kSegment + 1][2];  // h[t] before token t of the segment, h[t + 1] after it
        load_states(live ? a.saved + segment_row(a.seq, p.s, p.first, t0) * row + at : nullptr, n0, m, a.states, h[0]);
#pragma unroll
        for (int t = 0; t < kSegment; ++t) {
            if (t % 4 == 0) asm volatile("" ::: "memory");  // as below
            const float2 in = *reinterpret_cast<const float2 *>(&sh.in[t][c]);
            const float4 k = *reinterpret_cast<const float4 *>(&sh.k[t][copy][n0]);
            h[t + 1][0] = fma2(decay_of(in.x, rate[0]), h[t][0], mul2(both(in.y), make_float2(k.x, k.y)));
            h[t + 1][1] = fma2(decay_of(in.x, rate[1]), h[t][1], mul2(both(in.y), make_float2(k.z, k.w)));
        }
#pragma unroll
        for (int tb = kSegment - G::kBatch; tb >= 0; tb -= G::kBatch) {
            float sk[G::kBatch], sa[G::kBatch], sr[G::kBatch];
            asm volatile("" ::: "memory");  // keeps the compiler from loading later batches early, which spills
#pragma unroll
            for (int u = G::kBatch - 1; u >= 0; --u) {
                const int t = tb + u;
                const float4 in = sh.in[t][c];
                const float4 k4 = *reinterpret_cast<const float4 *>(&sh.k[t][copy][n0]);
                const float4 q4 = *reinterpret_cast<const float4 *>(&sh.q[t][copy][n0]);
                const float2 k[2] = {make_float2(k4.x, k4.y), make_float2(k4.z, k4.w)};
                const float2 q[2] = {make_float2(q4.x, q4.y), make_float2(q4.z, q4.w)};
                float2 dq[2], dk[2], pk = both(0.f), pa = both(0.f), pr = both(0.f);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float2 gh = fma2(q[j], both(in.z), g[j]);
                    dq[j] = mul2(both(in.z), h[t + 1][j]);
                    dk[j] = mul2(gh, both(in.y));
                    pr = fma2(q[j], h[t + 1][j], pr);
                    pk = fma2(gh, k[j], pk);
                    g[j] = mul2(decay_of(in.x, rate[j]), gh);
                    const float2 moved = mul2(g[j], h[t][j]);
                    pa = fma2(moved, rate[j], pa);
                    grate[j] = fma2(moved, both(in.x), grate[j]);
                }
                sk[u] = pk.x + pk.y;
                sa[u] = pa.x + pa.y;
                sr[u] = pr.x + pr.y;
                // over the warp's channels: states j and j ^ 2, then j ^ 1, then queries and keys
                float vq[2] = {dq[0].x + __shfl_xor_sync(0xffffffffu, dq[1].x, LPC),
                               dq[0].y + __shfl_xor_sync(0xffffffffu, dq[1].y, LPC)};
                float vk[2] = {dk[0].x + __shfl_xor_sync(0xffffffffu, dk[1].x, LPC),
                               dk[0].y + __shfl_xor_sync(0xffffffffu, dk[1].y, LPC)};
                float *part = sh.part[warp][t] + n0;
                if (G::kPerWarp == 2) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        part[j ^ m] = vq[j];
                        part[G::kStates + (j ^ m)] = vk[j];
                    }
                } else {
                    vq[0] += __shfl_xor_sync(0xffffffffu, vq[1], 2 * LPC);
                    vk[0] += __shfl_xor_sync(0xffffffffu, vk[1], 2 * LPC);
                    if (G::kPerWarp == 4) {
                        part[m] = vq[0];
                        part[G::kStates + m] = vk[0];
                    } else {
                        const bool keys_here = (in_warp & 4) != 0;
                        float v = (keys_here ? vk[0] : vq[0]) +
                                  __shfl_xor_sync(0xffffffffu, keys_here ? vq[0] : vk[0], 4 * LPC);
#pragma unroll
                        for (int off = 8 * LPC; off < 32; off *= 2) v += __shfl_xor_sync(0xffffffffu, v, off);
                        part[(keys_here ? G::kStates : 0) + m] = v;
                    }
                }
            }
            lane_sums<G::kBatch, LPC>(sk, sub);
            lane_sums<G::kBatch, LPC>(sa, sub);
            lane_sums<G::kBatch, LPC>(sr, sub);
#pragma unroll
            for (int i = 0; i < G::kBatch / LPC; ++i) {
                const int o = (tb + sub * (G::kBatch / LPC) + i) * G::kPitch + c;
                sh.gk[o] = sk[i];
                sh.ga[o] = sa[i];
                sh.r[o] = sr[i];
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kElems; ++i) {
            const int t = er + i * G::kRows;
            if (own && t < count) {
                const long r = p.first + t0 + t;
                const int o = t * G::kPitch + ec;
                const float4 in = sh.in[t][ec];
                const float2 slope = sh.slopes[t][ec];
                const float gd = fmaf(in.w, sh.gk[o], kLn2 * sh.ga[o]) * slope.x;  // rates were in powers of two
                static_cast<T *>(a.grad_values)[r * a.channels + cc] = from_float<T>(fmaf(in.x, sh.gk[o], skip * in.z));
                static_cast<T *>(a.grad_steps)[r * a.channels + cc] = from_float<T>(gd);
                if (gate != nullptr)
                    static_cast<T *>(a.grad_gate)[r * a.channels + cc] =
                        from_float<T>(slope.y * fmaf(skip, in.w, sh.r[o]));
                gbias += gd;
                gskip = fmaf(in.z, in.w, gskip);
            }
        }
        for (int i = tid; i < count * 2 * G::kStates; i += kThreads) {
            const int t = i / (2 * G::kStates), e = i % (2 * G::kStates);
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) v += sh.part[w][t][e];
            const int which = e / G::kStates, n = e % G::kStates;
            if (n < a.states)
                a.key_part[((tile * a.seq.tokens + p.first + t0 + t) * 2 + which) * a.states + n] = v;
        }
        __syncthreads();
    }
    const long entry = p.s * a.chunks + chunk;
    if (live && a.grad_state0 != nullptr && chunk == 0)
        store_states(a.grad_state0 + p.s * row + at, n0, m, a.states, g);
    if (live) store_states(a.rate_part + entry * row + at, n0, m, a.states, grate);
    // the skip's and step bias's sums over the CTA's token rows
    float *cs = sh.gk;  // [2][kRows][kChannels]
    cs[er * G::kChannels + ec] = gskip;
    cs[(G::kRows + er) * G::kChannels + ec] = gbias;
    __syncthreads();
    if (er == 0 && own) {
        float v = 0.f, w = 0.f;
        for (int i = 0; i < G::kRows; ++i) {
            v += cs[i * G::kChannels + ec];
            w += cs[(G::kRows + i) * G::kChannels + ec];
        }
        a.channel_part[entry * 2 * a.channels + cc] = v;
        a.channel_part[(entry * 2 + 1) * a.channels + cc] = w;
    }
}

// Keys' and queries' gradients: the rows of key_part [tiles][tokens][2][N] of
// each group's tiles, added in order of the tile.
template <typename T> __global__ void __launch_bounds__(kThreads) scan_sum_keys(const ScanArgs a, void *grad_keys,
                                                                                void *grad_queries) {
    const long cols = a.seq.tokens * 2 * a.states;
    const long i = static_cast<long>(blockIdx.x) * kThreads + threadIdx.x;
    if (i >= cols * a.groups) return;
    const long col = i % cols, group = i / cols;
    const long token = col / (2 * a.states);
    const int e = static_cast<int>(col % (2 * a.states)), which = e / a.states, n = e % a.states;
    float v = 0.f;
    for (int t = 0; t < a.tiles_per_group; ++t) v += a.key_part[(group * a.tiles_per_group + t) * cols + col];
    T *out = static_cast<T *>(which == 0 ? grad_queries : grad_keys);
    out[(token * a.groups + group) * a.states + n] = from_float<T>(v);
}

// Rates', skip's and step bias's gradients: the chunks' rows added in order.
__global__ void __launch_bounds__(kThreads) scan_sum_rows(const ScanArgs a, float *grad_rates, float *grad_skip,
                                                          float *grad_step_bias) {
    const long state = static_cast<long>(a.channels) * a.states, rows = a.seq.count * a.chunks;
    const long i = static_cast<long>(blockIdx.x) * kThreads + threadIdx.x;
    const long j = i - state;  // of 2 * channels: skip, then step bias
    if (j >= 2L * a.channels) return;
    const float *part = j < 0 ? a.rate_part + i : a.channel_part + j;
    const long pitch = j < 0 ? state : 2L * a.channels;
    float *out = j < 0 ? grad_rates + i
                 : j < a.channels ? (grad_skip == nullptr ? nullptr : grad_skip + j)
                                  : (grad_step_bias == nullptr ? nullptr : grad_step_bias + j - a.channels);
    if (out == nullptr) return;
    float v = 0.f;
#pragma unroll 8
    for (long r = 0; r < rows; ++r) v += part[r * pitch];
    *out = v;
}

template <typename T> __device__ __forceinline__ void load_row(const T *p, int n0, int states, float2 (&o)[2]) {
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = n0 + j < states ? to_float(p[j]) : 0.f;
    o[0] = make_float2(v[0], v[1]);
    o[1] = make_float2(v[2], v[3]);
}

// One token per sequence, the states [sequences][channels][N] moved on in place.
template <typename T, int LPC> __global__ void __launch_bounds__(kThreads) scan_step(const ScanArgs a, float *state) {
    const long id = static_cast<long>(blockIdx.x) * kThreads + threadIdx.x;
    const long row = id / LPC;  // sequence * channels + channel
    const int sub = static_cast<int>(id % LPC), n0 = 4 * sub;
    const bool ok = row < a.seq.count * a.channels;
    const bool live = ok && n0 < a.states;
    const long s = ok ? row / a.channels : 0, c = ok ? row % a.channels : 0;
    const long group = c / a.group_channels, col = group * a.states + n0;
    float sum = 0.f, x = 0.f;
    if (live) {
        x = to_float(static_cast<const T *>(a.values)[s * a.value_stride + c]);
        float d = to_float(static_cast<const T *>(a.steps)[s * a.step_stride + c]);
        if (a.step_bias != nullptr) d += a.step_bias[c];
        float2 h[2], rate[2], k[2], q[2];
        load_states(state + row * a.states + n0, n0, 0, a.states, h);
        load_states(a.rates + c * a.states + n0, n0, 0, a.states, rate);
        load_row(static_cast<const T *>(a.keys) + s * a.key_stride + col, n0, a.states, k);
        load_row(static_cast<const T *>(a.queries) + s * a.query_stride + col, n0, a.states, q);
        if (a.softplus) d = softplus_f(d);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            h[j] = fma2(decay_of(d, mul2(rate[j], both(kLog2e))), h[j], mul2(both(d * x), k[j]));
            const float2 y = mul2(q[j], h[j]);
            sum += y.x + y.y;
        }
        store_states(state + row * a.states + n0, n0, 0, a.states, h);
    }
#pragma unroll
    for (int off = LPC / 2; off >= 1; off /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (live && sub == 0) {
        if (a.skip != nullptr) sum = fmaf(a.skip[c], x, sum);
        if (a.gate != nullptr) {
            const float z = to_float(static_cast<const T *>(a.gate)[s * a.gate_stride + c]);
            sum *= z * sigmoid_f(z);
        }
        static_cast<T *>(a.out)[s * a.channels + c] = from_float<T>(sum);
    }
}

int lanes_per_channel(int states) {
    int lpc = 1;
    while (4 * lpc < states) lpc *= 2;
    return lpc;
}

void set_tiles(ScanArgs &a) {
    const int width = kWarps * 32 / lanes_per_channel(a.states);
    a.group_channels = a.channels / a.groups;
    a.tiles_per_group = (a.group_channels + width - 1) / width;
    a.tiles = a.tiles_per_group * a.groups;
}

unsigned blocks_for(long n) { return static_cast<unsigned>((n + kThreads - 1) / kThreads); }

// Chunks of a sequence that run as CTAs of their own.  Each costs a second
// pass of exponentials (the chunk's effect on the state that enters it), so a
// sequence is split only where its channels leave SMs idle.
void set_chunks(ScanArgs &a, long longest, int wanted_ctas, long shortest) {
    const long ctas = a.seq.count * a.tiles;
    a.chunks = 1;
    a.chunk = longest > 0 ? longest : 1;
    if (ctas == 0 || ctas * 2 > wanted_ctas) return;
    const long most = longest / shortest, wanted = wanted_ctas / ctas;
    const long chunks = wanted < most ? wanted : most;
    if (chunks < 2) return;
    a.chunk = ((longest + chunks - 1) / chunks + kSegment * 2 - 1) / (kSegment * 2) * (kSegment * 2);
    a.chunks = static_cast<int>((longest + a.chunk - 1) / a.chunk);
}
void set_forward_chunks(ScanArgs &a, long longest) { set_chunks(a, longest, 296, 128); }
void set_backward_chunks(ScanArgs &a, long longest) { set_chunks(a, longest, 296, 64); }

// Workspace, every part a multiple of 16 bytes: with a null base, its size.
long place_carry(ScanArgs &a, float *workspace) {
    if (a.chunks < 2) return 0;
    const long rows = a.seq.count * a.chunks * a.channels, states = (rows * a.states + 3) / 4 * 4;
    a.carry = workspace;
    a.span = workspace + states;
    return states + (rows + 3) / 4 * 4;
}
long place_backward(ScanArgs &a, float *workspace) {
    const long rows = a.seq.count * a.chunks * a.channels;
    long at = place_carry(a, workspace);
    a.rate_part = workspace + at;
    at += (rows * a.states + 3) / 4 * 4;
    a.channel_part = workspace + at;
    at += (rows * 2 + 3) / 4 * 4;
    a.key_part = workspace + at;
    return at + static_cast<long>(a.tiles) * a.seq.tokens * 2 * a.states;
}

ScanArgs shape_args(long tokens, long sequences, int channels, int states, int groups) {
    ScanArgs a{};
    a.seq = {nullptr, sequences, sequences > 0 ? tokens / sequences : 0, tokens};
    a.channels = channels; a.states = states; a.groups = groups;
    set_tiles(a);
    return a;
}

template <typename T, int LPC> int launch_forward(const ScanArgs &a, cudaStream_t st) {
    const dim3 grid(static_cast<unsigned>(a.seq.count * a.tiles), static_cast<unsigned>(a.chunks));
    if (a.chunks > 1) {
        scan_local<T, LPC, false><<<dim3(grid.x, grid.y - 1), kThreads, 0, st>>>(a);
        scan_join<false><<<blocks_for(a.seq.count * a.channels * a.states), kThreads, 0, st>>>(a);
    }
    scan_forward<T, LPC><<<grid, kThreads, 0, st>>>(a);
    return check_launch("selective_scan");
}
template <typename T, int LPC> int launch_backward(const ScanArgs &a, cudaStream_t st) {
    constexpr int bytes = static_cast<int>(sizeof(BackwardShared<LPC>));
    if (cudaError_t e = cudaFuncSetAttribute(scan_backward<T, LPC>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes))
        return fail(BSSM_ERR_CUDA, "selective_scan_backward: %s", cudaGetErrorString(e));
    const dim3 grid(static_cast<unsigned>(a.seq.count * a.tiles), static_cast<unsigned>(a.chunks));
    if (a.chunks > 1) {
        scan_local<T, LPC, true><<<dim3(grid.x, grid.y - 1), kThreads, 0, st>>>(a);
        scan_join<true><<<blocks_for(a.seq.count * a.channels * a.states), kThreads, 0, st>>>(a);
    }
    scan_backward<T, LPC><<<grid, kThreads, bytes, st>>>(a);
    return check_launch("selective_scan_backward");
}
template <typename T, int LPC> int launch_step(const ScanArgs &a, cudaStream_t st) {
    const long threads = a.seq.count * a.channels * LPC;
    scan_step<T, LPC><<<static_cast<unsigned>((threads + kThreads - 1) / kThreads), kThreads, 0, st>>>(a, a.state1);
    return check_launch("selective_step");
}

enum ScanKind { kScan, kScanBackward, kScanStep };

template <typename T, int LPC> int launch_kind(ScanKind kind, const ScanArgs &a, cudaStream_t st) {
    if (kind == kScan) return launch_forward<T, LPC>(a, st);
    if (kind == kScanBackward) return launch_backward<T, LPC>(a, st);
    return launch_step<T, LPC>(a, st);
}
template <typename T> int launch_lanes(ScanKind kind, const ScanArgs &a, cudaStream_t st) {
    switch (lanes_per_channel(a.states)) {
        case 1: return launch_kind<T, 1>(kind, a, st);
        case 2: return launch_kind<T, 2>(kind, a, st);
        case 4: return launch_kind<T, 4>(kind, a, st);
        case 8: return launch_kind<T, 8>(kind, a, st);
        default: return launch_kind<T, 16>(kind, a, st);
    }
}
int launch_scan(ScanKind kind, int dtype, const ScanArgs &a, cudaStream_t st) {
    switch (dtype) {
        case BSSM_F32: return launch_lanes<float>(kind, a, st);
        case BSSM_BF16: return launch_lanes<__nv_bfloat16>(kind, a, st);
        default: return launch_lanes<__half>(kind, a, st);
    }
}

int check_scan(const char *what, int dtype, int channels, int states, int groups, long sequences, long tokens,
               bool equal_length) {
    if (!io_dtype_known(dtype)) return fail(BSSM_ERR_UNSUPPORTED, "%s: unknown dtype", what);
    if (states < 1 || states > 64) return fail(BSSM_ERR_UNSUPPORTED, "%s: %d states (1 to 64 are built)", what, states);
    if (channels < 1 || groups < 1 || channels % groups != 0 || sequences < 0 || tokens < 0)
        return fail(BSSM_ERR_INVALID, "%s: bad sizes", what);
    if (sequences == 0 && tokens > 0) return fail(BSSM_ERR_INVALID, "%s: rows without a sequence", what);
    if (equal_length && sequences > 0 && tokens % sequences != 0)
        return fail(BSSM_ERR_INVALID, "%s: rows do not divide into sequences of one length", what);
    if (sequences > 0x7fffffffL / channels) return fail(BSSM_ERR_INVALID, "%s: too many rows", what);  // the grid
    return BSSM_OK;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace bssm

extern "C" long bssm_selective_saved_floats(long tokens, long sequences, int channels, int states) {
    return (tokens / bssm::kSegment + sequences) * channels * states;
}

extern "C" long bssm_selective_scan_floats(long tokens, long sequences, long longest, int channels, int states,
                                           int groups) {
    using namespace bssm;
    if (check_scan("selective_scan_floats", BSSM_F32, channels, states, groups, sequences, tokens, false)) return 0;
    ScanArgs a = shape_args(tokens, sequences, channels, states, groups);
    set_forward_chunks(a, longest);
    return place_carry(a, nullptr);
}

extern "C" int bssm_selective_scan(const void *values, long value_stride, const void *steps, long step_stride,
                                   const void *keys, long key_stride, const void *queries, long query_stride,
                                   const void *gate, long gate_stride, int dtype, const float *rates,
                                   const float *skip, const float *step_bias, int softplus, long tokens, int channels,
                                   int states, int groups, const long *offsets, long sequences, long longest,
                                   const float *state0, void *out, float *state1, float *saved, long saved_floats,
                                   float *workspace, long workspace_floats, void *stream) {
    using namespace bssm;
    if (int rc = check_scan("selective_scan", dtype, channels, states, groups, sequences, tokens, offsets == nullptr))
        return rc;
    if (sequences == 0) return BSSM_OK;
    if (rates == nullptr || (tokens > 0 && (values == nullptr || steps == nullptr || keys == nullptr ||
                                            queries == nullptr || out == nullptr)))
        return fail(BSSM_ERR_INVALID, "selective_scan: null pointer");
    if (saved != nullptr && saved_floats < bssm_selective_saved_floats(tokens, sequences, channels, states))
        return fail(BSSM_ERR_WORKSPACE, "selective_scan: buffer for the saved states too small");
    if (!aligned16(state1) || !aligned16(saved) || !aligned16(workspace))
        return fail(BSSM_ERR_ALIGNMENT, "selective_scan: states and workspace must be 16-byte aligned");
    ScanArgs a = shape_args(tokens, sequences, channels, states, groups);
    a.values = values; a.steps = steps; a.keys = keys; a.queries = queries; a.gate = gate;
    a.rates = rates; a.skip = skip; a.step_bias = step_bias; a.state0 = state0;
    a.value_stride = value_stride; a.step_stride = step_stride; a.key_stride = key_stride;
    a.query_stride = query_stride; a.gate_stride = gate_stride;
    a.seq.offsets = offsets;
    a.softplus = softplus;
    a.out = out; a.state1 = state1; a.saved = saved;
    set_forward_chunks(a, longest);
    const long needed = place_carry(a, workspace);
    if (workspace_floats < needed || (needed > 0 && workspace == nullptr))
        return fail(BSSM_ERR_WORKSPACE, "selective_scan: workspace too small");
    return launch_scan(kScan, dtype, a, static_cast<cudaStream_t>(stream));
}

extern "C" long bssm_selective_backward_floats(long tokens, long sequences, long longest, int channels, int states,
                                               int groups) {
    using namespace bssm;
    if (check_scan("selective_backward_floats", BSSM_F32, channels, states, groups, sequences, tokens, false)) return 0;
    ScanArgs a = shape_args(tokens, sequences, channels, states, groups);
    set_backward_chunks(a, longest);
    return place_backward(a, nullptr);
}

extern "C" int bssm_selective_scan_backward(
    const void *values, long value_stride, const void *steps, long step_stride, const void *keys, long key_stride,
    const void *queries, long query_stride, const void *gate, long gate_stride, int dtype, const float *rates,
    const float *skip, const float *step_bias, int softplus, long tokens, int channels, int states, int groups,
    const long *offsets, long sequences, long longest, const float *saved, const void *grad_out,
    const float *grad_state1, void *grad_values, void *grad_steps, float *grad_rates, void *grad_keys,
    void *grad_queries, float *grad_skip, void *grad_gate, float *grad_step_bias, float *grad_state0, float *workspace,
    long workspace_floats, void *stream) {
    using namespace bssm;
    if (int rc = check_scan("selective_scan_backward", dtype, channels, states, groups, sequences, tokens,
                            offsets == nullptr))
        return rc;
    if (rates == nullptr || grad_rates == nullptr || (gate != nullptr && grad_gate == nullptr && tokens > 0) ||
        (tokens > 0 && (values == nullptr || steps == nullptr || keys == nullptr || queries == nullptr ||
                        saved == nullptr || grad_values == nullptr || grad_steps == nullptr || grad_keys == nullptr ||
                        grad_queries == nullptr)))
        return fail(BSSM_ERR_INVALID, "selective_scan_backward: null pointer");
    if (!aligned16(grad_state0) || !aligned16(workspace))
        return fail(BSSM_ERR_ALIGNMENT, "selective_scan_backward: states and workspace must be 16-byte aligned");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    ScanArgs a = shape_args(tokens, sequences, channels, states, groups);
    a.values = values; a.steps = steps; a.keys = keys; a.queries = queries; a.gate = gate;
    a.rates = rates; a.skip = skip; a.step_bias = step_bias;
    a.value_stride = value_stride; a.step_stride = step_stride; a.key_stride = key_stride;
    a.query_stride = query_stride; a.gate_stride = gate_stride;
    a.seq.offsets = offsets;
    a.softplus = softplus;
    a.saved = const_cast<float *>(saved); a.grad_out = grad_out; a.grad_state1 = grad_state1;
    a.grad_values = grad_values; a.grad_steps = grad_steps; a.grad_gate = grad_gate; a.grad_state0 = grad_state0;
    set_backward_chunks(a, longest);
    const long needed = place_backward(a, workspace);
    if (workspace_floats < needed || (needed > 0 && workspace == nullptr))
        return fail(BSSM_ERR_WORKSPACE, "selective_scan_backward: workspace too small");
    if (sequences > 0)
        if (int rc = launch_scan(kScanBackward, dtype, a, st)) return rc;
    const long cols = tokens * 2 * states * groups;
    if (cols > 0) {
        const unsigned grid = blocks_for(cols);
        if (dtype == BSSM_F32) scan_sum_keys<float><<<grid, kThreads, 0, st>>>(a, grad_keys, grad_queries);
        else if (dtype == BSSM_BF16) scan_sum_keys<__nv_bfloat16><<<grid, kThreads, 0, st>>>(a, grad_keys, grad_queries);
        else scan_sum_keys<__half><<<grid, kThreads, 0, st>>>(a, grad_keys, grad_queries);
    }
    // rates', then skip's and step bias's rows added up, in one launch
    const long state = static_cast<long>(channels) * states;
    scan_sum_rows<<<blocks_for(state + 2L * channels), kThreads, 0, st>>>(a, grad_rates, grad_skip, grad_step_bias);
    return check_launch("selective_scan_backward");
}

extern "C" int bssm_selective_step(const void *values, long value_stride, const void *steps, long step_stride,
                                   const void *keys, long key_stride, const void *queries, long query_stride,
                                   const void *gate, long gate_stride, int dtype, const float *rates,
                                   const float *skip, const float *step_bias, int softplus, long sequences,
                                   int channels, int states, int groups, float *state, void *out, void *stream) {
    using namespace bssm;
    if (int rc = check_scan("selective_step", dtype, channels, states, groups, sequences, sequences, true)) return rc;
    if (sequences == 0) return BSSM_OK;
    if (values == nullptr || steps == nullptr || keys == nullptr || queries == nullptr || rates == nullptr ||
        state == nullptr || out == nullptr)
        return fail(BSSM_ERR_INVALID, "selective_step: null pointer");
    if (!aligned16(state)) return fail(BSSM_ERR_ALIGNMENT, "selective_step: states must be 16-byte aligned");
    ScanArgs a = shape_args(sequences, sequences, channels, states, groups);
    a.values = values; a.steps = steps; a.keys = keys; a.queries = queries; a.gate = gate;
    a.rates = rates; a.skip = skip; a.step_bias = step_bias;
    a.value_stride = value_stride; a.step_stride = step_stride; a.key_stride = key_stride;
    a.query_stride = query_stride; a.gate_stride = gate_stride;
    a.softplus = softplus;
    a.out = out; a.state1 = state;
    return launch_scan(kScanStep, dtype, a, static_cast<cudaStream_t>(stream));
}
