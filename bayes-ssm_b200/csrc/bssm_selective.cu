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
constexpr float kLog2e = 1.4426950408889634f;

struct ScanArgs {
    const void *values, *steps, *keys, *queries, *gate;
    const float *rates, *skip, *step_bias, *state0;
    long value_stride, step_stride, key_stride, query_stride, gate_stride;
    Sequences seq;
    int channels, states, groups, softplus;
    int tiles, tiles_per_group, group_channels;
    void *out;
    float *state1, *saved;
    // backward
    const void *grad_out;
    const float *grad_state1;
    void *grad_values, *grad_steps, *grad_gate;
    float *grad_state0, *key_part, *rate_part, *channel_part;
};

// exp(d A) with rate = A log2 e, by the multifunction unit's exp2 (relative error below 2^-22; subnormal results
// are zero).  The unit cuts its argument's low bits off: measured over d A in [-0.35, -1e-4], where a state
// remembers many tokens and a bias adds up, its results were 0.10 to 0.37 of 2^-24 low on average, and within
// -0.11 to 0.16 with 3 * 2^-27 added to the argument, which the multiplication takes along as an FMA.
__device__ __forceinline__ float decay_of(float d, float rate) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fmaf(d, rate, 3.f / 134217728.f)));
    return y;
}

// log(1 + exp(x)) = max(x, 0) + log1p(exp(-|x|)), and log1p(e) = 2 atanh(e / (2 + e)): with v = e / (2 + e) in
// (0, 1/3] the odd series 2 v (1 + v^2 / 3 + ... + v^14 / 15) is cut off below 2^-27 of its sum.  A step's error is
// one of the decay's exponent, so expf, which keeps the bits that rounding x log2 e would lose.
__device__ __forceinline__ float softplus_f(float x) {
    const float e = expf(-fabsf(x));
    const float v = __fdividef(e, 2.f + e), w = v * v;
    float p = 1.f / 15.f;
    p = fmaf(p, w, 1.f / 13.f);
    p = fmaf(p, w, 1.f / 11.f);
    p = fmaf(p, w, 1.f / 9.f);
    p = fmaf(p, w, 1.f / 7.f);
    p = fmaf(p, w, 1.f / 5.f);
    p = fmaf(p, w, 1.f / 3.f);
    return fmaxf(x, 0.f) + 2.f * v * fmaf(p, w, 1.f);
}

template <int LPC> struct Geometry {
    static constexpr int kStates = 4 * LPC;           // states a channel's lanes hold (N padded)
    static constexpr int kChannels = kWarps * 32 / LPC;
    static constexpr int kPerWarp = 32 / LPC;         // channels per warp
    static constexpr int kBatch = LPC < 4 ? 4 : LPC;  // tokens whose sums over the lanes are taken together
    static constexpr int kTile = LPC <= 2 ? 8 * LPC : 32;                     // forward tile, tokens
    static constexpr int kElems = kTile * kChannels / kThreads;
    static constexpr int kRows = kThreads / kChannels;                        // token rows a pass of the CTA covers
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
    int group, c0, width;  // group, first channel (of all channels), channels that exist
    long first, tokens, s;
};

template <int LPC> __device__ __forceinline__ Place place_of(const ScanArgs &a, long tile, long s) {
    Place p;
    p.group = static_cast<int>(tile) / a.tiles_per_group;
    const int in_group = (static_cast<int>(tile) - p.group * a.tiles_per_group) * Geometry<LPC>::kChannels;
    p.c0 = p.group * a.group_channels + in_group;
    p.width = min(Geometry<LPC>::kChannels, a.group_channels - in_group);
    p.s = s;
    p.first = a.seq.begin(s);
    p.tokens = max(0L, a.seq.end(s) - p.first);
    return p;
}

__device__ __forceinline__ void load_states(const float *p, int n0, int states, float (&o)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = p != nullptr && n0 + j < states ? p[j] : 0.f;
}
__device__ __forceinline__ void store_states(float *p, int n0, int states, const float (&v)[4]) {
    if ((states & 3) == 0) {
        if (n0 < states) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (n0 + j < states) p[j] = v[j];
}

// Row of `saved` for token t (a multiple of kSegment) of a sequence: segments
// of different sequences never share one.
__device__ __forceinline__ long segment_row(const Sequences &q, long s, long first, long t) {
    return (q.offsets == nullptr ? s * ((q.length + kSegment - 1) / kSegment) : first / kSegment + s) + t / kSegment;
}

template <typename T, int LPC> __global__ void __launch_bounds__(kThreads) scan_forward(const ScanArgs a) {
    using G = Geometry<LPC>;
    __shared__ float2 in_s[G::kTile][G::kChannels];  // (d, d x)
    __shared__ float sum_s[G::kTile * G::kPitch];
    __shared__ __align__(16) float k_s[G::kTile][G::kStates], q_s[G::kTile][G::kStates];
    const Place p = place_of<LPC>(a, blockIdx.x % a.tiles, blockIdx.x / a.tiles);
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
    float rate[4], h[4];
    load_states(live ? a.rates + (static_cast<long>(p.c0 + c) * a.states + n0) : nullptr, n0, a.states, rate);
#pragma unroll
    for (int j = 0; j < 4; ++j) rate[j] *= kLog2e;
    const long at = (p.s * a.channels + p.c0 + c) * a.states + n0;
    load_states(live && a.state0 != nullptr ? a.state0 + at : nullptr, n0, a.states, h);

    const T *values = static_cast<const T *>(a.values), *steps = static_cast<const T *>(a.steps);
    const T *keys = static_cast<const T *>(a.keys), *queries = static_cast<const T *>(a.queries);
    const T *gate = static_cast<const T *>(a.gate);
    for (long t0 = 0; t0 < p.tokens; t0 += G::kTile) {
        const int count = static_cast<int>(min(static_cast<long>(G::kTile), p.tokens - t0));
        float x[G::kElems], z[G::kElems];
#pragma unroll
        for (int i = 0; i < G::kElems; ++i) {
            const int t = er + i * G::kRows;
            float d = 0.f;
            x[i] = z[i] = 0.f;
            if (own && t < count) {
                const long g = p.first + t0 + t;
                d = to_float(steps[g * a.step_stride + cc]) + bias;
                x[i] = to_float(values[g * a.value_stride + cc]);
                if (gate != nullptr) z[i] = to_float(gate[g * a.gate_stride + cc]);
                if (a.softplus) d = softplus_f(d);
            }
            in_s[t][ec] = make_float2(d, d * x[i]);
        }
        for (int i = tid; i < G::kTile * G::kStates; i += kThreads) {
            const int t = i / G::kStates, n = i % G::kStates;
            const bool ok = t < count && n < a.states;
            const long g = p.first + t0 + t, col = static_cast<long>(p.group) * a.states + n;
            k_s[t][n] = ok ? to_float(keys[g * a.key_stride + col]) : 0.f;
            q_s[t][n] = ok ? to_float(queries[g * a.query_stride + col]) : 0.f;
        }
        __syncthreads();
        for (int tb = 0; tb < count; tb += G::kBatch) {
            if (a.saved != nullptr && (t0 + tb) % kSegment == 0 && live)
                store_states(a.saved + (segment_row(a.seq, p.s, p.first, t0 + tb) * a.channels + p.c0 + c) * a.states +
                                 n0, n0, a.states, h);
            float sum[G::kBatch];
#pragma unroll
            for (int u = 0; u < G::kBatch; ++u) {
                const float2 in = in_s[tb + u][c];
                const float4 k = *reinterpret_cast<const float4 *>(&k_s[tb + u][n0]);
                const float4 q = *reinterpret_cast<const float4 *>(&q_s[tb + u][n0]);
                h[0] = fmaf(decay_of(in.x, rate[0]), h[0], in.y * k.x);
                h[1] = fmaf(decay_of(in.x, rate[1]), h[1], in.y * k.y);
                h[2] = fmaf(decay_of(in.x, rate[2]), h[2], in.y * k.z);
                h[3] = fmaf(decay_of(in.x, rate[3]), h[3], in.y * k.w);
                sum[u] = fmaf(q.x, h[0], fmaf(q.y, h[1], fmaf(q.z, h[2], q.w * h[3])));
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
                float y = fmaf(skip, x[i], sum_s[t * G::kPitch + ec]);
                if (gate != nullptr) y *= z[i] * sigmoid_f(z[i]);
                static_cast<T *>(a.out)[(p.first + t0 + t) * a.channels + cc] = from_float<T>(y);
            }
        }
        // no barrier here: the next tile's in_s, k_s and q_s were last read before the one above, and its
        // sum_s is written after the next one
    }
    if (live && a.state1 != nullptr) store_states(a.state1 + at, n0, a.states, h);
}

// Sums over the lanes that hold different channels of the warp (lane bits LPC
// and up) of v[0 .. 8): each lane keeps 8 / min(8, channels per warp) of them,
// from entry `base` on.
template <int LPC> __device__ __forceinline__ int channel_sums(float (&v)[8], int lane) {
    int half = 4, base = 0;
#pragma unroll
    for (int off = 16; off >= LPC; off /= 2) {
        if (half > 0) {
            const bool upper = (lane & off) != 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (i < half) {
                    const float send = upper ? v[i] : v[i + half];
                    const float keep = upper ? v[i + half] : v[i];
                    v[i] = keep + __shfl_xor_sync(0xffffffffu, send, off);
                }
            }
            base += upper ? half : 0;
            half /= 2;
        } else {
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], off);
        }
    }
    return base;
}

template <int LPC> struct BackwardShared {
    using G = Geometry<LPC>;
    float d[kSegment][G::kChannels], dx[kSegment][G::kChannels], dr[kSegment][G::kChannels];
    float gk[kSegment * G::kPitch], ga[kSegment * G::kPitch], r[kSegment * G::kPitch];
    alignas(16) float k[kSegment][G::kStates];
    alignas(16) float q[kSegment][G::kStates];
    float part[kWarps][kSegment][2 * G::kStates];
};

// One CTA walks a sequence's segments of kSegment tokens from the last to the
// first: each is replayed from the state the forward saved at its start, its 16
// states kept in registers, then the adjoint runs back over them.  Keys' and
// queries' gradients are summed over the warp's channels by exchanges, over the
// CTA's warps in shared memory and written as one row per channel tile of
// key_part [tiles][tokens][2][N]; rates', skip's and step bias's as one row per
// sequence.  All are added up afterwards in a fixed order.
template <typename T, int LPC> __global__ void __launch_bounds__(kThreads) scan_backward(const ScanArgs a) {
    using G = Geometry<LPC>;
    constexpr int kElems = kSegment * G::kChannels / kThreads;
    extern __shared__ __align__(16) unsigned char raw[];
    BackwardShared<LPC> &sh = *reinterpret_cast<BackwardShared<LPC> *>(raw);
    const long tile = blockIdx.x % a.tiles;
    const Place p = place_of<LPC>(a, tile, blockIdx.x / a.tiles);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32;
    const int ec = tid % G::kChannels, er = tid / G::kChannels;
    const bool own = ec < p.width;
    const long cc = p.c0 + ec;
    const float bias = own && a.step_bias != nullptr ? a.step_bias[cc] : 0.f;
    const float skip = own && a.skip != nullptr ? a.skip[cc] : 0.f;
    const int sub = lane % LPC, c = warp * G::kPerWarp + lane / LPC, n0 = 4 * sub;
    const bool live = c < p.width && n0 < a.states;
    float rate[4], g[4], grate[4] = {};
    load_states(live ? a.rates + (static_cast<long>(p.c0 + c) * a.states + n0) : nullptr, n0, a.states, rate);
    float rate2[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) rate2[j] = rate[j] * kLog2e;
    const long at = (p.s * a.channels + p.c0 + c) * a.states + n0;
    load_states(live && a.grad_state1 != nullptr ? a.grad_state1 + at : nullptr, n0, a.states, g);
    float gskip = 0.f, gbias = 0.f;

    const T *values = static_cast<const T *>(a.values), *steps = static_cast<const T *>(a.steps);
    const T *keys = static_cast<const T *>(a.keys), *queries = static_cast<const T *>(a.queries);
    const T *gate = static_cast<const T *>(a.gate), *gy = static_cast<const T *>(a.grad_out);
    for (long t0 = (p.tokens - 1) / kSegment * kSegment; t0 >= 0 && p.tokens > 0; t0 -= kSegment) {
        const int count = static_cast<int>(min(static_cast<long>(kSegment), p.tokens - t0));
        float x[kElems], d[kElems], slope[kElems], dr[kElems], gz[kElems];
#pragma unroll
        for (int i = 0; i < kElems; ++i) {
            const int t = er + i * G::kRows;
            x[i] = d[i] = slope[i] = dr[i] = gz[i] = 0.f;
            if (own && t < count) {
                const long row = p.first + t0 + t;
                d[i] = to_float(steps[row * a.step_stride + cc]) + bias;
                x[i] = to_float(values[row * a.value_stride + cc]);
                dr[i] = gy == nullptr ? 0.f : to_float(gy[row * a.channels + cc]);
                slope[i] = 1.f;
                if (a.softplus) {
                    slope[i] = sigmoid_f(d[i]);
                    d[i] = softplus_f(d[i]);
                }
                if (gate != nullptr) {
                    const float z = to_float(gate[row * a.gate_stride + cc]), sg = sigmoid_f(z);
                    gz[i] = dr[i] * sg * fmaf(z, 1.f - sg, 1.f);
                    dr[i] *= z * sg;
                }
            }
            sh.d[t][ec] = d[i];
            sh.dx[t][ec] = d[i] * x[i];
            sh.dr[t][ec] = dr[i];
        }
        for (int i = tid; i < kSegment * G::kStates; i += kThreads) {
            const int t = i / G::kStates, n = i % G::kStates;
            const bool ok = t < count && n < a.states;
            const long row = p.first + t0 + t, col = static_cast<long>(p.group) * a.states + n;
            sh.k[t][n] = ok ? to_float(keys[row * a.key_stride + col]) : 0.f;
            sh.q[t][n] = ok ? to_float(queries[row * a.query_stride + col]) : 0.f;
        }
        __syncthreads();
        float h[kSegment + 1][4];  // h[t] before token t of the segment, h[t + 1] after it
        load_states(live ? a.saved + (segment_row(a.seq, p.s, p.first, t0) * a.channels + p.c0 + c) * a.states + n0
                         : nullptr, n0, a.states, h[0]);
#pragma unroll
        for (int t = 0; t < kSegment; ++t) {
            const float dt = sh.d[t][c], dx = sh.dx[t][c];
            const float4 k = *reinterpret_cast<const float4 *>(&sh.k[t][n0]);
            h[t + 1][0] = fmaf(decay_of(dt, rate2[0]), h[t][0], dx * k.x);
            h[t + 1][1] = fmaf(decay_of(dt, rate2[1]), h[t][1], dx * k.y);
            h[t + 1][2] = fmaf(decay_of(dt, rate2[2]), h[t][2], dx * k.z);
            h[t + 1][3] = fmaf(decay_of(dt, rate2[3]), h[t][3], dx * k.w);
        }
#pragma unroll
        for (int tb = kSegment - G::kBatch; tb >= 0; tb -= G::kBatch) {
            float sk[G::kBatch], sa[G::kBatch], sr[G::kBatch];
#pragma unroll
            for (int u = G::kBatch - 1; u >= 0; --u) {
                const int t = tb + u;
                const float dt = sh.d[t][c], dx = sh.dx[t][c], drt = sh.dr[t][c];
                const float4 k4 = *reinterpret_cast<const float4 *>(&sh.k[t][n0]);
                const float4 q4 = *reinterpret_cast<const float4 *>(&sh.q[t][n0]);
                const float k[4] = {k4.x, k4.y, k4.z, k4.w}, q[4] = {q4.x, q4.y, q4.z, q4.w};
                float v[8];
                sk[u] = sa[u] = sr[u] = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float gh = fmaf(q[j], drt, g[j]);
                    v[j] = drt * h[t + 1][j];
                    v[4 + j] = gh * dx;
                    sr[u] = fmaf(q[j], h[t + 1][j], sr[u]);
                    sk[u] = fmaf(gh, k[j], sk[u]);
                    g[j] = decay_of(dt, rate2[j]) * gh;
                    const float moved = g[j] * h[t][j];
                    sa[u] = fmaf(moved, rate[j], sa[u]);
                    grate[j] = fmaf(moved, dt, grate[j]);
                }
                const int base = channel_sums<LPC>(v, lane);
                constexpr int kKept = G::kPerWarp >= 8 ? 1 : 8 / G::kPerWarp;
#pragma unroll
                for (int i = 0; i < kKept; ++i) {
                    const int e = base + i;  // 0..3 queries, 4..7 keys
                    sh.part[warp][t][(e < 4 ? 0 : G::kStates) + n0 + (e & 3)] = v[i];
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
                const long row = p.first + t0 + t;
                const int o = t * G::kPitch + ec;
                const float gd = fmaf(x[i], sh.gk[o], sh.ga[o]) * slope[i];
                static_cast<T *>(a.grad_values)[row * a.channels + cc] =
                    from_float<T>(fmaf(d[i], sh.gk[o], skip * dr[i]));
                static_cast<T *>(a.grad_steps)[row * a.channels + cc] = from_float<T>(gd);
                if (gate != nullptr)
                    static_cast<T *>(a.grad_gate)[row * a.channels + cc] =
                        from_float<T>(gz[i] * fmaf(skip, x[i], sh.r[o]));
                gbias += gd;
                gskip = fmaf(dr[i], x[i], gskip);
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
    if (live && a.grad_state0 != nullptr) store_states(a.grad_state0 + at, n0, a.states, g);
    if (live) store_states(a.rate_part + at, n0, a.states, grate);
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
        a.channel_part[(p.s * 2) * a.channels + cc] = v;
        a.channel_part[(p.s * 2 + 1) * a.channels + cc] = w;
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

// out[i] = sum over `rows` of part[row * pitch + i], in order of the row.
__global__ void __launch_bounds__(kThreads) scan_sum_rows(const float *part, long rows, long pitch, long cols,
                                                          float *out) {
    const long i = static_cast<long>(blockIdx.x) * kThreads + threadIdx.x;
    if (i >= cols) return;
    float v = 0.f;
    for (long r = 0; r < rows; ++r) v += part[r * pitch + i];
    out[i] = v;
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
        float h[4], rate[4];
        load_states(state + row * a.states + n0, n0, a.states, h);
        load_states(a.rates + c * a.states + n0, n0, a.states, rate);
        if (a.softplus) d = softplus_f(d);
        const float dx = d * x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (n0 + j < a.states) {
                const float k = to_float(static_cast<const T *>(a.keys)[s * a.key_stride + col + j]);
                const float q = to_float(static_cast<const T *>(a.queries)[s * a.query_stride + col + j]);
                h[j] = fmaf(decay_of(d, kLog2e * rate[j]), h[j], dx * k);
                sum = fmaf(q, h[j], sum);
            }
        }
        store_states(state + row * a.states + n0, n0, a.states, h);
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

template <typename T, int LPC> int launch_forward(const ScanArgs &a, cudaStream_t st) {
    scan_forward<T, LPC><<<static_cast<unsigned>(a.seq.count * a.tiles), kThreads, 0, st>>>(a);
    return check_launch("selective_scan");
}
template <typename T, int LPC> int launch_backward(const ScanArgs &a, cudaStream_t st) {
    constexpr int bytes = static_cast<int>(sizeof(BackwardShared<LPC>));
    if (cudaError_t e = cudaFuncSetAttribute(scan_backward<T, LPC>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes))
        return fail(BSSM_ERR_CUDA, "selective_scan_backward: %s", cudaGetErrorString(e));
    scan_backward<T, LPC><<<static_cast<unsigned>(a.seq.count * a.tiles), kThreads, bytes, st>>>(a);
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

extern "C" int bssm_selective_scan(const void *values, long value_stride, const void *steps, long step_stride,
                                   const void *keys, long key_stride, const void *queries, long query_stride,
                                   const void *gate, long gate_stride, int dtype, const float *rates,
                                   const float *skip, const float *step_bias, int softplus, long tokens, int channels,
                                   int states, int groups, const long *offsets, long sequences, const float *state0,
                                   void *out, float *state1, float *saved, long saved_floats, void *stream) {
    using namespace bssm;
    if (int rc = check_scan("selective_scan", dtype, channels, states, groups, sequences, tokens, offsets == nullptr))
        return rc;
    if (sequences == 0) return BSSM_OK;
    if (rates == nullptr || (tokens > 0 && (values == nullptr || steps == nullptr || keys == nullptr ||
                                            queries == nullptr || out == nullptr)))
        return fail(BSSM_ERR_INVALID, "selective_scan: null pointer");
    if (saved != nullptr && saved_floats < bssm_selective_saved_floats(tokens, sequences, channels, states))
        return fail(BSSM_ERR_WORKSPACE, "selective_scan: buffer for the saved states too small");
    if (!aligned16(state1) || !aligned16(saved))
        return fail(BSSM_ERR_ALIGNMENT, "selective_scan: states must be 16-byte aligned");
    ScanArgs a{};
    a.values = values; a.steps = steps; a.keys = keys; a.queries = queries; a.gate = gate;
    a.rates = rates; a.skip = skip; a.step_bias = step_bias; a.state0 = state0;
    a.value_stride = value_stride; a.step_stride = step_stride; a.key_stride = key_stride;
    a.query_stride = query_stride; a.gate_stride = gate_stride;
    a.seq = {offsets, sequences, tokens / sequences, tokens};
    a.channels = channels; a.states = states; a.groups = groups; a.softplus = softplus;
    a.out = out; a.state1 = state1; a.saved = saved;
    set_tiles(a);
    return launch_scan(kScan, dtype, a, static_cast<cudaStream_t>(stream));
}

extern "C" long bssm_selective_backward_floats(long tokens, long sequences, int channels, int states, int groups) {
    bssm::ScanArgs a{};
    if (channels < 1 || states < 1 || groups < 1) return 0;
    a.channels = channels; a.states = states; a.groups = groups;
    bssm::set_tiles(a);
    const long state = (sequences * channels * states + 3) / 4 * 4;
    return state + sequences * 2 * channels + static_cast<long>(a.tiles) * tokens * 2 * states;
}

extern "C" int bssm_selective_scan_backward(
    const void *values, long value_stride, const void *steps, long step_stride, const void *keys, long key_stride,
    const void *queries, long query_stride, const void *gate, long gate_stride, int dtype, const float *rates,
    const float *skip, const float *step_bias, int softplus, long tokens, int channels, int states, int groups,
    const long *offsets, long sequences, const float *saved, const void *grad_out, const float *grad_state1,
    void *grad_values, void *grad_steps, float *grad_rates, void *grad_keys, void *grad_queries, float *grad_skip,
    void *grad_gate, float *grad_step_bias, float *grad_state0, float *workspace, long workspace_floats,
    void *stream) {
    using namespace bssm;
    if (int rc = check_scan("selective_scan_backward", dtype, channels, states, groups, sequences, tokens,
                            offsets == nullptr))
        return rc;
    if (rates == nullptr || grad_rates == nullptr || (gate != nullptr && grad_gate == nullptr && tokens > 0) ||
        (tokens > 0 && (values == nullptr || steps == nullptr || keys == nullptr || queries == nullptr ||
                        saved == nullptr || grad_values == nullptr || grad_steps == nullptr || grad_keys == nullptr ||
                        grad_queries == nullptr)))
        return fail(BSSM_ERR_INVALID, "selective_scan_backward: null pointer");
    if (workspace_floats < bssm_selective_backward_floats(tokens, sequences, channels, states, groups) ||
        (workspace == nullptr && sequences > 0))
        return fail(BSSM_ERR_WORKSPACE, "selective_scan_backward: workspace too small");
    if (!aligned16(grad_state0) || !aligned16(workspace))
        return fail(BSSM_ERR_ALIGNMENT, "selective_scan_backward: states and workspace must be 16-byte aligned");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    ScanArgs a{};
    a.values = values; a.steps = steps; a.keys = keys; a.queries = queries; a.gate = gate;
    a.rates = rates; a.skip = skip; a.step_bias = step_bias;
    a.value_stride = value_stride; a.step_stride = step_stride; a.key_stride = key_stride;
    a.query_stride = query_stride; a.gate_stride = gate_stride;
    a.seq = {offsets, sequences, sequences > 0 ? tokens / sequences : 0, tokens};
    a.channels = channels; a.states = states; a.groups = groups; a.softplus = softplus;
    a.saved = const_cast<float *>(saved); a.grad_out = grad_out; a.grad_state1 = grad_state1;
    a.grad_values = grad_values; a.grad_steps = grad_steps; a.grad_gate = grad_gate; a.grad_state0 = grad_state0;
    a.rate_part = workspace;
    a.channel_part = workspace + (sequences * channels * states + 3) / 4 * 4;
    a.key_part = a.channel_part + sequences * 2 * channels;
    set_tiles(a);
    if (sequences > 0)
        if (int rc = launch_scan(kScanBackward, dtype, a, st)) return rc;
    auto blocks = [](long n) { return static_cast<unsigned>((n + kThreads - 1) / kThreads); };
    const long cols = tokens * 2 * states * groups;
    if (cols > 0) {
        if (dtype == BSSM_F32) scan_sum_keys<float><<<blocks(cols), kThreads, 0, st>>>(a, grad_keys, grad_queries);
        else if (dtype == BSSM_BF16)
            scan_sum_keys<__nv_bfloat16><<<blocks(cols), kThreads, 0, st>>>(a, grad_keys, grad_queries);
        else scan_sum_keys<__half><<<blocks(cols), kThreads, 0, st>>>(a, grad_keys, grad_queries);
    }
    const long state = static_cast<long>(channels) * states;
    scan_sum_rows<<<blocks(state), kThreads, 0, st>>>(a.rate_part, sequences, state, state, grad_rates);
    if (grad_skip != nullptr)
        scan_sum_rows<<<blocks(channels), kThreads, 0, st>>>(a.channel_part, sequences, 2L * channels, channels,
                                                             grad_skip);
    if (grad_step_bias != nullptr)
        scan_sum_rows<<<blocks(channels), kThreads, 0, st>>>(a.channel_part + channels, sequences, 2L * channels,
                                                             channels, grad_step_bias);
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
    ScanArgs a{};
    a.values = values; a.steps = steps; a.keys = keys; a.queries = queries; a.gate = gate;
    a.rates = rates; a.skip = skip; a.step_bias = step_bias;
    a.value_stride = value_stride; a.step_stride = step_stride; a.key_stride = key_stride;
    a.query_stride = query_stride; a.gate_stride = gate_stride;
    a.seq = {nullptr, sequences, 1, sequences};
    a.channels = channels; a.states = states; a.groups = groups; a.softplus = softplus;
    a.out = out; a.state1 = state;
    set_tiles(a);
    return launch_scan(kScanStep, dtype, a, static_cast<cudaStream_t>(stream));
}
