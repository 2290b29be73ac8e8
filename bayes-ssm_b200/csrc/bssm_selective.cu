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
// Work split.  A lane holds 2 states of a channel and LPC = ceil(N / 2) lanes
// (a power of two, 1..32) hold the channel, so a warp advances 32 / LPC
// channels; tokens are walked in order.
// A CTA of 8 warps holds adjacent channels of one group and one sequence (32 of
// them at N = 16).  Its threads first turn a tile of tokens into d, d x (and
// dr) in shared memory, coalesced along the channels and once per element
// rather than once per lane; then every warp scans the tile; then the threads
// finish their own elements (skip, gate) and store them.  Sums and states are
// float32.  (Four states a lane need a tenth fewer instructions but have half
// the warps, and few rows are what this operator usually gets.)
//
// Bounds: one exp per state and token in the forward (16 a clock and SM: 3.6
// ps per channel-token at N = 16 against 1.2 ps for its bytes) and two in the
// backward, beside the other float32 instructions of the step.
#include <cuda_runtime.h>

#include <cfloat>
#include <cstdint>
#include <type_traits>

#include "bayes_ssm_b200.h"
#include "bssm_internal.h"
#include "bssm_io.cuh"

namespace bssm {
namespace {

constexpr int kThreads = 256, kWarps = 8;
constexpr int kChained = 24;  // chunks up to which every one chains those before it itself (a launch saved)
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
    int chunks, joined;  // joined: by scan_join, for more than kChained chunks
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
constexpr float kExponentBias = 3.f / 134217728.f;
__device__ __forceinline__ float exp2_unit(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float2 decay_of(float d, float2 rate) {
    const float2 e = fma2(both(d), rate, both(kExponentBias));
    return make_float2(exp2_unit(e.x), exp2_unit(e.y));
}

// log(1 + exp(x)) = max(x, 0) + log1p(e) with e = exp(-|x|), and log1p(e) = 2 atanh(v) = 2 v P(v^2) with
// v = e / (2 + e) in (0, 1/3]; P is atanh(v) / v fitted for the least relative error over v^2 in (0, 1/9], 2^-27.9
// (iterated weighted least squares).  A step's error is one of the decay's exponent, so e is taken with what
// rounding |x| log2 e lost: 2^(t + l) = 2^t (1 + l ln 2).  The slope is e's too: 1 / (1 + e) or e / (1 + e).
__device__ __forceinline__ float reciprocal(float x) {  // within 1 ulp
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <bool SLOPE> __device__ __forceinline__ float softplus_f(float x, float &slope) {
    constexpr float kLog2eLow = 1.925963033500e-8f;  // log2 e beyond its first 24 bits
    const float y = fabsf(x) > 128.f ? -128.f : -fabsf(x);  // a NaN stays one
    const float t = y * kLog2e, l = fmaf(y, kLog2eLow, fmaf(y, kLog2e, -t));
    float e = exp2_unit(t);
    e = fmaf(e, l * kLn2, e);
    const float v = e * reciprocal(2.f + e), w = v * v;
    float p = 0.14089173f;
    p = fmaf(p, w, 0.13980305f);
    p = fmaf(p, w, 0.20012454f);
    p = fmaf(p, w, 0.33333157f);
    p = fmaf(p, w, 1.f);
    if (SLOPE) slope = (x >= 0.f ? 1.f : e) * reciprocal(1.f + e);
    return fmaf(2.f * v, p, fmaxf(x, 0.f));
}

template <int LPC> struct Geometry {
    static constexpr int kStates = 2 * LPC;           // states a channel's lanes hold (N padded)
    static constexpr int kPerWarp = 32 / LPC;         // channels per warp
    static constexpr int kChannels = kWarps * kPerWarp;
    static constexpr int kRows = kThreads / kChannels;  // token rows a pass of the CTA covers
    static constexpr int kTile = LPC <= 2 ? 8 * LPC : 32;  // tokens of a tile
    static constexpr int kElems = kTile * kChannels / kThreads;
    static constexpr int kPairs = (kTile * LPC + kThreads - 1) / kThreads;  // pairs of states a thread loads
};

// Lanes.  In the forward adjacent lanes hold different channels and the same
// states: shared loads of 8 or 16 bytes take half the wavefronts where lanes
// 2 i and 2 i + 1 read the same address, and keys and queries are more bytes than
// a channel's (d, d x) (5 wavefronts a token become 4: 199 -> 193 us).  In the
// backward, which reads 16 bytes of a channel, adjacent lanes hold different
// states of one (the other way round it took 528 us against 514).
//
// Sums over a channel's lanes go through shared memory: every lane leaves its
// term at [token][channel][lane], and the thread that finishes the element adds the
// LPC neighbours (a store per token and a few wide loads per element; exchanges
// between the lanes would take a shuffle, an add and two selects a token).  The
// 16-byte loads of 8 neighbouring elements start at different vectors, so that
// they fall into different banks.
template <int LPC> __device__ __forceinline__ float sum_of(const float *token, int c) {
    if (LPC == 1) return token[c];
    if (LPC == 2) {
        const float2 v = reinterpret_cast<const float2 *>(token)[c];
        return v.x + v.y;
    }
    constexpr int kVecs = LPC < 4 ? 1 : LPC / 4, kShift = LPC == 8 ? 2 : LPC == 16 ? 1 : 0;
    float2 sum = both(0.f);
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
        const float4 v = reinterpret_cast<const float4 *>(token)[c * kVecs + ((j + (c >> kShift)) & (kVecs - 1))];
        sum = __fadd2_rn(sum, __fadd2_rn(make_float2(v.x, v.y), make_float2(v.z, v.w)));
    }
    return sum.x + sum.y;
}
template <int LPC> __device__ __forceinline__ float2 sums_of(const float2 *token, int c) {
    if (LPC == 1) return token[c];
    constexpr int kVecs = LPC < 2 ? 1 : LPC / 2, kShift = LPC == 4 ? 2 : LPC == 8 ? 1 : 0;
    float2 sum = both(0.f);
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
        const float4 v = reinterpret_cast<const float4 *>(token)[c * kVecs + ((j + (c >> kShift)) & (kVecs - 1))];
        sum = __fadd2_rn(sum, __fadd2_rn(make_float2(v.x, v.y), make_float2(v.z, v.w)));
    }
    return sum;
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
    // the same in every lane: said to the compiler, which then keeps addresses in uniform registers
    p.first = __shfl_sync(0xffffffffu, a.seq.begin(p.s), 0);
    p.tokens = __shfl_sync(0xffffffffu, max(0L, a.seq.end(p.s) - p.first), 0);
    p.begin = min(p.tokens, chunk * a.chunk);
    p.end = chunk == a.chunks - 1 ? p.tokens : min(p.tokens, p.begin + a.chunk);
    return p;
}

// A lane's two states n0 + (0 ^ m), n0 + (1 ^ m); those past N are zero.
__device__ __forceinline__ float2 load_states(const float *p, int n0, int m, int states) {
    float2 v = both(0.f);
    if (p != nullptr && n0 + m < states) v.x = p[m];
    if (p != nullptr && n0 + (1 ^ m) < states) v.y = p[1 ^ m];
    return v;
}
__device__ __forceinline__ void store_states(float *p, int n0, int m, int states, float2 v) {
    if ((states & 1) == 0) {
        if (n0 < states) *reinterpret_cast<float2 *>(p) = m == 0 ? v : make_float2(v.y, v.x);
        return;
    }
    if (n0 + m < states) p[m] = v.x;
    if (n0 + (1 ^ m) < states) p[1 ^ m] = v.y;
}

// A rate in powers of two.  One of -inf (a state that keeps nothing) becomes the
// lowest number, so that a step of zero keeps the state whatever its rate: as
// 0 * inf, the tokens that fill a tile up and the chunks past a short sequence's
// end would make it NaN.
__device__ __forceinline__ float in_powers_of_two(float rate) {
    rate *= kLog2e;
    return rate == -INFINITY ? -FLT_MAX : rate;
}
__device__ __forceinline__ float2 load_rates(const float *p, int n0, int m, int states) {
    const float2 rate = load_states(p, n0, m, states);
    return make_float2(in_powers_of_two(rate.x), in_powers_of_two(rate.y));
}

// The state after a chunk that h entered, exp(A D) h + local.  One of zero adds
// nothing, also where exp(A D) is past float32 (a positive rate; token by token
// it would never have been formed).
__device__ __forceinline__ float through_chunk(float exponent, float h, float local) {
    return h == 0.f ? local : fmaf(exp2f(exponent), h, local);
}

// The state that enters a chunk (BACKWARD: the adjoint, which enters at its
// end).  A few chunks before (after) it are chained here, from what scan_local
// found for each; more have been joined by scan_join.
template <bool BACKWARD>
__device__ __forceinline__ float2 entering(const ScanArgs &a, long s, int chunk, long c, long at, int n0, int m,
                                           bool live, float2 rate) {
    const long row = static_cast<long>(a.channels) * a.states;
    const float *start = BACKWARD ? a.grad_state1 : a.state0;
    const int first = BACKWARD ? a.chunks - 1 : 0, step = BACKWARD ? -1 : 1;
    if (a.joined && chunk != first)
        return load_states(live ? a.carry + (s * a.chunks + chunk - step) * row + at : nullptr, n0, m, a.states);
    float2 h = load_states(live && start != nullptr ? start + s * row + at : nullptr, n0, m, a.states);
#pragma unroll 4
    for (int k = first; k != chunk; k += step) {
        const long entry = s * a.chunks + k;
        const float span = live ? a.span[entry * a.channels + c] : 0.f;
        const float2 local = load_states(live ? a.carry + entry * row + at : nullptr, n0, m, a.states);
        h = make_float2(through_chunk(span * rate.x, h.x, local.x), through_chunk(span * rate.y, h.y, local.y));
    }
    return h;
}

// Row of `saved` for token t (a multiple of kSegment) of a sequence: segments
// of different sequences never share one.
__device__ __forceinline__ long segment_row(const Sequences &q, long s, long first, long t) {
    return (q.offsets == nullptr ? s * ((q.length + kSegment - 1) / kSegment) : first / kSegment + s) + t / kSegment;
}

// 1 / (1 + exp(-z)) of a gate.  Rows of 16 bits take the short form, whose
// exponent is rounded first (|z| 2^-24 of the result, far below the rows' own
// rounding).
template <typename T> __device__ __forceinline__ float gate_sigmoid(float z) {
    if (sizeof(T) == 4) return sigmoid_f(z);
    return reciprocal(1.f + exp2_unit(-kLog2e * z));
}

// An element between its load and its use: a whole register each.  As 16-bit
// variables, two of them are packed into one right behind their loads, which
// then wait there instead of running on under the tile before.
template <typename T> struct Raw {
    unsigned bits;
    __device__ __forceinline__ void load(const T *p) { bits = *reinterpret_cast<const unsigned short *>(p); }
    __device__ __forceinline__ float value() const;
};
template <> __device__ __forceinline__ float Raw<__nv_bfloat16>::value() const { return __uint_as_float(bits << 16); }
template <> __device__ __forceinline__ float Raw<__half>::value() const {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
}
template <> struct Raw<float> {
    unsigned bits;
    __device__ __forceinline__ void load(const float *p) { bits = __float_as_uint(*p); }
    __device__ __forceinline__ float value() const { return __uint_as_float(bits); }
};

// The rows of one operand as a CTA's threads read (or write) them, a tile of
// tokens at a time: the tile's first row and the CTA's first channel are the
// same for all threads (64 bits, moved on tile by tile), and what a thread adds
// to them is small.
template <typename T> struct Rows {
    T *tile;                // the tile's first row, at the CTA's first channel
    long advance;           // from one tile to the next
    unsigned offset, step;  // a thread's first element, and from one of its elements to the next
    __device__ __forceinline__ Rows(const void *p, long stride, long row, long c0, int t, int c, int rows, int tokens)
        : tile(const_cast<T *>(static_cast<const T *>(p)) + row * stride + c0), advance(tokens * stride),
          offset(t * static_cast<unsigned>(stride) + c), step(rows * static_cast<unsigned>(stride)) {}
    // o[i] is the element i * ROWS tokens on, zero where there is none; WHOLE: all of them exist
    template <bool WHOLE, int COUNT, int ROWS>
    __device__ __forceinline__ void load(Raw<T> (&o)[COUNT], int t, int count) {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            if (!WHOLE) o[i].bits = 0;
            if (WHOLE || t + i * ROWS < count) o[i].load(tile + (offset + i * step));
        }
        tile += advance;
    }
    __device__ __forceinline__ void store(int i, float v) const { tile[offset + i * step] = from_float<T>(v); }
};

// A tile's keys or queries, N padded to STATES, two states at a time: entries
// threadIdx.x + i * kThreads of [tile][STATES / 2].  PAIRED: both in one load
// (16-bit types: both in `first`).
template <typename T> struct KeyPair {
    Raw<T> first, second;
    __device__ __forceinline__ float2 value(bool paired) const {
        if (sizeof(T) == 4 || !paired) return make_float2(first.value(), second.value());
        return make_float2(Raw<T>{first.bits & 0xffffu}.value(), Raw<T>{first.bits >> 16}.value());
    }
};
template <typename T, int COUNT, int STATES>
__device__ __forceinline__ void load_keys(KeyPair<T> (&o)[COUNT], const T *&p, unsigned stride, long advance,
                                          int states, int count, bool paired) {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
        const unsigned e = threadIdx.x + i * kThreads, t = e / (STATES / 2), n = e % (STATES / 2) * 2;
        o[i].first.bits = o[i].second.bits = 0;
        if (t >= static_cast<unsigned>(count) || n >= static_cast<unsigned>(states)) continue;
        const T *q = p + (t * stride + n);
        if (sizeof(T) == 2 && paired) {
            o[i].first.bits = *reinterpret_cast<const unsigned *>(q);
        } else {
            o[i].first.load(q);
            if (n + 1 < static_cast<unsigned>(states)) o[i].second.load(q + 1);
        }
    }
    p += advance;
}
template <typename T> __device__ __forceinline__ bool keys_paired(const void *p, long stride, int states) {
    return (states & 1) == 0 && (stride & 1) == 0 && reinterpret_cast<uintptr_t>(p) % (2 * sizeof(T)) == 0;
}

// The next tile's rows are loaded while this one is scanned.
// bf16, N16, gate and skip: B8 T2048 C1024 with saved states 193 us (1.0 TB/s;
// 1.4e12 exponentials a second of 4.5e12), 24 ragged prompts C2048 316 us, the
// 9 chunks of B1 T8192 C1024 85 us.  Bound by issue slots (58 to 64 % used) and
// by what 16 to 24 warps an SM wait for; two adjacent channels a thread around
// the scan (half the loads and stores there) changed these by -3, +4 and -3 us.
template <typename T, int LPC> __global__ void __launch_bounds__(kThreads, 3) scan_forward(const ScanArgs a) {
    using G = Geometry<LPC>;
    __shared__ float2 in_s[G::kTile][G::kChannels];  // (d, d x)
    __shared__ float4 kq_s[G::kTile][LPC];           // (k, k, q, q) of a lane's states
    // q . h of a lane's states, [kTile][kThreads]: an object of its own, so that loads of the two above may be moved
    // over its stores
    extern __shared__ __align__(16) float part_s[];
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
    // scan: channel c, states n0 and n0 + 1
    const int sub = lane / G::kPerWarp, c = tid / 32 * G::kPerWarp + lane % G::kPerWarp, n0 = 2 * sub;
    const bool live = c < p.width && n0 < a.states;
    const long row = static_cast<long>(a.channels) * a.states, at = static_cast<long>(p.c0 + c) * a.states + n0;
    const float2 rate = load_rates(live ? a.rates + at : nullptr, n0, 0, a.states);
    float2 h = entering<false>(a, p.s, chunk, p.c0 + c, at, n0, 0, live, rate);

    const long row0 = p.first + p.begin;
    Rows<T> values(a.values, a.value_stride, row0, p.c0, er, ec, G::kRows, G::kTile);
    Rows<T> steps(a.steps, a.step_stride, row0, p.c0, er, ec, G::kRows, G::kTile);
    Rows<T> gate(a.gate, a.gate_stride, row0, p.c0, er, ec, G::kRows, G::kTile);
    Rows<T> out(a.out, a.channels, row0, p.c0, er, ec, G::kRows, G::kTile);
    const T *keys = static_cast<const T *>(a.keys) + row0 * a.key_stride + static_cast<long>(p.group) * a.states;
    const T *queries = static_cast<const T *>(a.queries) + row0 * a.query_stride + static_cast<long>(p.group) * a.states;
    const long keys_on = G::kTile * a.key_stride, queries_on = G::kTile * a.query_stride;
    const bool paired_k = keys_paired<T>(a.keys, a.key_stride, a.states);
    const bool paired_q = keys_paired<T>(a.queries, a.query_stride, a.states);
    float *saved = a.saved == nullptr ? nullptr : a.saved + segment_row(a.seq, p.s, p.first, p.begin) * row + at;
    const bool full_width = p.width == G::kChannels;
    Raw<T> next_x[G::kElems], next_s[G::kElems], next_z[G::kElems];
    KeyPair<T> next_k[G::kPairs], next_q[G::kPairs];
    auto load_rows = [&](auto whole, int count) {
        constexpr bool kWhole = decltype(whole)::value;
        steps.template load<kWhole, G::kElems, G::kRows>(next_s, er, count);
        values.template load<kWhole, G::kElems, G::kRows>(next_x, er, count);
        if (a.gate != nullptr) gate.template load<kWhole, G::kElems, G::kRows>(next_z, er, count);
    };
    auto load = [&](long left) {  // tokens from the tile's first on
        const int count = static_cast<int>(min(static_cast<long>(G::kTile), left));
        if (count == G::kTile && full_width) load_rows(std::true_type{}, count);
        else load_rows(std::false_type{}, own ? count : 0);
        load_keys<T, G::kPairs, G::kStates>(next_k, keys, static_cast<unsigned>(a.key_stride), keys_on, a.states, count,
                                            paired_k);
        load_keys<T, G::kPairs, G::kStates>(next_q, queries, static_cast<unsigned>(a.query_stride), queries_on,
                                            a.states, count, paired_q);
    };
    long left = p.end - p.begin;
    if (left > 0) load(left);
    int phase = 0;  // the tile's first token in its segment
    for (; left > 0; left -= G::kTile) {
        const int count = static_cast<int>(min(static_cast<long>(G::kTile), left));
        const bool whole = count == G::kTile && full_width;
        Raw<T> x[G::kElems], z[G::kElems];
        float d[G::kElems], unused;
#pragma unroll
        for (int i = 0; i < G::kElems; ++i) {
            x[i] = next_x[i];
            z[i] = next_z[i];
            d[i] = next_s[i].value() + bias;
        }
        if (a.softplus) {
#pragma unroll
            for (int i = 0; i < G::kElems; ++i) d[i] = softplus_f<false>(d[i], unused);
        }
        if (!whole) {
#pragma unroll
            for (int i = 0; i < G::kElems; ++i)
                if (!own || er + i * G::kRows >= count) d[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < G::kElems; ++i) {
            in_s[er + i * G::kRows][ec] = make_float2(d[i], d[i] * x[i].value());
        }
#pragma unroll
        for (int i = 0; i < G::kPairs; ++i) {
            const int e = tid + i * kThreads;
            if (G::kTile * LPC % kThreads == 0 || e < G::kTile * LPC) {
                const float2 k = next_k[i].value(paired_k), q = next_q[i].value(paired_q);
                (&kq_s[0][0])[e] = make_float4(k.x, k.y, q.x, q.y);
            }
        }
        if (left > G::kTile) load(left - G::kTile);
        __syncthreads();
        const float2 *in_at = &in_s[0][c];
        const float4 *kq_at = &kq_s[0][sub];
        float *part_at = part_s + c * LPC + sub;
        for (int tb = 0; tb < count; tb += 8) {
            if (saved != nullptr && (phase + tb) % kSegment == 0) {
                if (live) store_states(saved, n0, 0, a.states, h);
                saved += row;
            }
            // what does not depend on h first: only one FMA a token does
            float2 decay[8], inflow[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float2 in = in_at[u * G::kChannels], k = *reinterpret_cast<const float2 *>(kq_at + u * LPC);
                decay[u] = decay_of(in.x, rate);
                inflow[u] = mul2(both(in.y), k);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float2 q = *(reinterpret_cast<const float2 *>(kq_at + u * LPC) + 1);
                h = fma2(decay[u], h, inflow[u]);
                const float2 y = mul2(q, h);
                part_at[u * kThreads] = y.x + y.y;
            }
            in_at += 8 * G::kChannels;
            kq_at += 8 * LPC;
            part_at += 8 * kThreads;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < G::kElems; ++i) {
            const int t = er + i * G::kRows;
            float y = fmaf(skip, x[i].value(), sum_of<LPC>(part_s + t * kThreads, ec));
            if (a.gate != nullptr) y *= z[i].value() * gate_sigmoid<T>(z[i].value());
            if (whole || (own && t < count)) out.store(i, y);
        }
        out.tile += out.advance;
        phase = (phase + G::kTile) % kSegment;
        // no barrier here: the next tile's in and kq were last read before the one above, and its part is written
        // after the next one
    }
    if (live && a.state1 != nullptr && p.end == p.tokens) store_states(a.state1 + p.s * row + at, n0, 0, a.states, h);
}

// What a chunk does to the state that enters it, h -> exp(A D) h + local: the
// scan from a state of zero, its outputs left out, and the sum D of its steps.
// BACKWARD: the same of the adjoint, which enters at the chunk's end:
// g -> exp(A D) g + local with g_{t-1} = a_t (q_t dr_t + g_t).
// B1 T8192 C1024 N16 bf16, 9 chunks: 58 us, the exp2 unit at 51 %, the rest of
// the time waits of 16 warps an SM (two tiles in flight: 58.7 us against 56.8).
template <typename T, int LPC, bool BACKWARD>
__global__ void __launch_bounds__(kThreads, 3) scan_local(const ScanArgs a) {
    using G = Geometry<LPC>;
    __shared__ float2 in_s[G::kTile][G::kChannels];  // (d, d x) or (d, dr)
    __shared__ __align__(16) float k_s[G::kTile * G::kStates];
    const int chunk = static_cast<int>(blockIdx.y) + (BACKWARD ? 1 : 0);
    const Place p = place_of<LPC>(a, chunk);
    const int tid = threadIdx.x, lane = tid & 31;
    const int ec = tid % G::kChannels, er = tid / G::kChannels;
    const bool own = ec < p.width;
    const long cc = p.c0 + ec;
    const float bias = own && a.step_bias != nullptr ? a.step_bias[cc] : 0.f;
    const int sub = lane / G::kPerWarp, c = tid / 32 * G::kPerWarp + lane % G::kPerWarp, n0 = 2 * sub;
    const bool live = c < p.width && n0 < a.states;
    const long row = static_cast<long>(a.channels) * a.states, at = static_cast<long>(p.c0 + c) * a.states + n0;
    const float2 rate = load_rates(live ? a.rates + at : nullptr, n0, 0, a.states);
    float2 h = both(0.f);
    float span = 0.f;

    const long tiles = (p.end - p.begin + G::kTile - 1) / G::kTile;
    // BACKWARD walks the tiles from the last one down
    const long row0 = p.first + p.begin + (BACKWARD && tiles > 0 ? (tiles - 1) * G::kTile : 0);
    constexpr int kOn = BACKWARD ? -G::kTile : G::kTile;
    Rows<T> in(BACKWARD ? a.grad_out : a.values, BACKWARD ? a.channels : a.value_stride, row0, p.c0, er, ec, G::kRows,
               kOn);
    Rows<T> steps(a.steps, a.step_stride, row0, p.c0, er, ec, G::kRows, kOn);
    Rows<T> gate(a.gate, a.gate_stride, row0, p.c0, er, ec, G::kRows, kOn);
    const bool gated = BACKWARD && a.gate != nullptr, present = !BACKWARD || a.grad_out != nullptr;
    const long key_stride = BACKWARD ? a.query_stride : a.key_stride, keys_on = kOn * key_stride;
    const void *all_keys = BACKWARD ? a.queries : a.keys;
    const T *keys = static_cast<const T *>(all_keys) + row0 * key_stride + static_cast<long>(p.group) * a.states;
    const bool paired = keys_paired<T>(all_keys, key_stride, a.states), full_width = p.width == G::kChannels;
    Raw<T> x[G::kElems], s[G::kElems], z[G::kElems];
    KeyPair<T> k[G::kPairs];
    auto load_rows = [&](auto whole, int count) {
        constexpr bool kWhole = decltype(whole)::value;
        steps.template load<kWhole, G::kElems, G::kRows>(s, er, count);
        if (present) in.template load<kWhole, G::kElems, G::kRows>(x, er, count);
        else in.template load<false, G::kElems, G::kRows>(x, er, 0);
        if (gated) gate.template load<kWhole, G::kElems, G::kRows>(z, er, count);
    };
    auto load = [&](long tile) {
        const long t0 = p.begin + (BACKWARD ? tiles - 1 - tile : tile) * G::kTile;
        const int count = static_cast<int>(min(static_cast<long>(G::kTile), p.end - t0));
        if (count == G::kTile && full_width) load_rows(std::true_type{}, count);
        else load_rows(std::false_type{}, own ? count : 0);
        load_keys<T, G::kPairs, G::kStates>(k, keys, static_cast<unsigned>(key_stride), keys_on, a.states, count, paired);
        return count;
    };
    int count = tiles > 0 ? load(0) : 0;
    for (long tile = 0; tile < tiles; ++tile) {
        const bool whole = count == G::kTile && full_width;
        float d[G::kElems], unused;
#pragma unroll
        for (int i = 0; i < G::kElems; ++i) d[i] = s[i].value() + bias;
        if (a.softplus) {
#pragma unroll
            for (int i = 0; i < G::kElems; ++i) d[i] = softplus_f<false>(d[i], unused);
        }
        if (!whole) {
#pragma unroll
            for (int i = 0; i < G::kElems; ++i)
                if (!own || er + i * G::kRows >= count) d[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < G::kElems; ++i) {
            float v = x[i].value();
            if (gated) v *= z[i].value() * gate_sigmoid<T>(z[i].value());
            if (!BACKWARD) v *= d[i];
            span += d[i];
            in_s[er + i * G::kRows][ec] = make_float2(d[i], v);
        }
#pragma unroll
        for (int i = 0; i < G::kPairs; ++i) {
            const int e = tid + i * kThreads;
            if (G::kTile * LPC % kThreads == 0 || e < G::kTile * LPC)
                reinterpret_cast<float2 *>(k_s)[e] = k[i].value(paired);
        }
        if (tile + 1 < tiles) count = load(tile + 1);
        __syncthreads();
        for (int tb = 0; tb < G::kTile; tb += 8) {
            float2 decay[8], inflow[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int t = BACKWARD ? G::kTile - 1 - (tb + u) : tb + u;
                const float2 v = in_s[t][c], kk = *reinterpret_cast<const float2 *>(&k_s[t * G::kStates + n0]);
                decay[u] = decay_of(v.x, rate);
                inflow[u] = mul2(both(v.y), kk);
                if (BACKWARD) inflow[u] = mul2(decay[u], inflow[u]);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) h = fma2(decay[u], h, inflow[u]);
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
    const float rate = in_powers_of_two(a.rates[at]);
    const float *start = BACKWARD ? a.grad_state1 : a.state0;
    float h = start != nullptr ? start[i] : 0.f;
#pragma unroll 4
    for (int k = 0; k + 1 < a.chunks; ++k) {
        const long entry = s * a.chunks + (BACKWARD ? a.chunks - 1 - k : k);
        h = through_chunk(a.span[entry * a.channels + c] * rate, h, a.carry[entry * row + at]);
        a.carry[entry * row + at] = h;
    }
}

template <int LPC> struct BackwardShared {
    using G = Geometry<LPC>;
    static constexpr int kCopies = G::kPerWarp >= 2 ? 2 : 1;
    float4 in[kSegment][G::kChannels];      // d, d x, dr, x
    float2 slopes[kSegment][G::kChannels];  // d's slope in the step, dy silu'(z)
    // (k, k, q, q) of a lane's states, then (q, q, k, k) in the other order: both orders' keys in different banks
    float4 kq[kSegment][kCopies][LPC];
    float2 lane_ka[kSegment][kThreads];     // g . k and g . (A a h) of a lane's states
    float lane_r[kSegment][kThreads];       // q . h
    float part[kWarps][kSegment][2 * G::kStates];
};

// One CTA walks a chunk's segments of kSegment tokens from the last to the
// first: each is replayed from the state the forward saved at its start, its 16
// states kept in registers, then the adjoint runs back over them; the segment
// before it is loaded meanwhile.  Keys' and queries' gradients are summed over
// the warp's channels by exchanges, over the CTA's warps in shared memory and
// written as one row per channel tile of key_part [tiles][tokens][2][N];
// rates', skip's and step bias's as one row per chunk.  All are added up
// afterwards in a fixed order.
//
// A lane holds its two states in the order j ^ m, m the lowest bit that tells
// the warp's channels apart.  The two halves of the exchange over that bit then
// are the same registers in every lane and need no selects.
//
// B8 T2048 C1024 N16 bf16, gate and skip: 497 us, 1.1e12 exponentials a second
// of 4.5e12.  Bound by issue slots (54 %) and by shared memory's latency and
// queue: 128 registers leave 16 warps an SM.
template <typename T, int LPC> __global__ void __launch_bounds__(kThreads, LPC < 4 ? 1 : 2)
scan_backward(const ScanArgs a) {
    using G = Geometry<LPC>;
    using S = BackwardShared<LPC>;
    constexpr int kElems = (kSegment * G::kChannels + kThreads - 1) / kThreads;
    constexpr int kPairs = (kSegment * LPC + kThreads - 1) / kThreads;
    constexpr int kBatch = 8;  // tokens between which loads are kept apart (4: 528 us, 2: 546, against 514)
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
    const int sub = lane % LPC, in_warp = lane / LPC, c = warp * G::kPerWarp + in_warp, n0 = 2 * sub;
    const int m = G::kPerWarp >= 2 ? in_warp & 1 : 0, copy = S::kCopies == 2 ? m : 0;
    const bool keys_here = (in_warp & 2) != 0;
    const int part_at = (keys_here ? G::kStates : 0) + n0 + m;
    const bool live = c < p.width && n0 < a.states;
    const long row = static_cast<long>(a.channels) * a.states, at = static_cast<long>(p.c0 + c) * a.states + n0;
    const float2 rate = load_rates(live ? a.rates + at : nullptr, n0, m, a.states);
    float2 grate = both(0.f);
    float2 g = entering<true>(a, p.s, chunk, p.c0 + c, at, n0, m, live, rate);
    float gskip = 0.f, gbias = 0.f;

    const long segments = (p.end - p.begin + kSegment - 1) / kSegment;
    const long row0 = p.first + p.begin + (segments > 0 ? (segments - 1) * kSegment : 0);  // walked from the last down
    Rows<T> values(a.values, a.value_stride, row0, p.c0, er, ec, G::kRows, -kSegment);
    Rows<T> steps(a.steps, a.step_stride, row0, p.c0, er, ec, G::kRows, -kSegment);
    Rows<T> gate(a.gate, a.gate_stride, row0, p.c0, er, ec, G::kRows, -kSegment);
    Rows<T> above(a.grad_out, a.channels, row0, p.c0, er, ec, G::kRows, -kSegment);
    Rows<T> to_values(a.grad_values, a.channels, row0, p.c0, er, ec, G::kRows, -kSegment);
    T *to_steps = static_cast<T *>(a.grad_steps) + row0 * a.channels + p.c0;
    T *to_gate = static_cast<T *>(a.grad_gate) + row0 * a.channels + p.c0;
    float *key_part = a.key_part + (tile * a.seq.tokens + row0) * 2 * a.states;
    const T *keys = static_cast<const T *>(a.keys) + row0 * a.key_stride + static_cast<long>(p.group) * a.states;
    const T *queries = static_cast<const T *>(a.queries) + row0 * a.query_stride + static_cast<long>(p.group) * a.states;
    const bool paired_k = keys_paired<T>(a.keys, a.key_stride, a.states);
    const bool paired_q = keys_paired<T>(a.queries, a.query_stride, a.states);
    const bool full_width = p.width == G::kChannels && G::kRows <= kSegment;
    Raw<T> next_x[kElems], next_s[kElems], next_z[kElems], next_g[kElems];
    KeyPair<T> next_k[kPairs], next_q[kPairs];
    float2 next_h;
    auto load_rows = [&](auto whole, int count) {
        constexpr bool kWhole = decltype(whole)::value;
        steps.template load<kWhole, kElems, G::kRows>(next_s, er, count);
        values.template load<kWhole, kElems, G::kRows>(next_x, er, count);
        if (a.grad_out != nullptr) above.template load<kWhole, kElems, G::kRows>(next_g, er, count);
        else above.template load<false, kElems, G::kRows>(next_g, er, 0);
        if (a.gate != nullptr) gate.template load<kWhole, kElems, G::kRows>(next_z, er, count);
    };
    const float *saved = a.saved + segment_row(a.seq, p.s, p.first, row0 - p.first) * row + at;
    auto load = [&](int count) {
        if (count == kSegment && full_width) load_rows(std::true_type{}, count);
        else load_rows(std::false_type{}, own ? count : 0);
        load_keys<T, kPairs, G::kStates>(next_k, keys, static_cast<unsigned>(a.key_stride), -kSegment * a.key_stride,
                                         a.states, count, paired_k);
        load_keys<T, kPairs, G::kStates>(next_q, queries, static_cast<unsigned>(a.query_stride),
                                         -kSegment * a.query_stride, a.states, count, paired_q);
        next_h = load_states(live ? saved : nullptr, n0, m, a.states);
        saved -= row;
    };
    // only the last segment may be short
    int count = static_cast<int>(p.end - p.begin - (segments - 1) * kSegment);
    if (segments > 0) load(count);
    for (long seg = segments - 1; seg >= 0; --seg, count = kSegment) {
        const bool whole = count == kSegment && full_width;
#pragma unroll
        for (int i = 0; i < kElems; ++i) {
            const int t = er + i * G::kRows;
            if (G::kRows > kSegment && t >= kSegment) break;  // more threads than elements
            const float x = next_x[i].value();
            float d = next_s[i].value() + bias, dr = next_g[i].value(), slope = 1.f, gz = 0.f;
            if (a.softplus) d = softplus_f<true>(d, slope);
            if (!whole && (!own || t >= count)) d = 0.f;
            if (a.gate != nullptr) {
                const float z = next_z[i].value(), sg = gate_sigmoid<T>(z);
                gz = dr * sg * fmaf(z, 1.f - sg, 1.f);
                dr *= z * sg;
            }
            const float dx = d * x;
            sh.in[t][ec] = make_float4(d, dx, dr, x);
            sh.slopes[t][ec] = make_float2(slope, gz);  // read back by this thread only
        }
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            const int e = tid + i * kThreads, t = e / LPC, n = e % LPC;
            if (kSegment * LPC % kThreads == 0 || e < kSegment * LPC) {
                const float2 k = next_k[i].value(paired_k), q = next_q[i].value(paired_q);
                sh.kq[t][0][n] = make_float4(k.x, k.y, q.x, q.y);
                if (S::kCopies == 2) sh.kq[t][S::kCopies - 1][n] = make_float4(q.y, q.x, k.y, k.x);
            }
        }
        float2 h[kSegment + 1];  // h[t] before token t of the segment, h[t + 1] after it
        h[0] = next_h;
        if (seg > 0) load(kSegment);
        __syncthreads();
#pragma unroll
        for (int tb = 0; tb < kSegment; tb += 8) {
            asm volatile("" ::: "memory");  // as below
            float2 decay[8], inflow[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float2 in = *reinterpret_cast<const float2 *>(&sh.in[tb + u][c]);
                const float2 k = reinterpret_cast<const float2 *>(&sh.kq[tb + u][copy][sub])[copy];
                decay[u] = decay_of(in.x, rate);
                inflow[u] = mul2(both(in.y), k);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) h[tb + u + 1] = fma2(decay[u], h[tb + u], inflow[u]);
        }
#pragma unroll
        for (int tb = kSegment - kBatch; tb >= 0; tb -= kBatch) {
            asm volatile("" ::: "memory");  // keeps the compiler from loading later batches early, which spills
            float4 in[kBatch];
            float2 k[kBatch], q[kBatch], decay[kBatch], out_ka[kBatch], vqk[kBatch];
            float out_r[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                in[u] = sh.in[tb + u][c];
                k[u] = reinterpret_cast<const float2 *>(&sh.kq[tb + u][copy][sub])[copy];
                q[u] = reinterpret_cast<const float2 *>(&sh.kq[tb + u][copy][sub])[1 - copy];
            }
            // what does not depend on the adjoint first
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                decay[u] = decay_of(in[u].x, rate);
                const float2 pr = mul2(q[u], h[tb + u + 1]);
                out_r[u] = pr.x + pr.y;
            }
            float2 dk[kBatch];
#pragma unroll
            for (int u = kBatch - 1; u >= 0; --u) {
                const float2 gh = fma2(q[u], both(in[u].z), g);
                g = mul2(decay[u], gh);
                const float2 moved = mul2(g, h[tb + u]), pk = mul2(gh, k[u]), pa = mul2(moved, rate);
                dk[u] = mul2(gh, both(in[u].y));
                grate = fma2(moved, both(in[u].x), grate);
                out_ka[u] = make_float2(pk.x + pk.y, pa.x + pa.y);
            }
            // over the warp's channels: the states' exchange, then queries against keys, then plain sums
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const float2 dq = mul2(both(in[u].z), h[tb + u + 1]);
                if (G::kPerWarp == 1) {
                    float *part = sh.part[warp][tb + u] + n0;
                    *reinterpret_cast<float2 *>(part) = dq;
                    *reinterpret_cast<float2 *>(part + G::kStates) = dk[u];
                } else {
                    vqk[u] = make_float2(dq.x + __shfl_xor_sync(0xffffffffu, dq.y, LPC),
                                         dk[u].x + __shfl_xor_sync(0xffffffffu, dk[u].y, LPC));
                }
            }
            if (G::kPerWarp == 2) {
#pragma unroll
                for (int u = 0; u < kBatch; ++u) {
                    sh.part[warp][tb + u][n0 + m] = vqk[u].x;
                    sh.part[warp][tb + u][G::kStates + n0 + m] = vqk[u].y;
                }
            } else if (G::kPerWarp > 2) {
#pragma unroll
                for (int u = 0; u < kBatch; ++u) {
                    float v = (keys_here ? vqk[u].y : vqk[u].x) +
                              __shfl_xor_sync(0xffffffffu, keys_here ? vqk[u].x : vqk[u].y, 2 * LPC);
#pragma unroll
                    for (int off = 4 * LPC; off < 32; off *= 2) v += __shfl_xor_sync(0xffffffffu, v, off);
                    sh.part[warp][tb + u][part_at] = v;
                }
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                sh.lane_ka[tb + u][tid] = out_ka[u];
                sh.lane_r[tb + u][tid] = out_r[u];
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kElems; ++i) {
            const int t = er + i * G::kRows;
            if (whole || (own && t < count)) {
                const unsigned r = to_values.offset + i * to_values.step;
                const float4 in = sh.in[t][ec];
                const float x = in.w, dr = in.z;
                const float2 slope = sh.slopes[t][ec], ka = sums_of<LPC>(sh.lane_ka[t], ec);
                const float gd = fmaf(x, ka.x, kLn2 * ka.y) * slope.x;  // rates were in powers of two
                to_values.tile[r] = from_float<T>(fmaf(in.x, ka.x, skip * dr));
                to_steps[r] = from_float<T>(gd);
                if (a.gate != nullptr)
                    to_gate[r] = from_float<T>(slope.y * fmaf(skip, x, sum_of<LPC>(sh.lane_r[t], ec)));
                gbias += gd;
                gskip = fmaf(dr, x, gskip);
            }
        }
        const bool even = (a.states & 1) == 0;
        for (int i = tid; i < count * G::kStates; i += kThreads) {  // pairs of [token][2][kStates]
            const unsigned t = i / G::kStates, e = i % G::kStates * 2, which = e / G::kStates, n = e % G::kStates;
            float2 v = both(0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w)
                v = __fadd2_rn(v, *reinterpret_cast<const float2 *>(&sh.part[w][t][e]));
            float *o = key_part + (t * 2 + which) * a.states + n;
            if (even && n < a.states) {
                *reinterpret_cast<float2 *>(o) = v;
            } else if (n < a.states) {
                o[0] = v.x;
                if (n + 1 < a.states) o[1] = v.y;
            }
        }
        to_values.tile += to_values.advance;
        to_steps += to_values.advance;
        to_gate += to_values.advance;
        key_part -= kSegment * 2 * a.states;
        __syncthreads();
    }
    const long entry = p.s * a.chunks + chunk;
    if (live && a.grad_state0 != nullptr && chunk == 0)
        store_states(a.grad_state0 + p.s * row + at, n0, m, a.states, g);
    if (live) store_states(a.rate_part + entry * row + at, n0, m, a.states, grate);
    // the skip's and step bias's sums over the CTA's token rows
    float *cs = reinterpret_cast<float *>(&sh.in[0][0]);  // [2][kRows][kChannels]
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

// Everything that the chunks and tiles left in rows, added up in order: keys'
// and queries' gradients from key_part [tiles][tokens][2][N] (a group's tiles;
// VEC of N a thread), then rates', skip's and step bias's (the chunks).
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) scan_sums(const ScanArgs a, void *grad_keys, void *grad_queries,
                                                      float *grad_rates, float *grad_skip, float *grad_step_bias) {
    const long cols = a.seq.tokens * 2 * a.states, vecs = cols / VEC * a.groups;
    const long i = static_cast<long>(blockIdx.x) * kThreads + threadIdx.x;
    if (i < vecs) {
        const long group = a.groups == 1 ? 0 : i / (cols / VEC), col = (i - group * (cols / VEC)) * VEC;
        const long token = col / (2 * a.states);
        const int e = static_cast<int>(col - token * 2 * a.states), which = e >= a.states, n = e - which * a.states;
        const float *part = a.key_part + group * a.tiles_per_group * cols + col;
        float v[VEC] = {};
#pragma unroll 4
        for (int t = 0; t < a.tiles_per_group; ++t) {
            const Packed<float, VEC> p = load_packed<float, VEC>(part + t * cols);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] += p.e[j];
        }
        T *out = static_cast<T *>(which == 0 ? grad_queries : grad_keys);
        store_packed<T, VEC>(out + (token * a.groups + group) * a.states + n, v);
        return;
    }
    const long state = static_cast<long>(a.channels) * a.states, rows = a.seq.count * a.chunks;
    const long k = i - vecs;
    const long j = k - state;  // of 2 * channels: skip, then step bias
    if (j >= 2L * a.channels) return;
    const float *part = j < 0 ? a.rate_part + k : a.channel_part + j;
    const long pitch = j < 0 ? state : 2L * a.channels;
    float *out = j < 0 ? grad_rates + k
                 : j < a.channels ? (grad_skip == nullptr ? nullptr : grad_skip + j)
                                  : (grad_step_bias == nullptr ? nullptr : grad_step_bias + j - a.channels);
    if (out == nullptr) return;
    float v = 0.f;
#pragma unroll 8
    for (long r = 0; r < rows; ++r) v += part[r * pitch];
    *out = v;
}

// One token per sequence, the states [sequences][channels][N] moved on in
// place: bound by the states' traffic, 8 bytes each.  A lane holds VEC states
// (4 where N is a multiple of 4: 16-byte accesses) of a channel, LANES lanes (a
// power of two) the channel; it walks every gridDim.y-th sequence, so that
// rates and addresses are made once (77 -> 32 us), and loads a sequence ahead.
// B256 C4096 N16 bf16: 32 us for 143 MB, 4.4 TB/s, issue slots 72 % used; B1
// C1024 N16: 2.0 us, a launch's own time.
template <typename T, int VEC> struct StepKeys {  // VEC adjacent keys on their way: one word each, or packed
    unsigned w[VEC];
    __device__ __forceinline__ void load(const T *p, int n, bool wide) {
        if (sizeof(T) == 2 && VEC > 1 && wide) {
            const auto v = load_packed<unsigned, (VEC + 1) / 2>(reinterpret_cast<const unsigned *>(p));
#pragma unroll
            for (int j = 0; j < (VEC + 1) / 2; ++j) w[j] = v.e[j];
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                Raw<T> r{0};
                if (j < n) r.load(p + j);
                w[j] = r.bits;
            }
        }
    }
    __device__ __forceinline__ void values(bool wide, float (&o)[VEC]) const {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const unsigned pair = w[j / 2];
            const unsigned bits = sizeof(T) == 2 && VEC > 1 && wide ? (j % 2 == 0 ? pair & 0xffffu : pair >> 16) : w[j];
            o[j] = Raw<T>{bits}.value();
        }
    }
};

template <typename T, int VEC, int LANES>
__global__ void __launch_bounds__(kThreads, 4) scan_step(const ScanArgs a, float *state) {
    const int sub = threadIdx.x % LANES, n0 = VEC * sub;
    const int c = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
    const bool live = c < a.channels && n0 < a.states;
    const int n = live ? min(VEC, a.states - n0) : 0;
    const long group = a.groups == 1 ? 0 : c / a.group_channels;
    const long row = static_cast<long>(a.channels) * a.states, at = static_cast<long>(c) * a.states + n0;
    // whole vectors everywhere: VEC divides N, and the keys' rows are aligned to it
    const bool whole = a.states % VEC == 0;
    const auto aligned = [&](const void *p, long stride) {
        return whole && stride % VEC == 0 && reinterpret_cast<uintptr_t>(p) % (VEC * sizeof(T)) == 0;
    };
    const bool wide_k = aligned(a.keys, a.key_stride), wide_q = aligned(a.queries, a.query_stride);
    float rate[VEC], bias = 0.f, skip = 0.f;
#pragma unroll
    for (int j = 0; j < VEC; ++j) rate[j] = j < n ? in_powers_of_two(a.rates[at + j]) : 0.f;
    if (live && a.step_bias != nullptr) bias = a.step_bias[c];
    if (live && a.skip != nullptr) skip = a.skip[c];
    long s = blockIdx.y;
    float *h_at = state + s * row + at;
    const T *x_at = static_cast<const T *>(a.values) + s * a.value_stride + c;
    const T *d_at = static_cast<const T *>(a.steps) + s * a.step_stride + c;
    const T *z_at = static_cast<const T *>(a.gate) + s * a.gate_stride + c;
    const T *k_at = static_cast<const T *>(a.keys) + s * a.key_stride + group * a.states + n0;
    const T *q_at = static_cast<const T *>(a.queries) + s * a.query_stride + group * a.states + n0;
    T *out = static_cast<T *>(a.out) + s * a.channels + c;
    const long on = gridDim.y;
    float next_h[VEC];
    Raw<T> next_x{0}, next_d{0}, next_z{0};
    StepKeys<T, VEC> next_k{}, next_q{};
    auto load = [&]() {
        if (!live) return;
        if (whole) {
            const Packed<float, VEC> v = load_packed<float, VEC>(h_at);
#pragma unroll
            for (int j = 0; j < VEC; ++j) next_h[j] = v.e[j];
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) next_h[j] = j < n ? h_at[j] : 0.f;
        }
        next_x.load(x_at);
        next_d.load(d_at);
        if (a.gate != nullptr) next_z.load(z_at);
        next_k.load(k_at, n, wide_k);
        next_q.load(q_at, n, wide_q);
        x_at += on * a.value_stride;
        d_at += on * a.step_stride;
        z_at += on * a.gate_stride;
        k_at += on * a.key_stride;
        q_at += on * a.query_stride;
    };
#pragma unroll
    for (int j = 0; j < VEC; ++j) next_h[j] = 0.f;
    load();
    for (; s < a.seq.count; s += on) {
        float h[VEC], k[VEC], q[VEC], sum = 0.f, unused;
#pragma unroll
        for (int j = 0; j < VEC; ++j) h[j] = next_h[j];
        next_k.values(wide_k, k);
        next_q.values(wide_q, q);
        const float x = next_x.value(), z = next_z.value();
        float d = next_d.value() + bias;
        float *const to = h_at;
        h_at += on * row;
        if (s + on < a.seq.count) load();
        if (a.softplus) d = softplus_f<false>(d, unused);
        const float in = d * x;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            h[j] = fmaf(exp2_unit(fmaf(d, rate[j], kExponentBias)), h[j], in * k[j]);
            sum = fmaf(q[j], h[j], sum);
        }
        if (live && whole) {
            store_packed<float, VEC>(to, h);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (j < n) to[j] = h[j];
        }
#pragma unroll
        for (int off = LANES / 2; off >= 1; off /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        if (live && sub == 0) {
            sum = fmaf(skip, x, sum);
            if (a.gate != nullptr) sum *= z * gate_sigmoid<T>(z);
            *out = from_float<T>(sum);
        }
        out += on * a.channels;
    }
}

int lanes_per_channel(int states) {
    int lpc = 1;
    while (2 * lpc < states) lpc *= 2;
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
    a.joined = a.chunks > kChained;
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
    constexpr int bytes = Geometry<LPC>::kTile * kThreads * static_cast<int>(sizeof(float));
    if (cudaError_t e = cudaFuncSetAttribute(scan_forward<T, LPC>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes))
        return fail(BSSM_ERR_CUDA, "selective_scan: %s", cudaGetErrorString(e));
    const dim3 grid(static_cast<unsigned>(a.seq.count * a.tiles), static_cast<unsigned>(a.chunks));
    if (a.chunks > 1) {
        scan_local<T, LPC, false><<<dim3(grid.x, grid.y - 1), kThreads, 0, st>>>(a);
        if (a.joined) scan_join<false><<<blocks_for(a.seq.count * a.channels * a.states), kThreads, 0, st>>>(a);
    }
    scan_forward<T, LPC><<<grid, kThreads, bytes, st>>>(a);
    return check_launch("selective_scan");
}
template <typename T, int LPC> int launch_backward(const ScanArgs &a, cudaStream_t st) {
    constexpr int bytes = static_cast<int>(sizeof(BackwardShared<LPC>));
    if (cudaError_t e = cudaFuncSetAttribute(scan_backward<T, LPC>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes))
        return fail(BSSM_ERR_CUDA, "selective_scan_backward: %s", cudaGetErrorString(e));
    const dim3 grid(static_cast<unsigned>(a.seq.count * a.tiles), static_cast<unsigned>(a.chunks));
    if (a.chunks > 1) {
        scan_local<T, LPC, true><<<dim3(grid.x, grid.y - 1), kThreads, 0, st>>>(a);
        if (a.joined) scan_join<true><<<blocks_for(a.seq.count * a.channels * a.states), kThreads, 0, st>>>(a);
    }
    scan_backward<T, LPC><<<grid, kThreads, bytes, st>>>(a);
    return check_launch("selective_scan_backward");
}
template <typename T, int VEC, int LANES> int launch_step_as(const ScanArgs &a, cudaStream_t st) {
    // one wave of CTAs, four an SM
    const long columns = (static_cast<long>(a.channels) * LANES + kThreads - 1) / kThreads;
    long rows = 592 / columns;
    rows = rows < 1 ? 1 : rows < a.seq.count ? rows : a.seq.count;
    const dim3 grid(static_cast<unsigned>(columns), static_cast<unsigned>(rows));
    scan_step<T, VEC, LANES><<<grid, kThreads, 0, st>>>(a, a.state1);
    return check_launch("selective_step");
}
template <typename T, int LPC> int launch_step(const ScanArgs &a, cudaStream_t st) {
    if (a.states % 4 == 0) return launch_step_as<T, 4, LPC < 2 ? 1 : LPC / 2>(a, st);
    return launch_step_as<T, 2, LPC>(a, st);
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
        case 16: return launch_kind<T, 16>(kind, a, st);
        default: return launch_kind<T, 32>(kind, a, st);
    }
}
int launch_scan(ScanKind kind, int dtype, const ScanArgs &a, cudaStream_t st) {
    switch (dtype) {
        case BSSM_F32: return launch_lanes<float>(kind, a, st);
        case BSSM_BF16: return launch_lanes<__nv_bfloat16>(kind, a, st);
        default: return launch_lanes<__half>(kind, a, st);
    }
}

template <typename T>
void launch_sums_of(const ScanArgs &a, void *gk, void *gq, float *ga, float *gs, float *gb, cudaStream_t st) {
    const uintptr_t bits = reinterpret_cast<uintptr_t>(gk) | reinterpret_cast<uintptr_t>(gq);
    const long keys = a.seq.tokens * 2 * a.states * a.groups, rest = static_cast<long>(a.channels) * (a.states + 2);
    if (a.states % 4 == 0 && bits % (4 * sizeof(T)) == 0)
        scan_sums<T, 4><<<blocks_for(keys / 4 + rest), kThreads, 0, st>>>(a, gk, gq, ga, gs, gb);
    else
        scan_sums<T, 1><<<blocks_for(keys + rest), kThreads, 0, st>>>(a, gk, gq, ga, gs, gb);
}
void launch_sums(int dtype, const ScanArgs &a, void *gk, void *gq, float *ga, float *gs, float *gb, cudaStream_t st) {
    if (dtype == BSSM_F32) launch_sums_of<float>(a, gk, gq, ga, gs, gb, st);
    else if (dtype == BSSM_BF16) launch_sums_of<__nv_bfloat16>(a, gk, gq, ga, gs, gb, st);
    else launch_sums_of<__half>(a, gk, gq, ga, gs, gb, st);
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

// A tile's rows are addressed by 32-bit offsets from its first one.
bool strides_fit(const ScanArgs &a) {
    for (long stride : {a.value_stride, a.step_stride, a.key_stride, a.query_stride, a.gate_stride,
                        static_cast<long>(a.channels)})
        if (stride < 0 || stride > 0x7fffffffL / 64) return false;
    return true;
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
    if (!strides_fit(a)) return fail(BSSM_ERR_UNSUPPORTED, "selective_scan: row stride too large");
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
    if (!strides_fit(a)) return fail(BSSM_ERR_UNSUPPORTED, "selective_scan_backward: row stride too large");
    set_backward_chunks(a, longest);
    const long needed = place_backward(a, workspace);
    if (workspace_floats < needed || (needed > 0 && workspace == nullptr))
        return fail(BSSM_ERR_WORKSPACE, "selective_scan_backward: workspace too small");
    if (sequences > 0)
        if (int rc = launch_scan(kScanBackward, dtype, a, st)) return rc;
    launch_sums(dtype, a, grad_keys, grad_queries, grad_rates, grad_skip, grad_step_bias, st);
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
