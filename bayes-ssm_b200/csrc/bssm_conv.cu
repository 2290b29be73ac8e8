// bssm_conv.cu -- causal depthwise convolution over token rows, with SiLU.
//
//   u_t = bias + sum_j w_j x_{t-W+1+j},  y_t = u_t or u_t sigmoid(u_t)
//
// per channel, W = 2..4 taps, for sequences of equal length or packed one
// after the other.  Inputs before a sequence's start come from its state (its
// last W - 1 inputs, oldest first) or are zero; the state after the last token
// is written too, so a prompt can be continued in pieces or token by token.
// (catid/bayes-ssm's trainer has the length-4 form inside its mixer,
// example/train_6layer.py:160-191; bssm_envelope.cu fuses that one with the
// Bayesian mixer's features.)
//
// All of it is bound by the rows' traffic: x in and y out, or x and dy in and
// dx out.  A thread owns VEC adjacent channels (2 where the rows allow
// it) and walks a run of tokens with the window in registers, the next four
// tokens' loads in flight, so each row is read once apart from W - 1 rows per run.
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "bayes_ssm_b200.h"
#include "bssm_internal.h"
#include "bssm_io.cuh"

namespace bssm {
namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 4;  // tokens whose loads are in flight per thread

struct ConvArgs {
    const void *x, *weight, *bias, *state0, *grad_y, *grad_state1;
    void *y, *state1, *grad_x, *grad_state0;
    float *partial;
    long row_stride;
    Sequences seq;
    int channels, w_dtype, b_dtype, silu;
    long run, runs;
};

template <typename TW, int VEC, int W>
__device__ __forceinline__ void load_taps_of(const TW *weight, long c, float (&w)[W][VEC]) {
    constexpr int kCount = VEC * W;
    float v[kCount];
    constexpr int kStep = 16 / sizeof(TW) < kCount ? 16 / sizeof(TW) : kCount;
    const TW *p = weight + c * W;
    if (kCount % kStep == 0 && (kStep & (kStep - 1)) == 0 && reinterpret_cast<uintptr_t>(p) % (kStep * sizeof(TW)) == 0) {
#pragma unroll
        for (int o = 0; o < kCount; o += kStep) {
            const Packed<TW, kStep> q = load_packed<TW, kStep>(p + o);
#pragma unroll
            for (int e = 0; e < kStep; ++e) v[o + e] = to_float(q.e[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < kCount; ++e) v[e] = to_float(p[e]);
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) w[j][i] = v[i * W + j];
}
template <typename TW, int VEC> __device__ __forceinline__ void load_bias_of(const TW *bias, long c, float (&b)[VEC]) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) b[i] = to_float(bias[c + i]);
}
// The type is tested once, so that the loads go out together.
template <int VEC, int W>
__device__ __forceinline__ void load_taps(const ConvArgs &a, long c, float (&w)[W][VEC], float (&b)[VEC]) {
    if (a.w_dtype == BSSM_F32) load_taps_of(static_cast<const float *>(a.weight), c, w);
    else if (a.w_dtype == BSSM_BF16) load_taps_of(static_cast<const __nv_bfloat16 *>(a.weight), c, w);
    else load_taps_of(static_cast<const __half *>(a.weight), c, w);
    if (a.bias == nullptr) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) b[i] = 0.f;
    } else if (a.b_dtype == BSSM_F32) load_bias_of(static_cast<const float *>(a.bias), c, b);
    else if (a.b_dtype == BSSM_BF16) load_bias_of(static_cast<const __nv_bfloat16 *>(a.bias), c, b);
    else load_bias_of(static_cast<const __half *>(a.bias), c, b);
}

// The input at row `g` of sequence s, whose first row is `first`: a row before
// it is the state's (first - g of at most W - 1 back) or zero.
template <typename T, int VEC, int W>
__device__ __forceinline__ void load_input(const ConvArgs &a, long s, long first, long g, long c, float (&o)[VEC]) {
    if (g >= first) {
        widen(load_packed<T, VEC>(static_cast<const T *>(a.x) + g * a.row_stride + c), o);
    } else if (a.state0 != nullptr) {
        const long row = s * (W - 1) + (g - first + W - 1);
        widen(load_packed<T, VEC>(static_cast<const T *>(a.state0) + row * a.channels + c), o);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = 0.f;
    }
}

// acc += a b, two channels an instruction
template <int VEC>
__device__ __forceinline__ void fma_to(float (&acc)[VEC], const float (&a)[VEC], const float (&b)[VEC]) {
    if constexpr (VEC == 1) {
        acc[0] = fmaf(a[0], b[0], acc[0]);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
            const float2 r = __ffma2_rn(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]),
                                        make_float2(acc[i], acc[i + 1]));
            acc[i] = r.x;
            acc[i + 1] = r.y;
        }
    }
}

// u of one token from the window (the W - 1 inputs before it) and its own input
template <int VEC, int W>
__device__ __forceinline__ void preactivation(const float (&w)[W][VEC], const float (&b)[VEC],
                                              const float (&win)[W - 1][VEC], const float (&x)[VEC],
                                              float (&u)[VEC]) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) u[i] = b[i];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) fma_to(u, w[j], win[j]);
    fma_to(u, w[W - 1], x);
}

// 1 / (1 + exp(-u)).  Rows of 16 bits take the short form, whose exponent is
// rounded first (|u| 2^-24 of the result, far below the rows' own rounding).
template <typename T> __device__ __forceinline__ float sigmoid_for(float u) {
    if (sizeof(T) == 4) return sigmoid_f(u);
    return __fdividef(1.f, 1.f + __expf(-u));
}

template <int VEC, int ROWS> __device__ __forceinline__ void slide(float (&win)[ROWS][VEC], const float (&x)[VEC]) {
#pragma unroll
    for (int j = 0; j + 1 < ROWS; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) win[j][i] = win[j + 1][i];
#pragma unroll
    for (int i = 0; i < VEC; ++i) win[ROWS - 1][i] = x[i];
}

template <typename T> __device__ __forceinline__ float silu_slope(float u) {
    const float s = sigmoid_for<T>(u);
    return s * fmaf(u, 1.f - s, 1.f);
}

// Threads 0 .. nvec * runs - 1 walk one run of tokens each; the threads after
// them write the states after the last tokens, one state row each.
// B8 T2048 C2048 bf16, SiLU: 41 us for 134 MB, 3.3 TB/s, bound by issue slots
// (65 % used); 37 packed prompts of f32, C771: 18 us.
template <typename T, int VEC, int W> __global__ void __launch_bounds__(kThreads, 4) conv_forward(const ConvArgs a) {
    const long nvec = a.channels / VEC;
    const long id = static_cast<long>(blockIdx.x) * kThreads + threadIdx.x;
    const long c = id % nvec * VEC, r = id / nvec;
    if (r >= a.runs) {
        const long row = r - a.runs;  // s * (W - 1) + m
        if (row >= a.seq.count * (W - 1) || a.state1 == nullptr) return;
        const long s = row / (W - 1), m = row % (W - 1);
        const long first = a.seq.begin(s), last = max(first, a.seq.end(s));
        float v[VEC];
        load_input<T, VEC, W>(a, s, first, last - (W - 1) + m, c, v);
        store_packed<T, VEC>(static_cast<T *>(a.state1) + row * a.channels + c, v);
        return;
    }
    const T *x = static_cast<const T *>(a.x) + c;
    T *y = static_cast<T *>(a.y) + c;
    float w[W][VEC], b[VEC];
    load_taps<VEC, W>(a, c, w, b);
    auto emit = [&](long g, const float (&win)[W - 1][VEC], const float (&v)[VEC]) {
        float u[VEC];
        preactivation<VEC, W>(w, b, win, v, u);
        if (a.silu) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) u[i] *= sigmoid_for<T>(u[i]);
        }
        store_packed<T, VEC>(y + g * a.channels, u);
    };
    long g = r * a.run;
    const long stop = min(g + a.run, a.seq.tokens);
    for (long s = a.seq.find(g); g < stop && s < a.seq.count; ++s) {
        const long first = a.seq.begin(s), last = min(stop, a.seq.end(s));
        if (g < first) g = first;
        if (g >= last) continue;
        float win[W - 1][VEC];
#pragma unroll
        for (int j = 0; j < W - 1; ++j) load_input<T, VEC, W>(a, s, first, g - (W - 1) + j, c, win[j]);
        RawVec<T, VEC> p[kAhead];
        auto load = [&](long t) {
            if (t + kAhead > last) return;
#pragma unroll
            for (int k = 0; k < kAhead; ++k) p[k].load(x + (t + k) * a.row_stride);
        };
        load(g);
        for (; g + kAhead <= last; g += kAhead) {
            RawVec<T, VEC> now[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) now[k] = p[k];
            load(g + kAhead);
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                float v[VEC];
                now[k].values(v);
                emit(g + k, win, v);
                slide<VEC, W - 1>(win, v);
            }
        }
        for (; g < last; ++g) {
            float v[VEC];
            widen(load_packed<T, VEC>(x + g * a.row_stride), v);
            emit(g, win, v);
            slide<VEC, W - 1>(win, v);
        }
    }
}

// Backward.  With du_t = dy_t act'(u_t):
//   dx_t = sum_j w_j du_{t+W-1-j},  dw_j = sum_t du_t x_{t-W+1+j},  db = sum_t du_t
// within each sequence; dx of the last W - 1 rows also takes the final state's
// gradient.  u is computed again from x (its one extra pass over registers is
// cheaper than 2 bytes per element saved by the forward).  A thread walks W - 1
// tokens past its run for the du they need; the run's dw and db stay in
// registers and are written as one row of `partial` [runs][W + 1][channels],
// which conv_sum_partials adds up in a fixed order.
// B8 T2048 C2048 bf16, SiLU: 74 us for 201 MB, 2.7 TB/s, bound by issue slots
// (59 %) and by what 24 warps an SM wait for.
template <typename T, int VEC, int W> __global__ void __launch_bounds__(kThreads, 3) conv_backward(const ConvArgs a) {
    const long nvec = a.channels / VEC;
    const long id = static_cast<long>(blockIdx.x) * kThreads + threadIdx.x;
    const long c = id % nvec * VEC, r = id / nvec;
    const T *x = static_cast<const T *>(a.x) + c;
    const T *gy = static_cast<const T *>(a.grad_y) + c;
    const T *gs = static_cast<const T *>(a.grad_state1);
    float w[W][VEC], b[VEC];
    if (r >= a.runs) {
        // gradient of one row of the state a sequence began with: the input W - 1 - m rows before the start
        const long row = r - a.runs;
        if (row >= a.seq.count * (W - 1) || a.grad_state0 == nullptr) return;
        load_taps<VEC, W>(a, c, w, b);
        const long s = row / (W - 1), m = row % (W - 1);
        const long first = a.seq.begin(s), last = max(first, a.seq.end(s));
        float acc[VEC] = {};
        // tokens first .. first + m read it, with tap m - t
        for (long t = 0; t <= m && first + t < last; ++t) {
            float win[W - 1][VEC], v[VEC], u[VEC], dy[VEC];
#pragma unroll
            for (int j = 0; j < W - 1; ++j) load_input<T, VEC, W>(a, s, first, first + t - (W - 1) + j, c, win[j]);
            load_input<T, VEC, W>(a, s, first, first + t, c, v);
            preactivation<VEC, W>(w, b, win, v, u);
            widen(load_packed<T, VEC>(gy + (first + t) * a.channels), dy);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float du = a.silu ? dy[i] * silu_slope<T>(u[i]) : dy[i];
                float tap = 0.f;
#pragma unroll
                for (int j = 0; j < W - 1; ++j) tap = j == m - t ? w[j][i] : tap;
                acc[i] = fmaf(tap, du, acc[i]);
            }
        }
        // a sequence shorter than the state keeps some of it
        const long kept = m - (last - first);
        if (gs != nullptr && kept >= 0) {
            float v[VEC];
            widen(load_packed<T, VEC>(gs + (s * (W - 1) + kept) * a.channels + c), v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[i] += v[i];
        }
        store_packed<T, VEC>(static_cast<T *>(a.grad_state0) + row * a.channels + c, acc);
        return;
    }
    load_taps<VEC, W>(a, c, w, b);
    T *gx = static_cast<T *>(a.grad_x) + c;
    float dw[W][VEC] = {}, db[VEC] = {};
    long g = r * a.run;
    const long stop = min(g + a.run, a.seq.tokens);
    for (long s = a.seq.find(g); g < stop && s < a.seq.count; ++s) {
        const long first = a.seq.begin(s), last = a.seq.end(s);  // of the sequence
        if (g < first) g = first;
        const long lo = g, hi = min(stop, last);  // the piece whose dx this thread writes
        if (lo >= hi) continue;
        float win[W - 1][VEC], past[W - 1][VEC];  // inputs and du before the token at hand
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
            load_input<T, VEC, W>(a, s, first, lo - (W - 1) + j, c, win[j]);
#pragma unroll
            for (int i = 0; i < VEC; ++i) past[j][i] = 0.f;
        }
        // Token t: its du, the run's dw and db where t is the run's, and dx of W - 1 tokens before.  INNER: all of
        // these are the run's and no final state's gradient comes in.
        auto advance = [&](auto inner, long t, const float (&v)[VEC], float (&du)[VEC]) {
            constexpr bool kInner = decltype(inner)::value;
            if (a.silu) {
                float u[VEC];
                preactivation<VEC, W>(w, b, win, v, u);
#pragma unroll
                for (int i = 0; i < VEC; ++i) du[i] *= silu_slope<T>(u[i]);
            }
            if (kInner || t < hi) {
#pragma unroll
                for (int j = 0; j < W - 1; ++j) fma_to(dw[j], du, win[j]);
                fma_to(dw[W - 1], du, v);
#pragma unroll
                for (int i = 0; i < VEC; ++i) db[i] += du[i];
            }
            const long out = t - (W - 1);
            if (kInner || out >= lo) {
                float o[VEC] = {};
                const long kept = out - (last - (W - 1));
                if (!kInner && gs != nullptr && kept >= 0)
                    widen(load_packed<T, VEC>(gs + (s * (W - 1) + kept) * a.channels + c), o);
                fma_to(o, w[0], du);
#pragma unroll
                for (int j = 0; j < W - 1; ++j) fma_to(o, w[W - 1 - j], past[j]);
                store_packed<T, VEC>(gx + out * a.channels, o);
            }
            slide<VEC, W - 1>(win, v);
            slide<VEC, W - 1>(past, du);
        };
        auto edge = [&](long t) {  // a token at either end of the piece, or past the sequence's
            float v[VEC] = {}, du[VEC] = {};
            if (t < last) {
                widen(load_packed<T, VEC>(x + t * a.row_stride), v);
                widen(load_packed<T, VEC>(gy + t * a.channels), du);
            }
            advance(std::false_type{}, t, v, du);
        };
        long t = lo;
        for (; t < lo + W - 1 && t < hi + W - 1; ++t) edge(t);
        RawVec<T, VEC> next_x[kAhead], next_g[kAhead];
        auto load = [&](long from) {
            if (from + kAhead > hi) return;
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                next_x[k].load(x + (from + k) * a.row_stride);
                next_g[k].load(gy + (from + k) * a.channels);
            }
        };
        load(t);
        for (; t + kAhead <= hi; t += kAhead) {
            RawVec<T, VEC> px[kAhead], pg[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                px[k] = next_x[k];
                pg[k] = next_g[k];
            }
            load(t + kAhead);
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                float v[VEC], du[VEC];
                px[k].values(v);
                pg[k].values(du);
                advance(std::true_type{}, t + k, v, du);
            }
        }
        for (; t < hi + W - 1; ++t) edge(t);
        g = hi;
    }
    float *p = a.partial + r * (W + 1) * a.channels + c;
#pragma unroll
    for (int j = 0; j < W; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) p[static_cast<long>(j) * a.channels + i] = dw[j][i];
#pragma unroll
    for (int i = 0; i < VEC; ++i) p[static_cast<long>(W) * a.channels + i] = db[i];
}

// Rows of partial [runs][W + 1][channels] added up: grad_weight [channels][W]
// and grad_bias [channels].  A CTA takes `columns` of them, and its threads a
// column's runs in turn.  Few runs of wide rows want whole 128-byte lines (75
// runs of 20,480 columns: 4.3 us, against 7.7 by 8 columns), many runs of
// narrow rows more threads a column (8,192 runs of 320 columns: 7.7 us with
// 128 of them, 15.6 with 32, 39 with 8; 1,024 runs of 2,560: 6.7, 4.9, 7.5).
constexpr int kSumThreads = 1024;
__global__ void __launch_bounds__(kSumThreads) conv_sum_partials(const float *partial, long runs, int taps,
                                                                 long channels, int columns, void *grad_weight,
                                                                 int w_dtype, void *grad_bias, int b_dtype) {
    __shared__ float part[kSumThreads];
    const long cols = (taps + 1) * channels;
    const int in = threadIdx.x % columns, lane = threadIdx.x / columns, lanes = blockDim.x / columns;
    const long col = static_cast<long>(blockIdx.x) * columns + in;
    float acc = 0.f;
    if (col < cols) {
#pragma unroll 8
        for (long r = lane; r < runs; r += lanes) acc += partial[r * cols + col];
    }
    part[threadIdx.x] = acc;
    for (int half = lanes / 2; half > 0; half /= 2) {
        __syncthreads();
        if (lane < half) part[threadIdx.x] += part[threadIdx.x + half * columns];
    }
    if (lane != 0 || col >= cols) return;
    acc = part[in];
    const long j = col / channels, c = col % channels;
    if (j < taps) store_from_float(grad_weight, w_dtype, c * taps + j, acc);
    else if (grad_bias != nullptr) store_from_float(grad_bias, b_dtype, c, acc);
}

// One token per sequence: y from the state and x, and the state moved on.  B64
// C2048 f16: 2.1 us, a launch's own time.
template <typename T, int VEC, int W> __global__ void __launch_bounds__(kThreads) conv_step(const ConvArgs a) {
    const long nvec = a.channels / VEC;
    const long id = static_cast<long>(blockIdx.x) * kThreads + threadIdx.x;
    const long c = id % nvec * VEC, s = id / nvec;
    if (s >= a.seq.count) return;
    T *state = static_cast<T *>(a.state1) + s * (W - 1) * a.channels + c;
    Packed<T, VEC> rows[W];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) rows[j] = load_packed<T, VEC>(state + static_cast<long>(j) * a.channels);
    rows[W - 1] = load_packed<T, VEC>(static_cast<const T *>(a.x) + s * a.row_stride + c);
    float w[W][VEC], b[VEC], win[W - 1][VEC], v[VEC], u[VEC];
    load_taps<VEC, W>(a, c, w, b);
#pragma unroll
    for (int j = 0; j < W - 1; ++j) widen(rows[j], win[j]);
    widen(rows[W - 1], v);
    preactivation<VEC, W>(w, b, win, v, u);
    if (a.silu) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) u[i] *= sigmoid_for<T>(u[i]);
    }
    store_packed<T, VEC>(static_cast<T *>(a.y) + s * a.channels + c, u);
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
        *reinterpret_cast<Packed<T, VEC> *>(state + static_cast<long>(j) * a.channels) = rows[j + 1];
}

enum ConvKind { kForward, kBackward, kStep };

template <typename T, int VEC, int W> int launch_conv(ConvKind kind, const ConvArgs &a, cudaStream_t st) {
    const long nvec = a.channels / VEC;
    const long rows = kind == kStep ? a.seq.count : a.runs + a.seq.count * (W - 1);
    const long blocks = (nvec * rows + kThreads - 1) / kThreads;
    if (blocks > 0x7fffffffL) return fail(BSSM_ERR_INVALID, "causal_conv: too many rows");
    const unsigned grid = static_cast<unsigned>(blocks);
    if (kind == kForward) conv_forward<T, VEC, W><<<grid, kThreads, 0, st>>>(a);
    else if (kind == kBackward) conv_backward<T, VEC, W><<<grid, kThreads, 0, st>>>(a);
    else conv_step<T, VEC, W><<<grid, kThreads, 0, st>>>(a);
    return check_launch("causal_conv");
}

template <typename T, int VEC> int pick_taps(ConvKind kind, int taps, const ConvArgs &a, cudaStream_t st) {
    switch (taps) {
        case 2: return launch_conv<T, VEC, 2>(kind, a, st);
        case 3: return launch_conv<T, VEC, 3>(kind, a, st);
        default: return launch_conv<T, VEC, 4>(kind, a, st);
    }
}

// Two channels a thread where the channel count, the row stride and every
// address allow it.  Four or eight would make 8- or 16-byte loads, but taps,
// windows and loads in flight then leave few warps an SM or spill.
template <typename T> int pick_vector(ConvKind kind, int taps, const ConvArgs &a, cudaStream_t st) {
    uintptr_t bits = 0;
    for (const void *p : {a.x, a.state0, a.grad_y, a.grad_state1, static_cast<const void *>(a.y),
                          static_cast<const void *>(a.state1), static_cast<const void *>(a.grad_x),
                          static_cast<const void *>(a.grad_state0)})
        bits |= reinterpret_cast<uintptr_t>(p);
    bits |= static_cast<uintptr_t>(a.channels) * sizeof(T) | static_cast<uintptr_t>(a.row_stride) * sizeof(T);
    if (bits % (2 * sizeof(T)) == 0) return pick_taps<T, 2>(kind, taps, a, st);
    return pick_taps<T, 1>(kind, taps, a, st);
}

int pick_type(ConvKind kind, int dtype, int taps, const ConvArgs &a, cudaStream_t st) {
    switch (dtype) {
        case BSSM_F32: return pick_vector<float>(kind, taps, a, st);
        case BSSM_BF16: return pick_vector<__nv_bfloat16>(kind, taps, a, st);
        default: return pick_vector<__half>(kind, taps, a, st);
    }
}

// Tokens per run: long enough that the rows before (and, backward, after) it
// and its partial sums are a small part of its traffic, short enough to give
// every SM a few hundred threads.
long run_length(long tokens, long channels, long longest) {
    long run = longest;
    while (run > 4 && (tokens + run - 1) / run * channels / 4 < 148L * 512) run /= 2;
    return run;
}

int check_common(const char *what, int dtype, int channels, int taps, int w_dtype, int b_dtype, const void *bias,
                 long sequences, long tokens) {
    if (!io_dtype_known(dtype) || !io_dtype_known(w_dtype) || (bias != nullptr && !io_dtype_known(b_dtype)))
        return fail(BSSM_ERR_UNSUPPORTED, "%s: unknown dtype", what);
    if (taps < 2 || taps > 4) return fail(BSSM_ERR_UNSUPPORTED, "%s: %d taps (2, 3 and 4 are built)", what, taps);
    if (channels < 1 || sequences < 0 || tokens < 0) return fail(BSSM_ERR_INVALID, "%s: bad sizes", what);
    return BSSM_OK;
}

Sequences make_sequences(const long *offsets, long sequences, long tokens) {
    return {offsets, sequences, sequences > 0 ? tokens / sequences : 0, tokens};
}

}  // namespace
}  // namespace bssm

extern "C" int bssm_causal_conv(const void *x, int dtype, long row_stride, long tokens, int channels, int taps,
                                const void *weight, int weight_dtype, const void *bias, int bias_dtype, int silu,
                                const long *offsets, long sequences, const void *state0, void *y, void *state1,
                                void *stream) {
    using namespace bssm;
    if (int rc = check_common("causal_conv", dtype, channels, taps, weight_dtype, bias_dtype, bias, sequences, tokens))
        return rc;
    if (sequences == 0 && tokens > 0) return fail(BSSM_ERR_INVALID, "causal_conv: rows without a sequence");
    if (sequences == 0) return BSSM_OK;
    if (weight == nullptr || (tokens > 0 && (x == nullptr || y == nullptr)))
        return fail(BSSM_ERR_INVALID, "causal_conv: null pointer");
    if (offsets == nullptr && tokens % sequences != 0)
        return fail(BSSM_ERR_INVALID, "causal_conv: rows do not divide into sequences of one length");
    if (row_stride < channels) return fail(BSSM_ERR_INVALID, "causal_conv: row stride below the channels");
    ConvArgs a{};
    a.x = x; a.weight = weight; a.bias = bias; a.state0 = state0; a.y = y; a.state1 = state1;
    a.row_stride = row_stride; a.seq = make_sequences(offsets, sequences, tokens);
    a.channels = channels; a.w_dtype = weight_dtype; a.b_dtype = bias_dtype; a.silu = silu;
    a.run = run_length(tokens, channels, 32);
    a.runs = (tokens + a.run - 1) / a.run;
    return pick_type(kForward, dtype, taps, a, static_cast<cudaStream_t>(stream));
}

extern "C" long bssm_causal_conv_partial_floats(long tokens, int channels, int taps) {
    const long run = bssm::run_length(tokens, channels, 64);
    return (tokens + run - 1) / run * (taps + 1) * channels;
}

extern "C" int bssm_causal_conv_backward(const void *x, int dtype, long row_stride, long tokens, int channels,
                                         int taps, const void *weight, int weight_dtype, const void *bias,
                                         int bias_dtype, int silu, const long *offsets, long sequences,
                                         const void *state0, const void *grad_y, const void *grad_state1,
                                         void *grad_x, void *grad_weight, void *grad_bias, void *grad_state0,
                                         float *workspace, long workspace_floats, void *stream) {
    using namespace bssm;
    if (int rc = check_common("causal_conv_backward", dtype, channels, taps, weight_dtype, bias_dtype, bias, sequences,
                              tokens))
        return rc;
    if (sequences == 0 && tokens > 0) return fail(BSSM_ERR_INVALID, "causal_conv_backward: rows without a sequence");
    if (weight == nullptr || grad_weight == nullptr || (grad_bias != nullptr && bias == nullptr) ||
        (tokens > 0 && (x == nullptr || grad_y == nullptr || grad_x == nullptr || workspace == nullptr)))
        return fail(BSSM_ERR_INVALID, "causal_conv_backward: null pointer");
    if (offsets == nullptr && sequences > 0 && tokens % sequences != 0)
        return fail(BSSM_ERR_INVALID, "causal_conv_backward: rows do not divide into sequences of one length");
    if (row_stride < channels) return fail(BSSM_ERR_INVALID, "causal_conv_backward: row stride below the channels");
    if (workspace_floats < bssm_causal_conv_partial_floats(tokens, channels, taps))
        return fail(BSSM_ERR_WORKSPACE, "causal_conv_backward: workspace too small");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    ConvArgs a{};
    a.x = x; a.weight = weight; a.bias = bias; a.state0 = state0; a.grad_y = grad_y; a.grad_state1 = grad_state1;
    a.grad_x = grad_x; a.grad_state0 = grad_state0; a.partial = workspace;
    a.row_stride = row_stride; a.seq = make_sequences(offsets, sequences, tokens);
    a.channels = channels; a.w_dtype = weight_dtype; a.b_dtype = bias_dtype; a.silu = silu;
    a.run = run_length(tokens, channels, 64);
    a.runs = (tokens + a.run - 1) / a.run;
    if (sequences > 0)
        if (int rc = pick_type(kBackward, dtype, taps, a, st)) return rc;
    const long cols = static_cast<long>(taps + 1) * channels;
    const int columns = a.runs < 128 ? 32 : 8, threads = a.runs < 2048 ? 256 : kSumThreads;
    conv_sum_partials<<<static_cast<unsigned>((cols + columns - 1) / columns), threads, 0, st>>>(
        workspace, a.runs, taps, channels, columns, grad_weight, weight_dtype, grad_bias, bias_dtype);
    return check_launch("causal_conv_backward");
}

extern "C" int bssm_causal_conv_step(const void *x, int dtype, long row_stride, long sequences, int channels, int taps,
                                     const void *weight, int weight_dtype, const void *bias, int bias_dtype, int silu,
                                     void *state, void *y, void *stream) {
    using namespace bssm;
    if (int rc = check_common("causal_conv_step", dtype, channels, taps, weight_dtype, bias_dtype, bias, sequences, 0))
        return rc;
    if (sequences == 0) return BSSM_OK;
    if (x == nullptr || weight == nullptr || state == nullptr || y == nullptr)
        return fail(BSSM_ERR_INVALID, "causal_conv_step: null pointer");
    if (row_stride < channels) return fail(BSSM_ERR_INVALID, "causal_conv_step: row stride below the channels");
    ConvArgs a{};
    a.x = x; a.weight = weight; a.bias = bias; a.y = y; a.state1 = state; a.row_stride = row_stride;
    a.seq = {nullptr, sequences, 1, sequences};
    a.channels = channels; a.w_dtype = weight_dtype; a.b_dtype = bias_dtype; a.silu = silu;
    return pick_type(kStep, dtype, taps, a, static_cast<cudaStream_t>(stream));
}
