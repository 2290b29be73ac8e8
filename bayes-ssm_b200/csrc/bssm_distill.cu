// bssm_distill.cu -- distillation from a teacher's top logits.
//
// Per row: the teacher gives K logits t_k at vocabulary entries i_k (an entry
// below zero, or a logit of -inf, is empty), the student V logits s.  With
// p = softmax(t / tau) over the K entries and q = softmax(s / tau) over V,
//
//   loss = tau^2 sum_k p_k (log p_k - log q_{i_k})
//   ds_j = tau (q_j - sum_k [i_k = j] p_k) * upstream
//
// A row whose entries are all empty has no teacher: loss and gradient are
// zero, and a mean does not count it.  An entry at or past V, or a teacher's
// logit of NaN or +inf, makes the row's loss and gradient NaN (nothing is read
// or written out of range).
//
// The traffic of the logits bounds it: read once, and the gradient written
// once.  A CTA takes a row (where rows are few, a cluster of CTAs takes one,
// each a stretch of the vocabulary): a pass for the running reference and sum,
// and, where the gradient is wanted, a second one over logits that are then in
// L2 (6 CTAs an SM with stretches of up to 80 KB are 71 of its 126 MB; a row of
// more than 8 such stretches has longer ones, which may outgrow it).  The K
// entries are corrected afterwards, from the logits again rather than from the
// rounded gradient.  Sums are float32, taken in an order that sizes alone decide.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "bayes_ssm_b200.h"
#include "bssm_internal.h"
#include "bssm_io.cuh"

namespace bssm {
namespace {

constexpr int kThreadsAnSM = 1536;  // 6 CTAs of 256 threads, 12 of 128 or 24 of 64
constexpr int kRescaleThreadsAnSM = 1280;  // 48 registers: a loop over rows does not fit 40 (64: within 3 %)
constexpr long kStretchBytes = 81920;  // longest stretch of a row that a CTA takes while clusters allow it
constexpr int kMaxTop = 1024;
constexpr int kCounters = 148;       // partial counts of the rows with a teacher
// rows and entries up to which every CTA counts the rows with a teacher itself: a launch saved (2 us), where two warps
// take 0.23 us a row
constexpr long kCountRows = 16, kCountEntries = 4096;
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct DistillArgs {
    const void *logits, *teacher, *indices;
    long rows, row_stride;
    int vocab, top, teacher_dtype, wide_indices;
    float temperature;
    int mean;
    int *counts;             // kCounters partial counts (a mean's, null where every CTA counts itself)
    float *row_loss;         // forward
    float2 *row_stats;       // (reference, sum of exp2((s - reference) log2e / tau)); forward writes, backward reads
    void *grad;              // null: none
    const float *upstream;   // backward: null is 1
    int upstream_per_row;
    int words;               // of the bits of a stretch; 0: the stretch is too long for them
};

__device__ __forceinline__ float exp2_unit(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o /= 2) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// The maximum to subtract: where nothing but -inf was seen, any finite one.
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.f : m; }

// Running (reference, sum) pairs joined: by the larger reference.
__device__ __forceinline__ float2 join(float2 a, float2 b, float scale) {
    const float m = fmaxf(a.x, b.x), f = finite_max(m);
    return make_float2(m, a.y * exp2_unit((a.x - f) * scale) + b.y * exp2_unit((b.x - f) * scale));
}

__device__ __forceinline__ long entry_of(const DistillArgs &a, long i) {
    return a.wide_indices ? static_cast<const long *>(a.indices)[i] : static_cast<const int *>(a.indices)[i];
}
__device__ __forceinline__ bool is_entry(const DistillArgs &a, long i) {
    return entry_of(a, i) >= 0 && load_as_float(a.teacher, a.teacher_dtype, i) != -INFINITY;
}
// Rows of first, first + step, ... with a teacher, by one warp.
__device__ __forceinline__ int count_rows(const DistillArgs &a, long first, long step) {
    int n = 0;
    for (long r = first; r < a.rows; r += step) {
        bool any = false;
        for (int k = threadIdx.x % 32; k < a.top && !any; k += 32) any = is_entry(a, r * a.top + k);
        n += __any_sync(0xffffffffu, any) ? 1 : 0;
    }
    return n;
}
__global__ void __launch_bounds__(1024) distill_count(const DistillArgs a) {
    __shared__ int part[32];
    const int warp = threadIdx.x / 32;
    const int n = count_rows(a, blockIdx.x * 32 + warp, static_cast<long>(kCounters) * 32);
    if (threadIdx.x % 32 == 0) part[warp] = n;
    __syncthreads();
    if (warp != 0) return;
    const int total = __reduce_add_sync(0xffffffffu, part[threadIdx.x]);
    if (threadIdx.x == 0) a.counts[blockIdx.x] = total;
}
// All rows with a teacher, in every thread of the CTA; `part` is its scratch.
template <int WARPS> __device__ __forceinline__ int all_rows(const DistillArgs &a, int *part) {
    int n = 0;
    if (a.counts != nullptr) {
        for (int i = threadIdx.x % 32; i < kCounters; i += 32) n += a.counts[i];
        return __reduce_add_sync(0xffffffffu, n);
    }
    n = count_rows(a, threadIdx.x / 32, WARPS);
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) n += part[w];
    return n;
}

// A row's stretch [lo, hi): `head` single elements, `vecs` 16-byte vectors from
// the first aligned address on, then single elements again.
template <typename T> struct Stretch {
    static constexpr int kVec = 16 / sizeof(T);
    int lo, hi, body, vecs;
    __device__ __forceinline__ Stretch(const T *row, int vocab, int rank, int ranks) {
        // equal shares in whole vectors, counted from the row's first aligned element
        const int head = min(vocab, static_cast<int>((16 - reinterpret_cast<uintptr_t>(row) % 16) % 16 / sizeof(T)));
        const int all = (vocab - head) / kVec, share = (all + ranks - 1) / ranks;
        const int first = min(all, rank * share), last = min(all, first + share);
        body = head + first * kVec;
        vecs = last - first;
        lo = rank == 0 ? 0 : body;
        hi = rank == ranks - 1 ? vocab : head + last * kVec;
    }
    __device__ __forceinline__ int tail() const { return body + vecs * kVec; }
};

// A thread's running sum of exp2((v - reference) log2e / tau).  The reference
// follows the maximum lazily, once a value is 2^kSlack times its weight above
// it, so that few vectors rescale the sum: below 2^(17 + kSlack) for any row,
// far from float32's range.
constexpr float kSlack = 8.f;
struct Running {
    float reference = -INFINITY, shift = 0.f, limit = -INFINITY;  // shift: the reference, or 0 before the first value
    float2 sum = make_float2(0.f, 0.f);

    template <int VEC> __device__ __forceinline__ void add(float top, const float (&v)[VEC], float scale, float slack) {
        if (top > limit) {
            const float by = reference == -INFINITY ? 0.f : exp2_unit((reference - top) * scale);
            sum = make_float2(sum.x * by, sum.y * by);
            reference = shift = top;
            limit = top + slack;
        }
#pragma unroll
        for (int e = 0; e < VEC; e += 2) {
            const float2 x = __fmul2_rn(__fadd2_rn(make_float2(v[e], v[e + 1]), make_float2(-shift, -shift)),
                                        make_float2(scale, scale));
            sum = __fadd2_rn(sum, make_float2(exp2_unit(x.x), exp2_unit(x.y)));
        }
    }
};

// Row r by a CTA or, rank by rank, by its cluster.  BACKWARD: the reference and sum are the forward's.
// 8,192 x 32,000 bf16, K 64, loss and gradient: 204 us for 1.05 GB (5.1 TB/s,
// 0.80 of a copy's rate; the exp2 unit at 59 %); 2,048 x 32,000 f32, K 32: 112
// us (4.7 TB/s); 4 x 50,001 bf16 in clusters of 8: 10 us.  Rows of a few hundred
// logits are bound by their chain of round trips (65,536 x 256: 159 us, 2.4 ns a row).
template <typename T, bool BACKWARD, int THREADS>
__device__ __forceinline__ void distill_row(const DistillArgs &a, const long r) {
    constexpr int kVec = 16 / sizeof(T), kWarps = THREADS / 32;
    __shared__ float p_s[kMaxTop];
    __shared__ int i_s[kMaxTop];
    __shared__ float2 stat_s[kWarps], teacher_s[kWarps];
    __shared__ float loss_s[kWarps];
    __shared__ int bad_s[kWarps], count_s[kWarps], again_s;
    __shared__ float2 mine_s;           // this CTA's reference and sum, read by its cluster
    extern __shared__ unsigned named[]; // a bit for every logit of the stretch: named by the teacher
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = static_cast<int>(cluster.block_rank()), ranks = static_cast<int>(cluster.num_blocks());
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const T *row = static_cast<const T *>(a.logits) + r * a.row_stride;
    T *grad = a.grad == nullptr ? nullptr : static_cast<T *>(a.grad) + r * a.vocab;
    const Stretch<T> at(row, a.vocab, rank, ranks);
    const float scale = kLog2e / a.temperature;  // exponents in powers of two
    const bool counters = a.counts != nullptr;
    int counted = 0;
    if (counters)
        for (int i = lane; i < kCounters; i += 32) counted += a.counts[i];
    for (int i = tid; i < a.words; i += THREADS) named[i] = 0;
    if (tid == 0) again_s = 0;

    // the teacher's entries; -1 marks an empty one, -2 one past the vocabulary
    float top = -INFINITY, total = 0.f;
    bool bad = false;
    for (int k = tid; k < a.top; k += THREADS) {
        const long e = entry_of(a, r * a.top + k);
        const float t = e < 0 ? -INFINITY : load_as_float(a.teacher, a.teacher_dtype, r * a.top + k);
        const int j = t == -INFINITY ? -1 : e >= a.vocab ? -2 : static_cast<int>(e);
        p_s[k] = t;
        i_s[k] = j;
        bad |= j == -2;
        top = fmaxf(top, j == -1 ? -INFINITY : t);
    }
    const bool any = __any_sync(0xffffffffu, top != -INFINITY);
    bool nan = false;  // a NaN gives way in fmaxf, but is an entry
    for (int k = tid; k < a.top; k += THREADS) nan |= p_s[k] != p_s[k];
    top = warp_max(top);
    for (int k = tid; k < a.top; k += THREADS) total += exp2f((p_s[k] - finite_max(top)) * scale);
    total = warp_sum(total);
    bad = __any_sync(0xffffffffu, bad);
    if (lane == 0) {
        teacher_s[warp] = make_float2(top, total);
        bad_s[warp] = bad;
    }
    if (!__syncthreads_or(any || nan)) {  // no teacher
        if (!BACKWARD && tid == 0 && rank == 0) a.row_loss[r] = 0.f;
        if (grad != nullptr)
            for (int j = at.lo + tid; j < at.hi; j += THREADS) grad[j] = from_float<T>(0.f);
        return;  // every CTA of the cluster does
    }
    {
        const float2 w = teacher_s[lane % kWarps];
        top = warp_max(w.x);
        total = warp_sum(lane < kWarps ? w.y * exp2f((w.x - finite_max(top)) * scale) : 0.f);
        bad = __any_sync(0xffffffffu, bad_s[lane % kWarps] != 0);
    }
    for (int k = tid; k < a.top; k += THREADS) {
        const int j = i_s[k] - at.lo;
        if (a.words == 0 || i_s[k] < at.lo || i_s[k] >= at.hi) continue;
        const unsigned bit = 1u << (j % 32);
        if ((atomicOr(&named[j / 32], bit) & bit) != 0) again_s = 1;  // named twice
    }

    float2 stat;
    if (BACKWARD) {
        stat = a.row_stats[r];
    } else {
        Running run;
        const float slack = kSlack / scale;
        auto one = [&](int j) {
            const float v[2] = {to_float(row[j]), -INFINITY};
            run.add<2>(v[0], v, scale, slack);
        };
        for (int j = at.lo + tid; j < at.body; j += THREADS) one(j);
        for (int j = at.tail() + tid; j < at.hi; j += THREADS) one(j);
        const T *body = row + at.body;
        int i = tid;
        for (; i + 3 * THREADS < at.vecs; i += 4 * THREADS) {
            RawVec<T, kVec> p[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) p[u].load(body + (i + u * THREADS) * kVec);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                float v[kVec];
                p[u].values(v);
                run.add<kVec>(p[u].top(), v, scale, slack);
            }
        }
        for (; i < at.vecs; i += THREADS) {
            RawVec<T, kVec> p;
            float v[kVec];
            p.load(body + i * kVec);
            p.values(v);
            run.add<kVec>(p.top(), v, scale, slack);
        }
        stat = make_float2(run.reference, run.sum.x + run.sum.y);
        float2 all = make_float2(warp_max(stat.x), 0.f);
        all.y = warp_sum(stat.y * exp2_unit((stat.x - finite_max(all.x)) * scale));
        if (lane == 0) stat_s[warp] = all;
        __syncthreads();
        stat = stat_s[lane % kWarps];
        all.x = warp_max(stat.x);
        all.y = lane < kWarps ? stat.y * exp2_unit((stat.x - finite_max(all.x)) * scale) : 0.f;
        stat = make_float2(all.x, warp_sum(all.y));
        if (ranks > 1) {
            if (tid == 0) mine_s = stat;
            cluster.sync();
            stat = *cluster.map_shared_rank(&mine_s, 0);
            for (int w = 1; w < ranks; ++w) stat = join(stat, *cluster.map_shared_rank(&mine_s, w), scale);
            cluster.sync();  // no CTA leaves while another still reads its pair
        }
        if (a.row_stats != nullptr && tid == 0 && rank == 0) a.row_stats[r] = stat;
    }
    // a row of -inf alone has no distribution: m is -inf and what follows is NaN; so has a teacher's with a NaN or +inf
    const float m = stat.x, sum = stat.y, poison = bad || total != total ? NAN : 0.f, inverse = 1.f / sum + poison;

    if (!BACKWARD && rank == 0) {
        const float log_total = log2f(total), log_sum = log2f(sum);
        float loss = 0.f;
        for (int k = tid; k < a.top; k += THREADS) {
            if (i_s[k] < 0) continue;
            const float lp = (p_s[k] - top) * scale - log_total, p = exp2f(lp);
            const float lq = (to_float(row[i_s[k]]) - m) * scale - log_sum;
            if (p != 0.f) loss = fmaf(p, lp - lq, loss);
        }
        loss = warp_sum(loss);
        if (lane == 0) loss_s[warp] = loss;
    }
    float weight = a.temperature;
    if (grad != nullptr) {
        if (a.upstream != nullptr) weight *= a.upstream[a.upstream_per_row ? r : 0];
        if (a.mean) {
            const int n = counters ? __reduce_add_sync(0xffffffffu, counted) : all_rows<kWarps>(a, count_s);
            weight /= static_cast<float>(max(1, n));
        }
        const float factor = weight * inverse;
        auto one = [&](int j) { grad[j] = from_float<T>(exp2_unit((to_float(row[j]) - m) * scale) * factor); };
        auto gradients = [&](const RawVec<T, kVec> &p, float (&v)[kVec]) {
            p.values(v);
#pragma unroll
            for (int e = 0; e < kVec; e += 2) {
                const float2 x = __fmul2_rn(__fadd2_rn(make_float2(v[e], v[e + 1]), make_float2(-m, -m)),
                                            make_float2(scale, scale));
                const float2 g = __fmul2_rn(make_float2(exp2_unit(x.x), exp2_unit(x.y)), make_float2(factor, factor));
                v[e] = g.x;
                v[e + 1] = g.y;
            }
        };
        if ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(grad)) % 16 == 0) {
            for (int j = at.lo + tid; j < at.body; j += THREADS) one(j);
            for (int j = at.tail() + tid; j < at.hi; j += THREADS) one(j);
            const T *body = row + at.body;
            T *out = grad + at.body;
            int i = tid;
            for (; i + 3 * THREADS < at.vecs; i += 4 * THREADS) {
                RawVec<T, kVec> p[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) p[u].load(body + (i + u * THREADS) * kVec);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    float v[kVec];
                    gradients(p[u], v);
                    store_packed<T, kVec>(out + (i + u * THREADS) * kVec, v);
                }
            }
            for (; i < at.vecs; i += THREADS) {
                RawVec<T, kVec> p;
                float v[kVec];
                p.load(body + i * kVec);
                gradients(p, v);
                store_packed<T, kVec>(out + i * kVec, v);
            }
        } else {  // rows of logits and gradient fall differently on 16 bytes
            for (int j = at.lo + tid; j < at.hi; j += THREADS) one(j);
        }
    }
    __syncthreads();
    if (!BACKWARD && tid == 0 && rank == 0) {
        float loss = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) loss += loss_s[w];
        a.row_loss[r] = loss * kLn2 * a.temperature * a.temperature + poison + (sum != sum ? NAN : 0.f);
    }
    if (grad == nullptr) return;
    // the entries the teacher names: q - p, the p of an entry named twice added up by the first
    const float per = 1.f / total;
    const bool again = a.words == 0 || again_s != 0;
    for (int k = tid; k < a.top; k += THREADS) {
        const int j = i_s[k];
        if (j < at.lo || j >= at.hi) continue;
        float p = exp2f((p_s[k] - top) * scale) * per;
        if (again) {
            bool first = true;
            p = 0.f;
            for (int o = 0; o < a.top; ++o) {
                if (i_s[o] != j) continue;
                first &= o >= k;
                p += exp2f((p_s[o] - top) * scale) * per;
            }
            if (!first) continue;
        }
        grad[j] = from_float<T>(weight * (exp2_unit((to_float(row[j]) - m) * scale) * inverse - p));
    }
}
template <typename T, bool BACKWARD, int THREADS>
__global__ void __launch_bounds__(THREADS, kThreadsAnSM / THREADS) distill_rows(const DistillArgs a) {
    distill_row<T, BACKWARD, THREADS>(a, blockIdx.x / cooperative_groups::this_cluster().num_blocks());
}
// The gradient that the forward wrote, computed again for an upstream factor,
// which has to come before the rounding: a loss scale saves gradients that 16
// bits cannot hold.  Nothing at all where the factor is 1 (the loss was the end
// of the graph); one wave of CTAs, so that this is then over in 1 to 3 us.
// 8,192 x 32,000 bf16: 211 us (one read and one write of the logits' bytes, 5.0
// TB/s); 2,048 x 32,000 f32: 107; 65,536 x 256 bf16, by the rows' chains: 128.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, kRescaleThreadsAnSM / THREADS) distill_rescale(const DistillArgs a) {
    if (*a.upstream == 1.f) return;
    const unsigned ranks = cooperative_groups::this_cluster().num_blocks();
    for (unsigned r = blockIdx.x / ranks; r < a.rows; r += gridDim.x / ranks) {
        distill_row<T, true, THREADS>(a, r);
        __syncthreads();  // the row's entries have been read
    }
}

// The rows' losses added in a fixed order, and divided by the rows counted.
constexpr int kTotalThreads = 1024;
__global__ void __launch_bounds__(kTotalThreads) distill_total(const DistillArgs a, float *loss) {
    __shared__ float part[kTotalThreads / 32];
    __shared__ int count_s[kTotalThreads / 32];
    float v = 0.f;
#pragma unroll 8
    for (long r = threadIdx.x; r < a.rows; r += kTotalThreads) v += a.row_loss[r];
    v = warp_sum(v);
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = v;
    const int n = a.mean ? all_rows<kTotalThreads / 32>(a, count_s) : 1;
    __syncthreads();
    if (threadIdx.x >= 32) return;
    v = warp_sum(part[threadIdx.x]);
    if (threadIdx.x == 0) *loss = v / static_cast<float>(max(1, n));
}

enum RowsKind { kForward, kBackward, kRescale };

template <typename T, int THREADS>
cudaError_t launch_kernel(cudaLaunchConfig_t &config, unsigned ranks, const DistillArgs &a, RowsKind kind) {
    config.blockDim = dim3(THREADS);
    if (kind == kForward) return cudaLaunchKernelEx(&config, distill_rows<T, false, THREADS>, a);
    if (kind == kBackward) return cudaLaunchKernelEx(&config, distill_rows<T, true, THREADS>, a);
    const unsigned wave = 148u * (kRescaleThreadsAnSM / THREADS) / ranks * ranks;
    if (config.gridDim.x > wave) config.gridDim.x = wave;
    return cudaLaunchKernelEx(&config, distill_rescale<T, THREADS>, a);
}
template <typename T> int launch_rows(DistillArgs a, RowsKind kind, cudaStream_t st) {
    // Rows alone fill the SMs from 148 on; fewer are split down to 4,096 logits a CTA.  Long ones are split so
    // that the second pass finds its logits in L2: 6 CTAs an SM of 80 KB are 71 MB.  (When chosen: 8,192 x 32,000
    // bf16 unsplit 215 us, halved 297.  2,048 x 32,000 f32: halved 114, unsplit 133.  2,048 x 128,000 bf16: quarters,
    // 248.)
    int ranks = 1;
    while (ranks < kMaxCluster &&
           ((a.rows * ranks * 2 <= 296 && a.vocab / (ranks * 2) >= 4096) ||
            static_cast<long>(a.vocab) / ranks * static_cast<long>(sizeof(T)) > kStretchBytes))
        ranks *= 2;
    const long longest = static_cast<long>(a.vocab) / ranks + 64;  // shares are whole vectors, the ends ragged
    a.words = longest * static_cast<long>(sizeof(T)) <= 2 * kStretchBytes ? static_cast<int>((longest + 31) / 32) : 0;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(a.rows * ranks));
    config.dynamicSmemBytes = static_cast<size_t>(a.words) * sizeof(unsigned);
    config.stream = st;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = static_cast<unsigned>(ranks);
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = ranks > 1 ? 1 : 0;  // a cluster of one costs: 65,536 x 256 bf16 289 us with it, 159 without
    // Short rows are bound by a row's chain of round trips, so more of them at a time, by fewer threads each.  64, 128
    // and 256 threads: 65,536 x 256 bf16 159, 244, 452 us; 32,768 x 4,096 bf16 159, 196, 318; 32,768 x 4,096 f32 249,
    // 239, 321; 8,192 x 16,000 bf16 177, 118, 142; 8,192 x 32,000 bf16 -, 258 (12 rows an SM are more than L2), 204.
    const long bytes = static_cast<long>(a.vocab) * static_cast<long>(sizeof(T));
    const unsigned split = static_cast<unsigned>(ranks);
    const cudaError_t e = ranks > 1 || bytes > 32768 ? launch_kernel<T, 256>(config, split, a, kind)
                          : bytes > 8192             ? launch_kernel<T, 128>(config, split, a, kind)
                                                     : launch_kernel<T, 64>(config, split, a, kind);
    if (e != cudaSuccess) return fail(BSSM_ERR_CUDA, "distillation: %s", cudaGetErrorString(e));
    return check_launch("distillation");
}
int launch_rows(int dtype, const DistillArgs &a, RowsKind kind, cudaStream_t st) {
    switch (dtype) {
        case BSSM_F32: return launch_rows<float>(a, kind, st);
        case BSSM_BF16: return launch_rows<__nv_bfloat16>(a, kind, st);
        default: return launch_rows<__half>(a, kind, st);
    }
}

int *counts_of(int mean, long rows, int top, int *counts) {
    return mean && (rows > kCountRows || rows * top > kCountEntries) ? counts : nullptr;
}

int check_distill(const char *what, int dtype, long rows, int vocab, long row_stride, int top, int teacher_dtype,
                  int index_bytes, float temperature) {
    if (!io_dtype_known(dtype) || !io_dtype_known(teacher_dtype) || (index_bytes != 4 && index_bytes != 8))
        return fail(BSSM_ERR_UNSUPPORTED, "%s: unknown dtype", what);
    if (top < 1 || top > kMaxTop)
        return fail(BSSM_ERR_UNSUPPORTED, "%s: %d teacher logits a row (1 to %d are built)", what, top, kMaxTop);
    if (rows < 0 || rows > 0x7fffffffL / 8 || vocab < 1 || (rows > 1 && row_stride < vocab) || !(temperature > 0.f) ||
        !(temperature < INFINITY))
        return fail(BSSM_ERR_INVALID, "%s: bad sizes or temperature", what);
    return BSSM_OK;
}

}  // namespace
}  // namespace bssm

extern "C" int bssm_distillation_counters(void) { return bssm::kCounters; }

extern "C" int bssm_distillation(const void *logits, int dtype, long rows, int vocab, long row_stride,
                                 const void *teacher, int teacher_dtype, const void *indices, int index_bytes, int top,
                                 float temperature, int mean, float *row_loss, float *row_stats, float *loss,
                                 int *counts, void *grad, void *stream) {
    using namespace bssm;
    if (int rc = check_distill("distillation", dtype, rows, vocab, row_stride, top, teacher_dtype, index_bytes,
                               temperature))
        return rc;
    if ((rows > 0 && (logits == nullptr || teacher == nullptr || indices == nullptr || row_loss == nullptr)) ||
        (mean && counts == nullptr))
        return fail(BSSM_ERR_INVALID, "distillation: null pointer");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    DistillArgs a{};
    a.logits = logits; a.teacher = teacher; a.indices = indices; a.rows = rows; a.row_stride = row_stride;
    a.vocab = vocab; a.top = top; a.teacher_dtype = teacher_dtype; a.wide_indices = index_bytes == 8;
    a.temperature = temperature; a.mean = mean; a.counts = counts_of(mean, rows, top, counts); a.row_loss = row_loss;
    a.row_stats = reinterpret_cast<float2 *>(row_stats); a.grad = grad;
    if (a.counts != nullptr) {
        distill_count<<<kCounters, 1024, 0, st>>>(a);
        if (int rc = check_launch("distillation")) return rc;
    }
    if (rows > 0)
        if (int rc = launch_rows(dtype, a, kForward, st)) return rc;
    if (loss == nullptr) return BSSM_OK;
    distill_total<<<1, kTotalThreads, 0, st>>>(a, loss);
    return check_launch("distillation");
}

namespace bssm {
namespace {
int launch_backward(const char *what, const void *logits, int dtype, long rows, int vocab, long row_stride,
                    const void *teacher, int teacher_dtype, const void *indices, int index_bytes, int top,
                    float temperature, int mean, const float *row_stats, const int *counts, const float *upstream,
                    int upstream_per_row, RowsKind kind, void *grad, void *stream) {
    if (int rc = check_distill(what, dtype, rows, vocab, row_stride, top, teacher_dtype, index_bytes, temperature))
        return rc;
    if ((rows > 0 && (logits == nullptr || teacher == nullptr || indices == nullptr || row_stats == nullptr ||
                      grad == nullptr)) ||
        (mean && counts == nullptr) || (kind == kRescale && upstream == nullptr))
        return fail(BSSM_ERR_INVALID, "%s: null pointer", what);
    if (rows == 0) return BSSM_OK;
    DistillArgs a{};
    a.logits = logits; a.teacher = teacher; a.indices = indices; a.rows = rows; a.row_stride = row_stride;
    a.vocab = vocab; a.top = top; a.teacher_dtype = teacher_dtype; a.wide_indices = index_bytes == 8;
    a.temperature = temperature; a.mean = mean;
    a.counts = counts_of(mean, rows, top, const_cast<int *>(counts));
    a.row_stats = reinterpret_cast<float2 *>(const_cast<float *>(row_stats));
    a.grad = grad; a.upstream = upstream; a.upstream_per_row = upstream_per_row;
    return launch_rows(dtype, a, kind, static_cast<cudaStream_t>(stream));
}
}  // namespace
}  // namespace bssm

extern "C" int bssm_distillation_backward(const void *logits, int dtype, long rows, int vocab, long row_stride,
                                          const void *teacher, int teacher_dtype, const void *indices, int index_bytes,
                                          int top, float temperature, int mean, const float *row_stats,
                                          const int *counts, const float *upstream, int upstream_per_row, void *grad,
                                          void *stream) {
    return bssm::launch_backward("distillation_backward", logits, dtype, rows, vocab, row_stride, teacher,
                                 teacher_dtype, indices, index_bytes, top, temperature, mean, row_stats, counts,
                                 upstream, upstream_per_row, bssm::kBackward, grad, stream);
}

extern "C" int bssm_distillation_rescale(const void *logits, int dtype, long rows, int vocab, long row_stride,
                                         const void *teacher, int teacher_dtype, const void *indices, int index_bytes,
                                         int top, float temperature, int mean, const float *row_stats,
                                         const int *counts, const float *upstream, void *grad, void *stream) {
    return bssm::launch_backward("distillation_rescale", logits, dtype, rows, vocab, row_stride, teacher,
                                 teacher_dtype, indices, index_bytes, top, temperature, mean, row_stats, counts,
                                 upstream, 0, bssm::kRescale, grad, stream);
}
