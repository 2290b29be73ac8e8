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
// zero, and a mean does not count it.  An entry at or past V makes the row's
// loss and gradient NaN (nothing is read or written out of range).
//
// The traffic of the logits bounds it: read once, and the gradient written
// once.  One CTA takes one row: a pass for the running maximum and sum, and,
// where the gradient is wanted, a second one over a row that is then in L1 or
// L2 (148 rows of 128 KB are 19 MB of its 126).  The K entries are corrected
// afterwards, from the logits again rather than from the rounded gradient.
#include <cuda_runtime.h>

#include <cstdint>

#include "bayes_ssm_b200.h"
#include "bssm_internal.h"
#include "bssm_io.cuh"

namespace bssm {
namespace {

constexpr int kThreads = 512;
constexpr int kMaxTop = 1024;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct DistillArgs {
    const void *logits, *teacher, *indices;
    long rows, row_stride;
    int vocab, top, teacher_dtype, wide_indices;
    float temperature;
    int mean;
    const int *count;        // rows with a teacher (mean)
    float *row_loss;         // forward
    float2 *row_stats;       // (maximum, sum of exp2((s - maximum) log2e / tau)); forward writes, backward reads
    void *grad;              // null: none
    const float *upstream;   // backward: null is 1
    int upstream_per_row;
};

__device__ __forceinline__ long entry_of(const DistillArgs &a, long i) {
    return a.wide_indices ? static_cast<const long *>(a.indices)[i] : static_cast<const int *>(a.indices)[i];
}

// Reductions over the CTA; every thread gets the result.
__device__ __forceinline__ float block_max(float v, float *scratch) {
#pragma unroll
    for (int o = 16; o > 0; o /= 2) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if (threadIdx.x % 32 == 0) scratch[threadIdx.x / 32] = v;
    __syncthreads();
    v = scratch[threadIdx.x % (kThreads / 32)];
#pragma unroll
    for (int o = kThreads / 64; o > 0; o /= 2) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float block_sum(float v, float *scratch) {
#pragma unroll
    for (int o = 16; o > 0; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (threadIdx.x % 32 == 0) scratch[threadIdx.x / 32] = v;
    __syncthreads();
    v = scratch[threadIdx.x % (kThreads / 32)];
#pragma unroll
    for (int o = kThreads / 64; o > 0; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Rows with a teacher, added to *count: a warp per row.
__device__ __forceinline__ bool has_entry(const DistillArgs &a, long i) {
    return entry_of(a, i) >= 0 && load_as_float(a.teacher, a.teacher_dtype, i) != -INFINITY;
}
__global__ void __launch_bounds__(256) distill_count(const DistillArgs a, int *count) {
    const long warps = static_cast<long>(gridDim.x) * 8;
    int mine = 0;
    for (long r = static_cast<long>(blockIdx.x) * 8 + threadIdx.x / 32; r < a.rows; r += warps) {
        bool any = false;
        for (int k = threadIdx.x % 32; k < a.top && !any; k += 32) any = has_entry(a, r * a.top + k);
        mine += __any_sync(0xffffffffu, any) ? 1 : 0;
    }
    if (threadIdx.x % 32 == 0 && mine != 0) atomicAdd(count, mine);  // whole numbers: the order does not matter
}

// f(j, value) over a row's logits.  The row is walked in 16-byte vectors from
// the first aligned element on, the ends element by element.
template <typename T, typename F> __device__ __forceinline__ void for_row(const T *row, int n, F f) {
    constexpr int VEC = 16 / sizeof(T);
    const int head = min(n, static_cast<int>((16 - reinterpret_cast<uintptr_t>(row) % 16) % 16 / sizeof(T)));
    const int vecs = (n - head) / VEC;
    for (int j = threadIdx.x; j < head; j += kThreads) f(j, to_float(row[j]));
    for (int i = threadIdx.x; i < vecs; i += kThreads) {
        float v[VEC];
        widen(load_packed<T, VEC>(row + head + i * VEC), v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) f(head + i * VEC + e, v[e]);
    }
    for (int j = head + vecs * VEC + threadIdx.x; j < n; j += kThreads) f(j, to_float(row[j]));
}

// BACKWARD: the maximum and sum are the forward's.
template <typename T, bool BACKWARD> __global__ void __launch_bounds__(kThreads) distill_rows(const DistillArgs a) {
    __shared__ float scratch[kThreads / 32];
    __shared__ float p_s[kMaxTop];
    __shared__ int i_s[kMaxTop];
    __shared__ int bad_s;
    const long r = blockIdx.x;
    const T *row = static_cast<const T *>(a.logits) + r * a.row_stride;
    T *grad = a.grad == nullptr ? nullptr : static_cast<T *>(a.grad) + r * a.vocab;
    const float scale = kLog2e / a.temperature;  // exponents in powers of two

    // the teacher's softmax
    if (threadIdx.x == 0) bad_s = 0;
    __syncthreads();
    float top = -INFINITY;
    bool any = false;
    for (int k = threadIdx.x; k < a.top; k += kThreads) {
        const long e = entry_of(a, r * a.top + k);
        float t = e < 0 ? -INFINITY : load_as_float(a.teacher, a.teacher_dtype, r * a.top + k);
        if (e >= 0 && t != -INFINITY) any = true;
        if (e >= a.vocab) bad_s = 1;
        p_s[k] = t;
        i_s[k] = t == -INFINITY ? -1 : static_cast<int>(e >= a.vocab ? -1 : e);
        top = fmaxf(top, t);
    }
    any = __syncthreads_or(any);
    if (!any) {  // no teacher
        if (!BACKWARD && threadIdx.x == 0) a.row_loss[r] = 0.f;
        if (grad != nullptr)
            for (int j = threadIdx.x; j < a.vocab; j += kThreads) grad[j] = from_float<T>(0.f);
        return;
    }
    top = block_max(top, scratch);
    float part = 0.f;
    for (int k = threadIdx.x; k < a.top; k += kThreads) {
        const float e = p_s[k] == -INFINITY ? 0.f : exp2f((p_s[k] - top) * scale);
        part += e;
    }
    const float total = block_sum(part, scratch);

    float m, sum;
    if (BACKWARD) {
        m = a.row_stats[r].x;
        sum = a.row_stats[r].y;
    } else {
        m = -INFINITY;
        float s = 0.f;
        bool nan = false;
        for_row(row, a.vocab, [&](int, float v) {
            if (v > m) {
                s = s * exp2f((m - v) * scale);
                m = v;
            }
            nan |= v != v;
            s += m == -INFINITY ? 0.f : exp2f((v - m) * scale);
        });
        const float all = block_max(m, scratch);
        s = m == -INFINITY ? 0.f : s * exp2f((m - all) * scale);
        if (nan || all == INFINITY) s = NAN;
        sum = block_sum(s, scratch);
        m = all;
        if (a.row_stats != nullptr && threadIdx.x == 0) a.row_stats[r] = make_float2(m, sum);
    }
    const float bad = bad_s ? NAN : 0.f;
    const float inverse = 1.f / sum + bad;

    if (!BACKWARD) {
        const float log_total = log2f(total), log_sum = log2f(sum);
        float loss = 0.f;
        for (int k = threadIdx.x; k < a.top; k += kThreads) {
            if (i_s[k] < 0) continue;
            const float lp = (p_s[k] - top) * scale - log_total, p = exp2f(lp);
            const float lq = (to_float(row[i_s[k]]) - m) * scale - log_sum;
            if (p != 0.f) loss = fmaf(p, lp - lq, loss);
        }
        loss = block_sum(loss, scratch);
        if (threadIdx.x == 0) a.row_loss[r] = loss * kLn2 * a.temperature * a.temperature + bad + (sum != sum ? NAN : 0.f);
    }
    if (grad == nullptr) return;
    float weight = a.temperature;
    if (a.upstream != nullptr) weight *= a.upstream[a.upstream_per_row ? r : 0];
    if (a.mean) weight /= static_cast<float>(max(1, *a.count));
    if ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(grad)) % 16 == 0) {
        constexpr int VEC = 16 / sizeof(T);
        const int head = min(a.vocab, static_cast<int>((16 - reinterpret_cast<uintptr_t>(row) % 16) % 16 / sizeof(T)));
        const int vecs = (a.vocab - head) / VEC;
        auto one = [&](int j) { grad[j] = from_float<T>(weight * (exp2f((to_float(row[j]) - m) * scale) * inverse)); };
        for (int j = threadIdx.x; j < head; j += kThreads) one(j);
        for (int i = threadIdx.x; i < vecs; i += kThreads) {
            float v[VEC];
            widen(load_packed<T, VEC>(row + head + i * VEC), v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = weight * (exp2f((v[e] - m) * scale) * inverse);
            store_packed<T, VEC>(grad + head + i * VEC, v);
        }
        for (int j = head + vecs * VEC + threadIdx.x; j < a.vocab; j += kThreads) one(j);
    } else {
        for_row(row, a.vocab, [&](int j, float v) {
            grad[j] = from_float<T>(weight * (exp2f((v - m) * scale) * inverse));
        });
    }
    __syncthreads();
    // the entries the teacher names: q - p, the p of an entry named twice added up
    for (int k = threadIdx.x; k < a.top; k += kThreads) {
        const int j = i_s[k];
        if (j < 0) continue;
        float p = 0.f;
        bool first = true;
        for (int o = 0; o < a.top; ++o) {
            if (i_s[o] != j) continue;
            if (o < k) first = false;
            p += exp2f((p_s[o] - top) * scale) / total;
        }
        if (first) grad[j] = from_float<T>(weight * (exp2f((to_float(row[j]) - m) * scale) * inverse - p));
    }
}

// The rows' losses added in a fixed order, and divided by the rows counted.
__global__ void __launch_bounds__(kThreads) distill_total(const float *row_loss, long rows, int mean, const int *count,
                                                          float *loss) {
    __shared__ float scratch[kThreads / 32];
    float v = 0.f;
    for (long r = threadIdx.x; r < rows; r += kThreads) v += row_loss[r];
    v = block_sum(v, scratch);
    if (threadIdx.x == 0) *loss = mean ? v / static_cast<float>(max(1, *count)) : v;
}

// grad *= *factor, nothing at all where it is 1 (the loss was the end of the graph).
template <typename T> __global__ void __launch_bounds__(256) distill_scale(T *grad, long n, const float *factor) {
    const float f = *factor;
    if (f == 1.f) return;
    for (long i = static_cast<long>(blockIdx.x) * 256 + threadIdx.x; i < n; i += 256L * gridDim.x)
        grad[i] = from_float<T>(to_float(grad[i]) * f);
}

template <typename T> int launch_rows(const DistillArgs &a, bool backward, cudaStream_t st) {
    const unsigned grid = static_cast<unsigned>(a.rows);
    if (backward) distill_rows<T, true><<<grid, kThreads, 0, st>>>(a);
    else distill_rows<T, false><<<grid, kThreads, 0, st>>>(a);
    return check_launch("distillation");
}
int launch_rows(int dtype, const DistillArgs &a, bool backward, cudaStream_t st) {
    switch (dtype) {
        case BSSM_F32: return launch_rows<float>(a, backward, st);
        case BSSM_BF16: return launch_rows<__nv_bfloat16>(a, backward, st);
        default: return launch_rows<__half>(a, backward, st);
    }
}

int check_distill(const char *what, int dtype, long rows, int vocab, long row_stride, int top, int teacher_dtype,
                  int index_bytes, float temperature) {
    if (!io_dtype_known(dtype) || !io_dtype_known(teacher_dtype) || (index_bytes != 4 && index_bytes != 8))
        return fail(BSSM_ERR_UNSUPPORTED, "%s: unknown dtype", what);
    if (top < 1 || top > kMaxTop)
        return fail(BSSM_ERR_UNSUPPORTED, "%s: %d teacher logits a row (1 to %d are built)", what, top, kMaxTop);
    if (rows < 0 || rows > 0x7fffffffL || vocab < 1 || (rows > 1 && row_stride < vocab) || !(temperature > 0.f) ||
        !(temperature < INFINITY))
        return fail(BSSM_ERR_INVALID, "%s: bad sizes or temperature", what);
    return BSSM_OK;
}

int count_rows(const DistillArgs &a, int *count, cudaStream_t st) {
    if (cudaError_t e = cudaMemsetAsync(count, 0, sizeof(int), st))
        return fail(BSSM_ERR_CUDA, "distillation: %s", cudaGetErrorString(e));
    const long blocks = (a.rows + 7) / 8;
    if (blocks > 0) distill_count<<<static_cast<unsigned>(blocks < 592 ? blocks : 592), 256, 0, st>>>(a, count);
    return check_launch("distillation");
}

}  // namespace
}  // namespace bssm

extern "C" int bssm_distillation(const void *logits, int dtype, long rows, int vocab, long row_stride,
                                 const void *teacher, int teacher_dtype, const void *indices, int index_bytes, int top,
                                 float temperature, int mean, float *row_loss, float *row_stats, float *loss,
                                 int *count, void *grad, void *stream) {
    using namespace bssm;
    if (int rc = check_distill("distillation", dtype, rows, vocab, row_stride, top, teacher_dtype, index_bytes,
                               temperature))
        return rc;
    if ((rows > 0 && (logits == nullptr || teacher == nullptr || indices == nullptr || row_loss == nullptr)) ||
        (mean && count == nullptr))
        return fail(BSSM_ERR_INVALID, "distillation: null pointer");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    DistillArgs a{};
    a.logits = logits; a.teacher = teacher; a.indices = indices; a.rows = rows; a.row_stride = row_stride;
    a.vocab = vocab; a.top = top; a.teacher_dtype = teacher_dtype; a.wide_indices = index_bytes == 8;
    a.temperature = temperature; a.mean = mean; a.count = count; a.row_loss = row_loss;
    a.row_stats = reinterpret_cast<float2 *>(row_stats); a.grad = grad;
    if (mean)
        if (int rc = count_rows(a, count, st)) return rc;
    if (rows > 0)
        if (int rc = launch_rows(dtype, a, false, st)) return rc;
    if (loss == nullptr) return BSSM_OK;
    distill_total<<<1, kThreads, 0, st>>>(row_loss, rows, mean, count, loss);
    return check_launch("distillation");
}

extern "C" int bssm_distillation_backward(const void *logits, int dtype, long rows, int vocab, long row_stride,
                                          const void *teacher, int teacher_dtype, const void *indices, int index_bytes,
                                          int top, float temperature, int mean, const float *row_stats,
                                          const int *count, const float *upstream, int upstream_per_row, void *grad,
                                          void *stream) {
    using namespace bssm;
    if (int rc = check_distill("distillation_backward", dtype, rows, vocab, row_stride, top, teacher_dtype, index_bytes,
                               temperature))
        return rc;
    if ((rows > 0 && (logits == nullptr || teacher == nullptr || indices == nullptr || row_stats == nullptr ||
                      grad == nullptr)) ||
        (mean && count == nullptr))
        return fail(BSSM_ERR_INVALID, "distillation_backward: null pointer");
    if (rows == 0) return BSSM_OK;
    DistillArgs a{};
    a.logits = logits; a.teacher = teacher; a.indices = indices; a.rows = rows; a.row_stride = row_stride;
    a.vocab = vocab; a.top = top; a.teacher_dtype = teacher_dtype; a.wide_indices = index_bytes == 8;
    a.temperature = temperature; a.mean = mean; a.count = count;
    a.row_stats = reinterpret_cast<float2 *>(const_cast<float *>(row_stats));
    a.grad = grad; a.upstream = upstream; a.upstream_per_row = upstream_per_row;
    return launch_rows(dtype, a, true, static_cast<cudaStream_t>(stream));
}

extern "C" int bssm_distillation_scale(void *grad, int dtype, long n, const float *factor, void *stream) {
    using namespace bssm;
    if (!io_dtype_known(dtype)) return fail(BSSM_ERR_UNSUPPORTED, "distillation_scale: unknown dtype");
    if (n < 0 || factor == nullptr || (n > 0 && grad == nullptr))
        return fail(BSSM_ERR_INVALID, "distillation_scale: bad arguments");
    if (n == 0) return BSSM_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const long blocks = (n + 2047) / 2048;
    const unsigned grid = static_cast<unsigned>(blocks < 1184 ? blocks : 1184);
    if (dtype == BSSM_F32) distill_scale<<<grid, 256, 0, st>>>(static_cast<float *>(grad), n, factor);
    else if (dtype == BSSM_BF16) distill_scale<<<grid, 256, 0, st>>>(static_cast<__nv_bfloat16 *>(grad), n, factor);
    else distill_scale<<<grid, 256, 0, st>>>(static_cast<__half *>(grad), n, factor);
    return check_launch("distillation_scale");
}
