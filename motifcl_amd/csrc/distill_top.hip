// Distillation from a teacher's top logits.  With p = softmax(z / T) over the student's whole
// vocabulary and q = softmax(y / T) over the teacher's entries (id, y) of the row,
//     loss = T^2 sum q_i (log q_i - log p_id(i)),   d(weight loss)/dz_j = weight T (p_j sum q - sum over id(i) = j of q_i)
// sum q is 1, or 0 in a row without entries.  Bound by memory: the logits are read once and the gradient
// is written once.  A workgroup that holds its row in registers does both in one launch; longer rows
// are cut into stretches: statistics of the stretches, then the rows'
// losses, then the gradient from a second read.  The teacher's entries change `top` elements of a row: the
// gradient is written without them first and those elements are written again by the same workgroup
// behind a barrier, each by the first of the entries that name it.
#include <hip/hip_runtime.h>

#include <cmath>

#include "launch.hpp"
#include "row_softmax.hpp"
#include "row_values.hpp"

namespace mcc {
namespace {

// What the first wave knows of a row's teacher: lane l holds entries l and l + 64.
constexpr int kHeld = kMostTop / 64;
struct Entries {
    int id[kHeld];                // -1: none
    float z[kHeld], y[kHeld];     // the student's logit at id, the teacher's
    float q[kHeld], log_q[kHeld];
    float sum;                    // of q: 1, 0 without entries, NaN where the teacher has no distribution
};
// The logits of the entries in [from, from + n) alone are read.
template <typename T>
__device__ __forceinline__ Entries load_entries(const DistillTop& a, size_t row, int from, int n, int lane) {
    Entries e;
    const T* logits = static_cast<const T*>(a.logits) + row * a.stride;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int at = lane + 64 * i;
        e.id[i] = at < a.top ? a.ids[row * a.top + at] : -1;
        e.y[i] = at < a.top ? a.teacher[row * a.top + at] : 0.0f;
        if (e.id[i] < 0 || e.id[i] >= a.vocab) e.id[i] = -1, e.y[i] = -__builtin_inff();
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i) e.z[i] = e.id[i] >= from && e.id[i] - from < n ? (float)logits[e.id[i]] : 0.0f;
    return e;
}
__device__ __forceinline__ void weigh_entries(const DistillTop& a, Entries& e) {
    float largest = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < kHeld; ++i) largest = fmaxf(largest, e.y[i]);
    largest = shift_of(wave_reduce<Max>(largest));
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        e.log_q[i] = (e.y[i] - largest) * a.inv_temperature;
        e.q[i] = exp2_of(e.log_q[i] * kLog2E);
        sum += e.q[i];
    }
    sum = wave_reduce<Sum>(sum);
    const float log_sum = logf(sum), inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        e.log_q[i] -= log_sum;
        e.q[i] *= inv;
    }
    e.sum = sum == 0.0f ? 0.0f : sum * inv;
}
// T^2 sum q (log q - log p), in every lane of the first wave
__device__ __forceinline__ float loss_of(const DistillTop& a, const Entries& e, float m, float s) {
    const float log_s = logf(s);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const float log_p = s == 0.0f ? -__builtin_inff() : (e.z[i] - m) * a.inv_temperature - log_s;
        if (e.id[i] >= 0 && e.q[i] != 0.0f) sum += e.q[i] * (e.log_q[i] - log_p);
    }
    return a.temperature * a.temperature * wave_reduce<Sum>(sum);
}

// The entries for the patch.  Writing z here also waits for the load of z, so that behind a barrier
// the logits may be replaced by the gradient.
struct PatchScratch {
    int id[kMostTop];
    float q[kMostTop], z[kMostTop];
    float sum;
    __device__ __forceinline__ void put(const Entries& e, int lane) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            id[lane + 64 * i] = e.id[i];
            q[lane + 64 * i] = e.q[i];
            z[lane + 64 * i] = e.z[i];
        }
        if (lane == 0) sum = e.sum;
    }
};

// Gradient of a stretch whose logits are in registers: v = c 2^((z - m) k), and the teacher's entries in
// it once more, by the first wave.  A barrier lies between lds.put() and this.
template <typename T, int THREADS, int ITERS>
__device__ __forceinline__ void write_gradient(const DistillTop& a, size_t row, int from, int n,
                                               const RowVectors<T, THREADS, ITERS>& r, float m, float s,
                                               const PatchScratch& lds, int t) {
    typedef RowVectors<T, THREADS, ITERS> Row;
    const float weight = a.weight ? a.weight[row] : 1.0f, scale = weight * a.temperature, base = shift_of(m);
    // rows without weight or without entries, and rows of -inf alone, learn nothing
    const bool zero = weight == 0.0f || lds.sum == 0.0f || s == 0.0f;
    const float c = scale * lds.sum / s;
    T* out = static_cast<T*>(a.grad) + row * a.grad_stride;
#pragma unroll
    for (int j = 0; j < ITERS; ++j) {
        float v[Row::kVec];
#pragma unroll
        for (int k = 0; k < Row::kVec; ++k)
            v[k] = zero ? 0.0f : c * exp2_of(((float)r.raw[j][k] - base) * a.log2_scale);
        store_row_vector<T, THREADS, ITERS>(out + from, j, t, n, v);
    }
    __syncthreads();
    if (t >= 64 || zero) return;
    for (int at = t; at < a.top; at += 64) {
        const int id = lds.id[at];
        if (id < from || id - from >= n) continue;
        float q = 0.0f;
        bool first = true;
        for (int other = 0; other < a.top; ++other)
            if (lds.id[other] == id) {
                q += lds.q[other];
                first = first && other >= at;
            }
        if (first) out[id] = (T)(c * exp2_of((lds.z[at] - base) * a.log2_scale) - scale * q);
    }
}

// The row in one workgroup's registers: loss and gradient in one launch.
template <typename T, int THREADS, int PER_THREAD>
__global__ __launch_bounds__(THREADS) void distill_row_kernel(DistillTop a) {
    constexpr int kIters = PER_THREAD / Elements<T>::kVec, kWaves = THREADS / 64;
    typedef RowVectors<T, THREADS, kIters> Row;
    __shared__ float slots[3 * kWaves];
    __shared__ PatchScratch lds;
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63, n = a.vocab;
    const size_t row = blockIdx.x;
    Row r;
    r.load(static_cast<const T*>(a.logits) + row * a.stride, t, n);
    Entries e{};
    if (wave == 0) {
        e = load_entries<T>(a, row, 0, n, lane);
        weigh_entries(a, e);
        lds.put(e, lane);
    }
    r.fill_tail(t, n, (T)-__builtin_inff());
    float thread_max;
    const SoftmaxStats st = stats_of<Row, kWaves, kIters>(r, a.log2_scale, slots, wave, lane, thread_max);
    if (wave == 0 && a.loss) {
        const float loss = loss_of(a, e, st.m, st.s);
        if (lane == 0) a.loss[row] = loss;
    }
    __syncthreads();
    if (a.grad) write_gradient<T, THREADS, kIters>(a, row, 0, n, r, st.m, st.s, lds, t);
}

// Rows cut into stretches.  One wave a row joins the statistics into stats[row * segments] (the gradient
// reads them there) and writes the loss.
template <typename T>
__global__ __launch_bounds__(64) void distill_loss_kernel(DistillTop a, int segments, SoftmaxStats* stats) {
    const size_t row = blockIdx.x;
    Entries e = load_entries<T>(a, row, 0, a.vocab, threadIdx.x);
    SoftmaxStats st = stats[row * segments];
    for (int i = 1; i < segments; ++i) st = join_stats(st, stats[row * segments + i], a.log2_scale);
    weigh_entries(a, e);
    const float loss = loss_of(a, e, st.m, st.s);
    if (threadIdx.x == 0) {
        if (a.loss) a.loss[row] = loss;
        stats[row * segments] = st;
    }
}
template <typename T, int THREADS, int PER_THREAD>
__global__ __launch_bounds__(THREADS) void distill_gradient_kernel(DistillTop a, int segments, int length,
                                                                   const SoftmaxStats* stats) {
    constexpr int kIters = PER_THREAD / Elements<T>::kVec;
    typedef RowVectors<T, THREADS, kIters> Row;
    __shared__ PatchScratch lds;
    const int t = threadIdx.x;
    const size_t row = blockIdx.x / (unsigned)segments;
    const int from = (int)(blockIdx.x % (unsigned)segments) * length, n = a.vocab - from < length ? a.vocab - from : length;
    Row r;
    r.load(static_cast<const T*>(a.logits) + row * a.stride + from, t, n);
    if (t < 64) {  // another workgroup may have replaced the logits of the entries outside this stretch
        Entries e = load_entries<T>(a, row, from, n, t);
        weigh_entries(a, e);
        lds.put(e, t);
    }
    const SoftmaxStats st = stats[row * segments];
    __syncthreads();
    write_gradient<T, THREADS, kIters>(a, row, from, n, r, st.m, st.s, lds, t);
}

template <typename T>
hipError_t distill(hipStream_t stream, ElementType type, const DistillTop& a, void* workspace) {
    const RowCut c = cut_rows(a.vocab);
    if (c.segments > 1) {
        SoftmaxStats* stats = static_cast<SoftmaxStats*>(workspace);
        hipError_t e = launch_softmax_stats(stream, type, a.logits, a.stride, a.rows, a.vocab, a.log2_scale, c, stats);
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL(distill_loss_kernel<T>, dim3((unsigned)a.rows), dim3(64), 0, stream, a, c.segments, stats);
        e = hipGetLastError();
        if (e != hipSuccess || !a.grad) return e;
        hipLaunchKernelGGL((distill_gradient_kernel<T, 1024, 32>), dim3((unsigned)(a.rows * c.segments)), dim3(1024), 0,
                           stream, a, c.segments, c.length, stats);
        return hipGetLastError();
    }
#define MCC_DISTILL(THREADS, PER_THREAD)                                                                              \
    if (c.threads == THREADS && c.per_thread == PER_THREAD)                                                           \
    hipLaunchKernelGGL((distill_row_kernel<T, THREADS, PER_THREAD>), dim3((unsigned)a.rows), dim3(THREADS), 0, stream, a)
    MCC_DISTILL(64, 8);
    MCC_DISTILL(64, 32);
    MCC_DISTILL(256, 16);
    MCC_DISTILL(256, 32);
    MCC_DISTILL(512, 32);
    MCC_DISTILL(1024, 32);
#undef MCC_DISTILL
    return hipGetLastError();
}

}  // namespace

size_t distill_top_workspace_nbytes(size_t rows, int vocab) {
    const RowCut c = cut_rows(vocab);
    return c.segments == 1 ? 0 : rows * c.segments * sizeof(SoftmaxStats);
}

hipError_t launch_distill_top(hipStream_t stream, ElementType type, const DistillTop& a, void* workspace) {
    switch (type) {
        case ElementType::F32: return distill<float>(stream, type, a, workspace);
        case ElementType::F16: return distill<_Float16>(stream, type, a, workspace);
        case ElementType::BF16: return distill<__bf16>(stream, type, a, workspace);
    }
    return hipErrorInvalidValue;
}

}  // namespace mcc
