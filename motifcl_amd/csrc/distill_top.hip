// Distillation from a teacher's top logits.  With p = softmax(z / T) over the student's whole
// vocabulary and q = softmax(y / T) over the teacher's entries (id, y) of the row,
//     loss = T^2 sum q_i (log q_i - log p_id(i)),   d(weight loss)/dz_j = weight T (p_j sum q - sum over id(i) = j of q_i)
// sum q is 1, or 0 in a row without entries.  One workgroup a row, one launch.  Bound by memory: the logits are
// read once and the gradient is written once where the workgroup's registers hold the row; a longer row is read a
// second time, as far as the registers and caches do not hold it.  The teacher's entries change `top` elements of a
// row: the gradient is written without them first, and once all of it is in memory those elements are written again, each
// by the first of the entries that name it.  Measured: 4096 x 32768 f32 190 us = 5.7 TB/s; 2048 x 128011 f32 493 us, of
// whose 2.9 GB 0.8 are the second read.
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
    float q[kHeld], t_log_q[kHeld];  // q and T log q
    float sum;                    // of q: 1, 0 without entries, NaN where the teacher has no distribution
};
template <typename T>
__device__ __forceinline__ Entries load_entries(const DistillTop& a, size_t row, int lane) {
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
    for (int i = 0; i < kHeld; ++i) e.z[i] = e.id[i] >= 0 ? (float)logits[e.id[i]] : 0.0f;
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
        e.t_log_q[i] = e.y[i] - largest;
        e.q[i] = exp2_of(e.t_log_q[i] * a.inv_temperature * kLog2E);
        sum += e.q[i];
    }
    sum = wave_reduce<Sum>(sum);
    const float log_sum = logf(sum), inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        e.t_log_q[i] -= a.temperature * log_sum;
        e.q[i] *= inv;
    }
    e.sum = sum == 0.0f ? 0.0f : sum * inv;
}
// The entries in LDS.  Writing z here also waits for the load of z, so that behind a barrier the logits may
// be replaced by the gradient.
struct EntryScratch {
    int id[kMostTop];
    float q[kMostTop], t_log_q[kMostTop], z[kMostTop];
    float sum;
    __device__ __forceinline__ void put(const Entries& e, int lane) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            id[lane + 64 * i] = e.id[i];
            q[lane + 64 * i] = e.q[i];
            t_log_q[lane + 64 * i] = e.t_log_q[i];
            z[lane + 64 * i] = e.z[i];
        }
        if (lane == 0) sum = e.sum;
    }
};

// T sum q (T log q - T log p), in every lane of the first wave: neither T^2 nor a difference of logits over T is formed,
// of which a small T would leave 0 and infinity.
__device__ __forceinline__ float loss_of(const DistillTop& a, const EntryScratch& e, float m, float s, int lane) {
    const float t_log_s = a.temperature * logf(s);
    float sum = 0.0f;
#pragma unroll
    for (int i = lane; i < kMostTop; i += 64) {
        const float t_log_p = s == 0.0f ? -__builtin_inff() : e.z[i] - m - t_log_s;
        if (e.id[i] >= 0 && e.q[i] != 0.0f) sum += e.q[i] * (e.t_log_q[i] - t_log_p);
    }
    return a.temperature * wave_reduce<Sum>(sum);
}

// The gradient without the teacher's entries is c 2^((z - base) k).
struct GradientScale {
    float c, scale, base, log2_scale;
    bool zero;  // rows without weight or without entries, and rows of -inf alone, learn nothing
    __device__ __forceinline__ GradientScale(const DistillTop& a, size_t row, float m, float s, float sum_q) {
        const float weight = a.weight ? a.weight[row] : 1.0f;
        scale = weight * a.temperature;
        base = shift_of(m);
        log2_scale = a.log2_scale;
        zero = weight == 0.0f || sum_q == 0.0f || s == 0.0f;
        c = scale * sum_q / s;
    }
    __device__ __forceinline__ float at(float z) const { return zero ? 0.0f : c * exp2_of((z - base) * log2_scale); }
};
template <typename T, int THREADS, int ITERS>
__device__ __forceinline__ void write_stretch(const GradientScale& c, T* out, int n, const RowVectors<T, THREADS, ITERS>& r,
                                              int t) {
    typedef RowVectors<T, THREADS, ITERS> Row;
#pragma unroll
    for (int j = 0; j < ITERS; ++j) {
        float v[Row::kVec];
#pragma unroll
        for (int k = 0; k < Row::kVec; ++k) v[k] = c.at((float)r.raw[j][k]);
        r.store(out, j, t, n, v);
    }
}
// Once the whole row's gradient is written, the elements that the teacher's entries name, by the first wave.  All
// threads call it: first every wave waits until its stores are in memory, for another wave stores some of the same
// elements again, and a barrier alone waits for no store.
template <typename T>
__device__ __forceinline__ void patch_entries(const DistillTop& a, const GradientScale& c, T* out,
                                              const EntryScratch& lds, int t) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t >= 64 || c.zero) return;
    for (int at = t; at < a.top; at += 64) {
        const int id = lds.id[at];
        if (id < 0) continue;
        float q = 0.0f;
        bool first = true;
        for (int other = 0; other < a.top; ++other)
            if (lds.id[other] == id) {
                q += lds.q[other];
                first = first && other >= at;
            }
        if (first) out[id] = (T)(c.at(lds.z[at]) - c.scale * q);
    }
}

// The row in one workgroup's registers: loss and gradient in one launch.
template <typename T, int THREADS, int ITERS>
__global__ __launch_bounds__(THREADS, 8) void distill_row_kernel(DistillTop a) {
    constexpr int kWaves = THREADS / 64;
    typedef RowVectors<T, THREADS, ITERS> Row;
    __shared__ float slots[3 * kWaves];
    __shared__ EntryScratch lds;
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63, n = a.vocab;
    const size_t row = blockIdx.x;
    Row r;
    r.load(static_cast<const T*>(a.logits) + row * a.stride, t, n);
    if (wave == 0) {
        Entries e = load_entries<T>(a, row, lane);
        weigh_entries(a, e);
        lds.put(e, lane);
    }
    r.fill_tail(t, n, (T)-__builtin_inff());
    float thread_max;
    const SoftmaxStats st = stats_of<Row, kWaves, ITERS>(r, a.log2_scale, slots, wave, lane, thread_max);
    if (wave == 0 && a.loss) {
        const float loss = loss_of(a, lds, st.m, st.s, lane);
        if (lane == 0) a.loss[row] = loss;
    }
    __syncthreads();
    if (!a.grad) return;
    const GradientScale c(a, row, st.m, st.s, lds.sum);
    T* out = static_cast<T*>(a.grad) + row * a.grad_stride;
    write_stretch<T, THREADS, ITERS>(c, out, n, r, t);
    patch_entries(a, c, out, lds, t);
}

// A row longer than a workgroup's registers (2048 x 128011 f32: 493 us; stretches of rows in workgroups of their
// own, in a launch for the statistics, one for the losses and one for the gradient, 566 us): the workgroup sweeps
// the row in stretches, every thread with a maximum and a sum of its own, joins them, and sweeps back
// to write the gradient, from the last stretch, which it still holds, to the first.  A thread adds a stretch's numbers
// up by themselves and the stretches in binary64, so that the error of its sum does not grow with the row (of 34000
// equal numbers of a row of 35 million one running sum in binary32 was off by 3600 half steps).
template <typename T>
__global__ __launch_bounds__(1024, 8) void distill_sweep_kernel(DistillTop a, int segments, int length) {
    constexpr int kThreads = 1024, kIters = 8, kWaves = kThreads / 64;
    typedef RowVectors<T, kThreads, kIters> Row;
    __shared__ float slots[2 * kWaves];
    __shared__ EntryScratch lds;
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const size_t row = blockIdx.x;
    const T* logits = static_cast<const T*>(a.logits) + row * a.stride;
    if (wave == 0) {
        Entries e = load_entries<T>(a, row, lane);
        weigh_entries(a, e);
        lds.put(e, lane);
    }
    Row r;
    float m = -__builtin_inff();
    double s = 0.0;
    int from = 0, n = 0;
#pragma unroll 1
    for (int i = 0; i < segments; ++i) {
        from = i * length, n = a.vocab - from < length ? a.vocab - from : length;
        r.template load<false>(logits + from, again(t), n);  // read again below: kept in the caches
        r.fill_tail(t, n, (T)-__builtin_inff());
        float largest = m;
#pragma unroll
        for (int j = 0; j < kIters; ++j)
#pragma unroll
            for (int k = 0; k < Row::kVec; ++k) largest = fmaxf(largest, (float)r.raw[j][k]);
        r.convert_again();
        const float base = shift_of(largest);
        if (m != -__builtin_inff()) s *= (double)exp2_of((m - base) * a.log2_scale);
        m = largest;
        float part = 0.0f;
#pragma unroll
        for (int j = 0; j < kIters; ++j)
#pragma unroll
            for (int k = 0; k < Row::kVec; ++k) part += exp2_of(((float)r.raw[j][k] - base) * a.log2_scale);
        s += (double)part;
    }
    r.convert_again();
    float all_m[1] = {m}, all_s[1];
    row_reduce<Max, kWaves>(all_m, slots, wave, lane);
    all_s[0] = (float)s;
    if (m != -__builtin_inff()) all_s[0] *= exp2_of((m - shift_of(all_m[0])) * a.log2_scale);
    row_reduce<Sum, kWaves>(all_s, slots + kWaves, wave, lane);
    if (wave == 0 && a.loss) {
        const float loss = loss_of(a, lds, all_m[0], all_s[0], lane);
        if (lane == 0) a.loss[row] = loss;
    }
    if (!a.grad) return;
    const GradientScale c(a, row, all_m[0], all_s[0], lds.sum);
    T* out = static_cast<T*>(a.grad) + row * a.grad_stride;
#pragma unroll 1
    for (int i = segments - 1;; --i) {
        write_stretch<T, kThreads, kIters>(c, out + from, n, r, again(t));
        if (i == 0) break;
        from = (i - 1) * length, n = length;
        r.load(logits + from, again(t), n);
    }
    patch_entries(a, c, out, lds, t);
}
template <typename T>
hipError_t distill(hipStream_t stream, const DistillTop& a) {
    const RowCut c = cut_rows(a.vocab, Elements<T>::kVec);
    if (c.segments > 1) {
        hipLaunchKernelGGL(distill_sweep_kernel<T>, dim3((unsigned)a.rows), dim3(1024), 0, stream, a, c.segments, c.length);
        return hipGetLastError();
    }
    for_shape<T>(c, [&](auto threads, auto iters) {
        constexpr int THREADS = decltype(threads)::value, ITERS = decltype(iters)::value;
        hipLaunchKernelGGL((distill_row_kernel<T, THREADS, ITERS>), dim3((unsigned)a.rows), dim3(THREADS), 0, stream, a);
    });
    return hipGetLastError();
}

}  // namespace

hipError_t launch_distill_top(hipStream_t stream, ElementType type, const DistillTop& a) {
    hipError_t e = hipSuccess;
    for (size_t done = 0; done < a.rows && e == hipSuccess; done += kMostLaunchRows) {
        DistillTop p = a;
        p.rows = a.rows - done < kMostLaunchRows ? a.rows - done : kMostLaunchRows;
        p.logits = static_cast<const char*>(a.logits) + done * a.stride * element_size(type);
        p.ids = a.ids + done * a.top;
        p.teacher = a.teacher + done * a.top;
        if (a.weight) p.weight = a.weight + done;
        if (a.loss) p.loss = a.loss + done;
        if (a.grad) p.grad = static_cast<char*>(a.grad) + done * a.grad_stride * element_size(type);
        switch (type) {
            case ElementType::F32: e = distill<float>(stream, p); break;
            case ElementType::F16: e = distill<_Float16>(stream, p); break;
            case ElementType::BF16: e = distill<__bf16>(stream, p); break;
        }
    }
    return e;
}

}  // namespace mcc
