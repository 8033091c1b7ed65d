// Rows of numbers held in registers: element types, 16-byte accesses to rows of any alignment, and
// reductions over a wave and over the waves of a workgroup.  Shared by the row-wise operators (layer
// norm, token log probabilities, distillation loss).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace mcc {

// Element types of a tensor; everything computed from one is held in 32 bits and rounded once, to
// nearest even, when it is stored.
template <typename T>
struct Elements;
template <>
struct Elements<float> {
    static constexpr int kVec = 4;
    typedef float Vec __attribute__((ext_vector_type(4), aligned(4)));
};
template <>
struct Elements<_Float16> {
    static constexpr int kVec = 8;
    typedef _Float16 Vec __attribute__((ext_vector_type(8), aligned(2)));
};
template <>
struct Elements<__bf16> {
    static constexpr int kVec = 8;
    typedef __bf16 Vec __attribute__((ext_vector_type(8), aligned(2)));
};

// The vectors of 16 bytes that one of `threads` threads holds of a row of n elements: vector j of
// thread t covers the elements from (j * threads + t) * kVec.  A vector that would reach behind the
// row's end is read from the row's last kVec elements instead, so that every load is unconditional
// and in bounds; the elements it shares with the vector before it become `fill`, as do those of
// vectors that lie behind the end altogether.  Rows shorter than a vector are read one by one.
// 16-byte accesses need no more than the alignment of an element (unaligned access is enabled on
// this platform), so row strides and base pointers are free.  Rows are streamed past the caches' replacement
// order: every element is read once (32768 x 4096 bf16 backward: 156 -> 143 us; logits of 4096 x 32768 f32:
// 94 -> 85 us).  A row that does not begin on a cache line is read through them, for its waves share the lines
// where they meet (32768 x 4097 f32: 207 us, streamed 215 us).
__host__ __device__ inline bool streamed(const void* row) { return (reinterpret_cast<uintptr_t>(row) & 127) == 0; }

template <typename T, int THREADS, int ITERS>
struct RowVectors {
    static constexpr int kVec = Elements<T>::kVec;
    typedef typename Elements<T>::Vec Vec;
    Vec raw[ITERS];

    static __device__ __forceinline__ int first(int j, int t) { return (j * THREADS + t) * kVec; }
    // where vector j of thread t is read from (rows of at least kVec elements)
    static __device__ __forceinline__ int place(int j, int t, int n) {
        const int e = first(j, t);
        return e < n - kVec ? e : n - kVec;
    }

    template <bool STREAM>
    __device__ __forceinline__ void load_as(const T* row, int t, int n) {
        if (n >= kVec) {
#pragma unroll
            for (int j = 0; j < ITERS; ++j) {
                const Vec* p = reinterpret_cast<const Vec*>(row + place(j, t, n));
                raw[j] = STREAM ? __builtin_nontemporal_load(p) : *p;
            }
        } else {
#pragma unroll
            for (int j = 0; j < ITERS; ++j)
#pragma unroll
                for (int k = 0; k < kVec; ++k) raw[j][k] = first(j, t) + k < n ? row[first(j, t) + k] : (T)0.0f;
        }
    }
    __device__ __forceinline__ void load(const T* row, int t, int n) {
        if (streamed(row)) load_as<true>(row, t, n);
        else load_as<false>(row, t, n);
    }
    __device__ __forceinline__ void fill_tail(int t, int n, T fill) {
#pragma unroll
        for (int j = 0; j < ITERS; ++j) {
            if ((j + 1) * THREADS * kVec <= n) continue;  // the same for every thread
            const int e = first(j, t), at = n >= kVec ? place(j, t, n) : e;
#pragma unroll
            for (int k = 0; k < kVec; ++k)
                if (at + k < e || at + k >= n) raw[j][k] = fill;
        }
    }
    // Index of element k of vector j in the row; not less than n, or less than first(), for one that
    // fill_tail() filled.
    static __device__ __forceinline__ int index(int j, int k, int t, int n) {
        return (n >= kVec ? place(j, t, n) : first(j, t)) + k;
    }
    static __device__ __forceinline__ bool holds(int j, int k, int t, int n) {
        const int i = index(j, k, t, n);
        return i >= first(j, t) && i < n;
    }
};

// Stores vector j of thread t, past the caches as well: whole where it lies inside the row, else its elements one by one.
template <typename T, int THREADS, int ITERS>
__device__ __forceinline__ void store_row_vector(T* row, int j, int t, int n,
                                                 const float (&v)[Elements<T>::kVec]) {
    typedef RowVectors<T, THREADS, ITERS> Row;
    typedef typename Row::Vec Vec;
    const int e = Row::first(j, t);
    if (e + Row::kVec <= n) {
        Vec out;
#pragma unroll
        for (int k = 0; k < Row::kVec; ++k) out[k] = (T)v[k];
        __builtin_nontemporal_store(out, reinterpret_cast<Vec*>(row + e));
    } else if (e < n) {
#pragma unroll
        for (int k = 0; k < Row::kVec; ++k)
            if (Row::holds(j, k, t, n)) row[Row::index(j, k, t, n)] = (T)v[k];
    }
}

// ---- reductions: the same order on every call -------------------------------------------------
struct Sum {
    static __device__ __forceinline__ float identity() { return 0.0f; }
    static __device__ __forceinline__ float join(float a, float b) { return a + b; }
};
struct Max {
    static __device__ __forceinline__ float identity() { return -__builtin_inff(); }
    static __device__ __forceinline__ float join(float a, float b) { return fmaxf(a, b); }
};

// One step of a wave's reduction as a DPP operand; lanes without a source take `x`'s identity.
template <typename OP, int CTRL, int ROWS>
__device__ __forceinline__ float dpp_join(float x) {
    const int idle = (int)__float_as_uint(OP::identity());
    const int y = __builtin_amdgcn_update_dpp(idle, (int)__float_as_uint(x), CTRL, ROWS, 0xf, false);
    return OP::join(x, __uint_as_float((uint32_t)y));
}
// The reduction of all 64 lanes, in every lane (as a scalar).
template <typename OP>
__device__ __forceinline__ float wave_reduce(float x) {
    x = dpp_join<OP, 0x111, 0xf>(x);  // row_shr:1, 2, 4, 8 within 16 lanes
    x = dpp_join<OP, 0x112, 0xf>(x);
    x = dpp_join<OP, 0x114, 0xf>(x);
    x = dpp_join<OP, 0x118, 0xf>(x);
    x = dpp_join<OP, 0x142, 0xa>(x);  // row_bcast:15 into rows 1 and 3
    x = dpp_join<OP, 0x143, 0xc>(x);  // row_bcast:31 into rows 2 and 3
    return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x), 63));
}
// The reduction of N numbers over WAVES waves of one row, in every thread.  `slots` are WAVES * N
// floats of LDS that no wave still reads (two calls in a row take different ones); waves of
// workgroups that hold several rows call it together.
template <typename OP, int WAVES, int N>
__device__ __forceinline__ void row_reduce(float (&x)[N], float* slots, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = wave_reduce<OP>(x[i]);
    if (WAVES == 1) return;
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) slots[wave * N + i] = x[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (WAVES <= 4) {
            float a = slots[i];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) a = OP::join(a, slots[w * N + i]);
            x[i] = a;
        } else {  // one read a lane instead of one a wave: fewer registers
            x[i] = wave_reduce<OP>(lane < WAVES ? slots[lane * N + i] : OP::identity());
        }
    }
}

constexpr float kLog2E = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// 2^x by the hardware's instruction: within 2^-23 of the value, relative; results below 2^-126 are 0.
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

}  // namespace mcc
