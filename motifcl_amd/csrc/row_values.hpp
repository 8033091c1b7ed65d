// Rows of numbers held in registers: element types, 16-byte accesses to rows of any alignment, and
// reductions over a wave and over the waves of a workgroup.  Shared by the row-wise operators (layer
// norm, token log probabilities, distillation loss).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace mcc {

constexpr int kLineBytes = 128;  // of the L2 cache
__host__ __device__ inline bool whole_lines(const void* p) { return reinterpret_cast<uintptr_t>(p) % kLineBytes == 0; }

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

// The same number, which the compiler takes for a new one: indexes computed from it are computed where they are
// needed instead of being held in registers since the loads.
__device__ __forceinline__ int again(int t) {
    asm volatile("" : "+v"(t));
    return t;
}

// The vectors of 16 bytes that one of THREADS threads holds of a row of n elements: vector j of thread t
// covers the elements from first(j, t) = (j * THREADS + t) * kVec - lead.  lead is 0, so that a row's sums are
// taken in the same order wherever it lies, but for SHIFTED, where it moves the vectors back to the cache line
// that the row begins in: a wave's accesses are then whole lines whatever the row's alignment (gradients of
// 4096 x 32003 f32 logits: 196 us without).  A vector that reaches over an end of the row is read from the
// nearest kVec elements inside it, so that every load is unconditional and in bounds; those of them that are
// not its own, and all of a vector outside the row, become `fill`.  Rows shorter than a vector are read one
// by one.  16-byte accesses need no more than the alignment of an element (unaligned access is enabled on this
// platform).
// Rows are streamed past the caches' replacement order, for every element is read once (32768 x 4096 bf16 norm,
// backward: 156 -> 143 us; 4096 x 32768 f32 log probabilities: 94 -> 85 us).
template <typename T, int THREADS, int ITERS, bool SHIFTED = false>
struct RowVectors {
    static constexpr int kVec = Elements<T>::kVec;
    typedef typename Elements<T>::Vec Vec;
    Vec raw[ITERS];
    int lead;

    __device__ __forceinline__ int first(int j, int t) const { return (j * THREADS + t) * kVec - (SHIFTED ? lead : 0); }
    // where vector j of thread t is read from (rows of at least kVec elements)
    __device__ __forceinline__ int place(int j, int t, int n) const {
        const int e = first(j, t), f = SHIFTED && e < 0 ? 0 : e;
        return f < n - kVec ? f : n - kVec;
    }

    // STREAM false: the row is read again soon.  `before`: elements from the line's start to the row's (SHIFTED;
    // n + before at most what is held).
    template <bool STREAM = true>
    __device__ __forceinline__ void load(const T* row, int t, int n, int before = 0) {
        lead = n >= kVec ? before : 0;
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
                for (int k = 0; k < kVec; ++k) raw[j][k] = holds(j, k, t, n) ? row[index(j, k, t, n)] : (T)0.0f;
        }
    }
    // The same numbers, which the compiler takes for new ones: 16-bit numbers are then converted once more in the
    // pass that follows instead of being held as 32 bits since the last.
    __device__ __forceinline__ void convert_again() {
        if (sizeof(T) == 4) return;
        typedef uint32_t Words __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int j = 0; j < ITERS; ++j) {
            Words w = __builtin_bit_cast(Words, raw[j]);
            asm volatile("" : "+v"(w));
            raw[j] = __builtin_bit_cast(Vec, w);
        }
    }
    // whether vectors j of all threads lie inside the row (the same for every thread)
    __device__ __forceinline__ bool whole(int j, int n) const {
        return (j > 0 || !SHIFTED || lead == 0) && first(j + 1, 0) <= n;
    }
    __device__ __forceinline__ void fill_tail(int t, int n, T fill) {
#pragma unroll
        for (int j = 0; j < ITERS; ++j) {
            if (whole(j, n)) continue;
            const int u = again(t);
#pragma unroll
            for (int k = 0; k < kVec; ++k)
                if (!holds(j, k, u, n)) raw[j][k] = fill;
        }
    }
    // Index of element k of vector j in the row, and whether it is the vector's own.
    __device__ __forceinline__ int index(int j, int k, int t, int n) const {
        return (n >= kVec ? place(j, t, n) : first(j, t)) + k;
    }
    __device__ __forceinline__ bool holds(int j, int k, int t, int n) const {
        const int i = index(j, k, t, n), e = first(j, t);
        return i >= e && i < n && (!SHIFTED || i - e < kVec);
    }
    // Stores numbers for vector j of thread t, past the caches as well: whole where the vector lies inside the
    // row, else its own elements one by one.
    __device__ __forceinline__ void store(T* row, int j, int t, int n, const float (&v)[kVec]) const {
        const int e = first(j, t);
        if ((!SHIFTED || e >= 0) && e + kVec <= n) {
            Vec out;
#pragma unroll
            for (int k = 0; k < kVec; ++k) out[k] = (T)v[k];
            __builtin_nontemporal_store(out, reinterpret_cast<Vec*>(row + e));
        } else if (e < n) {
            const int u = again(t);
#pragma unroll
            for (int k = 0; k < kVec; ++k)
                if (holds(j, k, u, n)) row[index(j, k, u, n)] = (T)v[k];
        }
    }
};

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
