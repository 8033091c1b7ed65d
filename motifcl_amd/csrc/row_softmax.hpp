// The softmax statistics of a stretch of a row in registers, and how a row is cut into stretches.
// With d = (z - max) / temperature over the stretch:
//     m = max z,  s = sum e^d,  u = sum e^d d
// from which log sum e^(z / temperature) = m / temperature + log s and the entropy is log s - u / s.
// Stretches are joined by m = max m_i, r_i = e^((m_i - m) / temperature), s = sum r_i s_i,
// u = sum r_i (u_i + s_i (m_i - m) / temperature).  A stretch of -inf alone has m = -inf, s = u = 0; a NaN or
// +inf makes s (and with it everything taken from the row) NaN.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "launch.hpp"
#include "row_values.hpp"

namespace mcc {

struct SoftmaxStats {
    float m, s, u;
};

// What a maximum is subtracted as: 0 where there is none, so that -inf - (-inf) does not arise.
__device__ __forceinline__ float shift_of(float m) { return m == -__builtin_inff() ? 0.0f : m; }

// a joined to b; the order of the operands is the order of the stretches
__device__ __forceinline__ SoftmaxStats join_stats(SoftmaxStats a, SoftmaxStats b, float inv_temperature) {
    const float m = fmaxf(a.m, b.m), base = shift_of(m);
    const float da = (a.m - base) * inv_temperature, db = (b.m - base) * inv_temperature;
    const float ra = fast_exp(da), rb = fast_exp(db);
    // an empty stretch has d = -inf: its sums are zero and stay so
    return {m, ra * a.s + rb * b.s, ra * (a.u + a.s * fmaxf(da, -1e4f)) + rb * (b.u + b.s * fmaxf(db, -1e4f))};
}

// slots: 3 * WAVES floats of LDS that no wave still reads
template <typename ROW, int WAVES, int ITERS>
__device__ __forceinline__ SoftmaxStats stats_of(const ROW& r, float inv_temperature, float* slots, int wave, int lane,
                                                 float& thread_max) {
    SoftmaxStats st;
    float largest[1] = {-__builtin_inff()};
#pragma unroll
    for (int j = 0; j < ITERS; ++j)
#pragma unroll
        for (int k = 0; k < ROW::kVec; ++k) largest[0] = fmaxf(largest[0], (float)r.raw[j][k]);
    thread_max = largest[0];
    row_reduce<Max, WAVES>(largest, slots, wave, lane);
    st.m = largest[0];
    const float base = shift_of(st.m);
    float sums[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < ITERS; ++j)
#pragma unroll
        for (int k = 0; k < ROW::kVec; ++k) {
            const float d = ((float)r.raw[j][k] - base) * inv_temperature, e = fast_exp(d);
            sums[0] += e;
            sums[1] = fmaf(e, fmaxf(d, -1e4f), sums[1]);  // e is 0 long before the bound: 0 * -inf does not arise
        }
    row_reduce<Sum, WAVES>(sums, slots + WAVES, wave, lane);
    st.s = sums[0];
    st.u = sums[1];
    return st;
}

// A row of `vocab` numbers is cut into `segments` stretches of `length` numbers (the last may be
// shorter), each held by a workgroup of `threads` threads, `per_thread` numbers a thread.
struct RowCut {
    int threads, per_thread, segments, length;
};
// Workgroups that fill the device: two a CU.
constexpr size_t kFillGroups = 512;
inline RowCut cut_rows(size_t rows, int vocab) {
    // as long stretches as a workgroup's registers hold, shorter ones while the rows are too few to give every CU
    // work, but not under 4096 numbers: joining more stretches then costs what their loads save
    int most = 32768;
    while (most > 4096 && rows * (size_t)((vocab + (size_t)most - 1) / most) < kFillGroups) most /= 2;
    RowCut c;
    c.segments = (int)(((size_t)vocab + most - 1) / most);
    const size_t even = ((size_t)vocab + c.segments - 1) / c.segments;
    c.length = (int)((even + 7) / 8 * 8);  // stretches begin where 16-byte accesses of an aligned row do
    c.segments = (int)(((size_t)vocab + c.length - 1) / c.length);
    const int n = c.length < vocab ? c.length : vocab;
    if (n <= 512) c.threads = 64, c.per_thread = 8;
    else if (n <= 2048) c.threads = 64, c.per_thread = 32;
    else if (n <= 4096) c.threads = 256, c.per_thread = 16;
    else if (n <= 8192) c.threads = 256, c.per_thread = 32;
    else if (n <= 16384) c.threads = 512, c.per_thread = 32;
    else c.threads = 1024, c.per_thread = 32;
    return c;
}

// Statistics of every stretch of every row: stats[row * segments + segment].
hipError_t launch_softmax_stats(hipStream_t stream, ElementType type, const void* logits, size_t stride, size_t rows,
                                int vocab, float inv_temperature, const RowCut& cut, SoftmaxStats* stats);

}  // namespace mcc
