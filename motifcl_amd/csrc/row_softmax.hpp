// The softmax statistics of a stretch of a row in registers, and how a row is cut into stretches.
// With d = (z - max) k and k = log2(e) / temperature over the stretch:
//     m = max z,  s = sum 2^d,  u = sum 2^d d
// from which log sum e^(z / temperature) = m / temperature + log s and the entropy is log s - log(2) u / s.
// Stretches are joined by m = max m_i, r_i = 2^((m_i - m) k), s = sum r_i s_i, u = sum r_i (u_i + s_i (m_i - m) k).  A stretch of -inf alone has m = -inf, s = u = 0; a NaN or
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
__device__ __forceinline__ SoftmaxStats join_stats(SoftmaxStats a, SoftmaxStats b, float k) {
    const float m = fmaxf(a.m, b.m), base = shift_of(m);
    const float da = (a.m - base) * k, db = (b.m - base) * k;
    const float ra = exp2_of(da), rb = exp2_of(db);
    // an empty stretch has d = -inf: its sums are zero and stay so
    return {m, ra * a.s + rb * b.s, ra * (a.u + a.s * fmaxf(da, -1e4f)) + rb * (b.u + b.s * fmaxf(db, -1e4f))};
}

// scale is k above; slots: 3 * WAVES floats of LDS that no wave still reads
template <typename ROW, int WAVES, int ITERS>
__device__ __forceinline__ SoftmaxStats stats_of(const ROW& r, float scale, float* slots, int wave, int lane,
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
    // the difference first: of logits at the type's lowest value, as masks may leave a row, z k overflows
    const float base = shift_of(st.m);
    float sums[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < ITERS; ++j)
#pragma unroll
        for (int k = 0; k < ROW::kVec; ++k) {
            const float d = ((float)r.raw[j][k] - base) * scale, e = exp2_of(d);
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
constexpr int kMostHeld = 32768;  // numbers in the registers of a workgroup of 1024 threads
// Rows are cut only where a workgroup cannot hold one.  Cutting few rows further, so that more CUs read
// them, does not pay for the launch that joins the stretches: one row of 32768 f32 takes 30.7 us from call to
// end whole and 34.6 us in eight stretches, 200 rows 35 and 39 us, one row of 128011 37 us in four stretches
// and 45 us in 32.
inline RowCut cut_rows(int vocab) {
    RowCut c;
    c.segments = (int)(((size_t)vocab + kMostHeld - 1) / kMostHeld);
    const size_t even = ((size_t)vocab + c.segments - 1) / c.segments;
    c.length = (int)((even + 7) / 8 * 8);  // stretches begin where 16-byte accesses of an aligned row do
    if (c.segments > 1) c.threads = 1024, c.per_thread = 32;  // longer than half of what it holds
    else if (vocab <= 512) c.threads = 64, c.per_thread = 8;
    else if (vocab <= 2048) c.threads = 64, c.per_thread = 32;
    else if (vocab <= 4096) c.threads = 256, c.per_thread = 16;
    else if (vocab <= 8192) c.threads = 256, c.per_thread = 32;
    else if (vocab <= 16384) c.threads = 512, c.per_thread = 32;
    else c.threads = 1024, c.per_thread = 32;
    return c;
}

}  // namespace mcc
