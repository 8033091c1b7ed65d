// The softmax statistics of a stretch of a row in registers, and how a row is cut into stretches.
// With d = (z - max) k and k = log2(e) / temperature over the stretch:
//     m = max z,  s = sum 2^d,  u = sum 2^d d
// from which log sum e^(z / temperature) = m / temperature + log s and the entropy is log s - log(2) u / s.
// Stretches are joined by m = max m_i, r_i = 2^((m_i - m) k), s = sum r_i s_i, u = sum r_i (u_i + s_i (m_i - m) k).
// A stretch of -inf alone has m = -inf, s = u = 0; a NaN or +inf makes s (and with it everything taken from the
// row) NaN.
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

// A row's stretches, joined in their order.  The sums are binary64: a row may have 32768 stretches, and the error of a
// sum in binary32 grows with their number (16385 equal ones: 2300 half steps).
struct JoinedStats {
    float m;
    double s, u;
    __device__ __forceinline__ explicit JoinedStats(const SoftmaxStats& a) : m(a.m), s(a.s), u(a.u) {}
    __device__ __forceinline__ void join(const SoftmaxStats& b, float k) {
        const float most = fmaxf(m, b.m), base = shift_of(most);
        const float da = (m - base) * k, db = (b.m - base) * k;
        const double ra = exp2_of(da), rb = exp2_of(db);
        // an empty stretch has d = -inf: its sums are zero and stay so
        u = ra * (u + s * (double)fmaxf(da, -1e4f)) + rb * ((double)b.u + (double)b.s * (double)fmaxf(db, -1e4f));
        s = ra * s + rb * (double)b.s;
        m = most;
    }
    __device__ __forceinline__ SoftmaxStats stats() const { return {m, (float)s, (float)u}; }
};

// scale is k above; slots: 3 * WAVES floats of LDS that no wave still reads.  A thread adds its kVec * ITERS numbers, 32
// of f32 and at most 64 of 16 bits, one behind the other, and at most 12 joins follow.
template <typename ROW, int WAVES, int ITERS>
__device__ __forceinline__ SoftmaxStats stats_of(ROW& r, float scale, float* slots, int wave, int lane,
                                                 float& thread_max) {
    SoftmaxStats st;
    float largest[1] = {-__builtin_inff()};
#pragma unroll
    for (int j = 0; j < ITERS; ++j)
#pragma unroll
        for (int k = 0; k < ROW::kVec; ++k) largest[0] = fmaxf(largest[0], (float)r.raw[j][k]);
    thread_max = largest[0];
    row_reduce<Max, WAVES>(largest, slots, wave, lane);
    r.convert_again();
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
    r.convert_again();
    st.s = sums[0];
    st.u = sums[1];
    return st;
}

// A row of `vocab` numbers is cut into `segments` stretches of `length` numbers (the last may be
// shorter), each held by a workgroup of `threads` threads, `iters` vectors of `vec` numbers a thread.
struct RowCut {
    int threads, iters, segments, length;
};
// Rows are cut only where a workgroup cannot hold one, in at most 32 registers a thread.  Cutting few rows
// further, so that more CUs read them, does not pay for the launch that joins the stretches: one row of 32768
// f32 takes 30.7 us from call to end whole and 34.6 us in eight stretches, 200 rows 35 and 39 us.
// Sixteen-bit rows are bound by the vector units and want few waves, which share the work that is done once a
// wave: 64 numbers a thread (distillation of 16384 x 3001 bf16: 55 us in one wave, 67 us in four; of 4096 x 16384:
// 56 us with 256 or 512 threads, 72 us with 1024).  f32 rows are bound by memory and want many (of 16384 x 3001 f32:
// 83 us in two waves, 77 us in four; of 4096 x 16384: 114 us with 512 threads, 103 us with 1024).
inline RowCut cut_rows(int vocab, int vec) {
    RowCut c;
    const int most = 1024 * 8 * vec;
    c.segments = (int)(((size_t)vocab + most - 1) / most);
    const size_t even = ((size_t)vocab + c.segments - 1) / c.segments, line = kLineBytes / 2;
    // stretches of an aligned row begin on lines; at most `most`, so that none is left empty
    c.length = (int)((even + line - 1) / line * line);
    const int n = c.length < vocab ? c.length : vocab;
    if (c.segments > 1) c.threads = 1024, c.iters = 8;
    else if (n <= 512) c.threads = 64, c.iters = 8 / vec;
    else if (n <= 2048) c.threads = 64, c.iters = 32 / vec;
    else if (vec == 8) c.threads = n <= 4096 ? 64 : n <= 8192 ? 128 : n <= 16384 ? 256 : n <= 32768 ? 512 : 1024, c.iters = 8;
    else if (n <= 4096) c.threads = 256, c.iters = 4;
    else if (n <= 8192) c.threads = 256, c.iters = 8;
    else c.threads = 1024, c.iters = n <= 16384 ? 4 : 8;
    return c;
}

// Calls launch(threads, iters), both as types with a ::value, for the shape that a row of one stretch takes.
template <int V>
struct Int {
    static constexpr int value = V;
};
template <typename T, typename F>
void for_shape(const RowCut& c, F&& launch) {
    constexpr int vec = Elements<T>::kVec;
    if (c.threads == 64 && c.iters == 8 / vec) launch(Int<64>(), Int<8 / vec>());
    else if (c.threads == 64 && c.iters == 32 / vec) launch(Int<64>(), Int<32 / vec>());
    else if constexpr (vec == 8) {
        if (c.threads == 64) launch(Int<64>(), Int<8>());
        else if (c.threads == 128) launch(Int<128>(), Int<8>());
        else if (c.threads == 256) launch(Int<256>(), Int<8>());
        else if (c.threads == 512) launch(Int<512>(), Int<8>());
        else launch(Int<1024>(), Int<8>());
    } else {
        if (c.threads == 256 && c.iters == 4) launch(Int<256>(), Int<4>());
        else if (c.threads == 256) launch(Int<256>(), Int<8>());
        else if (c.iters == 4) launch(Int<1024>(), Int<4>());
        else launch(Int<1024>(), Int<8>());
    }
}

}  // namespace mcc
