// Layer norm of rows and its gradients.
//   mean = sum x / n,  rstd = 1 / sqrt(sum (x - mean)^2 / n + eps),  y = (x - mean) rstd gain + bias
//   h = dy gain,  xhat = (x - mean) rstd:  dx = rstd (h - sum h / n - xhat sum(h xhat) / n),
//   dgain = sum over rows of dy xhat,  dbias = sum over rows of dy
// All of it in binary32, long running sums in binary64; x, y, dy and dx have one element type of 32 or 16 bits.  Bound by memory: a
// row is read once into registers, where the mean is known before the squares are summed (no
// difference of large sums), and the backward pass adds its columns up in registers over all rows of a
// workgroup, so that only one partial row a workgroup is written and added up by a second launch.  No
// atomics: equal calls give equal bytes.  Measured: 32768 x 4096 f32 forward 179 us = 6.0 TB/s; bf16 backward of
// that shape 140 us = 5.7 TB/s; 8192 x 288 f32 forward 5.8 us, backward 10.0 + 3.8 us, both shorter than the calls.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "launch.hpp"
#include "row_values.hpp"

namespace mcc {
namespace {

// The kVec floats of a column vector (gain, bias) that belong to vector j of thread t.
template <typename ROW>
__device__ __forceinline__ void load_columns(const ROW& r, const float* p, int j, int t, int n, float none,
                                             float (&v)[ROW::kVec]) {
    if (!p) {
#pragma unroll
        for (int k = 0; k < ROW::kVec; ++k) v[k] = none;
    } else if (n >= ROW::kVec) {
        const int at = r.place(j, t, n);
#pragma unroll
        for (int k = 0; k < ROW::kVec; k += 4) {
            const Elements<float>::Vec q = *reinterpret_cast<const Elements<float>::Vec*>(p + at + k);
            v[k] = q[0], v[k + 1] = q[1], v[k + 2] = q[2], v[k + 3] = q[3];
        }
    } else {
#pragma unroll
        for (int k = 0; k < ROW::kVec; ++k) v[k] = r.holds(j, k, t, n) ? p[r.index(j, k, t, n)] : none;
    }
}

template <typename ROW>
__device__ __forceinline__ void store_columns(const ROW& r, float* p, int j, int t, int n, const float (&v)[ROW::kVec]) {
    const int e = r.first(j, t);
    if (e + ROW::kVec <= n) {
#pragma unroll
        for (int k = 0; k < ROW::kVec; k += 4) {
            const Elements<float>::Vec q = {v[k], v[k + 1], v[k + 2], v[k + 3]};
            *reinterpret_cast<Elements<float>::Vec*>(p + e + k) = q;
        }
    } else {
#pragma unroll
        for (int k = 0; k < ROW::kVec; ++k)
            if (r.holds(j, k, t, n)) p[r.index(j, k, t, n)] = v[k];
    }
}

__device__ __forceinline__ float inv_sqrt(float x) { return 1.0f / sqrtf(x); }

// THREADS threads hold a row, SLOTS rows share a workgroup (only where a row is one wave's), and each of them
// takes ROWS rows one behind the other, all read at once: gain and bias are then read once for ROWS rows,
// and a reduction serves them all.
template <typename T, int THREADS, int ITERS, int SLOTS, int ROWS>
__global__ __launch_bounds__(THREADS* SLOTS) void layer_norm_kernel(const T* x, size_t x_stride, const float* gain,
                                                                    const float* bias, T* y, size_t y_stride,
                                                                    float* mean_out, float* rstd_out, size_t rows,
                                                                    int n, float inv_n, float eps) {
    static_assert(SLOTS == 1 || THREADS == 64, "waves of a shared workgroup leave one by one");
    typedef RowVectors<T, THREADS, ITERS> Row;
    constexpr int kWaves = THREADS / 64;
    __shared__ float slots[2 * ROWS * kWaves];
    const int t = threadIdx.x % THREADS, wave = t >> 6, lane = threadIdx.x & 63;
    const size_t row = ((size_t)blockIdx.x * SLOTS + __builtin_amdgcn_readfirstlane(threadIdx.x / THREADS)) * ROWS;
    if (row >= rows) return;
    Row r[ROWS];
    float sum[ROWS], squares[ROWS], mean[ROWS], rstd[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {  // rows behind the last are the last once more
        r[i].load(x + (row + i < rows ? row + i : rows - 1) * x_stride, t, n);
        sum[i] = squares[i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        r[i].fill_tail(t, n, (T)0.0f);
#pragma unroll
        for (int j = 0; j < ITERS; ++j)
#pragma unroll
            for (int k = 0; k < Row::kVec; ++k) sum[i] += (float)r[i].raw[j][k];
    }
    row_reduce<Sum, kWaves>(sum, slots, wave, lane);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        mean[i] = sum[i] * inv_n;
#pragma unroll
        for (int j = 0; j < ITERS; ++j) {
            const bool whole = r[i].whole(j, n);
#pragma unroll
            for (int k = 0; k < Row::kVec; ++k) {
                const float d = (float)r[i].raw[j][k] - mean[i];
                if (whole || r[i].holds(j, k, t, n)) squares[i] = fmaf(d, d, squares[i]);
            }
        }
    }
    row_reduce<Sum, kWaves>(squares, slots + ROWS * kWaves, wave, lane);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        rstd[i] = inv_sqrt(squares[i] * inv_n + eps);
        if (t == 0 && row + i < rows) {
            if (mean_out) mean_out[row + i] = mean[i];
            if (rstd_out) rstd_out[row + i] = rstd[i];
        }
    }
#pragma unroll
    for (int j = 0; j < ITERS; ++j) {
        float g[Row::kVec], b[Row::kVec];
        load_columns(r[0], gain, j, t, n, 1.0f, g);
        load_columns(r[0], bias, j, t, n, 0.0f, b);
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            float v[Row::kVec];
#pragma unroll
            for (int k = 0; k < Row::kVec; ++k) v[k] = fmaf(((float)r[i].raw[j][k] - mean[i]) * rstd[i], g[k], b[k]);
            if (row + i < rows) r[i].store(y + (row + i) * y_stride, j, t, n, v);
        }
    }
}

// Rows longer than a workgroup's registers: three passes over the row, the later ones out of the caches.  A thread
// adds n / 1024 numbers, up to 2^20, one behind the other; in binary32 the error of such a sum grows with their number
// (a row of 2^22 numbers 1.1: 700 half steps), so these sums are binary64 until the threads' are joined.  One element an
// access and a workgroup a row: 2048 x 50000 f32 forward 322 us = 2.5 TB/s, backward 566 us; two rows of 2^22 3.7 ms.
constexpr int kLongThreads = 1024;
template <typename T>
__global__ __launch_bounds__(kLongThreads) void layer_norm_long_kernel(const T* x, size_t x_stride, const float* gain,
                                                                       const float* bias, T* y, size_t y_stride,
                                                                       float* mean_out, float* rstd_out, int n,
                                                                       float inv_n, float eps) {
    constexpr int kWaves = kLongThreads / 64;
    __shared__ float slots[2 * kWaves];
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const size_t row = blockIdx.x;
    const T* xr = x + row * x_stride;
    T* yr = y + row * y_stride;
    double mine = 0.0;
    for (int i = t; i < n; i += kLongThreads) mine += (double)(float)xr[i];
    float sum[1] = {(float)mine};
    row_reduce<Sum, kWaves>(sum, slots, wave, lane);
    const float mean = sum[0] * inv_n;
    mine = 0.0;
    for (int i = t; i < n; i += kLongThreads) {
        const float d = (float)xr[i] - mean;
        mine += (double)d * (double)d;
    }
    float squares[1] = {(float)mine};
    row_reduce<Sum, kWaves>(squares, slots + kWaves, wave, lane);
    const float rstd = inv_sqrt(squares[0] * inv_n + eps);
    if (t == 0) {
        if (mean_out) mean_out[row] = mean;
        if (rstd_out) rstd_out[row] = rstd;
    }
    for (int i = t; i < n; i += kLongThreads)  // y may be x: an element is read and written by one thread
        yr[i] = (T)fmaf(((float)xr[i] - mean) * rstd, gain ? gain[i] : 1.0f, bias ? bias[i] : 0.0f);
}

// ---- backward -----------------------------------------------------------------------------------
// A workgroup walks rows blockIdx * SLOTS + slot, + gridDim * SLOTS, ...; every thread keeps its
// columns' sums.  partial: [gridDim][2][n], the gain's and the bias's sums of the workgroup's rows.
template <typename T, int THREADS, int ITERS, int SLOTS>
__global__ __launch_bounds__(THREADS* SLOTS) void layer_norm_backward_kernel(
    const T* grad_out, size_t grad_out_stride, const T* x, size_t x_stride, const float* mean_in, const float* rstd_in,
    const float* gain, T* grad_x, size_t grad_x_stride, float* partial_gain, float* partial_bias, size_t partial_stride,
    size_t rows, int n, float inv_n) {
    typedef RowVectors<T, THREADS, ITERS> Row;
    constexpr int kWaves = THREADS / 64;
    __shared__ float slots[2][SLOTS][2 * kWaves];
    __shared__ float columns[SLOTS > 1 ? SLOTS / 2 : 1][SLOTS > 1 ? THREADS * ITERS * Row::kVec : 1];
    const int t = threadIdx.x % THREADS, slot = threadIdx.x / THREADS, wave = t >> 6, lane = threadIdx.x & 63;
    float dgain[ITERS][Row::kVec] = {}, dbias[ITERS][Row::kVec] = {};
    float g[ITERS][Row::kVec];
    Row rx, rd;
#pragma unroll
    for (int j = 0; j < ITERS; ++j) load_columns(rx, gain, j, t, n, 1.0f, g[j]);
    int turn = 0;
    for (size_t base = (size_t)blockIdx.x * SLOTS; base < rows; base += (size_t)gridDim.x * SLOTS, turn ^= 1) {
        const bool live = base + slot < rows;
        const size_t row = live ? base + slot : rows - 1;
        rx.load(x + row * x_stride, t, n);
        rd.load(grad_out + row * grad_out_stride, t, n);
        const float mean = mean_in[row], rstd = rstd_in[row];
        rd.fill_tail(t, n, (T)0.0f);  // the sums then need no other mask
        rx.fill_tail(t, n, (T)0.0f);
        float sums[2] = {0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < ITERS; ++j)
#pragma unroll
            for (int k = 0; k < Row::kVec; ++k) {
                const float d = (float)rd.raw[j][k], h = d * g[j][k];
                const float xhat = ((float)rx.raw[j][k] - mean) * rstd;
                sums[0] += h;
                sums[1] = fmaf(h, xhat, sums[1]);
                if (live) {
                    dgain[j][k] = fmaf(d, xhat, dgain[j][k]);
                    dbias[j][k] += d;
                }
            }
        row_reduce<Sum, kWaves>(sums, slots[turn][slot], wave, lane);
        if (grad_x && live) {
            const float a = sums[0] * inv_n, b = sums[1] * inv_n;
#pragma unroll
            for (int j = 0; j < ITERS; ++j) {
                float v[Row::kVec];
#pragma unroll
                for (int k = 0; k < Row::kVec; ++k) {
                    const float xhat = ((float)rx.raw[j][k] - mean) * rstd;
                    v[k] = rstd * ((float)rd.raw[j][k] * g[j][k] - a - xhat * b);
                }
                rd.store(grad_x + row * grad_x_stride, j, t, n, v);
            }
        }
    }
    // the slots' sums into slot 0: halves of the slots add the other half's, in a fixed order
#pragma unroll
    for (int half = SLOTS / 2; half >= 1; half /= 2) {
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            float(&mine)[ITERS][Row::kVec] = which ? dbias : dgain;
            __syncthreads();
            if (slot >= half && slot < 2 * half) {
#pragma unroll
                for (int j = 0; j < ITERS; ++j)
#pragma unroll
                    for (int k = 0; k < Row::kVec; ++k) columns[slot - half][(j * Row::kVec + k) * THREADS + t] = mine[j][k];
            }
            __syncthreads();
            if (slot < half) {
#pragma unroll
                for (int j = 0; j < ITERS; ++j)
#pragma unroll
                    for (int k = 0; k < Row::kVec; ++k) mine[j][k] += columns[slot][(j * Row::kVec + k) * THREADS + t];
            }
        }
    }
    if (slot != 0) return;
#pragma unroll
    for (int j = 0; j < ITERS; ++j) {
        if (partial_gain) store_columns(rx, partial_gain + (size_t)blockIdx.x * partial_stride, j, t, n, dgain[j]);
        if (partial_bias) store_columns(rx, partial_bias + (size_t)blockIdx.x * partial_stride, j, t, n, dbias[j]);
    }
}

// Rows longer than a workgroup's registers.  The columns' sums first (grad_x may overwrite grad_out):
// a workgroup takes kLongThreads columns of every gridDim.y-th row; then the rows' gradient in two passes.  Sums over
// rows and over a thread's columns are binary64, as in the forward pass.
template <typename T>
__global__ __launch_bounds__(kLongThreads) void layer_norm_columns_long_kernel(
    const T* grad_out, size_t grad_out_stride, const T* x, size_t x_stride, const float* mean, const float* rstd,
    float* partial_gain, float* partial_bias, size_t partial_stride, size_t rows, int n) {
    const int i = blockIdx.x * kLongThreads + threadIdx.x;
    if (i >= n) return;
    double dgain = 0.0, dbias = 0.0;
    for (size_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const float d = (float)grad_out[row * grad_out_stride + i];
        dgain += (double)d * (double)(((float)x[row * x_stride + i] - mean[row]) * rstd[row]);
        dbias += (double)d;
    }
    if (partial_gain) partial_gain[blockIdx.y * partial_stride + i] = (float)dgain;
    if (partial_bias) partial_bias[blockIdx.y * partial_stride + i] = (float)dbias;
}

template <typename T>
__global__ __launch_bounds__(kLongThreads) void layer_norm_grad_x_long_kernel(
    const T* grad_out, size_t grad_out_stride, const T* x, size_t x_stride, const float* mean_in, const float* rstd_in,
    const float* gain, T* grad_x, size_t grad_x_stride, int n, float inv_n) {
    constexpr int kWaves = kLongThreads / 64;
    __shared__ float slots[2 * kWaves];
    const int t = threadIdx.x;
    const size_t row = blockIdx.x;
    const T *xr = x + row * x_stride, *dr = grad_out + row * grad_out_stride;
    const float mean = mean_in[row], rstd = rstd_in[row];
    double sum_h = 0.0, sum_hx = 0.0;
    for (int i = t; i < n; i += kLongThreads) {
        const float h = (float)dr[i] * (gain ? gain[i] : 1.0f);
        sum_h += (double)h;
        sum_hx += (double)h * (double)(((float)xr[i] - mean) * rstd);
    }
    float sums[2] = {(float)sum_h, (float)sum_hx};
    row_reduce<Sum, kWaves>(sums, slots, t >> 6, t & 63);
    const float a = sums[0] * inv_n, b = sums[1] * inv_n;
    for (int i = t; i < n; i += kLongThreads) {  // grad_x may be grad_out or x: one thread owns an element
        const float h = (float)dr[i] * (gain ? gain[i] : 1.0f), xhat = ((float)xr[i] - mean) * rstd;
        grad_x[row * grad_x_stride + i] = (T)(rstd * (h - a - xhat * b));
    }
}

// out[i] = sum over the partial rows, of the gain (blockIdx.y 0) and of the bias (1); a workgroup adds
// 32 columns, 32 partial rows at a time with eight loads under way, and then the 32 sums in order, all in binary64.
constexpr int kJoinColumns = 32, kJoinRows = 32;
// Columns of one launch; wider rows go out as several, for at 1024 threads per 32 columns 2^27 columns would be the
// 2^32 threads that no launch may have.
constexpr int kMostJoinColumns = (int)kMostLaunchRows * kJoinColumns;
__global__ __launch_bounds__(kJoinColumns* kJoinRows) void layer_norm_join_kernel(
    const float* partial_gain, const float* partial_bias, size_t partial_stride, int partials, float* grad_gain,
    float* grad_bias, int n) {
    __shared__ double sums[kJoinRows][kJoinColumns];
    const float* p = blockIdx.y ? partial_bias : partial_gain;
    float* out = blockIdx.y ? grad_bias : grad_gain;
    if (!out) return;
    const int c = threadIdx.x % kJoinColumns, r = threadIdx.x / kJoinColumns, i = blockIdx.x * kJoinColumns + c;
    double a = 0.0;
    if (i < n) {
        int row = r;
        for (; row + 7 * kJoinRows < partials; row += 8 * kJoinRows) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = p[(row + k * kJoinRows) * partial_stride + i];
#pragma unroll
            for (int k = 0; k < 8; ++k) a += (double)v[k];
        }
        for (; row < partials; row += kJoinRows) a += (double)p[row * partial_stride + i];
    }
    sums[r][c] = a;
    __syncthreads();
    if (r == 0 && i < n) {
        for (int k = 1; k < kJoinRows; ++k) a += sums[k][c];
        out[i] = (float)a;
    }
}

// The shape of the backward kernel for rows of n elements: 64, 256, 512 or 1024 threads a row with at
// most 16 elements a thread (x, dy, gain and the two sums of an element are five registers), workgroups
// of 512 threads or one row; `threads` 0: the row is too long for registers.
struct BackwardShape {
    int threads, iters, slots;
};
BackwardShape backward_shape(int n, int vec) {
    const int vectors = (n + vec - 1) / vec, most = vec == 4 ? 4 : 2;
    if (vectors <= 64 * most) return {64, vectors <= 64 ? 1 : vectors <= 128 ? 2 : 4, 8};
    if (vectors <= 256 * most) return {256, vectors <= 256 ? 1 : vectors <= 512 ? 2 : 4, 2};
    if (vectors <= 512 * most) return {512, most, 1};
    if (vectors <= 1024 * most) return {1024, most, 1};
    return {0, 0, 1};
}
constexpr size_t kLongColumnRows = 64;  // partial rows where rows do not fit the registers

// Workgroups of the backward kernel, each of which writes a partial row: two of 512 threads a CU, and more where a thread
// would add more than 256 rows to its column's sum, whose error in binary32 grows with their number (8192 equal ones:
// 700 half steps).
constexpr size_t kMostRowsOfASum = 256;
size_t backward_groups(size_t rows, int n, int vec) {
    const BackwardShape s = backward_shape(n, vec);
    if (s.threads == 0) return rows < kLongColumnRows ? rows : kLongColumnRows;
    const size_t groups = (rows + s.slots - 1) / s.slots, resident = s.threads == 1024 ? 256 : 512;
    const size_t most = std::max(resident, (groups + kMostRowsOfASum - 1) / kMostRowsOfASum);
    return groups < most ? groups : most;
}

// Rows from which a wave or workgroup takes several (fewer are spread over the device).
constexpr size_t kManyRows = 4096;

template <typename T>
hipError_t forward(hipStream_t stream, const void* xv, size_t x_stride, const float* gain, const float* bias, void* yv,
                   size_t y_stride, float* mean, float* rstd, size_t rows, int n, float eps) {
    const T* x = static_cast<const T*>(xv);
    T* y = static_cast<T*>(yv);
    const float inv_n = 1.0f / (float)n;
    constexpr int vec = Elements<T>::kVec;
    const int vectors = (n + vec - 1) / vec;
#define MCC_NORM_AS(THREADS, ITERS, SLOTS, ROWS)                                                                   \
    hipLaunchKernelGGL((layer_norm_kernel<T, THREADS, ITERS, SLOTS, ROWS>),                                        \
                       dim3((unsigned)((rows + SLOTS * ROWS - 1) / (SLOTS * ROWS))), dim3(THREADS * SLOTS), 0, stream, \
                       x, x_stride, gain, bias, y, y_stride, mean, rstd, rows, n, inv_n, eps)
#define MCC_NORM(THREADS, ITERS, SLOTS, ROWS)                                          \
    do {                                                                               \
        if (rows < kManyRows) MCC_NORM_AS(THREADS, ITERS, SLOTS, 1);                   \
        else MCC_NORM_AS(THREADS, ITERS, SLOTS, ROWS);                                 \
    } while (0)
    // Gain and bias are 8 bytes an element from the caches, twice what a 16-bit row reads and writes: sharing them
    // pays there (16384 x 4096 bf16: 58 us alone, 53 us by two rows, 52 us by four; 8191 wide 145 us alone, 112 us by
    // two), and not for f32 (32768 x 4096: 178 us alone, 188 us by two).
    constexpr int kRows = vec == 8 ? 4 : 1, kRows4 = vec == 8 ? 2 : 1;
    // a row is a wave's up to 32 elements a thread, then a workgroup's of 256, then of 1024 threads
    if (vectors <= 64) MCC_NORM(64, 1, 4, kRows);
    else if (vectors <= 128) MCC_NORM(64, 2, 4, kRows);
    else if (vectors <= 256) MCC_NORM(64, 4, 4, kRows4);
    else if (vectors <= 512) MCC_NORM(256, 2, 1, kRows);
    else if (vectors <= 1024) MCC_NORM(256, 4, 1, kRows4);
    else if (vectors <= 2048) MCC_NORM(512, 4, 1, 1);
    else if (vectors <= 4096) MCC_NORM(1024, 4, 1, 1);
    else if (vectors <= 8192) MCC_NORM(1024, 8, 1, 1);
    else
        hipLaunchKernelGGL(layer_norm_long_kernel<T>, dim3((unsigned)rows), dim3(kLongThreads), 0, stream, x, x_stride,
                           gain, bias, y, y_stride, mean, rstd, n, inv_n, eps);
#undef MCC_NORM
#undef MCC_NORM_AS
    return hipGetLastError();
}

template <typename T>
hipError_t backward(hipStream_t stream, const void* dv, size_t d_stride, const void* xv, size_t x_stride,
                    const float* mean, const float* rstd, const float* gain, void* gv, size_t g_stride, float* grad_gain,
                    float* grad_bias, float* workspace, size_t rows, int n) {
    const T *d = static_cast<const T*>(dv), *x = static_cast<const T*>(xv);
    T* gx = static_cast<T*>(gv);
    const float inv_n = 1.0f / (float)n;
    constexpr int vec = Elements<T>::kVec;
    const BackwardShape shape = backward_shape(n, vec);
    const size_t groups = backward_groups(rows, n, vec);
    const bool join = groups > 1;  // one workgroup's sums are the result
    const size_t stride = join ? 2 * (size_t)n : 0;
    float* pg = !grad_gain ? nullptr : join ? workspace : grad_gain;
    float* pb = !grad_bias ? nullptr : join ? workspace + n : grad_bias;
#define MCC_NORM_BACKWARD(THREADS, ITERS, SLOTS)                                                                     \
    hipLaunchKernelGGL((layer_norm_backward_kernel<T, THREADS, ITERS, SLOTS>), dim3((unsigned)groups),               \
                       dim3(THREADS * SLOTS), 0, stream, d, d_stride, x, x_stride, mean, rstd, gain, gx, g_stride, pg, \
                       pb, stride, rows, n, inv_n)
    constexpr int most = vec == 4 ? 4 : 2;
    if (shape.threads == 64) {
        if (shape.iters == 1) MCC_NORM_BACKWARD(64, 1, 8);
        else if (shape.iters == 2) MCC_NORM_BACKWARD(64, 2, 8);
        else MCC_NORM_BACKWARD(64, most, 8);
    } else if (shape.threads == 256) {
        if (shape.iters == 1) MCC_NORM_BACKWARD(256, 1, 2);
        else if (shape.iters == 2) MCC_NORM_BACKWARD(256, 2, 2);
        else MCC_NORM_BACKWARD(256, most, 2);
    } else if (shape.threads == 512) {
        MCC_NORM_BACKWARD(512, most, 1);
    } else if (shape.threads == 1024) {
        MCC_NORM_BACKWARD(1024, most, 1);
    } else {
        if (pg || pb)
            hipLaunchKernelGGL(layer_norm_columns_long_kernel<T>,
                               dim3((unsigned)((n + kLongThreads - 1) / kLongThreads), (unsigned)groups),
                               dim3(kLongThreads), 0, stream, d, d_stride, x, x_stride, mean, rstd, pg, pb, stride, rows, n);
        for (size_t done = 0; gx && done < rows; done += kMostLaunchRows) {
            const size_t part = rows - done < kMostLaunchRows ? rows - done : kMostLaunchRows;
            hipLaunchKernelGGL(layer_norm_grad_x_long_kernel<T>, dim3((unsigned)part), dim3(kLongThreads), 0, stream,
                               d + done * d_stride, d_stride, x + done * x_stride, x_stride, mean + done, rstd + done, gain,
                               gx + done * g_stride, g_stride, n, inv_n);
        }
    }
#undef MCC_NORM_BACKWARD
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !join || (!pg && !pb)) return e;
    auto from = [](float* p, int column) { return p ? p + column : nullptr; };
    for (int done = 0; done < n; done += kMostJoinColumns) {
        const int part = n - done < kMostJoinColumns ? n - done : kMostJoinColumns;
        hipLaunchKernelGGL(layer_norm_join_kernel, dim3((unsigned)((part + kJoinColumns - 1) / kJoinColumns), 2),
                           dim3(kJoinColumns * kJoinRows), 0, stream, from(pg, done), from(pb, done), stride, (int)groups,
                           from(grad_gain, done), from(grad_bias, done), part);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_layer_norm(hipStream_t stream, ElementType type, const void* x, size_t x_stride, const float* gain,
                             const float* bias, void* y, size_t y_stride, float* mean, float* rstd, size_t rows, int n,
                             float eps) {
    hipError_t e = hipSuccess;
    for (size_t done = 0; done < rows && e == hipSuccess; done += kMostLaunchRows) {
        const size_t part = rows - done < kMostLaunchRows ? rows - done : kMostLaunchRows;
        const void* xp = static_cast<const char*>(x) + done * x_stride * element_size(type);
        void* yp = static_cast<char*>(y) + done * y_stride * element_size(type);
        float *m = mean ? mean + done : nullptr, *r = rstd ? rstd + done : nullptr;
        switch (type) {
            case ElementType::F32: e = forward<float>(stream, xp, x_stride, gain, bias, yp, y_stride, m, r, part, n, eps); break;
            case ElementType::F16: e = forward<_Float16>(stream, xp, x_stride, gain, bias, yp, y_stride, m, r, part, n, eps); break;
            case ElementType::BF16: e = forward<__bf16>(stream, xp, x_stride, gain, bias, yp, y_stride, m, r, part, n, eps); break;
        }
    }
    return e;
}

size_t layer_norm_backward_workspace_nbytes(ElementType type, size_t rows, int n) {
    const size_t groups = backward_groups(rows, n, type == ElementType::F32 ? 4 : 8);
    return groups > 1 ? groups * 2 * (size_t)n * sizeof(float) : 0;
}

hipError_t launch_layer_norm_backward(hipStream_t stream, ElementType type, const void* grad_out, size_t grad_out_stride,
                                      const void* x, size_t x_stride, const float* mean, const float* rstd,
                                      const float* gain, void* grad_x, size_t grad_x_stride, float* grad_gain,
                                      float* grad_bias, float* workspace, size_t rows, int n) {
    switch (type) {
        case ElementType::F32:
            return backward<float>(stream, grad_out, grad_out_stride, x, x_stride, mean, rstd, gain, grad_x, grad_x_stride,
                                   grad_gain, grad_bias, workspace, rows, n);
        case ElementType::F16:
            return backward<_Float16>(stream, grad_out, grad_out_stride, x, x_stride, mean, rstd, gain, grad_x,
                                      grad_x_stride, grad_gain, grad_bias, workspace, rows, n);
        case ElementType::BF16:
            return backward<__bf16>(stream, grad_out, grad_out_stride, x, x_stride, mean, rstd, gain, grad_x,
                                    grad_x_stride, grad_gain, grad_bias, workspace, rows, n);
    }
    return hipErrorInvalidValue;
}

}  // namespace mcc
