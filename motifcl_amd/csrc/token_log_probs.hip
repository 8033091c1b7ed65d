// Log probabilities of given tokens under softmax(logits / temperature), the entropy of that
// distribution, its `top` likeliest tokens, and the gradient of the logits.
//     log p_j = (z_j - m) / T - log s,  H = log s - log(2) u / s        (row_softmax.hpp)
//     dz_j = (g (delta_j,token - p_j) - h p_j (log p_j + H)) / T        for upstream gradients g of log p and h of H
// Bound by memory: the logits are read once, into registers, by one workgroup a row or, where rows are
// longer than it can hold, a stretch of a row; a second launch then joins the stretches.  The top entries are
// found in the registers: numbers below a bound that at least `top` numbers reach are passed over, and
// the few that are left are ranked.  Order: larger logit first, among equals the lower token, -0 = +0,
// NaN behind -inf; so equal calls give equal bytes whatever order the candidates were found in.
// Measured on 4096 x 32768 f32: 77 us = 7.0 TB/s without alternatives, 105 us with the top 64 (then bound by vector
// issue: 672 instructions a wave instead of 353); gradient of 8192 x 128000 bf16 712 us = 5.9 TB/s.
#include <hip/hip_runtime.h>

#include <cmath>

#include "launch.hpp"
#include "row_softmax.hpp"
#include "row_values.hpp"

namespace mcc {
namespace {

constexpr uint32_t kKeyLowest = 0x007fffffu;   // key of -inf
constexpr uint32_t kKeyHighest = 0xff800000u;  // key of +inf

// Unsigned integers in the order of the floats they stand for.
__device__ __forceinline__ uint32_t key_of(float z) {
    if (!(z == z)) return 0;
    const uint32_t b = __float_as_uint(z + 0.0f);  // -0 becomes +0
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
    if (k == 0) return __uint_as_float(0x7fc00000u);
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// A candidate: larger is likelier, and among equal logits the lower token is larger.
__device__ __forceinline__ uint64_t candidate(float z, uint32_t id) { return (uint64_t)key_of(z) << 32 | (uint32_t)~id; }

template <int WAVES>
struct TopScratch {
    static constexpr int kCandidates = WAVES == 1 ? 256 : 512;
    uint64_t list[kCandidates];
    int rank[kCandidates];
    uint32_t groups[WAVES == 1 ? 1 : 256], bound;
    int count;
    float totals[2][WAVES], least[WAVES];
};

// Sum over the workgroup of a count per wave; `turn` alternates between calls.
template <int WAVES>
__device__ __forceinline__ int total_of(int wave_count, float (&totals)[2][WAVES], int turn, int wave, int lane) {
    if (WAVES == 1) return wave_count;
    if (lane == 0) totals[turn][wave] = (float)wave_count;
    __syncthreads();
    return (int)wave_reduce<Sum>(lane < WAVES ? totals[turn][lane] : 0.0f);  // whole numbers below 2^24
}

// A number that at least `top` of the workgroup's numbers reach.  The threads' maxima are joined over groups
// of neighbouring lanes, and the first wave finds the top-th largest of the groups' maxima, each of which is a
// number of its own, by bisection over the leading 20 bits of its key: a compare and a population count a bit.
// Of random numbers about G ln(G / (G - top)) reach it, G groups: 256 from four waves on (75 for the top 64, 177 for
// the top 128), 128 of two waves, 64 of one (24 for the top 20, 89 for the top 48, 220 for the top 62).  Where top
// comes near G more numbers reach it than are listed, and beyond G it is -inf: those rows go to select_among_ties,
// ties or not.  That is one-wave rows (up to 2048 f32, 4096 16-bit numbers) from about the top 60 on and two-wave rows
// (16-bit, up to 8192) from about the top 126: 16384 x 3001 bf16 takes 45 us for the top 20, 79 for 48, 182 for 62 and
// 242 for 128, 16384 x 2000 f32 29, 64, 166 and 148, 16384 x 8000 bf16 74, 90, 107 and 762.
template <int WAVES>
__device__ __forceinline__ float lower_bound_of(float thread_max, int top, TopScratch<WAVES>& lds, int t, int wave, int lane) {
    constexpr int kLanes = WAVES > 4 ? WAVES / 4 : 1, kGroups = WAVES * 64 / kLanes, kHeld = kGroups / 64;
    static_assert(kLanes <= 4, "two steps join four lanes");
    if (kLanes >= 2) thread_max = dpp_join<Max, 0xB1, 0xf>(thread_max);  // quad_perm: lane ^ 1
    if (kLanes >= 4) thread_max = dpp_join<Max, 0x4E, 0xf>(thread_max);  // lane ^ 2
    uint32_t bound = 0;
    if (WAVES > 1) {
        if (lane % kLanes == 0) lds.groups[t / kLanes] = key_of(thread_max);
        __syncthreads();
    }
    if (wave == 0) {
        uint32_t held[kHeld];
#pragma unroll
        for (int i = 0; i < kHeld; ++i) held[i] = WAVES > 1 ? lds.groups[i * 64 + lane] : key_of(thread_max);
#pragma unroll
        for (int bit = 31; bit >= 12; --bit) {
            const uint32_t next = bound | 1u << bit;
            int reach = 0;
#pragma unroll
            for (int i = 0; i < kHeld; ++i) reach += __builtin_popcountll(__builtin_amdgcn_ballot_w64(held[i] >= next));
            if (reach >= top) bound = next;
        }
        if (WAVES > 1 && lane == 0) lds.bound = bound;
    }
    if (WAVES > 1) {
        __syncthreads();
        bound = lds.bound;
    }
    return bound <= kKeyLowest ? -__builtin_inff() : of_key(bound);
}

// The `top` candidates of a stretch into lds.list[0 .. top) when too many numbers reach the bound (ties, as of masked
// logits, or few groups) or too few (NaN): the top-th largest number, the numbers above it, and the
// first of those equal to it.  The smallest number that reaches the bound is tried first: in rows with
// fewer allowed tokens than `top` it is what the others were masked with (4096 x 32768 f32, 16 tokens allowed,
// top 64: 143 us against 107 us without masks; 330 us before it was tried first and NaN were looked for only
// where the sum says there are some).  Else the number is found by bisection over the bits of its key.
template <typename ROW, int WAVES, int ITERS>
__device__ __forceinline__ void select_among_ties(ROW& r, int n, uint32_t first_id, int top, float bound, bool no_nan,
                                                  TopScratch<WAVES>& lds, int t, int wave, int lane) {
    int turn = 0;
    auto count = [&](auto test) {
        int c = 0;
        r.convert_again();
#pragma unroll
        for (int j = 0; j < ITERS; ++j) {
            const int u = again(t);
#pragma unroll
            for (int k = 0; k < ROW::kVec; ++k)
                c += __builtin_popcountll(__builtin_amdgcn_ballot_w64(test((float)r.raw[j][k], j, k, u)));
        }
        turn ^= 1;
        return total_of<WAVES>(c, lds.totals, turn, wave, lane);
    };
    auto number = [&](float z, int j, int k, int u) { return z >= -__builtin_inff() && r.holds(j, k, u, n); };
    float f = 0.0f;
    int n_above = no_nan ? n : count(number);
    const bool numbers = n_above >= top;  // if not, all numbers are above and NaN are the ties
    if (numbers) {
        float least[1] = {__builtin_inff()};
        r.convert_again();
#pragma unroll
        for (int j = 0; j < ITERS; ++j)
#pragma unroll
            for (int k = 0; k < ROW::kVec; ++k) {
                const float z = (float)r.raw[j][k];
                least[0] = z >= bound && z < least[0] ? z : least[0];
            }
        least[0] = -wave_reduce<Max>(-least[0]);
        if (WAVES > 1) {
            if (lane == 0) lds.least[wave] = least[0];
            __syncthreads();
            least[0] = -wave_reduce<Max>(lane < WAVES ? -lds.least[lane] : -__builtin_inff());
        }
        f = least[0];
        n_above = count([&](float z, int, int, int) { return z > f; });
        if (n_above >= top) {
            uint32_t key = 0;
#pragma unroll 1
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t next = key | 1u << bit;
                if (next > kKeyHighest) continue;
                if (next > kKeyLowest) {  // at least `top` numbers reach -inf; above it the filled ones do not count
                    const float g = of_key(next);
                    if (count([&](float z, int, int, int) { return z >= g; }) < top) continue;
                }
                key = next;
            }
            f = of_key(key);
            n_above = count([&](float z, int, int, int) { return z > f; });
        }
    }
    auto above = [&](float z, int j, int k, int u) { return numbers ? z > f : number(z, j, k, u); };
    auto equal = [&](float z, int j, int k, int u) { return (numbers ? z == f : !(z == z)) && r.holds(j, k, u, n); };
    __syncthreads();
    if (t == 0) lds.count = 0;
    __syncthreads();
    if (n_above > 0) {
        r.convert_again();
#pragma unroll
        for (int j = 0; j < ITERS; ++j) {
            const int u = again(t);
#pragma unroll
            for (int k = 0; k < ROW::kVec; ++k) {
                const float z = (float)r.raw[j][k];
                if (above(z, j, k, u)) lds.list[atomicAdd(&lds.count, 1)] = candidate(z, first_id + r.index(j, k, u, n));
            }
        }
    }
    // ties in the order of their tokens: vector by vector, in it thread by thread, as many as are wanted
    int before = n_above;
    r.convert_again();
#pragma unroll
    for (int j = 0; j < ITERS; ++j) {
        if (before >= top) break;
        const int u = again(t);
        int of_wave = 0, lower = 0;
        const uint64_t below = ((uint64_t)1 << lane) - 1;
#pragma unroll
        for (int k = 0; k < ROW::kVec; ++k) {
            const uint64_t b = __builtin_amdgcn_ballot_w64(equal((float)r.raw[j][k], j, k, u));
            of_wave += __builtin_popcountll(b);
            lower += __builtin_popcountll(b & below);
        }
        turn ^= 1;
        const int all = total_of<WAVES>(of_wave, lds.totals, turn, wave, lane);
        int at = before + lower;
        for (int w = 0; w < wave; ++w) at += (int)lds.totals[turn][w];
#pragma unroll
        for (int k = 0; k < ROW::kVec; ++k) {
            const float z = (float)r.raw[j][k];
            if (equal(z, j, k, u)) {
                if (at < top) lds.list[at] = candidate(z, first_id + r.index(j, k, u, n));
                ++at;
            }
        }
        before += all;
    }
    __syncthreads();
}

// The candidates of a stretch, unordered, in lds.list; returns their number (at least `top`, at most
// kCandidates).  n >= top.
template <typename ROW, int WAVES, int ITERS>
__device__ __forceinline__ int find_candidates(ROW& r, int n, uint32_t first_id, int top, float thread_max, bool no_nan,
                                               TopScratch<WAVES>& lds, int t, int wave, int lane) {
    const float bound = lower_bound_of<WAVES>(thread_max, top, lds, t, wave, lane);
    // an address the compiler cannot see to be one for all lanes: it would add the lanes' ones up first, which costs
    // more than the one or two lanes that come here together
    const int none = again(0);
    auto push = [&](float z, int j, int k) {
        const int at = atomicAdd(&lds.count + none, 1);
        if (at < lds.kCandidates) lds.list[at] = candidate(z, first_id + r.index(j, k, again(t), n));
    };
    if (bound > -__builtin_inff()) {  // filled elements do not reach it
        if (thread_max >= bound) {
#pragma unroll
            for (int j = 0; j < ITERS; ++j)
#pragma unroll
                for (int k = 0; k < ROW::kVec; ++k) {
                    const float z = (float)r.raw[j][k];
                    if (z >= bound) push(z, j, k);
                }
        }
    } else if (n <= lds.kCandidates) {
#pragma unroll
        for (int j = 0; j < ITERS; ++j) {
            const int u = again(t);
#pragma unroll
            for (int k = 0; k < ROW::kVec; ++k) {
                const float z = (float)r.raw[j][k];
                if (z >= bound && r.holds(j, k, u, n)) push(z, j, k);
            }
        }
    }
    __syncthreads();
    const int found = lds.count;
    if (found >= top && found <= lds.kCandidates) return found;
    select_among_ties<ROW, WAVES, ITERS>(r, n, first_id, top, bound, no_nan, lds, t, wave, lane);
    return top;
}

// rank[i] += how many of the n candidates are likelier than list[i] (0 before).  All the workgroup's threads
// count: the list is read in parts, one by each group of a power of two of threads that holds the candidates.
template <int THREADS>
__device__ __forceinline__ void rank_candidates(const uint64_t* list, int n, int* rank, int t) {
    int bits = 32 - __builtin_clz(n > 1 ? n - 1 : 1);
    if ((1 << bits) > THREADS) bits = 31 - __builtin_clz(THREADS);
    const int held = 1 << bits, parts = THREADS >> bits, width = (n + parts - 1) / parts;
    const int from = (t >> bits) * width, to = from + width < n ? from + width : n;
    for (int i = t & (held - 1); i < n; i += held) {
        const uint64_t mine = list[i];
        int above = 0;
        for (int k = from; k < to; ++k) above += list[k] > mine ? 1 : 0;
        if (above) atomicAdd(&rank[i], above);
    }
    __syncthreads();
}

// What is left of a row's statistics once they are joined.
struct RowResult {
    float m, log_s, inv_temperature;
    bool empty;  // -inf alone
    __device__ __forceinline__ float log_prob(float z) const {
        return empty && z == z ? -__builtin_inff() : (z - m) * inv_temperature - log_s;
    }
};
__device__ __forceinline__ RowResult finish_row(const TokenLogProbs& a, size_t row, const SoftmaxStats& st, float token_logit,
                                                bool has_token, bool writes) {
    RowResult r;
    r.m = st.m;
    r.empty = st.s == 0.0f;
    r.log_s = logf(st.s);
    r.inv_temperature = a.inv_temperature;
    if (writes) {
        if (a.lse) a.lse[row] = r.empty ? -__builtin_inff() : st.m * a.inv_temperature + r.log_s;
        if (a.entropy) a.entropy[row] = r.empty ? 0.0f : r.log_s - kLn2 * (st.u / st.s);
        if (a.log_prob) a.log_prob[row] = has_token ? r.log_prob(token_logit) : 0.0f;
    }
    return r;
}

template <typename T>
__device__ __forceinline__ bool token_of(const TokenLogProbs& a, size_t row, float& z) {
    if (!a.tokens || !a.log_prob) return false;
    const int32_t token = a.tokens[row];
    if (token < 0 || token >= a.vocab) return false;  // an ignored position
    z = (float)static_cast<const T*>(a.logits)[row * a.stride + token];
    return true;
}

// One stretch a workgroup.  ONE: the row is one stretch, and the results are written; else `stats` and
// `best` [rows * segments][top] are.
template <typename T, int THREADS, int ITERS, bool TOP, bool ONE>
__global__ __launch_bounds__(THREADS, 8) void token_log_probs_kernel(TokenLogProbs a, int segments, int length,
                                                                  SoftmaxStats* stats, uint64_t* best) {
    constexpr int kWaves = THREADS / 64;
    typedef RowVectors<T, THREADS, ITERS> Row;
    __shared__ float slots[3 * kWaves];
    __shared__ TopScratch<TOP ? kWaves : 1> lds;
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    // between this and its use lies a barrier of the statistics, or there is one wave, whose LDS accesses keep their order
    if constexpr (TOP) {
        if (t == 0) lds.count = 0;
        for (int i = t; i < lds.kCandidates; i += THREADS) lds.rank[i] = 0;
    }
    const size_t row = ONE ? blockIdx.x : blockIdx.x / (unsigned)segments;
    const int segment = ONE ? 0 : (int)(blockIdx.x % (unsigned)segments);
    const int from = segment * length, n = a.vocab - from < length ? a.vocab - from : length;
    Row r;
    r.load(static_cast<const T*>(a.logits) + row * a.stride + from, t, n);
    float token_logit = 0.0f;
    const bool has_token = ONE && t == 0 && token_of<T>(a, row, token_logit);
    r.fill_tail(t, n, (T)-__builtin_inff());
    float thread_max;
    const SoftmaxStats st = stats_of<Row, kWaves, ITERS>(r, a.log2_scale, slots, wave, lane, thread_max);
    RowResult result{};
    if (ONE)
        result = finish_row(a, row, st, token_logit, has_token, t == 0);
    else if (t == 0)
        stats[row * segments + segment] = st;
    if constexpr (TOP) {
        const int top = a.top < n ? a.top : n;
        const int found = find_candidates<Row, kWaves, ITERS>(r, n, (uint32_t)from, top, thread_max, st.s == st.s, lds, t,
                                                                     wave, lane);
        rank_candidates<THREADS>(lds.list, found, lds.rank, t);
        for (int i = t; i < found; i += THREADS) {
            const uint64_t mine = lds.list[i];
            const int rank = lds.rank[i];
            if (rank >= top) continue;
            if (ONE) {
                if (a.top_ids) a.top_ids[row * a.top + rank] = (int32_t)~(uint32_t)mine;
                if (a.top_log_probs) a.top_log_probs[row * a.top + rank] = result.log_prob(of_key((uint32_t)(mine >> 32)));
            } else {
                best[(row * segments + segment) * a.top + rank] = mine;
            }
        }
        if (!ONE)
            for (int i = top + t; i < a.top; i += THREADS) best[(row * segments + segment) * a.top + i] = 0;
    }
}

// Joins a row's stretches.  The entries that reach the smallest of the stretches' ceil(top / segments)-th
// ones (at least `top` do) are ranked; where they are too many, as when one stretch holds most of the
// likely tokens, the top-th largest is found by bisection first.
constexpr int kJoinThreads = 256, kJoinCandidates = 1024;
template <typename T>
__global__ __launch_bounds__(kJoinThreads) void token_log_probs_join_kernel(TokenLogProbs a, int segments,
                                                                           const SoftmaxStats* stats,
                                                                           const uint64_t* best) {
    constexpr int kWaves = kJoinThreads / 64;
    __shared__ uint64_t list[kJoinCandidates];
    __shared__ int ranks[kJoinCandidates], count;
    __shared__ float totals[2][kWaves];
    __shared__ uint64_t bounds[kWaves];
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const size_t row = blockIdx.x;
    float token_logit = 0.0f;
    const bool has_token = t == 0 && token_of<T>(a, row, token_logit);
    JoinedStats joined(stats[row * segments]);
    for (int i = 1; i < segments; ++i) joined.join(stats[row * segments + i], a.log2_scale);
    const RowResult result = finish_row(a, row, joined.stats(), token_logit, has_token, t == 0);
    if (a.top == 0 || (!a.top_ids && !a.top_log_probs)) return;
    const uint64_t* entries = best + row * segments * a.top;
    const int all = segments * a.top, nth = (a.top + segments - 1) / segments;
    uint64_t bound = ~(uint64_t)0;
    for (int i = t; i < segments; i += kJoinThreads) {
        const uint64_t e = entries[i * a.top + nth - 1];
        bound = e < bound ? e : bound;
    }
    for (int s = 32; s >= 1; s >>= 1) {
        const uint64_t e = __shfl_xor(bound, s);
        bound = e < bound ? e : bound;
    }
    if (lane == 0) bounds[wave] = bound;
    if (t == 0) count = 0;
    for (int i = t; i < kJoinCandidates; i += kJoinThreads) ranks[i] = 0;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) bound = bounds[w] < bound ? bounds[w] : bound;
    auto gather = [&](uint64_t from) {
        for (int i = t; i < all; i += kJoinThreads) {
            const uint64_t e = entries[i];
            if (e >= from && e != 0) {  // 0: a stretch shorter than `top` has no such entry
                const int at = atomicAdd(&count, 1);
                if (at < kJoinCandidates) list[at] = e;
            }
        }
        __syncthreads();
    };
    gather(bound);
    int found = count;
    if (found > kJoinCandidates) {
        uint64_t kth = 0;
        int turn = 0;
        for (int bit = 63; bit >= 0; --bit) {
            const uint64_t next = kth | (uint64_t)1 << bit;
            int c = 0;
            for (int i = t; i < (all + 63) / 64 * 64; i += kJoinThreads)
                c += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < all && entries[i] >= next));
            turn ^= 1;
            if (total_of<kWaves>(c, totals, turn, wave, lane) >= a.top) kth = next;
        }
        __syncthreads();
        if (t == 0) count = 0;
        __syncthreads();
        gather(kth);
        found = count;
    }
    rank_candidates<kJoinThreads>(list, found, ranks, t);
    for (int i = t; i < found; i += kJoinThreads) {
        const uint64_t mine = list[i];
        const int rank = ranks[i];
        if (rank >= a.top) continue;
        if (a.top_ids) a.top_ids[row * a.top + rank] = (int32_t)~(uint32_t)mine;
        if (a.top_log_probs) a.top_log_probs[row * a.top + rank] = result.log_prob(of_key((uint32_t)(mine >> 32)));
    }
}

// ---- backward -----------------------------------------------------------------------------------
// A stream of logits in and gradients out; the row's numbers are known beforehand.  grad_logits may be
// logits (one thread owns an element).
constexpr int kGradThreads = 256, kGradPerThread = 16, kGradLength = kGradThreads * kGradPerThread;
template <typename T, bool ENTROPY>
__global__ __launch_bounds__(kGradThreads) void token_log_probs_backward_kernel(
    const T* logits, size_t stride, const int32_t* tokens, const float* lse, const float* entropy,
    const float* grad_log_prob, const float* grad_entropy, T* grad_logits, size_t grad_stride, int segments, int vocab,
    float inv_temperature) {
    constexpr int kIters = kGradPerThread / Elements<T>::kVec;
    typedef RowVectors<T, kGradThreads, kIters, true> Row;
    const int t = threadIdx.x;
    const size_t row = blockIdx.x / (unsigned)segments;
    const int segment = (int)(blockIdx.x % (unsigned)segments);
    // the row is cut at whole lines: the first stretch is shorter by what the row begins behind one
    const T* begin = logits + row * stride;
    const int behind = (int)((reinterpret_cast<uintptr_t>(begin) & (kLineBytes - 1)) / sizeof(T));
    const int from = segment ? segment * kGradLength - behind : 0;
    const int to = vocab - from < kGradLength - (segment ? 0 : behind) ? vocab : (segment + 1) * kGradLength - behind;
    const int n = to - from;
    if (n <= 0) return;
    Row r;
    r.load(begin + from, t, n, segment ? 0 : behind);
    const int32_t token = tokens ? tokens[row] : -1;
    const float l = lse[row], big_h = ENTROPY ? entropy[row] : 0.0f;
    const float g = grad_log_prob && token >= 0 && token < vocab ? grad_log_prob[row] : 0.0f;
    const float h = ENTROPY ? grad_entropy[row] : 0.0f;
    // nothing upstream, or a row of -inf alone: zeros, whatever the logits hold
    const bool zero = (g == 0.0f && h == 0.0f) || l == -__builtin_inff();
    const float gt = g * inv_temperature, ht = h * inv_temperature;
    const bool here = token >= from && token - from < n;  // the same for the whole workgroup
#pragma unroll
    for (int j = 0; j < kIters; ++j) {
        float v[Row::kVec];
#pragma unroll
        for (int k = 0; k < Row::kVec; ++k) {
            const float log_p = fmaf((float)r.raw[j][k], inv_temperature, -l), p = exp2_of(log_p * kLog2E);
            v[k] = -gt * p;
            if (ENTROPY) v[k] -= ht * (p * (fmaxf(log_p, -1e4f) + big_h));  // p is 0 long before the bound
        }
        if (here) {
#pragma unroll
            for (int k = 0; k < Row::kVec; ++k)
                if (from + r.index(j, k, t, n) == token) v[k] += gt;
        }
        if (zero) {
#pragma unroll
            for (int k = 0; k < Row::kVec; ++k) v[k] = 0.0f;
        }
        r.store(grad_logits + row * grad_stride + from, j, t, n, v);
    }
}

// Rows of one launch with `segments` workgroups a row.
size_t launch_rows(int segments) {
    const size_t rows = kMostLaunchRows / (size_t)segments;
    return rows > 0 ? rows : 1;
}

// Workspace of a row cut into stretches: their statistics, then their entries.
size_t stats_nbytes(size_t rows, const RowCut& c) { return (rows * c.segments * sizeof(SoftmaxStats) + 15) / 16 * 16; }

template <typename T, bool TOP>
hipError_t launch_whole(hipStream_t stream, const TokenLogProbs& a, const RowCut& c) {
    for_shape<T>(c, [&](auto threads, auto iters) {
        constexpr int THREADS = decltype(threads)::value, ITERS = decltype(iters)::value;
        hipLaunchKernelGGL((token_log_probs_kernel<T, THREADS, ITERS, TOP, true>), dim3((unsigned)a.rows), dim3(THREADS), 0,
                           stream, a, 1, c.length, (SoftmaxStats*)nullptr, (uint64_t*)nullptr);
    });
    return hipGetLastError();
}

template <typename T, bool TOP>
hipError_t launch_stretches(hipStream_t stream, const TokenLogProbs& a, const RowCut& c, SoftmaxStats* stats, uint64_t* best) {
    hipLaunchKernelGGL((token_log_probs_kernel<T, 1024, 8, TOP, false>), dim3((unsigned)(a.rows * c.segments)), dim3(1024),
                       0, stream, a, c.segments, c.length, stats, best);
    return hipGetLastError();
}

template <typename T>
hipError_t forward(hipStream_t stream, const TokenLogProbs& a, void* workspace) {
    const RowCut c = cut_rows(a.vocab, Elements<T>::kVec);
    const bool top = a.top > 0 && (a.top_ids || a.top_log_probs);
    if (c.segments == 1) return top ? launch_whole<T, true>(stream, a, c) : launch_whole<T, false>(stream, a, c);
    SoftmaxStats* stats = static_cast<SoftmaxStats*>(workspace);
    uint64_t* best = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + stats_nbytes(a.rows, c));
    const hipError_t e = top ? launch_stretches<T, true>(stream, a, c, stats, best)
                             : launch_stretches<T, false>(stream, a, c, stats, best);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(token_log_probs_join_kernel<T>, dim3((unsigned)a.rows), dim3(kJoinThreads), 0, stream, a, c.segments,
                       stats, best);
    return hipGetLastError();
}

template <typename T>
hipError_t backward(hipStream_t stream, const void* logits, size_t stride, const int32_t* tokens, const float* lse,
                    const float* entropy, const float* grad_log_prob, const float* grad_entropy, void* grad_logits,
                    size_t grad_stride, size_t rows, int vocab, float inv_temperature) {
    // one more line for rows that do not begin on one
    const bool aligned = whole_lines(logits) && (rows == 1 || stride * sizeof(T) % kLineBytes == 0);
    const size_t reach = (size_t)vocab + (aligned ? 0 : kLineBytes / sizeof(T) - 1);
    const int segments = (int)((reach + kGradLength - 1) / kGradLength);
    const dim3 grid((unsigned)(rows * segments)), block(kGradThreads);
    if (grad_entropy)
        hipLaunchKernelGGL((token_log_probs_backward_kernel<T, true>), grid, block, 0, stream, static_cast<const T*>(logits),
                           stride, tokens, lse, entropy, grad_log_prob, grad_entropy, static_cast<T*>(grad_logits),
                           grad_stride, segments, vocab, inv_temperature);
    else
        hipLaunchKernelGGL((token_log_probs_backward_kernel<T, false>), grid, block, 0, stream,
                           static_cast<const T*>(logits), stride, tokens, lse, entropy, grad_log_prob, grad_entropy,
                           static_cast<T*>(grad_logits), grad_stride, segments, vocab, inv_temperature);
    return hipGetLastError();
}

}  // namespace

size_t token_log_probs_workspace_nbytes(ElementType type, size_t rows, int vocab, int top) {
    const RowCut c = cut_rows(vocab, type == ElementType::F32 ? 4 : 8);
    if (c.segments == 1) return 0;
    const size_t part = launch_rows(c.segments) < rows ? launch_rows(c.segments) : rows;  // reused by the next
    return stats_nbytes(part, c) + part * c.segments * (size_t)top * sizeof(uint64_t);
}

hipError_t launch_token_log_probs(hipStream_t stream, ElementType type, const TokenLogProbs& a, void* workspace) {
    const size_t most = launch_rows(cut_rows(a.vocab, type == ElementType::F32 ? 4 : 8).segments);
    hipError_t e = hipSuccess;
    for (size_t done = 0; done < a.rows && e == hipSuccess; done += most) {
        TokenLogProbs p = a;
        p.rows = a.rows - done < most ? a.rows - done : most;
        p.logits = static_cast<const char*>(a.logits) + done * a.stride * element_size(type);
        if (a.tokens) p.tokens = a.tokens + done;
        if (a.log_prob) p.log_prob = a.log_prob + done;
        if (a.entropy) p.entropy = a.entropy + done;
        if (a.lse) p.lse = a.lse + done;
        if (a.top_ids) p.top_ids = a.top_ids + done * a.top;
        if (a.top_log_probs) p.top_log_probs = a.top_log_probs + done * a.top;
        switch (type) {
            case ElementType::F32: e = forward<float>(stream, p, workspace); break;
            case ElementType::F16: e = forward<_Float16>(stream, p, workspace); break;
            case ElementType::BF16: e = forward<__bf16>(stream, p, workspace); break;
        }
    }
    return e;
}

hipError_t launch_token_log_probs_backward(hipStream_t stream, ElementType type, const void* logits, size_t stride,
                                           const int32_t* tokens, const float* lse, const float* entropy,
                                           const float* grad_log_prob, const float* grad_entropy, void* grad_logits,
                                           size_t grad_stride, size_t rows, int vocab, float inv_temperature) {
    const size_t most = launch_rows(vocab / kGradLength + 2), size = element_size(type);
    hipError_t e = hipSuccess;
    for (size_t done = 0; done < rows && e == hipSuccess; done += most) {
        const size_t part = rows - done < most ? rows - done : most;
        const void* z = static_cast<const char*>(logits) + done * stride * size;
        void* g = static_cast<char*>(grad_logits) + done * grad_stride * size;
        auto at = [&](auto* p) { return p ? p + done : nullptr; };
        switch (type) {
            case ElementType::F32:
                e = backward<float>(stream, z, stride, at(tokens), at(lse), at(entropy), at(grad_log_prob), at(grad_entropy), g,
                                    grad_stride, part, vocab, inv_temperature);
                break;
            case ElementType::F16:
                e = backward<_Float16>(stream, z, stride, at(tokens), at(lse), at(entropy), at(grad_log_prob),
                                       at(grad_entropy), g, grad_stride, part, vocab, inv_temperature);
                break;
            case ElementType::BF16:
                e = backward<__bf16>(stream, z, stride, at(tokens), at(lse), at(entropy), at(grad_log_prob),
                                     at(grad_entropy), g, grad_stride, part, vocab, inv_temperature);
                break;
        }
    }
    return e;
}

}  // namespace mcc
