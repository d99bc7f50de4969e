// Sampling for gfx950: temperature, top-k, top-p and min-p over a row of logits, and the token
// that a given random number picks from what they keep.
//
// A token's weight is w = 2^((x - max) log2(e) / T), computed in f64 and rounded once to a whole
// number of 2^-F units (F = 44, or less for a vocabulary above 2^18, so that a row's sum fits 62
// bits). Sums of whole numbers do not depend on their order: histograms may be filled by atomics,
// and the choice is the same on every run. Ranks go by the logit's bits made monotonic (equal logits by index): a
// token's rank key is those bits over the complement of its index.
//
// What top-k and top-p keep is the tokens down to a cut in that order. A sort would find it; here
// a histogram does. Over slices of 4096 tokens, so that one row fills many CUs:
//  1. max: the slice's largest rank key;
//  2. histogram: tokens by their distance below the largest logit, in steps of 1/32 (of the
//     temperature where it is above 1), with each step's count and weight;
//  3. collect: every slice finds from the histogram the steps that can hold the cut, lists its
//     tokens of those steps, and sums the kept weights of the steps above them;
//  4. choose: one workgroup per row sorts the listed tokens, walks them to the exact cut, adds
//     what is kept of them to their slices' sums, and finds the token in its slice. Up to 512
//     listed tokens (a language model's logits list a few, up to some hundred where the cut lies
//     in the wide floor) are ranked by counting, a token per thread.
// Steps 2 and 3 do nothing for rows that need only the best token. A row whose steps list more
// than kListed tokens (many equal logits; logits of enormous range; a mask that leaves fewer tokens
// above -inf than top-k asks for) is solved by the choosing workgroup alone, by radix selection over
// the row: 10 live tokens of 151936, top-k 50, 0.67 ms, and 1.2 with top-p 0.9 (23 us at top-k 5).
//
// Bound by four dependent launches. One row of 151936 (top-k 50, top-p 0.9): 2.9, 5.1, 6.2 and 7.5
// us under a profiler, 22.3 in all; 64 rows of 32768: 4.5, 7.5, 11.2 and 12.2, 36 in all (8.4 MB, 1.6
// us of a large copy). With a row to one workgroup they took 444 and 184.
#include "eb_common.h"
#include "eb_internal.h"

#include <algorithm>
#include <cstdint>

namespace {

typedef unsigned long long u64;
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 512;   // of the choosing workgroup
constexpr int kWaves = kThreads / 64;
constexpr int kTile = 4096;     // tokens of a slice (of 2048: one row of 151936 22.0 -> 21.0 us, 64 rows 62.5 -> 93)
constexpr int kSliceThreads = 512;
constexpr int kPer = kTile / kSliceThreads;  // tokens per thread of a slice
constexpr int kDigits = 256;    // of a radix pass
constexpr int kBins = 1024;     // steps of the histogram
constexpr float kBinsPerUnit = 32.0f;
constexpr int kListed = 4096;   // most listed tokens of a row

// Per row, written by step 3.
struct Cut {
    u64 before_cut;   // weight of the steps above the first that can hold the cut
    u64 before_topk;  // and above the one that holds top-k's last token
    unsigned above;   // tokens above that one
    int topk_bin;     // that one (kBins: no top-k)
};

struct Args {
    eb::SampleArgs s;
    int frac;  // F
    int tiles;
    int per, groups;  // slices of a workgroup, workgroups of a row
    // workspace
    u64 *best;         // [rows, groups] rank keys
    u64 *tile_sum;     // [rows, tiles]
    u64 *hist_w;       // [rows, kBins]
    unsigned *hist_c;  // [rows, kBins]
    u64 *listed;       // [rows, kListed]
    unsigned *count;   // [rows]
    Cut *cut;          // [rows]
};

// The logit's bits in an order that follows its value; 0 for NaN. -0 counts as +0.
__device__ __forceinline__ unsigned key_of(float x) {
    if (x != x) return 0;
    unsigned u = __builtin_bit_cast(unsigned, x);
    if ((u & 0x7FFFFFFFu) == 0) u = 0;
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned key) {
    return __builtin_bit_cast(float, (key & 0x80000000u) ? key & 0x7FFFFFFFu : ~key);
}
__device__ __forceinline__ u64 rank_of(float x, unsigned i) { return (u64)key_of(x) << 32 | (u64)(unsigned)~i; }
__device__ __forceinline__ unsigned index_of(u64 rank) { return ~(unsigned)rank; }
constexpr u64 kLeastRank = 1ull << 32;  // at most every rank but NaN's

// 2^(y + F) for y <= 0 and whole F (0 from y = -900 on): y = n + f, |f| <= 1/2, the Taylor sum of
// e^(f ln 2) (the first term left out is below 2e-16), and n + F added to its exponent. Adding
// 1.5 * 2^52 leaves n in the low bits of the sum.
constexpr double kLn2 = 0.693147180559945309417232121458;
constexpr double term(int k) { return k == 0 ? 1.0 : term(k - 1) * kLn2 / k; }
template <int K>
__device__ __forceinline__ double horner(double p, double f) {
    constexpr double c = term(K);
    p = __builtin_fma(p, f, c);
    if constexpr (K > 0) return horner<K - 1>(p, f);
    return p;
}
__device__ __forceinline__ double exp2_scaled(double y, int frac) {
    y = fmax(y, -900.0);
    const double t = y + 6755399441055744.0;
    const double f = y - (t - 6755399441055744.0);
    constexpr double last = term(12);
    const double p = horner<11>(last, f);
    const u64 bits = __builtin_bit_cast(u64, p) + ((u64)((unsigned)__builtin_bit_cast(u64, t) + (unsigned)frac) << 52);
    return __builtin_bit_cast(double, bits);
}

// A row's parameters as given (loaded with a kernel's other first loads).
struct Params {
    float temperature, top_p, min_p;
    unsigned top_k;
    __device__ __forceinline__ Params(const Args &a, size_t r) {
        temperature = a.s.temperature ? a.s.temperature[r] : 1.0f;
        min_p = a.s.min_p ? a.s.min_p[r] : 0.0f;
        top_p = a.s.top_p ? a.s.top_p[r] : 1.0f;
        top_k = a.s.top_k ? a.s.top_k[r] : 0u;
    }
};

// And as used.
struct Row {
    double rate;    // log2(e) / T
    double one;     // 2^F
    double min_p;   // in the same units; 0: off
    float top;      // the largest logit
    float per_bin;  // steps per unit of distance
    float top_p;
    unsigned top_k;
    bool none, best, use_k, use_p;  // no candidate; only the best token; which cuts
    int frac;

    __device__ __forceinline__ Row(const Args &a, const Params &p, unsigned best_key) {
        const float temp = p.temperature, mp = p.min_p;
        top_p = p.top_p;
        top_k = p.top_k;
        none = best_key <= key_of(-INFINITY);  // (only -inf and NaN)
        best = !(temp > 0.0f) || mp > 1.0f || top_k == 1 || top_p <= 0.0f;
        use_k = top_k > 0 && top_k < (unsigned)a.s.vocab;
        use_p = top_p < 1.0f;
        rate = 1.4426950408889634073599 / (double)temp;
        frac = a.frac;
        one = ldexp(1.0, frac);
        min_p = mp > 0.0f ? (double)mp * one : 0.0;
        top = value_of(best_key);
        per_bin = kBinsPerUnit / fmaxf(temp, 1.0f);
    }
    // w in units of 2^-F, before its rounding.
    __device__ __forceinline__ double weight(float x) const {
        const double w = exp2_scaled(((double)x - (double)top) * rate, frac);
        // (top is finite or +inf; -inf has no weight, also where T is infinite)
        return x == top ? one : x == -INFINITY ? 0.0 : w;
    }
    // Rounded: below 2^51, adding 2^52 leaves the whole number in the sum's low bits.
    __device__ __forceinline__ u64 units(double w) const {
        return __builtin_bit_cast(u64, w + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
    }
    __device__ __forceinline__ u64 units_kept(double w) const { return w >= min_p ? units(w) : 0; }
    // The step a logit falls in; it rises as the logit falls.
    __device__ __forceinline__ int bin(float x) const {
        if (x == top) return 0;
        return (int)fminf((top - x) * per_bin, (float)(kBins - 1));
    }
};

// ---- workgroup reductions ---------------------------------------------------------------------

template <class T>
__device__ __forceinline__ T wave_total(T x) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) x += __shfl_xor(x, m);
    return x;
}
__device__ __forceinline__ u64 wave_best(u64 k) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) {
        const u64 o = __shfl_xor(k, m);
        k = o > k ? o : k;
    }
    return k;
}
// (each starts with a barrier, so that s_waves may be in use before)
template <int THREADS, class T>
__device__ __forceinline__ T block_total(T x, T *s_waves) {
    x = wave_total(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_waves[threadIdx.x >> 6] = x;
    __syncthreads();
    T t = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) t += s_waves[w];
    return t;
}
template <int THREADS>
__device__ __forceinline__ u64 block_best(u64 k, u64 *s_waves) {
    k = wave_best(k);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_waves[threadIdx.x >> 6] = k;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) k = s_waves[w] > k ? s_waves[w] : k;
    return k;
}
// Inclusive sums over the threads.
template <int THREADS, class T>
__device__ __forceinline__ T block_scan(T x, T *s_waves) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const T o = __shfl_up(x, d);
        if (lane >= d) x += o;
    }
    __syncthreads();
    if (lane == 63) s_waves[wave] = x;
    __syncthreads();
    for (int w = 0; w < wave; ++w) x += s_waves[w];
    return x;
}

// Two at once.
template <int THREADS>
__device__ __forceinline__ void block_scan2(unsigned &x, u64 &y, unsigned *s_x, u64 *s_y) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const unsigned o = __shfl_up(x, d);
        const u64 q = __shfl_up(y, d);
        if (lane >= d) {
            x += o;
            y += q;
        }
    }
    __syncthreads();
    if (lane == 63) {
        s_x[wave] = x;
        s_y[wave] = y;
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
        x += s_x[w];
        y += s_y[w];
    }
}
__device__ __forceinline__ u64 wave_scan(u64 x) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const u64 o = __shfl_up(x, d);
        if (lane >= d) x += o;
    }
    return x;
}

// ---- steps 1 to 3: one workgroup per run of slices -----------------------------------------------------

// The tokens of this thread in slice t: four at a time, NaN past the vocabulary.
struct Slice {
    float x[kPer];
    int base;
    __device__ __forceinline__ int at(int j) const { return base + j / 4 * kSliceThreads * 4 + j % 4; }
    __device__ __forceinline__ Slice(const float *row, int n, int t) {
        base = t * kTile + 4 * (int)threadIdx.x;
        if ((n & 3) == 0 && (reinterpret_cast<uintptr_t>(row) & 15) == 0) {
#pragma unroll
            for (int j = 0; j < kPer; j += 4) {
                const f32x4 nan = {__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
                const f32x4 v = at(j) < n ? *reinterpret_cast<const f32x4 *>(row + at(j)) : nan;
#pragma unroll
                for (int c = 0; c < 4; ++c) x[j + c] = v[c];
            }
        } else {
#pragma unroll
            for (int j = 0; j < kPer; ++j) x[j] = at(j) < n ? row[at(j)] : __builtin_nanf("");
        }
    }
};

// Step 1, and the clearing of the row's histogram and list.
__global__ __launch_bounds__(kSliceThreads) void sample_max_kernel(Args a) {
    __shared__ u64 s_waves[kSliceThreads / 64];
    const int g = blockIdx.x, tid = threadIdx.x;
    const size_t r = blockIdx.y;
    const float *row = a.s.logits + r * a.s.vocab;
    const int t0 = g * a.per, t1 = min(t0 + a.per, a.tiles);
    Slice s(row, (int)a.s.vocab, t0);
    for (int i = g * kSliceThreads + tid; i < kBins; i += a.groups * kSliceThreads) {
        a.hist_w[r * kBins + i] = 0;
        a.hist_c[r * kBins + i] = 0;
    }
    if (g == 0 && tid == 0) a.count[r] = 0;
    u64 k = 0;
    for (int t = t0;;) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const u64 o = rank_of(s.x[j], (unsigned)s.at(j));
            k = o > k ? o : k;
        }
        if (++t >= t1) break;
        s = Slice(row, (int)a.s.vocab, t);
    }
    k = block_best<kSliceThreads>(k, s_waves);
    if (tid == 0) a.best[r * a.groups + g] = k;
}

// The row's largest rank key, from step 1's (every wave by itself: no barrier).
__device__ __forceinline__ u64 row_best(const Args &a, size_t r) {
    u64 k = 0;
    for (int i = threadIdx.x & 63; i < a.groups; i += 64) {
        const u64 o = a.best[r * a.groups + i];
        k = o > k ? o : k;
    }
    return wave_best(k);
}

// Step 2: a histogram in LDS, its filled steps added to the row's.
__global__ __launch_bounds__(kSliceThreads) void sample_histogram_kernel(Args a) {
    __shared__ u64 s_w[kBins];
    __shared__ unsigned s_c[kBins];
    const int tid = threadIdx.x;
    const size_t r = blockIdx.y;
    const float *x = a.s.logits + r * a.s.vocab;
    const int t0 = blockIdx.x * a.per, t1 = min(t0 + a.per, a.tiles);
    Slice s(x, (int)a.s.vocab, t0);
    const Params params(a, r);
    for (int i = tid; i < kBins; i += kSliceThreads) {
        s_w[i] = 0;
        s_c[i] = 0;
    }
    const Row row(a, params, (unsigned)(row_best(a, r) >> 32));
    if (row.none || row.best || !(row.use_k || row.use_p)) return;  // (uniform)
    __syncthreads();
    for (int t = t0;;) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            if (s.x[j] != s.x[j]) continue;
            const int b = row.bin(s.x[j]);
            atomicAdd(&s_c[b], 1u);
            if (row.use_p) {
                const u64 w = row.units(row.weight(s.x[j]));
                if (w) atomicAdd(&s_w[b], w);
            }
        }
        if (++t >= t1) break;
        s = Slice(x, (int)a.s.vocab, t);
    }
    __syncthreads();
    for (int i = tid; i < kBins; i += kSliceThreads) {
        if (s_c[i]) atomicAdd(&a.hist_c[r * kBins + i], s_c[i]);
        if (s_w[i]) atomicAdd(&a.hist_w[r * kBins + i], s_w[i]);
    }
}

// Step 3. Top-k's last token lies in the first step by which top_k tokens are counted. The weight
// that top-k keeps lies between that of the steps above and that with the step's own; so the
// cut of top-p lies between the steps that reach top_p of the one and of the other.
__global__ __launch_bounds__(kSliceThreads) void sample_collect_kernel(Args a) {
    constexpr int PB = kBins / kSliceThreads;  // steps per thread
    __shared__ u64 s_waves[kSliceThreads / 64];
    __shared__ unsigned s_waves32[kSliceThreads / 64];
    __shared__ int s_topk, s_lo, s_hi;
    __shared__ u64 s_before_topk, s_at_topk, s_before_cut;
    __shared__ unsigned s_above, s_here, s_from;
    const int tid = threadIdx.x;
    const size_t r = blockIdx.y;
    const float *x = a.s.logits + r * a.s.vocab;
    const int t0 = blockIdx.x * a.per, t1 = min(t0 + a.per, a.tiles);
    Slice s(x, (int)a.s.vocab, t0);
    const Params params(a, r);
    unsigned c[PB];
    u64 w[PB];
#pragma unroll
    for (int i = 0; i < PB; ++i) {
        c[i] = a.hist_c[r * kBins + tid * PB + i];
        w[i] = a.hist_w[r * kBins + tid * PB + i];
    }
    const Row row(a, params, (unsigned)(row_best(a, r) >> 32));
    if (row.none || row.best) return;  // (uniform)
    // Steps below lo are kept; steps lo to hi, and topk, are listed (kBins: none).
    int lo = kBins, hi = kBins, topk = kBins;
    if (row.use_k || row.use_p) {
        unsigned csum = 0;
        u64 wsum = 0;
#pragma unroll
        for (int i = 0; i < PB; ++i) {
            csum += c[i];
            wsum += w[i];
        }
        unsigned cend = csum;
        u64 wend = wsum;
        block_scan2<kSliceThreads>(cend, wend, s_waves32, s_waves);
        if (tid == kSliceThreads - 1) {
            s_topk = s_lo = s_hi = kBins;
            s_here = 0;
            s_before_topk = wend;
            s_at_topk = s_before_cut = 0;
            s_above = cend;
        }
        __syncthreads();
        if (row.use_k && cend >= row.top_k && cend - csum < row.top_k) {  // (at most one thread)
            unsigned above = cend - csum;
            u64 before = wend - wsum;
            bool found = false;
#pragma unroll
            for (int i = 0; i < PB; ++i) {
                if (!found && above + c[i] >= row.top_k) {
                    found = true;
                    s_topk = tid * PB + i;
                    s_above = above;
                    s_before_topk = before;
                    s_at_topk = w[i];
                }
                above += c[i];
                before += w[i];
            }
        }
        __syncthreads();
        topk = s_topk;
        lo = hi = topk;
        if (row.use_p) {
            const double least = (double)row.top_p * (double)s_before_topk;
            const double most = (double)row.top_p * (double)(s_before_topk + s_at_topk);
            u64 before = wend - wsum;
#pragma unroll
            for (int i = 0; i < PB; ++i) {
                const u64 end = before + w[i];
                const int b = tid * PB + i;
                if ((double)end >= least && ((double)before < least || b == 0)) {  // (one step)
                    s_lo = b;
                    s_before_cut = before;
                }
                if ((double)end >= most && ((double)before < most || b == 0)) s_hi = b;
                before = end;
            }
            __syncthreads();
            lo = min(s_lo, topk);
            hi = min(s_hi, topk);
        }
        if (blockIdx.x == 0 && tid == 0)
            a.cut[r] = Cut{row.use_p ? s_before_cut : s_before_topk, s_before_topk, s_above, topk};
    }
    for (int t = t0;;) {
        u64 sum = 0;
        unsigned mine = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            if (s.x[j] != s.x[j]) continue;
            const int b = row.bin(s.x[j]);
            if (b < lo)
                sum += row.units_kept(row.weight(s.x[j]));
            else if (b <= hi || b == topk)
                ++mine;
        }
        if (lo < kBins) {
            // This slice's part of the list (in any order: it is sorted).
            unsigned at = mine ? atomicAdd(&s_here, mine) : 0;
            __syncthreads();
            if (tid == 0) {
                s_from = s_here ? atomicAdd(&a.count[r], s_here) : 0;
                s_here = 0;
            }
            __syncthreads();
            at += s_from;
            if (mine) {
#pragma unroll
                for (int j = 0; j < kPer; ++j) {
                    if (s.x[j] != s.x[j]) continue;
                    const int b = row.bin(s.x[j]);
                    if (b >= lo && (b <= hi || b == topk)) {
                        if (at < kListed) a.listed[r * kListed + at] = rank_of(s.x[j], (unsigned)s.at(j));
                        ++at;
                    }
                }
            }
        }
        sum = block_total<kSliceThreads>(sum, s_waves);
        if (tid == 0) a.tile_sum[r * a.tiles + t] = sum;
        if (++t >= t1) break;
        s = Slice(x, (int)a.s.vocab, t);
    }
}

// ---- step 4: one workgroup per row --------------------------------------------------------------

constexpr int kTokens = kTile / kThreads;  // tokens per thread of the chosen slice

struct Shared {
    u64 wsum[kDigits];
    unsigned csum[kDigits];
    u64 waves[kWaves];
    unsigned waves32[kWaves];
    unsigned digit;
    u64 above_w, cut;
    unsigned above_c, in_last;
    int last;
};

// A row by itself: its cut by radix selection (returned as the least rank that is kept), and the
// tiles' kept weights in s_tiles.
__device__ __noinline__ u64 solve_row(const Args &a, const Row &row, const float *x, u64 *s_tiles, unsigned *s_eq,
                                      Shared &s) {
    const int n = (int)a.s.vocab, tiles = a.tiles, tid = threadIdx.x;
    // Tokens with a larger key are in, and the first `equal` of those with this key.
    unsigned cut = 1, equal = 0xFFFFFFFFu;

    // Highest digit first; pick(weight, count) says whether the cut lies no lower.
    auto radix = [&](bool weights, auto &&pick) {
        unsigned prefix = 0;
        u64 above_w = 0;
        unsigned above_c = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            if (tid < kDigits) {
                s.wsum[tid] = 0;
                s.csum[tid] = 0;
            }
            __syncthreads();
            for (int i = tid; i < n; i += kThreads) {
                const float v = x[i];
                const unsigned k = key_of(v);
                if (k == 0 || (shift < 24 && (k >> (shift + 8)) != prefix)) continue;
                const unsigned d = (k >> shift) & 255u;
                atomicAdd(&s.csum[d], 1u);
                // (of the tokens at top-k's cut only the first are in: `spare` below)
                if (weights && k >= cut) atomicAdd(&s.wsum[d], row.units(row.weight(v)));
            }
            __syncthreads();
            if (tid == 0) {
                int d = kDigits - 1;
                for (; d > 0; --d) {
                    if (pick(above_w + s.wsum[d], above_c + s.csum[d])) break;
                    above_w += s.wsum[d];
                    above_c += s.csum[d];
                }
                s.digit = d;
                s.above_w = above_w;
                s.above_c = above_c;
            }
            __syncthreads();
            prefix = prefix << 8 | s.digit;
            above_w = s.above_w;
            above_c = s.above_c;
        }
        return prefix;
    };

    if (row.use_k) {
        const unsigned top_k = row.top_k;
        const unsigned c = radix(false, [&](u64, unsigned count) { return count >= top_k; });
        if (c) {  // (0: fewer than top_k tokens, all are in)
            cut = c;
            equal = top_k - s.above_c;
        }
    }
    if (row.use_p) {
        // The total of what top-k keeps: keys above the cut, and `equal` times the cut's weight.
        u64 part = 0, same = 0;
        for (int i = tid; i < n; i += kThreads) {
            const float v = x[i];
            const unsigned k = key_of(v);
            if (k > cut) part += row.units(row.weight(v));
            if (k == cut) ++same;
        }
        const u64 above = block_total<kThreads>(part, s.waves);
        const u64 eq = block_total<kThreads>(same, s.waves);
        const u64 in = eq < equal ? eq : equal;
        const u64 cut_w = eq ? row.units(row.weight(value_of(cut))) : 0;
        const u64 total = above + in * cut_w;
        const u64 spare = (eq - in) * cut_w;  // weight of the cut's tokens that are out
        const double target = (double)row.top_p * (double)total;
        const unsigned c = radix(true, [&](u64 w, unsigned count) {
            // (the digit that holds the cut's key counts its tokens that are out too; there the
            // target, at most the total, is reached whether they count or not)
            return count > 0 && ((double)w >= target || w >= total + spare);
        });
        const unsigned key = c < cut ? cut : c;
        const u64 w = row.units(row.weight(value_of(key)));
        const u64 before = s.above_w;
        // token j of this key is in while before + j w < target (and the row's first always)
        unsigned keep = 0xFFFFFFFFu;
        if (w > 0) {
            const double j = __builtin_ceil((target - (double)before) / (double)w);
            keep = j < 1.0 ? 1u : j < 4.0e9 ? (unsigned)j : 0xFFFFFFFFu;
        }
        equal = key == cut && equal < keep ? equal : keep;
        cut = key;
    }

    // The kept weights above the cut, and the tokens at it, tile by tile.
    __syncthreads();
    for (int t = tid; t < tiles; t += kThreads) {
        s_tiles[t] = 0;
        s_eq[t] = 0;
    }
    __syncthreads();
    for (int t = 0; t < tiles; ++t) {
        u64 part = 0;
        unsigned same = 0;
#pragma unroll
        for (int j = 0; j < kTile / kThreads; ++j) {
            const int i = t * kTile + j * kThreads + tid;
            if (i >= n) continue;
            const unsigned k = key_of(x[i]);
            if (k == cut) ++same;
            if (k > cut) part += row.units_kept(row.weight(x[i]));
        }
        part = wave_total(part);
        same = wave_total(same);
        if ((tid & 63) == 0) {
            if (part) atomicAdd(&s_tiles[t], part);
            if (same) atomicAdd(&s_eq[t], same);
        }
    }
    __syncthreads();
    if (tid == 0) {  // the first `equal` of the cut's tokens, in the tiles' order
        const u64 cut_w = row.units_kept(row.weight(value_of(cut)));
        unsigned room = equal;
        s.last = -1;
        s.cut = (u64)cut << 32;
        for (int t = 0; t < tiles && room; ++t) {
            const unsigned in = s_eq[t] < room ? s_eq[t] : room;
            if (in) {
                s.last = t;
                s.in_last = in;
            }
            s_tiles[t] += (u64)in * cut_w;
            room -= in;
        }
    }
    __syncthreads();
    if (s.last >= 0) {  // the rank of the in_last-th of them in its tile
        const int base = s.last * kTile + kTokens * tid;
        unsigned same = 0;
        for (int j = 0; j < kTokens; ++j) same += base + j < n && key_of(x[base + j]) == cut;
        unsigned before = block_scan<kThreads>(same, s.waves32) - same;
        for (int j = 0; j < kTokens; ++j)
            if (base + j < n && key_of(x[base + j]) == cut && ++before == s.in_last)
                s.cut = rank_of(x[base + j], (unsigned)(base + j));
    }
    __syncthreads();
    return s.cut;
}

// The cut from a list of up to kThreads tokens, one per thread (`rank`: 0 for none), in LDS too;
// the kept ones' weights join their slices' sums.
__device__ __forceinline__ u64 cut_of_few(u64 rank, const u64 *s_list, u64 *s_sorted, unsigned listed, const Cut &c,
                                          const Row &row, u64 best, u64 *s_tiles, Shared &s) {
    const int tid = threadIdx.x;
    // Its place, largest first, is the number of larger ones (ranks differ).
    unsigned place = 0;
    for (unsigned i = 0; i < listed; i += 4) {  // (past the list: zeros)
#pragma unroll
        for (int j = 0; j < 4; ++j) place += s_list[i + j] > rank;
    }
    if (rank) s_sorted[place] = rank;
    __syncthreads();
    rank = (unsigned)tid < listed ? s_sorted[tid] : 0ull;
    const float v = value_of((unsigned)(rank >> 32));
    bool in = rank != 0;
    const double f = in ? row.weight(v) : 0.0;
    const u64 w = row.units(f);
    // Top-k keeps the first top_k - above of its step (the last of the listed steps); what it keeps
    // weighs `total`.
    const bool topk = in && row.bin(v) == c.topk_bin;
    const int others = __syncthreads_count(in && !topk);
    if (topk) in = (unsigned)(tid - others) < row.top_k - c.above;
    // Top-p keeps a token while the weight before it is below the target.
    if (row.use_p) {
        const u64 mine = in ? w : 0;
        const u64 end = wave_scan(mine), of_topk = wave_total(topk ? mine : 0ull);
        if ((tid & 63) == 63) s.waves[tid >> 6] = end;
        if ((tid & 63) == 0) s.wsum[tid >> 6] = of_topk;
        __syncthreads();
        u64 before = c.before_cut + end - mine, total = c.before_topk;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            if (i < tid >> 6) before += s.waves[i];
            total += s.wsum[i];
        }
        in = in && (rank == best || (double)before < (double)row.top_p * (double)total);
    }
    if (in && w && f >= row.min_p) atomicAdd(&s_tiles[index_of(rank) / kTile], w);
    const int kept = __syncthreads_count(in);  // (the first `kept` of the order, at least one)
    return s_sorted[kept - 1];
}

// The same from a longer list, sorted in LDS, by the workgroup.
__device__ __noinline__ u64 cut_of_list(u64 *s_list, u64 *s_w, unsigned listed, const Cut &c, const Row &row, u64 best,
                                        u64 *s_tiles, Shared &s) {
    const int tid = threadIdx.x;
    int size = 1;
    while (size < (int)listed) size *= 2;  // (zeros pad the list)
    __syncthreads();
    for (int k = 2; k <= size; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            for (int i = tid; i < size / 2; i += kThreads) {
                const int p = 2 * i - (i & (j - 1)), q = p + j;
                const u64 u = s_list[p], v = s_list[q];
                if ((u < v) == ((p & k) == 0)) {
                    s_list[p] = v;
                    s_list[q] = u;
                }
            }
            __syncthreads();
        }
    // Thread tid has places from .. to - 1 of the order.
    const int pt = (size + kThreads - 1) / kThreads, from = min(pt * tid, (int)listed), to = min(from + pt, (int)listed);
    auto value = [&](int i) { return value_of((unsigned)(s_list[i] >> 32)); };
    unsigned here = 0;
    for (int i = from; i < to; ++i) {
        s_w[i] = row.units(row.weight(value(i)));
        here += row.bin(value(i)) == c.topk_bin;
    }
    unsigned place = block_scan<kThreads>(here, s.waves32) - here;
    const unsigned keep_k = row.use_k ? row.top_k - c.above : 0xFFFFFFFFu;
    u64 mine = 0, all = 0;
    int stop = to;  // this thread's first place that top-k does not keep
    for (int i = from; i < to; ++i) {
        const bool topk = row.bin(value(i)) == c.topk_bin;
        if (topk && place++ >= keep_k) {
            stop = i;
            break;
        }
        if (topk) mine += s_w[i];
        all += s_w[i];
    }
    const u64 total = c.before_topk + block_total<kThreads>(mine, s.waves);
    if (row.use_p) {
        const double target = (double)row.top_p * (double)total;
        u64 before = c.before_cut + block_scan<kThreads>(all, s.waves) - all;
        for (int i = from; i < stop; ++i) {
            if (s_list[i] != best && !((double)before < target)) {
                stop = i;
                break;
            }
            before += s_w[i];
        }
    }
    __syncthreads();
    if (tid == 0) s.cut = ~0ull;
    __syncthreads();
    for (int i = from; i < stop; ++i)
        if (s_w[i] && row.weight(value(i)) >= row.min_p) atomicAdd(&s_tiles[index_of(s_list[i]) / kTile], s_w[i]);
    if (stop > from) atomicMin(&s.cut, s_list[stop - 1]);
    __syncthreads();
    return s.cut;
}

__global__ __launch_bounds__(kThreads) void sample_choose_kernel(Args a) {
    __shared__ Shared s;
    __shared__ u64 s_list[kListed], s_w[kListed];
    extern __shared__ u64 s_tiles[];  // [tiles], then [tiles] u32
    unsigned *s_eq = reinterpret_cast<unsigned *>(s_tiles + a.tiles);
    const size_t r = blockIdx.x;
    const int n = (int)a.s.vocab, tiles = a.tiles, tid = threadIdx.x, lane = tid & 63;
    const float *x = a.s.logits + r * a.s.vocab;

    // (loads first; what a row does not need may be anything)
    u64 rank = a.listed[r * kListed + tid];
    const unsigned counted = a.count[r];
    const Cut c = a.cut[r];
    const float u = a.s.u[r];
    const Params params(a, r);
    for (int t = tid; t < tiles; t += kThreads) s_tiles[t] = a.tile_sum[r * tiles + t];
    const u64 best = row_best(a, r);
    const Row row(a, params, (unsigned)(best >> 32));
    if (row.none || row.best) {  // (uniform)
        if (tid == 0) a.s.out[r] = row.none ? 0u : index_of(best);
        return;
    }
    const unsigned listed = row.use_k || row.use_p ? counted : 0u;  // (0: every token is kept)
    u64 cut = kLeastRank;
    rank = (unsigned)tid < listed ? rank : 0ull;
    s_list[tid] = rank;
    __syncthreads();
    if (listed > kListed) {  // (uniform, as below)
        cut = solve_row(a, row, x, s_tiles, s_eq, s);
    } else if (listed > kThreads) {
        for (unsigned i = tid + kThreads; i < kListed; i += kThreads) s_list[i] = i < listed ? a.listed[r * kListed + i] : 0;
        cut = cut_of_list(s_list, s_w, listed, c, row, best, s_tiles, s);
    } else if (listed > 0) {
        cut = cut_of_few(rank, s_list, s_w, listed, c, row, best, s_tiles, s);
    }
    if (listed > kThreads) __syncthreads();

    // The slice that holds the token, found by every wave: lane l has `per` tiles from per * l on.
    int tile = 0;
    u64 left = 0;
    {
        const int per = (tiles + 63) / 64;
        u64 mine = 0;
        for (int t = per * lane; t < min(per * (lane + 1), tiles); ++t) mine += s_tiles[t];
        const u64 end = wave_scan(mine), total = __shfl(end, 63);
        const double place = u > 0.0f ? (double)u * (double)total : 0.0;
        u64 thr = place >= (double)total ? total - 1 : (u64)place;
        if (thr >= total) thr = total - 1;
        const bool here = thr < end && thr >= end - mine;  // (one lane)
        thr -= end - mine;
        int t = per * lane;
        while (here && thr >= s_tiles[t]) thr -= s_tiles[t++];
        const int l = __ffsll((long long)__ballot(here)) - 1;
        tile = __shfl(t, l);
        left = __shfl(thr, l);
    }
    // And the token in it: thread tid has tokens kTokens * tid ...
    const int base = tile * kTile + tid * kTokens;
    float v[kTokens];
    if ((n & 3) == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0) {
#pragma unroll
        for (int j = 0; j < kTokens; j += 4) {
            const f32x4 q = *reinterpret_cast<const f32x4 *>(x + min(base + j, n - 4));
#pragma unroll
            for (int i = 0; i < 4; ++i) v[j + i] = base + j < n ? q[i] : __builtin_nanf("");
        }
    } else {
#pragma unroll
        for (int j = 0; j < kTokens; ++j) v[j] = base + j < n ? x[base + j] : __builtin_nanf("");
    }
    u64 w[kTokens], mine = 0;
#pragma unroll
    for (int j = 0; j < kTokens; ++j) {
        w[j] = 0;
        if (v[j] == v[j] && rank_of(v[j], (unsigned)(base + j)) >= cut) w[j] = row.units_kept(row.weight(v[j]));
        mine += w[j];
    }
    u64 cum = block_scan<kThreads>(mine, s.waves) - mine;
    if (cum <= left && cum + mine > left) {  // (one thread)
#pragma unroll
        for (int j = 0; j < kTokens; ++j) {
            if (cum <= left && cum + w[j] > left) a.s.out[r] = (unsigned)(base + j);
            cum += w[j];
        }
    }
}

struct Layout {
    size_t best, tile_sum, hist_w, listed, cut, hist_c, count, floats;  // offsets in floats
};
Layout layout_of(size_t rows, size_t tiles) {
    Layout l{};
    size_t at = 0;
    auto take = [&](size_t floats) {
        const size_t here = at;
        at += (floats + 3) / 4 * 4;
        return here;
    };
    l.best = take(2 * rows * tiles);
    l.tile_sum = take(2 * rows * tiles);
    l.hist_w = take(2 * rows * kBins);
    l.listed = take(2 * rows * kListed);
    l.cut = take(sizeof(Cut) / 4 * rows);
    l.hist_c = take(rows * kBins);
    l.count = take(rows);
    l.floats = at;
    return l;
}

constexpr size_t kMaxVocab = (size_t)1 << 24;
// Where slices are more than this many for every CU, a workgroup of steps 1 to 3 takes several of a
// row, so that a row's parameters, largest logit and cut are found by fewer. Rows of 151936, top-k 50
// and top-p 0.9: 64 rows 57 us in runs of 2 and 65.5 a slice each, 256 rows 152 and 185.
constexpr size_t kGroupsPerCu = 7;
// A row's histogram and list take 45 KB whatever its vocabulary: rows beyond this many go through the
// same workspace after the others (65535 rows would ask for 3 GB; these take 185 MB). Another batch
// costs its launches and its tail: in batches of 1024, 2048 rows of 500 took 94 us instead of 81, 4096
// of 32000 616 instead of 547.
constexpr size_t kBatchRows = 4096;

eb_status launch_batch(hipStream_t st, const eb::SampleArgs &s, float *ws) {
    Args a{};
    a.s = s;
    a.frac = 44;
    while (((size_t)1 << (62 - a.frac)) < s.vocab) --a.frac;
    const size_t tiles = (s.vocab + kTile - 1) / kTile, cus = (size_t)eb::current_cu_count();
    a.tiles = (int)tiles;
    const size_t per = (tiles * s.rows + kGroupsPerCu * cus - 1) / (kGroupsPerCu * cus);
    a.groups = (int)((tiles + per - 1) / per);
    a.per = (a.tiles + a.groups - 1) / a.groups;
    a.groups = (a.tiles + a.per - 1) / a.per;
    const size_t lds = tiles * 12 + 8;
    const Layout l = layout_of(s.rows, tiles);
    a.best = reinterpret_cast<u64 *>(ws + l.best);
    a.tile_sum = reinterpret_cast<u64 *>(ws + l.tile_sum);
    a.hist_w = reinterpret_cast<u64 *>(ws + l.hist_w);
    a.hist_c = reinterpret_cast<unsigned *>(ws + l.hist_c);
    a.listed = reinterpret_cast<u64 *>(ws + l.listed);
    a.count = reinterpret_cast<unsigned *>(ws + l.count);
    a.cut = reinterpret_cast<Cut *>(ws + l.cut);
    const dim3 grid((unsigned)a.groups, (unsigned)s.rows);
    sample_max_kernel<<<grid, kSliceThreads, 0, st>>>(a);
    // (the parameters lie in device memory: which rows have a cut is known to the kernels alone)
    if (s.top_k || s.top_p) sample_histogram_kernel<<<grid, kSliceThreads, 0, st>>>(a);
    sample_collect_kernel<<<grid, kSliceThreads, 0, st>>>(a);
    sample_choose_kernel<<<(unsigned)s.rows, kThreads, lds, st>>>(a);
    return eb::check_launch("sample");
}

}  // namespace

namespace eb {

size_t sample_workspace_floats(size_t rows, size_t vocab) {
    return layout_of(std::min(rows, kBatchRows), (vocab + kTile - 1) / kTile).floats;
}

eb_status launch_sample(hipStream_t st, const SampleArgs &s, float *ws) {
    static const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&sample_choose_kernel),
                                                    hipFuncAttributeMaxDynamicSharedMemorySize,
                                                    (int)(kMaxVocab / kTile * 12 + 8));
    if (e != hipSuccess) return hip_fail(e, "sample launch set-up");
    for (size_t r = 0; r < s.rows; r += kBatchRows) {
        auto from = [&](auto *p) { return p ? p + r : nullptr; };
        const SampleArgs b{s.logits + r * s.vocab, s.u + r,         from(s.temperature),
                           from(s.top_k),          from(s.top_p),   from(s.min_p),
                           s.out + r,              std::min(kBatchRows, s.rows - r), s.vocab};
        const eb_status status = launch_batch(st, b, ws);
        if (status != EB_OK) return status;
    }
    return EB_OK;
}

}  // namespace eb
