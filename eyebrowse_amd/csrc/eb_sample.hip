// Sampling for gfx950: temperature, top-k, top-p and min-p over a row of logits, and the token
// that a given random number picks from what they keep.
//
// A token's weight is w = 2^((x - max) log2(e) / T), computed in f64 and rounded once to a whole
// number of 2^-F units (F = 62 - ceil(log2 vocab), so that a row's sum fits 64 bits). Sums of
// whole numbers do not depend on their order: histograms may be filled by atomics, and the choice
// is the same on every run. Ranks go by the logit's bits made monotonic (equal logits by index).
#include "eb_common.h"
#include "eb_internal.h"

#include <cstdint>

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kTile = 4096;   // tokens whose kept weights are summed together
constexpr int kDigits = 256;  // of a radix pass

struct Args {
    eb::SampleArgs s;
    int frac;  // F
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

// 2^y for y <= 0: 2^n times the Taylor sum of e^(f ln 2) for y = n + f, |f| <= 1/2 (the first term
// left out is below 2e-16).
__device__ __forceinline__ double exp2_f64(double y) {
    y = fmax(y, -2000.0);  // (0 from there on)
    const double n = __builtin_rint(y);
    const double f = (y - n) * 0.693147180559945309417232121458;
    double p = 1.0 / 479001600;
    p = __builtin_fma(p, f, 1.0 / 39916800);
    p = __builtin_fma(p, f, 1.0 / 3628800);
    p = __builtin_fma(p, f, 1.0 / 362880);
    p = __builtin_fma(p, f, 1.0 / 40320);
    p = __builtin_fma(p, f, 1.0 / 5040);
    p = __builtin_fma(p, f, 1.0 / 720);
    p = __builtin_fma(p, f, 1.0 / 120);
    p = __builtin_fma(p, f, 1.0 / 24);
    p = __builtin_fma(p, f, 1.0 / 6);
    p = __builtin_fma(p, f, 0.5);
    p = __builtin_fma(p, f, 1.0);
    p = __builtin_fma(p, f, 1.0);
    return ldexp(p, (int)n);
}

struct Row {
    double rate;    // log2(e) / T
    float top;      // the largest logit
    double min_p;   // 0: off
    int frac;
    __device__ __forceinline__ double weight(float x) const {
        if (x == top) return 1.0;  // (top is finite or +inf)
        if (x == -INFINITY) return 0.0;
        return exp2_f64(((double)x - (double)top) * rate);
    }
    __device__ __forceinline__ u64 units(double w) const { return (u64)(ldexp(w, frac) + 0.5); }
};

template <class T>
__device__ __forceinline__ T wave_total(T x) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) x += __shfl_xor(x, m);
    return x;
}

struct Shared {
    u64 wsum[kDigits];
    unsigned csum[kDigits];
    u64 red[kWaves];
    unsigned digit;
    u64 above_w;
    unsigned above_c;
};

__device__ __forceinline__ u64 block_total(u64 x, Shared &s) {
    x = wave_total(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.red[threadIdx.x >> 6] = x;
    __syncthreads();
    u64 t = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) t += s.red[w];
    return t;
}

// One workgroup per row.
__global__ __launch_bounds__(kThreads) void sample_row_kernel(Args a) {
    __shared__ Shared s;
    extern __shared__ u64 s_tiles[];  // [tiles] kept weight above the cut, then [tiles] u32 equal keys
    const size_t r = blockIdx.x;
    const int n = (int)a.s.vocab;
    const int tid = threadIdx.x;
    const float *x = a.s.logits + r * a.s.vocab;
    const int tiles = (n + kTile - 1) / kTile;
    unsigned *s_eq = reinterpret_cast<unsigned *>(s_tiles + tiles);

    // ---- the row's largest logit ----
    unsigned best = 0;
    for (int i = tid; i < n; i += kThreads) {
        const unsigned k = key_of(x[i]);
        best = k > best ? k : best;
    }
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) {
        const unsigned o = __shfl_xor(best, m);
        best = o > best ? o : best;
    }
    if ((tid & 63) == 0) s.red[tid >> 6] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) best = (unsigned)s.red[w] > best ? (unsigned)s.red[w] : best;
    __syncthreads();
    if (best <= key_of(-INFINITY)) {  // (only -inf and NaN)
        if (tid == 0) a.s.out[r] = 0;
        return;
    }
    const float temp = a.s.temperature ? a.s.temperature[r] : 1.0f;
    const float min_p = a.s.min_p ? a.s.min_p[r] : 0.0f;
    const float top_p = a.s.top_p ? a.s.top_p[r] : 1.0f;
    const bool greedy = !(temp > 0.0f) || min_p > 1.0f;
    unsigned top_k = a.s.top_k ? a.s.top_k[r] : 0u;
    if (greedy) top_k = 1;
    const bool use_k = top_k > 0 && top_k < (unsigned)n;
    const bool use_p = top_p < 1.0f && !greedy;
    Row row;
    row.rate = 1.4426950408889634073599 / (temp > 0.0f ? (double)temp : 1.0);
    row.top = value_of(best);
    row.min_p = min_p > 0.0f && !greedy ? (double)min_p : 0.0;
    row.frac = a.frac;

    // The cut: tokens with a larger key are in, and the first `equal` of those with this key.
    unsigned cut = 1, equal = 0xFFFFFFFFu;

    // Radix selection, highest digit first: digit(sums, above) names the digit that the cut has.
    auto radix = [&](bool weights, auto &&pick) {
        unsigned prefix = 0;
        u64 above_w = 0;
        unsigned above_c = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
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
                if (weights && k >= cut) {
                    // (of the keys at top-k's cut only the first `equal` are in: taken off below)
                    atomicAdd(&s.wsum[d], row.units(row.weight(v)));
                }
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

    if (use_k) {
        const unsigned c = radix(false, [&](u64, unsigned count) { return count >= top_k; });
        cut = c == 0 ? 1 : c;
        equal = c == 0 ? 0xFFFFFFFFu : top_k - s.above_c;  // (fewer than k tokens: all are in)
        __syncthreads();
    }
    if (use_p) {
        // The total of what top-k keeps: keys above the cut, and `equal` times the cut's weight.
        u64 part = 0;
        unsigned same = 0;
        for (int i = tid; i < n; i += kThreads) {
            const float v = x[i];
            const unsigned k = key_of(v);
            if (k > cut) part += row.units(row.weight(v));
            if (k == cut) ++same;
        }
        const u64 above = block_total(part, s);
        const u64 eq = block_total(same, s);
        const u64 in = eq < equal ? eq : equal;
        const u64 cut_w = eq ? row.units(row.weight(value_of(cut))) : 0;
        const u64 total = above + in * cut_w;
        const u64 spare = (eq - in) * cut_w;  // weight of the cut's tokens that are out
        const double target = (double)top_p * (double)total;
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
        if (key == cut)
            equal = keep < equal ? keep : equal;
        else
            equal = keep;
        cut = key;
        __syncthreads();
    }

    // ---- the kept weights, tile by tile ----
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
            const float v = x[i];
            const unsigned k = key_of(v);
            if (k == cut) ++same;
            if (k > cut) {
                const double w = row.weight(v);
                if (w >= row.min_p) part += row.units(w);
            }
        }
        part = wave_total(part);
        same = wave_total(same);
        if ((tid & 63) == 0) {
            if (part) atomicAdd(&s_tiles[t], part);
            if (same) atomicAdd(&s_eq[t], same);
        }
    }
    __syncthreads();
    const double cw = row.weight(value_of(cut));
    const u64 cut_w = cw >= row.min_p ? row.units(cw) : 0;
    __shared__ int s_tile;
    __shared__ u64 s_left;       // weight still to pass inside the tile
    __shared__ unsigned s_room;  // equal keys still in at its start
    if (tid == 0) {
        u64 total = 0;
        unsigned room = equal;
        for (int t = 0; t < tiles; ++t) {
            const unsigned in = s_eq[t] < room ? s_eq[t] : room;
            total += s_tiles[t] + (u64)in * cut_w;
            room -= in;
        }
        const float u = a.s.u[r];
        const double at = u > 0.0f ? (double)u * (double)total : 0.0;
        u64 thr = at >= (double)total ? total - 1 : (u64)at;
        if (thr >= total) thr = total - 1;
        room = equal;
        int t = 0;
        u64 cum = 0;
        for (; t < tiles; ++t) {
            const unsigned in = s_eq[t] < room ? s_eq[t] : room;
            const u64 w = s_tiles[t] + (u64)in * cut_w;
            if (cum + w > thr) break;
            cum += w;
            room -= in;
        }
        s_tile = t < tiles ? t : tiles - 1;
        s_left = thr - cum;
        s_room = room;
    }
    __syncthreads();

    // ---- the tile in order: thread tid has tokens 4 tid .. 4 tid + 3 ----
    const int base = s_tile * kTile + tid * 4;
    float v[4];
    unsigned same = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[j] = base + j < n ? x[base + j] : __builtin_nanf("");
        same += key_of(v[j]) == cut;
    }
    const int lane = tid & 63, wave = tid >> 6;
    auto exclusive = [&](u64 mine) {  // the sum over earlier threads
        u64 inc = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const u64 o = __shfl_up(inc, d);
            if (lane >= d) inc += o;
        }
        __syncthreads();
        if (lane == 63) s.red[wave] = inc;
        __syncthreads();
        u64 before = inc - mine;
        for (int w = 0; w < wave; ++w) before += s.red[w];
        return before;
    };
    unsigned rank = (unsigned)exclusive(same);
    u64 w[4], mine = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const unsigned k = key_of(v[j]);
        w[j] = 0;
        if (k == cut) {
            if (rank < s_room) w[j] = cut_w;
            ++rank;
        } else if (k > cut) {
            const double f = row.weight(v[j]);
            if (f >= row.min_p) w[j] = row.units(f);
        }
        mine += w[j];
    }
    u64 cum = exclusive(mine);
    if (cum <= s_left && cum + mine > s_left) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (cum <= s_left && cum + w[j] > s_left) a.s.out[r] = (unsigned)(base + j);
            cum += w[j];
        }
    }
}

}  // namespace

namespace eb {

size_t sample_workspace_floats(size_t rows, size_t vocab) {
    (void)rows;
    (void)vocab;
    return 0;
}

eb_status launch_sample(hipStream_t st, const SampleArgs &s, float *ws) {
    (void)ws;
    if (s.vocab > ((size_t)1 << 24))
        return fail(EB_UNSUPPORTED_CONFIG, "sample: vocab %zu (at most 2^24)", s.vocab);
    Args a{s, 62};
    while (((size_t)1 << (62 - a.frac)) < s.vocab) --a.frac;
    const size_t tiles = (s.vocab + kTile - 1) / kTile;
    const size_t lds = tiles * 12 + 8;
    sample_row_kernel<<<(unsigned)s.rows, kThreads, lds, st>>>(a);
    return check_launch("sample");
}

}  // namespace eb
