// Projections with 4-bit weights and group scales for gfx950:
//   y[i, o] = sum_g s[o, g] sum_{k in g} x[i, k] (q[o, k] - z[o, g])
// with x and y f32, q 4-bit codes (eight per word, lowest bits first), s half, z a byte (or 8).
//
// Both forms run on the matrix cores. A code less its zero point is a whole number, exact in f16.
// An x row is scaled by a power of two (its largest magnitude lands in [2^14, 2^15)) and split
// into f16 halves hi + lo, 22 bits of it; each product is exact in f32. The sum over a group is
// accumulated apart, then scaled and added in f32, so that no scale is rounded to f16.
//
// Unpacking a word gives four f16 pairs with nine instructions: (w & 0x000F000F) | 0x64006400 is
// the pair (1024 + k0, 1024 + k4), from which 1024 + z is subtracted; (w & 0x00F000F0) |
// 0x64006400 is (1024 + 16 k1, 1024 + 16 k5), times 1/16 less 64 + z; the same of w >> 8. So a
// word's contraction order is k0 k4 k1 k5 k2 k6 k3 k7, and x's halves are laid out in it.
#include "eb_common.h"
#include "eb_internal.h"

#include <algorithm>
#include <climits>

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct Seg {
    const uint32_t *w;
    const _Float16 *s;
    const uint8_t *z;
    float *y;
    int n;      // features
    int first;  // first 16-feature tile (or work unit) of the pair
};
struct Segs {
    Seg seg[eb::kLinearMaxSegs];
    int nseg, total;  // tiles of all pairs
};
__device__ __forceinline__ int seg_of(const Segs &s, int u) {
    int i = 0;
#pragma unroll
    for (int j = 1; j < eb::kLinearMaxSegs; ++j) i += (j < s.nseg && u >= s.seg[j].first) ? 1 : 0;
    return i;
}

// The four f16 pairs of a word: codes less their zero point.
struct Zero {
    f16x2 low, high;  // -(1024 + z), -(64 + z), twice each
};
// From byte i of z4: 0xE400 + z is f16 -(1024 + z).
__device__ __forceinline__ Zero zero_of(unsigned z4, int i) {
    const f16x2 up = {(_Float16)960.0f, (_Float16)960.0f};
    const unsigned sel = 0x04000400u | (unsigned)i * 0x00010001u;  // (z, 0xE4, z, 0xE4)
    const f16x2 low = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0xE4E4E4E4u, z4, sel));
    return Zero{low, low + up};
}
__device__ __forceinline__ f16x8 unpack(unsigned w, const Zero &z) {
    const f16x2 sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
    const unsigned v = w >> 8;
    const f16x2 a = __builtin_bit_cast(f16x2, (w & 0x000F000Fu) | 0x64006400u) + z.low;
    const f16x2 b = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (w & 0x00F000F0u) | 0x64006400u), sixteenth, z.high);
    const f16x2 c = __builtin_bit_cast(f16x2, (v & 0x000F000Fu) | 0x64006400u) + z.low;
    const f16x2 d = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (v & 0x00F000F0u) | 0x64006400u), sixteenth, z.high);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Eight values of a row (k0 .. k7), scaled by 2^-e, as hi and lo halves in a word's order.
__device__ __forceinline__ void split8(f32x4 a, f32x4 b, int e, f16x8 &hi, f16x8 &lo) {
    const float v[8] = {a[0], b[0], a[1], b[1], a[2], b[2], a[3], b[3]};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = ldexpf(v[i], -e);
        hi[i] = (_Float16)x;
        lo[i] = (_Float16)(x - (float)hi[i]);
    }
}

// The exponent e of a row's scale 2^-e, from its largest magnitude's bits: 0 for a zero row, and
// for one with a value that is not finite (which then reaches every output of the row).
__device__ __forceinline__ int row_exponent(unsigned top) {
    if (top == 0 || top >= 0x7F800000u) return 0;
    return ilogbf(__builtin_bit_cast(float, top)) - 14;
}
__device__ __forceinline__ unsigned max_bits(unsigned top, f32x4 x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned a = eb::magnitude_bits(x[i]);
        top = a > top ? a : top;
    }
    return top;
}

// ------------------------------------------------------------------------ up to 8 rows --------
// A wave takes tiles of 16 features: B of v_mfma_f32_16x16x32_f16 is 16 features' codes (lane
// (n, g) = lane n + 16 g: feature n), A the x rows, hi halves in rows 0..7 and lo halves in rows
// 8..15, so that one product serves both. A block is 128 of the contraction, 16 words of a
// feature: lane (n, g) loads words 4g .. 4g + 3 in one 16-byte load. Each of the block's four
// products takes one word of every lane, and these must lie in one group: at group 128 any
// word does; at 64 lane groups 0, 1 hold the first group and 2, 3 the second, and two swaps of
// wave halves bring each group's words together; at 32 a 4 x 4 transpose over lane groups and
// words does (four swaps). The rows' halves stay in LDS; a workgroup splits them once and then
// walks its tiles; kw waves share a tile's contraction.
constexpr int kGemvWaves = 8;
constexpr int kGemvThreads = kGemvWaves * 64;
constexpr int kDepth = 4;  // blocks of weights in flight per wave

template <int G>
struct Block {
    static constexpr int NG = 128 / G;  // groups
    unsigned w[4];
    unsigned s[(NG + 1) / 2];  // scales, two halves a word
    unsigned z;                // zero points, a byte each
};

// w[j] of lane group g for w[j'] of g', bit b of j and bit b of g exchanged (b = 1: wave halves,
// b = 0: neighbouring 16-lane rows).
__device__ __forceinline__ void swap_halves(unsigned &a, unsigned &b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}
__device__ __forceinline__ void swap_rows(unsigned &a, unsigned &b) {
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}

// VEC: a block's scales and zero points lie aligned in one load each (K % 128 == 0, aligned bases).
template <int G, bool ZERO, bool VEC>
__global__ __launch_bounds__(kGemvThreads, 4) void q4_gemv_kernel(const float *__restrict__ x, Segs segs, int m,
                                                                  int K, int kw) {
    using B = Block<G>;
    constexpr int NG = B::NG;
    extern __shared__ f16x8 lds[];  // [blocks * 16 chunks][2 m]: chunk c of row i: hi, then lo
    __shared__ unsigned s_top[kGemvWaves][8];
    __shared__ float s_part[kGemvWaves][8][16];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int nb = (K + 127) / 128;  // blocks of a row
    const int ngr = K / G;           // groups of a row
    const int nw = K / 8;            // words of a row

    // This wave's walk: tiles t0, t0 + units, ..., of each `per` blocks from b0 on. (Blocks past the
    // row's last and tiles past the last are skipped, but walked: waves that share a tile meet at
    // its end, in barriers of the workgroup.)
    const int units = (int)gridDim.x * (kGemvWaves / kw);
    const int t0 = (int)blockIdx.x * (kGemvWaves / kw) + wave / kw;
    const int per = (nb + kw - 1) / kw;
    const int b0 = wave % kw * per;
    const int steps = (segs.total + units - 1) / units * per;

    B ring[kDepth];
    int lt = t0, lb = 0;  // the next block to load
    auto load = [&](B &r) {
        if (lt < segs.total && b0 + lb < nb) {
            const Seg &sg = segs.seg[seg_of(segs, lt)];
            const int o = min((lt - sg.first) * 16 + n, sg.n - 1);
            const int b = b0 + lb;
            // (words past the row's end repeat its last ones, against zeros of x)
            const int at = VEC ? 16 * b + 4 * g : min(16 * b + 4 * g, nw - 4);
            const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(sg.w + (size_t)o * nw + at));
#pragma unroll
            for (int j = 0; j < 4; ++j) r.w[j] = v[j];
            const size_t gr = (size_t)o * ngr + b * NG;
            if constexpr (VEC && NG == 4) {
                const u32x2 q = *reinterpret_cast<const u32x2 *>(sg.s + gr);
                r.s[0] = q[0];
                r.s[1] = q[1];
                if constexpr (ZERO) r.z = *reinterpret_cast<const unsigned *>(sg.z + gr);
            } else if constexpr (VEC && NG == 2) {
                r.s[0] = *reinterpret_cast<const unsigned *>(sg.s + gr);
                if constexpr (ZERO) r.z = *reinterpret_cast<const uint16_t *>(sg.z + gr);
            } else {
                unsigned z = 0;
                unsigned sc[(NG + 1) / 2] = {};
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    const size_t gi = (size_t)o * ngr + min(b * NG + i, ngr - 1);
                    sc[i / 2] |= (unsigned)__builtin_bit_cast(uint16_t, sg.s[gi]) << (16 * (i % 2));
                    if constexpr (ZERO) z |= (unsigned)sg.z[gi] << (8 * i);
                }
#pragma unroll
                for (int i = 0; i < (NG + 1) / 2; ++i) r.s[i] = sc[i];
                r.z = z;
            }
        }
        if (++lb == per) {
            lb = 0;
            lt += units;
        }
    };
#pragma unroll
    for (int i = 0; i < kDepth; ++i) load(ring[i]);
    __builtin_amdgcn_sched_barrier(0);

    // The rows' exponents and halves; a thread's first chunk of each row stays in registers.
    f32x4 keep[8][2];
    const f32x4 z4 = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (i >= m) break;
        const f32x4 *p = reinterpret_cast<const f32x4 *>(x + (size_t)i * K);
        keep[i][0] = tid < nw ? p[2 * tid] : z4;
        keep[i][1] = tid < nw ? p[2 * tid + 1] : z4;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (i >= m) break;
        const f32x4 *p = reinterpret_cast<const f32x4 *>(x + (size_t)i * K);
        unsigned top = max_bits(max_bits(0u, keep[i][0]), keep[i][1]);
        for (int c = tid + kGemvThreads; c < nw; c += kGemvThreads) top = max_bits(max_bits(top, p[2 * c]), p[2 * c + 1]);
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            const unsigned o = __shfl_xor(top, d);
            top = o > top ? o : top;
        }
        if (lane == 0) s_top[wave][i] = top;
    }
    __syncthreads();
    auto exponent = [&](int i) {
        unsigned top = 0;
#pragma unroll
        for (int w = 0; w < kGemvWaves; ++w) top = s_top[w][i] > top ? s_top[w][i] : top;
        return row_exponent(top);
    };
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (i >= m) break;
        const f32x4 *p = reinterpret_cast<const f32x4 *>(x + (size_t)i * K);
        const int e = exponent(i);
        for (int c = tid; c < nb * 16; c += kGemvThreads) {
            f16x8 hi = {}, lo = {};
            if (c == tid)
                split8(keep[i][0], keep[i][1], e, hi, lo);  // (zeros past the row's end)
            else if (c < nw)
                split8(p[2 * c], p[2 * c + 1], e, hi, lo);
            lds[c * 2 * m + i] = hi;
            lds[c * 2 * m + m + i] = lo;
        }
    }
    __syncthreads();

    const int row = (n < 8 ? 0 : m) + min(n & 7, m - 1);  // (rows past m: the last, not stored)
    // The chunk of lane group g in product j: word 4 g' + j', bits of g and j exchanged.
    const int gw = G == 128 ? 4 * g : G == 64 ? 4 * (g & 1) + (g & 2) : g;
    auto word = [](int j) { return G == 128 ? j : G == 64 ? 4 * (j & 2) + (j & 1) : 4 * j; };
    const f16x8 *xa = lds + gw * 2 * m + row;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    int ct = t0, cb = 0;
    auto finish = [&] {
        // Rows 4 g + r: hi sums in lanes g 0, 1, lo sums 32 lanes on.
        float v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = acc[r] + eb::lane_xor32(acc[r]);
        if (kw == 1) {
            if (ct < segs.total) {
                const Seg &sg = segs.seg[seg_of(segs, ct)];
                const int o = (ct - sg.first) * 16 + n;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (g < 2 && o < sg.n && 4 * g + r < m)
                        sg.y[(size_t)(4 * g + r) * sg.n + o] = ldexpf(v[r], exponent(4 * g + r));
            }
        } else {
            if (g < 2)
#pragma unroll
                for (int r = 0; r < 4; ++r) s_part[wave][4 * g + r][n] = v[r];
            __syncthreads();
            // The first wave of each tile's waves adds their sums: lane (n, g) rows g and g + 4.
            if (wave % kw == 0 && ct < segs.total) {
                const Seg &sg = segs.seg[seg_of(segs, ct)];
                const int o = (ct - sg.first) * 16 + n;
#pragma unroll
                for (int i = g; i < 8; i += 4)
                    if (i < m && o < sg.n) {
                        float t = 0.0f;
                        for (int w = 0; w < kw; ++w) t += s_part[wave + w][i][n];
                        sg.y[(size_t)i * sg.n + o] = ldexpf(t, exponent(i));
                    }
            }
            __syncthreads();
        }
        acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        ct += units;
    };
    auto consume = [&](B &r) {
        if (ct < segs.total && b0 + cb < nb) {
            const f16x8 *xb = xa + (size_t)(b0 + cb) * 16 * 2 * m;
            if constexpr (G <= 64) {
                swap_halves(r.w[0], r.w[2]);
                swap_halves(r.w[1], r.w[3]);
            }
            if constexpr (G == 32) {
                swap_rows(r.w[0], r.w[1]);
                swap_rows(r.w[2], r.w[3]);
            }
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                const Zero z = zero_of(ZERO ? r.z : 0x08080808u, i);
                f32x4 t = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = i * (4 / NG); j < (i + 1) * (4 / NG); ++j)
                    t = __builtin_amdgcn_mfma_f32_16x16x32_f16(xb[word(j) * 2 * m], unpack(r.w[j], z), t, 0, 0, 0);
                acc += t * (float)__builtin_bit_cast(_Float16, (unsigned short)(r.s[i / 2] >> (16 * (i % 2))));
            }
        }
        if (++cb == per) {
            cb = 0;
            finish();
        }
    };
    for (int s = 0; s < steps; s += kDepth) {
#pragma unroll
        for (int i = 0; i < kDepth; ++i)
            if (s + i < steps) {  // (the same in every wave)
                consume(ring[i]);
                load(ring[i]);
            }
    }
}

// ------------------------------------------------------------------------ more rows -----------
// The rows are split once into the workspace, as operands: hi halves of 32-row block b, chunk c
// (8 of the contraction, in a word's order) and row r at chunk (b * KC + c) * 32 + r, the lo
// halves a plane on; rows past M and the contraction past K are zeros.
constexpr int kThreads = 256;

// 8 rows a workgroup, 128 threads each; a thread's first kSplitKept chunks stay in registers
// between the row's exponent and its halves (4096 of the contraction).
constexpr int kSplitThreads = 1024, kSplitKept = 4;
__global__ __launch_bounds__(kSplitThreads) void q4_split_kernel(const float *__restrict__ x, float *__restrict__ ex,
                                                                 f16x8 *__restrict__ hi, f16x8 *__restrict__ lo, int M,
                                                                 int K, int KC) {
    __shared__ unsigned s_top[kSplitThreads / 64][8];
    const int tid = threadIdx.x, i = tid & 7, l = tid >> 3;
    constexpr int L = kSplitThreads / 8;
    const int r = blockIdx.x * 8 + i, nw = K / 8;
    const f32x4 *p = reinterpret_cast<const f32x4 *>(x + (size_t)min(r, M - 1) * K);
    const int have = r < M ? nw : 0;  // chunks of the row
    const f32x4 z4 = {0.0f, 0.0f, 0.0f, 0.0f};
    f32x4 keep[kSplitKept][2];
#pragma unroll
    for (int j = 0; j < kSplitKept; ++j) {
        const int c = l + j * L;
        keep[j][0] = c < have ? p[2 * c] : z4;
        keep[j][1] = c < have ? p[2 * c + 1] : z4;
    }
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < kSplitKept; ++j) top = max_bits(max_bits(top, keep[j][0]), keep[j][1]);
    for (int c = l + kSplitKept * L; c < have; c += L) top = max_bits(max_bits(top, p[2 * c]), p[2 * c + 1]);
#pragma unroll
    for (int d = 32; d >= 8; d >>= 1) {
        const unsigned o = __shfl_xor(top, d);
        top = o > top ? o : top;
    }
    if ((tid & 63) < 8) s_top[tid >> 6][i] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSplitThreads / 64; ++w) top = s_top[w][i] > top ? s_top[w][i] : top;
    const int e = row_exponent(top);
    if (l == 0) ex[r] = (float)e;
    auto put = [&](int c, f32x4 a, f32x4 b) {
        f16x8 h, o;
        split8(a, b, e, h, o);
        const size_t at = ((size_t)(r / 32) * KC + c) * 32 + r % 32;
        hi[at] = h;
        lo[at] = o;
    };
#pragma unroll
    for (int j = 0; j < kSplitKept; ++j)
        if (l + j * L < KC) put(l + j * L, keep[j][0], keep[j][1]);
    for (int c = l + kSplitKept * L; c < KC; c += L) put(c, c < have ? p[2 * c] : z4, c < have ? p[2 * c + 1] : z4);
}

// Workgroup tile: 32 MB WM rows x 32 NB WN features, WM x WN waves of MB x NB blocks of 32 x 32
// (v_mfma_f32_32x32x16_f16: A = x rows, lane (r, h): row r, chunk 2 step + h; B = codes, lane
// (n, h): feature n). In a unit of U = min(G, 64) of the contraction, lane half h takes the U / 2
// values h * U / 2 .. as U / 16 words, step j word j.
template <int G, bool ZERO, int MB, int NB, int WM, int WN>
__global__ __launch_bounds__(kThreads, 1) void q4_gemm_kernel(const f16x8 *__restrict__ hi,
                                                              const f16x8 *__restrict__ lo,
                                                              const float *__restrict__ ex, Segs segs, int M, int K,
                                                              int KC) {
    constexpr int U = G < 64 ? G : 64, W = U / 16;  // a unit, and its words (and steps) per lane
    constexpr int S = 64 / U;                       // units per 64-deep stage
    constexpr int BM = 32 * MB * WM;
    constexpr int CH = 8 * BM;                      // chunks of a stage's plane
    constexpr int NLD = 2 * CH / kThreads;
    __shared__ f16x8 lds[2][2 * CH];                // hi then lo: [block][chunk][row]
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int n = lane & 31, h = lane >> 5;
    const int mt = blockIdx.x / segs.total, u = blockIdx.x % segs.total;
    const Seg &sg = segs.seg[seg_of(segs, u)];
    const int m0 = mt * BM, n0 = (u - sg.first) * 32 * NB * WN + wn * 32 * NB;
    const int ngr = K / G, nw = K / 8;
    const int stages = (K + 63) / 64;

    f16x8 rx[NLD];
    auto load_x = [&](int st) {
#pragma unroll
        for (int i = 0; i < NLD; ++i) {
            const int c = tid + i * kThreads;
            const int at = c % CH;
            const f16x8 *p = c < CH ? hi : lo;
            rx[i] = p[((size_t)(m0 / 32 + at / 256) * KC + st * 8) * 32 + at % 256];
        }
    };
    auto store_x = [&](int buf) {
#pragma unroll
        for (int i = 0; i < NLD; ++i) lds[buf][tid + i * kThreads] = rx[i];
    };
    unsigned rw[2][NB][S][W];
    auto load_w = [&](int st, unsigned (&r)[NB][S][W]) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int o = min(n0 + 32 * b + n, sg.n - 1);
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const int k = min(st * 64 + s * U, K - U);  // (past K: against zeros of x)
                const uint32_t *p = sg.w + (size_t)o * nw + k / 8 + h * W;
                if constexpr (W == 4) {
                    const u32x4 v = *reinterpret_cast<const u32x4 *>(p);
#pragma unroll
                    for (int j = 0; j < 4; ++j) r[b][s][j] = v[j];
                } else {
                    const u32x2 v = *reinterpret_cast<const u32x2 *>(p);
                    r[b][s][0] = v[0];
                    r[b][s][1] = v[1];
                }
            }
        }
    };
    floatx16 acc[MB][NB] = {}, t[MB][NB] = {};
    auto compute = [&](int st, int buf, const unsigned (&r)[NB][S][W]) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int gr = min((st * 64 + s * U) / G, ngr - 1);
            Zero z[NB];
            float sc[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int o = min(n0 + 32 * b + n, sg.n - 1);
                z[b] = zero_of(ZERO ? sg.z[(size_t)o * ngr + gr] : 8u, 0);
                sc[b] = (float)sg.s[(size_t)o * ngr + gr];
            }
#pragma unroll
            for (int j = 0; j < W; ++j) {
                f16x8 ah[MB], al[MB];
#pragma unroll
                for (int a = 0; a < MB; ++a) {
                    const int at = ((wm * MB + a) * 8 + s * (U / 8) + h * W + j) * 32 + n;
                    ah[a] = lds[buf][at];
                    al[a] = lds[buf][CH + at];
                }
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const f16x8 w = unpack(r[b][s][j], z[b]);
#pragma unroll
                    for (int a = 0; a < MB; ++a) {
                        t[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[a], w, t[a][b], 0, 0, 0);
                        t[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[a], w, t[a][b], 0, 0, 0);
                    }
                }
            }
            // The group's sum is complete (group 128: after its second stage).
            if (G <= 64 || (st & 1) || st + 1 == stages) {
#pragma unroll
                for (int a = 0; a < MB; ++a)
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        acc[a][b] += t[a][b] * sc[b];
                        t[a][b] = floatx16{};
                    }
            }
        }
    };
    load_x(0);
    load_w(0, rw[0]);
    store_x(0);
    __syncthreads();
    for (int st = 0; st < stages; ++st) {
        if (st + 1 < stages) {
            load_x(st + 1);
            load_w(st + 1, rw[1]);
        }
        compute(st, st & 1, rw[0]);
        if (st + 1 < stages) {
            store_x((st & 1) ^ 1);
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int s = 0; s < S; ++s)
#pragma unroll
                    for (int j = 0; j < W; ++j) rw[0][b][s][j] = rw[1][b][s][j];
        }
        __syncthreads();
    }
    // Lane (n, h) holds feature n, rows 8 (r / 4) + 4 h + r % 4 of each block.
#pragma unroll
    for (int a = 0; a < MB; ++a)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int row = m0 + (wm * MB + a) * 32 + 8 * (r >> 2) + 4 * h + (r & 3);
            if (row >= M) continue;
            const int e = (int)ex[row];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int o = n0 + 32 * b + n;
                if (o < sg.n) sg.y[(size_t)row * sg.n + o] = ldexpf(acc[a][b][r], e);
            }
        }
}

constexpr size_t kGemvLds = 144 * 1024;  // of the 160 KB, beside the kernel's own arrays
constexpr size_t kGemvRows = 8;
size_t gemv_lds(size_t m, size_t K) { return (K + 127) / 128 * 16 * 2 * m * 16; }
bool gemv(size_t m, size_t K) { return m <= kGemvRows && gemv_lds(m, K) <= kGemvLds; }

size_t round_up(size_t x, size_t to) { return (x + to - 1) / to * to; }
constexpr size_t kRowPad = 128;

int number(Segs &s, int per) {
    int t = 0;
    for (int i = 0; i < s.nseg; ++i) {
        s.seg[i].first = t;
        t += (s.seg[i].n + per - 1) / per;
    }
    return s.total = t;
}

// Waves that share a tile: the fewest that give every wave slot (two workgroups on a CU) a tile.
template <int G, bool ZERO, bool VEC>
hipError_t launch_gemv(hipStream_t st, const float *x, const Segs &s, int m, int K) {
    static const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&q4_gemv_kernel<G, ZERO, VEC>),
                                                    hipFuncAttributeMaxDynamicSharedMemorySize, (int)kGemvLds);
    if (e != hipSuccess) return e;
    const int slots = 2 * eb::current_cu_count();
    int kw = 1;
    while (kw < kGemvWaves && s.total * kw < slots * kGemvWaves) kw *= 2;
    const int tiles = kGemvWaves / kw;  // a workgroup's at a time
    const int grid = std::min((s.total + tiles - 1) / tiles, slots);
    q4_gemv_kernel<G, ZERO, VEC><<<grid, kGemvThreads, gemv_lds(m, K), st>>>(x, s, m, K, kw);
    return hipSuccess;
}

template <int G, bool ZERO>
hipError_t launch(hipStream_t st, const float *x, Segs s, int m, int K, float *ws) {
    if (gemv(m, K)) {
        number(s, 16);
        bool vec = K % 128 == 0;
        for (int i = 0; i < s.nseg; ++i)
            vec = vec && ((reinterpret_cast<uintptr_t>(s.seg[i].s) | 2 * reinterpret_cast<uintptr_t>(s.seg[i].z)) & 7) == 0;
        return vec ? launch_gemv<G, ZERO, true>(st, x, s, m, K) : launch_gemv<G, ZERO, false>(st, x, s, m, K);
    }
    const size_t mp = round_up(m, kRowPad), kp = round_up(K, 64);
    f16x8 *hi = reinterpret_cast<f16x8 *>(ws + mp), *lo = hi + mp * kp / 8;
    q4_split_kernel<<<(unsigned)(mp / 8), kSplitThreads, 0, st>>>(x, ws, hi, lo, m, K, (int)(kp / 8));
    if (m <= 64) {
        number(s, 128);
        q4_gemm_kernel<G, ZERO, 1, 1, 1, 4>
            <<<(unsigned)((m + 31) / 32 * s.total), kThreads, 0, st>>>(hi, lo, ws, s, m, K, (int)(kp / 8));
    } else {
        number(s, 128);
        q4_gemm_kernel<G, ZERO, 2, 2, 2, 2>
            <<<(unsigned)((m + 127) / 128 * s.total), kThreads, 0, st>>>(hi, lo, ws, s, m, K, (int)(kp / 8));
    }
    return hipSuccess;
}

}  // namespace

namespace eb {

size_t linear_q4_workspace_floats(size_t m, size_t in_f) {
    if (m == 0 || in_f == 0 || gemv(m, in_f)) return 0;
    return round_up(m, kRowPad) * (1 + round_up(in_f, 64));
}

eb_status launch_linear_q4(hipStream_t st, const float *x, const Q4Weight *w, float *const *y, int nseg, size_t m,
                           float *ws) {
    Segs s{};
    for (int i = 0; i < nseg; ++i)
        if (w[i].out_f > 0)
            s.seg[s.nseg++] = Seg{w[i].w, reinterpret_cast<const _Float16 *>(w[i].scales), w[i].zeros, y[i],
                                  (int)w[i].out_f, 0};
    if (s.nseg == 0) return EB_OK;
    const int K = (int)w[0].in_f, M = (int)m;
    const bool zero = w[0].zeros != nullptr;
    hipError_t e = hipSuccess;
    switch (w[0].group) {
        case 32: e = zero ? launch<32, true>(st, x, s, M, K, ws) : launch<32, false>(st, x, s, M, K, ws); break;
        case 64: e = zero ? launch<64, true>(st, x, s, M, K, ws) : launch<64, false>(st, x, s, M, K, ws); break;
        default: e = zero ? launch<128, true>(st, x, s, M, K, ws) : launch<128, false>(st, x, s, M, K, ws); break;
    }
    if (e != hipSuccess) return hip_fail(e, "linear_q4 launch set-up");
    return check_launch("linear_q4");
}

}  // namespace eb
