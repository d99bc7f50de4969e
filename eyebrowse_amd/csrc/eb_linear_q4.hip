// Projections with 4-bit weights and group scales for gfx950:
//   y[i, o] = sum_g s[o, g] sum_{k in g} x[i, k] (q[o, k] - z[o, g])
// with x and y f32, q 4-bit codes, s half, z a byte (or 8).
//
// All forms run on the matrix cores. A code less its zero point is a whole number, exact in f16.
// An x row is scaled by a power of two (its largest magnitude lands in [2^14, 2^15)) and split
// into f16 halves hi + lo, 22 bits of it; each product is exact in f32. The sum over a group is
// accumulated apart, then scaled and added in f32, so that no scale is rounded to f16.
//
// Weights are packed once (q4_pack_kernel) into tiles of 16 features, cut into blocks of 128 of the
// contraction: 1 KiB of codes, which lane n + 16 g of a wave reads as 16 bytes: word j holds the
// 8 codes of feature n from k = 32 j + 8 g on. So a product of 32 of the contraction (word j of
// every lane) lies in one group whatever the group's size, a wave's load is 1 KiB of memory, and a
// tile is one run of it. Read in the [out, in] layout, a wave's load was 16 pieces of 64 bytes in 16
// rows, and as many lines again for scales and zero points: a head of 1024 x 151936 took 30 us (3.1
// TB/s) whatever its instructions. Scales and zero points follow, [tile][block][16][128 / group]
// each. The contraction is padded to whole blocks and the features to whole tiles, with zero scales.
//
// In a word, codes k0, k2, k4, k6 are the nibbles of the low half, k1, k3, k5, k7 of the high one.
// Unpacking gives four f16 pairs in order with nine instructions: (w & 0x000F000F) | 0x64006400 is
// the pair (1024 + k0, 1024 + k1), from which 1024 + z is subtracted; (w & 0x00F000F0) |
// 0x64006400 is (1024 + 16 k2, 1024 + 16 k3), times 1/16 less 64 + z; the same of w >> 8.
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

constexpr int kBlock = 128;       // of the contraction
constexpr int kTileBytes = 1024;  // codes of a block of a tile
constexpr int kFeatures = 16;     // of a tile

// A packed weight: its planes, and the output.
struct Seg {
    const uint8_t *w;  // [tiles][blocks][1024]
    const _Float16 *s; // [tiles][blocks][16][128 / group]
    const uint8_t *z;  // the same, or null
    float *y;
    int n;      // features
    int first;  // first work unit of the pair
};
struct Segs {
    Seg seg[eb::kLinearMaxSegs];
    int nseg, total;  // units of all pairs
};
// The pair of unit u, by selects on the kernel's arguments (an index that varies would load from
// memory, and wait for it, wherever it is used).
__device__ __forceinline__ Seg seg_at(const Segs &s, int u) {
    Seg r = s.seg[0];
#pragma unroll
    for (int j = 1; j < eb::kLinearMaxSegs; ++j)
        if (j < s.nseg && u >= s.seg[j].first) r = s.seg[j];
    return r;
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
    // (the constant in a register: and + or are then one instruction, which takes no literals)
    unsigned magic = 0x64006400u;
    asm("" : "+v"(magic));
    const unsigned v = w >> 8;
    const f16x2 a = __builtin_bit_cast(f16x2, (w & 0x000F000Fu) | magic) + z.low;
    const f16x2 b = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (w & 0x00F000F0u) | magic), sixteenth, z.high);
    const f16x2 c = __builtin_bit_cast(f16x2, (v & 0x000F000Fu) | magic) + z.low;
    const f16x2 d = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (v & 0x00F000F0u) | magic), sixteenth, z.high);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ float half_of(unsigned w, int i) {
    return (float)__builtin_bit_cast(_Float16, (unsigned short)(w >> (16 * i)));
}

// Scales and zero points of a feature in a block, NG = 128 / group of each.
template <int NG>
struct Scales {
    unsigned s[(NG + 1) / 2];
    unsigned z;
    __device__ __forceinline__ float scale(int i) const { return half_of(s[i / 2], i % 2); }
};

// Eight values of a row, scaled by 2^-e, as hi and lo halves.
__device__ __forceinline__ void split8(f32x4 a, f32x4 b, int e, f16x8 &hi, f16x8 &lo) {
    const float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
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

// ------------------------------------------------------------------------ packing -------------
// One workgroup per block of a tile.
constexpr int kPackThreads = 256;
__global__ __launch_bounds__(kPackThreads) void q4_pack_kernel(const uint32_t *__restrict__ w,
                                                               const uint16_t *__restrict__ s,
                                                               const uint8_t *__restrict__ z, uint32_t *__restrict__ pw,
                                                               uint16_t *__restrict__ ps, uint8_t *__restrict__ pz, int N,
                                                               int K, int G, int nb) {
    const size_t at = blockIdx.x;  // tile * nb + block
    const int tile = (int)(at / nb), b = (int)(at % nb), tid = threadIdx.x;
    const int ng = kBlock / G, ngr = K / G, nw = K / 8;
    {
        const int lane = tid / 4, j = tid % 4, n = lane % 16, g = lane / 16;
        const int o = tile * kFeatures + n, word = b * 16 + 4 * j + g;
        uint32_t v = 0, r = 0;
        if (o < N && word < nw) v = w[(size_t)o * nw + word];
#pragma unroll
        for (int i = 0; i < 8; ++i) r |= (v >> (4 * i) & 15u) << (16 * (i % 2) + 4 * (i / 2));
        pw[at * (kTileBytes / 4) + tid] = r;
    }
    if (tid < kFeatures * ng) {
        const int o = tile * kFeatures + tid / ng, gr = b * ng + tid % ng;
        const bool in = o < N && gr < ngr;
        ps[at * kFeatures * ng + tid] = in ? s[(size_t)o * ngr + gr] : (uint16_t)0;
        if (pz) pz[at * kFeatures * ng + tid] = in && z ? z[(size_t)o * ngr + gr] : (uint8_t)0;
    }
}

// ------------------------------------------------------------------------ up to 8 rows --------
// A wave takes tiles: B of v_mfma_f32_16x16x32_f16 is the 16 features' codes, A the x rows, hi halves
// in rows 0..7 and lo halves in rows 8..15, so that one product serves both. The rows' halves stay in
// LDS; a workgroup splits them once and then walks its tiles; kw waves share a tile's contraction.
// Bound by its weights' loads past some 30 MB, by the ramp (x's halves, the first loads) below: 131072
// features of 4096, group 128, 51 us (5.5 TB/s of weights; a plain read reaches 6.4, and 7.1 with
// non-temporal loads, which were not tried here); 151936 of 1024, group 32 with zero points, 21.3 to
// 22.1 (4.4); 14336 of 4096 11.1; 14335 of 4096, three rows, group 64 with zero points, 13.3; 4096 of
// 4096 5.9; 2048 of 1024 4.9.
constexpr int kGemvWaves = 8;
constexpr int kGemvThreads = kGemvWaves * 64;
constexpr int kDepth = 4;  // blocks of weights in flight per wave

template <int NG>
struct Block {
    unsigned w[4];
    Scales<NG> f;
};

template <int G, bool ZERO>
__global__ __launch_bounds__(kGemvThreads, 4) void q4_gemv_kernel(const float *__restrict__ x, Segs segs, int m, int K,
                                                                  int kw) {
    constexpr int NG = kBlock / G;
    using B = Block<NG>;
    extern __shared__ f16x8 lds[];  // [blocks * 16 chunks][2 m]: chunk c of row i: hi, then lo
    __shared__ unsigned s_top[kGemvWaves][8];
    __shared__ int s_exp[8];
    __shared__ float s_part[kGemvWaves][8][16];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int nb = (K + kBlock - 1) / kBlock;
    const int nw = K / 8;  // chunks of a row

    // This wave's walk: tiles t0, t0 + units, ..., of each `per` blocks from b0 on. Blocks past the
    // row's last and tiles past the last are walked too, against zeros of x and without a store:
    // the loop has no branch around a load, so that kDepth of them stay in flight, and the waves
    // that share a tile meet at its end, in barriers of the workgroup.
    const int units = (int)gridDim.x * (kGemvWaves / kw);
    const int t0 = (int)blockIdx.x * (kGemvWaves / kw) + wave / kw;
    const int per = (nb + kw - 1) / kw;
    const int b0 = wave % kw * per;
    const int steps = (segs.total + units - 1) / units * per;

    // The next block to load; buffer resources over its tile (over nothing past the last).
    B ring[kDepth];
    int lt = t0, lb = 0;
    __amdgpu_buffer_rsrc_t wres, sres, zres;
    auto enter = [&] {
        const Seg sg = seg_at(segs, lt);
        const size_t at = (size_t)(lt - sg.first) * nb;
        const int have = lt < segs.total ? nb : 0;
        wres = eb::make_rsrc(sg.w + at * kTileBytes, have * kTileBytes);
        sres = eb::make_rsrc(sg.s + at * (kFeatures * NG), have * kFeatures * NG * 2);
        if constexpr (ZERO) zres = eb::make_rsrc(sg.z + at * (kFeatures * NG), have * kFeatures * NG);
    };
    enter();
    auto load = [&](B &r) {
        // (whole offsets in the vector operand: the scalar one is outside the range check)
        const int b = __builtin_amdgcn_readfirstlane(b0 + lb);
        const u32x4 v = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(wres, kTileBytes * b + 16 * lane, 0, 0));
#pragma unroll
        for (int j = 0; j < 4; ++j) r.w[j] = v[j];
        if constexpr (NG == 4) {
            const u32x2 q = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(sres, 128 * b + 8 * n, 0, 0));
            r.f.s[0] = q[0];
            r.f.s[1] = q[1];
            if constexpr (ZERO) r.f.z = __builtin_amdgcn_raw_buffer_load_b32(zres, 64 * b + 4 * n, 0, 0);
        } else if constexpr (NG == 2) {
            r.f.s[0] = __builtin_amdgcn_raw_buffer_load_b32(sres, 64 * b + 4 * n, 0, 0);
            if constexpr (ZERO) r.f.z = (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(zres, 32 * b + 2 * n, 0, 0);
        } else {
            r.f.s[0] = (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(sres, 32 * b + 2 * n, 0, 0);
            if constexpr (ZERO) r.f.z = (unsigned char)__builtin_amdgcn_raw_buffer_load_b8(zres, 16 * b + n, 0, 0);
        }
        if (++lb == per) {
            lb = 0;
            lt += units;
            enter();
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
    if (tid < m) {
        unsigned top = 0;
#pragma unroll
        for (int w = 0; w < kGemvWaves; ++w) top = s_top[w][tid] > top ? s_top[w][tid] : top;
        s_exp[tid] = row_exponent(top);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (i >= m) break;
        const f32x4 *p = reinterpret_cast<const f32x4 *>(x + (size_t)i * K);
        const int e = s_exp[i];
        for (int c = tid; c < kw * per * 16; c += kGemvThreads) {
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
    const f16x8 *xa = lds + g * 2 * m + row;               // word j of lane group g is chunk 4 j + g
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    int ct = t0, cb = 0;
    auto finish = [&] {
        // Rows 4 g + r: hi sums in lanes g 0, 1, lo sums 32 lanes on.
        float v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = acc[r] + eb::lane_xor32(acc[r]);
        const Seg sg = seg_at(segs, ct);
        const int o = (ct - sg.first) * kFeatures + n;
        const bool store = ct < segs.total && o < sg.n;
        if (kw == 1) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (store && g < 2 && 4 * g + r < m)
                    sg.y[(size_t)(4 * g + r) * sg.n + o] = ldexpf(v[r], s_exp[4 * g + r]);
        } else {
            if (g < 2)
#pragma unroll
                for (int r = 0; r < 4; ++r) s_part[wave][4 * g + r][n] = v[r];
            __syncthreads();
            // The first of a tile's waves adds their sums: lane (n, g) rows g and g + 4.
            if (wave % kw == 0 && store)
                for (int i = g; i < m; i += 4) {
                    float t = 0.0f;
                    for (int w = 0; w < kw; ++w) t += s_part[wave + w][i][n];
                    sg.y[(size_t)i * sg.n + o] = ldexpf(t, s_exp[i]);
                }
            __syncthreads();
        }
        acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        ct += units;
    };
    auto consume = [&](const B &r) {
        const f16x8 *xb = xa + (size_t)(b0 + cb) * 16 * 2 * m;
        f16x8 xv[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) xv[j] = xb[4 * j * 2 * m];
        f32x4 t[NG];
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const Zero z = zero_of(ZERO ? r.f.z : 0x08080808u, i);
            t[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = i * (4 / NG); j < (i + 1) * (4 / NG); ++j)
                t[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xv[j], unpack(r.w[j], z), t[i], 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < NG; ++i) acc += t[i] * r.f.scale(i);
        if (++cb == per) {
            cb = 0;
            finish();
        }
    };
    for (int s = 0; s < steps; s += kDepth) {
#pragma unroll
        for (int i = 0; i < kDepth; ++i) {
            if (s + i >= steps) break;  // (the same in every wave)
            consume(ring[i]);
            load(ring[i]);
        }
    }
}

// ------------------------------------------------------------------------ more rows -----------
// The rows are split once into the workspace, as operands: hi halves of 32-row block b, chunk c
// (8 of the contraction, in a word's order) and row r at chunk (b * KC + c) * 32 + r, the lo
// halves a plane on; rows past M and the contraction past K are zeros.

// 8 rows a workgroup, 128 threads each; a thread's first kSplitKept chunks stay in registers
// between the row's exponent and its halves (4096 of the contraction). 1000 rows of 4096: 10 us, 33
// MB read and written; of few rows 8, the chain of a workgroup's loads.
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

// B of v_mfma_f32_32x32x16_f16 for 32 features (two tiles): lane (n, h) is lane n + 32 h, feature n.
// In a block, lane half h reads the 16 bytes of slots g = h and g = 2 + h of its feature: word j of
// slot g is chunk 4 j + g, so product (q, j) takes chunk 4 j + 2 q + h of x, and lies in group j of
// 128 / G.
template <int NG>
struct Wide {
    unsigned w[2][4];  // slot 2 q + h, word j
    Scales<NG> f;
};
template <int NG, bool ZERO>
__device__ __forceinline__ void load_wide(Wide<NG> &r, const Seg &sg, int tile, int b, int nb, int n, int h) {
    const size_t at = (size_t)tile * nb + b;
    const u32x4 *p = reinterpret_cast<const u32x4 *>(sg.w + at * kTileBytes) + (n & 15) + 16 * h;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const u32x4 v = p[32 * q];
#pragma unroll
        for (int j = 0; j < 4; ++j) r.w[q][j] = v[j];
    }
    const size_t f = at * kFeatures + (n & 15);
    if constexpr (NG == 4) {
        const u32x2 q = *reinterpret_cast<const u32x2 *>(sg.s + f * 4);
        r.f.s[0] = q[0];
        r.f.s[1] = q[1];
        if constexpr (ZERO) r.f.z = *reinterpret_cast<const unsigned *>(sg.z + f * 4);
    } else if constexpr (NG == 2) {
        r.f.s[0] = *reinterpret_cast<const unsigned *>(sg.s + f * 2);
        if constexpr (ZERO) r.f.z = *reinterpret_cast<const uint16_t *>(sg.z + f * 2);
    } else {
        r.f.s[0] = *reinterpret_cast<const uint16_t *>(sg.s + f);
        if constexpr (ZERO) r.f.z = sg.z[f];
    }
}

// Four KiB from src (this lane's 16 bytes of the first) to LDS byte address dst, which m0 holds for
// all of them. A wait state follows the write of m0 (inside an asm block the compiler adds none).
__device__ __forceinline__ void copy_4kib(unsigned dst, const void *src) {
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\t"
        "global_load_lds_dwordx4 %1, off offset:1024\n\tglobal_load_lds_dwordx4 %1, off offset:2048\n\t"
        "global_load_lds_dwordx4 %1, off offset:%2"
        :
        : "s"(dst), "v"(src), "n"(3 * 1024)
        : "memory", "m0");
}

// Workgroup tile: 128 rows x 128 features, two sets of 2 x 2 waves (64 x 64 each); a stage is a
// block of 128, whose slots 2 q + h of q = 0 are the first set's and of q = 1 the second's: two
// waves on every SIMD, each with whole tiles of registers, where a launch has about one workgroup
// per CU. The sets' sums meet in LDS at the end. x's halves are copied memory-to-LDS a stage ahead
// (64 KiB; a wave copies one plane of one 32-row block), and the weights loaded a stage ahead. All
// of a stage's loads are waited for at its start; the empty asm on the weights there keeps the
// compiler from waiting for them, and with them for the next stage's copies, at their first use.
// Bound by the products: 1000 rows of 4096 to 4096 features, group 128, 74 to 76 us for 67 GFLOP of
// halves (880 to 900 TFLOP/s; a library's f16 product of 8192^3 reaches 1134 here).
constexpr int kTileRows = 128, kTileCols = 128;
constexpr int kTileThreads = 512;
template <int G, bool ZERO>
__global__ __launch_bounds__(kTileThreads, 2) void q4_tile_kernel(const f16x8 *__restrict__ hi, const f16x8 *__restrict__ lo,
                                                                  const float *__restrict__ ex, Segs segs, int M, int K,
                                                                  int KC, float *__restrict__ parts) {
    constexpr int NG = kBlock / G;
    constexpr int CH = 16 * kTileRows;  // chunks of a stage's plane: [row block][chunk][row]
    extern __shared__ f16x8 lds[];      // [2][hi CH, lo CH]
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q = wave >> 2, wm = (wave >> 1) & 1, wn = wave & 1;
    const int n = lane & 31, h = lane >> 5;
    const int mt = blockIdx.x / segs.total, u = blockIdx.x % segs.total;
    const Seg sg = seg_at(segs, u);
    const int m0 = mt * kTileRows, n0 = (u - sg.first) * kTileCols + wn * 64;
    const int nb = (K + kBlock - 1) / kBlock;
    const int last = (sg.n + kFeatures - 1) / kFeatures - 1;
    const int st0 = (int)((long long)nb * blockIdx.y / gridDim.y), st1 = (int)((long long)nb * (blockIdx.y + 1) / gridDim.y);

    // This wave's copies: plane wave / 4, row block wave % 4, 8 KiB a stage.
    const f16x8 *src = (wave < 4 ? hi : lo) + (size_t)(m0 / 32 + wave % 4) * KC * 32 + lane;
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    const unsigned dst0 = __builtin_amdgcn_readfirstlane(lds0 + ((wave / 4) * CH + (wave % 4) * 512) * 16);
    auto copy_stage = [&](int st) {
        const unsigned dst = dst0 + (st & 1) * 2 * CH * 16;
        copy_4kib(dst, src + (size_t)st * 512);
        copy_4kib(dst + 4096, src + (size_t)st * 512 + 256);
    };
    // This set's half of a block: slot 2 q + h of both blocks of 32 features.
    struct Half {
        unsigned w[4];
        Scales<NG> f;
    };
    size_t tile_at[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) tile_at[b] = (size_t)min((n0 + 32 * b + n) / kFeatures, last) * nb;
    auto load_w = [&](int st, Half (&r)[2]) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const size_t at = tile_at[b] + st;
            const u32x4 v = reinterpret_cast<const u32x4 *>(sg.w + at * kTileBytes)[(n & 15) + 16 * (2 * q + h)];
#pragma unroll
            for (int j = 0; j < 4; ++j) r[b].w[j] = v[j];
            const size_t f = at * kFeatures + (n & 15);
            r[b].f.z = 0x08080808u;
            if constexpr (NG == 4) {
                const u32x2 s = *reinterpret_cast<const u32x2 *>(sg.s + f * 4);
                r[b].f.s[0] = s[0];
                r[b].f.s[1] = s[1];
                if constexpr (ZERO) r[b].f.z = *reinterpret_cast<const unsigned *>(sg.z + f * 4);
            } else if constexpr (NG == 2) {
                r[b].f.s[0] = *reinterpret_cast<const unsigned *>(sg.s + f * 2);
                if constexpr (ZERO) r[b].f.z = *reinterpret_cast<const uint16_t *>(sg.z + f * 2);
            } else {
                r[b].f.s[0] = *reinterpret_cast<const uint16_t *>(sg.s + f);
                if constexpr (ZERO) r[b].f.z = sg.z[f];
            }
        }
    };
    auto arrived = [&](Half (&r)[2]) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
            for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(r[b].w[j]));
#pragma unroll
            for (int i = 0; i < (NG + 1) / 2; ++i) asm volatile("" : "+v"(r[b].f.s[i]));
            if constexpr (ZERO) asm volatile("" : "+v"(r[b].f.z));
        }
    };
    floatx16 acc[2][2] = {};
    auto compute = [&](int buf, const Half (&r)[2]) {
        const f16x8 *xb = lds + buf * 2 * CH + (wm * 2 * 16 + 2 * q + h) * 32 + n;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            floatx16 t[2][2];
            f16x8 w[2];
#pragma unroll
            for (int j = i * (4 / NG); j < (i + 1) * (4 / NG); ++j) {
                f16x8 ah[2], al[2];
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    ah[a] = xb[(a * 16 + 4 * j) * 32];
                    al[a] = xb[CH + (a * 16 + 4 * j) * 32];
                }
#pragma unroll
                for (int b = 0; b < 2; ++b) w[b] = unpack(r[b].w[j], zero_of(ZERO ? r[b].f.z : 0x08080808u, i));
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int b = 0; b < 2; ++b)
                        t[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                            ah[a], w[b], j == i * (4 / NG) ? floatx16{} : t[a][b], 0, 0, 0);
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int b = 0; b < 2; ++b)
                        t[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[a], w[b], t[a][b], 0, 0, 0);
            }
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int b = 0; b < 2; ++b) acc[a][b] += t[a][b] * r[b].f.scale(i);
            // (one group's sums at a time: two groups' do not fit the registers)
            if constexpr (NG > 1) __builtin_amdgcn_sched_barrier(0);
        }
    };
    Half wa[2], wb[2];
    copy_stage(st0);
    load_w(st0, wa);
    auto stage = [&](int st, Half (&now)[2], Half (&next)[2]) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        arrived(now);
        __syncthreads();  // stage st is there, and nobody reads the other buffer any more
        if (st + 1 < st1) {
            copy_stage(st + 1);
            load_w(st + 1, next);
        }
        __builtin_amdgcn_sched_barrier(0);
        compute(st & 1, now);
    };
    for (int st = st0; st < st1; st += 2) {
        stage(st, wa, wb);
        if (st + 1 < st1) stage(st + 1, wb, wa);
    }
    // The sets' sums meet in LDS: each takes one of the two blocks of 32 rows.
    float *part = reinterpret_cast<float *>(lds);
    __syncthreads();
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const floatx16 give = q ? acc[0][b] : acc[1][b];
#pragma unroll
        for (int r = 0; r < 16; ++r) part[((wave * 2 + b) * 16 + r) * 64 + lane] = give[r];
    }
    __syncthreads();
    // Lane (n, h) holds feature n, rows 8 (r / 4) + 4 h + r % 4 of each block.
    const int mr = (wm * 2 + q) * 32;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const floatx16 keep = q ? acc[1][b] : acc[0][b];
        const int o = n0 + 32 * b + n;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int at = mr + 8 * (r >> 2) + 4 * h + (r & 3), row = m0 + at;
            const float v = keep[r] + part[(((wave ^ 4) * 2 + b) * 16 + r) * 64 + lane];
            if (row >= M) continue;
            if (gridDim.y > 1)
                parts[((size_t)blockIdx.y * gridDim.x + blockIdx.x) * kTileRows * kTileCols + at * kTileCols + wn * 64 +
                      32 * b + n] = v;
            else if (o < sg.n)
                sg.y[(size_t)row * sg.n + o] = ldexpf(v, (int)ex[row]);
        }
    }
}

// The sums of a contraction that several workgroups shared, in their order. A workgroup takes eight
// rows of a tile, a thread four features of one; up to kJoinBatch shares' sums are in flight: 4.7 us
// for eight shares of 128 x 4096 (17.5 with a load, and a wait, a share at a time).
constexpr int kJoinRows = 8, kJoinThreads = 256, kJoinBatch = 8;
__global__ __launch_bounds__(kJoinThreads) void q4_join_kernel(const float *__restrict__ parts,
                                                               const float *__restrict__ ex, Segs segs, int M, int tiles,
                                                               int shares) {
    const int t = blockIdx.x, mt = t / segs.total, u = t % segs.total;
    const Seg sg = seg_at(segs, u);
    const int at = (int)blockIdx.y * kJoinRows + threadIdx.x / 32, row = mt * kTileRows + at;
    const int col = 4 * (threadIdx.x % 32), o = (u - sg.first) * kTileCols + col;
    if (row >= M || o >= sg.n) return;
    const float *p = parts + (size_t)t * kTileRows * kTileCols + at * kTileCols + col;
    const size_t step = (size_t)tiles * kTileRows * kTileCols;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < shares; s += kJoinBatch) {
        f32x4 v[kJoinBatch];
#pragma unroll
        for (int i = 0; i < kJoinBatch; ++i)
            v[i] = *reinterpret_cast<const f32x4 *>(p + (size_t)min(s + i, shares - 1) * step);
#pragma unroll
        for (int i = 0; i < kJoinBatch; ++i)
            if (s + i < shares) sum += v[i];
    }
    const int e = (int)ex[row];
    float *y = sg.y + (size_t)row * sg.n + o;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (o + i < sg.n) y[i] = ldexpf(sum[i], e);
}

// Up to 32 rows: a workgroup takes them all and 32 features, its eight waves sharing the contraction
// (wave w blocks w, w + 8, ...); x's halves come from L2 straight into the products' registers, and
// the waves' sums meet in LDS.
constexpr int kSlimWaves = 8;
template <int G, bool ZERO>
__global__ __launch_bounds__(kSlimWaves * 64, 2) void q4_slim_kernel(const f16x8 *__restrict__ hi,
                                                                     const f16x8 *__restrict__ lo,
                                                                     const float *__restrict__ ex, Segs segs, int M, int K) {
    constexpr int NG = kBlock / G;
    __shared__ float part[kSlimWaves][16][64];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, h = lane >> 5;
    const Seg sg = seg_at(segs, (int)blockIdx.x);
    const int n0 = ((int)blockIdx.x - sg.first) * 32;
    const int nb = (K + kBlock - 1) / kBlock;
    const int last = (sg.n + kFeatures - 1) / kFeatures - 1;
    const int tile = min((n0 + n) / kFeatures, last);
    floatx16 acc = {};
    Wide<NG> r;
    if (wave < nb) load_wide<NG, ZERO>(r, sg, tile, wave, nb, n, h);
    for (int b = wave; b < nb; b += kSlimWaves) {
        Wide<NG> next = r;
        if (b + kSlimWaves < nb) load_wide<NG, ZERO>(next, sg, tile, b + kSlimWaves, nb, n, h);
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const Zero z = zero_of(ZERO ? r.f.z : 0x08080808u, i);
            floatx16 t = {};
#pragma unroll
            for (int j = i * (4 / NG); j < (i + 1) * (4 / NG); ++j)
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const f16x8 w = unpack(r.w[q][j], z);
                    const int at = (b * 16 + 4 * j + 2 * q + h) * 32 + n;
                    t = __builtin_amdgcn_mfma_f32_32x32x16_f16(hi[at], w, t, 0, 0, 0);
                    t = __builtin_amdgcn_mfma_f32_32x32x16_f16(lo[at], w, t, 0, 0, 0);
                }
            acc += t * r.f.scale(i);
        }
        r = next;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) part[wave][i][lane] = acc[i];
    __syncthreads();
    // Lane (n, h): feature n, rows 8 (i / 4) + 4 h + i % 4; wave w takes i = w, w + 8.
#pragma unroll
    for (int i = wave; i < 16; i += kSlimWaves) {
        const int row = 8 * (i >> 2) + 4 * h + (i & 3), o = n0 + n;
        float t = 0.0f;
#pragma unroll
        for (int w = 0; w < kSlimWaves; ++w) t += part[w][i][lane];
        if (row < M && o < sg.n) sg.y[(size_t)row * sg.n + o] = ldexpf(t, (int)ex[row]);
    }
}

constexpr size_t kGemvLds = 144 * 1024;  // of the 160 KB, beside the kernel's own arrays
constexpr size_t kGemvRows = 8;
// (the blocks rounded up to what kGemvWaves waves share)
size_t gemv_lds(size_t m, size_t K) {
    return ((K + kBlock - 1) / kBlock + kGemvWaves - 1) / kGemvWaves * kGemvWaves * 16 * 2 * m * 16;
}
bool gemv(size_t m, size_t K) { return m <= kGemvRows && gemv_lds(m, K) <= kGemvLds; }

size_t round_up(size_t x, size_t to) { return (x + to - 1) / to * to; }
constexpr size_t kRowPad = 128;

// Where the tiles are fewer than the CUs, workgroups share a tile's contraction, as many as the CUs
// hold (one each, by its LDS), of at least kMinStages blocks of 128; kMaxParts bounds their sums.
// 4096 to 4096 features: 500 rows (128 tiles) 64 us whole, 32 + 5 in two shares; 128 rows (32 tiles)
// 17.5 + 4.7 in eight.
constexpr int kMaxParts = 256, kMinStages = 2;
// Up to this many rows the slim kernel: 16 rows of 4096 to 4096 features 9.1 us, against 17.5 + 4.7
// in shared tiles; to 14336 features 15.2 against 36.7 + 5. With two blocks of rows (64) it took
// 21.9 and 38.8, as the tiles do, and 200 rows of group 64 60 (the whole call 71, 41 in tiles).
constexpr int kSlimRows = 32;

int number(Segs &s, int per) {
    int t = 0;
    for (int i = 0; i < s.nseg; ++i) {
        s.seg[i].first = t;
        t += (s.seg[i].n + per - 1) / per;
    }
    return s.total = t;
}

template <int G, bool ZERO>
hipError_t launch(hipStream_t st, const float *x, Segs s, int m, int K, float *ws) {
    const int cus = eb::current_cu_count();
    if (gemv(m, K)) {
        static const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&q4_gemv_kernel<G, ZERO>),
                                                        hipFuncAttributeMaxDynamicSharedMemorySize, (int)kGemvLds);
        if (e != hipSuccess) return e;
        // Waves that share a tile: the fewest that give every wave slot (two workgroups on a CU) one.
        number(s, kFeatures);
        const int slots = 2 * cus;
        int kw = 1;
        while (kw < kGemvWaves && s.total * kw < slots * kGemvWaves) kw *= 2;
        const int tiles = kGemvWaves / kw;  // a workgroup's at a time
        const int grid = std::min((s.total + tiles - 1) / tiles, slots);
        q4_gemv_kernel<G, ZERO><<<grid, kGemvThreads, gemv_lds(m, K), st>>>(x, s, m, K, kw);
        return hipSuccess;
    }
    const size_t mp = round_up(m, kRowPad), kp = round_up(K, kBlock);
    f16x8 *hi = reinterpret_cast<f16x8 *>(ws + mp), *lo = hi + mp * kp / 8;
    const int KC = (int)(kp / 8);
    q4_split_kernel<<<(unsigned)(mp / 8), kSplitThreads, 0, st>>>(x, ws, hi, lo, m, K, KC);
    if (m > kSlimRows) {
        constexpr size_t lds = 2 * 2 * 16 * kTileRows * 16;
        static const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&q4_tile_kernel<G, ZERO>),
                                                        hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
        const int tiles = (m + kTileRows - 1) / kTileRows * number(s, kTileCols);
        const int shares = std::max(1, std::min(std::min(cus, kMaxParts) / tiles, KC / 16 / kMinStages));
        float *parts = ws + mp * (1 + kp);
        q4_tile_kernel<G, ZERO><<<dim3((unsigned)tiles, (unsigned)shares), kTileThreads, lds, st>>>(hi, lo, ws, s, m, K, KC,
                                                                                                   parts);
        if (shares > 1)
            q4_join_kernel<<<dim3((unsigned)tiles, (std::min(m, kTileRows) + kJoinRows - 1) / kJoinRows), kJoinThreads, 0, st>>>(
                parts, ws, s, m, tiles, shares);
        return hipSuccess;
    }
    number(s, 32);
    q4_slim_kernel<G, ZERO><<<(unsigned)s.total, kSlimWaves * 64, 0, st>>>(hi, lo, ws, s, m, K);
    return hipSuccess;
}

}  // namespace

namespace eb {

size_t linear_q4_workspace_floats(size_t m, size_t in_f) {
    if (m == 0 || in_f == 0 || gemv(m, in_f)) return 0;
    const size_t parts = m > kSlimRows ? (size_t)kMaxParts * kTileRows * kTileCols : 0;
    return round_up(m, kRowPad) * (1 + round_up(in_f, kBlock)) + parts;
}

// Planes: codes | scales | zero points; each a whole number of 16 bytes.
size_t q4_packed_bytes(size_t in_f, size_t out_f, size_t group, bool zeros) {
    const size_t blocks = (out_f + kFeatures - 1) / kFeatures * ((in_f + kBlock - 1) / kBlock);
    return blocks * (kTileBytes + kFeatures * (kBlock / group) * (zeros ? 3 : 2));
}

eb_status launch_q4_pack(hipStream_t st, const uint32_t *w, const uint16_t *scales, const uint8_t *zeros, uint8_t *packed,
                         size_t in_f, size_t out_f, size_t group) {
    const size_t nb = (in_f + kBlock - 1) / kBlock, blocks = (out_f + kFeatures - 1) / kFeatures * nb;
    if (blocks == 0) return EB_OK;
    uint8_t *ps = packed + blocks * kTileBytes, *pz = ps + blocks * kFeatures * (kBlock / group) * 2;
    q4_pack_kernel<<<(unsigned)blocks, kPackThreads, 0, st>>>(w, scales, zeros, reinterpret_cast<uint32_t *>(packed),
                                                              reinterpret_cast<uint16_t *>(ps), zeros ? pz : nullptr,
                                                              (int)out_f, (int)in_f, (int)group, (int)nb);
    return check_launch("q4_pack");
}

eb_status launch_linear_q4(hipStream_t st, const float *x, const Q4Weight *w, float *const *y, int nseg, size_t m,
                           float *ws) {
    Segs s{};
    for (int i = 0; i < nseg; ++i) {
        if (w[i].out_f == 0) continue;
        const size_t blocks = (w[i].out_f + kFeatures - 1) / kFeatures * ((w[i].in_f + kBlock - 1) / kBlock);
        const uint8_t *ps = w[i].packed + blocks * kTileBytes;
        s.seg[s.nseg++] = Seg{w[i].packed, reinterpret_cast<const _Float16 *>(ps),
                              ps + blocks * kFeatures * (kBlock / w[i].group) * 2, y[i], (int)w[i].out_f, 0};
    }
    if (s.nseg == 0) return EB_OK;
    const int K = (int)w[0].in_f, M = (int)m;
    const bool zero = w[0].zeros;
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
