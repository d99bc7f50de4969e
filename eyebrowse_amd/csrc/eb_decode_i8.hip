// Attention of a few query rows over the block-scaled 8-bit cache (eb_cache_i8.h) for gfx950:
// a single token, with its cache append folded in, or a short run of rows (a draft to verify, a
// short next chunk). Split keys, then the log-sum-exp merge of the decode path.
//
//   o[c] = sum_j 2^(s_cj - m) v_j / sum_j 2^(s_cj - m),   s_cj = scale log2(e) q_c . k_j
//
// over the keys j that column c sees. A column is one query head of one row; the up to 16 columns
// of a workgroup share a KV head, so that every key row is read once for all of them.
//
// Grid hkv x nsub x nsplit, 4 waves. A tile is 16 keys at an aligned position, hence inside one
// block of the cache: its two scales are the same for the whole tile. Lane (n, g) is lane
// n + 16 g.
//  - Scores S[key][column] = K q^T on v_mfma_f32_16x16x32_f16. A: lane (n, g) holds 16 dims of
//    key n per 64-dim piece, straight from one 16-byte load, converted to f16 (exact: whole
//    numbers up to 128). B: column n's q as f16 high and low halves of q * scale * log2(e) scaled
//    by a power of two (its largest |q| in [2^13, 2^14)). Lane (n, g) then holds the scores of
//    keys 4g .. 4g + 3 for column n; the tile's K scale and the column's power of two come back
//    in one multiply.
//  - Online softmax with a reference m per column that moves only when a score exceeds it by
//    more than kSlack.
//  - O[column][dim] += P V on v_mfma_f32_16x16x32_f16: the 32 contracted indices are the 16 keys
//    twice, with the weights' high halves and their remainders, against the same V. A: lane
//    (n, g)'s own score registers. B: lane (n, g) loads HD/16 dims of keys 4g .. 4g + 3.
//    No lane exchange and no LDS between the products.
//  - The weights carry the tile's V scale: p * 2^(ev - u + 7), u a whole number per column (the
//    unit of its accumulators) that moves, with a rescale, when a term would exceed it by more
//    than the slack. So a block of large values beside blocks of small ones costs neither range
//    nor the small ones' precision where the large ones have no weight.
// The products sum in f32; the f16 pairs keep 22 bits of q and of the weights.
//
// Bound by the codes' loads in long caches (32 heads over 8 of 128, 131071 keys: 49.5 us with the
// merge, 5.4 TB/s, where a plain read reaches 6.4, and 7.1 with non-temporal loads, which were not
// tried here), by the instructions of a tile (about 220 a wave for 16 keys) beside the ramp below: 32767
// keys 21.4, 8191 keys (16 heads) 13.1, 1000 keys 9.5; 100 keys, one launch on 8 workgroups, 6.8: a
// chain of q, scores, softmax and output. So every first load is issued before the first wait.
// Sixteen columns read the cache once: 4 rows at 8192 keys 15.0 us, 16 rows (64 columns) 23.2.
//
// Fused append (one row): the split with the fewest tiles owns the token's block; no other split
// reads it. Its waves take the block's tiles first, loaded with q as any first tile. The workgroup
// then normalises and rotates the new K and V rows and writes their codes, and the tile that holds
// the new row gets it out of LDS; only where the exponent grew, and the block's earlier codes are
// written again, are its tiles loaded again. Tiles beyond two per wave are loaded after the append
// anyway. With more than 16 columns several workgroups would read the block, and the append is a
// launch of its own.
#include "eb_cache_i8.h"

#include <algorithm>

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kTile = 16;    // keys per tile
constexpr int kCols = 16;    // columns per workgroup
constexpr float kSlack = 8.0f;  // log2 units a score may exceed its reference by
constexpr float kNoUnit = -100000.0f;  // u before the first tile

template <int HD>
struct Shape {
    static constexpr int NC = HD / 32;   // 32-dim chunks of a key row
    static constexpr int KL = HD / 64;   // 16-byte K loads per lane and tile
    static constexpr int DV = HD / 16;   // V dims per lane and row
    static constexpr int VW = DV / 4;    // words per lane and V row
    static constexpr int QS = HD + 4;    // floats per LDS row (bank spread)
    // LDS (floats): q [kCols][QS], later the waves' accumulators [kWaves][ncol][QS]; then the new
    // rows [2][HD]; column exponents [kCols]; m and l [kCols][kWaves] each; the new rows' codes
    // [2][HD / 4 words]; their block's exponents before and after, [2][2].
    static constexpr size_t lds_floats(int ncol) {
        const int a = kCols * QS, b = kWaves * ncol * QS;
        return (size_t)(a > b ? a : b) + 2 * HD + kCols + 2 * kCols * kWaves + 2 * HD / 4 + 4;
    }
};

struct Args {
    const float *q;  // [rows, h, hd]
    eb::CacheI8 c;
    const float *knew, *vnew;  // [hkv, hd] (null: no append)
    float *o;                  // [rows, h, hd]
    float *part_acc, *part_ml;
    int h, g, rows, ncols;  // ncols: columns of a KV head, rows * g
    int pos0;               // position of row 0
    int window;             // 0: none
    int tile0, tiles;       // the tiles dealt to the splits: tile0 .. tile0 + tiles - 1
    int owner, tails;        // the append's split; its block's tiles, behind the others
    unsigned g_inv;          // 2^32 / g, rounded up (exact below 65536 columns; a call has 192 at most)
    int nsplit, block_log2;
    float scale_log2;
    bool prologue;
    const float *qn_w, *kn_w, *vn_w;
    float eps;
    const float *rcos, *rsin;
};

// Two codes as packed f16, exact: their bytes (the sign bit flipped, so 0..255) become the low
// bits of 1024 + byte, from which 1152 is subtracted. sel picks the bytes of w (0..3).
__device__ __forceinline__ unsigned codes_f16(unsigned flipped, bool high) {
    const unsigned b = __builtin_amdgcn_perm(0x64646464u, flipped, high ? 0x04030402u : 0x04010400u);
    const f16x2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    return __builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2, b) + off);
}

__device__ __forceinline__ unsigned pk_f16(float a, float b) {  // (rounded toward zero)
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(a, b));
}
__device__ __forceinline__ float f16_lo(unsigned w) {
    return (float)__builtin_bit_cast(_Float16, (unsigned short)(w & 0xFFFFu));
}
__device__ __forceinline__ float f16_hi(unsigned w) {
    return (float)__builtin_bit_cast(_Float16, (unsigned short)(w >> 16));
}

// First dim of lane group g's 8 dims in 32-dim chunk c: a 16-byte load holds 16 dims, the first 8
// in chunk 2C, the rest in chunk 2C + 1.
__device__ __forceinline__ int chunk_dim(int c, int g) { return 64 * (c / 2) + 16 * g + 8 * (c % 2); }

// hd: the rows' head dim, at most HD; what a lane reads past it (the next head's codes, or zeros
// past the cache) meets q's zeros in the scores and is not stored from the output.
template <int HD>
__global__ __launch_bounds__(kThreads, 2) void decode_i8_kernel(Args a, int hd) {
    using S = Shape<HD>;
    constexpr int NC = S::NC, KL = S::KL, DV = S::DV, VW = S::VW, QS = S::QS;
    extern __shared__ float smem[];
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15;
    const int g4 = lane >> 4;
    const int hkv = (int)a.c.hkv;
    const int kvh = blockIdx.x;
    const int col0 = (int)blockIdx.y * kCols;
    const int ncol = min(kCols, a.ncols - col0);
    const int split = blockIdx.z;
    const bool owner = a.knew != nullptr && split == a.owner;
    auto row_of = [&](int cc) { return a.g == 1 ? cc : (int)__umulhi((unsigned)cc, a.g_inv); };  // cc / g
    const int lds_rows = max(kCols, kWaves * ncol);
    float *s_q = smem;
    float *s_new = smem + lds_rows * QS;
    int *s_qe = reinterpret_cast<int *>(s_new + 2 * HD);
    float *s_m = reinterpret_cast<float *>(s_qe + kCols);
    float *s_l = s_m + kCols * kWaves;
    unsigned *s_code = reinterpret_cast<unsigned *>(s_l + kCols * kWaves);
    unsigned *s_e = s_code + 2 * (HD / 4);

    // ---- tile loads ------------------------------------------------------------------------
    const int row_bytes = hkv * hd;
    const int end = a.pos0 + a.rows;  // keys held
    const int kvo = n * row_bytes + 16 * g4;
    const int vvo = 4 * g4 * row_bytes + DV * n;
    const uint8_t *kbase = a.c.k + (size_t)kvh * hd, *vbase = a.c.v + (size_t)kvh * hd;
    struct Tile {
        unsigned k[KL][4], v[4][VW];
        unsigned ek, ev;
    };
    // Tile t of the cache; one at or past the last key reads zeros and touches no memory.
    auto load_tile = [&](int t, Tile &x) {
        const int r0 = t * kTile;
        const int left = min(end - r0, kTile);
        const int nbytes = left > 0 ? (left - 1) * row_bytes + hd : 0;
        const size_t off = left > 0 ? (size_t)r0 * row_bytes : 0;
        const __amdgpu_buffer_rsrc_t kres = eb::make_rsrc(kbase + off, nbytes);
        const __amdgpu_buffer_rsrc_t vres = eb::make_rsrc(vbase + off, nbytes);
#pragma unroll
        for (int c = 0; c < KL; ++c) {
            const u32x4 w = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(kres, kvo + 64 * c, 0, 0));
#pragma unroll
            for (int i = 0; i < 4; ++i) x.k[c][i] = w[i];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int vo = vvo + r * row_bytes;
            if constexpr (VW == 4) {
                const u32x4 w = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(vres, vo, 0, 0));
#pragma unroll
                for (int i = 0; i < 4; ++i) x.v[r][i] = w[i];
            } else if constexpr (VW == 2) {
                const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(vres, vo, 0, 0));
                x.v[r][0] = w[0];
                x.v[r][1] = w[1];
            } else {
                x.v[r][0] = __builtin_amdgcn_raw_buffer_load_b32(vres, vo, 0, 0);
            }
        }
        const size_t b = left > 0 ? (size_t)(r0 >> a.block_log2) * hkv + kvh : 0;
        x.ek = a.c.ks[b];
        x.ev = a.c.vs[b];
    };
    // This wave's tiles (all waves and splits together walk one stretch of the cache). The owner's
    // first ones are the new token's block, right behind that stretch.
    const int stretch = a.tile0 + a.tiles, stride = kWaves * a.nsplit;
    const int first_tile = a.tile0 + wave * a.nsplit + split;
    bool in_tail = owner && wave < a.tails;
    int next = in_tail ? stretch + wave : first_tile;
    // The next tile, or one past the last key; then one further.
    auto advance = [&] {
        const int t = in_tail || next < stretch ? next : INT_MAX / kTile;
        const int up = next + (in_tail ? kWaves : stride);
        const bool back = in_tail && up >= stretch + a.tails;
        next = back ? first_tile : min(up, INT_MAX / kTile);
        in_tail = in_tail && !back;
        return t;
    };

    // ---- every first load at once: q, the new rows, what transforms them, two tiles ------------
    // Wave w takes columns w, w + 4, ... and, of the owner, wave 0 the new K row and wave 1 the new
    // V row. A lane owns the dim pairs (p, p + hd/2), so that RMSNorm and RoPE never read another
    // lane's dims. What is absent reads as zeros and is not used.
    constexpr int NP = (HD / 2 + 63) / 64, NJ = kCols / kWaves;
    const int half = hd / 2;
    const bool newrow = owner && wave < 2;
    float x1[NJ + 1][NP], x2[NJ + 1][NP], qw1[NP], qw2[NP], nw1[NP], nw2[NP], cs[NP], sn[NP];
    const float *nw = wave ? a.vn_w : a.kn_w;
    unsigned old_e = 0;
    {
        const int none = 0x7FFFFFF0;
        const auto qres = eb::make_rsrc(a.q, a.rows * a.h * hd * 4);
        const auto nres = eb::make_rsrc((wave ? a.vnew : a.knew) + (size_t)kvh * hd, newrow ? hd * 4 : 0);
        const auto qwres = eb::make_rsrc(a.qn_w, a.prologue && a.qn_w ? hd * 4 : 0);
        const auto nwres = eb::make_rsrc(nw, newrow && a.prologue && nw ? hd * 4 : 0);
        const size_t trow = (size_t)a.pos0 * half;
        const bool rope = a.prologue && a.rcos;
        const auto cres = eb::make_rsrc(a.rcos + trow, rope ? half * 4 : 0);
        const auto sres = eb::make_rsrc(a.rsin + trow, rope ? half * 4 : 0);
        auto get = [&](__amdgpu_buffer_rsrc_t r, int vo) {
            return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, vo, 0, 0));
        };
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int p = lane + 64 * i;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int cc = col0 + j * kWaves + wave, row = row_of(cc);
                const int at = (row * a.h + kvh * a.g + cc - row * a.g) * hd * 4;
                const bool have = j * kWaves + wave < ncol && p < half;
                x1[j][i] = get(qres, have ? at + 4 * p : none);
                x2[j][i] = get(qres, have ? at + 4 * (p + half) : none);
            }
            const int v1 = p < half ? 4 * p : none, v2 = p < half ? 4 * (p + half) : none;
            x1[NJ][i] = get(nres, v1);
            x2[NJ][i] = get(nres, v2);
            qw1[i] = get(qwres, v1);
            qw2[i] = get(qwres, v2);
            nw1[i] = get(nwres, v1);
            nw2[i] = get(nwres, v2);
            cs[i] = get(cres, v1);
            sn[i] = get(sres, v1);
        }
        old_e = (wave ? a.c.vs : a.c.ks)[(size_t)(a.pos0 >> a.block_log2) * hkv + kvh];
    }
    Tile ta, tb;
    int na = advance(), nb = advance();
    load_tile(na, ta);
    load_tile(nb, tb);

    // RMSNorm (x * (1 / sqrt(mean x^2 + eps)) * w), then RoPE, of a row's pairs.
    auto transform = [&](float (&y1)[NP], float (&y2)[NP], bool norm, const float (&w1)[NP], const float (&w2)[NP],
                         bool rope) {
        if (norm) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < NP; ++i) ss += y1[i] * y1[i] + y2[i] * y2[i];
            ss = eb::class_reduce<1, false>(ss);
            const float inv = 1.0f / sqrtf(ss / (float)hd + a.eps);
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                y1[i] = y1[i] * inv * w1[i];
                y2[i] = y2[i] * inv * w2[i];
            }
        }
        if (rope) {  // without fused multiply-adds as the row pass
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const float z1 = __fsub_rn(__fmul_rn(y1[i], cs[i]), __fmul_rn(y2[i], sn[i]));
                y2[i] = __fadd_rn(__fmul_rn(y2[i], cs[i]), __fmul_rn(y1[i], sn[i]));
                y1[i] = z1;
            }
        }
    };
    const bool rope = a.prologue && a.rcos;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        const int c = j * kWaves + wave;
        if (c < ncol) {  // (uniform) q * scale * log2(e), then the column's power of two
            transform(x1[j], x2[j], a.prologue && a.qn_w, qw1, qw2, rope);
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                x1[j][i] *= a.scale_log2;
                x2[j][i] *= a.scale_log2;
                top = fmaxf(top, fmaxf(fabsf(x1[j][i]), fabsf(x2[j][i])));
            }
            top = eb::class_reduce<1, true>(top);
            int ex = 0;
            if (top > 0.0f && top <= 3.0e38f) {
                frexpf(top, &ex);
                ex = 14 - ex;
            }
            if (lane == 0) s_qe[c] = -ex;
            float *x = s_q + c * QS;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int p = lane + 64 * i;
                if (p < half) {
                    x[p] = ldexpf(x1[j][i], ex);
                    x[p + half] = ldexpf(x2[j][i], ex);
                }
            }
            for (int p = hd + lane; p < HD; p += 64) x[p] = 0.0f;
        }
    }

    // ---- the append ---------------------------------------------------------------------------
    if (newrow) {  // wave 0: K, wave 1: V
        transform(x1[NJ], x2[NJ], a.prologue && nw, nw1, nw2, rope && wave == 0);
        uint8_t *codes = (wave ? a.c.v : a.c.k) + (size_t)kvh * hd;
        uint8_t *exps = wave ? a.c.vs : a.c.ks;
        float *x = s_new + wave * HD;
        const int b = a.pos0 >> a.block_log2, first = b << a.block_log2, lead = a.pos0 - first;
        if (!lead) old_e = 0;
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int p = lane + 64 * i;
            if (p < half) {
                x[p] = x1[NJ][i];
                x[p + half] = x2[NJ][i];
            }
            const unsigned u1 = eb::magnitude_bits(x1[NJ][i]), u2 = eb::magnitude_bits(x2[NJ][i]);
            top = p < half ? max(top, max(u1, u2)) : top;
        }
#pragma unroll
        for (int m = 32; m > 0; m >>= 1) top = max(top, __shfl_xor(top, m));
        unsigned e = eb::i8_exponent(top);
        if (lead) e = eb::i8_join(old_e, e);
        const int d = 4 * lane;
        if (d < hd) {
            const f32x4 y = *reinterpret_cast<const f32x4 *>(x + d);  // (this wave's own row)
            unsigned w = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) w |= eb::i8_code(y[i], e) << (8 * i);
            *reinterpret_cast<unsigned *>(codes + (size_t)a.pos0 * row_bytes + d) = w;
            s_code[wave * (HD / 4) + lane] = w;
        }
        if (lead && e != old_e && e != eb::kNanExponent) {
            const int per_row = hd / 4;
            for (int i = lane; i < lead * per_row; i += 64) {
                unsigned *p = reinterpret_cast<unsigned *>(codes + (size_t)(first + i / per_row) * row_bytes +
                                                           4 * (i % per_row));
                *p = eb::i8_recode(*p, old_e, e);
            }
        }
        if (lane == 0) {
            exps[(size_t)b * hkv + kvh] = (uint8_t)e;
            s_e[2 * wave] = lead ? old_e : e;
            s_e[2 * wave + 1] = e;
        }
    }
    if (owner) __threadfence_block();
    __syncthreads();
    if (owner) {  // (uniform over the workgroup)
        const unsigned k0 = s_e[0], k1 = s_e[1], v0 = s_e[2], v1 = s_e[3];
        auto appended = [&](int t, Tile &x) {
            if (t < stretch || t >= stretch + a.tails) return;
            if (k0 != k1 || v0 != v1) {
                load_tile(t, x);
                return;
            }
            const int at = a.pos0 - t * kTile;  // the new row, if in this tile
#pragma unroll
            for (int c = 0; c < KL; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n == at) x.k[c][i] = s_code[16 * c + 4 * g4 + i];
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int i = 0; i < VW; ++i)
                    if (4 * g4 + r == at) x.v[r][i] = s_code[HD / 4 + VW * n + i];
            x.ek = k1;
            x.ev = v1;
        };
        appended(na, ta);
        appended(nb, tb);
    }

    // ---- operands and state -------------------------------------------------------------------
    const int own = min(n, ncol - 1);  // this lane's column (the last one, repeated, past ncol)
    f16x8 qh[NC], ql[NC];
    const int qe = s_qe[own];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const float *src = s_q + own * QS + chunk_dim(c, g4);
        const f32x4 v0 = *reinterpret_cast<const f32x4 *>(src);
        const f32x4 v1 = *reinterpret_cast<const f32x4 *>(src + 4);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float v = j < 4 ? v0[j % 4] : v1[j % 4];
            const _Float16 hi = (_Float16)v;
            qh[c][j] = hi;
            ql[c][j] = (_Float16)(v - (float)hi);
        }
    }
    const int my_pos = a.pos0 + row_of(col0 + own);  // the column's last key
    const int my_first = a.window > 0 ? my_pos - a.window + 1 : 0;  // and its first
    // Tiles wholly inside every column's keys need no mask.
    const int safe_lo = a.window > 0 ? end - a.window : 0, safe_hi = a.pos0;
    f32x4 acc[DV];
#pragma unroll
    for (int e = 0; e < DV; ++e) acc[e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f, u = kNoUnit;  // per lane: of its own column

    auto consume = [&](int t, const Tile &x) {
        const int k0 = t * kTile;
        if (k0 >= end) return;  // (uniform)
        f32x4 s1 = {0.0f, 0.0f, 0.0f, 0.0f}, s2 = s1;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const unsigned w0 = x.k[c / 2][2 * (c % 2)] ^ 0x80808080u;
            const unsigned w1 = x.k[c / 2][2 * (c % 2) + 1] ^ 0x80808080u;
            const f16x8 kk = __builtin_bit_cast(f16x8, u32x4{codes_f16(w0, false), codes_f16(w0, true),
                                                             codes_f16(w1, false), codes_f16(w1, true)});
            s1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, qh[c], s1, 0, 0, 0);
            s2 = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, ql[c], s2, 0, 0, 0);
        }
        const float cs = eb::i8_scale(x.ek, qe);
        float sc[4], w[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[r] = (s1[r] + s2[r]) * cs;
        const bool edge = k0 < safe_lo || k0 + kTile - 1 > safe_hi;  // (uniform)
        if (edge) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int key = k0 + 4 * g4 + r;
                if (key > my_pos || key < my_first) sc[r] = -INFINITY;
            }
        }
        // A score above m + slack moves m; a term above 2^(u + slack) in V's units moves u (but
        // weights below 2^-126 are nothing, whatever their V's scale).
        const float ev = (float)((int)x.ev - 127);
        const float top = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
        const float over = top - m;
        if (__builtin_amdgcn_ballot_w64(over > fminf(kSlack, fmaxf(u + kSlack - ev, -126.0f)) ||
                                        (m == -INFINITY && top > -INFINITY)) != 0) {
            float t1 = fmaxf(top, eb::lane_xor16(top));
            t1 = fmaxf(t1, eb::lane_xor32(t1));  // the column's largest score in the tile
            const float mn = m == -INFINITY || t1 > m + kSlack ? t1 : m;
            const float d = mn == m ? 0.0f : mn - m;  // (infinite at the column's first keys)
            const float ub = d < 1.0e6f ? u - floorf(d) : kNoUnit;
            const float x1 = ceilf(t1 - mn);
            const float un = x1 > -126.0f && x1 + ev > ub + kSlack ? x1 + ev : ub;
            const float f = d < 1.0e6f ? eb::fast_exp2((u - un) - d) : 0.0f;
            l *= d < 1.0e6f ? eb::fast_exp2(-d) : 0.0f;
            m = mn;
            u = un;
            // the accumulators' columns are 4 g4 + r: their factors from those columns' lanes
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float fr = __shfl(f, 4 * g4 + r);
#pragma unroll
                for (int e = 0; e < DV; ++e) acc[e][r] *= fr;
            }
        }
        const float mref = m == -INFINITY ? 0.0f : m;
        const float vs = x.ev == eb::kNanExponent ? __builtin_nanf("") : ldexpf(1.0f, (int)fminf(ev - u + 7.0f, 126.0f));
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float p = eb::fast_exp2(sc[r] - mref);
            l += p;
            w[r] = p * vs;
        }
        if (edge) {  // (a NaN scale does not reach keys that the column does not see)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (sc[r] == -INFINITY) w[r] = 0.0f;
        }
        const unsigned h01 = pk_f16(w[0], w[1]), h23 = pk_f16(w[2], w[3]);
        const unsigned l01 = pk_f16(w[0] - f16_lo(h01), w[1] - f16_hi(h01));
        const unsigned l23 = pk_f16(w[2] - f16_lo(h23), w[3] - f16_hi(h23));
        const f16x8 pp = __builtin_bit_cast(f16x8, u32x4{h01, h23, l01, l23});
        unsigned vx[4][VW];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < VW; ++i) vx[r][i] = x.v[r][i] ^ 0x80808080u;
#pragma unroll
        for (int e = 0; e < DV; e += 2) {
            // bytes e, e + 1 of rows 0, 1 (and 2, 3) as [r0.e, r1.e, r0.e+1, r1.e+1]
            const unsigned k = (unsigned)(e % 4);
            const unsigned sel = k | (4u + k) << 8 | (k + 1u) << 16 | (5u + k) << 24;
            const unsigned b01 = __builtin_amdgcn_perm(vx[1][e / 4], vx[0][e / 4], sel);
            const unsigned b23 = __builtin_amdgcn_perm(vx[3][e / 4], vx[2][e / 4], sel);
            const unsigned c0 = codes_f16(b01, false), c1 = codes_f16(b23, false);
            const unsigned d0 = codes_f16(b01, true), d1 = codes_f16(b23, true);
            acc[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pp, __builtin_bit_cast(f16x8, u32x4{c0, c1, c0, c1}),
                                                            acc[e], 0, 0, 0);
            acc[e + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                pp, __builtin_bit_cast(f16x8, u32x4{d0, d1, d0, d1}), acc[e + 1], 0, 0, 0);
        }
    };

    // ---- the tiles, in pairs, each buffer refilled once consumed --------------------------------
    const int mine = a.tiles > split ? (a.tiles - split + a.nsplit - 1) / a.nsplit : 0;
    const int steps = (mine + kWaves - 1) / kWaves + (owner ? (a.tails + kWaves - 1) / kWaves : 0);
    for (int i = 0; i < steps; i += 2) {
        consume(na, ta);
        na = advance();
        load_tile(na, ta);
        if (i + 1 < steps) consume(nb, tb);
        nb = advance();
        load_tile(nb, tb);
    }

    // ---- the waves' states meet in LDS ----------------------------------------------------------
    l += eb::lane_xor16(l);
    l += eb::lane_xor32(l);
    __syncthreads();  // (q's rows are read no more)
    float *s_acc = smem + wave * ncol * QS;
    if (g4 == 0 && n < ncol) {
        s_m[n * kWaves + wave] = m;
        s_l[n * kWaves + wave] = l;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int c = 4 * g4 + r;
        const float back = ldexpf(1.0f, (int)fmaxf(__shfl(u, c) - 7.0f, -1000.0f));
        if (c < ncol) {
#pragma unroll
            for (int e = 0; e < DV; e += 4)
                *reinterpret_cast<f32x4 *>(s_acc + c * QS + DV * n + e) =
                    f32x4{acc[e][r] * back, acc[e + 1][r] * back, acc[e + 2][r] * back, acc[e + 3][r] * back};
        }
    }
    __syncthreads();
    for (int i = tid; i < ncol * (HD / 4); i += kThreads) {
        const int c = i / (HD / 4), d = 4 * (i % (HD / 4));
        if (d >= hd) continue;
        const f32x4 m4 = *reinterpret_cast<const f32x4 *>(s_m + c * kWaves);
        const f32x4 l4 = *reinterpret_cast<const f32x4 *>(s_l + c * kWaves);
        const float M = fmaxf(fmaxf(m4.x, m4.y), fmaxf(m4.z, m4.w));
        const float mref = M == -INFINITY ? 0.0f : M;
        f32x4 A = {0.0f, 0.0f, 0.0f, 0.0f};
        float L = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = eb::fast_exp2(m4[w] - mref);
            A += f * *reinterpret_cast<const f32x4 *>(smem + (w * ncol + c) * QS + d);
            L += f * l4[w];
        }
        const int cc = col0 + c, row = row_of(cc);
        const size_t at = (size_t)row * a.h + kvh * a.g + cc - row * a.g;
        if (a.nsplit == 1) {
            *reinterpret_cast<f32x4 *>(a.o + at * hd + d) = A / L;
        } else {
            const size_t slot = (size_t)split * a.rows * a.h + at;
            *reinterpret_cast<f32x4 *>(a.part_acc + slot * hd + d) = A;
            if (d == 0) {
                a.part_ml[slot * 2 + 0] = M;
                a.part_ml[slot * 2 + 1] = L;
            }
        }
    }
}

struct Plan {
    int nsub, nsplit, tile0, tiles, tails;
    bool fused;
};

// Splits: enough workgroups for two on every CU (32767 keys 21.1 us; for three 22.0, for four 25.3:
// a later workgroup's ramp), each wave with at least one tile; fewer than
// kMinSplitKeys keys stay in one workgroup (a second launch costs more than the split saves).
constexpr size_t kMinSplitKeys = 128;
constexpr int kWgsPerCu = 2;
constexpr size_t kMaxSplits = 256;
Plan plan_of(size_t h, size_t hkv, size_t pos0, size_t rows, size_t block, size_t window, bool append,
             int cu_count) {
    Plan p{};
    const size_t cols = rows * (h / hkv);
    p.nsub = (int)((cols + kCols - 1) / kCols);
    p.fused = append && p.nsub == 1;
    const size_t end = pos0 + rows;
    const size_t first = window > 0 && pos0 + 1 > window ? pos0 + 1 - window : 0;
    size_t stop = (end + kTile - 1) / kTile;
    p.tile0 = (int)(first / kTile);
    if (p.fused) {
        const size_t b0 = std::max(pos0 / block * block / kTile, (size_t)p.tile0);
        p.tails = (int)(stop - b0);
        stop = b0;
    }
    p.tiles = (int)(stop - p.tile0);
    size_t nsplit = std::max<size_t>(1, (size_t)cu_count * kWgsPerCu / (hkv * p.nsub));
    nsplit = std::min(nsplit, std::max<size_t>(1, (size_t)p.tiles / kWaves));
    nsplit = std::min(nsplit, kMaxSplits);
    if (end - first < kMinSplitKeys) nsplit = 1;
    p.nsplit = (int)nsplit;
    return p;
}

template <int HD>
hipError_t launch(hipStream_t st, const Args &a, const Plan &p, size_t hd) {
    const size_t lds = Shape<HD>::lds_floats(std::min(kCols, a.ncols)) * sizeof(float);
    static_assert(Shape<HD>::lds_floats(kCols) * sizeof(float) <= 80 * 1024, "two workgroups per CU");
    if (lds > 64 * 1024) {
        static const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&decode_i8_kernel<HD>),
                                                        hipFuncAttributeMaxDynamicSharedMemorySize, 80 * 1024);
        if (e != hipSuccess) return e;
    }
    decode_i8_kernel<HD><<<dim3((unsigned)a.c.hkv, (unsigned)p.nsub, (unsigned)p.nsplit), kThreads, lds, st>>>(a, (int)hd);
    return hipSuccess;
}

}  // namespace

namespace eb {

// Workspace (floats): part_acc [nsplit * rows * h * hd], part_ml [nsplit * rows * h * 2]; a
// window only lowers the splits.
size_t decode_i8_workspace_floats(size_t h, size_t hkv, size_t pos0, size_t rows, size_t hd, size_t block,
                                  int cu_count) {
    size_t n = 0;
    for (int append = 0; append < 2; ++append) {
        const Plan p = plan_of(h, hkv, pos0, rows, block, 0, append && rows == 1, cu_count);
        if (p.nsplit > 1) n = std::max(n, (size_t)p.nsplit * rows * h * (hd + 2));
    }
    return n;
}

eb_status launch_attn_decode_i8(hipStream_t st, const float *q, const CacheI8 &c, const float *knew,
                                const float *vnew, float *o, size_t h, size_t pos0, size_t rows, float scale,
                                size_t window, float *ws, size_t ws_floats, int cu_count,
                                const DecodePrologue *pro) {
    const Plan p = plan_of(h, c.hkv, pos0, rows, c.block, window, knew != nullptr, cu_count);
    if (knew && !p.fused) {
        if (pro) return fail(EB_OTHER, "attn_decode_i8: more than %d heads per KV head need the row pass", kCols);
        const eb_status s = launch_kv_write_i8(st, c, knew, vnew, pos0, 1);
        if (s != EB_OK) return s;
    }
    const size_t need = p.nsplit > 1 ? (size_t)p.nsplit * rows * h * (c.hd + 2) : 0;
    if (need > 0 && (!ws || ws_floats < need))
        return fail(EB_SHAPE_MISMATCH, "attn_decode_i8: workspace holds %zu floats, needs %zu", ws_floats, need);
    Args a{};
    a.q = q;
    a.c = c;
    a.knew = p.fused ? knew : nullptr;
    a.vnew = p.fused ? vnew : nullptr;
    a.o = o;
    a.part_acc = ws;
    a.part_ml = ws ? ws + (size_t)p.nsplit * rows * h * c.hd : nullptr;
    a.h = (int)h;
    a.g = (int)(h / c.hkv);
    a.g_inv = (unsigned)((((uint64_t)1 << 32) + a.g - 1) / a.g);
    a.rows = (int)rows;
    a.ncols = (int)(rows * (h / c.hkv));
    a.pos0 = (int)pos0;
    a.window = (int)std::min<size_t>(window, INT_MAX);
    a.tile0 = p.tile0;
    a.tiles = p.tiles;
    a.owner = p.tiles % p.nsplit;  // (the first split that has one tile less, if any)
    a.tails = p.tails;
    a.nsplit = p.nsplit;
    while ((size_t)1 << a.block_log2 < c.block) ++a.block_log2;
    a.scale_log2 = scale * kLog2e;
    if (pro) {
        a.prologue = true;
        a.qn_w = pro->q_norm;
        a.kn_w = pro->k_norm;
        a.vn_w = pro->v_norm;
        a.eps = pro->eps;
        a.rcos = pro->rope_cos;
        a.rsin = pro->rope_sin;
    }
    const hipError_t e = c.hd <= 64    ? launch<64>(st, a, p, c.hd)
                         : c.hd <= 128 ? launch<128>(st, a, p, c.hd)
                                       : launch<256>(st, a, p, c.hd);
    if (e != hipSuccess) return hip_fail(e, "attn_decode_i8 launch set-up");
    eb_status s = check_launch("attn_decode_i8");
    if (s != EB_OK || p.nsplit == 1) return s;
    return launch_decode_merge(st, a.part_acc, a.part_ml, o, rows * h, c.hkv, c.hd, p.nsplit);
}

}  // namespace eb
