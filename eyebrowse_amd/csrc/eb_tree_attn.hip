// Attention of a tree of drafted tokens over a KV cache for gfx950: node i sees the cached keys
// 0 .. pos - 1 (the last of them, with a window) and those drafted keys j whose bit is set in row i
// of the masks; the drafted rows are cache rows pos ...
//
//   o[c] = sum_j 2^(s_cj - m) v_j / sum_j 2^(s_cj - m),   s_cj = scale log2(e) q_c . k_j
//
// over the keys j that column c sees; a column is one query head of one node. All columns of a KV
// head read the same keys: a workgroup takes up to 128 of them, so that each key is fetched from
// memory, and brought into the matrix cores' format, once for all. Split keys, then a log-sum-exp
// merge.
//
// A workgroup walks tiles of T keys. Half of its waves fetch K, half V, a tile ahead, into
// registers; they become f16 operands on their way into LDS:
//  - f32 rows: scaled by a power of two (the row's largest element in [2^13, 2^14)) and split into
//    two halves, each rounded to nearest (22 bits; the product of the two low halves is left out:
//    three matrix products per result); the power comes back with the score (K) or in the weight (V);
//  - half and E4M3 rows, and the codes of a block-scaled cache: exact as they are (two products,
//    for the two halves of q or of the weight); a block's scales come back as those powers do.
// K lies in LDS by rows, V transposed, so that both are 16-byte operand reads; chunks are xor-ed
// with the row (K) or the dim (V), which spreads eight neighbouring lanes over the banks.
//
// Lane (n, g) is lane n + 16 g of a wave; a wave owns 16 or 32 columns.
//  - Scores S[key][column] on v_mfma_f32_16x16x32_f16: lane (n, g) ends with keys 4g .. 4g + 3 of
//    each of two 16-key halves of a 32-key group, for column n.
//  - O^T[dim][column] += V^T P^T, the 32 contracted indices being the group's keys in the order in
//    which lane (n, g) holds them: its own scores are the operand, no lane exchange. V's transposed
//    rows are stored in that order. Lane (n, g) ends with dims 4g .. 4g + 3 (+ 16 e) of column n, so
//    that m, l and every rescale belong to the lane's own column.
//  - Online softmax with a reference m per column that moves only when a score exceeds it by more
//    than kSlack. Where V rows have powers of two of their own (f32, block-scaled), the weights carry
//    them, in a unit per column (2^lcu) that moves when a term would pass 2^15: a row of large
//    values that a column does not see costs it nothing.
//
// A key that a column does not see has weight exactly 0, and its V row is finite where any column
// of the workgroup may not see it: in tiles with masked keys a row that is not finite is stored as
// zeros and its weight made NaN, which reaches the columns that see it and no others. A column
// that sees nothing gives zeros.
#include "eb_cache_i8.h"
#include "eb_tree.h"

#include <algorithm>
#include <climits>

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

using eb::TreeElem;

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr float kSlack = 8.0f;     // log2 units a score may exceed its reference by
constexpr float kTop = 32768.0f;   // largest weight of a term (f16 holds 65504)
constexpr float kUnit = 7.0f;      // log2 of a weight at its reference
constexpr int kNone = 0x7FFFFFF0;  // a byte offset past any tile

template <int HDP, TreeElem E, int CW, int NSET>
struct Shape {
    static constexpr bool F32 = E == TreeElem::F32;
    static constexpr bool SCALED = E == TreeElem::F32 || E == TreeElem::I8;
    static constexpr int ES = F32 ? 4 : E == TreeElem::F16 ? 2 : 1;  // bytes of an element
    static constexpr int PL = F32 ? 2 : 1;                           // f16 planes
    // 32-key groups per tile: about 32 KB of cache in flight per workgroup, at most 64 KB of LDS.
    static constexpr int KG = F32 ? (HDP == 64 ? 2 : 1) : HDP == 256 ? 2 : (ES == 2 && HDP == 128) ? 2 : 4;
    static constexpr int T = 32 * KG;
    static constexpr int KW = std::min(KG, kWaves / CW);  // waves that share a column's tile
    static constexpr int COLS = CW * NSET * 16;
    static constexpr int PLANE = T * HDP * 2;  // bytes of one plane of K, and of V
    static constexpr int TILE = 2 * PL * PLANE + 2 * T * 4;
    static constexpr int NBUF = TILE > 40 * 1024 ? 1 : 2;
    static constexpr int NC = HDP / 32;  // 32-dim steps of a score
    static constexpr int ND = HDP / 16;  // 16-dim groups of an output
    static constexpr int CH = HDP / 8;   // 8-dim chunks of a K row
    static constexpr int SW = (CH < 16 ? CH : 16) - 1;
    static constexpr int HT = kThreads / 2;
    static constexpr int KU = T * CH / HT;  // K chunks per thread
    static constexpr int VD = F32 ? 4 : 8;  // dims of a V unit (8 keys)
    static constexpr int VC = HDP / VD;
    static constexpr int VUNITS = 4 * KG * VC;
    static constexpr int VU = (VUNITS + HT - 1) / HT;
    static constexpr int RW = ES == 1 ? 2 : 4;  // words of a load
    static constexpr int NR = std::max(KU * (F32 ? 2 : 1), VU * 8);
    static_assert(KW == 1 || (KW - 1) * CW * NSET * (ND * 1024 + 768) <= TILE * NBUF, "room to join waves");
};

struct Args {
    const float *q;
    const char *k, *v;
    const uint8_t *ks, *vs;
    const unsigned *masks, *depths;
    float *o, *part_acc, *part_ml;
    int h, hkv, g, n, words, ncols, hd;
    unsigned g_inv;  // 2^32 / g, rounded up: exact for the at most 2^16 columns of a KV head
    int pos, window;
    int key0, tiles;  // the first key of tile 0; a tile at least
    int nsplit, ncb, pairs, block_log2;
    float scale_log2;
};

// The largest of N neighbouring lanes' values (N a power of two from 8 to 64), in each of them.
template <int N>
__device__ __forceinline__ float lanes_max(float x) {
    x = fmaxf(x, eb::dpp<eb::kDppQuadXor1>(x));
    x = fmaxf(x, eb::dpp<eb::kDppQuadXor2>(x));
    x = fmaxf(x, eb::dpp<eb::kDppRowHalfMirror>(x));
    if constexpr (N >= 16) x = fmaxf(x, eb::dpp<eb::kDppRowMirror>(x));
    if constexpr (N >= 32) x = fmaxf(x, eb::lane_xor16(x));
    if constexpr (N >= 64) x = fmaxf(x, eb::lane_xor32(x));
    return x;
}

// Powers of two of a row whose largest magnitude has biased exponent e (at least 14): what scales
// it into [2^13, 2^14), and what brings it back.
__device__ __forceinline__ unsigned biased_exponent(float magnitude) {
    const unsigned e = __builtin_bit_cast(unsigned, magnitude) >> 23;
    return e < 14u ? 14u : e;
}
__device__ __forceinline__ float pow2_biased(unsigned e) { return __builtin_bit_cast(float, e << 23); }

__device__ __forceinline__ unsigned f16x2_bits(f16x2 x) { return __builtin_bit_cast(unsigned, x); }

// Four E4M3 patterns, or codes of a block-scaled cache, as f16, exact.
template <TreeElem E>
__device__ __forceinline__ u32x2 narrow_f16(unsigned w) {
    if constexpr (E == TreeElem::E4M3) {
        return u32x2{f16x2_bits(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false)),
                     f16x2_bits(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true))};
    } else {  // (the sign bit flipped: bytes 0..255 as the low bits of 1024 + byte, less 1152)
        const f16x2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
        const unsigned f = w ^ 0x80808080u;
        const unsigned lo = __builtin_amdgcn_perm(0x64646464u, f, 0x04010400u);
        const unsigned hi = __builtin_amdgcn_perm(0x64646464u, f, 0x04030402u);
        return u32x2{f16x2_bits(__builtin_bit_cast(f16x2, lo) + off), f16x2_bits(__builtin_bit_cast(f16x2, hi) + off)};
    }
}

// x as two halves, each rounded to nearest: 22 bits.
__device__ __forceinline__ void split(f32x8 x, f16x8 &hi, f16x8 &lo) {
    hi = __builtin_convertvector(x, f16x8);
    lo = __builtin_convertvector(x - __builtin_convertvector(hi, f32x8), f16x8);
}

template <int HDP, TreeElem E, int CW, int NSET>
__global__ __launch_bounds__(kThreads, 2) void tree_attn_kernel(Args a) {
    using S = Shape<HDP, E, CW, NSET>;
    constexpr int ES = S::ES, T = S::T, KW = S::KW, PL = S::PL, PLANE = S::PLANE, HT = S::HT;
    extern __shared__ char smem[];
    // Consecutive workgroups of an XCD (dealt round robin) take the column blocks of one KV head and
    // split, which then share that XCD's L2.
    const int slot = blockIdx.x / 8;
    const int pair = (int)(blockIdx.x % 8) + 8 * (slot / a.ncb);
    const int cb = slot % a.ncb;
    if (pair >= a.pairs) return;
    const int kvh = pair % a.hkv, split_id = pair / a.hkv;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g4 = lane >> 4;
    const int hd = a.hd, end = a.pos + a.n;
    auto node_of = [&](int c) { return a.g == 1 ? c : (int)__umulhi((unsigned)c, a.g_inv); };  // c / g
    const int col0 = cb * S::COLS;
    const int node0 = node_of(col0);
    const int nodes = node_of(min(col0 + S::COLS, a.ncols) - 1) - node0 + 1;  // of this workgroup's columns
    unsigned *s_mask = reinterpret_cast<unsigned *>(smem + S::NBUF * S::TILE);  // [nodes][words]
    int *s_depth = reinterpret_cast<int *>(s_mask + nodes * a.words);           // [n] (with a window)

    // ---- tiles: fetched into registers, then stored as operands -----------------------------------
    const bool vside = wave >= kWaves / 2;
    const int ht = tid % HT;
    const size_t row_bytes = (size_t)a.hkv * hd * ES;
    const char *base = (vside ? a.v : a.k) + (size_t)kvh * hd * ES;
    unsigned raw[S::NR][S::RW];
    unsigned raw_e = 127;  // I8: the exponent of key ht (1 past the last)
    auto fetch = [&](int t) {
        const int r0 = a.key0 + t * T;
        const int left = min(end - r0, T);
        const int nbytes = left > 0 ? (int)((left - 1) * row_bytes) + hd * ES : 0;
        const __amdgpu_buffer_rsrc_t res = eb::make_rsrc(base + (left > 0 ? (size_t)r0 * row_bytes : 0), nbytes);
        auto get = [&](int i, int off) {
            if constexpr (S::RW == 4) {
                const u32x4 w = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(res, off, 0, 0));
#pragma unroll
                for (int j = 0; j < 4; ++j) raw[i][j] = w[j];
            } else {
                const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(res, off, 0, 0));
#pragma unroll
                for (int j = 0; j < 2; ++j) raw[i][j] = w[j];
            }
        };
        const int rb = (int)row_bytes;
        if (!vside) {
            const int c = ht % S::CH, r = ht / S::CH;
#pragma unroll
            for (int j = 0; j < S::KU; ++j) {
                const int off = (r + j * (HT / S::CH)) * rb + c * 8 * ES;
                if constexpr (S::F32) {
                    get(2 * j, 8 * c < hd ? off : kNone);
                    get(2 * j + 1, 8 * c + 4 < hd ? off + 16 : kNone);
                } else {
                    get(j, 8 * c < hd ? off : kNone);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < S::VU; ++j) {
                const int u = ht + j * HT, c = u % S::VC, sb = u / S::VC;
                const bool in = u < S::VUNITS && c * S::VD < hd;
                const int off = (32 * (sb / 4) + 4 * (sb % 4)) * rb + c * S::VD * ES;
#pragma unroll
                for (int i = 0; i < 8; ++i) get(8 * j + i, in ? off + (i + (i & 4) * 3) * rb : kNone);
            }
        }
        if constexpr (E == TreeElem::I8) {
            const int key = min(r0 + min(ht, T - 1), end - 1);
            raw_e = (vside ? a.vs : a.ks)[(size_t)(key >> a.block_log2) * a.hkv + kvh];
        }
    };
    // The operands of a tile in LDS: K [planes][T][HDP], V [planes][KG][HDP][32], scales [2][T].
    auto store = [&](char *buf, bool edge) {
        float *s_scale = reinterpret_cast<float *>(buf + 2 * PL * PLANE);
        if (!vside) {
            const int c = ht % S::CH, r0 = ht / S::CH;
#pragma unroll
            for (int j = 0; j < S::KU; ++j) {
                const int r = r0 + j * (HT / S::CH);
                char *at = buf + (r * S::CH + (c ^ (r & S::SW))) * 16;
                if constexpr (S::F32) {
                    f32x8 x;
                    float top = 0.0f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        x[i] = __uint_as_float(raw[2 * j + i / 4][i % 4]);
                        top = fmaxf(top, __uint_as_float(raw[2 * j + i / 4][i % 4] & 0x7FFFFFFFu));
                    }
                    const unsigned e = biased_exponent(lanes_max<S::CH>(top));
                    f16x8 hi, lo;
                    split(x * pow2_biased(267u - e), hi, lo);
                    *reinterpret_cast<f16x8 *>(at) = hi;
                    *reinterpret_cast<f16x8 *>(at + PLANE) = lo;
                    if (c == 0) s_scale[r] = pow2_biased(e - 13u);
                } else if constexpr (ES == 2) {
                    *reinterpret_cast<u32x4 *>(at) = u32x4{raw[j][0], raw[j][1], raw[j][2], raw[j][3]};
                } else {
                    const u32x2 x = narrow_f16<E>(raw[j][0]), y = narrow_f16<E>(raw[j][1]);
                    *reinterpret_cast<u32x4 *>(at) = u32x4{x[0], x[1], y[0], y[1]};
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < S::VU; ++j) {
                const int u = ht + j * HT, c = u % S::VC, sb = u / S::VC;
                const int kg = sb / 4, g = sb % 4;
                if (u >= S::VUNITS) break;
                char *vt = buf + PL * PLANE + kg * (HDP * 64);
                float *vs = s_scale + T + 32 * kg + 4 * g;  // keys i and 16 + i, i < 4
                if constexpr (S::F32) {
                    f32x4 x[8];
                    float back[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const unsigned *w = raw[8 * j + i];
                        x[i] = f32x4{__uint_as_float(w[0]), __uint_as_float(w[1]), __uint_as_float(w[2]),
                                     __uint_as_float(w[3])};
                        unsigned bits = 0;  // (as whole numbers: NaN is above infinity)
#pragma unroll
                        for (int d = 0; d < 4; ++d) bits = max(bits, w[d] & 0x7FFFFFFFu);
                        // What is not finite becomes infinity, which fmaxf keeps.
                        const float top = lanes_max<S::VC>(__uint_as_float(min(bits, 0x7F800000u)));
                        const unsigned e = biased_exponent(top);
                        const bool bad = e == 255u;
                        const float f = pow2_biased(267u - e);
#pragma unroll
                        for (int d = 0; d < 4; ++d) x[i][d] = bad ? 0.0f : x[i][d] * f;
                        back[i] = bad ? __builtin_nanf("") : pow2_biased(e - 13u);
                    }
                    if (c == 0) {
                        *reinterpret_cast<f32x4 *>(vs) = f32x4{back[0], back[1], back[2], back[3]};
                        *reinterpret_cast<f32x4 *>(vs + 16) = f32x4{back[4], back[5], back[6], back[7]};
                    }
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        const f32x8 col = {x[0][d], x[1][d], x[2][d], x[3][d], x[4][d], x[5][d], x[6][d], x[7][d]};
                        f16x8 hi, lo;
                        split(col, hi, lo);
                        char *at = vt + (4 * c + d) * 64 + ((g ^ (c & 3)) * 16);
                        *reinterpret_cast<f16x8 *>(at) = hi;
                        *reinterpret_cast<f16x8 *>(at + PLANE) = lo;
                    }
                } else {
                    unsigned x[8][4];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if constexpr (ES == 2) {
#pragma unroll
                            for (int d = 0; d < 4; ++d) x[i][d] = raw[8 * j + i][d];
                        } else {
                            const u32x2 p = narrow_f16<E>(raw[8 * j + i][0]), q = narrow_f16<E>(raw[8 * j + i][1]);
                            x[i][0] = p[0];
                            x[i][1] = p[1];
                            x[i][2] = q[0];
                            x[i][3] = q[1];
                        }
                    }
                    if constexpr (E != TreeElem::I8) {
                        if (edge) {
                            float back[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                bool bad = false;
#pragma unroll
                                for (int d = 0; d < 4; ++d)
                                    bad = bad || (x[i][d] & 0x7C00u) == 0x7C00u || (x[i][d] & 0x7C000000u) == 0x7C000000u;
                                bad = lanes_max<S::VC>(bad ? 1.0f : 0.0f) > 0.0f;
#pragma unroll
                                for (int d = 0; d < 4; ++d) x[i][d] = bad ? 0u : x[i][d];
                                back[i] = bad ? __builtin_nanf("") : 1.0f;
                            }
                            if (c == 0) {
                                *reinterpret_cast<f32x4 *>(vs) = f32x4{back[0], back[1], back[2], back[3]};
                                *reinterpret_cast<f32x4 *>(vs + 16) = f32x4{back[4], back[5], back[6], back[7]};
                            }
                        }
                    }
#pragma unroll
                    for (int d = 0; d < 8; ++d) {
                        const unsigned sel = d % 2 ? 0x07060302u : 0x05040100u;
                        u32x4 w;
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_perm(x[2 * i + 1][d / 2], x[2 * i][d / 2], sel);
                        const int dim = 8 * c + d;
                        *reinterpret_cast<u32x4 *>(vt + dim * 64 + ((g ^ ((dim >> 2) & 3)) * 16)) = w;
                    }
                }
            }
        }
        if constexpr (E == TreeElem::I8) {
            if (ht < T) s_scale[(vside ? T : 0) + ht] = eb::i8_scale(raw_e, 0);
        }
    };

    int t = split_id;
    fetch(t);

    // ---- the columns' queries, masks and first keys -------------------------------------------------
    const int cw = wave % CW, kw = wave / CW;
    const bool worker = kw < KW;  // (the others fetch and store only)
    f16x8 qh[NSET][S::NC], ql[NSET][S::NC];
    float qs[NSET];
    int my_node[NSET], my_first[NSET];
#pragma unroll
    for (int s = 0; s < NSET; ++s) {
        const int c = col0 + (cw * NSET + s) * 16 + n;
        const bool have = worker && c < a.ncols;
        const int node = node_of(min(c, a.ncols - 1));
        my_node[s] = node - node0;
        const auto res = eb::make_rsrc(a.q, a.n * a.h * hd * 4);
        const int at = (node * a.h + kvh * a.g + min(c, a.ncols - 1) - node * a.g) * hd;
        f32x8 x[S::NC];
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < S::NC; ++i) {
            const int d = 32 * i + 8 * g4;
            const f32x4 lo = __builtin_bit_cast(
                f32x4, __builtin_amdgcn_raw_buffer_load_b128(res, have && d < hd ? (at + d) * 4 : kNone, 0, 0));
            const f32x4 hi = __builtin_bit_cast(
                f32x4, __builtin_amdgcn_raw_buffer_load_b128(res, have && d + 4 < hd ? (at + d + 4) * 4 : kNone, 0, 0));
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[i][j] = (j < 4 ? lo[j % 4] : hi[j % 4]) * a.scale_log2;
                top = fmaxf(top, fabsf(x[i][j]));
            }
        }
        top = fmaxf(top, eb::lane_xor16(top));
        top = fmaxf(top, eb::lane_xor32(top));
        const unsigned e = biased_exponent(top);
        qs[s] = pow2_biased(e - 13u);
#pragma unroll
        for (int i = 0; i < S::NC; ++i) split(x[i] * pow2_biased(267u - e), qh[s][i], ql[s][i]);
    }
    for (int i = tid; i < nodes * a.words; i += kThreads) s_mask[i] = a.masks[(size_t)node0 * a.words + i];
    if (a.window > 0)
        for (int i = tid; i < a.n; i += kThreads) s_depth[i] = (int)min(a.depths[i], 1u << 27);
    __syncthreads();
    int safe_lo = 0;  // keys below it may be behind some column's window
    if (a.window > 0) {
        int deepest = 0;
        for (int i = lane; i < nodes; i += 64) deepest = max(deepest, s_depth[node0 + i]);
#pragma unroll
        for (int m = 32; m > 0; m >>= 1) deepest = max(deepest, __shfl_xor(deepest, m));
        safe_lo = __builtin_amdgcn_readfirstlane(a.pos + deepest - a.window + 1);
    }
#pragma unroll
    for (int s = 0; s < NSET; ++s)
        my_first[s] = a.window > 0 ? a.pos + s_depth[node0 + my_node[s]] - a.window + 1 : 0;

    // ---- state --------------------------------------------------------------------------------------
    f32x4 acc[NSET][S::ND];
    float m[NSET], l[NSET], lcu[NSET];
#pragma unroll
    for (int s = 0; s < NSET; ++s) {
        m[s] = -INFINITY;
        l[s] = 0.0f;
        lcu[s] = 0.0f;
#pragma unroll
        for (int e = 0; e < S::ND; ++e) acc[s][e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // One group of 32 keys from k0 on, in buf.
    auto consume = [&](const char *buf, int kg, int k0, bool edge) {
        const float *s_scale = reinterpret_cast<const float *>(buf + 2 * PL * PLANE);
        f32x4 sc[NSET][2];
#pragma unroll
        for (int s = 0; s < NSET; ++s) sc[s][0] = sc[s][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < S::NC; ++i) {
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                const int r = 32 * kg + 16 * sub + n;
                const char *at = buf + (r * S::CH + ((4 * i + g4) ^ (r & S::SW))) * 16;
                const f16x8 kh = *reinterpret_cast<const f16x8 *>(at);
                f16x8 kl;
                if constexpr (PL == 2) kl = *reinterpret_cast<const f16x8 *>(at + PLANE);
#pragma unroll
                for (int s = 0; s < NSET; ++s) {
                    sc[s][sub] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qh[s][i], sc[s][sub], 0, 0, 0);
                    sc[s][sub] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, ql[s][i], sc[s][sub], 0, 0, 0);
                    if constexpr (PL == 2)
                        sc[s][sub] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl, qh[s][i], sc[s][sub], 0, 0, 0);
                }
            }
        }
        f32x4 ks[2], vs[2];
        if constexpr (S::SCALED) {
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                ks[sub] = *reinterpret_cast<const f32x4 *>(s_scale + 32 * kg + 16 * sub + 4 * g4);
                vs[sub] = *reinterpret_cast<const f32x4 *>(s_scale + T + 32 * kg + 16 * sub + 4 * g4);
            }
        }
        f16x8 ph[NSET], pl[NSET];
#pragma unroll
        for (int s = 0; s < NSET; ++s) {
            float x[8], w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = sc[s][i / 4][i % 4];
                if constexpr (S::SCALED) x[i] *= ks[i / 4][i % 4];
                // (An infinite half of K meets q's two halves, whose signs may agree: infinity times 0
                // is NaN whatever they gave. f32 rows' split made it NaN, E4M3 has no infinity.)
                if constexpr (E == TreeElem::F16)
                    x[i] = __builtin_fmaf(x[i], qs[s], x[i] * 0.0f);
                else
                    x[i] *= qs[s];
            }
            unsigned seen = 0xFFu;
            if (edge) {
                const unsigned *mask = s_mask + my_node[s] * a.words;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int key = k0 + 16 * (i / 4) + 4 * g4 + i % 4, j = key - a.pos;
                    bool ok;
                    if (j < 0) {
                        ok = key >= my_first[s];
                    } else {
                        const int jj = min(j, a.n - 1);
                        ok = j < a.n && (mask[jj >> 5] >> (jj & 31)) & 1u;
                        if (a.window > 0) ok = ok && a.pos + s_depth[jj] >= my_first[s];
                    }
                    if (!ok) {
                        x[i] = -INFINITY;
                        seen &= ~(1u << i);
                    }
                }
            }
            const float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
            // Weights against the present reference and unit; true where they do not serve.
            float sum = 0.0f;
            auto weigh = [&] {
                const float ref = m[s] == -INFINITY ? 0.0f : S::SCALED ? m[s] : m[s] - kUnit;
                const float cu = ldexpf(1.0f, (int)lcu[s]);
                float most = 0.0f;
                sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float p = eb::fast_exp2(x[i] - ref);
                    sum += p;
                    w[i] = p;
                    if constexpr (S::SCALED) {
                        w[i] = p * vs[i / 4][i % 4] * cu;
                        most = fmaxf(most, w[i]);
                    }
                }
                return top > m[s] + kSlack || (m[s] == -INFINITY && top > -INFINITY) || most > kTop;
            };
            if (__builtin_amdgcn_ballot_w64(weigh()) != 0) {
                float t1 = fmaxf(top, eb::lane_xor16(top));
                t1 = fmaxf(t1, eb::lane_xor32(t1));  // the column's largest score of the group
                const float mn = m[s] == -INFINITY || t1 > m[s] + kSlack ? t1 : m[s];
                const float d = mn == m[s] ? 0.0f : m[s] - mn;  // (infinite at the column's first keys)
                float f = d;
                if constexpr (S::SCALED) {
                    const float ref = mn == -INFINITY ? 0.0f : mn;
                    float y = 0.0f;  // the group's largest term
#pragma unroll
                    for (int i = 0; i < 8; ++i) y = fmaxf(y, eb::fast_exp2(x[i] - ref) * vs[i / 4][i % 4]);
                    y = fmaxf(y, eb::lane_xor16(y));
                    y = fmaxf(y, eb::lane_xor32(y));
                    // Earlier terms lose 2^d: as much the unit may grow. Where this group's would pass
                    // 2^15 in it, its largest term becomes 2^6 to 2^7.
                    float unit = fminf(lcu[s] + floorf(-d), 120.0f);
                    const float ey = (float)__builtin_amdgcn_frexp_expf(y);
                    if (y > 0.0f && ey + unit > 15.0f) unit = 7.0f - ey;
                    f = d + (unit - lcu[s]);
                    lcu[s] = unit;
                }
                f = d < -1.0e6f ? 0.0f : eb::fast_exp2(f);
                l[s] *= d < -1.0e6f ? 0.0f : eb::fast_exp2(d);
                m[s] = mn;
#pragma unroll
                for (int e = 0; e < S::ND; ++e) acc[s][e] *= f;
                (void)weigh();
            }
            l[s] += sum;
            if (edge) {  // (a NaN scale does not reach what a column does not see)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if constexpr (!S::SCALED)
                        w[i] *= s_scale[T + 32 * kg + 16 * (i / 4) + 4 * g4 + i % 4];
                    if (!((seen >> i) & 1u)) w[i] = 0.0f;
                }
            }
            split(f32x8{w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]}, ph[s], pl[s]);
        }
        const char *vt = buf + PL * PLANE + kg * (HDP * 64);
#pragma unroll
        for (int e = 0; e < S::ND; ++e) {
            const char *at = vt + (16 * e + n) * 64 + ((g4 ^ ((n >> 2) & 3)) * 16);
            const f16x8 vh = *reinterpret_cast<const f16x8 *>(at);
            f16x8 vl;
            if constexpr (PL == 2) vl = *reinterpret_cast<const f16x8 *>(at + PLANE);
#pragma unroll
            for (int s = 0; s < NSET; ++s) {
                acc[s][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, ph[s], acc[s][e], 0, 0, 0);
                acc[s][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, pl[s], acc[s][e], 0, 0, 0);
                if constexpr (PL == 2)
                    acc[s][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, ph[s], acc[s][e], 0, 0, 0);
            }
        }
    };

    // ---- the tiles ----------------------------------------------------------------------------------
    for (int b = 0; t < a.tiles; t += a.nsplit, b ^= 1) {
        char *buf = smem + (S::NBUF == 2 && b ? S::TILE : 0);
        const int r0 = a.key0 + t * T;
        const bool edge = r0 + T > a.pos || r0 < safe_lo;  // (uniform)
        store(buf, edge);
        if (t + a.nsplit < a.tiles) fetch(t + a.nsplit);
        __syncthreads();
        if (worker) {
#pragma unroll 1
            for (int kg = kw; kg < S::KG; kg += KW) {
                if (r0 + 32 * kg >= end) break;
                consume(buf, kg, r0 + 32 * kg, edge);
            }
        }
        if constexpr (S::NBUF == 1) __syncthreads();
    }

    // ---- the waves' states meet ---------------------------------------------------------------------
#pragma unroll
    for (int s = 0; s < NSET; ++s) {
        l[s] += eb::lane_xor16(l[s]);
        l[s] += eb::lane_xor32(l[s]);
    }
    if constexpr (S::SCALED) {  // out of the columns' units
#pragma unroll
        for (int s = 0; s < NSET; ++s)
#pragma unroll
            for (int e = 0; e < S::ND; ++e)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[s][e][r] = ldexpf(acc[s][e][r], -(int)lcu[s]);
    }
    if constexpr (KW > 1) {
        constexpr int SLOT = NSET * (S::ND * 1024 + 512);  // bytes a wave leaves
        __syncthreads();
        if (worker && kw > 0) {
            char *at = smem + ((kw - 1) * CW + cw) * SLOT;
#pragma unroll
            for (int s = 0; s < NSET; ++s) {
#pragma unroll
                for (int e = 0; e < S::ND; ++e)
                    *reinterpret_cast<f32x4 *>(at + (s * S::ND + e) * 1024 + lane * 16) = acc[s][e];
                float *ml = reinterpret_cast<float *>(at + NSET * S::ND * 1024 + s * 512);
                ml[lane] = m[s];
                ml[64 + lane] = l[s];
            }
        }
        __syncthreads();
        if (kw > 0) return;
#pragma unroll
        for (int w = 1; w < KW; ++w) {
            const char *at = smem + ((w - 1) * CW + cw) * SLOT;
#pragma unroll
            for (int s = 0; s < NSET; ++s) {
                const float *ml = reinterpret_cast<const float *>(at + NSET * S::ND * 1024 + s * 512);
                const float m2 = ml[lane], mn = fmaxf(m[s], m2), ref = mn == -INFINITY ? 0.0f : mn;
                const float f1 = eb::fast_exp2(m[s] - ref), f2 = eb::fast_exp2(m2 - ref);
                l[s] = l[s] * f1 + ml[64 + lane] * f2;
                m[s] = mn;
#pragma unroll
                for (int e = 0; e < S::ND; ++e)
                    acc[s][e] = acc[s][e] * f1 +
                                f2 * *reinterpret_cast<const f32x4 *>(at + (s * S::ND + e) * 1024 + lane * 16);
            }
        }
    }
    if (!worker) return;
#pragma unroll
    for (int s = 0; s < NSET; ++s) {
        const int c = col0 + (cw * NSET + s) * 16 + n;
        if (c >= a.ncols) continue;
        const int node = node0 + my_node[s];
        const size_t row = (size_t)node * a.h + kvh * a.g + c - node * a.g;
        if (a.nsplit == 1) {
            const float inv = l[s] == 0.0f ? 0.0f : 1.0f / l[s];
#pragma unroll
            for (int e = 0; e < S::ND; ++e)
                if (16 * e + 4 * g4 < hd)
                    *reinterpret_cast<f32x4 *>(a.o + row * hd + 16 * e + 4 * g4) = acc[s][e] * inv;
        } else {
            const size_t at = (size_t)split_id * a.n * a.h + row;
#pragma unroll
            for (int e = 0; e < S::ND; ++e)
                if (16 * e + 4 * g4 < hd) *reinterpret_cast<f32x4 *>(a.part_acc + at * hd + 16 * e + 4 * g4) = acc[s][e];
            if (g4 == 0) {
                a.part_ml[at * 2] = m[s];
                a.part_ml[at * 2 + 1] = l[s];
            }
        }
    }
}

// o[row] = sum of the splits' sums, at one reference. Workgroup: one row (node and head); a group of
// lanes holds the row's dims, four each, the groups share the splits, four at a time in flight.
__global__ __launch_bounds__(kThreads) void tree_merge_kernel(const float *__restrict__ part_acc,
                                                              const float *__restrict__ part_ml, float *__restrict__ o,
                                                              int rows, int hd, int nsplit, int lanes_log2) {
    __shared__ float s_m[kThreads], s_l[kThreads];
    __shared__ f32x4 s_a[kThreads];
    const int tid = threadIdx.x, row = blockIdx.x;
    const int groups = kThreads >> lanes_log2;
    const int grp = tid >> lanes_log2, d = (tid & ((1 << lanes_log2) - 1)) * 4;
    const int at_d = d < hd ? d : 0;
    float M = -INFINITY, L = 0.0f;
    f32x4 A = {0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int B = 4;
    for (int s0 = grp; s0 < nsplit; s0 += groups * B) {
        float bm[B], bl[B];
        f32x4 ba[B];
#pragma unroll
        for (int j = 0; j < B; ++j) {
            const int s = min(s0 + j * groups, nsplit - 1);
            const size_t at = (size_t)s * rows + row;
            bm[j] = part_ml[at * 2];
            bl[j] = part_ml[at * 2 + 1];
            ba[j] = *reinterpret_cast<const f32x4 *>(part_acc + at * hd + at_d);
        }
        __builtin_amdgcn_sched_barrier(0);  // (all loads before the first use)
        float mn = M;
#pragma unroll
        for (int j = 0; j < B; ++j)
            if (s0 + j * groups < nsplit) mn = fmaxf(mn, bm[j]);
        const float ref = mn == -INFINITY ? 0.0f : mn;
        const float c = eb::fast_exp2(M - ref);
        L *= c;
        A *= c;
#pragma unroll
        for (int j = 0; j < B; ++j) {
            if (s0 + j * groups >= nsplit) continue;
            const float w = eb::fast_exp2(bm[j] - ref);
            L += w * bl[j];
            A += w * ba[j];
        }
        M = mn;
    }
    s_m[tid] = M;
    s_l[tid] = L;
    s_a[tid] = A;
    __syncthreads();
    if (grp > 0 || d >= hd) return;
    float mt = M;
    for (int g = 1; g < groups; ++g) mt = fmaxf(mt, s_m[(g << lanes_log2) + tid]);
    const float ref = mt == -INFINITY ? 0.0f : mt;
    float Lt = 0.0f;
    f32x4 At = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int g = 0; g < groups; ++g) {
        const int i = (g << lanes_log2) + tid;
        const float w = eb::fast_exp2(s_m[i] - ref);
        Lt += w * s_l[i];
        At += w * s_a[i];
    }
    const float inv = Lt == 0.0f ? 0.0f : 1.0f / Lt;  // (no key seen: zeros)
    *reinterpret_cast<f32x4 *>(o + (size_t)row * hd + d) = At * inv;
}

struct Plan {
    int hdp, cols, ncb, T, key0, tiles, nsplit;
};

int keys_per_tile(int hdp, TreeElem e) {
    switch (e) {
        case TreeElem::F32: return hdp == 64 ? 64 : 32;
        case TreeElem::F16: return hdp == 64 ? 128 : 64;
        default: return hdp == 256 ? 64 : 128;
    }
}

constexpr size_t kMinSplitKeys = 128;
constexpr int kWgsPerCu = 2;
Plan plan_of(size_t h, size_t hkv, size_t hd, size_t pos, size_t n, size_t window, TreeElem elem, int cu_count) {
    Plan p{};
    p.hdp = hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
    const size_t cols = n * (h / hkv);
    p.cols = cols <= 16 ? 16 : cols <= 64 || p.hdp == 256 ? 64 : 128;
    p.ncb = (int)((cols + p.cols - 1) / p.cols);
    p.T = keys_per_tile(p.hdp, elem);
    const size_t first = window > 0 && pos + 1 > window ? pos + 1 - window : 0;
    p.key0 = (int)(first & ~(size_t)15);
    p.tiles = (int)((pos + n - p.key0 + p.T - 1) / p.T);
    size_t nsplit = std::max<size_t>(1, (size_t)cu_count * kWgsPerCu / (hkv * p.ncb));
    nsplit = std::min(nsplit, (size_t)p.tiles);
    if (pos + n - first <= kMinSplitKeys) nsplit = 1;
    p.nsplit = (int)nsplit;
    return p;
}

template <int HDP, TreeElem E, int CW, int NSET>
hipError_t launch(hipStream_t st, const Args &a) {
    using S = Shape<HDP, E, CW, NSET>;
    const size_t nodes = std::min<size_t>(a.n, S::COLS);
    const size_t lds = (size_t)S::NBUF * S::TILE + (nodes * a.words + (a.window > 0 ? a.n : 0)) * 4;
    if (lds > 64 * 1024) {
        static const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&tree_attn_kernel<HDP, E, CW, NSET>),
                                                        hipFuncAttributeMaxDynamicSharedMemorySize, 80 * 1024);
        if (e != hipSuccess) return e;
    }
    static_assert(S::NBUF * S::TILE + (S::COLS * 8 + 256) * 4 <= 80 * 1024, "two workgroups per CU");
    const unsigned grid = (unsigned)((a.pairs + 7) / 8 * 8 * a.ncb);
    tree_attn_kernel<HDP, E, CW, NSET><<<grid, kThreads, lds, st>>>(a);
    return hipSuccess;
}

template <int HDP, TreeElem E>
hipError_t launch_cols(hipStream_t st, const Args &a, int cols) {
    if (cols == 16) return launch<HDP, E, 1, 1>(st, a);
    if constexpr (HDP < 256)
        if (cols == 128) return launch<HDP, E, 4, 2>(st, a);
    return launch<HDP, E, 4, 1>(st, a);
}

template <TreeElem E>
hipError_t launch_elem(hipStream_t st, const Args &a, const Plan &p) {
    return p.hdp == 64 ? launch_cols<64, E>(st, a, p.cols)
           : p.hdp == 128 ? launch_cols<128, E>(st, a, p.cols)
                          : launch_cols<256, E>(st, a, p.cols);
}

}  // namespace

namespace eb {

// part_acc [nsplit, n * h, hd], part_ml [nsplit, n * h, 2]; a window only lowers the splits.
size_t tree_attn_workspace_floats(size_t h, size_t hkv, size_t hd, size_t pos, size_t n, TreeElem elem, int cu_count) {
    if (n == 0) return 0;
    const Plan p = plan_of(h, hkv, hd, pos, n, 0, elem, cu_count);
    return p.nsplit > 1 ? (size_t)p.nsplit * n * h * (hd + 2) : 0;
}

eb_status launch_attn_tree(hipStream_t st, const TreeAttn &x, float *ws, size_t ws_floats, int cu_count) {
    const Plan p = plan_of(x.h, x.hkv, x.hd, x.pos, x.n, x.window, x.elem, cu_count);
    const size_t rows = x.n * x.h;
    const size_t need = p.nsplit > 1 ? (size_t)p.nsplit * rows * (x.hd + 2) : 0;
    if (need > 0 && (!ws || ws_floats < need))
        return fail(EB_SHAPE_MISMATCH, "attn_tree: workspace holds %zu floats, needs %zu", ws_floats, need);
    Args a{};
    a.q = x.q;
    a.k = static_cast<const char *>(x.k);
    a.v = static_cast<const char *>(x.v);
    a.ks = x.ks;
    a.vs = x.vs;
    a.masks = x.masks;
    a.depths = x.depths;
    a.o = x.o;
    a.part_acc = ws;
    a.part_ml = ws ? ws + (size_t)p.nsplit * rows * x.hd : nullptr;
    a.h = (int)x.h;
    a.hkv = (int)x.hkv;
    a.g = (int)(x.h / x.hkv);
    a.g_inv = (unsigned)((((uint64_t)1 << 32) + a.g - 1) / a.g);
    a.n = (int)x.n;
    a.words = (int)tree_words(x.n);
    a.ncols = (int)(x.n * a.g);
    a.hd = (int)x.hd;
    a.pos = (int)x.pos;
    a.window = (int)std::min<size_t>(x.window, (size_t)1 << 30);
    a.key0 = p.key0;
    a.tiles = p.tiles;
    a.nsplit = p.nsplit;
    a.ncb = p.ncb;
    a.pairs = (int)x.hkv * p.nsplit;
    while (x.block > 0 && (size_t)1 << a.block_log2 < x.block) ++a.block_log2;
    a.scale_log2 = x.scale * kLog2e;
    const hipError_t e = x.elem == TreeElem::F32    ? launch_elem<TreeElem::F32>(st, a, p)
                         : x.elem == TreeElem::F16  ? launch_elem<TreeElem::F16>(st, a, p)
                         : x.elem == TreeElem::E4M3 ? launch_elem<TreeElem::E4M3>(st, a, p)
                                                    : launch_elem<TreeElem::I8>(st, a, p);
    if (e != hipSuccess) return hip_fail(e, "attn_tree launch set-up");
    const eb_status s = check_launch("attn_tree");
    if (s != EB_OK || p.nsplit == 1) return s;
    int lanes_log2 = 0;
    while ((size_t)4 << lanes_log2 < x.hd) ++lanes_log2;
    tree_merge_kernel<<<(unsigned)rows, kThreads, 0, st>>>(a.part_acc, a.part_ml, x.o, (int)rows, (int)x.hd, p.nsplit,
                                                           lanes_log2);
    return check_launch("attn_tree (merge)");
}

}  // namespace eb
