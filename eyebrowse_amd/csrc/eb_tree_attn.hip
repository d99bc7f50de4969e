// Attention of a tree of drafted tokens over a KV cache for gfx950: node i sees the cached keys
// 0 .. pos - 1 (the last of them, with a window) and those drafted keys j whose bit is set in row i
// of the masks; the drafted rows are cache rows pos ...
//
//   o[c] = sum_j 2^(s_cj - m) v_j / sum_j 2^(s_cj - m),   s_cj = scale log2(e) q_c . k_j
//
// over the keys j that column c sees; a column is one query head of one node. All columns of a KV
// head read the same keys: a workgroup takes 16, 64 or 128 of them, so that each key is fetched from
// memory once for all of those. Split keys, then a log-sum-exp merge.
//
// A workgroup walks tiles of T keys; half of its waves fetch K, half V. Two ways to the matrix cores'
// f16 operands:
//  - Copied rows (half, E4M3 of whole 16-byte pieces, block-scaled codes) go from memory to LDS as they
//    are, up to four tiles ahead, no register on the way. K's pieces are the score's operand as read; V
//    is read across (16 lanes get 16 dims of 4 or 8 keys, each its own dim of all). Bytes become f16 at
//    use. Pieces are xor-ed with the row, against bank conflicts.
//  - Stored rows (f32; E4M3 rows that end inside a piece) pass through registers, a tile ahead, and
//    become f16 on their way into LDS, once for all columns. An f32 row is scaled by a power of two (its
//    largest element in [2^13, 2^14)) and split into two halves, each rounded to nearest (22 bits; the
//    product of the two low halves is left out: three matrix products per result); the power comes back
//    with the score (K) or in the weight (V). K lies by rows, V transposed.
// Half, E4M3 and code values are exact in f16 (two products, for the two halves of q or of the
// weight); a block's scales come back as those powers do.
//
// Lane (n, g) is lane n + 16 g of a wave; a wave owns 16 or 32 columns.
//  - Scores S[key][column] on v_mfma_f32_16x16x32_f16: lane (n, g) ends with keys 4g .. 4g + 3 of
//    each of two 16-key halves of a 32-key group, for column n.
//  - O^T[dim][column] += V^T P^T, the 32 contracted indices being the group's keys in the order in
//    which lane (n, g) holds them: its own scores are the operand, no lane exchange; V comes in that
//    order. Lane (n, g) ends with four dims of every 16 of column n, so that m, l and every rescale
//    belong to the lane's own column.
//  - Online softmax with a reference m per column that moves only when a score exceeds it by more
//    than kSlack. Where V rows have powers of two of their own (f32, block-scaled), the weights carry
//    them, in a unit per column (2^lcu) that moves when a term would pass 2^15: a row of large
//    values that a column does not see costs it nothing.
//
// A key that a column does not see has weight exactly 0, and its V row is finite where any column
// of the workgroup may not see it: in tiles with masked keys a row that is not finite becomes zeros
// and its weight NaN, which reaches the columns that see it and no others. Where all see it, a half or
// E4M3 row goes into the products as it is, and a column whose sums are not finite at the end is made
// NaN whole (finite rows' sums cannot pass f32's range). A column that sees nothing gives zeros.
//
// What binds it, with 32 heads over 8 of 128 (whole calls in a graph): 4 nodes, the cache's bytes (behind
// 30000 f32 keys 48 to 49 us, 5.0 to 5.1 TB/s: 1.26 times what they take at the 6.35 TB/s that a copy of cache
// rows reaches, the fixed parts below between); 64 nodes, matrix instructions and the softmax and conversions
// beside them, which two waves to a SIMD overlap in part (behind 32000 half keys 76 to 83 us, 406 to 440
// TFLOP/s of the formula's products, twice that issued; 30000 E4M3 71 to 76, block-scaled 90 to 91, f32 132 to
// 140 us); between, both, and the call's fixed parts: 3 to 5 us until a workgroup's first tile is there, 4 to
// 6 us for the merge and its launch (21 nodes behind 8191 block-scaled keys 24 us).
#include "eb_cache_i8.h"
#include "eb_tree.h"

#include <algorithm>
#include <climits>
#include <cmath>

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

using eb::TreeElem;

constexpr float kSlack = 8.0f;     // log2 units a score may exceed its reference by
constexpr float kTop = 32768.0f;   // largest weight of a term (f16 holds 65504)
constexpr float kUnit = 7.0f;      // log2 of a weight at its reference
constexpr float kNoRef = -3.4028235e38f;  // a reference below all scores (f32's lowest): no key yet
constexpr unsigned kNone = 0x7FFFFFF0u;  // a byte offset past any tile
// f32 K: a sum of up to 256 products of 2^14 times 2^14 times a row's power of two (2^-126 to 2^114) passes
// f32's range although the column's power, which comes last, brings it back: the rows' powers are kept times
// this (2^-149 at least, which f32 holds), the columns' times its inverse.
constexpr float kScoreShift = 0x1p-23f;
constexpr int kScoreShiftLog2 = 23;

// How a call is run: COPY moves the cache's rows to LDS as they are (half rows, E4M3 rows of whole
// 16-byte pieces, block-scaled codes); otherwise they pass through registers and become f16 there (f32
// rows, whose halves are the same for all columns; E4M3 rows that end inside a piece).
//
// Waves of a workgroup, and 32-key groups of a tile. One wave's columns (cw 1): the waves share the
// tile's keys. Up to 64: each wave has its own 16; more: its own 32. With eight waves the halves of a
// tile's keys go to four each, so that a split leaves half as much for the merge.
constexpr int waves_of(int cw, int nset, bool copy) { return nset == 2 || (copy && cw > 1) ? 8 : 4; }
constexpr int key_groups(int hdp, TreeElem e, int cw, int nset, bool copy) {
    const bool f32 = e == TreeElem::F32, f16 = e == TreeElem::F16;
    if (copy) return f16 ? hdp == 64 ? 4 : hdp == 128 || cw > 1 ? 2 : 1 : hdp == 256 ? 2 : 4;
    if (hdp == 256) return 1;
    if (f32) return hdp == 64 || nset == 2 ? 2 : 1;
    return 4;
}

template <int HDP, TreeElem E, int CW, int NSET, bool COPY>
struct Shape {
    static constexpr bool F32 = E == TreeElem::F32;
    static constexpr bool SCALED = E == TreeElem::F32 || E == TreeElem::I8;
    static constexpr int ES = F32 ? 4 : E == TreeElem::F16 ? 2 : 1;  // bytes of an element
    static constexpr int PL = F32 ? 2 : 1;                           // f16 planes
    static constexpr int WAVES = waves_of(CW, NSET, COPY), THREADS = WAVES * 64, HT = THREADS / 2;
    static constexpr int KG = key_groups(HDP, E, CW, NSET, COPY);
    static constexpr int T = 32 * KG;
    static constexpr int KW = std::min(KG, WAVES / CW);  // waves that share a column's tile
    static constexpr int COLS = CW * NSET * 16;
    static constexpr int NC = HDP / 32;  // 32-dim steps of a score
    static constexpr int ND = HDP / 16;  // 16-dim groups of an output
    static constexpr int LD = 16 / ES;   // dims of a 16-byte piece
    // ---- rows copied to LDS
    static constexpr int RB = HDP * ES, CR = RB / 16;             // bytes and pieces of a row
    static constexpr int CPW = T * CR / 64 / (WAVES / 2);         // copies per wave and tile
    static constexpr int CPT = CPW + (E == TreeElem::I8 ? 1 : 0);  // with the exponents'
    // ---- rows stored as operands
    static constexpr int CH = HDP / 8;  // 8-dim chunks of a K row in LDS
    static constexpr int SW = (CH < 16 ? CH : 16) - 1;
    static constexpr int PLANE = T * HDP * 2;  // bytes of one plane of K, and of V
    static constexpr int KL = HDP / (F32 ? 8 : LD);  // K units of a row: 8 dims (f32), or a load
    static constexpr int KU = T * KL / HT;           // and per thread
    // V units: 8 keys by VD dims, VW words of a row.
    static constexpr int VD = NSET == 2 && !F32 ? LD / 2 : LD;
    static constexpr int VW = VD * ES / 4;
    static constexpr int VC = HDP / VD;
    static constexpr int VUNITS = 4 * KG * VC;
    static constexpr int VU = (VUNITS + HT - 1) / HT;
    static constexpr int NR = COPY ? 1 : std::max(KU * (F32 ? 8 : 4), VU * 8 * VW);
    // ---- LDS
    static constexpr int TILE = COPY ? 2 * T * RB + (E == TreeElem::I8 ? 512 : 0) : 2 * PL * PLANE + 2 * T * 4;
    static constexpr int NBUF = COPY ? (WAVES == 8 && TILE <= 33 * 1024 ? 4 : 2)
                                : TILE > (NSET == 2 ? 66 : 40) * 1024 || (F32 && NSET == 2) ? 1 : 2;
    // q's low halves of 32 columns over f32 caches: in LDS, the registers do not hold them.
    static constexpr bool QLDS = F32 && NSET == 2;
    static constexpr int QBYTES = QLDS ? CW * NSET * NC * 1024 : 0;
    static constexpr int STEEP = F32 ? COLS * 4 : 0;  // what large queries leave of their power of two
    static constexpr int WGS = WAVES == 8 || (F32 && HDP == 256) ? 1 : 2;  // workgroups per CU
    // Operand reads from LDS that are on their way at once: units of two (16-key halves of a 32-dim
    // step, or two 16-dim groups of V), 8 registers each and plane.
    static constexpr int AHEAD = COPY ? (NSET == 2 || HDP == 256 ? 2 : std::min(NC, 4))
                                 : std::min(NC, HDP == 256 || NSET == 2 ? 1 : F32 ? 2 : 4);
    static_assert(NC % AHEAD == 0, "whole rounds");
    static_assert((KW - 1) * CW * (ND * 1024 + 512) <= TILE * NBUF, "room to join waves");
};

struct Args {
    const float *q;
    const char *k, *v;
    const uint8_t *ks, *vs;
    const char *tk, *tv;  // (block-scaled) rows from tail0 on
    const uint8_t *tks, *tvs, *bad;
    const unsigned *masks, *depths;
    float *o, *part_acc, *part_ml;
    int h, hkv, g, n, words, ncols, hd;
    unsigned g_inv;  // 2^32 / g, rounded up: exact for the at most 2^16 columns of a KV head
    int pos, window;
    int key0, tiles;  // the first key of tile 0; a tile at least
    int tail0;        // the first key of some tile
    int nsplit, ncb, pairs, block_log2;
    float scale;  // scale log2(e) / 2^scale_power
    int scale_power;
};

// 1 / l (to a step of f32: five of them meet in a result at most) for a sum of weights, which is at
// least about 1; 0 where no key was seen.
__device__ __forceinline__ float inverse(float l) { return l == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(l); }
// The largest of N neighbouring lanes' values, in each of them.
template <int N>
__device__ __forceinline__ float lanes_max(float x) {
    x = fmaxf(x, eb::dpp<eb::kDppQuadXor1>(x));
    x = fmaxf(x, eb::dpp<eb::kDppQuadXor2>(x));
    static_assert(N == 4 || N == 8 || N == 16 || N == 32 || N == 64, "a power of two from 4 to 64");
    if constexpr (N >= 8) x = fmaxf(x, eb::dpp<eb::kDppRowHalfMirror>(x));
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
// The scale of a block's exponent byte: 2^(e - 127), NaN for 255.
__device__ __forceinline__ float exponent_scale(unsigned e) {
    return __builtin_bit_cast(float, e == eb::kNanExponent ? 0x7FC00000u : e << 23);
}

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

// Where slot g (the keys of lane group g) of a dim lies in V's transposed rows of 64 bytes. Row
// (dim % 4) HDP / 4 + dim / 4: neighbouring lanes, whose dims are 4 apart where they store, and 4
// apart again where they read, meet neighbouring rows; the slots are xor-ed with the row.
template <int HDP>
__device__ __forceinline__ int v_row(int dim, int g) {
    const int row = (dim % 4) * (HDP / 4) + dim / 4;
    return row * 64 + ((g ^ ((row >> 2) & 3)) * 16);
}

// Whether one of four E4M3 patterns is NaN (0x7F and 0xFF: one more carries into the sign bit).
__device__ __forceinline__ bool has_nan_e4m3(unsigned w) { return (((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) != 0u; }
__device__ __forceinline__ bool has_nonfinite_f16(unsigned w) {
    return ((w & 0x7C00u) == 0x7C00u) | ((w & 0x7C000000u) == 0x7C000000u);
}

// x, computed here and not earlier: keeps what only rare branches need out of the common path.
template <class T>
__device__ __forceinline__ T here(T x) {
    asm volatile("" : "+v"(x));
    return x;
}

// x less the low (or high) half of h, one instruction (the compiler takes two).
__device__ __forceinline__ float less_low(float x, f16x2 h) {
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
    return r;
}
__device__ __forceinline__ float less_high(float x, f16x2 h) {
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
    return r;
}
// x as two halves, each rounded to nearest: 22 bits. x comes from ordinary vector instructions (no
// matrix instruction's result, which inline assembly would not wait for).
__device__ __forceinline__ void split(f32x8 x, f16x8 &hi, f16x8 &lo) {
    hi = __builtin_convertvector(x, f16x8);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const f16x2 h = {hi[i], hi[i + 1]};
        x[i] = less_low(x[i], h);
        x[i + 1] = less_high(x[i + 1], h);
    }
    lo = __builtin_convertvector(x, f16x8);
}

// Copies to LDS are inline assembly, which the compiler's wait counting does not see; they complete
// in issue order, so a tile is there when at most the later tiles' copies of this wave are under way
// (and, after a barrier, the other waves'). What the compiler itself waits for is then at worst waited
// for longer.
template <int N>
__device__ __forceinline__ void wait_copies() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Where piece c of row r lies in a copied row of RB bytes (in pieces): xor-ed with the row, so that
// neither 16 rows at one piece nor 4 rows at two meet a bank more often than their bytes ask for.
template <int RB>
__device__ __forceinline__ int piece_xor(int r) {
    return RB >= 256 ? r & 15 : RB == 128 ? (r >> 1) & 7 : (r >> 2) & 3;
}

// TAIL (block-scaled caches): keys from tail0 on are rows of the call's own, in place of the cache's, in blocks
// of 16.
template <int HDP, TreeElem E, int CW, int NSET, bool COPY, bool TAIL>
__global__ __launch_bounds__((Shape<HDP, E, CW, NSET, COPY>::THREADS),
                             (Shape<HDP, E, CW, NSET, COPY>::WGS * Shape<HDP, E, CW, NSET, COPY>::WAVES / 4))
void tree_attn_kernel(Args a) {
    using S = Shape<HDP, E, CW, NSET, COPY>;
    constexpr int ES = S::ES, T = S::T, KW = S::KW, PL = S::PL, PLANE = S::PLANE, HT = S::HT;
    constexpr int kWaves = S::WAVES, kThreads = S::THREADS;
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
    char *s_ql = smem + S::NBUF * S::TILE;  // [CW][NSET][NC][lane]
    float *s_steep = reinterpret_cast<float *>(s_ql + S::QBYTES);  // [columns] (f32 K)
    float *s_bad = reinterpret_cast<float *>(s_ql + S::QBYTES + S::STEEP);  // [T] (copied rows: 1, or NaN)
    int *s_any = reinterpret_cast<int *>(s_bad + T);  // (copied rows) a tile that has a row with NaN
    unsigned *s_mask = reinterpret_cast<unsigned *>(s_bad + (COPY ? T + 1 : 0));  // [nodes][words]
    int *s_depth = reinterpret_cast<int *>(s_mask + nodes * a.words);           // [n] (with a window)
    unsigned *s_nan = reinterpret_cast<unsigned *>(s_depth + (a.window > 0 ? a.n : 0));  // [8] (with a tail)

    // ---- tiles: fetched into registers, then stored as operands -----------------------------------
    const bool vside = wave >= kWaves / 2;
    const int ht = tid % HT;
    const size_t row_bytes = (size_t)a.hkv * hd * ES;
    const char *base = (vside ? a.v : a.k) + (size_t)kvh * hd * ES;
    const uint8_t *exps = vside ? a.vs : a.ks;
    // (so that the tail's rows and exponents are found by the same key)
    const char *tail_base = TAIL ? (vside ? a.tv : a.tk) + (size_t)kvh * hd - (size_t)a.tail0 * row_bytes : base;
    const uint8_t *tail_exps = TAIL ? (vside ? a.tvs : a.tks) - (size_t)(a.tail0 / 16) * a.hkv : exps;
    const unsigned lds0 = (unsigned)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char *)smem);
    unsigned piece[COPY ? S::CPW : 1];  // where this lane's pieces lie in a tile's rows
    if constexpr (COPY) {
#pragma unroll
        for (int i = 0; i < S::CPW; ++i) {
            const int at = ((wave % (kWaves / 2)) * S::CPW + i) * 64 + lane, r = at / S::CR;
            const int c = (at % S::CR) ^ piece_xor<S::RB>(r);
            piece[i] = c * S::LD < hd ? r * (unsigned)row_bytes + c * 16 : kNone;
        }
    }
    // Tile t to buffer b: rows [T][RB] of K, then of V; then the exponents of their 16-key pieces, [64]
    // words each. Past the last key, and past a row's dims, LDS gets zeros.
    auto copy = [&](int t, int b) {
        const int r0 = a.key0 + t * T;
        const int left = min(end - r0, T);
        const int nbytes = left > 0 ? (int)((left - 1) * row_bytes) + hd * ES : 0;
        const bool tail = TAIL && r0 >= a.tail0;
        const __amdgpu_buffer_rsrc_t res =
            eb::make_rsrc((tail ? tail_base : base) + (left > 0 ? (size_t)r0 * row_bytes : 0), nbytes);
        const unsigned dst = lds0 + b * S::TILE + (vside ? T * S::RB : 0) + (wave % (kWaves / 2)) * S::CPW * 1024;
#pragma unroll
        for (int i = 0; i < S::CPW; ++i)  // (a copy may read m0 one wait state after its write at the soonest)
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(dst + i * 1024),
                         "v"(piece[i]), "s"(res)
                         : "memory", "m0");
        if constexpr (E == TreeElem::I8) {  // (every wave the same words: the counts stay alike)
            const int bl = tail ? 4 : a.block_log2;
            const size_t b0 = left > 0 ? (size_t)(r0 >> bl) : 0;
            const int last = left > 0 ? (r0 + left - 1) >> bl : 0;
            const __amdgpu_buffer_rsrc_t eres = eb::make_rsrc(
                (tail ? tail_exps : exps) + b0 * a.hkv, left > 0 ? (last - (int)b0) * a.hkv + kvh + 1 : 0);
            const unsigned off = 16 * lane < left ? (((r0 + 16 * lane) >> bl) - (int)b0) * a.hkv + kvh : kNone;
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_ubyte %1, %2, 0 offen lds" ::"s"(
                             lds0 + b * S::TILE + 2 * T * S::RB + (vside ? 256 : 0)),
                         "v"(off), "s"(eres)
                         : "memory", "m0");
        }
    };
    unsigned raw[S::NR];
    auto fetch = [&](int t) {
        const int r0 = a.key0 + t * T;
        const int left = min(end - r0, T);
        const int nbytes = left > 0 ? (int)((left - 1) * row_bytes) + hd * ES : 0;
        const __amdgpu_buffer_rsrc_t res = eb::make_rsrc(base + (left > 0 ? (size_t)r0 * row_bytes : 0), nbytes);
        auto get = [&](int at, unsigned off) {
            const u32x4 w = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(res, off, 0, 0));
#pragma unroll
            for (int i = 0; i < 4; ++i) raw[at + i] = w[i];
        };
        // A lane whose dims the row does not have reads past the end from its first row on (unsigned
        // offsets do not wrap: kNone plus a tile's bytes).
        const unsigned rb = (unsigned)row_bytes;
        if (!vside) {
            const int c = ht % S::KL, r = ht / S::KL;
            if constexpr (S::F32) {
                const unsigned o0 = 8 * c < hd ? r * rb + c * 32 : kNone, o1 = 8 * c + 4 < hd ? o0 + 16 : kNone;
#pragma unroll
                for (int j = 0; j < S::KU; ++j) {
                    get(8 * j, o0 + j * (HT / S::KL) * rb);
                    get(8 * j + 4, o1 + j * (HT / S::KL) * rb);
                }
            } else {
                const unsigned o0 = c * S::LD < hd ? r * rb + c * 16 : kNone;
#pragma unroll
                for (int j = 0; j < S::KU; ++j) get(4 * j, o0 + j * (HT / S::KL) * rb);
            }
        } else {
#pragma unroll
            for (int j = 0; j < S::VU; ++j) {
                const int u = ht + j * HT, c = u % S::VC, sb = u / S::VC;
                const unsigned o0 = u < S::VUNITS && c * S::VD < hd ? (32 * (sb / 4) + 4 * (sb % 4)) * rb + c * S::VW * 4 : kNone;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const unsigned off = o0 + (i + (i & 4) * 3) * rb;
                    const int at = (8 * j + i) * S::VW;
                    if constexpr (S::VW == 4) {
                        get(at, off);
                    } else {
                        const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(res, off, 0, 0));
                        raw[at] = w[0];
                        raw[at + 1] = w[1];
                    }
                }
            }
        }
    };
    // The operands of a tile in LDS: K [planes][T][HDP], V [planes][KG][HDP][32], scales [2][T].
    auto store = [&](char *buf, bool edge) {
        float *s_scale = reinterpret_cast<float *>(buf + 2 * PL * PLANE);
        if (!vside) {
            const int c = ht % S::KL, r0 = ht / S::KL;
#pragma unroll
            for (int j = 0; j < S::KU; ++j) {
                const int r = r0 + j * (HT / S::KL);
                auto at = [&](int chunk) { return buf + (r * S::CH + (chunk ^ (r & S::SW))) * 16; };
                if constexpr (S::F32) {
                    f32x8 x;
                    float top = 0.0f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        x[i] = __uint_as_float(raw[8 * j + i]);
                        top = fmaxf(top, __uint_as_float(raw[8 * j + i] & 0x7FFFFFFFu));
                    }
                    const unsigned e = biased_exponent(lanes_max<S::KL>(top));
                    f16x8 hi, lo;
                    split(x * pow2_biased(267u - e), hi, lo);
                    *reinterpret_cast<f16x8 *>(at(c)) = hi;
                    *reinterpret_cast<f16x8 *>(at(c) + PLANE) = lo;
                    if (c == 0) s_scale[r] = pow2_biased(e - 13u) * kScoreShift;
                } else {
                    const bool whole = 16 * c + 8 < hd;  // (else the next head's)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const u32x2 x = narrow_f16<E>(raw[4 * j + 2 * half]), y = narrow_f16<E>(raw[4 * j + 2 * half + 1]);
                        u32x4 w = {x[0], x[1], y[0], y[1]};
                        if (half && !whole) w = u32x4{0u, 0u, 0u, 0u};
                        *reinterpret_cast<u32x4 *>(at(2 * c + half)) = w;
                    }
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
                        unsigned w[4];
#pragma unroll
                        for (int d = 0; d < 4; ++d) w[d] = raw[(8 * j + i) * 4 + d];
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
                        char *at = vt + v_row<HDP>(4 * c + d, g);
                        *reinterpret_cast<f16x8 *>(at) = hi;
                        *reinterpret_cast<f16x8 *>(at + PLANE) = lo;
                    }
                } else {
                    unsigned in[8][S::VW];
#pragma unroll
                    for (int i = 0; i < 8; ++i)
#pragma unroll
                        for (int d = 0; d < S::VW; ++d) in[i][d] = raw[(8 * j + i) * S::VW + d];
                    if (edge) {  // rows that are not finite: zeros, and NaN for the weight
                        float back[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            bool bad = false;
#pragma unroll
                            for (int d = 0; d < S::VW; ++d)  // (dims from hd on are the next head's)
                                bad = bad | (has_nan_e4m3(in[i][d]) & (c * S::VD + 4 * d < hd));
                            bad = lanes_max<S::VC>(bad ? 1.0f : 0.0f) > 0.0f;
#pragma unroll
                            for (int d = 0; d < S::VW; ++d) in[i][d] = bad ? 0u : in[i][d];
                            back[i] = bad ? __builtin_nanf("") : 1.0f;
                        }
                        if (c == 0) {
                            *reinterpret_cast<f32x4 *>(vs) = f32x4{back[0], back[1], back[2], back[3]};
                            *reinterpret_cast<f32x4 *>(vs + 16) = f32x4{back[4], back[5], back[6], back[7]};
                        }
                    }
#pragma unroll
                    for (int d0 = 0; d0 < S::VD; d0 += 4) {  // four dims: two words of f16 for each key
                        unsigned x[8][2];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const u32x2 p = narrow_f16<E>(in[i][d0 / 4]);
                            x[i][0] = p[0];
                            x[i][1] = p[1];
                        }
#pragma unroll
                        for (int d = 0; d < 4; ++d) {
                            const unsigned sel = d % 2 ? 0x07060302u : 0x05040100u;
                            u32x4 w;
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                w[i] = __builtin_amdgcn_perm(x[2 * i + 1][d / 2], x[2 * i][d / 2], sel);
                            const int dim = S::VD * c + d0 + d;
                            *reinterpret_cast<u32x4 *>(vt + v_row<HDP>(dim, g)) = w;
                        }
                    }
                }
            }
        }
    };

    int t = split_id;
    if constexpr (COPY)
        copy(t, 0);
    else
        fetch(t);

    // ---- the columns' queries, masks and first keys -------------------------------------------------
    const unsigned first_mask = tid < nodes * a.words ? a.masks[(size_t)node0 * a.words + tid] : 0u;
    const unsigned first_depth = a.window > 0 && tid < a.n ? a.depths[tid] : 0u;
    bool not_finite = false;  // (a node per thread) its row of K or V
    if constexpr (TAIL)
        if (tid < a.n) not_finite = (a.bad[(size_t)kvh * a.n + tid] | a.bad[(size_t)(a.hkv + kvh) * a.n + tid]) != 0;
    auto put_mask = [&](int i, unsigned w) {
        if (i % a.words == a.words - 1 && a.n % 32) w &= (1u << (a.n % 32)) - 1u;  // (no nodes past n)
        s_mask[i] = w;
    };
    const int cw = wave % CW, kw = wave / CW;
    const bool worker = kw < KW;  // (the others fetch and store only)
    // First of the 8 dims that a lane multiplies in 32-dim step i (copied bytes: a 16-byte piece holds
    // those of two steps).
    auto chunk_dim = [&](int i) { return COPY && ES == 1 ? 64 * (i / 2) + 16 * g4 + 8 * (i % 2) : 32 * i + 8 * g4; };
    f16x8 qh[NSET][S::NC], ql[NSET][S::QLDS ? 1 : S::NC];
    float qs[NSET];
    bool steep = false;  // (f32 K) a column's power of two, shifted, passes f32's range: s_steep has the rest
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
            const int d = chunk_dim(i);
            const f32x4 lo = __builtin_bit_cast(
                f32x4, __builtin_amdgcn_raw_buffer_load_b128(res, have && d < hd ? (unsigned)(at + d) * 4u : kNone, 0, 0));
            const f32x4 hi = __builtin_bit_cast(
                f32x4, __builtin_amdgcn_raw_buffer_load_b128(res, have && d + 4 < hd ? (unsigned)(at + d + 4) * 4u : kNone, 0, 0));
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[i][j] = j < 4 ? lo[j % 4] : hi[j % 4];
                top = fmaxf(top, fabsf(x[i][j]));
            }
        }
        top = fmaxf(top, eb::lane_xor16(top));
        top = fmaxf(top, eb::lane_xor32(top));
        // (q times scale log2(e), its largest in [2^13, 2^14) or, if the product rounds up, at 2^14; the scale as
        // a fraction and a power of two, which joins q's, since the product may pass f32's range)
        const unsigned e = biased_exponent(fabsf(top * a.scale));
        const int power = (int)e - 140 + a.scale_power + (S::F32 ? kScoreShiftLog2 : 0), most = min(power, 127);
        qs[s] = ldexpf(1.0f, most);
        if constexpr (S::F32) {
            steep = steep | (power > most);
            if (g4 == 0 && kw == 0) s_steep[(cw * NSET + s) * 16 + n] = ldexpf(1.0f, power - most);
        }
        const float f = pow2_biased(267u - e);
#pragma unroll
        for (int i = 0; i < S::NC; ++i) {
            f16x8 lo;
            split(x[i] * f * a.scale, qh[s][i], lo);
            if constexpr (S::QLDS) {
                if (kw == 0) *reinterpret_cast<f16x8 *>(s_ql + ((cw * NSET + s) * S::NC + i) * 1024 + lane * 16) = lo;
            } else {
                ql[s][i] = lo;
            }
        }
    }
    steep = __builtin_amdgcn_ballot_w64(steep) != 0;
    for (int i = tid; i < nodes * a.words; i += kThreads) put_mask(i, i == tid ? first_mask : a.masks[(size_t)node0 * a.words + i]);
    if (COPY && tid == 0) *s_any = -1;
    if (a.window > 0)
        if (tid < a.n) s_depth[tid] = (int)min(first_depth, 1u << 27);  // (a node per thread at most)
    if constexpr (TAIL) {
        const unsigned long long some = __builtin_amdgcn_ballot_w64(not_finite);
        if (lane < 2 && wave < 4) s_nan[2 * wave + lane] = (unsigned)(some >> (32 * lane));
    }
    __syncthreads();
    bool some_nan = false;  // (with a tail; uniform)
    if constexpr (TAIL) some_nan = __builtin_amdgcn_ballot_w64(s_nan[lane & 7] != 0u) != 0;
    int safe_lo = 0;  // keys below it may be behind some column's window
    bool shallow = true;  // no drafted key is behind any node's window
    if (a.window > 0) {
        int deepest = 0;
        for (int i = lane; i < nodes; i += 64) deepest = max(deepest, s_depth[node0 + i]);
#pragma unroll
        for (int m = 32; m > 0; m >>= 1) deepest = max(deepest, __shfl_xor(deepest, m));
        deepest = __builtin_amdgcn_readfirstlane(deepest);
        safe_lo = a.pos + deepest - a.window + 1;
        shallow = deepest < a.window;
    }
#pragma unroll
    for (int s = 0; s < NSET; ++s)
        my_first[s] = a.window > 0 ? a.pos + s_depth[node0 + my_node[s]] - a.window + 1 : 0;

    // ---- state --------------------------------------------------------------------------------------
    // ref: what a score's exponent is taken against (unscaled: less kUnit, so that weights and sums are
    // in units of 2^-kUnit); lcu: the unit of scaled weights.
    f32x4 acc[NSET][S::ND], lacc[NSET];
    float ref[NSET], l[NSET], lcu[NSET];
#pragma unroll
    for (int s = 0; s < NSET; ++s) {
        ref[s] = kNoRef;
        l[s] = 0.0f;
        lcu[s] = 0.0f;
        lacc[s] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < S::ND; ++e) acc[s][e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // One group of 32 keys from k0 on, in buf; edge: some may be hidden from some column.
    auto consume = [&](const char *buf, int kg, int k0, bool edge) {
        const float *s_scale = reinterpret_cast<const float *>(buf + 2 * PL * PLANE);  // (stored rows)
        const unsigned *s_exp = reinterpret_cast<const unsigned *>(buf + 2 * T * S::RB);  // (copied codes)
        f32x4 sc[NSET][2];
#pragma unroll
        for (int s = 0; s < NSET; ++s) sc[s][0] = sc[s][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        constexpr int AHEAD = S::AHEAD;
        constexpr bool BYTES = COPY && ES == 1;
        constexpr int VSHIFT = E == TreeElem::I8 ? 8 : 0;
        // Reads on their way: [unit][two][plane], as they lie in LDS (copied bytes: a K unit is the 16
        // dims of two steps, a V unit 8 bytes).
        u32x4 fr[AHEAD][2][PL];
        // Copied rows: piece c of a row is at its exclusive or with the row (piece_xor); a lane's own pieces
        // are those of step 0 (K) or group 0 (V) with the step's bits flipped, rows being aligned.
        typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
        const unsigned tile0 = (unsigned)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char *)buf);
        const int vr = BYTES ? 4 * g4 + ((n >> 1) & 3) : 4 * g4 + (n >> 2);  // (its row of the first 16)
        const unsigned k_at = tile0 + (32 * kg + n) * S::RB + ((g4 ^ piece_xor<S::RB>(n)) * 16);
        const unsigned v_at = tile0 + (T + 32 * kg + vr + (BYTES ? (n >> 3) * 16 : 0)) * S::RB + (n & 1) * 8 +
                              (((BYTES ? 0 : (n >> 1) & 1) ^ piece_xor<S::RB>(vr)) * 16);
        auto read_k = [&](int i) {
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                const int r = 32 * kg + 16 * sub + n;
                if constexpr (COPY) {
                    if (!BYTES || i % 2 == 0)
                        fr[i % AHEAD][sub][0] = *(const lds_u32x4 *)((k_at ^ (64 * (BYTES ? i / 2 : i))) + 16 * sub * S::RB);
                } else {
                    const char *at = buf + (r * S::CH + ((4 * i + g4) ^ (r & S::SW))) * 16;
#pragma unroll
                    for (int p = 0; p < PL; ++p) fr[i % AHEAD][sub][p] = *reinterpret_cast<const u32x4 *>(at + p * PLANE);
                }
            }
        };
        auto k_operand = [&](int i, int sub, int p) {
            if constexpr (BYTES) {
                const u32x4 w = fr[(i - i % 2) % AHEAD][sub][0];
                const u32x2 x = narrow_f16<E>(w[i % 2 * 2]), y = narrow_f16<E>(w[i % 2 * 2 + 1]);
                return __builtin_bit_cast(f16x8, u32x4{x[0], x[1], y[0], y[1]});
            } else {
                return __builtin_bit_cast(f16x8, fr[i % AHEAD][sub][p]);
            }
        };
        // V by keys in the lane's order: stored so (output group e = 4 q + d is dims 4 (16 q + n) + d, lane
        // n's row of V), or copied rows read across: 16 lanes read 16 dims of 4 keys (halves) or of 8 (bytes)
        // and get their own dim of each.
        const char *vt = buf + PL * PLANE + kg * (HDP * 64) + v_row<HDP>(4 * n, g4);  // (stored)
        auto read_v = [&](int u) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if constexpr (BYTES) {
                    const auto w = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                        (__attribute__((address_space(3))) i32x2 *)(v_at ^ (16 * (2 * u + e))));
                    fr[u % AHEAD][e][0][0] = w[0];
                    fr[u % AHEAD][e][0][1] = w[1];
                } else if constexpr (COPY) {
#pragma unroll
                    for (int sub = 0; sub < 2; ++sub) {
                        const auto w = __builtin_bit_cast(
                            u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((
                                       address_space(3))) i16x4 *)((v_at ^ (32 * (2 * u + e))) + 16 * sub * S::RB)));
                        fr[u % AHEAD][e][0][2 * sub] = w[0];
                        fr[u % AHEAD][e][0][2 * sub + 1] = w[1];
                    }
                } else {
#pragma unroll
                    for (int p = 0; p < PL; ++p)
                        fr[u % AHEAD][e][p] = *reinterpret_cast<const u32x4 *>(
                            vt + ((2 * u + e) % 4 * (HDP / 4) + (2 * u + e) / 4 * 16) * 64 + p * PLANE);
                }
            }
        };
        auto v_operand = [&](int u, int e, int p) {
            if constexpr (BYTES) {
                const u32x4 w = fr[u % AHEAD][e][0];
                const u32x2 x = narrow_f16<E>(w[0]), y = narrow_f16<E>(w[1]);
                return __builtin_bit_cast(f16x8, u32x4{x[0], x[1], y[0], y[1]});
            } else {
                return __builtin_bit_cast(f16x8, fr[u % AHEAD][e][p]);
            }
        };
        auto mfma = [](f16x8 x, f16x8 y, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0); };
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) read_k(i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < S::NC; ++i) {
            f16x8 lo[NSET];
#pragma unroll
            for (int s = 0; s < NSET; ++s) {
                if constexpr (S::QLDS)
                    lo[s] = *reinterpret_cast<const f16x8 *>(s_ql + ((cw * NSET + s) * S::NC + i) * 1024 + lane * 16);
                else
                    lo[s] = ql[s][i];
            }
            f16x8 k[2][PL];
#pragma unroll
            for (int sub = 0; sub < 2; ++sub)
#pragma unroll
                for (int p = 0; p < PL; ++p) k[sub][p] = k_operand(i, sub, p);
#pragma unroll
            for (int s = 0; s < NSET; ++s)
#pragma unroll
                for (int sub = 0; sub < 2; ++sub) sc[s][sub] = mfma(k[sub][0], qh[s][i], sc[s][sub]);
            if constexpr (PL == 2) {
#pragma unroll
                for (int s = 0; s < NSET; ++s)
#pragma unroll
                    for (int sub = 0; sub < 2; ++sub) sc[s][sub] = mfma(k[sub][PL - 1], qh[s][i], sc[s][sub]);
            }
#pragma unroll
            for (int s = 0; s < NSET; ++s)
#pragma unroll
                for (int sub = 0; sub < 2; ++sub) sc[s][sub] = mfma(k[sub][0], lo[s], sc[s][sub]);
            if constexpr (BYTES) {  // (a piece's second step frees it)
                if (i % 2 && i - 1 + AHEAD < S::NC) read_k(i - 1 + AHEAD);
            } else {
                if (i + AHEAD < S::NC) read_k(i + AHEAD);
            }
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) read_v(u);
        __builtin_amdgcn_sched_barrier(0);  // (on their way while the weights are formed)
        // Scales of the keys: one each (f32), or of their block, which 16 keys share (V's then times 2^-VSHIFT,
        // which the column's unit has instead: a weight of up to 2^8 times a scale of up to 2^122 stays finite).
        f32x4 ks[2], vs[2];
        if constexpr (S::SCALED) {
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                const float *at = s_scale + 32 * kg + 16 * sub;
                if constexpr (S::F32) {
                    ks[sub] = *reinterpret_cast<const f32x4 *>(at + 4 * g4);
                    vs[sub] = *reinterpret_cast<const f32x4 *>(at + T + 4 * g4);
                } else {
                    const float k1 = exponent_scale(s_exp[2 * kg + sub]);
                    const float v1 = exponent_scale(s_exp[64 + 2 * kg + sub]) * 0x1p-8f;
                    ks[sub] = f32x4{k1, k1, k1, k1};
                    vs[sub] = f32x4{v1, v1, v1, v1};
                }
            }
        }
        f16x8 ph[NSET], pl[NSET];
#pragma unroll
        for (int s = 0; s < NSET; ++s) {
            unsigned seen = 0xFFu;
            if (edge) {
                const unsigned *mask = s_mask + my_node[s] * a.words;
                seen = 0u;
#pragma unroll
                for (int sub = 0; sub < 2; ++sub) {  // four neighbouring keys; drafted from j = 0 on
                    const int key = k0 + 16 * sub + 4 * g4, j = key - a.pos, at = j >> 5;
                    const unsigned lo = at >= 0 && at < a.words ? mask[max(at, 0)] : 0u;
                    const unsigned hi = at + 1 >= 0 && at + 1 < a.words ? mask[max(at + 1, 0)] : 0u;
                    unsigned bits = __builtin_amdgcn_alignbit(hi, lo, (unsigned)j & 31u) & 15u;
                    if (!shallow) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int jj = min(max(j + i, 0), a.n - 1);
                            if (a.pos + s_depth[jj] < my_first[s]) bits &= ~(1u << i);
                        }
                    }
                    const unsigned cached = (1u << min(max(-j, 0), 4)) - 1u;
                    const unsigned before = (1u << min(max(my_first[s] - key, 0), 4)) - 1u;
                    seen |= ((bits & ~cached) | (cached & ~before)) << (4 * sub);
                }
            }
            float y[8], w[8], sum = 0.0f;  // y: scores before their column's factor
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                y[i] = sc[s][i / 4][i % 4];
                if constexpr (S::F32) y[i] *= ks[i / 4][i % 4];
            }
            if constexpr (S::F32)
                if (steep) {
                    const float rest = s_steep[(cw * NSET + s) * 16 + n];
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] *= rest;
                }
            // (Finite, so that a score of zero stays zero; a NaN block's stays NaN.)
            float qk[2] = {qs[s], qs[s]};
            if constexpr (E == TreeElem::I8)
#pragma unroll
                for (int i = 0; i < 2; ++i) qk[i] = __builtin_elementwise_minimum(qs[s] * ks[i][0], 0x1p127f);
            // Weights against the present reference and unit; where those do not serve, once more.
            for (bool again = true;; again = false) {
                const float cu = S::SCALED ? ldexpf(1.0f, (int)lcu[s] + VSHIFT) : 1.0f;
                float top = -INFINITY, least = INFINITY, most = 0.0f;
                sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    w[i] = __builtin_fmaf(y[i], qk[i / 4], -ref[s]);
                    if constexpr (E == TreeElem::F16) least = fminf(least, w[i]);
                }
                if constexpr (E == TreeElem::F16) least = here(least);
                if (edge) {
                    const unsigned bits = here(seen);
#pragma unroll
                    for (int i = 0; i < 8; ++i) w[i] = (bits >> i) & 1u ? w[i] : -INFINITY;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    top = fmaxf(top, w[i]);
                    w[i] = eb::fast_exp2(w[i]);
                    if constexpr (S::SCALED) {
                        sum += w[i];
                        // In this order: a row's scale and the column's unit together may pass f32's range
                        // beside a weight of zero or near it. What the first product loses below 2^-126 (2^-150)
                        // is, times a unit of at most 2^127, two of f16's least steps. (Block-scaled rows: eight
                        // products more a group than by a common factor, 0.5 to 2 % of a call.)
                        w[i] = w[i] * vs[i / 4][i % 4] * cu;
                        most = fmaxf(most, w[i]);
                    }
                }
                const bool over = (top > (S::SCALED ? kSlack : kSlack + kUnit)) | (most > kTop) | (least == -INFINITY);
                if (!again || __builtin_amdgcn_ballot_w64(over) == 0) break;
                float t1 = -INFINITY;
                const unsigned bits = here(seen);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    // (An infinite half of K meets q's two halves, whose signs may agree: infinity times 0
                    // is NaN whatever they gave. f32 rows' split made it NaN, E4M3 has no infinity.)
                    if constexpr (E == TreeElem::F16) y[i] = __builtin_fmaf(y[i], 0.0f, y[i]);
                    t1 = fmaxf(t1, (bits >> i) & 1u ? y[i] * qk[i / 4] : -INFINITY);
                }
                t1 = fmaxf(t1, eb::lane_xor16(t1));
                t1 = fmaxf(t1, eb::lane_xor32(t1));  // the column's largest score of the group
                if constexpr (!S::SCALED) t1 -= kUnit;
                const float rn = t1 > ref[s] + kSlack ? t1 : ref[s];
                const float d = ref[s] - rn;  // (-3e38 or so, or -inf, at the column's first keys)
                float f = d;
                if constexpr (S::SCALED) {
                    float big = 0.0f;  // the group's largest term
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float p = eb::fast_exp2(__builtin_fmaf(y[i], qk[i / 4], -rn)) * vs[i / 4][i % 4];
                        big = fmaxf(big, (bits >> i) & 1u ? p : 0.0f);
                    }
                    big = fmaxf(big, eb::lane_xor16(big));
                    big = fmaxf(big, eb::lane_xor32(big));
                    // Earlier terms lose 2^d: as much the unit may grow. Where this group's would pass
                    // 2^15 in it, its largest term becomes 2^6 to 2^7.
                    float unit = fminf(lcu[s] + floorf(-d), S::F32 ? 120.0f : 119.0f);
                    const float eb2 = (float)(__builtin_amdgcn_frexp_expf(big) + VSHIFT);
                    if (big > 0.0f && eb2 + unit > 15.0f) unit = 7.0f - eb2;
                    f = d + (unit - lcu[s]);
                    lcu[s] = unit;
                    l[s] *= eb::fast_exp2(d);
                }
                f = eb::fast_exp2(f);
                ref[s] = rn;
                lacc[s] *= f;
#pragma unroll
                for (int e = 0; e < S::ND; ++e) acc[s][e] *= f;
            }
            l[s] += sum;
            if (edge) {  // (a NaN scale does not reach what a column does not see)
                const unsigned bits = here(seen);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if constexpr (!S::SCALED)
                        w[i] *= (COPY ? s_bad : s_scale + T)[32 * kg + 16 * (i / 4) + 4 * g4 + i % 4];
                    if (!((bits >> i) & 1u)) w[i] = 0.0f;
                }
            }
            split(f32x8{w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]}, ph[s], pl[s]);
            if constexpr (!S::SCALED) {  // the weights' sum, as one more dim whose values are ones
                const _Float16 one = (_Float16)1.0f;
                const f16x8 ones = {one, one, one, one, one, one, one, one};
                lacc[s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, ph[s], lacc[s], 0, 0, 0);
                lacc[s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pl[s], lacc[s], 0, 0, 0);
            }
        }
#pragma unroll
        for (int u = 0; u < S::ND / 2; ++u) {
            f16x8 v[2][PL];
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int p = 0; p < PL; ++p) v[e][p] = v_operand(u, e, p);
#pragma unroll
            for (int s = 0; s < NSET; ++s)
#pragma unroll
                for (int e = 0; e < 2; ++e) acc[s][2 * u + e] = mfma(v[e][0], ph[s], acc[s][2 * u + e]);
            if constexpr (PL == 2) {
#pragma unroll
                for (int s = 0; s < NSET; ++s)
#pragma unroll
                    for (int e = 0; e < 2; ++e) acc[s][2 * u + e] = mfma(v[e][PL - 1], ph[s], acc[s][2 * u + e]);
            }
#pragma unroll
            for (int s = 0; s < NSET; ++s)
#pragma unroll
                for (int e = 0; e < 2; ++e) acc[s][2 * u + e] = mfma(v[e][0], pl[s], acc[s][2 * u + e]);
            if (u + AHEAD < S::ND / 2) read_v(u + AHEAD);
        }
    };

    // ---- the tiles ----------------------------------------------------------------------------------
    auto multiply = [&](const char *buf, int r0, bool edge) {
        if (!worker) return;
#pragma unroll 1
        for (int kg = kw; kg < S::KG; kg += KW) {
            if (r0 + 32 * kg >= end) break;
            consume(buf, kg, r0 + 32 * kg, edge);
        }
    };
    if constexpr (COPY) {
        constexpr int NB = S::NBUF;
        int b = 0;
#pragma unroll
        for (int i = 1; i < NB - 1; ++i) copy(t + i * a.nsplit, i);
        for (; t < a.tiles; t += a.nsplit) {
            char *buf = smem + b * S::TILE;
            const int r0 = a.key0 + t * T;
            const bool edge = r0 + T > a.pos || r0 < safe_lo;  // (uniform)
            wait_copies<(NB - 2) * S::CPT>();
            __syncthreads();  // tile t is there; tile t - 1's buffer is read no more
            copy(t + (NB - 1) * a.nsplit, b == 0 ? NB - 1 : b - 1);  // (past the last tile: of no keys)
            if constexpr (!S::SCALED) {
                if (edge) {  // V rows that are not finite: zeros, and NaN for the weight
                    for (int i = tid; i < T; i += kThreads) s_bad[i] = 1.0f;
                    u32x4 *v = reinterpret_cast<u32x4 *>(buf + T * S::RB);
                    auto is_bad = [&](int i) {
                        const u32x4 w = v[i];
                        bool bad = false;
#pragma unroll
                        for (int d = 0; d < 4; ++d) bad = bad | (ES == 2 ? has_nonfinite_f16(w[d]) : has_nan_e4m3(w[d]));
                        return bad;
                    };
                    bool any = false;
#pragma unroll
                    for (int i = 0; i < T * S::CR / kThreads; ++i) any = any | is_bad(i * kThreads + tid);
                    if (any) *s_any = t;
                    __syncthreads();
                    if (*s_any == t) {
                        for (int i = tid; i < T * S::CR; i += kThreads)
                            if (is_bad(i)) s_bad[i / S::CR] = __builtin_nanf("");
                        __syncthreads();
                        for (int i = tid; i < T * S::CR; i += kThreads)
                            if (s_bad[i / S::CR] != 1.0f) v[i] = u32x4{0u, 0u, 0u, 0u};
                        __syncthreads();
                    }
                }
            }
            multiply(buf, r0, edge);
            b = b == NB - 1 ? 0 : b + 1;
        }
        wait_copies<0>();  // (of no keys, but they write zeros to LDS)
    } else {
        for (int b = 0; t < a.tiles; t += a.nsplit, b ^= 1) {
            char *buf = smem + (S::NBUF == 2 && b ? S::TILE : 0);
            const int r0 = a.key0 + t * T;
            const bool edge = r0 + T > a.pos || r0 < safe_lo;
            store(buf, edge);
            if (t + a.nsplit < a.tiles) fetch(t + a.nsplit);
            __syncthreads();
            multiply(buf, r0, edge);
            if constexpr (S::NBUF == 1) __syncthreads();
        }
    }

    // ---- the waves' states meet ---------------------------------------------------------------------
    if constexpr (!S::SCALED) {
#pragma unroll
        for (int s = 0; s < NSET; ++s) l[s] = lacc[s][0];
    } else {
#pragma unroll
        for (int s = 0; s < NSET; ++s) {
            l[s] += eb::lane_xor16(l[s]);
            l[s] += eb::lane_xor32(l[s]);
        }
    }
    // A set's averages, out of their units. Where V may be of any size (SCALED) they are formed before
    // the waves' are joined: from there on nothing passes the size of V's own values.
    auto average = [&](int s) {
        const float inv = inverse(l[s]);
#pragma unroll
        for (int e = 0; e < S::ND; ++e) {
            acc[s][e] *= inv;
            if constexpr (S::SCALED)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[s][e][r] = ldexpf(acc[s][e][r], -(int)lcu[s]);
        }
    };
    if constexpr (S::SCALED)
#pragma unroll
        for (int s = 0; s < NSET; ++s) average(s);
    if constexpr (KW > 1) {  // a set at a time: into LDS, and to the first of the waves
        constexpr int SLOT = S::ND * 1024 + 512;  // bytes a wave leaves
#pragma unroll
        for (int s = 0; s < NSET; ++s) {
            __syncthreads();
            if (worker && kw > 0) {
                char *at = smem + ((kw - 1) * CW + cw) * SLOT;
#pragma unroll
                for (int e = 0; e < S::ND; ++e) *reinterpret_cast<f32x4 *>(at + e * 1024 + lane * 16) = acc[s][e];
                float *ml = reinterpret_cast<float *>(at + S::ND * 1024);
                ml[lane] = ref[s];
                ml[64 + lane] = l[s];
            }
            __syncthreads();
            if (kw == 0) {
#pragma unroll
                for (int w = 1; w < KW; ++w) {
                    const char *at = smem + ((w - 1) * CW + cw) * SLOT;
                    const float *ml = reinterpret_cast<const float *>(at + S::ND * 1024);
                    const float r2 = ml[lane], rn = fmaxf(ref[s], r2);
                    float f1 = eb::fast_exp2(ref[s] - rn), f2 = eb::fast_exp2(r2 - rn);
                    const float l1 = l[s] * f1, l2 = ml[64 + lane] * f2;
                    l[s] = l1 + l2;
                    ref[s] = rn;
                    if constexpr (S::SCALED) {
                        const float inv = inverse(l[s]);
                        f1 = l1 * inv;
                        f2 = l2 * inv;
                    }
#pragma unroll
                    for (int e = 0; e < S::ND; ++e)
                        acc[s][e] = acc[s][e] * f1 + f2 * *reinterpret_cast<const f32x4 *>(at + e * 1024 + lane * 16);
                }
            }
        }
        if (kw > 0) return;
    }
    if (!worker) return;
#pragma unroll
    for (int s = 0; s < NSET; ++s) {
        const int c = col0 + (cw * NSET + s) * 16 + n;
        if constexpr (!S::SCALED) {
            average(s);
            if (a.nsplit == 1) {  // (else the merge does so)
                float top[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // largest magnitudes (maximum, unlike fmaxf, keeps NaN)
#pragma unroll
                for (int e = 0; e < S::ND; ++e)
#pragma unroll
                    for (int r = 0; r < 4; ++r)  // (stored rows: dims from hd on are the next head's)
                        if (COPY || 64 * (e / 4) + 16 * g4 + 4 * r < hd)
                            top[r] = __builtin_elementwise_maximum(top[r], fabsf(acc[s][e][r]));
                float all = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top[0], top[1]),
                                                          __builtin_elementwise_maximum(top[2], top[3]));
                all = __builtin_elementwise_maximum(all, eb::lane_xor16(all));
                all = __builtin_elementwise_maximum(all, eb::lane_xor32(all));
                if (!(all < INFINITY)) {
                    const float nan = __builtin_nanf("");
#pragma unroll
                    for (int e = 0; e < S::ND; ++e) acc[s][e] = f32x4{nan, nan, nan, nan};
                }
            }
        }
        if (TAIL && some_nan) {  // drafted rows that are not finite: whom they reach
            bool hit = false;
            for (int w = 0; w < a.words; ++w)
                for (unsigned m = s_mask[my_node[s] * a.words + w] & s_nan[w]; m != 0; m &= m - 1)
                    hit = hit | (a.window == 0 || a.pos + s_depth[32 * w + __builtin_ctz(m)] >= my_first[s]);
            const float nan = __builtin_nanf("");
            if (hit)
#pragma unroll
                for (int e = 0; e < S::ND; ++e) acc[s][e] = f32x4{nan, nan, nan, nan};
        }
        if (c >= a.ncols) continue;
        const int node = node0 + my_node[s];
        const size_t row = (size_t)node * a.h + kvh * a.g + c - node * a.g;
        const size_t at = a.nsplit == 1 ? row : (size_t)split_id * a.n * a.h + row;
        float *out = (a.nsplit == 1 ? a.o : a.part_acc) + at * hd;
        if constexpr (COPY) {
#pragma unroll
            for (int e = 0; e < S::ND; ++e)
                if (16 * e + 4 * g4 < hd) *reinterpret_cast<f32x4 *>(out + 16 * e + 4 * g4) = acc[s][e];
        } else {
#pragma unroll
            for (int q = 0; q < S::ND / 4; ++q)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int d = 64 * q + 16 * g4 + 4 * r;
                    if (d < hd)
                        *reinterpret_cast<f32x4 *>(out + d) = f32x4{acc[s][4 * q][r], acc[s][4 * q + 1][r],
                                                                    acc[s][4 * q + 2][r], acc[s][4 * q + 3][r]};
                }
        }
        if (a.nsplit > 1 && g4 == 0) {
            a.part_ml[at * 2] = ref[s];
            a.part_ml[at * 2 + 1] = l[s];
        }
    }
}

// o[row] = average of the splits' averages, each weighed by its sum of weights at one reference. narrow: a
// row with a dim that is not finite becomes NaN (the sums of half and E4M3 values are finite otherwise).
// Workgroup: one row (node and head); a group of lanes holds the row's dims, four each, the groups share
// the splits, four at a time in flight. Bound by latency and its launch: 480 rows of 9 splits 4.0 us in a
// trace, 2048 rows of 16 (17 MB) 6.1 to 6.8.
constexpr int kMergeThreads = 256;
__global__ __launch_bounds__(kMergeThreads) void tree_merge_kernel(const float *__restrict__ part_acc,
                                                              const float *__restrict__ part_ml, float *__restrict__ o,
                                                              int rows, int hd, int nsplit, int lanes_log2,
                                                              bool narrow) {
    __shared__ float s_m[kMergeThreads], s_l[kMergeThreads];
    __shared__ f32x4 s_a[kMergeThreads];
    const int tid = threadIdx.x, row = blockIdx.x;
    const int groups = kMergeThreads >> lanes_log2;
    const int grp = tid >> lanes_log2, d = (tid & ((1 << lanes_log2) - 1)) * 4;
    const int at_d = d < hd ? d : 0;
    float M = kNoRef, L = 0.0f;
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
        float Ln = L * eb::fast_exp2(M - mn);
        const float had = Ln;
#pragma unroll
        for (int j = 0; j < B; ++j) {
            bl[j] = s0 + j * groups < nsplit ? bl[j] * eb::fast_exp2(bm[j] - mn) : 0.0f;
            Ln += bl[j];
        }
        const float inv = inverse(Ln);
        A *= had * inv;
#pragma unroll
        for (int j = 0; j < B; ++j)
            if (s0 + j * groups < nsplit) A += (bl[j] * inv) * ba[j];
        M = mn;
        L = Ln;
    }
    s_m[tid] = M;
    s_l[tid] = L;
    s_a[tid] = A;
    __syncthreads();
    if (grp > 0 || d >= hd) return;
    float mt = M;
    for (int g = 1; g < groups; ++g) mt = fmaxf(mt, s_m[(g << lanes_log2) + tid]);
    float Lt = 0.0f;
    for (int g = 0; g < groups; ++g) {
        const int i = (g << lanes_log2) + tid;
        Lt += eb::fast_exp2(s_m[i] - mt) * s_l[i];
    }
    const float inv = inverse(Lt);  // (no key seen: zeros)
    f32x4 At = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int g = 0; g < groups; ++g) {
        const int i = (g << lanes_log2) + tid;
        At += (eb::fast_exp2(s_m[i] - mt) * s_l[i] * inv) * s_a[i];
    }
    if (narrow) {  // (the row's lanes are one wave's)
        bool finite = true;
#pragma unroll
        for (int r = 0; r < 4; ++r) finite = finite & (fabsf(At[r]) < INFINITY);
        const float nan = __builtin_nanf("");
        if (__builtin_amdgcn_ballot_w64(!finite) != 0) At = f32x4{nan, nan, nan, nan};
    }
    *reinterpret_cast<f32x4 *>(o + (size_t)row * hd + d) = At;
}

struct Plan {
    int hdp, cols, ncb, key0, tiles, nsplit;
    bool copy;
};

// How many columns share a workgroup, and how many workgroups share the keys, by an estimate of the
// whole call's time (us): launch and a workgroup's start (queries, first tile), its tiles one after
// the other, and for several splits the merge's launch and what is written for it and read again. A
// tile costs its 32-key groups times 16-column sets at `set` each, times the workgroups that share the
// CU, but at least `chain` a group that one wave takes. Few columns start sooner and spread wider, many
// read each f32 key's operands and each half row for more of them. All sides measured (us; 32 heads over
// 8 of 128 unless said; in brackets the estimates for 16, 64 and 128 columns):
//   21 nodes behind 8191 block-scaled keys: 23.5, 27.5, 30.8 (23.7, 27.7, 27.5)
//   64 nodes behind  1000 half keys:        16.4, 18.0, 25.2 (17.1, 16.5, 19.2)
//   64 nodes behind 32000 half keys:         152,   86,   78 (174, 95.6, 82.9)
//   16 nodes behind 30000 half keys:          51, 35.3       (49.6, 33.2)
//   64 nodes behind  8000 f32 keys:                58.9, 52.9 (131, 60.8, 56.8)
//   16 nodes behind  8000 f32 keys:         41.7, 29.7       (41.3, 26.5)
//   16 nodes of 16 heads behind 200 E4M3 keys: 8.3 with one split, 10.9 with 64 columns (7.1, 10.7)
//   8 nodes of 16 heads behind 100 f32 keys: 10.5 with one split, 9.2 with four (16 columns)
// 64 nodes behind 1000 half keys thus take 64 columns where 16 are the faster by 1.6 us. The products grow with
// the dims and the softmax does not, hence the factor for other widths; 14 heads over 2 of 64, 16 over 8 of 256
// (16, 64 and 128 columns, each with its best splits; the rule takes the fastest of each row):
//   16 nodes of 64 behind 8000 half keys:   12.2, 12.8, 15.6 (12.4, 13.0, 15.0)
//   64 nodes of 64 behind 8000 half keys:   19.3, 17.5, 20.8 (20.0, 18.3, 19.5)
//   64 nodes of 64 behind 8000 f32 keys:    44.0, 25.7, 29.7 (45.4, 26.5, 26.8)
//   16 nodes of 64 behind 1000 block-scaled: 9.5, 12.0, 15.8 (9.7, 11.9, 13.7)
//   16 nodes of 256 behind 8000 f32 keys:   80.6, 51.2       (53.3, 35.0)
//   64 nodes of 256 behind 8000 half keys:  55.1, 38.2       (82.0, 35.2)
//   16 nodes of 256 behind 8000 block-scaled: 27.9, 29.8     (22.7, 23.7)
//   32 nodes of 256 behind 2000 E4M3 keys:  18.2, 23.0       (17.0, 18.0)
struct Cost {
    float set, chain;
};
Cost cost_of(int hdp, TreeElem e, int cols) {
    const int c = cols == 16 ? 0 : cols == 64 ? 1 : 2;
    static const Cost f32[3] = {{0.96f, 1.6f}, {0.335f, 1.6f}, {0.296f, 2.4f}};
    static const Cost f16[3] = {{0.28f, 1.3f}, {0.148f, 1.3f}, {0.112f, 2.0f}};
    static const Cost e4[3] = {{0.22f, 1.3f}, {0.15f, 1.3f}, {0.12f, 2.0f}};
    static const Cost i8[3] = {{0.24f, 1.5f}, {0.2f, 1.5f}, {0.15f, 2.2f}};
    const Cost *t = e == TreeElem::F32 ? f32 : e == TreeElem::F16 ? f16 : e == TreeElem::E4M3 ? e4 : i8;
    const float dims = (float)(hdp + 64) / 192.0f;  // (the products grow with the dims, the softmax does not)
    return Cost{t[c].set * dims, t[c].chain * dims};
}

bool copies(TreeElem e, size_t hd) { return e != TreeElem::F32 && (e != TreeElem::E4M3 || hd % 16 == 0); }

// The columns a workgroup may take, the largest number of splits, and the keys of a tile.
struct Width {
    int cols, cw, nset, wgs, T;
    size_t most;
};
int widths_of(size_t cols, size_t hkv, size_t hd, TreeElem e, int cu_count, Width (&w)[3]) {
    const int hdp = hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
    const bool copy = copies(e, hd);
    cu_count = std::min(cu_count, 1024);  // (a caller's number)
    int n = 0;
    for (const int c : {16, 64, 128}) {
        if ((c == 64 && cols <= 16) || (c == 128 && (cols <= 64 || hdp == 256))) continue;
        Width x{c, c == 16 ? 1 : 4, c == 128 ? 2 : 1, 0, 0, 0};
        x.wgs = waves_of(x.cw, x.nset, copy) == 8 || (e == TreeElem::F32 && hdp == 256) ? 1 : 2;
        x.T = 32 * key_groups(hdp, e, x.cw, x.nset, copy);
        x.most = std::max<size_t>(1, (size_t)cu_count * x.wgs / (hkv * ((cols + c - 1) / c)));
        w[n++] = x;
    }
    return n;
}

Plan plan_of(size_t h, size_t hkv, size_t hd, size_t pos, size_t n, size_t window, TreeElem elem, int cu_count) {
    const size_t cols = n * (h / hkv);
    Plan best{};
    best.hdp = hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
    best.copy = copies(elem, hd);
    best.key0 = (int)eb::tree_first_key(pos, window);
    const size_t keys = pos + n - best.key0;
    float least = 0.0f;
    Width widths[3];
    const int nw = widths_of(cols, hkv, hd, elem, cu_count, widths);
    for (int i = 0; i < nw; ++i) {
        const Width &w = widths[i];
        const size_t ncb = (cols + w.cols - 1) / w.cols, tiles = (keys + w.T - 1) / w.T;
        const Cost c = cost_of(best.hdp, elem, w.cols);
        const int sets = (int)std::min<size_t>(w.cols / 16, (cols + 15) / 16), kw = std::min(w.T / 32, w.cw == 1 ? 4 : w.nset == 2 || best.copy ? 2 : 1);
        const float start = 2.0f + (w.cols == 16 ? 2.5f : w.cols == 64 ? 3.5f : 4.5f);
        const size_t tries[] = {w.most, w.most * 3 / 4, w.most / 2, w.most / 3, w.most / 4, 4, 3, 2, 1};
        for (size_t s : tries) {
            s = std::min(std::min(std::max<size_t>(s, 1), w.most), tiles);
            const size_t per = (tiles + s - 1) / s;  // tiles of a split
            s = (tiles + per - 1) / per;
            const size_t wgs = hkv * ncb * s, room = (size_t)cu_count * w.wgs;
            const float shared = (float)std::min<size_t>(w.wgs, (wgs + cu_count - 1) / cu_count);
            const float tile = std::max(c.chain * (float)(w.T / 32 / kw), c.set * (float)(w.T / 32 * sets) * shared);
            float us = start + (float)((wgs + room - 1) / room) * tile * (float)per;
            if (s > 1) us += 4.0f + 8.0f * (float)(s * n * h * hd) / 4.0e6f;
            if (best.cols == 0 || us < least) {
                least = us;
                best.cols = w.cols;
                best.ncb = (int)ncb;
                best.tiles = (int)tiles;
                best.nsplit = (int)s;
            }
        }
    }
    return best;
}

template <int HDP, TreeElem E, int CW, int NSET, bool COPY, bool TAIL>
hipError_t launch(hipStream_t st, const Args &a) {
    using S = Shape<HDP, E, CW, NSET, COPY>;
    constexpr size_t kTiles = (size_t)S::NBUF * S::TILE + S::QBYTES + S::STEEP + (COPY ? S::T * 4 + 4 : 0);
    const size_t nodes = std::min<size_t>(a.n, S::COLS);
    const size_t lds = kTiles + (nodes * a.words + (a.window > 0 ? a.n : 0) + (TAIL ? 8 : 0)) * 4;
    constexpr size_t kMost = kTiles + (S::COLS * 8 + 256 + (TAIL ? 8 : 0)) * 4;
    static_assert(!TAIL || eb::kTailStep % S::T == 0, "a tail starts with a tile");
    static_assert(kMost <= 160 * 1024 / S::WGS, "LDS of a CU");
    const auto kernel = &tree_attn_kernel<HDP, E, CW, NSET, COPY, TAIL>;
    if (lds > 64 * 1024) {
        static const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                                        hipFuncAttributeMaxDynamicSharedMemorySize, (int)kMost);
        if (e != hipSuccess) return e;
    }
    const unsigned grid = (unsigned)((a.pairs + 7) / 8 * 8 * a.ncb);
    kernel<<<grid, S::THREADS, lds, st>>>(a);
    return hipSuccess;
}

template <int HDP, TreeElem E, bool COPY, bool TAIL>
hipError_t launch_cols(hipStream_t st, const Args &a, int cols) {
    if (cols == 16) return launch<HDP, E, 1, 1, COPY, TAIL>(st, a);
    if constexpr (HDP < 256)
        if (cols == 128) return launch<HDP, E, 4, 2, COPY, TAIL>(st, a);
    return launch<HDP, E, 4, 1, COPY, TAIL>(st, a);
}

template <TreeElem E, bool COPY, bool TAIL = false>
hipError_t launch_elem(hipStream_t st, const Args &a, const Plan &p) {
    if (p.hdp == 64) return launch_cols<64, E, COPY, TAIL>(st, a, p.cols);
    if constexpr (COPY || E == TreeElem::F32)  // (E4M3 rows that end inside a piece: at most 120 dims)
        if (p.hdp == 256) return launch_cols<256, E, COPY, TAIL>(st, a, p.cols);
    return launch_cols<128, E, COPY, TAIL>(st, a, p.cols);
}

}  // namespace

namespace eb {

// part_acc [nsplit, n * h, hd], part_ml [nsplit, n * h, 2], for the most splits that a call with any
// window may take.
size_t tree_attn_workspace_floats(size_t h, size_t hkv, size_t hd, size_t pos, size_t n, TreeElem elem, int cu_count) {
    if (n == 0) return 0;
    Width w[3];
    size_t splits = 1;
    for (int i = widths_of(n * (h / hkv), hkv, hd, elem, cu_count, w) - 1; i >= 0; --i)
        splits = std::max(splits, std::min(w[i].most, (pos + n + w[i].T - 1) / w[i].T));
    return splits > 1 ? splits * n * h * (hd + 2) : 0;
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
    if (x.tail) {
        a.tk = reinterpret_cast<const char *>(x.tail->k);
        a.tv = reinterpret_cast<const char *>(x.tail->v);
        a.tks = x.tail->ks;
        a.tvs = x.tail->vs;
        a.bad = x.tail->bad;
        a.tail0 = (int)x.tail->row0;
    }
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
    a.scale = std::frexp(x.scale * kLog2e, &a.scale_power);
    if (!std::isfinite(a.scale)) a.scale_power = 0;
    const hipError_t e = x.elem == TreeElem::F32   ? launch_elem<TreeElem::F32, false>(st, a, p)
                         : x.elem == TreeElem::F16 ? launch_elem<TreeElem::F16, true>(st, a, p)
                         : x.elem == TreeElem::I8  ? x.tail ? launch_elem<TreeElem::I8, true, true>(st, a, p)
                                                            : launch_elem<TreeElem::I8, true>(st, a, p)
                         : p.copy                  ? launch_elem<TreeElem::E4M3, true>(st, a, p)
                                                   : launch_elem<TreeElem::E4M3, false>(st, a, p);
    if (e != hipSuccess) return hip_fail(e, "attn_tree launch set-up");
    const eb_status s = check_launch("attn_tree");
    if (s != EB_OK || p.nsplit == 1) return s;
    int lanes_log2 = 0;
    while ((size_t)4 << lanes_log2 < x.hd) ++lanes_log2;
    tree_merge_kernel<<<(unsigned)rows, kMergeThreads, 0, st>>>(a.part_acc, a.part_ml, x.o, (int)rows, (int)x.hd, p.nsplit,
                                                           lanes_log2, x.elem == TreeElem::F16 || x.elem == TreeElem::E4M3);
    return check_launch("attn_tree (merge)");
}

}  // namespace eb
