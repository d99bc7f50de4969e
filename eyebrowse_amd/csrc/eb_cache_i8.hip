// Writing and reading the block-scaled 8-bit KV cache (eb_cache_i8.h) on gfx950. Both are bound
// by HBM: a write reads 4 bytes and stores 1 for each element, a read the reverse. 4096 rows of 8
// heads of 128, K and V: 10.1 and 9.6 us, 4.2 and 4.4 TB/s of the 5.1 that a large copy reaches; 37
// rows, a chain of loads: 4.3 and 2.6.
#include "eb_cache_i8.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kKept = 8;  // vectors of four that a thread keeps between its two passes

struct Side {  // K or V
    const float *src;  // [count, hkv, hd]
    uint8_t *codes;
    uint8_t *exps;
    uint32_t *tags;  // (eb::CacheI8)
};

// Workgroup (b, head, side): the new rows that fall into one block of one KV head, the block's
// earlier rows rounded again where its exponent grows. Two passes over the new rows: their
// largest magnitude, then their codes; the first kKept vectors of a thread stay in registers
// between them (a whole block of 64 rows of 128), the rest is read again, from L2. Earlier rows
// are touched only when the exponent grows. Nothing else writes these rows or this exponent, so
// there is no race and no atomic.
__global__ __launch_bounds__(kThreads) void kv_write_i8_kernel(Side k, Side v, int hkv, int hd, int block,
                                                               size_t dst, size_t count) {
    __shared__ unsigned s_max[kThreads / 64];
    const Side s = blockIdx.z ? v : k;
    const int head = blockIdx.y;
    const size_t b = dst / block + blockIdx.x;
    const size_t first = b * block;
    const size_t lo = first > dst ? first : dst;
    const size_t hi = first + block < dst + count ? first + block : dst + count;
    const int per_row = hd / 4;
    const int n = (int)(hi - lo) * per_row;  // vectors of four
    const size_t stride = (size_t)hkv * hd;
    const float *src = s.src + (lo - dst) * stride + (size_t)head * hd;
    uint8_t *codes = s.codes + (size_t)head * hd;
    const bool lead = first < lo;
    const unsigned old_e = lead ? s.exps[b * hkv + head] : 0u;

    auto load = [&](int i) {
        return *reinterpret_cast<const f32x4 *>(src + (size_t)(i / per_row) * stride + 4 * (i % per_row));
    };
    f32x4 kept[kKept];
    unsigned top = 0;  // largest magnitude, as bits: NaN is above infinity, both above all others
    auto take = [&](f32x4 x) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const unsigned a = eb::magnitude_bits(x[c]);
            top = a > top ? a : top;
        }
    };
#pragma unroll
    for (int j = 0; j < kKept; ++j) {
        const int i = (int)threadIdx.x + j * kThreads;
        kept[j] = i < n ? load(i) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
#pragma unroll
    for (int j = 0; j < kKept; ++j) take(kept[j]);
    for (int i = (int)threadIdx.x + kKept * kThreads; i < n; i += kThreads) take(load(i));
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) {
        const unsigned o = __shfl_xor(top, m);
        top = o > top ? o : top;
    }
    if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) top = s_max[w] > top ? s_max[w] : top;
    unsigned e = eb::i8_exponent(top);
    if (lead) e = eb::i8_join(old_e, e);

    auto store = [&](int i, f32x4 x) {
        unsigned w = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) w |= eb::i8_code(x[c], e) << (8 * c);
        *reinterpret_cast<unsigned *>(codes + (lo + i / per_row) * stride + 4 * (i % per_row)) = w;
    };
#pragma unroll
    for (int j = 0; j < kKept; ++j) {
        const int i = (int)threadIdx.x + j * kThreads;
        if (i < n) store(i, kept[j]);
    }
    for (int i = (int)threadIdx.x + kKept * kThreads; i < n; i += kThreads) store(i, load(i));
    if (lead && e != old_e && e != eb::kNanExponent) {
        const int m = (int)(lo - first) * per_row;
        for (int i = threadIdx.x; i < m; i += kThreads) {
            unsigned *p = reinterpret_cast<unsigned *>(codes + (first + i / per_row) * stride + 4 * (i % per_row));
            *p = eb::i8_recode(*p, old_e, e);
        }
    }
    if (threadIdx.x == 0) {
        s.exps[b * hkv + head] = (uint8_t)e;
        if (s.tags && blockIdx.x == 0) s.tags[eb::kTagWords * head] = 0;
    }
}

struct ReadSide {
    const uint8_t *codes, *exps;
    float *out;  // [count, hkv, hd]
};

// One thread per 8 codes: rows start.. of the cache as f32.
__global__ __launch_bounds__(kThreads) void kv_read_i8_kernel(ReadSide k, ReadSide v, int hkv, int hd, int block,
                                                              size_t start, size_t units) {
    const size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= units) return;
    const ReadSide s = blockIdx.y ? v : k;
    const size_t per_row = (size_t)hkv * hd / 8;
    const size_t row = start + i / per_row;
    const int head = (int)(i % per_row) * 8 / hd;
    const float f = eb::i8_scale(s.exps[row / block * hkv + head], 0);
    const u32x2 w = *reinterpret_cast<const u32x2 *>(s.codes + (start * per_row + i) * 8);
    f32x4 a, c;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        a[j] = eb::i8_f32(w[0], j) * f;
        c[j] = eb::i8_f32(w[1], j) * f;
    }
    f32x4 *out = reinterpret_cast<f32x4 *>(s.out + i * 8);
    out[0] = a;
    out[1] = c;
}

__global__ __launch_bounds__(kThreads) void fill_u8_kernel(uint8_t *p, uint8_t value, size_t n) {
    const size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x;
    if (i < n) p[i] = value;
}

}  // namespace

namespace eb {

// (a kernel, so that a captured graph holds one)
eb_status launch_fill_u8(hipStream_t st, uint8_t *p, uint8_t value, size_t n) {
    fill_u8_kernel<<<(unsigned)((n + kThreads - 1) / kThreads), kThreads, 0, st>>>(p, value, n);
    return check_launch("fill_u8");
}

eb_status launch_kv_write_i8(hipStream_t st, const CacheI8 &c, const float *k, const float *v, size_t dst,
                             size_t count) {
    const size_t blocks = (dst + count - 1) / c.block - dst / c.block + 1;
    const dim3 grid((unsigned)blocks, (unsigned)c.hkv, 2);
    kv_write_i8_kernel<<<grid, kThreads, 0, st>>>(Side{k, c.k, c.ks, c.tags},
                                                  Side{v, c.v, c.vs, c.tags ? c.tags + eb::kTagWords * c.hkv : nullptr},
                                                  (int)c.hkv, (int)c.hd, (int)c.block, dst, count);
    return check_launch("kv_write_i8");
}

eb_status launch_kv_read_i8(hipStream_t st, const CacheI8 &c, float *k, float *v, size_t start, size_t count) {
    const size_t units = count * c.hkv * c.hd / 8;
    const dim3 grid((unsigned)((units + kThreads - 1) / kThreads), 2);
    kv_read_i8_kernel<<<grid, kThreads, 0, st>>>(ReadSide{c.k, c.ks, k}, ReadSide{c.v, c.vs, v}, (int)c.hkv,
                                                 (int)c.hd, (int)c.block, start, units);
    return check_launch("kv_read_i8");
}

}  // namespace eb
