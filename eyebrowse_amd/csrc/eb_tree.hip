// A drafted tree's plan, the walk that accepts a branch of it, and the rows that are moved for that,
// for gfx950.
//
// Plan and walk are integers of at most kTreeMax nodes: one workgroup, a node per thread, bound by
// latency. Both follow parents by doubling: after r rounds a node knows its ancestors within 2^r
// steps, so a tree of depth d takes log2(d) rounds instead of d dependent reads. A round reads what was
// written to one half of LDS and the next one writes to the other, so one barrier parts them. Measured in
// a trace: 21 nodes 2.4 and 2.8 us, about what an empty launch takes; 256 nodes 5.4 to 5.8 and 4.4 to 4.9,
// four waves' LDS round trips and barriers (wider stores of the masks changed nothing).
//
// The copies are bound by HBM: every byte read once and written once.
#include "eb_cache_i8.h"
#include "eb_tree.h"

#include <algorithm>

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kNodes = (int)eb::kTreeMax;
constexpr int kWords = kNodes / 32;
constexpr int kThreads = 256;
constexpr unsigned kNobody = 0xFFFFFFFFu;
constexpr int kBlock = (int)eb::kTailBlock;

static_assert(kNodes == kThreads, "a node per thread");

// A parent is an earlier node; anything else is none.
__device__ __forceinline__ int parent_of(const int *parents, int i) {
    const int p = parents[i];
    return p >= 0 && p < i ? p : -1;
}

// Barrier of a round: whether any thread of the workgroup still has a way to go. What a thread wrote to
// half r of LDS before it is there for all after it.
__device__ __forceinline__ bool round_barrier(bool more, unsigned (&s_more)[kNodes / 64]) {
    const unsigned any = __ballot(more) != 0;
    if ((threadIdx.x & 63) == 0) s_more[threadIdx.x / 64] = any;
    __syncthreads();
    unsigned all = 0;
    for (unsigned w = 0; w * 64 < blockDim.x; ++w) all |= s_more[w];
    return all != 0;
}

// masks[i] = node i and its ancestors, as bits; depths[i] = how many ancestors it has.
__global__ __launch_bounds__(kThreads) void tree_plan_kernel(const int *__restrict__ parents,
                                                             unsigned *__restrict__ masks,
                                                             unsigned *__restrict__ depths, int n) {
    __shared__ u32x4 s_mask[2][kWords / 4][kNodes];
    __shared__ int s_up[2][kNodes];
    __shared__ unsigned s_more[2][kNodes / 64];
    const int i = threadIdx.x;
    const int words = (n + 31) / 32;
    int up = i < n ? parent_of(parents, i) : -1;
    u32x4 mask[kWords / 4];
#pragma unroll
    for (int w = 0; w < kWords; ++w) mask[w / 4][w % 4] = w == i / 32 ? 1u << (i % 32) : 0u;
    for (int r = 0;; r ^= 1) {
        s_up[r][i] = up;
#pragma unroll
        for (int w = 0; w < kWords / 4; ++w)
            if (4 * w < words) s_mask[r][w][i] = mask[w];
        if (!round_barrier(up >= 0, s_more[r])) break;
        if (up >= 0) {
#pragma unroll
            for (int w = 0; w < kWords / 4; ++w)
                if (4 * w < words) mask[w] |= s_mask[r][w][up];
            up = s_up[r][up];
        }
    }
    if (i >= n) return;
    int depth = -1;
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
        if (w >= words) continue;
        masks[i * words + w] = mask[w / 4][w % 4];
        depth += __popc(mask[w / 4][w % 4]);
    }
    depths[i] = (unsigned)depth;
}

// The branch that the model's own tokens follow from node 0: from a node on to its first child whose
// token is the node's sampled one. path[j] = its j-th node, emitted[j] = that node's sampled token.
__global__ __launch_bounds__(kThreads) void tree_accept_kernel(const unsigned *__restrict__ tokens,
                                                               const int *__restrict__ parents,
                                                               const unsigned *__restrict__ sampled,
                                                               unsigned *__restrict__ path,
                                                               unsigned *__restrict__ emitted,
                                                               unsigned *__restrict__ count, int n) {
    __shared__ unsigned s_sampled[kNodes], s_first[kNodes];
    __shared__ unsigned s_state[2][kNodes];  // whether taken so far, and the distance to `up`
    __shared__ int s_up[2][kNodes];
    __shared__ unsigned s_more[2][kNodes / 64];
    const int i = threadIdx.x;
    const bool in = i < n;
    int up = in && i > 0 ? parent_of(parents, i) : -1;
    const unsigned token = in ? tokens[i] : 0u, mine = in ? sampled[i] : 0u;
    s_sampled[i] = mine;
    s_first[i] = kNobody;
    __syncthreads();
    if (up >= 0 && token == s_sampled[up]) atomicMin(&s_first[up], (unsigned)i);
    __syncthreads();
    // Taken from its parent; then from all ancestors up to node 0, `dist` steps away.
    unsigned ok = i == 0 || (up >= 0 && s_first[up] == (unsigned)i);
    unsigned dist = up >= 0 ? 1 : 0;
    for (int r = 0;; r ^= 1) {
        s_state[r][i] = dist * 2 + ok;
        s_up[r][i] = up;
        if (!round_barrier(up >= 0, s_more[r])) break;
        if (up >= 0) {
            const unsigned state = s_state[r][up];
            ok &= state;
            dist += state >> 1;
            up = s_up[r][up];
        }
    }
    const int accepted = __syncthreads_count(in && ok);
    if (!in) return;
    if (i >= accepted) path[i] = emitted[i] = kNobody;
    if (ok) {
        path[dist] = (unsigned)i;
        emitted[dist] = mine;
    }
    if (i == 0) *count = (unsigned)accepted;
}

// A path of rows to move, as a kernel takes it: as long as its entries are nodes and increase, hence
// path[j] >= j, and a row is read before, or by the same thread that, another one is moved onto it.
// Returns its length; the entries are in s_path.
__device__ __forceinline__ int load_path(const unsigned *path, const unsigned *count, int n, unsigned *s_path,
                                         unsigned *s_end) {
    const int i = threadIdx.x;
    const unsigned c = *count;
    if (i == 0) *s_end = c < (unsigned)n ? c : (unsigned)n;
    const unsigned p = i < n ? path[i] : kNobody;
    s_path[i] = p;
    __syncthreads();
    if (i < n && (p >= (unsigned)n || (i > 0 && p <= s_path[i - 1]))) atomicMin(s_end, (unsigned)i);
    __syncthreads();
    return (int)*s_end;
}

constexpr int kMaxLayers = (int)eb::kMoveLayers;
struct CompactArgs {
    eb::CacheRows layer[kMaxLayers];
    const unsigned *path, *count;
    size_t pos;
    int n;
};

// Workgroup (x, layer and side): 256 vectors of V of each row. A thread moves its vector of every row,
// kBatch rows read before the first is written. Latency binds it (path and count, then the rows, two
// dependent reads): 5 of 21 rows in 28 layers of 4 KB rows 3.3 us, 12 of 64 in 32 layers 4.7.
template <class V>
__global__ __launch_bounds__(kThreads) void kv_compact_kernel(CompactArgs a) {
    __shared__ unsigned s_path[kNodes];
    __shared__ unsigned s_end;
    constexpr int kBatch = 8;
    const eb::CacheRows &layer = a.layer[blockIdx.y >> 1];
    V *cache = static_cast<V *>(blockIdx.y & 1 ? layer.v : layer.k);
    const size_t per_row = layer.row_bytes / sizeof(V);
    const int end = load_path(a.path, a.count, a.n, s_path, &s_end);
    const size_t x = (size_t)blockIdx.x * kThreads + threadIdx.x;
    if (x >= per_row) return;
    cache += a.pos * per_row + x;
    int j = 0;
    while (j < end && s_path[j] == (unsigned)j) ++j;  // (rows that stay)
    for (; j < end; j += kBatch) {
        V row[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
            if (j + b < end) row[b] = cache[s_path[j + b] * per_row];
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
            if (j + b < end) cache[(j + b) * per_row] = row[b];
    }
}

struct DraftSide {
    const float *rows;     // [n, hkv, hd]
    const uint8_t *codes, *exps;
    uint8_t *tail_codes, *tail_exps, *bad;
    unsigned *tags;
};
struct DraftArgs {
    DraftSide k, v;
    int row0, pos, n, hkv, hd, block_log2;
    u32x4 tag;  // as written: the cache's number, pos, n
};

// Workgroup (b, head, side): 16 rows of the tail, of one KV head: the cache's rows before pos, in the exponent
// that a write of the block's drafted rows gives it, and those rows' codes. A row that is not finite is zeros
// and a mark instead. The cache itself is not touched. Bound by latency: every load is on its way before the
// first wait (in a trace, 8 heads of 128: 8 nodes behind 100 keys 3.4 us, 21 behind 8191 3.5; a write of the
// same rows into the cache 3.1).
__global__ __launch_bounds__(kThreads) void kv_draft_i8_kernel(DraftArgs a) {
    __shared__ unsigned s_max[2][kThreads / 64];
    __shared__ unsigned s_bad[kBlock];
    constexpr int kNew = kBlock * 256 / 4 / kThreads;  // vectors of a thread, at the widest head
    static_assert(kBlock * 256 / 16 <= kThreads, "a vector of old rows a thread");
    const DraftSide &s = blockIdx.z ? a.v : a.k;
    const int head = blockIdx.y, tid = threadIdx.x;
    const int first = a.row0 + (int)blockIdx.x * kBlock, behind = first + kBlock;  // (row0 is a multiple of 16)
    const int lo = max(first, a.pos), hi = min(behind, a.pos + a.n);
    const int per_row = a.hd / 4, per_old = a.hd / 16;
    const int rows = max(hi - lo, 0), vecs = rows * per_row;  // drafted ones
    const int kept = max(min(behind, a.pos) - first, 0) * per_old;  // the cache's
    const size_t stride = (size_t)a.hkv * a.hd, head0 = (size_t)head * a.hd;
    const float *src = s.rows + (lo - a.pos) * stride + head0;
    uint8_t *new_dst = s.tail_codes + (lo - a.row0) * stride + head0;
    const bool lead = first < a.pos;
    auto load = [&](int i) {
        return *reinterpret_cast<const f32x4 *>(src + (size_t)(i / per_row) * stride + 4 * (i % per_row));
    };
    auto magnitude = [](f32x4 x) {
        unsigned top = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) top = max(top, eb::magnitude_bits(x[c]));
        return top;
    };
    auto join = [&](unsigned top, unsigned (&to_all)[kThreads / 64]) {  // the workgroup's largest
#pragma unroll
        for (int m = 32; m > 0; m >>= 1) top = max(top, __shfl_xor(top, m));
        if ((tid & 63) == 0) to_all[tid >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kThreads / 64; ++w) top = max(top, to_all[w]);
        return top;
    };
    const unsigned old_e = lead ? s.exps[(size_t)(first >> a.block_log2) * a.hkv + head] : 0u;
    f32x4 fresh[kNew];
    u32x4 old = {0u, 0u, 0u, 0u};
    const size_t old_at = (size_t)(tid / per_old) * stride + head0 + 16 * (tid % per_old);
#pragma unroll
    for (int j = 0; j < kNew; ++j)
        fresh[j] = tid + j * kThreads < vecs ? load(tid + j * kThreads) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (tid < kept) old = *reinterpret_cast<const u32x4 *>(s.codes + first * stride + old_at);
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < kNew; ++j) top = max(top, magnitude(fresh[j]));
    if (tid < rows) s_bad[tid] = 0;
    top = join(top, s_max[0]);
    const bool some_bad = top >= 0x7F800000u;  // (uniform)
    if (some_bad) {  // the rows that are not finite, and the others' largest
#pragma unroll
        for (int j = 0; j < kNew; ++j)
            if (magnitude(fresh[j]) >= 0x7F800000u) s_bad[(tid + j * kThreads) / per_row] = 1;
        __syncthreads();
        top = 0;
#pragma unroll
        for (int j = 0; j < kNew; ++j)
            if (tid + j * kThreads < vecs && !s_bad[(tid + j * kThreads) / per_row]) top = max(top, magnitude(fresh[j]));
        top = join(top, s_max[1]);
    }
    unsigned e = eb::i8_exponent(top);
    if (lead) e = rows > 0 ? eb::i8_join(old_e, e) : old_e;
#pragma unroll
    for (int j = 0; j < kNew; ++j) {
        const int i = tid + j * kThreads;
        if (i >= vecs) continue;
        unsigned w = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) w |= eb::i8_code(fresh[j][c], e) << (8 * c);
        if (some_bad && s_bad[i / per_row]) w = 0;
        *reinterpret_cast<unsigned *>(new_dst + (size_t)(i / per_row) * stride + 4 * (i % per_row)) = w;
    }
    if (tid < kept) {
        if (e != old_e && e != eb::kNanExponent)
#pragma unroll
            for (int c = 0; c < 4; ++c) old[c] = eb::i8_recode(old[c], old_e, e);
        *reinterpret_cast<u32x4 *>(s.tail_codes + (first - a.row0) * stride + old_at) = old;
    }
    if (tid < rows) s.bad[(size_t)head * a.n + (lo - a.pos) + tid] = (uint8_t)s_bad[tid];
    if (tid == 0) {
        s.tail_exps[blockIdx.x * a.hkv + head] = (uint8_t)e;
        if (blockIdx.x == 0) reinterpret_cast<u32x4 *>(s.tags)[head] = a.tag;
    }
}

struct CompactI8Args {
    struct Layer {
        uint8_t *codes[2], *exps[2];
        const float *draft[2];
        int hd;
    } layer[kMaxLayers];
    const unsigned *path, *count;
    unsigned *tags;  // of the first layer, and on
    unsigned id_lo, id_hi;
    size_t pos;
    int n, hkv, block;
};

// Workgroup (head, layer and side): the branch's rows as the values they stand for, written at pos as
// any rows are: block by block, with the least exponent that holds them and the block's earlier rows.
// They are the draft's that lies beside the cache, where that is one of pos, which is then done with; else
// the cache's own rows from pos on.
// All of these' codes and exponents are in LDS before the first is overwritten; no other workgroup touches them.
// Bound by latency (path, rows, then a block after another, with three barriers each): 8 heads of 128, the
// cache's rows: 5 of 21 in 28 layers 5.2 us, 8 of 64 in 32 layers 6.2, 64 of 256 12.4.
__global__ __launch_bounds__(kThreads) void kv_compact_i8_kernel(CompactI8Args a) {
    extern __shared__ unsigned s_code[];  // [n][hd / 4] (rows of the cache)
    __shared__ unsigned s_path[kNodes], s_exp[kNodes];
    __shared__ unsigned s_end, s_top;
    const CompactI8Args::Layer &layer = a.layer[blockIdx.y >> 1];
    const int side = blockIdx.y & 1, head = blockIdx.x, tid = threadIdx.x;
    const int per_row = layer.hd / 4;
    const size_t stride = (size_t)a.hkv * layer.hd;
    uint8_t *codes = layer.codes[side] + (size_t)head * layer.hd;
    uint8_t *exps = layer.exps[side] + head;
    u32x4 *tags = reinterpret_cast<u32x4 *>(a.tags) + (size_t)blockIdx.y * a.hkv + head;
    const u32x4 tag = *tags;
    const float *draft = nullptr;
    if (tag[0] == a.id_lo && tag[1] == a.id_hi && tag[2] == (unsigned)a.pos) draft = layer.draft[side];
    const int end = load_path(a.path, a.count, draft ? min(a.n, (int)tag[3]) : a.n, s_path, &s_end);
    if (tid == 0) *tags = u32x4{0u, 0u, 0u, 0u};  // (every thread has read it: load_path's barriers)
    if (draft) draft += (size_t)head * layer.hd;
    auto word = [&](size_t row, int w) { return reinterpret_cast<unsigned *>(codes + row * stride + 4 * w); };
    if (!draft) {
        for (int i = tid; i < end * per_row; i += kThreads) s_code[i] = *word(a.pos + s_path[i / per_row], i % per_row);
        if (tid < end) s_exp[tid] = exps[(a.pos + s_path[tid]) / a.block * a.hkv];
        __syncthreads();
    }
    auto values = [&](int i) {  // four of the branch's row i / per_row
        if (draft) return *reinterpret_cast<const f32x4 *>(draft + s_path[i / per_row] * stride + 4 * (i % per_row));
        const float f = eb::i8_scale(s_exp[i / per_row], 0);
        f32x4 x;
#pragma unroll
        for (int c = 0; c < 4; ++c) x[c] = eb::i8_f32(s_code[i], c) * f;
        return x;
    };
    for (int lo = 0; lo < end;) {
        const size_t b = (a.pos + lo) / a.block, first = b * a.block;
        const int hi = (int)(first + a.block - a.pos) < end ? (int)(first + a.block - a.pos) : end;
        const int lead = lo == 0 ? (int)(a.pos - first) : 0;  // earlier rows of the block
        if (tid == 0) s_top = 0;
        __syncthreads();
        unsigned top = 0;
        f32x4 kept = {0.0f, 0.0f, 0.0f, 0.0f};  // a thread's first
        for (int i = lo * per_row + tid, i0 = i; i < hi * per_row; i += kThreads) {
            const f32x4 x = values(i);
            if (i == i0) kept = x;
#pragma unroll
            for (int c = 0; c < 4; ++c) top = max(top, eb::magnitude_bits(x[c]));
        }
#pragma unroll
        for (int m = 32; m > 0; m >>= 1) top = max(top, __shfl_xor(top, m));
        if ((tid & 63) == 0) atomicMax(&s_top, top);
        const unsigned old_e = lead ? exps[b * a.hkv] : 0u;
        __syncthreads();
        unsigned e = eb::i8_exponent(s_top);
        if (lead) e = eb::i8_join(old_e, e);
        for (int i = lo * per_row + tid, i0 = i; i < hi * per_row; i += kThreads) {
            const f32x4 x = i == i0 ? kept : values(i);
            unsigned w = 0;
#pragma unroll
            for (int c = 0; c < 4; ++c) w |= eb::i8_code(x[c], e) << (8 * c);
            *word(a.pos + i / per_row, i % per_row) = w;
        }
        if (lead && e != old_e && e != eb::kNanExponent) {
            for (int i = tid; i < lead * per_row; i += kThreads) {
                unsigned *p = word(first + i / per_row, i % per_row);
                *p = eb::i8_recode(*p, old_e, e);
            }
        }
        __syncthreads();  // (every thread has read the old exponent and s_top)
        if (tid == 0) exps[b * a.hkv] = (uint8_t)e;
        lo = hi;
    }
}

constexpr int kMaxRuns = 2 * kMaxLayers;
constexpr size_t kRunChunk = (size_t)kThreads * 16;  // bytes a workgroup copies
struct RunArgs {
    eb::ByteRun run[kMaxRuns];
};

// Workgroup (x, run): chunk x of the run, one 16-byte vector a thread; a run's last 15 bytes one by
// one. The stores are non-temporal: nothing reads the copy soon. One vector a thread keeps more waves
// with a load on the way than several do: 64 runs of 16.4 MB (an 8000-row f16 cache of 32 layers) take
// 331 us (6.3 TB/s), with 2 vectors 354, with 4 337 to 368, with 8 493; 56 runs of 1.4 MB 23.0 us, with
// 8 vectors 43.4; stores that stay in the caches 342 and 22.7.
__global__ __launch_bounds__(kThreads) void copy_runs_kernel(RunArgs a) {
    const eb::ByteRun &r = a.run[blockIdx.y];
    const size_t at = (size_t)blockIdx.x * kRunChunk;
    if (at >= r.bytes) return;
    const size_t vecs = r.bytes / 16, v = at / 16 + threadIdx.x;
    if (v < vecs)
        __builtin_nontemporal_store(static_cast<const u32x4 *>(r.src)[v], static_cast<u32x4 *>(r.dst) + v);
    if (at + kRunChunk >= r.bytes && threadIdx.x < r.bytes % 16) {
        const size_t t = vecs * 16 + threadIdx.x;
        static_cast<uint8_t *>(r.dst)[t] = static_cast<const uint8_t *>(r.src)[t];
    }
}

}  // namespace

namespace eb {

static unsigned threads_of(size_t n) { return (unsigned)((n + 63) / 64 * 64); }

eb_status launch_tree_plan(hipStream_t st, const int32_t *parents, uint32_t *masks, uint32_t *depths, size_t n) {
    tree_plan_kernel<<<1, threads_of(n), 0, st>>>(parents, masks, depths, (int)n);
    return check_launch("tree_plan");
}

eb_status launch_tree_accept(hipStream_t st, const uint32_t *tokens, const int32_t *parents, const uint32_t *sampled,
                             uint32_t *path, uint32_t *emitted, uint32_t *count, size_t n) {
    tree_accept_kernel<<<1, threads_of(n), 0, st>>>(tokens, parents, sampled, path, emitted, count, (int)n);
    return check_launch("tree_accept");
}

eb_status launch_kv_compact(hipStream_t st, const CacheRows *layers, size_t n_layers, const uint32_t *path,
                            const uint32_t *count, size_t n, size_t pos) {
    CompactArgs a{};
    a.path = path;
    a.count = count;
    a.pos = pos;
    a.n = (int)n;
    size_t most = 0;
    bool wide = true;
    for (size_t l = 0; l < n_layers; ++l) {
        a.layer[l] = layers[l];
        most = std::max(most, layers[l].row_bytes);
        wide = wide && layers[l].row_bytes % 16 == 0;
    }
    if (most == 0) return EB_OK;
    const size_t per_wg = kThreads * (wide ? 16 : 4);
    const dim3 grid((unsigned)((most + per_wg - 1) / per_wg), (unsigned)(2 * n_layers));
    if (wide)
        kv_compact_kernel<u32x4><<<grid, kThreads, 0, st>>>(a);
    else
        kv_compact_kernel<unsigned><<<grid, kThreads, 0, st>>>(a);
    return check_launch("kv_compact");
}

eb_status launch_kv_draft_i8(hipStream_t st, const CacheI8 &c, const DraftRows &d, const DraftTail &t, size_t pos,
                             size_t n) {
    DraftArgs a{};
    a.k = DraftSide{d.k, c.k, c.ks, t.k, t.ks, t.bad, c.tags};
    a.v = DraftSide{d.v, c.v, c.vs, t.v, t.vs, t.bad + c.hkv * n, c.tags + kTagWords * c.hkv};
    a.row0 = (int)t.row0;
    a.pos = (int)pos;
    a.n = (int)n;
    a.hkv = (int)c.hkv;
    a.hd = (int)c.hd;
    a.tag = u32x4{(unsigned)c.id, (unsigned)(c.id >> 32), (unsigned)pos, (unsigned)n};
    while ((size_t)1 << a.block_log2 < c.block) ++a.block_log2;
    const size_t blocks = (pos + n - 1 - t.row0) / kTailBlock + 1;
    if (blocks > tree_tail_blocks(n) || pos + n - t.row0 > tree_tail_rows(n) || t.row0 % kTailBlock)
        return fail(EB_OTHER, "kv_draft_i8: rows %zu to %zu do not fit the tail", t.row0, pos + n);
    kv_draft_i8_kernel<<<dim3((unsigned)blocks, (unsigned)c.hkv, 2), kThreads, 0, st>>>(a);
    return check_launch("kv_draft_i8");
}

eb_status launch_kv_compact_i8(hipStream_t st, const CacheI8 *layers, const DraftRows *drafts, size_t n_layers,
                               const uint32_t *path, const uint32_t *count, size_t n, size_t pos) {
    CompactI8Args a{};
    static_assert(sizeof(a) <= 4096, "kernel arguments");
    a.path = path;
    a.count = count;
    a.pos = pos;
    a.n = (int)n;
    size_t hd = 0;
    for (size_t l = 0; l < n_layers; ++l) {
        const CacheI8 &c = layers[l];
        a.layer[l] = {{c.k, c.v}, {c.ks, c.vs}, {drafts[l].k, drafts[l].v}, (int)c.hd};
        hd = std::max(hd, c.hd);
    }
    a.tags = layers[0].tags;
    a.id_lo = (unsigned)layers[0].id;
    a.id_hi = (unsigned)(layers[0].id >> 32);
    a.hkv = (int)layers[0].hkv;
    a.block = (int)layers[0].block;
    constexpr int kMost = kNodes * 256;  // (the widest tree and head: 64 KB, beside 2 KB of paths)
    static const hipError_t room = hipFuncSetAttribute(reinterpret_cast<const void *>(&kv_compact_i8_kernel),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, kMost);
    if (room != hipSuccess) return hip_fail(room, "kv_compact_i8 launch set-up");
    kv_compact_i8_kernel<<<dim3((unsigned)a.hkv, (unsigned)(2 * n_layers)), kThreads, n * hd, st>>>(a);
    return check_launch("kv_compact_i8");
}

eb_status launch_copy_runs(hipStream_t st, const ByteRun *runs, size_t n) {
    RunArgs a{};
    size_t most = 0;
    for (size_t r = 0; r < n; ++r) {
        a.run[r] = runs[r];
        most = std::max(most, runs[r].bytes);
    }
    if (most == 0) return EB_OK;
    copy_runs_kernel<<<dim3((unsigned)((most + kRunChunk - 1) / kRunChunk), (unsigned)n), kThreads, 0, st>>>(a);
    return check_launch("kv_fork");
}

}  // namespace eb
