// Launchers for a tree of drafted tokens (eb_tree.hip, eb_tree_attn.hip). Arguments are checked by
// the caller (eb_draft.cpp); what lies in device memory (parents, masks, depths, paths, counts) is
// bounded by the kernels themselves, so that a captured graph may replay with another tree.
#pragma once

#include "eb_internal.h"

namespace eb {

constexpr size_t kTreeMax = 256;  // nodes of a tree: one workgroup of the plan and of the walk
inline size_t tree_words(size_t n) { return (n + 31) / 32; }

// The elements a cache holds, as the tree attention tells them apart.
enum class TreeElem { F32, F16, E4M3, I8 };

// A block-scaled layer's drafted rows beside the cache (eb_kv_cache; CacheI8::tags say whose they are).
struct DraftRows {
    float *k, *v;  // [up to kTreeMax, hkv, hd]
};
// A pass's own copy of such a cache from row0 on, in blocks of 16 rows, as a write of the drafted rows at pos
// would leave it, and which of them are not finite: those take no part in their block's exponent.
struct DraftTail {
    uint8_t *k, *v, *ks, *vs;  // codes [rows from row0, hkv, hd], exponents [blocks, hkv]
    uint8_t *bad;              // [K and V, hkv, n]
    size_t row0;
};
// The first key that some node may see (a multiple of 16, as the tiles are laid).
inline size_t tree_first_key(size_t pos, size_t window) {
    return (window > 0 && pos + 1 > window ? pos + 1 - window : 0) & ~(size_t)15;
}
// Where a tail starts: a tile of the attention (their sizes divide kTailStep) begins there, and pos's block of
// 16 does not begin before it, or no earlier key is seen.
constexpr size_t kTailStep = 128, kTailBlock = 16;
inline size_t tree_tail_row(size_t pos, size_t window) {
    const size_t key0 = tree_first_key(pos, window), b0 = pos & ~(kTailBlock - 1);
    return b0 > key0 ? key0 + (b0 - key0) / kTailStep * kTailStep : key0;
}
// Rows and blocks that a tail of n nodes has room for, wherever pos lies.
inline size_t tree_tail_rows(size_t n) { return kTailStep + kTailBlock + n; }
inline size_t tree_tail_blocks(size_t n) { return tree_tail_rows(n) / kTailBlock + 1; }
eb_status launch_kv_draft_i8(hipStream_t st, const CacheI8 &c, const DraftRows &d, const DraftTail &t, size_t pos,
                             size_t n);

struct TreeAttn {
    const float *q;  // [n, h, hd]
    const void *k, *v;         // caches [max_seq, hkv, hd], the drafted rows at pos..
    const uint8_t *ks, *vs;    // I8: exponents [ceil(max_seq / block), hkv]
    size_t block;              // I8
    TreeElem elem;
    const uint32_t *masks;     // [n, tree_words(n)]
    const uint32_t *depths;    // [n]; null without a window
    float *o;                  // [n, h, hd]
    size_t h, hkv, hd, pos, n, window;
    float scale;
    const DraftTail *tail;     // I8: keys from its row0 on are read there; or null
};
size_t tree_attn_workspace_floats(size_t h, size_t hkv, size_t hd, size_t pos, size_t n, TreeElem elem, int cu_count);
eb_status launch_attn_tree(hipStream_t st, const TreeAttn &a, float *ws, size_t ws_floats, int cu_count);

eb_status launch_tree_plan(hipStream_t st, const int32_t *parents, uint32_t *masks, uint32_t *depths, size_t n);
eb_status launch_tree_accept(hipStream_t st, const uint32_t *tokens, const int32_t *parents, const uint32_t *sampled,
                             uint32_t *path, uint32_t *emitted, uint32_t *count, size_t n);

// Copies within and between caches, for up to kMoveLayers layers a launch.
constexpr size_t kMoveLayers = 64;
// A layer's two caches as rows of bytes.
struct CacheRows {
    void *k, *v;
    size_t row_bytes;  // a multiple of 4
};
// Rows pos + path[j] to pos + j for j < *count, in place; of a block-scaled layer that has a draft of pos,
// its rows path[j], written there.
eb_status launch_kv_compact(hipStream_t st, const CacheRows *layers, size_t n_layers, const uint32_t *path,
                            const uint32_t *count, size_t n, size_t pos);
eb_status launch_kv_compact_i8(hipStream_t st, const CacheI8 *layers, const DraftRows *drafts, size_t n_layers,
                               const uint32_t *path, const uint32_t *count, size_t n, size_t pos);
// Up to 2 * kMoveLayers runs of bytes from one place to another, 16-byte aligned.
struct ByteRun {
    void *dst;
    const void *src;
    size_t bytes;
};
eb_status launch_copy_runs(hipStream_t st, const ByteRun *runs, size_t n);

}  // namespace eb
