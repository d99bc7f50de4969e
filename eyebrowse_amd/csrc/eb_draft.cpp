// Entry points that verify a drafted tree: its plan, its rows at their positions, its attention, the
// walk that accepts a branch, and the cache rows moved for that. Each checks its operands, then runs
// the launcher of its kernel translation unit (eb_tree.hip, eb_tree_attn.hip, eb_rows.hip).
#include <algorithm>
#include <cstdint>
#include <mutex>

#include "eb_handles.h"
#include "eb_internal.h"
#include "eb_tree.h"

using eb::fail;
using eb::Owned;

#define EB_TRY(expr)                      \
    do {                                  \
        eb_status eb_s_ = (expr);         \
        if (eb_s_ != EB_OK) return eb_s_; \
    } while (0)

namespace {

using WsLock = std::unique_lock<std::mutex>;

hipStream_t stream_of(eb_device *dev) { return static_cast<hipStream_t>(eb_device_stream(dev)); }
template <class T>
T *data(const eb_tensor *t) {
    return static_cast<T *>(eb_tensor_data(t));
}

// Rows and elements of a row that the kernels index with 32 bits (a whole cache may pass 2^31).
constexpr size_t kMaxRows = (size_t)1 << 27, kMaxRow = (size_t)1 << 20;

eb_status aligned(std::initializer_list<const void *> ps, uintptr_t n, const char *what) {
    for (const void *p : ps)
        if (reinterpret_cast<uintptr_t>(p) & (n - 1))
            return fail(EB_UNSUPPORTED_CONFIG, "%s must be %d-byte aligned", what, (int)n);
    return EB_OK;
}

eb_status nodes_checked(const char *what, size_t n) {
    if (n > eb::kTreeMax)
        return fail(EB_UNSUPPORTED_CONFIG, "%s: a tree of %zu nodes (at most %zu)", what, n, eb::kTreeMax);
    return EB_OK;
}

eb_status holds(size_t have, size_t need, const char *name) {
    if (have < need) return fail(EB_SHAPE_MISMATCH, "%s holds %zu elements, the shape needs %zu", name, have, need);
    return EB_OK;
}

// Node arrays: how many elements each holds, in device memory, 4-byte aligned.
struct NodeArray {
    const void *p;
    size_t have, need;
    const char *name;
};
eb_status arrays_checked(std::initializer_list<NodeArray> arrays) {
    for (const NodeArray &a : arrays) EB_TRY(holds(a.have, a.need, a.name));
    for (const NodeArray &a : arrays) {
        EB_TRY(eb::check_ptr(a.p, a.name));
        EB_TRY(aligned({a.p}, 4, a.name));
    }
    return EB_OK;
}

// ---- plan and walk ----------------------------------------------------------------------------

eb_status plan_checked(hipStream_t st, const int32_t *parents, size_t pn, uint32_t *masks, size_t mn, uint32_t *depths,
                       size_t dn, size_t n) {
    EB_TRY(nodes_checked("tree_plan", n));
    if (n == 0) return eb::ok();
    EB_TRY(arrays_checked({{parents, pn, n, "parents"}, {masks, mn, n * eb::tree_words(n), "masks"},
                           {depths, dn, n, "depths"}}));
    EB_TRY(eb::launch_tree_plan(st, parents, masks, depths, n));
    return eb::ok();
}

eb_status accept_checked(hipStream_t st, const uint32_t *tokens, size_t tn, const int32_t *parents, size_t pn,
                         const uint32_t *sampled, size_t sn, uint32_t *path, size_t hn, uint32_t *emitted, size_t en,
                         uint32_t *count, size_t cn, size_t n) {
    EB_TRY(nodes_checked("tree_accept", n));
    if (n == 0) return fail(EB_SHAPE_MISMATCH, "tree_accept: a tree has a root (n is 0)");
    EB_TRY(arrays_checked({{tokens, tn, n, "tokens"}, {parents, pn, n, "parents"}, {sampled, sn, n, "sampled"},
                           {path, hn, n, "path"}, {emitted, en, n, "emitted"}, {count, cn, 1, "count"}}));
    EB_TRY(eb::launch_tree_accept(st, tokens, parents, sampled, path, emitted, count, n));
    return eb::ok();
}

// ---- attention --------------------------------------------------------------------------------

eb::TreeElem elem_of(eb_dtype dt) {
    return dt == EB_F16 ? eb::TreeElem::F16 : dt == EB_F8E4M3 ? eb::TreeElem::E4M3 : eb::TreeElem::F32;
}

eb_status shape_checked(size_t h, size_t hkv, size_t hd, size_t max_seq, eb_dtype dt) {
    EB_TRY(eb::check_heads(h, hkv));
    if (!eb::attn_head_dim_supported(hd) || (dt != EB_F32 && hd < 8))
        return fail(EB_UNSUPPORTED_CONFIG,
                    "attn_tree: head_dim %zu (supported: 4 over f32 caches, multiples of 8 up to 128, multiples of 16 up "
                    "to 256)", hd);
    if (max_seq > kMaxRows || hkv > kMaxRow / hd || h > 65536 / eb::kTreeMax * hkv)
        return fail(EB_UNSUPPORTED_CONFIG, "attn_tree: %zu heads over caches [%zu, %zu, %zu] pass the index limits (2^27 "
                    "rows of 2^20 elements, 256 heads per KV head)", h, max_seq, hkv, hd);
    return EB_OK;
}

// What the caches do not decide: the nodes, their rows of the cache, q, o, masks and depths.
struct TreeOperands {
    const float *q;
    size_t qn;
    const uint32_t *masks;
    size_t mn;
    const uint32_t *depths;
    size_t dn;
    float *o;
    size_t on;
};
eb_status operands_checked(const TreeOperands &t, size_t h, size_t hd, size_t pos, size_t n, size_t max_seq,
                           size_t window) {
    EB_TRY(nodes_checked("attn_tree", n));
    if (pos > max_seq || n > max_seq - pos)
        return fail(EB_SHAPE_MISMATCH, "attn_tree: rows [%zu, %zu) exceed max_seq %zu", pos, pos + n, max_seq);
    EB_TRY(eb::check_numel(t.qn, {n, h, hd}, "q"));
    EB_TRY(eb::check_numel(t.on, {n, h, hd}, "o"));
    if (n * h * hd > ((size_t)1 << 29) - 1)
        return fail(EB_UNSUPPORTED_CONFIG, "attn_tree: q of %zu elements (below 2^29)", n * h * hd);
    if (n == 0) return EB_OK;
    EB_TRY(eb::check_ptr(t.q, "q"));
    EB_TRY(eb::check_ptr(t.o, "o"));
    EB_TRY(aligned({t.q, t.o}, 16, "attn_tree: q and o"));
    EB_TRY(arrays_checked({{t.masks, t.mn, n * eb::tree_words(n), "masks"}}));
    if (window > 0) EB_TRY(arrays_checked({{t.depths, t.dn, n, "depths (a window needs them)"}}));
    return EB_OK;
}

// Where the workspace comes from: the device's (dev), or the caller's.
struct Room {
    eb_device *dev = nullptr;
    float *ptr = nullptr;
    size_t floats = 0;
};

eb_status attend(hipStream_t st, const Room &room, const eb::TreeAttn &a, int cus) {
    const size_t need = eb::tree_attn_workspace_floats(a.h, a.hkv, a.hd, a.pos, a.n, a.elem, cus);
    float *ws = nullptr;
    WsLock lk;
    if (need > 0) {
        if (room.dev) {
            EB_TRY(eb::device_workspace(room.dev, need, &ws, lk));
        } else {
            if (room.floats < need)
                return fail(EB_SHAPE_MISMATCH, "attn_tree: workspace holds %zu floats, needs %zu", room.floats, need);
            EB_TRY(eb::check_ptr(room.ptr, "workspace"));
            EB_TRY(aligned({room.ptr}, 16, "the workspace"));
            ws = room.ptr;
        }
    }
    EB_TRY(eb::launch_attn_tree(st, a, ws, need, cus));
    return eb::ok();
}

eb_status tree_checked(hipStream_t st, const Room &room, int cus, const TreeOperands &t, const void *kc, size_t kcn,
                       const void *vc, size_t vcn, eb_dtype dt, size_t h, size_t hkv, size_t pos, size_t n, size_t hd,
                       size_t max_seq, float scale, size_t window) {
    EB_TRY(shape_checked(h, hkv, hd, max_seq, dt));
    EB_TRY(holds(kcn, max_seq * hkv * hd, "kcache"));
    EB_TRY(holds(vcn, max_seq * hkv * hd, "vcache"));
    EB_TRY(operands_checked(t, h, hd, pos, n, max_seq, window));
    if (n == 0) return eb::ok();
    EB_TRY(eb::check_ptr(kc, "kcache"));
    EB_TRY(eb::check_ptr(vc, "vcache"));
    EB_TRY(aligned({kc, vc}, 16, "attn_tree: the caches"));
    eb::TreeAttn a{t.q, kc, vc, nullptr, nullptr, 0, elem_of(dt), t.masks, window > 0 ? t.depths : nullptr, t.o,
                   h, hkv, hd, pos, n, window, scale, nullptr};
    return attend(st, room, a, cus);
}

// A block-scaled cache's layer, checked for its shape by the caller. tail: see TreeAttn.
eb_status tree_i8_checked(hipStream_t st, const Room &room, int cus, const TreeOperands &t, const eb::CacheI8 &c,
                          size_t h, size_t pos, size_t n, float scale, size_t window,
                          const eb::DraftTail *tail = nullptr) {
    EB_TRY(shape_checked(h, c.hkv, c.hd, c.max_seq, EB_I8));
    EB_TRY(operands_checked(t, h, c.hd, pos, n, c.max_seq, window));
    if (n == 0) return eb::ok();
    EB_TRY(eb::check_ptr(c.k, "k codes"));
    EB_TRY(eb::check_ptr(c.ks, "k exponents"));
    EB_TRY(eb::check_ptr(c.v, "v codes"));
    EB_TRY(eb::check_ptr(c.vs, "v exponents"));
    EB_TRY(aligned({c.k, c.v}, 16, "attn_tree: the codes"));
    eb::TreeAttn a{t.q, c.k, c.v, c.ks, c.vs, c.block, eb::TreeElem::I8, t.masks, window > 0 ? t.depths : nullptr, t.o,
                   h, c.hkv, c.hd, pos, n, window, scale, tail};
    return attend(st, room, a, cus);
}

eb_status operands_of(const eb_tensor *q, const eb_tensor *masks, const eb_tensor *depths, eb_tensor *o, eb_device *dev,
                      TreeOperands *t) {
    EB_TRY(eb::check_tensor(q, EB_F32, "q", dev));
    EB_TRY(eb::check_tensor(masks, EB_U32, "masks", dev));
    if (depths) EB_TRY(eb::check_tensor(depths, EB_U32, "depths", dev));
    EB_TRY(eb::check_tensor(o, EB_F32, "o", dev));
    *t = TreeOperands{data<float>(q), eb_tensor_numel(q), data<uint32_t>(masks), eb_tensor_numel(masks),
                      depths ? data<uint32_t>(depths) : nullptr, depths ? eb_tensor_numel(depths) : 0, data<float>(o),
                      eb_tensor_numel(o)};
    return EB_OK;
}

// ---- cache handles ----------------------------------------------------------------------------

eb_status layer_i8(const eb_kv_cache *kv, size_t layer, eb_device *dev, eb::CacheI8 *out) {
    EB_TRY(eb::check_tensor(kv->k[layer], EB_I8, "kv cache", dev));
    *out = eb::CacheI8{data<uint8_t>(kv->k[layer]), data<uint8_t>(kv->k_scale[layer]), data<uint8_t>(kv->v[layer]),
                       data<uint8_t>(kv->v_scale[layer]), kv->max_seq, kv->n_kv_heads,
                       eb_tensor_dim(kv->k[layer], 2), kv->block, eb::draft_tags(kv, layer), kv->id};
    return EB_OK;
}

// The layer's rows beside the cache. Room for the widest tree is taken once (whether it holds a draft is a tag on
// the device), so that a captured pass and a captured compaction agree about it, whichever was captured first.
eb_status draft_rows(eb_kv_cache *kv, size_t layer, eb_device *dev, eb::DraftRows *out) {
    if (!kv->draft_v[layer]) {
        const size_t shape[3] = {std::min(eb::kTreeMax, kv->max_seq), kv->n_kv_heads, eb_tensor_dim(kv->k[layer], 2)};
        eb_tensor *k = nullptr, *v = nullptr;
        EB_TRY(eb_tensor_empty(dev, shape, 3, EB_F32, &k));
        Owned guard(k);
        EB_TRY(eb_tensor_empty(dev, shape, 3, EB_F32, &v));
        kv->draft_k[layer] = guard.release();
        kv->draft_v[layer] = v;
    }
    *out = eb::DraftRows{data<float>(kv->draft_k[layer]), data<float>(kv->draft_v[layer])};
    return EB_OK;
}

// Memory for a pass's tail (eb::DraftTail), of a size that does not depend on pos.
eb_status tail_room(eb_device *dev, const eb::CacheI8 &c, size_t pos, size_t n, size_t window, Owned *hold,
                    eb::DraftTail *out) {
    const size_t codes = eb::tree_tail_rows(n) * c.hkv * c.hd;  // (a multiple of 16)
    const size_t exps = eb::tree_tail_blocks(n) * c.hkv, shape[1] = {2 * codes + 2 * exps + 2 * c.hkv * n};
    EB_TRY(eb_tensor_empty(dev, shape, 1, EB_U8, &hold->t));
    uint8_t *p = data<uint8_t>(hold->t);
    *out = eb::DraftTail{p, p + codes, p + 2 * codes, p + 2 * codes + exps, p + 2 * codes + 2 * exps,
                         eb::tree_tail_row(pos, window)};
    return EB_OK;
}

// The row pass's norms and tables, which reach `positions`.
eb_status rows_checked(const eb_attention_desc &d, const eb_rope_tables *rope, size_t positions, eb_device *dev) {
    for (const eb_tensor *n : {d.q_norm, d.k_norm, d.v_norm})
        if (n) EB_TRY(eb::check_tensor(n, EB_F32, "norm gain", dev));
    EB_TRY(eb::check_tensor(rope->cos, EB_F32, "rope cos", dev));
    EB_TRY(eb::check_tensor(rope->sin, EB_F32, "rope sin", dev));
    return eb::check_numel(std::min(eb_tensor_numel(rope->cos), eb_tensor_numel(rope->sin)),
                           {positions, d.head_dim / 2}, "rope tables");
}
const float *gain(const eb_tensor *t) { return t ? data<float>(t) : nullptr; }

size_t row_bytes(const eb_kv_cache *kv, size_t layer) {
    const eb_tensor *t = kv->k[layer];
    return kv->n_kv_heads * eb_tensor_dim(t, 2) * eb_dtype_size(eb_tensor_dtype(t));
}

// A cache on dev, whatever its elements.
eb_status cache_on(const eb_kv_cache *kv, const char *what, eb_device *dev) {
    if (!kv) return fail(EB_SHAPE_MISMATCH, "%s: kv cache is null", what);
    for (const eb_tensor *t : kv->k)
        if (eb::tensor_device(t) != dev) return fail(EB_OTHER, "%s: the kv cache lives on another device", what);
    return EB_OK;
}

}  // namespace

extern "C" {

eb_status eb_tree_plan(eb_recorder *rec, const eb_tensor *parents, eb_tensor *masks, eb_tensor *depths, size_t n) {
    eb_device *dev;
    EB_TRY(eb::recorder_ready(rec, &dev));
    EB_TRY(eb::check_tensor(parents, EB_I32, "parents", dev));
    EB_TRY(eb::check_tensor(masks, EB_U32, "masks", dev));
    EB_TRY(eb::check_tensor(depths, EB_U32, "depths", dev));
    return plan_checked(stream_of(dev), data<int32_t>(parents), eb_tensor_numel(parents), data<uint32_t>(masks),
                        eb_tensor_numel(masks), data<uint32_t>(depths), eb_tensor_numel(depths), n);
}

eb_status eb_launch_tree_plan(void *stream, const int32_t *parents, size_t parents_numel, uint32_t *masks,
                              size_t masks_numel, uint32_t *depths, size_t depths_numel, size_t n) {
    return plan_checked((hipStream_t)stream, parents, parents_numel, masks, masks_numel, depths, depths_numel, n);
}

eb_status eb_tree_accept(eb_recorder *rec, const eb_tensor *tokens, const eb_tensor *parents, const eb_tensor *sampled,
                         eb_tensor *path, eb_tensor *emitted, eb_tensor *count, size_t n) {
    eb_device *dev;
    EB_TRY(eb::recorder_ready(rec, &dev));
    EB_TRY(eb::check_tensor(tokens, EB_U32, "tokens", dev));
    EB_TRY(eb::check_tensor(parents, EB_I32, "parents", dev));
    EB_TRY(eb::check_tensor(sampled, EB_U32, "sampled", dev));
    EB_TRY(eb::check_tensor(path, EB_U32, "path", dev));
    EB_TRY(eb::check_tensor(emitted, EB_U32, "emitted", dev));
    EB_TRY(eb::check_tensor(count, EB_U32, "count", dev));
    return accept_checked(stream_of(dev), data<uint32_t>(tokens), eb_tensor_numel(tokens), data<int32_t>(parents),
                          eb_tensor_numel(parents), data<uint32_t>(sampled), eb_tensor_numel(sampled),
                          data<uint32_t>(path), eb_tensor_numel(path), data<uint32_t>(emitted), eb_tensor_numel(emitted),
                          data<uint32_t>(count), eb_tensor_numel(count), n);
}

eb_status eb_launch_tree_accept(void *stream, const uint32_t *tokens, size_t tokens_numel, const int32_t *parents,
                                size_t parents_numel, const uint32_t *sampled, size_t sampled_numel, uint32_t *path,
                                size_t path_numel, uint32_t *emitted, size_t emitted_numel, uint32_t *count, size_t n) {
    return accept_checked((hipStream_t)stream, tokens, tokens_numel, parents, parents_numel, sampled, sampled_numel,
                          path, path_numel, emitted, emitted_numel, count, 1, n);
}

eb_status eb_attn_tree(eb_recorder *rec, const eb_tensor *q, const eb_tensor *kcache, const eb_tensor *vcache,
                       const eb_tensor *masks, const eb_tensor *depths, eb_tensor *o, size_t h, size_t hkv, size_t pos,
                       size_t n, size_t hd, size_t max_seq, float scale, size_t window) {
    eb_device *dev;
    EB_TRY(eb::recorder_ready(rec, &dev));
    if (!kcache) return fail(EB_SHAPE_MISMATCH, "kcache is null");
    const eb_dtype dt = eb_tensor_dtype(kcache);
    if (dt != EB_F32 && dt != EB_F16 && dt != EB_F8E4M3)
        return fail(EB_SHAPE_MISMATCH, "kcache must be f32, f16 or f8e4m3");
    EB_TRY(eb::check_tensor(kcache, dt, "kcache", dev));
    EB_TRY(eb::check_tensor(vcache, dt, "vcache", dev));
    TreeOperands t;
    EB_TRY(operands_of(q, masks, depths, o, dev, &t));
    return tree_checked(stream_of(dev), Room{dev}, eb_device_cu_count(dev), t, data<void>(kcache),
                        eb_tensor_numel(kcache), data<void>(vcache), eb_tensor_numel(vcache), dt, h, hkv, pos, n, hd,
                        max_seq, scale, window);
}

eb_status eb_attn_tree_i8(eb_recorder *rec, const eb_tensor *q, const eb_kv_cache *kv, size_t layer,
                          const eb_tensor *masks, const eb_tensor *depths, eb_tensor *o, size_t h, size_t pos, size_t n,
                          float scale, size_t window) {
    eb_device *dev;
    EB_TRY(eb::recorder_ready(rec, &dev));
    if (!kv) return fail(EB_SHAPE_MISMATCH, "kv cache is null");
    if (!kv->block) return fail(EB_SHAPE_MISMATCH, "the kv cache is not block-scaled (eb_kv_cache_new_i8)");
    if (layer >= kv->k.size()) return fail(EB_SHAPE_MISMATCH, "layer %zu of %zu", layer, kv->k.size());
    eb::CacheI8 c;
    EB_TRY(layer_i8(kv, layer, dev, &c));
    TreeOperands t;
    EB_TRY(operands_of(q, masks, depths, o, dev, &t));
    return tree_i8_checked(stream_of(dev), Room{dev}, eb_device_cu_count(dev), t, c, h, pos, n, scale, window);
}

size_t eb_attn_tree_workspace_floats(size_t h, size_t hkv, size_t pos, size_t n, size_t hd, eb_dtype dtype,
                                     int cu_count) {
    if (n == 0 || n > eb::kTreeMax || pos > kMaxRows || shape_checked(h, hkv, hd, 0, dtype) != EB_OK) return 0;
    return eb::tree_attn_workspace_floats(h, hkv, hd, pos, n, dtype == EB_I8 ? eb::TreeElem::I8 : elem_of(dtype),
                                          cu_count > 0 ? cu_count : 256);
}

eb_status eb_launch_attn_tree(void *stream, const float *q, size_t q_numel, const void *kc, size_t kc_numel,
                              const void *vc, size_t vc_numel, eb_dtype dtype, const uint32_t *masks,
                              size_t masks_numel, const uint32_t *depths, size_t depths_numel, float *o, size_t o_numel,
                              size_t h, size_t hkv, size_t pos, size_t n, size_t hd, size_t max_seq, float scale,
                              size_t window, float *workspace, size_t workspace_floats, int cu_count) {
    if (dtype != EB_F32 && dtype != EB_F16 && dtype != EB_F8E4M3)
        return fail(EB_UNSUPPORTED_CONFIG, "attn_tree: caches must be f32, f16 or f8e4m3");
    const TreeOperands t{q, q_numel, masks, masks_numel, depths, depths_numel, o, o_numel};
    return tree_checked((hipStream_t)stream, Room{nullptr, workspace, workspace_floats}, cu_count > 0 ? cu_count : 256,
                        t, kc, kc_numel, vc, vc_numel, dtype, h, hkv, pos, n, hd, max_seq, scale, window);
}

eb_status eb_launch_attn_tree_i8(void *stream, const float *q, size_t q_numel, const eb_cache_i8 *cache,
                                 const uint32_t *masks, size_t masks_numel, const uint32_t *depths, size_t depths_numel,
                                 float *o, size_t o_numel, size_t h, size_t pos, size_t n, float scale, size_t window,
                                 float *workspace, size_t workspace_floats, int cu_count) {
    eb::CacheI8 c;
    EB_TRY(eb::cache_i8_of(cache, &c));
    const TreeOperands t{q, q_numel, masks, masks_numel, depths, depths_numel, o, o_numel};
    return tree_i8_checked((hipStream_t)stream, Room{nullptr, workspace, workspace_floats},
                           cu_count > 0 ? cu_count : 256, t, c, h, pos, n, scale, window);
}

eb_status eb_attn_prologue_tree(eb_recorder *rec, const eb_tensor *q, const eb_tensor *k, const eb_tensor *v,
                                const eb_tensor *depths, eb_tensor *q_out, eb_tensor *kcache, eb_tensor *vcache,
                                size_t rows, size_t h, size_t hkv, size_t hd, size_t base_pos, size_t max_seq,
                                const eb_tensor *q_norm, const eb_tensor *k_norm, const eb_tensor *v_norm, float eps,
                                const eb_tensor *rope_cos, const eb_tensor *rope_sin) {
    if (!depths) return fail(EB_SHAPE_MISMATCH, "depths is null");
    return eb::attn_rows_fused(rec, q, k, v, q_out, kcache, vcache, rows, h, hkv, hd, base_pos, max_seq, q_norm, k_norm,
                               v_norm, eps, rope_cos, rope_sin, depths);
}

// ---- moved rows ---------------------------------------------------------------------------------

eb_status eb_kv_compact(eb_recorder *rec, eb_kv_cache *kv, const eb_tensor *path, const eb_tensor *count, size_t n,
                        size_t pos) {
    eb_device *dev;
    EB_TRY(eb::recorder_ready(rec, &dev));
    EB_TRY(cache_on(kv, "kv_compact", dev));
    EB_TRY(eb::check_tensor(path, EB_U32, "path", dev));
    EB_TRY(eb::check_tensor(count, EB_U32, "count", dev));
    EB_TRY(nodes_checked("kv_compact", n));
    if (pos > kv->max_seq || n > kv->max_seq - pos)
        return fail(EB_SHAPE_MISMATCH, "kv_compact: rows [%zu, %zu) exceed max_seq %zu", pos, pos + n, kv->max_seq);
    const size_t layers = kv->k.size();
    if (n == 0 || layers == 0) return eb::ok();
    EB_TRY(arrays_checked({{data<uint32_t>(path), eb_tensor_numel(path), n, "path"},
                           {data<uint32_t>(count), eb_tensor_numel(count), 1, "count"}}));
    // Everything is checked before the first launch; then a launch for each group of layers.
    for (size_t l = 0; l < layers; ++l)
        if (!kv->block && row_bytes(kv, l) % 4)
            return fail(EB_UNSUPPORTED_CONFIG, "kv_compact: rows of %zu bytes (a multiple of 4)", row_bytes(kv, l));
    eb::CacheI8 caches[eb::kMoveLayers];
    eb::DraftRows drafts[eb::kMoveLayers];
    for (size_t l = 0; l < layers && kv->block; ++l) EB_TRY(draft_rows(kv, l, dev, &drafts[0]));  // (memory)
    const hipStream_t st = stream_of(dev);
    for (size_t l0 = 0; l0 < layers; l0 += eb::kMoveLayers) {
        const size_t nl = std::min(layers - l0, eb::kMoveLayers);
        if (kv->block) {
            for (size_t l = 0; l < nl; ++l) {
                EB_TRY(layer_i8(kv, l0 + l, dev, &caches[l]));
                EB_TRY(draft_rows(kv, l0 + l, dev, &drafts[l]));
            }
            EB_TRY(eb::launch_kv_compact_i8(st, caches, drafts, nl, data<uint32_t>(path), data<uint32_t>(count), n, pos));
        } else {
            eb::CacheRows c[eb::kMoveLayers];
            for (size_t l = 0; l < nl; ++l)
                c[l] = eb::CacheRows{data<void>(kv->k[l0 + l]), data<void>(kv->v[l0 + l]), row_bytes(kv, l0 + l)};
            EB_TRY(eb::launch_kv_compact(st, c, nl, data<uint32_t>(path), data<uint32_t>(count), n, pos));
        }
    }
    return eb::ok();
}

eb_status eb_kv_fork(eb_recorder *rec, eb_kv_cache *dst, const eb_kv_cache *src, size_t count) {
    eb_device *dev;
    EB_TRY(eb::recorder_ready(rec, &dev));
    EB_TRY(cache_on(dst, "kv_fork", dev));
    EB_TRY(cache_on(src, "kv_fork", dev));
    if (dst == src) return fail(EB_SHAPE_MISMATCH, "kv_fork: a cache cannot be copied into itself");
    const size_t layers = src->k.size();
    if (dst->k.size() != layers || dst->n_kv_heads != src->n_kv_heads || dst->block != src->block)
        return fail(EB_SHAPE_MISMATCH, "kv_fork: the caches' layers, KV heads or blocks differ");
    if (count > src->max_seq || count > dst->max_seq)
        return fail(EB_SHAPE_MISMATCH, "kv_fork: %zu rows of caches of %zu and %zu", count, src->max_seq, dst->max_seq);
    for (size_t l = 0; l < layers; ++l)
        if (eb_tensor_dtype(src->k[l]) != eb_tensor_dtype(dst->k[l]) || row_bytes(src, l) != row_bytes(dst, l))
            return fail(EB_SHAPE_MISMATCH, "kv_fork: layer %zu has other elements or another head_dim", l);
    if (count == 0) return eb::ok();
    // A launch's runs are of like length: a group of layers' rows, then their exponents.
    const hipStream_t st = stream_of(dev);
    if (std::any_of(dst->draft_v.begin(), dst->draft_v.end(), [](const eb_tensor *t) { return t != nullptr; }))
        EB_TRY(eb::drop_drafts(dst, st));
    eb::ByteRun runs[2 * eb::kMoveLayers];
    for (size_t l0 = 0; l0 < layers; l0 += eb::kMoveLayers) {
        const size_t nl = std::min(layers - l0, eb::kMoveLayers);
        for (size_t l = 0; l < nl; ++l) {
            const size_t bytes = count * row_bytes(src, l0 + l);
            runs[2 * l] = eb::ByteRun{data<void>(dst->k[l0 + l]), data<void>(src->k[l0 + l]), bytes};
            runs[2 * l + 1] = eb::ByteRun{data<void>(dst->v[l0 + l]), data<void>(src->v[l0 + l]), bytes};
        }
        EB_TRY(eb::launch_copy_runs(st, runs, 2 * nl));
        if (!src->block) continue;
        const size_t bytes = (count + src->block - 1) / src->block * src->n_kv_heads;
        for (size_t l = 0; l < nl; ++l) {
            runs[2 * l] = eb::ByteRun{data<void>(dst->k_scale[l0 + l]), data<void>(src->k_scale[l0 + l]), bytes};
            runs[2 * l + 1] = eb::ByteRun{data<void>(dst->v_scale[l0 + l]), data<void>(src->v_scale[l0 + l]), bytes};
        }
        EB_TRY(eb::launch_copy_runs(st, runs, 2 * nl));
    }
    return eb::ok();
}

// ---- Attention ------------------------------------------------------------------------------------

eb_status eb_attention_forward_tree_qkv(const eb_attention *attn, eb_recorder *rec, const eb_tensor *q,
                                        const eb_tensor *k, const eb_tensor *v, const eb_rope_tables *rope,
                                        eb_kv_cache *kv, size_t layer, const eb_tensor *masks, const eb_tensor *depths,
                                        size_t rows, size_t base_pos, eb_tensor **out) {
    if (!attn || !rec || !q || !k || !v || !rope || !kv || !out || !masks || !depths)
        return fail(EB_OTHER, "attention_forward_tree: null argument");
    *out = nullptr;
    eb_device *dev;
    EB_TRY(eb::recorder_ready(rec, &dev));
    const eb_attention_desc &d = attn->d;
    const size_t H = d.n_heads, Hkv = d.n_kv_heads, hd = d.head_dim;
    EB_TRY(nodes_checked("attention_forward_tree", rows));
    if (rows == 0) return fail(EB_SHAPE_MISMATCH, "attention_forward_tree: rows must be > 0");
    if (layer >= kv->k.size())
        return fail(EB_SHAPE_MISMATCH, "attention_forward_tree: layer %zu of %zu", layer, kv->k.size());
    if (rope->head_dim != hd)
        return fail(EB_SHAPE_MISMATCH, "attention_forward_tree: rope head_dim %zu != %zu", rope->head_dim, hd);
    if (kv->n_kv_heads != Hkv || eb_tensor_dim(kv->k[layer], 2) != hd)
        return fail(EB_SHAPE_MISMATCH, "attention_forward_tree: the cache layer is not [max_seq, %zu, %zu]", Hkv, hd);
    if (base_pos > kv->max_seq || rows > kv->max_seq - base_pos)
        return fail(EB_SHAPE_MISMATCH, "attention_forward_tree: rows [%zu, %zu) exceed max_seq %zu", base_pos,
                    base_pos + rows, kv->max_seq);
    EB_TRY(eb::check_tensor(q, EB_F32, "q", dev));
    EB_TRY(eb::check_tensor(k, EB_F32, "k", dev));
    EB_TRY(eb::check_tensor(v, EB_F32, "v", dev));
    EB_TRY(eb::check_tensor(masks, EB_U32, "masks", dev));
    EB_TRY(eb::check_tensor(depths, EB_U32, "depths", dev));
    if (eb_tensor_numel(q) != rows * H * hd || eb_tensor_numel(k) != rows * Hkv * hd ||
        eb_tensor_numel(v) != rows * Hkv * hd)
        return fail(EB_SHAPE_MISMATCH, "attention_forward_tree: q/k/v are not [rows, heads*head_dim]");
    // Before anything is written: the attention's own refusals.
    EB_TRY(shape_checked(H, Hkv, hd, kv->max_seq, eb_tensor_dtype(kv->k[layer])));
    EB_TRY(holds(eb_tensor_numel(masks), rows * eb::tree_words(rows), "masks"));
    EB_TRY(holds(eb_tensor_numel(depths), rows, "depths"));

    const size_t qshape[3] = {rows, H, hd}, oshape[2] = {rows, H * hd};
    eb_tensor *t = nullptr;
    EB_TRY(eb_tensor_empty(dev, qshape, 3, EB_F32, &t));
    Owned qr(t);
    EB_TRY(eb_tensor_empty(dev, oshape, 2, EB_F32, &t));
    Owned o(t);
    if (kv->block) {
        // The row pass into f32 rows beside the cache, then the attention over the cache's rows and, from a
        // copy of its end on, those rows' codes: written into the cache they would round the rows of pos's
        // block for good, whatever becomes of the draft. (The copy has blocks of 16, the fewest that the
        // attention tells apart, so that few rows are rounded to another's exponent even there.)
        eb::CacheI8 c;
        EB_TRY(layer_i8(kv, layer, dev, &c));
        EB_TRY(rows_checked(d, rope, base_pos + rows, dev));
        TreeOperands operands;
        EB_TRY(operands_of(qr.t, masks, depths, o.t, dev, &operands));
        eb::DraftRows beside;
        EB_TRY(draft_rows(kv, layer, dev, &beside));
        Owned hold;
        eb::DraftTail tail;
        EB_TRY(tail_room(dev, c, base_pos, rows, d.window, &hold, &tail));
        eb::RowsArgs a{};
        a.nseg = 3;
        a.seg[0] = eb::RowSeg{data<float>(q), data<float>(qr.t), gain(d.q_norm), (int)H, 0, true, 4};
        a.seg[1] = eb::RowSeg{data<float>(k), beside.k, gain(d.k_norm), (int)Hkv, 0, true, 4};
        a.seg[2] = eb::RowSeg{data<float>(v), beside.v, gain(d.v_norm), (int)Hkv, 0, false, 4};
        a.rows = (int)rows;
        a.hd = (int)hd;
        a.eps = d.norm_eps;
        a.cosb = data<float>(rope->cos);
        a.sinb = data<float>(rope->sin);
        a.rope_row0 = (int)base_pos;
        a.depths = data<uint32_t>(depths);
        EB_TRY(eb::launch_attn_rows(stream_of(dev), a));
        EB_TRY(eb::launch_kv_draft_i8(stream_of(dev), c, beside, tail, base_pos, rows));
        EB_TRY(tree_i8_checked(stream_of(dev), Room{dev}, eb_device_cu_count(dev), operands, c, H, base_pos, rows,
                               d.scale, d.window, &tail));
    } else {
        eb_tensor *kc = kv->k[layer], *vc = kv->v[layer];
        EB_TRY(eb::attn_rows_fused(rec, q, k, v, qr.t, kc, vc, rows, H, Hkv, hd, base_pos, kv->max_seq, d.q_norm,
                                   d.k_norm, d.v_norm, d.norm_eps, rope->cos, rope->sin, depths));
        EB_TRY(eb_attn_tree(rec, qr.t, kc, vc, masks, depths, o.t, H, Hkv, base_pos, rows, hd, kv->max_seq, d.scale,
                            d.window));
    }
    *out = o.release();
    return eb::ok();
}

}  // extern "C"
