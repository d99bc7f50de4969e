// Entry points of the quantised operators: 4-bit projections, block-scaled 8-bit KV caches, and
// the sampling that ends a token. Each checks its operands, then runs the launcher of its kernel
// translation unit (eb_linear_q4.hip, eb_cache_i8.hip, eb_decode_i8.hip, eb_prefill.hip,
// eb_sample.hip).
#include <algorithm>
#include <atomic>
#include <chrono>
#include <climits>
#include <cstdint>
#include <memory>
#include <mutex>

#include "eb_handles.h"
#include "eb_internal.h"

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

eb_status aligned(std::initializer_list<const void *> ps, uintptr_t n, const char *what) {
    for (const void *p : ps)
        if (reinterpret_cast<uintptr_t>(p) & (n - 1))
            return fail(EB_UNSUPPORTED_CONFIG, "%s must be %d-byte aligned", what, (int)n);
    return EB_OK;
}

// A set-up call's work belongs to no graph.
eb_status not_captured(hipStream_t st, const char *what) {
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    EB_HIP_TRY(hipStreamIsCapturing(st, &capture));
    if (capture != hipStreamCaptureStatusNone)
        return fail(EB_OTHER, "%s: not allowed while the device's stream is being captured", what);
    return EB_OK;
}

// ---- block-scaled caches --------------------------------------------------------------------

// A cache's number (eb::CacheI8): of 64 bits that no other one has and no memory holds by chance, the lower half
// not 0.
uint64_t cache_number(const void *at) {
    static std::atomic<uint64_t> count{0};
    uint64_t x = ++count * 0x9E3779B97F4A7C15u + (uint64_t)std::chrono::steady_clock::now().time_since_epoch().count() +
                 (uint64_t)reinterpret_cast<uintptr_t>(at);
    x = (x ^ (x >> 30)) * 0xBF58476D1CE4E5B9u;
    x = (x ^ (x >> 27)) * 0x94D049BB133111EBu;
    return (x ^ (x >> 31)) | 1;
}

// Rows and elements of a row that the kernels index with 32 bits (a whole cache may pass 2^31).
constexpr size_t kMaxRows = (size_t)1 << 27, kMaxRow = (size_t)1 << 20;

eb_status shape_i8(size_t max_seq, size_t hkv, size_t hd, size_t block) {
    if (hkv == 0) return fail(EB_SHAPE_MISMATCH, "head counts must be positive");
    if (hd % 16 != 0 || hd < 32 || hd > 256)
        return fail(EB_UNSUPPORTED_CONFIG, "block-scaled cache: head_dim %zu (multiples of 16 from 32 to 256)", hd);
    if (block < 16 || block > 256 || (block & (block - 1)))
        return fail(EB_UNSUPPORTED_CONFIG, "block-scaled cache: block %zu (a power of two from 16 to 256)", block);
    if (max_seq > kMaxRows || hkv > kMaxRow / hd)
        return fail(EB_UNSUPPORTED_CONFIG, "block-scaled cache: [%zu, %zu, %zu] passes the index limits (2^27 rows "
                    "of 2^20 elements)", max_seq, hkv, hd);
    return EB_OK;
}

eb_status cache_ready(const eb::CacheI8 &c) {
    EB_TRY(eb::check_ptr(c.k, "k codes"));
    EB_TRY(eb::check_ptr(c.ks, "k exponents"));
    EB_TRY(eb::check_ptr(c.v, "v codes"));
    EB_TRY(eb::check_ptr(c.vs, "v exponents"));
    return aligned({c.k, c.v}, 16, "block-scaled cache: the codes");
}

// The layer of a handle, on dev.
eb_status layer_of(const eb_kv_cache *kv, size_t layer, eb_device *dev, eb::CacheI8 *out) {
    if (!kv) return fail(EB_SHAPE_MISMATCH, "kv cache is null");
    if (!kv->block) return fail(EB_SHAPE_MISMATCH, "the kv cache is not block-scaled (eb_kv_cache_new_i8)");
    if (layer >= kv->k.size()) return fail(EB_SHAPE_MISMATCH, "layer %zu of %zu", layer, kv->k.size());
    EB_TRY(eb::check_tensor(kv->k[layer], EB_I8, "kv cache", dev));
    *out = eb::CacheI8{data<uint8_t>(kv->k[layer]), data<uint8_t>(kv->k_scale[layer]), data<uint8_t>(kv->v[layer]),
                       data<uint8_t>(kv->v_scale[layer]), kv->max_seq, kv->n_kv_heads,
                       eb_tensor_dim(kv->k[layer], 2), kv->block, eb::draft_tags(kv, layer), kv->id};
    return EB_OK;
}

eb_status rows_in(const char *what, size_t start, size_t count, size_t max_seq) {
    if (start > max_seq || count > max_seq - start)
        return fail(EB_SHAPE_MISMATCH, "%s: rows [%zu, %zu) exceed max_seq %zu", what, start, start + count, max_seq);
    return EB_OK;
}

// A count of f32 elements that is indexed with 64 bits.
eb_status holds(size_t have, size_t need, const char *name) {
    if (have < need) return fail(EB_SHAPE_MISMATCH, "%s holds %zu elements, the shape needs %zu", name, have, need);
    return EB_OK;
}

eb_status move_i8(hipStream_t st, const char *what, const eb::CacheI8 &c, const float *k, const float *v, size_t numel,
                  size_t count, size_t start, float *k_out, float *v_out) {
    EB_TRY(rows_in(what, start, count, c.max_seq));
    EB_TRY(holds(numel, count * c.hkv * c.hd, "k/v"));
    if (count == 0) return eb::ok();
    EB_TRY(cache_ready(c));
    EB_TRY(eb::check_ptr(k, "k"));
    EB_TRY(eb::check_ptr(v, "v"));
    EB_TRY(aligned({k, v}, 16, "k and v"));
    if (k_out)
        EB_TRY(eb::launch_kv_read_i8(st, c, k_out, v_out, start, count));
    else
        EB_TRY(eb::launch_kv_write_i8(st, c, k, v, start, count));
    return eb::ok();
}

// Rows whose columns (rows x heads of a KV head) number at most this many run the few-row kernel,
// which reads the cache once for every 16 of them; more rows run the prefill kernels over records.
// Both measured (us, few-row and prefill): 192 columns of 32 heads over 8 KV heads of 128 behind 1000
// keys 22.5 and 29.1, 8192 keys 47.0 and 56.3, 32000 keys 129 and 145; 256 columns 26.4 and 31.1, 57.0
// and 57.0, 157 and 150. One head per KV head, 8 of 128: 192 columns 22.6 and 30.0, 47.8 and 53.1, 128
// and 138, 256 columns 26.8 and 31.9, 57.4 and 56.3, 158 and 149. 14 over 2 heads of 64, 6 over 2 of
// 96: few-row the faster through 256 columns (32000 keys 35.9 and 65.9, 48.6 and 66.0). 16 over 8 of
// 256, 8192 keys: 128 columns 56.1 and 74.7. Where KV heads are many and short the sides meet
// earlier: 16 over 16 of 64, 128 columns 18.0 and 23.8, 40.6 and 44.6, 115 and 126, but 192 columns
// 20.3 and 23.5, 63.4 and 53.7, 197 and 159.
constexpr size_t kFewRowCols = 192;

size_t attn_workspace(size_t h, size_t hkv, size_t hd, size_t pos0, size_t rows, size_t window, size_t block, int cus) {
    if (rows * (h / hkv) <= kFewRowCols) return eb::decode_i8_workspace_floats(h, hkv, pos0, rows, hd, block, cus);
    return eb::prefill_i8_workspace_floats(h, hkv, hd, pos0, rows, window);
}

eb_status attn_checked(const eb::CacheI8 &c, const float *q, size_t qn, const float *o, size_t on, size_t h,
                       size_t pos0, size_t rows) {
    EB_TRY(eb::check_heads(h, c.hkv));
    EB_TRY(rows_in("attention over a block-scaled cache", pos0, rows, c.max_seq));
    EB_TRY(eb::check_numel(qn, {rows, h, c.hd}, "q"));
    EB_TRY(eb::check_numel(on, {rows, h, c.hd}, "o"));
    if (rows == 0) return EB_OK;
    EB_TRY(cache_ready(c));
    EB_TRY(eb::check_ptr(q, "q"));
    EB_TRY(eb::check_ptr(o, "o"));
    return aligned({q, o}, 16, "q and o");
}

eb_status step_checked(const eb::CacheI8 &c, const float *knew, const float *vnew, size_t n) {
    EB_TRY(holds(n, c.hkv * c.hd, "knew/vnew"));
    EB_TRY(eb::check_ptr(knew, "knew"));
    EB_TRY(eb::check_ptr(vnew, "vnew"));
    return aligned({knew, vnew}, 16, "knew and vnew");
}

// Where the workspace comes from: the device's (dev), or the caller's.
struct Room {
    eb_device *dev = nullptr;
    float *ptr = nullptr;
    size_t floats = 0;
};
eb_status room(const Room &r, size_t need, float **ws, WsLock &lk) {
    *ws = nullptr;
    if (need == 0) return EB_OK;
    if (r.dev) return eb::device_workspace(r.dev, need, ws, lk);
    if (r.floats < need)
        return fail(EB_SHAPE_MISMATCH, "workspace holds %zu floats, needs %zu", r.floats, need);
    EB_TRY(eb::check_ptr(r.ptr, "workspace"));
    EB_TRY(aligned({r.ptr}, 16, "the workspace"));
    *ws = r.ptr;
    return EB_OK;
}

// Checked attention of rows at pos0 (knew: one row, appended first).
eb_status attend_i8(hipStream_t st, const Room &src, int cus, const eb::CacheI8 &c, const float *q, const float *knew,
                    const float *vnew, float *o, size_t h, size_t pos0, size_t rows, float scale, size_t window,
                    const eb::DecodePrologue *pro = nullptr) {
    if (rows == 0) return eb::ok();
    const size_t need = attn_workspace(h, c.hkv, c.hd, pos0, rows, window, c.block, cus);
    float *ws;
    WsLock lk;
    EB_TRY(room(src, need, &ws, lk));
    if (rows * (h / c.hkv) <= kFewRowCols) {
        EB_TRY(eb::launch_attn_decode_i8(st, q, c, knew, vnew, o, h, pos0, rows, scale, window, ws, need, cus, pro));
    } else {
        if (knew) EB_TRY(eb::launch_kv_write_i8(st, c, knew, vnew, pos0, 1));
        EB_TRY(eb::launch_attn_prefill_i8(st, q, c, o, h, pos0, rows, scale, window, ws, need));
    }
    return eb::ok();
}

eb_status prologue_of(const eb_attention_desc &d, const eb_rope_tables *rope, size_t pos, eb_device *dev,
                      eb::DecodePrologue *p) {
    const eb_tensor *norms[3] = {d.q_norm, d.k_norm, d.v_norm};
    const float **slots[3] = {&p->q_norm, &p->k_norm, &p->v_norm};
    for (int i = 0; i < 3; ++i) {
        *slots[i] = nullptr;
        if (!norms[i]) continue;
        EB_TRY(eb::check_tensor(norms[i], EB_F32, "norm gain", dev));
        *slots[i] = data<float>(norms[i]);
    }
    EB_TRY(eb::check_tensor(rope->cos, EB_F32, "rope cos", dev));
    EB_TRY(eb::check_tensor(rope->sin, EB_F32, "rope sin", dev));
    if (pos >= rope->max_seq)
        return fail(EB_SHAPE_MISMATCH, "attention_forward: position %zu exceeds the rope tables (%zu)", pos,
                    rope->max_seq);
    p->eps = d.norm_eps;
    p->rope_cos = data<float>(rope->cos);
    p->rope_sin = data<float>(rope->sin);
    return EB_OK;
}

}  // namespace

eb_status eb::cache_i8_of(const eb_cache_i8 *c, CacheI8 *out) {
    if (!c) return fail(EB_SHAPE_MISMATCH, "cache is null");
    EB_TRY(shape_i8(c->max_seq, c->hkv, c->hd, c->block));
    const size_t codes = c->max_seq * c->hkv * c->hd;
    const size_t exps = (c->max_seq + c->block - 1) / c->block * c->hkv;
    if (c->code_numel < codes)
        return fail(EB_SHAPE_MISMATCH, "the cache's codes hold %zu elements, the shape needs %zu", c->code_numel, codes);
    if (c->exp_numel < exps)
        return fail(EB_SHAPE_MISMATCH, "the cache's exponents hold %zu bytes, the shape needs %zu", c->exp_numel, exps);
    *out = CacheI8{reinterpret_cast<uint8_t *>(c->k), c->k_exp, reinterpret_cast<uint8_t *>(c->v), c->v_exp,
                       c->max_seq, c->hkv, c->hd, c->block};
    return EB_OK;
}

uint32_t *eb::draft_tags(const eb_kv_cache *kv, size_t layer) {
    return data<uint32_t>(kv->draft_tags) + layer * 2 * kTagWords * kv->n_kv_heads;
}

eb_status eb::drop_drafts(eb_kv_cache *kv, hipStream_t st) {
    const size_t bytes = eb_tensor_numel(kv->draft_tags) * sizeof(uint32_t);
    return bytes == 0 ? EB_OK : launch_fill_u8(st, data<uint8_t>(kv->draft_tags), 0, bytes);
}

eb_status eb::attention_forward_i8(const eb_attention_desc &d, eb_recorder *rec, const eb_tensor *q,
                                   const eb_tensor *k, const eb_tensor *v, const eb_rope_tables *rope,
                                   eb_kv_cache *kv, size_t layer, size_t rows, size_t base_pos, eb_tensor **out) {
    eb_device *dev;
    EB_TRY(recorder_ready(rec, &dev));
    EB_TRY(check_tensor(q, EB_F32, "q", dev));
    EB_TRY(check_tensor(k, EB_F32, "k", dev));
    EB_TRY(check_tensor(v, EB_F32, "v", dev));
    CacheI8 c;
    EB_TRY(layer_of(kv, layer, dev, &c));
    if (c.hkv != d.n_kv_heads || c.hd != d.head_dim)
        return fail(EB_SHAPE_MISMATCH, "attention_forward: the block-scaled cache has %zu heads of %zu, not %zu of %zu",
                    c.hkv, c.hd, d.n_kv_heads, d.head_dim);
    const size_t H = d.n_heads, hd = d.head_dim, g = H / c.hkv;
    DecodePrologue pro{};
    EB_TRY(prologue_of(d, rope, base_pos + rows - 1, dev, &pro));
    EB_TRY(eb::check_numel(eb_tensor_numel(q), {rows, H, hd}, "q"));
    EB_TRY(eb::check_numel(eb_tensor_numel(k), {rows, c.hkv, hd}, "k"));
    const size_t oshape[2] = {rows, H * hd};
    eb_tensor *t = nullptr;
    EB_TRY(eb_tensor_empty(dev, oshape, 2, EB_F32, &t));
    Owned o(t);
    const Room src{dev};
    const int cus = eb_device_cu_count(dev);
    const hipStream_t st = stream_of(dev);
    if (rows == 1 && g <= kDecodeI8Cols) {
        EB_TRY(attend_i8(st, src, cus, c, data<float>(q), data<float>(k), data<float>(v), data<float>(o.t), H,
                         base_pos, 1, d.scale, d.window, &pro));
        *out = o.release();
        return eb::ok();
    }
    // The row pass (norms, RoPE) into f32 rows, their codes, then the attention.
    const size_t qshape[3] = {rows, H, hd}, kshape[3] = {rows, c.hkv, hd};
    EB_TRY(eb_tensor_empty(dev, qshape, 3, EB_F32, &t));
    Owned qr(t);
    EB_TRY(eb_tensor_empty(dev, kshape, 3, EB_F32, &t));
    Owned kr(t);
    EB_TRY(eb_tensor_empty(dev, kshape, 3, EB_F32, &t));
    Owned vr(t);
    RowsArgs a{};
    a.nseg = 3;
    a.seg[0] = RowSeg{data<float>(q), data<float>(qr.t), pro.q_norm, (int)H, 0, true, 4};
    a.seg[1] = RowSeg{data<float>(k), data<float>(kr.t), pro.k_norm, (int)c.hkv, 0, true, 4};
    a.seg[2] = RowSeg{data<float>(v), data<float>(vr.t), pro.v_norm, (int)c.hkv, 0, false, 4};
    a.rows = (int)rows;
    a.hd = (int)hd;
    a.eps = pro.eps;
    a.cosb = pro.rope_cos;
    a.sinb = pro.rope_sin;
    a.rope_row0 = (int)base_pos;
    EB_TRY(launch_attn_rows(st, a));
    EB_TRY(launch_kv_write_i8(st, c, data<float>(kr.t), data<float>(vr.t), base_pos, rows));
    EB_TRY(attend_i8(st, src, cus, c, data<float>(qr.t), nullptr, nullptr, data<float>(o.t), H, base_pos, rows,
                     d.scale, d.window));
    *out = o.release();
    return eb::ok();
}

extern "C" {

eb_status eb_kv_cache_new_i8(eb_device *dev, const size_t *head_dims, size_t n_layers, size_t max_seq,
                             size_t n_kv_heads, size_t block, eb_kv_cache **out) {
    if (!dev || !out || (n_layers > 0 && !head_dims)) return fail(EB_OTHER, "kv_cache: null argument");
    *out = nullptr;
    for (size_t l = 0; l < n_layers; ++l) EB_TRY(shape_i8(max_seq, n_kv_heads, head_dims[l], block));
    if (n_layers == 0) EB_TRY(shape_i8(max_seq, n_kv_heads, 32, block));
    EB_TRY(eb::make_current(dev));
    EB_TRY(not_captured(stream_of(dev), "kv_cache"));  // (a replay would clear the exponents)
    struct Release {
        void operator()(eb_kv_cache *kv) const { eb_kv_cache_release(kv); }
    };
    std::unique_ptr<eb_kv_cache, Release> kv(new eb_kv_cache());
    kv->max_seq = max_seq;
    kv->n_kv_heads = n_kv_heads;
    kv->block = block;
    const size_t blocks = (max_seq + block - 1) / block;
    for (size_t l = 0; l < n_layers; ++l) {
        const size_t shape[3] = {max_seq, n_kv_heads, head_dims[l]}, eshape[2] = {blocks, n_kv_heads};
        std::vector<eb_tensor *> *to[4] = {&kv->k, &kv->v, &kv->k_scale, &kv->v_scale};
        for (int i = 0; i < 4; ++i) {
            eb_tensor *t = nullptr;
            EB_TRY(i < 2 ? eb_tensor_empty(dev, shape, 3, EB_I8, &t) : eb_tensor_empty(dev, eshape, 2, EB_U8, &t));
            to[i]->push_back(t);
            // No row is written yet: the least exponent, so that a first row anywhere in a block
            // meets no old one.
            if (i >= 2 && blocks > 0)
                EB_TRY(eb::launch_fill_u8(stream_of(dev), data<uint8_t>(t), 1, blocks * n_kv_heads));
        }
    }
    kv->draft_k.resize(n_layers);
    kv->draft_v.resize(n_layers);
    const size_t tshape[4] = {n_layers, 2, n_kv_heads, eb::kTagWords};
    EB_TRY(eb_tensor_empty(dev, tshape, 4, EB_U32, &kv->draft_tags));
    kv->id = cache_number(kv.get());
    // Complete, as a tensor's write is: the next one to touch the exponents may be another stream,
    // which nothing orders behind this one.
    EB_HIP_TRY(hipStreamSynchronize(stream_of(dev)));
    *out = kv.release();
    return eb::ok();
}

eb_tensor *eb_kv_cache_k_scale(eb_kv_cache *kv, size_t layer) {
    return (kv && layer < kv->k_scale.size()) ? kv->k_scale[layer] : nullptr;
}
eb_tensor *eb_kv_cache_v_scale(eb_kv_cache *kv, size_t layer) {
    return (kv && layer < kv->v_scale.size()) ? kv->v_scale[layer] : nullptr;
}
size_t eb_kv_cache_block(const eb_kv_cache *kv) { return kv ? kv->block : 0; }

eb_status eb_kv_write_i8(eb_recorder *rec, eb_kv_cache *kv, size_t layer, const eb_tensor *k, const eb_tensor *v,
                         size_t count, size_t dst_start) {
    eb_device *dev;
    EB_TRY(eb::recorder_ready(rec, &dev));
    eb::CacheI8 c;
    EB_TRY(layer_of(kv, layer, dev, &c));
    EB_TRY(eb::check_tensor(k, EB_F32, "k", dev));
    EB_TRY(eb::check_tensor(v, EB_F32, "v", dev));
    return move_i8(stream_of(dev), "kv_write_i8", c, data<float>(k), data<float>(v),
                   std::min(eb_tensor_numel(k), eb_tensor_numel(v)), count, dst_start, nullptr, nullptr);
}

eb_status eb_kv_read_i8(eb_recorder *rec, const eb_kv_cache *kv, size_t layer, eb_tensor *k, eb_tensor *v,
                        size_t count, size_t src_start) {
    eb_device *dev;
    EB_TRY(eb::recorder_ready(rec, &dev));
    eb::CacheI8 c;
    EB_TRY(layer_of(kv, layer, dev, &c));
    EB_TRY(eb::check_tensor(k, EB_F32, "k", dev));
    EB_TRY(eb::check_tensor(v, EB_F32, "v", dev));
    return move_i8(stream_of(dev), "kv_read_i8", c, data<float>(k), data<float>(v),
                   std::min(eb_tensor_numel(k), eb_tensor_numel(v)), count, src_start, data<float>(k), data<float>(v));
}

static eb_status attn_handle(eb_recorder *rec, const eb_tensor *q, const eb_tensor *knew, const eb_tensor *vnew,
                             const eb_kv_cache *kv, size_t layer, eb_tensor *o, size_t h, size_t pos0, size_t rows,
                             float scale, size_t window, bool step) {
    eb_device *dev;
    EB_TRY(eb::recorder_ready(rec, &dev));
    eb::CacheI8 c;
    EB_TRY(layer_of(kv, layer, dev, &c));
    EB_TRY(eb::check_tensor(q, EB_F32, "q", dev));
    EB_TRY(eb::check_tensor(o, EB_F32, "o", dev));
    EB_TRY(attn_checked(c, data<float>(q), eb_tensor_numel(q), data<float>(o), eb_tensor_numel(o), h, pos0, rows));
    if (step) {
        EB_TRY(eb::check_tensor(knew, EB_F32, "knew", dev));
        EB_TRY(eb::check_tensor(vnew, EB_F32, "vnew", dev));
        EB_TRY(step_checked(c, data<float>(knew), data<float>(vnew),
                            std::min(eb_tensor_numel(knew), eb_tensor_numel(vnew))));
    }
    return attend_i8(stream_of(dev), Room{dev}, eb_device_cu_count(dev), c, data<float>(q),
                     step ? data<float>(knew) : nullptr, step ? data<float>(vnew) : nullptr, data<float>(o), h, pos0,
                     rows, scale, window);
}

eb_status eb_attn_decode_i8(eb_recorder *rec, const eb_tensor *q, const eb_kv_cache *kv, size_t layer, eb_tensor *o,
                            size_t h, size_t pos, float scale, size_t window) {
    return attn_handle(rec, q, nullptr, nullptr, kv, layer, o, h, pos, 1, scale, window, false);
}

eb_status eb_attn_decode_step_i8(eb_recorder *rec, const eb_tensor *q, const eb_tensor *knew, const eb_tensor *vnew,
                                 eb_kv_cache *kv, size_t layer, eb_tensor *o, size_t h, size_t pos, float scale,
                                 size_t window) {
    return attn_handle(rec, q, knew, vnew, kv, layer, o, h, pos, 1, scale, window, true);
}

eb_status eb_attn_prefill_chunk_i8(eb_recorder *rec, const eb_tensor *q, const eb_kv_cache *kv, size_t layer,
                                   eb_tensor *o, size_t h, size_t pos0, size_t rows, float scale, size_t window) {
    return attn_handle(rec, q, nullptr, nullptr, kv, layer, o, h, pos0, rows, scale, window, false);
}

eb_status eb_launch_kv_write_i8(void *stream, const eb_cache_i8 *cache, const float *k, const float *v, size_t numel,
                                size_t count, size_t dst_start) {
    eb::CacheI8 c;
    EB_TRY(eb::cache_i8_of(cache, &c));
    return move_i8((hipStream_t)stream, "kv_write_i8", c, k, v, numel, count, dst_start, nullptr, nullptr);
}

eb_status eb_launch_kv_read_i8(void *stream, const eb_cache_i8 *cache, float *k, float *v, size_t numel, size_t count,
                               size_t src_start) {
    eb::CacheI8 c;
    EB_TRY(eb::cache_i8_of(cache, &c));
    return move_i8((hipStream_t)stream, "kv_read_i8", c, k, v, numel, count, src_start, k, v);
}

size_t eb_attn_i8_workspace_floats(size_t h, size_t hkv, size_t hd, size_t pos0, size_t rows, size_t block,
                                   size_t window, int cu_count) {
    if (rows == 0 || hkv == 0 || h == 0 || h % hkv != 0 || shape_i8(0, hkv, hd, block) != EB_OK || pos0 > kMaxRows ||
        rows > kMaxRows)
        return 0;
    return attn_workspace(h, hkv, hd, pos0, rows, window, block, cu_count > 0 ? cu_count : 256);
}

eb_status eb_launch_attn_decode_i8(void *stream, const float *q, size_t q_numel, const float *knew, const float *vnew,
                                   size_t new_numel, const eb_cache_i8 *cache, float *o, size_t o_numel, size_t h,
                                   size_t pos, float scale, size_t window, float *workspace, size_t workspace_floats,
                                   int cu_count) {
    eb::CacheI8 c;
    EB_TRY(eb::cache_i8_of(cache, &c));
    EB_TRY(attn_checked(c, q, q_numel, o, o_numel, h, pos, 1));
    if (knew || vnew) EB_TRY(step_checked(c, knew, vnew, new_numel));
    return attend_i8((hipStream_t)stream, Room{nullptr, workspace, workspace_floats}, cu_count > 0 ? cu_count : 256, c,
                     q, knew, vnew, o, h, pos, 1, scale, window);
}

eb_status eb_launch_attn_prefill_chunk_i8(void *stream, const float *q, size_t q_numel, const eb_cache_i8 *cache,
                                          float *o, size_t o_numel, size_t h, size_t pos0, size_t rows, float scale,
                                          size_t window, float *workspace, size_t workspace_floats, int cu_count) {
    eb::CacheI8 c;
    EB_TRY(eb::cache_i8_of(cache, &c));
    EB_TRY(attn_checked(c, q, q_numel, o, o_numel, h, pos0, rows));
    return attend_i8((hipStream_t)stream, Room{nullptr, workspace, workspace_floats}, cu_count > 0 ? cu_count : 256, c,
                     q, nullptr, nullptr, o, h, pos0, rows, scale, window);
}

// ---- 4-bit projections ------------------------------------------------------------------------

// A weight's shape; its sizes are indexed with 32 bits.
static eb_status q4_shape(size_t in_f, size_t out_f, size_t group) {
    if (group != 32 && group != 64 && group != 128)
        return fail(EB_UNSUPPORTED_CONFIG, "4-bit weight: group %zu (32, 64 or 128)", group);
    if (in_f == 0 || in_f % group != 0)
        return fail(EB_SHAPE_MISMATCH, "4-bit weight: in_f %zu is not a positive multiple of the group %zu", in_f, group);
    if (in_f > ((size_t)1 << 24)) return fail(EB_UNSUPPORTED_CONFIG, "4-bit weight: in_f %zu (at most 2^24)", in_f);
    return eb::check_numel(SIZE_MAX, {out_f + 15, in_f / 8}, "4-bit weight");
}

size_t eb_q4_packed_bytes(size_t in_f, size_t out_f, size_t group, int zeros) {
    return q4_shape(in_f, out_f, group) == EB_OK ? eb::q4_packed_bytes(in_f, out_f, group, zeros != 0) : 0;
}

static eb_status pack_checked(hipStream_t st, const uint32_t *w, size_t words, const uint16_t *scales, size_t sn,
                              const uint8_t *zeros, size_t zn, size_t in_f, size_t out_f, size_t group, void *packed,
                              size_t bytes) {
    EB_TRY(q4_shape(in_f, out_f, group));
    EB_TRY(eb::check_numel(words, {out_f, in_f / 8}, "w"));
    EB_TRY(eb::check_numel(sn, {out_f, in_f / group}, "scales"));
    if (zeros) EB_TRY(eb::check_numel(zn, {out_f, in_f / group}, "zeros"));
    EB_TRY(holds(bytes, eb::q4_packed_bytes(in_f, out_f, group, zeros != nullptr), "packed"));
    if (out_f == 0) return eb::ok();
    EB_TRY(eb::check_ptr(w, "w"));
    EB_TRY(eb::check_ptr(scales, "scales"));
    EB_TRY(eb::check_ptr(packed, "packed"));
    EB_TRY(aligned({w}, 4, "q4_pack: w"));
    EB_TRY(aligned({scales}, 2, "q4_pack: scales"));
    EB_TRY(aligned({packed}, 16, "q4_pack: packed"));
    EB_TRY(eb::launch_q4_pack(st, w, scales, zeros, static_cast<uint8_t *>(packed), in_f, out_f, group));
    return eb::ok();
}

eb_status eb_q4_pack(eb_recorder *rec, const eb_tensor *w, const eb_tensor *scales, const eb_tensor *zeros, size_t in_f,
                     size_t out_f, size_t group, eb_tensor **packed) {
    if (!packed) return fail(EB_OTHER, "q4_pack: out is null");
    *packed = nullptr;
    eb_device *dev;
    EB_TRY(eb::recorder_ready(rec, &dev));
    EB_TRY(eb::check_tensor(w, EB_U32, "w", dev));
    EB_TRY(eb::check_tensor(scales, EB_F16, "scales", dev));
    if (zeros) EB_TRY(eb::check_tensor(zeros, EB_U8, "zeros", dev));
    EB_TRY(q4_shape(in_f, out_f, group));
    // Like a tensor's write, complete when it returns, and ordered behind the null stream, on which
    // other libraries fill weights; the sources are reused as soon as they are packed. (Not behind
    // every stream: a wait for the whole device would end a capture that another of its streams runs.)
    const hipStream_t st = stream_of(dev);
    EB_TRY(not_captured(st, "q4_pack"));
    EB_HIP_TRY(hipStreamSynchronize(nullptr));
    const size_t bytes = eb::q4_packed_bytes(in_f, out_f, group, zeros != nullptr);
    eb_tensor *t = nullptr;
    EB_TRY(eb_tensor_empty(dev, &bytes, 1, EB_U8, &t));
    Owned p(t);
    EB_TRY(pack_checked(st, data<uint32_t>(w), eb_tensor_numel(w), data<uint16_t>(scales),
                        eb_tensor_numel(scales), zeros ? data<uint8_t>(zeros) : nullptr, zeros ? eb_tensor_numel(zeros) : 0,
                        in_f, out_f, group, data<void>(p.t), bytes));
    EB_HIP_TRY(hipStreamSynchronize(st));
    *packed = p.release();
    return eb::ok();
}

eb_status eb_launch_q4_pack(void *stream, const uint32_t *w, size_t w_words, const uint16_t *scales, size_t scales_numel,
                            const uint8_t *zeros, size_t zeros_numel, size_t in_f, size_t out_f, size_t group,
                            void *packed, size_t packed_bytes) {
    return pack_checked((hipStream_t)stream, w, w_words, scales, scales_numel, zeros, zeros_numel, in_f, out_f, group,
                        packed, packed_bytes);
}

static eb_status q4_checked(hipStream_t st, const Room &src, const float *a, size_t an, const eb::Q4Weight *w,
                            const size_t *bytes, float *const *c, const size_t *cn, int n, size_t m) {
    const size_t in_f = w[0].in_f, group = w[0].group;
    for (int i = 0; i < n; ++i) {
        EB_TRY(q4_shape(w[i].in_f, w[i].out_f, w[i].group));
        if (w[i].in_f != in_f || w[i].group != group || w[i].zeros != w[0].zeros)
            return fail(EB_SHAPE_MISMATCH, "linear_q4: the weights of a launch share in_f and group, and have zero "
                        "points all or none");
        EB_TRY(holds(bytes[i], eb::q4_packed_bytes(in_f, w[i].out_f, group, w[i].zeros), "packed"));
        EB_TRY(eb::check_numel(cn[i], {m, w[i].out_f}, "c"));
    }
    EB_TRY(eb::check_numel(an, {m, in_f}, "a"));
    if (m == 0) return eb::ok();
    EB_TRY(eb::check_ptr(a, "a"));
    EB_TRY(aligned({a}, 16, "linear_q4: a"));
    for (int i = 0; i < n; ++i) {
        if (w[i].out_f == 0) continue;
        EB_TRY(eb::check_ptr(w[i].packed, "packed"));
        EB_TRY(eb::check_ptr(c[i], "c"));
        EB_TRY(aligned({w[i].packed}, 16, "linear_q4: packed"));
    }
    float *ws;
    WsLock lk;
    EB_TRY(room(src, eb::linear_q4_workspace_floats(m, in_f), &ws, lk));
    EB_TRY(eb::launch_linear_q4(st, a, w, c, n, m, ws));
    return eb::ok();
}

eb_status eb_linear_q4_multi(eb_recorder *rec, const eb_tensor *a, size_t n, const eb_q4_weight *w,
                             eb_tensor *const *c, size_t m) {
    eb_device *dev;
    EB_TRY(eb::recorder_ready(rec, &dev));
    constexpr int kMax = eb::kLinearMaxSegs;
    if (n < 1 || n > (size_t)kMax || !w || !c) return fail(EB_OTHER, "linear_q4: 1 to %d weights per launch", kMax);
    EB_TRY(eb::check_tensor(a, EB_F32, "a", dev));
    eb::Q4Weight q[kMax];
    float *y[kMax];
    size_t bytes[kMax], cn[kMax];
    for (size_t i = 0; i < n; ++i) {
        EB_TRY(eb::check_tensor(w[i].packed, EB_U8, "packed", dev));
        EB_TRY(eb::check_tensor(c[i], EB_F32, "c", dev));
        q[i] = eb::Q4Weight{data<uint8_t>(w[i].packed), w[i].in_f, w[i].out_f, w[i].group, w[i].zeros != 0};
        y[i] = data<float>(c[i]);
        bytes[i] = eb_tensor_numel(w[i].packed);
        cn[i] = eb_tensor_numel(c[i]);
    }
    return q4_checked(stream_of(dev), Room{dev}, data<float>(a), eb_tensor_numel(a), q, bytes, y, cn, (int)n, m);
}

eb_status eb_linear_q4(eb_recorder *rec, const eb_tensor *a, const eb_q4_weight *w, eb_tensor *c, size_t m) {
    return eb_linear_q4_multi(rec, a, 1, w, &c, m);
}

size_t eb_linear_q4_workspace_floats(size_t m, size_t in_f) { return eb::linear_q4_workspace_floats(m, in_f); }

eb_status eb_launch_linear_q4(void *stream, const float *a, size_t a_numel, const void *packed, size_t packed_bytes,
                              float *c, size_t c_numel, size_t m, size_t in_f, size_t out_f, size_t group, int zeros,
                              float *workspace, size_t workspace_floats) {
    const eb::Q4Weight q{static_cast<const uint8_t *>(packed), in_f, out_f, group, zeros != 0};
    return q4_checked((hipStream_t)stream, Room{nullptr, workspace, workspace_floats}, a, a_numel, &q, &packed_bytes, &c,
                      &c_numel, 1, m);
}

eb_status eb_attention_new_q4(const eb_attention_desc *desc, const eb_q4_weight proj[4], eb_attention **out) {
    if (!desc || !proj || !out) return fail(EB_OTHER, "attention_new: null argument");
    *out = nullptr;
    if (desc->q_proj || desc->k_proj || desc->v_proj || desc->o_proj)
        return fail(EB_SHAPE_MISMATCH, "attention_new_q4: the descriptor's projections must be null");
    if (desc->hidden == 0) return fail(EB_SHAPE_MISMATCH, "attention: hidden must be > 0");
    const size_t qd = desc->n_heads * desc->head_dim, kd = desc->n_kv_heads * desc->head_dim;
    const size_t outs[4] = {qd, kd, kd, desc->hidden}, ins[4] = {desc->hidden, desc->hidden, desc->hidden, qd};
    for (int i = 0; i < 4; ++i) {
        const eb_q4_weight &p = proj[i];
        if (p.out_f != outs[i] || p.in_f != ins[i])
            return fail(EB_SHAPE_MISMATCH, "attention: projection %d is [%zu, %zu], must be [%zu, %zu]", i, p.out_f,
                        p.in_f, outs[i], ins[i]);
        EB_TRY(q4_shape(p.in_f, p.out_f, p.group));
        if (!p.packed || eb_tensor_dtype(p.packed) != EB_U8 ||
            eb_tensor_numel(p.packed) < eb::q4_packed_bytes(p.in_f, p.out_f, p.group, p.zeros != 0))
            return fail(EB_SHAPE_MISMATCH, "attention: projection %d is not a packed 4-bit weight of its shape", i);
        if (i < 3 && (p.group != proj[0].group || (p.zeros != 0) != (proj[0].zeros != 0)))
            return fail(EB_SHAPE_MISMATCH, "attention: q, k and v share a group, and have zero points all or none");
    }
    eb_attention *a = nullptr;
    EB_TRY(eb_attention_new(desc, &a));
    a->q4 = true;
    for (int i = 0; i < 4; ++i) a->proj[i] = proj[i];
    *out = a;
    return eb::ok();
}

// ---- sampling -----------------------------------------------------------------------------------

static eb_status sample_checked(hipStream_t st, const Room &src, const eb::SampleArgs &a, size_t numel) {
    EB_TRY(eb::check_numel(numel, {a.rows, a.vocab}, "logits"));
    if (a.rows == 0) return eb::ok();
    if (a.vocab == 0) return fail(EB_SHAPE_MISMATCH, "sample: vocab must be > 0");
    if (a.vocab > ((size_t)1 << 24) || a.rows > 65535)
        return fail(EB_UNSUPPORTED_CONFIG, "sample: [%zu, %zu] logits (at most 65535 rows of a vocab of 2^24)", a.rows,
                    a.vocab);
    EB_TRY(eb::check_ptr(a.logits, "logits"));
    EB_TRY(eb::check_ptr(a.u, "u"));
    EB_TRY(eb::check_ptr(a.out, "out_idx"));
    float *ws;
    WsLock lk;
    EB_TRY(room(src, eb::sample_workspace_floats(a.rows, a.vocab), &ws, lk));
    EB_TRY(eb::launch_sample(st, a, ws));
    return eb::ok();
}

eb_status eb_sample(eb_recorder *rec, const eb_tensor *logits, const eb_tensor *u, eb_tensor *out_idx, size_t rows,
                    size_t vocab, const eb_tensor *temperature, const eb_tensor *top_k, const eb_tensor *top_p,
                    const eb_tensor *min_p) {
    eb_device *dev;
    EB_TRY(eb::recorder_ready(rec, &dev));
    EB_TRY(eb::check_tensor(logits, EB_F32, "logits", dev));
    EB_TRY(eb::check_tensor(u, EB_F32, "u", dev));
    EB_TRY(eb::check_tensor(out_idx, EB_U32, "out_idx", dev));
    const struct {
        const eb_tensor *t;
        eb_dtype dt;
        const char *name;
    } per_row[] = {{u, EB_F32, "u"}, {out_idx, EB_U32, "out_idx"}, {temperature, EB_F32, "temperature"},
                   {top_k, EB_U32, "top_k"}, {top_p, EB_F32, "top_p"}, {min_p, EB_F32, "min_p"}};
    for (const auto &p : per_row) {
        if (!p.t) continue;
        EB_TRY(eb::check_tensor(p.t, p.dt, p.name, dev));
        EB_TRY(eb::check_numel(eb_tensor_numel(p.t), rows, p.name));
    }
    eb::SampleArgs a{data<float>(logits), data<float>(u), temperature ? data<float>(temperature) : nullptr,
                     top_k ? data<uint32_t>(top_k) : nullptr, top_p ? data<float>(top_p) : nullptr,
                     min_p ? data<float>(min_p) : nullptr, data<uint32_t>(out_idx), rows, vocab};
    return sample_checked(stream_of(dev), Room{dev}, a, eb_tensor_numel(logits));
}

size_t eb_sample_workspace_floats(size_t rows, size_t vocab) {
    if (rows == 0 || vocab == 0) return 0;
    return eb::sample_workspace_floats(rows, vocab);
}

eb_status eb_launch_sample(void *stream, const float *logits, size_t logits_numel, const float *u, uint32_t *out_idx,
                           size_t rows, size_t vocab, const float *temperature, const uint32_t *top_k,
                           const float *top_p, const float *min_p, float *workspace, size_t workspace_floats) {
    const eb::SampleArgs a{logits, u, temperature, top_k, top_p, min_p, out_idx, rows, vocab};
    return sample_checked((hipStream_t)stream, Room{nullptr, workspace, workspace_floats}, a, logits_numel);
}

}  // extern "C"
