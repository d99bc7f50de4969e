// The handles of the nn layer, shared by the translation units that define its entry points.
#pragma once

#include <vector>

#include "eb_internal.h"

struct eb_rope_tables {
    eb_tensor *cos = nullptr;
    eb_tensor *sin = nullptr;
    size_t head_dim = 0;
    size_t max_seq = 0;
};

struct eb_kv_cache {
    std::vector<eb_tensor *> k, v;
    // A block-scaled 8-bit cache: its exponents per layer and the rows of a block (0: none).
    std::vector<eb_tensor *> k_scale, v_scale;
    size_t block = 0;
    size_t max_seq = 0;
    size_t n_kv_heads = 0;
};

struct eb_attention {
    eb_attention_desc d{};
    bool q4 = false;  // the projections are proj (q, k, v, o) instead of the descriptor's
    eb_q4_weight proj[4] = {};
};

namespace eb {

// Owns a tensor for the duration of a forward; released (back to the pool) on scope exit.
struct Owned {
    eb_tensor *t = nullptr;
    Owned() = default;
    explicit Owned(eb_tensor *x) : t(x) {}
    Owned(const Owned &) = delete;
    Owned &operator=(const Owned &) = delete;
    ~Owned() { eb_tensor_release(t); }
    eb_tensor *release() {
        eb_tensor *x = t;
        t = nullptr;
        return x;
    }
};

// Attention::forward between the projections over a block-scaled cache (eb_quant.cpp); the
// arguments are checked as far as eb_attention_forward_qkv checks them for every cache.
eb_status attention_forward_i8(const eb_attention_desc &d, eb_recorder *rec, const eb_tensor *q,
                               const eb_tensor *k, const eb_tensor *v, const eb_rope_tables *rope,
                               eb_kv_cache *kv, size_t layer, size_t rows, size_t base_pos, eb_tensor **out);

}  // namespace eb
