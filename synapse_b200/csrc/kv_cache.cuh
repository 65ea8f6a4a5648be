// Geometry of the KV caches behind syn_kv_cache (F16, Q8_0, Q4_0), shared by
// the kernels that write, read, move and attend over them.
#pragma once

#include "common.cuh"

namespace syn {

// Quants bytes of a block of 32 values in a planar cache.
__host__ __device__ constexpr int kv_block_bytes(int type) { return type == SYN_Q4_0 ? 16 : 32; }

// One layer of a cache, by value to the kernels.
struct KvView {
    char* k;
    char* v;
    size_t seq_stride;   // bytes between sequences
    size_t scale_plane;  // byte offset of the scales (quantised types)
    int n_seq, n_kv, hd, max_ctx;
};

__host__ __device__ inline size_t kv_quant_plane(int type, int n_kv, int hd, int max_ctx) {
    return align256(size_t(n_kv) * max_ctx * (hd / QK) * kv_block_bytes(type));
}

inline bool kv_type(int type) { return type == SYN_F16 || type == SYN_Q8_0 || type == SYN_Q4_0; }

// Checks of a syn_kv_cache and a layer of it.
inline int kv_check(const syn_kv_cache* c, int layer) {
    if (!c || !c->k || !c->v || c->n_layer <= 0 || c->n_seq <= 0 || c->n_kv <= 0 || c->max_ctx <= 0)
        return SYN_ERR_INVALID;
    if (layer < 0 || layer >= c->n_layer) return SYN_ERR_INVALID;
    if (!kv_type(c->type)) return SYN_ERR_UNSUPPORTED;
    const int unit = c->type == SYN_F16 ? 8 : QK;
    if (c->head_dim <= 0 || c->head_dim % unit || c->head_dim > 256) return SYN_ERR_UNSUPPORTED;
    const uintptr_t at = reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v) | c->seq_stride |
                         c->layer_stride;
    if (at & 15) return SYN_ERR_INVALID;
    const size_t bytes = syn_kv_cache_bytes(c->type, c->n_kv, c->head_dim, c->max_ctx);
    if (c->n_seq > 1 && c->seq_stride < bytes) return SYN_ERR_INVALID;
    if (c->n_layer > 1 && c->layer_stride < bytes) return SYN_ERR_INVALID;
    return SYN_OK;
}

inline KvView kv_view(const syn_kv_cache* c, int layer) {
    KvView w;
    const size_t off = size_t(layer) * c->layer_stride;
    w.k = static_cast<char*>(c->k) + off;
    w.v = static_cast<char*>(c->v) + off;
    w.seq_stride = c->seq_stride;
    w.scale_plane = c->type == SYN_F16 ? 0 : kv_quant_plane(c->type, c->n_kv, c->head_dim, c->max_ctx);
    w.n_seq = c->n_seq;
    w.n_kv = c->n_kv;
    w.hd = c->head_dim;
    w.max_ctx = c->max_ctx;
    return w;
}

}  // namespace syn
