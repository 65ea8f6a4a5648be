// What the two kernels of syn_tree_attention share (tree_attention.cu, tree_attention_tc.cu).
#pragma once

#include "kv_cache.cuh"

namespace syn {

constexpr float kPShift = 8.0f;      // probabilities carry 2^8, away from binary16's subnormals
constexpr int kMaxTree = 1024;

struct TreeParams {
    KvView c;
    const float* q;
    float* out;
    const int32_t* len;
    const uint32_t* mask;
    float2* part_ml;     // [n_seq][n_kv * row blocks][splits][R]: a part's maximum and sum of a row
    float* part_o;       // [n_seq][n_kv * row blocks][splits][R][hd]: its output, not divided
    size_t q_stride;
    int n_tree, n_head, group, rows, row_blocks, max_len, mask_words, splits;
    float scale_log2;    // scale * log2(e)
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 half2_of(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
// (x, y) as binary16 pairs hi + lo.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    hi = bits(h);
    lo = bits(__floats2half2_rn(x - f.x, y - f.y));
}
// Bytes i and j of x as binary16 integers 1024 + byte.
__device__ __forceinline__ __half2 bytes_h2(uint32_t x, uint32_t sel) { return half2_of(__byte_perm(x, 0x64646464u, sel)); }

// The power of two that brings a row of q with largest magnitude m to a
// maximum in [2^8, 2^9), and its inverse; zero, subnormal and non-finite rows
// take 2^8.
__device__ __forceinline__ void q_factor(float m, float& up, float& down) {
    const int e = int(__float_as_uint(m) >> 23);
    const bool plain = e < 32 || e > 250;
    up = plain ? 256.0f : __uint_as_float(uint32_t(254 + 8 - e) << 23);
    down = plain ? 1.0f / 256.0f : __uint_as_float(uint32_t(e - 8) << 23);
}
// Whether token tk of sequence seq sees the tree's row j >= 0.
__device__ __forceinline__ bool tree_sees(const TreeParams& a, int seq, int tk, int j) {
    if (j >= a.n_tree || tk >= a.n_tree) return false;
    return a.mask ? a.mask[(size_t(seq) * a.n_tree + tk) * a.mask_words + (j >> 5)] >> (j & 31) & 1u : j <= tk;
}
// The weight of a part with running maximum m and sum l among parts whose
// largest maximum is top: a NaN sum stays NaN, a part that saw nothing weighs 0.
__device__ __forceinline__ float part_weight(float m, float l, float top) {
    return m == -INFINITY ? (l != l ? 1.0f : 0.0f) : ex2(m - top);
}

}  // namespace syn

// The tcgen05 kernel (tree_attention_tc.cu): 128 rows of a KV head per CTA,
// heads of up to 128 dims; a.splits counts runs of 64 positions' tiles.
constexpr int kTcRows = 128, kTcTile = 64;
int syn_tree_attention_tc(const syn::TreeParams& a, int type, cudaStream_t s);
