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
    unsigned* arrived;   // [n_seq][n_kv * row blocks]: parts that are done; zero between calls
    int2* cuts;          // [n_seq]: a sequence's first part and number of parts, for tree_join_kernel; or NULL
    float2* part_ml;     // [parts][n_kv * row blocks][R]: a part's maximum and sum of a row
    float* part_o;       // [parts][n_kv * row blocks][R][hd]: its output, not divided
    size_t q_stride;
    int n_tree, n_head, group, rows, row_blocks, max_len, mask_words;
    int parts;           // that the contexts may be cut into, more than n_seq; 0: not cut
    float scale_log2;    // scale * log2(e)
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
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
// a += b, of two floats each.
__device__ __forceinline__ void add2(float& a0, float& a1, float b0, float b1) {
    asm("{\n .reg .b64 a, b;\n mov.b64 a, {%0, %1};\n mov.b64 b, {%2, %3};\n add.rn.f32x2 a, a, b;\n mov.b64 {%0, %1}, a;\n}\n"
        : "+f"(a0), "+f"(a1)
        : "f"(b0), "f"(b1));
}
// a *= b; a = a f + b; a += b c, of two floats each.
__device__ __forceinline__ void mul2(float& a0, float& a1, float b0, float b1) {
    asm("{\n .reg .b64 a, b;\n mov.b64 a, {%0, %1};\n mov.b64 b, {%2, %3};\n mul.rn.f32x2 a, a, b;\n mov.b64 {%0, %1}, a;\n}\n"
        : "+f"(a0), "+f"(a1)
        : "f"(b0), "f"(b1));
}
__device__ __forceinline__ void fma2(float& a0, float& a1, float f0, float f1, float b0, float b1) {
    asm("{\n .reg .b64 a, f, b;\n mov.b64 a, {%0, %1};\n mov.b64 f, {%2, %3};\n mov.b64 b, {%4, %5};\n"
        " fma.rn.f32x2 a, a, f, b;\n mov.b64 {%0, %1}, a;\n}\n"
        : "+f"(a0), "+f"(a1)
        : "f"(f0), "f"(f1), "f"(b0), "f"(b1));
}
__device__ __forceinline__ void fma2_to(float& a0, float& a1, float b0, float b1, float c0, float c1) {
    asm("{\n .reg .b64 a, b, c;\n mov.b64 a, {%0, %1};\n mov.b64 b, {%2, %3};\n mov.b64 c, {%4, %5};\n"
        " fma.rn.f32x2 a, b, c, a;\n mov.b64 {%0, %1}, a;\n}\n"
        : "+f"(a0), "+f"(a1)
        : "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
// (x, y) as binary16 pairs hi + lo.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    float2 f = __half22float2(h);
    fma2(f.x, f.y, -1.0f, -1.0f, x, y);
    hi = bits(h);
    lo = bits(__floats2half2_rn(f.x, f.y));
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
// How the sequences' contexts are cut into parts: of one length, `per` steps,
// whatever the sequences' lengths, numbered through the sequences, and the
// shortest of which there are at most a.parts (0: a part is a sequence).
struct Cutting {
    int seq;    // the part's sequence, -1: there are not so many parts
    int per;    // steps of a part
    int first;  // the sequence's first part
    int parts;  // and its number of parts
};
__device__ __forceinline__ int tree_len(const TreeParams& a, int seq) {
    return min(max(__ldg(a.len + seq), 0), a.max_len - a.n_tree);
}
__device__ __forceinline__ int tree_steps(const TreeParams& a, int seq, int step) {
    return (tree_len(a, seq) + a.n_tree + step - 1) / step;
}
// For a warp: the sequence that holds part `part`, and its cutting.
__device__ __forceinline__ Cutting tree_cutting(const TreeParams& a, int step, int part) {
    const int lane = threadIdx.x & 31, n = a.c.n_seq;
    if (a.parts == 0) return {part, 0x3fffffff, part, 1};
    if (n == 1) {
        const int steps = tree_steps(a, 0, step), per = (steps + a.parts - 1) / a.parts, parts = (steps + per - 1) / per;
        return {part < parts ? 0 : -1, per, 0, parts};
    }
    const int own = lane < n ? tree_steps(a, lane, step) : 0;
    int total = own;
    for (int s = 32 + lane; s < n; s += 32) total += tree_steps(a, s, step);
    total = __reduce_add_sync(0xffffffffu, total);
    // total / per + n parts are enough, so there are at most a.parts of the second length
    int per = (total + a.parts - 1) / a.parts, most = (total + a.parts - n - 1) / (a.parts - n);
    while (per < most) {
        const int mid = (per + most) / 2;
        int parts = (own + mid - 1) / mid;
        for (int s = 32 + lane; s < n; s += 32) parts += (tree_steps(a, s, step) + mid - 1) / mid;
        parts = __reduce_add_sync(0xffffffffu, parts);
        if (parts <= a.parts) most = mid;
        else per = mid + 1;
    }
    int before = 0;
    for (int s0 = 0; s0 < n; s0 += 32) {
        const int mine = s0 + lane < n ? (tree_steps(a, s0 + lane, step) + per - 1) / per : 0;
        int sum = mine;  // inclusive, over the lanes
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += x;
        }
        const unsigned who = __ballot_sync(0xffffffffu, s0 + lane < n && part < before + sum);
        if (who) {
            const int l = __ffs(who) - 1;
            return {s0 + l, per, before + __shfl_sync(0xffffffffu, sum - mine, l), __shfl_sync(0xffffffffu, mine, l)};
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    return {-1, per, 0, 0};
}
// By every CTA of a kernel whose parts tree_join_kernel joins.
__device__ __forceinline__ void note_cut(const TreeParams& a, const Cutting& cut) {
    if (a.cuts && threadIdx.x == 0 && blockIdx.y == 0 && int(blockIdx.x) == cut.first) a.cuts[cut.seq] = make_int2(cut.first, cut.parts);
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
// heads of up to 128 dims, a step of a part being a tile of 64 positions.
constexpr int kTcRows = 128, kTcTile = 64;
int syn_tree_attention_tc(const syn::TreeParams& a, int type, cudaStream_t s);
