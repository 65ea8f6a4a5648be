// Attention of a tree of drafted tokens over a KV cache (syn_tree_attention):
// out = softmax(scale q K^T) V over the committed rows and the tree's own rows
// that a token's mask names. n_tree = 1 is one-token decode.
//
// A KV head's work is one matrix product over the rows r = token * G + head of
// its group (G = n_head / n_kv): M = n_tree * G rows against every position,
// so the cache is read once for the whole tree. With many rows (cut_of, and
// head_dim <= 128) tree_attention_tc.cu takes the call; here is the kernel for
// few rows, where the cache's bytes are the bound.
//
// tree_attn_kernel: a CTA takes up to 16 of the M rows and a part of a
// sequence's context. Its four warps take every fourth step of 16 positions,
// each with a ring of its own in shared memory (16-byte asynchronous copies, no
// barrier between the warps), and keep a running maximum, sum and output of
// their own (one pass over K and V); the warps' results are joined at the end.
// The contexts of all sequences are cut into parts of one length, as many as
// fill the GPU whatever the sequences' own lengths; each CTA leaves (max, sum,
// output) in the scratch. With few rows (cut_of) the last of a sequence's CTAs to
// be done joins them, in their order; with more, and always of
// tree_attention_tc.cu's parts, tree_join_kernel does, which starts early and
// waits for the first kernel to end.
//
// Precision: the products run on binary16 tensor-core instructions with float
// accumulators. q is scaled by a power of two per row and split into two
// binary16 terms (22 bits), and so are the probabilities; K and V enter as
// stored. Quantised caches enter as integers (exact in binary16): a score is
// the sum over blocks of scale * (q . quants); for V the block's scale is
// m * 2^e, 2^e <= 2^5 applied to the integers (exact) and m (in [1, 2) unless
// the scale is beyond 2^6) to the float probabilities before they are split, so no
// value is rounded to binary16. Probabilities carry 2^8, and 2^8 m is within binary16
// up to scales of 8188; beyond them a row's output is NaN, and a warp that ends its
// steps with such rows goes through them again with those rows' maximum known and
// raised by 4, for probabilities of up to 2^4 (m < 2^11); the other rows come out the
// same. No append writes such scales, so the steps themselves do not ask for them
// (measured over 17 shapes: 0.8 % more time, against 2 to 3 % with the scales tested at
// every step). Each step's output is added to float registers outside the tensor core,
// whose accumulation truncates: kept there over 64 steps it cost 2e-6.
//
// Up to 8 rows, the usual decode step, the two terms share one product of 16
// rows: the high terms are rows 0-7, the low ones rows 8-15, and their results
// are added. For 16 sequences of 8192 positions, 8 KV heads of 128 and 4 rows
// that takes 60 us in Q8_0, against 92 with a product for each term.
//
// Bound: an F16 cache's bytes (16 sequences of 8192: 76 us, 5.4 TB/s, 83 % of
// the copy rate). A quantised cache's steps: some 600 instructions of a warp per
// 16 positions whatever the bytes' width (170 make binary16 of the bytes, 32 are
// products, the rest adds, splits, scales and addresses), issued in 57 % of the
// schedulers' active cycles, and uneven parts (60 us in Q8_0, 57 % of the copy rate,
// 61 in Q4_0, 30 %). One short sequence: the steps' latencies and the join (4096
// positions: 12.5 us).
#include "tree_attention.cuh"

#include <algorithm>

using namespace syn;

namespace {

constexpr int kWarps = 4;
constexpr int kStep = 16;            // positions per step of a warp
// F16 scores: products summed in the tensor core, which truncates, before a float add. The outputs' error (3000 positions)
// with all of them summed there is 1.4e-6 at 128 dims and 2.0e-6 at 256, with two 5e-7, in the same time.
constexpr int kChain = 2;
constexpr int kMostLen = 0x7fffffff - kMaxTree;  // of max_len: positions rounded up to a tile are still ints
constexpr size_t kCounterBytes = 4096;  // counters of parts that are done, at the start of the scratch
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
// C = A B; then C += A B, m16n8k16: lane = 4 g + t holds A[g | g + 8][2t.. | 2t + 8..], B[2t.. | 2t + 8..][g], C[g | g + 8][2t..].
__device__ __forceinline__ void mma0(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Shared memory of one warp's stage: K rows, V rows (pitches keep the
// fragment reads free of bank conflicts), then the scales of the 16 positions.
template <int TYPE, int HDP>
struct Stage {
    static constexpr int row = TYPE == SYN_F16 ? HDP * 2 : TYPE == SYN_Q8_0 ? HDP : HDP / 2;  // bytes
    static constexpr int k_pitch = row + (TYPE == SYN_Q8_0 ? 32 : 16);
    static constexpr int v_pitch = row + 16;
    static constexpr int nb = HDP / 32;
    static constexpr int scales = TYPE == SYN_F16 ? 0 : kStep * nb * 2 + 16;  // K's (V's alike), from a 16-byte boundary
    static constexpr int v_at = kStep * k_pitch;
    static constexpr int sk_at = v_at + kStep * v_pitch;
    static constexpr int sv_at = sk_at + scales;
    static constexpr int bytes = sv_at + scales;
};

template <int TYPE, int HDP, bool STACK>
struct Plan {
    using S = Stage<TYPE, HDP>;
    static constexpr bool quant = TYPE != SYN_F16;
    static constexpr int R = STACK ? 8 : 16;                         // rows of a CTA
    static constexpr int NR = R / 8;                                 // rows of a lane
    static constexpr int q_pitch = HDP * 2 + 16;
    static constexpr int q_bytes = 2 * R * q_pitch;                  // hi, then lo
    static constexpr int stages = !quant && HDP >= 256 ? 2 : 3;
    static constexpr int scale_bytes = quant ? kStep * (HDP / 32) * 10 : 0;  // a warp's scales as it uses them
    static constexpr int warp_bytes = stages * S::bytes + scale_bytes;
    static constexpr int ring = kWarps * warp_bytes;
    static constexpr int o_pitch = HDP + 4;                          // floats
    static constexpr int join = kWarps * R * (o_pitch + 2) * 4;      // the warps' results, over the ring
    static constexpr int smem = q_bytes + (ring > join ? ring : join) + R * 4;  // + the rows' score factors
    static constexpr int ctas = (STACK || HDP <= 64) && 3 * (smem + 1024) <= 227 * 1024 ? 3 : 2;  // per SM
};

// N floats (a multiple of 2) from shared memory.
template <int N>
__device__ __forceinline__ void load_floats(float (&x)[N], const float* p) {
#pragma unroll
    for (int i = 0; i < N; i += N % 4 ? 2 : 4) {
        if constexpr (N % 4 == 0) {
            const float4 v = *reinterpret_cast<const float4*>(p + i);
            x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
        } else {
            const float2 v = *reinterpret_cast<const float2*>(p + i);
            x[i] = v.x; x[i + 1] = v.y;
        }
    }
}

// Joins a row's parts, in their order, by a warp: row `row` of KV head kvh of sequence seq, whose parts' rows in the
// scratch are `first`, first + pitch, ...; B parts' loads at a time.
template <int B>
__device__ __forceinline__ void join_row(const TreeParams& a, int row, int kvh, int seq, size_t first, size_t pitch, int parts) {
    const int lane = threadIdx.x & 31, hd = a.c.hd;
    const float2* ml = a.part_ml + first;
    const float* o = a.part_o + first * hd;
    const float2 none = make_float2(-INFINITY, 0.0f);
    float2 s = lane < parts ? __ldcg(ml + lane * pitch) : none;
    float top = s.x;
    for (int x = 32 + lane; x < parts; x += 32) top = fmaxf(top, __ldcg(ml + x * pitch).x);
    top = warp_max(top);
    const bool in = 4 * lane < hd, in2 = 128 + 4 * lane < hd;
    float4 acc = make_float4(0, 0, 0, 0), acc2 = acc;
    float sum = 0.0f;
    auto add = [](float4& c, float f, const float4& v) {
        c.x = fmaf(f, v.x, c.x); c.y = fmaf(f, v.y, c.y); c.z = fmaf(f, v.z, c.z); c.w = fmaf(f, v.w, c.w);
    };
    for (int x0 = 0; x0 < parts; x0 += 32) {
        if (x0) s = x0 + lane < parts ? __ldcg(ml + (x0 + lane) * pitch) : none;
        const float w = part_weight(s.x, s.y, top);
        sum += warp_sum(w * s.y);
        const int n = min(32, parts - x0);
        auto half = [&](float4& c, int at, bool here) {
            for (int i0 = 0; i0 < n; i0 += B) {
                float4 v[B];
#pragma unroll
                for (int i = 0; i < B; ++i) {
                    v[i] = make_float4(0, 0, 0, 0);
                    if (i0 + i < n && here) v[i] = __ldcg(reinterpret_cast<const float4*>(o + (x0 + i0 + i) * pitch * hd) + at);
                }
#pragma unroll
                for (int i = 0; i < B; ++i) {
                    const float f = __shfl_sync(0xffffffffu, w, (i0 + i) & 31);
                    if (i0 + i < n) add(c, f, v[i]);
                }
            }
        };
        half(acc, lane, in);
        if (hd > 128) half(acc2, 32 + lane, in2);
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int tk = row / a.group, h = kvh * a.group + row - tk * a.group;
    float4* out = reinterpret_cast<float4*>(a.out + ((size_t(seq) * a.n_tree + tk) * a.n_head + h) * hd);
    if (in) out[lane] = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    if (in2) out[32 + lane] = make_float4(acc2.x * inv, acc2.y * inv, acc2.z * inv, acc2.w * inv);
}

template <int TYPE, int HDP, bool STACK>
__global__ void __launch_bounds__(kWarps * 32, Plan<TYPE, HDP, STACK>::ctas) tree_attn_kernel(const TreeParams a) {
    using S = Stage<TYPE, HDP>;
    using P = Plan<TYPE, HDP, STACK>;
    constexpr int R = P::R, NR = P::NR, KS = HDP / 16, NB = HDP / 32;
    constexpr bool kQuant = P::quant;
    constexpr bool kQReg = HDP <= 128;  // the q fragments stay in registers
    constexpr int QT = STACK ? 1 : 2;   // q fragments of a k step: both terms, or one each
    extern __shared__ __align__(128) unsigned char smem[];
    unsigned char* ring = smem + P::q_bytes;
    float* row_scale = reinterpret_cast<float*>(smem + P::smem - R * 4);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int hd = a.c.hd;
    const int kvh = blockIdx.y / a.row_blocks, rb = blockIdx.y - kvh * a.row_blocks;
    const int row0 = rb * R, rows = min(R, a.rows - row0);

    pdl_launch_dependents();
    pdl_wait();
    const Cutting cut = tree_cutting(a, kStep, blockIdx.x);
    const int seq = cut.seq;
    if (seq < 0) return;
    note_cut(a, cut);
    const int len = tree_len(a, seq), total = len + a.n_tree;
    const int steps = (total + kStep - 1) / kStep;
    const int s0 = (int(blockIdx.x) - cut.first) * cut.per, s1 = cut.per < steps - s0 ? s0 + cut.per : steps;

    // --- the ring -------------------------------------------------------------
    const int nb = hd / 32;  // blocks of a row (quantised)
    const char *kbase = a.c.k + size_t(seq) * a.c.seq_stride, *vbase = a.c.v + size_t(seq) * a.c.seq_stride;
    // a position's K (V) row of this head, and the bytes between positions
    const int row_bytes = TYPE == SYN_F16 ? hd * 2 : TYPE == SYN_Q8_0 ? hd : hd / 2;
    const size_t pos_pitch = TYPE == SYN_F16 ? size_t(a.c.n_kv) * hd * 2 : size_t(row_bytes);
    const size_t head_at = TYPE == SYN_F16 ? size_t(kvh) * hd * 2 : size_t(kvh) * a.c.max_ctx * row_bytes;
    const size_t scale_at = a.c.scale_plane + size_t(kvh) * a.c.max_ctx * nb * 2;
    const int scale_off = kQuant ? int(scale_at & 15) : 0;  // the same for every step: 16 positions are 32 nb bytes
    unsigned char* my_ring = ring + warp * P::warp_bytes;
    const uint32_t ring_s = smem_addr(my_ring);
    const int chunks = row_bytes / 16;
    constexpr int CP = S::row / 16;  // chunks of a full row
    const size_t lane_at = head_at + size_t(lane / CP) * pos_pitch + (lane % CP) * 16;
    const uint32_t lane_k = (lane / CP) * S::k_pitch + (lane % CP) * 16, lane_v = S::v_at + (lane / CP) * S::v_pitch + (lane % CP) * 16;
    auto load = [&](int step, int stage) {
        const uint32_t st = ring_s + stage * S::bytes;
        const int p0 = step * kStep;
        constexpr int rows_at_once = 32 / CP;
        const char *kp = kbase + lane_at + size_t(p0) * pos_pitch, *vp = vbase + lane_at + size_t(p0) * pos_pitch;
        if (hd == HDP && p0 + kStep <= total) {
#pragma unroll
            for (int i = 0; i < kStep / rows_at_once; ++i) {
                cp16(st + lane_k + i * rows_at_once * S::k_pitch, kp + i * rows_at_once * pos_pitch);
                cp16(st + lane_v + i * rows_at_once * S::v_pitch, vp + i * rows_at_once * pos_pitch);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kStep / rows_at_once; ++i) {
                const bool in = p0 + i * rows_at_once + lane / CP < total;
                const size_t at = in ? size_t(i) * rows_at_once * pos_pitch : 0;
                if (lane % CP < chunks) {
                    cp16(st + lane_k + i * rows_at_once * S::k_pitch, in ? kp + at : kbase, in);
                    cp16(st + lane_v + i * rows_at_once * S::v_pitch, in ? vp + at : vbase, in);
                }
            }
        }
        if (kQuant) {
            // the run of scales from its 16-byte boundary; the last chunk holds at least one of its bytes
            const int last = min(p0 + kStep, a.c.max_ctx);
            const size_t at = (scale_at + size_t(p0) * nb * 2) & ~size_t(15);
            const int n = (scale_off + (last - p0) * nb * 2 + 15) / 16;
            constexpr int most = S::scales / 16;
            const int which = lane / 16, c = lane % 16;
            const char* from = (which ? vbase : kbase) + at + c * 16;
            const uint32_t to = st + (which ? S::sv_at : S::sk_at) + c * 16;
            if (c < n) cp16(to, from);
            if (most > 16 && c + 16 < n) cp16(to + 256, from + 256);
        }
    };
    // q's rows are on their way before the tiles are
    float qx[R / kWarps][NB];
#pragma unroll
    for (int i = 0; i < R / kWarps; ++i) {
        const int r = i * kWarps + warp, row = row0 + r, qt = row / a.group, h = row - qt * a.group;
        const float* src = a.q + (size_t(seq) * a.n_tree + qt) * a.q_stride + size_t(kvh * a.group + h) * hd + lane;
#pragma unroll
        for (int b = 0; b < NB; ++b) qx[i][b] = r < rows && 32 * b + lane < hd ? __ldg(src + 32 * b) : 0.0f;
    }
    if (hd != HDP) {  // dims past the head stay zero
        for (int i = tid; i < P::ring / 16; i += kWarps * 32) reinterpret_cast<uint4*>(ring)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }
    int next;  // the next step to request
    auto request_first = [&] {
        next = s0 + warp;
#pragma unroll
        for (int i = 0; i < P::stages - 1; ++i) {
            if (next < s1) load(next, i);
            cp_commit();
            next += kWarps;
        }
    };
    request_first();

    // --- q: scaled to a row maximum in [2^8, 2^9), split, in the order of the K fragments -------
#pragma unroll
    for (int i = 0; i < R / kWarps; ++i) {
        const int r = i * kWarps + warp;
        float(&x)[NB] = qx[i];
        float m = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) m = fmaxf(m, fabsf(x[b]));
        float up, down;
        q_factor(warp_max(m), up, down);
        if (lane == 0) row_scale[r] = a.scale_log2 * down;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            // the k index of dim `lane` of the block in its two products of 16
            int s = lane >> 4, k = lane & 15;
            if (TYPE == SYN_Q8_0) {  // dim = 8 t + 4 s + e, e = 0..3: k = 2 t + (e & 1) + 8 (e >> 1)
                s = (lane >> 2) & 1;
                k = 2 * (lane >> 3) + (lane & 1) + 8 * ((lane >> 1) & 1);
            } else if (TYPE == SYN_Q4_0) {  // dim = 16 s + 4 t + e
                k = 2 * ((lane >> 2) & 3) + (lane & 1) + 8 * ((lane >> 1) & 1);
            }
            const float y = x[b] * up;
            const __half hi = __float2half_rn(y);
            const __half lo = __float2half_rn(y - __half2float(hi));
            unsigned char* at = smem + r * P::q_pitch + (32 * b + 16 * s + k) * 2;
            *reinterpret_cast<__half*>(at) = hi;
            *reinterpret_cast<__half*>(at + R * P::q_pitch) = lo;
        }
    }
    __syncthreads();

    // fragments of 16 rows: all high terms (with the low ones 16 rows on), or 8 high and 8 low
    const uint32_t q_s = smem_addr(smem) + (lane & 15) * P::q_pitch + (lane >> 4) * 16;
    uint32_t qf[kQReg ? KS : 1][QT][4];
    if (kQReg)
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int x = 0; x < QT; ++x) ldsm4(qf[k][x], q_s + x * 16 * P::q_pitch + k * 32);
    float rs[NR], m[NR], l[NR], o[HDP / 8][2 * NR];
    int tok[NR];
#pragma unroll
    for (int u = 0; u < NR; ++u) {
        rs[u] = row_scale[8 * u + g];
        tok[u] = (row0 + 8 * u + g) / a.group;
        m[u] = -INFINITY;
    }
    bool again = false;

    // --- the steps of this warp ----------------------------------------------------
[[maybe_unused]] pass:
#pragma unroll
    for (int u = 0; u < NR; ++u) l[u] = 0.0f;
#pragma unroll
    for (int n = 0; n < HDP / 8; ++n)
#pragma unroll
        for (int e = 0; e < 2 * NR; ++e) o[n][e] = 0.0f;
    int stage = 0;
    for (int step = s0 + warp; step < s1; step += kWarps) {
        cp_wait<P::stages - 2>();
        __syncwarp();
        {
            int to = stage + P::stages - 1;
            if (to >= P::stages) to -= P::stages;
            if (next < s1) load(next, to);
            cp_commit();
            next += kWarps;
        }
        unsigned char* st = my_ring + stage * S::bytes;
        const uint32_t st_s = ring_s + stage * S::bytes;
        const int p0 = step * kStep;

        // this step's scales as the lanes use them: K's, and V's as m (float) and 2^e (binary16)
        float* kds = reinterpret_cast<float*>(my_ring + P::stages * S::bytes);  // [16][NB]
        float* vms = kds + kStep * NB;                                          // [16][NB]
        uint16_t* ves = reinterpret_cast<uint16_t*>(vms + kStep * NB);          // [8 pairs][NB][2]
        if constexpr (kQuant) {
#pragma unroll
            for (int i = 0; i < kStep * NB / 32; ++i) {
                const int id = i * 32 + lane, r = id / NB, b = id % NB;
                // a position past the context has scales of 0; one with a scale that is not finite scores NaN (rows
                // that do not see it mask that): of K by an infinity times 0
                const bool ok = p0 + r < total && b < nb;
                const uint32_t dk = ok ? reinterpret_cast<const uint16_t*>(st + S::sk_at + scale_off)[r * nb + b] : 0u;
                const uint32_t dv = ok ? reinterpret_cast<const uint16_t*>(st + S::sv_at + scale_off)[r * nb + b] : 0u;
                const bool finite = (dv & 0x7c00u) != 0x7c00u;
                const uint32_t pow = finite ? min(max(dv & 0x7c00u, 0x0400u), 0x5000u) : 0x0400u;  // 2^-14 .. 2^5: 1152 * 2^5 is finite
                const float inv = __uint_as_float(0x7f000000u - __float_as_uint(f16_from_bits(uint16_t(pow))));
                const float kd = f16_from_bits(uint16_t(dk));
                kds[id] = finite ? __fmaf_rn(kd, 0.0f, kd) : __uint_as_float(0x7fffffffu);
                vms[id] = finite ? f16_from_bits(uint16_t(dv)) * inv : 0.0f;
                ves[((r >> 1) * NB + b) * 2 + (r & 1)] = uint16_t(pow);
            }
            __syncwarp();
        }

        // scores of 16 positions: n-tile u holds positions p0 + 8 u + {2t, 2t + 1}, for NR rows each
        float s[2][2 * NR];
        auto products = [&](float (&c)[2][4], int k, const uint32_t (&b)[2][2], bool first) {
            uint32_t f[QT][4];
            if (!kQReg)
#pragma unroll
                for (int x = 0; x < QT; ++x) ldsm4(f[x], q_s + x * 16 * P::q_pitch + k * 32);
#pragma unroll
            for (int x = 0; x < QT; ++x)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    if (first && x == 0) mma0(c[u], kQReg ? qf[kQReg ? k : 0][x] : f[x], b[u][0], b[u][1]);
                    else mma(c[u], kQReg ? qf[kQReg ? k : 0][x] : f[x], b[u][0], b[u][1]);
                }
        };
        if constexpr (!kQuant) {
            float c[2][4];
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t x[4];  // (n-tile 0: b0, b1), (n-tile 1: b0, b1)
                ldsm4(x, st_s + ((lane & 7) + ((lane >> 4) << 3)) * S::k_pitch + k * 32 + ((lane >> 3) & 1) * 16);
                const uint32_t b[2][2] = {{x[0], x[1]}, {x[2], x[3]}};
                products(c, k, b, k % kChain == 0);
                if (k % kChain == kChain - 1 || k == KS - 1)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        if (STACK) add2(c[u][0], c[u][1], c[u][2], c[u][3]);
#pragma unroll
                        for (int e = 0; e < 2 * NR; e += 2) {
                            if (k < kChain) {
                                s[u][e] = c[u][e];
                                s[u][e + 1] = c[u][e + 1];
                            } else {
                                add2(s[u][e], s[u][e + 1], c[u][e], c[u][e + 1]);
                            }
                        }
                    }
            }
        } else {
            float kd[4][NB];  // of positions 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
            for (int j = 0; j < 4; ++j) load_floats(kd[j], kds + (2 * t + (j & 1) + 8 * (j >> 1)) * NB);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float c[2][4];
                uint32_t w[2][2];  // [n-tile][product of 16 dims]: four quants as bytes
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const unsigned char* at = st + (8 * u + g) * S::k_pitch;
                    if (TYPE == SYN_Q8_0) {
                        const uint2 x = *reinterpret_cast<const uint2*>(at + 32 * b + 8 * t);
                        w[u][0] = x.x ^ 0x80808080u;
                        w[u][1] = x.y ^ 0x80808080u;
                    } else {
                        const uint32_t x = *reinterpret_cast<const uint32_t*>(at + 16 * b + 4 * t);
                        w[u][0] = x & 0x0f0f0f0fu;
                        w[u][1] = (x >> 4) & 0x0f0f0f0fu;
                    }
                }
                const __half2 zero = half2_of(TYPE == SYN_Q8_0 ? 0x64806480u : 0x64086408u);  // 1024 + 128 | 8
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t bb[2][2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        bb[u][0] = bits(__hsub2(bytes_h2(w[u][h], 0x4140), zero));
                        bb[u][1] = bits(__hsub2(bytes_h2(w[u][h], 0x4342), zero));
                    }
                    products(c, 2 * b + h, bb, h == 0);
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float d0 = kd[2 * u][b], d1 = kd[2 * u + 1][b];
                    if (STACK) add2(c[u][0], c[u][1], c[u][2], c[u][3]);
#pragma unroll
                    for (int e = 0; e < 2 * NR; e += 2) {
                        if (b == 0) {
                            s[u][e] = c[u][e] * d0;
                            s[u][e + 1] = c[u][e + 1] * d1;
                        } else {
                            fma2_to(s[u][e], s[u][e + 1], c[u][e], c[u][e + 1], d0, d1);
                        }
                    }
                }
            }
        }

        // an infinity in K may score -inf, which would drop its row in silence: NaN
        if (!kQuant)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 2 * NR; e += 2) fma2(s[u][e], s[u][e + 1], 0.0f, 0.0f, s[u][e], s[u][e + 1]);

        // the tree's own rows: what a token does not see scores -inf
        const bool edge = p0 + kStep > len;
        if (!kQuant && edge) {
            // V rows of the tree may hold values that are not finite where some token does not see them:
            // zeroed here (0 * inf is NaN), and the position scores NaN for the tokens that do see it
            unsigned bad = 0;
            const int r = lane & 15;
            if (p0 + r >= len && p0 + r < total) {
                for (int c = lane >> 4; c < row_bytes / 16; c += 2) {
                    uint16_t* x = reinterpret_cast<uint16_t*>(st + S::v_at + r * S::v_pitch + c * 16);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if ((x[e] & 0x7c00u) == 0x7c00u) {
                            x[e] = 0;
                            bad = 1;
                        }
                }
            }
            unsigned flags = __ballot_sync(0xffffffffu, bad);
            flags = (flags | flags >> 16) & 0xffffu;
            __syncwarp();
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 2 * NR; ++e)
                    if (flags >> (8 * u + 2 * t + (e & 1)) & 1u) s[u][e] = __uint_as_float(0x7fffffffu);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 2 * NR; ++e) s[u][e] *= rs[e >> 1];
        if (edge) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 2 * NR; ++e) {
                    const int j = p0 + 8 * u + 2 * t + (e & 1) - len;
                    const bool sees = j < 0 || tree_sees(a, seq, tok[e >> 1], j);
                    if (!sees) s[u][e] = -INFINITY;
                }
        }

        // running maximum, probabilities, sum
        float p[2][2 * NR], mn[NR];
        bool grows = false;
#pragma unroll
        for (int u = 0; u < NR; ++u) {
            float x = fmaxf(fmaxf(s[0][2 * u], s[0][2 * u + 1]), fmaxf(s[1][2 * u], s[1][2 * u + 1]));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
            mn[u] = fmaxf(m[u], x);
            grows |= mn[u] > m[u];
        }
        if (__any_sync(0xffffffffu, grows)) {
            float f[NR];
#pragma unroll
            for (int u = 0; u < NR; ++u) {
                f[u] = mn[u] > m[u] ? ex2(m[u] - mn[u]) : 1.0f;  // m = -inf: 0
                m[u] = mn[u];
                l[u] *= f[u];
            }
#pragma unroll
            for (int n = 0; n < HDP / 8; ++n)
#pragma unroll
                for (int e = 0; e < 2 * NR; ++e) o[n][e] *= f[e >> 1];
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 2 * NR; ++e) {
                const float mm = m[e >> 1];
                p[u][e] = ex2(s[u][e] - (mm == -INFINITY ? 0.0f : mm) + kPShift);
                l[e >> 1] += p[u][e];
            }

        // out += p V: the A fragments of the probabilities times four factors (one for each position of a lane)
        uint32_t pf[QT][4];
        auto split_p = [&](const float (&f)[4]) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 2 * NR; e += 2) {
                    float x = p[u][e], y = p[u][e + 1];
                    mul2(x, y, f[2 * u], f[2 * u + 1]);
                    if (STACK) split2(x, y, pf[0][2 * u], pf[0][2 * u + 1]);
                    else split2(x, y, pf[0][2 * u + e / 2], pf[QT - 1][2 * u + e / 2]);
                }
        };
        auto output = [&](float (&acc)[2 * NR], uint32_t b0, uint32_t b1) {
            float c[4];
            mma0(c, pf[0], b0, b1);
            if (!STACK) mma(c, pf[QT - 1], b0, b1);
            if (STACK) add2(c[0], c[1], c[2], c[3]);
            add2(acc[0], acc[1], c[0], c[1]);
            if (!STACK) add2(acc[2 * NR - 2], acc[2 * NR - 1], c[2], c[3]);
        };
        if constexpr (!kQuant) {
            split_p({1.0f, 1.0f, 1.0f, 1.0f});
#pragma unroll
            for (int n = 0; n < HDP / 16; ++n) {
                uint32_t b[4];
                ldsm4t(b, st_s + S::v_at + ((lane & 7) + ((lane >> 3) & 1) * 8) * S::v_pitch + n * 32 + (lane >> 4) * 16);
                output(o[2 * n], b[0], b[1]);
                output(o[2 * n + 1], b[2], b[3]);
            }
        } else {
            float vm[4][NB];
#pragma unroll
            for (int j = 0; j < 4; ++j) load_floats(vm[j], vms + (2 * t + (j & 1) + 8 * (j >> 1)) * NB);
            float ve[2][NB];  // binary16 pairs of positions 2t, 2t + 1 | 2t + 8, 2t + 9
#pragma unroll
            for (int j = 0; j < 2; ++j) load_floats(ve[j], reinterpret_cast<const float*>(ves) + (t + 4 * j) * NB);
            uint32_t r4[4];  // a block's bytes of 2 positions x 2 dims: (positions 0-7, 8-15) x (dims 0-15, 16-31)
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (TYPE == SYN_Q8_0)
                    ldsm4t(r4, st_s + S::v_at + ((lane & 7) + ((lane >> 3) & 1) * 8) * S::v_pitch + b * 32 + (lane >> 4) * 16);
                else if ((b & 1) == 0)  // two blocks of 16 bytes
                    ldsm4t(r4, st_s + S::v_at + ((lane & 7) + ((lane >> 3) & 1) * 8) * S::v_pitch + b * 16 + (lane >> 4) * 16);
                split_p({vm[0][b], vm[1][b], vm[2][b], vm[3][b]});
                const __half2 zero = half2_of(TYPE == SYN_Q8_0 ? 0xe480e480u : 0xe408e408u);
                const __half2 e0 = half2_of(__float_as_uint(ve[0][b])), e1 = half2_of(__float_as_uint(ve[1][b]));
                const __half2 z0 = __hmul2(zero, e0), z1 = __hmul2(zero, e1);  // -1152 * 2^e | -1032 * 2^e
                // n-tile 4 b + 2 half + odd: dims 32 b + 16 half + 2 n + odd
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t x0, x1;  // positions 2t, 2t + 1 | 2t + 8, 2t + 9: bytes (even, odd, even, odd)
                    if (TYPE == SYN_Q8_0) {
                        x0 = r4[2 * half] ^ 0x80808080u;
                        x1 = r4[2 * half + 1] ^ 0x80808080u;
                    } else {
                        x0 = (r4[2 * (b & 1)] >> (4 * half)) & 0x0f0f0f0fu;
                        x1 = (r4[2 * (b & 1) + 1] >> (4 * half)) & 0x0f0f0f0fu;
                    }
#pragma unroll
                    for (int odd = 0; odd < 2; ++odd) {
                        const uint32_t sel = odd ? 0x4341u : 0x4240u;
                        output(o[4 * b + 2 * half + odd], bits(__hfma2(bytes_h2(x0, sel), e0, z0)),
                               bits(__hfma2(bytes_h2(x1, sel), e1, z1)));
                    }
                }
            }
        }
        __syncwarp();
        if (++stage == P::stages) stage = 0;
    }
    cp_wait<0>();
    if constexpr (kQuant) {
        if (!again) {  // NaN in a row, in all dims of a block: a scale above 8188, or values that are not finite
            unsigned who[NR], any = 0;
#pragma unroll
            for (int u = 0; u < NR; ++u) {
                bool nan = false;
#pragma unroll
                for (int b = 0; b < NB; ++b) nan |= o[4 * b][2 * u] != o[4 * b][2 * u];
                who[u] = __ballot_sync(0xffffffffu, nan);
                any |= who[u];
            }
            if (any) {  // the other rows come out as before; a maximum to which 4 adds nothing goes up to the next float
#pragma unroll
                for (int u = 0; u < NR; ++u)
                    m[u] = who[u] >> (lane & 28) & 15u ? m[u] + fmaxf(4.0f, fabsf(m[u]) * 0x1p-23f) : -INFINITY;
                again = true;
                request_first();
                goto pass;
            }
        }
    }
    __syncthreads();  // every warp is done with the ring

    // --- the warps' results joined --------------------------------------------------
    float* jo = reinterpret_cast<float*>(ring);       // [kWarps][R][o_pitch]
    float* jm = jo + kWarps * R * P::o_pitch;          // [kWarps][R]
    float* jl = jm + kWarps * R;
#pragma unroll
    for (int u = 0; u < NR; ++u) {
        float sum = l[u];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        const int r = 8 * u + g;
        if (t == 0) {
            jm[warp * R + r] = m[u];
            jl[warp * R + r] = sum;
        }
        float* at = jo + (warp * R + r) * P::o_pitch;
        if constexpr (!kQuant) {
#pragma unroll
            for (int n = 0; n < HDP / 8; ++n)
                *reinterpret_cast<float2*>(at + 8 * n + 2 * t) = make_float2(o[n][2 * u], o[n][2 * u + 1]);
        } else {
#pragma unroll
            for (int n = 0; n < HDP / 16; ++n)  // (even, odd) n-tiles hold dims 4t, 4t + 2 and 4t + 1, 4t + 3
                *reinterpret_cast<float4*>(at + 16 * n + 4 * t) =
                    make_float4(o[2 * n][2 * u], o[2 * n + 1][2 * u], o[2 * n][2 * u + 1], o[2 * n + 1][2 * u + 1]);
        }
    }
    __syncthreads();
    const size_t part = (size_t(blockIdx.x) * gridDim.y + blockIdx.y) * R;
    for (int r = warp; r < rows; r += kWarps) {
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, jm[w * R + r]);
        float f[kWarps], sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            f[w] = part_weight(jm[w * R + r], jl[w * R + r], mx);
            sum += f[w] * jl[w * R + r];
        }
        const int row = row0 + r, tk = row / a.group, h = kvh * a.group + row - tk * a.group;
        const bool whole = a.parts == 0;
        float* out = whole ? a.out + ((size_t(seq) * a.n_tree + tk) * a.n_head + h) * hd : a.part_o + (part + r) * hd;
        const float inv = !whole ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
        for (int d = lane; d < hd; d += 32) {
            float acc = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) acc += f[w] * jo[(w * R + r) * P::o_pitch + d];
            out[d] = acc * inv;
        }
        if (!whole && lane == 0) a.part_ml[part + r] = make_float2(mx, sum);
    }
    if (!a.arrived) return;

    // --- the last of the sequence's parts to be done joins them ----------------------------
    __threadfence();
    __syncthreads();
    __shared__ bool last;
    if (tid == 0) {
        unsigned* arrived = a.arrived + size_t(seq) * gridDim.y + blockIdx.y;
        last = atomicAdd(arrived, 1u) == unsigned(cut.parts - 1);
        if (last) *arrived = 0;  // ready for the next call
        __threadfence();
    }
    __syncthreads();
    if (!last) return;
    const size_t first = (size_t(cut.first) * gridDim.y + blockIdx.y) * R;
    for (int r = warp; r < rows; r += kWarps) join_row<16>(a, row0 + r, kvh, seq, first + r, size_t(gridDim.y) * R, cut.parts);
}

// Joins the sequences' parts: a warp per row (token, head), whose cutting the first kernel has left in the scratch. The
// few-row kernel's parts are many, 32 at a time (16 rows of 8192 in Q8_0 18.0 us, against 19.5 with 16); of the other
// kernel there are few parts and many rows, and more registers mean fewer warps on an SM (16 sequences of 1000, 64 rows,
// F16: 33 us with 8 at a time, 36 with 16, 56 with 32 and the cutting found again by every warp).
template <int B>
__global__ void __launch_bounds__(128) tree_join_kernel(const TreeParams a, int R) {
    pdl_wait();
    const unsigned id = blockIdx.x * 4 + (threadIdx.x >> 5), per_seq = unsigned(a.c.n_kv) * a.rows;
    if (id >= unsigned(a.c.n_seq) * per_seq) return;
    const int seq = int(id / per_seq), row = int(id % per_seq) % a.rows, kvh = int(id % per_seq) / a.rows, rb = row / R;
    const int2 cut = __ldcg(a.cuts + seq);
    const size_t unit = size_t(a.c.n_kv) * a.row_blocks;
    join_row<B>(a, row, kvh, seq, (cut.x * unit + size_t(kvh) * a.row_blocks + rb) * R + row - rb * R, unit * R, cut.y);
}

// How a call is cut: rows of a CTA, CTAs over the rows, parts of the contexts
// (0: a part is a sequence).
struct Cut {
    bool tc, join;  // on tcgen05; parts joined by tree_join_kernel
    int R, row_blocks, parts;
    size_t rows;  // of all parts in the scratch
};
// CTAs of the few-row kernel on an SM (heads of more than 128 dims in F16 and Q8_0: shared memory lets one on it, and the
// parts take two waves).
template <int TYPE>
constexpr int slots(int hd, bool stack) {
    return hd <= 64    ? (stack ? Plan<TYPE, 64, true>::ctas : Plan<TYPE, 64, false>::ctas)
           : hd <= 128 ? (stack ? Plan<TYPE, 128, true>::ctas : Plan<TYPE, 128, false>::ctas)
                       : (stack ? Plan<TYPE, 256, true>::ctas : Plan<TYPE, 256, false>::ctas);
}
// More than 16 rows (32 of a quantised cache, whose tiles the tcgen05 kernel has to convert) go to tree_attention_tc.cu.
// Measured for 16 sequences of 8192 positions and 8 KV heads of 128, this kernel / that one, us: F16 16 rows 97 / 136, 20
// rows 145 / 136, 64 rows 247 / 149; Q8_0 32 rows 201 / 254, 48 rows 317 / 265; Q4_0 202 / 230, 311 / 236. For one
// sequence of 32768: F16 20 rows 45 / 42; Q8_0 32 rows 57 / 69, 48 rows 77 / 70.
Cut cut_of(int type, int n_seq, int n_tree, int n_head, int n_kv, int head_dim, int max_len) {
    Cut c;
    const int rows = n_tree * (n_head / n_kv);
    const size_t sms = size_t(syn_num_sms());
    c.tc = rows > (type == SYN_F16 ? 16 : 32) && head_dim <= 128;
    c.R = c.tc ? kTcRows : rows <= 8 ? 8 : 16;
    c.row_blocks = (rows + c.R - 1) / c.R;
    const size_t units = size_t(n_kv) * c.row_blocks;  // CTAs of a part
    if (c.tc) {
        // one CTA per SM: the parts whose last wave ends first
        const size_t tiles = size_t(max_len + kTcTile - 1) / kTcTile * n_seq;
        size_t best = ~size_t(0);
        c.parts = 0;
        for (size_t n = n_seq; n <= std::min(tiles, size_t(n_seq) * 128); ++n) {
            const size_t waves = (units * n + sms - 1) / sms, per = (tiles + n - 1) / n;
            const size_t cost = waves * (per + 8);  // a CTA's start and end take about 8 tiles
            if (waves > 4 && n > size_t(n_seq)) break;
            if (cost < best) {
                best = cost;
                c.parts = int(n);
            }
        }
    } else {
        // one wave of CTAs (two to four waves of shorter parts took 4 to 10 % more).
        // A part has two steps of every warp, or one while there are no more than the 16 parts that a join loads at a
        // time (one sequence of 1000: 7.9 -> 7.2 us; of 2000, with 32 parts, 8.0 -> 8.9).
        const bool stack = c.R == 8;
        const int per_sm = type == SYN_F16    ? slots<SYN_F16>(head_dim, stack)
                           : type == SYN_Q8_0 ? slots<SYN_Q8_0>(head_dim, stack)
                                              : slots<SYN_Q4_0>(head_dim, stack);
        const size_t turns = size_t(max_len + kWarps * kStep - 1) / (kWarps * kStep);  // steps of each warp
        const size_t most = std::max((turns + 1) / 2, std::min<size_t>(turns, 16)) * n_seq;
        c.parts = int(std::min(per_sm * sms / units, most));
    }
    if (c.parts <= n_seq) c.parts = 0;
    // The last CTA has a row a warp to join, or two of a few parts, in less time than a launch; with more it has them
    // one after another. Measured for one sequence of 8192, last CTA / kernel, us: 4 rows (of 4096) 10.8 / 11.7, 8 rows
    // 18.3 / 16.2, 16 rows 27.0 / 18.4; 4 sequences of 8192, 8 rows 27.5 / 28.4, 16 rows 33.2 / 31.5.
    c.join = c.parts && (c.tc || rows > 8 || (rows > 4 && c.parts > 16 * n_seq) || units * n_seq * sizeof(unsigned) > kCounterBytes);
    c.rows = size_t(c.parts) * units * c.R;
    return c;
}

template <int TYPE, int HDP, bool STACK>
int launch(const TreeParams& a, cudaStream_t s) {
    auto kernel = tree_attn_kernel<TYPE, HDP, STACK>;
    constexpr int smem = Plan<TYPE, HDP, STACK>::smem;
    static_assert(smem <= 227 * 1024, "shared memory of a CTA");
    const int st = syn_opt_in_smem(reinterpret_cast<const void*>(kernel), smem);
    if (st) return st;
    const dim3 grid{unsigned(a.parts ? a.parts : a.c.n_seq), unsigned(a.c.n_kv * a.row_blocks), 1};
    return syn_launch(kernel, grid, kWarps * 32, smem, s, a);
}

template <int TYPE>
int launch_type(const TreeParams& a, const Cut& c, cudaStream_t s) {
    if (a.c.hd <= 64) return c.R == 8 ? launch<TYPE, 64, true>(a, s) : launch<TYPE, 64, false>(a, s);
    if (a.c.hd <= 128) return c.R == 8 ? launch<TYPE, 128, true>(a, s) : launch<TYPE, 128, false>(a, s);
    return c.R == 8 ? launch<TYPE, 256, true>(a, s) : launch<TYPE, 256, false>(a, s);
}

}  // namespace

extern "C" size_t syn_tree_attention_scratch_bytes(int n_seq, int n_tree, int n_head, int n_kv, int head_dim,
                                                   int max_len) {
    if (n_seq <= 0 || n_tree <= 0 || n_tree > kMaxTree || n_kv <= 0 || n_head <= 0 || n_head % n_kv || head_dim <= 0 ||
        head_dim > 256 || max_len < n_tree || max_len > kMostLen)
        return 0;
    size_t rows = 0;  // the most of any type
    for (int type : {SYN_F16, SYN_Q8_0, SYN_Q4_0})
        rows = std::max(rows, cut_of(type, n_seq, n_tree, n_head, n_kv, head_dim, max_len).rows);
    return kCounterBytes + align256(size_t(n_seq) * 8) + align256(rows * 8) + align256(rows * head_dim * 4);
}

extern "C" int syn_tree_attention(const syn_kv_cache* c, int layer, const syn_tree_attention_args* x, void* stream) {
    int st = kv_check(c, layer);
    if (st) return st;
    if (!x || !x->q || !x->out || !x->len || !x->scratch) return SYN_ERR_INVALID;
    if (x->n_head <= 0 || x->n_head % c->n_kv || x->n_tree <= 0) return SYN_ERR_INVALID;
    if (x->max_len < x->n_tree || x->max_len > c->max_ctx) return SYN_ERR_INVALID;
    if (x->n_tree > kMaxTree || c->n_seq > 65535 || x->max_len > kMostLen) return SYN_ERR_UNSUPPORTED;
    const size_t q_row = size_t(x->n_head) * c->head_dim;
    if (x->q_stride && x->q_stride < q_row) return SYN_ERR_INVALID;
    if ((reinterpret_cast<uintptr_t>(x->scratch) | reinterpret_cast<uintptr_t>(x->out)) & 15) return SYN_ERR_INVALID;
    const Cut cut = cut_of(c->type, c->n_seq, x->n_tree, x->n_head, c->n_kv, c->head_dim, x->max_len);
    if (size_t(c->n_kv) * cut.row_blocks > 65535) return SYN_ERR_UNSUPPORTED;
    TreeParams a{};
    a.c = kv_view(c, layer);
    a.q = x->q; a.out = x->out; a.len = x->len; a.mask = x->mask;
    char* scratch = static_cast<char*>(x->scratch);
    a.arrived = cut.parts && !cut.join ? reinterpret_cast<unsigned*>(scratch) : nullptr;
    a.cuts = cut.join ? reinterpret_cast<int2*>(scratch + kCounterBytes) : nullptr;
    scratch += kCounterBytes + align256(size_t(c->n_seq) * 8);
    a.part_ml = reinterpret_cast<float2*>(scratch);
    a.part_o = reinterpret_cast<float*>(scratch + align256(cut.rows * 8));
    a.q_stride = x->q_stride ? x->q_stride : q_row;
    a.n_tree = x->n_tree; a.n_head = x->n_head;
    a.group = x->n_head / c->n_kv;
    a.rows = x->n_tree * a.group;
    a.row_blocks = cut.row_blocks;
    a.max_len = x->max_len;
    a.mask_words = (x->n_tree + 31) / 32;
    a.parts = cut.parts;
    a.scale_log2 = x->scale * 1.4426950408889634f;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (cut.tc) st = syn_tree_attention_tc(a, c->type, s);
    else if (c->type == SYN_F16) st = launch_type<SYN_F16>(a, cut, s);
    else if (c->type == SYN_Q8_0) st = launch_type<SYN_Q8_0>(a, cut, s);
    else st = launch_type<SYN_Q4_0>(a, cut, s);
    if (st || !cut.join) return st;
    const size_t rows = size_t(c->n_seq) * c->n_kv * a.rows;
    if (cut.tc) return syn_launch_pdl(true, tree_join_kernel<8>, unsigned((rows + 3) / 4), 128, 0, s, a, cut.R);
    return syn_launch_pdl(true, tree_join_kernel<32>, unsigned((rows + 3) / 4), 128, 0, s, a, cut.R);
}
