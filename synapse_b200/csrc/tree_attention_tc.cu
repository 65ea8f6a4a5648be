// syn_tree_attention on tcgen05: a CTA takes 128 rows (token * G + head) of a
// KV head and a run of the context in tiles of 64 positions.
//
// For a tile, S = Q K^T (128 x 64) and O = P V (128 x head_dim) are products
// with the A operand in tensor memory (Q for the whole call; P where S was)
// and the tile in shared memory. As in the other kernel q and the
// probabilities are two binary16 terms each, so S takes two products and O
// two; a quantised tile is also two terms (its scales times its integers: 18
// bits), so S and O take three (the product of the two low terms is under
// 2^-22). For that a position's row of K (V) is stored over the power of two
// of its largest scale; a score takes K's power back, and the probabilities
// take V's, their running maximum being that of probability times power, so
// that neither V nor the probabilities leave binary16's range. A tile's O is
// read from tensor memory and added to float registers, because sums in the
// tensor core's accumulators lose a little with every product.
//
// Warps: 0-3 softmax (a thread owns a row: no exchange between lanes), 4-7
// and 8-11 the two halves of O, 12-18 fill the tiles (F16: tensor copies;
// quantised: integers to binary16), 19 issues the products. Tensor
// memory: Q high | Q low | two S (then P) | two O.
//
// Bound: the products take 16 (F16) or 24 cycles per position and KV head
// whatever the number of rows up to 128, against 22 (F16), 12 (Q8_0) or 6
// (Q4_0) for the cache's bytes at head_dim 128. Measured: 64 tokens of 64 heads
// over 32768 F16 positions 138 us, the tensor cores busy 45 % of it: a tile
// takes some 2000 cycles of 1024, and leaving out the exponentials, the splitting
// or the reading of O changes that by 4 to 9 %: the roles wait for one
// another's latency. Before its first tile a CTA needs 9000 cycles (its 64 KB
// of q to tensor memory, the first tile), after the last 5000 (64 KB of O), which
// is most of a short context's time (32 rows of 8192 positions: 20 us).
// Tried and slower: two groups of softmax warps on alternate tiles (3 us more), two
// threads a row, the products issued by the oldest warp, the exponents by tile
// with a barrier, polling instead of sleeping waits, rolled loops.
#include "tcgen05.cuh"
#include "tree_attention.cuh"

using namespace syn;

namespace {

constexpr int kFillWarps = 7, kFillWarp0 = 12, kMmaWarp = kFillWarp0 + kFillWarps, kTcThreads = (kMmaWarp + 1) * 32;
constexpr int kFill = 32 * kFillWarps;  // threads that fill tiles
constexpr uint64_t kTcWaitNs = 2000000000ull;  // a wait gives up after 2 s
constexpr uint32_t kTcNapNs = 1000000;         // and sleeps in the barrier meanwhile: polling takes issue slots
constexpr int kEdgeTiles = kMaxTree / kTcTile + 2;  // tiles that hold rows of the tree

__device__ unsigned g_tree_timeouts = 0;  // bounded waits that gave up (syn_device_errors)

template <int TYPE, int HDP>
struct TcPlan {
    static constexpr bool quant = TYPE != SYN_F16;
    static constexpr int atom = kTcTile * 128;          // 64 positions x 64 dims
    static constexpr int tile = atom * (HDP / 64);      // one term of K or V
    static constexpr int k_lo = tile, v_hi = quant ? 2 * tile : tile;  // V's low term follows its high one
    static constexpr int stage = quant ? 4 * tile : 2 * tile;
    static constexpr int stages = quant ? (HDP == 64 ? 4 : 3) : 5;
    static constexpr int smem = stages * stage + 1024;  // from a 1024-byte boundary
    // tensor memory columns
    static constexpr int q_hi = 0, q_lo = HDP / 2, s = HDP, o = HDP + 2 * kTcTile;
    static_assert(o + 2 * HDP <= 512, "tensor memory");
};

// The F16 caches as tensors (column, position, sequence), boxes of 64 columns x 64 positions under the 128-byte
// swizzle; used where head_dim is a multiple of 64.
struct TcMaps {
    CUtensorMap k, v;
};
__device__ __forceinline__ void tma_load_tile(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar)) : "memory");
}

struct TcShared {
    uint64_t q_full, kv_full[5], kv_empty[5], s_full[2], p_full[4], o_full[2], o_empty[2], done;
    unsigned long long bad[kEdgeTiles];  // positions of a tree tile that hold values that are not finite
    float corr[4][kTcRows];              // a tile's factor of the rows' sums so far
    float k_pow[5][kTcTile];             // the powers of two of a stage's positions: K's,
    float v_log[5][kTcTile];             // V's logarithm,
    float v_inv[5][kTcTile];             // and V's inverse
    float m[kTcRows], l[kTcRows];
    float q_scale[kTcRows];              // the rows' factor of a product's scores
    uint32_t tmem;
    int abort;
};

// Waits for phase `parity`; false when it gave up, here or in another thread of the CTA. The way of a barrier that is
// not ready yet is a call: the loops stay small enough for the instruction cache that the roles share.
__device__ __noinline__ bool tc_wait_on(uint64_t* bar, uint32_t parity, TcShared& sh) {
    const uint64_t t0 = global_ns();
    for (;;) {
        if (mbar_try_wait_sleep(bar, parity, kTcNapNs)) return true;
        if (*reinterpret_cast<volatile int*>(&sh.abort)) return false;
        if (global_ns() - t0 > kTcWaitNs) {
            *reinterpret_cast<volatile int*>(&sh.abort) = 1;
            atomicAdd(&g_tree_timeouts, 1u);
            return false;
        }
    }
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, TcShared& sh) {
    bool ok = mbar_try_wait(bar, parity);
    if (!ok) ok = tc_wait_on(bar, parity, sh);
    return __all_sync(0xffffffffu, ok);
}

// Byte offset of 16-byte chunk c (8 dims) of position p in a swizzled tile.
__device__ __forceinline__ int tile_at(int p, int c) { return (c >> 3) * (kTcTile * 128) + p * 128 + (((c & 7) ^ (p & 7)) << 4); }

// The tile's positions that token tk sees: bit p for the tree's row j0 + p (a committed row where that is negative).
__device__ __forceinline__ unsigned long long tile_sees(const TreeParams& a, int seq, int tk, int j0) {
    uint32_t w[3];
    const int first = j0 >> 5, shift = j0 & 31;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const int wi = first + i, left = a.n_tree - 32 * wi;  // rows of the tree from this word on
        if (wi < 0) {
            w[i] = 0xffffffffu;
        } else if (left <= 0 || tk >= a.n_tree) {
            w[i] = 0;
        } else {
            const int most = a.mask ? left : min(left, tk + 1 - 32 * wi);
            w[i] = most <= 0 ? 0u : a.mask ? __ldg(a.mask + (size_t(seq) * a.n_tree + tk) * a.mask_words + wi) : 0xffffffffu;
            if (most > 0 && most < 32) w[i] &= (1u << most) - 1u;
        }
    }
    return (unsigned long long)(__funnelshift_r(w[1], w[2], shift)) << 32 | __funnelshift_r(w[0], w[1], shift);
}

template <int TYPE, int HDP>
__global__ void __launch_bounds__(kTcThreads, 1) tree_attn_tc_kernel(const TreeParams a, const __grid_constant__ TcMaps maps) {
    using P = TcPlan<TYPE, HDP>;
    extern __shared__ unsigned char raw[];
    __shared__ TcShared sh;
    unsigned char* tiles = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
    const uint32_t tiles_s = smem_addr(tiles);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int hd = a.c.hd;
    const int kvh = blockIdx.y / a.row_blocks, rb = blockIdx.y - kvh * a.row_blocks;
    const int row0 = rb * kTcRows, rows = min(kTcRows, a.rows - row0);

    pdl_launch_dependents();
    pdl_wait();
    const Cutting cut = tree_cutting(a, kTcTile, blockIdx.x);
    const int seq = cut.seq;
    if (seq < 0) return;
    note_cut(a, cut);
    const int len = tree_len(a, seq), total = len + a.n_tree;
    const int n_tiles = (total + kTcTile - 1) / kTcTile;
    const int t0 = (int(blockIdx.x) - cut.first) * cut.per, n = min(cut.per, n_tiles - t0);  // tiles t0 .. t0 + n - 1
    const int edge0 = len / kTcTile;  // the first tile with a row of the tree

    if (tid == 0) {
        mbar_init(&sh.q_full, 128);
        for (int i = 0; i < P::stages; ++i) {
            mbar_init(&sh.kv_full[i], kFillWarps);
            mbar_init(&sh.kv_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.o_full[i], 1);
            mbar_init(&sh.o_empty[i], 256);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&sh.p_full[i], 128);
        mbar_init(&sh.done, 1);
        mbar_init_fence();
        sh.abort = 0;
    }
    if (tid < kEdgeTiles) sh.bad[tid] = 0;
    if (warp == kMmaWarp) tmem_alloc_all(&sh.tmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = sh.tmem;

    // q, by all but the fill warps, which start on the tiles: a row at a time (lane = dims), as it is and then split in
    // place, in the tile memory that they leave free until q_full. Rows past the last stay what they are; they reach no other row's output.
    constexpr int kQPitch = HDP * 2 + 16;
    unsigned char* q_stage = tiles + P::stage;  // [row][high | low]
    if (warp < kFillWarp0) {
        constexpr int V = HDP / 32;
        const bool vec = ((reinterpret_cast<uintptr_t>(a.q) & 15) | (a.q_stride & 3)) == 0;
        const float* q = a.q + size_t(seq) * a.n_tree * a.q_stride + size_t(kvh) * a.group * hd;
        int tok = (row0 + warp) / a.group, h = row0 + warp - tok * a.group;
#pragma unroll 1
        for (int r = warp; r < rows; r += kFillWarp0) {
            const float* src = q + size_t(tok) * a.q_stride + h * hd;
            unsigned char* to = q_stage + r * 2 * kQPitch;
            if (vec) {
                if (4 * lane < HDP) cp16(smem_addr(to) + 16 * lane, 4 * lane < hd ? src + 4 * lane : src, 4 * lane < hd);
            } else {
#pragma unroll 1
                for (int d = lane; d < HDP; d += 32) reinterpret_cast<float*>(to)[d] = d < hd ? __ldg(src + d) : 0.0f;
            }
            for (h += kFillWarp0; h >= a.group; h -= a.group) ++tok;
        }
        cp_commit();
        cp_wait<0>();
        __syncwarp();
#pragma unroll 1
        for (int r = warp; r < rows; r += kFillWarp0) {
            unsigned char* row = q_stage + r * 2 * kQPitch;
            float x[V];
            uint32_t top = 0;
            if constexpr (V == 4) {
                const float4 f = reinterpret_cast<const float4*>(row)[lane];
                x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
            } else {
                const float2 f = reinterpret_cast<const float2*>(row)[lane];
                x[0] = f.x; x[1] = f.y;
            }
#pragma unroll
            for (int e = 0; e < V; ++e) top = max(top, __float_as_uint(fabsf(x[e])));
            float up, down;
            q_factor(__uint_as_float(__reduce_max_sync(0xffffffffu, top)), up, down);
            const float by = fabsf(a.scale_log2) * down;
            if (lane == 0) sh.q_scale[r] = by == 0.0f ? 0x1p-126f : by;  // masked scores, -inf, are multiplied by it
            if (a.scale_log2 < 0.0f) up = -up;  // the scores' factor is positive: maxima may be taken before it
            uint32_t hi[V / 2], lo[V / 2];
#pragma unroll
            for (int e = 0; e < V; e += 2) split2(x[e] * up, x[e + 1] * up, hi[e / 2], lo[e / 2]);
            if constexpr (V == 4) {
                reinterpret_cast<uint2*>(row)[lane] = make_uint2(hi[0], hi[1]);
                reinterpret_cast<uint2*>(row + kQPitch)[lane] = make_uint2(lo[0], lo[1]);
            } else {
                reinterpret_cast<uint32_t*>(row)[lane] = hi[0];
                reinterpret_cast<uint32_t*>(row + kQPitch)[lane] = lo[0];
            }
        }
        asm volatile("bar.sync 2, 384;" ::: "memory");
    }

    if (warp < 4) {
        // ---- softmax: thread = row -------------------------------------------------
        const bool live = 32 * (warp & 3) < rows;  // the warp has rows
        const int r = tid & 127, row = row0 + r;
        const int tok = row / a.group;
        const uint32_t lanes = tm + (uint32_t(32 * (warp & 3)) << 16);
        const float c = sh.q_scale[r];
        if (live) {
#pragma unroll
            for (int b = 0; b < HDP / 16; ++b) {  // 16 columns: 32 dims of the high, then of the low term
                const int term = b / (HDP / 32), at = b % (HDP / 32);
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint4 x = *reinterpret_cast<const uint4*>(q_stage + (r * 2 + term) * kQPitch + at * 64 + e * 16);
                    w[4 * e] = x.x; w[4 * e + 1] = x.y; w[4 * e + 2] = x.z; w[4 * e + 3] = x.w;
                }
                tmem_st16(lanes + (term ? P::q_lo : P::q_hi) + 16 * at, w);
            }
            tmem_wait_st();
        }
        tc_fence_before();
        fence_async_shared();
        mbar_arrive(&sh.q_full);
        float m = -INFINITY, l = 0.0f;
        for (int j = 0; j < n; ++j) {
            const int t = t0 + j, st = j % P::stages;
            const bool edge = t >= edge0;
            bool ok = warp_wait(&sh.s_full[j & 1], uint32_t(j >> 1) & 1, sh);
            if (ok && (P::quant || edge)) ok = warp_wait(&sh.kv_full[st], uint32_t(j / P::stages) & 1, sh);
            if (!ok) break;
            if (live) {
                tc_fence_after();
                float s[2][32];
                tmem_ld32(s[0], lanes + P::s + (j & 1) * kTcTile);
                tmem_ld32(s[1], lanes + P::s + (j & 1) * kTcTile + 32);
                tmem_wait_ld();
                // F16: raw scores, times c > 0 in the exponent; quantised: times K's power and c, plus the logarithm of V's
                auto each4 = [&](auto f) {
#pragma unroll
                    for (int e = 0; e < kTcTile; e += 4) f(reinterpret_cast<float(&)[4]>(s[e >> 5][e & 31]), e);
                };
                if (P::quant)
                    each4([&](float(&v)[4], int e) {
                        const float4 kp = *reinterpret_cast<const float4*>(sh.k_pow[st] + e), vl = *reinterpret_cast<const float4*>(sh.v_log[st] + e);
                        mul2(v[0], v[1], kp.x, kp.y);
                        mul2(v[2], v[3], kp.z, kp.w);
                        fma2(v[0], v[1], c, c, vl.x, vl.y);
                        fma2(v[2], v[3], c, c, vl.z, vl.w);
                    });
                else  // an infinity in K may score -inf, which would drop its row in silence: NaN (as a quantised one's low term is)
                    each4([&](float(&v)[4], int) {
                        fma2(v[0], v[1], 0.0f, 0.0f, v[0], v[1]);
                        fma2(v[2], v[3], 0.0f, 0.0f, v[2], v[3]);
                    });
                if (edge) {
                    const unsigned long long bad = sh.bad[t - edge0], sees = tile_sees(a, seq, tok, t * kTcTile - len);
                    const uint32_t bw[2] = {uint32_t(bad), uint32_t(bad >> 32)}, sw[2] = {uint32_t(sees), uint32_t(sees >> 32)};
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!(sw[u] >> e & 1u)) s[u][e] = -INFINITY;
                            else if (bw[u] >> e & 1u) s[u][e] = __uint_as_float(0x7fffffffu);
                }
                float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                each4([&](float(&v)[4], int e) {
                    float& y = x[(e >> 2) & 3];
                    y = fmaxf(fmaxf(fmaxf(y, v[0]), fmaxf(v[1], v[2])), v[3]);
                });
                const float most = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                const float mn = fmaxf(m, P::quant || most == -INFINITY ? most : most * c);
                const float corr = mn > m ? ex2(m - mn) : 1.0f;  // m = -inf: 0
                sh.corr[j & 3][r] = corr;
                m = mn;
                const float base = kPShift - (m == -INFINITY ? 0.0f : m);
                float sum[4] = {l * corr, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        float(&v)[4] = reinterpret_cast<float(&)[4]>(s[u >> 1][16 * (u & 1) + 2 * e]);
                        if (P::quant) {
                            add2(v[0], v[1], base, base);
                            add2(v[2], v[3], base, base);
                        } else {
                            fma2(v[0], v[1], c, c, base, base);
                            fma2(v[2], v[3], c, c, base, base);
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = ex2(v[i]);
                        if (P::quant) {  // the sum is the probabilities' own
                            const float4 vi = *reinterpret_cast<const float4*>(sh.v_inv[st] + 16 * u + 2 * e);
                            fma2_to(sum[0], sum[1], v[0], v[1], vi.x, vi.y);
                            fma2_to(sum[2], sum[3], v[2], v[3], vi.z, vi.w);
                        } else {
                            add2(sum[0], sum[1], v[0], v[1]);
                            add2(sum[2], sum[3], v[2], v[3]);
                        }
                        split2(v[0], v[1], hi[e], lo[e]);
                        split2(v[2], v[3], hi[e + 1], lo[e + 1]);
                    }
                    tmem_st8(lanes + P::s + (j & 1) * kTcTile + 8 * u, hi);
                    tmem_st8(lanes + P::s + (j & 1) * kTcTile + 32 + 8 * u, lo);
                }
                l = (sum[0] + sum[1]) + (sum[2] + sum[3]);
                tmem_wait_st();
            }
            tc_fence_before();
            mbar_arrive(&sh.p_full[j & 3]);
        }
        sh.m[r] = m;
        sh.l[r] = l;
    } else if (warp < 12) {
        // ---- O: thread = row, half of the dims -----------------------------------------
        constexpr int W = HDP / 2;
        const int half = (warp - 4) >> 2, r = tid & 127;
        const bool live = 32 * (warp & 3) < rows;
        const uint32_t from = tm + (uint32_t(32 * (warp & 3)) << 16) + P::o + half * W;
        float acc[W];
#pragma unroll
        for (int d = 0; d < W; ++d) acc[d] = 0.0f;
        for (int j = 0; j < n; ++j) {
            bool ok = warp_wait(&sh.p_full[j & 3], uint32_t(j >> 2) & 1, sh);
            ok = ok && warp_wait(&sh.o_full[j & 1], uint32_t(j >> 1) & 1, sh);
            if (!ok) break;
            if (live) {
                tc_fence_after();
                const float f = sh.corr[j & 3][r];
#pragma unroll
                for (int b = 0; b < W / 16; ++b) {
                    float o[16];
                    tmem_ld16(o, from + (j & 1) * HDP + 16 * b);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; e += 2)
                        fma2(acc[16 * b + e], acc[16 * b + e + 1], f, f, o[e], o[e + 1]);
                }
            }
            tc_fence_before();
            mbar_arrive(&sh.o_empty[j & 1]);
        }
        asm volatile("bar.sync 2, 384;" ::: "memory");  // the softmax warps' m and l
        const float l = sh.l[r];
        // through the tile memory (every product has read it: the last O was waited for), for whole-line stores
        constexpr int pitch = HDP + 4;
        float* stage = reinterpret_cast<float*>(tiles);
        const bool whole = a.parts == 0;
        const float inv = !whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
        const size_t part = (size_t(blockIdx.x) * gridDim.y + blockIdx.y) * kTcRows;
        if (live) {
#pragma unroll
            for (int d = 0; d < W; d += 4)
                *reinterpret_cast<float4*>(stage + r * pitch + half * W + d) =
                    make_float4(acc[d] * inv, acc[d + 1] * inv, acc[d + 2] * inv, acc[d + 3] * inv);
            if (!whole && half == 0 && r < rows) a.part_ml[part + r] = make_float2(sh.m[r], l);
        }
        asm volatile("bar.sync 3, 256;" ::: "memory");
        if (4 * lane < hd) {
            const float* from = stage + 4 * lane;
            if (!whole) {
                float* out = a.part_o + part * hd + 4 * lane;
#pragma unroll 2
                for (int x = warp - 4; x < rows; x += 8)
                    *reinterpret_cast<float4*>(out + x * hd) = *reinterpret_cast<const float4*>(from + x * pitch);
            } else {
#pragma unroll 1
                for (int x = warp - 4; x < rows; x += 8) {
                    const int row = row0 + x, tok = row / a.group, h = kvh * a.group + row - tok * a.group;
                    *reinterpret_cast<float4*>(a.out + ((size_t(seq) * a.n_tree + tok) * a.n_head + h) * hd + 4 * lane) =
                        *reinterpret_cast<const float4*>(from + x * pitch);
                }
            }
        }
    } else if (warp < kMmaWarp) {
        // ---- tiles ------------------------------------------------------------------------
        const int fw = warp - kFillWarp0, ft = fw * 32 + lane;
        const char *kb = a.c.k + size_t(seq) * a.c.seq_stride, *vb = a.c.v + size_t(seq) * a.c.seq_stride;
        auto full = [&](int j) {
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.kv_full[j % P::stages]);
        };
        if constexpr (!P::quant) {
            constexpr int CP = HDP / 8;  // chunks of a row
            const size_t pitch = size_t(a.c.n_kv) * hd * 2, head = size_t(kvh) * hd * 2;
            const int chunks = hd / 8;
            int j = 0;
            for (; j < n; ++j) {
                const int st = j % P::stages, t = t0 + j, p0 = t * kTcTile;
                if (j == 1 && !warp_wait(&sh.q_full, 0, sh)) break;
                if (j >= P::stages && !warp_wait(&sh.kv_empty[st], uint32_t(j / P::stages - 1) & 1, sh)) break;
                if (t < edge0 && hd % 64 == 0) {
                    if (lane == 0) {
                        if (fw == 0) {
                            const uint32_t to = tiles_s + st * P::stage;
                            fence_async_shared();  // q was staged here
                            mbar_expect_tx(&sh.kv_full[st], 2 * uint32_t(hd) * kTcTile * 2);
                            for (int i = 0; i < hd / 64; ++i) {
                                tma_load_tile(to + i * P::atom, &maps.k, kvh * hd + 64 * i, p0, seq, &sh.kv_full[st]);
                                tma_load_tile(to + P::v_hi + i * P::atom, &maps.v, kvh * hd + 64 * i, p0, seq, &sh.kv_full[st]);
                            }
                        } else {
                            mbar_arrive(&sh.kv_full[st]);
                        }
                    }
                    continue;
                }
                unsigned char* to = tiles + st * P::stage;
#pragma unroll 4
                for (int i = ft; i < kTcTile * CP; i += kFill) {
                    const int p = i / CP, ch = i % CP;
                    const bool in = p0 + p < total && ch < chunks;  // dims past the head are zero
                    const size_t at = in ? size_t(p0 + p) * pitch + head + ch * 16 : 0;
                    const int off = tile_at(p, ch);
                    const uint4 z = make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4*>(to + off) = in ? *reinterpret_cast<const uint4*>(kb + at) : z;
                    uint4 x = in ? *reinterpret_cast<const uint4*>(vb + at) : z;
                    if (p0 + p >= len) {
                        // a row of the tree: what is not finite becomes 0 (a probability of 0 times it would be
                        // NaN) and its position scores NaN for the tokens that see it
                        uint32_t w[4] = {x.x, x.y, x.z, x.w};
                        bool bad = false;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if ((w[e] & 0x7c00u) == 0x7c00u) { w[e] &= 0xffff0000u; bad = true; }
                            if ((w[e] & 0x7c000000u) == 0x7c000000u) { w[e] &= 0xffffu; bad = true; }
                        }
                        x = make_uint4(w[0], w[1], w[2], w[3]);
                        if (bad) atomicOr(&sh.bad[t - edge0], 1ull << p);
                    }
                    *reinterpret_cast<uint4*>(to + P::v_hi + off) = x;
                }
                full(j);
            }
            if (j < n)  // it gave up: its copies in flight land before it leaves
                for (int k = max(0, j - P::stages); k < j; ++k)
                    mbar_wait_bounded(&sh.kv_full[k % P::stages], uint32_t(k / P::stages) & 1, kTcWaitNs);
        } else {
            constexpr int VPC = TYPE == SYN_Q8_0 ? 16 : 32;          // values of 16 bytes of quants
            constexpr int CP = HDP / VPC, NI = kTcTile * CP / 32, N = (2 * NI + kFillWarps - 1) / kFillWarps;  // chunks of a row; sets of K; of a warp
            constexpr int PS = 32 / CP;  // positions of a set
            const int nb = hd / 32, chunks = hd / VPC;
            // A warp's share of a tile: sets of 32 chunks (16 bytes of quants) of K, then of V, every kFillWarps-th. A lane
            // has the same chunk `ch` of a row in all of them. A set of the next tile is requested as soon as this
            // tile's is in hand.
            const int ch = lane % CP, lp = lane / CP;
            const size_t row_at = size_t(kvh) * a.c.max_ctx + size_t(t0) * kTcTile + lp;
            const char *kq = kb + (row_at * chunks + ch) * 16, *ks = kb + a.c.scale_plane + (row_at * nb + ch * VPC / 32) * 2;
            const ptrdiff_t to_v = vb - kb;
            const uint32_t set_q = PS * chunks * 16, set_s = PS * nb * 2;
            uint4 q[N];
            uint32_t d[N];  // scale bits
            auto fetch = [&](int k, int j) {
                const int i = k * kFillWarps + fw;
                if (i >= 2 * NI) return;
                const bool v = i >= NI;
                const int ii = v ? i - NI : i;
                q[k] = make_uint4(0, 0, 0, 0);
                d[k] = 0;
                if (ch < chunks && (t0 + j) * kTcTile + ii * PS + lp < total) {
                    const char *qp = kq + (v ? to_v : 0), *sp = ks + (v ? to_v : 0);
                    q[k] = __ldg(reinterpret_cast<const uint4*>(qp + ii * set_q + size_t(j) * (kTcTile / PS) * set_q));
                    d[k] = __ldg(reinterpret_cast<const uint16_t*>(sp + ii * set_s + size_t(j) * (kTcTile / PS) * set_s));
                }
            };
            // a lane's place in a swizzled row: neighbouring lanes store different 16-byte columns at a time, those of the
            // second 64 dims take the chunk's eights in another order
            const int c0 = ch * (VPC / 8), turn = (c0 >> 3) * (VPC / 16);
            const uint32_t lane_at = (c0 >> 3) * P::atom + lp * 128;
            const __half2 zero = half2_of(TYPE == SYN_Q8_0 ? 0x64806480u : 0x64086408u);
            auto convert = [&](int k, int j, int st) {
                const int i = k * kFillWarps + fw;
                if (i >= 2 * NI) return;
                const bool v = i >= NI;
                const int ii = v ? i - NI : i, p = ii * PS + lp;
                uint32_t top = d[k] & 0x7fffu;
                bool bad = false;  // the position's row: NaN for who sees it, by its logarithm (V) or its values (K)
                if (__any_sync(0xffffffffu, top >= 0x7c00u)) {
                    const int t = t0 + j;
                    bad = __ballot_sync(0xffffffffu, top >= 0x7c00u) >> (lane - ch) & ((1u << CP) - 1u);
                    if (top >= 0x7c00u) {
                        if (t * kTcTile + p >= len) {
                            d[k] = 0;
                            atomicOr(&sh.bad[t - edge0], 1ull << p);
                        }
                        top = 0;
                    }
                }
                // the position's largest scale to [2^8, 2^9): 127 of it is finite, and the low term reaches 2^-33 of it
#pragma unroll
                for (int o = TYPE == SYN_Q8_0 ? 2 : 1; o < CP; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                const uint32_t e = max(top >> 10, 1u);
                const float up = __uint_as_float((150u - e) << 23), down = __uint_as_float((104u + e) << 23);  // 2^(23 - e), 2^(e - 23)
                if (ch == 0) {
                    if (!v) {
                        sh.k_pow[st][p] = down;
                    } else {
                        sh.v_log[st][p] = bad ? __uint_as_float(0x7fffffffu) : float(int(e) - 23);
                        sh.v_inv[st][p] = up;
                    }
                }
                const __half2 scale = __float2half2_rn(f16_from_bits(uint16_t(d[k])) * up);
                unsigned char* rowp = tiles + st * P::stage + (v ? P::v_hi : 0) + lane_at + ii * (PS * 128);
                const int col = (((c0 ^ p) & 7) ^ turn) << 4;
                uint32_t w[4] = {q[k].x, q[k].y, q[k].z, q[k].w};
                if (TYPE == SYN_Q8_0) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) w[x] ^= 0x80808080u;
                    if (turn) {
                        const uint32_t x = w[0], y = w[1];
                        w[0] = w[2]; w[1] = w[3]; w[2] = x; w[3] = y;
                    }
                }
                const int sh0 = TYPE == SYN_Q4_0 && turn ? 4 : 0;  // Q4_0: the high nibbles first
#pragma unroll
                for (int g = 0; g < VPC / 8; ++g) {  // 8 dims: one 16-byte column of each term
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int x2 = 0; x2 < 2; ++x2) {
                        uint32_t x = w[2 * (g & 1) + x2];
                        if (TYPE == SYN_Q4_0) x = x >> (g >> 1 ? 4 - sh0 : sh0) & 0x0f0f0f0fu;
#pragma unroll
                        for (int o = 0; o < 2; ++o) {
                            const __half2 n = __hsub2(bytes_h2(x, o ? 0x4342u : 0x4140u), zero);
                            const __half2 y = __hmul2(n, scale);
                            hi[2 * x2 + o] = bits(y);
                            lo[2 * x2 + o] = bits(__hfma2(n, scale, __hneg2(y)));
                        }
                    }
                    unsigned char* at = rowp + (col ^ (g << 4));
                    *reinterpret_cast<uint4*>(at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    *reinterpret_cast<uint4*>(at + P::tile) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
            };
#pragma unroll
            for (int k = 0; k < N; ++k) fetch(k, 0);
            int st = 0;
#pragma unroll 1
            for (int j = 0; j < n; ++j) {
                if (j == 1 && !warp_wait(&sh.q_full, 0, sh)) break;
                if (j >= P::stages && !warp_wait(&sh.kv_empty[st], uint32_t(j / P::stages - 1) & 1, sh)) break;
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    convert(k, j, st);
                    if (j + 1 < n) fetch(k, j + 1);
                }
                full(j);
                if (++st == P::stages) st = 0;
            }
        }
    } else {
        // ---- products (the whole warp runs the loop, one lane issues) ---------------------------
        constexpr uint32_t ds = mma_desc(128, kTcTile, false), dv = mma_desc(128, HDP, true);
        auto scores = [&](int j) {
            const int st = j % P::stages;
            if (!warp_wait(&sh.kv_full[st], uint32_t(j / P::stages) & 1, sh)) return false;
            tc_fence_after();
            const uint32_t d = tm + P::s + (j & 1) * kTcTile;
            const uint64_t k = smem_desc(tiles_s + st * P::stage, 16, 1024);
            if (elect_one()) {
#pragma unroll
                for (int term = P::quant ? 2 : 1; term >= 0; --term) {  // hi lo, lo hi, hi hi: the small first, for sums truncate
                    const uint32_t qa = tm + (term == 1 ? P::q_lo : P::q_hi);
#pragma unroll
                    for (int i = 0; i < HDP / 16; ++i)
                        mma_ts(d, qa + 8 * i, k + (((term == 2 ? P::k_lo : 0) + (i >> 2) * P::atom + (i & 3) * 32) >> 4), ds,
                               term < (P::quant ? 2 : 1) || i > 0);
                }
                mma_commit(&sh.s_full[j & 1]);
            }
            __syncwarp();
            return true;
        };
        bool ok = warp_wait(&sh.q_full, 0, sh);
        tc_fence_after();
        ok = ok && scores(0);
        for (int j = 0; ok && j < n; ++j) {
            if (j + 1 < n && !scores(j + 1)) break;
            if (!warp_wait(&sh.p_full[j & 3], uint32_t(j >> 2) & 1, sh)) break;
            if (j >= 2 && !warp_wait(&sh.o_empty[j & 1], uint32_t((j >> 1) - 1) & 1, sh)) break;
            tc_fence_after();
            const int st = j % P::stages;
            const uint32_t d = tm + P::o + (j & 1) * HDP, pa = tm + P::s + (j & 1) * kTcTile;
            const uint64_t v = smem_desc(tiles_s + st * P::stage + P::v_hi, P::atom, 1024);
            if (elect_one()) {
#pragma unroll
                for (int term = P::quant ? 2 : 1; term >= 0; --term) {
#pragma unroll
                    for (int i = 0; i < kTcTile / 16; ++i)
                        mma_ts(d, pa + (term == 1 ? 32 : 0) + 8 * i, v + (((term == 2 ? P::tile : 0) + i * 2048) >> 4), dv,
                               term < (P::quant ? 2 : 1) || i > 0);
                }
                mma_commit(&sh.o_full[j & 1]);
                mma_commit(&sh.kv_empty[st]);
            }
            __syncwarp();
        }
        // nothing of this CTA may be in flight when its tensor memory is freed
        if (elect_one()) mma_commit(&sh.done);
        __syncwarp();
        mbar_wait_bounded(&sh.done, 0, kTcWaitNs);
    }
    __syncwarp();
    if (warp < 4) asm volatile("bar.sync 2, 384;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kMmaWarp) tmem_free_all(tm);
}

int cache_map(const TreeParams& a, const char* base, CUtensorMap* m) {
    const auto encode = syn_tensor_map_encoder();
    if (!encode) {
        syn_set_error("cuTensorMapEncodeTiled is not available from the driver");
        return SYN_ERR_CUDA;
    }
    const cuuint64_t row = cuuint64_t(a.c.n_kv) * a.c.hd;
    const cuuint64_t dims[3] = {row, cuuint64_t(a.c.max_ctx), cuuint64_t(a.c.n_seq)};
    const cuuint64_t strides[2] = {row * 2, a.c.n_seq > 1 ? cuuint64_t(a.c.seq_stride) : row * 2 * a.c.max_ctx};
    const cuuint32_t box[3] = {64, kTcTile, 1}, estr[3] = {1, 1, 1};
    const CUresult r = encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<char*>(base), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        syn_set_error("cuTensorMapEncodeTiled rejected the KV cache geometry");
        return SYN_ERR_INVALID;
    }
    return SYN_OK;
}

template <int TYPE, int HDP>
int launch(const TreeParams& a, cudaStream_t s) {
    auto kernel = tree_attn_tc_kernel<TYPE, HDP>;
    constexpr int smem = TcPlan<TYPE, HDP>::smem;
    static_assert(smem + sizeof(TcShared) <= 227 * 1024, "shared memory of a CTA");
    int st = syn_opt_in_smem(reinterpret_cast<const void*>(kernel), smem);
    if (st) return st;
    TcMaps maps{};
    if (TYPE == SYN_F16 && a.c.hd % 64 == 0) {
        if ((st = cache_map(a, a.c.k, &maps.k))) return st;
        if ((st = cache_map(a, a.c.v, &maps.v))) return st;
    }
    const dim3 grid{unsigned(a.parts ? a.parts : a.c.n_seq), unsigned(a.c.n_kv * a.row_blocks), 1};
    return syn_launch(kernel, grid, kTcThreads, smem, s, a, maps);
}

}  // namespace

int syn_tree_attention_tc(const TreeParams& a, int type, cudaStream_t s) {
    if (a.c.hd <= 64)
        return type == SYN_F16 ? launch<SYN_F16, 64>(a, s) : type == SYN_Q8_0 ? launch<SYN_Q8_0, 64>(a, s) : launch<SYN_Q4_0, 64>(a, s);
    return type == SYN_F16 ? launch<SYN_F16, 128>(a, s) : type == SYN_Q8_0 ? launch<SYN_Q8_0, 128>(a, s) : launch<SYN_Q4_0, 128>(a, s);
}

// Bounded waits of the kernel that gave up on the current device (-1: unreadable).
int syn_tree_timeouts() {
    unsigned n = 0;
    if (cudaMemcpyFromSymbol(&n, g_tree_timeouts, sizeof n) != cudaSuccess) return -1;
    return int(n);
}
