// Logit processing between the output head and the choice of a token
// (syn_logits_process): biases, penalties for tokens already used, a grammar
// mask, and the pick of the largest, in one pass over the logits.
//
// Bound by memory: each logit is read and written once. A CTA takes a chunk
// of the vocabulary for the rows (tree nodes) of one sequence. It first
// counts the sequence's history and sums its biases for the chunk's tokens in
// shared memory (integer counts: the order of the atomics changes nothing)
// with a bit for every token that has either or that the tree has drafted.
// Then, row by row, a thread holds vectors of the row; for its marked tokens it
// computes the penalties (with the node's path added to their counts) in a loop
// over them, before the mask, the store and the maximum. Which of a thread's
// values are marked is the same in every row.
// Measured for 256 rows of 128256, histories of up to 4096, with a grammar:
// every value tested where it is held, 107 us (nearly every warp meets a marked
// token and takes the long way for each of a vector's values); marked tokens
// done afterwards in global memory, 111 us; marked tokens handed to a thread
// each through shared memory, 74 us (two barriers a row); as it is, 62 us, of
// which the bytes are 41 at the copy rate, and with 500 of history 55. The
// rest is the counting before the first row, one CTA of history per chunk. One
// row of 128256 takes 5.5 us, launch and counting. The picks are joined
// by a 64-bit maximum of (ordered value, lowest index), which does not depend on
// the order of arrival.
#include "common.cuh"

#include <algorithm>
#include <climits>

using namespace syn;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTree = 1024;
// Rows (nodes) of one CTA: few enough that the CTAs even out over the SMs, enough to pay for the counts. Measured with 8 /
// 4 / 2, us: 256 rows of 128256 62.3 / 61.6 / 69.3, 192 rows 48.7 / 44.4 / 47.8, 256 rows of 32000 28.2 / 20.2 / 21.7.
constexpr int kMaxRows = 4;

struct LogitParams {
    const float* x;
    float* out;
    int32_t* pick;
    size_t ld, out_ld, allowed_ld;
    const float* penalties;
    const int32_t *history, *history_len, *draft;
    const uint32_t* mask;
    const int32_t *bias_begin, *bias_token;
    const float* bias_value;
    const uint32_t* allowed;
    unsigned long long* key;  // [rows] best of the chunks seen so far, 0 = none
    unsigned* arrived;        // [rows]
    int n_tree, n_vocab, history_ld, n_bias, rows_per_cta;
};

// Counts: 32 bits in the short chunks, 16 (two to a word) in the long ones,
// whose CTAs then fit an SM four at a time; the host gives histories that
// could pass 16 bits to the short chunks.
template <int CHUNK>
struct Shared {
    static constexpr bool wide = CHUNK <= 1024;
    unsigned count[wide ? CHUNK : CHUNK / 2];
    float bias[CHUNK];
    float x[CHUNK];                   // a thread's own vectors, where it indexes them; before the rows, how often a bias names a token
    unsigned touched[CHUNK / 32];     // the tokens that may have a count or a bias
    unsigned drafted[CHUNK / 32];     // those some node of the tree has
    unsigned long long best[kMaxRows];
    unsigned short mine[kMaxTree];    // the nodes whose tokens are in this chunk
    int n_mine, thrice;
    __device__ __forceinline__ void add(int at) {
        if (wide) atomicAdd(&count[at], 1u);
        else atomicAdd(&count[at >> 1], 1u << (16 * (at & 1)));
    }
    __device__ __forceinline__ int counted(int at) const {
        return wide ? int(count[at]) : int(count[at >> 1] >> (16 * (at & 1)) & 0xffffu);
    }
};

// A float's bits in the order of the floats; 0 for NaN and -inf.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);  // -0 as +0
    return x > -INFINITY ? (b & 0x80000000u ? ~b : b | 0x80000000u) : 0u;
}

// A vector that is read once: not kept in L1, whose space in flight loads need.
__device__ __forceinline__ float4 load_once(const float* p) {
    float4 v;
    asm volatile("ld.global.L1::no_allocate.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
    return v;
}

template <int CHUNK, int VEC>
__global__ void __launch_bounds__(kThreads, 4) logits_kernel(const LogitParams a) {
    extern __shared__ __align__(16) unsigned char raw[];
    Shared<CHUNK>& sh = *reinterpret_cast<Shared<CHUNK>*>(raw);
    constexpr int kPer = CHUNK / (VEC * kThreads);  // vectors of a thread
    const int tid = threadIdx.x, lane = tid & 31;
    const int seq = blockIdx.z, v0 = blockIdx.x * CHUNK, span = min(CHUNK, a.n_vocab - v0);
    const int i0 = blockIdx.y * a.rows_per_cta, n_rows = min(a.rows_per_cta, a.n_tree - i0);
    for (int i = tid; i < CHUNK; i += kThreads) {
        if (i < int(sizeof(sh.count) / 4)) sh.count[i] = 0;
        sh.bias[i] = sh.x[i] = 0.0f;
        if (i < CHUNK / 32) sh.touched[i] = sh.drafted[i] = 0;
    }
    for (int i = tid; i < n_rows; i += kThreads) sh.best[i] = 0;
    if (tid == 0) sh.n_mine = sh.thrice = 0;
    __syncthreads();
    pdl_launch_dependents();
    pdl_wait();

    constexpr unsigned kAll = (1u << VEC) - 1u;
    const int words = (a.n_tree + 31) / 32;
    const bool full = span == CHUNK;
    float f[kPer][VEC];
    unsigned allowed = ~0u;  // a word of the grammar in each of the first kPer * VEC lanes
    auto load = [&](int i) {
        const size_t row = size_t(seq) * a.n_tree + i0 + i;
        const float* x = a.x + row * a.ld + v0 + tid * VEC;
        if (VEC == 4 && full) {
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                const float4 v = load_once(x + k * kThreads * VEC);
                f[k][0] = v.x; f[k][1 % VEC] = v.y; f[k][2 % VEC] = v.z; f[k][3 % VEC] = v.w;
            }
        } else {
#pragma unroll
            for (int k = 0; k < kPer; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int at = (k * kThreads + tid) * VEC + e;
                    f[k][e] = at < span ? x[k * kThreads * VEC + e] : -INFINITY;
                }
        }
        if (a.allowed && lane < kPer * VEC) {  // the warp's vectors k cover VEC words from k * 8 VEC + warp * VEC on
            const int w = lane / VEC * (kThreads * VEC / 32) + (tid >> 5) * VEC + lane % VEC;
            if (32 * w < span) allowed = __ldg(a.allowed + row * a.allowed_ld + (v0 >> 5) + w);
        }
    };
    load(0);  // on its way while the counts are made

    const int named0 = a.bias_begin ? __ldg(a.bias_begin + seq) : 0, named1 = a.bias_begin ? __ldg(a.bias_begin + seq + 1) : 0;
    auto touch = [&](int at) { atomicOr(&sh.touched[at >> 5], 1u << (at & 31)); };
    if (a.history) {
        const int n = min(a.history_len[seq], a.history_ld);
        const int32_t* h = a.history + size_t(seq) * a.history_ld;
        for (int i = tid; i < n; i += 8 * kThreads) {
            int tok[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) tok[j] = i + j * kThreads < n ? __ldg(h + i + j * kThreads) : -1;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (tok[j] >= v0 && tok[j] - v0 < span) {
                    sh.add(tok[j] - v0);
                    touch(tok[j] - v0);
                }
        }
    }
    // both in [0, n_bias], which leaves room for a CTA's steps below the largest int
    const int bias0 = min(max(named0, 0), a.n_bias), bias1 = min(max(named1, 0), a.n_bias);
    for (int i = bias0 + tid; i < bias1; i += kThreads) {
        const int tok = a.bias_token[i];
        if (tok >= v0 && tok - v0 < span) {
            atomicAdd(&sh.bias[tok - v0], a.bias_value[i]);
            if (atomicAdd(reinterpret_cast<unsigned*>(sh.x) + tok - v0, 1u) == 2) sh.thrice = 1;
            touch(tok - v0);
        }
    }
    const int32_t* draft = a.draft ? a.draft + size_t(seq) * a.n_tree : nullptr;
    if (draft)
        for (int j = tid; j < a.n_tree; j += kThreads) {
            const int tok = draft[j];
            if (tok >= v0 && tok - v0 < span) {
                sh.mine[atomicAdd(&sh.n_mine, 1)] = static_cast<unsigned short>(j);
                touch(tok - v0);
                atomicOr(&sh.drafted[(tok - v0) >> 5], 1u << ((tok - v0) & 31));
            }
        }
    __syncthreads();
    if (sh.thrice) {  // a sum of two is the same in either order; those of more are made again, in the list's order
        for (int at = tid; at < CHUNK; at += kThreads)
            if (__float_as_uint(sh.x[at]) > 2) {
                float sum = 0.0f;
                for (int i = bias0; i < bias1; ++i)
                    if (a.bias_token[i] == v0 + at) sum += a.bias_value[i];
                sh.bias[at] = sum;
            }
        __syncthreads();
    }
    const int n_mine = sh.n_mine;
    const float repeat = a.penalties ? a.penalties[3 * seq] : 1.0f;
    const float presence = a.penalties ? a.penalties[3 * seq + 1] : 0.0f;
    const float frequency = a.penalties ? a.penalties[3 * seq + 2] : 0.0f;
    unsigned some = 0;  // which of this thread's values may change
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const int at = (k * kThreads + tid) * VEC;
        some |= (sh.touched[at >> 5] >> (at & 31) & kAll) << (k * VEC);
    }

    for (int i = 0; i < n_rows; ++i) {
        const int node = i0 + i;
        const size_t row = size_t(seq) * a.n_tree + node;
        if (some) {  // through shared memory, for their indexes are not known to the compiler
            float* x = sh.x + tid * VEC;
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                if constexpr (VEC == 4) *reinterpret_cast<float4*>(x + k * kThreads * VEC) = make_float4(f[k][0], f[k][1], f[k][2], f[k][3]);
                else x[k * kThreads] = f[k][0];
            }
            for (unsigned left = some; left; left &= left - 1) {
                const int b = __ffs(left) - 1, at = (b / VEC * kThreads + tid) * VEC + b % VEC;
                float y = sh.x[at] + sh.bias[at];
                int c = sh.counted(at);
                if (n_mine && (sh.drafted[at >> 5] >> (at & 31) & 1u))
                    for (int d = 0; d < n_mine; ++d) {
                        const int j = sh.mine[d];
                        if (draft[j] == v0 + at && (a.mask ? a.mask[row * words + (j >> 5)] >> (j & 31) & 1u : j <= node)) ++c;
                    }
                if (c > 0) {
                    y = y > 0.0f ? __fdiv_rn(y, repeat) : y * repeat;
                    y -= float(c) * frequency + presence;
                }
                sh.x[at] = y;
            }
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                if constexpr (VEC == 4) {
                    const float4 v = *reinterpret_cast<const float4*>(x + k * kThreads * VEC);
                    f[k][0] = v.x; f[k][1] = v.y; f[k][2] = v.z; f[k][3] = v.w;
                } else {
                    f[k][0] = x[k * kThreads];
                }
            }
        }
        __syncwarp();
        if (a.allowed)
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                const unsigned may = __shfl_sync(0xffffffffu, allowed, k * VEC + lane * VEC / 32) >> (lane * VEC & 31);
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (!(may >> e & 1u)) f[k][e] = -INFINITY;
            }
        if (a.out) {
            float* out = a.out + row * a.out_ld + v0 + tid * VEC;
            if (VEC == 4 && full) {
#pragma unroll
                for (int k = 0; k < kPer; ++k)
                    __stcs(reinterpret_cast<float4*>(out + k * kThreads * VEC), make_float4(f[k][0], f[k][1 % VEC], f[k][2 % VEC], f[k][3 % VEC]));
            } else {
#pragma unroll
                for (int k = 0; k < kPer; ++k)
#pragma unroll
                    for (int e = 0; e < VEC; ++e)
                        if ((k * kThreads + tid) * VEC + e < span) out[k * kThreads * VEC + e] = f[k][e];
            }
        }
        if (a.pick) {
            float top = f[0][0];
#pragma unroll
            for (int k = 0; k < kPer * VEC; ++k) top = fmaxf(top, f[k / VEC][k % VEC]);  // a NaN loses
            const uint32_t o = ordered(top), best = __reduce_max_sync(0xffffffffu, o);
            // the warp's largest, where the CTA has none larger so far
            if (o == best && o && o >= uint32_t(*reinterpret_cast<volatile unsigned long long*>(&sh.best[i]) >> 32)) {
                int at = 0;
#pragma unroll
                for (int k = kPer * VEC - 1; k >= 0; --k)
                    if (f[k / VEC][k % VEC] == top) at = (k / VEC * kThreads + tid) * VEC + k % VEC;
                atomicMax(&sh.best[i], static_cast<unsigned long long>(o) << 32 | (0xffffffffu - uint32_t(v0 + at)));
            }
        }
        if (i + 1 < n_rows) load(i + 1);
    }
    if (!a.pick) return;
    __syncthreads();
    for (int i = tid; i < n_rows; i += kThreads) {
        const size_t row = size_t(seq) * a.n_tree + i0 + i;
        if (sh.best[i]) atomicMax(a.key + row, sh.best[i]);
        __threadfence();
        if (atomicAdd(a.arrived + row, 1u) == gridDim.x - 1) {  // the row's last chunk
            __threadfence();
            const unsigned long long k = atomicExch(a.key + row, 0ull);
            a.pick[row] = k ? int32_t(0xffffffffu - uint32_t(k)) : -1;
            a.arrived[row] = 0;
        }
    }
}

template <int CHUNK, int VEC>
int launch(LogitParams a, int n_seq, cudaStream_t s) {
    const int chunks = (a.n_vocab + CHUNK - 1) / CHUNK;
    // rows of a sequence stay in one CTA (its counts are made once) unless that leaves SMs idle
    const long ctas = long(chunks) * n_seq;
    const int groups = int(std::max<long>(1, 2l * syn_num_sms() / ctas));
    a.rows_per_cta = std::min(kMaxRows, (a.n_tree + groups - 1) / groups);
    const dim3 grid{unsigned(chunks), unsigned((a.n_tree + a.rows_per_cta - 1) / a.rows_per_cta), unsigned(n_seq)};
    const int st = syn_opt_in_smem(reinterpret_cast<const void*>(logits_kernel<CHUNK, VEC>), sizeof(Shared<CHUNK>));
    if (st) return st;
    return syn_launch(logits_kernel<CHUNK, VEC>, grid, kThreads, sizeof(Shared<CHUNK>), s, a);
}

}  // namespace

extern "C" size_t syn_logits_scratch_bytes(int n_rows) { return n_rows <= 0 ? 0 : align256(size_t(n_rows) * 12); }

extern "C" int syn_logits_process(const syn_logits_args* x, void* stream) {
    if (!x || !x->logits || (!x->out && !x->pick)) return SYN_ERR_INVALID;
    if (x->n_seq <= 0 || x->n_tree <= 0 || x->n_vocab <= 0) return SYN_ERR_INVALID;
    if (x->n_tree > kMaxTree || x->n_seq > 65535) return SYN_ERR_UNSUPPORTED;
    const size_t words = (size_t(x->n_vocab) + 31) / 32;
    LogitParams a{};
    a.x = x->logits; a.out = x->out; a.pick = x->pick;
    a.ld = x->ld ? x->ld : size_t(x->n_vocab);
    a.out_ld = x->out_ld ? x->out_ld : size_t(x->n_vocab);
    a.allowed_ld = x->allowed_ld ? x->allowed_ld : words;
    if (a.ld < size_t(x->n_vocab) || a.out_ld < size_t(x->n_vocab) || a.allowed_ld < words) return SYN_ERR_INVALID;
    if (x->out == x->logits && a.ld != a.out_ld) return SYN_ERR_INVALID;
    if (x->history && (!x->history_len || x->history_ld <= 0)) return SYN_ERR_INVALID;
    if (x->bias_begin && (!x->bias_token || !x->bias_value || x->n_bias < 0)) return SYN_ERR_INVALID;
    if (x->pick && (!x->scratch || (reinterpret_cast<uintptr_t>(x->scratch) & 7))) return SYN_ERR_INVALID;
    a.penalties = x->penalties;
    a.history = x->history; a.history_len = x->history_len; a.history_ld = x->history_ld;
    a.draft = x->draft; a.mask = x->mask;
    a.bias_begin = x->bias_begin; a.bias_token = x->bias_token; a.bias_value = x->bias_value;
    a.n_bias = x->n_bias && x->n_bias < INT_MAX - kThreads ? x->n_bias : INT_MAX - kThreads;
    a.allowed = x->allowed;
    const size_t rows = size_t(x->n_seq) * x->n_tree;
    a.key = static_cast<unsigned long long*>(x->scratch);
    a.arrived = x->scratch ? reinterpret_cast<unsigned*>(a.key + rows) : nullptr;
    a.n_tree = x->n_tree; a.n_vocab = x->n_vocab;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    // rows of 16-byte vectors where every row starts on a 16-byte boundary
    const uintptr_t at = reinterpret_cast<uintptr_t>(x->logits) | reinterpret_cast<uintptr_t>(x->out);
    const bool vec = (at & 15) == 0 && a.ld % 4 == 0 && (!x->out || a.out_ld % 4 == 0);
    // Short chunks while the rows' long ones would not give every SM a CTA. Measured, short / long, us: one row of
    // 128256 5.5 / 5.9, four 7.0 / 6.8, eight 9.2 / 7.2; 8 rows of 32000 6.2 / 7.0, 32 rows 10.0 / 7.5.
    const bool few = rows * ((size_t(x->n_vocab) + 4095) / 4096) < size_t(syn_num_sms()) ||
                     (x->history && size_t(x->history_ld) + x->n_tree > 0xffff);  // counts of more than 16 bits
    if (few) return vec ? launch<1024, 4>(a, x->n_seq, s) : launch<1024, 1>(a, x->n_seq, s);
    return vec ? launch<4096, 4>(a, x->n_seq, s) : launch<4096, 1>(a, x->n_seq, s);
}
