// Logit processing between the output head and the choice of a token
// (syn_logits_process): biases, penalties for tokens already used, a grammar
// mask, and the pick of the largest, in one pass over the logits.
//
// Bound by memory: each logit is read and written once. A CTA takes a chunk
// of the vocabulary for the rows (tree nodes) of one sequence. It first
// counts the sequence's history and sums its biases for the chunk's tokens in
// shared memory (integer counts: the order of the atomics changes nothing),
// with a bit per token that has either, so that the rows' pass reads the
// counts only where there is something. A node's own path adds to the counts
// before its row and is taken off after it, where a drafted token falls into
// the chunk at all. The picks are joined by a 64-bit maximum of (ordered
// value, lowest index), which does not depend on the order of arrival.
#include "common.cuh"

#include <algorithm>

using namespace syn;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTree = 1024;
constexpr int kMaxRows = 64;  // rows (nodes) of one CTA

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
    int n_tree, n_vocab, history_ld, rows_per_cta;
};

template <int CHUNK>
struct Shared {
    int count[CHUNK];
    float bias[CHUNK];
    unsigned touched[CHUNK / 32];  // tokens that may have a count or a bias
    unsigned long long best[kMaxRows];
    unsigned short mine[kMaxTree];  // drafted tokens in this chunk, by node
    int n_mine;
};

// A float's bits in the order of the floats; 0 for NaN and -inf.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);  // -0 as +0
    return x > -INFINITY ? (b & 0x80000000u ? ~b : b | 0x80000000u) : 0u;
}

template <int CHUNK, int VEC>
__global__ void __launch_bounds__(kThreads) logits_kernel(const LogitParams a) {
    extern __shared__ __align__(16) unsigned char raw[];
    Shared<CHUNK>& sh = *reinterpret_cast<Shared<CHUNK>*>(raw);
    const int tid = threadIdx.x, lane = tid & 31;
    const int seq = blockIdx.z, v0 = blockIdx.x * CHUNK;
    const int i0 = blockIdx.y * a.rows_per_cta, n_rows = min(a.rows_per_cta, a.n_tree - i0);
    for (int i = tid; i < CHUNK; i += kThreads) {
        sh.count[i] = 0;
        sh.bias[i] = 0.0f;
        if (i < CHUNK / 32) sh.touched[i] = 0;
    }
    for (int i = tid; i < n_rows; i += kThreads) sh.best[i] = 0;
    if (tid == 0) sh.n_mine = 0;
    __syncthreads();
    pdl_launch_dependents();
    pdl_wait();

    auto touch = [&](int at) { atomicOr(&sh.touched[at >> 5], 1u << (at & 31)); };
    const int span = min(CHUNK, a.n_vocab - v0);
    if (a.history) {
        const int n = min(a.history_len[seq], a.history_ld);
        const int32_t* h = a.history + size_t(seq) * a.history_ld;
        for (int i = tid; i < n; i += 4 * kThreads) {
            int tok[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) tok[j] = i + j * kThreads < n ? __ldg(h + i + j * kThreads) : -1;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = tok[j] - v0;
                if (tok[j] >= v0 && at < span) {
                    atomicAdd(&sh.count[at], 1);
                    touch(at);
                }
            }
        }
    }
    if (a.bias_begin) {
        const int end = a.bias_begin[seq + 1];
        for (int i = a.bias_begin[seq] + tid; i < end; i += kThreads) {
            const int tok = a.bias_token[i];
            if (tok >= v0 && tok - v0 < span) {
                atomicAdd(&sh.bias[tok - v0], a.bias_value[i]);
                touch(tok - v0);
            }
        }
    }
    const int32_t* draft = a.draft ? a.draft + size_t(seq) * a.n_tree : nullptr;
    if (draft)
        for (int j = tid; j < a.n_tree; j += kThreads) {
            const int tok = draft[j];
            if (tok >= v0 && tok - v0 < span) {
                sh.mine[atomicAdd(&sh.n_mine, 1)] = static_cast<unsigned short>(j);
                touch(tok - v0);
            }
        }
    __syncthreads();
    const int n_mine = sh.n_mine;
    const int words = (a.n_tree + 31) / 32;
    const float repeat = a.penalties ? a.penalties[3 * seq] : 1.0f;
    const float presence = a.penalties ? a.penalties[3 * seq + 1] : 0.0f;
    const float frequency = a.penalties ? a.penalties[3 * seq + 2] : 0.0f;

    constexpr int kPer = CHUNK / (VEC * kThreads);  // vectors of a thread
    for (int i = 0; i < n_rows; ++i) {
        const int node = i0 + i;
        const size_t row = size_t(seq) * a.n_tree + node;
        auto path = [&](int sign) {
            for (int k = tid; k < n_mine; k += kThreads) {
                const int j = sh.mine[k];
                const bool on = a.mask ? a.mask[row * words + (j >> 5)] >> (j & 31) & 1u : j <= node;
                if (on) atomicAdd(&sh.count[draft[j] - v0], sign);
            }
            __syncthreads();
        };
        const float* x = a.x + row * a.ld + v0;
        float f[kPer][VEC];
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const int at = (k * kThreads + tid) * VEC;
            const bool whole = VEC == 4 && at + 3 < span;
            if constexpr (VEC == 4) {
                if (whole) {
                    const float4 v = *reinterpret_cast<const float4*>(x + at);
                    f[k][0] = v.x; f[k][1] = v.y; f[k][2] = v.z; f[k][3] = v.w;
                }
            }
            if (!whole)
#pragma unroll
                for (int e = 0; e < VEC; ++e) f[k][e] = at + e < span ? x[at + e] : -INFINITY;
        }
        if (n_mine) path(1);
        uint32_t top = 0;
        int top_at = 0;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const int at = (k * kThreads + tid) * VEC;
            if (at >= span) continue;
            const unsigned some = sh.touched[at >> 5] >> (at & 31);
            unsigned allowed = ~0u;
            if (a.allowed) allowed = __ldg(a.allowed + row * a.allowed_ld + ((v0 + at) >> 5)) >> (at & 31);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                if (some >> e & 1u) {
                    const int c = sh.count[at + e];
                    float y = f[k][e] + sh.bias[at + e];
                    if (c > 0) {
                        y = y > 0.0f ? __fdiv_rn(y, repeat) : y * repeat;
                        y -= float(c) * frequency + presence;
                    }
                    f[k][e] = y;
                }
                if (!(allowed >> e & 1u)) f[k][e] = -INFINITY;
                const uint32_t o = at + e < span ? ordered(f[k][e]) : 0u;
                if (o > top) {
                    top = o;
                    top_at = at + e;
                }
            }
            if (a.out) {
                float* y = a.out + row * a.out_ld + v0;
                const bool whole = VEC == 4 && at + 3 < span;
                if constexpr (VEC == 4) {
                    if (whole)
                        *reinterpret_cast<float4*>(y + at) = make_float4(f[k][0], f[k][1], f[k][2], f[k][3]);
                }
                if (!whole)
#pragma unroll
                    for (int e = 0; e < VEC; ++e)
                        if (at + e < span) y[at + e] = f[k][e];
            }
        }
        if (a.pick) {
            const uint32_t best = __reduce_max_sync(0xffffffffu, top);
            const uint32_t at = __reduce_min_sync(0xffffffffu, top == best ? uint32_t(v0 + top_at) : 0xffffffffu);
            if (lane == 0 && best) atomicMax(&sh.best[i], static_cast<unsigned long long>(best) << 32 | (0xffffffffu - at));
        }
        if (n_mine) {
            __syncthreads();
            path(-1);
        }
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
    if (x->bias_begin && (!x->bias_token || !x->bias_value)) return SYN_ERR_INVALID;
    if (x->pick && (!x->scratch || (reinterpret_cast<uintptr_t>(x->scratch) & 7))) return SYN_ERR_INVALID;
    a.penalties = x->penalties;
    a.history = x->history; a.history_len = x->history_len; a.history_ld = x->history_ld;
    a.draft = x->draft; a.mask = x->mask;
    a.bias_begin = x->bias_begin; a.bias_token = x->bias_token; a.bias_value = x->bias_value;
    a.allowed = x->allowed;
    const size_t rows = size_t(x->n_seq) * x->n_tree;
    a.key = static_cast<unsigned long long*>(x->scratch);
    a.arrived = x->scratch ? reinterpret_cast<unsigned*>(a.key + rows) : nullptr;
    a.n_tree = x->n_tree; a.n_vocab = x->n_vocab;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    // rows of 16-byte vectors where every row starts on a 16-byte boundary
    const uintptr_t at = reinterpret_cast<uintptr_t>(x->logits) | reinterpret_cast<uintptr_t>(x->out);
    const bool vec = (at & 15) == 0 && a.ld % 4 == 0 && (!x->out || a.out_ld % 4 == 0);
    // short chunks while the long ones would not give every SM two CTAs
    const bool few = rows * ((size_t(x->n_vocab) + 4095) / 4096) < size_t(2) * syn_num_sms();
    if (few) return vec ? launch<1024, 4>(a, x->n_seq, s) : launch<1024, 1>(a, x->n_seq, s);
    return vec ? launch<4096, 4>(a, x->n_seq, s) : launch<4096, 1>(a, x->n_seq, s);
}
