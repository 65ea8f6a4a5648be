// KV caches in F16, Q8_0 and Q4_0: rows appended (RoPE, quantisation, store),
// read back as values, and moved together after a tree of drafted tokens has
// been verified. All three move each byte once; they are bound by memory for
// long inputs and by the launch for a decode step's few rows.
// Measured with 32 query and 8 KV heads of 128, against the copy rate of 6.5
// TB/s: 8192 tokens appended to an F16 cache in 66 us (86 %), to Q8_0 in 73 (74
// %: the divisions and roundings of a block are the rest), one token in 1.9 us;
// 32768 rows read as binary16 in 42 us from Q8_0 (75 %) and in 45 from F16 (92
// %), as floats from Q8_0 in 71 (73 %). Of append, a load of the next quad ahead
// of the work cost 14 % (registers: fewer CTAs on an SM).
#include "kv_cache.cuh"

using namespace syn;

namespace {

// ---- append -------------------------------------------------------------------
struct AppendParams {
    KvView c;
    const float *k, *v, *q;
    float* q_out;
    const int32_t *slot, *pos;
    const float2* table;
    size_t kv_stride, q_stride;
    int n, n_head, table_len;
    int neox;
};

// A thread takes 4 dims of a token's rows: n_head heads of q, then n_kv of K,
// then n_kv of V; 8 neighbouring lanes hold a block of 32. VEC: rows and
// strides allow 16-byte loads.
template <int TYPE, bool VEC, int THREADS = 256>
__global__ void __launch_bounds__(THREADS) kv_append_kernel(AppendParams a) {
    pdl_launch_dependents();
    pdl_wait();
    const int hd = a.c.hd, quads = hd / 4, half = hd / 2;
    const int nq = a.q ? a.n_head : 0, heads = nq + 2 * a.c.n_kv;
    const int tok = blockIdx.x;  // s * n + i
    const int slot = a.slot[tok];
    const int pos = a.pos ? a.pos[tok] : slot;
    if (slot < 0 || slot >= a.c.max_ctx) return;
    if (a.table && (pos < 0 || pos >= a.table_len)) return;
    const int s = tok / a.n, lane = threadIdx.x & 31;
    auto load4 = [](const float* p) {
        if (VEC) return *reinterpret_cast<const float4*>(p);
        return make_float4(p[0], p[1], p[2], p[3]);
    };
    const float2* cs = a.table ? a.table + size_t(pos) * half : nullptr;
    const int n = heads * quads;
    for (int w = blockIdx.y * blockDim.x + (threadIdx.x & ~31); w < n; w += gridDim.y * blockDim.x) {
        const int id = min(w + lane, n - 1);  // the last warp's spare lanes repeat the last quad and store nothing
        const bool in = w + lane < n;
        int h = id / quads;
        const int d = (id - h * quads) * 4;
        const int kind = h < nq ? 0 : h < nq + a.c.n_kv ? 1 : 2;  // q, K, V
        h -= kind == 0 ? 0 : kind == 1 ? nq : nq + a.c.n_kv;
        const float* row = kind == 0 ? a.q + size_t(tok) * a.q_stride : (kind == 1 ? a.k : a.v) + size_t(tok) * a.kv_stride;
        row += size_t(h) * hd;
        const float4 v = load4(row + d);
        float x[4] = {v.x, v.y, v.z, v.w};
        if (kind != 2 && cs) {
            if (a.neox) {  // pairs (i, i + hd / 2)
                const bool second = d >= half;
                const float4 o = load4(row + (second ? d - half : d + half));
                const float y[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 t = __ldg(cs + (second ? d - half : d) + e);
                    x[e] = second ? __fadd_rn(__fmul_rn(y[e], t.y), __fmul_rn(x[e], t.x))
                                  : __fsub_rn(__fmul_rn(x[e], t.x), __fmul_rn(y[e], t.y));
                }
            } else {  // pairs (2 i, 2 i + 1)
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const float2 t = __ldg(cs + (d + e) / 2);
                    const float y = x[e];
                    x[e] = __fsub_rn(__fmul_rn(y, t.x), __fmul_rn(x[e + 1], t.y));
                    x[e + 1] = __fadd_rn(__fmul_rn(y, t.y), __fmul_rn(x[e + 1], t.x));
                }
            }
        }
        char* base = (kind == 1 ? a.c.k : a.c.v) + size_t(s) * a.c.seq_stride;
        if (kind == 0) {
            if (in) *reinterpret_cast<float4*>(a.q_out + (size_t(tok) * a.n_head + h) * hd + d) = make_float4(x[0], x[1], x[2], x[3]);
        } else if (TYPE == SYN_F16) {
            const uint2 bits = make_uint2(uint32_t(f16_bits(x[0])) | uint32_t(f16_bits(x[1])) << 16,
                                          uint32_t(f16_bits(x[2])) | uint32_t(f16_bits(x[3])) << 16);
            if (in) *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(base) + (size_t(slot) * a.c.n_kv + h) * hd + d) = bits;
        }
        if (TYPE == SYN_F16 || __all_sync(0xffffffffu, kind == 0)) continue;
        // quantised rows hold finite values only: clamped to binary16's range, NaN as 0
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] = x[e] != x[e] ? 0.0f : fminf(fmaxf(x[e], -65504.0f), 65504.0f);
            top = max(top, __float_as_uint(fabsf(x[e])));
        }
        const uint32_t mine = top;
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const size_t block = (size_t(h) * a.c.max_ctx + slot) * (hd / QK) + d / QK;
        uint16_t* scale = reinterpret_cast<uint16_t*>(base + a.c.scale_plane) + block;
        if (TYPE == SYN_Q8_0) {
            const float dd = __fdiv_rn(__uint_as_float(top), 127.0f), id8 = __fdiv_rn(1.0f, dd);
            const uint16_t dh = min(f16_bits(dd), uint16_t(0x6007));  // 515.5: 127 times the next, 516, is beyond binary16
            uint32_t word = 0;  // a scale that rounds to zero stores zeros (and 1 / d may not be finite)
#pragma unroll
            for (int e = 0; e < 4; ++e) word |= (dh ? uint32_t(int(roundf(__fmul_rn(x[e], id8)))) & 255u : 0u) << (8 * e);
            if (in && kind != 0) {
                *reinterpret_cast<uint32_t*>(base + block * 32 + (d & 31)) = word;
                if ((lane & 7) == 0) *scale = dh;
            }
        } else {
            // d = (the value of largest magnitude, the first of equals) / -8, q = min(15, int(x / d + 8.5))
            float first = 0.0f;
#pragma unroll
            for (int e = 3; e >= 0; --e)
                if (__float_as_uint(fabsf(x[e])) == top) first = x[e];
            const unsigned who = __ballot_sync(0xffffffffu, mine == top) >> (lane & 24) & 255u;
            first = __shfl_sync(0xffffffffu, first, (lane & 24) + __ffs(who) - 1);
            const float dd = __fdiv_rn(first, -8.0f), id4 = __fdiv_rn(1.0f, dd);
            const uint16_t dh = f16_bits(dd);
            uint32_t word = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                word |= uint32_t((dh & 0x7fff) ? min(15, int(__fadd_rn(__fmul_rn(x[e], id4), 8.5f))) : 8) << (8 * e);
            const uint32_t high = __shfl_down_sync(0xffffffffu, word, 4);
            if (in && kind != 0 && (lane & 4) == 0) *reinterpret_cast<uint32_t*>(base + block * 16 + (d & 15)) = word | high << 4;
            if (in && kind != 0 && (lane & 7) == 0) *scale = dh;
        }
    }
}

// ---- read back --------------------------------------------------------------------
struct ReadParams {
    KvView c;
    const int32_t* rows;
    void *k_out, *v_out;
    int first, n, units;
};

constexpr int kReadRows = 4;  // rows of a thread, loaded together

// A CTA takes kReadRows * (256 / units) rows of one head of K or V of a
// sequence; a thread one unit (16 bytes of the output: 8 or 4 values) of
// kReadRows of them, so that a warp's stores are whole lines.
template <int TYPE, bool F16OUT>
__global__ void __launch_bounds__(256) kv_read_kernel(ReadParams a) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int V = F16OUT ? 8 : 4;
    const int hd = a.c.hd, h = blockIdx.y, s = blockIdx.z >> 1;
    const char* base = ((blockIdx.z & 1) ? a.c.v : a.c.k) + size_t(s) * a.c.seq_stride;
    void* out = (blockIdx.z & 1) ? a.v_out : a.k_out;
    const int per = 256 / a.units, r0 = threadIdx.x / a.units, u = threadIdx.x - r0 * a.units;
    if (!out || r0 >= per) return;
    const int i0 = blockIdx.x * per * kReadRows + r0;
    uint32_t x[kReadRows][V / (TYPE == SYN_F16 ? 2 : 4)];
    uint16_t d[kReadRows];
    auto load = [](auto& to, const char* p) {
        constexpr int n = sizeof(to) / 4;
        if constexpr (n == 4) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
            to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w;
        } else if constexpr (n == 2) {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
            to[0] = v.x; to[1] = v.y;
        } else {
            to[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
        }
    };
#pragma unroll
    for (int j = 0; j < kReadRows; ++j) {
        const int i = i0 + j * per;
        const int row = i >= a.n ? -1 : a.rows ? __ldg(a.rows + size_t(s) * a.n + i) : a.first + i;
        d[j] = 0;  // with a scale of 0 any quants are 0
#pragma unroll
        for (auto& w : x[j]) w = 0;
        if (row < 0 || row >= a.c.max_ctx) continue;
        if (TYPE == SYN_F16) {
            load(x[j], base + ((size_t(row) * a.c.n_kv + h) * hd + u * V) * 2);
        } else {
            const size_t block = (size_t(h) * a.c.max_ctx + row) * (hd / QK) + u * V / QK;
            const int in = u * V % QK;  // Q4_0: byte j of a block holds values j and j + 16
            load(x[j], base + (TYPE == SYN_Q8_0 ? block * 32 + in : block * 16 + in % 16));
            d[j] = __ldg(reinterpret_cast<const uint16_t*>(base + a.c.scale_plane) + block);
        }
    }
    const bool high = TYPE == SYN_Q4_0 && u * V % QK >= 16;
#pragma unroll
    for (int j = 0; j < kReadRows; ++j) {
        const int i = i0 + j * per;
        if (i >= a.n) continue;
        const size_t at = ((size_t(s) * a.n + i) * a.c.n_kv + h) * hd + u * V;
        const float scale = f16_from_bits(d[j]);
        float f[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (TYPE == SYN_F16) {
                f[e] = f16_from_bits(uint16_t(x[j][e >> 1] >> (16 * (e & 1))));
            } else {
                const uint32_t byte = x[j][e >> 2] >> (8 * (e & 3));
                const int q = TYPE == SYN_Q8_0 ? int(int8_t(byte)) : int((high ? byte >> 4 : byte) & 15u) - 8;
                f[e] = __fmul_rn(float(q), scale);
            }
        }
        if constexpr (F16OUT) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = uint32_t(f16_bits(f[2 * e])) | uint32_t(f16_bits(f[2 * e + 1])) << 16;
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            *reinterpret_cast<float4*>(static_cast<float*>(out) + at) = make_float4(f[0], f[1], f[2], f[3]);
        }
    }
}

// ---- move ---------------------------------------------------------------------------
struct MoveParams {
    KvView c;
    size_t layer_stride;
    const int32_t *path, *count, *begin;
    int path_ld, cols16, cols2;  // 16-byte columns of a row, then the 2-byte ones (scales)
    int rows16, rows2;           // columns of one head's row (quantised types)
};

constexpr int kMoveBatch = 8;

// One column of every row, in path order. A batch is read whole before it is
// written: row begin + i is written no earlier than row path[j] = begin + i,
// j <= i, was read, since the path ascends from begin.
template <typename T>
__device__ __forceinline__ void move_column(T* col, size_t pitch, const int32_t* path, int n, int begin, int max_ctx) {
    for (int i0 = 0; i0 < n; i0 += kMoveBatch) {
        T x[kMoveBatch];
        bool ok[kMoveBatch];
#pragma unroll
        for (int j = 0; j < kMoveBatch; ++j) {
            const int i = i0 + j, src = i < n ? path[i] : -1;
            ok[j] = src >= 0 && src < max_ctx && begin + i >= 0 && begin + i < max_ctx && src != begin + i;
            if (ok[j]) x[j] = col[size_t(src) * pitch];
        }
#pragma unroll
        for (int j = 0; j < kMoveBatch; ++j)
            if (ok[j]) col[size_t(begin + i0 + j) * pitch] = x[j];
    }
}

template <int TYPE>
__global__ void __launch_bounds__(128) kv_move_kernel(MoveParams a) {
    pdl_launch_dependents();
    pdl_wait();
    const int s = blockIdx.y, layer = blockIdx.z >> 1;
    char* base = ((blockIdx.z & 1) ? a.c.v : a.c.k) + size_t(layer) * a.layer_stride + size_t(s) * a.c.seq_stride;
    // from past the cache or n and more before it no row is moved: begin + i stays an int
    const int n = min(a.count[s], a.path_ld), begin = min(max(a.begin[s], -max(n, 0)), a.c.max_ctx);
    const int32_t* path = a.path + size_t(s) * a.path_ld;
    int col = blockIdx.x * blockDim.x + threadIdx.x;
    if (col < a.cols16) {
        uint4* p = reinterpret_cast<uint4*>(base);
        if (TYPE == SYN_F16) {
            move_column(p + col, a.cols16, path, n, begin, a.c.max_ctx);
        } else {
            const int h = col / a.rows16, x = col - h * a.rows16;
            move_column(p + size_t(h) * a.c.max_ctx * a.rows16 + x, a.rows16, path, n, begin, a.c.max_ctx);
        }
    } else if (col < a.cols16 + a.cols2) {
        col -= a.cols16;
        const int h = col / a.rows2, x = col - h * a.rows2;
        uint16_t* p = reinterpret_cast<uint16_t*>(base + a.c.scale_plane);
        move_column(p + size_t(h) * a.c.max_ctx * a.rows2 + x, a.rows2, path, n, begin, a.c.max_ctx);
    }
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace

extern "C" size_t syn_kv_cache_bytes(int type, int n_kv, int head_dim, int max_ctx) {
    if (!kv_type(type) || n_kv <= 0 || head_dim <= 0 || max_ctx <= 0 || head_dim > 256) return 0;
    if (head_dim % (type == SYN_F16 ? 8 : QK)) return 0;
    const size_t rows = size_t(n_kv) * max_ctx;
    if (type == SYN_F16) return rows * head_dim * 2;
    return kv_quant_plane(type, n_kv, head_dim, max_ctx) + align256(rows * (head_dim / QK) * 2);
}

extern "C" int syn_kv_append(const syn_kv_cache* c, int layer, const syn_kv_append_args* x, void* stream) {
    int st = kv_check(c, layer);
    if (st) return st;
    if (!x || !x->k || !x->v || !x->slot || x->n <= 0) return SYN_ERR_INVALID;
    if (x->q && (!x->q_out || x->n_head <= 0)) return SYN_ERR_INVALID;
    if (x->rope_mode != 0 && x->rope_mode != 1) return SYN_ERR_INVALID;
    if (x->rope_table && (x->table_len <= 0 || !aligned(x->rope_table, 8))) return SYN_ERR_INVALID;
    const size_t row = size_t(c->n_kv) * c->head_dim, q_row = size_t(x->n_head) * c->head_dim;
    AppendParams a{};
    a.c = kv_view(c, layer);
    a.k = x->k; a.v = x->v; a.q = x->q; a.q_out = x->q_out;
    a.slot = x->slot; a.pos = x->pos;
    a.table = reinterpret_cast<const float2*>(x->rope_table);
    a.kv_stride = x->kv_stride ? x->kv_stride : row;
    a.q_stride = x->q_stride ? x->q_stride : q_row;
    if (a.kv_stride < row || (x->q && a.q_stride < q_row)) return SYN_ERR_INVALID;
    if (x->q && x->q == x->q_out) return SYN_ERR_INVALID;  // pairs read each other's element
    a.n = x->n; a.n_head = x->q ? x->n_head : 0;
    a.table_len = x->table_len;
    a.neox = x->rope_mode;
    const size_t tokens = size_t(c->n_seq) * x->n;
    if (tokens > 0x7fffffff) return SYN_ERR_UNSUPPORTED;
    const int quads = (a.n_head + 2 * c->n_kv) * (c->head_dim / 4);
    // Few tokens: a thread per quad; many: a CTA per token. Measured, F16, the one / the other, us: 1 token 1.8 / 3.5,
    // 192 3.7 / 4.2, 256 4.5 / 4.2, 2048 25.0 / 18.5.
    const unsigned y = tokens < 256 ? unsigned((quads + 255) / 256) : 1u;
    const dim3 grid{unsigned(tokens), y, 1};
    const bool vec = aligned(x->k, 16) && aligned(x->v, 16) && aligned(x->q, 16) && a.kv_stride % 4 == 0 && a.q_stride % 4 == 0;
    if (x->q && !aligned(x->q_out, 16)) return SYN_ERR_INVALID;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (c->type == SYN_F16)
        return vec ? syn_launch(kv_append_kernel<SYN_F16, true>, grid, 256, 0, s, a) : syn_launch(kv_append_kernel<SYN_F16, false>, grid, 256, 0, s, a);
    // Q8_0's CTAs of 128 threads pay once there are more than an SM has room for at a time. Measured, 256 / 128 threads, us:
    // 512 tokens 7.5 / 9.3, 2048 23.6 / 22.0, 8192 81.5 / 73.1 (F16 65.9 / 65.1, Q4_0 75.9 / 80.5).
    if (c->type == SYN_Q8_0 && tokens > size_t(8) * syn_num_sms())
        return vec ? syn_launch(kv_append_kernel<SYN_Q8_0, true, 128>, grid, 128, 0, s, a) : syn_launch(kv_append_kernel<SYN_Q8_0, false, 128>, grid, 128, 0, s, a);
    if (c->type == SYN_Q8_0)
        return vec ? syn_launch(kv_append_kernel<SYN_Q8_0, true>, grid, 256, 0, s, a) : syn_launch(kv_append_kernel<SYN_Q8_0, false>, grid, 256, 0, s, a);
    return vec ? syn_launch(kv_append_kernel<SYN_Q4_0, true>, grid, 256, 0, s, a) : syn_launch(kv_append_kernel<SYN_Q4_0, false>, grid, 256, 0, s, a);
}

extern "C" int syn_kv_read(const syn_kv_cache* c, int layer, const int32_t* rows, int first, int n, int out_type,
                           void* k_out, void* v_out, void* stream) {
    int st = kv_check(c, layer);
    if (st) return st;
    if (n <= 0 || (!k_out && !v_out)) return SYN_ERR_INVALID;
    if (!rows && first < 0) return SYN_ERR_INVALID;
    if (out_type != SYN_F32 && out_type != SYN_F16) return SYN_ERR_UNSUPPORTED;
    if (!aligned(k_out, 16) || !aligned(v_out, 16)) return SYN_ERR_INVALID;
    ReadParams a{};
    a.c = kv_view(c, layer);
    a.k_out = k_out;
    a.v_out = v_out;
    a.rows = rows; a.first = first; a.n = n;
    a.units = c->head_dim / (out_type == SYN_F16 ? 8 : 4);
    const int per = 256 / a.units * kReadRows;
    if (c->n_kv > 65535 || c->n_seq > 32767) return SYN_ERR_UNSUPPORTED;
    const dim3 grid{unsigned((size_t(n) + per - 1) / per), unsigned(c->n_kv), unsigned(2 * c->n_seq)};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool h = out_type == SYN_F16;
    switch (c->type) {
    case SYN_F16:
        return h ? syn_launch(kv_read_kernel<SYN_F16, true>, grid, 256, 0, s, a)
                 : syn_launch(kv_read_kernel<SYN_F16, false>, grid, 256, 0, s, a);
    case SYN_Q8_0:
        return h ? syn_launch(kv_read_kernel<SYN_Q8_0, true>, grid, 256, 0, s, a)
                 : syn_launch(kv_read_kernel<SYN_Q8_0, false>, grid, 256, 0, s, a);
    default:
        return h ? syn_launch(kv_read_kernel<SYN_Q4_0, true>, grid, 256, 0, s, a)
                 : syn_launch(kv_read_kernel<SYN_Q4_0, false>, grid, 256, 0, s, a);
    }
}

extern "C" int syn_kv_move(const syn_kv_cache* c, const int32_t* path, int path_ld, const int32_t* count,
                           const int32_t* begin, void* stream) {
    int st = kv_check(c, 0);
    if (st) return st;
    if (!path || !count || !begin || path_ld <= 0) return SYN_ERR_INVALID;
    if (c->n_seq > 65535 || c->n_layer > 32767) return SYN_ERR_UNSUPPORTED;
    MoveParams a{};
    a.c = kv_view(c, 0);
    a.layer_stride = c->layer_stride;
    a.path = path; a.count = count; a.begin = begin; a.path_ld = path_ld;
    if (c->type == SYN_F16) {
        a.cols16 = c->n_kv * c->head_dim / 8;
    } else {
        a.rows16 = c->head_dim / QK * kv_block_bytes(c->type) / 16;
        a.rows2 = c->head_dim / QK;
        a.cols16 = c->n_kv * a.rows16;
        a.cols2 = c->n_kv * a.rows2;
    }
    const dim3 grid{unsigned((a.cols16 + a.cols2 + 127) / 128), unsigned(c->n_seq), unsigned(2 * c->n_layer)};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (c->type == SYN_F16) return syn_launch(kv_move_kernel<SYN_F16>, grid, 128, 0, s, a);
    if (c->type == SYN_Q8_0) return syn_launch(kv_move_kernel<SYN_Q8_0>, grid, 128, 0, s, a);
    return syn_launch(kv_move_kernel<SYN_Q4_0>, grid, 128, 0, s, a);
}
