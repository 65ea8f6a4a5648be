// KV caches in F16, Q8_0 and Q4_0: rows appended (RoPE, quantisation, store),
// read back as values, and moved together after a tree of drafted tokens has
// been verified. All three move each byte once; they are bound by memory for
// long inputs and by the launch for a decode step's few rows.
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
    int n, n_head, table_len, blocks_per_head;
    int neox;
};

// Q4_0 of one block of 32 values, one per lane: d = (the value of largest
// magnitude, the first of equals) / -8, q = min(15, int(x / d + 8.5)); the
// quant and the scale's bits.
__device__ __forceinline__ int quantize_q4_lane(float x, uint16_t& dh) {
    const uint32_t a = __float_as_uint(fabsf(x));
    const uint32_t amax = __reduce_max_sync(0xffffffffu, a);
    const int first = __ffs(__ballot_sync(0xffffffffu, a == amax)) - 1;
    const float d = __fdiv_rn(__shfl_sync(0xffffffffu, x, first), -8.0f);
    dh = f16_bits(d);
    const float id = __fdiv_rn(1.0f, d);
    // a scale that rounds to zero stores zeros (and 1 / d may not be finite)
    return (dh & 0x7fff) ? min(15, int(__fadd_rn(__fmul_rn(x, id), 8.5f))) : 8;
}

// A warp takes blocks of 32 dims of a token's rows: n_head heads of q, then
// n_kv of K, then n_kv of V, blocks_per_head each; lane = dim.
template <int TYPE>
__global__ void __launch_bounds__(256) kv_append_kernel(AppendParams a) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int hd = a.c.hd, bph = a.blocks_per_head;
    const int heads = (a.q ? a.n_head : 0) + 2 * a.c.n_kv;
    const int tok = blockIdx.x;  // s * n + i
    const int slot = a.slot[tok];
    const int pos = a.pos ? a.pos[tok] : slot;
    if (slot < 0 || slot >= a.c.max_ctx) return;
    if (a.table && (pos < 0 || pos >= a.table_len)) return;
    const int s = tok / a.n;
    const int w0 = blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5), step = gridDim.y * (blockDim.x >> 5);
    for (int w = w0; w < heads * bph; w += step) {
        int h = w / bph;
        const int b = w - h * bph, dim = b * 32 + lane;
        const int nq = a.q ? a.n_head : 0;
        const int kind = h < nq ? 0 : h < nq + a.c.n_kv ? 1 : 2;  // q, K, V
        h -= kind == 0 ? 0 : kind == 1 ? nq : nq + a.c.n_kv;
        const float* row = kind == 0 ? a.q + size_t(tok) * a.q_stride : (kind == 1 ? a.k : a.v) + size_t(tok) * a.kv_stride;
        row += size_t(h) * hd;
        const bool in = dim < hd;
        float x = in ? row[dim] : 0.0f;
        if (kind != 2 && a.table) {
            const int half = hd / 2;
            const bool second = a.neox ? dim >= half : (dim & 1);
            const int other = a.neox ? (second ? dim - half : dim + half) : dim ^ 1;
            const int pair = a.neox ? (second ? dim - half : dim) : dim >> 1;
            if (in) {
                const float y = row[other];
                const float2 cs = __ldg(a.table + size_t(pos) * half + pair);
                // first: x c - y s; second: y s + x c (y is the first)
                x = second ? __fadd_rn(__fmul_rn(y, cs.y), __fmul_rn(x, cs.x))
                           : __fsub_rn(__fmul_rn(x, cs.x), __fmul_rn(y, cs.y));
            }
        }
        if (kind == 0) {
            if (in) a.q_out[(size_t(tok) * a.n_head + h) * hd + dim] = x;
            continue;
        }
        char* base = (kind == 1 ? a.c.k : a.c.v) + size_t(s) * a.c.seq_stride;
        if (TYPE == SYN_F16) {
            if (in) reinterpret_cast<uint16_t*>(base)[(size_t(slot) * a.c.n_kv + h) * hd + dim] = f16_bits(x);
            continue;
        }
        // quantised rows hold finite values only: clamped to binary16's range, NaN as 0
        x = x != x ? 0.0f : fminf(fmaxf(x, -65504.0f), 65504.0f);
        const size_t block = (size_t(h) * a.c.max_ctx + slot) * bph + b;
        uint16_t* scale = reinterpret_cast<uint16_t*>(base + a.c.scale_plane) + block;
        if (TYPE == SYN_Q8_0) {
            const float d = __fdiv_rn(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(x)))), 127.0f);
            const uint16_t dh = f16_bits(d);
            const int q = dh ? int(roundf(__fmul_rn(x, __fdiv_rn(1.0f, d)))) : 0;
            reinterpret_cast<int8_t*>(base)[block * 32 + lane] = int8_t(q);
            if (lane == 0) *scale = dh;
        } else {
            uint16_t dh;
            const int q = quantize_q4_lane(x, dh);
            const int hi = __shfl_down_sync(0xffffffffu, q, 16);
            if (lane < 16) reinterpret_cast<uint8_t*>(base)[block * 16 + lane] = uint8_t(q | (hi << 4));
            if (lane == 0) *scale = dh;
        }
    }
}

// ---- read back --------------------------------------------------------------------
struct ReadParams {
    KvView c;
    const int32_t* rows;
    void *k_out, *v_out;
    size_t items;  // units of all rows of K (V alike)
    int first, n, units, f16;
};

template <bool F16OUT>
__device__ __forceinline__ void store8(void* out, size_t at, const float (&f)[8]) {
    if (F16OUT) {
        uint32_t h[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = uint32_t(f16_bits(f[2 * e])) | uint32_t(f16_bits(f[2 * e + 1])) << 16;
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at) = make_uint4(h[0], h[1], h[2], h[3]);
    } else {
        float4* o = reinterpret_cast<float4*>(static_cast<float*>(out) + at);
        o[0] = make_float4(f[0], f[1], f[2], f[3]);
        o[1] = make_float4(f[4], f[5], f[6], f[7]);
    }
}

// A thread takes one unit of 8 values of a row: consecutive threads take the
// units of one (row, head), then the next heads of the row.
template <int TYPE, bool F16OUT>
__global__ void __launch_bounds__(256) kv_read_kernel(ReadParams a) {
    pdl_launch_dependents();
    pdl_wait();
    const int hd = a.c.hd, upr = hd / 8;
    const char* plane = blockIdx.y ? a.c.v : a.c.k;
    void* out = blockIdx.y ? a.v_out : a.k_out;
    for (size_t i = size_t(blockIdx.x) * blockDim.x + threadIdx.x; i < a.items; i += size_t(gridDim.x) * blockDim.x) {
        const int u = int(i % upr);
        const size_t rh = i / upr;
        const int h = int(rh % a.c.n_kv);
        const size_t r = rh / a.c.n_kv;  // s * n + row
        const int s = int(r / a.n);
        const int row = a.rows ? a.rows[r] : a.first + int(r - size_t(s) * a.n);
        float f[8] = {};
        if (row >= 0 && row < a.c.max_ctx) {
            const char* base = plane + size_t(s) * a.c.seq_stride;
            if (TYPE == SYN_F16) {
                const uint4 x = __ldg(reinterpret_cast<const uint4*>(base + ((size_t(row) * a.c.n_kv + h) * hd + u * 8) * 2));
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    f[2 * e] = f16_from_bits(uint16_t(w[e]));
                    f[2 * e + 1] = f16_from_bits(uint16_t(w[e] >> 16));
                }
            } else {
                const int b = u >> 2, part = u & 3;
                const size_t block = (size_t(h) * a.c.max_ctx + row) * (hd / QK) + b;
                const float d = f16_from_bits(__ldg(reinterpret_cast<const uint16_t*>(base + a.c.scale_plane) + block));
                // Q4_0: values 0-15 are the block's low nibbles, 16-31 the high ones
                const uint2 x = __ldg(reinterpret_cast<const uint2*>(
                    base + (TYPE == SYN_Q8_0 ? block * 32 + part * 8 : block * 16 + (part & 1) * 8)));
                const uint32_t w[2] = {x.x, x.y};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t byte = w[e >> 2] >> (8 * (e & 3)) & 255u;
                    const int q = TYPE == SYN_Q8_0 ? int(int8_t(byte)) : int(part < 2 ? byte & 15u : byte >> 4) - 8;
                    f[e] = __fmul_rn(float(q), d);
                }
            }
        }
        store8<F16OUT>(out, i * 8, f);
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
    const int n = min(a.count[s], a.path_ld), begin = a.begin[s];
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
    a.blocks_per_head = (c->head_dim + 31) / 32;
    a.neox = x->rope_mode;
    const size_t tokens = size_t(c->n_seq) * x->n;
    if (tokens > 0x7fffffff) return SYN_ERR_UNSUPPORTED;
    const int tasks = (a.n_head + 2 * c->n_kv) * a.blocks_per_head;
    // few tokens: a warp per task; many: a CTA of 8 warps per token
    const unsigned y = tokens < 64 ? unsigned((tasks + 7) / 8) : 1u;
    const dim3 grid{unsigned(tokens), y, 1};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (c->type == SYN_F16) return syn_launch(kv_append_kernel<SYN_F16>, grid, 256, 0, s, a);
    if (c->type == SYN_Q8_0) return syn_launch(kv_append_kernel<SYN_Q8_0>, grid, 256, 0, s, a);
    return syn_launch(kv_append_kernel<SYN_Q4_0>, grid, 256, 0, s, a);
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
    if (!k_out) a.c.k = a.c.v;  // one output: plane 0 is V
    a.k_out = k_out ? k_out : v_out;
    a.v_out = v_out;
    a.rows = rows; a.first = first; a.n = n;
    a.items = size_t(c->n_seq) * n * c->n_kv * (c->head_dim / 8);
    const size_t blocks = (a.items + 255) / 256;
    const dim3 grid{unsigned(blocks < 0x7fffffff ? blocks : 0x7fffffff), k_out && v_out ? 2u : 1u, 1};
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
