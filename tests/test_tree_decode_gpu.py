"""KV caches in F16 / Q8_0 / Q4_0, attention of token trees over them, and logit processing, against plain
implementations in 64 bits (the quantised rows against the oracle's quantisers, bit for bit).

Tolerance of the attention (derived, per output): a score s = scale * sum q_d k_d is summed in float over at most
hd / 8 tensor-core products with an error of at most 2^-23 of the sum of magnitudes S each, q has 22 bits, and the
exponential 2^-22; a relative error e of every probability moves an output by at most 2 e max|v|; the sum over L
positions adds one rounding of 2^-23 max|v| for each product of 16 positions and its two terms. So
    |out - exact| <= (2 (hd / 8 + 8) 2^-23 S + (L / 8 + 64) 2^-23) max|v|.
As a whole the roundings are independent, and the relative 2-norm stays under 1e-5.
"""
import ctypes
import math

import numpy as np
import pytest

import oracle as orc

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
syn = pytest.importorskip("synapse_b200")

TYPES = [syn.F16, syn.Q8_0, syn.Q4_0]
SHAPES = [(32, 8, 128), (4, 2, 32), (6, 6, 64), (5, 1, 96), (16, 2, 256), (40, 8, 128)]


def gpu(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).cuda()


def blocks(x, type_):
    """The oracle's GGUF blocks of rows x [rows][dims]: (quants as bytes [rows][..], scale bits [rows][dims / 32])."""
    size = 18 if type_ == syn.Q4_0 else 34
    b = orc.quantize_weights(np.ascontiguousarray(x, np.float32), type_).reshape(x.shape[0], -1, size)
    return np.ascontiguousarray(b[..., 2:]).reshape(x.shape[0], -1), np.ascontiguousarray(b[..., :2]).view(np.uint16)[..., 0]


def planes(cache, which, layer=0):
    """Host views of a cache: F16 bits [n_seq][ctx][n_kv][hd], or (quant bytes, scale bits) [n_seq][n_kv][ctx][...]."""
    raw = (cache.k if which == 0 else cache.v)[layer].cpu().numpy()
    n, kv, hd, ctx = cache.n_seq, cache.n_kv, cache.head_dim, cache.max_ctx
    if cache.type == syn.F16:
        return np.ascontiguousarray(raw[:, :ctx * kv * hd * 2]).view(np.uint16).reshape(n, ctx, kv, hd)
    size = kv * ctx * hd // (1 if cache.type == syn.Q8_0 else 2)
    at = (size + 255) // 256 * 256
    scales = np.ascontiguousarray(raw[:, at:at + kv * ctx * hd // 16])
    return raw[:, :size].reshape(n, kv, ctx, -1), scales.view(np.uint16).reshape(n, kv, ctx, hd // 32)


def values(cache, which, layer=0):
    """A cache's values in 64 bits, [n_seq][ctx][n_kv][hd]."""
    p = planes(cache, which, layer)
    if cache.type == syn.F16:
        return p.view(np.float16).astype(np.float64)
    q, d = p
    d = d.view(np.float16).astype(np.float64)[..., None]
    if cache.type == syn.Q8_0:
        q = q.view(np.int8).astype(np.float64).reshape(*q.shape[:3], -1, 32)
    else:
        b = q.reshape(*q.shape[:3], -1, 16)
        q = np.concatenate([b & 15, b >> 4], -1).astype(np.float64) - 8
    return np.swapaxes((q * d).reshape(*q.shape[:3], -1), 1, 2)


def new_cache(type_, n_seq, n_kv, hd, ctx, n_layer=1):
    return syn.KVCache(type_, n_layer, n_seq, n_kv, hd, ctx)


def fill(cache, rng, rows, sigma=1.0, layer=0):
    """Rows 0 .. rows - 1 of every sequence appended from normal values."""
    n, w = cache.n_seq, cache.n_kv * cache.head_dim
    k = rng.standard_normal((n * rows, w), dtype=np.float32) * np.float32(sigma)
    v = rng.standard_normal((n * rows, w), dtype=np.float32) * np.float32(sigma)
    slot = np.tile(np.arange(rows, dtype=np.int32), n)
    syn.kv_append(cache, gpu(k), gpu(v), gpu(slot), layer=layer)
    return k, v


# ---- append -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("type_", [syn.Q8_0, syn.Q4_0])
@pytest.mark.parametrize("n_kv,hd,n_seq,n", [(8, 128, 1, 1), (2, 32, 3, 5), (1, 96, 2, 1), (2, 256, 1, 67)])
def test_append_quantises_as_the_oracle_bit_for_bit(type_, n_kv, hd, n_seq, n):
    rng = np.random.default_rng(hd + n)
    ctx = n + 9
    cache = new_cache(type_, n_seq, n_kv, hd, ctx, n_layer=2)
    k, v = (rng.standard_normal((n_seq * n, n_kv * hd), dtype=np.float32) for _ in "kv")
    k[0, :32] = 0.0
    k[0, 40 % (n_kv * hd)] = -50.0
    slot = np.concatenate([rng.permutation(ctx)[:n] for _ in range(n_seq)]).astype(np.int32)
    syn.kv_append(cache, gpu(k), gpu(v), gpu(slot), layer=1)
    for which, x in ((0, k), (1, v)):
        q, d = planes(cache, which, 1)
        wq, wd = blocks(x.reshape(-1, hd), type_)
        for i in range(n_seq * n):
            s = i // n
            for h in range(n_kv):
                assert np.array_equal(d[s, h, slot[i]], wd[i * n_kv + h])
                assert np.array_equal(q[s, h, slot[i]], wq[i * n_kv + h])
        assert not planes(cache, which, 0)[0].any()  # the other layer is untouched


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("mode", [0, 1])
@pytest.mark.parametrize("n_head,n_kv,hd", [(8, 2, 128), (3, 3, 32), (5, 1, 96)])
def test_append_rotates_as_rope(type_, mode, n_head, n_kv, hd):
    rng = np.random.default_rng(hd + mode)
    n, ctx = 7, 300
    theta = 10000.0 ** (-2.0 / hd)
    table = syn.rope_table(ctx, hd, theta)
    fused = gpu(rng.standard_normal((n, (n_head + 2 * n_kv) * hd), dtype=np.float32))  # rows of [q | k | v]
    q, k, v = fused.split([n_head * hd, n_kv * hd, n_kv * hd], 1)
    pos = gpu(np.array([0, 1, 2, 2, 3, 299, 17], np.int32))
    slot = gpu(np.arange(n, dtype=np.int32) + 3)
    cache, plain = new_cache(type_, 1, n_kv, hd, ctx), new_cache(type_, 1, n_kv, hd, ctx)
    out = syn.kv_append(cache, k, v, slot, pos=pos, rope_table=table, rope_mode=mode, q=q)
    assert torch.equal(out, syn.rope(q, pos, n_head, hd, theta, rope_mode=mode).view_as(out))
    syn.kv_append(plain, syn.rope(k, pos, n_kv, hd, theta, rope_mode=mode).view(n, -1), v.contiguous(), slot)
    assert torch.equal(cache.k, plain.k) and torch.equal(cache.v, plain.v)


def test_append_f16_is_the_sessions_cache():
    """The F16 layout is the one syn_rope_kv_append and syn_attention use."""
    rng = np.random.default_rng(5)
    n, n_kv, hd, ctx = 6, 4, 128, 32
    theta = 500000.0 ** (-2.0 / hd)
    k, v = (gpu(rng.standard_normal((n, n_kv * hd), dtype=np.float32)) for _ in "kv")
    pos = gpu(np.arange(n, dtype=np.int32) + 4)
    cache = new_cache(syn.F16, 1, n_kv, hd, ctx)
    syn.kv_append(cache, k, v, pos, rope_table=syn.rope_table(ctx, hd, theta))
    kc, vc = (torch.zeros(ctx * n_kv * hd, dtype=torch.int16, device="cuda") for _ in "kv")
    syn.rope_kv_append(k, v, kc, vc, pos, n_kv, hd, ctx, theta)
    assert torch.equal(cache.k.view(torch.int16).flatten(), kc) and torch.equal(cache.v.view(torch.int16).flatten(), vc)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("n_head,n_kv,hd", [(8, 2, 128), (5, 1, 96)])
def test_append_of_many_tokens_is_that_of_few(type_, n_head, n_kv, hd):
    """One call for 1500 tokens and calls of 100: the same bytes and the same rotated queries."""
    rng = np.random.default_rng(2)
    n = 1500
    q, k, v = (gpu(rng.standard_normal((n, h * hd), dtype=np.float32)) for h in (n_head, n_kv, n_kv))
    slot = gpu(rng.permutation(n).astype(np.int32))
    table = syn.rope_table(n, hd, 10000.0 ** (-2 / hd))
    one, many = new_cache(type_, 1, n_kv, hd, n), new_cache(type_, 1, n_kv, hd, n)
    whole = syn.kv_append(one, k, v, slot, rope_table=table, q=q)
    for i in range(0, n, 100):
        part = slice(i, i + 100)
        got = syn.kv_append(many, k[part], v[part], slot[part], rope_table=table, q=q[part])
        assert torch.equal(got, whole[part])
    assert torch.equal(one.k, many.k) and torch.equal(one.v, many.v)


@pytest.mark.parametrize("type_", [syn.Q8_0, syn.Q4_0])
def test_append_stores_finite_values_and_skips_bad_rows(type_):
    hd, ctx = 64, 8
    cache = new_cache(type_, 1, 1, hd, ctx)
    k = np.ones((4, hd), np.float32)
    k[0, 3], k[0, 40], k[1, 5] = np.inf, -np.inf, np.nan
    k[2] = 1e-30  # a scale that rounds to zero
    slot = gpu(np.array([0, 1, 2, 8], np.int32))  # the last is outside
    q = gpu(np.ones((4, hd), np.float32))
    table = syn.rope_table(3, hd, 0.9)
    before = cache.k.clone()
    out = syn.kv_append(cache, gpu(k), gpu(k), slot, q=q)
    x = values(cache, 0)[0, :, 0]
    assert np.isfinite(x).all() and not x[2].any() and not x[3:].any()
    assert 0.99 * 65504 <= x[0, 3] <= 1.01 * 65504 and -1.01 * 65504 <= x[0, 40] <= -0.99 * 65504
    assert x[1, 5] == 0 and abs(x[1, 6] - 1) < 0.01
    assert torch.equal(out[:3], q[:3])
    cache.k.copy_(before)
    syn.kv_append(cache, gpu(k), gpu(k), slot, pos=gpu(np.array([3, -1, 5, 0], np.int32)), rope_table=table)
    assert torch.equal(cache.k, before)  # positions outside the table, a slot outside the cache


# ---- read -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("n_kv,hd,n_seq", [(8, 128, 1), (2, 32, 3), (1, 96, 2), (3, 256, 2)])
def test_read_gives_the_stored_values(type_, dtype, n_kv, hd, n_seq):
    rng = np.random.default_rng(hd)
    ctx = 77
    cache = new_cache(type_, n_seq, n_kv, hd, ctx)
    fill(cache, rng, ctx)
    rows = rng.integers(-2, ctx + 2, (n_seq, 19)).astype(np.int32)
    rows[0, :2] = [-1, ctx]
    k, v = syn.kv_read(cache, 19, rows=gpu(rows), dtype=dtype)
    k2, v2 = syn.kv_read(cache, 40, first=33, dtype=dtype)  # runs past the cache's end? 33 + 40 < 77
    k3, _ = syn.kv_read(cache, 10, first=70, dtype=dtype)   # 70 .. 79: three rows outside
    for got, got2, which in ((k, k2, 0), (v, v2, 1)):
        x = values(cache, which).astype(np.float32)  # a product of 11 and 7 bits: exact in float
        x = x.astype(np.float16) if dtype == torch.float16 else x
        for s in range(n_seq):
            for i, r in enumerate(rows[s]):
                want = x[s, r] if 0 <= r < ctx else np.zeros((n_kv, hd), x.dtype)
                assert np.array_equal(got[s, i].cpu().numpy(), want)
        assert np.array_equal(got2.cpu().numpy(), x[:, 33:73])
    assert not k3[:, 7:].any() and k3[:, :7].any()


def test_read_one_of_the_two():
    cache = new_cache(syn.Q8_0, 1, 2, 64, 9)
    fill(cache, np.random.default_rng(0), 9)
    k, v = syn.kv_read(cache, 9)
    for which, want in ((0, k), (1, v)):
        out = torch.empty_like(want)
        p = [None, None]
        p[which] = out.data_ptr()
        assert syn.lib().syn_kv_read(cache.ref, 0, None, 0, 9, syn.F32, p[0], p[1], syn._stream()) == 0
        assert torch.equal(out, want)


# ---- move -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("n_kv,hd,n_seq,tree,n", [(8, 128, 2, 16, 5), (1, 32, 3, 40, 25), (2, 96, 1, 64, 64), (3, 64, 2, 1, 1)])
def test_move_gathers_the_path(type_, n_kv, hd, n_seq, tree, n):
    rng = np.random.default_rng(tree)
    ctx, layers = tree + 11, 3
    cache = new_cache(type_, n_seq, n_kv, hd, ctx, layers)
    raw = torch.randint(0, 256, cache.k.shape, dtype=torch.uint8, device="cuda")
    cache.k.copy_(raw)
    cache.v.copy_(raw.flip(-1))
    begin = rng.integers(0, ctx - tree + 1, n_seq).astype(np.int32)
    count = rng.integers(0, n + 1, n_seq).astype(np.int32)
    count[0] = n
    path = np.stack([b + np.sort(rng.choice(tree, n, replace=False)) for b in begin]).astype(np.int32)
    before = [[planes(cache, w, layer) for layer in range(layers)] for w in (0, 1)]
    syn.kv_move(cache, gpu(path), gpu(count), gpu(begin))
    for w in (0, 1):
        for layer in range(layers):
            got, want = planes(cache, w, layer), before[w][layer]
            for g, x in ((got, want),) if type_ == syn.F16 else zip(got, want):
                y = x.copy()
                for s in range(n_seq):
                    for i in range(count[s]):
                        if type_ == syn.F16:
                            y[s, begin[s] + i] = x[s, path[s, i]]
                        else:
                            y[s, :, begin[s] + i] = x[s, :, path[s, i]]
                assert np.array_equal(g, y)


def test_move_skips_rows_outside_the_cache():
    cache = new_cache(syn.Q8_0, 1, 1, 32, 8)
    fill(cache, np.random.default_rng(1), 8)
    before = cache.k.clone()
    syn.kv_move(cache, gpu(np.array([[8, 9]], np.int32)), gpu(np.array([2], np.int32)), gpu(np.array([7], np.int32)))
    syn.kv_move(cache, gpu(np.array([[3, 4]], np.int32)), gpu(np.array([-1], np.int32)), gpu(np.array([0], np.int32)))
    assert torch.equal(cache.k, before)


# ---- attention ----------------------------------------------------------------------------------------------------------
def random_masks(rng, n_seq, tree):
    """Trees as mask words and truth values."""
    sees = np.zeros((n_seq, tree, tree), bool)
    for s in range(n_seq):
        for i in range(tree):
            if i:
                sees[s, i] = sees[s, rng.integers(0, i)]
            sees[s, i, i] = True
    return pack(sees), sees


def pack(sees):
    n_seq, tree, _ = sees.shape
    words = np.zeros((n_seq, tree, (tree + 31) // 32), np.uint32)
    for j in range(tree):
        words[:, :, j // 32] |= sees[:, :, j].astype(np.uint32) << np.uint32(j % 32)
    return words.view(np.int32)


def exact_attention(q, k, v, lens, sees, n_head, scale):
    """q [n_seq][tree][n_head][hd], k, v [n_seq][ctx][n_kv][hd] in 64 bits -> (out, bound); unseen rows are left out."""
    n_seq, tree, _, hd = q.shape
    out, bound = np.zeros_like(q), np.zeros(q.shape[:3])
    for s in range(n_seq):
        for i in range(tree):
            rows = np.concatenate([np.arange(lens[s]), lens[s] + np.flatnonzero(sees[s, i])]).astype(int)
            if rows.size == 0:
                continue
            for h in range(n_head):
                g = h // (n_head // k.shape[2])
                kk, vv = k[s, rows, g], v[s, rows, g]
                x = kk @ q[s, i, h] * scale
                p = np.exp(x - x.max())
                out[s, i, h] = (p / p.sum()) @ vv
                most = (np.abs(kk) @ np.abs(q[s, i, h])).max() * abs(scale)
                bound[s, i, h] = (2 * (hd / 8 + 8) * 2.0 ** -23 * most + (rows.size / 8 + 64) * 2.0 ** -23) * np.abs(vv).max()
    return out, bound


def check_attention(type_, n_head, n_kv, hd, lens, tree, seed, mask="tree", ctx=None, sigma=1.0, scale=None, q_sigma=1.5,
                    max_len=None):
    rng = np.random.default_rng(seed)
    n_seq, most = len(lens), max(lens)
    ctx = ctx or most + tree
    cache = new_cache(type_, n_seq, n_kv, hd, ctx)
    cache.k.fill_(255)  # rows past a sequence's total hold NaN (F16) or scales that are NaN
    cache.v.fill_(255)
    w = n_kv * hd
    k, v = (rng.standard_normal((n_seq, most + tree, w), dtype=np.float32) * np.float32(sigma) for _ in "kv")
    k[:, :, ::7] *= 3
    slot = np.full((n_seq, most + tree), -1, np.int32)
    for s, n in enumerate(lens):
        slot[s, :n + tree] = np.arange(n + tree)
    syn.kv_append(cache, gpu(k.reshape(-1, w)), gpu(v.reshape(-1, w)), gpu(slot.reshape(-1)))
    q = rng.standard_normal((n_seq * tree, n_head * hd), dtype=np.float32) * np.float32(q_sigma)
    if mask == "tree":
        words, sees = random_masks(rng, n_seq, tree)
    else:
        words, sees = None, np.broadcast_to(np.tril(np.ones((tree, tree), bool)), (n_seq, tree, tree))
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    got = syn.tree_attention(cache, gpu(q), gpu(np.array(lens, np.int32)), n_head, scale, tree=tree,
                             mask=None if words is None else gpu(words), max_len=max_len)
    kk, vv = values(cache, 0), values(cache, 1)
    for s, n in enumerate(lens):  # never read by the check: what they hold is not finite
        kk[s, n + tree:], vv[s, n + tree:] = 0, 0
    want, bound = exact_attention(q.astype(np.float64).reshape(n_seq, tree, n_head, hd), kk, vv, lens, sees, n_head, scale)
    got = got.cpu().numpy().astype(np.float64).reshape(want.shape)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= bound[..., None]).all(), np.abs(got - want).max()
    assert np.linalg.norm(got - want) <= 1e-5 * np.linalg.norm(want)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("n_head,n_kv,hd", SHAPES)
@pytest.mark.parametrize("lens,tree", [([0], 1), ([1], 1), ([15, 16, 17], 1), ([63], 5), ([300, 1, 129], 16), ([40, 0], 33)])
def test_tree_attention(type_, n_head, n_kv, hd, lens, tree):
    check_attention(type_, n_head, n_kv, hd, lens, tree, seed=hd + tree)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("lens,tree", [([4095], 1), ([2047, 1000], 7), ([1500], 64), ([130], 100)])
def test_tree_attention_long(type_, lens, tree):
    check_attention(type_, 8, 2, 128, lens, tree, seed=tree)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("tree", [2, 3, 4, 5, 8, 9])
@pytest.mark.parametrize("lens", [[2500], [900, 3, 31]])
def test_attention_where_the_kernels_change(type_, tree, lens):
    check_attention(type_, 8, 2, 128, lens, tree, seed=tree)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("tree", [1, 3, 6])
def test_attention_of_many_ragged_sequences(type_, tree):
    """Far more sequences than the GPU has room for at a time, of lengths from none to several parts."""
    lens = [int(x) for x in np.random.default_rng(9).integers(0, 60, 400)]
    lens[3], lens[200], lens[399] = 1500, 700, 0
    check_attention(type_, 4, 2, 64, lens, tree, seed=tree)


@pytest.mark.parametrize("type_", TYPES)
def test_tree_attention_of_many_ragged_sequences(type_):
    """Trees of 40 tokens in more sequences than the GPU has room for at a time, one of several parts."""
    lens = [int(x) for x in np.random.default_rng(3).integers(0, 90, 170)]
    lens[5], lens[169] = 900, 0
    check_attention(type_, 4, 2, 64, lens, 40, seed=1)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("lens,tree", [([0], 70), ([100, 37], 9)])
def test_causal_chunk(type_, lens, tree):
    check_attention(type_, 6, 2, 64, lens, tree, seed=3, mask=None)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("sigma,q_sigma", [(1e-3, 1.0), (200.0, 0.01), (1.0, 1e-4), (1.0, 300.0)])
def test_tree_attention_over_the_range_of_values(type_, sigma, q_sigma):
    """Small and large keys, values and queries; q_sigma = 300 makes the softmax one-hot."""
    check_attention(type_, 4, 2, 64, [100, 33], 6, seed=11, sigma=sigma, q_sigma=q_sigma)


@pytest.mark.parametrize("n_head,n_kv,hd", [(3, 1, 48), (2, 2, 8), (4, 1, 200)])
def test_tree_attention_f16_head_sizes(n_head, n_kv, hd):
    check_attention(syn.F16, n_head, n_kv, hd, [50, 7], 5, seed=hd)


@pytest.mark.parametrize("type_", TYPES)
def test_tree_attention_odd_capacity_and_bound(type_):
    """A capacity that leaves the heads' scale rows unaligned, and a max_len far above the lengths."""
    check_attention(type_, 6, 3, 32, [70, 5], 4, seed=1, ctx=1237)
    check_attention(type_, 6, 3, 96, [70, 5], 4, seed=1, ctx=1237, max_len=1000)


@pytest.mark.parametrize("type_", TYPES)
def test_rows_that_see_nothing_are_zero_and_masked_rows_do_not_matter(type_):
    n_head, n_kv, hd, tree = 4, 2, 64, 6
    rng = np.random.default_rng(8)
    cache = new_cache(type_, 2, n_kv, hd, 40)
    fill(cache, rng, 40)
    sees = np.zeros((2, tree, tree), bool)
    sees[:, 1, 1] = sees[:, 2, 1] = sees[:, 2, 2] = sees[:, 5, 5] = True
    lens = gpu(np.array([0, 20], np.int32))
    q = gpu(rng.standard_normal((2 * tree, n_head * hd), dtype=np.float32))
    args = dict(tree=tree, mask=gpu(pack(sees)))
    want = syn.tree_attention(cache, q, lens, n_head, 0.125, **args)
    assert not want[[0, 3, 4]].any() and want[[1, 2, 5]].any(1).all() and want[6:].any(1).all()
    # node 3 is seen by nobody, node 2 by itself alone: infinities, NaN and unwritten rows there
    for bad in (float("inf"), float("nan"), -65504.0):
        for node in (3, 2):
            c = syn.KVCache(type_, 1, 2, n_kv, hd, 40)
            c.k.copy_(cache.k)
            c.v.copy_(cache.v)
            if type_ == syn.F16:
                for t in (c.k, c.v):
                    rows = t.view(torch.float16).view(2, 40, n_kv, hd)
                    rows[0, node], rows[1, 20 + node] = bad, bad
            else:  # scales that no append writes
                size = syn.kv_cache_bytes(type_, n_kv, hd, 40) - (n_kv * 40 * (hd // 32) * 2 + 255) // 256 * 256
                for t in (c.k, c.v):
                    rows = t[0, :, size:size + n_kv * 40 * (hd // 32) * 2].contiguous().view(torch.float16).view(2, n_kv, 40, -1)
                    rows[0, :, node], rows[1, :, 20 + node] = bad, bad
                    t[0, :, size:size + n_kv * 40 * (hd // 32) * 2] = rows.view(2, -1).view(torch.uint8)
            got = syn.tree_attention(c, q, lens, n_head, 0.125, **args)
            others = [i for i in range(2 * tree) if i % tree != node]
            assert torch.equal(got[others], want[others])
            if node == 2 and not math.isfinite(bad):
                assert got[[2, 8]].isnan().all()


def test_tree_attention_is_repeatable_and_leaves_its_scratch_ready():
    rng = np.random.default_rng(2)
    for type_ in TYPES:
        cache = new_cache(type_, 1, 2, 128, 3000)
        fill(cache, rng, 3000)
        q = gpu(rng.standard_normal((4, 8 * 128), dtype=np.float32))
        lens = gpu(np.array([2900], np.int32))
        scratch = syn.tree_attention_scratch(cache, 4, 8)
        first = syn.tree_attention(cache, q, lens, 8, 0.1, tree=4, scratch=scratch)
        small = syn.tree_attention(cache, q[:1], lens, 8, 0.1, scratch=scratch)  # another shape between
        for _ in range(20):
            assert torch.equal(syn.tree_attention(cache, q, lens, 8, 0.1, tree=4, scratch=scratch), first)
        assert torch.equal(syn.tree_attention(cache, q[:1], lens, 8, 0.1), small)


def test_tree_attention_matches_the_decode_attention():
    """One token over a session-layout cache: syn_attention's values, which round q and p to binary16."""
    rng = np.random.default_rng(4)
    n_head, n_kv, hd, L = 8, 2, 128, 700
    cache = new_cache(syn.F16, 1, n_kv, hd, L)
    fill(cache, rng, L)
    q = gpu(rng.standard_normal((1, n_head * hd), dtype=np.float32)).half().float()
    want = syn.attention(q, None, None, cache.k.view(torch.int16).flatten(), cache.v.view(torch.int16).flatten(),
                         gpu(np.array([L - 1], np.int32)), n_head, n_kv, hd, L, 1.0, 1 / math.sqrt(hd), append=False, rope=False)
    got = syn.tree_attention(cache, q, gpu(np.array([L - 1], np.int32)), n_head, 1 / math.sqrt(hd))
    assert torch.linalg.norm(got - want) <= 1e-3 * torch.linalg.norm(want)  # 2^-11 of each probability


def test_tree_attention_strided_queries_layers_and_streams():
    rng = np.random.default_rng(6)
    n_head, n_kv, hd, tree, L = 6, 2, 64, 5, 90
    cache = new_cache(syn.Q8_0, 2, n_kv, hd, L + tree, n_layer=3)
    for layer in range(3):
        fill(cache, rng, L + tree, layer=layer)
    qkv = gpu(rng.standard_normal((2 * tree, (n_head + 2 * n_kv) * hd), dtype=np.float32))
    q = qkv[:, :n_head * hd]
    lens = gpu(np.array([L, L - 30], np.int32))
    want = syn.tree_attention(cache, q.contiguous(), lens, n_head, 0.2, tree=tree, layer=2)
    one = syn.KVCache.over(syn.Q8_0, cache.k[2], cache.v[2], n_kv, hd, L + tree)
    assert torch.equal(syn.tree_attention(one, q, lens, n_head, 0.2, tree=tree), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = syn.tree_attention(cache, q, lens, n_head, 0.2, tree=tree, layer=2)
    side.synchronize()
    assert torch.equal(got, want)
    assert not torch.equal(syn.tree_attention(cache, q, lens, n_head, 0.2, tree=tree, layer=1), want)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("tree", [1, 9])
def test_unaligned_rows_and_a_stream_argument(type_, tree):
    """Rows of q, k and v that start and follow at no 16-byte boundary, and the calls' stream argument."""
    rng = np.random.default_rng(13)
    n_head, n_kv, hd, L = 8, 2, 128, 300
    wide = gpu(rng.standard_normal((tree, (n_head + 2 * n_kv) * hd + 3), dtype=np.float32))
    q, k, v = wide[:, 1:1 + n_head * hd], wide[:, 1 + n_head * hd:1 + (n_head + n_kv) * hd], wide[:, 1 + (n_head + n_kv) * hd:-2]
    table = syn.rope_table(L + tree, hd, 0.9)
    slot = gpu(np.arange(L, L + tree, dtype=np.int32))
    lens = gpu(np.array([L], np.int32))
    a, b = new_cache(type_, 1, n_kv, hd, L + tree), new_cache(type_, 1, n_kv, hd, L + tree)
    for c in (a, b):
        fill(c, np.random.default_rng(0), L)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for mode in (0, 1):
        qa = syn.kv_append(a, k, v, slot, rope_table=table, rope_mode=mode, q=q, stream=side)
        oa = syn.tree_attention(a, qa, lens, n_head, 0.1, tree=tree, stream=side)
        ua = syn.tree_attention(a, q, lens, n_head, 0.1, tree=tree, stream=side)
        _, pa = syn.logits_process(ua, 1, stream=side)
        ka, va = syn.kv_read(a, L + tree, stream=side)
        side.synchronize()
        qb = syn.kv_append(b, k.contiguous(), v.contiguous(), slot, rope_table=table, rope_mode=mode, q=q.contiguous())
        ob = syn.tree_attention(b, qb, lens, n_head, 0.1, tree=tree)
        ub = syn.tree_attention(b, q.contiguous(), lens, n_head, 0.1, tree=tree)
        kb, vb = syn.kv_read(b, L + tree)
        for x, y in ((qa, qb), (oa, ob), (ua, ub), (ka, kb), (va, vb)):
            assert torch.equal(x, y)
        assert torch.equal(pa, syn.logits_process(ub, 1)[1])


@pytest.mark.parametrize("type_", TYPES)
def test_wide_trees(type_):
    check_attention(type_, 2, 1, 64, [130, 5], 300, seed=21)
    check_attention(type_, 1, 1, 32, [40], 1024, seed=22)


@pytest.mark.parametrize("type_", TYPES)
def test_lengths_outside_the_bound_are_clamped(type_):
    rng = np.random.default_rng(14)
    for n_head, tree in ((2, 2), (24, 3)):
        cache = new_cache(type_, 3, 2, 64, 64)
        fill(cache, rng, 64)
        q = gpu(rng.standard_normal((3 * tree, n_head * 64), dtype=np.float32))
        got = syn.tree_attention(cache, q, gpu(np.array([-5, 1000, 2**31 - 1], np.int32)), n_head, 0.1, tree=tree, max_len=60)
        want = syn.tree_attention(cache, q, gpu(np.array([0, 60 - tree, 60 - tree], np.int32)), n_head, 0.1, tree=tree, max_len=60)
        assert torch.equal(got, want)


@pytest.mark.parametrize("type_", TYPES)
def test_negative_scale(type_):
    check_attention(type_, 4, 2, 64, [70], 3, seed=31, scale=-0.125)
    check_attention(type_, 24, 2, 64, [70], 3, seed=32, scale=-0.125)


def test_offsets_past_32_bits():
    """Rows past 2^32 bytes: written, read, moved and attended to; the scores of all but three rows are zero."""
    n_kv, hd = 8, 128
    ctx = (1 << 32) // (n_kv * hd * 2) + 1000
    cache = new_cache(syn.F16, 1, n_kv, hd, ctx)
    rng = np.random.default_rng(9)
    n = 3
    k = gpu(np.zeros((n, n_kv * hd), np.float32) + np.float32(0.5))
    v = gpu(rng.standard_normal((n, n_kv * hd), dtype=np.float32))
    slots = np.array([ctx - 900, ctx - 500, ctx - 2], np.int32)
    syn.kv_append(cache, k, v, gpu(slots))
    _, back = syn.kv_read(cache, n, rows=gpu(slots))
    assert torch.equal(back[0].view(n, -1), v.half().float())
    q = gpu(np.ones((1, n_kv * hd), np.float32))
    out = syn.tree_attention(cache, q, gpu(np.array([ctx - 1], np.int32)), n_kv, 0.25)  # scores 16 at three rows
    w = math.exp(16.0)
    want = w / (3 * w + ctx - 3) * v.half().double().sum(0)
    assert torch.linalg.norm(out[0].double() - want) <= 1e-5 * torch.linalg.norm(want)
    syn.kv_move(cache, gpu(slots[None]), gpu(np.array([n], np.int32)), gpu(np.array([ctx - 950], np.int32)))
    _, back = syn.kv_read(cache, n, first=ctx - 950)
    assert torch.equal(back[0].view(n, -1), v.half().float())
    del cache
    # sequences far apart
    stride = (1 << 32) + 4096
    data = torch.zeros(2 * stride, dtype=torch.uint8, device="cuda")
    size = syn.kv_cache_bytes(syn.Q4_0, 1, 64, 50)
    kv = [data[o:].as_strided((2, size), (stride, 1)) for o in (0, 65536)]
    far = syn.KVCache.over(syn.Q4_0, *kv, 1, 64, 50)
    near = new_cache(syn.Q4_0, 2, 1, 64, 50)
    for c in (far, near):
        fill(c, np.random.default_rng(1), 50)
    lens = gpu(np.array([30, 49], np.int32))
    q = gpu(rng.standard_normal((2, 4 * 64), dtype=np.float32))
    assert torch.equal(syn.tree_attention(far, q, lens, 4, 0.1), syn.tree_attention(near, q, lens, 4, 0.1))


# ---- logits -----------------------------------------------------------------------------------------------------------
def plain_logits(x, n_seq, pen, past, past_len, draft, sees, bias, allowed):
    """The definition, in float steps (each operation rounded once, as the kernel's)."""
    rows, vocab = x.shape
    tree = rows // n_seq
    y = x.astype(np.float32).copy()
    for r in range(rows):
        s, i = r // tree, r % tree
        count = np.zeros(vocab, np.int64)
        if past is not None:
            for t in past[s, :past_len[s]]:
                if 0 <= t < vocab:
                    count[t] += 1
        if draft is not None:
            for j in np.flatnonzero(sees[s, i]):
                if 0 <= draft[s, j] < vocab:
                    count[draft[s, j]] += 1
        if bias is not None:
            begin, tokens, vals = bias
            for e in range(begin[s], begin[s + 1]):
                if 0 <= tokens[e] < vocab:
                    y[r, tokens[e]] += vals[e]
        rep, pres, freq = (np.float32(p) for p in (pen[s] if pen is not None else (1, 0, 0)))
        hit = count > 0
        z = np.where(y[r] > 0, y[r] / rep, y[r] * rep).astype(np.float32)
        z = z - (count.astype(np.float32) * freq + pres)
        y[r] = np.where(hit, z, y[r])
        if allowed is not None:
            bits = (allowed[r].view(np.uint32)[np.arange(vocab) // 32] >> (np.arange(vocab) % 32).astype(np.uint32)) & 1
            y[r] = np.where(bits == 1, y[r], -np.inf)
    pick = np.full(rows, -1, np.int32)
    for r in range(rows):
        z = np.where(np.isnan(y[r]), -np.inf, y[r])
        if (z > -np.inf).any():
            pick[r] = int(np.argmax(z))
    return y, pick


@pytest.mark.parametrize("n_seq,tree,vocab", [(1, 1, 128256), (2, 5, 32000), (3, 1, 50257), (2, 40, 1000), (1, 3, 31), (1, 2, 1),
                                              (40, 4, 9000)])
@pytest.mark.parametrize("what", ["all", "penalties", "none"])
def test_logits_process(n_seq, tree, vocab, what):
    rng = np.random.default_rng(vocab + tree)
    rows = n_seq * tree
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    x[:, vocab // 2] = 0.0
    past = rng.integers(-3, vocab + 3, (n_seq, 700)).astype(np.int32)
    past[:, ::3] = rng.integers(0, min(vocab, 9), (n_seq, 234))
    past_len = rng.integers(0, 701, n_seq).astype(np.int32)
    past_len[0] = 700
    pen = np.stack([rng.uniform(0.8, 1.5, n_seq), rng.uniform(-0.5, 1, n_seq), rng.uniform(-0.2, 0.5, n_seq)], 1).astype(np.float32)
    draft = rng.integers(0, vocab, (n_seq, tree)).astype(np.int32)
    draft[:, tree // 2] = x.argmax(1).reshape(n_seq, tree)[:, 0]  # a likely token drafted: the paths differ in it
    words, sees = random_masks(rng, n_seq, tree)
    per = [min(vocab, 5 * s + 3) for s in range(n_seq)]
    begin = np.cumsum([0] + per).astype(np.int32)
    tokens = np.concatenate([rng.choice(vocab, n, replace=False) for n in per]).astype(np.int32)
    vals = (rng.standard_normal(tokens.size) * 5).astype(np.float32)
    allowed = rng.integers(0, 2**32, (rows, (vocab + 31) // 32), dtype=np.uint32)
    allowed[rows - 1] = 0  # a row whose mask leaves nothing
    kw, plain = {}, [None] * 7
    if what != "none":
        kw = dict(penalties=gpu(pen), history=gpu(past), history_len=gpu(past_len), draft=gpu(draft), mask=gpu(words))
        plain[:5] = [pen, past, past_len, draft, sees]
    if what == "all":
        kw.update(bias=(gpu(begin), gpu(tokens), gpu(vals)), allowed=gpu(allowed.view(np.int32)))
        plain[5:] = [(begin, tokens, vals), allowed]
    out, pick = syn.logits_process(gpu(x), n_seq, **kw)
    want, want_pick = plain_logits(x, n_seq, *plain)
    assert np.array_equal(out.cpu().numpy().view(np.int32), want.view(np.int32))
    assert np.array_equal(pick.cpu().numpy(), want_pick)
    if what == "all":
        assert pick[rows - 1] == -1


def test_logits_in_place_strided_ties_and_values_that_are_not_finite():
    rng = np.random.default_rng(0)
    wide = gpu(rng.standard_normal((3, 2056), dtype=np.float32))
    x = wide[:, 3:2003]
    x[0, 7] = x[0, 1999] = 50.0            # equal: the lowest index
    x[1, :] = float("nan")
    x[1, 100], x[1, 200] = -0.0, 0.0       # equal zeros, the first has its sign set
    x[2, 5], x[2, 6] = float("inf"), float("nan")
    before = wide.clone()
    out, pick = syn.logits_process(x, 3, out=x)
    assert out.data_ptr() == x.data_ptr() and pick.tolist() == [7, 100, 5]
    assert torch.equal(wide.nan_to_num(9.0), before.nan_to_num(9.0))
    x[1, :] = float("-inf")
    scratch = syn.logits_scratch(3)
    for _ in range(3):  # the scratch is left ready
        assert syn.logits_process(x, 1, scratch=scratch)[1].tolist() == [7, -1, 5]
        assert not scratch.any()
    assert syn.logits_process(x, 3, pick=False)[1] is None


@pytest.mark.parametrize("vocab", [1500, 64000])
def test_logits_biases_of_a_token_add_in_the_lists_order(vocab):
    """Sums whose value depends on the order, their entries far apart among others; long and short chunks."""
    rng = np.random.default_rng(5)
    rows = 1 if vocab < 4096 else 64
    tokens = rng.integers(0, vocab, 1200).astype(np.int32)
    values = rng.standard_normal(1200).astype(np.float32)
    for t in (7, vocab - 1):
        at = rng.choice(1200, 40, replace=False)
        tokens[at] = t
        values[at] = (rng.standard_normal(40) * 10.0 ** rng.integers(-3, 8, 40)).astype(np.float32)
    want = np.zeros(vocab, np.float32)
    for t, v in zip(tokens, values):
        want[t] = want[t] + v
    x = gpu(np.zeros((rows, vocab), np.float32))
    bias = (gpu(np.array([0, 1200], np.int32)), gpu(tokens), gpu(values))
    for _ in range(3):
        out, _ = syn.logits_process(x, 1, bias=bias)
        assert np.array_equal(out.cpu().numpy(), np.broadcast_to(want, (rows, vocab)))


def test_logits_bias_named_twice_counts_twice_and_draft_without_mask_is_a_chain():
    x = torch.zeros(3, 100, device="cuda")
    bias = (gpu(np.array([0, 2], np.int32)), gpu(np.array([5, 5], np.int32)), gpu(np.array([1.5, 2.0], np.float32)))
    draft = gpu(np.array([[9, 10, 9]], np.int32))
    pen = gpu(np.array([[1.0, 0.5, 0.25]], np.float32))
    out, pick = syn.logits_process(x, 1, penalties=pen, draft=draft, bias=bias)
    assert (out[:, 5] == 3.5).all() and pick.tolist() == [5, 5, 5]
    assert out[:, 9].tolist() == [-0.75, -0.75, -1.0] and out[:, 10].tolist() == [0.0, -0.75, -0.75]


# ---- refusals ---------------------------------------------------------------------------------------------------------
def test_refusals():
    cache = new_cache(syn.Q8_0, 2, 2, 64, 32)
    x = torch.zeros(2, 128, device="cuda")
    slot = torch.zeros(2, dtype=torch.int32, device="cuda")
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    L, st = syn.lib(), syn._stream()

    def desc(**kw):
        d = syn.KVCacheDesc(**{n: getattr(cache.desc, n) for n, _ in syn.KVCacheDesc._fields_})
        for n, v in kw.items():
            setattr(d, n, v)
        return d

    def append(d, layer=0, **kw):
        a = syn.KVAppendArgs(k=x.data_ptr(), v=x.data_ptr(), slot=slot.data_ptr(), n=1)
        for n, v in kw.items():
            setattr(a, n, v)
        return L.syn_kv_append(ctypes.byref(d), layer, ctypes.byref(a), st)

    INVALID, UNSUPPORTED = 1, 2
    assert append(desc()) == 0
    for d, want in ((desc(k=None), INVALID), (desc(type=syn.F32), UNSUPPORTED), (desc(type=syn.Q4_K), UNSUPPORTED),
                    (desc(head_dim=48), UNSUPPORTED), (desc(head_dim=288), UNSUPPORTED), (desc(max_ctx=0), INVALID),
                    (desc(seq_stride=cache.desc.seq_stride + 8), INVALID), (desc(seq_stride=16), INVALID),
                    (desc(k=cache.desc.k + 4), INVALID), (desc(n_layer=2), INVALID), (desc(n_seq=0), INVALID)):
        assert append(d) == want, d.type
    assert append(desc(), layer=1) == INVALID and append(desc(), layer=-1) == INVALID
    for kw in (dict(k=None), dict(slot=None), dict(n=0), dict(rope_mode=2), dict(kv_stride=64), dict(q=x.data_ptr()),
               dict(q=x.data_ptr(), q_out=x.data_ptr(), n_head=2), dict(rope_table=x.data_ptr())):
        assert append(desc(), **kw) == INVALID, kw
    assert L.syn_kv_read(cache.ref, 0, None, 0, 0, syn.F32, x.data_ptr(), None, st) == INVALID
    assert L.syn_kv_read(cache.ref, 0, None, 0, 1, syn.F32, None, None, st) == INVALID
    assert L.syn_kv_read(cache.ref, 0, None, -1, 1, syn.F32, x.data_ptr(), None, st) == INVALID
    assert L.syn_kv_read(cache.ref, 0, None, 0, 1, syn.Q8_0, x.data_ptr(), None, st) == UNSUPPORTED
    assert L.syn_kv_read(cache.ref, 0, None, 0, 1, syn.F32, x.data_ptr() + 4, None, st) == INVALID
    assert L.syn_kv_move(cache.ref, None, 1, slot.data_ptr(), slot.data_ptr(), st) == INVALID
    assert L.syn_kv_move(cache.ref, slot.data_ptr(), 0, slot.data_ptr(), slot.data_ptr(), st) == INVALID

    scratch = syn.tree_attention_scratch(cache, 1, 4)
    q = torch.zeros(2, 4 * 64, device="cuda")
    out = torch.empty_like(q)

    def attend(**kw):
        a = syn.TreeAttentionArgs(q=q.data_ptr(), out=out.data_ptr(), len=lens.data_ptr(), scratch=scratch.data_ptr(), n_tree=1,
                                  n_head=4, max_len=32, scale=1.0)
        for n, v in kw.items():
            setattr(a, n, v)
        return L.syn_tree_attention(cache.ref, 0, ctypes.byref(a), st)

    assert attend() == 0
    for kw in (dict(q=None), dict(out=None), dict(len=None), dict(scratch=None), dict(scratch=scratch.data_ptr() + 8), dict(n_head=3),
               dict(n_tree=0), dict(n_tree=33), dict(max_len=33), dict(max_len=0), dict(q_stride=100)):
        assert attend(**kw) == INVALID, kw
    assert syn.lib().syn_tree_attention_scratch_bytes(1, 0, 4, 2, 64, 32) == 0
    assert syn.kv_cache_bytes(syn.Q4_0, 2, 48, 32) == 0 and syn.kv_cache_bytes(syn.F16, 2, 48, 32) == 2 * 48 * 32 * 2

    logits = torch.zeros(2, 100, device="cuda")
    ls = syn.logits_scratch(2)
    pick = torch.empty(2, dtype=torch.int32, device="cuda")

    def process(**kw):
        a = syn.LogitsArgs(logits=logits.data_ptr(), pick=pick.data_ptr(), scratch=ls.data_ptr(), n_seq=2, n_tree=1, n_vocab=100)
        for n, v in kw.items():
            setattr(a, n, v)
        return L.syn_logits_process(ctypes.byref(a), st)

    assert process() == 0
    for kw in (dict(logits=None), dict(pick=None), dict(scratch=None), dict(n_vocab=0), dict(n_tree=0), dict(ld=99), dict(out_ld=99),
               dict(history=pick.data_ptr()), dict(bias_begin=pick.data_ptr()), dict(allowed_ld=3),
               dict(out=logits.data_ptr(), out_ld=104)):
        assert process(**kw) == INVALID, kw
    assert process(n_tree=2000) == UNSUPPORTED
    with pytest.raises(ValueError):
        syn.tree_attention(cache, q[:, :100], lens, 4, 1.0)
    with pytest.raises(ValueError):
        syn.tree_attention(cache, q, lens.long(), 4, 1.0)
    with pytest.raises(ValueError):
        syn.tree_attention(cache, q, lens, 4, 1.0, scratch=scratch[:100])
    with pytest.raises(ValueError):
        syn.kv_append(cache, x.half(), x, slot)
    with pytest.raises(ValueError):
        syn.logits_process(logits, 2, penalties=torch.zeros(5, device="cuda"))
    with pytest.raises(ValueError):
        syn.KVCache.over(syn.F16, torch.zeros(2, 100, dtype=torch.uint8, device="cuda"), torch.zeros(2, 100, dtype=torch.uint8, device="cuda"), 2, 64, 32)
    with pytest.raises(syn.SynapseError):
        syn.KVCache(syn.Q8_0, 1, 1, 2, 48, 32)
    torch.cuda.synchronize()


def test_refuses_tensors_that_are_not_on_the_current_device(monkeypatch):
    """As with a second GPU current: nothing is launched."""
    cache = new_cache(syn.Q8_0, 1, 2, 64, 32)
    i = gpu(np.zeros(1, np.int32))
    x, q = gpu(np.zeros((1, 128), np.float32)), gpu(np.zeros((1, 256), np.float32))
    scratch, small = syn.tree_attention_scratch(cache, 1, 4), syn.logits_scratch(1)
    monkeypatch.setattr(syn, "_here", lambda: 1)
    for call in (lambda: syn.kv_append(cache, x, x, i), lambda: syn.kv_read(cache, 1), lambda: syn.kv_move(cache, i, i, i),
                 lambda: syn.tree_attention(cache, q, i, 4, 1.0, scratch=scratch),
                 lambda: syn.logits_process(x, 1, scratch=small)):
        with pytest.raises(ValueError, match="current"):
            call()
    monkeypatch.undo()
    for call in (lambda: syn.kv_append(cache, x.cpu(), x, i), lambda: syn.tree_attention(cache, q, i.cpu(), 4, 1.0, scratch=scratch),
                 lambda: syn.logits_process(x.cpu(), 1), lambda: syn.logits_process(x, 1, scratch=small.cpu()),
                 lambda: syn.tree_attention(cache, q, i, 4, 1.0, scratch=scratch.cpu()),
                 lambda: syn.tree_attention(cache, q, i, 4, 1.0, scratch=scratch.new_zeros(2 * scratch.numel())[::2])):
        with pytest.raises(ValueError, match="current"):
            call()
