"""Tree attention and its caches at the edges of their types. Tolerances are those of test_tree_decode_gpu.py."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
syn = pytest.importorskip("synapse_b200")
from tests.test_tree_decode_gpu import exact_attention, fill, gpu, new_cache, random_masks, values  # noqa: E402

TYPES = [syn.F16, syn.Q8_0, syn.Q4_0]
# rows of a KV head on either side of every change of kernel: 1, 8, 12, 32 and 36
ROWS = [(2, 1), (8, 2), (6, 4), (8, 8), (24, 3)]


def scales(cache, which):
    """The scales of a quantised cache of one layer as a view, [n_seq][n_kv][ctx][hd / 32] binary16."""
    n, kv, hd, ctx = cache.n_seq, cache.n_kv, cache.head_dim, cache.max_ctx
    at = (kv * ctx * hd // (1 if cache.type == syn.Q8_0 else 2) + 255) // 256 * 256
    raw = (cache.k if which == 0 else cache.v)[0]
    return raw[:, at:at + kv * ctx * hd // 16].view(torch.float16).view(n, kv, ctx, hd // 32)


def rows16(cache, which):
    """An F16 cache of one layer as a view, [n_seq][ctx][n_kv][hd]."""
    raw = (cache.k if which == 0 else cache.v)[0]
    return raw.view(torch.float16).view(cache.n_seq, cache.max_ctx, cache.n_kv, cache.head_dim)


def copy_of(cache):
    c = new_cache(cache.type, cache.n_seq, cache.n_kv, cache.head_dim, cache.max_ctx)
    c.k.copy_(cache.k)
    c.v.copy_(cache.v)
    return c


def check_against_64_bits(cache, q, lens, tree, words, sees, n_head, scale):
    got = syn.tree_attention(cache, gpu(q), gpu(np.array(lens, np.int32)), n_head, scale, tree=tree, mask=gpu(words))
    q64 = q.astype(np.float64).reshape(len(lens), tree, n_head, cache.head_dim)
    want, bound = exact_attention(q64, values(cache, 0), values(cache, 1), lens, sees, n_head, scale)
    got = got.cpu().numpy().astype(np.float64).reshape(want.shape)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= bound[..., None]).all(), np.abs(got - want).max()
    assert np.linalg.norm(got - want) <= 1e-5 * np.linalg.norm(want)


# ---- scales ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("type_", [syn.Q8_0, syn.Q4_0])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n_head,tree", ROWS)
@pytest.mark.parametrize("where", ["all", "some", "tree"])
def test_attention_over_scales_of_any_finite_size(type_, hd, n_head, tree, where):
    """V's scales up to binary16's largest, of both signs, in every row, in a row here and there or in the tree's own."""
    rng = np.random.default_rng(hd + tree)
    n_kv, lens = 2, [400, 37]
    cache = new_cache(type_, 2, n_kv, hd, 400 + tree)
    fill(cache, rng, 400 + tree)
    d = scales(cache, 1)
    big = np.float16(rng.choice([8188, -8188, 8192, -8192, 10000, -16384, 40000, 65504, -65504, 4.0], d.shape))
    at = np.zeros(d.shape, bool)
    if where == "all":
        at[:] = True
    elif where == "some":
        at = rng.random(d.shape) < 0.01
        at[:, :, 5] = True
    else:
        for s, n in enumerate(lens):
            at[s, :, n:n + tree] = True
    d.copy_(torch.where(gpu(at), gpu(big), d))
    q = rng.standard_normal((2 * tree, n_head * hd), dtype=np.float32) * np.float32(1.5)
    words, sees = random_masks(rng, 2, tree)
    check_against_64_bits(cache, q, lens, tree, words, sees, n_head, hd ** -0.5)


@pytest.mark.parametrize("type_", [syn.Q8_0, syn.Q4_0])
@pytest.mark.parametrize("n_head,tree", ROWS)
def test_attention_over_large_scales_of_keys(type_, n_head, tree):
    rng = np.random.default_rng(tree)
    hd, lens = 64, [90, 300]
    cache = new_cache(type_, 2, 2, hd, 300 + tree)
    fill(cache, rng, 300 + tree)
    d = scales(cache, 0)
    d.copy_(gpu(np.float16(rng.choice([65504, -65504, 8192, 100], d.shape))))
    q = rng.standard_normal((2 * tree, n_head * hd), dtype=np.float32) * np.float32(1e-6)
    words, sees = random_masks(rng, 2, tree)
    check_against_64_bits(cache, q, lens, tree, words, sees, n_head, hd ** -0.5)


@pytest.mark.parametrize("type_", [syn.Q8_0, syn.Q4_0])
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("n_head,tree", [(4, 4), (4, 8), (24, 3)])
def test_large_scales_change_nothing_for_who_does_not_see_them(type_, hd, n_head, tree):
    rng = np.random.default_rng(hd + tree)
    n_kv, L = 2, 200
    cache = new_cache(type_, 1, n_kv, hd, L + tree)
    fill(cache, rng, L + tree)
    words, sees = random_masks(rng, 1, tree)
    q = gpu(rng.standard_normal((tree, n_head * hd), dtype=np.float32))
    lens = gpu(np.array([L], np.int32))
    want = syn.tree_attention(cache, q, lens, n_head, 0.125, tree=tree, mask=gpu(words)).view(tree, n_head, hd)
    scales(cache, 1)[0, 1, L + 1] = 65504.0
    got = syn.tree_attention(cache, q, lens, n_head, 0.125, tree=tree, mask=gpu(words)).view(tree, n_head, hd)
    hit = sees[0, :, 1]
    assert torch.equal(got[~hit], want[~hit]) and torch.equal(got[:, :n_head // 2], want[:, :n_head // 2])
    assert got.isfinite().all() and (got[hit][:, n_head // 2:] != want[hit][:, n_head // 2:]).any()


# ---- values that are not finite -------------------------------------------------------------------------------------
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("n_head,tree", [(4, 4), (24, 3)])
@pytest.mark.parametrize("which", [0, 1])
def test_one_value_that_is_not_finite(type_, hd, n_head, tree, which):
    """An infinity or NaN in one value of K (which = 0) or V: tokens that do not see its row and heads that do not read
    it are as without it. Who sees it gets NaN in the heads that read it, whatever the signs; of V in a committed row of
    an F16 cache, something that is not finite in the dim concerned, and the others as they were."""
    rng = np.random.default_rng(hd + tree)
    n_kv, lens = 2, [70, 200]
    group = n_head // n_kv
    cache = new_cache(type_, 2, n_kv, hd, 200 + tree)
    fill(cache, rng, 200 + tree)
    words, sees = random_masks(rng, 2, tree)
    q = gpu(rng.standard_normal((2 * tree, n_head * hd), dtype=np.float32))
    args = dict(tree=tree, mask=gpu(words))
    lens_gpu = gpu(np.array(lens, np.int32))
    want = syn.tree_attention(cache, q, lens_gpu, n_head, 0.125, **args).view(2, tree, n_head, hd)
    for bad in (float("inf"), -float("inf"), float("nan")):
        for row in (3, lens[1] + 1):  # committed, and the tree's
            c = copy_of(cache)
            dim = int(rng.integers(hd))
            if type_ == syn.F16:
                rows16(c, which)[1, row, 1, dim] = bad
            else:
                scales(c, which)[1, 1, row, dim // 32] = bad
            got = syn.tree_attention(c, q, lens_gpu, n_head, 0.125, **args).view(2, tree, n_head, hd)
            hit = np.ones(tree, bool) if row < lens[1] else sees[1, :, 1]
            assert torch.equal(got[0], want[0]) and torch.equal(got[:, :, :group], want[:, :, :group])
            assert torch.equal(got[1, ~hit], want[1, ~hit])
            heads = got[1, hit][:, group:]
            if which == 0 or type_ != syn.F16 or row >= lens[1]:
                assert heads.isnan().all()
            else:
                others = torch.arange(hd, device="cuda") != dim
                assert not heads[..., dim].isfinite().any() and torch.equal(heads[..., others], want[1, hit][:, group:][..., others])


# ---- a scale of zero --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("n_head,tree", ROWS)
def test_scale_of_zero_is_the_mean_of_what_is_seen(type_, hd, n_head, tree):
    rng = np.random.default_rng(hd + tree)
    lens = [130, 7]
    cache = new_cache(type_, 2, 2, hd, 130 + tree)
    fill(cache, rng, 130 + tree)
    q = rng.standard_normal((2 * tree, n_head * hd), dtype=np.float32)
    words, sees = random_masks(rng, 2, tree)
    check_against_64_bits(cache, q, lens, tree, words, sees, n_head, 0.0)


# ---- what an append stores --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("type_", [syn.Q8_0, syn.Q4_0])
def test_clamped_rows_read_back_finite_in_binary16(type_):
    """Values around and beyond binary16's range, of both signs, read back in both formats."""
    tops = [65400.0, 65469.0, 65499.0, 65500.25, 65500.5, 65503.0, 65504.0, 65519.0, 65520.0, 1e6, 3e38, float("inf")]
    tops += [-t for t in tops]
    cache = new_cache(type_, 1, 1, 64, len(tops))
    x = np.ones((len(tops), 64), np.float32)
    x[:, 5] = tops
    syn.kv_append(cache, gpu(x), gpu(x), gpu(np.arange(len(tops), dtype=np.int32)))
    f, _ = syn.kv_read(cache, len(tops))
    h, hv = syn.kv_read(cache, len(tops), dtype=torch.float16)
    assert f.isfinite().all() and h.isfinite().all() and torch.equal(h, hv)
    want = np.clip(np.array(tops), -65504.0, 65504.0)
    got = f[0, :, 0, 5].cpu().numpy()
    # the scale's rounding: 2^-11 of it, or from 516 down to 515.5
    assert (np.abs(got - want) <= 1.01 * 2.0 ** -10 * np.abs(want)).all()


@pytest.mark.parametrize("type_", TYPES)
def test_move_to_rows_near_the_largest_int(type_):
    """Rows begin + i outside the cache are skipped, wherever begin is; those inside are moved."""
    cache = new_cache(type_, 3, 2, 64, 16)
    fill(cache, np.random.default_rng(1), 16)
    k, v = syn.kv_read(cache, 16)
    path = np.array([[9, 10, 11], [9, 10, 11], [9, 10, 11]], np.int32)
    begin = np.array([2**31 - 2, -2, -2**31], np.int32)  # the second: rows -2, -1 and 0
    syn.kv_move(cache, gpu(path), gpu(np.array([3, 3, 3], np.int32)), gpu(begin))
    for x, y in zip((k, v), syn.kv_read(cache, 16)):
        x[1, 0] = x[1, 11]
        assert torch.equal(x, y)
