"""The tree operators in a captured graph, and over a session's own caches."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
syn = pytest.importorskip("synapse_b200")
from synapse_b200 import model  # noqa: E402
from tests.test_tree_decode_gpu import fill, gpu, new_cache, random_masks  # noqa: E402

TYPES = [syn.F16, syn.Q8_0, syn.Q4_0]


# (n_head, tree): one row and a few, joined by the last CTA; more, by the second kernel; on tcgen05
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("n_head,tree", [(2, 1), (4, 2), (6, 4), (24, 4)])
def test_a_captured_step_serves_every_length(type_, n_head, tree):
    """Append, attention, logits and move captured once and replayed over contexts of other lengths, with other inputs:
    what the same calls give outside the graph."""
    rng = np.random.default_rng(tree)
    n_seq, n_kv, hd, ctx = 2, 2, 64, 3000
    base = new_cache(type_, n_seq, n_kv, hd, ctx, n_layer=2)
    for layer in range(2):
        fill(base, rng, ctx, layer=layer)
    words, _ = random_masks(rng, n_seq, tree)
    mask, table = gpu(words), syn.rope_table(ctx, hd, 0.9)
    path_step = np.arange(tree)[::2]  # the nodes kept: every second

    def inputs(seed, lens):
        r = np.random.default_rng(seed)
        x = {n: gpu(r.standard_normal((n_seq * tree, h * hd), dtype=np.float32)) for n, h in (("q", n_head), ("k", n_kv), ("v", n_kv))}
        lens = np.array(lens, np.int32)
        x["len"] = gpu(lens)
        x["slot"] = gpu((lens[:, None] + np.arange(tree, dtype=np.int32)).reshape(-1))
        x["path"] = gpu((lens[:, None] + path_step).astype(np.int32))
        x["draft"] = gpu(r.integers(0, n_head * hd, (n_seq, tree)).astype(np.int32))
        return x

    def step(cache, x, attn_scratch, pick_scratch, count, pen):
        q = syn.kv_append(cache, x["k"], x["v"], x["slot"], rope_table=table, q=x["q"], layer=1)
        o = syn.tree_attention(cache, q, x["len"], n_head, 0.125, tree=tree, mask=mask, scratch=attn_scratch, layer=1)
        out, pick = syn.logits_process(o, n_seq, penalties=pen, draft=x["draft"], mask=mask, scratch=pick_scratch)
        syn.kv_move(cache, x["path"], count, x["len"])
        return q, o, out, pick

    cache = new_cache(type_, n_seq, n_kv, hd, ctx, n_layer=2)
    held = inputs(0, [5, 17])
    fixed = (syn.tree_attention_scratch(cache, tree, n_head), syn.logits_scratch(n_seq * tree),
             gpu(np.full(n_seq, len(path_step), np.int32)), gpu(np.array([[1.2, 0.1, 0.05]] * n_seq, np.float32)))
    step(cache, held, *fixed)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(cache, held, *fixed)
    for seed, lens in ((1, [0, 1]), (2, [ctx - tree, 700]), (3, [1500, 2900])):
        x = inputs(seed, lens)
        for n, t in x.items():
            held[n].copy_(t)
        for c in ("k", "v"):
            getattr(cache, c).copy_(getattr(base, c))
        graph.replay()
        plain = new_cache(type_, n_seq, n_kv, hd, ctx, n_layer=2)
        for c in ("k", "v"):
            getattr(plain, c).copy_(getattr(base, c))
        want = step(plain, x, *fixed)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert torch.equal(cache.k, plain.k) and torch.equal(cache.v, plain.v)


class Raw:
    """Device memory at an address, as bytes."""

    def __init__(self, at, n):
        self.__cuda_array_interface__ = {"data": (at, False), "shape": (n,), "typestr": "|u1", "version": 2}


def test_a_sessions_caches_as_they_are(tmp_path):
    """A syn_kv_cache that describes a session's F16 caches: rows read back and attended to are the session's own."""
    cfg = dict(n_layer=3, n_embd=128, n_ff=256, n_head=4, n_head_kv=2, head_dim=32, n_vocab=256, rms_eps=1e-5, rope_base=10000.0)
    p = tmp_path / "m.gguf"
    model.write_llama_gguf(str(p), cfg, model.random_llama_weights(cfg, seed=2), context_length=64)
    ctx, n_seq, n = 48, 2, 9
    s = syn.Session.open_ex(p, max_ctx=ctx, max_seqs=n_seq, max_batch=n_seq)
    for i in range(n):
        s.step_batch([i + 1, 100 + i], [i, i])
    torch.cuda.synchronize()
    at = [[s.kv_ptr(layer, w) for layer in range(3)] for w in (0, 1)]
    size = ctx * 2 * 32 * 2
    assert syn.kv_cache_bytes(syn.F16, 2, 32, ctx) == size and at[0][1] - at[0][0] == at[0][2] - at[0][1] == at[1][1] - at[1][0]
    desc = syn.KVCacheDesc(k=at[0][0], v=at[1][0], seq_stride=size, layer_stride=at[0][1] - at[0][0], type=syn.F16, n_layer=3, n_seq=n_seq,
                           n_kv=2, head_dim=32, max_ctx=ctx)
    q = gpu(np.random.default_rng(0).standard_normal((n_seq, 4 * 32), dtype=np.float32))
    lens = gpu(np.full(n_seq, n - 1, np.int32))
    for layer in range(3):
        raw = [torch.as_tensor(Raw(at[w][layer], n_seq * size), device="cuda").view(n_seq, size) for w in (0, 1)]
        copy = syn.KVCache.over(syn.F16, raw[0].clone(), raw[1].clone(), 2, 32, ctx)
        k, v = (torch.empty(n_seq, n, 2, 32, device="cuda") for _ in "kv")
        assert syn.lib().syn_kv_read(ctypes.byref(desc), layer, None, 0, n, syn.F32, k.data_ptr(), v.data_ptr(), syn._stream()) == 0
        want = syn.kv_read(copy, n)
        assert torch.equal(k, want[0]) and torch.equal(v, want[1]) and k.any(-1).all() and v.any(-1).all()
        out = torch.empty_like(q)
        scratch = syn.tree_attention_scratch(copy, 1, 4)
        a = syn.TreeAttentionArgs(q=q.data_ptr(), out=out.data_ptr(), len=lens.data_ptr(), scratch=scratch.data_ptr(), n_tree=1, n_head=4,
                                  max_len=ctx, scale=0.2)
        assert syn.lib().syn_tree_attention(ctypes.byref(desc), layer, ctypes.byref(a), syn._stream()) == 0
        assert torch.equal(out, syn.tree_attention(copy, q, lens, 4, 0.2))
    s.close()
