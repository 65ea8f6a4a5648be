"""The tree operators together (synapse_b200.tree_decode): decoding by trees of drafted tokens gives the tokens of
decoding one at a time, in fewer passes, over every cache type."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
syn = pytest.importorskip("synapse_b200")
from synapse_b200 import model as synmodel  # noqa: E402
from synapse_b200 import tree_decode as td  # noqa: E402


@pytest.mark.parametrize("cache", ["f16", "q8_0", "q4_0"])
@pytest.mark.parametrize("tree,n_head,n_kv,hd", [(12, 8, 2, 64), (5, 4, 4, 32)])
def test_trees_decode_what_single_tokens_do(cache, tree, n_head, n_kv, hd):
    cfg = dict(n_layer=2, n_embd=256, n_ff=512, n_head=n_head, n_head_kv=n_kv, head_dim=hd, n_vocab=512, rms_eps=1e-5, rope_base=10000.0)
    weights = synmodel.random_llama_weights(cfg, seed=3, type_layers=syn.F32, type_embd=syn.F32, tied=True, sigma=0.05)
    prompts = np.random.default_rng(4).integers(0, 512, (2, 10)).tolist()
    rules = td.default_rules(torch, cfg, 2, seed=5)
    m = td.TreeDecoder(cfg, weights, td.CACHES[cache], 2, 120, tree)
    one, passes = td.decode(m, prompts, 40, 1, rules)
    assert passes == 40
    m.corpus = td.changed([p + o for p, o in zip(prompts, one)], 512)
    many, fewer = td.decode(m, prompts, 40, tree, rules)
    assert many == one and fewer < 30
    # what is committed is what single tokens commit: the last layer's rows
    n = 10 + 38
    m.corpus = [()] * 2
    td.decode(m, prompts, 40, 1, rules)
    k1, v1 = syn.kv_read(m.cache, n, layer=1)
    m.corpus = td.changed([p + o for p, o in zip(prompts, one)], 512)
    td.decode(m, prompts, 40, tree, rules)
    k2, v2 = syn.kv_read(m.cache, n, layer=1)
    step = {"f16": 2.0 ** -10, "q8_0": 2.5 / 127, "q4_0": 2.5 / 8}[cache]  # a value may round to the neighbouring quant
    for x, y in ((k1, k2), (v1, v2)):
        assert (x - y).abs().max() <= step * x.abs().max()


def test_tree_helpers():
    words, depth = td.tree_mask([-1, 0, 0, 1, 3])
    assert words[:, 0].tolist() == [1, 3, 5, 11, 27] and depth.tolist() == [0, 1, 1, 2, 3]
    tokens, parents = td.draft_pairs([1, 2, 3, 1, 2, 4, 1], 6)
    assert tokens[0] == 1 and parents[0] == -1 and len(tokens) == len(parents) == 6
    assert all(0 <= p < i for i, p in enumerate(parents) if i)
    assert (tokens[1], parents[1]) == (2, 0)
    assert td.draft_pairs([7], 3) == ([7, 7, 7], [-1, 0, 0])
