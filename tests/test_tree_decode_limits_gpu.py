"""The limits of synapse_b200.tree_decode: what does not fit the cache is an error, not a wrong token."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
syn = pytest.importorskip("synapse_b200")
from synapse_b200 import model as synmodel  # noqa: E402
from synapse_b200 import tree_decode as td  # noqa: E402

CFG = dict(n_layer=1, n_embd=128, n_ff=256, n_head=4, n_head_kv=2, head_dim=32, n_vocab=256, rms_eps=1e-5, rope_base=10000.0)


def decoder(n_seq, max_ctx, tree, cache=syn.F16, n_layer=1):
    cfg = dict(CFG, n_layer=n_layer)
    weights = synmodel.random_llama_weights(cfg, seed=3, type_layers=syn.F32, type_embd=syn.F32, tied=True, sigma=0.05)
    return td.TreeDecoder(cfg, weights, cache, n_seq, max_ctx, tree)


def prompts(n_seq, n):
    return np.random.default_rng(4).integers(0, CFG["n_vocab"], (n_seq, n)).tolist()


def test_steps_past_the_cache_raise():
    m = decoder(2, 20, 8)
    m.start(prompts(2, 10))  # 9 rows
    m.step(8, {})            # 17 of 20, of which one at least stays
    before = [list(h) for h in m.histories], m.lens.copy()
    with pytest.raises(ValueError, match="cache"):
        m.step(11, {})
    assert m.histories == before[0] and (m.lens == before[1]).all()
    with pytest.raises(ValueError, match="cache"):
        m.start(prompts(2, 30))


def test_decode_fills_the_cache_to_its_last_row_and_no_further():
    """Sequences that draft well wait for the others, within a cache of just the prompt, the steps and a tree."""
    steps, tree, p = 30, 6, prompts(3, 5)
    m = decoder(3, 5 + steps + tree - 1, tree)
    one, _ = td.decode(m, p, steps, 1, {})
    m.corpus = [p[0] + one[0], [], []]  # the first sequence's drafts are all confirmed
    many, passes = td.decode(m, p, steps, tree, {})
    assert many == one and passes <= steps
    assert [len(h) for h in m.histories] == [5 + steps] * 3 and m.lens.tolist() == [4 + steps] * 3


@pytest.mark.parametrize("n", [1, 2, 1025, 1026, 2500])
def test_prompts_of_any_length(n):
    """A prompt of more tokens than a tree may have leaves the rows that its tokens leave in chains of 100."""
    m, by_100 = decoder(2, n + 4, 4, n_layer=2), decoder(2, n + 4, 4, n_layer=2)
    p = prompts(2, n)
    m.start(p)
    assert m.lens.tolist() == [n - 1] * 2
    for i in range(0, n - 1, 100):
        part = np.array([x[i:min(i + 100, n - 1)] for x in p], np.int32)
        by_100.forward(part, [list(range(-1, part.shape[1] - 1))] * 2)
        by_100.lens += part.shape[1]
    if n > 1:
        for x, y in zip(syn.kv_read(m.cache, n - 1, layer=1), syn.kv_read(by_100.cache, n - 1, layer=1)):
            assert (x - y).abs().max() <= 2.0 ** -10 * x.abs().max()  # a value may round to the neighbouring binary16
    assert all(len(new) >= 1 for new in m.step(4, {}))


def test_rules_that_leave_no_token_raise():
    m = decoder(2, 40, 4)
    m.start(prompts(2, 6))
    before = [list(h) for h in m.histories], m.lens.copy()
    with pytest.raises(ValueError, match="no token"):
        m.step(4, {"allowed": torch.zeros(1, CFG["n_vocab"] // 32, dtype=torch.int32, device="cuda")})
    assert m.histories == before[0] and (m.lens == before[1]).all()
    assert all(0 <= t < CFG["n_vocab"] for new in m.step(4, {}) for t in new)
