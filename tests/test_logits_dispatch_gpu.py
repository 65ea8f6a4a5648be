"""Logit processing on every side of its dispatch, against the definition, bit for bit: long chunks whose rows are not
16-byte vectors, and histories whose counts pass 16 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
syn = pytest.importorskip("synapse_b200")
from tests.test_tree_decode_gpu import gpu, plain_logits, random_masks  # noqa: E402


def everything(rng, n_seq, tree, vocab, history):
    """(x, arguments on the GPU, the definition's arguments)"""
    rows = n_seq * tree
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    past = rng.integers(-3, vocab + 3, (n_seq, history)).astype(np.int32)
    past[:, ::3] = rng.integers(0, 9, past[:, ::3].shape)
    past_len = rng.integers(0, history + 1, n_seq).astype(np.int32)
    pen = np.stack([rng.uniform(0.8, 1.5, n_seq), rng.uniform(-0.5, 1, n_seq), rng.uniform(-0.2, 0.5, n_seq)], 1).astype(np.float32)
    draft = rng.integers(0, vocab, (n_seq, tree)).astype(np.int32)
    draft[:, tree // 2] = x.argmax(1).reshape(n_seq, tree)[:, 0]
    words, sees = random_masks(rng, n_seq, tree)
    per = [5 * s + 3 for s in range(n_seq)]
    begin = np.cumsum([0] + per).astype(np.int32)
    tokens = np.concatenate([rng.choice(vocab, n, replace=False) for n in per]).astype(np.int32)
    vals = (rng.standard_normal(tokens.size) * 5).astype(np.float32)
    allowed = rng.integers(0, 2**32, (rows, (vocab + 31) // 32), dtype=np.uint32)
    allowed[rows - 1] = 0
    kw = dict(penalties=gpu(pen), history=gpu(past), history_len=gpu(past_len), draft=gpu(draft), mask=gpu(words),
              bias=(gpu(begin), gpu(tokens), gpu(vals)), allowed=gpu(allowed.view(np.int32)))
    return x, kw, (pen, past, past_len, draft, sees, (begin, tokens, vals), allowed)


@pytest.mark.parametrize("n_seq,tree,vocab", [(16, 4, 50257), (40, 2, 9001), (10, 30, 4097), (60, 3, 8191)])
@pytest.mark.parametrize("aligned", [True, False])
def test_many_rows_of_odd_vocabularies(n_seq, tree, vocab, aligned):
    """Rows of long chunks a value at a time; unaligned: rows that start at no 16-byte boundary, in place."""
    x, kw, plain = everything(np.random.default_rng(vocab), n_seq, tree, vocab, 700)
    want, want_pick = plain_logits(x, n_seq, *plain)
    if aligned:
        out, pick = syn.logits_process(gpu(x), n_seq, **kw)
    else:
        wide = torch.full((n_seq * tree, vocab + 5), 7.0, device="cuda")
        rows = wide[:, 3:3 + vocab]
        rows.copy_(gpu(x))
        out, pick = syn.logits_process(rows, n_seq, out=rows, **kw)
        assert (wide[:, :3] == 7).all() and (wide[:, 3 + vocab:] == 7).all()
    assert np.array_equal(out.cpu().numpy().view(np.int32), want.view(np.int32))
    assert np.array_equal(pick.cpu().numpy(), want_pick) and pick[-1] == -1


@pytest.mark.parametrize("history", [65495, 65496, 65536, 70000, 200000])
def test_counts_past_16_bits(history):
    """One even token all along a history, in rows enough for long chunks (with 65495 they take them, from there on not): its odd neighbour has no count of it."""
    n_seq, tree, vocab = 2, 40, 32000
    x = np.random.default_rng(1).standard_normal((n_seq * tree, vocab)).astype(np.float32)
    past = np.full((n_seq, history), 4242, np.int32)
    past[1, ::2] = 4243
    lens = np.full(n_seq, history, np.int32)
    draft = np.full((n_seq, tree), 4242, np.int32)
    pen = np.array([[1.0, 0.5, 2.0 ** -10]] * n_seq, np.float32)
    out, pick = syn.logits_process(gpu(x), n_seq, penalties=gpu(pen), history=gpu(past), history_len=gpu(lens), draft=gpu(draft))
    want = x.copy()
    for r in range(n_seq * tree):
        s, i = divmod(r, tree)
        for t in (4242, 4243):
            c = int((past[s] == t).sum()) + (i + 1 if t == 4242 else 0)  # without a mask a node's path is the nodes up to it
            if c:
                want[r, t] = want[r, t] - (np.float32(c) * pen[s, 2] + pen[s, 1])
    assert np.array_equal(out.cpu().numpy().view(np.int32), want.view(np.int32))
    assert np.array_equal(pick.cpu().numpy(), want.argmax(1))
