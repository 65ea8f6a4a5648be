"""Logit processing at its limits, against the definition in test_tree_decode_gpu.py, bit for bit."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
syn = pytest.importorskip("synapse_b200")
from tests.test_tree_decode_gpu import gpu, plain_logits  # noqa: E402


@pytest.mark.parametrize("n_seq,vocab", [(3, 1500), (3, 9001), (60, 9000)])
def test_bias_entries_outside_the_list_are_left_out(n_seq, vocab):
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((n_seq, vocab)).astype(np.float32)
    tokens = rng.integers(0, vocab, 50).astype(np.int32)
    tokens[[3, 30, 44]] = 7  # summed in the list's order
    values = (rng.standard_normal(50) * 3).astype(np.float32)
    begin = np.full(n_seq + 1, 50, np.int32)
    begin[:3] = [-2**31, 20, 2**31 - 1]  # sequence 0 has entries 0 .. 19, 1 has 20 .. 49, 2 has none
    out, pick = syn.logits_process(gpu(x), n_seq, bias=(gpu(begin), gpu(tokens), gpu(values)))
    sums = []  # a token's biases are added up, in the list's order, before its logit
    for part in (slice(0, 20), slice(20, 50)):
        sums.append({})
        for t, v in zip(tokens[part], values[part]):
            sums[-1][t] = np.float32(sums[-1].get(t, np.float32(0)) + v)
    clamped = np.full(n_seq + 1, len(sums[0]) + len(sums[1]), np.int32)
    clamped[:2] = [0, len(sums[0])]
    bias = clamped, np.array([t for d in sums for t in d], np.int32), np.array([v for d in sums for v in d.values()], np.float32)
    want, want_pick = plain_logits(x, n_seq, None, None, None, None, None, bias, None)
    assert np.array_equal(out.cpu().numpy().view(np.int32), want.view(np.int32))
    assert np.array_equal(pick.cpu().numpy(), want_pick)


def test_bias_count_is_checked():
    x, one = torch.zeros(1, 100, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    a = syn.LogitsArgs(logits=x.data_ptr(), out=x.data_ptr(), bias_begin=one.data_ptr(), bias_token=one.data_ptr(), bias_value=x.data_ptr(),
                       n_seq=1, n_tree=1, n_vocab=100, n_bias=-1)
    assert syn.lib().syn_logits_process(ctypes.byref(a), syn._stream()) == 1
