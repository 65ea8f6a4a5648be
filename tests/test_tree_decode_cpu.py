"""Sizes of the KV caches and of the tree operators' scratches, which need no GPU."""
import synapse_b200 as syn


def test_kv_cache_bytes():
    assert syn.kv_cache_bytes(syn.F16, 8, 128, 100) == 8 * 128 * 100 * 2
    assert syn.kv_cache_bytes(syn.F16, 3, 48, 7) == 3 * 48 * 7 * 2
    up = lambda n: (n + 255) // 256 * 256  # noqa: E731
    assert syn.kv_cache_bytes(syn.Q8_0, 2, 64, 33) == up(2 * 64 * 33) + up(2 * 33 * 2 * 2)
    assert syn.kv_cache_bytes(syn.Q4_0, 2, 64, 33) == up(2 * 64 * 33 // 2) + up(2 * 33 * 2 * 2)
    for bad in ((syn.F32, 2, 64, 8), (syn.Q4_K, 2, 64, 8), (syn.Q8_0, 2, 48, 8), (syn.F16, 2, 44, 8), (syn.Q8_0, 2, 288, 8),
                (syn.Q8_0, 0, 64, 8), (syn.Q8_0, 2, 64, 0)):
        assert syn.kv_cache_bytes(*bad) == 0, bad


def test_scratch_bytes():
    b = syn.lib().syn_tree_attention_scratch_bytes
    assert b(1, 1, 32, 8, 128, 4096) > 4096 and b(1, 1, 32, 8, 128, 16) >= 4096
    assert b(4, 16, 32, 8, 128, 4096) > b(1, 1, 32, 8, 128, 4096)
    for bad in ((0, 1, 32, 8, 128, 64), (1, 0, 32, 8, 128, 64), (1, 1, 30, 8, 128, 64), (1, 1, 32, 8, 264, 64), (1, 65, 32, 8, 128, 64),
                (1, 2000, 32, 8, 128, 4096)):
        assert b(*bad) == 0, bad
    assert syn.lib().syn_logits_scratch_bytes(0) == 0 and syn.lib().syn_logits_scratch_bytes(100) >= 1200
