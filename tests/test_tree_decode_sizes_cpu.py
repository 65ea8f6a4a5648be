"""Sizes of the tree operators near the largest int, which need no GPU."""
import synapse_b200 as syn


def test_lengths_whose_tiles_would_pass_the_largest_int_are_refused():
    b = syn.lib().syn_tree_attention_scratch_bytes
    for n_tree in (1, 64):
        assert b(1, n_tree, 8, 1, 8, 2**31 - 1) == 0 and b(1, n_tree, 8, 1, 8, 2**31 - 1024) == 0
        assert b(1, n_tree, 8, 1, 8, 2**31 - 1025) >= 4096
