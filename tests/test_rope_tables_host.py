"""The rotary tables a captured graph reads outlive a longer request."""
import gc
import weakref

import torch

from shardcompute_amd.parallel.attention import RoPE

CPU = torch.device("cpu")


def test_tables_replaced_by_longer_ones_stay_alive():
    rope = RoPE(64, max_position_embeddings=100)
    seen = []
    for length in (300, 5000, 5001, 300, 40000):
        pair = rope.tables(length, CPU)
        assert pair[0].shape == pair[1].shape and pair[0].shape[0] >= length
        seen += [(weakref.ref(t), t.data_ptr(), t.clone()) for t in pair]
        del pair
    gc.collect()
    for ref, ptr, values in seen:
        assert ref() is not None and ref().data_ptr() == ptr and torch.equal(ref(), values)
    # a request that fits takes what is there
    assert rope.tables(7, CPU)[0] is rope.tables(40000, CPU)[0]


def test_all_tables_together_are_at_most_twice_the_longest():
    rope = RoPE(64, max_position_embeddings=1)
    sizes = {}
    for length in range(1, 9000, 97):
        c, _ = rope.tables(length, CPU)
        sizes[c.data_ptr()] = c.shape[0]
    assert sum(sizes.values()) <= 2 * max(sizes.values())
