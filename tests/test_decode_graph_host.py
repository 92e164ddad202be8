"""What the decode graphs leave behind when a capture fails (no GPU calls)."""
import os

import pytest
import torch

from shardcompute_amd import executor
from shardcompute_amd.block_cache import BlockKVCache
from shardcompute_amd.build import LIB_PATH
from shardcompute_amd.executor import BlockDecodeGraph, DecodeGraph
from shardcompute_amd.kv_cache import KVCache

pytestmark = pytest.mark.skipif(not os.path.exists(LIB_PATH), reason="library not built")


def no_memory(*a, **kw):
    raise RuntimeError("out of memory")


def test_block_cache_counts_the_step_before_a_capture_that_fails(monkeypatch):
    """The first step has run on the device when its graph is captured: the host's lengths, free
    blocks and step number are those after it, also if the capture raises."""
    cache = BlockKVCache(1, 1, 64, num_blocks=4, max_sequences=2, max_length=64, block_size=16, device=torch.device("cpu"))
    cache.host_lengths, cache.host_free = [16, 3], 2
    dec = BlockDecodeGraph.__new__(BlockDecodeGraph)
    dec.cache, dec.use_graph, dec.graph, dec.logits = cache, True, None, None
    steps = []
    dec._step = lambda: steps.append(1) or len(steps)
    monkeypatch.setattr(executor.torch.cuda, "synchronize", no_memory)
    with pytest.raises(RuntimeError, match="out of memory"):
        dec.run(3)
    assert len(steps) == 1 and dec.logits == 1
    assert cache.host_lengths == [17, 4] and cache.host_free == 1 and cache.steps == 1
    # without graphs it goes on from there
    dec.use_graph = False
    dec.run(2)
    assert len(steps) == 3 and cache.host_lengths == [19, 6] and cache.steps == 3


def test_dense_cache_counts_the_step_before_a_capture_that_fails(monkeypatch):
    cache = KVCache(1, 1, 1, 64, 64, device=torch.device("cpu"))
    cache.length = 5
    dec = DecodeGraph.__new__(DecodeGraph)
    dec.cache, dec.use_graph, dec.steps_per_graph, dec.graph, dec.graph_n = cache, True, 8, None, None
    lengths = []

    def step():
        lengths.append(cache.length)
        dec.logits = len(lengths)
    dec._step = step
    monkeypatch.setattr(executor.torch.cuda, "synchronize", no_memory)
    with pytest.raises(RuntimeError, match="out of memory"):
        dec.run(2)
    assert lengths == [5] and dec.logits == 1 and cache.length == 6
    dec.use_graph = False
    dec.run(2)
    assert lengths == [5, 6, 7] and cache.length == 8
