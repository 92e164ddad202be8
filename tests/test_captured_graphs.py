"""Decode graphs that are kept while other work asks for longer tables or more scratch."""
import asyncio
import gc

import numpy as np
import pytest
import torch

from oracle.decoder import random_decoder_weights
from shardcompute_amd.executor import BlockDecodeGraph, DecodeGraph
from tests.test_gpu_model import SHAPE, build_model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def weights():
    return random_decoder_weights(SHAPE, seed=0)


def run(coro):
    return asyncio.run(coro)


def fill_memory(shape, n):
    """Fresh tensors where freed ones of their size lay."""
    gc.collect()
    return [torch.full(shape, float("nan"), device="cuda") for _ in range(n)]


def block_decoder(model, prompts, n):
    cache = model.new_block_cache(len(prompts), 128)
    logits = run(model.forward_blocks([t for p in prompts for t in p], cache.begin([len(p) for p in prompts])))
    out = torch.zeros((len(prompts), n), dtype=torch.int32, device="cuda")
    dec = BlockDecodeGraph(model, cache, out)
    out[:, 0] = dec.bufs.ids[:, 0] = logits.float().argmax(-1).to(torch.int32)
    dec.step.fill_(1)
    return dec, out


def dense_decoder(model, prompts, n):
    """The per-op graph over a dense cache: prompts of one length."""
    ids = torch.tensor(prompts, device="cuda")
    cache = model.new_cache(len(prompts), 128)
    logits, _ = run(model.forward(ids, past_key_values=cache, use_cache=True, last_only=True))
    out = torch.zeros((len(prompts), n), dtype=torch.int32, device="cuda")
    dec = DecodeGraph(model, cache, out, fused_trunk=False)
    out[:, 0] = dec.bufs.ids[:, 0] = logits.reshape(len(prompts), -1).float().argmax(-1).to(torch.int32)
    cache.counters[1:].fill_(1)
    return dec, out


@pytest.mark.parametrize("decoder", [block_decoder, dense_decoder])
def test_graph_outlives_longer_rotary_tables(device, weights, decoder):
    """Steps, a cache that needs longer rotary tables, steps again: the tokens of a run without it."""
    n = 24
    prompts = np.random.default_rng(2).integers(0, SHAPE.vocab_size, (3, 9)).tolist()
    quiet, want = decoder(build_model(SHAPE, weights), prompts, n)
    quiet.run(n - 1)
    model = build_model(SHAPE, weights)
    dec, out = decoder(model, prompts, n)
    dec.run(9)
    before = model.layers[0].attention.rope.tables(1, device)[0].shape
    big = model.new_block_cache(1, 3000)
    run(model.forward_blocks([1, 2, 3], big.begin([3])))
    assert model.layers[0].attention.rope.tables(1, device)[0].shape[0] > before[0]
    held = fill_memory(before, 4 * len(model.layers))
    dec.run(n - 10)
    assert torch.equal(out, want) and all(t.isnan().all() for t in held)
