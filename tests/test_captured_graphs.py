"""Decode graphs that are kept while other work asks for longer tables or more scratch."""
import asyncio
import gc

import numpy as np
import pytest
import torch

from oracle.decoder import random_decoder_weights
from shardcompute_amd import _lib
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


def product(g, M, N, K):
    x = torch.randn((M, K), generator=g, device="cuda").to(torch.bfloat16)
    return x, _lib.quantize(torch.randn((N, K), generator=g, device="cuda").mul_(0.02), bits=4)


def test_graph_outlives_a_larger_split_k_product(device):
    """Products that split K in a graph (9-32 rows, the band kernel), then one whose partials
    need more of the library's scratch, other allocations, and replays: the eager results."""
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    small = [product(g, 20, 128, 8192), product(g, 40, 256, 4096)]
    want = [_lib.qmm(x, *w) for x, w in small]
    outs = [torch.empty_like(y) for y in want]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for (x, w), y in zip(small, outs):
            _lib.qmm(x, *w, out=y)
    free = torch.cuda.mem_get_info()[0]
    x, w = product(g, 1000, 4096, 14336)                      # 4 x 1000 x 4096 partials
    big = _lib.qmm(x, *w)
    torch.cuda.synchronize()
    print(f"{(free - torch.cuda.mem_get_info()[0]) >> 20} MB more held", flush=True)
    held = [torch.full((n,), 7.0, device="cuda") for n in (1 << 16, 1 << 20, 1 << 24, 1 << 26)]
    for _ in range(3):
        for y in outs:
            y.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, z) for y, z in zip(outs, want))
        assert torch.equal(_lib.qmm(x, *w), big)
    assert all((t == 7).all() for t in held)
