"""The decoder over a block cache of 4- or 8-bit codes: the same model over a bf16 block cache whose
keys and values a test replaces by the ones the codes stand for."""
import asyncio

import numpy as np
import pytest
import torch

from oracle.decoder import random_decoder_weights
from shardcompute_amd import _lib
from shardcompute_amd.executor import BlockDecodeGraph, ParallelExecutor
from tests.test_gpu_block_model import close, f32, tokens
from tests.test_gpu_model import LOGIT_TOL, SHAPE, build_model

pytestmark = pytest.mark.gpu
BITS = [4, 8]


@pytest.fixture(scope="module")
def model():
    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")
    return build_model(SHAPE, random_decoder_weights(SHAPE, seed=0))


def run(coro):
    return asyncio.run(coro)


def rounded(x, bits):
    wq, s, b = _lib.quantize(x.float().reshape(-1, x.shape[-1]).contiguous(), bits=bits)
    return _lib.dequantize(wq, s, b, bits=bits).view(x.shape)


@pytest.fixture
def emulate(monkeypatch):
    """A bf16 block cache that holds quantized keys and values: what the append wrote is replaced."""
    def patch(bits):
        append = _lib.rope_append_blocks

        def both(qkv, H, Hkv, D, cos, sin, k, vt, slots, positions, out=None):
            q = append(qkv, H, Hkv, D, cos, sin, k, vt, slots, positions, out=out)
            s = slots[slots >= 0].long()
            b, off = s // k.shape[2], s % k.shape[2]
            k[b, :, off] = rounded(k[b, :, off], bits)
            vt[b, :, :, off] = rounded(vt[b, :, :, off], bits)
            return q
        monkeypatch.setattr(_lib, "rope_append_blocks", both)
    return patch


@pytest.mark.parametrize("prefix,lens,bs", [(0, [5, 1, 40], 16), (70, [1, 33, 2, 17], 64), (33, [3] * 12, 16)])
@pytest.mark.parametrize("bits", BITS)
def test_ragged_steps(model, emulate, prefix, lens, bs, bits):
    print(f"quantized blocks {bits} bits prefix={prefix} lens={lens} bs={bs}", flush=True)
    rng = np.random.default_rng(len(lens))
    pre, own = tokens(rng, prefix), [tokens(rng, n) for n in lens]
    more = [tokens(rng, (3 * i) % 4) for i in range(len(lens))]
    again = tokens(rng, 20)

    def steps(cache):
        out = []
        if prefix:
            cut = prefix // 3
            run(model.forward_blocks(pre[:cut], cache.begin_prefix(cut)))
            out.append(f32(run(model.forward_blocks(pre[cut:], cache.begin_prefix(prefix - cut)))))
        out.append(f32(run(model.forward_blocks([t for p in own for t in p], cache.begin(lens), all_rows=True))))
        step = cache.begin([len(m) for m in more])
        if step.rows:
            out.append(f32(run(model.forward_blocks([t for m in more for t in m], step, all_rows=True))))
        # the first sequence gives its blocks back and another takes its place
        release = [True] + [False] * (len(lens) - 1)
        step = cache.begin([20] + [0] * (len(lens) - 1), release=release)
        out.append(f32(run(model.forward_blocks(again, step)))[:1])
        cache.check_status()
        return out

    cache = model.new_block_cache(len(lens), 96, block_size=bs, max_prefix=prefix, bits=bits)
    got = steps(cache)
    whole = model.new_block_cache(len(lens), 96, block_size=bs, max_prefix=prefix)
    assert cache.nbytes * 16 == whole.nbytes * (bits + 0.5)
    emulate(bits)
    for a, b in zip(got, steps(whole)):
        assert close(a, b)


@pytest.mark.parametrize("bits", BITS)
def test_sequences_as_tuples(model, bits):
    """One sequence's keys and values behind the prefix, in the reference's layout; in the first
    layer those of the bf16 cache after the same steps, quantized."""
    rng = np.random.default_rng(2)
    pre, own = tokens(rng, 37), [tokens(rng, 21), tokens(rng, 3), tokens(rng, 40)]
    got = []
    for b in (bits, None):
        cache = model.new_block_cache(4, 64, block_size=16, max_prefix=48, bits=b)
        run(model.forward_blocks(pre, cache.begin_prefix(37)))
        run(model.forward_blocks([t for p in own for t in p], cache.begin([21, 3, 0, 40])))
        got.append([cache.as_tuple(0, r) for r in range(4)])
        with pytest.raises(IndexError):
            cache.as_tuple(0, 4)
    for r, ((k, v), (kw, vw)) in enumerate(zip(*got)):
        assert k.shape == v.shape == (1, SHAPE.num_kv_heads, 37 + [21, 3, 0, 40][r], SHAPE.head_dim)
        assert torch.equal(k, rounded(kw, bits)) and torch.equal(v, rounded(vw, bits))


@pytest.mark.parametrize("prefix,lens", [(50, [4, 1, 23]), (0, [7, 30])])
@pytest.mark.parametrize("bits", BITS)
def test_greedy_batch(model, emulate, prefix, lens, bits):
    """Graph and eager steps give the same tokens; each is the emulated cache's argmax up to the
    logits' tolerance, teacher-forced."""
    rng = np.random.default_rng(7)
    pre, prompts, n = tokens(rng, prefix), [tokens(rng, m) for m in lens], 24
    ex = ParallelExecutor(0, 1, None, model)
    out = run(ex.generate_batch(prompts, prefix=pre, max_new_tokens=n, kv_bits=bits))
    assert [len(t) for t in out] == [n] * len(lens)
    eager = ParallelExecutor(0, 1, None, model, use_graphs=False)
    assert run(eager.generate_batch(prompts, prefix=pre, max_new_tokens=n, kv_bits=bits)) == out
    sampled = run(ex.generate_batch(prompts, prefix=pre, max_new_tokens=4, temperature=0.7, kv_bits=bits))
    assert all(len(t) == 4 and all(0 <= x < SHAPE.vocab_size for x in t) for t in sampled)
    emulate(bits)
    cache = model.new_block_cache(len(lens), 64, block_size=64, max_prefix=prefix)
    if prefix:
        run(model.forward_blocks(pre, cache.begin_prefix(prefix)))
    rows = [p + t[:-1] for p, t in zip(prompts, out)]
    logits = f32(run(model.forward_blocks([x for r in rows for x in r], cache.begin([len(r) for r in rows]), all_rows=True)))
    at = 0
    for p, t, r in zip(prompts, out, rows):
        for i, tok in enumerate(t):
            row = logits[at + len(p) - 1 + i]
            assert row[tok] >= row.max() - 2 * LOGIT_TOL * np.abs(row).max(), (i, tok)
        at += len(r)


def test_two_graphs_of_one_cache_in_turn(model):
    """Two decode graphs of one quantized cache, replayed in turn, follow the eager steps."""
    rng = np.random.default_rng(11)
    prompts, n = [tokens(rng, 5), tokens(rng, 2)], 9
    want = run(ParallelExecutor(0, 1, None, model, use_graphs=False).generate_batch(prompts, max_new_tokens=n, kv_bits=4))
    cache = model.new_block_cache(2, 128, block_size=64, bits=4)
    out = torch.zeros((2, n), dtype=torch.int32, device="cuda")
    graphs = [BlockDecodeGraph(model, cache, out) for _ in range(2)]
    logits = run(model.forward_blocks(prompts[0] + prompts[1], cache.begin([5, 2])))
    first = logits.float().argmax(-1).to(torch.int32)
    out[:, 0] = first
    graphs[0].bufs.ids[:, 0] = first
    graphs[0].step.fill_(1)
    for i in range(1, n):
        g, other = graphs[(i - 1) % 2], graphs[i % 2]
        g.run(1)
        other.bufs.ids.copy_(g.bufs.ids)
        other.step.copy_(g.step)
    cache.check_status()
    assert out.tolist() == want


def test_refusals(model):
    with pytest.raises(ValueError, match="bits"):
        model.new_block_cache(2, 64, bits=6)
    with pytest.raises(ValueError, match="bits"):
        run(ParallelExecutor(0, 1, None, model).generate_batch([[1]], kv_bits=16))
