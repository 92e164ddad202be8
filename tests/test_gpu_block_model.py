"""The decoder over a block cache: ragged prompts behind a shared prefix against the same
model's dense path, sequence by sequence, on the small GQA decoder of test_gpu_model."""
import asyncio

import numpy as np
import pytest
import torch

from oracle.bf16 import bf16_to_f32
from oracle.decoder import random_decoder_weights
from shardcompute_amd.executor import BlockDecodeGraph, ParallelExecutor
from tests.gpu_util import host_u16
from tests.test_gpu_model import LOGIT_TOL, SHAPE, build_model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")
    return build_model(SHAPE, random_decoder_weights(SHAPE, seed=0))


def run(coro):
    return asyncio.run(coro)


def f32(t):
    return bf16_to_f32(host_u16(t.reshape(-1, t.shape[-1])))


def dense(model, ids):
    """Logits of every position of one sequence by the dense path."""
    logits, _ = run(model.forward(torch.tensor([ids])))
    return f32(logits)


def tokens(rng, n):
    return rng.integers(0, SHAPE.vocab_size, n).tolist()


def close(a, b):
    # both paths carry the roundings the oracle comparison's bar was set for, each against exact
    return np.abs(a - b).max() <= 2 * LOGIT_TOL * np.abs(b).max()


@pytest.mark.parametrize("prefix,lens,bs", [(0, [5, 1, 40], 16), (70, [1, 33, 2, 17], 64), (64, [9], 32),
                                            (33, [3] * 12, 16)])
def test_ragged_step_matches_dense(model, prefix, lens, bs):
    print(f"blocks prefix={prefix} lens={lens} bs={bs}", flush=True)
    rng = np.random.default_rng(len(lens))
    pre, own = tokens(rng, prefix), [tokens(rng, n) for n in lens]
    cache = model.new_block_cache(len(lens), 96, block_size=bs, max_prefix=prefix)
    if prefix:
        # the prefix in two pieces
        cut = prefix // 3
        run(model.forward_blocks(pre[:cut], cache.begin_prefix(cut)))
        run(model.forward_blocks(pre[cut:], cache.begin_prefix(prefix - cut)))
    got = run(model.forward_blocks([t for p in own for t in p], cache.begin(lens), all_rows=True))
    want = [dense(model, pre + p) for p in own]
    g, at = f32(got), 0
    for w, n in zip(want, lens):
        assert close(g[at:at + n], w[prefix:])
        at += n
    # some sequences get further positions, the others wait
    more = [tokens(rng, (3 * i) % 4) for i in range(len(lens))]
    step = cache.begin([len(m) for m in more])
    if step.rows:
        last = f32(run(model.forward_blocks([t for m in more for t in m], step)))
        for i, (p, m) in enumerate(zip(own, more)):
            if m:
                assert close(last[i], dense(model, pre + p + m)[-1])
    # the first sequence gives its blocks back and another takes its place
    again = tokens(rng, 20)
    release = [True] + [False] * (len(lens) - 1)
    last = f32(run(model.forward_blocks(again, cache.begin([20] + [0] * (len(lens) - 1), release=release))))
    assert close(last[0], dense(model, pre + again)[-1])
    cache.check_status()
    assert cache.host_lengths == cache.lengths.tolist() and cache.host_free == cache.n_free.item()
    assert cache.host_prefix == cache.prefix_len.item() == prefix


@pytest.mark.parametrize("prefix,lens", [(50, [4, 1, 23]), (0, [7, 30])])
@pytest.mark.parametrize("graphs", [True, False])
def test_greedy_batch_follows_dense_logits(model, prefix, lens, graphs):
    """Each token is the dense path's argmax up to the logits' tolerance, teacher-forced."""
    rng = np.random.default_rng(7)
    pre, prompts, n = tokens(rng, prefix), [tokens(rng, m) for m in lens], 40
    ex = ParallelExecutor(0, 1, None, model, use_graphs=graphs)
    out = run(ex.generate_batch(prompts, prefix=pre, max_new_tokens=n))
    assert [len(t) for t in out] == [n] * len(lens)
    for p, t in zip(prompts, out):
        logits = dense(model, pre + p + t)
        at = len(pre) + len(p) - 1
        for i, tok in enumerate(t):
            row = logits[at + i]
            assert row[tok] >= row.max() - 2 * LOGIT_TOL * np.abs(row).max(), (i, tok)
    # graph and eager steps are the same launches: the same tokens
    other = ParallelExecutor(0, 1, None, model, use_graphs=not graphs)
    assert run(other.generate_batch(prompts, prefix=pre, max_new_tokens=n)) == out


def test_stop_tokens_and_samples(model):
    rng = np.random.default_rng(3)
    pre, prompts = tokens(rng, 40), [tokens(rng, 3), tokens(rng, 8)]
    ex = ParallelExecutor(0, 1, None, model)
    full = run(ex.generate_batch(prompts, prefix=pre, max_new_tokens=30))
    stop = [full[0][5], full[1][20]]
    got = run(ex.generate_batch(prompts, prefix=pre, max_new_tokens=30, stop_tokens=stop))
    for f, g in zip(full, got):
        end = next((i + 1 for i, t in enumerate(f) if t in stop), 30)
        assert g == f[:end]
    # samples of one prompt: every token within the vocabulary, the asked number
    s = run(ex.generate_batch([prompts[0]] * 5, prefix=pre, max_new_tokens=6, temperature=0.8))
    assert len(s) == 5 and all(len(t) == 6 and all(0 <= x < SHAPE.vocab_size for x in t) for t in s)
    assert run(ex.generate_batch(prompts, max_new_tokens=0)) == [[], []]


def test_refusals(model):
    ex = ParallelExecutor(0, 1, None, model)
    with pytest.raises(ValueError, match="at least one token"):
        run(ex.generate_batch([[1], []]))
    with pytest.raises(ValueError, match="at least one token"):
        run(ex.generate_batch([]))
    cache = model.new_block_cache(2, 64, num_blocks=3, block_size=16, max_prefix=32)
    before = cache.n_free.item()
    with pytest.raises(RuntimeError, match="full"):
        cache.begin([40, 20])
    with pytest.raises(RuntimeError, match="table has room"):
        cache.begin([65, 0])
    with pytest.raises(RuntimeError, match="exceeds"):
        cache.begin_prefix(33)
    with pytest.raises(ValueError, match="every one"):
        cache.begin([1])
    assert cache.n_free.item() == before and cache.lengths.tolist() == [0, 0]
    step = cache.begin([2, 1])
    with pytest.raises(ValueError, match="step's rows"):
        run(model.forward_blocks([1, 2], step))
    with pytest.raises(RuntimeError, match="before the sequences"):
        cache.begin_prefix(1)
    layer = model.layers[0].attention
    qkv = torch.zeros((3, layer.qkv_width), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="no attention mask"):
        layer.attend_qkv(qkv, 1, 3, step[0], mask=torch.zeros((1, 3), device="cuda"))
    with pytest.raises(ValueError, match="3 rows"):
        layer.attend_qkv(qkv[:2], 1, 2, step[0])


def test_a_step_that_only_gives_back_and_one_that_is_over(model):
    cache = model.new_block_cache(3, 64, block_size=16)
    free = cache.host_free
    first = cache.begin([17, 1, 0])
    run(model.forward_blocks([3] * 18, first))
    second = cache.begin([1, 1, 1])
    with pytest.raises(RuntimeError, match="another step"):
        run(model.forward_blocks([3] * 18, first))
    run(model.forward_blocks([3] * 3, second))
    none = cache.begin([0, 0, 0], release=[True, False, True])
    with pytest.raises(ValueError, match="no rows"):
        run(model.forward_blocks([], none))
    assert cache.lengths.tolist() == cache.host_lengths == [0, 2, 0]
    assert cache.n_free.item() == cache.host_free == free - 1
    cache.check_status()


def test_decode_graph_made_before_its_prefix(model):
    rng = np.random.default_rng(11)
    pre, prompts, n = tokens(rng, 45), [tokens(rng, 5), tokens(rng, 2)], 12
    want = run(ParallelExecutor(0, 1, None, model).generate_batch(prompts, prefix=pre, max_new_tokens=n))
    cache = model.new_block_cache(2, 128, block_size=64, max_prefix=64)
    out = torch.zeros((2, n), dtype=torch.int32, device="cuda")
    dec = BlockDecodeGraph(model, cache, out)
    run(model.forward_blocks(pre, cache.begin_prefix(len(pre))))
    logits = run(model.forward_blocks(prompts[0] + prompts[1], cache.begin([5, 2])))
    out[:, 0] = dec.bufs.ids[:, 0] = logits.float().argmax(-1).to(torch.int32)
    dec.step.fill_(1)
    dec.run(n - 1)
    cache.check_status()
    assert out.tolist() == want


@pytest.mark.parametrize("prefix", [0, 70])
def test_positions_up_to_the_tables_room(device, prefix):
    """A sequence past max_length, up to the room of its table, behind more positions than the
    model's rotary tables hold by themselves."""
    m = build_model(SHAPE, random_decoder_weights(SHAPE, seed=0))
    rng = np.random.default_rng(5)
    pre, own, more = tokens(rng, prefix), tokens(rng, 255), tokens(rng, 200)
    cache = m.new_block_cache(1, 260, block_size=256, max_prefix=prefix)
    if prefix:
        run(m.forward_blocks(pre, cache.begin_prefix(prefix)))
    run(m.forward_blocks(own, cache.begin([255])))
    got = f32(run(m.forward_blocks(more, cache.begin([200]), all_rows=True)))
    assert close(got, dense(m, pre + own + more)[prefix + 255:])
    with pytest.raises(RuntimeError, match="room for 512"):
        cache.begin([58])
