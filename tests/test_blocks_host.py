"""Refusals of the block cache's entry points (argument checks only, no GPU calls)."""
import ctypes
import os

import pytest
import torch

from shardcompute_amd import _lib
from shardcompute_amd.build import LIB_PATH

pytestmark = pytest.mark.skipif(not os.path.exists(LIB_PATH), reason="library not built")
A = 1 << 12                     # a 16-byte aligned address nothing reads


def _tables(**kw):
    a = dict(lengths=A, new=A, release=None, tables=A, free=A, n_free=A, prefix=None, R=4, width=8, bs=64, cap=40, rows=4,
             lengths_out=A, n_free_out=A, row_starts=A, slots=A, positions=A, status=A)
    a.update(kw)
    return _lib.load().sc_block_tables_i32(*a.values(), None)


def _append(**kw):
    a = dict(qkv=A, qkv_stride=1536, q=A, q_stride=1024, N=3, H=8, Hkv=2, D=128, cos=A, sin=A, length=99, k=A, vt=A,
             n_blocks=10, bs=64, slots=A, positions=A)
    a.update(kw)
    return _lib.load().sc_rope_append_blocks_bf16(*a.values(), None)


def _attend(**kw):
    a = dict(q=A, q_stride=1024, k=A, vt=A, n_blocks=10, bs=64, row_starts=A, lengths=A, tables=A, width=4, prefix_table=A,
             prefix_width=5, prefix_len=A, out=A, out_stride=1024, N=3, R=3, H=8, Hkv=2, D=128, scale=0.1, max_new=1,
             workspace=A, workspace_bytes=1 << 30)
    a.update(kw)
    return _lib.load().sc_attention_shared_bf16(*a.values(), None)


@pytest.mark.parametrize("call,kw,message", [
    (_tables, dict(lengths=None), "null pointer"), (_tables, dict(tables=None), "null pointer"),
    (_tables, dict(status=None), "null pointer"), (_tables, dict(slots=None), "null pointer"),
    (_tables, dict(bs=48), "block size 48"), (_tables, dict(bs=8), "block size 8"), (_tables, dict(bs=512), "block size"),
    (_tables, dict(R=0), "sequences"), (_tables, dict(R=65537), "sequences"), (_tables, dict(width=0), "width"),
    (_tables, dict(width=1 << 25), "width"), (_tables, dict(cap=0), "stack"), (_tables, dict(cap=1 << 26), "stack"),
    (_tables, dict(rows=-1), "row count"),
    (_append, dict(qkv=None), "null pointer"), (_append, dict(slots=None), "null pointer"),
    (_append, dict(D=96), "head_dim 96"), (_append, dict(bs=20), "block size 20"), (_append, dict(Hkv=3), "bad shape"),
    (_append, dict(N=-1), "bad shape"), (_append, dict(n_blocks=0), "pool"), (_append, dict(n_blocks=1 << 25), "pool"),
    (_append, dict(qkv_stride=1528), "strides"), (_append, dict(qkv_stride=1540), "strides"),
    (_append, dict(q_stride=1020), "strides"), (_append, dict(k=A + 2), "aligned"), (_append, dict(cos=A + 4), "aligned"),
    (_attend, dict(q=None), "null pointer"), (_attend, dict(prefix_table=None), "null pointer"),
    (_attend, dict(prefix_len=None), "null pointer"), (_attend, dict(D=80), "head_dim 80"),
    (_attend, dict(bs=0), "block size 0"), (_attend, dict(H=9), "bad shape"), (_attend, dict(R=0), "bad shape"),
    (_attend, dict(R=2049), "bad shape"), (_attend, dict(width=0), "bad shape"), (_attend, dict(max_new=-1), "bad shape"),
    (_attend, dict(prefix_width=1 << 26), "bad shape"), (_attend, dict(n_blocks=0), "pool"),
    (_attend, dict(scale=0.0), "scale"), (_attend, dict(scale=-0.1), "scale"),
    (_attend, dict(scale=float("nan")), "scale"), (_attend, dict(scale=float("inf")), "scale"),
    (_attend, dict(q_stride=1023), "strides"), (_attend, dict(q_stride=1028), "strides"),
    (_attend, dict(out_stride=1000), "strides"), (_attend, dict(q=A + 8), "misaligned"),
    (_attend, dict(out=A + 4), "misaligned"), (_attend, dict(workspace=None), "workspace"),
    (_attend, dict(workspace_bytes=64), "workspace"), (_attend, dict(workspace=A + 8), "workspace"),
])
def test_refused(call, kw, message):
    assert call(**kw) in (-1, -2)
    assert message in _lib.load().sc_last_error().decode()


def test_no_rows_is_no_work():
    assert _append(N=0, qkv=None) == 0 and _attend(N=0, q=None) == 0
    lib = _lib.load()
    assert lib.sc_attention_shared_workspace_bytes(0, 3, 8, 2, 128, 256, 320, 1) == 0
    assert lib.sc_attention_shared_workspace_bytes(5, 3, 8, 3, 128, 256, 320, 1) == 0


def test_workspace_grows_with_rows_not_with_table_width():
    lib = _lib.load()
    small = lib.sc_attention_shared_workspace_bytes(64, 64, 32, 8, 128, 1 << 10, 1 << 13, 1)
    assert 0 < small <= lib.sc_attention_shared_workspace_bytes(128, 128, 32, 8, 128, 1 << 10, 1 << 13, 1)
    wide = lib.sc_attention_shared_workspace_bytes(64, 64, 32, 8, 128, 1 << 20, 1 << 13, 1)
    assert wide <= 2 * small + (16 << 20)


def test_wrappers_need_gpu_tensors():
    z = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        _lib.block_tables(z, z, z.view(4, 1), z, z, 64, 4)
    with pytest.raises(RuntimeError, match="GPU"):
        _lib.attention_shared(torch.zeros(1, 64, dtype=torch.bfloat16), 1, 1, 64, z, z, z, z, z, 1.0)
    assert ctypes.c_int64 in _lib.load().sc_attention_shared_bf16.argtypes


def test_cache_bookkeeping_on_the_host():
    from shardcompute_amd.block_cache import BlockKVCache
    c = BlockKVCache(2, 2, 64, num_blocks=5, max_sequences=3, max_length=40, block_size=16, max_prefix=20,
                     device=torch.device("cpu"))
    assert c.k.shape == (2, 5, 2, 16, 64) and c.vt.shape == (2, 5, 2, 64, 16) and c.tables.shape == (3, 3)
    assert c.prefix_table.shape == (2,) and c.max_positions == 60 and c.free_blocks.tolist() == [4, 3, 2, 1, 0]
    lengths, free = c._plan([17, 0, 16], None)
    assert lengths == [17, 0, 16] and free == 2
    c.host_lengths, c.host_free = lengths, free
    assert c._plan([15, 16, 16], None) == ([32, 16, 32], 0)
    assert c._plan([1, 40, 1], [True, False, True]) == ([1, 40, 1], 0)
    with pytest.raises(RuntimeError, match="full: the step needs 1 blocks more"):
        c.check_room([16, 16, 16])
    with pytest.raises(RuntimeError, match="sequence 0 would hold 49 positions"):
        c.check_room([32, 0, 0])
    with pytest.raises(ValueError, match="-1 new positions"):
        c.check_room([0, -1, 0])
    with pytest.raises(ValueError, match="block_size"):
        BlockKVCache(1, 1, 64, 4, 1, 64, block_size=48, device=torch.device("cpu"))
    with pytest.raises(ValueError, match="at least one"):
        BlockKVCache(1, 1, 64, 0, 1, 64, device=torch.device("cpu"))
    with pytest.raises(ValueError, match="at most 2048 sequences, got 2049"):
        BlockKVCache(1, 1, 64, 4, 2049, 64, device=torch.device("cpu"))


def test_more_key_blocks_than_32_bits_count_are_refused():
    """A workspace of 0 bytes is a refusal: 2048 sequences of 8 kv heads of 2^25 positions each."""
    from shardcompute_amd import _lib
    assert _lib.attention_shared_workspace_bytes(64, 2048, 32, 8, 128, 1 << 25, 0, 1) == 0
    assert _lib.attention_shared_workspace_bytes(64, 2048, 2048, 1, 128, 1 << 25, 0, 1) == 0       # 32 columns' 64s


@pytest.mark.parametrize("max_length,max_prefix,bs", [(2050, 0, 256), (2050, 300, 256), (17, 1, 16), (64, 128, 64)])
def test_rotary_tables_reach_every_position_a_table_has_room_for(max_length, max_prefix, bs, monkeypatch):
    """A sequence may grow to the room of its table, max_length rounded up to a block: the rotary
    tables that its layers ask for hold the last of these positions."""
    from types import SimpleNamespace

    from shardcompute_amd.block_cache import BlockBatch, BlockKVCache
    from shardcompute_amd.parallel import attention
    cpu = torch.device("cpu")
    c = BlockKVCache(1, 2, 64, num_blocks=40, max_sequences=1, max_length=max_length, block_size=bs,
                     max_prefix=max_prefix, device=cpu)
    room = c.tables.shape[1] * bs
    assert c._plan([room], None)[0] == [room]
    with pytest.raises(RuntimeError, match="room"):
        c._plan([room + 1], None)
    seen = []
    monkeypatch.setattr(attention._lib, "rope_append_blocks", lambda qkv, H, Hk, D, cos, *a, **kw: seen.append(cos.shape[0]))
    monkeypatch.setattr(attention._lib, "attention_shared", lambda *a, **kw: None)
    att = SimpleNamespace(local_num_heads=4, local_num_kv_heads=2, head_dim=64, scale=0.125,
                          rope=attention.RoPE(64, max_position_embeddings=1))
    step = c._buffers(1, 1, c.lengths)
    kv = BlockBatch(c, step, c.tables, 1, 1, False)[0]
    attention.ParallelAttention.attend_qkv(att, torch.zeros((1, 8 * 64), dtype=torch.bfloat16), 1, 1, kv)
    assert seen[0] >= max_prefix + room


@pytest.mark.parametrize("rows", [(1 << 30) - 1, 1 << 30, 1 << 40])
def test_more_rows_than_the_sums_count_are_refused(rows):
    """Sums of new positions saturate at 2^30 - 1: only row counts below that can tell a step that
    does not fit."""
    assert _tables(rows=rows) == -1 and "row count" in _lib.load().sc_last_error().decode()
