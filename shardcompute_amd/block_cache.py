"""A key/value cache in blocks for a ragged batch of sequences that share a prefix.

The dense :class:`~shardcompute_amd.kv_cache.KVCache` holds ``batch`` sequences of one
length.  Here every sequence has a length of its own, memory is taken by the block of
``block_size`` positions, and positions that all sequences share (a system prompt, a
document, the prompt of several samples) are held once:

* ``k``  ``[layers, blocks, kv_heads, block_size, head_dim]`` bf16
* ``vt`` ``[layers, blocks, kv_heads, head_dim, block_size]`` bf16 (values transposed)
* ``tables`` int32 ``[sequences, width]``: the blocks of each sequence's own positions, which
  follow the prefix; ``prefix_table`` the prefix's
* ``lengths`` int32 ``[sequences]``, ``prefix_len`` ``[1]``: positions held
* ``free_blocks`` / ``n_free``: a stack of the blocks nobody holds

With ``bits`` 4 or 8 keys and values are held as codes instead, in groups of 64 dims with a
bf16 scale and bias each (4.5 or 8.5 bits a value): ``pool`` uint8 ``[layers, blocks, kv_heads,
block_size / 16, bytes]`` in the place of ``k`` and ``vt``.  They are quantized as they are
appended, new ones included in what a step attends.

All of it is device memory and ``block_tables`` keeps it on the device, so a decode step
captured in a HIP graph replays as the sequences grow.  ``host_lengths`` and ``host_free``
are the host's mirror, from which a step that cannot fit is refused before its launch.

A model step is described by a :class:`BlockBatch` (``begin`` / ``begin_prefix``); indexed by
the layer it gives the :class:`BlockLayerKV` that ``ParallelAttention.attend_qkv`` takes.
"""
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib


def _cdiv(a: int, b: int) -> int:
    return -(-a // b)


class BlockLayerKV:
    """One layer's blocks and the step that reads and writes them."""

    def __init__(self, batch: "BlockBatch", layer: int):
        self.batch = batch
        self.bits = batch.cache.bits
        if self.bits is None:
            self.k = batch.cache.k[layer]
            self.vt = batch.cache.vt[layer]
        else:
            self.pool = batch.cache.pool[layer]


class BlockBatch:
    """The rows of one model step: ``step`` (slots, positions, row starts, lengths), whose rows
    belong to the sequences of ``tables`` behind ``prefix_table`` (None: no prefix)."""

    def __init__(self, cache: "BlockKVCache", step, tables, rows: int, max_new: int, prefix: bool):
        self.cache = cache
        self.step = step
        self.tables = tables
        self.rows = rows
        self.max_new = max_new
        self.number = cache.steps
        self.prefix_table = cache.prefix_table if prefix else None
        self.prefix_len = cache.prefix_len if prefix else None

    def __getitem__(self, layer: int) -> BlockLayerKV:
        return BlockLayerKV(self, layer)

    def check_current(self):
        """Raise if the cache has begun another step since (its lengths are that step's)."""
        if self.number != self.cache.steps:
            raise RuntimeError("the block cache has begun another step since this one")

    @property
    def last_rows(self) -> torch.Tensor:
        """The last row of each sequence (of one without rows: some row)."""
        return (self.step.row_starts[1:] - 1).clamp_(min=0).long()

    def workspace_bytes(self, H: int, Hkv: int, D: int) -> int:
        bs = self.cache.block_size
        pre = 0 if self.prefix_table is None else self.prefix_table.numel() * bs
        sizes = (self.rows, self.tables.shape[0], H, Hkv, D, self.tables.shape[1] * bs, pre, self.max_new)
        if self.cache.bits is not None:
            return _lib.attention_quantized_workspace_bytes(*sizes, bits=self.cache.bits)
        return _lib.attention_shared_workspace_bytes(*sizes)


class BlockKVCache:
    def __init__(self, num_layers: int, num_kv_heads: int, head_dim: int, num_blocks: int, max_sequences: int,
                 max_length: int, block_size: int = 64, max_prefix: int = 0, device: Optional[torch.device] = None,
                 bits: Optional[int] = None):
        if block_size not in _lib.BLOCK_SIZES:
            raise ValueError(f"block_size must be one of {_lib.BLOCK_SIZES}, got {block_size}")
        if min(num_layers, num_kv_heads, head_dim, num_blocks, max_sequences, max_length) < 1 or max_prefix < 0:
            raise ValueError("a block cache needs at least one layer, head, block, sequence and position")
        if max_sequences > _lib.SHARED_MAX_SEQUENCES:
            raise ValueError(f"at most {_lib.SHARED_MAX_SEQUENCES} sequences, got {max_sequences}")
        if bits is not None and bits not in _lib.CACHE_BITS:
            raise ValueError(f"a block cache holds bf16 (bits None) or {_lib.CACHE_BITS} bits, got {bits}")
        if device is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.num_layers, self.num_kv_heads, self.head_dim, self.bits = num_layers, num_kv_heads, head_dim, bits
        self.num_blocks, self.max_sequences, self.block_size = num_blocks, max_sequences, block_size
        self.max_length, self.max_prefix, self.device = max_length, max_prefix, device
        bf = torch.bfloat16
        if bits is None:
            self.k = torch.zeros((num_layers, num_blocks, num_kv_heads, block_size, head_dim), dtype=bf, device=device)
            self.vt = torch.zeros((num_layers, num_blocks, num_kv_heads, head_dim, block_size), dtype=bf, device=device)
        else:
            shape = _lib.quantized_pool_shape(num_blocks, num_kv_heads, block_size, head_dim, bits)
            self.pool = torch.zeros((num_layers, *shape), dtype=torch.uint8, device=device)

        def i32(*shape):
            return torch.zeros(shape, dtype=torch.int32, device=device)
        self.tables = i32(max_sequences, _cdiv(max_length, block_size))
        self.lengths = i32(max_sequences)
        self.prefix_table = i32(_cdiv(max_prefix, block_size)) if max_prefix else None
        self.prefix_len = i32(1)
        # popped from the end: block 0 first
        self.free_blocks = torch.arange(num_blocks - 1, -1, -1, dtype=torch.int32, device=device)
        self.n_free = torch.full((1,), num_blocks, dtype=torch.int32, device=device)
        self.status = i32(1)
        self.host_lengths: List[int] = [0] * max_sequences
        self.host_prefix = 0
        self.host_free = num_blocks
        self.steps = 0              # begun

    @property
    def max_positions(self) -> int:
        """Positions asked for: the longest prefix and the longest sequence behind it."""
        return self.max_prefix + self.max_length

    @property
    def rotary_positions(self) -> int:
        """Positions the tables have room for, whole blocks: what the rotary tables must hold."""
        blocks = self.tables.shape[1] + (0 if self.prefix_table is None else self.prefix_table.numel())
        return blocks * self.block_size

    @property
    def nbytes(self) -> int:
        return self.pool.numel() if self.bits is not None else 2 * self.k.numel() * self.k.element_size()

    def _plan(self, new: Sequence[int], release: Optional[Sequence[bool]]):
        """(lengths, free blocks) after a step, or an error if it does not fit."""
        if len(new) != self.max_sequences or (release is not None and len(release) != self.max_sequences):
            raise ValueError(f"a step names every one of the {self.max_sequences} sequences")
        bs, free, lengths = self.block_size, self.host_free, []
        for r, w in enumerate(new):
            if w < 0:
                raise ValueError(f"sequence {r}: {w} new positions")
            old = self.host_lengths[r]
            if release is not None and release[r]:
                free += _cdiv(old, bs)
                old = 0
            if old + w > self.tables.shape[1] * bs:
                raise RuntimeError(f"block cache: sequence {r} would hold {old + w} positions, its table has room for "
                                   f"{self.tables.shape[1] * bs}")
            free -= _cdiv(old + w, bs) - _cdiv(old, bs)
            lengths.append(old + w)
        if free < 0:
            raise RuntimeError(f"block cache full: the step needs {-free} blocks more than the {self.num_blocks} hold")
        return lengths, free

    def check_room(self, new: Sequence[int], release: Optional[Sequence[bool]] = None):
        self._plan(new, release)

    def _buffers(self, rows: int, R: int, lengths):
        i32 = dict(dtype=torch.int32, device=self.device)
        return _lib.BlockStep(lengths, self.n_free, torch.empty(R + 1, **i32), torch.empty(rows, **i32),
                              torch.empty(rows, **i32), self.status)

    def begin(self, new: Sequence[int], release: Optional[Sequence[bool]] = None) -> BlockBatch:
        """A model step in which sequence r gets ``new[r]`` positions; ``release[r]`` gives its
        blocks back first.  The step's rows are the sequences' new positions in order."""
        lengths, free = self._plan(new, release)
        rows = sum(new)
        step = self._buffers(rows, self.max_sequences, self.lengths)
        rel = None if release is None else torch.tensor([bool(x) for x in release], device=self.device)
        _lib.block_tables(self.lengths, torch.tensor(list(new), dtype=torch.int32, device=self.device), self.tables,
                          self.free_blocks, self.n_free, self.block_size, rows, prefix_len=self.prefix_len,
                          release=rel, out=step)
        self.host_lengths, self.host_free = lengths, free
        self.steps += 1
        return BlockBatch(self, step, self.tables, rows, max(new), self.host_prefix > 0)

    def begin_prefix(self, positions: int) -> BlockBatch:
        """A model step that appends ``positions`` to the shared prefix, before any sequence
        holds a position (theirs follow the prefix's)."""
        if any(self.host_lengths):
            raise RuntimeError("the shared prefix is filled before the sequences")
        have = self.host_prefix
        if positions < 1 or have + positions > self.max_prefix:
            raise RuntimeError(f"a prefix of {have} + {positions} positions exceeds the cache's {self.max_prefix}")
        need = _cdiv(have + positions, self.block_size) - _cdiv(have, self.block_size)
        if need > self.host_free:
            raise RuntimeError(f"block cache full: the prefix needs {need} blocks, {self.host_free} are free")
        tables = self.prefix_table.view(1, -1)
        step = self._buffers(positions, 1, self.prefix_len)
        _lib.block_tables(self.prefix_len, torch.full((1,), positions, dtype=torch.int32, device=self.device), tables,
                          self.free_blocks, self.n_free, self.block_size, positions, out=step)
        self.host_prefix += positions
        self.host_free -= need
        self.steps += 1
        return BlockBatch(self, step, tables, positions, positions, False)

    def as_tuple(self, layer: int, sequence: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """``(k, v)`` of one sequence in the reference layout ``[1, kv_heads, length, head_dim]``
        bf16, the shared prefix's positions first."""
        if not 0 <= sequence < self.max_sequences:
            raise IndexError(f"sequence {sequence} of {self.max_sequences}")
        bs = self.block_size

        def slots_of(table, n):
            p = torch.arange(n, dtype=torch.int32, device=self.device)
            return table[(p // bs).long()] * bs + p % bs
        slots = slots_of(self.tables[sequence], self.host_lengths[sequence])
        if self.host_prefix:
            slots = torch.cat([slots_of(self.prefix_table, self.host_prefix), slots])
        if self.bits is not None:
            k, v = _lib.read_quantized(self.pool[layer], self.num_kv_heads, self.head_dim, slots, bits=self.bits)
        else:
            b, off = (slots // bs).long(), (slots % bs).long()
            k, v = self.k[layer][b, :, off], self.vt[layer][b, :, :, off]
        return k.transpose(0, 1)[None].contiguous(), v.transpose(0, 1)[None].contiguous()

    def check_status(self):
        """Raise if a step was refused on the device (one captured in a graph and replayed
        past the cache's room); synchronises."""
        bits = int(self.status.item())
        if bits:
            why = [name for bit, name in ((1, "no free blocks"), (2, "a table is full"), (4, "too few rows"),
                                          (8, "the stack is full")) if bits & bit]
            raise RuntimeError("block cache: a step was refused (" + ", ".join(why) + ")")
