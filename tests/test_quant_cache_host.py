"""Refusals of the quantized cache's entry points (argument checks only, no GPU calls)."""
import os

import pytest
import torch

from shardcompute_amd import _lib
from shardcompute_amd.build import LIB_PATH

pytestmark = pytest.mark.skipif(not os.path.exists(LIB_PATH), reason="library not built")
A = 1 << 12                     # a 16-byte aligned address nothing reads


def _append(**kw):
    a = dict(qkv=A, qkv_stride=1536, q=A, q_stride=1024, N=3, H=8, Hkv=2, D=128, cos=A, sin=A, length=99, pool=A,
             n_blocks=10, bs=64, bits=4, slots=A, positions=A)
    a.update(kw)
    return _lib.load().sc_rope_append_quantized_bf16(*a.values(), None)


def _read(**kw):
    a = dict(pool=A, n_blocks=10, bs=64, bits=4, Hkv=2, D=128, slots=A, n=5, k=A, v=A)
    a.update(kw)
    return _lib.load().sc_read_quantized_bf16(*a.values(), None)


def _attend(**kw):
    a = dict(q=A, q_stride=1024, pool=A, n_blocks=10, bs=64, bits=8, row_starts=A, lengths=A, tables=A, width=4,
             prefix_table=A, prefix_width=5, prefix_len=A, out=A, out_stride=1024, N=3, R=3, H=8, Hkv=2, D=128, scale=0.1,
             max_new=1, workspace=A, workspace_bytes=1 << 30)
    a.update(kw)
    return _lib.load().sc_attention_quantized_bf16(*a.values(), None)


@pytest.mark.parametrize("call,kw,message", [
    (_append, dict(qkv=None), "null pointer"), (_append, dict(pool=None), "null pointer"),
    (_append, dict(slots=None), "null pointer"), (_append, dict(D=96), "head_dim 96"), (_append, dict(bits=3), "3 bits"),
    (_append, dict(bits=16), "16 bits"), (_append, dict(bs=20), "block size 20"), (_append, dict(bs=8), "block size 8"),
    (_append, dict(Hkv=3), "bad shape"), (_append, dict(N=-1), "bad shape"), (_append, dict(n_blocks=0), "pool"),
    (_append, dict(n_blocks=1 << 25), "pool"), (_append, dict(length=0), "table size"),
    (_append, dict(qkv_stride=1528), "strides"), (_append, dict(qkv_stride=1540), "strides"),
    (_append, dict(q_stride=1020), "strides"), (_append, dict(pool=A + 8), "aligned"), (_append, dict(cos=A + 4), "aligned"),
    (_append, dict(N=1 << 29), "too many rows"),
    (_read, dict(pool=None), "null pointer"), (_read, dict(k=None), "null pointer"), (_read, dict(D=32), "head_dim 32"),
    (_read, dict(bits=2), "2 bits"), (_read, dict(bs=512), "block size 512"), (_read, dict(n=-1), "bad shape"),
    (_read, dict(Hkv=0), "bad shape"), (_read, dict(n_blocks=0), "pool"), (_read, dict(v=A + 2), "aligned"),
    (_read, dict(n=1 << 29), "too many rows"),
    (_attend, dict(q=None), "null pointer"), (_attend, dict(pool=None), "null pointer"),
    (_attend, dict(prefix_table=None), "null pointer"), (_attend, dict(prefix_len=None), "null pointer"),
    (_attend, dict(D=80), "head_dim 80"), (_attend, dict(bits=5), "5 bits"), (_attend, dict(bs=0), "block size 0"),
    (_attend, dict(H=9), "bad shape"), (_attend, dict(R=0), "bad shape"), (_attend, dict(R=2049), "bad shape"),
    (_attend, dict(width=0), "bad shape"), (_attend, dict(max_new=-1), "bad shape"),
    (_attend, dict(prefix_width=1 << 26), "bad shape"), (_attend, dict(n_blocks=0), "pool"),
    (_attend, dict(scale=0.0), "scale"), (_attend, dict(scale=-0.1), "scale"),
    (_attend, dict(scale=float("nan")), "scale"), (_attend, dict(scale=float("inf")), "scale"),
    (_attend, dict(q_stride=1023), "strides"), (_attend, dict(q_stride=1028), "strides"),
    (_attend, dict(out_stride=1000), "strides"), (_attend, dict(q=A + 8), "misaligned"),
    (_attend, dict(out=A + 4), "misaligned"), (_attend, dict(pool=A + 4), "misaligned"),
])
def test_refused(call, kw, message):
    assert call(**kw) in (-1, -2)
    assert message in _lib.load().sc_last_error().decode()


def test_no_rows_is_no_work():
    assert _append(N=0, qkv=None) == 0 and _attend(N=0, q=None) == 0 and _read(n=0, k=None) == 0
    lib = _lib.load()
    assert lib.sc_attention_quantized_workspace_bytes(0, 3, 8, 2, 128, 256, 320, 1, 4) == 0
    assert lib.sc_attention_quantized_workspace_bytes(5, 3, 8, 3, 128, 256, 320, 1, 4) == 0


@pytest.mark.parametrize("D,bits", [(64, 4), (64, 8), (128, 4), (128, 8)])
def test_a_cell_holds_the_codes_a_scale_and_a_bias_per_64_values(D, bits):
    assert _lib.load().sc_kv_cell_bytes(D, bits) == 16 * (2 * D * bits // 8 + 2 * (D // 64) * 4)
    assert _lib.quantized_pool_shape(5, 3, 32, D, bits) == (5, 3, 2, 16 * (2 * D * bits // 8 + 2 * (D // 64) * 4))


def test_pools_refused():
    with pytest.raises(ValueError, match="bits"):
        _lib.quantized_pool_shape(5, 3, 32, 64, bits=6)
    with pytest.raises(ValueError, match="head_dim"):
        _lib.quantized_pool_shape(5, 3, 32, 96)
    with pytest.raises(ValueError, match="block_size"):
        _lib.quantized_pool_shape(5, 3, 48, 64)
    good = torch.zeros(_lib.quantized_pool_shape(5, 3, 32, 64, 4), dtype=torch.uint8)
    for pool, error, message in [(good.to(torch.int32), TypeError, "uint8"), (good[:, :2], ValueError, "must be"),
                                 (good[..., :64], ValueError, "must be"), (good.transpose(0, 1).contiguous(), ValueError, "must be"),
                                 (good[:, :, :1], ValueError, "contiguous"), (good, RuntimeError, "GPU")]:
        with pytest.raises(error, match=message):
            _lib._quantized(pool, 3, 64, 4, 0)
    with pytest.raises(ValueError, match="8 bits must be"):
        _lib._quantized(good, 3, 64, 8, 0)


def test_wrappers_need_gpu_tensors():
    z = torch.zeros(4, dtype=torch.int32)
    pool = torch.zeros(_lib.quantized_pool_shape(1, 1, 16, 64), dtype=torch.uint8)
    x = torch.zeros((4, 192), dtype=torch.bfloat16)
    for call in (lambda: _lib.rope_append_quantized(x, 1, 1, 64, z, z, pool, z, z),
                 lambda: _lib.read_quantized(pool, 1, 64, z),
                 lambda: _lib.attention_quantized(x, 1, 1, 64, pool, z, z, z, 1.0)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_cache_of_codes_on_the_host():
    from shardcompute_amd.block_cache import BlockKVCache
    cpu = torch.device("cpu")
    for bits in (4, 8):
        c = BlockKVCache(2, 3, 64, num_blocks=5, max_sequences=3, max_length=40, block_size=32, max_prefix=20, device=cpu,
                         bits=bits)
        assert c.pool.shape == (2, *_lib.quantized_pool_shape(5, 3, 32, 64, bits)) and c.pool.dtype is torch.uint8
        assert c.nbytes == 2 * 5 * 3 * 2 * 16 * (2 * 64 * bits // 8 + 8) and not c.pool.any()
        assert c._plan([17, 0, 16], None) == ([17, 0, 16], 3)
    with pytest.raises(ValueError, match="bits"):
        BlockKVCache(1, 1, 64, 4, 1, 64, device=cpu, bits=3)
    with pytest.raises(ValueError, match="head_dim"):
        BlockKVCache(1, 1, 80, 4, 1, 64, device=cpu, bits=4)


PARTS_SOURCE = r"""
#include "attn_shared_parts.h"
extern "C" void parts_of(const int *a, int *out) {
    const sc::OwnParts p = sc::own_parts_of(a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[8], a[9], a[10], a[11],
                                            a[12], a[13], a[14], a[15], a[16]);
    out[0] = p.first; out[1] = p.n; out[2] = p.step; out[3] = p.col;
}
"""


@pytest.fixture(scope="module")
def parts_of(tmp_path_factory):
    import ctypes
    import os
    import shutil
    import subprocess

    from shardcompute_amd import build

    if not (shutil.which("hipcc") or os.path.exists("/opt/rocm/bin/hipcc")):
        pytest.skip("no hipcc")
    d = tmp_path_factory.mktemp("parts")
    src, lib = d / "parts.hip", d / "parts.so"
    src.write_text(PARTS_SOURCE)
    subprocess.run([build.hipcc(), "--cuda-host-only", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", build.CSRC, str(src),
                    "-o", str(lib)], check=True, capture_output=True)
    fn = ctypes.CDLL(str(lib)).parts_of
    I17, I4 = ctypes.c_int * 17, ctypes.c_int * 4

    def call(*a):
        out = I4()
        fn(I17(*a), out)
        return tuple(out)
    return call


@pytest.mark.parametrize("rest", [0, 1, 2])
@pytest.mark.parametrize("seed", range(6))
def test_parts_of_units_with_rests(parts_of, rest, seed):
    """The parts that the merge reads are those of the runs that hold blocks of the row's unit:
    units' blocks and the empty places after them laid in a line, cut into equal runs."""
    import random

    rng = random.Random(seed)
    shift, small, hkv = 7, 16, rng.choice([1, 2, 8])
    G = rng.choice([1, 4, 8])
    R, wgs = rng.randint(1, 12), rng.choice([1, 3, 17, 64, 512])
    ns = [rng.choice([0, 1, 1, 1, 3, 16, 40]) for _ in range(R)]
    lens = [n + rng.choice([0, 0, 1, 100, 127, 128, 129, 3000]) for n in ns]
    line, off, unit, units, where = [], [], [], 0, {}
    for r, (n, ln) in enumerate(zip(ns, lens)):
        off.append(len(line))
        unit.append(units)
        kt = -(-ln // 128)
        if n == 0 or n > small or kt == 0:
            continue
        ct = -(-n * G // 64)
        for u in range(hkv * ct):
            where[(r, u)] = units
            line += [units] * kt + [None] * rest
            units += 1
    total = len(line)
    run = -(-total // wgs) if total else 1
    first = 0
    for r, (n, ln) in enumerate(zip(ns, lens)):
        for i in range(n):
            for hk in range(hkv):
                for g in range(G):
                    p_first, p_n, step, col = parts_of(first + i, first, n, ln, hk, g, G, small, off[r], unit[r], total, wgs,
                                                       1 << 28, 16, shift, 0, rest)
                    if n > small:
                        assert p_n == 0
                        continue
                    c = i * G + g
                    number = where[(r, hk * -(-n * G // 64) + c // 64)]
                    holders = sorted({t // run for t, x in enumerate(line) if x == number})
                    waves = [c // 16 % 4] if n * G > 16 else [0, 1, 2, 3]
                    want = [4 * (number + w) + v for w in holders for v in waves]
                    assert [p_first + step * j for j in range(p_n)] == want and col == c % 16
        first += n


def _up(v):
    return -(-v // 256) * 256


@pytest.mark.parametrize("rows,R,H,Hkv,D,own,prefix", [
    (24, 1, 32, 8, 128, 64, 0), (24, 1, 32, 8, 128, 4096, 0), (64, 1, 32, 8, 128, 131072, 0), (100, 3, 32, 4, 64, 700, 5000),
    (2049, 1, 32, 8, 128, 2112, 0), (2049, 1, 32, 8, 128, 131072, 0), (2079, 32, 32, 8, 128, 2112, 0), (9000, 16, 8, 1, 128, 1024, 4096),
])
def test_workspace_of_prompts_is_that_of_their_cut(rows, R, H, Hkv, D, own, prefix):
    """Column tiles of 256 (row, head) columns on 256 CUs, their keys cut into as many workgroups as
    make the walk (2 us a block of 64 keys, rounds of 256 workgroups) and the parts (2.5 TB/s and
    0.06 us each; none if uncut) least."""
    cus, G = 256, H // Hkv
    wgs, blocks = -(-rows * G // 256) * Hkv, -(-(own + prefix) // 64)

    def us(n):
        return blocks / n * 2.0 * -(-wgs * n // cus) + (n > 1) * n * (rows * H * (8 * D + 16) / 2.5e6 + 0.06)
    cut = min(range(1, min(64, blocks) + 1), key=us)
    small = max(64 // G, 1)                  # rows of a sequence whose own keys are the line's
    few = R * small < rows and cut == 1
    tile = cut * (R * small if few else rows) * H
    coltiles = min(R * -(-small * G // 64), R + rows * G // 64)
    keyblocks = coltiles * (-(-own // 128) + (R > 1))
    line = 4 * (Hkv * coltiles + max(min(2 * cus, Hkv * keyblocks), 1)) * min(small * G, 16)
    want = sum(_up(n * b) for n in (tile, line) for b in (4 * D, 8)) + _up((R + 1) * 8 + 8)
    assert _lib.attention_quantized_workspace_bytes(rows, R, H, Hkv, D, own, prefix, rows, bits=4) == want
