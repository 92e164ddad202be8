"""Where the merge of the shared attention looks for a row's parts, on the host: the header's
own code, compiled for the CPU."""
import ctypes
import random
import shutil
import subprocess

import pytest

from shardcompute_amd import build

SOURCE = r"""
#include "attn_shared_parts.h"
extern "C" void parts_of(const int *a, int *out) {
    const sc::OwnParts p = sc::own_parts_of(a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[8], a[9], a[10], a[11],
                                            a[12], a[13]);
    out[0] = p.first; out[1] = p.n; out[2] = p.step; out[3] = p.col;
}
extern "C" int tile_part_row(int row, int r, int i, int per_seq, int part_rows) {
    return sc::tile_part_row(row, r, i, per_seq, part_rows);
}
"""


@pytest.fixture(scope="module")
def library(tmp_path_factory):
    if not (shutil.which("hipcc") or shutil.os.path.exists("/opt/rocm/bin/hipcc")):
        pytest.skip("no hipcc")
    d = tmp_path_factory.mktemp("parts")
    src, lib = d / "parts.hip", d / "parts.so"
    src.write_text(SOURCE)
    subprocess.run([build.hipcc(), "--cuda-host-only", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", build.CSRC, str(src),
                    "-o", str(lib)], check=True, capture_output=True)
    return ctypes.CDLL(str(lib))


@pytest.fixture(scope="module")
def parts_of(library):
    fn = library.parts_of
    I14, I4 = ctypes.c_int * 14, ctypes.c_int * 4

    def call(*a):
        out = I4()
        fn(I14(*a), out)
        return tuple(out)
    return call


def cdiv(a, b):
    return -(-a // b)


def schedule(seqs, G, Hkv, small):
    """(first block, first unit) of every sequence (rows, keys), and the blocks of them all."""
    offs, t, u = [], 0, 0
    for n, ln in seqs:
        offs.append((t, u))
        if n <= small and n > 0 and ln > 0:
            units = Hkv * cdiv(n * G, 64)
            t, u = t + units * cdiv(ln, 64), u + units
    return offs, t, u


def inside(p, own_parts, part_cols):
    first, n, step, col = p
    return n == 0 or (n > 0 and 0 <= first and first + step * (n - 1) < own_parts and 0 <= col < part_cols)


@pytest.mark.parametrize("G,Hkv,max_rows,own_wgs", [(4, 8, 16, 512), (8, 1, 8, 256), (1, 3, 70, 7), (40, 1, 1, 64),
                                                    (96, 2, 1, 300), (5, 2, 30, 1)])
def test_parts_are_those_of_the_workgroups_that_have_the_unit(parts_of, G, Hkv, max_rows, own_wgs):
    """Every row of every sequence against a walk over the blocks: workgroup t // run has block
    t, its waves' parts of unit u are 4 (u + workgroup) + wave."""
    rng = random.Random(G)
    small = max(64 // G, 1)
    for _ in range(4):
        seqs = [(rng.randint(0, max_rows), rng.choice([0, 1, 63, 64, 65, rng.randint(1, 900)])) for _ in range(9)]
        offs, total, units = schedule(seqs, G, Hkv, small)
        own_parts, cols = 4 * (units + own_wgs), min(16, small * G)
        run, first = max(cdiv(total, own_wgs), 1), 0
        for (n, ln), (off, unit) in zip(seqs, offs):
            for row in range(first, first + n):
                for hk in range(Hkv):
                    for gq in (0, G - 1):
                        got = parts_of(row, first, n, ln, hk, gq, G, small, off, unit, total, own_wgs, own_parts, cols)
                        assert inside(got, own_parts, cols)
                        want = []
                        if n <= small and ln:
                            col, kt = (row - first) * G + gq, cdiv(ln, 64)
                            u = hk * cdiv(n * G, 64) + col // 64
                            wgs = sorted({t // run for t in range(off + u * kt, off + (u + 1) * kt)})
                            waves = [col // 16 % 4] if n * G > 16 else range(4)
                            want = [4 * (unit + u + g) + w for g in wgs for w in waves]
                            assert got[3] == col % 16
                        assert [got[0] + got[2] * i for i in range(got[1])] == want
            first += n


def test_rows_of_no_sequence_have_no_parts(parts_of):
    """A row before the first sequence's rows or past its sequence's (row starts that begin above
    0 or do not ascend) lies in no unit: nothing is looked up for it, least of all before the
    parts.  300 rows of 32 heads on 8, row starts 299, 300, 300."""
    own_parts = 4 * (8 * 2 + 512)
    for row in (0, 1, 150, 298, 300, 301, 100000):
        for hk in range(8):
            for gq in range(4):
                p = parts_of(row, 299, 1, 8192, hk, gq, 4, 16, 0, 0, 8 * 128, 512, own_parts, 16)
                assert p[1] == 0, (row, p)
    rng = random.Random(1)
    for _ in range(20000):
        G = rng.choice([1, 3, 4, 8, 40, 128])
        small = max(64 // G, 1)
        first, n, ln = rng.randint(0, 5000), rng.randint(0, 2 * small), rng.choice([0, 1, 700, 1 << 20, (1 << 30) - 1])
        row, total, wgs = rng.randint(0, 6000), rng.randint(0, (1 << 31) - 1), rng.randint(1, 512)
        parts = 4 * (rng.randint(0, 4000) + wgs)
        here = 8 * cdiv(n * G, 64) * cdiv(ln, 64)               # the sequence's blocks, among `total`
        if here > total:
            continue
        a = (row, first, n, ln, rng.randint(0, 7), rng.randint(0, G - 1), G, small, rng.randint(0, total - here),
             rng.randint(0, 4000), total, wgs, parts, 16)
        p = parts_of(*a)
        assert inside(p, parts, 16), (a, p)
        assert p[1] == 0 or first <= row < first + n


def test_rows_of_no_sequence_take_no_sequences_part(library):
    """attn_tile's parts by sequence, 3 of 16 rows each: every row of a sequence has a slot of its
    own, a row of no sequence none of them."""
    f = library.tile_part_row
    owned = [f(100 + 20 * r + i, r, i, 16, 48) for r in range(3) for i in range(16)]
    assert sorted(owned) == list(range(48))
    assert all(f(row, -1, 0, 16, 48) >= 48 for row in range(200))
    # a sequence of more rows keeps out of the next one's
    assert all(f(row, 0, row, 16, 48) >= 48 for row in range(16, 60))
    # by row: every row its own
    assert [f(row, r, 1, 0, 200) for row in range(200) for r in (-1, 2)] == [row for row in range(200) for _ in (0, 1)]
