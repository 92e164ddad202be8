"""The key/value cache in blocks on the GPU: tables of a step, rotation and append, attention
over a shared prefix and each sequence's own positions, against Python and float64."""
import random

import pytest
import torch

from shardcompute_amd import _lib
from tests.block_util import Cache, PlainTables, assert_attention, cdiv

pytestmark = pytest.mark.gpu


def i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------- tables


def _pool(rng, lengths, width, bs, spare):
    counts = [cdiv(n, bs) for n in lengths]
    order = list(range(sum(counts) + spare))
    rng.shuffle(order)
    tables, at = [], 0
    for c in counts:
        tables.append(order[at:at + c] + [-1] * (width - c))
        at += c
    return tables, order[at:] + [-1] * at, spare


# sequences, positions held at most, new ones at most, width, block size, rows beyond the step's,
# sequences given back (one in n), steps; up to one workgroup's sequences and rows and beyond
STEPS = [(1, 0, 1, 4, 16, 0, 0, 40), (1, 63, 1, 3, 64, 2, 0, 70), (3, 40, 9, 40, 16, 5, 2, 12),
         (64, 300, 1, 16, 32, 0, 7, 40), (255, 900, 3, 8, 256, 1, 5, 6), (300, 100, 40, 40, 16, 3, 0, 3),
         (1024, 50, 2, 12, 16, 0, 9, 3), (1025, 50, 2, 12, 16, 0, 9, 3), (2500, 33, 1, 5, 64, 4, 3, 3),
         (2500, 70, 5, 20, 16, 4, 3, 2), (40, 10, 700, 20, 128, 9, 0, 2), (1, 0, 5000, 40, 128, 0, 0, 1)]


@pytest.mark.parametrize("R,held,new,width,bs,pad,freed,steps", STEPS)
def test_tables(device, R, held, new, width, bs, pad, freed, steps):
    print(f"tables R={R} held={held} new={new} width={width} bs={bs}", flush=True)
    rng = random.Random(R * 1000 + new)
    lengths = [rng.randint(0, held) for _ in range(R)]
    tables, free, spare = _pool(rng, lengths, width, bs, R * width)
    plain = PlainTables(lengths, tables, free, spare, len(free), bs)
    ln, tb, fr, nf = i32(lengths), i32(tables), i32(free), i32([spare])
    prefix = i32([11])
    out = None
    for step in range(steps):
        w = [rng.randint(0, new) for _ in range(R)]
        w[0] = new                                              # one sequence always at the most
        if step == 1:
            w[-1] = -3 if R > 1 else w[-1]                      # counts as none
        gone = [bool(freed) and rng.randrange(freed) == 0 for _ in range(R)] if freed else None
        rows = sum(max(x, 0) for x in w) + pad
        rel = None if gone is None else torch.tensor(gone, device="cuda")
        # the lengths and the stack's height in place every other step
        if step % 2 and out is not None:
            out = _lib.BlockStep(ln, nf, i32([0] * (R + 1)), i32([5] * rows), i32([5] * rows), out.status)
        else:
            out = None
        out = _lib.block_tables(ln, i32(w), tb, fr, nf, bs, rows, prefix_len=prefix, release=rel, out=out)
        starts, slots, positions = plain.step(w, rows, 11, gone)
        assert out.status.item() == plain.status == 0
        assert out.row_starts.tolist() == starts and out.lengths.tolist() == plain.lengths
        assert out.slots.tolist() == slots and out.positions.tolist() == positions
        assert out.n_free.item() == plain.n_free and tb.tolist() == plain.tables
        assert fr.tolist() == plain.free
        ln, nf = out.lengths, out.n_free


@pytest.mark.parametrize("what", ["blocks", "table", "rows", "stack"])
@pytest.mark.parametrize("R", [5, 1500])
def test_tables_refused_step_changes_nothing(device, what, R):
    print(f"refused step: {what} R={R}", flush=True)
    rng, bs, width = random.Random(3), 16, 4
    lengths = [rng.randint(1, 40) for _ in range(R)]
    tables, free, spare = _pool(rng, lengths, width, bs, R * width)
    n_free = {"blocks": 1, "stack": len(free)}.get(what, spare)
    new, rows, release = [1] * R, R, None
    if what == "table":
        new[R // 2] = width * bs - lengths[R // 2] + 1
        rows += width * bs
    if what == "blocks":
        new, rows = [20] * R, 20 * R
    if what == "rows":
        rows = R - 1
    if what == "stack":
        release = [False] * R
        release[1] = True
    plain = PlainTables(lengths, tables, free, n_free, len(free), bs)
    starts, slots, positions = plain.step(new, rows, 0, release)
    ln, tb, fr, nf = i32(lengths), i32(tables), i32(free), i32([n_free])
    out = _lib.block_tables(ln, i32(new), tb, fr, nf, bs, rows,
                            release=None if release is None else torch.tensor(release, device="cuda"))
    bit = {"blocks": 1, "table": 2, "rows": 4, "stack": 8}[what]
    assert out.status.item() == plain.status == bit
    assert tb.tolist() == tables and fr.tolist() == free and out.lengths.tolist() == lengths
    assert out.n_free.item() == n_free and out.row_starts.tolist() == starts == [0] * (R + 1)
    assert out.slots.tolist() == slots and out.positions.tolist() == positions
    # a later step that fits runs, and the word keeps the reason
    ok = _lib.block_tables(out.lengths, i32([0] * R), tb, fr, out.n_free, bs, 0, out=out)
    assert ok.status.item() == bit and ok.lengths.tolist() == lengths


@pytest.mark.parametrize("R", [1, 3, 1500])
def test_tables_refused_step_names_every_reason(device, R):
    """One sequence with more positions than rows and more blocks than the stack holds."""
    bs, width, rows = 16, 80, 10
    tables, free = [[-1] * width for _ in range(R)], list(range(40))
    new = [1000] + [0] * (R - 1)
    plain = PlainTables([0] * R, tables, free, 2, len(free), bs)
    plain.step(new, rows)
    out = _lib.block_tables(i32([0] * R), i32(new), i32(tables), i32(free), i32([2]), bs, rows)
    assert out.status.item() == plain.status == _lib.BLOCKS_NO_ROWS | _lib.BLOCKS_NO_BLOCKS
    assert out.slots.tolist() == [-1] * rows and out.row_starts.tolist() == [0] * (R + 1)
    assert out.lengths.tolist() == [0] * R and out.n_free.item() == 2


# ---------------------------------------------------------------- rotation and append

# rows of each sequence, positions before them, block size, heads; single rows, runs at the edges
# of the 64-row groups and of the 8-slot pieces, rows without a slot between them
APPENDS = [([1], [0], 16, 4, 2, 64), ([1] * 70, list(range(70)), 64, 32, 8, 128), ([64], [0], 64, 8, 1, 128),
           ([65, 3, 200], [7, 8, 61], 16, 32, 4, 64), ([129, 130], [0, 127], 128, 6, 2, 128),
           ([7, 8, 9, 15, 16, 17], [1, 8, 0, 3, 16, 5], 32, 2, 2, 64), ([500], [3], 256, 24, 1, 128),
           ([1200, 1], [0, 40], 64, 32, 8, 128)]


@pytest.mark.parametrize("new,held,bs,H,Hkv,D", APPENDS)
@pytest.mark.parametrize("in_place", [False, True])
def test_append(device, new, held, bs, H, Hkv, D, in_place):
    print(f"append {new[:3]} held {held[:3]} bs={bs} H={H} Hkv={Hkv} D={D}", flush=True)
    g = torch.Generator(device="cuda")
    g.manual_seed(bs + D)
    n = sum(new)
    N, W = n + 3, (H + 2 * Hkv) * D
    buf = torch.randn((N, W + 8), generator=g, device="cuda").to(torch.bfloat16)
    qkv = buf[:, :W]                                             # a row stride wider than the rows
    counts = [cdiv(h + w, bs) for h, w in zip(held, new)]
    order = torch.randperm(sum(counts) + 1, generator=g, device="cuda").tolist()
    slots, positions, at = [], [], 0
    for h, w, c in zip(held, new, counts):
        slots += [order[at + p // bs] * bs + p % bs for p in range(h, h + w)]
        positions += [p + 5 for p in range(h, h + w)]
        at += c
    nb, L = len(order), max(positions) + 1
    # three rows left alone: no slot, a slot outside the pool, a position outside the tables
    slots, positions = slots + [-1, nb * bs, order[-1] * bs], positions + [0, 0, L]
    ang = torch.rand((L, D // 2), generator=g, device="cuda") * 6
    cos, sin = ang.cos(), ang.sin()
    k = torch.full((nb, Hkv, bs, D), 7.0, dtype=torch.bfloat16, device="cuda")
    vt = torch.full((nb, Hkv, D, bs), 7.0, dtype=torch.bfloat16, device="cuda")
    x = qkv.clone()
    out = qkv[:, :H * D] if in_place else torch.full((N, H * D), 9.0, dtype=torch.bfloat16, device="cuda")
    got = _lib.rope_append_blocks(qkv, H, Hkv, D, cos, sin, k, vt, i32(slots), i32(positions), out=out)
    assert got.data_ptr() == out.data_ptr()
    xd = x.double().view(N, H + 2 * Hkv, D)
    c, s = cos.double()[positions[:n]][:, None], sin.double()[positions[:n]][:, None]
    x1, x2 = xd[:n, :, :D // 2], xd[:n, :, D // 2:]
    rot = torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], -1)
    # two products and a sum rounded to fp32, then half a bf16 step
    size = torch.cat([(x1 * c).abs() + (x2 * s).abs()] * 2, -1).clamp(min=0)
    size = torch.maximum(size, torch.cat([(x2 * c).abs() + (x1 * s).abs()] * 2, -1))
    bound = 2.0 ** -8 * rot.abs() + 2.0 ** -22 * size

    def close(a, b, t):
        assert ((a.double() - b).abs() <= t).all()

    close(got[:n].view(n, H, D), rot[:, :H], bound[:, :H])
    sl = torch.tensor(slots[:n], device="cuda")
    close(k[sl // bs, :, sl % bs], rot[:, H:H + Hkv], bound[:, H:H + Hkv])
    assert torch.equal(vt[sl // bs, :, :, sl % bs], x.reshape(N, H + 2 * Hkv, D)[:n, H + Hkv:])
    # nothing else was written
    k[sl // bs, :, sl % bs] = 7.0
    vt[sl // bs, :, :, sl % bs] = 7.0
    assert (k == 7).all() and (vt == 7).all()
    assert torch.equal(got[n:], x[n:, :H * D] if in_place else torch.full_like(got[n:], 9.0))
    assert torch.equal(qkv[:, H * D:], x[:, H * D:])


@pytest.mark.parametrize("H,Hkv,D", [(32, 4, 64), (8, 2, 128)])
def test_append_equals_dense_append(device, H, Hkv, D):
    """One sequence: q, keys and values bit for bit those of the dense cache's append."""
    S, bs = 200, 32
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    qkv = torch.randn((S, (H + 2 * Hkv) * D), generator=g, device="cuda").to(torch.bfloat16)
    ang = torch.rand((256, D // 2), generator=g, device="cuda") * 6
    T = 224
    kc = torch.zeros((1, Hkv, T, D), dtype=torch.bfloat16, device="cuda")
    vt = torch.zeros((1, Hkv, D, T), dtype=torch.bfloat16, device="cuda")
    dense = qkv.clone()
    _lib.rope_append_kv(dense, 1, S, H, Hkv, D, ang.cos(), ang.sin(), kc, vt, i32([0, 0]), pos_offset=3)
    kb = torch.zeros((T // bs, Hkv, bs, D), dtype=torch.bfloat16, device="cuda")
    vb = torch.zeros((T // bs, Hkv, D, bs), dtype=torch.bfloat16, device="cuda")
    q = _lib.rope_append_blocks(qkv, H, Hkv, D, ang.cos(), ang.sin(), kb, vb, i32(list(range(S))),
                                i32(list(range(3, S + 3))))
    assert torch.equal(q, dense[:, :H * D])
    assert torch.equal(kb.transpose(0, 1).reshape(Hkv, T, D), kc[0])
    assert torch.equal(vb.permute(1, 2, 0, 3).reshape(Hkv, D, T), vt[0])


# ---------------------------------------------------------------- attention

# positions held, new ones, prefix, block size, q heads, kv heads, head_dim, rows behind the last
ATTEND = [
    # one token of one sequence: no prefix, a prefix of one, of a block's edge
    ([0], [1], 0, 16, 4, 4, 64, 0), ([0], [1], 1, 16, 8, 2, 128, 0), ([127], [1], 128, 64, 32, 4, 64, 0),
    ([4000], [1], 5, 256, 8, 1, 128, 2),
    # few rows: the prefix with them, and on its own at more columns
    ([5, 0, 300], [1, 1, 1], 700, 32, 32, 8, 128, 0), ([5, 0, 300, 64], [1, 0, 1, 0], 65, 128, 8, 1, 128, 1),
    (list(range(0, 620, 31)), [1] * 20, 1000, 64, 32, 8, 128, 0), ([63] * 33, [1] * 33, 333, 16, 32, 4, 64, 0),
    # a head each, ratios that no power of two divides, many heads on one
    ([10, 200], [1, 1], 77, 16, 6, 6, 64, 0), ([10, 200, 31], [2, 1, 3], 129, 32, 6, 2, 128, 0),
    ([40, 3], [1, 2], 64, 64, 24, 1, 64, 0), ([1, 2], [1, 2], 500, 16, 40, 1, 128, 3),
    ([9] * 5, [1] * 5, 200, 64, 64, 1, 128, 0), ([9] * 5, [3] * 5, 200, 64, 96, 1, 64, 0),
    # a few new ones each
    ([3, 90, 0, 511], [5, 5, 5, 5], 300, 16, 32, 4, 64, 3), ([3, 90, 0], [16, 16, 17], 300, 64, 32, 8, 128, 0),
    ([0, 500], [16, 15], 0, 32, 16, 4, 128, 0),
    # prompts: sequences within a workgroup's columns, over its edges, none between them
    ([0], [200], 0, 64, 32, 8, 128, 0), ([0], [333], 130, 16, 8, 1, 128, 5), ([100], [257], 64, 128, 32, 4, 64, 0),
    ([0, 40, 7, 0], [33, 0, 130, 64], 100, 32, 32, 8, 128, 2), ([0, 0, 0], [20, 300, 1], 511, 64, 4, 4, 64, 0),
    # prompts beside single tokens
    ([700, 0, 30, 5], [1, 400, 1, 18], 129, 64, 32, 8, 128, 0), ([50] * 9, [1, 1, 90, 1, 1, 1, 0, 70, 1], 0, 16, 8, 2, 64, 4),
    # many sequences; two hundred wait
    ([(37 * i) % 150 for i in range(300)], [1] * 300, 64, 16, 8, 2, 64, 0),
    ([(37 * i) % 150 for i in range(260)], [int(i % 5 == 3) for i in range(260)], 90, 32, 4, 1, 128, 0),
    # a long prefix over many workgroups, and a long sequence among short ones
    ([3, 4], [1, 1], 9001, 64, 32, 8, 128, 0), ([2, 6000, 9, 70], [1, 1, 1, 1], 100, 64, 16, 2, 64, 0),
]


@pytest.mark.parametrize("held,new,prefix,bs,H,Hkv,D,pad", ATTEND)
def test_attention(device, held, new, prefix, bs, H, Hkv, D, pad):
    print(f"attention {held[:4]} + {new[:4]} ({len(held)}) prefix={prefix} bs={bs} H={H} Hkv={Hkv} D={D}", flush=True)
    c = Cache(held, new, prefix, bs, H, Hkv, D, pad=pad)
    exact, mag = c.exact()
    rows = c.starts[-1]
    for max_new in (c.max_new, None):
        out = torch.full_like(c.q, 5.0)
        got = c.attend(max_new=max_new, out=out)
        assert got.data_ptr() == out.data_ptr()
        assert_attention(got, exact, mag, rows)
        assert (got[rows:] == 5).all()
        assert torch.equal(got, c.attend(max_new=max_new, out=torch.full_like(out, 5.0)))       # same bits again


@pytest.mark.parametrize("new", [[1, 3, 0, 1700, 2, 16, 17, 1], [2000] + [1] * 20, [1] * 5 + [900, 1, 900]])
def test_attention_of_few_decoded_rows_beside_prompts(device, new):
    """Sequences of few rows among long prompts, behind a prefix."""
    held = [(37 * i) % 200 for i in range(len(new))]
    c = Cache(held, new, 300, 64, 32, 8, 64, pad=3)
    exact, mag = c.exact()
    got = c.attend(max_new=c.max_new, out=torch.full_like(c.q, 5.0))
    assert_attention(got, exact, mag, c.starts[-1])
    assert (got[c.starts[-1]:] == 5).all()


@pytest.mark.parametrize("D,bs", [(64, 16), (128, 64)])
def test_attention_of_the_most_sequences(device, D, bs):
    """2048 sequences, one in three waiting, some without any position; one more is refused."""
    print(f"2048 sequences D={D} bs={bs}", flush=True)
    R = _lib.SHARED_MAX_SEQUENCES
    c = Cache([(11 * i) % 70 if i % 5 else 0 for i in range(R)], [i % 3 for i in range(R)], 90, bs, 4, 2, D, pad=1)
    exact, mag = c.exact()
    got = c.attend(max_new=2, out=torch.full_like(c.q, 5.0))
    assert_attention(got, exact, mag, c.starts[-1])
    assert (got[c.starts[-1]:] == 5).all()
    more = torch.cat([c.tables, c.tables[:1]])
    with pytest.raises(RuntimeError, match="at most 2048"):
        _lib.attention_shared(c.q, 4, 2, D, c.k, c.vt, torch.cat([c.row_starts, c.row_starts[-1:]]),
                              torch.cat([c.lens, c.lens[:1]]), more, c.scale)


@pytest.mark.parametrize("max_new", [1, 3, 20])
@pytest.mark.parametrize("prefix", [0, 700])
def test_attention_beyond_max_new_harms_nobody(device, max_new, prefix):
    """Sequences of more rows than max_new: the others' rows are right, and nothing is written
    outside the rows and the workspace."""
    new = [1, 5, 2, 40, 1, 16, 3]
    c = Cache([50, 3, 200, 0, 129, 10, 64], new, prefix, 64, 8, 2, 128, pad=2)
    exact, mag = c.exact()
    pre = 0 if c.prefix_table is None else c.prefix_table.numel() * c.bs
    need = _lib.attention_shared_workspace_bytes(c.N, len(new), 8, 2, 128, c.tables.shape[1] * c.bs, pre, max_new)
    buf = torch.full((need + 4096,), 77, dtype=torch.uint8, device="cuda")
    got = c.attend(max_new=max_new, out=torch.full_like(c.q, 5.0), workspace=buf[:need])
    assert (buf[need:] == 77).all() and (got[c.starts[-1]:] == 5).all()
    for r, n in enumerate(new):
        if n <= max_new:
            rows = slice(c.starts[r], c.starts[r + 1])
            assert_attention(got[rows], exact[rows], mag[rows], n)


def attend_without_first(c, max_new):
    """The call of c without its first sequence: row starts that begin above 0, and rows of nobody."""
    pre = dict(prefix_table=c.prefix_table, prefix_len=c.prefix_len) if c.prefix_table is not None else {}
    return _lib.attention_shared(c.q, c.H, c.Hkv, c.D, c.k, c.vt, c.row_starts[1:], c.lens[1:], c.tables[1:], c.scale,
                                 max_new=max_new, out=torch.full_like(c.q, 5.0), **pre)


# rows of the first sequence, which the call leaves out, and of the others; room of the tables in blocks
@pytest.mark.parametrize("held,new,prefix,bs,H,Hkv,D,width,max_new", [
    ([0, 700, 0], [299, 1, 0], 0, 64, 32, 8, 128, 128, None),       # cut tiles, merged row by row
    ([0, 40, 300, 3], [40, 30, 2, 40], 9000, 64, 8, 2, 64, 10, None),
    ([0, 40, 300, 3], [2, 1, 2, 1], 70, 16, 8, 2, 64, 30, 3),       # few rows, merged row by row
    ([0, 40, 300, 3], [9, 3, 2, 1], 0, 32, 32, 8, 128, 30, 3),      # few rows, by sequence
    ([0, 40, 30, 3], [120, 1, 50, 2], 100, 64, 32, 8, 128, 4, None),        # whole tiles, parts by sequence
    ([0, 40, 30, 3], [90, 5, 70, 8], 20, 16, 32, 4, 64, 8, None),
    ([0, 5], [700, 1], 33, 64, 4, 4, 64, 12, 1),                    # one row's slot behind 700 rows
])
def test_attention_leaves_rows_before_the_first_sequence(device, held, new, prefix, bs, H, Hkv, D, width, max_new):
    print(f"rows from {new[0]}: {new[1:]} prefix={prefix} bs={bs} H={H} Hkv={Hkv} D={D}", flush=True)
    c = Cache(held, new, prefix, bs, H, Hkv, D, pad=2, width=width)
    exact, mag = c.exact()
    got, rows = attend_without_first(c, max_new), slice(c.starts[1], c.starts[-1])
    assert_attention(got[rows], exact[rows], mag[rows], rows.stop - rows.start)
    assert (got[:rows.start] == 5).all() and (got[rows.stop:] == 5).all()


def test_attention_strides_scale_and_wide_tables(device):
    c = Cache([30, 2, 200], [1, 1, 40], 150, 32, 8, 2, 128, pad=2, width=50)
    wide = torch.zeros((c.N, 2 * 1024 + 8), dtype=torch.bfloat16, device="cuda")
    wide[:, :1024] = c.q
    for scale in (0.02, 1.0):
        exact, mag = c.exact(scale)
        out = torch.full((c.N, 1100), 5.0, dtype=torch.bfloat16, device="cuda")
        c.attend(q=wide[:, :1024], scale=scale, out=out[:, :1024])
        # |q k| scale is 11 times that of 1 / sqrt(128) at scale 1: the fp32 part of the bound with it
        got, rows = out[:, :1024].reshape(c.N, 8, 128)[:c.starts[-1]].double(), c.starts[-1]
        bound = 2.0 ** -8 * exact[:rows].abs() + (2.0 ** -8 + 2.0 ** -8.5) * mag[:rows]
        assert ((got - exact[:rows]).abs() <= bound).all()
        assert (out[:, 1024:] == 5).all() and (out[rows:] == 5).all()


@pytest.mark.parametrize("new,bs", [([1, 1, 1], 64), ([3, 2, 3], 16), ([60, 50, 70], 64), ([1, 200, 2], 32)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_attention_keeps_values_that_are_not_attended_out(device, new, bs, D, value):
    """A value that is not finite reaches the rows that attend it and no others: not another
    sequence's, not an earlier row's of its own."""
    print(f"not finite: {new} bs={bs} D={D} {value}", flush=True)
    held = [40, 70, 9]
    c = Cache(held, new, 100, bs, 8, 2, D)
    exact, mag = c.exact()
    # the middle sequence's second new position, or its last held one
    p = held[1] + 1 if new[1] > 1 else held[1] - 1
    c.vt[c.tables[1, p // bs].item(), :, :, p % bs] = value
    got = c.attend(max_new=c.max_new)
    sees = torch.zeros(c.N, dtype=torch.bool, device="cuda")
    sees[c.starts[1] + max(0, p - held[1]):c.starts[2]] = True
    assert not torch.isfinite(got[sees]).any()
    got = got.clone()
    got[sees], exact[sees], mag[sees] = 0, 0, 0
    assert_attention(got, exact, mag, c.N)


@pytest.mark.parametrize("new,prefix,bs", [([1, 1, 1], 0, 64), ([1, 1, 1], 2000, 16), ([3, 9, 3], 100, 64),
                                           ([1, 200, 2], 100, 32), ([90, 80, 2], 3000, 64)])
def test_attention_of_a_query_that_is_no_number(device, new, prefix, bs):
    """A query with a NaN makes its own row's head NaN and nothing else."""
    H, D = 8, 64
    c = Cache([40, 70, 9], new, prefix, bs, H, 2, D)
    exact, mag = c.exact()
    row, h = c.starts[2] - 1, 5
    c.q[row, h * D + 3] = float("nan")
    got = c.attend(max_new=c.max_new).clone().view(c.N, H, D)
    assert torch.isnan(got[row, h]).all()
    got[row, h], exact[row, h], mag[row, h] = 0, 0, 0
    assert_attention(got.view(c.N, H * D), exact, mag, c.N)


def test_attention_row_without_a_key_is_zero(device):
    """No prefix and a length below the rows given: the first rows have nothing to attend."""
    for n in (6, 100, 2000):
        c = Cache([0, 8], [n, 2], 0, 16, 8, 2, 64)
        c.lens[0] = n - 2
        got = c.attend(out=torch.full_like(c.q, 5.0))
        assert (got[:2] == 0).all() and torch.isfinite(got).all() and not (got[2:] == 5).any()


def test_attention_beyond_32_bit_offsets(device):
    """Blocks past the first 4 GB of the pool."""
    H, Hkv, D, bs = 8, 8, 128, 64
    nb = (1 << 32) // (Hkv * bs * D * 2) + 40
    c = Cache([100, 20], [1, 90], 130, bs, H, Hkv, D)
    k = torch.empty((nb, Hkv, bs, D), dtype=torch.bfloat16, device="cuda")
    vt = torch.empty((nb, Hkv, D, bs), dtype=torch.bfloat16, device="cuda")
    n = c.k.shape[0]
    k[-n:], vt[-n:] = c.k, c.vt
    exact, mag = c.exact()
    c.k, c.vt = k, vt
    c.tables += nb - n
    c.prefix_table += nb - n
    assert_attention(c.attend(), exact, mag, c.N)
    # and the append into them
    qkv = torch.randn((3, (H + 2 * Hkv) * D), device="cuda").to(torch.bfloat16)
    ones, zeros = torch.ones((4, D // 2), device="cuda"), torch.zeros((4, D // 2), device="cuda")
    last = nb * bs - 1
    _lib.rope_append_blocks(qkv, H, Hkv, D, ones, zeros, k, vt, i32([last, last - 9, -1]), i32([0, 1, 2]))
    x = qkv.view(3, H + 2 * Hkv, D)
    assert torch.equal(k[-1, :, -1], x[0, H:H + Hkv]) and torch.equal(k[-1, :, -10], x[1, H:H + Hkv])
    assert torch.equal(vt[-1, :, :, -1], x[0, H + Hkv:]) and torch.equal(vt[-1, :, :, -10], x[1, H + Hkv:])


# ---------------------------------------------------------------- together


@pytest.mark.parametrize("stream", ["default", "other"])
def test_captured_steps_of_two_graphs(device, stream):
    """Tables, append and attention of a decode step in a graph, replayed at growing lengths, two
    graphs over the same buffers and workspace in turn: bit for bit the eager steps, on a
    stream of their own too."""
    H, Hkv, D, bs, P, R = 8, 2, 64, 16, 50, 5
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    held = [0, 15, 16, 40, 3]
    cos, sin = torch.rand((200, D // 2), generator=g, device="cuda"), torch.rand((200, D // 2), generator=g, device="cuda")
    rowsrc = torch.randn((6, R, (H + 2 * Hkv) * D), generator=g, device="cuda").to(torch.bfloat16)

    def setup():
        c = Cache(held, [0] * R, P, bs, H, Hkv, D, seed=2, width=6)
        nb = c.k.shape[0]
        k = torch.cat([c.k, torch.zeros((40, Hkv, bs, D), dtype=torch.bfloat16, device="cuda")])
        vt = torch.cat([c.vt, torch.zeros((40, Hkv, D, bs), dtype=torch.bfloat16, device="cuda")])
        free = i32(list(range(nb, nb + 40)))
        step = _lib.block_step_buffers(R, R, "cuda")._replace(lengths=c.lens.clone(), n_free=i32([40]))
        return dict(c=c, k=k, vt=vt, free=free, step=step, qkv=torch.empty_like(rowsrc[0]),
                    q=torch.empty((R, H * D), dtype=torch.bfloat16, device="cuda"),
                    out=torch.empty((R, H * D), dtype=torch.bfloat16, device="cuda"),
                    ws=torch.empty(_lib.attention_shared_workspace_bytes(R, R, H, Hkv, D, 6 * bs,
                                                                         c.prefix_table.numel() * bs, 1),
                                   dtype=torch.uint8, device="cuda"), new=i32([1] * R))

    def one(s):
        st, c = s["step"], s["c"]
        _lib.block_tables(st.lengths, s["new"], c.tables, s["free"], st.n_free, bs, R, prefix_len=c.prefix_len, out=st)
        _lib.rope_append_blocks(s["qkv"], H, Hkv, D, cos, sin, s["k"], s["vt"], st.slots, st.positions, out=s["q"])
        _lib.attention_shared(s["q"], H, Hkv, D, s["k"], s["vt"], st.row_starts, st.lengths, c.tables, c.scale,
                              prefix_table=c.prefix_table, prefix_len=c.prefix_len, max_new=1, out=s["out"],
                              workspace=s["ws"])

    eager, want = setup(), []
    for i in range(6):
        eager["qkv"].copy_(rowsrc[i])
        one(eager)
        want.append(eager["out"].clone())
    st = torch.cuda.Stream() if stream == "other" else torch.cuda.current_stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        s = setup()
        lengths, n_free = s["step"].lengths.clone(), s["step"].n_free.clone()
        graphs = []
        for _ in range(2):
            torch.cuda.synchronize()
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                one(s)
            graphs.append(gr)
        s["step"].lengths.copy_(lengths)
        s["step"].n_free.copy_(n_free)
        for i in range(6):
            s["qkv"].copy_(rowsrc[i])
            graphs[i % 2].replay()
            assert torch.equal(s["out"], want[i]), i
        assert s["step"].lengths.tolist() == [h + 6 for h in held] and s["step"].status.item() == 0


def test_prompt_then_tokens_equals_dense_attention(device):
    """One sequence, no prefix: a prompt, then single tokens, the same positions attended as
    by the dense cache's kernels (within both sides' roundings)."""
    H, Hkv, D, bs, S = 8, 2, 128, 64, 150
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    qkv = torch.randn((S + 4, (H + 2 * Hkv) * D), generator=g, device="cuda").to(torch.bfloat16)
    ang = torch.rand((256, D // 2), generator=g, device="cuda") * 6
    cos, sin = ang.cos(), ang.sin()
    kc = torch.zeros((1, Hkv, 256, D), dtype=torch.bfloat16, device="cuda")
    vt = torch.zeros((1, Hkv, D, 256), dtype=torch.bfloat16, device="cuda")
    kb = torch.zeros((8, Hkv, bs, D), dtype=torch.bfloat16, device="cuda")
    vb = torch.zeros((8, Hkv, D, bs), dtype=torch.bfloat16, device="cuda")
    tables, free, nf, ln = i32([[0] * 4]), i32(list(range(8))), i32([8]), i32([0])
    for a, b in [(0, S)] + [(S + i, S + i + 1) for i in range(4)]:
        n = b - a
        dense = qkv[a:b].clone()
        _lib.rope_append_kv(dense, 1, n, H, Hkv, D, cos, sin, kc, vt, i32([a, 0]))
        want = _lib.attention(dense, 1, n, H, Hkv, D, kc, vt, i32([a, 0]), D ** -0.5)
        st = _lib.block_tables(ln, i32([n]), tables, free, nf, bs, n)
        q = _lib.rope_append_blocks(qkv[a:b], H, Hkv, D, cos, sin, kb, vb, st.slots, st.positions)
        got = _lib.attention_shared(q, H, Hkv, D, kb, vb, st.row_starts, st.lengths, tables, D ** -0.5)
        ln, nf = st.lengths, st.n_free
        # |v| <= 4.5 at these sizes: two roundings of each side, 4 * 2^-8 * the largest |v|
        assert (got.double() - want.double()).abs().max() <= 4 * 2.0 ** -8 * 4.5
        assert torch.nn.functional.cosine_similarity(got.double(), want.double()).min() > 0.9999
