"""The quantized key/value cache in blocks on the GPU: append, reading back and attention, against
``_lib.quantize`` and float64."""
import pytest
import torch

from shardcompute_amd import _lib
from tests.block_util import cdiv
from tests.quant_util import QuantCache, assert_attention, stored, write
from tests.test_gpu_blocks import APPENDS, ATTEND

pytestmark = pytest.mark.gpu
BITS = [4, 8]


def i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------- append and reading back


def _quantized_rows(x, bits):
    """bf16(scale code + bias) of x [..., D] by the weights' quantizer and dequantizer."""
    wq, s, b = _lib.quantize(x.float().reshape(-1, x.shape[-1]), bits=bits)
    return _lib.dequantize(wq, s, b, bits=bits).view(x.shape)


@pytest.mark.parametrize("new,held,bs,H,Hkv,D", APPENDS)
@pytest.mark.parametrize("bits", BITS)
def test_append_quantizes_what_the_bf16_append_writes(device, new, held, bs, H, Hkv, D, bits):
    """q, and the values the codes stand for, bit for bit those of rope_append_blocks followed by
    quantize and dequantize; nothing else is written."""
    print(f"append {bits} bits {new[:3]} held {held[:3]} bs={bs} H={H} Hkv={Hkv} D={D}", flush=True)
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
    k = torch.zeros((nb, Hkv, bs, D), dtype=torch.bfloat16, device="cuda")
    vt = torch.zeros((nb, Hkv, D, bs), dtype=torch.bfloat16, device="cuda")
    want = torch.full((N, H * D), 9.0, dtype=torch.bfloat16, device="cuda")
    _lib.rope_append_blocks(qkv, H, Hkv, D, ang.cos(), ang.sin(), k, vt, i32(slots), i32(positions), out=want)
    pool = _lib.quantized_pool(nb, Hkv, bs, D, bits=bits)
    got = torch.full_like(want, 9.0)
    assert _lib.rope_append_quantized(qkv, H, Hkv, D, ang.cos(), ang.sin(), pool, i32(slots), i32(positions), bits=bits,
                                      out=got) is got
    assert torch.equal(got, want)
    sl = torch.tensor(slots[:n], device="cuda")
    kr, vr = _lib.read_quantized(pool, Hkv, D, i32(slots[:n]), bits=bits)
    assert torch.equal(kr, _quantized_rows(k[sl // bs, :, sl % bs], bits))
    assert torch.equal(vr, _quantized_rows(vt[sl // bs, :, :, sl % bs], bits))
    # every other position of the pool is still zero, and so are its bytes
    rest = torch.ones(nb * bs, dtype=torch.bool, device="cuda")
    rest[sl] = False
    kr, vr = _lib.read_quantized(pool, Hkv, D, rest.nonzero()[:, 0].to(torch.int32), bits=bits)
    assert not kr.any() and not vr.any()
    # in place: the q part of qkv
    again = buf.clone()
    _lib.rope_append_quantized(again[:, :W], H, Hkv, D, ang.cos(), ang.sin(), pool.clone(), i32(slots), i32(positions),
                               bits=bits, out=again[:, :H * D])
    assert torch.equal(again[:n, :H * D], want[:n]) and torch.equal(again[n:], buf[n:])
    assert torch.equal(again[:, H * D:], buf[:, H * D:])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bits", BITS)
def test_append_of_edge_values(device, D, bits):
    """Groups of one value, of zeros, of both signs' zeros, tiny and large ones, values on the
    border of two codes: the quantizer's values bit for bit; neighbours written later or earlier
    do not matter."""
    n, Hkv = 48, 2
    g = torch.Generator(device="cuda")
    g.manual_seed(D + bits)
    x = torch.randn((n, 2 * Hkv, D), generator=g, device="cuda")
    x[0], x[1], x[2], x[3] = 0.0, -0.0, 1.5, -2.25
    x[4, :, ::2], x[5, :, 1:] = 0.0, 0.0
    x[6] *= 1e-9
    x[7] *= 1e25
    x[8] = x[8].abs()
    x[9] = -x[9].abs()
    x[10, :, 5] = 1000.0
    x[11] = torch.arange(D, device="cuda") - 20.0                # quotients on borders
    x[12] = (torch.arange(D, device="cuda") % 31) * 0.5
    x[13, :, :63], x[13, :, 63:] = 3.0, 3.015625
    x = x.to(torch.bfloat16)
    for order in (torch.arange(n), torch.arange(n - 1, -1, -1), torch.randperm(n)):
        pool = torch.full(_lib.quantized_pool_shape(3, Hkv, 16, D, bits), 255, dtype=torch.uint8, device="cuda")
        for part in order.split(7):                              # some rows at a time
            write(pool, x[part, :Hkv], x[part, Hkv:], part.to("cuda"), bits)
        k, v = _lib.read_quantized(pool, Hkv, D, torch.arange(n, dtype=torch.int32, device="cuda"), bits=bits)
        assert torch.equal(k, _quantized_rows(x[:, :Hkv], bits)) and torch.equal(v, _quantized_rows(x[:, Hkv:], bits))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bits", BITS)
def test_values_that_are_not_finite_stay_in_their_group(device, D, bits):
    x = torch.ones((40, 2, D), device="cuda").to(torch.bfloat16)
    x[:, 0] *= torch.arange(1, 41, device="cuda")[:, None]
    y = x.clone()
    y[7, 1, 3], y[21, 0, D - 1] = float("nan"), float("inf")
    pool = _lib.quantized_pool(3, 2, 16, D, bits=bits)
    write(pool, y, y, torch.arange(40, device="cuda"), bits)
    for i, got in enumerate(_lib.read_quantized(pool, 2, D, torch.arange(40, dtype=torch.int32, device="cuda"), bits=bits)):
        bad = torch.zeros_like(x, dtype=torch.bool)
        bad[7, 1, :64], bad[21, 0, D - 64:] = True, True
        if i == 0:               # a key's dims d and d + D / 2 are rotated together (inf * 0 is no number)
            bad[7, 1], bad[21, 0] = True, True
        assert not torch.isfinite(got[bad]).any()
        assert torch.equal(got[~bad], _quantized_rows(x, bits)[~bad])


@pytest.mark.parametrize("bits", BITS)
def test_read_back_any_slots(device, bits):
    """Slots outside the pool give zeros, the same slot twice the same values; one slot, none."""
    g = torch.Generator(device="cuda")
    g.manual_seed(bits)
    x = torch.randn((64, 6, 128), generator=g, device="cuda").to(torch.bfloat16)
    pool = _lib.quantized_pool(2, 3, 32, 128, bits=bits)
    write(pool, x[:, :3], x[:, 3:], torch.arange(64, device="cuda"), bits)
    slots = [5, -1, 63, 5, 64, 0, 1 << 30, -(1 << 31), 40]
    k, v = _lib.read_quantized(pool, 3, 128, i32(slots), bits=bits)
    for i, s in enumerate(slots):
        there = 0 <= s < 64
        assert torch.equal(k[i], _quantized_rows(x[s, :3], bits)) if there else not k[i].any()
        assert torch.equal(v[i], _quantized_rows(x[s, 3:], bits)) if there else not v[i].any()
    assert _lib.read_quantized(pool, 3, 128, i32([]), bits=bits)[0].shape == (0, 3, 128)


# ---------------------------------------------------------------- attention


@pytest.mark.parametrize("held,new,prefix,bs,H,Hkv,D,pad", ATTEND)
@pytest.mark.parametrize("bits", BITS)
def test_attention(device, held, new, prefix, bs, H, Hkv, D, pad, bits):
    print(f"attention {bits} bits {held[:4]} + {new[:4]} ({len(held)}) prefix={prefix} bs={bs} H={H} Hkv={Hkv} D={D}",
          flush=True)
    c = QuantCache(bits, held, new, prefix, bs, H, Hkv, D, pad=pad)
    exact, bound = c.exact()
    rows = c.starts[-1]
    for max_new in (c.max_new, None):
        out = torch.full_like(c.q, 5.0)
        got = c.attend(max_new=max_new, out=out)
        assert got.data_ptr() == out.data_ptr()
        assert_attention(got, exact, bound, rows)
        assert (got[rows:] == 5).all()
        assert torch.equal(got, c.attend(max_new=max_new, out=torch.full_like(out, 5.0)))       # same bits again


@pytest.mark.parametrize("new", [[1, 3, 0, 1700, 2, 16, 17, 1], [1] * 5 + [900, 1, 900]])
@pytest.mark.parametrize("bits", BITS)
def test_attention_of_few_decoded_rows_beside_prompts(device, new, bits):
    held = [(37 * i) % 200 for i in range(len(new))]
    c = QuantCache(bits, held, new, 300, 64, 32, 8, 64, pad=3)
    exact, bound = c.exact()
    got = c.attend(max_new=c.max_new, out=torch.full_like(c.q, 5.0))
    assert_attention(got, exact, bound, c.starts[-1])
    assert (got[c.starts[-1]:] == 5).all()


@pytest.mark.parametrize("D,bs,bits", [(64, 16, 8), (128, 64, 4)])
def test_attention_of_the_most_sequences(device, D, bs, bits):
    """2048 sequences, one in three waiting, some without any position; one more is refused."""
    R = _lib.SHARED_MAX_SEQUENCES
    c = QuantCache(bits, [(11 * i) % 70 if i % 5 else 0 for i in range(R)], [i % 3 for i in range(R)], 90, bs, 4, 2, D, pad=1)
    exact, bound = c.exact()
    got = c.attend(max_new=2, out=torch.full_like(c.q, 5.0))
    assert_attention(got, exact, bound, c.starts[-1])
    assert (got[c.starts[-1]:] == 5).all()
    more = torch.cat([c.tables, c.tables[:1]])
    with pytest.raises(RuntimeError, match="at most 2048"):
        _lib.attention_quantized(c.q, 4, 2, D, c.pool, torch.cat([c.row_starts, c.row_starts[-1:]]),
                                 torch.cat([c.lens, c.lens[:1]]), more, c.scale, bits=bits)


@pytest.mark.parametrize("max_new", [1, 3, 20])
@pytest.mark.parametrize("prefix", [0, 700])
@pytest.mark.parametrize("bits", BITS)
def test_attention_beyond_max_new_harms_nobody(device, max_new, prefix, bits):
    """Sequences of more rows than max_new: the others' rows are right, and nothing is written
    outside the rows and the workspace."""
    new = [1, 5, 2, 40, 1, 16, 3]
    c = QuantCache(bits, [50, 3, 200, 0, 129, 10, 64], new, prefix, 64, 8, 2, 128, pad=2)
    exact, bound = c.exact()
    need = c.workspace_bytes(max_new)
    buf = torch.full((need + 4096,), 77, dtype=torch.uint8, device="cuda")
    got = c.attend(max_new=max_new, out=torch.full_like(c.q, 5.0), workspace=buf[:need])
    assert (buf[need:] == 77).all() and (got[c.starts[-1]:] == 5).all()
    for r, n in enumerate(new):
        if n <= max_new:
            rows = slice(c.starts[r], c.starts[r + 1])
            assert_attention(got[rows], exact[rows], bound[rows], n)


# rows of the first sequence, which the call leaves out, and of the others; room of the tables in blocks
@pytest.mark.parametrize("held,new,prefix,bs,H,Hkv,D,width,max_new", [
    ([0, 700, 0], [299, 1, 0], 0, 64, 32, 8, 128, 128, None), ([0, 40, 300, 3], [40, 30, 2, 40], 9000, 64, 8, 2, 64, 150, None),
    ([0, 40, 300, 3], [2, 1, 2, 1], 70, 16, 8, 2, 64, 30, 3), ([0, 40, 300, 3], [9, 3, 2, 1], 0, 32, 32, 8, 128, 30, 3),
    ([0, 40, 30, 3], [120, 1, 50, 2], 100, 64, 32, 8, 128, 4, None), ([0, 5], [700, 1], 33, 64, 4, 4, 64, 12, 1),
])
@pytest.mark.parametrize("bits", BITS)
def test_attention_leaves_rows_before_the_first_sequence(device, held, new, prefix, bs, H, Hkv, D, width, max_new, bits):
    c = QuantCache(bits, held, new, prefix, bs, H, Hkv, D, pad=2, width=width)
    exact, bound = c.exact()
    rows = slice(c.starts[1], c.starts[-1])
    pre = dict(prefix_table=c.prefix_table, prefix_len=c.prefix_len) if prefix else {}
    got = _lib.attention_quantized(c.q, H, Hkv, D, c.pool, c.row_starts[1:], c.lens[1:], c.tables[1:], c.scale, bits=bits,
                                   max_new=max_new, out=torch.full_like(c.q, 5.0), **pre)
    assert_attention(got[rows], exact[rows], bound[rows], rows.stop - rows.start)
    assert (got[:rows.start] == 5).all() and (got[rows.stop:] == 5).all()


@pytest.mark.parametrize("bits", BITS)
def test_attention_strides_scale_and_wide_tables(device, bits):
    c = QuantCache(bits, [30, 2, 200], [1, 1, 40], 150, 32, 8, 2, 128, pad=2, width=50)
    wide = torch.zeros((c.N, 2 * 1024 + 8), dtype=torch.bfloat16, device="cuda")
    wide[:, :1024] = c.q
    for scale in (0.02, 0.3):
        exact, bound = c.exact(scale)
        out = torch.full((c.N, 1100), 5.0, dtype=torch.bfloat16, device="cuda")
        c.attend(q=wide[:, :1024], scale=scale, out=out[:, :1024])
        rows = c.starts[-1]
        got = out[:, :1024].reshape(c.N, 8, 128)[:rows].double()
        assert ((got - exact[:rows]).abs() <= bound[:rows]).all()
        assert (out[:, 1024:] == 5).all() and (out[rows:] == 5).all()


@pytest.mark.parametrize("new,bs", [([1, 1, 1], 64), ([3, 2, 3], 16), ([60, 50, 70], 64), ([1, 200, 2], 32)])
@pytest.mark.parametrize("D,bits", [(64, 4), (128, 4), (64, 8), (128, 8)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("where", ["key", "value"])
def test_attention_keeps_values_that_are_not_attended_out(device, new, bs, D, bits, value, where):
    """A key or value that is not finite reaches the rows that attend it and no others: not
    another sequence's, not an earlier row's of its own."""
    held = [40, 70, 9]
    c = QuantCache(bits, held, new, 100, bs, 8, 2, D)
    exact, bound = c.exact()
    # the middle sequence's second new position, or its last held one
    p = held[1] + 1 if new[1] > 1 else held[1] - 1
    b = c.tables[1, p // bs].item()
    k, v = c.k[b, :, p % bs].clone()[None], c.vt[b, :, :, p % bs].clone()[None]
    (k if where == "key" else v)[...] = value
    write(c.pool, k, v, i32([b * bs + p % bs]), bits)
    got = c.attend(max_new=c.max_new)
    sees = torch.zeros(c.N, dtype=torch.bool, device="cuda")
    sees[c.starts[1] + max(0, p - held[1]):c.starts[2]] = True
    assert not torch.isfinite(got[sees]).any()
    got = got.clone()
    got[sees], exact[sees], bound[sees] = 0, 0, 0
    assert_attention(got, exact, bound, c.N)


@pytest.mark.parametrize("new,prefix,bs", [([1, 1, 1], 0, 64), ([1, 1, 1], 2000, 16), ([3, 9, 3], 100, 64),
                                           ([1, 200, 2], 100, 32), ([90, 80, 2], 3000, 64)])
@pytest.mark.parametrize("bits", BITS)
def test_attention_of_a_query_that_is_no_number(device, new, prefix, bs, bits):
    """A query with a NaN makes its own row's head NaN and nothing else."""
    H, D = 8, 64
    c = QuantCache(bits, [40, 70, 9], new, prefix, bs, H, 2, D)
    exact, bound = c.exact()
    row, h = c.starts[2] - 1, 5
    c.q[row, h * D + 3] = float("nan")
    got = c.attend(max_new=c.max_new).clone().view(c.N, H, D)
    assert torch.isnan(got[row, h]).all()
    got[row, h], exact[row, h], bound[row, h] = 0, 0, 0
    assert_attention(got.view(c.N, H * D), exact, bound, c.N)


@pytest.mark.parametrize("bits", BITS)
def test_attention_row_without_a_key_is_zero(device, bits):
    """No prefix and a length below the rows given: the first rows have nothing to attend."""
    for n in (6, 100, 2000):
        c = QuantCache(bits, [0, 8], [n, 2], 0, 16, 8, 2, 64)
        c.lens[0] = n - 2
        got = c.attend(out=torch.full_like(c.q, 5.0))
        assert (got[:2] == 0).all() and torch.isfinite(got).all() and not (got[2:] == 5).any()


@pytest.mark.parametrize("scale_of_v,shift", [(1.0, 50.0), (1e-3, 4.0), (1e15, 0.0)])
@pytest.mark.parametrize("bits", BITS)
def test_attention_of_values_far_from_zero(device, scale_of_v, shift, bits):
    """Values whose groups lie on one side of zero, small and large ones, over keys that all weigh
    about the same: the codes' offset is taken off exactly enough."""
    c = QuantCache(bits, [3000, 40], [1, 2], 1500, 64, 8, 2, 128)
    for p in (c.k, c.vt):
        there = ~torch.isnan(p)
        p[there] = ((p[there].float() + shift) * scale_of_v).to(torch.bfloat16) if p is c.vt else (p[there].float() * 0.1).to(p.dtype)
    at = (~torch.isnan(c.k[:, 0, :, 0])).nonzero()
    write(c.pool, c.k[at[:, 0], :, at[:, 1]], c.vt[at[:, 0], :, :, at[:, 1]], at[:, 0] * c.bs + at[:, 1], bits)
    exact, bound = c.exact()
    assert_attention(c.attend(), exact, bound, c.N)


@pytest.mark.parametrize("bits", BITS)
def test_attention_beyond_32_bit_offsets(device, bits):
    """Blocks past the first 4 GB of the pool."""
    H, Hkv, D, bs = 8, 8, 128, 64
    shape = _lib.quantized_pool_shape(1, Hkv, bs, D, bits)
    c = QuantCache(bits, [100, 20], [1, 90], 130, bs, H, Hkv, D)
    nb, n = (1 << 32) // (Hkv * shape[2] * shape[3]) + 40, c.pool.shape[0]
    pool = torch.empty((nb, *shape[1:]), dtype=torch.uint8, device="cuda")
    pool[-n:] = c.pool
    exact, bound = c.exact()
    c.pool = pool
    c.tables += nb - n
    c.prefix_table += nb - n
    assert_attention(c.attend(), exact, bound, c.N)
    # and the append into them
    x = torch.randn((3, 2 * Hkv, D), device="cuda").to(torch.bfloat16)
    last = nb * bs - 1
    write(pool, x[:, :Hkv], x[:, Hkv:], i32([last, last - 9, -1]), bits)
    k, v = _lib.read_quantized(pool, Hkv, D, i32([last, last - 9]), bits=bits)
    assert torch.equal(k, _quantized_rows(x[:2, :Hkv], bits)) and torch.equal(v, _quantized_rows(x[:2, Hkv:], bits))


# ---------------------------------------------------------------- together


@pytest.mark.parametrize("stream", ["default", "other"])
@pytest.mark.parametrize("bits", BITS)
def test_captured_steps_of_two_graphs(device, stream, bits):
    """Tables, append, attention and reading back of a decode step in a graph, replayed at growing
    lengths, two graphs over the same buffers and workspace in turn: bit for bit the eager
    steps, on a stream of their own too."""
    H, Hkv, D, bs, P, R = 8, 2, 64, 16, 50, 5
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    held = [0, 15, 16, 40, 3]
    cos, sin = torch.rand((200, D // 2), generator=g, device="cuda"), torch.rand((200, D // 2), generator=g, device="cuda")
    rowsrc = torch.randn((6, R, (H + 2 * Hkv) * D), generator=g, device="cuda").to(torch.bfloat16)

    def setup():
        c = QuantCache(bits, held, [0] * R, P, bs, H, Hkv, D, seed=2, width=6, blocks_more=40)
        nb = c.k.shape[0]
        step = _lib.block_step_buffers(R, R, "cuda")._replace(lengths=c.lens.clone(), n_free=i32([40]))
        ws = _lib.attention_quantized_workspace_bytes(R, R, H, Hkv, D, 6 * bs, c.prefix_table.numel() * bs, 1, bits=bits)
        return dict(c=c, free=i32(list(range(nb, nb + 40))), step=step, qkv=torch.empty_like(rowsrc[0]),
                    q=torch.empty((R, H * D), dtype=torch.bfloat16, device="cuda"),
                    out=torch.empty((R, H * D), dtype=torch.bfloat16, device="cuda"),
                    ws=torch.empty(max(ws, 16), dtype=torch.uint8, device="cuda"), new=i32([1] * R))

    def one(s):
        st, c = s["step"], s["c"]
        _lib.block_tables(st.lengths, s["new"], c.tables, s["free"], st.n_free, bs, R, prefix_len=c.prefix_len, out=st)
        _lib.rope_append_quantized(s["qkv"], H, Hkv, D, cos, sin, c.pool, st.slots, st.positions, bits=bits, out=s["q"])
        _lib.attention_quantized(s["q"], H, Hkv, D, c.pool, st.row_starts, st.lengths, c.tables, c.scale, bits=bits,
                                 prefix_table=c.prefix_table, prefix_len=c.prefix_len, max_new=1, out=s["out"],
                                 workspace=s["ws"])
        s["read"] = _lib.read_quantized(c.pool, Hkv, D, st.slots, bits=bits)

    eager, want = setup(), []
    for i in range(6):
        eager["qkv"].copy_(rowsrc[i])
        one(eager)
        want.append((eager["out"].clone(), *(t.clone() for t in eager["read"])))
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
            graphs.append((gr, s["read"]))
        s["step"].lengths.copy_(lengths)
        s["step"].n_free.copy_(n_free)
        for i in range(6):
            s["qkv"].copy_(rowsrc[i])
            graphs[i % 2][0].replay()
            for a, b in zip((s["out"], *graphs[i % 2][1]), want[i]):
                assert torch.equal(a, b), i
        assert s["step"].lengths.tolist() == [h + 6 for h in held] and s["step"].status.item() == 0


@pytest.mark.parametrize("bits", BITS)
def test_prompt_then_tokens_is_the_bf16_caches_attention_of_the_read_values(device, bits):
    """One sequence, a prompt, then single tokens: as attention_shared over a bf16 cache that holds
    the values read back (their bf16 rounding, 2^-8 of a value, and both sides' roundings apart)."""
    H, Hkv, D, bs, S = 8, 2, 128, 64, 150
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    qkv = torch.randn((S + 4, (H + 2 * Hkv) * D), generator=g, device="cuda").to(torch.bfloat16)
    ang = torch.rand((256, D // 2), generator=g, device="cuda") * 6
    pool = _lib.quantized_pool(8, Hkv, bs, D, bits=bits)
    kb = torch.zeros((8, Hkv, bs, D), dtype=torch.bfloat16, device="cuda")
    vb = torch.zeros((8, Hkv, D, bs), dtype=torch.bfloat16, device="cuda")
    tables, free, nf, ln = i32([[0] * 4]), i32(list(range(8))), i32([8]), i32([0])
    for a, b in [(0, S)] + [(S + i, S + i + 1) for i in range(4)]:
        n = b - a
        st = _lib.block_tables(ln, i32([n]), tables, free, nf, bs, n)
        q = _lib.rope_append_quantized(qkv[a:b], H, Hkv, D, ang.cos(), ang.sin(), pool, st.slots, st.positions, bits=bits)
        k, v = _lib.read_quantized(pool, Hkv, D, st.slots, bits=bits)
        sl = st.slots.long()
        kb[sl // bs, :, sl % bs], vb[sl // bs, :, :, sl % bs] = k, v
        want = _lib.attention_shared(q, H, Hkv, D, kb, vb, st.row_starts, st.lengths, tables, D ** -0.5)
        got = _lib.attention_quantized(q, H, Hkv, D, pool, st.row_starts, st.lengths, tables, D ** -0.5, bits=bits)
        ln, nf = st.lengths, st.n_free
        # |v| <= 4.5 at these sizes: the roundings of both outputs, both weights and the value, 5 of
        # 2^-8; a score differs by the key's, e <= 2^-8 sum |q k| / sqrt(128) <= 2^-8 * 12 here, 2 e
        assert (got.double() - want.double()).abs().max() <= (5 + 24) * 2.0 ** -8 * 4.5
        assert torch.nn.functional.cosine_similarity(got.double(), want.double()).min() > 0.9999


def test_a_stored_value_is_the_quantizers(device):
    """quant_util's float64 values are the ones read back, up to their rounding to bf16."""
    x = torch.randn((9, 2, 128), device="cuda").to(torch.bfloat16)
    for bits in BITS:
        v = stored(x, bits)[0]
        assert ((_quantized_rows(x, bits).double() - v).abs() <= 2.0 ** -8 * v.abs() + 2.0 ** -20).all()


# factors of the keys, the values, q; every how many positions they are taken (1: everywhere)
MAGNITUDES = [(1, 3000, 1, 1), (1, 1e-5, 1, 1), (1, 2.0 ** -10, 1, 1), (3000, 1, 1 / 3000, 1), (1e-6, 1, 1e6, 1), (1e20, 1, 1e-20, 1),
              (1e-9, 1e23, 1e9, 1), (1, 1, 0, 1), (1, 2000, 1, 97), (2.0 ** -6, 1e-4, 1, 3), (0, 0, 1, 50)]


@pytest.mark.parametrize("kf,vf,qf,every", MAGNITUDES)
@pytest.mark.parametrize("new,H,Hkv", [([1, 1, 1], 8, 2), ([1, 200, 130], 8, 2), ([2, 300, 1], 4, 4)])
@pytest.mark.parametrize("D,bits", [(64, 4), (128, 4), (64, 8), (128, 8)])
def test_attention_over_the_range_of_bf16(device, kf, vf, qf, every, new, H, Hkv, D, bits):
    """Keys, values and q far from 1, some positions' or all: the column tiles take blocks whose
    values fp16 cannot hold as bf16.  The bound, relative to what a row's sums are of, holds for
    either: fp16 rounds to 2^-12 of a value, and what it drops of smaller ones is below 2^-12 of
    their group's largest."""
    print(f"magnitudes {kf} {vf} {qf} every {every} new={new} D={D} bits={bits}", flush=True)
    c = QuantCache(bits, [40, 300, 9], new, 500, 64, H, Hkv, D, pad=1)
    there = ~torch.isnan(c.k[:, 0, :, 0])
    chosen = torch.arange(there.numel(), device="cuda").view(there.shape) % every == 0
    c.k *= torch.where(chosen, kf, 1.0)[:, None, :, None].to(c.k.dtype)
    c.vt *= torch.where(chosen, vf, 1.0)[:, None, None, :].to(c.vt.dtype)
    c.q *= qf
    at = there.nonzero()
    write(c.pool, c.k[at[:, 0], :, at[:, 1]], c.vt[at[:, 0], :, :, at[:, 1]], at[:, 0] * c.bs + at[:, 1], bits)
    exact, bound = c.exact()
    rows = c.starts[-1]
    got = c.attend(max_new=c.max_new)[:rows].double().view(rows, H, D)
    assert torch.isfinite(got).all()
    err = (got - exact[:rows]).abs()
    assert (err <= bound[:rows] + 1e-36).all(), float((err / bound[:rows].clamp(min=1e-36)).max())


@pytest.mark.parametrize("slots", ["from 5", "every seventh missing", "any order"])
@pytest.mark.parametrize("D,bits", [(64, 4), (128, 4), (64, 8), (128, 8)])
def test_append_of_many_rows_leaves_what_few_at_a_time_do(device, D, bits, slots):
    """Runs of slots that begin and break anywhere, rows that are left out among them: the same
    bytes as row by row, and no others touched."""
    H, Hkv, n, nb, bs = 4, 2, 600, 12, 64
    g = torch.Generator(device="cuda")
    g.manual_seed(D + bits)
    at = {"from 5": torch.arange(5, 5 + n), "every seventh missing": torch.arange(nb * bs)[torch.arange(nb * bs) % 7 != 3][:n],
          "any order": torch.randperm(nb * bs, generator=torch.Generator().manual_seed(1))[:n]}[slots].to("cuda", torch.int32)
    at[17::40] = -1
    qkv = torch.randn((n, (H + 2 * Hkv) * D), generator=g, device="cuda").bfloat16()
    angles = torch.rand((50, D // 2), generator=g, device="cuda") * 6
    cos, sin = angles.cos().contiguous(), angles.sin().contiguous()
    pos = torch.arange(n, device="cuda", dtype=torch.int32) % 50
    shape = _lib.quantized_pool_shape(nb, Hkv, bs, D, bits)
    one, few = (torch.full(shape, 0xA5, dtype=torch.uint8, device="cuda") for _ in range(2))
    q = _lib.rope_append_quantized(qkv, H, Hkv, D, cos, sin, one, at, pos, bits=bits, out=torch.zeros((n, H * D), device="cuda").bfloat16())
    for i in range(0, n, 1 if slots == "any order" else 3):
        rows = slice(i, i + (1 if slots == "any order" else 3))
        part = _lib.rope_append_quantized(qkv[rows], H, Hkv, D, cos, sin, few, at[rows], pos[rows], bits=bits,
                                          out=torch.zeros((qkv[rows].shape[0], H * D), device="cuda").bfloat16())
        assert torch.equal(part, q[rows])
    assert torch.equal(one, few)


@pytest.mark.parametrize("held,new,prefix,bs,H,Hkv,D", [
    ([0], [24], 0, 64, 32, 8, 128), ([0], [64], 0, 16, 32, 8, 64), ([100, 0], [100, 1], 0, 64, 8, 2, 128),
    ([3, 0, 70, 500, 9], [40, 30, 1, 1, 0], 200, 32, 8, 1, 64), ([0, 10], [300, 90], 1000, 64, 8, 8, 128),
    ([0], [2049], 0, 64, 32, 8, 64),
])
@pytest.mark.parametrize("bits", BITS)
def test_attention_is_by_the_positions_held_not_by_the_tables_room(device, held, new, prefix, bs, H, Hkv, D, bits):
    """Many rows behind tables with room for 131072 positions: the bits of tables that end with the
    sequences, and no more of the workspace written than those need at all."""
    print(f"room {bits} bits {held} + {new} prefix={prefix} bs={bs} H={H} Hkv={Hkv} D={D}", flush=True)
    tight = QuantCache(bits, held, new, prefix, bs, H, Hkv, D, pad=2)
    want = tight.attend(out=torch.full_like(tight.q, 5.0))
    if tight.N < 1000:
        assert_attention(want, *tight.exact(), tight.starts[-1])
    most = tight.workspace_bytes(tight.N)
    wide = QuantCache(bits, held, new, prefix, bs, H, Hkv, D, pad=2, width=131072 // bs)
    assert torch.equal(wide.pool, tight.pool)
    if prefix:
        wide.prefix_table = torch.cat([wide.prefix_table, wide.prefix_table.new_full((100,), -3)])
    need = wide.workspace_bytes(wide.N)
    ws = torch.full((need,), 77, dtype=torch.uint8, device="cuda")
    got = wide.attend(out=torch.full_like(wide.q, 5.0), workspace=ws)
    assert torch.equal(got, want)
    assert int((ws != 77).sum()) <= most


# A rounding to bf16 of numbers spread over their range is 0.00166 of them (rms: half a step is 2^-8 at
# most, evenly spread within it, over numbers evenly spread within a factor of two).
ONE_ROUNDING = 0.00166


def _norm_off(got, exact, rows):
    got, exact = got[:rows].double().view(rows, *exact.shape[1:]), exact[:rows]
    return float((got - exact).norm() / exact.norm())


@pytest.mark.parametrize("held,new,prefix,H,Hkv", [([40, 300], [200, 130], 500, 8, 2), ([1000], [64], 0, 32, 8),
                                                   ([9, 0, 500], [70, 300, 90], 2100, 8, 1)])
@pytest.mark.parametrize("D,bits", [(64, 4), (128, 4), (64, 8), (128, 8)])
def test_column_tiles_keep_eleven_bits(device, held, new, prefix, H, Hkv, D, bits):
    """Many rows, keys, values and q of about 1: the output's own rounding and fp16's, an eighth of it,
    of keys, weights and values (with the scores' spread of 1: 0.0017 together).  One more rounding to
    8 bits makes it 0.0023 (bf16 values and weights 0.0033)."""
    c = QuantCache(bits, held, new, prefix, 64, H, Hkv, D)
    off = _norm_off(c.attend(max_new=c.max_new), c.exact()[0], c.starts[-1])
    assert off <= 1.2 * ONE_ROUNDING, off


@pytest.mark.parametrize("held,new,prefix,H,Hkv", [([300, 900, 77], [1, 1, 2], 0, 8, 2), ([700], [1], 600, 32, 8),
                                                   ([80, 200, 900], [5, 3, 8], 0, 8, 1), ([400, 90], [16, 9], 0, 4, 2)])
@pytest.mark.parametrize("D,bits", [(64, 4), (128, 4), (64, 8), (128, 8)])
def test_lines_round_the_weights_alone(device, held, new, prefix, H, Hkv, D, bits):
    """Few rows: the output's rounding and that of the weights, which meet values taken about the
    middle code (their squares 1.11 times the values': half a step of 0.3 and the range's middle, 0.3
    beside 0): 0.0024 together, one more of either 0.0029."""
    c = QuantCache(bits, held, new, prefix, 64, H, Hkv, D)
    off = _norm_off(c.attend(max_new=c.max_new), c.exact()[0], c.starts[-1])
    assert off <= 1.6 * ONE_ROUNDING, off


@pytest.mark.parametrize("D", [64, 128])
def test_column_tiles_of_groups_whose_scale_fp16_cannot_hold(device, D):
    """Keys of 8 bits in groups from 2^-11 to 2^-11 + 15 / 2^18, either sign: scales of 2^-22.1, of which
    fp16 (at 32 times them) drops up to 2^-30, 255 times as much of a key, below 2^-11 of the group's
    largest.  Scores of q about 2^12: 0.0006 off by the keys' rounding to 11 bits and by what is
    dropped; the output's rounding is 0.00166.  Keys rounded to bf16 would move scores by 0.0045."""
    c = QuantCache(8, [40, 300], [200, 130], 500, 64, 8, 2, D)
    there = ~torch.isnan(c.k[:, 0, :, 0])
    g = torch.Generator(device="cuda")
    g.manual_seed(D)
    nb, Hkv, bs = c.k.shape[:3]
    j = torch.randint(0, 16, c.k.shape, generator=g, device="cuda").view(nb, Hkv, bs, D // 64, 64)
    j[..., 0], j[..., 1] = 0, 15
    sign = torch.randint(0, 2, j.shape[:-1], generator=g, device="cuda")[..., None] * 2 - 1
    k = (sign * (2.0 ** -11 + j * 2.0 ** -18)).view(c.k.shape)
    c.k = torch.where(there[:, None, :, None], k, float("nan")).to(torch.bfloat16)
    assert torch.equal(c.k[there[:, None].expand(nb, Hkv, bs)].double(), k[there[:, None].expand(nb, Hkv, bs)].double())
    c.q *= 4096
    at = there.nonzero()
    write(c.pool, c.k[at[:, 0], :, at[:, 1]], c.vt[at[:, 0], :, :, at[:, 1]], at[:, 0] * bs + at[:, 1], 8)
    scales = stored(c.k[at[:, 0], :, at[:, 1]], 8)[1].abs()
    assert 2.0 ** -23 < scales.min() and scales.max() < 2.0 ** -22
    off = _norm_off(c.attend(max_new=c.max_new), c.exact()[0], c.starts[-1])
    assert off <= 1.2 * ONE_ROUNDING, off


@pytest.mark.parametrize("H,Hkv,D,bits", [(32, 8, 128, 4), (8, 1, 64, 8)])
def test_captured_prompts_of_growing_lengths(device, H, Hkv, D, bits):
    """Attention of many rows in a graph, tables with room for more than they hold: replayed as the
    lengths grow from one key block to hundreds, and as rows go from one sequence to another, bit for
    bit the eager call, two graphs over one workspace in turn."""
    bs, N = 64, 60
    c = QuantCache(bits, [20000 - 30, 700, 90], [30, 18, 12], 0, bs, H, Hkv, D, width=40000 // bs)
    need = c.workspace_bytes(N)
    ws, out = torch.empty(need, dtype=torch.uint8, device="cuda"), torch.empty_like(c.q)
    steps = [([0, 30, 48, 60], [30, 18, 12]), ([0, 30, 48, 60], [9000, 700, 12]), ([0, 30, 48, 60], [20000, 718, 102]),
             ([0, 1, 2, 60], [20000, 718, 64]), ([0, 0, 0, 60], [20000, 718, 102]), ([0, 60, 60, 60], [4000, 0, 5])]
    want = []
    for starts, lengths in steps:
        c.row_starts.copy_(i32(starts))
        c.lens.copy_(i32(lengths))
        want.append(c.attend(max_new=N).clone())
    graphs = []
    for _ in range(2):
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            c.attend(max_new=N, out=out, workspace=ws)
        graphs.append(gr)
    for i in range(2 * len(steps)):
        starts, lengths = steps[i % len(steps)]
        c.row_starts.copy_(i32(starts))
        c.lens.copy_(i32(lengths))
        out.fill_(5.0)
        ws.fill_(255)
        graphs[i % 2 if i < len(steps) else 1 - i % 2].replay()
        assert torch.equal(out, want[i % len(steps)]), i


@pytest.mark.parametrize("held,new,prefix,bs,H,Hkv,D", [
    ([100, 3000, 0], [1, 1, 1], 700, 64, 32, 8, 128), ([5000], [1], 0, 16, 8, 1, 64), ([40], [2], 900, 32, 32, 8, 128),
    ([(37 * i) % 900 for i in range(64)], [1] * 64, 5000, 64, 32, 8, 128), ([10, 600], [5, 8], 0, 64, 8, 1, 64),
    ([(61 * i) % 400 for i in range(200)], [1, 0, 2, 1] * 50, 90, 16, 32, 4, 64),
])
@pytest.mark.parametrize("bits", BITS)
def test_attention_of_few_rows_in_roomy_tables(device, held, new, prefix, bs, H, Hkv, D, bits):
    """Few rows a sequence: the same bits from tables that end with the sequences and from ones with
    room for 40000 positions, the prefix's too."""
    tight = QuantCache(bits, held, new, prefix, bs, H, Hkv, D, pad=1)
    want = tight.attend(max_new=tight.max_new, out=torch.full_like(tight.q, 5.0))
    wide = QuantCache(bits, held, new, prefix, bs, H, Hkv, D, pad=1, width=40000 // bs)
    if prefix:
        wide.prefix_table = torch.cat([wide.prefix_table, wide.prefix_table.new_full((500,), -3)])
    assert torch.equal(wide.attend(max_new=wide.max_new, out=torch.full_like(wide.q, 5.0)), want)


@pytest.mark.parametrize("D,bits", [(64, 8), (128, 4)])
def test_attention_of_prompts_among_the_most_sequences(device, D, bits):
    """2048 sequences, three of them with many rows, the last among them, in tables with room to spare:
    every sequence's length counts for the cut, wherever it is."""
    R = _lib.SHARED_MAX_SEQUENCES
    held, new = [(11 * i) % 70 if i % 5 else 0 for i in range(R)], [i % 2 for i in range(R)]
    held[70], new[70], new[1000], held[-1], new[-1] = 5, 90, 70, 1500, 40
    c = QuantCache(bits, held, new, 90, 64, 4, 2, D, pad=1, width=200)
    exact, bound = c.exact()
    got = c.attend(max_new=c.max_new, out=torch.full_like(c.q, 5.0))
    assert_attention(got, exact, bound, c.starts[-1])
    assert (got[c.starts[-1]:] == 5).all()
