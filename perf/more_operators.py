"""Measured calls of a key/value cache held in 4 or 8 bits, in blocks, behind a shared prefix.

Three operators and the calls a serving loop makes of them:

* ``append``: rotary embedding of a step's q and k rows, keys and values quantized in groups
  of 64 dims (the affine rule of the quantized weights) into the cache's blocks; the pass
  returns the rotated q and the values that the rows' codes stand for, read back;
* ``attend``: attention of a step's rows over the shared prefix and their own sequence;
* ``read``: the keys and values of some positions, as bfloat16.

Head layouts are those of the TinyLlama, Llama-3-8B and Llama-3-70B rank-0-of-8
configurations.  Lengths of a case follow from its numbers alone (a low-discrepancy
sequence between the case's bounds); values, block numbers and orders come from the seed.
"""
import math

import torch

own = False

GROUP = 64

# q heads, kv heads, head_dim, rotary base of one rank's share
HEADS = {
    "tinyllama": dict(H=32, Hkv=4, D=64, base=10000.0),
    "llama3-8b": dict(H=32, Hkv=8, D=128, base=500000.0),
    "llama3-70b/8": dict(H=8, Hkv=1, D=128, base=500000.0),
}


def _case(held, new, **rest):
    """A case whose sequences hold held[0] to held[1] positions and get new[0] to new[1]."""
    return dict(rest, held_min=held[0], held_max=held[1], new_min=new[0], new_max=new[1])


def listed():
    return [
        # the append of a 64-sequence decode step: latency
        _case(name="append_8b_decode64_4bit", kind="append", shape="llama3-8b", bits=4, R=64, held=(0, 1500), new=(1, 1),
              bs=64, prefix=2048, pad=0),
        # 24 ragged prompts of a serving step on TinyLlama's heads
        _case(name="append_tiny_24_prompts_4bit", kind="append", shape="tinyllama", bits=4, R=24, held=(0, 333),
              new=(1, 700), bs=32, prefix=333, pad=5),
        # long prompts taken in by the 70B shard
        _case(name="append_70b_8_prompts_8bit", kind="append", shape="llama3-70b/8", bits=8, R=8, held=(0, 0),
              new=(1500, 4100), bs=128, prefix=0, pad=0),
        # the smallest attention: one sequence's token behind a short prefix
        _case(name="attend_tiny_1_decode_4bit", kind="attend", shape="tinyllama", bits=4, R=1, held=(100, 100), new=(1, 1),
              bs=16, prefix=500, pad=0),
        # one user's session of 128 K positions, which is what a cache in 4 bits is kept for
        _case(name="attend_8b_1_session_4bit", kind="attend", shape="llama3-8b", bits=4, R=1, held=(131071, 131071),
              new=(1, 1), bs=256, prefix=0, pad=0),
        # 64 sequences sampled behind an 8192-token prefix
        _case(name="attend_8b_64_decode_4bit", kind="attend", shape="llama3-8b", bits=4, R=64, held=(0, 1023), new=(1, 1),
              bs=64, prefix=8192, pad=0),
        # 256 sequences of the 70B shard's heads, own parts as long as the prefix
        _case(name="attend_70b_256_decode_8bit", kind="attend", shape="llama3-70b/8", bits=8, R=256, held=(200, 4000),
              new=(1, 1), bs=128, prefix=2000, pad=0),
        # 24 sequences checking 5 guessed tokens each, odd lengths, small blocks
        _case(name="attend_tiny_24_guess_8bit", kind="attend", shape="tinyllama", bits=8, R=24, held=(3, 901), new=(5, 5),
              bs=16, prefix=1777, pad=3),
        # the questions of 16 ragged requests taken in behind a 4096-token prefix
        _case(name="attend_8b_16_prompts_4bit", kind="attend", shape="llama3-8b", bits=4, R=16, held=(0, 0),
              new=(24, 1000), bs=64, prefix=4096, pad=0),
        # no prefix: a 2048-token prompt taken in beside 31 sequences that decode
        _case(name="attend_8b_mixed_8bit", kind="attend", shape="llama3-8b", bits=8, R=32, held=(0, 1200), new=(1, 1),
              first=2048, bs=64, prefix=0, pad=0),
        # a long sequence handed on to another process
        _case(name="read_8b_long_4bit", kind="read", shape="llama3-8b", bits=4, R=1, held=(40000, 40000), new=(1, 1),
              bs=64, prefix=0, pad=0),
        # a ragged batch's keys and values, padded rows among them
        _case(name="read_tiny_32_ragged_8bit", kind="read", shape="tinyllama", bits=8, R=32, held=(0, 900), new=(1, 1),
              bs=16, prefix=0, pad=40),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "read"])
    bs, bits, shape = rng.choice([16, 32, 64, 64, 128, 256]), rng.choice([4, 8]), rng.choice(sorted(HEADS))
    if kind == "read":
        R = _log_int(rng, 1, 64)
        held = _log_int(rng, 1, 40000 // R)
        return _case(kind=kind, shape=shape, bits=bits, R=R, held=(rng.randint(0, held), held), new=(1, 1), bs=bs,
                     prefix=0, pad=rng.choice([0, rng.randint(1, 50)]))
    prompts = rng.random() < 0.5
    if kind == "append":
        R = _log_int(rng, 1, 12) if prompts else _log_int(rng, 1, 256)
        top = _log_int(rng, 2, 1500) if prompts else 1
        held = _log_int(rng, 1, 1000)
        return _case(kind=kind, shape=shape, bits=bits, R=R, held=(rng.randint(0, held), held),
                     new=(rng.randint(1, top), top), bs=bs, prefix=rng.choice([0, _log_int(rng, 1, 8000)]),
                     pad=rng.choice([0, rng.randint(1, 33)]))
    if prompts:
        R, top = _log_int(rng, 1, 10), _log_int(rng, 2, 700)
        held, prefix = _log_int(rng, 1, 800), _log_int(rng, 1, 3500)
    else:
        R, top = _log_int(rng, 1, 200), rng.choice([1, 1, 1, rng.randint(2, 8)])
        held, prefix = _log_int(rng, 1, min(100000, 200000 // R)), _log_int(rng, 16, 200000 // max(16, R))
    # a step in which some sequences wait has rows of the others only
    fewest = 0 if R >= 4 and rng.random() < 0.3 else rng.randint(1, top)
    return _case(kind=kind, shape=shape, bits=bits, R=R, held=(rng.randint(0, held), held), new=(fewest, top), bs=bs,
                 prefix=rng.choice([0, prefix, prefix, prefix]), pad=rng.choice([0, 0, rng.randint(1, 9)]))


# ---------------------------------------------------------------- inputs


def _spread(n, lo, hi, turn):
    """n whole numbers between the bounds, both included, spread evenly in a scrambled order."""
    return [lo + int((hi - lo + 1) * ((turn + i * 0.6180339887498949) % 1.0)) for i in range(n)]


def _lengths(case):
    """(positions held before the step, new positions) of every sequence."""
    held = _spread(case["R"], case["held_min"], case["held_max"], 0.13)
    new = _spread(case["R"], case["new_min"], case["new_max"], 0.57)
    if "first" in case:
        held[0], new[0] = 0, case["first"]
    return held, new


def _blocks(n, bs):
    return (n + bs - 1) // bs


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)


def _i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def _inputs(case, seed):
    """What both forms start from.  ``k`` and ``v``: the keys and values of every slot of the
    pool before they are quantized, [slots, kv heads, head_dim]."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind, bs, R, prefix = case["kind"], case["bs"], case["R"], case["prefix"]
    H, Hkv, D, base = (HEADS[case["shape"]][k] for k in ("H", "Hkv", "D", "base"))
    held, new = _lengths(case)
    after = [h + w for h, w in zip(held, new)]
    n = sum(after) if kind == "read" else sum(new)
    st = dict(kind=kind, bits=case["bits"], bs=bs, H=H, Hkv=Hkv, D=D, n=n, rows=n + case["pad"], prefix=prefix,
              max_new=max(new), scale=1.0 / math.sqrt(D), plan=list(zip(held, new)))
    # the blocks of the sequences and of the prefix, in random order
    counts = [_blocks(a, bs) for a in after] + [_blocks(prefix, bs)]
    st["blocks"] = sum(counts) + 3
    order = torch.randperm(st["blocks"], generator=g, device="cuda").to(torch.int32)
    tables = torch.zeros((R + 1, max(counts)), dtype=torch.int32, device="cuda")
    tables[torch.arange(max(counts), device="cuda")[None] < _i32(counts)[:, None]] = order[:sum(counts)]
    st["tables"] = tables[:R, :max(counts[:R])].contiguous()
    st["prefix_table"] = tables[R, :counts[R]].contiguous() if prefix else None
    # every slot holds something: whole blocks are handed out again without being cleared.  Some
    # channels of the keys are larger than others
    channel = torch.exp(0.5 * torch.randn((Hkv, D), generator=g, device="cuda"))
    st["k"] = (torch.randn((st["blocks"] * bs, Hkv, D), generator=g, device="cuda") * channel).to(torch.bfloat16)
    st["v"] = _randn(g, st["blocks"] * bs, Hkv, D)
    first = [0] * R if kind == "read" else held
    pos = torch.cat([torch.arange(a, b, device="cuda") for a, b in zip(first, after)])
    seq = torch.repeat_interleave(torch.arange(R, device="cuda"), _i32([b - a for a, b in zip(first, after)]))
    slots = torch.full((st["rows"],), -1, dtype=torch.int32, device="cuda")
    positions = slots.clone()
    slots[:n] = st["tables"][seq, pos // bs] * bs + (pos % bs).to(torch.int32)
    positions[:n] = (prefix + pos).to(torch.int32)
    st["slots"], st["positions"] = slots, positions
    if kind == "append":
        st["qkv"] = _randn(g, st["rows"], (H + 2 * Hkv) * D)
        ang = (torch.arange(prefix + max(after), dtype=torch.float64, device="cuda")[:, None]
               * base ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)[None])
        st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
        st["q"] = torch.zeros((st["rows"], H * D), dtype=torch.bfloat16, device="cuda")
    if kind == "attend":
        st["q"] = _randn(g, st["rows"], H * D)
        st["out"] = torch.zeros_like(st["q"])
        st["row_starts"], st["lengths"] = _i32([sum(new[:i]) for i in range(R + 1)]), _i32(after)
        st["prefix_len"] = _i32([prefix])
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    k, v = st.pop("k"), st.pop("v")
    if own:
        from shardcompute_amd import _lib
        # the cache's own layout, filled as a program fills it (rotated by no angle)
        Hkv, D = st["Hkv"], st["D"]
        st["pool"] = _lib.quantized_pool(st["blocks"], Hkv, st["bs"], D, bits=st["bits"], device=torch.device("cuda"))
        rows = torch.cat([torch.zeros_like(k), k, v], 1).view(k.shape[0], 3 * Hkv * D)
        one = torch.ones((1, D // 2), device="cuda")
        _lib.rope_append_quantized(rows, Hkv, Hkv, D, one, torch.zeros_like(one), st["pool"],
                                   torch.arange(k.shape[0], dtype=torch.int32, device="cuda"),
                                   torch.zeros(k.shape[0], dtype=torch.int32, device="cuda"), bits=st["bits"])
        if st["kind"] == "attend":
            need = _lib.attention_quantized_workspace_bytes(
                st["rows"], case["R"], st["H"], Hkv, D, st["tables"].shape[1] * st["bs"],
                0 if st["prefix_table"] is None else st["prefix_table"].numel() * st["bs"], st["max_new"],
                bits=st["bits"])
            st["workspace"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    else:
        st["kq"], st["vq"] = _quantize(k, st["bits"]), _quantize(v, st["bits"])
    return st


# ---------------------------------------------------------------- the calls


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(st):
    from shardcompute_amd import _lib
    H, Hkv, D, bits, pool = st["H"], st["Hkv"], st["D"], st["bits"], st["pool"]
    if st["kind"] == "append":
        q = _lib.rope_append_quantized(st["qkv"], H, Hkv, D, st["cos"], st["sin"], pool, st["slots"], st["positions"],
                                       bits=bits, out=st["q"])
        return q, *_lib.read_quantized(pool, Hkv, D, st["slots"], bits=bits)
    if st["kind"] == "read":
        return _lib.read_quantized(pool, Hkv, D, st["slots"], bits=bits)
    return _lib.attention_quantized(st["q"], H, Hkv, D, pool, st["row_starts"], st["lengths"], st["tables"], st["scale"],
                                    bits=bits, prefix_table=st["prefix_table"], prefix_len=st["prefix_len"],
                                    max_new=st["max_new"], out=st["out"], workspace=st["workspace"])


def _run_plain(st):
    return {"append": _plain_append, "read": _plain_read, "attend": _plain_attend}[st["kind"]](st)


def _quantize(x, bits):
    """(codes, scales, biases) of x [rows, heads, head_dim], a scale and a bias per 64 dims.  The
    rule says in which order its quotients are taken and rounded, in 32 bits: values of bfloat16
    often lie right on the border of two codes."""
    n = 2 ** bits - 1
    g = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    down = lo.abs() > hi.abs()
    # (a quotient by a plain number would be a product with its reciprocal)
    scale = ((hi - lo) / torch.full_like(hi, n)).clamp(min=1e-7)
    scale = torch.where(down, scale, -scale)
    edge = torch.where(down, lo, hi)
    q0 = torch.round(edge / scale)
    scale = torch.where(q0 != 0, edge / q0, scale)
    bias = torch.where(q0 != 0, edge, 0.0)
    codes = torch.round((g - bias) / scale).clamp(0, n).to(torch.uint8)
    return codes, scale.to(torch.bfloat16), bias.to(torch.bfloat16)


def _values(held, slots):
    """What the codes at these slots stand for, in 32 bits: [.., heads, head_dim]."""
    codes, scale, bias = (t[slots] for t in held)
    return (scale.float() * codes.float() + bias.float()).flatten(-2)


def _plain_append(st):
    H, Hkv, D, n = st["H"], st["Hkv"], st["D"], st["n"]
    x = st["qkv"][:n].float().view(n, H + 2 * Hkv, D)
    pos, slot = st["positions"][:n].long(), st["slots"][:n].long()
    c, s = st["cos"][pos][:, None], st["sin"][pos][:, None]
    x1, x2 = x[:, :H + Hkv, :D // 2], x[:, :H + Hkv, D // 2:]
    rot = torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], -1).to(torch.bfloat16)
    st["q"][:n] = rot[:, :H].reshape(n, H * D)
    for held, rows in ((st["kq"], rot[:, H:]), (st["vq"], x[:, H + Hkv:])):
        for all_slots, fresh in zip(held, _quantize(rows, st["bits"])):
            all_slots[slot] = fresh
    return st["q"], *_plain_read(st)


def _plain_read(st):
    there = (st["slots"] >= 0)[:, None, None]
    slot = st["slots"].long().clamp(min=0)
    return tuple(torch.where(there, _values(st[name], slot), 0.0).to(torch.bfloat16) for name in ("kq", "vq"))


def _slots_of(table, length, bs):
    p = torch.arange(length, device=table.device)
    return table.long()[p // bs] * bs + p % bs


def _plain_attend(st):
    H, Hkv, D, P, bs = st["H"], st["Hkv"], st["D"], st["prefix"], st["bs"]
    G, out, at = H // Hkv, st["out"], 0
    before = _slots_of(st["prefix_table"], P, bs) if P else torch.zeros(0, dtype=torch.int64, device=out.device)
    kp, vp = _values(st["kq"], before), _values(st["vq"], before)
    for r, (held, new) in enumerate(st["plan"]):
        if not new:
            continue
        mine = _slots_of(st["tables"][r], held + new, bs)
        k = torch.cat([kp, _values(st["kq"], mine)]).permute(1, 2, 0).contiguous()
        v = torch.cat([vp, _values(st["vq"], mine)]).transpose(0, 1).contiguous()
        last = P + held + torch.arange(new, device=k.device)
        hidden = torch.arange(v.shape[1], device=k.device)[None] > last[:, None]
        q = st["q"][at:at + new].float().view(new, Hkv, G, D).transpose(0, 1).reshape(Hkv, new * G, D)
        s = torch.bmm(q, k) * st["scale"]
        s.view(Hkv, new, G, -1).masked_fill_(hidden[:, None], -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.bmm(p, v) / p.sum(-1, keepdim=True)
        out[at:at + new] = o.view(Hkv, new, G, D).transpose(0, 1).reshape(new, H * D).to(torch.bfloat16)
        at += new
    return out


# ---------------------------------------------------------------- work


def work(case):
    held, new = _lengths(case)
    c, P = HEADS[case["shape"]], case["prefix"]
    H, Hkv, D = c["H"], c["Hkv"], c["D"]
    n = sum(new)
    position = Hkv * (2 * D * case["bits"] // 8 + 2 * D // GROUP * 4)        # bytes of one in the cache
    if case["kind"] == "append":
        angles = len({p for h, w in zip(held, new) for p in range(h, h + w)})
        return dict(bytes=4 * n * H * D + 8 * n * Hkv * D + n * position + 4 * angles * D + 8 * n,
                    flops=3 * n * (H + Hkv) * D + 8 * n * Hkv * D)
    if case["kind"] == "read":
        n = sum(held) + n
        return dict(bytes=n * (position + 4 * Hkv * D) + 4 * n, flops=4 * n * Hkv * D)
    keys = P + sum(h + w for h, w in zip(held, new) if w)
    pairs = sum(w * (P + h) + w * (w + 1) // 2 for h, w in zip(held, new))
    return dict(bytes=4 * n * H * D + keys * position, flops=4 * H * D * pairs)


# ---------------------------------------------------------------- 64 bits


def exact(case, seed):
    st = _inputs(case, seed)
    return {"append": _exact_append, "read": _exact_read, "attend": _exact_attend}[case["kind"]](case, st)


def _r32(x):
    """Rounded to 32 bits, where the operator's definition says so."""
    return x.to(torch.float32).double()


def _exact_stored(rows, bits):
    """The values a cache of ``bits`` bits holds for rows of bfloat16 [.., head_dim]."""
    top = (1 << bits) - 1
    out = torch.empty(rows.shape, dtype=torch.float64, device=rows.device)
    for d in range(0, rows.shape[-1], GROUP):
        x = rows[..., d:d + GROUP].double()
        most, least = x.max(-1).values, x.min(-1).values
        step = torch.maximum(_r32(_r32(most - least) / top), _r32(torch.tensor(1e-7, device=x.device)))
        from_least = least.abs() > most.abs()
        step[~from_least] *= -1
        anchor = most.clone()
        anchor[from_least] = least[from_least]
        turns = torch.round(_r32(anchor / step))
        some = turns != 0
        step[some] = _r32(anchor[some] / turns[some])
        anchor[~some] = 0
        code = torch.round(_r32(_r32(x - anchor[..., None]) / step[..., None])).clamp(0, top)
        step, anchor = step.to(torch.bfloat16).double(), anchor.to(torch.bfloat16).double()
        out[..., d:d + GROUP] = anchor[..., None] + code * step[..., None]
    return out


def _exact_append(case, st):
    H, Hkv, D = st["H"], st["Hkv"], st["D"]
    N, n = st["rows"], st["n"]
    x = st["qkv"].double().view(N, H + 2 * Hkv, D)
    pos = st["positions"].long().clamp(min=0)
    c, s = (st[name].double()[pos][:, None].repeat(1, 1, 2) for name in ("cos", "sin"))
    s[..., :D // 2] *= -1
    across = x.roll(D // 2, -1)
    q = x[:, :H] * c + across[:, :H] * s
    # the keys are rotated in 32 bits and rounded to bfloat16 before they are quantized
    k = (_r32(x[:, H:H + Hkv] * c) + _r32(across[:, H:H + Hkv] * s)).to(torch.float32).to(torch.bfloat16)
    k, v = _exact_stored(k, case["bits"]), _exact_stored(st["qkv"].view(N, -1, D)[:, H + Hkv:], case["bits"])
    q[n:], k[n:], v[n:] = 0, 0, 0
    return q.reshape(N, H * D), k, v


def _exact_read(case, st):
    at = st["slots"].long()
    k, v = (_exact_stored(st[name][at.clamp(min=0)], case["bits"]) for name in ("k", "v"))
    k[at < 0], v[at < 0] = 0, 0
    return k, v


def _exact_attend(case, st):
    H, Hkv, D, bs, P = st["H"], st["Hkv"], st["D"], st["bs"], case["prefix"]
    held, new = _lengths(case)
    out = st["out"].double()
    at = 0
    for r in range(case["R"]):
        if new[r] == 0:
            continue
        places = ([] if P == 0 else [int(b) * bs + j for b in st["prefix_table"].tolist() for j in range(bs)][:P])
        mine = st["tables"][r].tolist()
        places += [mine[p // bs] * bs + p % bs for p in range(held[r] + new[r])]
        there = torch.tensor(places, device="cuda")
        k, v = _exact_stored(st["k"][there], case["bits"]), _exact_stored(st["v"][there], case["bits"])
        keys = torch.arange(len(places), device="cuda")
        step = max(1, (1 << 26) // (len(places) * (H // Hkv)))                     # rows at a time
        for i in range(0, new[r], step):
            rows = torch.arange(i, min(i + step, new[r]), device="cuda")
            seen = keys[None] <= (P + held[r] + rows)[:, None]
            q = st["q"][at + rows].double().view(len(rows), H, D)
            for h in range(H):
                s = q[:, h] @ k[:, h * Hkv // H].T * st["scale"]
                p = torch.softmax(torch.where(seen, s, -math.inf), -1)
                out[at + rows, h * D:(h + 1) * D] = p @ v[:, h * Hkv // H]
        at += new[r]
    return out
