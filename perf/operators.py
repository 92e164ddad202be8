"""Measured calls of the key/value cache in blocks: a ragged batch behind one shared prefix.

Three operators and the calls a serving loop makes of them:

* ``step``: the block tables, row starts, slots and positions of one model step, from the
  sequences' lengths and their new positions;
* ``append``: rotary embedding of a step's q and k rows, keys and values into the cache's
  blocks through the slots;
* ``attend``: attention of a step's rows over the shared prefix and their own sequence.

Head layouts are those of the TinyLlama, Llama-3-8B and Llama-3-70B rank-0-of-8
configurations.  Lengths of a case follow from its numbers alone (a low-discrepancy
sequence between the case's bounds); values, block numbers and orders come from the seed.
"""
import math

import torch

own = False

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
        # one sequence's decode step: launch and host latency
        _case(name="step_1_decode", kind="step", R=1, held=(700, 700), new=(1, 1), bs=64, prefix=512, freed=0, pad=0),
        # a decode step of 256 sequences, every eighth of which has ended and starts anew
        _case(name="step_256_decode", kind="step", R=256, held=(1, 2000), new=(1, 1), bs=64, prefix=4096, freed=8,
              pad=0),
        # 512 prompts of up to 700 tokens taken in at once, rows padded to the step's width
        _case(name="step_512_prompts", kind="step", R=512, held=(0, 0), new=(0, 700), bs=16, prefix=1000, freed=0,
              pad=77),
        # the append of a 64-sequence decode step
        _case(name="append_8b_decode64", kind="append", shape="llama3-8b", R=64, held=(0, 1500), new=(1, 1), bs=64,
              prefix=2048, pad=0),
        # 24 ragged prompts of a serving step on TinyLlama's heads
        _case(name="append_tiny_24_prompts", kind="append", shape="tinyllama", R=24, held=(0, 333), new=(1, 700), bs=32,
              prefix=333, pad=5),
        # the smallest attention: one sequence's token behind a short prefix
        _case(name="attend_tiny_1_decode", kind="attend", shape="tinyllama", R=1, held=(100, 100), new=(1, 1), bs=16,
              prefix=500, pad=0),
        # 64 sequences sampled behind an 8192-token prefix
        _case(name="attend_8b_64_decode", kind="attend", shape="llama3-8b", R=64, held=(0, 1023), new=(1, 1), bs=64,
              prefix=8192, pad=0),
        # 256 sequences of the 70B shard's heads, own parts as long as the prefix
        _case(name="attend_70b_256_decode", kind="attend", shape="llama3-70b/8", R=256, held=(200, 4000), new=(1, 1),
              bs=128, prefix=2000, pad=0),
        # a long document asked 16 questions at once
        _case(name="attend_8b_16_long", kind="attend", shape="llama3-8b", R=16, held=(10, 300), new=(1, 1), bs=64,
              prefix=65536, pad=0),
        # 24 sequences checking 5 guessed tokens each, odd lengths, small blocks
        _case(name="attend_tiny_24_guess", kind="attend", shape="tinyllama", R=24, held=(3, 901), new=(5, 5), bs=16,
              prefix=1777, pad=3),
        # the questions of 16 ragged requests taken in behind a 4096-token prefix
        _case(name="attend_8b_16_prompts", kind="attend", shape="llama3-8b", R=16, held=(0, 0), new=(24, 1000), bs=64,
              prefix=4096, pad=0),
        # no prefix: a 2048-token prompt taken in beside 31 sequences that decode
        _case(name="attend_8b_mixed", kind="attend", shape="llama3-8b", R=32, held=(0, 1200), new=(1, 1), first=2048,
              bs=64, prefix=0, pad=0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["step", "append", "attend", "attend", "attend"])
    bs = rng.choice([16, 32, 64, 64, 128, 256])
    if kind == "step":
        R = _log_int(rng, 1, 512)
        prompts = rng.random() < 0.4
        top = _log_int(rng, 1, 350) if prompts else 1
        held = _log_int(rng, 1, 2000)
        return _case(kind=kind, R=R, held=(rng.randint(0, held), held), new=(rng.randint(0, top), top), bs=bs,
                    prefix=rng.choice([0, _log_int(rng, 1, 60000)]), freed=rng.choice([0, 0, 3, 11]),
                    pad=rng.choice([0, rng.randint(1, 99)]))
    shape = rng.choice(sorted(HEADS))
    prompts = rng.random() < 0.5
    if kind == "append":
        R = _log_int(rng, 1, 12) if prompts else _log_int(rng, 1, 256)
        top = _log_int(rng, 2, 250) if prompts else 1
        held = _log_int(rng, 1, 1000)
        return _case(kind=kind, shape=shape, R=R, held=(rng.randint(0, held), held), new=(rng.randint(1, top), top),
                    bs=bs, prefix=rng.choice([0, _log_int(rng, 1, 8000)]), pad=rng.choice([0, rng.randint(1, 33)]))
    if prompts:
        R, top = _log_int(rng, 1, 10), _log_int(rng, 2, 700)
        held, prefix = _log_int(rng, 1, 800), _log_int(rng, 1, 3500)
    else:
        R, top = _log_int(rng, 1, 200), rng.choice([1, 1, 1, rng.randint(2, 8)])
        held, prefix = _log_int(rng, 1, min(1500, 50000 // R)), _log_int(rng, 16, 200000 // max(16, R))
    # a step in which some sequences wait has rows of the others only
    fewest = 0 if R >= 4 and rng.random() < 0.3 else rng.randint(1, top)
    return _case(kind=kind, shape=shape, R=R, held=(rng.randint(0, held), held), new=(fewest, top), bs=bs,
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


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)


def _i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def _tables(g, counts, width, spare):
    """Tables [R, width] of counts[r] distinct blocks each in random order, and the blocks left over."""
    need = sum(counts)
    order = torch.randperm(need + spare, generator=g, device="cuda").to(torch.int32)
    tables = torch.zeros((len(counts), width), dtype=torch.int32, device="cuda")
    at = torch.arange(width, device="cuda")[None] < _i32(counts)[:, None]
    tables[at] = order[:need]
    return tables, order[need:].contiguous()


def _inputs(case, seed):
    g, kind, bs, R, prefix = _gen(seed), case["kind"], case["bs"], case["R"], case["prefix"]
    held, new = _lengths(case)
    n = sum(new)
    st = dict(kind=kind, bs=bs, n=n, rows=n + case["pad"], prefix=prefix, max_new=max(new))
    if kind == "step":
        release = [case["freed"] > 0 and i % case["freed"] == 1 for i in range(R)]
        counts = [_blocks(h, bs) for h in held]
        start = [0 if f else h for h, f in zip(held, release)]
        grow = sum(_blocks(s + w, bs) - _blocks(s, bs) for s, w in zip(start, new))
        width = max(max(_blocks(s + w, bs) for s, w in zip(start, new)), max(counts)) + 2
        st["tables"], free = _tables(g, counts, width, grow + 9)
        st["free"] = torch.zeros(sum(counts) + grow + 9, dtype=torch.int32, device="cuda")
        st["free"][:free.numel()] = free
        st["n_free"] = _i32([free.numel()])
        st["lengths"], st["new"], st["prefix_len"] = _i32(held), _i32(new), _i32([prefix])
        st["release"] = torch.tensor(release, device="cuda") if case["freed"] else None
        return st
    H, Hkv, D, base = (HEADS[case["shape"]][k] for k in ("H", "Hkv", "D", "base"))
    after = [h + w for h, w in zip(held, new)]
    width = max(_blocks(a, bs) for a in after)
    counts = [_blocks(a, bs) for a in after] + [_blocks(prefix, bs)]
    tables, _ = _tables(g, counts, max(width, counts[-1]), 3)
    st.update(H=H, Hkv=Hkv, D=D, scale=1.0 / math.sqrt(D), tables=tables[:R, :width].contiguous(),
              prefix_table=tables[R, :counts[-1]].contiguous() if prefix else None)
    nb = sum(counts) + 3
    # every slot of the pool holds something: whole blocks are handed out again without being cleared
    st["k"], st["vt"] = _randn(g, nb, Hkv, bs, D), _randn(g, nb, Hkv, D, bs)
    if kind == "append":
        st["qkv"] = _randn(g, st["rows"], (H + 2 * Hkv) * D)
        ang = (torch.arange(prefix + max(after), dtype=torch.float64, device="cuda")[:, None]
               * base ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)[None])
        st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
        pos = torch.cat([torch.arange(h, a, device="cuda") for h, a in zip(held, after)])
        seq = torch.repeat_interleave(torch.arange(R, device="cuda"), torch.tensor(new, device="cuda"))
        slots = torch.full((st["rows"],), -1, dtype=torch.int32, device="cuda")
        positions = slots.clone()
        slots[:n] = st["tables"][seq, pos // bs] * bs + (pos % bs).to(torch.int32)
        positions[:n] = (prefix + pos).to(torch.int32)
        st["slots"], st["positions"] = slots, positions
        st["q"] = torch.zeros((st["rows"], H * D), dtype=torch.bfloat16, device="cuda")
        return st
    st["q"] = _randn(g, st["rows"], H * D)
    st["out"] = torch.zeros_like(st["q"])
    st["row_starts"], st["lengths"] = _i32([sum(new[:i]) for i in range(R + 1)]), _i32(after)
    st["prefix_len"] = _i32([prefix])
    st["plan"] = list(zip(held, new))
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if own:
        from shardcompute_amd import _lib
        if st["kind"] == "step":
            st["out"] = _lib.block_step_buffers(case["R"], st["rows"], torch.device("cuda"))
            # a sequence that gives its blocks back gets others in their place: a further pass
            # starts from the tables as they were
            st["before"] = None if st["release"] is None else st["tables"].clone()
        if st["kind"] == "attend":
            need = _lib.attention_shared_workspace_bytes(
                st["rows"], case["R"], st["H"], st["Hkv"], st["D"], st["tables"].shape[1] * st["bs"],
                0 if st["prefix_table"] is None else st["prefix_table"].numel() * st["bs"], st["max_new"])
            st["workspace"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    return st


# ---------------------------------------------------------------- the calls


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(st):
    from shardcompute_amd import _lib
    if st["kind"] == "step":
        if st["before"] is not None:
            st["tables"].copy_(st["before"])
        s = _lib.block_tables(st["lengths"], st["new"], st["tables"], st["free"], st["n_free"], st["bs"], st["rows"],
                              prefix_len=st["prefix_len"], release=st["release"], out=st["out"])
        return dict(lengths=s.lengths, n_free=s.n_free, row_starts=s.row_starts, slots=s.slots, positions=s.positions,
                    tables=st["tables"], free=st["free"])
    if st["kind"] == "append":
        q = _lib.rope_append_blocks(st["qkv"], st["H"], st["Hkv"], st["D"], st["cos"], st["sin"], st["k"], st["vt"],
                                    st["slots"], st["positions"], out=st["q"])
        return q, st["k"], st["vt"]
    return _lib.attention_shared(st["q"], st["H"], st["Hkv"], st["D"], st["k"], st["vt"], st["row_starts"],
                                 st["lengths"], st["tables"], st["scale"], prefix_table=st["prefix_table"],
                                 prefix_len=st["prefix_len"], max_new=st["max_new"], out=st["out"],
                                 workspace=st["workspace"])


def _run_plain(st):
    return {"step": _plain_step, "append": _plain_append, "attend": _plain_attend}[st["kind"]](st)


def _plain_step(st):
    bs, rows, tables, dev = st["bs"], st["rows"], st["tables"], st["lengths"].device
    R, P = tables.shape
    lengths, new = st["lengths"].long(), st["new"].long().clamp(min=0)
    release = torch.zeros(R, dtype=torch.bool, device=dev) if st["release"] is None else st["release"]
    old = torch.where(release, 0, lengths)
    total, have = old + new, _blocks(old, bs)
    need = _blocks(total, bs) - have
    # blocks given back, onto the stack in the order of sequence and place
    col = torch.arange(P, device=dev)
    back = (col[None] < _blocks(lengths, bs)[:, None]) & release[:, None]
    cap = st["free"].numel()
    to = torch.where(back.reshape(-1), st["n_free"].long() + back.reshape(-1).long().cumsum(0) - 1, cap)
    free = torch.cat([st["free"], st["free"].new_zeros(1)])
    free[to.clamp(max=cap)] = tables.reshape(-1)
    top = st["n_free"].long() + back.sum()
    # blocks taken, from the stack's top
    first = need.cumsum(0) - need
    i = col[None] - have[:, None]
    taken = (i >= 0) & (i < need[:, None])
    after = torch.where(taken, free[(top - 1 - first[:, None] - i).clamp(min=0, max=cap)], tables)
    starts = torch.cat([new.new_zeros(1), new.cumsum(0)])
    row = torch.arange(rows, device=dev)
    seq = torch.zeros(rows + 1, dtype=torch.int64, device=dev)
    seq = (seq.index_add(0, starts[:-1].clamp(max=rows), torch.ones_like(new)).cumsum(0) - 1)[:rows]
    pos = old[seq] + row - starts[seq]
    at = after[seq, (pos // bs).clamp(max=P - 1)].long() * bs + pos % bs
    here = row < starts[-1]
    i32 = torch.int32
    return dict(lengths=total.to(i32), n_free=(top - need.sum()).to(i32), row_starts=starts.to(i32),
                slots=torch.where(here, at, -1).to(i32),
                positions=torch.where(here, st["prefix_len"].long() + pos, -1).to(i32), tables=after, free=free[:cap])


def _plain_append(st):
    H, Hkv, D, n, bs = st["H"], st["Hkv"], st["D"], st["n"], st["bs"]
    x = st["qkv"][:n].float().view(n, H + 2 * Hkv, D)
    pos, slot = st["positions"][:n].long(), st["slots"][:n].long()
    c, s = st["cos"][pos][:, None], st["sin"][pos][:, None]
    x1, x2 = x[:, :H + Hkv, :D // 2], x[:, :H + Hkv, D // 2:]
    rot = torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], -1).to(torch.bfloat16)
    st["q"][:n] = rot[:, :H].reshape(n, H * D)
    st["k"][slot // bs, :, slot % bs] = rot[:, H:]
    st["vt"][slot // bs, :, :, slot % bs] = st["qkv"][:n].view(n, H + 2 * Hkv, D)[:, H + Hkv:]
    return st["q"], st["k"], st["vt"]


def _gathered(st, table, length):
    """keys and values [Hkv, length, D] of the first positions of a table."""
    nb = _blocks(length, st["bs"])
    k = st["k"][table[:nb].long()].transpose(0, 1).reshape(st["Hkv"], nb * st["bs"], st["D"])[:, :length]
    v = st["vt"][table[:nb].long()].permute(1, 0, 3, 2).reshape(st["Hkv"], nb * st["bs"], st["D"])[:, :length]
    return k, v


def _plain_attend(st):
    H, Hkv, D, P = st["H"], st["Hkv"], st["D"], st["prefix"]
    G, out, at = H // Hkv, st["out"], 0
    empty = st["k"].new_zeros((Hkv, 0, D))
    kp, vp = _gathered(st, st["prefix_table"], P) if P else (empty, empty)
    kp, vp = kp.float(), vp.float()
    for r, (held, new) in enumerate(st["plan"]):
        if not new:
            continue
        k, v = _gathered(st, st["tables"][r], held + new)
        k, v = torch.cat([kp, k.float()], 1), torch.cat([vp, v.float()], 1)
        last = P + held + torch.arange(new, device=k.device)
        hidden = torch.arange(k.shape[1], device=k.device)[None] > last[:, None]
        q = st["q"][at:at + new].float().view(new, Hkv, G, D).transpose(0, 1).reshape(Hkv, new * G, D)
        s = torch.bmm(q, k.transpose(1, 2).contiguous()) * st["scale"]
        s.view(Hkv, new, G, -1).masked_fill_(hidden[:, None], -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.bmm(p, v) / p.sum(-1, keepdim=True)
        out[at:at + new] = o.view(Hkv, new, G, D).transpose(0, 1).reshape(new, H * D).to(torch.bfloat16)
        at += new
    return out


# ---------------------------------------------------------------- work


def work(case):
    held, new = _lengths(case)
    kind, R, bs, n, P = case["kind"], case["R"], case["bs"], sum(new), case["prefix"]
    if kind == "step":
        freed = [case["freed"] > 0 and i % case["freed"] == 1 for i in range(R)]
        old = [0 if f else h for h, f in zip(held, freed)]
        back = sum(_blocks(h, bs) for h, f in zip(held, freed) if f)
        grow = sum(_blocks(o + w, bs) - _blocks(o, bs) for o, w in zip(old, new))
        kept = sum(1 for o, w in zip(old, new) if w and o % bs)
        return dict(bytes=16 * R + 8 * (n + case["pad"]) + 8 * (back + grow) + 4 * kept, flops=4 * n)
    c = HEADS[case["shape"]]
    H, Hkv, D = c["H"], c["Hkv"], c["D"]
    if kind == "append":
        angles = len({p for h, w in zip(held, new) for p in range(h, h + w)})
        return dict(bytes=4 * n * (H + 2 * Hkv) * D + 4 * angles * D + 8 * n, flops=3 * n * (H + Hkv) * D)
    keys = P + sum(h + w for h, w in zip(held, new) if w)
    pairs = sum(w * (P + h) + w * (w + 1) // 2 for h, w in zip(held, new))
    return dict(bytes=4 * n * H * D + 4 * keys * Hkv * D, flops=4 * H * D * pairs)


# ---------------------------------------------------------------- 64 bits


def exact(case, seed):
    st = _inputs(case, seed)
    return {"step": _exact_step, "append": _exact_append, "attend": _exact_attend}[case["kind"]](case, st)


def _exact_step(case, st):
    """The same bookkeeping, one sequence and one position after the other."""
    bs = st["bs"]
    held, new = _lengths(case)
    tables, free = st["tables"].tolist(), st["free"].tolist()
    stack = free[:st["n_free"].item()]
    for r, gone in enumerate([] if st["release"] is None else st["release"].tolist()):
        if gone:
            stack += tables[r][:_blocks(held[r], bs)]
            held[r] = 0
    free[:len(stack)] = stack
    starts, slots, positions = [0], [], []
    for r, w in enumerate(new):
        for p in range(held[r], held[r] + w):
            if p % bs == 0:
                tables[r][p // bs] = stack.pop()
            slots.append(tables[r][p // bs] * bs + p % bs)
            positions.append(case["prefix"] + p)
        starts.append(len(slots))
    behind = [-1] * (st["rows"] - len(slots))
    return dict(lengths=_i32([h + w for h, w in zip(held, new)]), n_free=_i32([len(stack)]), row_starts=_i32(starts),
                slots=_i32(slots + behind), positions=_i32(positions + behind), tables=_i32(tables), free=_i32(free))


def _exact_append(case, st):
    H, Hkv, D, bs = st["H"], st["Hkv"], st["D"], st["bs"]
    q, k, vt = (st[name].double() for name in ("q", "k", "vt"))
    x = st["qkv"].double().view(st["rows"], H + 2 * Hkv, 2, D // 2)
    turn = torch.complex(st["cos"].double(), st["sin"].double())
    where = [s for s in st["slots"].tolist() if s >= 0]
    n = len(where)
    z = torch.complex(x[:n, :, 0], x[:n, :, 1]) * turn[st["positions"][:n].long()][:, None]
    z = torch.stack([z.real, z.imag], 2).reshape(n, H + 2 * Hkv, D)
    q[:n] = z[:, :H].reshape(n, H * D)
    block, off = torch.tensor(where, device="cuda") // bs, torch.tensor(where, device="cuda") % bs
    k[block, :, off] = z[:, H:H + Hkv]
    vt.transpose(2, 3)[block, :, off] = x.reshape(st["rows"], H + 2 * Hkv, D)[:n, H + Hkv:]
    return q, k, vt


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
        at_slot = torch.tensor(places, device="cuda")
        k = st["k"][at_slot // bs, :, at_slot % bs].double()                       # [keys, Hkv, D]
        v = st["vt"][at_slot // bs, :, :, at_slot % bs].double()
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
