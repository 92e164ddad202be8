"""A key/value cache in blocks in plain Python and float64: what the block tests compare with."""
import math

import torch


def cdiv(a, b):
    return -(-a // b)


class PlainTables:
    """``block_tables``'s bookkeeping, one sequence and one position after the other."""

    def __init__(self, lengths, tables, free, n_free, cap, bs):
        self.lengths, self.tables, self.bs, self.cap = list(lengths), [list(t) for t in tables], bs, cap
        self.free, self.n_free, self.status = list(free), n_free, 0

    def step(self, new, rows, prefix=0, release=None):
        bs, R = self.bs, len(self.lengths)
        width = len(self.tables[0])
        new = [max(w, 0) for w in new]
        gone = release or [False] * R
        old = [0 if f else n for n, f in zip(self.lengths, gone)]
        back = [b for r in range(R) if gone[r] for b in self.tables[r][:cdiv(self.lengths[r], bs)]]
        fits = [(r, o, w) for r, (o, w) in enumerate(zip(old, new)) if o + w <= width * bs]
        need = sum(cdiv(o + w, bs) - cdiv(o, bs) for _, o, w in fits)
        status = (1 if need > self.n_free + len(back) else 0) | (2 if len(fits) < R else 0)
        status |= (4 if sum(w for _, _, w in fits) > rows else 0) | (8 if self.n_free + len(back) > self.cap else 0)
        if status:
            self.status |= status
            return [0] * (R + 1), [-1] * rows, [-1] * rows
        for b in back:
            self.free[self.n_free] = b
            self.n_free += 1
        starts, slots, positions = [0], [], []
        for r in range(R):
            for p in range(old[r], old[r] + new[r]):
                if p % bs == 0:
                    self.n_free -= 1
                    self.tables[r][p // bs] = self.free[self.n_free]
                slots.append(self.tables[r][p // bs] * bs + p % bs)
                positions.append(prefix + p)
            starts.append(len(slots))
        self.lengths = [o + w for o, w in zip(old, new)]
        pad = [-1] * (rows - len(slots))
        return starts, slots + pad, positions + pad


def attention64(q, H, Hkv, D, k, vt, starts, lengths, tables, scale, prefix_table, prefix):
    """(out, softmax . |v|) [N, H, D] in float64, rows of the sequences only (0 elsewhere)."""
    N, bs, G = q.shape[0], k.shape[2], H // Hkv
    out = torch.zeros((N, H, D), dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)

    def gather(table, n):
        p = torch.arange(n, device=q.device)
        b = table.long()[p // bs]
        return k[b, :, p % bs].double(), vt[b, :, :, p % bs].double()          # [n, Hkv, D]

    kp, vp = gather(prefix_table, prefix) if prefix else (None, None)
    for r in range(len(lengths)):
        a, b = starts[r], starts[r + 1]
        if a == b:
            continue
        kk, vv = gather(tables[r], lengths[r])
        if prefix:
            kk, vv = torch.cat([kp, kk]), torch.cat([vp, vv])
        last = prefix + lengths[r] - (b - a) + torch.arange(b - a, device=q.device)
        hidden = torch.arange(kk.shape[0], device=q.device)[None] > last[:, None]
        for h in range(H):
            s = q[a:b, h * D:(h + 1) * D].double() @ kk[:, h // G].T.contiguous() * scale
            p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
            out[a:b, h] = p @ vv[:, h // G]
            mag[a:b, h] = p @ vv[:, h // G].abs()
    return out, mag


class Cache:
    """Random tables and a random pool: ``held[r] + new[r]`` positions of sequence r behind
    ``prefix`` shared ones, blocks in random order, everything no row attends NaN."""

    def __init__(self, held, new, prefix, bs, H, Hkv, D, pad=0, seed=0, width=None):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.H, self.Hkv, self.D, self.bs, self.prefix = H, Hkv, D, bs, prefix
        R = len(held)
        after = [h + w for h, w in zip(held, new)]
        counts = [cdiv(n, bs) for n in after]
        width = width or max(max(counts), 1)
        order = torch.randperm(sum(counts) + cdiv(prefix, bs) + 2, generator=g, device="cuda").to(torch.int32)
        nb, at = order.numel(), 0
        # entries past a sequence's last block hold nonsense
        self.tables = torch.full((R, width), -7, dtype=torch.int32, device="cuda")
        self.k = torch.full((nb, Hkv, bs, D), float("nan"), dtype=torch.bfloat16, device="cuda")
        self.vt = torch.full((nb, Hkv, D, bs), float("nan"), dtype=torch.bfloat16, device="cuda")

        def fill(table, n):
            nonlocal at
            c = cdiv(n, bs)
            table[:c] = order[at:at + c]
            at += c
            p = torch.arange(n, device="cuda")
            b = table[:c].long()[p // bs]
            self.k[b, :, p % bs] = torch.randn((n, Hkv, D), generator=g, device="cuda").to(torch.bfloat16)
            self.vt[b, :, :, p % bs] = torch.randn((n, Hkv, D), generator=g, device="cuda").to(torch.bfloat16)

        for r, n in enumerate(after):
            if n:
                fill(self.tables[r], n)
        self.prefix_table = None
        if prefix:
            self.prefix_table = torch.full((cdiv(prefix, bs) + 1,), 1 << 30, dtype=torch.int32, device="cuda")
            fill(self.prefix_table, prefix)
        self.starts = [sum(new[:i]) for i in range(R + 1)]
        self.lengths, self.max_new = after, max(new)
        self.row_starts = torch.tensor(self.starts, dtype=torch.int32, device="cuda")
        self.lens = torch.tensor(after, dtype=torch.int32, device="cuda")
        self.prefix_len = torch.tensor([prefix], dtype=torch.int32, device="cuda")
        self.N = self.starts[-1] + pad
        self.q = torch.randn((self.N, H * D), generator=g, device="cuda").to(torch.bfloat16)
        self.scale = 1.0 / math.sqrt(D)

    def attend(self, q=None, scale=None, **kw):
        from shardcompute_amd import _lib
        if self.prefix_table is not None:
            kw.setdefault("prefix_table", self.prefix_table)
            kw.setdefault("prefix_len", self.prefix_len)
        return _lib.attention_shared(self.q if q is None else q, self.H, self.Hkv, self.D, self.k, self.vt,
                                     self.row_starts, self.lens, self.tables, scale or self.scale, **kw)

    def exact(self, scale=None):
        return attention64(self.q, self.H, self.Hkv, self.D, self.k, self.vt, self.starts, self.lengths, self.tables,
                           scale or self.scale, self.prefix_table, self.prefix)


def assert_attention(got, out, mag, rows):
    """Every element within its roundings: the output's (half a bf16 step, 2^-8 of it) and the
    probabilities' (2^-8 of softmax . |v|), and 2^-12 of that for the fp32 scores, exponents and
    sums (D = 128 products of |q k| scale <= 40 in all: 128 * 40 * 2^-24 = 2^-11.7 at the worst,
    a fortieth of it usual)."""
    got = got[:rows].double().view(rows, out.shape[1], out.shape[2])
    out, mag = out[:rows], mag[:rows]
    assert torch.isfinite(got).all()
    err, bound = (got - out).abs(), 2.0 ** -8 * out.abs() + (2.0 ** -8 + 2.0 ** -12) * mag
    assert (err <= bound).all(), float((err / bound.clamp(min=1e-30)).max())
