"""A key/value cache in blocks of 4- or 8-bit codes in plain torch and float64: what the quantized
cache's tests compare with.  The codes are those of ``_lib.quantize``, which has tests of its own
against the oracle."""
import math

import torch

from shardcompute_amd import _lib
from tests.block_util import Cache

MID = {4: 8, 8: 128}


def stored(x, bits):
    """(values, scales, distance from the group's middle code) in float64 of x bf16 [..., D]."""
    D = x.shape[-1]
    wq, s, b = _lib.quantize(x.float().reshape(-1, D), bits=bits)
    words = wq.view(torch.int32).long() & 0xFFFFFFFF
    codes = ((words[..., None] >> (torch.arange(32 // bits, device=x.device) * bits)) & (2 ** bits - 1)).flatten(-2)
    s, b = s.double().repeat_interleave(64, -1), b.double().repeat_interleave(64, -1)
    return tuple(t.view(x.shape) for t in (s * codes + b, s.expand_as(codes).contiguous(), s * (codes - MID[bits])))


def rows_of(k, v):
    """qkv rows [n, 3 * Hkv * D] whose q is 0 and whose k and v [n, Hkv, D] are these."""
    n = k.shape[0]
    return torch.cat([torch.zeros_like(k), k, v], 1).reshape(n, -1).contiguous()


def write(pool, k, v, slots, bits):
    """k, v [n, Hkv, D] at ``slots``, rotated by no angle."""
    n, Hkv, D = k.shape
    one = torch.ones((1, D // 2), device=k.device)
    _lib.rope_append_quantized(rows_of(k, v), Hkv, Hkv, D, one, torch.zeros_like(one), pool, slots.to(torch.int32),
                               torch.zeros(n, dtype=torch.int32, device=k.device), bits=bits)


class QuantCache(Cache):
    """block_util's Cache with its attended positions quantized into ``pool``; every other byte is
    0xFF: scales, biases and the values of everything no row attends are NaN."""

    def __init__(self, bits, *a, blocks_more=0, **kw):
        super().__init__(*a, **kw)
        self.bits = bits
        nb = self.k.shape[0]
        shape = _lib.quantized_pool_shape(nb + blocks_more, self.Hkv, self.bs, self.D, bits)
        self.pool = torch.full(shape, 255, dtype=torch.uint8, device="cuda")
        at = (~torch.isnan(self.k[:, 0, :, 0])).nonzero()
        if at.numel():
            write(self.pool, self.k[at[:, 0], :, at[:, 1]], self.vt[at[:, 0], :, :, at[:, 1]],
                  at[:, 0] * self.bs + at[:, 1], bits)

    def attend(self, q=None, scale=None, **kw):
        if self.prefix_table is not None:
            kw.setdefault("prefix_table", self.prefix_table)
            kw.setdefault("prefix_len", self.prefix_len)
        return _lib.attention_quantized(self.q if q is None else q, self.H, self.Hkv, self.D, self.pool, self.row_starts,
                                        self.lens, self.tables, scale or self.scale, bits=self.bits, **kw)

    def workspace_bytes(self, max_new):
        pre = 0 if self.prefix_table is None else self.prefix_table.numel() * self.bs
        return _lib.attention_quantized_workspace_bytes(self.N, len(self.lengths), self.H, self.Hkv, self.D,
                                                        self.tables.shape[1] * self.bs, pre, max_new, bits=self.bits)

    def exact(self, scale=None):
        """(out, bound) [N, H, D] in float64, rows of the sequences only (0 elsewhere).

        The bound of each element, beside the output's own rounding: the weights are rounded to
        bf16 (2^-8) where they meet a value's distance from the middle of its group's codes, or
        the value itself; keys and values may be rounded to bf16 (2^-8 each) on their way into the
        matrix instructions, which moves a score by up to e = 2^-8 scale sum |q k| and a quotient
        of two sums of exponents by 2 e.  2^-12 of the values for the fp32 scores, exponents and sums,
        2^-11 of the values' scales for the sums of codes that are not centred."""
        scale, D, H, G, bs = scale or self.scale, self.D, self.H, self.H // self.Hkv, self.bs
        out = torch.zeros((self.N, H, D), dtype=torch.float64, device="cuda")
        bound = torch.zeros_like(out)

        def gather(table, n):
            p = torch.arange(n, device="cuda")
            b = table.long()[p // bs]
            return self.k[b, :, p % bs], self.vt[b, :, :, p % bs]               # [n, Hkv, D]

        pre = gather(self.prefix_table, self.prefix) if self.prefix else None
        for r, n in enumerate(self.lengths):
            a, b = self.starts[r], self.starts[r + 1]
            if a == b:
                continue
            k, v = gather(self.tables[r], n)
            if pre:
                k, v = torch.cat([pre[0], k]), torch.cat([pre[1], v])
            k = stored(k, self.bits)[0]
            v, vs, dev = stored(v, self.bits)
            last = self.prefix + n - (b - a) + torch.arange(b - a, device="cuda")
            hidden = torch.arange(k.shape[0], device="cuda")[None] > last[:, None]
            for h in range(H):
                q, kh = self.q[a:b, h * D:(h + 1) * D].double(), k[:, h // G].T.contiguous()
                p = torch.softmax((q @ kh * scale).masked_fill(hidden, -math.inf), -1)
                e = 2.0 ** -8 * scale * (q.abs() @ kh.abs()).masked_fill(hidden, 0).amax(-1, keepdim=True)
                out[a:b, h] = p @ v[:, h // G]
                mag = p @ v[:, h // G].abs()
                spread = torch.maximum(p @ dev[:, h // G].abs(), mag)
                bound[a:b, h] = (2.0 ** -8 * out[a:b, h].abs() + 2.0 ** -8 * spread + (2.0 ** -8 + 2 * e + 2.0 ** -12) * mag
                                 + 2.0 ** -11 * (p @ vs[:, h // G].abs()))
        return out, bound


def assert_attention(got, exact, bound, rows):
    """Every element within its bound, and all of them together within 2^-7 (2-norm): the four
    roundings of the bound are 0.0017 of their operand each in the mean (a uniform error of half
    a step, 2^-8 at most), that of the keys times a score's spread of 1.6 at most here, together
    0.0041; 2^-7 is 1.9 times that."""
    got = got[:rows].double().view(rows, exact.shape[1], exact.shape[2])
    exact, bound = exact[:rows], bound[:rows]
    assert torch.isfinite(got).all()
    err = (got - exact).abs()
    assert (err <= bound).all(), float((err / bound.clamp(min=1e-30)).max())
    if rows * exact.shape[1] >= 16:
        assert err.norm() <= 2.0 ** -7 * exact.norm(), float(err.norm() / exact.norm())
