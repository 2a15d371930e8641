"""Keys and values in eight bits, written out in 64 bits: rounding of a row, the pages' layout, attention over them."""
import math

import torch

PAGE = 64


def block(hd):
    return 64 if hd % 64 == 0 else 32 if hd % 32 == 0 else 16


def round_e4m3(y):
    """Doubles rounded to the nearest e4m3 number, ties to the even code, magnitudes above 448 to 448."""
    m, x = torch.frexp(y.abs())                                  # y = m 2^x, m in [1/2, 1)
    step = torch.ldexp(torch.ones_like(y), torch.clamp(x - 1, min=-6) - 3)
    return torch.copysign(torch.clamp(torch.round(y.abs() / step) * step, max=448.0), y)


def code_of(v):
    """The codes of e4m3 numbers."""
    m, x = torch.frexp(v.abs())
    normal = v.abs() >= 2.0 ** -6
    body = torch.where(normal, (x - 1 + 7) * 8 + torch.round((m * 2 - 1) * 8).long(), torch.round(v.abs() * 512).long())
    return (body + 128 * torch.signbit(v)).to(torch.uint8)


def quantise(x):
    """Rows ``x [..., hd]`` as ``(codes, exponent bytes, the doubles they stand for)``."""
    x = x.double()
    finite = torch.isfinite(x).all(-1)
    a = torch.where(finite, x.abs().amax(-1), 0.0)
    m, e = torch.frexp(a)                                         # 448 = 7/8 2^9
    e = torch.clamp(e - 9 + (m > 0.875), -117, 119)
    e = torch.where(a == 0, -117, e)
    scale = torch.ldexp(torch.ones_like(a), e)
    v = round_e4m3(torch.where(finite[..., None], x / scale[..., None], 0.0))
    value = torch.where(finite[..., None], v * scale[..., None], math.nan)
    return torch.where(finite[..., None], code_of(v), 127).to(torch.uint8), torch.where(finite, e + 127, 255).to(torch.uint8), value


class Held:
    """Sequences ``ks[s], vs[s] [len, nkv, hd]`` in pages that lie in random order; everything nobody wrote holds ``fill``."""

    def __init__(self, ks, vs, seed=0, fill=255, width=0):
        nkv, hd = ks[0].shape[1:]
        lens = [k.shape[0] for k in ks]
        counts = [-(-n // PAGE) for n in lens]
        W = max(counts + [width, 1])
        order = torch.randperm(sum(counts), generator=torch.Generator().manual_seed(seed)) + 1
        n, B = sum(counts) + 1, block(hd)
        full = lambda *shape: torch.full(shape, fill, dtype=torch.uint8)  # noqa: E731
        self.k, self.v = full(n, nkv, hd // B, PAGE, B), full(n, nkv, hd, PAGE)
        self.k_exp, self.v_exp = full(n, nkv, PAGE), full(n, nkv, PAGE)
        self.table, at = torch.zeros((len(ks), W), dtype=torch.int32), 0
        self.keys, self.values, self.lens = [], [], lens
        for s, c in enumerate(counts):
            self.table[s, :c] = order[at:at + c].int()
            at += c
        for s, (k, v) in enumerate(zip(ks, vs)):
            (kc, ke, kv), (vc, ve, vv) = quantise(k), quantise(v)
            self.keys.append(kv)
            self.values.append(vv)
            for j in range(lens[s]):
                p, r = int(self.table[s, j // PAGE]), j % PAGE
                self.k[p, :, :, r] = kc[j].view(nkv, hd // B, B)
                self.v[p, :, :, r] = vc[j]
                self.k_exp[p, :, r], self.v_exp[p, :, r] = ke[j], ve[j]

    def pages(self, device="cuda"):
        from synaptix_b200 import ops
        return ops.KV8Pages(*(t.to(device) for t in (self.k, self.v, self.k_exp, self.v_exp)))


def attend(q, keys, values, pos, scale, window=None, softcap=None, sinks=None, chunk=None):
    """Queries ``q [n, nh, hd]`` at positions ``pos [n]`` over ``keys, values [len, nkv, hd]``; ``(result, sum |w v|)`` in doubles."""
    n, nh, hd = q.shape
    G = nh // keys.shape[1]
    k, v = keys.repeat_interleave(G, 1), values.repeat_interleave(G, 1)
    s = torch.einsum("nhd,jhd->nhj", q.double(), k) * scale
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    j, pos = torch.arange(k.shape[0]), pos[:, None]
    seen = j <= pos
    if window:
        seen &= j > pos - window
    if chunk:
        seen &= torch.div(j, chunk, rounding_mode="floor") == torch.div(pos, chunk, rounding_mode="floor")
    s = torch.where(seen[:, None], s, -math.inf)
    if sinks is not None:
        s = torch.cat([s, sinks.double()[None, :, None].expand(n, nh, 1)], -1)
    w = torch.softmax(s, -1)[..., :k.shape[0]]
    w = torch.where(seen[:, None], w, 0.0)
    v = torch.where(seen.any(0)[:, None, None], v, 0.0)
    return torch.einsum("nhj,jhd->nhd", w, v).reshape(n, -1), torch.einsum("nhj,jhd->nhd", w, v.abs()).reshape(n, -1)
