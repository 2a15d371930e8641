"""Kernels of a cache in eight bits against 64-bit arithmetic, at the edges of pages, heads and types.

Writing without norm and rotation, and reading, are exact: every bit is compared.  A normed and rotated element is off by a few
roundings of 2^-24 of the row's largest in 32 bits before it is rounded to its type (bfloat16 2^-8 of itself, e4m3 2^-4).

Attention: a sum of n products is off by less than (n + 8) u of the sum of their magnitudes, with u = 2^-24 by FFMA and 2^-22 in the
tensor cores, which may truncate; there a query's elements below 2^-9 of its largest are off by up to 2^-18 of that.  With D = that bound on a score and N keys, a weight is off by 2 D + 8 2^-22 of itself (2^-11 more
where weights are rounded to half precision), the sum over keys by (N + 64) u of sum |w v|; then the result is rounded to its type."""
import math

import pytest
import torch

import plain_kv8 as P
import plain_qwen3 as Q
from helpers import BF16_REL, F32_REL, folder
from test_kv8_cpu import step
from tiny import random_tokens

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def on_gpu(ctx):
    for k, v in vars(ctx).items():
        if isinstance(v, torch.Tensor):
            setattr(ctx, k, v.cuda())
    return ctx


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


def prepare(x, held, pos, seq, nh, nkv, hd, wq=None, wk=None, freq=None, rot=0, col=0, write=True, q=True):
    """``kv8_prepare`` of rows ``x``; ``(q, the pages afterwards)``."""
    from synaptix_b200 import ops
    pages = held.pages()
    out = torch.full((x.shape[0], nh * hd), 7.0, dtype=x.dtype, device="cuda") if q else None
    a, b, f, p, s, t = cuda(wq, wk, freq, pos.int(), seq.int(), held.table)
    ops.kv8_prepare(x.cuda(), out, pages if write else None, a, b, f, rot, 1e-6, p, s, t, nh, nkv, hd, col=col)
    return (None if out is None else out.cpu()), pages


def written(pages, held, s, j, nkv, hd):
    """Codes and exponents of sequence ``s``, position ``j``: ``(k, k_exp, v, v_exp)``."""
    p, r = int(held.table[s, j // 64]), j % 64
    return (pages.k[p, :, :, r].reshape(nkv, hd).cpu(), pages.k_exp[p, :, r].cpu(), pages.v[p, :, :, r].cpu(), pages.v_exp[p, :, r].cpu())


def empty(lens, nkv, hd, fill=0xAB, **kw):
    held = P.Held([torch.zeros(n, nkv, hd) for n in lens], [torch.zeros(n, nkv, hd) for n in lens], fill=fill, **kw)
    for t in (held.k, held.v, held.k_exp, held.v_exp):
        t.fill_(fill)
    return held


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nh,nkv,hd", [(4, 2, 64), (3, 3, 16), (5, 1, 48), (8, 2, 128), (2, 1, 80), (2, 2, 256), (16, 8, 32), (1, 1, 144), (40, 8, 128), (80, 8, 128), (9, 9, 64)])
@pytest.mark.parametrize("past,new,col", [([0], [1], 0), ([63, 5, 127], [1, 1, 1], 8), ([60, 0], [9, 70], 0), ([0, 3], [300, 129], 24), ([130], [1], 3)])
def test_write(dtype, nh, nkv, hd, past, new, col):
    """Without norm and rotation: codes and exponents to the bit, queries unchanged, and not a byte beside them."""
    ctx = step([p + n for p, n in zip(past, new)], new)
    T, heads = sum(new), nh + 2 * nkv
    x = (randn(T, heads, hd, seed=hd + T) * torch.exp(3 * randn(T, heads, 1, seed=1))).to(dtype)
    rows = torch.full((T, col + heads * hd + (col and 5)), 3.0, dtype=dtype)
    rows[:, col:col + heads * hd] = x.view(T, -1)
    held = empty([p + n for p, n in zip(past, new)], nkv, hd)
    q, pages = prepare(rows, held, ctx.positions, ctx.seq_of_token, nh, nkv, hd, col=col)
    assert torch.equal(q, x[:, :nh].reshape(T, -1))
    want = empty([p + n for p, n in zip(past, new)], nkv, hd)
    kc, ke, _ = P.quantise(x[:, nh:nh + nkv])
    vc, ve, _ = P.quantise(x[:, nh + nkv:])
    for t in range(T):
        s, j = int(ctx.seq_of_token[t]), int(ctx.positions[t])
        p, r = int(held.table[s, j // 64]), j % 64
        want.k[p, :, :, r], want.v[p, :, :, r] = kc[t].view(nkv, hd // P.block(hd), -1), vc[t]
        want.k_exp[p, :, r], want.v_exp[p, :, r] = ke[t], ve[t]
    for name, got in zip(("k", "v", "k_exp", "v_exp"), pages):
        assert torch.equal(got.cpu(), getattr(want, name)), name


@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_at_the_formats_borders(dtype, tokens):
    """Largest magnitudes at and beside 1.75 2^x, zeros, the smallest and largest numbers, infinities and NaN."""
    hd = 64
    tops = [0.0, 1.75, 1.7578125, 1.75 * 2 ** -30, 448.0, 450.0, 2.0 ** -126, 2.0 ** -133, 2.0 ** -118, 1.9921875 * 2.0 ** 127, 1.75 * 2.0 ** 127, 1.0,
            math.inf, -math.inf, math.nan, 1.9921875]
    x = torch.clamp(randn(tokens, 3, len(tops), hd) / 4, -1, 1)
    nkv = len(tops)
    rows = torch.zeros(tokens, 3, nkv, hd)
    for i, a in enumerate(tops):
        row = x[:, :, i] * (a if math.isfinite(a) else 1.0)
        row[..., 7] = -a if i % 2 else a
        row[..., 9] = -0.0
        rows[:, :, i] = row
    rows = rows.to(dtype)
    held = empty([tokens], nkv, hd)
    _, pages = prepare(rows.view(tokens, -1), held, torch.arange(tokens), torch.zeros(tokens), nkv, nkv, hd)
    (kc, ke, _), (vc, ve, _) = P.quantise(rows[:, 1]), P.quantise(rows[:, 2])
    for t in range(tokens):
        got = written(pages, held, 0, t, nkv, hd)
        for name, a, b in zip(("k", "k_exp", "v", "v_exp"), got, (kc[t], ke[t], vc[t], ve[t])):
            assert torch.equal(a, b), (name, t, (a != b).nonzero()[:4])
    assert (ke[0, 12:15] == 255).all() and (kc[0, 12:15] == 127).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd,rot", [(128, 128), (64, 64), (64, 32), (80, 20), (256, 256), (32, 0), (128, 64)])
@pytest.mark.parametrize("normed", [True, False])
@pytest.mark.parametrize("first,T", [(0, 5), (99990, 1), (131000, 70), (1, 300)])
def test_norm_and_rotation(dtype, hd, rot, normed, first, T):
    nh, nkv = 6, 2
    x = randn(T, nh + 2 * nkv, hd, seed=rot + T).to(dtype)
    wq, wk = (1 + 0.2 * randn(hd, seed=2), 1 + 0.2 * randn(hd, seed=3)) if normed else (None, None)
    freq = (1e6 ** (-torch.arange(rot // 2).double() * 2 / max(rot, 1))).float() if rot else None
    held = empty([64 * 5], nkv, hd)
    pos = torch.arange(first, first + T)
    # far positions in a short table: the sequence's first pages are page 0 here
    held.table = torch.cat([torch.zeros(1, first // 64, dtype=torch.int32), held.table], 1)
    q, pages = prepare(x.view(T, -1), held, pos, torch.zeros(T), nh, nkv, hd, wq, wk, freq, rot)
    y = x[:, :nh + nkv].double()
    if normed:
        gain = torch.cat([wq.expand(nh, hd), wk.expand(nkv, hd)]).double()
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6) * gain
    if rot:
        t = pos.double()[:, None] * freq.double()
        c, s = torch.cos(t)[:, None], torch.sin(t)[:, None]
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        y = torch.cat([a * c - b * s, b * c + a * s, y[..., rot:]], -1)
    # 32-bit steps ahead of the rounding: the norm's sum and root (hd + 8 roundings), gain, two products and a sum, sine and cosine (2 ulp each)
    loose = 2 * y.abs().amax(-1, keepdim=True) * (hd / 2 + 24) * 2.0 ** -24
    half = HALF_STEP[dtype]
    want = y[:, :nh]
    assert ((q.double().view(T, nh, hd) - want).abs() <= want.abs() * half + loose[:, :nh] * (1 + half)).all()
    _, ve, vv = P.quantise(x[:, nh + nkv:])
    for i in range(T):
        k, ke, v, e = written(pages, held, 0, int(pos[i]), nkv, hd)
        assert torch.equal(e, ve[i]) and torch.equal(v.view(torch.float8_e4m3fn).double() * torch.exp2(e.double() - 127)[:, None], vv[i])
        power = torch.exp2(ke.double() - 127)[:, None]
        key = y[i, nh:]
        a = key.abs().amax(-1, keepdim=True)
        assert (a <= 448 * power * (1 + 2.0 ** -12)).all() and (a > 224 * power * (1 - 2.0 ** -12)).all()
        step_ = torch.maximum(key.abs() * 2.0 ** -4, power * 2.0 ** -10)
        assert ((k.view(torch.float8_e4m3fn).double() * power - key).abs() <= (step_ + loose[i, nh:]) * (1 + 2.0 ** -4)).all()


def test_prepare_without_pages_or_queries():
    x = randn(3, 4 * 64).bfloat16()
    held = empty([10], 2, 64)
    q, pages = prepare(x, held, torch.arange(3), torch.zeros(3), 4, 2, 64, write=False)
    assert torch.equal(q, x) and all((t.cpu() == 0xAB).all() for t in pages)
    _, pages = prepare(x, held, torch.arange(3), torch.zeros(3), 0, 2, 64, q=False)
    kc, _, _ = P.quantise(x.view(3, 4, 64)[:, :2])
    assert torch.equal(written(pages, held, 0, 2, 2, 64)[0], kc[2])
    prepare(x[:0], held, torch.arange(0), torch.zeros(0), 4, 2, 64, write=False)


def test_places_outside_the_table_or_the_pages_are_not_written():
    x = randn(3, 6 * 64).bfloat16()
    held = empty([64], 2, 64)
    held.table = torch.tensor([[77, -1]], dtype=torch.int32)
    _, pages = prepare(x, held, torch.tensor([5, 70, 5000]), torch.zeros(3), 2, 2, 64)
    assert all((t.cpu() == 0xAB).all() for t in pages)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nkv,hd", [(2, 64), (1, 16), (8, 128), (3, 96), (1, 256), (2, 80)])
@pytest.mark.parametrize("lens", [[1], [64, 63, 65], [0, 130, 1], [700]])
def test_read(dtype, nkv, hd, lens):
    from synaptix_b200 import ops
    ks, vs = ([randn(n, nkv, hd, seed=i + 7 * w) * torch.exp(4 * randn(n, nkv, 1, seed=i)) for i, n in enumerate(lens)] for w in (1, 2))
    held = P.Held(ks, vs, width=12)
    k, v, table = ops.kv8_read(held.pages(), on_gpu(step(lens, [0] * len(lens))), held.table.cuda(), dtype)
    assert k.shape == v.shape == (sum(-(-n // 64) for n in lens), nkv, 64, hd) and k.dtype == dtype
    for s, n in enumerate(lens):
        for got, want in ((k, held.keys), (v, held.values)):
            rows = got[table[s, :-(-n // 64)].long()].transpose(1, 2).reshape(-1, nkv, hd).cpu()
            assert torch.equal(rows[:n].double(), want[s]) and (rows[n:] == 0).all()


def test_read_of_a_window_and_of_a_row_that_was_not_finite():
    from synaptix_b200 import ops
    lens, new = [500, 300, 64], [3, 200, 1]
    ks, vs = ([randn(n, 2, 64, seed=i + 7 * w) for i, n in enumerate(lens)] for w in (1, 2))
    ks[0][450, 1, 3], vs[1][290, 0, 60] = math.inf, math.nan
    held = P.Held(ks, vs)
    for kw, firsts in ((dict(window=70), [497 - 69, 100 - 69, 0]), (dict(chunk=128), [384, 0, 0]), (dict(window=1), [497, 100, 63])):
        k, v, table = ops.kv8_read(held.pages(), on_gpu(step(lens, new)), held.table.cuda(), torch.float32, **kw)
        assert k.shape[0] == sum(-(-n // 64) - f // 64 for n, f in zip(lens, firsts)) and int(table.max()) < k.shape[0] and int(table.min()) >= 0
        for s, (n, f) in enumerate(zip(lens, firsts)):
            for got, want in ((k, held.keys), (v, held.values)):
                rows = got[table[s, :-(-n // 64)].long()].transpose(1, 2).reshape(-1, 2, 64).cpu().double()
                assert torch.equal(rows[f:n].nan_to_num(9e9), want[s][f:].nan_to_num(9e9))
                if kw.get("window", 0) != 1 and s < 2 and got is (k if s == 0 else v):
                    assert rows.isnan().any()


def bound(q, held, s, want, weight, pos, scale, dtype, hd, tensor_cores, softcap=None, portions=False):
    n = held.keys[s].shape[0]
    G = q.shape[1] // held.keys[s].shape[1]
    spread = torch.einsum("nhd,jhd->nhj", q.double().abs(), held.keys[s].nan_to_num(0.0).abs().repeat_interleave(G, 1)).amax().item() * scale
    u = 2.0 ** -22 if tensor_cores else 2.0 ** -24
    score = (hd + 8) * u * spread + (2.0 ** -20 * softcap if softcap else 0.0)
    if tensor_cores:
        score += 2.0 ** -18 * q.abs().amax().item() * held.keys[s].nan_to_num(0.0).abs().sum(-1).amax().item() * scale
    rel = 2 * score + 8 * 2.0 ** -22 + (2.0 ** -11 if tensor_cores else 0.0) + (n + 64) * u
    if portions:       # the kernels of the 16-bit cache round weights to bfloat16 (half a step: 2^-8 of themselves), those of the 32-bit one cut operands in pieces
        rel += 2.0 ** -8 if dtype == torch.bfloat16 else 8 * hd * 2.0 ** -23
    return want.abs() * HALF_STEP[dtype] + weight * rel * 1.01


def check(q, held, lens, new, nh, hd, dtype, tensor_cores, out_scale=1.0, out=None, out_col=0, window=None, softcap=None, sinks=None, chunk=None, scale=None):
    from synaptix_b200 import ops
    scale = hd ** -0.5 if scale is None else scale
    nkv = held.keys[0].shape[1]
    q = q.to(dtype)
    got = ops.kv8_attention(q.view(q.shape[0], -1).cuda(), held.pages(), on_gpu(step(lens, new)), held.table.cuda(), nh, nkv, hd, scale, window,
                            softcap=softcap, sinks=None if sinks is None else sinks.cuda(), chunk=chunk, out=out, out_col=out_col, out_scale=out_scale)
    assert got.dtype == dtype
    res = got.cpu().double()[:, out_col:out_col + nh * hd]
    at = 0
    for s, (n, m) in enumerate(zip(lens, new)):
        part = slice(at, at + m)
        at += m
        if m == 0:
            continue
        pos = torch.arange(n - m, n)
        want, weight = P.attend(q[part], held.keys[s], held.values[s], pos, scale, window, softcap, sinks, chunk)
        tol = bound(q[part], held, s, want, weight, pos, scale, dtype, hd, tensor_cores, softcap, max(new) > 1) * abs(out_scale)
        off = (res[part] - want * out_scale).abs()
        assert (off <= tol).all(), (s, n, m, (off / tol).max().item(), (off > tol).sum().item())
    return got


def filled(lens, nkv, hd, seed=0, loud=True, **kw):
    ks, vs = ([randn(n, nkv, hd, seed=seed + i + 100 * w) for i, n in enumerate(lens)] for w in (1, 2))
    if loud:                                                       # rows of unlike size, by factors of up to a thousand
        for v in vs:
            v *= torch.exp2(torch.randint(-5, 6, v.shape[:2] + (1,), generator=torch.Generator().manual_seed(seed)).float())
    return P.Held(ks, vs, seed=seed, **kw)


SINGLE_LENS = [[1], [64], [65, 1, 130], [5, 1000, 63, 2, 700], [3000]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nh,nkv,hd", [(4, 4, 64), (32, 8, 128), (10, 2, 64), (8, 1, 128), (16, 1, 64), (7, 1, 96), (4, 2, 256), (3, 1, 16), (40, 2, 32), (24, 1, 128)])
@pytest.mark.parametrize("lens", SINGLE_LENS)
def test_single_tokens(dtype, nh, nkv, hd, lens):
    held = filled(lens, nkv, hd, seed=nh)
    check(2 * randn(len(lens), nh, hd, seed=3), held, lens, [1] * len(lens), nh, hd, dtype, dtype == torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (32, 8, 128), (6, 2, 48)])
@pytest.mark.parametrize("options", [dict(window=1), dict(window=64), dict(window=100), dict(window=5000), dict(sinks=True), dict(window=70, sinks=True),
                                     dict(softcap=5.0), dict(chunk=100), dict(chunk=64, window=30, softcap=3.0, sinks=True)])
def test_single_tokens_with_options(dtype, nh, nkv, hd, options):
    lens = [1, 64, 129, 830, 200, 101]
    options = dict(options, sinks=randn(nh, seed=9) * 3) if options.get("sinks") else options
    check(2 * randn(len(lens), nh, hd, seed=3), filled(lens, nkv, hd), lens, [1] * len(lens), nh, hd, dtype, dtype == torch.bfloat16, **options)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [[1, 1], [1, 40]])
def test_output_among_other_columns(dtype, new):
    lens, nh, hd = [70, 90], 4, 64
    out = torch.full((sum(new), nh * hd + 10), 3.0, dtype=dtype, device="cuda")
    got = check(randn(sum(new), nh, hd), filled(lens, 2, hd), lens, new, nh, hd, dtype, dtype == torch.bfloat16, out=out, out_col=6, out_scale=-0.5)
    assert got is out and (out[:, :6] == 3).all() and (out[:, 6 + nh * hd:] == 3).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_are_not_finite(dtype):
    """A key or value that was not finite shows in the queries that see it and in no others; so does a query."""
    from synaptix_b200 import ops
    lens, hd, nh = [200, 200, 200, 200], 64, 4
    ks, vs = ([randn(n, 2, hd, seed=i + 7 * w) for i, n in enumerate(lens)] for w in (1, 2))
    ks[0][150, 0, 3], vs[1][150, 1, 5], ks[2][20, 0, 0], vs[2][20, 1, 0] = math.inf, math.nan, math.nan, math.inf
    held = P.Held(ks, vs)
    q = randn(4, nh, hd).to(dtype)
    q[3, 2, 1] = math.inf
    got = ops.kv8_attention(q.view(4, -1).cuda(), held.pages(), on_gpu(step(lens, [1] * 4)), held.table.cuda(), nh, 2, hd, 0.125, 100).cpu().view(4, nh, hd)
    bad = torch.zeros(4, nh, dtype=torch.bool)
    bad[0, :2] = bad[1, 2:] = bad[3, 2] = True
    assert torch.equal(got.isnan().any(-1), bad) and torch.equal(got.isnan().all(-1), bad)


@pytest.mark.parametrize("scale_k,scale_v,scale_q", [(1e-20, 1e20, 1e18), (1e15, 1e-30, 1e-16), (3e4, 1.0, 1.0), (1e-8, 1e-8, 1.0)])
def test_magnitudes_far_from_one(scale_k, scale_v, scale_q):
    lens, nh, hd = [300, 70], 8, 128
    ks, vs = ([randn(n, 2, hd, seed=i + 7 * w) * f for i, n in enumerate(lens)] for w, f in ((1, scale_k), (2, scale_v)))
    scale = hd ** -0.5 / (scale_k * scale_q) * (1.0 if scale_k != 3e4 else 3e4)
    check(randn(2, nh, hd) * scale_q, P.Held(ks, vs), lens, [1, 1], nh, hd, torch.bfloat16, True, scale=scale)


def test_one_value_outweighs_all_others():
    """Values of unlike size: one is 2^40 times the others, and its key has next to no weight."""
    lens, nh, hd = [260], 4, 64
    ks, vs = randn(260, 1, hd, seed=1), randn(260, 1, hd, seed=2)
    q = torch.ones(1, nh, hd)
    ks[77] = -6.0                                                  # score -48 below zero: weight 1e-21
    vs[77] *= 2.0 ** 40
    check(q, P.Held([ks], [vs]), lens, [1], nh, hd, torch.bfloat16, True, scale=1 / 8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (16, 4, 128), (4, 2, 80)])
@pytest.mark.parametrize("lens,new", [([5], [5]), ([200], [200]), ([64, 300, 1, 131], [2, 33, 1, 131]), ([1000, 70], [3, 64])])
@pytest.mark.parametrize("options", [{}, dict(window=50), dict(sinks=True), dict(softcap=4.0, chunk=96)])
def test_portions(dtype, nh, nkv, hd, lens, new, options):
    options = dict(options, sinks=randn(nh, seed=9)) if options.get("sinks") else options
    from synaptix_b200 import ops
    q = randn(sum(new), nh, hd, seed=3).to(dtype)
    held = filled(lens, nkv, hd)
    kw = {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in options.items()}
    got = ops.kv8_attention(q.view(q.shape[0], -1).cuda(), held.pages(), on_gpu(step(lens, new)), held.table.cuda(), nh, nkv, hd, hd ** -0.5, **kw).cpu().double()
    at = 0
    for s, (n, m) in enumerate(zip(lens, new)):
        part = slice(at, at + m)
        at += m
        pos = torch.arange(n - m, n)
        want, weight = P.attend(q[part], held.keys[s], held.values[s], pos, hd ** -0.5, **options)
        tol = bound(q[part], held, s, want, weight, pos, hd ** -0.5, dtype, hd, dtype == torch.bfloat16, options.get("softcap"), portions=True)
        assert ((got[part] - want).abs() <= tol).all(), (s, ((got[part] - want).abs() / tol).max().item())


@pytest.mark.parametrize("lens,new", [([6000], [70]), ([7000, 500, 129], [130, 300, 129]), ([8000, 64], [9, 6])])
@pytest.mark.parametrize("options", [{}, dict(window=4500), dict(sinks=True), dict(window=4001, sinks=True)])
def test_portions_over_long_caches(lens, new, options):
    """Few tiles of many keys: cut over the keys (``tc_parts``) and joined."""
    from synaptix_b200.ops.attention import tc_parts
    nh, nkv, hd = 16, 2, 128
    tiles = [(n - m + q0, min(n - m + q0 + 128, n) - 1) for n, m in zip(lens, new) for q0 in range(0, m, 128)]
    assert tc_parts(tiles, nh, options.get("window"), torch.device("cuda", 0))[1] > 1
    options = dict(options, sinks=randn(nh, seed=9) * 3) if options.get("sinks") else options
    check(2 * randn(sum(new), nh, hd, seed=3), filled(lens, nkv, hd), lens, new, nh, hd, torch.bfloat16, True, **options)


def test_when_keys_are_cut():
    from synaptix_b200.ops.attention import tc_parts
    d = torch.device("cuda", 0)
    assert tc_parts([(0, 127)], 32, None, d) == (0, 1)                       # one block of keys
    assert tc_parts([(128 * i, 128 * i + 127) for i in range(64)], 32, None, d) == (0, 1)   # a long prompt fills the SMs as it is
    chunk, parts = tc_parts([(100000, 100063)], 32, None, d)
    assert chunk * parts >= 782 > chunk * (parts - 1) and parts * 32 >= 148
    assert tc_parts([(100000, 100063)], 32, 500, d)[1] == 1                  # a window leaves few


@pytest.mark.parametrize("new", [[2], [4, 1, 8], [1, 4], [8, 1, 1]])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (32, 8, 128), (12, 1, 128), (5, 1, 64)])
@pytest.mark.parametrize("options", [{}, dict(window=33), dict(sinks=True)])
def test_a_few_tokens(new, nh, nkv, hd, options):
    """Portions of up to eight tokens attend over the codes, token by token."""
    lens = [m + past for m, past in zip(new, (300, 62, 0))]
    options = dict(options, sinks=randn(nh, seed=9)) if options.get("sinks") else options
    check(2 * randn(sum(new), nh, hd, seed=3), filled(lens, nkv, hd), lens, new, nh, hd, torch.bfloat16, True, **options)


@pytest.fixture
def over_the_codes(monkeypatch):
    """All portions attend over the codes, whatever is faster."""
    from synaptix_b200.ops import kv8
    calls, tile = [], kv8.kv8_tile
    monkeypatch.setattr(kv8, "FEW_NEW_TOKENS", 0)
    monkeypatch.setattr(kv8, "TILE_BF16_ROWS", {64: 1 << 30, 128: 1 << 30})
    monkeypatch.setattr(kv8, "kv8_tile", lambda *a, **kw: calls.append(1) or tile(*a, **kw))
    yield
    assert calls


# Bounds of portions over the codes.  bfloat16: those of single tokens (queries as two codes, weights as halves).  float32: queries and weights are two
# halves, off by 2^-22 of themselves; products are summed in chains of four instructions, each of which may drop 2^-22 of the sum so far, and chains by
# plain additions: a score is off by less than (4 + 2) 2^-22 + 8 2^-24, under (hd + 8) 2^-24, of its spread, the sum over keys by (2 + 4) 2^-22 + (n / 64 + 64) 2^-24.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (32, 8, 128), (64, 1, 128), (7, 1, 64), (24, 2, 128), (3, 3, 128)])
@pytest.mark.parametrize("lens,new", [([1], [1]), ([2, 65], [2, 1]), ([5000], [3]), ([64, 300, 1, 131], [2, 33, 1, 131]), ([2000, 64, 70], [150, 64, 0])])
@pytest.mark.parametrize("options", [{}, dict(window=1), dict(window=70, sinks=True), dict(softcap=4.0, chunk=96)])
def test_portions_over_the_codes(over_the_codes, dtype, nh, nkv, hd, lens, new, options):
    options = dict(options, sinks=randn(nh, seed=9) * 3) if options.get("sinks") else options
    held, ctx = filled(lens, nkv, hd, seed=nh), step(lens, new)
    ctx.all_single = False
    q = (2 * randn(sum(new), nh, hd, seed=3)).to(dtype)
    pages, table = held.pages(), held.table.cuda()
    from synaptix_b200 import ops
    kw = {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in options.items()}
    got, again = (ops.kv8_attention(q.view(q.shape[0], -1).cuda(), pages, on_gpu(ctx), table, nh, nkv, hd, hd ** -0.5, **kw).cpu() for _ in range(2))
    assert torch.equal(got, again)
    at = 0
    for s, (n, m) in enumerate(zip(lens, new)):
        part = slice(at, at + m)
        at += m
        if m:
            pos = torch.arange(n - m, n)
            want, weight = P.attend(q[part], held.keys[s], held.values[s], pos, hd ** -0.5, **options)
            tol = bound(q[part], held, s, want, weight, pos, hd ** -0.5, dtype, hd, dtype == torch.bfloat16, options.get("softcap"))
            assert ((got[part].double() - want).abs() <= tol).all(), (s, ((got[part].double() - want).abs() / tol).max().item())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("past", [0, 3000])
@pytest.mark.parametrize("window", [None, 50])
def test_portions_with_rows_that_are_not_finite(over_the_codes, dtype, past, window):
    """A key or value that was not finite shows in the tokens of a portion that see it, and leaves the others' results as they are without it."""
    from synaptix_b200 import ops
    hd, nh, new = 128, 4, 150
    ks, vs = ([randn(past + new, 2, hd, seed=i + 7 * w) for i in range(3)] for w in (1, 2))
    q = randn(3 * new, nh, hd).to(dtype)
    res = []
    for spoil in (False, True):
        if spoil:
            ks[0][past + 40, 0, 3], vs[1][past + 70, 1, 5] = math.inf, math.nan
            q = q.clone()
            q[2 * new + 9, 2, 1] = math.inf
        held = P.Held(ks, vs)
        ctx = step([past + new] * 3, [new] * 3)
        res.append(ops.kv8_attention(q.view(3 * new, -1).cuda(), held.pages(), on_gpu(ctx), held.table.cuda(), nh, 2, hd, 0.1, window).cpu().view(3, new, nh, hd))
    until = new if window is None else window
    bad = torch.zeros(3, new, nh, dtype=torch.bool)
    bad[0, 40:40 + until, :2] = bad[1, 70:70 + until, 2:] = bad[2, 9, 2] = True
    assert torch.equal(res[1].isnan().any(-1), bad) and torch.equal(res[1].isnan().all(-1), bad)
    assert torch.equal(res[0][~bad], res[1][~bad]) and not res[0].isnan().any()


@pytest.mark.parametrize("dtype,nh,nkv,hd,past", [(torch.bfloat16, 4, 2, 128, 0), (torch.bfloat16, 32, 2, 128, 3000), (torch.bfloat16, 4, 2, 128, 9000), (torch.bfloat16, 4, 2, 64, 70),
                                                  (torch.bfloat16, 4, 2, 32, 70), (torch.bfloat16, 4, 2, 96, 70), (torch.float32, 4, 2, 80, 70), (torch.float32, 4, 2, 32, 70)])
@pytest.mark.parametrize("window", [None, 50])
def test_portions_read_back_with_rows_that_are_not_finite(dtype, nh, nkv, hd, past, window):
    """The same where pages are read back: a row that is not finite shows in the tokens that see it and in no others."""
    from synaptix_b200 import ops
    new, G = 150, nh // nkv
    ks, vs = ([randn(past + new, nkv, hd, seed=i + 7 * w) for i in range(2)] for w in (1, 2))
    ks[0][past + 40, 0, 3], vs[1][past + 70, 1, 5] = math.inf, math.nan
    held = P.Held(ks, vs)
    got = ops.kv8_attention(randn(2 * new, nh * hd).to(dtype).cuda(), held.pages(), on_gpu(step([past + new] * 2, [new] * 2)), held.table.cuda(), nh, nkv, hd, 0.1, window)
    got = got.cpu().view(2, new, nh, hd)
    until = new if window is None else window
    bad = torch.zeros(2, new, nh, dtype=torch.bool)
    bad[0, 40:40 + until, :G] = bad[1, 70:70 + until, G:] = True
    assert torch.equal(got.isnan().any(-1), bad) and torch.equal(got.isnan().all(-1), bad)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale_k,scale_v,scale_q", [(1e-20, 1e20, 1e18), (1e15, 1e-30, 1e-16), (1e-8, 1e-8, 1.0)])
def test_portions_of_magnitudes_far_from_one(over_the_codes, dtype, scale_k, scale_v, scale_q):
    lens, new, nh, hd = [300, 70], [40, 70], 8, 128
    ks, vs = ([randn(n, 2, hd, seed=i + 7 * w) * f for i, n in enumerate(lens)] for w, f in ((1, scale_k), (2, scale_v)))
    check(randn(110, nh, hd) * scale_q, P.Held(ks, vs), lens, new, nh, hd, dtype, dtype == torch.bfloat16, scale=hd ** -0.5 / (scale_k * scale_q))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_portions_where_one_value_outweighs_all_others(over_the_codes, dtype):
    nh, hd = 4, 64
    ks, vs = randn(260, 1, hd, seed=1), randn(260, 1, hd, seed=2)
    ks[77] = -6.0                                                  # score -48 below zero: weight 1e-21
    vs[77] *= 2.0 ** 40
    check(torch.ones(120, nh, hd), P.Held([ks], [vs]), [260], [120], nh, hd, dtype, dtype == torch.bfloat16, scale=1 / 8)


def test_many_sequences_and_places_that_end_anywhere():
    """More pairs than blocks, pairs that end within a warp's stretch, empty sequences between: all rows of a batch against the same rows alone."""
    from synaptix_b200 import ops
    g = torch.Generator().manual_seed(5)
    nh, nkv, hd = 8, 4, 128
    lens = torch.randint(0, 400, (150,), generator=g).tolist()
    lens[3] = lens[4] = lens[149] = 0
    held = filled(lens, nkv, hd)
    q = (2 * randn(len(lens), nh, hd, seed=3)).bfloat16().view(len(lens), -1).cuda()
    pages, table = held.pages(), held.table.cuda()
    got = ops.kv8_attention(q, pages, on_gpu(step(lens, [1] * len(lens))), table, nh, nkv, hd, hd ** -0.5)
    for s in range(0, 150, 7):
        want, weight = P.attend(q[s:s + 1].cpu().view(1, nh, hd), held.keys[s], held.values[s], torch.tensor([lens[s] - 1]), hd ** -0.5) if lens[s] else (torch.zeros(1, nh * hd).double(),) * 2
        if lens[s] == 0:
            assert (got[s] == 0).all()
            continue
        tol = bound(q[s:s + 1].cpu().view(1, nh, hd), held, s, want, weight, None, hd ** -0.5, torch.bfloat16, hd, True)
        assert ((got[s].cpu().double() - want[0]).abs() <= tol[0]).all(), s
    again = ops.kv8_attention(q, pages, on_gpu(step(lens, [1] * len(lens))), table, nh, nkv, hd, hd ** -0.5)
    assert torch.equal(got, again)                                 # (no sum depends on which warp is first)


@pytest.mark.parametrize("nh,nkv,hd,dtype", [(32, 8, 128, torch.bfloat16), (8, 1, 64, torch.bfloat16), (24, 2, 128, torch.bfloat16), (4, 2, 96, torch.float32)])
def test_recorded_and_replayed(nh, nkv, hd, dtype):
    """A step of preparation and attention recorded once, replayed while the sequences grow, two graphs in turn and on two streams at once."""
    from synaptix_b200 import ops
    lens = [130, 700, 64]
    held = filled([n + 8 for n in lens], nkv, hd)
    pages, table = held.pages(), held.table.cuda()
    scale = hd ** -0.5

    class Step:
        def __init__(self, seed):
            self.ctx = on_gpu(step(lens, [1] * 3, host=None))
            self.ctx.max_len = table.shape[1] * 64
            self.pages = ops.KV8Pages(*(t.clone() for t in pages))
            self.qkv = torch.zeros(3, (nh + 2 * nkv) * hd, dtype=dtype, device="cuda")
            self.q = torch.zeros(3, nh * hd, dtype=dtype, device="cuda")
            self.run()
            torch.cuda.synchronize()
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self.out = self.run()
            self.rows = [randn(3, (nh + 2 * nkv) * hd, seed=seed + i).to(dtype).cuda() for i in range(4)]

        def run(self):
            ops.kv8_prepare(self.qkv, self.q, self.pages, None, None, None, 0, 0.0, self.ctx.positions, self.ctx.seq_of_token, table, nh, nkv, hd)
            return ops.kv8_attention(self.q, self.pages, self.ctx, table, nh, nkv, hd, scale)

        def at(self, i):
            self.qkv.copy_(self.rows[i])
            self.ctx.seq_lens.copy_(torch.tensor([n + i for n in lens], dtype=torch.int32))
            self.ctx.positions.copy_(torch.tensor([n + i - 1 for n in lens], dtype=torch.int32))

    a, b = Step(10), Step(20)
    want = []
    for s in (a, b):
        for i in range(4):
            s.at(i)
            want.append(s.run().clone())
    assert not torch.equal(a.pages.k, b.pages.k)
    for i in range(4):                                             # in turn
        for s, w in ((a, want[i]), (b, want[4 + i])):
            s.at(i)
            s.graph.replay()
            assert torch.equal(s.out, w)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in (3, 0, 2):                                            # at once
        for s in (a, b):
            s.at(i)
        torch.cuda.synchronize()
        for _ in range(5):
            for s, st in zip((a, b), streams):
                with torch.cuda.stream(st):
                    s.graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a.out, want[i]) and torch.equal(b.out, want[4 + i])


def test_what_is_not_contiguous_or_aligned():
    from synaptix_b200 import ops
    nh, nkv, hd, lens = 8, 2, 64, [200]
    held = filled(lens, nkv, hd)
    pages, table, ctx = held.pages(), held.table.cuda(), on_gpu(step(lens, [1]))
    wide = randn(1, 2 * nh * hd).bfloat16().cuda()
    with pytest.raises(ops.KernelError, match="contiguous"):
        ops.kv8_attention(wide[:, ::2], pages, ctx, table, nh, nkv, hd, 0.1)
    # (a row of a larger tensor that begins anywhere is fine for the heads' preparation, and refused where 16 bytes are loaded at once)
    odd = wide.view(-1)[1:1 + nh * hd].view(1, -1)
    with pytest.raises(ops.KernelError, match="misaligned"):
        ops.kv8_attention(odd, pages, ctx, table, nh, nkv, hd, 0.1)
    x = randn(70, 1 + (nh + 2 * nkv) * hd).bfloat16()
    held = empty([70], nkv, hd)
    q, got = prepare(x, held, torch.arange(70), torch.zeros(70), nh, nkv, hd, col=1)
    assert torch.equal(q, x[:, 1:1 + nh * hd])
    kc, _, _ = P.quantise(x[:, 1 + nh * hd:1 + (nh + nkv) * hd].reshape(70, nkv, hd))
    assert torch.equal(written(got, held, 0, 69, nkv, hd)[0], kc[69])


# ---- as a model uses them

def held_rows(engine, slot, layer, n):
    """Keys and values that the engine's cache holds of a sequence, as the doubles they stand for (NaN where a window gave the page back)."""
    view = engine.cache.view(layer)
    table = engine.cache.slots.table(slot, view.group)[:-(-n // 64)]
    at = torch.tensor([max(p, 0) for p in table], device="cuda")
    k, v, ke, ve = (t[at].cpu() for t in (view.pages8.k, view.pages8.v, view.pages8.k_exp, view.pages8.v_exp))
    power = [torch.exp2(e.double() - 127).transpose(1, 2).reshape(-1, e.shape[1], 1) for e in (ke, ve)]
    k = k.view(torch.float8_e4m3fn).double().permute(0, 3, 1, 2, 4).flatten(3).flatten(0, 1)
    v = v.view(torch.float8_e4m3fn).double().permute(0, 3, 1, 2).flatten(0, 1)
    gone = torch.tensor([p < 0 for p in table]).repeat_interleave(64)[:, None, None]
    return tuple(torch.where(gone, math.nan, x)[:n] for x in (k * power[0], v * power[1]))


def oracle8(name, tokens, held, slack):
    """The plain decoder whose attention reads the keys and values that the engine holds, each checked on the way: it is the plain decoder's own,
    rounded to eight bits (by at most half a step: 2^-4 of itself, or 2^-10 of the row's power of two, which is at most a / 224), where that
    is off by ``slack`` of the row's largest ahead of its rounding."""
    cfg, W = Q.load_folder(folder(name))
    whole, layer = Q.causal_gqa_attention, iter(range(1000))

    def attention(q, k, v, *a, **kw):
        rows = [torch.where(got.isnan(), P.quantise(own)[2], got) for got, own in zip(held[next(layer)], (k, v))]
        for got, own in zip(rows, (k, v)):
            top = own.double().abs().amax(-1, keepdim=True)
            assert ((got - own).abs() <= own.abs() * 2.0 ** -4 + top * (2.0 ** -10 / 224 + slack * (1 + 2.0 ** -4))).all()
        return whole(q, rows[0].float(), rows[1].float(), *a, **kw)
    Q.causal_gqa_attention = attention
    try:
        return Q.forward(cfg, W, list(tokens))
    finally:
        Q.causal_gqa_attention = whole


@pytest.mark.parametrize("name", ["A", "F", "O", "B", "W", "S", "G"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("graph", [True, False])
def test_engine(name, dtype, graph):
    """A prompt whole, in portions and token by token, against the plain decoder.  (An element that lies within its own error of the border
    between two e4m3 numbers may fall on either side of it, so the plain decoder is given what the cache holds.)"""
    import synaptix_b200
    from synaptix_b200.engine import Entry
    engine = synaptix_b200.LLM(folder(name), compute_dtype=dtype, max_tokens=1024, kv_dtype="fp8", graph=graph).engine
    tokens = random_tokens(engine.model.vocab_size, 150, 5)
    cfg, W = Q.load_folder(folder(name))
    full = Q.forward(cfg, W, list(tokens))
    for cuts in ([150], [70, 80], [64, 1, 1, 84], [140] + [1] * 10):
        s, at, rows = engine.open(), 0, []
        for n in cuts:
            rows.append(engine.step([Entry(s, tokens[at:at + n], list(range(n)))]).clone())
            at += n
        held = [held_rows(engine, s, i, 150) for i in range(cfg["num_hidden_layers"])]
        engine.close(s)
        rel = F32_REL if dtype == "f32" else BF16_REL
        want = oracle8(name, tokens, held, rel)
        scale = want.abs().max().item()
        assert (full - want).abs().max().item() > 1e-3 * scale      # eight bits show
        off = (torch.cat(rows).cpu() - want).abs().max().item() / scale
        assert off <= rel, (cuts, off)


def test_a_decoder_of_other_parts():
    """The Vemedra decoder (chunks, capped scores and sinks beside retention): where its keys and values have one size its cache may be in eight bits, and
    a prompt gives the same whole, in portions and token by token; where they have not, the engine says so."""
    import synaptix_b200
    import tiny_vemedra as V
    took = 0
    for name in V.CONFIGS:
        try:
            engine = synaptix_b200.LLM(V.folder(name), compute_dtype="f32", max_tokens=1024, kv_dtype="fp8").engine
        except ValueError as e:
            assert "eight bits" in str(e)
            continue
        took += 1
        tokens = random_tokens(engine.model.vocab_size, 150, 5)
        want = V.oracle_logits(name, tuple(tokens))
        scale = want.abs().max().item()
        from synaptix_b200.engine import Entry
        for cuts in ([150], [70, 80], [140] + [1] * 10):
            s, at, rows = engine.open(), 0, []
            for n in cuts:
                rows.append(engine.step([Entry(s, tokens[at:at + n], list(range(n)))]).clone())
                at += n
            engine.close(s)
            off = (torch.cat(rows).cpu() - want).abs().max().item() / scale
            # eight bits move an element of a key or value by 2^-4 of itself: half of that on average, mostly lost in sums of many
            assert 1e-6 < off < 2.0 ** -4, (name, cuts, off)
    assert took == 1


def test_generation_and_conversation():
    import synaptix_b200
    llm = synaptix_b200.LLM(folder("A"), compute_dtype="f32", max_tokens=2048, kv_dtype="fp8")
    wide = synaptix_b200.LLM(folder("A"), compute_dtype="f32", max_tokens=2048)
    assert llm.kv_bytes_per_token < wide.kv_bytes_per_token / 3
    prompts = [random_tokens(llm.vocab_size, n, n) for n in (5, 70, 130)]
    together = llm.generate(prompts, max_new_tokens=12, eos_token_ids=[])
    assert together == [llm.generate([p], max_new_tokens=12, eos_token_ids=[])[0] for p in prompts]
    assert together == llm.generate(prompts, max_new_tokens=12, eos_token_ids=[], prefill_batch=32)
    with llm.conversation() as chat:
        a = chat.generate(prompts[1], max_new_tokens=4, eos_token_ids=[])
        b = chat.generate(prompts[1] + a + [3, 4], max_new_tokens=4, eos_token_ids=[])
    assert b == llm.generate([prompts[1] + a + [3, 4]], max_new_tokens=4, eos_token_ids=[])[0]
