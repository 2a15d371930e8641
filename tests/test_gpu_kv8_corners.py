"""Attention over a cache in eight bits where its parts meet: rows that are not finite at the border of a stretch of keys, values and keys at the
format's smallest and largest powers, places nobody sees, a context that comes back with other lengths.  Bounds as in ``test_gpu_kv8``."""
import importlib
import math

import pytest
import torch

import plain_kv8 as P
from test_gpu_kv8 import bound, check, filled, on_gpu, over_the_codes, randn  # noqa: F401
from test_kv8_cpu import step
from test_kv8_corners_cpu import comes_back

pytestmark = pytest.mark.gpu


def attend(q, held, ctx, nh, nkv, hd, scale, window=None, **kw):
    from synaptix_b200 import ops
    return ops.kv8_attention(q.view(q.shape[0], -1).cuda(), held.pages(), on_gpu(ctx), held.table.cuda(), nh, nkv, hd, scale, window, **kw).cpu().view(-1, nh, hd)


@pytest.fixture
def read_back(monkeypatch):
    """All portions go through pages read back, whatever is faster."""
    from synaptix_b200.ops import kv8
    monkeypatch.setattr(kv8, "FEW_NEW_TOKENS", 0)
    for name in ("TILE_BF16_ROWS", "TILE_BF16_PAGES"):
        monkeypatch.setattr(kv8, name, {64: 0, 128: 0})


# ---- cut tiles (csrc/attn_tc.cu)

@pytest.mark.parametrize("what", ["key", "value"])
@pytest.mark.parametrize("sinks", [False, True])
def test_a_row_that_is_not_finite_begins_a_stretch_of_keys(what, sinks):
    """The first key of a stretch is the only one that its own token sees there."""
    from synaptix_b200.ops.attention import tc_parts
    past, new, nh, nkv, hd = 9156, 150, 4, 2, 128
    tiles = [(past + q0, min(past + q0 + 128, past + new) - 1) for _ in range(2) for q0 in (0, 128)]
    chunk, parts = tc_parts(tiles, nh, None, torch.device("cuda", 0))
    token = 60
    assert parts > 1 and (past + token) % (chunk * 128) == 0
    ks, vs = ([randn(past + new, nkv, hd, seed=i + 7 * w) for i in range(2)] for w in (1, 2))
    q, s, res = randn(2 * new, nh, hd).bfloat16(), randn(nh, seed=9).cuda() if sinks else None, []
    for spoil in (False, True):
        if spoil:
            (ks if what == "key" else vs)[1][past + token, 1, 5] = math.nan
        res.append(attend(q, P.Held(ks, vs), step([past + new] * 2, [new] * 2), nh, nkv, hd, 0.1, sinks=s).view(2, new, nh, hd))
    bad = torch.zeros(2, new, nh, dtype=torch.bool)
    bad[1, token:, 2:] = True
    assert torch.equal(res[1].isnan().any(-1), bad) and torch.equal(res[1].isnan().all(-1), bad)
    assert torch.equal(res[0][~bad], res[1][~bad]) and not res[0].isnan().any()


@pytest.mark.parametrize("window", [None, 130, 200])
def test_rows_that_are_not_finite_in_short_stretches(monkeypatch, window):
    """Stretches of 128 keys: spoiled keys at the first and the last place of a stretch, so that a window's lower end leaves that one key of it, and
    one among keys whose weights are nothing beside the others'."""
    cut = []
    monkeypatch.setattr(importlib.import_module("synaptix_b200.ops.attention"), "tc_parts", lambda *a: cut.append(1) or (1, 6))
    past, new, nh, nkv, hd = 500, 150, 16, 2, 128
    n = past + new
    ks, vs = ([randn(n, nkv, hd, seed=i + 7 * w) for i in range(4)] for w in (1, 2))
    q = randn(4 * new, nh, hd).bfloat16()
    q[3 * new:] = 1.0
    ks[3][:128], ks[3][128:] = -4.0, 0.0                           # scores of -256 and 0: weights of 2^-369 and 1
    spoiled = [512, 511, 383, 77]
    res = []
    for spoil in (False, True):
        if spoil:
            for s, j in enumerate(spoiled):
                (vs if s == 2 else ks)[s][j, 0, 3] = math.inf
        res.append(attend(q, P.Held(ks, vs), step([n] * 4, [new] * 4), nh, nkv, hd, 0.5, window).view(4, new, nh, hd))
    pos = torch.arange(past, n)
    bad = torch.zeros(4, new, nh, dtype=torch.bool)
    for s, j in enumerate(spoiled):
        bad[s, :, :8] = ((pos >= j) & (pos - (window or n) < j))[:, None]
    assert cut and torch.equal(res[1].isnan().any(-1), bad) and torch.equal(res[1].isnan().all(-1), bad)
    assert torch.equal(res[0][~bad], res[1][~bad]) and not res[0].isnan().any()


@pytest.mark.parametrize("sinks", [False, True])
def test_a_long_tile_among_many_short_ones_takes_no_room_for_them(sinks):
    """64 tokens behind 12,000 keys are cut; the 20 prompts beside them are not, and need no room for stretches."""
    from synaptix_b200 import ops
    lens, new, nh, nkv, hd = [12064] + [300] * 20, [64] + [300] * 20, 16, 2, 128
    held, q, s = filled(lens, nkv, hd), (2 * randn(sum(new), nh, hd, seed=3)).bfloat16(), randn(nh, seed=9) if sinks else None
    ctx, pages, table, x = on_gpu(step(lens, new)), held.pages(), held.table.cuda(), q.view(q.shape[0], -1).cuda()
    sink = None if s is None else s.cuda()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = ops.kv8_attention(x, pages, ctx, table, nh, nkv, hd, 0.1, sinks=sink)
    torch.cuda.synchronize()
    cut = ctx.scratch[("kv8_parts", nh, None)]
    assert cut[1] > 1
    read = 2 * sum(-(-n // 64) for n in lens) * nkv * 64 * hd * 2
    sums = cut[1] * 64 * nh * (hd + 4) * 4
    assert torch.cuda.max_memory_allocated() - before <= read + got.numel() * 2 + sums + (1 << 20)
    for i in (0, 1, 20):
        at = sum(new[:i])
        part, n, m = slice(at, at + new[i]), lens[i], new[i]
        want, weight = P.attend(q[part], held.keys[i], held.values[i], torch.arange(n - m, n), 0.1, sinks=s)
        tol = bound(q[part], held, i, want, weight, None, 0.1, torch.bfloat16, hd, True, portions=True)
        assert ((got[part].cpu().double() - want).abs() <= tol).all(), i


@pytest.mark.parametrize("new", [[700], [300, 400]])
@pytest.mark.parametrize("nh,nkv,hd", [(32, 8, 128), (64, 8, 64)])
def test_the_first_layer_of_a_step_takes_the_kernel_that_the_others_take(read_back, new, nh, nkv, hd):
    """What the first call makes for its context changes nothing but the time: the same bits from all calls, and those of the kernel itself."""
    from synaptix_b200 import ops
    held, q, ctx = filled(new, nkv, hd), (2 * randn(sum(new), nh, hd, seed=3)).bfloat16(), step(new, new)
    first, second = (attend(q, held, ctx, nh, nkv, hd, 0.1) for _ in range(2))
    k, v, table = ops.kv8_read(held.pages(), ctx, held.table.cuda(), torch.bfloat16)
    tiles = ops._query_tiles(ctx, 128 if hd == 128 else 64, k.device)
    whole = (ops.attn_prefill_tc if hd == 128 else ops.attn_prefill)(q.view(sum(new), -1).cuda(), k, v, *tiles, ctx.cu_seqlens, ctx.seq_past, ctx.seq_lens, table,
                                                                     nh, nkv, hd, 0.1, None)
    assert torch.equal(first, second) and torch.equal(first, whole.cpu().view(first.shape))


# ---- the format's ends

def values_of_exponents(lens, nkv, hd, exponents, seed=0):
    """Sequences whose value rows have these exponent bytes in turn."""
    held = filled(lens, nkv, hd, seed=seed, loud=False)
    vs = []
    for s, n in enumerate(lens):
        x = torch.clamp(randn(n, nkv, hd, seed=seed + 50 + s) / 4, -1, 1).double()
        x[..., 3] = 1.0
        e = torch.tensor(exponents)[torch.arange(n) % len(exponents)]
        vs.append((x * torch.exp2(e.double() - 127 + 8)[:, None, None]).float())       # a row of largest magnitude 2^x has e - 127 = x - 8
    ks = [k.float() for k in held.keys]
    held = P.Held(ks, vs, seed=seed)
    for s, n in enumerate(lens):
        for j in range(min(n, len(exponents))):
            assert int(held.v_exp[int(held.table[s, j // 64]), 0, j % 64]) == exponents[j]
    return held


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("exponents", [[e] for e in range(10, 18)] + [[10, 15], [10, 12, 30], [11, 127]])
@pytest.mark.parametrize("lens,new", [([40], [40]), ([2000, 70], [20, 12])])
def test_portions_over_values_at_the_formats_lower_end(over_the_codes, dtype, exponents, lens, new):  # noqa: F811
    nh, nkv, hd = 8, 2, 64
    check(2 * randn(sum(new), nh, hd, seed=3), values_of_exponents(lens, nkv, hd, exponents), lens, new, nh, hd, dtype, dtype == torch.bfloat16)


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 64), (torch.bfloat16, 96), (torch.float32, 64)])
@pytest.mark.parametrize("exponents", [[10], [12], [16], [10, 30]])
def test_single_tokens_over_values_at_the_formats_lower_end(dtype, hd, exponents):
    lens, nh, nkv = [40, 700], 8, 2
    check(2 * randn(2, nh, hd, seed=3), values_of_exponents(lens, nkv, hd, exponents), lens, [1, 1], nh, hd, dtype, dtype == torch.bfloat16)


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 64), (torch.bfloat16, 256), (torch.float32, 128)])
def test_single_tokens_over_keys_at_the_formats_upper_end(dtype, hd):
    """Keys of up to 3e38 and queries so small that scores are ordinary: codes times query elements times the power alone would pass float32's range."""
    lens, nh, nkv = [300, 70], 8, 2
    ks, vs = ([randn(n, nkv, hd, seed=i + 7 * w) for i, n in enumerate(lens)] for w in (1, 2))
    for k in ks:
        k.clamp_(-1, 1).mul_(3e38)
    scale = hd ** -0.5 * 2.0 ** -31                                # (powers of two beside the queries', which bfloat16 products hold from 2^-99 on)
    check(randn(2, nh, hd) * 2.0 ** -97, P.Held(ks, vs), lens, [1, 1], nh, hd, dtype, dtype == torch.bfloat16, scale=scale)


# ---- a context that comes back

@pytest.mark.parametrize("dtype,nh,nkv,hd,cut", [(torch.bfloat16, 32, 2, 128, False), (torch.bfloat16, 32, 2, 128, True), (torch.bfloat16, 64, 2, 64, False),
                                                 (torch.bfloat16, 4, 2, 96, False), (torch.float32, 4, 2, 80, False)])
def test_a_context_that_comes_back_with_other_portions(monkeypatch, dtype, nh, nkv, hd, cut):
    """As many tokens in all, dealt to the sequences in another way: what the first call made for the context is made anew."""
    from synaptix_b200 import ops
    module = importlib.import_module("synaptix_b200.ops.attention")
    if cut:
        monkeypatch.setattr(module, "tc_parts", lambda *a: (2, 6))
    read, reads = ops.kv8._read, []
    monkeypatch.setattr(ops.kv8, "_read", lambda *a: reads.append(1) or read(*a))
    ctx, scale = None, hd ** -0.5
    for lens, new in (([700, 1200], [150, 280]), ([800, 1100], [280, 150]), ([430, 900], [429, 1])):
        held = filled(lens, nkv, hd, seed=lens[0])
        ctx = step(lens, new) if ctx is None else comes_back(ctx, lens, new)
        q = (2 * randn(sum(new), nh, hd, seed=3)).to(dtype)
        got = attend(q, held, ctx, nh, nkv, hd, scale)
        assert torch.equal(got, attend(q, held, step(lens, new), nh, nkv, hd, scale))
        at = 0
        for s, (n, m) in enumerate(zip(lens, new)):
            part = slice(at, at + m)
            at += m
            want, weight = P.attend(q[part], held.keys[s], held.values[s], torch.arange(n - m, n), scale)
            tol = bound(q[part], held, s, want, weight, None, scale, dtype, hd, dtype == torch.bfloat16, portions=True)
            assert ((got[part].reshape(m, -1).double() - want).abs() <= tol).all(), (lens, s)
    assert len(reads) == 6


# ---- places that nobody sees

def littered(lens, new, nkv, hd, window=None, chunk=None, seed=0):
    """Sequences where the places that no token of the step sees hold arbitrary codes and exponents: NaN codes, powers up to 2^127."""
    held = filled(lens, nkv, hd, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    for s, (n, m) in enumerate(zip(lens, new)):
        p = n - m
        first = max(max(0, p - window + 1) if window else 0, p // chunk * chunk if chunk else 0)
        for j in [*range(first), *range(n, -(-n // 64) * 64)]:
            page, r = int(held.table[s, j // 64]), j % 64
            for t in (held.k, held.v, held.k_exp, held.v_exp):
                where = t[page, :, :, r] if t is held.k else t[page, ..., r]
                where.copy_(torch.randint(0, 256, where.shape, generator=g).byte())
            held.v[page, :, ::3, r] = 0x7f if j % 2 else 0xff
            held.v_exp[page, :, r] = 100 + (j * 7) % 155
    return held


OPTIONS = [{}, dict(window=50), dict(window=64), dict(window=200, chunk=96)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("options", OPTIONS)
def test_portions_over_the_codes_beside_places_nobody_sees(over_the_codes, dtype, hd, options):  # noqa: F811
    lens, new, nh, nkv = [300, 131, 1000], [33, 20, 100], 8, 2
    held = littered(lens, new, nkv, hd, **options)
    check(2 * randn(sum(new), nh, hd, seed=3), held, lens, new, nh, hd, dtype, dtype == torch.bfloat16, **options)


@pytest.mark.parametrize("dtype,nh,nkv,hd", [(torch.bfloat16, 8, 2, 128), (torch.bfloat16, 8, 2, 64), (torch.bfloat16, 4, 2, 32), (torch.bfloat16, 4, 2, 96),
                                             (torch.float32, 4, 2, 80), (torch.float32, 4, 2, 32)])
@pytest.mark.parametrize("options", OPTIONS)
def test_portions_read_back_beside_places_nobody_sees(read_back, dtype, nh, nkv, hd, options):
    lens, new = [300, 131, 1000], [33, 20, 100]
    held = littered(lens, new, nkv, hd, **options)
    check(2 * randn(sum(new), nh, hd, seed=3), held, lens, new, nh, hd, dtype, dtype == torch.bfloat16, **options)


def test_cut_tiles_beside_places_nobody_sees(read_back):
    lens, new, nh, nkv, hd = [6000, 300], [70, 300], 16, 2, 128
    options = dict(window=4500)
    check(2 * randn(sum(new), nh, hd, seed=3), littered(lens, new, nkv, hd, **options), lens, new, nh, hd, torch.bfloat16, True, **options)


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.bfloat16, 96), (torch.float32, 64)])
@pytest.mark.parametrize("new", [[1, 1, 1], [2, 8, 1]])
@pytest.mark.parametrize("options", OPTIONS)
def test_a_few_tokens_beside_places_nobody_sees(dtype, hd, new, options):
    lens, nh, nkv = [300, 131, 1000], 8, 2
    held = littered(lens, new, nkv, hd, **options)
    check(2 * randn(sum(new), nh, hd, seed=3), held, lens, new, nh, hd, dtype, dtype == torch.bfloat16, **options)
