"""Operators of a cache in eight bits, for measuring them: heads prepared and quantised as they are written into the cache,
the cache read back, and the attention that reads it, for single tokens and for portions of prompts.

A token's key (or value) of a head is held as one exponent byte ``e`` and ``hd`` e4m3 codes ``c``, and stands for
``c * 2^(e - 127)``.  With ``a`` the largest magnitude of the row, ``2^(e - 127)`` is the smallest power of two with
``a <= 448 * 2^(e - 127)``, kept in ``2^-117 .. 2^119``; codes are rounded to nearest even.  ``e = 255`` says that the row
was not finite.  Pages hold 64 tokens of all kv heads: keys as ``[pages, kv heads, hd / B, 64, B]`` (blocks of
``B = 64`` elements, of 32 or 16 where 64 does not divide ``hd``), values as ``[pages, kv heads, hd, 64]``, exponents as
``[pages, kv heads, 64]``.

Rows of a page behind a sequence's last token hold what an earlier sequence left there: here exponents that say "not
finite", which must show nowhere.  Pages lie in random order and page 0 belongs to nobody, as in the cache.
"""
import math
import random
import types

import torch

own = False

PAGE = 64
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    def case(name, op, seqs, past, new, nh=32, nkv=8, hd=128, dtype="bf16", window=0, sinks=False, norm=True):
        return {"name": name, "op": op, "seqs": seqs, "past": past, "new": new, "nh": nh, "nkv": nkv, "hd": hd, "dtype": dtype,
                "window": window, "sinks": sinks, "norm": norm}
    return [
        # heads of one user's next token: norm, rotation, eight bits; nothing but latency
        case("prepare_token", "prepare", 1, 1500, 1),
        # heads of a busy server's step, one token a sequence
        case("prepare_step_b48", "prepare", 48, 2000, 1),
        # a long document's heads
        case("prepare_prompt_8191", "prepare", 1, 0, 8191),
        # a short conversation read back (its next message is a prompt portion over it)
        case("read_chat", "read", 1, 611, 0),
        # several long conversations of unequal lengths read back
        case("read_batch", "read", 8, 12000, 0),
        # one user, a short context: launches and latency
        case("single_b1_short", "single", 1, 300, 1),
        # the benchmark's batch and context
        case("single_b8", "single", 8, 4096, 1),
        # a busy server whose layer sees a window of its keys, with a sink per head
        case("single_b64_window", "single", 64, 6000, 1, nh=64, nkv=8, hd=64, window=1000, sinks=True),
        # one user with a very long document
        case("single_b1_long", "single", 1, 131071, 1),
        # the benchmark's prompt
        case("portion_2048", "portion", 1, 0, 2048),
        # next messages of several users, over what the cache holds of each
        case("portion_ragged", "portion", 5, 9000, 127),
        # the 32-bit path: two short prompts
        case("portion_f32", "portion", 2, 40, 150, nh=16, dtype="f32"),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    op = rng.choice(["prepare", "read", "single", "single", "portion"])
    nkv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 4, 5, 8])
    dtype = "f32" if rng.random() < 0.2 else "bf16"
    case = {"op": op, "nh": nkv * group, "nkv": nkv, "hd": rng.choice([64, 128, 128]), "dtype": dtype, "window": 0, "sinks": rng.random() < 0.25,
            "norm": rng.random() < 0.7}
    if op == "prepare":
        new = rng.choice([1, log_int(2, 6000)])
        case.update(seqs=log_int(1, 64) if new == 1 else 1, past=log_int(1, 100000 if new > 1 else 4000), new=new, hd=rng.choice([32, 64, 96, 128, 128]))
    elif op == "read":
        seqs = log_int(1, 16)
        case.update(seqs=seqs, past=log_int(20, 60000 // seqs), new=0, hd=rng.choice([32, 64, 96, 128, 128]))
    elif op == "single":
        seqs = log_int(1, 64)
        past = log_int(30, 100000 // seqs)
        case.update(seqs=seqs, past=past, new=1, window=log_int(20, past) if rng.random() < 0.25 else 0, hd=rng.choice([32, 64, 96, 128, 128, 128]))
    else:
        seqs = log_int(1, 6)
        new = log_int(2, 1500 // seqs)
        past = rng.choice([0, log_int(1, 6000)])
        case.update(seqs=seqs, new=new, past=past, window=log_int(20, past + new) if rng.random() < 0.25 else 0)
    return case


def lengths(case):
    """``(past, new)`` of each sequence: the first has the case's own, the others are shorter by an amount that the sizes fix."""
    rng = random.Random(case["seqs"] * 1000003 + case["past"] * 101 + case["new"])
    past = [case["past"]] + [int(case["past"] * rng.uniform(0.3, 1.0)) for _ in range(case["seqs"] - 1)]
    new = [case["new"]] + [max(1, int(case["new"] * rng.uniform(0.5, 1.0))) if case["new"] else 0 for _ in range(case["seqs"] - 1)]
    return past, new


def block(hd):
    return 64 if hd % 64 == 0 else 32 if hd % 32 == 0 else 16


def power(e):
    """``2^(e - 127)`` of exponent bytes, NaN for 255."""
    return torch.where(e == 255, torch.full_like(e, 0x7fc00000, dtype=torch.int32), e.to(torch.int32) << 23).view(torch.float32)


def quantise(x):
    """``x [..., hd]`` float32 as ``(codes uint8 [..., hd], exponents uint8 [...])``."""
    a = x.abs().amax(-1)
    bits = a.view(torch.int32)
    e = (bits >> 23) - torch.where((bits & 0x7fffff) <= 0x600000, 8, 7)
    e = torch.where(a == 0, 10, e.clamp(10, 246))
    finite = torch.isfinite(x).all(-1)
    inverse = ((254 - e) << 23).to(torch.int32).view(torch.float32)
    y = torch.where(finite[..., None], x * inverse[..., None], 0.0).clamp(-448.0, 448.0)
    return y.to(torch.float8_e4m3fn).view(torch.uint8), torch.where(finite, e, 255).to(torch.uint8)


def prepare(case, seed):
    past, new = lengths(case)
    S, nh, nkv, hd, op = case["seqs"], case["nh"], case["nkv"], case["hd"], case["op"]
    dtype, dev = DTYPES[case["dtype"]], "cuda"
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    host = random.Random(seed)
    lens = [p + n for p, n in zip(past, new)]
    pages = [-(-n // PAGE) for n in lens]
    order = list(range(1, sum(pages) + 1))
    host.shuffle(order)
    W = max(pages)
    tables, at = torch.zeros((S, W), dtype=torch.int32), 0
    for s, n in enumerate(pages):
        tables[s, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    n_pages = len(order) + 1
    tables = tables.to(dev)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    T = sum(new)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    seq = [s for s in range(S) for _ in range(new[s])]
    pos = [past[s] + i for s in range(S) for i in range(new[s])]

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=dev)

    B = block(hd)
    state = {"case": dict(case), "lens": lens, "n_pages": n_pages}
    k = torch.empty((n_pages, nkv, hd // B, PAGE, B), dtype=torch.uint8, device=dev)
    v = torch.empty((n_pages, nkv, hd, PAGE), dtype=torch.uint8, device=dev)
    ke = torch.full((n_pages, nkv, PAGE), 255, dtype=torch.uint8, device=dev)
    ve = torch.full((n_pages, nkv, PAGE), 255, dtype=torch.uint8, device=dev)
    if op == "prepare":
        k.zero_()
        v.zero_()
    else:
        # what lies where a sequence's tokens are; the rest of its last page is an earlier sequence's
        held = torch.zeros((n_pages, PAGE), dtype=torch.bool, device=dev)
        places = torch.arange(W * PAGE, device=dev)[None, :] < ints(lens)[:, None]
        held[tables.long()] = places.view(S, W, PAGE)
        held[0] = False
        level = torch.exp(0.5 * randn(nkv, 1, 1))                # heads of unlike size
        for first in range(0, n_pages, 2048):
            part = slice(first, min(first + 2048, n_pages))
            n = part.stop - part.start
            loud = 1.0 + 4.0 * (torch.rand((1, nkv, PAGE, 1), generator=gen, device=dev) < 0.05)       # some tokens' keys and values are larger
            c, e = quantise(randn(n, nkv, PAGE, hd))
            k[part] = c.view(n, nkv, PAGE, hd // B, B).transpose(2, 3)
            ke[part] = torch.where(held[part, None, :], e, 255)
            c, e = quantise(randn(n, nkv, PAGE, hd) * level * loud)
            v[part] = c.transpose(2, 3)
            ve[part] = torch.where(held[part, None, :], e, 255)
    state.update(k=k, v=v, k_exp=ke, v_exp=ve, table=tables)
    state["sinks"] = randn(nh) if case["sinks"] and op in ("single", "portion") else None
    if op == "prepare":
        state["qkv"] = (randn(T, (nh + 2 * nkv) * hd) * torch.exp(0.5 * randn(1, nh + 2 * nkv, 1)).expand(1, -1, hd).reshape(1, -1)).to(dtype)
        state["wq"], state["wk"] = (1.0 + 0.1 * randn(hd), 1.0 + 0.1 * randn(hd)) if case["norm"] else (None, None)
        state["inv_freq"] = torch.tensor([1e6 ** (-2.0 * i / hd) for i in range(hd // 2)], dtype=torch.float64).to(torch.float32).to(dev) if case["norm"] else None
        state["q_out"] = torch.empty((T, nh * hd), dtype=dtype, device=dev)
    elif op != "read":
        state["q"] = (2.0 * randn(T, nh * hd)).to(dtype)          # normed heads with a gain: a few keys stand out
    state["ctx"] = types.SimpleNamespace(
        n_tokens=T, n_seqs=S, max_new=max(max(new), 1), max_len=max(lens), all_single=op == "single", cu_seqlens=ints(cu), seq_past=ints(past),
        seq_lens=ints(lens), positions=ints(pos), seq_of_token=ints(seq), scratch={},
        host={"cu_seqlens": cu, "seq_past": past, "seq_lens": lens})
    return state


def run(state):
    if own:
        return run_own(state)
    return {"prepare": plain_prepare, "read": plain_read, "single": plain_single, "portion": plain_portion}[state["case"]["op"]](state)


def run_own(state):
    from synaptix_b200 import ops
    c, ctx = state["case"], state["ctx"]
    pages = ops.KV8Pages(state["k"], state["v"], state["k_exp"], state["v_exp"])
    if c["op"] == "prepare":
        ops.kv8_prepare(state["qkv"], state["q_out"], pages, state["wq"], state["wk"], state["inv_freq"],
                        c["hd"] if c["norm"] else 0, 1e-6, ctx.positions, ctx.seq_of_token, state["table"], c["nh"], c["nkv"], c["hd"])
        return written(state)
    if c["op"] == "read":
        k, v, _ = ops.kv8_read(pages, ctx, state["table"], DTYPES[c["dtype"]])
        return k, v
    return ops.kv8_attention(state["q"], pages, ctx, state["table"], c["nh"], c["nkv"], c["hd"], c["hd"] ** -0.5, c["window"] or None,
                             sinks=state["sinks"])


def written(state):
    """The prepared queries, and the cache as the values it holds: e4m3 codes and their rows' powers of two."""
    return {"q": state["q_out"], "k": state["k"].view(torch.float8_e4m3fn), "v": state["v"].view(torch.float8_e4m3fn),
            "k_exp": state["k_exp"].view(torch.float8_e8m0fnu), "v_exp": state["v_exp"].view(torch.float8_e8m0fnu)}


# ---- the plain forms

def plain_prepare(state):
    c, ctx = state["case"], state["ctx"]
    nh, nkv, hd = c["nh"], c["nkv"], c["hd"]
    x = state["qkv"].float().view(-1, nh + 2 * nkv, hd)
    qk, v = x[:, :nh + nkv], x[:, nh + nkv:]
    if c["norm"]:
        gain = torch.cat([state["wq"].expand(nh, hd), state["wk"].expand(nkv, hd)])
        qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + 1e-6) * gain
        angle = ctx.positions.double()[:, None] * state["inv_freq"].double()
        cos, sin = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
        a, b = qk[..., :hd // 2], qk[..., hd // 2:]
        qk = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    state["q_out"].copy_(qk[:, :nh].reshape(-1, nh * hd))
    page = state["table"][ctx.seq_of_token.long(), (ctx.positions // PAGE).long()].long()
    row = (ctx.positions % PAGE).long()
    codes, exps = quantise(qk[:, nh:])
    state["k"][page, :, :, row] = codes.view(-1, nkv, hd // block(hd), block(hd))
    state["k_exp"][page, :, row] = exps
    codes, exps = quantise(v)
    state["v"][page, :, :, row] = codes
    state["v_exp"][page, :, row] = exps
    return written(state)


def keys_of(state, at):
    """Keys of the pages ``at [...]`` as float32 ``[..., kv heads, 64, hd]``."""
    c = state["k"][at].view(torch.float8_e4m3fn).float().transpose(-3, -2).flatten(-2)
    return c * power(state["k_exp"][at])[..., None]


def values_of(state, at):
    c = state["v"][at].view(torch.float8_e4m3fn).float().transpose(-2, -1)
    return c * power(state["v_exp"][at])[..., None]


def plain_read(state):
    c, ctx = state["case"], state["ctx"]
    places = torch.arange(state["table"].shape[1] * PAGE, device="cuda")[None, :] < ctx.seq_lens[:, None]
    rows = places.view(c["seqs"], -1, PAGE)
    mine = rows[..., 0]
    at, rows = state["table"][mine].long(), rows[mine][:, None, :, None]
    return tuple(torch.where(rows, f(state, at), 0.0).to(DTYPES[c["dtype"]]) for f in (keys_of, values_of))


def attend(state, q, pos):
    """Attention of padded queries ``q [seqs, n, nh, hd]`` at positions ``pos [seqs, n]`` over the whole cache."""
    c, ctx = state["case"], state["ctx"]
    S, n, nh, hd = q.shape
    nkv, at = c["nkv"], state["table"].long()
    L = at.shape[1] * PAGE
    k, v = (f(state, at).transpose(1, 2).reshape(S, nkv, L, hd) for f in (keys_of, values_of))
    j = torch.arange(L, device="cuda")
    held = (j < ctx.seq_lens[:, None])[:, None, :, None]
    k, v = torch.where(held, k, 0.0), torch.where(held, v, 0.0)
    q = q.view(S, n, nkv, nh // nkv, hd).permute(0, 2, 3, 1, 4).reshape(S, nkv, -1, hd)
    s = torch.matmul(q, k.transpose(-1, -2)).view(S, nkv, nh // nkv, n, L) * hd ** -0.5
    seen = j <= pos[..., None]
    if c["window"]:
        seen = seen & (j > pos[..., None] - c["window"])
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    sink = None if state["sinks"] is None else state["sinks"].view(1, nkv, -1, 1, 1)
    if sink is not None:
        top = torch.maximum(top, sink)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink - top)
    o = torch.matmul((p / total).view(S, nkv, -1, L), v)
    return o.view(S, nkv, nh // nkv, n, hd).permute(0, 3, 1, 2, 4).reshape(S, n, nh * hd).to(DTYPES[c["dtype"]])


def plain_single(state):
    c, ctx = state["case"], state["ctx"]
    return attend(state, state["q"].float().view(c["seqs"], 1, c["nh"], c["hd"]), ctx.positions[:, None])[:, 0]


def plain_portion(state):
    c, ctx = state["case"], state["ctx"]
    col = ctx.positions - ctx.seq_past[ctx.seq_of_token.long()]
    at = (ctx.seq_of_token.long(), col.long())
    q = torch.zeros((c["seqs"], ctx.max_new, c["nh"], c["hd"]), device="cuda")
    q[at] = state["q"].float().view(-1, c["nh"], c["hd"])
    pos = ctx.seq_past[:, None] + torch.arange(ctx.max_new, device="cuda")
    return attend(state, q, pos)[at]


# ---- the definitions in 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    ctx, nh, nkv, hd = state["ctx"], case["nh"], case["nkv"], case["hd"]
    B = block(hd)
    if case["op"] == "prepare":
        x = state["qkv"].double().view(-1, nh + 2 * nkv, hd)
        heads = {"q": x[:, :nh], "k": x[:, nh:nh + nkv], "v": x[:, nh + nkv:]}
        if case["norm"]:
            for name, gain in (("q", state["wq"]), ("k", state["wk"])):
                y = heads[name]
                y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / hd + 1e-6) * gain.double()
                rotated = torch.empty_like(y)
                for i in range(hd // 2):
                    t = ctx.positions.double()[:, None] * float(state["inv_freq"][i])
                    rotated[..., i] = y[..., i] * torch.cos(t) - y[..., i + hd // 2] * torch.sin(t)
                    rotated[..., i + hd // 2] = y[..., i + hd // 2] * torch.cos(t) + y[..., i] * torch.sin(t)
                heads[name] = rotated
        out = {"q": heads["q"].reshape(-1, nh * hd)}
        page = state["table"][ctx.seq_of_token.long(), (ctx.positions // PAGE).long()].long()
        row = (ctx.positions % PAGE).long()
        for name in ("k", "v"):
            y = heads[name]
            m, x = torch.frexp(y.abs().amax(-1))                     # m 2^x with m from 1/2 on; 448 = 7/8 2^9
            scale = torch.ldexp(torch.ones_like(m), x - 9 + (m > 0.875))
            codes = state[name].view(torch.float8_e4m3fn).to(torch.float64)
            scales = torch.full(state[name + "_exp"].shape, math.nan, dtype=torch.float64, device="cuda")
            codes_new = y / scale[..., None]
            for h in range(nkv):
                if name == "k":
                    codes[page, h, :, row] = codes_new[:, h].view(-1, hd // B, B)
                else:
                    codes[page, h, :, row] = codes_new[:, h]
                scales[page, h, row] = scale[:, h]
            out[name], out[name + "_exp"] = codes, scales
        return out
    k_all, v_all = [], []
    for s, n in enumerate(state["lens"]):
        pages = state["table"][s, :-(-n // PAGE)].long()
        k = state["k"][pages].view(torch.float8_e4m3fn).to(torch.float64).permute(1, 0, 3, 2, 4).reshape(nkv, -1, hd)
        v = state["v"][pages].view(torch.float8_e4m3fn).to(torch.float64).permute(1, 0, 3, 2).reshape(nkv, -1, hd)
        for x, e, to in ((k, state["k_exp"], k_all), (v, state["v_exp"], v_all)):
            x = x * torch.exp2(e[pages].permute(1, 0, 2).reshape(nkv, -1, 1).double() - 127)
            x[:, n:] = 0.0
            to.append(x)
    if case["op"] == "read":
        return tuple(torch.cat([x.view(nkv, -1, PAGE, hd).transpose(0, 1) for x in all_]) for all_ in (k_all, v_all))
    outs = []
    for s, n in enumerate(state["lens"]):
        first, last = ctx.host["cu_seqlens"][s], ctx.host["cu_seqlens"][s + 1]
        q = state["q"][first:last].double().view(-1, nh, hd)
        o = torch.empty_like(q)
        at = torch.arange(n - (last - first), n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None, :]
        hidden = (j > at) | (j <= at - case["window"] if case["window"] else j < 0)
        for h in range(nh):
            w = (q[:, h] @ k_all[s][h * nkv // nh, :n].T) / math.sqrt(hd)
            w[hidden] = -math.inf
            if state["sinks"] is not None:
                w = torch.cat([w, state["sinks"][h].double().expand(len(w), 1)], 1)
            o[:, h] = torch.softmax(w, 1)[:, :n] @ v_all[s][h * nkv // nh, :n]
        outs.append(o.view(-1, nh * hd))
    return torch.cat(outs)


def work(case):
    past, new = lengths(case)
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    es, T = (2 if case["dtype"] == "bf16" else 4), sum(new)
    if case["op"] == "prepare":
        return {"bytes": T * ((2 * nh + 2 * nkv) * hd * es + 2 * nkv * (hd + 1)), "flops": 12 * T * (nh + 2 * nkv) * hd}
    if case["op"] == "read":
        rows = sum(-(-p // PAGE) * PAGE for p in past)
        return {"bytes": 2 * nkv * (sum(past) * (hd + 1) + rows * hd * es), "flops": 2 * nkv * sum(past) * hd}
    w = case["window"] or 1 << 60
    held = sum(min(p + n, w + n - 1) for p, n in zip(past, new))
    pairs = sum(min(p + i + 1, w) for p, n in zip(past, new) for i in range(n))
    return {"bytes": 2 * nkv * held * (hd + 1) + 2 * T * nh * hd * es, "flops": 4 * nh * hd * pairs}
