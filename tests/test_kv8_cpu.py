"""A cache in eight bits, as far as it goes without a GPU: the format's arithmetic, storage, options and refusals."""
import dataclasses
import math
import types

import pytest
import torch

import plain_kv8 as P
from synaptix_b200 import cli, ops
from synaptix_b200.cache import Cache, KVRequest
from synaptix_b200.csrc.build import KernelsUnavailable
from synaptix_b200.ops import KernelError


def test_the_oracles_codes_are_e4m3():
    every = torch.arange(256, dtype=torch.uint8)
    every = every[(every & 127) != 127]                          # (the two NaN)
    v = every.view(torch.float8_e4m3fn).double()
    assert torch.equal(P.code_of(v), every) and torch.equal(P.round_e4m3(v), v)
    x = torch.randn(4096, generator=torch.Generator().manual_seed(0)).double() * 20
    assert torch.equal(P.code_of(P.round_e4m3(x)), x.float().to(torch.float8_e4m3fn).view(torch.uint8))
    assert P.round_e4m3(torch.tensor([500.0, -1e30]).double()).tolist() == [448.0, -448.0]


@pytest.mark.parametrize("scale", [1e-30, 1e-3, 1.0, 77.0, 1e30])
def test_a_row_is_off_by_half_a_step(scale):
    """Elements down to 2^-14 of the row's largest are off by at most 2^-4 of themselves; smaller ones by half the smallest step,
    2^-10 2^E <= 2^-10 2 a / 448."""
    x = torch.randn(300, 96, generator=torch.Generator().manual_seed(1)).double() * scale
    _, e, v = P.quantise(x)
    a = x.abs().amax(-1, keepdim=True)
    assert ((v - x).abs() <= torch.maximum(x.abs() * 2.0 ** -4, a * (2.0 ** -9 / 448))).all()
    power = torch.exp2(e.double() - 127)[:, None]
    assert (a <= 448 * power).all() and (a > 224 * power).all()


def test_storage():
    c = Cache([KVRequest(2, 96, eight_bit=True), KVRequest(4, 64, window=100, eight_bit=True), KVRequest(2, 96, eight_bit=True)],
              max_tokens=300, max_seqs=3, dtype=torch.bfloat16, device="cpu", kv_dtype="fp8")
    a, b, a2 = (c.view(i) for i in range(3))
    assert tuple(a.pages8.k.shape) == (6, 2, 3, 64, 32) and tuple(a.pages8.v.shape) == (6, 2, 96, 64) and tuple(a.pages8.k_exp.shape) == (6, 2, 64)
    assert tuple(b.pages8.k.shape) == (6, 4, 1, 64, 64) and b.window == 100 and a2.group == a.group
    assert a.pages8.k.data_ptr() != a2.pages8.k.data_ptr() and all(t.dtype == torch.uint8 and t.is_contiguous() for t in a.pages8)
    assert c.kv_bytes_per_token == 2 * 2 * 2 * 97 + 2 * 4 * 65 and c.bytes() == c.kv_bytes_per_token * 6 * 64
    wide = Cache([KVRequest(2, 96, eight_bit=True)], max_tokens=300, max_seqs=3, dtype=torch.bfloat16, device="cpu")
    assert wide.view(0).pages8 is None and wide.kv_bytes_per_token == 2 * 2 * 96 * 2


def test_what_cannot_be_held_in_eight_bits_is_refused():
    def cache(*requests, **kw):
        return Cache(requests, max_tokens=64, max_seqs=1, dtype=torch.bfloat16, device="cpu", **kw)
    for bad in ((KVRequest(2, 64),), (KVRequest(2, 64, eight_bit=True), KVRequest(1, 576, keys_only=True)), ()):
        with pytest.raises(ValueError, match="fp8"):
            cache(*bad, kv_dtype="fp8")
    with pytest.raises(ValueError, match="int8"):
        cache(KVRequest(2, 64, eight_bit=True), kv_dtype="int8")
    from synaptix_b200.parts import Attention, NoPosition
    for hd, vd, takes in ((64, None, True), (16, None, True), (256, None, True), (40, None, False), (320, None, False), (64, 32, False)):
        r = Attention("", 64, 4, 2, hd, position=NoPosition(), v_head_dim=vd).cache_request()
        assert r.eight_bit is takes and r == dataclasses.replace(r, eight_bit=False)


def test_command_line():
    p = cli.build_parser()
    assert p.parse_args(["run", "MODEL"]).kv_dtype == "auto" and p.parse_args(["bench", "MODEL", "--kv-dtype", "fp8"]).kv_dtype == "fp8"
    assert [cli._kv_dtype_arg(s) for s in ("auto", "FP8", "mxfp8")] == [None, "fp8", "fp8"]
    with pytest.raises(SystemExit):
        cli._kv_dtype_arg("int4")


def step(lens, new, **kw):
    past = [a - b for a, b in zip(lens, new)]
    cu = [sum(new[:i]) for i in range(len(new) + 1)]
    ints = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return types.SimpleNamespace(**{**dict(
        all_single=all(n == 1 for n in new), n_seqs=len(lens), n_tokens=sum(new), max_new=max(new), max_len=max(lens), seq_lens=ints(lens),
        seq_past=ints(past), cu_seqlens=ints(cu), positions=ints([p + i for p, n in zip(past, new) for i in range(n)]),
        seq_of_token=ints([s for s, n in enumerate(new) for _ in range(n)]), scratch={},
        host={"cu_seqlens": cu, "seq_past": past, "seq_lens": list(lens)}), **kw})


def pages(n=3, nkv=2, hd=64):
    return ops.KV8Pages(*(torch.zeros(s, dtype=torch.uint8) for s in (lambda k, v, e: (k, v, e, e))(*ops.kv8_shapes(n, nkv, hd))))


def test_prepare_refuses():
    ok = dict(qkv=torch.zeros(2, 8 * 64), q_out=torch.zeros(2, 4 * 64), pages=pages(), wq=torch.zeros(64), wk=torch.zeros(64),
              inv_freq=torch.zeros(16), rotary_dim=32, eps=1e-6, positions=torch.zeros(2, dtype=torch.int32),
              seq_of_token=torch.zeros(2, dtype=torch.int32), block_table=torch.zeros((1, 2), dtype=torch.int32), nh=4, nkv=2, hd=64, col=0)
    with pytest.raises(KernelsUnavailable):
        ops.kv8_prepare(**ok)                                    # nothing wrong but the device
    bad = [dict(nkv=1), dict(hd=32), dict(col=1), dict(col=-1), dict(nh=5), dict(nh=-1), dict(q_out=None), dict(q_out=torch.zeros(2, 4 * 64).bfloat16()),
           dict(qkv=torch.zeros(2, 8 * 64).half(), q_out=torch.zeros(2, 4 * 64).half()), dict(wq=torch.zeros(63)), dict(wk=torch.zeros(64).bfloat16()),
           dict(rotary_dim=30), dict(rotary_dim=66), dict(positions=torch.zeros(2)), dict(positions=torch.zeros(1, dtype=torch.int32)),
           dict(seq_of_token=torch.zeros(2, dtype=torch.int64)), dict(block_table=torch.zeros(2, dtype=torch.int32)),
           dict(pages=pages()._replace(k=torch.zeros(3, 2, 64, 64, dtype=torch.uint8))), dict(pages=pages()._replace(v_exp=torch.zeros(3, 2, 64))),
           dict(pages=pages(hd=48), hd=48), dict(pages=pages(n=0)), dict(pages=None, hd=40, nh=1, q_out=torch.zeros(2, 40))]
    for change in bad:
        with pytest.raises(KernelError):
            ops.kv8_prepare(**{**ok, **change})


def test_read_refuses():
    ok = dict(pages=pages(), ctx=step([70], [0]), block_table=torch.zeros((1, 2), dtype=torch.int32), dtype=torch.float32)
    with pytest.raises(KernelsUnavailable):
        ops.kv8_read(**ok)
    for change in (dict(ctx=step([70], [0], host=None)), dict(ctx=step([129], [0])), dict(block_table=torch.zeros((0, 2), dtype=torch.int32)),
                   dict(dtype=torch.float16), dict(window=0), dict(chunk=-1), dict(ctx=step([70], [0], seq_lens=torch.tensor([70.0])))):
        with pytest.raises(KernelError):
            ops.kv8_read(**{**ok, **change})


@pytest.mark.parametrize("new", [1, 5])
def test_attention_refuses(new):
    q = torch.zeros(new, 4 * 64)
    ok = dict(q=q, pages=pages(), ctx=step([70], [new]), block_table=torch.zeros((1, 2), dtype=torch.int32), nh=4, nkv=2, hd=64, scale=1.0)
    with pytest.raises(KernelsUnavailable):
        ops.kv8_attention(**ok)
    bad = [dict(nh=3), dict(nkv=1), dict(hd=32), dict(q=torch.zeros(new, 65)), dict(q=q.half()), dict(sinks=torch.zeros(3)), dict(sinks=torch.zeros(4).bfloat16()),
           dict(window=0), dict(chunk=0), dict(softcap=-1.0), dict(softcap=math.nan), dict(out=torch.zeros(new, 4 * 64).bfloat16()),
           dict(out=torch.zeros(new + 1, 4 * 64)), dict(out=torch.zeros(new, 4 * 64), out_col=8), dict(out=torch.zeros(new, 8 * 64)[:, ::2]),
           dict(block_table=torch.zeros((1, 2))), dict(block_table=torch.zeros((0, 2), dtype=torch.int32))]
    if new > 1:
        bad += [dict(ctx=step([70], [new], host=None)), dict(ctx=step([70], [new], cu_seqlens=torch.tensor([0.0, 5.0]))),
                dict(ctx=step([70], [new], seq_past=torch.tensor([65]))), dict(ctx=step([70], [new], cu_seqlens=torch.zeros(1, dtype=torch.int32))),
                dict(ctx=step([70], [new + 1])), dict(ctx=step([70], [new - 1])), dict(ctx=step([129], [new])),
                dict(ctx=step([70], [new], seq_of_token=torch.zeros(new - 1, dtype=torch.int32)))]
    for change in bad:
        with pytest.raises(KernelError):
            ops.kv8_attention(**{**ok, **change})
