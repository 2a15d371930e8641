"""Python faces of the kernels of a cache in eight bits (``csrc/kv8.cu``): heads prepared and quantised into the pages, pages
read back, and attention over them.

A token's key (or value) of a head is one exponent byte ``e`` and ``hd`` e4m3 codes ``c`` and stands for ``c * 2^(e - 127)``
(``csrc/kv8.cuh`` says how a row is rounded and why).  A row that held an infinity or NaN reads as NaN as a whole; magnitudes above
``448 * 2^119`` saturate.  Head sizes are multiples of 16 up to 256, keys and values of one size."""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Tuple

import numpy as np
import torch

from ._lib import KernelError, c_float, c_int, check, dt_code, fn, ptr, require_cuda, stream
from .decode import sm_count

PAGE = 64
MAX_HEAD_DIM = 256


class KV8Pages(NamedTuple):
    """A cache entry in eight bits: uint8 codes ``k [n_pages, kv heads, hd / B, 64, B]`` (``B`` the largest of 64, 32, 16 that
    divides ``hd``) and ``v [n_pages, kv heads, hd, 64]``, uint8 exponents ``k_exp``, ``v_exp`` ``[n_pages, kv heads, 64]``."""
    k: torch.Tensor
    v: torch.Tensor
    k_exp: torch.Tensor
    v_exp: torch.Tensor

    @property
    def n_kv_heads(self) -> int:
        return self.v.shape[1]

    @property
    def head_dim(self) -> int:
        return self.v.shape[2]


def kv8_supported(hd: int, vd: Optional[int] = None) -> bool:
    """Whether keys and values of this size can be held in eight bits."""
    return vd in (None, hd) and 0 < hd <= MAX_HEAD_DIM and hd % 16 == 0


def kv8_shapes(n_pages: int, nkv: int, hd: int) -> Tuple[tuple, tuple, tuple]:
    """Shapes of the codes of keys and values and of their exponents."""
    b = 64 if hd % 64 == 0 else 32 if hd % 32 == 0 else 16
    return (n_pages, nkv, hd // b, PAGE, b), (n_pages, nkv, hd, PAGE), (n_pages, nkv, PAGE)


def _check_pages(pages: KV8Pages, what: str, nkv: Optional[int] = None, hd: Optional[int] = None) -> Tuple[int, int, int]:
    if any(t.dtype != torch.uint8 for t in pages):
        raise KernelError(f"{what}: codes and exponents are uint8")
    if pages.v.dim() != 4:
        raise KernelError(f"{what}: values are [n_pages, kv heads, head size, 64]")
    n, kv, d = pages.v.shape[:3]
    if (nkv is not None and nkv != kv) or (hd is not None and hd != d):
        raise KernelError(f"{what}: the pages hold {kv} heads of {d}, not {nkv} of {hd}")
    if not kv8_supported(d):
        raise KernelError(f"{what}: head sizes are multiples of 16 up to {MAX_HEAD_DIM}")
    ks, vs, es = kv8_shapes(n, kv, d)
    if tuple(pages.k.shape) != ks or tuple(pages.v.shape) != vs or tuple(pages.k_exp.shape) != es or tuple(pages.v_exp.shape) != es:
        raise KernelError(f"{what}: codes or exponents have the wrong shape (want {ks}, {vs}, {es})")
    if n < 1 or kv < 1:
        raise KernelError(f"{what}: no pages, or no heads")
    return n, kv, d


def _check_index(what: str, *tensors: torch.Tensor) -> None:
    if any(t.dtype != torch.int32 for t in tensors):
        raise KernelError(f"{what}: index tensors are int32")


def _check_device(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """Behind all other checks: contiguous tensors of the current CUDA device."""
    device = next(t.device for t in tensors if t is not None)
    if any(t is not None and t.device != device for t in tensors):
        raise KernelError(f"{what}: tensors lie on several devices")
    require_cuda(*tensors)
    if device.index is not None and device.index != torch.cuda.current_device():
        raise KernelError(f"{what}: the tensors lie on {device}, the current device is cuda:{torch.cuda.current_device()}")


def kv8_prepare(qkv: torch.Tensor, q_out: Optional[torch.Tensor], pages: Optional[KV8Pages], wq: Optional[torch.Tensor],
                wk: Optional[torch.Tensor], inv_freq: Optional[torch.Tensor], rotary_dim: int, eps: float,
                positions: torch.Tensor, seq_of_token: torch.Tensor, block_table: torch.Tensor, nh: int, nkv: int, hd: int,
                col: int = 0) -> None:
    """Per-head RMSNorm (gains ``wq``, ``wk`` float32 ``[hd]``; optional) and rotate-half rotation (``inv_freq`` float32
    ``[rotary_dim / 2]``; optional) of the step's heads, and the write of keys and values into pages of eight bits.

    ``qkv [T, row]`` (bfloat16 or float32): q heads, then k and v heads from column ``col`` on, other columns around them.  q heads
    go to ``q_out [T, nh * hd]`` in ``qkv``'s dtype (``nh = 0``: none); keys and values into the pages of each token's sequence at its position.
    Two tokens of a call never share a sequence and a position.  Without ``pages`` nothing is written (a layer that reads another layer's
    cache; ``qkv`` may then hold the q heads alone)."""
    n_pages = 0
    if pages is not None:
        n_pages, _, _ = _check_pages(pages, "kv8_prepare", nkv, hd)
    elif not kv8_supported(hd):
        raise KernelError(f"kv8_prepare: head sizes are multiples of 16 up to {MAX_HEAD_DIM}")
    _check_index("kv8_prepare", positions, seq_of_token, block_table)
    if qkv.dim() != 2 or block_table.dim() != 2 or positions.numel() < qkv.shape[0] or seq_of_token.numel() < qkv.shape[0]:
        raise KernelError("kv8_prepare: qkv is [T, row], with a position and a sequence per token and a table [sequences, pages]")
    T, row = qkv.shape
    if nh < 0 or nkv < 1 or col < 0 or col + (nh + (2 * nkv if pages is not None else 0)) * hd > row:
        raise KernelError("kv8_prepare: the heads do not fit the rows of qkv")
    if nh and (q_out is None or q_out.dtype != qkv.dtype or tuple(q_out.shape) != (T, nh * hd)):
        raise KernelError("kv8_prepare: q_out is [T, nh * hd] in qkv's dtype")
    if any(w is not None and (w.dtype != torch.float32 or w.numel() != hd) for w in (wq, wk)):
        raise KernelError("kv8_prepare: gains are float32, one per element of a head")
    if inv_freq is None:
        rotary_dim = 0
    elif inv_freq.dtype != torch.float32 or rotary_dim % 2 or not 0 < rotary_dim <= hd or inv_freq.numel() != rotary_dim // 2:
        raise KernelError("kv8_prepare: inv_freq is float32 with a frequency per rotated pair of the head")
    dt_code(qkv.dtype)
    k, v, ke, ve = pages if pages is not None else (None,) * 4
    _check_device("kv8_prepare", qkv, q_out, k, v, ke, ve, wq, wk, inv_freq, positions, seq_of_token, block_table)
    check(fn("kv8", "sx_kv8_prepare")(
        ptr(qkv if col == 0 else qkv.view(-1)[col:]), ptr(q_out), ptr(k), ptr(v), ptr(ke), ptr(ve), ptr(wq), ptr(wk), ptr(inv_freq),
        c_int(rotary_dim), c_float(eps), ptr(positions), ptr(seq_of_token), ptr(block_table), c_int(block_table.shape[1]), c_int(T), c_int(nh),
        c_int(nkv), c_int(hd), c_int(n_pages), c_int(row), c_int(dt_code(qkv.dtype)), stream()), "kv8_prepare",
        launches=1 if T and (nh or pages is not None) else 0)


def _read_plan(ctx, width: int, window: Optional[int], chunk: Optional[int], device):
    """Which pages of which sequence are read, in order, and the table that finds them again, made once a step."""
    key = ("kv8_read", width, window, chunk)
    plan = ctx.scratch.get(key)
    if plan is None:
        past, lens = ctx.host["seq_past"], ctx.host["seq_lens"]
        seqs, idx, table = [], [], np.zeros((len(lens), width), dtype=np.int32)
        for s, (p, n) in enumerate(zip(past, lens)):
            first = max(0, p - window + 1) if window else 0              # the first key that the step's first token sees
            if chunk:
                first = max(first, p // chunk * chunk)
            a, b = first // PAGE, -(-n // PAGE)
            at = len(idx)
            table[s, :b] = at + np.maximum(np.arange(b) - a, 0)
            seqs += [s] * (b - a)
            idx += range(a, b)
        flat = np.concatenate([table.reshape(-1), np.asarray(seqs + idx, dtype=np.int32)])
        dev = torch.from_numpy(flat).to(device, non_blocking=True)
        n = len(idx)
        plan = ctx.scratch[key] = (dev[:table.size].view(table.shape), dev[table.size:table.size + n], dev[table.size + n:], n)
    return plan


def _check_host(what: str, ctx, block_table: torch.Tensor) -> None:
    _check_index(what, ctx.seq_lens, block_table)
    if ctx.host is None:
        raise KernelError(f"{what}: the step's lengths are not known on the host (a captured step)")
    lens = ctx.host["seq_lens"]
    if block_table.dim() != 2 or block_table.shape[0] < len(lens) or ctx.seq_lens.numel() < len(lens):
        raise KernelError(f"{what}: a row of the table and a length per sequence")
    if any(-(-n // PAGE) > block_table.shape[1] for n in lens):
        raise KernelError(f"{what}: the table is too narrow for the sequences")


def kv8_read(pages: KV8Pages, ctx, block_table: torch.Tensor, dtype: torch.dtype, window: Optional[int] = None,
             chunk: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """What the cache holds of the step's sequences, back in ``dtype`` (exactly, in bfloat16 and float32): ``(k, v, table)`` with
    ``k``, ``v`` ``[n, kv heads, 64, hd]`` the pages one sequence after the other and ``table`` int32 ``[sequences, pages]`` the page
    of each.  Rows behind a sequence's end are zero.  With ``window`` or ``chunk`` pages that no token of the step sees are left
    out (their place in the table names another page).  Needs the step's lengths on the host."""
    n_pages, nkv, hd = _check_pages(pages, "kv8_read")
    _check_host("kv8_read", ctx, block_table)
    if (window is not None and window < 1) or (chunk is not None and chunk < 1):
        raise KernelError("kv8_read: window and chunk are positive")
    dt = dt_code(dtype)
    _check_device("kv8_read", *pages, ctx.seq_lens, block_table)
    table, seqs, idx, n = _read_plan(ctx, block_table.shape[1], window, chunk, pages.k.device)
    k = torch.empty((n, nkv, PAGE, hd), dtype=dtype, device=pages.k.device)
    v = torch.empty_like(k)
    check(fn("kv8", "sx_kv8_read")(
        ptr(pages.k), ptr(pages.v), ptr(pages.k_exp), ptr(pages.v_exp), ptr(k), ptr(v), ptr(seqs), ptr(idx), c_int(n), ptr(ctx.seq_lens),
        ptr(block_table), c_int(block_table.shape[1]), c_int(nkv), c_int(hd), c_int(n_pages), c_int(dt), stream()), "kv8_read",
        launches=1 if n else 0)
    return k, v, table


def _rows_splits(S: int, nh: int, nkv: int, max_pages: int, device) -> int:
    """Shares of a sequence's pages: as many as keep all blocks in one wave (two fit an SM), each with a page a warp."""
    blocks = max(1, S * nkv * -(-(nh // nkv) // 4))
    return max(1, min(-(-max_pages // 8), 2 * sm_count(device) // blocks))


def kv8_rows(q: torch.Tensor, pages: KV8Pages, seq_lens: torch.Tensor, block_table: torch.Tensor, nh: int, scale: float,
             window: Optional[int], max_len: int, *, softcap: Optional[float] = None, sinks: Optional[torch.Tensor] = None,
             chunk: Optional[int] = None, out: Optional[torch.Tensor] = None, out_col: int = 0, out_scale: float = 1.0) -> torch.Tensor:
    """One query token a sequence (row ``s`` of ``q``) by the kernel that takes every head size, type and option."""
    n_pages, nkv, hd = pages.v.shape[:3]
    S = q.shape[0]
    if out is None:
        out = torch.empty((S, nh * hd), dtype=q.dtype, device=q.device)
    splits = _rows_splits(S, nh, nkv, -(-max_len // PAGE), q.device)
    part_o = part_ml = None
    if splits > 1:
        part_o = torch.empty(S * nh * splits * hd, dtype=torch.float32, device=q.device)
        part_ml = torch.empty(S * nh * splits * 2, dtype=torch.float32, device=q.device)
    o = out if out_col == 0 else out.view(-1)[out_col:]
    check(fn("kv8", "sx_kv8_rows")(
        ptr(q), ptr(o), ptr(pages.k), ptr(pages.v), ptr(pages.k_exp), ptr(pages.v_exp), ptr(seq_lens), ptr(block_table), c_int(block_table.shape[1]),
        c_int(S), c_int(nh), c_int(nkv), c_int(hd), c_int(n_pages), c_float(scale), c_int(window or 0), c_float(softcap or 0.0), ptr(sinks),
        c_int(chunk or 0), c_int(out.shape[1]), c_float(out_scale), c_int(splits), ptr(part_o), ptr(part_ml), c_int(dt_code(q.dtype)), stream()),
        "kv8_attention", launches=2 if splits > 1 else 1)
    return out


DECODE_HEAD_DIMS = (64, 128)
DECODE_MAX_GROUP = 16
DECODE_MAX_SEQS = 2047


def kv8_decode_supported(dtype, nh: int, nkv: int, hd: int, S: int) -> bool:
    """Whether single tokens of these sizes attend on the tensor cores (``csrc/kv8_decode.cu``)."""
    return dtype == torch.bfloat16 and hd in DECODE_HEAD_DIMS and nh // nkv <= DECODE_MAX_GROUP and S <= DECODE_MAX_SEQS


def kv8_decode(q: torch.Tensor, pages: KV8Pages, seq_lens: torch.Tensor, block_table: torch.Tensor, nh: int, scale: float,
               window: Optional[int], max_len: int, sinks: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One query token a sequence (row ``s`` of ``q``) on the tensor cores; sizes as ``kv8_decode_supported`` says."""
    n_pages, nkv, hd = pages.v.shape[:3]
    S = q.shape[0]
    max_pages = min(-(-max_len // PAGE), block_table.shape[1]) if window is None else min(-(-max_len // PAGE), block_table.shape[1], (window + 126) // PAGE)
    floats = ctypes.c_longlong(0)
    launches = fn("kv8_decode", "sx_kv8_decode_plan")(c_int(S), c_int(nh), c_int(nkv), c_int(hd), c_int(max_pages), ctypes.byref(floats))
    out = torch.empty_like(q)
    part = torch.empty(floats.value, dtype=torch.float32, device=q.device)
    check(fn("kv8_decode", "sx_kv8_decode")(
        ptr(q), ptr(out), ptr(pages.k), ptr(pages.v), ptr(pages.k_exp), ptr(pages.v_exp), ptr(seq_lens), ptr(block_table), c_int(block_table.shape[1]),
        c_int(S), c_int(nh), c_int(nkv), c_int(hd), c_int(n_pages), c_float(scale), c_int(window or 0), ptr(sinks), ptr(part), c_int(max_pages), stream()),
        "kv8_attention", launches=launches)
    return out


def kv8_decode_status(reset: bool = False) -> int:
    """0, or 1: a bounded wait of ``kv8_decode`` ran out in a launch the host has already waited for.  ``reset`` puts it back to 0."""
    v = ctypes.c_int(0)
    check(fn("kv8_decode", "sx_kv8_decode_status")(ctypes.byref(v), c_int(1 if reset else 0)), "kv8_decode_status", launches=0)
    return int(v.value)


def kv8_attention(q: torch.Tensor, pages: KV8Pages, ctx, block_table: torch.Tensor, nh: int, nkv: int, hd: int, scale: float,
                  window: Optional[int] = None, *, softcap: Optional[float] = None, sinks: Optional[torch.Tensor] = None,
                  chunk: Optional[int] = None, out: Optional[torch.Tensor] = None, out_col: int = 0,
                  out_scale: float = 1.0) -> torch.Tensor:
    """Causal attention of the step's packed queries ``q [T, nh * hd]`` over a cache in eight bits that already holds the step's
    keys and values: ``[T, nh * hd]`` in ``q``'s dtype.  The options are those of ``ops.attention``.

    Single tokens attend over the codes.  Portions of prompts read the pages back once (``kv8_read``) and attend over the result
    with the kernels of the 16- and 32-bit cache: a page serves many rows there, and turning its codes again in every block that
    reads it would cost more than writing it out once."""
    n_pages, _, _ = _check_pages(pages, "kv8_attention", nkv, hd)
    _check_index("kv8_attention", ctx.seq_lens, block_table)
    dt_code(q.dtype)
    if nh < 1 or nh % nkv or q.dim() != 2 or q.shape[1] != nh * hd:
        raise KernelError("kv8_attention: q is [T, nh * hd], and every kv head serves as many query heads")
    if sinks is not None and (sinks.dtype != torch.float32 or sinks.numel() != nh):
        raise KernelError("kv8_attention: sinks are float32, one per query head")
    if (window is not None and window < 1) or (chunk is not None and chunk < 1) or (softcap is not None and not softcap > 0):
        raise KernelError("kv8_attention: window, chunk and softcap are positive")
    if out is not None and (out.dtype != q.dtype or out.dim() != 2 or out.shape[0] != q.shape[0] or out_col < 0
                            or out_col + nh * hd > out.shape[1] or not out.is_contiguous()):
        raise KernelError("kv8_attention: the output does not fit")
    if ctx.all_single and ctx.n_seqs == q.shape[0]:
        if block_table.dim() != 2 or block_table.shape[0] < ctx.n_seqs or ctx.seq_lens.numel() < ctx.n_seqs:
            raise KernelError("kv8_attention: a row of the table and a length per sequence")
        _check_device("kv8_attention", q, *pages, ctx.seq_lens, block_table, sinks, out)
        if out is None and softcap is None and chunk is None and out_scale == 1.0 and kv8_decode_supported(q.dtype, nh, nkv, hd, q.shape[0]):
            return kv8_decode(q, pages, ctx.seq_lens, block_table, nh, scale, window, ctx.max_len, sinks)
        return kv8_rows(q, pages, ctx.seq_lens, block_table, nh, scale, window, ctx.max_len, softcap=softcap, sinks=sinks, chunk=chunk,
                        out=out, out_col=out_col, out_scale=out_scale)
    from . import attention
    _check_host("kv8_attention", ctx, block_table)
    _check_device("kv8_attention", q, *pages, ctx.seq_lens, block_table, sinks, out)
    k, v, table = kv8_read(pages, ctx, block_table, q.dtype, window, chunk)
    return attention(q, k, v, ctx, table, nh, nkv, hd, scale, window, softcap=softcap, sinks=sinks, chunk=chunk, out=out, out_col=out_col,
                     out_scale=out_scale)
