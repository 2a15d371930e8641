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

from ._lib import KernelError, c_int, check, dt_code, fn, launcher, raw_stream, require_cuda
from .decode import sm_count

current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)

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


_SHAPES = {}                    # of the values' shape: those of keys and exponents, or what is wrong with it


def _shapes_beside(v_shape, what: str):
    both = _SHAPES.get(v_shape)
    if both is None:
        if len(v_shape) != 4 or v_shape[3] != PAGE:
            raise KernelError(f"{what}: values are [n_pages, kv heads, head size, 64]")
        n, kv, d = v_shape[:3]
        if not kv8_supported(d):
            raise KernelError(f"{what}: head sizes are multiples of 16 up to {MAX_HEAD_DIM}")
        if n < 1 or kv < 1:
            raise KernelError(f"{what}: no pages, or no heads")
        k, _, e = kv8_shapes(n, kv, d)
        both = _SHAPES[v_shape] = (torch.Size(k), torch.Size(e))
    return both


def _check_pages(pages: KV8Pages, what: str, nkv: Optional[int] = None, hd: Optional[int] = None):
    k, v, ke, ve = pages
    u8 = torch.uint8
    if k.dtype is not u8 or v.dtype is not u8 or ke.dtype is not u8 or ve.dtype is not u8:
        raise KernelError(f"{what}: codes and exponents are uint8")
    vs = v.shape
    ks, es = _SHAPES.get(vs) or _shapes_beside(vs, what)
    if k.shape != ks or ke.shape != es or ve.shape != es:
        raise KernelError(f"{what}: codes or exponents have the wrong shape (want %s, %s, %s)" % (tuple(ks), tuple(vs), tuple(es)))
    if nkv is not None and (nkv != vs[1] or hd != vs[2]):
        raise KernelError(f"{what}: the pages hold {vs[1]} heads of {vs[2]}, not {nkv} of {hd}")
    return vs


def _check_device(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """Behind all other checks: contiguous tensors of the current CUDA device."""
    device = tensors[0].get_device()
    for t in tensors:
        if t is not None and (t.get_device() != device or not t.is_contiguous()):
            require_cuda(t)
            raise KernelError(f"{what}: tensors lie on several devices")
    if device < 0:
        require_cuda(tensors[0])
    if device != current_device():
        raise KernelError(f"{what}: the tensors lie on cuda:{device}, the current device is cuda:{current_device()}")


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


# at least this many tokens: the kernels that take four tokens' queries and keys, and 16 tokens' values, a block
WIDE_MIN_TOKENS = 64


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
    k = v = ke = ve = None
    n_pages = 0
    if pages is not None:
        n_pages = _check_pages(pages, "kv8_prepare", nkv, hd)[0]
        k, v, ke, ve = pages
    elif not kv8_supported(hd):
        raise KernelError(f"kv8_prepare: head sizes are multiples of 16 up to {MAX_HEAD_DIM}")
    i32, f32 = torch.int32, torch.float32
    if positions.dtype is not i32 or seq_of_token.dtype is not i32 or block_table.dtype is not i32:
        raise KernelError("kv8_prepare: index tensors are int32")
    if qkv.dim() != 2 or block_table.dim() != 2:
        raise KernelError("kv8_prepare: qkv is [T, row], with a position and a sequence per token and a table [sequences, pages]")
    T, row = qkv.shape
    if positions.numel() < T or seq_of_token.numel() < T:
        raise KernelError("kv8_prepare: qkv is [T, row], with a position and a sequence per token and a table [sequences, pages]")
    if nh < 0 or nkv < 1 or col < 0 or col + (nh + (2 * nkv if pages is not None else 0)) * hd > row:
        raise KernelError("kv8_prepare: the heads do not fit the rows of qkv")
    if nh and (q_out is None or q_out.dtype != qkv.dtype or q_out.shape != (T, nh * hd)):
        raise KernelError("kv8_prepare: q_out is [T, nh * hd] in qkv's dtype")
    if (wq is not None and (wq.dtype is not f32 or wq.numel() != hd)) or (wk is not None and (wk.dtype is not f32 or wk.numel() != hd)):
        raise KernelError("kv8_prepare: gains are float32, one per element of a head")
    if inv_freq is None:
        rotary_dim = 0
    elif inv_freq.dtype is not f32 or rotary_dim % 2 or not 0 < rotary_dim <= hd or inv_freq.numel() != rotary_dim // 2:
        raise KernelError("kv8_prepare: inv_freq is float32 with a frequency per rotated pair of the head")
    dt = dt_code(qkv.dtype)
    _check_device("kv8_prepare", qkv, q_out, k, v, ke, ve, wq, wk, inv_freq, positions, seq_of_token, block_table)
    es = 4 if dt == 0 else 2
    a_qkv, a_q, a_wq, a_wk = qkv.data_ptr() + col * es, _ptr(q_out), _ptr(wq), _ptr(wk)
    a_k, a_v = _ptr(k), _ptr(v)
    wide = (T >= WIDE_MIN_TOKENS and hd in (64, 128) and (inv_freq is None or rotary_dim == hd)
            and not (row * es | a_qkv | (a_q or 0) | (a_k or 0) | (a_v or 0) | (a_wq or 0) | (a_wk or 0)) & 15)
    check(launcher("kv8", "sx_kv8_prepare")(
        a_qkv, a_q, a_k, a_v, _ptr(ke), _ptr(ve), a_wq, a_wk, _ptr(inv_freq), rotary_dim, eps, positions.data_ptr(), seq_of_token.data_ptr(),
        block_table.data_ptr(), block_table.shape[1], T, nh, nkv, hd, n_pages, row, wide, dt, raw_stream()), "kv8_prepare",
        launches=1 if T and (nh or k is not None) else 0)


def _read_plan(ctx, width: int, window: Optional[int], chunk: Optional[int], device):
    """The table that finds the pages read again, which pages of which sequence they are, in order, and from which row on tokens of the step
    see them, made once a step (and anew where a context is used for other lengths)."""
    past, lens = ctx.host["seq_past"], ctx.host["seq_lens"]
    plan = ctx.scratch.get(("kv8_read", width, window, chunk))
    if plan is not None and plan[4] == past and plan[5] == lens:
        return plan
    seqs, idx, rows, table = [], [], [], np.zeros((len(lens), width), dtype=np.int32)
    for s, (p, n) in enumerate(zip(past, lens)):
        first = max(0, p - window + 1) if window else 0                  # the first key that the step's first token sees
        if chunk:
            first = max(first, p // chunk * chunk)
        a, b = first // PAGE, -(-n // PAGE)
        at = len(idx)
        table[s, :b] = at + np.maximum(np.arange(b) - a, 0)
        seqs += [s] * (b - a)
        idx += range(a, b)
        rows += [max(0, first - PAGE * i) for i in range(a, b)]
    flat = np.concatenate([table.reshape(-1), np.asarray(seqs + idx + rows, dtype=np.int32)])
    dev = torch.from_numpy(flat).to(device, non_blocking=True)
    n, at = len(idx), table.size
    plan = ctx.scratch[("kv8_read", width, window, chunk)] = (dev[:at].view(table.shape), dev[at:at + n], dev[at + n:at + 2 * n], dev[at + 2 * n:], list(past),
                                                              list(lens))
    return plan


def _check_host(what: str, ctx, block_table: torch.Tensor) -> None:
    if not (ctx.seq_lens.dtype == block_table.dtype == torch.int32):
        raise KernelError(f"{what}: index tensors are int32")
    if ctx.host is None:
        raise KernelError(f"{what}: the step's lengths are not known on the host (a captured step)")
    lens = ctx.host["seq_lens"]
    if block_table.dim() != 2 or block_table.shape[0] < len(lens) or ctx.seq_lens.numel() < len(lens):
        raise KernelError(f"{what}: a row of the table and a length per sequence")
    if lens and -(-max(lens) // PAGE) > block_table.shape[1]:
        raise KernelError(f"{what}: the table is too narrow for the sequences")


def kv8_read(pages: KV8Pages, ctx, block_table: torch.Tensor, dtype: torch.dtype, window: Optional[int] = None,
             chunk: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """What the cache holds of the step's sequences, back in ``dtype`` (exactly, in bfloat16 and float32): ``(k, v, table)`` with
    ``k``, ``v`` ``[n, kv heads, 64, hd]`` the pages one sequence after the other and ``table`` int32 ``[sequences, pages]`` the page
    of each.  Rows behind a sequence's end are zero.  With ``window`` or ``chunk`` pages that no token of the step sees are left
    out (their place in the table names another page).  Needs the step's lengths on the host."""
    _check_pages(pages, "kv8_read")
    _check_host("kv8_read", ctx, block_table)
    if (window is not None and window < 1) or (chunk is not None and chunk < 1):
        raise KernelError("kv8_read: window and chunk are positive")
    dt_code(dtype)
    _check_device("kv8_read", *pages, ctx.seq_lens, block_table)
    return _read(pages, ctx, block_table, dtype, window, chunk, False)


def _read(pages: KV8Pages, ctx, block_table: torch.Tensor, dtype: torch.dtype, window: Optional[int], chunk: Optional[int], for_attention: bool):
    """``kv8_read`` of what has been checked.  ``for_attention``: rows that no token of the step sees are zeros; so are value rows that are not
    finite, and their keys are NaN."""
    k8, v8, ke, ve = pages
    n_pages, nkv, hd, _ = v8.shape
    device, width = v8.device, block_table.shape[1]
    table, seqs, idx, rows, _, _ = _read_plan(ctx, width, window, chunk, device)
    n = idx.numel()
    k = torch.empty((n, nkv, PAGE, hd), dtype=dtype, device=device)
    v = torch.empty_like(k)
    check(launcher("kv8", "sx_kv8_read")(
        k8.data_ptr(), v8.data_ptr(), ke.data_ptr(), ve.data_ptr(), k.data_ptr(), v.data_ptr(), seqs.data_ptr(), idx.data_ptr(),
        rows.data_ptr() if for_attention else None, n, ctx.seq_lens.data_ptr(), block_table.data_ptr(), width, nkv, hd, n_pages, dt_code(dtype),
        raw_stream()), "kv8_read", 1 if n else 0)
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
    check(launcher("kv8", "sx_kv8_rows")(
        q.data_ptr(), out.data_ptr() + out_col * out.element_size(), *(t.data_ptr() for t in pages), seq_lens.data_ptr(), block_table.data_ptr(),
        block_table.shape[1], S, nh, nkv, hd, n_pages, scale, window or 0, softcap or 0.0, _ptr(sinks), chunk or 0, out.shape[1], out_scale, splits,
        _ptr(part_o), _ptr(part_ml), dt_code(q.dtype), raw_stream()), "kv8_attention", launches=2 if splits > 1 else 1)
    return out


DECODE_HEAD_DIMS = (64, 128)
DECODE_MAX_GROUP = 16
DECODE_MAX_SEQS = 2047
# Portions of up to this many tokens a sequence: every token attends by itself over the codes.  Measured, us, reading back and by token, 32 heads over 8
# of 128: 2 tokens over 2,000 keys 20 and 11.5, over 20,000 80 and 22; 8 tokens 20 and 16, 80 and 48, of 32 sequences with 3,000 keys 260 and 107;
# 16 tokens 20 and 20, 81 and 80, 260 and 199, but 5 x 16 over 9,000 135 and 118 and 32 tokens 84 and 146
FEW_NEW_TOKENS = 8


def kv8_decode_supported(dtype, nh: int, nkv: int, hd: int, S: int) -> bool:
    """Whether single tokens of these sizes attend on the tensor cores (``csrc/kv8_decode.cu``)."""
    return dtype == torch.bfloat16 and hd in DECODE_HEAD_DIMS and nh // nkv <= DECODE_MAX_GROUP and S <= DECODE_MAX_SEQS


_DECODE_PLANS = {}              # of a shape: kernels, floats of scratch


def kv8_decode(q: torch.Tensor, pages: KV8Pages, seq_lens: torch.Tensor, block_table: torch.Tensor, nh: int, scale: float,
               window: Optional[int], max_len: int, sinks: Optional[torch.Tensor] = None,
               row_seq: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One query token a sequence (row ``s`` of ``q``) on the tensor cores; sizes as ``kv8_decode_supported`` says.  With ``row_seq`` a row is any
    token: ``row_seq`` names its sequence and ``seq_lens`` holds its position."""
    k, v, ke, ve = pages
    n_pages, nkv, hd, _ = v.shape
    S, maxp = q.shape[0], block_table.shape[1]
    max_pages = min(-(-max_len // PAGE), maxp)
    if window is not None:
        max_pages = min(max_pages, (window + 126) // PAGE)
    device = q.get_device()
    shape = (S, nh, nkv, hd, max_pages, device)
    plan = _DECODE_PLANS.get(shape)
    if plan is None:
        floats = ctypes.c_longlong(0)
        launches = fn("kv8_decode", "sx_kv8_decode_plan")(*map(c_int, shape[:5]), ctypes.byref(floats))
        plan = _DECODE_PLANS[shape] = (launches, floats.value)
    out = torch.empty_like(q)
    part = torch.empty(plan[1], dtype=torch.float32, device=q.device) if plan[1] else None
    check(launcher("kv8_decode", "sx_kv8_decode")(
        q.data_ptr(), out.data_ptr(), k.data_ptr(), v.data_ptr(), ke.data_ptr(), ve.data_ptr(), seq_lens.data_ptr(), _ptr(row_seq),
        0 if row_seq is None else 1, block_table.data_ptr(), maxp, S, nh, nkv, hd, n_pages, scale, window or 0, _ptr(sinks), _ptr(part), max_pages,
        raw_stream()), "kv8_attention", plan[0])
    return out


def kv8_decode_status(reset: bool = False) -> int:
    """0, or 1: a bounded wait of ``kv8_decode`` ran out in a launch the host has already waited for.  ``reset`` puts it back to 0."""
    v = ctypes.c_int(0)
    check(fn("kv8_decode", "sx_kv8_decode_status")(ctypes.byref(v), c_int(1 if reset else 0)), "kv8_decode_status", launches=0)
    return int(v.value)


TILE_HEAD_DIMS = (64, 128)
TILE_ROWS = 64                  # query heads of a kv head x tokens that a block of csrc/kv8_tile.cu serves
# float32 portions of any length attend over the codes: us, 32 heads over 8 of 128, reading back (with FFMA products) and so: 150 tokens of two
# sequences 57 and 17.5, 64 over 6,000 keys 447 and 52, a prompt of 1,500 638 and 160.  bfloat16 ones of up to one tile of rows a kv head at head size 128
# (16 tokens of 4 heads a kv head over 2,000 keys 17.9 and 16.5, over 20,000 91 and 48, of 32 sequences with 3,000 260 and 156), two at head size 64 (32
# tokens of 4 heads 44 and 13, 374 and 47, 159 and 147); with more the tcgen05 products are worth the pages' way through memory (5 x 32 over 9,000
# at head size 128 135 and 164, 5 x 64 at 64 229 and 252).
TILE_BF16_ROWS = {128: 64, 64: 128}
# And where the pages of all tiles together are few: one launch is 17 us for the host (21 with a cut), reading back and attending 33.  Device time of both, 32
# heads over 8 of 128: a prompt of 128 (128 pages of tiles) 9.4 and 12.0, of 200 (416) 11.0 and 14.9, five of 60 behind 60 (320) 14.8 and 15.0, but 300
# (760) 12.3 and 22.0; at head size 64 300 tokens (760) 11.5 and 13.5, 64 behind 2,000 (1,056) 60 and 17.6, 500 behind 200 (2,816) 23.8 and 26.5, 1,024 (8,192) 36 and 52.
TILE_BF16_PAGES = {128: 512, 64: 2816}


def kv8_tile_supported(q: torch.Tensor, nh: int, nkv: int, hd: int, S: int) -> bool:
    """Whether portions of these sizes attend over the codes (``csrc/kv8_tile.cu``)."""
    return hd in TILE_HEAD_DIMS and nh // nkv <= TILE_ROWS and q.shape[0] > 0 and S <= 65535 and q.data_ptr() % 16 == 0


def _tile_better(S: int, max_new: int, nh: int, nkv: int, hd: int, max_len: int, window: Optional[int]) -> bool:
    """Whether bfloat16 portions go by ``kv8_tile`` (else pages are read back)."""
    if max_new * (nh // nkv) <= TILE_BF16_ROWS[hd]:
        return True
    tokens = TILE_ROWS // (nh // nkv)
    return S * nkv * -(-max_new // tokens) * _tile_pages(max_len, tokens, window) <= TILE_BF16_PAGES[hd]


def _tile_pages(max_len: int, tokens: int, window: Optional[int]) -> int:
    """Pages of a tile of ``tokens`` tokens at most."""
    pages = -(-max_len // PAGE)
    return pages if window is None else min(pages, (window + tokens + 125) // PAGE)


def _tile_splits(S: int, max_new: int, nh: int, nkv: int, max_pages: int, device) -> int:
    """Shares of a tile's pages: as many as fit the GPU at once (two blocks an SM), of four pages or more."""
    blocks = S * nkv * -(-max_new // (TILE_ROWS // (nh // nkv)))
    return max(1, min(-(-max_pages // 4), 2 * sm_count(device) // blocks))


def kv8_tile(q: torch.Tensor, pages: KV8Pages, ctx, block_table: torch.Tensor, nh: int, scale: float, window: Optional[int], *,
             softcap: Optional[float] = None, sinks: Optional[torch.Tensor] = None, chunk: Optional[int] = None,
             out: Optional[torch.Tensor] = None, out_col: int = 0, out_scale: float = 1.0) -> torch.Tensor:
    """Packed queries of portions over the codes; sizes as ``kv8_tile_supported`` says."""
    k, v, ke, ve = pages
    n_pages, nkv, hd, _ = v.shape
    T, S, maxp = q.shape[0], ctx.n_seqs, block_table.shape[1]
    max_pages = min(_tile_pages(ctx.max_len, TILE_ROWS // (nh // nkv), window), maxp)
    splits = _tile_splits(S, ctx.max_new, nh, nkv, max_pages, q.device)
    if out is None:
        out = torch.empty_like(q)
    part = torch.empty(T * nh * splits * (hd + 2), dtype=torch.float32, device=q.device) if splits > 1 else None
    part_o = _ptr(part)
    check(launcher("kv8_tile", "sx_kv8_tile")(
        q.data_ptr(), out.data_ptr() + out_col * out.element_size(), k.data_ptr(), v.data_ptr(), ke.data_ptr(), ve.data_ptr(),
        ctx.cu_seqlens.data_ptr(), ctx.seq_past.data_ptr(), block_table.data_ptr(), maxp, S, T, ctx.max_new, nh, nkv, hd, n_pages, scale, window or 0,
        softcap or 0.0, _ptr(sinks), chunk or 0, out.shape[1], out_scale, splits, part_o, part_o + 4 * T * nh * splits * hd if part_o else 0,
        dt_code(q.dtype), raw_stream()), "kv8_attention", 2 if splits > 1 else 1)
    return out


def kv8_attention(q: torch.Tensor, pages: KV8Pages, ctx, block_table: torch.Tensor, nh: int, nkv: int, hd: int, scale: float,
                  window: Optional[int] = None, *, softcap: Optional[float] = None, sinks: Optional[torch.Tensor] = None,
                  chunk: Optional[int] = None, out: Optional[torch.Tensor] = None, out_col: int = 0,
                  out_scale: float = 1.0) -> torch.Tensor:
    """Causal attention of the step's packed queries ``q [T, nh * hd]`` over a cache in eight bits that already holds the step's
    keys and values: ``[T, nh * hd]`` in ``q``'s dtype.  The options are those of ``ops.attention``.

    ``q`` has a row for every token of the step; places of the cache that the step's tokens do not see may hold anything.  Kernels on the codes load
    queries 16 bytes at a time and refuse a ``q`` that does not begin at a multiple of 16.

    A bfloat16 query goes into the products over the codes as two e4m3 numbers: elements down to 2^-9 of the row's largest are exact, smaller ones off by at most
    2^-18 of it; rows whose largest magnitude is below 2^-99 lose more.  Weights are rounded to half precision there, to bfloat16 by the 16-bit cache's
    kernels (denominators sum them as they are), and kept to 22 bits in float32.  Results are divided at the end: values times the number of keys seen stay below 2^127.

    Single tokens, portions of a few tokens and float32 portions attend over the codes.  Longer portions read the pages back once
    (``kv8_read``) and attend over the result with the kernels of the 16- and 32-bit cache: a page serves many rows there, and
    turning its codes again in every block that reads it would cost more than writing it out once.  What is read back takes ``2 nkv hd`` elements of ``q``'s
    dtype a token of the step's sequences (131,072 tokens of 8 heads of 128 in bfloat16: 537 MB) until the call's kernels are done."""
    _check_pages(pages, "kv8_attention", nkv, hd)
    seq_lens = ctx.seq_lens
    if seq_lens.dtype is not torch.int32 or block_table.dtype is not torch.int32:
        raise KernelError("kv8_attention: index tensors are int32")
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
        if block_table.dim() != 2 or block_table.shape[0] < ctx.n_seqs or seq_lens.numel() < ctx.n_seqs:
            raise KernelError("kv8_attention: a row of the table and a length per sequence")
        k, v, ke, ve = pages
        _check_device("kv8_attention", q, k, v, ke, ve, seq_lens, block_table, sinks, out)
        if out is None and softcap is None and chunk is None and out_scale == 1.0 and kv8_decode_supported(q.dtype, nh, nkv, hd, q.shape[0]):
            return kv8_decode(q, pages, seq_lens, block_table, nh, scale, window, ctx.max_len, sinks)
        return kv8_rows(q, pages, seq_lens, block_table, nh, scale, window, ctx.max_len, softcap=softcap, sinks=sinks, chunk=chunk,
                        out=out, out_col=out_col, out_scale=out_scale)
    T = q.shape[0]
    if ctx.host is not None and ctx.host["cu_seqlens"][ctx.n_seqs] != T:
        raise KernelError("kv8_attention: q has a row for every token of the step and no others")
    if (ctx.max_new <= FEW_NEW_TOKENS and out is None and softcap is None and chunk is None and out_scale == 1.0
            and kv8_decode_supported(q.dtype, nh, nkv, hd, q.shape[0])):
        if not (ctx.positions.dtype == ctx.seq_of_token.dtype == torch.int32) or min(ctx.positions.numel(), ctx.seq_of_token.numel()) < T or block_table.dim() != 2:
            raise KernelError("kv8_attention: a position and a sequence per token (int32), and a table [sequences, pages]")
        _check_device("kv8_attention", q, *pages, ctx.positions, ctx.seq_of_token, block_table, sinks)
        return kv8_decode(q, pages, ctx.positions, block_table, nh, scale, window, ctx.max_len, sinks, ctx.seq_of_token)
    _check_host("kv8_attention", ctx, block_table)
    S = ctx.n_seqs
    if (not (ctx.cu_seqlens.dtype == ctx.seq_past.dtype == ctx.seq_of_token.dtype == torch.int32) or ctx.cu_seqlens.numel() <= S
            or ctx.seq_past.numel() < S or ctx.seq_of_token.numel() < T):
        raise KernelError("kv8_attention: a first token and a length before the step per sequence, and a sequence per token (int32)")
    if kv8_tile_supported(q, nh, nkv, hd, S) and (q.dtype == torch.float32 or _tile_better(S, ctx.max_new, nh, nkv, hd, ctx.max_len, window)):
        _check_device("kv8_attention", q, *pages, ctx.cu_seqlens, ctx.seq_past, block_table, sinks, out)
        return kv8_tile(q, pages, ctx, block_table, nh, scale, window, softcap=softcap, sinks=sinks, chunk=chunk, out=out, out_col=out_col,
                        out_scale=out_scale)
    from . import TC_TILE_ROWS, _query_tiles, attention, tc_prefill_supported
    from .attention import attn_prefill_tc_parts, tc_part_rows, tc_parts
    _check_device("kv8_attention", q, *pages, ctx.seq_lens, block_table, sinks, out)
    k, v, table = _read(pages, ctx, block_table, q.dtype, window, chunk, True)
    if out is None and softcap is None and chunk is None and out_scale == 1.0 and tc_prefill_supported(q.dtype, nh, nkv, hd):
        cu, past = ctx.host["cu_seqlens"], ctx.host["seq_past"]
        cut = ctx.scratch.get(("kv8_parts", nh, window))
        if cut is None or cut[4] != cu or cut[5] != past:
            tiles = [(p + q0, min(p + q0 + TC_TILE_ROWS, p + b - a) - 1) for a, b, p in zip(cu, cu[1:], past) for q0 in range(0, b - a, TC_TILE_ROWS)]
            blocks, parts = tc_parts(tiles, nh, window, q.device)
            places = rows = None
            if parts > 1:
                places, rows = tc_part_rows(tiles, blocks, window)
                places = torch.from_numpy(np.asarray(places, dtype=np.int32)).to(q.device, non_blocking=True)
            cut = ctx.scratch[("kv8_parts", nh, window)] = (blocks, parts, places, rows, list(cu), list(past))
        if cut[1] > 1:
            tile_seq, tile_q0 = _query_tiles(ctx, TC_TILE_ROWS, q.device)
            return attn_prefill_tc_parts(q, k, v, tile_seq, tile_q0, cut[2], cut[3], ctx.cu_seqlens, ctx.seq_past, ctx.seq_lens, table, nh, nkv, hd,
                                         scale, window, cut[0], cut[1], sinks=sinks)
    return attention(q, k, v, ctx, table, nh, nkv, hd, scale, window, softcap=softcap, sinks=sinks, chunk=chunk, out=out, out_col=out_col,
                     out_scale=out_scale)
