"""The 8-bit K/V cache: rotary positions, the quantising write, the read-back and attention over it.

    rotary_table, rotary_embed   positions: half or interleaved pairs, part of the head, scaled for long contexts
    append_q8                    new rows into the cache as they are written (rotating K, and q, on the way)
    read_q8                      a range of the cache as float32 or bfloat16
    attend_q8                    attention over the cache: single tokens, prompt chunks, sliding window with sinks

One layer's cache (`Q8Cache`) holds K and V as e4m3 codes [B,G,C,128] and one int8 exponent per block of 64 tokens of
each (batch, group): value = code * 2^exponent, the exponent the smallest with amax <= 448 * 2^e. A value is rounded
when it is written; if a later token of its block raises the exponent, the codes already there are rounded again (a
shift by a power of two: exact except where it enters e4m3's subnormals). NaN and infinities become the NaN code.

`lengths` says how many tokens of each request are in the cache once this step's T rows are: an int for every request,
or an int32 device tensor [B]. Row t of T sits at position length - T + t; rows at negative positions are padding (a
ragged batch of prompts is padded on the left). A device length outside [0, C] is clamped and sets error bit 4
(`_lib.device_status()`); an int is checked here.

As in `ops`: tensors live on one CUDA device, float32 or bfloat16, head_dim 128, work goes to the current stream,
nothing synchronises, ValueError for shapes, dtypes and ranges.
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch

from . import _lib
from .ops import _code, _cuda, _scale, _stream

BLOCK = 64                     # tokens that share one exponent
HEAD_DIM = 128
LAYOUTS = {"half": 0, "interleaved": 1}
_CODES = torch.float8_e4m3fn


class Q8Cache(NamedTuple):
    """One layer's cache: codes k, v float8_e4m3fn [B,G,C,128] and exponents k_exp, v_exp int8 [B,G,ceil(C/64)]."""

    k: torch.Tensor
    v: torch.Tensor
    k_exp: torch.Tensor
    v_exp: torch.Tensor

    @classmethod
    def empty(cls, batch: int, groups: int, capacity: int, device, head_dim: int = HEAD_DIM) -> "Q8Cache":
        """An empty cache. Codes are left as the allocator gave them: no operator reads a row past a length."""
        if int(capacity) <= 0:
            raise ValueError("capacity must be positive")
        shape, nb = (batch, groups, capacity, head_dim), (batch, groups, -(-capacity // BLOCK))
        return cls(torch.empty(shape, dtype=_CODES, device=device), torch.empty(shape, dtype=_CODES, device=device),
                   torch.zeros(nb, dtype=torch.int8, device=device), torch.zeros(nb, dtype=torch.int8, device=device))


def _check_q8(cache):
    k, v, ke, ve = cache
    if k.dim() != 4 or k.shape != v.shape:
        raise ValueError(f"the codes must be [B,G,C,d] of one shape, got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype != _CODES or v.dtype != _CODES:
        raise ValueError(f"the codes must be float8_e4m3fn, got {k.dtype} and {v.dtype}")
    B, G, C, d = k.shape
    if ke.shape != (B, G, -(-C // BLOCK)) or ve.shape != ke.shape or ke.dtype != torch.int8 or ve.dtype != torch.int8:
        raise ValueError("the exponents must be int8 [B,G,ceil(C/64)]")
    if not (k.is_contiguous() and v.is_contiguous() and ke.is_contiguous() and ve.is_contiguous()):
        raise ValueError("codes and exponents must be contiguous")
    return B, G, C, d


def _check_lengths(lengths, B: int, what: str, least: int, most: int):
    """(device pointer or None, int)"""
    if isinstance(lengths, torch.Tensor):
        if lengths.dtype != torch.int32 or lengths.shape != (B,) or not lengths.is_contiguous():
            raise ValueError("lengths must be an int or a contiguous int32 tensor [B]")
        return lengths.data_ptr(), 0
    n = int(lengths)
    if not least <= n <= most:
        raise ValueError(f"{what}: length {n} outside [{least}, {most}]")
    return None, n


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x itself when its rows can be read in 16-byte pieces, else a contiguous copy."""
    unit = 16 // x.element_size()
    s = x.stride()
    if s[-1] == 1 and x.data_ptr() % 16 == 0:
        for i in s[:-1]:
            if i % unit:
                break
        else:
            return x
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _check_table(table: torch.Tensor, layout: str) -> int:
    if layout not in LAYOUTS:
        raise ValueError(f"unknown layout {layout!r}; choose from {tuple(LAYOUTS)}")
    if table.dim() != 2 or table.dtype != torch.float32 or not table.is_contiguous():
        raise ValueError("the rotary table must be a contiguous float32 [length, rotary_dim] tensor")
    return LAYOUTS[layout]


def rotary_table(length: int, rotary_dim: int = HEAD_DIM, *, base: float = 10000.0, scaling=None,
                 device="cuda") -> torch.Tensor:
    """The rotary table [length, rotary_dim] (float32: cosines, then sines) of positions 0 .. length - 1 at frequencies
    base^(-2i/rotary_dim), computed in float64. `scaling` stretches the context by `factor`:

        {"type": "linear", "factor": s}      every position divided by s
        {"type": "ntk", "factor": s}         base times s^(rotary_dim / (rotary_dim - 2))
        {"type": "yarn", "factor": s, "original": n}   frequencies that turn more than `fast` (32) times in the original
            context of n positions kept, those that turn less than `slow` (1) times divided by s, a ramp between; table
            entries times `amplitude` (default 0.1 ln s + 1)
    """
    length, rot = int(length), int(rotary_dim)
    if length < 1 or rot < 2 or rot % 2:
        raise ValueError("need length >= 1 and an even rotary_dim >= 2")
    scaling = dict(scaling or {"type": "none"})
    kind, s = scaling.pop("type", None), float(scaling.pop("factor", 1.0))
    if not s > 0:
        raise ValueError("the scaling factor must be positive")
    i = torch.arange(rot // 2, dtype=torch.float64, device=device)
    pos = torch.arange(length, dtype=torch.float64, device=device)
    amp = 1.0
    if kind == "ntk":
        if rot < 4:
            raise ValueError("ntk scaling needs rotary_dim >= 4")
        base = base * s ** (rot / (rot - 2))
    freq = float(base) ** (-2.0 * i / rot)
    if kind == "linear":
        pos = pos / s
    elif kind == "yarn":
        if "original" not in scaling:
            raise ValueError("yarn scaling needs the original context length")
        fast, slow = float(scaling.pop("fast", 32.0)), float(scaling.pop("slow", 1.0))
        if not fast > slow:
            raise ValueError("yarn scaling needs fast > slow")
        turns = freq * float(scaling.pop("original")) / (2 * math.pi)
        keep = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
        freq = freq * keep + freq / s * (1.0 - keep)
        amp = float(scaling.pop("amplitude", 0.1 * math.log(s) + 1.0))
    elif kind not in ("none", "ntk"):
        raise ValueError(f"unknown scaling type {kind!r}")
    if scaling:
        raise ValueError(f"unknown scaling entries {sorted(scaling)}")
    ang = pos[:, None] * freq
    return torch.cat([ang.cos() * amp, ang.sin() * amp], dim=1).float().contiguous()


def rotary_embed(q: torch.Tensor, k, table: torch.Tensor, positions, *, layout: str = "half", inverse: bool = False):
    """q [B,H,T,d] and k [B,G,T,d] (or None) rotated to their positions, in one launch: pairs (a, b) become
    (a c - b s, b c + a s) in float32, rounded once; dimensions past the table's rotary_dim are copied. `positions` is
    an int (row t at positions + t) or int64 [B,T] (or [T]); negative ones are padding (zeros), one past the table gives
    zeros and error bit 4. `inverse` rotates back: the gradient of the forward rotation. Returns (q', k')."""
    dev = _cuda(q, k, table, positions if isinstance(positions, torch.Tensor) else None)
    lay = _check_table(table, layout)
    if q.dim() != 4:
        raise ValueError(f"q must be [B,H,T,d], got {tuple(q.shape)}")
    B, H, T, d = q.shape
    code = _code(q, "q")
    q = _rows(q)
    Hk, kp, ks, ko, k_out = 0, None, None, None, None
    if k is not None:
        if k.dim() != 4 or k.shape[0] != B or k.shape[2] != T or k.shape[3] != d or k.dtype != q.dtype:
            raise ValueError("k must be [B,G,T,d] of q's dtype")
        k = _rows(k)
        Hk, kp, ks = k.shape[1], k.data_ptr(), _lib.strides(k, 3)
        k_out = torch.empty((B, Hk, T, d), dtype=q.dtype, device=dev)
        ko = k_out.data_ptr()
    pp, pst, start = None, None, 0
    if isinstance(positions, torch.Tensor):
        if positions.dtype != torch.int64:
            raise ValueError("positions must be int64")
        pos = positions.expand(B, T) if positions.dim() < 2 or positions.shape[0] == 1 else positions
        if tuple(pos.shape) != (B, T):
            raise ValueError(f"positions must be [B,T] = [{B},{T}], got {tuple(positions.shape)}")
        pp, pst = pos.data_ptr(), _lib.strides(pos, 2)
    else:
        start = int(positions)
        if start < 0 or start + T > table.shape[0]:
            raise ValueError(f"positions [{start}, {start + T}) outside the table's {table.shape[0]} rows")
    out = torch.empty((B, H, T, d), dtype=q.dtype, device=dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.load().al_rotary(
            q.data_ptr(), _lib.strides(q, 3), H, kp, ks, Hk, code, table.data_ptr(), table.shape[0], table.shape[1], lay,
            pp, pst, start, B, T, d, int(bool(inverse)), out.data_ptr(), ko, _stream(dev)))
    return out, k_out


def append_q8(cache, lengths, k_new: torch.Tensor, v_new: torch.Tensor, *, q=None, table=None, layout: str = "half"):
    """Write k_new, v_new [B,G,T,d] at the ends of the requests (see `lengths` above). With a rotary `table` k_new is
    rotated to its positions first (in float32, then rounded to codes once), and q [B,G,h,T,d], when given, is returned
    rotated ([B,G,h,T,d] contiguous, zeros in padding rows); without a table q must be None. One launch."""
    k, v, ke, ve = cache
    dev = _cuda(k, v, ke, ve, k_new, v_new, q, table, lengths if isinstance(lengths, torch.Tensor) else None)
    B, G, C, d = _check_q8(cache)
    if k_new.dim() != 4 or k_new.shape[0] != B or k_new.shape[1] != G or k_new.shape[3] != d or v_new.shape != k_new.shape:
        raise ValueError("k_new and v_new must be [B,G,T,d] matching the cache")
    if v_new.dtype != k_new.dtype:
        raise ValueError("k_new and v_new must share one dtype")
    T, code = k_new.shape[2], _code(k_new, "k_new")
    lp, length = _check_lengths(lengths, B, "append", T, C)
    tp, trows, rot, lay = None, 0, 0, 0
    if table is not None:
        lay = _check_table(table, layout)
        tp, trows, rot = table.data_ptr(), table.shape[0], table.shape[1]
    qp, qst, h, q_out, qo = None, None, 0, None, None
    if q is not None:
        if table is None:
            raise ValueError("q is rotated: it needs a table")
        if q.dim() != 5 or q.shape[0] != B or q.shape[1] != G or q.shape[3] != T or q.shape[4] != d or q.dtype != k_new.dtype:
            raise ValueError("q must be [B,G,h,T,d] of k_new's dtype")
        q = _rows(q)
        h = q.shape[2]
        q_out = torch.empty((B, G, h, T, d), dtype=q.dtype, device=dev)
        qp, qst, qo = q.data_ptr(), _lib.strides(q, 4), q_out.data_ptr()
    k_new, v_new = _rows(k_new), _rows(v_new)
    with torch.cuda.device(dev):
        _lib.check(_lib.load().al_append_q8(
            k.data_ptr(), v.data_ptr(), ke.data_ptr(), ve.data_ptr(), lp, length, k_new.data_ptr(),
            _lib.strides(k_new, 3), v_new.data_ptr(), _lib.strides(v_new, 3), code, tp, trows, rot, lay, qp, qst, h, qo,
            B, G, T, C, d, _stream(dev)))
    return q_out


def read_q8(cache, lo: int, hi: int, *, dtype=torch.bfloat16):
    """Positions [lo, hi) of the cache as values: (k, v), each [B,G,hi-lo,d] of dtype."""
    k, v, ke, ve = cache
    dev = _cuda(k, v, ke, ve)
    B, G, C, d = _check_q8(cache)
    lo, hi = int(lo), int(hi)
    if not 0 <= lo <= hi <= C:
        raise ValueError(f"need 0 <= lo <= hi <= capacity {C}, got lo={lo} hi={hi}")
    ko, vo = (torch.empty((B, G, hi - lo, d), dtype=dtype, device=dev) for _ in range(2))
    code = _code(ko, "dtype")
    with torch.cuda.device(dev):
        _lib.check(_lib.load().al_read_q8(k.data_ptr(), v.data_ptr(), ke.data_ptr(), ve.data_ptr(), B, G, C, d, lo, hi,
                                          code, ko.data_ptr(), vo.data_ptr(), _stream(dev)))
    return ko, vo


def attend_q8(q: torch.Tensor, cache, lengths, *, window: int = 0, sinks: int = 0, scale=None, max_length=None):
    """Attention of q [B,G,h,T,d] over the cache, causal: the query at position p sees the tokens j <= p, with a
    `window` > 0 only those with j > p - window or j < sinks. A row that sees nothing is zero. `max_length` (default: the
    capacity) is what the caller knows of the largest length; it chooses how the work is split, never the result's rows.
    Returns [B,G,h,T,d] of q's dtype."""
    k, v, ke, ve = cache
    dev = _cuda(q, k, v, ke, ve, lengths if isinstance(lengths, torch.Tensor) else None)
    B, G, C, d = _check_q8(cache)
    if q.dim() != 5 or q.shape[0] != B or q.shape[1] != G or q.shape[4] != d:
        raise ValueError(f"q must be [B,G,h,T,d] matching the cache, got {tuple(q.shape)}")
    _, _, h, T, _ = q.shape
    code = _code(q, "q")
    window, sinks = int(window), int(sinks)
    if window < 0 or sinks < 0:
        raise ValueError(f"window and sinks must not be negative, got {window} and {sinks}")
    lp, length = _check_lengths(lengths, B, "attend", 0, C)
    most = length if lp is None else (C if max_length is None else int(max_length))
    q = _rows(q)
    out = torch.empty((B, G, h, T, d), dtype=q.dtype, device=dev)
    lib = _lib.load()
    need = ctypes.c_size_t(0)
    with torch.cuda.device(dev):
        _lib.check(lib.al_attend_q8_workspace(B, G, h, T, C, window, sinks, most, ctypes.byref(need)))
        work = torch.empty(need.value, dtype=torch.uint8, device=dev) if need.value else None
        _lib.check(lib.al_attend_q8(
            q.data_ptr(), _lib.strides(q, 4), code, k.data_ptr(), v.data_ptr(), ke.data_ptr(), ve.data_ptr(), lp, length,
            B, G, h, T, C, d, window, sinks, _scale(d, scale), most, out.data_ptr(),
            None if work is None else work.data_ptr(), need.value, _stream(dev)))
    return out
