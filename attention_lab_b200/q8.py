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
import functools
import math
from typing import NamedTuple

import torch

from . import _lib

BLOCK = 64                     # tokens that share one exponent
HEAD_DIM = 128
LAYOUTS = {"half": 0, "interleaved": 1}
_CODES = torch.float8_e4m3fn
_DTYPES = {torch.float32: _lib.AL_F32, torch.bfloat16: _lib.AL_BF16}

# These operators also serve calls of a few microseconds (a decode step of one request), where the wrapper's own time
# counts: tensors are compared by device ordinal, the stream handle is taken without building a Stream object, and the
# device is switched only when it is not the current one.
_raw_stream = torch._C._cuda_getCurrentRawStream


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


def _call_on(dev: int, entry, *args) -> None:
    """entry(*args) with device `dev` current."""
    if torch.cuda.current_device() == dev:
        rc = entry(*args)
    else:
        with torch.cuda.device(dev):
            rc = entry(*args)
    if rc:
        _lib.check(rc)


def _call(dev: int, entry, *args) -> None:
    """entry(*args, stream) on device `dev`, on its current stream."""
    _call_on(dev, entry, *args, _raw_stream(dev))


def _same_device(dev: int, *ts) -> None:
    if dev < 0:
        raise ValueError("every tensor must live on a CUDA device (the CUDA path has no CPU fallback)")
    for t in ts:
        if t is not None and t.get_device() != dev:
            if not t.is_cuda:
                raise ValueError("every tensor must live on a CUDA device (the CUDA path has no CPU fallback)")
            raise ValueError("all inputs must live on the same device")


def _code(dtype, what: str) -> int:
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"{what} must be float32 or bfloat16, got {dtype}")
    return code


def _check_q8(cache):
    """(codes and exponents as given, their shape, device ordinal)"""
    k, v, ke, ve = cache
    shape = k.shape
    if len(shape) != 4 or v.shape != shape:
        raise ValueError(f"the codes must be [B,G,C,d] of one shape, got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype != _CODES or v.dtype != _CODES:
        raise ValueError(f"the codes must be float8_e4m3fn, got {k.dtype} and {v.dtype}")
    B, G, C, d = shape
    if ke.shape != (B, G, -(-C // BLOCK)) or ve.shape != ke.shape or ke.dtype != torch.int8 or ve.dtype != torch.int8:
        raise ValueError("the exponents must be int8 [B,G,ceil(C/64)]")
    if not (k.is_contiguous() and v.is_contiguous() and ke.is_contiguous() and ve.is_contiguous()):
        raise ValueError("codes and exponents must be contiguous")
    dev = k.get_device()
    _same_device(dev, v, ke, ve)
    return B, G, C, d, dev


def _check_lengths(lengths, B: int, dev: int, what: str, least: int, most: int):
    """(device pointer or None, int)"""
    if isinstance(lengths, torch.Tensor):
        if lengths.dtype != torch.int32 or lengths.shape != (B,) or not lengths.is_contiguous():
            raise ValueError("lengths must be an int or a contiguous int32 tensor [B]")
        _same_device(dev, lengths)
        return lengths.data_ptr(), 0
    n = int(lengths)
    if not least <= n <= most:
        raise ValueError(f"{what}: length {n} outside [{least}, {most}]")
    return None, n


def _rows(x: torch.Tensor):
    """(x, its address, its strides); a contiguous copy of x when its rows cannot be read in 16-byte pieces."""
    s, p = x.stride(), x.data_ptr()
    bits = 0
    for i in s[:-1]:
        bits |= i
    if s[-1] != 1 or p & 15 or bits & (16 // x.element_size() - 1):
        x = x.contiguous()
        if x.data_ptr() & 15:
            x = x.clone()
        s, p = x.stride(), x.data_ptr()
    return x, p, s


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
    lay = _check_table(table, layout)
    shape = q.shape
    if len(shape) != 4:
        raise ValueError(f"q must be [B,H,T,d], got {tuple(q.shape)}")
    B, H, T, d = shape
    dev, dtype = q.get_device(), q.dtype
    code = _code(dtype, "q")
    _same_device(dev, table, k)
    q, qp, qs = _rows(q)
    Hk, kp, ks, ko, k_out = 0, None, (0, 0, 0), None, None
    if k is not None:
        Hk = k.shape[1] if k.dim() == 4 else 0
        if k.shape != (B, Hk, T, d) or k.dtype != dtype:
            raise ValueError("k must be [B,G,T,d] of q's dtype")
        k, kp, ks = _rows(k)
        k_out = q.new_empty((B, Hk, T, d))
        ko = k_out.data_ptr()
    pp, pst, start = None, (0, 0), 0
    if isinstance(positions, torch.Tensor):
        if positions.dtype != torch.int64:
            raise ValueError("positions must be int64")
        _same_device(dev, positions)
        if positions.dim() < 2 or positions.shape[0] == 1:
            positions = positions.expand(B, T)
        if positions.shape != (B, T):
            raise ValueError(f"positions must be [B,T] = [{B},{T}], got {tuple(positions.shape)}")
        pp, pst = positions.data_ptr(), positions.stride()
    else:
        start = int(positions)
        if start < 0 or start + T > table.shape[0]:
            raise ValueError(f"positions [{start}, {start + T}) outside the table's {table.shape[0]} rows")
    out = q.new_empty(shape)
    _call(dev, _lib.load().al_rotary, qp, qs[0], qs[1], qs[2], H, kp, ks[0], ks[1], ks[2], Hk, code, table.data_ptr(),
          table.shape[0], table.shape[1], lay, pp, pst[0], pst[1], start, B, T, d, int(bool(inverse)), out.data_ptr(), ko)
    return out, k_out


def append_q8(cache, lengths, k_new: torch.Tensor, v_new: torch.Tensor, *, q=None, table=None, layout: str = "half"):
    """Write k_new, v_new [B,G,T,d] at the ends of the requests (see `lengths` above). With a rotary `table` k_new is
    rotated to its positions first (in float32, then rounded to codes once), and q [B,G,h,T,d], when given, is returned
    rotated ([B,G,h,T,d] contiguous, zeros in padding rows); without a table q must be None. One launch."""
    k, v, ke, ve = cache
    B, G, C, d, dev = _check_q8(cache)
    shape, dtype = k_new.shape, k_new.dtype
    if len(shape) != 4 or shape[0] != B or shape[1] != G or shape[3] != d or v_new.shape != shape:
        raise ValueError("k_new and v_new must be [B,G,T,d] matching the cache")
    if v_new.dtype != dtype:
        raise ValueError("k_new and v_new must share one dtype")
    _same_device(dev, k_new, v_new, table, q)
    T, code = shape[2], _code(dtype, "k_new")
    lp, length = _check_lengths(lengths, B, dev, "append", T, C)
    tp, trows, rot, lay = None, 0, 0, 0
    if table is not None:
        lay = _check_table(table, layout)
        tp, (trows, rot) = table.data_ptr(), table.shape
    qp, qs, h, q_out, qo = None, (0, 0, 0, 0), 0, None, None
    if q is not None:
        if table is None:
            raise ValueError("q is rotated: it needs a table")
        h = q.shape[2] if q.dim() == 5 else 0
        if q.shape != (B, G, h, T, d) or q.dtype != dtype:
            raise ValueError("q must be [B,G,h,T,d] of k_new's dtype")
        q, qp, qs = _rows(q)
        q_out = q.new_empty((B, G, h, T, d))
        qo = q_out.data_ptr()
    k_new, kp, ks = _rows(k_new)
    v_new, vp, vs = _rows(v_new)
    _call(dev, _lib.load().al_append_q8, k.data_ptr(), v.data_ptr(), ke.data_ptr(), ve.data_ptr(), lp, length,
          kp, ks[0], ks[1], ks[2], vp, vs[0], vs[1], vs[2], code, tp, trows, rot, lay,
          qp, qs[0], qs[1], qs[2], qs[3], h, qo, B, G, T, C, d)
    return q_out


def read_q8(cache, lo: int, hi: int, *, dtype=torch.bfloat16):
    """Positions [lo, hi) of the cache as values: (k, v), each [B,G,hi-lo,d] of dtype."""
    k, v, ke, ve = cache
    B, G, C, d, dev = _check_q8(cache)
    lo, hi = int(lo), int(hi)
    if not 0 <= lo <= hi <= C:
        raise ValueError(f"need 0 <= lo <= hi <= capacity {C}, got lo={lo} hi={hi}")
    code = _code(dtype, "dtype")
    k_out = torch.empty((B, G, hi - lo, d), dtype=dtype, device=k.device)
    v_out = torch.empty_like(k_out)
    _call(dev, _lib.load().al_read_q8, k.data_ptr(), v.data_ptr(), ke.data_ptr(), ve.data_ptr(), B, G, C, d, lo, hi, code,
          k_out.data_ptr(), v_out.data_ptr())
    return k_out, v_out


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(dev: int, B: int, G: int, h: int, T: int, C: int, window: int, sinks: int, most: int) -> int:
    """What al_attend_q8 needs for a call of these sizes (the answer depends on nothing else)."""
    need = ctypes.c_size_t(0)
    _call_on(dev, _lib.load().al_attend_q8_workspace, B, G, h, T, C, window, sinks, most, ctypes.byref(need))
    return need.value


def attend_q8(q: torch.Tensor, cache, lengths, *, window: int = 0, sinks: int = 0, scale=None, max_length=None):
    """Attention of q [B,G,h,T,d] over the cache, causal: the query at position p sees the tokens j <= p, with a
    `window` > 0 only those with j > p - window or j < sinks. A row that sees nothing is zero. `max_length` (default: the
    capacity) is what the caller knows of the largest length; it chooses how the work is split, never the result's rows.
    Returns [B,G,h,T,d] of q's dtype."""
    k, v, ke, ve = cache
    B, G, C, d, dev = _check_q8(cache)
    shape = q.shape
    if len(shape) != 5 or shape[0] != B or shape[1] != G or shape[4] != d:
        raise ValueError(f"q must be [B,G,h,T,d] matching the cache, got {tuple(q.shape)}")
    _same_device(dev, q)
    h, T = shape[2], shape[3]
    code = _code(q.dtype, "q")
    window, sinks = int(window), int(sinks)
    if window < 0 or sinks < 0:
        raise ValueError(f"window and sinks must not be negative, got {window} and {sinks}")
    lp, length = _check_lengths(lengths, B, dev, "attend", 0, C)
    most = length if lp is None else (C if max_length is None else int(max_length))
    q, qp, qs = _rows(q)
    out = q.new_empty(shape)
    lib = _lib.load()
    wn = _workspace_bytes(dev, B, G, h, T, C, window, sinks, most)
    work = torch.empty(wn, dtype=torch.uint8, device=q.device) if wn else None
    wp = work.data_ptr() if wn else None
    _call(dev, lib.al_attend_q8, qp, qs[0], qs[1], qs[2], qs[3], code, k.data_ptr(), v.data_ptr(), ke.data_ptr(),
          ve.data_ptr(), lp, length, B, G, h, T, C, d, window, sinks, 1.0 / math.sqrt(d) if scale is None else float(scale),
          most, out.data_ptr(), wp, wn)
    return out
