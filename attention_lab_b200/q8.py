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
nothing synchronises, ValueError for shapes, dtypes and ranges. rotary_embed takes part in autograd; the cache holds
codes, through which no gradient passes: append_q8 and attend_q8 return tensors without one.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch


class _Binding:
    """The operators' compiled binding (csrc/bind_q8.cpp: argument checks, outputs and the C-ABI call), loaded with the
    CUDA library it is linked to at the first call of an operator: importing this module maps neither."""

    NAMES = ("rotary_embed", "append_q8", "read_q8", "attend_q8")

    def __getattr__(self, name):                 # reached until the functions below are attributes
        if name not in self.NAMES:
            raise AttributeError(name)
        try:
            from . import _q8_bind
        except ImportError as e:
            raise RuntimeError(f"the 8-bit cache's binding is not built ({e}): run `python -m attention_lab_b200.build` "
                               "(these operators have no fallback)") from e
        for n in self.NAMES:
            setattr(self, n, getattr(_q8_bind, n))
        return getattr(self, name)


_bind = _Binding()

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


def _layout(layout: str) -> int:
    try:
        return LAYOUTS[layout]
    except KeyError:
        raise ValueError(f"unknown layout {layout!r}; choose from {tuple(LAYOUTS)}") from None


def rotary_table(length: int, rotary_dim: int = HEAD_DIM, *, base: float = 10000.0, scaling=None, frequencies=None,
                 amplitude: float = 1.0, device="cuda") -> torch.Tensor:
    """The rotary table [length, rotary_dim] (float32: cosines, then sines) of positions 0 .. length - 1 at frequencies
    base^(-2i/rotary_dim), computed in float64. `scaling` stretches the context by `factor`:

        {"type": "linear", "factor": s}      every position divided by s
        {"type": "ntk", "factor": s}         base times s^(rotary_dim / (rotary_dim - 2))
        {"type": "yarn", "factor": s, "original": n}   frequencies that turn more than `fast` (32) times in the original
            context of n positions kept, those that turn less than `slow` (1) times divided by s, between them a ramp that
            is linear in the pair's index, from the whole index below the one of `fast` turns to the one above that of
            `slow` (checkpoints trained with YaRN run with this ramp, not with the one linear in turns); table entries
            times `amplitude` (default 0.1 ln s + 1, and 1 for s <= 1)
    """
    length, rot = int(length), int(rotary_dim)
    if length < 1 or rot < 2 or rot % 2:
        raise ValueError("need length >= 1 and an even rotary_dim >= 2")
    if frequencies is not None:
        if scaling is not None or frequencies.shape != (rot // 2,):
            raise ValueError("frequencies must be [rotary_dim / 2], without scaling")
        ang = torch.arange(length, dtype=torch.float64, device=device)[:, None] * frequencies.to(device).double()
        return (torch.cat([ang.cos(), ang.sin()], dim=1) * amplitude).float().contiguous()
    scaling = dict(scaling or {"type": "none"})
    kind, s = scaling.pop("type", None), float(scaling.pop("factor", 1.0))
    if not s > 0:
        raise ValueError("the scaling factor must be positive")
    i = torch.arange(rot // 2, dtype=torch.float64, device=device)
    pos = torch.arange(length, dtype=torch.float64, device=device)
    amp = float(amplitude)
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
        original = float(scaling.pop("original"))
        if not (fast > slow > 0 and original > 0 and base > 1):
            raise ValueError("yarn scaling needs fast > slow > 0, original > 0 and base > 1")
        # pair i turns original base^(-2i/rot) / (2 pi) times: the index of so many turns, not rounded
        index = lambda turns: rot * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base))
        first, last = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), rot - 1)
        keep = 1.0 - ((i - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)
        freq = freq * keep + freq / s * (1.0 - keep)
        amp *= float(scaling.pop("amplitude", 0.1 * math.log(s) + 1.0 if s > 1 else 1.0))
    elif kind not in ("none", "ntk"):
        raise ValueError(f"unknown scaling type {kind!r}")
    if scaling:
        raise ValueError(f"unknown scaling entries {sorted(scaling)}")
    ang = pos[:, None] * freq
    return torch.cat([ang.cos() * amp, ang.sin() * amp], dim=1).float().contiguous()


class _Rotation(torch.autograd.Function):
    """The rotation as an operation of autograd: a pair's gradient is the output's, turned the other way."""

    @staticmethod
    def forward(ctx, q, k, table, positions, layout, inverse):
        at = positions if isinstance(positions, torch.Tensor) else None
        ctx.save_for_backward(table, at)
        ctx.start, ctx.layout, ctx.inverse = (positions if at is None else None), layout, inverse
        return _bind.rotary_embed(q, k, table, positions, layout, inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        table, at = ctx.saved_tensors
        turn = lambda x, y: _rotate(x, y, table, ctx.start if at is None else at, ctx.layout, not ctx.inverse)
        if ctx.needs_input_grad[0]:
            gq, gk = turn(dq, dk if ctx.needs_input_grad[1] else None)
        else:
            gq, gk = None, turn(dk, None)[0]
        return gq, gk, None, None, None, None


def _rotate(q, k, table, positions, layout, inverse):
    if torch.is_grad_enabled() and (getattr(q, "requires_grad", False) or getattr(k, "requires_grad", False)):
        return _Rotation.apply(q, k, table, positions, layout, inverse)
    return _bind.rotary_embed(q, k, table, positions, layout, inverse)


def rotary_embed(q: torch.Tensor, k, table: torch.Tensor, positions, *, layout: str = "half", inverse: bool = False):
    """q [B,H,T,d] and k [B,G,T,d] (or None) rotated to their positions, in one launch: pairs (a, b) become
    (a c - b s, b c + a s) in float32, rounded once; dimensions past the table's rotary_dim are copied. `positions` is
    an int (row t at positions + t) or int64 [B,T] (or [T]); negative ones are padding (zeros), one past the table gives
    zeros and error bit 4. `inverse` turns the other way (s becomes -s): the gradient of the forward rotation, which
    autograd takes through q and k by itself (the table has none). Returns (q', k')."""
    return _rotate(q, k, table, positions, _layout(layout), bool(inverse))


def append_q8(cache, lengths, k_new: torch.Tensor, v_new: torch.Tensor, *, q=None, table=None, layout: str = "half"):
    """Write k_new, v_new [B,G,T,d] at the ends of the requests (see `lengths` above). With a rotary `table` k_new is
    rotated to its positions first (in float32, then rounded to codes once), and q [B,G,h,T,d], when given, is returned
    rotated ([B,G,h,T,d] contiguous, zeros in padding rows); without a table q must be None. One launch."""
    return _bind.append_q8(cache, lengths, k_new, v_new, q, table, _layout(layout))


def read_q8(cache, lo: int, hi: int, *, dtype=torch.bfloat16):
    """Positions [lo, hi) of the cache as values: (k, v), each [B,G,hi-lo,d] of dtype."""
    if dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"dtype must be float32 or bfloat16, got {dtype}")
    return _bind.read_q8(cache, lo, hi, dtype == torch.float32)


def attend_q8(q: torch.Tensor, cache, lengths, *, window: int = 0, sinks: int = 0, scale=None, max_length=None):
    """Attention of q [B,G,h,T,d] over the cache, causal: the query at position p sees the tokens j <= p, with a
    `window` > 0 only those with j > p - window or j < sinks. A row that sees nothing is zero. `max_length` (default: the
    capacity) is what the caller knows of the largest length; it chooses how the work is split, never the result's rows.
    Returns [B,G,h,T,d] of q's dtype.

    Precision: the cache's values are exact, q too (32-bit q to 2^-22 of its row's largest element); scores, maxima,
    denominators and outputs are summed in 32 bits. A softmax weight meets V as f16 terms: two (2^-21 of the weight) for
    32-bit q, and for 16-bit q up to 16 rows (T * h) a group, or 128 over few tokens; one (2^-11) for longer 16-bit chunks,
    where the output is rounded to 2^-8 in any case. Either ends 2^-31 below the row's largest 2^(score + exponent of the
    V block): values of V that are so much quieter than a visible block leave nothing in the output, though their tokens
    count in the denominator in full. A NaN code in a visible token makes the row (K) or its dimension (V) NaN, whatever
    the token's weight; hidden tokens' codes never show."""
    return _bind.attend_q8(q, cache, lengths, window, sinks, scale, max_length)
