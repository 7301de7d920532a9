"""Rotary positions with several axes on MI355X: ``rotary``.

Channels in pairs (x, y) are turned by the angle of their axis' position and their own
frequency, x' = x cos - y sin, y' = x sin + y cos, for queries and keys in one launch.
A token of a video has three axes, time, height and width, each with a section of the
channels; ``grid`` numbers tokens as ``TubeletEmbedding3D`` lays them out
(nope_gdn_mlx.py:98-150: frame by frame, rows of a frame, tokens of a row).  The
reference's model has no positions; this is for what is built beside it.

Angles are formed in fp64 (at a position p they are within 2^-52 p), rows in fp32 and
rounded once.  Differentiable in q and k, by turning back; a second derivative and tracing are
refused.  A backward pass is captured into a graph as torch's own nodes are: while no eager graph
of the same leaves is alive.  There is no CPU path.
"""
from __future__ import annotations

import math
from array import array
from functools import lru_cache
from operator import index
from struct import Struct
from typing import Optional, Sequence, Tuple, Union

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .kda import _DTYPE_CODE
from .linear import _grad_enabled, _is_tracing, _on, _raw_stream

MAX_HEAD_DIM, MAX_AXES, MAX_TOKENS = 256, 4, (1 << 31) - 1
_POSITIONS = {torch.int32: 0, torch.int64: 1, torch.float32: 2}


@lru_cache(maxsize=64)
def _axes(D: int, sections, base: float) -> Tuple[int, Tuple[int, ...], array]:
    """Validated: how many axes, their sections filled up with zeros, and turns a unit of position of
    every pair, base^(-2 i / section) / 2 pi."""
    given, sections = sections, (D,) if sections is None else sections
    if not 1 <= len(sections) <= MAX_AXES or any(s < 0 or s % 2 for s in sections) or sum(sections) > D:
        raise ValueError(f"rotary: sections={given}: expected 1 to {MAX_AXES} even numbers that make up at most {D}")
    if not 0.0 < base < math.inf:
        raise ValueError(f"rotary: base={base}: expected a positive number")
    turns = array("d", [base ** (-2 * i / s) / (2 * math.pi) for s in sections for i in range(s // 2)])
    return len(sections), sections + (0,) * (MAX_AXES - len(sections)), turns


def _whole(sections) -> Optional[Tuple[int, ...]]:
    try:
        return sections if sections is None else tuple(map(index, sections))
    except TypeError:
        raise ValueError(f"rotary: sections={sections}: expected 1 to {MAX_AXES} even numbers") from None


def _unit(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 else t.contiguous()


def _rows(t: torch.Tensor):
    return (t.data_ptr(), *t.stride()[:3], t.shape[2])


_NONE = (0, 0, 0, 0, 1)
_pack = Struct("32q").pack      # kda_rotary_args


def _turn(q, k, how, sign: int):
    """Queries and keys (either may be None) turned by ``how``, sign -1: back."""
    positions, where, (axes, sections, turns), interleaved = how
    first, second = (k, None) if q is None else (q, k)
    B, T, _, D = first.shape
    dev = first.device
    with _on(dev):
        first = _unit(first)
        y, z = torch.empty(first.shape, dtype=first.dtype, device=dev), None
        if second is not None:
            second = _unit(second)
            z = torch.empty(second.shape, dtype=second.dtype, device=dev)
        rc = _lib.load().kda_rotary(
            _pack(*_rows(first), *(_NONE if second is None else _rows(second)), y.data_ptr(), 0 if z is None else z.data_ptr(),
                  0 if positions is None else positions.data_ptr(), *where, axes, *sections, turns.buffer_info()[0], interleaved, sign,
                  B, T, D, _DTYPE_CODE[first.dtype]), _raw_stream(dev.index))
        if rc:
            _lib.check(rc, "kda_rotary")
    return (None, y) if q is None else (y, z)


class RotaryFunction(torch.autograd.Function):
    """``rotary`` as one node; keeps the positions."""

    @staticmethod
    def forward(ctx, q, k, how):
        ctx.save_for_backward(how[0])
        ctx.how = how[1:]
        ctx.set_materialize_grads(False)
        y = _turn(q, k, how, 1)
        return y[0] if k is None else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk=None):
        dq, dk = (d if need else None for d, need in zip((dq, dk), ctx.needs_input_grad))
        if dq is None and dk is None:
            return None, None, None
        return (*_turn(dq, dk, (*ctx.saved_tensors, *ctx.how), -1), None)


def rotary(q: torch.Tensor, k: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None, *,
           grid: Optional[Tuple[int, int]] = None, start: int = 0, sections: Optional[Sequence[int]] = None,
           base: float = 10000.0, interleaved: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """q (B, T, heads, D) and k (B, T, heads, D), bf16 or fp32, turned by their tokens' positions,
    differentiable.  Returns q', or (q', k') with k.

    ``positions``: (T,), (axes, T) or (axes, B, T), int32, int64 or fp32, on the same device; or
    ``grid`` = (height, width), the tokens of a frame: token t is number n = start + t of its
    video, with positions n // (height width), n // width % height and n % width.
    ``sections``: the channels of each axis, even, in order (default: all for one axis); channels
    behind them stay as they are.  Pair i of an axis with s channels turns by base^(-2 i / s) a
    position; its channels are i and s / 2 + i of the section, or with ``interleaved`` 2 i and
    2 i + 1.  D even, at most 256, at most 4 axes; any strides."""
    what = "rotary"
    if not isinstance(q, torch.Tensor) or not (k is None or isinstance(k, torch.Tensor)):
        raise TypeError("rotary: q and k must be torch.Tensors")
    if q.dim() != 4:
        raise ValueError(f"{what}: q must be (B, T, heads, D); got shape {tuple(q.shape)}")
    B, T, heads, D = q.shape
    if q.dtype not in _DTYPE_CODE:
        raise ValueError(f"{what}: q dtype {q.dtype} unsupported: use float32 or bfloat16")
    if D < 2 or D % 2 or D > MAX_HEAD_DIM or heads < 1:
        raise ValueError(f"{what}: {heads} heads of head_dim={D}: expected an even number up to {MAX_HEAD_DIM}")
    if B * T > MAX_TOKENS:
        raise ValueError(f"{what}: q of shape {tuple(q.shape)} has more than {MAX_TOKENS} tokens")
    dev = q.device
    if k is not None:
        if k.dim() != 4 or k.shape[:2] != (B, T) or k.shape[3] != D or k.shape[2] < 1:
            raise ValueError(f"{what}: k shape {tuple(k.shape)} does not match q's {tuple(q.shape)}")
        if k.dtype != q.dtype:
            raise ValueError(f"{what}: k has dtype {k.dtype}; expected {q.dtype}")
        if k.device != dev:
            raise ValueError(f"{what}: k is on {k.device}, q on {dev}")
    how = _axes(D, _whole(sections), float(base))
    n = how[0]
    if (positions is None) == (grid is None):
        raise ValueError(f"{what}: expected either positions or grid")
    if grid is not None:
        try:
            h, w = grid
            h, w, first = index(h), index(w), index(start)
        except (TypeError, ValueError):
            raise ValueError(f"{what}: grid={grid}, start={start}: expected (height, width) and a number, whole numbers") from None
        if not (1 <= h < 1 << 31 and 1 <= w < 1 << 31 and n <= 3 and 0 <= first < 1 << 62):
            raise ValueError(f"{what}: grid={grid}, start={start} with {n} sections: expected (height, width), "
                             "start >= 0 and at most 3 axes")
        where = (0, 0, 0, 0, h, w, first)
    else:
        if not isinstance(positions, torch.Tensor):
            raise TypeError("rotary: positions must be a torch.Tensor")
        if start:
            raise ValueError(f"{what}: start={start} goes with grid, not with positions")
        shape = tuple(positions.shape)
        if shape not in ((n, T), (n, B, T)) and not (n == 1 and shape == (T,)):
            raise ValueError(f"{what}: positions shape {shape}: expected ({n}, {T}) or ({n}, {B}, {T})")
        if positions.dtype not in _POSITIONS:
            raise ValueError(f"{what}: positions dtype {positions.dtype} unsupported: use int32, int64 or float32")
        if positions.device != dev:
            raise ValueError(f"{what}: positions is on {positions.device}, q on {dev}")
        if positions.requires_grad and _grad_enabled():
            raise ValueError(f"{what} has no gradient for positions")
        s = positions.stride()
        where = (_POSITIONS[positions.dtype], *((0, 0, s[0]) if len(s) == 1 else (s[0], 0, s[1]) if len(s) == 2 else s), 1, 1, 0)
    if dev.type != "cuda":
        raise ValueError(f"{what} runs on a ROCm device; got tensors on {dev}")
    if _is_tracing():
        raise RuntimeError(f"{what} cannot be traced: its launches are no part of a traced graph")
    how = positions, where, how, bool(interleaved)
    if _grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)) or forward_ad._current_level >= 0:
        return RotaryFunction.apply(q, k, how)
    y = _turn(q, k, how, 1)
    return y[0] if k is None else y
