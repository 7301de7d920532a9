"""Linear attention with a decay for each head on MI355X: ``chunk_decay`` over whole
sequences, ``decay_step`` for one token.

    S_t = e^{g_t} S_{t-1} + v_t k_t^T,   o_t = S_t q_t

the recurrence of ``chunk_gdn`` without the delta rule (nope_gdn_mlx.py:641-650), in
``chunk_kda``'s layouts: q, k, v (B, T, heads, D), the state (B, H, D, D) fp32 as
``S[i_v, j_k]``; q is not scaled inside.  What differs:

* the decay ``g`` is a log-decay (<= 0) of every token and head, (B, T, H), or one of each
  head, (H,);
* q, k and v may have fewer heads than the H of the state: head h takes theirs of
  index h // (H / heads);
* sequences of different lengths may lie packed in one row: ``cu_seqlens``.

Differentiable in every tensor but ``cu_seqlens``; a second derivative and tracing are
refused.  Sums and states are fp32; each output is rounded once, to its input's dtype.
There is no CPU path.  A backward pass is captured into a graph as torch's own nodes are: while no
eager graph of the same leaves is alive.  Gradients of g are fp32 sums of what reaches the tokens from one on
from before it, and those of shared heads are summed before they are rounded.
"""
from __future__ import annotations

from functools import lru_cache
from struct import Struct
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .kda import FWD_HEAD_DIMS, _DTYPE_CODE
from .linear import _grad_enabled, _is_tracing, _on, _raw_stream

HEAD_DIMS = FWD_HEAD_DIMS
_increment_version = torch._C._increment_version
MAX_TOKENS, MAX_TOKEN_STRIDE = (1 << 31) - 8192, 1 << 24


def _pieces(t: torch.Tensor) -> torch.Tensor:
    """t (..., heads, D) as the kernels read it, rows in whole 16-byte pieces; a copy where it is not."""
    if not t.data_ptr() & 15:
        if t.is_contiguous():
            return t
        n = 16 // t.element_size()
        if (t.stride(-1) == 1 and t.stride(0 if t.dim() == 3 else 1) <= MAX_TOKEN_STRIDE
                and not any(s % n for s, m in zip(t.stride()[:-1], t.shape[:-1]) if m > 1)):
            return t
    return t.clone(memory_format=torch.contiguous_format)


def _rows(t: torch.Tensor):
    """kda_decay_rows of t (B, T, heads, D).  (Of a dimension of one the stride does not count.)"""
    B, T, h, D = t.shape
    if t.is_contiguous():
        return t.data_ptr(), T * h * D, h * D, D, h
    b, m, s, _ = t.stride()
    return t.data_ptr(), b if B > 1 else 0, m if T > 1 else 0, s if h > 1 else 0, h


_NONE = (0,) * 5
_pack = Struct("46q").pack      # kda_decay_args


@lru_cache(maxsize=1024)
def _space(pass_: int, B: int, T: int, H: int, D: int, code: int, hq: int, hk: int, hv: int, nseq: int, dg: int) -> int:
    """``kda_decay_workspace_size`` by sizes; nseq -1: not packed; dg 0: not wanted, 1 [B][T][H], 2 [H]."""
    none = (0, 0, 0, 0)
    return _lib.load().kda_decay_workspace_size(pass_, _pack(
        *none, hq, *none, hk, *none, hv, *none, H, *none, 0, nseq >= 0, max(nseq, 0), 0, 0, 0, 0, 0, 0, dg > 0, dg == 2, 0, B, T, H, D,
        code, *none, 0))


def _new(n: int, dev: torch.device) -> Optional[torch.Tensor]:
    return torch.empty(n, dtype=torch.uint8, device=dev) if n else None


def _p(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _matches(n: int, q, k, v, g) -> bool:
    """What ``_check_operands`` asks for, in one expression."""
    try:
        *head, hq, D = q.shape
        *kh, hk, kd = k.shape
        *vh, hv, vd = v.shape
        H, dt, dev = g.shape[-1], q.dtype, q.get_device()
        return (len(head) == n and head == kh == vh and D == kd == vd and D in HEAD_DIMS and dt in _DTYPE_CODE
                and k.dtype is dt and v.dtype is dt and g.dtype in _DTYPE_CODE and not (H % hq or H % hk or H % hv) and H > 0
                and (g.dim() == 1 or g.shape == (*head, H)) and dev == k.get_device() == v.get_device() == g.get_device())
    except (AttributeError, TypeError, ValueError, IndexError, ZeroDivisionError):
        return False


def _check_operands(what: str, q, k, v, g, lead: Tuple[str, ...]) -> int:
    """Validate q, k, v (*lead, heads, D) and g (*lead, H) or (H,); returns H."""
    if _matches(len(lead), q, k, v, g):
        return g.shape[-1]
    for name, t in (("q", q), ("k", k), ("v", v), ("g", g)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what}: {name} must be a torch.Tensor")
    n = len(lead)
    if q.dim() != n + 2:
        raise ValueError(f"{what}: q must be ({', '.join(lead)}, heads, D); got shape {tuple(q.shape)}")
    head, D = q.shape[:n], q.shape[-1]
    if D not in HEAD_DIMS:
        raise ValueError(f"{what}: head_dim={D}: expected one of {HEAD_DIMS}")
    if q.dtype not in _DTYPE_CODE:
        raise ValueError(f"{what}: q dtype {q.dtype} unsupported: use float32 or bfloat16")
    if g.dim() != 1 and (g.dim() != n + 1 or g.shape[:n] != head):
        raise ValueError(f"{what}: g shape {tuple(g.shape)}: expected {tuple(head)} and the heads, or the heads alone")
    if g.dtype not in _DTYPE_CODE:
        raise ValueError(f"{what}: g dtype {g.dtype} unsupported: use float32 or bfloat16")
    H = g.shape[-1]
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != n + 2 or t.shape[:n] != head or t.shape[-1] != D:
            raise ValueError(f"{what}: {name} shape {tuple(t.shape)} does not match q's {tuple(q.shape)}")
        if t.shape[n] < 1 or H < 1 or H % t.shape[n]:
            raise ValueError(f"{what}: {name} has {t.shape[n]} heads, which do not divide g's {H}")
        if t.dtype != q.dtype:
            raise ValueError(f"{what}: {name} has dtype {t.dtype}; expected {q.dtype}")
    for name, t in (("k", k), ("v", v), ("g", g)):
        if t.device != q.device:
            raise ValueError(f"{what}: {name} is on {t.device}, q on {q.device}")
    return H


def _check_states(what: str, name: str, t: torch.Tensor, shape: Tuple[int, ...], dev: torch.device) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: {name} must be a torch.Tensor")
    if tuple(t.shape) != shape:
        raise ValueError(f"{what}: {name} shape {tuple(t.shape)} != {shape}")
    if t.dtype != torch.float32:
        raise ValueError(f"{what}: {name} has dtype {t.dtype}; expected torch.float32")
    if t.device != dev:
        raise ValueError(f"{what}: {name} is on {t.device}, q on {dev}")


def _check_device(what: str, dev: torch.device) -> None:
    if dev.type != "cuda":
        raise ValueError(f"{what} runs on a ROCm device; got tensors on {dev}")
    if _is_tracing():
        raise RuntimeError(f"{what} cannot be traced: its launches are no part of a traced graph")


def _aligned(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """States: contiguous, rows on 16 bytes."""
    if t is None or (t.is_contiguous() and not t.data_ptr() & 15):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _call(fn, q, k, v, do, g, *rest):
    one = g.dim() == 1
    B, T, _, D = q.shape
    s0, cu, o, s_final, ds, dq, dk, dv, dg, ds0, ws, kept, train = rest
    rc = fn(_pack(*_rows(q), *_rows(k), *_rows(v), *(_NONE if do is None else _rows(do)), g.data_ptr(),
                  *((0, 0, g.stride(0)) if one else g.stride()), _p(s0), _p(cu), 0 if cu is None else cu.numel() - 1, _p(o),
                  _p(s_final), _p(ds), _p(dq), _p(dk), _p(dv), _p(dg), one, _p(ds0), B, T, g.shape[-1], D, _DTYPE_CODE[q.dtype],
                  _p(ws), 0 if ws is None else ws.numel(), _p(kept), 0 if kept is None else kept.numel(), train),
            _raw_stream(q.get_device()))
    if rc:
        _lib.check(rc, fn.__name__)


def _forward(q, k, v, g, s0, cu, train: bool):
    B, T, hq, D = q.shape
    H, dev, nseq = g.shape[-1], q.device, -1 if cu is None else cu.numel() - 1
    with _on(dev):
        q, k, v, s0 = _pieces(q), _pieces(k), _pieces(v), _aligned(s0)
        o = torch.empty((B, T, H, D), dtype=q.dtype, device=dev)
        s_final = torch.empty((B if cu is None else nseq, H, D, D), dtype=torch.float32, device=dev)
        ws = _new(_space(_lib.KDA_PASS_TRAIN if train else _lib.KDA_PASS_FWD, B, T, H, D, _DTYPE_CODE[q.dtype], hq, k.shape[2],
                         v.shape[2], nseq, 0), dev)
        _call(_lib.load().kda_decay_fwd, q, k, v, None, g, s0, cu, o, s_final, None, None, None, None, None, None,
              None if train else ws, ws if train else None, train)
    return q, k, v, s0, ws, o, s_final


class ChunkDecayFunction(torch.autograd.Function):
    """``chunk_decay`` as one node; keeps its inputs, the final state and the states that
    the kernels share a sequence out by."""

    @staticmethod
    def forward(ctx, q, k, v, g, s0, cu):
        *kept, o, s_final = _forward(q, k, v, g, s0, cu, True)
        ctx.save_for_backward(*kept, g, cu, s_final)
        # an unused output's cotangent comes as None
        ctx.set_materialize_grads(False)
        return o, s_final

    @staticmethod
    @once_differentiable
    def backward(ctx, do, ds):
        q, k, v, s0, kept, g, cu, s_final = ctx.saved_tensors
        need_g, need_s = ctx.needs_input_grad[3:5]
        B, T, hq, D = q.shape
        H, dev = g.shape[-1], q.device
        with _on(dev):
            do = torch.zeros((B, T, H, D), dtype=q.dtype, device=dev) if do is None else _pieces(do)
            dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k, v))
            dg = torch.empty(g.shape, dtype=torch.float32, device=dev) if need_g else None
            ds0 = torch.empty(s0.shape, dtype=torch.float32, device=dev) if need_s else None
            ws = _new(_space(_lib.KDA_PASS_BWD, B, T, H, D, _DTYPE_CODE[q.dtype], hq, k.shape[2], v.shape[2],
                             -1 if cu is None else cu.numel() - 1, (2 if g.dim() == 1 else 1) if need_g else 0), dev)
            _call(_lib.load().kda_decay_bwd, q, k, v, do, g, s0, cu, None, s_final, _aligned(ds), dq, dk, dv, dg, ds0, ws, kept, 0)
        return dq, dk, dv, dg, ds0, None


def chunk_decay(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor,
                initial_state: Optional[torch.Tensor] = None, cu_seqlens: Optional[torch.Tensor] = None
                ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Decayed linear attention over whole sequences, differentiable.  Returns (o (B, T, H, D)
    in q's dtype, final_state (B, H, D, D) fp32).

    q, k, v (B, T, heads, D), bf16 or fp32, D 32, 64, 96 or 128, any strides (rows that
    are not whole 16-byte pieces are copied first).  g (B, T, H) or (H,), fp32 or bf16;
    g = -inf starts the state anew, and so does everything below -200.  A value that is not
    finite reaches the outputs of its sequence from its token on, and all of its dg.

    ``cu_seqlens`` (N + 1,) int32 on the same device: token cu[i] to cu[i + 1] - 1 of the one
    row (B = 1) are sequence i; states are then (N, H, D, D).  The limits are read on the
    device: one below its predecessor counts as that, one past T as T; rows of no sequence
    get zeros."""
    H = _check_operands("chunk_decay", q, k, v, g, ("B", "T"))
    B, T, _, D = q.shape
    dev = q.device
    if B * T > MAX_TOKENS:
        raise ValueError(f"chunk_decay: q of shape {tuple(q.shape)} has more than {MAX_TOKENS} tokens")
    if cu_seqlens is not None:
        if not isinstance(cu_seqlens, torch.Tensor):
            raise TypeError("chunk_decay: cu_seqlens must be a torch.Tensor")
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1 or cu_seqlens.dtype != torch.int32:
            raise ValueError(f"chunk_decay: cu_seqlens must be (N + 1,) int32; got {tuple(cu_seqlens.shape)} {cu_seqlens.dtype}")
        if B != 1:
            raise ValueError(f"chunk_decay: cu_seqlens with B={B}: packed sequences lie in one row")
        if cu_seqlens.device != dev:
            raise ValueError(f"chunk_decay: cu_seqlens is on {cu_seqlens.device}, q on {dev}")
        cu_seqlens = cu_seqlens.contiguous()
    if initial_state is not None:
        n = B if cu_seqlens is None else cu_seqlens.numel() - 1
        _check_states("chunk_decay", "initial_state", initial_state, (n, H, D, D), dev)
    _check_device("chunk_decay", dev)
    g = g if g.dtype == torch.float32 else g.float()
    if (_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, g, initial_state))
            or forward_ad._current_level >= 0):
        return ChunkDecayFunction.apply(q, k, v, g, initial_state, cu_seqlens)
    return _forward(q, k, v, g, initial_state, cu_seqlens, False)[5:]


def decay_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, state: torch.Tensor,
               slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of each row, S <- e^g S + v k^T, o = S q, on states that stay where they are:
    ``state`` (N, H, D, D) fp32, contiguous, is updated.  Returns o (B, H, D) in q's dtype.

    q, k, v (B, heads, D), g (B, H) or (H,), types and heads as in ``chunk_decay``, whose
    final_state a sequence goes on from.  ``slots`` (B,) int32 on the same device: the state of each
    row (without it row b's is b, N = B).  A row whose slot is none of 0 to N - 1 is left out, its o
    zero; rows of one slot follow each other (which is looked for among all rows: thousands of them
    cost more than their states).  No gradients: ``chunk_decay`` with T = 1 has them."""
    H = _check_operands("decay_step", q, k, v, g, ("B",))
    B, _, D = q.shape
    dev = q.device
    if not isinstance(state, torch.Tensor):
        raise TypeError("decay_step: state must be a torch.Tensor")
    N = B if slots is None else state.shape[0] if state.dim() else 0
    _check_states("decay_step", "state", state, (N, H, D, D), dev)
    if slots is not None:
        if not isinstance(slots, torch.Tensor):
            raise TypeError("decay_step: slots must be a torch.Tensor")
        if slots.shape != (B,) or slots.dtype != torch.int32:
            raise ValueError(f"decay_step: slots must be ({B},) int32; got {tuple(slots.shape)} {slots.dtype}")
        if slots.device != dev:
            raise ValueError(f"decay_step: slots is on {slots.device}, q on {dev}")
        slots = slots.contiguous()
    if not state.is_contiguous() or state.data_ptr() & 15:
        raise ValueError(f"decay_step: state must be contiguous and 16-byte aligned; got strides {state.stride()}")
    _check_device("decay_step", dev)
    if (_grad_enabled() and any(t.requires_grad for t in (q, k, v, g, state))) or forward_ad._current_level >= 0:
        raise RuntimeError("decay_step has no gradient: run it under torch.no_grad(), or chunk_decay with T = 1")
    g = g if g.dtype == torch.float32 else g.float()
    with _on(dev):
        q, k, v = _pieces(q), _pieces(k), _pieces(v)
        o = torch.empty((B, H, D), dtype=q.dtype, device=dev)
        gb, gh = (0, g.stride(0)) if g.dim() == 1 else g.stride()
        fields = []
        for t in (q, k, v):
            b, h, _ = t.stride()
            fields += (t.data_ptr(), b if B > 1 else 0, 0, h if t.shape[1] > 1 else 0, t.shape[1])
        rc = _lib.load().kda_decay_step(
            _pack(*fields, *_NONE, g.data_ptr(), gb, 0, gh, state.data_ptr(), 0, 0, o.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, B, 1, H, D,
                  _DTYPE_CODE[q.dtype], 0, 0, 0, 0, 0), None if slots is None else slots.data_ptr(), N, _raw_stream(dev.index))
        if rc:
            _lib.check(rc, "kda_decay_step")
    if not state.is_inference():
        _increment_version((state,))   # a graph that holds the state as it was has to notice
    return o
