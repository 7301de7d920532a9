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
There is no CPU path.  Gradients of g are fp32 sums of what reaches the tokens from one on
from before it, and those of shared heads are summed before they are rounded.
"""
from __future__ import annotations

from array import array
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
    n = 16 // t.element_size()
    if (t.data_ptr() & 15 or t.stride(-1) != 1 or t.stride(-3) > MAX_TOKEN_STRIDE
            or any(s % n for s, m in zip(t.stride()[:-1], t.shape[:-1]) if m > 1)):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _field(t: Optional[torch.Tensor], lead: int):
    """Address, ``lead`` strides and the heads of an operand (zeros: not there).  Of a dimension of
    one the stride does not count."""
    if t is None:
        return [0] * (lead + 2)
    return [t.data_ptr(), *(s if n > 1 else 0 for s, n in zip(t.stride()[:lead], t.shape)), t.shape[lead - 1]]


def _check_operands(what: str, q, k, v, g, lead: Tuple[str, ...]) -> int:
    """Validate q, k, v (*lead, heads, D) and g (*lead, H) or (H,); returns H."""
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


def _args(q, k, v, g, s0, cu, do=None, o=None, s_final=None, ds_final=None, dq=None, dk=None, dv=None, dg=None, ds0=None):
    """``kda_decay_args`` as 64-bit fields; the last five are the workspace, what is kept and train."""
    B, T, _, D = q.shape
    p = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    gs = (0, 0, g.stride(0)) if g.dim() == 1 else g.stride()
    return array("q", [*_field(q, 3), *_field(k, 3), *_field(v, 3), *_field(do, 3), p(g), *gs, p(s0), p(cu),
                       0 if cu is None else cu.numel() - 1, p(o), p(s_final), p(ds_final), p(dq), p(dk), p(dv), p(dg),
                       int(g.dim() == 1), p(ds0), B, T, g.shape[-1], D, _DTYPE_CODE[q.dtype], 0, 0, 0, 0, 0])


def _space(lib, pass_: int, at: int, dev: torch.device) -> Optional[torch.Tensor]:
    n = lib.kda_decay_workspace_size(pass_, at)
    return torch.empty(n, dtype=torch.uint8, device=dev) if n else None


def _aligned(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """States: contiguous, rows on 16 bytes."""
    if t is None or (t.is_contiguous() and not t.data_ptr() & 15):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _forward(q, k, v, g, s0, cu, train: bool):
    B, T, _, D = q.shape
    H, dev = g.shape[-1], q.device
    with _on(dev):
        q, k, v, s0 = _pieces(q), _pieces(k), _pieces(v), _aligned(s0)
        o = torch.empty((B, T, H, D), dtype=q.dtype, device=dev)
        s_final = torch.empty((B if cu is None else cu.numel() - 1, H, D, D), dtype=torch.float32, device=dev)
        args, lib = _args(q, k, v, g, s0, cu, o=o, s_final=s_final), _lib.load()
        at = args.buffer_info()[0]
        ws = _space(lib, _lib.KDA_PASS_TRAIN if train else _lib.KDA_PASS_FWD, at, dev)
        if ws is not None:
            i = -3 if train else -5
            args[i], args[i + 1] = ws.data_ptr(), ws.numel()
        args[-1] = int(train)
        rc = lib.kda_decay_fwd(at, _raw_stream(dev.index))
        if rc:
            _lib.check(rc, "kda_decay_fwd")
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
        B, T, _, D = q.shape
        H, dev = g.shape[-1], q.device
        with _on(dev):
            do = torch.zeros((B, T, H, D), dtype=q.dtype, device=dev) if do is None else _pieces(do)
            ds = _aligned(ds)
            new = lambda t: torch.empty(t.shape, dtype=t.dtype, device=dev)  # noqa: E731
            dq, dk, dv = new(q), new(k), new(v)
            dg = new(g) if need_g else None
            ds0 = new(s0) if need_s else None
            args, lib = _args(q, k, v, g, s0, cu, do, None, s_final, ds, dq, dk, dv, dg, ds0), _lib.load()
            at = args.buffer_info()[0]
            ws = _space(lib, _lib.KDA_PASS_BWD, at, dev)
            if ws is not None:
                args[-5], args[-4] = ws.data_ptr(), ws.numel()
            if kept is not None:
                args[-3], args[-2] = kept.data_ptr(), kept.numel()
            rc = lib.kda_decay_bwd(at, _raw_stream(dev.index))
            if rc:
                _lib.check(rc, "kda_decay_bwd")
        return dq, dk, dv, dg, ds0, None


def chunk_decay(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor,
                initial_state: Optional[torch.Tensor] = None, cu_seqlens: Optional[torch.Tensor] = None
                ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Decayed linear attention over whole sequences, differentiable.  Returns (o (B, T, H, D)
    in q's dtype, final_state (B, H, D, D) fp32).

    q, k, v (B, T, heads, D), bf16 or fp32, D 32, 64, 96 or 128, any strides (rows that
    are not whole 16-byte pieces are copied first).  g (B, T, H) or (H,), fp32 or bf16;
    g = -inf starts the state anew, and so does everything below -200.  A
    value that is not finite reaches all outputs of its sequence from its 64 tokens on.

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
    zero; rows of one slot follow each other.  No gradients: ``chunk_decay`` with T = 1 has them."""
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
        gs = (0, g.stride(0)) if g.dim() == 1 else g.stride()
        rows = lambda t: (t.data_ptr(), t.stride(0) if B > 1 else 0, 0, t.stride(1) if t.shape[1] > 1 else 0, t.shape[1])  # noqa: E731
        args = array("q", [*rows(q), *rows(k), *rows(v), 0, 0, 0, 0, 0, g.data_ptr(), gs[0], 0, gs[1], state.data_ptr(), 0, 0,
                           o.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, B, 1, H, D, _DTYPE_CODE[q.dtype], 0, 0, 0, 0, 0])
        rc = _lib.load().kda_decay_step(args.buffer_info()[0], None if slots is None else slots.data_ptr(), N,
                                        _raw_stream(dev.index))
        if rc:
            _lib.check(rc, "kda_decay_step")
    if not state.is_inference():
        _increment_version((state,))   # a graph that holds the state as it was has to notice
    return o
