"""Linear maps with their epilogue on MI355X: ``linear_act`` and ``mlp``.

``linear_act(x, weight, bias, residual, activation)`` is

    y = act(x weight^T + bias) + residual

and ``mlp`` two of them, the reference's block MLP with its skip connection
(nope_gdn_mlx.py:216-262, 4009-4091):

    y = act(x w1^T + b1) w2^T + b2 + residual

One kernel forms a product and its epilogue; the backward pass applies the
activation's derivative in the epilogue of the product that needs it, and forms
weight and bias gradients in one launch.  Sums, epilogues and activations are
fp32; each tensor that is stored (y, and for the backward pass the value before
the activation and the hidden layer) is rounded once to the inputs' dtype, bf16
or fp32.  fp32 products split each operand exactly into three bf16 parts and
keep what is at least 2^-16 of the largest product, fp32's own accuracy; an
infinite fp32 operand gives NaN where fp32 arithmetic may give an infinity.

Differentiable in every tensor; a second derivative is refused.  There is no CPU
path.
"""
from __future__ import annotations

import contextlib
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .kda import _DTYPE_CODE, _ptr, _stream

ACTIVATIONS = {None: 0, "gelu": 1, "silu": 2}
FEW_ROWS = 64        # up to here a forward's operands may have any alignment (kda_linear_fwd)
MAX_STRIDE = 1 << 21
_NULL = contextlib.nullcontext()


def _on(dev: torch.device):
    """Launches go to the tensors' device, whatever the current one is."""
    return _NULL if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)


def _padded(M: int, n: int, like: torch.Tensor) -> torch.Tensor:
    """An (M, n) matrix whose rows begin on 16 bytes and can be read in whole
    16-byte pieces (n rounded up to 8)."""
    return torch.empty((M, -(-n // 8) * 8), dtype=like.dtype, device=like.device)[:, :n]


def _mat(t: torch.Tensor, dma: bool) -> torch.Tensor:
    """t (M, n) as the kernels read it: rows at an even stride, with ``dma`` as
    ``_padded`` lays them out; a copy where it is not."""
    M, n = t.shape
    if (n > 1 and t.stride(1) != 1) or (M > 1 and not n <= t.stride(0) <= MAX_STRIDE):
        t = t.contiguous()
    if dma and (t.data_ptr() & 15 or n & 7 or (M > 1 and t.stride(0) & 7)):
        return _padded(M, n, t).copy_(t)
    return t


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else -(-t.shape[1] // 8) * 8


def _forward(x2: torch.Tensor, w: torch.Tensor, bias, res2, act: int, want_z: bool, pad: bool = False):
    """(y, z or None, x2, w) of matrices x2 (M, K), w (N, K): the last two as the
    kernel read them.  pad: y and z with rows as ``_padded`` lays them out."""
    M, K = x2.shape
    N = w.shape[0]
    code = _DTYPE_CODE[x2.dtype]
    dma = code == 1 and M > FEW_ROWS
    x2, w = _mat(x2, dma), _mat(w, dma)
    new = _padded if pad else lambda m, n, like: torch.empty((m, n), dtype=like.dtype, device=like.device)
    y = new(M, N, x2)
    z = new(M, N, x2) if want_z else None
    if M:
        if bias is not None:
            bias = bias.contiguous()
        if res2 is not None:
            res2 = _mat(res2, False)
        rc = _lib.load().kda_linear_fwd(
            _ptr(x2), _ld(x2), _ptr(w), _ld(w), _ptr(bias), _ptr(res2), 0 if res2 is None else _ld(res2), _ptr(y), _ld(y),
            _ptr(z), 0 if z is None else _ld(z), M, N, K, act, code, _stream(x2.device))
        _lib.check(rc, "kda_linear_fwd")
    return y, z, x2, w


def _dgrad(dz: torch.Tensor, w: torch.Tensor, z: Optional[torch.Tensor], act: int, pad: bool = False) -> torch.Tensor:
    """(dz w) * act'(z) for dz (M, N), w (N, K)."""
    M, N = dz.shape
    K = w.shape[1]
    code = _DTYPE_CODE[dz.dtype]
    dz, w = _mat(dz, code == 1), _mat(w, code == 1)
    dx = _padded(M, K, dz) if pad else torch.empty((M, K), dtype=dz.dtype, device=dz.device)
    rc = _lib.load().kda_linear_dgrad(_ptr(dz), _ld(dz), _ptr(w), _ld(w), _ptr(z) if act else None, _ld(z) if act else 0,
                                      _ptr(dx), _ld(dx), M, N, K, act, code, _stream(dz.device))
    _lib.check(rc, "kda_linear_dgrad")
    return dx


def _act_bwd(dy: torch.Tensor, z: torch.Tensor, act: int) -> torch.Tensor:
    M, N = dy.shape
    dz = _padded(M, N, dy)
    dy = _mat(dy, False)
    rc = _lib.load().kda_linear_act_bwd(_ptr(dy), _ld(dy), _ptr(z), _ld(z), _ptr(dz), _ld(dz), M, N, act,
                                        _DTYPE_CODE[dy.dtype], _stream(dy.device))
    _lib.check(rc, "kda_linear_act_bwd")
    return dz


def _wgrad(problems, M: int):
    """[(dw, db or None)] for each (dz (M, N), x (M, K), bias)."""
    dev = problems[0][0].device
    if M == 0:
        z = dict(dtype=problems[0][0].dtype, device=dev)
        return [(torch.zeros((d.shape[1], x.shape[1]), **z), torch.zeros(d.shape[1], **z) if b else None)
                for d, x, b in problems]
    if problems[0][0].dtype == torch.bfloat16:
        from .layer import weight_grads
        wide, ks = [], []
        for d, x, b in problems:
            k = x.shape[1]
            ks.append(k)
            if k & 7:   # rows of whole 16-byte pieces: the columns past k give columns of dw that are left out
                x = _mat(x, True)
                x = x.as_strided((M, -(-k // 8) * 8), (_ld(x), 1))
            wide.append((d, x, b))
        return [(dw if dw.shape[1] == k else dw[:, :k].contiguous(), db) for (dw, db), k in zip(weight_grads(wide, M), ks)]
    out = []
    lib = _lib.load()
    for d, x, b in problems:
        d, x = _mat(d, False), _mat(x, False)
        N, K = d.shape[1], x.shape[1]
        dw = torch.empty((N, K), dtype=torch.float32, device=dev)
        db = torch.empty((N,), dtype=torch.float32, device=dev) if b else None
        ws = torch.empty(lib.kda_linear_wgrad_workspace_size(M, N, K), dtype=torch.uint8, device=dev)
        rc = lib.kda_linear_wgrad(_ptr(d), _ld(d), _ptr(x), _ld(x), _ptr(dw), _ptr(db), M, N, K, _ptr(ws), ws.numel(),
                                  _stream(dev))
        _lib.check(rc, "kda_linear_wgrad")
        out.append((dw, db))
    return out


def _check(what: str, x: torch.Tensor, maps, residual: Optional[torch.Tensor], activation) -> int:
    """Validate x (..., K), the maps' (weight, bias) in turn and the residual;
    returns the activation's code."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"{what}: activation={activation!r}: expected one of {tuple(ACTIVATIONS)}")
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{what}: x must be a torch.Tensor")
    if x.dtype not in _DTYPE_CODE:
        raise ValueError(f"{what}: x dtype {x.dtype} unsupported: use float32 or bfloat16")
    if x.dim() < 1:
        raise ValueError(f"{what}: x must be (..., K); got shape {tuple(x.shape)}")
    n, named = x.shape[-1], []
    for i, (w, b) in enumerate(maps):
        tag = str(i + 1) if len(maps) > 1 else ""
        if w.dim() != 2 or w.shape[1] != n or w.shape[0] < 1 or n < 1:
            raise ValueError(f"{what}: weight{tag} shape {tuple(w.shape)} does not take {n} columns")
        n = w.shape[0]
        if b is not None and tuple(b.shape) != (n,):
            raise ValueError(f"{what}: bias{tag} shape {tuple(b.shape)} != {(n,)}")
        named += [("weight" + tag, w), ("bias" + tag, b)]
    if residual is not None and tuple(residual.shape) != (*x.shape[:-1], n):
        raise ValueError(f"{what}: residual shape {tuple(residual.shape)} != {(*x.shape[:-1], n)}")
    for name, t in (*named, ("residual", residual)):
        if t is None:
            continue
        if t.dtype != x.dtype:
            raise ValueError(f"{what}: {name} has dtype {t.dtype}; expected {x.dtype}")
        if t.device != x.device:
            raise ValueError(f"{what}: {name} is on {t.device}, x on {x.device}")
    if x.device.type != "cuda":
        raise ValueError(f"{what} runs on a ROCm device; got tensors on {x.device}")
    return ACTIVATIONS[activation]


def _needs_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _flat(t: Optional[torch.Tensor], n: int) -> Optional[torch.Tensor]:
    return None if t is None else t.reshape(-1, n)


class LinearActFunction(torch.autograd.Function):
    """``linear_act`` as one node; keeps its input, weight and, with an
    activation, the value before it."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        N, K = weight.shape
        with _on(x.device):
            y, z, x2, w = _forward(_flat(x, K), weight, bias, _flat(residual, N), act, bool(act))
        ctx.save_for_backward(x2, w, z)
        ctx.act, ctx.bias, ctx.shape = act, bias is not None, x.shape
        return y.view(*x.shape[:-1], N)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x2, w, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        M, N = x2.shape[0], w.shape[0]
        dx = dw = db = None
        with _on(x2.device):
            if M == 0:
                dx = x2.new_zeros(ctx.shape) if need_x else None
                if need_w or need_b:
                    ((dw, db),) = _wgrad([(dy.reshape(M, N), x2, ctx.bias)], M)
            elif need_x or need_w or need_b:
                dz = dy.reshape(M, N)
                dz = _act_bwd(dz, z, ctx.act) if ctx.act else _mat(dz, dz.dtype == torch.bfloat16)
                if need_x:
                    dx = _dgrad(dz, w, None, 0).view(ctx.shape)
                if need_w or need_b:
                    ((dw, db),) = _wgrad([(dz, x2, ctx.bias and need_b)], M)
        return dx, dw if need_w else None, db if need_b else None, dy if need_r else None, None


class MLPFunction(torch.autograd.Function):
    """``mlp`` as one node; keeps x, the weights, the hidden layer and the value
    before its activation."""

    @staticmethod
    def forward(ctx, x, w1, b1, w2, b2, residual, act):
        N, K = w1.shape
        out = w2.shape[0]
        with _on(x.device):
            h, z, x2, w1 = _forward(_flat(x, K), w1, b1, None, act, bool(act), pad=True)
            y, _, _, w2 = _forward(h, w2, b2, _flat(residual, out), 0, False)
        ctx.save_for_backward(x2, w1, z, h, w2)
        ctx.act, ctx.biases, ctx.shape = act, (b1 is not None, b2 is not None), x.shape
        return y.view(*x.shape[:-1], out)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x2, w1, z, h, w2 = ctx.saved_tensors
        need_x, need_w1, need_b1, need_w2, need_b2, need_r = ctx.needs_input_grad[:6]
        M, out = x2.shape[0], w2.shape[0]
        dx = dw1 = db1 = dw2 = db2 = None
        with _on(x2.device):
            dy2 = dy.reshape(M, out)
            first, second = need_w1 or need_b1, need_w2 or need_b2
            problems = []
            if M == 0:
                dx = x2.new_zeros(ctx.shape) if need_x else None
                dz = x2.new_zeros((0, w1.shape[0]))
            else:
                dy2 = _mat(dy2, dy2.dtype == torch.bfloat16)
                if need_x or first:
                    dz = _dgrad(dy2, w2, z, ctx.act, pad=True)
                if need_x:
                    dx = _dgrad(dz, w1, None, 0).view(ctx.shape)
            if first:
                problems.append((dz, x2, ctx.biases[0] and need_b1))
            if second:
                problems.append((dy2, h, ctx.biases[1] and need_b2))
            grads = _wgrad(problems, M) if problems else []
            if second:
                dw2, db2 = grads.pop()
            if first:
                dw1, db1 = grads.pop()
        return (dx, dw1 if need_w1 else None, db1, dw2 if need_w2 else None, db2, dy if need_r else None, None)


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
               residual: Optional[torch.Tensor] = None, activation: Optional[str] = None) -> torch.Tensor:
    """act(x weight^T + bias) + residual, differentiable.  x (..., K), weight (N, K),
    bias (N,), residual (..., N), all bf16 or all fp32; ``activation`` None, "gelu"
    (z Phi(z)) or "silu".  Rows and weights at any stride; bf16 rows that do not
    begin on 16 bytes, or whose K is no multiple of 8, are copied first when there
    are more than 64 of them."""
    act = _check("linear_act", x, ((weight, bias),), residual, activation)
    if _needs_grad(x, weight, bias, residual):
        return LinearActFunction.apply(x, weight, bias, residual, act)
    N, K = weight.shape
    with _on(x.device):
        return _forward(_flat(x, K), weight, bias, _flat(residual, N), act, False)[0].view(*x.shape[:-1], N)


def mlp(x: torch.Tensor, w1: torch.Tensor, b1: Optional[torch.Tensor], w2: torch.Tensor, b2: Optional[torch.Tensor],
        residual: Optional[torch.Tensor] = None, activation: Optional[str] = "gelu") -> torch.Tensor:
    """act(x w1^T + b1) w2^T + b2 + residual, differentiable.  x (..., K), w1 (N, K),
    w2 (K', N), biases or None, residual (..., K'), all bf16 or all fp32.  The hidden
    layer is rounded to their dtype between the two maps."""
    act = _check("mlp", x, ((w1, b1), (w2, b2)), residual, activation)
    if _needs_grad(x, w1, b1, w2, b2, residual):
        return MLPFunction.apply(x, w1, b1, w2, b2, residual, act)
    out = w2.shape[0]
    with _on(x.device):
        h = _forward(_flat(x, w1.shape[1]), w1, b1, None, act, False, pad=True)[0]
        return _forward(h, w2, b2, _flat(residual, out), 0, False)[0].view(*x.shape[:-1], out)
