"""Linear maps with their epilogue on MI355X: ``linear_act`` and ``mlp``.

``linear_act(x, weight, bias, residual, activation)`` is

    y = act(x weight^T + bias) + residual

and ``mlp`` two of them, the reference's block MLP with its skip connection
(nope_gdn_mlx.py:216-262, 4009-4091):

    y = act(x w1^T + b1) w2^T + b2 + residual

One kernel forms a product and its epilogue; the backward pass applies the
activation's derivative in the epilogue of the product that needs it, and forms
weight and bias gradients in one launch.  Sums and epilogues are fp32, and so are
activations: of fp32 results to its own accuracy, of bf16's gelu within 1e-5 of its
value.  Each tensor that is stored is rounded once, y and the hidden layer to the
inputs' dtype, bf16 or fp32; what the backward pass reads again too: the value before
the activation to fp16 where that is bf16, its gradient to bf16, the operand of the
next products.  So bf16 gradients are off by two roundings, 2^1/2 of one.  fp32
products split each operand exactly into three bf16 parts and keep what is at least
2^-16 of the largest product, fp32's own accuracy; there an infinite operand gives
NaN where fp32 arithmetic may give an infinity, which forwards of at most 1024 pieces
of 16 x 16 (2048 up to 8 rows), formed otherwise, do give.

Differentiable in every tensor; a second derivative and tracing are refused.  There
is no CPU path.  A backward pass is captured into a graph as torch's own nodes are:
while no eager graph of the same leaves is alive.
"""
from __future__ import annotations

import contextlib
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .kda import _DTYPE_CODE

ACTIVATIONS = {None: 0, "gelu": 1, "silu": 2}
_PRE = {torch.float32: torch.float32, torch.bfloat16: torch.float16}    # what the value before the activation is kept in
MAX_STRIDE, MAX_ROWS = 1 << 21, (1 << 31) - 1
_NULL = contextlib.nullcontext()
_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
_grad_enabled, _is_tracing = torch.is_grad_enabled, torch._C._is_tracing


def _on(dev: torch.device):
    """Launches go to the tensors' device, whatever the current one is."""
    return _NULL if dev.index == _current_device() else torch.cuda.device(dev)


def _few(M: int, N: int) -> bool:
    """A bf16 forward's operands may have any alignment (kda_linear_fwd)."""
    return (M + 15 >> 4) * (N + 15 >> 4) <= (512 if M <= 8 else 256)


def _up8(n: int) -> int:
    return -(-n // 8) * 8


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t (M, n) with unit column stride and rows at an even stride; a copy where it is not."""
    M, n = t.shape
    s0, s1 = t.stride()
    if (n > 1 and s1 != 1) or (M > 1 and not n <= s0 <= MAX_STRIDE):
        return t.contiguous()
    return t


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else _up8(t.shape[1])


def _whole(t: torch.Tensor) -> bool:
    """Rows begin on 16 bytes and are whole 16-byte pieces."""
    return not (t.shape[1] & 7 or t.data_ptr() & 15 or (t.shape[0] > 1 and t.stride(0) & 7))


def _whole_rows(x: torch.Tensor, w: torch.Tensor, stream: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """bf16 matrices as the tiles' DMA reads them: copies, in one launch, of those
    that are not, their columns rounded up to 8."""
    jobs, out = [], [x, w]
    for i, t in enumerate((x, w)):
        if not _whole(t):
            M, n = t.shape
            out[i] = torch.empty((M, _up8(n)), dtype=t.dtype, device=t.device)
            jobs += [t.data_ptr(), _ld(t), M, n, out[i].data_ptr()]
    if jobs:
        jobs += [None, 0, 0, 0, None] * (2 - len(jobs) // 5)
        _lib.check(_lib.load().kda_linear_pad(*jobs, stream), "kda_linear_pad")
    return out[0], out[1]


def _forward(x2: torch.Tensor, K: int, w: torch.Tensor, bias, res2, act: int, y: int, ld_y: int, z: Optional[int],
             ld_z: int, train: bool):
    """y <- act(x2 w^T + bias) + res2 for x2 (M, K or wider), w (N, K); y and z: addresses
    and row strides of (M, N) outputs.  Returns x2 and w as the kernels read them,
    with ``train`` also the backward's."""
    M, N = x2.shape[0], w.shape[0]
    code = _DTYPE_CODE[w.dtype]
    stream = _raw_stream(w.get_device())
    x2, w = _rows(x2), _rows(w)
    if code and (train or not _few(M, N)):
        x2, w = _whole_rows(x2, w, stream)
    if M:
        if bias is not None and not bias.is_contiguous():
            bias = bias.contiguous()
        if res2 is not None:
            res2 = _rows(res2)
        rc = _lib.load().kda_linear_fwd(
            x2.data_ptr(), _ld(x2), w.data_ptr(), _ld(w), None if bias is None else bias.data_ptr(),
            None if res2 is None else res2.data_ptr(), 0 if res2 is None else _ld(res2), y, ld_y, z, ld_z, M, N, K, act,
            code, stream)
        if rc:
            _lib.check(rc, "kda_linear_fwd")
    return x2, w


def _check(what: str, x: torch.Tensor, maps, residual: Optional[torch.Tensor], activation) -> int:
    """Validate x (..., K), the maps' (weight, bias) in turn and the residual;
    returns the activation's code."""
    act = ACTIVATIONS.get(activation, -1)
    if act < 0:
        raise ValueError(f"{what}: activation={activation!r}: expected one of {tuple(ACTIVATIONS)}")
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{what}: x must be a torch.Tensor")
    dtype, dev, shape = x.dtype, x.device, x.shape
    if dtype not in _DTYPE_CODE:
        raise ValueError(f"{what}: x dtype {dtype} unsupported: use float32 or bfloat16")
    if len(shape) < 1:
        raise ValueError(f"{what}: x must be (..., K); got shape {tuple(shape)}")
    n = shape[-1]
    named = []
    for w, b in maps:
        ws = w.shape
        if len(ws) != 2 or ws[1] != n or ws[0] < 1 or n < 1:
            tag = str(len(named) // 2 + 1) if len(maps) > 1 else ""
            raise ValueError(f"{what}: weight{tag} shape {tuple(ws)} does not take {n} columns")
        n = ws[0]
        if b is not None and b.shape != (n,):
            tag = str(len(named) // 2 + 1) if len(maps) > 1 else ""
            raise ValueError(f"{what}: bias{tag} shape {tuple(b.shape)} != {(n,)}")
        named += (w, b)
    if residual is not None and (residual.shape[-1:] != (n,) or residual.shape[:-1] != shape[:-1]):
        raise ValueError(f"{what}: residual shape {tuple(residual.shape)} != {(*shape[:-1], n)}")
    for i, t in enumerate((*named, residual)):
        if t is not None and (t.dtype != dtype or t.device != dev):
            name = "residual" if i == len(named) else ("weight", "bias")[i & 1] + (str(i // 2 + 1) if len(maps) > 1 else "")
            if t.dtype != dtype:
                raise ValueError(f"{what}: {name} has dtype {t.dtype}; expected {dtype}")
            raise ValueError(f"{what}: {name} is on {t.device}, x on {dev}")
    if dev.type != "cuda":
        raise ValueError(f"{what} runs on a ROCm device; got tensors on {dev}")
    if _is_tracing():
        raise RuntimeError(f"{what} cannot be traced: its launches are no part of a traced graph")
    if x.numel() > MAX_ROWS * shape[-1]:
        raise ValueError(f"{what}: x of shape {tuple(shape)} has more than {MAX_ROWS} rows")
    return act


def _flat(t: Optional[torch.Tensor], n: int) -> Optional[torch.Tensor]:
    return t if t is None or t.dim() == 2 else t.reshape(-1, n)


def _new(like: torch.Tensor, *shape) -> torch.Tensor:
    return torch.empty(shape, dtype=like.dtype, device=like.device)


def _out(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _zeros(like: torch.Tensor, *wanted):
    """Gradients over no rows: (shape, whether it is wanted)."""
    return [like.new_zeros(shape) if need else None for shape, need in wanted]


class LinearActFunction(torch.autograd.Function):
    """``linear_act`` as one node; keeps its input, weight and, with an
    activation, the value before it."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        N, K = weight.shape
        with _on(x.device):
            x2 = _flat(x, K)
            M = x2.shape[0]
            y = _new(x, *x.shape[:-1], N)
            z = torch.empty((M, _up8(N)), dtype=_PRE[x.dtype], device=x.device) if act else None
            x2, w = _forward(x2, K, weight, bias, _flat(residual, N), act, y.data_ptr(), N, _out(z), _up8(N), True)
        ctx.save_for_backward(x2, w, z)
        ctx.act, ctx.shape, ctx.N = act, x.shape, N
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x2, w, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        act, N, K, M = ctx.act, ctx.N, ctx.shape[-1], x2.shape[0]
        dx = dw = db = None
        if M == 0:
            dx, dw, db = _zeros(x2, (ctx.shape, need_x), ((N, K), need_w), ((N,), need_b))
        elif need_x or need_w or need_b:
            with _on(x2.device):
                d = _rows(_flat(dy, N))
                if need_x:
                    dx = _new(x2, *ctx.shape)
                if need_w or need_b:
                    dw = _new(x2, N, K)
                    db = _new(x2, N) if need_b else None
                lib, code, pd, ld = _lib.load(), _DTYPE_CODE[x2.dtype], d.data_ptr(), _ld(d)
                n = lib.kda_linear_bwd_workspace_size(pd, ld, M, N, K, act, code)
                ws = torch.empty(n, dtype=torch.uint8, device=x2.device)
                rc = lib.kda_linear_bwd(pd, ld, x2.data_ptr(), _ld(x2), w.data_ptr(), _ld(w), _out(z),
                                        z.stride(0) if act else 0, _out(dx), K, _out(dw), _out(db), M, N, K, act, code,
                                        ws.data_ptr(), n, _raw_stream(x2.device.index))
                if rc:
                    _lib.check(rc, "kda_linear_bwd")
        return dx, dw if need_w else None, db, dy if need_r else None, None


class MLPFunction(torch.autograd.Function):
    """``mlp`` as one node; keeps x, the weights, the hidden layer and the value
    before its activation."""

    @staticmethod
    def forward(ctx, x, w1, b1, w2, b2, residual, act):
        (N, K), O = w1.shape, w2.shape[0]
        with _on(x.device):
            x2 = _flat(x, K)
            M = x2.shape[0]
            h = _new(x, M, _up8(N))
            z = torch.empty((M, _up8(N)), dtype=_PRE[x.dtype], device=x.device) if act else None
            y = _new(x, *x.shape[:-1], O)
            x2, w1 = _forward(x2, K, w1, b1, None, act, h.data_ptr(), _up8(N), _out(z), _up8(N), True)
            h, w2 = _forward(h, N, w2, b2, _flat(residual, O), 0, y.data_ptr(), O, None, 0, True)
        ctx.save_for_backward(x2, w1, z, h, w2)
        ctx.act, ctx.shape, ctx.sizes = act, x.shape, (N, O)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x2, w1, z, h, w2 = ctx.saved_tensors
        need_x, need_w1, need_b1, need_w2, need_b2, need_r = ctx.needs_input_grad[:6]
        act, (N, O), K, M = ctx.act, ctx.sizes, ctx.shape[-1], x2.shape[0]
        dx = dw1 = db1 = dw2 = db2 = None
        if M == 0:
            dx, dw1, db1, dw2, db2 = _zeros(x2, (ctx.shape, need_x), ((N, K), need_w1), ((N,), need_b1),
                                            ((O, N), need_w2), ((O,), need_b2))
        elif need_x or need_w1 or need_b1 or need_w2 or need_b2:
            with _on(x2.device):
                d = _rows(_flat(dy, O))
                if need_x:
                    dx = _new(x2, *ctx.shape)
                if need_w1 or need_b1:
                    dw1 = _new(x2, N, K)
                    db1 = _new(x2, N) if need_b1 else None
                if need_w2 or need_b2:
                    dw2 = _new(x2, O, N)
                    db2 = _new(x2, O) if need_b2 else None
                lib, code, pd, ld = _lib.load(), _DTYPE_CODE[x2.dtype], d.data_ptr(), _ld(d)
                n = lib.kda_mlp_bwd_workspace_size(pd, ld, M, N, K, O, act, code)
                ws = torch.empty(n, dtype=torch.uint8, device=x2.device)
                rc = lib.kda_mlp_bwd(pd, ld, x2.data_ptr(), _ld(x2), w1.data_ptr(), _ld(w1), _out(z),
                                     z.stride(0) if act else 0, h.data_ptr(), _ld(h), w2.data_ptr(), _ld(w2), _out(dx), K,
                                     _out(dw1), _out(db1), _out(dw2), _out(db2), M, N, K, O, act, code, ws.data_ptr(), n,
                                     _raw_stream(x2.device.index))
                if rc:
                    _lib.check(rc, "kda_mlp_bwd")
        return (dx, dw1 if need_w1 else None, db1, dw2 if need_w2 else None, db2, dy if need_r else None, None)


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
               residual: Optional[torch.Tensor] = None, activation: Optional[str] = None) -> torch.Tensor:
    """act(x weight^T + bias) + residual, differentiable.  x (..., K), weight (N, K),
    bias (N,), residual (..., N), all bf16 or all fp32; ``activation`` None, "gelu"
    (z Phi(z)) or "silu".  Rows and weights at any stride; bf16 rows that do not
    begin on 16 bytes, or whose K is no multiple of 8, are copied first when y has
    more than 256 pieces of 16 x 16 (512 up to 8 rows) or a gradient is needed."""
    act = _check("linear_act", x, ((weight, bias),), residual, activation)
    # (a forward-mode tangent: the node refuses it, the kernels would drop it)
    if _grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                            or (residual is not None and residual.requires_grad)) or forward_ad._current_level >= 0:
        return LinearActFunction.apply(x, weight, bias, residual, act)
    N, K = weight.shape
    y = torch.empty((*x.shape[:-1], N), dtype=x.dtype, device=x.device)
    px, pw, M, code = x.data_ptr(), weight.data_ptr(), x.numel() // K, _DTYPE_CODE[x.dtype]
    if (M and x.is_contiguous() and weight.is_contiguous() and (bias is None or bias.is_contiguous())
            and (residual is None or residual.is_contiguous()) and not (code and ((px | pw) & 15 or K & 7) and not _few(M, N))
            and K <= MAX_STRIDE and N <= MAX_STRIDE and x.get_device() == _current_device()):
        # as they lie: half the time of such a call is the host's
        rc = _lib.load().kda_linear_fwd(
            px, K, pw, K, None if bias is None else bias.data_ptr(), None if residual is None else residual.data_ptr(), N,
            y.data_ptr(), N, None, 0, M, N, K, act, code, _raw_stream(x.get_device()))
        if rc:
            _lib.check(rc, "kda_linear_fwd")
        return y
    with _on(x.device):
        _forward(_flat(x, K), K, weight, bias, _flat(residual, N), act, y.data_ptr(), N, None, 0, False)
    return y


def mlp(x: torch.Tensor, w1: torch.Tensor, b1: Optional[torch.Tensor], w2: torch.Tensor, b2: Optional[torch.Tensor],
        residual: Optional[torch.Tensor] = None, activation: Optional[str] = "gelu") -> torch.Tensor:
    """act(x w1^T + b1) w2^T + b2 + residual, differentiable.  x (..., K), w1 (N, K),
    w2 (K', N), biases or None, residual (..., K'), all bf16 or all fp32.  The hidden
    layer is rounded to their dtype between the two maps."""
    act = _check("mlp", x, ((w1, b1), (w2, b2)), residual, activation)
    if (_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w1, b1, w2, b2, residual))
            or forward_ad._current_level >= 0):
        return MLPFunction.apply(x, w1, b1, w2, b2, residual, act)
    (N, K), O = w1.shape, w2.shape[0]
    with _on(x.device):
        x2 = _flat(x, K)
        h, y = _new(x, x2.shape[0], _up8(N)), _new(x, *x.shape[:-1], O)
        _forward(x2, K, w1, b1, None, act, h.data_ptr(), _up8(N), None, 0, False)
        _forward(h, N, w2, b2, _flat(residual, O), 0, y.data_ptr(), O, None, 0, False)
    return y
