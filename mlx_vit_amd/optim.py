"""AdamW over all of a model's tensors in a few launches: ``FusedAdamW``.

The update is ``train.AdamW``'s (the reference's, train_mlx_k400.py:548-549), with
the gradients' global norm and clip (train_mlx_k400.py:241-252) folded into it:
the norm is one pass over the gradients, and the update multiplies each gradient
by the clip factor as it reads it, so no gradient is rewritten.  What differs is
what the moments are held in: fp32 whatever the weights' dtype, or 8 bits with a
scale for each 256 elements, and on request an fp32 copy of the weights
(``master_weights``) that bf16 weights are the rounding of, so that updates below
half a bf16 step add up.

8-bit moments: m = s (k / 127) |k / 127|, k in [-127, 127], s the block's largest
|m|; v = (s (k / 255)^2)^2, k in [0, 255], s the block's largest sqrt(v); k / 127 and
k / 255 are products with the fp32 numbers next to 1 / 127 and 1 / 255.  The update
uses the new moments before they are rounded.  A gradient that is not finite makes its
whole block of 8-bit moments NaN.
"""
from __future__ import annotations

from array import array
from operator import attrgetter
from typing import Dict, Iterable, List, Optional, Tuple

import torch
import torch.nn as nn

from . import _lib
from .kda import _DTYPE_CODE, _ptr, _stream
from .linear import _on, _raw_stream

BLOCK = 256      # elements that share a scale; a tensor's moments begin on a multiple of it
_STATES = {"fp32": 0, "int8": 1}
_increment_version = torch._C._increment_version
_data_ptr, _contiguous, _nbytes = torch.Tensor.data_ptr, torch.Tensor.is_contiguous, attrgetter("nbytes")


def _overlap(spans: List[Tuple[int, int]]) -> bool:
    """Do any two of these (address, bytes) share memory?"""
    spans = sorted(s for s in spans if s[1])
    return any(a + n > b for (a, n), (b, _) in zip(spans, spans[1:]))


class FusedAdamW:
    """AdamW with moments of their own dtype.  A captured step replays with the learning
    rate, and the bias corrections, that it was captured with, on the weights' memory of
    then, which the optimizer keeps; it needs the optimizer and those gradients alive.

    ``states``: "fp32" or "int8"; ``master_weights``: keep and update fp32 copies of
    the weights; ``bias_correction``: divide the moments by 1 - beta^step (off in
    the reference).  ``state``: buffers to use (not copied), as the attribute
    ``state`` of an optimizer over the same tensors holds them: "m", "v" (fp32, or
    int8 and uint8 with "m_scale" and "v_scale"), "master"; parameter i's part
    begins at ``offsets[i]`` and what lies between two parameters' is zero.

    With ``master_weights`` a weight that is changed other than by ``step`` gets its
    master's value back at the next one.

    Parameters are contiguous fp32 or bf16 tensors on one ROCm device, and stay so;
    gradients have their dtype.  Those without a gradient at a step are left out of it."""

    def __init__(self, params: Iterable[nn.Parameter], lr: float = 3e-4, betas=(0.9, 0.95), eps: float = 1e-8,
                 weight_decay: float = 0.05, states: str = "fp32", master_weights: bool = False,
                 bias_correction: bool = False, state: Optional[Dict[str, torch.Tensor]] = None):
        if states not in _STATES:
            raise ValueError(f"states={states!r}: expected one of {tuple(_STATES)}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0) or not eps >= 0.0:
            raise ValueError(f"betas={betas}, eps={eps}: expected betas in [0, 1) and eps >= 0")
        self.params: List[nn.Parameter] = [p for p in params if p.requires_grad]
        if not self.params:
            raise ValueError("no parameters to optimise")
        self.lr, self.betas, self.eps, self.weight_decay = lr, betas, eps, weight_decay
        self.states, self.bias_correction = states, bias_correction
        self.steps = 0
        self.device = self.params[0].device
        for p in self.params:
            if p.device.type != "cuda" or p.device != self.device:
                raise ValueError(f"FusedAdamW runs on one ROCm device; got parameters on {p.device} and {self.device}")
            if p.dtype not in _DTYPE_CODE or not p.is_contiguous():
                raise ValueError("parameters must be contiguous float32 or bfloat16 tensors; got "
                                 f"{p.dtype}, shape {tuple(p.shape)}, strides {p.stride()}")
        self._dtypes = [p.dtype for p in self.params]
        self._numels = [p.numel() for p in self.params]
        self._bytes = [p.nbytes for p in self.params]
        self.offsets: List[int] = []
        at = 0
        for n in self._numels:
            self.offsets.append(at)
            at += -(-n // BLOCK) * BLOCK
        self.total = at
        self._state = self._new_state(master_weights) if state is None else self._given_state(state, master_weights)
        # the streams that the buffers' memory waits for (the one it was allocated on; of given ones that is not known)
        self._state_streams = {_raw_stream(self.device.index)} if state is None else set()
        # p, g, n, offset, dtype of each parameter
        self._ptrs: List[int] = []
        self._plan: Optional[torch.Tensor] = None
        self._captured: List[tuple] = []
        self._table = array("q", [v for n, o, t in zip(self._numels, self.offsets, self._dtypes)
                                  for v in (0, 0, n, o, _DTYPE_CODE[t])])
        self._check_params(list(map(_data_ptr, self.params)))

    # ---- state -----------------------------------------------------------
    def _specs(self, master: bool) -> Dict[str, Tuple[torch.dtype, int]]:
        n = self.total
        if self.states == "fp32":
            specs = {"m": (torch.float32, n), "v": (torch.float32, n)}
        else:
            specs = {"m": (torch.int8, n), "v": (torch.uint8, n), "m_scale": (torch.float32, n // BLOCK),
                     "v_scale": (torch.float32, n // BLOCK)}
        if master:
            specs["master"] = (torch.float32, n)
        return specs

    def _new_state(self, master: bool) -> Dict[str, torch.Tensor]:
        state = {k: torch.zeros(n, dtype=t, device=self.device) for k, (t, n) in self._specs(master).items()}
        if master:
            with torch.no_grad():
                torch._foreach_copy_(self.views(state["master"]), self.params)
        return state

    def _given_state(self, state: Dict[str, torch.Tensor], master: bool) -> Dict[str, torch.Tensor]:
        specs = self._specs(master)
        if set(state) != set(specs):
            raise ValueError(f"state holds {sorted(state)}; expected {sorted(specs)}")
        for k, (t, n) in specs.items():
            s = state[k]
            if (s.dtype != t or tuple(s.shape) != (n,) or s.device != self.device or not s.is_contiguous()
                    or s.data_ptr() & 15):
                raise ValueError(f"state[{k!r}] must be a contiguous 16-byte aligned {t} tensor of {n} elements on "
                                 f"{self.device}; got {s.dtype}, shape {tuple(s.shape)} on {s.device}")
        if _overlap([(s.data_ptr(), s.nbytes) for s in state.values()]):
            raise ValueError("state's buffers overlap in memory")
        return dict(state)

    @property
    def state(self) -> Dict[str, torch.Tensor]:
        """The buffers of moments (and masters) by name."""
        return dict(self._state)

    def views(self, flat: torch.Tensor) -> List[torch.Tensor]:
        """Each parameter's part of a buffer laid out as the moments."""
        return [flat[o:o + n].view(p.shape) for p, o, n in zip(self.params, self.offsets, self._numels)]

    def moments(self, dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
        """(m, v) as buffers of values (``views`` gives the parameters' parts): with
        fp32 states the state's own buffers, in another dtype copies."""
        m, v = self._state["m"], self._state["v"]
        with _on(self.device):
            self._use()
        if self.states == "fp32":
            return m.to(dtype), v.to(dtype)
        if dtype not in _DTYPE_CODE:
            raise ValueError(f"dtype {dtype} unsupported: use float32 or bfloat16")
        mo = torch.empty(self.total, dtype=dtype, device=self.device)
        vo = torch.empty_like(mo)
        with _on(self.device):
            _lib.check(_lib.load().kda_adamw_moments(
                _ptr(m), _ptr(v), _ptr(self._state["m_scale"]), _ptr(self._state["v_scale"]), _ptr(mo), _ptr(vo),
                self.total, _DTYPE_CODE[dtype], _stream(self.device)), "kda_adamw_moments")
        return mo, vo

    def state_dict(self) -> dict:
        return {"steps": self.steps, **self._state}

    def load_state_dict(self, state: dict) -> None:
        """Copy a ``state_dict`` of an optimizer over the same tensors into this one's buffers."""
        if set(state) != {"steps", *self._state}:
            raise ValueError(f"state holds {sorted(state)}; expected {sorted(('steps', *self._state))}")
        for k, t in self._state.items():
            if state[k].dtype != t.dtype or state[k].shape != t.shape:
                raise ValueError(f"state[{k!r}] is {state[k].dtype} {tuple(state[k].shape)}; expected {t.dtype} "
                                 f"{tuple(t.shape)}")
        with _on(self.device):
            self._use()
        for k, t in self._state.items():
            t.copy_(state[k])
        self.steps = int(state["steps"])

    # ---- the step --------------------------------------------------------
    def _check_params(self, ptrs: List[int]) -> None:
        """The parameters' addresses are new: are they still what the optimizer was made for?"""
        for p, t, n in zip(self.params, self._dtypes, self._numels):
            if p.dtype != t or p.numel() != n or not p.is_contiguous() or p.device != self.device:
                raise ValueError(f"a parameter of {n} elements of {t} is now {tuple(p.shape)}, {p.dtype}, strides "
                                 f"{p.stride()} on {p.device}: make a new optimizer")
            # (a step looks at the gradients' sizes in bytes: half precision's are bf16's)
            if getattr(p, "grad_dtype", t) != t:
                raise ValueError(f"a parameter of {t} takes gradients of grad_dtype={p.grad_dtype}: expected its own dtype")
        if _overlap([(a, p.nbytes) for a, p in zip(ptrs, self.params)]):
            raise ValueError("parameters overlap in memory (one of them is given twice, or two share a storage)")
        if self._plan is not None and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("parameters were moved since the last step: take one outside the capture first")
        table = array("q", self._table)
        table[0::5] = array("q", ptrs)
        lib, at, count = _lib.load(), table.buffer_info()[0], len(self.params)
        host = torch.empty(lib.kda_adamw_plan_size(at, count), dtype=torch.uint8)
        _lib.check(lib.kda_adamw_plan(at, count, host.data_ptr(), host.numel()), "kda_adamw_plan")
        parts = lib.kda_adamw_step_workspace_size(at, count) // 8
        storages = [p.untyped_storage() for p in self.params]
        if self._plan is not None:
            torch.cuda.synchronize(self.device)   # a step may be reading the old plan, on any stream
        plan = host.to(self.device)
        # all at once, the addresses last: after a failure above the next step comes here again
        # (while the storages are held no other tensor can come to lie at the same address)
        self._table, self._plan, self._parts, self._storages = table, plan, parts, storages
        self._plan_streams = {_raw_stream(self.device.index)}
        self._ptrs = ptrs

    def _use(self) -> bool:
        """Work on the device's current stream uses the buffers: their memory must not be given away
        before it has ended, even if the optimizer is dropped.  A stream once recorded stays so.
        Returns whether the stream is being captured (a graph's user keeps the optimizer)."""
        if torch.cuda.is_current_stream_capturing():
            return True
        stream = _raw_stream(self.device.index)
        for known, buffers in ((self._state_streams, self._state.values()), (self._plan_streams, (self._plan,))):
            if stream not in known:
                current = torch.cuda.current_stream(self.device)
                for t in buffers:
                    t.record_stream(current)
                known.add(stream)
        return False

    def _gradients(self) -> Tuple[List[Optional[torch.Tensor]], List[nn.Parameter]]:
        """Fill the descriptors for a step; returns the gradients, to be kept until the
        launches, and the parameters that have one."""
        ptrs = list(map(_data_ptr, self.params))
        if ptrs != self._ptrs:
            self._check_params(ptrs)
        gs = present = [p.grad for p in self.params]
        sizes = self._bytes
        # (each such look at 436 tensors is 15 us of the host's)
        try:
            fits, missing = list(map(_nbytes, gs)) == sizes, False
        except AttributeError:   # None
            missing = True
            present = [g for g in gs if g is not None]
            fits = [g.nbytes for g in present] == [n for n, g in zip(sizes, gs) if g is not None]
        if not fits:
            raise ValueError("a gradient's size or dtype is not that of its parameter when the optimizer was made")
        if not all(map(_contiguous, present)):
            # gradients lie as their parameters do
            if not all(map(_contiguous, self.params)):
                raise ValueError("a parameter is no longer contiguous: make a new optimizer")
            gs = [g if g is None else g.detach().contiguous() for g in gs]
        self._table[1::5] = array("q", [0 if g is None else g.data_ptr() for g in gs] if missing
                                  else list(map(_data_ptr, gs)))
        return gs, [p for p, g in zip(self.params, gs) if g is not None] if missing else self.params

    def step(self, max_norm: Optional[float] = None) -> Optional[torch.Tensor]:
        """One update.  With ``max_norm`` the gradients count scaled by
        min(max_norm / (G + 1e-6), 1), G their global norm, which is returned (0-d
        fp32); the gradients themselves stay as they are."""
        if max_norm is not None and not max_norm > 0.0:
            raise ValueError(f"max_norm={max_norm}: expected a positive number or None")
        gs, updated = self._gradients()   # (gs: alive until the launches)
        b1, b2 = self.betas
        c1 = 1.0 / (1.0 - b1 ** (self.steps + 1)) if self.bias_correction else 1.0
        c2 = 1.0 / (1.0 - b2 ** (self.steps + 1)) if self.bias_correction else 1.0
        lib, at, count = _lib.load(), self._table.buffer_info()[0], len(self.params)
        plan = self._plan.data_ptr()
        get = self._state.get
        buffers = [None if t is None else t.data_ptr()
                   for t in (get("m"), get("v"), get("m_scale"), get("v_scale"), get("master"))]
        clip, pc, pw, parts = None, None, None, 0
        with _on(self.device):
            stream = _raw_stream(self.device.index)
            if self._use() and not any(kept[0] is self._plan for kept in self._captured):
                # the graph reads the plan at each replay, and writes the weights that it names, also after they moved
                self._captured.append((self._plan, self._storages))
            if max_norm is not None:
                # the norm and the clip factor; the norm's partial sums (fp64), behind them while they
                # are few, since who keeps the norm keeps what it lies in
                parts = self._parts
                clip = torch.empty(2 + 2 * parts if parts < 256 else 2, dtype=torch.float32, device=self.device)
                pc = clip.data_ptr()
                pw = pc + 8
                if parts >= 256:
                    sums = torch.empty(parts, dtype=torch.float64, device=self.device)
                    pw = sums.data_ptr()
            rc = lib.kda_adamw_step(at, count, plan, _STATES[self.states], *buffers, max_norm or 0.0, pc, self.lr, b1, b2,
                                    self.eps, self.weight_decay, c1, c2, pw, 8 * parts, stream)
            if rc:
                _lib.check(rc, "kda_adamw_step")
        self.steps += 1
        # a graph that holds the weights as they were has to notice
        _increment_version(updated)
        return None if clip is None else clip[0]

    def zero_grad(self) -> None:
        for p in self.params:
            p.grad = None
