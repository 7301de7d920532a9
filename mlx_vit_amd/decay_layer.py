"""DecayAttentionLayer: linear attention with a decay for each head and rotary positions.

The place of ``GatedDeltaLayer`` in a block (the same state, the same call but for the tokens'
numbers), without the delta rule and the short convolutions, so without a write gate, and with positions on a video's
axes instead: queries and keys are turned (``rotary``), mixed by ``chunk_decay`` and
normalised and gated by ``RMSNormGated`` (nope_gdn_mlx.py:340-366).  The decay is the
reference's decay gate for one head (nope_gdn_mlx.py:812-819),
g = -exp(A_log) softplus(a_proj(x) + dt_bias).
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import torch
import torch.nn as nn
import torch.nn.functional as F

from .decay import HEAD_DIMS, chunk_decay, decay_step
from .layer import RMSNormGated
from .positions import rotary


def video_sections(head_dim: int) -> Tuple[int, int, int]:
    """Channels for time, height and width: three eighths or less for each of the latter, the rest for time."""
    space = head_dim // 32 * 12
    return head_dim - 2 * space, space, space


class DecayAttentionLayer(nn.Module):
    """``forward(x, state=None, start=None) -> (out, new_state)``, x (B, L, hidden_size), state
    (B, H, D, D) fp32 or None; ``start``: the first token's number in its video, a number for all rows
    (a captured graph keeps it) or (B,) int32 or int64 on x's device, each row's (a graph reads it
    anew).  A state holds keys turned by their positions, so whoever goes on from one says from
    where; without a state it is 0.
    ``grid`` = (height, width): the tokens of a frame.  ``num_kv_heads``: key and value heads, each
    shared by num_heads / num_kv_heads heads (default: one each)."""

    def __init__(self, hidden_size: int, num_heads: int = 6, head_dim: int = 64, num_kv_heads: Optional[int] = None,
                 grid: Tuple[int, int] = (14, 14), sections: Optional[Sequence[int]] = None, base: float = 10000.0):
        super().__init__()
        kv = num_heads if num_kv_heads is None else num_kv_heads
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim={head_dim}: expected one of {HEAD_DIMS}")
        if kv < 1 or num_heads % kv:
            raise ValueError(f"num_kv_heads={kv} does not divide num_heads={num_heads}")
        self.hidden_size, self.num_heads, self.head_dim, self.num_kv_heads = hidden_size, num_heads, head_dim, kv
        self.grid, self.base = tuple(grid), base
        self.sections = video_sections(head_dim) if sections is None else tuple(sections)
        self.scale = head_dim ** -0.5
        total = num_heads * head_dim
        self.q_proj = nn.Linear(hidden_size, total, bias=False)
        self.k_proj = nn.Linear(hidden_size, kv * head_dim, bias=False)
        self.v_proj = nn.Linear(hidden_size, kv * head_dim, bias=False)
        self.a_proj = nn.Linear(hidden_size, num_heads, bias=False)
        self.A_log = nn.Parameter(torch.empty(num_heads).uniform_(0.01, 1.0).log_())
        self.dt_bias = nn.Parameter(torch.zeros(num_heads))
        self.g_proj = nn.Linear(hidden_size, total, bias=False)
        self.o_norm = RMSNormGated(head_dim, eps=1e-5)
        self.o_proj = nn.Linear(total, hidden_size, bias=False)

    def _where(self, x: torch.Tensor, start: Union[int, torch.Tensor]) -> dict:
        """rotary's positions of x's tokens."""
        if not isinstance(start, torch.Tensor) or not start.dim():
            return dict(grid=self.grid, start=start)
        if start.shape != x.shape[:1] or start.dtype not in (torch.int32, torch.int64) or start.device != x.device:
            raise ValueError(f"start must be a number or ({x.shape[0]},) int32 or int64 on {x.device}; "
                             f"got {tuple(start.shape)} {start.dtype} on {start.device}")
        h, w = self.grid
        n = start[:, None] + torch.arange(x.shape[1], device=x.device)
        return dict(positions=torch.stack([n // (h * w), n // w % h, n % w][:len(self.sections)]))

    def _operands(self, x: torch.Tensor, start: Union[int, torch.Tensor]):
        if x.dim() != 3 or x.shape[-1] != self.hidden_size:
            raise ValueError(f"x must be (B, L, {self.hidden_size}); got {tuple(x.shape)}")
        D = self.head_dim
        q, k, v = (p(x).unflatten(-1, (-1, D)) for p in (self.q_proj, self.k_proj, self.v_proj))
        q, k = rotary(q * self.scale, k, **self._where(x, start), sections=self.sections, base=self.base)
        g = -torch.exp(self.A_log.float()) * F.softplus(self.a_proj(x).float() + self.dt_bias.float())
        return q, k, v, g

    def forward(self, x: torch.Tensor, state: Optional[torch.Tensor] = None,
                start: Union[None, int, torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        if start is None:
            if state is not None:
                raise ValueError("a state was given without start, the number of the first token in its video")
            start = 0
        o, new_state = chunk_decay(*self._operands(x, start), state)
        return self.o_proj(self.o_norm(o, self.g_proj(x))), new_state

    @torch.no_grad()
    def step(self, x: torch.Tensor, state: torch.Tensor, start: Union[int, torch.Tensor],
             slots: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The next token of each row, x (B, 1, hidden_size), number ``start`` of its video, as in forward; ``state``
        is updated: (B, H, D, D), or (N, H, D, D) with ``slots`` (B,) int32, the state of each row (``decay_step``)."""
        q, k, v, g = self._operands(x, start)
        if x.shape[1] != 1:
            raise ValueError(f"a step takes one token of each row; got {x.shape[1]}")
        o = decay_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], state, slots)
        return self.o_proj(self.o_norm(o[:, None], self.g_proj(x)))
