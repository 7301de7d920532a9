"""``chunk_decay`` and ``decay_step`` in 64 bits, token after token, from the definitions.

Called on absolute values the same functions give what an error of rounding grows
with: every output is a sum of products of the inputs, with e^g > 0 between."""
import torch


def heads(t, H):
    """(..., heads, D) -> (..., H, D) in 64 bits, on the CPU."""
    return t.detach().double().cpu().repeat_interleave(H // t.shape[-2], -2)


def spans(T, cu, B):
    """(first token, behind the last, its states) of each sequence."""
    if cu is None:
        return [(0, T, slice(0, B))]
    return [(cu[i], cu[i + 1], slice(i, i + 1)) for i in range(len(cu) - 1)]


def forward(q, k, v, g, s0=None, cu=None):
    """o, the final states; q, k, v (B, T, heads, D), g (B, T, H) or (H,), cu a list."""
    H, (B, T, _, D) = g.shape[-1], q.shape
    q, k, v = heads(q, H), heads(k, H), heads(v, H)
    f = torch.exp(g.detach().double().cpu()).expand(B, T, H)[..., None, None]
    n = B if cu is None else len(cu) - 1
    S = torch.zeros(n, H, D, D, dtype=torch.float64) if s0 is None else s0.detach().double().cpu().clone()
    o = torch.zeros(B, T, H, D, dtype=torch.float64)
    for lo, hi, own in spans(T, cu, B):
        s = S[own]
        for t in range(lo, hi):
            s = torch.where(f[:, t] == 0, 0.0, f[:, t] * s) + v[:, t, :, :, None] * k[:, t, :, None, :]
            o[:, t] = (s * q[:, t, :, None, :]).sum(-1)
        S[own] = s
    return o, S


def backward(q, k, v, g, s0, cu, do, ds):
    """dq, dk, dv, dg, ds0 of <o, do> + <final states, ds> (do, ds: may be None)."""
    H, (B, T, _, D), one = g.shape[-1], q.shape, g.dim() == 1
    shares = [t.shape[2] for t in (q, k, v)]
    q, k, v = heads(q, H), heads(k, H), heads(v, H)
    f = torch.exp(g.detach().double().cpu()).expand(B, T, H)[..., None, None]
    n = B if cu is None else len(cu) - 1
    zero = torch.zeros(n, H, D, D, dtype=torch.float64)
    S = zero.clone() if s0 is None else s0.detach().double().cpu().clone()
    dS = zero.clone() if ds is None else ds.detach().double().cpu().clone()
    do = torch.zeros(B, T, H, D, dtype=torch.float64) if do is None else do.detach().double().cpu()
    dq, dk, dv = (torch.zeros(B, T, H, D, dtype=torch.float64) for _ in range(3))
    dg = torch.zeros(B, T, H, dtype=torch.float64)
    for lo, hi, own in spans(T, cu, B):
        s, kept = S[own], []
        for t in range(lo, hi):
            kept.append(f[:, t] * s)
            s = kept[-1] + v[:, t, :, :, None] * k[:, t, :, None, :]
            dq[:, t] = (s * do[:, t, :, :, None]).sum(-2)
        d = dS[own]
        for t in range(hi - 1, lo - 1, -1):
            d = d + do[:, t, :, :, None] * q[:, t, :, None, :]
            dv[:, t] = (d * k[:, t, :, None, :]).sum(-1)
            dk[:, t] = (d * v[:, t, :, :, None]).sum(-2)
            dg[:, t] = (d * kept[t - lo]).sum((-1, -2))
            d = f[:, t] * d
        dS[own] = d
    group = lambda t, n: t.unflatten(2, (n, -1)).sum(3)  # noqa: E731
    return (group(dq, shares[0]), group(dk, shares[1]), group(dv, shares[2]), dg.sum((0, 1)) if one else dg,
            None if s0 is None else dS)


def step(q, k, v, g, state, slots=None):
    """o and the states after one token of each row; a slot outside the states is left out, rows
    of one slot follow each other."""
    H = g.shape[-1]
    q, k, v, S = heads(q, H), heads(k, H), heads(v, H), state.detach().double().cpu().clone()
    f = torch.exp(g.detach().double().cpu()).expand(q.shape[0], H)
    o = torch.zeros_like(q)
    for b, n in enumerate(range(len(q)) if slots is None else slots):
        if 0 <= n < len(S):
            S[n] = f[b, :, None, None] * S[n] + v[b, :, :, None] * k[b, :, None, :]
            o[b] = (S[n] * q[b, :, None, :]).sum(-1)
    return o, S
