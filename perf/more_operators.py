"""Linear attention with a decay for each head and the rotary positions of its queries
and keys, as measurable cases.

* ``rotary``: queries and keys turned by positions on several axes (time, height,
  width), with the gradients in training;
* ``decay``: ``chunk_decay``, S_t = e^{g_t} S_{t-1} + v_t k_t^T, o_t = S_t q_t over whole
  prompts, padded to one length or packed, with the gradients in training;
* ``step``: ``decay_step``, the same for one token of each sequence, on states that
  stay where they are.

A case is a dict of plain values: ``B`` sequences of ``T`` tokens (``lens``, if not empty:
one packed row of sequences of these lengths), ``H`` heads of ``D`` channels (``HK`` key
and value heads, or key heads alone), ``dtype``, ``train``.  ``rotary``: ``sections``, the
channels of each axis; ``grid``, the tokens of a frame's height and width, or "" for
positions given as numbers from ``start`` on; ``pairs``: "halves" or "neighbours".
``decay`` and ``step``: ``g`` "token", a log-decay of every token, or "head", one for each
head; ``state``: it starts from a state and returns the last one.  ``step``: ``N`` states.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
DEVICE = "cuda"
CHUNK = 64                  # tokens of a block of the plain form
BASE = 10000.0              # wave lengths of an axis: 2 pi to 2 pi BASE


def _rotary(name, B, T, H, HK, D, sections, grid="", start=0, pairs="halves", dtype="bf16", train=False):
    c = dict(kind="rotary", B=B, T=T, H=H, HK=HK, D=D, sections=sections, grid=grid, start=start, pairs=pairs, dtype=dtype,
             train=train)
    return dict(name=name, **c) if name else c


def _decay(name, B, T, H, HK, D, g="token", state=False, lens="", dtype="bf16", train=False):
    c = dict(kind="decay", B=B, T=T, H=H, HK=HK, D=D, g=g, state=state, lens=lens, dtype=dtype, train=train)
    return dict(name=name, **c) if name else c


def _step(name, B, N, H, HK, D, g="token", dtype="bf16"):
    c = dict(kind="step", B=B, N=N, T=1, H=H, HK=HK, D=D, g=g, dtype=dtype, train=False)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # streaming inference: the next tubelet's 196 tokens of one clip, far into the video
        _rotary("rotary-stream", 1, 196, 6, 6, 64, "16,24,24", "14,14", 196 * 300),
        # training the default classifier's width on 8 clips of 3136 tokens
        _rotary("rotary-train", 8, 3136, 6, 6, 64, "16,24,24", "14,14", train=True),
        # a long prompt with few key heads, one axis, positions beyond a million
        _rotary("rotary-long", 1, 65537, 16, 4, 128, "128", "", 1 << 20, "neighbours"),
        # streaming inference: the next tubelet from the state that the last one left
        _decay("decay-stream", 1, 196, 6, 6, 64, state=True),
        # classifying 8 clips of 1568 tokens at width 768
        _decay("decay-clips", 8, 1568, 12, 12, 64),
        # the same in training, the decay with a gradient too
        _decay("decay-train", 8, 1568, 12, 12, 64, train=True),
        # training in fp32 (the parity mode), odd length, from a state and with the last state's gradient
        _decay("decay-train-fp32", 2, 1571, 6, 6, 32, state=True, dtype="fp32", train=True),
        # prompts of different lengths in one row, four heads to a key and value head, fixed decays
        _decay("decay-packed-train", 1, 20000, 16, 4, 128, "head", lens="1,8191,0,63,700,4096,65,1999,128,4757", train=True),
        # one long video: few heads, so the length has to be shared out
        _decay("decay-long", 1, 65536, 12, 12, 64),
        # one stream's next token, where latency counts
        _step("step-one", 1, 1, 6, 6, 64),
        # 200 streams served together out of 256 states
        _step("step-batch", 200, 256, 12, 12, 64),
        # large heads, few of them keys: the states' bytes
        _step("step-wide", 256, 256, 32, 8, 128, "head"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng, most):
    """Heads, and the key heads they share."""
    H = rng.randint(1, most)
    return H, rng.choice([n for n in range(1, H + 1) if H % n == 0] + [H] * 4)


def draw(rng):
    kind = rng.choice(["rotary", "decay", "decay", "decay", "step"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    D = rng.choice([32, 64, 64, 96, 128])
    H, HK = _heads(rng, 24)
    if kind == "step":
        N = _log_int(rng, 1, 512)
        while N * H * D * D > 128e6:
            N //= 2
        return _step(None, rng.randint(max(1, N // 2), N), N, H, HK, D, rng.choice(["token", "head"]), dtype)
    B, T = _log_int(rng, 1, 16), _log_int(rng, 1, 16384)
    if kind == "rotary":
        while B * T * (H + HK) * D > 1.3e8:
            T //= 2
        third = D // 32 * 12        # a multiple of four below D / 2
        sections = rng.choice([str(D), str(D // 2), "%d,%d" % (D // 2, D // 2), "%d,%d,%d" % (D - 2 * third, third, third)])
        grid = "14,14" if sections.count(",") == 2 and rng.random() < 0.7 else ""
        return _rotary(None, B, T, H, HK, D, sections, grid, rng.choice([0, 0, _log_int(rng, 1, 1 << 21)]),
                       rng.choice(["halves", "neighbours"]), dtype, rng.random() < 0.5)
    train = rng.random() < 0.6
    most = 6e6 if train else 4e7    # token channels; a training case's states are kept by exact()
    while B * T * H * D > most:
        T //= 2
    lens = ""
    if rng.random() < 0.4 and T > 8:
        B, total = 1, min(B * T, 40000)
        cuts = sorted(rng.randint(0, total) for _ in range(rng.randint(1, 12)))
        lens = ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [total]))
        T = total
    return _decay(None, B, max(T, 1), H, HK, D, rng.choice(["token", "token", "head"]), rng.random() < 0.5, lens, dtype, train)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE)


def _lens(case):
    return [int(n) for n in case["lens"].split(",")] if case.get("lens") else []


def _log_decay(case, gen, *shape):
    """Log-decays: heads that forget within a few tokens to heads that keep hundreds,
    each token's by a softplus around its head's."""
    H = case["H"]
    head = -torch.exp2(-1 - 7 * torch.arange(H, device=DEVICE) / max(1, H - 1)) * (1 + 0.1 * _randn(gen, H))
    if case["g"] == "head":
        return head
    return head * torch.nn.functional.softplus(_randn(gen, *shape, H))


def _inputs(case, seed):
    """Tensors by name, None where the case has none: queries and keys as projections
    of a normed input leave them, queries scaled by D^-1/2."""
    B, T, H, HK, D = (case[n] for n in ("B", "T", "H", "HK", "D"))
    dt, gen, rows = DTYPES[case["dtype"]], torch.Generator(device=DEVICE).manual_seed(seed), _lens(case)
    lead = (B,) if case["kind"] == "step" else (B, T)
    x = {"q": (_randn(gen, *lead, H, D) * D ** -0.5).to(dt), "k": (_randn(gen, *lead, HK, D) * D ** -0.5).to(dt)}
    if case["kind"] == "rotary":
        if not case["grid"]:
            axes = case["sections"].count(",") + 1
            at = torch.arange(T, device=DEVICE) + case["start"]
            x["positions"] = torch.stack([at // 7 ** a for a in range(axes)])     # the later axes advance more slowly
        if case["train"]:
            x["dq"], x["dk"] = _randn(gen, B, T, H, D).to(dt), _randn(gen, B, T, HK, D).to(dt)
        return x
    x["v"] = _randn(gen, *lead, HK, D).to(dt)
    x["g"] = _log_decay(case, gen, *lead)
    if case["kind"] == "step":
        x["s"] = 0.3 * _randn(gen, case["N"], H, D, D)
        x["slots"] = torch.randperm(case["N"], generator=gen, device=DEVICE)[:B].to(torch.int32)
        return x
    n = len(rows) or B
    x["s0"] = 0.3 * _randn(gen, n, H, D, D) if case["state"] else None
    if case["train"]:
        x["do"] = _randn(gen, B, T, H, D).to(dt)
        x["ds"] = 0.1 * _randn(gen, n, H, D, D) if case["state"] else None
    if rows:
        x["cu"] = torch.cumsum(torch.tensor([0] + rows, device=DEVICE), 0).to(torch.int32)
    return x


def prepare(case, seed):
    x = _inputs(case, seed)
    names = ("q", "k") if case["kind"] == "rotary" else ("q", "k", "v", "g", "s0")
    leaves = [x[n] for n in names if x.get(n) is not None] if case["train"] else []
    for t in leaves:
        t.requires_grad_(True)
    state = dict(case=case, x=x, leaves=leaves)
    if _lens(case):     # the plain form's: where sequence n's token t lies, and which are there
        rows = torch.tensor(_lens(case), device=DEVICE)
        t = torch.arange(max(_lens(case)), device=DEVICE)
        there = t < rows[:, None]
        state["rows"] = torch.where(there, t + (torch.cumsum(rows, 0) - rows)[:, None], 0), there
    return state


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _angles(case, x):
    """(tokens, pairs) in 64 bits: the positions on the axes times the axes' frequencies."""
    T, sections = case["T"], [int(s) for s in case["sections"].split(",")]
    if case["grid"]:
        h, w = (int(n) for n in case["grid"].split(","))
        at = torch.arange(T, device=DEVICE) + case["start"]
        positions = torch.stack([at // (h * w), at // w % h, at % w])
    else:
        positions = x["positions"]
    return torch.cat([p.double()[:, None] * BASE ** (-torch.arange(0, s, 2, device=DEVICE).double() / s)
                      for p, s in zip(positions, sections)], 1)


def _pairs(case):
    """The channels of every pair's two members, and those that no axis turns."""
    first, second, at = [], [], 0
    for s in (int(n) for n in case["sections"].split(",")):
        if case["pairs"] == "halves":
            a, b = range(at, at + s // 2), range(at + s // 2, at + s)
        else:
            a, b = range(at, at + s, 2), range(at + 1, at + s, 2)
        first, second, at = first + list(a), second + list(b), at + s
    return torch.tensor([first, second], device=DEVICE)


def _turn(t, cos, sin, pairs):
    y, t = t.clone(), t.float()
    a, b = t[..., pairs[0]], t[..., pairs[1]]
    y[..., pairs[0]] = (a * cos - b * sin).to(y.dtype)
    y[..., pairs[1]] = (a * sin + b * cos).to(y.dtype)
    return y


def _plain_rotary(case, x):
    angles, pairs = _angles(case, x), _pairs(case)
    cos, sin = torch.cos(angles).float()[:, None], torch.sin(angles).float()[:, None]
    out = [_turn(x["q"], cos, sin, pairs), _turn(x["k"], cos, sin, pairs)]
    if case["train"]:       # a rotation's transpose turns back
        out += [_turn(x["dq"], cos, -sin, pairs), _turn(x["dk"], cos, -sin, pairs)]
    return out


def _shared(t, H):
    """(n, T, heads, D) -> fp32 (n, H, T, D), each head with its copy."""
    return t.float().repeat_interleave(H // t.shape[2], 2).transpose(1, 2)


def _blocks(t, T):
    """(n, H, T, ...) -> (n, H, blocks, CHUNK, ...), zeros behind T."""
    pad = -T % CHUNK
    t = torch.cat([t, t.new_zeros(*t.shape[:2], pad, *t.shape[3:])], 2)
    return t.reshape(*t.shape[:2], -1, CHUNK, *t.shape[3:])


def _decays(g):
    """Of log-decays (n, H, blocks, CHUNK), sums in 64 bits: to each token from its block's
    start, from each token to its block's end, between two tokens of a block (row t, column s, zero
    where s > t), and from the end of block j to the start of block i."""
    c = g.double().cumsum(-1)
    end = c[..., -1:].cumsum(-2)                                       # to each block's end, from the sequence's start
    n = torch.arange(CHUNK, device=DEVICE)
    inner = torch.exp(torch.where(n[:, None] >= n, c[..., :, None] - c[..., None, :], -math.inf)).float()
    m = torch.arange(end.shape[2], device=DEVICE)
    across = torch.where(m[:, None] > m, end - c[..., -1:] - end.transpose(-1, -2), -math.inf)
    start = torch.exp(end - c[..., -1:]).float()                        # from the sequence's start to each block's
    return torch.exp(c).float(), torch.exp(c[..., -1:] - c).float(), inner, torch.exp(across).float(), start


def _states(add, across, start, s0):
    """Each block's first state, (n, H, blocks, D, D), from what every block adds by its end."""
    n, H, m, D = add.shape[:4]
    s = (across @ add.reshape(n, H, m, D * D)).reshape(add.shape)
    return s if s0 is None else s + start[..., None] * s0[:, :, None]


def _plain_decay_padded(H, train, q, k, v, g, s0, do, ds):
    """chunk_decay over (n, T, heads, D) in 32 bits: o, the last state and, with do, the
    gradients of q, k, v (for each of the H heads), g and s0."""
    T = q.shape[1]
    Q, K, V = (_blocks(_shared(t, H), T) for t in (q, k, v))
    up, down, inner, across, start = _decays(_blocks(g.transpose(1, 2), T))
    add = V.transpose(-1, -2) @ (K * down[..., None])
    S = _states(add, across, start, s0)
    A = (Q @ K.transpose(-1, -2)) * inner
    flat = lambda t: t.reshape(*t.shape[:2], -1, *t.shape[4:])[:, :, :T].transpose(1, 2)  # noqa: E731
    o = flat(A @ V + up[..., None] * (Q @ S.transpose(-1, -2)))
    last = up[:, :, -1, -1, None, None] * S[:, :, -1] + add[:, :, -1]
    if not train:
        return o, last
    # adjoints of the states at the blocks' ends: the same sums from the other side
    dO = _blocks(_shared(do, H), T)
    add_d = dO.transpose(-1, -2) @ (Q * up[..., None])
    dS = _states(add_d, across.transpose(-1, -2), torch.zeros_like(start), None)
    if ds is not None:
        behind = torch.exp(_behind(g, T)).float()                      # from each block's end to the sequence's
        dS = dS + behind[..., None, None] * ds[:, :, None]
    dA = (dO @ V.transpose(-1, -2)) * inner
    from_s = up[..., None] * (dO @ S)
    dq = dA @ K + from_s
    to_s = down[..., None] * (V @ dS)
    dk = dA.transpose(-1, -2) @ Q + to_s
    dv = A.transpose(-1, -2) @ dO + down[..., None] * (K @ dS.transpose(-1, -2))
    # dg_t: everything that passes from before t to t or later, the block's own pairs, what enters and what leaves it
    E = A * (dO @ V.transpose(-1, -2))
    rev = lambda t: t.flip(-1).cumsum(-1).flip(-1)  # noqa: E731
    pairs = rev(E.double().sum(-1)) - rev(E.double().sum(-2))
    entering, leaving = (Q * from_s).sum(-1).double(), (K * to_s).sum(-1).double()
    through = up[..., -1].double() * (S * dS).sum((-1, -2)).double()
    dg = pairs + rev(entering) + leaving.cumsum(-1) - leaving + through[..., None]
    ds0 = None
    if s0 is not None:
        ds0 = up[:, :, 0, -1, None, None] * dS[:, :, 0] + add_d[:, :, 0]
    return o, last, flat(dq), flat(dk), flat(dv), dg.reshape(*dg.shape[:2], -1)[:, :, :T].transpose(1, 2).float(), ds0


def _behind(g, T):
    """Log-decay from each block's end to the sequence's, in 64 bits."""
    c = _blocks(g.transpose(1, 2), T).double().sum(-1)
    return c.flip(-1).cumsum(-1).flip(-1) - c


def _group(t, heads):
    """Gradients (n, T, H, D) of a tensor whose heads are shared."""
    return t.reshape(*t.shape[:2], heads, -1, t.shape[-1]).sum(3)


def _plain_decay(state):
    case, x = state["case"], {n: None if t is None else t.detach() for n, t in state["x"].items()}
    dt, H, HK, B, T, train = DTYPES[case["dtype"]], case["H"], case["HK"], case["B"], case["T"], case["train"]
    g = x["g"] if case["g"] == "token" else x["g"].expand(B, T, H)
    q, k, v, do = x["q"], x["k"], x["v"], x.get("do")
    at = None
    if "rows" in state:
        at, there = state["rows"]
        q, k, v, g, do = (None if t is None else torch.where(there[..., None, None] if t.dim() == 4 else there[..., None],
                                                              t[0][at], torch.zeros((), dtype=t.dtype, device=DEVICE))
                          for t in (q, k, v, g, do))
    out = _plain_decay_padded(H, train, q, k, v, g, x["s0"], do, x.get("ds"))

    def back(t):
        if at is None:
            return t
        y = t.new_zeros(1, T, *t.shape[2:])
        y[0, at[there]] = t[there]
        return y
    o, last = back(out[0]).to(dt), out[1]
    res = [o, last] if case["state"] or not train else [o]
    if not train:
        return res
    dq, dk, dv, dg, ds0 = out[2:]
    dg = back(dg) if case["g"] == "token" else back(dg).double().sum((0, 1)).float()
    res += [back(dq).to(dt), back(_group(dk, HK)).to(dt), back(_group(dv, HK)).to(dt), dg]
    return res if ds0 is None else [*res, ds0]


def _plain_step(case, x):
    H, slots = case["H"], x["slots"].long()
    q, k, v = (t.float().repeat_interleave(H // t.shape[1], 1) for t in (x["q"], x["k"], x["v"]))
    g = x["g"] if case["g"] == "token" else x["g"].expand(case["B"], H)
    s = torch.exp(g)[..., None, None] * x["s"][slots] + v[..., :, None] * k[..., None, :]
    x["s"][slots] = s
    return [(s @ q[..., None])[..., 0].to(x["q"].dtype), x["s"]]


def run(state):
    case, x = state["case"], state["x"]
    if own:
        return {"rotary": _own_rotary, "decay": _own_decay, "step": _own_step}[case["kind"]](state)
    with torch.no_grad():
        if case["kind"] == "decay":
            return _plain_decay(state)
        return (_plain_rotary if case["kind"] == "rotary" else _plain_step)(case, {n: t.detach() for n, t in x.items()})


# ---------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------
def _own_rotary(state):
    from mlx_vit_amd import rotary
    case, x = state["case"], state["x"]
    where = dict(positions=x.get("positions"))
    if case["grid"]:
        where = dict(grid=tuple(int(n) for n in case["grid"].split(",")), start=case["start"])
    y = rotary(x["q"], x["k"], sections=tuple(int(s) for s in case["sections"].split(",")), base=BASE,
               interleaved=case["pairs"] == "neighbours", **where)
    return [*y, *torch.autograd.grad(y, state["leaves"], (x["dq"], x["dk"]))] if case["train"] else list(y)


def _own_decay(state):
    from mlx_vit_amd import chunk_decay
    case, x = state["case"], state["x"]
    o, last = chunk_decay(x["q"], x["k"], x["v"], x["g"], x["s0"], cu_seqlens=x.get("cu"))
    if not case["train"]:
        return [o, last]
    if case["state"]:
        return [o, last, *torch.autograd.grad((o, last), state["leaves"], (x["do"], x["ds"]))]
    return [o, *torch.autograd.grad(o, state["leaves"], x["do"])]


def _own_step(state):
    from mlx_vit_amd import decay_step
    x = state["x"]
    return [decay_step(x["q"], x["k"], x["v"], x["g"], x["s"], slots=x["slots"]), x["s"]]


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    B, T, H, HK, D, train = (case[n] for n in ("B", "T", "H", "HK", "D", "train"))
    es = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "rotary":
        elems = B * T * (H + HK) * D * (2 if train else 1)
        at = 0 if case["grid"] else 8 * T * (case["sections"].count(",") + 1)
        return {"bytes": 2 * es * elems + at, "flops": 3 * elems}
    ins = B * T * (H + 2 * HK) * D              # q, k, v
    g = 4 * (B * T * H if case["g"] == "token" else H)
    if case["kind"] == "step":
        return {"bytes": es * (ins + B * H * D) + g + 4 * B + 8 * B * H * D * D, "flops": 5 * B * H * D * D}
    s = 4 * (len(_lens(case)) or B) * H * D * D if case["state"] or not train else 0
    nbytes, flops = es * (ins + B * T * H * D) + g + s * (2 if case["state"] else 1), 4 * B * T * H * D * D
    if train:       # do in; the gradients of q, k, v and g out, with a state also that of the last one in and of the first one out
        nbytes += es * (B * T * H * D + ins) + g + (2 * s if case["state"] else 0)
        flops *= 3
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------
# the same results in 64 bits, from the definitions: token after token
# ---------------------------------------------------------------------------
def _exact_rotary(case, seed):
    x = _inputs(case, seed)
    T, D = case["T"], case["D"]
    at = torch.arange(T, device=DEVICE, dtype=torch.float64)
    turns, lo = torch.zeros(T, D, dtype=torch.complex128, device=DEVICE), 0
    for a, s in enumerate(int(n) for n in case["sections"].split(",")):
        if case["grid"]:
            h, w = (int(n) for n in case["grid"].split(","))
            n = at.long() + case["start"]
            row = torch.div(n, w, rounding_mode="floor")
            p = (torch.div(row, h, rounding_mode="floor"), row.remainder(h), n.remainder(w))[a].double()
        else:
            p = x["positions"][a].double()
        for i in range(s // 2):
            turns[:, lo + i] = torch.polar(torch.ones_like(at), p * math.pow(BASE, -2 * i / s))
        lo += s

    def turned(t, back):
        z, y = t.double(), t.double().clone()
        lo = 0
        for s in (int(n) for n in case["sections"].split(",")):
            for i in range(s // 2):
                a, b = (lo + i, lo + s // 2 + i) if case["pairs"] == "halves" else (lo + 2 * i, lo + 2 * i + 1)
                e = turns[:, lo + i, None]
                c = torch.complex(z[..., a], z[..., b]) * (e.conj() if back else e)
                y[..., a], y[..., b] = c.real, c.imag
            lo += s
        return y
    out = [turned(x["q"], False), turned(x["k"], False)]
    return out + [turned(x["dq"], True), turned(x["dk"], True)] if case["train"] else out


def _exact_decay(case, seed):
    x = _inputs(case, seed)
    B, T, H, D, train = case["B"], case["T"], case["H"], case["D"], case["train"]
    if train and B * T * H * D * D * 8 > 6e10:
        return None
    wide = lambda t: t.double().repeat_interleave(H // t.shape[-2], -2)  # noqa: E731
    q, k, v = wide(x["q"]), wide(x["k"]), wide(x["v"])
    f = torch.exp(x["g"].double()).expand(B, T, H)[..., None, None]
    o, rows = torch.zeros(B, T, H, D, dtype=torch.float64, device=DEVICE), _lens(case)
    spans, at = [], 0
    for i, n in enumerate(rows or [T]):         # (first token, behind the last, its states)
        spans.append((at, at + n, slice(i, i + 1) if rows else slice(0, B)))
        at += n
    zero = torch.zeros(len(rows) or B, H, D, D, dtype=torch.float64, device=DEVICE)
    S = zero.clone() if x["s0"] is None else x["s0"].double()
    kept = torch.zeros(T if train else 0, B, H, D, D, dtype=torch.float64, device=DEVICE)
    for lo, hi, own_rows in spans:
        s = S[own_rows]
        for t in range(lo, hi):
            s = f[:, t] * s
            if train:
                kept[t] = s                     # what the decay let through
            s = s + v[:, t, :, :, None] * k[:, t, :, None, :]
            o[:, t] = torch.matmul(s, q[:, t, :, :, None])[..., 0]
        S[own_rows] = s
    out = [o, S] if case["state"] or not train else [o]
    if not train:
        return out
    do = x["do"].double()
    dq, dk, dv = (torch.zeros_like(o) for _ in range(3))
    dg = torch.zeros(B, T, H, dtype=torch.float64, device=DEVICE)
    dS = zero if x["ds"] is None else x["ds"].double()
    for lo, hi, own_rows in spans:
        d = dS[own_rows]
        for t in range(hi - 1, lo - 1, -1):
            s = kept[t] + v[:, t, :, :, None] * k[:, t, :, None, :]
            dq[:, t] = torch.matmul(s.transpose(-1, -2), do[:, t, :, :, None])[..., 0]
            d = d + do[:, t, :, :, None] * q[:, t, :, None, :]
            dv[:, t] = torch.matmul(d, k[:, t, :, :, None])[..., 0]
            dk[:, t] = torch.matmul(d.transpose(-1, -2), v[:, t, :, :, None])[..., 0]
            dg[:, t] = (d * kept[t]).sum((-1, -2))
            d = f[:, t] * d
        dS[own_rows] = d
    heads = lambda t: t.unflatten(2, (case["HK"], -1)).sum(3)  # noqa: E731
    out += [dq, heads(dk), heads(dv), dg if case["g"] == "token" else dg.sum((0, 1))]
    return [*out, dS] if x["s0"] is not None else out


def _exact_step(case, seed):
    x = _inputs(case, seed)
    H, s = case["H"], x["s"].double()
    o = torch.zeros(case["B"], H, case["D"], dtype=torch.float64, device=DEVICE)
    for h in range(H):
        q, k, v = (x[n][:, h * x[n].shape[1] // H].double() for n in ("q", "k", "v"))
        f = torch.exp((x["g"][:, h] if case["g"] == "token" else x["g"][h]).double())
        new = s[x["slots"].long(), h] * f.reshape(-1, 1, 1) + v[:, :, None] * k[:, None, :]
        s[x["slots"].long(), h] = new
        o[:, h] = (new * q[:, None, :]).sum(-1)
    return [o, s]


def exact(case, seed):
    with torch.no_grad():
        return {"rotary": _exact_rotary, "decay": _exact_decay, "step": _exact_step}[case["kind"]](case, seed)
