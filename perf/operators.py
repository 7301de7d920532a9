"""The work of a training step around the recurrence layer, as measurable cases.

* ``linear``: ``linear_act``, one linear map with its bias, activation and
  residual: y = act(x W^T + b) + r;
* ``mlp``: ``mlp``, a block's two maps: y = act(x W1^T + b1) W2^T + b2 + r;
* ``adamw``: ``FusedAdamW.step``, the clip by the gradients' global norm and the
  AdamW update over all of a model's tensors, with moments held in 32 bits or
  in 8 (blocks of 256).

A case is a dict of plain values.  ``linear`` and ``mlp``: ``M`` rows, widths ``K``
-> ``N`` (``mlp``: K -> N -> K), ``dtype``, ``act``, ``bias``, ``res`` (a residual),
``train`` (the gradients too).  ``adamw``: a model of ``depth`` blocks of ``width``,
the parameters' ``dtype``, the moments' ``states``, ``master`` (fp32 copies of
bf16 weights) and ``clip`` (the largest norm; 0 leaves the gradients as they are).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
DEVICE = "cuda"
LR, B1, B2, EPS, WD = 3e-4, 0.9, 0.95, 1e-8, 0.05      # the trainer's AdamW
BLOCK = 256                                            # elements that share a scale of the 8-bit moments


def _linear(name, M, K, N, dtype="bf16", act="none", bias=True, res=False, train=False, kind="linear"):
    c = dict(kind=kind, M=M, K=K, N=N, dtype=dtype, act=act, bias=bias, res=res, train=train)
    return dict(name=name, **c) if name else c


def _mlp(name, M, K, N, dtype="bf16", act="gelu", res=True, train=False):
    return _linear(name, M, K, N, dtype, act, True, res, train, "mlp")


def _adamw(name, width, depth, dtype="bf16", states="fp32", master=False, clip=1.0):
    c = dict(kind="adamw", width=width, depth=depth, dtype=dtype, states=states, master=master, clip=clip)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # the class scores of one clip: 174 classes from one row of the default width, where latency counts
        _linear("linear-scores", 1, 384, 174),
        # streaming inference: the next tubelet's 196 tokens through a block's first map
        _linear("linear-stream", 196, 384, 1536, act="gelu"),
        # odd sizes in training, every input with a gradient: none of them a multiple of eight
        _linear("linear-odd-train", 1571, 772, 395, act="silu", res=True, train=True),
        # the largest product: a wide model's first map over a long batch
        _linear("linear-wide", 16384, 2048, 8192, act="gelu"),
        # classifying 8 clips: the MLP of a block of the default classifier (3136 tokens a clip)
        _mlp("mlp-classify", 25088, 384, 1536),
        # the same in training
        _mlp("mlp-train", 25088, 384, 1536, train=True),
        # training in fp32 (the parity mode), 2 clips
        _mlp("mlp-train-fp32", 6272, 384, 1536, "fp32", train=True),
        # fine-tuning one small block, fp32 throughout: launches and latency
        _adamw("adamw-block", 128, 1, "fp32"),
        # the default classifier's 16 blocks in bf16 with fp32 master weights
        _adamw("adamw-default", 384, 16, master=True),
        # a large model, 300 million parameters, fp32 moments
        _adamw("adamw-large", 1024, 24),
        # the default classifier with 8-bit moments
        _adamw("adamw8-default", 384, 16, states="int8"),
        # the large model with 8-bit moments
        _adamw("adamw8-large", 1024, 24, states="int8"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width: a multiple of 64 or of 8 in most models, any number in some."""
    n = _log_int(rng, lo, hi)
    step = rng.choice([64, 64, 8, 1])
    return max(step, n // step * step)


def draw(rng):
    kind = rng.choice(["linear", "linear", "mlp", "adamw", "adamw"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    if kind == "linear":
        M, K, N = _log_int(rng, 1, 25088), _width(rng, 32, 4096), _width(rng, 8, 4096)
        train = rng.random() < 0.5
        while M * K * N * (3 if train else 1) > 1.2e11:
            M //= 2
        return _linear(None, M, K, N, dtype, rng.choice(["none", "gelu", "silu"]), rng.random() < 0.8,
                       rng.random() < 0.5, train)
    if kind == "mlp":
        K = _width(rng, 64, 1024)
        M, N = _log_int(rng, 1, 25088), K * rng.choice([2, 3, 4])
        train = rng.random() < 0.6
        while 2 * M * K * N * (3 if train else 1) > 1.2e11:
            M //= 2
        return _mlp(None, M, K, N, dtype, rng.choice(["gelu", "gelu", "silu"]), rng.random() < 0.7, train)
    width, depth = 64 * rng.randint(1, 14), rng.randint(1, 24)
    states = rng.choice(["fp32", "int8"])
    return _adamw(None, width, depth, dtype, states, dtype == "bf16" and rng.random() < 0.5, rng.choice([0.0, 1.0, 1.0]))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE)


def _map_inputs(case, seed):
    """Operands by name, None where the case has none: x as a LayerNorm leaves it,
    weights at their initial spread."""
    M, K, N = case["M"], case["K"], case["N"]
    dt, gen = DTYPES[case["dtype"]], _gen(seed)
    out = N if case["kind"] == "linear" else K
    x = {"x": _randn(gen, M, K).to(dt)}
    x["w1"] = (_randn(gen, N, K) * K ** -0.5).to(dt)
    x["b1"] = (0.1 * _randn(gen, N)).to(dt) if case["bias"] else None
    if case["kind"] == "mlp":
        x["w2"] = (_randn(gen, K, N) * N ** -0.5).to(dt)
        x["b2"] = (0.1 * _randn(gen, K)).to(dt)
    x["res"] = _randn(gen, M, out).to(dt) if case["res"] else None
    x["dy"] = _randn(gen, M, out).to(dt) if case["train"] else None
    return x


def _shapes(width, depth):
    """The parameters of ``depth`` blocks of a recurrence layer and an MLP, and of
    a classifier of 174 classes."""
    d, h, r = width, max(1, width // 64), 64
    block = [(d,), (d,), (d, d), (d, d), (d, d), (r, d), (d, r), (h,), (d,), (h, d), (d, 4, 1), (d,), (d, 4, 1), (d,),
             (d, 4, 1), (d,), (r, d), (d, r), (d,), (r,), (d, d), (d,), (d,), (4 * d, d), (4 * d,), (d, 4 * d), (d,)]
    return block * depth + [(d,), (d,), (174, d), (174,)]


def _layout(width, depth):
    """(shape, first element, elements) of each tensor in one flat buffer where each
    begins on a multiple of BLOCK, and the buffer's length."""
    at, rows = 0, []
    for s in _shapes(width, depth):
        n = math.prod(s)
        rows.append((s, at, n))
        at += -(-n // BLOCK) * BLOCK
    return rows, at


def _adamw_inputs(case, seed):
    """Flat buffers: weights p, gradients g, moments (codes and scales in 8 bits), fp32
    masters.  What lies between two tensors is zero and stays so."""
    rows, total = _layout(case["width"], case["depth"])
    dt, gen = DTYPES[case["dtype"]], _gen(seed)
    ends = torch.tensor([a + n for _, a, n in rows], device=DEVICE)
    starts = torch.tensor([a for _, a, _ in rows], device=DEVICE)
    at = torch.arange(total, device=DEVICE)
    used = at < ends[torch.searchsorted(starts, at, right=True) - 1]
    x = {}
    p = 0.02 * _randn(gen, total) * used
    x["p"] = p.to(dt)
    x["g"] = (1e-3 * _randn(gen, total) * used).to(dt)
    x["master"] = p if case["master"] else None
    m, v = 1e-4 * _randn(gen, total) * used, (1e-4 * _randn(gen, total) * used).square()
    if case["states"] == "fp32":
        x["m"], x["v"] = m, v
    else:
        x["m"], x["m_scale"] = _encode_m(m)
        x["v"], x["v_scale"] = _encode_v(v.sqrt())
    return x


def prepare(case, seed):
    if case["kind"] != "adamw":
        x = _map_inputs(case, seed)
        leaves = [x[n] for n in ("x", "w1", "b1", "w2", "b2", "res") if x.get(n) is not None]
        if case["train"]:
            for t in leaves:
                t.requires_grad_(True)
        return dict(case=case, x=x, leaves=leaves)
    x = _adamw_inputs(case, seed)
    params = []
    for s, a, n in _layout(case["width"], case["depth"])[0]:
        p = torch.nn.Parameter(x["p"][a:a + n].view(s))
        p.grad = x["g"][a:a + n].view(s)
        params.append(p)
    return dict(case=case, x=x, params=params)


# ---------------------------------------------------------------------------
# the 8-bit moments: blocks of BLOCK elements
# ---------------------------------------------------------------------------
def _encode_m(m):
    """m -> (codes in [-127, 127], scales): m = s (k / 127) |k / 127|, s the block's largest |m|."""
    b = m.view(-1, BLOCK)
    s = b.abs().amax(1, keepdim=True)
    k = torch.round(127 * torch.sqrt(b.abs() / torch.where(s > 0, s, 1))) * torch.sign(b)
    return k.to(torch.int8).view(-1), s.view(-1)


def _encode_v(r):
    """sqrt(v) -> (codes in [0, 255], scales): sqrt(v) = s (k / 255)^2, s the block's largest
    sqrt(v); what is above zero keeps a code above zero."""
    b = r.view(-1, BLOCK)
    s = b.amax(1, keepdim=True)
    k = torch.maximum(torch.round(255 * torch.sqrt(b / torch.where(s > 0, s, 1))), (b > 0).to(b.dtype))
    return k.to(torch.uint8).view(-1), s.view(-1)


def _decode_m(k, s, dt=torch.float32):
    f = k.to(dt).view(-1, BLOCK) / 127
    return (s.to(dt).view(-1, 1) * f * f.abs()).view(-1)


def _decode_sqrt_v(k, s, dt=torch.float32):
    f = k.to(dt).view(-1, BLOCK) / 255
    return (s.to(dt).view(-1, 1) * f * f).view(-1)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _act(z, act):
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z * torch.sigmoid(z) if act == "silu" else z


def _act_grad(z, act):
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * math.sqrt(0.5 / math.pi)
    s = torch.sigmoid(z)
    return s * (1 + z * (1 - s)) if act == "silu" else torch.ones_like(z)


def _plain_map(case, x):
    """The formulas in 32 bits, each result rounded once."""
    dt, act, mlp = DTYPES[case["dtype"]], case["act"], case["kind"] == "mlp"
    f = {n: None if t is None else t.detach().float() for n, t in x.items()}
    z = f["x"] @ f["w1"].t()
    if f["b1"] is not None:
        z = z + f["b1"]
    h = _act(z, act)
    y = h @ f["w2"].t() + f["b2"] if mlp else h
    if f["res"] is not None:
        y = y + f["res"]
    if not case["train"]:
        return [y.to(dt)]
    dy = f["dy"]
    dh = dy @ f["w2"] if mlp else dy
    dz = dh * _act_grad(z, act)
    grads = [dz @ f["w1"], dz.t() @ f["x"]]
    if f["b1"] is not None:
        grads.append(dz.sum(0))
    if mlp:
        grads += [dy.t() @ h, dy.sum(0)]
    if f["res"] is not None:
        grads.append(dy)
    return [t.to(dt) for t in [y, *grads]]


def _own_map(state):
    from mlx_vit_amd import linear_act, mlp
    case, x = state["case"], state["x"]
    act = None if case["act"] == "none" else case["act"]
    if case["kind"] == "mlp":
        y = mlp(x["x"], x["w1"], x["b1"], x["w2"], x["b2"], x["res"], act)
    else:
        y = linear_act(x["x"], x["w1"], x["b1"], x["res"], act)
    return [y, *torch.autograd.grad(y, state["leaves"], x["dy"])] if case["train"] else [y]


def _plain_adamw(case, x):
    """The update over the flat buffers, in place; the norm's sum in 64 bits."""
    out = []
    g = x["g"].float()
    if case["clip"]:
        norm = g.double().square().sum().sqrt()
        g = g * torch.clamp(case["clip"] / (norm + 1e-6), max=1.0).float()
        out.append(norm.float())
    small = case["states"] == "int8"
    m = _decode_m(x["m"], x["m_scale"]) if small else x["m"]
    v = _decode_sqrt_v(x["v"], x["v_scale"]).square() if small else x["v"]
    m = B1 * m + (1 - B1) * g
    v = B2 * v + (1 - B2) * g * g
    r = v.sqrt()
    p = x["p"].float() if x["master"] is None else x["master"]
    p = p * (1 - LR * WD) - LR * m / (r + EPS)
    x["p"].copy_(p)
    out.insert(0, x["p"])
    if x["master"] is not None:
        x["master"].copy_(p)
        out.append(x["master"])
    if not small:
        x["m"].copy_(m)
        x["v"].copy_(v)
        return [*out, x["m"], x["v"]]
    for n, (k, s) in (("m", _encode_m(m)), ("v", _encode_v(r))):
        x[n].copy_(k)
        x[n + "_scale"].copy_(s)
    # what the codes stand for
    return [*out, _decode_m(x["m"], x["m_scale"]).bfloat16(),
            _decode_sqrt_v(x["v"], x["v_scale"]).square().bfloat16()]


def _own_adamw(state):
    from mlx_vit_amd import FusedAdamW
    case, x = state["case"], state["x"]
    if "opt" not in state:      # a program makes its optimizer once, here over moments as a checkpoint gives them
        names = ("m", "v", "m_scale", "v_scale", "master")
        state["opt"] = FusedAdamW(state["params"], lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD,
                                  states=case["states"], master_weights=case["master"],
                                  state={n: x[n] for n in names if x.get(n) is not None})
    opt = state["opt"]
    norm = opt.step(max_norm=case["clip"] or None)
    out = [x["p"]] if norm is None else [x["p"], norm]
    if case["master"]:
        out.append(x["master"])
    return [*out, x["m"], x["v"]] if case["states"] == "fp32" else [*out, *opt.moments(torch.bfloat16)]


def run(state):
    if own:
        return _own_adamw(state) if state["case"]["kind"] == "adamw" else _own_map(state)
    with torch.no_grad():
        return (_plain_adamw if state["case"]["kind"] == "adamw" else _plain_map)(state["case"], state["x"])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["kind"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(case["width"], case["depth"]))
        es = 2 if case["dtype"] == "bf16" else 4
        small = case["states"] == "int8"
        # g read (the norm's and the update's share where it fits no cache: once), p read and written
        # (with a master only written), the moments read and written and, in 8 bits, the values they stand for
        per = es + (es + 8 if case["master"] else 2 * es) + (4 + 16 / BLOCK + 4 if small else 16)
        return {"bytes": n * per, "flops": 20 * n}
    M, K, N, mlp, train = case["M"], case["K"], case["N"], case["kind"] == "mlp", case["train"]
    es = 2 if case["dtype"] == "bf16" else 4
    out = K if mlp else N
    weights = N * K + (N if case["bias"] else 0) + (N * K + K if mlp else 0)
    ins = M * K + weights + (M * out if case["res"] else 0)
    elems, flops = ins + M * out, 2 * M * N * K * (2 if mlp else 1)
    if train:
        elems += M * out + ins              # dy in, a gradient for every input out
        flops *= 3
    return {"bytes": es * elems, "flops": flops}


# ---------------------------------------------------------------------------
# the same results in 64 bits, from the definitions: autograd through the
# formula for the maps, tensor by tensor for the update
# ---------------------------------------------------------------------------
def _exact_map(case, seed):
    t = {n: None if v is None else v.double() for n, v in _map_inputs(case, seed).items()}
    dy = t.pop("dy")
    leaves = [t[n].requires_grad_(case["train"]) for n in ("x", "w1", "b1", "w2", "b2", "res") if t.get(n) is not None]

    def phi(z):
        if case["act"] == "gelu":
            return z * torch.special.ndtr(z)
        return z / (1 + torch.exp(-z)) if case["act"] == "silu" else z

    with torch.set_grad_enabled(case["train"]):
        y = t["x"].matmul(t["w1"].transpose(0, 1))
        y = phi(y if t["b1"] is None else y + t["b1"])
        if case["kind"] == "mlp":
            y = y.matmul(t["w2"].transpose(0, 1)) + t["b2"]
        y = y if t["res"] is None else y + t["res"]
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)] if case["train"] else [y]


def _exact_adamw(case, seed):
    x = _adamw_inputs(case, seed)
    rows, total = _layout(case["width"], case["depth"])
    small, master = case["states"] == "int8", case["master"]
    norm = math.sqrt(sum(float(x["g"][a:a + n].double().pow(2).sum()) for _, a, n in rows))
    scale = min(case["clip"] / (norm + 1e-6), 1.0) if case["clip"] else 1.0
    P, M, V = (torch.zeros(total, dtype=torch.float64, device=DEVICE) for _ in range(3))
    for _, a, n in rows:
        e = a + -(-n // BLOCK) * BLOCK      # to the end of the tensor's last block, which holds zeros
        g = x["g"][a:e].double() * scale
        if small:
            blocks = slice(a // BLOCK, e // BLOCK)
            m, v = x["m"][a:e].double() / 127, x["v"][a:e].double() / 255
            m = m.abs() * m * x["m_scale"][blocks].double().repeat_interleave(BLOCK)
            v = v.pow(4) * x["v_scale"][blocks].double().pow(2).repeat_interleave(BLOCK)
        else:
            m, v = x["m"][a:e].double(), x["v"][a:e].double()
        m = m + (1 - B1) * (g - m)
        v = v + (1 - B2) * (g.pow(2) - v)
        w = (x["master"] if master else x["p"])[a:e].double()
        P[a:e] = w - LR * (WD * w + m / (torch.sqrt(v) + EPS))
        if small:                           # the nearest code's value
            top = m.abs().view(-1, BLOCK).amax(1).repeat_interleave(BLOCK)
            k = torch.where(top > 0, (m.abs() / top).sqrt() * 127, 0).round()
            m = torch.sign(m) * top * (k / 127).pow(2)
            top = v.view(-1, BLOCK).amax(1).repeat_interleave(BLOCK)
            k = torch.where(top > 0, (v / top).pow(0.25) * 255, 0).round().clamp(min=1) * (v > 0)
            v = top * (k / 255).pow(4)
        M[a:e], V[a:e] = m, v
    out = [P]
    if case["clip"]:
        out.append(torch.tensor(norm, dtype=torch.float64))
    return [*out, *([P] if master else []), M, V]


def exact(case, seed):
    return _exact_adamw(case, seed) if case["kind"] == "adamw" else _exact_map(case, seed)
