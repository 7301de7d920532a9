"""FusedAdamW against the update in 64 bits, tensor by tensor: odd sizes, mixed
dtypes, unaligned tensors, more tensors than a launch takes, 8-bit moments,
master weights, the clip, missing gradients, graph replays, and a training step
of a small model through it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BLOCK = 256
SIZES = [(1,), (7,), (255,), (256,), (257,), (12, 64), (4095,), (4097,), (3, 5, 7), (130, 129), (40000,)]


def _params(sizes, dtypes, seed=0, scale=0.05):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter((scale * torch.randn(*s, generator=g)).to(d).to(DEV)) for s, d in zip(sizes, dtypes)]


def _grads(params, seed, scale=1e-2):
    g = torch.Generator().manual_seed(seed)
    for p in params:
        p.grad = (scale * torch.randn(p.shape, generator=g)).to(p.dtype).to(DEV)


class Plain:
    """The update in 64 bits from given moments and weights."""

    def __init__(self, lr, betas, eps, wd, correct=False):
        self.h = lr, betas, eps, wd, correct

    def __call__(self, w, g, m, v, scale, step):
        lr, (b1, b2), eps, wd, correct = self.h
        g = g * scale
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g * g
        c1, c2 = (1 / (1 - b1 ** step), 1 / (1 - b2 ** step)) if correct else (1.0, 1.0)
        u = c1 * m / ((c2 * v).sqrt() + eps)
        return w * (1 - lr * wd) - lr * u, m, v, u


def _clip(params, max_norm):
    n = math.sqrt(sum(p.grad.double().square().sum().item() for p in params if p.grad is not None))
    return n, 1.0 if max_norm is None else min(max_norm / (n + 1e-6), 1.0)


def _check_step(opt, before, plain, max_norm, params):
    """``before``: weights (or masters) and moment values before the step, fp64."""
    norm, scale = _clip(params, max_norm)
    got = opt.step(max_norm=max_norm)
    if max_norm is None:
        assert got is None
    else:
        # fp32 sums of at most 64 squares a lane, then a tree: below 100 * 2^-24
        assert got.dtype == torch.float32 and abs(got.item() - norm) <= 1e-5 * norm
    m_all, v_all = opt.moments()
    masters = opt.views(opt.state["master"]) if "master" in opt.state else [None] * len(params)
    for p, (w, m, v), mo, vo, ma, o in zip(params, before, opt.views(m_all), opt.views(v_all), masters, opt.offsets):
        if p.grad is None:
            assert torch.equal(p.detach().double(), w) and torch.equal(mo.double(), m) and torch.equal(vo.double(), v)
            continue
        W, M, V, u = plain(w, p.grad.double(), m, v, scale, opt.steps)
        # fp32 arithmetic: a few roundings each (16 * 2^-24), m's of its two terms, which may cancel
        # (the clip factor itself is within 1e-5 where there is one)
        rel = 2.0 ** -20 + (1e-5 if max_norm is not None else 0.0)
        terms = 0.9 * m.abs() + 0.1 * scale * p.grad.double().abs()
        lr, (b1, b2), eps, _, correct = plain.h
        c1, c2 = (1 / (1 - b1 ** opt.steps), 1 / (1 - b2 ** opt.steps)) if correct else (1.0, 1.0)
        tol_m = rel * terms
        tol_u = 4 * rel * u.abs() + c1 * tol_m / ((c2 * V).sqrt() + eps)
        tol_w = 2.0 ** -22 * W.abs() + lr * tol_u
        if ma is not None:
            assert ((ma.double() - W).abs() <= tol_w).all()
            assert torch.equal(p.detach(), ma.to(p.dtype))
        else:
            half = torch.finfo(p.dtype).eps / 2
            assert ((p.detach().double() - W).abs() <= tol_w + half * (W.abs() + tol_w)).all()
        if opt.states == "fp32":
            assert ((mo.double() - M).abs() <= tol_m).all()
            assert ((vo.double() - V).abs() <= 4 * rel * V + 2.0 ** -126).all()
        else:
            _check_codes(opt, o, p.numel(), M.reshape(-1), V.reshape(-1), rel)


def _blocks(x):
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def _check_codes(opt, o, n, M, V, rel):
    """Scales are the blocks' largest values; a code is the nearest of the companded value,
    up to rel of it; a v above zero has a code above zero; what lies past n is zero."""
    end = o + -(-n // BLOCK) * BLOCK
    blk = slice(o // BLOCK, end // BLOCK)
    s, t = opt.state["m_scale"][blk].double().unsqueeze(1), opt.state["v_scale"][blk].double().unsqueeze(1)
    m, r = _blocks(M), _blocks(V.sqrt())
    assert ((s.squeeze(1) - m.abs().amax(1)).abs() <= 8 * rel * s.squeeze(1) + 1e-30).all()
    assert ((t.squeeze(1) - r.amax(1)).abs() <= 8 * rel * t.squeeze(1) + 1e-30).all()
    km, kv = opt.state["m"][o:end].view(-1, BLOCK).double(), opt.state["v"][o:end].view(-1, BLOCK).double()
    x = 127 * torch.where(s > 0, m.abs() / torch.where(s > 0, s, 1), 0).sqrt() * m.sign()
    y = 255 * torch.where(t > 0, r / torch.where(t > 0, t, 1), 0).sqrt()
    # m's terms may cancel, so its companded value is off by more near zero: sqrt(rel) codes of 127
    assert ((km - x).abs() <= 0.5 + 127 * 4 * rel ** 0.5 * (x.abs() < 4) + 127 * 8 * rel).all()
    assert ((kv - y).abs() <= torch.where((r > 0) & (y < 0.5), 1.0, 0.5 + 255 * 8 * rel)).all()
    assert ((kv >= 1) | (r == 0)).all()
    pad = torch.arange(end - o, device=DEV).view(-1, BLOCK) >= n
    assert not km[pad].any() and not kv[pad].any()


def _before(opt, params):
    m, v = opt.moments()
    ws = opt.views(opt.state["master"]) if "master" in opt.state else [p.detach() for p in params]
    return [(w.double().clone(), a.double().clone(), b.double().clone())
            for w, a, b in zip(ws, opt.views(m), opt.views(v))]


@pytest.mark.parametrize("correct", [False, True], ids=["plain", "corrected"])
@pytest.mark.parametrize("states", ["fp32", "int8"])
@pytest.mark.parametrize("kind", ["bf16", "fp32", "mixed", "master"])
def test_steps(kind, states, correct):
    from mlx_vit_amd import FusedAdamW
    dts = {"bf16": [torch.bfloat16], "fp32": [torch.float32], "mixed": [torch.bfloat16, torch.float32],
           "master": [torch.bfloat16, torch.bfloat16, torch.float32]}[kind]
    params = _params(SIZES, [dts[i % len(dts)] for i in range(len(SIZES))])
    h = dict(lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.05)
    opt = FusedAdamW(params, states=states, master_weights=kind == "master", bias_correction=correct, **h)
    plain = Plain(h["lr"], h["betas"], h["eps"], h["weight_decay"], correct)
    for k, (max_norm, scale) in enumerate([(None, 1e-2), (1.0, 1e-2), (0.5, 1e-1), (1e6, 1e-4)]):
        print(kind, states, correct, "step", k, flush=True)
        _grads(params, 10 + k, scale)
        kept = [p.grad.clone() for p in params]
        _check_step(opt, _before(opt, params), plain, max_norm, params)
        assert all(torch.equal(p.grad, g) for p, g in zip(params, kept))


def test_more_tensors_than_a_launch_takes():
    from mlx_vit_amd import FusedAdamW
    sizes = [(1 + 37 * i % 700,) for i in range(301)] + [(70000,)]
    params = _params(sizes, [torch.bfloat16 if i % 3 else torch.float32 for i in range(302)], seed=1)
    opt = FusedAdamW(params, lr=1e-2)
    for k in range(2):
        _grads(params, 20 + k)
        _check_step(opt, _before(opt, params), Plain(1e-2, (0.9, 0.95), 1e-8, 0.05), 1.0, params)


@pytest.mark.parametrize("states", ["fp32", "int8"])
def test_unaligned_tensors_and_gradients(states):
    """Weights and gradients that begin on any element, gradients of another stride,
    parameters without a gradient; what surrounds the weights stays."""
    from mlx_vit_amd import FusedAdamW
    for dt in (torch.bfloat16, torch.float32):
        buf = (0.05 * torch.randn(5000, device=DEV)).to(dt)
        keep = buf.clone()
        spans = [(1, 300), (302, 1030), (1333, 3), (1337, 2049)]
        params = [torch.nn.Parameter(buf[a:a + n]) for a, n in spans] + _params([(40, 30), (17,)], [dt, dt], seed=3)
        opt = FusedAdamW(params, lr=1e-2, states=states)
        gbuf = (1e-2 * torch.randn(6000, device=DEV)).to(dt)
        for k in range(2):
            for i, (a, n) in enumerate(spans):
                params[i].grad = gbuf[a + 2 + k:a + 2 + k + n]
            params[4].grad = (1e-2 * torch.randn(30, 40, device=DEV)).to(dt).t()
            params[5].grad = None
            _check_step(opt, _before(opt, params), Plain(1e-2, (0.9, 0.95), 1e-8, 0.05), 0.2, params)
        inside = torch.zeros(5000, dtype=torch.bool, device=DEV)
        for a, n in spans:
            inside[a:a + n] = True
        assert torch.equal(buf[~inside], keep[~inside]) and not torch.equal(buf[inside], keep[inside])


def test_nothing_to_do():
    from mlx_vit_amd import FusedAdamW
    params = _params([(10,), (0,)], [torch.float32] * 2)
    opt = FusedAdamW(params)
    w = params[0].detach().clone()
    assert opt.step() is None and opt.step(max_norm=1.0).item() == 0.0
    assert torch.equal(params[0], w)
    params[1].grad = torch.zeros(0, device=DEV)
    opt.step(max_norm=1.0)
    params[0].grad = torch.zeros(10, device=DEV)       # a block of zeros: no division by its scale
    for states in ("fp32", "int8"):
        opt = FusedAdamW(params, states=states, lr=0.1, weight_decay=0.5)
        w = params[0].detach().double()
        opt.step(max_norm=1.0)
        assert ((params[0].double() - w * 0.95).abs() <= 2.0 ** -22 * w.abs()).all()
        assert not any(t.any() for t in opt.moments())


def test_non_finite_gradients():
    """They reach the weights they belong to, through a clip all; an 8-bit block with one is NaN,
    its neighbours are not."""
    from mlx_vit_amd import FusedAdamW
    for states in ("fp32", "int8"):
        for bad in (float("nan"), float("inf")):
            (p,) = _params([(1000,)], [torch.float32])
            _grads([p], 5)
            p.grad[300] = bad
            opt = FusedAdamW([p], states=states)
            opt.step()
            assert not p[300].isfinite() and p.isfinite().sum() == 999
            m, v = opt.moments()
            assert not m[300].isfinite() and not v[300].isfinite()
            if states == "int8":
                assert not m[256:512].isfinite().any() and m[:256].isfinite().all() and m[512:].isfinite().all()
            norm = opt.step(max_norm=1.0)
            assert not norm.isfinite() and not p[300].isfinite()
            if bad != bad:
                assert p.isnan().all()


def test_tiny_and_large_gradients_in_8_bits():
    """Ten decades of gradients in one block: small roots of v round to their code of at
    least one, and no update exceeds what 64 bits give from the same moments."""
    from mlx_vit_amd import FusedAdamW
    (p,) = _params([(512,)], [torch.float32])
    opt = FusedAdamW([p], lr=1e-2, states="int8")
    plain = Plain(1e-2, (0.9, 0.95), 1e-8, 0.05)
    for k in range(4):
        g = torch.randn(512, generator=torch.Generator().manual_seed(k)) * 10.0 ** torch.linspace(-9, 1, 512)
        p.grad = g.to(DEV)
        _check_step(opt, _before(opt, [p]), plain, None, [p])
    p.grad = torch.full((512,), 1e-25, device=DEV)      # their squares are not normal numbers, or zero
    opt = FusedAdamW([p], states="int8")
    opt.step()
    assert p.isfinite().all() and all(t.isfinite().all() for t in opt.moments())


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_codes_are_those_of_fp32_arithmetic(dtype):
    """Codes and scales, over steps with the clip at work, equal those of torch's fp32
    operations in the same order, each rounded by itself: two programs that take the
    same steps keep the same moments."""
    from mlx_vit_amd import FusedAdamW
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    n, b1, b2 = 3_000_064, 0.9, 0.95
    (p,) = _params([(n,)], [dt], seed=11)
    opt = FusedAdamW([p], betas=(b1, b2), states="int8")
    k, s, q, t = (opt.state[i].clone() for i in ("m", "m_scale", "v", "v_scale"))
    rows = lambda x: torch.nn.functional.pad(x, (0, -n % BLOCK)).view(-1, BLOCK)  # noqa: E731
    for step in range(4):
        g = torch.Generator(device=DEV).manual_seed(step)
        p.grad = (torch.randn(n, generator=g, device=DEV) * torch.rand(n, generator=g, device=DEV) ** 4).to(dt)
        norm = p.grad.double().square().sum().sqrt()
        c = torch.clamp(0.5 / (norm + 1e-6), max=1.0).float()
        assert opt.step(max_norm=0.5).item() == norm.float().item()
        x = rows(p.grad.float() * c)
        f = k.float().view(-1, BLOCK) / 127
        m = b1 * (s.view(-1, 1) * f * f.abs()) + (1 - b1) * x
        f = q.float().view(-1, BLOCK) / 255
        v = b2 * (t.view(-1, 1) * f * f).square() + (1 - b2) * x * x
        r = v.sqrt()
        s, t = m.abs().amax(1, keepdim=True), r.amax(1, keepdim=True)
        k = (torch.round(127 * torch.sqrt(m.abs() / s)) * m.sign()).to(torch.int8).view(-1)
        q = torch.maximum(torch.round(255 * torch.sqrt(r / t)), (r > 0).float()).to(torch.uint8).view(-1)
        for name, want in (("m_scale", s.view(-1)), ("v_scale", t.view(-1)), ("m", k), ("v", q)):
            assert torch.equal(opt.state[name], want), (step, name, (opt.state[name] != want).sum().item())


@pytest.mark.parametrize("states", ["fp32", "int8"])
def test_state_is_carried(states):
    """The state of one optimizer, given or copied to another, continues it bit for bit."""
    from mlx_vit_amd import FusedAdamW
    a = _params(SIZES, [torch.bfloat16] * len(SIZES))
    opt = FusedAdamW(a, states=states, master_weights=True, bias_correction=True)
    for k in range(2):
        _grads(a, k)
        opt.step(1.0)
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    c = [torch.nn.Parameter(p.detach().clone()) for p in a]
    given = FusedAdamW(b, states=states, master_weights=True, bias_correction=True,
                       state={k: t.clone() for k, t in opt.state.items()})
    given.steps = opt.steps
    copied = FusedAdamW(c, states=states, master_weights=True, bias_correction=True)
    copied.load_state_dict(opt.state_dict())
    for ps, o in ((a, opt), (b, given), (c, copied)):
        _grads(ps, 9)
        o.step(1.0)
    for p, q, r in zip(a, b, c):
        assert torch.equal(p, q) and torch.equal(p, r)
    for k in opt.state:
        assert torch.equal(opt.state[k], given.state[k]) and torch.equal(opt.state[k], copied.state[k])


def test_master_weights_collect_small_updates():
    """Updates of a tenth of a bf16 half step: without masters no weight moves, with them all do."""
    from mlx_vit_amd import FusedAdamW
    for master in (False, True):
        p = torch.nn.Parameter(torch.ones(500, dtype=torch.bfloat16, device=DEV))
        opt = FusedAdamW([p], lr=2.0 ** -8 / 20, weight_decay=0.0, master_weights=master)
        for _ in range(60):
            p.grad = torch.ones_like(p)
            opt.step()
        assert bool((p == 1).all()) != master


def test_graph_replays_of_a_step():
    from mlx_vit_amd import FusedAdamW
    for states in ("fp32", "int8"):
        a, b = (_params(SIZES, [torch.bfloat16] * len(SIZES), seed=4) for _ in range(2))
        oa, ob = (FusedAdamW(ps, states=states, master_weights=True) for ps in (a, b))
        _grads(a, 1)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norm = oa.step(max_norm=0.3)
        for k in range(3):
            _grads(b, 30 + k)
            for p, q in zip(a, b):
                p.grad.copy_(q.grad)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(norm, ob.step(max_norm=0.3))
            assert all(torch.equal(p, q) for p, q in zip(a, b))
            assert all(torch.equal(oa.state[n], ob.state[n]) for n in oa.state)


def test_other_stream():
    from mlx_vit_amd import FusedAdamW
    a, b = (_params(SIZES, [torch.float32] * len(SIZES), seed=5) for _ in range(2))
    oa, ob = FusedAdamW(a), FusedAdamW(b)
    for ps in (a, b):
        _grads(ps, 2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        na = oa.step(1.0)
    s.synchronize()
    assert torch.equal(na, ob.step(1.0)) and all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("states", ["fp32", "int8"])
def test_optimizer_dropped_behind_a_step_on_another_stream(states):
    """Its memory is not given to others before the step has ended."""
    from mlx_vit_amd import FusedAdamW
    a, b = (_params(SIZES, [torch.float32] * len(SIZES), seed=12) for _ in range(2))
    for ps in (a, b):
        _grads(ps, 6)
    FusedAdamW(b, states=states).step(1.0)
    opt = FusedAdamW(a, states=states)
    sizes = [t.numel() * t.element_size() for t in (*opt.state.values(), opt._plan)]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)   # some milliseconds
        opt.step(1.0)
    del opt
    others = [torch.full((n,), 1, dtype=torch.uint8, device=DEV) for n in sizes for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and len(others) == 4 * len(sizes)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("states", ["fp32", "int8"])
def test_training_step_of_a_block(states, dtype):
    """The operators as they are used together: a block's MLP forward and backward, then the
    clipped update, against the same step in 64 bits from the gradients that it made."""
    from mlx_vit_amd import FusedAdamW, mlp
    import linear_reference as L
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    g = torch.Generator().manual_seed(0)
    x, dy = (torch.randn(150, 96, generator=g).to(dt).to(DEV) for _ in range(2))
    params = _params([(384, 96), (384,), (96, 384), (96,)], [dt] * 4, seed=6)
    opt = FusedAdamW(params, lr=1e-2, states=states, master_weights=dt == torch.bfloat16)
    for _ in range(3):
        want = L.mlp(x, *params, x, "gelu", dy)
        opt.zero_grad()
        y = mlp(x, *params, residual=x)
        y.backward(dy)
        L.check("y", y, want["y"])
        for p, n in zip(params, ("dw1", "db1", "dw2", "db2")):
            L.check(n, p.grad, want[n])
        _check_step(opt, _before(opt, params), Plain(1e-2, (0.9, 0.95), 1e-8, 0.05), 1.0, params)


@pytest.mark.parametrize("states", ["fp32", "int8"])
def test_train_step_of_a_classifier(states):
    """TrainStep with the fused MLPs and FusedAdamW: its first update is 64 bits' from the
    gradients of that step, every parameter with a gradient moves, the schedule sets the rate."""
    from mlx_vit_amd import model as M
    from mlx_vit_amd import train as TR
    torch.manual_seed(0)
    model = M.to_bf16(M.NoPEGDNClassifier(img_size=64, num_frames=10, encoder_dim=32, encoder_depth=1, encoder_heads=2,
                                          processor_dim=64, processor_depth=4, processor_heads=2, gdn_ratio=3,
                                          num_classes=7)).to(DEV)
    M.set_fused_mlp(model)
    step = TR.TrainStep(model, lr=1e-2, grad_clip=1.0, total_steps=10, warmup_steps=2, step_offset=1,
                        optimizer_states=states, master_weights=True)
    before = _before(step.opt, step.opt.params)
    g = torch.Generator().manual_seed(1)
    video = torch.randn(2, 10, 64, 64, 3, generator=g).to(torch.bfloat16).to(DEV)
    loss = step(video, torch.tensor([3, 5], device=DEV))
    assert loss.isfinite() and step.opt.lr == TR.cosine_warmup_lr(1, 10, 2, 1e-2)
    _, scale = _clip(step.opt.params, 1.0)
    plain = Plain(step.opt.lr, (0.9, 0.95), 1e-8, 0.05)
    for p, (w, m, v), ma in zip(step.opt.params, before, step.opt.views(step.opt.state["master"])):
        if p.grad is None:
            continue
        W, _, _, u = plain(w, p.grad.double(), m, v, scale, 1)
        # u = (1 - b1) g / (sqrt(1 - b2) |g| + eps): at most 0.45, within 1e-4 of it for the clip factor
        assert ((ma.double() - W).abs() <= 2.0 ** -20 * W.abs() + step.opt.lr * 1e-4).all()
        assert torch.equal(p.detach(), ma.to(p.dtype))


def test_moved_parameters():
    """Weights that were given new memory between two steps; one of another size is refused, as are
    parameters that share memory."""
    from mlx_vit_amd import FusedAdamW
    a, b = (_params(SIZES, [torch.bfloat16] * len(SIZES), seed=8) for _ in range(2))
    oa, ob = FusedAdamW(a), FusedAdamW(b)
    for k in range(2):
        for ps, o in ((a, oa), (b, ob)):
            _grads(ps, 40 + k)
            o.step(1.0)
        for p in a:
            p.data = p.data.clone()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    a[3].grad = None
    a[3].data = torch.zeros(5, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="make a new optimizer"):
        oa.step()
    buf = torch.zeros(300, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        FusedAdamW([torch.nn.Parameter(buf[:200]), torch.nn.Parameter(buf[100:])])
    with pytest.raises(ValueError, match="overlap"):
        FusedAdamW([b[0], b[0]])
    with pytest.raises(ValueError, match="contiguous"):
        FusedAdamW([torch.nn.Parameter(buf.view(30, 10).t())])
    with pytest.raises(ValueError, match="state"):
        FusedAdamW(b, state={"m": buf})
    with pytest.raises(ValueError, match="elements"):
        FusedAdamW(b, state={"m": buf, "v": buf})
    with pytest.raises(ValueError, match="buffers overlap"):
        FusedAdamW([torch.nn.Parameter(torch.zeros(256, device=DEV))], state={"m": buf[:256], "v": buf[:256]})


def test_parameters_changed_in_place_are_refused():
    """The same address, other elements: a part of the parameter, its transpose."""
    from mlx_vit_amd import FusedAdamW
    p = torch.nn.Parameter(torch.zeros(32, 16, device=DEV))
    whole = p.data
    opt = FusedAdamW([p])
    for other, match in ((whole[:8], "size or dtype"), (whole.t(), "make a new optimizer")):
        p.grad = None
        p.data = other
        p.grad = torch.ones_like(p)
        with pytest.raises(ValueError, match=match):
            opt.step()
    assert opt.steps == 0 and bool((whole == 0).all())
    p.grad = None
    p.data = whole
    p.grad = torch.ones_like(p)
    opt.step()
    assert bool((whole != 0).all())


def test_graph_of_a_step_before_parameters_moved():
    """A captured step goes on updating the memory that it was captured with."""
    from mlx_vit_amd import FusedAdamW
    a, b = (_params(SIZES, [torch.bfloat16] * len(SIZES), seed=9) for _ in range(2))
    oa, ob = FusedAdamW(a), FusedAdamW(b)
    for ps in (a, b):
        _grads(ps, 3)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        norm = oa.step(0.5)
    old = [p.data for p in a]
    grads = [p.grad for p in a]
    for p in a:
        p.grad = None
        p.data = p.data.clone()
    oa.step()      # the plan is made again; no gradients: nothing moves
    for k in range(3):
        junk = [torch.full((4096,), -1, dtype=torch.int64, device=DEV) for _ in range(8)]   # noqa: F841 (takes freed memory)
        g.replay()
        assert torch.equal(norm, ob.step(0.5))
        assert all(torch.equal(x, q) for x, q in zip(old, b)) and len(grads) == len(a)


@pytest.mark.parametrize("n", [(1 << 23) - 5, (1 << 23) + 5])
def test_norm_of_many_elements(n):
    """2048 partial sums of the norm and 2049: joined by the update itself, by a launch before it."""
    from mlx_vit_amd import FusedAdamW
    (p,) = params = _params([(n,)], [torch.bfloat16], seed=10)
    _grads(params, 4)
    opt = FusedAdamW(params, lr=1e-2)
    _check_step(opt, _before(opt, params), Plain(1e-2, (0.9, 0.95), 1e-8, 0.05), 1.0, params)
    exact = p.grad.double().square().sum().sqrt()
    assert torch.equal(opt.step(1.0), exact.float())


def test_autograd_sees_that_weights_changed():
    from mlx_vit_amd import FusedAdamW
    p = torch.nn.Parameter(torch.ones(16, device=DEV))
    x = torch.ones(16, device=DEV, requires_grad=True)
    opt = FusedAdamW([p])
    y = (x * p).sum()
    p.grad = torch.ones_like(p)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    q = torch.nn.Parameter(torch.ones(16, device=DEV))
    opt = FusedAdamW([p, q])
    y = (x * q).sum()
    opt.step()               # q has no gradient: it stays
    y.backward()
    assert torch.equal(x.grad, q.detach())


def test_a_kept_norm_keeps_little():
    from mlx_vit_amd import FusedAdamW
    params = _params([(1 << 21,)], [torch.bfloat16], seed=11)
    _grads(params, 5)
    assert FusedAdamW(params).step(1.0).untyped_storage().nbytes() <= 4096


@pytest.mark.parametrize("states", ["fp32", "int8"])
def test_offsets_past_32_bits(states):
    """A tensor of more than 2^31 elements and one behind it: what a small one of the same values gets."""
    from mlx_vit_amd import FusedAdamW
    n = (1 << 31) + 300

    def params(*sizes):
        ps = [torch.nn.Parameter(torch.full((k,), 0.25, dtype=torch.bfloat16, device=DEV)) for k in sizes]
        for p in ps:
            p.grad = torch.full_like(p, 0.5)
        return ps

    (big, behind), (small,) = params(n, 300), params(300)
    opt, ref = FusedAdamW([big, behind], lr=1e-2, states=states), FusedAdamW([small], lr=1e-2, states=states)
    opt.step()
    ref.step()
    assert bool((small != 0.25).all())
    assert bool((big == small[0]).all()) and torch.equal(behind, small)
    for k in opt.state:
        a, b = opt.state[k], ref.state[k]
        assert torch.equal(a[-b.numel():], b), k
    norm = opt.step(1.0)
    exact = 0.5 * (n + 300) ** 0.5
    assert abs(norm.item() - exact) <= 2.0 ** -23 * exact


@pytest.mark.parametrize("states", ["fp32", "int8"])
def test_moved_parameters_in_a_capture(states):
    """A step in a capture refuses weights that were moved, as often as it is asked; the step outside that it asks
    for updates the new ones, and the memory that they were moved from stays as it was."""
    from mlx_vit_amd import FusedAdamW
    a, b = (_params(SIZES, [torch.bfloat16] * len(SIZES), seed=13) for _ in range(2))
    oa, ob = (FusedAdamW(ps, states=states, master_weights=True) for ps in (a, b))
    for ps, o in ((a, oa), (b, ob)):
        _grads(ps, 50)
        o.step(1.0)
    old = [p.data for p in a]
    for p in a:
        p.data = p.data.clone()
    kept = [t.clone() for t in old]
    for ps in (a, b):
        _grads(ps, 51)
    torch.cuda.synchronize()
    for _ in range(2):
        with pytest.raises(RuntimeError, match="outside the capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                oa.step(1.0)
    assert oa.steps == 1
    for k in range(2):
        for ps, o in ((a, oa), (b, ob)):
            _grads(ps, 52 + k)
            o.step(1.0)
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and oa.steps == ob.steps
    assert all(torch.equal(oa.state[k], ob.state[k]) for k in oa.state)
    assert all(torch.equal(p, q) for p, q in zip(old, kept))


def test_a_plan_that_cannot_be_made(monkeypatch):
    """Whatever fails while the plan of moved weights is made, the next step makes it."""
    from mlx_vit_amd import FusedAdamW
    a, b = (_params(SIZES, [torch.float32] * len(SIZES), seed=14) for _ in range(2))
    oa, ob = FusedAdamW(a), FusedAdamW(b)
    for p in a:
        p.data = p.data.clone()
    for ps in (a, b):
        _grads(ps, 60)
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "synchronize", lambda *_: (_ for _ in ()).throw(RuntimeError("no memory")))
        with pytest.raises(RuntimeError, match="no memory"):
            oa.step(1.0)
    oa.step(1.0)
    ob.step(1.0)
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and oa.steps == 1


@pytest.mark.parametrize("states", ["fp32", "int8"])
@pytest.mark.parametrize("how", ["moved", "given", "given-moved", "loaded"])
def test_optimizer_dropped_behind_work_on_another_stream(how, states):
    """The same where the weights' plan is made on that stream, where the moments came from a caller who made
    them on a third one, and behind a state that is being loaded."""
    from mlx_vit_amd import FusedAdamW
    a, b = (_params(SIZES, [torch.float32] * len(SIZES), seed=15) for _ in range(2))
    for ps in (a, b):
        _grads(ps, 70)
    ref = FusedAdamW(b, states=states)
    made, stepped = torch.cuda.Stream(), torch.cuda.Stream()
    if how.startswith("given"):
        with torch.cuda.stream(made):
            given = {k: torch.zeros_like(t) for k, t in ref.state.items()}
        torch.cuda.synchronize()
        opt = FusedAdamW(a, states=states, state=given)
        del given
    else:
        opt = FusedAdamW(a, states=states)
    sizes = [t.nbytes for t in (*opt.state.values(), opt._plan)]
    state = ref.state_dict() if how == "loaded" else None
    ref.step(1.0)
    if how.endswith("moved"):
        for p in a:
            p.data = p.data.clone()
    torch.cuda.synchronize()
    if how == "given":
        stepped = torch.cuda.default_stream()
    with torch.cuda.stream(stepped):
        torch.cuda._sleep(20_000_000)   # some milliseconds (over before the plan of moved weights: it waits)
        if how == "loaded":
            opt.load_state_dict({k: t if k == "steps" else t.clone() for k, t in state.items()})
        else:
            opt.step(1.0)
            torch.cuda._sleep(20_000_000)
            opt.moments(torch.bfloat16)
    del opt
    others = []
    for s in (torch.cuda.default_stream(), made):
        with torch.cuda.stream(s):
            others += [torch.full((n,), 1, dtype=torch.uint8, device=DEV) for n in sizes for _ in range(4)]
    torch.cuda.synchronize()
    assert all(bool((t == 1).all()) for t in others)
    if how != "loaded":
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_graph_of_a_step_keeps_the_weights_it_writes():
    """Nobody but the optimizer holds the memory that the weights were moved from: no other tensor comes to lie
    there, and a replay goes on updating it."""
    from mlx_vit_amd import FusedAdamW
    a, b = (_params(SIZES, [torch.bfloat16] * len(SIZES), seed=16) for _ in range(2))
    oa, ob = FusedAdamW(a), FusedAdamW(b)
    for ps in (a, b):
        _grads(ps, 80)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        norm = oa.step(0.5)
    grads = [p.grad for p in a]
    spans = [(p.data_ptr(), p.nbytes) for p in a]
    for p in a:
        p.grad = None
        p.data = p.data.clone()
    oa.step()      # the plan is made again; no gradients: nothing moves
    moved = [p.detach().clone() for p in a]
    junk = [torch.full((n,), 7, dtype=torch.uint8, device=DEV) for _, n in spans for _ in range(16)]
    for x, n in ((t.data_ptr(), t.nbytes) for t in junk):
        assert not any(x < y + m and y < x + n for y, m in spans)
    for _ in range(3):
        g.replay()
        assert torch.equal(norm, ob.step(0.5))
    assert all(bool((t == 7).all()) for t in junk) and all(torch.equal(p, q) for p, q in zip(a, moved))
    assert len(grads) == len(a)


@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("states", ["fp32", "int8"])
@pytest.mark.parametrize("how", ["eps 0", "no factor", "infinite"])
def test_what_lies_between_the_weights_stays_zero(how, states, master):
    """With eps = 0 (0 / 0 there), with a clip factor that is NaN, with gradients that are infinite: whatever becomes
    of the weights, the buffers are zero between them, and load as a state does."""
    from mlx_vit_amd import FusedAdamW
    params = _params(SIZES, [torch.bfloat16] * len(SIZES), seed=17)
    opt = FusedAdamW(params, states=states, master_weights=master, eps=0.0 if how == "eps 0" else 1e-8)
    for k in range(2):
        _grads(params, 90 + k)
        if how != "eps 0":
            for p in params:
                p.grad.view(-1)[-1] = float("nan" if how == "no factor" else "inf")
        opt.step(1.0 if how == "no factor" else None)
    between = torch.ones(opt.total, dtype=torch.bool, device=DEV)
    for v in opt.views(between):
        v.fill_(False)
    assert between.any()
    for name in ("m", "v", "master"):
        if name in opt.state:
            assert not opt.state[name][between].any(), name
    if how == "eps 0":
        assert all(p.isfinite().all() for p in params)


@pytest.mark.parametrize("max_norm", [None, 1.0])
def test_a_step_that_fails_does_not_count(max_norm, monkeypatch):
    """No memory for the norm, a rate that the library refuses: the next step is the one that failed."""
    from mlx_vit_amd import FusedAdamW
    a, b = (_params(SIZES, [torch.float32] * len(SIZES), seed=18) for _ in range(2))
    oa, ob = (FusedAdamW(ps, bias_correction=True) for ps in (a, b))
    for ps in (a, b):
        _grads(ps, 95)
    if max_norm is not None:
        with monkeypatch.context() as m:
            m.setattr(torch, "empty", lambda *a, **k: (_ for _ in ()).throw(RuntimeError("no memory")))
            with pytest.raises(RuntimeError, match="no memory"):
                oa.step(max_norm)
    betas, oa.betas = oa.betas, (1.5, 0.95)
    with pytest.raises((RuntimeError, ValueError)):
        oa.step(max_norm)
    oa.betas = betas
    assert oa.steps == 0
    oa.step(max_norm)
    ob.step(max_norm)
    assert oa.steps == 1 and all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("dtype", [torch.float16, None], ids=["half", "any"])
def test_gradients_of_another_dtype_are_refused(dtype):
    """Half precision's bytes would be read as bf16's."""
    from mlx_vit_amd import FusedAdamW
    (p,) = _params([(300,)], [torch.bfloat16], seed=19)
    if not hasattr(p, "grad_dtype"):
        pytest.skip("this torch lets no gradient have another dtype")
    p.grad_dtype = dtype
    with pytest.raises(ValueError, match="grad_dtype"):
        FusedAdamW([p])
    p.grad_dtype = torch.bfloat16
    opt = FusedAdamW([p])
    p.grad = torch.ones_like(p)
    opt.step()
    p.grad = None
    p.grad_dtype = dtype
    p.data = p.data.clone()
    p.grad = torch.ones(300, dtype=torch.float16, device=DEV)
    w = p.detach().clone()
    with pytest.raises(ValueError, match="grad_dtype"):
        opt.step()
    assert torch.equal(p, w)
