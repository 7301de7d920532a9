"""What linear_act, mlp and FusedAdamW refuse, on the CPU: shapes, dtypes, devices,
and the C ABI's own checks, which come before any device work."""
import ctypes

import pytest
import torch

from mlx_vit_amd import FusedAdamW, _lib, linear_act, mlp
from mlx_vit_amd import train as TR

X, W, B, R = torch.zeros(4, 8), torch.zeros(6, 8), torch.zeros(6), torch.zeros(4, 6)


@pytest.mark.parametrize("args,match", [
    ((X, torch.zeros(6, 7)), "does not take 8 columns"),
    ((X, torch.zeros(6, 8, 1)), "does not take"),
    ((X, torch.zeros(0, 8)), "does not take"),
    ((torch.zeros(4, 0), torch.zeros(6, 0)), "does not take"),
    ((X, W, torch.zeros(5)), "bias shape"),
    ((X, W, B, torch.zeros(6)), "residual shape"),
    ((X, W, B, torch.zeros(1, 6)), "residual shape"),
    ((X, W, B, R, "relu"), "activation"),
    ((X.half(), W.half()), "unsupported"),
    ((X, W.bfloat16()), "expected torch.float32"),
    ((X.bfloat16(), W.bfloat16(), B), "bias has dtype"),
    ((X, W, B, R.double()), "residual has dtype"),
    ((torch.zeros(()), W), "must be"),
    ((X, W, B, R), "ROCm device"),
])
def test_linear_act_refuses(args, match):
    with pytest.raises(ValueError, match=match):
        linear_act(*args)


def test_mlp_refuses():
    w2, b2 = torch.zeros(8, 6), torch.zeros(8)
    for args, match in (((X, W, B, torch.zeros(8, 5), b2), "weight2 shape"), ((X, W, B, w2, torch.zeros(6)), "bias2 shape"),
                        ((X, W, B, w2, b2, R), "residual shape"), ((X, W, B, w2, b2, X, "tanh"), "activation"),
                        ((X, W, B, w2, b2, X), "ROCm device")):
        with pytest.raises(ValueError, match=match):
            mlp(*args)
    with pytest.raises(TypeError):
        mlp([1.0], W, B, w2, b2)


def test_fused_adamw_refuses():
    p = torch.nn.Parameter(torch.zeros(4))
    for kw, match in ((dict(states="fp8"), "states"), (dict(betas=(1.0, 0.9)), "betas"), (dict(eps=-1.0), "eps"),
                      (dict(), "ROCm device")):
        with pytest.raises(ValueError, match=match):
            FusedAdamW([p], **kw)
    with pytest.raises(ValueError, match="no parameters"):
        FusedAdamW([torch.nn.Parameter(torch.zeros(1), requires_grad=False)])
    with pytest.raises(ValueError, match="master_weights needs"):
        TR.TrainStep(torch.nn.Linear(2, 2), master_weights=True)


def _fwd(lib, **kw):
    a = dict(x=4096, ld_x=64, w=8192, ld_w=64, bias=None, res=None, ld_r=0, y=16384, ld_y=32, z=None, ld_z=0, M=9000, N=32,
             K=64, act=0, dtype=1, stream=None)
    a.update(kw)
    return lib.kda_linear_fwd(*a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=2), -2), (dict(act=3), -2), (dict(M=-1), -1), (dict(N=0), -1), (dict(K=0), -1), (dict(K=(1 << 20) + 1), -1),
    (dict(x=None), -1), (dict(w=None), -1), (dict(y=None), -1), (dict(x=4098), -1), (dict(w=8200), -1), (dict(ld_x=60), -1),
    (dict(ld_x=63, K=63), -1), (dict(ld_w=68), -1), (dict(ld_y=31), -1), (dict(res=4096, ld_r=16), -1),
    (dict(z=4097, ld_z=32), -1), (dict(bias=4097), -1), (dict(ld_x=(1 << 21) + 8), -1), (dict(dtype=0, x=4098), -1),
    (dict(M=(1 << 31) - 1, N=1 << 20, ld_y=1 << 20), -2),
])
def test_c_abi_linear_fwd_refuses(kw, rc):
    lib = _lib.load()
    assert _fwd(lib, **kw) == rc and _lib.last_error()


def test_c_abi_linear_nothing_to_do():
    lib = _lib.load()
    assert _fwd(lib, M=0, x=None) == 0
    assert lib.kda_linear_bwd_workspace_size(4096, 16, 0, 16, 16, 0, 0) == 0
    assert lib.kda_linear_pad(None, 0, 0, 0, None, None, 0, 0, 0, None, None) == 0


def test_c_abi_backward_workspace():
    """fp32: at least one partial gradient; dz where an activation is, or a bf16 dy cannot be read as it is."""
    lib = _lib.load()
    size = lambda dy=4096, ld=32, M=100, N=32, K=64, act=0, dtype=1: lib.kda_linear_bwd_workspace_size(dy, ld, M, N, K, act, dtype)  # noqa: E731
    assert size(dtype=0) >= 4 * (32 * 64 + 32)
    assert size(act=1) >= size() + 2 * 100 * 32
    assert size(dy=4098) >= size() + 2 * 100 * 32 and size(ld=33) >= size() + 2 * 100 * 32
    assert size(K=63) >= size() + 2 * 32 * 64
    assert lib.kda_mlp_bwd_workspace_size(4096, 32, 100, 128, 64, 32, 1, 1) >= 2 * 100 * 128


def test_c_abi_backward_refuses():
    lib = _lib.load()
    a0 = dict(dy=4096, ld_dy=32, x=4096, ld_x=64, w=8192, ld_w=64, z=4096, ld_z=32, dx=16384, ld_dx=64, dw=4096, db=4096,
              M=100, N=32, K=64, act=1, dtype=1, ws=4096, n=1 << 30, st=None)
    for kw, rc in ((dict(dy=None), -1), (dict(x=None), -1), (dict(w=None), -1), (dict(z=None), -1), (dict(dw=None), -1),
                   (dict(ld_dy=31), -1), (dict(ld_x=60), -1), (dict(x=4104), -1), (dict(w=8200), -1), (dict(ld_dx=63), -1),
                   (dict(dw=4104), -1), (dict(act=5), -2), (dict(dtype=7), -2), (dict(M=0), -1), (dict(ws=None), -1),
                   (dict(ws=4100), -1), (dict(n=16), -3), (dict(dtype=0, dy=4098), -1)):
        assert lib.kda_linear_bwd(*{**a0, **kw}.values()) == rc, kw
    m0 = dict(dy=4096, ld_dy=32, x=4096, ld_x=64, w1=8192, ld_w1=64, z=4096, ld_z=128, h=4096, ld_h=128, w2=4096, ld_w2=128,
              dx=16384, ld_dx=64, dw1=4096, db1=4096, dw2=4096, db2=4096, M=100, N=128, K=64, O=32, act=1, dtype=1, ws=4096,
              n=1 << 30, st=None)
    for kw, rc in ((dict(dy=None), -1), (dict(x=None), -1), (dict(w1=None), -1), (dict(w2=None), -1), (dict(z=None), -1),
                   (dict(h=None), -1), (dict(dw1=None), -1), (dict(dw2=None), -1), (dict(h=4104), -1), (dict(ld_h=127), -1),
                   (dict(O=0), -1), (dict(M=-1), -1), (dict(act=3), -2), (dict(ws=None), -1), (dict(n=16), -3)):
        assert lib.kda_mlp_bwd(*{**m0, **kw}.values()) == rc, kw
    p0 = dict(s0=4096, ld0=10, r0=4, c0=9, d0=4096, s1=None, ld1=0, r1=0, c1=0, d1=None, st=None)
    for kw, rc in ((dict(s0=None), -1), (dict(d0=None), -1), (dict(d0=4104), -1), (dict(ld0=8), -1), (dict(c0=0), -1),
                   (dict(r0=-1), -1), (dict(d1=4096), -1)):
        assert lib.kda_linear_pad(*{**p0, **kw}.values()) == rc, kw


def _tensor(p=4096, g=8192, n=10, offset=0, dtype=1):
    return (ctypes.c_int64 * 5)(p, g, n, offset, dtype)


def _step(lib, t, count=1, states=0, m=4096, v=8192, ms=None, vs=None, master=None, b1=0.9, b2=0.95, eps=1e-8, c1=1.0, c2=1.0, plan=4096,
          norm=0.0, clip=4096, ws=8192, n=1 << 10):
    return lib.kda_adamw_step(t, count, plan, states, m, v, ms, vs, master, norm, clip, 1e-3, b1, b2, eps, 0.05, c1, c2, ws, n,
                              None)


def test_c_abi_adamw_refuses():
    lib = _lib.load()
    for t, rc in ((_tensor(p=0), -1), (_tensor(p=4097), -1), (_tensor(g=8194, dtype=0), -1),
                  (_tensor(n=-1), -1), (_tensor(offset=100), -1), (_tensor(offset=-256), -1), (_tensor(dtype=2), -2), (_tensor(n=1 << 36), -2)):
        assert _step(lib, t) == rc, list(t)
    t = _tensor()
    for kw, rc in ((dict(count=-1), -1), (dict(states=2), -2), (dict(m=None), -1), (dict(v=8196), -1), (dict(master=4100), -1),
                   (dict(states=1), -1), (dict(states=1, ms=4096, vs=4098), -1), (dict(b1=1.0), -1), (dict(b2=-0.1), -1),
                   (dict(eps=-1.0), -1), (dict(c1=0.0), -1), (dict(c2=float("nan")), -1), (dict(plan=None), -1), (dict(plan=4100), -1)):
        assert _step(lib, t, **kw) == rc, kw
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 15) & ~15
    n = lib.kda_adamw_plan_size(t, 1)
    assert 0 < n <= 64 and lib.kda_adamw_plan(t, 1, at, n) == 0
    assert lib.kda_adamw_plan(t, 1, at, n - 1) == -3 and lib.kda_adamw_plan(t, 1, None, n) == -1
    assert lib.kda_adamw_plan(_tensor(p=0), 1, at, n) == -1
    assert _step(lib, None, count=1) == -1 and _step(lib, None, count=0) == 0
    for kw, rc in ((dict(clip=None), -1), (dict(clip=4098), -1), (dict(norm=-1.0), -1), (dict(norm=float("nan")), -1),
                   (dict(ws=None), -1), (dict(ws=8196), -1), (dict(n=0), -3)):
        assert _step(lib, t, **{"norm": 1.0, **kw}) == rc, kw
    assert lib.kda_adamw_step_workspace_size(_tensor(n=100000), 1) >= 8
    mom = lambda **kw: lib.kda_adamw_moments(*{**dict(m=4096, v=4096, ms=4096, vs=4096, mo=4096, vo=4096, n=256, dt=1, st=None), **kw}.values())  # noqa: E731
    for kw, rc in ((dict(n=100), -1), (dict(n=-256), -1), (dict(dt=3), -2), (dict(m=None), -1), (dict(mo=4100), -1), (dict(ms=None), -1)):
        assert mom(**kw) == rc, kw
    assert mom(n=0) == 0
