"""What chunk_decay, decay_step and rotary refuse, on the CPU: shapes, dtypes, devices, and
the C ABI's own checks, which come before any device work."""
import ctypes

import pytest
import torch

from mlx_vit_amd import _lib, chunk_decay, decay_step, rotary

Q, G, S = torch.zeros(2, 5, 4, 32), torch.zeros(2, 5, 4), torch.zeros(2, 4, 32, 32)
ROW = Q[:1]
CU = torch.tensor([0, 2, 5], dtype=torch.int32)


@pytest.mark.parametrize("args,match", [
    ((Q[0], Q, Q, G), "q must be"),
    ((torch.zeros(2, 5, 4, 48),) * 3 + (G,), "head_dim=48"),
    ((Q.half(), Q.half(), Q.half(), G), "unsupported"),
    ((Q, Q[:, :4], Q, G), "k shape"),
    ((Q, Q, Q[..., :16], G), "v shape"),
    ((Q, Q.bfloat16(), Q, G), "k has dtype"),
    ((Q, torch.zeros(2, 5, 3, 32), Q, G), "do not divide"),
    ((Q, Q, torch.zeros(2, 5, 8, 32), G), "do not divide"),
    ((Q, Q, Q, G[:1]), "g shape"),
    ((Q, Q, Q, torch.zeros(2, 5, 4, 32)), "g shape"),
    ((Q, Q, Q, torch.zeros(6)), "do not divide"),
    ((Q, Q, Q, G.double()), "g dtype"),
    ((Q, Q, Q, G, S[:1]), "initial_state shape"),
    ((Q, Q, Q, G, S.bfloat16()), "initial_state has dtype"),
    ((ROW, ROW, ROW, G[:1], S, CU.long()), "int32"),
    ((ROW, ROW, ROW, G[:1], S, CU[None]), "int32"),
    ((ROW, ROW, ROW, G[:1], S, CU[:0]), "int32"),
    ((Q, Q, Q, G, S, CU), "one row"),
    ((ROW, ROW, ROW, G[:1], S[:1], CU), "initial_state shape"),
    ((Q, Q, Q, G, S), "ROCm device"),
    ((ROW, ROW, ROW, torch.zeros(4), S, CU), "ROCm device"),
])
def test_chunk_decay_refuses(args, match):
    with pytest.raises(ValueError, match=match):
        chunk_decay(*args)


def test_not_tensors():
    for f in (lambda: chunk_decay(Q, Q, Q, 0.5), lambda: chunk_decay(Q, Q, [1.0], G), lambda: chunk_decay(Q, Q, Q, G, 1.0),
              lambda: chunk_decay(ROW, ROW, ROW, G[:1], None, [0, 5]), lambda: decay_step(Q[:, 0], Q[:, 0], Q[:, 0], G[:, 0], None),
              lambda: decay_step(Q[:, 0], Q[:, 0], Q[:, 0], G[:, 0], S, [0, 1]), lambda: rotary(Q, [1.0], grid=(2, 2)),
              lambda: rotary(Q, None, [0, 1, 2, 3, 4])):
        with pytest.raises(TypeError):
            f()


@pytest.mark.parametrize("args,match", [
    ((Q, Q, Q, G, S), "q must be"),
    ((Q[:, 0], Q[:1, 0], Q[:, 0], G[:, 0], S), "k shape"),
    ((Q[:, 0], Q[:, 0], Q[:, 0], G[:, 0], S[:1]), "state shape"),
    ((Q[:, 0], Q[:, 0], Q[:, 0], G[:, 0], S.bfloat16()), "state has dtype"),
    ((Q[:, 0], Q[:, 0], Q[:, 0], G[:, 0], S.transpose(2, 3)), "contiguous"),
    ((Q[:, 0], Q[:, 0], Q[:, 0], G[:, 0], S, CU), "slots must be"),
    ((Q[:, 0], Q[:, 0], Q[:, 0], G[:, 0], S, CU[:2].long()), "slots must be"),
    ((Q[:, 0], Q[:, 0], Q[:, 0], G[:, 0], torch.zeros(()), CU[:2]), "state shape"),
    ((Q[:, 0], Q[:, 0], Q[:, 0], G[:, 0], S), "ROCm device"),
])
def test_decay_step_refuses(args, match):
    with pytest.raises(ValueError, match=match):
        decay_step(*args)


P = torch.arange(5)


@pytest.mark.parametrize("args,kw,match", [
    ((Q[0],), dict(grid=(2, 2)), "q must be"),
    ((Q.half(),), dict(grid=(2, 2)), "unsupported"),
    ((torch.zeros(1, 2, 3, 7), None, P[:2]), {}, "head_dim=7"),
    ((torch.zeros(1, 2, 3, 260), None, P[:2]), {}, "head_dim=260"),
    ((Q, Q[:, :4]), dict(grid=(2, 2)), "k shape"),
    ((Q, Q.bfloat16()), dict(grid=(2, 2)), "k has dtype"),
    ((Q,), {}, "either positions or grid"),
    ((Q, None, P), dict(grid=(2, 2)), "either positions or grid"),
    ((Q, None, P[:4]), {}, "positions shape"),
    ((Q, None, P), dict(sections=(8, 8)), "positions shape"),
    ((Q, None, P.double()), {}, "positions dtype"),
    ((Q, None, P), dict(start=3), "start=3"),
    ((Q, None, P), dict(sections=(5,)), "sections"),
    ((Q, None, P), dict(sections=(34,)), "sections"),
    ((Q, None, P), dict(sections=()), "sections"),
    ((Q, None, P), dict(sections=(2, 2, 2, 2, 2)), "sections"),
    ((Q, None, P), dict(base=0.0), "base"),
    ((Q,), dict(grid=(0, 2)), "grid"),
    ((Q,), dict(grid=(2, 2), start=-1), "grid"),
    ((Q,), dict(grid=(2, 2), sections=(8, 8, 8, 8)), "grid"),
    ((Q, None, P.float().requires_grad_(True)), {}, "no gradient for positions"),
    ((Q, Q, P), {}, "ROCm device"),
])
def test_rotary_refuses(args, kw, match):
    with pytest.raises(ValueError, match=match):
        rotary(*args, **kw)


class Rows(ctypes.Structure):
    _fields_ = [("p", ctypes.c_void_p)] + [(n, ctypes.c_int64) for n in ("batch", "token", "head", "heads")]


class Decay(ctypes.Structure):
    _fields_ = ([(n, Rows) for n in ("q", "k", "v", "dout")] + [("g", ctypes.c_void_p)]
                + [(n, ctypes.c_int64) for n in ("g_batch", "g_token", "g_head")]
                + [("s0", ctypes.c_void_p), ("cu", ctypes.c_void_p), ("nseq", ctypes.c_int64)]
                + [(n, ctypes.c_void_p) for n in ("o", "s_final", "ds_final", "dq", "dk", "dv", "dg")]
                + [("dg_heads", ctypes.c_int64), ("ds0", ctypes.c_void_p)]
                + [(n, ctypes.c_int64) for n in ("B", "T", "H", "D", "dtype")] + [("workspace", ctypes.c_void_p), ("ws_bytes", ctypes.c_int64), ("kept", ctypes.c_void_p), ("kept_bytes", ctypes.c_int64), ("train", ctypes.c_int64)])


def _decay(**kw):
    a = Decay(B=2, T=300, H=4, D=64, dtype=1)
    for i, n in enumerate(("q", "k", "v", "dout")):
        setattr(a, n, Rows(4096 * (i + 1), 300 * 256, 256, 64, 4))
    for i, n in enumerate(("g", "o", "s_final", "dq", "dk", "dv", "dg", "workspace", "kept")):
        setattr(a, n, 65536 * (i + 1))
    a.ws_bytes = a.kept_bytes = 1 << 40
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw,code,match", [
    (dict(dtype=2), _lib.KDA_E_UNSUPPORTED, "dtype"),
    (dict(D=48), _lib.KDA_E_UNSUPPORTED, "D=48"),
    (dict(H=0), _lib.KDA_E_INVALID, "H=0"),
    (dict(T=-1), _lib.KDA_E_INVALID, "T=-1"),
    (dict(H=6), _lib.KDA_E_INVALID, "do not divide"),
    (dict(q=Rows(4097, 0, 256, 64, 4)), _lib.KDA_E_INVALID, "q is NULL or not"),
    (dict(k=Rows(4096, 0, 252, 64, 4)), _lib.KDA_E_INVALID, "k: strides"),
    (dict(v=Rows(None, 0, 256, 64, 4)), _lib.KDA_E_INVALID, "v is NULL"),
    (dict(g=None), _lib.KDA_E_INVALID, "g is NULL"),
    (dict(s0=8), _lib.KDA_E_INVALID, "s0"),
    (dict(B=2, cu=4096, nseq=2), _lib.KDA_E_INVALID, "one row"),
    (dict(workspace=None), _lib.KDA_E_INVALID, "workspace"),
    (dict(ws_bytes=16), _lib.KDA_E_WORKSPACE, "needs"),
    (dict(q=Rows(4096, 0, (1 << 24) + 8, 64, 4)), _lib.KDA_E_INVALID, "token stride"),
    (dict(B=1 << 30, T=4096), _lib.KDA_E_UNSUPPORTED, "too many workgroups"),
    (dict(B=1 << 22, T=1), _lib.KDA_E_UNSUPPORTED, "too many workgroups"),   # 2^32 threads
])
def test_decay_abi_refuses(kw, code, match):
    lib = _lib.load()
    a = _decay(**{**dict(B=1, T=100000), **kw})
    for f in (lib.kda_decay_fwd, lib.kda_decay_bwd):
        assert f(ctypes.addressof(a), None) == code
        assert match in _lib.last_error()


def test_decay_abi_refuses_its_own():
    lib = _lib.load()
    for f, kw, match in ((lib.kda_decay_fwd, dict(o=None), "o is NULL"), (lib.kda_decay_fwd, dict(s_final=4), "s_final"),
                         (lib.kda_decay_bwd, dict(dq=None), "dq"), (lib.kda_decay_bwd, dict(dg=2), "dg"),
                         (lib.kda_decay_bwd, dict(ds_final=65536, s_final=None), "s_final (of the forward"),
                         (lib.kda_decay_bwd, dict(B=1, T=100000, kept=None), "kept is NULL"),
                         (lib.kda_decay_fwd, dict(B=1, T=100000, train=1, kept=None), "kept is NULL")):
        a = _decay(**kw)
        assert f(ctypes.addressof(a), None) == _lib.KDA_E_INVALID
        assert match in _lib.last_error()
    assert lib.kda_decay_fwd(None, None) == lib.kda_decay_bwd(None, None) == lib.kda_rotary(None, None) == _lib.KDA_E_INVALID
    a = _decay(T=2)
    assert lib.kda_decay_step(ctypes.addressof(a), None, 2, None) == _lib.KDA_E_INVALID and "T=2" in _lib.last_error()
    a = _decay(T=1)
    assert lib.kda_decay_step(ctypes.addressof(a), None, 3, None) == _lib.KDA_E_INVALID and "3 states" in _lib.last_error()
    a = _decay(T=1, B=1 << 21)
    assert lib.kda_decay_step(ctypes.addressof(a), None, 1 << 21, None) == _lib.KDA_E_UNSUPPORTED
    a = _decay(T=1, s0=None)
    assert lib.kda_decay_step(ctypes.addressof(a), None, 2, None) == _lib.KDA_E_INVALID and "s0" in _lib.last_error()


def test_decay_workspace():
    """None where no sequence is shared out; the states between its parts where one is."""
    lib = _lib.load()
    size = lambda pass_, **kw: lib.kda_decay_workspace_size(pass_, ctypes.addressof(_decay(**kw)))  # noqa: E731
    assert size(_lib.KDA_PASS_FWD, B=256, T=1568, H=12) == 0
    assert size(_lib.KDA_PASS_FWD, B=1, T=64) == 0
    n = size(_lib.KDA_PASS_FWD, B=1, T=65536, H=12)
    assert n and n % (12 * 4) == 0 and n > 12 * 4 * 64 * 64 * 2
    # a training pass keeps the states at its slots' starts, a backward pass makes as many adjoints
    own = Rows(4096, 0, 768, 64, 12)
    many = dict(B=1, T=65536, H=12, dg=None, q=own, k=own, v=own)
    assert size(_lib.KDA_PASS_TRAIN, **many) == size(_lib.KDA_PASS_BWD, **many) > 12 * 4 * 64 * 64 * 2
    assert size(_lib.KDA_PASS_BWD, **{**many, "dg": 64}) - size(_lib.KDA_PASS_BWD, **many) >= 4 * 65536 * 12
    assert size(_lib.KDA_PASS_BWD, **{**many, "k": Rows(4096, 0, 64, 64, 1)}) - size(_lib.KDA_PASS_BWD, **many) == 2 * 4 * 65536 * 12 * 64
    assert size(_lib.KDA_PASS_FWD, dtype=5) == 0 and "dtype" in _lib.last_error()
    # packed: a slot for every sequence, and for what lies around them
    many = size(_lib.KDA_PASS_FWD, B=1, T=64, cu=4096, nseq=1000)
    assert many >= 1000 * 4 * 64 * 64 * 4
