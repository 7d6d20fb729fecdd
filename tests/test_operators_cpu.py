"""CPU: what the dense-layer operators (orthogonalised updates, 8-bit linear layers) refuse, and how they read their arguments."""
import ctypes

import pytest
import torch

from point2cyl_amd import _lib, ops, optim, train

ONE = ctypes.c_void_p(16)              # a non-null, 16-byte aligned dummy: arguments are checked before anything is dereferenced


def _mats(*shapes, batch=1, src=16, dst=16, mom=16):
    a = (_lib.NsMatrix * len(shapes))()
    for m, (r, c) in zip(a, shapes):
        m.src, m.dst, m.mom, m.rows, m.cols, m.batch = src, dst, mom, r, c, batch
        m.src_rs = m.dst_rs = c
        m.src_cs = m.dst_cs = 1
    return a


def test_newton_schulz_entry_refuses_bad_arguments():
    L = _lib.lib()
    co = ops.ns_coefficients(5, ops.NS_COEFFS)
    big = 1 << 40
    assert L.p2c_newton_schulz_ws_bytes(None, 1) == 0 and L.p2c_newton_schulz_ws_bytes(_mats((-1, 4)), 1) == 0
    assert L.p2c_newton_schulz(None, 1, 0, 5, co, 1e-7, ONE, big, None) == -1
    assert L.p2c_newton_schulz(_mats((64, 64)), 0, 0, 5, co, 1e-7, ONE, big, None) == -1
    assert L.p2c_newton_schulz(_mats((64, -1)), 1, 0, 5, co, 1e-7, ONE, big, None) == -1
    assert L.p2c_newton_schulz(_mats((1 << 20, 1 << 20)), 1, 0, 5, co, 1e-7, ONE, big, None) == -1      # more than 2^31 elements
    assert L.p2c_newton_schulz(_mats((64, 64), src=0), 1, 0, 5, co, 1e-7, ONE, big, None) == -1
    assert L.p2c_newton_schulz(_mats((64, 64)), 1, 3, 5, co, 1e-7, ONE, big, None) == -1                # no such type
    assert L.p2c_newton_schulz(_mats((64, 64)), 1, 0, 17, co, 1e-7, ONE, big, None) == -1
    assert L.p2c_newton_schulz(_mats((64, 64)), 1, 0, 5, co, 0.0, ONE, big, None) == -1
    assert L.p2c_newton_schulz(_mats((64, 64)), 1, 0, 5, co, float("nan"), ONE, big, None) == -1
    assert L.p2c_newton_schulz(_mats((64, 64)), 1, 0, 5, None, 1e-7, ONE, big, None) == -1
    need = L.p2c_newton_schulz_ws_bytes(_mats((100, 300)), 1)
    assert need > 0 and L.p2c_newton_schulz(_mats((100, 300)), 1, 0, 5, co, 1e-7, ONE, need - 1, None) == -1   # workspace too small
    assert L.p2c_newton_schulz(_mats((100, 300)), 1, 0, 5, co, 1e-7, ctypes.c_void_p(8), big, None) == -1       # ... or not aligned
    wild = (ctypes.c_float * 15)(*([10.0, 20.0, 30.0] * 5))
    assert L.p2c_newton_schulz(_mats((64, 64)), 1, 0, 5, wild, 1e-7, ONE, big, None) == -1
    nan = (ctypes.c_float * 15)(*([float("nan")] * 15))
    assert L.p2c_newton_schulz(_mats((64, 64)), 1, 0, 5, nan, 1e-7, ONE, big, None) == -1
    assert L.p2c_muon_step_f32(_mats((64, 64), mom=0), 1, 0.95, 1, 5, co, 1e-7, ONE, big, None) == -1
    assert L.p2c_muon_step_f32(_mats((64, 64)), 1, 1.0, 1, 5, co, 1e-7, ONE, big, None) == -1                # momentum outside [0, 1)
    assert L.p2c_muon_step_f32(_mats((64, 64), batch=2), 1, 0.5, 1, 5, co, 1e-7, ONE, big, None) == -1
    assert L.p2c_newton_schulz(_mats((0, 5), (7, 0)), 2, 0, 5, co, 1e-7, None, 0, None) == 0                  # nothing to do: no launch, no workspace


def test_int8_entries_refuse_bad_arguments():
    L = _lib.lib()
    assert L.p2c_int8_padded(1) == 64 and L.p2c_int8_padded(64) == 64 and L.p2c_int8_padded(65) == 128 and L.p2c_int8_padded(0) == 0
    assert L.p2c_int8_padded_out(1) == 256 and L.p2c_int8_padded_out(257) == 512
    assert L.p2c_int8_few_supported(32, 2048) == 1 and L.p2c_int8_few_supported(33, 8) == 0 and L.p2c_int8_few_supported(1, 2049) == 0
    assert L.p2c_int8_requant_supported(512, 2, 20.0) == 1 and L.p2c_int8_requant_supported(513, 0, 20.0) == 0
    assert L.p2c_int8_requant_supported(8, 2, 5.0) == 0 and L.p2c_int8_requant_supported(8, 1, 5.0) == 1
    q = lambda **k: L.p2c_quantize_rows(*[dict(x=ONE, dt=0, ld=8, M=2, K=8, Kp=64, q=ONE, s=ONE, st=None, **{})[n] if n not in k else k[n]  # noqa: E731
                                          for n in ("x", "dt", "ld", "M", "K", "Kp", "q", "s", "st")])
    assert q(M=0) == 0                                             # no rows: no launch
    assert q(x=None) == -1 and q(q=None) == -1 and q(s=None) == -1 and q(dt=3) == -1 and q(K=0) == -1 and q(Kp=60) == -1 and q(K=65) == -1
    assert q(K=131073, Kp=131136) == -1 and q(M=-1) == -1 and q(ld=-8) == -1 and q(q=ctypes.c_void_p(8)) == -2
    assert L.p2c_dequantize_rows(None, ONE, 2, 8, 64, ONE, 0, None) == -1 and L.p2c_dequantize_rows(ONE, ONE, 2, 8, 64, ONE, 4, None) == -1
    names = ("xq", "ldx", "sx", "wq", "sw", "bias", "add", "ldadd", "act", "beta", "thr", "out", "ldo", "dt", "M", "N", "K", "Kp", "st")
    good = dict(xq=ONE, ldx=64, sx=ONE, wq=ONE, sw=ONE, bias=None, add=None, ldadd=0, act=0, beta=1.0, thr=20.0, out=ONE, ldo=8, dt=0, M=4, N=8, K=8, Kp=64, st=None)
    lin = lambda **k: L.p2c_int8_linear(*[{**good, **k}[n] for n in names])  # noqa: E731
    assert lin(M=0) == 0
    for bad in (dict(xq=None), dict(sx=None), dict(wq=None), dict(sw=None), dict(out=None), dict(ldx=32), dict(act=3), dict(act=2, beta=0.0),
                dict(act=2, beta=float("nan")), dict(dt=3), dict(ldo=7), dict(add=ONE, ldadd=7), dict(N=0), dict(K=0), dict(Kp=100)):
        assert lin(**bad) == -1, bad
    assert lin(xq=ctypes.c_void_p(8)) == -2 and lin(wq=ctypes.c_void_p(8)) == -2 and lin(ldx=72) == -2
    rq = lambda **k: L.p2c_int8_linear_requant(*[{**good, "ldo": 64, "so": ONE, **k}[n] for n in (*names[:13], "so", *names[14:])])  # noqa: E731
    assert rq(M=0) == 0 and rq(N=513, ldo=576) == -1 and rq(ldo=128) == -1 and rq(so=None) == -1 and rq(out=ctypes.c_void_p(8)) == -2
    few = lambda **k: L.p2c_int8_linear_few(*[{**good, "x": ONE, "xdt": 0, "ldx": 8, **k}[n] for n in ("x", "xdt", "ldx", "wq", *names[4:])])  # noqa: E731
    assert few(M=33) == -1 and few(K=2049, Kp=2112) == -1 and few(x=None) == -1 and few(xdt=5) == -1 and few(M=0) == -1
    flo = lambda **k: L.p2c_int8_linear_float(*[{**good, "x": ONE, "xdt": 0, "ldx": 8, "M": 40, "ws": ONE, **k}[n]  # noqa: E731
                                                for n in ("x", "xdt", "ldx", "wq", *names[4:18], "ws", "st")])
    assert flo(M=0) == 0 and flo(M=0, ws=None, x=None) == 0
    for bad in (dict(x=None), dict(ws=None), dict(wq=None), dict(sw=None), dict(out=None), dict(xdt=5), dict(ldx=-1), dict(act=3), dict(act=2, beta=0.0), dict(dt=3), dict(ldo=7),
                dict(add=ONE, ldadd=7), dict(N=0), dict(K=0), dict(Kp=100), dict(M=-1), dict(M=4, x=None), dict(M=4, K=2049, Kp=2112, ws=None)):
        assert flo(**bad) == -1, bad
    assert flo(wq=ctypes.c_void_p(8)) == -2 and flo(ws=ctypes.c_void_p(8)) == -2
    rqf = lambda **k: L.p2c_int8_linear_requant_float(*[{**good, "x": ONE, "xdt": 0, "ldx": 8, "ldo": 64, "so": ONE, "ws": ONE, **k}[n]  # noqa: E731
                                                        for n in ("x", "xdt", "ldx", "wq", *names[4:13], "so", *names[14:18], "ws", "st")])
    assert rqf(M=0) == 0 and rqf(N=513, ldo=576) == -1 and rqf(ldo=128) == -1 and rqf(so=None) == -1 and rqf(ws=None) == -1 and rqf(x=None) == -1 and rqf(M=-1) == -1
    assert rqf(act=2, thr=5.0) == -1 and rqf(out=ctypes.c_void_p(8)) == -2 and rqf(wq=ctypes.c_void_p(8)) == -2


def test_coefficients():
    assert list(ops.ns_coefficients(2, (1.5, -0.5, 0.0))) == [1.5, -0.5, 0.0, 1.5, -0.5, 0.0]
    assert len(ops.ns_coefficients(2, ((3.0, -3.0, 1.0), (1.5, -0.5, 0.0)))) == 6
    for steps, co in ((0, ops.NS_COEFFS), (17, ops.NS_COEFFS), (2, (1.0, 2.0)), (3, ((1.5, -0.5, 0.0),)), (5, (10.0, 20.0, 30.0)), (2, (float("nan"), 0.0, 0.0))):
        with pytest.raises(ValueError):
            ops.ns_coefficients(steps, co)


def test_no_cpu_path():
    for f in (lambda: ops.newton_schulz(torch.zeros(4, 4)), lambda: ops.quantize_rows(torch.zeros(4, 4)), lambda: ops.Int8Weight(torch.zeros(4, 4))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            f()
    assert ops.newton_schulz([]) == []
    p = torch.nn.Parameter(torch.zeros(4, 4))
    p.grad = torch.zeros(4, 4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        optim.Muon([p]).step()


def test_muon_refuses_bad_settings():
    p = torch.nn.Parameter(torch.zeros(4, 4))
    for kw in (dict(momentum=1.0), dict(momentum=-0.1), dict(adjust="size"), dict(eps=0.0), dict(ns_steps=0), dict(ns_coeffs=(9.0, 9.0, 9.0))):
        with pytest.raises(ValueError):
            optim.Muon([p], **kw)
    o = optim.Muon([p])
    with pytest.raises(ValueError):
        o.add_param_group({"params": [torch.nn.Parameter(torch.zeros(2, 2))], "momentum": 2.0})


def test_the_8_bit_decoder_flag_needs_the_decoder():
    from point2cyl_amd import eval as ev
    with pytest.raises(SystemExit, match="with_sketch_fit"):
        ev.main(["--int8_decoder", "--synthetic", "2"])


def test_trainer_flags_choose_the_update_rule():
    p = train.build_parser()
    net = torch.nn.Sequential(torch.nn.Linear(4, 3), torch.nn.Linear(3, 2))
    groups = [{"params": list(net.parameters()), "lr": 0.5}]
    a = p.parse_args([])
    assert type(optim.from_arguments(a, groups)) is optim.Adam
    with pytest.raises(SystemExit):
        optim.from_arguments(p.parse_args(["--weight_decay", "0.1"]), groups)
    a = p.parse_args(["--optimizer", "muon", "--weight_decay", "0.1", "--muon_momentum", "0.9"])
    o = optim.from_arguments(a, groups, heads=list(net[1].parameters()))
    assert type(o) is optim.Muon and [g["use_muon"] for g in o.param_groups] == [True, False] and [g["source"] for g in o.param_groups] == [0, 0]
    assert all(g["lr"] == 0.5 and g["weight_decay"] == 0.1 and g["momentum"] == 0.9 for g in o.param_groups)
    assert [len(g["params"]) for g in o.param_groups] == [2, 2]
