"""CPU: the ends of what the dense-layer operators accept - launch sizes, row counts, settings - and what they refuse there."""
import copy
import ctypes
import pickle

import pytest
import torch

from point2cyl_amd import _lib, backbone, ops, optim, sketch, train_sketch

ONE = ctypes.c_void_p(16)              # a non-null, 16-byte aligned dummy: arguments are checked before anything is dereferenced


def test_quantize_launches_fit_a_grid():
    """A launch holds fewer than 2^32 threads; a workgroup of 256 takes four rows of up to 1024 elements or one longer row."""
    L = _lib.lib()
    assert L.p2c_quantize_rows_at_once(0) == 0
    for K in (1, 64, 1000, 1024, 1025, 2048, 5000, 131072):
        rows = L.p2c_quantize_rows_at_once(K)
        assert rows >= 1 << 20 and (rows + 3) // 4 * 256 < 1 << 32
        if K > 1024:
            assert rows * 256 < 1 << 32
    top = (1 << 30) - 64               # ... and a tile of 64 rows is a workgroup of 256 in the requantising product
    assert -(-top // 64) * 256 < 1 << 32
    for M in (top + 1, (1 << 31) - 1):
        assert L.p2c_quantize_rows(ONE, 0, 8, M, 8, 64, ONE, ONE, None) == -1
        assert L.p2c_int8_linear_requant(ONE, 64, ONE, ONE, ONE, None, None, 0, 0, 1.0, 20.0, ONE, 64, ONE, M, 8, 8, 64, None) == -1


def test_newton_schulz_refuses_steps_that_amplify_too_much():
    """The operands' floor of 2^-37 may grow to 2^-22 of one, not further: by the steps from any one to the last."""
    L = _lib.lib()
    a = (ctypes.c_float * 48)
    need = 1 << 40
    m = (_lib.NsMatrix * 1)()
    m[0].rows, m[0].cols, m[0].batch, m[0].src, m[0].dst, m[0].src_rs, m[0].src_cs, m[0].dst_rs, m[0].dst_cs = 0, 4, 1, 16, 16, 4, 1, 4, 1       # no rows: nothing is launched
    entry = lambda steps, co: L.p2c_newton_schulz(m, 1, 0, steps, a(*[v for c in co for v in c]), 1e-7, ONE, need, None)  # noqa: E731
    weak, flat, strong = (1.875, -1.25, 0.375), (1.0, 0.0, 0.0), ops.NS_COEFFS
    for co in ([strong] * 8, [weak] * 16, [strong] * 5 + [weak] * 4, [flat] * 8 + [strong] * 8, [(0.1, 0.0, 0.0)] * 4 + [strong] * 8):
        assert len(ops.ns_coefficients(len(co), co)) == 3 * len(co) and entry(len(co), co) == 0, co
    for co in ([strong] * 9, [strong] * 16, [strong] * 8 + [weak] * 2, [(0.1, 0.0, 0.0)] * 4 + [strong] * 9):
        with pytest.raises(ValueError, match="2\\^15"):
            ops.ns_coefficients(len(co), co)
        assert entry(len(co), co) == -1, co
    with pytest.raises(ValueError, match="2\\^15"):
        optim.Muon([torch.nn.Parameter(torch.zeros(4, 4))], ns_steps=16)


@pytest.mark.parametrize("name", ["Adam", "Muon"])
def test_adams_rule_runs_on_the_parameters_device(name, monkeypatch):
    """The launch (and its stream) belong to the device of the group's parameters, not to the current one."""
    seen, inside = [], []

    class On:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            inside.append(self.device)

        def __exit__(self, *a):
            inside.pop()
    monkeypatch.setattr(_lib, "require_device", lambda *t: None)
    monkeypatch.setattr(_lib, "on", On)
    monkeypatch.setattr(optim, "stream", lambda: 0)
    monkeypatch.setattr(optim, "call", lambda f, *a, **k: seen.append((f, list(inside))))
    p = torch.nn.Parameter(torch.zeros(5))
    p.grad = torch.ones(5)
    o = getattr(optim, name)([p])
    o.step()
    assert seen == [("p2c_adam_multi_f32", [p.device])] and not inside
    q = torch.nn.Parameter(torch.zeros(3, device="meta"))
    q.grad = torch.ones(3, device="meta")
    o.add_param_group({"params": [q]})
    o.param_groups[0]["params"].append(q)
    with pytest.raises(RuntimeError, match="one device"):
        o.step()


def test_a_group_can_leave_muons_rule(monkeypatch):
    """A matrix that has a momentum and no moments yet takes Adam's rule from then on."""
    seen = []
    monkeypatch.setattr(_lib, "require_device", lambda *t: None)
    monkeypatch.setattr(_lib, "on", lambda d: _lib._HERE_ALREADY)
    monkeypatch.setattr(optim, "stream", lambda: 0)
    monkeypatch.setattr(optim, "call", lambda f, *a, **k: seen.append(f))
    p = torch.nn.Parameter(torch.zeros(5, 4))
    p.grad = torch.ones(5, 4)
    o = optim.Muon([p])
    o.state[p]["momentum_buffer"] = torch.zeros(5, 4)
    o.param_groups[0]["use_muon"] = False
    o.step()
    o.step()
    assert seen == ["p2c_adam_multi_f32"] * 2 and o.state[p]["step"] == 2 and set(o.state[p]) == {"momentum_buffer", "step", "exp_avg", "exp_avg_sq"}


@pytest.mark.parametrize("name", ["Adam", "Muon"])
def test_optimizers_can_be_copied_and_pickled(name):
    p = torch.nn.Parameter(torch.zeros(5, 4))
    o = getattr(optim, name)([p], lr=0.5)
    o._captured.append("a captured step's table")
    for c in (copy.deepcopy(o), pickle.loads(pickle.dumps(o))):
        assert type(c) is type(o) and c.param_groups[0]["lr"] == 0.5 and c._tables == {} and c._captured == []
        assert name == "Adam" or c._mats == {}
        c.param_groups[0]["params"][0].grad = torch.ones(5, 4)
        with pytest.raises(RuntimeError, match="no CPU path"):       # (as far as a step gets here)
            c.step()
    o._tables[0] = "old"
    o.load_state_dict(o.state_dict())
    assert o._tables == {} and o._captured


def test_requantising_softplus_refuses_a_small_beta():
    """Its epilogue holds the rows times 1.44 beta: below 0.7 a row in the normal range would leave it there (ops.linear_int8 takes the unfused form)."""
    L = _lib.lib()
    entry = lambda act, beta: L.p2c_int8_linear_requant(ONE, 64, ONE, ONE, ONE, None, None, 0, act, beta, 20.0, ONE, 64, ONE, 0, 8, 8, 64, None)  # noqa: E731
    assert entry(2, 100.0) == 0 and entry(2, 0.75) == 0 and entry(1, 0.01) == 0
    assert entry(2, 0.69) == -1 and entry(2, 0.01) == -1 and entry(2, float("nan")) == -1


def test_newton_schulz_refuses_an_infinite_eps():
    L = _lib.lib()
    co = ops.ns_coefficients(5, ops.NS_COEFFS)
    m = (_lib.NsMatrix * 1)()
    m[0].rows, m[0].cols, m[0].batch = 0, 4, 1
    for eps, rc in ((1e-7, 0), (1e-300, 0), (float("inf"), -1), (0.0, -1)):
        assert L.p2c_newton_schulz(m, 1, 0, 5, co, eps, ONE, 1 << 20, None) == rc
    with pytest.raises(ValueError, match="finite"):
        optim.Muon([torch.nn.Parameter(torch.zeros(4, 4))], eps=float("inf"))
    with pytest.raises(ValueError, match="finite"):
        ops.newton_schulz([torch.zeros(4, 4)], eps=float("inf"))


def test_newton_schulz_size_limits():
    L = _lib.lib()

    def need(r, c, batch=1):
        m = (_lib.NsMatrix * 1)()
        m[0].rows, m[0].cols, m[0].batch, m[0].src, m[0].dst = r, c, batch, 16, 16
        return L.p2c_newton_schulz_ws_bytes(m, 1)
    # padded sides, three images of X, two of the small side's square
    assert need(64, 1 << 23) >= 3 * 4 * 64 << 23 and need(1 << 23, 256) >= 3 * 4 * 256 << 23
    assert need(64, (1 << 23) + 1) == 0 and need(300, 1 << 23) == 0 and need(64, 200, (1 << 16) + 1) == 0 and need(64, 2000, 1 << 16) > 0
    for r, c in ((1, (1 << 23) + 1), (1 << 23, 257), ((1 << 31) + 7, 1)):
        with pytest.raises(ValueError, match="2\\^23"):
            ops.ns_check_size(r, c, "x")
    ops.ns_check_size(1 << 23, 256, "x")


@pytest.mark.parametrize("pc,im", [(True, True), (True, False), (False, True)])
def test_sketch_trainer_leaves_output_layers_to_adam(pc, im):
    """--optimizer muon: the backbone's heads and the sketch encoder's output layer keep Adam's rule, and a schedule of their group reaches them."""
    a = train_sketch.build_parser().parse_args(["--optimizer", "muon"])
    a.is_pc_train, a.is_im_train = pc, im
    model, enc = backbone.backbone(output_sizes=[3, 16]), sketch.PointNetEncoder(256, 2, with_normals=True)
    o = train_sketch.make_optimizer(a, model, enc)
    rule = {id(p): g["use_muon"] for g in o.param_groups for p in g["params"]}
    heads = [p for on, m in ((pc, model.fc2), (im, enc.fc)) if on for p in m.parameters()]
    assert heads and not any(rule[id(p)] for p in heads)
    others = [p for on, m in ((pc, model), (im, enc)) if on for p in m.parameters() if not any(p is h for h in heads)]
    assert all(rule[id(p)] for p in others) and len(rule) == len(heads) + len(others)
    assert [(g["source"], g["use_muon"]) for g in o.param_groups] == [(k, m) for k in range(pc + im) for m in (True, False)]
    assert [g["lr"] for g in o.param_groups] == [lr for on, lr in ((pc, a.learning_rate), (im, 0.001)) if on for _ in range(2)]


def test_settings_changed_after_construction_are_checked(monkeypatch):
    monkeypatch.setattr(_lib, "require_device", lambda *t: None)
    monkeypatch.setattr(_lib, "on", lambda d: _lib._HERE_ALREADY)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(optim, "stream", lambda: 0)
    monkeypatch.setattr(optim, "call", lambda f, *a, **k: None)
    p = torch.nn.Parameter(torch.zeros(5, 4))
    p.grad = torch.ones(5, 4)
    for key, bad in (("adjust", "spectrall"), ("ns_steps", 0), ("ns_coeffs", (9.0, 9.0, 9.0)), ("ns_steps", 12)):
        o = optim.Muon([p])
        o.step()
        o.param_groups[0][key] = bad
        with pytest.raises(ValueError):
            o.step()


def test_few_rows_refuse_columns_that_do_not_fit_the_workgroup():
    """The rows of a one-launch product lie in LDS, padded: K was checked, the padded width was not."""
    L = _lib.lib()
    few = lambda M, K, Kp: L.p2c_int8_linear_few(ONE, 0, 8, ONE, ONE, None, None, 0, 0, 1.0, 20.0, ONE, 8, 0, M, 8, K, Kp, None)  # noqa: E731
    flo = lambda M, K, Kp: L.p2c_int8_linear_float(ONE, 0, 8, ONE, ONE, None, None, 0, 0, 1.0, 20.0, ONE, 8, 0, M, 8, K, Kp, ONE, None)  # noqa: E731
    for f in (few, flo):
        assert f(4, 8, 2112) == -1 and f(4, 2048, 1 << 20) == -1
