"""Adam for the trainers (train_Point2Cyl_without_sketch.py:204: torch.optim.Adam(model.parameters(), lr) with torch's defaults).

torch's fused / foreach Adam hands every 65,536-element chunk of every tensor to one thread block: the backbone's 1.4 M
parameters in 123 tensors become ~140 blocks in two launches, 88 us per step on an MI355X whose 256 CUs could do the whole
update in a few microseconds.  Here the update of ALL tensors of a parameter group is ONE launch of
csrc/bn.hip:adam_multi_kernel with 1024-element work items (p2c_adam_multi_f32), driven by a device-resident table of
(param, grad, exp_avg, exp_avg_sq) pointers.  The table is rebuilt only when a gradient tensor moved (eager steps; under the HIP
graph the gradient tensors are static), never during a capture; a captured one is kept.  Same update rule and operation order as torch.optim.Adam (no weight decay, no amsgrad);
`param_groups`, `zero_grad`, `state_dict` keep torch's shapes so schedules that poke `param_groups[i]["lr"]` keep working.
"""
import ctypes

import torch

from . import _lib, ops
from ._lib import call, ptr, stream


class Adam(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8):
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps))
        self._tables, self._captured = {}, []

    def _key(self, ps):
        """Every pointer and size a table holds (after load_state_dict, or anything else that replaces exp_avg / exp_avg_sq, a cached table would otherwise
        keep pointing at the old, freed moment tensors, and after p.data = p.data[:k] at elements behind the parameter); None: there are no moments yet."""
        key = []
        try:
            for p in ps:
                st = self.state[p]
                key += p.data_ptr(), p.numel(), p.grad.data_ptr(), st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr()
        except KeyError:
            return None
        return key

    def _table(self, gi, ps):
        key = self._key(ps)
        cached = self._tables.get(gi)
        capturing = ps[0].is_cuda and torch.cuda.is_current_stream_capturing()
        if cached is not None and key is not None and cached[0] == key:
            if capturing and not any(cached is c for c in self._captured):
                self._captured.append(cached)          # the graph's replays read this table, also after an eager step with other gradients has replaced it
            return cached
        if capturing:       # (a copy from host memory that is gone, and zeroed moments, would be part of the graph)
            raise RuntimeError("point2cyl_amd.optim.%s: take one step with the same gradient tensors before capturing one" % type(self).__name__)
        dev = ps[0].device
        rows, numel, chunks = [], [], []
        for t, p in enumerate(ps):
            _lib.require_device(p, p.grad)
            if p.dtype != torch.float32 or not p.is_contiguous() or not p.grad.is_contiguous():
                raise RuntimeError("point2cyl_amd.optim.Adam takes contiguous fp32 parameters and gradients")
            if p.device != dev or p.grad.device != dev:
                raise RuntimeError("point2cyl_amd.optim.Adam: the parameters of a group are on one device (got %s and %s)" % (dev, p.device))
            st = self.state[p]
            if "exp_avg" not in st:        # (a matrix whose group left Muon's rule has its momentum here)
                st["step"] = 0
                st["exp_avg"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
            for s in (p.grad, st["exp_avg"], st["exp_avg_sq"]):
                if s.shape != p.shape or s.dtype != p.dtype or not s.is_contiguous():
                    raise RuntimeError("point2cyl_amd.optim.Adam: a gradient or moment of %s %s does not fit its parameter %s"
                                       % (s.dtype, tuple(s.shape), tuple(p.shape)))
            rows.append([p.data_ptr(), p.grad.data_ptr(), st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr()])
            numel.append(p.numel())
            chunks += [[t, c] for c in range((p.numel() + 1023) // 1024)]
        tab = torch.tensor(rows, dtype=torch.int64).to(dev, non_blocking=True)
        nel = torch.tensor(numel, dtype=torch.int64).to(dev, non_blocking=True)
        chk = torch.tensor(chunks, dtype=torch.int32).to(dev, non_blocking=True)
        cached = (self._key(ps), tab, nel, chk, len(chunks), ps)
        self._tables[gi] = cached
        return cached

    def __setstate__(self, state):         # copies, pickles and load_state_dict come through here; tables of captured steps stay with their optimizer
        super().__setstate__(state)
        self._tables = {}
        self.__dict__.setdefault("_captured", [])

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        self._tables = {}

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for gi, group in enumerate(self.param_groups):
            ps = [p for p in group["params"] if p.grad is not None]
            if ps:
                self._adam(gi, ps, group["lr"], group["betas"], group["eps"])
        return loss

    def _adam(self, gi, ps, lr, betas, eps):
        _lib.require_device(ps[0])
        with _lib.on(ps[0].device):
            _, tab, nel, chk, n_chunks, ps = self._table(gi, ps)
            for p in ps:
                self.state[p]["step"] += 1
            steps = {int(self.state[p]["step"]) for p in ps}
            if len(steps) != 1:     # one bias correction per launch: every tensor of the group must have taken the same number of updates
                raise RuntimeError("point2cyl_amd.optim.Adam: parameters of one group have different step counts %s (a parameter that first "
                                   "received a gradient later than the others); put it in its own param group" % sorted(steps))
            b1, b2 = betas
            call("p2c_adam_multi_f32", ptr(tab), ptr(nel), ptr(chk), n_chunks, float(lr), float(b1), float(b2), float(eps),
                 int(self.state[ps[0]]["step"]), stream())


class Muon(Adam):
    """Orthogonalised momentum for matrices, Adam for the rest.

    A parameter of two or more dimensions is a matrix (its first dimension against the others: a 1x1 convolution (Co, Ci, 1, 1) is Co x Ci):
        m <- momentum m + (1 - momentum) g;   u = (1 - momentum) g + momentum m with nesterov, else m
        p <- (1 - lr weight_decay) p - lr s newton_schulz(u)
    with s = 0.2 sqrt(max(rows, columns)) for adjust="rms" (an update of the size Adam's has: Adam's learning rates and schedules carry over) or
    sqrt(max(1, rows / columns)) for "spectral".  All matrices of a parameter group go through csrc/muon.hip together, 24 at a time: 17 launches
    (one if they all fit a workgroup each), momentum, norm, normalisation, decay and update included.  Vectors and scalars (biases, BatchNorm), and every parameter of a
    group with use_muon=False, take Adam's rule with the group's `betas` and `adam_eps` in one launch, without decay.

    fp32, contiguous; `param_groups`, `state_dict` keep torch's shapes (state: "momentum_buffer" for matrices, Adam's three for the others).  A step can
    be captured into a graph after one eager step has made the state - where vectors take part, with the same gradient tensors; its replays keep the learning
    rates (and Adam's step count) of the capture and need the optimizer's state, so the optimizer has to stay."""

    def __init__(self, params, lr=1e-3, momentum=0.95, nesterov=True, weight_decay=0.0, ns_steps=5, ns_coeffs=ops.NS_COEFFS, eps=1e-7, adjust="rms",
                 betas=(0.9, 0.999), adam_eps=1e-8, use_muon=True):
        torch.optim.Optimizer.__init__(self, params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, ns_steps=ns_steps,
                                                          ns_coeffs=ns_coeffs, eps=eps, adjust=adjust, betas=betas, adam_eps=adam_eps, use_muon=use_muon))
        self._tables, self._captured, self._mats = {}, [], {}

    @staticmethod
    def _check_group(g):
        if not 0.0 <= g["momentum"] < 1.0:
            raise ValueError("Muon: momentum = %r is outside [0, 1)" % (g["momentum"],))
        if g["adjust"] not in ("rms", "spectral"):
            raise ValueError("Muon: adjust %r is neither rms nor spectral" % (g["adjust"],))
        if not 0.0 < g["eps"] < float("inf"):
            raise ValueError("Muon: eps = %r has to be positive and finite" % (g["eps"],))
        ops.ns_coefficients(g["ns_steps"], g["ns_coeffs"])

    def __setstate__(self, state):
        super().__setstate__(state)
        self._mats = {}

    def add_param_group(self, param_group):
        self._check_group({**self.defaults, **param_group})
        super().add_param_group(param_group)
        self._mats = {}

    def _matrices(self, gi, ps, group):
        """Descriptors of the group's matrices, rebuilt when a tensor, the learning rate or the decay changed."""
        for p in ps:
            if "momentum_buffer" not in self.state[p]:
                if torch.cuda.is_current_stream_capturing():       # (the zeros would be part of the graph: every replay would start the momentum again)
                    raise RuntimeError("point2cyl_amd.optim.Muon: take one step before capturing one (a parameter has no momentum yet)")
                self.state[p]["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
        lr, wd, adjust = float(group["lr"]), float(group["weight_decay"]), group["adjust"]
        key = [lr, wd, adjust, group["ns_steps"], repr(group["ns_coeffs"])]
        for p in ps:
            d, m = p.grad, self.state[p]["momentum_buffer"]
            key += (p.data_ptr(), p.shape, p.stride(), d.data_ptr(), d.shape, d.stride(), m.data_ptr(), m.shape)
        hit = self._mats.get(gi)
        if hit is not None and hit[0] == key:
            return hit
        self._check_group(group)                   # (its settings may have been changed since it was added)
        dev = ps[0].device
        recs = []
        for p in ps:
            m = self.state[p]["momentum_buffer"]
            _lib.require_device(p, p.grad, m)
            for t in (p, p.grad, m):
                if t.dtype != torch.float32 or not t.is_contiguous() or t.shape != p.shape or t.device != dev:
                    raise RuntimeError("point2cyl_amd.optim.Muon takes contiguous fp32 parameters, gradients and momenta of one device (got %s %s on %s)"
                                       % (t.dtype, tuple(t.shape), t.device))
            r = p.shape[0]
            c = p.numel() // r if r else 0
            if not p.numel():
                continue
            ops.ns_check_size(r, c, "point2cyl_amd.optim.Muon")
            s = 0.2 * max(r, c) ** 0.5 if adjust == "rms" else max(1.0, r / c) ** 0.5
            recs.append(ops._NS_RECORD.pack(p.grad.data_ptr(), m.data_ptr(), p.data_ptr(), c, 1, 0, c, 1, 0, r, c, 1, lr * s, 1.0 - lr * wd))
        buf = ctypes.create_string_buffer(b"".join(recs), max(1, len(recs) * ops._NS_RECORD.size))
        mats = ctypes.cast(buf, ctypes.POINTER(_lib.NsMatrix))
        nb = _lib.lib().p2c_newton_schulz_ws_bytes(mats, len(recs)) if recs else 0
        hit = self._mats[gi] = (key, mats, len(recs), nb, ops.ns_coefficients(group["ns_steps"], group["ns_coeffs"]), buf)
        return hit

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for gi, group in enumerate(self.param_groups):
            ps = [p for p in group["params"] if p.grad is not None]
            mats = [p for p in ps if p.dim() >= 2] if group["use_muon"] else []
            rest = [p for p in ps if p.dim() < 2] if group["use_muon"] else ps
            if mats:
                _lib.require_device(*mats)
                with _lib.on(mats[0].device):
                    _, rec, n, nb, co, _ = self._matrices(gi, mats, group)
                    if n:
                        ws = torch.empty(max(nb, 16), dtype=torch.uint8, device=mats[0].device)        # (of this call: a captured step keeps its own)
                        call("p2c_muon_step_f32", rec, n, float(group["momentum"]), int(bool(group["nesterov"])), int(group["ns_steps"]), co,
                             float(group["eps"]), ptr(ws), ws.numel(), stream())
            if rest:
                self._adam(gi, rest, group["lr"], group["betas"], group["adam_eps"])
        return loss


def add_arguments(p):
    """The trainers' flags for the choice of the update rule."""
    p.add_argument("--optimizer", choices=("adam", "muon"), default="adam", help="muon: orthogonalised momentum for the weight matrices (optim.Muon), Adam "
                   "for biases, BatchNorm and the output heads; the learning rates mean the same")
    p.add_argument("--muon_momentum", type=float, default=0.95)
    p.add_argument("--weight_decay", type=float, default=0.0, help="decoupled decay of the matrices (--optimizer muon only)")


def from_arguments(a, groups, heads=()):
    """The trainers' optimizer from their flags: groups = [{"params": [...], "lr": ...}, ...]; heads: parameters of output layers, whose rows
    are separate regressions and not one operator - muon leaves them to Adam, in a group of their own behind the one they came from."""
    if a.optimizer == "adam":
        if a.weight_decay:
            raise SystemExit("--weight_decay belongs to --optimizer muon (the reference's Adam has none)")
        return Adam(groups)
    out, ids = [], {id(p) for p in heads}
    for k, g in enumerate(groups):                           # "source": a schedule of group k moves every part of it
        ps = list(g["params"])
        out.append({**g, "params": [p for p in ps if id(p) not in ids], "source": k})
        own = [p for p in ps if id(p) in ids]
        if own:
            out.append({**g, "params": own, "use_muon": False, "source": k})
    return Muon(out, momentum=a.muon_momentum, weight_decay=a.weight_decay)
