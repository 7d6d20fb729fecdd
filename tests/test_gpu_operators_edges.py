"""GPU: the dense-layer operators at the ends of what they accept: very many rows, very long matrices, large batches, extreme scales, optimizers that
are copied, shrunk or captured."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g, device="cuda")


@pytest.mark.parametrize("M,K,dtype", [((1 << 26) + 5, 3, torch.float32), ((1 << 24) + 3, 1025, torch.bfloat16)])
def test_quantize_more_rows_than_a_launch_holds(M, K, dtype):
    """Rows overlap in memory (row i starts at element i), so that the input stays small.  Rows around the launches' borders against the definition,
    and every row's scale."""
    from point2cyl_amd import _lib, ops
    most = _lib.lib().p2c_quantize_rows_at_once(K)
    assert M > most
    buf = torch.rand(M + K, device="cuda", dtype=torch.float32).to(dtype)
    x = buf.as_strided((M, K), (1, 1))
    r = ops.quantize_rows(x)
    assert r.shape == (M, K)
    for lo in sorted({0, most - 3, most, most // 2, *range(2 * most - 2, M - 4, most), M - 6}):
        if not 0 <= lo <= M - 6:
            continue
        v = x[lo:lo + 6].float()
        s = v.abs().amax(1) * torch.tensor(1.0 / 127.0, device="cuda")
        assert torch.equal(r.scale[lo:lo + 6], s), lo
        assert torch.equal(r.q[lo:lo + 6], torch.round(v.double() / s.double()[:, None]).to(torch.int8)), lo
        assert not r.store[lo:lo + 6, K:].any()
    assert bool((r.scale > 0).all())


def test_int8_row_counts_past_32_bits_are_refused():
    """The entries count rows in 32 bits: 2^32 + 5 rows must not become 5.  (Views that repeat one row: nothing of that size is allocated.)"""
    from point2cyl_amd import ops
    one = torch.ones(1, 1, device="cuda")
    w = ops.Int8Weight(one)
    for M in ((1 << 32) + 5, (1 << 31) + 5, (1 << 30) - 63):
        x = one.expand(M, 1)
        for f in (lambda: ops.linear_int8(x, w), lambda: ops.linear_int8(x, w, requantize=True), lambda: ops.quantize_rows(x), lambda: ops.linear_int8(x.view(1, M, 1), w)):
            with pytest.raises(ValueError, match="rows"):
                f()
    for N in ((1 << 20) + 1, (1 << 32) + 5):
        with pytest.raises(ValueError, match="channels|rows"):
            ops.Int8Weight(one.expand(N, 1))


NSC = (3.4445, -4.7750, 2.0315)


@pytest.mark.parametrize("shape", [(64, 128), (200, 60), (256, 1024), (12, 300)])
@pytest.mark.parametrize("kind", ["half", "fall8", "fall12"])
def test_newton_schulz_weak_rows_after_eight_steps(shape, kind):
    """Rows far below the others, brought up by the most steps that are accepted.  An operand's absolute floor of 2^-38 enters X through A, B (|b| + 2 |c| |A| + 1 <= 12.6 of
    them) and X itself: at most sqrt(m) 12.6 2^-38 |X| in a row's norm, m 12.6 2^-38 x 1.26 in the Frobenius norm, amplified by the steps that follow (sum of 3.4445^k).  Beside it
    the roundings of 32-bit arithmetic: four times what the plain 32-bit form makes of the same matrix."""
    from point2cyl_amd import ops
    m, n = shape
    f = {"half": torch.where(torch.arange(m) % 2 == 0, 1.0, 1e-9), "fall8": torch.logspace(0, -8, m), "fall12": torch.logspace(0, -12, m)}[kind].cuda()
    G = gen(31)(m, n) * f[:, None]

    def plain(dtype):
        X = (G.double() / (G.double().norm() + 1e-7)).to(dtype)
        X = X.t().contiguous() if m > n else X
        for _ in range(8):
            A = X @ X.t().contiguous()
            X = NSC[0] * X + (NSC[1] * A + NSC[2] * (A @ A)) @ X
        return X.t() if m > n else X
    want = plain(torch.float64)
    err = lambda o: (o.double() - want).norm().item()  # noqa: E731
    floor = min(m, n) * 12.6 * 1.26 * 2.0 ** -38 * sum(NSC[0] ** k for k in range(8))
    assert err(ops.newton_schulz(G, steps=8)) <= 4.0 * err(plain(torch.float32)) + floor
    assert floor <= 4e-5 * want.norm().item()


@pytest.mark.parametrize("use_muon", [True, False])
def test_a_parameter_that_shrank_is_refused(use_muon):
    """p.data = p.data[:k] keeps every address: the step must not go on with the sizes of the one before."""
    from point2cyl_amd import optim
    r = gen(32)
    for cls, kw in ((optim.Muon, dict(use_muon=use_muon)), (optim.Adam, {})):
        whole = r(64, 32)
        p = torch.nn.Parameter(whole)
        p.grad = r(64, 32)
        o = cls([dict(params=[p], **kw)], lr=0.01)
        o.step()
        grad, keep = p.grad, whole.clone()
        p.grad = None
        p.data = whole[:32]
        p.grad = grad[:32]
        with pytest.raises(RuntimeError, match="fit|takes"):
            o.step()
        assert torch.equal(whole, keep)
        # with moments of its size the shorter parameter is stepped, what lies behind it stays
        o.state[p].clear()
        o.step()
        assert torch.equal(whole[32:], keep[32:]) and not torch.equal(whole[:32], keep[:32])


@pytest.mark.parametrize("name", ["Muon", "Adam"])
def test_captured_step_survives_steps_with_other_gradients(name):
    """Vectors go by a table in device memory: the one a graph was captured with stays when an eager step makes another."""
    from point2cyl_amd import optim
    r = gen(33)
    make = lambda ps: getattr(optim, name)(ps, lr=0.01)  # noqa: E731
    base = [r(300), r(64, 48), r(5)]
    ps, qs = ([torch.nn.Parameter(t.clone()) for t in base] for _ in range(2))
    g0, g1 = ([r(*t.shape) for t in base] for _ in range(2))
    o, o2 = make(ps), make(qs)
    give = lambda ts, gs: [setattr(t, "grad", g) for t, g in zip(ts, gs)]  # noqa: E731
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        give(ps, g0), o.step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            o.step()
        moved = [g.clone() for g in g0]
        give(ps, moved)
        with pytest.raises(RuntimeError, match="same gradient tensors"), torch.cuda.graph(torch.cuda.CUDAGraph(), stream=st):
            make(ps).step() if name == "Adam" else o.step()
        give(ps, g0)
    torch.cuda.synchronize()
    counts = {p: o.state[p]["step"] for p in ps if "step" in o.state[p]}
    step = max(counts.values())                                  # of the capture: what every replay takes for the bias correction
    give(qs, g0), o2.step()

    def replayed():
        for q in qs:
            if "step" in o2.state[q]:
                o2.state[q]["step"] = step - 1
        give(qs, g0), o2.step()
    for k in range(4):
        graph.replay(), replayed()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs)), k
        for t, oo in ((ps, o), (qs, o2)):                         # an eager step with other gradient tensors
            for p in t:
                if "step" in oo.state[p]:
                    oo.state[p]["step"] = 10 + k
            give(t, g1), oo.step()
        junk = [torch.full((n,), -1, dtype=torch.int64, device="cuda") for n in (8, 16, 64, 512, 4096) for _ in range(20)]
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs)), k
        del junk


@pytest.mark.parametrize("name", ["Muon", "Adam"])
def test_a_copied_optimizer_goes_on_alone(name):
    from point2cyl_amd import optim
    r = gen(34)
    ps = [torch.nn.Parameter(r(60, 40)), torch.nn.Parameter(r(7))]
    o = getattr(optim, name)(ps, lr=0.01)
    gs = [[r(*p.shape) for p in ps] for _ in range(4)]

    def steps(opt, some):
        for g in some:
            for p, d in zip(opt.param_groups[0]["params"], g):
                p.grad = d.clone()
            opt.step()
    steps(o, gs[:2])
    c = copy.deepcopy(o)
    keep = [p.detach().clone() for p in ps]
    steps(c, gs[2:])
    assert all(torch.equal(p, k) for p, k in zip(ps, keep))
    steps(o, gs[2:])
    assert all(torch.equal(p, q) and not torch.equal(p, k) for p, q, k in zip(ps, c.param_groups[0]["params"], keep))


@pytest.mark.parametrize("beta", [0.01, 0.5, 0.75, 1.0, 100.0])
def test_requantised_softplus_far_below_zero(beta):
    """Arguments z with beta z from -80 to -86: values of e^(beta z) / beta, down to 2^-124 / beta, next to the end of the range.  The rows given back are within half a quantum of the
    floats (plus their relative error: 2^-22 beta |z| on either side), rows below 2^-119 are zero."""
    from point2cyl_amd import ops
    r = gen(35)
    M, K, N = 70, 64, 40
    w = ops.Int8Weight(1e-3 * r(N, K) / beta, torch.full((N,), -80.0 / beta, device="cuda"))
    x = r(M, K)
    add = -torch.linspace(0, 6, M, device="cuda")[:, None].expand(M, N).contiguous() / beta
    y = ops.linear_int8(x, w, act="softplus", beta=beta, add=add)
    h = ops.linear_int8(x, w, act="softplus", beta=beta, add=add, requantize=True)
    top = y.abs().amax(1)
    live = top > 2.0 ** -118
    assert (h.scale[live] > 0).all() and (h.scale[top < 2.0 ** -120] == 0).all()
    assert bool(live.any()) == (beta < 100.0)                    # (e^-80 / 100 = 1.8e-37 is below 2^-119 = 1.5e-36 already)
    s = h.scale.double()[:, None]
    off = (h.q.double() * s - y.double()).abs()
    assert (off <= 0.5001 * s + 2.0 ** -21 * 87 * y.double())[live].all()
    assert (h.q.abs().amax(1) >= 126)[live].all() and not h.q[h.scale == 0].any()


@pytest.mark.parametrize("shape", [(5, 70), (16, 16), (80, 90), (300, 200)])
@pytest.mark.parametrize("eps", [1e-30, 1e-80, 1e-160, 1e-310])
def test_newton_schulz_zero_matrix_and_a_tiny_eps(shape, eps):
    """Every kernel: zeros stay zeros and do not touch their neighbours; the smallest matrices that are not zero go by the formula (where eps outweighs their norm they stay small).
    Bound: 2^-20 of every step's result and the operands' floor, carried on by at most 3.4445 a step (as in the other tests of these kernels)."""
    from point2cyl_amd import ops
    G = torch.zeros(3, *shape, device="cuda")
    G[1] = gen(36)(*shape)
    G[2] = G[1].sign() * 2.0 ** -140                        # (subnormal)
    o = ops.newton_schulz(G, eps=eps)
    assert not o[0].any()
    m = min(shape)
    for k in (1, 2):
        X = G[k].double()
        X = X / (X.norm() + eps)
        X = X.t().contiguous() if shape[0] > shape[1] else X
        bound = 2.0 ** -20 * X.norm().item()
        for _ in range(5):
            A = X @ X.t().contiguous()
            X = NSC[0] * X + (NSC[1] * A + NSC[2] * (A @ A)) @ X
            bound = NSC[0] * bound + 2.0 ** -20 * X.norm().item() + m * 12.6 * 1.26 * 2.0 ** -38
        X = X.t() if shape[0] > shape[1] else X
        assert (o[k].double() - X).norm().item() <= bound, k


def ns64(G):
    """-> (result in 64 bits, bound on the Frobenius error: 2^-20 of every step's result, carried on, and half a unit of the type)"""
    X = G.double()
    X = X / (X.norm() + 1e-7)
    X = X.t() if G.shape[0] > G.shape[1] else X
    bound = 2.0 ** -20 * X.norm().item()
    for _ in range(5):
        A = X @ X.t().contiguous()
        X = NSC[0] * X + (NSC[1] * A + NSC[2] * (A @ A)) @ X.contiguous()
        bound = NSC[0] * bound + 2.0 ** -20 * X.norm().item()
    return X.t() if G.shape[0] > G.shape[1] else X, bound + {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[G.dtype] * X.norm().item()


@pytest.mark.parametrize("shape,dtype", [((70000, 3, 3), torch.float32), ((65537, 20, 24), torch.bfloat16), ((2, 131075, 6), torch.float32)])
def test_newton_schulz_batches_larger_than_a_descriptor(shape, dtype):
    from point2cyl_amd import ops
    G = gen(37)(*shape).to(dtype)
    o = ops.newton_schulz(G)
    for k in {0, 1, 65535, 65536, shape[0] - 1}:
        if k < shape[0]:
            want, bound = ns64(G[k])
            assert (o[k].double() - want).norm().item() <= bound, k
    v = G.transpose(-1, -2)
    lo = max(0, shape[0] - 5)
    assert torch.equal(ops.newton_schulz(v)[lo:], ops.newton_schulz(v[lo:]))


@pytest.mark.parametrize("shape,dtype", [((3, 2000000), torch.float32), ((1200000, 64), torch.bfloat16), ((20, (1 << 20) + 33), torch.float32)])
def test_newton_schulz_and_muon_on_very_long_matrices(shape, dtype):
    from point2cyl_amd import ops, optim
    G = gen(38)(*shape).to(dtype)
    want, bound = ns64(G)
    assert (ops.newton_schulz(G).double() - want).norm().item() <= bound
    if dtype == torch.float32:
        p = torch.nn.Parameter(torch.zeros_like(G))
        p.grad = G
        optim.Muon([p], lr=1.0, momentum=0.0, adjust="spectral").step()
        scale = max(1.0, shape[0] / shape[1]) ** 0.5
        assert (p.detach().double() + scale * want).norm().item() <= scale * bound


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_quantized_rows_by_what_they_stand_for(dtype):
    """Without the kernel's own expression for the scale: within a unit of max / 127 (one rounding of 1 / 127 and one of the product), the largest element 127, and every element within half
    a step (the quotients are rounded exactly)."""
    from point2cyl_amd import ops
    r = gen(39)
    M, K = 4000, 200
    mags = torch.logspace(-30 if dtype != torch.float16 else -3, 30 if dtype != torch.float16 else 3, M, device="cuda")[:, None]
    x = (r(M, K).clamp(-5, 5) * torch.exp(r(M, 1)) * mags).to(dtype)
    h = ops.quantize_rows(x)
    v, s = x.double(), h.scale.double()
    top = v.abs().amax(1)
    assert ((s - top / 127.0).abs() <= 2.0 ** -23 * top / 127.0).all()
    assert (h.q.abs().amax(1) == 127).all() and int(h.q.min()) >= -127
    assert ((h.q.double() * s[:, None] - v).abs() <= 0.5 * s[:, None] * (1.0 + 2.0 ** -30)).all()


@pytest.mark.parametrize("kind", ["gauss", "lowrank", "decay"])
@pytest.mark.parametrize("shapes,batch", [([(128, 128)], 0), ([(50, 256)], 0), ([(200, 1000)], 0), ([(1024, 512)], 0), ([(700, 500)], 12), ([(12, 400)], 0),
                                          ([(8, 512), (16, 500), (3, 128), (512, 512)], 0), ([(8, 120), (60, 90), (1, 100)], 0)])
def test_newton_schulz_is_as_exact_as_32_bits(shapes, batch, kind):
    """Operands of 22 bits at least, products and sums of 32-bit size: at most four times (two bits) the error that plain 32-bit arithmetic makes of the same matrix, beside two units of
    rounding of the result itself."""
    from point2cyl_amd import ops
    r = gen(40)

    def make(m, n):
        if kind == "lowrank":
            k = max(1, min(m, n) // 16)
            return r(m, k) @ r(k, n) / k ** 0.5 + 0.3 * r(m, n)
        return r(m, n) * (torch.logspace(0, -3, m, device="cuda")[:, None] if kind == "decay" else 1.0)

    def plain(G, dtype):
        X = (G.double() / (G.double().norm() + 1e-7)).to(dtype)
        X = X.t().contiguous() if G.shape[0] > G.shape[1] else X
        for _ in range(5):
            A = X @ X.t().contiguous()
            X = NSC[0] * X + (NSC[1] * A + NSC[2] * (A @ A)) @ X
        return X.t() if G.shape[0] > G.shape[1] else X
    Gs = [make(*shapes[0]) for _ in range(batch)] if batch else [make(*s) for s in shapes]
    os_ = list(ops.newton_schulz(torch.stack(Gs))) if batch else ops.newton_schulz(Gs)
    for G, o in zip(Gs, os_):
        want = plain(G, torch.float64)
        err = lambda x: (x.double() - want).norm().item()  # noqa: E731
        assert err(o) <= 4.0 * err(plain(G, torch.float32)) + 2.0 ** -22 * want.norm().item(), tuple(G.shape)


def test_newton_schulz_refuses_large_matrices_before_it_allocates():
    from point2cyl_amd import ops
    one = torch.ones(1, 1, device="cuda")
    before = torch.cuda.max_memory_allocated()
    for shape in ((1 << 24, 1 << 16), ((1 << 23) + 1, 2), (1 << 32, 1), (1 << 16, (1 << 15) + 1)):
        for G in (one.expand(*shape), one.expand(2, *shape), [one, one.expand(*shape)]):
            with pytest.raises(ValueError, match="2\\^23"):
                ops.newton_schulz(G)
    assert torch.cuda.max_memory_allocated() < before + (1 << 20)
    assert ops.newton_schulz(one.expand(1, 1)[:0].expand(0, 1 << 24)).shape == (0, 1 << 24)


def test_int8_decoder_runs_on_its_rows_device(monkeypatch):
    """Every launch of the 8-bit decoder, the 32-bit ones among them, is made with the rows' device current; rows elsewhere than the weights are refused."""
    from point2cyl_amd import _lib, implicit
    net = implicit.ImplicitNet(d_in=6, dims=[64, 40, 48], skip_in=(2,), geometric_init=True, radius_init=1, beta=100).cuda()
    q = implicit.Int8ImplicitNet(net)
    x = gen(41)(300, 6)
    want, inside, products, on, prod = q(x), [], [], _lib.on, implicit._prod_nt

    class On:
        def __init__(self, device):
            self.device, self.real = device, on(device)

        def __enter__(self):
            inside.append(self.device)
            self.real.__enter__()

        def __exit__(self, *a):
            inside.pop()
            return self.real.__exit__(*a)
    monkeypatch.setattr(_lib, "on", On)
    monkeypatch.setattr(implicit, "_prod_nt", lambda *a, **k: (products.append(list(inside)), prod(*a, **k))[1])
    assert torch.equal(q(x), want) and len(products) == 3 and all(p == [x.device] for p in products)
    q.first = tuple(t.cpu() for t in q.first)
    with pytest.raises(ValueError, match="weights on"):
        q(x)


def test_int8_products_of_rows_past_32_bit_offsets():
    """2^26 + 700 rows of 64 bytes: the last ones lie beyond 2^32 bytes.  They are the numbers that a call on them alone gives (a row's sums are exact, its scaling its own)."""
    from point2cyl_amd import ops
    M, K, N = (1 << 26) + 700, 5, 6
    r = gen(42)
    x = r(M + K).as_strided((M, K), (1, 1))
    w = ops.Int8Weight(r(N, K), r(N))
    tail, mid = slice(M - 700, M), slice((1 << 25) - 300, (1 << 25) + 300)
    y = ops.linear_int8(x, w, out_dtype=torch.bfloat16)
    for part in (tail, mid):
        assert torch.equal(y[part], ops.linear_int8(x[part], w, out_dtype=torch.bfloat16))
    del y
    h = ops.linear_int8(x, w, act="relu", requantize=True)
    for part in (tail, mid):
        p = ops.linear_int8(x[part], w, act="relu", requantize=True)
        assert torch.equal(h.q[part], p.q) and torch.equal(h.scale[part], p.scale)
    d = h.dequantize(torch.float16)
    assert torch.equal(d[mid], p.dequantize(torch.float16))
    assert torch.equal(d[tail], ops.linear_int8(x[tail], w, act="relu", requantize=True).dequantize(torch.float16))
