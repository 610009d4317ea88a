"""GPU parity: the routed-experts operators (choice, plan, products, join, their gradients) against the 64-bit oracle.

Tolerances.  u = 2^-24 is half a step of fp32, h half a step of the 16-bit type (fp16 2^-11, bf16 2^-8).  A sum of n products in
32 bits is off by at most (n + 2) * 2 * u * sum |terms| whatever its order (2 u a step: the matrix instructions may cut instead
of rounding); its one rounding to 16 bits adds h * |result|, and fp16 below 2^-14 half of its smallest step, 2^-25."""
import numpy as np
import pytest
import torch

from oracle import experts as ox

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=["native", "functions"])
def way(request, monkeypatch):
    """Every test runs both ways through the host: the native nodes that plain arguments take, and the Functions for all others."""
    from nersemble_amd import experts as X
    if request.param == "functions":
        class Never:
            def __getattr__(self, name):
                return lambda *args: None
        monkeypatch.setattr(X, "_fast", Never())
    return request.param

U = 2.0 ** -24
HALF = {torch.float16: (2.0 ** -11, 2.0 ** -25), torch.bfloat16: (2.0 ** -8, 2.0 ** -130)}
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _f64(t):
    return t.detach().double().cpu().numpy()


def _close(got, want, tol, what):
    got = _f64(got) if isinstance(got, torch.Tensor) else got
    off = np.abs(got - want)
    worst = np.max(np.where(tol > 0, off / np.where(tol > 0, tol, 1), np.where(off > 0, np.inf, 0))) if off.size else 0.0
    assert np.isfinite(got).all() and worst <= 1.0, f"{what}: {worst:.3g} of the tolerance, largest error {off.max():.3g}"


# ---------------------------------------------------------------------------------------------------------------------
# choice
# ---------------------------------------------------------------------------------------------------------------------
def _route_tol(x, w, k):
    """Relative: x - max is off by u of its size (at most the logits' span), exp by 2 steps, sums and divisions by u a term."""
    span = np.nanmax(np.where(np.isfinite(x), np.abs(x), 0.0), initial=0.0) * 2
    return (span + k + 10) * 2 * U * np.abs(w) + 1e-37


ROUTES = [
    # E, k, scores, bias, groups, top_groups, group_top, renorm, scale
    (1, 1, "softmax", False, 1, 1, 1, True, 1.0),
    (2, 1, "softmax", False, 1, 1, 1, False, 1.0),
    (3, 3, "sigmoid", False, 1, 1, 1, True, 2.5),
    (16, 2, "softmax", False, 1, 1, 1, True, 1.0),
    (32, 2, "softmax", True, 1, 1, 1, False, 1.0),
    (61, 7, "sigmoid", True, 1, 1, 1, True, 1.0),
    (64, 6, "softmax", False, 1, 1, 1, False, 16.0),
    (256, 8, "sigmoid", True, 8, 4, 2, True, 2.5),
    (160, 6, "softmax", False, 8, 3, 1, False, 16.0),
    (20, 4, "sigmoid", True, 4, 2, 2, True, 1.0),
    (24, 5, "softmax", True, 3, 2, 1, True, 1.0),
    (50, 3, "sigmoid", False, 5, 2, 2, False, 1.0),
    (512, 16, "softmax", True, 1, 1, 1, True, 1.0),
    (495, 9, "sigmoid", True, 33, 5, 2, True, 1.0),
]


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("cfg", ROUTES, ids=lambda c: f"E{c[0]}k{c[1]}{c[2][:3]}{'b' if c[3] else ''}g{c[4]}")
def test_route(cfg, dtype, cuda):
    from nersemble_amd import experts as X
    E, k, sc, has_bias, G, tg, gt, renorm, scale = cfg
    for T in (1, 7, 130):
        rng = np.random.default_rng(E * 7 + T)
        x = torch.from_numpy((rng.standard_normal((T, E)) * 2).astype(np.float32)).to(DT[dtype])
        bias = torch.from_numpy((rng.standard_normal(E) * 0.1).astype(np.float32)) if has_bias else None
        xd = x.to(cuda).requires_grad_(True)
        w, c = X.route_experts(xd, k, scores=sc, bias=None if bias is None else bias.to(cuda), n_groups=G, top_groups=tg,
                               group_top=gt, renormalise=renorm, scale=scale)
        assert w.dtype == torch.float32 and c.dtype == torch.int32 and w.shape == c.shape == (T, k)
        x64 = _f64(x)
        ww, wc = ox.route(x64, k, sc == "sigmoid", None if bias is None else _f64(bias), G, tg, gt, renorm, scale)
        assert np.array_equal(c.cpu().numpy(), wc)
        _close(w, ww, _route_tol(x64, ww, k), "weights")
        g = rng.standard_normal((T, k)).astype(np.float32)
        (d,) = torch.autograd.grad(w, [xd], torch.from_numpy(g).to(cuda))
        want = ox.route_bwd(x64, ww, wc, g, sc == "sigmoid", renorm, scale)
        # every term of a gradient is a weight (or score) times g: off relatively as the weights are, plus the sum's own steps
        size = np.zeros_like(x64)
        total = (np.abs(g) * ww).sum(1, keepdims=True)
        for j in range(k):
            size[np.arange(T), wc[:, j]] += ww[:, j] * (np.abs(g[:, j]) + (total[:, 0] / scale if renorm else 0.0))
        if sc == "softmax" and not renorm:
            size += ox.scores(x64, False) * total
        tol = 3 * _route_tol(x64, size, k)
        if dtype != "fp32":
            h, tiny = HALF[DT[dtype]]
            tol = tol + h * np.abs(want) + tiny
        assert d.dtype == DT[dtype]
        _close(d, want, tol, "dlogits")


def test_route_gradient_against_differences(cuda):
    """The gradient against central differences of the forward (16 experts whose choice does not change under the step)."""
    from nersemble_amd import experts as X
    rng = np.random.default_rng(0)
    for sc, renorm in (("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)):
        x = np.stack([rng.permutation(16) * 0.25 for _ in range(4)])            # gaps of 0.25
        g = rng.standard_normal((4, 3))
        xd = torch.tensor(x, dtype=torch.float32, device=cuda, requires_grad=True)
        w, _ = X.route_experts(xd, 3, scores=sc, renormalise=renorm)
        (d,) = torch.autograd.grad(w, [xd], torch.tensor(g, dtype=torch.float32, device=cuda))
        step = 2.0 ** -6
        for e in range(16):
            hi, lo = x.copy(), x.copy()
            hi[:, e] += step
            lo[:, e] -= step
            f = [(_f64(X.route_experts(torch.tensor(v, dtype=torch.float32, device=cuda), 3, scores=sc, renormalise=renorm)[0]) * g).sum(1)
                 for v in (hi, lo)]
            diff = (f[0] - f[1]) / (2 * step)
            # third derivative of a softmax weight <= 1: step^2 / 6 * sum|g|; rounding of the forward: 16 u * sum|g| / step
            tol = (step ** 2 / 6 + 32 * U / step) * np.abs(g).sum(1)
            assert (np.abs(_f64(d)[:, e] - diff) <= tol).all()


def test_route_rows_without_experts_and_odd_values(cuda):
    from nersemble_amd import experts as X
    inf, nan = float("inf"), float("nan")
    rows = np.array([[0.5, 1.0, -1.0, 2.0], [-inf, -inf, -inf, -inf], [-inf, 3.0, -inf, -inf], [nan, 1.0, 2.0, 3.0],
                     [inf, 1.0, 2.0, 3.0], [1.0, 1.0, 1.0, 1.0], [-200.0, -201.0, -300.0, -250.0], [0.0, -0.0, 0.0, -inf]], np.float32)
    lowest = np.finfo(np.float32).min
    rows = np.concatenate([rows, np.full((1, 4), lowest, np.float32)])
    sel = np.ones(len(rows), np.uint8)
    for sc in ("softmax", "sigmoid"):
        for bias in (None, np.array([0.0, 0.125, 0.0, 0.0], np.float32)):
            for renorm in (True, False):
                for selector in (None, sel * (np.arange(len(rows)) % 3 != 0)):
                    xd = torch.from_numpy(rows).to(cuda).requires_grad_(True)
                    w, c = X.route_experts(xd, 2, scores=sc, renormalise=renorm, bias=None if bias is None else torch.from_numpy(bias).to(cuda),
                                           selector=None if selector is None else torch.from_numpy(selector.astype(np.uint8)).to(cuda))
                    ww, wc = ox.route(rows, 2, sc == "sigmoid", bias, renormalise=renorm, selector=selector)
                    assert np.array_equal(c.cpu().numpy(), wc), (sc, renorm)
                    got = _f64(w)
                    assert np.array_equal(np.isnan(got), np.isnan(ww))
                    # (a span of 100 in the sixth row; the last one's scores are equal or 0)
                    assert np.allclose(got, ww, rtol=(800 + 12) * 2 * U, atol=1e-37, equal_nan=True)
                    (d,) = torch.autograd.grad(w, [xd], torch.ones_like(w))
                    d = _f64(d)
                    fine = ~np.isnan(ww).any(1)
                    assert np.isfinite(d[fine]).all() and (d[(wc < 0).all(1)] == 0).all()


def test_route_equal_values_go_by_index(cuda):
    from nersemble_amd import experts as X
    x = torch.zeros((5, 256), device=cuda, dtype=torch.bfloat16)
    x[1, 100:] = 1
    for bias in (None, torch.zeros(256, device=cuda)):
        _, c = X.route_experts(x, 8, bias=bias)
        assert c[0].tolist() == list(range(8)) and c[1].tolist() == list(range(100, 108))
        _, c = X.route_experts(x, 8, bias=bias, n_groups=8, top_groups=2, group_top=2)
        # (experts 100 .. 127 are in group 3, whose two best are as good as those of the groups behind it)
        assert c[0].tolist() == list(range(8)) and c[1].tolist() == list(range(100, 108))
        x[2, 127:] = 1                                        # group 3 has one such expert only: 4 and 5 come before it
        _, c = X.route_experts(x, 8, bias=bias, n_groups=8, top_groups=2, group_top=2)
        assert c[2].tolist() == list(range(128, 136))


@pytest.mark.parametrize("layout", ["strided", "transposed", "offset", "one_row"])
def test_route_layouts(layout, cuda):
    from nersemble_amd import experts as X
    g = torch.Generator(device=cuda).manual_seed(1)
    base = torch.randn((40, 24), generator=g, device=cuda)
    x = {"strided": torch.randn((40, 100), generator=g, device=cuda)[:, 3:27], "transposed": torch.randn((24, 40), generator=g, device=cuda).t(),
         "offset": torch.randn(40 * 24 + 1, generator=g, device=cuda)[1:].view(40, 24), "one_row": base[3:4].expand(1, 24)}[layout]
    x = x.requires_grad_(True)
    y = x.detach().contiguous().clone().requires_grad_(True)
    wa, ca = X.route_experts(x, 3)
    wb, cb = X.route_experts(y, 3)
    assert torch.equal(wa, wb) and torch.equal(ca, cb)
    go = torch.randn(wa.shape, generator=g, device=cuda)
    assert torch.equal(torch.autograd.grad(wa, [x], go)[0], torch.autograd.grad(wb, [y], go)[0])


# ---------------------------------------------------------------------------------------------------------------------
# plan
# ---------------------------------------------------------------------------------------------------------------------
def _check_plan(plan, want):
    for got, w in zip((plan.offsets, plan.rows, plan.positions), want):
        assert got.dtype == torch.int32 and np.array_equal(got.cpu().numpy(), w)


@pytest.mark.parametrize("T,k,E", [(0, 2, 4), (1, 1, 1), (1, 8, 64), (63, 1, 3), (257, 3, 512), (1000, 2, 16), (4096, 2, 16),
                                   (3001, 7, 61), (20000, 8, 256), (300001, 2, 33), (150001, 3, 30), (100000, 8, 200), (1200000, 2, 7)])
def test_plan(T, k, E, cuda):
    from nersemble_amd import experts as X
    rng = np.random.default_rng(T + E)
    c = rng.integers(0, E, (T, k)).astype(np.int32)
    c[rng.random(T) < 0.2] = -1
    if T > 10:
        c[5, 0], c[6, 0], c[7, :] = E, 2 ** 31 - 1, -2 ** 31          # outside the experts
    _check_plan(X.expert_plan(torch.from_numpy(c).to(cuda), E), ox.plan(np.where((c >= 0) & (c < E), c, -1), E))


def test_plan_of_one_expert_and_of_none(cuda):
    from nersemble_amd import experts as X
    for T in (5, 5000, 200000):
        for fill in (-1, 0, 7):
            c = np.full((T, 2), fill, np.int32)
            _check_plan(X.expert_plan(torch.from_numpy(c).to(cuda), 8), ox.plan(c, 8))


# ---------------------------------------------------------------------------------------------------------------------
# products and join
# ---------------------------------------------------------------------------------------------------------------------
def _chosen(rng, T, k, E, masked, spread=None):
    """Distinct experts per row; ``spread``: only that many experts are ever chosen (the others stay without rows)."""
    use = min(E, spread or E)
    c = np.argsort(rng.random((T, use)), axis=1)[:, :k].astype(np.int32)
    c[rng.random(T) < masked] = -1
    return c


def _linear_case(cuda, T, k, E, K, N, dtype, gather, relu, master, masked, spread=None, seed=0):
    from nersemble_amd import experts as X
    rng = np.random.default_rng(seed + T + K + N)
    dt = DT[dtype]
    chosen = _chosen(rng, T, k, E, masked, spread)
    plan = X.expert_plan(torch.from_numpy(chosen).to(cuda), E)
    offsets, rows, positions = ox.plan(chosen, E)
    R = T * k
    x = torch.from_numpy(rng.standard_normal((T if gather else R, K)).astype(np.float32)).to(dt)
    wf = torch.from_numpy((rng.standard_normal((E, N, K)) / np.sqrt(K)).astype(np.float32))
    w16 = wf.to(dt)
    dy = torch.from_numpy(rng.standard_normal((R, N)).astype(np.float32)).to(dt)
    xd = x.to(cuda).requires_grad_(True)
    wd = (wf if master else w16).to(cuda).requires_grad_(True)
    y = X.expert_linear(xd, wd, plan, gather=gather, relu=relu)
    h, tiny = HALF[dt]
    want, mag = ox.linear(_f64(x), _f64(w16), offsets, rows, k, gather, relu)
    assert y.dtype == dt and y.shape == (R, N)
    _close(y, want, h * np.abs(want) + tiny + (K + 2) * 2 * U * mag, "y")
    with torch.no_grad():
        assert torch.equal(X.expert_linear(xd, wd, plan, gather=gather, relu=relu), y)
    dx, dw = torch.autograd.grad(y, [xd, wd], dy.to(cuda))
    assert dx.dtype == dt and dx.shape == x.shape and dw.dtype == wd.dtype
    dz = np.where(_f64(y) > 0, _f64(dy), 0.0) if relu else _f64(dy)     # (a value next to 0 falls where the kernel's fell)
    wx, mx, ww, mw = ox.linear_bwd(_f64(x), _f64(w16), offsets, rows, k, gather, dz)
    n_e = np.diff(offsets)[:, None, None]
    tw = (n_e + 2 + 64) * 2 * U * mw + ((h * np.abs(ww) + tiny) if not master else 0)
    _close(dw, ww, tw, "dw")
    tx = h * np.abs(wx) + tiny + (N + 2) * 2 * U * mx                    # in the plan's order
    if gather:
        one = np.ones((T, k))
        tx = ox.combine(tx, one, positions)[0]
        wx, _ = ox.combine(wx, one, positions)
        tx = tx + h * np.abs(wx) + tiny
    _close(dx, wx, tx * (1 + 4 * U * k), "dx")


WIDTHS = [(8, 8), (16, 8), (32, 64), (64, 16), (64, 64), (40, 24), (176, 128), (128, 128), (72, 200), (264, 520), (1024, 136)]


@pytest.mark.parametrize("K,N", WIDTHS)
@pytest.mark.parametrize("dtype,gather,relu,master", [("fp16", True, True, False), ("bf16", True, False, False), ("fp16", False, False, True),
                                                      ("bf16", False, True, True)])
def test_linear_widths(K, N, dtype, gather, relu, master, cuda):
    _linear_case(cuda, 211, 2, 5, K, N, dtype, gather, relu, master, 0.1)


@pytest.mark.parametrize("T,k,E,spread", [(1, 1, 1, None), (1, 2, 8, None), (4, 3, 64, None), (17, 1, 3, None), (64, 2, 2, None), (65, 4, 9, 5),
                                          (300, 1, 40, 7), (1025, 3, 7, None), (5000, 2, 16, None), (2600, 1, 1, None)])
@pytest.mark.parametrize("masked", [0.0, 0.4, 1.0])
def test_linear_rows(T, k, E, spread, masked, cuda):
    _linear_case(cuda, T, k, E, 72, 48, "fp16", True, True, False, masked, spread, seed=1)
    _linear_case(cuda, T, k, E, 48, 72, "bf16", False, False, True, masked, spread, seed=2)


@pytest.mark.parametrize("K,N,T,k,E", [(512, 768, 700, 2, 6), (1024, 512, 1500, 1, 3), (32, 64, 30000, 2, 16), (64, 16, 30000, 2, 5),
                                       (2048, 1024, 5, 4, 64), (1024, 2048, 40, 4, 32)])
def test_linear_larger(K, N, T, k, E, cuda):
    _linear_case(cuda, T, k, E, K, N, "bf16", True, False, False, 0.1)
    _linear_case(cuda, T, k, E, K, N, "fp16", False, True, False, 0.0)


@pytest.mark.parametrize("K,N", [(8, 8), (8, 64), (16, 32), (32, 64), (64, 16), (64, 32), (40, 24), (24, 48), (64, 64)])
@pytest.mark.parametrize("gather,relu,master", [(True, True, False), (True, False, True), (False, True, True), (False, False, False)])
def test_linear_narrow_layers(K, N, gather, relu, master, cuda):
    """Rows enough that both gradients of a narrow layer are made at once; segments of other lengths than its steps."""
    _linear_case(cuda, 2501, 2, 7, K, N, "fp16", gather, relu, master, 0.2, seed=3)
    _linear_case(cuda, 9001, 3, 3, K, N, "bf16", gather, relu, master, 0.0, 3, seed=4)


def test_linear_row_of_infinities_stays_in_its_row(cuda):
    """What is not finite in one row (or in one expert's weights) reaches that row (those rows) alone."""
    from nersemble_amd import experts as X
    T, E, K, N = 150, 3, 40, 24
    rng = np.random.default_rng(3)
    c = torch.from_numpy(rng.integers(0, E, (T, 1)).astype(np.int32)).to(cuda)
    plan = X.expert_plan(c, E)
    x = torch.from_numpy(rng.standard_normal((T, K)).astype(np.float16)).to(cuda)
    w = torch.from_numpy(rng.standard_normal((E, N, K)).astype(np.float16)).to(cuda)
    clean = X.expert_linear(x, w, plan)
    x2 = x.clone()
    x2[7], x2[11, 3] = float("inf"), float("nan")
    got = X.expert_linear(x2, w, plan)
    hit = torch.zeros(T, dtype=torch.bool, device=cuda)
    hit[plan.positions[[7, 11], 0].long()] = True
    assert torch.equal(got[~hit], clean[~hit]) and not torch.isfinite(got[hit]).any()
    w2 = w.clone()
    w2[1] = float("nan")
    got = X.expert_linear(x, w2, plan)
    mine = torch.zeros(T, dtype=torch.bool, device=cuda)
    mine[int(plan.offsets[1]):int(plan.offsets[2])] = True
    assert torch.equal(got[~mine], clean[~mine]) and torch.isnan(got[mine]).all()
    assert torch.isnan(X.expert_linear(x2, w, plan, relu=True)[plan.positions[11, 0].long()]).all()


@pytest.mark.parametrize("K,N", [(32, 64), (64, 16), (16, 64), (128, 64), (64, 128), (256, 256)])
def test_linear_rows_behind_the_last_segment_are_zero_whatever_the_weights(K, N, cuda):
    from nersemble_amd import experts as X
    T, E = 700, 3
    c = torch.full((T, 2), -1, dtype=torch.int32, device=cuda)
    c[::3, 1] = 1
    plan = X.expert_plan(c, E)
    n = int(plan.offsets[-1])
    x = torch.randn((T, K), device=cuda).half().requires_grad_(True)
    w = torch.randn((E, N, K), device=cuda).half()
    w[0], w[2] = float("inf"), float("nan")
    w.requires_grad_(True)
    y = X.expert_linear(x, w, plan)
    assert (y[n:] == 0).all() and torch.isfinite(y).all() and (y[:n] != 0).any()
    dx, dw = torch.autograd.grad(y, [x, w], torch.ones_like(y))
    off = (c < 0).all(1)
    assert torch.isfinite(dx).all() and (dx[off] == 0).all() and (dw[[0, 2]] == 0).all() and torch.isfinite(dw).all()
    dh, = torch.autograd.grad(X.expert_linear(x.detach().repeat(2, 1).requires_grad_(True), w, plan, gather=False).sum(), [w])
    assert (dh[[0, 2]] == 0).all()


@pytest.mark.parametrize("T,k,E,K,N", [(16384, 2, 17, 1000, 2056), (9000, 3, 70, 776, 776), (20000, 2, 5, 264, 520), (40001, 1, 3, 512, 256)])
@pytest.mark.parametrize("dtype,relu,master", [("bf16", False, False), ("fp16", True, False), ("fp16", False, True)])
def test_linear_largest_tiles(T, k, E, K, N, dtype, relu, master, cuda):
    """Products of thousands of tiles, one expert with a third of the rows, against 64-bit products of each segment."""
    from nersemble_amd import experts as X
    g = torch.Generator(device=cuda).manual_seed(T)
    dt, (h, tiny) = DT[dtype], HALF[DT[dtype]]
    logits = torch.randn((T, E), generator=g, device=cuda)
    logits[:, min(3, E - 1)] += 2
    _, c = X.route_experts(logits, k)
    c[::10] = -1
    plan = X.expert_plan(c, E)
    x = torch.randn((T, K), generator=g, device=cuda).to(dt).requires_grad_(True)
    wf = torch.randn((E, N, K), generator=g, device=cuda) / K ** 0.5
    w = (wf if master else wf.to(dt)).requires_grad_(True)
    y = X.expert_linear(x, w, plan, relu=relu)
    dy = torch.randn(y.shape, generator=g, device=cuda).to(dt)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    off = plan.offsets.tolist()
    assert (y[off[-1]:] == 0).all()
    wx, tx = torch.zeros((T, K), dtype=torch.float64, device=cuda), torch.zeros((T, K), dtype=torch.float64, device=cuda)

    def inside(got, want, tol, what):
        assert ((got.double() - want).abs() <= tol).all(), what
    for e in range(E):
        a, b = off[e], off[e + 1]
        r = (plan.rows[a:b] // k).long()
        xe, we = x.detach()[r].double(), wf[e].to(dt).double()
        want, mag = xe @ we.t(), xe.abs() @ we.t().abs()
        if relu:
            want = want.clamp(min=0)
        inside(y[a:b], want, h * want.abs() + tiny + (K + 2) * 2 * U * mag, "y")
        dz = dy[a:b].double() * (y[a:b] > 0) if relu else dy[a:b].double()
        want, mag = dz.t() @ xe, dz.t().abs() @ xe.abs()
        inside(dw[e], want, (b - a + 66) * 2 * U * mag + (0 if master else h * want.abs() + tiny), "dw")
        want, mag = dz @ we, dz.abs() @ we.abs()
        wx.index_add_(0, r, want)
        tx.index_add_(0, r, h * want.abs() + tiny + (N + 2 + k) * 2 * U * mag)
    inside(dx, wx, (tx + h * wx.abs() + h * tx + tiny) * (1 + 4 * U * k), "dx")


def test_linear_layouts(cuda):
    """Strided, transposed and misaligned rows, gradients and weights give what their contiguous copies give."""
    from nersemble_amd import experts as X
    g = torch.Generator(device=cuda).manual_seed(2)
    T, k, E, K, N = 90, 2, 4, 32, 48
    c = torch.randint(0, E, (T, k), generator=g, device=cuda, dtype=torch.int32)
    plan = X.expert_plan(c, E)

    def rnd(*s):
        return torch.randn(s, generator=g, device=cuda).half()
    xs = [rnd(T, 56)[:, 8:40], rnd(T, 41)[:, 3:35], rnd(K, T).t(), rnd(T * K + 1)[1:].view(T, K), rnd(1, K).expand(T, K)]
    ws = [rnd(E, N, K), rnd(E, K, N).transpose(1, 2), rnd(E * N * K + 1)[1:].view(E, N, K), rnd(E, N, K), rnd(E, N, K)]
    dys = [rnd(T * k, N), rnd(T * k, 64)[:, 8:56], rnd(N, T * k).t(), rnd(T * k, 49)[:, 1:], rnd(1, N).expand(T * k, N)]
    for x, w, dy in zip(xs, ws, dys):
        a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        a2, b2 = x.detach().contiguous().clone().requires_grad_(True), w.detach().contiguous().clone().requires_grad_(True)
        y, y2 = X.expert_linear(a, b, plan, relu=True), X.expert_linear(a2, b2, plan, relu=True)
        assert torch.equal(y, y2)
        for p, q in zip(torch.autograd.grad(y, [a, b], dy), torch.autograd.grad(y2, [a2, b2], dy.contiguous().clone())):
            assert torch.equal(p, q)


@pytest.mark.parametrize("T,k,N", [(1, 1, 8), (3, 5, 16), (130, 2, 64), (1000, 8, 24), (77, 3, 520), (50, 4, 2048), (20000, 2, 16)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("masked", [0.0, 0.5, 1.0])
def test_combine(T, k, N, dtype, masked, cuda):
    from nersemble_amd import experts as X
    rng = np.random.default_rng(T + N)
    E, dt = 9, DT[dtype]
    chosen = _chosen(rng, T, k, E, masked)
    chosen[rng.random((T, k)) < 0.1] = -1                 # single choices as well
    plan = X.expert_plan(torch.from_numpy(chosen).to(cuda), E)
    _, _, positions = ox.plan(chosen, E)
    y = torch.from_numpy(rng.standard_normal((T * k, N)).astype(np.float32)).to(dt)
    w = rng.random((T, k)).astype(np.float32)
    g = torch.from_numpy(rng.standard_normal((T, N)).astype(np.float32)).to(dt)
    yd, wd = y.to(cuda).requires_grad_(True), torch.from_numpy(w).to(cuda).requires_grad_(True)
    out = X.expert_combine(yd, wd, plan)
    h, tiny = HALF[dt]
    want, mag = ox.combine(_f64(y), w, positions)
    assert out.dtype == dt
    _close(out, want, h * np.abs(want) + tiny + (k + 2) * 2 * U * mag, "out")
    dy, dw = torch.autograd.grad(out, [yd, wd], g.to(cuda))
    g64, y64 = _f64(g), _f64(y)
    wdy, wdw, mdw = np.zeros_like(y64), np.zeros((T, k)), np.zeros((T, k))
    for t in range(T):
        for j in range(k):
            if positions[t, j] >= 0:
                p = positions[t, j]
                wdy[p] = w[t, j].astype(np.float64) * g64[t]
                wdw[t, j], mdw[t, j] = (g64[t] * y64[p]).sum(), (np.abs(g64[t]) * np.abs(y64[p])).sum()
    _close(dy, wdy, (h + 2 * U) * np.abs(wdy) + tiny, "dy")
    _close(dw, wdw, (N + 2) * 2 * U * mdw, "dweights")


def test_plans_of_other_numbers_stay_inside_the_arrays(cuda):
    """A plan whose numbers are not a plan's gives other results, but the kernels bound every index that they take from it."""
    from nersemble_amd import experts as X
    T, k, E, K, N = 64, 2, 4, 32, 48
    x = torch.randn((T, K), device=cuda).half().requires_grad_(True)
    w = torch.randn((E, N, K), device=cuda).half().requires_grad_(True)
    wt = torch.rand((T, k), device=cuda, requires_grad=True)
    big, low = 2 ** 31 - 1, -2 ** 31
    offs = [[0, 500, 100, -7, big], [big, big, 0, 5, 9], [low, -1, low, 128, 128]]
    fill = [big, low, 129]
    for o, f in zip(offs, fill):
        plan = X.ExpertPlan(torch.tensor(o, dtype=torch.int32, device=cuda), torch.full((T * k,), f, dtype=torch.int32, device=cuda),
                            torch.full((T, k), f, dtype=torch.int32, device=cuda))
        y = X.expert_linear(x, w, plan, relu=True)
        out = X.expert_combine(y, wt, plan)
        grads = torch.autograd.grad(out, [x, w, wt], torch.ones_like(out))
        torch.cuda.synchronize()
        assert out.shape == (T, N) and (out == 0).all() and all((q == 0).all() for q in grads)


# ---------------------------------------------------------------------------------------------------------------------
# a run of them
# ---------------------------------------------------------------------------------------------------------------------
def _mixture(x, logits, w1, w2, E, k, selector=None, bias=None):
    """The whole path of a routed network with one hidden layer."""
    from nersemble_amd import experts as X
    weights, chosen = X.route_experts(logits, k, bias=bias, selector=selector)
    plan = X.expert_plan(chosen, E)
    h = X.expert_linear(x, w1, plan, gather=True, relu=True)
    y = X.expert_linear(h, w2, plan, gather=False)
    return X.expert_combine(y, weights, plan)


def _mixture64(x, logits, w1, w2, k, selector=None):
    """The same, densely: every expert on every row, in 64 bits; rows without experts are 0."""
    s = torch.softmax(logits, 1)
    top = torch.sort(s, dim=1, descending=True, stable=True).indices[:, :k]
    u = s.gather(1, top)
    w = u / u.sum(1, keepdim=True)
    if selector is not None:
        w = w * selector[:, None]
    y = torch.relu(torch.matmul(x, w1.transpose(1, 2).contiguous()))                    # [E, T, hidden]
    y = torch.matmul(y, w2.transpose(1, 2).contiguous()).transpose(0, 1)                # [T, E, n]
    return (w[..., None] * y.gather(1, top[..., None].expand(-1, -1, y.shape[2]))).sum(1)


def _mixture_inputs(T, E, K, H, N, seed, dev):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)                               # noqa: E731
    x, logits = r(T, K).half(), r(T, E)
    w1, w2 = (r(E, H, K) / K ** 0.5).half(), (r(E, N, H) / H ** 0.5).half()
    return [v.to(dev).requires_grad_(True) for v in (x, logits, w1, w2)], r(T, N).half().to(dev)


@pytest.mark.parametrize("T,E,k,K,H,N", [(1, 4, 2, 32, 64, 16), (501, 8, 2, 32, 64, 16), (333, 5, 3, 40, 128, 24)])
def test_routed_chain(T, E, k, K, H, N, cuda):
    """Route -> plan -> linear -> linear -> combine with all gradients, against dense 64-bit autograd.  Tolerance: the hidden row
    is rounded to 16 bits (h of each term), as are y, dy and dh on the way; every one of the at most 4 roundings a path passes
    moves a result by h times a norm-like sum of its terms, so 8 h relative to the largest entry of the tensor, and a hidden
    unit that changes sides next to 0 by no more than that either."""
    (x, logits, w1, w2), go = _mixture_inputs(T, E, K, H, N, 5, cuda)
    sel = (torch.arange(T, device=cuda) % 5 != 3).to(torch.uint8)
    out = _mixture(x, logits, w1, w2, E, k, sel)
    grads = torch.autograd.grad(out, [x, logits, w1, w2], go)
    leaves = [v.detach().double().cpu().requires_grad_(True) for v in (x, logits, w1, w2)]
    want = _mixture64(*leaves, k, sel.double().cpu())
    wg = torch.autograd.grad(want, leaves, go.double().cpu())
    for name, a, b in zip(("out", "dx", "dlogits", "dw1", "dw2"), (out,) + grads, (want,) + wg):
        tol = 8 * 2.0 ** -11 * float(b.abs().max())
        assert float((a.detach().double().cpu() - b).abs().max()) <= tol, name


def test_calls_repeat_bit_for_bit_and_on_another_stream(cuda):
    (x, logits, w1, w2), go = _mixture_inputs(3000, 16, 32, 64, 16, 6, cuda)
    first = None
    for where in range(3):
        s = torch.cuda.Stream() if where == 2 else torch.cuda.current_stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            out = _mixture(x, logits, w1, w2, 16, 2)
            got = [out.detach()] + list(torch.autograd.grad(out, [x, logits, w1, w2], go))
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        if first is None:
            first = got
        assert all(torch.equal(a, b) for a, b in zip(got, first))


def test_two_graphs_of_a_step_replay(cuda):
    """Forward and backward captured twice (two batches), replayed in turn with eager work between: every replay is the eager
    result of what its inputs hold then."""
    def inputs(seed, T):
        return _mixture_inputs(T, 8, 32, 64, 16, seed, cuda)

    def step(leaves, go):
        leaves = [v.detach().requires_grad_(True) for v in leaves]
        out = _mixture(*leaves, 8, 2)
        return [out.detach()] + list(torch.autograd.grad(out, leaves, go))
    graphs = []
    side = torch.cuda.Stream()
    for seed, T in ((1, 700), (2, 90000)):
        leaves, go = inputs(seed, T)
        static = [v.detach().clone() for v in leaves]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(static, go)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step(static, go)
        graphs.append((graph, static, go, res, T))
    for turn in range(3):
        for n, (graph, static, go, res, T) in enumerate(graphs):
            new, _ = inputs(10 * turn + n, T)
            for s, v in zip(static, new):
                s.copy_(v.detach())
            graph.replay()
            want = step(static, go)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(res, want)), (turn, n)


def test_device_side_row_count(cuda):
    """Under ``device_count`` the rows behind the count are neither routed nor written, whatever they hold."""
    from nersemble_amd import _lib
    from nersemble_amd import experts as X
    T, n, E, k = 600, 437, 8, 2
    (x, logits, w1, w2), go = _mixture_inputs(T, E, 32, 64, 16, 7, cuda)
    with torch.no_grad():
        want = _mixture(x[:n], logits[:n], w1, w2, E, k)
        x2, l2 = x.detach().clone(), logits.detach().clone()
        x2[n:], l2[n:] = float("nan"), float("nan")
        for count in (n, 0, T, -3):
            c = torch.tensor([count], dtype=torch.int64, device=cuda)
            with _lib.device_count(c, T):
                weights, chosen = X.route_experts(l2 if count <= n else logits, k)
                plan = X.expert_plan(chosen, E)
                h = X.expert_linear(x2 if count <= n else x, w1, plan, relu=True)
                out = X.expert_combine(X.expert_linear(h, w2, plan, gather=False), weights, plan)
            routed = max(0, min(count, T)) * k
            assert int(plan.offsets[-1]) == routed and (plan.rows[routed:] == -1).all() and (plan.positions[routed // k:] == -1).all()
            assert torch.isfinite(h).all()
            m = min(n, max(0, count))
            assert torch.equal(out[:m], want[:m])
    # gradients: weights see the valid rows alone
    c = torch.tensor([n], dtype=torch.int64, device=cuda)
    leaves = [v.detach().clone().requires_grad_(True) for v in (x2, l2, w1, w2)]
    ref = [v.detach().clone().requires_grad_(True) for v in (x[:n], logits[:n], w1, w2)]
    want = torch.autograd.grad(_mixture(*ref, E, k), ref, go[:n])
    with _lib.device_count(c, T):
        got = torch.autograd.grad(_mixture(*leaves, E, k), leaves, go)
    assert torch.equal(got[2], want[2]) and torch.equal(got[3], want[3])
    assert torch.equal(got[0][:n], want[0]) and torch.equal(got[1][:n], want[1])


def test_the_same_tensor_twice_and_shared_plans(cuda):
    """One weight in two products, one plan for two inputs, the gradients of both uses added."""
    from nersemble_amd import experts as X
    (x, logits, w1, _), _ = _mixture_inputs(200, 4, 64, 64, 16, 8, cuda)
    _, chosen = X.route_experts(logits.detach(), 2)
    plan = X.expert_plan(chosen, 4)
    y = X.expert_linear(X.expert_linear(x, w1, plan, relu=True), w1, plan, gather=False)
    dx, dw = torch.autograd.grad(y.float().sum(), [x, w1])
    a, b = w1.detach().clone().requires_grad_(True), w1.detach().clone().requires_grad_(True)
    y2 = X.expert_linear(X.expert_linear(x, a, plan, relu=True), b, plan, gather=False)
    dx2, da, db = torch.autograd.grad(y2.float().sum(), [x, a, b])
    assert torch.equal(dx, dx2) and torch.equal(dw, da + db)


@pytest.mark.parametrize("n_in,n_out,n_hidden,routing", [
    (32, 16, 1, dict(n_experts=4, top_k=2)), (35, 3, 2, dict(n_experts=6, top_k=1, renormalise=False)),
    (16, 8, 1, dict(n_experts=8, top_k=3, scores="sigmoid", n_groups=4, top_groups=2, balance=True))])
def test_routed_network(n_in, n_out, n_hidden, routing, cuda):
    """tcnn.RoutedNetwork trains: finite gradients of every parameter, equal to those of the same mixture evaluated expert by
    expert in 64 bits (tolerance as for the chain, one more rounding per hidden layer), and a step changes its output."""
    from nersemble_amd import tcnn
    net = tcnn.RoutedNetwork(n_in, n_out, {"n_neurons": 64, "n_hidden_layers": n_hidden}, routing).to(cuda)
    g = torch.Generator().manual_seed(n_in)
    x = torch.randn((301, n_in), generator=g).half()
    go = torch.randn((301, n_out), generator=g).half()
    xd = x.to(cuda).requires_grad_(True)
    out = net(xd)
    assert out.shape == (301, n_out) and out.dtype == torch.float16
    got = torch.autograd.grad(out, [xd, net.gate, net.params], go.to(cuda))
    # 64 bits, densely (the choice is the network's own: gaps of the scores are far above the rounding of the logits)
    x64 = x.double().requires_grad_(True)
    gate, params = (p.detach().double().cpu().requires_grad_(True) for p in (net.gate, net.params))
    logits = x64 @ gate.t()
    s = torch.sigmoid(logits) if routing.get("scores") == "sigmoid" else torch.softmax(logits, 1)
    E, k = routing["n_experts"], routing["top_k"]
    from nersemble_amd import experts as X
    _, chosen = X.route_experts((xd.detach().float() @ net.gate.detach().t()), k, bias=net.balance, **net.routing)
    idx = chosen.long().cpu()
    u = s.gather(1, idx)
    w = u / u.sum(1, keepdim=True) if routing.get("renormalise", True) else u
    h = torch.nn.functional.pad(x64, (0, net.shapes[0][2] - n_in)).expand(E, -1, -1)
    for n, (m, shape) in enumerate(zip(torch.split(params, [a * b * c for a, b, c in net.shapes]), net.shapes)):
        m16 = m + (m.detach().half().double() - m.detach())                  # the fp16 values, the fp32 parameters' gradient
        h = torch.matmul(h, m16.view(shape).transpose(1, 2))
        h = torch.relu(h) if n < len(net.shapes) - 1 else h
    y = h.transpose(0, 1).gather(1, idx[..., None].expand(-1, -1, h.shape[2]))
    want = (w[..., None] * y).sum(1)[:, :n_out]
    wg = torch.autograd.grad(want, [x64, gate, params], go.double())
    for name, a, b in zip(("out", "dx", "dgate", "dparams"), (out,) + got, (want,) + wg):
        tol = (6 + 4 * n_hidden) * 2.0 ** -11 * float(b.abs().max())
        assert float((a.detach().double().cpu() - b).abs().max()) <= tol, name
    assert int(net.load.sum()) == 301 * k
    opt = torch.optim.Adam(net.parameters(), lr=1e-2)
    net.gate.grad, net.params.grad = got[1], got[2]
    opt.step()
    assert not torch.equal(net(xd), out)
    assert (net(xd, selector=torch.zeros(301, dtype=torch.uint8, device=cuda)) == 0).all()
    if routing.get("balance"):
        net.rebalance(0.5)
        assert set(net.balance.abs().tolist()) <= {0.0, 0.5}
    else:
        with pytest.raises(RuntimeError):
            net.rebalance()


# ---------------------------------------------------------------------------------------------------------------------
# corners
# ---------------------------------------------------------------------------------------------------------------------
def test_no_rows_at_all(cuda):
    """Zero rows: empty results, a weight gradient of zeros, through every call."""
    from nersemble_amd import experts as X
    E, K, N = 3, 32, 48
    for k in (1, 2):
        logits = torch.empty((0, E), device=cuda, requires_grad=True)
        w, c = X.route_experts(logits, k)
        plan = X.expert_plan(c, E)
        x = torch.empty((0, K), dtype=torch.float16, device=cuda, requires_grad=True)
        m = torch.randn((E, N, K), device=cuda).half().requires_grad_(True)
        y = X.expert_linear(x, m, plan, relu=True)
        out = X.expert_combine(y, w, plan)
        assert w.shape == (0, k) and y.shape == (0, N) and out.shape == (0, N) and (plan.offsets == 0).all()
        dl, dx, dm = torch.autograd.grad(out, [logits, x, m], torch.empty_like(out))
        assert dl.shape == (0, E) and dx.shape == (0, K) and (dm == 0).all()


def test_gradients_of_some_inputs_only(cuda):
    """Each input's gradient alone is the one that is computed beside the others'."""
    from nersemble_amd import experts as X
    (x, logits, w1, w2), go = _mixture_inputs(150, 5, 32, 64, 16, 9, cuda)
    full = torch.autograd.grad(_mixture(x, logits, w1, w2, 5, 2), [x, logits, w1, w2], go)
    for n in range(4):
        leaves = [v.detach().requires_grad_(i == n) for i, v in enumerate((x, logits, w1, w2))]
        (g,) = torch.autograd.grad(_mixture(*leaves, 5, 2), [leaves[n]], go)
        assert torch.equal(g, full[n])
    # and a second differentiation is refused, not wrong
    g = torch.autograd.grad(_mixture(x, logits, w1, w2, 5, 2), [w1], go, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.float().sum(), [x])


def test_what_is_not_routed_is_not_read(cuda):
    """Rows, gradients and outputs that no segment holds may be anything."""
    from nersemble_amd import experts as X
    nan = float("nan")
    T, E, k = 300, 4, 2
    (x, logits, w1, w2), go = _mixture_inputs(T, E, 32, 64, 16, 10, cuda)
    sel = (torch.arange(T, device=cuda) % 3 > 0).to(torch.uint8)
    off = sel == 0
    want = _mixture(x, logits, w1, w2, E, k, sel)
    wg = torch.autograd.grad(want, [x, logits, w1, w2], go)
    x2, l2, go2 = x.detach().clone(), logits.detach().clone(), go.clone()
    x2[off], l2[off], go2[off] = nan, nan, nan
    leaves = [v.detach().requires_grad_(True) for v in (x2, l2, w1, w2)]
    got = _mixture(*leaves, E, k, sel)
    gg = torch.autograd.grad(got, leaves, go2)
    assert torch.equal(got, want) and (got[off] == 0).all()
    for a, b in zip(gg, wg):
        assert torch.equal(a, b)
    # the gradient of a product's rows behind the last segment
    _, c = X.route_experts(l2, k, selector=sel)
    plan = X.expert_plan(c, E)
    xa, wa = x.detach().requires_grad_(True), w1.detach().requires_grad_(True)
    y = X.expert_linear(xa, wa, plan)
    n = int(plan.offsets[-1])
    dy = torch.randn(y.shape, device=cuda).half()
    a = torch.autograd.grad(y, [xa, wa], dy, retain_graph=True)
    dy[n:] = nan
    b = torch.autograd.grad(y, [xa, wa], dy)
    assert n < y.shape[0] and (y[n:] == 0).all() and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_more_than_2_31_elements(cuda):
    """Ordered rows whose elements pass 2^31 (and whose bytes pass 2^32): products, gradients and join at the far end."""
    from nersemble_amd import experts as X
    T, E, K, N = (1 << 20) + 5, 3, 8, 2056
    g = torch.Generator(device=cuda).manual_seed(0)
    c = torch.randint(0, E, (T, 1), generator=g, device=cuda, dtype=torch.int32)
    plan = X.expert_plan(c, E)
    x = torch.randn((T, K), generator=g, device=cuda).half().requires_grad_(True)
    w = torch.randn((E, N, K), generator=g, device=cuda).half().requires_grad_(True)
    y = X.expert_linear(x, w, plan)
    assert y.numel() > 2 ** 31
    last = plan.rows[-200:].long()
    want = x.detach().float()[last] @ w.detach().float()[E - 1].t()
    tol = 2.0 ** -11 * want.abs() + 2.0 ** -25 + (K + 2) * 2 * U * (x.detach().float().abs()[last] @ w.detach().float().abs()[E - 1].t())
    assert ((y.detach()[-200:].float() - want).abs() <= tol).all()
    wt = torch.ones((T, 1), device=cuda)
    out = X.expert_combine(y.detach(), wt, plan)
    assert torch.equal(out[last], y.detach()[-200:])
    del out
    # dx of the last rows alone: dy is zero before them (a sum over 2056 outputs), dW then is theirs as well
    dy = torch.zeros_like(y)
    dy[-200:] = torch.randn((200, N), generator=g, device=cuda).half()
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    far = dy[-200:].float()
    want = far @ w.detach().float()[E - 1]
    tol = 2 * (2.0 ** -11 * want.abs() + 2.0 ** -25) + (N + 2) * 2 * U * (far.abs() @ w.detach().float().abs()[E - 1])
    assert ((dx[last].float() - want).abs() <= tol).all() and int((dx != 0).any(1).sum()) == 200
    want = far.t() @ x.detach().float()[last]
    tol = 2.0 ** -11 * want.abs() + 2.0 ** -25 + (200 + 66) * 2 * U * (far.abs().t() @ x.detach().float().abs()[last])
    assert ((dw[E - 1].float() - want).abs() <= tol).all() and (dw[:E - 1] == 0).all()


def test_route_choice_where_32_bits_do_not_tell(cuda):
    """Scores plus a bias that lie closer than 32 bits resolve, and equal ones: the choice is that of 64 bits."""
    from nersemble_amd import experts as X
    rng = np.random.default_rng(4)
    for E, G, tg, gt in ((64, 1, 1, 1), (64, 8, 3, 2), (256, 8, 4, 2)):
        x = (rng.standard_normal((257, E)) * 0.5).astype(np.float32)
        # neighbours one step of fp32 apart, in a shuffled order
        for t in range(0, 257, 2):
            base = np.float32(rng.standard_normal())
            x[t] = base + np.float32(2.0 ** -22) * rng.permutation(E).astype(np.float32)
        x[1::4] = np.round(x[1::4] * 4) / 4                                   # many equal
        for bias in (np.zeros(E, np.float32), (rng.integers(0, 3, E) * 2.0 ** -20).astype(np.float32)):
            for sc in ("sigmoid", "softmax"):
                w, c = X.route_experts(torch.from_numpy(x).to(cuda), 6, scores=sc, bias=torch.from_numpy(bias).to(cuda), n_groups=G, top_groups=tg, group_top=gt)
                s = ox.scores(x, sc == "sigmoid") + bias
                _, wc = ox.route(x, 6, sc == "sigmoid", bias, G, tg, gt)
                got = c.cpu().numpy()
                # (64-bit sums of a softmax depend on their order by 1e-16: a row counts where no two values are that close but not equal)
                v = np.sort(s, axis=1)
                d = np.diff(v, axis=1)
                clear = ~((d > 0) & (d < 1e-13)).any(1)
                if G > 1:
                    by = np.sort(np.sort(s.reshape(len(s), G, -1), axis=2)[:, :, -gt:].sum(2), axis=1)
                    dg = np.diff(by, axis=1)
                    clear &= ~((dg > 0) & (dg < 1e-13)).any(1)
                assert clear.mean() > 0.5 and np.array_equal(got[clear], wc[clear]), (E, G, sc)


def test_the_same_expert_twice_for_a_row(cuda):
    """Choices made by hand: a row that names one expert several times is several entries of it, gradients add up."""
    from nersemble_amd import experts as X
    T, E, K, N = 70, 3, 24, 40
    g = torch.Generator(device=cuda).manual_seed(3)
    c = torch.randint(0, E, (T, 1), generator=g, device=cuda, dtype=torch.int32)
    x = torch.randn((T, K), generator=g, device=cuda).half().requires_grad_(True)
    w = torch.randn((E, N, K), generator=g, device=cuda).half().requires_grad_(True)
    go = torch.randn((T, N), generator=g, device=cuda).half()
    one, three = X.expert_plan(c, E), X.expert_plan(c.expand(T, 3), E)
    wt = torch.tensor([0.5, 0.25, 0.25], device=cuda).expand(T, 3)
    a = X.expert_combine(X.expert_linear(x, w, one), torch.ones((T, 1), device=cuda), one)
    b = X.expert_combine(X.expert_linear(x, w, three), wt, three)
    assert torch.equal(a, b)                                         # (weights that are powers of two: nothing rounds)
    ga, gb = torch.autograd.grad(a, [x, w], go), torch.autograd.grad(b, [x, w], go)
    # dw: the same terms (scaled exactly) in another order; dx: three scaled copies of one gradient, each rounded
    h, tiny = HALF[torch.float16]
    x64, w64, g64 = x.detach().double(), w.detach().double(), go.double()
    for e in range(E):
        m = c[:, 0] == e
        mag = g64[m].t().abs() @ x64[m].abs()
        tol = 2 * (h * ga[1][e].double().abs() * 2 + tiny) + 2 * (3 * int(m.sum()) + 66) * 2 * U * mag
        assert ((ga[1][e].double() - gb[1][e].double()).abs() <= tol).all()
        mag = g64[m].abs() @ w64[e].abs()
        tol = 2 * (2 * h * ga[0][m].double().abs() + 4 * tiny) + 2 * (N + 6) * 2 * U * mag + h * h * mag
        assert ((ga[0][m].double() - gb[0][m].double()).abs() <= tol).all()


def test_products_against_differences(cuda):
    """Gradients of the products and of the join against differences: both are linear in each input, so a step of 1 in one
    value changes the loss by the gradient, up to the roundings of the outputs."""
    from nersemble_amd import experts as X
    g = torch.Generator(device=cuda).manual_seed(8)
    T, k, E, K, N = 9, 2, 3, 8, 16
    _, c = X.route_experts(torch.randn((T, E), generator=g, device=cuda), k)
    plan = X.expert_plan(c, E)
    # small whole numbers: every product, sum and difference is exact in fp16 and fp32
    x = torch.randint(-3, 4, (T, K), generator=g, device=cuda).half()
    w = torch.randint(-3, 4, (E, N, K), generator=g, device=cuda).half()
    wt = torch.randint(-2, 3, (T, k), generator=g, device=cuda).float()
    go = torch.randint(-1, 2, (T, N), generator=g, device=cuda).half()

    def loss(x, w, wt):
        return (X.expert_combine(X.expert_linear(x, w, plan), wt, plan).double() * go.double()).sum()
    leaves = [v.clone().requires_grad_(True) for v in (x, w, wt)]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    base = loss(x, w, wt)
    for n, v in enumerate((x, w, wt)):
        for i in range(0, v.numel(), 5):
            args = [u.clone() for u in (x, w, wt)]
            args[n].view(-1)[i] += 1
            assert float(loss(*args) - base) == float(grads[n].reshape(-1)[i]), (n, i)


def test_two_runs_at_once_on_two_streams(cuda):
    """Two steps enqueued on two streams without waiting for each other give what they give alone."""
    a, ga = _mixture_inputs(3000, 8, 64, 128, 32, 11, cuda)
    b, gb = _mixture_inputs(2500, 5, 32, 64, 16, 12, cuda)

    def step(v, go, E):
        out = _mixture(*v, E, 2)
        return [out] + list(torch.autograd.grad(out, v, go))
    want = step(a, ga, 8), step(b, gb, 5)
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (v, go, E) in enumerate(((a, ga, 8), (b, gb, 5))):
            with torch.cuda.stream(s[i]):
                got[i].append(step(v, go, E))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            for p, q in zip(r, want[i]):
                assert torch.equal(p, q)


def test_routed_network_rows_that_are_not_evaluated(cuda):
    """What `selector` leaves out may hold anything: outputs 0, gradients as if the rows were not there; no rows at all work too."""
    from nersemble_amd import tcnn
    net = tcnn.RoutedNetwork(20, 5, {"n_neurons": 64, "n_hidden_layers": 2}, {"n_experts": 6, "top_k": 2}).to(cuda)
    g = torch.Generator().manual_seed(6)
    x = torch.randn((300, 20), generator=g).to(cuda)
    sel = (torch.arange(300, device=cuda) % 4 != 0).to(torch.uint8)
    go = torch.randn((300, 5), generator=g).half().to(cuda)
    grads = []
    for fill in (0.0, float("nan"), float("inf")):
        v = x.clone()
        v[sel == 0] = fill
        v.requires_grad_(True)
        out = net(v, sel)
        assert (out[sel == 0] == 0).all()
        grads.append([out] + list(torch.autograd.grad(out, [v, net.params, net.gate], go)))
    for other in grads[1:]:
        for a, b in zip(grads[0], other):
            assert torch.isfinite(b).all() and torch.equal(a, b)
    assert (grads[0][1][sel == 0] == 0).all()
    empty = net(x[:0].requires_grad_(True))
    assert empty.shape == (0, 5)
    (gp,) = torch.autograd.grad(empty.sum(), [net.params])
    assert (gp == 0).all()


def test_graph_of_a_wide_step_replays(cuda):
    """Wide layers behind a ReLU (dy masked in a pass of its own, chunks of large tiles) captured and replayed: the eager result."""
    T, E, shape = 6000, 3, (1024, 520, 264)

    def step(leaves, go):
        leaves = [v.detach().requires_grad_(True) for v in leaves]
        out = _mixture(*leaves, E, 2)
        return [out.detach()] + list(torch.autograd.grad(out, leaves, go))
    leaves, go = _mixture_inputs(T, E, *shape, 21, cuda)
    static = [v.detach().clone() for v in leaves]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static, go)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step(static, go)
    for turn in range(3):
        new, _ = _mixture_inputs(T, E, *shape, 30 + turn, cuda)
        for s, v in zip(static, new):
            s.copy_(v.detach())
        graph.replay()
        want = step(static, go)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, want)), turn


def test_a_plan_changed_before_the_backward_pass_is_refused(cuda):
    from nersemble_amd import experts as X
    (x, logits, w1, w2), go = _mixture_inputs(40, 4, 32, 64, 16, 5, cuda)
    weights, chosen = X.route_experts(logits.detach(), 2)
    plan = X.expert_plan(chosen, 4)
    h = X.expert_linear(x, w1, plan, relu=True)
    out = X.expert_combine(X.expert_linear(h, w2, plan, gather=False), weights, plan)
    torch.autograd.grad(out, [x, w1], go, retain_graph=True)
    plan.rows.add_(0)
    with pytest.raises(RuntimeError, match="inplace operation"):
        torch.autograd.grad(out, [x, w1], go)


def test_plain_arguments_run_natively(cuda, way, monkeypatch):
    """The native nodes are what runs where nothing stands against it; a row count on the device, a profiler or another layout do."""
    from nersemble_amd import _lib
    from nersemble_amd import experts as X
    called = []
    if way != "native":
        return
    X.expert_plan(torch.zeros((1, 1), dtype=torch.int32, device=cuda), 1)          # (loads it)
    native = X._fast

    class Watch:
        def __getattr__(self, name):
            def call(*args):
                out = getattr(native, name)(*args)
                called.append((name, out is not None))
                return out
            return call
    monkeypatch.setattr(X, "_fast", Watch())
    (x, logits, w1, w2), go = _mixture_inputs(50, 4, 32, 64, 16, 5, cuda)
    out = _mixture(x, logits, w1, w2, 4, 2)
    assert called == [("route_experts", True), ("plan", True), ("expert_linear", True), ("expert_linear", True), ("expert_combine", True)]
    want = torch.autograd.grad(out, [x, logits, w1, w2], go)
    called.clear()
    strided = torch.randn((50, 48), device=cuda).half()[:, 8:40]
    X.expert_linear(strided, w1, X.expert_plan(torch.zeros((50, 1), dtype=torch.int32, device=cuda), 4))
    assert called == [("plan", True), ("expert_linear", False)]
    called.clear()
    with _lib.device_count(torch.tensor([50], device=cuda), 50):
        again = _mixture(x, logits, w1, w2, 4, 2)
        got = torch.autograd.grad(again, [x, logits, w1, w2], go)
    assert not called and torch.equal(again, out) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("E,k,G,tg,gt", [(64, 6, 1, 1, 1), (61, 8, 1, 1, 1), (256, 8, 8, 4, 2), (64, 64, 1, 1, 1), (9, 9, 1, 1, 1), (20, 1, 4, 2, 1)])
@pytest.mark.parametrize("sc", ["sigmoid", "softmax"])
def test_route_pairs_that_32_bits_do_not_tell(E, k, G, tg, gt, sc, cuda):
    """Rows with one pair of sums a few 1e-9 apart, anywhere in the order: the choice is that of 64 bits."""
    from nersemble_amd import experts as X
    rng = np.random.default_rng(E + k)
    T = 400
    bias = (rng.standard_normal(E) * 0.1).astype(np.float32)
    x = (rng.standard_normal((T, E)) * 1.5).astype(np.float32)
    sig = sc == "sigmoid"
    for t in range(T):
        s = ox.scores(x[t:t + 1], sig)[0] + bias
        order = np.argsort(-s)
        a, b = order[t % min(E - 1, k + 1)], order[t % min(E - 1, k + 1) + 1]
        if sig:                                                              # the logit that puts b beside a
            p = s[a] - bias[b]
            if 0 < p < 1:
                x[t, b] = np.log(p / (1 - p))
        else:
            e, delta = np.exp(x[t].astype(np.float64)), np.float64(bias[a]) - np.float64(bias[b])
            eb = (e[a] + delta * (e.sum() - e[b])) / (1 - delta)
            if eb > 0:
                x[t, b] = np.log(eb)
    s = ox.scores(x, sig) + bias
    gaps = np.diff(np.sort(s, axis=1), axis=1)
    assert ((gaps > 0) & (gaps < 1e-7)).any(1).mean() > 0.2                  # (there are such pairs)
    clear = ~((gaps > 0) & (gaps < 1e-13)).any(1)
    w, c = X.route_experts(torch.from_numpy(x).to(cuda), k, scores=sc, bias=torch.from_numpy(bias).to(cuda), n_groups=G, top_groups=tg, group_top=gt)
    ww, wc = ox.route(x, k, sig, bias, G, tg, gt)
    assert clear.mean() > 0.9 and np.array_equal(c.cpu().numpy()[clear], wc[clear])
    _close(w.cpu()[clear], ww[clear], _route_tol(x, ww, k)[clear], "weights")


# ---------------------------------------------------------------------------------------------------------------------
# gathered gradients are rounded once
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,k,E,K,N,relu,only_x", [
    (211, 2, 5, 72, 48, False, False), (900, 3, 7, 264, 136, True, False), (9000, 2, 7, 32, 64, True, False), (9000, 2, 7, 64, 64, False, False),
    (5003, 8, 16, 16, 24, False, False), (4000, 3, 7, 32, 64, True, True), (4000, 2, 5, 64, 64, False, True), (700, 1, 4, 40, 72, False, False),
    (3, 64, 70, 1024, 64, False, False), (6000, 2, 3, 1024, 264, True, False), (16384, 2, 17, 1000, 2056, False, False)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_gathered_gradient_is_rounded_once(T, k, E, K, N, relu, only_x, dtype, cuda):
    """dx of a gathered product: a row's choices are summed in 32 bits (off by at most (N + 2 + k) 2 u sum |terms|) and the sum is rounded,
    not its terms: h * |sum|, where h more of each term would pass it by far."""
    from nersemble_amd import experts as X
    g = torch.Generator(device=cuda).manual_seed(T + K)
    dt, (h, tiny) = DT[dtype], HALF[DT[dtype]]
    c = torch.rand((T, E), generator=g, device=cuda).topk(k, dim=1).indices.int()
    c[::7] = -1
    plan = X.expert_plan(c, E)
    x = torch.randn((T, K), generator=g, device=cuda).to(dt).requires_grad_(True)
    w = (torch.randn((E, N, K), generator=g, device=cuda) / K ** 0.5).to(dt).requires_grad_(not only_x)
    y = X.expert_linear(x, w, plan, relu=relu)
    dy = torch.randn(y.shape, generator=g, device=cuda).to(dt)
    dx = torch.autograd.grad(y, [x] if only_x else [x, w], dy)[0].double()
    want, mag = torch.zeros((T, K), dtype=torch.float64, device=cuda), torch.zeros((T, K), dtype=torch.float64, device=cuda)
    off = plan.offsets.tolist()
    for e in range(E):
        a, b = off[e], off[e + 1]
        r = (plan.rows[a:b] // k).long()
        dz, we = dy[a:b].double(), w.detach()[e].double()
        if relu:
            dz = dz * (y[a:b] > 0)
        want.index_add_(0, r, dz @ we)
        mag.index_add_(0, r, dz.abs() @ we.abs())
    tol = h * want.abs() + tiny + (1 + h) * (N + 2 + k) * 2 * U * mag
    worst = ((dx - want).abs() / tol).max()
    assert worst <= 1.0, float(worst)


@pytest.mark.parametrize("T,K,N", [(40, 8, 8), (40, 72, 80), (3000, 32, 64), (3000, 8, 8), (600, 256, 136)])
def test_gathered_gradient_whose_terms_alone_pass_fp16(T, K, N, cuda):
    """Two choices whose gradients are +80000 and -79600 (fp16 ends at 65504): their sum is 400, exactly."""
    from nersemble_amd import experts as X
    plan = X.expert_plan(torch.tensor([[0, 1]], dtype=torch.int32, device=cuda).repeat(T, 1), 2)
    x = torch.ones((T, K), dtype=torch.float16, device=cuda, requires_grad=True)
    w = torch.zeros((2, N, K), dtype=torch.float16, device=cuda)
    w[0, :8], w[1, :8] = 200.0, -199.0
    w.requires_grad_(True)
    y = X.expert_linear(x, w, plan)
    dx, _ = torch.autograd.grad(y, [x, w], torch.full_like(y, 50.0))
    assert (dx == 400).all()


# ---------------------------------------------------------------------------------------------------------------------
# groups whose members have large biases of opposite signs
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("big", [8.0, 64.0, 1000.0, 30000.0])
@pytest.mark.parametrize("E,G,tg", [(4, 2, 1), (32, 4, 2), (64, 8, 3)])
@pytest.mark.parametrize("sc", ["sigmoid", "softmax"])
def test_route_groups_of_large_biases_that_cancel(E, G, tg, big, sc, cuda):
    """A group's two best are s + B and s' - B: their sum is of the size of a score, its error in 32 bits of the size of B's steps.  Sums of
    two groups a few 1e-6 apart: the groups that stay are those of 64 bits."""
    from nersemble_amd import experts as X
    rng = np.random.default_rng(E)
    T, per = 2000, E // G
    bias = np.full((G, per), -2 * big, np.float32)
    bias[:, 0], bias[:, 1] = big, -big
    s = rng.uniform(0.1, 0.9, (T, G, per))
    # groups in pairs: the second's sum is the first's and a few 1e-6
    other = s[:, 0::2, 0] + s[:, 0::2, 1] - s[:, 1::2, 0] + rng.uniform(-4e-6, 4e-6, (T, G // 2))
    fine = (other > 0.05) & (other < 0.95)
    s[:, 1::2, 1] = np.where(fine, other, s[:, 1::2, 1])
    s = s.reshape(T, E)
    x = (np.log(s / (1 - s)) if sc == "sigmoid" else np.log(s)).astype(np.float32)
    bias = bias.reshape(-1)
    k = min(3, tg * per)
    _, wc = ox.route(x, k, sc == "sigmoid", bias, G, tg, 2)
    by = np.sort((ox.scores(x, sc == "sigmoid") + bias).reshape(T, G, per), axis=2)[:, :, -2:].sum(2)
    gaps = np.diff(np.sort(by, axis=1), axis=1)
    clear = (gaps > big * 2.0 ** -48).all(1)                                # (64-bit sums are themselves off by steps of B)
    assert clear.mean() > 0.9 and (gaps < 1e-5).any(1).mean() > 0.5
    _, c = X.route_experts(torch.from_numpy(x).to(cuda), k, scores=sc, bias=torch.from_numpy(bias).to(cuda), n_groups=G, top_groups=tg, group_top=2)
    wrong = (c.cpu().numpy()[clear] != wc[clear]).any(1).mean()
    assert wrong == 0, wrong


# ---------------------------------------------------------------------------------------------------------------------
# autocast, forward mode, refusals
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_routed_network_under_autocast_is_the_one_without(dtype, cuda):
    """The router's product stays in 32 bits where the step runs under autocast (as a trainer's does): equal bits, forward and backward."""
    from nersemble_amd import tcnn
    net = tcnn.RoutedNetwork(20, 5, {"n_neurons": 64, "n_hidden_layers": 2}, {"n_experts": 32, "top_k": 2}).to(cuda)
    g = torch.Generator().manual_seed(6)
    for fill in (torch.float32, torch.float16):
        x = torch.randn((3000, 20), generator=g).to(fill).to(cuda).requires_grad_(True)
        sel = (torch.arange(3000, device=cuda) % 4 != 0).to(torch.uint8)
        go = torch.randn((3000, 5), generator=g).half().to(cuda)
        for s in (None, sel):
            res = []
            for on in (False, True):
                with torch.autocast(device_type="cuda", dtype=dtype, enabled=on, cache_enabled=False):
                    out = net(x, s)
                res.append([out.detach()] + list(torch.autograd.grad(out, [x, net.gate, net.params], go)))
            for name, a, b in zip(("out", "dx", "dgate", "dparams"), *res):
                assert a.dtype == b.dtype and torch.equal(a, b), name


def test_forward_mode_derivatives_are_refused(cuda):
    """A dual tensor has a tangent that these calls do not carry: refused, not dropped."""
    import torch.autograd.forward_ad as fwd
    from nersemble_amd import experts as X
    (x, logits, w1, w2), _ = _mixture_inputs(30, 4, 32, 64, 16, 5, cuda)
    x, logits, w1 = x.detach(), logits.detach(), w1.detach()
    weights, chosen = X.route_experts(logits, 2)
    plan = X.expert_plan(chosen, 4)
    y = X.expert_linear(x, w1, plan)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))                # noqa: E731
        for call in (lambda: X.route_experts(dual(logits), 2), lambda: X.expert_linear(dual(x), w1, plan),
                     lambda: X.expert_linear(x, dual(w1), plan), lambda: X.expert_combine(dual(y), weights, plan),
                     lambda: X.expert_combine(y, dual(weights), plan), lambda: X.expert_linear(x, dual(w1.float()), plan, w16=w1)):
            with pytest.raises(NotImplementedError):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError):
                call()
        # (what has no tangent goes through inside a level too)
        assert torch.equal(X.expert_linear(x, w1, plan), y)


def test_route_says_what_it_refuses(cuda):
    """The reason of this call, not that of an earlier failure."""
    from nersemble_amd import experts as X
    with pytest.raises(RuntimeError, match="scale"):
        X.route_experts(torch.zeros((4, 16), device=cuda), 2, scale=0.0)
    for E, k in ((16, 0), (16, 17), (128, 65), (16, -1), (4, 1 << 40)):
        with pytest.raises(RuntimeError, match="top_k"):
            X.route_experts(torch.zeros((4, E), device=cuda), k)
    for E in (0, 513):
        with pytest.raises(RuntimeError, match="n_experts|top_k"):
            X.route_experts(torch.zeros((4, E), device=cuda), 1)
    with pytest.raises(RuntimeError, match="n_experts"):
        X.route_experts(torch.zeros((4, 513), device=cuda, requires_grad=True), 1)


# ---------------------------------------------------------------------------------------------------------------------
# choice in large batches (8 and 16 values per lane)
# ---------------------------------------------------------------------------------------------------------------------
def _route64(x, k, sigmoid, bias, G, tg, gt, renorm, scale, selector):
    """(weights, chosen, scores, rows whose order 64 bits tell beyond the order of their own sums) on the device, in 64 bits."""
    T, E = x.shape
    xd = x.double()
    live = xd > -np.inf
    any_live = live.any(1, keepdim=True)
    s = torch.sigmoid(xd) if sigmoid else torch.where(any_live, torch.softmax(torch.where(any_live, xd, torch.zeros_like(xd)), 1), torch.zeros_like(xd))
    s = torch.where(live, s, torch.zeros_like(s))
    c = s if bias is None else s + bias.double()
    c = torch.where(live, c, torch.full_like(c, -np.inf))

    def close(v):
        d = torch.diff(torch.sort(v, dim=1).values, dim=1)
        return ((d > 0) & (d < 1e-13)).any(1)
    clear = ~close(c)
    if tg < G:
        by = torch.sort(c.view(T, G, E // G), dim=2, descending=True).values[..., :gt].sum(2)
        clear &= ~close(by)
        kept = torch.sort(by, dim=1, descending=True, stable=True).indices[:, :tg]
        on = torch.zeros((T, G), dtype=torch.bool, device=x.device).scatter_(1, kept, True)
        c = torch.where(on.repeat_interleave(E // G, 1), c, torch.full_like(c, -np.inf))
    top = torch.sort(c, dim=1, descending=True, stable=True)
    chosen, there = top.indices[:, :k], top.values[:, :k] > -np.inf
    if selector is not None:
        there = there & (selector != 0)[:, None]
    u = torch.where(there, s.gather(1, chosen), torch.zeros((), dtype=torch.float64, device=x.device))
    w = scale * (u / u.sum(1, keepdim=True).clamp(min=1e-300) if renorm else u)
    return w, torch.where(there, chosen, -1), s, clear


LARGE_ROUTES = [
    # rows, E, k, scores, bias, groups, top_groups, group_top, renorm, scale
    (131075, 32, 2, "softmax", False, 1, 1, 1, True, 1.0),               # above 2^22 values: 16 per lane
    (131075, 32, 5, "softmax", True, 1, 1, 1, False, 2.5),
    (131075, 32, 32, "sigmoid", True, 1, 1, 1, True, 1.0),               # entries of many choices: fewer values per lane
    (131075, 32, 31, "softmax", True, 1, 1, 1, True, 1.0),
    (131075, 32, 32, "softmax", False, 1, 1, 1, False, 1.0),
    (65541, 64, 64, "softmax", True, 1, 1, 1, True, 1.0),
    (65541, 64, 32, "sigmoid", False, 2, 1, 2, True, 1.0),
    (65541, 64, 64, "sigmoid", True, 2, 2, 1, True, 1.0),
    (65541, 64, 6, "sigmoid", True, 1, 1, 1, True, 1.0),
    (131075, 33, 3, "softmax", True, 1, 1, 1, True, 1.0),
    (131075, 48, 4, "sigmoid", True, 3, 2, 2, True, 1.0),
    (524291, 8, 8, "softmax", True, 1, 1, 1, True, 1.0),
    (262147, 16, 16, "sigmoid", True, 1, 1, 1, False, 1.0),
    (16411, 256, 8, "sigmoid", True, 8, 4, 2, True, 2.5),
    (16411, 256, 8, "softmax", False, 8, 3, 1, False, 16.0),
    (16411, 256, 8, "softmax", False, 1, 1, 1, True, 1.0),
    (8209, 512, 64, "softmax", True, 1, 1, 1, True, 1.0),
    (8209, 512, 16, "sigmoid", True, 16, 4, 2, True, 1.0),
    (8195, 96, 7, "softmax", True, 1, 1, 1, True, 1.0),                  # between 2^19 and 2^22: 8 per lane
    (8195, 64, 64, "sigmoid", True, 1, 1, 1, True, 1.0),
    (4111, 256, 8, "sigmoid", True, 8, 4, 2, True, 2.5),
    (20011, 160, 6, "softmax", True, 8, 3, 2, False, 16.0),
    (17003, 32, 32, "softmax", False, 1, 1, 1, True, 1.0),
]


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("cfg", LARGE_ROUTES, ids=lambda c: f"T{c[0]}E{c[1]}k{c[2]}{c[3][:3]}{'b' if c[4] else ''}g{c[5]}")
def test_route_of_large_batches(cfg, dtype, cuda):
    """Choice, weights and gradient against 64 bits: ordinary rows, rows of equal values, of values that 32-bit scores do not tell apart, rows
    with experts taken out and rows that are not routed; rows side by side and strided ones."""
    from nersemble_amd import experts as X
    T, E, k, sc, has_bias, G, tg, gt, renorm, scale = cfg
    sig = sc == "sigmoid"
    g = torch.Generator(device=cuda).manual_seed(E * 100 + k)
    x = torch.randn((T, E), generator=g, device=cuda) * 2
    x[1::5] = torch.round(x[1::5] * 2) / 2                                    # equal ones
    near = torch.rand((T, E), generator=g, device=cuda).argsort(1)[2::5].float()
    x[2::5] = torch.randn((T, 1), generator=g, device=cuda)[2::5] + near * 2.0 ** -22      # neighbours a step of fp32 apart
    x[3::5][torch.rand((T, E), generator=g, device=cuda)[3::5] < 0.3] = -np.inf
    x[7] = -np.inf
    x = x.to(DT[dtype])
    bias = torch.randn(E, generator=g, device=cuda) * 0.1 if has_bias else None
    if has_bias:
        bias[E // 2:] = bias[:E - E // 2].clone()                                     # (equal biases as well)
    sel = (torch.rand(T, generator=g, device=cuda) > 0.1).to(torch.uint8)
    dw = torch.randn((T, k), generator=g, device=cuda)
    for layout in ("side by side", "strided"):
        if layout == "strided":
            wide = torch.zeros((T, E + 40), dtype=x.dtype, device=cuda)
            wide[:, 3:3 + E] = x
            xd, s = wide[:, 3:3 + E].requires_grad_(True), sel
        else:
            xd, s = x.detach().clone().requires_grad_(True), None
        w, c = X.route_experts(xd, k, scores=sc, bias=bias, n_groups=G, top_groups=tg, group_top=gt, renormalise=renorm, scale=scale, selector=s)
        ww, wc, score, clear = _route64(x, k, sig, bias, G, tg, gt, renorm, scale, s)
        assert clear.double().mean() > 0.75
        assert torch.equal(c[clear].long(), wc[clear])
        # as _route_tol: span of the logits (what is taken out has none)
        span = float(torch.where(torch.isfinite(x), x.double().abs(), torch.zeros((), dtype=torch.float64, device=cuda)).max()) * 2
        rel = (span + (k if renorm else E) + 10) * 2 * U
        assert ((w.double() - ww).abs() <= rel * ww.abs() + 1e-37)[clear].all()
        (d,) = torch.autograd.grad(w, [xd], dw)
        assert d.dtype == x.dtype and d.shape == x.shape
        on, at = (wc >= 0).double(), wc.clamp(min=0)
        gw = dw.double() * ww * on
        total = gw.sum(1, keepdim=True)
        mag = gw.abs().sum(1, keepdim=True)
        val = gw - ww * total / scale if renorm else gw
        size = gw.abs() + (ww.abs() * mag / abs(scale) if renorm else 0.0)
        if sig:
            val, size = val * torch.sigmoid(-x.double()).gather(1, at), size * torch.sigmoid(-x.double()).gather(1, at)
        want = torch.zeros((T, E), dtype=torch.float64, device=cuda).scatter_add_(1, at, val * on)
        size = torch.zeros((T, E), dtype=torch.float64, device=cuda).scatter_add_(1, at, size * on)
        if not sig and not renorm:
            want, size = want - score * total, size + score * mag
        tol = 3 * (rel * size + 1e-37)
        if dtype != "fp32":
            h, tiny = HALF[DT[dtype]]
            tol = tol + h * want.abs() + tiny
        assert torch.isfinite(d).all() and ((d.double() - want).abs() <= tol)[clear].all()


@pytest.mark.parametrize("k", [1, 2, 3, 7, 16, 30, 32])
@pytest.mark.parametrize("T", [50, 16500, 131075])
def test_route_rows_that_are_compared_whole_in_64_bits(k, T, cuda):
    """Every row has more candidates in doubt than one: the wide entries of the redo move over to the narrow ones, which lie in the same
    memory, at 4, 8 and 16 values per lane."""
    from nersemble_amd import experts as X
    g = torch.Generator(device=cuda).manual_seed(k)
    E = 32
    x = torch.rand((T, E), generator=g, device=cuda).argsort(1).float() * 2.0 ** -23 + 0.25
    bias = torch.zeros(E, device=cuda)
    for sc in ("sigmoid", "softmax"):
        w, c = X.route_experts(x, k, scores=sc, bias=bias)
        ww, wc, _, clear = _route64(x, k, sc == "sigmoid", bias, 1, 1, 1, True, 1.0, None)
        assert clear.all() and torch.equal(c.long(), wc)
        assert ((w.double() - ww).abs() <= (1 + k + 10) * 2 * U * ww).all()


@pytest.mark.parametrize("sc", ["sigmoid", "softmax"])
def test_route_groups_with_infinite_biases_and_one_expert_left(sc, cuda):
    """A group whose second expert is taken out counts nothing, whatever the first one's bias: no more groups stay than were asked for."""
    from nersemble_amd import experts as X
    inf = np.float32(np.inf)
    rng = np.random.default_rng(1)
    E, G, T = 32, 8, 300
    x = rng.standard_normal((T, E)).astype(np.float32)
    bias = (rng.standard_normal(E) * 0.1).astype(np.float32)
    bias[8] = inf                                    # group 2: one expert with an infinite bias, the others taken out
    x[:, 9:12] = -inf
    bias[20], bias[21] = inf, inf                    # group 5: two of them
    bias[25] = -inf                                  # (an infinite bias takes out as well)
    x[::3, 28:31] = -inf
    for tg, k in ((1, 3), (2, 5), (3, 8)):
        with np.errstate(invalid="ignore"):
            ww, wc = ox.route(x, k, sc == "sigmoid", bias, G, tg, 2)
        w, c = X.route_experts(torch.from_numpy(x).to(cuda), k, scores=sc, bias=torch.from_numpy(bias).to(cuda), n_groups=G, top_groups=tg, group_top=2)
        assert np.array_equal(c.cpu().numpy(), wc), (tg, k)
        _close(w, ww, _route_tol(x, ww, k), "weights")


def test_routed_network_follows_its_weights_through_captured_steps(cuda):
    """Weights that change without a word to the autograd engine -- a captured optimizer's replays, ``.data`` -- and replays of a forward whose
    weights an eager step changed: what runs next reads them as they are."""
    from nersemble_amd import tcnn
    args = (20, 5, {"n_neurons": 64, "n_hidden_layers": 2}, {"n_experts": 6, "top_k": 2})
    net, fresh = tcnn.RoutedNetwork(*args).to(cuda), tcnn.RoutedNetwork(*args).to(cuda)
    g = torch.Generator(device=cuda).manual_seed(3)
    x = torch.randn((700, 20), generator=g, device=cuda)
    go = torch.randn((700, 5), generator=g, device=cuda).half()

    def now():
        """What a network made for these weights says."""
        other = tcnn.RoutedNetwork(*args).to(cuda)
        other.load_state_dict(net.state_dict())
        with torch.no_grad():
            return other(x)

    def step():
        out = net(x)
        (d,) = torch.autograd.grad(out, [net.params], go)
        with torch.no_grad():
            net.params.sub_(d, alpha=0.01)
        return out.detach()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    with torch.no_grad():
        net(x)                                          # (whatever a forward keeps, it has now)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for turn in range(3):
        want = now()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(res, want), turn             # the captured forward read the weights of its time
        with torch.no_grad():
            assert torch.equal(net(x), now()), turn     # an eager one those that the replay left
            net.params.data.mul_(1.01)
            assert torch.equal(net(x), now()), turn
            net.params.copy_(fresh.params * (1 + turn))
