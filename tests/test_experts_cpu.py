"""CPU: the routed-experts oracle against torch's autograd in 64 bits, and the refusals of the entry points (all argument checks
come before anything is launched, so they need no GPU)."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import experts as ox


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("renorm", [False, True])
def test_oracle_route_gradient_is_autograds(sigmoid, renorm):
    rng = np.random.default_rng(0)
    x, g = rng.standard_normal((6, 12)), rng.standard_normal((6, 4))
    bias = rng.standard_normal(12) * 0.1
    w, c = ox.route(x, 4, sigmoid, bias, 3, 2, 2, renorm, 2.5)
    t = torch.tensor(x, requires_grad=True)
    s = torch.sigmoid(t) if sigmoid else torch.softmax(t, 1)
    u = s.gather(1, torch.tensor(c).long())
    wt = 2.5 * (u / u.sum(1, keepdim=True) if renorm else u)
    assert np.allclose(wt.detach().numpy(), w, rtol=1e-12)
    (d,) = torch.autograd.grad(wt, [t], torch.tensor(g))
    assert np.allclose(d.numpy(), ox.route_bwd(x, w, c, g, sigmoid, renorm, 2.5), rtol=1e-9, atol=1e-13)


def test_oracle_route_choice_by_hand():
    x = np.log(np.array([[0.1, 0.4, 0.2, 0.3]]))
    w, c = ox.route(x, 2)
    assert c.tolist() == [[1, 3]] and np.allclose(w, [[4 / 7, 3 / 7]])
    w, c = ox.route(x, 2, renormalise=False, bias=np.array([1.0, 0, 0, 0]))
    assert c.tolist() == [[0, 1]] and np.allclose(w, [[0.1, 0.4]])
    w, c = ox.route(x, 2, n_groups=2, top_groups=1, group_top=2)          # 0.5 against 0.5 and a rounding: by sums
    assert set(c[0].tolist()) in ({0, 1}, {2, 3})
    w, c = ox.route(np.full((1, 4), -np.inf), 2)
    assert c.tolist() == [[-1, -1]] and (w == 0).all()


def test_oracle_products_and_join_are_autograds():
    rng = np.random.default_rng(1)
    T, k, E, K, N = 20, 3, 5, 6, 4
    chosen = np.argsort(rng.random((T, E)), axis=1)[:, :k].astype(np.int32)
    chosen[3] = -1
    offsets, rows, positions = ox.plan(chosen, E)
    assert offsets[-1] == (T - 1) * k and (np.sort(rows[:offsets[-1]]) == np.flatnonzero(chosen.reshape(-1) >= 0)).all()
    x, w, wt = rng.standard_normal((T, K)), rng.standard_normal((E, N, K)), rng.random((T, k))
    tx, tw, tt = (torch.tensor(v, requires_grad=True) for v in (x, w, wt))
    out = torch.zeros((T, N), dtype=torch.float64)
    for t in range(T):
        for j in range(k):
            if chosen[t, j] >= 0:
                out = out.index_add(0, torch.tensor([t]), (tt[t, j] * torch.relu(tw[chosen[t, j]] @ tx[t]))[None])
    g = rng.standard_normal((T, N))
    dx, dw, dt = torch.autograd.grad(out, [tx, tw, tt], torch.tensor(g))
    y, _ = ox.linear(x, w, offsets, rows, k, True, True)
    assert np.allclose(ox.combine(y, wt, positions)[0], out.detach().numpy())
    dy = np.zeros_like(y)
    for t in range(T):
        for j in range(k):
            if positions[t, j] >= 0:
                dy[positions[t, j]] = wt[t, j] * g[t]
                assert np.isclose(dt[t, j], (g[t] * y[positions[t, j]]).sum())
    ox_dx, _, ox_dw, _ = ox.linear_bwd(x, w, offsets, rows, k, True, np.where(y > 0, dy, 0))
    assert np.allclose(ox.combine(ox_dx, np.ones((T, k)), positions)[0], dx.numpy()) and np.allclose(ox_dw, dw.numpy())


def _refused(rc, *words):
    from nersemble_amd import _lib
    msg = _lib.lib().nsx_last_error().decode()
    assert rc < 0 and all(w in msg for w in words), (rc, msg)


def test_c_abi_refuses_bad_arguments():
    from nersemble_amd import _lib
    L = _lib.lib()
    P = ctypes.c_void_p(16)                    # (never dereferenced: every call below is refused or has nothing to do)

    def route(dtype=0, T=4, E=16, stride=16, k=2, G=1, tg=1, gt=1, scale=1.0, logits=P):
        return L.nsx_expert_route_fwd(logits, dtype, T, E, stride, None, None, k, 0, G, tg, gt, 1, scale, P, P, None, None)
    _refused(route(dtype=3), "dtype")
    _refused(route(E=0), "n_experts")
    _refused(route(E=513, stride=513), "n_experts")
    _refused(route(k=17), "top_k")
    _refused(route(k=0), "top_k")
    _refused(route(k=65, E=128, stride=128), "top_k")
    _refused(route(T=-1), "rows")
    _refused(route(T=1 << 30), "too many")
    _refused(route(stride=15), "stride")
    _refused(route(G=3), "groups")
    _refused(route(G=128, E=256, stride=256), "groups")
    _refused(route(G=4, tg=5), "top_groups")
    _refused(route(G=4, tg=1, k=5), "choices")
    _refused(route(G=16, tg=4, gt=2), "group_top")
    _refused(route(gt=3), "group_top")
    _refused(route(scale=0.0), "scale")
    _refused(route(scale=float("nan")), "scale")
    _refused(route(logits=None), "NULL")
    _refused(route(T=1 << 27, E=512, stride=512), "one launch")
    assert route(T=0) == 0
    rbwd = lambda **o: L.nsx_expert_route_bwd(o.get("x", P), 0, o.get("T", 4), 16, o.get("s", 16), 2, 0, 1, 1.0, P, P, o.get("g", P), P, None, None)  # noqa: E731
    _refused(rbwd(s=3), "stride")
    _refused(rbwd(g=None), "NULL")
    assert rbwd(T=0) == 0
    _refused(L.nsx_expert_plan_workspace(-1, 4), "entries")
    _refused(L.nsx_expert_plan_workspace(4, 0), "n_experts")
    assert L.nsx_expert_plan_workspace(4096, 16) > 0
    _refused(L.nsx_expert_plan(P, 4, 2, 4, None, P, P, P, None, None), "NULL")
    _refused(L.nsx_expert_plan(P, 1 << 30, 2, 4, P, P, P, P, None, None), "too many")
    _refused(L.nsx_expert_plan(None, 4, 2, 4, P, P, P, P, None, None), "NULL")

    def lin(dtype=1, stride=32, x_rows=8, rows=P, k=2, K=32, N=64, E=4, R=16, x=P, w=P, y=P, off=P):
        return L.nsx_expert_linear_fwd(x, dtype, stride, x_rows, rows, k, w, K, N, E, off, R, 0, y, None)
    _refused(lin(dtype=0), "16-bit")
    _refused(lin(K=30), "multiples of 8")
    _refused(lin(N=0), "multiples of 8")
    _refused(lin(N=16392), "multiples of 8")
    _refused(lin(stride=24), "stride")
    _refused(lin(stride=36), "stride")
    _refused(lin(x=ctypes.c_void_p(24)), "unaligned")
    _refused(lin(w=None), "NULL")
    _refused(lin(off=None), "offsets")
    _refused(lin(rows=None), "rows")
    _refused(lin(R=1 << 31), "ordered rows")
    assert lin(R=0) == 0

    def bwd(x=P, dtype=1, x_stride=32, x_rows=8, rows=P, positions=P, k=2, w=P, dy=P, dy_stride=64, y=None, y_stride=0, K=32, N=64, E=4,
            R=16, dx=P, dw=P, ws=P):
        return L.nsx_expert_linear_bwd(x, dtype, x_stride, x_rows, rows, positions, k, w, dy, dy_stride, y, y_stride, K, N, E, P, R, dx, 0,
                                       dw, ws, None)
    _refused(bwd(dtype=0), "16-bit")
    _refused(bwd(dy_stride=60), "strides")
    _refused(bwd(dy_stride=(1 << 20) + 8), "strides")
    _refused(bwd(y=P, y_stride=8), "strides")
    _refused(bwd(dy=None), "NULL")
    _refused(bwd(x_rows=7), "x has 7 rows")
    _refused(bwd(rows=None), "x has 8 rows")
    _refused(bwd(positions=None), "positions")
    _refused(bwd(w=None), "weight")
    _refused(bwd(x=None), "dw needs")
    _refused(bwd(x_stride=24), "dw needs")
    _refused(bwd(dw=ctypes.c_void_p(8)), "dw needs")
    _refused(bwd(ws=None), "workspace")
    _refused(bwd(x_rows=1 << 20, R=1 << 21, dx=None, ws=None), "workspace")
    assert bwd(R=0, x_rows=0, dw=None) == 0 and bwd(dx=None, dw=None) == 0
    _refused(L.nsx_expert_linear_bwd_workspace(16, 4, 33, 64, 1, 1, 1, 0), "multiples of 8")
    assert L.nsx_expert_linear_bwd_workspace(16, 4, 32, 64, 1, 1, 0, 1) == 16 * 32 * 2
    assert L.nsx_expert_linear_bwd_workspace(16, 4, 32, 64, 1, 0, 0, 1) == 0
    _refused(L.nsx_expert_combine_fwd(P, 1, 60, 16, 64, None, P, 8, 2, P, None, None), "stride")
    _refused(L.nsx_expert_combine_fwd(P, 0, 64, 16, 64, None, P, 8, 2, P, None, None), "16-bit")
    _refused(L.nsx_expert_combine_fwd(P, 1, 64, 16, 64, None, None, 8, 2, P, None, None), "NULL")
    _refused(L.nsx_expert_combine_bwd(P, 1, 64, 16, 64, P, P, None, 8, 2, P, P, P, None, None), "NULL")
    _refused(L.nsx_expert_combine_bwd(P, 1, 64, 16, 12, P, P, P, 8, 2, P, P, P, None, None), "multiple of 8")


def test_python_layer_refuses_bad_arguments():
    from nersemble_amd import experts as X
    T, k, E = 4, 2, 3
    i32 = torch.int32
    plan = X.ExpertPlan(torch.zeros(E + 1, dtype=i32), torch.zeros(T * k, dtype=i32), torch.zeros((T, k), dtype=i32))
    half = lambda *s: torch.zeros(s, dtype=torch.float16)  # noqa: E731
    bad = [
        lambda: X.route_experts(torch.zeros(4), 2),
        lambda: X.route_experts(torch.zeros((4, 4), dtype=torch.float64), 2),
        lambda: X.route_experts(torch.zeros((4, 4)), 2, scores="relu"),
        lambda: X.route_experts(torch.zeros((4, 4)), 2, bias=torch.zeros(3)),
        lambda: X.route_experts(torch.zeros((4, 4)), 2, selector=torch.zeros(3, dtype=torch.uint8)),
        lambda: X.expert_plan(torch.zeros((4, 2), dtype=torch.int64), 3),
        lambda: X.expert_plan(torch.zeros(4, dtype=i32), 3),
        lambda: X.expert_linear(torch.zeros((T, 8)), torch.zeros((E, 8, 8)), plan),
        lambda: X.expert_linear(half(T, 8), torch.zeros((E, 8, 8), dtype=torch.bfloat16), plan),
        lambda: X.expert_linear(half(T, 8), half(E + 1, 8, 8), plan),
        lambda: X.expert_linear(half(T, 16), half(E, 8, 8), plan),
        lambda: X.expert_linear(half(T * k, 8), half(E, 8, 8), plan, gather=True),
        lambda: X.expert_linear(half(T, 8), half(E, 8, 8), plan, gather=False),
        lambda: X.expert_linear(half(T, 8), torch.zeros((E, 8, 8)), plan, w16=half(E, 8, 16)),
        lambda: X.expert_linear(half(T, 8), half(E, 8, 8), X.ExpertPlan(plan.offsets, plan.rows[1:], plan.positions)),
        lambda: X.expert_combine(half(T, 8), torch.zeros((T, k)), plan),
        lambda: X.expert_combine(half(T * k, 8), torch.zeros((T, k + 1)), plan),
        lambda: X.expert_combine(half(T * k, 8), torch.zeros((T, k), dtype=i32), plan),
    ]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()
    with pytest.raises(AttributeError):                       # (checked once, in the constructor)
        plan.rows = plan.rows[:1]
    for f in (lambda: X.route_experts(torch.zeros((4, 4)), 2), lambda: X.expert_plan(torch.zeros((4, 2), dtype=i32), 3),
              lambda: X.expert_linear(half(T, 8), half(E, 8, 8), plan), lambda: X.expert_combine(half(T * k, 8), torch.zeros((T, k)), plan)):
        with pytest.raises(RuntimeError, match="device tensors"):
            f()


def test_workspace_of_a_gathered_gradient():
    """One choice of a row is rounded as it is; the terms of more are kept in 32 bits until they are summed."""
    from nersemble_amd import _lib
    ws = _lib.lib().nsx_expert_linear_bwd_workspace
    assert ws(16, 4, 32, 64, 1, 1, 0, 0) == 16 * 32 * 2
    assert ws(16, 4, 32, 64, 1, 2, 0, 0) == ws(16, 4, 32, 64, 1, 8, 0, 0) == 16 * 32 * 4
    assert ws(16, 4, 32, 64, 1, 0, 0, 0) == 0
    _refused(ws(16, 4, 32, 64, 1, -1, 0, 0), "choices")
    _refused(ws(16, 4, 32, 64, 1, 65, 0, 0), "choices")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_routed_networks_logits_are_32_bits_under_autocast(dtype, monkeypatch):
    from nersemble_amd import experts as X
    from nersemble_amd import tcnn
    net = tcnn.RoutedNetwork(20, 5, {"n_neurons": 64}, {"n_experts": 6, "top_k": 2})
    seen = []

    def route(logits, *args, **kw):
        seen.append(logits)
        raise InterruptedError
    monkeypatch.setattr(X, "route_experts", route)
    x = torch.randn((30, 20), generator=torch.Generator().manual_seed(0))
    for on in (False, True):
        with torch.autocast("cpu", dtype=dtype, enabled=on), pytest.raises(InterruptedError):
            net(x)
    assert seen[1].dtype == torch.float32 and torch.equal(seen[0], seen[1])


def test_forward_mode_derivatives_are_refused():
    """A dual tensor has no ``requires_grad``: its tangent would be lost without a word."""
    import torch.autograd.forward_ad as fwd
    from nersemble_amd import experts as X
    T, k, E = 4, 2, 3
    i32 = torch.int32
    plan = X.ExpertPlan(torch.zeros(E + 1, dtype=i32), torch.zeros(T * k, dtype=i32), torch.zeros((T, k), dtype=i32))
    half = lambda *s: torch.zeros(s, dtype=torch.float16)                    # noqa: E731
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))                # noqa: E731
        for call in (lambda: X.route_experts(dual(torch.zeros((T, E))), k), lambda: X.expert_linear(dual(half(T, 8)), half(E, 8, 8), plan),
                     lambda: X.expert_linear(half(T, 8), dual(half(E, 8, 8)), plan),
                     lambda: X.expert_linear(half(T, 8), dual(torch.zeros((E, 8, 8))), plan, w16=half(E, 8, 8)),
                     lambda: X.expert_linear(half(T, 8), torch.zeros((E, 8, 8)), plan, w16=dual(half(E, 8, 8))),
                     lambda: X.expert_combine(dual(half(T * k, 8)), torch.zeros((T, k)), plan),
                     lambda: X.expert_combine(half(T * k, 8), dual(torch.zeros((T, k))), plan)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with pytest.raises(RuntimeError, match="device tensors"):            # (no tangent: as outside)
            X.route_experts(torch.zeros((T, E)), k)


@pytest.mark.parametrize("E,k", [(16, 0), (16, 17), (128, 65), (16, -1), (4, 1 << 40), (0, 1), (513, 1)])
def test_route_refuses_sizes_before_it_makes_results(E, k):
    from nersemble_amd import experts as X
    with pytest.raises(RuntimeError, match="n_experts" if E in (0, 513) else "top_k"):
        X.route_experts(torch.zeros((4, E)), k)


def test_binding_of_another_torch_is_built_again(tmp_path, monkeypatch):
    from nersemble_amd.csrc import build
    so, stamp, src = (str(tmp_path / n) for n in ("b.so", "b.txt", "b.cpp"))
    open(src, "w").close()
    assert build.binding_is_stale(so, stamp, [src])
    open(so, "w").close()
    assert build.binding_is_stale(so, stamp, [src])                     # (nothing says what it was built against)
    with open(stamp, "w") as f:
        f.write(build._built_against())
    assert not build.binding_is_stale(so, stamp, [src])
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert build.binding_is_stale(so, stamp, [src])


@pytest.mark.parametrize("what", ["nsx_version", "torch_version"])
def test_binding_of_another_library_or_torch_is_not_used(what, monkeypatch):
    """Its calls would pass other arguments, or tensors of another layout."""
    from nersemble_amd import csrc, experts as X
    X._FastNotLoaded().plan                                             # (loads the one that is there)
    from nersemble_amd.csrc import _experts

    class Other:
        nsx_version, torch_version, plan = _experts.nsx_version, _experts.torch_version, None
    setattr(Other, what, "other")
    monkeypatch.setattr(csrc, "_experts", Other)
    monkeypatch.setattr(X, "_fast", X._FastNotLoaded())
    with pytest.raises(RuntimeError, match="Build it again"):
        X.expert_plan(torch.zeros((4, 2), dtype=torch.int32), 3)
