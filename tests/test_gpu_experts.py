"""Routing, layout by expert and combination on the device against the float64 oracle (oracle/experts_oracle.py).

Tolerances, u = 2^-24 (2^-53 for float64): the chosen experts and the plan are integers and must be equal.  Weights that are formed in
64 bits carry one rounding; the plain softmax carries its exponentials (argument rounding |x - max| u, function 2 u), a sum of at most 16
terms a lane and 6 steps across lanes, a division and a product: (|x - max| + 32) u.  A result of a 16-bit type adds half a step, eps / 2.
"""
import numpy as np
import pytest
import torch

from oak import experts as ox
from oracle import experts_oracle as eo

pytestmark = pytest.mark.gpu
DT = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def unit(dtype):
    return 2.0 ** -53 if dtype == "f64" else 2.0 ** -24


def half_step(dtype, ref):
    """Half a step of the type around ref; float16 numbers below 2^-14 are 2^-24 apart."""
    return torch.finfo(DT[dtype]).eps / 2 * np.abs(ref) + (2.0 ** -25 if dtype == "f16" else 0.0)


def tensor(a, dtype=None, pad=0):
    """On the device; ``pad`` puts the rows into a wider array one element off its start."""
    t = torch.as_tensor(np.ascontiguousarray(a)).to("cuda")
    t = t if dtype is None else t.to(DT[dtype])
    if pad:
        store = torch.full((t.shape[0], t.shape[1] + pad), float("nan") if t.is_floating_point() else 0, dtype=t.dtype, device="cuda")
        store[:, 1:1 + t.shape[1]] = t
        t = store[:, 1:1 + t.shape[1]]
    return t


def back(t):
    return t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def scores_of(rng, n, e, dtype, pad=0, spread=1.5):
    t = tensor(rng.standard_normal((n, e)) * spread, dtype, pad)
    return t, back(t)


ROUTE = [
    # n, E, k, dtype, options
    (1, 1, 1, "f32", {}),
    (5, 2, 2, "bf16", {"score": "sigmoid"}),
    (257, 7, 3, "f32", {"renormalise": False}),
    (33, 16, 16, "f16", {}),
    (100, 17, 4, "bf16", {"bias": True}),
    (301, 24, 2, "f32", {"renormalise": False, "pad": 5}),
    (64, 33, 5, "f64", {"mask": 0.5}),
    (130, 64, 6, "bf16", {"pad": 3}),
    (70, 65, 8, "f32", {"score": "sigmoid", "bias": True, "scale": 2.5}),
    (50, 128, 1, "bf16", {"renormalise": False, "mask": 0.1}),
    (43, 160, 6, "bf16", {"renormalise": False, "mask": 0.9}),
    (90, 256, 8, "bf16", {"score": "sigmoid", "bias": True, "n_groups": 8, "top_groups": 4, "group_score": "top2", "scale": 2.5}),
    (31, 300, 16, "f16", {"bias": True, "n_groups": 10, "top_groups": 3}),
    (20, 513, 64, "f32", {"score": "sigmoid", "renormalise": False}),
    (9, 1024, 33, "f64", {"bias": True, "mask": 0.7, "n_groups": 64, "top_groups": 9, "group_score": "top2"}),
    (200, 60, 4, "bf16", {"n_groups": 6, "top_groups": 2, "mask": 0.15}),
    (65, 64, 3, "f32", {"n_groups": 64, "top_groups": 3, "group_score": "top2"}),
    (65, 64, 3, "f32", {"n_groups": 1, "mask": "shared"}),
]


def route_case(n, e, k, dtype, opt, seed=0):
    rng = np.random.default_rng(seed + 1000 * e + n)
    opt = dict(opt)
    x, xr = scores_of(rng, n, e, dtype, opt.pop("pad", 0))
    kw = dict(opt)
    host = dict(opt)
    if opt.get("bias"):
        b = torch.as_tensor(rng.standard_normal(e) * 0.05, dtype=torch.float32, device="cuda")
        kw["bias"], host["bias"] = b, back(b)
    if "mask" in opt:
        m = rng.random(e) < 0.5 if opt["mask"] == "shared" else rng.random((n, e)) < opt["mask"]
        if opt["mask"] != "shared" and n > 2:
            m[n // 2] = False                                            # a row that is left nothing
        kw["mask"], host["mask"] = torch.as_tensor(m, device="cuda"), m
    return x, xr, kw, host


def check_weights(w, ref, xr, experts, dtype, kw):
    formed_wide = kw.get("renormalise", True) or kw.get("score") == "sigmoid"
    far = np.ptp(np.where(np.isfinite(xr), xr, 0.0)) if xr.size else 0.0
    tol = (2 if formed_wide and dtype != "f64" else far + 32) * unit(dtype)
    np.testing.assert_allclose(w, ref, rtol=tol, atol=1e-37)


@pytest.mark.parametrize("n,e,k,dtype,opt", ROUTE)
def test_route(n, e, k, dtype, opt):
    x, xr, kw, host = route_case(n, e, k, dtype, opt)
    ex, w = ox.route(x, k, **kw)
    er, wr = eo.route(xr, k, **host)
    assert ex.dtype == torch.int32 and w.dtype == (torch.float64 if dtype == "f64" else torch.float32)
    np.testing.assert_array_equal(back(ex), er)
    check_weights(back(w), wr, xr, er, dtype, kw)


@pytest.mark.parametrize("n,e,k,dtype,opt", ROUTE)
def test_route_grad(n, e, k, dtype, opt):
    x, xr, kw, host = route_case(n, e, k, dtype, opt)
    ex, _ = ox.route(x, k, **kw)
    for name in ("bias", "n_groups", "top_groups", "group_score"):
        kw.pop(name, None), host.pop(name, None)
    rng = np.random.default_rng(7)
    dw = torch.as_tensor(rng.standard_normal((n, k)), dtype=torch.float64 if dtype == "f64" else torch.float32, device="cuda")
    dx = ox.route_grad(x, ex, dw, **kw)
    assert dx.dtype == x.dtype and dx.shape == x.shape
    ref = eo.route_grad(xr, back(ex), back(dw), **host)
    # every probability carries (|x - max| + 32) u, the bracket a few u of its two parts; the result one rounding
    far = np.ptp(xr) if xr.size else 0.0
    g = kw.get("scale", 1.0) * np.abs(back(dw)).max(initial=0.0)
    one = np.exp(xr - xr.max(1, keepdims=True)) if kw.get("score", "softmax") == "softmax" else np.ones_like(xr)
    tol = 2 * (far + 40) * unit(dtype) * 2 * g * np.minimum(one * e, 1.0) + half_step(dtype, ref) + 1e-37
    assert (np.abs(back(dx) - ref) <= tol).all(), np.abs(back(dx) - ref).max()


def test_route_ties_go_to_the_lowest_expert():
    x = torch.zeros(3, 100, device="cuda", dtype=torch.bfloat16)
    x[1, 40:60] = 1.0
    x[2] = torch.arange(100, device="cuda") % 2
    ex, w = ox.route(x, 5)
    np.testing.assert_array_equal(back(ex), [[0, 1, 2, 3, 4], [40, 41, 42, 43, 44], [1, 3, 5, 7, 9]])
    np.testing.assert_allclose(back(w), 0.2, rtol=2 * 2.0 ** -24)
    ex, _ = ox.route(x, 5, bias=torch.zeros(100, device="cuda"), score="sigmoid", n_groups=10, top_groups=2)
    np.testing.assert_array_equal(back(ex)[0], [0, 1, 2, 3, 4])
    np.testing.assert_array_equal(back(ex)[1], [40, 41, 42, 43, 44])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [True, False])
def test_route_infinities_nan_and_lowest_values(score, renormalise):
    inf, nan, low = np.inf, np.nan, float(np.finfo(np.float32).min)
    x = np.array([[1.0, -inf, 2.0, 0.0], [-inf, -inf, -inf, -inf], [1.0, nan, 2.0, 0.0], [inf, 1.0, 0.0, 0.0], [low, low, low, low],
                  [low, 3.0, low, -inf], [nan, inf, 1.0, 2.0], [-200.0, -201.0, -300.0, -250.0]])
    mask = np.ones_like(x, bool)
    mask[6, :2] = False                                                  # NaN and infinity in masked places do no harm
    t, m = tensor(x, "f32"), torch.as_tensor(mask, device="cuda")
    kw = dict(score=score, renormalise=renormalise, mask=m)
    ex, w = ox.route(t, 3, **kw)
    er, wr = eo.route(back(t), 3, score=score, renormalise=renormalise, mask=mask)
    np.testing.assert_array_equal(back(ex), er)
    np.testing.assert_allclose(back(w), wr, rtol=64 * 2.0 ** -24, atol=1e-37)
    dw = torch.ones(len(x), 3, device="cuda") * torch.arange(1, 4, device="cuda")
    dx = back(ox.route_grad(t, ex, dw, **kw))
    ref = eo.route_grad(back(t), er, back(dw), score=score, renormalise=renormalise, mask=mask)
    assert (dx[1] == 0).all() and (dx[2] == 0).all() and (dx[3] == 0).all()    # rows without experts
    np.testing.assert_allclose(dx, ref, rtol=64 * 2.0 ** -24, atol=256 * 2.0 ** -24)


def test_route_strides_offsets_and_empty():
    rng = np.random.default_rng(3)
    base = tensor(rng.standard_normal((40, 50)), "bf16")
    ex, w = ox.route(base.t(), 4)                                        # columns not consecutive
    er, wr = eo.route(back(base).T, 4)
    np.testing.assert_array_equal(back(ex), er)
    one = base[:1].expand(9, 50)                                         # row stride 0
    ex, _ = ox.route(one, 2)
    np.testing.assert_array_equal(back(ex), np.repeat(eo.route(back(base[:1]), 2)[0], 9, 0))
    ex, w = ox.route(base[:0], 4)
    assert ex.shape == (0, 4) and w.shape == (0, 4)
    assert ox.route_grad(base[:0], ex, w).shape == (0, 50)


PLANS = [(0, 2, 5), (1, 1, 1), (3, 2, 16), (64, 1, 7), (1000, 6, 160), (4096, 4, 1024), (4097, 4, 24), (5000, 4, 1025), (40000, 2, 3),
         (70001, 8, 333), (6000, 3, 4096), (16385, 1, 1), (100003, 3, 24), (30000, 6, 32),
         (30000, 6, 33), (1 << 20, 1, 2), (349526, 3, 32)]


@pytest.mark.parametrize("n,k,e", PLANS)
def test_plan(n, k, e):
    rng = np.random.default_rng(n + e)
    ex = rng.integers(-1, e, (n, k))
    ex[rng.random((n, k)) < 0.3] = e // 2                                # one much sought after
    p = ox.plan(torch.as_tensor(ex, dtype=torch.int32, device="cuda"), e)
    for got, ref in zip(p[:4], eo.plan(ex, e)):
        np.testing.assert_array_equal(back(got), ref)
    p64 = ox.plan(torch.as_tensor(ex, dtype=torch.int64, device="cuda"), e)
    np.testing.assert_array_equal(back(p64.positions), back(p.positions))


def test_plan_of_labels_and_of_numbers_that_are_no_experts():
    labels = np.array([2, 0, 2, 1, 0, 2], dtype=np.int32)
    p = ox.plan(torch.as_tensor(labels, device="cuda"), 3)
    np.testing.assert_array_equal(back(p.rows), [1, 4, 3, 0, 2, 5])
    np.testing.assert_array_equal(back(p.offsets), [0, 2, 3, 6])
    assert p.positions.shape == (6,)
    for dtype in (torch.int32, torch.int64):
        odd = torch.as_tensor([[0, 7], [-5, 1], [2 ** 31 - 1, 2]], dtype=dtype, device="cuda")
        p = ox.plan(odd, 3)
        np.testing.assert_array_equal(back(p.positions), [[0, -1], [-1, 1], [-1, 2]])
        np.testing.assert_array_equal(back(p.rows), [0, 1, 2, -1, -1, -1])
    p = ox.plan(torch.as_tensor([2 ** 32, 0], dtype=torch.int64, device="cuda"), 3)
    np.testing.assert_array_equal(back(p.positions), [-1, 0])


MIXES = [(1, 1, 1, 1, "f32", 0), (3, 2, 16, 64, "f32", 0), (50, 2, 5, 17, "f64", 0), (200, 6, 40, 33, "bf16", 3), (129, 4, 7, 257, "f16", 1),
         (64, 8, 8, 2048, "bf16", 0), (31, 3, 3, 4100, "f32", 5), (2500, 2, 24, 3, "bf16", 0), (10, 64, 64, 8, "f64", 0)]


@pytest.mark.parametrize("n,k,e,c,dtype,pad", MIXES)
def test_dispatch_combine_and_gradients(n, k, e, c, dtype, pad):
    rng = np.random.default_rng(n * c + k)
    ex = np.stack([rng.permutation(e)[:k] for _ in range(n)])
    ex[rng.random((n, k)) < 0.2] = -1
    p = ox.plan(torch.as_tensor(ex, dtype=torch.int32, device="cuda"), e)
    used, pos = int(p.offsets[e]), back(p.positions)
    wide = torch.float64 if dtype == "f64" else torch.float32
    u = unit(dtype)
    X = tensor(rng.standard_normal((n, c)), dtype, pad)
    laid = ox.dispatch(X, p)
    np.testing.assert_array_equal(back(laid), eo.dispatch(back(X), back(p.rows)))
    F = tensor(rng.standard_normal((n * k, c)), dtype, pad)
    F[used:] = float("nan")                                              # never read
    w = torch.as_tensor(rng.standard_normal((n, k)), dtype=wide, device="cuda")
    y = ox.combine(F, w, p)
    Fr, wr = back(F), back(w)
    ref = eo.combine(Fr, wr, pos)
    size = eo.combine(np.abs(Fr), np.abs(wr), pos)
    assert (np.abs(back(y) - ref) <= (k + 1) * u * size + half_step(dtype, ref)).all()
    dy = tensor(rng.standard_normal((n, c)), dtype, pad)
    dF, dw = ox.combine_grad(F, w, p, dy)
    dFr, dwr = eo.combine_grad(np.where(np.isnan(Fr), 0.0, Fr), wr, pos, back(dy))
    assert (np.abs(back(dF) - dFr) <= u * np.abs(dFr) + half_step(dtype, dFr)).all()
    assert (back(dF)[used:] == 0).all()
    _, sizes = eo.combine_grad(np.abs(np.where(np.isnan(Fr), 0.0, Fr)), wr, pos, np.abs(back(dy)))
    assert (np.abs(back(dw) - dwr) <= (c / 8 + 20) * u * sizes).all() and dw.dtype == wide
    dX = ox.dispatch_grad(F, p)
    ones = np.ones((n, k))
    dXr = eo.combine(Fr, ones, pos)
    assert (np.abs(back(dX) - dXr) <= (k + 1) * u * eo.combine(np.abs(Fr), ones, pos) + half_step(dtype, dXr)).all()


def test_combine_shows_the_weights_of_a_row_without_an_answer():
    x = torch.tensor([[0.0, 1.0], [float("nan"), 0.0]], device="cuda")
    ex, w = ox.route(x, 1)
    p = ox.plan(ex, 2)
    y = ox.combine(torch.ones(2, 3, device="cuda"), w, p)
    assert (back(y)[0] == 1).all() and np.isnan(back(y)[1]).all()


def test_mix_of_vectors_and_of_nothing():
    p = ox.plan(torch.tensor([1, 0, 1], dtype=torch.int32, device="cuda"), 2)
    X = torch.tensor([1.0, 2.0, 3.0], device="cuda")
    laid = ox.dispatch(X, p)
    np.testing.assert_array_equal(back(laid), [2, 1, 3])
    np.testing.assert_array_equal(back(ox.combine(laid, torch.ones(3, 1, device="cuda"), p)), [1, 2, 3])
    np.testing.assert_array_equal(back(ox.dispatch_grad(laid, p)), [1, 2, 3])
    empty = ox.plan(torch.empty(0, 2, dtype=torch.int32, device="cuda"), 4)
    assert ox.dispatch(torch.empty(0, 5, device="cuda"), empty).shape == (0, 5)
    assert ox.dispatch(torch.empty(3, 0, device="cuda"), p).shape == (3, 0)


def test_numpy_arrays_give_the_same_numbers():
    rng = np.random.default_rng(11)
    x, b = rng.standard_normal((77, 20)), rng.standard_normal(20) * 0.05
    m = rng.random((77, 20)) < 0.6
    for kw in (dict(), dict(score="sigmoid", bias=b, n_groups=4, top_groups=2), dict(renormalise=False, mask=m), dict(mask=m[0])):
        ex, w = ox.route(x, 3, **kw)
        er, wr = eo.route(x, 3, **kw)
        np.testing.assert_array_equal(ex, er)
        np.testing.assert_allclose(w, wr, rtol=1e-13, atol=1e-300)
        kw = {k: v for k, v in kw.items() if k in ("score", "renormalise", "mask")}
        dw = rng.standard_normal((77, 3))
        np.testing.assert_allclose(ox.route_grad(x, ex, dw, **kw), eo.route_grad(x, er, dw, **kw), rtol=1e-12, atol=1e-14)
    for shape, e in (((77, 3), 20), ((9000, 4), 50), ((30,), 4), ((0, 2), 3)):
        ex = rng.integers(-1, e, shape)
        p = ox.plan(ex, e)
        for got, ref in zip(p[:4], eo.plan(ex, e)):
            np.testing.assert_array_equal(got, ref)
    ex = rng.integers(-1, 20, (77, 3))
    p = ox.plan(ex, 20)
    X, F, w, dy = rng.standard_normal((77, 5)), rng.standard_normal((231, 5)), rng.standard_normal((77, 3)), rng.standard_normal((77, 5))
    np.testing.assert_array_equal(ox.dispatch(X, p), eo.dispatch(X, p.rows))
    np.testing.assert_allclose(ox.combine(F, w, p), eo.combine(F, w, p.positions), rtol=1e-12, atol=1e-13)
    for got, ref in zip(ox.combine_grad(F, w, p, dy), eo.combine_grad(F, w, p.positions, dy)):
        np.testing.assert_allclose(got, ref, rtol=1e-12, atol=1e-13)
    np.testing.assert_allclose(ox.dispatch_grad(F, p), eo.combine(F, np.ones((77, 3)), p.positions), rtol=1e-12, atol=1e-13)


def test_gradients_against_differences():
    """sum(c * combine(F, route(x))) differentiated through the calls of this module and by central differences (float64)."""
    rng = np.random.default_rng(5)
    n, e, k, c = 12, 9, 3, 4
    x, coef = rng.standard_normal((n, e)) * 1.5, rng.standard_normal((n, c))
    F = rng.standard_normal((n * k, c))
    for kw in (dict(), dict(renormalise=False), dict(score="sigmoid", scale=1.7), dict(score="sigmoid", renormalise=False)):
        ex, w = ox.route(x, k, **kw)
        p = ox.plan(ex, e)
        dF, dw = ox.combine_grad(F, w, p, coef)
        dx = ox.route_grad(x, ex, dw, **kw)

        def value(xx, ff):
            ee, ww = ox.route(xx, k, **kw)
            assert (ee == ex).all()
            return (coef * ox.combine(ff, ww, p)).sum()

        h = 1e-5
        for i, j in ((0, ex[0, 0]), (3, ex[3, 1]), (7, ex[7, 2]), (5, int(np.argmin(x[5])))):
            up, down = x.copy(), x.copy()
            up[i, j] += h
            down[i, j] -= h
            assert abs((value(up, F) - value(down, F)) / (2 * h) - dx[i, j]) <= 1e-8
        for s, j in ((0, 0), (20, 3)):
            up, down = F.copy(), F.copy()
            up[s, j] += h
            down[s, j] -= h
            assert abs((value(x, up) - value(x, down)) / (2 * h) - dF[s, j]) <= 1e-8


def test_streams_and_captured_graphs():
    """Another stream than the default one, and a captured step that is replayed on new inputs between eager work."""
    rng = np.random.default_rng(2)
    n, e, k, c = 3000, 40, 4, 96
    x, X, dy = tensor(rng.standard_normal((n, e)), "f32"), tensor(rng.standard_normal((n, c)), "bf16"), tensor(rng.standard_normal((n, c)), "bf16")

    def step():
        ex, w = ox.route(x, k, renormalise=False)
        p = ox.plan(ex, e)
        laid = ox.dispatch(X, p)
        y = ox.combine(laid, w, p)
        dF, dw = ox.combine_grad(laid, w, p, dy)
        return ex, w, p.rows, p.positions, p.offsets, laid, y, dF, dw, ox.route_grad(x, ex, dw, renormalise=False), ox.dispatch_grad(dF, p)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(step(), other):
        assert torch.equal(a, b)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.cuda.graph(second):
        held2 = step()
    for seed in range(4):
        x.copy_(tensor(np.random.default_rng(seed).standard_normal((n, e)), "f32"))
        X.copy_(tensor(np.random.default_rng(seed + 50).standard_normal((n, c)), "bf16"))
        graph.replay()
        second.replay()
        torch.cuda.synchronize()
        for a, b, c2 in zip(step(), held, held2):
            assert torch.equal(a, b) and torch.equal(a, c2)


def test_offsets_beyond_32_bits():
    """Rows whose offset in elements passes 2^31: strided scores, a laid-out array of more than 2^32 bytes."""
    rng = np.random.default_rng(9)
    far = (1 << 30) + 7
    store = torch.zeros(2 * far + 64, device="cuda", dtype=torch.bfloat16)
    x = store.as_strided((3, 64), (far, 1))
    x.copy_(tensor(rng.standard_normal((3, 64)), "bf16"))
    ex, w = ox.route(x, 4)
    er, wr = eo.route(back(x), 4)
    np.testing.assert_array_equal(back(ex), er)
    p = ox.plan(ex, 64)
    laid = ox.dispatch(x, p)
    np.testing.assert_array_equal(back(laid), eo.dispatch(back(x), back(p.rows)))
    del store, x
    n, c = 300_000, 8192                                                 # 2.46e9 elements laid out
    ex = torch.arange(n, device="cuda", dtype=torch.int32).flip(0) % 7
    p = ox.plan(ex, 7)
    X = torch.arange(n, device="cuda", dtype=torch.float32).remainder(251).to(torch.bfloat16)[:, None].expand(n, c)
    laid = ox.dispatch(X, p)
    rows = p.rows.long()
    at = torch.tensor([0, 1, n // 2, n - 2, n - 1], device="cuda")
    assert torch.equal(laid[at], X[rows[at]])
    y = ox.combine(laid, torch.ones(n, 1, device="cuda"), p)
    assert torch.equal(y[at], X[at])
    dF, dw = ox.combine_grad(laid, torch.ones(n, 1, device="cuda"), p, y)
    assert torch.equal(dF[at], laid[at])
    np.testing.assert_allclose(back(dw[at, 0]), c * back(X[at, 0]) ** 2, rtol=1e-5)


def test_more_rows_than_one_launch_takes():
    """The rows of a call are walked in several launches beyond 2^23 workgroups (inputs with row stride 0 keep them small)."""
    n = (1 << 30) + 5
    ex, w = ox.route(torch.tensor([[1.0, 3.0]], device="cuda", dtype=torch.float16).expand(n, 2), 1)
    for part in (slice(0, 3), slice((1 << 30) - 3, (1 << 30) + 5)):
        assert (ex[part] == 1).all() and (w[part] == 1).all()
    assert int(ex.min()) == 1
    del ex, w
    n, c = (1 << 23) + 3, 1032                                           # 129 units a row: one row a workgroup
    p = ox.plan(torch.zeros(n, device="cuda", dtype=torch.int32), 1)
    y = ox.combine(torch.full((1, c), 2.0, device="cuda", dtype=torch.bfloat16).expand(n, c), torch.full((n, 1), 3.0, device="cuda"), p)
    assert (y[-4:] == 6).all() and (y[:2] == 6).all() and bool((y[:, 0] == 6).all())


def test_refusals_on_the_device():
    x = torch.randn(4, 6, device="cuda")
    ex, w = ox.route(x, 2)
    p = ox.plan(ex, 6)
    cases = [
        lambda: ox.route(x.clone().requires_grad_(), 2), lambda: ox.route(x, 2, bias=np.zeros(6)), lambda: ox.route(x, 2, bias=torch.zeros(6)),
        lambda: ox.route(x.to(torch.int32), 2), lambda: ox.route(x, 7), lambda: ox.route(x, 0), lambda: ox.route(x, 2 ** 32 + 1),
        lambda: ox.route(x, 1.5), lambda: ox.route(x, 2, mask=torch.ones(4, 5, device="cuda", dtype=torch.bool)),
        lambda: ox.route(x, 2, mask=torch.ones(4, 6, device="cuda")), lambda: ox.route(torch.randn(2, 1025, device="cuda"), 2),
        lambda: ox.route_grad(x, ex, w[:, :1]), lambda: ox.route_grad(x, ex.float(), w), lambda: ox.route_grad(x, back(ex), w),
        lambda: ox.plan(ex, 2 ** 32 + 6), lambda: ox.plan(ex.float(), 6), lambda: ox.plan(ex[:, None], 6), lambda: ox.plan(ex, 5000),
        lambda: ox.dispatch(back(x), p), lambda: ox.dispatch(x[:3], p), lambda: ox.combine(x, w, p), lambda: ox.combine(torch.zeros(8, 3), w, p),
        lambda: ox.combine(torch.zeros(8, 3, device="cuda"), w, p._replace(positions=p.positions[:2])),
        lambda: ox.combine(torch.zeros(8, 3, device="cuda"), w, p._replace(positions=p.positions.long())),
        lambda: ox.combine(torch.zeros(8, 3, device="cuda"), w, p._replace(n_experts=9)),
        lambda: ox.combine_grad(torch.zeros(8, 3, device="cuda"), w, p, torch.zeros(4, 2, device="cuda")),
    ]
    for i, call in enumerate(cases):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"case {i} was not refused")


def test_two_threads_at_once():
    """Device calls share no state: two threads on streams of their own get what one gets."""
    import threading
    rng = np.random.default_rng(0)
    xs = [tensor(rng.standard_normal((5000, 48)), "bf16") for _ in range(2)]
    ref = [ox.route(x, 4, renormalise=False) for x in xs]
    plans = [ox.plan(r[0], 48) for r in ref]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                ex, w = ox.route(xs[i], 4, renormalise=False)
                p = ox.plan(ex, 48)
                torch.cuda.current_stream().synchronize()
                if not (torch.equal(ex, ref[i][0]) and torch.equal(w, ref[i][1]) and torch.equal(p.positions, plans[i].positions)):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [True, False])
def test_float64_at_the_ends_of_its_range(score, renormalise):
    """Finite scores stay open, the lowest double among them; sigmoids far out on both sides; saturated probabilities do not tie."""
    low, high = float(np.finfo(np.float64).min), 1e300
    x = np.array([[low, low, -np.inf, low], [low, 1.0, low, 2.0], [800.0, -800.0, 750.0, -750.0], [-800.0, -900.0, -1e5, -1e6],
                  [50.0, 60.0, 55.0, 40.0], [high, 0.0, -high, 1.0], [0.0, -0.0, 0.0, -0.0]])
    dw = np.arange(1.0, 1.0 + x.shape[0] * 3).reshape(-1, 3)
    ex, w = ox.route(x, 3, score=score, renormalise=renormalise)
    er, wr = eo.route(x, 3, score=score, renormalise=renormalise)
    np.testing.assert_array_equal(ex, er)
    np.testing.assert_allclose(w, wr, rtol=1e-13, atol=1e-300)
    dx, ref = ox.route_grad(x, ex, dw, score=score, renormalise=renormalise), eo.route_grad(x, er, dw, score=score, renormalise=renormalise)
    np.testing.assert_allclose(dx, ref, rtol=1e-12, atol=1e-13)
    grouped = dict(score=score, renormalise=renormalise, n_groups=2, top_groups=1, group_score="top2")
    ex, w = ox.route(x[1:], 2, **grouped)
    np.testing.assert_array_equal(ex, eo.route(x[1:], 2, **grouped)[0])


def test_saturated_probabilities_do_not_tie_without_a_bias():
    """Scores whose sigmoids agree in every bit that 64 bits hold are still told apart: the choice goes by the scores."""
    x = torch.tensor([[40.0, 41.0, 39.0, 42.0, 45.0, 44.0, 43.0, 46.0]], device="cuda")
    for dtype in ("f32", "bf16", "f64"):
        ex, _ = ox.route(x.to(DT[dtype]), 3, score="sigmoid", n_groups=2, top_groups=2, group_score="top2")
        np.testing.assert_array_equal(back(ex), [[7, 4, 5]])
        ex, _ = ox.route(x.to(DT[dtype]), 3, score="sigmoid")
        np.testing.assert_array_equal(back(ex), [[7, 4, 5]])


def test_types_of_experts():
    """The smaller integers count like int32; unsigned ones whose numbers 32 bits would wrap are refused."""
    ex = torch.tensor([[0, 2], [1, 3], [3, 0]], dtype=torch.int32, device="cuda")
    p = ox.plan(ex, 4)
    for dtype in (torch.int8, torch.uint8, torch.int16, torch.int64):
        for got, ref in zip(ox.plan(ex.to(dtype), 4)[:4], p[:4]):
            np.testing.assert_array_equal(back(got), back(ref))
    for dtype in (torch.uint32, torch.uint64, torch.bool, torch.float32):
        with pytest.raises(ValueError):
            ox.plan(torch.zeros(3, 2, dtype=dtype, device="cuda"), 4)


def test_two_threads_with_numpy_arrays():
    """Host calls share the process's context and wait for each other."""
    import threading
    rng = np.random.default_rng(1)
    xs = [rng.standard_normal((n, 24)) for n in (3000, 500)]
    ref = [ox.route(x, 3) for x in xs]
    wrong = []

    def work(i):
        for _ in range(20):
            ex, w = ox.route(xs[i], 3)
            if not (np.array_equal(ex, ref[i][0]) and np.array_equal(w, ref[i][1])):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


def test_views_that_negate_when_they_are_read():
    z = torch.randn(7, 1, dtype=torch.complex64, device="cuda")
    x = z.conj().imag
    assert x.is_neg()
    p = ox.plan(torch.zeros(7, 1, dtype=torch.int32, device="cuda"), 1)
    np.testing.assert_array_equal(back(ox.dispatch(x, p)), -back(z.imag.contiguous()))


@pytest.mark.parametrize("dtype", ["f64", "f32", "bf16", "f16"])
@pytest.mark.parametrize("opt", [{}, dict(renormalise=False), dict(score="sigmoid"), dict(n_groups=4, top_groups=2, group_score="top2"),
                                 dict(score="sigmoid", n_groups=4, top_groups=3, renormalise=False), dict(n_groups=20, top_groups=5)])
def test_bias_closes_experts_and_what_is_no_number_shows(dtype, opt):
    """-inf in the bias closes its expert for every row; rows for which an expert of bias NaN or +inf is open hold -1 and NaN."""
    rng = np.random.default_rng(17)
    n, e, k = 90, 60, 5
    x, xr = scores_of(rng, n, e, dtype)
    mask = rng.random((n, e)) < 0.9
    mask[:40, [7, 33]] = False
    bias = rng.standard_normal(e) * 0.05
    for odd in ((-np.inf, -np.inf), (np.nan, -np.inf), (-np.inf, np.inf), (np.nan, np.inf)):
        bias[[7, 33]] = odd
        bias[[0, 12, 50, 59]] = -np.inf
        b32 = bias.astype(np.float32)
        for b in (torch.as_tensor(b32, device="cuda"), torch.as_tensor(b32.astype(np.float64), device="cuda")):
            ex, w = ox.route(x, k, bias=b, mask=torch.as_tensor(mask, device="cuda"), **opt)
            er, wr = eo.route(xr, k, bias=b32, mask=mask, **opt)
            np.testing.assert_array_equal(back(ex), er)
            check_weights(back(w), wr, xr, er, dtype, opt)
            assert not np.isin(back(ex), [0, 12, 50, 59]).any() and (back(ex)[:40] >= 0).all()
            assert (back(ex)[40:][mask[40:, 7] & ~np.isneginf(odd[0])] == -1).all()
    bias[:] = -np.inf
    ex, w = ox.route(x, k, bias=torch.as_tensor(bias, device="cuda"), **opt)
    assert (ex == -1).all() and (w == 0).all()


def test_bias_of_numpy_arrays_may_close_experts():
    rng = np.random.default_rng(18)
    x, bias = rng.standard_normal((50, 12)), rng.standard_normal(12) * 0.05
    bias[[0, 5]] = -np.inf
    for kw in (dict(), dict(score="sigmoid", n_groups=3, top_groups=2, group_score="top2"), dict(renormalise=False)):
        ex, w = ox.route(x, 3, bias=bias, **kw)
        er, wr = eo.route(x, 3, bias=bias, **kw)
        np.testing.assert_array_equal(ex, er)
        np.testing.assert_allclose(w, wr, rtol=1e-13, atol=1e-300)
        assert not np.isin(ex, [0, 5]).any()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("c", [65536, 1 << 20, (1 << 20) + 5])
def test_weights_gradient_of_long_flat_rows(c, dtype):
    """A long row of equal terms: one running sum in 32 bits would round the same way at every step.  Of the terms of a 16-byte unit each
    carries a product's and at most 7 additions' roundings, the units are added in 64 bits, the result is rounded once: 9 u, and 2 u for the
    elements left over, at most 7 of them a lane."""
    p = ox.plan(torch.zeros(3, dtype=torch.int32, device="cuda"), 1)
    F = torch.full((3, c), 1.0, device="cuda", dtype=DT[dtype])
    dy = torch.full((3, c), 1.0, device="cuda", dtype=DT[dtype])
    F[1], dy[1] = 0.2998046875, 0.2001953125
    F[2], dy[2] = 1.0078125, 0.7109375
    _, dw = ox.combine_grad(F, torch.ones(3, 1, device="cuda"), p, dy)
    ref = (F.double() * dy.double()).sum(1).cpu().numpy()
    assert (np.abs(back(dw)[:, 0] - ref) <= 11 * 2.0 ** -24 * ref).all(), (back(dw)[:, 0] / ref - 1) * 2.0 ** 24


def test_zeros_without_storage_are_refused():
    """torch's zero tensors, which have no memory (tangents of what does not vary, for one), were taken for an array left out."""
    z = torch._efficientzerotensor((2, 2), device="cuda")
    p = ox.plan(torch.tensor([[0, 1], [1, 2]], dtype=torch.int32, device="cuda"), 3)
    F, dy = torch.ones(4, 3, device="cuda"), torch.ones(2, 3, device="cuda")
    for call in (lambda: ox.combine(F, z, p), lambda: ox.dispatch(z, p), lambda: ox.combine_grad(F, z, p, dy), lambda: ox.route(z, 1),
                 lambda: ox.route(F, 1, bias=torch._efficientzerotensor((3,), device="cuda"))):
        with pytest.raises(ValueError, match="without storage"):
            call()
    assert (ox.combine(F, z.clone(), p) == 0).all()


def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as fwd
    p = ox.plan(torch.tensor([[0, 1], [1, 2]], dtype=torch.int32, device="cuda"), 3)
    F, w = torch.ones(4, 3, device="cuda"), torch.ones(2, 2, device="cuda")
    with fwd.dual_level():
        for call in (lambda: ox.combine(fwd.make_dual(F, F), w, p), lambda: ox.combine(F, fwd.make_dual(w, w), p), lambda: ox.route(fwd.make_dual(w, w), 1)):
            with pytest.raises(ValueError, match="tangent"):
                call()
        assert (ox.combine(F, w, p) == 2).all()


@pytest.mark.parametrize("numpy", [False, True])
def test_weights_of_slots_without_a_place(numpy):
    """Their answer is a row of zeros: a finite weight leaves no trace, a NaN or infinite one shows, and the weight's gradient is 0."""
    rng = np.random.default_rng(12)
    ex = np.array([[0, -1], [-1, -1], [1, -1], [-1, 2], [2, 0], [-1, 1]], dtype=np.int32)
    w = rng.standard_normal(ex.shape)
    w[0, 1], w[1, 1], w[3, 0] = np.inf, np.nan, -np.inf
    F, dy = rng.standard_normal((12, 5)), rng.standard_normal((6, 5))
    put = (lambda a: a) if numpy else (lambda a: torch.as_tensor(a, device="cuda"))
    get = (lambda a: a) if numpy else back
    p = ox.plan(put(ex), 3)
    y = get(ox.combine(put(F), put(w), p))
    np.testing.assert_allclose(y, eo.combine(F, w, get(p.positions)), rtol=1e-13, atol=1e-13)
    assert np.isnan(y[[0, 1, 3]]).all() and np.isfinite(y[[2, 4, 5]]).all()
    dF, dw = map(get, ox.combine_grad(put(F), put(w), p, put(dy)))
    for got, ref in zip((dF, dw), eo.combine_grad(F, w, get(p.positions), dy)):
        np.testing.assert_allclose(got, ref, rtol=1e-13, atol=1e-13)
    assert (dw[ex < 0] == 0).all() and np.isfinite(dF).all()
