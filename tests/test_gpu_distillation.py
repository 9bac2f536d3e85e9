"""Distillation from a teacher's top logits on the device against the float64 oracle (oracle/experts_oracle.py).

Tolerances, u = 2^-24 (2^-53 for float64).  log z carries d = (far / tau + V / 64 + 16) u: the argument's rounding is u of the
distance ``far`` of the logits, the exponential's two, and a sum of V terms by at least 64 threads takes at most V / 64 + 12 roundings.  A
divergence adds d (and a few u of its terms, ``size`` of the oracle) to its value; a gradient entry carries 2 d of both of its parts and
one rounding to its type, half a step.  Teacher probabilities are formed in 64 bits everywhere, so they only count for float64: the rounding
of t / tau - lse, (|t| / tau + |lse|) 2^-53, and as much again in the oracle, which works in the same 64 bits.  The reverse direction
holds log p_rest, p_rest = 1 - sum p: that error and the k roundings of the sum over p_rest.
"""
import numpy as np
import pytest
import torch

from oak import distillation as od
from oracle import experts_oracle as eo

pytestmark = pytest.mark.gpu
DT = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def back(t):
    return t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def problem(n, v, k, dtype, tail, tau=1.0, seed=0, pad=0, index_64=True, spread=2.0):
    rng = np.random.default_rng(seed + v)
    teacher = rng.standard_normal((n, v)) * spread
    s = torch.as_tensor(0.8 * teacher + rng.standard_normal((n, v)), device="cuda").to(DT[dtype])
    store = torch.full((n, v + pad), float("nan"), dtype=DT[dtype], device="cuda")
    off = 1 if pad else 0
    store[:, off:off + v] = s
    s = store[:, off:off + v]
    wide = torch.float64 if dtype == "f64" else torch.float32
    order = np.argsort(-teacher, 1)[:, :k].copy()
    top = torch.as_tensor(np.take_along_axis(teacher, order, 1), device="cuda").to(wide)
    m = teacher.max(1, keepdims=True) / tau
    lse = torch.as_tensor((m + np.log(np.exp(teacher / tau - m).sum(1, keepdims=True)))[:, 0], device="cuda").to(wide) if tail else None
    return s, top, torch.as_tensor(order, dtype=torch.int64 if index_64 else torch.int32, device="cuda"), lse


def compare(s, top, idx, lse, tau, direction, weight, dtype):
    kw = dict(top_lse=lse, temperature=tau, direction=direction, row_weight=weight)
    loss, grad = od.distill_grad(s, top, idx, **kw)
    only = od.distill(s, top, idx, **kw)
    assert torch.equal(torch.nan_to_num(only, nan=7.0), torch.nan_to_num(loss, nan=7.0))
    assert grad.dtype == s.dtype and loss.dtype == (torch.float64 if dtype == "f64" else torch.float32)
    x = back(s)
    n, v = x.shape
    resolution = 2.0 ** -53 if dtype == "f64" else 2.0 ** -24
    ref, gref, size = eo.distill(x, back(top), back(idx), None if lse is None else back(lse), tau, direction,
                                 None if weight is None else back(weight), resolution)
    u = 2.0 ** -53 if dtype == "f64" else 2.0 ** -24
    finite = np.where(np.isfinite(x), x, np.nan)
    far = np.array([np.ptp(r[np.isfinite(r)]) if np.isfinite(r).any() else 0.0 for r in finite])
    far = np.minimum(far, 110.0 * tau)                                   # further down an exponential is 0 in 32 bits
    d = (far / tau + v / 64 + 16) * u
    if dtype == "f64":
        t = np.where((back(idx) >= 0) & np.isfinite(back(top)), np.abs(back(top)), 0.0).max(1)
        t = t / tau + (0.0 if lse is None else np.abs(back(lse)))
        d = d + 2 * t * u
        if direction == "reverse":
            there = (back(idx) >= 0) & np.isfinite(back(top))
            p = np.where(there, np.exp(np.where(there, back(top), 0.0) / tau - back(lse)[:, None]), 0.0)
            d = d + 2 * (t + top.shape[1]) * u / np.maximum(1.0 - p.sum(1), 2.0 ** -53)
    assert np.array_equal(np.isnan(back(loss)), np.isnan(ref)) and np.array_equal(np.isinf(back(loss)), np.isinf(ref))
    ok = np.isfinite(ref)
    err, tol = np.abs(back(loss) - np.where(ok, ref, 0)), (2 * d + 4 * u) * (size + np.abs(np.where(ok, ref, 0)))
    # exact zeros of the oracle's size (rows of weight 0, empty teachers) are zeros here
    assert (err[ok] <= tol[ok]).all(), (err[ok].max(), tol[ok][err[ok].argmax()])
    q = np.exp(x / tau - (x / tau).max(1, keepdims=True))
    q = q / q.sum(1, keepdims=True)
    w = np.ones(n) if weight is None else back(weight)
    half = torch.finfo(DT[dtype]).eps / 2
    gok = np.isfinite(gref)
    part = np.where(gok, np.abs(gref), 0) + tau * np.abs(w)[:, None] * np.nan_to_num(q)
    gtol = 2 * d[:, None] * (part + np.nan_to_num(q) * (size / tau)[:, None]) + half * np.abs(np.where(gok, gref, 0)) + 1e-37
    if dtype == "f16":
        gtol = gtol + 2.0 ** -25                                         # half a step of the smallest float16 numbers
    gerr = np.abs(back(grad) - np.where(gok, gref, 0))
    assert (gerr[gok] <= gtol[gok]).all(), (gerr - gtol)[gok].max()
    return loss, grad, ref, gref


CASES = [
    # n, V, k, dtype, tail, tau, direction, pad, index_64
    (1, 1, 1, "f32", False, 1.0, "forward", 0, True),
    (4, 2, 1, "bf16", True, 1.0, "reverse", 0, False),
    (7, 10, 10, "f32", True, 1.0, "forward", 0, True),                  # the entries are all the classes: no rest
    (7, 10, 10, "f32", True, 1.0, "reverse", 0, True),
    (70, 100, 5, "f64", True, 2.0, "reverse", 3, True),
    (33, 1000, 10, "f32", False, 2.0, "forward", 0, False),
    (20, 1024, 256, "bf16", True, 1.0, "forward", 0, True),
    (6, 1024, 300, "f16", True, 0.7, "forward", 1, True),
    (9, 1025, 3, "bf16", True, 4.0, "forward", 1, True),
    (5, 4099, 64, "f16", False, 1.0, "forward", 0, True),
    (3, 8191, 1024, "f32", True, 1.5, "reverse", 11, False),
    (4, 16384, 20, "bf16", True, 1.0, "forward", 0, True),
    (2, 50021, 33, "f32", True, 1.5, "reverse", 3, True),
    (3, 49157, 20, "f16", True, 1.0, "forward", 0, True),
    (2, 131072, 128, "bf16", True, 1.0, "forward", 0, True),
    (2, 140001, 7, "bf16", False, 1.0, "forward", 0, True),
    (2, 30000, 17, "f64", True, 1.0, "forward", 1, True),
    (1, 1 << 20, 1024, "bf16", True, 1.0, "forward", 0, True),
]


@pytest.mark.parametrize("n,v,k,dtype,tail,tau,direction,pad,index_64", CASES)
def test_distill(n, v, k, dtype, tail, tau, direction, pad, index_64):
    s, top, idx, lse = problem(n, v, k, dtype, tail, tau, 0, pad, index_64)
    w = torch.rand(n, device="cuda", dtype=top.dtype) + 0.5
    compare(s, top, idx, lse, tau, direction, w, dtype)


@pytest.mark.parametrize("v", [50, 3000, 40000])
@pytest.mark.parametrize("direction", ["forward", "reverse"])
def test_ragged_teachers_masked_rows_and_wrong_indices(v, direction):
    s, top, idx, lse = problem(12, v, 9, "bf16", True, seed=3)
    s, top, idx = s.clone(), top.clone(), idx.clone()
    idx[0, 4:] = -1                                                      # padding by index,
    top[1, 2:] = -float("inf")                                           # by value,
    idx[2] = -1                                                          # a teacher that kept nothing
    s[3] = float("nan")                                                  # a row that is left out may hold anything
    idx[3, 0] = v + 5
    idx[4, 3] = v                                                        # no class
    idx[5, 0] = -2
    s[6, :v // 2] = -float("inf")                                        # classes the student rules out ...
    top[6, 0], idx[6, 0] = 1.0, 0                                        # ... one of which the teacher holds
    s[7, 3] = float("nan")
    s[8] = torch.finfo(torch.bfloat16).min                               # all at the type's lowest value: uniform
    w = torch.ones(12, device="cuda")
    w[3] = 0
    loss, grad, _, _ = compare(s, top, idx, lse, 1.0, direction, w, "bf16")
    loss, grad = back(loss), back(grad)
    assert loss[2] == 0 and loss[3] == 0 and (grad[2] == 0).all() and (grad[3] == 0).all()
    assert np.isnan(loss[[4, 5, 7]]).all() and np.isnan(grad[4]).all() and np.isnan(grad[5]).all()
    if direction == "forward":
        assert np.isposinf(loss[6])
    assert np.isfinite(loss[[0, 1, 8, 9, 10, 11]]).all()


@pytest.mark.parametrize("v", [40, 5000])
@pytest.mark.parametrize("direction", ["forward", "reverse"])
def test_entries_of_one_class_are_merged(v, direction):
    s, top, idx, lse = problem(6, v, 12, "f32", True, seed=8)
    idx = idx.clone()
    idx[0, 5] = idx[0, 2]
    idx[1, :] = idx[1, 0]
    idx[2, 11] = idx[2, 0]
    lse = torch.logsumexp(top, 1) + 0.3
    compare(s, top, idx, lse, 1.0, direction, None, "f32")
    if direction == "forward":
        compare(s, top, idx, None, 1.0, direction, None, "f32")


@pytest.mark.parametrize("v", [64, 4096])
def test_a_student_that_is_sure_of_itself_keeps_its_rest(v):
    """The rest's mass far below the rounding of the top's: its logarithm has to come from the rest itself."""
    s = torch.zeros(2, v, device="cuda", dtype=torch.float64)
    s[0, 5], s[1, 5] = 60.0, 300.0
    for dtype in ("f32", "f64", "bf16"):
        top = torch.full((2, 1), 3.0, device="cuda", dtype=torch.float64 if dtype == "f64" else torch.float32)
        idx = torch.full((2, 1), 5, device="cuda")
        lse = torch.full((2,), 3.5, device="cuda", dtype=top.dtype)
        compare(s.to(DT[dtype]), top, idx, lse, 1.0, "forward", None, dtype)


def test_types_of_the_teacher():
    s, top, idx, lse = problem(20, 300, 8, "bf16", True)
    for t in (torch.bfloat16, torch.float16, torch.float64):
        compare(s, top.to(t), idx.to(torch.int32), lse.double(), 1.0, "forward", torch.ones(20, device="cuda", dtype=t), "bf16")
    s32, top, idx, lse = problem(20, 300, 8, "f64", True)
    compare(s32, top.float(), idx, lse.float(), 1.0, "forward", None, "f64")


def test_strides():
    s, top, idx, lse = problem(16, 200, 6, "f32", True)
    wide = torch.zeros(16, 20, device="cuda")
    wide[:, 3:9] = top
    compare(s.t().contiguous().t(), wide[:, 3:9], idx.t().contiguous().t(), lse, 1.0, "forward", None, "f32")
    one = s[:1].expand(5, 200)                                           # one row for all
    loss = od.distill(one, top[:1].expand(5, 6), idx[:1].expand(5, 6), top_lse=lse[:1].expand(5))
    assert torch.equal(loss, od.distill(s[:1], top[:1], idx[:1], top_lse=lse[:1]).expand(5))
    loss, grad = od.distill_grad(s[:0], top[:0], idx[:0])
    assert loss.shape == (0,) and grad.shape == (0, 200)


def test_numpy_arrays_and_differences():
    rng = np.random.default_rng(1)
    n, v, k = 9, 30, 5
    teacher, s = rng.standard_normal((n, v)) * 2, rng.standard_normal((n, v))
    idx = np.argsort(-teacher, 1)[:, :k].copy()
    top, lse = np.take_along_axis(teacher, idx, 1), np.log(np.exp(teacher / 1.3).sum(1))
    idx[2, 3:] = -1
    w = rng.random(n) + 0.2
    for direction, given in (("forward", None), ("forward", lse), ("reverse", lse)):
        kw = dict(top_lse=given, temperature=1.3, direction=direction, row_weight=w)
        loss, grad = od.distill_grad(s, top, idx, **kw)
        ref, gref, _ = eo.distill(s, top, idx, given, 1.3, direction, w)
        np.testing.assert_allclose(loss, ref, rtol=1e-12, atol=1e-13)
        np.testing.assert_allclose(grad, gref, rtol=1e-11, atol=1e-13)
        np.testing.assert_array_equal(od.distill(s, top, idx, **kw), loss)
        np.testing.assert_allclose(grad.sum(1), 0, atol=1e-12)           # a shift of all logits changes nothing
        for i, j in ((0, idx[0, 0]), (2, 7), (5, idx[5, 4]), (8, 29)):
            up, down = s.copy(), s.copy()
            up[i, j] += 1e-5
            down[i, j] -= 1e-5
            fd = (od.distill(up, top, idx, **kw).sum() - od.distill(down, top, idx, **kw).sum()) / 2e-5
            assert abs(fd - grad[i, j]) <= 1e-8


def test_streams_and_captured_graphs():
    s, top, idx, lse = problem(40, 9000, 16, "bf16", True)
    s = s.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = od.distill_grad(s, top, idx, top_lse=lse)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(od.distill_grad(s, top, idx, top_lse=lse), other):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = od.distill_grad(s, top, idx, top_lse=lse)
    for seed in range(4):
        s.copy_(torch.randn(s.shape, generator=torch.Generator().manual_seed(seed)).to("cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(od.distill_grad(s, top, idx, top_lse=lse), held):
            assert torch.equal(a, b)


def test_offsets_beyond_32_bits():
    far = (1 << 30) + 3
    store = torch.zeros(2 * far + 5000, device="cuda", dtype=torch.bfloat16)
    s = store.as_strided((3, 5000), (far, 1))
    small, top, idx, lse = problem(3, 5000, 9, "bf16", True, seed=4)
    s.copy_(small)
    compare(s, top, idx, lse, 1.0, "forward", None, "bf16")


@pytest.mark.parametrize("n,v", [((1 << 28) + 70, 2), ((1 << 22) + 3, 9000)])
def test_more_rows_than_one_launch_takes(n, v):
    """Beyond 2^22 workgroups a workgroup walks on to further rows; the rows are one row n times over (row stride 0)."""
    s, top, idx, lse = problem(1, v, 1, "f16", True)
    one = od.distill(s, top, idx, top_lse=lse)
    loss = od.distill(s.expand(n, v), top.expand(n, 1), idx.expand(n, 1), top_lse=lse.expand(n))
    assert bool((loss == one).all())


def test_rows_differ_from_launch_to_launch_row():
    """A workgroup's second row must not see the first one's entries: rows with entries in different places, few workgroups' worth each."""
    for n, v, k in ((3000, 40, 3), (700, 600, 20), (300, 9000, 40)):
        s, top, idx, lse = problem(n, v, k, "f32", True, seed=n)
        compare(s, top, idx, lse, 1.0, "forward", None, "f32")


def test_refusals_on_the_device():
    s, top, idx, lse = problem(4, 30, 3, "f32", True)
    cases = [
        lambda: od.distill(s.clone().requires_grad_(), top, idx), lambda: od.distill(s, top.cpu(), idx), lambda: od.distill(s, back(top), idx),
        lambda: od.distill(s, top, idx.float()), lambda: od.distill(s, top, idx[:, :2]), lambda: od.distill(s, top[:3], idx[:3]),
        lambda: od.distill(s, top, idx, top_lse=lse[:3]), lambda: od.distill(s, top, idx, direction="reverse"),
        lambda: od.distill(s, top, idx, temperature=0.0), lambda: od.distill(s, top, idx, row_weight=lse[:, None]),
        lambda: od.distill(s.to(torch.int32), top, idx), lambda: od.distill(s[0], top, idx),
        lambda: od.distill(torch.zeros(1, (1 << 20) + 1, device="cuda"), top[:1], idx[:1]),
    ]
    for i, call in enumerate(cases):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"case {i} was not refused")


@pytest.mark.parametrize("n,v,k,dtype,tail,direction,pad", [
    (1, 131072, 128, "bf16", True, "forward", 0), (2, 131075, 64, "bf16", True, "reverse", 5), (3, 70001, 1, "f16", False, "forward", 1),
    (128, 66003, 20, "bf16", True, "forward", 0), (129, 66003, 20, "bf16", True, "forward", 0), (17, 32773, 300, "f32", True, "forward", 3),
    (5, 16384, 7, "f64", True, "reverse", 0), (5, 16383, 7, "f64", False, "forward", 1), (8, 65535, 9, "bf16", True, "forward", 0), (1, 262147, 3, "f32", True, "forward", 0),
])
def test_few_rows_cut_into_slices(n, v, k, dtype, tail, direction, pad):
    """Sizes around the rule that cuts a row into slices, entries on both sides of the cuts."""
    s, top, idx, lse = problem(n, v, k, dtype, tail, 1.0, 1, pad)
    idx = idx.clone()
    if v > 40000 and k > 3:
        idx[0, :4] = torch.tensor([0, v - 1, v // 2, v // 2 - 1], device="cuda")   # ends, and the middle cut of an even number of slices
    w = torch.rand(n, device="cuda", dtype=top.dtype) + 0.5
    if n > 2:
        w[1] = 0
        s[1] = float("nan")
    compare(s, top, idx, lse, 1.0, direction, w, dtype)


def test_slices_merge_entries_of_one_class():
    s, top, idx, lse = problem(3, 90000, 12, "bf16", True, seed=8)
    idx = idx.clone()
    idx[0, 5] = idx[0, 2]
    idx[1, :] = idx[1, 0]
    idx[2, 3] = 90000
    lse = torch.logsumexp(top, 1) + 0.3
    for direction in ("forward", "reverse"):
        compare(s, top, idx, lse, 1.0, direction, None, "bf16")


def test_two_graphs_of_split_rows_do_not_share_scratch():
    a, b = problem(2, 100000, 9, "bf16", True, seed=1), problem(4, 90000, 9, "bf16", True, seed=2)
    ref = [od.distill_grad(p[0], p[1], p[2], top_lse=p[3]) for p in (a, b)]
    graphs, held = [], []
    for p in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(od.distill_grad(p[0], p[1], p[2], top_lse=p[3]))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for h, r in zip(held, ref):
            assert torch.equal(h[0], r[0]) and torch.equal(h[1], r[1])


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32", "f64"])
@pytest.mark.parametrize("direction", ["forward", "reverse"])
def test_every_small_number_of_classes(dtype, direction):
    """1 .. 70 classes: every count of elements left over behind the 16-byte units, many rows, some of them left out."""
    for v in range(1, 71):
        k = 1 + v % min(v, 17)
        s, top, idx, lse = problem(300, v, k, dtype, True, 1.0, v, pad=v % 3)
        w = torch.rand(300, device="cuda", dtype=top.dtype) + 0.5
        w[::7] = 0
        compare(s, top, idx, lse, 1.0, direction, w, dtype)


@pytest.mark.parametrize("units", [16, 64, 128, 256, 512, 1024, 2048, 4096])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_around_the_sizes_where_the_team_changes(units, dtype):
    per = 8 if dtype == "bf16" else 4
    for v in (units * per - 1, units * per, units * per + 1, units * per + per - 1):
        for k, n in ((9, 270), (33, 260)):
            s, top, idx, lse = problem(n, v, min(k, v), dtype, True, 1.0, v + k)
            compare(s, top, idx, lse, 1.0, "forward", None, dtype)


@pytest.mark.parametrize("k,shift", [(11, 0.4), (11, -0.7), (4, -0.7), (4, 0.4)])
def test_gradient_where_the_kept_mass_is_not_what_top_lse_leaves(k, shift):
    """A rounded top_lse (or one entry that is kept twice): the entries' mass passes 1, or they are all the classes and stay below it.  The
    loss as it stands is differentiated: against differences, and a shift of all logits changes nothing."""
    rng = np.random.default_rng(21)
    n, v, tau = 5, 11, 1.3
    s, top = rng.standard_normal((n, v)), rng.standard_normal((n, k)) * 2
    idx = np.argsort(rng.random((n, v)), 1)[:, :k].copy()
    lse = np.log(np.exp(top / tau).sum(1)) + shift                       # the entries' mass is exp(-shift)
    kw = dict(top_lse=lse, temperature=tau)
    loss, grad = od.distill_grad(s, top, idx, **kw)
    ref, gref, _ = eo.distill(s, top, idx, lse, tau)
    np.testing.assert_allclose(loss, ref, rtol=1e-12, atol=1e-13)
    np.testing.assert_allclose(grad, gref, rtol=1e-11, atol=1e-13)
    np.testing.assert_allclose(grad.sum(1), 0, atol=1e-12)
    for i, j in ((0, idx[0, 0]), (2, 7), (3, idx[3, 2]), (4, 10)):
        up, down = s.copy(), s.copy()
        up[i, j] += 1e-5
        down[i, j] -= 1e-5
        fd = (od.distill(up, top, idx, **kw).sum() - od.distill(down, top, idx, **kw).sum()) / 2e-5
        assert abs(fd - grad[i, j]) <= 1e-8


@pytest.mark.parametrize("v", [40, 5000, 140001])
@pytest.mark.parametrize("dtype", ["bf16", "f32", "f64"])
def test_top_lse_of_16_bits(v, dtype):
    s, top, idx, lse = problem(6, v, 9, dtype, True, spread=6.0, seed=2)  # nearly all of the teacher's mass is kept
    for low in (lse.to(torch.bfloat16), (lse - 0.02).to(torch.float16)):
        compare(s, top, idx, low, 1.0, "forward", None, dtype)


@pytest.mark.parametrize("v", [70, 5000, 70001])
def test_lowest_values_are_entries_of_no_mass_and_not_padding(v):
    """-inf is padding, the type's lowest value is not, whatever the temperature makes of it: its class stays out of the rest."""
    s, top, idx, lse = problem(3, v, 6, "f64", True, 0.5)
    low, far = top.clone(), top.clone()
    for t, value in ((low, torch.finfo(torch.float64).min), (far, -1e5)):
        t[0, 3:] = value
        t[1] = value
    for given in (lse, None):
        for a, b in zip(od.distill_grad(s, low, idx, top_lse=given, temperature=0.5), od.distill_grad(s, far, idx, top_lse=given, temperature=0.5)):
            assert torch.equal(a, b)
        assert torch.equal(od.distill(s, low, idx, top_lse=given, temperature=0.5), od.distill(s, far, idx, top_lse=given, temperature=0.5))
    ref, gref, _ = eo.distill(back(s), back(far), back(idx), back(lse), 0.5)
    loss, grad = od.distill_grad(s, low, idx, top_lse=lse, temperature=0.5)
    np.testing.assert_allclose(back(loss), ref, rtol=1e-11)
    np.testing.assert_allclose(back(grad), gref, rtol=1e-10, atol=1e-14)


@pytest.mark.parametrize("n,v", [(300, 4096), (300, 32768), (300, 131072), (2, 131072), (128, 1 << 20), (130, 1 << 20)])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("t", [-1.25, -0.3125])
def test_flat_rows_keep_the_digits_of_their_sum(n, v, dtype, t):
    """Every 16-byte unit holds one 0 and otherwise t, so that a running sum in 32 bits would round alike at every step of every lane (at 2^20
    classes by 179 u and more of the sum).  One sure class against the rest's sum S: L = log(1 + S e^-x).  A term carries |t| u of
    its argument and 2 u of the exponential, a unit's sum at most as many additions as it has terms; everything else is 64 bits, the result one u."""
    vn = 4 if dtype == "f32" else 8
    row = torch.full((v,), t, dtype=torch.float64)
    row[::vn] = 0.0
    rest = float(row.exp().sum()) - 1.0                                  # without class 0, the teacher's
    x = float(round(np.log(rest)))
    row[0] = x
    s = row.to("cuda").to(DT[dtype]).expand(n, v).contiguous()
    ref = np.log1p(rest * np.exp(-x))
    share = rest * np.exp(-x - ref)
    top, idx = torch.zeros(n, 1, device="cuda"), torch.zeros(n, 1, dtype=torch.int64, device="cuda")
    u = 2.0 ** -24
    tol = share * (abs(t) + 2 + vn) * u + u * ref
    loss = back(od.distill(s, top, idx))
    assert (np.abs(loss - ref) <= tol).all(), (np.abs(loss - ref).max() / u, tol / u)


@pytest.mark.parametrize("teams,n,v,k,dtype,grad", [
    (1 << 27, (1 << 27) + 100, 2, 1, "f16", True), (1 << 28, (1 << 28) + 100, 20, 2, "f64", False), (1 << 26, (1 << 26) + 100, 136, 2, "bf16", True),
    (1 << 24, (1 << 24) + 100, 2100, 40, "bf16", False), (1 << 22, (1 << 22) + 100, 8200, 3, "bf16", True),
    (1 << 22, (1 << 22) + 100, 33000, 70, "f16", False)])
def test_a_teams_next_row_sees_nothing_of_its_last(teams, n, v, k, dtype, grad):
    """A launch has teams for ``teams`` rows; the rows behind them are their second ones, whose teachers kept other classes (the student's row is
    one row n times over).  A few rows in one launch are the reference, to the bit."""
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 2 * n * v * (2 if grad else 0) + (24 << 30):
        pytest.skip("not enough free device memory")
    rng = np.random.default_rng(v)
    s = torch.as_tensor(rng.standard_normal((1, v)), device="cuda").to(DT[dtype])
    top = torch.as_tensor(rng.standard_normal((1, k)), device="cuda", dtype=torch.float64 if dtype == "f64" else torch.float32)
    lse = torch.logsumexp(top, 1) + 0.7
    place = torch.arange(k, device="cuda", dtype=torch.int32) * max(1, v // (2 * k))

    def run(rows, call):
        r = torch.arange(rows, device="cuda", dtype=torch.int32)
        first = (r + r // teams) % v                                     # classes of a team's second row: one further
        out = call(s.expand(rows, v), top.expand(rows, k), (first[:, None] + place) % v, top_lse=lse.expand(rows))
        return first, out

    few = max(v, 257)                                                    # up to 256 rows another rule holds
    _, (ref, gref) = run(few, od.distill_grad)
    assert len(ref[:v].unique()) > 1
    first, out = run(n, od.distill_grad if grad else od.distill)
    loss = out[0] if grad else out
    for a in range(0, n, 1 << 24):
        assert torch.equal(loss[a:a + (1 << 24)], ref[first[a:a + (1 << 24)].long()]), a
    if grad:
        assert torch.equal(out[1][teams - 50:], gref[first[teams - 50:].long()])
    del out, loss, gref, first
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", ["f64", "f32"])
def test_kept_mass_within_single_precision_of_1_is_1(dtype):
    """All classes kept, top_lse rounded to float32: the gradient is q - p."""
    s, top, idx, _ = problem(200, 20, 20, dtype, False)
    low = torch.logsumexp(top.double(), 1).float()
    loss, grad, _, _ = compare(s, top, idx, low.to(top.dtype), 1.0, "forward", None, dtype)
    p = torch.exp(top.double() - low.double()[:, None])
    want = torch.softmax(s.double(), 1).scatter_add_(1, idx, -p)
    # beside the softmax's own error (see above; distances below 16 here) one rounding of the result
    u = 2.0 ** -53 if dtype == "f64" else 2.0 ** -24
    assert ((grad.double() - want).abs() <= 2 * (16 + 16) * u * (want.abs() + torch.softmax(s.double(), 1)) + (64 * u if dtype == "f64" else 0)).all()
