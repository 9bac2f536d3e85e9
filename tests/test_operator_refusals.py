"""What the mixture and distillation operators refuse, before anything reaches a device (runs without one)."""
import ctypes

import numpy as np
import pytest

from oak import _capi, distillation, experts

FAKE = ctypes.create_string_buffer(64)          # an address that is never read: every call below is refused first


def refused(name, args, match):
    with pytest.raises(ValueError, match=match):
        _capi.call_device(name, None, 0, args)


def route_args(**kw):
    base = dict(n_rows=2, ld_scores=4, n_experts=4, top_k=2, n_groups=1, top_groups=1, dtype=1, scale=1.0, ld_dscores=4)
    a = _capi.RouteArgs(**{**base, **kw})
    for f in ("scores", "experts", "weights", "dweights", "dscores"):
        if f not in kw:
            setattr(a, f, ctypes.addressof(FAKE))
    return a


@pytest.mark.parametrize("kw,match", [
    (dict(n_experts=0), "n_experts"), (dict(n_experts=1025), "n_experts"), (dict(top_k=0), "top_k"), (dict(top_k=5), "top_k"),
    (dict(n_groups=3), "n_groups"), (dict(n_groups=0), "n_groups"), (dict(n_groups=2, top_groups=3), "top_groups"),
    (dict(n_groups=4, top_groups=1, top_k=2), "top_k"), (dict(dtype=9), "type"), (dict(score=2), "score"), (dict(group_score=-1), "group score"),
    (dict(scale=float("inf")), "scale"), (dict(n_rows=-1), "n_rows"), (dict(n_rows=1 << 31), "slots"), (dict(n_rows=1 << 62, top_k=4), "slots"), (dict(scores=None), "NULL"),
    (dict(weights=None), "NULL"), (dict(ld_scores=-4), "stride"),
])
def test_route_refuses(kw, match):
    refused("route", route_args(**kw), match)


def test_route_grad_refuses():
    refused("route_grad", route_args(dscores=None), "NULL")
    refused("route_grad", route_args(ld_dscores=3), "overlap")


def plan_args(**kw):
    a = _capi.PlanArgs(**{**dict(n_rows=2, top_k=2, n_experts=4), **kw})
    for f in ("experts", "rows", "positions", "counts", "offsets"):
        if f not in kw:
            setattr(a, f, ctypes.addressof(FAKE))
    return a


@pytest.mark.parametrize("kw,match", [
    (dict(n_experts=0), "n_experts"), (dict(n_experts=4097), "n_experts"), (dict(top_k=0), "experts"), (dict(top_k=65), "experts"),
    (dict(n_rows=1 << 30), "slots"), (dict(n_rows=1 << 62, top_k=4), "slots"), (dict(rows=None), "NULL"), (dict(n_rows=1 << 20), "workspace"),
])
def test_plan_refuses(kw, match):
    refused("plan", plan_args(**kw), match)


def mix_args(**kw):
    a = _capi.MixArgs(**{**dict(n_rows=2, top_k=2, n_experts=4, n_cols=3, ld_rows=3, ld_slots=3, ld_grad=3, dtype=1), **kw})
    for f in ("positions", "offsets", "weights", "src", "dst", "dout", "dslots", "dweights"):
        if f not in kw:
            setattr(a, f, ctypes.addressof(FAKE))
    return a


@pytest.mark.parametrize("name,kw,match", [
    ("dispatch", dict(n_cols=0), "n_cols"), ("dispatch", dict(dtype=4), "type"), ("dispatch", dict(ld_slots=2), "overlap"),
    ("combine", dict(ld_rows=2), "overlap"), ("combine", dict(dst=None), "NULL"), ("combine", dict(positions=None), "NULL"),
    ("combine", dict(ld_slots=-3), "stride"), ("combine_grad", dict(weights=None), "NULL"), ("combine_grad", dict(dout=None), "NULL"),
])
def test_mixture_refuses(name, kw, match):
    refused(name, mix_args(**kw), match)


def distill_args(**kw):
    a = _capi.DistillArgs(**{**dict(n_rows=2, n_classes=8, top_k=2, dtype=1, top_dtype=1, temperature=1.0, ld_logits=8, ld_top=2, ld_index=2,
                                    ld_dlogits=8), **kw})
    for f in ("logits", "top", "index", "loss", "dlogits"):
        if f not in kw:
            setattr(a, f, ctypes.addressof(FAKE))
    return a


@pytest.mark.parametrize("kw,match", [
    (dict(n_classes=0), "n_classes"), (dict(n_classes=(1 << 20) + 1), "n_classes"), (dict(top_k=0), "top_k"), (dict(top_k=1025), "top_k"),
    (dict(temperature=0.0), "temperature"), (dict(temperature=float("nan")), "temperature"), (dict(temperature=1e9), "temperature"),
    (dict(direction=1), "top_lse"), (dict(direction=2), "direction"), (dict(top_dtype=7), "type"), (dict(loss=None), "NULL"),
    (dict(ld_dlogits=7), "overlap"), (dict(n_rows=1 << 31), "n_rows"),
])
def test_distill_refuses(kw, match):
    refused("distill", distill_args(**kw), match)


def test_null_arguments_and_contexts():
    lib = _capi.load_library()
    for name in ("route", "route_grad", "plan", "dispatch", "combine", "combine_grad", "distill"):
        assert getattr(lib, f"oak_{name}")(None, None) == _capi.OAK_E_ARG
        assert getattr(lib, f"oak_{name}_device")(None, None, None) == _capi.OAK_E_ARG
    with pytest.raises(ValueError):
        _capi.check_device_pointer(None, ctypes.addressof(FAKE))
    assert _capi.plan_workspace(None, 1 << 20, 2, 24) == 0 and _capi.distill_workspace(None, 1, 1 << 17, 2) == 0
    for name, args in (("route", route_args()), ("plan", plan_args()), ("combine", mix_args()), ("distill", distill_args())):
        refused(name, args, "ctx is NULL")


def test_python_layer_refuses():
    x = np.zeros((4, 6))
    for bad in (dict(score="argmax"), dict(group_score="mean"), dict(mask=np.ones((3, 6), bool)), dict(bias=np.zeros(5)), dict(bias=np.full(6, np.inf))):
        with pytest.raises(ValueError):
            experts.route(x, 2, **bad)
    with pytest.raises(ValueError):
        experts.route(np.zeros(6), 2)
    with pytest.raises(ValueError):
        experts.route_grad(x, np.zeros((3, 2), int), np.zeros((4, 2)))
    with pytest.raises(ValueError):
        experts.route_grad(x, np.full((4, 2), 6), np.zeros((4, 2)))
    with pytest.raises(ValueError):
        experts.plan(np.array([[0, 9]]), 4)
    with pytest.raises(ValueError):
        experts.plan(np.array([[0.5, 1.0]]), 4)
    with pytest.raises(ValueError):
        experts.plan(np.zeros((2, 2, 2), int), 4)
    p = experts.Plan(np.zeros(4, np.int32), np.zeros((2, 2), np.int32), np.zeros(3, np.int32), np.zeros(4, np.int32), 2, 2, 3)
    with pytest.raises(ValueError):
        experts.dispatch(np.zeros((3, 5)), p)
    with pytest.raises(ValueError):
        experts.combine(np.zeros((4, 5)), None, p)
    with pytest.raises(ValueError):
        experts.combine(np.zeros((4, 5)), np.zeros((2, 3)), p)
    with pytest.raises(ValueError):
        experts.combine_grad(np.zeros((4, 5)), np.zeros((2, 2)), p, np.zeros((2, 4)))
    with pytest.raises(ValueError):
        experts.dispatch(np.zeros((2, 5)), ("not", "a", "plan"))
    top, idx = np.zeros((4, 2)), np.zeros((4, 2), int)
    for bad in (dict(direction="sideways"), dict(top_lse=np.zeros(3)), dict(row_weight=np.zeros((4, 1)))):
        with pytest.raises(ValueError):
            distillation.distill(x, top, idx, **bad)
    for t, i in ((top[:3], idx[:3]), (top, idx[:, :1]), (top, idx + 6), (top, idx - 2), (top, idx * 0.5)):
        with pytest.raises(ValueError):
            distillation.distill(x, t, i)


def test_a_library_without_a_device_says_so():
    if _capi.device_count() > 0:
        pytest.skip("a HIP device is present")
    with pytest.raises(_capi.OakHipError):
        experts.route(np.zeros((4, 6)), 2)
    with pytest.raises(_capi.OakHipError):
        distillation.distill(np.zeros((4, 6)), np.zeros((4, 2)), np.zeros((4, 2), int))


@pytest.mark.parametrize("torch_first", [True, False])
def test_a_second_copy_of_the_hip_runtime_is_noticed(torch_first):
    """torch brings its own HIP runtime: loaded first it serves the library too, loaded second there are two (nothing here touches a device)."""
    import subprocess
    import sys
    lines = ["import torch", "from oak import _capi; _capi.load_library()"]
    code = "; ".join((lines if torch_first else lines[::-1]) + ["from oak import _capi; print(len(_capi.hip_runtimes()))"])
    out = subprocess.run([sys.executable, "-c", f"import sys; sys.path.insert(0, {str(_capi._PKG_ROOT)!r}); {code}"], capture_output=True, text=True)
    assert out.returncode == 0, out.stderr
    assert int(out.stdout) == (1 if torch_first else 2)


def call_on_host_tensors():
    """The checks a device call makes of every tensor, here on tensors of the host (which are on "device" -1)."""
    import torch
    from oak import _arrays
    t = torch.zeros(1)
    old, _arrays._contexts[-1] = _arrays._contexts.get(-1), type("Context", (), {"_h": 1})()
    d = _arrays.Device(t)
    if old is None:
        del _arrays._contexts[-1]
    return torch, d


def test_zeros_without_storage_are_no_array_left_out():
    torch, d = call_on_host_tensors()
    from oak import _arrays
    z = torch._efficientzerotensor((3, 2))
    for a in (d.tensor(z, "a"), d.matrix(z, "a"), d.dense(z, "a", (3, 2))):
        assert a.data_ptr() == 0
        with pytest.raises(ValueError, match="without storage"):
            _arrays.ptr(a)
    for a in (d.dense(z, "a", (3, 2), torch.float64), d.matrix(z.t(), "a")):           # the copy is an array of zeros
        assert _arrays.ptr(a) is not None and (a == 0).all()
    assert _arrays.ptr(d.matrix(z.clone(), "a")) is not None and _arrays.ptr(d.matrix(torch.zeros(0, 2), "a")) is None


def test_forward_mode_tangents_are_refused():
    import torch
    import torch.autograd.forward_ad as fwd
    x = torch.ones(3, 2)
    with fwd.dual_level():
        _, d = call_on_host_tensors()
        for make in (lambda t: fwd.make_dual(t, torch.ones_like(t)), lambda t: fwd.make_dual(t, torch.ones_like(t)).t()):
            for call in (lambda t: d.tensor(t, "weights"), lambda t: d.matrix(t, "weights"), lambda t: d.dense(t, "weights", tuple(t.shape))):
                with pytest.raises(ValueError, match="weights carries a forward-mode tangent"):
                    call(make(x))
        with torch.no_grad():
            with pytest.raises(ValueError, match="tangent"):
                d.tensor(fwd.make_dual(x, x), "weights")
        assert d.tensor(x, "weights") is x                   # within a level, without a tangent
        assert d.tensor(fwd.unpack_dual(fwd.make_dual(x, x)).primal, "weights").shape == x.shape
    _, d = call_on_host_tensors()
    assert d.tensor(x, "weights") is x


@pytest.mark.parametrize("name", ["route", "route_grad"])
def test_route_refuses_masks_that_run_backwards(name):
    """Rows of a mask at a negative stride would be read from before its start, as those of scores would."""
    refused(name, route_args(mask=ctypes.addressof(FAKE), ld_mask=-4), "stride")
    for kw in (dict(mask=ctypes.addressof(FAKE), ld_mask=-4, n_rows=1), dict(mask=None, ld_mask=-4)):        # not used
        refused(name, route_args(**kw), "ctx is NULL")
