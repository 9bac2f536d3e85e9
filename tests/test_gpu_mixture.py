"""Routing, experts, combination and distillation run together, as a mixture of additive models taught by a classifier would run them."""
import numpy as np
import pytest
import torch

from oak import _capi, distillation, experts

pytestmark = pytest.mark.gpu


def teacher_entries(rng, n, v, k, tau):
    logits = rng.standard_normal((n, v)) * 2.0
    index = np.argsort(-logits, 1)[:, :k].copy()
    return np.take_along_axis(logits, index, 1), index, np.log(np.exp(logits / tau).sum(1))


@pytest.mark.parametrize("score,renormalise", [("softmax", True), ("softmax", False), ("sigmoid", True)])
def test_mixture_of_additive_models(hip, score, renormalise):
    """Rows go to the additive models of their nearest k-means centres; logits = OAK Gram features times each model's weights.
    Gradients of the distillation loss with respect to weights and router against central differences (float64)."""
    rng = np.random.default_rng(4)
    n, d, n_experts, v, m, k = 60, 3, 4, 6, 8, 2
    X = rng.standard_normal((n, d))
    centres, labels, _, _ = hip.kmeans(X, X[:n_experts])
    Z = X[:m]
    desc = [_capi.KernelDesc({"dims": [{"type": "rbf", "lengthscale": 0.7 + 0.2 * e, "variance": 1.0, "measure": ("gaussian", 0.0, 1.0)}] * d,
                              "order_variances": [0.5, 1.0, 0.3], "max_interaction_depth": 2, "share_var_across_orders": True})
            for e in range(n_experts)]
    A = rng.standard_normal((n_experts, m, v))
    scores = -((X[:, None, :] - centres[None]) ** 2).sum(2)
    top, index, lse = teacher_entries(rng, n, v, 3, 1.5)     # top_lse is at the temperature of the call
    by_label = experts.plan(labels, n_experts)                           # hard assignment: the same layout, one expert a row
    assert (labels[by_label.rows] == np.repeat(np.arange(n_experts), by_label.counts)).all()

    def forward(s, weights_of):
        chosen, w = experts.route(s, k, score=score, renormalise=renormalise)
        p = experts.plan(chosen, n_experts)
        rows = experts.dispatch(X, p)
        answers, features = np.zeros((n * k, v)), np.zeros((n * k, m))
        for e in range(n_experts):
            mine = slice(p.offsets[e], p.offsets[e + 1])
            if p.counts[e]:
                features[mine] = hip.gram(desc[e], rows[mine], Z)
                answers[mine] = features[mine] @ weights_of[e]
        logits = experts.combine(answers, w, p)
        return chosen, w, p, features, answers, logits

    chosen, w, p, features, answers, logits = forward(scores, A)
    loss, dlogits = distillation.distill_grad(logits, top, index, top_lse=lse, temperature=1.5)
    danswers, dw = experts.combine_grad(answers, w, p, dlogits)
    dscores = experts.route_grad(scores, chosen, dw, score=score, renormalise=renormalise)
    dA = np.stack([features[p.offsets[e]:p.offsets[e + 1]].T @ danswers[p.offsets[e]:p.offsets[e + 1]] for e in range(n_experts)])
    # a logit's gradient sums to 0 over the classes, and so does everything linear in it
    np.testing.assert_allclose(dlogits.sum(1), 0, atol=1e-12)

    def value(s, weights_of):
        return distillation.distill(forward(s, weights_of)[-1], top, index, top_lse=lse, temperature=1.5).sum()

    h = 1e-5
    for e, i, j in ((0, 0, 0), (1, 3, 2), (3, 7, 5)):
        up, down = A.copy(), A.copy()
        up[e, i, j] += h
        down[e, i, j] -= h
        assert abs((value(scores, up) - value(scores, down)) / (2 * h) - dA[e, i, j]) <= 1e-6 * (1 + abs(dA[e, i, j]))
    for i, j in ((0, 0), (7, 1), (21, 0), (40, 1)):
        up, down = scores.copy(), scores.copy()
        up[i, chosen[i, j]] += h
        down[i, chosen[i, j]] -= h
        got = dscores[i, chosen[i, j]]
        assert abs((value(up, A) - value(down, A)) / (2 * h) - got) <= 1e-6 * (1 + abs(got))


def test_training_step_on_the_device_against_autograd():
    """The same chain on tensors in place: every gradient against float64 autograd of the formulas on the CPU."""
    g = torch.Generator().manual_seed(0)
    n, e, k, c, v = 300, 6, 2, 16, 50
    x = torch.randn(n, c, generator=g)
    gate, heads = torch.randn(c, e, generator=g) * 0.5, torch.randn(e, c, v, generator=g) * 0.5
    t = torch.randn(n, v, generator=g) * 2
    top, index = t.topk(5, 1)
    lse = torch.logsumexp(t, 1)
    bias = torch.linspace(-0.05, 0.05, e)
    dev = [a.cuda() for a in (x, gate, heads, top, index, lse, bias)]
    xd, gated, headsd, topd, indexd, lsed, biasd = dev
    scores = xd @ gated
    chosen, w = experts.route(scores, k, bias=biasd)
    p = experts.plan(chosen, e)
    rows = experts.dispatch(xd, p)
    off = p.offsets.tolist()
    answers = torch.cat([rows[off[i]:off[i + 1]] @ headsd[i] for i in range(e)])
    logits = experts.combine(answers, w, p)
    loss, dlogits = distillation.distill_grad(logits, topd, indexd, top_lse=lsed)
    danswers, dw = experts.combine_grad(answers, w, p, dlogits)
    dscores = experts.route_grad(scores, chosen, dw)
    dheads = torch.stack([rows[off[i]:off[i + 1]].T @ danswers[off[i]:off[i + 1]] for i in range(e)])
    drows = torch.cat([danswers[off[i]:off[i + 1]] @ headsd[i].T for i in range(e)])
    dx = experts.dispatch_grad(drows, p) + dscores @ gated.T

    X, G, H = (a.double().requires_grad_() for a in (x, gate, heads))
    S = X @ G
    picked = chosen.long().cpu()
    W = torch.softmax(S, 1).gather(1, picked)
    W = W / W.sum(1, keepdim=True)
    L = sum(W[:, j, None] * torch.bmm(X[:, None, :], H[picked[:, j]])[:, 0] for j in range(k))
    lq = torch.log_softmax(L, 1)
    lp = top.double() - lse.double()[:, None]
    pr = 1 - lp.exp().sum(1)
    qr = 1 - lq.gather(1, index).exp().sum(1)
    ref = (lp.exp() * (lp - lq.gather(1, index))).sum(1) + pr * (pr.log() - qr.log())
    ref.sum().backward()
    # products of float32 sums of at most 300 terms: 300 * 2^-24 of the terms, a few times over
    for got, want in ((loss, ref), (dheads, H.grad), (dx, X.grad), (xd.T @ dscores, G.grad)):
        want = want.detach()
        assert (got.double().cpu() - want).abs().max() <= 1e-4 * want.abs().max()
