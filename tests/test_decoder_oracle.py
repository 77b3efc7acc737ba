"""The fp64 oracle of residual_norm, token_logprobs and distill_topk: its written-out gradients against
autograd of its forward formulas and against central differences, and its conventions on small rows.
Central differences of step h in fp64 carry an error of about h^2 (third derivatives are of order one
here) + 1e-16 / h: 1e-6 with room at h = 1e-4."""
import math

import pytest
import torch

from oracle import decoder_ops as D

F64 = torch.float64


def _differences(f, x, h=1e-4):
    grad = torch.zeros_like(x)
    flat, out = x.view(-1), grad.view(-1)
    for i in range(flat.numel()):
        keep = float(flat[i])
        flat[i] = keep + h
        up = float(f(x))
        flat[i] = keep - h
        down = float(f(x))
        flat[i] = keep
        out[i] = (up - down) / (2 * h)
    return grad


@pytest.mark.parametrize("post,gated", [(True, True), (True, False), (False, True), (False, False)])
def test_residual_norm_gradient(post, gated):
    torch.manual_seed(3)
    rows, cols, scale = 3, 7, 0.8
    leaves = {"block": torch.randn(rows, cols, dtype=F64), "residual": torch.randn(rows, cols, dtype=F64),
              "post": torch.rand(cols, dtype=F64) + 0.5, "gate": torch.rand(cols, dtype=F64) + 0.2,
              "pre": torch.rand(cols, dtype=F64) + 0.5}
    dout, dy = torch.randn(rows, cols, dtype=F64), torch.randn(rows, cols, dtype=F64)

    def loss(t):
        out, y, _, _ = D.residual_norm_forward(t["block"], t["residual"], t["post"] if post else None,
                                               t["gate"] if gated else None, t["pre"], scale)
        return (out * dout).sum() + (y * dy).sum()

    tracked = {k: v.clone().requires_grad_() for k, v in leaves.items()}
    loss(tracked).backward()
    out, _, r1, r2 = D.residual_norm_forward(leaves["block"], leaves["residual"], leaves["post"] if post else None,
                                             leaves["gate"] if gated else None, leaves["pre"], scale)
    (db, dr, dpost, dgate, dpre), mags = D.residual_norm_backward(
        dy, dout, leaves["block"], out, leaves["post"] if post else None, leaves["gate"] if gated else None,
        leaves["pre"], r1, r2, scale)
    got = {"block": db, "residual": dr, "post": dpost, "gate": dgate, "pre": dpre}
    for name, g in got.items():
        if g is None:
            assert tracked[name].grad is None
            continue
        torch.testing.assert_close(g, tracked[name].grad, rtol=1e-10, atol=1e-12)
        diff = _differences(lambda v, n=name: loss({**leaves, n: v}), leaves[name].clone())
        torch.testing.assert_close(g, diff, rtol=1e-6, atol=1e-6)
    for g, mag in zip((db, dr, dpre), (mags[0], mags[1], mags[4])):
        assert bool((g.abs() <= mag * (1 + 1e-12)).all())


@pytest.mark.parametrize("temperature", [0.7, 1.0, 2.0])
def test_token_logprobs_gradient(temperature):
    torch.manual_seed(4)
    rows, cols = 4, 9
    x = torch.randn(rows, cols, dtype=F64) * 2
    x[1, 3] = -math.inf
    targets = torch.tensor([0, 8, -1, 4])
    g, gh = torch.randn(rows, dtype=F64), torch.randn(rows, dtype=F64)

    def loss(v):
        logprob, _, entropy, _, _ = D.token_logprobs_forward(v, targets, temperature)
        return (logprob * g).sum() + (entropy * gh).sum()

    _, stats, entropy, _, _ = D.token_logprobs_forward(x, targets, temperature)
    grad, _, _ = D.token_logprobs_backward(x, targets, stats, entropy, g, gh, temperature)
    diff = _differences(loss, x.clone())
    diff[1, 3] = 0.0     # differences of a masked logit do not exist
    torch.testing.assert_close(grad, diff, rtol=1e-6, atol=1e-6)
    assert float(grad[2].abs().max()) == 0.0 and float(grad[1, 3]) == 0.0


def test_token_logprobs_conventions():
    inf = math.inf
    x = torch.tensor([[1.0, 3.0, 3.0, -inf], [-inf] * 4, [0.0, math.nan, 2.0, -inf], [inf, 1.0, 1.0, 1.0]], dtype=F64)
    lp, stats, h, tlp, ti = D.token_logprobs_forward(x, torch.tensor([0, 1, 2, 1]), top_k=3)
    assert ti.tolist() == [[1, 2, 0], [-1, -1, -1], [1, 2, 0], [0, 1, 2]]
    assert float(lp[1]) == -inf and float(h[1]) == 0.0 and stats[1].tolist() == [-inf, 0.0]
    assert bool(torch.isnan(lp[2:]).all()) and bool(torch.isnan(h[2:]).all())
    want = torch.log_softmax(x[0], -1)
    torch.testing.assert_close(tlp[0], want[[1, 2, 0]])
    torch.testing.assert_close(lp[0], want[0])
    lowest = torch.full((1, 5), torch.finfo(torch.float32).min, dtype=F64)   # every logit the lowest value: uniform
    lp, _, h, _, _ = D.token_logprobs_forward(lowest, torch.tensor([2]))
    torch.testing.assert_close(lp, torch.tensor([-math.log(5)], dtype=F64))
    torch.testing.assert_close(h, torch.tensor([math.log(5)], dtype=F64))


@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("temperature", [1.0, 1.7])
def test_distill_gradient(tail, temperature):
    torch.manual_seed(5)
    rows, cols, k = 5, 11, 4
    x = torch.randn(rows, cols, dtype=F64)
    index = torch.stack([torch.randperm(cols)[:k] for _ in range(rows)])
    logprob = torch.log_softmax(torch.randn(rows, k, dtype=F64), -1) + math.log(0.8)
    index[1, 2] = -1                                  # an unused place
    index[2, 3] = index[2, 0]                         # the same column twice
    index[3] = -1                                     # no teacher
    logprob[4] = logprob[4] + math.log(1.5)           # a list of more than 1
    dloss = torch.randn(rows, dtype=F64)

    def loss(v):
        return (D.distill_topk_forward(v, index, logprob, temperature, tail)[0] * dloss).sum()

    value, stats = D.distill_topk_forward(x, index, logprob, temperature, tail)
    assert float(value[3]) == 0.0 and bool((value[[0, 1, 4]] >= 0).all())
    grad, _ = D.distill_topk_backward(x, index, logprob, stats, dloss, temperature)
    torch.testing.assert_close(grad, _differences(loss, x.clone()), rtol=1e-6, atol=1e-6)


def test_distill_of_the_student_itself_is_zero():
    """A teacher list taken from the student's own distribution: loss 0, gradient 0."""
    torch.manual_seed(6)
    x = torch.randn(2, 30, dtype=F64)
    _, _, _, tlp, ti = D.token_logprobs_forward(x, None, top_k=7)
    loss, stats = D.distill_topk_forward(x, ti, tlp)
    assert float(loss.abs().max()) < 1e-14
    grad, _ = D.distill_topk_backward(x, ti, tlp, stats, torch.ones(2))
    assert float(grad.abs().max()) < 1e-14


def test_distill_edges():
    x = torch.tensor([[0.0, 1.0, -math.inf, -math.inf]] * 2 + [[-math.inf] * 4], dtype=F64)
    index = torch.tensor([[0, 1], [2, 0], [0, 1]])
    logprob = torch.log(torch.tensor([[0.5, 0.25], [0.5, 0.25], [0.5, 0.25]], dtype=F64))
    loss, stats = D.distill_topk_forward(x, index, logprob)
    # nothing left outside the list: the teacher is renormalised (2/3, 1/3)
    p = torch.tensor([2 / 3, 1 / 3], dtype=F64)
    torch.testing.assert_close(loss[0], (p * (p.log() - torch.log_softmax(x[0, :2], -1))).sum())
    assert float(loss[1]) == math.inf and float(loss[2]) == math.inf
    grad, _ = D.distill_topk_backward(x, index, logprob, stats, torch.ones(3))
    assert bool(torch.isfinite(grad).all()) and float(grad[2].abs().max()) == 0.0
    torch.testing.assert_close(grad[1, 2], torch.tensor(-0.5, dtype=F64))
