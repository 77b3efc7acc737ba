"""The gradient of residual_norm against differences of the forward pass, tight enough that neither of the two mean
terms (which make it the gradient of a norm) can be missing: with t = dy w_pre, v = h' r2, D = dh' + r2 (t - v mean(t v)),
n = o r1, the terms r2 v mean(t v) and r1 n mean(D c n). The entries that are looked at are those that the terms
change most.

Differences: f' = (8 (f(h) - f(-h)) - (f(2h) - f(-2h))) / 12 h at h = 0.1, of L = sum(residual_out dresidual_out) + sum(y dy).
What they may be off by, u = 2^-24:
* their own error (order h^4), which the same differences of the fp64 oracle show exactly: |differences - gradient| there;
* the roundings of the fp32 forward outputs. Rows of 64 in fp32: a square sum goes through at most 4 + 5 + 2 additions,
  its mean and eps 2, rsqrt 2 more ulps: r1 is off by (13 / 2 + 4) u < 11 u. n adds 3 roundings, the join one of its
  sum: |n| 14 u + |out| u. r2: the relative error of the row's entries, at most (|n| 14 u + |out| u) in the norm of the
  row, and its own 11 u; y: that twice (its entry and its r2) and 13 u. So at most e_out = 14 u |n| + u |out| and
  e_y = r2 w_pre (e_out + |out| (rms(e_out) r2 + 13 u)). The four evaluations weigh 18 / 12 h:
  1.5 / h (sum |dresidual_out| e_out + sum |dy| e_y) over the rows that the entry reaches, at the unperturbed point, and
  a tenth of that again for the perturbed ones;
* the kernel's gradient: 100 u of its magnitude, (rows + 200) u for the column sums, as in test_gpu_decoder_ops.py.
The entry moves by h up to 0.2 of values of order 1, which the oracle's differences follow exactly."""
import math

import pytest
import torch

from credit_b200 import launchers as L
from oracle import decoder_ops as D

U = 2.0 ** -24
ROWS, COLS, SCALE, EPS, H = 3, 64, 0.7, 1e-5, 0.1
NAMES = ("block", "residual", "post_weight", "gate", "pre_weight")


def _inputs():
    gen = torch.Generator().manual_seed(12)
    ins = [torch.randn(ROWS, COLS, generator=gen) for _ in range(2)]
    ins += [torch.rand(COLS, generator=gen) + 0.5 for _ in range(3)]
    # one direction in common with the values, so that the means are of order 1 and not of order 1 / sqrt(cols)
    dy, dout = (torch.randn(ROWS, COLS, generator=gen) + 0.5 * ins[0] + 0.5 * ins[1] for _ in range(2))
    return ins, dy, dout


def _gradient(ins, dy, dout, pre_mean=True, post_mean=True):
    """The fp64 formulas, with either mean term left out on demand."""
    o, r, w1, g, w2 = (t.double() for t in ins)
    dy, dout, c = dy.double(), dout.double(), w1 * g
    out, _, r1, r2 = D.residual_norm_forward(o, r, w1, g, w2, SCALE, EPS)
    r1, r2 = r1[:, None], r2[:, None]
    v, t, n = out * r2, dy * w2, o * r1
    total = dout + r2 * (t - v * (t * v).mean(-1, keepdim=True) * pre_mean)
    dn = c * total
    shared = (total * n).sum(0)
    return (r1 * (dn - n * (dn * n).mean(-1, keepdim=True) * post_mean), SCALE * total, g * shared, w1 * shared, (dy * v).sum(0))


def _differences(loss, ins, which, i):
    flat = ins[which].view(-1)
    keep = flat[i].clone()
    values = []
    for step in (H, -H, 2 * H, -2 * H):
        flat[i] = keep + step
        values.append((loss(ins), float(flat[i]) - float(keep)))
    flat[i] = keep
    (up, a), (down, b), (up2, c), (down2, d) = values
    # the steps as stored: a - b = 2 h and c - d = 4 h up to a rounding of h
    return (8 * (up - down) * (2 * H / (a - b)) - (up2 - down2) * (4 * H / (c - d))) / (12 * H)


def _loss64(dy, dout):
    def loss(ins):
        out, y, _, _ = D.residual_norm_forward(*ins, SCALE, EPS)
        return float((out * dout.double()).sum() + (y * dy.double()).sum())
    return loss


def _entries():
    """(input, place, gradient, tolerance, what leaving out each term changes) of the entries looked at."""
    ins, dy, dout = _inputs()
    full = _gradient(ins, dy, dout)
    without = [_gradient(ins, dy, dout, False, True), _gradient(ins, dy, dout, True, False)]
    o, r, w1, g, w2 = (t.double() for t in ins)
    out, _, r1, r2 = D.residual_norm_forward(o, r, w1, g, w2, SCALE, EPS)
    n = (out - SCALE * r).abs()
    e_out = 14 * U * n + U * out.abs()
    rms = e_out.square().mean(-1).sqrt() * r2
    e_y = r2[:, None] * w2 * (e_out + out.abs() * (rms[:, None] + 13 * U))
    rounding = (1.65 / H) * ((dout.double().abs() * e_out).sum(-1) + (dy.double().abs() * e_y).sum(-1))
    _, mags = D.residual_norm_backward(dy, dout, o, out, w1, g, w2, r1, r2, SCALE)
    ins64 = [t.double() for t in ins]
    entries = []
    for which in range(5):
        change = [(full[which] - w[which]).abs().view(-1) for w in without]
        places = {int(c.argmax()) for c in change} | {0, full[which].numel() - 1}
        for i in sorted(places):
            want = float(full[which].reshape(-1)[i])
            own = abs(_differences(_loss64(dy, dout), ins64, which, i) - want)
            reach = float(rounding[i // COLS] if which < 2 else rounding.sum())
            kernel = U * (100 if which < 2 else ROWS + 200) * float(mags[which].reshape(-1)[i])
            entries.append((which, i, want, own + reach + kernel, [float(c[i]) for c in change]))
    return ins, dy, dout, full, entries


def test_a_missing_term_exceeds_the_tolerance():
    """Each of the terms, left out of any gradient that holds it, is seen at some entry by at least four tolerances."""
    _, _, _, full, entries = _entries()
    for term in (0, 1):
        for which in ((0, 1, 2, 3) if term == 0 else (0,)):      # dpre_weight holds neither, the others the first
            ratio = max(change[term] / tol for w, _, _, tol, change in entries if w == which)
            assert ratio > 4.0, (NAMES[which], term, ratio)
    for which, i, want, tol, _ in entries:
        assert abs(want - float(full[which].reshape(-1)[i])) == 0.0 and tol < 0.05


def test_the_formulas_are_those_of_the_oracle():
    ins, dy, dout = _inputs()
    wide = [t.double() for t in ins]
    out, _, r1, r2 = D.residual_norm_forward(*wide, SCALE, EPS)
    want, _ = D.residual_norm_backward(dy, dout, wide[0], out, wide[2], wide[3], wide[4], r1, r2, SCALE)
    for a, b in zip(_gradient(ins, dy, dout), want):
        torch.testing.assert_close(a, b, rtol=1e-12, atol=1e-14)


@pytest.mark.gpu
def test_kernel_gradient_against_differences_of_the_kernel(native_lib):
    ins, dy, dout, _, entries = _entries()
    dev = torch.device("cuda:0")
    ins = [t.to(dev) for t in ins]
    dy, dout = dy.to(dev), dout.to(dev)

    def forward(leaves):
        outs = L.allocate_outputs("residual_norm_forward", tuple(leaves))
        L.launch_residual_norm_forward(tuple(leaves), outs, residual_scale=SCALE, eps=EPS)
        return outs

    def loss(leaves):
        outs = forward(leaves)
        return float((outs[0].double() * dout).sum() + (outs[1].double() * dy).sum())

    out, _, r1, r2 = forward(ins)
    bwd = (dy, dout, ins[0], out, *ins[2:], r1, r2)
    grads = L.allocate_outputs("residual_norm_backward", bwd)
    L.launch_residual_norm_backward(bwd, grads, residual_scale=SCALE)
    for which, i, want, tol, _ in entries:
        got = float(grads[which].view(-1)[i])
        assert math.isfinite(got)
        assert abs(got - _differences(loss, ins, which, i)) <= tol, (NAMES[which], i)
        assert abs(got - want) <= tol, (NAMES[which], i)
