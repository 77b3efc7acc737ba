"""distill_topk with teacher lists far from log probabilities: raw logits a long way from zero, lists whose
exponentials leave the range of 64 bits, above and below. The result depends on the differences inside the list
alone, so the tolerances are those of an ordinary list (test_gpu_decoder_ops.py) and hold no term of its offset:
the differences are exact or rounded once, their exponentials are off by 4 u + 2 u |log w|, the normaliser by
8 u, within the 24 u |log w| of the loss and the 64 u of the gradient."""
import math

import pytest
import torch

from credit_b200 import _native as N
from credit_b200 import launchers as L
from oracle import decoder_ops as D
from test_gpu_decoder_ops import DEV, NAN, TYPES, U, _launch, _logits, _poisoned, _rounding, _within

pytestmark = pytest.mark.gpu


def _inputs(dtype, cols, k, offset):
    x, _ = _logits(5, cols, dtype, 7)
    gen = torch.Generator().manual_seed(8)
    index = torch.stack([torch.randperm(cols, generator=gen)[:k] for _ in range(5)])
    # multiples of 2^-6, which fp32 holds up to 2^18: the same list at every offset but the last
    value = (torch.randn(5, k, generator=gen) * 128).round() / 64 + offset
    keep = x[1, index[1]].clone()
    x[1] = -math.inf
    x[1, index[1]] = keep                   # nothing left outside the list
    index[2, 4] = index[2, 1]               # a column twice
    index[3, 2:] = -1                       # unused places
    value[3, 2:] = NAN                      # are not read
    value[4, 3:] = -math.inf                # entries without mass
    return x, index, value


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("offset", [-3e5, -16384.0, -800.0, -80.0, 0.0, 7.0, 80.0, 800.0, 16384.0, 3e5])
@pytest.mark.parametrize("cluster", [1, 4])
def test_lists_far_from_zero(native_lib, dtype, tail, offset, cluster):
    cols, k, temperature = 1003, 12, 1.3
    x, index, value = _inputs(dtype, cols, k, offset)
    logits = x.to(DEV)
    ins = (logits, index.to(DEV), value.to(DEV))
    outs = _poisoned(L.allocate_outputs("distill_topk_forward", ins))
    _launch("distill_topk_forward", ins, outs, cluster_size=cluster, temperature=temperature, tail=tail)
    loss, stats = D.distill_topk_forward(x, index, value, temperature, tail)
    m, ls, m2, ls2, norm, rest = stats.unbind(-1)
    log_n = math.log2(cols)
    e_sum = (128 + 64 * log_n) * U
    logw = torch.where(index >= 0, value.double() - norm[:, None], -math.inf)
    w = logw.exp()
    logq = (x.double().gather(1, index.clamp(min=0)) - m[:, None]) / temperature - ls[:, None]
    size = torch.where(w > 0, w * (logw.abs() + logq.abs() + 4 * log_n), 0.0).sum(-1)
    tail_size = (torch.log(rest).abs() + ((m2 - m) / temperature + ls2 - ls).abs()).nan_to_num(0.0, 0.0, 0.0)
    _within(outs[0], loss, (size + rest * tail_size) * 24 * U + 3 * e_sum, "loss")

    dloss = torch.randn(5, generator=torch.Generator().manual_seed(3))
    (grad,) = _poisoned(L.allocate_outputs("distill_topk_backward", (logits,)))
    _launch("distill_topk_backward", (*ins, outs[1], dloss.to(DEV)), (grad,), temperature=temperature, tail=tail)
    want, mag = D.distill_topk_backward(x, index, value, stats, dloss, temperature)
    far = ((x.double() - m[:, None]).abs() + (x.double() - m2[:, None]).abs()).nan_to_num(0.0, 0.0, 0.0) / temperature
    extra = ls.abs() + ls2.abs() + ((m - m2).abs() / temperature).nan_to_num(0.0, 0.0, 0.0)
    _within(grad, want, mag * U * (64 + 16 * far + 16 * extra[:, None]) + _rounding(dtype, want), "dlogits")
    assert N.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("cluster", [1, 4])
def test_nan_and_inf_at_a_used_place(native_lib, dtype, tail, cluster):
    """NaN throughout such a row; the rows beside it, and the same values at unused places, are as they were."""
    x, index, value = _inputs(dtype, 1003, 12, -2.0)
    want_ins = (x.to(DEV), index.to(DEV), value.to(DEV))
    value, index = value.clone(), index.clone()
    value[0, 5], value[2, 0] = NAN, math.inf
    value[3, 2], value[3, 3] = math.inf, NAN           # unused places
    dloss = torch.ones(5, device=DEV)
    results = []
    for ins in (want_ins, (x.to(DEV), index.to(DEV), value.to(DEV))):
        outs = _poisoned(L.allocate_outputs("distill_topk_forward", ins))
        _launch("distill_topk_forward", ins, outs, cluster_size=cluster, tail=tail)
        (grad,) = _poisoned(L.allocate_outputs("distill_topk_backward", ins))
        _launch("distill_topk_backward", (*ins, outs[1], dloss), (grad,), tail=tail)
        results.append((outs[0], grad))
    (loss, grad), (got_loss, got_grad) = results
    broken = torch.tensor([True, False, True, False, False], device=DEV)
    assert bool(torch.isnan(got_loss[broken]).all()) and bool(torch.isnan(got_grad[broken]).all())
    assert torch.equal(got_loss[~broken], loss[~broken]) and torch.equal(got_grad[~broken], grad[~broken])
    assert N.device_status() == 0
