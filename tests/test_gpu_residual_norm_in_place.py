"""residual_norm in place at widths that no 16 bytes divide. A row is then copied in whole 16-byte pieces that hold the
ends of the rows before and behind it, which other clusters may be writing: those bytes must not reach any result. In
place and out of place have to agree in every bit, with as many rows as keep every cluster busy for several steps."""
import pytest
import torch

from credit_b200 import _native as N
from credit_b200 import launchers as L
from test_gpu_decoder_ops import (DEV, TYPES, _check_norm_forward, _launch, _norm_inputs, _on_gpu, _poisoned)

pytestmark = pytest.mark.gpu
SHAPES = [(5000, 37, 0, 0), (3001, 1003, 0, 0), (2500, 1003, 4, 1), (1300, 5003, 0, 0), (600, 9001, 0, 1), (300, 40001, 0, 0),
          (2000, 1000, 0, 1)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,cluster,shift", SHAPES)
@pytest.mark.parametrize("post,gate", [(True, True), (False, False)])
def test_forward(native_lib, dtype, rows, cols, cluster, shift, post, gate):
    inputs = _norm_inputs(rows, cols, dtype, rows + cols, post, gate)
    ins = tuple(_on_gpu(t, shift=shift) for t in inputs)
    want = _poisoned(L.allocate_outputs("residual_norm_forward", ins))
    _launch("residual_norm_forward", ins, want, cluster_size=cluster, residual_scale=0.7, eps=1e-5)
    _check_norm_forward(inputs, want, 0.7, 1e-5, dtype)
    for swapped in (False, True):      # the sum in the residual's place and y in the block's, and the other way round
        mine = tuple(_on_gpu(t, shift=shift) for t in inputs)
        fresh = L.allocate_outputs("residual_norm_forward", mine)
        outs = (mine[0] if swapped else mine[1], mine[1] if swapped else mine[0], fresh[2], fresh[3])
        _launch("residual_norm_forward", mine, outs, cluster_size=cluster, residual_scale=0.7, eps=1e-5)
        for a, b in zip(outs, want):
            assert (a is None and b is None) or torch.equal(a, b)
    assert N.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,cluster,shift", SHAPES)
@pytest.mark.parametrize("post", [True, False])
def test_backward(native_lib, dtype, rows, cols, cluster, shift, post):
    block, residual, weight, gate, pre = _norm_inputs(rows, cols, dtype, rows + cols, post, True)
    gen = torch.Generator().manual_seed(9)
    dy, dout = (torch.randn(rows, cols, generator=gen).to(dtype) for _ in range(2))
    r1, r2 = (torch.rand(rows, generator=gen) + 0.5 for _ in range(2))
    given = (dy, dout, block, residual, weight, gate, pre, r1 if post else None, r2)
    ins = tuple(_on_gpu(t, shift=shift) for t in given)
    want = _poisoned(L.allocate_outputs("residual_norm_backward", ins))
    _launch("residual_norm_backward", ins, want, cluster_size=cluster, residual_scale=0.7)
    for place in (2, 0):               # dblock in the block's place, and in dy's; dresidual in dresidual_out's
        mine = tuple(_on_gpu(t, shift=shift) for t in given)
        outs = (mine[place], mine[1], *L.allocate_outputs("residual_norm_backward", mine)[2:])
        _launch("residual_norm_backward", mine, outs, cluster_size=cluster, residual_scale=0.7)
        for a, b in zip(outs, want):
            assert (a is None and b is None) or torch.equal(a, b)
    assert N.device_status() == 0
