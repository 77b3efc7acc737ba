"""token_logprobs with as many rows as fill the device, on both sides of the row length at which the CTAs of rows with
alternatives change size (224 KiB), against fp64 torch on the GPU. Tolerances as in test_gpu_decoder_ops.py."""
import math

import pytest
import torch

from credit_b200 import _native as N
from credit_b200 import launchers as L
from test_gpu_decoder_ops import DEV, U, _launch, _poisoned

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,cols", [(torch.bfloat16, 114687), (torch.bfloat16, 114688), (torch.float32, 57343),
                                        (torch.float32, 57344)])
@pytest.mark.parametrize("top_k", [0, 20])
def test_both_sides_of_the_border(native_lib, dtype, cols, top_k):
    rows = 8 * torch.cuda.get_device_properties(DEV).multi_processor_count
    gen = torch.Generator(device=DEV).manual_seed(cols)
    x = (torch.randn(rows, cols, generator=gen, device=DEV) * 2.0).to(dtype)
    targets = torch.randint(0, cols, (rows,), generator=gen, device=DEV)
    outs = _poisoned(L.allocate_outputs("token_logprobs_forward", (x, targets), top_k=top_k))
    _launch("token_logprobs_forward", (x, targets), outs)
    log_n = math.log2(cols)
    e_sum = (128 + 64 * log_n) * U
    for r in range(0, rows, 148):
        logp = torch.log_softmax(x[r:r + 148].double(), -1)
        at = slice(r, r + logp.shape[0])
        size = logp.gather(1, targets[at, None])[:, 0]
        assert bool(((outs[0][at] - size).abs() <= e_sum + 8 * U * (size.abs() + 2 * log_n)).all())
        entropy = -(logp.exp() * logp).sum(-1)
        assert float((outs[2][at] - entropy).abs().max()) <= e_sum * (2 + log_n) + 8 * U * log_n
        if top_k:
            value, index = torch.sort(x[at], dim=-1, descending=True, stable=True)
            want = logp.gather(1, index[:, :top_k])
            assert torch.equal(outs[4][at], index[:, :top_k])
            assert bool(((outs[3][at] - want).abs() <= e_sum + 8 * U * (want.abs() + 2 * log_n)).all())
    assert N.device_status() == 0
