"""The registry's entries of residual_norm, token_logprobs and distill_topk: seeded inputs, what the backward
inputs hold of a forward pass, byte accounting, and that every entry has its launcher. No GPU needed."""
import math

import pytest
import torch

from credit_b200 import launchers as L
from credit_b200 import workloads as W
from oracle import decoder_ops as D

NAMES = [f"{op}_{way}" for op in ("residual_norm", "token_logprobs", "distill_topk") for way in ("forward", "backward")]


@pytest.mark.parametrize("name", NAMES)
def test_entries_are_seeded_and_have_launchers(name):
    spec = W.WORKLOADS[name]
    assert spec.name == name and name in L.NATIVE_LAUNCHERS
    a, b = (spec.input_factory(3, 200, torch.device("cpu"), seed=5) for _ in range(2))
    for s, t in zip(a, b):
        assert torch.equal(s, t)
    assert a[0].shape == (3, 200) and a[0].dtype == spec.dtype
    assert not torch.equal(a[0], spec.input_factory(3, 200, torch.device("cpu"), seed=6)[0])


def test_byte_accounting():
    assert W.algorithmic_bytes("residual_norm_forward", 10, 64) == 4 * 10 * 64 * 2 + 3 * 64 * 4 + 2 * 10 * 4
    assert W.algorithmic_bytes("residual_norm_backward", 10, 64) == 6 * 10 * 64 * 2 + 6 * 64 * 4 + 2 * 10 * 4
    assert W.algorithmic_bytes("token_logprobs_backward", 10, 1000) == 2 * 10 * 1000 * 2 + 280
    assert W.algorithmic_bytes("distill_topk_forward", 10, 1000) == 10 * 1000 * 2 + 10 * (12 * 64 + 28)


def test_backward_inputs_hold_the_forward_pass():
    # fp32 sums of 300 terms against fp64: 300 * 2^-24 relative, logarithms of order 10
    logits, targets, stats, entropy, _, _ = W.make_token_logprobs_backward_inputs(4, 300, "cpu")
    _, want, h, _, _ = D.token_logprobs_forward(logits, targets)
    assert float((stats.double() - want).abs().max()) < 1e-4 and float((entropy.double() - h).abs().max()) < 1e-4
    logits, index, value, stats, _ = W.make_distill_topk_backward_inputs(4, 300, "cpu")
    assert all(len(set(row)) == 64 for row in index.tolist())
    assert float((value.exp().sum(-1) - 0.9).abs().max()) < 1e-5
    _, want = D.distill_topk_forward(logits, index, value)
    assert float((stats.double() - want).abs().max()) < 1e-4 and math.isclose(float(stats[0, 5]), 0.1, rel_tol=1e-4)
    ins = W.make_residual_norm_backward_inputs(4, 300, "cpu")
    assert float((ins[7].double() - (ins[2].double().square().mean(-1) + 1e-6).rsqrt()).abs().max()) < 1e-5
