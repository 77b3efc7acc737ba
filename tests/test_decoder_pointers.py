"""Addresses that are not aligned to their elements are refused by residual_norm, token_logprobs and
distill_topk before any device is touched: addresses here are numbers that nothing dereferences. No GPU needed."""
import pytest

from credit_b200 import _native as N
from test_decoder_refusals import (BAD, P, _distill, _distill_bwd, _logprobs, _logprobs_bwd, _norm, _norm_bwd, _refused)


@pytest.mark.parametrize("dtype,off", [(N.BF16, 1), (N.BF16, 15), (N.F32, 1), (N.F32, 2), (N.F32, 14)])
@pytest.mark.parametrize("name", ["block", "residual", "out", "y"])
def test_residual_norm_forward_matrices(native_lib, name, dtype, off):
    _refused(_norm(native_lib, dtype=dtype, **{name: 5 * P + off}), BAD, "aligned")


@pytest.mark.parametrize("name", ["post", "gate", "pre", "r1", "r2"])
@pytest.mark.parametrize("off", [1, 2, 6])
def test_residual_norm_forward_vectors(native_lib, name, off):
    _refused(_norm(native_lib, **{name: P + off}), BAD, "aligned")


@pytest.mark.parametrize("dtype,off", [(N.BF16, 1), (N.BF16, 15), (N.F32, 1), (N.F32, 2), (N.F32, 14)])
@pytest.mark.parametrize("name", ["dy", "dout", "block", "out", "db", "dr"])
def test_residual_norm_backward_matrices(native_lib, name, dtype, off):
    _refused(_norm_bwd(native_lib, dtype=dtype, **{name: 7 * P + off}), BAD, "aligned")


@pytest.mark.parametrize("name", ["post", "gate", "pre", "r1", "r2", "dpost", "dgate", "dpre"])
@pytest.mark.parametrize("off", [1, 2, 6])
def test_residual_norm_backward_vectors(native_lib, name, off):
    _refused(_norm_bwd(native_lib, **{name: P + off}), BAD, "aligned")


@pytest.mark.parametrize("name,off", [("logits", 2), ("targets", 4), ("logprob", 2), ("stats", 1), ("entropy", 3), ("top", 2),
                                      ("index", 4)])
def test_token_logprobs_forward(native_lib, name, off):
    _refused(_logprobs(native_lib, **{name: P + off}), BAD, "aligned")


@pytest.mark.parametrize("name,off", [("logits", 2), ("targets", 4), ("stats", 1), ("entropy", 3), ("g", 2), ("gh", 2),
                                      ("dlogits", 2)])
def test_token_logprobs_backward(native_lib, name, off):
    _refused(_logprobs_bwd(native_lib, **{name: 3 * P + off}), BAD, "aligned")


@pytest.mark.parametrize("name,off", [("logits", 2), ("index", 4), ("teacher", 2), ("loss", 1), ("stats", 2)])
def test_distill_forward(native_lib, name, off):
    _refused(_distill(native_lib, **{name: P + off}), BAD, "aligned")


@pytest.mark.parametrize("name,off", [("logits", 2), ("index", 4), ("teacher", 2), ("stats", 2), ("g", 1), ("dlogits", 2)])
def test_distill_backward(native_lib, name, off):
    _refused(_distill_bwd(native_lib, **{name: 3 * P + off}), BAD, "aligned")
