"""What residual_norm, token_logprobs and distill_topk refuse, through the C ABI, before any device is
touched: addresses here are numbers that nothing dereferences. No GPU needed."""
import pytest
import torch

from credit_b200 import _native as N
from credit_b200 import launchers as L

P = 1 << 20          # a 16-byte aligned address
BAD, UNSUPPORTED = N.ERR_INVALID_ARGUMENT, N.ERR_UNSUPPORTED


def _refused(code, want, word):
    assert code == want and word in N.last_error(), (code, N.last_error())


def _logprobs(lib, *, logits=P, ld=100, targets=P, logprob=P, stats=P, entropy=P, top=P, index=P, k=4, rows=2, cols=100,
              t=1.0, dtype=N.F32, opts=None):
    return lib.credit_token_logprobs_forward(logits, ld, targets, logprob, stats, entropy, top, index, k, rows, cols, t,
                                             dtype, N.opts_ref(opts), None)


@pytest.mark.parametrize("change,code,word", [
    (dict(logits=None), BAD, "logits"), (dict(logits=P + 2), BAD, "aligned"), (dict(ld=99), BAD, "row_stride"),
    (dict(ld=1 << 31), BAD, "row_stride"), (dict(targets=None), BAD, "go together"), (dict(logprob=None), BAD, "go together"),
    (dict(stats=None), BAD, "stats"), (dict(k=-1), BAD, "top_k"), (dict(k=129), BAD, "top_k"), (dict(top=None), BAD, "top_logprob"),
    (dict(index=None), BAD, "top_index"), (dict(rows=-1), BAD, "rows"), (dict(cols=0), BAD, "cols"),
    (dict(cols=1 << 23, ld=1 << 23), UNSUPPORTED, "columns"), (dict(t=0.0), BAD, "temperature"), (dict(t=-1.0), BAD, "temperature"),
    (dict(t=float("nan")), BAD, "temperature"), (dict(t=float("inf")), BAD, "temperature"), (dict(t=1e-45), BAD, "temperature"),
    (dict(dtype=7), BAD, "dtype"), (dict(opts={"cluster_size": 3}), BAD, "cluster_size"),
    (dict(opts={"threads": 256}), BAD, "cluster_size only"),
    (dict(targets=None, logprob=None, entropy=None, k=0), BAD, "nothing"),
])
def test_token_logprobs_forward_refuses(native_lib, change, code, word):
    _refused(_logprobs(native_lib, **change), code, word)


def test_no_rows_is_no_work(native_lib):
    assert _logprobs(native_lib, logits=None, targets=None, logprob=None, stats=None, rows=0) == N.CREDIT_OK
    assert _logprobs_bwd(native_lib, logits=None, dlogits=None, rows=0) == N.CREDIT_OK
    assert _distill(native_lib, logits=None, index=None, rows=0) == N.CREDIT_OK
    assert _distill_bwd(native_lib, logits=None, dlogits=None, rows=0) == N.CREDIT_OK
    assert _norm(native_lib, block=None, rows=0) == N.CREDIT_OK


def _logprobs_bwd(lib, *, logits=P, ld=100, targets=P, stats=P, entropy=P, g=P, gh=P, dlogits=2 * P, out_ld=100, rows=2,
                  cols=100, t=1.0, dtype=N.F32, opts=None):
    return lib.credit_token_logprobs_backward(logits, ld, targets, stats, entropy, g, gh, dlogits, out_ld, rows, cols, t,
                                              dtype, N.opts_ref(opts), None)


@pytest.mark.parametrize("change,word", [
    (dict(targets=None), "targets"), (dict(stats=None), "stats"), (dict(g=None), "dlogprob"), (dict(entropy=None), "entropy"),
    (dict(dlogits=None), "dlogits"), (dict(out_ld=99), "dlogits_row_stride"), (dict(dlogits=P + 4), "overlap"),
    (dict(dlogits=P, out_ld=101), "overlap"), (dict(dlogits=P + 199 * 4), "overlap"), (dict(dlogits=2 * P + 1), "aligned"),
    (dict(opts={"cluster_size": 2}), "elementwise"), (dict(opts={"stages": 2}), "cluster_size only"),
])
def test_token_logprobs_backward_refuses(native_lib, change, word):
    _refused(_logprobs_bwd(native_lib, **change), BAD, word)


def _distill(lib, *, logits=P, ld=100, index=P, teacher=P, k=4, loss=P, stats=P, rows=2, cols=100, t=1.0, tail=1,
             dtype=N.F32, opts=None):
    return lib.credit_distill_topk_forward(logits, ld, index, teacher, k, loss, stats, rows, cols, t, tail, dtype,
                                           N.opts_ref(opts), None)


def _distill_bwd(lib, *, logits=P, ld=100, index=P, teacher=P, k=4, stats=P, g=P, dlogits=2 * P, out_ld=100, rows=2,
                 cols=100, t=1.0, dtype=N.F32, opts=None):
    return lib.credit_distill_topk_backward(logits, ld, index, teacher, k, stats, g, dlogits, out_ld, rows, cols, t, dtype,
                                            N.opts_ref(opts), None)


@pytest.mark.parametrize("change,word", [
    (dict(index=None), "teacher_index"), (dict(teacher=None), "teacher_logprob"), (dict(k=0), "top_k"), (dict(k=129), "top_k"),
    (dict(loss=None), "loss"), (dict(stats=None), "stats"), (dict(t=0.0), "temperature"), (dict(ld=50), "row_stride"),
    (dict(opts={"schedule": 1}), "cluster_size only"),
])
def test_distill_forward_refuses(native_lib, change, word):
    _refused(_distill(native_lib, **change), BAD, word)


@pytest.mark.parametrize("change,word", [
    (dict(index=None), "teacher_index"), (dict(k=200), "top_k"), (dict(stats=None), "stats"), (dict(g=None), "dloss"),
    (dict(dlogits=P + 16), "overlap"), (dict(opts={"cluster_size": 8}), "elementwise"),
])
def test_distill_backward_refuses(native_lib, change, word):
    _refused(_distill_bwd(native_lib, **change), BAD, word)


def _norm(lib, *, block=P, residual=2 * P, post=P, gate=P, pre=P, out=3 * P, y=4 * P, r1=P, r2=P, rows=2, cols=128, scale=1.0,
          eps=1e-6, dtype=N.BF16, opts=None):
    return lib.credit_residual_norm_forward(block, residual, post, gate, pre, out, y, r1, r2, rows, cols, scale, eps, dtype,
                                            N.opts_ref(opts), None)


@pytest.mark.parametrize("change,code,word", [
    (dict(block=None), BAD, "block"), (dict(residual=None), BAD, "residual"), (dict(pre=None), BAD, "pre_weight"),
    (dict(out=None), BAD, "residual_out"), (dict(y=None), BAD, "y"), (dict(r2=None), BAD, "pre_rstd"),
    (dict(post=None), BAD, "go together"), (dict(r1=None), BAD, "go together"), (dict(y=3 * P), BAD, "differ"),
    (dict(eps=0.0), BAD, "eps"), (dict(eps=float("nan")), BAD, "eps"), (dict(scale=float("inf")), BAD, "residual_scale"),
    (dict(cols=1 << 18), UNSUPPORTED, "columns"), (dict(cols=20000, opts={"cluster_size": 1}), UNSUPPORTED, "columns"),
    (dict(opts={"variant": 1}), BAD, "cluster_size only"),
])
def test_residual_norm_forward_refuses(native_lib, change, code, word):
    _refused(_norm(native_lib, **change), code, word)


def _norm_bwd(lib, *, dy=P, dout=2 * P, block=3 * P, out=4 * P, post=P, gate=P, pre=P, r1=P, r2=P, db=5 * P, dr=6 * P, dpost=P,
              dgate=P, dpre=P, rows=2, cols=128, scale=1.0, dtype=N.BF16, opts=None, ws=P, ws_bytes=1 << 30):
    return lib.credit_residual_norm_backward(dy, dout, block, out, post, gate, pre, r1, r2, db, dr, dpost, dgate, dpre, rows,
                                             cols, scale, dtype, N.opts_ref(opts), ws, ws_bytes, None)


@pytest.mark.parametrize("change,word", [
    (dict(dy=None), "dy"), (dict(block=None), "block"), (dict(out=None), "residual_out"), (dict(db=None), "dblock"),
    (dict(dr=None), "dresidual"), (dict(dpre=None), "gradient"), (dict(dgate=None), "gradient"), (dict(post=None), "gradient"),
    (dict(r1=None), "go together"), (dict(dr=5 * P), "differ"), (dict(scale=float("nan")), "residual_scale"),
])
def test_residual_norm_backward_refuses(native_lib, change, word):
    _refused(_norm_bwd(native_lib, **change), BAD, word)


def test_workspace_of_a_refused_shape_is_zero(native_lib):
    assert native_lib.credit_residual_norm_backward_workspace_bytes(4, 1 << 20, N.BF16, None) == 0
    assert native_lib.credit_residual_norm_backward_workspace_bytes(-1, 128, N.BF16, None) == 0


def test_launchers_refuse_host_tensors():
    x = torch.zeros(2, 8)
    for name in ("token_logprobs_forward", "distill_topk_forward", "residual_norm_forward"):
        outs = (None,) * 5 if name == "token_logprobs_forward" else (None,) * (2 if name.startswith("distill") else 4)
        ins = {"token_logprobs_forward": (x, None), "distill_topk_forward": (x, None, None),
               "residual_norm_forward": (x, x, None, None, x)}[name]
        with pytest.raises(ValueError, match="CUDA tensor"):
            L.NATIVE_LAUNCHERS[name](ins, outs)
