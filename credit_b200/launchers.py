"""In-process launcher table of the native backend.

Same convention as the reference's Triton table
(`dsmem_eval/triton_kernels.py:300-414`): `launcher(inputs, outputs, ...)`
takes caller-owned device tensors, enqueues on the current CUDA stream and
returns nothing; `allocate_outputs(name, inputs)` pre-allocates the outputs. The
Triton knobs (`block_size`, `num_warps`) have no meaning for these kernels; the
knobs here are the cluster size and the other launch options of the C ABI.

torch is used for device memory and streams only; every kernel is in
`libcredit_b200.so`.
"""
from __future__ import annotations

import torch

from . import _native as N

_DTYPES = {torch.float32: N.F32, torch.bfloat16: N.BF16}


def _stream_ptr() -> int:
    return torch.cuda.current_stream().cuda_stream


def _check_matrix(name: str, t: torch.Tensor, dtype=None, shape=None) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must have dtype {dtype}, got {t.dtype}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _row_dtype(x: torch.Tensor) -> int:
    if x.dtype not in _DTYPES:
        raise ValueError(f"unsupported dtype {x.dtype}: float32 and bfloat16 only")
    return _DTYPES[x.dtype]


def _opts(cluster_size: int, opts) -> "N.LaunchOpts | None":
    o = N.make_opts(opts)
    if cluster_size:
        if o is None:
            o = N.LaunchOpts()
        else:
            o = N.LaunchOpts(**{name: getattr(o, name) for name, _ in N.LaunchOpts._fields_})
        o.cluster_size = int(cluster_size)
    return o


def _ref(o):
    import ctypes
    return None if o is None else ctypes.byref(o)


def launch_rmsnorm_forward(inputs, outputs, cluster_size: int = 0, opts=None, eps: float = 1.0e-6) -> None:
    x, gamma = inputs
    (y,) = outputs
    _check_matrix("x", x)
    rows, cols = x.shape
    _check_matrix("gamma", gamma, torch.float32, (cols,))
    _check_matrix("y", y, x.dtype, x.shape)
    o = _opts(cluster_size, opts)
    with torch.cuda.device(x.device):
        N.check(N.load().credit_rmsnorm_forward(
            x.data_ptr(), gamma.data_ptr(), y.data_ptr(), rows, cols, eps, _row_dtype(x), _ref(o),
            _stream_ptr()))


def launch_row_reduce(inputs, outputs, cluster_size: int = 0, opts=None) -> None:
    (x,) = inputs
    row_sum, row_max, row_argmax = outputs
    _check_matrix("x", x, torch.float32)
    rows, cols = x.shape
    _check_matrix("sum", row_sum, torch.float32, (rows,))
    _check_matrix("max", row_max, torch.float32, (rows,))
    _check_matrix("argmax", row_argmax, torch.int64, (rows,))
    o = _opts(cluster_size, opts)
    with torch.cuda.device(x.device):
        N.check(N.load().credit_row_reduce(
            x.data_ptr(), row_sum.data_ptr(), row_max.data_ptr(), row_argmax.data_ptr(), rows, cols,
            _ref(o), _stream_ptr()))


def launch_layernorm_forward(inputs, outputs, cluster_size: int = 0, opts=None, eps: float = 1.0e-5) -> None:
    x, gamma, beta = inputs
    y, mean, rstd = outputs
    _check_matrix("x", x)
    rows, cols = x.shape
    _check_matrix("gamma", gamma, torch.float32, (cols,))
    _check_matrix("beta", beta, torch.float32, (cols,))
    _check_matrix("y", y, x.dtype, x.shape)
    _check_matrix("mean", mean, torch.float32, (rows,))
    _check_matrix("rstd", rstd, torch.float32, (rows,))
    o = _opts(cluster_size, opts)
    with torch.cuda.device(x.device):
        N.check(N.load().credit_layernorm_forward(
            x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), y.data_ptr(), mean.data_ptr(),
            rstd.data_ptr(), rows, cols, eps, _row_dtype(x), _ref(o), _stream_ptr()))


def launch_layernorm_backward(inputs, outputs, cluster_size: int = 0, opts=None, eps: float = 1.0e-5) -> None:
    """dx with statistics recomputed from x: the reference workload
    (`launch_layernorm_backward`, triton_kernels.py:300-312)."""
    x, dy, gamma = inputs
    (dx,) = outputs
    _check_matrix("x", x)
    rows, cols = x.shape
    _check_matrix("dy", dy, x.dtype, x.shape)
    _check_matrix("gamma", gamma, torch.float32, (cols,))
    _check_matrix("dx", dx, x.dtype, x.shape)
    o = _opts(cluster_size, opts)
    with torch.cuda.device(x.device):
        N.check(N.load().credit_layernorm_backward(
            x.data_ptr(), dy.data_ptr(), gamma.data_ptr(), dx.data_ptr(), rows, cols, eps,
            _row_dtype(x), _ref(o), _stream_ptr()))


def layernorm_backward_stats_workspace_bytes(rows: int, cols: int, dtype: torch.dtype,
                                             cluster_size: int = 0, opts=None) -> int:
    o = _opts(cluster_size, opts)
    # credit_plan raises with the precise status if the shape or options are unusable
    N.plan(N.WL_LAYERNORM_BACKWARD_STATS, rows, cols, _DTYPES[dtype], o)
    return int(N.load().credit_layernorm_backward_stats_workspace_bytes(
        rows, cols, _DTYPES[dtype], _ref(o)))


def launch_layernorm_backward_stats(inputs, outputs, cluster_size: int = 0, opts=None,
                                    workspace: torch.Tensor | None = None) -> None:
    """dx, dgamma, dbeta from x, dy, gamma and the saved fp32 mean/rstd. `workspace` is a
    uint8 CUDA tensor of at least `layernorm_backward_stats_workspace_bytes(...)` bytes; when
    omitted one is allocated through torch's caching allocator for this call."""
    x, dy, gamma, mean, rstd = inputs
    if len(outputs) == 1:
        (dx,), dgamma, dbeta = outputs, None, None
    else:
        dx, dgamma, dbeta = outputs
    _check_matrix("x", x)
    rows, cols = x.shape
    _check_matrix("dy", dy, x.dtype, x.shape)
    _check_matrix("gamma", gamma, torch.float32, (cols,))
    _check_matrix("mean", mean, torch.float32, (rows,))
    _check_matrix("rstd", rstd, torch.float32, (rows,))
    _check_matrix("dx", dx, x.dtype, x.shape)
    o = _opts(cluster_size, opts)
    ws_ptr, ws_bytes = 0, 0
    if dgamma is not None:
        _check_matrix("dgamma", dgamma, torch.float32, (cols,))
        _check_matrix("dbeta", dbeta, torch.float32, (cols,))
        if workspace is None:
            need = layernorm_backward_stats_workspace_bytes(rows, cols, x.dtype, 0, o)
            workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=x.device)
        _check_matrix("workspace", workspace, torch.uint8)
        ws_ptr, ws_bytes = workspace.data_ptr(), workspace.numel()
    with torch.cuda.device(x.device):
        N.check(N.load().credit_layernorm_backward_stats(
            x.data_ptr(), dy.data_ptr(), gamma.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
            dx.data_ptr(), 0 if dgamma is None else dgamma.data_ptr(),
            0 if dbeta is None else dbeta.data_ptr(), rows, cols, _row_dtype(x), _ref(o), ws_ptr,
            ws_bytes, _stream_ptr()))


def pack_ffn_weight(w: torch.Tensor) -> torch.Tensor:
    """[k, n] bf16 row-major weight -> the K-major [n, k] form the FFN GEMMs take (done once per
    weight, on the device)."""
    _check_matrix("w", w, torch.bfloat16)
    k, n = w.shape
    packed = torch.empty((n, k), dtype=torch.bfloat16, device=w.device)
    with torch.cuda.device(w.device):
        N.check(N.load().credit_ffn_pack_weight(w.data_ptr(), packed.data_ptr(), k, n, _stream_ptr()))
    return packed


def ffn_workspace_bytes(m: int, d: int, h: int) -> int:
    return int(N.load().credit_ffn_workspace_bytes(m, d, h))


def launch_ffn_forward(inputs, outputs, cluster_size: int = 0, opts=None, eps: float = 1.0e-6,
                       workspace: torch.Tensor | None = None) -> None:
    """Y = RMSNorm(GELU(X W1) W2 + X) * gamma. inputs = (x [m, d] bf16, w1_packed [h, d],
    w2_packed [d, h], gamma [d] fp32) with the weights from `pack_ffn_weight`. The cluster size
    is fixed by the width (d / 256 CTAs span a row); `cluster_size` and `opts` are accepted for
    the common launcher signature and must be left at their defaults."""
    x, w1p, w2p, gamma = inputs
    (y,) = outputs
    if cluster_size or opts:
        raise ValueError("the FFN takes no launch options: its cluster size is d / 256")
    _check_matrix("x", x, torch.bfloat16)
    m, d = x.shape
    h = w1p.shape[0]
    _check_matrix("w1_packed", w1p, torch.bfloat16, (h, d))
    _check_matrix("w2_packed", w2p, torch.bfloat16, (d, h))
    _check_matrix("gamma", gamma, torch.float32, (d,))
    _check_matrix("y", y, torch.bfloat16, (m, d))
    if workspace is None:
        workspace = torch.empty(max(ffn_workspace_bytes(m, d, h), 16), dtype=torch.uint8, device=x.device)
    _check_matrix("workspace", workspace, torch.uint8)
    with torch.cuda.device(x.device):
        N.check(N.load().credit_ffn_forward(
            x.data_ptr(), w1p.data_ptr(), w2p.data_ptr(), gamma.data_ptr(), y.data_ptr(), m, d, h, eps,
            workspace.data_ptr(), workspace.numel(), _stream_ptr()))


def _check_like(name: str, t, device: torch.device, dtype, shape) -> "int | None":
    """The checks of `_check_matrix` and that the tensor lies on `device`; returns its address (NULL when it
    is empty). What is in order costs a handful of attribute reads: small calls are bound by their host side."""
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.device == device
            and t.is_contiguous()):
        _check_matrix(name, t, dtype, shape)
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    return t.data_ptr() or None


def _check_optional(name: str, t, device: torch.device, dtype, shape) -> "int | None":
    return None if t is None else _check_like(name, t, device, dtype, shape)


def _options(cluster_size: int, opts):
    return None if not cluster_size and opts is None else _ref(_opts(cluster_size, opts))


# The current stream's address without a Stream object around it (0.1 us instead of 2.2 us a call).
_current_stream_ptr = getattr(torch._C, "_cuda_getCurrentRawStream",
                              lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(entry, device: torch.device, *args) -> None:
    """Runs a C entry point with `device` current, on that device's current stream."""
    index = device.index
    if index == torch.cuda.current_device():
        status = entry(*args, _current_stream_ptr(index))
    else:
        with torch.cuda.device(device):
            status = entry(*args, _current_stream_ptr(index))
    if status:
        N.check(status)


def launch_residual_norm_forward(inputs, outputs, cluster_size: int = 0, opts=None, residual_scale: float = 1.0,
                                 eps: float = 1.0e-6) -> None:
    """The norms after and before a block with its gate and the scaled residual:

        n = rmsnorm(block) * post_weight   (block without post_weight)
        residual_out = residual_scale * residual + gate * n;   y = rmsnorm(residual_out) * pre_weight

    inputs = (block, residual, post_weight | None, gate | None, pre_weight), outputs = (residual_out, y,
    post_rstd | None, pre_rstd). residual_out may be residual or block, y block or residual."""
    block, residual, post_weight, gate, pre_weight = inputs
    residual_out, y, post_rstd, pre_rstd = outputs
    _check_matrix("block", block)
    rows, cols = shape = block.shape
    device, dtype, f32 = block.device, block.dtype, torch.float32
    if (post_weight is None) != (post_rstd is None):
        raise ValueError("post_weight and post_rstd go together")
    _call(N.load().credit_residual_norm_forward, device, block.data_ptr() or None,
          _check_like("residual", residual, device, dtype, shape),
          _check_optional("post_weight", post_weight, device, f32, (cols,)),
          _check_optional("gate", gate, device, f32, (cols,)),
          _check_like("pre_weight", pre_weight, device, f32, (cols,)),
          _check_like("residual_out", residual_out, device, dtype, shape), _check_like("y", y, device, dtype, shape),
          _check_optional("post_rstd", post_rstd, device, f32, (rows,)),
          _check_like("pre_rstd", pre_rstd, device, f32, (rows,)),
          rows, cols, residual_scale, eps, _row_dtype(block), _options(cluster_size, opts))


def residual_norm_backward_workspace_bytes(rows: int, cols: int, dtype: torch.dtype, cluster_size: int = 0,
                                           opts=None) -> int:
    """For the current device; enough for every call of the shape, with or without post norm."""
    return int(N.load().credit_residual_norm_backward_workspace_bytes(
        rows, cols, _DTYPES[dtype], _ref(_opts(cluster_size, opts))))


def launch_residual_norm_backward(inputs, outputs, cluster_size: int = 0, opts=None, residual_scale: float = 1.0,
                                  workspace: torch.Tensor | None = None) -> None:
    """Gradient of `launch_residual_norm_forward`. inputs = (dy, dresidual_out | None, block, residual_out,
    post_weight | None, gate | None, pre_weight, post_rstd | None, pre_rstd); outputs = (dblock, dresidual,
    dpost_weight | None, dgate | None, dpre_weight). dresidual may be dresidual_out. `workspace` is a uint8
    CUDA tensor of at least `residual_norm_backward_workspace_bytes(...)` bytes; when omitted one is
    allocated through torch's caching allocator for this call."""
    dy, dresidual_out, block, residual_out, post_weight, gate, pre_weight, post_rstd, pre_rstd = inputs
    dblock, dresidual, dpost_weight, dgate, dpre_weight = outputs
    _check_matrix("dy", dy)
    rows, cols = shape = dy.shape
    device, dtype, f32 = dy.device, dy.dtype, torch.float32
    for name, t, d in (("post_weight", post_weight, dpost_weight), ("gate", gate, dgate),
                       ("pre_weight", pre_weight, dpre_weight)):
        if (t is None) != (d is None):
            raise ValueError(f"{name} and d{name} go together")
    if (post_weight is None) != (post_rstd is None):
        raise ValueError("post_weight and post_rstd go together")
    if workspace is None:
        with torch.cuda.device(device):
            need = residual_norm_backward_workspace_bytes(rows, cols, dtype, cluster_size, opts)
        workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=device)
    elif workspace.dim() != 1:
        raise ValueError("workspace must have one dimension")
    _call(N.load().credit_residual_norm_backward, device, dy.data_ptr() or None,
          _check_optional("dresidual_out", dresidual_out, device, dtype, shape),
          _check_like("block", block, device, dtype, shape),
          _check_like("residual_out", residual_out, device, dtype, shape),
          _check_optional("post_weight", post_weight, device, f32, (cols,)),
          _check_optional("gate", gate, device, f32, (cols,)),
          _check_like("pre_weight", pre_weight, device, f32, (cols,)),
          _check_optional("post_rstd", post_rstd, device, f32, (rows,)),
          _check_like("pre_rstd", pre_rstd, device, f32, (rows,)),
          _check_like("dblock", dblock, device, dtype, shape), _check_like("dresidual", dresidual, device, dtype, shape),
          _check_optional("dpost_weight", dpost_weight, device, f32, (cols,)),
          _check_optional("dgate", dgate, device, f32, (cols,)),
          _check_like("dpre_weight", dpre_weight, device, f32, (cols,)),
          rows, cols, residual_scale, _row_dtype(dy), _options(cluster_size, opts),
          _check_like("workspace", workspace, device, torch.uint8, workspace.shape), workspace.numel())


def _check_logits(name: str, t, device=None, dtype=None, shape=None) -> int:
    """Row stride of a [rows, cols] matrix whose rows are contiguous, whole or as the leading columns of a
    wider (padded) buffer."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dim() != 2:
        raise ValueError(f"{name} must have two dimensions, got {t.dim()}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must have dtype {dtype}, got {t.dtype}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    rows, cols = t.shape
    stride, step = t.stride()
    if (cols > 1 and step != 1) or (rows > 1 and stride < cols):
        raise ValueError(f"{name} must have contiguous rows that do not overlap")
    return stride if rows > 1 else cols


def launch_token_logprobs_forward(inputs, outputs, cluster_size: int = 0, opts=None, temperature: float = 1.0) -> None:
    """Log probabilities of given tokens under softmax(logits / temperature). inputs = (logits [rows, cols],
    targets int64 [rows] | None), outputs = (logprob [rows] | None, stats [rows, 2], entropy [rows] | None,
    top_logprob [rows, k] | None, top_index int64 [rows, k] | None). The logits may be the leading columns
    of a wider buffer. A negative target is an ignored row."""
    logits, targets = inputs
    logprob, stats, entropy, top_logprob, top_index = outputs
    stride = _check_logits("logits", logits)
    rows, cols = logits.shape
    device, f32 = logits.device, torch.float32
    if (targets is None) != (logprob is None):
        raise ValueError("targets and logprob go together")
    if (top_logprob is None) != (top_index is None):
        raise ValueError("top_logprob and top_index go together")
    if top_index is not None and top_index.dim() != 2:
        raise ValueError("top_index must have two dimensions")
    top_k = 0 if top_index is None else top_index.shape[1]
    _call(N.load().credit_token_logprobs_forward, device, logits.data_ptr() or None, stride,
          _check_optional("targets", targets, device, torch.int64, (rows,)),
          _check_optional("logprob", logprob, device, f32, (rows,)), _check_like("stats", stats, device, f32, (rows, 2)),
          _check_optional("entropy", entropy, device, f32, (rows,)),
          _check_optional("top_logprob", top_logprob, device, f32, (rows, top_k)),
          _check_optional("top_index", top_index, device, torch.int64, (rows, top_k)),
          top_k, rows, cols, temperature, _row_dtype(logits), _options(cluster_size, opts))


def launch_token_logprobs_backward(inputs, outputs, cluster_size: int = 0, opts=None, temperature: float = 1.0) -> None:
    """dlogits of sum(dlogprob * logprob) + sum(dentropy * entropy). inputs = (logits, targets, stats,
    entropy | None, dlogprob, dentropy | None), outputs = (dlogits,), which may be the logits themselves."""
    logits, targets, stats, entropy, dlogprob, dentropy = inputs
    (dlogits,) = outputs
    stride = _check_logits("logits", logits)
    rows, cols = logits.shape
    device, f32 = logits.device, torch.float32
    out_stride = _check_logits("dlogits", dlogits, device, logits.dtype, logits.shape)
    if dentropy is None:
        entropy = None
    elif entropy is None:
        raise ValueError("dentropy needs the entropy of the forward pass")
    _call(N.load().credit_token_logprobs_backward, device, logits.data_ptr() or None, stride,
          _check_like("targets", targets, device, torch.int64, (rows,)),
          _check_like("stats", stats, device, f32, (rows, 2)), _check_optional("entropy", entropy, device, f32, (rows,)),
          _check_like("dlogprob", dlogprob, device, f32, (rows,)),
          _check_optional("dentropy", dentropy, device, f32, (rows,)), dlogits.data_ptr() or None, out_stride, rows, cols,
          temperature, _row_dtype(logits), _options(cluster_size, opts))


def _teacher_size(index) -> int:
    if not isinstance(index, torch.Tensor) or index.dim() != 2:
        raise ValueError("teacher_index must be a tensor of two dimensions")
    return index.shape[1]


def launch_distill_topk_forward(inputs, outputs, cluster_size: int = 0, opts=None, temperature: float = 1.0,
                                tail: bool = True) -> None:
    """KL(teacher || softmax(logits / temperature)) per row, the teacher given by its top log probabilities.
    inputs = (logits [rows, cols], teacher_index int64 [rows, k], teacher_logprob [rows, k]), outputs =
    (loss [rows], stats [rows, 6]). `tail`: what the list leaves of 1 is one more outcome; otherwise
    the teacher is renormalised over its list. A negative index is an unused place."""
    logits, index, value = inputs
    loss, stats = outputs
    stride = _check_logits("logits", logits)
    rows, cols = logits.shape
    device, f32 = logits.device, torch.float32
    top_k = _teacher_size(index)
    _call(N.load().credit_distill_topk_forward, device, logits.data_ptr() or None, stride,
          _check_like("teacher_index", index, device, torch.int64, (rows, top_k)),
          _check_like("teacher_logprob", value, device, f32, (rows, top_k)), top_k,
          _check_like("loss", loss, device, f32, (rows,)), _check_like("stats", stats, device, f32, (rows, 6)),
          rows, cols, temperature, 1 if tail else 0, _row_dtype(logits), _options(cluster_size, opts))


def launch_distill_topk_backward(inputs, outputs, cluster_size: int = 0, opts=None, temperature: float = 1.0,
                                 tail: bool = True) -> None:
    """dlogits of sum(dloss * loss). inputs = (logits, teacher_index, teacher_logprob, stats, dloss), outputs =
    (dlogits,), which may be the logits themselves. `stats` says whether the forward call had a tail;
    `tail` is accepted for one signature with it."""
    logits, index, value, stats, dloss = inputs
    (dlogits,) = outputs
    stride = _check_logits("logits", logits)
    rows, cols = logits.shape
    device, f32 = logits.device, torch.float32
    out_stride = _check_logits("dlogits", dlogits, device, logits.dtype, logits.shape)
    top_k = _teacher_size(index)
    _call(N.load().credit_distill_topk_backward, device, logits.data_ptr() or None, stride,
          _check_like("teacher_index", index, device, torch.int64, (rows, top_k)),
          _check_like("teacher_logprob", value, device, f32, (rows, top_k)), top_k,
          _check_like("stats", stats, device, f32, (rows, 6)), _check_like("dloss", dloss, device, f32, (rows,)),
          dlogits.data_ptr() or None, out_stride, rows, cols, temperature, _row_dtype(logits),
          _options(cluster_size, opts))


# name -> (workload id, staged inputs, per-row input?, row-major outputs, per-row output?)
_ROW_OPS = {
    "weighted_var_backward": (N.WL_WEIGHTED_VAR_BACKWARD, 3, False, 1, False),
    "pearson_backward": (N.WL_PEARSON_BACKWARD, 2, True, 2, False),
    "softmax_logits_backward": (N.WL_SOFTMAX_LOGITS_BACKWARD, 2, False, 1, False),
    "lars_momentum": (N.WL_LARS_MOMENTUM, 3, False, 2, False),
    "rowwise_quant": (N.WL_ROWWISE_QUANT, 1, False, 1, True),
}


def _make_row_op_launcher(name: str):
    workload, nin, has_row_in, nout, has_row_out = _ROW_OPS[name]

    def launch(inputs, outputs, cluster_size: int = 0, opts=None) -> None:
        if len(inputs) != nin + int(has_row_in) or len(outputs) != nout + int(has_row_out):
            raise ValueError(f"{name}: expected {nin + int(has_row_in)} inputs and {nout + int(has_row_out)} outputs")
        x = inputs[0]
        _check_matrix("input 0", x, torch.float32)
        rows, cols = x.shape
        for i in range(1, nin):
            _check_matrix(f"input {i}", inputs[i], torch.float32, (rows, cols))
        row_in = None
        if has_row_in:      # the reference passes it as [rows, 1]
            row_in = inputs[nin]
            if row_in.numel() != rows:
                raise ValueError(f"{name}: the per-row input must have {rows} elements")
            _check_matrix("per-row input", row_in, torch.float32)
        out_dtype = torch.int8 if name == "rowwise_quant" else torch.float32
        for i in range(nout):
            _check_matrix(f"output {i}", outputs[i], out_dtype, (rows, cols))
        row_out = None
        if has_row_out:
            row_out = outputs[nout]
            _check_matrix("per-row output", row_out, torch.float32, (rows,))
        ptr = [t.data_ptr() if rows else None for t in inputs[:nin]] + [None] * (3 - nin)
        N.check(N.load().credit_row_op(
            workload, ptr[0], ptr[1], ptr[2], row_in.data_ptr() if has_row_in and rows else None,
            outputs[0].data_ptr() if rows else None, outputs[1].data_ptr() if nout > 1 and rows else None,
            row_out.data_ptr() if has_row_out and rows else None, rows, cols, _ref(_opts(cluster_size, opts)),
            _stream_ptr()))

    launch.__name__ = f"launch_{name}"
    launch.__doc__ = (f"{name} of the reference sweep (dsmem_eval/workloads.py), fp32, through credit_row_op; "
                      "same launcher convention as the others.")
    return launch


NATIVE_LAUNCHERS = {
    "rmsnorm_forward": launch_rmsnorm_forward,
    "row_reduce": launch_row_reduce,
    "layernorm_forward": launch_layernorm_forward,
    "layernorm_backward": launch_layernorm_backward,
    "layernorm_backward_stats": launch_layernorm_backward_stats,
    "ffn_forward": launch_ffn_forward,
    "residual_norm_forward": launch_residual_norm_forward,
    "residual_norm_backward": launch_residual_norm_backward,
    "token_logprobs_forward": launch_token_logprobs_forward,
    "token_logprobs_backward": launch_token_logprobs_backward,
    "distill_topk_forward": launch_distill_topk_forward,
    "distill_topk_backward": launch_distill_topk_backward,
    **{name: _make_row_op_launcher(name) for name in _ROW_OPS},
}


def allocate_outputs(name: str, inputs: tuple[torch.Tensor, ...], top_k: int = 0,
                     entropy: bool = True) -> tuple[torch.Tensor, ...]:
    """Output tensors for one call (reference: allocate_outputs, triton_kernels.py:403-414). `top_k` and
    `entropy` say which optional outputs token_logprobs_forward has; absent ones are None."""
    x = inputs[0]
    rows, cols = x.shape
    dev = x.device

    def fp32(*shape):
        return torch.empty(shape, device=dev, dtype=torch.float32)

    if name == "residual_norm_forward":
        return (torch.empty_like(x), torch.empty_like(x), None if inputs[2] is None else fp32(rows), fp32(rows))
    if name == "residual_norm_backward":
        return (torch.empty_like(x), torch.empty_like(x), None if inputs[4] is None else fp32(cols),
                None if inputs[5] is None else fp32(cols), fp32(cols))
    if name == "token_logprobs_forward":
        return (None if inputs[1] is None else fp32(rows), fp32(rows, 2), fp32(rows) if entropy else None,
                fp32(rows, top_k) if top_k else None,
                torch.empty((rows, top_k), device=dev, dtype=torch.int64) if top_k else None)
    if name == "distill_topk_forward":
        return (fp32(rows), fp32(rows, 6))
    if name in ("token_logprobs_backward", "distill_topk_backward"):
        # rows that start at the same place between two 16-byte boundaries as the logits' do, without their padding
        vec = 16 // x.element_size()
        stride = cols + (max(int(x.stride(0)), cols) - cols) % vec
        shift = x.data_ptr() % 16 // x.element_size()
        flat = torch.empty(shift + rows * stride, device=dev, dtype=x.dtype)
        return (flat[shift:].view(rows, stride)[:, :cols],)
    if name == "row_reduce":
        return (
            torch.empty(rows, device=dev, dtype=torch.float32),
            torch.empty(rows, device=dev, dtype=torch.float32),
            torch.empty(rows, device=dev, dtype=torch.int64),
        )
    if name == "layernorm_forward":
        return (
            torch.empty_like(x),
            torch.empty(rows, device=dev, dtype=torch.float32),
            torch.empty(rows, device=dev, dtype=torch.float32),
        )
    if name == "layernorm_backward_stats":
        return (
            torch.empty_like(x),
            torch.empty(cols, device=dev, dtype=torch.float32),
            torch.empty(cols, device=dev, dtype=torch.float32),
        )
    if name in ("rmsnorm_forward", "layernorm_backward", "ffn_forward", "weighted_var_backward",
                "softmax_logits_backward"):
        return (torch.empty_like(x),)
    if name in ("pearson_backward", "lars_momentum"):
        return (torch.empty_like(x), torch.empty_like(x))
    if name == "rowwise_quant":
        return (torch.empty(rows, cols, device=dev, dtype=torch.int8),
                torch.empty(rows, device=dev, dtype=torch.float32))
    raise KeyError(f"unknown workload {name!r}")
