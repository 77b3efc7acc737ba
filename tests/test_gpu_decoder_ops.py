"""residual_norm, token_logprobs and distill_topk on the GPU against the fp64 oracle
(`oracle/decoder_ops.py`), through the launcher table.

Tolerances count roundings, u = 2^-24 in fp32:
* a row sum of exponentials: ex2.approx 4 u relative, its argument up to 4 roundings of |d|, at most 64
  additions on any path (8 a chunk of each of four chains, chunks, warps, ranks): relative error
  (128 + 8 |d|) u, with |d| <= log n + entropy-weighted distances, taken as 8 log2 n;
* log probabilities and entropies: that, plus 8 roundings of each term that is added;
* gradients: the sum of the absolute terms ("magnitude", from the oracle) times (64 + 16 |log p| + 8 |log sum|) u,
  as the exponent of p is a difference of those two;
* the norms: sums of at most 16 + 32 + 16 + 16 additions, 100 u of the magnitude with the elementwise
  arithmetic, column sums (rows + 100) u;
* bf16 results: one rounding more, 2^-8 of the value.
Results below 2^-126 may be flushed to zero (the absolute 1e-37)."""
import math

import pytest
import torch

from credit_b200 import _native as N
from credit_b200 import launchers as L
from oracle import decoder_ops as D

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16]
NAN = float("nan")


def _within(got, want, tol, what=""):
    """|got - want| <= tol where want is finite; equal infinities and NaN elsewhere."""
    got, want = got.detach().cpu().double(), want.double()
    # beyond fp32's largest value and half a step, its infinities
    want = torch.where(want.abs() >= 2.0 ** 128 - 2.0 ** 103, want.sign() * math.inf, want)
    tol = torch.as_tensor(tol, dtype=torch.float64).expand_as(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    special = ~torch.isfinite(want)
    assert torch.equal(got[special].nan_to_num(nan=0.0), want[special].nan_to_num(nan=0.0)), what
    err = torch.where(special, torch.zeros_like(want), (got - want).abs())
    over = err - torch.where(special, torch.zeros_like(want), tol)
    assert not bool((over > 0).any()), f"{what}: {float(over.max()):.3e} above the tolerance at {int(over.argmax())}"


def _rounding(dtype, want):
    return want.abs().nan_to_num(0.0, 0.0, 0.0) * (2.0 ** -8 if dtype == torch.bfloat16 else 0.0) + 1e-37


def _launch(name, inputs, outputs, **kw):
    L.NATIVE_LAUNCHERS[name](inputs, outputs, **kw)
    torch.cuda.synchronize()


def _on_gpu(t, ld=None, shift=0):
    """A copy on the GPU: the leading columns of rows `ld` apart, `shift` elements behind an aligned address;
    everything around it holds NaN."""
    if t is None:
        return None
    if t.dim() != 2 or (ld is None and shift == 0):
        return t.to(DEV)
    rows, cols = t.shape
    ld = cols if ld is None else ld
    buffer = torch.full((rows * ld + shift + 64,), NAN, device=DEV, dtype=t.dtype)
    view = buffer[shift:shift + rows * ld].view(rows, ld)[:, :cols]
    view.copy_(t)
    return view


def _poisoned(outputs):
    for o in outputs:
        if o is not None:
            o.fill_(-77 if o.dtype == torch.int64 else NAN)
    return outputs


# --------------------------------------------------------------------------------------------
# norms around a block
# --------------------------------------------------------------------------------------------
def _norm_inputs(rows, cols, dtype, seed, post=True, gate=True):
    gen = torch.Generator().manual_seed(seed)
    block, residual = (torch.randn(rows, cols, generator=gen).to(dtype) for _ in range(2))
    weights = [torch.rand(cols, generator=gen) + 0.5 for _ in range(3)]
    return block, residual, weights[0] if post else None, weights[1] if gate else None, weights[2]


def _check_norm_forward(inputs, got, scale, eps, dtype):
    block, residual, post, gate, pre = inputs
    out, y, r1, r2 = D.residual_norm_forward(*inputs, scale, eps)
    n = (out - scale * residual.double()).abs()
    tol_out = 100 * U * ((scale * residual.double()).abs() + n)
    _within(got[0], out, tol_out + _rounding(dtype, out), "residual_out")
    rel = 100 * U * (1 + (tol_out.square().mean(-1) / out.square().mean(-1).clamp_min(1e-300)).sqrt() / (100 * U))
    _within(got[3], r2, rel * r2, "pre_rstd")
    tol_y = (tol_out + out.abs() * rel[:, None]) * r2[:, None] * pre.double().abs()
    _within(got[1], y, tol_y + _rounding(dtype, y), "y")
    if post is not None:
        _within(got[2], r1, 100 * U * r1, "post_rstd")


NORM_SHAPES = [(1, 1, 0), (3, 7, 0), (2, 64, 2), (5, 1000, 0), (4, 1024, 4), (300, 1024, 0), (3, 4099, 0), (2, 8192, 16),
               (2, 8200, 0), (3, 16384, 0), (2, 16392, 0), (2, 33333, 16), (1, 65536, 0), (700, 72, 0), (40, 9000, 0), (900, 5000, 2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,cluster", NORM_SHAPES)
@pytest.mark.parametrize("post,gate", [(True, True), (False, False)])
def test_residual_norm_forward(native_lib, dtype, rows, cols, cluster, post, gate):
    inputs = _norm_inputs(rows, cols, dtype, rows + cols, post, gate)
    ins = tuple(_on_gpu(t) for t in inputs)
    outs = _poisoned(L.allocate_outputs("residual_norm_forward", ins))
    _launch("residual_norm_forward", ins, outs, cluster_size=cluster, residual_scale=0.7, eps=1e-5)
    _check_norm_forward(inputs, outs, 0.7, 1e-5, dtype)
    assert N.device_status() == 0


def _norm_backward(inputs, saved, dy, dout, scale, cluster=0, shift=0, workspace=None):
    block, _, post, gate, pre = inputs
    out, r1, r2 = saved
    ins = tuple(_on_gpu(t, shift=shift) for t in (dy, dout, block, out, post, gate, pre, r1, r2))
    outs = _poisoned(L.allocate_outputs("residual_norm_backward", ins))
    _launch("residual_norm_backward", ins, outs, cluster_size=cluster, residual_scale=scale, workspace=workspace)
    want, mags = D.residual_norm_backward(dy, dout, block, out, post, gate, pre, r1, r2, scale)
    rows = dy.shape[0]
    for i, name in enumerate(("dblock", "dresidual", "dpost_weight", "dgate", "dpre_weight")):
        assert (outs[i] is None) == (want[i] is None)
        if want[i] is not None:
            tol = mags[i] * U * (100 if i < 2 else rows + 200)
            _within(outs[i], want[i], tol + (_rounding(dy.dtype, want[i]) if i < 2 else 1e-37), name)
    return outs


def _saved(inputs, dtype, scale=0.7, eps=1e-5):
    out, _, r1, r2 = D.residual_norm_forward(*inputs, scale, eps)
    return out.to(dtype), None if r1 is None else r1.float(), r2.float()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,cluster", NORM_SHAPES)
@pytest.mark.parametrize("post,gate,upstream", [(True, True, True), (True, False, False), (False, True, True),
                                                (False, False, True)])
def test_residual_norm_backward(native_lib, dtype, rows, cols, cluster, post, gate, upstream):
    inputs = _norm_inputs(rows, cols, dtype, rows + cols, post, gate)
    gen = torch.Generator().manual_seed(9)
    dy, dout = (torch.randn(rows, cols, generator=gen).to(dtype) for _ in range(2))
    _norm_backward(inputs, _saved(inputs, dtype), dy, dout if upstream else None, 0.7, cluster)
    assert N.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_residual_norm_unaligned_and_in_place(native_lib, dtype):
    rows, cols = 37, 2048
    inputs = _norm_inputs(rows, cols, dtype, 5)
    ins = tuple(_on_gpu(t, shift=1) for t in inputs)              # rows off the 16-byte boundary
    outs = _poisoned(L.allocate_outputs("residual_norm_forward", ins))
    _launch("residual_norm_forward", ins, outs, residual_scale=0.7, eps=1e-5)
    _check_norm_forward(inputs, outs, 0.7, 1e-5, dtype)
    for cluster in (1, 4):                                          # the sum in the residual's place, y in the block's
        ins = tuple(_on_gpu(t) for t in inputs)
        fresh = L.allocate_outputs("residual_norm_forward", ins)
        outs = (ins[1], ins[0], fresh[2], fresh[3])
        _launch("residual_norm_forward", ins, outs, cluster_size=cluster, residual_scale=0.7, eps=1e-5)
        _check_norm_forward(inputs, outs, 0.7, 1e-5, dtype)
    gen = torch.Generator().manual_seed(6)
    dy, dout = (torch.randn(rows, cols, generator=gen).to(dtype) for _ in range(2))
    saved = _saved(inputs, dtype)
    _norm_backward(inputs, saved, dy, dout, 0.7, shift=1)
    block, _, post, gate, pre = inputs
    for cluster in (1, 4):
        ins = tuple(_on_gpu(t) for t in (dy, dout, block, saved[0], post, gate, pre, saved[1], saved[2]))
        want = L.allocate_outputs("residual_norm_backward", ins)
        _launch("residual_norm_backward", ins, want, cluster_size=cluster, residual_scale=0.7)
        outs = (ins[2], ins[1], *L.allocate_outputs("residual_norm_backward", ins)[2:])   # in place
        _launch("residual_norm_backward", ins, outs, cluster_size=cluster, residual_scale=0.7)
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_residual_norm_rows_of_zero(native_lib):
    rows, cols = 3, 512
    inputs = list(_norm_inputs(rows, cols, torch.float32, 8))
    inputs[0][1] = 0.0
    inputs[0][2] = inputs[1][2] = 0.0
    ins = tuple(_on_gpu(t) for t in inputs)
    outs = _poisoned(L.allocate_outputs("residual_norm_forward", ins))
    _launch("residual_norm_forward", ins, outs, residual_scale=0.7, eps=1e-5)
    _check_norm_forward(inputs, outs, 0.7, 1e-5, torch.float32)
    assert float(outs[1][2].abs().max()) == 0.0


def test_residual_norm_no_rows(native_lib):
    ins = tuple(_on_gpu(t) for t in _norm_inputs(0, 256, torch.float32, 1))
    L.launch_residual_norm_forward(ins, L.allocate_outputs("residual_norm_forward", ins))
    e = ins[0]
    bwd = (e, None, e, e, ins[2], ins[3], ins[4], torch.empty(0, device=DEV), torch.empty(0, device=DEV))
    outs = _poisoned(L.allocate_outputs("residual_norm_backward", bwd))
    _launch("residual_norm_backward", bwd, outs)
    for o in outs[2:]:
        assert float(o.abs().max()) == 0.0


def test_residual_norm_gradient_against_differences(native_lib):
    """The kernels' gradient against central differences of the kernels' forward, fp32. Rounding of the forward
    outputs (sum of 2 * 3 * 64 values of order 1, 100 u each) over 2 h = 0.02 and h^2 times third derivatives of
    order 10: 384 * 100 * u / 0.02 + 1e-3 < 0.12 in the worst case; the observed scale is far below it, entries are
    of order 1."""
    rows, cols, h = 3, 64, 0.01
    inputs = _norm_inputs(rows, cols, torch.float32, 12)
    gen = torch.Generator().manual_seed(13)
    dy, dout = torch.randn(rows, cols, generator=gen), torch.randn(rows, cols, generator=gen)

    def forward(ins):
        outs = L.allocate_outputs("residual_norm_forward", ins)
        L.launch_residual_norm_forward(ins, outs, residual_scale=0.7, eps=1e-5)
        return outs

    def loss(ins):
        outs = forward(ins)
        return float((outs[0].double().cpu() * dout).sum() + (outs[1].double().cpu() * dy).sum())

    ins = [t.to(DEV) for t in inputs]
    out, _, r1, r2 = forward(tuple(ins))
    bwd = (dy.to(DEV), dout.to(DEV), ins[0], out, ins[2], ins[3], ins[4], r1, r2)
    outs = L.allocate_outputs("residual_norm_backward", bwd)
    _launch("residual_norm_backward", bwd, outs, residual_scale=0.7)
    for which, grad in ((0, outs[0]), (1, outs[1]), (2, outs[2]), (3, outs[3]), (4, outs[4])):
        flat = ins[which].view(-1)
        for i in (0, flat.numel() // 2, flat.numel() - 1):
            keep = float(flat[i])
            flat[i] = keep + h
            up = loss(tuple(ins))
            flat[i] = keep - h
            down = loss(tuple(ins))
            flat[i] = keep
            assert abs((up - down) / (2 * h) - float(grad.view(-1)[i])) < 0.12


# --------------------------------------------------------------------------------------------
# log probabilities
# --------------------------------------------------------------------------------------------
def _logits(rows, cols, dtype, seed, masked=0.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=gen) * 3.0
    for r in range(rows):
        x[r, int(torch.randint(0, cols, (1,), generator=gen))] = 9.0
    if masked:
        x[torch.rand(rows, cols, generator=gen) < masked] = -math.inf
    targets = torch.randint(0, cols, (rows,), generator=gen)
    return x.to(dtype), targets


def _check_logprobs(x, targets, got, temperature, top_k):
    logprob, stats, entropy, top_logprob, top_index = got
    cols = x.shape[1]
    want = D.token_logprobs_forward(x, targets, temperature, top_k)
    log_n = math.log2(max(cols, 2))
    e_sum = (128 + 64 * log_n) * U           # relative error of the sum = absolute error of its logarithm

    def tol(lp):
        size = lp.abs().nan_to_num(0.0, 0.0, 0.0)
        return e_sum + 8 * U * (size + 2 * log_n)
    if targets is not None:
        _within(logprob, want[0], tol(want[0]), "logprob")
    _within(stats[:, 0], want[1][:, 0], 0.0, "max")
    _within(stats[:, 1], want[1][:, 1], e_sum + 8 * U * log_n, "log sum")
    if entropy is not None:
        _within(entropy, want[2], e_sum * (2 + log_n) + 8 * U * log_n, "entropy")
    if top_k:
        assert torch.equal(top_index.cpu(), want[4])
        _within(top_logprob, want[3], tol(want[3]), "top_logprob")


def _run_logprobs(x, targets, top_k=0, temperature=1.0, cluster=0, ld=None, shift=0, entropy=True):
    ins = (_on_gpu(x, ld, shift), _on_gpu(targets))
    outs = _poisoned(L.allocate_outputs("token_logprobs_forward", ins, top_k=top_k, entropy=entropy))
    _launch("token_logprobs_forward", ins, outs, cluster_size=cluster, temperature=temperature)
    return outs


LOGIT_SHAPES = [(1, 1, None, 0), (3, 2, None, 0), (2, 7, 9, 3), (5, 255, None, 1), (4, 257, 320, 0), (3, 1000, 1024, 8),
                (2, 4099, None, 5), (3, 8192, None, 0), (2, 8200, 8260, 1), (2, 50001, None, 0), (2, 131072, None, 0),
                (1, 262147, 262400, 7), (300, 520, None, 0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,ld,shift", LOGIT_SHAPES)
@pytest.mark.parametrize("cluster,top_k", [(0, 0), (0, 5), (1, 20), (2, 0), (4, 1), (16, 128)])
def test_token_logprobs_forward(native_lib, dtype, rows, cols, ld, shift, cluster, top_k):
    x, targets = _logits(rows, cols, dtype, rows + cols)
    _check_logprobs(x, targets, _run_logprobs(x, targets, top_k, 0.8, cluster, ld, shift), 0.8, top_k)
    assert N.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cluster", [1, 8])
def test_token_logprobs_masks_and_special_values(native_lib, dtype, cluster):
    cols = 9000
    lowest = torch.finfo(dtype).min
    x, targets = _logits(14, cols, dtype, 2, masked=0.5)
    x[0] = -math.inf                                       # nothing left
    x[1, :-1] = -math.inf                                  # one left, in the last place
    x[2] = lowest                                          # the lowest value as a mask, everywhere
    x[3] = lowest                                          # and with a few tokens left
    x[3, [5, 4000, 8999]] = torch.tensor([1.0, 2.0, 1.0], dtype=dtype)
    x[4] = 0.0                                             # all equal: columns in order
    x[5] = -0.0
    x[5, ::2] = 0.0                                        # signed zeros are equal
    x[6, 17] = NAN
    x[7, 17] = math.inf
    x[8, [3, 8000]] = NAN
    x[8, 20] = math.inf
    x[9] = torch.arange(cols).to(dtype)                    # ascending: every element is a candidate
    x[10] = torch.arange(cols).flip(0).to(dtype)
    x[11] = (torch.arange(cols) % 3).to(dtype)             # thousands of ties at the top
    x[12, :] = -math.inf
    x[12, 100:103] = torch.tensor([-5.0, -5.0, 2.0], dtype=dtype)   # fewer left than asked for
    x[13] = 30000.0 + torch.arange(cols).to(dtype) % 7     # far from zero
    targets[3], targets[12] = 4000, 101
    for top_k in (0, 3, 64, 128):
        _check_logprobs(x, targets, _run_logprobs(x, targets, top_k, 1.0, cluster), 1.0, top_k)
    assert N.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_top_alternatives_of_sorted_and_constant_wide_rows(native_lib, dtype):
    """Rows that bring more candidates than the buffer holds, over many chunks."""
    cols = 100000
    x = torch.zeros(4, cols, dtype=dtype)
    x[0] = torch.linspace(-8, 8, cols).to(dtype)
    x[1] = 2.5
    x[2] = torch.linspace(-8, 8, cols).to(dtype)
    x[2, 50000:] = -math.inf
    x[3] = torch.linspace(8, -8, cols).to(dtype)
    for cluster in (1, 2):
        for top_k in (7, 128):
            _check_logprobs(x, None, _run_logprobs(x, None, top_k, 1.0, cluster), 1.0, top_k)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows_with_masks_and_special_values(native_lib, dtype):
    """More rows than are resident at once, of every kind next to one another."""
    rows, cols = 900, 9001
    x, targets = _logits(rows, cols, dtype, 50)
    x[1::9] = -math.inf
    x[2::9, 100:] = -math.inf
    x[3::9] = torch.finfo(dtype).min
    x[4::9, 17] = NAN
    x[5::9, 8000] = math.inf
    x[6::9] = torch.arange(cols).to(dtype)
    x[7::9] = 1.5
    targets[8::9] = -1
    x[8::18] = NAN
    clean = x.clone()
    clean[targets < 0] = 0.0
    for top_k in (0, 20):
        _check_logprobs(clean, targets, _run_logprobs(x, targets, top_k), 1.0, top_k)
    assert N.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,ld,shift", [(1184, 1, None, 0), (1300, 37, 40, 1), (1300, 4099, None, 5),
                                                (1201, 8200, 8260, 1), (1500, 1031, None, 0)])
@pytest.mark.parametrize("entropy", [True, False])
def test_as_many_rows_as_fill_the_device(native_lib, dtype, rows, cols, ld, shift, entropy):
    """Rows of every kind next to one another, without alternatives, at lengths below and above a CTA's chunk."""
    _check_mixed_rows(dtype, rows, cols, ld, shift, entropy, 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,ld,shift,top_k", [(1184, 1, None, 0, 3), (1300, 37, 40, 1, 32), (1300, 4099, None, 5, 20),
                                                      (1201, 8200, 8260, 1, 31), (1190, 9001, None, 0, 33), (1500, 1031, None, 0, 1)])
def test_alternatives_of_as_many_rows_as_fill_the_device(native_lib, dtype, rows, cols, ld, shift, top_k):
    _check_mixed_rows(dtype, rows, cols, ld, shift, True, top_k)


def _check_mixed_rows(dtype, rows, cols, ld, shift, entropy, top_k):
    x, targets = _logits(rows, cols, dtype, rows + cols)
    x[1::9] = -math.inf
    x[2::9, cols // 3 + 1:] = -math.inf
    x[3::9] = torch.finfo(dtype).min
    x[4::9, cols // 2] = NAN
    x[5::9, cols - 1] = math.inf
    x[6::9] = torch.arange(cols).to(dtype)
    x[7::9] = 1.5
    targets[8::9] = -1
    x[8::18] = NAN
    clean = x.clone()
    clean[targets < 0] = 0.0
    _check_logprobs(clean, targets, _run_logprobs(x, targets, top_k, 0.8, 0, ld, shift, entropy), 0.8, top_k)
    assert N.device_status() == 0


def _far_rows(dtype, cols, seed):
    """Rows far from zero: log2(e) times their maximum is large, near 2^24, or beyond fp32's resolution of 1."""
    x, targets = _logits(10, cols, torch.float32, seed)
    x[0] = -1e9                     # a finite mask that leaves nothing
    x[1] = -1e10
    x[2] = -1e20
    x[3] += 1e10
    x[4, cols // 2:] = -1e10
    step = torch.arange(cols) % 24  # maxima on both sides of 2^24 / log2(e)
    x[5] = 11629068.0 + step
    x[6] = -11629090.0 + step
    x[7] = 11629068.0 + 24.0 * torch.arange(cols) / cols
    x[8] = 3e38
    x[9] = 1e25 * torch.arange(cols)
    return x.to(dtype), targets


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols,cluster,top_k", [(9001, 1, 0), (9001, 4, 0), (9001, 1, 12), (257, 0, 3)])
def test_token_logprobs_rows_far_from_zero(native_lib, dtype, cols, cluster, top_k):
    x, targets = _far_rows(dtype, cols, 90)
    _check_logprobs(x, targets, _run_logprobs(x, targets, top_k, 1.0, cluster), 1.0, top_k)
    assert N.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [1e-12, 1e-9, 1e-6, 1e6, 1e12, 1e22])
def test_token_logprobs_extreme_temperatures(native_lib, dtype, temperature):
    """Logits on the temperature's own scale, some masked, and (near greedy) on the ordinary one."""
    x, targets = _logits(6, 5003, torch.float32, 91)
    x[:4] *= temperature
    x = x.to(dtype)
    x[1::2, 7::3] = -math.inf
    x[3, :] = torch.where(x[3] < 0, torch.finfo(dtype).min, x[3].double()).to(dtype)
    for cluster in (1, 4):
        _check_logprobs(x, targets, _run_logprobs(x, targets, 5, temperature, cluster), temperature, 5)
    _check_logprob_gradient(x[:4], targets[:4], temperature, True)
    assert N.device_status() == 0


def test_token_logprobs_ignored_and_bad_targets(native_lib):
    x, targets = _logits(5, 700, torch.float32, 3)
    targets[1], targets[4] = -1, -100
    x[1] = NAN                                              # not read
    _check_logprobs(x.nan_to_num(0.0), targets, _run_logprobs(x, targets, 4), 1.0, 4)
    assert N.device_status() == 0
    targets[2] = 700
    outs = _run_logprobs(x, targets, 4)
    assert N.device_status() == N.STATUS_BAD_INDEX and math.isnan(float(outs[0][2]))
    _check_logprobs(x.nan_to_num(0.0), targets, outs, 1.0, 4)
    assert N.device_status() == 0


def test_token_logprobs_optional_outputs_agree(native_lib):
    x, targets = _logits(6, 3000, torch.bfloat16, 4)
    full = _run_logprobs(x, targets, 9)
    alone = _run_logprobs(x, targets, 0, entropy=False)
    assert torch.equal(full[0], alone[0]) and torch.equal(full[1], alone[1])
    listed = _run_logprobs(x, None, 9, entropy=False)
    assert torch.equal(full[3], listed[3]) and torch.equal(full[4], listed[4])
    again = _run_logprobs(x, targets, 9)
    for a, b in zip(full, again):
        assert torch.equal(a, b)


def _check_logprob_gradient(x, targets, temperature, use_entropy, ld=None, shift=0, out_ld=None, out_shift=None,
                            in_place=False, seed=1):
    gen = torch.Generator().manual_seed(seed)
    rows, cols = x.shape
    clean = x.clone()
    clean[targets < 0] = 0.0
    _, stats, entropy, _, _ = (None if t is None else t.float() for t in
                               D.token_logprobs_forward(clean, targets, temperature))
    g, gh = torch.randn(rows, generator=gen), torch.randn(rows, generator=gen)
    logits = _on_gpu(x, ld, shift)
    ins = (logits, *(t.to(DEV) for t in (targets, stats, entropy, g)), gh.to(DEV) if use_entropy else None)
    out = logits
    if not in_place:
        out = _on_gpu(torch.full((rows, cols), NAN, dtype=x.dtype), out_ld or ld, shift if out_shift is None else out_shift)
    _launch("token_logprobs_backward", ins, (out,), temperature=temperature)
    want, mag, logp = D.token_logprobs_backward(clean, targets, stats, entropy, g, gh if use_entropy else None, temperature)
    finite = logp.abs().nan_to_num(0.0, 0.0, 0.0)
    tol = mag * U * (64 + 16 * finite + 8 * stats[:, 1:].abs().nan_to_num(0.0))
    _within(out, want, tol.nan_to_num(0.0) + _rounding(x.dtype, want), "dlogits")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,ld,shift", LOGIT_SHAPES)
@pytest.mark.parametrize("use_entropy", [True, False])
def test_token_logprobs_backward(native_lib, dtype, rows, cols, ld, shift, use_entropy):
    x, targets = _logits(rows, cols, dtype, rows + cols)
    _check_logprob_gradient(x, targets, 0.8, use_entropy, ld, shift)
    _check_logprob_gradient(x, targets, 0.8, use_entropy, ld, shift, in_place=True)
    # another stride and phase for the gradient: the scalar path
    _check_logprob_gradient(x, targets, 0.8, use_entropy, ld, shift, out_ld=(ld or cols) + 3, out_shift=shift + 1)
    assert N.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("use_entropy", [True, False])
def test_token_logprobs_backward_masks_and_special_values(native_lib, dtype, use_entropy):
    cols = 5000
    x, targets = _logits(9, cols, dtype, 7, masked=0.3)
    x[0] = -math.inf
    x[1] = NAN
    targets[1] = -1
    x[2, 9] = NAN
    x[3, 9] = math.inf
    x[4] = torch.finfo(dtype).min
    x[5] = -math.inf
    x[5, 77] = 3.0                                         # p = 1 at the target: gradient 0
    targets[5] = 77
    x[6, 11] = 40.0                                        # p close to 1: 1 - p without cancellation
    targets[6] = 11
    _check_logprob_gradient(x, targets, 1.0, use_entropy)
    assert N.device_status() == 0
    targets[8] = cols + 5
    _check_logprob_gradient(x, targets, 1.0, use_entropy)
    assert N.device_status() == N.STATUS_BAD_INDEX


# --------------------------------------------------------------------------------------------
# distillation
# --------------------------------------------------------------------------------------------
def _teacher(x, k, seed, kept=0.9):
    gen = torch.Generator().manual_seed(seed)
    rows, cols = x.shape
    index = torch.stack([torch.randperm(cols, generator=gen)[:k] if k <= cols else
                         torch.cat([torch.randperm(cols, generator=gen), torch.full((k - cols,), -1)]) for _ in range(rows)])
    logprob = torch.log_softmax(torch.randn(rows, k, generator=gen) * 2.0, -1) + math.log(kept)
    return index, logprob


def _check_distill(x, index, logprob, temperature, tail, cluster=0, ld=None, shift=0, out_ld=None, out_shift=None,
                   in_place=False):
    rows, cols = x.shape
    logits = _on_gpu(x, ld, shift)
    ins = (logits, index.to(DEV), logprob.to(DEV))
    outs = _poisoned(L.allocate_outputs("distill_topk_forward", ins))
    _launch("distill_topk_forward", ins, outs, cluster_size=cluster, temperature=temperature, tail=tail)
    loss, stats = D.distill_topk_forward(x, index, logprob, temperature, tail)
    log_n = math.log2(max(cols, 2))
    e_sum = (128 + 64 * log_n) * U
    m, ls, m2, ls2, norm, rest = stats.unbind(-1)
    broken = torch.isnan(m)
    good = ~broken
    for i, tol in ((0, 0.0), (1, e_sum + 8 * U * log_n), (2, 0.0), (3, e_sum + 8 * U * log_n), (4, 4 * U * (1 + norm.abs())),
                   (5, 2 * U * rest)):
        keep = torch.as_tensor(tol).expand(rows)[good]
        _within(outs[1][:, i].cpu()[good], stats[good, i], keep, f"stats[{i}]")
    _within(outs[1][:, 0], stats[:, 0], 0.0, "stats[0]")
    # each entry: weight (8 u) times log weight and log q (its own roundings, and the logarithms' of the sums)
    w = torch.where((index >= 0) & (index < cols), (logprob.double() - norm[:, None]).exp(), 0.0).nan_to_num(0.0)
    logq = ((x.double().gather(1, index.clamp(0, cols - 1)) - m[:, None]) / temperature - ls[:, None])
    size = (logprob.double() - norm[:, None]).abs() + logq.abs() + 4 * log_n
    tol = (torch.where(w > 0, w * size, 0.0)).nan_to_num(0.0, 0.0, 0.0).sum(-1) * 24 * U + 3 * e_sum
    tail_size = (torch.log(rest).abs() + ((m2 - m) / temperature + ls2 - ls).abs()).nan_to_num(0.0, 0.0, 0.0)
    _within(outs[0], loss, tol + rest * tail_size * 24 * U, "loss")

    gen = torch.Generator().manual_seed(3)
    dloss = torch.randn(rows, generator=gen)
    saved = stats.float()
    out = logits
    if not in_place:
        out = _on_gpu(torch.full((rows, cols), NAN, dtype=x.dtype), out_ld or ld, shift if out_shift is None else out_shift)
    _launch("distill_topk_backward", (*ins, saved.to(DEV), dloss.to(DEV)), (out,), temperature=temperature, tail=tail)
    want, mag = D.distill_topk_backward(x, index, logprob, saved, dloss, temperature)
    far = ((x.double() - m[:, None]).abs() / temperature).nan_to_num(0.0, 0.0, 0.0) + \
        ((x.double() - m2[:, None]).abs() / temperature).nan_to_num(0.0, 0.0, 0.0)
    extra = (ls.abs() + ls2.abs() + norm.abs()).nan_to_num(0.0)[:, None] + \
        ((m - m2).abs() / temperature).nan_to_num(0.0, 0.0, 0.0)[:, None]
    _within(out, want, (mag * U * (64 + 16 * far + 16 * extra)).nan_to_num(0.0) + _rounding(x.dtype, want), "dlogits")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,ld,shift", LOGIT_SHAPES)
@pytest.mark.parametrize("cluster,k,tail", [(0, 20, True), (0, 20, False), (1, 1, True), (2, 33, True), (16, 128, False),
                                            (16, 128, True)])
def test_distill_topk(native_lib, dtype, rows, cols, ld, shift, cluster, k, tail):
    x, _ = _logits(rows, cols, dtype, rows + cols)
    index, logprob = _teacher(x, k, 5)
    _check_distill(x, index, logprob, 1.3, tail, cluster, ld, shift)
    _check_distill(x, index, logprob, 1.3, tail, cluster, ld, shift, in_place=True)
    _check_distill(x, index, logprob, 1.3, tail, cluster, ld, shift, out_ld=(ld or cols) + 3, out_shift=shift + 1)
    assert N.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("cluster", [1, 4])
def test_distill_lists_and_masks(native_lib, dtype, tail, cluster):
    cols, k = 6000, 8
    x, _ = _logits(14, cols, dtype, 11)
    index, logprob = _teacher(x, k, 12)
    index[0] = -1                                          # no teacher
    index[1, 2:] = -1                                      # two places used
    index[2, 5] = index[2, 1]                              # a column three times
    index[2, 7] = index[2, 1]
    index[3, :] = index[3, 0]                              # one column only
    logprob[4] = -math.inf                                 # a list without mass
    logprob[5, 3] = -math.inf
    logprob[6] = logprob[6] + 0.5                          # a list of more than 1
    x[7] = -math.inf                                       # nothing left
    x[8, int(index[8, 0])] = -math.inf                     # teacher mass on a masked column: loss +inf
    keep = x[9, index[9]].clone()
    x[9] = -math.inf
    x[9, index[9]] = keep                                  # nothing left outside the list
    x[10, index[10]] = 60.0                                # the student's tail has mass e^-50
    x[11, 5] = NAN
    x[12, 5] = math.inf
    x[13] = torch.finfo(dtype).min
    _check_distill(x, index, logprob, 1.0, tail, cluster)
    assert N.device_status() == 0


@pytest.mark.parametrize("tail", [True, False])
def test_distill_many_rows(native_lib, tail):
    """Rows that one CTA each takes, lists and masks of every kind next to one another."""
    rows, cols, k = 700, 9001, 8
    x, _ = _logits(rows, cols, torch.bfloat16, 51)
    index, logprob = _teacher(x, k, 52)
    index[1::11] = -1
    index[2::11, 5] = index[2::11, 1]
    index[2::11, 7] = index[2::11, 1]
    index[3::11, :] = index[3::11, :1]
    logprob[4::11] = -math.inf
    logprob[5::11] = logprob[5::11] + 0.5
    x[6::11] = -math.inf
    for r in range(7, rows, 11):
        keep = x[r, index[r]].clone()
        x[r] = -math.inf
        x[r, index[r]] = keep
    x[8::11, 5] = NAN
    x[9::11, cols - 1] = math.inf
    _check_distill(x, index, logprob, 1.0, tail)
    assert N.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("cluster", [1, 4])
def test_distill_rows_far_from_zero(native_lib, dtype, tail, cluster):
    x, _ = _far_rows(dtype, 9001, 92)
    index, logprob = _teacher(_logits(10, 9001, torch.float32, 93)[0], 8, 94)
    _check_distill(x, index, logprob, 1.0, tail, cluster)
    x, _ = _logits(4, 5003, torch.float32, 95)
    x[1::2, 7::3] = -math.inf
    index, logprob = _teacher(x, 8, 96)
    for temperature in (1e-9, 1e12):
        _check_distill((x * temperature).to(dtype), index, logprob, temperature, tail, cluster)
    assert N.device_status() == 0


def test_distill_bad_index(native_lib):
    x, _ = _logits(4, 500, torch.float32, 13)
    index, logprob = _teacher(x, 6, 14)
    index[2, 3] = 500
    for tail in (True, False):
        _check_distill(x, index, logprob, 1.0, tail)
        assert N.device_status() == N.STATUS_BAD_INDEX
    index[2, 3] = -(1 << 32) + 5                           # negative, whatever its low bits say
    _check_distill(x, index, logprob, 1.0, True)
    assert N.device_status() == 0


def test_distill_gradient_against_differences(native_lib):
    """Kernel gradient against central differences of the kernel's loss, fp32: rounding 2e-6 over 2 h = 0.1 and
    h^2 / 6 times third derivatives below 1: 5e-4."""
    rows, cols, h = 2, 40, 0.05
    x, _ = _logits(rows, cols, torch.float32, 15)
    index, logprob = _teacher(x, 6, 16)
    dev = (index.to(DEV), logprob.to(DEV))

    def forward(v):
        outs = L.allocate_outputs("distill_topk_forward", (v, *dev))
        L.launch_distill_topk_forward((v, *dev), outs)
        return outs

    v = x.to(DEV)
    _, stats = forward(v)
    (grad,) = L.allocate_outputs("distill_topk_backward", (v,))
    _launch("distill_topk_backward", (v, *dev, stats, torch.ones(rows, device=DEV)), (grad,))
    for r in range(rows):
        for c in (0, int(index[r, 0]), 17, cols - 1):
            keep = float(v[r, c])
            v[r, c] = keep + h
            up = float(forward(v)[0][r])
            v[r, c] = keep - h
            down = float(forward(v)[0][r])
            v[r, c] = keep
            assert abs((up - down) / (2 * h) - float(grad[r, c])) < 5e-4


# --------------------------------------------------------------------------------------------
# together, captured, on other streams
# --------------------------------------------------------------------------------------------
class _Step:
    """The end of a training step: join + norm, head product, log probabilities and distillation, and back
    to the block and the residual. Buffers are allocated once, as a training loop keeps them."""

    def __init__(self, rows, cols, vocab, dtype, seed):
        gen = torch.Generator().manual_seed(seed)
        self.host = _norm_inputs(rows, cols, dtype, seed)
        self.ins = tuple(t.to(DEV) for t in self.host)
        self.head = (torch.randn(vocab, cols, generator=gen) / cols ** 0.5 * 2).to(dtype).to(DEV)
        self.targets = torch.randint(0, vocab, (rows,), generator=gen).to(DEV)
        self.targets[1] = -1
        self.teacher = torch.randn(rows, vocab, generator=gen).to(dtype).to(DEV)
        self.g, self.gh, self.gd = (torch.randn(rows, generator=gen).to(DEV) for _ in range(3))
        self.norm = L.allocate_outputs("residual_norm_forward", self.ins)
        self.logits = torch.empty(rows, vocab, device=DEV, dtype=dtype)
        self.lp = L.allocate_outputs("token_logprobs_forward", (self.logits, self.targets))
        self.listed = L.allocate_outputs("token_logprobs_forward", (self.teacher, None), top_k=16, entropy=False)
        self.kd = L.allocate_outputs("distill_topk_forward", (self.logits,))
        (self.d1,) = L.allocate_outputs("token_logprobs_backward", (self.logits,))
        (self.d2,) = L.allocate_outputs("distill_topk_backward", (self.logits,))
        self.dy = torch.empty_like(self.ins[0])
        self.back_in = (self.dy, None, self.ins[0], self.norm[0], *self.ins[2:], self.norm[2], self.norm[3])
        self.back = L.allocate_outputs("residual_norm_backward", self.back_in)
        need = L.residual_norm_backward_workspace_bytes(rows, cols, dtype)
        self.workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)

    def __call__(self):
        t = L.NATIVE_LAUNCHERS
        t["residual_norm_forward"](self.ins, self.norm, residual_scale=0.9)
        torch.matmul(self.norm[1], self.head.T, out=self.logits)
        t["token_logprobs_forward"]((self.logits, self.targets), self.lp, temperature=0.8)
        t["token_logprobs_forward"]((self.teacher, None), self.listed)
        lists = (self.listed[4], self.listed[3])
        t["distill_topk_forward"]((self.logits, *lists), self.kd)
        t["token_logprobs_backward"]((self.logits, self.targets, self.lp[1], self.lp[2], self.g, self.gh), (self.d1,),
                                     temperature=0.8)
        t["distill_topk_backward"]((self.logits, *lists, self.kd[1], self.gd), (self.d2,))
        torch.matmul(self.d1 + self.d2, self.head, out=self.dy)
        t["residual_norm_backward"](self.back_in, self.back, residual_scale=0.9, workspace=self.workspace)

    def results(self):
        return [o for o in (*self.norm, *self.lp, *self.listed, *self.kd, self.d1, self.d2, *self.back) if o is not None]


def test_end_of_a_training_step(native_lib):
    rows, cols, vocab = 12, 512, 3001
    step = _Step(rows, cols, vocab, torch.float32, 21)
    step()
    torch.cuda.synchronize()
    assert N.device_status() == 0
    # the same chain in fp64 by autograd over the oracle's forward formulas
    leaves = [t.double().requires_grad_() for t in step.host]
    out, y, _, _ = D.residual_norm_forward(*leaves, 0.9)
    z = y @ step.head.cpu().double().T
    targets = step.targets.cpu()
    logp = torch.log_softmax(z / 0.8, -1)
    used = (targets >= 0).double()
    lp = logp.gather(1, targets.clamp(min=0)[:, None])[:, 0] * used
    entropy = -(logp.exp() * logp).sum(-1) * used
    index, listed = step.listed[4].cpu(), step.listed[3].cpu().double()
    logq = torch.log_softmax(z, -1)
    rest = 1.0 - listed.exp().sum(-1)
    outside = torch.logsumexp(logq.scatter(1, index, -math.inf), -1)
    kd = (listed.exp() * (listed - logq.gather(1, index))).sum(-1) + rest * (rest.log() - outside)
    (lp @ step.g.cpu().double() + entropy @ step.gh.cpu().double() + kd @ step.gd.cpu().double()).backward()
    # fp32 through a product of 512 terms of order 1 (about 512 u) and logits of order 5 in the exponents
    for got, want in ((step.lp[0], lp), (step.lp[2], entropy), (step.kd[0], kd)):
        assert float((got.cpu().double() - want.detach()).abs().max()) < 2e-3
    for got, leaf in zip(step.back, leaves):
        scale = float(leaf.grad.abs().max())
        assert float((got.cpu().double() - leaf.grad).abs().max()) < 2e-3 * scale


@pytest.mark.parametrize("dtype", TYPES)
def test_captured_step_replays_on_new_inputs(native_lib, dtype):
    step, other = _Step(9, 256, 2500, dtype, 22), _Step(9, 256, 2500, dtype, 23)
    step()
    other()
    torch.cuda.synchronize()
    want = [o.clone() for o in other.results()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for mine, theirs in zip((*step.ins, step.head, step.targets, step.teacher, step.g, step.gh, step.gd),
                            (*other.ins, other.head, other.targets, other.teacher, other.g, other.gh, other.gd)):
        mine.copy_(theirs)
    for o in step.results():
        o.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(step.results(), want):
        assert torch.equal(a, b)
    assert N.device_status() == 0


def test_two_streams_at_once(native_lib):
    steps = [_Step(64, 512, 9000, torch.bfloat16, 30 + i) for i in range(2)]
    want = []
    for s in steps:
        s()
        torch.cuda.synchronize()
        want.append([o.clone() for o in s.results()])
    streams = [torch.cuda.Stream() for _ in steps]
    for o in (o for s in steps for o in s.results()):
        o.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        for s, stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                s()
    torch.cuda.synchronize()
    for s, w in zip(steps, want):
        for a, b in zip(s.results(), w):
            assert torch.equal(a, b)


def test_bytes_around_the_logits_stay(native_lib):
    """Padding columns and the memory around the gradient are not written."""
    rows, cols, ld = 5, 1003, 1024
    for dtype in TYPES:
        buffer = torch.full((rows + 2, ld), 7.0, device=DEV, dtype=dtype)
        out = buffer[1:-1, :cols]
        x, targets = _logits(rows, cols, dtype, 40)
        logits = _on_gpu(x, ld)
        index, logprob = _teacher(x, 10, 41)
        _, stats, _, _, _ = D.token_logprobs_forward(x, targets)
        _launch("token_logprobs_backward", (logits, targets.to(DEV), stats.float().to(DEV), None,
                                            torch.ones(rows, device=DEV), None), (out,))
        _, saved = D.distill_topk_forward(x, index, logprob)
        _launch("distill_topk_backward", (logits, index.to(DEV), logprob.to(DEV), saved.float().to(DEV),
                                          torch.ones(rows, device=DEV)), (out,))
        assert bool((buffer[0] == 7).all()) and bool((buffer[-1] == 7).all()) and bool((buffer[:, cols:] == 7).all())


def test_gradient_buffers_take_the_vector_form_without_the_padding(native_lib):
    """allocate_outputs: the logits' alignment, not their row stride."""
    for dtype in TYPES:
        wide = torch.zeros(6, 5000, device=DEV, dtype=dtype)
        for view in (wide[:, :1000], wide[:, 3:1003], wide[:, :999], wide[1:2, 7:8], wide[:0, :40], wide):
            (out,) = L.allocate_outputs("token_logprobs_backward", (view,))
            vec = 16 // view.element_size()
            assert out.shape == view.shape and out.dtype == dtype
            if view.shape[0] > 1:
                assert (out.data_ptr() - view.data_ptr()) % 16 == 0 and (out.stride(0) - view.stride(0)) % vec == 0
                assert out.stride(0) < view.shape[1] + vec
    x, targets = _logits(6, 1000, torch.bfloat16, 60)
    wide = torch.zeros(6, 5000, device=DEV, dtype=torch.bfloat16)
    logits = wide[:, 3:1003]
    logits.copy_(x)
    _, stats, _, _, _ = D.token_logprobs_forward(x, targets)
    ins = (logits, targets.to(DEV), stats.float().to(DEV), None, torch.ones(6, device=DEV), None)
    (out,) = L.allocate_outputs("token_logprobs_backward", ins)
    _launch("token_logprobs_backward", ins, (out,))
    want, mag, logp = D.token_logprobs_backward(x, targets, stats.float(), None, torch.ones(6))
    _within(out, want, mag * U * (64 + 16 * logp.abs() + 8 * 20) + _rounding(torch.bfloat16, want), "dlogits")


def test_launchers_refuse(native_lib):
    x, targets = _logits(4, 600, torch.float32, 61)
    logits, targets = x.to(DEV), targets.to(DEV)
    outs = L.allocate_outputs("token_logprobs_forward", (logits, targets), top_k=4)
    index, value = (t.to(DEV) for t in _teacher(x, 6, 62))
    kd = L.allocate_outputs("distill_topk_forward", (logits,))
    f32 = torch.zeros(4, device=DEV)

    def bad(name, inputs, outputs, match, **kw):
        with pytest.raises((ValueError, N.CreditError), match=match):
            L.NATIVE_LAUNCHERS[name](inputs, outputs, **kw)

    bad("token_logprobs_forward", (logits.half(), targets), outs, "dtype")
    bad("token_logprobs_forward", (logits.T, targets), outs, "contiguous rows")
    bad("token_logprobs_forward", (logits[:1].expand(4, 600), targets), outs, "contiguous rows")
    bad("token_logprobs_forward", (logits[0], targets), outs, "two dimensions")
    bad("token_logprobs_forward", (logits, targets.int()), outs, "targets must have dtype")
    bad("token_logprobs_forward", (logits, targets[:3]), outs, "targets must have shape")
    bad("token_logprobs_forward", (logits, targets.cpu()), outs, "targets must be a CUDA tensor")
    bad("token_logprobs_forward", (logits, None), outs, "go together")
    bad("token_logprobs_forward", (logits, targets), (*outs[:3], None, outs[4]), "go together")
    bad("token_logprobs_forward", (logits, targets), outs, "temperature", temperature=0.0)
    bad("token_logprobs_forward", (logits, targets), outs, "cluster_size", cluster_size=5)
    wide = torch.zeros(4, 129, device=DEV)
    bad("token_logprobs_forward", (logits, targets), (*outs[:3], wide, wide.long()), "top_k")
    bad("token_logprobs_backward", (logits, targets, outs[1], None, f32, f32), (torch.empty_like(logits),), "entropy")
    shifted = torch.zeros(4 * 600 + 1, device=DEV)
    bad("token_logprobs_backward", (shifted[:-1].view(4, 600), targets, outs[1], None, f32, None),
        (shifted[1:].view(4, 600),), "overlap")
    bad("distill_topk_forward", (logits, index[:, :5], value), kd, "teacher_index must be contiguous")
    bad("distill_topk_forward", (logits, index, value.double()), kd, "teacher_logprob must have dtype")
    bad("distill_topk_forward", (logits, index, value), (kd[0], kd[1][:, :5].contiguous()), "stats must have shape")
    norm = tuple(_on_gpu(t) for t in _norm_inputs(4, 512, torch.float32, 63))
    outs = L.allocate_outputs("residual_norm_forward", norm)
    bad("residual_norm_forward", (norm[0], norm[1].bfloat16(), *norm[2:]), outs, "residual must have dtype")
    bad("residual_norm_forward", (*norm[:2], None, *norm[3:]), outs, "go together")
    bad("residual_norm_forward", norm, (outs[0], outs[0], *outs[2:]), "differ")
    bad("residual_norm_forward", norm, outs, "eps", eps=0.0)
    back = (norm[0], None, norm[0], outs[0], *norm[2:], outs[2], outs[3])
    grads = L.allocate_outputs("residual_norm_backward", back)
    bad("residual_norm_backward", back, grads, "workspace", workspace=torch.empty(64, dtype=torch.uint8, device=DEV))
    bad("residual_norm_backward", back, (*grads[:3], None, grads[4]), "go together")
    assert N.device_status() == 0


def test_one_value_more_than_32_bits_of_elements(native_lib):
    """Offsets past 2^31 elements: the last rows of a matrix of 2.2e9 logits, and of one as wide of the norms."""
    rows, cols = 17000, 131072
    buffer = torch.empty(rows, cols, device=DEV, dtype=torch.bfloat16)
    x, targets = _logits(2, cols, torch.bfloat16, 64)
    buffer[-2:] = x.to(DEV)
    target = torch.full((rows,), -1, device=DEV)
    target[-2:] = targets.to(DEV)
    outs = L.allocate_outputs("token_logprobs_forward", (buffer, target), top_k=3)
    _launch("token_logprobs_forward", (buffer, target), outs)
    _check_logprobs(x, targets, [o[-2:] for o in outs], 1.0, 3)
    g = torch.ones(rows, device=DEV)
    _launch("token_logprobs_backward", (buffer, target, outs[1], None, g, None), (buffer,))     # in place
    _, stats, _, _, _ = D.token_logprobs_forward(x, targets)
    want, mag, logp = D.token_logprobs_backward(x, targets, outs[1][-2:].cpu(), None, torch.ones(2))
    _within(buffer[-2:], want, mag * U * (64 + 16 * logp.abs() + 8 * 20) + _rounding(torch.bfloat16, want), "dlogits")
    assert float(buffer[:-2].abs().max()) == 0.0
    del buffer
    rows, cols = 540000, 4096
    block = torch.zeros(rows, cols, device=DEV, dtype=torch.bfloat16)
    last = _norm_inputs(2, cols, torch.bfloat16, 65)
    block[-2:] = last[0].to(DEV)
    residual = torch.zeros_like(block)
    residual[-2:] = last[1].to(DEV)
    ins = (block, residual, *(t.to(DEV) for t in last[2:]))
    outs = L.allocate_outputs("residual_norm_forward", ins)
    _launch("residual_norm_forward", ins, outs, residual_scale=0.7, eps=1e-5)
    _check_norm_forward(last, [o[-2:] for o in outs], 0.7, 1e-5, torch.bfloat16)
    assert N.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(2, 1 << 22), (1, (1 << 22) - 5), (150000, 33)])
def test_widest_and_most_rows(native_lib, dtype, rows, cols):
    """The largest width, and more rows than two grid dimensions of 65535 would hold, against fp64 torch on the GPU.
    Tolerances as in _check_logprobs and _check_logprob_gradient (512 additions a chain at the largest width)."""
    gen = torch.Generator(device=DEV).manual_seed(71)
    x = (torch.randn(rows, cols, generator=gen, device=DEV) * 2.0).to(dtype)
    targets = torch.randint(0, cols, (rows,), generator=gen, device=DEV)
    outs = _poisoned(L.allocate_outputs("token_logprobs_forward", (x, targets), top_k=5))
    _launch("token_logprobs_forward", (x, targets), outs)
    z = x.double()
    logp = torch.log_softmax(z, -1)
    log_n = math.log2(cols)
    e_sum = (768 + 64 * log_n) * U
    assert float((outs[0] - logp.gather(1, targets[:, None])[:, 0]).abs().max()) < e_sum + 8 * U * 40
    entropy = -(logp.exp() * logp).sum(-1)
    assert float((outs[2] - entropy).abs().max()) < e_sum * (2 + log_n) + 8 * U * log_n
    value, index = torch.sort(x, dim=-1, descending=True, stable=True)
    assert torch.equal(outs[4], index[:, :5])
    del value, index
    g = torch.rand(rows, generator=gen, device=DEV)
    (grad,) = L.allocate_outputs("token_logprobs_backward", (x,))
    _launch("token_logprobs_backward", (x, targets, outs[1], None, g, None), (grad,))
    want = -logp.exp() * g[:, None].double()
    want.scatter_add_(1, targets[:, None], g[:, None].double())
    tol = (64 + 16 * 40 + 8 * 20) * U * logp.exp() + 768 * U * logp.exp() + 1e-37
    tol.scatter_add_(1, targets[:, None], torch.full((rows, 1), (64 + 8 * 20) * U, device=DEV, dtype=torch.float64))
    tol += want.abs() * (2.0 ** -8 if dtype == torch.bfloat16 else 0.0)
    assert bool(((grad.double() - want).abs() <= tol).all())
    del want, tol
    k = 16
    teacher = torch.arange(k, device=DEV) * (cols // k) + torch.randint(0, cols // k, (rows, k), generator=gen, device=DEV)
    weight = torch.log_softmax(torch.randn(rows, k, generator=gen, device=DEV), -1) + math.log(0.9)
    outs = _poisoned(L.allocate_outputs("distill_topk_forward", (x, teacher, weight)))
    _launch("distill_topk_forward", (x, teacher, weight), outs)
    w, rest = weight.double(), 1.0 - weight.double().exp().sum(-1)
    outside = torch.logsumexp(logp.scatter(1, teacher, -math.inf), -1)
    loss = (w.exp() * (w - logp.gather(1, teacher))).sum(-1) + rest * (rest.log() - outside)
    assert float((outs[0] - loss).abs().max()) < 3 * e_sum + 24 * U * 60
    (grad,) = L.allocate_outputs("distill_topk_backward", (x,))
    _launch("distill_topk_backward", (x, teacher, weight, outs[1], g), (grad,))
    want = (logp - outside[:, None]).exp() * (outside.exp() - rest)[:, None]
    want.scatter_(1, teacher, logp.gather(1, teacher).exp() - w.exp())
    want *= g[:, None].double()
    size = (logp - outside[:, None]).exp() + logp.exp()
    size.scatter_add_(1, teacher, w.exp())
    tol = size * U * (64 + 32 * 40 + 1536) + want.abs() * (2.0 ** -8 if dtype == torch.bfloat16 else 0.0) + 1e-37
    assert bool(((grad.double() - want).abs() <= tol).all())
    assert N.device_status() == 0


def test_first_launch_of_a_form_inside_a_capture(native_lib):
    """The device's first call sets the library up; any other form of a kernel may then meet its first launch in a
    capture."""
    warm = torch.zeros(2, 64, device=DEV)
    L.launch_token_logprobs_forward((warm, None), L.allocate_outputs("token_logprobs_forward", (warm, None)))
    x, targets = _logits(3, 777, torch.bfloat16, 72)
    index, value = _teacher(x, 5, 73)
    logits, targets_d, index_d, value_d = (t.to(DEV) for t in (x, targets, index, value))
    outs = L.allocate_outputs("token_logprobs_forward", (logits, targets_d), top_k=7)
    kd = L.allocate_outputs("distill_topk_forward", (logits,))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        L.launch_token_logprobs_forward((logits, targets_d), outs, cluster_size=2)
        L.launch_distill_topk_forward((logits, index_d, value_d), kd, cluster_size=2, tail=False)
    graph.replay()
    torch.cuda.synchronize()
    _check_logprobs(x, targets, outs, 1.0, 7)
