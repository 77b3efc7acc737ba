"""Alternatives of rows in which thousands of elements share the value that bounds them: finite masks that leave few
tokens, anywhere in the row, and rows with too many elements above the bound as well. Every path of the selection has to
give the value-descending, column-ascending list. Rows beyond the slowest path's border are timed against ordinary ones."""
import math

import pytest
import torch

from credit_b200 import _native as N
from credit_b200 import launchers as L
from test_gpu_decoder_ops import DEV, NAN, TYPES, U, _check_logprobs, _run_logprobs, _within

pytestmark = pytest.mark.gpu


def _rows(dtype, cols, mask):
    gen = torch.Generator().manual_seed(cols)
    x = torch.full((17, cols), mask).to(dtype)
    free = (torch.randn(cols, generator=gen) * 3).to(dtype)
    for r, left in enumerate((0, 1, 3, 8, 19, 20, 21, 60)):          # rows 0...7: tokens left at random places
        places = torch.randperm(cols, generator=gen)[:left]
        x[r, places] = free[places]
    x[8, :9] = free[:9]                                             # at the row's start, at its end
    x[9, -9:] = free[-9:]
    x[10, -1] = 5.0
    run = min(cols, 1900)
    x[11, cols - run:] = free[cols - run:]                          # contiguous tokens that some warps do not see
    warp = (torch.arange(cols) // (16 // x.element_size()) // 32) % 8
    x[12] = torch.where(warp < 7, free.float(), torch.tensor(float(mask))).to(dtype)   # an eighth masked, by warps:
    x[13] = torch.where(warp == 0, free.float(), torch.tensor(float(mask))).to(dtype)  # more above the bound than places
    x[14, ::2] = -math.inf                                          # both kinds of mask
    x[14, 101:105] = 1.0
    x[15, 7] = NAN                                                  # NaN above the mask, fewer than asked for
    x[15, cols // 2] = math.inf
    x[16, : cols // 2] = mask / 2                                   # two finite masks
    x[16, 3] = 2.0
    return x


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask", [-1e9, -3.3895e38, -30000.0, 0.0])
@pytest.mark.parametrize("cols,ld,shift", [(20000, None, 0), (16411, 16500, 3), (40001, None, 1)])
def test_finite_masks(native_lib, dtype, mask, cols, ld, shift):
    x = _rows(dtype, cols, mask)
    for cluster in (1, 2, 8):
        for top_k in (1, 20, 128):
            _check_logprobs(x, None, _run_logprobs(x, None, top_k, 1.0, cluster, ld, shift), 1.0, top_k)
    assert N.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [9001, 40001])
def test_as_many_rows_as_fill_the_device(native_lib, dtype, cols):
    """The form with half the threads a row, rows of every kind next to one another. Copies of a row lie at different
    places between two 16-byte boundaries and add their terms in different orders: their lists are equal, their real
    results are each within _check_logprobs's tolerance (here its largest, that of the entropy) of one value, so
    within twice that of one another."""
    x = _rows(dtype, cols, -1e9).repeat(71, 1)       # 1207 rows
    outs = _run_logprobs(x, None, 32)
    _check_logprobs(x[:17], None, [None if o is None else o[:17] for o in outs], 1.0, 32)
    log_n = math.log2(cols)
    for o in outs:
        if o is None:
            continue
        copies = o.view(71, 17, -1)
        first = copies[:1].expand_as(copies)
        if o.dtype == torch.int64:
            assert torch.equal(copies, first)
        else:
            size = first.double().abs().nan_to_num(0.0, 0.0, 0.0)
            tol = (128 + 64 * log_n) * U * (2 + log_n) + 8 * U * (size + 2 * log_n)
            _within(copies, first.cpu(), 2 * tol.cpu())
    assert N.device_status() == 0


def test_a_finite_mask_costs_no_more_than_a_few_reads(native_lib):
    """592 rows of 131072, 8 tokens left, 20 asked for: within four times an ordinary row's time (once it was 64 times). A
    timing test with that much room fails only for a path that reads the row many times."""
    x = torch.randn(592, 131072, device=DEV).bfloat16()
    masked = torch.full_like(x, -1e9)
    masked[:, 5:131072:16384] = x[:, 5:131072:16384]

    def time(logits):
        outs = L.allocate_outputs("token_logprobs_forward", (logits, None), top_k=20)
        best = math.inf
        for _ in range(5):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            torch.cuda.synchronize()
            start.record()
            for _ in range(4):
                L.launch_token_logprobs_forward((logits, None), outs)
            end.record()
            torch.cuda.synchronize()
            best = min(best, start.elapsed_time(end))
        return best

    time(x)
    assert time(masked) < 4.0 * time(x)
