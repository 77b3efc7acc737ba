"""CPU oracle of the operators at the end of a decoder (residual_norm, token_logprobs, distill_topk),
in fp64 from the stored inputs. TEST INFRASTRUCTURE ONLY, like `reference_ops`; nothing in
`credit_b200/` imports it. The reference has no function for these, so they restate the formulas; the
gradients are written out and checked against autograd and differences by the CPU tests.

The conventions are those of `include/credit_b200.h`: -inf is a masked logit, a negative target an
ignored row, a negative teacher index an unused place, a row holding NaN or +inf has NaN results.
"""
from __future__ import annotations

import math

import torch

F64 = torch.float64


def residual_norm_forward(block, residual, post_weight, gate, pre_weight, residual_scale=1.0, eps=1e-6):
    """(residual_out, y, post_rstd | None, pre_rstd), all fp64."""
    n = block.to(F64)
    post_rstd = None
    if post_weight is not None:
        post_rstd = (n.square().mean(-1) + eps).rsqrt()
        n = n * post_rstd[:, None] * post_weight.to(F64)
    if gate is not None:
        n = n * gate.to(F64)
    out = residual_scale * residual.to(F64) + n
    pre_rstd = (out.square().mean(-1) + eps).rsqrt()
    return out, out * pre_rstd[:, None] * pre_weight.to(F64), post_rstd, pre_rstd


def residual_norm_backward(dy, dresidual_out, block, residual_out, post_weight, gate, pre_weight, post_rstd, pre_rstd,
                           residual_scale=1.0):
    """((dblock, dresidual, dpost_weight | None, dgate | None, dpre_weight), magnitudes): the second
    holds, for each output, the sum of the absolute values of the terms it is made of (what rounding
    errors are relative to)."""
    dy, o, h = dy.to(F64), block.to(F64), residual_out.to(F64)
    d = torch.zeros_like(dy) if dresidual_out is None else dresidual_out.to(F64)
    one = torch.ones(o.shape[1], dtype=F64)
    w1 = one if post_weight is None else post_weight.to(F64)
    g = one if gate is None else gate.to(F64)
    c = w1 * g
    r2 = pre_rstd.to(F64)[:, None]
    v, t = h * r2, dy * pre_weight.to(F64)
    total = d + r2 * (t - v * (t * v).mean(-1, keepdim=True))
    m_total = d.abs() + r2 * (t.abs() + v.abs() * (t * v).abs().mean(-1, keepdim=True))
    if post_weight is None:
        n, dblock, m_block = o, c * total, c.abs() * m_total
    else:
        r1 = post_rstd.to(F64)[:, None]
        n = o * r1
        dn = c * total
        dblock = r1 * (dn - n * (dn * n).mean(-1, keepdim=True))
        m_dn = c.abs() * m_total
        m_block = r1 * (m_dn + n.abs() * (m_dn * n.abs()).mean(-1, keepdim=True))
    shared, m_shared = (total * n).sum(0), (m_total * n.abs()).sum(0)
    outs = (dblock, residual_scale * total, None if post_weight is None else g * shared,
            None if gate is None else w1 * shared, (dy * v).sum(0))
    mags = (m_block, abs(residual_scale) * m_total, None if post_weight is None else g.abs() * m_shared,
            None if gate is None else w1.abs() * m_shared, (dy * v).abs().sum(0))
    return outs, mags


def _row_softmax(x, temperature):
    """(max, log sum, d = (x - max) / T with masked logits at -inf, p) of fp64 rows."""
    m = x.amax(-1)
    m = torch.where(torch.isnan(x).any(-1), torch.full_like(m, math.nan), m)
    d = (x - torch.where(m == -math.inf, torch.zeros_like(m), m)[:, None]) / temperature
    d = torch.where(x == -math.inf, torch.full_like(d, -math.inf), d)
    total = d.exp().sum(-1)
    broken = ~(m < math.inf)
    log_sum = torch.where(m == -math.inf, torch.zeros_like(m), total.log())
    log_sum = torch.where(broken, torch.full_like(m, math.nan), log_sum)
    return m, log_sum, d


def token_logprobs_forward(logits, targets=None, temperature=1.0, top_k=0):
    """(logprob | None, stats, entropy, top_logprob | None, top_index | None)."""
    x = logits.to(F64)
    rows, cols = x.shape
    m, log_sum, d = _row_softmax(x, temperature)
    logp = d - log_sum[:, None]
    empty, broken = m == -math.inf, ~(m < math.inf)
    terms = torch.where(torch.isinf(logp), torch.zeros_like(logp), logp.exp() * logp)
    entropy = torch.where(broken, torch.full_like(m, math.nan), -terms.sum(-1))
    stats = torch.stack([m, log_sum], -1)
    logprob = None
    used = torch.ones(rows, dtype=torch.bool)
    if targets is not None:
        used = targets >= 0
        logprob = logp.gather(1, targets.clamp(0, cols - 1)[:, None])[:, 0]
        logprob = torch.where(empty, torch.full_like(m, -math.inf), logprob)
        logprob = torch.where(broken | (targets >= cols), torch.full_like(m, math.nan), logprob)
        logprob = torch.where(used, logprob, torch.zeros_like(m))
    stats = torch.where(used[:, None], stats, torch.zeros_like(stats))
    entropy = torch.where(used, entropy, torch.zeros_like(entropy))
    top_logprob = top_index = None
    if top_k:
        top_logprob = torch.full((rows, top_k), -math.inf, dtype=F64)
        top_index = torch.full((rows, top_k), -1, dtype=torch.int64)
        for r in range(rows):
            if not bool(used[r]):
                continue
            # NaN first, then values descending; Python's sort is stable: columns ascend among equals
            row = x[r].tolist()
            order = [j for j in range(cols) if row[j] != -math.inf]
            order.sort(key=lambda j: (0, 0.0) if math.isnan(row[j]) else (1, -row[j]))
            order = order[:top_k]
            top_index[r, :len(order)] = torch.tensor(order, dtype=torch.int64)
            if order:
                top_logprob[r, :len(order)] = math.nan if bool(broken[r]) else logp[r, order]
    return logprob, stats, entropy, top_logprob, top_index


def token_logprobs_backward(logits, targets, stats, entropy, dlogprob, dentropy=None, temperature=1.0):
    """(dlogits, magnitudes, log p); stats and entropy are the forward call's, as stored."""
    x = logits.to(F64)
    m, log_sum = stats.to(F64).unbind(-1)
    logp = (x - m[:, None]) / temperature - log_sum[:, None]
    logp = torch.where(x == -math.inf, torch.full_like(x, -math.inf), logp)
    p = logp.exp()
    g = dlogprob.to(F64)[:, None]
    weight, m_weight = g.expand_as(p), g.abs().expand_as(p)
    if dentropy is not None:
        gh, h = dentropy.to(F64)[:, None], entropy.to(F64)[:, None]
        finite = torch.where(p > 0, logp, torch.zeros_like(logp))
        weight = weight + gh * (finite + h)
        m_weight = m_weight + gh.abs() * (finite.abs() + h.abs())
    grad, mag = -p * weight, p * m_weight
    valid = (targets >= 0) & (m != -math.inf)
    hit = torch.arange(x.shape[1])[None, :] == targets[:, None]
    at = -torch.expm1(logp) * g + torch.where(p > 0, grad + p * g, torch.zeros_like(p))
    grad = torch.where(hit, at, grad)
    mag = torch.where(hit, mag + (torch.expm1(logp) * g).abs(), mag)
    broken = ~(m < math.inf) | (targets >= x.shape[1])
    grad = torch.where(broken[:, None], torch.full_like(grad, math.nan), grad)
    zero = torch.zeros_like(grad)
    return (torch.where(valid[:, None], grad, zero) / temperature, torch.where(valid[:, None], mag, zero) / temperature,
            logp)


def distill_topk_forward(logits, index, logprob, temperature=1.0, tail=True):
    """(loss, stats [rows, 6]); row by row, as the header words it."""
    rows, cols = logits.shape
    loss = torch.zeros(rows, dtype=F64)
    stats = torch.zeros(rows, 6, dtype=F64)
    for r in range(rows):
        x = logits[r].to(F64)
        places = [(int(c), float(v)) for c, v in zip(index[r], logprob[r].to(F64)) if int(c) >= 0]
        if any(c >= cols for c, _ in places):
            loss[r] = stats[r, 0] = math.nan
            continue
        values = torch.tensor([v for _, v in places], dtype=F64)
        mass = float(values.exp().sum())
        log_mass = float(torch.logsumexp(values, 0)) if places else -math.inf    # also where mass leaves fp64's range
        stats[r, 0] = -math.inf
        if not places or (not tail and log_mass == -math.inf):
            continue
        m, log_sum, d = (t[0] for t in _row_softmax(x[None], temperature))
        columns = torch.tensor([c for c, _ in places])
        outside = x.clone()
        if tail:
            outside[columns] = -math.inf
        m2, log_sum2, _ = (t[0] for t in _row_softmax(outside[None], temperature))
        norm, rest = 0.0, 0.0
        if not tail:
            norm = log_mass
        elif m2 == -math.inf or mass > 1.0:
            if log_mass == -math.inf:
                continue
            norm = log_mass
        else:
            rest = 1.0 - mass
        total = 0.0
        for c, v in places:
            w = math.exp(v - norm)
            if w > 0.0:
                total += w * (v - norm) - w * float(d[c] - log_sum if m != -math.inf else -math.inf)
        if rest > 0.0:
            log_rest = float((m2 - m) / temperature + log_sum2 - log_sum)
            total += rest * (math.log(rest) - log_rest)
        stats[r] = torch.stack([m, log_sum, m2, log_sum2, torch.tensor(norm, dtype=F64), torch.tensor(rest, dtype=F64)])
        broken = not bool(m < math.inf)
        loss[r] = math.nan if broken else total
        if broken:
            stats[r, 0] = math.nan
    return loss, stats


def distill_topk_backward(logits, index, logprob, stats, dloss, temperature=1.0):
    """(dlogits, magnitudes); stats as stored by the forward call."""
    rows, cols = logits.shape
    grad = torch.zeros(rows, cols, dtype=F64)
    mag = torch.zeros(rows, cols, dtype=F64)
    for r in range(rows):
        x, s = logits[r].to(F64), stats[r].to(F64)
        m, log_sum, m2, log_sum2, norm, rest = (float(v) for v in s)
        places = [(int(c), float(v)) for c, v in zip(index[r], logprob[r].to(F64)) if int(c) >= 0]
        if any(c >= cols for c, _ in places) or math.isnan(m):
            grad[r] = math.nan
            continue
        if not places or m == -math.inf:
            continue
        q = ((x - m) / temperature - log_sum).exp()
        if m2 == -math.inf:
            row, size = torch.zeros_like(x), torch.zeros_like(x)
        else:
            share = ((x - m2) / temperature - log_sum2).exp()
            outside = math.exp((m2 - m) / temperature + log_sum2 - log_sum)
            row, size = share * (outside - rest), share * (outside + rest)
        w = torch.zeros_like(x)
        listed = torch.zeros(cols, dtype=torch.bool)
        for c, v in places:
            w[c] += math.exp(v - norm)
            listed[c] = True
        scale = float(dloss[r]) / temperature
        grad[r] = torch.where(listed, q - w, row) * scale
        mag[r] = torch.where(listed, q + w, size) * abs(scale)
    return grad, mag
