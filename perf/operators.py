"""What is measured of three operators at the end of a decoder, in both directions:

* `residual_norm`: the norms after and before a block, fused with the block's gate and the scaled
  residual;
* `token_logprobs`: log probabilities of given tokens with entropy and top alternatives;
* `distill_topk`: distillation from a teacher's top logits.

`run` computes them in plain torch, in 32 bits, or (`own`) by the launchers of `credit_b200`.
Definitions that the formulas leave open:

* a logit of -inf is masked: probability 0, never an alternative (index -1, log probability -inf);
* a row whose target is negative is ignored: zeros in its outputs and in its gradient;
* `stats` holds the row maximum of the logits and log(sum(exp((x - max) / temperature)));
* ties among alternatives go to the lowest index.
"""
from __future__ import annotations

import math

import torch

own = False

_TORCH = {"bf16": torch.bfloat16, "f32": torch.float32}
DEV = "cuda"


def listed():
    return [
        # --- norms around a block ------------------------------------------------------------
        # one decode step of a few sequences: latency
        dict(name="norm_fwd_decode", op="norm_fwd", rows=8, cols=4096, dtype="bf16", post=True, gate=True),
        # a training micro-batch at a wide model
        dict(name="norm_fwd_train", op="norm_fwd", rows=16384, cols=8192, dtype="bf16", post=True, gate=True),
        # the same step's backward
        dict(name="norm_bwd_train", op="norm_bwd", rows=16384, cols=4096, dtype="bf16", post=True, gate=True),
        # fp32 and a width that no vector divides, no gate: a small model under test
        dict(name="norm_bwd_odd", op="norm_bwd", rows=2049, cols=5003, dtype="f32", post=True, gate=False),
        # --- log probabilities -----------------------------------------------------------------
        # a decode step that reports alternatives to its client
        dict(name="logprob_decode", op="logprob_fwd", rows=8, cols=131072, ld=131072, dtype="bf16", top_k=20,
             entropy=True, temperature=1.0, masked=0.0, ignored=0.0),
        # scoring a rollout batch under the policy, padded tokens among it
        dict(name="logprob_score", op="logprob_fwd", rows=4096, cols=131072, ld=131072, dtype="bf16", top_k=0,
             entropy=True, temperature=0.7, masked=0.0, ignored=0.05),
        # a teacher's pass that lists alternatives; fp32, odd width, rows not 16-byte aligned, masked logits
        dict(name="logprob_list_odd", op="logprob_fwd", rows=1023, cols=50001, ld=50001, dtype="f32", top_k=64,
             entropy=True, temperature=1.0, masked=0.1, ignored=0.0),
        # gradient of a policy loss with an entropy bonus
        dict(name="logprob_bwd", op="logprob_bwd", rows=4096, cols=65536, ld=65536, dtype="bf16", entropy=True,
             temperature=0.7, masked=0.0, ignored=0.05),
        # fp32 with a padded vocabulary
        dict(name="logprob_bwd_padded", op="logprob_bwd", rows=777, cols=32003, ld=32064, dtype="f32", entropy=False,
             temperature=1.0, masked=0.1, ignored=0.1),
        # --- distillation ----------------------------------------------------------------------
        # a student's batch against 64 stored teacher logits, the rest of the mass in one bucket
        dict(name="distill_fwd", op="distill_fwd", rows=2048, cols=131072, ld=131072, dtype="bf16", top_k=64,
             tail=True, temperature=1.0),
        # its gradient
        dict(name="distill_bwd", op="distill_bwd", rows=2048, cols=131072, ld=131072, dtype="bf16", top_k=64,
             tail=True, temperature=1.0),
        # a small fp32 student, teacher renormalised over its list
        dict(name="distill_bwd_small", op="distill_bwd", rows=64, cols=32768, ld=32768, dtype="f32", top_k=20,
             tail=False, temperature=2.0),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm_fwd", "norm_bwd", "logprob_fwd", "logprob_bwd", "distill_fwd", "distill_bwd"])
    dtype = rng.choice(["bf16", "f32"])
    wide = 2 if dtype == "f32" else 1
    if op.startswith("norm"):
        cols = _log_uniform(rng, 512, 16384)
        if rng.random() < 0.7:
            cols -= cols % 64
        limit = (16384 * 8192 if op == "norm_fwd" else 16384 * 4096) // wide
        rows = min(_log_uniform(rng, 1, 32768), limit // cols)
        return dict(op=op, rows=rows, cols=cols, dtype=dtype, post=rng.random() < 0.75, gate=rng.random() < 0.5)
    cols = _log_uniform(rng, 8000, 262144)
    if rng.random() < 0.6:
        cols -= cols % 64
    limit = {"logprob_fwd": 4096 * 131072, "logprob_bwd": 4096 * 65536,
             "distill_fwd": 2048 * 131072, "distill_bwd": 2048 * 131072}[op] // wide
    ld = cols if rng.random() < 0.6 else (cols + 127) // 128 * 128
    rows = min(_log_uniform(rng, 1, 8192), limit // ld)
    case = dict(op=op, rows=rows, cols=cols, ld=ld, dtype=dtype, temperature=rng.choice([0.6, 1.0, 1.5]))
    if op.startswith("logprob"):
        case.update(entropy=rng.random() < 0.6, masked=rng.choice([0.0, 0.3]), ignored=0.0)
        if op == "logprob_fwd":
            case["top_k"] = rng.choice([0, 0, 1, 5, 20, 64, 128])
        if case.get("top_k", 0) == 0:
            case["ignored"] = rng.choice([0.0, 0.1])
    else:
        case.update(top_k=rng.choice([8, 20, 64, 128]), tail=rng.random() < 0.5)
    return case


# --------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------
def _generator(seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return gen


def _normal(shape, std, gen):
    return torch.empty(shape, device=DEV, dtype=torch.float32).normal_(0.0, std, generator=gen)


def _uniform(shape, low, high, gen):
    return torch.empty(shape, device=DEV, dtype=torch.float32).uniform_(low, high, generator=gen)


def _row_blocks(rows, cols):
    step = max(1, (1 << 26) // cols)
    return [(r, min(rows, r + step)) for r in range(0, rows, step)]


def _logits(case, gen):
    """Logits as a head gives them: a broad normal bulk, one likely token a row, a few runners-up, and
    the masked columns of a grammar. Returns the [rows, cols] view of a [rows, ld] buffer, and the
    likely tokens."""
    rows, cols, ld = case["rows"], case["cols"], case["ld"]
    buffer = torch.zeros(rows, ld, device=DEV, dtype=_TORCH[case["dtype"]])
    likely = torch.randint(0, cols, (rows,), device=DEV, generator=gen)
    runners = torch.randint(0, cols, (rows, 8), device=DEV, generator=gen)
    peak = _uniform((rows,), 8.0, 18.0, gen)
    steps = _uniform((rows, 8), 5.0, 12.0, gen)
    for a, b in _row_blocks(rows, cols):
        x = _normal((b - a, cols), 2.5, gen)
        x.scatter_(1, runners[a:b], steps[a:b])
        if case.get("masked", 0.0):
            hidden = _uniform((b - a, cols), 0.0, 1.0, gen) < case["masked"]
            x.masked_fill_(hidden, -math.inf)
        x.scatter_(1, likely[a:b, None], peak[a:b, None])
        buffer[a:b, :cols] = x
    return buffer[:, :cols], likely


def _targets(case, likely, gen):
    rows = case["rows"]
    other = torch.randint(0, case["cols"], (rows,), device=DEV, generator=gen)
    # under a mask every given token is one that the mask leaves
    swap = (_uniform((rows,), 0.0, 1.0, gen) < 0.3) & (case["masked"] == 0.0)
    targets = torch.where(swap, other, likely)
    ignored = _uniform((rows,), 0.0, 1.0, gen) < case["ignored"]
    return torch.where(ignored, torch.full_like(targets, -1), targets)


def _teacher(case, logits, likely, gen):
    """A teacher that mostly agrees with the student: distinct random columns, the likely token among
    them, log probabilities that leave part of the mass outside the list."""
    rows, cols, k = case["rows"], case["cols"], case["top_k"]
    stride = cols // k
    index = torch.arange(k, device=DEV) * stride + torch.randint(0, stride, (rows, k), device=DEV, generator=gen)
    slot = torch.clamp(likely // stride, max=k - 1)
    inside = likely < k * stride
    index = index.scatter(1, slot[:, None], torch.where(inside, likely, index.gather(1, slot[:, None])[:, 0])[:, None])
    value = _normal((rows, k), 2.0, gen)
    value.scatter_(1, slot[:, None], _uniform((rows, 1), 4.0, 9.0, gen))
    kept = _uniform((rows, 1), 0.6, 0.99, gen)
    logprob = torch.log_softmax(value.double(), -1) + torch.log(kept.double())
    order = torch.argsort(logprob, dim=-1, descending=True)
    return index.gather(1, order).contiguous(), logprob.gather(1, order).float().contiguous()


def _safe(m):
    return torch.where(torch.isinf(m), torch.zeros_like(m), m)


def _saved_stats(logits, temperature):
    """What a forward pass leaves for the backward one: stats [rows, 2] and the entropy, from 64 bits."""
    rows = logits.shape[0]
    stats = torch.empty(rows, 2, device=DEV)
    entropy = torch.empty(rows, device=DEV)
    for a, b in _row_blocks(rows, 2 * logits.shape[1]):
        x = logits[a:b].double()
        m = x.amax(-1, keepdim=True)
        d = (x - _safe(m)) / temperature
        e = torch.exp(d)
        total = e.sum(-1)
        stats[a:b, 0] = m[:, 0].float()
        stats[a:b, 1] = torch.log(total).float()
        entropy[a:b] = (torch.log(total) - torch.where(e > 0, e * d, 0.0).sum(-1) / total).float()
    return stats, entropy


def _saved_distill_stats(logits, index, logprob, temperature, tail):
    """stats [rows, 6]: maximum and log sum of all logits, of those outside the list (of all without
    a tail), the teacher's log normaliser, its mass outside the list; from 64 bits."""
    rows = logits.shape[0]
    stats = torch.empty(rows, 6, device=DEV)
    for a, b in _row_blocks(rows, 3 * logits.shape[1]):
        x = logits[a:b].double()
        m = x.amax(-1)
        stats[a:b, 0] = m.float()
        stats[a:b, 1] = torch.log(torch.exp((x - m[:, None]) / temperature).sum(-1)).float()
        v = logprob[a:b].double()
        if tail:
            x = x.scatter(1, index[a:b], -math.inf)
            stats[a:b, 4] = 0.0
            stats[a:b, 5] = (1.0 - torch.exp(v).sum(-1)).float()
        else:
            stats[a:b, 4] = torch.logsumexp(v, -1).float()
            stats[a:b, 5] = 0.0
        m = x.amax(-1)
        stats[a:b, 2] = m.float()
        stats[a:b, 3] = torch.log(torch.exp((x - m[:, None]) / temperature).sum(-1)).float()
    return stats


def prepare(case, seed):
    gen = _generator(seed)
    op, rows, cols = case["op"], case["rows"], case["cols"]
    dtype = _TORCH[case["dtype"]]
    st = {"case": case}
    if op.startswith("norm"):
        def matrix(std):
            return _normal((rows, cols), std, gen).to(dtype)
        st["block"] = matrix(0.4)
        st["post_weight"] = _uniform((cols,), 0.5, 1.5, gen) if case["post"] else None
        st["gate"] = _uniform((cols,), 0.2, 1.2, gen) if case["gate"] else None
        st["pre_weight"] = _uniform((cols,), 0.5, 1.5, gen)
        st["residual_scale"], st["eps"] = 0.9, 1.0e-6
        if op == "norm_fwd":
            st["residual"] = matrix(1.5)
        else:
            st["residual_out"] = matrix(1.8)
            st["dy"], st["dresidual_out"] = matrix(0.02), matrix(0.02)
            st["post_rstd"] = torch.rsqrt(st["block"].float().square().mean(-1) + st["eps"]) if case["post"] else None
            st["pre_rstd"] = torch.rsqrt(st["residual_out"].float().square().mean(-1) + st["eps"])
    else:
        st["logits"], likely = _logits(case, gen)
        if op.startswith("logprob"):
            st["targets"] = _targets(case, likely, gen)
        else:
            st["index"], st["logprob"] = _teacher(case, st["logits"], likely, gen)
        if op == "logprob_bwd":
            st["stats"], entropy = _saved_stats(st["logits"], case["temperature"])
            st["entropy"] = entropy if case["entropy"] else None
            st["dlogprob"] = _normal((rows,), 1.0 / rows, gen)
            st["dentropy"] = _uniform((rows,), 0.0, 0.01 / rows, gen) if case["entropy"] else None
        if op == "distill_bwd":
            st["stats"] = _saved_distill_stats(st["logits"], st["index"], st["logprob"], case["temperature"],
                                               case["tail"])
            st["dloss"] = _uniform((rows,), 0.5 / rows, 1.5 / rows, gen)
    if own:
        _prepare_own(st)
    return st


def _prepare_own(st):
    """The output buffers (and the workspace) that a program keeps from call to call."""
    from credit_b200 import launchers as L

    case = st["case"]
    op = case["op"]
    if op == "norm_fwd":
        st["inputs"] = (st["block"], st["residual"], st["post_weight"], st["gate"], st["pre_weight"])
        st["outputs"] = L.allocate_outputs("residual_norm_forward", st["inputs"])
    elif op == "norm_bwd":
        st["inputs"] = (st["dy"], st["dresidual_out"], st["block"], st["residual_out"], st["post_weight"], st["gate"],
                        st["pre_weight"], st["post_rstd"], st["pre_rstd"])
        st["outputs"] = L.allocate_outputs("residual_norm_backward", st["inputs"])
        need = L.residual_norm_backward_workspace_bytes(case["rows"], case["cols"], st["dy"].dtype)
        st["workspace"] = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
    elif op == "logprob_fwd":
        st["inputs"] = (st["logits"], st["targets"])
        st["outputs"] = L.allocate_outputs("token_logprobs_forward", st["inputs"], top_k=case["top_k"],
                                           entropy=case["entropy"])
    elif op == "logprob_bwd":
        st["inputs"] = (st["logits"], st["targets"], st["stats"], st["entropy"], st["dlogprob"], st["dentropy"])
        st["outputs"] = L.allocate_outputs("token_logprobs_backward", st["inputs"])
    elif op == "distill_fwd":
        st["inputs"] = (st["logits"], st["index"], st["logprob"])
        st["outputs"] = L.allocate_outputs("distill_topk_forward", st["inputs"])
    else:
        st["inputs"] = (st["logits"], st["index"], st["logprob"], st["stats"], st["dloss"])
        st["outputs"] = L.allocate_outputs("distill_topk_backward", st["inputs"])


# --------------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------------
def run(st):
    return (_run_own if own else _run_plain)(st)


def _run_own(st):
    from credit_b200.launchers import NATIVE_LAUNCHERS as launch

    case = st["case"]
    op, ins, outs = case["op"], st["inputs"], st["outputs"]
    if op == "norm_fwd":
        launch["residual_norm_forward"](ins, outs, residual_scale=st["residual_scale"], eps=st["eps"])
    elif op == "norm_bwd":
        launch["residual_norm_backward"](ins, outs, residual_scale=st["residual_scale"], workspace=st["workspace"])
    elif op == "logprob_fwd":
        launch["token_logprobs_forward"](ins, outs, temperature=case["temperature"])
    elif op == "logprob_bwd":
        launch["token_logprobs_backward"](ins, outs, temperature=case["temperature"])
    elif op == "distill_fwd":
        launch["distill_topk_forward"](ins, outs, temperature=case["temperature"], tail=case["tail"])
    else:
        launch["distill_topk_backward"](ins, outs, temperature=case["temperature"], tail=case["tail"])
    return [o for o in outs if o is not None]


def _run_plain(st):
    case = st["case"]
    return {"norm_fwd": _norm_fwd, "norm_bwd": _norm_bwd, "logprob_fwd": _logprob_fwd, "logprob_bwd": _logprob_bwd,
            "distill_fwd": _distill_fwd, "distill_bwd": _distill_bwd}[case["op"]](st, case)


def _norm_fwd(st, case):
    o, h = st["block"].float(), st["residual"].float()
    outs = []
    n = o
    if case["post"]:
        r1 = torch.rsqrt((o * o).mean(-1) + st["eps"])
        n = o * r1[:, None] * st["post_weight"]
        outs.append(r1)
    if case["gate"]:
        n = n * st["gate"]
    joined = st["residual_scale"] * h + n
    r2 = torch.rsqrt((joined * joined).mean(-1) + st["eps"])
    y = joined * r2[:, None] * st["pre_weight"]
    dtype = st["block"].dtype
    return [joined.to(dtype), y.to(dtype), *outs, r2]


def _norm_bwd(st, case):
    dy, dres = st["dy"].float(), st["dresidual_out"].float()
    o, joined = st["block"].float(), st["residual_out"].float()
    r2 = st["pre_rstd"][:, None]
    v = joined * r2
    t = dy * st["pre_weight"]
    total = dres + r2 * (t - v * (t * v).mean(-1, keepdim=True))
    dresidual = st["residual_scale"] * total
    n = o * st["post_rstd"][:, None] if case["post"] else o
    b = total
    if case["gate"]:
        b = b * st["gate"]
    if case["post"]:
        b = b * st["post_weight"]
        b = st["post_rstd"][:, None] * (b - n * (b * n).mean(-1, keepdim=True))
    dtype = st["dy"].dtype
    outs = [b.to(dtype), dresidual.to(dtype)]
    shared = (total * n).sum(0) if case["post"] or case["gate"] else None
    if case["post"]:
        outs.append(shared * st["gate"] if case["gate"] else shared)
    if case["gate"]:
        outs.append(shared * st["post_weight"] if case["post"] else shared)
    outs.append((dy * v).sum(0))
    return outs


def _logprob_fwd(st, case):
    x, targets = st["logits"].float(), st["targets"]
    used = targets >= 0
    s = 1.0 / case["temperature"]
    m = x.amax(-1, keepdim=True)
    d = (x - _safe(m)) * s
    e = torch.exp(d)
    total = e.sum(-1)
    log_total = torch.log(total)
    picked = d.gather(1, targets.clamp(min=0)[:, None])[:, 0] - log_total
    outs = [torch.where(used, picked, 0.0),
            torch.where(used[:, None], torch.stack([m[:, 0], log_total], -1), 0.0)]
    if case["entropy"]:
        mean = torch.where(e > 0, e * d, 0.0).sum(-1) / total
        outs.append(torch.where(used, log_total - mean, 0.0))
    k = case["top_k"]
    if k:
        # descending by value, ascending by index among equals: one integer key for both
        bits = (x + 0.0).view(torch.int32).long()
        ordered = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
        column = torch.arange(x.shape[1], device=x.device)
        top = torch.topk((ordered << 32) | (0x7FFFFFFF - column), k, dim=-1).indices
        value = d.gather(1, top)
        outs += [value - log_total[:, None], torch.where(torch.isinf(value), -1, top)]
    return outs


def _logprob_bwd(st, case):
    x, targets = st["logits"].float(), st["targets"]
    s = 1.0 / case["temperature"]
    logp = (x - st["stats"][:, :1]) * s - st["stats"][:, 1:]
    p = torch.exp(logp)
    weight = st["dlogprob"][:, None]
    if case["entropy"]:
        weight = weight + torch.where(p > 0, st["dentropy"][:, None] * (logp + st["entropy"][:, None]), 0.0)
    grad = -p * weight
    grad.scatter_add_(1, targets.clamp(min=0)[:, None], st["dlogprob"][:, None])
    grad = torch.where(targets[:, None] >= 0, grad * s, 0.0)
    return [grad.to(st["logits"].dtype)]


def _distill_fwd(st, case):
    x, index, v = st["logits"].float(), st["index"], st["logprob"]
    s = 1.0 / case["temperature"]
    m = x.amax(-1)
    log_total = torch.log(torch.exp((x - m[:, None]) * s).sum(-1))
    logq = (x.gather(1, index) - m[:, None]) * s - log_total[:, None]
    if case["tail"]:
        norm = torch.zeros_like(m)
        rest = (1.0 - torch.exp(v.double()).sum(-1)).float()
        outside = x.scatter(1, index, -math.inf)
        m2 = outside.amax(-1)
        log_total2 = torch.log(torch.exp((outside - m2[:, None]) * s).sum(-1))
        log_rest = (m2 - m) * s + log_total2 - log_total
        tail = rest * (torch.log(rest) - log_rest)
    else:
        norm = torch.logsumexp(v, -1)
        rest, tail, m2, log_total2 = torch.zeros_like(m), 0.0, m, log_total
    logw = v - norm[:, None]
    loss = (torch.exp(logw) * (logw - logq)).sum(-1) + tail
    return [loss, torch.stack([m, log_total, m2, log_total2, norm, rest], -1)]


def _distill_bwd(st, case):
    x, index, v, stats = st["logits"].float(), st["index"], st["logprob"], st["stats"]
    s = 1.0 / case["temperature"]
    m, log_total, m2, log_total2, norm, rest = (c[:, None] for c in stats.unbind(-1))
    q = torch.exp((x.gather(1, index) - m) * s - log_total)
    grad = torch.exp((x - m2) * s - log_total2)
    if case["tail"]:
        grad = grad * (torch.exp((m2 - m) * s + log_total2 - log_total) - rest)
    grad.scatter_(1, index, q - torch.exp(v - norm))
    return [(grad * (s * st["dloss"][:, None])).to(st["logits"].dtype)]


# --------------------------------------------------------------------------------------------
# floors
# --------------------------------------------------------------------------------------------
def work(case):
    n = case["rows"] * case["cols"]
    size = 4 if case["dtype"] == "f32" else 2
    rows, cols, op = case["rows"], case["cols"], case["op"]
    params = 4 * cols * (1 + int(case.get("post", False)) + int(case.get("gate", False)))
    per_row = 4 * rows * (1 + int(case.get("post", False)))
    if op == "norm_fwd":
        return {"bytes": 4 * n * size + params + per_row, "flops": 10 * n}
    if op == "norm_bwd":
        return {"bytes": 6 * n * size + 2 * params + per_row, "flops": 26 * n}
    if op == "logprob_fwd":
        # an ignored row needs no logits
        read = n * (1.0 - case["ignored"]) * size
        out = rows * (8 + 4 + 8 + (4 if case["entropy"] else 0) + 12 * case["top_k"])
        return {"bytes": int(read + out), "flops": (7 if case["entropy"] else 5) * n}
    if op == "logprob_bwd":
        read = n * (1.0 - case["ignored"]) * size
        return {"bytes": int(read + n * size + rows * 28), "flops": (8 if case["entropy"] else 5) * n}
    if op == "distill_fwd":
        return {"bytes": n * size + rows * (12 * case["top_k"] + 28), "flops": 5 * n}
    return {"bytes": 2 * n * size + rows * (12 * case["top_k"] + 28), "flops": 5 * n}


# --------------------------------------------------------------------------------------------
# the same from the definitions in 64 bits
# --------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    op, rows, cols = case["op"], case["rows"], case["cols"]
    parts = []
    sums = None
    for a, b in _row_blocks(rows, 2 * cols):
        part, column_sums = _EXACT[op](st, case, slice(a, b))
        parts.append(part)
        if column_sums is not None:
            sums = column_sums if sums is None else [u + w for u, w in zip(sums, column_sums)]
    outs = [torch.cat(column) for column in zip(*parts)]
    if op != "norm_bwd":
        return outs
    shared, dpre = sums
    one = torch.ones(cols, device=DEV, dtype=torch.float64)
    if case["post"]:
        outs.append(shared * (st["gate"].double() if case["gate"] else one))
    if case["gate"]:
        outs.append(shared * (st["post_weight"].double() if case["post"] else one))
    return outs + [dpre]


def _channel_scale(st):
    scale = torch.ones(st["block"].shape[1], device=DEV, dtype=torch.float64)
    for name in ("post_weight", "gate"):
        if st[name] is not None:
            scale = scale * st[name].double()
    return scale


def _exact_norm_fwd(st, case, rows):
    o, h = st["block"][rows].double(), st["residual"][rows].double()
    outs = []
    if case["post"]:
        rms = (o.square().sum(-1) / o.shape[1] + st["eps"]).sqrt()
        o = o / rms[:, None]
        outs.append(1.0 / rms)
    joined = st["residual_scale"] * h + o * _channel_scale(st)
    rms = (joined.square().sum(-1) / joined.shape[1] + st["eps"]).sqrt()
    return [joined, joined / rms[:, None] * st["pre_weight"].double(), *outs, 1.0 / rms], None


def _exact_norm_bwd(st, case, rows):
    dy, dres = st["dy"][rows].double(), st["dresidual_out"][rows].double()
    o, joined = st["block"][rows].double(), st["residual_out"][rows].double()
    cols = o.shape[1]
    r2 = st["pre_rstd"][rows].double()[:, None]
    weighted = dy * st["pre_weight"].double()
    total = dres + r2 * weighted - r2 ** 3 / cols * joined * (weighted * joined).sum(-1, keepdim=True)
    dn = total * _channel_scale(st)
    n = o
    if case["post"]:
        r1 = st["post_rstd"][rows].double()[:, None]
        n = o * r1
        dn = r1 * dn - r1 ** 3 / cols * o * (dn * o).sum(-1, keepdim=True)
    return [dn, st["residual_scale"] * total], [(total * n).sum(0), (dy * joined * r2).sum(0)]


def _exact_logprob_fwd(st, case, rows):
    x, targets = st["logits"][rows].double(), st["targets"][rows]
    z = x / case["temperature"]
    logp = torch.log_softmax(z, -1)
    used = targets >= 0
    at = logp.gather(1, targets.clamp(min=0)[:, None])[:, 0]
    m = x.amax(-1)
    stats = torch.stack([m, torch.logsumexp(z, -1) - m / case["temperature"]], -1)
    zero = torch.zeros_like(at)
    outs = [torch.where(used, at, zero), torch.where(used[:, None], stats, zero[:, None])]
    if case["entropy"]:
        outs.append(torch.where(used, torch.special.entr(logp.exp()).sum(-1), zero))
    if case["top_k"]:
        value, index = torch.sort(st["logits"][rows], dim=-1, descending=True, stable=True)
        value, index = value[:, :case["top_k"]], index[:, :case["top_k"]]
        outs += [logp.gather(1, index), index.masked_fill(value == -math.inf, -1)]
    return outs, None


def _exact_logprob_bwd(st, case, rows):
    x, targets = st["logits"][rows].double(), st["targets"][rows]
    stats = st["stats"][rows].double()
    logp = (x - stats[:, :1]) / case["temperature"] - stats[:, 1:]
    p = logp.exp()
    g = st["dlogprob"][rows].double()[:, None]
    grad = -g * p
    if case["entropy"]:
        # d entropy / d z = -p (log p + entropy), p log p -> 0 as p -> 0
        plogp = -torch.special.entr(p)
        grad -= st["dentropy"][rows].double()[:, None] * (plogp + p * st["entropy"][rows].double()[:, None])
    hit = torch.arange(x.shape[1], device=x.device) == targets[:, None]
    grad = torch.where(hit, grad + g, grad) / case["temperature"]
    return [grad * (targets >= 0)[:, None]], None


def _list_mask(index, cols):
    mask = torch.zeros(index.shape[0], cols, device=index.device, dtype=torch.bool)
    return mask.scatter_(1, index, True)


def _exact_distill_fwd(st, case, rows):
    x, index, v = st["logits"][rows].double(), st["index"][rows], st["logprob"][rows].double()
    z = x / case["temperature"]
    m, lse = x.amax(-1), torch.logsumexp(z, -1)
    logq = z.gather(1, index) - lse[:, None]
    if case["tail"]:
        outside = z.masked_fill(_list_mask(index, x.shape[1]), -math.inf)
        m2, lse2 = outside.amax(-1) * case["temperature"], torch.logsumexp(outside, -1)
        norm = torch.zeros_like(m)
        rest = -torch.expm1(torch.logsumexp(v, -1))
        extra = torch.xlogy(rest, rest) - rest * (lse2 - lse)
    else:
        m2, lse2, norm = m, lse, torch.logsumexp(v, -1)
        rest = extra = torch.zeros_like(m)
    w = torch.exp(v - norm[:, None])
    loss = (w * (v - norm[:, None]) - w * logq).sum(-1) + extra
    t = case["temperature"]
    return [loss, torch.stack([m, lse - m / t, m2, lse2 - m2 / t, norm, rest], -1)], None


def _exact_distill_bwd(st, case, rows):
    x, index, v = st["logits"][rows].double(), st["index"][rows], st["logprob"][rows].double()
    m, l1, m2, l2, norm, rest = (c[:, None] for c in st["stats"][rows].double().unbind(-1))
    t = case["temperature"]
    q = torch.exp((x - m) / t - l1)
    w = torch.zeros_like(x).scatter_(1, index, torch.exp(v - norm))
    if case["tail"]:
        share = torch.exp((x - m2) / t - l2)
        listed_here = _list_mask(index, x.shape[1])
        outside_mass = torch.exp((m2 - m) / t + l2 - l1)
        grad = torch.where(listed_here, q - w, share * (outside_mass - rest))
    else:
        grad = q - w
    return [grad * st["dloss"][rows].double()[:, None] / t], None


_EXACT = {"norm_fwd": _exact_norm_fwd, "norm_bwd": _exact_norm_bwd, "logprob_fwd": _exact_logprob_fwd,
          "logprob_bwd": _exact_logprob_bwd, "distill_fwd": _exact_distill_fwd, "distill_bwd": _exact_distill_bwd}
