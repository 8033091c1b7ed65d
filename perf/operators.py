"""Performance cases of the operators around the counter layers: layer norm in front of them, and the
log probabilities and the distillation loss behind the vocabulary head.

`run` computes a case in its plain form (elementary torch operations in 32 bits), or through
`motifcl_amd.ops` where `own` is true.  `exact` gives the same outputs in 64 bits.

Kinds of cases:
  norm           y = (x - mean) / sqrt(var + eps) * gain + bias, with the rows' mean and 1 / sqrt(var + eps)
  norm_grad      the gradients of x, gain and bias from those two numbers of a row
  log_probs      of softmax(logits / temperature): the given token's log probability, the entropy, the log of the
                 sum, and the `top` likeliest tokens with theirs
  log_probs_grad the gradient of the logits from the gradients of the token's log probability and of the entropy
  distill        temperature^2 * KL(teacher's top logits || student) of each row, and the weighted gradient
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5


def listed():
    return [
        # serving: the norm in front of a 4096-wide layer, one token
        {"name": "norm_one_token", "kind": "norm", "rows": 1, "cols": 4096, "dtype": "f32", "bias": True, "pad": 0},
        # training: a step of the 15M-shaped model, 288 wide (288 floats: no multiple of a wave's accesses)
        {"name": "norm_288", "kind": "norm", "rows": 8192, "cols": 288, "dtype": "f32", "bias": True, "pad": 0},
        # training: the 7B-shaped layer at 32768 tokens, in the layers' own type
        {"name": "norm_4096", "kind": "norm", "rows": 32768, "cols": 4096, "dtype": "f32", "bias": False, "pad": 0},
        # the backward pass of the 15M-shaped model's step
        {"name": "norm_grad_288", "kind": "norm_grad", "rows": 8192, "cols": 288, "dtype": "f32", "bias": True, "pad": 0},
        # the backward pass of the 7B-shaped layer, activations kept in 16 bits
        {"name": "norm_grad_4096", "kind": "norm_grad", "rows": 32768, "cols": 4096, "dtype": "bf16", "bias": True, "pad": 0},
        # serving: one decoded token with its alternatives
        {"name": "log_probs_one_token", "kind": "log_probs", "rows": 1, "vocab": 32768, "dtype": "f32", "top": 20,
         "temperature": 1.0, "pad": 0},
        # serving: a batch of decoded tokens over a large ragged vocabulary, in 16 bits
        {"name": "log_probs_batch", "kind": "log_probs", "rows": 61, "vocab": 128011, "dtype": "bf16", "top": 8,
         "temperature": 0.7, "pad": 53},
        # a teacher's pass over a step's tokens: its 64 top logits for every token
        {"name": "log_probs_teacher", "kind": "log_probs", "rows": 4096, "vocab": 32768, "dtype": "f32", "top": 64,
         "temperature": 1.0, "pad": 0},
        # policy gradient with an entropy bonus on a short batch, odd sizes
        {"name": "log_probs_grad_odd", "kind": "log_probs_grad", "rows": 509, "vocab": 32003, "dtype": "f32",
         "entropy": True, "temperature": 1.0, "pad": 0},
        # cross entropy of a step's tokens, large vocabulary
        {"name": "log_probs_grad_large", "kind": "log_probs_grad", "rows": 8192, "vocab": 128000, "dtype": "bf16",
         "entropy": False, "temperature": 1.0, "pad": 0},
        # distillation of the 15M-shaped model: a step of 4096 tokens over its 32k vocabulary
        {"name": "distill_32k", "kind": "distill", "rows": 4096, "vocab": 32768, "dtype": "f32", "top": 64,
         "temperature": 2.0, "pad": 0},
        # distillation over a large ragged vocabulary, rows longer than a compute unit's registers
        {"name": "distill_large", "kind": "distill", "rows": 2048, "vocab": 128011, "dtype": "f32", "top": 100,
         "temperature": 1.0, "pad": 5},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm_grad", "log_probs", "log_probs_grad", "distill"])
    case = {"kind": kind, "dtype": rng.choice(["f32", "f32", "bf16", "f16"]), "pad": rng.choice([0, 0, 0, 1, 8, 53])}
    if kind in ("norm", "norm_grad"):
        case["cols"] = _log_int(rng, 16, 16384)
        case["rows"] = min(_log_int(rng, 1, 65536), (1 << 27) // case["cols"])
        case["bias"] = rng.random() < 0.5
        return case
    case["vocab"] = _log_int(rng, 96, 131072)
    case["rows"] = min(_log_int(rng, 1, 16384), (1 << 27) // case["vocab"])
    case["temperature"] = rng.choice([0.7, 1.0, 1.0, 2.0])
    if kind == "log_probs":
        case["top"] = rng.choice([0, 1, _log_int(rng, 2, 64)])
    elif kind == "log_probs_grad":
        case["entropy"] = rng.random() < 0.5
    else:
        case["top"] = _log_int(rng, 1, min(128, case["vocab"] // 2))
    return case


def _rows_of(g, rows, cols, pad, dtype, spread):
    """[rows, cols] normal numbers, each row `pad` elements behind the end of the one before it."""
    whole = torch.randn(rows, cols + pad, generator=g, device="cuda", dtype=torch.float32).mul_(spread).to(dtype)
    return whole[:, :cols]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype, rows, pad = DTYPES[case["dtype"]], case["rows"], case["pad"]

    def uniform(*size):
        return torch.rand(*size, generator=g, device="cuda", dtype=torch.float32)

    s = {"case": case}
    if case["kind"] in ("norm", "norm_grad"):
        cols = case["cols"]
        x = _rows_of(g, rows, cols, pad, dtype, 1.5)
        x += (0.5 * uniform(rows, 1)).to(dtype)  # activations are not centred
        s["x"], s["gain"] = x, 0.5 + uniform(cols)
        s["bias"] = uniform(cols) - 0.5 if case["bias"] else None
        if case["kind"] == "norm_grad":
            s["grad_out"] = _rows_of(g, rows, cols, pad, dtype, 0.01)
            wide = x.float()
            s["mean"] = wide.mean(1)
            s["rstd"] = 1.0 / torch.sqrt((wide - s["mean"][:, None]).square().mean(1) + EPS)
        return s
    vocab = case["vocab"]
    # a mean over the rows; in fp16 a training program scales its loss, or most of the gradients would be zero
    scale = 1024.0 if case["dtype"] == "f16" else 1.0 / rows
    logits = _rows_of(g, rows, vocab, pad, dtype, 2.0)
    s["tokens"] = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    logits.scatter_add_(1, s["tokens"].long()[:, None], (6.0 * uniform(rows, 1)).to(dtype))  # the model knows something
    logits[:, vocab - vocab // 64:] = -math.inf  # the head is wider than the vocabulary
    s["tokens"].clamp_(max=vocab - vocab // 64 - 1)
    s["logits"] = logits
    if case["kind"] == "log_probs_grad":
        padding = uniform(rows) < 0.05
        s["tokens"] = torch.where(padding, torch.full_like(s["tokens"], -100), s["tokens"])
        s["grad_log_prob"] = torch.where(padding, 0.0, -scale * (0.5 + uniform(rows)))
        s["grad_entropy"] = -0.1 * scale * uniform(rows) if case["entropy"] else None
        z = logits.float() / case["temperature"]
        top = z.max(1).values
        e = torch.exp(z - top[:, None])
        total = e.sum(1)
        s["lse"] = top + torch.log(total)
        finite = torch.where(e > 0, z - top[:, None], 0.0)
        s["entropy"] = torch.log(total) - (e * finite).sum(1) / total
    if case["kind"] == "distill":
        top = case["top"]
        span = (vocab - vocab // 64) // top  # one id in each of `top` stretches, in a random order
        ids = torch.arange(top, device="cuda") * span + (uniform(rows, top) * span).long().clamp_(max=span - 1)
        ids = torch.gather(ids, 1, uniform(rows, top).argsort(1))
        teacher = torch.sort(torch.randn(rows, top, generator=g, device="cuda") * 2.0 + 6.0, 1, descending=True).values
        near = 0.7 * teacher + 0.5 * torch.randn(rows, top, generator=g, device="cuda")
        logits.scatter_add_(1, ids, near.to(dtype))  # a student that is on its way
        fewer = torch.arange(top, device="cuda") >= (top * (0.75 + uniform(rows, 1))).long().clamp_(min=1)
        s["teacher_ids"] = torch.where(fewer, -1, ids).to(torch.int32)  # some rows hold fewer alternatives
        s["teacher_logits"] = teacher
        s["weight"] = torch.where(uniform(rows) < 0.05, 0.0, scale * (0.5 + uniform(rows)))  # padding counts nothing
    return s


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "norm":
        x = s["x"].float()
        mean = x.sum(1) / case["cols"]
        d = x - mean[:, None]
        rstd = 1.0 / torch.sqrt((d * d).sum(1) / case["cols"] + EPS)
        y = d * rstd[:, None] * s["gain"]
        if s["bias"] is not None:
            y = y + s["bias"]
        return {"y": y.to(s["x"].dtype), "mean": mean, "rstd": rstd}
    if kind == "norm_grad":
        xhat = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
        dy = s["grad_out"].float()
        h = dy * s["gain"]
        a, b = h.sum(1) / case["cols"], (h * xhat).sum(1) / case["cols"]
        grad_x = s["rstd"][:, None] * (h - a[:, None] - xhat * b[:, None])
        out = {"grad_x": grad_x.to(s["x"].dtype), "grad_gain": (dy * xhat).sum(0)}
        if s["bias"] is not None:
            out["grad_bias"] = dy.sum(0)
        return out
    logits = s["logits"]
    z = logits.float() / case["temperature"]
    if kind == "log_probs":
        largest = z.max(1).values
        d = z - largest[:, None]
        e = torch.exp(d)
        total = e.sum(1)
        lse = largest + torch.log(total)
        entropy = torch.log(total) - (e * torch.where(e > 0, d, 0.0)).sum(1) / total
        log_prob = torch.gather(z, 1, s["tokens"].long()[:, None])[:, 0] - lse
        out = {"log_prob": log_prob, "entropy": entropy, "lse": lse}
        if case["top"]:
            # one whole number for each logit, in their order, with the lower index first among equals
            bits = (logits.float() + 0.0).view(torch.int32)
            order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 32)
            order = order + ((1 << 32) - 1 - torch.arange(case["vocab"], device=z.device))
            best = torch.topk(order, case["top"], dim=1).values
            ids = (1 << 32) - 1 - (best & ((1 << 32) - 1))
            out["top_ids"] = ids.to(torch.int32)
            out["top_log_probs"] = torch.gather(z, 1, ids) - lse[:, None]
        return out
    if kind == "log_probs_grad":
        log_p = z - s["lse"][:, None]
        p = torch.exp(log_p)
        token = s["tokens"].long()[:, None]
        given = torch.where(token[:, 0] >= 0, s["grad_log_prob"], 0.0)
        grad = -given[:, None] * p
        if s["grad_entropy"] is not None:
            log_p = torch.where(p > 0, log_p, 0.0)
            grad = grad - s["grad_entropy"][:, None] * p * (log_p + s["entropy"][:, None])
        grad = grad.scatter_add_(1, token.clamp(min=0), given[:, None])
        return {"grad_logits": (grad / case["temperature"]).to(logits.dtype)}
    t = case["temperature"]
    d = z - z.max(1).values[:, None]
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    ids = s["teacher_ids"].long()
    there = ids >= 0
    ids = ids.clamp(min=0)
    y = torch.where(there, s["teacher_logits"] / t, -math.inf)
    y = y - y.max(1).values[:, None]
    log_q = y - torch.log(torch.exp(y).sum(1, keepdim=True))
    q = torch.exp(log_q)
    log_p = torch.gather(d, 1, ids) - torch.log(total)
    loss = t * t * (q * torch.where(there, log_q - log_p, 0.0)).sum(1)
    grad = (e / total).scatter_add_(1, ids, -q)
    grad = grad * (s["weight"] * t)[:, None]
    return {"loss": loss, "grad_logits": grad.to(logits.dtype)}


def run(state):
    if not own:
        return _plain(state)
    from motifcl_amd import ops

    s, case = state, state["case"]
    kind = case["kind"]
    if kind == "norm":
        y, mean, rstd = ops.layer_norm(s["x"], s["gain"], s["bias"], EPS)
        return {"y": y, "mean": mean, "rstd": rstd}
    if kind == "norm_grad":
        grad_x, grad_gain, grad_bias = ops.layer_norm_backward(s["grad_out"], s["x"], s["mean"], s["rstd"], s["gain"],
                                                               bias=s["bias"] is not None)
        out = {"grad_x": grad_x, "grad_gain": grad_gain}
        if grad_bias is not None:
            out["grad_bias"] = grad_bias
        return out
    if kind == "log_probs":
        r = ops.token_log_probs(s["logits"], s["tokens"], top=case["top"], temperature=case["temperature"])
        out = {"log_prob": r.log_prob, "entropy": r.entropy, "lse": r.lse}
        if case["top"]:
            out["top_ids"], out["top_log_probs"] = r.top_ids, r.top_log_probs
        return out
    if kind == "log_probs_grad":
        return {"grad_logits": ops.token_log_probs_backward(
            s["logits"], s["tokens"], s["lse"], s["entropy"], s["grad_log_prob"], s["grad_entropy"],
            temperature=case["temperature"])}
    loss, grad = ops.distill_top(s["logits"], s["teacher_ids"], s["teacher_logits"], temperature=case["temperature"],
                                 weight=s["weight"])
    return {"loss": loss, "grad_logits": grad}


def exact(case, seed):
    s = prepare(case, seed)
    kind, wide = case["kind"], torch.float64
    if kind in ("norm", "norm_grad"):
        x = s["x"].to(wide).requires_grad_()
        gain = s["gain"].to(wide).requires_grad_()
        bias = s["bias"].to(wide).requires_grad_() if s["bias"] is not None else None
        if kind == "norm":
            y = torch.nn.functional.layer_norm(x, (case["cols"],), gain, bias, EPS)
            var, mean = torch.var_mean(x, 1, correction=0)
            return {"y": y.detach(), "mean": mean.detach(), "rstd": torch.rsqrt(var + EPS).detach()}
        y = torch.nn.functional.layer_norm(x, (case["cols"],), gain, bias, EPS)
        leaves = [x, gain] + ([bias] if bias is not None else [])
        grads = torch.autograd.grad(y, leaves, s["grad_out"].to(wide))
        return dict(zip(("grad_x", "grad_gain", "grad_bias"), grads))
    z = s["logits"].to(wide)
    if kind == "log_probs":
        z = z / case["temperature"]
        log_p = torch.log_softmax(z, 1)
        out = {"log_prob": log_p.gather(1, s["tokens"].long()[:, None]).squeeze(1),
               "entropy": torch.special.entr(log_p.exp()).sum(1), "lse": torch.logsumexp(z, 1)}
        if case["top"]:
            out["top_ids"], out["top_log_probs"] = None, log_p.topk(case["top"], 1).values
        return out
    if kind == "log_probs_grad":
        log_p = torch.log_softmax(z / case["temperature"], 1)
        p = log_p.exp()
        grad = torch.zeros_like(z).scatter_(1, s["tokens"].long().clamp(min=0)[:, None], 1.0).sub_(p)
        grad.mul_(s["grad_log_prob"].to(wide).unsqueeze(1))  # zero in the padding rows
        if s["grad_entropy"] is not None:
            surprise = torch.special.entr(p)
            grad.add_((surprise - p * surprise.sum(1, keepdim=True)) * s["grad_entropy"].to(wide).unsqueeze(1))
        return {"grad_logits": grad.div_(case["temperature"])}
    z.requires_grad_()
    t, there = case["temperature"], s["teacher_ids"] >= 0
    q = torch.softmax((s["teacher_logits"].to(wide) / t).masked_fill(~there, -math.inf), 1)
    log_p = torch.log_softmax(z / t, 1).gather(1, s["teacher_ids"].long().clamp(min=0))
    loss = t * t * (torch.special.xlogy(q, q) - torch.where(there, q * log_p, 0.0)).sum(1)
    grad = torch.autograd.grad((loss * s["weight"].to(wide)).sum(), z)[0]
    return {"loss": loss.detach(), "grad_logits": grad}


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    rows = case["rows"]
    if case["kind"] == "norm":
        n = rows * case["cols"]
        return {"bytes": 2 * size * n + 8 * rows + (8 if case["bias"] else 4) * case["cols"], "flops": 8 * n}
    if case["kind"] == "norm_grad":
        n = rows * case["cols"]
        return {"bytes": 3 * size * n + 8 * rows + (12 if case["bias"] else 8) * case["cols"], "flops": 14 * n}
    n = rows * case["vocab"]
    if case["kind"] == "log_probs":
        return {"bytes": size * n + rows * (16 + 8 * case["top"]), "flops": 7 * n}
    if case["kind"] == "log_probs_grad":
        return {"bytes": 2 * size * n + rows * 20, "flops": 5 * n}
    return {"bytes": 2 * size * n + rows * (8 + 8 * case["top"]), "flops": 8 * n}
