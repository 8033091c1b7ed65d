"""The row-wise operators in 64 bits, written from their definitions (torch tensors on any device), and the
tolerances their tests use.  A rounding to a type is off by at most half a step, relative to the value."""
import math

import torch

U = 2.0 ** -24  # half a step of binary32, in which everything is computed
HALF = {torch.float32: U, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}  # half the smallest step of float16


def close(got, want, scale, steps, what):
    """|got - want| <= half a step of got's type + `steps` half steps of binary32 at `scale`; the same infinities
    and NaN."""
    got64 = got.double()
    assert torch.equal(torch.isnan(got64), torch.isnan(want)), what + ": NaN differ"
    finite = torch.isfinite(want)
    assert torch.equal(got64[~finite & ~torch.isnan(want)], want[~finite & ~torch.isnan(want)]), what + ": infinities differ"
    bound = HALF[got.dtype] * want.abs() + TINY[got.dtype] + steps * U * scale
    off = (got64 - want).abs()
    bad = finite & ~(off <= bound * torch.ones_like(off))
    assert not bad.any(), "%s: %d values off, worst %.3g of its bound" % (
        what, int(bad.sum()), float((off / bound)[bad].max()))


def layer_norm(x, gain, bias, eps):
    x = x.double()
    mean = x.mean(-1)
    d = x - mean[..., None]
    rstd = 1.0 / ((d * d).mean(-1) + eps).sqrt()
    y = d * rstd[..., None]
    y = y * gain.double() if gain is not None else y
    return y + bias.double() if bias is not None else y, mean, rstd


def layer_norm_backward(dy, x, mean, rstd, gain):
    dy, xhat = dy.double(), (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    h = dy * gain.double() if gain is not None else dy
    n = x.shape[1]
    dx = rstd.double()[:, None] * (h - h.sum(1, keepdim=True) / n - xhat * (h * xhat).sum(1, keepdim=True) / n)
    return dx, (dy * xhat).sum(0), dy.sum(0)


def softmax_parts(logits, temperature):
    """(log probabilities, probabilities, lse) with the definitions for rows of -inf alone."""
    z = logits.double() / temperature
    m = z.max(-1, keepdim=True).values
    empty = m == -math.inf
    shift = torch.where(empty, torch.zeros_like(m), m)
    s = (z - shift).exp().sum(-1, keepdim=True)
    lse = m + s.log()
    lse = torch.where(empty & ~s.isnan(), torch.full_like(lse, -math.inf), lse)
    log_p = torch.where(empty & ~s.isnan(), torch.full_like(z, -math.inf), z - lse)
    return log_p, log_p.exp(), lse[..., 0]


def entropy_of(log_p, p):
    return -(p * torch.where(p == 0, torch.zeros_like(log_p), log_p)).sum(-1)


def token_log_probs(logits, tokens, temperature):
    log_p, p, lse = softmax_parts(logits, temperature)
    there = (tokens >= 0) & (tokens < logits.shape[-1])
    picked = log_p.gather(-1, torch.where(there, tokens, 0).long()[:, None])[:, 0]
    return torch.where(there, picked, torch.zeros_like(picked)), entropy_of(log_p, p), lse


def top_ids(logits, top):
    """Larger logit first, equal ones by the lower index, NaN last."""
    z = logits.float() + 0.0
    order = torch.sort(torch.where(z.isnan(), torch.full_like(z, -math.inf), z), dim=-1, descending=True, stable=True).indices
    nan = z.gather(-1, order).isnan()
    order = order.gather(-1, torch.sort(nan.to(torch.int8), dim=-1, stable=True).indices)
    return order[..., :top].to(torch.int32)


def token_log_probs_backward(logits, tokens, g, h, temperature):
    log_p, p, lse = softmax_parts(logits, temperature)
    vocab = logits.shape[-1]
    there = (tokens >= 0) & (tokens < vocab)
    g = torch.where(there, g.double(), 0.0) if g is not None else torch.zeros_like(lse)
    out = -g[:, None] * p
    out[there, tokens[there].long()] += g[there]
    if h is not None:
        bounded = torch.where(p == 0, torch.zeros_like(log_p), log_p)
        out = out - h.double()[:, None] * p * (bounded + entropy_of(log_p, p)[:, None])
    zero = (g == 0) & (h.double() == 0 if h is not None else True) | (lse == -math.inf)
    return torch.where(zero[:, None], torch.zeros_like(out), out / temperature), p


def distill_top(logits, ids, teacher, weight, temperature):
    t = temperature
    log_p, p, lse = softmax_parts(logits, t)
    there = (ids >= 0) & (ids < logits.shape[-1])
    y = torch.where(there, teacher.double() / t, -math.inf)
    m = y.max(-1, keepdim=True).values
    e = (y - torch.where(m == -math.inf, torch.zeros_like(m), m)).exp()
    total = e.sum(-1, keepdim=True)
    q = torch.where(total == 0, torch.zeros_like(e), e / total)
    at = torch.where(there, ids, 0).long()
    inside = log_p.gather(-1, at)
    terms = torch.where(there & (q != 0), q * (q.log() - inside), torch.zeros_like(q))
    loss = t * t * terms.sum(-1)
    w = weight.double() if weight is not None else torch.ones_like(lse)
    grad = p * q.sum(-1, keepdim=True)
    grad = grad.scatter_add(-1, at, torch.where(there, -q, torch.zeros_like(q)))
    zero = (w == 0) | (total[:, 0] == 0) | (lse == -math.inf)
    scale = (w * t)[:, None]
    return loss, torch.where(zero[:, None], torch.zeros_like(grad), scale * grad), q, torch.where(zero[:, None], 0.0, scale.abs() * p)
