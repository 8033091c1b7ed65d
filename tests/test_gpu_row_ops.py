"""Layer norm, token log probabilities and the distillation loss against their definitions in 64 bits.

Bounds, in half steps of binary32 (U = 2^-24).  A thread adds at most 64 numbers (32 of f32) one behind the other and at
most 12 joins follow, so a sum is off by at most 76 U (f32: 44 U) of the sum of magnitudes; the norm's tests hold all of
them to 64 U.  Longer running sums, of long rows and of swept rows, are binary64 between stretches of as many numbers.
e^d is off by (3 |d| + 4) U of itself: the difference, the temperature's reciprocal and its product, the hardware's
exponential; with |d| e^d <= 1 a sum of e^d, which is at least 1, is off by at most (76 + 3 ln(vocab) + 4) U of itself,
128 U up to vocabularies of 8 million, and its logarithm by that."""
import math

import pytest

from . import rows64

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS = 1e-5


@pytest.fixture(scope="module")
def ops():
    import motifcl_amd
    motifcl_amd.load()
    from motifcl_amd import ops as _ops
    assert torch.cuda.is_available()
    return _ops


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def rows_of(g, rows, cols, dtype, pad=0, spread=1.0, offset=0.0):
    return (torch.randn(rows, cols + pad, generator=g, device="cuda") * spread + offset).to(dtype)[:, :cols]


# ---- layer norm ------------------------------------------------------------------------------------
NORM_SHAPES = [(1, 1), (3, 2), (5, 3), (2, 7), (4, 8), (3, 9), (17, 16), (1, 255), (6, 256), (9, 257), (33, 288), (7, 511),
               (5, 513), (3, 1000), (2, 1025), (130, 768), (1, 2047), (3, 2049), (1, 4096), (70, 4096), (3, 4097),
               (2, 8191), (2, 11008), (2, 16384), (2, 16385), (2, 32768), (2, 32771), (1, 65537), (3, 70001)]


@pytest.mark.parametrize("rows, cols", NORM_SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm(ops, rows, cols, dtype):
    g = generator(rows * 131 + cols)
    x = rows_of(g, rows, cols, dtype, pad=cols % 3, spread=2.0, offset=1.0)
    gain = torch.rand(cols, generator=g, device="cuda") + 0.5 if cols % 2 else None
    bias = torch.randn(cols, generator=g, device="cuda") if rows % 2 else None
    y, mean, rstd = ops.layer_norm(x, gain, bias, EPS)
    want, want_mean, want_rstd = rows64.layer_norm(x, gain, bias, EPS)
    largest = x.double().abs().max(1).values
    # the mean is off by 64 U of the mean magnitude; so is each difference, and the variance by twice that at most:
    # where a row's variance is far below eps or the mean, the scale is 1 / sqrt(eps)
    rows64.close(mean, want_mean, largest, 66, "mean")
    slack = 64 * rows64.U * largest * want_rstd  # error of a difference in units of the deviation
    relative = 70 * rows64.U + 2 * slack
    assert ((rstd.double() - want_rstd).abs() <= want_rstd * relative).all()
    scale = (x.double() - want_mean[:, None]).abs() * want_rstd[:, None]
    weight = gain.double() if gain is not None else 1.0
    at = (scale * (relative[:, None] + 4 * rows64.U) + slack[:, None]) * weight
    shift = bias.double().abs() if bias is not None else 0.0
    rows64.close(y, want, at / rows64.U + scale * weight + shift, 1, "y")


@pytest.mark.parametrize("rows, cols", NORM_SHAPES + [(1000, 288), (2500, 40), (1200, 2048), (600, 6000)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_backward(ops, rows, cols, dtype):
    g = generator(rows * 137 + cols)
    x = rows_of(g, rows, cols, dtype, pad=cols % 3, spread=2.0, offset=1.0)
    dy = rows_of(g, rows, cols, dtype, pad=rows % 2)
    gain = torch.rand(cols, generator=g, device="cuda") + 0.5 if cols % 2 else None
    _, mean, rstd = ops.layer_norm(x, gain, None, EPS)
    dx, dgain, dbias = ops.layer_norm_backward(dy, x, mean, rstd, gain)
    want_dx, want_dgain, want_dbias = rows64.layer_norm_backward(dy, x, mean, rstd, gain)
    xhat = ((x.double() - mean.double()[:, None]) * rstd.double()[:, None]).abs()
    h = dy.double().abs() * (gain.double() if gain is not None else 1.0)
    # rstd (h - a - xhat b): every term and the two sums (64 U of their magnitudes), xhat within 3 U of |x| + |mean|
    near = (x.double().abs() + mean.double().abs()[:, None]) * rstd.double()[:, None]
    scale = rstd.double()[:, None] * (h + h.mean(1, keepdim=True) + near * (h * near).mean(1, keepdim=True))
    rows64.close(dx, want_dx, scale, 80, "dx")
    # a workgroup adds up to rows / 512 + 1 rows one after the other, then at most 512 partial rows in 16 sums
    steps = rows / 512 + 1 + 32 + 16 + 8
    if gain is None:
        assert dgain is None
    else:
        rows64.close(dgain, want_dgain, (dy.double().abs() * near).sum(0), steps, "dgain")
    rows64.close(dbias, want_dbias, dy.double().abs().sum(0), steps, "dbias")
    del xhat


def test_layer_norm_constant_and_far_rows(ops):
    # a row of one number has deviation 0: y is the bias; far from zero the differences still count
    x = torch.full((2, 640), 7.25, device="cuda")
    y, mean, rstd = ops.layer_norm(x, None, None, EPS)
    assert torch.equal(y, torch.zeros_like(y)) and torch.equal(mean, x[:, 0])
    assert ((rstd.double() - EPS ** -0.5).abs() <= 8 * rows64.U * EPS ** -0.5).all()
    far = torch.randn(4, 1024, generator=generator(1), device="cuda") + 4096.0
    y, _, _ = ops.layer_norm(far, None, None, EPS)
    want, _, _ = rows64.layer_norm(far, None, None, EPS)
    # the mean alone is rounded, to 2^-12 of a deviation here (4096 U); every y moves by that at most twice
    assert (y.double() - want).abs().max() <= 2 * 2.0 ** -12


@pytest.mark.parametrize("cols", [40, 1000, 5000, 70001])
def test_layer_norm_in_place_and_in_halves(ops, cols):
    g = generator(cols)
    x, dy = (rows_of(g, 37, cols, torch.float32) for _ in range(2))
    gain, bias = torch.rand(cols, generator=g, device="cuda"), torch.rand(cols, generator=g, device="cuda")
    y, mean, rstd = ops.layer_norm(x, gain, bias, EPS)
    dx, dgain, dbias = ops.layer_norm_backward(dy, x, mean, rstd, gain)
    wide = torch.full((37, 2 * cols + 3), 9.0, device="cuda")
    wide[:, :cols] = x
    ops.layer_norm(wide[:, :cols], gain, bias, EPS, out=wide[:, cols:2 * cols])
    assert torch.equal(wide[:, cols:2 * cols], y) and torch.equal(wide[:, :cols], x)
    assert (wide[:, 2 * cols:] == 9.0).all()
    again = x.clone()
    assert torch.equal(ops.layer_norm(again, gain, bias, EPS, out=again)[0], y)
    for out in (dy.clone(), None):
        got = ops.layer_norm_backward(out if out is not None else dy, x, mean, rstd, gain, out=out)
        assert torch.equal(got[0], dx) and torch.equal(got[1], dgain) and torch.equal(got[2], dbias)
    over_x = x.clone()
    got = ops.layer_norm_backward(dy, over_x, mean, rstd, gain, out=over_x)
    assert torch.equal(got[0], dx) and torch.equal(got[1], dgain)
    assert ops.layer_norm_backward(dy, x, mean, rstd, gain, bias=False, input_grad=False)[0] is None
    only = ops.layer_norm_backward(dy, x, mean, rstd, None, bias=False)
    assert only[1] is None and only[2] is None


def test_layer_norm_gradient_by_differences(ops):
    g = generator(5)
    x, w = rows_of(g, 3, 24, torch.float32), rows_of(g, 3, 24, torch.float32)
    gain, bias = torch.rand(24, generator=g, device="cuda") + 0.5, torch.rand(24, generator=g, device="cuda")
    _, mean, rstd = ops.layer_norm(x, gain, bias, EPS)
    dx, dgain, dbias = ops.layer_norm_backward(w, x, mean, rstd, gain)

    def f(x, gain, bias):
        return float((ops.layer_norm(x, gain, bias, EPS)[0].double() * w.double()).sum())
    step = 2.0 ** -7
    # a difference of two sums of 72 products, each within a few U, over 2 step: 72 * 8 * U / step, and step^2 times
    # the third derivative, which is of order rstd^3 here
    bound = 72 * 8 * rows64.U / step + 8 * step * step * float(rstd.max()) ** 3
    for r, c in [(0, 0), (1, 23), (2, 11)]:
        moved = [x.clone(), x.clone()]
        moved[0][r, c] += step
        moved[1][r, c] -= step
        assert abs((f(moved[0], gain, bias) - f(moved[1], gain, bias)) / (2 * step) - float(dx[r, c])) <= bound
    for c in (0, 13):
        up, down = gain.clone(), gain.clone()
        up[c] += step
        down[c] -= step
        assert abs((f(x, up, bias) - f(x, down, bias)) / (2 * step) - float(dgain[c])) <= bound
        up, down = bias.clone(), bias.clone()
        up[c] += step
        down[c] -= step
        assert abs((f(x, gain, up) - f(x, gain, down)) / (2 * step) - float(dbias[c])) <= bound


# ---- log probabilities -------------------------------------------------------------------------------
# (rows, vocab): every kernel variant whole and cut into stretches, vectors that reach behind the end
LOGIT_SHAPES = [(1, 1), (3, 2), (2, 3), (4, 7), (3, 8), (2, 9), (5, 100), (1, 511), (3, 513), (600, 515), (2, 2047), (5, 2051),
                (7, 4096), (3, 4099), (600, 4100), (2, 8191), (540, 8195), (1, 16389), (520, 16381), (520, 16390),
                (1, 32768), (515, 32765), (2, 32771), (9, 50001), (61, 65539), (130, 128011), (1, 200003)]


def logits_of(g, rows, vocab, dtype, pad=0):
    z = rows_of(g, rows, vocab, dtype, pad=pad, spread=2.5)
    at = torch.randint(0, vocab, (rows, 1), generator=g, device="cuda")
    z.scatter_(1, at, (8.0 * torch.rand(rows, 1, generator=g, device="cuda")).to(dtype))
    return z


def check_log_probs(ops, z, tokens, top, temperature):
    r = ops.token_log_probs(z, tokens, top=top, temperature=temperature)
    want, want_h, want_lse = rows64.token_log_probs(z, tokens, temperature)
    wide = z.double() / temperature
    finite = torch.where(torch.isfinite(wide), wide, torch.zeros_like(wide)).abs().max(1).values
    there = (tokens >= 0) & (tokens < z.shape[1])
    rows64.close(r.lse, want_lse, 130.0 + 4 * finite, 1, "lse")
    rows64.close(r.log_prob, want, torch.where(there, 130.0 + 8 * finite, torch.zeros_like(finite)), 1, "log_prob")
    # u = sum e^d d adds |d| <= ln(vocab) + entropy terms: its error and that of log s, each 128 U of their magnitude
    rows64.close(r.entropy, want_h, 1.0 + math.log(z.shape[1]), 300, "entropy")
    if top == 0:
        assert r.top_ids is None and r.top_log_probs is None
        return r
    ids = rows64.top_ids(z, top)
    assert torch.equal(r.top_ids, ids)
    log_p = rows64.softmax_parts(z, temperature)[0].gather(1, ids.long())
    rows64.close(r.top_log_probs, log_p, (130.0 + 8 * finite)[:, None], 1, "top_log_probs")
    return r


@pytest.mark.parametrize("rows, vocab", LOGIT_SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_token_log_probs(ops, rows, vocab, dtype):
    g = generator(rows * 139 + vocab)
    z = logits_of(g, rows, vocab, dtype, pad=vocab % 5)
    tokens = torch.randint(-1, vocab + 1, (rows,), generator=g, device="cuda", dtype=torch.int32)
    for top, temperature in ((0, 1.0), (min(vocab, 20), 0.7), (min(vocab, 128), 2.0), (1, 1.0)):
        check_log_probs(ops, z, tokens, top, temperature)


@pytest.mark.parametrize("rows, vocab", [(3, 300), (2, 5000), (600, 700), (530, 20000), (2, 40000), (520, 32768)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_token_log_probs_of_masked_and_tied_rows(ops, rows, vocab, dtype):
    g = generator(vocab)
    lowest = torch.finfo(dtype).min
    for what in ("masked", "lowest", "constant", "few values", "sorted", "zeros", "one"):
        z = logits_of(g, rows, vocab, dtype)
        allowed = torch.rand(rows, vocab, generator=g, device="cuda") < 5.0 / vocab
        allowed[:, vocab // 2] = True
        if what == "masked":
            z = torch.where(allowed, z, torch.full_like(z, -math.inf))
        elif what == "lowest":
            z = torch.where(allowed, z, torch.full_like(z, lowest))
        elif what == "constant":
            z = torch.full_like(z, 1.5)
        elif what == "few values":
            z = torch.randint(0, 3, (rows, vocab), generator=g, device="cuda").to(dtype)
        elif what == "sorted":
            z = torch.sort(z, 1, descending=True).values
        elif what == "zeros":
            z = torch.where(allowed, torch.zeros_like(z), -torch.zeros_like(z))
        else:
            z = torch.full_like(z, -math.inf)
            z[:, vocab - 1] = 3.0
        tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
        for top in (1, 20, 128):
            if what == "lowest":  # (lowest - m) / T may leave the range: T = 1 keeps it
                check_lowest(ops, z, tokens, top)
            else:
                check_log_probs(ops, z, tokens, top, 1.0)


def check_lowest(ops, z, tokens, top):
    """Logits of the type's lowest value: probability 0 like -inf, log probability of its size."""
    r = ops.token_log_probs(z, tokens, top=top)
    log_p, p, lse = rows64.softmax_parts(z, 1.0)
    assert torch.equal(r.top_ids, rows64.top_ids(z, top))
    want = log_p.gather(1, r.top_ids.long()).float()  # beyond the range of binary32 it is -inf
    assert torch.allclose(r.top_log_probs, want, rtol=1e-5, atol=1e-4)
    rows64.close(r.lse, lse, 300.0, 1, "lse")
    rows64.close(r.entropy, rows64.entropy_of(log_p, p), 1.0 + math.log(z.shape[1]), 300, "entropy")


@pytest.mark.parametrize("vocab", [5, 600, 5000, 40000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_the_lowest_value_are_uniform(ops, vocab, dtype):
    # everything masked with the type's lowest value: (z - m) / T is 0 wherever z / T is out of range
    z = torch.full((3, vocab), torch.finfo(dtype).min, device="cuda", dtype=dtype)
    tokens = torch.tensor([0, vocab - 1, -1], dtype=torch.int32, device="cuda")
    for temperature in (0.5, 1.0, 2.0):
        r = ops.token_log_probs(z, tokens, top=3, temperature=temperature)
        uniform = torch.full((3,), -math.log(vocab), dtype=torch.float64, device="cuda")
        rows64.close(r.log_prob[:2], uniform[:2], 1.0, 200, "log_prob")
        rows64.close(r.entropy, -uniform, 1.0, 300, "entropy")
        rows64.close(r.top_log_probs, uniform[:, None].expand(3, 3), 1.0, 200, "top_log_probs")
        assert r.top_ids.tolist() == [[0, 1, 2]] * 3
        ids = torch.tensor([[0, 1]] * 3, dtype=torch.int32, device="cuda")
        loss, grad = ops.distill_top(z, ids, torch.zeros(3, 2, device="cuda"), temperature)
        want = temperature ** 2 * (math.log(vocab) - math.log(2)) + 0 * uniform
        rows64.close(loss, want, 4.0, 400, "loss")
        at = torch.full((vocab,), temperature / vocab, dtype=torch.float64, device="cuda")
        at[:2] -= 0.5 * temperature
        rows64.close(grad, at.expand(3, vocab), 1.0, 400, "grad")


@pytest.mark.parametrize("vocab", [5, 600, 5000, 40000])
def test_token_log_probs_of_empty_and_invalid_rows(ops, vocab):
    g = generator(vocab)
    inf, nan = math.inf, math.nan
    z = rows_of(g, 6, vocab, torch.float32)
    z[1] = -inf
    z[2, vocab // 3] = nan
    z[3, 1] = inf
    z[4] = nan
    z[5, : vocab // 2] = -inf
    tokens = torch.tensor([0, 1, 2, 1, 0, 0], dtype=torch.int32, device="cuda")
    top = min(vocab, 7)
    r = ops.token_log_probs(z, tokens, top=top)
    assert r.lse[1] == -inf and r.entropy[1] == 0 and r.log_prob[1] == -inf
    assert (r.top_log_probs[1] == -inf).all() and r.log_prob[5] == -inf
    for bad in (2, 3, 4):
        for out in (r.lse, r.entropy, r.log_prob):
            assert out[bad].isnan()
        assert r.top_log_probs[bad].isnan().all()
    assert torch.equal(r.top_ids, rows64.top_ids(z, top))
    good = torch.tensor([0, 5], device="cuda")
    alone = ops.token_log_probs(z[good].contiguous(), tokens[good].contiguous(), top=top)
    for a, b in zip(r, alone):
        assert torch.equal(a[good], b)
    # the gradient of an empty row is zero, of a NaN row with nothing upstream too
    up = torch.tensor([1.0, 1.0, 0.0, 0.0, 0.0, 1.0], device="cuda")
    grad = ops.token_log_probs_backward(z, tokens, r.lse, r.entropy, up, torch.where(up == 0, 0.0, 0.5))
    assert (grad[1:5] == 0).all() and grad[0].isfinite().all() and grad[5].isfinite().all()


@pytest.mark.parametrize("rows, vocab", LOGIT_SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_token_log_probs_backward(ops, rows, vocab, dtype):
    g = generator(rows * 149 + vocab)
    z = logits_of(g, rows, vocab, dtype, pad=vocab % 3)
    if vocab > 8:
        z[:, vocab - vocab // 8:] = -math.inf
    tokens = torch.randint(-1, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    up, up_h = (torch.randn(rows, generator=g, device="cuda") for _ in range(2))
    up[rows // 2] = 0.0
    for temperature, a, b in ((1.0, up, None), (0.7, up, up_h), (2.0, None, up_h)):
        r = ops.token_log_probs(z, tokens, temperature=temperature)
        got = ops.token_log_probs_backward(z, tokens, r.lse, r.entropy, a, b, temperature=temperature)
        want, p = rows64.token_log_probs_backward(z, tokens, a, b, temperature)
        wide = z.double() / temperature
        finite = torch.where(torch.isfinite(wide), wide, torch.zeros_like(wide)).abs().max(1, keepdim=True).values
        there = torch.zeros_like(want)
        inside = tokens >= 0
        there[inside, tokens[inside].long()] = 1.0
        # p is off by the errors of z / T - lse (4 |z| / T + 130 for lse) and of the exponential
        steps = 140.0 + 8 * finite
        # at the token g / T (1 - p): 1 / T is rounded, its product with g is, and the product with p <= 1 is: three
        # half steps of |g| / T; the rounding of the sum is that of the result
        size = 0.0 if a is None else a.double().abs()[:, None] * (p * steps + 3 * there)
        if b is not None:
            size = size + b.double().abs()[:, None] * p * (math.log(vocab) + 1 + finite) * (steps + 300)
        rows64.close(got, want, size / temperature, 1, "grad")
        again = z.clone()
        assert torch.equal(ops.token_log_probs_backward(again, tokens, r.lse, r.entropy, a, b, temperature=temperature,
                                                        out=again), got)


# ---- distillation ------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows, vocab", LOGIT_SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_distill_top(ops, rows, vocab, dtype):
    g = generator(rows * 151 + vocab)
    z = logits_of(g, rows, vocab, dtype, pad=vocab % 4)
    for top, temperature in ((1, 1.0), (5, 0.7), (64, 2.0), (128, 1.0)):
        # ids with repetitions, some outside the vocabulary, a row without any, a row without weight
        ids = torch.randint(-2, vocab + 2, (rows, top), generator=g, device="cuda", dtype=torch.int32)
        teacher = torch.randn(rows, top, generator=g, device="cuda") * 2
        teacher[:, top // 2] = -math.inf if top > 2 else 0.0
        weight = torch.randn(rows, generator=g, device="cuda")
        ids[rows // 2] = -1
        weight[rows // 3] = 0.0
        loss, grad = ops.distill_top(z, ids, teacher, temperature, weight)
        want_loss, want, q, p = rows64.distill_top(z, ids, teacher, weight, temperature)
        wide = z.double().abs().max(1).values / temperature
        t2 = temperature * temperature
        # q within (3 * 16 + 16) U, log p and log q within 130 + 8 |z| / T
        rows64.close(loss, want_loss, t2 * (400.0 + 16 * wide + 16 * math.log(vocab)), 1, "loss")
        at = torch.where((ids >= 0) & (ids < vocab), ids, 0).long()
        taken = torch.zeros_like(want).scatter_add(1, at, torch.where((ids >= 0) & (ids < vocab), q, 0.0))
        scale = (140.0 + 8 * wide)[:, None] * p + 140.0 * (weight.double().abs() * temperature)[:, None] * taken
        rows64.close(grad, want, scale, 1, "grad")
        assert torch.equal(ops.distill_top(z, ids, teacher, temperature, weight, grad=False)[0], loss)
        again = z.clone()
        loss2, grad2 = ops.distill_top(again, ids, teacher, temperature, weight, out=again)
        assert torch.equal(loss2, loss) and torch.equal(grad2, grad)


@pytest.mark.parametrize("vocab", [6, 600, 5000, 40000])
def test_distill_top_of_empty_and_invalid_rows(ops, vocab):
    g = generator(vocab)
    inf, nan = math.inf, math.nan
    z = rows_of(g, 7, vocab, torch.float32)
    ids = torch.tensor([[0, 1, 2]] * 7, dtype=torch.int32, device="cuda")
    teacher = torch.tensor([[1.0, 0.5, -inf]] * 7, device="cuda")
    z[1] = -inf             # a student row that holds nothing
    z[2, 1] = -inf          # a token the teacher wants is masked
    z[3, 2] = nan
    teacher[4] = -inf       # no entry has weight
    teacher[5, 0] = nan
    z[6] = nan              # padding
    weight = torch.tensor([1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 0.0], device="cuda")
    loss, grad = ops.distill_top(z, ids, teacher, 1.0, weight)
    want_loss, want, _, _ = rows64.distill_top(z, ids, teacher, weight, 1.0)
    assert loss[1] == inf and (grad[1] == 0).all()
    assert loss[2] == inf and grad[2].isfinite().all() and grad[2, 1] < 0
    assert loss[3].isnan() and grad[3].isnan().all()
    assert loss[4] == 0 and (grad[4] == 0).all()
    assert loss[5].isnan() and grad[5].isnan().all()
    assert (grad[6] == 0).all()
    for row in (0, 2):
        rows64.close(grad[row], want[row], 1.0, 300, "grad")
    rows64.close(loss[:1], want_loss[:1], 1.0, 500, "loss")


def test_loss_gradients_by_differences(ops):
    g = generator(9)
    z = rows_of(g, 2, 40, torch.float32, spread=1.5)
    tokens = torch.tensor([3, 39], dtype=torch.int32, device="cuda")
    ids = torch.tensor([[1, 5, 39], [0, 0, 7]], dtype=torch.int32, device="cuda")
    teacher = torch.tensor([[2.0, 1.0, 0.0], [0.5, 0.25, 1.0]], device="cuda")
    up, up_h = torch.tensor([0.7, -1.3], device="cuda"), torch.tensor([0.4, 0.9], device="cuda")
    t = 1.5

    def f(z):
        r = ops.token_log_probs(z, tokens, temperature=t)
        return float((r.log_prob.double() * up.double() + r.entropy.double() * up_h.double()).sum())

    def d(z):
        return float((ops.distill_top(z, ids, teacher, t, grad=False)[0].double() * up.double()).sum())
    r = ops.token_log_probs(z, tokens, temperature=t)
    grads = (ops.token_log_probs_backward(z, tokens, r.lse, r.entropy, up, up_h, temperature=t),
             ops.distill_top(z, ids, teacher, t, weight=up)[1])
    step = 2.0 ** -6
    bound = 2 * 500 * rows64.U * 4 / step + step * step  # both functions within 500 U, third derivatives below 6
    for fn, grad in zip((f, d), grads):
        for row, c in [(0, 1), (0, 3), (0, 39), (1, 0), (1, 20), (1, 39)]:
            up_z, down_z = z.clone(), z.clone()
            up_z[row, c] += step
            down_z[row, c] -= step
            assert abs((fn(up_z) - fn(down_z)) / (2 * step) - float(grad[row, c])) <= bound


@pytest.mark.parametrize("temperature", [0.03, 60.0])
@pytest.mark.parametrize("rows, vocab", [(5, 3001), (2, 70001)])
def test_sharp_and_flat_temperatures(ops, rows, vocab, temperature):
    g = generator(vocab)
    z = logits_of(g, rows, vocab, torch.float32)
    tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    check_log_probs(ops, z, tokens, 10, temperature)


def test_without_tokens_and_with_the_entropy_alone(ops):
    g = generator(21)
    z = logits_of(g, 6, 900, torch.float32)
    r = ops.token_log_probs(z, top=5)
    assert r.log_prob is None
    whole = ops.token_log_probs(z, torch.zeros(6, dtype=torch.int32, device="cuda"), top=5)
    for a, b in zip(r[1:], whole[1:]):
        assert torch.equal(a, b)
    up_h = torch.randn(6, generator=g, device="cuda")
    got = ops.token_log_probs_backward(z, None, r.lse, r.entropy, None, up_h)
    none = torch.full((6,), -1, dtype=torch.int32, device="cuda")
    assert torch.equal(got, ops.token_log_probs_backward(z, none, r.lse, r.entropy, None, up_h))
    want, p = rows64.token_log_probs_backward(z, none, None, up_h, 1.0)
    rows64.close(got, want, up_h.double().abs()[:, None] * p * (math.log(900) + 12) * 600, 1, "grad")


# ---- how they are called --------------------------------------------------------------------------
def test_shapes_and_workspaces(ops):
    g = generator(3)
    z = torch.randn(2, 3, 40000, generator=g, device="cuda")
    tokens = torch.randint(0, 40000, (2, 3), generator=g, device="cuda", dtype=torch.int32)
    r = ops.token_log_probs(z, tokens, top=4)
    flat = ops.token_log_probs(z.view(6, 40000), tokens.view(6), top=4)
    assert r.top_ids.shape == (2, 3, 4) and r.entropy.shape == (2, 3)
    for a, b in zip(r, flat):
        assert torch.equal(a.reshape(b.shape), b)
    one = ops.token_log_probs(z[0, 0], tokens[0, 0], top=4)
    assert one.lse.shape == () and torch.equal(one.top_ids, ops.token_log_probs(z[0, :1], tokens[0, :1], top=4).top_ids[0])
    need = ops.token_log_probs_workspace_nbytes(6, 40000, 4, torch.float32)
    assert need > 0
    lent = torch.full((need + 64,), 0xAB, dtype=torch.uint8, device="cuda")
    again = ops.token_log_probs(z, tokens, top=4, workspace=lent[:need])
    for a, b in zip(r, again):
        assert torch.equal(a, b)
    assert (lent[need:] == 0xAB).all()
    x = torch.randn(2, 5, 64, generator=g, device="cuda")
    y, mean, rstd = ops.layer_norm(x)
    dx, _, db = ops.layer_norm_backward(y, x, mean, rstd)
    assert y.shape == x.shape and mean.shape == (2, 5) and dx.shape == x.shape and db.shape == (64,)
    need = ops.layer_norm_backward_workspace_nbytes(10, 64, torch.float32)
    lent = torch.full((need + 64,), 0xAB, dtype=torch.uint8, device="cuda")
    assert torch.equal(ops.layer_norm_backward(y, x, mean, rstd, workspace=lent[:need])[2], db)
    assert (lent[need:] == 0xAB).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_is_written_outside_the_rows(ops, dtype):
    g = generator(4)
    for rows, n in [(5, 37), (3, 4001), (2, 40003), (600, 131)]:
        pad = 13
        whole = torch.full((rows + 2, n + pad), 3.0, dtype=dtype, device="cuda")
        out = whole[1:-1, 5:5 + n]
        z = logits_of(g, rows, n, dtype)
        tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
        ids = torch.randint(0, n, (rows, 3), generator=g, device="cuda", dtype=torch.int32)
        r = ops.token_log_probs(z, tokens)
        _, mean, rstd = ops.layer_norm(z)
        for call in (lambda: ops.layer_norm(z, out=out), lambda: ops.layer_norm_backward(z, z, mean, rstd, out=out),
                     lambda: ops.token_log_probs_backward(z, tokens, r.lse, r.entropy, r.lse, out=out),
                     lambda: ops.distill_top(z, ids, torch.zeros(rows, 3, device="cuda"), out=out)):
            whole.fill_(3.0)
            call()
            inside = out.clone()
            assert not (inside == 3.0).all()
            out.fill_(3.0)
            assert (whole == 3.0).all()


def test_rows_beyond_32_bit_offsets(ops):
    rows, vocab = 66000, 65536 + 8  # 4.3 G elements
    z = torch.empty(rows, vocab, dtype=torch.bfloat16, device="cuda")
    z.normal_(generator=generator(6))
    last = z[-600:]
    tokens = torch.randint(0, vocab, (rows,), generator=generator(7), device="cuda", dtype=torch.int32)
    ids = torch.randint(0, vocab, (rows, 4), generator=generator(8), device="cuda", dtype=torch.int32)
    teacher = torch.zeros(rows, 4, device="cuda")
    r, tail = ops.token_log_probs(z, tokens, top=3), ops.token_log_probs(last, tokens[-600:], top=3)
    for a, b in zip(r, tail):
        assert torch.equal(a[-600:], b)
    want = ops.distill_top(last, ids[-600:], teacher[-600:])
    want_grad = ops.token_log_probs_backward(last, tokens[-600:], tail.lse, tail.entropy, tail.entropy)
    want_y, mean, rstd = ops.layer_norm(last)
    want_dx = ops.layer_norm_backward(last, last, mean, rstd, bias=False)[0]
    out = torch.empty_like(z)
    assert torch.equal(ops.token_log_probs_backward(z, tokens, r.lse, r.entropy, r.entropy, out=out)[-600:], want_grad)
    loss, _ = ops.distill_top(z, ids, teacher, out=out)
    assert torch.equal(loss[-600:], want[0]) and torch.equal(out[-600:], want[1])
    _, mean, rstd = ops.layer_norm(z, out=out)
    assert torch.equal(out[-600:], want_y)
    ops.layer_norm_backward(z, z, mean, rstd, bias=False, out=out)
    assert torch.equal(out[-600:], want_dx)


@pytest.mark.parametrize("vocab, dtype", [(8650753, torch.float32), (9000001, torch.float32), (35000003, torch.bfloat16)])
def test_rows_of_very_many_stretches(ops, vocab, dtype):
    # hundreds of stretches a row: every one holds something, and their entries are more than are ranked at once
    z = logits_of(generator(vocab), 2, vocab, dtype)
    tokens = torch.tensor([vocab - 1, 0], dtype=torch.int32, device="cuda")
    check_log_probs(ops, z, tokens, 100, 1.0)
    ids = torch.tensor([[vocab - 1, 0, 7]] * 2, dtype=torch.int32, device="cuda")
    teacher = torch.tensor([[1.0, 0.5, 0.0]] * 2, device="cuda")
    loss, grad = ops.distill_top(z, ids, teacher)
    want_loss, want, _, p = rows64.distill_top(z, ids, teacher, None, 1.0)
    wide = float(z.double().abs().max())
    rows64.close(loss, want_loss, 400.0 + 16 * wide + 16 * math.log(vocab), 1, "loss")
    scale = (140.0 + 8 * wide) * p
    scale[:, [0, 7, vocab - 1]] += 140.0
    rows64.close(grad, want, scale, 1, "grad")


@pytest.mark.parametrize("rows, n", [((1 << 21) + 5, 3), ((1 << 20) + 3, 8200)])
def test_more_rows_than_a_launch_takes(ops, rows, n):
    # 2^21 workgroups a launch: one a row, or, in the gradient of the log probabilities, one a stretch of 4096
    g = generator(n)
    z = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    z.normal_(generator=g)
    tokens = torch.randint(0, n, (rows,), generator=g, device="cuda", dtype=torch.int32)
    ids = torch.randint(0, n, (rows, 2), generator=g, device="cuda", dtype=torch.int32)
    teacher = torch.randn(rows, 2, generator=g, device="cuda")
    r = ops.token_log_probs(z, tokens, top=2)
    loss, dz = ops.distill_top(z, ids, teacher)
    grad = ops.token_log_probs_backward(z, tokens, r.lse, r.entropy, r.entropy)
    y, mean, rstd = ops.layer_norm(z)
    for at in (slice(0, 5000), slice(rows // 2 - 2500, rows // 2 + 2500), slice(rows - 5000, rows)):
        part = ops.token_log_probs(z[at], tokens[at], top=2)
        for a, b in zip(r, part):
            assert torch.equal(a[at], b)
        part = ops.distill_top(z[at], ids[at], teacher[at])
        assert torch.equal(loss[at], part[0]) and torch.equal(dz[at], part[1])
        assert torch.equal(grad[at], ops.token_log_probs_backward(z[at], tokens[at], r.lse[at], r.entropy[at], r.entropy[at]))
        part = ops.layer_norm(z[at])
        assert torch.equal(y[at], part[0]) and torch.equal(mean[at], part[1]) and torch.equal(rstd[at], part[2])


def run_all(ops, z, x, gain, tokens, ids, teacher):
    y, mean, rstd = ops.layer_norm(x, gain, None)
    dx, dgain, dbias = ops.layer_norm_backward(y, x, mean, rstd, gain)
    r = ops.token_log_probs(z, tokens, top=10)
    grad = ops.token_log_probs_backward(z, tokens, r.lse, r.entropy, r.log_prob, r.entropy)
    loss, dz = ops.distill_top(z, ids, teacher, 2.0)
    return [y, mean, rstd, dx, dgain, dbias, *r, grad, loss, dz]


@pytest.mark.parametrize("rows, vocab", [(3, 20000), (700, 3001), (5, 70001)])
def test_equal_calls_captured_and_on_another_stream(ops, rows, vocab):
    g = generator(rows)
    z, x = rows_of(g, rows, vocab, torch.float32), rows_of(g, rows * 5, 320, torch.float32)
    gain = torch.rand(320, generator=g, device="cuda")
    tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    ids = torch.randint(0, vocab, (rows, 6), generator=g, device="cuda", dtype=torch.int32)
    teacher = torch.randn(rows, 6, generator=g, device="cuda")
    want = run_all(ops, z, x, gain, tokens, ids, teacher)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run_all(ops, z, x, gain, tokens, ids, teacher)
    busy = run_all(ops, z, x, gain, tokens, ids, teacher)  # at the same time, with workspaces of its own
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, busy):
        assert torch.equal(a, b) and torch.equal(a, c)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run_all(ops, z, x, gain, tokens, ids, teacher)
    first, first_x = z.clone(), x.clone()
    for turn in range(4):
        z.copy_(first * (1 + turn))
        x.copy_(first_x + turn)
        graph.replay()
        eager = run_all(ops, z, x, gain, tokens, ids, teacher)
        torch.cuda.synchronize()
        for a, b in zip(held, eager):
            assert torch.equal(a, b), turn


def test_front_refuses(ops):
    from motifcl_amd.lib import MccError
    z = torch.randn(4, 64, device="cuda")
    tokens = torch.zeros(4, dtype=torch.int32, device="cuda")
    row = torch.zeros(4, device="cuda")
    with pytest.raises(ValueError, match="device tensor"):
        ops.layer_norm(z.cpu())
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        ops.layer_norm(z.double())
    with pytest.raises(ValueError, match="contiguous rows"):
        ops.layer_norm(z.t())
    with pytest.raises(ValueError, match="gain: expected shape"):
        ops.layer_norm(z, torch.ones(63, device="cuda"))
    with pytest.raises(ValueError, match="expected dtype"):
        ops.layer_norm(z, torch.ones(64, device="cuda", dtype=torch.float64))
    with pytest.raises(ValueError, match="out: expected shape"):
        ops.layer_norm(z, out=z.half())
    with pytest.raises(MccError, match="y overlaps x"):
        ops.layer_norm(z[:3], out=z[1:])
    with pytest.raises(MccError, match="stride shorter"):
        ops.layer_norm(torch.randn(1, 64, device="cuda").expand(4, 64))
    with pytest.raises(MccError, match="non-zero dimensions"):
        ops.layer_norm(z[:0])
    with pytest.raises(ValueError, match="expected dtype"):
        ops.token_log_probs(z, tokens.long())
    with pytest.raises(MccError, match="alternatives"):
        ops.token_log_probs(z, tokens, top=65)
    with pytest.raises(MccError, match="alternatives"):
        ops.token_log_probs(torch.randn(2, 200, device="cuda"), top=129)
    with pytest.raises(MccError, match="alternatives"):
        ops.token_log_probs(z, tokens, top=-1)
    with pytest.raises(MccError, match="temperature"):
        ops.token_log_probs(z, tokens, temperature=0.0)
    with pytest.raises(MccError, match="no upstream"):
        ops.token_log_probs_backward(z, tokens, row, row, None)
    with pytest.raises(MccError, match="null buffer"):
        ops.token_log_probs_backward(z, None, row, row, row)
    with pytest.raises(ValueError, match="teacher_logits: expected shape"):
        ops.distill_top(z, tokens[:, None], torch.zeros(4, 2, device="cuda"))
    with pytest.raises(MccError, match="1 to 128"):
        ops.distill_top(z, torch.zeros(4, 129, dtype=torch.int32, device="cuda"), torch.zeros(4, 129, device="cuda"))
    with pytest.raises(MccError, match="workspace is too small"):
        ops.token_log_probs(torch.randn(2, 40000, device="cuda"), top=4,
                            workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))


def test_distillation_step_of_a_counter_layer(ops):
    """A student of norm, counter layer and head learns from a teacher's top log probabilities: the calls a training
    step makes, one after the other, against the same step in 64 bits."""
    g = generator(11)
    rows, width, vocab, top, C = 96, 64, 1000, 16, 11
    teacher_logits = logits_of(g, rows, vocab, torch.float32)
    teacher = ops.token_log_probs(teacher_logits, top=top)
    x = rows_of(g, rows, width, torch.float32)
    gain, bias = torch.rand(width, generator=g, device="cuda") + 0.5, torch.zeros(width, device="cuda")
    state = torch.empty(vocab * (width // 4) * 3, dtype=torch.uint8, device="cuda")
    ops.fill_counter_state(state, 5, 3 * (2 * C - 1))
    scale = torch.full((vocab,), 0.3, device="cuda")
    w = ops.decode_weight(state, scale, C, width, vocab).double()
    tokens = teacher.top_ids[:, 0].contiguous()

    h, mean, rstd = ops.layer_norm(x, gain, bias)
    logits = ops.forward(h, state, scale, C, vocab)
    loss, grad_logits = ops.distill_top(logits, teacher.top_ids, teacher.top_log_probs, 2.0,
                                        weight=torch.full((rows,), 1.0 / rows, device="cuda"))
    grad_h = ops.backward_input(grad_logits, state, scale, C, width)
    grad_x, grad_gain, grad_bias = ops.layer_norm_backward(grad_h, x, mean, rstd, gain)
    before = ops.token_log_probs(logits, tokens)

    leaves = [t.double().requires_grad_() for t in (x, gain, bias)]
    d = leaves[0] - leaves[0].mean(1, keepdim=True)
    out = d / (d.square().mean(1, keepdim=True) + 1e-5).sqrt() * leaves[1] + leaves[2]
    z = out @ w.t()
    q = torch.softmax(teacher.top_log_probs.double() / 2.0, 1)
    log_p = (z / 2.0).log_softmax(1)
    picked = torch.stack([log_p[i, teacher.top_ids[i].long()] for i in range(rows)])
    want_loss = 4.0 * (q * (q.log() - picked)).sum(1)
    want = torch.autograd.grad(want_loss.mean(), leaves)
    # logits are sums of 64 products (|z| <= 40), so within 64 U of 64; everything behind is smooth in them
    rows64.close(loss, want_loss.detach(), 40.0, 1000, "loss")
    for got, exact in zip((grad_x, grad_gain, grad_bias), want):
        rows64.close(got, exact, exact.abs().max() + 1.0 / rows, 4000, "gradient")
    assert (before.log_prob.double() - z.detach().log_softmax(1).gather(1, tokens.long()[:, None])[:, 0]).abs().max() < 1e-3

    v, m = torch.zeros(vocab, device="cuda"), [torch.zeros(width, device="cuda") for _ in range(4)]
    ws = torch.empty(ops.fused_workspace_nbytes(width, vocab, rows), dtype=torch.uint8, device="cuda")
    kept = state.clone()
    ops.apply_update_fused(state, scale, v, grad_logits, h, ws, C, 3e-3, 0.0, 0.9, 1e-3, 1)
    ops.adam_update(gain, grad_gain, m[0], m[1], 1e-2, 0.9, 0.999, 1e-8, 1)
    ops.adam_update(bias, grad_bias, m[2], m[3], 1e-2, 0.9, 0.999, 1e-8, 1)
    assert not torch.equal(state, kept) and v.isfinite().all() and (v > 0).any() and gain.isfinite().all()
