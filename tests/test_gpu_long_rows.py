"""The row-wise operators on rows, vocabularies and batches far longer than a workgroup's registers.

A rounding of binary32 is U = 2^-24 of the value; `steps` below counts the roundings on the longest path of a sum."""
import math

import pytest

from . import rows64
from .test_gpu_row_ops import ops  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def test_column_gradients_of_the_widest_rows(ops):
    # from 2^27 columns on one launch does not hold the threads that join the partial rows
    cols = (1 << 27) + 5
    g = torch.Generator(device="cuda").manual_seed(3)
    x, dy = (torch.randn(2, cols, generator=g, device="cuda") for _ in range(2))
    gain = torch.ones(cols, device="cuda")
    mean, rstd = torch.tensor([0.25, -0.5], device="cuda"), torch.tensor([0.75, 1.25], device="cuda")
    _, dgain, dbias = ops.layer_norm_backward(dy, x, mean, rstd, gain, input_grad=False)
    for at in (slice(0, 1 << 20), slice((1 << 26) - 70, (1 << 26) + 70), slice(cols - (1 << 20), cols)):
        xhat = (x[:, at].double() - mean.double()[:, None]) * rstd.double()[:, None]
        near = (x[:, at].double().abs() + mean.double().abs()[:, None]) * rstd.double()[:, None]
        d = dy[:, at].double()
        # x - mean, its product with rstd, the product with dy, the sum of the two rows
        rows64.close(dgain[at], (d * xhat).sum(0), (d.abs() * near).sum(0), 4, "dgain")
        rows64.close(dbias[at], d.sum(0), d.abs().sum(0), 1, "dbias")


# Sums of a row that a workgroup's registers do not hold: a thread's own is rounded once, then a tree of 6 + 6 joins, the
# rounded 1 / n and its product: at most 16 U of the mean magnitude, whatever the length.
LONG_SUM = 16


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("spread", [0.0, 2.0 ** -5])
def test_norm_of_long_rows_far_from_zero(ops, dtype, spread):
    rows, cols, eps = 2, (1 << 22) + 3, 1e-5
    g = torch.Generator(device="cuda").manual_seed(cols)
    x = (1.1 + spread * torch.randn(rows, cols, generator=g, device="cuda")).to(dtype)
    y, mean, rstd = ops.layer_norm(x, None, None, eps)
    want, want_mean, want_rstd = rows64.layer_norm(x, None, None, eps)
    largest = x.double().abs().max(1).values
    rows64.close(mean, want_mean, largest, LONG_SUM, "mean")
    # a difference is off by the mean's error and its own rounding, the variance by twice that against the deviation,
    # by its square (small here: below 2^-12 of itself, where the deviation is 0 it is compared with eps) and its sum
    slack = (LONG_SUM + 1) * rows64.U * largest * want_rstd
    relative = (LONG_SUM + 6) * rows64.U + 2 * slack
    assert ((rstd.double() - want_rstd).abs() <= want_rstd * relative).all()
    scale = (x.double() - want_mean[:, None]).abs() * want_rstd[:, None]
    rows64.close(y, want, (scale * (relative[:, None] + 4 * rows64.U) + slack[:, None]) / rows64.U, 1, "y")


def test_norm_gradient_of_long_rows_far_from_zero(ops):
    rows, cols = 2, (1 << 22) + 3
    g = torch.Generator(device="cuda").manual_seed(cols)
    x = torch.randn(rows, cols, generator=g, device="cuda")
    dy = torch.full_like(x, 0.7)  # equal numbers round the same way every time
    _, mean, rstd = ops.layer_norm(x)
    dx, _, _ = ops.layer_norm_backward(dy, x, mean, rstd, bias=False)
    want, _, _ = rows64.layer_norm_backward(dy, x, mean, rstd, None)
    near = (x.double().abs() + mean.double().abs()[:, None]) * rstd.double()[:, None]
    h = dy.double().abs()
    # xhat within 3 U of |x| + |mean|; h - a - xhat b and its product with rstd: 5 roundings
    scale = rstd.double()[:, None] * (h + h.mean(1, keepdim=True) + near * (h * near).mean(1, keepdim=True))
    rows64.close(dx, want, scale, LONG_SUM + 10, "dx")


def test_column_gradients_of_many_long_rows(ops):
    # 1024 rows to each partial row of a matrix wider than the registers
    rows, cols = 1 << 16, 16392
    x = torch.ones(rows, cols, device="cuda")
    dy = torch.full_like(x, 0.7)
    mean, rstd = torch.full((rows,), 0.25, device="cuda"), torch.full((rows,), 0.75, device="cuda")
    _, dgain, dbias = ops.layer_norm_backward(dy, x, mean, rstd, torch.ones(cols, device="cuda"), input_grad=False)
    total = torch.full((cols,), float(dy[0, 0]) * rows, device="cuda", dtype=torch.float64)
    # the thread's sum is rounded once, the partial rows are added in two steps and 31
    rows64.close(dbias, total, total, 34, "dbias")
    rows64.close(dgain, 0.5625 * total, total, 36, "dgain")


def test_distillation_of_rows_of_equal_logits(ops):
    # 534 stretches of 65536: one running sum of equal numbers in binary32 would be off by thousands of roundings
    vocab, rows = 35000003, 2
    z = torch.full((rows, vocab), -0.357, device="cuda", dtype=torch.bfloat16)
    z[:, :65536] = 0.0  # every thread's largest
    ids = torch.tensor([[5, vocab - 1]] * rows, dtype=torch.int32, device="cuda")
    loss, grad = ops.distill_top(z, ids, torch.zeros(rows, 2, device="cuda"))
    want_loss, want, _, _ = rows64.distill_top(z, ids, torch.zeros(rows, 2, device="cuda"), None, 1.0)
    # e^d with |d| < 1 is off by 7 U, a thread's 64 of them by 64 U, 12 joins, the rescaling: s within 90 U of itself;
    # log p by that, the rounding of log s (18 U at most) and of their difference
    rows64.close(loss, want_loss, 1.0, 150, "loss")
    # p = e^d / s, rounded with T, q and the product; at the two entries q is subtracted
    entries = torch.zeros(vocab, dtype=torch.float64, device="cuda")
    entries[ids[0].long()] = 1.0
    rows64.close(grad, want, want.abs() + entries, 105, "grad")


def test_log_probs_of_the_most_stretches(ops):
    # 16385 stretches of nearly equal sums
    vocab = (1 << 29) + 3
    z = torch.full((1, vocab), -0.5, device="cuda")
    z[:, ::16384] = 0.0  # every stretch's largest
    tokens = torch.tensor([vocab - 1], dtype=torch.int32, device="cuda")
    r = ops.token_log_probs(z, tokens)
    ones = (vocab + 16383) // 16384
    e = math.exp(-0.5)
    s, u = ones + (vocab - ones) * e, -0.5 * (vocab - ones) * e
    # a stretch's s and u: e^d within 6 U, a thread's 32 of them 32 U, 12 joins; then log s (20 at most) and its sum
    for got, want in ((r.lse, math.log(s)), (r.log_prob, -0.5 - math.log(s)), (r.entropy, math.log(s) - u / s)):
        assert abs(float(got[0]) - want) <= (2 * 50 + 2 * 21) * rows64.U


def test_column_gradients_of_very_many_rows(ops):
    # 33 million rows: no thread adds more than 256 of them up in binary32
    rows, cols = (1 << 25) + 3, 16
    x = torch.ones(rows, cols, device="cuda")
    dy = torch.full_like(x, 0.7)
    mean, rstd = torch.full((rows,), 0.25, device="cuda"), torch.full((rows,), 0.75, device="cuda")
    _, dgain, dbias = ops.layer_norm_backward(dy, x, mean, rstd, torch.ones(cols, device="cuda"), input_grad=False)
    total = torch.full((cols,), float(dy[0, 0]) * rows, device="cuda", dtype=torch.float64)
    # a thread's 256 rows, three joins of a workgroup's eight, the products; the partial rows' sum is rounded once
    rows64.close(dbias, total, total, 259, "dbias")
    rows64.close(dgain, 0.5625 * total, total, 261, "dgain")
