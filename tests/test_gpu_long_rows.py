"""The row-wise operators on rows, vocabularies and batches far longer than a workgroup's registers.

A rounding of binary32 is U = 2^-24 of the value; `steps` below counts the roundings on the longest path of a sum."""
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
