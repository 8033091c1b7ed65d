"""The distillation loss at the smallest temperatures that are accepted, where temperature^2 and the logits over the
temperature leave the range of binary32 though the loss does not."""
import pytest

from . import rows64
from .test_gpu_row_ops import ops  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("temperature", [1e-3, 1e-21, 1e-30, 2e-38])
@pytest.mark.parametrize("vocab", [50, 40000])
def test_distillation_at_small_temperatures(ops, vocab, temperature):
    g = torch.Generator(device="cuda").manual_seed(vocab)
    z = 3.0 * torch.randn(4, vocab, generator=g, device="cuda")
    ids = torch.randint(0, vocab, (4, 6), generator=g, device="cuda", dtype=torch.int32)
    teacher = torch.randn(4, 6, generator=g, device="cuda")
    weight = torch.rand(4, generator=g, device="cuda") + 0.5
    # the temperature as the kernels have it
    temperature = float(torch.tensor(temperature, dtype=torch.float32))
    loss, grad = ops.distill_top(z, ids, teacher, temperature, weight)
    want_loss, want, q, p = rows64.distill_top(z, ids, teacher, weight, temperature)
    # T log q and T log p are a difference, T's product with a logarithm (within 130 U as everywhere) and their
    # difference; 6 terms of at most the largest difference of logits; T's product
    largest = (z.double().max(1).values[:, None] - z.double()).max(1).values + 2 * teacher.double().abs().max(1).values
    rows64.close(loss, want_loss, temperature * (largest * 20 + temperature * 400), 1, "loss")
    # p and q are 0 or 1 but for logits within a few temperatures of the largest; |d| U at T = 1e-3, where d <= 20 counts
    scale = (weight.double() * temperature)[:, None] * (400.0 * torch.ones_like(want))
    rows64.close(grad, want, scale, 1, "grad")
