"""Layer norm whose input and summand nearly cancel: the sum is taken first, as it is exact (both have about the same magnitude), and only then the
mean, in the forward and in every form of the backward pass."""
import pytest
import torch

from tests.test_gpu_layernorm_training import near, reference, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,channels", [(40, 64), (30, 256), (30, 400), (20, 1024), (20, 1001), (9, 2048), (7, 4096), (5, 8192), (5, 8191), (3, 9000)])
def test_a_summand_that_cancels(ctx, rows, channels):
    """x and ext are about 1e4 and their sum about 1, with x's last digits worth 2^-10 each.  The sum is exact in fp32, so the tolerances are those of an input
    of that size without a summand (test_gpu_layernorm_training.py)."""
    gen = torch.Generator(device="cuda").manual_seed(channels)
    x = torch.randn((rows, channels), device="cuda", generator=gen) * 100 + 1.0e4
    s = torch.randn((rows, channels), device="cuda", generator=gen) * 1.5 + 0.25
    ext = s - x
    w, b, dy = torch.rand(channels, device="cuda", generator=gen) + 0.5, torch.randn(channels, device="cuda", generator=gen), torch.randn((rows, channels), device="cuda", generator=gen)
    assert torch.equal((x + ext).double(), x.double() + ext.double())
    y, stats, dx, dw, db = run(ctx, x, ext, w, b, dy, torch.float32)
    wy, ws, wdx, dw_terms, db_terms = reference(x, ext, w, b, dy)
    near(y, wy, torch.float32)
    near(stats, ws, torch.float32)
    near(dx, wdx, torch.float32, magnitude=(ws[:, 1:] * dy.double().abs().amax(1, keepdim=True) * 4).clamp(min=1e-30))
    for got, terms in ((dw, dw_terms), (db, db_terms)):
        assert bool(((got.double() - terms.sum(0)).abs() <= (rows + 32) * 2.0 ** -24 * terms.abs().sum(0) + 1e-5 * terms.abs().amax(0) + 1e-30).all())
