"""GPU: the 8-bit checkpoint layers where values are not finite."""
import pytest
import torch

from test_act8_gpu import make

pytestmark = pytest.mark.gpu

# sizes of every weight-gradient kernel: both gradients in one, 64 x 64, 64 x 32, 32 x 64 tiles, 128 x 128
SIZES = [(2, 40, 300, 24), (2, 100, 300, 80), (2, 20, 300, 100), (2, 100, 300, 20), (17, 130, 4100, 200)]


def finite(t):
    return bool(torch.isfinite(t).all())


@pytest.mark.parametrize("mode", ["batch", "frozen"])
@pytest.mark.parametrize("B,K,L,N", SIZES)
def test_nan_in_a_norms_parameters(B, K, L, N, mode):
    """a NaN of gamma or beta is in every value of its channel, and with them in the channel's weight gradients; no other channel has it"""
    from pointcloudsegmentation_amd import quant
    for which in ("weight", "bias"):
        x, W, b, g, norm = make(B, K, L, N, True)
        norm.train(mode == "batch")
        with torch.no_grad():
            getattr(norm, which)[3] = float("nan")
        h = quant.act8_linear(x, W, b, norm=norm)
        assert bool(torch.isnan(h).all())
        dx, dW, db, dgamma, dbeta = torch.autograd.grad(h, [x, W, b, norm.weight, norm.bias], g)
        assert bool(torch.isnan(dW[:, 3]).all()), which
        keep = torch.arange(K, device="cuda") != 3
        assert finite(dW[:, keep]) and finite(db) and finite(dx[:, keep]) and finite(dgamma[keep]) and finite(dbeta)
        assert bool(torch.isnan(dx[:, 3]).all()) == (which == "weight")


@pytest.mark.parametrize("B,K,L,N", SIZES)
def test_a_channel_switched_off_by_minus_infinity(B, K, L, N):
    """beta = -inf: ReLU leaves zeros, so the channel has no weight gradient and gives none on"""
    from pointcloudsegmentation_amd import quant
    x, W, b, g, norm = make(B, K, L, N, True)
    with torch.no_grad():
        norm.bias[3] = -float("inf")
    h = quant.act8_linear(x, W, b, norm=norm)
    dx, dW, dgamma, dbeta = torch.autograd.grad(h, [x, W, norm.weight, norm.bias], g)
    assert finite(h) and finite(dx) and finite(dW)
    assert bool((dW[:, 3] == 0).all()) and bool((dx[:, 3] == 0).all()) and dgamma[3] == 0 and dbeta[3] == 0


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("B,K,L,N", SIZES)
def test_frozen_statistics_keep_a_bad_point_to_itself(B, K, L, N, value):
    """with frozen statistics dx = gamma r dy: a point that is not finite changes no other point's gradient, though it shares its scale"""
    from pointcloudsegmentation_amd import quant
    x, W, b, g, norm = make(B, K, L, N, True)
    norm.eval()
    clean, = torch.autograd.grad(quant.act8_linear(x, W, b, norm=norm), [x], g)
    cleany, = torch.autograd.grad(quant.act8_norm_relu(x, norm), [x], clean)
    with torch.no_grad():
        x[1, 3, 200] = value
    keep = torch.ones_like(x, dtype=torch.bool)
    keep[1, 3, 200] = False
    dx, = torch.autograd.grad(quant.act8_linear(x, W, b, norm=norm), [x], g)
    assert torch.equal(dx[keep], clean[keep])
    dy, = torch.autograd.grad(quant.act8_norm_relu(x, norm), [x], clean)
    assert torch.equal(dy[keep], cleany[keep])
