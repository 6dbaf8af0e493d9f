"""The 64-bit formulas that the GPU tests compare with, against central differences of what they differentiate."""
import pytest
import torch

from tests import dense_helpers as H

STEP = 1e-6
# a central difference in 64 bits is off by STEP^2 |f'''| / 6 and eps64 |f| / STEP: below 1e-9 of sizes around 1
CLOSE = 2e-8


def difference(f, x):
    out = torch.zeros_like(x)
    flat, grad = x.view(-1), out.view(-1)
    for i in range(flat.numel()):
        keep = float(flat[i])
        flat[i] = keep + STEP
        up = float(f())
        flat[i] = keep - STEP
        grad[i] = (up - float(f())) / (2 * STEP)
        flat[i] = keep
    return out


@pytest.mark.parametrize("name", ["none", "relu", "gelu", "silu"])
def test_slopes(name):
    z = torch.linspace(-6.03, 6.01, 301, dtype=torch.float64)   # (not through relu's corner)
    slope = (H.act(z + STEP, name) - H.act(z - STEP, name)) / (2 * STEP)
    assert float((H.slope(z, name) - slope).abs().max()) < CLOSE


def test_epilogue_gradient():
    g = torch.Generator().manual_seed(1)
    z, dy, bias = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((3, 4), (3, 4), (4,)))
    (dz, _), (dbias, _) = H.epilogue_grad(dy, z + bias, "gelu", "f32")
    assert float((difference(lambda: (H.act(z + bias, "gelu") * dy).sum(), z) - dz).abs().max()) < CLOSE
    assert float((difference(lambda: (H.act(z + bias, "gelu") * dy).sum(), bias) - dbias).abs().max()) < CLOSE


def test_layer_norm_gradient():
    g = torch.Generator().manual_seed(2)
    x, dy, r = (torch.randn((3, 7), generator=g, dtype=torch.float64) for _ in range(3))
    gamma, beta = (torch.randn((7,), generator=g, dtype=torch.float64) for _ in range(2))

    def objective():   # y's part, and x's own on the residual stream
        return (H.layer_norm(x, gamma, beta, 1e-3, "f32")[0][0] * dy).sum() + (x * r).sum()

    (_, _), (mean, _), (rstd, _) = H.layer_norm(x, gamma, beta, 1e-3, "f32")
    (dx, _), (dgamma, _), (dbeta, _) = H.layer_norm_grad(dy, x, gamma, mean, rstd, r, "f32")
    for variable, grad in ((x, dx), (gamma, dgamma), (beta, dbeta)):
        assert float((difference(objective, variable) - grad).abs().max()) < CLOSE


@pytest.mark.parametrize("sigmoid", [False, True])
def test_balance_gradient(sigmoid):
    g = torch.Generator().manual_seed(3)
    x = torch.randn((6, 5), generator=g, dtype=torch.float64)
    ids = torch.tensor([[0, 1], [1, 2], [-1, -1], [1, 4], [1, -1], [9, 1]])
    counts, (loss, _), (grad, _) = H.balance(x, ids, sigmoid, 0.7, 1.3, "f32")
    assert counts.tolist() == [1, 5, 1, 0, 1]
    found = difference(lambda: 1.3 * H.balance(x, ids, sigmoid, 0.7, 1.0, "f32")[1][0], x)
    assert float((found - grad).abs().max()) < CLOSE
    assert float(loss) > 0.7   # (an uneven load of the likelier experts costs more than an even one)


def test_even_load_costs_the_coefficient():
    x = torch.zeros((8, 4), dtype=torch.float64)
    ids = torch.arange(8).reshape(8, 1) % 4
    _, (loss, _), (grad, _) = H.balance(x, ids, False, 0.25, 1.0, "f32")
    assert float(loss) == pytest.approx(0.25, abs=1e-15) and float(grad.abs().max()) == 0
