"""Layer normalisation of constant rows: y is beta up to the mean's own roundings.

A row's sum is a tree over at most 16 elements a lane, 64 lanes and 16 waves (wider rows: one more addition
for every 16384 columns and element): at most `chain` additions one behind another, each off by u = 2^-24 of
its result, then a quotient; so |mean - x| <= (chain + 1) u |x| =: e, and the centred values are e in
size (their difference is exact: mean and x are neighbours).  The variance is e^2, so for epsilon >> e^2 the
normalised value is at most e / sqrt(epsilon), with two more roundings.
"""
import pytest
import torch

from agents_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("value", [0.1, 100.1, -3000.7, 2.0])
@pytest.mark.parametrize("width", [7, 37, 1000, 4099, 9001, 20011])
def test_constant_rows(dev, value, width):
    x = torch.full((5, width), value, device=dev)
    gen = torch.Generator(device=dev).manual_seed(1)
    gamma, beta = torch.randn(width, generator=gen, device=dev), torch.randn(width, generator=gen, device=dev)
    y, stats = ops.layer_norm_forward(x, gamma, beta, 1e-3)
    exact = float(x[0, 0])
    e = (16 + 6 + 16 + 16 * (width / 16384.0) + 1) * U * abs(exact)
    assert float((stats[:, 0].double() - exact).abs().max()) <= e
    off = (y.double() - beta.double()).abs()
    tol = e / 1e-3 ** 0.5 * gamma.double().abs() * (1 + 4 * U) + 2 * U * beta.double().abs()
    assert bool((off <= tol).all()), float((off / tol).max())
    print(f"value {value} width {width}: mean off by {float((stats[:, 0].double() - exact).abs().max()):.3g}, "
          f"y - beta at most {float((off / gamma.double().abs()).max()):.3g} gamma")
