"""The float64 statements behind the token operators' GPU tests: gradients against central differences,
the corners that the kernels' documentation names (CPU)."""
import numpy as np
import pytest

from oracle import categorical as ocat
from oracle import grad_clip as oclip
from oracle import layer_norm as oln


def _differences(f, x, h=1e-5):
    d = np.zeros_like(x)
    flat, out = x.reshape(-1), d.reshape(-1)
    for i in range(flat.size):
        keep = flat[i]
        flat[i] = keep + h
        up = f()
        flat[i] = keep - h
        out[i] = (up - f()) / (2 * h)
        flat[i] = keep
    return d


@pytest.mark.parametrize("temperature", [1.0, 0.6])
@pytest.mark.parametrize("masked", [False, True])
def test_categorical_gradient_vs_differences(temperature, masked):
    rng = np.random.RandomState(0)
    x = rng.randn(5, 7) * 2
    act = np.array([0, 3, 6, -1, 2])
    mask = None
    if masked:
        mask = rng.rand(5, 7) < 0.6
        mask[np.arange(5), np.maximum(act, 0)] = True
        mask[4] = False
        act[4] = 2
    g, h = rng.randn(5), rng.randn(5)

    def loss():
        lp, en, *_ = ocat.forward(x, act, mask, temperature)
        lp = np.where(np.isfinite(lp), lp, 0.0)
        return float((g * lp + h * en).sum())

    # central differences of a smooth function: error h^2 |f'''| / 6 + 2^-52 |f| / h < 1e-8
    np.testing.assert_allclose(ocat.gradient(x, act, g, h, mask, temperature),
                               _differences(loss, x), atol=1e-8)


def test_layer_norm_gradient_vs_differences():
    rng = np.random.RandomState(1)
    x, gamma, beta, dy = rng.randn(4, 6), 1 + 0.2 * rng.randn(6), rng.randn(6), rng.randn(4, 6)

    def loss():
        return float((dy * oln.forward(x, gamma, beta)[0]).sum())

    dx, dg, db = oln.backward(dy, x, gamma)
    np.testing.assert_allclose(dx, _differences(loss, x), atol=1e-8)
    np.testing.assert_allclose(dg, _differences(loss, gamma), atol=1e-8)
    np.testing.assert_allclose(db, _differences(loss, beta), atol=1e-8)


def test_categorical_corners():
    inf, nan = np.inf, np.nan
    x = np.array([[1.0, 2.0, 2.0], [-inf, -inf, -inf], [0.0, nan, 0.0], [0.0, inf, 1.0],
                  [1.0, 1.0, 1.0], [0.0, -inf, 0.0]])
    mask = np.ones((6, 3), bool)
    mask[4] = False
    lp, en, ids, top, _ = ocat.forward(x, np.array([0, 0, 0, 0, 0, 1]), mask, 1.0, 2)
    assert ids.tolist() == [[1, 2], [-1, -1], [-1, -1], [-1, -1], [-1, -1], [0, 2]]
    assert lp[1] == -inf and lp[4] == -inf and lp[5] == -inf
    assert np.isnan(lp[2]) and np.isnan(lp[3]) and np.isnan(en[2])
    assert en[1] == 0 and en[4] == 0
    np.testing.assert_allclose(en[5], np.log(2.0), rtol=1e-15)


def test_clip_statements():
    t = [np.array([3.0]), np.array([0.0, 4.0]), np.zeros((0,))]
    got, norm = oclip.clip_by_global_norm(t, 2.5)
    assert norm == 5.0 and got[0][0] == 1.5 and got[1][1] == 2.0
    got, norms = oclip.clip_by_norms(t, 3.5)
    assert norms.tolist() == [3.0, 4.0, 0.0] and got[0][0] == 3.0 and got[1][1] == 3.5
    assert np.isnan(oclip.clip_by_global_norm([np.array([np.inf, 1.0])], 1.0)[0][0]).all()
