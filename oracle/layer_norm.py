"""float64 numpy statement of layer normalisation over the last axis and its gradient (TEST
INFRASTRUCTURE): keras LayerNormalization, biased variance."""
import numpy as np


def forward(x, gamma=None, beta=None, epsilon=1e-3):
    x = np.asarray(x, np.float64)
    mean = x.mean(-1, keepdims=True)
    rstd = 1.0 / np.sqrt(((x - mean) ** 2).mean(-1, keepdims=True) + epsilon)
    y = (x - mean) * rstd
    if gamma is not None:
        y = y * np.asarray(gamma, np.float64)
    if beta is not None:
        y = y + np.asarray(beta, np.float64)
    return y, mean[..., 0], rstd[..., 0]


def backward(dy, x, gamma=None, epsilon=1e-3):
    """(dx, dgamma, dbeta) of sum(dy * y)."""
    x, dy = np.asarray(x, np.float64), np.asarray(dy, np.float64)
    h, _, rstd = forward(x, None, None, epsilon)
    g = dy if gamma is None else dy * np.asarray(gamma, np.float64)
    dx = rstd[..., None] * (g - g.mean(-1, keepdims=True) - h * (g * h).mean(-1, keepdims=True))
    rows = tuple(range(x.ndim - 1))
    return dx, (dy * h).sum(rows), dy.sum(rows)
