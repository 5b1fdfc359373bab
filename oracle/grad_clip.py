"""float64 numpy statement of tf.clip_by_global_norm and tf.clip_by_norm per tensor (TEST
INFRASTRUCTURE).  A norm that is not finite makes what it scales NaN."""
import numpy as np


def _scale(norm, clip):
    return np.nan if not np.isfinite(norm) else 1.0 if norm <= clip else clip / norm


def clip_by_global_norm(tensors, clip):
    ts = [np.asarray(t, np.float64) for t in tensors]
    norm = np.sqrt(sum((t * t).sum() for t in ts))
    return [t * _scale(norm, clip) for t in ts], norm


def clip_by_norms(tensors, clip):
    ts = [np.asarray(t, np.float64) for t in tensors]
    norms = np.array([np.sqrt((t * t).sum()) for t in ts])
    return [t * _scale(n, clip) for t, n in zip(ts, norms)], norms
