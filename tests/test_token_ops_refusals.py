"""Arguments that the token operators refuse before anything reaches the device (CPU)."""
import ctypes

import pytest
import torch

from agents_amd import _lib, ops


pytestmark = pytest.mark.usefixtures("lib")


def bad(fn, *a, **kw):
    with pytest.raises((ValueError, _lib.AgentsAmdError)):
        fn(*a, **kw)


def test_categorical_refusals():
    f = ops.categorical_log_prob
    x, a = torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64)
    bad(f, x, a)                                              # host tensors
    bad(f, x.double(), a)
    bad(f, x[0], a[0])
    bad(f, torch.zeros(3, 0), a)
    bad(f, torch.zeros(5, 3).t(), torch.zeros(3, dtype=torch.int64))
    bad(f, x, a.float())
    bad(f, x, a[:2])
    bad(f, x, a, mask=torch.ones(3, 5))
    bad(f, x, a, mask=torch.ones(3, 1, dtype=torch.bool))
    bad(f, x, a, mask=torch.ones(2, 5, dtype=torch.bool))
    bad(f, x, a, mask=torch.ones(1, 3, 5, dtype=torch.bool))
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-31):
        bad(f, x, a, temperature=t)
    bad(f, x, a, top_k=65)
    bad(f, x, a, top_k=-1)
    y = torch.zeros(2, 3, 4, 5).permute(2, 0, 1, 3)[::2]
    bad(f, y, torch.zeros(2, 2, 3, dtype=torch.int64))
    r = ops.CategoricalLogProb(torch.zeros(3), torch.zeros(3), None, None, torch.zeros(3, 2))
    g = ops.categorical_log_prob_backward
    bad(g, x, a, r)
    bad(g, x, None, r, torch.zeros(3))
    bad(g, x, a, r, torch.zeros(3).double())
    bad(g, x, a, r, torch.zeros(2))
    bad(g, x, a, r._replace(stats=torch.zeros(3, 3)), torch.zeros(3))
    bad(g, x, a, r, torch.zeros(3), out=torch.zeros(3, 5).half())


def test_clip_refusals():
    for f in (ops.clip_by_global_norm, ops.clip_by_norms):
        bad(f, [], 1.0)
        bad(f, [torch.zeros(3)], 0.0)
        bad(f, [torch.zeros(3)], float("nan"))
        bad(f, [torch.zeros(3)], 1.0)                         # host tensors
        bad(f, [torch.zeros(3, dtype=torch.int32)], 1.0)
        bad(f, [torch.zeros(3), torch.zeros(3).half()], 1.0)
        bad(f, [torch.zeros(3, 4).t()], 1.0)


def test_layer_norm_refusals():
    x, w = torch.zeros(3, 5), torch.zeros(5)
    f, g, st = ops.layer_norm_forward, ops.layer_norm_backward, torch.zeros(3, 2)
    bad(f, x, w, w)                                           # host tensors
    bad(f, x.double(), w, w)
    bad(f, x[0], w, w)
    bad(f, x, w[:4], w)
    bad(f, x, w, w.half())
    bad(f, x, w, w, epsilon=-1.0)
    bad(f, x, w, w, epsilon=float("nan"))
    bad(f, x, w, w, out=torch.zeros(3, 5).half())
    bad(f, torch.zeros(5, 3).t(), torch.zeros(3), torch.zeros(3))
    bad(g, x.half(), x, w, st)
    bad(g, x, x, w, torch.zeros(2, 2))
    bad(g, x, x, w, st, param_grads=False, input_grad=False)
    bad(g, x, x, w, st, dgamma=torch.zeros(4))


def test_entry_points_refuse(lib):
    """The C entries check what they are given before any launch."""
    d = _lib.CategoricalDesc(rows=1, inner=1, vocab=5, logits=64, action_bytes=8, temperature=1.0)
    w = lib.aa_categorical_workspace_bytes
    assert w(ctypes.byref(d)) == 0
    big = _lib.CategoricalDesc(rows=1, inner=1, vocab=100000, logits=64, temperature=1.0)
    assert w(ctypes.byref(big)) > 0
    assert lib.aa_categorical_log_prob(ctypes.byref(big), None, 0, None) == -34
    for k, v in (("rows", 0), ("vocab", 0), ("inner", 0), ("logits", None), ("dtype", 3), ("dtype", -1),
                 ("top_k", 6), ("top_k", -1), ("temperature", 0.0)):
        b = _lib.CategoricalDesc.from_buffer_copy(d)
        setattr(b, k, v)
        assert w(ctypes.byref(b)) == -1, k
        assert lib.aa_categorical_log_prob(ctypes.byref(b), None, 0, None) == -22, k
    b = _lib.CategoricalDesc.from_buffer_copy(d)
    b.actions = 64                                            # without log_prob
    assert lib.aa_categorical_log_prob(ctypes.byref(b), None, 0, None) == -22
    b.log_prob, b.action_bytes = 64, 2
    assert lib.aa_categorical_log_prob(ctypes.byref(b), None, 0, None) == -22
    b.action_bytes, b.mask, b.mask_bytes = 8, 64, 2
    assert lib.aa_categorical_log_prob(ctypes.byref(b), None, 0, None) == -22
    assert lib.aa_categorical_log_prob_backward(ctypes.byref(d), None, None, 64, 5, 0, None) == -22
    n = (ctypes.c_int64 * 2)(3, -1)
    p = (ctypes.c_void_p * 2)(64, 64)
    assert lib.aa_clip_tensors_workspace_bytes(n, 2) == -1
    n[1] = 4
    assert lib.aa_clip_tensors_workspace_bytes(n, 0) == -1
    need = lib.aa_clip_tensors_workspace_bytes(n, 2)
    assert need > 0
    assert lib.aa_clip_tensors(p, p, n, 2, 0, 1.0, 0, 64, 64, need - 1, None) == -34
    assert lib.aa_clip_tensors(p, p, n, 2, 0, 0.0, 0, 64, 64, need, None) == -22
    assert lib.aa_clip_tensors(p, None, n, 2, 0, 1.0, 1, 64, 64, need, None) == -22
    assert lib.aa_clip_tensors(p, p, n, 2, 7, 1.0, 0, 64, 64, need, None) == -22
    ln = _lib.LayerNormDesc(rows=2, inner=1, width=4, x=64, y=64, epsilon=1e-3)
    for k, v in (("rows", 0), ("width", 0), ("x", None), ("y", None), ("dtype", 3), ("mask_act", 9)):
        b = _lib.LayerNormDesc.from_buffer_copy(ln)
        setattr(b, k, v)
        assert lib.aa_layer_norm_forward(ctypes.byref(b), None) == -22, k
    ln.dy, ln.stats, ln.dx, ln.dgamma = 64, 64, 64, 64
    assert lib.aa_layer_norm_backward_workspace_bytes(ctypes.byref(ln)) == 0     # one workgroup
    ln.rows = 5000
    need = lib.aa_layer_norm_backward_workspace_bytes(ctypes.byref(ln))
    assert need > 0
    assert lib.aa_layer_norm_backward(ctypes.byref(ln), None, 0, None) == -34
    ln.dx = ln.dgamma = None
    assert lib.aa_layer_norm_backward(ctypes.byref(ln), None, 0, None) == -22
