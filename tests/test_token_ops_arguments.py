"""Each check of the token operators' arguments by its own message (CPU: types, shapes and layouts are
looked at before the device is, so host tensors reach every check but the last one)."""
import pytest
import torch

from agents_amd import _lib, ops

pytestmark = pytest.mark.usefixtures("lib")

I64, I32, F16, F64 = torch.int64, torch.int32, torch.float16, torch.float64


def z(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


X, A = z(3, 5), z(3, dtype=I64)
R = ops.CategoricalLogProb(z(3), z(3), None, None, z(3, 2))


def refused(text, fn, *a, error=ValueError, **kw):
    with pytest.raises(error, match=text) as e:
        fn(*a, **kw)
    assert "device tensors" not in str(e.value)


CATEGORICAL = {
    "type": ("logits must be", dict(logits=z(3, 5, dtype=F64))),
    "scalar": ("logits must be", dict(logits=z(), actions=None)),
    "no actions": ("no actions", dict(logits=z(3, 0))),
    "last axis": ("last axis of logits", dict(logits=z(5, 3).t())),
    "action type": ("int32 or int64", dict(actions=z(3))),
    "action shape": ("actions .* for logits", dict(actions=z(2, dtype=I64))),
    "action axes": ("actions .* for logits", dict(logits=z(5), actions=z(1, dtype=I64))),
    "mask type": ("mask must be", dict(mask=z(3, 5))),
    "mask last axis": ("mask .* for logits", dict(mask=z(3, 1, dtype=torch.bool))),
    "mask rows": ("mask .* for logits", dict(mask=z(2, 5, dtype=torch.bool))),
    "mask axes": ("mask .* for logits", dict(mask=z(1, 3, 5, dtype=torch.bool))),
    "mask strides": ("last axis of mask", dict(mask=z(5, 3, dtype=torch.bool).t())),
    "temperature 0": ("temperature", dict(temperature=0.0)),
    "temperature < 0": ("temperature", dict(temperature=-1.0)),
    "temperature nan": ("temperature", dict(temperature=float("nan"))),
    "temperature inf": ("temperature", dict(temperature=float("inf"))),
    "temperature tiny": ("temperature", dict(temperature=1e-31)),
    "top_k 65": ("top_k", dict(top_k=65)),
    "top_k -1": ("top_k", dict(top_k=-1)),
    "fold": ("do not fold", dict(logits=z(3, 5, 4, 5)[:, :4, :3], actions=z(3, 4, 3, dtype=I64))),
}


@pytest.mark.parametrize("name", list(CATEGORICAL))
def test_categorical(name):
    text, kw = CATEGORICAL[name]
    refused(text, ops.categorical_log_prob, **{**dict(logits=X, actions=A), **kw})
    if not name.startswith("top_k"):
        kw = {**dict(logits=X, actions=A, forward=R, dentropy=None), **kw}
        lead = kw["logits"].shape[:-1]
        if lead != (3,):
            kw["forward"] = ops.CategoricalLogProb(z(*lead), z(*lead), None, None, z(*lead, 2))
        if kw["actions"] is None:
            kw["dentropy"] = z(*lead)
        else:
            kw["dlog_prob"] = z(*lead)
        refused(text, ops.categorical_log_prob_backward, **kw)


BACKWARD = {
    "nothing": ("needs dlog_prob or dentropy", dict(dlog_prob=None)),
    "no actions": ("needs actions", dict(actions=None)),
    "dlog_prob type": ("dlog_prob must be", dict(dlog_prob=z(3, dtype=F64))),
    "dlog_prob shape": ("dlog_prob must be", dict(dlog_prob=z(2))),
    "dentropy type": ("dentropy must be", dict(dentropy=z(3, dtype=F16))),
    "dentropy shape": ("dentropy must be", dict(dentropy=z(3, 1))),
    "stats shape": ("forward.stats", dict(forward=R._replace(stats=z(3, 3)))),
    "stats type": ("forward.stats", dict(forward=R._replace(stats=z(3, 2, dtype=F64)))),
    "stats layout": ("forward.stats", dict(forward=R._replace(stats=z(2, 3).t()))),
    "entropy shape": ("forward.entropy", dict(forward=R._replace(entropy=z(2)))),
    "entropy type": ("forward.entropy", dict(forward=R._replace(entropy=z(3, dtype=F16)))),
    "entropy layout": ("forward.entropy", dict(forward=R._replace(entropy=z(6)[::2]))),
    "out type": ("out must be", dict(out=z(3, 5, dtype=F16))),
    "out shape": ("out must be", dict(out=z(3, 4))),
    "out layout": ("out must be", dict(out=z(5, 3).t())),
}


@pytest.mark.parametrize("name", list(BACKWARD))
def test_categorical_backward(name):
    text, kw = BACKWARD[name]
    refused(text, ops.categorical_log_prob_backward,
            **{**dict(logits=X, actions=A, forward=R, dlog_prob=z(3)), **kw})


@pytest.mark.parametrize("each", [False, True])
def test_clip(each):
    f = ops.clip_by_norms if each else ops.clip_by_global_norm
    refused("no tensors", f, [], 1.0)
    for limit in (0.0, -1.0, float("nan")):
        refused("clip_norm must be positive", f, [z(3)], limit)
    refused("must be float32", f, [z(3, dtype=I32)], 1.0)
    refused("of one type", f, [z(3), z(3, dtype=F16)], 1.0)
    refused("contiguous", f, [z(3), z(3, 4).t()], 1.0)
    refused("must be a tensor", f, [z(3), None], 1.0, error=TypeError)
    refused("must be a number", f, [z(3)], "one", error=TypeError)
    for out in ([z(3)], [z(3), z(4, dtype=F16)], [z(3), z(2, 2)], [z(3), z(8)[::2]]):
        refused("out must mirror", f, [z(3), z(4)], 1.0, out=out)


W, ST = z(5), z(3, 2)
NORM = {
    "type": ("x must be", dict(x=z(3, 5, dtype=F64))),
    "no columns": ("x must be", dict(x=z(3, 0))),
    "last axis": ("contiguous last axis", dict(x=z(5, 3).t(), gamma=z(3), beta=z(3))),
    "gamma length": ("gamma must be", dict(gamma=z(4))),
    "gamma type": ("gamma must be", dict(gamma=z(5, dtype=F16))),
    "gamma layout": ("gamma must be", dict(gamma=z(10)[::2])),
    "beta axes": ("beta must be", dict(beta=z(1, 5))),
    "epsilon < 0": ("epsilon", dict(epsilon=-1.0)),
    "epsilon nan": ("epsilon", dict(epsilon=float("nan"))),
    "out type": ("out must be", dict(out=z(3, 5, dtype=F16))),
    "out shape": ("out must be", dict(out=z(2, 5))),
    "out layout": ("out must be", dict(out=z(5, 3).t())),
    "stats shape": ("stats must be", dict(stats=z(3))),
    "stats type": ("stats must be", dict(stats=z(3, 2, dtype=F64))),
    "fold": ("do not fold", dict(x=z(3, 5, 4, 5)[:, :4, :3])),
}


@pytest.mark.parametrize("name", list(NORM))
def test_layer_norm(name):
    text, kw = NORM[name]
    refused(text, ops.layer_norm_forward, **{**dict(x=X, gamma=W, beta=W), **kw})


NORM_BACKWARD = {
    "dy type": ("dy must be", dict(dy=z(3, 5, dtype=F16))),
    "dy shape": ("dy must be", dict(dy=z(2, 5))),
    "dy layout": ("dy must be", dict(dy=z(5, 3).t())),
    "gamma length": ("gamma must be", dict(gamma=z(4))),
    "stats shape": ("stats must be", dict(stats=z(2, 2))),
    "stats layout": ("stats must be", dict(stats=z(2, 3).t())),
    "nothing": ("nothing to compute", dict(param_grads=False, input_grad=False)),
    "dx type": ("dx must be", dict(dx=z(3, 5, dtype=F16))),
    "dx shape": ("dx must be", dict(dx=z(3, 4))),
    "dgamma length": ("dgamma must be", dict(dgamma=z(4))),
    "dbeta type": ("dbeta must be", dict(dbeta=z(5, dtype=F16))),
    "fold": ("do not fold", dict(x=z(3, 5, 4, 5)[:, :4, :3], dy=z(3, 4, 3, 5), stats=z(3, 4, 3, 2))),
}


@pytest.mark.parametrize("name", list(NORM_BACKWARD))
def test_layer_norm_backward(name):
    text, kw = NORM_BACKWARD[name]
    refused(text, ops.layer_norm_backward, **{**dict(dy=z(3, 5), x=X, gamma=W, stats=ST), **kw})


def test_host_tensors():
    """Calls that pass every other check."""
    for call in (lambda: ops.categorical_log_prob(X, A, mask=z(5, dtype=torch.bool), top_k=3),
                 lambda: ops.categorical_log_prob_backward(X, A, R, z(3), z(3)),
                 lambda: ops.categorical_log_prob_backward(X, A, R, z(3), out=z(3, 5)),
                 lambda: ops.categorical_log_prob(z(0, 5), z(0, dtype=I64)),
                 lambda: ops.clip_by_global_norm([z(3), z(2, 2)], 1.0),
                 lambda: ops.clip_by_norms([z(3)], 1.0, out=[z(3)]),
                 lambda: ops.global_norm([z(3)]),
                 lambda: ops.layer_norm_forward(X, W, W, out=z(3, 5), stats=ST),
                 lambda: ops.layer_norm_forward(z(0, 5), W, W),
                 lambda: ops.layer_norm_backward(z(3, 5), X, W, ST),
                 lambda: ops.layer_norm_backward(z(3, 5), X, W, ST, dx=z(3, 5), dgamma=z(5), dbeta=z(5))):
        with pytest.raises(_lib.AgentsAmdError, match="device tensors"):
            call()
