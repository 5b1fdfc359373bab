"""Results of the token operators over their inputs: refused exactly where a byte is shared, unless the
result is the input itself (CPU: the check runs before the one for device tensors)."""
import random

import numpy as np
import pytest
import torch

from agents_amd import _lib, ops

pytestmark = pytest.mark.usefixtures("lib")


def outcome(fn, *a, **kw):
    """"overlaps", "twice", or "" for a call that passes every check but the one for device tensors."""
    try:
        fn(*a, **kw)
    except _lib.AgentsAmdError as e:
        assert "device tensors" in str(e)
        return ""
    except ValueError as e:
        for word in ("overlaps", "twice"):
            if word in str(e):
                return word
        raise
    raise AssertionError("host tensors were taken")


def norm_over(x, out):
    return outcome(ops.layer_norm_forward, x, None, None, out=out)


def grad_over(x, out):
    a = torch.zeros(x.shape[:-1], dtype=torch.int64)
    r = ops.CategoricalLogProb(None, torch.zeros(x.shape[:-1]), None, None, torch.zeros(*x.shape[:-1], 2))
    return outcome(ops.categorical_log_prob_backward, x, a, r, torch.zeros(x.shape[:-1]), out=out)


def dx_over(x, out):
    return outcome(ops.layer_norm_backward, torch.zeros(x.shape), x, None, torch.zeros(*x.shape[:-1], 2), dx=out)


def dx_over_dy(dy, out):
    return outcome(ops.layer_norm_backward, dy, torch.zeros(dy.shape), None, torch.zeros(*dy.shape[:-1], 2), dx=out)


CALLS = [norm_over, grad_over, dx_over, dx_over_dy]


@pytest.mark.parametrize("call", CALLS)
def test_shifted_slices(call):
    buf = torch.zeros(3, 6, 10)
    assert call(buf[:, :-1], buf[:, 1:]) == "overlaps"
    assert call(buf[:, 1:], buf[:, :-1]) == "overlaps"
    assert call(buf[:, :, :8], buf[:, :, 2:]) == "overlaps"
    assert call(buf[:, :-1], buf[:, :-1]) == ""                  # itself
    assert call(buf[:, :3], buf[:, 3:]) == ""
    assert call(buf[:, 0::2], buf[:, 1::2]) == ""                # rows in turn
    assert call(buf[:, :, :5], buf[:, :, 5:]) == ""              # columns beside each other
    assert call(buf[:, :, :5], buf[:, :, 4:9]) == "overlaps"
    assert call(buf[:2, :, 1:4], buf[1:, :, 4:7]) == ""
    assert call(buf[:2, :, 1:4], buf[1:, :, 3:6]) == "overlaps"
    flat = torch.zeros(200)
    assert call(flat[:40].view(4, 10), flat[5:45].view(4, 10)) == "overlaps"
    assert call(flat[:40].view(4, 10), flat[40:80].view(4, 10)) == ""


@pytest.mark.parametrize("call", CALLS)
def test_the_same_memory_in_another_order(call):
    flat = torch.zeros(60)
    x = flat.view(2, 3, 10)
    assert call(x, flat.view(3, 2, 10).transpose(0, 1)) == "overlaps"
    # a row of one: its stride is no difference
    one = flat[:10].view(1, 10)
    assert call(one, flat.as_strided((1, 10), (33, 1))) == ""


@pytest.mark.parametrize("call", CALLS)
def test_a_result_that_meets_itself(call):
    flat = torch.zeros(100)
    x = torch.zeros(4, 10)
    assert call(x, flat[:13].unfold(0, 10, 1)) == "twice"
    assert call(x, flat[:10].expand(4, 10)) == "twice"
    w = flat[:13].unfold(0, 10, 1)
    assert call(w, w) == "twice"
    assert call(w, torch.zeros(4, 10)) == ""                     # rows that share memory may be read
    assert call(torch.zeros(2, 2, 10), flat.as_strided((2, 2, 10), (20, 20, 1))) == "twice"


def test_large_tensors_take_no_search():
    """Interleaved slices of many rows (the check must not walk them)."""
    buf = torch.empty(1 << 12, 1 << 8, 8)
    for call in CALLS[:1]:
        assert call(buf[..., :4], buf[..., 4:]) == ""
        assert call(buf[:, ::2, :4], buf[:, 1::2, :4]) == ""
        assert call(buf[:, :-1], buf[:, 1:]) == "overlaps"


def test_random_layouts():
    """Against the sets of element addresses."""
    rng = random.Random(7)
    seen = {"": 0, "overlaps": 0, "twice": 0}
    for _ in range(4000):
        buf = torch.zeros(400)
        lead, width = [rng.randint(1, 4) for _ in range(2)], rng.randint(1, 6)

        def strides():
            s1 = rng.choice([0, width, width + 1, 2 * width, rng.randint(1, 12)])
            s0 = rng.choice([0, s1 * lead[1], s1 * lead[1] + 1, 2 * s1 * lead[1], rng.randint(1, 40)])
            return rng.choice([(s0, s1, 1), (s1, s0, 1)])

        def make(st):
            reach = (lead[0] - 1) * st[0] + (lead[1] - 1) * st[1] + width
            return buf.as_strided((*lead, width), st, rng.randint(0, 60)) if reach < 300 else None

        st = strides()
        x, out = make(st), make(st if rng.random() < 0.6 else strides())
        if x is None or out is None:
            continue

        def places(t):
            i = np.indices(t.shape).reshape(3, -1)
            return t.storage_offset() + (i * np.array(t.stride())[:, None]).sum(0)

        px, po = places(x), places(out)
        want = "twice" if len(set(po)) < len(po) else \
            "overlaps" if set(px) & set(po) and not np.array_equal(px, po) else ""
        try:
            got = norm_over(x, out)
        except ValueError as e:
            assert "do not fold" in str(e)
            continue
        assert got == want, (x.shape, x.stride(), x.storage_offset(), out.stride(), out.storage_offset())
        seen[got] += 1
    assert min(seen.values()) > 200, seen


def test_other_tensors_of_the_call():
    x, flat = torch.zeros(4, 10), torch.zeros(400)
    rows = flat.as_strided((4, 10), (20, 1))                     # room between the rows
    w_between, w_inside = flat[10:20], flat[15:25]
    f = ops.layer_norm_forward
    assert outcome(f, x, w_between, None, out=rows) == ""
    assert outcome(f, x, None, w_between, out=rows) == ""
    assert outcome(f, x, w_inside, None, out=rows) == "overlaps"
    assert outcome(f, x, None, w_inside, out=rows) == "overlaps"
    assert outcome(f, rows, None, None, stats=flat[10:18].view(4, 2)) == ""
    assert outcome(f, rows, None, None, stats=flat[14:22].view(4, 2)) == "overlaps"
    g, st = ops.layer_norm_backward, torch.zeros(4, 2)
    assert outcome(g, x, rows, None, st, dgamma=w_between) == ""
    assert outcome(g, x, rows, None, st, dgamma=w_inside) == "overlaps"
    assert outcome(g, rows, x, None, st, dbeta=w_inside) == "overlaps"
    assert outcome(g, x, x, None, st, dx=rows, dbeta=w_inside) == "overlaps"
    a = torch.zeros(4, dtype=torch.int64)
    r = ops.CategoricalLogProb(None, torch.zeros(4), None, None, st)
    b = ops.categorical_log_prob_backward
    assert outcome(b, x, a, r, flat[10:14], out=rows) == ""
    assert outcome(b, x, a, r, flat[18:22], out=rows) == "overlaps"
    assert outcome(b, x, a, r._replace(stats=flat[58:66].view(4, 2)), torch.zeros(4), out=rows) == "overlaps"
    ints = flat.view(torch.int64)                                # (places 5 .. 9 lie between two rows)
    assert outcome(b, x, ints[5:9], r, torch.zeros(4), out=rows) == ""
    assert outcome(b, x, ints[7:11], r, torch.zeros(4), out=rows) == "overlaps"
    mask = flat.view(torch.int32).as_strided((4, 10), (20, 1), 10)
    assert outcome(b, x, a, r, torch.zeros(4), mask=mask, out=rows) == ""
    assert outcome(b, x, a, r, torch.zeros(4), mask=flat.view(torch.int32)[15:25], out=rows) == "overlaps"
