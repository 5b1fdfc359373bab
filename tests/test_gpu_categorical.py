"""categorical_log_prob and its gradient against the float64 statement (oracle/categorical.py).

Tolerances (u = 2^-24, the kernels' arithmetic; inputs are exact in float64):
  ln S: a term e^z carries 3 u |z| (difference, scale, exponential), the row's sum `depth` u for the
    longest chain of additions (V / team + joins); so |d ln S| <= u (3 E|z| + depth + 4), E|z| over p;
  log_prob = z_a - ln S: 3 u |z_a| + d ln S;   entropy = ln S - E z: twice d ln S and 3 u E|z| more;
  d logits: p (1 + d ln S + 3 u |z|) times its factor, then half a step of the logits' type.
E|z| <= H + ln S <= 2 ln V + the reference's margin.
"""
import numpy as np
import pytest
import torch

from agents_amd import ops
from oracle import categorical as ocat

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def f64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def chain(vocab):
    return vocab / 64.0 + 40.0 + 6.0 * np.log(vocab + 1.0)


def check(logits, actions, mask, temperature, top_k, r, n_first=0):
    V = logits.shape[-1]
    x = f64(logits).reshape(-1, V)
    a = None if actions is None else actions.cpu().numpy().reshape(-1) - n_first
    m = None if mask is None else mask.expand(logits.shape).cpu().numpy().reshape(-1, V)
    lp, en, ids, top, logp = ocat.forward(x, a, m, temperature, top_k)
    dls = U * (chain(V) + 10)

    def near(got, want, tol):
        got = f64(got).reshape(want.shape)
        bad = ~np.isfinite(want)
        np.testing.assert_array_equal(got[bad], want[bad])
        assert np.all(np.abs(got[~bad] - want[~bad]) <= tol[~bad]), \
            (np.abs(got[~bad] - want[~bad]) / tol[~bad]).max()

    fin = np.where(np.isfinite(lp), np.abs(lp), 0.0)
    span = np.log(V + 1.0) + 4
    if actions is not None:
        near(r.log_prob, lp, dls + 4 * U * (fin + span))
    near(r.entropy, en, np.full(en.shape, 2 * dls + 8 * U * span))
    if top_k > 0:
        np.testing.assert_array_equal(r.top_ids.cpu().numpy().reshape(ids.shape), ids)
        near(r.top_log_prob, top, dls + 4 * U * (np.where(np.isfinite(top), np.abs(top), 0.0) + span))
    return lp, en, logp


def check_grad(logits, actions, mask, temperature, g, h, out, n_first=0):
    V = logits.shape[-1]
    x = f64(logits).reshape(-1, V)
    a = None if actions is None else actions.cpu().numpy().reshape(-1) - n_first
    m = None if mask is None else mask.expand(logits.shape).cpu().numpy().reshape(-1, V)
    gn = None if g is None else f64(g).reshape(-1)
    hn = None if h is None else f64(h).reshape(-1)
    want = ocat.gradient(x, a, gn, hn, m, temperature)
    lp, en, _, _, logp = ocat.forward(x, a, m, temperature)
    p = np.exp(logp)
    size = np.zeros(len(x))
    if gn is not None:
        size = size + np.abs(gn)
    rel = U * (2 * chain(V) + 40)
    near = np.where(p > 0, np.abs(logp), 0.0)
    tol = p * (rel + 6 * U * near) * (size[:, None])
    if hn is not None:
        tol = tol + np.abs(hn)[:, None] * p * (rel + 6 * U * near) * (near + np.abs(en)[:, None] + 1)
    if gn is not None:       # the action's own entry: g / T rounded, then the sum
        tol = tol + 4 * U * size[:, None] * (np.arange(V)[None, :] == (a if a is not None else
                                                                        np.full(len(x), -1))[:, None])
    tol = tol / temperature
    half = torch.finfo(logits.dtype).eps / 2
    # (results below the normal range: half the spacing there; exp2 flushes below 2^-126)
    tiny = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}[
        logits.dtype]
    tol = tol * (1 + half) + half * np.abs(want) + tiny * (1 + size[:, None])
    got = f64(out).reshape(want.shape)
    bad = ~np.isfinite(want)
    np.testing.assert_array_equal(np.isnan(got[bad]), np.isnan(want[bad]))
    assert np.all(np.abs(got[~bad] - want[~bad]) <= tol[~bad]), \
        (np.abs(got[~bad] - want[~bad]) / tol[~bad]).max()


def inputs(shape, dtype, mask_kind, dev, seed, pad=True):
    gen = torch.Generator(device=dev).manual_seed(seed)
    logits = (torch.randn(*shape, generator=gen, device=dev) * 3).to(dtype)
    V = shape[-1]
    actions = torch.randint(0, V, shape[:-1], generator=gen, device=dev)
    mask = None
    if mask_kind is not None:
        mask = torch.rand(*shape, generator=gen, device=dev) < 0.7
        mask.scatter_(-1, actions[..., None], True)
        mask = mask.to(mask_kind)
    if pad and actions.numel() > 2:
        actions.view(-1)[1] = -1
    g = torch.randn(*shape[:-1], generator=gen, device=dev)
    h = torch.randn(*shape[:-1], generator=gen, device=dev) * 0.1
    return logits, actions, mask, g, h


@pytest.mark.parametrize("shape", [(1, 1), (3, 2), (37, 18), (9, 64), (130, 65), (5, 1000), (2, 4096),
                                   (3, 4097), (2, 4, 5003), (1, 30011)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask_kind", [None, torch.bool, torch.int32])
def test_values_and_gradient(dev, shape, dtype, mask_kind):
    logits, actions, mask, g, h = inputs(shape, dtype, mask_kind, dev, 1)
    t = 0.7 if shape[-1] % 2 else 1.0
    r = ops.categorical_log_prob(logits, actions, mask=mask, temperature=t)
    check(logits, actions, mask, t, 0, r)
    for gg, hh in ((g, h), (g, None), (None, h)):
        d = ops.categorical_log_prob_backward(logits, actions, r, gg, hh, mask=mask, temperature=t)
        check_grad(logits, actions, mask, t, gg, hh, d)


@pytest.mark.parametrize("vocab", [8, 9, 63, 127, 128, 129, 200, 256, 257, 300, 511, 512, 513])
@pytest.mark.parametrize("rows", [1, 15, 33])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask_kind", [None, torch.bool, torch.int32])
def test_few_actions(dev, vocab, rows, dtype, mask_kind):
    """Around the sizes at which a row's team changes, rows at every alignment."""
    logits, actions, mask, g, h = inputs((rows, vocab + 1), dtype, mask_kind, dev, vocab)
    logits, actions = logits[:, 1:], actions.clamp(max=vocab - 1)
    mask = None if mask is None else mask[:, 1:]
    r = ops.categorical_log_prob(logits, actions, mask=mask)
    check(logits, actions, mask, 1.0, 0, r)
    d = ops.categorical_log_prob_backward(logits, actions, r, g, h, mask=mask)
    check_grad(logits, actions, mask, 1.0, g, h, d)


@pytest.mark.parametrize("shape", [(9, 18), (33, 700), (5, 5003), (1, 60001), (300, 20011)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask_kind", [torch.bool, torch.int32])
def test_alternatives_under_masks(dev, shape, dtype, mask_kind):
    logits, actions, mask, _, _ = inputs(shape[:1] + (shape[1] + 3,), dtype, mask_kind, dev, 31)
    logits, mask, actions = logits[:, 3:], mask[:, 3:], actions.clamp(max=shape[1] - 1)
    for k in (1, 11):
        r = ops.categorical_log_prob(logits, actions, mask=mask, top_k=k)
        check(logits, actions, mask, 1.0, k, r)


@pytest.mark.parametrize("rows", [1, 3, 700])
@pytest.mark.parametrize("vocab,top_k", [(2, 2), (7, 64), (300, 5), (4096, 20), (4099, 64), (40003, 1),
                                         (131072, 20)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_alternatives(dev, rows, vocab, top_k, dtype):
    if rows * vocab > 5_000_000:
        rows = 30
    logits, actions, mask, _, _ = inputs((rows, vocab), dtype, torch.uint8 if rows == 3 else None, dev,
                                         rows + vocab)
    r = ops.categorical_log_prob(logits, actions, mask=mask, top_k=top_k)
    check(logits, actions, mask, 1.0, top_k, r)


@pytest.mark.parametrize("order", ["ascending", "descending", "equal", "two-values", "zeros"])
@pytest.mark.parametrize("vocab", [100, 3000, 20001])
def test_alternatives_of_ordered_rows(dev, order, vocab):
    i = torch.arange(vocab, device=dev)
    x = {"ascending": i / 100.0, "descending": -i / 100.0, "equal": torch.full((vocab,), 2.5, device=dev),
         "two-values": (i % 3 == 0).float(), "zeros": torch.where(i % 2 == 0, 0.0, -0.0)}[order]
    logits = x.float().repeat(2, 1)
    actions = torch.tensor([0, vocab - 1], device=dev)
    for k in (1, 33, 64):
        check(logits, actions, None, 1.0, k, ops.categorical_log_prob(logits, actions, top_k=k))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [6, 5000, 40001])
def test_corners(dev, dtype, vocab):
    corners(dev, dtype, vocab, 4)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [6, 60, 100, 200, 300, 600, 5000, 40001])
def test_corners_without_alternatives(dev, dtype, vocab):
    corners(dev, dtype, vocab, 0)


def corners(dev, dtype, vocab, top_k):
    """Empty masks, the type's lowest value, infinities and NaN in masked and in allowed places, an
    action that its mask excludes, one past the end, padding."""
    inf, nan, low = float("inf"), float("nan"), torch.finfo(dtype).min
    n = 14
    logits = (torch.randn(n, vocab, generator=torch.Generator().manual_seed(3)) * 2).to(dtype).to(dev)
    mask = torch.ones(n, vocab, dtype=torch.bool, device=dev)
    actions = torch.zeros(n, dtype=torch.int32, device=dev)
    mask[0] = False                                   # nothing left
    logits[1] = -inf                                  # no finite logit
    logits[2] = low                                   # all the lowest: uniform
    logits[3, 1:] = low                               # all but one
    logits[4, 2], mask[4, 2] = nan, False             # masked NaN, infinities
    logits[5, 2], mask[5, 2] = inf, False
    logits[6, 2], mask[6, 2] = -inf, False
    logits[7, vocab - 1] = nan                        # allowed NaN, infinities
    logits[8, vocab - 1] = inf
    logits[9, vocab - 1] = -inf
    mask[10, 0] = False                               # the action's own place
    actions[11] = vocab                               # past the end
    actions[12] = -7                                  # padding; its logits are not used
    logits[12] = nan
    logits[13, 0] = -inf                              # the action's logit is -inf
    r = ops.categorical_log_prob(logits, actions, mask=mask, top_k=top_k)
    check(logits, actions, mask, 1.0, top_k, r)
    g = torch.linspace(-1, 1, n, device=dev)
    h = torch.linspace(0.5, -0.5, n, device=dev)
    d = ops.categorical_log_prob_backward(logits, actions, r, g, h, mask=mask)
    check_grad(logits, actions, mask, 1.0, g, h, d)
    assert (d[0] == 0).all() and (d[1] == 0).all() and (d[12] == 0).all()
    assert (d[~mask] == 0).all()


@pytest.mark.parametrize("scale", [1e-4, 1.0, 1e4])
def test_offsets_and_scales(dev, scale):
    """A common offset of the logits costs no accuracy, whatever its size (exact in float32)."""
    x = torch.randint(-64, 64, (4, 9001), generator=torch.Generator().manual_seed(5)).float().to(dev)
    logits = x * 0.125 + 8192.0 * 16
    actions = torch.tensor([5, 9000, 17, 4000], device=dev)
    t = 1.0 if scale == 1.0 else scale
    check(logits, actions, None, t, 3, ops.categorical_log_prob(logits, actions, temperature=t, top_k=3))


def test_strides(dev):
    """Sliced sequences, rows of a wider buffer at odd offsets, broadcast masks, actions of both widths
    and with an offset."""
    gen = torch.Generator(device=dev).manual_seed(9)
    B, T, V = 3, 6, 777
    full = torch.randn(B, T, V, generator=gen, device=dev).half()
    tokens = torch.randint(0, V, (B, T), generator=gen, device=dev)
    logits, actions = full[:, :-1], tokens[:, 1:]
    vocab_mask = torch.rand(V, generator=gen, device=dev) < 0.9
    per_row = torch.rand(B, 1, V, generator=gen, device=dev) < 0.9
    g = torch.randn(B, 1, device=dev, generator=gen).expand(B, T - 1)
    for mask in (None, vocab_mask, per_row):
        r = ops.categorical_log_prob(logits, actions, mask=mask, top_k=3)
        check(logits, actions, mask, 1.0, 3, r)
        assert r.log_prob.shape == (B, T - 1) and r.top_ids.shape == (B, T - 1, 3)
        d = ops.categorical_log_prob_backward(logits, actions, r, g, None, mask=mask)
        check_grad(logits, actions, mask, 1.0, g, None, d)
    wide = torch.randn(11, 5000, generator=gen, device=dev)
    part = wide[:, 3:3 + 4501]
    acts = torch.randint(10, 10 + 4501, (11,), generator=gen, device=dev, dtype=torch.int32)
    r = ops.categorical_log_prob(part, acts, first_action=10, top_k=2)
    check(part, acts, None, 1.0, 2, r, n_first=10)
    # out with strides of its own: what lies around it stays
    buf = torch.full((11, 4510), 7.0, device=dev)
    g1 = torch.ones(11, device=dev)
    d = ops.categorical_log_prob_backward(part, acts, r, g1, None, first_action=10,
                                          out=buf[:, 5:5 + 4501])
    check_grad(part, acts, None, 1.0, g1, None, d, n_first=10)
    assert (buf[:, :5] == 7).all() and (buf[:, 5 + 4501:] == 7).all()
    same = torch.zeros(1, 4501, device=dev).expand(8, 4501)      # one row for all
    a8 = torch.arange(8, device=dev)
    check(same, a8, None, 1.0, 0, ops.categorical_log_prob(same, a8))


def test_one_row_without_leading_axes(dev):
    logits = torch.randn(700, device=dev, generator=torch.Generator(device=dev).manual_seed(1))
    action = torch.tensor(9, device=dev)
    mask = torch.ones(700, dtype=torch.bool, device=dev)
    r = ops.categorical_log_prob(logits, action, mask=mask, top_k=3)
    assert r.log_prob.shape == () and r.top_ids.shape == (3,)
    check(logits[None], action[None], mask[None], 1.0, 3, r)
    g = torch.tensor(2.0, device=dev)
    d = ops.categorical_log_prob_backward(logits, action, r, g, mask=mask)
    check_grad(logits[None], action[None], mask[None], 1.0, g[None], None, d)


def test_results_over_inputs_are_refused(dev):
    buf = torch.randn(4, 20, device=dev)
    logits, actions = buf[:, :10], torch.zeros(4, dtype=torch.int64, device=dev)
    r = ops.categorical_log_prob(logits, actions)
    g = torch.ones(4, device=dev)
    with pytest.raises(ValueError, match="twice"):
        ops.categorical_log_prob_backward(logits, actions, r, g,
                                          out=torch.zeros(1, 10, device=dev).expand(4, 10))
    flat = torch.randn(100, device=dev)
    logits = flat[:40].view(4, 10)
    r = ops.categorical_log_prob(logits, actions)
    with pytest.raises(ValueError, match="overlaps"):
        ops.categorical_log_prob_backward(logits, actions, r, g, out=flat[5:45].view(4, 10))
    ops.categorical_log_prob_backward(logits, actions, r, g, out=flat[40:80].view(4, 10))


def test_in_place_gradient(dev):
    for dtype, V in ((torch.float32, 37), (torch.bfloat16, 5001)):
        logits, actions, _, g, h = inputs((6, V), dtype, None, dev, 11)
        r = ops.categorical_log_prob(logits, actions)
        want = ops.categorical_log_prob_backward(logits, actions, r, g, h)
        got = logits.clone()
        ops.categorical_log_prob_backward(got, actions, r, g, h, out=got)
        assert torch.equal(got, want)


def test_entropy_without_actions(dev):
    logits, _, mask, _, h = inputs((5, 6001), torch.float32, torch.bool, dev, 12)
    r = ops.categorical_log_prob(logits, mask=mask, top_k=7)
    assert r.log_prob is None
    check(logits, None, mask, 1.0, 7, r)
    d = ops.categorical_log_prob_backward(logits, None, r, None, h, mask=mask)
    check_grad(logits, None, mask, 1.0, None, h, d)


def test_no_rows(dev):
    r = ops.categorical_log_prob(torch.empty(0, 5, device=dev),
                                 torch.empty(0, dtype=torch.int64, device=dev), top_k=2)
    assert r.log_prob.shape == (0,) and r.top_ids.shape == (0, 2)
    d = ops.categorical_log_prob_backward(
        torch.empty(0, 5, device=dev), torch.empty(0, dtype=torch.int64, device=dev), r,
        torch.empty(0, device=dev))
    assert d.shape == (0, 5)


def test_many_rows(dev):
    """More rows than one grid axis takes workgroups."""
    n, V = (1 << 22) + 5, 3
    logits = torch.randn(n, V, device=dev, generator=torch.Generator(device=dev).manual_seed(2))
    actions = torch.arange(n, device=dev) % V
    r = ops.categorical_log_prob(logits, actions)
    want = torch.log_softmax(logits.double(), 1)
    assert (r.log_prob.double() - want.gather(1, actions[:, None])[:, 0]).abs().max() < 64 * U
    g = torch.ones(n, device=dev)
    d = ops.categorical_log_prob_backward(logits, actions, r, g)
    hot = torch.nn.functional.one_hot(actions, V)
    assert (d.double() - (hot - want.exp())).abs().max() < 64 * U


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_gradients(dev, dtype):
    """Gradients that are stored past the caches are those of a part of the rows, bit for bit."""
    V = 33001
    rows = (140 << 20) // (V * dtype.itemsize)
    gen = torch.Generator(device=dev).manual_seed(4)
    logits = torch.randn(rows, V, generator=gen, device=dev).to(dtype)
    actions = torch.randint(0, V, (rows,), generator=gen, device=dev)
    g = torch.randn(rows, generator=gen, device=dev)
    r = ops.categorical_log_prob(logits, actions)
    d = ops.categorical_log_prob_backward(logits, actions, r, g, g)
    cut = slice(rows - 5, rows)
    part = type(r)(r.log_prob[cut], r.entropy[cut], None, None, r.stats[cut])
    want = ops.categorical_log_prob_backward(logits[cut], actions[cut], part, g[cut], g[cut])
    assert torch.equal(d[cut], want)
    check_grad(logits[cut], actions[cut], None, 1.0, g[cut], g[cut], want)


def test_offsets_past_32_bits(dev):
    V, stride = 4099, (1 << 31) + 4099
    buf = torch.empty(stride + V, dtype=torch.bfloat16, device=dev)
    logits = buf.as_strided((2, V), (stride, 1))
    logits.copy_(torch.randn(2, V, generator=torch.Generator().manual_seed(1)))
    actions = torch.tensor([7, 4098], device=dev)
    r = ops.categorical_log_prob(logits, actions, top_k=2)
    check(logits, actions, None, 1.0, 2, r)
    g = torch.ones(2, device=dev)
    want = ops.categorical_log_prob_backward(logits, actions, r, g)
    ops.categorical_log_prob_backward(logits, actions, r, g, out=logits)
    assert torch.equal(logits, want)


def test_same_bits_on_two_streams_and_in_a_graph(dev):
    """Two calls at once on streams of their own, and a captured pair of calls replayed between eager
    work, give the bits of the eager call (one token over split rows, and a batch)."""
    for shape, k in (((1, 60001), 9), ((300, 999), 0)):
        logits, actions, _, g, h = inputs(shape, torch.bfloat16, None, dev, 21, pad=False)
        other, oact, _, _, _ = inputs(shape, torch.bfloat16, None, dev, 22, pad=False)

        def both(x, a):
            r = ops.categorical_log_prob(x, a, top_k=k)
            return r, ops.categorical_log_prob_backward(x, a, r, g, h)

        want, wd = both(logits, actions)
        want2, wd2 = both(other, oact)
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        outs = []
        for _ in range(20):
            with torch.cuda.stream(s1):
                outs.append((both(logits, actions), want, wd))
            with torch.cuda.stream(s2):
                outs.append((both(other, oact), want2, wd2))
        torch.cuda.synchronize()
        for (r, d), w, wdd in outs:
            for x, y in zip(r, w):
                assert x is None or torch.equal(x, y)
            assert torch.equal(d, wdd)
        x = logits.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r, d = both(x, actions)
        for i in range(6):
            x.copy_(logits if i % 2 == 0 else other)
            graph.replay()
            eager, ed = both(x, actions)
            torch.cuda.synchronize()
            for p, q in zip(r, eager):
                assert p is None or torch.equal(p, q)
            assert torch.equal(d, ed)
