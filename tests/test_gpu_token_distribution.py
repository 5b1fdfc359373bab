"""Categorical distributions of the discrete policies where actions are excluded, out of the action spec
or without a distribution, against the float64 statement (oracle/categorical.py).

Tolerances (u = 2^-24): q / T is rounded once (u |z|), the operator adds 3 u |z| and ln S with at most 12 u
for rows of up to six values; |z| <= 16 here, so 100 u.
"""
import numpy as np
import pytest
import torch

from agents_amd import ops
from agents_amd.networks import layers as L
from agents_amd.networks import sequential
from agents_amd.policies import boltzmann_policy, q_policy
from agents_amd.specs import tensor_spec
from agents_amd.trajectories import time_step as ts
from oracle import categorical as ocat

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
INF, NAN = float("inf"), float("nan")


def make_policy(lo, hi, dtype=torch.int64, masked=True):
    obs = tensor_spec.TensorSpec((3,), torch.float32)
    spec, splitter = obs, None
    if masked:
        spec = {"x": obs, "mask": tensor_spec.BoundedTensorSpec((hi - lo + 1,), torch.int32, 0, 1)}
        splitter = lambda o: (o["x"], o["mask"])
    net = sequential.Sequential([L.Dense(hi - lo + 1)], input_spec=obs, seed=4)
    policy = q_policy.QPolicy(ts.time_step_spec(spec), tensor_spec.BoundedTensorSpec((), dtype, lo, hi),
                              q_network=net, observation_and_action_constraint_splitter=splitter)
    return policy, net


def close(got, want):
    got, want = got.detach().double().cpu().numpy(), np.asarray(want, np.float64)
    fin = np.isfinite(want)
    np.testing.assert_array_equal(got[~fin], want[~fin])
    assert np.all(np.abs(got[fin] - want[fin]) <= 100 * U)


@pytest.mark.parametrize("lo", [2, 0, -3])
@pytest.mark.parametrize("temperature", [None, 0.5, 3.0])
def test_excluded_actions_have_no_probability(dev, lo, temperature):
    policy, net = make_policy(lo, lo + 4)
    x = torch.randn(5, 3, generator=torch.Generator().manual_seed(0)).to(dev)
    mask = torch.tensor([[1, 1, 1, 1, 1], [0, 0, 0, 1, 0], [1, 0, 0, 0, 1], [0, 1, 0, 0, 0],
                         [0, 0, 0, 0, 0]], dtype=torch.int32, device=dev)
    p = policy if temperature is None else boltzmann_policy.BoltzmannPolicy(policy, temperature)
    dist = p.distribution(ts.restart({"x": x, "mask": mask}, batch_size=5)).action
    q, m = net.forward(x).double().cpu().numpy(), mask.cpu().numpy()
    for a in range(5):
        actions = np.full(5, a)
        lp, en, ids, top, _ = ocat.forward(q, actions, m, temperature or 1.0, 4)
        close(dist.log_prob(torch.from_numpy(actions + lo).to(dev)), lp)
    close(dist.entropy(), en)
    got_ids, got_top = dist.most_likely(4)
    np.testing.assert_array_equal(got_ids.cpu().numpy(), np.where(ids < 0, ids, ids + lo))
    close(got_top, top)
    # the most likely action is the mode wherever there is one
    assert torch.equal(got_ids[:4, 0], dist.mode()[:4])


def test_the_mask_is_the_one_of_the_time_step(dev):
    """An observation buffer that is written again does not change a distribution."""
    policy, net = make_policy(0, 4)
    x = torch.randn(2, 3, generator=torch.Generator().manual_seed(1)).to(dev)
    mask = torch.tensor([[1, 0, 1, 0, 1], [0, 1, 1, 0, 0]], dtype=torch.int32, device=dev)
    dist = policy.distribution(ts.restart({"x": x, "mask": mask}, batch_size=2)).action
    before = dist.most_likely(5) + (dist.entropy(), dist.log_prob(torch.tensor([1, 1], device=dev)))
    x.zero_()
    mask.fill_(1)
    after = dist.most_likely(5) + (dist.entropy(), dist.log_prob(torch.tensor([1, 1], device=dev)))
    for a, b in zip(before, after):
        assert torch.equal(a, b)
    assert float(before[3][0]) == -INF and (before[0][1, 2:] == -1).all()


@pytest.mark.parametrize("lo", [2, -3])
def test_no_alternative_is_no_action(dev, lo):
    """The marker of a missing alternative is -1 whatever the spec's minimum."""
    policy, net = make_policy(lo, lo + 4, masked=False)
    dist = policy.distribution(ts.restart(torch.zeros(3, 3, device=dev), batch_size=3)).action
    dist.logits[0] = torch.tensor([1.0, NAN, 0.0, 2.0, 3.0])
    dist.logits[1] = torch.tensor([-INF, 4.0, -INF, -INF, 1.0])
    dist.logits[2] = -INF
    ids, top = dist.most_likely(3)
    assert ids.tolist() == [[-1, -1, -1], [lo + 1, lo + 4, -1], [-1, -1, -1]]
    assert top[0].isnan().all() and float(top[1, 2]) == -INF and (top[2] == -INF).all()


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("lo", [2, -3])
def test_actions_outside_the_spec(dev, lo, dtype):
    policy, net = make_policy(lo, lo + 4, dtype, masked=False)
    low, high = torch.iinfo(dtype).min, torch.iinfo(dtype).max
    actions = torch.tensor([lo, lo - 1, lo - 2, low, lo + 4, lo + 5, high, low + 2], dtype=dtype, device=dev)
    x = torch.randn(len(actions), 3, generator=torch.Generator().manual_seed(2)).to(dev)
    dist = policy.distribution(ts.restart(x, batch_size=len(actions))).action
    want, *_ = ocat.forward(net.forward(x).double().cpu().numpy(), np.array([0, 9, 9, 9, 4, 9, 9, 9]))
    close(dist.log_prob(actions), want)


def test_how_many_alternatives(dev):
    """More than there are actions: all of them; none at all is refused, 64 of many is the limit."""
    policy, net = make_policy(2, 6, masked=False)
    x = torch.randn(2, 3, generator=torch.Generator().manual_seed(2)).to(dev)
    dist = policy.distribution(ts.restart(x, batch_size=2)).action
    all_ids, all_top = dist.most_likely(5)
    for k in (6, 64, 65, 1000):
        ids, top = dist.most_likely(k)
        assert torch.equal(ids, all_ids) and torch.equal(top, all_top)
    for k in (0, -1):
        with pytest.raises(ValueError, match="at least 1"):
            dist.most_likely(k)
    many, _ = make_policy(0, 99, masked=False)
    dist = many.distribution(ts.restart(x, batch_size=2)).action
    assert dist.most_likely(64)[0].shape == (2, 64)
    with pytest.raises(ValueError, match="top_k"):
        dist.most_likely(65)
