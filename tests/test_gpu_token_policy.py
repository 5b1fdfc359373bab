"""The token operators as a policy's training and serving use them together: LayerNormalization inside
Sequential, the log-probability loss on its head with the gradient, clipping, the optimizer; Categorical
distributions of the discrete policies; clipping of (gradient, variable) pairs.

Reference: torch autograd in float64 on the CPU.  A gradient of these networks passes at most six
products of at most 150 terms and as many normalisations of at most 64: with 2^-24 a rounding, chains of
at most 400 additions in all and a norm of |terms| over |sum| below 8, tensors agree to
400 * 8 * 2^-24 = 2e-4 of their largest entry.
"""
import numpy as np
import pytest
import torch

from agents_amd import ops, optimizers
from agents_amd.agents.dqn import dqn_agent
from agents_amd.drivers import dynamic_step_driver
from agents_amd.environments import random_tf_environment
from agents_amd.networks import layers as L
from agents_amd.networks import sequential
from agents_amd.policies import boltzmann_policy, q_policy
from agents_amd.replay_buffers import tf_uniform_replay_buffer as rb_lib
from agents_amd.specs import tensor_spec
from agents_amd.train import learner
from agents_amd.trajectories import time_step as ts
from agents_amd.utils import common, eager_utils, graph

pytestmark = pytest.mark.gpu

TOL = 2e-4


def close(got, want, tol=TOL):
    want = want.detach().double()
    scale = max(float(want.abs().max()), 1e-6)
    err = float((got.detach().double().cpu() - want).abs().max())
    assert err <= tol * scale, (err, scale)


def act(x, name):
    return torch.relu(x) if name == "relu" else torch.tanh(x) if name == "tanh" else x


def reference(layers, weights, x):
    """The stack in float64 with autograd; weights: leaves in `variables` order."""
    w = iter(weights)
    h = x.double()
    for l in layers:
        if isinstance(l, L.Flatten):
            h = h.reshape(h.shape[0], -1)
        elif isinstance(l, L.Dense):
            k, b = next(w), next(w)
            h = act(h.reshape(h.shape[0], -1) @ k + b, l.activation)
        elif isinstance(l, L.Conv2D):
            k, b = next(w), next(w)
            y = torch.nn.functional.conv2d(h.permute(0, 3, 1, 2), k.permute(3, 2, 0, 1), b, l.stride)
            h = act(y.permute(0, 2, 3, 1), l.activation)
        else:
            g, b = next(w), next(w)
            m = h.mean(-1, keepdim=True)
            h = (h - m) / (((h - m) ** 2).mean(-1, keepdim=True) + l.epsilon).sqrt() * g + b
    return h


STACKS = {
    "dense": ((20,), lambda: [L.Dense(48, "relu"), L.LayerNormalization(), L.Dense(33, "tanh"),
                              L.LayerNormalization(epsilon=1e-5), L.Dense(7)]),
    "first": ((31,), lambda: [L.LayerNormalization(), L.Dense(64, "tanh"), L.Dense(6)]),
    "last": ((12,), lambda: [L.Dense(70, "tanh"), L.LayerNormalization()]),
    "twice": ((12,), lambda: [L.Dense(70), L.LayerNormalization(), L.LayerNormalization(), L.Dense(3)]),
    "conv": ((8, 8, 4), lambda: [L.Conv2D(16, 3, 1, "tanh"), L.LayerNormalization(),
                                 L.Conv2D(12, 2, 2, "tanh"), L.LayerNormalization(), L.Flatten(),
                                 L.Dense(40, "tanh"), L.LayerNormalization(), L.Dense(5)]),
    "conv-flat": ((9, 9, 4), lambda: [L.Conv2D(16, 3, 2, "tanh"), L.Flatten(), L.LayerNormalization(),
                                      L.Dense(40, "tanh"), L.Dense(5)]),
    "conv-unflattened": ((9, 9, 4), lambda: [L.Conv2D(16, 3, 2, "tanh"), L.LayerNormalization(),
                                             L.Dense(5)]),
    "before-conv": ((9, 9, 4), lambda: [L.LayerNormalization(), L.Conv2D(16, 3, 1, "tanh"),
                                        L.Conv2D(16, 3, 1, "tanh"), L.Flatten(), L.Dense(5)]),
}


def build(name, dev, seed=3):
    shape, make = STACKS[name]
    net = sequential.Sequential(make(), input_spec=tensor_spec.TensorSpec(shape, torch.float32),
                                seed=seed)
    net.create_variables(device=dev)
    rng = np.random.RandomState(seed)
    net.set_weights([w + 0.1 * rng.randn(*w.shape).astype(np.float32) for w in net.get_weights()])
    return net, shape


@pytest.mark.parametrize("name", list(STACKS))
@pytest.mark.parametrize("side", [False, True])
def test_sequential_with_layer_normalization(dev, name, side):
    net, shape = build(name, dev)
    B = 9
    x = torch.randn(B, *shape, generator=torch.Generator().manual_seed(1))
    leaves = [v.detach().cpu().double().requires_grad_() for v in net.variables]
    xr = x.double().requires_grad_()
    want = reference(net.layers, leaves, xr)
    y = net.forward(x.to(dev), slot="t", need_grad=True)
    close(y, want)
    dout = torch.randn(want.shape, generator=torch.Generator().manual_seed(2))
    (want * dout.double()).sum().backward()
    stream = ops.new_side_stream(dev) if side else None
    dense_first = not name.startswith("conv")
    dx = torch.zeros(B, *shape, device=dev) if dense_first else None
    net.backward(dout.to(dev), slot="t", side_stream=stream, input_grad=dx)
    torch.cuda.synchronize()
    for g, l in zip(net.gradients, leaves):
        close(g, l.grad)
    if dense_first:
        close(dx, xr.grad)
        # the input-gradient chain alone leaves the weights' gradients as they are
        before = net.flat_grads.clone()
        dx2 = torch.zeros_like(dx)
        net.backward(dout.to(dev), slot="t", param_grads=False, input_grad=dx2)
        assert torch.equal(before, net.flat_grads) and torch.equal(dx, dx2)
    assert len(net.kernels) == sum(isinstance(l, (L.Dense, L.Conv2D)) for l in net.layers)
    # a copy has the same values
    assert torch.equal(net.copy().forward(x.to(dev)), net.forward(x.to(dev)))


def test_layer_normalization_refusals():
    for kw in (dict(axis=1), dict(center=False), dict(scale=False)):
        with pytest.raises(NotImplementedError):
            L.LayerNormalization(**kw)
    with pytest.raises(ValueError):
        L.LayerNormalization(epsilon=-1.0)
    net = sequential.Sequential([L.Rescale(255.0), L.LayerNormalization()],
                                input_spec=tensor_spec.TensorSpec((4,), torch.float32))
    net.create_variables(device="cuda")
    with pytest.raises(NotImplementedError):
        net.forward(torch.zeros(2, 4, device="cuda"))


V = 151


def token_step(net, opt, x, tokens, mask, adv):
    """One policy-gradient step over [B] tokens: logits, log-probabilities, -mean(adv log p) -
    0.01 mean H, its gradient, clipped by the global norm, Adam."""
    B = x.shape[0]
    logits = net.forward(x, slot="t", need_grad=True)
    r = ops.categorical_log_prob(logits, tokens, mask=mask, top_k=4)
    d = ops.categorical_log_prob_backward(logits, tokens, r, -adv / B,
                                          torch.full_like(adv, -0.01 / B), mask=mask)
    net.backward(d, slot="t")
    clipped, norm = ops.clip_by_global_norm(net.gradients, 0.05, out=net.gradients)
    opt.apply_flat(net.flat_params, net.flat_grads)
    return r, norm


def token_net(dev):
    net = sequential.Sequential(
        [L.Dense(64, "tanh"), L.LayerNormalization(), L.Dense(64, "tanh"), L.LayerNormalization(),
         L.Dense(V)], input_spec=tensor_spec.TensorSpec((24,), torch.float32), seed=1)
    net.create_variables(device=dev)
    return net


def token_batch(dev, seed):
    g = torch.Generator().manual_seed(seed)
    x, adv = torch.randn(32, 24, generator=g), torch.randn(32, generator=g)
    mask = torch.rand(32, V, generator=g) < 0.7
    tokens = torch.randint(0, V, (32,), generator=g)
    mask[torch.arange(32), tokens] = True
    tokens[3] = -1
    return [t.to(dev) for t in (x, tokens, mask, adv)]


def test_training_step_of_a_token_policy(dev):
    net, opt = token_net(dev), optimizers.Adam(1e-3)
    x, tokens, mask, adv = token_batch(dev, 0)
    leaves = [v.detach().cpu().double().requires_grad_() for v in net.variables]
    logits = reference(net.layers, leaves, x.cpu())
    logp = torch.log_softmax(logits.masked_fill(~mask.cpu(), float("-inf")), 1)
    real = tokens.cpu() >= 0
    lp = logp.gather(1, tokens.cpu().clamp(min=0)[:, None])[:, 0]
    ent = -(logp.exp() * logp.masked_fill(~mask.cpu(), 0.0)).sum(1)
    loss = -(adv.cpu().double() * lp + 0.01 * ent)[real].sum() / 32
    loss.backward()
    norm = torch.sqrt(sum((l.grad ** 2).sum() for l in leaves))
    r, n = token_step(net, opt, x, tokens, mask, adv)
    close(r.log_prob, torch.where(real, lp, torch.zeros_like(lp)))
    close(r.entropy, torch.where(real, ent, torch.zeros_like(ent)))
    close(n.reshape(1), norm.reshape(1))
    for g, l in zip(net.gradients, leaves):
        close(g, l.grad * min(1.0, 0.05 / float(norm)))


def test_training_step_replays_from_a_graph(dev):
    """The captured step, replayed between eager work, walks the parameters of the eager one."""
    eager, graphed = token_net(dev), token_net(dev)
    oe, og = optimizers.Adam(1e-3), optimizers.Adam(1e-3)
    batches = [token_batch(dev, s) for s in range(4)]
    live = [t.clone() for t in batches[0]]
    for net, opt in ((eager, oe), (graphed, og)):
        token_step(net, opt, *batches[0])              # workspaces, slots
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rg, ng = token_step(graphed, og, *live)
    for i in range(8):
        for a, b in zip(live, batches[i % 4]):
            a.copy_(b)
        g.replay()
        re, ne = token_step(eager, oe, *batches[i % 4])
        torch.cuda.synchronize()
        assert torch.equal(ne, ng)
        for p, q in zip(re, rg):
            assert torch.equal(p, q)
        assert torch.equal(eager.flat_params, graphed.flat_params)


def test_dqn_agent_with_layer_normalization_graphs_match_eager(dev):
    def stack(ring):
        obs = tensor_spec.TensorSpec((12, 12, 4), torch.uint8, "observation")
        aspec = tensor_spec.BoundedTensorSpec((), torch.int64, 0, 3, "action")
        tss = ts.time_step_spec(obs)
        env = random_tf_environment.RandomTFEnvironment(tss, aspec, batch_size=8, seed=11,
                                                        episode_end_probability=0.2, device=dev)
        net = sequential.Sequential(
            [L.Rescale(255.0), L.Conv2D(8, 4, 4, "relu"), L.LayerNormalization(), L.Flatten(),
             L.Dense(32, "relu"), L.LayerNormalization(), L.Dense(4)], seed=3)
        agent = dqn_agent.DqnAgent(tss, aspec, q_network=net, optimizer=optimizers.Adam(1e-3),
                                   td_errors_loss_fn=common.element_wise_huber_loss, gamma=0.9,
                                   epsilon_greedy=0.3, target_update_period=3, seed=5)
        agent.initialize()
        rb = rb_lib.TFUniformReplayBuffer(agent.collect_data_spec, batch_size=8, max_length=64,
                                          device=dev, seed=9, dataset_ring=ring)
        drv = dynamic_step_driver.DynamicStepDriver(env, agent.collect_policy,
                                                    observers=[rb.add_batch], num_steps=1)
        return agent, rb, drv, net

    ag_e, rb_e, drv_e, net_e = stack(0)
    ag_g, rb_g, drv_g, net_g = stack(8)
    run_g = common.function(drv_g.run)
    lrn = learner.Learner(None, common.Variable(0), ag_g)
    for _ in range(4):
        drv_e.run()
        run_g()
    it_g = iter(rb_g.as_dataset(sample_batch_size=16, num_steps=2))
    ts_e = ts_g = None
    start = net_e.flat_params.clone()
    for i in range(20):
        ts_e, _ = drv_e.run(ts_e)
        exp_e, _ = rb_e.get_next(16, 2)
        li_e = ag_e.train(exp_e)
        ts_g, _ = run_g(ts_g)
        li_g = lrn.run(iterations=1, iterator=it_g)
        assert torch.equal(net_e.flat_params, net_g.flat_params), f"params diverged at step {i}"
        assert float(li_e.loss) == float(li_g.loss)
    assert not torch.equal(start, net_e.flat_params)
    assert graph.graphed_train(ag_g).replays > 10


# ---- distributions of the discrete policies -----------------------------------------------------
def test_categorical_distribution_of_a_policy(dev):
    obs = {"x": tensor_spec.TensorSpec((3,), torch.float32),
           "mask": tensor_spec.BoundedTensorSpec((5,), torch.int32, 0, 1)}
    aspec = tensor_spec.BoundedTensorSpec((), torch.int64, 2, 6, "action")
    net = sequential.Sequential([L.Dense(5)], input_spec=obs["x"], seed=4)
    policy = q_policy.QPolicy(ts.time_step_spec(obs), aspec, q_network=net,
                              observation_and_action_constraint_splitter=lambda o: (o["x"], o["mask"]))
    net.set_weights([w + 0.3 for w in net.get_weights()])
    x = torch.randn(4, 3, generator=torch.Generator().manual_seed(0)).to(dev)
    mask = torch.tensor([[1, 1, 1, 1, 1], [1, 0, 1, 0, 1], [0, 0, 0, 1, 0], [1, 1, 0, 0, 0]],
                        dtype=torch.int32, device=dev)
    step = ts.restart({"x": x, "mask": mask}, batch_size=4)
    for temperature in (None, 0.5):
        p = policy if temperature is None else boltzmann_policy.BoltzmannPolicy(policy, temperature)
        dist = p.distribution(step).action
        q = net.forward(x).double().cpu() / (temperature or 1.0)
        want = torch.log_softmax(q.masked_fill(mask.cpu() == 0, float("-inf")), 1)
        actions = torch.tensor([2, 4, 5, 3], device=dev)
        lp = common.log_probability(dist, actions)
        # four values of size below 4: a few roundings each
        close(lp, want.gather(1, (actions.cpu() - 2)[:, None])[:, 0], 1e-6)
        close(common.entropy(dist), -(want.exp() * want.clamp(min=-1e30)).sum(1), 1e-6)
        ids, best = dist.most_likely(2)
        top = want.sort(1, descending=True)
        assert torch.equal(ids.cpu()[:2], top.indices[:2, :2] + 2)
        assert int(ids[2, 0]) == 5 and torch.equal(ids[:, :1].cpu(), dist.mode().cpu()[:, None])
        close(best[:2], top.values[:2, :2], 1e-6)
        both = common.log_probability((dist, dist), (actions, actions))
        assert torch.equal(both, lp + lp)


# ---- (gradient, variable) pairs -------------------------------------------------------------------
def test_clipping_of_pairs(dev):
    gen = torch.Generator(device=dev).manual_seed(0)
    shapes = [(17, 5), (5,), (3, 3, 2), ()]
    grads = [torch.randn(s, generator=gen, device=dev) for s in shapes]
    vs = [torch.zeros(s, device=dev) for s in shapes] + [torch.zeros(2, device=dev)]
    pairs = list(zip(grads[:2] + [None] + grads[2:], vs[:2] + [vs[4]] + vs[2:4]))
    got = eager_utils.clip_gradient_norms(pairs, 1.5)
    assert got[2][0] is None and all(a[1] is b[1] for a, b in zip(got, pairs))
    for (g, _), (o, _) in zip(got, pairs):
        if o is not None:
            n = float(o.double().norm())
            # factor, product and the comparison's own rounding: 3 * 2^-24
            close(g, o.double().cpu() * min(1.0, 1.5 / n), 4 * 2.0 ** -24)
    got, norm = eager_utils.clip_gradients_by_global_norm(pairs, 0.7)
    n = float(torch.cat([g.reshape(-1) for g in grads]).double().norm())
    assert abs(float(norm) - n) <= 2.0 ** -23 * n
    for (g, _), (o, _) in zip(got, pairs):
        if o is not None:
            close(g, o.double().cpu() * 0.7 / n, 4 * 2.0 ** -24)
    optimizers.SGD(0.5).apply_gradients(got)
    for (g, v), _ in zip(got, pairs):
        if g is not None:
            assert torch.equal(v, -0.5 * g)
    none = [(None, vs[0])]
    assert eager_utils.clip_gradient_norms(none, 1.0) == none
    assert eager_utils.clip_gradients_by_global_norm(none, 1.0) == (none, None)
