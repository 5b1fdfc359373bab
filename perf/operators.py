"""Cases of three groups of operators, their plain forms and the calls of this package for them.

  categorical   log-probabilities of given tokens (actions) under softmax(logits / temperature), with the
                entropy and the most likely alternatives; for training the gradient with respect to the logits
  clip          the norm of many gradient tensors and the clipped tensors, over all of them together
                (`global`) or over each by itself (`each`)
  layer_norm    layer normalisation; for training its gradient with respect to the input and both weights

Where `own` is false `run` computes them with elementary torch operations in 32 bits, rounded once at the end;
where it is true it calls agents_amd.  `exact` gives the same outputs in 64 bits from the definitions.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_MASK_BYTES = {"none": 0, "byte": 1, "int32": 4}

# what the largest listed cases hold; a drawn case stays below
_MOST_LOGITS = 4096 * 32768
_MOST_GRADS = 200_000_000
_MOST_NORM = 8192 * 4096

# trunk of a token policy, [vocabulary x width] and blocks of [width x 4 width] matrices
_TRUNK = "32000x2048 2048 2048x6144 2048x2048 2048x8192 8192x2048 2048 2048 2048x6144 2048x2048 2048x8192 8192x2048 2048 2048"
# the Atari Q-network: three convolutions, 512 units, 6 actions; a kernel and a bias each
_ATARI = "8x8x4x32 32 4x4x32x64 64 3x3x64x64 64 3136x512 512 512x6 6"
# a 256-256 actor and its two critics on a 376-dimensional observation and 17 actions
_ACTOR_CRITICS = ("376x256 256 256x256 256 256x34 34 393x256 256 256x256 256 256x1 1 "
                  "393x256 256 256x256 256 256x1 1")


def listed():
    return [
        # one token of one sequence is chosen: its alternatives are shown beside it
        {"name": "serve-1x131072-bf16", "op": "categorical", "outer": 1, "inner": 1, "cut": 0, "vocab": 131072,
         "type": "bf16", "mask": "none", "temperature": 1.0, "top": 20, "train": False},
        # a batch of sequences, one token each, with a grammar's mask and a temperature
        {"name": "serve-64x50001-f32", "op": "categorical", "outer": 64, "inner": 1, "cut": 0, "vocab": 50001,
         "type": "f32", "mask": "byte", "temperature": 0.7, "top": 8, "train": False},
        # a minibatch of an agent with a small set of actions and an action mask
        {"name": "actions-4096x18-f32", "op": "categorical", "outer": 4096, "inner": 1, "cut": 0, "vocab": 18,
         "type": "f32", "mask": "int32", "temperature": 1.0, "top": 0, "train": True},
        # a minibatch of tokens
        {"name": "tokens-4096x32768-bf16", "op": "categorical", "outer": 4096, "inner": 1, "cut": 0, "vocab": 32768,
         "type": "bf16", "mask": "none", "temperature": 1.0, "top": 0, "train": True},
        # whole sequences: position t's logits against token t + 1, so both are slices; an odd vocabulary
        {"name": "shifted-4x511x50001-f16", "op": "categorical", "outer": 4, "inner": 512, "cut": 1, "vocab": 50001,
         "type": "f16", "mask": "none", "temperature": 1.0, "top": 0, "train": True},
        # a step of the Atari agent
        {"name": "clip-atari-global", "op": "clip", "shapes": _ATARI, "type": "f32", "mode": "global", "share": 0.4},
        # a step of an actor-critic agent that clips each tensor by itself
        {"name": "clip-actor-critics-each", "op": "clip", "shapes": _ACTOR_CRITICS, "type": "f32", "mode": "each",
         "share": 0.4},
        # a step of a token policy
        {"name": "clip-trunk-global", "op": "clip", "shapes": _TRUNK, "type": "bf16", "mode": "global", "share": 0.4},
        # one token of one sequence
        {"name": "norm-1x4096-bf16", "op": "layer_norm", "rows": 1, "width": 4096, "type": "bf16", "train": False},
        # a hidden layer of 512 units at the Atari agent's batch
        {"name": "norm-256x512-f32", "op": "layer_norm", "rows": 256, "width": 512, "type": "f32", "train": True},
        # odd sizes
        {"name": "norm-3001x1003-f16", "op": "layer_norm", "rows": 3001, "width": 1003, "type": "f16", "train": True},
        # a minibatch of tokens
        {"name": "norm-8192x4096-bf16", "op": "layer_norm", "rows": 8192, "width": 4096, "type": "bf16", "train": True},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["categorical", "categorical", "clip", "layer_norm"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op == "categorical":
        vocab = _spread(rng, 2, 160_000)
        train = rng.random() < 0.5
        # half of what the largest listed case holds where the type is twice as wide or a mask is read too
        inner = rng.choice([1, _spread(rng, 2, 64)])
        outer = _spread(rng, 1, max(1, min(8192, _MOST_LOGITS // (2 * vocab * inner))))
        return {"op": op, "outer": outer, "inner": inner, "cut": 1 if inner > 1 else 0, "vocab": vocab, "type": kind,
                "mask": rng.choice(["none", "none", "byte", "int32"]), "temperature": rng.choice([1.0, 0.7, 1.3]),
                "top": 0 if train else rng.randint(0, 24), "train": train}
    if op == "clip":
        total = _spread(rng, 1000, _MOST_GRADS // (2 if kind == "f32" else 1))
        parts = [rng.random() ** 3 + 1e-6 for _ in range(rng.randint(1, 24))]
        return {"op": op, "shapes": " ".join(str(max(1, int(total * p / sum(parts)))) for p in parts), "type": kind,
                "mode": rng.choice(["global", "global", "each"]), "share": rng.choice([0.1, 0.5, 2.0])}
    width = _spread(rng, 2, 20_000)
    rows = _spread(rng, 1, max(1, min(65_536, _MOST_NORM // (2 * width))))
    return {"op": op, "rows": rows, "width": width, "type": kind, "train": rng.random() < 0.7}


def _shapes(case):
    return [tuple(int(n) for n in s.split("x")) for s in case["shapes"].split()]


def _positions(case):
    return case["inner"] - case["cut"]


# ---- inputs ---------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 11)
    dtype = _TYPES[case["type"]]

    def normal(*shape, scale=1.0, mean=0.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale + mean

    if case["op"] == "categorical":
        n, t, vocab, keep = case["outer"], case["inner"], case["vocab"], _positions(case)
        logits = normal(n, t, vocab, scale=2.5)
        tokens = torch.randint(0, vocab, (n, t), generator=g, device="cuda")
        # the tokens of a sequence are mostly ones that its policy finds likely
        lift = normal(n, t, 1, scale=3.0, mean=6.0)
        if t > 1:
            logits[:, :-1].scatter_add_(2, tokens[:, 1:, None], lift[:, 1:])
        else:
            logits.scatter_add_(2, tokens[:, :, None], lift)
        logits = logits.to(dtype)[:, :keep]
        tokens = tokens[:, t - keep:]
        mask = None
        if case["mask"] != "none":
            mask = torch.rand(n, keep, vocab, generator=g, device="cuda") < 0.8
            mask.scatter_(2, tokens[:, :, None], True)
            mask = mask.to(torch.int32) if case["mask"] == "int32" else mask
        state = {"logits": logits, "tokens": tokens, "mask": mask}
        if case["train"]:
            # padding behind the end of some sequences
            pad = torch.rand(n, keep, generator=g, device="cuda") < 0.03
            state["tokens"] = torch.where(pad, torch.full_like(tokens, -1), tokens)
            state["dlog_prob"] = normal(n, keep)
            state["dentropy"] = torch.full((n, keep), -0.01, device="cuda")
        return {"case": case, **state}
    if case["op"] == "clip":
        grads = [normal(*s, scale=0.02).to(dtype) for s in _shapes(case)]
        largest = max(x.numel() for x in grads) if case["mode"] == "each" else sum(x.numel() for x in grads)
        return {"case": case, "grads": grads, "limit": case["share"] * 0.02 * math.sqrt(largest)}
    rows, width = case["rows"], case["width"]
    state = {"x": normal(rows, width, scale=1.5, mean=0.3).to(dtype), "gamma": normal(width, scale=0.1, mean=1.0),
             "beta": normal(width, scale=0.1), "epsilon": 1e-3}
    if case["train"]:
        state["dy"] = normal(rows, width).to(dtype)
    return {"case": case, **state}


# ---- plain forms ------------------------------------------------------------------------------
def _plain_categorical(s):
    case, logits, tokens = s["case"], s["logits"], s["tokens"]
    x = logits.float() / case["temperature"]
    raw = logits.float() + 0.0
    if s["mask"] is not None:
        allowed = s["mask"] != 0
        x = torch.where(allowed, x, -math.inf)
        raw = torch.where(allowed, raw, -math.inf)
    high = x.amax(-1, keepdim=True)
    e = (x - high).exp()
    total = e.sum(-1, keepdim=True)
    log_p = x - high - total.log()
    p = e / total
    entropy = -torch.where(p > 0, p * log_p, 0.0).sum(-1)
    real = tokens >= 0
    at = tokens.clamp(min=0)[..., None]
    log_prob = torch.where(real, log_p.gather(-1, at)[..., 0], 0.0)
    entropy = torch.where(real, entropy, 0.0)
    if case["train"]:
        g = s["dlog_prob"][..., None]
        h = s["dentropy"][..., None]
        dx = -g * p - h * torch.where(p > 0, p * (log_p + entropy[..., None]), 0.0)
        dx = dx.scatter_add(-1, at, g) / case["temperature"]
        dx = torch.where(real[..., None], dx, 0.0)
        if s["mask"] is not None:
            dx = torch.where(allowed, dx, 0.0)
        return {"log_prob": log_prob, "entropy": entropy, "dlogits": dx.to(logits.dtype)}
    out = {"log_prob": log_prob, "entropy": entropy}
    if case["top"]:
        # larger logits first and, among equal ones, the lower index: both in one whole number
        bits = raw.view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        vocab = raw.shape[-1]
        keys = order * (1 << 20) + (vocab - 1 - torch.arange(vocab, device=raw.device))
        k = min(case["top"], vocab)
        ids = vocab - 1 - (keys.topk(k, -1).values & ((1 << 20) - 1))
        best = log_p.gather(-1, ids)
        out["top_ids"] = torch.where(raw.gather(-1, ids) > -math.inf, ids, -1)
        out["top_log_prob"] = best
    return out


def _plain_clip(s):
    grads, limit = s["grads"], s["limit"]
    squares = torch.stack([x.float().square().sum(dtype=torch.float64) for x in grads])
    if s["case"]["mode"] == "global":
        squares = squares.sum().reshape(1)
    norms = squares.sqrt().float()
    scales = limit / norms.clamp(min=limit)
    scales = scales.expand(len(grads)).unbind(0)
    out = norms.reshape(()) if s["case"]["mode"] == "global" else norms
    return {"norm": out, "clipped": [(x.float() * c).to(x.dtype) for x, c in zip(grads, scales)]}


def _plain_layer_norm(s):
    x = s["x"].float()
    mean = x.mean(-1, keepdim=True)
    centred = x - mean
    rstd = 1.0 / (centred.square().mean(-1, keepdim=True) + s["epsilon"]).sqrt()
    hat = centred * rstd
    y = hat * s["gamma"] + s["beta"]
    out = {"y": y.to(s["x"].dtype)}
    if s["case"]["train"]:
        dy = s["dy"].float()
        d = dy * s["gamma"]
        dx = rstd * (d - d.mean(-1, keepdim=True) - hat * (d * hat).mean(-1, keepdim=True))
        out["dx"] = dx.to(s["x"].dtype)
        out["dgamma"] = (dy * hat).sum(0)
        out["dbeta"] = dy.sum(0)
    return out


# ---- the package's calls --------------------------------------------------------------------------
def _own_categorical(s):
    from agents_amd import ops
    case, logits, tokens, mask = s["case"], s["logits"], s["tokens"], s["mask"]
    r = ops.categorical_log_prob(logits, tokens, mask=mask, temperature=case["temperature"], top_k=case["top"])
    out = {"log_prob": r.log_prob, "entropy": r.entropy}
    if case["train"]:
        out["dlogits"] = ops.categorical_log_prob_backward(logits, tokens, r, s["dlog_prob"], s["dentropy"], mask=mask,
                                                           temperature=case["temperature"])
    elif case["top"]:
        out["top_ids"], out["top_log_prob"] = r.top_ids, r.top_log_prob
    return out


def _own_clip(s):
    from agents_amd import ops
    if s["case"]["mode"] == "global":
        clipped, norm = ops.clip_by_global_norm(s["grads"], s["limit"])
    else:
        clipped, norm = ops.clip_by_norms(s["grads"], s["limit"])
    return {"norm": norm, "clipped": clipped}


def _own_layer_norm(s):
    from agents_amd import ops
    y, stats = ops.layer_norm_forward(s["x"], s["gamma"], s["beta"], s["epsilon"])
    out = {"y": y}
    if s["case"]["train"]:
        out["dx"], out["dgamma"], out["dbeta"] = ops.layer_norm_backward(s["dy"], s["x"], s["gamma"], stats)
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"categorical": _own_categorical, "clip": _own_clip, "layer_norm": _own_layer_norm}[op](state)
    return {"categorical": _plain_categorical, "clip": _plain_clip, "layer_norm": _plain_layer_norm}[op](state)


# ---- the definitions in 64 bits -------------------------------------------------------------------
def _exact_categorical(s):
    case = s["case"]
    shape = s["tokens"].shape
    rows = s["tokens"].numel()
    vocab = case["vocab"]
    z = s["logits"].reshape(rows, vocab)
    ids = s["tokens"].reshape(rows)
    keep = None if s["mask"] is None else s["mask"].reshape(rows, vocab)
    parts = {"log_prob": [], "entropy": [], "dlogits": [], "top_log_prob": []}
    step = max(1, 40_000_000 // vocab)
    for a in range(0, rows, step):
        b = min(rows, a + step)
        u = z[a:b].double() / case["temperature"]
        if keep is not None:
            u = u.masked_fill(keep[a:b] == 0, -math.inf)
        lse = torch.logsumexp(u, 1)
        lp = u - lse[:, None]
        prob = lp.exp()
        ent = torch.special.entr(prob).sum(1)
        padded = ids[a:b] < 0
        tok = ids[a:b].masked_fill(padded, 0)
        hit = lp[torch.arange(b - a, device=lp.device), tok]
        parts["log_prob"].append(hit.masked_fill(padded, 0.0))
        parts["entropy"].append(ent.masked_fill(padded, 0.0))
        if case["train"]:
            g = s["dlog_prob"].reshape(rows)[a:b].double()
            h = s["dentropy"].reshape(rows)[a:b].double()
            d = torch.zeros_like(prob)
            d[torch.arange(b - a, device=lp.device), tok] = g
            d -= prob * g[:, None]
            d += h[:, None] * (torch.special.entr(prob) - prob * ent[:, None])
            d /= case["temperature"]
            d[padded] = 0.0
            if keep is not None:
                d = d.masked_fill(keep[a:b] == 0, 0.0)
            parts["dlogits"].append(d)
        elif case["top"]:
            parts["top_log_prob"].append(lp.sort(1, descending=True).values[:, :min(case["top"], vocab)])
    out = {"log_prob": torch.cat(parts["log_prob"]).reshape(shape), "entropy": torch.cat(parts["entropy"]).reshape(shape)}
    if case["train"]:
        out["dlogits"] = torch.cat(parts["dlogits"]).reshape(*shape, vocab)
    elif case["top"]:
        out["top_ids"] = None
        out["top_log_prob"] = torch.cat(parts["top_log_prob"]).reshape(*shape, -1)
    return out


def _exact_clip(s):
    limit = float(s["limit"])
    lengths = [torch.linalg.vector_norm(x.double().flatten()) for x in s["grads"]]
    if s["case"]["mode"] == "global":
        length = torch.linalg.vector_norm(torch.stack(lengths))
        lengths, norm = [length] * len(lengths), length
    else:
        norm = torch.stack(lengths)
    clipped = [x.double() * min(1.0, limit / float(n)) if float(n) > 0 else x.double()
               for x, n in zip(s["grads"], lengths)]
    return {"norm": norm, "clipped": clipped}


def _exact_layer_norm(s):
    x = s["x"].double()
    n = x.shape[1]
    m = x.sum(1) / n
    var = (x * x).sum(1) / n - m * m
    r = (var + s["epsilon"]).rsqrt()
    gamma = s["gamma"].double()
    y = (x - m[:, None]) * (r[:, None] * gamma) + s["beta"].double()
    out = {"y": y}
    if s["case"]["train"]:
        dy = s["dy"].double()
        hat = (x - m[:, None]) * r[:, None]
        # the product of the three parts' Jacobians, each with respect to x
        dhat = dy * gamma
        dvar = -0.5 * (dhat * (x - m[:, None])).sum(1) * r ** 3
        dmean = -(dhat.sum(1) * r)
        out["dx"] = dhat * r[:, None] + dvar[:, None] * 2.0 * (x - m[:, None]) / n + dmean[:, None] / n
        out["dgamma"] = (dy * hat).sum(0)
        out["dbeta"] = dy.sum(0)
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return {"categorical": _exact_categorical, "clip": _exact_clip, "layer_norm": _exact_layer_norm}[case["op"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------
def work(case):
    if case["op"] == "categorical":
        rows = case["outer"] * _positions(case)
        n = rows * case["vocab"]
        size = n * (_BYTES[case["type"]] * (2 if case["train"] else 1) + _MASK_BYTES[case["mask"]])
        size += rows * (8 + 4 + 4 + (8 if case["train"] else 12 * case["top"]))
        return {"bytes": size, "flops": n * (14 if case["train"] else 6)}
    if case["op"] == "clip":
        n = sum(math.prod(s) for s in _shapes(case))
        return {"bytes": n * 2 * _BYTES[case["type"]], "flops": n * 3}
    n = case["rows"] * case["width"]
    return {"bytes": n * _BYTES[case["type"]] * (4 if case["train"] else 2) + case["width"] * (16 if case["train"] else 8),
            "flops": n * (20 if case["train"] else 8)}
