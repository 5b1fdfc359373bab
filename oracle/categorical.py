"""float64 numpy statement of Categorical(logits / temperature) with an action mask (TEST
INFRASTRUCTURE): log_prob, entropy, most likely alternatives, gradient with respect to the logits.

Rows are independent.  A masked action has probability 0 and gradient 0; a negative action marks a
padding row (log_prob, entropy, gradient 0; no alternatives); a row without an allowed finite logit has
log_prob -inf, entropy 0, gradient 0; NaN or +inf in an allowed place makes the row NaN.
"""
import numpy as np


def _masked(logits, mask):
    x = np.asarray(logits, np.float64)
    return x if mask is None else np.where(np.asarray(mask) != 0, x, -np.inf)


def forward(logits, actions, mask=None, temperature=1.0, top_k=0):
    """[N, A] logits, [N] actions -> (log_prob, entropy, ids, top log-probabilities, log p [N, A])."""
    x = _masked(logits, mask)
    n, a = x.shape
    log_prob, entropy = np.zeros(n), np.zeros(n)
    k = min(top_k, a)
    ids = np.full((n, k), -1, np.int64)
    top = np.full((n, k), -np.inf)
    logp = np.full((n, a), -np.inf)
    for i in range(n):
        act = -1 if actions is None else int(actions[i])
        if actions is not None and act < 0:
            continue
        row = x[i]
        if np.isnan(row).any() or (row == np.inf).any():
            logp[i] = log_prob[i] = entropy[i] = np.nan
            top[i] = np.nan
            continue
        if (row == -np.inf).all():
            log_prob[i] = -np.inf if actions is None or act < a else np.nan
            continue
        z = (row - row.max()) / temperature
        lp = z - np.log(np.exp(z).sum())
        logp[i] = lp
        p = np.exp(lp)
        entropy[i] = -(p[p > 0] * lp[p > 0]).sum()
        if actions is not None:
            log_prob[i] = lp[act] if act < a else np.nan
        order = np.lexsort((np.arange(a), -row))[:k]
        real = row[order] > -np.inf
        ids[i, :len(order)] = np.where(real, order, -1)
        top[i, :len(order)] = np.where(real, lp[order], -np.inf)
    return log_prob, entropy, ids, top, logp


def gradient(logits, actions, dlog_prob, dentropy, mask=None, temperature=1.0):
    """sum_r dlog_prob[r] d log_prob[r] + dentropy[r] d entropy[r] with respect to the logits."""
    _, entropy, _, _, logp = forward(logits, actions, mask, temperature)
    p = np.exp(logp)
    n, a = p.shape
    g = np.zeros(n) if dlog_prob is None else np.asarray(dlog_prob, np.float64)
    h = np.zeros(n) if dentropy is None else np.asarray(dentropy, np.float64)
    safe = np.where(p > 0, logp, 0.0)
    d = -g[:, None] * p - h[:, None] * p * (safe + entropy[:, None])
    for i in range(n):
        act = -1 if actions is None else int(actions[i])
        if (actions is not None and act < 0) or (logp[i] == -np.inf).all():
            d[i] = 0.0
        elif actions is not None and dlog_prob is not None:
            if act < a:
                d[i, act] += g[i]
            else:
                d[i] = np.nan
    d /= temperature
    return d if mask is None else np.where(np.asarray(mask) != 0, d, 0.0)
