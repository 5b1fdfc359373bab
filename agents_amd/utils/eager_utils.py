"""Clipping of (gradient, variable) pairs before an optimizer's `apply_gradients`.

  clip_gradient_norms              tf_agents/utils/eager_utils.py:227-246  every gradient by its own norm
  clip_gradients_by_global_norm    tf.clip_by_global_norm over the pairs (ppo_agent.py:948-949)

Gradients are contiguous device tensors of one type in storage of their own; None stays None (a variable
that the loss does not reach).  Networks whose gradients lie in one flat buffer are clipped there
(aa_clip_by_norm); these take any list in two launches (csrc/grad_clip.hip).
"""
from agents_amd import ops


def _clip(gradients_to_variables, clip):
    pairs = list(gradients_to_variables)
    grads = [g for g, _ in pairs if g is not None]
    if not grads:
        return pairs, None
    clipped, norm = clip(grads)
    clipped = iter(clipped)
    return [(None if g is None else next(clipped), v) for g, v in pairs], norm


def clip_gradient_norms(gradients_to_variables, max_norm):
    """[(gradient * max_norm / max(its norm, max_norm), variable)] of a list of pairs."""
    return _clip(gradients_to_variables, lambda g: ops.clip_by_norms(g, max_norm))[0]


def clip_gradients_by_global_norm(gradients_to_variables, clip_norm):
    """([(gradient * clip_norm / max(global norm, clip_norm), variable)], global norm): the norm of all
    gradients together, a float32 scalar on the device (None without a gradient)."""
    return _clip(gradients_to_variables, lambda g: ops.clip_by_global_norm(g, clip_norm))
