"""CPU: the clipping calls own the tensors of their lists for as long as the call lasts."""
import weakref

import pytest
import torch

from agents_amd import _lib, ops

pytestmark = pytest.mark.usefixtures("lib")


@pytest.mark.parametrize("fn", [ops.clip_by_global_norm, ops.clip_by_norms])
def test_a_list_emptied_during_the_call(fn):
    """Whatever runs during a call (a number's own conversion, another thread while a launch waits) may
    change the caller's list; the tensors stay."""
    grads = [torch.zeros(5), torch.zeros(3, 2)]
    seen = [weakref.ref(g) for g in grads]
    alive = []

    class Limit:
        def __float__(self):
            grads.clear()
            alive.extend(r() is not None for r in seen)
            return 1.0

    with pytest.raises(_lib.AgentsAmdError, match="device tensors"):
        fn(grads, Limit())
    assert alive == [True, True]
    assert [r() for r in seen] == [None, None]       # and are released with it


def test_any_sequence():
    with pytest.raises(_lib.AgentsAmdError, match="device tensors"):
        ops.clip_by_global_norm((t for t in (torch.zeros(3), torch.zeros(2))), 1.0)
    with pytest.raises(TypeError):
        ops.clip_by_global_norm(None, 1.0)
