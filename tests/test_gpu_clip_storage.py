"""What a kept norm keeps: its own values, not the scratch of the call it came from."""
import pytest
import torch

from agents_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_a_norm_is_an_allocation_of_its_own(dev, dtype):
    gen = torch.Generator(device=dev).manual_seed(1)
    grads = [torch.randn(n, generator=gen, device=dev).to(dtype) for n in (5, 300_001, 1, 0, 77)]
    plain = torch.cat([g.double() for g in grads]).norm()
    place = [torch.empty_like(g) for g in grads]
    for out in (None, place, grads):
        keep = [g.clone() for g in grads]
        clipped, norm = ops.clip_by_global_norm(grads, 2.0, out=out)
        assert norm.untyped_storage().nbytes() == 4
        # rounded once from a sum in float64
        assert abs(float(norm.double() - plain)) <= 2.0 ** -23 * float(plain)
        want, _ = ops.clip_by_global_norm(keep, 2.0)
        assert all(torch.equal(a, b) for a, b in zip(clipped, want))
    norms = ops.clip_by_norms(keep, 2.0)[1]
    assert norms.untyped_storage().nbytes() == 4 * len(keep)
    assert ops.global_norm(keep).untyped_storage().nbytes() == 4


def test_results_of_calls_in_a_row_stay(dev):
    """The scratch behind one call's results is not another call's."""
    gen = torch.Generator(device=dev).manual_seed(2)
    lists = [[torch.randn(n, generator=gen, device=dev).half() for n in (4097, 3, 70_000)] for _ in range(6)]
    got = [ops.clip_by_global_norm(g, 1.0) for g in lists]
    for (clipped, norm), g in zip(got, lists):
        again, n2 = ops.clip_by_global_norm([t.clone() for t in g], 1.0)
        assert torch.equal(norm, n2) and all(torch.equal(a, b) for a, b in zip(clipped, again))
