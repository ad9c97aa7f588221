"""Reordering of states together with what else a search keeps for each beam: lengths, token ids, rows of odd sizes."""
import pytest
import torch

from test_gpu_beam_masks import _time

pytestmark = pytest.mark.gpu

B, K = 64, 4


def _tensors(cuda):
    g = torch.Generator().manual_seed(3)
    states = [torch.randn(B * K, 32, 64, 64, generator=g).to(cuda), torch.randn(B * K, 2, 2048, generator=g).bfloat16().to(cuda)]
    small = [torch.arange(B * K, device=cuda), torch.arange(B * K, device=cuda, dtype=torch.int32).mul(7),
             torch.randn(B * K, 3, generator=g).bfloat16().to(cuda), torch.randn(B * K, 5, 2, generator=g).to(cuda)]
    parents = torch.randint(0, K, (B, K), generator=g, dtype=torch.int32).to(cuda)
    return states, small, parents


@pytest.mark.parametrize("in_place", [False, True])
def test_tensors_of_all_row_sizes(pkg, cuda, in_place):
    states, small, parents = _tensors(cuda)
    both = [t for pair in zip(small, states + states) for t in pair][:6] + small[3:]   # (in between one another)
    both = [t.clone() for t in both]
    rows = (torch.arange(B, device=cuda)[:, None] * K + parents).flatten()
    want = [t[rows] for t in both]
    out = None if in_place else [torch.empty_like(t) for t in both]
    got = pkg.beam_reorder(both, parents, out=out)
    assert pkg.read_device_status(0) == 0
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("which", [0, 1, 2])
def test_a_small_tensor_does_not_slow_the_states_down(pkg, cuda, which):
    states, small, parents = _tensors(cuda)
    out = [torch.empty_like(t) for t in states]
    alone = _time(lambda: pkg.beam_reorder(states, parents, out=out))
    with_small = _time(lambda: pkg.beam_reorder([*states, small[which]], parents, out=[*out, torch.empty_like(small[which])]))
    # one launch more at most, 5 of 38 us
    assert with_small < 1.4 * alone, (alone, with_small)
