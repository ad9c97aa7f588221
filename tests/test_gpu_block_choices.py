"""Every choice that beam search makes in a model of linear attention between its norms is one of the definition's, on the logits that
the model had at that step and the scores it went on from, in both types."""
import pytest
import torch

import block_reference as ref
from test_gpu_block_decode import BEAMS, V, Kernels, Plain, _decode, _weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("forced", [False, True])
def test_choices_are_the_definitions(pkg, cuda, dtype, forced):
    weights = _weights(dtype, cuda)
    prompts = torch.randint(0, V, (2, 150), generator=torch.Generator().manual_seed(5)).to(cuda)
    lens = torch.tensor([150, 61], dtype=torch.int32, device=cuda)
    follow = None
    if forced:
        wide = ([{n: t.double() for n, t in w.items()} for w in weights[0]], weights[1].double(), weights[2].double())
        follow = [(s.float(), p.int(), t, None) for s, p, t, _ in _decode(Plain(cuda), wide, prompts, lens, 6)[0]]
    trace, _ = _decode(Kernels(pkg, cuda), weights, prompts, lens, 6, force=follow)
    assert pkg.read_device_status(0) == 0
    before = torch.zeros(2, 1, device=cuda)
    for step, (scores, parents, tokens, logits) in enumerate(trace):
        best, want_parents, want_tokens = ref.beam_select(logits.view(2, before.shape[1], V), before, BEAMS)
        assert torch.equal(parents.long(), want_parents) and torch.equal(tokens.long(), want_tokens), step
        # a sum of 97 exponentials, each within two steps, and half a step of the score
        assert float((scores.double() - best).abs().max()) <= (97 / 256 + 24) * ref.U + ref.U * float(best.abs().max()), step
        before = scores if follow is None else follow[step][0]


def test_a_wrong_choice_would_be_seen(pkg, cuda):
    """The states follow the parents: two beams exchanged give other logits."""
    weights = _weights(torch.float32, cuda)
    prompts = torch.randint(0, V, (2, 40), generator=torch.Generator().manual_seed(6)).to(cuda)
    trace, _ = _decode(Kernels(pkg, cuda), weights, prompts, None, 3)

    class Exchanged(Kernels):
        def reorder(self, states, parents):
            return super().reorder(states, parents.flip(1).contiguous())

    other, _ = _decode(Exchanged(pkg, cuda), weights, prompts, None, 3, force=trace)
    moved = any(not torch.equal(p, p.flip(1)) for _, p, _, _ in trace[1:3])
    assert moved and not all(torch.equal(a[3], b[3]) for a, b in zip(trace, other))
