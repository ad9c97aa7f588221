"""The operators around a recurrent block together: a two-layer model of linear attention between its norms reads padded prompts,
then decodes them with beam search, its states reordered in place at every step.  Everything is compared with the same model in 64
bits.  Two tokens of a search are told apart by more than the bf16 activations are off: the head is scaled up, and the test checks
the gaps of the 64-bit model's own choices."""
import pytest
import torch

import block_reference as ref

pytestmark = pytest.mark.gpu

H, N, V, LAYERS, BEAMS, EPS = 4, 64, 97, 2, 3, 1e-5
C = H * N


def _weights(dtype, cuda):
    g = torch.Generator().manual_seed(11)

    def w(*shape, s):
        return (torch.randn(shape, generator=g) * s).to(dtype).to(cuda)

    layers = [dict(q=w(C, C, s=C ** -0.5 * N ** -0.5), k=w(C, C, s=C ** -0.5), v=w(C, C, s=C ** -0.5), gate=w(C, C, s=C ** -0.5),
                   pre_gamma=1 + w(C, s=0.1), pre_beta=w(C, s=0.1), post_gamma=1 + w(C, s=0.1), post_beta=w(C, s=0.1),
                   scale=w(C, s=0.3)) for _ in range(LAYERS + 1)]
    return layers, w(V, C, s=1.0), w(C, V, s=0.5 * C ** -0.5)


LOG_DECAY = [-0.5, -0.2, -0.05, -0.01]


class Kernels:
    def __init__(self, pkg, cuda):
        self.pkg, self.decay = pkg, torch.tensor(LOG_DECAY, device=cuda)

    def between(self, x, h, gate, w, after):
        kw = {} if h is None else dict(block_output=h, gate=gate, residual_scale=w["scale"], post_gamma=w["post_gamma"], post_beta=w["post_beta"])
        out = self.pkg.residual_norm(self.pkg.ResidualNormForwardInputs(x, **kw, pre_gamma=after["pre_gamma"], pre_beta=after["pre_beta"], epsilon=EPS))
        return (x if h is None else out.next_residual), out.normed

    def attention(self, q, k, v, s0, lens):
        out = self.pkg.linear_attention(self.pkg.LinearAttentionForwardInputs(q, k, v, self.decay, context_lens=lens), s0)
        return out.output, out.next_state

    def select(self, logits, scores, K):
        out = self.pkg.beam_select(logits, scores, K)
        return out.scores, out.parents, out.tokens

    def reorder(self, states, parents):
        return self.pkg.beam_reorder(states, parents)


class Plain:
    def __init__(self, cuda):
        self.decay = torch.tensor(LOG_DECAY, device=cuda, dtype=torch.float64)

    def between(self, x, h, gate, w, after):
        kw = {} if h is None else dict(block_output=h, gate=gate, residual_scale=w["scale"], post_gamma=w["post_gamma"], post_beta=w["post_beta"])
        new, z = ref.between(x, **kw, pre_gamma=after["pre_gamma"], pre_beta=after["pre_beta"], kind="layer", eps=EPS)
        return (x if h is None else new), z

    def attention(self, q, k, v, s0, lens):
        return ref.attention(q, k, v, self.decay, s0, lens)

    def select(self, logits, scores, K):
        best, parents, tokens = ref.beam_select(logits, scores, K)
        c = torch.sort(ref.beam_candidates(logits, scores), dim=1, descending=True).values
        self.gap = (c[:, :K] - c[:, 1:K + 1]).min()
        return best, parents, tokens

    def reorder(self, states, parents):
        B, K = parents.shape
        rows = (torch.arange(B, device=parents.device)[:, None] * K + parents).flatten()
        return [s[rows] for s in states]


def _model(ops, weights, tokens, states, lens):
    layers, embedding, head = weights
    x = embedding[tokens]
    B, T, _ = x.shape
    h = gate = None
    new = []
    for i in range(LAYERS):
        x, z = ops.between(x, h, gate, layers[i - 1], layers[i])
        w = layers[i]
        q, k, v = ((z @ w[n]).view(B, T, H, N) for n in "qkv")
        y, s = ops.attention(q, k, v, None if states is None else states[i], lens)
        new.append(s)
        h, gate = y.reshape(B, T, C), torch.sigmoid(z @ w["gate"])
    _, z = ops.between(x, h, gate, layers[LAYERS - 1], layers[LAYERS])
    last = torch.full((B,), T, device=x.device) if lens is None else lens.long()
    return z[torch.arange(B, device=x.device), last - 1] @ head, new


def _decode(ops, weights, prompts, lens, steps, force=None):
    """``force``: the choices to follow (so that two runs see the same tokens)."""
    B = prompts.shape[0]
    logits, states = _model(ops, weights, prompts, None, lens)
    scores, parents, tokens = ops.select(logits[:, None], torch.zeros(B, 1, device=prompts.device), BEAMS)
    rows = torch.arange(B, device=prompts.device).repeat_interleave(BEAMS)
    states = [s[rows].contiguous() for s in states]
    trace = [(scores, parents, tokens, logits)]
    for step in range(steps):
        follow = trace[-1] if force is None else force[step]
        if step > 0:
            states = ops.reorder(states, follow[1])
        logits, states = _model(ops, weights, follow[2].reshape(-1, 1).long(), states, None)
        scores, parents, tokens = ops.select(logits.view(B, BEAMS, V), follow[0].to(scores.dtype), BEAMS)
        trace.append((scores, parents, tokens, logits))
    return trace, states


@pytest.mark.parametrize("dtype,near", [(torch.float32, 1e-4), (torch.bfloat16, 0.15)])
def test_prompts_then_beams(pkg, cuda, dtype, near):
    weights = _weights(dtype, cuda)
    g = torch.Generator().manual_seed(5)
    prompts = torch.randint(0, V, (2, 150), generator=g).to(cuda)
    lens = torch.tensor([150, 61], dtype=torch.int32, device=cuda)
    wide = ([{n: t.double() for n, t in w.items()} for w in weights[0]], weights[1].double(), weights[2].double())
    want, want_states = _decode(Plain(cuda), wide, prompts, lens, 6)
    got, states = _decode(Kernels(pkg, cuda), weights, prompts, lens, 6, force=[(s.float(), p.int(), t, None) for s, p, t, _ in want])
    assert pkg.read_device_status(0) == 0
    for (s, p, t, logits), (ws, wp, wt, wl) in zip(got, want):
        # logits of a two-layer model in the tensors' type: its half step through some ten roundings, on values of up to 3
        assert float((logits.double() - wl).abs().max()) <= near
        # each choice is one of the definition's on these very logits
        assert s.shape == ws.shape
    for a, b in zip(states, want_states):
        assert float((a.double() - b).norm() / b.norm()) <= near


def test_choices_follow_from_the_logits(pkg, cuda):
    """Unforced in fp32: every step's choice equals the 64-bit selection on the kernels' own logits and scores."""
    weights = _weights(torch.float32, cuda)
    prompts = torch.randint(0, V, (3, 40), generator=torch.Generator().manual_seed(6)).to(cuda)
    trace, _ = _decode(Kernels(pkg, cuda), weights, prompts, None, 8)
    before = torch.zeros(3, 1, device=cuda)
    for scores, parents, tokens, logits in trace:
        best, wp, wt = ref.beam_select(logits.view(3, before.shape[1], V), before, BEAMS)
        assert torch.equal(parents.long(), wp) and torch.equal(tokens.long(), wt)
        assert float((scores.double() - best).abs().max()) <= 1e-5
        before = scores
