"""The operators around a recurrent block with one decay per head, over the sizes they are called with.

Linear attention with a decay for each head (one token, prompts, a training step), the norms before and after a block
fused with its gate and residual scale (forward, and a training step), and beam search over the vocabulary with the
reordering of the recurrent states.  Widths are those of the benchmark configurations: head size 64; 12, 16, 32, 40 and 64
heads; a vocabulary of 65 536.

``run`` computes the plain form in 32-bit torch operations, or, where ``own`` is set, calls the package.
"""
from __future__ import annotations

import math

import torch

own = False

N = 64
EPS = 1e-5
HEADS = (12, 16, 32, 40, 64)
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _package():
    from __graft_entry__ import load_package
    return load_package()


def listed():
    return [
        # The next token of one chat, one layer of the 32-head model: the latency of a call.
        dict(name="attention_step_one", op="attention", B=1, T=1, H=32, dtype="bf16", ragged=False),
        # A loaded server: one layer-step of 512 sequences of 40 heads, 335 MB of state in and out.
        dict(name="attention_step_batch", op="attention", B=512, T=1, H=40, dtype="bf16", ragged=False),
        # A chat prompt of odd length behind a carried state.
        dict(name="attention_prompt", op="attention", B=1, T=333, H=32, dtype="bf16", ragged=False),
        # A padded batch of prompts of different lengths.
        dict(name="attention_prompts", op="attention", B=8, T=4096, H=32, dtype="bf16", ragged=True),
        # One long document, few heads: work has to be found along the sequence.
        dict(name="attention_document", op="attention", B=1, T=32768, H=12, dtype="bf16", ragged=False),
        # fp32 tensors, the element type of the reference's own tests.
        dict(name="attention_f32", op="attention", B=2, T=1000, H=12, dtype="f32", ragged=False),
        # A training step of the layer: forward, then the gradients of the sequence and of the state.
        dict(name="attention_train", op="attention_train", B=4, T=2048, H=32, dtype="bf16"),
        # What stands between two blocks in a decode step of 16 sequences.
        dict(name="norm_step", op="norm", rows=16, C=2048, kind="layer", dtype="bf16"),
        # The same in a training step, odd number of tokens.
        dict(name="norm_train", op="norm_train", rows=4 * 4095, C=2048, kind="layer", dtype="bf16"),
        # One request, four beams: select, then move the states of all twelve layers.
        dict(name="beam_one", op="beam", B=1, beams=4, V=65536, layers=12, H=12, dtype="f32"),
        # Sixteen requests of four beams in a 24-layer model of 2048 channels.
        dict(name="beam_batch", op="beam", B=16, beams=4, V=65536, layers=24, H=32, dtype="bf16"),
        # The selection alone for many wide searches: 512 rows of the vocabulary.
        dict(name="beam_select", op="beam", B=64, beams=8, V=65536, layers=0, H=32, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(("step", "attention", "attention", "attention_train", "norm", "norm_train", "beam", "beam"))
    H = rng.choice(HEADS)
    dtype = rng.choice(("bf16", "bf16", "bf16", "f32"))
    if op == "step":
        return dict(op="attention", B=_log(rng, 1, 512 * 40 // H), T=1, H=H, dtype=dtype, ragged=False)
    if op == "attention":
        if dtype == "f32":
            T = _log(rng, 2, 2048)
            return dict(op=op, B=_log(rng, 1, max(1, min(16, 16384 * 12 // (T * H)))), T=T, H=H, dtype=dtype, ragged=rng.random() < 0.5)
        T = _log(rng, 2, 16384)
        return dict(op=op, B=_log(rng, 1, max(1, min(64, 8 * 4096 * 32 // (T * H)))), T=T, H=H, dtype=dtype, ragged=rng.random() < 0.5)
    if op == "attention_train":
        T = _log(rng, 16, 4096 if dtype == "bf16" else 1024)
        return dict(op=op, B=_log(rng, 1, max(1, min(16, (4 * 2048 * 32 if dtype == "bf16" else 8192 * 12) // (T * H)))), T=T, H=H, dtype=dtype)
    if op in ("norm", "norm_train"):
        C = rng.choice((768, 1024, 2048, 2560, 4096, _log(rng, 64, 4096)))
        return dict(op=op, rows=_log(rng, 1, 16384 * 2048 // C), C=C, kind=rng.choice(("layer", "rms")), dtype=dtype)
    layers, H = rng.choice((0, 2, 12, 24)), rng.choice((12, 16, 32))
    beams = _log(rng, 1, 16)
    B = _log(rng, 1, max(1, min(64, 512 // beams, (56 * 24 * 32 // (layers * H * beams)) if layers else 512)))
    return dict(op="beam", B=B, beams=beams, V=rng.choice((65536, 65529, 32768, 8192)), layers=layers, H=H, dtype=dtype)


def _lens(case):
    """The lengths of a padded batch, in the order before it is shuffled: from half the longest up."""
    B, T = case["B"], case["T"]
    return [T - i * (T // 2) // B for i in range(B)]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(104651 * (seed + 1))
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dtype):
        return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)

    s = dict(case)
    if case["op"] in ("attention", "attention_train"):
        B, T, H = case["B"], case["T"], case["H"]
        # queries come scaled by 1/sqrt(N), as a caller folds the scale into its projection
        s["q"], s["k"], s["v"] = normal(B, T, H, N, scale=N ** -0.5), normal(B, T, H, N), normal(B, T, H, N)
        s["state"] = normal(B, H, N, N, scale=0.5, dtype=torch.float32)
        # memories of 2 to 256 tokens, spread over the heads
        s["log_decay"] = -(2.0 ** -(1.0 + 7.0 * torch.arange(H, device="cuda", dtype=torch.float32) / max(H - 1, 1)))
        s["lens"] = None
        if case.get("ragged"):
            order = torch.randperm(B, generator=g, device="cuda")
            s["lens"] = torch.tensor(_lens(case), device="cuda", dtype=torch.int32)[order]
        if case["op"] == "attention_train":
            s["dy"], s["dstate"] = normal(B, T, H, N), normal(B, H, N, N, scale=0.1, dtype=torch.float32)
    elif case["op"] in ("norm", "norm_train"):
        R, C = case["rows"], case["C"]
        s["x"], s["h"] = normal(1, R, C, scale=2.0), normal(1, R, C, scale=0.7)
        s["gate"] = torch.sigmoid(normal(1, R, C, dtype=torch.float32)).to(dtype)
        s["scale"], s["post_gamma"], s["pre_gamma"] = normal(C, scale=0.3), 1 + normal(C, scale=0.1), 1 + normal(C, scale=0.1)
        s["post_beta"] = s["pre_beta"] = None
        if case["kind"] == "layer":
            s["post_beta"], s["pre_beta"] = normal(C, scale=0.1), normal(C, scale=0.1)
        if case["op"] == "norm_train":
            s["dx"], s["dz"] = normal(1, R, C, scale=0.5), normal(1, R, C)
    else:
        B, beams = case["B"], case["beams"]
        s["logits"] = normal(B, beams, case["V"], scale=3.0)
        s["scores"] = -30.0 + torch.sort(normal(B, beams, scale=2.0, dtype=torch.float32), dim=1, descending=True).values
        # per layer a state and two shifted tokens for each beam, and the buffers that the next step reads
        s["states"] = [t for _ in range(case["layers"])
                       for t in (normal(B * beams, case["H"], N, N, dtype=torch.float32), normal(B * beams, 2, case["H"] * N, dtype=torch.bfloat16))]
        s["next"] = [torch.empty_like(t) for t in s["states"]]
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------------


def _plain_attention(q, k, v, state, log_decay, lens):
    """Chunks of 128 tokens: products inside a chunk, and one matrix over the chunks that carries their states on."""
    B, T, H, _ = q.shape
    L = min(128, T)
    n = -(-T // L)
    pos = torch.arange(T, device=q.device)
    if lens is not None:
        inside = (pos < lens[:, None])[:, :, None, None]
        q, k, v = torch.where(inside, q, 0.0), torch.where(inside, k, 0.0), torch.where(inside, v, 0.0)

    def chunks(x):
        return torch.nn.functional.pad(x, (0, 0, 0, 0, 0, n * L - T)).view(B, n, L, H, N).permute(0, 3, 1, 2, 4)   # B H n L N

    qc, kc, vc = chunks(q), chunks(k), chunks(v)
    i = torch.arange(L, device=q.device)
    gap = i[:, None] - i[None, :]
    inner = torch.where(gap >= 0, torch.exp(log_decay[:, None, None] * gap.clamp_min(0)), 0.0)
    y = ((qc @ kc.transpose(-1, -2)) * inner[:, None]) @ vc
    added = vc.transpose(-1, -2) @ (kc * torch.exp(log_decay[:, None, None, None] * (L - 1 - i)[:, None]))           # B H n N N
    c = torch.arange(n, device=q.device)
    far = c[:, None] - 1 - c[None, :]
    carry = torch.where(far >= 0, torch.exp(log_decay[:, None, None] * (L * far.clamp_min(0))), 0.0)
    before = (carry @ added.reshape(B, H, n, N * N)).view(B, H, n, N, N)
    before = before + torch.exp(log_decay[:, None] * (L * c))[:, :, None, None] * state[:, :, None]
    y = y + (qc @ before.transpose(-1, -2)) * torch.exp(log_decay[:, None] * (i + 1))[:, None, :, None]
    y = y.permute(0, 2, 3, 1, 4).reshape(B, n * L, H, N)[:, :T]
    end = torch.full((B, 1), T, device=q.device) if lens is None else lens[:, None]
    weight = torch.exp(log_decay * (end - 1 - pos).clamp_min(0)[:, :, None])                                         # B T H
    last = v.permute(0, 2, 3, 1) @ (k * weight[..., None]).permute(0, 2, 1, 3)
    return y, torch.exp(log_decay * end)[:, :, None, None] * state + last


def _plain_norm(x, gamma, beta, kind):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gamma
    return y if beta is None else y + beta


def _plain_between(x, h, gate, scale, post_gamma, post_beta, pre_gamma, pre_beta, kind):
    x = x + scale * (gate * _plain_norm(h, post_gamma, post_beta, kind))
    return x, _plain_norm(x, pre_gamma, pre_beta, kind)


def _plain_select(logits, scores):
    # (64 bits: which of two candidates is larger hangs on their last bits)
    z = logits.double()
    z = z - z.amax(-1, keepdim=True)
    c = scores.double()[..., None] + z - torch.log(torch.exp(z).sum(-1, keepdim=True))
    best, where = torch.sort(c.flatten(1), dim=1, descending=True, stable=True)
    K, V = scores.shape[1], logits.shape[-1]
    best, where = best[:, :K], where[:, :K]
    return best.float(), (where // V).int(), (where % V).int()


def _floats(s, names):
    return [None if s[n] is None else s[n].float() for n in names]


_NORM = ("x", "h", "gate", "scale", "post_gamma", "post_beta", "pre_gamma", "pre_beta")


def run(s):
    op = s["op"]
    if own:
        pkg = _package()
        if op in ("attention", "attention_train"):
            inputs = pkg.LinearAttentionForwardInputs(s["q"], s["k"], s["v"], s["log_decay"], context_lens=s["lens"])
            out = pkg.linear_attention(inputs, s["state"])
            if op == "attention":
                return out.output, out.next_state
            grads, dstate = pkg.linear_attention_backward(inputs, s["dy"], s["dstate"], initial_state=s["state"])
            return out.output, out.next_state, *grads, dstate
        if op in ("norm", "norm_train"):
            inputs = pkg.ResidualNormForwardInputs(
                s["x"], s["h"], gate=s["gate"], residual_scale=s["scale"], post_gamma=s["post_gamma"], post_beta=s["post_beta"],
                pre_gamma=s["pre_gamma"], pre_beta=s["pre_beta"], kind=s["kind"], epsilon=EPS)
            out = pkg.residual_norm(inputs)
            if op == "norm":
                return out.next_residual, out.normed
            return out.next_residual, out.normed, pkg.residual_norm_backward(inputs, s["dx"], s["dz"])
        best = pkg.beam_select(s["logits"], s["scores"], s["beams"])
        if s["states"]:
            pkg.beam_reorder(s["states"], best.parents, out=s["next"])
        return best.scores, best.parents, best.tokens, s["next"]
    if op == "attention":
        y, state = _plain_attention(*_floats(s, ("q", "k", "v", "state", "log_decay")), s["lens"])
        return y.to(s["q"].dtype), state
    if op == "attention_train":
        leaves = [t.detach().requires_grad_() for t in _floats(s, ("q", "k", "v", "state"))]
        y, state = _plain_attention(*leaves, s["log_decay"], None)
        grads = torch.autograd.grad((y, state), leaves, (s["dy"].float(), s["dstate"]))
        t = s["q"].dtype
        return y.detach().to(t), state.detach(), grads[0].to(t), grads[1].to(t), grads[2].to(t), grads[3]
    if op == "norm":
        return tuple(t.to(s["x"].dtype) for t in _plain_between(*_floats(s, _NORM), s["kind"]))
    if op == "norm_train":
        leaves = [None if t is None else t.detach().requires_grad_() for t in _floats(s, _NORM)]
        x, z = _plain_between(*leaves, s["kind"])
        given = [t for t in leaves if t is not None]
        grads = dict(zip([n for n, t in zip(_NORM, leaves) if t is not None],
                         torch.autograd.grad((x, z), given, (s["dx"].float(), s["dz"].float()))))
        t = s["x"].dtype
        return x.detach().to(t), z.detach().to(t), tuple(grads[n].to(t) if n in grads else None for n in _NORM)
    scores, parents, tokens = _plain_select(s["logits"], s["scores"])
    rows = (torch.arange(s["B"], device=parents.device)[:, None] * s["beams"] + parents).flatten()
    return scores, parents, tokens, [t.index_select(0, rows) for t in s["states"]]


# ---- work ----------------------------------------------------------------------------------------------------------------


def work(case):
    op, size = case["op"], DTYPES[case["dtype"]].itemsize
    if op in ("attention", "attention_train"):
        B, T, H = case["B"], case["T"], case["H"]
        tokens = sum(_lens(case)) if case.get("ragged") else B * T
        state = 4 * N * N * B * H
        if op == "attention":     # q, k, v of the tokens there are, y of all; S <- d S + v k^T and S q
            return {"bytes": size * N * H * (3 * tokens + B * T) + 2 * state + 4 * (H + B), "flops": 4 * N * N * tokens * H}
        # forward; then q, k, v, dy in and three gradients out; S^T dy, G k, G^T v and the two states again
        return {"bytes": 11 * size * N * H * tokens + 5 * state + 4 * H, "flops": 14 * N * N * tokens * H}
    if op == "norm":
        return {"bytes": size * case["C"] * (5 * case["rows"] + 5), "flops": 18 * case["C"] * case["rows"]}
    if op == "norm_train":
        return {"bytes": size * case["C"] * (13 * case["rows"] + 10), "flops": 60 * case["C"] * case["rows"]}
    rows = case["B"] * case["beams"]
    states = rows * case["layers"] * case["H"] * (4 * N * N + 4 * N)
    return {"bytes": rows * (size * case["V"] + 16) + 2 * states, "flops": 4 * rows * case["V"]}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------


def _exact_attention(s, train):
    """Token by token."""
    q, k, v, S = (s[n].double() for n in ("q", "k", "v", "state"))
    B, T, H, _ = q.shape
    d = torch.exp(s["log_decay"].double())[:, None, None]
    ends = [T] * B if s["lens"] is None else s["lens"].tolist()
    y = torch.zeros_like(q)
    dq = torch.zeros_like(q)
    shortest = min(ends)
    live = torch.ones(B, 1, 1, 1, device=q.device, dtype=torch.bool)
    for t in range(max(ends)):
        new = d * S + v[:, t, :, :, None] * k[:, t, :, None, :]
        if t >= shortest:
            live = torch.tensor([t < e for e in ends], device=q.device)[:, None, None, None]
        S = new if t < shortest else torch.where(live, new, S)
        y[:, t] = (S @ q[:, t, :, :, None])[..., 0] if t < shortest else torch.where(live[..., 0], (S @ q[:, t, :, :, None])[..., 0], 0.0)
        if train:
            dq[:, t] = (S.transpose(-1, -2) @ s["dy"][:, t].double()[..., None])[..., 0]
    if not train:
        return y, S
    G = s["dstate"].double()
    dk, dv = torch.zeros_like(q), torch.zeros_like(q)
    for t in reversed(range(T)):
        G = G + s["dy"][:, t].double()[..., None] * q[:, t, :, None, :]
        dv[:, t] = (G @ k[:, t, :, :, None])[..., 0]
        dk[:, t] = (G.transpose(-1, -2) @ v[:, t, :, :, None])[..., 0]
        G = d * G
    return y, S, dq, dk, dv, G


class _ExactNorm:
    def __init__(self, x, gamma, beta, kind):
        self.layer, self.gamma = kind == "layer", gamma
        mean = x.mean(-1, keepdim=True) if self.layer else 0.0
        self.r = ((x - mean).square().mean(-1, keepdim=True) + EPS) ** -0.5
        self.hat = (x - mean) * self.r
        self.y = self.hat * gamma + (0.0 if beta is None else beta)

    def back(self, dy):
        """Gradients of the input, gamma and beta."""
        g = dy * self.gamma
        dx = g - self.hat * (g * self.hat).mean(-1, keepdim=True)
        if self.layer:
            dx = dx - g.mean(-1, keepdim=True)
        return self.r * dx, (dy * self.hat).sum((0, 1)), dy.sum((0, 1)) if self.layer else None


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("attention", "attention_train"):
        return _exact_attention(s, op == "attention_train")
    if op in ("norm", "norm_train"):
        x, h, gate, scale, post_gamma, post_beta, pre_gamma, pre_beta = (None if s[n] is None else s[n].double() for n in _NORM)
        post = _ExactNorm(h, post_gamma, post_beta, case["kind"])
        x1 = x + scale * gate * post.y
        pre = _ExactNorm(x1, pre_gamma, pre_beta, case["kind"])
        if op == "norm":
            return x1, pre.y
        dx, dpre_gamma, dpre_beta = pre.back(s["dz"].double())
        dx = dx + s["dx"].double()
        dh, dpost_gamma, dpost_beta = post.back(dx * scale * gate)
        return x1, pre.y, (dx, dh, dx * scale * post.y, (dx * gate * post.y).sum((0, 1)), dpost_gamma, dpost_beta, dpre_gamma, dpre_beta)
    z = s["logits"].double()
    c = s["scores"].double()[..., None] + z - torch.logsumexp(z, -1, keepdim=True)
    best = torch.topk(c.flatten(1), case["beams"], dim=1).values
    return best, None, None, [None] * len(s["next"])
