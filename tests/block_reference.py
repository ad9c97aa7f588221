"""Plain 64-bit forms of linear attention with a decay per head, the norms around a block and beam search, and bounds on what
fp32 arithmetic can be off by, for the tests of those operators."""
import torch

U = 2.0 ** -24                                                       # half a step of fp32
HALF_STEP = {torch.float32: U, torch.bfloat16: 2.0 ** -8}            # torch.finfo(t).eps / 2


def attention(q, k, v, log_decay, s0=None, lens=None):
    """``(y, state)`` in 64 bits, every pair of tokens at once; differentiable."""
    q, k, v, log_decay = q.double(), k.double(), v.double(), log_decay.double()
    B, T, H, N = q.shape
    pos = torch.arange(T, device=q.device)
    lens = torch.full((B,), T, device=q.device) if lens is None else lens.clamp(0, T).long()
    live = (pos < lens[:, None])[:, :, None, None]
    zero = torch.zeros((), dtype=torch.float64, device=q.device)
    q, k, v = (torch.where(live, t, zero) for t in (q, k, v))
    gap = pos[:, None] - pos[None, :]
    decay = torch.where(gap >= 0, torch.exp(log_decay[:, None, None] * gap.clamp_min(0)), zero)     # H T T
    y = torch.einsum("bhij,bjhn->bihn", torch.einsum("bihn,bjhn->bhij", q, k) * decay, v)
    left = torch.where(live[..., 0], torch.exp(log_decay * (lens[:, None] - 1 - pos).clamp_min(0)[..., None]), zero)   # B T H
    state = torch.einsum("bthi,bthj,bth->bhij", v, k, left)
    if s0 is not None:
        s0 = s0.double()
        y = y + torch.einsum("bhij,bthj,th->bthi", s0, q, torch.exp((pos[:, None] + 1) * log_decay))
        state = state + s0 * torch.exp(lens[:, None] * log_decay)[:, :, None, None]
    return torch.where(live, y, zero), state


def attention_grads(q, k, v, log_decay, dy, ds, s0=None, lens=None):
    leaves = [t.detach().double().requires_grad_() for t in (q, k, v)]
    if s0 is not None:
        leaves.append(s0.detach().double().requires_grad_())
    y, s = attention(*leaves[:3], log_decay, leaves[3] if s0 is not None else None, lens)
    total = (y * dy.double()).sum()
    if ds is not None:
        total = total + (s * ds.double()).sum()
    return torch.autograd.grad(total, leaves)


def attention_bound(T, N, magnitude, dtype):
    """What a result may be off by before it is rounded itself.  ``magnitude``: the same sum over absolute values.  fp32 sums: a
    term passes at most T + N additions, T products with a decay that is itself off by two steps, and a decay over a long
    distance has an exponent of at most 88 in fp32.  bf16: scores inside a chunk are rounded to bf16 once."""
    return ((4 * T + N + 96) * U + (HALF_STEP[dtype] if dtype == torch.bfloat16 else 0.0)) * magnitude


def norm(x, gamma, beta, kind, eps):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    y = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * gamma
    return y if beta is None else y + beta


def between(residual, block_output=None, gate=None, residual_scale=None, post_gamma=None, post_beta=None, pre_gamma=None, pre_beta=None, *,
            kind, eps):
    """``(next_residual or None, normed or None)`` of tensors in 64 bits."""
    x = residual
    if block_output is not None:
        u = block_output if post_gamma is None else norm(block_output, post_gamma, post_beta, kind, eps)
        u = u if gate is None else gate * u
        x = x + (u if residual_scale is None else residual_scale * u)
    return (x if block_output is not None else None), (None if pre_gamma is None else norm(x, pre_gamma, pre_beta, kind, eps))


def beam_candidates(logits, scores, finished=None, pad_token=0):
    """Every candidate's score in 64 bits, ``[B, I * V]``."""
    z = logits.double()
    z = torch.where(torch.isnan(z), torch.full_like(z, -torch.inf), z).clamp_max(torch.finfo(torch.float32).max)
    top = z.amax(-1, keepdim=True)
    top = torch.where(top == -torch.inf, torch.zeros_like(top), top)
    z = z - top
    lp = z - torch.log(torch.exp(z).sum(-1, keepdim=True))
    lp = torch.where(z == -torch.inf, z, lp)
    s = scores.double()
    s = torch.where(torch.isnan(s), torch.full_like(s, -torch.inf), s).clamp_max(torch.finfo(torch.float32).max)
    c = s[..., None] + lp
    if finished is not None:
        only = torch.full_like(c, -torch.inf)
        only[..., pad_token] = s
        c = torch.where((finished != 0)[..., None], only, c)
    return c.flatten(1)


def beam_select(logits, scores, K, finished=None, pad_token=0):
    c = beam_candidates(logits, scores, finished, pad_token)
    best, where = torch.sort(c, dim=1, descending=True, stable=True)
    V = logits.shape[-1]
    return best[:, :K], where[:, :K] // V, where[:, :K] % V
