"""Beam search's selection and the reordering of states against their 64-bit form.

Parents and tokens are equal to the definition's; the inputs' next two scores are far enough apart for that (checked).  A score is
off by half a step of fp32 and by the logarithm of a sum of V exponentials in fp32, each within two steps, added by 256 threads or
more in trees."""
import pytest
import torch

import block_reference as ref

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _check(pkg, logits, scores, K, finished=None, pad_token=0):
    out = pkg.beam_select(logits, scores, K, finished=finished, pad_token=pad_token)
    torch.cuda.synchronize()
    assert pkg.read_device_status(0) == 0
    c = ref.beam_candidates(logits, scores, finished, pad_token)
    best, where = torch.sort(c, dim=1, descending=True, stable=True)
    V = logits.shape[-1]
    lse = (V / 256 + 24) * ref.U
    # what decides: neighbours in the order are the same number or further apart than the arithmetic is off
    finite = torch.where(best[:, :K + 1] == -torch.inf, torch.full_like(best[:, :K + 1], -1e30), best[:, :K + 1])
    gaps = finite[:, :-1] - finite[:, 1:]
    assert bool(((gaps == 0) | (gaps > 2 * lse)).all()), "inputs too close for the test"
    assert torch.equal(out.parents.long(), where[:, :K] // V), "parents"
    assert torch.equal(out.tokens.long(), where[:, :K] % V), "tokens"
    want = best[:, :K]
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(out.scores), fine)
    off = (out.scores.double() - want).abs()[fine]
    assert bool((off <= ref.U * want[fine].abs() + lse).all()), float(off.max())
    return out


def _random(cuda, B, I, V, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + V)
    logits = (torch.randn(B, I, V, generator=g) * 3).to(dtype).to(cuda)
    scores = (torch.randn(B, I, generator=g) * 2 - 20).to(cuda)
    return logits, scores


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,I,V,K", [(1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 2, 6), (3, 4, 100, 4), (1, 4, 1000, 8), (2, 1, 4097, 4), (5, 8, 8191, 8),
                                     (1, 32, 2000, 32), (2, 4, 65529, 4), (1, 5, 65536, 5), (3, 2, 33, 32), (40, 4, 8192, 4)])
def test_select(pkg, cuda, B, I, V, K, dtype):
    _check(pkg, *_random(cuda, B, I, V, dtype, seed=K), K)


@pytest.mark.parametrize("V", [7, 300, 8200])
def test_equal_candidates_go_by_index(pkg, cuda, V):
    """All logits equal; few values; two equal beams: the lowest beam, then the lowest token."""
    scores = torch.zeros(2, 3, device=cuda)
    _check(pkg, torch.zeros(2, 3, V, device=cuda), scores, 6)
    g = torch.Generator().manual_seed(V)
    few = torch.randint(0, 3, (2, 1, V), generator=g).float().to(cuda)
    _check(pkg, few.expand(2, 3, V).contiguous(), scores, 9)
    _check(pkg, few.expand(2, 3, V).contiguous().bfloat16(), scores, 9)


def test_first_step_of_a_search(pkg, cuda):
    """One beam alive, its copies at -inf: all come from it, and -inf fills up what is missing."""
    logits, _ = _random(cuda, 2, 4, 50, F32)
    logits = logits[:, :1].expand(2, 4, 50).contiguous()
    scores = torch.tensor([[0.0] + [float("-inf")] * 3] * 2, device=cuda)
    out = _check(pkg, logits, scores, 4)
    assert bool((out.parents == 0).all())
    logits[:, :, 3:] = float("-inf")
    _check(pkg, logits, scores, 8)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_masked_and_broken_logits(pkg, cuda, dtype):
    logits, scores = _random(cuda, 3, 4, 600, dtype)
    logits[0, 0] = float("-inf")                                   # a row without a token
    logits[0, 1, :590] = float("-inf")
    logits[1, 2, 5] = float("nan")
    logits[1, 3] = float("nan")
    logits[2, 0, 77] = float("inf")
    logits[2, 1] = torch.finfo(dtype).min                          # masked by the type's lowest value throughout
    logits[2, 1, 9] = 1.0
    _check(pkg, logits, scores, 8)
    _check(pkg, torch.full((1, 2, 40), float("-inf"), dtype=dtype, device=cuda), scores[:1, :2].contiguous(), 5)


def test_broken_scores(pkg, cuda):
    logits, scores = _random(cuda, 2, 3, 64, F32)
    scores[0, 1] = float("nan")
    scores[1] = float("-inf")
    _check(pkg, logits, scores, 5)


@pytest.mark.parametrize("pad", [0, 17, 63])
def test_finished_beams(pkg, cuda, pad):
    logits, scores = _random(cuda, 3, 4, 64, BF16)
    scores[0, 2] = -19.0
    finished = torch.tensor([[0, 0, 1, 0], [1, 1, 1, 1], [0, 5, 0, 0]], dtype=torch.int32, device=cuda)
    logits[0, 2] = float("nan")                                    # not looked at
    _check(pkg, logits, scores, 4, finished, pad)
    _check(pkg, logits, scores, 32, finished, pad)


def test_other_stream_and_graph(pkg, cuda):
    logits, scores = _random(cuda, 2, 4, 9000, F32, seed=1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a = pkg.beam_select(logits, scores, 4)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b = pkg.beam_select(logits, scores, 4)
    new = _random(cuda, 2, 4, 9000, F32, seed=2)
    logits.copy_(new[0])
    scores.copy_(new[1])
    graph.replay()
    want = _check(pkg, logits, scores, 4)
    torch.cuda.synchronize()
    assert torch.equal(b.tokens, want.tokens) and torch.equal(b.scores, want.scores) and torch.equal(b.parents, want.parents)
    assert not torch.equal(a.tokens, want.tokens)


# ---- reordering -----------------------------------------------------------------------------------------------------------------


def _states(cuda, rows, seed=0):
    g = torch.Generator().manual_seed(seed)
    shapes = [((2, 64, 64), F32), ((64,), BF16), ((3,), F32), ((5,), BF16), ((1,), BF16), ((7, 2), torch.int64), ((), torch.int32), ((0, 4), F32)]
    return [(torch.randn(rows, *s, generator=g) * 100).to(t).to(cuda) for s, t in shapes]


@pytest.mark.parametrize("B,I,K", [(1, 1, 1), (2, 4, 4), (1, 1, 4), (3, 4, 2), (2, 5, 5), (1, 16, 16), (2, 32, 32), (1, 3, 32)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_reorder(pkg, cuda, B, I, K, dtype):
    states = _states(cuda, B * I, seed=B + I)
    g = torch.Generator().manual_seed(K)
    parents = torch.randint(0, I, (B, K), generator=g, dtype=dtype).to(cuda)
    rows = (torch.arange(B, device=cuda)[:, None] * I + parents).flatten()
    want = [t[rows] for t in states]
    out = [torch.full((B * K, *t.shape[1:]), 9, dtype=t.dtype, device=cuda) for t in states]
    kept = [t.clone() for t in states]
    assert pkg.beam_reorder(states, parents, out=out)[0] is out[0]
    assert all(torch.equal(a, b) for a, b in zip(out, want)) and all(torch.equal(a, b) for a, b in zip(states, kept))
    if I == K:
        pkg.beam_reorder(states, parents)
        assert all(torch.equal(a, b) for a, b in zip(states, want))
    assert pkg.read_device_status(0) == 0


def test_reorder_cycles_in_place(pkg, cuda):
    """A rotation: every row is read before any is written."""
    states = _states(cuda, 2 * 8)
    parents = torch.stack([torch.arange(8).roll(1), torch.arange(8).flip(0)]).int().to(cuda)
    want = [torch.cat([t[:8].roll(1, 0), t[8:].flip(0)]) for t in states]
    pkg.beam_reorder(states, parents)
    assert all(torch.equal(a, b) for a, b in zip(states, want))


def test_reorder_many_tensors(pkg, cuda):
    g = torch.Generator().manual_seed(0)
    states = [torch.randn(6, 33, generator=g).to(cuda) for _ in range(101)]
    parents = torch.tensor([[2, 0, 0], [1, 1, 2]], dtype=torch.int32, device=cuda)
    want = [t[torch.tensor([2, 0, 0, 4, 4, 5], device=cuda)] for t in states]
    pkg.beam_reorder(states, parents)
    assert all(torch.equal(a, b) for a, b in zip(states, want))
    assert pkg.beam_reorder([], parents) == []


def test_bad_parents_leave_their_rows(pkg, cuda):
    """A parent outside the beams (the kernel checks it before it reads) is reported and its row stays as it was."""
    states = _states(cuda, 2 * 3)
    kept = [t.clone() for t in states]
    parents = torch.tensor([[1, -1, 0], [3, 2, 1]], dtype=torch.int32, device=cuda)
    pkg.beam_reorder(states, parents)
    torch.cuda.synchronize()
    assert pkg.read_device_status(0) == 13
    rows = torch.tensor([1, 1, 0, 3, 5, 4], device=cuda)
    assert all(torch.equal(a, b[rows]) for a, b in zip(states, kept))
    assert pkg.read_device_status(0) == 0


def test_reorder_captured(pkg, cuda):
    states = _states(cuda, 4)
    out = [torch.zeros_like(t) for t in states]
    parents = torch.tensor([[0, 1, 2, 3]], dtype=torch.int32, device=cuda)
    pkg.beam_reorder(states, parents, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.beam_reorder(states, parents, out=out)
    parents.copy_(torch.tensor([[3, 3, 0, 1]], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b[parents[0].long()]) for a, b in zip(out, states))


@pytest.mark.parametrize("order", ["rising", "falling", "late", "plateau"])
def test_rows_in_an_order(pkg, cuda, order):
    """Many rows, so that a CTA goes over all of one: every logit larger than those before it; the best at the end; few above -inf in
    front of many; a flood of equal ones."""
    B, I, V = 200, 4, 40000
    x = torch.arange(V, dtype=F32) / 64
    if order == "falling":
        x = x.flip(0)
    elif order == "late":
        x = torch.cat([torch.full((8180,), float("-inf")), torch.tensor([9.0, 3.0, 11.0]), torch.full((V - 8183 - 9000,), float("-inf")), x[:9000] / 16])
    elif order == "plateau":
        x = torch.where(x > 300, torch.full_like(x, 300.0), x)
    assert x.numel() == V
    logits = x.expand(B, I, V).contiguous().to(cuda)
    scores = -torch.arange(I, dtype=F32).expand(B, I).contiguous().to(cuda) / 7
    for K in (1, 4, 32):
        _check(pkg, logits, scores, K)


@pytest.mark.parametrize("I,K", [(32, 32), (32, 1), (8, 32), (20, 7)])
@pytest.mark.parametrize("equal", [False, True])
def test_rows_that_many_share(pkg, cuda, I, K, equal):
    """Few rows, each gone over by many: hundreds of lists to choose from, and all of them alike."""
    logits, scores = _random(cuda, 1, I, 65529, F32, seed=9)
    if equal:
        logits, scores = torch.zeros_like(logits), torch.zeros_like(scores)
    _check(pkg, logits, scores, K)
