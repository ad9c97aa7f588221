"""Beam selection where most of the vocabulary is masked, as constrained decoding leaves it, in rows that a CTA goes through in many pieces."""
import pytest
import torch

from test_gpu_beam_search import BF16, F32, _check
from test_gpu_beam_search import _random as _unrounded

pytestmark = pytest.mark.gpu

V = 65536


def _random(cuda, B, I, dtype, seed):
    """A row's logits are the same numbers or far apart."""
    logits, scores = _unrounded(cuda, B, I, V, BF16, seed=seed)
    return logits.to(dtype), scores


def _allowed(cuda, B, I, kind):
    """What is left of each row: a run of tokens, tokens all over it, or three."""
    g = torch.Generator().manual_seed(12)
    t = torch.arange(V)
    if kind == "run":
        first = torch.randint(0, V - 6000, (B, I, 1), generator=g)
        allowed = (t >= first) & (t < first + 6000)
    elif kind == "scattered":
        allowed = torch.rand(B, I, V, generator=g) < 0.1
    else:
        allowed = torch.zeros(B, I, V, dtype=torch.bool)
        allowed.scatter_(2, torch.randint(0, V // 3, (B, I, 3), generator=g) * 3 + torch.arange(3), True)
    return allowed.to(cuda)


def _time(call):
    """Milliseconds on the device, of four calls in a graph (a busy host counts for nothing)."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(4):
            call()
    times = []
    for _ in range(7):
        ends = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        ends[0].record()
        graph.replay()
        ends[1].record()
        torch.cuda.synchronize()
        times.append(ends[0].elapsed_time(ends[1]))
    return sorted(times)[3]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["run", "scattered"])
@pytest.mark.parametrize("B,I,K", [(64, 8, 8), (2, 4, 4)])
def test_a_vocabulary_masked_with_the_lowest_number(pkg, cuda, B, I, K, kind, dtype):
    logits, scores = _random(cuda, B, I, dtype, seed=7)
    masked = torch.where(_allowed(cuda, B, I, kind), logits, torch.finfo(dtype).min)
    _check(pkg, masked, scores, K)
    if B > 2:   # it is no other work: the slow way, one pass for each that is chosen, takes five times as long and more
        plain, slow = (_time(lambda: pkg.beam_select(x, scores, K)) for x in (logits, masked))
        assert slow < 2 * plain, (plain, slow)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["run", "scattered", "three"])
@pytest.mark.parametrize("B,I,K", [(512, 1, 8), (64, 8, 8), (3, 1, 32), (1, 2, 7)])
def test_a_vocabulary_masked_with_infinity(pkg, cuda, B, I, K, kind, dtype):
    """With less left than is chosen the rest are masked tokens, by their index."""
    logits, scores = _random(cuda, B, I, dtype, seed=7)
    masked = logits.masked_fill(~_allowed(cuda, B, I, kind), -torch.inf)
    _check(pkg, masked, scores, K)
    if B == 512:
        plain, slow = (_time(lambda: pkg.beam_select(x, scores, K)) for x in (logits, masked))
        assert slow < 2 * plain, (plain, slow)


@pytest.mark.parametrize("left", [(0, 1, 2), (1,), (5, 40, 65535), tuple(range(0, 14, 2)), ()])
def test_tokens_that_fill_up_pass_over_those_that_are_left(pkg, cuda, left):
    logits = torch.full((300, 1, V), -torch.inf, device=cuda)
    for j, t in enumerate(left):
        logits[:, 0, t] = 1.0 - 0.25 * (j * 3 % 7)
    _check(pkg, logits, torch.zeros(300, 1, device=cuda), 8)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("values", [1, 3])
def test_few_different_logits(pkg, cuda, values, dtype):
    """Thousands of equals above all others: the lowest tokens of them, in about the time that other rows take."""
    logits = torch.randint(0, values, (512, 1, V), generator=torch.Generator().manual_seed(5)).to(dtype).to(cuda)
    scores = torch.zeros(512, 1, device=cuda)
    _check(pkg, logits, scores, 8)
    other = _random(cuda, 512, 1, dtype, seed=7)[0]
    plain, slow = (_time(lambda: pkg.beam_select(x, scores, 8)) for x in (other, logits))
    assert slow < 2 * plain, (plain, slow)
