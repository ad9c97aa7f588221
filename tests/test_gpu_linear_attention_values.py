"""Linear attention on values at the edges: decays above one, long memories, infinities, and how many bits of a state are kept.

Bounds are those of ``block_reference``, or are derived at the test."""
import pytest
import torch

import block_reference as ref
from test_gpu_linear_attention import BF16, F32, _abs, _call, _close, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,lens", [(100, None), (300, [100, 57]), (3000, [100, 0])])
def test_states_that_double_every_token(pkg, cuda, T, lens, dtype):
    """exp(0.7 x 100) is a number, exp(0.7 x 128) is not: powers behind a sequence's end are part of nothing, in either direction, in
    one piece or in segments."""
    B = 1 if lens is None else len(lens)
    x, dy, ds = _inputs(cuda, B, T, 2, 64, dtype, seed=T, lens=lens)
    x["log_decay"] = torch.tensor([0.7, 0.35], device=cuda)
    out = _call(pkg, x)
    inputs = pkg.LinearAttentionForwardInputs(x["q"], x["k"], x["v"], x["log_decay"], context_lens=x["lens"])
    grads, ds0 = pkg.linear_attention_backward(inputs, dy, ds, initial_state=x["s0"])
    live = T if lens is None else max(lens)   # (the 64-bit form takes powers of every place)
    y = {n: t[:, :live] if n in ("q", "k", "v") else t for n, t in x.items()}
    inside = torch.arange(live, device=cuda) < (torch.full((B,), T, device=cuda) if lens is None else x["lens"])[:, None]
    dy0 = torch.where(inside[:, :, None, None], dy[:, :live], torch.zeros_like(dy[:, :live]))
    wants = [*ref.attention(**y), *ref.attention_grads(**y, dy=dy0, ds=ds)]
    mags = [*ref.attention(**_abs(y)), *ref.attention_grads(**_abs(y), dy=dy0.abs(), ds=ds.abs())]
    for name, got, w, m in zip(("output", "state", "query", "key", "value", "state gradient"), (out.output, out.next_state, *grads, ds0), wants, mags):
        if got.dim() == 4 and got.shape[1] == T and name not in ("state", "state gradient"):
            assert bool((got[:, live:] == 0).all()), name
            got = got[:, :live]
        _close(got, w, m, live, 64, dtype, name)


@pytest.mark.parametrize("dtype,pieces,scalings", [(BF16, "one", 256), (BF16, "segments", 18 + 15), (F32, "one", 2048), (F32, "segments", 148 + 14)])
def test_a_long_memory_does_not_drift(pkg, cuda, dtype, pieces, scalings):
    """Without values the state is S0 d^T.  Each of the chunks, blocks or segments that it is scaled over rounds an entry, by half a step at
    most and this way or that, so that a head's norm is off by the root of their number times a half step; the powers by which it is scaled
    are off together by a step or two, however many they are."""
    T, H = 32768, 8
    x = _inputs(cuda, 1, T, H, 64, dtype, seed=4)[0]
    x["v"].zero_()
    x["log_decay"] = -1.3e-5 * torch.arange(1, H + 1, device=cuda, dtype=F32)
    workspace = torch.empty(0, dtype=torch.uint8, device=cuda) if pieces == "one" else None
    got = _call(pkg, x, workspace=workspace).next_state.double()
    want = x["s0"].double() * torch.exp(x["log_decay"].double() * T)[:, None, None]
    off = ((got - want).flatten(2).norm(dim=2) / want.flatten(2).norm(dim=2)).flatten() / ref.U
    assert bool((off <= 2 + scalings ** 0.5).all()), off.tolist()


@pytest.mark.parametrize("dtype,T", [(BF16, 148 * 16 * 128 - 77), (F32, 148 * 8 * 16 * 2 - 5)])
def test_every_entry_that_is_not_finite_is_found_in_segments(pkg, cuda, dtype, T):
    """One column of the values in each of 64 chunks in a row, so that a column's later tokens and its row of the state hang on
    a single entry of one segment, with entries of other columns in the chunks around it."""
    step = 128 if dtype == BF16 else 16
    x = _inputs(cuda, 1, T, 1, 64, dtype, seed=8)[0]
    x["log_decay"] = torch.tensor([-0.01], device=cuda)
    first = torch.tensor([T // 3 // step * step + step * c + 11 * c % step for c in range(64)], device=cuda)
    for c, t in enumerate(first.tolist()):
        x["v"][0, t, 0, (29 * c) % 64] = (float("inf"), float("-inf"), float("nan"))[c % 3]
    got = _call(pkg, x)
    assert pkg.read_device_status(0) == 0
    of_column = torch.empty_like(first)
    of_column[(29 * torch.arange(64, device=cuda)) % 64] = first
    reached = torch.arange(T, device=cuda)[:, None] >= of_column
    assert torch.equal(torch.isfinite(got.output[0, :, 0].float()), ~reached)
    assert not bool(torch.isfinite(got.next_state).any())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T", [1, 16, 17, 33, 200, 1500])
def test_infinite_states_stay_infinite(pkg, cuda, T, dtype):
    """One entry of a state that is infinite: it stays, it makes one row of the outputs and one of the queries' gradient infinite, with
    the sign that the formula gives them, and nothing else is touched."""
    x, dy, ds = _inputs(cuda, 2, T, 2, 64, dtype, seed=T)
    x["log_decay"] = torch.tensor([-0.01, -0.002], device=cuda)

    def call():
        inputs = pkg.LinearAttentionForwardInputs(x["q"], x["k"], x["v"], x["log_decay"])
        out = _call(pkg, x)
        (dq, dk, dv), ds0 = pkg.linear_attention_backward(inputs, dy, ds, initial_state=x["s0"])
        return out.output.clone(), out.next_state.clone(), dq, dk, dv, ds0

    want = call()
    inf = float("inf")
    for row, column, entry in ((5, 9, inf), (7, 3, -inf)):
        x["s0"][0, 1, row, column] = entry
        want[1][0, 1, row, column] = entry
        want[0][0, :, 1, row] = entry * x["q"][0, :, 1, column].float().sign()
        want[2][0, :, 1, column] = entry * dy[0, :, 1, row].float().sign()
    for name, a, b in zip(("output", "state", "query", "key", "value", "state gradient"), call(), want):
        assert torch.equal(a, b), name


@pytest.mark.parametrize("T", [60, 200])
def test_states_beyond_the_largest_bf16_number(pkg, cuda, T):
    """fp32 goes on for half a step of bf16 behind bf16's largest number."""
    x = _inputs(cuda, 1, T, 2, 64, BF16)[0]
    x["s0"][0, 1, 5, 9], x["s0"][0, 1, 7, 3] = 3.4e38, -3.4e38
    x["log_decay"] = torch.tensor([-0.01, -0.002], device=cuda)
    out = _call(pkg, x)
    y, s = ref.attention(**x)
    my, ms = ref.attention(**_abs(x))
    _close(out.output, y, my, T, 64, BF16, "output")
    _close(out.next_state, s, ms, T, 64, BF16, "state")
