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


@pytest.mark.parametrize("T,pieces", [(200, "one"), (1500, "segments")])
def test_a_state_keeps_all_bits_of_its_terms(pkg, cuda, T, pieces):
    """One token has a value, so the state is one product: nothing is added that could hide what its parts leave out.  Its decay is taken as two
    powers at most, with exponents down to -2: each within 4 half steps (expf) and the rounding of its exponent, 2 more; the product with the
    value, the three sums of its parts and the state's own scalings add a half step or (a sum on the tensor cores) two each."""
    H = 32 if pieces == "one" else 4
    x = _inputs(cuda, 5, T, H, 64, BF16, state=False, seed=6)[0]
    x["log_decay"] = -(2.0 / T) * torch.rand(H, generator=torch.Generator().manual_seed(1)).to(cuda)
    at = torch.randint(0, T, (5, H), generator=torch.Generator().manual_seed(2)).to(cuda)
    only = torch.arange(T, device=cuda)[None, :, None] == at[:, None]
    x["v"] = torch.where(only[..., None], x["v"], torch.zeros_like(x["v"]))
    got = _call(pkg, x).next_state.double()
    v, k = (x[n].double()[only.nonzero(as_tuple=True)].view(-1, 64) for n in "vk")
    where = only.nonzero()
    want = torch.empty_like(got)
    power = torch.exp(x["log_decay"].double()[where[:, 2]] * (T - 1 - where[:, 1]))
    want[where[:, 0], where[:, 2]] = power[:, None, None] * v[:, :, None] * k[:, None, :]
    scalings = T // 128 + 1
    off = ((got - want).abs() / want.abs().clamp_min(1e-30)).max() / ref.U
    # (without the last eight bits of a weighted value: up to 64)
    assert float(off) <= 2 * 6 + 1 + 3 * 2 + 3 * scalings, float(off)


def test_a_carried_state_enters_the_outputs_with_sixteen_bits(pkg, cuda):
    """A query of one component and no values: an output is one entry of the state and its decay, rounded to bf16 once, with what the state's
    two bf16 parts (2^-17 of it) and fp32 (16 half steps) leave out before that."""
    T = 100
    x = _inputs(cuda, 2, T, 40, 64, BF16, seed=9)[0]
    x["v"].zero_()
    one = torch.randint(0, 64, (2, T, 40), generator=torch.Generator().manual_seed(3)).to(cuda)
    x["q"] = torch.nn.functional.one_hot(one, 64).bfloat16()
    got = _call(pkg, x).output.double()
    picked = x["s0"].double().transpose(-1, -2)[torch.arange(2, device=cuda)[:, None, None], torch.arange(40, device=cuda), one]   # B T H N
    want = picked * torch.exp(x["log_decay"].double() * (torch.arange(T, device=cuda)[:, None] + 1))[None, ..., None]
    half = torch.exp2(torch.floor(torch.log2(want.abs().clamp_min(1e-300)))) * 2.0 ** -8   # of a step of bf16 there
    # (by the first part alone 2^-9 more)
    assert bool(((got - want).abs() <= half * (1 + 2.0 ** -7) + (2.0 ** -17 + 16 * ref.U) * want.abs()).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N", [32, 128])
def test_padded_batches_of_other_head_sizes_in_segments(pkg, cuda, N, dtype):
    lens = [700, 0, 333]
    x, dy, ds = _inputs(cuda, 3, 700, 2, N, dtype, lens=lens, seed=N)
    for b, e in enumerate(lens):
        for t in (x["q"], x["k"], x["v"], dy):
            t[b, e:] = float("nan")
    assert pkg.linear_attention_workspace_bytes(3, 700, 2, N, dtype) > 0   # (there are segments)
    out = _call(pkg, x)
    inputs = pkg.LinearAttentionForwardInputs(x["q"], x["k"], x["v"], x["log_decay"], context_lens=x["lens"])
    grads, ds0 = pkg.linear_attention_backward(inputs, dy, ds, initial_state=x["s0"])
    dy0 = torch.nan_to_num(dy, nan=0.0)
    wants = [*ref.attention(**x), *ref.attention_grads(**x, dy=dy0, ds=ds)]
    mags = [*ref.attention(**_abs(x)), *ref.attention_grads(**_abs(x), dy=dy0.abs(), ds=ds.abs())]
    for name, got, w, m in zip(("output", "state", "query", "key", "value", "state gradient"), (out.output, out.next_state, *grads, ds0), wants, mags):
        _close(got, w, m, 700, N, dtype, name)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T", [1, 33, 200, 1500])
def test_infinite_gradients_of_the_final_state_stay_infinite(pkg, cuda, T, dtype):
    x, dy, ds = _inputs(cuda, 2, T, 2, 64, dtype, seed=T)
    x["log_decay"] = torch.tensor([-0.01, -0.002], device=cuda)

    def call():
        (dq, dk, dv), ds0 = pkg.linear_attention_backward(pkg.LinearAttentionForwardInputs(x["q"], x["k"], x["v"], x["log_decay"]), dy, ds,
                                                          initial_state=x["s0"])
        return dq, dk, dv, ds0

    want = call()
    inf = float("inf")
    for row, column, entry in ((5, 9, inf), (7, 3, -inf)):
        ds[1, 0, row, column] = entry
        want[3][1, 0, row, column] = entry
        want[2][1, :, 0, row] = entry * x["k"][1, :, 0, column].float().sign()
        want[1][1, :, 0, column] = entry * x["v"][1, :, 0, row].float().sign()
    for name, a, b in zip(("query", "key", "value", "state gradient"), call(), want):
        assert torch.equal(a, b), name


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T", [1, 40, 200, 1500])
def test_what_is_not_finite_reaches_its_own(pkg, cuda, T, dtype):
    """One key, then one query, of a head: columns of the state, outputs from that token on or of that token; everything else as without it."""
    x = _inputs(cuda, 2, T, 2, 64, dtype, seed=T + 1)[0]
    x["log_decay"] = torch.tensor([-0.01, -0.002], device=cuda)
    clean = _call(pkg, x)
    t = T // 2
    for bad in (float("inf"), float("-inf"), float("nan")):
        k = x["k"].clone()
        k[1, t, 0, 11] = bad
        out = _call(pkg, dict(x, k=k))
        reached = torch.zeros_like(out.output, dtype=torch.bool)
        reached[1, t:, 0] = True
        assert torch.equal(torch.isfinite(out.output), ~reached) and torch.equal(out.output[~reached], clean.output[~reached])
        column = torch.zeros_like(out.next_state, dtype=torch.bool)
        column[1, 0, :, 11] = True
        assert torch.equal(torch.isfinite(out.next_state), ~column) and torch.equal(out.next_state[~column], clean.next_state[~column])
        q = x["q"].clone()
        q[1, t, 0, 11] = bad
        out = _call(pkg, dict(x, q=q))
        reached = torch.zeros_like(out.output, dtype=torch.bool)
        reached[1, t, 0] = True
        assert torch.equal(torch.isfinite(out.output), ~reached) and torch.equal(out.output[~reached], clean.output[~reached])
        assert torch.equal(out.next_state, clean.next_state)
