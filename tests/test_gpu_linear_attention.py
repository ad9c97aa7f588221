"""Linear attention with a decay per head against its 64-bit form.

Tolerances (``block_reference.attention_bound``): a result is off by half a step of its type, plus, on the same sum over absolute
values, the roundings of fp32 sums and, for bf16 tensors, one rounding of the scores."""
import pytest
import torch

import block_reference as ref

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _inputs(cuda, B, T, H, N, dtype, seed=0, state=True, lens=None):
    g = torch.Generator().manual_seed(1000 * seed + 7)
    q, k, v, dy = ((torch.randn(B, T, H, N, generator=g) * s).to(dtype).to(cuda) for s in (N ** -0.5, 1.0, 1.0, 1.0))
    s0, ds = ((torch.randn(B, H, N, N, generator=g) * s).to(cuda) for s in (0.5, 0.1))
    log_decay = -(2.0 ** -(1.0 + 7.0 * torch.arange(H, dtype=F32) / max(H - 1, 1))).to(cuda)
    lens = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=cuda)
    return dict(q=q, k=k, v=v, log_decay=log_decay, s0=s0 if state else None, lens=lens), dy, ds


def _call(pkg, x, **kw):
    inputs = pkg.LinearAttentionForwardInputs(x["q"], x["k"], x["v"], x["log_decay"], context_lens=x["lens"])
    return pkg.linear_attention(inputs, x["s0"], **kw)


def _abs(x):
    return {n: t.abs() if n in ("q", "k", "v", "s0") and t is not None else t for n, t in x.items()}


def _close(got, want, magnitude, T, N, dtype, what):
    assert got.dtype in (F32, dtype)
    bound = ref.attention_bound(T, N, magnitude, dtype) + ref.HALF_STEP[got.dtype] * want.abs()
    if got.dtype == F32 and dtype == BF16:   # a state: its sums take no rounded scores
        bound = ref.attention_bound(T, N, magnitude, F32) + ref.U * want.abs()
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"{what}: {int((off > bound).sum())} beyond, worst {float((off / bound.clamp_min(1e-300)).max()):.3g} of the bound"


def _check_forward(pkg, x, dtype):
    out = _call(pkg, x)
    torch.cuda.synchronize()
    assert pkg.read_device_status(0) == 0
    B, T, H, N = x["q"].shape
    y, s = ref.attention(**x)
    my, ms = ref.attention(**_abs(x))
    _close(out.output, y, my, T, N, dtype, "output")
    _close(out.next_state, s, ms, T, N, dtype, "state")
    return out


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N", [32, 64, 128])
@pytest.mark.parametrize("B,T,H", [(1, 1, 1), (2, 1, 3), (3, 2, 2), (2, 5, 2), (1, 16, 2), (2, 17, 3), (1, 127, 1), (2, 128, 2), (1, 129, 3), (2, 300, 2), (1, 1000, 2)])
def test_forward(pkg, cuda, B, T, H, N, dtype):
    _check_forward(pkg, _inputs(cuda, B, T, H, N, dtype, seed=T)[0], dtype)


@pytest.mark.parametrize("T,ragged", [(64, False), (130, True), (300, True), (1100, True)])
def test_more_chains_than_the_device_holds(pkg, cuda, T, ragged):
    """Short sequences: a CTA goes over several chains, some without a token; longer ones: more CTAs than SMs.  Every chain has its own
    decay, state and length."""
    B, H = 60, 9
    lens = [(37 * b) % (T + 1) if ragged else T for b in range(B)]
    x, dy, ds = _inputs(cuda, B, T, H, 64, BF16, seed=T, lens=lens)
    for t in (x["q"], x["k"], x["v"], dy):
        for b, e in enumerate(lens):
            t[b, e:] = float("nan")
    _check_forward(pkg, x, BF16)
    inputs = pkg.LinearAttentionForwardInputs(x["q"], x["k"], x["v"], x["log_decay"], context_lens=x["lens"])
    grads, ds0 = pkg.linear_attention_backward(inputs, dy, ds, initial_state=x["s0"])
    dy0 = torch.nan_to_num(dy, nan=0.0)
    for part in (slice(0, 20), slice(20, 40), slice(40, 60)):   # (the 64-bit form takes every pair of tokens at once)
        y = {n: t if n == "log_decay" else t[part] for n, t in x.items()}
        want = ref.attention_grads(**y, dy=dy0[part], ds=ds[part])
        mag = ref.attention_grads(**_abs(y), dy=dy0[part].abs(), ds=ds[part].abs())
        for name, got, w, m in zip(("query", "key", "value", "state"), (*grads, ds0), want, mag):
            _close(got[part], w, m, T, 64, BF16, name)
    assert pkg.read_device_status(0) == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T", [1, 31, 200])
def test_zero_state_and_no_state_wanted(pkg, cuda, T, dtype):
    x = _inputs(cuda, 2, T, 3, 64, dtype, state=False)[0]
    out = _check_forward(pkg, x, dtype)
    alone = _call(pkg, x, want_state=False)
    assert alone.next_state is None and torch.equal(alone.output, out.output)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,lens", [(1, [0, 1, 1, 0]), (40, [0, 1, 39, 40]), (300, [0, 128, 129, 300]), (1024, [1, 127, 1023, 640])])
def test_padded_batches(pkg, cuda, T, lens, dtype):
    """Lengths from none to all; what stands in the padding (NaN here) reaches nothing."""
    x = _inputs(cuda, 4, T, 2, 64, dtype, lens=lens)[0]
    for n in "qkv":
        for b, e in enumerate(lens):
            x[n][b, e:] = float("nan")
    out = _check_forward(pkg, x, dtype)
    for b, e in enumerate(lens):
        assert bool((out.output[b, e:] == 0).all())
        if e == 0:
            assert torch.equal(out.next_state[b], x["s0"][b])


def test_lengths_outside_the_sequence_count_as_its_ends(pkg, cuda):
    x = _inputs(cuda, 2, 50, 2, 64, BF16, lens=[-3, 1 << 30])[0]
    got = _call(pkg, x)
    want = _call(pkg, dict(x, lens=torch.tensor([0, 50], dtype=torch.int32, device=cuda)))
    assert torch.equal(got.output, want.output) and torch.equal(got.next_state, want.next_state)


@pytest.mark.parametrize("T", [1, 3, 150, 700])
def test_state_in_place_and_carried_on(pkg, cuda, T):
    """A sequence cut in two with its state carried on in place is the sequence in one call."""
    x = _inputs(cuda, 2, 2 * T, 2, 64, BF16, seed=3)[0]
    cut = [dict(x, **{n: x[n][:, i * T:(i + 1) * T].contiguous() for n in "qkv"}) for i in (0, 1)]
    state = x["s0"].clone()
    y = []
    for part in cut:
        out = _call(pkg, dict(part, s0=state), next_state=state)
        assert out.next_state is state
        y.append(out.output)
    want_y, want_s = ref.attention(**x)
    my, ms = ref.attention(**_abs(x))
    _close(torch.cat(y, 1), want_y, my, 2 * T, 64, BF16, "output")
    _close(state, want_s, ms, 2 * T, 64, BF16, "state")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("value", [0.0, -1e-6, -30.0, -1e4, float("-inf"), 0.01])
def test_decays_from_none_to_all(pkg, cuda, value, dtype):
    x = _inputs(cuda, 1, 260, 2, 64, dtype)[0]
    x["log_decay"] = torch.full((2,), value, device=cuda)
    if value == float("-inf"):   # every token stands alone
        out = _call(pkg, x)
        y = (x["q"].double() * x["k"].double()).sum(-1, keepdim=True) * x["v"].double()
        my = (x["q"].double() * x["k"].double()).abs().sum(-1, keepdim=True) * x["v"].double().abs()
        _close(out.output, y, my, 260, 64, dtype, "output")
        s = x["v"][:, -1].double()[..., None] * x["k"][:, -1].double()[..., None, :]
        _close(out.next_state, s, s.abs(), 260, 64, dtype, "state")
    else:
        _check_forward(pkg, x, dtype)


def test_infinities_stay_in_their_sequence_and_head(pkg, cuda):
    x = _inputs(cuda, 2, 200, 2, 64, BF16)[0]
    want = _call(pkg, x)
    bad = dict(x, v=x["v"].clone())
    bad["v"][0, 100, 1] = float("inf")
    got = _call(pkg, bad)
    assert torch.equal(got.output[1], want.output[1]) and torch.equal(got.output[0, :, 0], want.output[0, :, 0])
    assert torch.equal(got.output[0, :100, 1], want.output[0, :100, 1])
    assert not bool(torch.isfinite(got.next_state[0, 1]).any())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,T,H,N,state,lens", [
    (1, 1, 1, 64, True, None), (2, 7, 2, 64, True, None), (2, 128, 2, 64, True, None), (1, 129, 3, 64, False, None),
    (2, 300, 2, 64, True, None), (3, 260, 2, 64, True, [0, 129, 260]), (1, 900, 1, 64, True, None), (2, 65, 2, 32, True, None),
    (1, 70, 2, 128, True, [33])])
def test_backward(pkg, cuda, B, T, H, N, state, lens, dtype):
    x, dy, ds = _inputs(cuda, B, T, H, N, dtype, seed=T, state=state, lens=lens)
    if lens is not None:
        for b, e in enumerate(lens):
            for t in (x["q"], x["k"], x["v"], dy):
                t[b, e:] = float("nan")
    inputs = pkg.LinearAttentionForwardInputs(x["q"], x["k"], x["v"], x["log_decay"], context_lens=x["lens"])
    grads, ds0 = pkg.linear_attention_backward(inputs, dy, ds, initial_state=x["s0"], want_state_grad=state)
    torch.cuda.synchronize()
    live = torch.ones(B, T, 1, 1, dtype=torch.bool, device=cuda)
    if lens is not None:
        live = (torch.arange(T, device=cuda) < x["lens"][:, None])[:, :, None, None]
    dy0 = torch.where(live, dy, torch.zeros_like(dy))
    want = ref.attention_grads(**x, dy=dy0, ds=ds)
    mag = ref.attention_grads(**_abs(x), dy=dy0.abs(), ds=ds.abs())
    for name, got, w, m in zip(("query", "key", "value"), grads, want, mag):
        _close(got, w, m, T, N, dtype, name)
        assert bool((torch.where(live, torch.zeros_like(got), got) == 0).all())
    if state:
        _close(ds0, want[3], mag[3], T, N, dtype, "state")
    else:
        assert ds0 is None


def test_gradients_against_differences(pkg, cuda):
    """The operator is linear in each of query, key, value and state, so a difference quotient has no error but roundings."""
    x, dy, ds = _inputs(cuda, 2, 70, 2, 64, F32, seed=5)
    leaves = {n: x[n].clone().requires_grad_() for n in ("q", "k", "v", "s0")}
    inputs = pkg.LinearAttentionForwardInputs(leaves["q"], leaves["k"], leaves["v"], x["log_decay"])
    y, s = pkg.linear_attention_autograd(leaves["s0"], inputs)
    grads = dict(zip(leaves, torch.autograd.grad((y, s), list(leaves.values()), (dy, ds))))
    g = torch.Generator().manual_seed(1)
    for n in leaves:
        d = torch.randn(x[n].shape, generator=g).to(cuda)
        ends = []
        for sign in (1.0, -1.0):
            out = _call(pkg, dict(x, **{n: x[n] + sign * d}))
            ends.append((out.output.double() * dy).sum() + (out.next_state.double() * ds).sum())
        m = _abs(dict(x, **{n: x[n].abs() + d.abs()}))
        my, ms = ref.attention(**m)
        bound = 4 * ref.attention_bound(70, 64, float((my * dy.abs()).sum() + (ms * ds.abs()).sum()), F32)
        assert abs(float((ends[0] - ends[1]) / 2 - (grads[n].double() * d.double()).sum())) <= bound, n


def test_autograd_without_some_gradients(pkg, cuda):
    x, dy, ds = _inputs(cuda, 1, 40, 2, 64, BF16)
    q = x["q"].clone().requires_grad_()
    y, s = pkg.linear_attention_autograd(x["s0"], pkg.LinearAttentionForwardInputs(q, x["k"], x["v"], x["log_decay"]))
    a, = torch.autograd.grad(y, q, dy, retain_graph=True)
    b, = torch.autograd.grad((y, s), q, (dy, ds))
    assert torch.equal(a, b)   # the final state does not hang on the queries
    y, s = pkg.linear_attention_autograd(None, pkg.LinearAttentionForwardInputs(x["q"], x["k"].requires_grad_(), x["v"], x["log_decay"]))
    g, = torch.autograd.grad(s, x["k"], ds)
    want = ref.attention_grads(x["q"], x["k"], x["v"], x["log_decay"], torch.zeros_like(dy), ds)[1]
    mag = ref.attention_grads(x["q"].abs(), x["k"].abs(), x["v"].abs(), x["log_decay"], torch.zeros_like(dy), ds.abs())[1]
    _close(g, want, mag, 40, 64, BF16, "key")


@pytest.mark.parametrize("T", [1, 200, 1500])
def test_captured_and_replayed_with_new_values(pkg, cuda, T):
    x, dy, ds = _inputs(cuda, 1, T, 3, 64, BF16, seed=1)
    inputs = pkg.LinearAttentionForwardInputs(x["q"], x["k"], x["v"], x["log_decay"])

    def step():
        return _call(pkg, x), pkg.linear_attention_backward(inputs, dy, ds, initial_state=x["s0"])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, (grads, ds0) = step()
    new = _inputs(cuda, 1, T, 3, 64, BF16, seed=2)
    for n in ("q", "k", "v", "s0"):
        x[n].copy_(new[0][n])
    dy.copy_(new[1])
    ds.copy_(new[2])
    graph.replay()
    want, (want_grads, want_ds0) = step()
    torch.cuda.synchronize()
    for a, b in zip((out.output, out.next_state, *grads, ds0), (want.output, want.next_state, *want_grads, want_ds0)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("T", [1, 1500])
def test_two_streams_at_once(pkg, cuda, T):
    xs = [_inputs(cuda, 2, T, 2, 64, BF16, seed=i)[0] for i in range(2)]
    want = [_call(pkg, x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(_call(pkg, xs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert torch.equal(o.output, want[i].output) and torch.equal(o.next_state, want[i].next_state)


def test_smaller_workspaces_are_taken(pkg, cuda):
    """Down to none: fewer parts of a sequence at once, the same sums."""
    B, T, H, N = 1, 4100, 2, 64
    x = _inputs(cuda, B, T, H, N, BF16)[0]
    y, s = ref.attention(**x)
    my, ms = ref.attention(**_abs(x))
    full = pkg.linear_attention_workspace_bytes(B, T, H, N, BF16)
    for nbytes in (full, full // 2, full // 7, 0):
        ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=cuda)[:nbytes] if nbytes else torch.empty(0, dtype=torch.uint8, device=cuda)
        out = _call(pkg, x, workspace=ws)
        _close(out.output, y, my, T, N, BF16, f"output, {nbytes} bytes")
        _close(out.next_state, s, ms, T, N, BF16, f"state, {nbytes} bytes")
    with pytest.raises(pkg.KernelInputsError) as e:
        _call(pkg, x, workspace=torch.empty(64, dtype=torch.uint8, device=cuda)[8:])
    assert e.value.kind == "Unsupported"


@pytest.mark.parametrize("B,T,H", [(40, 17, 5), (40, 47, 5), (40, 48, 5), (1, 32, 148), (1, 47, 149), (1, 513, 40)])
def test_few_tokens_of_many_chains(pkg, cuda, B, T, H):
    """On both sides of what decides between the kernels."""
    _check_forward(pkg, _inputs(cuda, B, T, H, 64, BF16)[0], BF16)


@pytest.mark.parametrize("T", [1, 200])
def test_autograd_captured(pkg, cuda, T):
    x, dy, ds = _inputs(cuda, 1, T, 3, 64, BF16, seed=1)
    leaves = [x[n].requires_grad_() for n in ("q", "k", "v", "s0")]

    def step():
        y, s = pkg.linear_attention_autograd(x["s0"], pkg.LinearAttentionForwardInputs(x["q"], x["k"], x["v"], x["log_decay"]))
        return torch.autograd.grad((y, s), leaves, (dy, ds))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = step()
    new = _inputs(cuda, 1, T, 3, 64, BF16, seed=2)
    with torch.no_grad():
        for n in ("q", "k", "v", "s0"):
            x[n].copy_(new[0][n])
        dy.copy_(new[1])
        ds.copy_(new[2])
    graph.replay()
    want = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(grads, want))


def test_autograd_of_strided_inputs(pkg, cuda):
    """Views of a projection of all three and a state out of a larger one: the autograd form lays them out itself."""
    x, dy, ds = _inputs(cuda, 2, 40, 2, 64, BF16)
    want = torch.autograd.grad(pkg.linear_attention_autograd(
        x["s0"], pkg.LinearAttentionForwardInputs(*(x[n].requires_grad_() for n in ("q", "k", "v")), x["log_decay"])),
        [x[n] for n in ("q", "k", "v")], (dy, ds))
    qkv = torch.stack([x[n].detach() for n in ("q", "k", "v")], dim=3).requires_grad_()
    s0 = torch.stack([x["s0"], x["s0"]], dim=-1)[..., 0]
    out = pkg.linear_attention_autograd(s0, pkg.LinearAttentionForwardInputs(*qkv.unbind(3), x["log_decay"]))
    got, = torch.autograd.grad(out, qkv, (dy, ds))
    assert all(torch.equal(a, b) for a, b in zip(got.unbind(3), want))
