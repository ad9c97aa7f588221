"""The norms before and after a block with its gate and residual scale against their 64-bit form.

Tolerances: a result is off by half a step of its type, plus the roundings of fp32 arithmetic on the same expression over absolute
values: a row's sums are trees of at most 8 + 10 additions and pass through under 30 more operations in all; a parameter's
gradient adds one addition for each row that it is summed over."""
import pytest
import torch

import block_reference as ref

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
NAMES = ("residual", "block_output", "gate", "residual_scale", "post_gamma", "post_beta", "pre_gamma", "pre_beta")
FULL = NAMES
FORMS = {
    "full": FULL,
    "cell": ("residual", "block_output", "pre_gamma", "pre_beta"),               # residual addition and the next norm
    "first": ("residual", "pre_gamma", "pre_beta"),                              # in front of the first block
    "last": ("residual", "block_output", "gate", "residual_scale", "post_gamma"),
    "gated": ("residual", "block_output", "gate", "pre_gamma"),
    "sum": ("residual", "block_output"),
}


def _inputs(cuda, B, T, C, dtype, names, seed=0, mean=0.0):
    g = torch.Generator().manual_seed(seed + 17 * C)
    t = {}
    for n in NAMES:
        shape, scale, shift = ((B, T, C), 1.5, mean) if n in NAMES[:3] else ((C,), 0.2, 1.0 if n.endswith("gamma") else 0.0)
        x = (torch.randn(shape, generator=g) * scale + shift).to(dtype).to(cuda)
        if n in names:
            t[n] = x
    grads = [(torch.randn(B, T, C, generator=g) * s).to(dtype).to(cuda) for s in (0.5, 1.0)]
    return t, grads


def _norm_magnitude(x, gamma, beta, kind, eps, mx):
    """|norm| over absolute values: mx bounds what x was computed from."""
    mean = mx.mean(-1, keepdim=True) if kind == "layer" else 0.0
    centred = x - x.mean(-1, keepdim=True) if kind == "layer" else x
    r = (centred.square().mean(-1, keepdim=True) + eps).rsqrt()
    # a relative error of the root is that of the mean square: once for the summation, twice for its terms' own
    spread = ((mx + mean) * centred.abs()).mean(-1, keepdim=True) * r * r
    y = ((mx + mean) * r + centred.abs() * r * (1 + spread)) * gamma.abs()
    return y if beta is None else y + beta.abs()


def _forward_magnitudes(t, kind, eps):
    d = {n: x.double() for n, x in t.items()}
    x, mx = d["residual"], d["residual"].abs()
    if "block_output" in d:
        h = d["block_output"]
        mu = h.abs() if "post_gamma" not in d else _norm_magnitude(h, d["post_gamma"], d.get("post_beta"), kind, eps, h.abs())
        mx = mx + d.get("residual_scale", torch.ones((), dtype=torch.float64)).abs().to(h.device) * d.get("gate", torch.ones_like(h)).abs() * mu
        x = ref.between(d["residual"], d["block_output"], d.get("gate"), d.get("residual_scale"), d.get("post_gamma"), d.get("post_beta"),
                        kind=kind, eps=eps)[0]
    mz = None if "pre_gamma" not in d else _norm_magnitude(x, d["pre_gamma"], d.get("pre_beta"), kind, eps, mx)
    return mx, mz


def _within(got, want, magnitude, steps, what):
    bound = ref.HALF_STEP[got.dtype] * want.abs() + steps * ref.U * magnitude
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"{what}: {int((off > bound).sum())} beyond, worst {float((off / bound.clamp_min(1e-300)).max()):.3g} of the bound"


def _check_forward(pkg, cuda, B, T, C, dtype, kind, form, mean=0.0, eps=1e-5):
    t, _ = _inputs(cuda, B, T, C, dtype, FORMS[form], mean=mean)
    out = pkg.residual_norm(pkg.ResidualNormForwardInputs(**t, kind=kind, epsilon=eps))
    want = ref.between(**{n: x.double() for n, x in t.items()}, kind=kind, eps=eps)
    for name, got, w, m in zip(("next_residual", "normed"), (out.next_residual, out.normed), want, _forward_magnitudes(t, kind, eps)):
        assert (got is None) == (w is None), name
        if w is not None:
            _within(got, w, m, 48, name)
    return t, out


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("C", [1, 7, 64, 100, 768, 2047, 2048, 2560, 8191, 8192])
def test_forward(pkg, cuda, C, kind, dtype):
    _check_forward(pkg, cuda, 2, 3, C, dtype, kind, "full")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("form", list(FORMS))
def test_parts_left_out(pkg, cuda, form, kind, dtype):
    _check_forward(pkg, cuda, 3, 5, 256, dtype, kind, form)


def test_one_row_and_many(pkg, cuda):
    _check_forward(pkg, cuda, 1, 1, 2048, BF16, "layer", "full")
    _check_forward(pkg, cuda, 3, 1111, 768, BF16, "layer", "full")


def test_a_mean_far_from_zero(pkg, cuda):
    """The variance is taken from the differences: a mean of a thousand deviations costs what its own rounding costs."""
    _check_forward(pkg, cuda, 2, 4, 1024, F32, "layer", "full", mean=1000.0)


def test_no_rows(pkg, cuda):
    t, grads = _inputs(cuda, 0, 5, 64, F32, FULL)
    out = pkg.residual_norm(pkg.ResidualNormForwardInputs(**t))
    assert out.normed.shape == (0, 5, 64)
    g = pkg.residual_norm_backward(pkg.ResidualNormForwardInputs(**t), *grads)
    assert all(bool((x == 0).all()) for x in g[3:])


def test_constant_rows_and_zero_epsilon(pkg, cuda):
    x = torch.full((1, 3, 64), 2.0, device=cuda)
    w = torch.ones(64, device=cuda)
    out = pkg.residual_norm(pkg.ResidualNormForwardInputs(x, pre_gamma=w, epsilon=1e-5))
    assert bool((out.normed == 0).all())
    out = pkg.residual_norm(pkg.ResidualNormForwardInputs(x, pre_gamma=w, kind="rms", epsilon=0.0))
    assert bool((out.normed == 1).all())


def test_rows_do_not_touch_one_another(pkg, cuda):
    t, out = _check_forward(pkg, cuda, 1, 9, 200, BF16, "layer", "full")
    t["block_output"][0, 4, 3] = float("nan")
    again = pkg.residual_norm(pkg.ResidualNormForwardInputs(**t))
    keep = [i for i in range(9) if i != 4]
    assert torch.equal(again.normed[:, keep], out.normed[:, keep]) and bool(torch.isnan(again.normed[0, 4]).all())


def test_in_place(pkg, cuda):
    t, out = _check_forward(pkg, cuda, 2, 5, 300, BF16, "layer", "full")
    got = pkg.residual_norm(pkg.ResidualNormForwardInputs(**t), next_residual=t["residual"], normed=t["block_output"])
    assert got.next_residual is t["residual"] and torch.equal(t["residual"], out.next_residual) and torch.equal(t["block_output"], out.normed)


def _grads_64(t, grads, kind, eps):
    leaves = {n: x.double().requires_grad_() for n, x in t.items()}
    outs = ref.between(**leaves, kind=kind, eps=eps)
    pairs = [(o, g.double()) for o, g in zip(outs, grads) if o is not None]
    got = torch.autograd.grad([o for o, _ in pairs], list(leaves.values()), [g for _, g in pairs])
    return dict(zip(leaves, got))


def _magnitudes_back(t, grads, kind, eps):
    """The backward pass over absolute values; `spread` terms as in the forward pass."""
    d = {n: x.double() for n, x in t.items()}
    one = torch.ones_like(d["residual"])
    h = d.get("block_output")
    mh = mu = u_hat_r = None
    if h is not None and "post_gamma" in d:
        mu = _norm_magnitude(h, d["post_gamma"], d.get("post_beta"), kind, eps, h.abs())
        mh = _norm_magnitude(h, torch.ones_like(d["post_gamma"]), None, kind, eps, h.abs())
        c = h - h.mean(-1, keepdim=True) if kind == "layer" else h
        u_hat_r = (c.square().mean(-1, keepdim=True) + eps).rsqrt()
    elif h is not None:
        mu = h.abs()
    mx, _ = _forward_magnitudes(t, kind, eps)
    x = d["residual"] if h is None else ref.between(**{n: v for n, v in d.items() if not n.startswith("pre")}, kind=kind, eps=eps)[0]

    def back(g, hat, r):
        # (the root's own relative error counts as in the magnitudes of the forward pass: hat holds it)
        total = g + (g.mean(-1, keepdim=True) if kind == "layer" else 0.0) + hat * (g * hat).mean(-1, keepdim=True)
        return r * total * (1 + hat.square().mean(-1, keepdim=True))

    m = {}
    dx = torch.zeros_like(one)
    if "pre_gamma" in d:
        dz = grads[1].double().abs()
        hat = _norm_magnitude(x, torch.ones_like(d["pre_gamma"]), None, kind, eps, mx)
        c = x - x.mean(-1, keepdim=True) if kind == "layer" else x
        r = (c.square().mean(-1, keepdim=True) + eps).rsqrt()
        m["pre_gamma"], m["pre_beta"] = (dz * hat).sum((0, 1)), dz.sum((0, 1))
        dx = back(dz * d["pre_gamma"].abs(), hat, r)
    if h is not None:
        dx = dx + grads[0].double().abs()
        gate, scale = d.get("gate", one).abs(), d.get("residual_scale", torch.ones(one.shape[-1], dtype=torch.float64, device=one.device)).abs()
        m["residual_scale"] = (dx * gate * mu).sum((0, 1))
        m["gate"] = dx * scale * mu
        du = dx * scale * gate
        m["block_output"] = du
        if "post_gamma" in d:
            m["post_gamma"], m["post_beta"] = (du * mh).sum((0, 1)), du.sum((0, 1))
            m["block_output"] = back(du * d["post_gamma"].abs(), mh, u_hat_r)
    m["residual"] = dx
    return m


def _check_backward(pkg, cuda, B, T, C, dtype, kind, form, eps=1e-5):
    t, grads = _inputs(cuda, B, T, C, dtype, FORMS[form], seed=3)
    given = [g if wanted else None for g, wanted in zip(grads, ("block_output" in t, "pre_gamma" in t))]
    got = dict(zip(NAMES, pkg.residual_norm_backward(pkg.ResidualNormForwardInputs(**t, kind=kind, epsilon=eps), *given)))
    want, mag = _grads_64(t, grads, kind, eps), _magnitudes_back(t, grads, kind, eps)
    for n in NAMES:
        assert (got[n] is None) == (n not in t), n
        if n in t:
            _within(got[n], want[n], mag[n], 96 + (B * T if want[n].dim() == 1 else 0), n)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("B,T,C", [(1, 1, 64), (2, 3, 7), (3, 100, 768), (1, 301, 1001), (2, 5, 2048), (1, 3, 8192), (1, 2, 8191)])
def test_backward(pkg, cuda, B, T, C, kind, dtype):
    _check_backward(pkg, cuda, B, T, C, dtype, kind, "full")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("form", list(FORMS))
def test_backward_of_parts(pkg, cuda, form, kind, dtype):
    _check_backward(pkg, cuda, 2, 33, 256, dtype, kind, form)


def test_gradients_against_differences(pkg, cuda):
    """Central differences of step e in fp32: the error of third order is e^2 of the derivative's own size, roundings are 2^-24 / e of
    the values summed; with e = 2^-8 both are a few 1e-5 of the sum of absolute products."""
    t, grads = _inputs(cuda, 1, 6, 64, F32, FULL, seed=9)
    inputs = pkg.ResidualNormForwardInputs(**{n: x.clone().requires_grad_() for n, x in t.items()})
    x, z = pkg.residual_norm_autograd(inputs)
    got = torch.autograd.grad((x, z), inputs.eight(), grads)
    g = torch.Generator().manual_seed(2)
    e = 2.0 ** -8
    for n, grad in zip(NAMES, got):
        d = torch.randn(t[n].shape, generator=g).to(cuda)
        ends = []
        for sign in (1.0, -1.0):
            out = pkg.residual_norm(pkg.ResidualNormForwardInputs(**dict(t, **{n: t[n] + sign * e * d})))
            ends.append((out.next_residual.double() * grads[0]).sum() + (out.normed.double() * grads[1]).sum())
        mag = float((out.next_residual.double() * grads[0]).abs().sum() + (out.normed.double() * grads[1]).abs().sum())
        assert abs(float((ends[0] - ends[1]) / (2 * e) - (grad.double() * d.double()).sum())) <= 2e-3 * mag, n


def test_autograd_without_some_gradients(pkg, cuda):
    t, grads = _inputs(cuda, 2, 3, 64, BF16, FORMS["cell"])
    for n in t:
        t[n].requires_grad_()
    x, z = pkg.residual_norm_autograd(pkg.ResidualNormForwardInputs(**t))
    only = torch.autograd.grad(x, [t["residual"], t["block_output"]], grads[0], retain_graph=True)
    assert all(torch.equal(g, grads[0]) for g in only)
    want = _grads_64({n: v.detach() for n, v in t.items()}, [torch.zeros_like(grads[0]), grads[1]], "layer", 1e-5)
    mag = _magnitudes_back({n: v.detach() for n, v in t.items()}, [torch.zeros_like(grads[0]), grads[1]], "layer", 1e-5)
    for n, g in zip(t, torch.autograd.grad(z, list(t.values()), grads[1])):
        _within(g, want[n], mag[n], 128, n)


def test_sums_over_rows_do_not_change_from_call_to_call(pkg, cuda):
    t, grads = _inputs(cuda, 4, 501, 512, BF16, FULL)
    inputs = pkg.ResidualNormForwardInputs(**t)
    first = pkg.residual_norm_backward(inputs, *grads)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, pkg.residual_norm_backward(inputs, *grads)))


def test_captured_and_replayed_with_new_values(pkg, cuda):
    t, grads = _inputs(cuda, 2, 40, 768, BF16, FULL)
    inputs = pkg.ResidualNormForwardInputs(**t)

    def step():
        return pkg.residual_norm(inputs), pkg.residual_norm_backward(inputs, *grads)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, back = step()
    new, new_grads = _inputs(cuda, 2, 40, 768, BF16, FULL, seed=77)
    for n in t:
        t[n].copy_(new[n])
    for a, b in zip(grads, new_grads):
        a.copy_(b)
    graph.replay()
    want, want_back = step()
    torch.cuda.synchronize()
    assert torch.equal(out.next_residual, want.next_residual) and torch.equal(out.normed, want.normed)
    assert all(torch.equal(a, b) for a, b in zip(back, want_back))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_autograd_of_strided_and_broadcast_inputs(pkg, cuda, dtype):
    """A gate that all rows share, a block output out of a larger projection, parameters out of one tensor: the autograd form lays them out, and
    the gradients come back in the places they were taken from."""
    B, T, C = 2, 5, 96
    t, grads = _inputs(cuda, B, T, C, dtype, FULL, seed=5)
    want_in = dict(t, gate=t["gate"][:1, :1].expand(B, T, C).contiguous())
    want = dict(zip(NAMES, pkg.residual_norm_backward(pkg.ResidualNormForwardInputs(**want_in), *grads)))
    gate = t["gate"][:1, :1].clone().requires_grad_()
    wide = torch.stack([t["block_output"], t["residual"]], dim=2).requires_grad_()
    params = torch.stack([t[n] for n in NAMES[3:]], dim=1).requires_grad_()
    strided = dict(zip(NAMES[3:], params.unbind(1)), residual=t["residual"].transpose(0, 1).contiguous().transpose(0, 1), block_output=wide[:, :, 0],
                   gate=gate.expand(B, T, C))
    x, z = pkg.residual_norm_autograd(pkg.ResidualNormForwardInputs(**strided))
    of_gate, of_wide, of_params = torch.autograd.grad((x, z), (gate, wide, params), grads)
    assert torch.equal(of_wide[:, :, 0], want["block_output"]) and bool((of_wide[:, :, 1] == 0).all())
    assert all(torch.equal(of_params[:, i], want[n]) for i, n in enumerate(NAMES[3:]))
    assert torch.equal(of_gate, want["gate"].sum((0, 1), keepdim=True))
