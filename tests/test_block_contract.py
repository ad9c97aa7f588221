"""Refusals of linear attention, the residual norms and beam search: wrong calls fail on the host, before any CUDA call."""
import ctypes

import pytest
import torch


def _attention(pkg, shape=(2, 5, 3, 64), dtype=torch.float32, **change):
    t = dict(query=torch.zeros(shape, dtype=dtype), key=torch.zeros(shape, dtype=dtype), value=torch.zeros(shape, dtype=dtype),
             log_decay=torch.zeros(shape[2]), context_lens=None)
    t.update(change)
    return pkg.LinearAttentionForwardInputs(**t)


def _refused(pkg, kind, call, match=None):
    with pytest.raises(pkg.KernelInputsError, match=match) as e:
        call()
    assert e.value.kind == kind, (e.value.kind, str(e.value))


def test_linear_attention_refusals(pkg):
    z = torch.zeros
    bad = [
        ("ShapeMismatch", dict(key=z(2, 5, 3, 32)), "key"),
        ("ShapeMismatch", dict(value=z(2, 4, 3, 64)), "value"),
        ("ShapeMismatch", dict(query=z(2, 5, 192)), "query"),
        ("DTypeMismatch", dict(key=z(2, 5, 3, 64, dtype=torch.bfloat16)), "key"),
        ("NotContiguous", dict(key=z(2, 3, 5, 64).transpose(1, 2)), "key"),
        ("ShapeMismatch", dict(log_decay=z(2)), "log_decay"),
        ("DTypeMismatch", dict(log_decay=z(3, dtype=torch.bfloat16)), "log_decay"),
        ("ShapeMismatch", dict(context_lens=z(3, dtype=torch.int32)), "context_lens"),
        ("DTypeMismatch", dict(context_lens=z(2, dtype=torch.int64)), "context_lens"),
    ]
    for kind, change, name in bad:
        _refused(pkg, kind, lambda: pkg.linear_attention(_attention(pkg, **change)), name)
    _refused(pkg, "EmptyAxis", lambda: pkg.linear_attention(_attention(pkg, (2, 0, 3, 64))))
    _refused(pkg, "Unsupported", lambda: pkg.linear_attention(_attention(pkg, (2, 5, 3, 48))), "head sizes")
    _refused(pkg, "Unsupported", lambda: pkg.linear_attention(_attention(pkg, dtype=torch.float16)))
    _refused(pkg, "NotContiguous", lambda: pkg.linear_attention(_attention(pkg), z(2, 64, 3, 64).transpose(1, 2)), "initial_state")
    _refused(pkg, "ShapeMismatch", lambda: pkg.linear_attention(_attention(pkg), z(2, 3, 64, 32)), "initial_state")
    _refused(pkg, "DTypeMismatch", lambda: pkg.linear_attention(_attention(pkg), z(2, 3, 64, 64, dtype=torch.bfloat16)), "initial_state")
    inputs = _attention(pkg)
    _refused(pkg, "BadArgument", lambda: pkg.linear_attention(inputs, output=inputs.value), "share memory")
    two = z(2 * 2 * 3 * 64 * 64)
    half = two.numel() // 4
    _refused(pkg, "BadArgument", lambda: pkg.linear_attention(
        inputs, two[:2 * half].view(2, 3, 64, 64), next_state=two[half:3 * half].view(2, 3, 64, 64)), "share memory")
    _refused(pkg, "NotContiguous", lambda: pkg.linear_attention_backward(inputs, z(2, 3, 5, 64).transpose(1, 2)), "output_grad")
    _refused(pkg, "ShapeMismatch", lambda: pkg.linear_attention_backward(inputs, z(2, 5, 3, 64), z(2, 3, 64)), "next_state_grad")
    inputs.log_decay.requires_grad_()
    _refused(pkg, "Unsupported", lambda: pkg.linear_attention_autograd(None, inputs), "no gradient")


def test_linear_attention_of_no_chain_is_nothing(pkg):
    out = pkg.linear_attention(_attention(pkg, (0, 5, 3, 64)))
    assert out.output.shape == (0, 5, 3, 64) and out.next_state.shape == (0, 3, 64, 64)


def test_residual_norm_refusals(pkg):
    z, x, w = torch.zeros, torch.zeros(2, 3, 16), torch.zeros(16)

    def call(*args, out=None, **kw):
        return lambda: pkg.residual_norm(pkg.ResidualNormForwardInputs(*args, **kw), **(out or {}))

    _refused(pkg, "NullPointer", call(x), "block_output, pre_gamma")
    _refused(pkg, "NullPointer", call(x, gate=x, pre_gamma=w), "gate needs block_output")
    _refused(pkg, "NullPointer", call(x, x.clone(), post_beta=w), "post_beta needs post_gamma")
    _refused(pkg, "NullPointer", call(x, x.clone(), pre_beta=w), "pre_beta needs pre_gamma")
    _refused(pkg, "ShapeMismatch", call(z(6, 16), pre_gamma=w))
    _refused(pkg, "ShapeMismatch", call(x, z(2, 3, 8)), "block_output")
    _refused(pkg, "ShapeMismatch", call(x, pre_gamma=z(15)), "pre_gamma")
    _refused(pkg, "DTypeMismatch", call(x, pre_gamma=w.bfloat16()), "pre_gamma")
    _refused(pkg, "NotContiguous", call(z(2, 16, 3).transpose(1, 2), pre_gamma=w), "residual")
    _refused(pkg, "EmptyAxis", call(z(2, 3, 0), pre_gamma=z(0)))
    _refused(pkg, "Unsupported", call(z(1, 1, 8193), pre_gamma=z(8193)), "8193 channels")
    _refused(pkg, "Unsupported", call(x.half(), pre_gamma=w.half()))
    _refused(pkg, "BadArgument", call(x, pre_gamma=w, kind="group"))
    for eps in (-1.0, float("nan"), float("inf")):
        _refused(pkg, "BadArgument", call(x, pre_gamma=w, epsilon=eps))
    same = torch.zeros(2, 3, 16)
    _refused(pkg, "BadArgument", call(x, x.clone(), pre_gamma=w, out=dict(next_residual=same, normed=same)), "share memory")
    _refused(pkg, "NullPointer", call(x, pre_gamma=w, out=dict(next_residual=same)), "next_residual")
    _refused(pkg, "NullPointer", lambda: pkg.residual_norm_backward(pkg.ResidualNormForwardInputs(x, pre_gamma=w), x), "normed_grad")
    _refused(pkg, "NullPointer", lambda: pkg.residual_norm_backward(pkg.ResidualNormForwardInputs(x, x.clone()), x, x.clone()), "normed_grad")


def test_beam_select_refusals(pkg):
    z = torch.zeros
    logits, scores = z(2, 4, 10), z(2, 4)

    def call(*args, **kw):
        return lambda: pkg.beam_select(*args, **kw)

    _refused(pkg, "ShapeMismatch", call(z(8, 10), scores, 4), "logits")
    _refused(pkg, "ShapeMismatch", call(logits, z(2, 3), 4), "scores")
    _refused(pkg, "DTypeMismatch", call(logits, scores.bfloat16(), 4), "scores")
    _refused(pkg, "DTypeMismatch", call(logits, scores, 4, finished=z(2, 4)), "finished")
    _refused(pkg, "EmptyAxis", call(z(2, 4, 0), scores, 4))
    _refused(pkg, "NotContiguous", call(z(2, 10, 4).transpose(1, 2), scores, 4), "logits")
    _refused(pkg, "Unsupported", call(logits.half(), scores, 4))
    for k in (0, 33):
        _refused(pkg, "Unsupported", call(logits, scores, k), "beam_select")
    _refused(pkg, "Unsupported", call(z(1, 2, 3), z(1, 2), 7), "beam_select")
    _refused(pkg, "Unsupported", call(z(1, 33, 3), z(1, 33), 4), "beam_select")
    for pad in (-1, 10):
        _refused(pkg, "BadArgument", call(logits, scores, 4, finished=z(2, 4, dtype=torch.int32), pad_token=pad), "pad_token")
    _refused(pkg, "WorkspaceTooSmall", call(logits, scores, 4, workspace=z(16, dtype=torch.uint8)))


def test_beam_reorder_refusals(pkg):
    z = torch.zeros
    state, parents = z(8, 3, 4), z(2, 4, dtype=torch.int32)

    def call(*args, **kw):
        return lambda: pkg.beam_reorder(*args, **kw)

    _refused(pkg, "DTypeMismatch", call([state], z(2, 4)), "parents")
    _refused(pkg, "ShapeMismatch", call([state], z(8, dtype=torch.int32)), "parents")
    _refused(pkg, "ShapeMismatch", call([z(6, 3)], parents), "rows")
    _refused(pkg, "ShapeMismatch", call([z(7, 3)], parents, out=[z(8, 3)]), "rows")
    _refused(pkg, "ShapeMismatch", call([state], parents, out=[z(8, 3, 5)]), "out")
    _refused(pkg, "DTypeMismatch", call([state], parents, out=[state.bfloat16()]))
    _refused(pkg, "NotContiguous", call([z(8, 4, 3).transpose(1, 2)], parents), "states")
    _refused(pkg, "BadArgument", call([state, state], parents), "share memory")
    _refused(pkg, "BadArgument", call([state], parents, out=[state]), "share memory")
    _refused(pkg, "Unsupported", call([z(66, 2)], z(2, 33, dtype=torch.int32)), "33 beams")
    with pytest.raises(ValueError):
        pkg.beam_reorder([state], parents, out=[])
    with pytest.raises(TypeError):
        pkg.beam_reorder([None], parents)


def test_null_descriptors(pkg):
    L = pkg.lib()
    null = ctypes.c_void_p(0)
    assert L.rwkv7_fused_linear_attention(*[null] * 9, ctypes.c_size_t(0), null) == 9
    assert L.rwkv7_beam_reorder(null, ctypes.c_int32(1), null, null, null) == 9
    p = pkg.describe(torch.zeros(2, 4, dtype=torch.int32))
    assert L.rwkv7_beam_reorder(null, ctypes.c_int32(1), ctypes.byref(p), null, null) == 9
    assert L.rwkv7_beam_reorder(null, ctypes.c_int32(-1), ctypes.byref(p), null, null) == 14
