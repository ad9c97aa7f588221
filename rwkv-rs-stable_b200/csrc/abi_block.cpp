// extern "C" entry points of the operators around a recurrent block that the reference does not have: linear attention with a
// decay per head, the norms before and after a block, beam search.  Checks in the order and with the messages of abi.cpp.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <memory>
#include <new>

#include "abi_common.h"
#include "check.h"
#include "kernels.h"
#include "rwkv7_b200.h"
#include "trace.h"

using namespace rwkv7;

namespace {

size_t bytes_of(const rwkv7_tensor *t) { return (size_t)num_elements(t) * dtype_size(t->dtype); }

bool overlap(const rwkv7_tensor *a, const rwkv7_tensor *b) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(a->data), q = reinterpret_cast<uintptr_t>(b->data);
    return p < q + bytes_of(b) && q < p + bytes_of(a);
}

// What is written may not share memory with what is read (or written) beside it.
int check_apart(const TensorInfo &a, const TensorInfo &b) {
    if (a.t == nullptr || b.t == nullptr || !overlap(a.t, b.t)) return RWKV7_OK;
    return fail(RWKV7_ERR_BAD_ARGUMENT, "BadArgument: %s and %s share memory", a.name, b.name);
}
int check_same_or_apart(const TensorInfo &a, const TensorInfo &b) {
    return a.t != nullptr && b.t != nullptr && a.t->data == b.t->data ? RWKV7_OK : check_apart(a, b);
}

int check_dtype(const TensorInfo &x, int32_t dtype) {
    if (x.t->dtype == dtype) return RWKV7_OK;
    return fail(RWKV7_ERR_DTYPE_MISMATCH, "DTypeMismatch: %s must be %s, got %s", x.name, dtype_name(dtype), dtype_name(x.t->dtype));
}

int check_float(const TensorInfo &x, const char *op) {
    if (float_dtype_supported(x.t->dtype)) return RWKV7_OK;
    return fail(RWKV7_ERR_UNSUPPORTED, "Unsupported: %s computes F32 or BF16, got %s", op, dtype_name(x.t->dtype));
}

int check_like(const TensorInfo &ref, const TensorInfo &x) {
    RWKV7_TRY(check_present(x, ref.t->ndim));
    RWKV7_TRY(check_shape(x, ref.t->shape, ref.t->ndim));
    RWKV7_TRY(check_same_dtype({ref, x}));
    RWKV7_TRY(check_same_device({ref, x}));
    return check_contiguous(x);
}

int check_of(const TensorInfo &ref, const TensorInfo &x, std::initializer_list<int64_t> shape, int32_t dtype) {
    RWKV7_TRY(check_present(x, (int)shape.size()));
    RWKV7_TRY(check_shape(x, shape));
    RWKV7_TRY(check_dtype(x, dtype));
    RWKV7_TRY(check_same_device({ref, x}));
    return check_contiguous(x);
}

// A workspace of fewer than `need` bytes is refused; so is one that vector accesses cannot reach.
int check_workspace(const char *op, const void *workspace, size_t bytes, size_t need) {
    if (need > 0 && (workspace == nullptr || bytes < need))
        return fail(RWKV7_ERR_WORKSPACE_TOO_SMALL, "WorkspaceTooSmall: %s needs %zu workspace bytes, got %zu", op, need,
                    workspace == nullptr ? (size_t)0 : bytes);
    if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)
        return fail(RWKV7_ERR_UNSUPPORTED, "Unsupported: the %s workspace must be 16-byte aligned", op);
    return RWKV7_OK;
}

int current_sms() {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || num_sms(dev, &sms) != RWKV7_OK) return 0;
    return sms;
}

// ---- linear attention ----------------------------------------------------------------------------------------------------

// The contract that both directions share; `p` gets the sizes.
int check_linear_attention(const TensorInfo &s0, const TensorInfo (&qkv)[3], const TensorInfo &decay, const TensorInfo &lens,
                           LinearAttentionPass &p) {
    const TensorInfo &q = qkv[0];
    RWKV7_TRY(check_present(q, 4));
    RWKV7_TRY(check_axis_non_empty(q, 1));
    for (int i = 1; i < 3; ++i) {
        RWKV7_TRY(check_present(qkv[i], 4));
        RWKV7_TRY(check_shape(qkv[i], q.t->shape, 4));
    }
    RWKV7_TRY(check_same_dtype(qkv, 3));
    RWKV7_TRY(check_same_device(qkv, 3));
    for (const TensorInfo &x : qkv) RWKV7_TRY(check_contiguous(x));
    RWKV7_TRY(check_float(q, "linear_attention"));
    if (!linear_attention_supported(q.dim(3)))
        return fail(RWKV7_ERR_UNSUPPORTED, "Unsupported: linear_attention computes head sizes 32, 64 and 128, got %lld", (long long)q.dim(3));
    p.B = q.dim(0); p.T = q.dim(1); p.H = q.dim(2); p.N = q.dim(3);
    if (p.T > INT32_MAX - 256 || p.H > INT32_MAX / p.N || (p.H > 0 && p.B > INT32_MAX / p.H))
        return fail(RWKV7_ERR_UNSUPPORTED, "Unsupported: linear_attention of %s", shape_string(q.t->shape, 4).c_str());
    RWKV7_TRY(check_of(q, decay, {p.H}, RWKV7_F32));
    if (lens.t != nullptr) RWKV7_TRY(check_of(q, lens, {p.B}, RWKV7_I32));
    if (s0.t != nullptr) RWKV7_TRY(check_of(q, s0, {p.B, p.H, p.N, p.N}, RWKV7_F32));
    p.log_decay = static_cast<const float *>(decay.t->data);
    p.lens = lens.t == nullptr ? nullptr : static_cast<const int *>(lens.t->data);
    p.bf16 = q.t->dtype == RWKV7_BF16;
    p.device = q.t->device;
    return RWKV7_OK;
}

size_t attention_workspace(int64_t B, int64_t T, int64_t H, int64_t N, int32_t dtype) {
    LinearAttentionPass p{};
    p.B = B; p.T = T; p.H = H; p.N = N;
    p.bf16 = dtype == RWKV7_BF16;
    p.num_sms = current_sms();
    return B <= 0 || T <= 0 || H <= 0 || !float_dtype_supported(dtype) || !linear_attention_supported(N) ? 0 : linear_attention_workspace_bytes(p);
}

}  // namespace

extern "C" {

size_t rwkv7_linear_attention_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t N, int32_t dtype) {
    return attention_workspace(B, T, H, N, dtype);
}

// (its passes use it in turn)
size_t rwkv7_linear_attention_backward_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t N, int32_t dtype) {
    return attention_workspace(B, T, H, N, dtype);
}

int rwkv7_fused_linear_attention(const rwkv7_tensor *s0_t, const rwkv7_tensor *q_t, const rwkv7_tensor *k_t, const rwkv7_tensor *v_t,
                                 const rwkv7_tensor *decay_t, const rwkv7_tensor *lens_t, rwkv7_tensor *y_t, rwkv7_tensor *s_t,
                                 void *workspace, size_t workspace_bytes, rwkv7_stream stream) {
    RWKV7_TRACE("rwkv.infer.model.linear_attention");
    clear_error();
    const TensorInfo s0{"initial_state", s0_t}, qkv[3] = {{"query", q_t}, {"key", k_t}, {"value", v_t}}, decay{"log_decay", decay_t},
        lens{"context_lens", lens_t}, y{"output", y_t}, s{"next_state", s_t};
    LinearAttentionPass p{};
    RWKV7_TRY(check_linear_attention(s0, qkv, decay, lens, p));
    RWKV7_TRY(check_like(qkv[0], y));
    if (s_t != nullptr) {
        RWKV7_TRY(check_of(qkv[0], s, {p.B, p.H, p.N, p.N}, RWKV7_F32));
        RWKV7_TRY(check_same_or_apart(s, s0));
    }
    for (const TensorInfo &x : {qkv[0], qkv[1], qkv[2], s0, s, decay, lens}) RWKV7_TRY(check_apart(y, x));
    for (const TensorInfo &x : {qkv[0], qkv[1], qkv[2], decay, lens}) RWKV7_TRY(check_apart(s, x));
    RWKV7_TRY(check_workspace("linear_attention", workspace, workspace_bytes, 0));
    if (p.B == 0 || p.H == 0) return RWKV7_OK;
    DeviceGuard guard(p.device);
    if (guard.error() != cudaSuccess) return cuda_fail("cudaSetDevice", (int)guard.error());
    RWKV7_TRY(num_sms(p.device, &p.num_sms));
    p.a = q_t->data; p.b = k_t->data; p.c = v_t->data; p.y = y_t->data;
    p.s_in = s0_t == nullptr ? nullptr : static_cast<const float *>(s0_t->data);
    p.s_out = s_t == nullptr ? nullptr : static_cast<float *>(s_t->data);
    if (int e = launch_linear_attention(p, workspace, workspace_bytes, (cudaStream_t)stream)) return cuda_fail("linear_attention launch", e);
    return RWKV7_OK;
}

int rwkv7_fused_linear_attention_backward(const rwkv7_tensor *s0_t, const rwkv7_tensor *q_t, const rwkv7_tensor *k_t,
                                          const rwkv7_tensor *v_t, const rwkv7_tensor *decay_t, const rwkv7_tensor *lens_t,
                                          const rwkv7_tensor *dy_t, const rwkv7_tensor *ds_t, rwkv7_tensor *dq_t, rwkv7_tensor *dk_t,
                                          rwkv7_tensor *dv_t, rwkv7_tensor *ds0_t, void *workspace, size_t workspace_bytes,
                                          rwkv7_stream stream) {
    RWKV7_TRACE("rwkv.train.model.linear_attention");
    clear_error();
    const TensorInfo s0{"initial_state", s0_t}, qkv[3] = {{"query", q_t}, {"key", k_t}, {"value", v_t}}, decay{"log_decay", decay_t},
        lens{"context_lens", lens_t}, dy{"output_grad", dy_t}, ds{"next_state_grad", ds_t},
        grads[4] = {{"query_grad", dq_t}, {"key_grad", dk_t}, {"value_grad", dv_t}, {"initial_state_grad", ds0_t}};
    LinearAttentionPass p{};
    RWKV7_TRY(check_linear_attention(s0, qkv, decay, lens, p));
    RWKV7_TRY(check_like(qkv[0], dy));
    if (ds_t != nullptr) RWKV7_TRY(check_of(qkv[0], ds, {p.B, p.H, p.N, p.N}, RWKV7_F32));
    for (int i = 0; i < 3; ++i) RWKV7_TRY(check_like(qkv[0], grads[i]));
    if (ds0_t != nullptr) RWKV7_TRY(check_of(qkv[0], grads[3], {p.B, p.H, p.N, p.N}, RWKV7_F32));
    for (int i = 0; i < 4; ++i) {
        for (const TensorInfo &x : {qkv[0], qkv[1], qkv[2], s0, decay, lens, dy, ds}) RWKV7_TRY(check_apart(grads[i], x));
        for (int j = 0; j < i; ++j) RWKV7_TRY(check_apart(grads[i], grads[j]));
    }
    RWKV7_TRY(check_workspace("linear_attention_backward", workspace, workspace_bytes, 0));
    if (p.B == 0 || p.H == 0) return RWKV7_OK;
    DeviceGuard guard(p.device);
    if (guard.error() != cudaSuccess) return cuda_fail("cudaSetDevice", (int)guard.error());
    RWKV7_TRY(num_sms(p.device, &p.num_sms));
    const float *state = s0_t == nullptr ? nullptr : static_cast<const float *>(s0_t->data);
    const float *state_grad = ds_t == nullptr ? nullptr : static_cast<const float *>(ds_t->data);
    LinearAttentionPass dq = p, dv = p, dk = p;
    dq.a = dy_t->data; dq.b = v_t->data; dq.c = k_t->data; dq.y = dq_t->data;
    dq.s_in = state; dq.s_in_transposed = true;
    dv.a = k_t->data; dv.b = q_t->data; dv.c = dy_t->data; dv.y = dv_t->data; dv.reversed = true;
    dv.s_in = state_grad;
    dv.s_out = ds0_t == nullptr ? nullptr : static_cast<float *>(ds0_t->data);
    dk.a = v_t->data; dk.b = dy_t->data; dk.c = q_t->data; dk.y = dk_t->data; dk.reversed = true;
    dk.s_in = state_grad; dk.s_in_transposed = true;
    for (const LinearAttentionPass *pass : {&dq, &dv, &dk})
        if (int e = launch_linear_attention(*pass, workspace, workspace_bytes, (cudaStream_t)stream)) return cuda_fail("linear_attention_backward launch", e);
    return RWKV7_OK;
}

// ---- norms before and after a block -----------------------------------------------------------------------------------------

}  // extern "C"

namespace {

struct NormTensors {
    TensorInfo residual, block_output, gate, scale, post_gamma, post_beta, pre_gamma, pre_beta;
};

int check_norm(const NormTensors &t, int32_t kind, double epsilon, ResidualNormArgs &p) {
    const TensorInfo &x = t.residual;
    RWKV7_TRY(check_present(x, 3));
    RWKV7_TRY(check_axis_non_empty(x, 2));
    RWKV7_TRY(check_contiguous(x));
    RWKV7_TRY(check_float(x, "residual_norm"));
    p.C = x.dim(2);
    if (p.C > residual_norm_max_channels())
        return fail(RWKV7_ERR_UNSUPPORTED, "Unsupported: residual_norm of %lld channels, at most %lld", (long long)p.C,
                    (long long)residual_norm_max_channels());
    if (x.dim(1) > 0 && x.dim(0) > INT32_MAX / x.dim(1))
        return fail(RWKV7_ERR_UNSUPPORTED, "Unsupported: residual_norm of %s", shape_string(x.t->shape, 3).c_str());
    p.rows = x.dim(0) * x.dim(1);
    if (t.block_output.t != nullptr) RWKV7_TRY(check_like(x, t.block_output));
    for (const TensorInfo &part : {t.gate, t.scale, t.post_gamma})
        if (part.t != nullptr && t.block_output.t == nullptr)
            return fail(RWKV7_ERR_NULL_POINTER, "NullPointer: %s needs block_output", part.name);
    if (t.gate.t != nullptr) RWKV7_TRY(check_like(x, t.gate));
    if (t.post_beta.t != nullptr && t.post_gamma.t == nullptr) return fail(RWKV7_ERR_NULL_POINTER, "NullPointer: post_beta needs post_gamma");
    if (t.pre_beta.t != nullptr && t.pre_gamma.t == nullptr) return fail(RWKV7_ERR_NULL_POINTER, "NullPointer: pre_beta needs pre_gamma");
    if (t.block_output.t == nullptr && t.pre_gamma.t == nullptr)
        return fail(RWKV7_ERR_NULL_POINTER, "NullPointer: residual_norm needs block_output, pre_gamma or both");
    for (const TensorInfo &w : {t.scale, t.post_gamma, t.post_beta, t.pre_gamma, t.pre_beta}) {
        if (w.t == nullptr) continue;
        RWKV7_TRY(check_present(w, w.t->ndim));
        if (num_elements(w.t) != p.C)
            return fail(RWKV7_ERR_SHAPE_MISMATCH, "ShapeMismatch: %s is %s, expected %lld elements", w.name,
                        shape_string(w.t->shape, w.t->ndim).c_str(), (long long)p.C);
        RWKV7_TRY(check_same_dtype({x, w}));
        RWKV7_TRY(check_same_device({x, w}));
        RWKV7_TRY(check_contiguous(w));
    }
    if (kind != RWKV7_NORM_LAYER && kind != RWKV7_NORM_RMS) return fail(RWKV7_ERR_BAD_ARGUMENT, "BadArgument: norm kind %d", kind);
    if (!(epsilon >= 0.0) || !std::isfinite(epsilon))
        return fail(RWKV7_ERR_BAD_ARGUMENT, "BadArgument: epsilon must be non-negative, got %g", epsilon);
    auto data = [](const TensorInfo &i) { return i.t == nullptr ? nullptr : (const void *)i.t->data; };
    p.residual = data(x); p.block_output = data(t.block_output); p.gate = data(t.gate);
    p.residual_scale = data(t.scale); p.post_gamma = data(t.post_gamma); p.post_beta = data(t.post_beta);
    p.pre_gamma = data(t.pre_gamma); p.pre_beta = data(t.pre_beta);
    p.epsilon = (float)epsilon;
    p.layer = kind == RWKV7_NORM_LAYER;
    p.bf16 = x.t->dtype == RWKV7_BF16;
    return RWKV7_OK;
}

// An output is given if and only if its input is.
int check_paired(const TensorInfo &out, const TensorInfo &in) {
    if ((out.t == nullptr) == (in.t == nullptr)) return RWKV7_OK;
    return fail(RWKV7_ERR_NULL_POINTER, "NullPointer: %s must be given if and only if %s is", out.name, in.name);
}

}  // namespace

extern "C" {

int rwkv7_fused_residual_norm(const rwkv7_tensor *x_t, const rwkv7_tensor *h_t, const rwkv7_tensor *g_t, const rwkv7_tensor *scale_t,
                              const rwkv7_tensor *post_g_t, const rwkv7_tensor *post_b_t, const rwkv7_tensor *pre_g_t,
                              const rwkv7_tensor *pre_b_t, int32_t kind, double epsilon, rwkv7_tensor *next_t, rwkv7_tensor *normed_t,
                              rwkv7_stream stream) {
    RWKV7_TRACE("rwkv.infer.model.residual_norm");
    clear_error();
    const NormTensors t{{"residual", x_t}, {"block_output", h_t}, {"gate", g_t}, {"residual_scale", scale_t}, {"post_gamma", post_g_t},
                        {"post_beta", post_b_t}, {"pre_gamma", pre_g_t}, {"pre_beta", pre_b_t}};
    const TensorInfo next{"next_residual", next_t}, normed{"normed", normed_t};
    ResidualNormArgs p{};
    RWKV7_TRY(check_norm(t, kind, epsilon, p));
    RWKV7_TRY(check_paired(next, t.block_output));
    RWKV7_TRY(check_paired(normed, t.pre_gamma));
    for (const TensorInfo &out : {next, normed}) {
        if (out.t == nullptr) continue;
        RWKV7_TRY(check_like(t.residual, out));
        for (const TensorInfo &in : {t.residual, t.block_output, t.gate}) RWKV7_TRY(check_same_or_apart(out, in));
        for (const TensorInfo &in : {t.scale, t.post_gamma, t.post_beta, t.pre_gamma, t.pre_beta}) RWKV7_TRY(check_apart(out, in));
    }
    RWKV7_TRY(check_apart(next, normed));
    if (p.rows == 0) return RWKV7_OK;
    p.next_residual = next_t == nullptr ? nullptr : next_t->data;
    p.normed = normed_t == nullptr ? nullptr : normed_t->data;
    DeviceGuard guard(x_t->device);
    if (guard.error() != cudaSuccess) return cuda_fail("cudaSetDevice", (int)guard.error());
    RWKV7_TRY(num_sms(x_t->device, &p.num_sms));
    if (int e = launch_residual_norm(p, (cudaStream_t)stream)) return cuda_fail("residual_norm launch", e);
    return RWKV7_OK;
}

size_t rwkv7_residual_norm_backward_workspace_bytes(int64_t rows, int64_t C) {
    return rows <= 0 || C <= 0 ? 0 : residual_norm_backward_workspace_bytes(rows, C, current_sms());
}

int rwkv7_fused_residual_norm_backward(const rwkv7_tensor *x_t, const rwkv7_tensor *h_t, const rwkv7_tensor *g_t,
                                       const rwkv7_tensor *scale_t, const rwkv7_tensor *post_g_t, const rwkv7_tensor *post_b_t,
                                       const rwkv7_tensor *pre_g_t, const rwkv7_tensor *pre_b_t, int32_t kind, double epsilon,
                                       const rwkv7_tensor *dnext_t, const rwkv7_tensor *dnormed_t, rwkv7_tensor *const grads[8],
                                       void *workspace, size_t workspace_bytes, rwkv7_stream stream) {
    RWKV7_TRACE("rwkv.train.model.residual_norm");
    clear_error();
    const NormTensors t{{"residual", x_t}, {"block_output", h_t}, {"gate", g_t}, {"residual_scale", scale_t}, {"post_gamma", post_g_t},
                        {"post_beta", post_b_t}, {"pre_gamma", pre_g_t}, {"pre_beta", pre_b_t}};
    const TensorInfo inputs[10] = {t.residual, t.block_output, t.gate, t.scale, t.post_gamma, t.post_beta, t.pre_gamma, t.pre_beta,
                                   {"next_residual_grad", dnext_t}, {"normed_grad", dnormed_t}};
    static const char *const names[8] = {"residual_grad", "block_output_grad", "gate_grad", "residual_scale_grad",
                                         "post_gamma_grad", "post_beta_grad", "pre_gamma_grad", "pre_beta_grad"};
    ResidualNormBackwardArgs p{};
    RWKV7_TRY(check_norm(t, kind, epsilon, p.f));
    if (dnext_t != nullptr) RWKV7_TRY(check_like(t.residual, inputs[8]));
    RWKV7_TRY(check_paired(inputs[9], t.pre_gamma));
    if (dnormed_t != nullptr) RWKV7_TRY(check_like(t.residual, inputs[9]));
    if (grads == nullptr) return fail(RWKV7_ERR_NULL_POINTER, "NullPointer: grads array is null");
    for (int i = 0; i < 8; ++i) {
        const TensorInfo out{names[i], grads[i]};
        RWKV7_TRY(check_paired(out, inputs[i]));
        if (out.t == nullptr) continue;
        RWKV7_TRY(check_like(inputs[i], out));
        for (const TensorInfo &in : inputs) RWKV7_TRY(check_apart(out, in));
        for (int j = 0; j < i; ++j) RWKV7_TRY(check_apart(out, TensorInfo{names[j], grads[j]}));
    }
    DeviceGuard guard(x_t->device);
    if (guard.error() != cudaSuccess) return cuda_fail("cudaSetDevice", (int)guard.error());
    if (p.f.rows == 0) {   // no row: the sums are empty
        for (int i = 3; i < 8; ++i) {
            if (grads[i] == nullptr) continue;
            const cudaError_t e = cudaMemsetAsync(grads[i]->data, 0, bytes_of(grads[i]), (cudaStream_t)stream);
            if (e != cudaSuccess) return cuda_fail("residual_norm_backward", (int)e);
        }
        return RWKV7_OK;
    }
    RWKV7_TRY(num_sms(x_t->device, &p.f.num_sms));
    RWKV7_TRY(check_workspace("residual_norm_backward", workspace, workspace_bytes,
                              residual_norm_backward_workspace_bytes(p.f.rows, p.f.C, p.f.num_sms)));
    p.next_residual_grad = dnext_t == nullptr ? nullptr : dnext_t->data;
    p.normed_grad = dnormed_t == nullptr ? nullptr : dnormed_t->data;
    p.residual_grad = grads[0]->data;
    p.block_output_grad = grads[1] == nullptr ? nullptr : grads[1]->data;
    p.gate_grad = grads[2] == nullptr ? nullptr : grads[2]->data;
    for (int i = 0; i < 5; ++i) p.param_grads[i] = grads[3 + i] == nullptr ? nullptr : grads[3 + i]->data;
    if (int e = launch_residual_norm_backward(p, workspace, (cudaStream_t)stream)) return cuda_fail("residual_norm_backward launch", e);
    return RWKV7_OK;
}

// ---- beam search ------------------------------------------------------------------------------------------------------------

size_t rwkv7_beam_select_workspace_bytes(int64_t B, int64_t I, int64_t V, int64_t K) {
    if (B <= 0 || I <= 0 || V <= 0 || K <= 0 || I > 32 || K > 32) return 0;
    BeamSelectArgs p{};
    p.B = B; p.V = V; p.I = (int)I; p.K = (int)K;
    p.num_sms = current_sms();
    const size_t f32 = beam_select_workspace_bytes(p);
    p.bf16 = true;
    return std::max(f32, beam_select_workspace_bytes(p));
}

int rwkv7_beam_select(const rwkv7_tensor *logits_t, const rwkv7_tensor *scores_t, const rwkv7_tensor *finished_t, int64_t pad_token,
                      rwkv7_tensor *next_t, rwkv7_tensor *parents_t, rwkv7_tensor *tokens_t, void *workspace, size_t workspace_bytes,
                      rwkv7_stream stream) {
    RWKV7_TRACE("rwkv.infer.beam_select");
    clear_error();
    const TensorInfo logits{"logits", logits_t}, scores{"scores", scores_t}, finished{"finished", finished_t}, next{"next_scores", next_t},
        parents{"parents", parents_t}, tokens{"tokens", tokens_t};
    RWKV7_TRY(check_present(logits, 3));
    RWKV7_TRY(check_axis_non_empty(logits, 1));
    RWKV7_TRY(check_axis_non_empty(logits, 2));
    RWKV7_TRY(check_contiguous(logits));
    RWKV7_TRY(check_float(logits, "beam_select"));
    const int64_t B = logits.dim(0), I = logits.dim(1), V = logits.dim(2);
    RWKV7_TRY(check_of(logits, scores, {B, I}, RWKV7_F32));
    if (finished_t != nullptr) {
        RWKV7_TRY(check_of(logits, finished, {B, I}, RWKV7_I32));
        if (pad_token < 0 || pad_token >= V)
            return fail(RWKV7_ERR_BAD_ARGUMENT, "BadArgument: pad_token %lld is no token of %lld", (long long)pad_token, (long long)V);
    }
    RWKV7_TRY(check_present(next, 2));
    const int64_t K = next.dim(1);
    RWKV7_TRY(check_of(logits, next, {B, K}, RWKV7_F32));
    RWKV7_TRY(check_of(logits, parents, {B, K}, RWKV7_I32));
    RWKV7_TRY(check_of(logits, tokens, {B, K}, RWKV7_I32));
    if (K < 1 || K > 32 || I > 32 || V > INT32_MAX || K > I * V || B > INT32_MAX / 32 / I)
        return fail(RWKV7_ERR_UNSUPPORTED, "Unsupported: beam_select of %lld out of %lld beams of %lld tokens, %lld searches (1 to 32 of at most 32)",
                    (long long)K, (long long)I, (long long)V, (long long)B);
    const TensorInfo outs[3] = {next, parents, tokens};
    for (int i = 0; i < 3; ++i) {
        for (const TensorInfo &in : {logits, scores, finished}) RWKV7_TRY(check_apart(outs[i], in));
        for (int j = 0; j < i; ++j) RWKV7_TRY(check_apart(outs[i], outs[j]));
    }
    if (B == 0) return RWKV7_OK;
    BeamSelectArgs p{};
    p.logits = logits_t->data;
    p.scores = static_cast<const float *>(scores_t->data);
    p.finished = finished_t == nullptr ? nullptr : static_cast<const int *>(finished_t->data);
    p.next_scores = static_cast<float *>(next_t->data);
    p.parents = static_cast<int *>(parents_t->data);
    p.tokens = static_cast<int *>(tokens_t->data);
    p.B = B; p.V = V; p.pad_token = pad_token; p.I = (int)I; p.K = (int)K;
    p.bf16 = logits_t->dtype == RWKV7_BF16;
    RWKV7_TRY(check_workspace("beam_select", workspace, workspace_bytes, beam_select_min_workspace_bytes(p)));
    DeviceGuard guard(logits_t->device);
    if (guard.error() != cudaSuccess) return cuda_fail("cudaSetDevice", (int)guard.error());
    RWKV7_TRY(num_sms(logits_t->device, &p.num_sms));
    if (int e = launch_beam_select(p, workspace, workspace_bytes, (cudaStream_t)stream)) return cuda_fail("beam_select launch", e);
    return RWKV7_OK;
}

int rwkv7_beam_reorder(const rwkv7_tensor *const *states, int32_t n, const rwkv7_tensor *parents_t, rwkv7_tensor *const *out,
                       rwkv7_stream stream) {
    RWKV7_TRACE("rwkv.infer.beam_reorder");
    clear_error();
    const TensorInfo parents{"parents", parents_t};
    RWKV7_TRY(check_present(parents, 2));
    RWKV7_TRY(check_contiguous(parents));
    if (parents_t->dtype != RWKV7_I32 && parents_t->dtype != RWKV7_I64)
        return fail(RWKV7_ERR_DTYPE_MISMATCH, "DTypeMismatch: parents must be I32 or I64, got %s", dtype_name(parents_t->dtype));
    const int64_t B = parents.dim(0), K = parents.dim(1);
    if (n < 0) return fail(RWKV7_ERR_BAD_ARGUMENT, "BadArgument: %d tensors", n);
    if (n > 0 && states == nullptr) return fail(RWKV7_ERR_NULL_POINTER, "NullPointer: states array is null");
    if (K < 1 || K > 32) return fail(RWKV7_ERR_UNSUPPORTED, "Unsupported: beam_reorder to %lld beams (1 to 32)", (long long)K);
    int64_t I = out == nullptr ? K : 0;   // (otherwise what the first tensor has)
    for (int i = 0; i < n; ++i) {
        const TensorInfo s{"states", states[i]};
        if (s.t == nullptr) return fail(RWKV7_ERR_NULL_POINTER, "NullPointer: tensor descriptor states[%d] is null", i);
        if (s.t->ndim < 1 || s.t->ndim > RWKV7_MAX_DIMS)
            return fail(RWKV7_ERR_SHAPE_MISMATCH, "ShapeMismatch: states[%d] has %d axes", i, s.t->ndim);
        RWKV7_TRY(check_present(s, s.t->ndim));
        RWKV7_TRY(check_same_device({parents, s}));
        RWKV7_TRY(check_contiguous(s));
        if (I == 0 && B > 0) I = s.dim(0) / B;
        if (s.dim(0) != B * I)
            return fail(RWKV7_ERR_SHAPE_MISMATCH, "ShapeMismatch: states[%d] has %lld rows, expected %lld searches of %lld beams", i,
                        (long long)s.dim(0), (long long)B, (long long)I);
        if (out != nullptr) {
            const TensorInfo o{"out", out[i]};
            RWKV7_TRY(check_present(o, s.t->ndim));
            int64_t shape[RWKV7_MAX_DIMS];
            for (int d = 0; d < s.t->ndim; ++d) shape[d] = d == 0 ? B * K : s.dim(d);
            RWKV7_TRY(check_shape(o, shape, s.t->ndim));
            RWKV7_TRY(check_same_dtype({s, o}));
            RWKV7_TRY(check_same_device({s, o}));
            RWKV7_TRY(check_contiguous(o));
        }
    }
    // What is written stays apart from everything else; states that are only read may be the same.  (Places once a tensor: n (3 n - 1) / 2
    // pairs are compared.)
    struct Place {
        uintptr_t from, to;
        bool meets(const Place &x) const { return from < x.to && x.from < to; }
    };
    auto place = [](const rwkv7_tensor *t) {
        const uintptr_t from = reinterpret_cast<uintptr_t>(t->data);
        return Place{from, from + bytes_of(t)};
    };
    const std::unique_ptr<Place[]> places(new (std::nothrow) Place[2 * (size_t)n]);
    if (places == nullptr) return fail(RWKV7_ERR_BAD_ARGUMENT, "BadArgument: %d tensors", n);
    Place *const read = places.get(), *const written = read + n;
    for (int i = 0; i < n; ++i) {
        read[i] = place(states[i]);
        written[i] = out == nullptr ? read[i] : place(out[i]);
    }
    const char *name = out == nullptr ? "states" : "out";
    const Place chosen = place(parents_t);
    for (int i = 0; i < n; ++i) {
        const char *met = written[i].meets(chosen) ? "parents" : nullptr;
        for (int j = 0; j < i && met == nullptr; ++j)
            if (written[i].meets(written[j])) met = name;
        for (int j = 0; out != nullptr && j < n && met == nullptr; ++j)
            if (written[i].meets(read[j])) met = "states";
        if (met != nullptr) return fail(RWKV7_ERR_BAD_ARGUMENT, "BadArgument: %s and %s share memory", name, met);
    }
    if (I > 32 || (n > 0 && B > 0 && I < 1))
        return fail(RWKV7_ERR_UNSUPPORTED, "Unsupported: beam_reorder from %lld beams (1 to 32)", (long long)I);
    if (B == 0 || n == 0) return RWKV7_OK;
    BeamReorderArgs p{};
    p.parents = parents_t->data;
    p.parents_i64 = parents_t->dtype == RWKV7_I64;
    p.B = B; p.I = (int)I; p.K = (int)K;
    DeviceGuard guard(parents_t->device);
    if (guard.error() != cudaSuccess) return cuda_fail("cudaSetDevice", (int)guard.error());
    RWKV7_TRY(num_sms(parents_t->device, &p.num_sms));
    if (int e = device_status_ptr(parents_t->device, &p.status)) return cuda_fail("device status word", e);
    for (const int unit : kReorderUnits) {
        for (int i = 0; i < n; ++i) {
            const int64_t row = (int64_t)(bytes_of(states[i]) / (size_t)(B * I));
            if (row > 0 && beam_reorder_unit(row) == unit) p.tensors[p.n++] = {states[i]->data, out == nullptr ? states[i]->data : out[i]->data, row};
            if (p.n == kMaxReordered || (i == n - 1 && p.n > 0)) {
                if (int e = launch_beam_reorder(p, unit, (cudaStream_t)stream)) return cuda_fail("beam_reorder launch", e);
                p.n = 0;
            }
        }
    }
    return RWKV7_OK;
}

}  // extern "C"
