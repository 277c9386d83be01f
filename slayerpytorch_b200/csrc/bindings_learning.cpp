// Python module `slayerCuda`, second part: the losses of rows of logits (actionLogProb, policyLoss, preferenceLoss) as autograd
// functions - a step of a small network is bound by the host, and these are half as long there as their Python form - and the
// orthogonalised updates (orthogonalize, muonStep).  They take float32, bfloat16 and float16 logits, matrices and weights; everything
// that belongs to a row, and the momenta, are float32.
#include "bindings_common.h"

#include <cuda_runtime_api.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <math.h>

#include <algorithm>

using namespace sb200py;

namespace {

int dtype_code(const torch::Tensor &x, const char *name)
{
    switch (x.scalar_type()) {
    case torch::kFloat32: return SLAYER_B200_F32;
    case torch::kBFloat16: return SLAYER_B200_BF16;
    case torch::kFloat16: return SLAYER_B200_F16;
    default: TORCH_CHECK(false, name, " must be a float32, bfloat16 or float16 tensor");
    }
}

// [rows, V] with the entries of a row next to each other; any distance between rows
void check_logits(const torch::Tensor &x)
{
    TORCH_CHECK(x.is_cuda(), "logits must be a CUDA tensor");
    TORCH_CHECK(x.dim() == 2, "logits must be [rows, entries]");
    TORCH_CHECK(x.size(1) >= 1, "logits must have at least one entry per row");
    TORCH_CHECK(x.size(1) == 1 || x.stride(1) == 1, "the entries of a row of logits must be next to each other");
    dtype_code(x, "logits");
}

void check_rows(const torch::Tensor &v, const char *name, torch::ScalarType dtype, int64_t count, const torch::Tensor &like)
{
    TORCH_CHECK(v.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(v.is_contiguous(), name, " must be contiguous");
    TORCH_CHECK(v.scalar_type() == dtype, name, " has the wrong dtype (", v.scalar_type(), ")");
    TORCH_CHECK(v.numel() == count, name, " must have ", count, " entries, it has ", v.numel());
    check_device(v, like, name, "logits");
}

template <typename T>
T *or_null(const c10::optional<torch::Tensor> &x) { return x.has_value() ? x->data_ptr<T>() : nullptr; }

const uint8_t *mask_of(const c10::optional<torch::Tensor> &mask, int64_t rows, const torch::Tensor &like)
{
    if (!mask.has_value()) return nullptr;
    check_rows(*mask, "mask", torch::kBool, rows, like);
    return reinterpret_cast<const uint8_t *>(mask->data_ptr<bool>());
}

// Which stream capture the current stream of a tensor's device is in; 0: none.
int64_t capture_id(torch::Tensor like)
{
    TORCH_CHECK(like.is_cuda(), "captureId takes a CUDA tensor");
    c10::cuda::CUDAGuard guard(like.device());
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (cudaStreamGetCaptureInfo((cudaStream_t)current_stream(), &status, &id) != cudaSuccess) return -1;
    return status == cudaStreamCaptureStatusActive ? (int64_t)id : 0;
}

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

// ---- arguments: logits [..., V], what belongs to a row of the shape in front of V
void check_logits_shape(const torch::Tensor &logits, const torch::Tensor &action, const c10::optional<torch::Tensor> &mask, double scale, const char *op)
{
    TORCH_CHECK_VALUE(logits.dim() >= 1 && action.sizes() == logits.sizes().slice(0, logits.dim() - 1), op,
                      ": action must have the shape of logits without its last dimension, got ", action.sizes(), " for ", logits.sizes());
    TORCH_CHECK_TYPE(action.scalar_type() == torch::kInt64 || action.scalar_type() == torch::kInt32, op, ": action must be int64 or int32, got ",
                     action.scalar_type());
    TORCH_CHECK_VALUE(!mask.has_value() || mask->sizes() == action.sizes(), op, ": mask must have the shape of action");
    TORCH_CHECK_VALUE(logits.size(-1) >= 1, op, ": logits must have at least one entry per row");
    TORCH_CHECK_VALUE(scale > 0.0 && scale < INFINITY, op, ": scale must be positive and finite, got ", scale);
}

// constants: no gradient flows into them
torch::Tensor flat(const torch::Tensor &x, torch::ScalarType dtype) { return x.detach().to(dtype).reshape({-1}).contiguous(); }

torch::Tensor per_row(const torch::Tensor &x, at::IntArrayRef shape, const char *what)
{
    TORCH_CHECK_VALUE(x.sizes() == shape, what, " must have the shape ", shape, ", got ", x.sizes());
    return flat(x, torch::kFloat32);
}

c10::optional<torch::Tensor> flat_mask(const c10::optional<torch::Tensor> &mask)
{
    if (!mask.has_value()) return c10::nullopt;
    return (mask->scalar_type() == torch::kBool ? *mask : mask->ne(0)).reshape({-1}).contiguous();
}

// the rows of logits, a view where there is one
torch::Tensor rows_of(const torch::Tensor &logits)
{
    const int64_t V = logits.size(-1);
    auto rows = logits.reshape({logits.numel() / V, V});
    if (V > 1 && rows.size(0) > 0 && rows.stride(1) != 1) rows = rows.contiguous();
    check_logits(rows);
    return rows;
}

// What the backward passes need, in one buffer: stats (two floats a row) and coef, and behind them what the forward pass works with.
struct RowBuffer {
    torch::Tensor all;
    float *stats, *coef;
    void *workspace;
    RowBuffer(const torch::Tensor &like, int64_t rows, int64_t coefs, int64_t workspace_bytes)
        : RowBuffer(torch::empty({2 + 2 * rows + coefs + (workspace_bytes + 3) / 4}, like.options().dtype(torch::kFloat32)), rows, coefs)
    {
    }
    RowBuffer(torch::Tensor buffer, int64_t rows, int64_t coefs) : all(std::move(buffer))
    {
        const int64_t even = (2 * rows + coefs + 1) / 2 * 2;       // the workspace is aligned to 8 bytes
        stats = all.data_ptr<float>();
        coef = stats + 2 * rows;
        workspace = stats + even;
    }
};

torch::Tensor logit_grad(const torch::Tensor &logits, const torch::Tensor &action, const torch::Tensor &mask, const float *stats, const float *coef,
                         int64_t coef_len, const torch::Tensor &up, double scale, const torch::Tensor *into, const char *op)
{
    const auto x = rows_of(logits);
    const int64_t rows = x.size(0), V = x.size(1);
    c10::cuda::CUDAGuard guard(x.device());
    auto grad = into ? *into : torch::empty({rows, V}, x.options());
    const bool by_row = up.dim() > 0;
    const auto upstream = up.to(torch::kFloat32).contiguous();
    if (rows > 0)
        check_rc(slayer_b200_logit_grad(grad.data_ptr(), x.data_ptr(), dtype_code(x, "logits"), action.data_ptr<int64_t>(),
                                        mask.defined() ? reinterpret_cast<const uint8_t *>(mask.data_ptr<bool>()) : nullptr, stats, coef, coef_len,
                                        upstream.data_ptr<float>(), by_row, into != nullptr, rows, V, x.stride(0), (float)scale, current_stream()),
                 op);
    grad = grad.view(logits.sizes());
    if (!at::GradMode::is_enabled()) return grad;
    // create_graph: the gradient can be had, its derivative cannot (and must not read as zero)
    grad = grad.detach().set_requires_grad(true);
    return (*std::make_shared<torch::autograd::DelayedError>(std::string(op) + ": has first derivatives only", 1))({grad})[0];
}

// Forward reads the logits once and keeps two floats per row; backward reads them again and writes their gradient.
struct ActionLogProb : public torch::autograd::Function<ActionLogProb> {
    static torch::Tensor forward(AutogradContext *ctx, const torch::Tensor &logits, const torch::Tensor &action,
                                 const c10::optional<torch::Tensor> &mask, double scale)
    {
        const auto x = rows_of(logits);
        const int64_t rows = x.size(0);
        const auto act = flat(action, torch::kInt64);
        const auto keep = flat_mask(mask);
        check_rows(act, "action", torch::kInt64, rows, x);
        const uint8_t *m = mask_of(keep, rows, x);
        c10::cuda::CUDAGuard guard(x.device());
        auto logp = torch::empty(action.sizes(), x.options().dtype(torch::kFloat32));
        auto stats = torch::empty({2 * rows}, logp.options());
        check_rc(slayer_b200_log_prob(logp.data_ptr<float>(), stats.data_ptr<float>(), x.data_ptr(), dtype_code(x, "logits"), act.data_ptr<int64_t>(), m,
                                      rows, x.size(1), x.stride(0), (float)scale, current_stream()),
                 "actionLogProb");
        ctx->save_for_backward({logits, act, keep.value_or(torch::Tensor()), stats});
        ctx->saved_data["scale"] = scale;
        return logp;
    }
    static variable_list backward(AutogradContext *ctx, variable_list up)
    {
        const auto v = ctx->get_saved_variables();
        const double scale = ctx->saved_data["scale"].toDouble();
        torch::Tensor by_row = up[0];
        if (by_row.dim() == 0) by_row = by_row.reshape({1});
        return {logit_grad(v[0], v[1], v[2], v[3].data_ptr<float>(), nullptr, 1, by_row, scale, nullptr, "actionLogProb"), Variable(), Variable(),
                Variable()};
    }
};

// Value and gradient from one pass over the logits.  The gradient for an upstream gradient of one is written in the forward pass
// and handed over by the first backward, which checks on the device whether the upstream gradient is one and forms the
// gradient anew if not (rounding it once); later backward passes form it anew.  Half-precision logits get theirs in the
// backward pass alone: their losses are scaled up before it, and unscaled gradients would be lost below 6e-8.
struct PolicyLoss : public torch::autograd::Function<PolicyLoss> {
    static variable_list forward(AutogradContext *ctx, const torch::Tensor &logits, const torch::Tensor &action, const torch::Tensor &old,
                                 const torch::Tensor &advantage, const c10::optional<torch::Tensor> &ref, const c10::optional<torch::Tensor> &mask,
                                 int64_t seqLen, double scale, double low, double high, double kl, int64_t reduction, bool want)
    {
        const auto x = rows_of(logits);
        const int64_t rows = x.size(0), V = x.size(1);
        const auto act = flat(action, torch::kInt64);
        const auto keep = flat_mask(mask);
        check_rows(act, "action", torch::kInt64, rows, x);
        check_rows(old, "oldLogProb", torch::kFloat32, rows, x);
        if (ref.has_value()) check_rows(*ref, "refLogProb", torch::kFloat32, rows, x);
        const uint8_t *m = mask_of(keep, rows, x);
        const int64_t advLen = rows == 0 || advantage.numel() == rows ? 1 : seqLen;
        check_rows(advantage, "advantage", torch::kFloat32, rows == 0 ? advantage.numel() : rows / advLen, x);   // its shape has been checked
        c10::cuda::CUDAGuard guard(x.device());
        auto loss = torch::empty({}, x.options().dtype(torch::kFloat32));
        auto logp = torch::empty(action.sizes(), loss.options());       // the caller's own: nothing here reads it again
        RowBuffer buffer(x, rows, rows, slayer_b200_policy_loss_workspace(rows, seqLen));
        const bool early = want && x.scalar_type() != torch::kFloat16;
        torch::Tensor grad;
        if (early) grad = torch::empty({rows, V}, x.options());
        check_rc(slayer_b200_policy_loss(loss.data_ptr<float>(), early ? grad.data_ptr() : nullptr, logp.data_ptr<float>(), buffer.stats, buffer.coef,
                                         buffer.workspace, x.data_ptr(), dtype_code(x, "logits"), act.data_ptr<int64_t>(), old.data_ptr<float>(),
                                         advantage.data_ptr<float>(), advLen, or_null<float>(ref), m, rows, seqLen, V, x.stride(0), (float)scale,
                                         (float)low, (float)high, (float)kl, (int)reduction, current_stream()),
                 "policyLoss");
        if (want) {
            ctx->save_for_backward({logits, act, keep.value_or(torch::Tensor()), buffer.all});
            ctx->saved_data["scale"] = scale;
            if (early) {
                ctx->saved_data["early"] = grad;
                ctx->saved_data["capture"] = capture_id(x);
            }
        }
        ctx->mark_non_differentiable({logp});
        return {loss, logp};
    }
    static variable_list backward(AutogradContext *ctx, variable_list up)
    {
        const auto v = ctx->get_saved_variables();
        const int64_t rows = v[1].numel();
        const RowBuffer buffer(v[3], rows, rows);
        torch::Tensor early;
        const auto it = ctx->saved_data.find("early");
        if (it != ctx->saved_data.end()) {
            early = it->second.toTensor();
            ctx->saved_data.erase(it);
            // replayed without its forward pass, a captured backward pass would hand over a buffer that is the user's by then
            if (capture_id(v[0]) != ctx->saved_data["capture"].toInt()) early = torch::Tensor();
        }
        variable_list out(13);
        out[0] = logit_grad(v[0], v[1], v[2], buffer.stats, buffer.coef, 1, up[0], ctx->saved_data["scale"].toDouble(), early.defined() ? &early : nullptr,
                            "policyLoss");
        return out;
    }
};

// The pairs' coefficients need every sequence's sum: the logits are read for those, and again where the gradient is written.
struct PreferenceLoss : public torch::autograd::Function<PreferenceLoss> {
    static torch::Tensor forward(AutogradContext *ctx, const torch::Tensor &logits, const torch::Tensor &action, const torch::Tensor &ref,
                                 const torch::Tensor &pairs, const c10::optional<torch::Tensor> &mask, double beta, double smoothing, double scale,
                                 int64_t reduction)
    {
        const auto x = rows_of(logits);
        const int64_t rows = x.size(0), S = logits.size(0), L = logits.size(1);
        const auto act = flat(action, torch::kInt64);
        const auto keep = flat_mask(mask);
        check_rows(act, "action", torch::kInt64, rows, x);
        check_rows(ref, "refLogProb", torch::kFloat32, S, x);
        check_rows(pairs, "pairs", torch::kInt64, pairs.numel(), x);
        const uint8_t *m = mask_of(keep, rows, x);
        c10::cuda::CUDAGuard guard(x.device());
        auto loss = torch::empty({}, x.options().dtype(torch::kFloat32));
        const int64_t bytes = slayer_b200_preference_loss_workspace(S);
        RowBuffer buffer(x, rows, S, bytes + 4 * rows);
        float *logp = (float *)((char *)buffer.workspace + bytes);
        check_rc(slayer_b200_log_prob(logp, buffer.stats, x.data_ptr(), dtype_code(x, "logits"), act.data_ptr<int64_t>(), m, rows, x.size(1),
                                      x.stride(0), (float)scale, current_stream()),
                 "preferenceLoss");
        check_rc(slayer_b200_preference_loss(loss.data_ptr<float>(), buffer.coef, buffer.workspace, logp, ref.data_ptr<float>(),
                                             pairs.data_ptr<int64_t>(), S, L, pairs.size(0), (float)beta, (float)smoothing, (int)reduction,
                                             current_stream()),
                 "preferenceLoss");
        ctx->save_for_backward({logits, act, keep.value_or(torch::Tensor()), buffer.all});
        ctx->saved_data["scale"] = scale;
        return loss;
    }
    static variable_list backward(AutogradContext *ctx, variable_list up)
    {
        const auto v = ctx->get_saved_variables();
        const int64_t rows = v[1].numel(), S = v[0].size(0), L = v[0].size(1);
        const RowBuffer buffer(v[3], rows, S);
        variable_list out(9);
        out[0] = logit_grad(v[0], v[1], v[2], buffer.stats, buffer.coef, L > 0 ? L : 1, up[0], ctx->saved_data["scale"].toDouble(), nullptr,
                            "preferenceLoss");
        return out;
    }
};

torch::Tensor actionLogProbCuda(const torch::Tensor &logits, const torch::Tensor &action, const c10::optional<torch::Tensor> &mask, double scale)
{
    check_logits_shape(logits, action, mask, scale, "actionLogProb");
    return ActionLogProb::apply(logits, action, mask, scale);
}

// (loss, the rows' log-probabilities)
std::vector<torch::Tensor> policyLossCuda(const torch::Tensor &logits, const torch::Tensor &action, const torch::Tensor &oldLogProb,
                                          const torch::Tensor &advantage, const c10::optional<torch::Tensor> &refLogProb,
                                          const c10::optional<torch::Tensor> &mask, double clipLow, double clipHigh, double klCoef, double scale,
                                          int64_t reduction)
{
    check_logits_shape(logits, action, mask, scale, "policyLoss");
    const auto shape = action.sizes();
    TORCH_CHECK_VALUE(reduction != SLAYER_B200_SEQUENCE || !shape.empty(), "policyLoss: reduction 'sequence' needs a dimension of choices");
    const auto old = per_row(oldLogProb, shape, "policyLoss: oldLogProb");
    c10::optional<torch::Tensor> ref;
    if (refLogProb.has_value()) ref = per_row(*refLogProb, shape, "policyLoss: refLogProb");
    const bool by_sequence = !shape.empty() && advantage.sizes() != shape && advantage.sizes() == shape.slice(0, shape.size() - 1);
    const auto adv = per_row(advantage, by_sequence ? shape.slice(0, shape.size() - 1) : shape, "policyLoss: advantage");
    const int64_t seqLen = shape.empty() ? 1 : std::max<int64_t>(1, shape.back());
    const bool want = at::GradMode::is_enabled() && logits.requires_grad();
    return PolicyLoss::apply(logits, action, old, adv, ref, mask, seqLen, scale, clipLow, clipHigh, klCoef, reduction, want);
}

torch::Tensor preferenceLossCuda(const torch::Tensor &logits, const torch::Tensor &action, const torch::Tensor &refLogProb,
                                 const c10::optional<torch::Tensor> &pairs, const c10::optional<torch::Tensor> &mask, double beta, double smoothing,
                                 double scale, int64_t reduction)
{
    TORCH_CHECK_VALUE(logits.dim() == 3, "preferenceLoss: logits must be [sequences, choices, entries], got ", logits.sizes());
    check_logits_shape(logits, action, mask, scale, "preferenceLoss");
    const int64_t S = logits.size(0);
    const auto ref = per_row(refLogProb, {S}, "preferenceLoss: refLogProb");
    torch::Tensor pair;
    if (pairs.has_value()) {
        TORCH_CHECK_VALUE(pairs->dim() == 2 && pairs->size(1) == 2 && (pairs->scalar_type() == torch::kInt64 || pairs->scalar_type() == torch::kInt32),
                          "preferenceLoss: pairs must be [P, 2] integers, got ", pairs->sizes(), " ", pairs->scalar_type());
        pair = pairs->to(torch::kInt64).contiguous();
    } else {
        TORCH_CHECK_VALUE(S % 2 == 0, "preferenceLoss: without pairs the number of sequences must be even, got ", S);
        const auto first = torch::arange(S / 2, logits.options().dtype(torch::kInt64));
        pair = torch::stack({first, first + S / 2}, 1);
    }
    return PreferenceLoss::apply(logits, action, ref, pair, mask, beta, smoothing, scale, reduction);
}

void check_matrix(const torch::Tensor &x, const char *name)
{
    TORCH_CHECK(x.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(x.is_contiguous(), name, " must be contiguous");
    TORCH_CHECK(x.dim() >= 2, name, " must have at least two dimensions, it has ", x.dim());
}

// bytes that are not a negative code
int64_t size_of(int64_t bytes, const char *op)
{
    if (bytes < 0) check_rc((int)bytes, op);
    return bytes;
}

// A matrix, or a stack of them, made near orthogonal.
torch::Tensor orthogonalizeCuda(torch::Tensor x, int64_t steps, double a, double b, double c, double eps)
{
    check_matrix(x, "matrix");
    const int dtype = dtype_code(x, "matrix");
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t rows = x.size(-2), cols = x.size(-1), batch = x.numel() ? x.numel() / (rows * cols) : 0;
    auto workspace = torch::empty({size_of(slayer_b200_orthogonalize_workspace(batch, rows, cols, dtype), "orthogonalize")}, x.options().dtype(torch::kUInt8));
    auto out = torch::empty_like(x);
    check_rc(slayer_b200_orthogonalize(out.data_ptr(), x.data_ptr(), dtype, batch, rows, cols, (int)std::clamp<int64_t>(steps, 0, 1 << 20),
                                       (float)a, (float)b, (float)c, (float)eps, workspace.data_ptr(), current_stream()),
             "orthogonalize");
    return out;
}

// One optimiser step, in place: [d0, d1, ...] is a matrix of d0 rows.  Weights of one type on one device are worked on together; whatever
// can be refused is, before the first of them changes.
void muonStepCuda(std::vector<torch::Tensor> weights, const std::vector<torch::Tensor> &grads, std::vector<torch::Tensor> momenta, double lr,
                  double momentum, bool nesterov, double weightDecay, int64_t adjust, int64_t steps, double a, double b, double c, double eps)
{
    TORCH_CHECK(weights.size() == grads.size() && weights.size() == momenta.size(), "as many gradients and momenta as weights");
    struct Group {
        torch::Tensor first, workspace;
        int dtype;
        std::vector<slayer_b200_muon_matrix> list;
    };
    std::vector<Group> groups;
    for (size_t i = 0; i < weights.size(); ++i) {
        const torch::Tensor &w = weights[i], &g = grads[i], &m = momenta[i];
        check_matrix(w, "weight");
        check_matrix(g, "grad");
        check_matrix(m, "momentum");
        const int dtype = dtype_code(w, "weight");
        TORCH_CHECK(g.scalar_type() == w.scalar_type(), "grad must have the dtype of its weight");
        TORCH_CHECK(m.scalar_type() == torch::kFloat32, "momentum must be a float32 tensor");
        TORCH_CHECK(g.sizes() == w.sizes() && m.sizes() == w.sizes(), "grad and momentum must have the shape of their weight");
        check_device(g, w, "grad", "weight");
        check_device(m, w, "momentum", "weight");
        TORCH_CHECK(c10::InferenceMode::is_enabled() || !(w.is_inference() || m.is_inference()),
                    "weights and momenta made in inference mode are updated in it only");
        const int64_t rows = w.size(0);
        size_t at = 0;
        while (at < groups.size() && !(groups[at].dtype == dtype && groups[at].first.device() == w.device())) ++at;
        if (at == groups.size()) groups.push_back({w, torch::Tensor(), dtype, {}});
        groups[at].list.push_back({w.data_ptr(), g.data_ptr(), m.data_ptr<float>(), rows, w.numel() ? w.numel() / rows : 0});
    }
    for (Group &k : groups) {
        c10::cuda::CUDAGuard guard(k.first.device());
        k.workspace = torch::empty({size_of(slayer_b200_muon_step_workspace(k.list.data(), (int64_t)k.list.size(), k.dtype), "muonStep")},
                                   k.first.options().dtype(torch::kUInt8));
    }
    for (Group &k : groups) {
        c10::cuda::CUDAGuard guard(k.first.device());
        check_rc(slayer_b200_muon_step(k.list.data(), (int64_t)k.list.size(), k.dtype, (float)lr, (float)momentum, nesterov, (float)weightDecay,
                                       (int)adjust, (int)std::clamp<int64_t>(steps, 0, 1 << 20), (float)a, (float)b, (float)c, (float)eps,
                                       k.workspace.data_ptr(), current_stream()),
                 "muonStep");
    }
    for (auto &w : weights) w.unsafeGetTensorImpl()->bump_version();      // autograd sees that they changed
    for (auto &m : momenta) m.unsafeGetTensorImpl()->bump_version();
}

}  // namespace

void bind_learning(pybind11::module_ &m)
{
    m.def("actionLogProb", &actionLogProbCuda, "Log-probability of the chosen entry of each row of logits, differentiable (CUDA)");
    m.def("policyLoss", &policyLossCuda, "Clipped policy loss with a KL term, value and gradient in one pass, differentiable (CUDA)");
    m.def("preferenceLoss", &preferenceLossCuda, "Loss of paired sequences of choices, differentiable (CUDA)");
    m.def("orthogonalize", &orthogonalizeCuda, "Matrices made near orthogonal by Newton-Schulz products (CUDA)");
    m.def("muonStep", &muonStepCuda, "Momentum, orthogonalised update and decay of a list of weights, in place (CUDA)");
}
