// Python module `slayerCuda`, second part: the operators behind the losses on logits (logProb, policyLoss, preferenceLoss,
// logitGrad), and the orthogonalised updates (orthogonalize, muonStep).  They take float32, bfloat16 and float16 logits, matrices
// and weights; everything that belongs to a row, and the momenta, are float32.
#include "bindings_common.h"

#include <cuda_runtime_api.h>

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

// (logp [rows], stats [rows, 2])
std::vector<torch::Tensor> logProbCuda(torch::Tensor logits, torch::Tensor action, c10::optional<torch::Tensor> mask, float scale)
{
    check_logits(logits);
    const int64_t rows = logits.size(0);
    check_rows(action, "action", torch::kInt64, rows, logits);
    const uint8_t *m = mask_of(mask, rows, logits);
    c10::cuda::CUDAGuard guard(logits.device());
    auto logp = torch::empty({rows}, logits.options().dtype(torch::kFloat32));
    auto stats = torch::empty({rows, 2}, logp.options());
    check_rc(slayer_b200_log_prob(logp.data_ptr<float>(), stats.data_ptr<float>(), logits.data_ptr(), dtype_code(logits, "logits"),
                                  action.data_ptr<int64_t>(), m, rows, logits.size(1), logits.stride(0), scale, current_stream()),
             "logProb");
    return {logp, stats};
}

// d / d logits of sum_r upstream * coef[r / coefLen] * logp[r].  into: a buffer that holds the gradient for an upstream of one
// already, which is kept if upstream is one.
torch::Tensor logitGradCuda(torch::Tensor logits, torch::Tensor action, c10::optional<torch::Tensor> mask, torch::Tensor stats,
                            c10::optional<torch::Tensor> coef, int64_t coefLen, torch::Tensor upstream, float scale,
                            c10::optional<torch::Tensor> into)
{
    check_logits(logits);
    const int64_t rows = logits.size(0), V = logits.size(1);
    check_rows(action, "action", torch::kInt64, rows, logits);
    const uint8_t *m = mask_of(mask, rows, logits);
    check_rows(stats, "stats", torch::kFloat32, 2 * rows, logits);
    TORCH_CHECK(coefLen >= 1 && rows % coefLen == 0, "coefLen must divide the rows");
    if (coef.has_value() && rows > 0) check_rows(*coef, "coef", torch::kFloat32, rows / coefLen, logits);
    const bool by_row = upstream.dim() > 0;
    check_rows(upstream, "upstream", torch::kFloat32, by_row ? rows : 1, logits);
    c10::cuda::CUDAGuard guard(logits.device());
    if (rows == 0) return torch::empty({0, V}, logits.options());
    torch::Tensor grad;
    if (into.has_value()) {
        grad = *into;
        check_rows(grad, "into", logits.scalar_type(), rows * V, logits);
        TORCH_CHECK(!by_row, "a gradient that is there already needs one upstream value");
    } else {
        grad = torch::empty({rows, V}, logits.options());
    }
    check_rc(slayer_b200_logit_grad(grad.data_ptr(), logits.data_ptr(), dtype_code(logits, "logits"), action.data_ptr<int64_t>(), m,
                                    stats.data_ptr<float>(), or_null<float>(coef), coefLen, upstream.data_ptr<float>(), by_row,
                                    into.has_value(), rows, V, logits.stride(0), scale, current_stream()),
             "logitGrad");
    return grad;
}

// (loss [], logp [rows], stats [rows, 2], coef [rows], gradient [rows, V] or an empty tensor)
std::vector<torch::Tensor> policyLossCuda(torch::Tensor logits, torch::Tensor action, torch::Tensor oldLogProb, torch::Tensor advantage,
                                          c10::optional<torch::Tensor> refLogProb, c10::optional<torch::Tensor> mask, int64_t seqLen,
                                          float scale, float clipLow, float clipHigh, float klCoef, int64_t reduction, bool wantGrad)
{
    check_logits(logits);
    const int64_t rows = logits.size(0), V = logits.size(1);
    check_rows(action, "action", torch::kInt64, rows, logits);
    check_rows(oldLogProb, "oldLogProb", torch::kFloat32, rows, logits);
    if (refLogProb.has_value()) check_rows(*refLogProb, "refLogProb", torch::kFloat32, rows, logits);
    const uint8_t *m = mask_of(mask, rows, logits);
    TORCH_CHECK(seqLen >= 1 && rows % seqLen == 0, "the rows must be whole sequences");
    const int64_t advLen = advantage.numel() == rows ? 1 : seqLen;
    check_rows(advantage, "advantage", torch::kFloat32, rows / advLen, logits);
    c10::cuda::CUDAGuard guard(logits.device());
    auto f32 = logits.options().dtype(torch::kFloat32);
    auto loss = torch::empty({}, f32);
    auto logp = torch::empty({rows}, f32), stats = torch::empty({rows, 2}, f32), coef = torch::empty({rows}, f32);
    auto grad = wantGrad ? torch::empty({rows, V}, logits.options()) : torch::empty({0}, logits.options());
    auto workspace = torch::empty({slayer_b200_policy_loss_workspace(rows, seqLen)}, logits.options().dtype(torch::kUInt8));
    check_rc(slayer_b200_policy_loss(loss.data_ptr<float>(), wantGrad ? grad.data_ptr() : nullptr, logp.data_ptr<float>(),
                                     stats.data_ptr<float>(), coef.data_ptr<float>(), workspace.data_ptr(), logits.data_ptr(),
                                     dtype_code(logits, "logits"), action.data_ptr<int64_t>(), oldLogProb.data_ptr<float>(),
                                     advantage.data_ptr<float>(), advLen, or_null<float>(refLogProb), m, rows, seqLen, V,
                                     logits.stride(0), scale, clipLow, clipHigh, klCoef, (int)reduction, current_stream()),
             "policyLoss");
    return {loss, logp, stats, coef, grad};
}

// (loss [], coef [sequences])
std::vector<torch::Tensor> preferenceLossCuda(torch::Tensor logp, torch::Tensor refLogProb, torch::Tensor pairs, int64_t sequences,
                                              float beta, float smoothing, int64_t reduction)
{
    TORCH_CHECK(logp.is_cuda() && logp.is_contiguous() && logp.scalar_type() == torch::kFloat32, "logp must be a contiguous float32 CUDA tensor");
    TORCH_CHECK(sequences >= 0 && (sequences ? logp.numel() % sequences == 0 : logp.numel() == 0), "logp must hold whole sequences");
    check_rows(refLogProb, "refLogProb", torch::kFloat32, sequences, logp);
    TORCH_CHECK(pairs.dim() == 2 && pairs.size(1) == 2, "pairs must be [pairs, 2]");
    check_rows(pairs, "pairs", torch::kInt64, pairs.numel(), logp);
    c10::cuda::CUDAGuard guard(logp.device());
    auto loss = torch::empty({}, logp.options());
    auto coef = torch::empty({sequences}, logp.options());
    auto workspace = torch::empty({slayer_b200_preference_loss_workspace(sequences)}, logp.options().dtype(torch::kUInt8));
    check_rc(slayer_b200_preference_loss(loss.data_ptr<float>(), coef.data_ptr<float>(), workspace.data_ptr(), logp.data_ptr<float>(),
                                         refLogProb.data_ptr<float>(), pairs.data_ptr<int64_t>(), sequences,
                                         sequences ? logp.numel() / sequences : 0, pairs.size(0), beta, smoothing, (int)reduction,
                                         current_stream()),
             "preferenceLoss");
    return {loss, coef};
}

void check_matrix(const torch::Tensor &x, const char *name)
{
    TORCH_CHECK(x.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(x.is_contiguous(), name, " must be contiguous");
    TORCH_CHECK(x.dim() >= 2, name, " must have at least two dimensions, it has ", x.dim());
}

// A matrix, or a stack of them, made near orthogonal.
torch::Tensor orthogonalizeCuda(torch::Tensor x, int64_t steps, double a, double b, double c, double eps)
{
    check_matrix(x, "matrix");
    const int dtype = dtype_code(x, "matrix");
    c10::cuda::CUDAGuard guard(x.device());
    auto out = torch::empty_like(x);
    const int64_t rows = x.size(-2), cols = x.size(-1), batch = x.numel() ? x.numel() / (rows * cols) : 0;
    auto workspace = torch::empty({slayer_b200_orthogonalize_workspace(batch, rows, cols, dtype)}, x.options().dtype(torch::kUInt8));
    check_rc(slayer_b200_orthogonalize(out.data_ptr(), x.data_ptr(), dtype, batch, rows, cols, (int)std::min<int64_t>(steps, 1 << 20),
                                       (float)a, (float)b, (float)c, (float)eps, workspace.data_ptr(), current_stream()),
             "orthogonalize");
    return out;
}

// One optimiser step, in place, of weights of one type on one device: [d0, d1, ...] is a matrix of d0 rows.
void muonStepCuda(std::vector<torch::Tensor> weights, const std::vector<torch::Tensor> &grads, std::vector<torch::Tensor> momenta, double lr,
                  double momentum, bool nesterov, double weightDecay, int64_t adjust, int64_t steps, double a, double b, double c, double eps)
{
    TORCH_CHECK(weights.size() == grads.size() && weights.size() == momenta.size(), "as many gradients and momenta as weights");
    if (weights.empty()) return;
    const int dtype = dtype_code(weights[0], "weight");
    std::vector<slayer_b200_muon_matrix> list;
    list.reserve(weights.size());
    for (size_t i = 0; i < weights.size(); ++i) {
        const torch::Tensor &w = weights[i], &g = grads[i], &m = momenta[i];
        check_matrix(w, "weight");
        check_matrix(g, "grad");
        check_matrix(m, "momentum");
        TORCH_CHECK(w.scalar_type() == weights[0].scalar_type(), "the weights of one call must have one dtype");
        TORCH_CHECK(g.scalar_type() == w.scalar_type(), "grad must have the dtype of its weight");
        TORCH_CHECK(m.scalar_type() == torch::kFloat32, "momentum must be a float32 tensor");
        TORCH_CHECK(g.sizes() == w.sizes() && m.sizes() == w.sizes(), "grad and momentum must have the shape of their weight");
        check_device(w, weights[0], "weight", "the first weight");
        check_device(g, w, "grad", "weight");
        check_device(m, w, "momentum", "weight");
        const int64_t rows = w.size(0);
        list.push_back({w.data_ptr(), g.data_ptr(), m.data_ptr<float>(), rows, w.numel() ? w.numel() / rows : 0});
    }
    c10::cuda::CUDAGuard guard(weights[0].device());
    auto workspace = torch::empty({slayer_b200_muon_step_workspace(list.data(), (int64_t)list.size(), dtype)},
                                  weights[0].options().dtype(torch::kUInt8));
    check_rc(slayer_b200_muon_step(list.data(), (int64_t)list.size(), dtype, (float)lr, (float)momentum, nesterov, (float)weightDecay,
                                   (int)adjust, (int)std::min<int64_t>(steps, 1 << 20), (float)a, (float)b, (float)c, (float)eps,
                                   workspace.data_ptr(), current_stream()),
             "muonStep");
    for (auto &w : weights) w.unsafeGetTensorImpl()->bump_version();      // autograd sees that they changed
    for (auto &m : momenta) m.unsafeGetTensorImpl()->bump_version();
}

}  // namespace

void bind_learning(pybind11::module_ &m)
{
    m.def("logProb", &logProbCuda, "Log-probability of the chosen entry of each row of logits (CUDA)");
    m.def("logitGrad", &logitGradCuda, "Gradient of rows' log-probabilities with respect to the logits (CUDA)");
    m.def("policyLoss", &policyLossCuda, "Clipped policy loss with a KL term: value and gradient in one pass (CUDA)");
    m.def("preferenceLoss", &preferenceLossCuda, "Loss of paired sequences and its derivative by each sequence's log-probability (CUDA)");
    m.def("orthogonalize", &orthogonalizeCuda, "Matrices made near orthogonal by Newton-Schulz products (CUDA)");
    m.def("muonStep", &muonStepCuda, "Momentum, orthogonalised update and decay of a list of weights, in place (CUDA)");
    m.def("captureId", &capture_id, "Which stream capture the current stream of a tensor's device is in (0: none)");
}
