// Python module `slayerCuda`, third part: the gated leaky integrator (gatedLeak, an autograd function in C++ as the losses of choices are;
// gatedLeakStep), and tensors kept in 8 bits (compress8, restore8, spikeGrad8, weightGrad8).  Rows are all dimensions but the last,
// which is time.
#include "bindings_common.h"

#include <torch/csrc/autograd/functions/basic_ops.h>

#include <numeric>

using namespace sb200py;

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

int dtype_code(const torch::Tensor &x, const char *name)
{
    switch (x.scalar_type()) {
    case torch::kFloat32: return SLAYER_B200_F32;
    case torch::kBFloat16: return SLAYER_B200_BF16;
    case torch::kFloat16: return SLAYER_B200_F16;
    default: TORCH_CHECK(false, name, " must be a float32, bfloat16 or float16 tensor");
    }
}

int64_t size_of(int64_t bytes, const char *op)
{
    if (bytes < 0) check_rc((int)bytes, op);
    return bytes;
}

int64_t product(at::IntArrayRef sizes, int64_t from, int64_t to)
{
    return std::accumulate(sizes.begin() + from, sizes.begin() + to, (int64_t)1, std::multiplies<int64_t>());
}

// itself, or a copy where it does not begin at 16 bytes
torch::Tensor aligned(const torch::Tensor &x) { return (uintptr_t)x.data_ptr() % 16 ? x.clone() : x; }

// A gate that is broadcast to x, as the kernels take it: a value per step (period 0), or one for each group of rows at all steps.
struct Gate {
    torch::Tensor values;
    int64_t inner = 1, period = 0;
};

Gate gate_of(const torch::Tensor &gate, const torch::Tensor &x, const char *op)
{
    const int64_t d = x.dim(), lead = d - gate.dim();
    bool fits = lead >= 0, full = lead == 0;
    for (int64_t i = 0; i < d && fits; ++i) {
        const int64_t n = i < lead ? 1 : gate.size(i - lead);
        fits = n == 1 || n == x.size(i);
        full = full && n == x.size(i);
    }
    TORCH_CHECK_VALUE(fits, op, ": gate ", gate.sizes(), " does not broadcast to x ", x.sizes());
    const auto steps = [&](const torch::Tensor &g) {
        TORCH_CHECK_TYPE(g.scalar_type() == x.scalar_type(), op, ": a gate for every step must have the type of x (", x.scalar_type(), "), got ",
                         g.scalar_type());
        return Gate{aligned(g.contiguous())};
    };
    if (full && (gate.size(-1) != 1 || gate.scalar_type() == x.scalar_type())) return steps(gate);      // (of one step: either)
    if (x.numel() == 0) return {gate.expand(x.sizes()).to(x.scalar_type()).contiguous()};       // nothing to do, and no rows to divide
    if (gate.dim() > 0 && gate.size(-1) != 1) return steps(gate.expand(x.sizes()));
    // the same at every step: the dimensions that it has must lie next to each other
    int64_t a = d - 1, b = 0;
    for (int64_t i = 0; i < d - 1; ++i)
        if (i >= lead && gate.size(i - lead) != 1) a = std::min(a, i), b = i + 1;
    bool together = true;
    for (int64_t i = a; i < b; ++i) together = together && gate.size(i - lead) == x.size(i);
    if (a >= b) return {gate.reshape({1}), product(x.sizes(), 0, d - 1), 1};
    if (together) return {gate.reshape({-1}).contiguous(), product(x.sizes(), b, d - 1), product(x.sizes(), a, b)};
    auto rows = x.sizes().vec();
    rows.back() = 1;
    return {gate.expand(rows).reshape({-1}).contiguous(), 1, product(x.sizes(), 0, d - 1)};
}

// what has a first derivative and no second must not read as zero under create_graph
torch::Tensor first_only(torch::Tensor grad)
{
    if (!grad.defined() || !at::GradMode::is_enabled()) return grad;
    grad = grad.detach().set_requires_grad(true);
    return (*std::make_shared<torch::autograd::DelayedError>("gatedLeak: has first derivatives only", 1))({grad})[0];
}

struct Shape {
    int64_t rows, T, sample_rows, inner, period;
    int dtype, flags;
    Shape(const torch::Tensor &x, int64_t inner_, int64_t period_, int64_t flags_)
        : rows(product(x.sizes(), 0, x.dim() - 1)), T(x.size(-1)), sample_rows(std::max<int64_t>(1, x.dim() > 1 ? product(x.sizes(), 1, x.dim() - 1) : 1)),
          inner(inner_), period(period_), dtype(dtype_code(x, "x")), flags((int)flags_)
    {
    }
    // (the backward pass adds up the gradients of a gate per row there, too)
    torch::Tensor workspace(const torch::Tensor &x, bool backward) const
    {
        return torch::empty({size_of(slayer_b200_leak_workspace(rows, T, dtype, inner, backward ? period : 0), "gatedLeak")}, x.options().dtype(torch::kUInt8));
    }
};

// Forward keeps x, the gate and a state for each dozen steps; backward forms the other states from them again.
struct GatedLeak : public torch::autograd::Function<GatedLeak> {
    static variable_list forward(AutogradContext *ctx, const torch::Tensor &x, const torch::Tensor &gate, const c10::optional<torch::Tensor> &initial,
                                 const c10::optional<torch::Tensor> &lengths, int64_t inner, int64_t period, int64_t flags, bool wantState, bool want)
    {
        const Shape s(x, inner, period, flags);
        c10::cuda::CUDAGuard guard(x.device());
        auto y = torch::empty(x.sizes(), x.options());
        const auto floats = x.options().dtype(torch::kFloat32);
        torch::Tensor state, starts;
        if (wantState) state = torch::empty(x.sizes().slice(0, x.dim() - 1), floats);
        if (want) starts = torch::empty({s.rows, slayer_b200_leak_states(s.T)}, floats);
        const auto workspace = s.workspace(x, false);
        check_rc(slayer_b200_leak_forward(y.data_ptr(), wantState ? state.data_ptr<float>() : nullptr, want ? starts.data_ptr<float>() : nullptr, x.data_ptr(),
                                          gate.data_ptr(), initial.has_value() ? initial->data_ptr<float>() : nullptr, s.dtype, s.flags, s.rows, s.T,
                                          lengths.has_value() ? lengths->data_ptr<int64_t>() : nullptr, s.sample_rows, inner, period,
                                          workspace.data_ptr(), current_stream()),
                 "gatedLeak");
        if (want) {
            ctx->save_for_backward({x, gate, starts, lengths.value_or(torch::Tensor())});
            ctx->saved_data["inner"] = inner;
            ctx->saved_data["period"] = period;
            ctx->saved_data["flags"] = flags;
            ctx->saved_data["initial"] = initial.has_value();
        }
        ctx->set_materialize_grads(false);
        return wantState ? variable_list{y, state} : variable_list{y};
    }
    static variable_list backward(AutogradContext *ctx, variable_list up)
    {
        const auto v = ctx->get_saved_variables();
        const auto &x = v[0], &gate = v[1], &starts = v[2], &lengths = v[3];
        const Shape s(x, ctx->saved_data["inner"].toInt(), ctx->saved_data["period"].toInt(), ctx->saved_data["flags"].toInt());
        variable_list out(9);
        const bool some = up[0].defined() || (up.size() > 1 && up[1].defined());
        if (!some) return out;
        c10::cuda::CUDAGuard guard(x.device());
        const auto g = up[0].defined() ? aligned(up[0].contiguous()) : torch::zeros_like(x);
        torch::Tensor gstate;
        if (up.size() > 1 && up[1].defined()) gstate = up[1].contiguous();
        if (ctx->needs_input_grad(0)) out[0] = torch::empty_like(x);
        if (ctx->needs_input_grad(1)) out[1] = torch::empty_like(gate);
        if (ctx->saved_data["initial"].toBool() && ctx->needs_input_grad(2)) out[2] = torch::empty(x.sizes().slice(0, x.dim() - 1), starts.options());
        const auto workspace = s.workspace(x, true);
        check_rc(slayer_b200_leak_backward(out[0].defined() ? out[0].data_ptr() : nullptr, out[1].defined() ? out[1].data_ptr() : nullptr,
                                           out[2].defined() ? out[2].data_ptr<float>() : nullptr, g.data_ptr(),
                                           gstate.defined() ? gstate.data_ptr<float>() : nullptr, starts.data_ptr<float>(), x.data_ptr(), gate.data_ptr(),
                                           s.dtype, s.flags, s.rows, s.T, lengths.defined() ? lengths.data_ptr<int64_t>() : nullptr, s.sample_rows, s.inner,
                                           s.period, workspace.data_ptr(), current_stream()),
                 "gatedLeak");
        if (s.rows == 0 && out[1].defined()) out[1].zero_();
        for (auto &o : out) o = first_only(o);
        return out;
    }
};

void check_same_device(const torch::Tensor &y, const torch::Tensor &x, const char *name, const char *op)
{
    TORCH_CHECK(y.is_cuda(), op, ": ", name, " must be a CUDA tensor");
    check_device(x, y, "x", name);
}

// (y), or (y, the state after the last step)
std::vector<torch::Tensor> gatedLeakCuda(const torch::Tensor &x, const torch::Tensor &gate, const c10::optional<torch::Tensor> &initial,
                                         const c10::optional<torch::Tensor> &lengths, int64_t flags, bool wantState)
{
    const char *op = "gatedLeak";
    TORCH_CHECK_VALUE(x.dim() >= 1, op, ": x must have a time dimension");
    const auto outer = x.sizes().slice(0, x.dim() - 1);
    TORCH_CHECK(x.is_cuda(), op, ": x must be a CUDA tensor");
    dtype_code(x, "x");
    dtype_code(gate, "gate");
    const Gate g = gate_of(gate, x, op);
    TORCH_CHECK_VALUE(!initial.has_value() || initial->sizes() == outer, op, ": initial must have the shape of x without time, got ", initial->sizes(), " for ",
                      x.sizes());
    TORCH_CHECK_VALUE(!lengths.has_value() || (x.dim() >= 2 && lengths->dim() == 1 && lengths->size(0) == x.size(0)), op,
                      ": lengths must hold one number for each of the first dimension of x, got ", lengths->sizes(), " for ", x.sizes());
    TORCH_CHECK_TYPE(!lengths.has_value() || lengths->scalar_type() == torch::kInt64 || lengths->scalar_type() == torch::kInt32, op,
                     ": lengths must be int64 or int32, got ", lengths->scalar_type());
    check_same_device(gate, x, "gate", op);
    c10::optional<torch::Tensor> first, steps;
    if (initial.has_value()) {
        check_same_device(*initial, x, "initial", op);
        first = initial->to(torch::kFloat32).contiguous();
    }
    if (lengths.has_value()) {
        check_same_device(*lengths, x, "lengths", op);
        steps = lengths->to(torch::kInt64).contiguous();
    }
    const auto values = g.period ? g.values.to(torch::kFloat32) : g.values;
    const bool want = at::GradMode::is_enabled() && (x.requires_grad() || gate.requires_grad() || (initial.has_value() && initial->requires_grad()));
    return GatedLeak::apply(aligned(x.contiguous()), values, first, steps, g.inner, g.period, flags, wantState, want);
}

torch::Tensor gatedLeakStepCuda(const torch::Tensor &x, const torch::Tensor &gate, torch::Tensor state, int64_t flags)
{
    const char *op = "gatedLeakStep";
    TORCH_CHECK_VALUE(!(at::GradMode::is_enabled() && (x.requires_grad() || gate.requires_grad() || state.requires_grad())), op,
                      ": no gradient flows through it; use gatedLeak, or torch.no_grad()");
    TORCH_CHECK(x.is_cuda(), op, ": x must be a CUDA tensor");
    const int dtype = dtype_code(x, "x");
    dtype_code(gate, "gate");
    const auto rows = x.unsqueeze(-1);
    const Gate g = gate_of(gate.unsqueeze(-1), rows, op);
    TORCH_CHECK_VALUE(state.sizes() == x.sizes(), op, ": state must have the shape of x, got ", state.sizes(), " for ", x.sizes());
    TORCH_CHECK_TYPE(state.scalar_type() == torch::kFloat32, op, ": state must be float32, got ", state.scalar_type());
    TORCH_CHECK_VALUE(state.is_contiguous(), op, ": state must be contiguous");
    check_same_device(gate, x, "gate", op);
    check_same_device(state, x, "state", op);
    TORCH_CHECK(c10::InferenceMode::is_enabled() || !state.is_inference(), op, ": a state made in inference mode is updated in it only");
    auto values = g.values;
    if (values.scalar_type() != x.scalar_type()) values = values.to(torch::kFloat32);
    c10::cuda::CUDAGuard guard(x.device());
    const auto in = x.contiguous();
    // a thread would read what another has written
    const auto apart = [&](const torch::Tensor &v) {
        const auto a = (uintptr_t)v.data_ptr(), b = (uintptr_t)state.data_ptr();
        return a + v.nbytes() <= b || b + state.nbytes() <= a;
    };
    TORCH_CHECK_VALUE(apart(in) && apart(gate.is_contiguous() ? gate : values), op, ": state must not share memory with x or gate");
    auto y = torch::empty(x.sizes(), x.options());
    check_rc(slayer_b200_leak_step(y.data_ptr(), state.data_ptr<float>(), in.data_ptr(), values.data_ptr(), dtype, dtype_code(values, "gate"), (int)flags,
                                   x.numel(), g.inner, g.period, current_stream()),
             op);
    if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();      // autograd sees that it changed
    return y;
}

// what compress8 returned for a tensor of these sizes
void check_kept(const torch::Tensor &q, const torch::Tensor &scale, at::IntArrayRef sizes, const char *op)
{
    const int64_t rows = product(sizes, 0, (int64_t)sizes.size() - 1), groups = (sizes.back() + 31) / 32;
    TORCH_CHECK(q.is_cuda() && scale.is_cuda(), op, ": a checkpoint must be on a CUDA device");
    check_device(q, scale, "q", "scale");
    TORCH_CHECK_VALUE(q.sizes() == at::IntArrayRef({rows, groups * 32}) && scale.sizes() == at::IntArrayRef({groups, rows}), op, ": a checkpoint of ",
                      sizes, " has values ", at::IntArrayRef({rows, groups * 32}), " and scales ", at::IntArrayRef({groups, rows}), ", got ", q.sizes(), " and ",
                      scale.sizes());
    TORCH_CHECK(q.scalar_type() == torch::kInt8 && scale.scalar_type() == torch::kUInt8 && q.is_contiguous() && scale.is_contiguous(), op,
                ": a checkpoint has contiguous int8 values and uint8 scales");
}

std::vector<torch::Tensor> compress8Cuda(const torch::Tensor &x)
{
    TORCH_CHECK_VALUE(x.dim() >= 1, "compress: x must have a time dimension");
    TORCH_CHECK(x.is_cuda(), "compress: x must be a CUDA tensor");
    const int dtype = dtype_code(x, "x");
    c10::cuda::CUDAGuard guard(x.device());
    const auto in = x.detach().contiguous();
    const int64_t rows = product(x.sizes(), 0, x.dim() - 1), T = x.size(-1), groups = (T + 31) / 32;
    auto q = torch::empty({rows, groups * 32}, x.options().dtype(torch::kInt8)), scale = torch::empty({groups, rows}, x.options().dtype(torch::kUInt8));
    check_rc(slayer_b200_compress8(q.data_ptr<int8_t>(), scale.data_ptr<uint8_t>(), in.data_ptr(), dtype, rows, T, current_stream()), "compress");
    return {q, scale};
}

torch::Tensor restore8Cuda(const torch::Tensor &q, const torch::Tensor &scale, std::vector<int64_t> sizes, const torch::Tensor &like)
{
    TORCH_CHECK_VALUE(!sizes.empty(), "restore: a checkpoint has a time dimension");
    check_kept(q, scale, sizes, "restore");
    c10::cuda::CUDAGuard guard(q.device());
    auto out = torch::empty(sizes, q.options().dtype(like.scalar_type()));
    const int dtype = dtype_code(out, "restore: the result");
    check_rc(slayer_b200_restore8(out.data_ptr(), q.data_ptr<int8_t>(), scale.data_ptr<uint8_t>(), dtype, product(sizes, 0, (int64_t)sizes.size() - 1),
                                  sizes.back(), current_stream()),
             "restore");
    return out;
}

torch::Tensor spikeGrad8Cuda(const torch::Tensor &grad, const torch::Tensor &q, const torch::Tensor &scaleBytes, float theta, float tau, float scale)
{
    TORCH_CHECK_VALUE(grad.dim() >= 1, "spikeGrad: grad must have a time dimension");
    check_input(grad, "grad");
    check_kept(q, scaleBytes, grad.sizes(), "spikeGrad");
    check_device(grad, q, "grad", "the checkpoint");
    c10::cuda::CUDAGuard guard(grad.device());
    auto out = torch::empty_like(grad);
    const auto g = aligned(grad);
    check_rc(slayer_b200_spike_grad8(out.data_ptr<float>(), g.data_ptr<float>(), q.data_ptr<int8_t>(), scaleBytes.data_ptr<uint8_t>(),
                                     product(grad.sizes(), 0, grad.dim() - 1), grad.size(-1), theta, tau, scale, current_stream()),
             "spikeGrad");
    return out;
}

// grad [N, O, 1 ..., T] and a checkpoint of [N, sizes ..., T]: [O, sizes ..., 1]
torch::Tensor weightGrad8Cuda(const torch::Tensor &grad, const torch::Tensor &q, const torch::Tensor &scale, std::vector<int64_t> sizes)
{
    const int64_t d = (int64_t)sizes.size();
    TORCH_CHECK_VALUE(d >= 3, "weightGrad: the layer's input must be [samples, neurons ..., T]");
    TORCH_CHECK_VALUE(grad.dim() == d && grad.size(0) == sizes[0] && grad.size(-1) == sizes.back() && product(grad.sizes(), 2, d - 1) == 1,
                      "weightGrad: grad must be [samples, outputs, 1 ..., T] for an input ", at::IntArrayRef(sizes), ", got ", grad.sizes());
    check_input(grad, "grad");
    check_kept(q, scale, sizes, "weightGrad");
    check_device(grad, q, "grad", "the checkpoint");
    c10::cuda::CUDAGuard guard(grad.device());
    const int64_t N = sizes[0], O = grad.size(1), I = product(sizes, 1, d - 1), T = sizes.back();
    sizes.front() = O;
    sizes.back() = 1;
    auto out = torch::empty(sizes, grad.options());
    const auto g = aligned(grad);
    auto workspace = torch::empty({size_of(slayer_b200_weight_grad8_workspace(N, O, I, T), "weightGrad")}, grad.options().dtype(torch::kUInt8));
    check_rc(slayer_b200_weight_grad8(out.data_ptr<float>(), g.data_ptr<float>(), q.data_ptr<int8_t>(), scale.data_ptr<uint8_t>(), N, O, I, T,
                                      workspace.data_ptr(), current_stream()),
             "weightGrad");
    return out;
}

}  // namespace

void bind_sequence(pybind11::module_ &m)
{
    m.def("gatedLeak", &gatedLeakCuda, "Gated leaky integrator along time, differentiable (CUDA)");
    m.def("gatedLeakStep", &gatedLeakStepCuda, "One time step of the gated leaky integrator, its state in place (CUDA)");
    m.def("compress8", &compress8Cuda, "A tensor in 8 bits with a scale for each 32 time steps (CUDA)");
    m.def("restore8", &restore8Cuda, "What a tensor in 8 bits stands for (CUDA)");
    m.def("spikeGrad8", &spikeGrad8Cuda, "Surrogate gradient on a membrane potential kept in 8 bits (CUDA)");
    m.def("weightGrad8", &weightGrad8Cuda, "Weight gradient of a dense layer whose input is kept in 8 bits (CUDA)");
}
