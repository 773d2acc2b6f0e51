// Python bindings of what stands around the routed experts of a block: norm, choice of the experts, experts for a few tokens.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <pybind11/functional.h>
#include <pybind11/stl.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>

#include <tuple>

#include "../kernels/block_api.h"
#include "../kernels/few_ring.h"

namespace py = pybind11;

int* gemm_error_word(int device);  // gemm_bindings.cpp
long long gemm_wait_cycles(int device, double timeout_ms);

namespace {

#define DXB_CHECK(cond, what, msg)                                                                      \
    do {                                                                                                \
        if (!(cond)) throw std::invalid_argument(std::string("deepep_efa_b200.") + (what) + ": " + (msg)); \
    } while (0)

void launched(cudaError_t e, const char* what) {
    if (e != cudaSuccess) {
        cudaGetLastError();
        throw std::runtime_error(std::string("deepep_efa_b200.") + what + ": " + cudaGetErrorString(e));
    }
}

cudaStream_t stream_of(const torch::Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

bool aligned16(const torch::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

// Rows of a bf16 matrix that the kernels read in pieces of 16 bytes: neighbouring channels together, rows any multiple of eight elements apart.
bool rows_fit(const torch::Tensor& t) {
    return t.size(0) == 0 || t.size(1) == 0 || ((t.size(1) == 1 || t.stride(1) == 1) && t.stride(0) % 8 == 0 && t.stride(0) >= 0 && aligned16(t));
}
torch::Tensor fitting(const torch::Tensor& t) { return rows_fit(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

// Short steps wait for the host, which an allocation through the dispatcher takes a microsecond of.
torch::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const torch::Tensor& like) { return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt); }

// Refuses to drop a graph silently.
void forward_only(const char* what, std::initializer_list<const torch::Tensor*> tensors) {
    if (!at::GradMode::is_enabled()) return;
    for (const torch::Tensor* t : tensors) DXB_CHECK(!t->requires_grad(), what, "forward only; call it under torch.no_grad()");
}

// There are no forward-mode derivatives, under no_grad either: refuses to drop a tangent silently, as autograd does for the CPU forms.
void no_tangents(const char* what, std::initializer_list<const torch::Tensor*> tensors) {
    for (const torch::Tensor* t : tensors)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(0).defined(), "deepep_efa_b200.", what, ": no forward-mode derivative");
}

int sms_of(const torch::Tensor& t) { return at::cuda::getDeviceProperties(t.device().index())->multiProcessorCount; }

// x [N, H] (+ residual) -> (y, q, scales, total), with None for what was not asked for
std::tuple<c10::optional<torch::Tensor>, c10::optional<torch::Tensor>, c10::optional<torch::Tensor>, c10::optional<torch::Tensor>> rms_norm(
    const torch::Tensor& x_in, const torch::Tensor& weight, c10::optional<torch::Tensor> residual, double eps, bool rows, bool quantize, bool round_scale) {
    const char* what = "rms_norm";
    no_tangents(what, {&x_in, &weight, residual.has_value() ? &*residual : &x_in});
    DXB_CHECK(x_in.is_cuda() && x_in.dim() == 2 && x_in.scalar_type() == torch::kBFloat16, what, "x must be a CUDA bf16 matrix [N, H]");
    const int64_t N = x_in.size(0), H = x_in.size(1);
    DXB_CHECK(H > 0 && H % 8 == 0 && H <= dx::kNormMaxHidden, what, "hidden must be a multiple of 8, at most 32768");
    DXB_CHECK(!quantize || H % 128 == 0, what, "FP8 rows need a hidden size that is a multiple of 128");
    DXB_CHECK(weight.device() == x_in.device() && weight.dim() == 1 && weight.size(0) == H && (weight.scalar_type() == torch::kBFloat16 || weight.scalar_type() == torch::kFloat32),
              what, "weight must be bf16 or fp32 [H] on x's device");
    DXB_CHECK(!residual.has_value() || (residual->device() == x_in.device() && residual->scalar_type() == torch::kBFloat16 && residual->sizes() == x_in.sizes()), what,
              "residual must be bf16 of x's shape on x's device");
    DXB_CHECK(N <= 0x7fffffff, what, "too many rows");
    c10::cuda::CUDAGuard guard(x_in.device());
    const torch::Tensor x = fitting(x_in), res = residual.has_value() ? fitting(*residual) : x;
    const torch::Tensor w = weight.is_contiguous() && aligned16(weight) ? weight : weight.clone(at::MemoryFormat::Contiguous);
    c10::optional<torch::Tensor> y, q, scales, total;
    dx::NormArgs a{};
    if (rows) a.y = (y = fresh({N, H}, at::kBFloat16, x))->data_ptr();
    if (quantize) {
        a.q = static_cast<uint8_t*>((q = fresh({N, H}, at::kFloat8_e4m3fn, x))->data_ptr());
        a.scales = (scales = fresh({N, H / 128}, at::kFloat, x))->data_ptr<float>();
    }
    if (residual.has_value()) {
        a.residual = res.data_ptr();
        a.residual_stride = res.stride(0);
        a.total = (total = fresh({N, H}, at::kBFloat16, x))->data_ptr();
    }
    a.x = x.data_ptr();
    a.x_stride = x.stride(0);
    a.weight = w.data_ptr();
    a.weight_f32 = w.scalar_type() == torch::kFloat32;
    a.round_scale = round_scale;
    a.rows = N;
    a.hidden = (int)H;
    a.eps = (float)eps;
    launched(dx::launch_rms_norm(a, stream_of(x)), what);
    return {y, q, scales, total};
}

// ((q, scales), y or None, total or None)
std::tuple<std::tuple<torch::Tensor, torch::Tensor>, c10::optional<torch::Tensor>, c10::optional<torch::Tensor>> rms_norm_fp8(
    const torch::Tensor& x, const torch::Tensor& weight, const c10::optional<torch::Tensor>& residual, double eps, bool round_scale, bool keep_rows) {
    forward_only("rms_norm_fp8", {&x, &weight, residual.has_value() ? &*residual : &x});
    const auto [y, q, scales, total] = rms_norm(x, weight, residual, eps, keep_rows, true, round_scale);
    return {{*q, *scales}, y, total};
}

// -> (dx, dweight)
std::tuple<torch::Tensor, torch::Tensor> rms_norm_bwd(const torch::Tensor& total_in, const torch::Tensor& weight, const torch::Tensor& dy_in, c10::optional<torch::Tensor> dtotal,
                                                      double eps) {
    const char* what = "rms_norm_bwd";
    auto like = [&](const torch::Tensor& t) { return t.device() == total_in.device() && t.scalar_type() == torch::kBFloat16 && t.sizes() == total_in.sizes(); };
    DXB_CHECK(total_in.is_cuda() && total_in.dim() == 2 && total_in.scalar_type() == torch::kBFloat16, what, "the normed rows must be a CUDA bf16 matrix [N, H]");
    const int64_t N = total_in.size(0), H = total_in.size(1);
    DXB_CHECK(H > 0 && H % 8 == 0 && H <= dx::kNormMaxHidden, what, "hidden must be a multiple of 8, at most 32768");
    DXB_CHECK(like(dy_in) && (!dtotal.has_value() || like(*dtotal)), what, "gradients must be bf16 of the rows' shape on their device");
    DXB_CHECK(weight.device() == total_in.device() && weight.dim() == 1 && weight.size(0) == H && (weight.scalar_type() == torch::kBFloat16 || weight.scalar_type() == torch::kFloat32),
              what, "weight must be bf16 or fp32 [H] on the rows' device");
    c10::cuda::CUDAGuard guard(total_in.device());
    const torch::Tensor t = fitting(total_in), dy = fitting(dy_in), dt = dtotal.has_value() ? fitting(*dtotal) : dy;
    const torch::Tensor w = weight.is_contiguous() && aligned16(weight) ? weight : weight.clone(at::MemoryFormat::Contiguous);
    const int sms = sms_of(t), ctas = dx::norm_bwd_ctas(N, (int)H, sms);
    const torch::Tensor dx_out = fresh({N, H}, at::kBFloat16, t), dw = fresh({H}, w.scalar_type(), t), partial = fresh({ctas, H}, at::kFloat, t);
    dx::NormBwdArgs a{};
    a.total = t.data_ptr();
    a.dy = dy.data_ptr();
    a.dtotal = dtotal.has_value() ? dt.data_ptr() : nullptr;
    a.total_stride = t.stride(0);
    a.dy_stride = dy.stride(0);
    a.dtotal_stride = dt.stride(0);
    a.weight = w.data_ptr();
    a.weight_f32 = w.scalar_type() == torch::kFloat32;
    a.dx = dx_out.data_ptr();
    a.partial = partial.data_ptr<float>();
    a.dweight = dw.data_ptr();
    a.rows = N;
    a.hidden = (int)H;
    a.eps = (float)eps;
    launched(dx::launch_rms_norm_bwd(a, sms, stream_of(t)), what);
    return {dx_out, dw};
}

dx::SelectArgs select_args(const char* what, const torch::Tensor& logits, int64_t topk, bool renormalize) {
    DXB_CHECK(logits.is_cuda() && logits.dim() == 2 && (logits.scalar_type() == torch::kFloat32 || logits.scalar_type() == torch::kBFloat16), what,
              "logits must be a CUDA matrix [T, E] in fp32 or bf16");
    DXB_CHECK(logits.size(1) >= 1 && logits.size(1) <= dx::kRouterMaxExperts, what, "1 to 1024 experts");
    DXB_CHECK(topk >= 1 && topk <= dx::kRouterMaxTopk && topk <= logits.size(1), what, "num_topk must be 1 to 32 and at most the number of experts");
    DXB_CHECK(logits.size(0) <= 0x7fffffff / 32, what, "too many tokens");
    dx::SelectArgs a{};
    a.bf16 = logits.scalar_type() == torch::kBFloat16;
    a.tokens = (int)logits.size(0);
    a.experts = (int)logits.size(1);
    a.topk = (int)topk;
    a.renormalize = renormalize;
    return a;
}
torch::Tensor logit_rows(const torch::Tensor& t) { return t.size(1) == 1 || t.stride(1) == 1 ? t : t.clone(at::MemoryFormat::Contiguous); }

std::tuple<torch::Tensor, torch::Tensor> select_experts(const torch::Tensor& logits_in, int64_t topk, bool renormalize) {
    const char* what = "select_experts";
    no_tangents(what, {&logits_in});
    dx::SelectArgs a = select_args(what, logits_in, topk, renormalize);
    c10::cuda::CUDAGuard guard(logits_in.device());
    const torch::Tensor logits = logit_rows(logits_in);
    const torch::Tensor idx = fresh({a.tokens, a.topk}, at::kLong, logits), weights = fresh({a.tokens, a.topk}, at::kFloat, logits);
    a.logits = logits.data_ptr();
    a.logits_stride = logits.stride(0);
    a.idx = idx.data_ptr<int64_t>();
    a.weights = weights.data_ptr<float>();
    launched(dx::launch_select_experts(a, stream_of(logits)), what);
    return {idx, weights};
}

torch::Tensor select_experts_bwd(const torch::Tensor& logits_in, const torch::Tensor& idx, const torch::Tensor& weights, const torch::Tensor& dweights_in, bool renormalize) {
    const char* what = "select_experts_bwd";
    DXB_CHECK(idx.dim() == 2, what, "idx must be [T, K]");
    dx::SelectArgs a = select_args(what, logits_in, idx.size(1), renormalize);
    auto fits = [&](const torch::Tensor& t) { return t.device() == logits_in.device() && t.dim() == 2 && t.size(0) == a.tokens && t.size(1) == a.topk; };
    DXB_CHECK(fits(idx) && idx.scalar_type() == torch::kInt64 && idx.is_contiguous(), what, "idx must be contiguous int64 [T, K] on the logits' device");
    DXB_CHECK(fits(weights) && weights.scalar_type() == torch::kFloat32 && weights.is_contiguous(), what, "weights must be contiguous fp32 [T, K] on the logits' device");
    DXB_CHECK(fits(dweights_in) && dweights_in.scalar_type() == torch::kFloat32, what, "the weights' gradient must be fp32 [T, K] on the logits' device");
    c10::cuda::CUDAGuard guard(logits_in.device());
    const torch::Tensor logits = logit_rows(logits_in), dweights = dweights_in.contiguous(), dlogits = fresh({a.tokens, a.experts}, logits.scalar_type(), logits);
    a.logits = logits.data_ptr();
    a.logits_stride = logits.stride(0);
    a.idx = idx.data_ptr<int64_t>();
    a.weights = weights.data_ptr<float>();
    a.dweights = dweights.data_ptr<float>();
    a.dlogits = dlogits.data_ptr();
    launched(dx::launch_select_experts_bwd(a, stream_of(logits)), what);
    return dlogits;
}

// What a backward pass computed, where it was asked for with a graph: a node that refuses to be differentiated stands between it and `from`, what it depends on. Without
// one second-order terms would be lost without a word.
template <typename... T>
torch::autograd::variable_list once(const char* what, torch::autograd::variable_list results, const T&... from) {
    if (!at::GradMode::is_enabled() || !(from.requires_grad() || ...)) return results;
    const auto refusal = std::make_shared<torch::autograd::Error>(std::string("deepep_efa_b200.") + what + ": the gradient is not differentiable",
                                                                  torch::autograd::collect_next_edges(from...));
    for (const auto& t : results) torch::autograd::set_history(t, refusal);
    return results;
}

// The two with gradients as nodes of the autograd graph. In C++, since a step's launches are short: choice and gradient of 8192 x 64, us, as a Python function 70, so 58.
struct RMSNorm : torch::autograd::Function<RMSNorm> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& weight,
                                                  const c10::optional<torch::Tensor>& residual, double eps) {
        ctx->set_materialize_grads(false);
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["residual"] = residual.has_value();
        const auto [y, q, scales, total] = rms_norm(x, weight, residual, eps, true, false, false);
        ctx->save_for_backward({residual.has_value() ? *total : x, weight});
        if (residual.has_value()) return {*y, *total};
        return {*y};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const bool residual = ctx->saved_data["residual"].toBool();
        c10::optional<torch::Tensor> past;
        if (residual && grads[1].defined()) past = grads[1];
        if (!grads[0].defined()) {
            const torch::Tensor dx = past.has_value() ? *past : torch::Tensor();
            return {dx, torch::Tensor(), residual ? dx : torch::Tensor(), torch::Tensor()};
        }
        const auto [dx, dw] = rms_norm_bwd(saved[0], saved[1], grads[0], past, ctx->saved_data["eps"].toDouble());
        const auto out = once("rms_norm", {dx, dw}, saved[0], saved[1], grads[0], past.has_value() ? *past : grads[0]);
        return {out[0], out[1], residual ? out[0] : torch::Tensor(), torch::Tensor()};
    }
};
torch::autograd::variable_list rms_norm_grad(const torch::Tensor& x, const torch::Tensor& weight, const c10::optional<torch::Tensor>& residual, double eps) {
    if (!at::GradMode::is_enabled() || !(x.requires_grad() || weight.requires_grad() || (residual.has_value() && residual->requires_grad()))) {
        const auto [y, q, scales, total] = rms_norm(x, weight, residual, eps, true, false, false);
        if (total.has_value()) return {*y, *total};
        return {*y};
    }
    return RMSNorm::apply(x, weight, residual, eps);
}

struct SelectExperts : torch::autograd::Function<SelectExperts> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const torch::Tensor& logits, int64_t topk, bool renormalize) {
        ctx->set_materialize_grads(false);
        ctx->saved_data["renormalize"] = renormalize;
        const auto [idx, weights] = select_experts(logits, topk, renormalize);
        ctx->mark_non_differentiable({idx});
        ctx->save_for_backward({logits, idx, weights});
        return {idx, weights};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        if (!grads[1].defined()) return {torch::Tensor(), torch::Tensor(), torch::Tensor()};
        const torch::Tensor dlogits = select_experts_bwd(saved[0], saved[1], saved[2], grads[1], ctx->saved_data["renormalize"].toBool());
        return {once("select_experts", {dlogits}, saved[0], grads[1])[0], torch::Tensor(), torch::Tensor()};
    }
};
std::tuple<torch::Tensor, torch::Tensor> select_experts_grad(const torch::Tensor& logits, int64_t topk, bool renormalize) {
    const auto out = SelectExperts::apply(logits, topk, renormalize);
    return {out[0], out[1]};
}

torch::Tensor few_tokens(const torch::Tensor& x_in, const torch::Tensor& idx_in, const torch::Tensor& weights_in, const torch::Tensor& w13, const torch::Tensor& w2,
                         c10::optional<torch::Tensor> s13, c10::optional<torch::Tensor> s2, int64_t first, c10::optional<torch::Tensor> out) {
    const char* what = "few_token_experts";
    const auto dev = x_in.device();
    forward_only(what, {&x_in, &weights_in, &w13, &w2, out.has_value() ? &*out : &x_in});
    no_tangents(what, {&x_in, &weights_in, &w13, &w2});
    DXB_CHECK(x_in.is_cuda() && x_in.dim() == 2 && x_in.scalar_type() == torch::kBFloat16, what, "x must be a CUDA bf16 matrix [T, H]");
    const int64_t T = x_in.size(0), H = x_in.size(1);
    DXB_CHECK(T <= dx::kFewMaxTokens, what, "at most 32 tokens");
    DXB_CHECK(idx_in.device() == dev && idx_in.scalar_type() == torch::kInt64 && idx_in.dim() == 2 && idx_in.size(0) == T && idx_in.size(1) >= 1 && idx_in.size(1) <= dx::kFewMaxTopk,
              what, "topk_idx must be int64 [T, K] on x's device, K from 1 to 32");
    DXB_CHECK(weights_in.device() == dev && weights_in.scalar_type() == torch::kFloat32 && weights_in.sizes() == idx_in.sizes(), what,
              "topk_weights must be fp32 of topk_idx's shape on x's device");
    const bool fp8 = w13.scalar_type() == torch::kFloat8_e4m3fn;
    DXB_CHECK((fp8 || w13.scalar_type() == torch::kBFloat16) && w2.scalar_type() == w13.scalar_type(), what, "w13 and w2 must both be bf16 or both float8_e4m3fn");
    DXB_CHECK(w13.device() == dev && w2.device() == dev && w13.dim() == 3 && w2.dim() == 3, what, "w13 [L, 2 I, H] and w2 [L, H, I] must be on x's device");
    const int64_t L = w13.size(0), I = w13.size(1) / 2;
    DXB_CHECK(L >= 1 && L <= dx::kFewMaxExperts, what, "1 to 1024 experts");
    DXB_CHECK(w13.size(1) == 2 * I && I > 0 && w13.size(2) == H && w2.size(0) == L && w2.size(1) == H && w2.size(2) == I, what, "w13 must be [L, 2 I, H] and w2 [L, H, I]");
    DXB_CHECK(w13.is_contiguous() && w2.is_contiguous() && aligned16(w13) && aligned16(w2), what, "weights must be contiguous and 16-byte aligned");
    const int unit = fp8 ? 128 : 8;
    DXB_CHECK(H % unit == 0 && I % unit == 0, what, fp8 ? "FP8 weights need H and I that are multiples of 128" : "H and I must be multiples of 8");
    DXB_CHECK(2 * I <= 0x7fffffff && H <= 0x7fffffff, what, "the weights are too large");
    auto scales_fit = [&](const c10::optional<torch::Tensor>& s, int64_t n, int64_t k) {
        return s.has_value() && s->device() == dev && s->scalar_type() == torch::kFloat32 && s->is_contiguous() && s->dim() == 3 && s->size(0) == L && s->size(1) == n / 128 &&
               s->size(2) == k / 128;
    };
    DXB_CHECK(fp8 ? scales_fit(s13, 2 * I, H) && scales_fit(s2, H, I) : !s13.has_value() && !s2.has_value(), what,
              "FP8 weights need contiguous fp32 scales [L, N / 128, K / 128] on x's device, bf16 weights none");
    DXB_CHECK(!out.has_value() || (out->device() == dev && out->scalar_type() == torch::kBFloat16 && out->is_contiguous() && out->sizes() == x_in.sizes()), what,
              "out must be contiguous bf16 [T, H] on x's device");
    c10::cuda::CUDAGuard guard(dev);
    const torch::Tensor x = fitting(x_in), idx = idx_in.contiguous(), weights = weights_in.contiguous();
    const torch::Tensor y = out.has_value() ? *out : fresh({T, H}, at::kBFloat16, x);
    dx::FewTokensArgs a{};
    a.x = x.data_ptr();
    a.x_stride = x.stride(0);
    a.idx = idx.data_ptr<int64_t>();
    a.weights = weights.data_ptr<float>();
    a.w13 = w13.data_ptr();
    a.w2 = w2.data_ptr();
    a.s13 = fp8 ? s13->data_ptr<float>() : nullptr;
    a.s2 = fp8 ? s2->data_ptr<float>() : nullptr;
    a.out = y.data_ptr();
    a.first = first;
    a.tokens = (int)T;
    a.topk = (int)idx.size(1);
    a.experts = (int)L;
    a.hidden = (int)H;
    a.inter = (int)I;
    a.fp8 = fp8;
    a.error_flag = gemm_error_word(dev.index());
    a.wait_limit = gemm_wait_cycles(dev.index(), 2000.0);
    const torch::Tensor scratch = fresh({(int64_t)dx::few_tokens_scratch(a)}, at::kByte, x);
    a.scratch = scratch.data_ptr();
    launched(dx::launch_few_tokens(a, sms_of(x), stream_of(x)), what);
    if (out.has_value() && !out->is_inference()) torch::autograd::impl::bump_version(*out);  // a graph that has kept `out` notices
    return y;
}

}  // namespace

void bind_block(py::module_& m) {
    m.def("rms_norm", &rms_norm);
    m.def("rms_norm_fp8", &rms_norm_fp8);
    m.def("rms_norm_grad", &rms_norm_grad);
    m.def("rms_norm_bwd", &rms_norm_bwd);
    m.def("select_experts", &select_experts);
    m.def("select_experts_grad", &select_experts_grad);
    m.def("select_experts_bwd", &select_experts_bwd);
    m.def("few_tokens", &few_tokens);
    // (for tests without a GPU: what the warps of the experts for a few tokens keep of their rings)
    py::class_<dx::RingState>(m, "FewTokensRing")
        .def(py::init<int>())
        .def("started", &dx::RingState::started)
        .def("taken", &dx::RingState::taken)
        .def("give_up", [](dx::RingState& r, const std::function<void(int, int)>& wait) { r.give_up(wait); })
        .def_readonly("fill", &dx::RingState::fill)
        .def_readonly("slot", &dx::RingState::slot)
        .def_readonly("parity", &dx::RingState::parity)
        .def_readonly("flying", &dx::RingState::flying)
        .def_readonly("alive", &dx::RingState::alive);
}
