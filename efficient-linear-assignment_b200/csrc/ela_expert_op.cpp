// ela_expert_op.cpp -- the expert-layer operators as C++ torch operators over
// the C ABI (include/ela_expert.h), with their autograd.
//
//   ela_native::expert_plan(expert, num_experts) -> (offsets, position, source)
//   ela_native::expert_dispatch(x, position, offsets) -> rows
//   ela_native::expert_combine(y, position, offsets, weights?) -> out
//   ela_native::expert_linear(x, weight, bias?, residual?, offsets?, activation) -> y
//
// Arguments are checked here, with Python's TypeError and ValueError, and host tensors
// are refused by CPU kernels that raise: the Python functions only forward, since a
// small call is bound by host time.  As in ela_torch_op.cpp: device guard, outputs and workspaces from the caching
// allocator, the current stream, no synchronisation.  Autograd is here for
// the same reason.  The backward passes launch kernels that autograd does not see, so asking for a gradient of
// a gradient (create_graph) raises; so does a forward-mode derivative, whose tangents would be lost.
#include <torch/library.h>
#include <torch/csrc/autograd/custom_function.h>
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <tuple>

#include "ela_expert.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> OptTensor;

int code_of(const Tensor& t) {
    switch (t.scalar_type()) {
    case at::kFloat: return ELA_DTYPE_F32;
    case at::kHalf: return ELA_DTYPE_F16;
    case at::kBFloat16: return ELA_DTYPE_BF16;
    default: return -1;
    }
}

[[noreturn]] void refuse(const char* name) { TORCH_CHECK(false, name, " needs CUDA tensors (there is no CPU path)"); }

void check_rc(int rc, const char* where) {
    TORCH_CHECK(rc == ELA_OK, where, ": ", ela_status_string(rc), " (status ", rc, ")");
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
const void* ptr(const OptTensor& t) { return t.has_value() ? t->data_ptr() : nullptr; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// Unit stride inside a row; any (non-negative) distance between rows.
Tensor rows_of(const Tensor& t) {
    return (t.size(-1) <= 1 || t.stride(-1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(-1)) ? t : t.contiguous();
}
int64_t ld(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(-1); }

// An uninitialised tensor on like's device from the caching allocator (straight from it:
// at::empty's dispatch costs as much again).
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
    return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}
Tensor fresh(at::IntArrayRef sizes, const Tensor& like) { return fresh(sizes, like.scalar_type(), like); }

Tensor workspace(size_t bytes, const Tensor& like) {
    return bytes ? fresh({(int64_t)bytes}, at::kByte, like) : Tensor();
}

void no_second_derivative() {
    TORCH_CHECK(!at::GradMode::is_enabled(), "the expert operators have no second derivative (create_graph=True)");
}

// ---- plan
std::tuple<Tensor, Tensor, Tensor> plan(const Tensor& expert_in, int64_t E) {
    TORCH_CHECK_TYPE(expert_in.scalar_type() == at::kInt || expert_in.scalar_type() == at::kLong,
                     "expert_plan: expert must be int32 or int64, not ", expert_in.scalar_type());
    TORCH_CHECK_VALUE(expert_in.dim() == 1 || expert_in.dim() == 2, "expert_plan: expert must be (T,) or (T, k)");
    TORCH_CHECK_VALUE(E >= 1 && E <= ELA_EXPERT_MAX, "expert_plan: num_experts must be 1..", ELA_EXPERT_MAX);
    TORCH_CHECK_VALUE(expert_in.numel() <= INT32_MAX, "expert_plan: more than 2^31 - 1 choices");
    c10::cuda::CUDAGuard guard(expert_in.device());
    const Tensor expert = expert_in.contiguous();
    Tensor offsets = fresh({E + 1}, at::kInt, expert), source = fresh({expert.numel()}, at::kInt, expert);
    Tensor position = fresh({expert.size(0), expert.dim() == 1 ? 1 : expert.size(1)}, at::kInt, expert);
    const size_t bytes = ela_expert_plan_workspace_bytes(expert.numel(), E);
    Tensor ws = workspace(bytes, expert);
    check_rc(ela_expert_plan(expert.data_ptr(), (int)expert.element_size(), expert.numel(), E, offsets.data_ptr<int32_t>(),
                             position.data_ptr<int32_t>(), source.data_ptr<int32_t>(), ptr(ws), bytes, stream_of(expert)),
             "ela_expert_plan");
    return {offsets, position, source};
}

void check_rows(const char* name, const Tensor& rows, int64_t want, const Tensor& position, const Tensor& offsets) {
    if (!rows.is_cuda()) refuse(name);
    TORCH_CHECK_TYPE(code_of(rows) >= 0, name, ": unsupported dtype ", rows.scalar_type());
    TORCH_CHECK_VALUE(position.scalar_type() == at::kInt && offsets.scalar_type() == at::kInt && position.dim() == 2 &&
                          offsets.dim() == 1 && offsets.numel() >= 2 && position.is_contiguous() && offsets.is_contiguous() &&
                          position.device() == rows.device() && offsets.device() == rows.device(),
                      name, ": the plan's position (T, k) and offsets (E+1,) must be contiguous int32 on the rows' device");
    TORCH_CHECK_VALUE(rows.dim() == 2 && rows.size(0) == want, name, ": a matrix of ", want, " rows is needed");
}

// ---- dispatch and combine
Tensor dispatch_raw(const Tensor& x_in, const Tensor& position, const Tensor& offsets) {
    check_rows("expert_dispatch", x_in, position.dim() == 2 ? position.size(0) : -1, position, offsets);
    const int code = code_of(x_in);
    c10::cuda::CUDAGuard guard(x_in.device());
    const Tensor x = rows_of(x_in);
    Tensor rows = fresh({position.numel(), x.size(1)}, x);
    check_rc(ela_expert_dispatch(x.data_ptr(), code, x.size(0), position.size(1), x.size(1), ld(x),
                                 position.data_ptr<int32_t>(), offsets.data_ptr<int32_t>(), offsets.numel() - 1,
                                 rows.data_ptr(), stream_of(x)),
             "ela_expert_dispatch");
    return rows;
}

Tensor combine_raw(const Tensor& y_in, const Tensor& position, const Tensor& offsets, const OptTensor& weights) {
    check_rows("expert_combine", y_in, position.numel(), position, offsets);
    const int code = code_of(y_in);
    if (weights.has_value()) {
        TORCH_CHECK_TYPE(weights->scalar_type() == at::kFloat || weights->scalar_type() == y_in.scalar_type(),
                         "expert_combine: weights must be float32 or y's dtype, not ", weights->scalar_type());
        TORCH_CHECK_VALUE((weights->sizes() == position.sizes() || (weights->dim() == 1 && position.size(1) == 1 && weights->size(0) == position.size(0))) &&
                              weights->device() == y_in.device(), "expert_combine: weights must be (T, k) on y's device");
    }
    c10::cuda::CUDAGuard guard(y_in.device());
    const Tensor y = rows_of(y_in);
    const OptTensor w = weights.has_value() ? OptTensor(weights->contiguous()) : OptTensor();
    Tensor out = fresh({position.size(0), y.size(1)}, y);
    check_rc(ela_expert_combine(y.data_ptr(), code, position.size(0), position.size(1), y.size(1), ld(y),
                                position.data_ptr<int32_t>(), offsets.data_ptr<int32_t>(), offsets.numel() - 1, ptr(w),
                                w.has_value() ? code_of(*w) : ELA_DTYPE_F32, out.data_ptr(), stream_of(y)),
             "ela_expert_combine");
    return out;
}

// (dy, dweights); the one that is not needed comes back empty
std::tuple<Tensor, Tensor> combine_grad_raw(const Tensor& dout_in, const OptTensor& y_in, const Tensor& position,
                                            const Tensor& offsets, const OptTensor& weights, bool need_y, bool need_w) {
    const Tensor dout = rows_of(dout_in);
    const OptTensor y = y_in.has_value() ? OptTensor(rows_of(*y_in)) : OptTensor();
    const OptTensor w = weights.has_value() ? OptTensor(weights->contiguous()) : OptTensor();
    c10::cuda::CUDAGuard guard(dout.device());
    Tensor dy = fresh({need_y ? position.numel() : 0, dout.size(1)}, dout);
    Tensor dw = need_w ? fresh(w->sizes(), *w) : fresh({0}, dout);
    check_rc(ela_expert_combine_grad(dout.data_ptr(), ptr(y), code_of(dout), position.size(0), position.size(1),
                                     dout.size(1), ld(dout), y.has_value() ? ld(*y) : 0, position.data_ptr<int32_t>(),
                                     offsets.data_ptr<int32_t>(), offsets.numel() - 1, ptr(w),
                                     w.has_value() ? code_of(*w) : ELA_DTYPE_F32, need_y ? dy.data_ptr() : nullptr,
                                     need_w ? dw.data_ptr() : nullptr, stream_of(dout)),
             "ela_expert_combine_grad");
    return {dy, dw};
}

// ---- linear
struct LinearSizes {
    int64_t R, E, K, N;
    Tensor x, w;  // unit stride inside rows
    int64_t stride_e, ldw;
};

Tensor weight_rows(const Tensor& w) {
    const Tensor v = w.dim() == 2 ? w.unsqueeze(0) : w;
    const bool ok = (v.size(2) <= 1 || v.stride(2) == 1) && (v.size(1) <= 1 || v.stride(1) >= v.size(2)) &&
                    (v.size(0) <= 1 || v.stride(0) > 0);
    return ok ? v : v.contiguous();
}

LinearSizes linear_sizes(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual,
                         const OptTensor& offsets) {
    if (!x.is_cuda()) refuse("expert_linear");
    TORCH_CHECK_TYPE(x.scalar_type() == at::kHalf || x.scalar_type() == at::kBFloat16,
                     "expert_linear: x must be float16 or bfloat16, not ", x.scalar_type());
    auto operand = [&](const char* name, const Tensor& t) {
        TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type(), "expert_linear: ", name, " must be ", x.scalar_type(), ", not ", t.scalar_type());
        TORCH_CHECK_VALUE(t.device() == x.device(), "expert_linear: ", name, " must be on x's device");
    };
    operand("weight", weight);
    TORCH_CHECK_VALUE(x.dim() == 2 && (weight.dim() == 2 || weight.dim() == 3) && weight.size(-1) == x.size(1),
                      "expert_linear: x must be (R, K), weight (E, N, K) or (N, K)");
    TORCH_CHECK_VALUE(weight.numel() > 0 && (weight.dim() == 2 || weight.size(0) <= ELA_EXPERT_MAX),
                      "expert_linear: E must be 1..", ELA_EXPERT_MAX, ", N and K at least 1");
    LinearSizes s;
    s.x = rows_of(x);
    s.w = weight_rows(weight);
    s.R = x.size(0);
    s.E = s.w.size(0);
    s.K = x.size(1);
    s.N = s.w.size(1);
    s.stride_e = s.E > 1 ? s.w.stride(0) : 0;
    s.ldw = s.N > 1 ? s.w.stride(1) : s.K;
    if (bias.has_value()) {
        operand("bias", *bias);
        TORCH_CHECK_VALUE(weight.dim() == 3 ? bias->dim() == 2 && bias->size(0) == s.E && bias->size(1) == s.N
                                            : bias->dim() == 1 && bias->size(0) == s.N,
                          "expert_linear: bias must be (E, N), or (N,) for one matrix");
    }
    if (residual.has_value()) {
        operand("residual", *residual);
        TORCH_CHECK_VALUE(residual->dim() == 2 && residual->size(0) == s.R && residual->size(1) == s.N,
                          "expert_linear: residual must be (R, N)");
    }
    if (offsets.has_value())
        TORCH_CHECK_VALUE(offsets->scalar_type() == at::kInt && offsets->is_contiguous() && offsets->dim() == 1 &&
                              offsets->numel() == s.E + 1 && offsets->device() == x.device(),
                          "expert_linear: offsets must be contiguous int32 (E+1,) on x's device");
    TORCH_CHECK_VALUE(offsets.has_value() || s.E == 1, "expert_linear: offsets are needed for more than one expert");
    return s;
}

// What z is kept in: the slope of GELU and SiLU is taken from an unrounded z, ReLU's from its sign.
at::ScalarType kept_type(const Tensor& x, int64_t act) {
    return act == ELA_ACT_GELU || act == ELA_ACT_SILU ? at::kFloat : x.scalar_type();
}

int aligned(const Tensor& t, int64_t ldt, int64_t stride_e = 0) {
    const int64_t es = t.element_size();
    return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && ldt * es % 16 == 0 && stride_e * es % 16 == 0;
}

const int32_t* off_ptr(const OptTensor& o) { return o.has_value() ? o->data_ptr<int32_t>() : nullptr; }

std::tuple<Tensor, Tensor> linear_raw(const Tensor& x, const Tensor& weight, const OptTensor& bias,
                                      const OptTensor& residual, const OptTensor& offsets, int64_t act, bool want_z) {
    const LinearSizes s = linear_sizes(x, weight, bias, residual, offsets);
    c10::cuda::CUDAGuard guard(x.device());
    const OptTensor b = bias.has_value() ? OptTensor(bias->contiguous()) : OptTensor();
    const OptTensor r = residual.has_value() ? OptTensor(rows_of(*residual)) : OptTensor();
    Tensor y = fresh({s.R, s.N}, s.x);
    Tensor z = fresh({want_z ? s.R : 0, s.N}, kept_type(x, act), s.x);  // rows of no expert stay unwritten
    const int al = aligned(s.x, ld(s.x)) && aligned(s.w, s.ldw, s.stride_e);
    const size_t bytes = ela_expert_linear_workspace_bytes(ELA_LINEAR_FORWARD, s.R, s.E, s.K, s.N, al);
    Tensor ws = workspace(bytes, x);
    check_rc(ela_expert_linear(s.x.data_ptr(), s.w.data_ptr(), ptr(b), ptr(r), off_ptr(offsets), code_of(x), s.R, s.E, s.K,
                               s.N, ld(s.x), s.stride_e, s.ldw, r.has_value() ? ld(*r) : 0, (int)act, y.data_ptr(), want_z ? z.data_ptr() : nullptr,
                               ptr(ws), bytes, stream_of(x)),
             "ela_expert_linear");
    return {y, z};
}

// The gradients asked for; the others come back empty.
std::tuple<Tensor, Tensor, Tensor> linear_grad_raw(const Tensor& dy_in, const OptTensor& z, const OptTensor& x_in,
                                                   const OptTensor& weight, const OptTensor& offsets, int64_t act,
                                                   at::IntArrayRef wsizes, at::IntArrayRef bsizes, bool need_x,
                                                   bool need_w, bool need_b) {
    const Tensor dy = dy_in.contiguous();
    c10::cuda::CUDAGuard guard(dy.device());
    const int64_t R = dy.size(0), N = dy.size(1), K = wsizes.back(), E = wsizes.size() == 3 ? wsizes[0] : 1;
    const int code = code_of(dy);
    void* stream = stream_of(dy);
    Tensor dx = fresh({need_x ? R : 0, K}, dy);
    Tensor dw = need_w ? fresh(wsizes, dy) : fresh({0}, dy);
    Tensor db = need_b ? fresh(bsizes, dy) : fresh({0}, dy);
    Tensor dz = dy;
    if (need_b || act != ELA_ACT_NONE) {
        const bool write = act != ELA_ACT_NONE && (need_x || need_w);
        if (write) dz = fresh(dy.sizes(), dy);
        const size_t bytes = ela_expert_linear_workspace_bytes(ELA_LINEAR_GRAD_ACT, R, E, K, N, 1);
        Tensor ws = workspace(bytes, dy);
        check_rc(ela_expert_linear_grad_act(dy.data_ptr(), ptr(z), off_ptr(offsets), code, R, E, N, (int)act,
                                            write ? dz.data_ptr() : nullptr, need_b ? db.data_ptr() : nullptr, ptr(ws),
                                            bytes, stream),
                 "ela_expert_linear_grad_act");
    }
    if (need_x) {
        const Tensor w = weight_rows(*weight);
        const int64_t se = E > 1 ? w.stride(0) : 0, ldw = N > 1 ? w.stride(1) : K;
        const size_t bytes = ela_expert_linear_workspace_bytes(ELA_LINEAR_GRAD_INPUT, R, E, K, N,
                                                               aligned(dz, N) && aligned(w, ldw, se));
        Tensor ws = workspace(bytes, dy);
        check_rc(ela_expert_linear_grad_input(dz.data_ptr(), w.data_ptr(), off_ptr(offsets), code, R, E, K, N, se, ldw,
                                              dx.data_ptr(), ptr(ws), bytes, stream),
                 "ela_expert_linear_grad_input");
    }
    if (need_w) {
        const Tensor x = rows_of(*x_in);
        const size_t bytes = ela_expert_linear_workspace_bytes(ELA_LINEAR_GRAD_WEIGHT, R, E, K, N,
                                                               aligned(dz, N) && aligned(x, ld(x)));
        Tensor ws = workspace(bytes, dy);
        check_rc(ela_expert_linear_grad_weight(dz.data_ptr(), x.data_ptr(), off_ptr(offsets), code, R, E, K, N, ld(x),
                                               dw.data_ptr(), ptr(ws), bytes, stream),
                 "ela_expert_linear_grad_weight");
    }
    return {dx, dw, db};
}

Tensor linear_cuda(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual,
                   const OptTensor& offsets, int64_t act) {
    return std::get<0>(linear_raw(x, weight, bias, residual, offsets, act, false));
}

// ---- autograd: every pass is a registered operator, so that traced graphs see them
template <typename F> auto op(const char* name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
Tensor given(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

Tensor call_dispatch(const Tensor& x, const Tensor& position, const Tensor& offsets) {
    static auto f = op<Tensor(const Tensor&, const Tensor&, const Tensor&)>("ela_native::expert_dispatch");
    return f.call(x, position, offsets);
}
Tensor call_combine(const Tensor& y, const Tensor& position, const Tensor& offsets, const OptTensor& weights) {
    static auto f = op<Tensor(const Tensor&, const Tensor&, const Tensor&, const OptTensor&)>("ela_native::expert_combine");
    return f.call(y, position, offsets, weights);
}

struct Dispatch : torch::autograd::Function<Dispatch> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& position, const Tensor& offsets) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({position, offsets});
        return call_dispatch(x, position, offsets);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        no_second_derivative();
        const auto saved = ctx->get_saved_variables();
        return {call_combine(grads[0], saved[0], saved[1], OptTensor()), Tensor(), Tensor()};
    }
};

struct Combine : torch::autograd::Function<Combine> {
    static Tensor forward(AutogradContext* ctx, const Tensor& y, const Tensor& position, const Tensor& offsets,
                          const OptTensor& weights) {
        const bool need_w = weights.has_value() && weights->requires_grad();
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({need_w ? y : Tensor(), position, offsets, given(weights)});
        return call_combine(y, position, offsets, weights);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        no_second_derivative();
        static auto f = op<std::tuple<Tensor, Tensor>(const Tensor&, const OptTensor&, const Tensor&, const Tensor&,
                                                      const OptTensor&, bool, bool)>("ela_native::expert_combine_grad");
        const auto saved = ctx->get_saved_variables();
        const bool need_y = ctx->needs_input_grad(0), need_w = saved[0].defined() && ctx->needs_input_grad(3);
        auto g = f.call(grads[0], opt(saved[0]), saved[1], saved[2], opt(saved[3]), need_y, need_w);
        return {need_y ? std::get<0>(g) : Tensor(), Tensor(), Tensor(), need_w ? std::get<1>(g) : Tensor()};
    }
};

struct Linear : torch::autograd::Function<Linear> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& bias,
                          const OptTensor& residual, const OptTensor& offsets, int64_t act) {
        static auto f = op<std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const OptTensor&, const OptTensor&,
                                                      const OptTensor&, int64_t, bool)>("ela_native::expert_linear_z");
        const bool gx = x.requires_grad(), gw = weight.requires_grad(), gb = bias.has_value() && bias->requires_grad();
        at::AutoDispatchBelowADInplaceOrView below;
        const bool want_z = act != ELA_ACT_NONE && (gx || gw || gb);
        auto out = f.call(x, weight, bias, residual, offsets, act, want_z);
        ctx->save_for_backward({gw ? x : Tensor(), gx ? weight : Tensor(), want_z ? std::get<1>(out) : Tensor(),
                                given(offsets)});
        ctx->saved_data["act"] = act;
        ctx->saved_data["residual"] = residual.has_value();
        ctx->saved_data["wsizes"] = weight.sizes().vec();
        ctx->saved_data["bsizes"] = bias.has_value() ? bias->sizes().vec() : std::vector<int64_t>{};
        return std::get<0>(out);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        no_second_derivative();
        static auto f = op<std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const OptTensor&, const OptTensor&,
                                                              const OptTensor&, const OptTensor&, int64_t,
                                                              at::IntArrayRef, at::IntArrayRef, bool, bool, bool)>(
            "ela_native::expert_linear_grad");
        const auto saved = ctx->get_saved_variables();
        const auto wsizes = ctx->saved_data["wsizes"].toIntVector(), bsizes = ctx->saved_data["bsizes"].toIntVector();
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1),
                   need_b = !bsizes.empty() && ctx->needs_input_grad(2);
        const int residual_at = bsizes.empty() ? 2 : 3;  // an absent bias has no edge
        variable_list out(6);
        if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(residual_at)) out[3] = grads[0];
        if (!need_x && !need_w && !need_b) return out;
        auto g = f.call(grads[0], opt(saved[2]), opt(saved[0]), opt(saved[1]), opt(saved[3]),
                        ctx->saved_data["act"].toInt(), wsizes, bsizes, need_x, need_w, need_b);
        if (need_x) out[0] = std::get<0>(g);
        if (need_w) out[1] = std::get<1>(g);
        if (need_b) out[2] = std::get<2>(g);
        return out;
    }
};

// A tensor of a forward-mode derivative (a dual tensor) need not require a gradient.
bool dual(const Tensor& t) { return t._fw_grad(/*level=*/0).defined(); }
bool dual(const OptTensor& t) { return t.has_value() && dual(*t); }
template <typename... Ts> void no_forward_mode(const Ts&... ts) {
    TORCH_CHECK(!(dual(ts) || ...), "the expert operators have no forward-mode derivative");
}

// Without a gradient to prepare, the operator itself: the graph's bookkeeping costs more
// host time than a small call's kernel.
bool tracked(const Tensor& t) { return t.requires_grad() && at::GradMode::is_enabled(); }
bool tracked(const OptTensor& t) { return t.has_value() && tracked(*t); }

Tensor dispatch_autograd(const Tensor& x, const Tensor& position, const Tensor& offsets) {
    no_forward_mode(x);
    if (!tracked(x)) {
        at::AutoDispatchBelowADInplaceOrView below;
        return call_dispatch(x, position, offsets);
    }
    return Dispatch::apply(x, position, offsets);
}
Tensor combine_autograd(const Tensor& y, const Tensor& position, const Tensor& offsets, const OptTensor& weights) {
    no_forward_mode(y, weights);
    if (!tracked(y) && !tracked(weights)) {
        at::AutoDispatchBelowADInplaceOrView below;
        return call_combine(y, position, offsets, weights);
    }
    return Combine::apply(y, position, offsets, weights);
}
Tensor linear_autograd(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual,
                       const OptTensor& offsets, int64_t act) {
    no_forward_mode(x, weight, bias, residual);
    if (!tracked(x) && !tracked(weight) && !tracked(bias) && !tracked(residual)) {
        static auto f = op<Tensor(const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, const OptTensor&,
                                  int64_t)>("ela_native::expert_linear");
        at::AutoDispatchBelowADInplaceOrView below;
        return f.call(x, weight, bias, residual, offsets, act);
    }
    return Linear::apply(x, weight, bias, residual, offsets, act);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(ela_native, m) {
    m.def("expert_plan(Tensor expert, int num_experts) -> (Tensor, Tensor, Tensor)");
    m.def("expert_dispatch(Tensor x, Tensor position, Tensor offsets) -> Tensor");
    m.def("expert_combine(Tensor y, Tensor position, Tensor offsets, Tensor? weights) -> Tensor");
    m.def("expert_combine_grad(Tensor dout, Tensor? y, Tensor position, Tensor offsets, Tensor? weights, "
          "bool need_y, bool need_w) -> (Tensor, Tensor)");
    m.def("expert_linear(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, Tensor? offsets, int activation) -> Tensor");
    m.def("expert_linear_z(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, Tensor? offsets, int activation, "
          "bool want_z) -> (Tensor, Tensor)");
    m.def("expert_linear_grad(Tensor dy, Tensor? z, Tensor? x, Tensor? weight, Tensor? offsets, int activation, "
          "int[] wsizes, int[] bsizes, bool need_x, bool need_w, bool need_b) -> (Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(ela_native, CUDA, m) {
    m.impl("expert_plan", &plan);
    m.impl("expert_dispatch", &dispatch_raw);
    m.impl("expert_combine", &combine_raw);
    m.impl("expert_combine_grad", &combine_grad_raw);
    m.impl("expert_linear", &linear_cuda);
    m.impl("expert_linear_z", &linear_raw);
    m.impl("expert_linear_grad", &linear_grad_raw);
}

TORCH_LIBRARY_IMPL(ela_native, CPU, m) {
    m.impl("expert_plan", [](const Tensor&, int64_t) -> std::tuple<Tensor, Tensor, Tensor> { refuse("expert_plan"); });
    m.impl("expert_dispatch", [](const Tensor&, const Tensor&, const Tensor&) -> Tensor { refuse("expert_dispatch"); });
    m.impl("expert_combine", [](const Tensor&, const Tensor&, const Tensor&, const OptTensor&) -> Tensor { refuse("expert_combine"); });
    m.impl("expert_linear", [](const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, const OptTensor&, int64_t) -> Tensor {
        refuse("expert_linear");
    });
}

TORCH_LIBRARY_IMPL(ela_native, AutogradCUDA, m) {
    m.impl("expert_dispatch", &dispatch_autograd);
    m.impl("expert_combine", &combine_autograd);
    m.impl("expert_linear", &linear_autograd);
}
