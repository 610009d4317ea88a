// experts_torch.cpp -- the routed-experts calls with plain arguments, from torch's tensors to the C entry points and back.
//
// A call of a few rows is as long as its way through the host: the same autograd nodes in Python take 81 us forward and backward
// (the engine's thread and the caller's then share the interpreter), these 55; without gradients 7.2 and 4.4.  Every function
// here returns None where an argument is not as plain as it takes it (another layout, type or device, a wrong shape): experts.py
// then goes its own way, which copies or says what is wrong.  Under a device-side row count and while calls are
// profiled, experts.py does not come here.
#include <ATen/ATen.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <optional>
#include <stdexcept>

#include "nsx.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream((c10::DeviceIndex)t.get_device()).stream(); }
int dtype_of(const Tensor& t) {
    return t.scalar_type() == at::kFloat ? NSX_DTYPE_F32 : t.scalar_type() == at::kHalf ? NSX_DTYPE_F16 : t.scalar_type() == at::kBFloat16 ? NSX_DTYPE_BF16 : -1;
}
bool aligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
bool here(const Tensor& t) { return t.is_cuda() && t.get_device() == c10::hip::current_device(); }
// forward-mode derivatives are refused (by experts.py)
bool dual(const Tensor& t) { return t._fw_grad(0).defined(); }
// consecutive values on the current device
bool plain(const Tensor& t, int64_t dims) { return t.dim() == dims && t.is_contiguous() && here(t); }
bool half_rows(const Tensor& t) { return plain(t, 2) && dtype_of(t) > 0 && t.size(1) % 8 == 0 && aligned(t); }
bool plan_at(const Tensor& offsets, const Tensor& rows, const Tensor& positions) { return here(offsets) && here(rows) && here(positions); }
void must(int rc, const char* what) {
    if (rc != NSX_OK) throw std::runtime_error(std::string("libnsx ") + what + " failed (rc=" + std::to_string(rc) + "): " + nsx_last_error());
}
Tensor like_rows(Tensor g) {
    g = g.contiguous();
    return aligned(g) ? g : g.clone();
}
// Results of a backward pass whose own derivative is asked for: differentiating them raises.
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list given;
    std::vector<size_t> places;
    for (size_t i = 0; i < grads.size(); ++i)
        if (grads[i].defined()) {
            given.push_back(grads[i].detach().set_requires_grad(true));
            places.push_back(i);
        }
    auto raise = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that was marked with @once_differentiable",
                                                                 (int64_t)given.size());
    given = (*raise)(std::move(given));
    for (size_t i = 0; i < places.size(); ++i) grads[places[i]] = given[i];
    return grads;
}

// ---- choice -----------------------------------------------------------------------------------------------------------
struct Choice { Tensor bias, selector; int64_t top_k, sigmoid, n_groups, top_groups, group_top, renormalise; double scale; };

int route(const Tensor& x, const Choice& c, Tensor& weights, Tensor& chosen) {
    const int64_t T = x.size(0), E = x.size(1);
    weights = at::empty({T, c.top_k}, x.options().dtype(at::kFloat));
    chosen = at::empty({T, c.top_k}, x.options().dtype(at::kInt));
    return nsx_expert_route_fwd(x.data_ptr(), dtype_of(x), T, (int)E, E, c.bias.defined() ? c.bias.data_ptr<float>() : nullptr,
                                c.selector.defined() ? c.selector.data_ptr<uint8_t>() : nullptr, (int)c.top_k, (int)c.sigmoid, (int)c.n_groups,
                                (int)c.top_groups, (int)c.group_top, (int)c.renormalise, (float)c.scale, weights.data_ptr<float>(),
                                chosen.data_ptr<int>(), nullptr, stream_of(x));
}

struct RouteNode : torch::autograd::Function<RouteNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Choice& c) {
        Tensor w, e;
        must(route(x, c, w, e), "nsx_expert_route_fwd");
        ctx->save_for_backward({x, w, e});
        ctx->mark_non_differentiable({e});
        ctx->set_materialize_grads(false);
        ctx->saved_data["sigmoid"] = c.sigmoid;
        ctx->saved_data["renormalise"] = c.renormalise;
        ctx->saved_data["scale"] = c.scale;
        return {w, e};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        Tensor none;
        if (!grads[0].defined()) return {none, none};
        auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &c = saved[2], g = grads[0].to(at::kFloat).contiguous();
        Tensor d = at::empty(x.sizes(), x.options());
        must(nsx_expert_route_bwd(x.data_ptr(), dtype_of(x), x.size(0), (int)x.size(1), x.size(1), (int)w.size(1), (int)ctx->saved_data["sigmoid"].toInt(),
                                  (int)ctx->saved_data["renormalise"].toInt(), (float)ctx->saved_data["scale"].toDouble(), w.data_ptr<float>(),
                                  c.data_ptr<int>(), g.data_ptr<float>(), d.data_ptr(), nullptr, stream_of(x)), "nsx_expert_route_bwd");
        return once({d, none});
    }
};

std::optional<std::pair<Tensor, Tensor>> route_experts(const Tensor& logits, int64_t top_k, int64_t sigmoid, const std::optional<Tensor>& bias,
                                                       const std::optional<Tensor>& selector, int64_t n_groups, int64_t top_groups, int64_t group_top,
                                                       int64_t renormalise, double scale) {
    if (!plain(logits, 2) || dtype_of(logits) < 0 || dual(logits)) return {};
    const int64_t T = logits.size(0), E = logits.size(1);
    if (E < 1 || E > NSX_MAX_EXPERTS || top_k < 1 || top_k > std::min<int64_t>(E, NSX_MAX_TOP_K)) return {};
    Choice c{{}, {}, top_k, sigmoid, n_groups, top_groups, group_top, renormalise, scale};
    if (bias) {
        if (!plain(*bias, 1) || bias->size(0) != E || bias->scalar_type() != at::kFloat) return {};
        c.bias = *bias;
    }
    if (selector) {
        if (!plain(*selector, 1) || selector->size(0) != T || selector->scalar_type() != at::kByte) return {};
        c.selector = *selector;
    }
    if (logits.requires_grad() && at::GradMode::is_enabled()) {
        auto out = RouteNode::apply(logits, c);
        return std::make_pair(out[0], out[1]);
    }
    Tensor w, e;
    must(route(logits, c, w, e), "nsx_expert_route_fwd");
    return std::make_pair(w, e);
}

// ---- plan -------------------------------------------------------------------------------------------------------------
std::optional<std::tuple<Tensor, Tensor, Tensor>> plan(const Tensor& chosen, int64_t E) {
    if (!plain(chosen, 2) || chosen.scalar_type() != at::kInt || E < 1 || E > NSX_MAX_EXPERTS) return {};
    const int64_t T = chosen.size(0), k = chosen.size(1), n = T * k, o = (E + 4) / 4 * 4, r = (n + 3) / 4 * 4;
    if (n > NSX_MAX_EXPERT_ENTRIES) return {};
    // one allocation: offsets | rows | positions | workspace (16-byte steps)
    Tensor all = at::empty({o + 2 * r + nsx_expert_plan_workspace(n, (int)E) / 4}, chosen.options());
    int* p = all.data_ptr<int>();
    must(nsx_expert_plan(chosen.data_ptr<int>(), T, (int)k, (int)E, p, p + o, p + o + r, p + o + 2 * r, nullptr, stream_of(chosen)), "nsx_expert_plan");
    return std::make_tuple(all.as_strided({E + 1}, {1}, 0), all.as_strided({n}, {1}, o), all.as_strided({T, k}, {k, 1}, o + r));
}

// ---- products ---------------------------------------------------------------------------------------------------------
int linear(const Tensor& x, const Tensor& w, const Tensor& offsets, const Tensor& rows, int64_t top_k, bool gather, bool relu, Tensor& y) {
    const int64_t R = rows.size(0), E = w.size(0), N = w.size(1), K = w.size(2);
    y = at::empty({R, N}, x.options());
    return nsx_expert_linear_fwd(x.data_ptr(), dtype_of(x), K, x.size(0), gather ? rows.data_ptr<int>() : nullptr, (int)top_k, w.data_ptr(), (int)K, (int)N,
                                 (int)E, offsets.data_ptr<int>(), R, relu, y.data_ptr(), stream_of(x));
}

struct Plan { Tensor offsets, rows, positions; };

struct LinearNode : torch::autograd::Function<LinearNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& w16, const Plan& p, bool gather, bool relu) {
        Tensor y, none;
        must(linear(x, w16, p.offsets, p.rows, p.positions.size(1), gather, relu, y), "nsx_expert_linear_fwd");
        ctx->save_for_backward({weight.requires_grad() ? x : none, x.requires_grad() ? w16 : none, relu ? y : none, p.offsets, p.rows, p.positions});
        ctx->saved_data["gather"] = gather;
        ctx->saved_data["f32"] = weight.scalar_type() == at::kFloat;
        ctx->saved_data["sizes"] = std::vector<int64_t>{x.size(0), w16.size(0), w16.size(1), w16.size(2)};
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w16 = saved[1], &y = saved[2], &offsets = saved[3], &rows = saved[4], &positions = saved[5];
        const bool gather = ctx->saved_data["gather"].toBool(), f32 = ctx->saved_data["f32"].toBool(), need_x = w16.defined(), need_w = x.defined();
        const auto sizes = ctx->saved_data["sizes"].toIntVector();
        const int64_t x_rows = sizes[0], E = sizes[1], N = sizes[2], K = sizes[3], R = rows.size(0);
        const Tensor g = like_rows(grads[0]);
        const int64_t need = nsx_expert_linear_bwd_workspace(R, (int)E, (int)K, (int)N, need_x, gather ? (int)positions.size(1) : 0, need_w, y.defined());
        if (need < 0) must((int)need, "nsx_expert_linear_bwd_workspace");
        Tensor ws, dx, dw, none;
        if (need) ws = at::empty({need}, g.options().dtype(at::kByte));
        if (need_x) dx = at::empty({x_rows, K}, g.options());
        if (need_w) dw = at::empty({E, N, K}, f32 ? g.options().dtype(at::kFloat) : g.options());
        must(nsx_expert_linear_bwd(need_w ? x.data_ptr() : nullptr, dtype_of(g), K, x_rows, gather ? rows.data_ptr<int>() : nullptr, positions.data_ptr<int>(),
                                   (int)positions.size(1), need_x ? w16.data_ptr() : nullptr, g.data_ptr(), N, y.defined() ? y.data_ptr() : nullptr, N, (int)K, (int)N,
                                   (int)E, offsets.data_ptr<int>(), R, need_x ? dx.data_ptr() : nullptr, f32, need_w ? dw.data_ptr() : nullptr,
                                   need ? ws.data_ptr() : nullptr, stream_of(g)), "nsx_expert_linear_bwd");
        return once({dx, dw, none, none, none, none});
    }
};

std::optional<Tensor> expert_linear(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& copy, const Tensor& offsets, const Tensor& rows,
                                    const Tensor& positions, bool gather, bool relu) {
    const Tensor& w16 = copy ? *copy : weight;
    if (!half_rows(x) || !plain(w16, 3) || w16.scalar_type() != x.scalar_type() || !aligned(w16) || !plan_at(offsets, rows, positions) ||
        dual(x) || dual(weight) || dual(w16)) return {};
    if (copy && (!here(weight) || weight.sizes() != w16.sizes() || (weight.scalar_type() != at::kFloat && weight.scalar_type() != x.scalar_type()))) return {};
    if (w16.size(0) != offsets.size(0) - 1 || w16.size(2) != x.size(1) || x.size(0) != (gather ? positions.size(0) : rows.size(0))) return {};
    if (w16.size(1) < 8 || w16.size(1) % 8 || w16.size(1) > NSX_MAX_EXPERT_WIDTH || x.size(1) < 8 || x.size(1) > NSX_MAX_EXPERT_WIDTH) return {};
    if ((x.requires_grad() || weight.requires_grad()) && at::GradMode::is_enabled()) return LinearNode::apply(x, weight, w16, Plan{offsets, rows, positions}, gather, relu);
    Tensor y;
    must(linear(x, w16, offsets, rows, positions.size(1), gather, relu, y), "nsx_expert_linear_fwd");
    return y;
}

// ---- join -------------------------------------------------------------------------------------------------------------
int combine(const Tensor& y, const Tensor& w, const Tensor& positions, Tensor& out) {
    const int64_t T = positions.size(0), n = y.size(1);
    out = at::empty({T, n}, y.options());
    return nsx_expert_combine_fwd(y.data_ptr(), dtype_of(y), n, y.size(0), (int)n, w.data_ptr<float>(), positions.data_ptr<int>(), T, (int)positions.size(1),
                                  out.data_ptr(), nullptr, stream_of(y));
}

struct CombineNode : torch::autograd::Function<CombineNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& y, const Tensor& w, const Plan& p) {
        Tensor out;
        must(combine(y, w, p.positions, out), "nsx_expert_combine_fwd");
        ctx->save_for_backward({y, w, p.offsets, p.positions});
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        auto saved = ctx->get_saved_variables();
        const Tensor &y = saved[0], &w = saved[1], &offsets = saved[2], &positions = saved[3], g = like_rows(grads[0]);
        const int64_t T = positions.size(0), n = y.size(1);
        Tensor dy = at::empty(y.sizes(), y.options()), dw = at::empty(w.sizes(), w.options()), none;
        must(nsx_expert_combine_bwd(y.data_ptr(), dtype_of(y), n, y.size(0), (int)n, w.data_ptr<float>(), positions.data_ptr<int>(),
                                    offsets.data_ptr<int>() + offsets.size(0) - 1, T, (int)positions.size(1), g.data_ptr(), dy.data_ptr(), dw.data_ptr<float>(),
                                    nullptr, stream_of(y)), "nsx_expert_combine_bwd");
        return once({dy, dw, none});
    }
};

std::optional<Tensor> expert_combine(const Tensor& y, const Tensor& w, const Tensor& offsets, const Tensor& rows, const Tensor& positions) {
    if (!half_rows(y) || !plain(w, 2) || w.scalar_type() != at::kFloat || !plan_at(offsets, rows, positions) || dual(y) || dual(w)) return {};
    if (w.sizes() != positions.sizes() || y.size(0) != rows.size(0) || y.size(1) < 8 || y.size(1) > NSX_MAX_EXPERT_WIDTH) return {};
    if ((y.requires_grad() || w.requires_grad()) && at::GradMode::is_enabled()) return CombineNode::apply(y, w, Plan{offsets, rows, positions});
    Tensor out;
    must(combine(y, w, positions, out), "nsx_expert_combine_fwd");
    return out;
}

}  // namespace

PYBIND11_MODULE(_experts, m) {
    m.attr("nsx_version") = NSX_VERSION;           // (experts.py compares both with what runs)
    m.attr("torch_version") = NSX_TORCH;
    m.def("route_experts", &route_experts);
    m.def("plan", &plan);
    m.def("expert_linear", &expert_linear);
    m.def("expert_combine", &expert_combine);
}
