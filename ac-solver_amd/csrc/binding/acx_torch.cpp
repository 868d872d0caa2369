// acx_torch.cpp -- the recurrent agent's operators on torch tensors: checks of arguments, outputs and scratch memory, autograd nodes, and the
// calls of libacx's C ABI (include/acx.h).  Host code only, no kernels: a backward pass runs on autograd's own thread, where a Python function
// costs several times what it does in the foreground (75 us of a 165 us pass over a short scan), and the operators' smallest calls are host
// time altogether.
// The functions of the ABI come from Python as addresses (bind): there is one libacx in the process, the one that ac_solver._acx loaded.
#define __HIP_PLATFORM_AMD__ 1
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>
#include <string>
#include <tuple>
#include <type_traits>

#include "../../../include/acx.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

namespace {

#define ACX_FUNCTIONS(X)                                                                                                                    \
    X(acx_last_error) X(acx_scan_bounds_bytes) X(acx_scan_workspace_bytes) X(acx_scan_forward) X(acx_scan_backward) X(acx_block_workspace_bytes) \
        X(acx_block_forward) X(acx_block_backward) X(acx_block_step) X(acx_act8_pack) X(acx_act8_unpack) X(acx_act8_workspace_bytes)            \
            X(acx_act8_weight_grad)
#define ACX_POINTER(f) decltype(&::f) f = nullptr;
struct Functions {
    ACX_FUNCTIONS(ACX_POINTER)
} api;

struct AcxFailure : std::runtime_error {
    using std::runtime_error::runtime_error;
};
void check(int rc, const char* what) {
    if (rc == ACX_E_INVAL) throw py::value_error(api.acx_last_error());
    if (rc != ACX_OK) throw AcxFailure(std::string(what) + " failed (code " + std::to_string(rc) + "): " + api.acx_last_error());
}

[[noreturn]] void value_error(const std::string& s) { throw py::value_error(s); }
[[noreturn]] void type_error(const std::string& s) { throw py::type_error(s); }

std::string shape_text(at::IntArrayRef s) {
    std::string t = "(";
    for (size_t i = 0; i < s.size(); i++) t += (i ? ", " : "") + std::to_string(s[i]);
    return t + (s.size() == 1 ? ",)" : ")");
}
std::string type_text(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return "float32";
        case at::kDouble: return "float64";
        case at::kHalf: return "float16";
        case at::kBFloat16: return "bfloat16";
        case at::kChar: return "int8";
        case at::kByte: return "uint8";
        case at::kBool: return "bool";
        case at::kInt: return "int32";
        case at::kLong: return "int64";
        default: return c10::toString(t);
    }
}

struct NoForwardMode : std::runtime_error {  // (NotImplementedError, as torch raises for its own functions)
    using std::runtime_error::runtime_error;
};
// Every operand that can carry one passes here: outputs without its tangent would read as a derivative of zero.  (Inside a function of autograd forward
// mode is off, and there is nothing to be seen: the operands are looked at in front of it, by wants_grad.)
void require_no_tangent(const Tensor& t, const char* name) {
    if (t._fw_grad(0).defined()) throw NoForwardMode(std::string(name) + " has a tangent: forward mode derivatives of this operator are not implemented");
}

Tensor tensor(py::handle o, const char* name) {
    if (!THPVariable_Check(o.ptr())) type_error(std::string(name) + " has to be a tensor, not " + Py_TYPE(o.ptr())->tp_name);
    return THPVariable_Unpack(o.ptr());
}
Maybe maybe(py::handle o, const char* name) {
    if (o.is_none()) return std::nullopt;
    return tensor(o, name);
}

int code_of(at::ScalarType t) { return t == at::kFloat ? ACX_F32 : t == at::kBFloat16 ? ACX_BF16 : t == at::kHalf ? ACX_F16 : -1; }

// An activation as a kernel reads it: float32 / bfloat16 / float16, last axis contiguous (a copy of one whose is not, such as the expanded gradient
// of a sum).
Tensor activation(Tensor t, const char* name, const Tensor* like = nullptr, std::optional<at::IntArrayRef> shape = std::nullopt) {
    if (code_of(t.scalar_type()) < 0) type_error(std::string(name) + " has to be float32, bfloat16 or float16, not " + type_text(t.scalar_type()));
    require_no_tangent(t, name);
    if (like && (t.scalar_type() != like->scalar_type() || t.device() != like->device()))
        value_error(std::string(name) + " is " + type_text(t.scalar_type()) + " on " + t.device().str() + ", the other activations are " + type_text(like->scalar_type()) + " on " +
                    like->device().str());
    if (shape && t.sizes() != *shape) value_error(std::string(name) + " has the shape " + shape_text(t.sizes()) + ", expected " + shape_text(*shape));
    if (t.is_contiguous() || (t.dim() && (t.size(-1) == 1 || t.stride(-1) == 1))) return t;
    return t.contiguous();
}
// a contiguous tensor of exactly this type, shape and device (parameters, states)
Tensor plain(Tensor t, const char* name, at::IntArrayRef shape, at::Device device, at::ScalarType type = at::kFloat) {
    if (t.scalar_type() != type) type_error(std::string(name) + " has to be " + type_text(type) + ", not " + type_text(t.scalar_type()));
    require_no_tangent(t, name);
    if (t.sizes() != shape) value_error(std::string(name) + " has the shape " + shape_text(t.sizes()) + ", expected " + shape_text(shape));
    if (t.device() != device) value_error(std::string(name) + " lives on " + t.device().str() + ", the activations on " + device.str());
    return t.is_contiguous() ? t : t.contiguous();
}
// bool or uint8 flags
Tensor flags(Tensor t, const char* name, at::IntArrayRef shape, at::Device device) { return plain(t, name, shape, device, t.scalar_type() == at::kBool ? at::kBool : at::kByte); }
void require_gpu(const Tensor& t) {
    if (!t.is_cuda()) value_error("the activations have to live on a GPU, not on " + t.device().str() + ": there is no CPU path");
}

// whether two tensors have no element in common, as far as it is told easily: memory apart, or other columns of the same rows
bool apart(const Tensor& a, const Tensor& b) {
    if (!a.numel() || !b.numel()) return true;
    auto bytes = [](const Tensor& t) {
        int64_t n = 1;
        for (int64_t k = 0; k < t.dim(); k++) n += (t.size(k) - 1) * t.stride(k);
        return n * (int64_t)t.element_size();
    };
    const int64_t between = static_cast<const char*>(b.data_ptr()) - static_cast<const char*>(a.data_ptr());
    if (between >= bytes(a) || -between >= bytes(b)) return true;
    if (a.scalar_type() != b.scalar_type() || a.sizes() != b.sizes()) return false;
    int64_t row = 0;
    for (int64_t k = 0; k + 1 < a.dim(); k++) {
        if (a.size(k) == 1) continue;
        if (a.stride(k) != b.stride(k)) return false;
        row = row && row < a.stride(k) ? row : a.stride(k);
    }
    const int64_t columns = (between < 0 ? -between : between) / (int64_t)a.element_size();
    return columns >= a.size(-1) && columns + a.size(-1) <= row;
}
void require_apart(const Tensor& t, const char* name, std::initializer_list<const Maybe*> others) {
    for (const Maybe* o : others)
        if (*o && !apart(t, **o)) value_error(std::string(name) + " lies in the memory of another operand");
}
// a caller's tensor that results are written into: contiguous last axis, no element named twice, nothing that is still read
void require_target(const Tensor& t, const char* name, const Tensor& like, std::initializer_list<const Maybe*> others) {
    if (!activation(t, name, &like, like.sizes()).is_same(t)) value_error(std::string(name) + " has to have a contiguous last axis");
    int64_t extent = t.size(-1), before = 0;  // of the axes so far, from the narrowest stride to the widest
    for (int64_t n = 0; n + 1 < t.dim(); n++) {
        int64_t axis = -1;
        for (int64_t k = 0; k + 1 < t.dim(); k++)
            if (t.size(k) > 1 && t.stride(k) > before && (axis < 0 || t.stride(k) < t.stride(axis))) axis = k;
        for (int64_t k = 0; k + 1 < t.dim(); k++)
            if (t.size(k) > 1 && (t.stride(k) < t.size(-1) || (axis >= 0 && k != axis && t.stride(k) == t.stride(axis)))) value_error(std::string(name) + " has rows that overlap");
        if (axis < 0) break;
        if (t.stride(axis) < extent) value_error(std::string(name) + " has rows that overlap");
        before = t.stride(axis);
        extent += before * (t.size(axis) - 1);
    }
    require_apart(t, name, others);
}

// a caller's tensor has been written into: what autograd kept of it elsewhere is not what it was
void count_change(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void* ptr(const Tensor& t) { return t.data_ptr(); }
void* ptr(const Maybe& t) { return t ? t->data_ptr() : nullptr; }
template <class T> T* ptr_as(const Tensor& t) { return static_cast<T*>(t.data_ptr()); }
template <class T> T* ptr_as(const Maybe& t) { return t ? static_cast<T*>(t->data_ptr()) : nullptr; }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
Tensor floats(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options().dtype(at::kFloat)); }
Tensor same(const Tensor& like, at::IntArrayRef shape) { return at::empty(shape, like.options()); }
Maybe scratch(int64_t bytes, const Tensor& like) {
    if (!bytes) return std::nullopt;
    return at::empty({bytes}, like.options().dtype(at::kByte));
}
int64_t bytes_of(const Maybe& t) { return t ? t->numel() : 0; }
bool wants_grad(std::initializer_list<const Maybe*> ts) {
    for (const Maybe* t : ts)
        if (*t) require_no_tangent(**t, "an operand");
    if (!at::GradMode::is_enabled()) return false;
    for (const Maybe* t : ts)
        if (*t && (*t)->requires_grad()) return true;
    return false;
}
// The gradients of a backward pass that is itself recorded (create_graph), from those of the outputs: differentiating them again raises.  They hang on every operand
// of the forward pass (the edges of the node that runs), whether it was kept or not, so that no way from them to an operand leaves a term out.
variable_list once(variable_list grads, const variable_list& from) {
    if (!at::GradMode::is_enabled()) return grads;
    torch::autograd::edge_list edges;
    if (const auto node = torch::autograd::get_current_node())
        for (const auto& e : node->next_edges())
            if (e.is_valid()) edges.push_back(e);
    for (const auto& t : from)
        if (t.defined() && t.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(t));
    const auto error = std::make_shared<torch::autograd::Error>("the gradients of this operator cannot be differentiated again", std::move(edges));
    for (auto& g : grads)
        if (g.defined()) {
            g = g.detach();
            torch::autograd::create_gradient_edge(g, error);
        }
    return grads;
}
Maybe opt(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }
Tensor orundef(const Maybe& t) { return t ? *t : Tensor(); }

// ---- the recurrence ---------------------------------------------------------------------------------------------------------------
struct ScanOperands {
    Tensor c, z;
    Maybe reset, state;
    int64_t steps, rows, width;
};
ScanOperands scan_operands(const Tensor& candidate, const Tensor& gate, const Maybe& reset, const Maybe& state) {
    ScanOperands o;
    o.c = activation(candidate, "candidate");
    if (o.c.dim() != 3) value_error("candidate has to be [steps, rows, features], not " + shape_text(o.c.sizes()));
    o.z = activation(gate, "gate", &o.c, o.c.sizes());
    o.steps = o.c.size(0), o.rows = o.c.size(1), o.width = o.c.size(2);
    if (o.steps < 1) value_error("a scan needs at least one step");
    if (reset) o.reset = flags(*reset, "reset", {o.steps, o.rows}, o.c.device());
    if (state) o.state = plain(*state, "state", {o.rows, o.width}, o.c.device());
    require_gpu(o.c);
    return o;
}
// -> hidden, last state, what the backward pass needs besides the operands
std::tuple<Tensor, Tensor, Maybe> scan_forward(const Tensor& candidate, const Tensor& gate, const Maybe& reset, const Maybe& state, bool save) {
    const ScanOperands o = scan_operands(candidate, gate, reset, state);
    const c10::OptionalDeviceGuard guard(o.c.device());
    const int code = code_of(o.c.scalar_type());
    Tensor hidden = same(o.c, o.c.sizes()), last = floats({o.rows, o.width}, o.c);
    Maybe bounds, work = scratch(api.acx_scan_workspace_bytes(o.steps, o.rows, o.width, code), o.c);
    if (save) bounds = floats({api.acx_scan_bounds_bytes(o.steps, o.rows, o.width) / 4}, o.c);
    check(api.acx_scan_forward(ptr(o.c), o.c.stride(0), o.c.stride(1), ptr(o.z), o.z.stride(0), o.z.stride(1), code, ptr_as<uint8_t>(o.reset), ptr_as<float>(o.state), o.steps, o.rows, o.width,
                               ptr(hidden), ptr_as<float>(last), ptr_as<float>(bounds), ptr(work), bytes_of(work), stream_of(o.c)),
          "acx_scan_forward");
    return {hidden, last, bounds};
}
// -> gradients of candidate, gate, state (if wanted); the first two into `dc`, `dz` where these are given
std::tuple<Tensor, Tensor, Maybe> scan_backward(const Tensor& d_hidden, const Maybe& d_last, const Tensor& candidate, const Tensor& gate, const Maybe& reset, const Tensor& bounds, bool want_state,
                                                Maybe dc = std::nullopt, Maybe dz = std::nullopt) {
    const ScanOperands o = scan_operands(candidate, gate, reset, std::nullopt);
    const Tensor dh = activation(d_hidden, "d_hidden", &o.c, o.c.sizes());
    Maybe dl;
    if (d_last) dl = plain(*d_last, "d_last", {o.rows, o.width}, o.c.device());
    const Tensor b = plain(bounds, "bounds", {api.acx_scan_bounds_bytes(o.steps, o.rows, o.width) / 4}, o.c.device());
    const c10::OptionalDeviceGuard guard(o.c.device());
    const Maybe operands[] = {o.c, o.z, dh, b};
    auto target = [&](Maybe& t, const char* name, const Maybe* other) {
        if (t) require_target(*t, name, o.c, {&operands[0], &operands[1], &operands[2], &operands[3], &dl, &o.reset, other});
        else t = same(o.c, o.c.sizes());
    };
    target(dc, "out[0]", &dz), target(dz, "out[1]", &dc);
    const int code = code_of(o.c.scalar_type());
    Maybe ds, work = scratch(api.acx_scan_workspace_bytes(o.steps, o.rows, o.width, code), o.c);
    if (want_state) ds = floats({o.rows, o.width}, o.c);
    check(api.acx_scan_backward(ptr(o.c), o.c.stride(0), o.c.stride(1), ptr(o.z), o.z.stride(0), o.z.stride(1), ptr(dh), dh.stride(0), dh.stride(1), code, ptr_as<uint8_t>(o.reset),
                                ptr_as<float>(b), ptr_as<float>(dl), o.steps, o.rows, o.width, ptr(*dc), dc->stride(0), dc->stride(1), ptr(*dz), dz->stride(0), dz->stride(1),
                                ptr_as<float>(ds), ptr(work), bytes_of(work), stream_of(o.c)),
          "acx_scan_backward");
    count_change(*dc), count_change(*dz);
    return {*dc, *dz, ds};
}

struct GatedScan : torch::autograd::Function<GatedScan> {
    static variable_list forward(AutogradContext* ctx, const Tensor& candidate, const Tensor& gate, const Maybe& reset, const Maybe& state) {
        auto [hidden, last, bounds] = scan_forward(candidate, gate, reset, state, true);
        ctx->save_for_backward({candidate, gate, orundef(reset), *bounds});
        ctx->saved_data["state"] = state.has_value() && state->requires_grad();
        ctx->set_materialize_grads(false);
        return {hidden, last};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        if (!g[0].defined() && !g[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        const auto saved = ctx->get_saved_variables();
        variable_list out;
        {
            const at::NoGradGuard no_grad;
            const Tensor d_hidden = g[0].defined() ? g[0] : at::zeros({}, saved[0].options()).expand(saved[0].sizes());
            auto [dc, dz, ds] = scan_backward(d_hidden, opt(g[1]), saved[0], saved[1], opt(saved[2]), saved[3], ctx->saved_data["state"].toBool());
            out = {dc, dz, Tensor(), orundef(ds)};
        }
        return once(std::move(out), g);
    }
};

// ---- the end of a block -----------------------------------------------------------------------------------------------------------
constexpr int64_t kMaxWidth = 4096;

struct BlockOperands {
    Tensor x;
    Maybe y, g, w, s, n;
    int64_t rows, width;
};
void check_width(int64_t width, double eps) {
    if (width > kMaxWidth) value_error("rows of up to " + std::to_string(kMaxWidth) + " features are handled, not " + std::to_string(width));
    if (!(eps >= 0.0)) value_error("eps has to be a number of at least 0, not " + std::to_string(eps));
}
BlockOperands block_operands(const Tensor& x, const Maybe& y, const Maybe& gate, const Maybe& weight, const Maybe& scale, const Maybe& next_weight, double eps) {
    BlockOperands o;
    o.x = activation(x, "x");
    if (o.x.dim() < 1) value_error("x has to have a feature axis");
    o.width = o.x.size(-1);
    check_width(o.width, eps);
    o.rows = o.width ? o.x.numel() / o.width : 0;
    const at::Device dev = o.x.device();
    if (y) {
        o.y = activation(*y, "y", &o.x, o.x.sizes());
        if (!weight) type_error("weight has to be a tensor, not NoneType");
        o.w = plain(*weight, "weight", {o.width}, dev);
    }
    if (gate) {
        if (!y) value_error("a gate without y");
        o.g = activation(*gate, "gate", &o.x, o.x.sizes());
    }
    if (scale) o.s = plain(*scale, "scale", {o.width}, dev);
    if (next_weight) o.n = plain(*next_weight, "next_weight", {o.width}, dev);
    require_gpu(o.x);
    return o;
}
// [..., width] as rows with one stride between them (a copy only where the leading axes have none in common)
Tensor rows_of(const Tensor& t) { return t.dim() == 2 ? t : t.reshape({-1, t.size(-1)}); }
struct Rows {
    Tensor t;
    void* p = nullptr;
    int64_t stride = 0;
    explicit Rows(const Maybe& m) {
        if (m) t = rows_of(*m), p = t.data_ptr(), stride = t.stride(0);
    }
};

std::tuple<Maybe, Maybe, Maybe> block_forward(const Tensor& x, const Maybe& y, const Maybe& gate, const Maybe& weight, const Maybe& scale, const Maybe& next_weight, double eps, bool save) {
    const BlockOperands o = block_operands(x, y, gate, weight, scale, next_weight, eps);
    const c10::OptionalDeviceGuard guard(o.x.device());
    Maybe out, u, stats;
    if (o.y) out = same(o.x, o.x.sizes());
    if (o.n) u = same(o.x, o.x.sizes());
    if (save) stats = floats({o.rows, 2}, o.x);
    if (o.rows) {
        const Rows rx(o.x), ry(o.y), rg(o.g);
        check(api.acx_block_forward(rx.p, rx.stride, ry.p, ry.stride, rg.p, rg.stride, code_of(o.x.scalar_type()), ptr_as<float>(o.w), ptr_as<float>(o.s), ptr_as<float>(o.n), (float)eps, o.rows,
                                    o.width, ptr(out), ptr(u), ptr_as<float>(stats), stream_of(o.x)),
              "acx_block_forward");
    }
    return {out, u, stats};
}
// -> gradients of x, y, gate, weight, scale, next_weight (none for an operand that is none)
std::tuple<Tensor, Maybe, Maybe, Maybe, Maybe, Maybe> block_backward(const Maybe& d_new, const Maybe& d_u, const Tensor& x, const Maybe& y, const Maybe& gate, const Maybe& weight, const Maybe& scale,
                                                                     const Maybe& next_weight, const Tensor& stats, Maybe dg = std::nullopt) {
    const BlockOperands o = block_operands(x, y, gate, weight, scale, next_weight, 0.0);
    if (d_u && !o.n) value_error("a gradient of u without next_weight");
    Maybe gn, gu;
    if (d_new) gn = activation(*d_new, "d_new", &o.x, o.x.sizes());
    if (d_u) gu = activation(*d_u, "d_u", &o.x, o.x.sizes());
    const Tensor st = plain(stats, "stats", {o.rows, 2}, o.x.device());
    const c10::OptionalDeviceGuard guard(o.x.device());
    Tensor dx = same(o.x, o.x.sizes());
    Maybe dy, dg_rows;
    if (o.y) dy = same(o.x, o.x.sizes());
    if (o.g) {
        const Maybe operands[] = {o.x, st};
        if (dg) require_target(*dg, "d_gate_out", o.x, {&operands[0], &operands[1], &o.y, &o.g, &gn, &gu, &o.w, &o.s, &o.n});
        else dg = same(o.x, o.x.sizes());
    } else {
        dg = std::nullopt;
    }
    Tensor weights = o.rows ? floats({3, o.width}, o.x) : at::zeros({3, o.width}, o.x.options().dtype(at::kFloat));
    if (o.rows) {
        if (dg) dg_rows = dg->dim() == 2 ? *dg : dg->view({-1, o.width});  // (raises where the rows have no common stride: the result has to land in the caller's tensor)
        const Rows rx(o.x), ry(o.y), rg(o.g), rn(gn), ru(gu), rdg(dg_rows);
        const int code = code_of(o.x.scalar_type());
        Maybe work = scratch(api.acx_block_workspace_bytes(o.rows, o.width, code), o.x);
        check(api.acx_block_backward(rx.p, rx.stride, ry.p, ry.stride, rg.p, rg.stride, rn.p, rn.stride, ru.p, ru.stride, code, ptr_as<float>(o.w), ptr_as<float>(o.s), ptr_as<float>(o.n),
                                     ptr_as<float>(st), o.rows, o.width, ptr(dx), ptr(dy), rdg.p, rdg.stride, ptr_as<float>(weights), ptr(work), bytes_of(work), stream_of(o.x)),
              "acx_block_backward");
        if (dg) count_change(*dg);
    }
    Maybe dw, ds, dn;
    if (o.y) dw = weights.select(0, 0);
    if (o.y && o.s) ds = weights.select(0, 1);
    if (o.n) dn = weights.select(0, 2);
    return {dx, dy, dg, dw, ds, dn};
}

struct BlockOutput : torch::autograd::Function<BlockOutput> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& y, const Maybe& gate, const Maybe& weight, const Maybe& scale, const Maybe& next_weight, double eps) {
        auto [out, u, stats] = block_forward(x, y, gate, weight, scale, next_weight, eps, true);
        ctx->save_for_backward({x, orundef(y), orundef(gate), orundef(weight), orundef(scale), orundef(next_weight), *stats});
        ctx->saved_data["new"] = out.has_value();
        ctx->saved_data["u"] = u.has_value();
        ctx->set_materialize_grads(false);
        variable_list r;
        if (out) r.push_back(*out);
        if (u) r.push_back(*u);
        return r;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        variable_list out(7);
        const bool has_new = ctx->saved_data["new"].toBool(), has_u = ctx->saved_data["u"].toBool();
        const Tensor d_new = has_new ? g[0] : Tensor(), d_u = has_u ? g[has_new ? 1 : 0] : Tensor();
        if (!d_new.defined() && !d_u.defined()) return out;
        const auto s = ctx->get_saved_variables();
        {
            const at::NoGradGuard no_grad;
            auto [dx, dy, dg, dw, ds, dn] = block_backward(opt(d_new), opt(d_u), s[0], opt(s[1]), opt(s[2]), opt(s[3]), opt(s[4]), opt(s[5]), s[6]);
            out = {dx, orundef(dy), orundef(dg), orundef(dw), orundef(ds), orundef(dn), Tensor()};
            // (an argument that does not belong to the result, such as the scale without y, has a gradient of nothing)
            for (int i = 3; i < 6; i++)
                if (s[i].defined() && !out[i].defined()) out[i] = at::zeros(s[i].sizes(), s[i].options());
        }
        return once(std::move(out), g);
    }
};

// ---- activations in 8 bits ----------------------------------------------------------------------------------------------------------
constexpr int64_t kBlock = 32;

std::tuple<Tensor, Tensor> pack8(const Tensor& x_) {
    const Tensor x = activation(x_, "x");
    if (x.dim() < 1) value_error("x has to have a feature axis");
    require_gpu(x);
    const c10::OptionalDeviceGuard guard(x.device());
    const int64_t width = x.size(-1);
    auto shape = x.sizes().vec();
    Tensor q = at::empty(shape, x.options().dtype(at::kChar));
    shape.back() = (width + kBlock - 1) / kBlock;
    Tensor e = at::empty(shape, x.options().dtype(at::kByte));
    if (x.numel()) {
        const Rows r(x);
        check(api.acx_act8_pack(r.p, r.stride, code_of(x.scalar_type()), x.numel() / width, width, ptr_as<int8_t>(q), ptr_as<uint8_t>(e), stream_of(x)), "acx_act8_pack");
    }
    return {q, e};
}
std::tuple<Tensor, Tensor> checkpoint(const Tensor& q_, const Tensor& e_) {
    const Tensor q = plain(q_, "q", q_.sizes(), q_.device(), at::kChar);
    if (q.dim() < 1) value_error("q has to have a feature axis");
    auto shape = q.sizes().vec();
    shape.back() = (shape.back() + kBlock - 1) / kBlock;
    return {q, plain(e_, "exponent", shape, q.device(), at::kByte)};
}
Tensor unpack8(const Tensor& q_, const Tensor& e_, at::ScalarType dtype) {
    if (code_of(dtype) < 0) type_error("dtype has to be float32, bfloat16 or float16, not " + type_text(dtype));
    const auto [q, e] = checkpoint(q_, e_);
    require_gpu(q);
    const c10::OptionalDeviceGuard guard(q.device());
    Tensor x = at::empty(q.sizes(), q.options().dtype(dtype));
    if (q.numel())
        check(api.acx_act8_unpack(ptr_as<int8_t>(q), ptr_as<uint8_t>(e), q.numel() / q.size(-1), q.size(-1), ptr(x), code_of(dtype), stream_of(q)), "acx_act8_unpack");
    return x;
}
std::tuple<Tensor, Tensor> weight_grad8(const Tensor& d_out_, const Tensor& q_, const Tensor& e_) {
    const Tensor d_out = activation(d_out_, "d_out");
    const auto [q, e] = checkpoint(q_, e_);
    if (d_out.dim() < 1 || d_out.dim() != q.dim() || d_out.sizes().slice(0, d_out.dim() - 1) != q.sizes().slice(0, q.dim() - 1) || d_out.device() != q.device())
        value_error("d_out " + shape_text(d_out.sizes()) + " on " + d_out.device().str() + " and q " + shape_text(q.sizes()) + " on " + q.device().str() + " do not have their rows in common");
    const int64_t outputs = d_out.size(-1), inputs = q.size(-1);
    if (outputs > 65536 || inputs > 65536 || outputs * inputs > (1 << 29)) value_error("up to 65536 outputs and inputs, 2^29 weights");
    require_gpu(d_out);
    const c10::OptionalDeviceGuard guard(d_out.device());
    const int64_t rows = inputs ? q.numel() / inputs : 0;
    if (!rows || !outputs)
        return {at::zeros({outputs, inputs}, d_out.options().dtype(at::kFloat)),
                outputs && d_out.numel() ? d_out.reshape({-1, outputs}).to(at::kFloat).sum(0) : at::zeros({outputs}, d_out.options().dtype(at::kFloat))};
    Tensor g = rows_of(d_out);
    if (rows > 1 && (g.stride(0) < outputs || g.stride(0) >= (1 << 24))) g = g.contiguous();  // (the expanded gradient of a sum over the rows, say)
    Tensor dw = floats({outputs, inputs}, d_out), db = floats({outputs}, d_out);
    Maybe work = scratch(api.acx_act8_workspace_bytes(rows, outputs, inputs), d_out);
    check(api.acx_act8_weight_grad(ptr(g), rows > 1 ? g.stride(0) : outputs, code_of(d_out.scalar_type()), ptr_as<int8_t>(q), ptr_as<uint8_t>(e), rows, outputs, inputs, ptr_as<float>(dw),
                                   ptr_as<float>(db), ptr(work), bytes_of(work), stream_of(d_out)),
          "acx_act8_weight_grad");
    return {dw, db};
}

// ---- a block over a rollout, and for one step ----------------------------------------------------------------------------------------
struct RecurrentBlock : torch::autograd::Function<RecurrentBlock> {
    static Tensor third(const Tensor& t, int64_t k) {
        const int64_t width = t.size(-1) / 3;
        return t.narrow(-1, k * width, width);
    }
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& projected, const Maybe& reset, const Maybe& state, const Maybe& weight, const Maybe& scale,
                                 const Maybe& next_weight, double eps, bool pack) {
        auto [hidden, last, bounds] = scan_forward(third(projected, 0), third(projected, 1), reset, state, true);
        auto [out, u, stats] = block_forward(x, hidden, third(projected, 2), weight, scale, next_weight, eps, true);
        Tensor kept = hidden, exponent;
        if (pack) std::tie(kept, exponent) = pack8(hidden);  // (autograd's hooks pack x and projected; hidden is nobody's input)
        ctx->save_for_backward({x, projected, orundef(reset), orundef(weight), orundef(scale), orundef(next_weight), *bounds, *stats, kept, exponent});
        ctx->saved_data["state"] = state.has_value() && state->requires_grad();
        ctx->set_materialize_grads(false);
        if (u) return {*out, last, *u};
        return {*out, last};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        variable_list out(9);
        const Tensor d_new = g[0], d_last = g[1], d_u = g.size() > 2 ? g[2] : Tensor();
        if (!d_new.defined() && !d_last.defined() && !d_u.defined()) return out;
        const auto s = ctx->get_saved_variables();
        {
            const at::NoGradGuard no_grad;
            const Tensor &x = s[0], &projected = s[1], hidden = s[9].defined() ? unpack8(s[8], s[9], x.scalar_type()) : s[8];
            Tensor d_projected = same(x, projected.sizes());
            auto [dx, dh, dg, dw, ds, dn] = block_backward(opt(d_new), opt(d_u), x, hidden, third(projected, 2), opt(s[3]), opt(s[4]), opt(s[5]), s[7], third(d_projected, 2));
            auto [dc, dz, d_state] = scan_backward(*dh, opt(d_last), third(projected, 0), third(projected, 1), opt(s[2]), s[6], ctx->saved_data["state"].toBool(), third(d_projected, 0),
                                                   third(d_projected, 1));
            out = {dx, d_projected, Tensor(), orundef(d_state), orundef(dw), orundef(ds), orundef(dn), Tensor(), Tensor()};
        }
        return once(std::move(out), g);
    }
};

std::tuple<Tensor, Maybe, Tensor> recurrent_step(const Tensor& x_, const Tensor& projected_, const Tensor& state_, const Maybe& weight, const Maybe& scale, const Maybe& next_weight, const Maybe& reset_,
                                                 const Maybe& next_state, double eps) {
    const Tensor x = activation(x_, "x");
    if (x.dim() != 2) value_error("x has to be [rows, features], not " + shape_text(x.sizes()));
    const int64_t rows = x.size(0), width = x.size(1);
    check_width(width, eps);
    const at::Device dev = x.device();
    const int64_t wide[2] = {rows, 3 * width};
    const Tensor projected = activation(projected_, "projected", &x, at::IntArrayRef(wide, 2)), state = plain(state_, "state", {rows, width}, dev);
    if (!weight) type_error("weight has to be a tensor, not NoneType");
    const Maybe w = plain(*weight, "weight", {width}, dev);
    Maybe s, n, reset;
    if (scale) s = plain(*scale, "scale", {width}, dev);
    if (next_weight) n = plain(*next_weight, "next_weight", {width}, dev);
    if (reset_) reset = flags(*reset_, "reset", {rows}, dev);
    if (next_state && !plain(*next_state, "next_state", {rows, width}, dev).is_same(*next_state)) value_error("next_state has to be contiguous");
    if (next_state) {
        const Maybe operands[] = {x, projected, state};
        require_apart(*next_state, "next_state", {&operands[0], &operands[1], &w, &s, &n, &reset});
        if (ptr(*next_state) != ptr(state)) require_apart(*next_state, "next_state", {&operands[2]});
    }
    require_gpu(x);
    const c10::OptionalDeviceGuard guard(dev);
    const Tensor next = next_state ? *next_state : floats({rows, width}, x);
    Tensor out = same(x, x.sizes());
    Maybe u;
    if (n) u = same(x, x.sizes());
    if (rows && width)
        check(api.acx_block_step(ptr(x), x.stride(0), ptr(projected), projected.stride(0), code_of(x.scalar_type()), ptr_as<uint8_t>(reset), ptr_as<float>(state), ptr_as<float>(w), ptr_as<float>(s),
                                 ptr_as<float>(n), (float)eps, rows, width, ptr_as<float>(next), ptr(out), ptr(u), stream_of(x)),
              "acx_block_step");
    if (next_state) count_change(next);
    return {out, u, next};
}

// ---- Python -------------------------------------------------------------------------------------------------------------------------
py::object wrap(const Tensor& t) { return py::reinterpret_steal<py::object>(THPVariable_Wrap(t)); }
py::object wrap(const Maybe& t) { return t ? wrap(*t) : py::none(); }
template <class... T> py::tuple wrap_all(const T&... t) { return py::make_tuple(wrap(t)...); }

// the operators' own work runs without the interpreter's lock (hooks on saved tensors take it themselves)
template <class F> auto unlocked(F&& f) {
    const py::gil_scoped_release release;
    return f();
}

}  // namespace

PYBIND11_MODULE(acx_torch, m) {
    using H = py::handle;
    m.def("bind", [](const py::dict& addresses, py::object acx_error) {
#define ACX_BIND(f) api.f = reinterpret_cast<decltype(api.f)>(addresses[#f].cast<uintptr_t>());
        ACX_FUNCTIONS(ACX_BIND)
        static PyObject* error = nullptr;
        error = acx_error.release().ptr();
        py::register_exception_translator([](std::exception_ptr p) {
            try {
                if (p) std::rethrow_exception(p);
            } catch (const AcxFailure& e) {
                PyErr_SetString(error, e.what());
            } catch (const NoForwardMode& e) {
                PyErr_SetString(PyExc_NotImplementedError, e.what());
            }
        });
    });
    m.def("gated_scan_forward", [](H c, H z, H r, H s, bool save) {
        const Tensor ct = tensor(c, "candidate"), zt = tensor(z, "gate");
        const Maybe rt = maybe(r, "reset"), st = maybe(s, "state");
        auto [hidden, last, bounds] = unlocked([&] { return scan_forward(ct, zt, rt, st, save); });
        return wrap_all(hidden, last, bounds);
    });
    m.def("gated_scan_backward", [](H dh, H dl, H c, H z, H r, H b, bool want_state, H dc, H dz) {
        const Tensor dht = tensor(dh, "d_hidden"), ct = tensor(c, "candidate"), zt = tensor(z, "gate"), bt = tensor(b, "bounds");
        const Maybe dlt = maybe(dl, "d_last"), rt = maybe(r, "reset"), dct = maybe(dc, "out[0]"), dzt = maybe(dz, "out[1]");
        auto [a, d, e] = unlocked([&] { return scan_backward(dht, dlt, ct, zt, rt, bt, want_state, dct, dzt); });
        return wrap_all(a, d, e);
    });
    m.def("gated_scan", [](H c, H z, H r, H s) {
        const Maybe ct = tensor(c, "candidate"), zt = tensor(z, "gate"), rt = maybe(r, "reset"), st = maybe(s, "state");
        auto out = unlocked([&]() -> variable_list {
            if (wants_grad({&ct, &zt, &st})) return GatedScan::apply(*ct, *zt, rt, st);
            auto [hidden, last, bounds] = scan_forward(*ct, *zt, rt, st, false);
            return {hidden, last};
        });
        return wrap_all(out[0], out[1]);
    });
    m.def("block_output_forward", [](H x, H y, H g, H w, H s, H n, double eps, bool save) {
        const Tensor xt = tensor(x, "x");
        const Maybe yt = maybe(y, "y"), gt = maybe(g, "gate"), wt = maybe(w, "weight"), st = maybe(s, "scale"), nt = maybe(n, "next_weight");
        auto [a, b, c] = unlocked([&] { return block_forward(xt, yt, gt, wt, st, nt, eps, save); });
        return wrap_all(a, b, c);
    });
    m.def("block_output_backward", [](H dn, H du, H x, H y, H g, H w, H s, H n, H stats, H dg) {
        const Tensor xt = tensor(x, "x"), stt = tensor(stats, "stats");
        const Maybe dnt = maybe(dn, "d_new"), dut = maybe(du, "d_u"), yt = maybe(y, "y"), gt = maybe(g, "gate"), wt = maybe(w, "weight"), st = maybe(s, "scale"), nt = maybe(n, "next_weight"),
                    dgt = maybe(dg, "d_gate_out");
        auto [a, b, c, d, e, f] = unlocked([&] { return block_backward(dnt, dut, xt, yt, gt, wt, st, nt, stt, dgt); });
        return wrap_all(a, b, c, d, e, f);
    });
    m.def("block_output", [](H x, H y, H g, H w, H s, H n, double eps) {
        const Maybe xt = tensor(x, "x"), yt = maybe(y, "y"), gt = maybe(g, "gate"), wt = maybe(w, "weight"), st = maybe(s, "scale"), nt = maybe(n, "next_weight");
        Maybe out, u, stats;
        unlocked([&] {
            if (wants_grad({&xt, &yt, &gt, &wt, &st, &nt})) {
                auto r = BlockOutput::apply(*xt, yt, gt, wt, st, nt, eps);
                size_t k = 0;
                if (yt) out = r[k++];
                if (nt) u = r[k++];
            } else {
                std::tie(out, u, stats) = block_forward(*xt, yt, gt, wt, st, nt, eps, false);
            }
        });
        return wrap_all(out, u);
    });
    m.def("recurrent_block", [](H x, H p, H r, H st, H w, H s, H n, double eps, bool pack) {
        const Maybe xt = tensor(x, "x"), pt = tensor(p, "projected"), rt = maybe(r, "reset"), stt = maybe(st, "state"), wt = tensor(w, "weight"), sct = maybe(s, "scale"),
                    nt = maybe(n, "next_weight");
        if (xt->dim() != 3) value_error("x has to be [steps, rows, features]");
        auto wide = xt->sizes().vec();
        wide.back() *= 3;
        const Tensor xa = activation(*xt, "x");
        activation(*pt, "projected", &xa, at::IntArrayRef(wide));
        Maybe out, u, last, bounds, stats, hidden;
        unlocked([&] {
            if (wants_grad({&xt, &pt, &stt, &wt, &sct, &nt})) {
                auto v = RecurrentBlock::apply(*xt, *pt, rt, stt, wt, sct, nt, eps, pack);
                out = v[0], last = v[1];
                if (nt) u = v[2];
            } else {
                std::tie(hidden, last, bounds) = scan_forward(RecurrentBlock::third(*pt, 0), RecurrentBlock::third(*pt, 1), rt, stt, false);
                std::tie(out, u, stats) = block_forward(*xt, hidden, RecurrentBlock::third(*pt, 2), wt, sct, nt, eps, false);
            }
        });
        return wrap_all(out, u, last);
    });
    m.def("recurrent_step", [](H x, H p, H st, H w, H s, H n, H r, H ns, double eps) {
        const Tensor xt = tensor(x, "x"), pt = tensor(p, "projected"), stt = tensor(st, "state");
        const Maybe wt = maybe(w, "weight"), sct = maybe(s, "scale"), nt = maybe(n, "next_weight"), rt = maybe(r, "reset"), nst = maybe(ns, "next_state");
        const at::NoGradGuard no_grad;
        auto [a, b, c] = recurrent_step(xt, pt, stt, wt, sct, nt, rt, nst, eps);
        return py::make_tuple(wrap(a), wrap(b), ns.is_none() ? wrap(c) : py::reinterpret_borrow<py::object>(ns));
    });
    m.def("once", [](const py::sequence& grads, H from) {  // (of a backward pass in Python: a tuple of tensors and None)
        variable_list g;
        for (H t : grads) g.push_back(orundef(maybe(t, "a gradient")));
        g = once(std::move(g), {tensor(from, "d_out")});
        py::tuple out(g.size());
        for (size_t k = 0; k < g.size(); k++) out[k] = wrap(opt(g[k]));
        return out;
    });
    m.def("pack8", [](H x) {
        const Tensor xt = tensor(x, "x");
        const at::NoGradGuard no_grad;
        auto [q, e] = pack8(xt);
        return wrap_all(q, e);
    });
    m.def("unpack8", [](H q, H e, H dtype) {
        const Tensor qt = tensor(q, "q"), et = tensor(e, "exponent");
        const at::NoGradGuard no_grad;
        return wrap(unpack8(qt, et, reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type));
    });
    m.def("weight_grad8", [](H d, H q, H e) {
        const Tensor dt = tensor(d, "d_out"), qt = tensor(q, "q"), et = tensor(e, "exponent");
        const at::NoGradGuard no_grad;
        auto [dw, db] = weight_grad8(dt, qt, et);
        return wrap_all(dw, db);
    });
}
