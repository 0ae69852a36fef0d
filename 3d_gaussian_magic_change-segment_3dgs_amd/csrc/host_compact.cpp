// host_compact.cpp -- the host side of the compact-scene operators in C++ (part of the torch
// extension "gsr_host"): allocation, the libgsr calls of include/gsr_compact.h and the autograd
// functions, as gsr_train/compact.py does them over ctypes, with its checks and messages: small calls
// are bound by the host (10k Gaussians: colours 18 us through Python and ctypes, 3 us on the GPU).
#include <torch/extension.h>
#include <ATen/TracerMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <cstdint>
#include <stdexcept>
#include <string>
#include <tuple>
#include <unordered_set>
#include <vector>

#include "gsr_compact.h"

namespace {

void check(int rc) {
    if (rc) throw std::runtime_error(gsr_last_error());
}
void* cur_stream() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }
using Guard = c10::hip::HIPGuardMasqueradingAsCUDA;

int64_t words(int64_t K) { return (K + 7) / 8; }
int64_t blocks(int64_t K) { return (K + GSR_MX_BLOCK - 1) / GSR_MX_BLOCK; }
at::TensorOptions like(const at::Tensor& t, at::ScalarType type) {
    return at::TensorOptions().dtype(type).device(t.device());
}
const uint32_t* code_ptr(const at::Tensor& t) { return reinterpret_cast<const uint32_t*>(t.data_ptr<uint8_t>()); }
uint32_t* code_out(at::Tensor& t) { return reinterpret_cast<uint32_t*>(t.data_ptr<uint8_t>()); }

}  // namespace

namespace {

[[noreturn]] void refuse(const std::string& text) { throw std::runtime_error(text); }

void check_float(const char* what, const char* name, const at::Tensor& t) {
    if (t.scalar_type() != at::kFloat)
        refuse(std::string(what) + ": " + name + " must be a torch.float32 tensor (got " +
               c10::toString(t.scalar_type()) + ")");
}
void check_gpu(const char* what, const at::Tensor& t) {
    if (!t.is_cuda()) refuse(std::string(what) + ": tensors must be on the GPU (the HIP path has no CPU fallback)");
}
void check_device(const char* what, const char* name, const at::Tensor& t, const at::Tensor& first) {
    if (t.device() != first.device())
        refuse(std::string(what) + ": " + name + " is on " + t.device().str() + ", expected " + first.device().str());
}

// A tracer would record the allocations and not the kernels: what it made would return uninitialised memory.
bool jit_traced() { return at::tracer::impl::is_dispatch_enabled(); }
bool fx_traced() {
    using namespace c10::impl;
    return TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY).has_value();
}
void check_traced(const char* what, bool traced = jit_traced() || fx_traced()) {
    if (traced) refuse(std::string(what) + ": cannot be traced");
}

// A write through the pointer, which autograd has to know of.
void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// (the library takes a width as an int)
void check_width(const char* what, int64_t K) {
    if (K > GSR_MAX_WIDTH) refuse(std::string(what) + ": rows of more than 2^20 values");
}

}  // namespace

std::tuple<at::Tensor, at::Tensor> mx4_quantize(const at::Tensor& rows) {
    check_traced("mx4_quantize");
    check_float("mx4_quantize", "x", rows);
    if (rows.dim() != 2) refuse("mx4_quantize: x must have shape (rows, values)");
    if (rows.size(0)) check_width("mx4_quantize", rows.size(1));
    check_gpu("mx4_quantize", rows);
    Guard guard(rows.device());
    const bool apart = rows.numel() && ((rows.size(1) > 1 && rows.stride(1) != 1) ||
                                        (rows.size(0) > 1 && rows.stride(0) < rows.size(1)));
    const at::Tensor x = apart ? rows.contiguous() : rows;
    const int64_t R = x.size(0), K = x.size(1);
    at::Tensor codes = at::empty({R, 4 * words(K)}, like(x, at::kByte));
    at::Tensor scales = at::empty({R, blocks(K)}, like(x, at::kByte));
    if (R && K)
        check(gsr_mx4_quantize(R, (int)K, x.data_ptr<float>(), x.stride(0), code_out(codes),
                               scales.data_ptr<uint8_t>(), cur_stream()));
    return {codes, scales};
}

at::Tensor mx4_dequantize(const at::Tensor& codes, const at::Tensor& scales, int64_t K) {
    check_traced("MX4Rows.dequantize");
    if (codes.size(0)) check_width("MX4Rows.dequantize", K);
    check_gpu("MX4Rows.dequantize", codes);
    Guard guard(codes.device());
    at::Tensor x = at::empty({codes.size(0), K}, like(codes, at::kFloat));
    if (x.numel())
        check(gsr_mx4_dequantize(codes.size(0), (int)K, code_ptr(codes), scales.data_ptr<uint8_t>(),
                                 x.data_ptr<float>(), cur_stream()));
    return x;
}

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

at::Tensor colors_for(const at::Tensor& xyz, int64_t V, bool single) {
    const int64_t P = xyz.size(0);
    return single ? at::empty({P, 3}, like(xyz, at::kFloat)) : at::empty({V, P, 3}, like(xyz, at::kFloat));
}

at::Tensor colors_of(const at::Tensor& xyz, const at::Tensor& dc, const at::Tensor& campos, const at::Tensor& codes,
                     const at::Tensor& scales, int64_t degree, int64_t M, bool single, at::Tensor* mask) {
    const int64_t P = xyz.size(0), V = campos.size(0);
    at::Tensor colors = colors_for(xyz, V, single);
    if (mask) *mask = at::empty({V, P}, like(xyz, at::kByte));
    if (P)
        check(gsr_sh_colors((int)P, (int)V, (int)degree, (int)M, xyz.data_ptr<float>(), dc.data_ptr<float>(),
                            dc.stride(0), code_ptr(codes), scales.data_ptr<uint8_t>(), campos.data_ptr<float>(),
                            colors.data_ptr<float>(), mask ? mask->data_ptr<uint8_t>() : nullptr, cur_stream()));
    return colors;
}

// scales and mask: defined, or behind the codes in one buffer (quantized_of).
void keep(AutogradContext* ctx, const at::Tensor& xyz, const at::Tensor& campos, const at::Tensor& codes,
          const at::Tensor& scales, const at::Tensor& mask, int64_t degree, int64_t M) {
    if (scales.defined()) ctx->save_for_backward({xyz, campos, codes, scales, mask});
    else ctx->save_for_backward({xyz, campos, codes});
    ctx->saved_data["degree"] = degree;
    ctx->saved_data["M"] = M;
}

// Stands for the derivative of a gradient.  Its edges lead to what the gradient is a function of, so that every
// backward pass towards one of those, grad() of a single input too, comes through here and is refused.
struct NoSecondDerivative : torch::autograd::Node {
    variable_list apply(variable_list&&) override {
        throw std::runtime_error("sh_colors: trying to differentiate twice (the colours are once_differentiable)");
    }
    std::string name() const override { return "NoSecondDerivative"; }
};

void once_differentiable(at::Tensor& gradient, const std::vector<torch::autograd::Edge>& of) {
    torch::autograd::edge_list edges;
    for (const auto& e : of)
        if (e.is_valid()) edges.push_back(e);
    if (!gradient.defined() || edges.empty()) return;  // a constant
    std::shared_ptr<torch::autograd::Node> node(new NoSecondDerivative, torch::autograd::deleteNode);
    node->set_next_edges(std::move(edges));
    torch::autograd::set_history(gradient, node);
}

// The gradients wanted of (dxyz, ddc or dfeatures); a second derivative is refused when it is taken.
variable_list gradients(AutogradContext* ctx, const at::Tensor& g_in, bool features) {
    const auto sv = ctx->get_saved_variables();
    const at::Tensor &xyz = sv[0], &campos = sv[1], &codes = sv[2];
    const int64_t P = xyz.size(0), M = ctx->saved_data["M"].toInt(), degree = ctx->saved_data["degree"].toInt();
    const bool apart = sv.size() > 3;
    const uint8_t* scales = apart ? sv[3].data_ptr<uint8_t>() : codes.data_ptr<uint8_t>() + P * 4 * words(3 * (M - 1));
    const uint8_t* mask = apart ? sv[4].data_ptr<uint8_t>() : scales + P * blocks(3 * (M - 1));
    Guard guard(xyz.device());
    variable_list out(2);
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const at::Tensor g = g_in.contiguous();
        if (ctx->needs_input_grad(0)) out[0] = at::empty({P, 3}, like(xyz, at::kFloat));
        if (ctx->needs_input_grad(1))
            out[1] = features ? at::empty({P, M, 3}, like(xyz, at::kFloat)) : at::empty({P, 3}, like(xyz, at::kFloat));
        float* second = out[1].defined() ? out[1].data_ptr<float>() : nullptr;
        if (P)
            check(gsr_sh_colors_backward((int)P, (int)campos.size(0), (int)degree, (int)M, xyz.data_ptr<float>(),
                                         code_ptr(codes), scales, campos.data_ptr<float>(), mask, g.data_ptr<float>(),
                                         out[0].defined() ? out[0].data_ptr<float>() : nullptr,
                                         features ? nullptr : second, features ? second : nullptr, cur_stream()));
    }
    if (at::GradMode::is_enabled()) {
        // dxyz is a function of the upstream gradient, the positions and the coefficients above the constant one (and 0
        // at degree 0); ddc is one of the upstream gradient alone, dfeatures of the positions too (straight through the
        // rounding: not of the features).
        const auto node = torch::autograd::get_current_node();
        const torch::autograd::Edge up = torch::autograd::impl::gradient_edge(g_in);
        const torch::autograd::Edge place = degree > 0 ? node->next_edge(0) : torch::autograd::Edge();
        if (degree > 0) {
            if (features) once_differentiable(out[0], {up, place, node->next_edge(1)});
            else once_differentiable(out[0], {up, place});
        }
        if (features) once_differentiable(out[1], {up, place});
        else once_differentiable(out[1], {up});
    }
    return out;
}

struct ShColorsFn : public torch::autograd::Function<ShColorsFn> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& xyz, const at::Tensor& dc,
                              const at::Tensor& campos, const at::Tensor& codes, const at::Tensor& scales,
                              int64_t degree, int64_t M, bool single) {
        at::Tensor mask;
        at::Tensor colors = colors_of(xyz, dc, campos, codes, scales, degree, M, single, &mask);
        keep(ctx, xyz, campos, codes, scales, mask, degree, M);
        return colors;
    }
    static variable_list backward(AutogradContext* ctx, variable_list go) {
        const variable_list g = gradients(ctx, go[0], false);
        return {g[0], g[1], {}, {}, {}, {}, {}, {}};
    }
};

// What the backward needs of a call goes into one buffer: the codes, the scales, the mask.
at::Tensor quantized_of(const at::Tensor& xyz, const at::Tensor& features, const at::Tensor& campos, int64_t degree,
                        bool single, at::Tensor& held) {
    const int64_t P = xyz.size(0), V = campos.size(0), M = features.size(1), K = 3 * (M - 1);
    held = at::empty({P * (4 * words(K) + blocks(K) + V)}, like(xyz, at::kByte));
    at::Tensor colors = colors_for(xyz, V, single);
    if (P) {
        uint8_t* codes = held.data_ptr<uint8_t>();
        uint8_t* scales = codes + P * 4 * words(K);
        check(gsr_sh_colors_quantize((int)P, (int)V, (int)degree, (int)M, xyz.data_ptr<float>(),
                                     features.data_ptr<float>(), campos.data_ptr<float>(),
                                     reinterpret_cast<uint32_t*>(codes), scales, scales + P * blocks(K),
                                     colors.data_ptr<float>(), cur_stream()));
    }
    return colors;
}

struct ShColorsQuantizedFn : public torch::autograd::Function<ShColorsQuantizedFn> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& xyz, const at::Tensor& features,
                              const at::Tensor& campos, int64_t degree, bool single) {
        at::Tensor held;
        at::Tensor colors = quantized_of(xyz, features, campos, degree, single, held);
        keep(ctx, xyz, campos, held, {}, {}, degree, features.size(1));
        return colors;
    }
    static variable_list backward(AutogradContext* ctx, variable_list go) {
        const variable_list g = gradients(ctx, go[0], true);
        return {g[0], g[1], {}, {}, {}};
    }
};

// In a capture, every node that the gradients will flow through has to belong to the capturing stream: the
// backward pass would make another node's stream wait for it, which breaks the capture beyond repair.  Such
// nodes are an eager graph's: one that the inputs come from, or the accumulators of the same leaves, which live
// as long as any graph of them.
void check_capture(const char* what, const at::Tensor& a, const at::Tensor& b) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    const auto here = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA();
    if (hipStreamIsCapturing(here.stream(), &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;
    std::vector<std::shared_ptr<torch::autograd::Node>> todo;
    std::unordered_set<torch::autograd::Node*> seen;
    for (const at::Tensor* t : {&a, &b}) {
        if (!t->requires_grad()) continue;
        auto node = t->grad_fn() ? t->grad_fn() : torch::autograd::impl::try_get_grad_accumulator(*t);
        if (node && seen.insert(node.get()).second) todo.push_back(node);
    }
    while (!todo.empty()) {
        const auto node = todo.back();
        todo.pop_back();
        const auto stream = node->stream();
        if (stream && *stream != here.unwrap())
            refuse(std::string(what) + ": captured while an eager graph of the same tensors is alive (" + node->name() +
                   " is on another stream): drop it, or make it in the capture");
        for (const auto& e : node->next_edges())
            if (e.function && seen.insert(e.function.get()).second) todo.push_back(e.function);
    }
}

// A tangent on an input would be lost: refused, as autograd refuses it for a function without a forward-mode form.
void check_forward(const char* what, std::initializer_list<const at::Tensor*> inputs) {
    for (const at::Tensor* t : inputs)
        if (t->_fw_grad(0).defined()) refuse(std::string(what) + ": there is no forward-mode derivative");
}

bool wanted(const char* what, const at::Tensor& a, const at::Tensor& b) {
    const bool yes = at::GradMode::is_enabled() && (a.requires_grad() || b.requires_grad());
    if (yes) check_capture(what, a, b);
    return yes;
}

}  // namespace

namespace {
void check_sh(const char* what, const at::Tensor& xyz, const at::Tensor& campos, int64_t degree, int64_t M) {
    check_float(what, "xyz", xyz);
    check_float(what, "campos", campos);
    if (xyz.dim() != 2 || xyz.size(1) != 3 || xyz.size(0) >= (1LL << 31))
        refuse(std::string(what) + ": xyz must have shape (P, 3), P below 2^31");
    const bool one = campos.dim() == 1 && campos.size(0) == 3;
    const bool many = campos.dim() == 2 && campos.size(1) == 3 && campos.size(0) >= 1 && campos.size(0) <= GSR_MAX_VIEWS;
    if (!one && !many)
        refuse(std::string(what) + ": campos must have shape (3,) or (V, 3) with V of 1.." + std::to_string(GSR_MAX_VIEWS));
    if (degree < 0 || degree > 3 || (degree + 1) * (degree + 1) > M)
        refuse(std::string(what) + ": degree must be 0..3 and the features must hold its coefficients (degree " +
               std::to_string(degree) + ", " + std::to_string(M) + " coefficients)");
}
at::Tensor views_of(const at::Tensor& campos) {
    const at::Tensor c = campos.requires_grad() ? campos.detach() : campos;
    return (c.dim() == 1 ? c.unsqueeze(0) : c).contiguous();
}
}  // namespace

at::Tensor sh_colors(const at::Tensor& xyz_, const at::Tensor& features_dc, const at::Tensor& codes,
                     const at::Tensor& scales, int64_t width, const at::Tensor& campos_, int64_t degree) {
    if (jit_traced()) return {};  // the caller's Python function, which the tracer records as a whole
    check_traced("sh_colors", fx_traced());
    if (width % 3 || width > 45) refuse("sh_colors: rest must be MX4Rows of 3 (M - 1) values, M of 1..16");
    const int64_t M = width / 3 + 1;
    check_sh("sh_colors", xyz_, campos_, degree, M);
    check_float("sh_colors", "features_dc", features_dc);
    const int64_t P = xyz_.size(0), dims = features_dc.dim();
    if (!((dims == 2 || (dims == 3 && features_dc.size(1) == 1)) && features_dc.size(0) == P &&
          features_dc.size(dims - 1) == 3))
        refuse("sh_colors: features_dc must have shape (" + std::to_string(P) + ", 1, 3) or (" + std::to_string(P) +
               ", 3)");
    if (codes.size(0) != P)
        refuse("sh_colors: rest must have " + std::to_string(P) + " rows (got " + std::to_string(codes.size(0)) + ")");
    check_gpu("sh_colors", xyz_);
    check_device("sh_colors", "features_dc", features_dc, xyz_);
    check_device("sh_colors", "rest", codes, xyz_);
    check_device("sh_colors", "campos", campos_, xyz_);
    check_forward("sh_colors", {&xyz_, &features_dc, &campos_});
    Guard guard(xyz_.device());
    const bool single = campos_.dim() == 1, grad = wanted("sh_colors", xyz_, features_dc);
    const at::Tensor xyz = xyz_.contiguous(), campos = views_of(campos_);
    at::Tensor dc = dims == 3 ? features_dc.squeeze(1) : features_dc;
    if (P && (dc.stride(1) != 1 || (P > 1 && dc.stride(0) < 3))) dc = dc.contiguous();
    if (grad) return ShColorsFn::apply(xyz, dc, campos, codes, scales, degree, M, single);
    return colors_of(xyz, dc, campos, codes, scales, degree, M, single, nullptr);
}

at::Tensor sh_colors_quantized(const at::Tensor& xyz_, const at::Tensor& features_, const at::Tensor& campos_,
                               int64_t degree) {
    const char* what = "sh_colors_quantized";
    if (jit_traced()) return {};  // (as sh_colors)
    check_traced(what, fx_traced());
    check_float(what, "features", features_);
    if (features_.dim() != 3 || features_.size(2) != 3 || features_.size(1) < 1 || features_.size(1) > 16)
        refuse(std::string(what) + ": features must have shape (P, M, 3), M of 1..16");
    check_sh(what, xyz_, campos_, degree, features_.size(1));
    if (features_.size(0) != xyz_.size(0))
        refuse(std::string(what) + ": features must have " + std::to_string(xyz_.size(0)) + " rows (got " +
               std::to_string(features_.size(0)) + ")");
    check_gpu(what, xyz_);
    check_device(what, "features", features_, xyz_);
    check_device(what, "campos", campos_, xyz_);
    check_forward(what, {&xyz_, &features_, &campos_});
    Guard guard(xyz_.device());
    const bool single = campos_.dim() == 1, grad = wanted(what, xyz_, features_);
    const at::Tensor xyz = xyz_.contiguous(), features = features_.contiguous(), campos = views_of(campos_);
    if (grad) return ShColorsQuantizedFn::apply(xyz, features, campos, degree, single);
    at::Tensor held;
    return quantized_of(xyz, features, campos, degree, single, held);
}

void accumulate_weights(const at::Tensor& acc, const at::Tensor& weights, double decay) {
    const char* what = "accumulate_weights";
    check_traced(what);
    check_float(what, "acc", acc);
    check_float(what, "weights", weights);
    const int64_t P = acc.numel();
    if (P >= (1LL << 31)) refuse("accumulate_weights: at most 2^31 - 1 weights");
    if (!acc.is_contiguous() || weights.dim() != 1 || weights.size(0) != P)
        refuse("accumulate_weights: acc must be contiguous and weights have shape (P,), P values each");
    check_gpu(what, acc);
    check_device(what, "weights", weights, acc);
    Guard guard(acc.device());
    if (!P) return;
    check(gsr_accumulate_weights((int)P, weights.data_ptr<float>(), weights.stride(0), (float)decay,
                                 acc.data_ptr<float>(), cur_stream()));
    written(acc);
}

at::Tensor keep_heaviest(const at::Tensor& weights, const std::vector<std::tuple<int, int, int, int>>& plan) {
    check_traced("keep_heaviest");
    Guard guard(weights.device());
    std::vector<gsr_keep_group> g;
    int64_t n = 0;
    for (const auto& [a, b, k, r] : plan) {
        g.push_back({a, b, k, r});
        n += k;
    }
    at::Tensor ids = at::empty({n}, like(weights, at::kInt));
    if (n) {
        const int P = (int)weights.numel();
        const int64_t bytes = (int64_t)gsr_keep_ws_bytes(P);
        at::Tensor ws = bytes ? at::empty({bytes}, like(weights, at::kByte)) : at::Tensor();
        check(gsr_keep_heaviest(P, weights.data_ptr<float>(), (int)g.size(), g.data(), ids.data_ptr<int>(),
                                bytes ? ws.data_ptr() : nullptr, cur_stream()));
    }
    return ids;
}

// compact.py _take: the tensors' checks, the outputs where none are given, one gsr_take_rows.
std::vector<at::Tensor> take_rows(const at::Tensor& ids, const std::vector<at::Tensor>& tensors,
                                  std::vector<at::Tensor> out, const std::vector<int>& pad, bool given) {
    check_traced("take_rows");
    const int64_t K = ids.size(0);
    auto fine = [&](const at::Tensor& t) {
        return (t.scalar_type() == at::kFloat || t.scalar_type() == at::kInt) && t.dim() >= 1 && t.is_contiguous() &&
               t.device() == ids.device() && t.size(0) < (1LL << 31);
    };
    auto bad = [&](const char* name, size_t n) {
        refuse("take_rows: " + std::string(name) + "[" + std::to_string(n) +
               "] must be a contiguous float32 or int32 tensor of rows on " + ids.device().str());
    };
    Guard guard(ids.device());
    std::vector<gsr_rows> table;
    table.reserve(tensors.size());
    for (size_t n = 0; n < tensors.size(); ++n) {
        const at::Tensor& t = tensors[n];
        if (!fine(t)) bad("tensors", n);
        int64_t width = 1;
        for (int64_t d = 1; d < t.dim(); ++d) width *= t.size(d);
        check_width("take_rows", width);
        if (!given) {
            std::vector<int64_t> shape = t.sizes().vec();
            shape[0] = K;
            out.push_back(at::empty(shape, t.options().requires_grad(false)));
        } else {
            const at::Tensor& o = out[n];
            if (!fine(o)) bad("out", n);
            if (o.scalar_type() != t.scalar_type() || o.size(0) != K || o.sizes().slice(1) != t.sizes().slice(1))
                refuse("take_rows: out[" + std::to_string(n) + "] must be " + c10::toString(t.scalar_type()) + " of " +
                       std::to_string(K) + " rows like tensors[" + std::to_string(n) + "]");
        }
        table.push_back({t.data_ptr(), out[n].data_ptr(), (int)width, (int)t.size(0), pad.empty() ? 0 : pad[n]});
    }
    if (!table.empty()) check(gsr_take_rows((int)K, ids.data_ptr<int>(), (int)table.size(), table.data(), cur_stream()));
    if (given)
        for (const at::Tensor& o : out) written(o);
    return out;
}

void bind_compact(pybind11::module_& mod) {
    namespace py = pybind11;
    mod.def("mx4_quantize", &mx4_quantize, py::call_guard<py::gil_scoped_release>());
    mod.def("mx4_dequantize", &mx4_dequantize, py::call_guard<py::gil_scoped_release>());
    mod.def("sh_colors", &sh_colors, py::call_guard<py::gil_scoped_release>());
    mod.def("sh_colors_quantized", &sh_colors_quantized, py::call_guard<py::gil_scoped_release>());
    mod.def("accumulate_weights", &accumulate_weights, py::call_guard<py::gil_scoped_release>());
    mod.def("keep_heaviest", &keep_heaviest, py::call_guard<py::gil_scoped_release>());
    mod.def("take_rows", &take_rows, py::call_guard<py::gil_scoped_release>());
}
