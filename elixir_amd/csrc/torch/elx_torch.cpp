// Autograd of layer_norm and embedding over the C ABI of libelx_ops.so (include/elx_ops.h), as a Python extension, and the
// reading of 8-bit moments, which a program may ask of many small tensors in turn.
//
// A backward pass runs on torch's own thread for the device.  A Python function called from there has to wait for the
// interpreter to change threads and then spends tens of microseconds on its bookkeeping, more than many of these kernels
// take: a training pass through a layer norm took 140 us of host time with the same steps written in Python, two thirds
// of it in backward.  No kernel lives here.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/autograd.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include "elx_ops.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kMaxTokens = 1ll << 26, kMaxRows = 1ll << 30, kMaxCols = 1ll << 20, kMaxElems = 1ll << 34;    // of elx_embedding_*

void check(const char *func, int code) { TORCH_CHECK(code == 0, func, " failed with code ", code); }

int code_of(const Tensor &t) {
    return t.scalar_type() == at::kFloat ? ELX_F32 : t.scalar_type() == at::kHalf ? ELX_F16 : t.scalar_type() == at::kBFloat16 ? ELX_BF16 : ELX_NONE;
}

void *stream_of(const Tensor &t) {
    return (void *)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

// NULL for a tensor that is not there -- and for no other: a tensor without memory of its own (a wrapper) is refused
void *ptr(const Tensor &t) {
    if (!t.defined()) return nullptr;
    void *p = t.data_ptr();
    TORCH_CHECK(p || t.numel() == 0, "a tensor without memory");
    return p;
}

// A transform that would see the allocations of a call but not its launches must not record it.
void check_transforms(const char *name, std::initializer_list<const Tensor *> tensors) {
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing() &&
                                    !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(),
                                name, " cannot be traced");
    for (const Tensor *t : tensors)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), name, " has no forward-mode derivative");
}

// `x` as rows of `cols` elements: the tensor to read them from and the distance of two rows.  A tensor whose rows do not
// lie at one distance, or whose elements do not lie side by side, is copied.
std::pair<Tensor, int64_t> rows_of(const Tensor &any, int64_t cols) {
    const Tensor x = any.resolve_neg();
    if (x.is_contiguous()) return {x, cols};
    const int64_t dims = x.dim();
    if (dims >= 1 && x.size(-1) == cols && (x.stride(-1) == 1 || cols == 1)) {
        int64_t step = 0, expect = 0;
        bool even = true;
        for (int64_t d = dims - 2; d >= 0; --d) {    // from the innermost row dimension out
            if (x.size(d) == 1) continue;
            if (expect == 0) {
                step = x.stride(d);
                even = step >= cols;
            } else {
                even = x.stride(d) == expect;
            }
            if (!even) break;
            expect = x.stride(d) * x.size(d);
        }
        if (even) return {x, step == 0 ? cols : step};
    }
    return {x.contiguous(), cols};
}

Tensor packed(const Tensor &t) { return t.defined() ? t.resolve_neg().contiguous() : t; }

// What a hook on the saved tensors hands back is laid out as what it was given.
void check_saved(const char *name, const Tensor &t, c10::ScalarType type, const c10::Device &device, int64_t numel) {
    TORCH_CHECK(t.scalar_type() == type && t.device() == device && t.numel() == numel, name, ": a saved tensor came back as ", t.numel(),
                " elements of ", c10::getDtypeNames(t.scalar_type()).first, " on ", t.device());
}

void check_devices(const char *name, const Tensor &first, const Tensor &other) {
    if (!other.defined()) return;
    TORCH_CHECK(other.is_cuda(), name, " runs on the GPU: its tensors must live in device memory");
    TORCH_CHECK(other.device() == first.device(), name, ": tensors on ", first.device(), " and ", other.device());
}

void check_types(const char *name, const Tensor &first, const Tensor &other) {
    TORCH_CHECK_TYPE(code_of(first) != ELX_NONE, name, " takes float32, float16 or bfloat16, not ", c10::getDtypeNames(first.scalar_type()).first);
    if (other.defined())
        TORCH_CHECK_TYPE(other.scalar_type() == first.scalar_type(), name, ": tensors of ", c10::getDtypeNames(first.scalar_type()).first, " and ",
                         c10::getDtypeNames(other.scalar_type()).first);
}

// ------------------------------------------------------------------------------------------------------------ layer norm

Tensor layer_norm_forward(const Tensor &x, const Tensor &weight, const Tensor &bias, int64_t cols, double eps, const Tensor &stats) {
    Tensor y = at::empty(x.sizes(), x.options());
    const int64_t rows = x.numel() / cols;
    if (rows == 0) return y;
    const auto [src, stride] = rows_of(x, cols);
    const Tensor w = packed(weight), b = packed(bias);
    float *mean = stats.defined() ? stats.data_ptr<float>() : nullptr;
    check("elx_layer_norm_fwd", elx_layer_norm_fwd(ptr(src), ptr(w), ptr(b), ptr(y), mean, mean ? mean + rows : nullptr, rows,
                                                   (uint32_t)cols, stride, (float)eps, code_of(x), stream_of(x)));
    return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const std::optional<Tensor> &weight_, const std::optional<Tensor> &bias_,
                          int64_t dims, int64_t cols, double eps) {
        const Tensor weight = weight_.value_or(Tensor()), bias = bias_.value_or(Tensor());
        const Tensor stats = at::empty({2, x.numel() / cols}, x.options().dtype(at::kFloat));    // mean and rstd of every row
        ctx->save_for_backward({x, weight, stats});
        ctx->saved_data["dims"] = dims;
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["affine"] = (int64_t)(weight.defined() ? 1 : 0) | (bias.defined() ? 2 : 0);
        return layer_norm_forward(x, weight, bias, cols, eps, stats);
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], stats = packed(saved[2]);
        const Tensor &grad = grads[0];
        const int64_t dims = ctx->saved_data["dims"].toInt(), affine = ctx->saved_data["affine"].toInt();
        const c10::DeviceGuard guard(grad.device());
        const auto shape = grad.sizes().slice(grad.dim() - dims);
        check_saved("layer_norm", x, grad.scalar_type(), grad.device(), grad.numel());
        if (weight.defined()) check_saved("layer_norm", weight, grad.scalar_type(), grad.device(), c10::multiply_integers(shape));
        TORCH_CHECK(x.sizes() == grad.sizes(), "layer_norm: a saved tensor came back in another shape");
        const int64_t cols = c10::multiply_integers(shape), rows = x.numel() / cols;
        check_saved("layer_norm", stats, at::kFloat, grad.device(), 2 * rows);
        size_t edge = 0;    // inputs that are not there have no edge
        const bool want_x = ctx->needs_input_grad(edge++);
        const bool want_w = (affine & 1) && ctx->needs_input_grad(edge++);
        const bool want_b = (affine & 2) && ctx->needs_input_grad(edge++);
        Tensor dx, dw, db;
        if (at::GradMode::is_enabled() || !grad.has_storage()) {    // to be differentiated, or many at once: torch's operators
            const bool create_graph = at::GradMode::is_enabled();
            const at::AutoGradMode record(true);
            // With respect to aliases: the saved tensors carry their history, and where one of them is an ancestor of the
            // other (one norm in two layers) the derivative would run on through it, a path that is the outer pass's.
            const Tensor a = x.view_as(x), w = weight.defined() ? weight.view_as(weight) : weight;
            const Tensor b = want_b ? at::zeros(shape, x.options()).requires_grad_() : Tensor();
            variable_list leaves;
            if (want_x) leaves.push_back(a);
            if (want_w) leaves.push_back(w);
            if (want_b) leaves.push_back(b);
            const Tensor y = at::layer_norm(a, shape, w, b, ctx->saved_data["eps"].toDouble());
            auto got = torch::autograd::grad({y}, leaves, {grad}, std::nullopt, create_graph);
            size_t i = 0;
            if (want_x) dx = got[i++];
            if (want_w) dw = got[i++];
            if (want_b) db = got[i++];
            return {dx, dw, db, Tensor(), Tensor(), Tensor()};
        }
        if (want_x) dx = at::empty(x.sizes(), x.options());
        if (want_w) dw = at::empty(shape, x.options());
        if (want_b) db = at::empty(shape, x.options());
        if (rows == 0) {
            if (want_w) dw.zero_();
            if (want_b) db.zero_();
        } else if (want_x || want_w || want_b) {
            const auto [src, x_stride] = rows_of(x, cols);
            const auto [dy, dy_stride] = rows_of(grad, cols);
            const Tensor w = packed(weight);
            Tensor workspace;
            const uint64_t bytes = want_w || want_b ? elx_layer_norm_bwd_workspace(rows, (uint32_t)cols) : 0;
            if (bytes) workspace = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
            const float *mean = stats.data_ptr<float>();
            check("elx_layer_norm_bwd",
                  elx_layer_norm_bwd(ptr(dy), ptr(src), ptr(w), mean, mean + rows, ptr(dx), ptr(dw), ptr(db), ptr(workspace),
                                     bytes, rows, (uint32_t)cols, dy_stride, x_stride, code_of(x), stream_of(x)));
        }
        return {dx, dw, db, Tensor(), Tensor(), Tensor()};
    }
};

Tensor layer_norm(const Tensor &input, const std::optional<Tensor> &weight_, const std::optional<Tensor> &bias_, double eps,
                  const std::optional<std::vector<int64_t>> &normalized_shape) {
    const Tensor weight = weight_.value_or(Tensor()), bias = bias_.value_or(Tensor());
    const at::IntArrayRef shape = normalized_shape    ? at::IntArrayRef(*normalized_shape)
                                  : weight.defined() ? weight.sizes()
                                  : bias.defined()   ? bias.sizes()
                                                     : input.sizes().slice(input.dim() ? input.dim() - 1 : 0);
    check_transforms("layer_norm", {&input, &weight, &bias});
    const int64_t dims = (int64_t)shape.size();
    TORCH_CHECK_VALUE(dims > 0 && dims <= input.dim() && input.sizes().slice(input.dim() - dims) == shape, "layer_norm over ", shape,
                      " of an input of shape ", input.sizes());
    TORCH_CHECK_VALUE(!weight.defined() || weight.sizes() == shape, "layer_norm: weight has shape ", weight.sizes(), ", not ", shape);
    TORCH_CHECK_VALUE(!bias.defined() || bias.sizes() == shape, "layer_norm: bias has shape ", bias.sizes(), ", not ", shape);
    check_devices("layer_norm", input, input);
    check_devices("layer_norm", input, weight);
    check_devices("layer_norm", input, bias);
    check_types("layer_norm", input, weight);
    check_types("layer_norm", input, bias);
    const int64_t cols = c10::multiply_integers(shape), most = elx_layer_norm_max_cols();
    TORCH_CHECK_VALUE(cols >= 1 && cols <= most, "layer_norm takes rows of 1 to ", most, " elements, not ", cols);
    const c10::DeviceGuard guard(input.device());
    if (at::GradMode::is_enabled() &&
        (input.requires_grad() || (weight.defined() && weight.requires_grad()) || (bias.defined() && bias.requires_grad())))
        return LayerNorm::apply(input, weight_, bias_, dims, cols, eps);
    return layer_norm_forward(input, weight, bias, cols, eps, Tensor());
}

// ------------------------------------------------------------------------------------------------------------- embedding

Tensor embedding_forward(const Tensor &index, const Tensor &table, double scale) {
    auto shape = index.sizes().vec();
    shape.push_back(table.size(1));
    Tensor y = at::empty(shape, table.options());
    if (y.numel() == 0) return y;
    const Tensor t = packed(table);
    check("elx_embedding_fwd", elx_embedding_fwd(index.data_ptr(), (int)index.element_size(), index.numel(), t.data_ptr(), t.size(0),
                                                 (uint32_t)t.size(1), (float)scale, y.data_ptr(), code_of(t), stream_of(t)));
    return y;
}

struct Embedding : torch::autograd::Function<Embedding> {
    static Tensor forward(AutogradContext *ctx, const Tensor &index, const Tensor &table, int64_t padding, double scale) {
        ctx->save_for_backward({index});
        ctx->saved_data["table"] = at::empty({0}, table.options());    // type and device; the table itself is not kept
        ctx->saved_data["wide"] = index.scalar_type() == at::kLong;
        ctx->saved_data["rows"] = table.size(0);
        ctx->saved_data["cols"] = table.size(1);
        ctx->saved_data["padding"] = padding;
        ctx->saved_data["scale"] = scale;
        return embedding_forward(index, table, scale);
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const Tensor index = ctx->get_saved_variables()[0].contiguous();
        const Tensor &grad = grads[0];
        const auto options = ctx->saved_data["table"].toTensor().options();
        const int64_t rows = ctx->saved_data["rows"].toInt(), cols = ctx->saved_data["cols"].toInt();
        const int64_t padding = ctx->saved_data["padding"].toInt();
        const double scale = ctx->saved_data["scale"].toDouble();
        const c10::DeviceGuard guard(grad.device());
        TORCH_CHECK(cols == 0 || index.numel() == grad.numel() / cols, "embedding: a saved tensor came back in another shape");
        check_saved("embedding", index, ctx->saved_data["wide"].toBool() ? at::kLong : at::kInt, grad.device(), index.numel());
        if (at::GradMode::is_enabled() || !grad.has_storage()) {    // to be differentiated, or many at once: torch's operators
            const bool create_graph = at::GradMode::is_enabled();
            const at::AutoGradMode record(true);
            const Tensor inside = index.ge(0).logical_and(index.lt(rows));
            const Tensor table = at::zeros({rows, cols}, options).requires_grad_();
            const Tensor y = at::embedding(table, index.where(inside, at::zeros_like(index)), padding);
            const Tensor dy = (grad * scale).masked_fill(inside.logical_not().unsqueeze(-1), 0);
            return {Tensor(), torch::autograd::grad({y}, {table}, {dy}, std::nullopt, create_graph)[0], Tensor(), Tensor()};
        }
        Tensor dtable = at::empty({rows, cols}, options);
        const int64_t n = index.numel();
        if (n == 0 || dtable.numel() == 0) return {Tensor(), dtable.zero_(), Tensor(), Tensor()};
        const auto [dy, stride] = rows_of(grad, cols);
        const uint64_t bytes = elx_embedding_bwd_workspace(n, rows, (uint32_t)cols);
        const Tensor workspace = at::empty({(int64_t)bytes}, options.dtype(at::kByte));
        check("elx_embedding_bwd",
              elx_embedding_bwd(index.data_ptr(), (int)index.element_size(), n, dy.data_ptr(), stride, dtable.data_ptr(), rows,
                                (uint32_t)cols, (float)scale, padding, workspace.data_ptr(), bytes, code_of(dtable), stream_of(index)));
        return {Tensor(), dtable, Tensor(), Tensor()};
    }
};

Tensor embedding(const Tensor &input, const Tensor &weight, const std::optional<int64_t> &padding_idx, double scale) {
    check_transforms("embedding", {&weight});
    TORCH_CHECK_VALUE(weight.dim() == 2, "embedding takes a table of two dimensions, not ", weight.dim());
    TORCH_CHECK_TYPE(input.scalar_type() == at::kLong || input.scalar_type() == at::kInt, "embedding takes int64 or int32 indices, not ",
                     c10::getDtypeNames(input.scalar_type()).first);
    check_devices("embedding", weight, weight);
    check_devices("embedding", weight, input);
    check_types("embedding", weight, Tensor());
    const int64_t rows = weight.size(0), cols = weight.size(1);
    TORCH_CHECK_VALUE(input.numel() <= kMaxTokens && rows <= kMaxRows && cols <= kMaxCols && (rows > 0 || input.numel() == 0) &&
                          rows * cols <= kMaxElems && input.numel() * cols <= kMaxElems,
                      "embedding takes up to ", kMaxTokens, " tokens and a table of 1 to ", kMaxRows, " rows of up to ", kMaxCols,
                      " elements, at most ", kMaxElems, " elements each in the table and in the embedded tokens");
    int64_t padding = -1;
    if (padding_idx) {
        TORCH_CHECK_VALUE(*padding_idx >= -rows && *padding_idx < rows, "padding_idx ", *padding_idx, " lies outside a table of ", rows, " rows");
        padding = *padding_idx < 0 ? *padding_idx + rows : *padding_idx;
    }
    const c10::DeviceGuard guard(weight.device());
    const Tensor index = input.contiguous();
    if (at::GradMode::is_enabled() && weight.requires_grad()) return Embedding::apply(index, weight, padding, scale);
    return embedding_forward(index, weight, scale);
}

// --------------------------------------------------------------------------------------------------------- 8-bit moments

// Values of the elements [begin, end) of a buffer, in the memory of `device`; codes and exponents lie there or in pinned memory.
std::pair<Tensor, Tensor> state8_read(const Tensor &m, const Tensor &v, const Tensor &scales, int64_t begin, int64_t end, bool bf16,
                                      int64_t device) {
    for (const Tensor *t : {&m, &v, &scales}) {
        TORCH_CHECK(t->is_cuda() || t->is_pinned(), "HybridAdam runs on the GPU: an 8-bit state lives in device memory or in pinned host memory");
        TORCH_CHECK(t->scalar_type() == at::kByte && t->is_contiguous(), "an 8-bit state is held in contiguous uint8 tensors");
    }
    TORCH_CHECK(v.numel() == m.numel() && scales.numel() == 2 * ((m.numel() + 255) / 256) && 0 <= begin && begin <= end && end <= m.numel(),
                "elements [", begin, ", ", end, ") of an 8-bit state of ", m.numel(), " elements");
    const c10::Device where(at::kCUDA, (c10::DeviceIndex)device);
    const c10::DeviceGuard guard(where);
    const auto options = at::TensorOptions().device(where).dtype(bf16 ? at::kBFloat16 : at::kFloat);
    const Tensor mo = at::empty({end - begin}, options), vo = at::empty({end - begin}, options);
    const int64_t piece = 1ll << 32, es = bf16 ? 2 : 4;    // a call takes up to 2^33 elements
    for (int64_t b = begin; b < end; b += piece)
        check("elx_state8_read", elx_state8_read(m.data_ptr<uint8_t>(), v.data_ptr<uint8_t>(), (const uint16_t *)scales.data_ptr(), b,
                                                 std::min(piece, end - b), (char *)mo.data_ptr() + (b - begin) * es,
                                                 (char *)vo.data_ptr() + (b - begin) * es, bf16 ? ELX_BF16 : ELX_F32, stream_of(mo)));
    return {mo, vo};
}

}    // namespace

PYBIND11_MODULE(_elx_torch, m) {
    m.attr("stamp") = "elx_torch built from [" ELX_TORCH_STAMP "]";
    m.def("layer_norm", &layer_norm, py::call_guard<py::gil_scoped_release>());
    m.def("embedding", &embedding, py::call_guard<py::gil_scoped_release>());
    m.def("rows_of", &rows_of);
    m.def("state8_read", &state8_read, py::call_guard<py::gil_scoped_release>());
}
