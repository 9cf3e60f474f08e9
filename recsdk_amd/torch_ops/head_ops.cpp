// The training head over the looked-up rows as torch operators for ROCm tensors, over librecsdk_hip.so:
//
//   recsdk::dropout(x, p, seed, offset=0, step=None)                  mask drawn from a counter, stored nowhere
//   recsdk::layer_norm(x, weight=None, bias=None, eps=1e-5)           over the last dimension
//   recsdk::softmax_loss(x, table, target, item_bias=None, scale=1)   per-row loss against every row of the table
//
// with autograd, and the passes one by one (recsdk::layer_norm_forward, ..._backward, recsdk::softmax_loss_forward,
// ..._backward; the backward of dropout is dropout of the gradient) for callers that run or capture their backward pass
// themselves.  They stand behind the pooled lookup (fbgemm::split_embedding_codegen_lookup_*_function), whose output they take
// and whose backward takes their gradient.  No counterpart in the reference, whose models take these from their framework.
//
// Every call runs on the caller's current stream of the tensors' device and takes its workspace from torch's allocator.
// Tensors whose rows are not laid out as the library takes them (last dimension not contiguous, rows of x or table that
// do not start on 16-byte borders) are copied first.
#include <array>
#include <tuple>

#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>
#include <torch/autograd.h>
#include <torch/library.h>

#include "recsdk_hip.h"

namespace {

using at::Tensor;
using c10::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check(int rc, const char* what)
{
    TORCH_CHECK(rc == RECSDK_OK, what, " failed: ", recsdk_last_error());
}

void* current_stream(const Tensor& t)
{
    return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

int32_t float_type(const Tensor& t, const char* what)
{
    switch (t.scalar_type()) {
        case at::kFloat:
            return RECSDK_DT_F32;
        case at::kHalf:
            return RECSDK_DT_F16;
        case at::kBFloat16:
            return RECSDK_DT_BF16;
        default:
            TORCH_CHECK(false, what, ": expected float32, float16 or bfloat16, got ", t.scalar_type());
    }
}

void same_device(const Tensor& t, const Tensor& x, const char* what)
{
    TORCH_CHECK(t.device() == x.device(), what, ": all tensors must be on the device of x");
}

bool has(const optional<Tensor>& t)
{
    return t.has_value() && t->defined();
}

void once_only(const char* what)
{
    TORCH_CHECK(!at::GradMode::is_enabled(), what, ": the backward pass cannot be differentiated again (create_graph)");
}

Tensor bytes(int64_t n, const Tensor& like)
{
    return at::empty({n}, like.options().dtype(at::kByte));
}

// ---- dropout ---------------------------------------------------------------------------------------------------------

Tensor dropout_cuda(const Tensor& x_, double p, int64_t seed, int64_t offset, const optional<Tensor>& step)
{
    constexpr const char* what = "recsdk::dropout";
    TORCH_CHECK(x_.is_cuda(), what, ": x must be on a ROCm device");
    const int32_t dt = float_type(x_, what);
    const int64_t* word = nullptr;
    if (has(step)) {
        same_device(*step, x_, what);
        TORCH_CHECK(step->scalar_type() == at::kLong && step->numel() == 1, what, ": step must hold one int64");
        word = step->data_ptr<int64_t>();
    }
    const c10::DeviceGuard guard(x_.device());
    const Tensor x = x_.contiguous();
    Tensor y = at::empty_like(x);
    check(recsdk_dropout(x.data_ptr(), x.numel(), dt, p, (uint64_t)seed, (uint64_t)offset, word, y.data_ptr(),
                         current_stream(x)),
          what);
    return y;
}

class Dropout : public torch::autograd::Function<Dropout> {
public:
    static Tensor forward(AutogradContext* ctx, const Tensor& x, double p, int64_t seed, int64_t offset,
                          const optional<Tensor>& step)
    {
        if (has(step)) {
            ctx->save_for_backward({*step});   // a word that was advanced before the backward pass is an error there
        }
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["offset"] = offset;
        return dropout_cuda(x, p, seed, offset, step);
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        once_only("recsdk::dropout");
        const auto saved = ctx->get_saved_variables();
        variable_list out(5);
        if (grads[0].defined()) {
            out[0] = dropout_cuda(grads[0], ctx->saved_data["p"].toDouble(), ctx->saved_data["seed"].toInt(),
                                  ctx->saved_data["offset"].toInt(), saved.empty() ? optional<Tensor>() : saved[0]);
        }
        return out;
    }
};

Tensor dropout_autograd(const Tensor& x, double p, int64_t seed, int64_t offset, const optional<Tensor>& step)
{
    if (!at::GradMode::is_enabled() || !x.requires_grad()) {
        return dropout_cuda(x, p, seed, offset, step);
    }
    return Dropout::apply(x, p, seed, offset, step);
}

// ---- layer norm ------------------------------------------------------------------------------------------------------

// x as rows of its last dimension: a tensor to read from and the elements between its rows
std::tuple<Tensor, int64_t> norm_rows(const Tensor& x)
{
    const int64_t dim = x.size(-1);
    if (x.dim() == 2 && (x.stride(1) == 1 || dim == 1) && (x.stride(0) >= dim || x.size(0) == 1)) {
        return {x, x.size(0) == 1 ? dim : x.stride(0)};
    }
    return {x.contiguous(), dim};
}

int32_t norm_params(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias, const char* what)
{
    TORCH_CHECK(x.is_cuda(), what, ": x must be on a ROCm device");
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, what, ": x needs a last dimension to normalise over");
    float_type(x, what);
    TORCH_CHECK(x.size(-1) < (int64_t(1) << 31), what, ": the last dimension is too long");
    at::ScalarType type = has(weight) ? weight->scalar_type() : has(bias) ? bias->scalar_type() : at::kFloat;
    for (const auto* p : {&weight, &bias}) {
        if (has(*p)) {
            same_device(**p, x, what);
            TORCH_CHECK((*p)->dim() == 1 && (*p)->size(0) == x.size(-1), what,
                        ": weight and bias must hold one value per column");
            TORCH_CHECK((*p)->scalar_type() == type, what, ": weight and bias must be of one type");
        }
    }
    TORCH_CHECK(type == at::kFloat || type == x.scalar_type(), what, ": weight and bias must be float32 or of the type of x");
    return type == at::kFloat ? RECSDK_DT_F32 : float_type(x, what);
}

std::tuple<Tensor, Tensor, Tensor> norm_forward(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias,
                                                double eps, bool stats, const char* what)
{
    const int32_t wt = norm_params(x, weight, bias, what);
    const c10::DeviceGuard guard(x.device());
    const auto [rowsOf, stride] = norm_rows(x);
    const int64_t dim = x.size(-1);
    const int64_t rows = x.numel() / dim;
    const Tensor w = has(weight) ? weight->contiguous() : Tensor();
    const Tensor b = has(bias) ? bias->contiguous() : Tensor();
    Tensor y = at::empty(x.sizes(), x.options());
    Tensor mean, rstd;
    if (stats) {
        mean = at::empty({rows}, x.options().dtype(at::kFloat));
        rstd = at::empty({rows}, x.options().dtype(at::kFloat));
    }
    check(recsdk_layer_norm_forward(rowsOf.data_ptr(), rows, (int32_t)dim, stride, float_type(x, what),
                                    w.defined() ? w.data_ptr() : nullptr, b.defined() ? b.data_ptr() : nullptr, wt, (float)eps,
                                    y.data_ptr(), stats && rows > 0 ? mean.data_ptr<float>() : nullptr,
                                    stats && rows > 0 ? rstd.data_ptr<float>() : nullptr, current_stream(x)),
          what);
    return {y, mean, rstd};
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_forward(const Tensor& x, const optional<Tensor>& weight,
                                                      const optional<Tensor>& bias, double eps)
{
    return norm_forward(x, weight, bias, eps, true, "recsdk::layer_norm_forward");
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_backward(const Tensor& grad_, const Tensor& x, const optional<Tensor>& weight,
                                                       const Tensor& mean, const Tensor& rstd, std::array<bool, 3> wanted)
{
    constexpr const char* what = "recsdk::layer_norm_backward";
    const int32_t wt = norm_params(x, weight, optional<Tensor>(), what);
    const int64_t dim = x.size(-1);
    const int64_t rows = x.numel() / dim;
    same_device(grad_, x, what);
    TORCH_CHECK(grad_.sizes() == x.sizes() && grad_.scalar_type() == x.scalar_type(), what,
                ": the gradient must have the shape and type of x");
    for (const Tensor* t : {&mean, &rstd}) {
        same_device(*t, x, what);
        TORCH_CHECK(t->scalar_type() == at::kFloat && t->is_contiguous() && t->numel() == rows, what,
                    ": mean and rstd must be what the forward pass returned");
    }
    const c10::DeviceGuard guard(x.device());
    const auto [rowsOf, stride] = norm_rows(x);
    const Tensor grad = grad_.contiguous();
    const Tensor w = has(weight) ? weight->contiguous() : Tensor();
    const auto params = x.options().dtype(wt == RECSDK_DT_F32 ? at::kFloat : x.scalar_type());
    Tensor dx, dweight, dbias, space;
    if (wanted[0]) {
        dx = at::empty(x.sizes(), x.options());
    }
    if (wanted[1]) {
        dweight = at::empty({dim}, params);
    }
    if (wanted[2]) {
        dbias = at::empty({dim}, params);
    }
    int64_t need = 0;
    if (wanted[1] || wanted[2]) {
        check(recsdk_layer_norm_workspace(rows, (int32_t)dim, &need), what);
        space = bytes(need, x);
    }
    auto ptr = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
    check(recsdk_layer_norm_backward(grad.data_ptr(), rowsOf.data_ptr(), rows, (int32_t)dim, stride, float_type(x, what), ptr(w),
                                     wt, mean.data_ptr<float>(), rstd.data_ptr<float>(), ptr(dx), ptr(dweight), ptr(dbias),
                                     ptr(space), need, current_stream(x)),
          what);
    return {dx, dweight, dbias};
}

class LayerNorm : public torch::autograd::Function<LayerNorm> {
public:
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias,
                          double eps)
    {
        auto [y, mean, rstd] = norm_forward(x, weight, bias, eps, true, "recsdk::layer_norm");
        ctx->save_for_backward({x, mean, rstd, has(weight) ? *weight : Tensor()});
        ctx->saved_data["biased"] = has(bias);
        ctx->saved_data["bias_type"] = has(bias) ? (int64_t)bias->scalar_type() : (int64_t)at::kFloat;
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        once_only("recsdk::layer_norm");
        variable_list out(4);
        if (!grads[0].defined()) {
            return out;
        }
        const auto saved = ctx->get_saved_variables();
        const optional<Tensor> weight = saved[3].defined() ? optional<Tensor>(saved[3]) : optional<Tensor>();
        // the inputs that are tensors are counted: the bias is the second of them without a weight
        const bool weighted = weight.has_value();
        const std::array<bool, 3> wanted = {ctx->needs_input_grad(0), weighted && ctx->needs_input_grad(1),
                                            ctx->saved_data["biased"].toBool() && ctx->needs_input_grad(weighted ? 2 : 1)};
        auto [dx, dw, db] = layer_norm_backward(grads[0], saved[0], weight, saved[1], saved[2], wanted);
        out[0] = dx;
        out[1] = dw;
        if (db.defined()) {
            out[2] = db.to((at::ScalarType)ctx->saved_data["bias_type"].toInt());   // a bias without a weight
        }
        return out;
    }
};

Tensor layer_norm_cuda(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias, double eps)
{
    return std::get<0>(norm_forward(x, weight, bias, eps, false, "recsdk::layer_norm"));
}

Tensor layer_norm_autograd(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias, double eps)
{
    const bool wanted = x.requires_grad() || (has(weight) && weight->requires_grad()) || (has(bias) && bias->requires_grad());
    if (!at::GradMode::is_enabled() || !wanted) {
        return layer_norm_cuda(x, weight, bias, eps);
    }
    return LayerNorm::apply(x, weight, bias, eps);
}

// ---- softmax loss ----------------------------------------------------------------------------------------------------

struct LossInputs {
    Tensor x, table, target, bias;
    int64_t rows, items, xStride, tableStride;
    int32_t dim, type;
    float* bias_ptr() const { return bias.defined() ? bias.data_ptr<float>() : nullptr; }
};

// rows with their columns side by side, starting on a 16-byte border, and the elements between them
std::tuple<Tensor, int64_t> loss_rows(const Tensor& t)
{
    const int64_t n = t.size(0);
    const int64_t dim = t.size(1);
    const bool side_by_side = (t.stride(1) == 1 || dim == 1) && (n <= 1 || t.stride(0) >= dim);
    const bool aligned = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    if (side_by_side && aligned) {
        return {t, n <= 1 ? dim : t.stride(0)};
    }
    return {t.clone(at::MemoryFormat::Contiguous), dim};
}

LossInputs loss_inputs(const Tensor& x, const Tensor& table, const Tensor& target, const optional<Tensor>& item_bias,
                       const char* what)
{
    TORCH_CHECK(x.is_cuda(), what, ": x must be on a ROCm device");
    for (const Tensor* t : {&table, &target}) {
        same_device(*t, x, what);
    }
    TORCH_CHECK(x.dim() == 2 && table.dim() == 2 && x.size(1) == table.size(1), what,
                ": x and table must be matrices with the same number of columns");
    TORCH_CHECK(x.scalar_type() == table.scalar_type(), what, ": x and table must be of one type, got ", x.scalar_type(), " and ",
                table.scalar_type());
    TORCH_CHECK(target.dim() == 1 && target.size(0) == x.size(0), what, ": target must hold one item per row of x");
    TORCH_CHECK(target.scalar_type() == at::kLong || target.scalar_type() == at::kInt, what, ": target must be int64 or int32");
    LossInputs l;
    l.type = float_type(x, what);
    l.rows = x.size(0);
    l.items = table.size(0);
    TORCH_CHECK(x.size(1) <= 256, what, ": at most 256 columns, got ", x.size(1));
    l.dim = (int32_t)x.size(1);
    std::tie(l.x, l.xStride) = loss_rows(x);
    std::tie(l.table, l.tableStride) = loss_rows(table);
    l.target = target.to(at::kLong).contiguous();
    if (has(item_bias)) {
        same_device(*item_bias, x, what);
        TORCH_CHECK(item_bias->scalar_type() == at::kFloat && item_bias->dim() == 1 && item_bias->size(0) == l.items, what,
                    ": item_bias must hold one float32 per row of the table");
        l.bias = item_bias->contiguous();
    }
    return l;
}

std::tuple<Tensor, Tensor> softmax_loss_forward(const Tensor& x, const Tensor& table, const Tensor& target,
                                                const optional<Tensor>& item_bias, double scale)
{
    constexpr const char* what = "recsdk::softmax_loss";
    const c10::OptionalDeviceGuard guard(x.is_cuda() ? optional<c10::Device>(x.device()) : optional<c10::Device>());
    const LossInputs l = loss_inputs(x, table, target, item_bias, what);
    int64_t need = 0;
    int64_t unused = 0;
    check(recsdk_softmax_loss_workspace(l.rows, l.items, l.dim, l.type, l.xStride, l.tableStride, &need, &unused), what);
    Tensor loss = at::empty({l.rows}, x.options().dtype(at::kFloat));
    Tensor lse = at::empty({l.rows}, x.options().dtype(at::kFloat));
    const Tensor space = bytes(need, x);
    check(recsdk_softmax_loss_forward(l.x.data_ptr(), l.rows, l.xStride, l.table.data_ptr(), l.items, l.tableStride, l.dim, l.type,
                                      l.target.data_ptr<int64_t>(), l.bias_ptr(), (float)scale, loss.data_ptr<float>(),
                                      lse.data_ptr<float>(), space.data_ptr(), need, current_stream(x)),
          what);
    return {loss, lse};
}

std::tuple<Tensor, Tensor> softmax_loss_backward(const Tensor& grad_, const Tensor& x, const Tensor& table, const Tensor& target,
                                                 const Tensor& lse, const optional<Tensor>& item_bias, double scale,
                                                 std::array<bool, 2> wanted)
{
    constexpr const char* what = "recsdk::softmax_loss_backward";
    const c10::OptionalDeviceGuard guard(x.is_cuda() ? optional<c10::Device>(x.device()) : optional<c10::Device>());
    const LossInputs l = loss_inputs(x, table, target, item_bias, what);
    for (const Tensor* t : {&grad_, &lse}) {
        same_device(*t, x, what);
        TORCH_CHECK(t->scalar_type() == at::kFloat && t->dim() == 1 && t->size(0) == l.rows, what,
                    ": the gradient and lse must hold one float32 per row of x");
    }
    const Tensor grad = grad_.contiguous();
    const Tensor l2 = lse.contiguous();
    int64_t need = 0;
    int64_t unused = 0;
    check(recsdk_softmax_loss_workspace(l.rows, l.items, l.dim, l.type, l.xStride, l.tableStride, &unused, &need), what);
    Tensor dx, dtable;
    if (wanted[0]) {
        dx = at::empty({l.rows, l.dim}, x.options());
    }
    if (wanted[1]) {
        dtable = at::empty({l.items, l.dim}, x.options());
    }
    const Tensor space = bytes(need, x);
    check(recsdk_softmax_loss_backward(grad.data_ptr<float>(), l.x.data_ptr(), l.rows, l.xStride, l.table.data_ptr(), l.items,
                                       l.tableStride, l.dim, l.type, l.target.data_ptr<int64_t>(), l.bias_ptr(), (float)scale,
                                       l2.data_ptr<float>(), dx.defined() ? dx.data_ptr() : nullptr,
                                       dtable.defined() ? dtable.data_ptr() : nullptr, space.data_ptr(), need, current_stream(x)),
          what);
    return {dx, dtable};
}

class SoftmaxLoss : public torch::autograd::Function<SoftmaxLoss> {
public:
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& table, const Tensor& target,
                          const optional<Tensor>& item_bias, double scale)
    {
        auto [loss, lse] = softmax_loss_forward(x, table, target, item_bias, scale);
        ctx->save_for_backward({x, table, target, lse, has(item_bias) ? *item_bias : Tensor()});
        ctx->saved_data["scale"] = scale;
        return loss;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        once_only("recsdk::softmax_loss");
        variable_list out(5);
        if (!grads[0].defined()) {
            return out;
        }
        const auto saved = ctx->get_saved_variables();
        const optional<Tensor> bias = saved[4].defined() ? optional<Tensor>(saved[4]) : optional<Tensor>();
        std::tie(out[0], out[1]) =
            softmax_loss_backward(grads[0], saved[0], saved[1], saved[2], saved[3], bias, ctx->saved_data["scale"].toDouble(),
                                  {ctx->needs_input_grad(0), ctx->needs_input_grad(1)});
        return out;
    }
};

Tensor softmax_loss_cuda(const Tensor& x, const Tensor& table, const Tensor& target, const optional<Tensor>& item_bias,
                         double scale)
{
    return std::get<0>(softmax_loss_forward(x, table, target, item_bias, scale));
}

Tensor softmax_loss_autograd(const Tensor& x, const Tensor& table, const Tensor& target, const optional<Tensor>& item_bias,
                             double scale)
{
    TORCH_CHECK(!at::GradMode::is_enabled() || !has(item_bias) || !item_bias->requires_grad(),
                "recsdk::softmax_loss: item_bias takes no gradient");
    if (!at::GradMode::is_enabled() || (!x.requires_grad() && !table.requires_grad())) {
        return softmax_loss_cuda(x, table, target, item_bias, scale);
    }
    return SoftmaxLoss::apply(x, table, target, item_bias, scale);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(recsdk, m)
{
    m.def("dropout(Tensor x, float p, int seed, int offset=0, Tensor? step=None) -> Tensor");
    m.def("layer_norm(Tensor x, Tensor? weight=None, Tensor? bias=None, float eps=1e-05) -> Tensor");
    m.def("layer_norm_forward(Tensor x, Tensor? weight=None, Tensor? bias=None, float eps=1e-05) -> (Tensor, Tensor, Tensor)");
    m.def("layer_norm_backward(Tensor grad, Tensor x, Tensor? weight, Tensor mean, Tensor rstd, bool[3] wanted) "
          "-> (Tensor, Tensor, Tensor)");
    m.def("softmax_loss(Tensor x, Tensor table, Tensor target, Tensor? item_bias=None, float scale=1.0) -> Tensor");
    m.def("softmax_loss_forward(Tensor x, Tensor table, Tensor target, Tensor? item_bias=None, float scale=1.0) "
          "-> (Tensor, Tensor)");
    m.def("softmax_loss_backward(Tensor grad, Tensor x, Tensor table, Tensor target, Tensor lse, Tensor? item_bias, "
          "float scale, bool[2] wanted) -> (Tensor, Tensor)");
}

// ROCm tensors carry the CUDA dispatch key.
TORCH_LIBRARY_IMPL(recsdk, CUDA, m)
{
    m.impl("dropout", TORCH_FN(dropout_cuda));
    m.impl("layer_norm", TORCH_FN(layer_norm_cuda));
    m.impl("layer_norm_forward", TORCH_FN(layer_norm_forward));
    m.impl("layer_norm_backward", TORCH_FN(layer_norm_backward));
    m.impl("softmax_loss", TORCH_FN(softmax_loss_cuda));
    m.impl("softmax_loss_forward", TORCH_FN(softmax_loss_forward));
    m.impl("softmax_loss_backward", TORCH_FN(softmax_loss_backward));
}

TORCH_LIBRARY_IMPL(recsdk, Autograd, m)
{
    m.impl("dropout", TORCH_FN(dropout_autograd));
    m.impl("layer_norm", TORCH_FN(layer_norm_autograd));
    m.impl("softmax_loss", TORCH_FN(softmax_loss_autograd));
}
