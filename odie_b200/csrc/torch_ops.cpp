// The routed-expert row operators as differentiable torch functions: checks, allocations and autograd nodes around the
// C-ABI (odie_b200/experts.py has their documentation).
//
// In C++ because of what a small call costs on the host: a layer of 1021 rows, forward and backward, took 143 us
// through autograd nodes written in Python (the engine's thread waits for the interpreter at every node), more than
// its kernels.
#include <torch/extension.h>
#include <torch/csrc/autograd/engine.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include "odie_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

void done(int status, const char* name) { TORCH_CHECK(status == 0, name, " failed: ", status == -1 ? odie_error() : "CUDA error"); }
uint64_t stream_of(const Tensor& t) {
    return reinterpret_cast<uint64_t>(c10::cuda::getCurrentCUDAStream(t.get_device()).stream());
}
void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor rows_like(const Tensor& t, at::IntArrayRef shape) { return at::empty(shape, t.options().requires_grad(false)); }
Tensor scratch(const Tensor& t, int64_t bytes) {
    return bytes ? at::empty({bytes}, t.options().dtype(at::kByte).requires_grad(false)) : Tensor();
}
// Absent tensors: std::nullopt as arguments of an autograd function, undefined inside.
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }
Tensor present(const Maybe& t) { return t ? *t : Tensor(); }
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }

int row_type(const Tensor& t) {
    return t.scalar_type() == at::kHalf ? 0 : t.scalar_type() == at::kBFloat16 ? 1 : t.scalar_type() == at::kFloat ? 2 : -1;
}
void check_rows(const Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(t.is_cuda() && row_type(t) >= 0 && t.dim() == 2 && t.size(1) > 0, name,
                      " must be a CUDA fp16, bf16 or fp32 tensor [rows, width] with at least one column");
}
void check_ids(const Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(t.is_cuda() && (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong), name,
                      " must be a CUDA int32 or int64 tensor");
}
void check_device(const Tensor& t, const Tensor& as, const char* name) {
    TORCH_CHECK_VALUE(t.device() == as.device(), name, " is on ", t.device(), ", not ", as.device());
}

// Forward-mode derivatives are refused: the kernels' results would have no tangent, and the derivative be wrong.
bool dual(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool dual(const Maybe& t) { return t && dual(*t); }
template <typename... Tensors>
void refuse_tangents(const Tensors&... tensors) {
    TORCH_CHECK_NOT_IMPLEMENTED(!(c10::AutogradState::get_tls_state().get_fw_grad_mode() && (dual(tensors) || ...)),
                                "the row operators of odie_b200 have no forward-mode derivatives");
}

// What a backward pass returns.  Asked for a graph of it (create_graph), it hangs by a node that refuses to be
// differentiated from the tensors that it depends on: `from`, and the first `arguments` of the forward pass (by the
// running node's edges to them, so that none is kept for it).
variable_list once(variable_list gradients, const variable_list& from, size_t arguments = 0) {
    if (!at::GradMode::is_enabled()) return gradients;
    torch::autograd::edge_list edges = torch::autograd::collect_next_edges(from);
    if (arguments) {
        const auto node = torch::autograd::get_current_node();
        TORCH_CHECK(node && node->num_outputs() >= arguments, "a backward pass outside of its node");
        for (size_t i = 0; i < arguments; ++i) edges.push_back(node->next_edge(i));
    }
    for (Tensor& g : gradients) {
        if (!g.defined()) continue;
        g = g.detach();
        torch::autograd::set_history(g, std::make_shared<torch::autograd::Error>("the row operators of odie_b200 are differentiable once",
                                                                                 torch::autograd::edge_list(edges)));
    }
    return gradients;
}

// ---------------------------------------------------------------- order
std::tuple<Tensor, Tensor, Tensor> sort_rows(const Tensor& expert, int64_t bins) {
    check_ids(expert, "expert");
    TORCH_CHECK_VALUE(expert.dim() == 1 || (expert.dim() == 2 && expert.size(1) > 0), "expert must have the shape [rows] or [rows, choices]");
    TORCH_CHECK_VALUE(bins >= 1 && bins < (int64_t(1) << 30), "bins must be 1 to 2^30 - 1");
    const int64_t rows = expert.size(0), choices = expert.dim() == 1 ? 1 : expert.size(1), n = rows * choices;
    TORCH_CHECK_VALUE(n < (int64_t(1) << 31) - 4096, "too many (row, choice) pairs");
    const c10::cuda::CUDAGuard guard(expert.device());
    const Tensor keys = expert.contiguous();
    const auto options = expert.options().dtype(at::kInt);
    Tensor order = at::empty({n}, options), slot = at::empty({rows, choices}, options), offsets = at::empty({bins + 1}, options);
    const Tensor work = scratch(expert, odie_sort_rows_scratch(n, int(bins)));
    done(odie_sort_rows(data(keys), int(keys.element_size()), n, int(bins), static_cast<int32_t*>(data(order)),
                        static_cast<int32_t*>(data(slot)), static_cast<int32_t*>(data(offsets)), data(work), stream_of(expert)),
         "odie_sort_rows");
    return {order, slot, offsets};
}

// ---------------------------------------------------------------- dispatch and combine
struct Order {
    Tensor order, slot;
    int64_t rows() const { return slot.size(0); }
    int64_t choices() const { return slot.size(1); }
    const int32_t* order_data() const { return static_cast<const int32_t*>(data(order)); }
    const int32_t* slot_data() const { return static_cast<const int32_t*>(data(slot)); }
};

Order check_order(const Tensor& order, const Tensor& slot) {
    TORCH_CHECK_VALUE(slot.is_cuda() && slot.scalar_type() == at::kInt && slot.dim() == 2 && slot.size(1) > 0 && slot.is_contiguous() &&
                          order.device() == slot.device() && order.scalar_type() == at::kInt && order.dim() == 1 &&
                          order.size(0) == slot.numel() && order.is_contiguous(),
                      "order must hold contiguous CUDA int32 tensors: order [rows * choices] and slot [rows, choices]");
    return {order, slot};
}

Tensor dispatched(const Tensor& x, const Order& o, const Tensor& weights) {
    const c10::cuda::CUDAGuard guard(x.device());
    Tensor out = rows_like(x, {o.rows() * o.choices(), x.size(1)});
    done(odie_dispatch(data(x), o.rows(), int(o.choices()), x.size(1), row_type(x), o.order_data(), o.slot_data(),
                       static_cast<const float*>(data(weights)), data(out), stream_of(x)),
         "odie_dispatch");
    return out;
}
Tensor combined(const Tensor& rows, const Order& o, const Tensor& weights) {
    const c10::cuda::CUDAGuard guard(rows.device());
    Tensor out = rows_like(rows, {o.rows(), rows.size(1)});
    done(odie_combine(data(rows), o.rows(), int(o.choices()), rows.size(1), row_type(rows), o.slot_data(),
                      static_cast<const float*>(data(weights)), data(out), stream_of(rows)),
         "odie_combine");
    return out;
}
// (d rows, d weights); rows are the sorted ones, needed for d weights.
std::pair<Tensor, Tensor> combine_gradients(const Tensor& d_out, const Tensor& rows, const Order& o, const Tensor& weights, bool need_rows,
                                            bool need_weights) {
    const c10::cuda::CUDAGuard guard(d_out.device());
    Tensor d_rows, d_weights;
    if (need_rows) d_rows = rows_like(d_out, {o.rows() * o.choices(), d_out.size(1)});
    if (need_weights) d_weights = at::empty({o.rows(), o.choices()}, d_out.options().dtype(at::kFloat));
    done(odie_combine_backward(data(d_out), data(rows), o.rows(), int(o.choices()), d_out.size(1), row_type(d_out), o.order_data(),
                               o.slot_data(), static_cast<const float*>(data(weights)), data(d_rows), static_cast<float*>(data(d_weights)),
                               stream_of(d_out)),
         "odie_combine_backward");
    return {d_rows, d_weights};
}

struct Dispatch : torch::autograd::Function<Dispatch> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& maybe_weights, const Tensor& order, const Tensor& slot,
                          bool need_x, bool need_weights) {
        const Tensor weights = present(maybe_weights);
        ctx->save_for_backward({need_weights ? x : Tensor(), weights, order, slot});
        ctx->saved_data["need"] = int64_t(need_x) | int64_t(need_weights) << 1;
        return dispatched(x, {order, slot}, weights);
    }
    static variable_list backward(AutogradContext* ctx, variable_list gradients) {
        refuse_tangents(gradients[0]);
        const auto saved = ctx->get_saved_variables();
        const int64_t need = ctx->saved_data["need"].toInt();
        const Order o{saved[2], saved[3]};
        const Tensor d_rows = gradients[0].contiguous();
        Tensor d_x, d_weights;
        if (need & 1) d_x = combined(d_rows, o, saved[1]);
        // d weights[t, j] = <x[t], d rows[slot]>: the same product as combine's, the rows' roles exchanged
        if (need & 2) d_weights = combine_gradients(saved[0], d_rows, o, Tensor(), false, true).second;
        return once({d_x, d_weights, Tensor(), Tensor(), Tensor(), Tensor()}, {gradients[0], saved[0], saved[1]});
    }
};

struct Combine : torch::autograd::Function<Combine> {
    static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Maybe& maybe_weights, const Tensor& order, const Tensor& slot,
                          bool need_rows, bool need_weights) {
        const Tensor weights = present(maybe_weights);
        ctx->save_for_backward({need_weights ? rows : Tensor(), weights, order, slot});
        ctx->saved_data["need"] = int64_t(need_rows) | int64_t(need_weights) << 1;
        return combined(rows, {order, slot}, weights);
    }
    static variable_list backward(AutogradContext* ctx, variable_list gradients) {
        refuse_tangents(gradients[0]);
        const auto saved = ctx->get_saved_variables();
        const int64_t need = ctx->saved_data["need"].toInt();
        const auto [d_rows, d_weights] =
            combine_gradients(gradients[0].contiguous(), saved[0], {saved[2], saved[3]}, saved[1], need & 1, need & 2);
        return once({d_rows, d_weights, Tensor(), Tensor(), Tensor(), Tensor()}, {gradients[0], saved[0], saved[1]});
    }
};

// fp32 [rows, choices]; differentiable, so that the gradient takes the weights' own type and shape.
Tensor check_weights(const Maybe& weights, const Order& o, const Tensor& x) {
    if (!weights) return Tensor();
    TORCH_CHECK_VALUE(weights->is_cuda() && weights->is_floating_point(), "weights must be a CUDA floating-point tensor");
    TORCH_CHECK_VALUE(weights->sizes() == o.slot.sizes() || (o.choices() == 1 && weights->dim() == 1 && weights->size(0) == o.rows()),
                      "weights must have the shape of the choices ", o.slot.sizes(), ", not ", weights->sizes());
    check_device(*weights, x, "weights");
    return weights->to(at::kFloat).reshape(o.slot.sizes()).contiguous();
}

Tensor dispatch(const Tensor& x, const Tensor& order, const Tensor& slot, const Maybe& weights) {
    check_rows(x, "x");
    refuse_tangents(x, weights);
    const Order o = check_order(order, slot);
    TORCH_CHECK_VALUE(x.size(0) == o.rows(), "x has ", x.size(0), " rows, the order ", o.rows());
    check_device(slot, x, "order");
    const Tensor w = check_weights(weights, o, x), rows = x.contiguous();
    if (at::GradMode::is_enabled() && (wants(rows) || wants(w))) return Dispatch::apply(rows, maybe(w), order, slot, wants(rows), wants(w));
    return dispatched(rows, o, w);
}

Tensor combine(const Tensor& rows, const Tensor& order, const Tensor& slot, const Maybe& weights) {
    check_rows(rows, "rows");
    refuse_tangents(rows, weights);
    const Order o = check_order(order, slot);
    TORCH_CHECK_VALUE(rows.size(0) == o.rows() * o.choices(), "rows has ", rows.size(0), " rows, the order ", o.rows(), " x ", o.choices());
    check_device(slot, rows, "order");
    const Tensor w = check_weights(weights, o, rows), sorted = rows.contiguous();
    if (at::GradMode::is_enabled() && (wants(sorted) || wants(w))) return Combine::apply(sorted, maybe(w), order, slot, wants(sorted), wants(w));
    return combined(sorted, o, w);
}

// ---------------------------------------------------------------- linear
bool on_16_bytes(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
// Contiguous, starting on a 16-byte boundary (a view of an odd offset is copied), as every new tensor does.
Tensor aligned(const Tensor& t) {
    const Tensor c = t.contiguous();
    return on_16_bytes(c) ? c : c.clone();
}
struct Sizes {
    int64_t rows, inputs, outputs, groups;
    Sizes(const Tensor& x, const Tensor& weight)
        : rows(x.size(0)), inputs(x.size(1)), outputs(weight.size(-2)), groups(weight.dim() == 3 ? weight.size(0) : 1) {}
};

Tensor linear_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual, const Tensor& offsets,
                      int64_t activation, bool keep_slope, Tensor& slope) {
    const c10::cuda::CUDAGuard guard(x.device());
    const Sizes s(x, weight);
    Tensor y = rows_like(x, {s.rows, s.outputs});
    if (keep_slope)  // a ReLU's as bits
        slope = activation == 1 ? at::empty({s.rows, (s.outputs + 7) / 8}, x.options().dtype(at::kByte).requires_grad(false))
                                : at::empty({s.rows, s.outputs}, x.options().dtype(at::kShort).requires_grad(false));
    const bool on_16 = !residual.defined() || on_16_bytes(residual);  // the others are
    const Tensor work = scratch(x, odie_linear_scratch_for(s.rows, int(s.inputs), int(s.outputs), int(s.groups), offsets.defined(), on_16));
    done(odie_linear(data(x), data(weight), data(bias), data(residual), s.rows, int(s.inputs), int(s.outputs), int(s.groups),
                     static_cast<const int32_t*>(data(offsets)), row_type(x), int(activation), data(y), data(slope), data(work), stream_of(x)),
         "odie_linear");
    return y;
}

struct Linear : torch::autograd::Function<Linear> {
    // need: bits of x, weight, bias, residual
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Maybe& maybe_bias, const Maybe& maybe_residual,
                          const Maybe& maybe_offsets, int64_t activation, int64_t need) {
        const Tensor bias = present(maybe_bias), residual = present(maybe_residual), offsets = present(maybe_offsets);
        Tensor slope;
        Tensor y = linear_forward(x, weight, bias, residual, offsets, activation, (need & 7) && activation != 0, slope);
        ctx->save_for_backward({need & 2 ? x : Tensor(), need & 1 ? weight : Tensor(), slope, offsets});
        ctx->saved_data["need"] = need;
        ctx->saved_data["activation"] = activation;
        ctx->saved_data["slope of"] = int64_t(bias.defined() ? 3 : 2);
        ctx->saved_data["inputs"] = x.size(1);
        ctx->saved_data["weight"] = weight.sizes().vec();
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list gradients) {
        refuse_tangents(gradients[0]);
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &slope = saved[2], &offsets = saved[3];
        // without a slope (only the residual's gradient is wanted) there is no activation to undo
        const int64_t activation = slope.defined() ? ctx->saved_data["activation"].toInt() : 0;
        const int64_t need = ctx->saved_data["need"].toInt(), inputs = ctx->saved_data["inputs"].toInt();
        const auto shape = ctx->saved_data["weight"].toIntVector();
        const int64_t groups = shape.size() == 3 ? shape[0] : 1, outputs = shape[shape.size() - 2];
        const Tensor d_y = aligned(gradients[0]);
        const int64_t rows = d_y.size(0);
        const c10::cuda::CUDAGuard guard(d_y.device());
        Tensor d_x, d_weight, d_bias, d_residual;
        if (need & 1) d_x = rows_like(d_y, {rows, inputs});
        if (need & 2) d_weight = rows_like(d_y, shape);
        if (need & 4) d_bias = rows_like(d_y, at::IntArrayRef(shape.data(), shape.size() - 1));
        if (need & 8) d_residual = offsets.defined() ? rows_like(d_y, {rows, outputs}) : d_y;  // every row is a group's row
        if ((need & 7) || (need & 8 && offsets.defined())) {
            const Tensor work = scratch(d_y, odie_linear_backward_scratch_for(rows, int(inputs), int(outputs), int(groups), 1));  // (see aligned)
            done(odie_linear_backward(data(d_y), data(slope), int(activation), data(x), data(weight), rows,
                                      int(inputs), int(outputs), int(groups), static_cast<const int32_t*>(data(offsets)), row_type(d_y),
                                      data(d_x), data(d_weight), data(d_bias), offsets.defined() ? data(d_residual) : nullptr, data(work),
                                      stream_of(d_y)),
                 "odie_linear_backward");
        }
        return once({d_x, d_weight, d_bias, d_residual, Tensor(), Tensor(), Tensor()}, {gradients[0], x, weight},
                    slope.defined() && activation != 1 ? ctx->saved_data["slope of"].toInt() : 0);
    }
};

Tensor linear(const Tensor& x, const Tensor& weight, const Maybe& bias, const Maybe& residual, int64_t activation, const Maybe& offsets) {
    TORCH_CHECK_VALUE(x.is_cuda() && (x.scalar_type() == at::kHalf || x.scalar_type() == at::kBFloat16) && x.dim() >= 1 && x.size(-1) > 0,
                      "x must be a CUDA fp16 or bf16 tensor with at least one column");
    TORCH_CHECK_VALUE(weight.dim() == (offsets ? 3 : 2) && weight.size(-1) == x.size(-1) && weight.numel() > 0, "weight must be [",
                      offsets ? "experts, " : "", "outputs, ", x.size(-1), "], not ", weight.sizes());
    TORCH_CHECK_VALUE(weight.size(-1) <= (1 << 20) && weight.size(-2) <= (1 << 20), "at most 2^20 inputs and outputs");
    TORCH_CHECK_VALUE(!bias || bias->sizes() == weight.sizes().slice(0, weight.dim() - 1), "bias must be ",
                      weight.sizes().slice(0, weight.dim() - 1), ", not ", bias ? bias->sizes() : at::IntArrayRef());
    auto check = [&](const Tensor& t, const char* name) {
        TORCH_CHECK_VALUE(t.scalar_type() == x.scalar_type(), name, " must have the type of x, ", x.scalar_type());
        check_device(t, x, name);
    };
    check(weight, "weight");
    if (bias) check(*bias, "bias");
    if (residual) check(*residual, "residual");
    if (offsets) {
        TORCH_CHECK_VALUE(x.dim() == 2, "x must be [rows, inputs] with offsets");
        TORCH_CHECK_VALUE(weight.size(0) <= 1024, "at most 1024 experts");
        TORCH_CHECK_VALUE(offsets->is_cuda() && offsets->scalar_type() == at::kInt && offsets->dim() == 1 && offsets->size(0) == weight.size(0) + 1,
                          "offsets must be CUDA int32 [", weight.size(0) + 1, "]");
        check_device(*offsets, x, "offsets");
    }
    refuse_tangents(x, weight, bias, residual);
    const int64_t outputs = weight.size(-2);
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = outputs;
    int64_t rows = 1;
    for (int64_t i = 0; i + 1 < x.dim(); ++i) rows *= x.size(i);
    const bool flat = x.dim() == 2;
    const Tensor in = aligned(flat ? x : x.reshape({rows, x.size(-1)}));
    const Tensor w = aligned(weight), b = bias ? bias->contiguous() : Tensor(), o = offsets ? offsets->contiguous() : Tensor();
    Tensor r;
    if (residual) {
        r = residual->sizes() == at::IntArrayRef(shape) ? *residual : residual->expand(shape);
        r = (flat ? r : r.reshape({rows, outputs})).contiguous();
    }
    const int64_t need = at::GradMode::is_enabled() ? int64_t(wants(in)) | int64_t(wants(w)) << 1 | int64_t(wants(b)) << 2 | int64_t(wants(r)) << 3 : 0;
    Tensor slope;
    const Tensor y = need ? Linear::apply(in, w, maybe(b), maybe(r), maybe(o), activation, need) : linear_forward(in, w, b, r, o, activation, false, slope);
    return flat ? y : y.reshape(shape);
}

// ---------------------------------------------------------------- learned rows by id
Tensor embedded(const Tensor& ids, const Tensor& table, double scale) {
    const c10::cuda::CUDAGuard guard(table.device());
    Tensor out = rows_like(table, {ids.numel(), table.size(1)});
    done(odie_embed(data(ids), int(ids.element_size()), ids.numel(), data(table), table.size(0), table.size(1), row_type(table), float(scale),
                    data(out), stream_of(table)),
         "odie_embed");
    return out;
}

struct Embed : torch::autograd::Function<Embed> {
    static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& table, double scale) {
        ctx->save_for_backward({ids});
        ctx->saved_data["rows"] = table.size(0);
        ctx->saved_data["scale"] = scale;
        return embedded(ids, table, scale);
    }
    static variable_list backward(AutogradContext* ctx, variable_list gradients) {
        refuse_tangents(gradients[0]);
        const Tensor ids = ctx->get_saved_variables()[0];
        const int64_t rows = ctx->saved_data["rows"].toInt();
        const Tensor d_out = gradients[0].contiguous();
        const c10::cuda::CUDAGuard guard(d_out.device());
        const int64_t width = d_out.size(1);
        Tensor d_table = rows_like(d_out, {rows, width});
        const Tensor work = scratch(d_out, odie_embed_backward_scratch(ids.numel(), rows, width));
        done(odie_embed_backward(data(ids), int(ids.element_size()), ids.numel(), data(d_out), rows, width, row_type(d_out),
                                 float(ctx->saved_data["scale"].toDouble()), data(d_table), data(work), stream_of(d_out)),
             "odie_embed_backward");
        return once({Tensor(), d_table, Tensor()}, {gradients[0]});
    }
};

Tensor embed(const Tensor& ids, const Tensor& table, double scale) {
    check_ids(ids, "ids");
    check_rows(table, "table");
    refuse_tangents(table);
    TORCH_CHECK_VALUE(table.size(0) >= 1 && table.size(0) < (int64_t(1) << 30), "the table must have 1 to 2^30 - 1 rows");
    TORCH_CHECK_VALUE(ids.numel() < (int64_t(1) << 31) - 4096, "too many ids");
    check_device(ids, table, "ids");
    const Tensor flat = ids.contiguous(), rows = table.contiguous();
    const Tensor out = at::GradMode::is_enabled() && wants(rows) ? Embed::apply(flat, rows, scale) : embedded(flat, rows, scale);
    if (ids.dim() == 1) return out;
    std::vector<int64_t> shape = ids.sizes().vec();
    shape.push_back(table.size(1));
    return out.view(shape);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("sort_rows", &sort_rows);
    m.def("dispatch", &dispatch);
    m.def("combine", &combine);
    m.def("linear", &linear);
    m.def("embed", &embed);
}
