// PyTorch operators of the training step over the C ABI (csrc/norm.hip, csrc/adamw.hip):
//
//   layer_norm                         layer norm, its result in x's type or float32; the transformer camera head of
//                                      the reference's network (nnutils/mesh_net.py:468-536) ends its blocks in one
//   layer_norm_stats / _backward       the same with the rows' statistics, and what they are kept for
//   grad_square_sums                   squares of a list of gradients, summed (the norm that clipping needs)
//   adamw_step                         unscale, clip and AdamW over a list of tensors (nnutils/train_utils.py:201-214),
//                                      32-bit or 8-bit moments
//   moment_values                      what 8-bit moments stand for
//
// GPU and Meta kernels for each, an Autograd kernel for layer_norm; no CPU kernels.
#include "torch_util.h"

#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <algorithm>

namespace {

int32_t type_of(const Tensor &t, const char *name)
{
    switch (t.scalar_type()) {
    case at::kFloat: return SV3D_F32;
    case at::kHalf: return SV3D_F16;
    case at::kBFloat16: return SV3D_BF16;
    default: TORCH_CHECK_VALUE(false, name, " must be float32, float16 or bfloat16, got ", t.scalar_type());
    }
}

void *ptr(const Tensor &t) { return t.defined() && t.numel() > 0 ? t.data_ptr() : nullptr; }

// ---- layer norm ---------------------------------------------------------------------------------
// x as rows of `cols` contiguous elements a fixed stride apart; a copy only where its strides say otherwise.
struct Rows {
    Tensor t;
    int64_t count, stride;
};

Rows rows_of(const Tensor &x, int64_t cols)
{
    const int64_t count = cols > 0 ? x.numel() / cols : 0;
    int64_t d = x.dim() - 1, inner = 1, stride = 0, run = 0;
    bool fits = true;
    for (; d >= 0 && inner < cols; --d) {
        if (x.size(d) != 1 && x.stride(d) != inner) fits = false;
        inner *= x.size(d);
    }
    for (; d >= 0; --d) {
        if (x.size(d) == 1) continue;
        if (run == 0) {
            stride = x.stride(d);
            run = x.size(d);
        } else {
            if (x.stride(d) != stride * run) fits = false;
            run *= x.size(d);
        }
    }
    if (count <= 1) stride = cols;
    if (fits && inner == cols) return {x, count, stride};
    return {x.contiguous(), count, cols};
}

int64_t check_norm(const Tensor &x, IntList shape, const optional<Tensor> &weight, const optional<Tensor> &bias)
{
    type_of(x, "x");
    TORCH_CHECK_VALUE(!shape.empty() && (int64_t)shape.size() <= x.dim() &&
                          x.sizes().slice(x.dim() - shape.size()) == shape,
                      "normalized_shape ", shape, " must be the last sizes of x, got ", x.sizes());
    int64_t cols = 1;
    for (auto s : shape) cols *= s;
    TORCH_CHECK_VALUE(cols > 0 && cols <= (1 << 24), "normalized_shape ", shape, " must hold 1 to 2^24 elements");
    for (const auto &pr : {std::make_pair(&weight, "weight"), std::make_pair(&bias, "bias")}) {
        if (!pr.first->has_value() || !(*pr.first)->defined()) continue;
        const Tensor &t = **pr.first;
        TORCH_CHECK_VALUE(t.sizes() == shape, pr.second, " must be ", shape, ", got ", t.sizes());
        type_of(t, pr.second);
        same_device(x, t, pr.second);
    }
    return cols;
}

bool given(const optional<Tensor> &t) { return t.has_value() && t->defined(); }

// weights are read in x's type where all of them have it, in fp32 otherwise
at::ScalarType param_type(const Tensor &x, const optional<Tensor> &weight, const optional<Tensor> &bias)
{
    const bool same = (!given(weight) || weight->scalar_type() == x.scalar_type()) &&
                      (!given(bias) || bias->scalar_type() == x.scalar_type()) && (given(weight) || given(bias));
    return same ? x.scalar_type() : at::kFloat;
}

Tensor as_param(const optional<Tensor> &t, at::ScalarType type)
{
    if (!given(t)) return Tensor();
    return (t->scalar_type() == type ? *t : t->to(type)).contiguous();
}

int32_t code_of(at::ScalarType t) { return t == at::kFloat ? SV3D_F32 : t == at::kHalf ? SV3D_F16 : SV3D_BF16; }

using NormOut = std::tuple<Tensor, Tensor, Tensor>;

// mean and rstd may be undefined: nobody will call the backward
void run_layer_norm(const Tensor &x, int64_t cols, const optional<Tensor> &weight, const optional<Tensor> &bias, double eps,
                    Tensor &y, Tensor *mean, Tensor *rstd)
{
    TORCH_CHECK_VALUE(eps >= 0.0, "eps must not be negative, got ", eps);
    Launch L(x);
    const Rows r = rows_of(x, cols);
    const auto pt = param_type(x, weight, bias);
    const Tensor w = as_param(weight, pt), b = as_param(bias, pt);
    const sv3d_layer_norm_params p = {r.count, cols, r.stride, cols, code_of(x.scalar_type()), code_of(y.scalar_type()),
                                      code_of(pt), (float)eps};
    check_status(sv3d_layer_norm_forward(&p, ptr(r.t), ptr(w), ptr(b), ptr(y), mean ? (float *)ptr(*mean) : nullptr,
                                         rstd ? (float *)ptr(*rstd) : nullptr, L.stream),
                 "sv3d_layer_norm_forward");
}

Tensor norm_output(const Tensor &x, bool f32_out)
{
    return at::empty(x.sizes(), x.options().dtype(f32_out ? at::kFloat : x.scalar_type()));
}

Tensor layer_norm_gpu(const Tensor &x, IntList shape, const optional<Tensor> &weight, const optional<Tensor> &bias, double eps,
                      bool f32_out)
{
    const int64_t cols = check_norm(x, shape, weight, bias);
    Tensor y = norm_output(x, f32_out);
    run_layer_norm(x, cols, weight, bias, eps, y, nullptr, nullptr);
    return y;
}

Tensor layer_norm_meta(const Tensor &x, IntList shape, const optional<Tensor> &weight, const optional<Tensor> &bias, double,
                       bool f32_out)
{
    check_norm(x, shape, weight, bias);
    return norm_output(x, f32_out);
}

NormOut layer_norm_stats_gpu(const Tensor &x, IntList shape, const optional<Tensor> &weight, const optional<Tensor> &bias,
                             double eps, bool f32_out)
{
    const int64_t cols = check_norm(x, shape, weight, bias);
    Tensor y = norm_output(x, f32_out);
    Tensor mean = at::empty({x.numel() / cols}, x.options().dtype(at::kFloat)), rstd = at::empty_like(mean);
    run_layer_norm(x, cols, weight, bias, eps, y, &mean, &rstd);
    return {y, mean, rstd};
}

NormOut layer_norm_stats_meta(const Tensor &x, IntList shape, const optional<Tensor> &weight, const optional<Tensor> &bias,
                              double, bool f32_out)
{
    const int64_t cols = check_norm(x, shape, weight, bias);
    Tensor mean = at::empty({x.numel() / cols}, x.options().dtype(at::kFloat));
    return {norm_output(x, f32_out), mean, at::empty_like(mean)};
}

void check_norm_backward(const Tensor &dy, const Tensor &x, int64_t cols, const Tensor &mean, const Tensor &rstd)
{
    TORCH_CHECK_VALUE(dy.sizes() == x.sizes() && (dy.scalar_type() == x.scalar_type() || dy.scalar_type() == at::kFloat),
                      "grad_y must be ", x.sizes(), " in x's type or float32, got ", dy.scalar_type(), " ", dy.sizes());
    same_device(x, dy, "grad_y");
    for (const auto &pr : {std::make_pair(&mean, "mean"), std::make_pair(&rstd, "rstd")}) {
        TORCH_CHECK_VALUE(pr.first->scalar_type() == at::kFloat && pr.first->is_contiguous() &&
                              pr.first->numel() == x.numel() / cols,
                          pr.second, " must be float32 with one element per row (an output of the forward operator), got ",
                          pr.first->scalar_type(), " ", pr.first->sizes());
        same_device(x, *pr.first, pr.second);
    }
}

NormOut layer_norm_backward_gpu(const Tensor &dy, const Tensor &x, IntList shape, const optional<Tensor> &weight,
                                const optional<Tensor> &bias, const Tensor &mean, const Tensor &rstd, bool need_x,
                                bool need_weight, bool need_bias)
{
    const int64_t cols = check_norm(x, shape, weight, bias);
    check_norm_backward(dy, x, cols, mean, rstd);
    Launch L(x);
    const Rows r = rows_of(x, cols), g = rows_of(dy, cols);
    const auto pt = param_type(x, weight, bias);
    const Tensor w = as_param(weight, pt);
    Tensor dx, dw, db, ws;
    if (need_x) dx = at::empty(x.sizes(), x.options());
    if (need_weight) dw = at::empty(shape, x.options().dtype(pt));
    if (need_bias) db = at::empty(shape, x.options().dtype(pt));
    const sv3d_layer_norm_params p = {r.count, cols, r.stride, g.stride, code_of(x.scalar_type()), code_of(dy.scalar_type()),
                                      code_of(pt), 0.f};
    size_t bytes = 0;
    if (need_weight || need_bias) {
        check_status(sv3d_layer_norm_workspace(&p, &bytes), "sv3d_layer_norm_workspace");
        ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    }
    check_status(sv3d_layer_norm_backward(&p, ptr(r.t), ptr(g.t), ptr(w), (const float *)ptr(mean), (const float *)ptr(rstd),
                                          ptr(dx), ptr(dw), ptr(db), ptr(ws), bytes, L.stream),
                 "sv3d_layer_norm_backward");
    // an operator returns tensors: what was not asked for comes back empty
    const auto none = [&] { return at::empty({0}, x.options()); };
    return {need_x ? dx : none(), need_weight ? cast_like(dw, given(weight) ? weight->scalar_type() : pt) : none(),
            need_bias ? cast_like(db, given(bias) ? bias->scalar_type() : pt) : none()};
}

NormOut layer_norm_backward_meta(const Tensor &dy, const Tensor &x, IntList shape, const optional<Tensor> &weight,
                                 const optional<Tensor> &bias, const Tensor &mean, const Tensor &rstd, bool need_x,
                                 bool need_weight, bool need_bias)
{
    const int64_t cols = check_norm(x, shape, weight, bias);
    check_norm_backward(dy, x, cols, mean, rstd);
    const auto pt = param_type(x, weight, bias);
    const auto none = [&] { return at::empty({0}, x.options()); };
    return {need_x ? at::empty(x.sizes(), x.options()) : none(),
            need_weight ? at::empty(shape, x.options().dtype(given(weight) ? weight->scalar_type() : pt)) : none(),
            need_bias ? at::empty(shape, x.options().dtype(given(bias) ? bias->scalar_type() : pt)) : none()};
}

// The graph's node, with its members as C++ holds them: the generic Function keeps shapes and flags in a dictionary and costs
// 6 to 12 us more per backward, of the 65 us that forward and backward of a small layer take on the host.
struct LayerNormBackward : public torch::autograd::Node {
    using torch::autograd::Node::Node;
    torch::autograd::SavedVariable x, weight, bias, mean, rstd;
    std::vector<int64_t> shape;
    bool released = false;

    std::string name() const override { return "LayerNormBackward"; }

    void release_variables() override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        x.reset_data();
        weight.reset_data();
        bias.reset_data();
        mean.reset_data();
        rstd.reset_data();
        released = true;
    }

    variable_list apply(variable_list &&grads) override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(3);
        if (!grads[0].defined()) return out;
        TORCH_CHECK(!released, torch::autograd::ERR_BACKWARD_TWICE);
        TORCH_CHECK(!at::GradMode::is_enabled(), "sv3d::layer_norm has no second derivative: create_graph=True asks for one, "
                    "and so does torch.func.grad");
        const Tensor xt = x.unpack();
        optional<Tensor> wt, bt;
        if (const Tensor t = weight.unpack(); t.defined()) wt = t;
        if (const Tensor t = bias.unpack(); t.defined()) bt = t;
        const bool need[3] = {task_should_compute_output(0), wt && task_should_compute_output(1), bt && task_should_compute_output(2)};
        static auto op = find_op<NormOut(const Tensor &, const Tensor &, IntList, const optional<Tensor> &,
                                         const optional<Tensor> &, const Tensor &, const Tensor &, bool, bool, bool)>(
            "sv3d::layer_norm_backward");
        const auto g = op.call(grads[0], xt, shape, wt, bt, mean.unpack(), rstd.unpack(), need[0], need[1], need[2]);
        if (need[0]) out[0] = std::get<0>(g);
        if (need[1]) out[1] = std::get<1>(g);
        if (need[2]) out[2] = std::get<2>(g);
        return out;
    }
};

Tensor layer_norm_autograd(const Tensor &x, IntList shape, const optional<Tensor> &weight, const optional<Tensor> &bias,
                           double eps, bool f32_out)
{
    const Tensor w = given(weight) ? *weight : Tensor(), b = given(bias) ? *bias : Tensor();
    for (const Tensor *t : {&x, &w, &b})
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), "sv3d::layer_norm has no forward-mode derivative");
    if (!torch::autograd::compute_requires_grad(x, w, b)) {
        // no gradient will be asked for: without the statistics of the rows
        at::AutoDispatchBelowADInplaceOrView guard;
        static auto op = find_op<Tensor(const Tensor &, IntList, const optional<Tensor> &, const optional<Tensor> &, double, bool)>(
            "sv3d::layer_norm");
        return op.call(x, shape, weight, bias, eps, f32_out);
    }
    auto node = std::shared_ptr<LayerNormBackward>(new LayerNormBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, w, b));
    Tensor y, mean, rstd;
    {
        at::AutoDispatchBelowADInplaceOrView guard;
        static auto op = find_op<NormOut(const Tensor &, IntList, const optional<Tensor> &, const optional<Tensor> &, double,
                                         bool)>("sv3d::layer_norm_stats");
        std::tie(y, mean, rstd) = op.call(x, shape, weight, bias, eps, f32_out);
    }
    node->x = torch::autograd::SavedVariable(x, false);
    node->weight = torch::autograd::SavedVariable(w, false);
    node->bias = torch::autograd::SavedVariable(b, false);
    node->mean = torch::autograd::SavedVariable(mean, false);
    node->rstd = torch::autograd::SavedVariable(rstd, false);
    node->shape = shape.vec();
    torch::autograd::set_history(y, node);
    return y;
}

// ---- optimizer ------------------------------------------------------------------------------------
using TensorList = at::TensorList;

bool same_layout(const Tensor &a, const Tensor &b)
{
    if (a.sizes() != b.sizes()) return false;
    for (int64_t d = 0; d < a.dim(); ++d)
        if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
    return true;
}

// The elements of a tensor in the order that they lie in memory, if nothing lies between them.
void check_dense(const Tensor &t, const char *name, size_t i)
{
    TORCH_CHECK_VALUE(t.layout() == at::kStrided && t.is_non_overlapping_and_dense(), name, "[", i,
                      "] must be a dense tensor without gaps or overlap, got sizes ", t.sizes(), " strides ", t.strides());
}

Tensor grad_square_sums_gpu(TensorList grads)
{
    TORCH_CHECK_VALUE(!grads.empty(), "grads must not be empty");
    std::vector<sv3d_adamw_tensor> list(grads.size());
    std::vector<Tensor> keep;
    Launch L(grads[0]);
    for (size_t i = 0; i < grads.size(); ++i) {
        const Tensor &g = grads[i];
        TORCH_CHECK_VALUE(g.layout() == at::kStrided, "grads[", i, "] must be a dense tensor");
        same_device(grads[0], g, "grads");
        list[i] = {};
        list[i].type = type_of(g, "grads");
        list[i].numel = g.numel();
        if (g.is_non_overlapping_and_dense()) {
            list[i].grad = ptr(g);
        } else {
            keep.push_back(g.contiguous());
            list[i].grad = ptr(keep.back());
        }
    }
    int32_t count = 0;
    check_status(sv3d_grad_square_sums_count(list.data(), (int32_t)list.size(), &count), "sv3d_grad_square_sums_count");
    Tensor sums = at::empty({count}, grads[0].options().dtype(at::kDouble));
    check_status(sv3d_grad_square_sums(list.data(), (int32_t)list.size(), (double *)ptr(sums), count, L.stream),
                 "sv3d_grad_square_sums");
    return sums;
}

Tensor grad_square_sums_meta(TensorList grads)
{
    std::vector<sv3d_adamw_tensor> list(grads.size());
    for (size_t i = 0; i < grads.size(); ++i) {
        list[i] = {};
        list[i].type = type_of(grads[i], "grads");
        list[i].numel = grads[i].numel();
        list[i].grad = &list[i];            // the count looks at sizes and types only
    }
    int32_t count = 0;
    check_status(sv3d_grad_square_sums_count(list.data(), (int32_t)list.size(), &count), "sv3d_grad_square_sums_count");
    return at::empty({count}, grads[0].options().dtype(at::kDouble));
}

const float *scalar_ptr(const optional<Tensor> &t, const Tensor &ref, const char *name)
{
    if (!given(t)) return nullptr;
    TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat && t->numel() == 1, name, " must hold one float32, got ", t->scalar_type(),
                      " ", t->sizes());
    same_device(ref, *t, name);
    return t->data_ptr<float>();
}

void check_adamw(TensorList params, TensorList grads, TensorList exp_avgs, TensorList exp_avg_sqs, TensorList scales,
                 TensorList steps)
{
    const size_t n = params.size();
    TORCH_CHECK_VALUE(n > 0, "params must not be empty");
    TORCH_CHECK_VALUE(grads.size() == n && exp_avgs.size() == n && exp_avg_sqs.size() == n && steps.size() == n &&
                          (scales.empty() || scales.size() == n),
                      "params, grads, exp_avgs, exp_avg_sqs, steps (and scales) must be lists of one length");
    for (size_t i = 0; i < n; ++i) {
        const Tensor &p = params[i], &g = grads[i], &m = exp_avgs[i], &v = exp_avg_sqs[i], &s = steps[i];
        type_of(p, "params");
        check_dense(p, "params", i);
        TORCH_CHECK_VALUE(g.layout() == at::kStrided && g.scalar_type() == p.scalar_type() && g.sizes() == p.sizes(), "grads[", i,
                          "] must be a dense ", p.scalar_type(), " ", p.sizes(), ", got ", g.layout(), " ", g.scalar_type(), " ",
                          g.sizes());
        const bool eight = m.scalar_type() == at::kByte;
        TORCH_CHECK_VALUE((eight || m.scalar_type() == at::kFloat) && v.scalar_type() == m.scalar_type(), "exp_avgs[", i,
                          "] and exp_avg_sqs[", i, "] must both be float32 or both uint8, got ", m.scalar_type(), " and ",
                          v.scalar_type());
        TORCH_CHECK_VALUE(same_layout(p, m) && same_layout(p, v), "exp_avgs[", i, "] and exp_avg_sqs[", i,
                          "] must have the sizes and strides of params[", i, "]: ", p.sizes(), " ", p.strides());
        TORCH_CHECK_VALUE(s.scalar_type() == at::kFloat && s.numel() == 1, "steps[", i, "] must hold one float32");
        for (const Tensor *t : {&p, &g, &m, &v, &s}) same_device(params[0], *t, "every tensor of the step");
        if (!eight) continue;
        TORCH_CHECK_VALUE(!scales.empty(), "scales must be given with 8-bit moments");
        const int64_t blocks = (p.numel() + SV3D_STATE_BLOCK - 1) / SV3D_STATE_BLOCK;
        const Tensor &e = scales[i];
        TORCH_CHECK_VALUE(e.scalar_type() == at::kByte && e.is_contiguous() && e.numel() == 2 * blocks, "scales[", i,
                          "] must be contiguous uint8 [", blocks, ",2], got ", e.scalar_type(), " ", e.sizes());
        same_device(params[0], e, "scales");
    }
}

// Nothing may be written twice: a tensor that is in the lists twice, or overlaps another one, is updated by two
// workgroups at once.  Nor may a gradient lie where something is written; two weights may share one.
void check_apart(const std::vector<sv3d_adamw_tensor> &list)
{
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;
    spans.reserve(5 * list.size());
    const auto add = [&](const void *at, int64_t bytes) {
        if (at && bytes > 0) spans.emplace_back((uintptr_t)at, (uintptr_t)at + (uintptr_t)bytes);
    };
    for (const auto &t : list) {
        const int64_t state = t.state_bits / 8;
        add(t.param, t.numel * (t.type == SV3D_F32 ? 4 : 2));
        add(t.exp_avg, t.numel * state);
        add(t.exp_avg_sq, t.numel * state);
        add(t.scales, (t.numel + SV3D_STATE_BLOCK - 1) / SV3D_STATE_BLOCK * 2);
        add(t.step, 4);
    }
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i)
        TORCH_CHECK_VALUE(spans[i - 1].second <= spans[i].first,
                          "a weight, moment, scale or step count is in the lists twice, or overlaps another one");
    for (const auto &t : list) {
        if (!t.grad || t.numel == 0) continue;
        const uintptr_t from = (uintptr_t)t.grad, to = from + (uintptr_t)(t.numel * (t.type == SV3D_F32 ? 4 : 2));
        const auto behind = std::lower_bound(spans.begin(), spans.end(), std::make_pair(to, (uintptr_t)0));
        TORCH_CHECK_VALUE(behind == spans.begin() || (behind - 1)->second <= from,
                          "a gradient overlaps a weight, moment, scale or step count");
    }
}

Tensor adamw_step_gpu(TensorList params, TensorList grads, TensorList exp_avgs, TensorList exp_avg_sqs, TensorList scales,
                      TensorList steps, const optional<Tensor> &lr_tensor, const optional<Tensor> &grad_scale,
                      const optional<Tensor> &found_inf, const optional<Tensor> &square_sums, double lr, double beta1,
                      double beta2, double eps, double weight_decay, double max_norm, bool maximize, int64_t seed)
{
    check_adamw(params, grads, exp_avgs, exp_avg_sqs, scales, steps);
    const Tensor &ref = params[0];
    Launch L(ref);
    std::vector<sv3d_adamw_tensor> list(params.size());
    std::vector<Tensor> keep;
    for (size_t i = 0; i < list.size(); ++i) {
        sv3d_adamw_tensor &t = list[i];
        const bool eight = exp_avgs[i].scalar_type() == at::kByte;
        const void *g = ptr(grads[i]);
        if (!same_layout(params[i], grads[i])) {        // a gradient laid out otherwise than its weight is copied
            keep.push_back(at::empty_strided(params[i].sizes(), params[i].strides(), grads[i].options()).copy_(grads[i]));
            g = ptr(keep.back());
        }
        t = {ptr(params[i]), g, ptr(exp_avgs[i]), ptr(exp_avg_sqs[i]), eight ? (uint8_t *)ptr(scales[i]) : nullptr,
             steps[i].data_ptr<float>(), params[i].numel(), code_of(params[i].scalar_type()), eight ? 8 : 32};
    }
    check_apart(list);
    sv3d_adamw_params p = {};
    p.lr = lr;
    p.beta1 = beta1;
    p.beta2 = beta2;
    p.eps = eps;
    p.weight_decay = weight_decay;
    p.max_norm = max_norm;
    p.lr_device = scalar_ptr(lr_tensor, ref, "lr");
    p.grad_scale = scalar_ptr(grad_scale, ref, "grad_scale");
    p.found_inf = scalar_ptr(found_inf, ref, "found_inf");
    p.maximize = maximize ? 1 : 0;
    p.seed = (uint32_t)seed;
    Tensor norm = at::empty({}, ref.options().dtype(at::kFloat));
    if (max_norm > 0.0) p.total_norm = norm.data_ptr<float>();
    Tensor none;
    if (max_norm > 0.0 && given(square_sums)) {
        TORCH_CHECK_VALUE(square_sums->scalar_type() == at::kDouble && square_sums->is_contiguous() && square_sums->dim() == 1,
                          "square_sums must be what grad_square_sums returns");
        same_device(ref, *square_sums, "square_sums");
        if (square_sums->numel() == 0) none = at::empty({1}, square_sums->options());       // the norm of nothing
        p.square_sums = none.defined() ? none.data_ptr<double>() : square_sums->data_ptr<double>();
        p.num_square_sums = (int32_t)square_sums->numel();
    }
    size_t bytes = 0;
    check_status(sv3d_adamw_workspace(&p, list.data(), (int32_t)list.size(), &bytes), "sv3d_adamw_workspace");
    Tensor ws = at::empty({(int64_t)bytes}, ref.options().dtype(at::kByte));
    check_status(sv3d_adamw_step(&p, list.data(), (int32_t)list.size(), ws.data_ptr(), bytes, L.stream), "sv3d_adamw_step");
    // a graph that saved a weight for its backward has to see that the weight is another one now
    for (const auto *tensors : {&params, &exp_avgs, &exp_avg_sqs, &scales, &steps})
        for (const Tensor &t : *tensors)
            if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    return norm;
}

Tensor adamw_step_meta(TensorList params, TensorList grads, TensorList exp_avgs, TensorList exp_avg_sqs, TensorList scales,
                       TensorList steps, const optional<Tensor> &, const optional<Tensor> &, const optional<Tensor> &,
                       const optional<Tensor> &, double, double, double, double, double, double, bool, int64_t)
{
    check_adamw(params, grads, exp_avgs, exp_avg_sqs, scales, steps);
    return at::empty({}, params[0].options().dtype(at::kFloat));
}

// Without kernels of their own these operators would pass autograd's generic check, which takes the lists apart once more (five
// lists of 72 tensors: 71 us with that check, 36 us without).
Tensor adamw_step_autograd(TensorList params, TensorList grads, TensorList exp_avgs, TensorList exp_avg_sqs, TensorList scales,
                           TensorList steps, const optional<Tensor> &lr_tensor, const optional<Tensor> &grad_scale,
                           const optional<Tensor> &found_inf, const optional<Tensor> &square_sums, double lr, double beta1,
                           double beta2, double eps, double weight_decay, double max_norm, bool maximize, int64_t seed)
{
    if (at::GradMode::is_enabled())
        for (const auto *tensors : {&params, &exp_avgs, &exp_avg_sqs})
            for (const Tensor &t : *tensors)
                TORCH_CHECK(!t.requires_grad(), "sv3d::adamw_step changes tensors that require a gradient: call it under torch.no_grad()");
    at::AutoDispatchBelowADInplaceOrView guard;
    using O = const optional<Tensor> &;
    static auto op = find_op<Tensor(TensorList, TensorList, TensorList, TensorList, TensorList, TensorList, O, O, O, O, double,
                                    double, double, double, double, double, bool, int64_t)>("sv3d::adamw_step");
    return op.call(params, grads, exp_avgs, exp_avg_sqs, scales, steps, lr_tensor, grad_scale, found_inf, square_sums, lr, beta1,
                   beta2, eps, weight_decay, max_norm, maximize, seed);
}

int64_t check_moments(const Tensor &exp_avg, const Tensor &exp_avg_sq, const Tensor &scales)
{
    TORCH_CHECK_VALUE(exp_avg.scalar_type() == at::kByte && exp_avg_sq.scalar_type() == at::kByte && same_layout(exp_avg, exp_avg_sq) &&
                          exp_avg.layout() == at::kStrided && exp_avg.is_non_overlapping_and_dense(),
                      "exp_avg and exp_avg_sq must be dense uint8 tensors of one layout");
    const int64_t n = exp_avg.numel(), blocks = (n + SV3D_STATE_BLOCK - 1) / SV3D_STATE_BLOCK;
    TORCH_CHECK_VALUE(scales.scalar_type() == at::kByte && scales.is_contiguous() && scales.numel() == 2 * blocks,
                      "scales must be contiguous uint8 [", blocks, ",2], got ", scales.scalar_type(), " ", scales.sizes());
    same_device(exp_avg, exp_avg_sq, "exp_avg_sq");
    same_device(exp_avg, scales, "scales");
    return n;
}

std::tuple<Tensor, Tensor> moment_values_gpu(const Tensor &exp_avg, const Tensor &exp_avg_sq, const Tensor &scales)
{
    const int64_t n = check_moments(exp_avg, exp_avg_sq, scales);
    Launch L(exp_avg);
    Tensor m = at::empty_like(exp_avg, exp_avg.options().dtype(at::kBFloat16)), v = at::empty_like(m);
    check_status(sv3d_moment_values((const uint8_t *)ptr(exp_avg), (const uint8_t *)ptr(exp_avg_sq), (const uint8_t *)ptr(scales), n,
                                    ptr(m), ptr(v), L.stream),
                 "sv3d_moment_values");
    return {m, v};
}

std::tuple<Tensor, Tensor> moment_values_meta(const Tensor &exp_avg, const Tensor &exp_avg_sq, const Tensor &scales)
{
    check_moments(exp_avg, exp_avg_sq, scales);
    Tensor m = at::empty_like(exp_avg, exp_avg.options().dtype(at::kBFloat16));
    return {m, at::empty_like(m)};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(sv3d, m)
{
    m.def("layer_norm(Tensor x, int[] normalized_shape, Tensor? weight, Tensor? bias, float eps, bool f32_out) -> Tensor");
    m.def("layer_norm_stats(Tensor x, int[] normalized_shape, Tensor? weight, Tensor? bias, float eps, bool f32_out) "
          "-> (Tensor, Tensor, Tensor)");
    m.def("layer_norm_backward(Tensor grad_y, Tensor x, int[] normalized_shape, Tensor? weight, Tensor? bias, Tensor mean, "
          "Tensor rstd, bool need_x, bool need_weight, bool need_bias) -> (Tensor, Tensor, Tensor)");
    m.def("grad_square_sums(Tensor[] grads) -> Tensor");
    m.def("adamw_step(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] exp_avgs, Tensor(c!)[] exp_avg_sqs, "
          "Tensor(d!)[] scales, Tensor(e!)[] steps, Tensor? lr_tensor, Tensor? grad_scale, Tensor? found_inf, "
          "Tensor? square_sums, float lr, float beta1, float beta2, float eps, float weight_decay, float max_norm, "
          "bool maximize, int seed) -> Tensor");
    m.def("moment_values(Tensor exp_avg, Tensor exp_avg_sq, Tensor scales) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(sv3d, CUDA, m)
{
    m.impl("layer_norm", layer_norm_gpu);
    m.impl("layer_norm_stats", layer_norm_stats_gpu);
    m.impl("layer_norm_backward", layer_norm_backward_gpu);
    m.impl("grad_square_sums", grad_square_sums_gpu);
    m.impl("adamw_step", adamw_step_gpu);
    m.impl("moment_values", moment_values_gpu);
}

TORCH_LIBRARY_IMPL(sv3d, Meta, m)
{
    m.impl("layer_norm", layer_norm_meta);
    m.impl("layer_norm_stats", layer_norm_stats_meta);
    m.impl("layer_norm_backward", layer_norm_backward_meta);
    m.impl("grad_square_sums", grad_square_sums_meta);
    m.impl("adamw_step", adamw_step_meta);
    m.impl("moment_values", moment_values_meta);
}

TORCH_LIBRARY_IMPL(sv3d, Autograd, m)
{
    m.impl("layer_norm", layer_norm_autograd);
    m.impl("adamw_step", adamw_step_autograd);
    // no gradients: what comes back requires none
    m.impl("layer_norm_stats", torch::CppFunction::makeFallthrough());
    m.impl("layer_norm_backward", torch::CppFunction::makeFallthrough());
    m.impl("grad_square_sums", torch::CppFunction::makeFallthrough());
    m.impl("moment_values", torch::CppFunction::makeFallthrough());
}
