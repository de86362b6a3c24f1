// Calls of the routing and layer entry points from torch, with their autograd nodes.
//
// A small layer takes a few microseconds on the card; a call through Python takes ten, a backward pass through Python nodes some
// thirty more.  Here the arguments are looked over, the results allocated and the entry points of mtp_accel.h called without
// Python between them: a forward and a backward pass of a 64 x 96 layer with gelu take the host 62 us, 35 of which the engine takes
// for a node that does nothing.  A call whose arguments are not as they have to be returns None: the Python front end then finds
// out what is wrong and raises.
#include <torch/extension.h>

#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <array>
#include <optional>

#include "mtp_accel.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

constexpr int64_t MOST = 0x7fffffff;
constexpr int64_t MOST_SIZE = 65536, MOST_SETS = 65535, MOST_MODALITIES = 4096, MOST_TOPK = 128;
enum { NONE = 0, RELU = 1 };

void *stream_of(const Tensor &t) {
    return static_cast<void *>(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream());
}
void *at_(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
void check(int rc, const char *what) { TORCH_CHECK(rc == MTP_OK, what, " failed (rc=", rc, "): ", mtp_last_error()); }

int type_code(const Tensor &t) {
    switch (t.scalar_type()) {
        case at::kFloat: return MTP_FLOAT;
        case at::kBFloat16: return MTP_BFLOAT16;
        case at::kHalf: return MTP_HALF;
        default: return -1;
    }
}
// elements from row to row of a matrix with contiguous rows that do not overlap, -1 otherwise
int64_t row_distance(const Tensor &t) {
    const int64_t rows = t.size(0), cols = t.size(1);
    if (rows <= 1 && (cols <= 1 || t.stride(1) == 1)) return cols > 1 ? cols : 1;
    if ((cols > 1 && t.stride(1) != 1) || (rows > 1 && t.stride(0) < cols)) return -1;
    return t.stride(0);
}
// (a tensor with the negative bit holds the negatives of its values)
bool matrix(const Tensor &t) { return t.is_cuda() && t.dim() == 2 && t.layout() == at::kStrided && type_code(t) >= 0 && !t.is_neg(); }
bool like(const Tensor &t, at::ScalarType type, const Tensor &ref, at::IntArrayRef shape) {
    return t.scalar_type() == type && t.device() == ref.device() && t.sizes() == shape && t.is_contiguous() && !t.is_neg();
}
// A result or a workspace on ref's device.  Past the dispatcher, which would take the host as long again as the allocation; each has a
// storage of its own, so that it can grow, move to another stream and go by itself.
Tensor fresh(const Tensor &ref, at::ScalarType type, at::IntArrayRef sizes) {
    return Tensor(at::detail::empty_cuda(sizes, type, ref.device(), std::nullopt));
}
Tensor workspace(int64_t bytes, const Tensor &ref) { return bytes > 0 ? fresh(ref, at::kByte, {bytes}) : Tensor(); }

// Under capture a backward pass must not meet a node that was made on another stream: the engine would make that stream wait for
// the captured one, which fails inside its own thread and ends the process.  Such a node exists where an input is a result
// from outside the capture, or a leaf that a result from outside still refers to.
void refuse_foreign_nodes(const char *what, std::initializer_list<const Tensor *> inputs) {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    for (const Tensor *t : inputs) {
        if (!t->defined() || !t->requires_grad()) continue;
        const auto node = t->grad_fn() ? t->grad_fn() : torch::autograd::impl::try_get_grad_accumulator(*t);
        if (!node) continue;
        const auto stream = node->stream();
        TORCH_CHECK(!stream || *stream == c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t->device().index()).unwrap(), what,
                    ": an input belongs to an autograd graph that was begun outside this capture; its backward pass cannot be captured "
                    "(let go of the eager results that refer to it first)");
    }
}

// A tracer records what goes through the dispatcher.  The kernels do not: a trace would hold the results' allocation without what fills
// it, or their values as constants.
void refuse_tracing(const char *what) {
    TORCH_CHECK(!torch::jit::tracer::isTracing() &&
                    !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(),
                what, " cannot be traced: its kernels are not seen by a tracer");
}

// no derivative in forward mode: a tangent must not get lost in silence
void refuse_tangents(const char *what, std::initializer_list<const Tensor *> inputs) {
    for (const Tensor *t : inputs)
        TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), what, " has no derivative in forward mode");
}

// A node of the operators below with an edge to each of its inputs.  (Nodes of their own rather than torch::autograd::Function: its
// bookkeeping takes the host some 5 us of a forward and a backward pass.)
template <typename N, typename... Inputs>
std::shared_ptr<N> node_with_edges(const Inputs &...inputs) {
    std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(inputs...));
    return node;
}

// Hooks on saved tensors may give back what they like: what the kernels read has to be what the node kept.  `rows`: rows at any
// distance will do.
void refuse_changed(const char *what, const Tensor &t, at::ScalarType type, c10::Device device, at::IntArrayRef sizes, bool rows = false) {
    TORCH_CHECK(t.defined() && t.layout() == at::kStrided && t.scalar_type() == type && t.device() == device && t.sizes() == sizes && !t.is_neg() &&
                    (rows ? row_distance(t) >= 0 : t.is_contiguous()),
                what, ": a saved tensor has come back from its hook with another layout, type, size or device");
}

// What a backward pass returns can be differentiated no further: trying to says so.  `from`: what it was computed from.
variable_list no_further(variable_list out, variable_list from, const char *what) {
    if (!at::GradMode::is_enabled()) return out;
    const size_t n = out.size();
    auto node = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " has no second derivative",
                                                                (int64_t)(n + from.size()));
    variable_list in = std::move(out);
    for (auto &t : from) in.push_back(t);  // the error stands between the result and these
    variable_list got = (*node)(std::move(in));
    got.resize(n);
    return got;
}

// ---- linear layers ----
struct Sizes {
    int code, act;
    int64_t rows, in, out, sets;
};

Tensor run_linear(const Sizes &z, const Tensor &x, const Tensor &w, const Tensor &bias, const Tensor &residual, const Tensor &offsets,
                  Tensor *pre, Tensor *laid_out = nullptr) {
    const Tensor y = fresh(x, x.scalar_type(), {z.rows, z.out});
    if (pre != nullptr) *pre = fresh(x, x.scalar_type(), {z.rows, z.out});
    const int64_t ldx = row_distance(x);
    const int64_t bytes = mtp_linear_workspace_bytes(z.code, MTP_LINEAR_FORWARD, z.rows, (int)z.in, (int)z.out, (int)z.sets, at_(x),
                                                     ldx, at_(w), z.in);
    const Tensor ws = workspace(bytes, x);
    check(mtp_linear(z.code, at_(x), z.rows, (int)z.in, ldx, at_(w), (int)z.out, at_(bias), z.act, at_(residual),
                     residual.defined() ? row_distance(residual) : 0, static_cast<const int32_t *>(at_(offsets)), (int)z.sets, at_(y),
                     pre != nullptr ? at_(*pre) : nullptr, at_(ws), (size_t)bytes, stream_of(x)),
          "mtp_linear");
    if (laid_out != nullptr) *laid_out = ws;
    return y;
}

struct LinearNode : Node {
    Sizes z;
    bool has_bias, has_residual, pre_kept, offsets_kept, rows_kept, weights_kept;
    SavedVariable x_, w_, pre_, offsets_, rows_, weights_;

    std::string name() const override { return "LinearBackward"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable *v : {&x_, &w_, &pre_, &offsets_, &rows_, &weights_}) v->reset_data();
    }
    // edges: x, weight, bias, residual
    variable_list apply(variable_list &&grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        if (!grads[0].defined()) return variable_list(4);
        const Tensor x = x_.unpack(), w = w_.unpack(), pre = pre_.unpack(getptr()), offsets = offsets_.unpack();
        const Tensor rows = rows_.unpack(), weights = weights_.unpack();
        const auto type = grads[0].scalar_type();
        const auto device = grads[0].device();
        refuse_changed("linear", x, type, device, {z.rows, z.in}, true);
        if (offsets_kept) {
            refuse_changed("linear", w, type, device, {z.sets, z.out, z.in});
            refuse_changed("linear", offsets, at::kInt, device, {z.sets + 1});
        } else {
            refuse_changed("linear", w, type, device, {z.out, z.in});
        }
        if (pre_kept) refuse_changed("linear", pre, type, device, {z.rows, z.out});
        if (rows_kept) refuse_changed("linear", rows, type, device, {z.rows, z.in}, true);
        if (weights_kept) refuse_changed("linear", weights, type, device, {z.sets * z.out, z.in}, true);
        Tensor dx, dw, db, dr;
        {
            at::NoGradGuard off;
            const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
            const Tensor g = grads[0].resolve_neg().contiguous();
            const bool want_x = task_should_compute_output(0), want_b = has_bias && task_should_compute_output(2);
            const bool want_w = task_should_compute_output(1) || want_b;
            const int32_t *sets = static_cast<const int32_t *>(at_(offsets));
            if (want_x || want_w) {
                const Tensor &xs = rows.defined() ? rows : x, &wt = weights.defined() ? weights : w;
                // hooks on saved tensors may have given the copies other distances
                const int64_t ldx = row_distance(xs), ldw = weights.defined() ? row_distance(weights) : z.in;
                const int64_t ws_bytes = mtp_linear_backward_workspace_bytes(z.code, z.rows, (int)z.in, (int)z.out, (int)z.sets, z.act,
                                                                             at_(g), at_(wt), ldw, at_(xs), ldx, want_x, want_w);
                const bool many = offsets.defined();
                const std::array<int64_t, 2> x_size{z.rows, z.in};
                const std::array<int64_t, 3> w_size{z.sets, z.out, z.in};
                const auto w_sizes = at::IntArrayRef(w_size).slice(many ? 0 : 1), b_sizes = w_sizes.slice(0, w_sizes.size() - 1);
                if (want_x) dx = fresh(x, type, x_size);
                if (want_w) dw = fresh(x, type, w_sizes);
                if (want_b) db = fresh(x, type, b_sizes);
                const Tensor ws = workspace(ws_bytes, x);
                if (want_w || z.rows > 0)  // else dx has no elements
                    check(mtp_linear_backward(z.code, at_(g), at_(pre), z.act, at_(xs), z.rows, (int)z.in, ldx, at_(wt), (int)z.out,
                                              ldw, sets, (int)z.sets, at_(dx), at_(dw), at_(db), at_(ws), (size_t)ws_bytes, stream_of(x)),
                          "mtp_linear_backward");
            }
            if (has_residual && task_should_compute_output(3)) {
                if (offsets.defined()) {  // rows behind the last set have none
                    dr = fresh(g, type, g.sizes());
                    check(mtp_linear_mask_rows(z.code, at_(g), z.rows, (int)z.out, sets, (int)z.sets, at_(dr), stream_of(x)),
                          "mtp_linear_mask_rows");
                } else {
                    dr = g;
                }
            }
            if (!task_should_compute_output(1)) dw = Tensor();
        }
        return no_further({dx, dw, db, dr}, {x, w, grads[0]}, "linear");
    }
};

Tensor linear_with_node(const Tensor &x, const Tensor &w, const Tensor &bias, const Tensor &residual, const Tensor &offsets,
                        const Sizes &z) {
    const auto node = node_with_edges<LinearNode>(x, w, bias, residual);
    // relu's slope can be read off y where nothing was added to it
    const bool from_y = z.act == RELU && !residual.defined();
    Tensor pre, ws, y, rows, weights;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        y = run_linear(z, x, w, bias, residual, offsets, z.act != NONE && !from_y ? &pre : nullptr, &ws);
        // rows that do not start where the products want them have been laid out there: once for both passes
        const int64_t ld = (z.in + 7) / 8 * 8;
        if (ws.defined()) {
            const Tensor all = ws.view(x.scalar_type());
            int64_t at = 0;
            auto take = [&](const Tensor &t, int64_t n, int64_t distance) {
                if (mtp_linear_rows_aligned(z.code, at_(t), distance)) return Tensor();
                const int64_t from = at;
                at += (n * ld * x.element_size() + 255) / 256 * 256 / x.element_size();
                return all.as_strided({n, z.in}, {ld, 1}, from);
            };
            rows = take(x, z.rows, row_distance(x));
            weights = take(w, z.sets * z.out, z.in);
        }
    }
    torch::autograd::set_history(y, node);
    node->z = z;
    node->has_bias = bias.defined();
    node->has_residual = residual.defined();
    node->x_ = SavedVariable(x, false);
    node->w_ = SavedVariable(w, false);
    node->pre_kept = from_y || pre.defined();
    node->offsets_kept = offsets.defined();
    node->rows_kept = rows.defined();
    node->weights_kept = weights.defined();
    if (from_y) node->pre_ = SavedVariable(y, true);
    else if (pre.defined()) node->pre_ = SavedVariable(pre, false);
    if (offsets.defined()) node->offsets_ = SavedVariable(offsets, false);
    if (rows.defined()) node->rows_ = SavedVariable(rows, false);
    if (weights.defined()) node->weights_ = SavedVariable(weights, false);
    return y;
}

std::optional<Tensor> linear(const Tensor &x, const Tensor &w, const std::optional<Tensor> &bias_, int act,
                             const std::optional<Tensor> &residual_, const std::optional<Tensor> &offsets_) {
    refuse_tracing("linear");
    const Tensor bias = bias_.value_or(Tensor()), residual = residual_.value_or(Tensor()), offsets = offsets_.value_or(Tensor());
    const bool many = offsets.defined();
    if (!matrix(x) || row_distance(x) < 0 || w.dim() != (many ? 3 : 2) || !w.is_contiguous() || w.is_neg() || w.scalar_type() != x.scalar_type() ||
        w.device() != x.device())
        return std::nullopt;
    const Sizes z{type_code(x), act, x.size(0), x.size(1), w.size(many ? 1 : 0), many ? w.size(0) : 1};
    if (w.size(many ? 2 : 1) != z.in || z.rows > MOST || z.in < 1 || z.in > MOST_SIZE || z.out < 1 || z.out > MOST_SIZE || z.sets < 1 ||
        z.sets > MOST_SETS)
        return std::nullopt;
    if (many && !like(offsets, at::kInt, x, {z.sets + 1})) return std::nullopt;
    if (bias.defined() && !like(bias, x.scalar_type(), x, w.sizes().slice(0, w.dim() - 1))) return std::nullopt;
    if (residual.defined() && (!matrix(residual) || residual.scalar_type() != x.scalar_type() || residual.device() != x.device() ||
                               residual.size(0) != z.rows || residual.size(1) != z.out || row_distance(residual) < 0))
        return std::nullopt;
    refuse_tangents("linear", {&x, &w, &bias, &residual});
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
    if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || (bias.defined() && bias.requires_grad()) ||
                                       (residual.defined() && residual.requires_grad())))
    {
        refuse_foreign_nodes("linear", {&x, &w, &bias, &residual});
        return linear_with_node(x, w, bias, residual, offsets, z);
    }
    return run_linear(z, x, w, bias, residual, offsets, nullptr);
}

// ---- router ----
struct RouteNode : Node {
    bool normalize;
    int64_t modalities;
    at::ScalarType type;
    SavedVariable scores_, ids_, weights_, stats_;

    std::string name() const override { return "RouteTopkBackward"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable *v : {&scores_, &ids_, &weights_, &stats_}) v->reset_data();
    }
    variable_list apply(variable_list &&grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        if (!grads[0].defined()) return variable_list(1);
        const Tensor scores = scores_.unpack(), ids = ids_.unpack(), weights = weights_.unpack(getptr()), stats = stats_.unpack();
        const auto device = grads[0].device();
        const int64_t n = grads[0].size(0), k = grads[0].size(1);
        refuse_changed("route_topk", scores, type, device, {n, modalities}, true);
        refuse_changed("route_topk", ids, at::kInt, device, {n, k});
        refuse_changed("route_topk", weights, at::kFloat, device, {n, k});
        refuse_changed("route_topk", stats, at::kFloat, device, {n, 2});
        Tensor out;
        {
            at::NoGradGuard off;
            const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(scores.device());
            const Tensor g = grads[0].resolve_neg().contiguous();
            out = fresh(scores, type, {n, modalities});
            check(mtp_route_topk_grad(type_code(scores), at_(scores), scores.size(0), (int)scores.size(1), row_distance(scores),
                                      (int)ids.size(1), normalize, static_cast<const int32_t *>(at_(ids)),
                                      static_cast<const float *>(at_(weights)), static_cast<const float *>(at_(stats)),
                                      static_cast<const float *>(at_(g)), at_(out), stream_of(scores)),
                  "mtp_route_topk_grad");
        }
        return no_further({out}, {scores, grads[0]}, "route_topk");
    }
};

std::optional<std::tuple<Tensor, Tensor>> route_topk(const Tensor &scores, int64_t k, bool normalize) {
    refuse_tracing("route_topk");
    if (!matrix(scores)) return std::nullopt;
    const int64_t n = scores.size(0), e = scores.size(1), ld = row_distance(scores);
    if (ld < 0 || n > MOST || e < 1 || e > MOST_MODALITIES || k < 1 || k > e || k > MOST_TOPK) return std::nullopt;
    refuse_tangents("route_topk", {&scores});
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(scores.device());
    const bool train = at::GradMode::is_enabled() && scores.requires_grad();
    if (train) refuse_foreign_nodes("route_topk", {&scores});
    Tensor ids, weights, stats;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        ids = fresh(scores, at::kInt, {n, k});
        weights = fresh(scores, at::kFloat, {n, k});
        if (train) stats = fresh(scores, at::kFloat, {n, 2});
        check(mtp_route_topk(type_code(scores), at_(scores), n, (int)e, ld, (int)k, normalize, static_cast<int32_t *>(at_(ids)),
                             static_cast<float *>(at_(weights)), static_cast<float *>(at_(stats)), stream_of(scores)),
              "mtp_route_topk");
    }
    if (train) {
        const auto node = node_with_edges<RouteNode>(scores);
        torch::autograd::set_history(weights, node);
        node->normalize = normalize;
        node->modalities = e;
        node->type = scores.scalar_type();
        node->scores_ = SavedVariable(scores, false);
        node->ids_ = SavedVariable(ids, false);
        node->weights_ = SavedVariable(weights, true);
        node->stats_ = SavedVariable(stats, false);
    }
    return std::make_tuple(ids, weights);
}

// ---- pairs ----
std::optional<std::tuple<Tensor, Tensor, Tensor>> sort_pairs(const Tensor &ids, int64_t e) {
    refuse_tracing("sort_pairs");
    if (!ids.is_cuda() || ids.scalar_type() != at::kInt || ids.dim() != 2 || !ids.is_contiguous() || ids.is_neg() || e < 1 || e > MOST_MODALITIES ||
        ids.numel() > MOST)
        return std::nullopt;
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(ids.device());
    const int64_t pairs = ids.numel(), bytes = mtp_sort_pairs_workspace_bytes(pairs, (int)e);
    const Tensor offsets = fresh(ids, at::kInt, {e + 1}), order = fresh(ids, at::kInt, {pairs});
    const Tensor position = fresh(ids, at::kInt, ids.sizes()), ws = workspace(bytes, ids);
    check(mtp_sort_pairs(static_cast<const int32_t *>(at_(ids)), pairs, (int)e, static_cast<int32_t *>(at_(offsets)),
                         static_cast<int32_t *>(at_(order)), static_cast<int32_t *>(at_(position)), at_(ws), (size_t)bytes,
                         stream_of(ids)),
          "mtp_sort_pairs");
    return std::make_tuple(offsets, order, position);
}

// the device's count of pairs that have a modality
const int32_t *held(const Tensor &offsets) { return static_cast<const int32_t *>(at_(offsets)) + (offsets.numel() - 1); }
const int32_t *places(const Tensor &position) { return static_cast<const int32_t *>(at_(position)); }

Tensor run_dispatch(const Tensor &x, const Tensor &position, const Tensor &offsets) {
    const int64_t n = x.size(0), d = x.size(1), k = position.size(1);
    Tensor rows = fresh(x, x.scalar_type(), {n * k, d});
    check(mtp_dispatch_rows(type_code(x), at_(x), n, (int)d, row_distance(x), (int)k, places(position), held(offsets), at_(rows),
                            stream_of(x)),
          "mtp_dispatch_rows");
    return rows;
}
Tensor run_combine(const Tensor &rows, const Tensor &position, const Tensor &offsets, const Tensor &weights) {
    const int64_t n = position.size(0), d = rows.size(1), k = position.size(1);
    Tensor y = fresh(rows, rows.scalar_type(), {n, d});
    check(mtp_combine_rows(type_code(rows), at_(rows), n, (int)d, (int)k, places(position), held(offsets),
                           static_cast<const float *>(at_(weights)), at_(y), stream_of(rows)),
          "mtp_combine_rows");
    return y;
}

struct DispatchNode : Node {
    int64_t agents, choices, modalities;  // the plan's sizes
    SavedVariable position_, offsets_;

    std::string name() const override { return "DispatchBackward"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        position_.reset_data();
        offsets_.reset_data();
    }
    variable_list apply(variable_list &&grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        if (!grads[0].defined()) return variable_list(1);
        const Tensor position = position_.unpack(), offsets = offsets_.unpack();
        refuse_changed("dispatch", position, at::kInt, grads[0].device(), {agents, choices});
        refuse_changed("dispatch", offsets, at::kInt, grads[0].device(), {modalities + 1});
        Tensor dx;
        {
            at::NoGradGuard off;
            const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(grads[0].device());
            dx = run_combine(grads[0].resolve_neg().contiguous(), position, offsets, Tensor());
        }
        return no_further({dx}, {grads[0]}, "dispatch");
    }
};

struct CombineNode : Node {
    int64_t choices, modalities;
    SavedVariable rows_, weights_, position_, offsets_;
    bool weighted;

    std::string name() const override { return "CombineBackward"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable *v : {&rows_, &weights_, &position_, &offsets_}) v->reset_data();
    }
    // edges: rows, weights
    variable_list apply(variable_list &&grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        if (!grads[0].defined()) return variable_list(2);
        const Tensor rows = rows_.unpack(), weights = weights_.unpack(), position = position_.unpack(), offsets = offsets_.unpack();
        const auto device = grads[0].device();
        const int64_t n = grads[0].size(0), d = grads[0].size(1);
        if (weighted) {
            refuse_changed("combine", rows, grads[0].scalar_type(), device, {n * choices, d});
            refuse_changed("combine", weights, at::kFloat, device, {n, choices});
        }
        refuse_changed("combine", position, at::kInt, device, {n, choices});
        refuse_changed("combine", offsets, at::kInt, device, {modalities + 1});
        Tensor dr, dw;
        {
            at::NoGradGuard off;
            const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(grads[0].device());
            const Tensor g = grads[0].resolve_neg().contiguous();
            if (!weighted) {
                dr = run_dispatch(g, position, offsets);
            } else {
                const bool want_r = task_should_compute_output(0), want_w = task_should_compute_output(1);
                if (want_r) dr = fresh(rows, rows.scalar_type(), rows.sizes());
                if (want_w) dw = fresh(rows, at::kFloat, weights.sizes());
                check(mtp_combine_rows_grad(type_code(rows), at_(rows), at_(g), g.size(0), (int)g.size(1), (int)position.size(1),
                                            places(position), held(offsets), static_cast<const float *>(at_(weights)), at_(dr),
                                            static_cast<float *>(at_(dw)), stream_of(g)),
                      "mtp_combine_rows_grad");
            }
        }
        return no_further({dr, dw}, {rows, weights, grads[0]}, "combine");
    }
};

bool plan_for(const Tensor &t, const Tensor &position, const Tensor &offsets) {
    return position.dim() == 2 && like(position, at::kInt, t, position.sizes()) && offsets.dim() == 1 && offsets.numel() >= 1 &&
           like(offsets, at::kInt, t, offsets.sizes());
}

std::optional<Tensor> dispatch(const Tensor &x, const Tensor &position, const Tensor &offsets) {
    refuse_tracing("dispatch");
    if (!matrix(x) || row_distance(x) < 0 || !plan_for(x, position, offsets) || position.size(0) != x.size(0) || x.size(1) < 1 ||
        position.size(1) < 1)
        return std::nullopt;
    refuse_tangents("dispatch", {&x});
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
    const bool train = at::GradMode::is_enabled() && x.requires_grad();
    if (train) refuse_foreign_nodes("dispatch", {&x});
    const Tensor rows = run_dispatch(x, position, offsets);
    if (train) {
        const auto node = node_with_edges<DispatchNode>(x);
        torch::autograd::set_history(rows, node);
        node->agents = position.size(0);
        node->choices = position.size(1);
        node->modalities = offsets.numel() - 1;
        node->position_ = SavedVariable(position, false);
        node->offsets_ = SavedVariable(offsets, false);
    }
    return rows;
}

std::optional<Tensor> combine(const Tensor &rows, const Tensor &position, const Tensor &offsets, const std::optional<Tensor> &weights_) {
    refuse_tracing("combine");
    const Tensor weights = weights_.value_or(Tensor());
    if (!matrix(rows) || !rows.is_contiguous() || !plan_for(rows, position, offsets) || rows.size(0) != position.numel() ||
        rows.size(1) < 1 || position.size(1) < 1)
        return std::nullopt;
    if (weights.defined() && !like(weights, at::kFloat, rows, position.sizes())) return std::nullopt;
    refuse_tangents("combine", {&rows, &weights});
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(rows.device());
    const bool train = at::GradMode::is_enabled() && (rows.requires_grad() || (weights.defined() && weights.requires_grad()));
    if (train) refuse_foreign_nodes("combine", {&rows, &weights});
    const Tensor y = run_combine(rows, position, offsets, weights);
    if (train) {
        const auto node = node_with_edges<CombineNode>(rows, weights);
        torch::autograd::set_history(y, node);
        node->weighted = weights.defined();
        node->choices = position.size(1);
        node->modalities = offsets.numel() - 1;
        if (weights.defined()) {  // the rows themselves are needed for the weights' gradient only
            node->rows_ = SavedVariable(rows, false);
            node->weights_ = SavedVariable(weights, false);
        }
        node->position_ = SavedVariable(position, false);
        node->offsets_ = SavedVariable(offsets, false);
    }
    return y;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("linear", &linear);
    m.def("route_topk", &route_topk);
    m.def("sort_pairs", &sort_pairs);
    m.def("dispatch", &dispatch);
    m.def("combine", &combine);
}
