// Autograd binding of the fine-tuning operators (ops.py checks the arguments and calls these).
//
// The C entry points of include/clipvit.h take no torch types; this module is the torch side of them: operands'
// strides, outputs and workspaces from the caching allocator, the current stream, and the autograd nodes. It is native
// because a node written in Python runs under the interpreter on autograd's own thread: a training step of a small Linear
// took 130 us of host time that way, most of it handing the interpreter over and waking the threads.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <unordered_set>

#include "clipvit.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

namespace {

struct Api {
    decltype(&clipvit_linear) linear;
    decltype(&clipvit_linear_workspace) linear_workspace;
    decltype(&clipvit_linear_grad) linear_grad;
    decltype(&clipvit_linear_grad_workspace) linear_grad_workspace;
    decltype(&clipvit_lora_linear) lora;
    decltype(&clipvit_lora_linear_workspace) lora_workspace;
    decltype(&clipvit_lora_linear_grad) lora_grad;
    decltype(&clipvit_lora_linear_grad_workspace) lora_grad_workspace;
    decltype(&clipvit_dropout) dropout;
    decltype(&clipvit_last_error) last_error;
    int (*is_capturing)(void* stream, int* status);
} api{};
PyObject* error_class = nullptr;

struct Failure : std::runtime_error {
    int code;
    Failure(int c, const std::string& m) : std::runtime_error(m), code(c) {}
};
void check(int rc) {
    if (rc) throw Failure(rc, api.last_error());
}

int type_of(at::ScalarType t) { return t == at::kFloat ? CLIPVIT_F32 : t == at::kBFloat16 ? CLIPVIT_BF16 : CLIPVIT_F16; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void set_strides(int64_t (&to)[2], const Tensor& t) {
    for (int i = 0; i < 2; ++i) to[i] = t.defined() ? t.stride(i) : 0;
}

constexpr int64_t MAX_LD = 1 << 22;

// [..., n] as [rows, n] with unit column stride and rows that do not overlap (a copy only where the strides are
// something else); `ld`: also a row stride that the matrix products address
Tensor rows_of(const Tensor& t, bool ld) {
    Tensor r = t;
    if (t.dim() != 2) {
        int64_t rows = 1;
        for (int64_t i = 0; i + 1 < t.dim(); ++i) rows *= t.size(i);
        r = t.reshape({rows, t.size(-1)});
    }
    const bool several = r.size(0) > 1;
    if ((r.size(1) > 1 && r.stride(1) != 1) || (several && (r.stride(0) < r.size(1) || (ld && r.stride(0) >= MAX_LD)))) r = r.contiguous();
    return r;
}
// a matrix operand: one unit stride, rows (or columns) that do not overlap, the other stride below 2^22
Tensor panel_of(const Tensor& t) {
    const int64_t r = t.size(0), c = t.size(1), s0 = t.stride(0), s1 = t.stride(1);
    if ((s1 == 1 || c == 1) && (r <= 1 || (c <= s0 && s0 < MAX_LD))) return t;
    if ((s0 == 1 || r == 1) && (c <= 1 || (r <= s1 && s1 < MAX_LD))) return t;
    return t.contiguous();
}

auto current_stream(const Tensor& t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()); }

// the tensors' device as the current one, and its current stream
struct On {
    c10::DeviceGuard guard;
    void* stream;
    explicit On(const Tensor& t) : guard(t.device()) {
        stream = current_stream(t).stream();
    }
};

struct Workspace {
    Tensor t;
    void* p = nullptr;
    size_t bytes = 0;
    template <class Args>
    Workspace(int (*need)(const Args*, size_t*), const Args& a, const Tensor& like) {
        check(need(&a, &bytes));
        if (bytes) {
            t = at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
            p = t.data_ptr();
        }
    }
};

clipvit_dropout_args drop_of(double p, uint64_t seed, uint64_t offset, const Tensor& offset_dev) {
    return clipvit_dropout_args{p, seed, offset, (const int64_t*)ptr(offset_dev)};
}

// A leaf's gradient node keeps the stream of the graph that it was made for, for as long as one of its graphs lives. A
// backward pass captured on another stream would draw that stream into the capture, which ends the process, so such a
// capture is refused before anything of the call is recorded. The leaves are the operands and those behind them: the search
// goes through what was computed on the capturing stream (or on none), and stops at a graph made before, which the capture
// may treat as its input. (A capture happens once: the search costs an eager call nothing.)
void check_capture(const Tensor& first, std::initializer_list<const Tensor*> operands) {
    int status = 0;
    const auto current = current_stream(first);
    const int rc = api.is_capturing(current.stream(), &status);
    TORCH_CHECK(rc == 0, "whether a graph is capturing the current stream could not be asked (HIP error ", rc, "); a backward pass needs to know");
    if (status == 0) return;
    const c10::Stream stream = current.unwrap();
    std::vector<std::shared_ptr<Node>> todo;
    std::unordered_set<Node*> seen;
    const auto visit = [&](std::shared_ptr<Node> node) {
        if (node && seen.insert(node.get()).second) todo.push_back(std::move(node));
    };
    for (const Tensor* t : operands)
        if (t->defined() && t->requires_grad()) visit(t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t) : t->grad_fn());
    while (!todo.empty()) {
        const auto node = std::move(todo.back());
        todo.pop_back();
        const auto made = node->stream();
        const bool elsewhere = made && *made != stream;
        TORCH_CHECK(!elsewhere || node->num_outputs(),
                    "a graph capture would differentiate a leaf whose earlier autograd graph, made on another stream, is still alive: "
                    "delete that graph's outputs (or run it on the capturing stream) first");
        if (elsewhere) continue;
        for (const auto& edge : node->next_edges()) visit(edge.function);
    }
}
// The library fills the outputs outside torch's dispatcher, so a trace would record their allocation alone and replay
// uninitialised memory.
void check_eager() {
    TORCH_CHECK(!torch::jit::tracer::isTracing() && !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY) &&
                    !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::FAKE),
                "the fine-tuning operators cannot be traced (torch.jit.trace, make_fx, fake tensors): call them eagerly or capture a graph");
}
bool wants_grad(std::initializer_list<const Tensor*> ts) {
    check_eager();
    for (const Tensor* t : ts)
        TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), "the fine-tuning operators have no forward-mode derivative");
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}
std::vector<int64_t> shape_with(const Tensor& x, int64_t n) {
    auto s = x.sizes().vec();
    s.back() = n;
    return s;
}

// What the operators' autograd nodes share: the dropout of the forward (a tensor offset is saved, so that autograd notices
// when it changes before the backward pass) and the release of what is saved.
struct OpNode : Node {
    clipvit_dropout_args drop{};
    SavedVariable offset_dev;
    bool released = false;

    void begin() const {
        TORCH_CHECK(!released, torch::autograd::ERR_BACKWARD_TWICE);
        TORCH_CHECK(!at::GradMode::is_enabled(), "the fine-tuning operators are differentiable once: their backward takes no create_graph");
    }
    // the dropout arguments for a backward pass that draws the mask again; `off` keeps their tensor
    clipvit_dropout_args mask(Tensor& off, const Tensor& dy) const {
        off = offset_dev.unpack();
        TORCH_CHECK(!off.defined() || !dy.defined() || (off.device() == dy.device() && off.scalar_type() == at::kLong && off.numel() == 1),
                    "a saved tensor came back with another size, type or device than it was saved with");
        clipvit_dropout_args d = drop;
        d.offset_dev = (const int64_t*)ptr(off);
        return d;
    }
    void set_dropout(const clipvit_dropout_args& d, const Tensor& off) {
        drop = d;
        drop.offset_dev = nullptr;  // (the saved tensor's, in mask)
        offset_dev = SavedVariable(off, false);
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        released = true;
        offset_dev.reset_data();
        release_saved();
    }
    virtual void release_saved() {}
};
// A saved tensor as it was saved: a saved-tensor hook may have given back another layout, and must not another size or type.
Tensor unpacked(const SavedVariable& v, at::IntArrayRef shape, at::ScalarType type, const Tensor& like) {
    const Tensor t = v.unpack();
    TORCH_CHECK(t.defined() && t.sizes() == shape && t.scalar_type() == type && t.device() == like.device(),
                "a saved tensor came back with another size, type or device than it was saved with");
    return t;
}
int64_t rows_in(at::IntArrayRef shape) {
    int64_t m = 1;
    for (size_t i = 0; i + 1 < shape.size(); ++i) m *= shape[i];
    return m;
}
template <class N, class... Inputs>
std::shared_ptr<N> new_node(const Inputs&... inputs) {
    std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(inputs...));
    return node;
}

// ---- linear ----
struct LinearOut {
    Tensor y, slope;
};
LinearOut linear_forward(at::IntArrayRef shape, const Tensor& x2, const Tensor& w, const Tensor& bias, const Tensor& res2, int act, const clipvit_dropout_args& drop, bool save) {
    LinearOut o;
    const On on(x2);
    const int64_t m = x2.size(0), n = w.size(0);
    o.y = at::empty(shape, x2.options());
    if (save && act) o.slope = at::empty({m, n}, x2.options().dtype(at::kShort));
    clipvit_linear_args a{};
    a.dtype = type_of(x2.scalar_type());
    a.activation = act;
    a.bias_dtype = bias.defined() ? type_of(bias.scalar_type()) : a.dtype;
    a.M = m;
    a.N = n;
    a.K = x2.size(1);
    a.x = ptr(x2);
    a.x_stride[0] = x2.stride(0);
    a.x_stride[1] = x2.stride(1);
    a.w = ptr(w);
    a.w_stride[0] = w.stride(0);
    a.w_stride[1] = w.stride(1);
    a.bias = ptr(bias);
    a.residual = ptr(res2);
    a.residual_stride = res2.defined() ? res2.stride(0) : 0;
    a.y = ptr(o.y);
    a.y_stride = n;
    a.slope = (int16_t*)ptr(o.slope);
    a.dropout = drop;
    const Workspace ws(api.linear_workspace, a, x2);
    check(api.linear(on.stream, &a, ws.p, ws.bytes));
    return o;
}

struct LinearNode : OpNode {
    SavedVariable x, w, slope;  // x where the weight's gradient reads it, w where x's does
    bool has_slope = false;
    std::vector<int64_t> x_shape;
    at::ScalarType bias_type = at::ScalarType::Undefined;  // (none)

    std::string name() const override { return "LinearBackward"; }
    void release_saved() override {
        x.reset_data();
        w.reset_data();
        slope.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        begin();
        const Tensor& dy = grads[0];
        if (!dy.defined()) return variable_list(4);
        const int64_t m = rows_in(x_shape), k = x_shape.back(), n = dy.size(-1);
        const at::ScalarType type = dy.scalar_type();
        const bool nx = task_should_compute_output(0), nw = task_should_compute_output(1);
        const bool nb = bias_type != at::ScalarType::Undefined && task_should_compute_output(2), nr = task_should_compute_output(3);
        const Tensor x2 = nw ? panel_of(unpacked(x, {m, k}, type, dy)) : Tensor(), w2 = nx ? panel_of(unpacked(w, {n, k}, type, dy)) : Tensor();
        const Tensor slope2 = has_slope && (nx || nw || nb) ? unpacked(slope, {m, n}, at::kShort, dy).contiguous() : Tensor();
        Tensor dx, dw, db;
        if (nx || nw || nb) {
            const On on(dy);
            const Tensor dy2 = rows_of(dy, true);
            if (nx) dx = at::empty(x_shape, dy.options());
            if (nw) dw = at::empty({n, k}, dy.options());
            if (nb) db = at::empty({n}, dy.options().dtype(bias_type));
            clipvit_linear_grad_args a{};
            a.dtype = type_of(type);
            a.bias_dtype = nb ? type_of(bias_type) : a.dtype;
            a.M = m;
            a.N = n;
            a.K = k;
            a.dy = ptr(dy2);
            a.dy_stride = dy2.stride(0);
            a.x = ptr(x2);
            set_strides(a.x_stride, x2);
            a.w = ptr(w2);
            set_strides(a.w_stride, w2);
            a.slope = (const int16_t*)ptr(slope2);
            a.dx = ptr(dx);
            a.dw = ptr(dw);
            a.db = ptr(db);
            Tensor offset_keep;
            a.dropout = mask(offset_keep, dy);
            const Workspace ws(api.linear_grad_workspace, a, dy);
            check(api.linear_grad(on.stream, &a, ws.p, ws.bytes));
        }
        return {dx, dw, db, nr ? dy : Tensor()};
    }
};

Tensor opt(const std::optional<Tensor>& t) { return t ? *t : Tensor(); }

Tensor linear(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias_, const std::optional<Tensor>& residual_, int64_t act, double p,
              uint64_t seed, uint64_t offset, const std::optional<Tensor>& offset_dev) {
    Tensor bias = opt(bias_);
    const Tensor residual = opt(residual_), off = opt(offset_dev);
    if (bias.defined() && bias.stride(0) != 1) bias = bias.contiguous();
    const bool grad = wants_grad({&x, &weight, &bias, &residual});
    if (grad) check_capture(x, {&x, &weight, bias_ ? &*bias_ : &bias, &residual});
    Tensor x2, w, res2;
    {
        const at::NoGradGuard no_grad;
        x2 = panel_of(rows_of(x, false));
        w = panel_of(weight);
        if (residual.defined()) res2 = rows_of(residual, false);
    }
    const bool product = grad && (x.requires_grad() || weight.requires_grad() || (bias.defined() && bias.requires_grad()));  // (not the residual alone)
    const auto drop = drop_of(p, seed, offset, off);
    const LinearOut o = linear_forward(shape_with(x, w.size(0)), x2, w, bias, res2, (int)act, drop, product);
    if (grad) {
        const auto node = new_node<LinearNode>(x, weight, bias, residual);
        node->set_dropout(drop, product ? off : Tensor());
        if (weight.requires_grad()) node->x = SavedVariable(x2, false);
        if (x.requires_grad()) node->w = SavedVariable(w, false);
        node->slope = SavedVariable(o.slope, false);
        node->has_slope = o.slope.defined();
        node->x_shape = x.sizes().vec();
        if (bias.defined()) node->bias_type = bias.scalar_type();
        torch::autograd::set_history(o.y, node);
    }
    return o.y;
}

// ---- dropout ----
Tensor dropout_call(const Tensor& x, const Tensor& residual, const clipvit_dropout_args& drop) {
    const at::NoGradGuard no_grad;
    const On on(x);
    const Tensor x2 = rows_of(x, false), res2 = residual.defined() ? rows_of(residual, false) : Tensor();
    const Tensor y = at::empty(x.sizes(), x.options());
    check(api.dropout(on.stream, type_of(x.scalar_type()), ptr(x2), x2.stride(0), ptr(res2), res2.defined() ? res2.stride(0) : 0, ptr(y), x2.size(1),
                      x2.size(0), x2.size(1), &drop));
    return y;
}

struct DropoutNode : OpNode {
    std::string name() const override { return "DropoutBackward"; }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        begin();
        const Tensor& dy = grads[0];
        if (!dy.defined()) return variable_list(2);
        Tensor offset_keep, dx;
        if (task_should_compute_output(0)) dx = dropout_call(dy, Tensor(), mask(offset_keep, dy));
        return {dx, task_should_compute_output(1) ? dy : Tensor()};
    }
};

Tensor dropout(const Tensor& x, const std::optional<Tensor>& residual_, double p, uint64_t seed, uint64_t offset, const std::optional<Tensor>& offset_dev) {
    const Tensor residual = opt(residual_), off = opt(offset_dev);
    const bool grad = wants_grad({&x, &residual});
    if (grad) check_capture(x, {&x, &residual});
    const auto drop = drop_of(p, seed, offset, off);
    const Tensor y = dropout_call(x, residual, drop);
    if (grad) {
        const auto node = new_node<DropoutNode>(x, residual);
        node->set_dropout(drop, x.requires_grad() ? off : Tensor());
        torch::autograd::set_history(y, node);
    }
    return y;
}

// ---- LoRA linear ----
struct LoraOut {
    Tensor y, u;
};
LoraOut lora_forward(at::IntArrayRef shape, const Tensor& x2, const Tensor& w, const Tensor& A, const Tensor& B, const Tensor& bias, double scaling,
                     const clipvit_dropout_args& drop) {
    LoraOut o;
    const On on(x2);
    const int64_t m = x2.size(0), n = w.size(0), r = A.size(1);
    o.y = at::empty(shape, x2.options());
    o.u = at::empty({m, (r + 31) / 32 * 32}, x2.options());
    clipvit_lora_args a{};
    a.dtype = type_of(x2.scalar_type());
    a.bias_dtype = bias.defined() ? type_of(bias.scalar_type()) : a.dtype;
    a.M = m;
    a.N = n;
    a.K = x2.size(1);
    a.rank = r;
    a.x = ptr(x2);
    a.x_stride = x2.stride(0);
    a.w = ptr(w);
    a.w_stride[0] = w.stride(0);
    a.w_stride[1] = w.stride(1);
    a.a = ptr(A);
    a.a_stride[0] = A.stride(0);
    a.a_stride[1] = A.stride(1);
    a.b = ptr(B);
    a.b_stride[0] = B.stride(0);
    a.b_stride[1] = B.stride(1);
    a.bias = ptr(bias);
    a.y = ptr(o.y);
    a.u = ptr(o.u);
    a.scaling = (float)scaling;
    a.dropout = drop;
    const Workspace ws(api.lora_workspace, a, x2);
    check(api.lora(on.stream, &a, ws.p, ws.bytes));
    return o;
}

struct LoraNode : OpNode {
    SavedVariable x, w, a_factor, b_factor, u;  // each where a wanted gradient reads it
    std::vector<int64_t> x_shape;
    int64_t rank = 0;
    at::ScalarType bias_type = at::ScalarType::Undefined;  // (none)
    float scaling = 1;

    std::string name() const override { return "LoraLinearBackward"; }
    void release_saved() override {
        for (SavedVariable* v : {&x, &w, &a_factor, &b_factor, &u}) v->reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        begin();
        const Tensor& dy = grads[0];
        if (!dy.defined()) return variable_list(5);
        const int64_t m = rows_in(x_shape), k = x_shape.back(), n = dy.size(-1), r = rank;
        const at::ScalarType type = dy.scalar_type();
        const bool nx = task_should_compute_output(0), nw = task_should_compute_output(1), nA = task_should_compute_output(2);
        const bool nB = task_should_compute_output(3), nb = bias_type != at::ScalarType::Undefined && task_should_compute_output(4);
        const Tensor x2 = nw || nA ? rows_of(unpacked(x, {m, k}, type, dy), true) : Tensor(), w2 = nx ? panel_of(unpacked(w, {n, k}, type, dy)) : Tensor();
        const Tensor A = nx ? unpacked(a_factor, {k, r}, type, dy) : Tensor(), B = nx || nA ? unpacked(b_factor, {r, n}, type, dy) : Tensor();
        const Tensor u2 = nB ? unpacked(u, {m, (r + 31) / 32 * 32}, type, dy).contiguous() : Tensor();
        const On on(dy);
        const Tensor dy2 = rows_of(dy, true);
        Tensor dx, dw, dA, dB, db;
        if (nx) dx = at::empty(x_shape, dy.options());
        if (nw) dw = at::empty({n, k}, dy.options());
        if (nA) dA = at::empty({k, r}, dy.options());
        if (nB) dB = at::empty({r, n}, dy.options());
        if (nb) db = at::empty({n}, dy.options().dtype(bias_type));
        clipvit_lora_grad_args a{};
        a.dtype = type_of(type);
        a.bias_dtype = nb ? type_of(bias_type) : a.dtype;
        a.M = m;
        a.N = n;
        a.K = k;
        a.rank = r;
        a.dy = ptr(dy2);
        a.dy_stride = dy2.stride(0);
        a.x = ptr(x2);
        a.x_stride = x2.defined() ? x2.stride(0) : 0;
        a.w = ptr(w2);
        set_strides(a.w_stride, w2);
        a.a = ptr(A);
        set_strides(a.a_stride, A);
        a.b = ptr(B);
        set_strides(a.b_stride, B);
        a.u = ptr(u2);
        a.dx = ptr(dx);
        a.dw = ptr(dw);
        a.da = ptr(dA);
        a.db_factor = ptr(dB);
        a.dbias = ptr(db);
        a.scaling = scaling;
        Tensor offset_keep;
        a.dropout = drop;
        if (nx || nA) a.dropout = mask(offset_keep, dy);  // (du's scale is 1 / (1 - p) all the same)
        const Workspace ws(api.lora_grad_workspace, a, dy);
        check(api.lora_grad(on.stream, &a, ws.p, ws.bytes));
        return {dx, dw, dA, dB, db};
    }
};

Tensor lora_linear(const Tensor& x, const Tensor& weight, const Tensor& A, const Tensor& B, const std::optional<Tensor>& bias_, double scaling, double p,
                   uint64_t seed, uint64_t offset, const std::optional<Tensor>& offset_dev) {
    Tensor bias = opt(bias_);
    const Tensor off = opt(offset_dev);
    if (bias.defined() && bias.stride(0) != 1) bias = bias.contiguous();
    const bool grad = wants_grad({&x, &weight, &A, &B, &bias});
    if (grad) check_capture(x, {&x, &weight, &A, &B, bias_ ? &*bias_ : &bias});
    Tensor x2, w;
    {
        const at::NoGradGuard no_grad;
        x2 = rows_of(x, true);
        w = panel_of(weight);
    }
    const auto drop = drop_of(p, seed, offset, off);
    const LoraOut o = lora_forward(shape_with(x, w.size(0)), x2, w, A, B, bias, scaling, drop);
    if (grad) {
        const auto node = new_node<LoraNode>(x, weight, A, B, bias);
        const bool gx = x.requires_grad(), gA = A.requires_grad();
        node->set_dropout(drop, gx || gA ? off : Tensor());  // (dB's mask is in u)
        if (weight.requires_grad() || gA) node->x = SavedVariable(x2, false);
        if (gx) node->w = SavedVariable(w, false);
        if (gx) node->a_factor = SavedVariable(A, false);
        if (gx || gA) node->b_factor = SavedVariable(B, false);
        if (B.requires_grad()) node->u = SavedVariable(o.u, false);
        node->x_shape = x.sizes().vec();
        if (bias.defined()) node->bias_type = bias.scalar_type();
        node->rank = A.size(1);
        node->scaling = (float)scaling;
        torch::autograd::set_history(o.y, node);
    }
    return o.y;
}

// the library's entry points by address (whichever build of it the package loaded), the query of the HIP runtime that it is
// linked to, and the package's error class
void set_library(const std::map<std::string, uint64_t>& f, py::object error) {
    auto get = [&](auto& p, const char* name) {
        const auto at = f.find(name);
        if (at == f.end() || !at->second) throw std::runtime_error(std::string("the library has no ") + name);
        p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(at->second);
    };
    get(api.linear, "clipvit_linear");
    get(api.linear_workspace, "clipvit_linear_workspace");
    get(api.linear_grad, "clipvit_linear_grad");
    get(api.linear_grad_workspace, "clipvit_linear_grad_workspace");
    get(api.lora, "clipvit_lora_linear");
    get(api.lora_workspace, "clipvit_lora_linear_workspace");
    get(api.lora_grad, "clipvit_lora_linear_grad");
    get(api.lora_grad_workspace, "clipvit_lora_linear_grad_workspace");
    get(api.dropout, "clipvit_dropout");
    get(api.last_error, "clipvit_last_error");
    get(api.is_capturing, "hipStreamIsCapturing");
    error_class = error.release().ptr();
}

}  // namespace

PYBIND11_MODULE(_ops_torch, m) {
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Failure& e) {
            PyErr_SetObject(error_class, py::make_tuple(e.code, e.what()).ptr());
        }
    });
    const auto no_gil = py::call_guard<py::gil_scoped_release>();
    m.def("set_library", &set_library);
    m.def("linear", &linear, no_gil);
    m.def("dropout", &dropout, no_gil);
    m.def("lora_linear", &lora_linear, no_gil);
}
