// Autograd nodes of the codebook operators (ops.embedding, loss.linear_cross_entropy, loss.linear_distillation) in C++: what
// their small calls cost is the host's time, and a node in Python cost as much in the backward thread as all the launches of
// the pass (lookup of 256 x 48 with its gradient: 71 us a call that way, here 46, of which 7 on the GPU).  The entry points of
// librisesdf_hip.so come in as addresses (bind), so that this module works with whichever build of the library is loaded.
// Host code only: no kernels here.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <atomic>
#include <unordered_set>

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Error : std::runtime_error { using std::runtime_error::runtime_error; };

struct Entries {
    const char *(*last_error)();
    int (*embedding_fwd)(const int64_t *, int64_t, const void *, int64_t, int, int, float, int64_t, void *, int32_t *, void *);
    int64_t (*embedding_bwd_workspace_bytes)(int64_t, int64_t, int);
    int (*embedding_bwd)(const int64_t *, int64_t, const void *, int64_t, int, int, float, int64_t, void *, void *, int64_t, void *);
    int64_t (*class_head_workspace_bytes)(int64_t, int64_t, int, int, int);
    int (*class_head_fwd)(const void *, const void *, int64_t, int64_t, int, int, const int64_t *, const float *, int, int64_t, float, int,
                          float *, float *, float *, float *, float *, int32_t *, void *, int64_t, void *);
    int (*class_head_bwd)(const void *, const void *, int64_t, int64_t, int, int, const int64_t *, const float *, const float *, int, float,
                          const float *, const float *, const float *, int, void *, void *, void *, int64_t, void *);
} E = {};

void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

void check(int rc, const char *what)
{
    if (rc == 0) return;
    const char *msg = E.last_error();
    throw Error(std::string(what) + " failed (code " + std::to_string(rc) + "): " + (msg != nullptr ? msg : ""));
}

// Timers and the debug log of the Python layer (_lib._watch): called before each entry point with its name and scalar arguments; what it
// returns is called behind it.
std::atomic<bool> watched{false};
py::object *watcher = nullptr;             // (only touched with the interpreter's lock; kept for the life of the process)

template <class F, class... A> void entry(const char *name, F call, A... scalars)
{
    if (!watched.load(std::memory_order_relaxed)) {
        check(call(), name);
        return;
    }
    py::gil_scoped_acquire lock;
    const py::object done = watched.load() ? (*watcher)(name, py::make_tuple(scalars...)) : py::none();
    int rc;
    {
        py::gil_scoped_release free;
        rc = call();
    }
    if (!done.is_none()) done();
    check(rc, name);
}

int dtype_id(const Tensor &t)
{
    return t.scalar_type() == at::kFloat ? 0 : (t.scalar_type() == at::kBFloat16 ? 1 : 2);       // (the caller checked)
}

Tensor bytes_on(int64_t n, const Tensor &like)
{
    return at::empty({n}, like.options().dtype(at::kByte).requires_grad(false));
}

template <class T> T *address(const Tensor &t) { return t.defined() ? (T *)t.data_ptr() : nullptr; }

// whether a stream of this device is being captured
bool captured(const c10::Stream &s)
{
    if (s.id() == c10::hip::getDefaultHIPStream(s.device_index()).id()) return false;
    const c10::DeviceGuard guard(c10::Device(c10::DeviceType::CUDA, s.device_index()));
    const auto now = c10::hip::getCurrentHIPStream(s.device_index());
    c10::hip::setCurrentHIPStream(c10::hip::HIPStream(
        c10::hip::HIPStream::UNCHECKED, c10::Stream(c10::Stream::UNSAFE, c10::Device(c10::DeviceType::HIP, s.device_index()), s.id())));
    const bool yes = c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None;
    c10::hip::setCurrentHIPStream(now);
    return yes;
}

// A leaf remembers the stream on which a graph that is still alive first used it, and its gradient is accumulated there.  Inside a
// capture that would tie an eager stream to the captured one, which ends the process, so the call is refused while it can be.  All
// leaves behind the operand count: it may be a view, a cast or a layer's output.
void check_leaves(const Tensor &t, const char *what)
{
    if (!at::GradMode::is_enabled() || !t.requires_grad()) return;
    const c10::DeviceGuard guard(t.device());
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    const auto node = t.is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(t) : t.grad_fn();
    std::vector<torch::autograd::Node *> todo{node.get()};
    std::unordered_set<torch::autograd::Node *> seen;
    while (!todo.empty()) {
        auto *n = todo.back();
        todo.pop_back();
        if (n == nullptr || !seen.insert(n).second) continue;
        for (const auto &e : n->next_edges()) todo.push_back(e.function.get());
        if (dynamic_cast<torch::autograd::AccumulateGrad *>(n) == nullptr) continue;
        const auto there = n->stream();
        // (by id: one of the two calls the device HIP, the other CUDA)
        if (there.has_value() && there->id() != c10::hip::getCurrentHIPStream(there->device_index()).id() && !captured(*there))
            throw Error(std::string(what) + ": a leaf of this captured pass is part of a graph that was recorded on another stream and is "
                        "still alive; drop that graph (its outputs and losses) before the capture");
    }
}

// gradients of a node that cannot be differentiated again: under create_graph a second derivative raises instead of being zero
variable_list once(variable_list grads, const char *what)
{
    if (!at::GradMode::is_enabled()) return grads;
    variable_list there;
    for (auto &g : grads)
        if (g.defined()) there.push_back(g.detach().requires_grad_(true));
    if (there.empty()) return grads;
    auto error = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " cannot be differentiated twice", (int)there.size());
    auto out = (*error)(std::move(there));
    size_t i = 0;
    for (auto &g : grads)
        if (g.defined()) g = out[i++];
    return grads;
}

struct Embedding : torch::autograd::Function<Embedding> {
    static Tensor forward(AutogradContext *ctx, const Tensor &ids, const Tensor &table_, double scale, int64_t padding, int64_t bad_ids)
    {
        const Tensor table = table_.contiguous();
        const c10::DeviceGuard guard(table.device());
        const int64_t v = table.size(0), d = table.size(1);
        auto shape = ids.sizes().vec();
        shape.push_back(d);
        Tensor out = at::empty(shape, table.options().requires_grad(false));
        entry("embedding_fwd", [&] {
            return E.embedding_fwd(address<const int64_t>(ids), ids.numel(), address<const void>(table), v, (int)d, dtype_id(table), (float)scale,
                                   padding, address<void>(out), (int32_t *)bad_ids, stream_of(table));
        }, ids.numel(), v, d, dtype_id(table));
        ctx->save_for_backward({ids});
        ctx->saved_data["v"] = v;
        ctx->saved_data["d"] = d;
        ctx->saved_data["type"] = (int64_t)table.scalar_type();
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["padding"] = padding;
        return out;
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        const Tensor ids = ctx->get_saved_variables()[0];
        const int64_t v = ctx->saved_data["v"].toInt(), d = ctx->saved_data["d"].toInt(), n = ids.numel();
        const c10::DeviceGuard guard(ids.device());
        const Tensor g = grads[0].detach().to((at::ScalarType)ctx->saved_data["type"].toInt()).contiguous();
        Tensor dt = at::empty({v, d}, g.options());
        const int64_t bytes = E.embedding_bwd_workspace_bytes(n, v, (int)d);
        const Tensor ws = bytes > 0 ? bytes_on(bytes, g) : Tensor();
        entry("embedding_bwd", [&] {
            return E.embedding_bwd(address<const int64_t>(ids), n, address<const void>(g), v, (int)d, dtype_id(g),
                                   (float)ctx->saved_data["scale"].toDouble(), ctx->saved_data["padding"].toInt(), address<void>(dt),
                                   address<void>(ws), bytes, stream_of(g));
        }, n, v, d, dtype_id(g));
        return once({Tensor(), dt, Tensor(), Tensor(), Tensor()}, "embedding");
    }
};

// contiguous and 16-byte aligned (a view into the middle of a storage may be neither)
Tensor aligned(const Tensor &t)
{
    const Tensor c = t.detach().contiguous();
    return ((uintptr_t)c.data_ptr() & 15) == 0 ? c : c.clone();
}

// both losses: no logits = labels (k = 1), else a teacher's listed classes
struct ClassHead : torch::autograd::Function<ClassHead> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x_, const Tensor &w_, const Tensor &ids, const c10::optional<Tensor> &logits,
                          int64_t k, int64_t ignore, double temperature, int64_t reduction, int64_t bad_ids)
    {
        const Tensor x = aligned(x_), w = aligned(w_);
        const c10::DeviceGuard guard(x.device());
        const int64_t n = x.size(0), d = x.size(1), v = w.size(0);
        const bool teacher = logits.has_value();
        const int64_t bytes = E.class_head_workspace_bytes(n, v, (int)d, dtype_id(x), 0);
        if (bytes < 0) check(1, "class_head_workspace_bytes");
        const Tensor ws = bytes_on(bytes, x);
        const auto f32 = x.options().dtype(at::kFloat).requires_grad(false);
        // lse [2, n], count [1], and for a teacher q, listed logits [n, k]: one allocation, kept for the backward
        const Tensor keep = at::empty({2 * n + 1 + (teacher ? 2 * n * k : 0)}, f32);
        Tensor loss = reduction == 0 ? at::empty({n}, f32) : at::empty({}, f32);
        float *a = address<float>(keep), *q = teacher ? a + 2 * n + 1 : nullptr;
        entry("class_head_fwd", [&] {
            return E.class_head_fwd(address<const void>(x), address<const void>(w), n, v, (int)d, dtype_id(x), address<const int64_t>(ids),
                                    teacher ? address<const float>(*logits) : nullptr, (int)k, ignore, (float)temperature, (int)reduction,
                                    address<float>(loss), a, a + 2 * n, q, teacher ? q + n * k : nullptr, (int32_t *)bad_ids,
                                    address<void>(ws), bytes, stream_of(x));
        }, n, v, d, dtype_id(x), k);
        ctx->save_for_backward({x, w, ids, keep});
        ctx->saved_data["k"] = k;
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["reduction"] = reduction;
        ctx->saved_data["teacher"] = teacher;
        return loss;
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &ids = saved[2], &keep = saved[3];
        const int64_t n = x.size(0), d = x.size(1), v = w.size(0), k = ctx->saved_data["k"].toInt();
        const int64_t reduction = ctx->saved_data["reduction"].toInt();
        const bool teacher = ctx->saved_data["teacher"].toBool();
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
        variable_list out(9);
        if (!need_x && !need_w) return out;
        const c10::DeviceGuard guard(x.device());
        const Tensor g = grads[0].detach().to(at::kFloat).contiguous();
        if (need_x) out[0] = at::empty_like(x);
        if (need_w) out[1] = at::empty_like(w);
        const int64_t bytes = E.class_head_workspace_bytes(n, v, (int)d, dtype_id(x), (need_x ? 1 : 0) + (need_w ? 2 : 0));
        const Tensor ws = bytes_on(bytes, x);
        float *a = address<float>(keep), *q = teacher ? a + 2 * n + 1 : nullptr;
        entry("class_head_bwd", [&] {
            return E.class_head_bwd(address<const void>(x), address<const void>(w), n, v, (int)d, dtype_id(x), address<const int64_t>(ids), q,
                                    teacher ? q + n * k : nullptr, (int)k, (float)ctx->saved_data["temperature"].toDouble(), a,
                                    reduction == 1 ? a + 2 * n : nullptr, address<const float>(g), reduction == 0, address<void>(out[0]),
                                    address<void>(out[1]), address<void>(ws), bytes, stream_of(x));
        }, n, v, d, dtype_id(x), k);
        return once(std::move(out), "the losses of a linear head");
    }
};

void bind(const std::vector<uintptr_t> &a, py::object error)
{
    TORCH_CHECK(a.size() == 7, "seven entry points");
    static py::object *type = nullptr;       // (kept for the life of the process)
    if (type != nullptr) return;
    type = new py::object(error);
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Error &e) {
            PyErr_SetString(type->ptr(), e.what());
        }
    });
    E.last_error = (decltype(E.last_error))a[0];
    E.embedding_fwd = (decltype(E.embedding_fwd))a[1];
    E.embedding_bwd_workspace_bytes = (decltype(E.embedding_bwd_workspace_bytes))a[2];
    E.embedding_bwd = (decltype(E.embedding_bwd))a[3];
    E.class_head_workspace_bytes = (decltype(E.class_head_workspace_bytes))a[4];
    E.class_head_fwd = (decltype(E.class_head_fwd))a[5];
    E.class_head_bwd = (decltype(E.class_head_bwd))a[6];
}

}  // namespace

PYBIND11_MODULE(_codebook, m)
{
    m.def("bind", &bind);
    m.def("watch", [](py::object call) {
        watched = false;
        if (watcher == nullptr) watcher = new py::object();
        *watcher = call;
        watched = !call.is_none();
    });
    m.def("embedding", [](const Tensor &ids, const Tensor &table, double scale, int64_t padding, int64_t bad_ids) {
        py::gil_scoped_release free;
        check_leaves(table, "embedding");
        return Embedding::apply(ids, table, scale, padding, bad_ids);
    });
    m.def("class_head", [](const Tensor &x, const Tensor &w, const Tensor &ids, const c10::optional<Tensor> &logits, int64_t k, int64_t ignore,
                           double temperature, int64_t reduction, int64_t bad_ids) {
        py::gil_scoped_release free;
        check_leaves(x, "the losses of a linear head");
        check_leaves(w, "the losses of a linear head");
        return ClassHead::apply(x, w, ids, logits, k, ignore, temperature, reduction, bad_ids);
    });
}
