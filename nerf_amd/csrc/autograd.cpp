// What of the package's host side is in C++: the two operators that enter autograd's graph from here, ops.embedding and
// ops.linear_scan, and the pointer lists and step counts of the clipped optimiser step.  A backward pass written in
// Python costs a small call more than its kernels -- autograd's thread has to take the interpreter's lock and run cold
// code -- so allocation, launch and graph node are here; ops.py checks the arguments.  Host code only: every kernel is
// reached through the C ABI, whose functions ops.py's binding hands over (bind), so that both use one library.
// A training call of a lookup of 2^20 ids: 58 us (its kernels 53), with the node in Python 86; of 4096 rays x 192 x 3 55, 84.
#include <torch/extension.h>

#include <unordered_set>

#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include "../../include/nerf_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptionalTensor = std::optional<Tensor>;

#define NERF_ENTRIES(X) \
    X(nerf_last_error) X(nerf_embedding_fwd) X(nerf_embedding_bwd_workspace_bytes) X(nerf_embedding_bwd) X(nerf_linear_scan_carry_floats) \
    X(nerf_linear_scan_workspace_floats) X(nerf_linear_scan_fwd) X(nerf_linear_scan_bwd) X(nerf_grad_norm_workspace_doubles) X(nerf_grad_norm) \
    X(nerf_adam_step_scaled)

struct Entries {
#define X(name) decltype(&::name) name = nullptr;
    NERF_ENTRIES(X)
#undef X
} entry;

PyObject* error_class = PyExc_RuntimeError;   // kept to the process's end
struct EntryError : std::runtime_error {
    using std::runtime_error::runtime_error;
};
void check(int rc, const char* name) {
    if (rc != 0) throw EntryError(std::string(name) + " failed (" + std::to_string(rc) + "): " + entry.nerf_last_error());
}

int type_code(const Tensor& t) { return t.scalar_type() == at::kFloat ? NERF_F32 : t.scalar_type() == at::kBFloat16 ? NERF_BF16 : NERF_F16; }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
void* ptr(const OptionalTensor& t) { return t && t->numel() ? t->data_ptr() : nullptr; }
// Dense view or copy that starts on a 16-byte boundary.
Tensor dense(const Tensor& t) {
    Tensor c = t.contiguous();
    return (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15) == 0 ? c : c.clone();
}
OptionalTensor floats(const Tensor& like, size_t n) {
    return n ? OptionalTensor(at::empty({(int64_t)n}, like.options().dtype(at::kFloat))) : std::nullopt;
}

// A node's backward runs on the stream that was current when it was made, and a leaf's gradient is accumulated on the stream
// where the first graph over it that is still alive was made.  A captured backward pass draws such a stream into the capture
// and joins it again, but the default stream cannot be captured: that ends the process.  So everything that the operand was
// formed from is looked at, down to the leaves.
void refuse_eager_graph(const Tensor& t) {
    if (!t.requires_grad()) return;
    std::vector<std::shared_ptr<torch::autograd::Node>> next{t.is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(t) : t.grad_fn()};
    std::unordered_set<torch::autograd::Node*> seen;
    while (!next.empty()) {
        const auto node = std::move(next.back());
        next.pop_back();
        if (!node || !seen.insert(node.get()).second) continue;
        const auto stream = node->stream();
        if (stream && stream->id() == 0)   // the default one
            throw EntryError("a graph over this tensor that was made outside the capture, on the default stream, is still alive: drop or detach its outputs before capturing");
        for (const auto& edge : node->next_edges()) next.push_back(edge.function);
    }
}
bool capturing() { return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None; }

// A gradient that a kernel formed.  Where a graph of the gradients is asked for, differentiating it raises, whatever it
// depends on; otherwise this does nothing.
struct Once : torch::autograd::Function<Once> {
    static Tensor forward(AutogradContext*, const Tensor& anchor, const Tensor& formed) { return formed.detach(); }
    static variable_list backward(AutogradContext*, variable_list) {
        throw std::runtime_error("this operator of nerf_amd is differentiable once: its gradients have no gradient");
    }
};
Tensor once(const Tensor& formed) {
    if (!formed.defined() || !at::GradMode::is_enabled()) return formed;
    return Once::apply(at::empty({0}, formed.options()).set_requires_grad(true), formed);
}

// ---- embedding ----
Tensor embedding_fwd(const Tensor& table, const Tensor& ids, double scale) {
    auto shape = ids.sizes().vec();
    shape.push_back(table.size(1));
    Tensor out = at::empty(shape, table.options());
    check(entry.nerf_embedding_fwd(table.data_ptr(), type_code(table), table.size(0), (int)table.size(1), ids.data_ptr(), (int)ids.element_size(), ids.numel(),
                                   (float)scale, out.data_ptr(), stream_of(table)),
          "nerf_embedding_fwd");
    return out;
}

struct Embedding : torch::autograd::Function<Embedding> {
    static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& ids, double scale, int64_t padding) {
        ctx->save_for_backward({ids});
        ctx->saved_data["meta"] = std::vector<int64_t>{table.size(0), table.size(1), padding};
        ctx->saved_data["scale"] = scale;
        return embedding_fwd(dense(table), ids, scale);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor ids = ctx->get_saved_variables()[0];
        const auto meta = ctx->saved_data["meta"].toIntVector();
        const float scale = (float)ctx->saved_data["scale"].toDouble();
        c10::DeviceGuard guard(ids.device());
        const Tensor d_out = dense(grads[0].detach());
        const int64_t N = ids.numel(), V = meta[0], D = meta[1];
        const size_t bytes = entry.nerf_embedding_bwd_workspace_bytes(N, V, (int)D);
        OptionalTensor work;
        if (bytes) work = at::empty({(int64_t)bytes}, d_out.options().dtype(at::kByte));
        Tensor d_table = at::empty({V, D}, d_out.options());
        check(entry.nerf_embedding_bwd(d_out.data_ptr(), type_code(d_out), ids.data_ptr(), (int)ids.element_size(), N, V, (int)D, scale, meta[2], d_table.data_ptr(),
                                       ptr(work), bytes, stream_of(d_out)),
              "nerf_embedding_bwd");
        return {once(d_table), Tensor(), Tensor(), Tensor()};
    }
};

// ids dense, of 32 or 64 bits, on the table's device
Tensor embedding(const Tensor& ids, const Tensor& table, double scale, int64_t padding) {
    c10::DeviceGuard guard(table.device());
    if (at::GradMode::is_enabled() && table.requires_grad()) {
        if (capturing()) refuse_eager_graph(table);
        return Embedding::apply(table, ids, scale, padding);
    }
    return embedding_fwd(dense(table), ids, scale);
}

// ---- linear recurrence ----
struct Scanned {
    Tensor h;
    OptionalTensor last, carry;
};
// gate [B,T,G], x [B,T,C], state [B,C]: dense.  keep: with what the backward pass needs.
Scanned scan_fwd(const Tensor& gate, const Tensor& x, const OptionalTensor& state, bool reverse, bool blend, bool want_last, bool keep) {
    Scanned r;
    r.h = at::empty_like(x);
    const int64_t B = x.size(0), T = x.size(1);
    const int C = (int)x.size(2), G = (int)gate.size(2);
    if (x.numel() == 0) {   // the state passes through
        if (want_last) r.last = state ? state->detach().clone() : at::zeros({B, C}, x.options().dtype(at::kFloat));
        return r;
    }
    if (want_last) r.last = at::empty({B, C}, x.options().dtype(at::kFloat));
    if (keep) r.carry = floats(r.h, entry.nerf_linear_scan_carry_floats(B, T, C, G));
    const OptionalTensor work = floats(r.h, entry.nerf_linear_scan_workspace_floats(B, T, C, G, 0));
    check(entry.nerf_linear_scan_fwd(gate.data_ptr(), type_code(gate), x.data_ptr(), type_code(x), static_cast<const float*>(ptr(state)), B, T, C, G, reverse, blend,
                                     r.h.data_ptr(), static_cast<float*>(ptr(r.last)), static_cast<float*>(ptr(r.carry)), static_cast<float*>(ptr(work)), stream_of(x)),
          "nerf_linear_scan_fwd");
    return r;
}

struct LinearScan : torch::autograd::Function<LinearScan> {
    static variable_list forward(AutogradContext* ctx, const Tensor& gate_in, const Tensor& x_in, const OptionalTensor& state_in, bool reverse, bool blend, bool want_last) {
        const Tensor gate = dense(gate_in), x = dense(x_in);
        const OptionalTensor state = state_in ? OptionalTensor(dense(*state_in)) : std::nullopt;
        Scanned r = scan_fwd(gate, x, state, reverse, blend, want_last, true);
        ctx->save_for_backward({gate, x, state.value_or(Tensor()), r.carry.value_or(Tensor())});
        ctx->saved_data["flags"] = (int64_t)(reverse | blend << 1);
        ctx->set_materialize_grads(false);
        return want_last ? variable_list{r.h, *r.last} : variable_list{r.h};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &gate = saved[0], &x = saved[1], &state = saved[2], &carry = saved[3];
        const int64_t flags = ctx->saved_data["flags"].toInt();
        c10::DeviceGuard guard(x.device());
        const auto option = [](const Tensor& t) { return t.defined() ? OptionalTensor(t) : std::nullopt; };
        const auto like = [](const Tensor& t, bool wanted) { return wanted ? OptionalTensor(at::empty_like(t)) : std::nullopt; };
        const OptionalTensor d_h = grads[0].defined() ? OptionalTensor(dense(grads[0].detach())) : std::nullopt,
                             d_last = grads.size() > 1 && grads[1].defined() ? OptionalTensor(dense(grads[1].detach())) : std::nullopt;
        const bool needs_state = state.defined() && ctx->needs_input_grad(2);
        OptionalTensor d_gate = like(gate, ctx->needs_input_grad(0)), d_x = like(x, ctx->needs_input_grad(1)), d_state = like(state, needs_state);
        if (x.numel() == 0) {   // the state passes through; a gate may have elements where there are no channels
            if (d_gate) d_gate->zero_();
            if (d_state) d_last ? (void)d_state->copy_(*d_last) : (void)d_state->zero_();
        } else {
            const int64_t B = x.size(0), T = x.size(1);
            const int C = (int)x.size(2), G = (int)gate.size(2);
            const OptionalTensor work = floats(x.detach(), entry.nerf_linear_scan_workspace_floats(B, T, C, G, 1));
            check(entry.nerf_linear_scan_bwd(gate.data_ptr(), type_code(gate), x.data_ptr(), type_code(x), static_cast<const float*>(ptr(option(state))),
                                             static_cast<const float*>(ptr(option(carry))), ptr(d_h), static_cast<const float*>(ptr(d_last)), B, T, C, G, flags & 1,
                                             flags >> 1, ptr(d_gate), ptr(d_x), static_cast<float*>(ptr(d_state)), static_cast<float*>(ptr(work)), stream_of(x)),
                  "nerf_linear_scan_bwd");
        }
        return {once(d_gate.value_or(Tensor())), once(d_x.value_or(Tensor())), once(d_state.value_or(Tensor())), Tensor(), Tensor(), Tensor()};
    }
};

// gate [B,T,G], x [B,T,C], state [B,C] float32 on one device -> h, last (None unless want_last)
std::pair<Tensor, OptionalTensor> linear_scan(const Tensor& gate, const Tensor& x, const OptionalTensor& state, bool reverse, bool blend, bool want_last) {
    c10::DeviceGuard guard(x.device());
    if (at::GradMode::is_enabled() && (gate.requires_grad() || x.requires_grad() || (state && state->requires_grad()))) {
        if (capturing()) {
            refuse_eager_graph(gate);
            refuse_eager_graph(x);
            if (state) refuse_eager_graph(*state);
        }
        auto out = LinearScan::apply(gate, x, state, reverse, blend, want_last);
        return {out[0], want_last ? OptionalTensor(out[1]) : std::nullopt};
    }
    Scanned r = scan_fwd(dense(gate), dense(x), state ? OptionalTensor(dense(*state)) : std::nullopt, reverse, blend, want_last, false);
    return {r.h, r.last};
}

// ---- clipped Adam (FusedAdam) ----
using Tensors = std::vector<Tensor>;
template <class T>
std::vector<T*> pointers(const Tensors& list) {
    std::vector<T*> out;
    for (const Tensor& t : list) out.push_back(static_cast<T*>(t.data_ptr()));
    return out;
}
std::vector<int64_t> counts(const Tensors& list) {
    std::vector<int64_t> out;
    for (const Tensor& t : list) out.push_back(t.numel());
    return out;
}

// The norm of grads and the coefficient that it leads to -> norm[0], norm[1].  Returns the gradients as the optimiser's
// kernels take them if they are not so already.
std::optional<Tensors> grad_norm(const Tensors& params, Tensors grads, double max_norm, const Tensor& norm) {
    bool changed = false;
    for (size_t i = 0; i < params.size(); ++i) {
        const Tensor& p = params[i];
        Tensor& g = grads[i];
        if (g.layout() != at::kStrided) throw EntryError("FusedAdam does not take sparse gradients");
        if (p.scalar_type() != at::kFloat || !p.is_contiguous()) throw EntryError("FusedAdam needs contiguous float32 parameters");
        if (!p.is_cuda()) throw EntryError("nerf_amd ops run on the GPU only: got a tensor on " + p.device().str());
        if (p.device() != norm.device() || g.device() != norm.device()) throw EntryError("FusedAdam: all parameters and gradients must be on one device");
        if (g.scalar_type() == at::kFloat && g.is_contiguous()) continue;
        g = g.to(at::kFloat).contiguous();
        changed = true;
    }
    c10::DeviceGuard guard(norm.device());
    const auto n = counts(grads);
    const auto at = pointers<const float>(grads);
    const Tensor partials = at::empty({(int64_t)entry.nerf_grad_norm_workspace_doubles((int)n.size(), n.data())}, norm.options().dtype(at::kDouble));
    check(entry.nerf_grad_norm((int)n.size(), at.data(), n.data(), (float)max_norm, static_cast<double*>(partials.data_ptr()), static_cast<float*>(norm.data_ptr()),
                               stream_of(norm)),
          "nerf_grad_norm");
    return changed ? std::optional<Tensors>(std::move(grads)) : std::nullopt;
}

// Step counts as torch's Adam keeps them, a float each in host memory (a state loaded from elsewhere may hold another kind).
float* host_float(const Tensor& t) { return t.is_cpu() && t.scalar_type() == at::kFloat && t.numel() == 1 ? static_cast<float*>(t.data_ptr()) : nullptr; }
std::vector<int64_t> steps(const Tensors& list) {
    std::vector<int64_t> out;
    for (const Tensor& t : list) {
        const float* at = host_float(t);
        out.push_back((int64_t)(at ? *at : t.item<double>()));
    }
    return out;
}
void count_step(const Tensors& list) {   // in place
    for (const Tensor& t : list) {
        if (float* at = host_float(t)) *at += 1.0f;
        else t.add_(1);
    }
}

// One update with the gradients times norm[1]; `state`: of a group whose count and rate are in device memory.
void adam_step(const Tensors& params, const Tensors& grads, const Tensors& m, const Tensors& v, int64_t step, const OptionalTensor& state, double lr, double beta1,
               double beta2, double eps, double weight_decay, const Tensor& norm) {
    c10::DeviceGuard guard(norm.device());
    const auto n = counts(params);
    const auto p_at = pointers<float>(params), m_at = pointers<float>(m), v_at = pointers<float>(v);
    const auto g_at = pointers<const float>(grads);
    check(entry.nerf_adam_step_scaled((int)n.size(), p_at.data(), g_at.data(), m_at.data(), v_at.data(), n.data(), step, static_cast<float*>(ptr(state)), (float)lr,
                                      beta1, beta2, (float)eps, (float)weight_decay, static_cast<const float*>(norm.data_ptr()) + 1, stream_of(norm)),
          "nerf_adam_step_scaled");
}

// addresses: of the C ABI's functions, by name; error: what a failing entry point raises
void bind(const std::map<std::string, uintptr_t>& addresses, py::object error) {
#define X(name) entry.name = reinterpret_cast<decltype(entry.name)>(addresses.at(#name));
    NERF_ENTRIES(X)
#undef X
    error_class = error.release().ptr();
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const EntryError& e) {
            PyErr_SetString(error_class, e.what());
        }
    });
    m.def("bind", &bind);
    m.def("embedding", &embedding, py::call_guard<py::gil_scoped_release>());
    m.def("linear_scan", &linear_scan, py::call_guard<py::gil_scoped_release>());
    m.def("grad_norm", &grad_norm, py::call_guard<py::gil_scoped_release>());
    m.def("steps", &steps, py::call_guard<py::gil_scoped_release>());
    m.def("count_step", &count_step, py::call_guard<py::gil_scoped_release>());
    m.def("adam_step", &adam_step, py::call_guard<py::gil_scoped_release>());
    m.attr("entries") = std::vector<std::string>{
#define X(name) #name,
        NERF_ENTRIES(X)
#undef X
    };
}
