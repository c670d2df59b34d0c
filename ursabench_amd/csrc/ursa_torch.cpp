// ursa_torch.cpp — K15 / K16 (include/ursa_hip.h) as autograd nodes, and K17's two calls. The backward pass of a node runs on autograd's device thread:
// written in Python it has to wait there for the interpreter, which costs more than the launches of a small layer (mnist's first
// layer, forward + backward: 138 us with Python nodes, 46 with these). What may be called and with what is checked by the Python callers
// (fused_linear, fused_norm); this file allocates, launches on the current stream of the tensors' device and keeps what the
// backward pass needs.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/ursa_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

int32_t type_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return URSA_F32;
        case at::kBFloat16: return URSA_BF16;
        case at::kHalf: return URSA_F16;
        default: TORCH_CHECK_TYPE(false, "float32, bfloat16 or float16 wanted, got ", t.scalar_type());
    }
}

void ok(int rc, const char* what) {
    if (rc < 0) TORCH_CHECK_VALUE(false, what, ": ", ursa_strerror(rc), " (ursa error ", rc, ")");
    TORCH_CHECK(rc == 0, what, ": HIP error ", rc, ": ", ursa_strerror(rc));
}

ursa_stream_t stream_of(const Tensor& t) { return (ursa_stream_t)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void* at_(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor bytes(const Tensor& like, int64_t n) { return n ? at::empty({n}, like.options().dtype(at::kByte)) : Tensor(); }

Tensor given(const Maybe& t) { return t.has_value() && t->defined() ? *t : Tensor(); }

Tensor packed(const Tensor& t) { return t.defined() ? t.contiguous() : t; }

// What a backward pass finds of a tensor that its forward kept: a saved_tensors_hooks pair may hand back another one. The same values
// in other places (strides, a copy) are laid out again; anything that the launch would misread raises.
Tensor kept(const Tensor& t, at::IntArrayRef sizes, at::ScalarType type, const Tensor& dy) {
    if (!t.defined()) return t;
    TORCH_CHECK(t.layout() == at::kStrided && t.device() == dy.device() && t.scalar_type() == type && t.sizes() == sizes,
                "ursabench_amd: a saved tensor came back as ", t.scalar_type(), " ", t.sizes(), " on ", t.device(), ", saved was ", type, " ", sizes, " on ", dy.device());
    return t.contiguous();
}

bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }

// Whether a tensor is its memory and no more: not the wrapper of a function transform or of a dispatching subclass, nor a dual tensor,
// whose tangent a launch would drop.
bool memory(const Tensor& t) {
    return !t.defined() || (t.has_storage() && !t.key_set().has(c10::DispatchKey::Python) && !t._fw_grad(0).defined());
}

// Whether a launch on the operands' memory is all that a call is to torch: not inside a function transform (vmap, grad, jvp), under a
// dispatch mode (fake tensors, tracing to a graph, counters) or torch.jit.trace, all of which see operators only.
bool plain(std::initializer_list<const Tensor*> operands) {
    if (c10::impl::tls_local_dispatch_key_set().included_.has(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) ||
        c10::impl::TorchDispatchModeTLS::any_modes_set() || torch::jit::tracer::isTracing()) return false;
    for (const Tensor* t : operands)
        if (!memory(*t)) return false;
    return true;
}

void only_memory(const variable_list& grads) {
    for (const auto& g : grads)
        TORCH_CHECK(memory(g), "ursabench_amd: batched (is_grads_batched) and dual gradients are not offered in the backward pass; "
                               "fused_linear.enabled(False) / fused_norm.enabled(False) before the forward pass select the stock ops");
}

// x as rows of `width`
Tensor rows_of(const Tensor& x, int64_t width) { return (x.dim() == 2 && x.size(1) == width ? x : x.reshape({width ? x.numel() / width : 0, width})).contiguous(); }

struct Packed8 { Tensor q, e; };

// room for the 8-bit form of x2
Packed8 room8(const Tensor& x2) {
    const int64_t blocks = (x2.size(1) + 31) / 32;
    Packed8 p{at::empty({x2.size(0), 32 * blocks}, x2.options().dtype(at::kChar)), at::empty({x2.size(0), blocks}, x2.options().dtype(at::kChar))};
    return p;
}

// What a gradient of a once differentiable node is a function of when a graph is recorded: whoever differentiates it any further comes
// through here.
struct DoubleBackward : torch::autograd::Node {
    variable_list apply(variable_list&&) override { TORCH_CHECK(false, "ursabench_amd: double backward is not offered"); }
};

// Gradients of a node that is differentiable once. Under create_graph each depends on all the node's
// inputs and on the incoming gradients, whether or not one of those is tracked: a gradient of a sum has a constant coming in, and
// depends on the weights all the same. The edges to them are what makes a second differentiation with respect to one of them arrive.
variable_list once(variable_list grads, const variable_list& incoming, bool create_graph) {
    if (!create_graph) return grads;
    torch::autograd::edge_list edges;
    if (const auto self = torch::autograd::get_current_node())
        for (const auto& e : self->next_edges())
            if (e.is_valid()) edges.push_back(e);
    for (const auto& g : incoming)
        if (wants(g)) edges.push_back(torch::autograd::impl::gradient_edge(g));
    const auto refusal = std::make_shared<DoubleBackward>();
    refusal->set_next_edges(std::move(edges));
    for (auto& g : grads)
        if (g.defined()) {
            g = g.detach();
            torch::autograd::create_gradient_edge(g, refusal);
        }
    return grads;
}

// y (, z) = act(x w' + b) + r for 2-d contiguous operands
Tensor linear_forward(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& r, int64_t act, at::IntArrayRef shape, Tensor* z) {
    const c10::DeviceGuard guard(x.device());
    const int64_t M = x.size(0), N = w.size(0), K = w.size(1);
    const int32_t dt = type_of(x);
    Tensor y = at::empty(shape, x.options());
    if (z) *z = at::empty({M, N}, x.options());
    const Tensor ws = bytes(x, ursa_linear_ws_bytes(M, N, K, dt));
    ok(ursa_linear_act(at_(x), at_(w), at_(b), at_(r), at_(y), z ? at_(*z) : nullptr, at_(ws), M, N, K, dt, (int32_t)act, stream_of(x)), "ursa_linear_act");
    return y;
}

// Which of a node's gradients this backward pass wants. `given`: bit i is set where operand i was a tensor; autograd numbers those.
struct Wanted {
    const AutogradContext* ctx;
    int64_t given;
    bool operator()(int i) const { return given >> i & 1 && ctx->needs_input_grad(__builtin_popcountll(given & ((1ll << i) - 1))); }
};

struct LinearAct : torch::autograd::Function<LinearAct> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Maybe& b_, const Maybe& r_, int64_t act, bool save8) {
        const Tensor b = given(b_), r = given(r_);
        const bool nx = wants(x), nw = wants(w), nb = wants(b);
        at::NoGradGuard no_grad;
        const int64_t N = w.size(0), K = w.size(1);
        const Tensor x2 = rows_of(x, K), wc = w.contiguous();
        std::vector<int64_t> shape = x.sizes().vec();
        shape.back() = N;
        Tensor z;
        const Tensor y = linear_forward(x2, wc, packed(b), r.defined() ? rows_of(r, N) : r, act, shape, act && (nx || nw || nb) ? &z : nullptr);
        Packed8 p;
        if (nw && save8) {
            p = room8(x2);
            const c10::DeviceGuard guard(x.device());
            ok(ursa_act8_pack(at_(x2), (int8_t*)at_(p.q), (int8_t*)at_(p.e), x2.size(0), K, type_of(x2), stream_of(x2)), "ursa_act8_pack");
        }
        ctx->save_for_backward({nw && !save8 ? x2 : Tensor(), nx ? wc : Tensor(), z, p.q, p.e});
        ctx->saved_data["act"] = act;
        ctx->saved_data["given"] = (int64_t)(3 + 4 * b.defined() + 8 * r.defined());
        ctx->saved_data["x"] = x.sizes().vec();
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        only_memory(grads);
        const bool create_graph = at::GradMode::is_enabled();
        at::NoGradGuard no_grad;
        const int64_t act = ctx->saved_data["act"].toInt();
        const Wanted wanted{ctx, ctx->saved_data["given"].toInt()};
        const bool nx = wanted(0), nw = wanted(1), nb = wanted(2);
        const auto saved = ctx->get_saved_variables();
        const Tensor& dy_ = grads[0];
        variable_list out(6);
        if (nx || nw || nb) {
            const std::vector<int64_t> shape = ctx->saved_data["x"].toIntVector();
            const int64_t K = shape.back(), N = dy_.size(-1);
            const Tensor dy = rows_of(dy_, N);
            const int64_t M = dy.size(0);
            const c10::DeviceGuard guard(dy.device());
            const int32_t dt = type_of(dy);
            const at::ScalarType t = dy.scalar_type();
            const int64_t blocks = (K + 31) / 32;
            Tensor x, w, q, e;
            const Tensor z = kept(saved[2], {M, N}, t, dy);
            if (nx) w = kept(saved[1], {N, K}, t, dy);
            if (nw) x = kept(saved[0], {M, K}, t, dy), q = kept(saved[3], {M, 32 * blocks}, at::kChar, dy), e = kept(saved[4], {M, blocks}, at::kChar, dy);
            if (nx) out[0] = at::empty(shape, dy.options());
            if (nw) out[1] = at::empty({N, K}, dy.options());
            if (nb) out[2] = at::empty({N}, dy.options());
            const Tensor ws = bytes(dy, ursa_linear_bwd_ws_bytes(M, N, K, dt, (int32_t)act, nx, nw, nb));
            ok(ursa_linear_bwd(at_(dy), at_(x), (const int8_t*)at_(q), (const int8_t*)at_(e), at_(w), at_(z), at_(out[0]), at_(out[1]), at_(out[2]), at_(ws), M,
                               N, K, dt, (int32_t)act, stream_of(dy)), "ursa_linear_bwd");
        }
        if (wanted(3)) out[3] = dy_;
        return once(std::move(out), grads, create_graph);
    }
};

// None where the call is the stock ops' (plain)
Maybe linear_act(const Tensor& x, const Tensor& w, const Maybe& b_, const Maybe& r_, int64_t act, bool save8) {
    const Tensor b = given(b_), r = given(r_);
    if (!plain({&x, &w, &b, &r})) return {};
    if (at::GradMode::is_enabled() && (wants(x) || wants(w) || wants(b) || wants(r))) return LinearAct::apply(x, w, b_, r_, act, save8);
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = w.size(0);
    return linear_forward(rows_of(x, w.size(1)), w.contiguous(), packed(b), r.defined() ? rows_of(r, w.size(0)) : r, act, shape, nullptr);
}

struct NormOut { Tensor z, y, stats, q, e; };

// of 2-d contiguous x (and addend); z and y in `shape`
NormOut norm_forward(const Tensor& x, const Tensor& r, const Tensor& w, const Tensor& b, double eps, at::IntArrayRef shape, bool stats, bool save8) {
    const c10::DeviceGuard guard(x.device());
    const int64_t M = x.size(0), D = x.size(1);
    NormOut o;
    if (r.defined()) o.z = at::empty(shape, x.options());
    o.y = at::empty(shape, x.options());
    if (stats) o.stats = at::empty({2, M}, x.options().dtype(at::kFloat));
    Packed8 p;
    if (save8) p = room8(x);
    float* m = (float*)at_(o.stats);
    ok(ursa_layer_norm_fwd(at_(x), at_(r), at_(o.z), at_(o.y), at_(w), at_(b), m, m ? m + M : nullptr, (int8_t*)at_(p.q), (int8_t*)at_(p.e), M, D, (float)eps,
                           type_of(x), w.defined() ? type_of(w) : b.defined() ? type_of(b) : type_of(x), stream_of(x)), "ursa_layer_norm_fwd");
    o.q = p.q, o.e = p.e;
    return o;
}

// z: what was normalised, in any shape (of an output: that tensor itself, so that changes in place are noticed)
void norm_keep(AutogradContext* ctx, const Tensor& z, const NormOut& o, const Tensor& w, const Tensor& b, const Tensor& x, int64_t width, int64_t given, bool save8) {
    ctx->save_for_backward({save8 ? Tensor() : z, o.q, o.e, o.stats, w});
    ctx->saved_data["given"] = given;
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["kept"] = z.sizes().vec();
    ctx->saved_data["width"] = width;
    ctx->saved_data["type"] = (int64_t)(w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : z.scalar_type());
}

// dx in the input's shape, dgamma and dbeta [D]
std::array<Tensor, 3> norm_backward(AutogradContext* ctx, const Tensor& dy_, const Tensor& dz_, bool nx, bool nw, bool nb) {
    const auto saved = ctx->get_saved_variables();
    const int64_t D = ctx->saved_data["width"].toInt();
    const auto ptype = (at::ScalarType)ctx->saved_data["type"].toInt();
    const Tensor dy = rows_of(dy_, D), dz = dz_.defined() ? rows_of(dz_, D) : dz_;
    const int64_t M = dy.size(0);
    const int64_t blocks = (D + 31) / 32;
    const Tensor x = kept(saved[0], ctx->saved_data["kept"].toIntVector(), dy.scalar_type(), dy), q = kept(saved[1], {M, 32 * blocks}, at::kChar, dy),
                 e = kept(saved[2], {M, blocks}, at::kChar, dy), stats = kept(saved[3], {2, M}, at::kFloat, dy), w = kept(saved[4], {D}, ptype, dy);
    const c10::DeviceGuard guard(dy.device());
    std::array<Tensor, 3> out;
    if (nx) out[0] = at::empty(ctx->saved_data["shape"].toIntVector(), dy.options());
    if (nw) out[1] = at::empty({D}, dy.options().dtype(ptype));
    if (nb) out[2] = at::empty({D}, dy.options().dtype(ptype));
    const Tensor ws = nw || nb ? bytes(dy, 4 * ursa_layer_norm_ws_floats(M, D)) : Tensor();
    const float* m = (const float*)at_(stats);
    ok(ursa_layer_norm_bwd(at_(x), (const int8_t*)at_(q), (const int8_t*)at_(e), at_(dy), at_(dz), at_(w), m, m + M, at_(out[0]),
                           at_(out[1]), at_(out[2]), (float*)at_(ws), M, D, type_of(dy), ptype == at::kFloat ? URSA_F32 : ptype == at::kHalf ? URSA_F16 : URSA_BF16,
                           stream_of(dy)), "ursa_layer_norm_bwd");
    return out;
}

// w, b: [D] contiguous
struct Norm : torch::autograd::Function<Norm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& w_, const Maybe& b_, int64_t width, double eps, bool save8) {
        const Tensor w = given(w_), b = given(b_);
        at::NoGradGuard no_grad;
        const Tensor x2 = rows_of(x, width);
        const NormOut o = norm_forward(x2, Tensor(), w, b, eps, x.sizes(), true, save8);
        norm_keep(ctx, x2, o, w, b, x, width, 1 + 2 * w.defined() + 4 * b.defined(), save8);
        return o.y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        only_memory(grads);
        const bool create_graph = at::GradMode::is_enabled();
        at::NoGradGuard no_grad;
        const Wanted wanted{ctx, ctx->saved_data["given"].toInt()};
        const auto g = norm_backward(ctx, grads[0], Tensor(), wanted(0), wanted(1), wanted(2));
        return once({g[0], g[1], g[2], Tensor(), Tensor(), Tensor()}, grads, create_graph);
    }
};

struct AddNorm : torch::autograd::Function<AddNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& a, const Tensor& r, const Maybe& w_, const Maybe& b_, int64_t width, double eps, bool save8) {
        const Tensor w = given(w_), b = given(b_);
        const bool constant = !wants(a) && !wants(r);
        at::NoGradGuard no_grad;
        ctx->set_materialize_grads(false);                     // an unused output's gradient arrives undefined, not as zeros
        const NormOut o = norm_forward(rows_of(a, width), rows_of(r, width), w, b, eps, a.sizes(), true, save8);
        norm_keep(ctx, o.z, o, w, b, a, width, 3 + 4 * w.defined() + 8 * b.defined(), save8);
        if (constant) ctx->mark_non_differentiable({o.z});     // as the stock sum: only y depends on what needs a gradient
        return {o.z, o.y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        only_memory(grads);
        const bool create_graph = at::GradMode::is_enabled();
        at::NoGradGuard no_grad;
        const Wanted wanted{ctx, ctx->saved_data["given"].toInt()};
        const bool na = wanted(0), nr = wanted(1);
        variable_list out(7);
        const Tensor &dz = grads[0], &dy = grads[1];
        if (!dy.defined()) {                                   // y unused: only the sum's own gradient flows
            if (na) out[0] = dz;
            if (nr) out[1] = dz;
            return once(std::move(out), grads, create_graph);
        }
        const auto g = norm_backward(ctx, dy, dz, na || nr, wanted(2), wanted(3));
        if (na) out[0] = g[0];
        if (nr) out[1] = g[0];
        out[2] = g[1], out[3] = g[2];
        return once(std::move(out), grads, create_graph);
    }
};

bool recorded(const Tensor& x, const Tensor& r, const Tensor& w, const Tensor& b) {
    return at::GradMode::is_enabled() && (wants(x) || wants(r) || wants(w) || wants(b));
}

// None where the call is the stock ops' (plain)
Maybe layer_norm(const Tensor& x, const Maybe& w_, const Maybe& b_, int64_t width, double eps, bool save8) {
    const Tensor w = given(w_), b = given(b_);
    if (!plain({&x, &w, &b})) return {};
    if (recorded(x, Tensor(), w, b)) return Norm::apply(x, w_, b_, width, eps, save8);
    return norm_forward(rows_of(x, width), Tensor(), w, b, eps, x.sizes(), false, false).y;
}

std::optional<std::pair<Tensor, Tensor>> add_layer_norm(const Tensor& a, const Tensor& r, const Maybe& w_, const Maybe& b_, int64_t width, double eps, bool save8) {
    const Tensor w = given(w_), b = given(b_);
    if (!plain({&a, &r, &w, &b})) return {};
    if (recorded(a, r, w, b)) {
        auto out = AddNorm::apply(a, r, w_, b_, width, eps, save8);
        return std::make_pair(out[0], out[1]);
    }
    const NormOut o = norm_forward(rows_of(a, width), rows_of(r, width), w, b, eps, a.sizes(), false, false);
    return std::make_pair(o.z, o.y);
}

void only_plain(std::initializer_list<const Tensor*> operands, const char* what) {
    TORCH_CHECK_VALUE(plain(operands), what, ": a plain tensor wanted, outside of function transforms, dispatch modes and tracing");
}

std::pair<Tensor, Tensor> act8_pack(const Tensor& x) {
    only_plain({&x}, "act8.pack");
    at::NoGradGuard no_grad;
    const int64_t D = x.size(-1);
    const Tensor x2 = rows_of(x, D);
    const c10::DeviceGuard guard(x.device());
    const Packed8 p = room8(x2);
    ok(ursa_act8_pack(at_(x2), (int8_t*)at_(p.q), (int8_t*)at_(p.e), x2.size(0), D, type_of(x2), stream_of(x2)), "ursa_act8_pack");
    return {p.q, p.e};
}

// q, e: contiguous, of `shape`'s rows and features
Tensor act8_unpack(const Tensor& q, const Tensor& e, const std::vector<int64_t>& shape, const Tensor& like) {
    only_plain({&q, &e}, "act8.unpack");
    const c10::DeviceGuard guard(q.device());
    Tensor x = at::empty(shape, like.options().device(q.device()));
    ok(ursa_act8_unpack((const int8_t*)at_(q), (const int8_t*)at_(e), at_(x), q.size(0), shape.back(), type_of(x), stream_of(q)), "ursa_act8_unpack");
    return x;
}

}  // namespace

PYBIND11_MODULE(_ursa_torch, m) {
    namespace py = pybind11;
    m.attr("abi_version") = URSA_ABI_VERSION;
    m.def("act8_pack", &act8_pack, py::call_guard<py::gil_scoped_release>());
    m.def("act8_unpack", &act8_unpack, py::call_guard<py::gil_scoped_release>());
    m.def("linear_act", &linear_act, py::call_guard<py::gil_scoped_release>());
    m.def("layer_norm", &layer_norm, py::call_guard<py::gil_scoped_release>());
    m.def("add_layer_norm", &add_layer_norm, py::call_guard<py::gil_scoped_release>());
}
