// binding.cpp -- the sequence operators' C entry points (include/mmn_sequence.h) as functions of torch tensors: argument checks,
// outputs and workspaces from torch's allocator, the call.  Host code only; multimodn_amd/sequence.py is its one user.
// (In Python the checks and the descriptors of a one-step pair of calls took 38 of 44 us.)
#include <torch/extension.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <dlfcn.h>
#include <unordered_set>

#include "mmn_sequence.h"

#ifndef MMN_SOURCE_HASH
#define MMN_SOURCE_HASH "unknown"
#endif

namespace py = pybind11;
using at::Tensor;
using Opt = std::optional<Tensor>;
using Shape = c10::IntArrayRef;

namespace {

// ------------------------------------------------------------------------------------------------ the library
#define ENTRIES(X)                                                                                                         \
    X(mmn_seq_embed) X(mmn_seq_embed_grad_bytes) X(mmn_seq_embed_grad) X(mmn_seq_conv) X(mmn_seq_conv_grad_bytes) X(mmn_seq_conv_grad) \
    X(mmn_seq_conv_step) X(mmn_seq_scan_marks) X(mmn_seq_scan_bytes) X(mmn_seq_scan) X(mmn_seq_scan_grad) X(mmn_seq_scan_step)
struct Lib {
#define X(name) decltype(&::name) name = nullptr;
    ENTRIES(X)
#undef X
    PyObject *error = nullptr, *stream = nullptr, *check = nullptr;      // hip.MmnError, the current stream's handle by device, hip.check
} lib;

void bind(const std::string& path, py::object error, py::object stream, py::object check) {
    void* h = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
    if (!h) throw std::runtime_error(std::string("cannot load ") + path + ": " + dlerror());
#define X(name)                                                                                     \
    lib.name = reinterpret_cast<decltype(&::name)>(dlsym(h, #name));                                \
    if (!lib.name) throw std::runtime_error(path + " does not export " #name);
    ENTRIES(X)
#undef X
    lib.error = error.release().ptr();
    lib.stream = stream.release().ptr();
    lib.check = check.release().ptr();
}

// ------------------------------------------------------------------------------------------------ arguments
constexpr int64_t LIMIT = 0x7fffffff, MOST_SIZE = (int64_t)1 << 30, MOST_STEP = (int64_t)1 << 23;

[[noreturn]] void refuse(const std::string& what) { throw py::value_error(what); }
#define NEED(ok, what) do { if (!(ok)) refuse(what); } while (0)

std::string show(Shape s) {
    std::string o = "[";
    for (size_t i = 0; i < s.size(); ++i) o += (i ? ", " : "") + std::to_string(s[i]);
    return o + "]";
}
bool is_data(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }
int type_code(at::ScalarType t) { return t == at::kFloat ? MMN_SEQ_F32 : t == at::kBFloat16 ? MMN_SEQ_BF16 : MMN_SEQ_F16; }

// A call's device: that of its first tensor, a GPU.
struct On {
    at::Device device;
    void* stream;
    c10::OptionalDeviceGuard guard;
    explicit On(const Tensor& first) : device(first.device()) {
        if (device.type() != at::kCUDA) {
            PyErr_Format(lib.error, "the sequence operators only run on an AMD GPU (torch device 'cuda' on ROCm), not on %s; there is no CPU fallback",
                         device.str().c_str());
            throw py::error_already_set();
        }
        guard.reset_device(device);
        stream = (void*)py::handle(lib.stream)(device.index()).cast<uintptr_t>();
    }
    void also(const char* name, const Tensor& t) const { NEED(t.device() == device, std::string(name) + " is on " + t.device().str() + ", not on " + device.str()); }
    void also(const char* name, const Opt& t) const { if (t) also(name, *t); }
    Tensor bytes(size_t n) const { return at::empty({(int64_t)(n > 256 ? n : 256)}, at::TensorOptions().dtype(at::kByte).device(device)); }
};
void ok(int rc, const char* what) {
    if (rc != 0) py::handle(lib.check)(rc, what);                    // (raises hip.MmnError with the library's own text)
}

// Data of the call's type.  Channels adjacent; the kernels address a stretch of a row's steps with 32-bit offsets, so steps further
// apart than 2^23 elements are brought together, and steps that share memory taken apart.
Tensor data(const char* name, const Tensor& t, at::ScalarType type, Shape shape) {
    NEED(t.scalar_type() == type, std::string(name) + " must be a " + c10::toString(type) + " tensor, as the other data of the call");
    NEED(t.sizes() == shape, std::string(name) + " must be " + show(shape) + ", not " + show(t.sizes()));
    const int64_t width = shape.back();
    if (t.stride(-1) == 1) {
        if (shape.size() < 3 || shape[1] <= 1) return t;
        if (t.stride(1) >= width && t.stride(1) <= MOST_STEP) return t;
        return t.clone(at::MemoryFormat::Contiguous);
    }
    return t.contiguous();
}
Tensor dense(const char* name, const Tensor& t, at::ScalarType type, Shape shape) { return data(name, t, type, shape).contiguous(); }
Tensor floats(const char* name, const Tensor& t, Shape shape) {
    NEED(t.scalar_type() == at::kFloat, std::string(name) + " must be a float32 tensor");
    NEED(t.sizes() == shape, std::string(name) + " must be " + show(shape) + ", not " + show(t.sizes()));
    return t.contiguous();
}
Opt floats(const char* name, const Opt& t, Shape shape) { return t ? Opt(floats(name, *t, shape)) : Opt(); }
Opt lengths_of(const Opt& t, int64_t batch) {
    if (!t) return {};
    NEED(t->scalar_type() == at::kInt || t->scalar_type() == at::kLong, "lengths must be an int32 or int64 tensor");
    NEED(t->dim() == 1 && t->size(0) == batch, "lengths must be [" + std::to_string(batch) + "], not " + show(t->sizes()));
    // (int64 values outside int32 would wrap: the kernels clamp to [0, steps])
    return t->scalar_type() == at::kInt ? t->contiguous() : t->clamp(0, LIMIT).to(at::kInt);
}
void check_x(const Tensor& x, int64_t dims) {
    NEED(is_data(x.scalar_type()), "data must be float32, bfloat16 or float16");
    NEED(x.dim() == dims && x.size(-1) >= 1, "x must have " + std::to_string(dims) + " dimensions, the last of at least one channel, not shape " + show(x.sizes()));
    for (const int64_t s : x.sizes()) NEED(s <= MOST_SIZE, "sizes above 2^30 are not supported");
}
bool wants_grad(const Tensor& t) { return t.requires_grad(); }
bool wants_grad(const Opt& t) { return t && t->requires_grad(); }
template <typename... Ts> void serving(const Ts&... ts) {
    NEED(!(at::GradMode::is_enabled() && (wants_grad(ts) || ...)),
         "the one-step forms have no gradient: call them under torch.no_grad(), or the whole sequence's operator");
}
// Where a one-step form leaves the state
Tensor state_pair(const Opt& state, const Opt& out_state) {
    NEED(state.has_value(), "state must be a tensor");
    const Tensor& out = out_state ? *out_state : *state;
    NEED(out.scalar_type() == state->scalar_type() && out.sizes() == state->sizes() && out.device() == state->device(), "out_state must be like state");
    NEED(state->is_contiguous() && out.is_contiguous(), "state and out_state must be contiguous");
    const char *a = (const char*)state->data_ptr(), *b = (const char*)out.data_ptr();
    const int64_t n = (int64_t)state->nbytes();
    NEED(a == b || a + n <= b || b + n <= a, "out_state overlaps state without being the same memory");
    return out;
}
// ... which no other operand shares: the kernels write it while other threads still read theirs
void apart(const Tensor& out, const char* name, const Tensor& t) {
    if (t.numel() == 0 || out.numel() == 0) return;
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    const char *a = (const char*)out.data_ptr(), *b = (const char*)t.data_ptr();
    NEED(a + out.nbytes() <= b || b + (last + 1) * t.element_size() <= a, std::string(name) + " shares memory with the state that the step writes");
}
void apart(const Tensor& out, const char* name, const Opt& t) { if (t) apart(out, name, *t); }
void moved(const Tensor& t) {                                        // written through its address: autograd's saved copies are stale
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
// Does a backward pass from one of these tensors meet a node, or a leaf's accumulator, that was made on another stream than the current
// one?  Autograd runs each node, and adds to each leaf, on the stream on which it was made.  A captured backward pass may not go there:
// on the default stream that ends the process.
bool made_elsewhere(const std::vector<Opt>& tensors) {
    const c10::impl::VirtualGuardImpl guard(at::kCUDA);
    std::vector<torch::autograd::Node*> todo;
    std::unordered_set<torch::autograd::Node*> seen;
    std::vector<std::shared_ptr<torch::autograd::Node>> kept;            // (an accumulator is held by the graphs that use it)
    auto take = [&](const std::shared_ptr<torch::autograd::Node>& node) {
        if (node && seen.insert(node.get()).second) { kept.push_back(node); todo.push_back(node.get()); }
    };
    for (const Opt& t : tensors)
        if (t && t->requires_grad()) take(t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t) : t->grad_fn());
    while (!todo.empty()) {
        torch::autograd::Node* const node = todo.back();
        todo.pop_back();
        const auto stream = node->stream();
        if (stream && stream->device_type() == at::kCUDA && *stream != guard.getStream(stream->device())) return true;
        for (const auto& edge : node->next_edges()) take(edge.function);
    }
    return false;
}
const void* ptr(const Opt& t) { return t ? t->data_ptr() : nullptr; }
template <typename T> T* at_of(const Opt& t) { return t ? (T*)t->data_ptr() : nullptr; }

// ------------------------------------------------------------------------------------------------ embedding
Tensor ids_of(const Tensor& ids) {
    NEED(ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong, "ids must be an int32 or int64 tensor");
    NEED(ids.numel() <= LIMIT, "more than 2^31 - 1 ids");
    return ids.contiguous();
}
std::vector<int64_t> with(Shape s, int64_t last) {
    std::vector<int64_t> o(s.begin(), s.end());
    o.push_back(last);
    return o;
}
Tensor embed(const Tensor& ids_, const Tensor& weight_, double scale) {
    const Tensor ids = ids_of(ids_);
    NEED(is_data(weight_.scalar_type()), "the table must be float32, bfloat16 or float16");
    NEED(weight_.dim() == 2 && weight_.size(0) >= 1 && weight_.size(1) >= 1 && weight_.size(0) <= MOST_SIZE && weight_.size(1) <= MOST_SIZE,
         "the table must be [vocabulary, width], not " + show(weight_.sizes()));
    const On on(weight_);
    on.also("ids", ids);
    const Tensor weight = weight_.contiguous();
    const Tensor out = at::empty(with(ids.sizes(), weight.size(1)), weight.options());
    ok(lib.mmn_seq_embed(ids.data_ptr(), ids.scalar_type() == at::kLong, weight.data_ptr(), out.data_ptr(), ids.numel(), weight.size(0), (int)weight.size(1),
                         type_code(weight.scalar_type()), (float)scale, on.stream), "mmn_seq_embed");
    return out;
}
Tensor embed_grad(const Tensor& grad_, const Tensor& ids_, int64_t vocab, double scale) {
    const Tensor ids = ids_of(ids_);
    NEED(is_data(grad_.scalar_type()), "grad must be float32, bfloat16 or float16");
    NEED(grad_.dim() == ids.dim() + 1 && grad_.sizes().slice(0, ids.dim()) == ids.sizes() && grad_.size(-1) >= 1 && grad_.size(-1) <= MOST_SIZE,
         "grad must be [*ids.shape, width], not " + show(grad_.sizes()) + " for ids " + show(ids.sizes()));
    NEED(vocab >= 1 && vocab <= MOST_SIZE, "num_embeddings must be in [1, 2^30]");
    const On on(grad_);
    on.also("ids", ids);
    const Tensor grad = grad_.contiguous();
    const int width = (int)grad.size(-1);
    const Tensor out = at::empty({vocab, width}, grad.options());
    const Tensor ws = on.bytes(lib.mmn_seq_embed_grad_bytes(ids.numel(), vocab, width));
    ok(lib.mmn_seq_embed_grad(ids.data_ptr(), ids.scalar_type() == at::kLong, grad.data_ptr(), out.data_ptr(), ids.numel(), vocab, width,
                              type_code(grad.scalar_type()), (float)scale, ws.data_ptr(), ws.nbytes(), on.stream), "mmn_seq_embed_grad");
    return out;
}

// ------------------------------------------------------------------------------------------------ convolution
struct Conv {
    mmn_seq_conv_desc c{};
    Tensor x, weight;
    Opt bias, lengths, state;
    Conv(const Tensor& x_, const Tensor& weight_, const Opt& bias_, bool silu, const Opt& lengths_, const Opt& state_, int64_t dims) {
        check_x(x_, dims);
        const int64_t batch = x_.size(0), steps = dims == 3 ? x_.size(1) : 1, width = x_.size(-1);
        NEED(weight_.dim() == 2 && weight_.size(1) >= 2 && weight_.size(1) <= 4, "weight must be [width, taps] with 2 to 4 taps");
        const int64_t taps = weight_.size(1);
        x = data("x", x_, x_.scalar_type(), x_.sizes());
        weight = floats("weight", weight_, {width, taps});
        bias = floats("bias", bias_, {width});
        lengths = lengths_of(lengths_, batch);
        if (state_) state = dense("state", *state_, x.scalar_type(), {batch, taps - 1, width});
        c.x = x.data_ptr(); c.state = ptr(state);
        c.weight = (const float*)weight.data_ptr(); c.bias = at_of<const float>(bias); c.lengths = at_of<const int32_t>(lengths);
        c.batch = batch; c.x_row = x.stride(0); c.x_step = dims == 3 ? x.stride(1) : 0;
        c.steps = (int32_t)steps; c.width = (int32_t)width; c.taps = (int32_t)taps; c.silu = silu; c.type = type_code(x.scalar_type());
    }
    void check(const On& on) const {
        on.also("weight", weight); on.also("bias", bias); on.also("lengths", lengths); on.also("state", state);
    }
};
std::pair<Tensor, Opt> conv(const Tensor& x, const Tensor& weight, const Opt& bias, bool silu, const Opt& lengths, const Opt& state, bool return_state) {
    Conv k(x, weight, bias, silu, lengths, state, 3);
    const On on(k.x);
    k.check(on);
    const Tensor y = at::empty(x.sizes(), k.x.options());
    Opt out;
    if (return_state) out = at::empty({x.size(0), k.c.taps - 1, x.size(2)}, k.x.options());
    k.c.y = y.data_ptr();
    k.c.state_out = at_of<void>(out);
    ok(lib.mmn_seq_conv(&k.c, on.stream), "mmn_seq_conv");
    return {y, out};
}
std::tuple<Tensor, Tensor, Tensor, Opt> conv_grad(const Tensor& dy_, const Tensor& x, const Tensor& weight, const Opt& bias, bool silu, const Opt& lengths,
                                                  const Opt& state, const Opt& state_grad_) {
    check_x(x, 3);
    const Tensor dy = data("dy", dy_, x.scalar_type(), x.sizes());
    Conv k(x, weight, bias, silu, lengths, state, 3);
    const int64_t batch = x.size(0), steps = x.size(1), width = x.size(2), taps = k.c.taps;
    Opt state_grad;
    if (state_grad_) state_grad = dense("state_grad", *state_grad_, x.scalar_type(), {batch, taps - 1, width});
    const On on(k.x);
    k.check(on);
    on.also("dy", dy);
    on.also("state_grad", state_grad);
    const Tensor dx = at::empty(x.sizes(), k.x.options());
    Opt dstate;
    if (state) dstate = at::empty({batch, taps - 1, width}, k.x.options());
    const Tensor params = at::empty({width * (taps + 1)}, weight.options());
    const Tensor dweight = params.narrow(0, 0, width * taps).view({width, taps}), dbias = params.narrow(0, width * taps, width);
    if (batch == 0 || steps == 0) {
        params.zero_();
        if (dstate) { if (state_grad) dstate->copy_(*state_grad); else dstate->zero_(); }
        return {dx, dweight, dbias, dstate};
    }
    k.c.dy = dy.data_ptr(); k.c.dstate_out = ptr(state_grad); k.c.dx = dx.data_ptr(); k.c.dstate = at_of<void>(dstate);
    k.c.dy_row = dy.stride(0); k.c.dy_step = dy.stride(1);
    k.c.dweight = (float*)params.data_ptr(); k.c.dbias = k.c.dweight + width * taps;
    const Tensor ws = on.bytes(lib.mmn_seq_conv_grad_bytes(&k.c));
    ok(lib.mmn_seq_conv_grad(&k.c, ws.data_ptr(), ws.nbytes(), on.stream), "mmn_seq_conv_grad");
    return {dx, dweight, dbias, dstate};
}
Tensor conv_step(const Tensor& x, const Tensor& weight, const Opt& bias, bool silu, const Opt& state, const Opt& out_state) {
    serving(x, weight, bias, state);
    const Tensor out = state_pair(state, out_state);
    Conv k(x, weight, bias, silu, {}, state, 2);
    apart(out, "x", k.x); apart(out, "weight", k.weight); apart(out, "bias", k.bias);
    const On on(k.x);
    k.check(on);
    const Tensor y = at::empty(x.sizes(), k.x.options());
    k.c.y = y.data_ptr();
    k.c.state_out = out.data_ptr();
    ok(lib.mmn_seq_conv_step(&k.c, on.stream), "mmn_seq_conv_step");
    moved(out);
    return y;
}

// ------------------------------------------------------------------------------------------------ scan
struct Scan {
    mmn_seq_scan_desc s{};
    Tensor x, dt, a, b, c;
    Opt d, z, dt_bias, lengths, state;
    static Tensor grouped(const char* name, const Tensor& t, const Tensor& x, int64_t states) {
        NEED(t.dim() == x.dim() || t.dim() == x.dim() + 1, std::string(name) + " must be [.., states] or [.., groups, states]");
        const Tensor g = t.dim() == x.dim() ? t.unsqueeze(-2) : t;
        std::vector<int64_t> shape = with(x.sizes().slice(0, x.dim() - 1), g.size(-2));
        shape.push_back(states);
        NEED(g.scalar_type() == x.scalar_type(), std::string(name) + " must be of the other data's type");
        NEED(g.sizes() == Shape(shape), std::string(name) + " must be " + show(shape) + ", not " + show(g.sizes()));
        return g.stride(-1) == 1 ? g : g.contiguous();
    }
    Scan(const Tensor& x_, const Tensor& dt_, const Tensor& a_, const Tensor& b_, const Tensor& c_, const Opt& d_, const Opt& z_, const Opt& dt_bias_, bool softplus,
         const Opt& lengths_, const Opt& state_, int64_t dims) {
        check_x(x_, dims);
        const int64_t batch = x_.size(0), steps = dims == 3 ? x_.size(1) : 1, width = x_.size(-1);
        NEED(a_.dim() == 2 && a_.size(1) >= 1 && a_.size(1) <= MMN_SEQ_MAX_STATES, "a must be [width, states] with 1 to 32 states");
        const int64_t states = a_.size(1);
        b = grouped("b", b_, x_, states);
        c = grouped("c", c_, x_, states);
        const int64_t groups = b.size(-2);
        NEED(c.size(-2) == groups && groups >= 1 && width % groups == 0, "b and c need the same number of groups, which divides the width");
        x = data("x", x_, x_.scalar_type(), x_.sizes());
        dt = data("dt", dt_, x_.scalar_type(), x_.sizes());
        if (z_) z = data("z", *z_, x_.scalar_type(), x_.sizes());
        a = floats("a", a_, {width, states});
        d = floats("d", d_, {width});
        dt_bias = floats("dt_bias", dt_bias_, {width});
        state = floats("state", state_, {batch, width, states});
        lengths = lengths_of(lengths_, batch);
        s.x = x.data_ptr(); s.dt = dt.data_ptr(); s.b = b.data_ptr(); s.c = c.data_ptr(); s.z = ptr(z);
        s.a = (const float*)a.data_ptr(); s.d = at_of<const float>(d); s.dt_bias = at_of<const float>(dt_bias);
        s.state = at_of<const float>(state); s.lengths = at_of<const int32_t>(lengths);
        s.batch = batch; s.steps = (int32_t)steps; s.width = (int32_t)width; s.groups = (int32_t)groups; s.states = (int32_t)states;
        s.softplus = softplus; s.type = type_code(x.scalar_type());
        s.x_row = x.stride(0); s.dt_row = dt.stride(0); s.b_row = b.stride(0); s.c_row = c.stride(0);
        s.b_group = b.stride(-2); s.c_group = c.stride(-2);
        if (dims == 3) { s.x_step = x.stride(1); s.dt_step = dt.stride(1); s.b_step = b.stride(1); s.c_step = c.stride(1); }
        if (z) { s.z_row = z->stride(0); s.z_step = dims == 3 ? z->stride(1) : 0; }
    }
    void check(const On& on) const {
        on.also("dt", dt); on.also("a", a); on.also("b", b); on.also("c", c); on.also("d", d); on.also("z", z); on.also("dt_bias", dt_bias);
        on.also("lengths", lengths); on.also("state", state);
    }
};
py::tuple scan(const Tensor& x, const Tensor& dt, const Tensor& a, const Tensor& b, const Tensor& c, const Opt& d, const Opt& z, const Opt& dt_bias, bool softplus,
               const Opt& lengths, const Opt& state, bool return_state, bool save) {
    Scan k(x, dt, a, b, c, d, z, dt_bias, softplus, lengths, state, 3);
    const On on(k.x);
    k.check(on);
    const Tensor y = at::empty(x.sizes(), k.x.options());
    Opt out, marks;
    if (return_state) out = at::empty({x.size(0), x.size(2), k.s.states}, k.a.options());
    if (save) marks = at::empty({(int64_t)lib.mmn_seq_scan_marks(&k.s)}, k.a.options());
    k.s.y = y.data_ptr();
    k.s.state_out = at_of<float>(out);
    k.s.marks = marks && marks->numel() ? (float*)marks->data_ptr() : nullptr;
    const Tensor ws = on.bytes(lib.mmn_seq_scan_bytes(&k.s, 0));
    ok(lib.mmn_seq_scan(&k.s, ws.data_ptr(), ws.nbytes(), on.stream), "mmn_seq_scan");
    if (!save) return py::make_tuple(y, out);
    return py::make_tuple(y, out, k.x, k.dt, k.a, k.b, k.c, k.d, k.z, k.dt_bias, k.lengths, k.state, marks);
}
py::tuple scan_grad(const Tensor& dy_, const Tensor& x, const Tensor& dt, const Tensor& a, const Tensor& b, const Tensor& c, const Opt& d, const Opt& z, const Opt& dt_bias,
                    const Opt& lengths, const Opt& state, const Tensor& marks, bool softplus, const Opt& state_grad_) {
    Scan k(x, dt, a, b, c, d, z, dt_bias, softplus, lengths, state, 3);
    const int64_t batch = x.size(0), steps = x.size(1), width = x.size(2), states = k.s.states;
    const Tensor dy = data("dy", dy_, x.scalar_type(), x.sizes());
    const Opt state_grad = floats("state_grad", state_grad_, {batch, width, states});
    NEED(marks.scalar_type() == at::kFloat && marks.is_contiguous() && (size_t)marks.numel() == lib.mmn_seq_scan_marks(&k.s), "marks are not those of these inputs");
    const On on(k.x);
    k.check(on);
    on.also("dy", dy);
    on.also("state_grad", state_grad);
    on.also("marks", marks);
    const Tensor dx = at::empty(x.sizes(), k.x.options()), ddt = at::empty(x.sizes(), k.x.options());
    const Tensor db = at::empty(k.b.sizes(), k.x.options()), dc = at::empty(k.b.sizes(), k.x.options());
    Opt dz, dstate;
    if (z) dz = at::empty(x.sizes(), k.x.options());
    if (state) dstate = at::empty({batch, width, states}, k.a.options());
    const int64_t n = width * states;
    const Tensor params = at::empty({n + 2 * width}, k.a.options());
    const Tensor da = params.narrow(0, 0, n).view({width, states}), dd = params.narrow(0, n, width), dbias = params.narrow(0, n + width, width);
    if (batch == 0 || steps == 0) {
        params.zero_();
        if (dstate) { if (state_grad) dstate->copy_(*state_grad); else dstate->zero_(); }
    } else {
        k.s.marks = (float*)marks.data_ptr(); k.s.dy = dy.data_ptr(); k.s.dstate_out = at_of<const float>(state_grad);
        k.s.dy_row = dy.stride(0); k.s.dy_step = dy.stride(1);
        k.s.dx = dx.data_ptr(); k.s.ddt = ddt.data_ptr(); k.s.db = db.data_ptr(); k.s.dc = dc.data_ptr(); k.s.dz = at_of<void>(dz);
        k.s.dparams = (float*)params.data_ptr(); k.s.dstate = at_of<float>(dstate);
        const Tensor ws = on.bytes(lib.mmn_seq_scan_bytes(&k.s, 1));
        ok(lib.mmn_seq_scan_grad(&k.s, ws.data_ptr(), ws.nbytes(), on.stream), "mmn_seq_scan_grad");
    }
    return py::make_tuple(dx, ddt, da, db, dc, dd, dz, dbias, dstate);
}
Tensor scan_step(const Tensor& x, const Tensor& dt, const Tensor& a, const Tensor& b, const Tensor& c, const Opt& d, const Opt& z, const Opt& dt_bias, bool softplus,
                 const Opt& state, const Opt& out_state) {
    serving(x, dt, a, b, c, d, z, dt_bias, state);
    const Tensor out = state_pair(state, out_state);
    Scan k(x, dt, a, b, c, d, z, dt_bias, softplus, {}, state, 2);
    apart(out, "x", k.x); apart(out, "dt", k.dt); apart(out, "a", k.a); apart(out, "b", k.b); apart(out, "c", k.c); apart(out, "d", k.d);
    apart(out, "z", k.z); apart(out, "dt_bias", k.dt_bias);
    const On on(k.x);
    k.check(on);
    const Tensor y = at::empty(x.sizes(), k.x.options());
    k.s.y = y.data_ptr();
    k.s.state_out = (float*)out.data_ptr();
    ok(lib.mmn_seq_scan_step(&k.s, on.stream), "mmn_seq_scan_step");
    moved(out);
    return y;
}

}  // namespace

PYBIND11_MODULE(_binding, m) {
    m.def("bind", &bind);
    m.def("source_hash", [] { return std::string(MMN_SOURCE_HASH); });
    m.def("made_elsewhere", &made_elsewhere);
    m.def("embed", &embed);
    m.def("embed_grad", &embed_grad);
    m.def("conv", &conv);
    m.def("conv_grad", &conv_grad);
    m.def("conv_step", &conv_step);
    m.def("scan", &scan);
    m.def("scan_grad", &scan_grad);
    m.def("scan_step", &scan_step);
}
