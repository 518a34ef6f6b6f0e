// PyTorch binding of the entry points whose calls are short: argument checks, allocation, stream and autograd node in
// C++ instead of Python.  A call of a few microseconds on the device took 20 to 60 microseconds through ctypes and
// torch.autograd.Function, a training step of one 200; everything else of the C ABI stays on ctypes (_lib.py).
// It holds no kernel and no arithmetic: each function fills in a call of include/loractl_b200.h.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>

#include <algorithm>
#include <vector>

#include "../../include/loractl_b200.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
namespace py = pybind11;

struct LqFailure : std::runtime_error {
    int status;
    explicit LqFailure(int s) : std::runtime_error(lq_last_error()), status(s) {}
};
inline void check(int status) {
    if (status != LQ_OK) throw LqFailure(status);
}

inline int dtype_code(const Tensor& t) {
    if (t.scalar_type() == at::kBFloat16) return LQ_BF16;
    TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat, "unsupported activation dtype ", t.scalar_type(),
                     ": the b200 backend computes in f32 or bf16");
    return LQ_F32;
}
inline void require_cuda(const Tensor& t, const char* what) {
    TORCH_CHECK(t.is_cuda(), what, " must live on a CUDA device: the b200 backend has no CPU path");
}
inline void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
inline const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
inline void* mut(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
inline Tensor defined(const std::optional<Tensor>& t) { return t ? *t : Tensor(); }

// The last axis contiguous (any other strides), a copy otherwise.
inline Tensor rows_of(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }

// Contiguous and on 16 bytes, a copy if it is not.
inline Tensor whole(const Tensor& t) {
    const Tensor c = t.contiguous();
    return (uintptr_t)ptr(c) % 16 ? c.clone() : c;
}

// A saved tensor as unpacking gave it back.  Under saved-tensor hooks (checkpointing, offloading) that is another tensor than the
// forward's, of any strides and at any address; so it is after a swap of `.data`.
Tensor restored(const Tensor& t, at::IntArrayRef sizes, at::ScalarType type, at::Device device, const char* name) {
    if (!t.defined()) return t;
    TORCH_CHECK(t.sizes() == sizes && t.scalar_type() == type && t.device() == device, "the saved ", name, " came back as ", t.sizes(), " ",
                t.scalar_type(), " on ", t.device(), ", it was ", sizes, " ", type, " on ", device);
    return rows_of(t);
}

inline bool wants_grad(std::initializer_list<const Tensor*> inputs) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : inputs)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}
// A forward-mode tangent that the node would drop is refused, as torch.autograd.Function does without a jvp.
void no_tangents(std::initializer_list<const Tensor*> inputs, const char* name) {
    for (const Tensor* t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), name, " has no forward-mode derivative");
}
// Gradients that are themselves to be differentiated (create_graph) fail when that is tried, as torch's
// once_differentiable does.
variable_list once(variable_list&& grads, const char* name) {
    if (!at::GradMode::is_enabled()) return std::move(grads);
    variable_list marked;
    for (const Tensor& g : grads) marked.push_back(g.defined() ? g.detach().requires_grad_(true) : g);
    auto error = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " is differentiable once only", (int64_t)grads.size());
    return (*error)(std::move(marked));
}

// ---- residual norm ----------------------------------------------------------------------------------

// A modulation vector as a [b, h] view in `type`.
Tensor vector_of(const Tensor& v, int64_t b, int64_t h, at::ScalarType type, const char* name) {
    TORCH_CHECK_VALUE(v.dim() >= 1 && v.size(-1) == h && v.size(0) == b && v.numel() == b * h, name, " must be [b = ", b, ", h = ", h,
                      "] or [b, 1, h], got ", v.sizes());
    Tensor t = v.scalar_type() == type ? v : v.to(type);
    if (t.dim() != 2) t = t.reshape({b, h});
    return t.stride(1) == 1 || h == 1 ? t : t.contiguous();
}
Tensor weight_of(const Tensor& w, int64_t h, const char* name) {
    if (!w.defined()) return w;
    TORCH_CHECK_VALUE(w.numel() == h, name, " must hold ", h, " values, got ", w.sizes());
    Tensor t = w.scalar_type() == at::kFloat ? w : w.to(at::kFloat);
    if (t.dim() != 1) t = t.reshape({h});
    return t.is_contiguous() ? t : t.contiguous();
}

struct Like {
    bool there = false;
    std::vector<int64_t> shape;
    at::ScalarType type = at::kFloat;
    void of(const Tensor& t) {
        there = t.defined();
        if (there) shape = t.sizes().vec(), type = t.scalar_type();
    }
    Tensor back(const Tensor& g) const { return g.scalar_type() == type ? g : g.to(type); }
};

// What a call reads, with contiguous rows: x, y [b, t, h], vectors [b, h], weights f32 [h]; y, gate and weights may be undefined.
struct ResidualNormInputs {
    Tensor x, y, gate, shift, scale, weight, post_weight;
    void put(lq_residual_norm_args& a) const {
        a.x = ptr(x), a.x_sample = x.stride(0), a.x_token = x.stride(1);
        if (y.defined()) a.y = ptr(y), a.y_sample = y.stride(0), a.y_token = y.stride(1), a.gate = ptr(gate), a.gate_sample = gate.stride(0);
        a.shift = ptr(shift), a.shift_sample = shift.stride(0), a.scale = ptr(scale), a.scale_sample = scale.stride(0);
        a.weight = (const float*)ptr(weight), a.post_weight = (const float*)ptr(post_weight);
    }
};

struct ResidualNormBackward : public Node {
    lq_residual_norm_args args;  // of the inputs, only which there are: their addresses are those of what unpacking gives
    SavedVariable x, y, gate, shift, scale, weight, post_weight;  // r and z are not read by the backward
    Tensor stats;
    Like like[5];  // gate, shift, scale, weight, post_weight
    bool two = false, released = false;

    std::string name() const override { return "ResidualNormBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable* v : {&x, &y, &gate, &shift, &scale, &weight, &post_weight}) v->reset_data();
        stats.reset();
        released = true;
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        TORCH_CHECK(!released, "Trying to backward through the graph a second time: specify retain_graph=True");
        return once(gradients(std::move(grads)), "gated_residual_norm");
    }
    variable_list gradients(variable_list&& grads) {
        variable_list out(7);
        Tensor dr = two ? grads[0] : Tensor(), dz = grads[two ? 1 : 0];
        if (!dr.defined() && !dz.defined()) return out;
        no_tangents({&dr, &dz}, "the residual norm's backward");
        // unpacking checks that none was changed in place; the tensors keep their memory through the launch
        const Tensor tensors[7] = {x.unpack(), y.unpack(), gate.unpack(), shift.unpack(), scale.unpack(), weight.unpack(), post_weight.unpack()};
        at::NoGradGuard no_grad;
        const auto device = stats.device();
        c10::cuda::OptionalCUDAGuard guard(device);
        const int64_t b = args.samples, h = args.h;
        const auto type = args.dtype == LQ_F32 ? at::kFloat : at::kBFloat16, mod = args.mod_f32 ? at::kFloat : at::kBFloat16;
        const int64_t rows[] = {b, args.tokens, h}, vectors[] = {b, h}, columns[] = {h};
        const ResidualNormInputs in = {restored(tensors[0], rows, type, device, "x"), restored(tensors[1], rows, type, device, "y"),
                                       restored(tensors[2], vectors, mod, device, "gate"), restored(tensors[3], vectors, mod, device, "shift"),
                                       restored(tensors[4], vectors, mod, device, "scale"), restored(tensors[5], columns, at::kFloat, device, "weight"),
                                       restored(tensors[6], columns, at::kFloat, device, "post_weight")};
        const Tensor& xs = in.x;
        const auto opts = xs.options().requires_grad(false);
        lq_residual_norm_args args = this->args;
        in.put(args);
        lq_residual_norm_grads g = {};
        auto token = [&](int i) {
            if (!task_should_compute_output(i)) return Tensor();
            return at::empty({b, args.tokens, h}, opts);
        };
        out[0] = token(0);
        if (args.y) out[2] = token(2);
        const int places[5] = {1, 3, 4, 5, 6};
        bool sums = false;
        for (int i = 0; i < 5; ++i) {
            if (!like[i].there || !task_should_compute_output(places[i])) continue;
            sums = true;
            out[places[i]] = at::empty(like[i].shape, opts.dtype(i >= 3 || args.mod_f32 ? at::kFloat : at::kBFloat16));  // b * h or h values
        }
        if (dr.defined()) {
            dr = rows_of(dr);
            g.dr = ptr(dr), g.dr_sample = dr.stride(0), g.dr_token = dr.stride(1);
        }
        if (dz.defined()) {
            dz = rows_of(dz);
            g.dz = ptr(dz), g.dz_sample = dz.stride(0), g.dz_token = dz.stride(1);
        }
        g.dx = mut(out[0]), g.dy = mut(out[2]), g.dgate = mut(out[1]), g.dshift = mut(out[3]), g.dscale = mut(out[4]);
        g.dweight = (float*)mut(out[5]), g.dpost_weight = (float*)mut(out[6]);
        Tensor ws;  // of this call alone: from the pool of the current stream, or of the graph being captured
        if (sums) ws = at::empty({(int64_t)lq_residual_norm_workspace_bytes(b, args.tokens, h)}, opts.dtype(at::kByte));
        check(lq_residual_norm_bwd(&args, &g, mut(ws), sums ? ws.numel() : 0, stream_of(xs)));
        for (int i = 0; i < 5; ++i)
            if (out[places[i]].defined()) out[places[i]] = like[i].back(out[places[i]]);
        return out;
    }
};

// r (undefined without y) and z.
std::vector<Tensor> residual_norm(const Tensor& x_, const std::optional<Tensor>& gate_, const std::optional<Tensor>& y_, const Tensor& shift_,
                                  const Tensor& scale_, const std::optional<Tensor>& weight_, const std::optional<Tensor>& post_weight_,
                                  bool layer, double alpha, double eps) {
    const Tensor gate0 = defined(gate_), y0 = defined(y_), weight0 = defined(weight_), post0 = defined(post_weight_);
    no_tangents({&x_, &gate0, &y0, &shift_, &scale_, &weight0, &post0}, "the residual norm");
    require_cuda(x_, "x");
    TORCH_CHECK_VALUE(x_.dim() == 3, "expected [b, tokens, h], got ", x_.sizes());
    const int64_t b = x_.size(0), t = x_.size(1), h = x_.size(2);
    lq_residual_norm_args a = {};
    a.dtype = dtype_code(x_);
    if (y0.defined())
        TORCH_CHECK_VALUE(y0.sizes() == x_.sizes() && y0.scalar_type() == x_.scalar_type(), "x and y must agree in shape and dtype, got ",
                          x_.sizes(), " ", x_.scalar_type(), " / ", y0.sizes(), " ", y0.scalar_type());
    const std::pair<const char*, const Tensor*> named[] = {{"gate", &gate0}, {"y", &y0}, {"shift", &shift_}, {"scale", &scale_},
                                                           {"weight", &weight0}, {"post_weight", &post0}};
    for (const auto& [name, v] : named)
        TORCH_CHECK(!v->defined() || v->device() == x_.device(), name, " is on ", v->device(), ", x on ", x_.device());
    // one type for the modulation vectors: theirs when they agree on f32 or bf16, else f32
    at::ScalarType type = shift_.scalar_type();
    for (const Tensor* v : {&gate0, &shift_, &scale_}) {
        if (!v->defined()) continue;
        TORCH_CHECK_TYPE(v->scalar_type() == at::kFloat || v->scalar_type() == at::kBFloat16, "unsupported dtype ", v->scalar_type(),
                         " of gate, shift or scale: f32 or bf16");
        if (v->scalar_type() != type) type = at::kFloat;
    }
    TORCH_CHECK_VALUE(y0.defined() == gate0.defined(), "gate and y go together");
    const bool grad = wants_grad({&x_, &gate0, &y0, &shift_, &scale_, &weight0, &post0});
    ResidualNormInputs in;
    Tensor r, z, stats;
    c10::cuda::OptionalCUDAGuard guard(x_.device());
    {
        at::NoGradGuard no_grad;
        in.x = rows_of(x_), in.shift = vector_of(shift_, b, h, type, "shift"), in.scale = vector_of(scale_, b, h, type, "scale");
        in.weight = weight_of(weight0, h, "weight"), in.post_weight = weight_of(post0, h, "post_weight");
        const auto opts = x_.options().requires_grad(false);
        z = at::empty({b, t, h}, opts);
        if (y0.defined()) {
            in.y = rows_of(y0), in.gate = vector_of(gate0, b, h, type, "gate"), r = at::empty({b, t, h}, opts);
            a.r = mut(r);
        }
        if (grad) {
            stats = at::empty({3, b * t}, opts.dtype(at::kFloat));
            a.mean = stats.data_ptr<float>(), a.rstd = a.mean + b * t, a.post_rstd = a.rstd + b * t;
        }
        in.put(a);
        a.z = mut(z);
        a.samples = b, a.tokens = t, a.h = h, a.mod_f32 = type == at::kFloat, a.layer = layer, a.alpha = (float)alpha, a.eps = (float)eps;
        check(lq_residual_norm_fwd(&a, stream_of(x_)));
    }
    if (grad) {
        auto node = std::shared_ptr<ResidualNormBackward>(new ResidualNormBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x_, gate0, y0, shift_, scale_, weight0, post0));
        node->args = a;
        node->x = SavedVariable(in.x, false), node->y = SavedVariable(in.y, false), node->gate = SavedVariable(in.gate, false);
        node->shift = SavedVariable(in.shift, false), node->scale = SavedVariable(in.scale, false);
        node->weight = SavedVariable(in.weight, false), node->post_weight = SavedVariable(in.post_weight, false);
        node->stats = stats;
        node->two = r.defined();
        const Tensor* vectors[5] = {&gate0, &shift_, &scale_, &weight0, &post0};
        for (int i = 0; i < 5; ++i) node->like[i].of(*vectors[i]);
        if (r.defined()) torch::autograd::set_history(r, node);
        torch::autograd::set_history(z, node);
    }
    return r.defined() ? std::vector<Tensor>{r, z} : std::vector<Tensor>{z};
}

// ---- gradient norm ----------------------------------------------------------------------------------

// A list or tuple of tensors, read without pybind's casters (60 ns an element, a third of a call on hundreds of tensors).
std::vector<Tensor> tensors_of(const py::object& list, const char* what) {
    const py::object items = py::reinterpret_steal<py::object>(PySequence_Fast(list.ptr(), "a sequence of tensors is needed"));
    if (!items) throw py::error_already_set();
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(items.ptr());
    std::vector<Tensor> v;
    v.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject* o = PySequence_Fast_GET_ITEM(items.ptr(), i);
        TORCH_CHECK_TYPE(THPVariable_Check(o), what, " must be tensors, got ", Py_TYPE(o)->tp_name, " at place ", i);
        v.push_back(THPVariable_Unpack(o));
    }
    return v;
}

// Leaves that require grad are refused where they would be scaled, as torch's in-place operators do: they are most likely parameters
// in place of their gradients.
inline void no_parameter(const Tensor& t) {
    TORCH_CHECK(!t.requires_grad() || !t.is_leaf(), "a leaf that requires grad would be scaled in place: clip_grad_norm takes gradients, not parameters");
}

struct Gradients {
    std::vector<const void*> at;
    std::vector<int64_t> counts;
    std::vector<int32_t> types;
    explicit Gradients(const std::vector<Tensor>& grads, bool scaled = false) {
        TORCH_CHECK_VALUE(!grads.empty(), "no gradient tensors");
        at.reserve(grads.size()), counts.reserve(grads.size()), types.reserve(grads.size());
        for (const Tensor& t : grads) {
            TORCH_CHECK(t.device() == grads[0].device(), "gradients must live on one CUDA device, got ", grads[0].device(), " and ", t.device());
            const auto type = t.scalar_type();
            TORCH_CHECK_TYPE(type == at::kFloat || type == at::kBFloat16, "unsupported gradient dtype ", type, ": f32 or bf16");
            at.push_back(t.const_data_ptr());
            counts.push_back(t.numel());
            types.push_back(type == at::kFloat ? LQ_F32 : LQ_BF16);
            if (scaled) no_parameter(t);
        }
        require_cuda(grads[0], "gradients");
    }
};

void grad_norm_call(const Gradients& g, const std::vector<const void*>& at, const std::vector<const void*>* outs, double grad_scale,
                    double max_norm, const Tensor& norm, const Tensor& coef, const Tensor& flag) {
    const int n = (int)at.size();
    Tensor ws = at::empty({(int64_t)lq_grad_norm_workspace_bytes(n)}, norm.options().dtype(at::kByte));
    check(lq_grad_norm(at.data(), outs ? (void* const*)outs->data() : nullptr, g.counts.data(), g.types.data(), n, (float)grad_scale,
                       (float)max_norm, (float*)mut(norm), (float*)mut(coef), (int*)mut(flag), ws.data_ptr(), ws.numel(), stream_of(norm)));
}

std::vector<Tensor> contiguous(const std::vector<Tensor>& v) {
    std::vector<Tensor> c;
    for (const Tensor& t : v) c.push_back(t.contiguous());
    return c;
}
bool all_contiguous(const std::vector<Tensor>& v) {
    return std::all_of(v.begin(), v.end(), [](const Tensor& t) { return t.is_contiguous(); });
}

Tensor global_grad_norm(const py::object& list, double grad_scale) {
    at::NoGradGuard no_grad;
    const std::vector<Tensor> grads = tensors_of(list, "gradients");
    Gradients g(grads);
    c10::cuda::OptionalCUDAGuard guard(grads[0].device());
    Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat).requires_grad(false));
    std::vector<Tensor> copies;  // of strided gradients, alive until the launch is enqueued
    if (!all_contiguous(grads)) {
        copies = contiguous(grads);
        for (size_t i = 0; i < copies.size(); ++i) g.at[i] = copies[i].const_data_ptr();
    }
    grad_norm_call(g, g.at, nullptr, grad_scale, 0.0, norm, Tensor(), Tensor());
    return norm;
}

// Spans of bytes [first, second) that are not empty, by their start.
typedef std::vector<std::pair<uintptr_t, uintptr_t>> Spans;
Spans spans_of(const std::vector<const void*>& at, const std::vector<int64_t>& bytes) {
    Spans s;
    s.reserve(at.size());
    for (size_t i = 0; i < at.size(); ++i)
        if (bytes[i] > 0) s.emplace_back((uintptr_t)at[i], (uintptr_t)at[i] + bytes[i]);
    if (!std::is_sorted(s.begin(), s.end())) std::sort(s.begin(), s.end());
    return s;
}

// The bytes from a tensor's first element to the end of its last; a strided one counts with the gaps between.
int64_t extent_of(const Tensor& t) {
    if (t.numel() == 0 || t.is_contiguous()) return t.nbytes();
    int64_t last = 0;
    for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
    return (last + 1) * t.element_size();
}

// Outputs (contiguous, `bytes` each) may be the gradients themselves, one for one, and share no byte with anything else;
// `extents` are those of the gradients.
void check_outputs(const std::vector<const void*>& at, const std::vector<int64_t>& extents, const std::vector<const void*>& out,
                   const std::vector<int64_t>& bytes) {
    const Spans o = spans_of(out, bytes);
    for (size_t i = 1; i < o.size(); ++i)
        TORCH_CHECK_VALUE(o[i - 1].second <= o[i].first, "the clipped tensors overlap one another (the same tensor twice?)");
    if (&at == &out) return;
    // the usual call, whose outputs are all apart from the gradients: one walk along both
    const Spans g = spans_of(at, extents);
    bool apart = true;
    for (size_t i = 0, j = 0; apart && i < g.size(); ++i) {
        while (j < o.size() && o[j].second <= g[i].first) ++j;
        apart = j == o.size() || o[j].first >= g[i].second;
    }
    if (apart) return;
    std::vector<uintptr_t> starts, ends;
    for (const auto& s : g) starts.push_back(s.first), ends.push_back(s.second);
    std::sort(ends.begin(), ends.end());
    for (size_t i = 0; i < out.size(); ++i) {
        if (bytes[i] == 0) continue;
        const uintptr_t lo = (uintptr_t)out[i], hi = lo + bytes[i];
        // gradients that begin before the output ends, less those that end before it begins: its own alone may be one
        const auto met = (std::lower_bound(starts.begin(), starts.end(), hi) - starts.begin()) - (std::upper_bound(ends.begin(), ends.end(), lo) - ends.begin());
        TORCH_CHECK_VALUE(met <= (out[i] == at[i] ? 1 : 0), "an output overlaps a gradient tensor other than its own");
    }
}
// The same check for Python (tests run it on CPU tensors).
void check_outputs_py(const py::object& grad_list, const py::object& out_list) {
    const std::vector<Tensor> grads = tensors_of(grad_list, "gradients"), outs = tensors_of(out_list, "outputs");
    std::vector<const void*> at, out;
    std::vector<int64_t> extents, bytes;
    for (const Tensor& t : grads) at.push_back(t.const_data_ptr()), extents.push_back(extent_of(t));
    for (const Tensor& t : outs) out.push_back(t.const_data_ptr()), bytes.push_back(t.nbytes());
    if (at == out) check_outputs(at, extents, at, bytes);
    else check_outputs(at, extents, out, bytes);
}

Tensor clip_grad_norm(const py::object& list, double max_norm, const py::object& out_list, double grad_scale) {
    const std::vector<Tensor> grads = tensors_of(list, "gradients");
    const bool out = !out_list.is_none();
    const std::vector<Tensor> given = out ? tensors_of(out_list, "outputs") : std::vector<Tensor>();
    const bool grad_mode = at::GradMode::is_enabled();
    if (grad_mode)
        for (const Tensor& t : given) no_parameter(t);
    at::NoGradGuard no_grad;
    Gradients g(grads, grad_mode && !out);
    TORCH_CHECK_VALUE(max_norm >= 0.0, "max_norm must be >= 0, got ", max_norm);
    const std::vector<Tensor>& outs = out ? given : grads;
    std::vector<const void*> to;
    if (out) {
        Gradients o(outs);
        bool same = outs.size() == grads.size() && o.types == g.types;
        for (size_t i = 0; same && i < outs.size(); ++i) same = outs[i].sizes() == grads[i].sizes();
        TORCH_CHECK_VALUE(same, "out must hold one tensor of the same shape and type for each gradient");
        TORCH_CHECK(outs[0].device() == grads[0].device(), "gradients must live on one CUDA device, got ", grads[0].device(), " and ", outs[0].device());
        to = o.at;
    }
    TORCH_CHECK_VALUE(all_contiguous(outs), out ? "out tensors must be contiguous" : "gradients that are clipped in place must be contiguous");
    std::vector<int64_t> bytes;
    for (size_t i = 0; i < grads.size(); ++i) bytes.push_back(g.counts[i] * (g.types[i] == LQ_F32 ? 4 : 2));
    const bool strided = out && !all_contiguous(grads);
    std::vector<int64_t> extents;
    if (strided)
        for (const Tensor& t : grads) extents.push_back(extent_of(t));
    check_outputs(g.at, strided ? extents : bytes, out ? to : g.at, bytes);
    c10::cuda::OptionalCUDAGuard guard(grads[0].device());
    std::vector<Tensor> copies;
    std::vector<const void*> at = g.at;
    if (strided) {
        copies = contiguous(grads);
        for (size_t i = 0; i < copies.size(); ++i) at[i] = copies[i].const_data_ptr();
    }
    Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat).requires_grad(false));
    grad_norm_call(g, at, out ? &to : &at, grad_scale, max_norm, norm, Tensor(), Tensor());
    for (const Tensor& t : outs) torch::autograd::impl::bump_version(t);
    return norm;
}

// norm, coef and the non-finite flag of one flat f32 bucket.
std::vector<Tensor> bucket_norm(const Tensor& bucket, double max_norm, double grad_scale, const Tensor& flag) {
    at::NoGradGuard no_grad;
    Gradients g({bucket});
    TORCH_CHECK_VALUE(max_norm >= 0.0, "max_norm must be >= 0, got ", max_norm);
    c10::cuda::OptionalCUDAGuard guard(bucket.device());
    Tensor norm = at::empty({}, bucket.options()), coef = at::empty({}, bucket.options());
    grad_norm_call(g, g.at, nullptr, grad_scale, max_norm, norm, coef, flag);
    return {norm, coef};
}

// ---- microscaled 4-bit ------------------------------------------------------------------------------

constexpr int64_t kBlock = 32;

// [rows, k] with contiguous rows that do not overlap.
Tensor matrix_of(const Tensor& x, int64_t k) {
    Tensor m = x.dim() == 2 ? x : x.reshape({-1, k});
    return m.stride(1) == 1 && (m.stride(0) >= k || m.size(0) == 1) ? m : m.contiguous();
}

std::pair<Tensor, Tensor> mx4_quantize(const Tensor& x_) {
    at::NoGradGuard no_grad;
    require_cuda(x_, "x");
    const int type = dtype_code(x_);
    const int64_t k = x_.dim() ? x_.size(-1) : 0;
    TORCH_CHECK_VALUE(k > 0 && k % kBlock == 0, "the last axis must be a positive multiple of ", kBlock, ", got ", x_.sizes());
    c10::cuda::OptionalCUDAGuard guard(x_.device());
    const Tensor x = matrix_of(x_, k);
    const int64_t rows = x.size(0);
    const auto bytes = x.options().dtype(at::kByte).requires_grad(false);
    Tensor codes = at::empty({rows, k / 2}, bytes), scales = at::empty({(int64_t)lq_mx4_scale_bytes(rows, k)}, bytes);
    check(lq_mx4_quantize(ptr(x), type, rows, k, x.stride(0), mut(codes), mut(scales), stream_of(x)));
    return {codes, scales};
}

Tensor mx4_dequantize(const Tensor& codes, const Tensor& scales, int64_t rows, int64_t k, at::ScalarType dtype) {
    require_cuda(codes, "codes");
    c10::cuda::OptionalCUDAGuard guard(codes.device());
    Tensor out = at::empty({rows, k}, codes.options().dtype(dtype));
    check(lq_mx4_dequantize(ptr(codes), ptr(scales), rows, k, mut(out), dtype_code(out), stream_of(codes)));
    return out;
}

Tensor bias_of(const std::optional<Tensor>& bias, const Tensor& w, int64_t m) {
    if (!bias) return Tensor();
    TORCH_CHECK_VALUE(bias->numel() == m && bias->device() == w.device(), "bias must hold ", m, " values on ", w.device(), ", got ", bias->sizes(),
                      " on ", bias->device());
    return bias->scalar_type() == at::kFloat && bias->is_contiguous() ? *bias : bias->to(at::kFloat).contiguous();
}

Tensor mx4_matmul(const Tensor& xc, const Tensor& xs, int64_t n, const Tensor& wc, const Tensor& ws, int64_t m, int64_t k,
                  const std::optional<Tensor>& bias_, at::ScalarType dtype) {
    at::NoGradGuard no_grad;
    require_cuda(xc, "x");
    TORCH_CHECK(xc.device() == wc.device(), "x is on ", xc.device(), ", w on ", wc.device());
    c10::cuda::OptionalCUDAGuard guard(xc.device());
    const Tensor bias = bias_of(bias_, wc, m);
    Tensor y = at::empty({n, m}, xc.options().dtype(dtype));
    check(lq_mx4_matmul(ptr(xc), ptr(xs), n, ptr(wc), ptr(ws), m, k, (const float*)ptr(bias), mut(y), dtype_code(y), stream_of(xc)));
    return y;
}

Tensor mx4_matmul_dx(const Tensor& dy_, const Tensor& wc, const Tensor& ws, int64_t m, int64_t k) {
    at::NoGradGuard no_grad;
    require_cuda(dy_, "dy");
    TORCH_CHECK_VALUE(dy_.dim() == 2 && dy_.size(1) == m, "dy must be [n, ", m, "], got ", dy_.sizes());
    TORCH_CHECK(dy_.device() == wc.device(), "dy is on ", dy_.device(), ", w on ", wc.device());
    const int type = dtype_code(dy_);
    c10::cuda::OptionalCUDAGuard guard(dy_.device());
    const Tensor dy = whole(dy_);
    const int64_t n = dy.size(0);
    Tensor dx = at::empty({n, k}, dy.options().requires_grad(false));
    // of this call alone: from the pool of the current stream, or of the graph being captured
    Tensor space = at::empty({(int64_t)lq_mx4_matmul_dx_workspace_bytes(n, m, k, type)}, wc.options());
    check(lq_mx4_matmul_dx(ptr(dy), type, n, ptr(wc), ptr(ws), m, k, mut(dx), mut(space), space.numel(), stream_of(dy)));
    return dx;
}

struct Mx4LinearBackward : public Node {
    Tensor codes, scales;  // the weight is state, never a graph parent
    int64_t m = 0, k = 0;
    std::vector<int64_t> shape;

    std::string name() const override { return "Mx4LinearBackward"; }
    variable_list apply(variable_list&& grads) override {
        const bool asked = at::GradMode::is_enabled();
        if (!grads[0].defined() || !task_should_compute_output(0)) return {Tensor()};
        no_tangents({&grads[0]}, "Mx4Linear's backward");
        at::NoGradGuard no_grad_in_here;
        const Tensor dy = grads[0].dim() == 2 ? grads[0] : grads[0].reshape({-1, m});
        variable_list out = {mx4_matmul_dx(dy, codes, scales, m, k).view(shape)};
        at::AutoGradMode as_asked(asked);
        return once(std::move(out), "Mx4Linear");
    }
};

// dequant(quant(x)) . dequant(w)^T + bias over the last axis of x; backward dy . dequant(w).
Tensor mx4_linear(const Tensor& x_, const Tensor& wc, const Tensor& ws, int64_t m, int64_t k, const std::optional<Tensor>& bias_) {
    const Tensor bias0 = defined(bias_);
    no_tangents({&x_, &bias0}, "Mx4Linear");
    require_cuda(x_, "x");
    TORCH_CHECK_VALUE(x_.dim() >= 1 && x_.size(-1) == k, "last dim ", x_.dim() ? x_.size(-1) : 0, " != d_in ", k);
    TORCH_CHECK(x_.device() == wc.device(), "x is on ", x_.device(), ", w on ", wc.device());
    const int type = dtype_code(x_);
    c10::cuda::OptionalCUDAGuard guard(x_.device());
    Tensor y;
    {
        at::NoGradGuard no_grad;
        const Tensor x = matrix_of(x_, k), bias = bias_of(bias_, wc, m);
        const int64_t n = x.size(0);
        auto shape = x_.sizes().vec();
        shape.back() = m;
        y = at::empty(shape, x.options().requires_grad(false));
        Tensor space = at::empty({(int64_t)lq_mx4_linear_workspace_bytes(n, k)}, wc.options());
        check(lq_mx4_linear(ptr(x), type, n, x.stride(0), ptr(wc), ptr(ws), m, k, (const float*)ptr(bias), mut(y), mut(space), space.numel(),
                            stream_of(x)));
    }
    if (wants_grad({&x_})) {
        auto node = std::shared_ptr<Mx4LinearBackward>(new Mx4LinearBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x_));
        node->codes = wc, node->scales = ws, node->m = m, node->k = k, node->shape = x_.sizes().vec();
        torch::autograd::set_history(y, node);
    }
    return y;
}

// With an adapter on the same input: quant(x) . W^T + bias + scaling * (x . A) . B in bf16.
struct Mx4LoraBackward : public Node {
    Tensor codes, scales, mirror, h;   // state, never graph parents
    Tensor bucket_a, bucket_b;         // views of a flat gradient buffer, or undefined
    SavedVariable x, a, b;             // a and b for their versions and .grad: the mirror holds their values
    int64_t n = 0, m = 0, k = 0, rank = 0;
    double scaling = 1.0;
    std::vector<int64_t> shape;
    bool released = false;

    std::string name() const override { return "Mx4LoraBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable* v : {&x, &a, &b}) v->reset_data();
        h.reset();
        released = true;
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        TORCH_CHECK(!released, "Trying to backward through the graph a second time: specify retain_graph=True");
        return once(gradients(std::move(grads)), "the microscaled linear with an adapter");
    }
    variable_list gradients(variable_list&& grads) {
        variable_list out(3);
        if (!grads[0].defined()) return out;
        no_tangents({&grads[0]}, "the backward of the microscaled linear with an adapter");
        const Tensor saved = x.unpack(), as = a.unpack(), bs = b.unpack();
        at::NoGradGuard no_grad;
        c10::cuda::OptionalCUDAGuard guard(codes.device());
        const Tensor xs = whole(restored(saved, {n, k}, at::kBFloat16, codes.device(), "x")), dy = whole(grads[0].reshape({n, m}));
        // straight into the flat buffer only while the factors' .grad are its views: whoever reset them expects autograd's
        auto lives = [](const Tensor& p, const Tensor& view) {
            return view.defined() && p.grad().defined() && p.grad().const_data_ptr() == view.const_data_ptr();
        };
        const bool direct = lives(as, bucket_a) && lives(bs, bucket_b);
        const auto opts = xs.options().requires_grad(false);
        Tensor da, db;
        if (task_should_compute_output(0)) out[0] = at::empty({n, k}, opts);
        if (task_should_compute_output(1)) da = direct ? bucket_a : at::empty({k, rank}, opts.dtype(at::kFloat));
        if (task_should_compute_output(2)) db = direct ? bucket_b : at::empty({rank, m}, opts.dtype(at::kFloat));
        // of this call alone: from the pool of the current stream, or of the graph being captured
        Tensor space = at::empty({(int64_t)lq_mx4_lora_workspace_bytes(n, m, k, (int)rank, 1)}, opts.dtype(at::kByte));
        check(lq_mx4_lora_bwd(ptr(dy), ptr(xs), (const float*)ptr(h), n, ptr(codes), ptr(scales), m, k, ptr(mirror), (int)rank, (float)scaling,
                              mut(out[0]), (float*)mut(da), (float*)mut(db), direct, mut(space), space.numel(), stream_of(xs)));
        if (out[0].defined()) out[0] = out[0].view(shape);
        if (!direct) out[1] = da, out[2] = db;
        return out;
    }
};

Tensor mx4_lora_linear(const Tensor& x_, const Tensor& wc, const Tensor& ws, int64_t m, int64_t k, const std::optional<Tensor>& bias_,
                       const Tensor& a, const Tensor& b, double scaling, const Tensor& mirror, const std::optional<Tensor>& bucket_a,
                       const std::optional<Tensor>& bucket_b) {
    const Tensor bias0 = defined(bias_);
    no_tangents({&x_, &a, &b, &bias0}, "the microscaled linear with an adapter");
    require_cuda(x_, "x");
    TORCH_CHECK_VALUE(x_.dim() >= 1 && x_.size(-1) == k, "last dim ", x_.dim() ? x_.size(-1) : 0, " != d_in ", k);
    TORCH_CHECK_TYPE(x_.scalar_type() == at::kBFloat16, "the fused adapter takes bf16 activations, got ", x_.scalar_type());
    const std::pair<const char*, const Tensor*> named[] = {{"w", &wc}, {"lora_a", &a}, {"lora_b", &b}, {"the mirror", &mirror}};
    for (const auto& [name, v] : named) TORCH_CHECK(v->device() == x_.device(), name, " is on ", v->device(), ", x on ", x_.device());
    TORCH_CHECK_TYPE(a.scalar_type() == at::kFloat && b.scalar_type() == at::kFloat, "LoRA factors must be f32, got ", a.scalar_type(), " and ",
                     b.scalar_type());
    const int64_t rank = a.dim() == 2 ? a.size(1) : 0;
    TORCH_CHECK_VALUE(rank > 0 && a.size(0) == k && b.dim() == 2 && b.size(0) == rank && b.size(1) == m, "lora_a must be [", k,
                      ", rank], lora_b [rank, ", m, "], got ", a.sizes(), " and ", b.sizes());
    TORCH_CHECK_VALUE(mirror.is_contiguous() && mirror.nbytes() >= lq_lora_mirror_bytes(k, m, (int)rank), "the mirror is too small");
    c10::cuda::OptionalCUDAGuard guard(x_.device());
    const bool grad = wants_grad({&x_, &a, &b});
    Tensor x, y, h;
    {
        at::NoGradGuard no_grad;
        x = whole(x_.reshape({-1, k}));
        const Tensor bias = bias_of(bias_, wc, m);
        const int64_t n = x.size(0);
        auto shape = x_.sizes().vec();
        shape.back() = m;
        const auto opts = x.options().requires_grad(false);
        y = at::empty(shape, opts);
        if (grad) h = at::empty({n, rank}, opts.dtype(at::kFloat));
        Tensor space = at::empty({(int64_t)lq_mx4_lora_workspace_bytes(n, m, k, (int)rank, 0)}, wc.options());
        check(lq_mx4_lora_fwd(ptr(x), n, ptr(wc), ptr(ws), m, k, (const float*)ptr(bias), ptr(mirror), (int)rank, (float)scaling, mut(y),
                              (float*)mut(h), mut(space), space.numel(), stream_of(x)));
    }
    if (grad) {
        auto node = std::shared_ptr<Mx4LoraBackward>(new Mx4LoraBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x_, a, b));
        node->x = SavedVariable(x, false), node->a = SavedVariable(a, false), node->b = SavedVariable(b, false);
        node->codes = wc, node->scales = ws, node->mirror = mirror, node->h = h;
        node->bucket_a = defined(bucket_a), node->bucket_b = defined(bucket_b);
        node->n = x.size(0), node->m = m, node->k = k, node->rank = rank, node->scaling = scaling, node->shape = x_.sizes().vec();
        torch::autograd::set_history(y, node);
    }
    return y;
}

}  // namespace

PYBIND11_MODULE(_lq_torch, mod) {
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const LqFailure& e) {
            py::object type = py::module_::import("loractl_b200._lib").attr("LqError");
            PyErr_SetObject(type.ptr(), type(e.status, std::string(e.what())).ptr());
        }
    });
    mod.def("residual_norm", &residual_norm);
    mod.def("global_grad_norm", &global_grad_norm);
    mod.def("clip_grad_norm", &clip_grad_norm);
    mod.def("check_outputs", &check_outputs_py);
    mod.def("bucket_norm", &bucket_norm);
    mod.def("mx4_quantize", &mx4_quantize);
    mod.def("mx4_dequantize", &mx4_dequantize);
    mod.def("mx4_matmul", &mx4_matmul);
    mod.def("mx4_matmul_dx", &mx4_matmul_dx);
    mod.def("mx4_linear", &mx4_linear);
    mod.def("mx4_lora_linear", &mx4_lora_linear);
}
