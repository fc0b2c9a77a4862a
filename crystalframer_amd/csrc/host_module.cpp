// Host side of the whole-model pass and of the optimizer, as a Python extension module: what stands between the framework's
// tensors and the entry points of the library for every pass, in native code.
//
// A pass of the library is 30 (inference) to 80 launches; around them Python spent 90 us on looking the model and the batch
// over, 190 us on the gradients' tensors and the bookkeeping of the autograd function and 100 us on the optimizer's job
// table, per training step of the 4-layer model with its 65 parameters, as long as the GPU takes for a step on 13 crystals.
//
// The residual norms (norms.py) are here for the same reason: their launches take 3 to 10 us on the sizes of a crystal batch, and the
// checks, the argument structure and the autograd function in Python took 140 us per forward and backward pass.
//
// The entry points are called through addresses that the Python side hands over: the module does not link the library.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/SavedTensorHooks.h>

#include <mutex>

#include "../../include/crystalframer_hip.h"

namespace py = pybind11;

namespace {

struct Library {
    int64_t (*sizes)(const cfh_model*, const cfh_model_batch*, size_t*) = nullptr;
    int (*forward)(const cfh_model*, const cfh_model_batch*, float*) = nullptr;
    int (*backward)(const cfh_model*, const cfh_model_batch*, const float*, void*, size_t, float*) = nullptr;
    const char* (*last_error)() = nullptr;
} g_lib;

void check(int rc, const char* what) {
    TORCH_CHECK(rc == 0, what, " failed (", rc, "): ", g_lib.last_error ? g_lib.last_error() : "");
}

// The launches of a pass share the scratch of their stream, and a backward pass is enqueued by a thread of the autograd engine
// without the interpreter's lock: no other thread's launches come between those of a pass.  (Nothing that is done with this
// held waits for the interpreter.)
std::mutex g_enqueue;

at::Tensor bytes(size_t n, const c10::Device& dev) {
    return at::empty({(int64_t)n}, at::TensorOptions().dtype(at::kByte).device(dev));
}
// Memory of a pass.  Sizes are rounded up to an eighth of their power of two: the batches of an epoch differ a little from each
// other, and the framework's allocator then finds a block to use again.
at::Tensor arena(size_t n, const c10::Device& dev) {
    size_t step = 512;
    int bits = 0;
    for (size_t v = n; v; v >>= 1) bits++;
    if (bits > 4 && ((size_t)1 << (bits - 4)) > step) step = (size_t)1 << (bits - 4);
    return bytes((n + step - 1) / step * step, dev);
}

// Memory whose address the library was given: kept, and still where it was.
struct Held {
    c10::Storage storage;
    const void* base;
    explicit Held(const at::Tensor& t) : storage(t.storage()), base(storage.data()) {}
    bool there() const { return storage.data() == base; }
};

// What a plan's passes share (see model_pass._Plan).
struct Shared {
    std::vector<at::Tensor> params;            // in the order of the library's gradients
    std::vector<at::Tensor> gauss;
    std::vector<Held> held;                    // of params and gauss as the plan was made
    std::vector<std::vector<int64_t>> sizes;   // of params
    std::vector<int64_t> offset;               // of a parameter's gradient, in floats
    c10::Device device{c10::kCPU};
    int64_t feat = 0, D = 0, H = 0, out_features = 0;
};

// Structures of the library call, kept alive by the Python object that made them.
struct Model {
    const cfh_model* m;
    std::shared_ptr<void> owner;               // drops a reference to the Python object, with the GIL held
};
std::shared_ptr<void> hold(py::object o) {
    return std::shared_ptr<void>(o.release().ptr(), [](void* p) {
        if (!Py_IsInitialized()) return;
        py::gil_scoped_acquire gil;
        Py_DECREF(reinterpret_cast<PyObject*>(p));
    });
}

struct ModelPassBackward : public torch::autograd::Node {
    std::shared_ptr<Shared> plan;
    Model model;
    cfh_model_batch b;
    int64_t total;
    size_t scratch_bytes;
    std::vector<uint64_t> seeds;
    at::Tensor arena_, workspace_;
    std::vector<torch::autograd::SavedVariable> data;
    std::vector<Held> held;                    // of the batch
    std::vector<at::Tensor> first;
    std::vector<int64_t> versions;
    bool released = false;

    std::string name() const override { return "ModelPassHIPBackward"; }
    void release_variables() override {
        released = true;
        arena_.reset();
        workspace_.reset();
        data.clear();
        held.clear();
        first.clear();
    }
    static std::vector<int64_t> current_versions(const Shared& P) {
        std::vector<int64_t> v;
        v.reserve(P.params.size() + P.gauss.size());
        for (auto& p : P.params) v.push_back((int64_t)p._version());
        for (auto& p : P.gauss) v.push_back((int64_t)p._version());
        return v;
    }
    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
        TORCH_CHECK(!released, "the backward pass of this model output has been made and what its forward pass kept is given back; to "
                    "make it a second time, make the first one with retain_graph=True");
        // The .data of a parameter or of the batch was exchanged since the forward pass: the addresses are those of the storages
        // before, which are held, and the gradients those of what the forward pass computed.
        const size_t n = plan->params.size();
        torch::autograd::variable_list out(n);
        if (!grads[0].defined()) return out;
        TORCH_CHECK(current_versions(*plan) == versions,
                    "a parameter of the model was modified by an inplace operation between its forward and its backward pass");
        for (auto& s : data) s.unpack(shared_from_this());       // (says so if an input was changed in place)
        for (auto* list : {&plan->held, &held})
            for (auto& h : *list)
                TORCH_CHECK(h.there(), "the memory of a parameter of the model or of the batch was resized or given back between the "
                            "forward and the backward pass");
        const at::Tensor gout = grads[0].detach().to(at::kFloat).contiguous();
        c10::DeviceGuard guard(plan->device);
        const at::Tensor flat = at::empty({total}, at::TensorOptions().dtype(at::kFloat).device(plan->device));
        const at::Tensor scratch = arena(scratch_bytes, plan->device);
        cfh_model_batch q = b;
        q.workspace = workspace_.data_ptr();
        q.workspace_bytes = (size_t)workspace_.numel();
        q.stream = (void*)c10::hip::getCurrentHIPStream(plan->device.index()).stream();
        int rc;
        {
            std::lock_guard<std::mutex> lock(g_enqueue);
            rc = g_lib.backward(model.m, &q, gout.data_ptr<float>(), scratch.data_ptr(), (size_t)scratch.numel(),
                                flat.data_ptr<float>());
        }
        check(rc, "cfh_model_backward");
        // a tensor of its own per parameter over the common storage (autograd adopts it as .grad: nobody else holds it)
        const c10::Storage& storage = flat.storage();
        for (size_t i = 0; i < n; i++) {
            if (!task_should_compute_output(i)) continue;
            auto t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(storage), flat.key_set(), flat.dtype());
            c10::TensorImpl* impl = t.unsafeGetTensorImpl();
            impl->set_storage_offset(plan->offset[i]);
            impl->set_sizes_contiguous(plan->sizes[i]);
            out[i] = std::move(t);
        }
        return out;
    }
};

struct Plan {
    std::shared_ptr<Shared> S = std::make_shared<Shared>();
    // Borrowed: the Python object that owns the plan keeps them (a reference from here would close a cycle that the garbage
    // collector cannot see).
    struct Link { PyObject *dict, *key, *value; };
    std::vector<Link> links;
    struct Walked { PyObject* dict; Py_ssize_t entries; };
    std::vector<Walked> walked;
    struct Layout { void* ptr; std::vector<int64_t> sizes; };
    std::vector<Layout> layout;                // of params, then gauss; all of them contiguous float32

    Plan(py::list links_, py::list walked_, std::vector<at::Tensor> params, std::vector<at::Tensor> gauss, int64_t feat, int64_t D,
         int64_t H, int64_t out_features) {
        for (auto l : links_) {
            auto t = py::reinterpret_borrow<py::tuple>(l);
            links.push_back({PyTuple_GET_ITEM(t.ptr(), 0), PyTuple_GET_ITEM(t.ptr(), 1), PyTuple_GET_ITEM(t.ptr(), 2)});
        }
        for (auto w : walked_) {
            auto t = py::reinterpret_borrow<py::tuple>(w);
            walked.push_back({PyTuple_GET_ITEM(t.ptr(), 0), PyLong_AsSsize_t(PyTuple_GET_ITEM(t.ptr(), 1))});
        }
        S->params = std::move(params);
        S->gauss = std::move(gauss);
        int64_t off = 0;
        for (auto& p : S->params) {
            S->offset.push_back(off);
            off += p.numel();
        }
        for (auto* list : {&S->params, &S->gauss})
            for (auto& p : *list) {
                layout.push_back({p.data_ptr(), p.sizes().vec()});
                S->held.emplace_back(p);
            }
        for (auto& p : S->params) S->sizes.push_back(p.sizes().vec());
        S->device = S->params[0].device();
        S->feat = feat; S->D = D; S->H = H; S->out_features = out_features;
    }
    // Whether the modules and parameters are still those the plan was made from, no more and no fewer, in the same storages
    // and with the same layout.
    bool current() const {
        for (auto& w : walked)
            if (PyDict_GET_SIZE(w.dict) != w.entries) return false;
        for (auto& l : links) {
            PyObject* v = PyDict_GetItemWithError(l.dict, l.key);
            if (v != l.value) {
                if (!v && PyErr_Occurred()) throw py::error_already_set();
                if (v || l.value != Py_None) return false;
            }
        }
        const Layout* l = layout.data();
        for (auto* list : {&S->params, &S->gauss})
            for (auto& p : *list) {
                if (p.data_ptr() != l->ptr || p.scalar_type() != at::kFloat || !p.is_contiguous() || p.sizes() != l->sizes)
                    return false;
                l++;
            }
        return true;
    }
    // The batch is one that the library call takes: it reads as many words of each tensor as x and trans have rows.
    bool accepts(const at::Tensor& x, const at::Tensor& pos, const at::Tensor& batch, const at::Tensor& trans,
                 const at::Tensor& sizes) const {
        auto good = [&](const at::Tensor& t, at::ScalarType ty) {
            return t.scalar_type() == ty && t.device() == S->device && t.is_contiguous();
        };
        return good(x, at::kFloat) && good(pos, at::kFloat) && good(trans, at::kFloat) && good(batch, at::kLong) &&
               good(sizes, at::kLong) && x.dim() == 2 && x.size(1) == S->feat && x.size(0) > 0 &&
               pos.dim() == 2 && pos.size(0) == x.size(0) && pos.size(1) == 3 && batch.dim() == 1 && batch.size(0) == x.size(0) &&
               trans.dim() == 3 && trans.size(1) == 3 && trans.size(2) == 3 && sizes.dim() == 1 && sizes.size(0) == trans.size(0);
    }
    // How many of the parameters want a gradient: 0 none, 1 some, 2 all.
    int wanted() const {
        size_t n = 0;
        for (auto& p : S->params) n += p.requires_grad() ? 1 : 0;
        return n == 0 ? 0 : (n == S->params.size() ? 2 : 1);
    }
    // out (B, features).  workspace: called with a size, gives the scratch of the current stream.  x0, qkv0: see
    // cfh_model_batch (undefined: made by the library).  noise: seeds of the layers' frame searches, or empty.
    at::Tensor forward(uintptr_t model, py::object owner, const at::Tensor& x, const at::Tensor& pos, const at::Tensor& batch,
                       const at::Tensor& trans, const at::Tensor& sizes, int64_t E, bool keep, py::function workspace,
                       std::vector<uint64_t> noise, std::vector<at::Tensor> first) {
        const cfh_model* m = reinterpret_cast<const cfh_model*>(model);
        cfh_model_batch b;
        std::memset(&b, 0, sizeof(b));
        b.x = x.data_ptr<float>(); b.pos = pos.data_ptr<float>(); b.batch = batch.data_ptr<int64_t>();
        b.tvecs = trans.data_ptr<float>(); b.sizes = sizes.data_ptr<int64_t>();
        b.N = x.size(0); b.B = trans.size(0); b.E = E;
        b.keep = keep ? 1 : 0;
        if (!first.empty()) { b.x0 = first[0].data_ptr<float>(); b.qkv0 = first[1].data_ptr<float>(); }
        if (!noise.empty()) b.noise_seeds = noise.data();
        size_t nbytes[4] = {0, 0, 0, 0};
        const int64_t total = g_lib.sizes(m, &b, nbytes);
        if (total < 0) check((int)total, "cfh_model_sizes");
        at::Tensor arena_ = arena(nbytes[0], S->device);
        at::Tensor ws = py::cast<at::Tensor>(workspace(keep ? std::max(nbytes[1], nbytes[3]) : nbytes[1]));
        at::Tensor out = at::empty({b.B, S->out_features}, at::TensorOptions().dtype(at::kFloat).device(S->device));
        b.arena = arena_.data_ptr(); b.arena_bytes = (size_t)arena_.numel();
        b.workspace = ws.data_ptr(); b.workspace_bytes = (size_t)ws.numel();
        b.stream = (void*)c10::hip::getCurrentHIPStream(S->device.index()).stream();
        int rc;
        {
            std::lock_guard<std::mutex> lock(g_enqueue);
            rc = g_lib.forward(m, &b, out.data_ptr<float>());
        }
        check(rc, "cfh_model_forward");
        if (!keep) return out;
        auto node = std::shared_ptr<ModelPassBackward>(new ModelPassBackward(), torch::autograd::deleteNode);
        node->plan = S;
        node->model = Model{m, hold(std::move(owner))};
        node->seeds = std::move(noise);            // (the vector's memory moves along: b.noise_seeds stays right)
        node->b = b;
        node->total = total;
        node->scratch_bytes = nbytes[2];
        node->arena_ = std::move(arena_);
        node->workspace_ = std::move(ws);
        node->first = std::move(first);
        node->versions = ModelPassBackward::current_versions(*S);
        for (const at::Tensor* t : {&x, &pos, &batch, &trans, &sizes}) {
            node->data.emplace_back(*t, false);
            node->held.emplace_back(*t);
        }
        torch::autograd::edge_list edges;
        edges.reserve(S->params.size());
        for (auto& p : S->params) edges.push_back(torch::autograd::impl::gradient_edge(p));
        node->set_next_edges(std::move(edges));
        torch::autograd::set_history(out, node);
        return out;
    }
};

// Who would see the framework's operations in this thread beside autograd's backward pass.
enum : int { WATCHED = 1, FUNCTION_MODE = 2, SAVED_TENSOR_HOOKS = 4 };
int watchers() {
    int seen = 0;
    if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::stack_len() > 0 ||
        c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode))
        seen |= WATCHED;
    if (at::impl::PythonTorchFunctionTLS::stack_len() > 0) seen |= FUNCTION_MODE;
    if (at::SavedTensorDefaultHooks::get_hooks().has_value()) seen |= SAVED_TENSOR_HOOKS;
    return seen;
}

// ---- residual norms ------------------------------------------------------------------------------------------------------------
struct NormLibrary {
    int (*forward)(const cfh_residual_norm*, void*, void*, float*, void*) = nullptr;
    size_t (*backward_bytes)(const cfh_residual_norm*) = nullptr;
    int (*backward)(const cfh_residual_norm*, const float*, const void*, const void*, void*, void*, void*, void*, void*, void*, void*, void*,
                    size_t, void*) = nullptr;
} g_norm;

constexpr int64_t NORM_MAX_DIM = 16384;
enum { X, BLOCK, GATE, WEIGHT, BIAS, BLOCK_WEIGHT, BLOCK_BIAS, NORM_TENSORS };
const char* const NORM_NAMES[NORM_TENSORS] = {"x", "block", "gate", "weight", "bias", "block_weight", "block_bias"};
using NormTensors = std::array<at::Tensor, NORM_TENSORS>;

struct NormSpec {
    int norm, block_norm;
    float eps, block_eps, residual_scale, block_scale;
    bool keep, twice;
};

int element_type(at::ScalarType t) {
    return t == at::kFloat ? CFH_FLOAT32 : t == at::kBFloat16 ? CFH_BFLOAT16 : t == at::kHalf ? CFH_FLOAT16 : -1;
}

// How many rows the gate has: 1 (a factor per channel), one for as many rows of x after one another, or one for each.
int64_t gate_rows(const at::Tensor& gate, const at::Tensor& x) {
    const int64_t D = x.size(-1);
    if (gate.dim() == 1 && gate.size(0) == D) return 1;
    if (gate.dim() == x.dim() && gate.dim() > 0 && gate.size(-1) == D) {
        int64_t k = 0, rows = 1;
        while (k + 1 < gate.dim() && gate.size(k) == x.size(k)) rows *= gate.size(k++);
        while (k + 1 < gate.dim() && gate.size(k) == 1) k++;
        if (k + 1 == gate.dim()) return rows;
    }
    TORCH_CHECK_VALUE(false, "gate of shape ", gate.sizes(), " for x of shape ", x.sizes(), ": its last dimension must be that of x, and its "
                      "leading dimensions none, or those of x up to some dimension and 1 from there on");
}

// A tensor whose class makes the framework's operations itself: it has no memory of its own (its address is NULL, which the library
// takes for an argument left out).
bool wrapped(const at::Tensor& t) { return t.defined() && t.unsafeGetTensorImpl()->is_python_dispatch(); }

void check_norm(const NormTensors& t, const NormSpec& s) {
    const at::Tensor& x = t[X];
    for (int k = 0; k < NORM_TENSORS; k++) TORCH_CHECK_TYPE(!wrapped(t[k]), NORM_NAMES[k], " is a tensor of a class with operations of its own: one in memory is needed");
    for (const auto& u : t)
        TORCH_CHECK(!u.defined() || u.is_cuda(), "crystalframer_amd operators run on a HIP device only (tensor on ", u.device(),
                    "); there is no CPU path");
    TORCH_CHECK_TYPE(element_type(x.scalar_type()) >= 0, "x of ", x.scalar_type(), ": float32, bfloat16 or float16");
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= NORM_MAX_DIM, "x of shape ", x.sizes(), ": 1 to ", NORM_MAX_DIM, " channels");
    TORCH_CHECK_VALUE(s.eps >= 0.0f && s.block_eps >= 0.0f, "eps and block_eps must not be negative");
    TORCH_CHECK_VALUE(s.norm || s.keep, "norm None with keep_residual False: nothing is left to return");
    TORCH_CHECK_VALUE(s.norm || !(t[WEIGHT].defined() || t[BIAS].defined()), "weight and bias belong to a norm");
    TORCH_CHECK_VALUE(s.block_norm || !(t[BLOCK_WEIGHT].defined() || t[BLOCK_BIAS].defined()), "block_weight and block_bias belong to a block_norm");
    TORCH_CHECK_VALUE(t[BLOCK].defined() || !(t[GATE].defined() || s.block_norm), "gate and block_norm belong to a block");
    for (int k : {BLOCK, GATE})
        TORCH_CHECK_TYPE(!t[k].defined() || t[k].scalar_type() == x.scalar_type(), NORM_NAMES[k], " of ", t[k].scalar_type(), ", x of ",
                         x.scalar_type(), ": they must have one type");
    TORCH_CHECK_VALUE(!t[BLOCK].defined() || t[BLOCK].sizes() == x.sizes(), "block of shape ", t[BLOCK].sizes(), ", x of shape ", x.sizes());
    c10::optional<at::ScalarType> kind;
    for (int k : {WEIGHT, BIAS, BLOCK_WEIGHT, BLOCK_BIAS}) {
        if (!t[k].defined()) continue;
        const at::ScalarType type = t[k].scalar_type();
        TORCH_CHECK_VALUE(t[k].dim() == 1 && t[k].size(0) == x.size(-1), NORM_NAMES[k], " of shape ", t[k].sizes(), " for ", x.size(-1), " channels");
        TORCH_CHECK_TYPE((type == x.scalar_type() || type == at::kFloat) && (!kind || *kind == type), NORM_NAMES[k], " of ", type,
                         ": weights and biases have one type, that of x or float32");
        kind = type;
    }
    for (const auto& u : t) TORCH_CHECK(!u.defined() || u.device() == x.device(), "the tensors are on different devices");
    if (t[GATE].defined()) gate_rows(t[GATE], x);
    TORCH_CHECK_VALUE(!s.twice || (s.norm == CFH_NORM_LAYER && !s.block_norm && !t[GATE].defined() && s.residual_scale == 1.0f && s.block_scale == 1.0f),
                      "second derivatives are those of a layer norm of x or of x + block");
}

// t as rows of its last dimension, `stride` elements apart: in place if they lie evenly and their elements next to each other.
at::Tensor rows_of(const at::Tensor& t, int64_t& stride) {
    stride = t.size(-1);
    if (t.is_contiguous()) return t;
    if (t.dim() == 2 && t.stride(1) == 1 && t.stride(0) >= t.size(1)) {
        stride = t.stride(0);
        return t;
    }
    return t.contiguous();
}

// The library's arguments; `t` becomes the tensors that they point to.
cfh_residual_norm norm_args(NormTensors& t, const NormSpec& s) {
    cfh_residual_norm a;
    std::memset(&a, 0, sizeof(a));
    a.struct_size = (int32_t)sizeof(a);
    a.dtype = a.weight_dtype = element_type(t[X].scalar_type());
    a.norm = s.norm; a.block_norm = s.block_norm;
    a.eps = s.eps; a.block_eps = s.block_eps; a.residual_scale = s.residual_scale; a.block_scale = s.block_scale;
    a.dim = t[X].size(-1);
    a.rows = t[X].numel() / a.dim;
    if (t[GATE].defined()) a.gate_rows = gate_rows(t[GATE], t[X]);
    t[X] = rows_of(t[X], a.x_stride);
    if (t[BLOCK].defined()) t[BLOCK] = rows_of(t[BLOCK], a.block_stride);
    for (int k = GATE; k < NORM_TENSORS; k++) {
        if (!t[k].defined()) continue;
        t[k] = t[k].contiguous();
        if (k >= WEIGHT) a.weight_dtype = element_type(t[k].scalar_type());
    }
    auto p = [&](int k) { return t[k].defined() ? t[k].data_ptr() : nullptr; };
    a.x = p(X); a.block = p(BLOCK); a.gate = p(GATE); a.weight = p(WEIGHT); a.bias = p(BIAS); a.block_weight = p(BLOCK_WEIGHT);
    a.block_bias = p(BLOCK_BIAS);
    return a;
}
void* raw_stream(const at::Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// A gradient of a leaf that an eager graph still holds is accumulated on that graph's stream, which a backward pass under capture must
// not wait for: that ends the process, so it is refused here, before this pass records anything.
void check_capture(const torch::autograd::Node& node, const c10::Device& device, const char* what) {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    const c10::StreamId now = c10::hip::getCurrentHIPStream(device.index()).unwrap().id();
    for (const auto& edge : node.next_edges()) {
        const auto* const leaf = dynamic_cast<const torch::autograd::AccumulateGrad*>(edge.function.get());
        if (!leaf) continue;
        const auto stream = edge.function->stream();
        TORCH_CHECK(!stream || stream->device_index() != device.index() || stream->id() == now, "the backward pass of ", what, " is captured while a graph that was made on another stream "
                    "still holds one of its parameters or inputs: let go of that graph's outputs (a loss, a prediction) first");
    }
}

struct ResidualNormBackward : public torch::autograd::Node {
    NormSpec spec;
    bool joined = false;                       // `saved[X]` is h (the last of the outputs that are kept for this)
    std::vector<int64_t> shape;
    at::ScalarType weight_type = at::kFloat;   // of weight and bias
    std::array<torch::autograd::SavedVariable, NORM_TENSORS> saved;
    at::Tensor stats;
    bool released = false;

    std::string name() const override { return "ResidualNormHIPBackward"; }
    void release_variables() override {
        released = true;
        for (auto& s : saved) s.reset_data();
        stats.reset();
    }
    // The same gradients by the framework's operations, which have derivatives of their own: for a backward pass that is recorded
    // (create_graph) through a layer norm with at most an addition before it.
    torch::autograd::variable_list differentiable_gradients(const at::Tensor& gh, const at::Tensor& gy) {
        torch::autograd::variable_list out(NORM_TENSORS);
        at::Tensor dh = gh;
        if (gy.defined()) {
            auto wide = [&](int k) {
                const at::Tensor t = saved[k].unpack(shared_from_this());
                return t.defined() ? c10::optional<at::Tensor>(t.to(at::kFloat)) : c10::nullopt;
            };
            at::Tensor h = *wide(X);
            if (const auto block = wide(BLOCK)) h = h + *block;
            const auto weight = wide(WEIGHT), bias = wide(BIAS);
            at::Tensor mean, inverse, dweight, dbias, dx;
            std::tie(std::ignore, mean, inverse) = at::native_layer_norm(h.detach(), {shape.back()}, c10::nullopt, c10::nullopt, spec.eps);
            std::tie(dx, dweight, dbias) = at::native_layer_norm_backward(
                gy.to(at::kFloat), h, {shape.back()}, mean, inverse, weight, bias,
                {task_should_compute_output(X) || task_should_compute_output(BLOCK), task_should_compute_output(WEIGHT), task_should_compute_output(BIAS)});
            if (dx.defined()) dh = (gh.defined() ? gh.to(at::kFloat) + dx : dx).to(gy.scalar_type());
            if (dweight.defined()) out[WEIGHT] = dweight.to(weight_type);
            if (dbias.defined()) out[BIAS] = dbias.to(weight_type);
        }
        for (int k : {X, BLOCK})
            if (task_should_compute_output(k)) out[k] = dh;
        return out;
    }
    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
        TORCH_CHECK(!released, "Trying to backward through a residual norm a second time: make the first pass with retain_graph=True");
        torch::autograd::variable_list out(NORM_TENSORS);
        at::Tensor gh = spec.keep ? grads[0] : at::Tensor(), gy = spec.norm ? grads[spec.keep ? 1 : 0] : at::Tensor();
        if (!gh.defined() && !gy.defined()) return out;
        NormTensors t;
        for (int k = 0; k < NORM_TENSORS; k++) {
            t[k] = saved[k].unpack(shared_from_this());
            if (t[k].defined()) t[k] = t[k].detach();
        }
        c10::DeviceGuard guard(t[X].device());
        check_capture(*this, t[X].device(), "a residual norm");
        const bool differentiable = at::GradMode::is_enabled();
        if (differentiable && spec.twice) return differentiable_gradients(gh, gy);
        {
            at::AutoDispatchBelowADInplaceOrView below;
            const auto options = t[X].options();
            for (int k = GATE; k < NORM_TENSORS; k++)
                if (t[k].defined() && task_should_compute_output(k)) out[k] = at::empty(t[k].sizes(), t[k].options());
            cfh_residual_norm a = norm_args(t, spec);
            a.joined = joined ? 1 : 0;
            const bool same = !t[GATE].defined() && !spec.block_norm && spec.residual_scale == spec.block_scale;
            if (task_should_compute_output(X)) out[X] = at::empty(shape, options);
            if (task_should_compute_output(BLOCK)) out[BLOCK] = same && out[X].defined() ? out[X] : at::empty(shape, options);
            if (a.rows == 0) {
                for (int k = GATE; k < NORM_TENSORS; k++)
                    if (out[k].defined()) out[k].zero_();
            } else {
                if (gh.defined()) gh = gh.detach().contiguous();
                if (gy.defined()) gy = gy.detach().contiguous();
                // (scratch of its own for every call: two captured passes never share it)
                const at::Tensor scratch = bytes(g_norm.backward_bytes(&a), t[X].device());
                auto p = [](const at::Tensor& u) { return u.defined() ? u.data_ptr() : nullptr; };
                check(g_norm.backward(&a, stats.data_ptr<float>(), p(gh), p(gy), p(out[X]), p(out[BLOCK]), p(out[GATE]), p(out[WEIGHT]), p(out[BIAS]),
                                      p(out[BLOCK_WEIGHT]), p(out[BLOCK_BIAS]), scratch.data_ptr(), (size_t)scratch.numel(), raw_stream(t[X])),
                      "cfh_residual_norm_backward");
            }
        }
        if (differentiable) {                  // a gradient of this gradient would be wrong without a word
            auto error = std::make_shared<torch::autograd::DelayedError>(
                "the gradients of a residual norm are not differentiable", (int64_t)out.size());
            torch::autograd::variable_list given = out;
            for (auto& g : given)
                if (g.defined()) g = g.detach().requires_grad_(true);
            given = (*error)(std::move(given));
            for (size_t k = 0; k < out.size(); k++)
                if (out[k].defined()) out[k] = given[k];
        }
        return out;
    }
};

py::object residual_norm(const at::Tensor& x, const c10::optional<at::Tensor>& block, const c10::optional<at::Tensor>& gate,
                         const c10::optional<at::Tensor>& weight, const c10::optional<at::Tensor>& bias,
                         const c10::optional<at::Tensor>& block_weight, const c10::optional<at::Tensor>& block_bias, int norm, double eps,
                         int block_norm, double block_eps, double residual_scale, double block_scale, bool keep, bool twice) {
    auto given = [](const c10::optional<at::Tensor>& t) { return t ? *t : at::Tensor(); };
    const NormTensors inputs = {x, given(block), given(gate), given(weight), given(bias), given(block_weight), given(block_bias)};
    const NormSpec s{norm, block_norm, (float)eps, (float)block_eps, (float)residual_scale, (float)block_scale, keep, twice};
    check_norm(inputs, s);
    TORCH_CHECK(!(watchers() & WATCHED), "a residual norm is one call of the library: it cannot be traced or transformed");
    bool train = false;
    if (at::GradMode::is_enabled())
        for (const auto& t : inputs) train = train || (t.defined() && t.requires_grad());
    c10::DeviceGuard guard(x.device());
    NormTensors t = inputs;
    at::Tensor h, y, stats;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const cfh_residual_norm a = norm_args(t, s);
        if (keep) h = at::empty(x.sizes(), x.options());
        if (norm) y = at::empty(x.sizes(), x.options());
        if (train) stats = at::empty({a.rows, 4}, x.options().dtype(at::kFloat));
        check(g_norm.forward(&a, keep ? h.data_ptr() : nullptr, norm ? y.data_ptr() : nullptr, train ? stats.data_ptr<float>() : nullptr, raw_stream(x)),
              "cfh_residual_norm_forward");
    }
    if (train) {
        auto node = std::shared_ptr<ResidualNormBackward>(new ResidualNormBackward(), torch::autograd::deleteNode);
        node->spec = s;
        node->shape = x.sizes().vec();
        for (int k : {WEIGHT, BIAS})
            if (inputs[k].defined()) node->weight_type = inputs[k].scalar_type();
        node->stats = std::move(stats);
        torch::autograd::edge_list edges;
        for (const auto& u : inputs)
            edges.push_back(u.defined() && u.requires_grad() ? torch::autograd::impl::gradient_edge(u) : torch::autograd::Edge());
        node->set_next_edges(std::move(edges));
        if (keep) torch::autograd::set_history(h, node);
        if (norm) torch::autograd::set_history(y, node);
        // In float32 h is what the norm saw: where it is there anyway, and nothing else needs the block's output, it is kept instead of x
        // and block.  16 bits hold it rounded: the backward pass puts it together again.
        node->joined = keep && x.scalar_type() == at::kFloat && !inputs[GATE].defined() && !block_norm;
        for (int k = 0; k < NORM_TENSORS; k++) {
            if (!inputs[k].defined() || (k == BLOCK && node->joined)) continue;
            if (k == X && node->joined) node->saved[k] = torch::autograd::SavedVariable(h, true);
            else node->saved[k] = torch::autograd::SavedVariable(inputs[k], false);
        }
    }
    if (!norm) return py::cast(h);
    if (!keep) return py::cast(y);
    return py::make_tuple(py::cast(h), py::cast(y));
}

// ---- attention between sequences ---------------------------------------------------------------------------------------------------
struct AttentionLibrary {
    size_t (*forward_bytes)(const cfh_attention*) = nullptr;
    int (*forward)(const cfh_attention*, void*, void*, float*, void*, size_t, void*) = nullptr;
    size_t (*backward_bytes)(const cfh_attention*) = nullptr;
    int (*backward)(const cfh_attention*, const void*, const void*, const float*, const void*, const int64_t*, void*, void*, void*, void*, void*, size_t, void*) = nullptr;
} g_attention;

enum { QUERY, KEY, VALUE, TABLE, ATTENTION_LEAVES, BUCKETS = ATTENTION_LEAVES, QUERY_STARTS, KEY_STARTS, QUERY_SIZES, KEY_SIZES, KEY_MASK, ATTENTION_TENSORS };
const char* const ATTENTION_NAMES[ATTENTION_TENSORS] = {"query", "key", "value", "table", "buckets", "query_starts", "key_starts", "query_sizes",
                                                       "key_sizes", "key_mask"};
using AttentionTensors = std::array<at::Tensor, ATTENTION_TENSORS>;

struct AttentionSpec {
    double scale;                              // 0: one over the root of the channels
    bool causal, last;
};

void check_attention(const AttentionTensors& t, const AttentionSpec& s) {
    const at::Tensor &q = t[QUERY], &k = t[KEY], &v = t[VALUE];
    for (int n = 0; n < ATTENTION_TENSORS; n++)
        TORCH_CHECK_TYPE(!wrapped(t[n]), ATTENTION_NAMES[n], " is a tensor of a class with operations of its own: one in memory is needed");
    for (const auto& u : t) {
        TORCH_CHECK(!u.defined() || u.is_cuda(), "crystalframer_amd operators run on a HIP device only (tensor on ", u.device(),
                    "); there is no CPU path");
        TORCH_CHECK(!u.defined() || u.layout() == at::kStrided, "a tensor of layout ", u.layout(), ": strided ones are needed");
    }
    TORCH_CHECK_TYPE(element_type(q.scalar_type()) >= 0, "query of ", q.scalar_type(), ": float32, bfloat16 or float16");
    TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "query of ", q.scalar_type(), ", key of ",
                     k.scalar_type(), ", value of ", v.scalar_type(), ": they must have one type");
    TORCH_CHECK_VALUE(q.dim() == 3 || q.dim() == 4, "query of shape ", q.sizes(), ": (rows, heads, channels) of packed sequences, or (batch, positions, heads, channels)");
    const bool packed = q.dim() == 3;
    TORCH_CHECK_VALUE(k.dim() == q.dim() && k.sizes() == v.sizes(), "query of shape ", q.sizes(), ", key of shape ", k.sizes(), ", value of shape ", v.sizes());
    const int64_t H = q.size(-2), G = k.size(-2), D = q.size(-1);
    TORCH_CHECK_VALUE(k.size(-1) == D && D >= 1 && D <= CFH_ATTENTION_MAX_DIM, "heads of ", D, " and ", k.size(-1), " channels: as many, from 1 to ", CFH_ATTENTION_MAX_DIM);
    TORCH_CHECK_VALUE(H >= 1 && G >= 1 && H % G == 0, H, " heads of the query, ", G, " of key and value: each of these has to serve as many of those");
    for (const auto& u : t) TORCH_CHECK(!u.defined() || u.device() == q.device(), "the tensors are on different devices");
    int64_t batch = 0;
    if (packed) {
        TORCH_CHECK_VALUE(t[QUERY_STARTS].defined() && t[KEY_STARTS].defined(), "packed sequences need query_starts and key_starts");
        TORCH_CHECK_VALUE(!t[QUERY_SIZES].defined() && !t[KEY_SIZES].defined(), "query_sizes and key_sizes are of sequences that are not packed");
        for (int n : {QUERY_STARTS, KEY_STARTS})
            TORCH_CHECK_VALUE(t[n].dim() == 1 && t[n].size(0) >= 1 && t[n].size(0) == t[QUERY_STARTS].size(0), ATTENTION_NAMES[n], " of shape ", t[n].sizes(),
                              ": where each sequence begins and, behind them, where the last ends, for queries and keys alike");
        batch = t[QUERY_STARTS].size(0) - 1;
    } else {
        batch = q.size(0);
        TORCH_CHECK_VALUE(k.size(0) == batch, "batches of ", batch, " and ", k.size(0), " sequences");
        TORCH_CHECK_VALUE(!t[QUERY_STARTS].defined() && !t[KEY_STARTS].defined(), "query_starts and key_starts are of packed sequences");
        for (int n : {QUERY_SIZES, KEY_SIZES})
            TORCH_CHECK_VALUE(!t[n].defined() || (t[n].dim() == 1 && t[n].size(0) == batch), ATTENTION_NAMES[n], " of shape ", t[n].sizes(), " for ", batch, " sequences");
    }
    TORCH_CHECK_VALUE(batch <= 0x7fffffffLL, batch, " sequences");
    for (int n : {QUERY_STARTS, KEY_STARTS, QUERY_SIZES, KEY_SIZES})
        TORCH_CHECK_TYPE(!t[n].defined() || t[n].scalar_type() == at::kLong, ATTENTION_NAMES[n], " of ", t[n].scalar_type(), ": int64");
    if (t[KEY_MASK].defined()) {
        TORCH_CHECK_TYPE(t[KEY_MASK].scalar_type() == at::kBool, "key_mask of ", t[KEY_MASK].scalar_type(), ": bool, true for keys that are there");
        TORCH_CHECK_VALUE(t[KEY_MASK].sizes() == k.sizes().slice(0, k.dim() - 2), "key_mask of shape ", t[KEY_MASK].sizes(), " for keys of shape ", k.sizes());
    }
    if (t[TABLE].defined()) {
        const at::Tensor& of = t[BUCKETS];
        TORCH_CHECK_TYPE(t[TABLE].scalar_type() == q.scalar_type() || t[TABLE].scalar_type() == at::kFloat, "table of ", t[TABLE].scalar_type(),
                         ": the type of the query, or float32");
        TORCH_CHECK_VALUE(t[TABLE].dim() == 2 && t[TABLE].size(0) >= 1 && t[TABLE].size(0) <= 65535 && t[TABLE].size(1) == H, "table of shape ",
                          t[TABLE].sizes(), ": (buckets, ", H, " heads)");
        TORCH_CHECK_TYPE(of.scalar_type() == at::kInt, "buckets of ", of.scalar_type(), ": int32");
        TORCH_CHECK_VALUE(of.dim() == 1 && of.size(0) % 2 == 1 && of.size(0) <= 2 * CFH_ATTENTION_MAX_REACH + 1, "buckets of shape ", of.sizes(),
                          ": one for each relative position from -reach to reach, up to ", CFH_ATTENTION_MAX_REACH);
    }
    TORCH_CHECK_VALUE(s.scale == 0.0 || (s.scale <= CFH_ATTENTION_MAX_SCALE && (float)s.scale > 0.0f), "scale ", s.scale, " must be positive, up to ", CFH_ATTENTION_MAX_SCALE);
    TORCH_CHECK_VALUE(s.scale == 0.0 || !t[TABLE].defined() || (s.scale >= 0x1p-64 && s.scale <= 0x1p64), "scale ", s.scale, ": from 2^-64 to 2^64 with a table");
}

// t as the library reads it: rows of neighbouring channels that begin at multiples of 16 bytes and fill them, and lie apart from one
// another (not one row for all positions); others are laid out again.
at::Tensor aligned_rows(const at::Tensor& t) {
    const int64_t size = (int64_t)t.element_size(), D = t.size(-1), n = t.dim();
    uint64_t all = (uint64_t)reinterpret_cast<uintptr_t>(t.data_ptr());
    for (int64_t d = 0; d + 1 < n; d++)
        if (t.size(d) > 1) all |= (uint64_t)(t.stride(d) * size);
    const bool fit = t.size(n - 3) <= 1 || (t.stride(n - 3) >= D && t.stride(n - 3) * size < 1 << 24);
    if (D * size % 16) {      // (at::constant_pad_nd would keep the order of t's dimensions in memory)
        std::vector<int64_t> filled = t.sizes().vec();
        filled.back() += (16 - D * size % 16) / size;
        const at::Tensor y = at::zeros(filled, t.options().memory_format(at::MemoryFormat::Contiguous));
        y.narrow(-1, 0, D).copy_(t);
        return y;
    }
    return (D == 1 || t.stride(-1) == 1) && !(all & 15) && fit ? t : t.clone(at::MemoryFormat::Contiguous);
}
// Strides of (batch, row, head); of a dimension that has one entry, 0.
void strides_of(const at::Tensor& t, int64_t* out) {
    const int64_t n = t.dim();
    for (int64_t d = 0; d < 3; d++) {
        const int64_t at = n - 4 + d;
        out[d] = at < 0 || t.size(at) <= 1 ? 0 : t.stride(at);
    }
}
// The library's arguments; `t` becomes the tensors that they point to.
cfh_attention attention_args(AttentionTensors& t, const AttentionSpec& s) {
    cfh_attention a;
    std::memset(&a, 0, sizeof(a));
    const int64_t channels = t[QUERY].size(-1);
    for (int n : {QUERY, KEY, VALUE}) t[n] = aligned_rows(t[n]);
    for (int n = TABLE; n < ATTENTION_TENSORS; n++)
        if (t[n].defined()) t[n] = t[n].contiguous();
    const at::Tensor &q = t[QUERY], &k = t[KEY];
    a.struct_size = (int32_t)sizeof(a);
    a.dtype = a.table_dtype = element_type(q.scalar_type());
    a.packed = q.dim() == 3;
    a.causal = s.causal; a.queries_last = s.last;
    a.batch = (int32_t)(a.packed ? t[QUERY_STARTS].size(0) - 1 : q.size(0));
    a.heads = (int32_t)q.size(-2); a.kv_heads = (int32_t)k.size(-2); a.dim = (int32_t)channels;
    a.scale = s.scale == 0.0 ? (float)(1.0 / std::sqrt((double)a.dim)) : (float)s.scale;
    a.query_rows = q.size(-3); a.key_rows = k.size(-3);
    strides_of(q, a.q_stride);
    strides_of(k, a.k_stride);
    strides_of(t[VALUE], a.v_stride);
    auto p = [&](int n) { return t[n].defined() ? t[n].data_ptr() : nullptr; };
    a.q = p(QUERY); a.k = p(KEY); a.v = p(VALUE);
    a.key_mask = static_cast<const uint8_t*>(p(KEY_MASK));
    a.query_starts = static_cast<const int64_t*>(p(QUERY_STARTS)); a.key_starts = static_cast<const int64_t*>(p(KEY_STARTS));
    a.query_sizes = static_cast<const int64_t*>(p(QUERY_SIZES)); a.key_sizes = static_cast<const int64_t*>(p(KEY_SIZES));
    if (t[TABLE].defined()) {
        a.table = p(TABLE);
        a.table_dtype = element_type(t[TABLE].scalar_type());
        a.buckets = (int32_t)t[TABLE].size(0);
        a.reach = (int32_t)(t[BUCKETS].size(0) / 2);
        a.bucket_of = static_cast<const int32_t*>(p(BUCKETS));
    }
    return a;
}

struct SequenceAttentionBackward : public torch::autograd::Node {
    AttentionSpec spec;
    std::array<torch::autograd::SavedVariable, ATTENTION_TENSORS> saved;
    torch::autograd::SavedVariable out;
    at::Tensor stats, rest;                    // rest: what rounding to 16 bits left of the output
    bool released = false;

    std::string name() const override { return "SequenceAttentionHIPBackward"; }
    void release_variables() override {
        released = true;
        for (auto& s : saved) s.reset_data();
        out.reset_data();
        stats.reset();
        rest.reset();
    }
    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
        TORCH_CHECK(!released, "Trying to backward through an attention a second time: make the first pass with retain_graph=True");
        torch::autograd::variable_list result(ATTENTION_LEAVES);
        if (!grads[0].defined()) return result;
        AttentionTensors t;
        for (int n = 0; n < ATTENTION_TENSORS; n++) {
            t[n] = saved[n].unpack();
            if (t[n].defined()) t[n] = t[n].detach();
        }
        const at::Tensor o = out.unpack(shared_from_this()).detach();
        c10::DeviceGuard guard(o.device());
        check_capture(*this, o.device(), "an attention");
        {
            at::AutoDispatchBelowADInplaceOrView below;
            const std::array<bool, ATTENTION_LEAVES> wanted = {task_should_compute_output(QUERY), task_should_compute_output(KEY),
                                                               task_should_compute_output(VALUE), task_should_compute_output(TABLE)};
            const at::Tensor dq = at::empty(t[QUERY].sizes(), o.options());
            at::Tensor dk, dv, dtable;
            if (wanted[KEY] || wanted[VALUE]) {
                dk = at::empty(t[KEY].sizes(), o.options());
                dv = at::empty(t[KEY].sizes(), o.options());
            }
            if (wanted[TABLE]) dtable = at::empty(t[TABLE].sizes(), t[TABLE].options());
            const at::Tensor go = aligned_rows(grads[0].detach());
            const cfh_attention a = attention_args(t, spec);
            int64_t go_stride[3];
            strides_of(go, go_stride);
            // (scratch of its own for every call: two captured passes never share it)
            const at::Tensor scratch = bytes(g_attention.backward_bytes(&a), o.device());
            auto p = [](const at::Tensor& u) { return u.defined() ? u.data_ptr() : nullptr; };
            check(g_attention.backward(&a, p(o), p(rest), stats.data_ptr<float>(), p(go), go_stride, p(dq), p(dk), p(dv), p(dtable), scratch.data_ptr(),
                                       (size_t)scratch.numel(), raw_stream(o)),
                  "cfh_attention_backward");
            if (wanted[QUERY]) result[QUERY] = dq;
            if (wanted[KEY]) result[KEY] = dk;
            if (wanted[VALUE]) result[VALUE] = dv;
            if (wanted[TABLE]) result[TABLE] = dtable;
        }
        if (at::GradMode::is_enabled()) {      // a gradient of this gradient would be wrong without a word
            auto error = std::make_shared<torch::autograd::DelayedError>("the gradients of an attention are not differentiable", (int64_t)result.size());
            torch::autograd::variable_list given = result;
            for (auto& g : given)
                if (g.defined()) g = g.detach().requires_grad_(true);
            given = (*error)(std::move(given));
            for (size_t n = 0; n < result.size(); n++)
                if (result[n].defined()) result[n] = given[n];
        }
        return result;
    }
};

at::Tensor sequence_attention(const at::Tensor& query, const at::Tensor& key, const at::Tensor& value, const c10::optional<at::Tensor>& table,
                              const c10::optional<at::Tensor>& buckets, const c10::optional<at::Tensor>& query_starts,
                              const c10::optional<at::Tensor>& key_starts, const c10::optional<at::Tensor>& query_sizes,
                              const c10::optional<at::Tensor>& key_sizes, const c10::optional<at::Tensor>& key_mask, double scale, bool causal, bool last) {
    auto given = [](const c10::optional<at::Tensor>& t) { return t ? *t : at::Tensor(); };
    const AttentionTensors inputs = {query, key, value, given(table), given(buckets), given(query_starts), given(key_starts), given(query_sizes),
                                     given(key_sizes), given(key_mask)};
    const AttentionSpec s{scale, causal, last};
    check_attention(inputs, s);
    TORCH_CHECK(!(watchers() & WATCHED), "an attention is one call of the library: it cannot be traced or transformed");
    bool train = false;
    if (at::GradMode::is_enabled())
        for (int n = 0; n < ATTENTION_LEAVES; n++) train = train || (inputs[n].defined() && inputs[n].requires_grad());
    c10::DeviceGuard guard(query.device());
    AttentionTensors t = inputs;
    at::Tensor out, stats, rest;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const cfh_attention a = attention_args(t, s);
        out = at::empty(query.sizes(), query.options().memory_format(at::MemoryFormat::Contiguous));
        if (train) stats = at::empty({query.numel() / query.size(-1), 2}, query.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous));
        if (train && query.scalar_type() != at::kFloat) rest = at::empty_like(out);
        const size_t need = g_attention.forward_bytes(&a);
        const at::Tensor scratch = need ? bytes(need, query.device()) : at::Tensor();
        check(g_attention.forward(&a, out.data_ptr(), rest.defined() ? rest.data_ptr() : nullptr, train ? stats.data_ptr<float>() : nullptr, need ? scratch.data_ptr() : nullptr, need, raw_stream(query)),
              "cfh_attention_forward");
    }
    if (train) {
        auto node = std::shared_ptr<SequenceAttentionBackward>(new SequenceAttentionBackward(), torch::autograd::deleteNode);
        node->spec = s;
        node->stats = std::move(stats);
        node->rest = std::move(rest);
        torch::autograd::edge_list edges;
        for (int n = 0; n < ATTENTION_LEAVES; n++)
            edges.push_back(inputs[n].defined() && inputs[n].requires_grad() ? torch::autograd::impl::gradient_edge(inputs[n]) : torch::autograd::Edge());
        node->set_next_edges(std::move(edges));
        torch::autograd::set_history(out, node);
        for (int n = 0; n < ATTENTION_TENSORS; n++)
            if (inputs[n].defined()) node->saved[n] = torch::autograd::SavedVariable(inputs[n], false);
        node->out = torch::autograd::SavedVariable(out, true);
    }
    return out;
}

// Addresses of an optimizer's launch: fills the jobs of the parameters that have a gradient.  Returns how many, or -1 when a
// gradient is one that the Python side has to look at (not contiguous, sparse, another type) or does not fit the moments:
// the kernel goes over as many words of parameter, gradient and moments as the parameter had when these were made.
struct Updates {
    std::vector<at::Tensor> params;
    std::vector<int64_t> offset;               // of a parameter's moments, in floats (-1: none)
    std::vector<int64_t> numel;                // of a parameter's moments
    c10::Device device;                        // of the moments
    Updates(std::vector<at::Tensor> p, std::vector<int64_t> o, std::vector<int64_t> n, const at::Tensor& moments)
        : params(std::move(p)), offset(std::move(o)), numel(std::move(n)), device(moments.device()) {}
    // Whether these are the tensors of the list, in its order.
    bool of(py::object list) const {
        py::object seq = py::reinterpret_steal<py::object>(PySequence_Fast(list.ptr(), "the parameters of a group"));
        if (!seq) throw py::error_already_set();
        if (PySequence_Fast_GET_SIZE(seq.ptr()) != (Py_ssize_t)params.size()) return false;
        PyObject** const items = PySequence_Fast_ITEMS(seq.ptr());
        for (size_t i = 0; i < params.size(); i++)
            if (!THPVariable_Check(items[i]) || THPVariable_Unpack(items[i]).unsafeGetTensorImpl() != params[i].unsafeGetTensorImpl())
                return false;
        return true;
    }
    int64_t fill(uintptr_t jobs, uintptr_t m, uintptr_t v) const {
        cfh_adamw_job* const J = reinterpret_cast<cfh_adamw_job*>(jobs);
        int64_t n = 0;
        for (size_t i = 0; i < params.size(); i++) {
            const at::Tensor& p = params[i];
            const at::Tensor& g = p.grad();
            if (!g.defined()) continue;
            if (offset[i] < 0 || g.layout() != at::kStrided || g.scalar_type() != at::kFloat || !g.is_contiguous() ||
                !p.is_contiguous() || p.scalar_type() != at::kFloat || p.numel() != numel[i] || g.numel() != numel[i] ||
                p.device() != device || g.device() != device)
                return -1;
            cfh_adamw_job& j = J[n++];
            j.param = reinterpret_cast<float*>(p.data_ptr());
            j.grad = reinterpret_cast<const float*>(g.data_ptr());
            j.exp_avg = reinterpret_cast<float*>(m) + offset[i];
            j.exp_avg_sq = reinterpret_cast<float*>(v) + offset[i];
            j.n = p.numel();
        }
        return n;
    }
    // The same for cfh_adamw_step_moments, whose tensors have types of their own and whose moments are given by their place.
    int64_t fill_params(uintptr_t jobs) const {
        cfh_param_job* const J = reinterpret_cast<cfh_param_job*>(jobs);
        int64_t n = 0;
        for (size_t i = 0; i < params.size(); i++) {
            const at::Tensor& p = params[i];
            const at::Tensor& g = p.grad();
            if (!g.defined()) continue;
            const at::ScalarType t = p.scalar_type();
            if (offset[i] < 0 || g.layout() != at::kStrided || g.scalar_type() != t || !g.is_contiguous() || !p.is_contiguous() ||
                p.numel() != numel[i] || g.numel() != numel[i] || p.device() != device || g.device() != device ||
                !(t == at::kFloat || t == at::kBFloat16 || t == at::kHalf))
                return -1;
            cfh_param_job& j = J[n++];
            j.param = p.data_ptr();
            j.grad = g.data_ptr();
            j.n = numel[i];
            j.first = offset[i];
            j.dtype = t == at::kFloat ? CFH_FLOAT32 : t == at::kBFloat16 ? CFH_BFLOAT16 : CFH_FLOAT16;
            j.reserved0 = 0;
        }
        return n;
    }
    // every .grad becomes None
    void drop() {
        for (auto& p : params) p.mutable_grad().reset();
    }
};

}  // namespace

PYBIND11_MODULE(_host, mod) {
    mod.def("bind", [](uintptr_t sizes, uintptr_t forward, uintptr_t backward, uintptr_t last_error) {
        g_lib.sizes = reinterpret_cast<decltype(g_lib.sizes)>(sizes);
        g_lib.forward = reinterpret_cast<decltype(g_lib.forward)>(forward);
        g_lib.backward = reinterpret_cast<decltype(g_lib.backward)>(backward);
        g_lib.last_error = reinterpret_cast<decltype(g_lib.last_error)>(last_error);
    });
    mod.def("bind_norm", [](uintptr_t forward, uintptr_t backward_bytes, uintptr_t backward) {
        g_norm.forward = reinterpret_cast<decltype(g_norm.forward)>(forward);
        g_norm.backward_bytes = reinterpret_cast<decltype(g_norm.backward_bytes)>(backward_bytes);
        g_norm.backward = reinterpret_cast<decltype(g_norm.backward)>(backward);
    });
    mod.def("residual_norm", &residual_norm);
    mod.def("bind_attention", [](uintptr_t forward_bytes, uintptr_t forward, uintptr_t backward_bytes, uintptr_t backward) {
        g_attention.forward_bytes = reinterpret_cast<decltype(g_attention.forward_bytes)>(forward_bytes);
        g_attention.forward = reinterpret_cast<decltype(g_attention.forward)>(forward);
        g_attention.backward_bytes = reinterpret_cast<decltype(g_attention.backward_bytes)>(backward_bytes);
        g_attention.backward = reinterpret_cast<decltype(g_attention.backward)>(backward);
    });
    mod.def("sequence_attention", &sequence_attention);
    mod.def("gate_rows", &gate_rows);
    mod.attr("abi") = CFH_ABI_VERSION;
    mod.attr("WATCHED") = (int)WATCHED;
    mod.attr("FUNCTION_MODE") = (int)FUNCTION_MODE;
    mod.attr("SAVED_TENSOR_HOOKS") = (int)SAVED_TENSOR_HOOKS;
    mod.def("watchers", &watchers);
    py::class_<Plan>(mod, "Plan")
        .def(py::init<py::list, py::list, std::vector<at::Tensor>, std::vector<at::Tensor>, int64_t, int64_t, int64_t, int64_t>())
        .def("current", &Plan::current)
        .def("accepts", &Plan::accepts)
        .def("wanted", &Plan::wanted)
        .def("forward", &Plan::forward);
    py::class_<Updates>(mod, "Updates")
        .def(py::init<std::vector<at::Tensor>, std::vector<int64_t>, std::vector<int64_t>, const at::Tensor&>())
        .def("of", &Updates::of)
        .def("fill", &Updates::fill)
        .def("fill_params", &Updates::fill_params)
        .def("drop", &Updates::drop);
}
