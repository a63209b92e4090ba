// Host work that Python is too slow for.  A CPython extension, no kernels in it: the library that holds those stays a plain C ABI, whose
// functions are handed in by address.
//
// Tables of the multi-tensor entry points: reads lists of torch tensors, checks them and writes the descriptors of include/semseg_hip.h.
// An optimiser step over a few hundred tensors asks each of them for its address, type, device, size and layout; from Python that
// costs about 2 us a tensor (0.48 ms for the 168 tensors of ResNet50dilated + PPM with 8-bit states, twice the time of the kernels), here
// about 20 ns.
//
// The backward node of the per-row losses (label log probability, policy loss): autograd runs it on a thread of its own, where a Python
// node first has to get the interpreter lock from the thread that waits for it.  Loss and gradient of 2 x 64 x 64 pixels are 14 us of GPU
// time.
#include <Python.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <algorithm>
#include <exception>
#include <vector>

#include "semseg_hip.h"

namespace {

struct Refused {};                      // a Python error has been set

struct Seq {                            // a list or tuple, held
    PyObject* fast;
    explicit Seq(PyObject* o, const char* what) : fast(PySequence_Fast(o, what)) {
        if (!fast) throw Refused();
    }
    ~Seq() { Py_DECREF(fast); }
    Seq(const Seq&) = delete;
    Seq& operator=(const Seq&) = delete;
    Py_ssize_t size() const { return PySequence_Fast_GET_SIZE(fast); }
    PyObject* operator[](Py_ssize_t i) const { return PySequence_Fast_GET_ITEM(fast, i); }
};

[[noreturn]] void refuse(PyObject* type, const char* format, ...) {
    va_list args;
    va_start(args, format);
    PyErr_FormatV(type, format, args);
    va_end(args);
    throw Refused();
}

thread_local bool duals = false;        // whether tensors with a forward-mode tangent exist at all: asked once a call (20 ns a tensor otherwise)

const at::Tensor& tensor(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s: expected a tensor, got %s", what, Py_TYPE(o)->tp_name);
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || t.layout() != at::kStrided) refuse(PyExc_TypeError, "%s: tensors must be strided", what);
    // a result without a tangent would say that the derivative is zero
    if (duals && t._fw_grad(0).defined()) refuse(PyExc_NotImplementedError, "%s: there is no forward-mode derivative", what);
    return t;
}

int type_code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return SEMSEG_TYPE_F32;
        case at::kBFloat16: return SEMSEG_TYPE_BF16;
        case at::kHalf: return SEMSEG_TYPE_F16;
        default: return -1;
    }
}

// elements of two tensors follow each other in memory in the same order; strides of axes of one element say nothing
bool same_order(const at::Tensor& a, const at::Tensor& b) {
    if (a.sizes() != b.sizes()) return false;          // equal strides alone may stand for other elements, or for fewer in memory
    const auto sa = a.strides(), sb = b.strides();
    if (sa == sb) return true;
    for (size_t i = 0; i < sa.size(); ++i)
        if (a.size(i) != 1 && sa[i] != sb[i]) return false;
    return true;
}

void* address(const at::Tensor& t) { return const_cast<void*>(t.const_data_ptr()); }

typedef std::vector<std::pair<uintptr_t, uintptr_t>> Ranges;
// what a call writes: no element twice (blocks of two tensors would race)
void disjoint(Ranges& r, const char* what) {
    std::sort(r.begin(), r.end());
    for (size_t i = 1; i < r.size(); ++i)
        if (r[i].first < r[i - 1].second)
            refuse(PyExc_ValueError, "%s: the same tensor twice among parameters, states, copies and step counts of a call (or overlapping ones)", what);
}
// what it reads: nothing that it writes (`w`, sorted and disjoint) -- another block's results would be read as gradients
void unwritten(const Ranges& w, const void* at, int64_t bytes, const char* what) {
    const uintptr_t begin = (uintptr_t)at, end = begin + (uintptr_t)bytes;
    const auto behind = std::lower_bound(w.begin(), w.end(), std::make_pair(end, (uintptr_t)0));
    if (bytes && behind != w.begin() && std::prev(behind)->second > begin)
        refuse(PyExc_ValueError, "%s: a gradient shares memory with a parameter, state, copy or step count of the call", what);
}
void add(Ranges& r, const void* at, int64_t bytes) {
    if (bytes) r.emplace_back((uintptr_t)at, (uintptr_t)at + (uintptr_t)bytes);
}

// the part that both AdamW tables share; returns false for a tensor without elements
template <class ENTRY>
bool common(ENTRY& e, const char* what, const at::Tensor& p, PyObject* grad, PyObject* step, PyObject* wd, PyObject* copy,
            const at::Device& dev, Ranges& written) {
    const at::Tensor& g = tensor(grad, what);
    const at::Tensor& s = tensor(step, what);
    if (p.scalar_type() != at::kFloat)
        refuse(PyExc_TypeError, "%s: parameters must be float32 (a 16-bit copy goes into `copies`)", what);
    if (type_code(g) < 0) refuse(PyExc_TypeError, "%s: gradients must be float32, bfloat16 or float16", what);
    if (s.scalar_type() != at::kInt || s.numel() != 1) refuse(PyExc_TypeError, "%s: a step count is one int32 on the device", what);
    if (p.device() != dev || g.device() != dev || s.device() != dev)
        refuse(PyExc_ValueError, "%s: all tensors of a call must be on one HIP device", what);
    if (!p.is_non_overlapping_and_dense() || !same_order(p, g))
        refuse(PyExc_RuntimeError, "%s: a parameter of %zd elements and its gradient differ in layout or are not dense", what,
               (Py_ssize_t)p.numel());
    e.copy = nullptr;
    e.copy_type = 0;
    if (copy && copy != Py_None) {
        const at::Tensor& c = tensor(copy, what);
        if (type_code(c) <= SEMSEG_TYPE_F32 || c.device() != dev || !same_order(p, c))
            refuse(PyExc_RuntimeError, "%s: a copy must be bfloat16 or float16 in its parameter's layout on its device", what);
        e.copy = address(c);
        e.copy_type = type_code(c);
    }
    const double decay = PyFloat_AsDouble(wd);
    if (decay == -1.0 && PyErr_Occurred()) throw Refused();
    e.param = address(p);
    e.grad = address(g);
    e.step = (int*)address(s);
    e.numel = p.numel();
    e.weight_decay = (float)decay;
    e.grad_type = type_code(g);
    if (e.numel == 0) return false;
    add(written, e.param, 4 * e.numel);
    add(written, e.copy, e.copy ? 2 * e.numel : 0);
    add(written, e.step, 4);
    return true;
}

template <class ENTRY, class FILL>
PyObject* adam_table(PyObject* const* args, Py_ssize_t n_states, FILL fill) {
    const char* what = PyUnicode_AsUTF8(args[0]);
    if (!what) throw Refused();
    const char* lists = "expected a list of tensors";
    Seq params(args[1], lists), grads(args[2], lists), steps(args[3], lists), wds(args[4], "expected a list of numbers");
    const bool copying = args[5] != Py_None;
    Seq copies(copying ? args[5] : args[1], lists);
    const Py_ssize_t n = params.size();
    bool even = grads.size() == n && steps.size() == n && wds.size() == n && copies.size() == n;
    std::vector<std::unique_ptr<Seq>> states;
    for (Py_ssize_t k = 0; k < n_states; ++k) {
        states.emplace_back(new Seq(args[6 + k], lists));
        even = even && states.back()->size() == n;
    }
    if (!even) refuse(PyExc_ValueError, "%s: the lists differ in length", what);
    std::vector<ENTRY> table;
    table.reserve(n);
    Ranges written;
    written.reserve(7 * n);
    for (Py_ssize_t i = 0; i < n; ++i) {
        const at::Tensor& p = tensor(params[i], what);
        const at::Device dev = THPVariable_Unpack(params[0]).device();
        ENTRY e{};
        const bool live = common(e, what, p, grads[i], steps[i], wds[i], copying ? copies[i] : nullptr, dev, written);
        fill(e, what, p, dev, states, i, written);
        if (live) table.push_back(e);
    }
    disjoint(written, what);
    for (const ENTRY& e : table) unwritten(written, e.grad, e.numel * (e.grad_type == SEMSEG_TYPE_F32 ? 4 : 2), what);
    PyObject* bytes = PyBytes_FromStringAndSize((const char*)table.data(), (Py_ssize_t)(table.size() * sizeof(ENTRY)));
    if (!bytes) throw Refused();
    return Py_BuildValue("Nn", bytes, (Py_ssize_t)table.size());
}

void fill32(semseg_adamw_tensor& e, const char* what, const at::Tensor& p, const at::Device& dev,
            const std::vector<std::unique_ptr<Seq>>& states, Py_ssize_t i, Ranges& written) {
    const at::Tensor& m = tensor((*states[0])[i], what);
    const at::Tensor& v = tensor((*states[1])[i], what);
    if (m.scalar_type() != at::kFloat || v.scalar_type() != at::kFloat || m.device() != dev || v.device() != dev || !same_order(p, m) ||
        !same_order(p, v))
        refuse(PyExc_RuntimeError, "%s: the states of a parameter of %zd elements must be float32 in its layout on its device", what,
               (Py_ssize_t)p.numel());
    e.exp_avg = address(m);
    e.exp_avg_sq = address(v);
    add(written, e.exp_avg, 4 * p.numel());
    add(written, e.exp_avg_sq, 4 * p.numel());
}

void fill8(semseg_adamw8_tensor& e, const char* what, const at::Tensor& p, const at::Device& dev,
           const std::vector<std::unique_ptr<Seq>>& states, Py_ssize_t i, Ranges& written) {
    Seq state((*states[0])[i], "expected an AdamW8State");
    const int64_t n = p.numel(), blocks = (n + 255) / 256;
    bool ok = state.size() == 4;
    void* at_[4] = {};
    for (int k = 0; ok && k < 4; ++k) {
        const at::Tensor& t = tensor(state[k], what);
        const bool codes = k % 2 == 0;
        const auto type = t.scalar_type();
        ok = (codes ? type == at::kByte || type == at::kFloat8_e4m3fn : type == at::kFloat) && t.numel() == (codes ? n : blocks) &&
             t.is_contiguous() && t.device() == dev;
        at_[k] = address(t);
    }
    if (!ok)
        refuse(PyExc_RuntimeError, "%s: the state of a parameter of %zd elements must be as many codes and %zd float32 scales, twice, on its "
               "device (adamw8_state)", what, (Py_ssize_t)n, (Py_ssize_t)blocks);
    e.m_codes = at_[0];
    e.m_scales = at_[1];
    e.r_codes = at_[2];
    e.r_scales = at_[3];
    add(written, e.m_codes, n);
    add(written, e.r_codes, n);
    add(written, e.m_scales, 4 * blocks);
    add(written, e.r_scales, 4 * blocks);
}

template <class F>
PyObject* guarded(F f) {
    try {
        duals = torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr;
        return f();
    } catch (const Refused&) {
        return nullptr;
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// (what, params, grads, steps, weight_decays, copies or None, exp_avgs, exp_avg_sqs) -> (table, entries)
PyObject* adamw_table(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 8) return PyErr_Format(PyExc_TypeError, "adamw_table: 8 arguments");
    return guarded([&] { return adam_table<semseg_adamw_tensor>(args, 2, fill32); });
}
// (what, params, grads, steps, weight_decays, copies or None, states) -> (table, entries)
PyObject* adamw8_table(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 7) return PyErr_Format(PyExc_TypeError, "adamw8_table: 7 arguments");
    return guarded([&] { return adam_table<semseg_adamw8_tensor>(args, 1, fill8); });
}
// (grads,) -> (table, entries)
PyObject* grad_table(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 1) return PyErr_Format(PyExc_TypeError, "grad_table: 1 argument");
    return guarded([&]() -> PyObject* {
        const char* what = "grad_norm";
        Seq grads(args[0], "expected a list of tensors");
        std::vector<semseg_grad_tensor> table;
        table.reserve(grads.size());
        for (Py_ssize_t i = 0; i < grads.size(); ++i) {
            const at::Tensor& g = tensor(grads[i], what);
            if (type_code(g) < 0) refuse(PyExc_TypeError, "%s: gradients must be float32, bfloat16 or float16", what);
            if (g.device() != THPVariable_Unpack(grads[0]).device()) refuse(PyExc_ValueError, "%s: all gradients must be on one HIP device", what);
            if (!g.is_non_overlapping_and_dense()) refuse(PyExc_RuntimeError, "%s: a gradient of %zd elements is not dense", what, (Py_ssize_t)g.numel());
            semseg_grad_tensor e{};
            e.grad = address(g);
            e.numel = g.numel();
            e.grad_type = type_code(g);
            if (e.numel) table.push_back(e);
        }
        PyObject* bytes = PyBytes_FromStringAndSize((const char*)table.data(), (Py_ssize_t)(table.size() * sizeof(table[0])));
        if (!bytes) throw Refused();
        return Py_BuildValue("Nn", bytes, (Py_ssize_t)table.size());
    });
}

// ---------------------------------------------------------------- backward of the per-row losses -------------------------------
typedef int (*LogpBackward)(const void*, int, int64_t, const int64_t*, int64_t, const float*, const float*, const float*, const float*, int64_t,
                            int, void*, void*);
typedef int (*ScaleBy)(float*, const float*, int64_t, const float*, void*);

void* stream_of(const at::Tensor& t) {
    return t.is_cuda() ? (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream() : nullptr;
}
// number of the recording (stream capture) that calls on this tensor go into now, 0 for none
unsigned long long recording_of(const at::Tensor& t) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (!t.is_cuda()) return 0;
    if (hipStreamGetCaptureInfo((hipStream_t)stream_of(t), &status, &id) != hipSuccess) {
        (void)hipGetLastError();                      // the default stream beside another one's capture: nothing is recorded on it
        return 0;
    }
    return status == hipStreamCaptureStatusActive ? id : 0;
}
void check(int rc, const char* what) {
    TORCH_CHECK(rc == 0, what, " failed with code ", rc, rc >= 900 && rc <= 908 ? " (stream capture)" : "");
}

// d logits of label_log_prob (kept: {maximum, log sum} per row) and of policy_loss (kept: scratch, the same, gradient per row, 1 / rows
// that count; `written`: the gradient for an upstream gradient of 1, where the forward pass has written it).
// `written` is scaled in place and handed out where the forward pass runs once for every backward pass: both eager, or both in one recording.
// Where the forward pass was recorded apart (its replays write `written` again), the product goes to memory of its own.  A backward pass that is
// recorded while its forward pass was eager is refused: every replay would scale `written` once more, and what is kept for it is the
// eager pass's memory, free for other tensors once the node is gone.
struct RowsBackward : public torch::autograd::Node {
    torch::autograd::SavedVariable z, label, kept;
    at::Tensor written;
    std::vector<int64_t> shape, strides;              // of the logits, and of `z`
    int64_t ld = 0, ignore = 0;
    unsigned long long recording = 0;                 // of the forward pass
    bool loss = false;
    LogpBackward logp_bwd = nullptr;
    ScaleBy scale_by = nullptr;

    std::string name() const override { return loss ? "PolicyLossBackward" : "LabelLogProbBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        z.reset_data();
        label.reset_data();
        kept.reset_data();
        written.reset();
    }
    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
        if (!grads[0].defined()) return {at::Tensor()};
        at::Tensor zt, lab, keep, dz, again;
        {
            std::lock_guard<std::mutex> lock(mutex_);
            zt = z.unpack(shared_from_this());
            lab = label.unpack(shared_from_this());
            keep = kept.unpack(shared_from_this());
            const auto now = recording_of(zt);
            TORCH_CHECK(!now || recording, name(), ": a backward pass cannot be recorded apart from its forward pass: record both");
            if (now == recording) std::swap(dz, written);
            else again = written;
        }
        {
            at::AutoDispatchBelowADInplaceOrView below;
            const c10::DeviceGuard guard(zt.device());
            int64_t pitch = ld;
            if (zt.strides() != strides) {            // saved through hooks (on the CPU, say) that keep values and not layouts
                zt = shape.size() == 2 ? zt.contiguous()
                                       : zt.permute({0, 2, 3, 1}).contiguous().permute({0, 3, 1, 2});
                pitch = shape[1];
            }
            const at::Tensor g = grads[0].to(at::kFloat).contiguous();
            const int64_t P = lab.numel();
            const float* kp = (const float*)keep.const_data_ptr();
            const float* inv = loss && P ? kp + keep.numel() - 1 : nullptr;
            const float* coef = loss ? inv - P : nullptr;
            if (again.defined()) dz = at::empty_strided(again.sizes(), again.strides(), again.options());
            if (dz.defined()) {                       // handed out once: a second eager backward pass computes its own
                const void* from = again.defined() ? again.const_data_ptr() : dz.const_data_ptr();
                check(scale_by((float*)dz.mutable_data_ptr(), (const float*)from, dz.numel(), (const float*)g.const_data_ptr(), stream_of(zt)), "scale_by");
            } else {
                dz = shape.size() == 2 ? at::empty(shape, zt.options())
                                       : at::empty({shape[0], shape[2], shape[3], shape[1]}, zt.options()).permute({0, 3, 1, 2});
                if (P)
                    check(logp_bwd(zt.const_data_ptr(), type_code(zt), pitch, (const int64_t*)lab.const_data_ptr(), ignore,
                                   loss ? coef - 2 * P : kp, loss ? coef : (const float*)g.const_data_ptr(),
                                   loss ? (const float*)g.const_data_ptr() : nullptr, inv, P, (int)shape[1], dz.mutable_data_ptr(),
                                   stream_of(zt)),
                          "label_logp_bwd");
            }
        }
        if (at::GradMode::is_enabled()) {             // create_graph: the result has no gradient of its own
            auto refused = std::make_shared<torch::autograd::DelayedError>(name() + ": the gradient cannot be differentiated again", 1);
            return (*refused)({dz.set_requires_grad(true)});
        }
        return {dz};
    }
};

// Logits that are a leaf keep the node that accumulates their gradient as long as any graph made with them lives, and with it the stream
// of that graph.  A backward pass that is being captured would draw that stream into the capture, which ends the process here: refused
// while there is something to refuse.
void refuse_foreign_leaf(const at::Tensor& z) {
    if (!z.is_cuda() || z.grad_fn()) return;
    const auto held = torch::autograd::impl::try_get_grad_accumulator(z);
    if (!held || c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    const auto of = held->stream();
    if (of && *of != c10::hip::getCurrentHIPStream(z.get_device()).unwrap())
        refuse(PyExc_RuntimeError, "a backward pass of these logits cannot be captured while a graph that was made with them on another stream "
               "is alive: drop the earlier loss, or detach() the logits first");
}

// (out, z, z as rows, label, kept, written or None, pitch, ignore_index, loss, address of label_logp_bwd, address of scale_by): `out`
// becomes differentiable in z
PyObject* attach_rows(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 11) return PyErr_Format(PyExc_TypeError, "attach_rows: 11 arguments");
    return guarded([&]() -> PyObject* {
        const char* what = "attach_rows";
        const at::Tensor& out = tensor(args[0], what);
        const at::Tensor& z = tensor(args[1], what);
        refuse_foreign_leaf(z);
        auto node = std::shared_ptr<RowsBackward>(new RowsBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(z));
        node->shape = z.sizes().vec();
        node->strides = tensor(args[2], what).strides().vec();
        node->z = torch::autograd::SavedVariable(tensor(args[2], what), false);
        node->label = torch::autograd::SavedVariable(tensor(args[3], what), false);
        node->kept = torch::autograd::SavedVariable(tensor(args[4], what), false);
        if (args[5] != Py_None) node->written = tensor(args[5], what);
        node->recording = recording_of(z);
        node->ld = PyLong_AsLongLong(args[6]);
        node->ignore = PyLong_AsLongLong(args[7]);
        node->loss = PyObject_IsTrue(args[8]) == 1;
        node->logp_bwd = (LogpBackward)PyLong_AsVoidPtr(args[9]);
        node->scale_by = (ScaleBy)PyLong_AsVoidPtr(args[10]);
        if (PyErr_Occurred()) throw Refused();
        torch::autograd::set_history(out, node);
        Py_RETURN_NONE;
    });
}

// (what, *tensors or None): refuses tensors that carry a tangent
PyObject* no_tangents(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const char* what = n ? PyUnicode_AsUTF8(args[0]) : "";
        if (!what) throw Refused();
        for (Py_ssize_t i = 1; i < n; ++i)
            if (args[i] != Py_None) tensor(args[i], what);
        Py_RETURN_NONE;
    });
}

PyMethodDef methods[] = {{"no_tangents", (PyCFunction)(void*)no_tangents, METH_FASTCALL, nullptr},
                         {"attach_rows", (PyCFunction)(void*)attach_rows, METH_FASTCALL, nullptr},
                         {"adamw_table", (PyCFunction)(void*)adamw_table, METH_FASTCALL, nullptr},
                         {"adamw8_table", (PyCFunction)(void*)adamw8_table, METH_FASTCALL, nullptr},
                         {"grad_table", (PyCFunction)(void*)grad_table, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
