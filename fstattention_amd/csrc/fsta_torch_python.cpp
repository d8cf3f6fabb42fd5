// The extension module `_fsta_torch`: the entry points of the package as plain C functions for calls that need nothing of
// torch's dispatcher (ordinary tensors on the GPU, no gradient, no mode that wants to see the call).  A call through the
// registered operator costs about 3 us of schema matching and boxing, and the lookup of the packed inputs another 1.5 us in
// Python; a launch of the smallest kernels takes less than that on the GPU.  Every function returns NotImplemented for a
// call it does not want to judge; the caller then takes the ordinary way, which also raises the errors.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <ATen/record_function.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <pybind11/pybind11.h>

#include <algorithm>
#include <cstring>
#include <limits>
#include <vector>

#include "../../include/fsta.h"
#include "fsta_torch.h"

using fsta_torch::fresh;

namespace {

PyObject* g_packed_type = nullptr;      // attention.PackedTreeMask
PyObject* g_packed_table = nullptr;     // attention._PACKED: id of a mask -> (weak reference, key, packed)

PyObject* not_implemented() { Py_RETURN_NOTIMPLEMENTED; }

// An ordinary torch.Tensor object (no subclass) in GPU memory
const at::Tensor* gpu_tensor(PyObject* o) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.defined() && t.is_cuda() && t.layout() == at::kStrided && !t.key_set().has(c10::DispatchKey::Python) &&
                   !t.key_set().has(c10::DispatchKey::FuncTorchGradWrapper) && !t.key_set().has(c10::DispatchKey::FuncTorchBatched) &&
                   !t.is_conj() && !t.is_neg()
               ? &t
               : nullptr;
}

// Nobody stands between the dispatcher and the kernels (dispatch modes, functorch, tracing).  Inference mode only takes
// ADInplaceOrView out of the default set, which looks after views of and writes to arguments: there are none here.
bool plain_dispatch() {
    const auto included = c10::impl::tls_local_dispatch_key_set().included_ | c10::DispatchKeySet(c10::DispatchKey::ADInplaceOrView);
    return included == c10::default_included_set;
}
// .. and nobody has asked to see calls from Python
bool plain_context() { return plain_dispatch() && !at::impl::torch_function_mode_enabled(); }

bool wants_grad(const at::Tensor& t) { return t.requires_grad(); }
// .. a gradient now, or forward-mode derivatives
bool wants_derivative(const at::Tensor& t) { return (c10::GradMode::is_enabled() && wants_grad(t)) || t._fw_grad(0).defined(); }

bool as_int(PyObject* o, int64_t* out) {
    if (!PyLong_Check(o)) return false;
    *out = PyLong_AsLongLong(o);
    if (*out == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}

struct Packed {
    const at::Tensor *bits, *count, *plan;     // plan may be null
    int64_t block_m, max_ancestors, key_shift, key_limit;
    bool has_limit;
};

bool read_packed(PyObject* o, Packed* p) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 7) return false;
    p->bits = gpu_tensor(PyTuple_GET_ITEM(o, 0));
    p->count = gpu_tensor(PyTuple_GET_ITEM(o, 1));
    PyObject* plan = PyTuple_GET_ITEM(o, 4);
    p->plan = plan == Py_None ? nullptr : gpu_tensor(plan);
    PyObject* limit = PyTuple_GET_ITEM(o, 6);
    p->has_limit = limit != Py_None;
    return p->bits && p->count && (plan == Py_None || p->plan) && as_int(PyTuple_GET_ITEM(o, 2), &p->block_m) &&
           as_int(PyTuple_GET_ITEM(o, 3), &p->max_ancestors) && as_int(PyTuple_GET_ITEM(o, 5), &p->key_shift) &&
           (!p->has_limit || as_int(limit, &p->key_limit));
}

// The packed form remembered for the bool tensor `mask`, if it is the one of these three tensors as they are now
// (attention.recall_packed and attention._cache_key, read from C); a borrowed reference or null.
PyObject* recall(PyObject* mask_obj, const at::Tensor& mask, const at::Tensor& a_idx, const at::Tensor& l_idx) {
    if (mask.is_inference() || a_idx.is_inference() || l_idx.is_inference()) return nullptr;
    PyObject* id = PyLong_FromVoidPtr(mask_obj);
    PyObject* entry = id ? PyDict_GetItem(g_packed_table, id) : nullptr;
    Py_XDECREF(id);
    if (!entry || !PyTuple_Check(entry) || PyTuple_GET_SIZE(entry) != 3) return nullptr;
    PyObject* ref = PyTuple_GET_ITEM(entry, 0);
    if (!PyWeakref_Check(ref) || PyWeakref_GET_OBJECT(ref) != mask_obj) return nullptr;
    PyObject* key = PyTuple_GET_ITEM(entry, 1);
    if (!PyTuple_Check(key) || PyTuple_GET_SIZE(key) != 6) return nullptr;
    const int64_t want[5] = {(int64_t)mask._version(), (int64_t)a_idx._version(), (int64_t)l_idx._version(),
                             (int64_t)(uintptr_t)a_idx.data_ptr(), (int64_t)(uintptr_t)l_idx.data_ptr()};
    for (int i = 0; i < 5; ++i) {
        int64_t v;
        if (!as_int(PyTuple_GET_ITEM(key, i), &v) || v != want[i]) return nullptr;
    }
    PyObject* shape = PyTuple_GET_ITEM(key, 5);
    if (!PyTuple_Check(shape) || PyTuple_GET_SIZE(shape) != mask.dim()) return nullptr;
    for (int64_t d = 0; d < mask.dim(); ++d) {
        int64_t v;
        if (!as_int(PyTuple_GET_ITEM(shape, d), &v) || v != mask.size(d)) return nullptr;
    }
    return PyTuple_GET_ITEM(entry, 2);
}

// Profilers and other observers see a call under the name of the registered operator
__attribute__((noinline)) void report(c10::optional<at::RecordFunction>& seen, at::StepCallbacks&& callbacks, const at::Tensor& q,
                                      const at::Tensor& k, const at::Tensor& v, const at::Tensor& a_idx, const Packed& p,
                                      const at::Tensor& l_idx) {
    seen.emplace(std::move(callbacks));
    if (seen->needsInputs()) {
        const c10::IValue inputs[] = {q, k, v, a_idx, *p.bits, *p.count, l_idx};
        seen->before("fsta::attention_fwd", c10::ArrayRef<const c10::IValue>(inputs, 7));
    } else {
        seen->before("fsta::attention_fwd");
    }
}

// attention(q, k, v, ancestor_idx, ancestor_mask, leaf_idx, sm_scale, BLOCK_M, MAX_ANCESTORS, out_dtype, return_lse, flags,
//           k_scale, v_scale): attention.fst_attention with its switches as FSTA_FLAG_* bits
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 14 || !g_packed_table || !plain_context()) return not_implemented();
    const at::Tensor *q = gpu_tensor(args[0]), *k = gpu_tensor(args[1]), *v = gpu_tensor(args[2]);
    const at::Tensor *a_idx = gpu_tensor(args[3]), *l_idx = gpu_tensor(args[5]);
    if (!q || !k || !v || !a_idx || !l_idx) return not_implemented();
    if (c10::GradMode::is_enabled() && (wants_grad(*q) || wants_grad(*k) || wants_grad(*v))) return not_implemented();
    if (q->dim() != 4 || k->dim() != 4 || v->dim() != 4) return not_implemented();
    const int64_t d = q->size(3);
    if (k->size(3) != d || v->size(3) != d || (d != 16 && d != 32 && d != 64 && d != 128)) return not_implemented();
    int64_t block_m, max_anc, flags;
    if (!as_int(args[7], &block_m) || !as_int(args[8], &max_anc) || !as_int(args[11], &flags) || block_m <= 0) return not_implemented();
    const double sm_scale = PyFloat_CheckExact(args[6]) ? PyFloat_AS_DOUBLE(args[6]) : PyFloat_AsDouble(args[6]);
    if (sm_scale == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        return not_implemented();
    }
    const bool return_lse = args[10] == Py_True;
    if (!return_lse && args[10] != Py_False) return not_implemented();
    const int in_code = fsta_torch::dtype_code(q->scalar_type());
    int out_code = in_code;
    if (args[9] != Py_None) {
        if (!THPDtype_Check(args[9])) return not_implemented();
        out_code = fsta_torch::dtype_code(reinterpret_cast<THPDtype*>(args[9])->scalar_type);
    }
    if (in_code < 0 || out_code < 0) return not_implemented();

    Packed p;
    if (Py_TYPE(args[4]) == reinterpret_cast<PyTypeObject*>(g_packed_type)) {
        if (!read_packed(args[4], &p)) return not_implemented();
        if (p.plan && !p.has_limit && p.key_shift != k->size(2) - q->size(2)) return not_implemented();
    } else {
        const at::Tensor* mask = gpu_tensor(args[4]);
        if (!mask || mask->dim() != 3 || a_idx->dim() != 2 || mask->size(0) != a_idx->size(0) || mask->size(1) != block_m ||
            mask->size(2) != max_anc)
            return not_implemented();
        PyObject* packed = recall(args[4], *mask, *a_idx, *l_idx);
        if (!packed || !read_packed(packed, &p) || (p.has_limit && p.key_limit != k->size(2))) return not_implemented();
    }
    if (p.block_m != block_m || p.max_ancestors != max_anc) return not_implemented();
    c10::optional<at::Tensor> k_scale, v_scale;
    for (int i = 0; i < 2; ++i)
        if (args[12 + i] != Py_None) {
            const at::Tensor* s = gpu_tensor(args[12 + i]);
            if (!s) return not_implemented();
            (i ? v_scale : k_scale) = *s;
        }
    try {
        c10::optional<at::RecordFunction> seen;
        if (auto callbacks = at::getStepCallbacksUnlessEmpty(at::RecordScope::FUNCTION))
            report(seen, std::move(*callbacks), *q, *k, *v, *a_idx, p, *l_idx);
        const auto out = fsta_torch::attention_fwd(*q, *k, *v, *a_idx, *p.bits, *p.count, *l_idx,
                                                   p.plan ? c10::optional<at::Tensor>(*p.plan) : c10::nullopt, p.key_shift, sm_scale,
                                                   block_m, max_anc, out_code, return_lse, flags, k_scale, v_scale);
        PyObject* o = THPVariable_Wrap(std::get<0>(out));
        if (!o || !return_lse) return o;
        PyObject* lse = THPVariable_Wrap(std::get<1>(out));
        PyObject* both = lse ? PyTuple_Pack(2, o, lse) : nullptr;
        Py_DECREF(o);
        Py_XDECREF(lse);
        return both;
    } catch (const std::exception&) {
        return not_implemented();      // (the ordinary way meets the same condition and raises it)
    }
}

// ---- front-end of a decoding step (integer work; outputs are new tensors, arguments are checked in precompute.py) -------
// A return code of the library other than FSTA_OK comes back as a Python int.

const at::Tensor& tensor_arg(PyObject* o) {
    TORCH_CHECK_TYPE(THPVariable_Check(o), "expected a torch.Tensor");
    return THPVariable_Unpack(o);
}

int64_t int_arg(PyObject* o) {
    int64_t v;
    TORCH_CHECK_TYPE(as_int(o, &v), "expected an int");
    return v;
}

struct OnStream {      // the tensors' device and torch's current stream on it
    explicit OnStream(const at::Tensor& t)
        : guard(t.device()), stream(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream()) {}
    const c10::hip::HIPGuardMasqueradingAsCUDA guard;
    const hipStream_t stream;
};

// The status word of a call: the caller's or a zeroed one
at::Tensor status_word(PyObject* given, const at::Tensor& like) {
    return given != Py_None ? tensor_arg(given) : at::zeros({1}, like.options().dtype(at::kInt));
}

template <class... T> PyObject* as_tuple(const T&... tensors) {      // undefined tensors become None
    PyObject* tuple = PyTuple_New(sizeof...(T));
    if (!tuple) return nullptr;
    Py_ssize_t i = 0;
    auto put = [&](const at::Tensor& t) {
        PyObject* o = t.defined() ? THPVariable_Wrap(t) : (Py_INCREF(Py_None), Py_None);
        PyTuple_SET_ITEM(tuple, i++, o);
        return o != nullptr;
    };
    if ((put(tensors) && ...)) return tuple;
    Py_DECREF(tuple);
    return nullptr;
}

// Watches the words of fsta_precompute_from_parents_flags until all of them are set (a wait for the stream costs 10 us more
// than the kernel takes).  Asks the runtime now and then, so that a launch that failed ends the wait with its error.
long watch_flags(const volatile int32_t* words, int64_t n, hipStream_t stream) {
    long found = 0;
    int spins = 0;
    bool drained = false;
    for (int64_t j = 0; j < n;) {
        if (const int32_t word = words[j]) {
            found |= word >> 1;
            ++j;
            continue;
        }
        TORCH_CHECK(!drained, "kernel_inputs_from_parents_gpu: the kernel ended without reporting");
        if (++spins % 4096 == 0) {
            const hipError_t err = hipStreamQuery(stream);
            TORCH_CHECK(err == hipSuccess || err == hipErrorNotReady, "kernel_inputs_from_parents_gpu: ", hipGetErrorString(err));
            drained = err == hipSuccess;      // (the word is looked at once more)
        }
        __builtin_ia32_pause();
    }
    return found;
}

template <class T> T* data_or_null(const at::Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }

// dfs_order(parent, light_first, read_status, status or None) -> (perm, rank, status)
PyObject* dfs_order(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n_args == 4, "dfs_order takes 4 arguments");
    const at::Tensor parent = tensor_arg(args[0]).contiguous();
    const OnStream on(parent);
    const int64_t n = parent.size(0);
    at::Tensor perm = fresh({n}, at::kLong, parent), rank = fresh({n}, at::kLong, parent);
    // (a status word that nobody reads is one int more of workspace)
    const int64_t ints = (int64_t)FSTA_DFS_ORDER_WORKSPACE_INTS(n);
    at::Tensor work = fresh({ints + 1}, at::kInt, parent), status;
    if (args[3] != Py_None || args[2] == Py_True) status = status_word(args[3], parent);
    uint32_t* word = status.defined() ? static_cast<uint32_t*>(status.data_ptr()) : reinterpret_cast<uint32_t*>(work.data_ptr<int32_t>() + ints);
    const int rc = fsta_dfs_order(parent.data_ptr<int64_t>(), n, args[1] == Py_True, perm.data_ptr<int64_t>(), rank.data_ptr<int64_t>(),
                                  work.data_ptr<int32_t>(), word, on.stream);
    return rc != FSTA_OK ? PyLong_FromLong(rc) : as_tuple(perm, rank, status);
    END_HANDLE_TH_ERRORS
}

// renumber_parents(parent, rank) -> new_parent
PyObject* renumber_parents(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n_args == 2, "renumber_parents takes 2 arguments");
    const at::Tensor parent = tensor_arg(args[0]).contiguous(), rank = tensor_arg(args[1]).contiguous();
    const OnStream on(parent);
    at::Tensor out = fresh(parent.sizes(), at::kLong, parent);
    const int rc = fsta_renumber_parents(parent.data_ptr<int64_t>(), rank.data_ptr<int64_t>(), parent.size(0), out.data_ptr<int64_t>(),
                                         on.stream);
    return rc != FSTA_OK ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// inputs_from_parents(parent, block_m, max_ancestors, width, check, want_bool_mask, want_lineage, status or None)
//   -> (ancestor_idx, ancestor_mask, leaf_idx, mask_bits, anc_count, plan, lineage, level_lookup, status), bits
// `check` (then no status word is used or returned): waits until every block has reported, bits are the FSTA_PRE_* conditions;
// else 0
PyObject* inputs_from_parents(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n_args == 8, "inputs_from_parents takes 8 arguments");
    const at::Tensor parent = tensor_arg(args[0]).contiguous();
    const int64_t n = parent.size(0), block_m = int_arg(args[1]), max_anc = int_arg(args[2]), width = int_arg(args[3]);
    const bool check = args[4] == Py_True, want_mask = args[5] == Py_True, want_lineage = args[6] == Py_True;
    TORCH_CHECK_VALUE(block_m > 0 && block_m <= INT32_MAX && max_anc > 0 && max_anc <= INT32_MAX && width > 0,
                      "block_m, max_ancestors and width must be positive");
    const OnStream on(parent);
    if (check) {      // (before anything is recorded: a replay would report into memory that has gone to others)
        hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
        TORCH_CHECK(hipStreamIsCapturing(on.stream, &capture) == hipSuccess && capture == hipStreamCaptureStatusNone,
                    "kernel_inputs_from_parents_gpu: check=True waits for the GPU, which a stream that is being captured does not");
    }
    const int64_t nb = (n + block_m - 1) / block_m;
    at::Tensor a_idx = fresh({nb, max_anc}, at::kLong, parent), l_idx = fresh({nb, block_m}, at::kLong, parent), a_mask, lineage, level, plan;
    if (want_mask) a_mask = fresh({nb, block_m, max_anc}, at::kBool, parent);
    at::Tensor bits = fresh({nb, (int64_t)fsta_mask_words((int32_t)max_anc), block_m}, at::kInt, parent), count = fresh({nb}, at::kInt, parent);
    const size_t plan_bytes = fsta_block_plan_bytes((int32_t)nb, (int32_t)block_m, (int32_t)max_anc);
    if (plan_bytes) plan = fresh({(int64_t)(plan_bytes / 4)}, at::kInt, parent);
    if (want_lineage) {
        lineage = fresh({n, width}, at::kLong, parent);
        level = fresh({n}, at::kLong, parent);
    }
    // A caller that waits is told through pinned host memory, a word per block; a word in device memory is for those that
    // look later.
    at::Tensor flags, status;
    if (check && nb > 0) {
        flags = at::empty({nb}, at::TensorOptions().dtype(at::kInt).pinned_memory(true));
        memset(flags.data_ptr(), 0, (size_t)nb * sizeof(int32_t));
    }
    if (!check) status = status_word(args[7], parent);
    const int rc = fsta_precompute_from_parents_flags(
        parent.data_ptr<int64_t>(), n, width, (int32_t)block_m, (int32_t)max_anc, 1, data_or_null<int64_t>(lineage),
        data_or_null<int64_t>(level), a_idx.data_ptr<int64_t>(), data_or_null<uint8_t>(a_mask), l_idx.data_ptr<int64_t>(),
        static_cast<uint32_t*>(bits.data_ptr()), count.data_ptr<int32_t>(), data_or_null<uint32_t>(plan),
        data_or_null<uint32_t>(status), data_or_null<uint32_t>(flags), on.stream);
    if (rc != FSTA_OK) return PyLong_FromLong(rc);
    long found = 0;
    if (check && nb > 0) {
        pybind11::gil_scoped_release no_gil;
        found = watch_flags(flags.data_ptr<int32_t>(), nb, on.stream);
    }
    PyObject* tensors = as_tuple(a_idx, a_mask, l_idx, bits, count, plan, lineage, level, status);
    return tensors ? Py_BuildValue("Nl", tensors, found) : nullptr;
    END_HANDLE_TH_ERRORS
}

// medusa_parents(probs, n, read_status, status or None) -> (parent, status)
PyObject* medusa_parents(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n_args == 4, "medusa_parents takes 4 arguments");
    const at::Tensor probs = tensor_arg(args[0]).contiguous();
    const int64_t n = int_arg(args[1]);
    const OnStream on(probs);
    const int32_t depths = (int32_t)probs.size(0), topk = (int32_t)probs.size(1);
    const int32_t code = probs.scalar_type() == at::kFloat ? FSTA_F32 : FSTA_F64;
    at::Tensor parent = fresh({n}, at::kLong, probs);
    at::Tensor status = args[3] != Py_None || args[2] == Py_True ? status_word(args[3], probs) : fresh({1}, at::kInt, probs);
    const size_t need = fsta_medusa_workspace_bytes(depths, topk);
    at::Tensor work;      // (stream-ordered: free again after the launches)
    if (need) work = fresh({(int64_t)need}, at::kByte, probs);
    uint32_t* word = static_cast<uint32_t*>(status.data_ptr());
    const int rc = need ? fsta_medusa_tree_ws(probs.data_ptr(), code, depths, topk, (int32_t)n, parent.data_ptr<int64_t>(), word,
                                              work.data_ptr(), need, on.stream)
                        : fsta_medusa_tree(probs.data_ptr(), code, depths, topk, (int32_t)n, parent.data_ptr<int64_t>(), word, on.stream);
    return rc != FSTA_OK ? PyLong_FromLong(rc) : as_tuple(parent, status);
    END_HANDLE_TH_ERRORS
}

// shift_index(ancestor_idx, leaf_idx, shift) -> both with `shift` added to the entries that are not negative; NotImplemented
// for anything but ordinary int64 tensors on one GPU
PyObject* shift_index(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 3 || !plain_context()) return not_implemented();
    const at::Tensor *a = gpu_tensor(args[0]), *b = gpu_tensor(args[1]);
    int64_t shift;
    if (!a || !b || a->scalar_type() != at::kLong || b->scalar_type() != at::kLong || a->device() != b->device() || !as_int(args[2], &shift))
        return not_implemented();
    const at::Tensor ac = a->contiguous(), bc = b->contiguous();
    const OnStream on(ac);
    at::Tensor out_a = fresh(ac.sizes(), at::kLong, ac), out_b = fresh(bc.sizes(), at::kLong, bc);
    const int rc = fsta_shift_index(ac.data_ptr<int64_t>(), ac.numel(), bc.data_ptr<int64_t>(), bc.numel(), shift,
                                    out_a.data_ptr<int64_t>(), out_b.data_ptr<int64_t>(), on.stream);
    return rc != FSTA_OK ? not_implemented() : as_tuple(out_a, out_b);
    END_HANDLE_TH_ERRORS
}

// quantizes(k, v): True if the operator for the 8-bit storage, whose only implementation is a kernel, takes both: ordinary GPU
// tensors of one shape and type, in slices of whole 16-byte pieces, that nobody transforms, traces below the dispatcher or
// differentiates, in either direction.  (A mode that watches calls from Python, such as a default device, sees the operator.)
PyObject* quantizes(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n_args == 2, "quantizes takes 2 arguments");
    if (!plain_dispatch()) Py_RETURN_FALSE;
    const at::Tensor* t[2];
    for (int i = 0; i < 2; ++i) {
        t[i] = gpu_tensor(args[i]);
        if (!t[i] || wants_derivative(*t[i])) Py_RETURN_FALSE;
    }
    const at::Tensor &k = *t[0], &v = *t[1];
    if (k.dim() != 4 || v.sizes() != k.sizes() || v.device() != k.device() || v.scalar_type() != k.scalar_type() ||
        fsta_torch::dtype_code(k.scalar_type()) < 0 || k.numel() == 0 || k.size(2) * k.size(3) % 16 != 0 ||
        k.size(0) * k.size(1) > (int64_t)1 << 20 ||      // (a workgroup of 1024 threads per slice of both: a grid ends at 2^32)
        (uintptr_t)k.data_ptr() % 16 != 0 || (uintptr_t)v.data_ptr() % 16 != 0)
        Py_RETURN_FALSE;
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// setup(PackedTreeMask, packed_table)
PyObject* setup(PyObject*, PyObject* args) {
    PyObject *type, *table;
    if (!PyArg_ParseTuple(args, "OO!", &type, &PyDict_Type, &table)) return nullptr;
    Py_INCREF(type);
    Py_INCREF(table);
    Py_XSETREF(g_packed_type, type);
    Py_XSETREF(g_packed_table, table);
    Py_RETURN_NONE;
}

// ---- the paged KV cache: calls that paged.py has nothing to complain about; it judges and raises for all others --------

int half_code(at::ScalarType t) { return t == at::kHalf ? FSTA_F16 : t == at::kBFloat16 ? FSTA_BF16 : -1; }

struct Pool {      // paged.PagedKV
    const at::Tensor *k, *v, *exps[2];      // exps: null but for 8-bit rows
    uint8_t *k_exp, *v_exp;
    int32_t pages, heads, page_size, head_dim, code;
};

bool read_pool(PyObject* o, Pool* p) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) return false;
    p->k = gpu_tensor(PyTuple_GET_ITEM(o, 0));
    p->v = gpu_tensor(PyTuple_GET_ITEM(o, 1));
    if (!p->k || !p->v || p->k->dim() != 4 || p->v->sizes() != p->k->sizes() || p->v->scalar_type() != p->k->scalar_type() ||
        p->v->device() != p->k->device() || !p->k->is_contiguous() || !p->v->is_contiguous() ||
        wants_derivative(*p->k) || wants_derivative(*p->v))
        return false;
    const bool fp8 = p->k->scalar_type() == at::kFloat8_e4m3fn;
    p->code = fp8 ? FSTA_FP8 : half_code(p->k->scalar_type());
    uint8_t* exps[2] = {nullptr, nullptr};
    p->exps[0] = p->exps[1] = nullptr;
    for (int i = 0; i < 2; ++i) {
        PyObject* item = PyTuple_GET_ITEM(o, 2 + i);
        if (fp8 != (item != Py_None)) return false;
        if (!fp8) continue;
        const at::Tensor* e = gpu_tensor(item);
        if (!e || e->scalar_type() != at::kByte || e->sizes() != p->k->sizes().slice(0, 3) || !e->is_contiguous() || e->device() != p->k->device())
            return false;
        p->exps[i] = e;
        exps[i] = static_cast<uint8_t*>(e->data_ptr());
    }
    p->k_exp = exps[0];
    p->v_exp = exps[1];
    for (int64_t i = 0; i < 4; ++i)
        if (p->k->size(i) > INT32_MAX) return false;
    p->pages = (int32_t)p->k->size(0);
    p->heads = (int32_t)p->k->size(1);
    p->page_size = (int32_t)p->k->size(2);
    p->head_dim = (int32_t)p->k->size(3);
    return p->code >= 0;
}

const int32_t* int32_array(PyObject* o, const at::Tensor& like, int64_t dims, int64_t size) {
    const at::Tensor* t = gpu_tensor(o);
    return t && t->scalar_type() == at::kInt && t->dim() == dims && t->size(0) == size && t->is_contiguous() && t->device() == like.device()
               ? static_cast<const int32_t*>(t->data_ptr())
               : nullptr;
}

struct Batch {
    const int32_t *table, *lens, *starts;
    int32_t batch, width;
};
// starts == null: not wanted
bool read_batch(const Pool& pool, PyObject* table, PyObject* lens, PyObject* starts, Batch* b) {
    const at::Tensor* t = gpu_tensor(table);
    if (!t || t->dim() != 2 || t->size(0) == 0 || t->size(1) == 0 || t->size(0) > INT32_MAX || t->size(1) > INT32_MAX) return false;
    b->batch = (int32_t)t->size(0);
    b->width = (int32_t)t->size(1);
    b->table = int32_array(table, *pool.k, 2, b->batch);
    b->lens = int32_array(lens, *pool.k, 1, b->batch);
    b->starts = starts ? int32_array(starts, *pool.k, 1, (int64_t)b->batch + 1) : nullptr;
    return b->table && b->lens && (b->starts || !starts);
}

// Packed rows [tokens, heads, head_dim], at least one
const at::Tensor* read_rows(PyObject* o, const Pool& pool) {
    const at::Tensor* t = gpu_tensor(o);
    if (!t || t->dim() != 3 || t->numel() == 0 || t->size(0) > INT32_MAX || t->size(2) != pool.head_dim || t->stride(2) != 1 ||
        t->device() != pool.k->device() || wants_derivative(*t))
        return nullptr;
    const int code = half_code(t->scalar_type());
    return code >= 0 && (pool.code == FSTA_FP8 || pool.code == code) ? t : nullptr;
}
int64_t stride_of(const at::Tensor& t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }

// paged_write(cache, k, v, page_table, kv_lens, q_starts) -> None
PyObject* paged_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Pool pool;
    Batch b;
    if (n != 6 || !plain_context() || !read_pool(args[0], &pool) || !read_batch(pool, args[3], args[4], args[5], &b)) return not_implemented();
    const at::Tensor *k = read_rows(args[1], pool), *v = read_rows(args[2], pool);
    if (!k || !v || k->sizes() != v->sizes() || k->size(1) != pool.heads || k->scalar_type() != v->scalar_type()) return not_implemented();
    try {
        const OnStream on(*pool.k);
        if (fsta_paged_write(k->data_ptr(), v->data_ptr(), stride_of(*k, 0), stride_of(*k, 1), stride_of(*v, 0), stride_of(*v, 1),
                             pool.k->data_ptr(), pool.v->data_ptr(), pool.k_exp, pool.v_exp, b.table, b.lens, b.starts, b.batch, b.width,
                             (int32_t)k->size(0), pool.pages, pool.page_size, pool.heads, pool.head_dim, half_code(k->scalar_type()),
                             pool.code, on.stream) != FSTA_OK)
            return not_implemented();
        // autograd is told, as by torch's own operations in place (inference tensors have no version counter)
        for (const at::Tensor* t : {pool.k, pool.v, pool.exps[0], pool.exps[1]})
            if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    } catch (const std::exception&) {
        return not_implemented();
    }
    Py_RETURN_NONE;
}

// paged_read(cache, page_table, kv_lens, max_len, dtype or None) -> (k, v)
PyObject* paged_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Pool pool;
    Batch b;
    int64_t max_len;
    if (n != 5 || !plain_context() || !read_pool(args[0], &pool) || !read_batch(pool, args[1], args[2], nullptr, &b) || !as_int(args[3], &max_len) ||
        max_len < 0 || max_len > INT32_MAX)
        return not_implemented();
    at::ScalarType type = pool.code == FSTA_FP8 ? at::kBFloat16 : pool.k->scalar_type();
    if (args[4] != Py_None) {
        if (!THPDtype_Check(args[4])) return not_implemented();
        const at::ScalarType asked = reinterpret_cast<THPDtype*>(args[4])->scalar_type;
        if (half_code(asked) < 0 || (pool.code != FSTA_FP8 && asked != type)) return not_implemented();
        type = asked;
    }
    try {
        const OnStream on(*pool.k);
        const at::Tensor k = fresh({b.batch, pool.heads, max_len, pool.head_dim}, type, *pool.k), v = fresh(k.sizes(), type, *pool.k);
        if (fsta_paged_read(pool.k->data_ptr(), pool.v->data_ptr(), pool.k_exp, pool.v_exp, b.table, b.lens, k.data_ptr(), v.data_ptr(), b.batch,
                            b.width, (int32_t)max_len, pool.pages, pool.page_size, pool.heads, pool.head_dim, half_code(type), pool.code,
                            on.stream) != FSTA_OK)
            return not_implemented();
        return as_tuple(k, v);
    } catch (const std::exception&) {
        return not_implemented();
    }
}

// paged_attention(q, cache, page_table, kv_lens, q_starts, sm_scale, causal, tree_bits or None, max_q_len or None, return_lse)
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Pool pool;
    Batch b;
    if (n != 10 || !plain_context() || !read_pool(args[1], &pool) || !read_batch(pool, args[2], args[3], args[4], &b) || !PyFloat_Check(args[5]))
        return not_implemented();
    const at::Tensor* q = read_rows(args[0], pool);
    const double sm_scale = PyFloat_AS_DOUBLE(args[5]);
    if (!q || q->size(1) % std::max(pool.heads, 1) || pool.heads == 0 || pool.pages == 0 || !(sm_scale > 0)) return not_implemented();
    const int32_t tokens = (int32_t)q->size(0), heads = (int32_t)std::min<int64_t>(q->size(1), INT32_MAX);
    if (!PyBool_Check(args[6]) || !PyBool_Check(args[9])) return not_implemented();
    const uint32_t* bits = nullptr;
    int32_t words = 0, mask = args[6] == Py_True ? FSTA_PAGED_CAUSAL : FSTA_PAGED_ALL;
    if (args[7] != Py_None) {
        bits = reinterpret_cast<const uint32_t*>(int32_array(args[7], *q, 2, tokens));
        if (!bits) return not_implemented();
        words = (int32_t)THPVariable_Unpack(args[7]).size(1);
        mask = FSTA_PAGED_TREE;
    }
    int64_t most = 0;
    if (args[8] != Py_None && (!as_int(args[8], &most) || most < 0 || most > INT32_MAX)) return not_implemented();
    try {
        const OnStream on(*q);
        const at::Tensor o = fresh(q->sizes(), q->scalar_type(), *q);
        const at::Tensor lse = args[9] == Py_True ? fresh({tokens, heads}, at::kFloat, *q) : at::Tensor();
        const size_t need = fsta_paged_attention_workspace_bytes(b.batch, tokens, (int32_t)most, heads, pool.heads, pool.head_dim, pool.code);
        const at::Tensor work = fresh({(int64_t)need}, at::kByte, *q);
        if (fsta_paged_attention(q->data_ptr(), stride_of(*q, 0), stride_of(*q, 1), pool.k->data_ptr(), pool.v->data_ptr(), pool.k_exp, pool.v_exp,
                                 b.table, b.lens, b.starts, bits, words, o.data_ptr(), data_or_null<float>(lse), b.batch, b.width, tokens,
                                 (int32_t)most, pool.pages, pool.page_size, heads, pool.heads, pool.head_dim, half_code(q->scalar_type()), pool.code,
                                 mask, (float)sm_scale, work.data_ptr(), need, on.stream) != FSTA_OK)
            return not_implemented();
        return lse.defined() ? as_tuple(o, lse) : THPVariable_Wrap(o);
    } catch (const std::exception&) {
        return not_implemented();
    }
}

// tree_bits(parent, q_starts, max_nodes): paged.tree_mask_bits of a batch
PyObject* tree_bits(PyObject*, PyObject* const* args, Py_ssize_t n) {
    int64_t most;
    if (n != 3 || !plain_context() || !as_int(args[2], &most) || most <= 0 || most > INT32_MAX - 32) return not_implemented();
    const at::Tensor *parent = gpu_tensor(args[0]), *starts = gpu_tensor(args[1]);
    if (!parent || !starts || parent->dim() != 1 || parent->scalar_type() != at::kLong || parent->size(0) == 0 || parent->size(0) > INT32_MAX ||
        !parent->is_contiguous() || starts->dim() != 1 || starts->size(0) < 2 || starts->size(0) > INT32_MAX)
        return not_implemented();
    const int32_t* first = int32_array(args[1], *parent, 1, starts->size(0));
    if (!first) return not_implemented();
    try {
        const OnStream on(*parent);
        const at::Tensor bits = fresh({parent->size(0), (most + 31) / 32}, at::kInt, *parent);
        if (fsta_tree_bits(parent->data_ptr<int64_t>(), first, (int32_t)(starts->size(0) - 1), (int32_t)parent->size(0), (int32_t)bits.size(1),
                           static_cast<uint32_t*>(bits.data_ptr()), on.stream) != FSTA_OK)
            return not_implemented();
        return THPVariable_Wrap(bits);
    } catch (const std::exception&) {
        return not_implemented();
    }
}

// ---- what happens between two passes of a model: drafts.py and pages.py judge and raise for all other calls --------------

// A float tensor [nodes, vocabulary] whose rows are contiguous
const at::Tensor* read_logits(PyObject* o) {
    const at::Tensor* t = gpu_tensor(o);
    return t && t->dim() == 2 && t->numel() > 0 && t->size(0) <= INT32_MAX && t->size(1) <= INT32_MAX - 65536 && (t->size(1) == 1 || t->stride(1) == 1) &&
                   (t->scalar_type() == at::kFloat || half_code(t->scalar_type()) >= 0)
               ? t
               : nullptr;
}
int float_code(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? FSTA_F32 : half_code(t.scalar_type()); }
int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// The data of a contiguous tensor [size] of one type on like's device
template <typename T> const T* array_of(PyObject* o, const at::Tensor& like, at::ScalarType type, int64_t size) {
    const at::Tensor* t = gpu_tensor(o);
    return t && t->scalar_type() == type && t->dim() == 1 && t->size(0) == size && t->is_contiguous() && t->device() == like.device()
               ? static_cast<const T*>(t->data_ptr())
               : nullptr;
}

// verify_drafts(logits, tokens, parent, q_starts, u_accept, u_next, max_path, temperature, draft_probs or None) -> (path, counts, next)
PyObject* verify_drafts(PyObject*, PyObject* const* args, Py_ssize_t n) {
    int64_t most;
    if (n != 9 || !plain_context() || !as_int(args[6], &most) || most < 1 || most > INT32_MAX) return not_implemented();
    const at::Tensor *logits = read_logits(args[0]), *starts = gpu_tensor(args[3]), *draft = nullptr;
    if (!logits || !starts || starts->dim() != 1 || starts->size(0) < 2 || starts->size(0) > INT32_MAX) return not_implemented();
    const int64_t nodes = logits->size(0), batch = starts->size(0) - 1;
    const int64_t *tokens = array_of<int64_t>(args[1], *logits, at::kLong, nodes), *parent = array_of<int64_t>(args[2], *logits, at::kLong, nodes);
    const int32_t* first = array_of<int32_t>(args[3], *logits, at::kInt, batch + 1);
    const float *u_accept = array_of<float>(args[4], *logits, at::kFloat, nodes), *u_next = array_of<float>(args[5], *logits, at::kFloat, batch);
    if (!tokens || !parent || !first || !u_accept || !u_next) return not_implemented();
    const float* temperatures = nullptr;
    double temperature = 0;
    if (PyFloat_Check(args[7])) {
        temperature = PyFloat_AS_DOUBLE(args[7]);
        if (!(temperature >= 0) || (float)temperature > std::numeric_limits<float>::max()) return not_implemented();
    } else if (!(temperatures = array_of<float>(args[7], *logits, at::kFloat, batch))) {
        return not_implemented();
    }
    if (args[8] != Py_None) {
        draft = read_logits(args[8]);
        if (!draft || draft->sizes() != logits->sizes() || draft->device() != logits->device()) return not_implemented();
    }
    try {
        const OnStream on(*logits);
        const at::Tensor path = fresh({batch, most}, at::kInt, *logits), counts = fresh({batch}, at::kInt, *logits),
                         next = fresh({batch}, at::kLong, *logits);
        const size_t need = fsta_verify_workspace_bytes((int32_t)batch, (int32_t)nodes, (int32_t)logits->size(1), (int32_t)most, draft != nullptr);
        const at::Tensor work = need ? fresh({(int64_t)need}, at::kByte, *logits) : at::Tensor();
        if (fsta_verify_drafts(logits->data_ptr(), row_stride(*logits), float_code(*logits), draft ? draft->data_ptr() : nullptr,
                               draft ? row_stride(*draft) : 0, draft ? float_code(*draft) : FSTA_F32, tokens, parent, first, u_accept, u_next,
                               temperatures, (float)temperature, path.data_ptr<int32_t>(), counts.data_ptr<int32_t>(), next.data_ptr<int64_t>(),
                               (int32_t)batch, (int32_t)nodes, (int32_t)logits->size(1), (int32_t)most, need ? work.data_ptr() : nullptr, need,
                               on.stream) != FSTA_OK)
            return not_implemented();
        return as_tuple(path, counts, next);
    } catch (const std::exception&) {
        return not_implemented();
    }
}

// The caches of all layers: a PagedKV, or a list or tuple of them
struct Pools {
    std::vector<fsta_paged_pool> layers;
    std::vector<const at::Tensor*> tensors;      // what a call that writes to them changes
    const at::Tensor* k = nullptr;               // of the first
    int32_t pages = 0, page_size = 0;
};
bool read_pools(PyObject* o, Pools* p) {
    const bool list = PyList_CheckExact(o);
    if (!list && !PyTuple_Check(o)) return false;
    PyObject** items = list ? reinterpret_cast<PyListObject*>(o)->ob_item : reinterpret_cast<PyTupleObject*>(o)->ob_item;
    Py_ssize_t n = Py_SIZE(o);
    if (n == 0) return false;
    if (!list && THPVariable_Check(items[0])) items = &o, n = 1;      // a PagedKV itself
    p->layers.resize(n);
    p->tensors.reserve(2 * n);
    for (Py_ssize_t i = 0; i < n; ++i) {
        Pool pool;
        if (!read_pool(items[i], &pool)) return false;
        if (i == 0) p->k = pool.k, p->pages = pool.pages, p->page_size = pool.page_size;
        if (pool.pages != p->pages || pool.page_size != p->page_size || pool.k->device() != p->k->device()) return false;
        p->layers[i] = fsta_paged_pool{pool.k->data_ptr(), pool.v->data_ptr(), pool.k_exp, pool.v_exp, pool.heads, pool.head_dim, pool.code, 0};
        for (const at::Tensor* t : {pool.k, pool.v, pool.exps[0], pool.exps[1]})
            if (t) p->tensors.push_back(t);
    }
    return true;
}
void moved(const at::Tensor* t) {
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}
void moved(const Pools& p) {
    for (const at::Tensor* t : p.tensors) moved(t);
}

// [batch, width] of a page table on the pools' device, or false
bool read_table(PyObject* o, const Pools& p, int32_t* batch, int32_t* width, const int32_t** data) {
    const at::Tensor* t = gpu_tensor(o);
    if (!t || t->dim() != 2 || t->size(0) == 0 || t->size(0) > INT32_MAX || t->size(1) > INT32_MAX) return false;
    *batch = (int32_t)t->size(0);
    *width = (int32_t)t->size(1);
    *data = int32_array(o, *p.k, 2, *batch);
    return *data != nullptr;
}

// compact_paged_kv(caches, path, counts, page_table, kv_lens, q_starts) -> lengths
PyObject* compact_paged_kv(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        Pools pools;
        int32_t batch, width;
        const int32_t* table;
        if (n != 6 || !plain_context() || !read_pools(args[0], &pools) || !read_table(args[3], pools, &batch, &width, &table)) return not_implemented();
        const int32_t *path = int32_array(args[1], *pools.k, 2, batch), *counts = int32_array(args[2], *pools.k, 1, batch);
        const int32_t *lens = int32_array(args[4], *pools.k, 1, batch), *starts = int32_array(args[5], *pools.k, 1, (int64_t)batch + 1);
        if (!path || !counts || !lens || !starts || THPVariable_Unpack(args[1]).size(1) > INT32_MAX) return not_implemented();
        const OnStream on(*pools.k);
        const at::Tensor out = fresh({batch}, at::kInt, *pools.k);
        if (fsta_compact_paged_kv(pools.layers.data(), (int32_t)pools.layers.size(), pools.pages, pools.page_size, path,
                                  (int32_t)THPVariable_Unpack(args[1]).size(1), counts, table, lens, starts, batch, width, out.data_ptr<int32_t>(),
                                  on.stream) != FSTA_OK)
            return not_implemented();
        moved(pools);
        return THPVariable_Wrap(out);
    } catch (const std::exception&) {
        return not_implemented();
    }
}

// copy_pages(caches, sources, targets, into or None) -> None
PyObject* copy_pages(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        Pools pools, others;
        if (n != 4 || !plain_context() || !read_pools(args[0], &pools)) return not_implemented();
        const bool elsewhere = args[3] != Py_None;
        if (elsewhere && (!read_pools(args[3], &others) || others.layers.size() != pools.layers.size() || others.page_size != pools.page_size ||
                          others.k->device() != pools.k->device()))
            return not_implemented();
        const Pools& into = elsewhere ? others : pools;
        const at::Tensor* t = gpu_tensor(args[1]);
        if (!t || t->dim() != 1 || t->size(0) > INT32_MAX) return not_implemented();
        const int32_t *sources = int32_array(args[1], *pools.k, 1, t->size(0)), *targets = int32_array(args[2], *pools.k, 1, t->size(0));
        if (!sources || !targets) return not_implemented();
        const OnStream on(*pools.k);
        if (fsta_copy_pages(pools.layers.data(), into.layers.data(), (int32_t)pools.layers.size(), pools.pages, into.pages, pools.page_size, sources,
                            targets, (int32_t)t->size(0), on.stream) != FSTA_OK)
            return not_implemented();
        moved(into);
    } catch (const std::exception&) {
        return not_implemented();
    }
    Py_RETURN_NONE;
}

// fit_pages(caches, refs, page_table, lens) -> missing
PyObject* fit_pages(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        Pools pools;
        int32_t batch, width;
        const int32_t* table;
        if (n != 4 || !plain_context() || !read_pools(args[0], &pools) || !read_table(args[2], pools, &batch, &width, &table)) return not_implemented();
        const int32_t *refs = int32_array(args[1], *pools.k, 1, pools.pages), *lens = int32_array(args[3], *pools.k, 1, batch);
        if (!refs || !lens) return not_implemented();
        const OnStream on(*pools.k);
        const at::Tensor missing = fresh({batch}, at::kInt, *pools.k);
        const size_t need = fsta_fit_pages_workspace_bytes(batch, pools.pages);
        const at::Tensor work = fresh({(int64_t)need}, at::kByte, *pools.k);
        if (fsta_fit_pages(pools.layers.data(), (int32_t)pools.layers.size(), pools.pages, pools.page_size, const_cast<int32_t*>(refs),
                           const_cast<int32_t*>(table), lens, batch, width, missing.data_ptr<int32_t>(), work.data_ptr(), need, on.stream) != FSTA_OK)
            return not_implemented();
        moved(pools);
        moved(&THPVariable_Unpack(args[1]));
        moved(&THPVariable_Unpack(args[2]));
        return THPVariable_Wrap(missing);
    } catch (const std::exception&) {
        return not_implemented();
    }
}

// fork_pages(caches, refs, page_table, lens, sources, targets) -> missing
PyObject* fork_pages(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        Pools pools;
        int32_t batch, width;
        const int32_t* table;
        if (n != 6 || !plain_context() || !read_pools(args[0], &pools) || !read_table(args[2], pools, &batch, &width, &table)) return not_implemented();
        const int32_t *refs = int32_array(args[1], *pools.k, 1, pools.pages), *lens = int32_array(args[3], *pools.k, 1, batch);
        const at::Tensor* t = gpu_tensor(args[4]);
        if (!refs || !lens || !t || t->dim() != 1 || t->size(0) > INT32_MAX) return not_implemented();
        const int32_t pairs = (int32_t)t->size(0);
        const int32_t *sources = int32_array(args[4], *pools.k, 1, pairs), *targets = int32_array(args[5], *pools.k, 1, pairs);
        if (!sources || !targets) return not_implemented();
        const OnStream on(*pools.k);
        const at::Tensor missing = fresh({pairs}, at::kInt, *pools.k);
        const size_t need = fsta_fork_pages_workspace_bytes(pairs, width, pools.pages);
        const at::Tensor work = fresh({(int64_t)need}, at::kByte, *pools.k);
        if (fsta_fork_pages(pools.layers.data(), (int32_t)pools.layers.size(), pools.pages, pools.page_size, const_cast<int32_t*>(refs),
                            const_cast<int32_t*>(table), const_cast<int32_t*>(lens), batch, width, sources, targets, pairs, missing.data_ptr<int32_t>(),
                            work.data_ptr(), need, on.stream) != FSTA_OK)
            return not_implemented();
        moved(pools);
        for (int i : {1, 2, 3}) moved(&THPVariable_Unpack(args[i]));
        return THPVariable_Wrap(missing);
    } catch (const std::exception&) {
        return not_implemented();
    }
}

#define FSTA_FASTCALL(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&f)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {
    FSTA_FASTCALL(attention),
    FSTA_FASTCALL(dfs_order),
    FSTA_FASTCALL(renumber_parents),
    FSTA_FASTCALL(inputs_from_parents),
    FSTA_FASTCALL(medusa_parents),
    FSTA_FASTCALL(shift_index),
    FSTA_FASTCALL(quantizes),
    FSTA_FASTCALL(paged_write),
    FSTA_FASTCALL(paged_read),
    FSTA_FASTCALL(paged_attention),
    FSTA_FASTCALL(tree_bits),
    FSTA_FASTCALL(verify_drafts),
    FSTA_FASTCALL(compact_paged_kv),
    FSTA_FASTCALL(copy_pages),
    FSTA_FASTCALL(fit_pages),
    FSTA_FASTCALL(fork_pages),
    {"setup", &setup, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fsta_torch", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fsta_torch(void) { return PyModule_Create(&kModule); }
