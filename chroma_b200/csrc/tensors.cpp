// The operators on CUDA tensors: checks of their arguments, outputs and workspace from Torch's allocator, and calls of the C
// ABI (include/chroma_b200.h) on the current stream of the tensors' device. A Python extension module
// (chroma_b200/_src/_tensors.so) rather than ctypes: a call takes about 4 microseconds of host time where ctypes and Python
// checks took 9 to 23, and single tokens are decided by that.
//
// The entry points of libchroma_b200.so are handed over once by `bind` (chroma_b200/_src/paged.py), so that the module follows
// whichever library the process has loaded.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "../../include/chroma_b200.h"

namespace {

using at::Tensor;

#define ENTRY(name) decltype(&chroma_b200_##name) name = nullptr
struct Entries {
    ENTRY(paged_append);
    ENTRY(paged_attention);
    ENTRY(attention_workspace);
    ENTRY(step_pages);
    ENTRY(step_pages_uncut);
    ENTRY(compact_pages);
    ENTRY(pages_workspace);
    ENTRY(process_logits);
    ENTRY(logits_workspace);
} native;
#undef ENTRY

// An argument that has to be a tensor, or may be None.
const Tensor& tensor(PyObject* o, const char* name) {
    TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor, not ", Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}
const Tensor* optional(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }

int integer(PyObject* o, const char* name) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    TORCH_CHECK_VALUE(v >= 0 && v <= INT32_MAX, name, " must be nonnegative and below 2^31, got ", v);
    return int(v);
}

bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw python_error();
    return v;
}

int storage_of(const Tensor& t, const char* what) {
    const auto type = t.scalar_type();
    TORCH_CHECK_VALUE(type == at::kFloat || type == at::kBFloat16, what, " must be float32 or bfloat16, got ", type);
    return type == at::kBFloat16 ? CHROMA_B200_BF16 : CHROMA_B200_FP32;
}

// The tensors of one call: all on one CUDA device, which is the current one while the call lasts.
struct Call {
    c10::cuda::OptionalCUDAGuard guard;
    at::Device device;
    explicit Call(const Tensor& first) : device(first.device()) {
        TORCH_CHECK_VALUE(first.is_cuda(), "tensors must be on a CUDA device");
        guard.set_device(device);
    }
    void with(const Tensor& t) const { TORCH_CHECK_VALUE(t.device() == device, "tensors on different devices"); }
    void with(const Tensor* t) const {
        if (t) with(*t);
    }
    void* stream() const { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }
    Tensor empty(at::IntArrayRef shape, at::ScalarType type) const { return at::empty(shape, at::TensorOptions().dtype(type).device(device)); }
};

// The operators have no gradients. What comes of a tensor that wants one says so when it is differentiated; what is written in
// place counts its version up, so that a graph which still needs the old values says so.
using Inputs = std::initializer_list<const Tensor*>;
bool wanted(Inputs inputs) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : inputs)
        if (t && t->requires_grad()) return true;
    return false;
}
void no_gradient(const char* name, Inputs inputs, Inputs outputs) {
    if (!wanted(inputs)) return;
    for (const Tensor* out : outputs) {
        if (!out->defined()) continue;
        torch::autograd::edge_list edges;
        for (const Tensor* t : inputs)
            if (t && t->requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(*t));
        std::shared_ptr<torch::autograd::Node> node(new torch::autograd::NotImplemented(name), torch::autograd::deleteNode);
        node->set_next_edges(std::move(edges));
        torch::autograd::set_history(*out, node);
    }
}
void written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void check_out(const Tensor* out, Inputs inputs) {
    TORCH_CHECK_VALUE(!out || !(wanted(inputs) || wanted({out})), "out cannot be given where a gradient is wanted (torch.no_grad() turns them off)");
}

void run(int status, const char* err) {
    TORCH_CHECK_VALUE(status != CHROMA_B200_VALUE, err);
    TORCH_CHECK_INDEX(status != CHROMA_B200_INDEX, err);
    TORCH_CHECK(status == CHROMA_B200_OK, err);
}

const int32_t* ints(const Call& call, const Tensor& t, int64_t n, const char* name) {
    call.with(t);
    TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous(), name,
                      " must be contiguous int32 [", n, "], got ", t.scalar_type(), " ", t.sizes());
    return t.const_data_ptr<int32_t>();
}
const int32_t* ints(const Call& call, const Tensor* t, int64_t n, const char* name) { return t ? ints(call, *t, n, name) : nullptr; }

chroma_b200_pages pages_of(const Call& call, const Tensor& keys, const Tensor& values, const Tensor& table, const Tensor& lengths,
                           bool layered) {
    call.with(keys), call.with(values), call.with(table);
    chroma_b200_pages p{};
    p.storage = storage_of(keys, "pools");
    TORCH_CHECK_VALUE(values.scalar_type() == keys.scalar_type(), "pools are of one type, got ", keys.scalar_type(), " and ", values.scalar_type());
    const int64_t rank = keys.dim();
    TORCH_CHECK_VALUE(values.sizes() == keys.sizes() && (rank == 4 || (layered && rank == 5)), "pools must be [",
                      layered ? "layers, " : "", "pages, rows, heads, dim], alike, got ", keys.sizes(), " and ", values.sizes());
    TORCH_CHECK_VALUE(keys.stride(rank - 1) == 1 && values.stride(rank - 1) == 1, "a head's row must be contiguous");
    TORCH_CHECK_VALUE(table.scalar_type() == at::kInt && table.dim() == 2 && table.stride(1) == 1, "table must be int32 [slots, width] with contiguous rows");
    const int64_t first = rank - 4;
    for (int i = 0; i < 5; ++i) {
        const int64_t at = first - 1 + i;  // layers, pages, rows, heads, dim
        const int64_t size = at < 0 ? 1 : keys.size(at);
        TORCH_CHECK_VALUE(size <= INT32_MAX, "pool too large");
        (&p.layers)[i] = int32_t(size);
        if (i < 4) {
            p.key_strides[i] = at < 0 ? 0 : keys.stride(at);
            p.value_strides[i] = at < 0 ? 0 : values.stride(at);
        }
    }
    TORCH_CHECK_VALUE(table.size(0) <= INT32_MAX && table.size(1) <= INT32_MAX, "table too large");
    p.slots = int32_t(table.size(0));
    p.width = int32_t(table.size(1));
    p.table_stride = table.stride(0);
    p.keys = keys.data_ptr();
    p.values = values.data_ptr();
    p.table = table.const_data_ptr<int32_t>();
    p.lengths = ints(call, lengths, p.slots, "lengths");
    return p;
}

void count_args(Py_ssize_t n, Py_ssize_t want) { TORCH_CHECK_TYPE(n == want, "expected ", want, " arguments, got ", n); }

PyObject* paged_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count_args(n, 7);
    const Tensor &keys = tensor(args[0], "keys"), &nk = tensor(args[2], "new_keys"), &nv = tensor(args[3], "new_values"), &table = tensor(args[4], "table");
    const Tensor* starts = optional(args[6], "starts");
    const Call call(keys);
    const auto p = pages_of(call, keys, tensor(args[1], "values"), table, tensor(args[5], "lengths"), false);
    call.with(nk), call.with(nv);
    for (const Tensor* t : {&nk, &nv})
        TORCH_CHECK_VALUE(t->dim() == 3 && t->size(0) == nk.size(0) && t->size(1) == p.kv_heads && t->size(2) == p.head_dim && t->scalar_type() == keys.scalar_type(),
                          "new rows must be [tokens, ", p.kv_heads, ", ", p.head_dim, "] ", keys.scalar_type(), ", got ", t->sizes(), " ", t->scalar_type());
    TORCH_CHECK_VALUE(nk.stride(2) == 1 && nv.stride(2) == 1, "a head's row must be contiguous");
    TORCH_CHECK_VALUE(nk.size(0) <= INT32_MAX, "too many rows");
    const int64_t strides[4] = {nk.stride(0), nk.stride(1), nv.stride(0), nv.stride(1)};
    char err[512];
    run(native.paged_append(&p, nk.const_data_ptr(), nv.const_data_ptr(), strides, ints(call, starts, int64_t(p.slots) + 1, "starts"),
                            int32_t(nk.size(0)), call.stream(), err, sizeof err), err);
    written(keys), written(tensor(args[1], "values"));
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count_args(n, 12);
    const Tensor &q = tensor(args[0], "q"), &keys = tensor(args[1], "keys"), &table = tensor(args[3], "table");
    const Tensor *starts = optional(args[5], "starts"), *sinks = optional(args[9], "sinks"), *given = optional(args[11], "out");
    const Call call(q);
    const auto p = pages_of(call, keys, tensor(args[2], "values"), table, tensor(args[4], "lengths"), false);
    TORCH_CHECK_VALUE(q.dim() == 3 && q.scalar_type() == keys.scalar_type() && q.size(2) == p.head_dim, "q must be [tokens, heads, ", p.head_dim,
                      "] ", keys.scalar_type(), ", got ", q.sizes(), " ", q.scalar_type());
    TORCH_CHECK_VALUE(q.size(0) <= INT32_MAX && q.size(1) <= INT32_MAX, "too many rows");
    chroma_b200_attention g{};
    g.tokens = int32_t(q.size(0));
    g.heads = int32_t(q.size(1));
    g.scale = args[6] == Py_None ? 1.0f / std::sqrt(float(p.head_dim)) : float(PyFloat_AsDouble(args[6]));
    if (PyErr_Occurred()) throw python_error();
    g.window = integer(args[7], "window");
    g.first = integer(args[8], "first");
    const bool lse = truth(args[10]);
    const Inputs inputs = {&q, &keys, &tensor(args[2], "values"), sinks};
    check_out(given, inputs);
    if (given) {
        call.with(given);
        TORCH_CHECK_VALUE(given->sizes() == q.sizes() && given->scalar_type() == q.scalar_type(), "out must be ", q.sizes(), " ", q.scalar_type(),
                          ", got ", given->sizes(), " ", given->scalar_type());
    }
    const Tensor out = given ? *given : call.empty(q.sizes(), q.scalar_type());
    TORCH_CHECK_VALUE(q.stride(2) == 1 && out.stride(2) == 1, "a head's row must be contiguous");
    Tensor logs;
    if (lse) {
        logs = call.empty({q.size(0), q.size(1)}, at::kFloat);
        g.lse = logs.data_ptr<float>();
    }
    if (sinks) {
        call.with(sinks);
        TORCH_CHECK_VALUE(sinks->dim() == 1 && sinks->size(0) == g.heads && sinks->is_contiguous() &&
                              (sinks->scalar_type() == q.scalar_type() || sinks->scalar_type() == at::kFloat),
                          "sinks must be contiguous [", g.heads, "] ", q.scalar_type(), " or float32, got ", sinks->sizes(), " ", sinks->scalar_type());
        g.sinks = sinks->const_data_ptr();
        g.sinks_fp32 = sinks->scalar_type() == at::kFloat;
    }
    g.q = q.const_data_ptr();
    g.out = out.data_ptr();
    g.starts = ints(call, starts, int64_t(p.slots) + 1, "starts");
    g.q_strides[0] = q.stride(0), g.q_strides[1] = q.stride(1);
    g.out_strides[0] = out.stride(0), g.out_strides[1] = out.stride(1);
    Tensor room;
    g.workspace_bytes = native.attention_workspace(&p, &g);
    if (g.workspace_bytes > 0) {
        room = call.empty({g.workspace_bytes}, at::kByte);
        g.workspace = room.data_ptr();
    }
    char err[512];
    run(native.paged_attention(&p, &g, call.stream(), err, sizeof err), err);
    if (given) written(out);
    no_gradient("paged_attention", inputs, {&out, &logs});
    return lse ? Py_BuildValue("(NN)", THPVariable_Wrap(out), THPVariable_Wrap(logs)) : THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

PyObject* step_pages(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count_args(n, 7);
    const Tensor &table = tensor(args[0], "table"), &lengths = tensor(args[1], "lengths"), &keys = tensor(args[4], "keys");
    const Call call(keys);
    const auto p = pages_of(call, keys, tensor(args[5], "values"), table, lengths, true);
    const int32_t *parents = ints(call, tensor(args[2], "parents"), p.slots, "parents"), *counts = ints(call, tensor(args[3], "counts"), p.slots, "counts");
    const int64_t room = native.pages_workspace(p.pages, p.slots);
    const Tensor new_table = call.empty({p.slots, p.width}, at::kInt), new_lengths = call.empty({p.slots}, at::kInt), info = call.empty({3}, at::kInt),
                 workspace = call.empty({room}, at::kByte);
    char err[512];
    const bool cut = truth(args[6]);
    run((cut ? native.step_pages : native.step_pages_uncut)(&p, parents, counts, new_table.data_ptr<int32_t>(), new_lengths.data_ptr<int32_t>(), info.data_ptr<int32_t>(),
                          workspace.data_ptr(), room, call.stream(), err, sizeof err), err);
    written(keys), written(tensor(args[5], "values"));
    return Py_BuildValue("(NNN)", THPVariable_Wrap(new_table), THPVariable_Wrap(new_lengths), THPVariable_Wrap(info));
    END_HANDLE_TH_ERRORS
}

PyObject* compact_pages(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count_args(n, 4);
    const Tensor &table = tensor(args[0], "table"), &keys = tensor(args[2], "keys");
    const Call call(keys);
    const auto p = pages_of(call, keys, tensor(args[3], "values"), table, tensor(args[1], "lengths"), true);
    const int64_t room = native.pages_workspace(p.pages, p.slots);
    const Tensor new_table = call.empty({p.slots, p.width}, at::kInt), info = call.empty({2}, at::kInt), workspace = call.empty({room}, at::kByte);
    char err[512];
    run(native.compact_pages(&p, new_table.data_ptr<int32_t>(), info.data_ptr<int32_t>(), workspace.data_ptr(), room, call.stream(), err, sizeof err), err);
    written(keys), written(tensor(args[3], "values"));
    return Py_BuildValue("(NN)", THPVariable_Wrap(new_table), THPVariable_Wrap(info));
    END_HANDLE_TH_ERRORS
}

const float* floats(const Call& call, const Tensor* t, int64_t rows, const char* name) {
    if (!t) return nullptr;
    call.with(t);
    TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat && t->dim() == 1 && t->size(0) == rows && t->is_contiguous(), name, " must be contiguous float32 [",
                      rows, "], got ", t->scalar_type(), " ", t->sizes());
    return t->const_data_ptr<float>();
}

// The row stride of a matrix whose rows are contiguous (rows that are all one row, stride 0, are fine).
int64_t matrix(const Call& call, const Tensor& t, at::ScalarType type, int64_t rows, int64_t cols, const char* name) {
    call.with(t);
    TORCH_CHECK_VALUE(t.scalar_type() == type && t.dim() == 2 && t.size(0) == rows && (cols < 0 || t.size(1) == cols) && (t.stride(1) == 1 || t.size(1) < 2) &&
                          t.size(1) <= INT32_MAX,
                      name, " must be ", type, " [", rows, ", ", cols, "] (-1: any) with contiguous rows, got ", t.scalar_type(), " ", t.sizes());
    return t.stride(0);
}

PyObject* process_logits(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count_args(n, 13);
    static const char* names[13] = {"logits", "history", "lengths", "prompts", "repetition", "presence", "frequency",
                                    "bias_ids", "bias", "mask", "temperature", "out", "argmax"};
    const Tensor& logits = tensor(args[0], names[0]);
    const Tensor* t[12];
    for (int i = 1; i < 12; ++i) t[i] = optional(args[i], names[i]);
    const Tensor *history = t[1], *bias_ids = t[7], *bias = t[8], *mask = t[9], *given = t[11];
    const Call call(logits);
    chroma_b200_logits g{};
    g.storage = storage_of(logits, "logits");
    TORCH_CHECK_VALUE(logits.dim() == 2 && logits.size(1) > 0 && logits.stride(1) == 1 && logits.size(0) <= INT32_MAX && logits.size(1) <= INT32_MAX,
                      "logits must be [rows, vocab] with contiguous rows, got ", logits.sizes());
    const int64_t rows = logits.size(0), vocab = logits.size(1);
    const Inputs inputs = {&logits, t[4], t[5], t[6], bias, t[10]};
    check_out(given, inputs);
    if (given) {
        call.with(given);
        TORCH_CHECK_VALUE(given->sizes() == logits.sizes() && given->scalar_type() == logits.scalar_type() && given->stride(1) == 1 &&
                              (given->stride(0) >= vocab || rows < 2),
                          "out must be ", logits.sizes(), " ", logits.scalar_type(), " with contiguous rows");
    }
    const Tensor out = given ? *given : call.empty(logits.sizes(), logits.scalar_type());
    g.rows = int32_t(rows), g.vocab = int32_t(vocab);
    g.logits = logits.const_data_ptr(), g.out = out.data_ptr();
    g.stride = logits.stride(0), g.out_stride = out.stride(0);
    if (history) {
        TORCH_CHECK_VALUE(t[2], "a history needs its lengths");
        g.history_stride = matrix(call, *history, at::kInt, rows, -1, "history");
        g.history = history->const_data_ptr<int32_t>(), g.width = int32_t(history->size(1));
        g.lengths = ints(call, t[2], rows, "lengths"), g.prompts = ints(call, t[3], rows, "prompts");
    } else {
        TORCH_CHECK_VALUE(!t[4] && !t[5] && !t[6], "penalties need a history");
    }
    g.repetition = floats(call, t[4], rows, names[4]), g.presence = floats(call, t[5], rows, names[5]);
    g.frequency = floats(call, t[6], rows, names[6]), g.temperature = floats(call, t[10], rows, names[10]);
    TORCH_CHECK_VALUE(!bias_ids == !bias, "bias_ids and bias go together");
    if (bias_ids) {
        g.bias_ids_stride = matrix(call, *bias_ids, at::kInt, rows, -1, "bias_ids");
        g.bias_stride = matrix(call, *bias, at::kFloat, rows, bias_ids->size(1), "bias");
        g.biases = int32_t(bias_ids->size(1));
        g.bias_ids = bias_ids->const_data_ptr<int32_t>(), g.bias = bias->const_data_ptr<float>();
    }
    if (mask) {
        g.mask_stride = matrix(call, *mask, at::kInt, rows, (vocab + 31) / 32, "mask");
        g.mask = mask->const_data_ptr<int32_t>();
    }
    Tensor best, room;
    const bool argmax = truth(args[12]);
    if (argmax) {
        best = call.empty({rows}, at::kLong);
        g.argmax = best.data_ptr<int64_t>();
    }
    if (argmax || g.history || g.bias_ids) {
        g.workspace_bytes = native.logits_workspace(g.rows, g.vocab);
        room = call.empty({g.workspace_bytes}, at::kByte);
        g.workspace = room.data_ptr();
    }
    char err[512];
    run(native.process_logits(&g, call.stream(), err, sizeof err), err);
    if (given) written(out);
    no_gradient("process_logits", inputs, {&out});
    // `out` comes back as the object that was given.
    PyObject* result = given ? Py_NewRef(args[11]) : THPVariable_Wrap(out);
    return argmax ? Py_BuildValue("(NN)", result, THPVariable_Wrap(best)) : result;
    END_HANDLE_TH_ERRORS
}

// bind(addresses): the entry points of the native library, in the order of Entries.
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    constexpr int kEntries = sizeof(Entries) / sizeof(void*);
    void* at[kEntries];
    count_args(n, kEntries);
    for (int i = 0; i < kEntries; ++i) {
        at[i] = PyLong_AsVoidPtr(args[i]);
        if (PyErr_Occurred()) throw python_error();
    }
    int i = 0;
#define ENTRY(name) native.name = reinterpret_cast<decltype(native.name)>(at[i++])
    ENTRY(paged_append);
    ENTRY(paged_attention);
    ENTRY(attention_workspace);
    ENTRY(step_pages);
    ENTRY(step_pages_uncut);
    ENTRY(compact_pages);
    ENTRY(pages_workspace);
    ENTRY(process_logits);
    ENTRY(logits_workspace);
#undef ENTRY
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(paged_append), METHOD(paged_attention), METHOD(step_pages), METHOD(compact_pages), METHOD(process_logits),
                         METHOD(bind), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "built_for", BUILT_FOR) < 0) Py_CLEAR(m);
    return m;
}
