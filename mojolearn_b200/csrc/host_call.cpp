// The host side of calls on device tensors, in native code: torch_ops.product without bias, activation or `out`, and paged.append and
// paged.attention.
//
// The checks, allocations and argument conversions of a one-row product take 15.5 us of host time a call in Python and ctypes and
// 6.5 here, on the tensors themselves, with output and workspace from torch's allocator and the C ABI called directly. A loop of
// int8 [768, 768] rows went from 15.3 to 6.4 us a call. One of [11008, 4096] rows takes 16.4 either way, also when it is queued
// behind other work: a 14.5 us kernel (graph replay) and what the device leaves between two plain launches.
//
// It takes the plain case only: exact torch tensors (no subclass, no functorch or python-dispatch wrapper) of the storage
// types, contiguous, on the current device, extents that agree, no torch mode active. For anything else it returns None and the
// caller's Python path decides, so refusals keep their exceptions and messages.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <cstdint>
#include <map>

namespace {

constexpr int64_t OP_NN = 0, OP_NT = 1, OP_TN = 2, W_F32 = 0, W_BF16 = 1, W_INT8_EXP = 2, W_INT8_SCALE = 3, PLAN_AUTO = -1;
constexpr int64_t ERR_CAP = 512;

using GemmFn = int64_t (*)(int64_t, void *, float *, const float *, const void *, const void *, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t,
                           void *, int64_t, char *, int64_t);
using NeedFn = int64_t (*)(int64_t, int64_t, int64_t, int64_t, int64_t);
GemmFn g_gemm = nullptr;      // b200i_gemm_w_plan
NeedFn g_auto_need = nullptr; // b200i_product_workspace_bytes
NeedFn g_plan_need = nullptr; // b200i_plan_workspace_bytes
using AppendFn = int64_t (*)(int64_t, void *, void *, void *, void *, const void *, const void *, const void *, int64_t, int64_t, int64_t, int64_t, int64_t, const float *,
                             const float *, int64_t, int64_t, const float *, const float *, double, int64_t, const int32_t *, const int32_t *, const int32_t *, int64_t, int64_t,
                             int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, char *, int64_t);
using AttendFn = int64_t (*)(int64_t, void *, void *, const void *, int64_t, const void *, const void *, int64_t, int64_t, const int32_t *, const int32_t *, const int32_t *, int64_t,
                             int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, double, int64_t, double, void *, int64_t, char *, int64_t);
using AttendNeedFn = int64_t (*)(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t);
AppendFn g_append = nullptr;            // b200i_paged_append
AttendFn g_attend = nullptr;            // b200i_paged_attention
AttendNeedFn g_attend_need = nullptr;   // b200i_paged_attention_workspace_bytes
PyObject *g_error = nullptr;  // the package's exception for a refusal

// Workspace sizes by the call's form: a pure function of it and of the device's SM count. Reached with the GIL held; bounded.
std::map<std::array<int64_t, 8>, int64_t> g_need;
constexpr size_t MAX_NEEDS = 4096;

bool plain(PyObject *o, at::Tensor &t, bool contiguous = true) {
    if (!THPVariable_CheckExact(o)) return false;
    t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided) return false;
    const c10::DispatchKeySet keys = t.key_set();
    if (keys.has(c10::DispatchKey::FuncTorchBatched) || keys.has(c10::DispatchKey::FuncTorchGradWrapper) || keys.has(c10::DispatchKey::Batched) ||
        keys.has(c10::DispatchKey::Python) || keys.has(c10::DispatchKey::Negative) || keys.has(c10::DispatchKey::Functionalize) || keys.has(c10::DispatchKey::ZeroTensor))
        return false;
    return t.has_storage() && (!contiguous || t.is_contiguous());
}

PyObject *bind(PyObject *, PyObject *args) {
    unsigned long long gemm, auto_need, plan_need, append, attend, attend_need;
    PyObject *error;
    if (!PyArg_ParseTuple(args, "KKKKKKO", &gemm, &auto_need, &plan_need, &append, &attend, &attend_need, &error)) return nullptr;
    g_append = reinterpret_cast<AppendFn>(static_cast<uintptr_t>(append));
    g_attend = reinterpret_cast<AttendFn>(static_cast<uintptr_t>(attend));
    g_attend_need = reinterpret_cast<AttendNeedFn>(static_cast<uintptr_t>(attend_need));
    g_gemm = reinterpret_cast<GemmFn>(static_cast<uintptr_t>(gemm));
    g_auto_need = reinterpret_cast<NeedFn>(static_cast<uintptr_t>(auto_need));
    g_plan_need = reinterpret_cast<NeedFn>(static_cast<uintptr_t>(plan_need));
    Py_XINCREF(error);
    Py_XDECREF(g_error);
    g_error = error;
    g_need.clear();
    Py_RETURN_NONE;
}

// product(a, b, bscale or None, wkind, op, plan, group_leaves) -> the output tensor, or None where this is not the plain case
PyObject *product(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    // (a torch mode wants to see the allocations)
    if (nargs != 7 || !g_gemm || c10::impl::TorchDispatchModeTLS::any_modes_set() || at::impl::PythonTorchFunctionTLS::stack_len() > 0) Py_RETURN_NONE;
    int64_t v[4];
    for (int i = 0; i < 4; i++) {
        if (!PyLong_Check(args[3 + i])) Py_RETURN_NONE;
        v[i] = PyLong_AsLongLong(args[3 + i]);
        if (v[i] == -1 && PyErr_Occurred()) {
            PyErr_Clear();
            Py_RETURN_NONE;
        }
    }
    const int64_t wkind = v[0], op = v[1], plan = v[2], group_leaves = v[3];
    at::Tensor a, b, scale;
    if (!plain(args[0], a) || !plain(args[1], b) || a.dim() != 2 || b.dim() != 2 || a.scalar_type() != at::kFloat) Py_RETURN_NONE;
    const at::ScalarType stored = b.scalar_type();
    const bool int8 = wkind == W_INT8_EXP || wkind == W_INT8_SCALE;
    if (wkind == W_F32 ? stored != at::kFloat
                       : (wkind == W_BF16 ? stored != at::kUInt16 && stored != at::kShort && stored != at::kBFloat16 : !int8 || stored != at::kChar))
        Py_RETURN_NONE;
    const int64_t k = op == OP_TN ? a.size(0) : a.size(1), m = op == OP_TN ? a.size(1) : a.size(0);
    const int64_t n = op == OP_NT ? b.size(0) : b.size(1), k2 = op == OP_NT ? b.size(1) : b.size(0);
    if ((op != OP_NN && op != OP_NT && op != OP_TN) || k != k2 || m <= 0 || n <= 0 || k <= 0) Py_RETURN_NONE;
    if (int8 != (args[2] != Py_None)) Py_RETURN_NONE;
    if (int8 && (!plain(args[2], scale) || scale.scalar_type() != (wkind == W_INT8_EXP ? at::kInt : at::kFloat) || scale.dim() != 1 || scale.size(0) != n ||
                 scale.device() != a.device()))
        Py_RETURN_NONE;
    const c10::Device dev = a.device();
    if (b.device() != dev || c10::cuda::current_device() != dev.index()) Py_RETURN_NONE;

    const std::array<int64_t, 8> form{dev.index(), m, n, k, op, wkind, plan, group_leaves};
    auto found = g_need.find(form);
    if (found == g_need.end()) {
        if (g_need.size() >= MAX_NEEDS) g_need.clear();
        found = g_need.emplace(form, plan == PLAN_AUTO ? g_auto_need(m, n, k, op, wkind) : g_plan_need(m, n, k, plan, group_leaves)).first;
    }
    const int64_t need = found->second;
    at::Tensor out = at::empty({m, n}, a.options().requires_grad(false)), ws;
    if (need > 0) ws = at::empty({need < 16 ? 16 : need}, a.options().requires_grad(false).dtype(at::kByte));
    char message[ERR_CAP] = "";
    int64_t status;
    Py_BEGIN_ALLOW_THREADS;
    status = g_gemm(dev.index(), c10::cuda::getCurrentCUDAStream(dev.index()).stream(), static_cast<float *>(out.data_ptr()),
                    static_cast<const float *>(a.const_data_ptr()), b.const_data_ptr(), int8 ? scale.const_data_ptr() : nullptr, wkind, m, n, k, op, plan, group_leaves,
                    need > 0 ? ws.data_ptr() : nullptr, need, message, ERR_CAP);
    Py_END_ALLOW_THREADS;
    if (status != 0) {
        PyErr_SetString(g_error, message[0] ? message : "b200i_gemm_w_plan failed");
        return nullptr;
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// ---- the paged cache ----

bool modes() { return c10::impl::TorchDispatchModeTLS::any_modes_set() || at::impl::PythonTorchFunctionTLS::stack_len() > 0; }

// What the two calls share. Each part is false where the call is not a plain one, which the Python path then looks at.
struct Pages {
    at::Tensor k, v, table, cu, lengths;
    int64_t batch = 0, pages = 0, kv = 0, page = 0, hd = 0, type = 0;
    bool read(PyObject *const *args, c10::Device dev) { // k_cache, v_cache, page_table, cu, lengths
        if (!plain(args[0], k) || !plain(args[1], v) || !plain(args[2], table) || !plain(args[3], cu) || !plain(args[4], lengths)) return false;
        if (k.dim() != 4 || v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type() || (k.scalar_type() != at::kFloat && k.scalar_type() != at::kBFloat16)) return false;
        if (table.scalar_type() != at::kInt || cu.scalar_type() != at::kInt || lengths.scalar_type() != at::kInt || table.dim() != 2 || cu.dim() != 1 || lengths.dim() != 1) return false;
        batch = lengths.size(0), pages = k.size(0), kv = k.size(1), page = k.size(2), hd = k.size(3), type = k.scalar_type() == at::kBFloat16;
        return table.size(0) == batch && cu.size(0) == batch + 1 && k.device() == dev && v.device() == dev && table.device() == dev && cu.device() == dev && lengths.device() == dev;
    }
};
// Rows [total, heads, hd] whose heads stand side by side.
bool rows_of(PyObject *o, at::Tensor &t, int64_t *heads, int64_t hd, int64_t total, int64_t *ld) {
    if (!plain(o, t, false) || t.dim() != 3 || t.size(2) != hd || (total >= 0 && t.size(0) != total)) return false;
    *heads = t.size(1);
    if (t.stride(2) != 1 || (t.size(1) > 1 && t.stride(1) != hd)) return false;
    *ld = t.size(0) > 1 ? t.stride(0) : t.size(1) * hd;
    return true;
}
bool vector_of(PyObject *o, at::Tensor &t, int64_t n, c10::Device dev, const float **at) {
    *at = nullptr;
    if (o == Py_None) return true;
    if (!plain(o, t) || t.scalar_type() != at::kFloat || t.dim() != 1 || t.size(0) != n || t.device() != dev) return false;
    *at = static_cast<const float *>(t.const_data_ptr());
    return true;
}
bool integer(PyObject *o, int64_t *v) {
    if (!PyLong_CheckExact(o)) return false;
    *v = PyLong_AsLongLong(o);
    if (*v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}
bool real(PyObject *o, double *v) {
    if (!PyFloat_CheckExact(o)) return false;
    *v = PyFloat_AS_DOUBLE(o);
    return true;
}
PyObject *refusal(const char *message, const char *otherwise) {
    PyErr_SetString(g_error, message[0] ? message : otherwise);
    return nullptr;
}

// paged_append(q, k, v, k_cache, v_cache, page_table, cu, lengths, cos, sin, q_norm, k_norm, eps, norm kind) -> the rotated queries, or None
PyObject *paged_append(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 14 || !g_append || modes()) Py_RETURN_NONE;
    at::Tensor q, k, v, cos, sin, wq, wk;
    if (!plain(args[0], q, false) || q.dim() != 3 || (q.scalar_type() != at::kFloat && q.scalar_type() != at::kBFloat16)) Py_RETURN_NONE;
    const c10::Device dev = q.device();
    Pages c;
    if (!c.read(args + 3, dev) || c10::cuda::current_device() != dev.index()) Py_RETURN_NONE;
    int64_t heads, kv1, kv2, ldq, ldk, ldv, kind, half = 0, positions = 0;
    double eps;
    const int64_t rows = q.size(0), type = q.scalar_type() == at::kBFloat16;
    if (!rows_of(args[0], q, &heads, c.hd, rows, &ldq) || !rows_of(args[1], k, &kv1, c.hd, rows, &ldk) || !rows_of(args[2], v, &kv2, c.hd, rows, &ldv) || kv1 != c.kv || kv2 != c.kv ||
        k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() || k.device() != dev || v.device() != dev || rows == 0)
        Py_RETURN_NONE;
    const float *pcos = nullptr, *psin = nullptr, *pq, *pk;
    if ((args[8] == Py_None) != (args[9] == Py_None)) Py_RETURN_NONE;
    if (args[8] != Py_None) {
        if (!plain(args[8], cos) || !plain(args[9], sin) || cos.scalar_type() != at::kFloat || sin.scalar_type() != at::kFloat || cos.dim() != 2 || sin.sizes() != cos.sizes() ||
            cos.device() != dev || sin.device() != dev)
            Py_RETURN_NONE;
        positions = cos.size(0), half = cos.size(1);
        if (half < 1 || 2 * half > c.hd) Py_RETURN_NONE;
        pcos = static_cast<const float *>(cos.const_data_ptr()), psin = static_cast<const float *>(sin.const_data_ptr());
    }
    if (!vector_of(args[10], wq, c.hd, dev, &pq) || !vector_of(args[11], wk, c.hd, dev, &pk) || !real(args[12], &eps) || !integer(args[13], &kind)) Py_RETURN_NONE;
    at::Tensor out = at::empty(q.sizes(), q.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
    // written, so storage that is shared until then (a lazy clone) becomes this tensor's own, before addresses into it are taken
    void *const k_cache = c.k.mutable_data_ptr(), *const v_cache = c.v.mutable_data_ptr();
    char message[ERR_CAP] = "";
    int64_t status;
    Py_BEGIN_ALLOW_THREADS;
    status = g_append(dev.index(), c10::cuda::getCurrentCUDAStream(dev.index()).stream(), out.data_ptr(), k_cache, v_cache, q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), ldq, ldk, ldv, type, c.type, pcos, psin, 2 * half, positions, pq, pk, eps,
                      kind, static_cast<const int32_t *>(c.table.const_data_ptr()), static_cast<const int32_t *>(c.cu.const_data_ptr()), static_cast<const int32_t *>(c.lengths.const_data_ptr()),
                      rows, c.batch, heads, c.kv, c.hd, c.pages, c.page, c.table.size(1), message, ERR_CAP);
    Py_END_ALLOW_THREADS;
    if (status != 0) return refusal(message, "b200i_paged_append failed");
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// paged_attention(q, k_cache, v_cache, page_table, cu, lengths, max_new, max_length, scale, window, softcap) -> the output, or None
PyObject *paged_attention(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 11 || !g_attend || !g_attend_need || modes()) Py_RETURN_NONE;
    at::Tensor q;
    if (!plain(args[0], q, false) || q.dim() != 3 || (q.scalar_type() != at::kFloat && q.scalar_type() != at::kBFloat16)) Py_RETURN_NONE;
    const c10::Device dev = q.device();
    Pages c;
    if (!c.read(args + 1, dev) || c10::cuda::current_device() != dev.index()) Py_RETURN_NONE;
    int64_t heads, ldq, max_new, max_length, window;
    double scale, softcap;
    const int64_t rows = q.size(0), type = q.scalar_type() == at::kBFloat16;
    if (type > c.type || !rows_of(args[0], q, &heads, c.hd, rows, &ldq) || rows == 0) Py_RETURN_NONE;
    if (!integer(args[6], &max_new) || !integer(args[7], &max_length) || !real(args[8], &scale) || !integer(args[9], &window) || !real(args[10], &softcap)) Py_RETURN_NONE;
    const int64_t need = g_attend_need(dev.index(), type, c.type, rows, c.batch, heads, c.kv, c.hd, max_new, max_length, window);
    at::Tensor out = at::empty(q.sizes(), q.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous)), ws;
    if (need > 0) ws = at::empty({need}, q.options().requires_grad(false).dtype(at::kByte));
    char message[ERR_CAP] = "";
    int64_t status;
    Py_BEGIN_ALLOW_THREADS;
    status = g_attend(dev.index(), c10::cuda::getCurrentCUDAStream(dev.index()).stream(), out.data_ptr(), q.const_data_ptr(), ldq, c.k.const_data_ptr(), c.v.const_data_ptr(), type, c.type,
                      static_cast<const int32_t *>(c.table.const_data_ptr()), static_cast<const int32_t *>(c.cu.const_data_ptr()), static_cast<const int32_t *>(c.lengths.const_data_ptr()), rows,
                      c.batch, heads, c.kv, c.hd, c.pages, c.page, c.table.size(1), max_new, max_length, scale, window, softcap, need > 0 ? ws.data_ptr() : nullptr, need, message, ERR_CAP);
    Py_END_ALLOW_THREADS;
    if (status != 0) return refusal(message, "b200i_paged_attention failed");
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

PyMethodDef METHODS[] = {{"bind", bind, METH_VARARGS, "addresses of the C entry points, and the exception of a refusal"},
                         {"product", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(product)), METH_FASTCALL, "a product of plain device tensors, or None"},
                         {"paged_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paged_append)), METH_FASTCALL, "rows into a paged cache, or None"},
                         {"paged_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paged_attention)), METH_FASTCALL, "attention over a paged cache, or None"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef MODULE = {PyModuleDef_HEAD_INIT, "_host_call", "native host side of a product call", -1, METHODS, nullptr, nullptr, nullptr, nullptr};

} // namespace

// BUILT_FOR, of the compiler's command line: the versions of torch and Python whose headers this was compiled with. The package
// does not use a module of others.
PyMODINIT_FUNC PyInit__host_call() {
    PyObject *m = PyModule_Create(&MODULE);
    if (m && PyModule_AddStringConstant(m, "BUILT_FOR", BUILT_FOR) < 0) Py_CLEAR(m);
    return m;
}
