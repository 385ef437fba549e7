// torch_binding.cpp -- the operators of include/fklhip.h on torch tensors: the module fusedkernellibrary_amd._attention, whose
// functions fusedkernellibrary_amd/attention.py documents and calls with all their arguments in order.
//
// A serving step makes a handful of calls of a few microseconds each, and reading some thirty fields of tensors takes longer in
// Python than a small kernel runs; here a call is checked, its outputs are allocated and its kernels are launched in about
// two microseconds. Shapes, types and places of tensors are checked here, everything else by the C ABI.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/TracerMode.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>

#include <fklhip.h>

#include <cmath>
#include <string>

namespace {

using at::Tensor;

[[noreturn]] void refuse(const std::string& what) {
    PyErr_SetString(PyExc_ValueError, what.c_str());
    throw python_error();
}

const Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(std::string(name) + " has to be a tensor");
    return THPVariable_Unpack(o);
}
int type_of(const Tensor& t, const char* name) {
    if (t.scalar_type() == at::kBFloat16) return FKLHIP_BF16;
    if (t.scalar_type() == at::kHalf) return FKLHIP_F16;
    refuse(std::string(name) + " has to be torch.bfloat16 or torch.float16");
}
std::string shape_text(at::IntArrayRef s) {
    std::string t = "[";
    for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
    return t + "]";
}
// The current stream of a tensor's device, which has to be the current one: kernels are launched on that.
void* stream_of(const Tensor& t, const char* name) {
    if (!t.is_cuda()) refuse(std::string(name) + " has to be on a GPU");
    if (t.device().index() != c10::hip::current_device()) refuse(std::string(name) + " is on a device that is not the current one");
    return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}
// A storage may have been resized to less than its tensor needs (such tensors exist between a sharded model's steps).
void holds(const Tensor& t, const char* name) {
    int64_t last = t.storage_offset();
    for (int64_t i = 0; i < t.dim(); ++i) {
        if (t.size(i) == 0) return;
        last += (t.size(i) - 1) * t.stride(i);
    }
    if (int64_t(t.storage().nbytes() / t.element_size()) <= last) refuse(std::string(name) + "'s storage is smaller than the tensor");
}
// A gradient or a tangent would be lost without a word.
void serves(const Tensor& t, const char* name) {
    if (t.requires_grad() && at::GradMode::is_enabled()) refuse(std::string(name) + " asks for a gradient, which these operators do not have (torch.no_grad())");
    if (t._fw_grad(0).defined()) refuse(std::string(name) + " carries a forward-mode tangent, which these operators do not have");
}
fklhip_rows rows(const Tensor& t, const char* name, int64_t tokens, int64_t heads, int64_t dim, const Tensor& like) {
    if (t.dim() != 3 || t.size(0) != tokens || t.size(1) != heads || t.size(2) != dim || t.scalar_type() != like.scalar_type() || t.device() != like.device() ||
        (dim > 1 && t.stride(2) != 1))
        refuse(std::string(name) + " has to be " + shape_text({tokens, heads, dim}) + " of " + c10::toString(like.scalar_type()) + " on " + like.device().str() +
               " with a tight last dimension, not " + shape_text(t.sizes()) + " of " + c10::toString(t.scalar_type()) + " on " + t.device().str());
    serves(t, name);
    holds(t, name);
    return {t.data_ptr(), t.stride(0), t.stride(1)};
}
// A contiguous tensor of one type and shape on a device.
void* plain(const Tensor& t, const char* name, at::ScalarType type, at::IntArrayRef shape, c10::Device device) {
    if (t.scalar_type() != type || t.sizes() != shape || t.device() != device || !t.is_contiguous())
        refuse(std::string(name) + " has to be " + shape_text(shape) + " of " + c10::toString(type) + " on " + device.str() + ", contiguous");
    serves(t, name);
    holds(t, name);
    return t.data_ptr();
}
bool none(PyObject* o) { return o == Py_None; }
Tensor empty(at::IntArrayRef shape, at::ScalarType type, c10::Device device) { return at::empty(shape, at::TensorOptions().dtype(type).device(device)); }
// What was given, or a new one.
Tensor output(PyObject* o, const char* name, at::IntArrayRef shape, at::ScalarType type, c10::Device device) {
    return none(o) ? empty(shape, type, device) : tensor(o, name);
}
// What a call wrote to and the caller had before: autograd finds out by the version whether a tensor that it saved still is what it was.
void written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
// `given`, or a Python object of the tensor that was allocated.
PyObject* result(PyObject* given, const Tensor& t) {
    if (none(given)) return THPVariable_Wrap(t);
    written(t);
    Py_INCREF(given);
    return given;
}
void check(int rc, const char* what) {
    if (rc == FKLHIP_OK) return;
    if (rc == FKLHIP_EINVAL) {
        const char* text = "";
        fklhip_argument_error(&text);
        refuse(std::string(what) + ": " + text);
    }
    throw std::runtime_error(std::string("GPU Error: ") + fklhip_error_string(rc) + " (" + what + ", code " + std::to_string(rc) + ")");
}
int64_t whole(PyObject* o) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}
int32_t whole32(PyObject* o, const char* name) {
    const int64_t v = whole(o);
    if (v != int32_t(v)) refuse(std::string(name) + " is out of range");
    return int32_t(v);
}
double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}
// What every call begins with. The calls are no operators of torch's dispatcher: a tracer would record their outputs as they
// happened to be, or as empty tensors.
void expect(Py_ssize_t have, Py_ssize_t want) {
    if (at::tracer::impl::is_dispatch_enabled() ||
        (c10::impl::TorchDispatchModeTLS::any_modes_set() && c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY)))
        refuse("a tracer cannot record this call");
    if (have != want) refuse("called with " + std::to_string(have) + " arguments and not " + std::to_string(want));
}

// ---- caches: (k, v, k_scale, v_scale), read anew by every call ---------------------------------------------------------

// The description is of what the tensors are at the call: one that got other memory since the last call (through set_ or .data,
// or because its storage was resized) is taken, or refused, as it is now.
struct CacheView {
    fklhip_kv_cache c;
    int device;
};
CacheView cache_of(PyObject* o) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) refuse("not a cache's tensors");
    const Tensor &k = tensor(PyTuple_GET_ITEM(o, 0), "k"), &v = tensor(PyTuple_GET_ITEM(o, 1), "v"), &ks = tensor(PyTuple_GET_ITEM(o, 2), "k_scale"), &vs = tensor(PyTuple_GET_ITEM(o, 3), "v_scale");
    const bool int8 = k.scalar_type() == at::kChar;
    if (k.dim() != 4 || !(int8 || k.scalar_type() == at::kFloat8_e4m3fn))
        refuse("k has to be [pages, kv_heads, page_tokens, head_dim] of torch.int8 or torch.float8_e4m3fn");
    if (!k.is_cuda()) refuse("k has to be on a GPU");
    const int64_t pages = k.size(0), heads = k.size(1), page = k.size(2), dim = k.size(3);
    const c10::Device device = k.device();
    CacheView b{};
    b.c.k = plain(k, "k", k.scalar_type(), {pages, heads, page, dim}, device);
    b.c.v = plain(v, "v", k.scalar_type(), {pages, heads, page / 4, dim, 4}, device);
    b.c.k_scale = static_cast<float*>(plain(ks, "k_scale", at::kFloat, {pages, heads, page}, device));
    b.c.v_scale = static_cast<float*>(plain(vs, "v_scale", at::kFloat, {pages, heads, page}, device));
    if (heads > 65535 || page > 65535 || dim > 65535) refuse("a cache's heads, pages or rows are too large");
    b.c.pages = pages; b.c.kv_heads = int32_t(heads); b.c.page_tokens = int32_t(page); b.c.head_dim = int32_t(dim);
    b.c.codes = int8 ? FKLHIP_CODES_INT8 : FKLHIP_CODES_E4M3;
    b.device = device.index();
    return b;
}
void written(PyObject* cache) {
    for (Py_ssize_t i = 0; i < 4; ++i) written(THPVariable_Unpack(PyTuple_GET_ITEM(cache, i)));
}
// The check that a cache gets when it is made.
PyObject* check_cache(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 1);
    const CacheView c = cache_of(a[0]);
    check(fklhip_kv_read(&c.c, nullptr, 0, nullptr, nullptr, FKLHIP_BF16, nullptr), "KvCache");      // (of no tokens: looks at the cache alone)
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}
void on_device(const Tensor& t, const char* name, const CacheView& c) {
    if (!t.is_cuda() || t.device().index() != c.device) refuse(std::string(name) + " is on another device than the cache");
}

// ---- heads ------------------------------------------------------------------------------------------------------------

// q, k, q_weight, k_weight, cos, sin, positions, eps, pairs
void heads_of(PyObject* const* a, fklhip_heads& h) {
    const Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k");
    if (q.dim() != 3 || k.dim() != 3) refuse("q and k have to be [tokens, heads, head_dim]");
    h.type = type_of(q, "q");
    const int64_t tokens = q.size(0), dim = q.size(2);
    h.tokens = tokens;
    if (q.size(1) > 65535 || k.size(1) > 65535 || dim > 65535) refuse("too many heads, or heads that are too large");
    h.q_heads = int32_t(q.size(1)); h.kv_heads = int32_t(k.size(1)); h.head_dim = int32_t(dim);
    h.q = rows(q, "q", tokens, h.q_heads, dim, q);
    h.k = rows(k, "k", tokens, h.kv_heads, dim, q);
    if (none(a[2]) != none(a[3])) refuse("weights for both of q and k, or for none");
    if (!none(a[2])) {
        h.q_weight = plain(tensor(a[2], "q_weight"), "q_weight", q.scalar_type(), {dim}, q.device());
        h.k_weight = plain(tensor(a[3], "k_weight"), "k_weight", q.scalar_type(), {dim}, q.device());
    }
    if (none(a[4]) != none(a[5])) refuse("cos and sin, or neither");
    if (!none(a[4])) {
        const Tensor& cos = tensor(a[4], "cos");
        if (cos.dim() != 2 || cos.size(1) > dim) refuse("cos and sin have to be [positions, rotated / 2]");
        h.table_rows = cos.size(0);
        h.rot_dim = int32_t(2 * cos.size(1));
        h.cos = static_cast<const float*>(plain(cos, "cos", at::kFloat, cos.sizes(), q.device()));
        h.sin = static_cast<const float*>(plain(tensor(a[5], "sin"), "sin", at::kFloat, cos.sizes(), q.device()));
        h.positions = static_cast<const int32_t*>(plain(tensor(a[6], "positions"), "positions", at::kInt, {tokens}, q.device()));
    }
    h.eps = float(number(a[7]));
    h.pairs = PyObject_IsTrue(a[8]);
}

// ..., q_out, k_out
PyObject* qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 11);
    at::AutoDispatchBelowAutograd quick;
    fklhip_heads h{};
    heads_of(a, h);
    const Tensor &q = THPVariable_Unpack(a[0]), &k = THPVariable_Unpack(a[1]);
    void* stream = stream_of(q, "q");
    const Tensor q_out = output(a[9], "q_out", q.sizes(), q.scalar_type(), q.device()), k_out = output(a[10], "k_out", k.sizes(), q.scalar_type(), q.device());
    h.q_out = rows(q_out, "q_out", h.tokens, h.q_heads, h.head_dim, q);
    h.k_out = rows(k_out, "k_out", h.tokens, h.kv_heads, h.head_dim, q);
    check(fklhip_qk_norm_rope(&h, stream), "qk_norm_rope");
    PyObject* both = PyTuple_New(2);
    if (!both) throw python_error();
    PyTuple_SET_ITEM(both, 0, result(a[9], q_out));
    PyTuple_SET_ITEM(both, 1, result(a[10], k_out));
    return both;
    END_HANDLE_TH_ERRORS
}

// ..., v, slots, cache, q_out
PyObject* qkv_to_cache(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 13);
    at::AutoDispatchBelowAutograd quick;
    fklhip_heads h{};
    heads_of(a, h);
    const Tensor& q = THPVariable_Unpack(a[0]);
    const CacheView c = cache_of(a[11]);
    on_device(q, "q", c);
    void* stream = stream_of(q, "q");
    h.v = rows(tensor(a[9], "v"), "v", h.tokens, h.kv_heads, h.head_dim, q);
    h.slots = static_cast<const int32_t*>(plain(tensor(a[10], "slots"), "slots", at::kInt, {h.tokens}, q.device()));
    const Tensor q_out = output(a[12], "q_out", q.sizes(), q.scalar_type(), q.device());
    h.q_out = rows(q_out, "q_out", h.tokens, h.q_heads, h.head_dim, q);
    check(fklhip_qkv_to_cache(&h, &c.c, stream), "qkv_to_cache");
    written(a[11]);
    return result(a[12], q_out);
    END_HANDLE_TH_ERRORS
}

// ---- cache ------------------------------------------------------------------------------------------------------------

// cache, k, v, slots
PyObject* kv_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 4);
    const CacheView c = cache_of(a[0]);
    const Tensor &k = tensor(a[1], "k"), &v = tensor(a[2], "v"), &slots = tensor(a[3], "slots");
    if (k.dim() != 3) refuse("k has to be [tokens, kv_heads, head_dim]");
    on_device(k, "k", c);
    const int type = type_of(k, "k");
    const int64_t tokens = k.size(0);
    const fklhip_rows kr = rows(k, "k", tokens, c.c.kv_heads, c.c.head_dim, k), vr = rows(v, "v", tokens, c.c.kv_heads, c.c.head_dim, k);
    const auto* s = static_cast<const int32_t*>(plain(slots, "slots", at::kInt, {tokens}, k.device()));
    check(fklhip_kv_write(&c.c, &kr, &vr, s, tokens, type, stream_of(k, "k")), "kv_write");
    written(a[0]);
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// cache, slots, half precision or not, k_out, v_out
PyObject* kv_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 5);
    at::AutoDispatchBelowAutograd quick;
    const CacheView c = cache_of(a[0]);
    const Tensor& slots = tensor(a[1], "slots");
    on_device(slots, "slots", c);
    if (slots.dim() != 1) refuse("slots has to have one dimension");
    const int64_t tokens = slots.size(0);
    const auto* s = static_cast<const int32_t*>(plain(slots, "slots", at::kInt, {tokens}, slots.device()));
    const at::ScalarType type = PyObject_IsTrue(a[2]) ? at::kHalf : at::kBFloat16;
    const int64_t shape[3] = {tokens, c.c.kv_heads, c.c.head_dim};
    const Tensor k = output(a[3], "k_out", shape, type, slots.device()), v = output(a[4], "v_out", shape, type, slots.device());
    if (k.scalar_type() != type) refuse("k_out has to be of the type asked for");
    on_device(k, "k_out", c);
    const fklhip_rows kr = rows(k, "k_out", tokens, shape[1], shape[2], k), vr = rows(v, "v_out", tokens, shape[1], shape[2], k);
    check(fklhip_kv_read(&c.c, s, tokens, &kr, &vr, type == at::kHalf ? FKLHIP_F16 : FKLHIP_BF16, stream_of(slots, "slots")), "kv_read");
    PyObject* both = PyTuple_New(2);
    if (!both) throw python_error();
    PyTuple_SET_ITEM(both, 0, result(a[3], k));
    PyTuple_SET_ITEM(both, 1, result(a[4], v));
    return both;
    END_HANDLE_TH_ERRORS
}

// ---- attention --------------------------------------------------------------------------------------------------------

// q, cache, page_table, context, q_start, max_new, max_context, mask, scale, out, lse
PyObject* tree_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 11);
    at::AutoDispatchBelowAutograd quick;
    const Tensor& q = tensor(a[0], "q");
    const CacheView c = cache_of(a[1]);
    const Tensor& table = tensor(a[2], "page_table");
    fklhip_attention f{};
    if (q.dim() != 3) refuse("q has to be [tokens, q_heads, head_dim]");
    f.type = type_of(q, "q");
    on_device(q, "q", c);
    const int64_t tokens = q.size(0), heads = q.size(1), dim = q.size(2);
    if (dim != c.c.head_dim) refuse("q and the cache have heads of different sizes");
    if (heads > 65535) refuse("too many heads");
    if (table.dim() != 2 || table.size(0) > 65535) refuse("page_table has to be [batch, pages of a sequence], batch up to 65535");
    f.tokens = tokens; f.q_heads = int32_t(heads); f.batch = int32_t(table.size(0)); f.page_table_stride = table.size(1);
    f.q = rows(q, "q", tokens, heads, dim, q);
    f.page_table = static_cast<const int32_t*>(plain(table, "page_table", at::kInt, table.sizes(), q.device()));
    f.context = static_cast<const int32_t*>(plain(tensor(a[3], "context"), "context", at::kInt, {table.size(0)}, q.device()));
    f.q_start = static_cast<const int32_t*>(plain(tensor(a[4], "q_start"), "q_start", at::kInt, {table.size(0) + 1}, q.device()));
    f.max_new = whole32(a[5], "max_new");
    f.max_context = whole32(a[6], "max_context");
    if (!none(a[7])) {
        const Tensor& mask = tensor(a[7], "mask");
        if (mask.dim() != 2 || mask.size(1) > 1 << 20) refuse("mask has to be [tokens, words]");
        f.mask = static_cast<const uint64_t*>(plain(mask, "mask", at::kLong, {tokens, mask.size(1)}, q.device()));
        f.mask_words = int32_t(mask.size(1));
        if (f.mask == nullptr && tokens != 0) refuse("mask has to have a word at least");
    }
    f.scale = none(a[8]) ? float(1.0 / std::sqrt(double(dim))) : float(number(a[8]));
    void* stream = stream_of(q, "q");
    const Tensor out = output(a[9], "out", q.sizes(), q.scalar_type(), q.device());
    f.out = rows(out, "out", tokens, heads, dim, q);
    if (!none(a[10])) f.lse = static_cast<float*>(plain(tensor(a[10], "lse"), "lse", at::kFloat, {tokens, heads}, q.device()));
    uint64_t bytes = 0;
    check(fklhip_tree_attention_workspace(&f, &c.c, &bytes), "tree_attention");
    Tensor workspace;                                          // (given back to torch's allocator, in the stream's order, on return)
    if (bytes) {
        workspace = empty({int64_t(bytes)}, at::kByte, q.device());
        f.workspace = workspace.data_ptr();
        f.workspace_bytes = bytes;
    }
    check(fklhip_tree_attention(&f, &c.c, stream), "tree_attention");
    if (tokens != 0 && (f.batch == 0 || f.max_new == 0)) {     // (nothing was launched)
        Tensor(out).zero_();
        if (!none(a[10])) Tensor(THPVariable_Unpack(a[10])).fill_(-HUGE_VAL);
    }
    if (!none(a[10])) written(THPVariable_Unpack(a[10]));
    return result(a[9], out);
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
#define FUNCTION(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
    FUNCTION(check_cache), FUNCTION(qk_norm_rope), FUNCTION(qkv_to_cache), FUNCTION(kv_write), FUNCTION(kv_read), FUNCTION(tree_attention),
#undef FUNCTION
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_attention", "Calls of fusedkernellibrary_amd.attention", -1, methods, nullptr, nullptr, nullptr, nullptr};

} // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__attention() { return PyModule_Create(&module); }
