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

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <memory>
#include <string>
#include <vector>

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

// Axes of pairs: None, or a sequence of whole numbers, and positions [axes, tokens] then.
struct AxesView : fklhip_axes {
    bool given = false;
};
AxesView axes_of(PyObject* o, int64_t pairs) {
    AxesView x{};
    if (none(o)) return x;
    PyObject* items = PySequence_Fast(o, "axes has to be a sequence of whole numbers");
    if (!items) throw python_error();
    const std::unique_ptr<PyObject, void (*)(PyObject*)> held(items, [](PyObject* p) { Py_DECREF(p); });
    if (PySequence_Fast_GET_SIZE(items) != pairs || pairs > 128) refuse("axes has to have an axis for each of " + std::to_string(pairs) + " pairs, up to 128");
    for (int64_t i = 0; i < pairs; ++i) {
        const int64_t axis = whole(PySequence_Fast_GET_ITEM(items, i));
        if (axis < 0 || axis > 3) refuse("an axis has to be 0 to 3");
        x.of_pair[i] = uint8_t(axis);
    }
    x.given = true;
    return x;
}

// q, k, q_weight, k_weight, cos, sin, positions, eps, pairs; axes
AxesView heads_of(PyObject* const* a, PyObject* of_pairs, fklhip_heads& h) {
    AxesView axes{};
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
        axes = axes_of(of_pairs, cos.size(1));
        const Tensor& positions = tensor(a[6], "positions");
        if (axes.given) {
            if (positions.dim() != 2 || positions.size(0) < 1 || positions.size(0) > 4) refuse("positions has to be [axes, tokens] with axes, of 1 to 4");
            axes.count = int32_t(positions.size(0));
            axes.stride = tokens;
            h.positions = static_cast<const int32_t*>(plain(positions, "positions", at::kInt, {positions.size(0), tokens}, q.device()));
        } else {
            h.positions = static_cast<const int32_t*>(plain(positions, "positions", at::kInt, {tokens}, q.device()));
        }
    } else if (!none(of_pairs)) {
        refuse("axes without cos and sin");
    }
    h.eps = float(number(a[7]));
    h.pairs = PyObject_IsTrue(a[8]);
    return axes;
}

// ..., q_out, k_out, axes
PyObject* qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 12);
    at::AutoDispatchBelowAutograd quick;
    fklhip_heads h{};
    const AxesView axes = heads_of(a, a[11], h);
    const Tensor &q = THPVariable_Unpack(a[0]), &k = THPVariable_Unpack(a[1]);
    void* stream = stream_of(q, "q");
    const Tensor q_out = output(a[9], "q_out", q.sizes(), q.scalar_type(), q.device()), k_out = output(a[10], "k_out", k.sizes(), q.scalar_type(), q.device());
    h.q_out = rows(q_out, "q_out", h.tokens, h.q_heads, h.head_dim, q);
    h.k_out = rows(k_out, "k_out", h.tokens, h.kv_heads, h.head_dim, q);
    check(axes.given ? fklhip_qk_norm_rope_axes(&h, &axes, stream) : fklhip_qk_norm_rope(&h, stream), "qk_norm_rope");
    PyObject* both = PyTuple_New(2);
    if (!both) throw python_error();
    PyTuple_SET_ITEM(both, 0, result(a[9], q_out));
    PyTuple_SET_ITEM(both, 1, result(a[10], k_out));
    return both;
    END_HANDLE_TH_ERRORS
}

// ..., v, slots, cache, q_out, axes
PyObject* qkv_to_cache(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 14);
    at::AutoDispatchBelowAutograd quick;
    fklhip_heads h{};
    const AxesView axes = heads_of(a, a[13], h);
    const Tensor& q = THPVariable_Unpack(a[0]);
    const CacheView c = cache_of(a[11]);
    on_device(q, "q", c);
    void* stream = stream_of(q, "q");
    h.v = rows(tensor(a[9], "v"), "v", h.tokens, h.kv_heads, h.head_dim, q);
    h.slots = static_cast<const int32_t*>(plain(tensor(a[10], "slots"), "slots", at::kInt, {h.tokens}, q.device()));
    const Tensor q_out = output(a[12], "q_out", q.sizes(), q.scalar_type(), q.device());
    h.q_out = rows(q_out, "q_out", h.tokens, h.q_heads, h.head_dim, q);
    check(axes.given ? fklhip_qkv_to_cache_axes(&h, &axes, &c.c, stream) : fklhip_qkv_to_cache(&h, &c.c, stream), "qkv_to_cache");
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

// q, cache, page_table, context, q_start, max_new, max_context, mask, scale, out, lse; cap, slopes, positions, first, prefix
PyObject* tree_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 16);
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
    fklhip_scores h{};
    const bool shaped = !none(a[11]) || !none(a[12]) || !none(a[14]) || !none(a[15]);
    if (!none(a[11])) {
        h.cap = float(number(a[11]));
        if (!(h.cap > 0.0f)) refuse("cap has to be above 0, or None");
    }
    if (!none(a[12])) h.slopes = static_cast<const float*>(plain(tensor(a[12], "slopes"), "slopes", at::kFloat, {heads}, q.device()));
    const auto of_rows = [&](PyObject* o, const char* name, int64_t n) { return none(o) ? nullptr : static_cast<const int32_t*>(plain(tensor(o, name), name, at::kInt, {n}, q.device())); };
    h.positions = of_rows(a[13], "positions", tokens);
    h.first = of_rows(a[14], "first", tokens);
    h.prefix = of_rows(a[15], "prefix", table.size(0));
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
    check(shaped ? fklhip_shaped_attention(&f, &h, &c.c, stream) : fklhip_tree_attention(&f, &c.c, stream), "tree_attention");
    if (tokens != 0 && (f.batch == 0 || f.max_new == 0)) {     // (nothing was launched)
        Tensor(out).zero_();
        if (!none(a[10])) Tensor(THPVariable_Unpack(a[10])).fill_(-HUGE_VAL);
    }
    if (!none(a[10])) written(THPVariable_Unpack(a[10]));
    return result(a[9], out);
    END_HANDLE_TH_ERRORS
}

// ---- a step's tables --------------------------------------------------------------------------------------------------

int32_t* ints(PyObject* o, const char* name, at::IntArrayRef shape, c10::Device device) { return static_cast<int32_t*>(plain(tensor(o, name), name, at::kInt, shape, device)); }
// Several small results in one allocation, each a tensor of its own behind the last: one takes 0.9 us, a tensor of what is there 0.15.
class Block {
    int64_t m_bytes = 0;
    Tensor m_block;
public:
    // where `count` elements of a type will be (16-byte pieces)
    int64_t room(int64_t count, int64_t size) {
        const int64_t at = m_bytes;
        m_bytes += (count * size + 15) / 16 * 16;
        return at;
    }
    void allocate(c10::Device device) { m_block = empty({m_bytes}, at::kByte, device); }
    void* data(int64_t at) const { return static_cast<char*>(m_block.data_ptr()) + at; }
    Tensor tensor(int64_t at, at::ScalarType type, at::IntArrayRef shape) const {
        auto impl = c10::make_intrusive<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(m_block.storage()), m_block.key_set(), c10::scalarTypeToTypeMeta(type));
        impl->set_storage_offset(at / int64_t(c10::elementSize(type)));
        impl->set_sizes_contiguous(shape);
        return Tensor(std::move(impl));
    }
};
PyObject* tuple_of(std::initializer_list<const Tensor*> tensors) {
    PyObject* all = PyTuple_New(Py_ssize_t(tensors.size()));
    if (!all) throw python_error();
    Py_ssize_t i = 0;
    for (const Tensor* t : tensors) {
        PyObject* o = Py_None;
        if (t) o = THPVariable_Wrap(*t);
        else Py_INCREF(o);
        PyTuple_SET_ITEM(all, i++, o);
    }
    return all;
}

// page_table, held, context, new, free, available, page_tokens, tokens, max_new, parents
PyObject* step_tables(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 10);
    at::AutoDispatchBelowAutograd quick;
    const Tensor &table = tensor(a[0], "page_table"), &free = tensor(a[4], "free");
    if (table.dim() != 2 || table.size(0) > 65535) refuse("page_table has to be [batch, pages of a sequence], batch up to 65535");
    if (free.dim() != 1) refuse("free has to have one dimension");
    void* stream = stream_of(table, "page_table");
    const c10::Device device = table.device();
    const int64_t batch = table.size(0), tokens = whole(a[7]);
    if (tokens < 0 || tokens >= int64_t(1) << 30) refuse("tokens has to be 0 or more, below 2^30");
    fklhip_tables t{};
    t.page_table = ints(a[0], "page_table", table.sizes(), device);
    t.held = ints(a[1], "held", {batch}, device);
    t.context = ints(a[2], "context", {batch}, device);
    t.fresh = ints(a[3], "new", {batch}, device);
    t.free_pages = ints(a[4], "free", free.sizes(), device);
    t.available = ints(a[5], "available", {1}, device);
    t.page_table_stride = table.size(1); t.free_count = free.size(0); t.tokens = tokens; t.batch = int32_t(batch);
    t.page_tokens = whole32(a[6], "page_tokens");
    t.max_new = whole32(a[8], "max_new");
    const bool trees = !none(a[9]);
    if (trees) t.parents = ints(a[9], "parents", {tokens}, device);
    if (t.max_new < 0) refuse("max_new has to be 0 or more");
    t.mask_words = trees ? std::max(1, int32_t((int64_t(t.max_new) + 63) / 64)) : 0;
    if (trees && int64_t(t.mask_words) * tokens >= int64_t(1) << 31) refuse("masks of more than 2^31 words");
    Block block;
    const int64_t at_mask = block.room(trees ? tokens * t.mask_words : 0, 8), at_start = block.room(batch + 1, 4), at_slots = block.room(tokens, 4), at_positions = block.room(tokens, 4),
                  at_held = block.room(batch, 4), at_left = block.room(1, 4);
    block.allocate(device);
    t.q_start = static_cast<int32_t*>(block.data(at_start)); t.slots = static_cast<int32_t*>(block.data(at_slots)); t.positions = static_cast<int32_t*>(block.data(at_positions));
    t.held_out = static_cast<int32_t*>(block.data(at_held)); t.left = static_cast<int32_t*>(block.data(at_left));
    if (trees) t.mask = static_cast<uint64_t*>(block.data(at_mask));
    check(fklhip_step_tables(&t, stream), "step_tables");
    written(table);
    const Tensor q_start = block.tensor(at_start, at::kInt, {batch + 1}), slots = block.tensor(at_slots, at::kInt, {tokens}), positions = block.tensor(at_positions, at::kInt, {tokens}),
                 held = block.tensor(at_held, at::kInt, {batch}), left = block.tensor(at_left, at::kInt, {1}), mask = trees ? block.tensor(at_mask, at::kLong, {tokens, t.mask_words}) : Tensor();
    return tuple_of({&q_start, &slots, &positions, &held, &left, trees ? &mask : nullptr});
    END_HANDLE_TH_ERRORS
}

// target, tokens, q_start, uniforms, max_new, draft, parents
PyObject* verify_drafts(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 7);
    at::AutoDispatchBelowAutograd quick;
    const Tensor &target = tensor(a[0], "target"), &q_start = tensor(a[2], "q_start");
    fklhip_drafts d{};
    if (target.dim() != 2 || target.size(1) < 1 || target.size(1) > 1 << 24) refuse("target has to be [tokens, vocabulary], of 1 to 2^24");
    if (q_start.dim() != 1 || q_start.size(0) < 1 || q_start.size(0) > 65536) refuse("q_start has to be [batch + 1], batch up to 65535");
    d.type = target.scalar_type() == at::kFloat ? FKLHIP_F32 : target.scalar_type() == at::kBFloat16 ? FKLHIP_BF16 : target.scalar_type() == at::kHalf ? FKLHIP_F16 : -1;
    if (d.type < 0) refuse("target has to be torch.float32, torch.bfloat16 or torch.float16");
    void* stream = stream_of(target, "target");
    const c10::Device device = target.device();
    const int64_t tokens = target.size(0), vocab = target.size(1), batch = q_start.size(0) - 1;
    const auto table = [&](const Tensor& t, const char* name, int64_t& stride) -> const void* {
        if (t.dim() != 2 || t.size(0) != tokens || t.size(1) != vocab || t.scalar_type() != target.scalar_type() || t.device() != device || (vocab > 1 && t.stride(1) != 1))
            refuse(std::string(name) + " has to be " + shape_text({tokens, vocab}) + " of " + c10::toString(target.scalar_type()) + " on " + device.str() + " with a tight last dimension");
        serves(t, name);
        holds(t, name);
        stride = t.stride(0);
        return t.data_ptr();
    };
    d.target = table(target, "target", d.target_stride);
    d.ids = ints(a[1], "tokens", {tokens}, device);
    d.q_start = ints(a[2], "q_start", {batch + 1}, device);
    d.uniforms = static_cast<const float*>(plain(tensor(a[3], "uniforms"), "uniforms", at::kFloat, {tokens}, device));
    d.max_new = whole32(a[4], "max_new");
    if (d.max_new < 0 || d.max_new > 1024) refuse("max_new has to be up to 1024");
    if (!none(a[5])) d.draft = table(tensor(a[5], "draft"), "draft", d.draft_stride);
    if (!none(a[6])) d.parents = ints(a[6], "parents", {tokens}, device);
    if (!none(a[5]) && !none(a[6])) refuse("draft's probabilities are of chains: not with parents");
    d.tokens = tokens; d.batch = int32_t(batch); d.vocab = int32_t(vocab);
    uint64_t bytes = 0;
    check(fklhip_verify_drafts_workspace(&d, &bytes), "verify_drafts");
    // (a small workspace is in the results' allocation; a large one is given back to torch's allocator, in the stream's order, on return)
    const bool small = bytes <= 1 << 18;
    Block block;
    const int64_t at_path = block.room(batch * d.max_new, 4), at_count = block.room(batch, 4), at_out = block.room(batch * d.max_new, 4), at_work = block.room(small ? int64_t(bytes) : 0, 1);
    block.allocate(device);
    d.path = static_cast<int32_t*>(block.data(at_path)); d.count = static_cast<int32_t*>(block.data(at_count)); d.out = static_cast<int32_t*>(block.data(at_out));
    Tensor workspace;
    if (bytes) {
        if (!small) workspace = empty({int64_t(bytes)}, at::kByte, device);
        d.workspace = small ? block.data(at_work) : workspace.data_ptr();
        d.workspace_bytes = bytes;
    }
    check(fklhip_verify_drafts(&d, stream), "verify_drafts");
    const Tensor path = block.tensor(at_path, at::kInt, {batch, d.max_new}), count = block.tensor(at_count, at::kInt, {batch}), out = block.tensor(at_out, at::kInt, {batch, d.max_new});
    if (batch != 0 && d.max_new == 0) Tensor(count).zero_();   // (nothing was launched)
    return tuple_of({&path, &count, &out});
    END_HANDLE_TH_ERRORS
}

// caches (a tuple of their tensors), page_table, context, path, count
PyObject* kv_keep(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 5);
    if (!PyTuple_Check(a[0])) refuse("not caches");
    const Py_ssize_t layers = PyTuple_GET_SIZE(a[0]);
    if (layers > 1024) refuse("more than 1024 caches");
    const Tensor &table = tensor(a[1], "page_table"), &path = tensor(a[3], "path");
    if (table.dim() != 2 || table.size(0) > 65535) refuse("page_table has to be [batch, pages of a sequence], batch up to 65535");
    if (path.dim() != 2 || path.size(1) > 1 << 20) refuse("path has to be [batch, max_new], max_new up to 2^20");
    void* stream = stream_of(table, "page_table");
    const c10::Device device = table.device();
    const int64_t batch = table.size(0);
    std::vector<fklhip_kv_cache> caches;
    caches.reserve(size_t(layers));
    for (Py_ssize_t i = 0; i < layers; ++i) {
        const CacheView c = cache_of(PyTuple_GET_ITEM(a[0], i));
        on_device(table, "page_table", c);
        caches.push_back(c.c);
    }
    const int32_t *t = ints(a[1], "page_table", table.sizes(), device), *context = ints(a[2], "context", {batch}, device), *p = ints(a[3], "path", {batch, path.size(1)}, device),
                  *count = ints(a[4], "count", {batch}, device);
    check(fklhip_kv_keep(caches.data(), int32_t(layers), t, table.size(1), context, p, count, int32_t(batch), int32_t(path.size(1)), stream), "kv_keep");
    for (Py_ssize_t i = 0; i < layers; ++i) written(PyTuple_GET_ITEM(a[0], i));
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
#define FUNCTION(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
    FUNCTION(check_cache), FUNCTION(qk_norm_rope), FUNCTION(qkv_to_cache), FUNCTION(kv_write), FUNCTION(kv_read), FUNCTION(tree_attention), FUNCTION(step_tables), FUNCTION(verify_drafts), FUNCTION(kv_keep),
#undef FUNCTION
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_attention", "Calls of fusedkernellibrary_amd.attention", -1, methods, nullptr, nullptr, nullptr, nullptr};

} // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__attention() { return PyModule_Create(&module); }
