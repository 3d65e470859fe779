// tensor_args.cpp — the Python binding's view of torch tensors, in C++: shape, type, device and layout of a tensor and its address in about a tenth of
// a microsecond, and the parameter blocks of flb_kv8.h and of scored attention calls filled from them.  From Python every attribute of a tensor costs that much, and a decode call
// names a dozen tensors: its host time would be that of three kernel launches (8-bit decode: 4.2 us from Python, 1.2 us from here).  Python
// module `_tensor_args`.
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cmath>
#include <cstring>
#include <string>

#include "../../include/flb_attn.h"
#include "../../include/flb_kv8.h"

namespace {

struct Refused {}; // thrown with a Python exception set, caught where Python calls

constexpr at::ScalarType kAnyType = at::ScalarType::Undefined;
constexpr int kAnyDevice = INT_MIN;

template <typename... A> [[noreturn]] void refuse(const char *format, A... a) {
    PyErr_Format(PyExc_ValueError, format, a...);
    throw Refused();
}

// Where a tensor has to be: on this device; `pinned`: or in pinned host memory.
struct Place {
    int dev;
    bool pinned;
    Place(int d, bool p = false) : dev(d), pinned(p) {}
};
const at::Tensor &tensor(PyObject *o, const char *name, Place at) {
    if (!THPVariable_Check(o)) refuse("%s must be a torch tensor", name);
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.device().is_cuda() && !t.device().is_cpu()) refuse("%s must lie in CUDA or host memory", name);
    if (at.dev != kAnyDevice && t.get_device() != at.dev && !(at.pinned && t.device().is_cpu() && t.is_pinned()))
        refuse("%s is on another device (%d) than the cache (%d)", name, (int)t.get_device(), at.dev);
    if (t.layout() != at::kStrided) refuse("%s must be a strided tensor", name);
    return t;
}

const at::Tensor &shaped(PyObject *o, const char *name, at::IntArrayRef shape, at::ScalarType type, Place dev) {
    const at::Tensor &t = tensor(o, name, dev);
    if (t.sizes() != shape || (type != kAnyType && t.scalar_type() != type)) {
        std::string want;
        for (int64_t n : shape) want += (want.empty() ? "" : ",") + std::to_string(n);
        refuse("%s must be a %s tensor of shape [%s]", name, type == kAnyType ? "dense" : c10::toString(type), want.c_str());
    }
    return t;
}

// address of a dense tensor
void *dense(PyObject *o, const char *name, at::IntArrayRef shape, at::ScalarType type, Place dev) {
    const at::Tensor &t = shaped(o, name, shape, type, dev);
    if (!t.is_contiguous()) refuse("%s must be a dense tensor", name);
    return t.data_ptr();
}
template <typename P> P *opt(PyObject *o, const char *name, at::IntArrayRef shape, at::ScalarType type, Place dev) {
    return o == Py_None ? nullptr : static_cast<P *>(dense(o, name, shape, type, dev));
}

int as_int(int64_t n, const char *name) {
    if (n < INT_MIN || n > INT_MAX) refuse("%s is out of range", name);
    return (int)n;
}
int integer(PyObject *o, const char *name) {
    const long long n = PyLong_AsLongLong(o);
    if (n == -1 && PyErr_Occurred()) throw Refused();
    return as_int(n, name);
}
float number(PyObject *o) {
    const double x = PyFloat_AsDouble(o);
    if (x == -1.0 && PyErr_Occurred()) throw Refused();
    return (float)x;
}
int truth(PyObject *o) {
    const int x = PyObject_IsTrue(o);
    if (x < 0) throw Refused();
    return x;
}

// q, k or v [B,S,heads,d]: dense heads, one stride between tokens
void *rows(PyObject *o, const char *name, at::IntArrayRef shape, at::ScalarType type, Place dev, int64_t &row) {
    const at::Tensor &t = shaped(o, name, shape, type, dev);
    if (t.dim() != 4) refuse("%s must be [B,S,heads,d]", name);
    const int64_t B = t.size(0), S = t.size(1), H = t.size(2), d = t.size(3);
    row = H * d;
    if (!t.is_contiguous()) {
        row = S > 1 ? t.stride(1) : (B > 1 ? t.stride(0) : H * d);
        if (t.stride(3) != 1 || (H > 1 && t.stride(2) != d) || (S > 1 && t.stride(1) != row) || (B > 1 && t.stride(0) != S * row) || row < H * d)
            refuse("%s must be [B,S,heads,d] with unit element stride, head stride d and one stride between tokens", name);
    }
    return t.data_ptr();
}
// k and v of the tokens; their stride
int kv_rows(PyObject *ko, PyObject *vo, at::IntArrayRef shape, at::ScalarType type, Place dev, const void *&k, const void *&v) {
    int64_t rk, rv;
    k = rows(ko, "k", shape, type, dev, rk);
    v = rows(vo, "v", shape, type, dev, rv);
    if (rk != rv) refuse("k and v must share one token-row stride");
    return as_int(rk, "the stride of k");
}

int input_mode(const at::Tensor &t) {
    switch (t.scalar_type()) {
    case at::kInt: return FLB_IN_INT32;
    case at::kFloat: return FLB_IN_F32;
    case at::kHalf: return FLB_IN_F16;
    default: refuse("q, k and v must be int32, float32 or float16");
    }
}
// activation scale of int32 inputs, one per token
const float *act_scale(PyObject *o, int64_t tokens, int dev) {
    if (o == Py_None) refuse("int32 inputs need act_scale and the weight scales");
    const at::Tensor &t = tensor(o, "act_scale", dev);
    if (t.numel() != tokens) refuse("act_scale must hold one value per token");
    return static_cast<const float *>(dense(o, "act_scale", t.sizes(), at::kFloat, dev));
}
const float *w_scale(PyObject *o, const char *name, int64_t n, int dev) {
    if (o == Py_None) refuse("int32 inputs need act_scale and the weight scales");
    return static_cast<const float *>(dense(o, name, {n}, at::kFloat, dev));
}
const float *rope(PyObject *o, int64_t d, int dev, int &n) {
    n = 0;
    if (o == Py_None) return nullptr;
    const at::Tensor &t = tensor(o, "freq_cis", dev);
    if (t.dim() != 2 || t.size(0) == 0) refuse("freq_cis must have a row for every position");
    n = as_int(t.size(0), "the length of freq_cis");
    return static_cast<const float *>(dense(o, "freq_cis", {t.size(0), d}, at::kFloat, dev));
}
void *scratch(PyObject *o, int dev, size_t &bytes) {
    bytes = 0;
    if (o == Py_None) return nullptr;
    const at::Tensor &t = tensor(o, "scratch", dev);
    if (!t.is_contiguous()) refuse("scratch must be a dense tensor");
    bytes = t.nbytes();
    return t.data_ptr();
}

// k, v, k_scale, v_scale, row_pos -> the cache block; the index of its device (-1: host memory, for the checks alone)
int cache_of(PyObject *const *a, flb_kv8_cache &c) {
    const at::Tensor &k = tensor(a[0], "k", kAnyDevice), &ks = tensor(a[2], "k_scale", kAnyDevice);
    const at::ScalarType type = k.scalar_type();
    if (k.dim() != 4 || (type != at::kChar && type != at::kFloat8_e4m3fn)) refuse("cache codes must be int8 or float8_e4m3fn tensors [B,Hkv,T,d]");
    const int dev = (int)k.get_device();
    const int64_t B = k.size(0), H = k.size(1), T = k.size(2), n = ks.dim() ? ks.size(-1) : 0;
    if (n <= 0 || T % n) refuse("cache scales must be [B,Hkv,T/block_len]");
    c.batch_size = as_int(B, "the batch");
    c.kv_head_num = as_int(H, "the number of heads");
    c.size_per_head = as_int(k.size(3), "the head size");
    c.total_len = as_int(T, "the cache's length");
    c.block_len = as_int(T / n, "the block");
    c.code_type = type == at::kChar ? FLB_KV8_I8 : FLB_KV8_E4M3;
    c.k_codes = dense(a[0], "k", k.sizes(), type, dev);
    c.v_codes = dense(a[1], "v", k.sizes(), type, dev);
    c.k_scale = static_cast<float *>(dense(a[2], "k_scale", {B, H, n}, at::kFloat, dev));
    c.v_scale = static_cast<float *>(dense(a[3], "v_scale", {B, H, n}, at::kFloat, dev));
    c.row_pos = opt<int>(a[4], "row_pos", {B, H, T}, at::kInt, dev);
    return dev;
}

// f(block) fills a parameter block and gives its device -> (bytes of the block, device)
template <typename Block, int ARGS, typename F> PyObject *block(Py_ssize_t n, F fill) {
    if (n != ARGS) return PyErr_Format(PyExc_TypeError, "expected %d arguments", ARGS);
    Block p;
    memset(&p, 0, sizeof p);
    try {
        const int dev = fill(p);
        PyObject *bytes = PyBytes_FromStringAndSize(reinterpret_cast<const char *>(&p), sizeof p);
        return bytes ? Py_BuildValue("(Ni)", bytes, dev) : nullptr;
    } catch (const Refused &) {
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

PyObject *kv8_append(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return block<flb_kv8_append_params, 16>(n, [a](flb_kv8_append_params &p) {
        const int dev = cache_of(a, p.cache);
        const int64_t B = p.cache.batch_size, H = p.cache.kv_head_num, d = p.cache.size_per_head;
        const at::Tensor &k = tensor(a[5], "k", dev);
        if (k.dim() != 4) refuse("k must be [B,S,heads,d]");
        const int64_t S = k.size(1);
        p.seq_len = as_int(S, "the number of tokens");
        p.input_mode = input_mode(k);
        p.kv_row_stride = kv_rows(a[5], a[6], {B, S, H, d}, k.scalar_type(), dev, p.k, p.v);
        p.start_pos = integer(a[7], "start_pos");
        p.past_lens = opt<int>(a[8], "past_lens", {B}, at::kInt, dev);
        p.new_lens = opt<int>(a[9], "new_lens", {B}, at::kInt, dev);
        p.token_pos = opt<int>(a[10], "token_pos", {B}, at::kInt, dev);
        if (p.input_mode == FLB_IN_INT32) {
            p.act_scale = act_scale(a[11], B * S, dev);
            p.k_w_scale = w_scale(a[12], "k_w_scale", H * d, dev);
            p.v_w_scale = w_scale(a[13], "v_w_scale", H * d, dev);
        }
        p.freq_cis = rope(a[14], d, dev, p.freq_rows);
        size_t bytes;
        p.status = static_cast<unsigned *>(scratch(a[15], dev, bytes));
        if (a[15] != Py_None && bytes < sizeof(unsigned)) refuse("scratch must hold the status word");
        return dev;
    });
}

PyObject *kv8_decode(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return block<flb_kv8_decode_params, 27>(n, [a](flb_kv8_decode_params &p) {
        const int dev = cache_of(a, p.cache);
        const int64_t B = p.cache.batch_size, Hkv = p.cache.kv_head_num, T = p.cache.total_len, d = p.cache.size_per_head;
        const at::Tensor &q = tensor(a[5], "q", dev), &out = tensor(a[8], "out", dev);
        if (q.dim() != 4) refuse("q must be [B,1,heads,d]");
        if (out.scalar_type() != at::kFloat && out.scalar_type() != at::kHalf) refuse("out must be float32 or float16");
        const int64_t Hq = q.size(2);
        int64_t row;
        p.head_num = as_int(Hq, "the number of heads");
        p.input_mode = input_mode(q);
        p.q = rows(a[5], "q", {B, 1, Hq, d}, q.scalar_type(), dev, row);
        p.q_row_stride = as_int(row, "the stride of q");
        p.kv_row_stride = kv_rows(a[6], a[7], {B, 1, Hkv, d}, q.scalar_type(), dev, p.k, p.v);
        p.out = dense(a[8], "out", {B, Hq, 1, d}, out.scalar_type(), dev);
        p.out_dtype = out.scalar_type() == at::kFloat ? FLB_F32 : FLB_F16;
        p.start_pos = integer(a[9], "start_pos");
        p.past_lens = opt<int>(a[10], "past_lens", {B}, at::kInt, dev);
        p.max_past_len = integer(a[11], "max_past_len");
        p.token_pos = opt<int>(a[12], "token_pos", {B}, at::kInt, dev);
        if (p.input_mode == FLB_IN_INT32) {
            p.act_scale = act_scale(a[13], B, dev);
            p.q_w_scale = w_scale(a[14], "q_w_scale", Hq * d, dev);
            p.k_w_scale = w_scale(a[15], "k_w_scale", Hkv * d, dev);
            p.v_w_scale = w_scale(a[16], "v_w_scale", Hkv * d, dev);
        }
        p.freq_cis = rope(a[17], d, dev, p.freq_rows);
        p.softmax_scale = a[18] == Py_None ? (float)(1.0 / std::sqrt((double)d)) : number(a[18]);
        p.softcap = number(a[19]);
        p.alibi_slopes = opt<float>(a[20], "alibi_slopes", {Hq}, at::kFloat, dev);
        p.key_begin = opt<int>(a[21], "key_begin", {B}, at::kInt, dev);
        p.weight_in = opt<float>(a[22], "weight_in", {B, Hkv, T}, at::kFloat, dev);
        p.weight_out = opt<float>(a[23], "weight_out", {B, Hkv, T}, at::kFloat, dev);
        p.scratch = scratch(a[24], dev, p.scratch_bytes);
        p.scratch_zeroed = truth(a[25]);
        p.split_len = integer(a[26], "split_len");
        return dev;
    });
}

PyObject *kv8_evict(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return block<flb_kv8_evict_params, 16>(n, [a](flb_kv8_evict_params &p) {
        const int dev = cache_of(a, p.cache);
        const int64_t B = p.cache.batch_size, H = p.cache.kv_head_num, T = p.cache.total_len;
        p.start_pos = integer(a[5], "start_pos");
        p.past_lens = opt<int>(a[6], "past_lens", {B}, at::kInt, dev);
        p.len_out = static_cast<int *>(dense(a[7], "len_out", {B}, at::kInt, dev));
        p.budget = integer(a[8], "budget");
        p.recent = integer(a[9], "recent");
        p.sinks = integer(a[10], "sinks");
        p.next_pos = opt<int>(a[11], "next_pos", {B}, at::kInt, dev);
        p.weight = static_cast<const float *>(dense(a[12], "weight", {B, H, T}, at::kFloat, dev));
        p.weight_out = static_cast<float *>(dense(a[13], "weight_out", {B, H, T}, at::kFloat, dev));
        p.pos_out = static_cast<int *>(dense(a[14], "pos_out", {B, H, T}, at::kInt, dev));
        p.scratch = scratch(a[15], dev, p.scratch_bytes);
        return dev;
    });
}

// A dense tensor of so many elements, in whatever shape; null for None
template <typename P> P *flat(PyObject *o, const char *name, at::ScalarType type, int64_t n, Place dev) {
    if (o == Py_None) return nullptr;
    const at::Tensor &t = tensor(o, name, dev);
    if (t.scalar_type() != type || !t.is_contiguous()) refuse("%s must be a dense %s tensor", name, c10::toString(type));
    if (n >= 0 && t.numel() != n) refuse("%s must hold %lld elements", name, (long long)n);
    return static_cast<P *>(t.data_ptr());
}
int dtype_of(const at::Tensor &t) {
    if (t.scalar_type() != at::kFloat && t.scalar_type() != at::kHalf) refuse("caches and out must be float32 or float16");
    return t.scalar_type() == at::kFloat ? FLB_F32 : FLB_F16;
}

// The blocks of flb_attn.h with a score form.  What a call can read and write has to be there: host memory is left for the checks alone (the
// cache there too), or, pinned, for what a decode call may read from and write to it.
PyObject *scored(PyObject *, PyObject *const *a, Py_ssize_t n) {
    flb_score_form f;
    memset(&f, 0, sizeof f);
    PyObject *first = block<flb_attn_params, 30>(n, [a, &f](flb_attn_params &p) {
        const at::Tensor &kc = tensor(a[3], "k_cache", kAnyDevice);
        const int dev = (int)kc.get_device();
        const at::Tensor &q = tensor(a[0], "q", kAnyDevice), &k = tensor(a[1], "k", kAnyDevice), &out = tensor(a[5], "out", kAnyDevice);
        if (q.dim() != 4 || k.dim() != 4 || kc.dim() != 4) refuse("q and k must be [B,S,heads,d], k_cache [B,Hkv,T,d]");
        const int64_t B = q.size(0), S = q.size(1), H = q.size(2), d = q.size(3), Hkv = k.size(2), T = kc.size(2);
        const Place near(dev, S == 1);
        if (Hkv <= 0 || H % Hkv) refuse("the number of K/V heads must divide that of the q heads");
        p.batch_size = as_int(B, "the batch");
        p.head_num = as_int(H, "the number of heads");
        p.size_per_head = as_int(d, "the head size");
        p.seq_len = as_int(S, "the number of tokens");
        p.total_len = as_int(T, "the cache's length");
        p.input_mode = input_mode(q);
        int64_t row;
        p.q = rows(a[0], "q", q.sizes(), q.scalar_type(), near, row);
        p.qkv_row_stride = row == H * d ? 0 : as_int(row, "the stride of q");
        f.kv_head_num = as_int(Hkv, "the number of K/V heads");
        f.kv_row_stride = kv_rows(a[1], a[2], {B, S, Hkv, d}, q.scalar_type(), near, p.k, p.v);
        p.cache_dtype = dtype_of(kc);
        p.k_cache = dense(a[3], "k_cache", {B, Hkv, T, d}, kc.scalar_type(), dev);
        p.v_cache = dense(a[4], "v_cache", {B, Hkv, T, d}, kc.scalar_type(), dev);
        p.out_dtype = dtype_of(out);
        p.out = dense(a[5], "out", {B, H, S, d}, out.scalar_type(), near);
        f.softcap = number(a[6]);
        f.alibi_slopes = opt<float>(a[7], "alibi_slopes", {H}, at::kFloat, near);
        const int64_t bounds[2] = {B, S};
        const at::IntArrayRef bound_shape(bounds, S == 1 ? 1 : 2);
        f.key_begin = opt<int>(a[8], "key_begin", bound_shape, at::kInt, near);
        f.key_end = opt<int>(a[9], "key_end", bound_shape, at::kInt, near);
        p.scratch = scratch(a[10], dev, p.scratch_bytes);
        p.start_pos = integer(a[11], "start_pos");
        p.past_lens = opt<int>(a[12], "past_lens", {B}, at::kInt, near);
        p.max_past_len = integer(a[13], "max_past_len");
        const bool scaled = p.input_mode == FLB_IN_INT32; // the scales are read
        p.act_scale = flat<float>(a[14], "act_scale", at::kFloat, scaled ? B * S : -1, near);
        p.q_w_scale = flat<float>(a[15], "q_w_scale", at::kFloat, scaled ? H * d : -1, near);
        p.k_w_scale = flat<float>(a[16], "k_w_scale", at::kFloat, scaled ? Hkv * d : -1, near);
        p.v_w_scale = flat<float>(a[17], "v_w_scale", at::kFloat, scaled ? Hkv * d : -1, near);
        p.freq_cis = flat<float>(a[18], "freq_cis", at::kFloat, -1, near);
        p.rope_pos0 = integer(a[19], "rope_pos0");
        p.rope_add_past = truth(a[20]);
        // rows that the call can reach: of a prompt its own, else up to the host's bound on the cached ones
        const int64_t most = S > 1 ? S - 1 : !p.past_lens ? p.start_pos : p.max_past_len > 0 ? p.max_past_len : T - 1;
        const int64_t last = (int64_t)p.rope_pos0 + (S > 1 || p.rope_add_past ? most : 0);
        if (a[18] != Py_None && d > 0 && THPVariable_Unpack(a[18]).numel() / d <= last) refuse("freq_cis must have a row of the head size for every position up to %lld", (long long)last);
        p.mask_mode = integer(a[21], "mask_mode");
        p.attn_mask = flat<float>(a[22], "attn_mask", at::kFloat, -1, near);
        p.mask_row_stride = integer(a[23], "mask_row_stride");
        if (a[22] != Py_None && !p.mask_row_stride) p.mask_row_stride = as_int(THPVariable_Unpack(a[22]).size(-1), "the mask's row");
        if (a[22] != Py_None && p.mask_mode == FLB_MASK_GENERIC && THPVariable_Unpack(a[22]).numel() <= most * p.mask_row_stride + most)
            refuse("attn_mask must have rows and columns for every position up to %lld", (long long)most);
        p.softmax_scale = a[24] == Py_None ? (float)(1.0 / std::sqrt((double)d)) : number(a[24]);
        p.scratch_zeroed = truth(a[25]);
        p.split_len = integer(a[26], "split_len");
        p.out_q8 = flat<int8_t>(a[27], "out_q8", at::kChar, B * S * H * d, near);
        p.out_q8_scale = flat<float>(a[28], "out_q8_scale", at::kFloat, B * S, near);
        p.early_start = integer(a[29], "early_start");
        return dev;
    });
    if (!first) return nullptr;
    PyObject *bytes = PyBytes_FromStringAndSize(reinterpret_cast<const char *>(&f), sizeof f);
    PyObject *both = bytes ? Py_BuildValue("(ONO)", PyTuple_GET_ITEM(first, 0), bytes, PyTuple_GET_ITEM(first, 1)) : nullptr;
    Py_DECREF(first);
    return both;
}

using Fast = PyObject *(*)(PyObject *, PyObject *const *, Py_ssize_t);
PyCFunction fast(Fast f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }

PyMethodDef methods[] = {
    {"kv8_append", fast(kv8_append), METH_FASTCALL, "parameter block of an append, and its device"},
    {"kv8_decode", fast(kv8_decode), METH_FASTCALL, "parameter block of a decode, and its device"},
    {"kv8_evict", fast(kv8_evict), METH_FASTCALL, "parameter block of an eviction, and its device"},
    {"scored", fast(scored), METH_FASTCALL, "parameter block and score form of an attention call, and their device"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_args", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

} // namespace

PyMODINIT_FUNC PyInit__tensor_args(void) {
    // what a tensor looks like in memory is torch's own affair, of one version
    PyObject *torch = PyImport_ImportModule("torch"), *version = torch ? PyObject_GetAttrString(torch, "__version__") : nullptr, *text = version ? PyObject_Str(version) : nullptr;
    const char *is = text ? PyUnicode_AsUTF8(text) : nullptr;
    const bool same = is && !strcmp(is, FLB_BUILT_FOR_TORCH);
    if (is && !same) PyErr_Format(PyExc_ImportError, "_tensor_args was built for torch " FLB_BUILT_FOR_TORCH ", this is %s: run python -m fasterllama_b200.build", is);
    Py_XDECREF(text);
    Py_XDECREF(version);
    Py_XDECREF(torch);
    return same ? PyModule_Create(&module) : nullptr;
}
