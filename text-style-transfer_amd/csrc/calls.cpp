// The prompted-decoding calls from Python, checked and issued natively: _tst_calls, an extension module beside libtst_hip.so.
//
// These kernels take a few microseconds, and a decode loop outside this package makes several such calls per token.  Asking a tensor for
// its type, shape, strides, device and address costs about 0.8 us in Python and a foreign call with 17 arguments 1.3; here both are field
// accesses.  Host time per call, checks included, against the same checks in Python over ctypes: page plan 4.4 us (8.2), attention over the
// cache 4.9 (8.2), rules on logits 4.4 (10.3), prompt attention 4.2 (8.3); most of what is left is the launch itself.
//
// Contains no GPU code and no arithmetic: every function checks its arguments, asks for torch's current device and stream, and calls the
// entry point of libtst_hip.so whose address bind() was given (whichever build of the library the process loaded).
#include "tst_hip.h"
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>
#include <stdarg.h>
#include <stdio.h>
#include <cmath>
#include <exception>

namespace {

struct Refused {};   // thrown with a Python exception set

[[noreturn]] void refuse(PyObject* type, const char* format, ...) {
    char text[512];
    va_list list;
    va_start(list, format);
    vsnprintf(text, sizeof text, format, list);
    va_end(list);
    PyErr_SetString(type, text);
    throw Refused();
}

PyObject *device_fn = nullptr, *stream_fn = nullptr, *error_type = nullptr;

#define TST_CALLS(X)                                                                                                                       \
    X(tst_last_error) X(tst_attn_prompt_f32) X(tst_attn_prompt_bf16) X(tst_page_plan) X(tst_page_step) X(tst_cache4_write_f32)             \
    X(tst_cache4_write_bf16) X(tst_cache4_read_f32) X(tst_cache4_read_bf16) X(tst_attn_cache4_f32) X(tst_attn_cache4_bf16)                 \
    X(tst_adjust_logits_f32) X(tst_adjust_logits_bf16) X(tst_grammar_next)
struct Entries {
#define X(name) decltype(&::name) name;
    TST_CALLS(X)
#undef X
} entry;

int64_t as_int(PyObject* o, const char* name) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse(PyExc_TypeError, "%s must be an integer", name);
    }
    return v;
}
int64_t current_device() {
    PyObject* o = PyObject_CallNoArgs(device_fn);
    if (o == nullptr) throw Refused();
    const int64_t v = PyLong_AsLongLong(o);
    Py_DECREF(o);
    return v;
}
void* current_stream(int64_t dev) {
    PyObject* n = PyLong_FromLongLong(dev);
    PyObject* o = n != nullptr ? PyObject_CallOneArg(stream_fn, n) : nullptr;
    Py_XDECREF(n);
    if (o == nullptr) throw Refused();
    void* v = PyLong_AsVoidPtr(o);
    Py_DECREF(o);
    return v;
}
const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s must be a tensor", name);
    return THPVariable_Unpack(o);
}
int64_t where(const at::Tensor& t) { return t.is_cuda() ? t.get_device() : -1; }
[[noreturn]] void wrong_tensor(const at::Tensor& t, const char* name, const char* what) {
    char shape[128];
    int at = 0;
    shape[0] = 0;
    for (int64_t i = 0; i < t.dim() && at < 100; ++i) at += snprintf(shape + at, sizeof shape - at, "%s%lld", i ? ", " : "", (long long)t.size(i));
    refuse(PyExc_ValueError, "%s must be a %s on the current GPU, got %s (%s) on %s", name, what, c10::toString(t.scalar_type()), shape, t.device().str().c_str());
}

const at::ScalarType I32 = at::kInt, F32 = at::kFloat, BF16 = at::kBFloat16;

// a 2-D view whose rows the kernels can read 16 bytes at a time
struct Rows {
    char* p;
    int64_t ld;
};
Rows rows2d(const at::Tensor& t, at::ScalarType type, int64_t dev, int64_t n_rows, int64_t n_cols, const char* name) {
    if (t.scalar_type() != type || t.dim() != 2 || where(t) != dev || (t.stride(1) != 1 && t.size(1) > 1))
        wrong_tensor(t, name, type == F32 ? "2-D torch.float32 tensor with unit inner stride" : "2-D torch.bfloat16 tensor with unit inner stride");
    if (t.size(0) < n_rows || t.size(1) < n_cols)
        refuse(PyExc_ValueError, "%s must hold [%lld, %lld], got (%lld, %lld)", name, (long long)n_rows, (long long)n_cols, (long long)t.size(0), (long long)t.size(1));
    const int64_t unit = type == F32 ? 4 : 8;
    int64_t ld = t.stride(0);
    if (n_rows <= 1) ld = ((ld > n_cols ? ld : n_cols) + unit - 1) / unit * unit;
    else if (ld < n_cols || ld % unit != 0)
        refuse(PyExc_ValueError, "rows of %s must not overlap and start at multiples of %d elements (16 bytes)", name, (int)unit);
    char* p = static_cast<char*>(t.data_ptr());
    if (reinterpret_cast<uintptr_t>(p) & 15) refuse(PyExc_ValueError, "%s must start at a 16-byte boundary", name);
    return {p, ld};
}
// a 1-D int32 tensor of at least n entries (None: a null pointer)
int32_t* ints(PyObject* o, int64_t n, int64_t dev, const char* name, int64_t* have = nullptr) {
    if (o == Py_None) return nullptr;
    const at::Tensor& t = tensor(o, name);
    if (t.scalar_type() != I32 || t.dim() != 1 || t.numel() < n || where(t) != dev || !t.is_contiguous()) {
        char what[64];
        snprintf(what, sizeof what, "contiguous int32 tensor [%lld]", (long long)n);
        wrong_tensor(t, name, what);
    }
    if (have != nullptr) *have = t.numel();
    return static_cast<int32_t*>(t.data_ptr());
}
int32_t* given_ints(PyObject* o, int64_t n, int64_t dev, const char* name, int64_t* have) {
    tensor(o, name);
    return ints(o, n, dev, name, have);
}
struct Table {
    int32_t* p;
    int64_t rows, width;
};
Table table2d(PyObject* o, int64_t dev, const char* name) {
    const at::Tensor& t = tensor(o, name);
    if (t.scalar_type() != I32 || t.dim() != 2 || where(t) != dev || !t.is_contiguous()) wrong_tensor(t, name, "contiguous 2-D int32 tensor");
    return {static_cast<int32_t*>(t.data_ptr()), t.size(0), t.size(1)};
}
// raises if the first n_rows rows of two views share a byte's range
void disjoint(const char* a, int64_t lda, const char* b, int64_t ldb, int64_t n_rows, int64_t cols_a, int64_t cols_b, int64_t size, const char* what) {
    if (n_rows > 0 && a < b + ((n_rows - 1) * ldb + cols_b) * size && b < a + ((n_rows - 1) * lda + cols_a) * size)
        refuse(PyExc_ValueError, "%s", what);
}
bool is_bf16(const at::Tensor& t, const char* what) {
    if (t.scalar_type() != BF16 && t.scalar_type() != F32) refuse(PyExc_ValueError, "%s must be fp32 or bf16", what);
    return t.scalar_type() == BF16;
}
float scale_or(PyObject* o, int64_t dh) {
    if (o == Py_None) return (float)(1.0 / std::sqrt((double)dh));
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Refused();
    return (float)v;
}
const tst_cache4* cache_at(PyObject* o) { return static_cast<const tst_cache4*>(PyLong_AsVoidPtr(o)); }

void done(int rc, const char* name) {
    if (rc == TST_OK) return;
    char text[640];
    snprintf(text, sizeof text, "%s failed (%d): %s", name, rc, entry.tst_last_error());
    PyErr_SetString(error_type, text);
    throw Refused();
}
// the entry point runs without the interpreter's lock, as a foreign call would
template <typename F, typename... A>
void issue(const char* name, F f, A... a) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f(a...);
    Py_END_ALLOW_THREADS
    done(rc, name);
}

// q, k, v, cu, out, heads, kv_heads, scale
void attn_prompt(PyObject* const* a) {
    const at::Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k"), &v = tensor(a[2], "v"), &out = tensor(a[4], "out");
    const int64_t heads = as_int(a[5], "heads"), kv_heads = a[6] == Py_None ? heads : as_int(a[6], "kv_heads"), dev = current_device();
    const bool low = is_bf16(q, "q");
    if (q.dim() != 2 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || q.size(1) % heads != 0)
        refuse(PyExc_ValueError, "q must be [tokens, heads * head size], heads a multiple of kv_heads");
    const int64_t N = q.size(0), wq = q.size(1), dh = wq / heads, wk = kv_heads * dh, unit = low ? 8 : 4, size = low ? 2 : 4;
    if (dh % unit != 0 || dh <= 0 || dh > 256) refuse(PyExc_ValueError, "head size %lld is not a multiple of %d up to 256", (long long)dh, (int)unit);
    const at::ScalarType type = q.scalar_type();
    const Rows rq = rows2d(q, type, dev, N, wq, "q"), rk = rows2d(k, type, dev, N, wk, "k"), rv = rows2d(v, type, dev, N, wk, "v"),
               ro = rows2d(out, type, dev, N, wq, "out");
    int64_t n_cu = 0;
    const int32_t* cu = given_ints(a[3], 1, dev, "cu", &n_cu);
    disjoint(ro.p, ro.ld, rq.p, rq.ld, N, wq, wq, size, "out must not overlap q, k or v");
    disjoint(ro.p, ro.ld, rk.p, rk.ld, N, wq, wk, size, "out must not overlap q, k or v");
    disjoint(ro.p, ro.ld, rv.p, rv.ld, N, wq, wk, size, "out must not overlap q, k or v");
    const float scale = scale_or(a[7], dh);
    void* st = current_stream(dev);
    if (low) issue("tst_attn_prompt_bf16", entry.tst_attn_prompt_bf16, rq.p, rq.ld, rk.p, rk.ld, rv.p, rv.ld, cu, n_cu - 1, ro.p, ro.ld, N, heads, kv_heads,
                   dh, scale, st);
    else issue("tst_attn_prompt_f32", entry.tst_attn_prompt_f32, (const float*)rq.p, rq.ld, (const float*)rk.p, rk.ld, (const float*)rv.p, rv.ld, cu, n_cu - 1,
               (float*)ro.p, ro.ld, N, heads, kv_heads, dh, scale, st);
}

// lens, room, pages, page, table, cu, slots, pos, seq, used
void page_plan(PyObject* const* a) {
    const int64_t dev = current_device(), page = as_int(a[3], "page");
    int64_t B = 0, N = 0, n_pages = 0;
    const int32_t* lens = given_ints(a[0], 0, dev, "lens", &B);
    int32_t* slots = given_ints(a[6], 0, dev, "slots", &N);
    const int32_t* pages = given_ints(a[2], 0, dev, "pages", &n_pages);
    const Table t = table2d(a[4], dev, "table");
    if (t.rows != B) refuse(PyExc_ValueError, "table must be [sequences, width]");
    if (page > 0 && n_pages > 0x7fffffff / page) refuse(PyExc_ValueError, "pages * page exceeds 2^31 - 1: slots are 32-bit");
    issue("tst_page_plan", entry.tst_page_plan, lens, (const int32_t*)ints(a[1], B, dev, "room"), B, pages, n_pages, page, t.p, t.width,
          ints(a[5], B + 1, dev, "cu"), slots, ints(a[7], N, dev, "pos"), ints(a[8], N, dev, "seq"), N, ints(a[9], 1, dev, "used"), current_stream(dev));
}

// base, sent, t, table, page, slots, pos, lens, n_rows
void page_step(PyObject* const* a) {
    const int64_t dev = current_device(), n = as_int(a[8], "n_rows");
    const Table t = table2d(a[3], dev, "table");
    issue("tst_page_step", entry.tst_page_step, (const int32_t*)ints(a[0], t.rows, dev, "base"), (const int32_t*)ints(a[1], n, dev, "sent"), as_int(a[2], "t"),
          (const int32_t*)t.p, t.width, t.rows, as_int(a[4], "page"), ints(a[5], n, dev, "slots"), ints(a[6], n, dev, "pos"), ints(a[7], n, dev, "lens"), n,
          current_stream(dev));
}

int64_t cache_device(PyObject* o) {
    const int64_t at = as_int(o, "cache"), dev = current_device();
    if (at != dev) refuse(PyExc_ValueError, "the cache is on cuda:%lld, the current device is cuda:%lld", (long long)at, (long long)dev);
    return dev;
}

// cache address, cache device, k, v, slots, n_rows
void cache4_write(PyObject* const* a) {
    const tst_cache4* c = cache_at(a[0]);
    const at::Tensor &k = tensor(a[2], "k"), &v = tensor(a[3], "v");
    const bool low = is_bf16(k, "rows");
    const int64_t dev = cache_device(a[1]), n = as_int(a[5], "n_rows"), w = (int64_t)c->kv_heads * c->dh;
    const Rows rk = rows2d(k, k.scalar_type(), dev, n, w, "k"), rv = rows2d(v, k.scalar_type(), dev, n, w, "v");
    const int32_t* slots = ints(a[4], n, dev, "slots");
    void* st = current_stream(dev);
    if (low) issue("tst_cache4_write_bf16", entry.tst_cache4_write_bf16, c, rk.p, rk.ld, rv.p, rv.ld, slots, n, st);
    else issue("tst_cache4_write_f32", entry.tst_cache4_write_f32, c, (const float*)rk.p, rk.ld, (const float*)rv.p, rv.ld, slots, n, st);
}

// cache address, cache device, slots, k, v, n_rows
void cache4_read(PyObject* const* a) {
    const tst_cache4* c = cache_at(a[0]);
    const at::Tensor &k = tensor(a[3], "k"), &v = tensor(a[4], "v");
    const bool low = is_bf16(k, "rows");
    const int64_t dev = cache_device(a[1]), n = as_int(a[5], "n_rows"), w = (int64_t)c->kv_heads * c->dh;
    const int32_t* slots = ints(a[2], n, dev, "slots");
    const Rows rk = rows2d(k, k.scalar_type(), dev, n, w, "k"), rv = rows2d(v, k.scalar_type(), dev, n, w, "v");
    void* st = current_stream(dev);
    if (low) issue("tst_cache4_read_bf16", entry.tst_cache4_read_bf16, c, slots, rk.p, rk.ld, rv.p, rv.ld, n, st);
    else issue("tst_cache4_read_f32", entry.tst_cache4_read_f32, c, slots, (float*)rk.p, rk.ld, (float*)rv.p, rv.ld, n, st);
}

// cache address, cache device, q, table, lens, out, n_rows, heads, max_len, seq, scale, work
void attn_cache4(PyObject* const* a) {
    const tst_cache4* c = cache_at(a[0]);
    const at::Tensor &q = tensor(a[2], "q"), &out = tensor(a[5], "out");
    const bool low = is_bf16(q, "q");
    const int64_t dev = cache_device(a[1]), n = as_int(a[6], "n_rows"), heads = as_int(a[7], "heads"), max_len = as_int(a[8], "max_len"), dh = c->dh;
    if (heads < 1 || heads % c->kv_heads != 0) refuse(PyExc_ValueError, "heads must be a multiple of the cache's %d", (int)c->kv_heads);
    const int64_t w = heads * dh;
    const Rows rq = rows2d(q, q.scalar_type(), dev, n, w, "q"), ro = rows2d(out, q.scalar_type(), dev, n, w, "out");
    disjoint(ro.p, ro.ld, rq.p, rq.ld, n, w, w, low ? 2 : 4, "out must not overlap q");
    const Table t = table2d(a[3], dev, "table");
    float* work = nullptr;
    int64_t n_work = 0;
    if (a[11] != Py_None) {
        const at::Tensor& s = tensor(a[11], "work");
        if (s.scalar_type() != F32 || where(s) != dev || !s.is_contiguous())
            refuse(PyExc_ValueError, "work must be a contiguous fp32 tensor on the current GPU");
        work = static_cast<float*>(s.data_ptr());
        n_work = s.numel();
    }
    const int32_t *seq = ints(a[9], n, dev, "seq"), *lens = ints(a[4], n, dev, "lens");
    const float scale = scale_or(a[10], dh);
    void* st = current_stream(dev);
    if (low) issue("tst_attn_cache4_bf16", entry.tst_attn_cache4_bf16, c, rq.p, rq.ld, t.p, t.width, t.rows, seq, lens, max_len, ro.p, ro.ld, n, heads, scale,
                   work, n_work, st);
    else issue("tst_attn_cache4_f32", entry.tst_attn_cache4_f32, c, (const float*)rq.p, rq.ld, t.p, t.width, t.rows, seq, lens, max_len, (float*)ro.p, ro.ld, n, heads,
               scale, work, n_work, st);
}

// address, leading dimension and rows of a bias or mask table
struct RuleRows {
    void* p;
    int64_t ld, rows;
};
RuleRows rule_rows(const at::Tensor& t, at::ScalarType type, int64_t width, int64_t dev, const char* name) {
    if (t.scalar_type() != type || t.dim() != 2 || where(t) != dev || t.size(1) < width || (t.stride(1) != 1 && t.size(1) > 1) ||
        (t.size(0) > 1 && t.stride(0) < width))
        refuse(PyExc_ValueError, "%s must be a 2-D %s tensor [n, %lld] with unit inner stride on the current GPU", name, type == F32 ? "torch.float32" : "torch.int32",
               (long long)width);
    return {t.data_ptr(), t.stride(0) > width ? t.stride(0) : width, t.size(0)};
}

// logits, n_rows, n_cols, out, params, sent, hist, hist_len, prompt, prompt_cu, bias, bias_row, mask, mask_row
void adjust_logits(PyObject* const* a) {
    const at::Tensor &x = tensor(a[0], "logits"), &out = tensor(a[3], "out");
    const int64_t n = as_int(a[1], "n_rows"), V = as_int(a[2], "n_cols"), dev = current_device();
    const bool low = is_bf16(x, "logits");
    int64_t ld[2];
    const at::Tensor* both[2] = {&x, &out};
    for (int i = 0; i < 2; ++i) {
        const at::Tensor& t = *both[i];
        if (t.scalar_type() != x.scalar_type() || t.dim() != 2 || where(t) != dev || (t.stride(1) != 1 && t.size(1) > 1))
            refuse(PyExc_ValueError, "logits and out must be 2-D tensors of one type with unit inner stride on the current GPU");
        if (t.size(0) < n || t.size(1) < V || (n > 1 && t.stride(0) < V))
            refuse(PyExc_ValueError, "%s must hold [%lld, %lld] without overlapping rows", i ? "out" : "logits", (long long)n, (long long)V);
        ld[i] = t.stride(0) > V ? t.stride(0) : V;
    }
    char *p_in = static_cast<char*>(x.data_ptr()), *p_out = static_cast<char*>(out.data_ptr());
    if (p_in != p_out) disjoint(p_out, ld[1], p_in, ld[0], n, V, V, low ? 2 : 4, "out must be logits or not overlap it");
    tst_logit_rules r = {};
    if (a[4] != Py_None) {
        const at::Tensor& t = tensor(a[4], "params");
        if (t.scalar_type() != F32 || t.dim() != 2 || t.size(1) != 3 || where(t) != dev || !t.is_contiguous() || (a[5] == Py_None && t.size(0) < n))
            refuse(PyExc_ValueError, "params must be a contiguous fp32 tensor [sentences, 3] on the current GPU");
        r.params = static_cast<const float*>(t.data_ptr());
        r.n_sent = t.size(0);
    } else if (a[6] != Py_None || a[8] != Py_None) {
        refuse(PyExc_ValueError, "hist and prompt need params");
    }
    r.sent = ints(a[5], n, dev, "sent");
    if (a[6] != Py_None) {
        const at::Tensor& t = tensor(a[6], "hist");
        if (t.scalar_type() != I32 || t.dim() != 2 || where(t) != dev || t.size(0) < n || (t.stride(1) != 1 && t.size(1) > 1) ||
            (n > 1 && t.stride(0) < t.size(1)))
            refuse(PyExc_ValueError, "hist must be int32 [rows, tokens] with unit inner stride on the current GPU");
        r.hist = static_cast<const int32_t*>(t.data_ptr());
        r.n_hist = t.size(1);
        r.ld_hist = t.stride(0) > r.n_hist ? t.stride(0) : r.n_hist;
        r.hist_len = ints(a[7], n, dev, "hist_len");
    }
    if (a[8] != Py_None) {
        if (a[9] == Py_None) refuse(PyExc_ValueError, "prompt needs prompt_cu");
        r.prompt = given_ints(a[8], 0, dev, "prompt", &r.n_prompt);
        r.prompt_cu = ints(a[9], r.n_sent + 1, dev, "prompt_cu");
    }
    if (a[10] != Py_None) {
        const RuleRows t = rule_rows(tensor(a[10], "bias"), F32, V, dev, "bias");
        r.bias = static_cast<const float*>(t.p);
        r.ld_bias = t.ld;
        r.n_bias = t.rows;
        r.bias_row = ints(a[11], n, dev, "bias_row");
    }
    if (a[12] != Py_None) {
        const RuleRows t = rule_rows(tensor(a[12], "mask"), I32, (V + 31) / 32, dev, "mask");
        r.mask = static_cast<const uint32_t*>(t.p);
        r.ld_mask = t.ld;
        r.n_masks = t.rows;
        r.mask_row = ints(a[13], n, dev, "mask_row");
    }
    void* st = current_stream(dev);
    if (low) issue("tst_adjust_logits_bf16", entry.tst_adjust_logits_bf16, p_in, ld[0], n, V, &r, p_out, ld[1], st);
    else issue("tst_adjust_logits_f32", entry.tst_adjust_logits_f32, (const float*)p_in, ld[0], n, V, &r, (float*)p_out, ld[1], st);
}

// table, state, parent, tok, out, n_rows
void grammar_next(PyObject* const* a) {
    const int64_t dev = current_device(), n = as_int(a[5], "n_rows");
    const Table t = table2d(a[0], dev, "table");
    int64_t n_state = 0;
    const int32_t* state = given_ints(a[1], 0, dev, "state", &n_state);
    int32_t* out = ints(a[4], n, dev, "out");
    if (n > 0 && out == state) refuse(PyExc_ValueError, "out must not be state");
    issue("tst_grammar_next", entry.tst_grammar_next, (const int32_t*)t.p, t.rows, t.width, state, n_state, (const int32_t*)ints(a[2], n, dev, "parent"),
          (const int32_t*)ints(a[3], n, dev, "tok"), out, n, current_stream(dev));
}

template <void (*F)(PyObject* const*), int COUNT>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != COUNT) {
        PyErr_Format(PyExc_TypeError, "%d arguments wanted, %zd given", COUNT, n);
        return nullptr;
    }
    try {
        F(args);
    } catch (const Refused&) {
        return nullptr;
    } catch (const std::exception& e) {   // a tensor without memory, strides ...
        PyErr_SetString(PyExc_ValueError, e.what());
        return nullptr;
    }
    Py_RETURN_NONE;
}

// bind({entry point: address}, current device, current stream of a device, error class)
PyObject* bind(PyObject*, PyObject* args) {
    PyObject *addresses, *dev, *stream, *error;
    if (!PyArg_ParseTuple(args, "O!OOO", &PyDict_Type, &addresses, &dev, &stream, &error)) return nullptr;
    Entries e;
#define X(name)                                                                          \
    {                                                                                    \
        PyObject* at = PyDict_GetItemString(addresses, #name);                           \
        void* p = at != nullptr ? PyLong_AsVoidPtr(at) : nullptr;                        \
        if (p == nullptr) {                                                              \
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_KeyError, #name);               \
            return nullptr;                                                              \
        }                                                                                \
        e.name = reinterpret_cast<decltype(e.name)>(p);                                  \
    }
    TST_CALLS(X)
#undef X
    entry = e;
    Py_INCREF(dev);
    Py_INCREF(stream);
    Py_INCREF(error);
    device_fn = dev;
    stream_fn = stream;
    error_type = error;
    Py_RETURN_NONE;
}

#define FAST(name, count) {#name, (PyCFunction)(void (*)(void))guarded<name, count>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, nullptr}, FAST(attn_prompt, 8), FAST(page_plan, 10), FAST(page_step, 9), FAST(cache4_write, 6),
                         FAST(cache4_read, 6), FAST(attn_cache4, 12), FAST(adjust_logits, 14), FAST(grammar_next, 6), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tst_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__tst_calls() {
    PyObject* m = PyModule_Create(&module);
    // the tensor fields read here lie where this torch puts them: whoever loads the module compares
    if (m != nullptr && PyModule_AddStringConstant(m, "built_for", TORCH_VERSION) != 0) Py_CLEAR(m);
    return m;
}
