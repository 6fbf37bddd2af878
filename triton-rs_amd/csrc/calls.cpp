// Python's side of the calls that a program makes once a layer and step (norm, rotary positions, the caches'
// attention, the 8-bit cache): checks of the tensors, then the C-ABI entry point, without a Python object on the
// way. A decode step makes hundreds of these calls, of a few microseconds of GPU time each; in Python the checks and
// ctypes' conversions made a call of rms_norm 9.9 us, which takes 4.2 here.
//
// A module for CPython (built by build.py beside the library, imported by __init__.py): functions of positional
// arguments, called by the functions of the same names there, which have the documentation.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/core/DeviceGuard.h>

#include <cstdarg>
#include <cstdio>
#include <stdexcept>
#include <string>

#include "../../include/w4a16.h"

namespace {

PyObject *invalid_argument, *check, *current_stream;   // set by setup()

struct Refused { std::string what; };
struct PythonError {};   // (an exception is set)

[[noreturn]] __attribute__((format(printf, 1, 2))) void refuse(const char* fmt, ...) {
    char text[512];
    va_list a;
    va_start(a, fmt);
    vsnprintf(text, sizeof(text), fmt, a);
    va_end(a);
    throw Refused{text};
}

std::string text(at::IntArrayRef s) {
    std::string r = "[";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + "]";
}

// ------------------------------------------------------------------ arguments

bool none(PyObject* o) { return o == Py_None; }

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse("%s must be a torch tensor", name);
    return THPVariable_Unpack(o);
}
bool is_elem(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }

void check_type(const at::Tensor& t, const char* name, at::ScalarType type) {
    if (t.scalar_type() != type) refuse("%s has dtype %s, expected %s", name, toString(t.scalar_type()), toString(type));
}
// A tensor that decides the call's device; then others, which must be there too.
int device_of(const at::Tensor& t, const char* name) {
    if (!t.is_cuda()) refuse("%s must be on the GPU", name);
    return t.get_device();
}
const at::Tensor& on(PyObject* o, const char* name, int device, at::ScalarType type) {
    const at::Tensor& t = tensor(o, name);
    if (!t.is_cuda()) refuse("%s must be on the GPU", name);
    if (t.get_device() != device) refuse("%s is on cuda:%d, expected cuda:%d", name, (int)t.get_device(), device);
    check_type(t, name, type);
    return t;
}
const at::Tensor& elements(PyObject* o, const char* name) {
    const at::Tensor& t = tensor(o, name);
    if (!t.is_cuda()) refuse("%s must be on the GPU", name);
    if (!is_elem(t.scalar_type())) refuse("%s has dtype %s, expected float16 or bfloat16", name, toString(t.scalar_type()));
    return t;
}

// Tensors that a call writes. There is no backward pass: written in place, a tensor of a graph that is being recorded would go
// on without what was done to it. And whoever has saved one for a backward pass of its own is told by its version.
struct Written {
    const at::Tensor* t[4];
    int n = 0;
    void add(const at::Tensor& x, const char* name, bool any = false) {   // any: gradients or not
        if (!any && x.requires_grad() && at::GradMode::is_enabled())
            refuse("%s requires grad and would be written, and there is no backward pass: call under torch.no_grad(), or give a tensor of its own to write to", name);
        t[n++] = &x;
    }
    void done() const {
        for (int i = 0; i < n; ++i)
            if (!t[i]->is_inference()) t[i]->unsafeGetTensorImpl()->bump_version();
    }
};

int elem_flag(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? W4A16_BF16 : 0; }

int64_t integer(PyObject* o) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw PythonError{};
    return v;
}
double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw PythonError{};
    return v;
}
bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw PythonError{};
    return v != 0;
}

// Sizes and strides of the C entries are 32-bit.
int32_t size32(int64_t v, const char* name) {
    if (v > INT32_MAX || v < INT32_MIN) refuse("%s is 32-bit (%lld)", name, (long long)v);
    return (int32_t)v;
}

struct Rows { void* p; int32_t st, sh; };
constexpr Rows NO_ROWS{nullptr, 0, 0};

// Rows [T, H, D] with contiguous D (two_d: or [T, D]); shape: as they have to be (null: any).
Rows rows(const at::Tensor& t, const char* name, const at::IntArrayRef* shape, bool two_d = false) {
    const auto s = t.sizes();
    if (shape ? s != *shape : s.size() != 3 && !(two_d && s.size() == 2))
        refuse("%s must be %s, not %s", name, shape ? text(*shape).c_str() : two_d ? "[T, K] or [T, H, K]" : "[T, heads, D]", text(s).c_str());
    const auto st = t.strides();
    if (st.back() != 1 && s.back() > 1) refuse("%s must be contiguous along its last dimension", name);
    const int64_t a = st[0], b = s.size() == 3 ? st[1] : 0;
    if (a > INT32_MAX || b > INT32_MAX || s[0] > INT32_MAX || s[1] > INT32_MAX || s.back() > INT32_MAX)
        refuse("%s: rows and strides are 32-bit (%s at %s)", name, text(s).c_str(), text(st).c_str());
    return {t.data_ptr(), (int32_t)a, (int32_t)b};
}
const int32_t* indices(PyObject* o, const char* name, int device, int64_t n) {
    const at::Tensor& t = on(o, name, device, at::kInt);
    if (t.dim() != 1 || t.size(0) != n || !t.is_contiguous()) refuse("%s must be a contiguous int32 tensor [%lld]", name, (long long)n);
    return t.data_ptr<int32_t>();
}

// ------------------------------------------------------------------ calls

void* stream_of(int device) {
    PyObject* i = PyLong_FromLong(device);
    PyObject* s = i ? PyObject_CallOneArg(current_stream, i) : nullptr;
    Py_XDECREF(i);
    if (!s) throw PythonError{};
    void* p = PyLong_AsVoidPtr(s);
    Py_DECREF(s);
    if (!p && PyErr_Occurred()) throw PythonError{};
    return p;
}
// f(stream) on the device's current stream, with the device as the current one; its status as Python's exception.
template <typename F>
void call_on(int device, F f) {
    void* stream = stream_of(device);
    int rc;
    {
        const c10::DeviceGuard guard(c10::Device(c10::kCUDA, (c10::DeviceIndex)device));
        PyThreadState* released = PyEval_SaveThread();
        rc = f(stream);
        PyEval_RestoreThread(released);
    }
    if (rc == W4A16_OK) return;
    PyObject* r = PyObject_CallFunction(check, "i", rc);   // raises
    Py_XDECREF(r);
    throw PythonError{};
}

template <typename F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F f) {
    if (n != want) {
        PyErr_Format(PyExc_TypeError, "%zd arguments, not %zd", want, n);
        return nullptr;
    }
    HANDLE_TH_ERRORS   // torch's exceptions as torch's own functions raise them (memory that is not there: torch.OutOfMemoryError)
    try {
        return f();
    } catch (const Refused& e) {
        PyErr_SetString(invalid_argument, e.what.c_str());
    } catch (const PythonError&) {
    }
    return nullptr;
    END_HANDLE_TH_ERRORS
}
PyObject* given(PyObject* o) {
    Py_INCREF(o);
    return o;
}

// (x, weight, eps, residual, residual_out, out, scales, group or None) -> out, or (out, scales)
PyObject* rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 8, [&]() -> PyObject* {
        const at::Tensor& x = elements(a[0], "x");
        const int device = x.get_device();
        const auto type = x.scalar_type();
        const Rows xr = rows(x, "x", nullptr, true);
        const at::IntArrayRef shape = x.sizes();
        const int32_t T = (int32_t)shape[0], H = shape.size() == 3 ? (int32_t)shape[1] : 1, K = (int32_t)shape.back();
        const at::Tensor& w = on(a[1], "weight", device, type);
        if (w.dim() != 1 || w.size(0) != K || !w.is_contiguous()) refuse("weight must be a contiguous [%d] tensor", K);
        const float eps = (float)number(a[2]);
        Rows r = NO_ROWS, ro = NO_ROWS;
        Written written;
        if (!none(a[3])) {
            const at::Tensor& residual = on(a[3], "residual", device, type);
            r = ro = rows(residual, "residual", &shape, true);
            if (!none(a[4])) ro = rows(on(a[4], "residual_out", device, type), "residual_out", &shape, true);
            written.add(none(a[4]) ? residual : THPVariable_Unpack(a[4]), none(a[4]) ? "residual" : "residual_out");
        } else if (!none(a[4])) {
            refuse("residual_out without residual");
        }
        const bool bytes = !none(a[7]);
        const auto out_type = bytes ? at::kFloat8_e4m3fn : type;
        at::Tensor made, made_scales;
        if (none(a[5])) made = at::empty(shape, x.options().dtype(out_type));
        const at::Tensor& out = none(a[5]) ? made : on(a[5], "out", device, out_type);
        const Rows o = rows(out, "out", &shape, true);
        if (!none(a[5])) written.add(out, "out");
        const void* weight = w.data_ptr();
        const int flag = elem_flag(x);
        if (!bytes) {
            call_on(device, [&](void* s) {
                return w4a16_rms_norm(s, flag, xr.p, xr.st, xr.sh, r.p, r.st, r.sh, ro.p, ro.st, ro.sh, weight, o.p, o.st, o.sh, T, H, K, eps);
            });
            written.done();
            return none(a[5]) ? THPVariable_Wrap(made) : given(a[5]);
        }
        const int64_t group = integer(a[7]);
        if (group < 0 || (group && K % group)) refuse("group %lld: 0 (a row), or a divisor of %d", (long long)group, K);
        std::vector<int64_t> want(shape.begin(), shape.end());
        want.back() = K ? K / (group ? group : K) : 0;
        if (none(a[6])) made_scales = at::empty(want, x.options().dtype(at::kFloat));
        const at::Tensor& scales = none(a[6]) ? made_scales : on(a[6], "scales", device, at::kFloat);
        if (scales.sizes() != at::IntArrayRef(want) || !scales.is_contiguous()) refuse("scales must be a contiguous %s tensor", text(want).c_str());
        if (!none(a[6])) written.add(scales, "scales");
        float* sp = scales.data_ptr<float>();
        call_on(device, [&](void* s) {
            return w4a16_rms_norm_8bit(s, flag, xr.p, xr.st, xr.sh, r.p, r.st, r.sh, ro.p, ro.st, ro.sh, weight, o.p, o.st, o.sh, sp, T, H, K, (int32_t)group, eps);
        });
        written.done();
        PyObject *po = none(a[5]) ? THPVariable_Wrap(made) : given(a[5]), *ps = none(a[6]) ? THPVariable_Wrap(made_scales) : given(a[6]);
        PyObject* both = po && ps ? PyTuple_Pack(2, po, ps) : nullptr;
        Py_XDECREF(po);
        Py_XDECREF(ps);
        return both;
    });
}

struct Turn { const double* f = nullptr; float magnitude = 0.f; int32_t rot = 0, interleaved = 0; };
Turn turn(PyObject* inv_freq, PyObject* magnitude, PyObject* interleaved, int device) {
    const at::Tensor& f = on(inv_freq, "rope.inv_freq", device, at::kDouble);
    if (f.dim() != 1 || !f.is_contiguous() || f.size(0) > (1 << 20)) refuse("rope.inv_freq must be a contiguous [rot / 2] tensor");
    return {f.data_ptr<double>(), (float)number(magnitude), (int32_t)(2 * f.size(0)), truth(interleaved)};
}

// (q, positions, inv_freq, magnitude, interleaved, k, q_out, k_out)
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 8, [&]() -> PyObject* {
        const at::Tensor& q = elements(a[0], "q");
        const int device = q.get_device();
        const auto type = q.scalar_type();
        const Rows qr = rows(q, "q", nullptr);
        const at::IntArrayRef shape = q.sizes();
        const at::Tensor& q_out = none(a[6]) ? q : on(a[6], "q_out", device, type);
        const Rows qo = rows(q_out, "q_out", &shape);
        Written written;
        written.add(q_out, none(a[6]) ? "q" : "q_out");
        const int32_t T = (int32_t)shape[0], Hq = (int32_t)shape[1], D = (int32_t)shape[2];
        const int32_t* positions = indices(a[1], "positions", device, T);
        const Turn t = turn(a[2], a[3], a[4], device);
        int32_t Hkv = 0;
        Rows kr = NO_ROWS, ko = NO_ROWS;
        if (!none(a[5])) {
            const at::Tensor& k = on(a[5], "k", device, type);
            const int64_t want[3] = {T, k.dim() == 3 ? k.size(1) : 0, D};
            const at::IntArrayRef ks(want, 3);
            kr = rows(k, "k", &ks);
            Hkv = (int32_t)want[1];
            const at::Tensor& k_out = none(a[7]) ? k : on(a[7], "k_out", device, type);
            ko = rows(k_out, "k_out", &ks);
            written.add(k_out, none(a[7]) ? "k" : "k_out");
        } else if (!none(a[7])) {
            refuse("k_out without k");
        }
        const int flag = elem_flag(q);
        call_on(device, [&](void* s) {
            return w4a16_rope(s, flag, qr.p, qr.st, qr.sh, qo.p, qo.st, qo.sh, kr.p, kr.st, kr.sh, ko.p, ko.st, ko.sh, positions, t.f, t.magnitude, T, Hq,
                              Hkv, D, t.rot, t.interleaved);
        });
        written.done();
        Py_RETURN_NONE;
    });
}

// A cache of either format: [pages, kv heads, page_size / 16, bytes of a block].
struct Cache { void* p; int device; int32_t pages, Hkv, page, D; };
Cache cache_of(PyObject* o, int bits) {
    const at::Tensor& t = tensor(o, "cache");
    const int device = device_of(t, "cache");
    check_type(t, "cache", at::kByte);
    const int per = bits == 4 ? 16 : 32, tail = bits == 4 ? 128 : 16;
    if (t.dim() != 4 || !t.is_contiguous()) refuse("cache must be a contiguous [pages, kv heads, page_size / 16, %d D + %d] tensor", per, tail);
    const int64_t width = t.size(3), D = (width - tail) / per;
    if (D < 1 || width != per * D + tail) refuse("cache has blocks of %lld bytes, not %d D + %d", (long long)width, per, tail);
    return {t.data_ptr(), device, size32(t.size(0), "cache"), size32(t.size(1), "cache"), size32(t.size(2) * 16, "cache"), size32(D, "cache")};
}
struct Table { const int32_t* p; int32_t B, per; };
Table table_of(PyObject* o, int device) {
    const at::Tensor& t = on(o, "page_table", device, at::kInt);
    if (t.dim() != 2 || !t.is_contiguous()) refuse("page_table must be a contiguous [sequences, pages per sequence] tensor");
    return {t.data_ptr<int32_t>(), size32(t.size(0), "page_table"), size32(t.size(1), "page_table")};
}

// (k, v, cache, page_table, kv_lens, cu_q, max_q_len, inv_freq, magnitude, interleaved, positions, q, q_out)
PyObject* kv8_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 13, [&]() -> PyObject* {
        const Cache c = cache_of(a[2], 8);
        const at::Tensor& k = elements(a[0], "k");
        const auto type = k.scalar_type();
        on(a[0], "k", c.device, type);
        const int64_t want[3] = {k.dim() ? k.size(0) : 0, c.Hkv, c.D};
        const at::IntArrayRef shape(want, 3);
        const Rows kr = rows(k, "k", &shape), vr = rows(on(a[1], "v", c.device, type), "v", &shape);
        const int32_t T = (int32_t)want[0];
        const Table t = table_of(a[3], c.device);
        const int32_t* lens = indices(a[4], "kv_lens", c.device, t.B);
        const int32_t* cu = none(a[5]) ? nullptr : indices(a[5], "cu_q", c.device, (int64_t)t.B + 1);
        const int32_t max_q = none(a[6]) ? (cu && T > 1 ? T : 1) : size32(integer(a[6]), "max_q_len");
        Turn r;
        const int32_t* positions = nullptr;
        Rows qr = NO_ROWS, qo = NO_ROWS;
        int32_t Hq = 0;
        Written written;
        written.add(THPVariable_Unpack(a[2]), "cache");
        if (!none(a[7])) {
            r = turn(a[7], a[8], a[9], c.device);
            if (!none(a[10])) positions = indices(a[10], "positions", c.device, T);
            if (!none(a[11])) {
                const at::Tensor& q = on(a[11], "q", c.device, type);
                const int64_t qs[3] = {T, q.dim() == 3 ? q.size(1) : 0, c.D};
                const at::IntArrayRef qshape(qs, 3);
                qr = rows(q, "q", &qshape);
                Hq = (int32_t)qs[1];
                const at::Tensor& q_out = none(a[12]) ? q : on(a[12], "q_out", c.device, type);
                qo = rows(q_out, "q_out", &qshape);
                written.add(q_out, none(a[12]) ? "q" : "q_out");
            }
        } else if (!none(a[10]) || !none(a[11])) {
            refuse("positions and q are for a rotation: give rope");
        }
        if (none(a[11]) && !none(a[12])) refuse("q_out without q");
        if (T > 0 && (t.B > 0 || (qr.p && positions))) {   // (without sequences queries are rotated at most)
            const int flag = elem_flag(k);
            call_on(c.device, [&](void* s) {
                return w4a16_kv8_write(s, flag, kr.p, kr.st, kr.sh, vr.p, vr.st, vr.sh, qr.p, qr.st, qr.sh, qo.p, qo.st, qo.sh, positions, r.f, r.magnitude,
                                       r.rot, r.interleaved, c.p, t.p, lens, cu, T, t.B, Hq, c.Hkv, c.D, c.pages, c.page, t.B > 0 ? t.per : std::max(1, t.per), max_q);
            });
            written.done();
        }
        return given(a[2]);
    });
}

// (cache, slots, k_out, v_out)
PyObject* kv8_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 4, [&]() -> PyObject* {
        const Cache c = cache_of(a[0], 8);
        const at::Tensor& slots = on(a[1], "slots", c.device, at::kInt);
        if (slots.dim() != 1 || !slots.is_contiguous()) refuse("slots must be a contiguous 1-D tensor");
        const int64_t want[3] = {slots.size(0), c.Hkv, c.D};
        const at::IntArrayRef shape(want, 3);
        const at::Tensor& k = elements(a[2], "k_out");
        on(a[2], "k_out", c.device, k.scalar_type());
        const at::Tensor& v = on(a[3], "v_out", c.device, k.scalar_type());
        const Rows kr = rows(k, "k_out", &shape), vr = rows(v, "v_out", &shape);
        Written written;
        written.add(k, "k_out");
        written.add(v, "v_out");
        const int32_t* sp = slots.data_ptr<int32_t>();
        const int flag = elem_flag(k);
        call_on(c.device, [&](void* s) {
            return w4a16_kv8_read(s, flag, c.p, sp, kr.p, kr.st, kr.sh, vr.p, vr.st, vr.sh, c.pages, (int32_t)want[0], c.Hkv, c.D, c.page);
        });
        written.done();
        Py_RETURN_NONE;
    });
}

struct Format {
    int bits;
    size_t (*workspace)(int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t);
    decltype(&w4a16_kv8_attention) attention;
};
Format format_of(PyObject* o) {
    return integer(o) == 4 ? Format{4, w4a16_kv4_attention_workspace_size, w4a16_kv4_attention}
                           : Format{8, w4a16_kv8_attention_workspace_size, w4a16_kv8_attention};
}
at::Tensor new_workspace(const Format& f, const Cache& c, at::TensorOptions options, int64_t T, int64_t B, int64_t Hq, int64_t max_q, int64_t max_kv) {
    if (std::max({T, B, Hq, max_q, max_kv}) > INT32_MAX || std::min({T, B, Hq, max_q, max_kv}) < INT32_MIN)
        refuse("sizes are 32-bit (%lld, %lld, %lld, %lld, %lld)", (long long)T, (long long)B, (long long)Hq, (long long)max_q, (long long)max_kv);
    const size_t need = f.workspace((int32_t)T, (int32_t)B, (int32_t)Hq, c.Hkv, c.D, (int32_t)max_q, (int32_t)max_kv);
    if (!need) {
        PyObject* r = PyObject_CallFunction(check, "i", (int)W4A16_ERR_INVALID_ARG);
        Py_XDECREF(r);
        throw PythonError{};
    }
    at::Tensor ws = at::empty({(int64_t)need}, options.dtype(at::kByte));
    ws.narrow(0, 0, W4A16_KV8_COUNTER_BYTES).zero_();
    return ws;
}
static_assert(W4A16_KV4_COUNTER_BYTES == W4A16_KV8_COUNTER_BYTES, "one area of counters");

// (bits, rows of q, its heads, cache, num_seqs, max_q_len, max_kv_len)
PyObject* attention_workspace(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 7, [&]() -> PyObject* {
        const Format f = format_of(a[0]);
        const Cache c = cache_of(a[3], f.bits);
        return THPVariable_Wrap(new_workspace(f, c, tensor(a[3], "cache").options(), integer(a[1]), integer(a[4]), integer(a[2]), integer(a[5]), integer(a[6])));
    });
}

// (bits, q, cache, page_table, kv_lens, cu_q, max_q_len, max_kv_len, scale, causal, window, out, lse, workspace) -> out
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 14, [&]() -> PyObject* {
        const Format f = format_of(a[0]);
        const Cache c = cache_of(a[2], f.bits);
        const at::Tensor& q = elements(a[1], "q");
        const auto type = q.scalar_type();
        on(a[1], "q", c.device, type);
        const Rows qr = rows(q, "q", nullptr);
        const at::IntArrayRef shape = q.sizes();
        const int64_t T = shape[0], Hq = shape[1];
        if (shape[2] != c.D) refuse("q has heads of %lld dimensions, the cache %d", (long long)shape[2], c.D);
        const Table t = table_of(a[3], c.device);
        const int32_t* lens = indices(a[4], "kv_lens", c.device, t.B);
        const int32_t* cu = nullptr;
        if (!none(a[5])) cu = indices(a[5], "cu_q", c.device, (int64_t)t.B + 1);
        else if (T != t.B)   // (also where one is 0, and there would be nothing to launch)
            refuse("without cu_q every sequence has one query (%lld queries, %d sequences)", (long long)T, t.B);
        const int64_t max_q = none(a[6]) ? (cu ? std::max<int64_t>(1, T) : 1) : integer(a[6]);
        const int64_t max_kv = none(a[7]) ? (int64_t)t.per * c.page : integer(a[7]), window = integer(a[10]);
        if (std::max({max_q, max_kv, window}) > INT32_MAX || std::min({max_q, max_kv, window}) < INT32_MIN)
            refuse("max_q_len, max_kv_len and window are 32-bit (%lld, %lld, %lld)", (long long)max_q, (long long)max_kv, (long long)window);
        const float scale = none(a[8]) ? (float)(1.0 / std::sqrt((double)c.D)) : (float)number(a[8]);
        const bool causal = truth(a[9]);
        at::Tensor made, made_workspace;
        if (none(a[11])) made = cu ? at::zeros(shape, q.options()) : at::empty(shape, q.options());
        const at::Tensor& out = none(a[11]) ? made : on(a[11], "out", c.device, type);
        const Rows o = rows(out, "out", &shape);
        Written written;
        if (!none(a[11])) written.add(out, "out", f.bits == 4);   // (the 4-bit cache's calls have always taken one that requires grad)
        float* lse = nullptr;
        if (!none(a[12])) {
            const at::Tensor& l = on(a[12], "lse", c.device, at::kFloat);
            if (l.dim() != 2 || l.size(0) != T || l.size(1) != Hq || !l.is_contiguous()) refuse("lse must be a contiguous [%lld, %lld] tensor", (long long)T, (long long)Hq);
            written.add(l, "lse", f.bits == 4);
            lse = l.data_ptr<float>();
        }
        if (T > 0 && t.B > 0) {
            if (none(a[13])) made_workspace = new_workspace(f, c, tensor(a[2], "cache").options(), T, t.B, Hq, max_q, max_kv);
            const at::Tensor& ws = none(a[13]) ? made_workspace : on(a[13], "workspace", c.device, at::kByte);
            if (!ws.is_contiguous()) refuse("workspace must be contiguous");
            void* wp = ws.data_ptr();
            const size_t bytes = (size_t)ws.numel();
            const int flag = elem_flag(q);
            call_on(c.device, [&](void* s) {
                return f.attention(s, flag, qr.p, qr.st, qr.sh, c.p, t.p, lens, cu, o.p, o.st, o.sh, lse, (int32_t)T, t.B, (int32_t)Hq, c.Hkv, c.D, c.pages,
                                   c.page, t.per, (int32_t)max_q, (int32_t)max_kv, scale, causal, (int32_t)window, wp, bytes);
            });
            written.done();
        }
        return none(a[11]) ? THPVariable_Wrap(made) : given(a[11]);
    });
}

// (the exception class, the function that raises a status, the current stream of a device)
PyObject* setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 3, [&]() -> PyObject* {
        invalid_argument = given(a[0]);
        check = given(a[1]);
        current_stream = given(a[2]);
        Py_RETURN_NONE;
    });
}

PyMethodDef methods[] = {
    {"setup", (PyCFunction)(void (*)())setup, METH_FASTCALL, nullptr},
    {"rms_norm", (PyCFunction)(void (*)())rms_norm, METH_FASTCALL, nullptr},
    {"rope", (PyCFunction)(void (*)())rope, METH_FASTCALL, nullptr},
    {"kv8_write", (PyCFunction)(void (*)())kv8_write, METH_FASTCALL, nullptr},
    {"kv8_read", (PyCFunction)(void (*)())kv8_read, METH_FASTCALL, nullptr},
    {"attention", (PyCFunction)(void (*)())attention, METH_FASTCALL, nullptr},
    {"attention_workspace", (PyCFunction)(void (*)())attention_workspace, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__calls() { return PyModule_Create(&module_def); }
