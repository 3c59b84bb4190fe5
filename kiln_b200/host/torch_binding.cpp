// Compiled binding of the 4-bit, rotary and dropout calls for torch tensors (kiln_b200/ops.py has the functions that users call and their documentation).
//
// The shortest of these calls take the GPU 2-5 us, and what Python and ctypes do for one - a buffer or two, a dozen tensor attributes, seventeen
// converted arguments - took 6-9 us more: a projection of one token, quantisation and product, 22 us of host time for 6 us of device time. Here a call reads the
// tensors' own structures and goes straight through the C ABI, whose addresses ops.py hands over once (bind), so both use one loaded library.
// It checks what the C ABI cannot see: shapes, types, strides, that a 4-bit matrix's buffers still hold it, and that every tensor lies on the current device.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <structmember.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Device.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdarg>
#include <limits>
#include <string>

#include "../../include/kiln_b200.h"

namespace {

decltype(&kb_quant4) f_quant4;
decltype(&kb_dequant4) f_dequant4;
decltype(&kb_linear4) f_linear4;
decltype(&kb_linear4_dx) f_linear4_dx;
decltype(&kb_rope) f_rope;
decltype(&kb_dropout) f_dropout;
PyObject* kiln_error = nullptr;       // ops.KilnError

struct Refused {};                    // a Python exception is set

[[noreturn]] void refuse(const char* format, ...) {
    va_list args;
    va_start(args, format);
    PyErr_FormatV(PyExc_ValueError, format, args);
    va_end(args);
    throw Refused();
}

void check(int code, const char* what) {
    if (code == KB_OK) return;
    PyObject* args = Py_BuildValue("is", code, what);
    if (args) { PyErr_SetObject(kiln_error, args); Py_DECREF(args); }
    throw Refused();
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse("%s is no tensor", name);
    return THPVariable_Unpack(o);
}

int to_int(PyObject* o) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw Refused();
    if (v < std::numeric_limits<int>::min() || v > std::numeric_limits<int>::max()) refuse("%ld does not fit 32 bits", v);
    return (int)v;
}
double to_double(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Refused();
    return v;
}
bool to_bool(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Refused();
    return v != 0;
}

int dtype_code(const at::Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case at::kHalf: return KB_F16;
        case at::kBFloat16: return KB_BF16;
        case at::kFloat: return KB_F32;
        default: refuse("%s is fp16, bf16 or fp32", name);
    }
}

// A [rows, cols] matrix with elements side by side along a row
struct Mat {
    void* p;
    int rows, cols, ld, dtype, device;
};
Mat matrix(const at::Tensor& t, const char* name) {
    if (t.dim() != 2) refuse("%s is a matrix [rows, cols]", name);
    const int64_t rows = t.size(0), cols = t.size(1), most = std::numeric_limits<int>::max();
    if (rows > most || cols > most) refuse("%s is too large", name);
    if (cols > 1 && t.stride(1) != 1) refuse("the elements of a row of %s lie side by side", name);
    int64_t ld = t.stride(0);
    if (rows <= 1) ld = (cols + 7) / 8 * 8;         // the stride of a single row is never used, and may be anything
    if (ld > most || ld < 0) refuse("%s has a row stride beyond 32 bits", name);
    return {t.data_ptr(), (int)rows, (int)cols, (int)ld, dtype_code(t, name), t.is_cuda() ? (int)t.get_device() : -1};
}

// the current device, which every tensor has to lie on, and its current stream
struct Here {
    int device;
    void* stream;
    Here() : device((int)c10::cuda::current_device()), stream(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream()) {}
    void have(int where, const char* name) const {
        if (where != device) refuse(where < 0 ? "%s does not lie on a GPU; the current device is cuda:%d" : "%s lies on another device than the current cuda:%d", name, device);
    }
};

at::Tensor new_bytes(int64_t n, const at::Device& device) { return at::empty({n}, at::TensorOptions().dtype(at::kByte).device(device)); }

at::Device to_device(PyObject* o) {
    if (THPDevice_Check(o)) {
        at::Device d = reinterpret_cast<THPDevice*>(o)->device;
        return d.is_cuda() && !d.has_index() ? at::Device(d.type(), c10::cuda::current_device()) : d;
    }
    const char* s = PyUnicode_Check(o) ? PyUnicode_AsUTF8(o) : nullptr;
    if (!s) refuse("device is a torch.device or its name");
    at::Device d{std::string(s)};
    return d.is_cuda() && !d.has_index() ? at::Device(d.type(), c10::cuda::current_device()) : d;
}

// ---------------------------------------------------------------- Quant4
struct Quant4 {
    PyObject_HEAD
    PyObject *codes, *scales, *both;    // `both`: the one buffer of a matrix made here, whose two views are made when they are asked for
    int rows, cols, fmt, exp;
};
PyTypeObject* quant4_type = nullptr;

int row_bytes(int cols) { return (cols + 31) / 32 * 16; }
int64_t scale_bytes(int rows, int cols, int fmt) {
    const int piece = fmt == KB_NV4 ? 64 : 128;
    return ((int64_t)rows + 127) / 128 * ((cols + piece - 1) / piece) * 512;
}
void check_size(int rows, int cols, int fmt) {
    if (rows < 0 || rows > KB_MAX_Q4_ROWS || cols <= 0 || cols > KB_MAX_Q4_COLS || (fmt != KB_MX4 && fmt != KB_NV4)) refuse("no 4-bit matrix of %d x %d, format %d", rows, cols, fmt);
}
// The power of two of a whole matrix. quant4 takes 0 alone for MX4, but a product may carry one, and every product takes what a handle holds.
constexpr int MOST_EXP = 64;
int check_exp(int exp) {
    if (exp < -MOST_EXP || exp > MOST_EXP) refuse("exp lies between %d and %d, not %d", -MOST_EXP, MOST_EXP, exp);
    return exp;
}

// Where a matrix lies. A tensor can be given another memory at any time (`codes.data = ...`, which is what moving a parameter to another device does, or
// storage().resize_()), so this is asked for in every call and kept by none.
struct Buffers {
    void *codes, *scales;
    int ld, device;                     // bytes of a row of codes; -1: the CPU
};
// bytes [first, first + n) of a tensor's storage exist
bool exists(const at::Tensor& t, int64_t first, int64_t n) { return n <= 0 || (int64_t)t.storage().nbytes() >= first + n; }

Buffers buffers(const Quant4& q, const char* name) {
    const int wide = row_bytes(q.cols);
    const int64_t n_codes = (int64_t)q.rows * wide, n_scales = scale_bytes(q.rows, q.cols, q.fmt);
    Buffers b = {nullptr, nullptr, wide, -1};
    const at::Tensor* both = q.both ? &THPVariable_Unpack(q.both) : nullptr;
    at::Device codes_device(at::kCPU), scales_device(at::kCPU);
    if (q.codes) {
        const at::Tensor& t = THPVariable_Unpack(q.codes);
        if (t.element_size() != 1 || t.dim() != 2) refuse("%s: codes are a [rows, bytes] matrix of bytes", name);
        if (t.size(0) < q.rows || t.size(1) < wide || t.stride(1) != 1) refuse("%s: codes do not hold %d rows of %d columns", name, q.rows, q.cols);
        const int64_t ld = q.rows <= 1 ? wide : t.stride(0);
        if (ld > std::numeric_limits<int>::max()) refuse("%s: codes have a row stride beyond 32 bits", name);
        if (!exists(t, t.storage_offset(), q.rows ? (q.rows - 1) * ld + wide : 0)) refuse("%s: the memory behind its codes is gone", name);
        b.ld = (int)ld;
        b.codes = t.data_ptr();
        codes_device = t.device();
    } else if (both) {
        if (!exists(*both, both->storage_offset(), n_codes)) refuse("%s: the memory behind its codes is gone", name);
        b.codes = both->data_ptr();
        codes_device = both->device();
    } else {
        refuse("%s has no buffers", name);
    }
    if (q.scales) {
        const at::Tensor& t = THPVariable_Unpack(q.scales);
        if (t.element_size() != 1 || !t.is_contiguous()) refuse("%s: scales are contiguous bytes", name);
        if (t.numel() < n_scales) refuse("%s: scales do not hold %d rows of %d columns", name, q.rows, q.cols);
        if (!exists(t, t.storage_offset(), n_scales)) refuse("%s: the memory behind its scales is gone", name);
        b.scales = t.data_ptr();
        scales_device = t.device();
    } else if (both) {
        if (!exists(*both, both->storage_offset() + n_codes, n_scales)) refuse("%s: the memory behind its scales is gone", name);
        b.scales = static_cast<char*>(both->data_ptr()) + n_codes;
        scales_device = both->device();
    } else {
        refuse("%s has no buffers", name);
    }
    if (codes_device != scales_device) refuse("%s: codes and scales lie on one device", name);
    b.device = codes_device.is_cuda() ? (int)codes_device.index() : -1;
    return b;
}

Quant4* new_quant4() {
    Quant4* q = reinterpret_cast<Quant4*>(quant4_type->tp_alloc(quant4_type, 0));
    if (!q) throw Refused();
    return q;
}

Quant4* make_quant4(int rows, int cols, int fmt, int exp, const at::Device& device) {
    check_size(rows, cols, fmt);
    check_exp(exp);
    const int64_t codes = (int64_t)rows * row_bytes(cols);
    at::Tensor both = new_bytes(codes + scale_bytes(rows, cols, fmt), device);
    Quant4* q = new_quant4();
    q->rows = rows; q->cols = cols; q->fmt = fmt; q->exp = exp;
    q->both = THPVariable_Wrap(std::move(both));
    if (!q->both) { Py_DECREF(q); throw Refused(); }
    return q;
}

const Quant4& quant4_arg(PyObject* o, const char* name) {
    if (Py_TYPE(o) != quant4_type) refuse("%s is a Quant4", name);
    return *reinterpret_cast<Quant4*>(o);
}

PyObject* guard(PyObject* (*body)(PyObject* const*, Py_ssize_t), PyObject* const* args, Py_ssize_t n) {
    try {
        return body(args, n);
    } catch (const Refused&) {
        return nullptr;
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}
void expect(Py_ssize_t n, Py_ssize_t want) {
    if (n != want) refuse("%zd arguments, not %zd", want, n);
}

int quant4_init(PyObject* self, PyObject* args, PyObject* kwargs) {
    static const char* names[] = {"codes", "scales", "rows", "cols", "fmt", "exp", nullptr};
    PyObject *codes_o, *scales_o;
    int rows, cols, fmt, exp = 0;
    if (!PyArg_ParseTupleAndKeywords(args, kwargs, "OOiii|i", const_cast<char**>(names), &codes_o, &scales_o, &rows, &cols, &fmt, &exp)) return -1;
    try {
        check_size(rows, cols, fmt);
        check_exp(exp);
        tensor(codes_o, "codes");
        tensor(scales_o, "scales");
        Quant4 fresh = {};                              // looked over before `self` changes
        fresh.codes = codes_o; fresh.scales = scales_o;
        fresh.rows = rows; fresh.cols = cols; fresh.fmt = fmt; fresh.exp = exp;
        buffers(fresh, "Quant4");
        Quant4* q = reinterpret_cast<Quant4*>(self);
        q->rows = rows; q->cols = cols; q->fmt = fmt; q->exp = exp;
        Py_INCREF(codes_o);
        Py_INCREF(scales_o);
        Py_XSETREF(q->codes, codes_o);
        Py_XSETREF(q->scales, scales_o);
        Py_CLEAR(q->both);
        return 0;
    } catch (const Refused&) {
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return -1;
}
void quant4_dealloc(PyObject* self) {
    Quant4* q = reinterpret_cast<Quant4*>(self);
    Py_XDECREF(q->codes);
    Py_XDECREF(q->scales);
    Py_XDECREF(q->both);
    PyTypeObject* type = Py_TYPE(self);
    type->tp_free(self);
    Py_DECREF(type);
}
PyObject* view_of(Quant4* q, PyObject** slot, bool scales) {
    try {
        if (!*slot) {
            if (!q->both) refuse("this Quant4 has no buffers");
            const at::Tensor& both = THPVariable_Unpack(q->both);
            const int64_t wide = row_bytes(q->cols), codes = q->rows * wide;
            *slot = scales ? THPVariable_Wrap(both.narrow(0, codes, both.numel() - codes)) : THPVariable_Wrap(both.narrow(0, 0, codes).view({q->rows, wide}));
        }
        Py_XINCREF(*slot);
        return *slot;
    } catch (const Refused&) {
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}
PyObject* get_codes(PyObject* self, void*) { Quant4* q = reinterpret_cast<Quant4*>(self); return view_of(q, &q->codes, false); }
PyObject* get_scales(PyObject* self, void*) { Quant4* q = reinterpret_cast<Quant4*>(self); return view_of(q, &q->scales, true); }
// copy, deepcopy and pickle: the type's own arguments
PyObject* quant4_reduce(PyObject* self, PyObject*) {
    const Quant4* q = reinterpret_cast<Quant4*>(self);
    PyObject *codes = get_codes(self, nullptr), *scales = codes ? get_scales(self, nullptr) : nullptr;
    PyObject* made = scales ? Py_BuildValue("O(OOiiii)", reinterpret_cast<PyObject*>(Py_TYPE(self)), codes, scales, q->rows, q->cols, q->fmt, q->exp) : nullptr;
    Py_XDECREF(codes);
    Py_XDECREF(scales);
    return made;
}
PyMethodDef quant4_methods[] = {{"__reduce__", quant4_reduce, METH_NOARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
enum { WHERE_CODES, WHERE_SCALES, WHERE_LD, WHERE_DEVICE };
PyObject* get_where(PyObject* self, void* what) {
    try {
        const Buffers b = buffers(*reinterpret_cast<Quant4*>(self), "Quant4");
        switch ((int)(intptr_t)what) {
            case WHERE_CODES: return PyLong_FromUnsignedLongLong((uintptr_t)b.codes);
            case WHERE_SCALES: return PyLong_FromUnsignedLongLong((uintptr_t)b.scales);
            case WHERE_LD: return PyLong_FromLong(b.ld);
            default: return PyLong_FromLong(b.device);
        }
    } catch (const Refused&) {
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

PyObject* get_exp(PyObject* self, void*) { return PyLong_FromLong(reinterpret_cast<Quant4*>(self)->exp); }
int set_exp(PyObject* self, PyObject* value, void*) {
    try {
        if (!value) refuse("exp cannot be deleted");
        reinterpret_cast<Quant4*>(self)->exp = check_exp(to_int(value));
        return 0;
    } catch (const Refused&) {
        return -1;
    }
}

PyMemberDef quant4_members[] = {
    {"rows", T_INT, offsetof(Quant4, rows), READONLY, nullptr},
    {"cols", T_INT, offsetof(Quant4, cols), READONLY, nullptr},
    {"fmt", T_INT, offsetof(Quant4, fmt), READONLY, "MX4 or NV4"},
    {nullptr, 0, 0, 0, nullptr}};
PyGetSetDef quant4_getset[] = {
    {"codes", get_codes, nullptr, "uint8 [rows, ld]", nullptr},
    {"scales", get_scales, nullptr, "uint8, flat", nullptr},
    {"exp", get_exp, set_exp, "the whole matrix is times 2^exp", nullptr},
    {"ld", get_where, nullptr, "bytes from a row of codes to the next", (void*)(intptr_t)WHERE_LD},
    {"device", get_where, nullptr, "index of the GPU, -1 for the CPU", (void*)(intptr_t)WHERE_DEVICE},
    {"codes_ptr", get_where, nullptr, "where the codes lie now", (void*)(intptr_t)WHERE_CODES},
    {"scales_ptr", get_where, nullptr, "where the scales lie now", (void*)(intptr_t)WHERE_SCALES},
    {nullptr, nullptr, nullptr, nullptr, nullptr}};
PyType_Slot quant4_slots[] = {
    {Py_tp_doc, const_cast<char*>("Quant4(codes, scales, rows, cols, fmt, exp=0): a matrix [rows, cols] of 4-bit numbers in blocks (kb_quant4): codes uint8 [rows, >= 16 ceil(cols / 32)], "
                                  "scales uint8, fmt MX4 or NV4, all of it times 2^exp, exp from -64 to 64. quant4 makes MX4 matrices with 0 alone; "
                                  "another one counts in products, and dequant4 and linear4_dx refuse it.")},
    {Py_tp_init, (void*)quant4_init}, {Py_tp_new, (void*)PyType_GenericNew}, {Py_tp_dealloc, (void*)quant4_dealloc},
    {Py_tp_members, quant4_members}, {Py_tp_methods, quant4_methods}, {Py_tp_getset, quant4_getset}, {0, nullptr}};
PyType_Spec quant4_spec = {"kiln_b200.ops.Quant4", sizeof(Quant4), 0, Py_TPFLAGS_DEFAULT, quant4_slots};

inline void* ptr(unsigned long long p) { return reinterpret_cast<void*>((uintptr_t)p); }
inline PyObject* same(PyObject* o) { Py_INCREF(o); return o; }

// ---------------------------------------------------------------- calls
PyObject* py_quant4_empty(PyObject* const* a, Py_ssize_t n) {      // rows, cols, fmt, device, exp
    expect(n, 5);
    return reinterpret_cast<PyObject*>(make_quant4(to_int(a[0]), to_int(a[1]), to_int(a[2]), to_int(a[4]), to_device(a[3])));
}

PyObject* py_padded_empty(PyObject* const* a, Py_ssize_t n) {      // rows, cols, dtype, device
    expect(n, 4);
    if (!THPDtype_Check(a[2])) refuse("dtype is a torch.dtype");
    const at::ScalarType type = reinterpret_cast<THPDtype*>(a[2])->scalar_type;
    const int64_t rows = to_int(a[0]), cols = to_int(a[1]), step = 16 / (int64_t)c10::elementSize(type);
    if (rows < 0 || cols < 0 || step < 1) refuse("no such matrix");
    const int64_t wide = (cols + step - 1) / step * step;
    at::Tensor t = at::empty({rows, wide}, at::TensorOptions().dtype(type).device(to_device(a[3])));
    return THPVariable_Wrap(wide == cols ? std::move(t) : t.narrow(1, 0, cols));
}

PyObject* py_quant4(PyObject* const* a, Py_ssize_t n) {            // x, fmt, exp, out
    expect(n, 4);
    const at::Tensor& xt = tensor(a[0], "x");
    const Mat x = matrix(xt, "x");
    const int fmt = to_int(a[1]), exp = to_int(a[2]);
    Quant4* q;
    if (a[3] == Py_None) {
        q = make_quant4(x.rows, x.cols, fmt, exp, xt.device());
    } else {
        const Quant4& out = quant4_arg(a[3], "out");
        if (out.rows != x.rows || out.cols != x.cols || out.fmt != fmt || out.exp != exp) refuse("out was made for another matrix");
        q = reinterpret_cast<Quant4*>(same(a[3]));
    }
    try {
        const Here here;
        here.have(x.device, "x");
        const Buffers out = buffers(*q, "out");
        here.have(out.device, "out");
        if (x.rows) check(f_quant4(out.codes, out.ld, out.scales, x.p, x.ld, x.dtype, x.rows, x.cols, fmt, exp, here.stream), "kb_quant4");
    } catch (...) {
        Py_DECREF(q);
        throw;
    }
    return reinterpret_cast<PyObject*>(q);
}

PyObject* py_dequant4(PyObject* const* a, Py_ssize_t n) {          // y, q, transpose
    expect(n, 3);
    const Mat y = matrix(tensor(a[0], "y"), "y");
    const Quant4& q = quant4_arg(a[1], "q");
    const bool t = to_bool(a[2]);
    if (y.rows != (t ? q.cols : q.rows) || y.cols != (t ? q.rows : q.cols)) refuse("y is %d x %d for a matrix of %d x %d", y.rows, y.cols, q.rows, q.cols);
    const Here here;
    const Buffers b = buffers(q, "q");
    here.have(y.device, "y");
    here.have(b.device, "q");
    if (q.rows) check(f_dequant4(y.p, y.ld, y.dtype, b.codes, b.ld, b.scales, q.rows, q.cols, q.fmt, q.exp, t, here.stream), "kb_dequant4");
    return same(a[0]);
}

PyObject* py_linear4(PyObject* const* a, Py_ssize_t n) {           // C, A, W, epi, gate, alpha
    expect(n, 6);
    const Quant4 &A = quant4_arg(a[1], "A"), &W = quant4_arg(a[2], "W");
    const int M = A.rows, N = W.rows, K = A.cols, epi = to_int(a[3]);
    const Buffers ab = buffers(A, "A"), wb = buffers(W, "W");
    if (W.cols != K || W.fmt != A.fmt) refuse("A and W have to agree in columns and format");
    void *out, *scales = nullptr;
    int ldc, where;
    if (epi == KB_EPI_GELU4) {
        const Quant4& C = quant4_arg(a[0], "C of EPI_GELU4");
        if (C.rows != M || C.cols != N || C.fmt != A.fmt || C.exp != 0) refuse("EPI_GELU4 goes into a Quant4 [M, N] of the operands' format with exp 0");
        const Buffers cb = buffers(C, "C");
        out = cb.codes; scales = cb.scales; ldc = cb.ld; where = cb.device;
    } else {
        const Mat C = matrix(tensor(a[0], "C"), "C");
        if (C.rows != M || C.cols != N || C.dtype != (epi == KB_EPI_F32 || epi == KB_EPI_RESID ? KB_F32 : KB_F16)) refuse("C is [M, N] of its epilogue's type");
        out = C.p; ldc = C.ld; where = C.device;
    }
    const Here here;
    const float* gate = nullptr;
    if (a[4] != Py_None) {
        const at::Tensor& g = tensor(a[4], "gate");
        if (g.scalar_type() != at::kFloat || g.numel() < N || !g.is_contiguous()) refuse("gate is fp32 [N]");
        here.have(g.is_cuda() ? (int)g.get_device() : -1, "gate");
        gate = static_cast<const float*>(g.data_ptr());
    }
    here.have(where, "C");
    here.have(ab.device, "A");
    here.have(wb.device, "W");
    const double alpha = std::ldexp(to_double(a[5]), A.exp + W.exp);
    // within a rounding of 32 bits, which infinities, NaN and what vanishes are not
    if (!(std::fabs((double)(float)alpha - alpha) <= 0x1p-24 * std::fabs(alpha))) refuse("alpha and both powers of two make a factor that 32 bits do not hold");
    if (M) check(f_linear4(out, ldc, scales, ab.codes, ab.ld, ab.scales, wb.codes, wb.ld, wb.scales, M, N, K, A.fmt, epi, (float)alpha, gate,
                           here.stream), "kb_linear4");
    return same(a[0]);
}

PyObject* py_linear4_dx(PyObject* const* a, Py_ssize_t n) {        // dx, dy, W, workspace
    expect(n, 4);
    const at::Tensor& dyt = tensor(a[1], "dy");
    const Mat dx = matrix(tensor(a[0], "dx"), "dx"), dy = matrix(dyt, "dy");
    const Quant4& W = quant4_arg(a[2], "W");
    if (dy.cols != W.rows || dx.rows != dy.rows || dx.cols != W.cols || dy.dtype != KB_F16) refuse("dy is fp16 [M, N], dx [M, K] for a weight of [N, K]");
    const Here here;
    here.have(dx.device, "dx");
    here.have(dy.device, "dy");
    const Buffers wb = buffers(W, "W");
    here.have(wb.device, "W");
    if (!dy.rows) return same(a[0]);
    at::Tensor made;
    const bool given = a[3] != Py_None;
    if (!given) made = new_bytes((int64_t)2 * W.rows * W.cols, dyt.device());     // kb_linear4_dx_workspace_bytes
    const at::Tensor& ws = given ? tensor(a[3], "workspace") : made;
    if (given) here.have(ws.is_cuda() ? (int)ws.get_device() : -1, "workspace");
    if (!ws.is_contiguous()) refuse("the workspace is contiguous");
    check(f_linear4_dx(dx.p, dx.ld, dx.dtype, dy.p, dy.ld, wb.codes, wb.ld, wb.scales, dy.rows, W.rows, W.cols, W.fmt, W.exp, ws.data_ptr(), ws.nbytes(),
                       here.stream), "kb_linear4_dx");
    return same(a[0]);
}

// a one-dimensional contiguous host array of this kind ('d' or 'i')
struct HostArray {
    Py_buffer b;
    bool open = false;
    HostArray() = default;
    HostArray(const HostArray&) = delete;
    void get(PyObject* o, char kind, const char* name) {
        if (PyObject_GetBuffer(o, &b, PyBUF_FORMAT | PyBUF_C_CONTIGUOUS) != 0) throw Refused();
        open = true;
        if (b.ndim != 1 || !b.format || b.format[0] != kind || b.format[1] != 0) refuse("%s is one-dimensional, float64 (freq) or int32 (axis)", name);
    }
    ~HostArray() { if (open) PyBuffer_Release(&b); }
};

PyObject* py_rope(PyObject* const* a, Py_ssize_t n_args) {         // outs, xs, heads, head_dim, pos, freq, axis, layout, amplitude, inverse
    expect(n_args, 10);
    struct List {
        PyObject* seq;
        explicit List(PyObject* o) : seq(PySequence_Fast(o, "outs, xs and heads are sequences")) { if (!seq) throw Refused(); }
        List(const List&) = delete;
        ~List() { Py_DECREF(seq); }
        Py_ssize_t size() const { return PySequence_Fast_GET_SIZE(seq); }
        PyObject* operator[](Py_ssize_t i) const { return PySequence_Fast_GET_ITEM(seq, i); }
    };
    const List outs(a[0]), xs(a[1]), heads(a[2]);
    const Py_ssize_t n = xs.size();
    if (n < 1 || n > 4 || outs.size() != n || heads.size() != n) refuse("one to four tensors, an output and a number of heads each");
    const int head_dim = to_int(a[3]);
    void *px[4], *po[4];
    int lx[4], lo[4], nh[4], where[8], rows = 0, dtype = 0;
    for (Py_ssize_t i = 0; i < n; i++) {
        const Mat x = matrix(tensor(xs[i], "x"), "x"), o = matrix(tensor(outs[i], "out"), "out");
        nh[i] = to_int(heads[i]);
        if (i == 0) { rows = x.rows; dtype = x.dtype; }
        const int64_t wide = (int64_t)nh[i] * head_dim;
        if (x.rows != rows || o.rows != rows || x.dtype != dtype || o.dtype != dtype || x.cols < wide || o.cols < wide) refuse("tensors are [rows, heads * head_dim] of one type");
        px[i] = x.p; po[i] = o.p; lx[i] = x.ld; lo[i] = o.ld; where[2 * i] = x.device; where[2 * i + 1] = o.device;
    }
    const at::Tensor& pos = tensor(a[4], "pos");
    if (pos.scalar_type() != at::kInt || pos.dim() != 2 || (pos.size(1) > 1 && pos.stride(1) != 1)) refuse("pos is int32 [rows, axes]");
    const int64_t pos_rows = pos.size(0), axes = pos.size(1), ld_pos = pos_rows > 1 ? pos.stride(0) : axes, most = std::numeric_limits<int>::max();
    if (pos_rows > most || axes > most || ld_pos > most || ld_pos < 0) refuse("pos is too large");
    HostArray freq, axis;
    freq.get(a[5], 'd', "freq");
    if (a[6] != Py_None) {
        axis.get(a[6], 'i', "axis");
        if (axis.b.shape[0] != freq.b.shape[0]) refuse("axis has an entry per pair, as freq");
    }
    if (freq.b.shape[0] > 1 << 20) refuse("freq has too many pairs");
    const int layout = to_int(a[7]), inverse = to_bool(a[9]);
    const float amplitude = (float)to_double(a[8]);
    const Here here;
    for (Py_ssize_t i = 0; i < 2 * n; i++) here.have(where[i], i & 1 ? "out" : "x");
    here.have(pos.is_cuda() ? (int)pos.get_device() : -1, "pos");
    if (rows)
        check(f_rope((int)n, po, lo, px, lx, nh, dtype, rows, head_dim, 2 * (int)freq.b.shape[0], layout, static_cast<const int*>(pos.data_ptr()), (int)pos_rows, (int)ld_pos,
                     (int)axes, static_cast<const double*>(freq.b.buf), axis.open ? static_cast<const int*>(axis.b.buf) : nullptr, amplitude, inverse, here.stream), "kb_rope");
    return same(a[0]);
}

PyObject* py_dropout(PyObject* const* a, Py_ssize_t n) {           // out, x, rng, p, resid
    expect(n, 5);
    const Mat out = matrix(tensor(a[0], "out"), "out"), x = matrix(tensor(a[1], "x"), "x");
    const at::Tensor& rng = tensor(a[2], "rng");
    if (rng.element_size() != 8 || !at::isIntegralType(rng.scalar_type(), false) || rng.numel() != 2 || !rng.is_contiguous()) refuse("rng is int64 [2]: seed and offset");
    Mat res = {nullptr, 0, 0, 0, 0, 0};
    const bool has = a[4] != Py_None;
    if (has) res = matrix(tensor(a[4], "resid"), "resid");
    if (out.rows != x.rows || out.cols != x.cols || (has && (res.rows != x.rows || res.cols != x.cols || res.dtype != out.dtype)))
        refuse("out, x and resid have one shape, out and resid one type");
    const double p = to_double(a[3]);
    const Here here;
    here.have(out.device, "out");
    here.have(x.device, "x");
    here.have(rng.is_cuda() ? (int)rng.get_device() : -1, "rng");
    if (has) here.have(res.device, "resid");
    if (x.rows)
        check(f_dropout(out.p, out.ld, out.dtype, x.p, x.ld, x.dtype, res.p, res.ld, x.rows, x.cols, p, static_cast<const unsigned long long*>(rng.data_ptr()), here.stream),
              "kb_dropout");
    return same(a[0]);
}

PyObject* py_bind(PyObject* const* a, Py_ssize_t n) {              // KilnError, then the addresses of the calls in the order below
    expect(n, 7);
    unsigned long long p[6];
    for (int i = 0; i < 6; i++) {
        p[i] = PyLong_AsUnsignedLongLong(a[1 + i]);
        if (PyErr_Occurred()) throw Refused();
    }
    f_quant4 = reinterpret_cast<decltype(f_quant4)>(ptr(p[0]));
    f_dequant4 = reinterpret_cast<decltype(f_dequant4)>(ptr(p[1]));
    f_linear4 = reinterpret_cast<decltype(f_linear4)>(ptr(p[2]));
    f_linear4_dx = reinterpret_cast<decltype(f_linear4_dx)>(ptr(p[3]));
    f_rope = reinterpret_cast<decltype(f_rope)>(ptr(p[4]));
    f_dropout = reinterpret_cast<decltype(f_dropout)>(ptr(p[5]));
    Py_INCREF(a[0]);
    Py_XSETREF(kiln_error, a[0]);
    Py_RETURN_NONE;
}

template <PyObject* (*BODY)(PyObject* const*, Py_ssize_t)>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) { return guard(BODY, args, n); }

#define ENTRY(name) {#name, (PyCFunction)(void (*)(void))entry<py_##name>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(bind), ENTRY(quant4_empty), ENTRY(padded_empty), ENTRY(quant4), ENTRY(dequant4), ENTRY(linear4), ENTRY(linear4_dx), ENTRY(rope), ENTRY(dropout),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_kiln_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kiln_torch() {
    PyObject* m = PyModule_Create(&module_def);
    if (!m) return nullptr;
    quant4_type = reinterpret_cast<PyTypeObject*>(PyType_FromSpec(&quant4_spec));
    // in brackets in the file as well, where the build looks for it
    static const char built_for[] = "[" KB_BUILT_FOR "]";
    if (PyModule_AddObject(m, "built_for", PyUnicode_FromStringAndSize(built_for + 1, sizeof(built_for) - 3)) < 0) { Py_DECREF(m); return nullptr; }
    if (!quant4_type || PyModule_AddObjectRef(m, "Quant4", reinterpret_cast<PyObject*>(quant4_type)) < 0) { Py_DECREF(m); return nullptr; }
    return m;
}
