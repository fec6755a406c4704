// The dense products' calls from Python in native code: mmv(x, w, out_bf16, multi_col) and linear(x, w, gemv_tokens, chunk_bytes);
// those of 4-bit weights with group scales, int4_mmv and int4_moe_experts; the selection, router_topk_grouped; and those in 8-bit
// floating point, fp8_mm, fp8_moe_experts and add_rmsnorm_fp8.
//
// A small product is bound by the host's call (512 x 2048, one token: the kernel takes 3 us, the call with its checks, result
// and argument block in Python 9.2).  This does the same for the plain case: a two-dimensional tensor of the plain class on the
// current device, all of the weight's buffers there.  Whatever it does not take, wrong arguments among it, it answers with
// None, and the Python layer goes its general way, whose checks and messages hold; nothing is kept from one call for the next.
#include <Python.h>

#include <algorithm>

#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/gil.h>
#include <torch/csrc/autograd/python_variable.h>

#include "bf16n_c.h"

namespace {

typedef int (*mmv_fn)(const bf16n_weight *, const bf16n_mmv_args *, void *, int);
typedef int (*max_tokens_fn)(const bf16n_weight *, int *);
typedef int (*dequant_fn)(const bf16n_weight *, int64_t, int64_t, uint16_t *, void *);
mmv_fn g_mmv = nullptr; // of the library that the Python layer loaded
max_tokens_fn g_max_tokens = nullptr;
dequant_fn g_dequant = nullptr;
PyObject * s_plane, * s_aux, * s_meta, * s_format, * s_K, * s_rows, * s_R, * s_cm, * s_frag, * s_w64, * s_off[4];

// a tensor of the plain class with memory of its own on a device (no tracer, batch or gradient wrapper)
const at::Tensor * plain(PyObject * o) {
    if (!THPVariable_CheckExact(o)) {
        return nullptr;
    }
    const at::Tensor & t = THPVariable_Unpack(o);
    constexpr c10::DispatchKeySet other({c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot, c10::DispatchKey::FuncTorchBatched,
                                         c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize, c10::DispatchKey::Conjugate,
                                         c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor});
    if (!t.is_cuda() || t.layout() != c10::kStrided || t.key_set().has_any(other) || !t.has_storage()) {
        return nullptr;
    }
    return &t;
}

struct ref { // an owned attribute
    PyObject * o;
    ref(PyObject * of, PyObject * name) : o(PyObject_GetAttr(of, name)) {}
    ~ref() { Py_XDECREF(o); }
};
bool number(PyObject * of, PyObject * name, int64_t & out) {
    const ref a(of, name);
    if (!a.o || !PyLong_Check(a.o)) { // (bool is a number too)
        return false;
    }
    out = PyLong_AsLongLong(a.o);
    return out >= 0; // -1: an error too
}

PyObject * not_taken() {
    PyErr_Clear();
    Py_RETURN_NONE;
}

// x [tokens, K] and a weight on the current device, checked as the Python layer checks them
struct operands {
    const at::Tensor * x;
    bf16n_weight w;
    int device;
    bool x_bf16;
    bool get(PyObject * px, PyObject * pw) {
        if (!g_mmv || at::impl::torch_function_mode_enabled() || c10::impl::dispatch_mode_enabled()) {
            return false;
        }
        x = plain(px);
        if (!x || x->dim() != 2) {
            return false;
        }
        device = c10::hip::current_device();
        x_bf16 = x->scalar_type() == at::kBFloat16;
        const ref pl(pw, s_plane), au(pw, s_aux), me(pw, s_meta);
        if (!pl.o || !au.o || !me.o) {
            return false;
        }
        const at::Tensor * plane = plain(pl.o), * aux = plain(au.o);
        int64_t fmt, K, rows, R, cm, frag, w64, off[4];
        bool ok = plane && aux && x->get_device() == device && plane->get_device() == device && aux->get_device() == device &&
                  number(me.o, s_format, fmt) && number(me.o, s_K, K) && number(me.o, s_rows, rows) && number(me.o, s_R, R) &&
                  number(me.o, s_cm, cm) && number(me.o, s_frag, frag) && number(me.o, s_w64, w64);
        for (int i = 0; ok && i < 4; i++) {
            ok = number(me.o, s_off[i], off[i]) && off[i] < aux->numel();
        }
        if (!ok || plane->scalar_type() != at::kByte || aux->scalar_type() != at::kByte || !plane->is_contiguous() || !aux->is_contiguous() ||
            rows <= 0 || K <= 0 || plane->numel() != rows * K || fmt > INT32_MAX || R > INT32_MAX) {
            return false;
        }
        w = {};
        w.plane = (decltype(w.plane)) plane->data_ptr();
        w.aux = (decltype(w.aux)) aux->data_ptr();
        w.format = (int32_t) fmt;
        w.R = (int32_t) R;
        w.K = K;
        w.rows = rows;
        w.flags = (cm ? 1u : 0u) | (frag ? 2u : 0u) | (w64 ? 4u : 0u);
        w.off_a = (uint64_t) off[0];
        w.off_b = (uint64_t) off[1];
        w.off_c = (uint64_t) off[2];
        w.off_d = (uint64_t) off[3];
        return x->size(0) > 0 && x->size(0) <= 65535 && x->size(1) == K && x->stride(1) == 1 && x->stride(0) * (x_bf16 ? 2 : 4) % 16 == 0 &&
               (((uintptr_t) x->data_ptr() | (uintptr_t) w.plane | (uintptr_t) w.aux) & 15) == 0;
    }
    void * stream() const { return (void *) c10::hip::getCurrentHIPStream((c10::DeviceIndex) device).stream(); }
    PyObject * product(bool out_bf16, bool multi_col) const {
        at::Tensor y = at::empty({x->size(0), w.rows}, x->options().dtype(out_bf16 ? at::kBFloat16 : at::kFloat).requires_grad(false));
        bf16n_mmv_args a = {};
        a.x = (decltype(a.x)) x->data_ptr();
        a.y = (decltype(a.y)) y.data_ptr();
        a.x_tok = x->stride(0) * (x_bf16 ? 2 : 4);
        a.y_tok = w.rows * (out_bf16 ? 2 : 4);
        a.rows_per_matrix = w.rows;
        a.nrows = w.rows;
        a.ncols = (int32_t) x->size(0);
        a.n_used = 1;
        a.x_per_slot = 1;
        a.x_bf16 = x_bf16;
        a.y_bf16 = out_bf16;
        int status;
        {
            pybind11::gil_scoped_release free; // (the queue may be full)
            status = g_mmv(&w, &a, stream(), multi_col);
        }
        return status == 0 ? THPVariable_Wrap(y) : PyLong_FromLong(status);
    }
};

PyObject * mmv(PyObject *, PyObject * const * args, Py_ssize_t n) {
    try {
        operands o;
        if (n != 4 || !o.get(args[0], args[1]) || (!o.x_bf16 && o.x->scalar_type() != at::kFloat)) {
            return not_taken();
        }
        return o.product(args[2] == Py_True, args[3] == Py_True);
    } catch (const std::exception &) { // (out of memory: the general way meets it again and says so)
        return not_taken();
    }
}

// the GEMV up to gemv_tokens or bf16n_gemv_max_tokens tokens, beyond it the whole matrix decoded, if it is one piece of
// chunk_bytes, and torch's product
PyObject * linear(PyObject *, PyObject * const * args, Py_ssize_t n) {
    try {
        operands o;
        if (n != 4 || !o.get(args[0], args[1]) || !o.x_bf16) {
            return not_taken();
        }
        const int64_t gemv_tokens = PyLong_AsLongLong(args[2]), chunk_bytes = PyLong_AsLongLong(args[3]), T = o.x->size(0);
        if (gemv_tokens < 0 || chunk_bytes < 0) {
            return not_taken();
        }
        int most = 0;
        if (T > gemv_tokens && g_max_tokens(&o.w, &most) != 0) {
            return not_taken();
        }
        if (T <= gemv_tokens || T <= most) {
            return o.product(true, true);
        }
        const int64_t unit = o.w.format == 1 ? 1 : o.w.R; // (the 4-bit code has no units)
        if (unit <= 0 || std::max(chunk_bytes / (o.w.K * 2) / unit * unit, unit) < o.w.rows) {
            return not_taken();
        }
        at::Tensor d = at::empty({o.w.rows, o.w.K}, o.x->options().requires_grad(false)), y;
        int status;
        {
            pybind11::gil_scoped_release free;
            status = g_dequant(&o.w, 0, o.w.rows, (uint16_t *) d.data_ptr(), o.stream());
            if (status == 0) {
                y = at::linear(*o.x, d);
            }
        }
        return status == 0 ? THPVariable_Wrap(y) : PyLong_FromLong(status);
    } catch (const std::exception &) {
        return not_taken();
    }
}

// ---------------------------------------------------------------- 4-bit weights with group scales, selection in groups

typedef int (*int4_bytes_fn)(const bf16n_int4_weight *, int64_t, int64_t, int, uint64_t *);
typedef int (*int4_mmv_fn)(const bf16n_int4_weight *, const bf16n_int4_weight *, const bf16n_mmv_args *, int, void *, uint64_t, void *);
typedef int (*int4_route_fn)(const void *, int, int64_t, int64_t, int, int, int, int32_t *, int32_t *, void *);
typedef int (*int4_mm_ids_fn)(const bf16n_int4_weight *, const bf16n_int4_weight *, const void *, int64_t, int, const int32_t *, const int32_t *, void *,
                              int, int64_t, int, int, int, void *, uint64_t, void *);
typedef int (*combine_fn)(const float *, const void *, int, void *, int, int, int, int64_t, void *);
typedef int (*router_fn)(const float *, int64_t, const float *, int, int, int, int, int, int, int, int, float, int32_t *, float *, int64_t, void *);
int4_bytes_fn g_int4_bytes = nullptr;
int4_mmv_fn g_int4_mmv = nullptr;
int4_route_fn g_int4_route = nullptr;
int4_mm_ids_fn g_int4_mm_ids = nullptr;
combine_fn g_combine = nullptr;
router_fn g_router = nullptr;
PyObject * s_codes, * s_scales, * s_zeros, * s_group;

bool native() { return g_int4_mmv && !at::impl::torch_function_mode_enabled() && !c10::impl::dispatch_mode_enabled(); }

at::TensorOptions on(const at::Tensor & like, at::ScalarType t) { return like.options().dtype(t).requires_grad(false); }
void * stream_of(int device) { return (void *) c10::hip::getCurrentHIPStream((c10::DeviceIndex) device).stream(); }

// an Int4Weight on the device, its tensors as their class has checked them
bool int4_matrix(PyObject * o, int device, bf16n_int4_weight & w) {
    const ref co(o, s_codes), sc(o, s_scales), ze(o, s_zeros);
    if (!co.o || !sc.o || !ze.o) {
        return false;
    }
    const at::Tensor * c = plain(co.o), * s = plain(sc.o), * z = ze.o == Py_None ? nullptr : plain(ze.o);
    int64_t group;
    if (!c || !s || (!z && ze.o != Py_None) || !number(o, s_group, group) || c->dim() != 2 || s->dim() != 2 || group < 32 || group > 1 << 30 ||
        (group & (group - 1)) || c->scalar_type() != at::kByte || !c->is_contiguous() || !s->is_contiguous()) {
        return false;
    }
    w = {};
    w.rows = c->size(0);
    w.K = 2 * c->size(1);
    w.group = (int32_t) group;
    w.scales_f16 = s->scalar_type() == at::kHalf;
    const int64_t groups = (w.K + group - 1) / group;
    if (c->get_device() != device || s->get_device() != device || (!w.scales_f16 && s->scalar_type() != at::kBFloat16) || s->size(0) != w.rows || s->size(1) != groups ||
        (z && (z->get_device() != device || z->scalar_type() != at::kByte || !z->is_contiguous() || z->dim() != 2 || z->size(0) != w.rows || z->size(1) != groups))) {
        return false;
    }
    w.codes = (const uint8_t *) c->data_ptr();
    w.scales = s->data_ptr();
    w.zeros = z ? (const uint8_t *) z->data_ptr() : nullptr;
    return w.rows > 0;
}
bool alike(const bf16n_int4_weight & a, const bf16n_int4_weight & b) { return a.rows == b.rows && a.K == b.K && a.group == b.group && !a.zeros == !b.zeros; }

// rows of K activations, 16-byte aligned as the kernels read them
const at::Tensor * int4_x(PyObject * o, int device, int64_t K) {
    const at::Tensor * x = plain(o);
    if (!x || x->dim() != 2 || x->get_device() != device || (x->scalar_type() != at::kBFloat16 && x->scalar_type() != at::kFloat) || x->size(0) <= 0 ||
        x->size(0) > 1 << 24 || x->size(1) != K || x->stride(1) != 1 || x->stride(0) * x->element_size() % 16 != 0 || (uintptr_t) x->data_ptr() % 16 != 0) {
        return nullptr;
    }
    return x;
}

bf16n_mmv_args int4_args(const at::Tensor & x, const at::Tensor & y, int64_t rows) {
    bf16n_mmv_args a = {};
    a.x = (decltype(a.x)) x.data_ptr();
    a.y = (decltype(a.y)) y.data_ptr();
    a.x_tok = x.stride(0) * x.element_size();
    a.y_tok = y.stride(0) * y.element_size();
    a.rows_per_matrix = a.nrows = rows;
    a.ncols = (int32_t) x.size(0);
    a.n_used = a.x_per_slot = 1;
    a.x_bf16 = x.scalar_type() == at::kBFloat16;
    a.y_bf16 = y.scalar_type() == at::kBFloat16;
    return a;
}

// int4_mmv(x, w, up or None, out_bf16, few_tokens): dense
PyObject * int4_mmv(PyObject *, PyObject * const * args, Py_ssize_t n) {
    try {
        if (n != 5 || !native()) {
            return not_taken();
        }
        const int device = c10::hip::current_device();
        bf16n_int4_weight w, up;
        const bool glu = args[2] != Py_None;
        if (!int4_matrix(args[1], device, w) || (glu && (!int4_matrix(args[2], device, up) || !alike(w, up)))) {
            return not_taken();
        }
        const at::Tensor * x = int4_x(args[0], device, w.K);
        const int64_t few = PyLong_AsLongLong(args[4]);
        if (!x || few < 0) {
            return not_taken();
        }
        at::Tensor y = at::empty({x->size(0), w.rows}, on(*x, args[3] == Py_True ? at::kBFloat16 : at::kFloat)), space;
        const bf16n_mmv_args a = int4_args(*x, y, w.rows);
        uint64_t bytes = 0;
        if (a.x_bf16 && x->size(0) > few) {
            if (g_int4_bytes(&w, x->size(0), 0, 0, &bytes) != 0) {
                return not_taken();
            }
            space = at::empty({(int64_t) bytes}, on(*x, at::kByte));
        }
        int status;
        {
            pybind11::gil_scoped_release free;
            status = g_int4_mmv(&w, glu ? &up : nullptr, &a, 0, bytes ? space.data_ptr() : nullptr, bytes, stream_of(device));
        }
        return status == 0 ? THPVariable_Wrap(y) : PyLong_FromLong(status);
    } catch (const std::exception &) {
        return not_taken();
    }
}

// int4_moe_experts(x, gate, up, down, topk_weights, topk_ids, n_experts, batched): the launches of the Python layer's, in its order
PyObject * int4_moe_experts(PyObject *, PyObject * const * args, Py_ssize_t n) {
    try {
        if (n != 8 || !native()) {
            return not_taken();
        }
        const int device = c10::hip::current_device();
        bf16n_int4_weight gate, up, down;
        if (!int4_matrix(args[1], device, gate) || !int4_matrix(args[2], device, up) || !int4_matrix(args[3], device, down) || !alike(gate, up)) {
            return not_taken();
        }
        const at::Tensor * x = int4_x(args[0], device, gate.K), * wts = plain(args[4]), * ids = plain(args[5]);
        const int64_t E = PyLong_AsLongLong(args[6]);
        const bool batched = args[7] == Py_True;
        if (!x || !wts || !ids || E <= 0 || E > 65534 || gate.rows % E || down.rows % E || down.K != gate.rows / E || !x->is_contiguous() || ids->dim() != 2 ||
            (ids->scalar_type() != at::kInt && ids->scalar_type() != at::kLong) || ids->get_device() != device || ids->size(0) != x->size(0) || ids->size(1) <= 0 ||
            ids->stride(1) != 1 || wts->dim() != 2 || wts->get_device() != device || !wts->is_contiguous() ||
            (wts->scalar_type() != at::kFloat && wts->scalar_type() != at::kBFloat16) || wts->size(0) != ids->size(0) || wts->size(1) != ids->size(1)) {
            return not_taken();
        }
        const int64_t T = ids->size(0), slots = ids->size(1), mid = gate.rows / E, out = down.rows / E, pairs = T * slots;
        const bool x_bf16 = x->scalar_type() == at::kBFloat16;
        if (T > 65535 || pairs > (batched ? 1 << 28 : 65535) || (batched && !x_bf16) || gate.rows / E > 1 << 30) {
            return not_taken();
        }
        const int i64 = ids->scalar_type() == at::kLong, isz = i64 ? 8 : 4;
        at::Tensor hidden = at::empty({pairs, mid}, on(*x, batched ? at::kBFloat16 : at::kFloat));
        at::Tensor ys = at::empty({pairs, out}, on(*x, at::kFloat)), y = at::empty({T, out}, on(*x, at::kBFloat16)), lists, space;
        uint64_t bytes = 0;
        if (batched) {
            uint64_t second = 0;
            if (g_int4_bytes(&gate, T, pairs, (int) E, &bytes) != 0 || g_int4_bytes(&down, pairs, pairs, (int) E, &second) != 0) {
                return not_taken();
            }
            bytes = std::max(bytes, second);
            lists = at::empty({pairs + E + 2}, on(*x, at::kInt));
            space = at::empty({(int64_t) bytes}, on(*x, at::kByte));
        }
        void * const stream = stream_of(device);
        int status;
        {
            pybind11::gil_scoped_release free;
            if (batched) {
                int32_t * const sorted = (int32_t *) lists.data_ptr(), * const bounds = sorted + pairs;
                status = g_int4_route(ids->data_ptr(), i64, isz, ids->stride(0) * isz, (int) E, (int) T, (int) slots, sorted, bounds, stream);
                status = status ? status : g_int4_mm_ids(&gate, &up, x->data_ptr(), gate.K, 0, sorted, bounds, hidden.data_ptr(), 1, mid, (int) E, (int) T, (int) slots,
                                                         space.data_ptr(), bytes, stream);
                status = status ? status : g_int4_mm_ids(&down, nullptr, hidden.data_ptr(), mid, 1, sorted, bounds, ys.data_ptr(), 0, out, (int) E, (int) T, (int) slots,
                                                         space.data_ptr(), bytes, stream);
            } else {
                bf16n_mmv_args a = int4_args(*x, hidden, mid);
                a.ids = (decltype(a.ids)) ids->data_ptr();
                a.ids_s0 = isz;
                a.ids_s1 = ids->stride(0) * isz;
                a.ncols = (int32_t) pairs;
                a.n_used = (int32_t) slots;
                a.y_slot = mid * 4;
                a.y_tok = slots * a.y_slot;
                bf16n_mmv_args b = int4_args(hidden, ys, out);
                b.ids = a.ids;
                b.ids_s0 = a.ids_s0;
                b.ids_s1 = a.ids_s1;
                b.n_used = b.x_per_slot = (int32_t) slots;
                b.x_slot = a.y_slot;
                b.x_tok = a.y_tok;
                b.y_slot = out * 4;
                b.y_tok = slots * b.y_slot;
                status = g_int4_mmv(&gate, &up, &a, i64, nullptr, 0, stream);
                status = status ? status : g_int4_mmv(&down, nullptr, &b, i64, nullptr, 0, stream);
            }
            status = status ? status : g_combine((const float *) ys.data_ptr(), wts->data_ptr(), wts->scalar_type() == at::kBFloat16, y.data_ptr(), 1, (int) T, (int) slots, out, stream);
        }
        return status == 0 ? THPVariable_Wrap(y) : PyLong_FromLong(status);
    } catch (const std::exception &) {
        return not_taken();
    }
}

// router_topk_grouped(logits, k, bias or None, n_groups, topk_groups, sigmoid, top2, renorm, scale) -> (weights, ids)
PyObject * router_topk_grouped(PyObject *, PyObject * const * args, Py_ssize_t n) {
    try {
        if (n != 9 || !native()) {
            return not_taken();
        }
        const int device = c10::hip::current_device();
        const at::Tensor * lg = plain(args[0]), * bias = args[2] == Py_None ? nullptr : plain(args[2]);
        int64_t v[3];
        for (int i = 0; i < 3; i++) {
            PyObject * o = args[i ? 2 + i : 1];
            if (!PyLong_Check(o)) {
                return not_taken();
            }
            v[i] = PyLong_AsLongLong(o);
        }
        const double scale = PyFloat_AsDouble(args[8]);
        if (PyErr_Occurred() || !lg || (!bias && args[2] != Py_None) || lg->dim() != 2 || lg->get_device() != device || lg->scalar_type() != at::kFloat || lg->stride(1) != 1 ||
            lg->size(0) <= 0 || lg->size(0) > INT32_MAX || lg->size(1) > 1024 || v[0] <= 0 || v[0] > 64 || v[1] <= 0 || v[1] > 64 || v[2] <= 0 || v[2] > 64 ||
            (bias && (bias->get_device() != device || bias->scalar_type() != at::kFloat || !bias->is_contiguous() || bias->numel() != lg->size(1)))) {
            return not_taken();
        }
        const int64_t T = lg->size(0);
        at::Tensor wts = at::empty({T, v[0]}, on(*lg, at::kFloat)), ids = at::empty({T, v[0]}, on(*lg, at::kInt));
        const int status = g_router((const float *) lg->data_ptr(), lg->stride(0), bias ? (const float *) bias->data_ptr() : nullptr, (int) T, (int) lg->size(1), (int) v[1], (int) v[2],
                                    (int) v[0], args[5] == Py_True, args[6] == Py_True, args[7] == Py_True, (float) scale, (int32_t *) ids.data_ptr(), (float *) wts.data_ptr(), v[0],
                                    stream_of(device));
        if (status != 0) {
            return PyLong_FromLong(status);
        }
        PyObject * a = THPVariable_Wrap(wts), * b = THPVariable_Wrap(ids);
        PyObject * both = a && b ? PyTuple_Pack(2, a, b) : nullptr;
        Py_XDECREF(a);
        Py_XDECREF(b);
        return both;
    } catch (const std::exception &) {
        return not_taken();
    }
}

// ---------------------------------------------------------------- 8-bit floating point with a scale for every block of 128

typedef int (*fp8_bytes_fn)(const bf16n_fp8_weight *, int, int, int, int64_t, int64_t, int, uint64_t *);
typedef int (*fp8_mm_fn)(const bf16n_fp8_weight *, const bf16n_fp8_weight *, const bf16n_fp8_rows *, const bf16n_fp8_rows *, int64_t, void *, uint64_t, void *);
typedef int (*fp8_experts_bytes_fn)(const bf16n_fp8_weight *, const bf16n_fp8_weight *, int, int, int, int, uint64_t *);
typedef int (*fp8_experts_fn)(const bf16n_fp8_weight *, const bf16n_fp8_weight *, const bf16n_fp8_weight *, const bf16n_fp8_rows *, const void *, int, int64_t, int64_t,
                              const void *, int, const bf16n_fp8_rows *, int, int, void *, uint64_t, void *);
typedef int (*fp8_norm_fn)(const uint16_t *, const uint16_t *, const uint16_t *, const float *, const void *, int, int, const uint16_t *, const bf16n_fp8_rows *, uint16_t *,
                           uint16_t *, int, int64_t, float, void *);
fp8_bytes_fn g_fp8_bytes = nullptr;
fp8_mm_fn g_fp8_mm = nullptr;
fp8_experts_bytes_fn g_fp8_experts_bytes = nullptr;
fp8_experts_fn g_fp8_experts = nullptr;
fp8_norm_fn g_fp8_norm = nullptr;
PyObject * s_n_matrices;

bool native_fp8() { return g_fp8_mm && !at::impl::torch_function_mode_enabled() && !c10::impl::dispatch_mode_enabled(); }
int64_t blocks_of(int64_t n) { return (n + 127) / 128; }

// an Fp8Weight on the device, its tensors as their class has checked them
bool fp8_matrix(PyObject * o, int device, bf16n_fp8_weight & w) {
    const ref co(o, s_codes), sc(o, s_scales);
    if (!co.o || !sc.o) {
        return false;
    }
    const at::Tensor * c = plain(co.o), * s = plain(sc.o);
    int64_t n;
    if (!c || !s || !number(o, s_n_matrices, n) || n <= 0 || c->dim() != 2 || s->dim() != 2 || c->scalar_type() != at::kFloat8_e4m3fn || !c->is_contiguous() ||
        !s->is_contiguous() || c->get_device() != device || s->get_device() != device || c->size(0) <= 0 || c->size(0) % n) {
        return false;
    }
    w = {};
    w.codes = (const uint8_t *) c->data_ptr();
    w.scales = s->data_ptr();
    w.K = c->size(1);
    w.rows = c->size(0);
    w.n_matrices = n;
    w.scales_bf16 = s->scalar_type() == at::kBFloat16;
    return (w.scales_bf16 || s->scalar_type() == at::kFloat) && s->size(0) == n * blocks_of(w.rows / n) && s->size(1) == blocks_of(w.K);
}
bool alike(const bf16n_fp8_weight & a, const bf16n_fp8_weight & b) { return a.rows == b.rows && a.K == b.K && a.n_matrices == b.n_matrices && a.scales_bf16 == b.scales_bf16; }

struct fp8_x {
    bf16n_fp8_rows r;
    int64_t rows;
    at::TensorOptions like;
    // BF16 or FP32 rows of K values, or Fp8Rows
    bool get(PyObject * o, int device, int64_t K) {
        r = {};
        const at::Tensor * x;
        if (THPVariable_CheckExact(o)) {
            x = plain(o);
            if (!x || (x->scalar_type() != at::kBFloat16 && x->scalar_type() != at::kFloat)) {
                return false;
            }
            r.kind = x->scalar_type() == at::kBFloat16 ? BF16N_FP8_BF16 : BF16N_FP8_F32;
            return rest(*x, device, K);
        }
        const ref co(o, s_codes), sc(o, s_scales); // (the object keeps its tensors for the call)
        if (!co.o || !sc.o) {
            return false;
        }
        x = plain(co.o);
        const at::Tensor * s = plain(sc.o);
        if (!x || !s || x->scalar_type() != at::kFloat8_e4m3fn || s->scalar_type() != at::kFloat || s->get_device() != device || x->dim() != 2 || s->dim() != 2 ||
            s->size(0) != x->size(0) || s->size(1) != blocks_of(K)) {
            return false;
        }
        r.kind = BF16N_FP8_CODES;
        r.scales = (float *) s->data_ptr();
        r.scale_row = s->stride(0);
        r.scale_block = s->stride(1);
        return rest(*x, device, K);
    }
    bool rest(const at::Tensor & x, int device, int64_t K) {
        if (x.dim() != 2 || x.get_device() != device || x.size(0) <= 0 || x.size(0) > 1 << 28 || x.size(1) != K || x.stride(1) != 1) {
            return false;
        }
        r.at = x.data_ptr();
        r.row = x.stride(0) * x.element_size();
        rows = x.size(0);
        like = x.options().requires_grad(false);
        return r.row % 16 == 0 && (uintptr_t) r.at % 16 == 0;
    }
};

// a tensor beside `first`, which torch has just made, from the same allocator and past the dispatcher (0.3 us less than at::empty)
at::Tensor beside(const at::Tensor & first, at::IntArrayRef sizes, at::IntArrayRef strides, at::ScalarType type) {
    return at::Tensor(at::detail::empty_strided_generic(sizes, strides, first.storage().allocator(), first.key_set(), type));
}

// results: a tensor, or codes and scales
struct fp8_y {
    at::Tensor y, scales;
    bf16n_fp8_rows r = {};
    fp8_y(int64_t rows, int64_t n, int kind, const at::TensorOptions & like) {
        r.kind = kind;
        if (kind != BF16N_FP8_CODES) {
            y = at::empty({rows, n}, like.dtype(kind == BF16N_FP8_BF16 ? at::kBFloat16 : at::kFloat));
            r.at = y.data_ptr();
            r.row = n * y.element_size();
            return;
        }
        // (a storage for each: torch neither saves nor traces tensors of two types that share one)
        const int64_t blocks = blocks_of(n);
        y = at::empty({rows, n}, like.dtype(at::kFloat8_e4m3fn));
        scales = beside(y, {rows, blocks}, {1, rows}, at::kFloat);
        r.at = y.data_ptr();
        r.row = n;
        r.scales = (float *) scales.data_ptr();
        r.scale_row = 1;
        r.scale_block = rows;
    }
};

PyObject * tuple_of(std::initializer_list<const at::Tensor *> tensors) { // those that are there
    Py_ssize_t n = 0, i = 0;
    for (const at::Tensor * t : tensors) {
        n += t->defined();
    }
    PyObject * all = PyTuple_New(n);
    for (const at::Tensor * t : tensors) {
        if (all && t->defined()) {
            PyObject * o = THPVariable_Wrap(*t);
            if (!o) {
                Py_DECREF(all);
                return nullptr;
            }
            PyTuple_SET_ITEM(all, i++, o);
        }
    }
    return all;
}

// fp8_mm(x, w, up or None, kind of the result): the product, or (codes, scales)
PyObject * fp8_mm(PyObject *, PyObject * const * args, Py_ssize_t n) {
    try {
        if (n != 4 || !native_fp8()) {
            return not_taken();
        }
        const int device = c10::hip::current_device();
        bf16n_fp8_weight w, up;
        const bool glu = args[2] != Py_None;
        const int64_t kind = PyLong_AsLongLong(args[3]);
        fp8_x x;
        if (kind < 0 || kind > BF16N_FP8_F32 || !fp8_matrix(args[1], device, w) || w.n_matrices != 1 || (glu && (!fp8_matrix(args[2], device, up) || !alike(w, up))) ||
            !x.get(args[0], device, w.K) || (kind == BF16N_FP8_CODES && (!glu || w.rows % 16))) {
            return not_taken();
        }
        uint64_t bytes = 0;
        if (g_fp8_bytes(&w, glu, x.r.kind, (int) kind, x.rows, 0, 0, &bytes) != 0) {
            return not_taken();
        }
        fp8_y y(x.rows, w.rows, (int) kind, x.like);
        at::Tensor space;
        if (bytes) {
            space = at::empty({(int64_t) bytes}, x.like.dtype(at::kByte));
        }
        int status;
        {
            pybind11::gil_scoped_release free;
            status = g_fp8_mm(&w, glu ? &up : nullptr, &x.r, &y.r, x.rows, bytes ? space.data_ptr() : nullptr, bytes, stream_of(device));
        }
        return status != 0 ? PyLong_FromLong(status) : kind == BF16N_FP8_CODES ? tuple_of({&y.y, &y.scales}) : THPVariable_Wrap(y.y);
    } catch (const std::exception &) {
        return not_taken();
    }
}

// fp8_moe_experts(x, gate, up, down, topk_weights, topk_ids, n_experts) -> BF16 rows
PyObject * fp8_moe_experts(PyObject *, PyObject * const * args, Py_ssize_t n) {
    try {
        if (n != 7 || !native_fp8()) {
            return not_taken();
        }
        const int device = c10::hip::current_device();
        bf16n_fp8_weight gate, up, down;
        const int64_t E = PyLong_AsLongLong(args[6]);
        if (E <= 0 || !fp8_matrix(args[1], device, gate) || !fp8_matrix(args[2], device, up) || !fp8_matrix(args[3], device, down) || !alike(gate, up) || gate.n_matrices != E ||
            down.n_matrices != E || down.K != gate.rows / E) {
            return not_taken();
        }
        fp8_x x;
        const at::Tensor * wts = plain(args[4]), * ids = plain(args[5]);
        if (!wts || !ids || !x.get(args[0], device, gate.K) || ids->dim() != 2 || (ids->scalar_type() != at::kInt && ids->scalar_type() != at::kLong) || ids->get_device() != device ||
            ids->size(0) != x.rows || ids->size(1) <= 0 || ids->size(1) >= 1024 || x.rows > 65535 || ids->stride(1) != 1 || wts->dim() != 2 || wts->get_device() != device ||
            !wts->is_contiguous() || (wts->scalar_type() != at::kFloat && wts->scalar_type() != at::kBFloat16) || wts->size(0) != x.rows || wts->size(1) != ids->size(1)) {
            return not_taken();
        }
        const int T = (int) x.rows, slots = (int) ids->size(1), i64 = ids->scalar_type() == at::kLong, isz = i64 ? 8 : 4;
        uint64_t bytes = 0;
        if (g_fp8_experts_bytes(&gate, &down, x.r.kind, 1, T, slots, &bytes) != 0) {
            return not_taken();
        }
        fp8_y y(T, down.rows / E, BF16N_FP8_BF16, x.like);
        at::Tensor space = at::empty({(int64_t) bytes}, x.like.dtype(at::kByte));
        int status;
        {
            pybind11::gil_scoped_release free;
            status = g_fp8_experts(&gate, &up, &down, &x.r, ids->data_ptr(), i64, isz, ids->stride(0) * isz, wts->data_ptr(), wts->scalar_type() == at::kBFloat16, &y.r, T, slots,
                                   space.data_ptr(), bytes, stream_of(device));
        }
        return status != 0 ? PyLong_FromLong(status) : THPVariable_Wrap(y.y);
    } catch (const std::exception &) {
        return not_taken();
    }
}

// add_rmsnorm_fp8(a, b, c, ys, topk_weights, gamma (each of these five or None), eps, want_sum, want_norm) -> (codes, scales[, sum][, norm])
PyObject * add_rmsnorm_fp8(PyObject *, PyObject * const * args, Py_ssize_t n) {
    try {
        if (n != 9 || !native_fp8()) {
            return not_taken();
        }
        const int device = c10::hip::current_device();
        const at::Tensor * t[6];
        for (int i = 0; i < 6; i++) {
            t[i] = args[i] == Py_None ? nullptr : plain(args[i]);
            if (args[i] != Py_None && (!t[i] || t[i]->get_device() != device || !t[i]->is_contiguous())) {
                return not_taken();
            }
        }
        const at::Tensor * a = t[0], * ys = t[3], * wts = t[4], * gamma = t[5];
        const double eps = PyFloat_AsDouble(args[6]);
        if (PyErr_Occurred() || !a || a->dim() != 2 || a->size(0) <= 0 || a->size(0) > INT32_MAX || (gamma && (gamma->scalar_type() != at::kBFloat16 || gamma->numel() != a->size(1)))) {
            return not_taken();
        }
        const int64_t T = a->size(0), K = a->size(1);
        for (int i = 0; i < 3; i++) {
            if (t[i] && (t[i]->scalar_type() != at::kBFloat16 || t[i]->dim() != 2 || t[i]->size(0) != T || t[i]->size(1) != K)) {
                return not_taken();
            }
        }
        int64_t slots = 0;
        if (ys) {
            slots = ys->dim() == 3 ? ys->size(1) : 0;
            if (slots <= 0 || ys->scalar_type() != at::kFloat || ys->size(0) != T || ys->size(2) != K || !wts || wts->dim() != 2 || wts->size(0) != T || wts->size(1) != slots ||
                (wts->scalar_type() != at::kFloat && wts->scalar_type() != at::kBFloat16)) {
                return not_taken();
            }
        }
        if (K % 16 || K < 16 || K > 16384) {
            return not_taken();
        }
        fp8_y y(T, K, BF16N_FP8_CODES, on(*a, at::kBFloat16));
        at::Tensor sum, norm;
        if (args[7] == Py_True) {
            sum = beside(y.y, {T, K}, {K, 1}, at::kBFloat16);
        }
        if (args[8] == Py_True) {
            norm = beside(y.y, {T, K}, {K, 1}, at::kBFloat16);
        }
        const auto at_of = [](const at::Tensor * v) { return v ? v->data_ptr() : nullptr; };
        int status;
        {
            pybind11::gil_scoped_release free;
            status = g_fp8_norm((const uint16_t *) a->data_ptr(), (const uint16_t *) at_of(t[1]), (const uint16_t *) at_of(t[2]), (const float *) at_of(ys), ys ? at_of(wts) : nullptr,
                                ys && wts->scalar_type() == at::kBFloat16, (int) slots, (const uint16_t *) at_of(gamma), &y.r, sum.defined() ? (uint16_t *) sum.data_ptr() : nullptr,
                                norm.defined() ? (uint16_t *) norm.data_ptr() : nullptr, (int) T, K, (float) eps, stream_of(device));
        }
        return status != 0 ? PyLong_FromLong(status) : tuple_of({&y.y, &y.scales, &sum, &norm});
    } catch (const std::exception &) {
        return not_taken();
    }
}

PyObject * bind_fp8(PyObject *, PyObject * const * args, Py_ssize_t n) {
    if (n != 5) {
        PyErr_SetString(PyExc_TypeError, "bind_fp8: five addresses");
        return nullptr;
    }
    g_fp8_bytes = (fp8_bytes_fn) PyLong_AsVoidPtr(args[0]);
    g_fp8_experts_bytes = (fp8_experts_bytes_fn) PyLong_AsVoidPtr(args[2]);
    g_fp8_experts = (fp8_experts_fn) PyLong_AsVoidPtr(args[3]);
    g_fp8_norm = (fp8_norm_fn) PyLong_AsVoidPtr(args[4]);
    g_fp8_mm = (fp8_mm_fn) PyLong_AsVoidPtr(args[1]);
    if (PyErr_Occurred()) {
        g_fp8_mm = nullptr;
        return nullptr;
    }
    Py_RETURN_NONE;
}

PyObject * bind_int4(PyObject *, PyObject * const * args, Py_ssize_t n) {
    if (n != 6) {
        PyErr_SetString(PyExc_TypeError, "bind_int4: six addresses");
        return nullptr;
    }
    g_int4_bytes = (int4_bytes_fn) PyLong_AsVoidPtr(args[0]);
    g_int4_route = (int4_route_fn) PyLong_AsVoidPtr(args[2]);
    g_int4_mm_ids = (int4_mm_ids_fn) PyLong_AsVoidPtr(args[3]);
    g_combine = (combine_fn) PyLong_AsVoidPtr(args[4]);
    g_router = (router_fn) PyLong_AsVoidPtr(args[5]);
    g_int4_mmv = (int4_mmv_fn) PyLong_AsVoidPtr(args[1]);
    if (PyErr_Occurred()) {
        g_int4_mmv = nullptr;
        return nullptr;
    }
    Py_RETURN_NONE;
}

PyObject * bind(PyObject *, PyObject * const * args, Py_ssize_t n) {
    if (n != 3) {
        PyErr_SetString(PyExc_TypeError, "bind: three addresses");
        return nullptr;
    }
    g_mmv = (mmv_fn) PyLong_AsVoidPtr(args[0]);
    g_max_tokens = (max_tokens_fn) PyLong_AsVoidPtr(args[1]);
    g_dequant = (dequant_fn) PyLong_AsVoidPtr(args[2]);
    if (PyErr_Occurred()) {
        g_mmv = nullptr;
        return nullptr;
    }
    Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"mmv", (PyCFunction) (void (*)(void)) mmv, METH_FASTCALL, "the product, a status of the C ABI, or None: not taken"},
    {"linear", (PyCFunction) (void (*)(void)) linear, METH_FASTCALL, "the same for BF16 in and out and any number of tokens"},
    {"int4_mmv", (PyCFunction) (void (*)(void)) int4_mmv, METH_FASTCALL, "the dense product, plain or gated, of 4-bit weights with group scales"},
    {"int4_moe_experts", (PyCFunction) (void (*)(void)) int4_moe_experts, METH_FASTCALL, "routed experts on such weights"},
    {"router_topk_grouped", (PyCFunction) (void (*)(void)) router_topk_grouped, METH_FASTCALL, "(weights, ids), a status of the C ABI, or None"},
    {"bind_int4", (PyCFunction) (void (*)(void)) bind_int4, METH_FASTCALL,
     "the addresses of bf16n_int4_workspace_bytes, _mmv, _route, _mm_ids, bf16n_moe_combine, bf16n_router_topk_grouped"},
    {"fp8_mm", (PyCFunction) (void (*)(void)) fp8_mm, METH_FASTCALL, "the dense product in 8 bits, plain or gated: results, (codes, scales), a status or None"},
    {"fp8_moe_experts", (PyCFunction) (void (*)(void)) fp8_moe_experts, METH_FASTCALL, "routed experts in 8 bits"},
    {"add_rmsnorm_fp8", (PyCFunction) (void (*)(void)) add_rmsnorm_fp8, METH_FASTCALL, "(codes, scales[, sum][, norm]), a status of the C ABI, or None"},
    {"bind_fp8", (PyCFunction) (void (*)(void)) bind_fp8, METH_FASTCALL,
     "the addresses of bf16n_fp8_workspace_bytes, _fp8_mm, _fp8_moe_experts_workspace_bytes, _fp8_moe_experts, bf16n_add_rmsnorm_fp8"},
    {"bind", (PyCFunction) (void (*)(void)) bind, METH_FASTCALL, "the addresses of bf16n_mmv, bf16n_gemv_max_tokens, bf16n_dequant"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

} // namespace

PyMODINIT_FUNC PyInit__host(void) {
    PyObject ** const names[] = {&s_plane, &s_aux, &s_meta, &s_format, &s_K, &s_rows, &s_R, &s_cm, &s_frag, &s_w64, &s_off[0], &s_off[1], &s_off[2], &s_off[3],
                                 &s_codes, &s_scales, &s_zeros, &s_group, &s_n_matrices};
    const char * const text[] = {"plane", "aux", "meta", "format", "K", "rows", "R", "chunk_major", "frag_order", "wave64", "off_a", "off_b", "off_c", "off_d",
                                 "codes", "scales", "zeros", "group", "n_matrices"};
    for (size_t i = 0; i < sizeof(text) / sizeof(text[0]); i++) {
        if (!(*names[i] = PyUnicode_InternFromString(text[i]))) {
            return nullptr;
        }
    }
    // the release of torch whose internals are inlined above; the Python layer uses the module with no other
    PyObject * m = PyModule_Create(&g_module);
    if (m && PyModule_AddStringConstant(m, "built_for", BUILT_FOR) != 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
