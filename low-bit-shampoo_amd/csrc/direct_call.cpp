// qtensor/_direct: the host side of one quantize or dequantize call of qtensor/functional.py, or of one call of an attention cache
// (qtensor/cache.py), in native code.
//
// A call on a small matrix is bound by its host side: kernels of 4 to 6 us, and 9 us of Python around each (checks, two or
// three torch.empty, data_ptr, ctypes, the error slot).  This is the same sequence behind one call: what the tensors are is
// checked, buffers that are not given come from torch's allocator, the launch goes to torch's current stream through the
// library's entry point, the error slot is read.  Quantized and dequantized with an exact diagonal, calls back to back: 256 x 256
// 17.9 -> 12.1 us (the kernels are what is left), 1200 x 1200 17.7 -> 11.1.
//
// It takes plainly good calls only.  Anything else -- an argument that is not what it should be, a device that is not the current one, a
// tensor subclass or wrapper, a function or dispatch mode, a transformation (torch.func) or trace around the call -- returns None,
// nothing launched, and the caller's own checks say what is wrong or do it the long way: there is one place that words errors.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cmath>

#include "qtensor_hip.h"

namespace {

using Plain = void (*)(const void *, const void *, int, void *, void *, int, void *);
using WithDiagonal = void (*)(const void *, const void *, int, void *, void *, void *, int, void *);
// [quantize, dequantize][4, 8 bits][fp32, bf16][plain, exact diagonal]: entry points of libqtensor_hip.so (include/qtensor_hip.h)
void *entry[2][2][2][2];
int (*last_error)();
const char *(*last_error_string)();

using K = c10::DispatchKey;

// Memory of the GPU `device` and nothing around it: no wrapper that a transformation or mode has made.
bool in_memory(const at::Tensor &t, int device) {
    static const c10::DispatchKeySet wrapped({K::Python, K::PythonTLSSnapshot, K::FuncTorchBatched, K::FuncTorchGradWrapper, K::Functionalize,
                                              K::Batched, K::Conjugate, K::Negative, K::ZeroTensor});
    return t.defined() && t.is_cuda() && t.layout() == at::kStrided && !t.key_set().has_any(wrapped) && t.has_storage() &&
           t.get_device() == device;
}
bool in_plain_memory(const at::Tensor &t, int device) { return in_memory(t, device) && t.is_contiguous(); }

// A tensor that is itself (no subclass), in plain memory of the current GPU.
const at::Tensor *plain(PyObject *obj, int device) {
    if (!THPVariable_CheckExact(obj)) return nullptr;
    const at::Tensor &t = THPVariable_Unpack(obj);
    return in_plain_memory(t, device) ? &t : nullptr;
}

// Whether something is set up around the call that would see, or wrap, the tensors it makes: with plain inputs, too, what
// at::empty returns inside a level of torch.func is a wrapper without memory of its own.
bool watched() {
    static const c10::DispatchKeySet levels({K::Python, K::PythonTLSSnapshot, K::PythonDispatcher, K::PreDispatch, K::Functionalize, K::Tracer,
                                             K::FuncTorchVmapMode, K::VmapMode, K::FuncTorchDynamicLayerFrontMode,
                                             K::FuncTorchDynamicLayerBackMode});
    return c10::impl::tls_local_dispatch_key_set().included_.has_any(levels) || at::impl::torch_function_mode_enabled();
}

// A buffer of `numel` elements: false where what is given does not fit; made if nothing is given.
bool buffer(PyObject *given, int device, long long numel, at::ScalarType type, const at::TensorOptions &like, at::Tensor &out) {
    if (given == Py_None) {
        out = at::empty({numel}, like.dtype(type));
        return in_plain_memory(out, device);
    }
    const at::Tensor *t = plain(given, device);
    if (t == nullptr || t->scalar_type() != type || t->numel() != numel) return false;
    out = *t;
    return true;
}

bool whole(PyObject *obj, long long &value) {
    if (!PyLong_CheckExact(obj)) return false;
    int overflow = 0;
    value = PyLong_AsLongLongAndOverflow(obj, &overflow);
    return overflow == 0;
}

struct Format { long long order, blocksize, bits, codes, maxima; int device; };
bool format(PyObject *data, PyObject *order, PyObject *blocksize, PyObject *bits, Format &f) {
    // (before the device is asked for: that would start the GPU's runtime for a tensor that is not there)
    if (!THPVariable_CheckExact(data) || !THPVariable_Unpack(data).is_cuda()) return false;
    if (!whole(order, f.order) || !whole(blocksize, f.blocksize) || !whole(bits, f.bits)) return false;
    if (f.bits != 4 && f.bits != 8) return false;
    if (f.blocksize < 64 || f.blocksize > 2048 || (f.blocksize & (f.blocksize - 1)) != 0) return false;
    if (f.order < 1 || f.order > 46340 || watched()) return false;
    f.codes = (f.order * f.order * f.bits + 7) / 8;
    f.maxima = f.order * ((f.order + f.blocksize - 1) / f.blocksize);
    f.device = c10::hip::current_device();
    return true;
}

const at::Tensor *code_table(PyObject *obj, const Format &f) {
    const at::Tensor *t = plain(obj, f.device);
    return t != nullptr && t->scalar_type() == at::kFloat && t->dim() == 1 && t->numel() == (1ll << f.bits) ? t : nullptr;
}

int slot_of(at::ScalarType type) { return type == at::kFloat ? 0 : type == at::kBFloat16 ? 1 : -1; }

// The launch itself, without the interpreter's lock (a full queue blocks); false with a Python error set.  Addresses first:
// asking for one may throw (a lazy copy that has to be made, memory that is not there), and nothing may between letting go
// of the lock and taking it again.
bool launch(void *fn, const at::Tensor &a, const at::Tensor &code, const Format &f, const at::Tensor &absmax, const at::Tensor *diag,
            const at::Tensor &out) {
    void *stream = c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(f.device)).stream();
    const void *from = a.data_ptr(), *table = code.data_ptr();
    void *maxima = absmax.data_ptr(), *diagonal = diag != nullptr ? diag->data_ptr() : nullptr, *to = out.data_ptr();
    const int order = (int)f.order, blocksize = (int)f.blocksize;
    const bool with_diag = diag != nullptr;
    int error = 0;
    Py_BEGIN_ALLOW_THREADS
    if (with_diag) reinterpret_cast<WithDiagonal>(fn)(from, table, order, maxima, diagonal, to, blocksize, stream);
    else reinterpret_cast<Plain>(fn)(from, table, order, maxima, to, blocksize, stream);
    error = last_error();
    Py_END_ALLOW_THREADS
    if (error == 0) return true;
    PyErr_Format(PyExc_RuntimeError, "libqtensor_hip: %s", last_error_string());
    return false;
}

// quantize(A, code, order, absmax, diag, out, blocksize, bits, with_diag) -> (out, absmax[, diag]) or None
PyObject *quantize_checked(PyObject *const *args) {
    Format f;
    if (!format(args[0], args[2], args[6], args[7], f)) Py_RETURN_NONE;
    const bool with_diag = args[8] == Py_True;
    const at::Tensor *a = plain(args[0], f.device), *code = code_table(args[1], f);
    if (a == nullptr || code == nullptr || a->numel() != f.order * f.order) Py_RETURN_NONE;
    const int slot = slot_of(a->scalar_type());
    if (slot < 0) Py_RETURN_NONE;
    const at::TensorOptions like = at::TensorOptions().device(a->device());
    at::Tensor out, absmax, diag;
    if (!buffer(args[3], f.device, f.maxima, at::kFloat, like, absmax) ||
        (with_diag && !buffer(args[4], f.device, f.order, at::kFloat, like, diag)) ||
        !buffer(args[5], f.device, f.codes, at::kByte, like, out)) Py_RETURN_NONE;
    if (!launch(entry[0][f.bits == 8][slot][with_diag], *a, *code, f, absmax, with_diag ? &diag : nullptr, out)) return nullptr;
    PyObject *result = PyTuple_New(with_diag ? 3 : 2);
    if (result == nullptr) return nullptr;
    auto put = [&](int i, PyObject *given, at::Tensor &t) {
        if (given != Py_None) Py_INCREF(given);
        PyTuple_SET_ITEM(result, i, given != Py_None ? given : THPVariable_Wrap(std::move(t)));
    };
    put(0, args[5], out);
    put(1, args[3], absmax);
    if (with_diag) put(2, args[4], diag);
    return result;
}

// dequantize(A, code, order, absmax, diag, outdtype, out, blocksize, bits, with_diag) -> out or None
PyObject *dequantize_checked(PyObject *const *args) {
    Format f;
    if (!format(args[0], args[2], args[7], args[8], f)) Py_RETURN_NONE;
    const bool with_diag = args[9] == Py_True;
    const at::Tensor *a = plain(args[0], f.device), *code = code_table(args[1], f), *absmax = plain(args[3], f.device);
    if (a == nullptr || code == nullptr || absmax == nullptr) Py_RETURN_NONE;
    if (a->scalar_type() != at::kByte || a->numel() != f.codes || absmax->scalar_type() != at::kFloat || absmax->numel() != f.maxima) Py_RETURN_NONE;
    const at::Tensor *diag = with_diag ? plain(args[4], f.device) : nullptr;
    if (with_diag && (diag == nullptr || diag->scalar_type() != at::kFloat || diag->numel() != f.order)) Py_RETURN_NONE;
    at::Tensor out;
    if (args[6] == Py_None) {
        if (!THPDtype_Check(args[5])) Py_RETURN_NONE;
        const at::ScalarType type = reinterpret_cast<THPDtype *>(args[5])->scalar_type;
        if (slot_of(type) < 0) Py_RETURN_NONE;
        out = at::empty({f.order, f.order}, at::TensorOptions().device(a->device()).dtype(type));
        if (!in_plain_memory(out, f.device)) Py_RETURN_NONE;
    } else {
        const at::Tensor *t = plain(args[6], f.device);
        if (t == nullptr || t->numel() != f.order * f.order) Py_RETURN_NONE;
        out = *t;
    }
    const int slot = slot_of(out.scalar_type());
    if (slot < 0) Py_RETURN_NONE;
    if (!launch(entry[1][f.bits == 8][slot][with_diag], *a, *code, f, *absmax, diag, out)) return nullptr;
    if (args[6] != Py_None) {
        Py_INCREF(args[6]);
        return args[6];
    }
    return THPVariable_Wrap(std::move(out));
}

// C++ exceptions (out of memory, a failed look-up) end here, with the interpreter's lock held: the caller's long way meets
// the same one and raises it in torch's words.
template <PyObject *(*body)(PyObject *const *), Py_ssize_t COUNT>
PyObject *guarded(PyObject *, PyObject *const *args, Py_ssize_t count) {
    if (count != COUNT || last_error == nullptr) Py_RETURN_NONE;
    try {
        return body(args);
    } catch (...) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
}

// bind(addresses): the sixteen entry points in the order of `entry`, the two of the error slot
PyObject *bind(PyObject *, PyObject *list) {
    void *address[18];
    PyObject *items = PySequence_Fast(list, "bind takes a sequence of addresses");
    if (items == nullptr) return nullptr;
    if (PySequence_Fast_GET_SIZE(items) != 18) {
        Py_DECREF(items);
        PyErr_SetString(PyExc_ValueError, "bind takes eighteen addresses");
        return nullptr;
    }
    for (int i = 0; i < 18; ++i) address[i] = PyLong_AsVoidPtr(PySequence_Fast_GET_ITEM(items, i));
    Py_DECREF(items);
    if (PyErr_Occurred()) return nullptr;
    for (int i = 0; i < 18; ++i)
        if (address[i] == nullptr) {
            PyErr_SetString(PyExc_ValueError, "bind: null address");
            return nullptr;
        }
    for (int i = 0; i < 16; ++i) entry[i >> 3][(i >> 2) & 1][(i >> 1) & 1][i & 1] = address[i];
    last_error_string = reinterpret_cast<const char *(*)()>(address[17]);
    last_error = reinterpret_cast<int (*)()>(address[16]);
    Py_RETURN_NONE;
}

// ------------------------------------------------------------------------------------------------ the attention cache
using Copy = decltype(&qtensor_hip_cache_write);
Copy cache_write_entry, cache_read_entry;
decltype(&qtensor_hip_cache_attend) cache_attend_entry;
decltype(&qtensor_hip_cache_attend_workspace) cache_workspace_entry;

struct CacheCall {
    qtensor_cache cache;
    qtensor_cache_places places;
    int device;
};

// codes, scales, page_size, kv_heads, head_dim, blocksize
bool cache_of(PyObject *const *args, CacheCall &c) {
    if (!THPVariable_CheckExact(args[0]) || !THPVariable_Unpack(args[0]).is_cuda() || watched()) return false;
    c.device = c10::hip::current_device();
    const at::Tensor *codes = plain(args[0], c.device), *scales = plain(args[1], c.device);
    long long page_size, heads, dim, blocksize;
    if (codes == nullptr || scales == nullptr || !whole(args[2], page_size) || !whole(args[3], heads) || !whole(args[4], dim) || !whole(args[5], blocksize))
        return false;
    if (page_size < 16 || page_size > 4096 || heads < 1 || heads > 32767 || dim < 1 || dim > 256 || (blocksize != 64 && blocksize != 128 && blocksize != 256))
        return false;
    if (codes->scalar_type() != at::kByte || scales->scalar_type() != at::kFloat || codes->dim() != 5 || scales->dim() != 5) return false;
    const long long pages = codes->size(1), row = 16 * ((dim + 31) / 32), segments = (dim + blocksize - 1) / blocksize;
    if (pages < 1 || pages > INT_MAX || codes->numel() != 2 * pages * heads * page_size * row || scales->numel() != 2 * pages * heads * page_size * segments)
        return false;
    auto *bytes = static_cast<unsigned char *>(codes->data_ptr());
    auto *floats = static_cast<float *>(scales->data_ptr());
    c.cache = {{bytes, bytes + codes->numel() / 2}, {floats, floats + scales->numel() / 2}, (int)pages, (int)page_size, (int)heads, (int)dim, (int)blocksize};
    return true;
}

// table, lengths, starts
bool places_of(PyObject *const *args, CacheCall &c, long long tokens) {
    if (!THPVariable_CheckExact(args[0])) return false;
    const at::Tensor &table = THPVariable_Unpack(args[0]);
    const at::Tensor *lengths = plain(args[1], c.device);
    if (!in_memory(table, c.device) || lengths == nullptr || table.scalar_type() != at::kInt || lengths->scalar_type() != at::kInt) return false;
    const long long batch = lengths->numel();
    if (batch < 1 || batch > INT_MAX || table.dim() != 2 || table.size(0) != batch || table.size(1) < 1 || table.size(1) > INT_MAX ||
        (table.size(1) > 1 && table.stride(1) != 1) || tokens < 0 || tokens > INT_MAX)
        return false;
    const int *starts = nullptr;
    if (args[2] != Py_None) {
        const at::Tensor *t = plain(args[2], c.device);
        if (t == nullptr || t->scalar_type() != at::kInt || t->numel() != batch + 1) return false;
        starts = static_cast<const int *>(t->data_ptr());
    } else if (tokens != batch) {
        return false;
    }
    c.places = {static_cast<const int *>(table.data_ptr()), static_cast<const int *>(lengths->data_ptr()), starts, table.stride(0), (int)table.size(1),
                (int)batch, (int)tokens};
    return true;
}

// Vectors [tokens, heads, dim] of fp32 or bf16 (of `like`'s type, if given); tokens or heads of -1: as they come.
const at::Tensor *vectors_of(PyObject *obj, const CacheCall &c, const at::Tensor *like, long long tokens, long long heads, qtensor_cache_vectors &out) {
    if (!THPVariable_CheckExact(obj)) return nullptr;
    const at::Tensor &t = THPVariable_Unpack(obj);
    if (!in_memory(t, c.device) || t.dim() != 3 || slot_of(t.scalar_type()) < 0 || t.size(2) != c.cache.head_dim || (t.size(2) > 1 && t.stride(2) != 1)) return nullptr;
    if ((like != nullptr && t.scalar_type() != like->scalar_type()) || (tokens >= 0 && t.size(0) != tokens) || (heads >= 0 && t.size(1) != heads)) return nullptr;
    if (t.requires_grad() && c10::GradMode::is_enabled()) return nullptr;
    out = {t.data_ptr(), slot_of(t.scalar_type()), t.stride(0), t.stride(1)};
    return &t;
}

template <typename Launch>
bool launched(Launch launch) {
    int error = 0;
    Py_BEGIN_ALLOW_THREADS
    launch();
    error = last_error();
    Py_END_ALLOW_THREADS
    if (error == 0) return true;
    PyErr_Format(PyExc_RuntimeError, "libqtensor_hip: %s", last_error_string());
    return false;
}

void *stream_of(const CacheCall &c) { return c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(c.device)).stream(); }

// cache_write(codes, scales, page_size, kv_heads, head_dim, blocksize, keys, values, table, lengths, starts) -> True or None
PyObject *cache_write_checked(PyObject *const *args) {
    CacheCall c;
    qtensor_cache_vectors keys, values;
    if (cache_write_entry == nullptr || !cache_of(args, c)) Py_RETURN_NONE;
    const at::Tensor *k = vectors_of(args[6], c, nullptr, -1, c.cache.kv_heads, keys);
    if (k == nullptr || vectors_of(args[7], c, k, k->size(0), c.cache.kv_heads, values) == nullptr || !places_of(args + 8, c, k->size(0))) Py_RETURN_NONE;
    void *stream = stream_of(c);
    if (!launched([&] { cache_write_entry(&c.cache, &c.places, &keys, &values, stream); })) return nullptr;
    Py_RETURN_TRUE;
}

// cache_read(codes, scales, page_size, kv_heads, head_dim, blocksize, table, lengths, starts, tokens, dtype) -> (keys, values) or None
PyObject *cache_read_checked(PyObject *const *args) {
    CacheCall c;
    long long tokens;
    if (cache_read_entry == nullptr || !cache_of(args, c) || !whole(args[9], tokens) || !places_of(args + 6, c, tokens) || !THPDtype_Check(args[10])) Py_RETURN_NONE;
    const at::ScalarType type = reinterpret_cast<THPDtype *>(args[10])->scalar_type;
    if (slot_of(type) < 0) Py_RETURN_NONE;
    const at::TensorOptions like = at::TensorOptions().device(at::kCUDA, static_cast<c10::DeviceIndex>(c.device)).dtype(type);
    at::Tensor out[2];
    qtensor_cache_vectors vectors[2];
    for (int i = 0; i < 2; ++i) {
        out[i] = at::empty({tokens, c.cache.kv_heads, c.cache.head_dim}, like);
        if (!in_plain_memory(out[i], c.device)) Py_RETURN_NONE;
        vectors[i] = {out[i].data_ptr(), slot_of(type), out[i].stride(0), out[i].stride(1)};
    }
    void *stream = stream_of(c);
    if (!launched([&] { cache_read_entry(&c.cache, &c.places, &vectors[0], &vectors[1], stream); })) return nullptr;
    PyObject *result = PyTuple_New(2);
    if (result == nullptr) return nullptr;
    for (int i = 0; i < 2; ++i) PyTuple_SET_ITEM(result, i, THPVariable_Wrap(std::move(out[i])));
    return result;
}

// cache_attend(codes, scales, page_size, kv_heads, head_dim, blocksize, q, table, lengths, starts, scale, window, sinks, out) -> out or None
PyObject *cache_attend_checked(PyObject *const *args) {
    CacheCall c;
    qtensor_cache_vectors q, result;
    long long window = 0, sinks;
    if (cache_attend_entry == nullptr || !cache_of(args, c)) Py_RETURN_NONE;
    const at::Tensor *t = vectors_of(args[6], c, nullptr, -1, -1, q);
    if (t == nullptr || t->size(1) < 1 || t->size(1) > 32767 || t->size(1) % c.cache.kv_heads != 0 || !places_of(args + 7, c, t->size(0))) Py_RETURN_NONE;
    double scale = 1.0 / std::sqrt((double)c.cache.head_dim);
    if (args[10] != Py_None) {
        if (!PyFloat_CheckExact(args[10])) Py_RETURN_NONE;
        scale = PyFloat_AS_DOUBLE(args[10]);
    }
    if (args[11] != Py_None && (!whole(args[11], window) || window < 1)) Py_RETURN_NONE;
    if (!whole(args[12], sinks) || sinks < 0 || sinks > INT_MAX || window > INT_MAX || (sinks != 0 && window == 0) || !std::isfinite((float)scale)) Py_RETURN_NONE;
    at::Tensor out;
    if (args[13] == Py_None) {
        out = at::empty({t->size(0), t->size(1), t->size(2)}, at::TensorOptions().device(t->device()).dtype(t->scalar_type()));
        if (!in_plain_memory(out, c.device)) Py_RETURN_NONE;
        result = {out.data_ptr(), q.is_bf16, out.stride(0), out.stride(1)};
    } else if (vectors_of(args[13], c, t, t->size(0), t->size(1), result) == nullptr) {
        Py_RETURN_NONE;
    }
    const int heads = (int)t->size(1);
    const long long size = cache_workspace_entry(&c.cache, heads, q.is_bf16, c.places.starts != nullptr);
    if (size <= 0) Py_RETURN_NONE;
    at::Tensor scratch = at::empty({size}, at::TensorOptions().device(t->device()).dtype(at::kByte));
    if (!in_plain_memory(scratch, c.device)) Py_RETURN_NONE;
    void *stream = stream_of(c), *workspace = scratch.data_ptr();
    if (!launched([&] { cache_attend_entry(&c.cache, &c.places, &q, &result, heads, (float)scale, (int)window, (int)sinks, workspace, size, stream); })) return nullptr;
    if (args[13] != Py_None) {
        Py_INCREF(args[13]);
        return args[13];
    }
    return THPVariable_Wrap(std::move(out));
}

// bind_cache(addresses): write, read, attend, attend's workspace
PyObject *bind_cache(PyObject *, PyObject *list) {
    PyObject *items = PySequence_Fast(list, "bind_cache takes a sequence of addresses");
    if (items == nullptr) return nullptr;
    void *address[4] = {};
    const bool four = PySequence_Fast_GET_SIZE(items) == 4;
    for (int i = 0; four && i < 4; ++i) address[i] = PyLong_AsVoidPtr(PySequence_Fast_GET_ITEM(items, i));
    Py_DECREF(items);
    if (PyErr_Occurred()) return nullptr;
    if (!four || address[0] == nullptr || address[1] == nullptr || address[2] == nullptr || address[3] == nullptr) {
        PyErr_SetString(PyExc_ValueError, "bind_cache takes four addresses");
        return nullptr;
    }
    cache_write_entry = reinterpret_cast<Copy>(address[0]);
    cache_read_entry = reinterpret_cast<Copy>(address[1]);
    cache_attend_entry = reinterpret_cast<decltype(cache_attend_entry)>(address[2]);
    cache_workspace_entry = reinterpret_cast<decltype(cache_workspace_entry)>(address[3]);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", bind, METH_O, "addresses of the library's entry points"},
    {"quantize", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<quantize_checked, 9>)), METH_FASTCALL,
     "quantize(A, code, order, absmax, diag, out, blocksize, bits, with_diag): (out, absmax[, diag]), None if not taken"},
    {"dequantize", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<dequantize_checked, 10>)), METH_FASTCALL,
     "dequantize(A, code, order, absmax, diag, outdtype, out, blocksize, bits, with_diag): out, None if not taken"},
    {"bind_cache", bind_cache, METH_O, "addresses of the library's entry points for attention caches"},
    {"cache_write", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<cache_write_checked, 11>)), METH_FASTCALL,
     "cache_write(codes, scales, page_size, kv_heads, head_dim, blocksize, keys, values, table, lengths, starts): True, None if not taken"},
    {"cache_read", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<cache_read_checked, 11>)), METH_FASTCALL,
     "cache_read(codes, scales, page_size, kv_heads, head_dim, blocksize, table, lengths, starts, tokens, dtype): (keys, values), None if not taken"},
    {"cache_attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<cache_attend_checked, 14>)), METH_FASTCALL,
     "cache_attend(codes, scales, page_size, kv_heads, head_dim, blocksize, q, table, lengths, starts, scale, window, sinks, out): out, None if not taken"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_direct", "one quantize, dequantize or attention cache call in native code", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// torch_version: what this was compiled against.  It reads torch's objects as they lie in memory, which no other torch promises.
PyMODINIT_FUNC PyInit__direct() {
    PyObject *made = PyModule_Create(&module);
    if (made != nullptr && PyModule_AddStringConstant(made, "torch_version", QT_TORCH_VERSION) != 0) {
        Py_DECREF(made);
        return nullptr;
    }
    return made;
}
