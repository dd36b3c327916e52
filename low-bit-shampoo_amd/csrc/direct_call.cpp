// qtensor/_direct: the host side of one quantize or dequantize call of qtensor/functional.py, or of one call of an attention cache
// (qtensor/cache.py), of a projection (qtensor/linear.py) or of rotary positions (qtensor/rotary.py), in native code.
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
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <array>
#include <climits>
#include <cmath>
#include <initializer_list>
#include <memory>
#include <optional>
#include <utility>
#include <vector>

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
// A forward-mode derivative (torch.autograd.forward_ad): an ordinary tensor carries it, whatever the mode of gradients is.
bool has_tangent(const at::Tensor &t) { return t.unsafeGetTensorImpl()->autograd_meta() != nullptr && t._fw_grad(/*level=*/0).defined(); }
// Whether a derivative is asked for that a call without one would lose.
bool differentiated(const at::Tensor &t) { return (t.requires_grad() && c10::GradMode::is_enabled()) || has_tangent(t); }

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

// Whether a tensor has the shape that it was made with: as many elements in another order are not what the kernels read.
bool shaped(const at::Tensor &t, std::initializer_list<int64_t> sizes) { return t.sizes() == at::IntArrayRef(sizes.begin(), sizes.size()); }

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
// the same one and raises it in torch's words.  Python's own go through: they come from hooks on what a gradient saves, which have been called by then, and may be
// raised to be caught by whoever set them (a recomputed region ends in that way).
template <PyObject *(*body)(PyObject *const *), Py_ssize_t COUNT>
PyObject *guarded(PyObject *, PyObject *const *args, Py_ssize_t count) {
    if (count != COUNT || last_error == nullptr) Py_RETURN_NONE;
    try {
        return body(args);
    } catch (python_error &e) {
        e.restore();
    } catch (pybind11::error_already_set &e) {
        e.restore();
    } catch (...) {
    }
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
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
decltype(&qtensor_hip_cache_write_turned) write_turned_entry;
decltype(&qtensor_hip_cache_weigh) weigh_entry;
decltype(&qtensor_hip_cache_weigh_workspace) weigh_workspace_entry;
decltype(&qtensor_hip_cache_evict) evict_entry;
decltype(&qtensor_hip_cache_evict_workspace) evict_workspace_entry;
decltype(&qtensor_hip_linear_product) linear_entry;
decltype(&qtensor_hip_rotary_turn) turn_entry;

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
    if (codes->scalar_type() != at::kByte || scales->scalar_type() != at::kFloat || codes->dim() != 5) return false;
    const long long pages = codes->size(1), row = 16 * ((dim + 31) / 32), segments = (dim + blocksize - 1) / blocksize;
    if (pages < 1 || pages > INT_MAX || !shaped(*codes, {2, pages, heads, page_size, row}) || !shaped(*scales, {2, pages, heads, segments, page_size})) return false;
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
    if (differentiated(t)) return nullptr;
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

struct Angles { qtensor_rotary rotary; const at::Tensor *frequencies; };

// frequencies, magnitude, dims, interleaved: in heads of up to `most` elements
bool angles_of(PyObject *const *args, int device, long long most, Angles &a) {
    long long dims;
    a.frequencies = plain(args[0], device);
    if (a.frequencies == nullptr || !PyFloat_CheckExact(args[1]) || !whole(args[2], dims) || !PyBool_Check(args[3])) return false;
    if (dims < 2 || dims % 2 != 0 || dims > most || a.frequencies->scalar_type() != at::kDouble || !shaped(*a.frequencies, {dims / 2})) return false;
    a.rotary = {static_cast<const double *>(a.frequencies->data_ptr()), PyFloat_AS_DOUBLE(args[1]), (int)dims, args[3] == Py_True, 0};
    return true;
}

// First and last byte of a tensor's elements.
std::pair<const char *, const char *> span(const at::Tensor &t) {
    long long last = 0;
    for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
    const char *first = static_cast<const char *>(t.data_ptr());
    return {first, first + (last + 1) * t.element_size()};
}
// Whether the elements of a tensor [tokens, heads, head_dim] lie apart from each other.
bool apart_within(const at::Tensor &t) {
    const int64_t near = std::min(t.stride(0), t.stride(1)), far = std::max(t.stride(0), t.stride(1)), of_near = t.stride(0) < t.stride(1) ? t.size(0) : t.size(1);
    if (t.size(0) < 2 || t.size(1) < 2) return t.numel() == 0 || std::max(t.size(0), t.size(1)) < 2 || (t.size(0) < 2 ? t.stride(1) : t.stride(0)) >= t.size(2);
    return near >= t.size(2) && far >= near * (of_near - 1) + t.size(2);
}
bool apart(const at::Tensor &a, const at::Tensor &b) {
    if (a.numel() == 0 || b.numel() == 0) return true;
    const auto x = span(a), y = span(b);
    return x.second <= y.first || y.second <= x.first;
}

// cache_write_turned(codes, scales, page_size, kv_heads, head_dim, blocksize, frequencies, magnitude, dims, interleaved, q, keys, values, table,
// lengths, starts, positions, out) -> out or None
PyObject *cache_write_turned_checked(PyObject *const *args) {
    CacheCall c;
    Angles angles;
    qtensor_cache_vectors q, keys, values, result;
    if (write_turned_entry == nullptr || !cache_of(args, c) || !angles_of(args + 6, c.device, c.cache.head_dim, angles)) Py_RETURN_NONE;
    const at::Tensor *t = vectors_of(args[10], c, nullptr, -1, -1, q);
    if (t == nullptr || t->size(1) < 1 || t->size(1) > 32767) Py_RETURN_NONE;
    const at::Tensor *k = vectors_of(args[11], c, t, t->size(0), c.cache.kv_heads, keys), *v = vectors_of(args[12], c, t, t->size(0), c.cache.kv_heads, values);
    if (k == nullptr || v == nullptr || !places_of(args + 13, c, t->size(0))) Py_RETURN_NONE;
    const void *positions = nullptr;
    bool long_positions = false;
    if (args[16] != Py_None) {
        const at::Tensor *p = plain(args[16], c.device);
        if (p == nullptr || p->dim() != 1 || p->numel() != t->size(0) || (p->scalar_type() != at::kInt && p->scalar_type() != at::kLong)) Py_RETURN_NONE;
        positions = p->data_ptr(), long_positions = p->scalar_type() == at::kLong;
    }
    at::Tensor out;
    if (args[17] == Py_None) {
        out = at::empty({t->size(0), t->size(1), t->size(2)}, at::TensorOptions().device(t->device()).dtype(t->scalar_type()));
        if (!in_plain_memory(out, c.device)) Py_RETURN_NONE;
        result = {out.data_ptr(), q.is_bf16, out.stride(0), out.stride(1)};
    } else {
        const at::Tensor *given = vectors_of(args[17], c, t, t->size(0), t->size(1), result);
        if (given == nullptr || !apart_within(*given) || !apart(*given, *t) || !apart(*given, *k) || !apart(*given, *v)) Py_RETURN_NONE;
    }
    const int heads = (int)t->size(1);
    void *stream = stream_of(c);
    if (!launched([&] { write_turned_entry(&c.cache, &c.places, &angles.rotary, &q, &result, heads, &keys, &values, positions, long_positions, stream); })) return nullptr;
    if (args[17] != Py_None) {
        Py_INCREF(args[17]);
        return args[17];
    }
    return THPVariable_Wrap(std::move(out));
}

// Totals of the call's sequences, heads and places.
const at::Tensor *totals_of(PyObject *obj, const CacheCall &c) {
    const at::Tensor *t = plain(obj, c.device);
    return t != nullptr && t->scalar_type() == at::kFloat && t->dim() == 3 && t->size(0) == c.places.batch && t->size(1) == c.cache.kv_heads &&
                   t->size(2) >= (long long)c.places.table_pages * c.cache.page_size && c.places.batch <= 65535
               ? t
               : nullptr;
}

// cache_weigh(codes, scales, page_size, kv_heads, head_dim, blocksize, totals, q, table, lengths, starts, scale, window, sinks) -> totals or None
PyObject *cache_weigh_checked(PyObject *const *args) {
    CacheCall c;
    qtensor_cache_vectors q;
    long long window = 0, sinks;
    if (weigh_entry == nullptr || !cache_of(args, c)) Py_RETURN_NONE;
    const at::Tensor *t = vectors_of(args[7], c, nullptr, -1, -1, q);
    if (t == nullptr || t->size(1) < 1 || t->size(1) > 32767 || t->size(1) % c.cache.kv_heads != 0 || !places_of(args + 8, c, t->size(0))) Py_RETURN_NONE;
    const at::Tensor *totals = totals_of(args[6], c);
    const int heads = (int)t->size(1);
    if (totals == nullptr || t->size(0) * (heads / c.cache.kv_heads) >= 1ll << 27 || !apart(*totals, *t)) Py_RETURN_NONE;
    double scale = 1.0 / std::sqrt((double)c.cache.head_dim);
    if (args[11] != Py_None) {
        if (!PyFloat_CheckExact(args[11])) Py_RETURN_NONE;
        scale = PyFloat_AS_DOUBLE(args[11]);
    }
    if (args[12] != Py_None && (!whole(args[12], window) || window < 1)) Py_RETURN_NONE;
    if (!whole(args[13], sinks) || sinks < 0 || sinks > INT_MAX || window > INT_MAX || (sinks != 0 && window == 0) || !std::isfinite((float)scale)) Py_RETURN_NONE;
    const long long size = weigh_workspace_entry(&c.cache, &c.places, heads);
    if (size <= 0) Py_RETURN_NONE;
    at::Tensor scratch = at::empty({size}, at::TensorOptions().device(t->device()).dtype(at::kByte));
    if (!in_plain_memory(scratch, c.device)) Py_RETURN_NONE;
    void *stream = stream_of(c), *workspace = scratch.data_ptr();
    float *sums = static_cast<float *>(totals->data_ptr());
    const long long of_sequence = totals->stride(0), of_head = totals->stride(1);
    if (!launched([&] { weigh_entry(&c.cache, &c.places, &q, heads, (float)scale, (int)window, (int)sinks, sums, of_sequence, of_head, workspace, size, stream); }))
        return nullptr;
    Py_INCREF(args[6]);
    return args[6];
}

// cache_evict(codes, scales, page_size, kv_heads, head_dim, blocksize, totals, table, lengths, keep, recent, sinks) -> new lengths or None
PyObject *cache_evict_checked(PyObject *const *args) {
    CacheCall c;
    long long keep, recent, sinks;
    if (evict_entry == nullptr || !cache_of(args, c) || !THPVariable_CheckExact(args[8])) Py_RETURN_NONE;
    PyObject *where[3] = {args[7], args[8], Py_None};
    if (!places_of(where, c, THPVariable_Unpack(args[8]).numel())) Py_RETURN_NONE;
    const at::Tensor *totals = totals_of(args[6], c);
    if (totals == nullptr || !whole(args[9], keep) || !whole(args[10], recent) || !whole(args[11], sinks)) Py_RETURN_NONE;
    if (keep < 1 || recent < 0 || sinks < 0 || recent > keep || sinks > keep - recent) Py_RETURN_NONE;
    const long long size = evict_workspace_entry(&c.cache, &c.places, keep);
    if (size <= 0) Py_RETURN_NONE;
    const at::TensorOptions like = at::TensorOptions().device(totals->device());
    at::Tensor scratch = at::empty({size}, like.dtype(at::kByte)), out = at::empty({c.places.batch}, like.dtype(at::kInt));
    if (!in_plain_memory(scratch, c.device) || !in_plain_memory(out, c.device)) Py_RETURN_NONE;
    void *stream = stream_of(c), *workspace = scratch.data_ptr();
    float *sums = static_cast<float *>(totals->data_ptr());
    int *lengths = static_cast<int *>(out.data_ptr());
    const long long of_sequence = totals->stride(0), of_head = totals->stride(1);
    if (!launched([&] { evict_entry(&c.cache, &c.places, sums, of_sequence, of_head, keep, recent, sinks, lengths, workspace, size, stream); })) return nullptr;
    return THPVariable_Wrap(std::move(out));
}

// ------------------------------------------------------------------------------------------------ projections
// linear_product(codes, scales, inputs, outputs, blocksize, x, bias, out) -> out or None
PyObject *linear_product_checked(PyObject *const *args) {
    long long inputs, outputs, blocksize;
    if (linear_entry == nullptr || !THPVariable_CheckExact(args[0]) || !THPVariable_Unpack(args[0]).is_cuda() || watched()) Py_RETURN_NONE;
    const int device = c10::hip::current_device();
    const at::Tensor *codes = plain(args[0], device), *scales = plain(args[1], device);
    if (codes == nullptr || scales == nullptr || !whole(args[2], inputs) || !whole(args[3], outputs) || !whole(args[4], blocksize)) Py_RETURN_NONE;
    if (inputs < 1 || inputs > 1 << 24 || outputs < 1 || outputs > 1 << 24 || (blocksize != 64 && blocksize != 128 && blocksize != 256)) Py_RETURN_NONE;
    const long long tiles = (outputs + 15) / 16;
    if (codes->scalar_type() != at::kByte || scales->scalar_type() != at::kFloat || !shaped(*codes, {tiles, (inputs + 127) / 128, 1024}) ||
        !shaped(*scales, {tiles, (inputs + blocksize - 1) / blocksize, 16}))
        Py_RETURN_NONE;
    if (!THPVariable_CheckExact(args[5])) Py_RETURN_NONE;
    const at::Tensor &x = THPVariable_Unpack(args[5]);
    if (!in_memory(x, device) || slot_of(x.scalar_type()) < 0 || x.dim() < 1 || x.size(-1) != inputs || differentiated(x)) Py_RETURN_NONE;
    if (x.dim() == 2 ? inputs > 1 && x.stride(1) != 1 : !x.is_contiguous()) Py_RETURN_NONE;
    const long long tokens = x.numel() / inputs;
    const at::Tensor *bias = nullptr;
    if (args[6] != Py_None) {
        bias = plain(args[6], device);
        if (bias == nullptr || bias->numel() != outputs || (bias->scalar_type() != at::kFloat && bias->scalar_type() != x.scalar_type()) || differentiated(*bias))
            Py_RETURN_NONE;
    }
    at::Tensor out;
    if (args[7] == Py_None) {
        c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
        shape.back() = outputs;
        out = at::empty(shape, at::TensorOptions().device(x.device()).dtype(x.scalar_type()));
        if (!in_plain_memory(out, device)) Py_RETURN_NONE;
    } else {
        const at::Tensor *given = plain(args[7], device);
        if (given == nullptr || given->scalar_type() != x.scalar_type() || given->dim() != x.dim() || given->size(-1) != outputs || differentiated(*given) || !apart(*given, x) ||
            (bias != nullptr && !apart(*given, *bias)))
            Py_RETURN_NONE;
        for (int64_t d = 0; d + 1 < x.dim(); ++d)
            if (given->size(d) != x.size(d)) Py_RETURN_NONE;
        out = *given;
    }
    const qtensor_linear weights = {static_cast<unsigned char *>(codes->data_ptr()), static_cast<float *>(scales->data_ptr()), (int)inputs, (int)outputs, (int)blocksize};
    const qtensor_linear_call call = {x.data_ptr(), bias != nullptr ? bias->data_ptr() : nullptr, out.data_ptr(), x.dim() == 2 ? x.stride(0) : inputs, outputs, tokens,
                                      slot_of(x.scalar_type()), bias != nullptr && bias->scalar_type() == at::kBFloat16};
    void *stream = c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(device)).stream();
    if (!launched([&] { linear_entry(&weights, &call, stream); })) return nullptr;
    if (args[7] != Py_None) {
        Py_INCREF(args[7]);
        return args[7];
    }
    return THPVariable_Wrap(std::move(out));
}

// ------------------------------------------------------------------------------------------------ rotary positions
// Queries and keys (which may be undefined) that turn_fits has passed, turned or turned back.
bool turn_fits(const at::Tensor &t, const at::Tensor &first, int device, long long dims) {
    return in_memory(t, device) && t.scalar_type() == first.scalar_type() && slot_of(t.scalar_type()) >= 0 && (t.dim() == 3 || t.dim() == 4) && t.dim() == first.dim() &&
           t.size(-1) == first.size(-1) && t.size(-3) == first.size(-3) && t.size(0) == first.size(0) && t.size(-1) >= dims && t.size(-1) <= 1024 && t.size(-2) >= 1 &&
           t.size(-2) <= 32767 && t.stride(-1) == 1 && !has_tangent(t);
}
bool positions_fit(const at::Tensor &p, const at::Tensor &first, int device) {
    if (!in_memory(p, device) || (p.scalar_type() != at::kInt && p.scalar_type() != at::kLong) || p.dim() < 1 || p.dim() > first.dim() - 2) return false;
    return p.size(-1) == first.size(-3) && (p.dim() == 1 || p.size(0) == first.size(0)) && (p.size(-1) < 2 || p.stride(-1) == 1);
}
std::array<at::Tensor, 2> turned(const qtensor_rotary &rotary, const at::Tensor &q, const at::Tensor &k, const at::Tensor &positions) {
    std::array<at::Tensor, 2> out;
    qtensor_rotary_call call = {};
    for (const at::Tensor *t : {&q, &k}) {
        if (!t->defined()) continue;
        at::Tensor &y = out[t == &k];
        y = at::empty(t->sizes(), at::TensorOptions().device(t->device()).dtype(t->scalar_type()));
        TORCH_CHECK(in_plain_memory(y, (int)t->get_device()), "a result that is not in memory");
        const bool batch = t->dim() == 4;
        call.part[call.parts++] = {t->data_ptr(), y.data_ptr(), batch ? t->stride(0) : 0, t->stride(-3), t->stride(-2), batch ? y.stride(0) : 0, y.stride(-3), y.stride(-2),
                                   (int)t->size(-2)};
    }
    call.head_dim = (int)q.size(-1), call.is_bf16 = slot_of(q.scalar_type()), call.long_positions = positions.scalar_type() == at::kLong;
    call.batch = q.dim() == 4 ? q.size(0) : 1, call.tokens = q.size(-3), call.position_batch = positions.dim() == 2 ? positions.stride(0) : 0;
    call.positions = positions.data_ptr();
    turn_entry(&rotary, &call, c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(q.get_device())).stream());
    TORCH_CHECK(last_error() == 0, "libqtensor_hip: ", last_error_string());
    return out;
}

// The gradient of turning is turning back.  It is given what fits the kernel; gradients come as they are.
struct Turn : torch::autograd::Function<Turn> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const at::Tensor &q, const std::optional<at::Tensor> &k, const at::Tensor &positions,
                                                  const at::Tensor &frequencies, double magnitude, int64_t dims, bool interleaved, bool back) {
        ctx->save_for_backward({positions, frequencies});
        ctx->set_materialize_grads(false);
        ctx->saved_data["magnitude"] = magnitude, ctx->saved_data["dims"] = dims, ctx->saved_data["interleaved"] = interleaved, ctx->saved_data["back"] = back;
        const qtensor_rotary rotary = {static_cast<const double *>(frequencies.data_ptr()), magnitude, (int)dims, interleaved, back};
        std::array<at::Tensor, 2> out = turned(rotary, q, k.value_or(at::Tensor()), positions);
        return out[1].defined() ? torch::autograd::variable_list{out[0], out[1]} : torch::autograd::variable_list{out[0]};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
        torch::autograd::variable_list out(8);
        std::vector<at::Tensor> given;
        std::vector<int> whose;
        for (int i = 0; i < (int)grads.size(); ++i) {
            if (!grads[i].defined() || !ctx->needs_input_grad(i)) continue;
            given.push_back(grads[i].stride(-1) == 1 ? grads[i] : grads[i].contiguous());
            whose.push_back(i);
        }
        if (given.empty()) return out;
        // (what was saved comes back from hooks, which may give anything, and gradients are of whoever calls: a kernel reads them)
        const auto saved = ctx->get_saved_variables();
        const int device = (int)given[0].get_device();
        const int64_t dims = ctx->saved_data["dims"].toInt();
        for (const at::Tensor &d : given) TORCH_CHECK(turn_fits(d, given[0], device, dims), "gradients of turned queries and keys that are not in the GPU's memory");
        TORCH_CHECK(positions_fit(saved[0], given[0], device) && in_plain_memory(saved[1], device) && saved[1].scalar_type() == at::kDouble && shaped(saved[1], {dims / 2}),
                    "positions or frequencies that have come back from saved-tensor hooks as something else");
        const c10::OptionalDeviceGuard guard(given[0].device());
        const auto back = Turn::apply(given[0], given.size() > 1 ? std::optional<at::Tensor>(given[1]) : std::nullopt, saved[0], saved[1], ctx->saved_data["magnitude"].toDouble(),
                                      dims, ctx->saved_data["interleaved"].toBool(), !ctx->saved_data["back"].toBool());
        for (size_t n = 0; n < whose.size(); ++n) out[whose[n]] = back[n];
        return out;
    }
};

// rotary_turn(frequencies, magnitude, dims, interleaved, q, k, positions) -> (q, k) or None
PyObject *rotary_turn_checked(PyObject *const *args) {
    Angles angles;
    if (turn_entry == nullptr || !THPVariable_CheckExact(args[0]) || !THPVariable_Unpack(args[0]).is_cuda() || watched()) Py_RETURN_NONE;
    const int device = c10::hip::current_device();
    if (!angles_of(args, device, 1024, angles) || !THPVariable_CheckExact(args[4]) || !THPVariable_CheckExact(args[6])) Py_RETURN_NONE;
    const at::Tensor &q = THPVariable_Unpack(args[4]), &positions = THPVariable_Unpack(args[6]);
    if (!turn_fits(q, q, device, angles.rotary.dims) || !positions_fit(positions, q, device)) Py_RETURN_NONE;
    at::Tensor k;
    if (args[5] != Py_None) {
        if (!THPVariable_CheckExact(args[5])) Py_RETURN_NONE;
        k = THPVariable_Unpack(args[5]);
        if (!turn_fits(k, q, device, angles.rotary.dims)) Py_RETURN_NONE;
    }
    std::array<at::Tensor, 2> out;
    struct Unlocked {                       // (a full queue blocks; exceptions pass with the lock taken again)
        PyThreadState *state = PyEval_SaveThread();
        ~Unlocked() { PyEval_RestoreThread(state); }
    };
    const bool saves = c10::GradMode::is_enabled() && (q.requires_grad() || (k.defined() && k.requires_grad()));
    // (what torch does not save: found out before hooks on the rest have been called)
    if (saves && (angles.frequencies->is_inference() || positions.is_inference())) Py_RETURN_NONE;
    auto unlocked = std::make_unique<Unlocked>();
    if (saves) {
        const auto both = Turn::apply(q, k.defined() ? std::optional<at::Tensor>(k) : std::nullopt, positions, *angles.frequencies, angles.rotary.magnitude, (int64_t)angles.rotary.dims, angles.rotary.interleaved != 0, false);
        out = {both[0], both.size() > 1 ? both[1] : at::Tensor()};
    } else {
        out = turned(angles.rotary, q, k, positions);
    }
    unlocked.reset();
    PyObject *result = PyTuple_New(2);
    if (result == nullptr) return nullptr;
    PyTuple_SET_ITEM(result, 0, THPVariable_Wrap(std::move(out[0])));
    if (out[1].defined()) {
        PyTuple_SET_ITEM(result, 1, THPVariable_Wrap(std::move(out[1])));
    } else {
        Py_INCREF(Py_None);
        PyTuple_SET_ITEM(result, 1, Py_None);
    }
    return result;
}

// Takes `count` addresses from a sequence; false with a Python error set.
bool addresses_of(PyObject *list, const char *what, Py_ssize_t count, void **address) {
    PyObject *items = PySequence_Fast(list, "a sequence of addresses is wanted");
    if (items == nullptr) return false;
    bool good = PySequence_Fast_GET_SIZE(items) == count;
    for (Py_ssize_t i = 0; good && i < count; ++i) {
        address[i] = PyLong_AsVoidPtr(PySequence_Fast_GET_ITEM(items, i));
        good = address[i] != nullptr;
    }
    Py_DECREF(items);
    if (!good && !PyErr_Occurred()) PyErr_Format(PyExc_ValueError, "%s takes %zd addresses", what, count);
    return good;
}

// bind_model(addresses): the linear product, rotary turn, the cache's write_turned, weigh, weigh's workspace, evict, evict's workspace
PyObject *bind_model(PyObject *, PyObject *list) {
    void *address[7];
    if (!addresses_of(list, "bind_model", 7, address)) return nullptr;
    linear_entry = reinterpret_cast<decltype(linear_entry)>(address[0]);
    turn_entry = reinterpret_cast<decltype(turn_entry)>(address[1]);
    write_turned_entry = reinterpret_cast<decltype(write_turned_entry)>(address[2]);
    weigh_entry = reinterpret_cast<decltype(weigh_entry)>(address[3]);
    weigh_workspace_entry = reinterpret_cast<decltype(weigh_workspace_entry)>(address[4]);
    evict_entry = reinterpret_cast<decltype(evict_entry)>(address[5]);
    evict_workspace_entry = reinterpret_cast<decltype(evict_workspace_entry)>(address[6]);
    Py_RETURN_NONE;
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
    {"cache_write_turned", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<cache_write_turned_checked, 18>)), METH_FASTCALL,
     "cache_write_turned(codes, scales, page_size, kv_heads, head_dim, blocksize, frequencies, magnitude, dims, interleaved, q, keys, values, table, lengths, starts, positions, out): out, None if not taken"},
    {"cache_weigh", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<cache_weigh_checked, 14>)), METH_FASTCALL,
     "cache_weigh(codes, scales, page_size, kv_heads, head_dim, blocksize, totals, q, table, lengths, starts, scale, window, sinks): totals, None if not taken"},
    {"cache_evict", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<cache_evict_checked, 12>)), METH_FASTCALL,
     "cache_evict(codes, scales, page_size, kv_heads, head_dim, blocksize, totals, table, lengths, keep, recent, sinks): new lengths, None if not taken"},
    {"bind_model", bind_model, METH_O, "addresses of the library's entry points for projections, rotary positions and eviction"},
    {"linear_product", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<linear_product_checked, 8>)), METH_FASTCALL,
     "linear_product(codes, scales, inputs, outputs, blocksize, x, bias, out): out, None if not taken"},
    {"rotary_turn", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<rotary_turn_checked, 7>)), METH_FASTCALL,
     "rotary_turn(frequencies, magnitude, dims, interleaved, q, k, positions): (q, k), None if not taken"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_direct", "one call of the quantizers, an attention cache, a projection or rotary positions in native code", -1, methods, nullptr, nullptr, nullptr, nullptr};

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
