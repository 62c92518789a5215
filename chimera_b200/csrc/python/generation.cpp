// Python module chimera_b200._generation: the generation operators over torch
// tensors.  It checks what tensors can get wrong (kinds, devices, shapes,
// layouts), allocates outputs where none are given, and calls the C ABI on the
// current stream of the tensors' device.  chimera_b200/attention.py documents
// the calls; these functions take the same arguments by position.
//
// A call here costs the host a few microseconds; the same checks in Python cost
// 25 to 40, more than the small calls' kernels.
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/Functions.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "chimera_b200.h"

namespace {

using at::ScalarType;
using at::Tensor;

int type_of(ScalarType t) {
    switch (t) {
        case ScalarType::Float: return CHM_FP32;
        case ScalarType::Half: return CHM_FP16;
        case ScalarType::BFloat16: return CHM_BF16;
        case ScalarType::Char: return CHM_INT8;
        case ScalarType::Float8_e4m3fn: return CHM_E4M3;
        default: return -1;
    }
}
bool is_vector_type(int t) { return t == CHM_FP32 || t == CHM_FP16 || t == CHM_BF16; }

// The tensor an argument holds.  It must be strided memory on a CUDA device,
// and must not ask for a gradient that the call would not give it.
const Tensor& tensor(PyObject* o, const char* name) {
    TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor");
    const Tensor& x = THPVariable_Unpack(o);
    TORCH_CHECK_TYPE(x.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK_TYPE(x.layout() == c10::kStrided && !x.is_neg() && !x.is_conj(), name, " must be a plain strided tensor");
    TORCH_CHECK_VALUE(!(x.requires_grad() && at::GradMode::is_enabled()), name,
                      " requires a gradient, which this call does not record: detach it, or call under "
                      "torch.no_grad() (rotary's gradient is rotary with inverse=True)");
    TORCH_CHECK_VALUE(!(c10::AutogradState::get_tls_state().get_fw_grad_mode() && x._fw_grad(0).defined()), name,
                      " has a forward-mode tangent, which this call does not carry on: take its primal "
                      "(torch.autograd.forward_ad.unpack_dual)");
    return x;
}

// The same for the arguments after the first: on the first one's device.
const Tensor& tensor_on(c10::Device device, PyObject* o, const char* name) {
    TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor");
    const Tensor& x = THPVariable_Unpack(o);
    TORCH_CHECK_VALUE(x.device() == device, name, " is on ", x.device(), ", not on ", device);
    return tensor(o, name);
}

chm_heads heads_of(const Tensor& x, const char* name, bool batch, bool token) {
    const int64_t n = x.dim();
    TORCH_CHECK_VALUE(x.size(n - 1) <= 1 || x.stride(n - 1) == 1 || x.numel() == 0, "the last axis of ", name,
                      " must be contiguous");
    TORCH_CHECK_VALUE(x.size(n - 2) <= (1 << 16), name, " has more than 65536 heads");
    chm_heads h{};
    h.data = x.data_ptr();
    h.heads = (int32_t)x.size(n - 2);
    h.head_stride = x.stride(n - 2);
    if (token) h.token_stride = x.stride(n - 3);
    if (batch) h.batch_stride = x.stride(0);
    return h;
}

// Whether vectors of x may share memory: an axis, from the smallest stride up, that does not
// step past all that the ones before it span.
bool overlaps_itself(const Tensor& x) {
    const int64_t n = x.dim();
    if (x.numel() == 0) return false;
    int64_t extent = x.size(n - 1), done_axes = 0;
    for (int64_t done = 0; done < n - 1; ++done) {
        int64_t best = -1;  // the smallest stride of an axis of more than one that is not done
        for (int64_t i = 0; i < n - 1; ++i)
            if (x.size(i) > 1 && !(done_axes >> i & 1) && (best < 0 || x.stride(i) < x.stride(best))) best = i;
        if (best < 0) break;
        if (x.stride(best) < extent) return true;
        extent += x.stride(best) * (x.size(best) - 1);
        done_axes |= int64_t{1} << best;
    }
    return false;
}
// What a call writes must not overlap itself, nor two outputs stand in one place.
void check_written(const Tensor& x, const char* name) {
    TORCH_CHECK_VALUE(!overlaps_itself(x), name, " is written and must not overlap itself");
}
void check_apart(const Tensor& x, const Tensor& y, const char* names) {
    TORCH_CHECK_VALUE(x.numel() == 0 || y.numel() == 0 || x.data_ptr() != y.data_ptr(), names,
                      " are written and must not overlap");
}

// An output given by the caller, or a new one.
Tensor output(PyObject* o, c10::IntArrayRef shape, ScalarType type, c10::Device device, const char* name) {
    // (not at::empty: its dispatch is a third of a small call)
    if (o == Py_None) return at::detail::empty_cuda(shape, type, device, std::nullopt);
    const Tensor& x = tensor_on(device, o, name);
    TORCH_CHECK_VALUE(x.sizes() == shape && x.scalar_type() == type, name, " must be ", c10::toString(type),
                      " of shape ", shape);
    check_written(x, name);
    return x;
}

// Tells autograd that a caller's tensor was written (one it saved is then refused by
// backward).  Tensors of inference mode have no count, and cannot be saved.
void written(const Tensor& x) {
    if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
}
void written(PyObject* o) {
    if (o != Py_None) written(THPVariable_Unpack(o));
}

bool flag(PyObject* o) {
    const int r = PyObject_IsTrue(o);
    if (r < 0) throw python_error();
    return r;
}
double number(PyObject* o) {
    const double x = PyFloat_AsDouble(o);
    if (x == -1.0 && PyErr_Occurred()) throw python_error();
    return x;
}

// A status as an exception: ValueError for an argument the C ABI refused,
// chimera_b200.capi.ChmError for the rest.
void check(chm_status s, const char* where) {
    if (s == CHM_OK) return;
    TORCH_CHECK_VALUE(s != CHM_ERR_INVALID, chm_last_error());
    PyObject* m = PyImport_ImportModule("chimera_b200.capi");
    PyObject* kind = m ? PyObject_GetAttrString(m, "ChmError") : nullptr;
    PyObject* e = kind ? PyObject_CallFunction(kind, "is", (int)s, where) : nullptr;
    if (e) PyErr_SetObject(kind, e);
    Py_XDECREF(e);
    Py_XDECREF(kind);
    Py_XDECREF(m);
    throw python_error();
}

void* stream_of(c10::Device d) { return c10::cuda::getCurrentCUDAStream(d.index()).stream(); }

PyObject* pair(PyObject* a, PyObject* b) {
    PyObject* t = PyTuple_New(2);
    if (!t) throw python_error();
    PyTuple_SET_ITEM(t, 0, a);
    PyTuple_SET_ITEM(t, 1, b);
    return t;
}

// q, k or None, positions, freqs, interleaved, inverse, scale, q_out, k_out
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 9, "rotary takes 9 arguments");
    const Tensor& q = tensor(a[0], "q");
    const bool both = a[1] != Py_None;
    const c10::Device dev = q.device();
    const int type = type_of(q.scalar_type());
    TORCH_CHECK_TYPE(is_vector_type(type), "q must be float32, float16 or bfloat16");
    const int64_t dims = q.dim();
    TORCH_CHECK_VALUE(dims == 3 || dims == 4, "q must be [batch, tokens, heads, dim] or [tokens, heads, dim]");
    const int64_t batch = dims == 4 ? q.size(0) : 1, tokens = q.size(dims - 3), dim = q.size(dims - 1);
    TORCH_CHECK_VALUE(dim <= 4096, "dim is at most 4096");
    const Tensor& pos = tensor_on(dev, a[2], "positions");
    TORCH_CHECK_TYPE(pos.scalar_type() == ScalarType::Long || pos.scalar_type() == ScalarType::Int,
                     "positions must be int64 or int32");
    const bool per_row = pos.dim() == 2 && pos.size(0) == batch && pos.size(1) == tokens;
    TORCH_CHECK_VALUE(per_row || (pos.dim() == 1 && pos.size(0) == tokens), "positions must be [batch, tokens] or [tokens]");
    const Tensor& freqs = tensor_on(dev, a[3], "freqs");
    TORCH_CHECK_TYPE(freqs.scalar_type() == ScalarType::Double && freqs.dim() == 1 && freqs.is_contiguous(),
                     "freqs must be a contiguous float64 vector");
    TORCH_CHECK_VALUE(freqs.size(0) <= 2048, "freqs has more than 2048 pairs");
    const int flags = (flag(a[4]) ? CHM_ROTARY_INTERLEAVED : 0) | (flag(a[5]) ? CHM_ROTARY_INVERSE : 0);
    const float scale = (float)number(a[6]);
    TORCH_CHECK_VALUE(both || a[8] == Py_None, "k_out without k");
    const Tensor* k = nullptr;
    if (both) {
        k = &tensor_on(dev, a[1], "k");
        TORCH_CHECK_TYPE(k->scalar_type() == q.scalar_type(), "k must have q's type");
        bool alike = k->dim() == dims && k->size(dims - 1) == dim;
        for (int64_t i = 0; alike && i < dims - 2; ++i) alike = k->size(i) == q.size(i);
        TORCH_CHECK_VALUE(alike, "k must agree with q but for its heads");
    }
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor qo = output(a[7], q.sizes(), q.scalar_type(), dev, "q_out");
    chm_heads in[2], out[2];
    in[0] = heads_of(q, "q", dims == 4, true);
    out[0] = heads_of(qo, "q_out", dims == 4, true);
    Tensor ko;
    if (both) {
        ko = output(a[8], k->sizes(), k->scalar_type(), dev, "k_out");
        in[1] = heads_of(*k, "k", dims == 4, true);
        out[1] = heads_of(ko, "k_out", dims == 4, true);
        check_apart(qo, ko, "q_out and k_out");
    }
    check(chm_rotary(in, out, both ? 2 : 1, type, batch, tokens, (int32_t)dim, 2 * (int32_t)freqs.size(0),
                     pos.data_ptr(), (int32_t)pos.element_size(), per_row ? pos.stride(0) : 0,
                     pos.stride(per_row ? 1 : 0), freqs.data_ptr<double>(), scale, flags, stream_of(dev)),
          "rotary");
    written(a[7]);
    written(a[8]);
    PyObject* r0 = a[7] != Py_None ? Py_NewRef(a[7]) : THPVariable_Wrap(qo);
    PyObject* r1 = !both ? Py_NewRef(Py_None) : a[8] != Py_None ? Py_NewRef(a[8]) : THPVariable_Wrap(ko);
    return pair(r0, r1);
    END_HANDLE_TH_ERRORS
}

// k_pages, v_pages, k_scale, v_scale
chm_kv_cache cache_of(PyObject* const* a, c10::Device dev) {
    const Tensor& k = tensor_on(dev, a[0], "k_pages");
    const Tensor& v = tensor_on(dev, a[1], "v_pages");
    const int type = type_of(k.scalar_type());
    TORCH_CHECK_TYPE(type > CHM_FP32, "pages must be float16, bfloat16, int8 or float8_e4m3fn");
    TORCH_CHECK_VALUE(k.dim() == 4, "pages must be [num_pages, heads, page_size, dim]");
    bool alike = v.scalar_type() == k.scalar_type() && v.sizes() == k.sizes();
    int64_t stride[3] = {};  // of an axis of one any stride will do
    for (int i = 0; alike && i < 4; ++i) {
        alike = k.size(i) <= 1 || v.stride(i) == k.stride(i);
        if (i < 3 && k.size(i) > 1) stride[i] = k.stride(i);
    }
    TORCH_CHECK_VALUE(alike, "k_pages and v_pages must be alike in type, shape and strides");
    TORCH_CHECK_VALUE(k.stride(3) == 1 || k.size(3) <= 1, "the last axis of the pages must be contiguous");
    TORCH_CHECK_VALUE(k.size(1) <= (1 << 16) && k.size(2) <= INT32_MAX && k.size(3) <= 256,
                      "pages have at most 65536 heads, 2^31 - 1 tokens and 256 dimensions");
    chm_kv_cache c{};
    c.k = k.data_ptr();
    c.v = v.data_ptr();
    c.num_pages = k.size(0);
    c.heads = (int32_t)k.size(1);
    c.page_size = (int32_t)k.size(2);
    c.dim = (int32_t)k.size(3);
    c.page_stride = stride[0];
    c.head_stride = stride[1];
    c.token_stride = stride[2];
    c.type = type;
    if (type == CHM_INT8 || type == CHM_E4M3) {
        for (int i = 0; i < 2; ++i) {
            TORCH_CHECK_VALUE(a[2 + i] != Py_None, "an 8-bit cache needs k_scale and v_scale");
            const Tensor& s = tensor_on(dev, a[2 + i], "scales");
            TORCH_CHECK_VALUE(s.scalar_type() == ScalarType::Float && s.dim() == 3 && s.size(0) == c.num_pages &&
                                  s.size(1) == c.heads && s.size(2) == c.page_size && s.is_contiguous(),
                              "scales must be contiguous float32 [num_pages, heads, page_size]");
            (i ? c.v_scale : c.k_scale) = s.data_ptr<float>();
        }
    } else {
        TORCH_CHECK_VALUE(a[2] == Py_None && a[3] == Py_None, "a 16-bit cache has no scales");
    }
    return c;
}

const Tensor& slots_of(PyObject* o, c10::Device dev) {
    const Tensor& s = tensor_on(dev, o, "slots");
    TORCH_CHECK_TYPE(s.scalar_type() == ScalarType::Long && s.dim() == 1 && s.is_contiguous(),
                     "slots must be a contiguous int64 vector");
    return s;
}

// k, v, slots, then a cache
PyObject* cache_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 7, "cache_write takes 7 arguments");
    const Tensor& k = tensor(a[0], "k");
    const c10::Device dev = k.device();
    const Tensor& v = tensor_on(dev, a[1], "v");
    const int type = type_of(k.scalar_type());
    TORCH_CHECK_TYPE(is_vector_type(type) && v.scalar_type() == k.scalar_type(),
                     "k and v must be float32, float16 or bfloat16, and alike");
    const Tensor& slots = slots_of(a[2], dev);
    const chm_kv_cache c = cache_of(a + 3, dev);
    TORCH_CHECK_VALUE(k.dim() == 3 && k.size(0) == slots.size(0) && k.size(1) == c.heads && k.size(2) == c.dim &&
                          v.sizes() == k.sizes(),
                      "k and v must be [", slots.size(0), ", ", c.heads, ", ", c.dim, "]");
    const chm_heads kh = heads_of(k, "k", false, true), vh = heads_of(v, "v", false, true);
    const Tensor &kp = THPVariable_Unpack(a[3]), &vp = THPVariable_Unpack(a[4]);
    check_written(kp, "k_pages");  // v_pages has the same strides
    check_apart(kp, vp, "k_pages and v_pages");
    if (c.k_scale) check_apart(THPVariable_Unpack(a[5]), THPVariable_Unpack(a[6]), "k_scale and v_scale");
    const c10::cuda::CUDAGuard guard(dev);
    check(chm_cache_write(&c, &kh, &vh, type, slots.size(0), slots.data_ptr<int64_t>(), stream_of(dev)), "cache_write");
    for (int i = 3; i < 7; ++i) written(a[i]);
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// slots, a cache, dtype, k_out, v_out
PyObject* cache_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 8, "cache_read takes 8 arguments");
    const c10::Device dev = tensor(a[1], "k_pages").device();
    const chm_kv_cache c = cache_of(a + 1, dev);
    TORCH_CHECK_TYPE(THPDtype_Check(a[5]), "dtype must be a torch.dtype");
    const ScalarType st = reinterpret_cast<THPDtype*>(a[5])->scalar_type;
    const int type = type_of(st);
    TORCH_CHECK_TYPE(is_vector_type(type), "dtype must be float32, float16 or bfloat16");
    const Tensor& slots = slots_of(a[0], dev);
    const int64_t shape[3] = {slots.size(0), c.heads, c.dim};
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor k = output(a[6], shape, st, dev, "k_out"), v = output(a[7], shape, st, dev, "v_out");
    const chm_heads kh = heads_of(k, "k_out", false, true), vh = heads_of(v, "v_out", false, true);
    check_apart(k, v, "k_out and v_out");
    check(chm_cache_read(&c, slots.data_ptr<int64_t>(), slots.size(0), &kh, &vh, type, stream_of(dev)), "cache_read");
    written(a[6]);
    written(a[7]);
    PyObject* r0 = a[6] != Py_None ? Py_NewRef(a[6]) : THPVariable_Wrap(k);
    PyObject* r1 = a[7] != Py_None ? Py_NewRef(a[7]) : THPVariable_Wrap(v);
    return pair(r0, r1);
    END_HANDLE_TH_ERRORS
}

// q, a cache, tables, lens, starts, scale or None, out, lse, workspace
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 12, "paged_attention takes 12 arguments");
    const Tensor& q = tensor(a[0], "q");
    const c10::Device dev = q.device();
    const chm_kv_cache c = cache_of(a + 1, dev);
    const int type = type_of(q.scalar_type());
    TORCH_CHECK_TYPE(type == CHM_FP16 || type == CHM_BF16, "q must be float16 or bfloat16");
    TORCH_CHECK_VALUE(q.dim() == 3 && q.size(2) == c.dim, "q must be [batch, q_heads, ", c.dim, "]");
    const int64_t batch = q.size(0), heads = q.size(1);
    const Tensor& tables = tensor_on(dev, a[5], "tables");
    TORCH_CHECK_VALUE(tables.scalar_type() == ScalarType::Int && tables.dim() == 2 && tables.size(0) == batch &&
                          (tables.size(1) <= 1 || tables.stride(1) == 1) && tables.size(1) <= INT32_MAX,
                      "tables must be int32 [batch, width], contiguous along the width");
    const int32_t width = (int32_t)tables.size(1);
    const int32_t* bounds[2] = {nullptr, nullptr};
    for (int i = 0; i < 2; ++i) {
        const char* name = i ? "starts" : "lens";
        if (i && a[7] == Py_None) continue;
        const Tensor& x = tensor_on(dev, a[6 + i], name);
        TORCH_CHECK_VALUE(x.scalar_type() == ScalarType::Int && x.dim() == 1 && x.size(0) == batch && x.is_contiguous(),
                          name, " must be contiguous int32 [batch]");
        bounds[i] = x.data_ptr<int32_t>();
    }
    const float scale = a[8] == Py_None ? (float)(1.0 / std::sqrt((double)c.dim)) : (float)number(a[8]);
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor out = output(a[9], q.sizes(), q.scalar_type(), dev, "out");
    const int64_t rows[2] = {batch, heads};
    const Tensor lse = output(a[10], rows, ScalarType::Float, dev, "lse");
    TORCH_CHECK_VALUE(lse.is_contiguous(), "lse must be contiguous");
    const chm_heads qh = heads_of(q, "q", true, false), oh = heads_of(out, "out", true, false);
    const size_t need = chm_paged_attention_workspace_bytes(&c, batch, (int32_t)heads, width);
    c10::DataPtr own;  // back to the allocator at the end: it gives the memory out again on this stream
    void* ws;
    size_t ws_bytes = need;
    if (a[11] == Py_None) {
        own = c10::cuda::CUDACachingAllocator::get()->allocate(need);
        ws = own.get();
    } else {
        const Tensor& x = tensor_on(dev, a[11], "workspace");
        ws = x.data_ptr();
        ws_bytes = (size_t)x.numel();
        TORCH_CHECK_VALUE(x.scalar_type() == ScalarType::Byte && x.is_contiguous() && ws_bytes >= need &&
                              (uintptr_t)ws % 256 == 0,
                          "workspace must be contiguous uint8, 256-byte aligned, of ", need, " bytes or more");
    }
    check(chm_paged_attention(&c, &qh, &oh, type, batch, tables.data_ptr<int32_t>(), tables.stride(0), width, bounds[0],
                              bounds[1], scale, lse.data_ptr<float>(), ws, ws_bytes,
                              stream_of(dev)),
          "paged_attention");
    written(a[9]);
    written(a[10]);
    written(a[11]);
    PyObject* r0 = a[9] != Py_None ? Py_NewRef(a[9]) : THPVariable_Wrap(out);
    PyObject* r1 = a[10] != Py_None ? Py_NewRef(a[10]) : THPVariable_Wrap(lse);
    return pair(r0, r1);
    END_HANDLE_TH_ERRORS
}

// a cache, batch, q_heads, table_width
PyObject* paged_attention_workspace(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 7, "paged_attention_workspace takes 7 arguments");
    const c10::Device dev = tensor(a[0], "k_pages").device();
    const chm_kv_cache c = cache_of(a, dev);
    int64_t v[3];
    for (int i = 0; i < 3; ++i) {
        v[i] = PyLong_AsLongLong(a[4 + i]);
        if (v[i] == -1 && PyErr_Occurred()) throw python_error();
        TORCH_CHECK_VALUE(v[i] >= 0 && v[i] <= INT32_MAX, "sizes must be from 0 to 2^31 - 1");
    }
    const c10::cuda::CUDAGuard guard(dev);
    const size_t need = chm_paged_attention_workspace_bytes(&c, v[0], (int32_t)v[1], (int32_t)v[2]);
    TORCH_CHECK_VALUE(need > 0, chm_last_error());
    return PyLong_FromSize_t(need);
    END_HANDLE_TH_ERRORS
}

#define CHM_METHOD(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {CHM_METHOD(rotary),     CHM_METHOD(cache_write),     CHM_METHOD(cache_read),
                         CHM_METHOD(paged_attention), CHM_METHOD(paged_attention_workspace), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_generation", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__generation(void) { return PyModule_Create(&module); }
