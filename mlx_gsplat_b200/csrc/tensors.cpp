// Reads many tensors' metadata into a gs_tensor table without a Python
// operation per tensor and property (1.0 us for a gradient and its output
// through Python, most of a call over a few hundred small tensors).
//
// The fast path only: whatever is not a dense strided tensor of the three types,
// of the expected shape, on the expected device, makes a function return 1, and
// the caller's own checks then find out what it is and say so.  Nothing is kept
// from call to call.  Called with the GIL held (ctypes.PyDLL); no exception
// leaves a function.
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <utility>
#include <vector>

#include "gsplat_b200.h"

namespace {

int type_code(at::ScalarType t) {
    return t == at::kFloat ? GS_F32 : t == at::kBFloat16 ? GS_BF16 : t == at::kHalf ? GS_F16 : -1;
}

const at::Tensor* tensor_of(PyObject* o) { return o && THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

// The type's code of a dense tensor on CUDA device ``device``, else -1.
int dense_type(const at::Tensor& t, int device) {
    if (!t.defined() || t.layout() != at::kStrided || !t.is_cuda() || t.get_device() != device || !t.is_contiguous() ||
        t.is_conj() || t.is_neg())
        return -1;
    return type_code(t.scalar_type());
}

// Whether ``p`` still has the type, shape and strides of ``was``, a strided tensor (the
// sizes of other layouts throw).
bool same_form(const at::Tensor& p, const at::Tensor& was) {
    const auto *a = p.unsafeGetTensorImpl(), *b = was.unsafeGetTensorImpl();
    const int64_t n = a->dim();
    if (n != b->dim() || a->dtype() != b->dtype() || p.is_neg()) return false;
    const int64_t *size = a->sizes().data(), *stride = a->strides().data();
    const int64_t *size0 = b->sizes().data(), *stride0 = b->strides().data();
    for (int64_t k = 0; k < n; ++k)
        if ((size[k] != size0[k]) | (stride[k] != stride0[k])) return false;
    return true;
}

void changed(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// See gst_fill.  ``may_miss``: a name that the dict lacks or that has None, or a parameter
// without ``grad``, has a null one; ``present`` counts the others.
bool fill(PyObject* items, PyObject* names, PyObject* owners, PyObject* like, gs_tensor* e, Py_ssize_t n, int device,
          bool may_miss, Py_ssize_t& present) {
    present = 0;
    try {
        const bool list = PyList_Check(items), dict = PyDict_Check(items);
        if (!(list || dict || items == Py_None) || !PyList_Check(like) || PyList_GET_SIZE(like) != n ||
            (list && PyList_GET_SIZE(items) != n) ||
            (dict && ((!may_miss && PyDict_GET_SIZE(items) != n) || !PyList_Check(names) ||
                      PyList_GET_SIZE(names) != n)) ||
            (items == Py_None && owners == Py_None) ||
            (owners != Py_None && (!PyList_Check(owners) || PyList_GET_SIZE(owners) != n)))
            return false;
        Py_ssize_t named = 0;
        for (Py_ssize_t k = 0; k < n; ++k) {
            const at::Tensor* p = tensor_of(PyList_GET_ITEM(like, k));
            if (!p) return false;
            const at::Tensor *g = nullptr, *owner = nullptr;
            if (owners != Py_None && (!(owner = tensor_of(PyList_GET_ITEM(owners, k))) || !same_form(*owner, *p)))
                return false;
            bool none = false;
            if (list) {
                g = tensor_of(PyList_GET_ITEM(items, k));
            } else if (dict) {
                PyObject* item = PyDict_GetItem(items, PyList_GET_ITEM(names, k));
                named += item != nullptr;
                none = !item || item == Py_None;
                g = tensor_of(item);
            } else {
                g = &owner->grad();
                none = !g->defined();
            }
            if (none && may_miss) {
                e[k].grad = nullptr;
                continue;
            }
            if (!g) return false;
            const int type = dense_type(*g, device);
            if (type < 0 || g->sizes() != p->sizes()) return false;
            e[k].grad = g->const_data_ptr();
            if (!e[k].grad && g->numel() > 0) return false;
            e[k].grad_type = type;
            e[k].grad_stride = e[k].cols;
            ++present;
        }
        return !dict || named == PyDict_GET_SIZE(items);
    } catch (...) {
        return false;
    }
}

struct Span {
    uintptr_t lo, hi;
    bool operator<(const Span& o) const { return lo < o.lo; }
};

}  // namespace

// What this file was compiled against: a loader refuses it under anything else.
extern "C" const char* gst_abi() { return GST_ABI; }

// Fills ``e[k].grad`` and its type and row stride from the k-th of ``n`` tensors
// shaped like ``like[k]``: those of the list ``items``, or those of the dict
// ``items`` under ``names``, or (None) the ``grad`` of ``owners[k]``.  ``owners``, where
// given, must still have the form of ``like``.
extern "C" int gst_fill(PyObject* items, PyObject* names, PyObject* owners, PyObject* like, gs_tensor* e, Py_ssize_t n,
                        int device) {
    Py_ssize_t present;
    return fill(items, names, owners, like, e, n, device, false, present) ? 0 : 1;
}

// Whether the parameters still lie where the entries say, and if so tells autograd
// that they are written.
extern "C" int gst_params_unmoved(PyObject* params, const gs_tensor* e, Py_ssize_t n) {
    try {
        if (!PyList_Check(params) || PyList_GET_SIZE(params) != n) return 1;
        for (Py_ssize_t k = 0; k < n; ++k) {
            const at::Tensor* p = tensor_of(PyList_GET_ITEM(params, k));
            // (an address to write to: memory shared with a lazy copy becomes the parameter's own)
            if (!p || p->mutable_data_ptr() != e[k].param) return 1;
        }
        for (Py_ssize_t k = 0; k < n; ++k) changed(THPVariable_Unpack(PyList_GET_ITEM(params, k)));
        return 0;
    } catch (...) {
        return 1;
    }
}

// A step's entries: gradients as gst_fill takes them, where any may be missing, for
// parameters that still are where the entries say, which are then told to be
// written.  ``found``: the gradients that are there, and whether they have any element.
extern "C" int gst_step(PyObject* grads, PyObject* names, PyObject* params, PyObject* like, gs_tensor* e, Py_ssize_t n,
                        int device, Py_ssize_t* found) {
    if (params == Py_None || PyList_Check(grads) ||
        !fill(grads, names, params, like, e, n, device, true, found[0]))
        return 1;
    found[1] = 0;
    for (Py_ssize_t k = 0; k < n; ++k) found[1] |= e[k].grad && e[k].n;
    if (found[0] == n) return gst_params_unmoved(params, e, n);
    try {
        for (Py_ssize_t k = 0; k < n; ++k)
            if (THPVariable_Unpack(PyList_GET_ITEM(params, k)).mutable_data_ptr() != e[k].param) return 1;
        for (Py_ssize_t k = 0; k < n; ++k)
            if (e[k].grad) changed(THPVariable_Unpack(PyList_GET_ITEM(params, k)));
        return 0;
    } catch (...) {
        return 1;
    }
}

// Whether the parameters are the memory, types and layouts that the entries and
// ``like`` were taken from.
extern "C" int gst_params_as_taken(PyObject* params, PyObject* like, const gs_tensor* e, Py_ssize_t n) {
    try {
        if (!PyList_Check(params) || PyList_GET_SIZE(params) != n || !PyList_Check(like) || PyList_GET_SIZE(like) != n)
            return 1;
        for (Py_ssize_t k = 0; k < n; ++k) {
            const at::Tensor *p = tensor_of(PyList_GET_ITEM(params, k)), *was = tensor_of(PyList_GET_ITEM(like, k));
            if (!p || !was || p->mutable_data_ptr() != e[k].param || !same_form(*p, *was)) return 1;
        }
        return 0;
    } catch (...) {
        return 1;
    }
}

// The entries of gradients and of the tensors their clipped values go to (the same
// list: in place), where all are dense and on one device (returned) and nothing
// that is written overlaps anything but its own gradient's memory.  ``e`` comes
// zeroed; ``found``: the device, and whether there is any element.
extern "C" int gst_clip(PyObject* grads, PyObject* outs, gs_tensor* e, Py_ssize_t n, int* found) {
    try {
        if (!PyList_Check(grads) || !PyList_Check(outs) || PyList_GET_SIZE(grads) != n || PyList_GET_SIZE(outs) != n || n == 0)
            return 1;
        const at::Tensor* first = tensor_of(PyList_GET_ITEM(grads, 0));
        if (!first || !first->defined() || !first->is_cuda()) return 1;
        const int device = first->get_device();
        bool any = false;
        std::vector<Span> written(n), read;
        for (Py_ssize_t k = 0; k < n; ++k) {
            const at::Tensor* g = tensor_of(PyList_GET_ITEM(grads, k));
            const at::Tensor* o = tensor_of(PyList_GET_ITEM(outs, k));
            if (!g || !o) return 1;
            const int g_type = dense_type(*g, device), o_type = dense_type(*o, device);
            if (g_type < 0 || o_type < 0 || g->sizes() != o->sizes()) return 1;
            gs_tensor& t = e[k];
            t.n = g->numel();
            any |= t.n > 0;
            t.param = o->mutable_data_ptr();
            t.grad = g->const_data_ptr();
            t.param_type = o_type;
            t.grad_type = g_type;
            t.cols = t.param_stride = t.grad_stride = t.n ? t.n : 1;
            const uintptr_t at_o = reinterpret_cast<uintptr_t>(t.param), at_g = reinterpret_cast<uintptr_t>(t.grad);
            written[k] = {at_o, at_o + (uintptr_t)t.n * o->element_size()};
            if (at_o != at_g || o_type != g_type) read.push_back({at_g, at_g + (uintptr_t)t.n * g->element_size()});
        }
        std::sort(written.begin(), written.end());
        for (Py_ssize_t k = 1; k < n; ++k)
            if (written[k].lo < written[k - 1].hi) return 1;
        for (const Span& r : read) {
            // the last written span that begins below the end of what is read
            auto w = std::lower_bound(written.begin(), written.end(), Span{r.hi, 0});
            if (w != written.begin() && (w - 1)->hi > r.lo) return 1;
        }
        for (Py_ssize_t k = 0; k < n; ++k) changed(*tensor_of(PyList_GET_ITEM(outs, k)));
        found[0] = device;
        found[1] = any;
        return 0;
    } catch (...) {
        return 1;
    }
}
