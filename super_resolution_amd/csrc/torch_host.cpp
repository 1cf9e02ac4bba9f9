// Host side of the optimizers: reads the gradients of thousands of parameters in one call.
//
// A training step of RRDBNet-FDConv has 8380 parameter tensors whose `.grad` are new tensors every step.  Reading 8380 data
// pointers and checking dtype, device and layout takes Python 4 ms, the same walk over the tensors' C++ objects 0.07 ms -- and the
// kernels that then run take 0.1.  Built as libsr_amd_torch.so (the only file that sees torch's C++ headers); Python calls it
// through ctypes with the GIL held.  No exception leaves a function: they return SRT_FAILED and keep the message.
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <algorithm>
#include <cstring>
#include <string>
#include <vector>

#define SRT_FAILED (-1)
#define SRT_API extern "C" __attribute__((visibility("default")))

namespace {
thread_local std::string g_message;

template <typename F>
int64_t guarded(F f) {
    try {
        return f();
    } catch (const std::exception& e) {
        g_message = e.what();
    } catch (...) {
        g_message = "unknown C++ exception";
    }
    return SRT_FAILED;
}

const at::Tensor& tensor_of(PyObject* o) {
    // (THPVariable_Check asks the metaclass, 0.1 us for a Parameter)
    TORCH_CHECK(THPVariableClass && PyObject_TypeCheck(o, (PyTypeObject*)THPVariableClass), "not a tensor");
    return THPVariable_Unpack(o);
}

struct Tracked {
    std::vector<at::Tensor> params;
    struct Was {
        const void* data;
        int64_t numel;
        caffe2::TypeMeta dtype;
        bool counts;  // has a version counter
        bool contiguous;
        const c10::StorageImpl* storage;
    };
    std::vector<Was> was;
    // the storages' data may go, their objects stay: no other storage takes an address in `was`
    std::vector<c10::weak_intrusive_ptr<c10::StorageImpl>> storages;
    std::vector<std::vector<int64_t>> strides;  // of the tensors that are not contiguous
};

struct Span {
    uint64_t g;
    int64_t n;
};
// the gradients that this thread's last srt_spans found: float32, bfloat16 (another thread may run between it and srt_take_spans)
thread_local std::vector<Span> g_found[2];
thread_local int64_t g_longest = 1;

// autograd's part of a tensor, where its gradient is; NULL: none
const at::Tensor* gradient_of(const c10::TensorImpl* t) {
    const auto* meta = static_cast<const torch::autograd::AutogradMeta*>(t->autograd_meta());
    return meta && meta->grad_.defined() ? &meta->grad_ : nullptr;
}
// takes a bump_version back: the tensor was not written after all
void unbump_version(c10::TensorImpl* t) {
    c10::VariableVersion v = t->version_counter();  // (shares the tensor's counter)
    v.set_version((int64_t)v.current_version() - 1);
}
// the gradients of the first `count` tensors of a list whose versions srt_spans moved
void unbump_gradients(PyObject* list, int of_params, Py_ssize_t count) {
    for (Py_ssize_t i = 0; i < count; ++i) {
        c10::TensorImpl* g = tensor_of(PyList_GET_ITEM(list, i)).unsafeGetTensorImpl();
        const at::Tensor* grad = of_params ? gradient_of(g) : nullptr;
        if (of_params && !grad) continue;
        if (grad) g = grad->unsafeGetTensorImpl();
        if (!g->is_inference()) unbump_version(g);
    }
}
// the same memory order: element i of one is element i of the other
bool same_layout(const c10::TensorImpl* a, const c10::TensorImpl* b) {
    return (a->is_contiguous() && b->is_contiguous()) || (a->strides().equals(b->strides()) && a->is_non_overlapping_and_dense());
}
}  // namespace

SRT_API const char* srt_message() { return g_message.c_str(); }

// holds the tensors of a list (they stay alive); NULL on failure
SRT_API void* srt_track(PyObject* list) {
    Tracked* t = nullptr;
    const int64_t rc = guarded([&]() -> int64_t {
        TORCH_CHECK(PyList_Check(list), "not a list");
        t = new Tracked;
        for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); ++i) {
            const at::Tensor& p = tensor_of(PyList_GET_ITEM(list, i));
            t->params.push_back(p);
            const c10::TensorImpl* impl = p.unsafeGetTensorImpl();
            t->was.push_back({impl->data(), impl->numel(), impl->dtype(), !p.is_inference(), impl->is_contiguous(),
                              impl->storage().unsafeGetStorageImpl()});
            t->storages.push_back(impl->storage().getWeakStorageImpl());
            if (!impl->is_contiguous()) t->strides.push_back(impl->strides().vec());
        }
        return 0;
    });
    if (rc) {
        delete t;
        return nullptr;
    }
    return t;
}
SRT_API void srt_untrack(void* h) { delete (Tracked*)h; }

// out[i] = address of the gradient of tensor i, 0 without one.  Returns the number of tensors without a gradient.
// odd[0 .. *nodd): tensors whose gradient cannot be read as it lies (other shape, strides, dtype or device: out[i] = 0, not counted
// as missing).  *moved: tensors that are not where, or what, they were when the list was made, or that lie in another storage or in
// another order of their elements (an address may come back with another one).  Shapes are not compared: in the same storage and
// contiguous as before, the elements are where they were, and reading 8380 shapes costs a fifth of the walk (30 us).  Tensors with a
// gradient are about to be written in place: their version counters move (autograd's saved-tensor checks and caches keyed on them must
// see it; here and not in a walk of its own, which costs a third as much again).
SRT_API int64_t srt_gradients(void* h, uint64_t* out, int64_t* odd, int64_t* nodd, int64_t* moved) {
    return guarded([&]() -> int64_t {
        const Tracked& t = *(const Tracked*)h;
        const size_t n = t.params.size();
        int64_t missing = 0;
        *nodd = *moved = 0;
        size_t strided = 0;
        for (size_t i = 0; i < n; ++i) {
            c10::TensorImpl* p = t.params[i].unsafeGetTensorImpl();
            const Tracked::Was& was = t.was[i];
            const bool contiguous = p->is_contiguous();
            bool stayed = p->unsafe_storage().unsafeGetStorageImpl() == was.storage && p->data() == was.data && p->numel() == was.numel &&
                          p->dtype() == was.dtype;  // (another device: another storage)
            if (!(contiguous && was.contiguous)) {
                stayed = stayed && contiguous == was.contiguous && p->strides().equals(t.strides[strided]);
                strided += !was.contiguous;
            }
            *moved += !stayed;
            const at::Tensor* grad = gradient_of(p);
            out[i] = 0;
            if (!grad) {
                ++missing;
                continue;
            }
            if (was.counts) p->bump_version();
            const c10::TensorImpl* g = grad->unsafeGetTensorImpl();
            // (equal key sets: the same kind of tensor; torch keeps a gradient on its parameter's device)
            if (g->key_set() == p->key_set() && g->numel() == was.numel && g->dtype() == was.dtype && ((contiguous && g->is_contiguous()) || same_layout(g, p)))
                out[i] = g->numel() ? (uint64_t)(uintptr_t)g->data() : 16;  // (of an empty tensor nothing is read, but it has one)
            else
                odd[(*nodd)++] = (int64_t)i;
        }
        return missing;
    });
}
// The step that srt_gradients prepared does not take place: the version counters go back.
SRT_API int64_t srt_not_written(void* h) {
    return guarded([&]() -> int64_t {
        const Tracked& t = *(const Tracked*)h;
        for (size_t i = 0; i < t.params.size(); ++i) {
            c10::TensorImpl* p = t.params[i].unsafeGetTensorImpl();
            if (t.was[i].counts && gradient_of(p)) unbump_version(p);
        }
        return 0;
    });
}

// The gradients of a list of parameters (of_params) or of a list of gradients, as spans of consecutive values of at most
// `longest` (0: by the total, see below); counts[0 / 1]: spans in float32 / bfloat16, counts[2]: tensors.  Returns 0, or
//   1 + i: tensor i is neither float32 nor bfloat16, or not on GPU `device` (device < 0: that of the first, put into *device)
//   -2 - i: gradient i has holes or repeats its elements
// and SRT_FAILED.  Gradients that share memory fail: they would be scaled twice.  The version counters of the gradients move, as they
// are about to be written, but not where the call fails.
SRT_API int64_t srt_spans(PyObject* list, int of_params, int* device, int64_t* counts) {
    return guarded([&]() -> int64_t {
        TORCH_CHECK(PyList_Check(list), "not a list");
        std::vector<Span>(&found)[2] = g_found;
        found[0].clear();
        found[1].clear();
        counts[0] = counts[1] = counts[2] = 0;
        int64_t total = 0;
        uint64_t last = 0;
        bool ascending = true;
        const Py_ssize_t size = PyList_GET_SIZE(list);
        found[0].reserve(size);
        c10::DispatchKeySet usual;  // of the first gradient: those with the same keys are of the same kind
        Py_ssize_t i = 0;
        const auto refuse = [&](int64_t code) {
            unbump_gradients(list, of_params, i);
            return code;
        };
        try {
            for (; i < size; ++i) {
                c10::TensorImpl* g = tensor_of(PyList_GET_ITEM(list, i)).unsafeGetTensorImpl();
                if (of_params) {
                    const at::Tensor* grad = gradient_of(g);
                    if (!grad) continue;
                    g = grad->unsafeGetTensorImpl();
                }
                ++counts[2];
                if (!(g->key_set() == usual)) {
                    if (g->layout() != at::kStrided || !g->device().is_cuda()) return refuse(1 + i);
                    if (*device < 0) *device = g->device().index();
                    if (!g->is_inference()) usual = g->key_set();
                }
                const int kind = g->dtype() == caffe2::TypeMeta::Make<float>() ? 0 : g->dtype() == caffe2::TypeMeta::Make<at::BFloat16>() ? 1 : -1;
                if (kind < 0 || g->device().index() != *device) return refuse(1 + i);
                if (!g->is_contiguous() && !g->is_non_overlapping_and_dense()) return refuse(-2 - i);
                if (g->key_set() == usual) g->bump_version();  // (not that of an inference tensor, which has none)
                const int64_t n = g->numel();
                if (!n) continue;
                const uint64_t at = (uint64_t)(uintptr_t)g->data();
                ascending &= at >= last;
                last = at + (uint64_t)n * (kind ? 2 : 4);
                found[kind].push_back({at, n});
                total += n;
            }
            if (!ascending) {
                std::vector<std::pair<uint64_t, uint64_t>> all;
                for (int k = 0; k < 2; ++k)
                    for (const Span& s : found[k]) all.emplace_back(s.g, s.g + (uint64_t)s.n * (k ? 2 : 4));
                std::sort(all.begin(), all.end());
                for (size_t i = 1; i < all.size(); ++i) TORCH_CHECK(all[i].first >= all[i - 1].second, "two gradients share memory");
            }
        } catch (...) {
            refuse(0);
            throw;
        }
        // a wave takes a span at a time and 8192 waves run at once: equal shares of long tensors, none below 4096 values
        const int64_t longest = std::max<int64_t>(4096, (total / 8192 + 1023) / 1024 * 1024);
        g_longest = longest;
        for (int k = 0; k < 2; ++k)
            for (const Span& s : found[k]) counts[k] += s.n <= longest ? 1 : (s.n + longest - 1) / longest;
        return 0;
    });
}
// The gradients that srt_spans walked are not written: the version counters go back.
SRT_API int64_t srt_spans_not_written(PyObject* list, int of_params) {
    return guarded([&]() -> int64_t {
        unbump_gradients(list, of_params, PyList_GET_SIZE(list));
        return 0;
    });
}
// writes them out, float32 first (long lists straight into pinned memory: they are read once, by a kernel)
SRT_API void srt_take_spans(void* dst) {
    Span* to = (Span*)dst;
    for (int k = 0; k < 2; ++k) {
        for (const Span& s : g_found[k])
            for (int64_t at = 0; at < s.n; at += g_longest) *to++ = {s.g + (uint64_t)at * (k ? 2 : 4), std::min(g_longest, s.n - at)};
        g_found[k].clear();
    }
}
