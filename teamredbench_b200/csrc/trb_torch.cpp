// trb_torch.cpp -- the short way from torch tensors to the C ABI, for calls that take a few microseconds.
//
// One function for each front end of teamredbench_b200/kernels.py that has one here.  It takes the tensors, and where
// everything is as the front end wants it (types, shapes, one device that is the current one, contiguous) it makes the
// call on the current stream and returns True.  Anything else, an error of the call's own included, returns False without
// a trace, and the front end goes its usual way, which names what is wrong.  Asked from Python, the same checks, pointers
// and conversions take longer than the launch (combine of 40 tokens: 6.9 us, of which the launch 2.4).
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/trb_b200.h"

namespace {

constexpr int64_t kLargest = 0x7fffffff;

int dtype_code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return TRB_FLOAT32;
        case at::kBFloat16: return TRB_BFLOAT16;
        case at::kHalf: return TRB_FLOAT16;
        default: return -1;
    }
}

// The tensors of one call.
struct Call {
    at::Tensor t[6];
    bool there[6] = {};
    c10::DeviceIndex device = -1;

    // Arguments as they are, None for the optional ones (a bit of `optional` each).
    bool take(PyObject* const* args, Py_ssize_t given, Py_ssize_t wanted, unsigned optional) {
        if (given != wanted) return false;
        for (Py_ssize_t i = 0; i < wanted; ++i) {
            if (args[i] == Py_None && (optional >> i & 1)) continue;
            if (!THPVariable_Check(args[i])) return false;
            t[i] = THPVariable_Unpack(args[i]);
            there[i] = true;
            if (!t[i].is_cuda() || !t[i].is_contiguous()) return false;
            if (device < 0) device = t[i].get_device();
            if (t[i].get_device() != device) return false;
            for (const int64_t size : t[i].sizes())
                if (size > kLargest) return false;
        }
        return c10::cuda::current_device() == device;
    }
    const void* in(int i) const { return there[i] ? t[i].const_data_ptr() : nullptr; }
    void* out(int i) const { return there[i] ? t[i].mutable_data_ptr() : nullptr; }
    int size(int i, int d) const { return (int)t[i].size(d); }
    bool is(int i, at::ScalarType type, int dim) const { return t[i].scalar_type() == type && t[i].dim() == dim; }
    bool same_shape(int i, int j) const { return t[i].sizes() == t[j].sizes(); }
    void* stream() const { return c10::cuda::getCurrentCUDAStream(device).stream(); }
    // q and scales, uint8, belong together.
    bool fp4(int q, int scales) const {
        const int dim = (int)t[q].dim();
        if (t[q].scalar_type() != at::kByte || !is(scales, at::kByte, dim)) return false;
        for (int d = 0; d + 1 < dim; ++d)
            if (t[q].size(d) != t[scales].size(d)) return false;
        return t[scales].size(dim - 1) == (t[q].size(dim - 1) / 16 + 15) / 16 * 16 && t[q].size(dim - 1) <= kLargest / 2;
    }
};

// Runs `call`, which returns a status or -1 where the arguments are not what it takes, without the interpreter's lock.
template <typename F>
bool launched(const F& call) {
    int status;
    Py_BEGIN_ALLOW_THREADS;
    status = call();
    Py_END_ALLOW_THREADS;
    return status == TRB_OK;
}

template <typename F>
PyObject* answer(const F& f) {
    bool done = false;
    try {
        done = f();
    } catch (...) {  // a tensor without memory of its own, for one
        PyErr_Clear();
    }
    return PyBool_FromLong(done);
}

PyObject* expert_sort(PyObject*, PyObject* const* args, Py_ssize_t n) {  // experts, offsets, slots
    return answer([&] {
        Call c;
        if (!c.take(args, n, 3, 0)) return false;
        const bool wide = c.t[0].scalar_type() == at::kLong;
        if (!c.is(0, wide ? at::kLong : at::kInt, 2) || !c.is(1, at::kInt, 1) || !c.is(2, at::kInt, 2) ||
            !c.same_shape(0, 2) || c.size(1, 0) < 2)
            return false;
        const void* const ids = c.in(0);
        int* const offsets = static_cast<int*>(c.out(1));
        int* const slots = static_cast<int*>(c.out(2));
        void* const stream = c.stream();
        return launched([&] {
            return trb_expert_sort_launch(wide ? 8 : 4, c.size(0, 0), c.size(0, 1), c.size(1, 0) - 1, ids, offsets, slots,
                                          stream);
        });
    });
}

// x, slots, out, weights or y, slots, out, weights
PyObject* move(PyObject* const* args, Py_ssize_t n, bool back) {
    return answer([&] {
        Call c;
        if (!c.take(args, n, 4, 8)) return false;
        const int tokens_side = back ? 2 : 0, rows_side = 2 - tokens_side, dtype = dtype_code(c.t[0]);
        if (dtype < 0 || c.t[0].dim() != 2 || !c.is(2, c.t[0].scalar_type(), 2) || !c.is(1, at::kInt, 2) ||
            c.size(0, 1) != c.size(2, 1) || c.size(1, 0) != c.size(tokens_side, 0))
            return false;
        const int weight_dtype = c.there[3] ? dtype_code(c.t[3]) : dtype;
        if (c.there[3] && (weight_dtype < 0 || !c.same_shape(3, 1))) return false;
        const void *const src = c.in(0), *const weights = c.in(3);
        const int* const slots = static_cast<const int*>(c.in(1));
        void *const dst = c.out(2), *const stream = c.stream();
        return launched([&] {
            return (back ? trb_expert_combine_launch : trb_expert_dispatch_launch)(
                dtype, weight_dtype, c.size(1, 0), c.size(1, 1), c.size(rows_side, 0), c.size(0, 1), src, slots, weights,
                dst, stream);
        });
    });
}
PyObject* expert_dispatch(PyObject*, PyObject* const* args, Py_ssize_t n) { return move(args, n, false); }
PyObject* expert_combine(PyObject*, PyObject* const* args, Py_ssize_t n) { return move(args, n, true); }

PyObject* expert_combine_grad(PyObject*, PyObject* const* args, Py_ssize_t n) {  // grad, y, slots, weights, grad_y, grad_weights
    return answer([&] {
        Call c;
        if (!c.take(args, n, 6, 0)) return false;
        const int dtype = dtype_code(c.t[0]), weight_dtype = dtype_code(c.t[3]);
        const at::ScalarType type = c.t[0].scalar_type(), weight_type = c.t[3].scalar_type();
        if (dtype < 0 || weight_dtype < 0 || c.t[0].dim() != 2 || !c.is(1, type, 2) || !c.is(2, at::kInt, 2) ||
            c.t[3].dim() != 2 || !c.is(4, type, 2) || !c.is(5, weight_type, 2) || c.size(0, 1) != c.size(1, 1) ||
            c.size(2, 0) != c.size(0, 0) || !c.same_shape(3, 2) || !c.same_shape(4, 1) || !c.same_shape(5, 3))
            return false;
        const void *const grad = c.in(0), *const y = c.in(1), *const weights = c.in(3);
        const int* const slots = static_cast<const int*>(c.in(2));
        void *const grad_y = c.out(4), *const grad_weights = c.out(5), *const stream = c.stream();
        return launched([&] {
            return trb_expert_combine_grad_launch(dtype, weight_dtype, c.size(2, 0), c.size(2, 1), c.size(1, 0),
                                                  c.size(0, 1), grad, y, slots, weights, grad_y, grad_weights, stream);
        });
    });
}

PyObject* quantize_fp4(PyObject*, PyObject* const* args, Py_ssize_t n) {  // x, q, scales, slots
    return answer([&] {
        Call c;
        if (!c.take(args, n, 4, 8)) return false;
        const int dtype = dtype_code(c.t[0]);
        if (dtype < 0 || c.t[0].dim() != 2 || c.t[1].dim() != 2 || !c.fp4(1, 2) || 2 * c.t[1].size(1) != c.t[0].size(1))
            return false;
        if (c.there[3] ? !c.is(3, at::kInt, 2) || c.size(3, 0) != c.size(0, 0) : c.size(1, 0) != c.size(0, 0)) return false;
        const void* const x = c.in(0);
        const int* const slots = static_cast<const int*>(c.in(3));
        void *const q = c.out(1), *const scales = c.out(2), *const stream = c.stream();
        return launched([&] {
            return trb_quantize_fp4_launch(dtype, c.size(0, 0), c.size(0, 1), x, slots ? c.size(3, 1) : 1, slots,
                                           c.size(1, 0), q, scales, stream);
        });
    });
}

PyObject* dequantize_fp4(PyObject*, PyObject* const* args, Py_ssize_t n) {  // q, scales, out
    return answer([&] {
        Call c;
        if (!c.take(args, n, 3, 0)) return false;
        const int dtype = dtype_code(c.t[2]);
        if (dtype < 0 || c.t[0].dim() != 2 || c.t[2].dim() != 2 || !c.fp4(0, 1) || c.size(0, 0) != c.size(2, 0) ||
            2 * c.t[0].size(1) != c.t[2].size(1))
            return false;
        const void *const q = c.in(0), *const scales = c.in(1);
        void *const out = c.out(2), *const stream = c.stream();
        return launched([&] {
            return trb_dequantize_fp4_launch(dtype, c.size(2, 0), c.size(2, 1), q, scales, out, stream);
        });
    });
}

PyObject* gemm_fp4(PyObject*, PyObject* const* args, Py_ssize_t n) {  // a, a_scales, b, b_scales, out, offsets
    return answer([&] {
        Call c;
        if (!c.take(args, n, 6, 32)) return false;
        const int dtype = dtype_code(c.t[4]), dim = (int)c.t[2].dim();
        if (dtype < 0 || c.t[0].dim() != 2 || (dim != 2 && dim != 3) || c.t[4].dim() != 2 || !c.fp4(0, 1) || !c.fp4(2, 3))
            return false;
        const int groups = dim == 2 ? 1 : c.size(2, 0), outputs = c.size(2, dim - 2);
        if (c.size(2, dim - 1) != c.size(0, 1) || c.size(4, 0) != c.size(0, 0) || c.size(4, 1) != outputs) return false;
        if (c.there[5] ? !c.is(5, at::kInt, 1) || c.t[5].numel() != (int64_t)groups + 1 : groups != 1) return false;
        const void *const a = c.in(0), *const a_scales = c.in(1), *const b = c.in(2), *const b_scales = c.in(3);
        const int* const offsets = static_cast<const int*>(c.in(5));
        void *const out = c.out(4), *const stream = c.stream();
        return launched([&] {
            return trb_gemm_fp4_launch(dtype, groups, c.size(0, 0), outputs, 2 * c.size(0, 1), a, a_scales, b, b_scales,
                                       offsets, out, stream);
        });
    });
}

#define TRB_METHOD(NAME) {#NAME, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(NAME)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {TRB_METHOD(expert_sort),  TRB_METHOD(expert_dispatch), TRB_METHOD(expert_combine),
                         TRB_METHOD(expert_combine_grad), TRB_METHOD(quantize_fp4), TRB_METHOD(dequantize_fp4),
                         TRB_METHOD(gemm_fp4),     {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "trb_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_trb_torch(void) { return PyModule_Create(&module); }
