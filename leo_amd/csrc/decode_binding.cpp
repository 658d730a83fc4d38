// The Python face of include/leo_decode.h for torch tensors: checks, results and
// the call in compiled code. A step of generation makes these calls once a byte,
// and for short rows the same work in Python took longer than the kernels: one
// host call from Python and from here, timed in turn on one card, took 7.4 and
// 4.1 us for the 4-bit product of one row and 257 outputs, 10.9 and 4.1 us for the
// control and 10.0 and 4.9 us for the draw of a row of 257 symbols.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <string>

#include "leo_decode.h"
#include "leo_hip.h"

namespace {

PyObject* g_error = nullptr;      // native.LeoError
PyObject* g_stream_of = nullptr;  // the stream of a device's number

struct Refusal {
    int code;
    std::string message;
};

[[noreturn]] void refuse(const std::string& message) { throw Refusal{LEO_ERR_INVALID_ARGUMENT, message}; }

void check(int32_t status) {
    if (status == LEO_OK) return;
    char message[4096] = "";
    leo_hip_last_error(message, sizeof(message));
    throw Refusal{status, message};
}

constexpr int kFloating = -1;

int type_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return LEO_TYPE_F32;
        case at::kHalf: return LEO_TYPE_F16;
        case at::kBFloat16: return LEO_TYPE_BF16;
        default: return -1;
    }
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor on the GPU");
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda()) refuse(std::string(name) + " must be a tensor on the GPU");
    return t;
}

void same_device(const at::Tensor& t, const char* name, int index) {
    if (t.get_device() != index)
        refuse(std::string(name) + " is on GPU " + std::to_string(t.get_device()) + ", not on " + std::to_string(index));
}

struct Matrix {
    const void* data;
    int64_t rows, width, stride;
    int type;
};

// A 2-D tensor whose last axis is dense, of the type or (kFloating) one of the three floating ones.
Matrix matrix(const at::Tensor& t, const char* name, int index, int type) {
    same_device(t, name, index);
    const int own = type_of(t.scalar_type());
    if (type == kFloating ? own < 0 : t.scalar_type() != static_cast<at::ScalarType>(type))
        refuse(std::string(name) + " has type " + c10::toString(t.scalar_type()));
    if (t.dim() != 2) refuse(std::string(name) + " must have two axes, not " + std::to_string(t.dim()));
    if (t.size(1) > 1 && t.stride(1) != 1) refuse(std::string(name) + "'s last axis must be dense");
    return {t.const_data_ptr(), t.size(0), t.size(1), t.stride(0), own};
}

// The data of a dense 1-D tensor of `count` entries (any number below 0), null for None.
template <class T>
const T* vector(PyObject* o, const char* name, at::ScalarType type, int index, int64_t count, int64_t* size = nullptr) {
    if (o == Py_None) return nullptr;
    const at::Tensor& t = tensor(o, name);
    same_device(t, name, index);
    if (t.scalar_type() != type)
        refuse(std::string(name) + " must have type " + c10::toString(type) + ", not " + c10::toString(t.scalar_type()));
    if (t.dim() != 1 || !t.is_contiguous() || (count >= 0 && t.numel() != count))
        refuse(std::string(name) + " must be a dense vector" + (count >= 0 ? " of " + std::to_string(count) + " entries" : ""));
    if (size) *size = t.numel();
    return static_cast<const T*>(t.const_data_ptr());
}

void* stream_of(int index) {
    PyObject* number = PyLong_FromLong(index);
    PyObject* stream = number ? PyObject_CallOneArg(g_stream_of, number) : nullptr;
    Py_XDECREF(number);
    if (!stream) throw python_error();
    void* p = PyLong_AsVoidPtr(stream);
    Py_DECREF(stream);
    if (!p && PyErr_Occurred()) throw python_error();
    return p;
}

at::Tensor workspace(uint64_t bytes, const at::Tensor& like) {  // free again in the stream's order
    return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}

template <class F>
PyObject* guarded(F&& f) {
    try {
        return f();
    } catch (const Refusal& r) {
        PyObject* value = PyObject_CallFunction(g_error, "is", r.code, r.message.c_str());
        if (value) PyErr_SetObject(g_error, value);
        Py_XDECREF(value);
    } catch (python_error& e) {
        e.restore();
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

bool given(Py_ssize_t n, Py_ssize_t wanted) {
    if (n == wanted) return true;
    PyErr_Format(PyExc_TypeError, "%zd arguments are needed, not %zd", wanted, n);
    return false;
}

// q4_matvec(x, layout, shape as bytes, bias, out or the result's type as LEO_TYPE_* (-1: x's))
PyObject* q4_matvec(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!given(n, 5)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor& layout = tensor(args[1], "layout");
        const int index = layout.get_device();
        LeoQ4Product p{};
        if (!PyBytes_Check(args[2]) || PyBytes_GET_SIZE(args[2]) != sizeof(p.shape)) refuse("shape must be a LeoQ4Shape");
        memcpy(&p.shape, PyBytes_AS_STRING(args[2]), sizeof(p.shape));
        const at::Tensor& input = tensor(args[0], "x");
        const Matrix x = matrix(input, "x", index, kFloating);
        if (static_cast<uint64_t>(x.width) != p.shape.inputs)
            refuse("x has " + std::to_string(x.width) + " inputs, the weight " + std::to_string(p.shape.inputs));
        const int64_t outputs = static_cast<int64_t>(p.shape.outputs);
        at::Tensor out;
        if (PyLong_Check(args[4])) {
            static constexpr at::ScalarType kTypes[] = {at::kFloat, at::kHalf, at::kBFloat16};
            const long type = PyLong_AsLong(args[4]);
            if (type < -1 || type > 2) refuse("the result must be float32, float16 or bfloat16");
            out = at::empty({x.rows, outputs}, type < 0 ? input.options() : input.options().dtype(kTypes[type]));
        } else {
            out = tensor(args[4], "out");
        }
        const Matrix y = matrix(out, "out", index, kFloating);
        if (y.rows != x.rows || y.width != outputs)
            refuse("out must be (" + std::to_string(x.rows) + ", " + std::to_string(outputs) + ")");
        p.layout = layout.const_data_ptr();
        p.layout_bytes = static_cast<uint64_t>(layout.numel());
        p.rows = static_cast<uint64_t>(x.rows);
        p.x = x.data;
        p.x_stride = x.stride;
        p.x_type = x.type;
        p.bias = vector<float>(args[3], "bias", at::kFloat, index, outputs);
        p.y = out.data_ptr();
        p.y_stride = y.stride;
        p.y_type = y.type;
        const c10::DeviceGuard guard(input.device());
        check(leo_q4_workspace_bytes(&p.shape, p.rows, p.x_type, &p.workspace_bytes));
        at::Tensor space;
        if (p.workspace_bytes) {
            space = workspace(p.workspace_bytes, input);
            p.workspace = space.data_ptr();
        }
        check(leo_q4_matvec(&p, stream_of(index)));
        return THPVariable_Wrap(out);
    });
}

// control_logits(logits, history, history offsets, repetition, presence, frequency, bias ids, values, offsets, masks,
// mask_rows, out); None for what is not given
PyObject* control_logits(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!given(n, 12)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor& logits = tensor(args[0], "logits");
        const int index = logits.get_device();
        const Matrix z = matrix(logits, "logits", index, kFloating);
        at::Tensor out = args[11] == Py_None ? at::empty({z.rows, z.width}, logits.options()) : tensor(args[11], "out");
        const Matrix to = matrix(out, "out", index, static_cast<int>(logits.scalar_type()));
        if (to.rows != z.rows || to.width != z.width)
            refuse("out must be (" + std::to_string(z.rows) + ", " + std::to_string(z.width) + ")");
        LeoLogitControl c{};
        c.rows = static_cast<uint64_t>(z.rows);
        c.symbols = static_cast<uint64_t>(z.width);
        c.logits = z.data;
        c.logits_stride = z.stride;
        c.out = out.data_ptr();
        c.out_stride = to.stride;
        c.type = z.type;
        int64_t count = 0;
        if ((args[1] == Py_None) != (args[2] == Py_None)) refuse("history needs its offsets");
        c.history = vector<int32_t>(args[1], "history", at::kInt, index, -1, &count);
        c.history_count = static_cast<uint64_t>(count);
        c.history_offsets = vector<int64_t>(args[2], "history offsets", at::kLong, index, z.rows + 1);
        c.repetition = vector<float>(args[3], "repetition", at::kFloat, index, z.rows);
        c.presence = vector<float>(args[4], "presence", at::kFloat, index, z.rows);
        c.frequency = vector<float>(args[5], "frequency", at::kFloat, index, z.rows);
        if ((args[6] == Py_None) != (args[7] == Py_None) || (args[6] == Py_None) != (args[8] == Py_None))
            refuse("bias needs ids, values and offsets");
        count = 0;
        c.bias_ids = vector<int32_t>(args[6], "bias ids", at::kInt, index, -1, &count);
        c.bias_values = vector<float>(args[7], "bias values", at::kFloat, index, count);
        c.bias_count = static_cast<uint64_t>(count);
        c.bias_offsets = vector<int64_t>(args[8], "bias offsets", at::kLong, index, z.rows + 1);
        if (args[9] != Py_None) {
            const Matrix m = matrix(tensor(args[9], "masks"), "masks", index, static_cast<int>(at::kInt));
            if (m.width != (z.width + 31) / 32)
                refuse("masks of " + std::to_string(z.width) + " symbols have " + std::to_string((z.width + 31) / 32) +
                       " words, not " + std::to_string(m.width));
            if (m.rows < 1) refuse("masks have no rows");
            c.masks = static_cast<const int32_t*>(m.data);
            c.masks_stride = m.stride;
            c.mask_count = static_cast<uint64_t>(m.rows);
        } else if (args[10] != Py_None) {
            refuse("mask_rows without masks");
        }
        c.mask_rows = vector<int32_t>(args[10], "mask_rows", at::kInt, index, z.rows);
        const c10::DeviceGuard guard(logits.device());
        check(leo_control_logits(&c, stream_of(index)));
        return THPVariable_Wrap(out);
    });
}

// sample(logits, noise, temperature, top_k, top_p, min_p); None for what is not given
PyObject* sample(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!given(n, 6)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor& logits = tensor(args[0], "logits");
        const int index = logits.get_device();
        const Matrix z = matrix(logits, "logits", index, kFloating);
        if (z.width < 1) refuse("no symbols to draw from");
        LeoSample s{};
        s.rows = static_cast<uint64_t>(z.rows);
        s.symbols = static_cast<uint64_t>(z.width);
        s.logits = z.data;
        s.logits_stride = z.stride;
        s.type = z.type;
        if (args[1] != Py_None) {
            const Matrix g = matrix(tensor(args[1], "noise"), "noise", index, static_cast<int>(at::kFloat));
            if (g.rows != z.rows || g.width != z.width)
                refuse("noise must be (" + std::to_string(z.rows) + ", " + std::to_string(z.width) + ")");
            s.noise = static_cast<const float*>(g.data);
            s.noise_stride = g.stride;
        }
        s.temperature = vector<float>(args[2], "temperature", at::kFloat, index, z.rows);
        s.top_k = vector<int32_t>(args[3], "top_k", at::kInt, index, z.rows);
        s.top_p = vector<float>(args[4], "top_p", at::kFloat, index, z.rows);
        s.min_p = vector<float>(args[5], "min_p", at::kFloat, index, z.rows);
        const c10::DeviceGuard guard(logits.device());
        at::Tensor drawn = at::empty({z.rows}, logits.options().dtype(at::kInt));
        at::Tensor logprobs = at::empty({z.rows}, logits.options().dtype(at::kFloat));
        s.out_symbols = static_cast<int32_t*>(drawn.data_ptr());
        s.out_logprobs = static_cast<float*>(logprobs.data_ptr());
        check(leo_sample_workspace_bytes(s.rows, s.symbols, &s.workspace_bytes));
        at::Tensor space;
        if (s.workspace_bytes) {
            space = workspace(s.workspace_bytes, logits);
            s.workspace = space.data_ptr();
        }
        check(leo_sample(&s, stream_of(index)));
        PyObject* first = THPVariable_Wrap(drawn);
        PyObject* second = THPVariable_Wrap(logprobs);
        PyObject* both = first && second ? PyTuple_Pack(2, first, second) : nullptr;
        Py_XDECREF(first);
        Py_XDECREF(second);
        return both;
    });
}

// setup(LeoError, stream_of)
PyObject* setup(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!given(n, 2)) return nullptr;
    for (int i = 0; i < 2; ++i) Py_INCREF(args[i]);
    Py_XSETREF(g_error, args[0]);
    Py_XSETREF(g_stream_of, args[1]);
    Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"q4_matvec", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(q4_matvec)), METH_FASTCALL, nullptr},
    {"control_logits", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(control_logits)), METH_FASTCALL, nullptr},
    {"sample", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(sample)), METH_FASTCALL, nullptr},
    {"setup", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(setup)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "leo_decode_binding", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_leo_decode_binding() { return PyModule_Create(&kModule); }
