// The Python face of include/leo_decode.h for torch tensors: checks, results and
// the call in compiled code. A step of generation makes these calls once a byte,
// and for short rows the same work in Python took longer than the kernels: one
// host call from Python and from here, timed in turn on one card, took 7.4 and
// 4.1 us for the 4-bit product of one row and 257 outputs, 10.9 and 4.1 us for the
// control and 10.0 and 4.9 us for the draw of a row of 257 symbols.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/DimVector.h>
#include <ATen/core/Tensor.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/util/SmallVector.h>
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

// A new dense tensor, without the dispatch that torch.empty goes through first.
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
    return at::Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}

at::Tensor workspace(uint64_t bytes, const at::Tensor& like) {  // free again in the stream's order
    return fresh({static_cast<int64_t>(bytes)}, at::kByte, like);
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

struct Q4 {
    using Product = LeoQ4Product;
    static constexpr const char* kShape = "shape must be a LeoQ4Shape";
    static constexpr auto workspace_bytes = leo_q4_workspace_bytes;
    static constexpr auto call = leo_q4_matvec;
};
struct Q8 {
    using Product = LeoQ8Product;
    static constexpr const char* kShape = "shape must be a LeoQ8Shape";
    static constexpr auto workspace_bytes = leo_q8_workspace_bytes;
    static constexpr auto call = leo_q8_matmul;
};

// product(x, layout, shape as bytes, bias, out or the result's type as LEO_TYPE_* (-1: x's))
template <class Q>
PyObject* product(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!given(n, 5)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor& layout = tensor(args[1], "layout");
        const int index = layout.get_device();
        typename Q::Product p{};
        if (!PyBytes_Check(args[2]) || PyBytes_GET_SIZE(args[2]) != sizeof(p.shape)) refuse(Q::kShape);
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
            out = fresh({x.rows, outputs}, type < 0 ? input.scalar_type() : kTypes[type], input);
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
        check(Q::workspace_bytes(&p.shape, p.rows, p.x_type, &p.workspace_bytes));
        at::Tensor space;
        if (p.workspace_bytes) {
            space = workspace(p.workspace_bytes, input);
            p.workspace = space.data_ptr();
        }
        check(Q::call(&p, stream_of(index)));
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
        at::Tensor out = args[11] == Py_None ? fresh({z.rows, z.width}, logits.scalar_type(), logits) : tensor(args[11], "out");
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
        at::Tensor drawn = fresh({z.rows}, at::kInt, logits);
        at::Tensor logprobs = fresh({z.rows}, at::kFloat, logits);
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

// A dense 2-D tensor of a type.
const at::Tensor& table(PyObject* o, const char* name, at::ScalarType type, int index) {
    const at::Tensor& t = tensor(o, name);
    same_device(t, name, index);
    if (t.scalar_type() != type)
        refuse(std::string(name) + " must have type " + c10::toString(type) + ", not " + c10::toString(t.scalar_type()));
    if (t.dim() != 2 || !t.is_contiguous()) refuse(std::string(name) + " must be dense with two axes");
    return t;
}

// beam_select(logits, scores, kept, finished, lengths, length_penalty, end); None for what is not given
PyObject* beam_select(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!given(n, 7)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor& logits = tensor(args[0], "logits");
        const int index = logits.get_device();
        const Matrix z = matrix(logits, "logits", index, kFloating);
        const at::Tensor& scores = table(args[1], "scores", at::kFloat, index);
        LeoBeams b{};
        const int64_t groups = scores.size(0), beams = scores.size(1);
        const int64_t kept = args[2] == Py_None ? beams : PyLong_AsLongLong(args[2]);
        if (PyErr_Occurred()) throw python_error();
        if (beams < 1 || beams > 64) refuse("scores have 1 to 64 beams, not " + std::to_string(beams));
        if (z.rows != groups * beams)
            refuse("logits have " + std::to_string(z.rows) + " rows, the scores " + std::to_string(groups * beams) + " entries");
        b.groups = static_cast<uint64_t>(groups);
        b.beams = static_cast<uint64_t>(beams);
        b.kept = static_cast<uint64_t>(kept);
        b.symbols = static_cast<uint64_t>(z.width);
        b.logits = z.data;
        b.logits_stride = z.stride;
        b.type = z.type;
        b.scores = static_cast<const float*>(scores.const_data_ptr());
        const auto beside = [&](PyObject* o, const char* name, at::ScalarType type) -> const void* {
            if (o == Py_None) return nullptr;
            const at::Tensor& t = table(o, name, type, index);
            if (t.size(0) != groups || t.size(1) != beams)
                refuse(std::string(name) + " must be (" + std::to_string(groups) + ", " + std::to_string(beams) + ")");
            return t.const_data_ptr();
        };
        b.finished = static_cast<const uint8_t*>(beside(args[3], "finished", at::kBool));
        b.lengths = static_cast<const int32_t*>(beside(args[4], "lengths", at::kInt));
        b.length_penalty = PyFloat_AsDouble(args[5]);
        if (PyErr_Occurred()) throw python_error();
        b.end = -1;
        if (args[6] != Py_None) {
            b.end = PyLong_AsLongLong(args[6]);
            if (PyErr_Occurred()) throw python_error();
            if (b.end < 0) refuse("end must be a symbol");
        }
        const c10::DeviceGuard guard(logits.device());
        check(leo_beam_workspace_bytes(b.groups, b.beams, b.kept, b.symbols, &b.workspace_bytes));
        at::Tensor outs[5];
        const auto out = [&](int i, at::ScalarType type) {
            outs[i] = fresh({groups, kept}, type, logits);
            return outs[i].data_ptr();
        };
        b.out_symbols = static_cast<int32_t*>(out(0, at::kInt));
        b.out_parents = static_cast<int32_t*>(out(1, at::kInt));
        b.out_scores = static_cast<float*>(out(2, at::kFloat));
        if (b.finished || args[6] != Py_None) b.out_finished = static_cast<uint8_t*>(out(3, at::kBool));
        if (b.lengths) b.out_lengths = static_cast<int32_t*>(out(4, at::kInt));
        at::Tensor space;
        if (b.workspace_bytes) {
            space = workspace(b.workspace_bytes, logits);
            b.workspace = space.data_ptr();
        }
        check(leo_beam_select(&b, stream_of(index)));
        PyObject* result = PyTuple_New(5);
        if (!result) throw python_error();
        for (int i = 0; i < 5; ++i) {
            PyObject* o = Py_None;
            if (outs[i].defined()) o = THPVariable_Wrap(outs[i]);
            else Py_INCREF(o);
            if (!o) {
                Py_DECREF(result);
                throw python_error();
            }
            PyTuple_SET_ITEM(result, i, o);
        }
        return result;
    });
}

// A state's rows as pieces of dense bytes: every axis but the first joined to the
// one behind it where it can be, and one more beside.
struct Pieces {
    int64_t row, outer, width;  // bytes
    uint64_t count;
    bool fits;
};
Pieces pieces(const at::Tensor& t) {
    const int64_t e = static_cast<int64_t>(t.element_size());
    Pieces p{t.stride(0) * e, 0, e, 1, true};
    for (int64_t d = t.dim() - 1; d > 0; --d) {
        const int64_t size = t.size(d), stride = t.stride(d) * e;
        if (size == 1) continue;
        if (p.count == 1 && stride == p.width) {
            p.width *= size;
        } else if (p.count == 1) {
            p.outer = stride;
            p.count = static_cast<uint64_t>(size);
        } else if (stride == p.outer * static_cast<int64_t>(p.count)) {
            p.count *= static_cast<uint64_t>(size);
        } else {
            p.fits = false;
        }
    }
    return p;
}

// reorder_states(states as a tuple, parents, outs as a tuple or None): a list of the results
PyObject* reorder_states(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!given(n, 3)) return nullptr;
    return guarded([&]() -> PyObject* {
        if (!PyTuple_Check(args[0]) || (args[2] != Py_None && !PyTuple_Check(args[2]))) refuse("states and outs must be tuples");
        const at::Tensor& order = tensor(args[1], "parents");
        const int index = order.get_device();
        table(args[1], "parents", at::kInt, index);
        const Py_ssize_t count = PyTuple_GET_SIZE(args[0]);
        if (args[2] != Py_None && PyTuple_GET_SIZE(args[2]) != count) refuse("out needs a tensor for each of the states");
        const int64_t groups = order.size(0), kept = order.size(1);
        if (kept < 1 || kept > 64) refuse("parents have 1 to 64 places a row, not " + std::to_string(kept));
        const c10::DeviceGuard guard(order.device());
        c10::SmallVector<at::Tensor, 16> outs;
        c10::SmallVector<LeoStateArray, 16> arrays;
        int64_t beams = 0;
        for (Py_ssize_t i = 0; i < count; ++i) {
            const at::Tensor& t = tensor(PyTuple_GET_ITEM(args[0], i), "a state");
            same_device(t, "a state", index);
            if (t.layout() != at::kStrided || t.is_conj() || t.is_neg()) refuse("a state must be a dense tensor, its values as they are in memory");
            if (t.dim() < 1) refuse("a state needs an axis of rows");
            if (groups > 0 && (t.size(0) % groups || t.size(0) == 0 || (i && t.size(0) != groups * beams)))
                refuse("a state has " + std::to_string(t.size(0)) + " rows for " + std::to_string(groups) + " groups" +
                       (i ? " of " + std::to_string(beams) + " beams" : ""));
            if (groups == 0 && t.size(0)) refuse("a state has rows, the parents none");
            beams = groups ? t.size(0) / groups : 1;
            at::DimVector sizes(t.sizes());
            sizes[0] = groups * kept;
            if (args[2] == Py_None) {
                outs.push_back(fresh(sizes, t.scalar_type(), t));
            } else {
                const at::Tensor& out = tensor(PyTuple_GET_ITEM(args[2], i), "out");
                same_device(out, "out", index);
                if (out.layout() != at::kStrided || out.is_conj() || out.is_neg() || out.scalar_type() != t.scalar_type() || out.sizes() != at::IntArrayRef(sizes))
                    refuse("out must have the states' types, and their shapes with " + std::to_string(groups * kept) + " rows");
                outs.push_back(out);
            }
            if (t.numel() == 0) continue;
            Pieces from = pieces(t), to = pieces(outs.back());
            if (!from.fits || !to.fits) refuse("a state's axes behind the first must join to two at most, the last of them dense");
            // the wider side in the other's pieces
            if (from.count == 1 && to.count > 1) {
                from.outer = to.width;
                from.width = to.width;
                from.count = to.count;
            } else if (to.count == 1 && from.count > 1) {
                to.outer = from.width;
                to.width = from.width;
                to.count = from.count;
            }
            if (from.count != to.count || from.width != to.width) refuse("a state and its out must join to the same pieces");
            arrays.push_back({t.const_data_ptr(), outs.back().data_ptr(), from.count, static_cast<uint64_t>(from.width),
                              from.row, from.outer, to.row, to.outer});
        }
        if (beams > 64) refuse("64 beams are the most, not " + std::to_string(beams));
        LeoReorder r{};
        r.arrays = arrays.data();
        r.count = arrays.size();
        r.groups = static_cast<uint64_t>(groups);
        r.beams = static_cast<uint64_t>(count ? beams : 1);
        r.kept = static_cast<uint64_t>(kept);
        r.parents = static_cast<const int32_t*>(order.const_data_ptr());
        check(leo_reorder_states(&r, stream_of(index)));
        PyObject* result = PyList_New(count);
        if (!result) throw python_error();
        for (Py_ssize_t i = 0; i < count; ++i) {
            PyObject* o = THPVariable_Wrap(outs[static_cast<size_t>(i)]);
            if (!o) {
                Py_DECREF(result);
                throw python_error();
            }
            PyList_SET_ITEM(result, i, o);
        }
        return result;
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
    {"q4_matvec", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(product<Q4>)), METH_FASTCALL, nullptr},
    {"q8_matmul", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(product<Q8>)), METH_FASTCALL, nullptr},
    {"control_logits", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(control_logits)), METH_FASTCALL, nullptr},
    {"sample", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(sample)), METH_FASTCALL, nullptr},
    {"beam_select", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(beam_select)), METH_FASTCALL, nullptr},
    {"reorder_states", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(reorder_states)), METH_FASTCALL, nullptr},
    {"setup", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(setup)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "leo_decode_binding", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_leo_decode_binding() { return PyModule_Create(&kModule); }
