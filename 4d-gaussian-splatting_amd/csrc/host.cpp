// fdgs._host: the per-tensor host work of the entry points over lists of tensors.
//
// A step over 200 tensors looks at 1400 tensors' types, sizes, layouts, devices and addresses.  From Python each look
// costs 0.1 to 0.4 us, 5 to 7 us a tensor, several times what the GPU needs for the step; here the whole list costs
// about 0.3 us a tensor.  Every check raises the Python exception that a caller sees; nothing is launched from here.
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <algorithm>
#include <cstring>
#include <stdexcept>
#include <string>
#include <vector>
#include "fdgs.h"

namespace {

struct Refused { PyObject* type; std::string what; };
[[noreturn]] void value_error(const std::string& s) { throw Refused{PyExc_ValueError, s}; }
struct Raised {};                                    // a Python exception is set

struct Ref {                                         // an owned reference
    PyObject* p;
    explicit Ref(PyObject* o) : p(o) { if (!p) throw Raised(); }
    ~Ref() { Py_XDECREF(p); }
    Ref(const Ref&) = delete;
    Ref& operator=(const Ref&) = delete;
    PyObject* give() { PyObject* o = p; p = nullptr; return o; }
};

struct List {                                        // a list or tuple (anything else is made one)
    Ref seq;
    explicit List(PyObject* o) : seq(PySequence_Fast(o, "a list of tensors is needed")) {}
    Py_ssize_t size() const { return PySequence_Fast_GET_SIZE(seq.p); }
    PyObject* at(Py_ssize_t i) const { return PySequence_Fast_GET_ITEM(seq.p, i); }
};

const at::Tensor& tensor(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) throw Refused{PyExc_TypeError, std::string(what) + ": a tensor is needed, not " + Py_TYPE(o)->tp_name};
    return THPVariable_Unpack(o);
}

// One number for all of n tensors, or a list or tuple of n.
struct Each {
    PyObject* o;
    bool many;
    Each(PyObject* x, Py_ssize_t n, const char* what) : o(x), many(PyList_Check(x) || PyTuple_Check(x)) {
        if (many && PySequence_Fast_GET_SIZE(o) != n)
            value_error(std::string(what) + ": one value, or one for each of the " + std::to_string(n) + " tensors");
    }
    PyObject* at(Py_ssize_t i) const { return many ? PySequence_Fast_GET_ITEM(o, i) : o; }
    double number(Py_ssize_t i) const {
        const double v = PyFloat_AsDouble(at(i));
        if (v == -1.0 && PyErr_Occurred()) throw Raised();
        return v;
    }
    long long whole(Py_ssize_t i) const {
        Ref n(PyNumber_Index(at(i)));
        const long long v = PyLong_AsLongLong(n.p);
        if (v == -1 && PyErr_Occurred()) throw Raised();
        return v;
    }
    uint32_t low32(Py_ssize_t i) const {             // the low 32 bits of any whole number
        Ref n(PyNumber_Index(at(i)));
        const unsigned long v = PyLong_AsUnsignedLongMask(n.p);
        if (v == (unsigned long)-1 && PyErr_Occurred()) throw Raised();
        return (uint32_t)v;
    }
};

std::string name_of(const at::Tensor& t) { return std::string("torch.") + (t.scalar_type() == at::kFloat ? "float32" : t.scalar_type() == at::kBFloat16 ? "bfloat16" : c10::toString(t.scalar_type())); }

struct Moment { const at::Tensor *codes, *exps; bool is_signed; };

bool is_moment(PyObject* o, PyObject* cls) { return (PyObject*)Py_TYPE(o) == cls || PyObject_IsInstance(o, cls) == 1; }

Moment moment8(PyObject* o, PyObject* cls, int64_t numel, const at::Device& device, const std::string& what) {
    if (!is_moment(o, cls)) value_error(what + ": an 8-bit moment is an adamw.Moment8; do not mix moments in 8 and in 32 bits");
    const at::Tensor &c = tensor(PyTuple_GET_ITEM(o, 0), "codes"), &e = tensor(PyTuple_GET_ITEM(o, 1), "exponents");
    const int truth = PyObject_IsTrue(PyTuple_GET_ITEM(o, 2));
    if (truth < 0) throw Raised();
    if (c.scalar_type() != at::kByte || e.scalar_type() != at::kByte || !c.is_contiguous() || !e.is_contiguous())
        value_error(what + ": codes and exponents are contiguous uint8 tensors");
    if (c.numel() != numel || e.numel() != (numel + FDGS_MOMENT8_BLOCK - 1) / FDGS_MOMENT8_BLOCK)
        value_error(what + ": one code per element, one exponent per " + std::to_string(FDGS_MOMENT8_BLOCK) + " elements");
    if (c.device() != device || e.device() != device) value_error(what + ": every tensor of a call is on one device");
    return {&c, &e, truth != 0};
}

void on_gpu(const at::Tensor& t) {
    if (!t.is_cuda()) throw Refused{PyExc_RuntimeError, "libfdgs kernels run on the GPU only; got a tensor on " + t.device().str()};
}

// adamw_records(params, grads, exp_avgs, exp_avg_sqs, residuals | None, steps, lr, weight_decay, keys | None, Moment8)
//   -> (records, param type, state bits, copies of gradients to keep until the launch)
PyObject* adamw_records(PyObject* a) {
    PyObject *po, *go, *mo, *vo, *ro, *so, *lo, *wo, *ko, *cls;
    if (!PyArg_ParseTuple(a, "OOOOOOOOOO", &po, &go, &mo, &vo, &ro, &so, &lo, &wo, &ko, &cls)) throw Raised();
    List p(po), g(go), m(mo), v(vo);
    const Py_ssize_t n = p.size();
    if (g.size() != n || m.size() != n || v.size() != n) value_error("params, grads and moments have to be lists of the same length");
    if (n == 0) value_error("no tensors");
    const Each steps(so, n, "steps"), lr(lo, n, "lr"), wd(wo, n, "weight_decay");
    const at::Tensor& first = tensor(p.at(0), "params");
    const at::ScalarType type = first.scalar_type();
    const at::Device device = first.device();
    const bool bf16 = type == at::kBFloat16;
    if (!bf16 && type != at::kFloat) value_error("adamw_step takes float32 and bfloat16 parameters, not " + name_of(first));
    on_gpu(first);
    Py_ssize_t nr = 0;
    std::vector<PyObject*> low;
    Ref rseq(ro == Py_None ? PyTuple_New(0) : PySequence_Fast(ro, "residuals: a list of tensors is needed"));
    nr = PySequence_Fast_GET_SIZE(rseq.p);
    if (bf16 && nr != n) value_error("bfloat16 parameters need residuals: an int16 tensor for each");
    const bool eight = is_moment(m.at(0), cls);
    if (eight && (ko == Py_None || !(PyList_Check(ko) || PyTuple_Check(ko)) || PySequence_Fast_GET_SIZE(ko) != n))
        value_error("8-bit moments need keys: a number for each tensor, others at every step");
    Ref hold(PyList_New(0));
    Ref bytes(PyBytes_FromStringAndSize(nullptr, n * (Py_ssize_t)sizeof(fdgs_adamw_tensor)));
    fdgs_adamw_tensor* out = (fdgs_adamw_tensor*)PyBytes_AS_STRING(bytes.p);
    std::vector<uintptr_t> written;
    written.reserve(3 * n);
    for (Py_ssize_t i = 0; i < n; ++i) {
        const at::Tensor &pt = tensor(p.at(i), "params"), &gt = tensor(g.at(i), "grads");
        const int64_t numel = pt.numel();
        fdgs_adamw_tensor r;
        memset(&r, 0, sizeof(r));
        if (pt.scalar_type() != type || gt.scalar_type() != type)
            value_error("parameters and gradients of one step have one type: " + name_of(first) + ", " + name_of(pt) + " and " + name_of(gt) + " given");
        if (gt.numel() != numel || !pt.is_contiguous()) value_error("a parameter has to be contiguous, and its gradient of its size");
        if (pt.device() != device || gt.device() != device) value_error("every tensor of a call is on one device");
        r.grad = gt.data_ptr();
        if (!gt.is_contiguous()) {
            // rows that are contiguous runs a constant distance apart are read in place
            int64_t len = 1;
            bool rows = gt.dim() >= 2 && gt.size(0) > 0 && gt.stride(0) > 0;
            for (int64_t d = gt.dim() - 1; rows && d >= 1; --d) {
                if (gt.size(d) != 1 && gt.stride(d) != len) rows = false;
                len *= gt.size(d);
            }
            if (rows && len > 0 && gt.stride(0) >= len && len <= INT32_MAX) {
                r.grad_row_len = (int32_t)len;
                r.grad_row_stride = gt.stride(0);
            } else {
                const at::Tensor copy = gt.detach().contiguous();
                r.grad = copy.data_ptr();
                Ref held(THPVariable_Wrap(copy));
                if (PyList_Append(hold.p, held.p) < 0) throw Raised();
            }
        }
        if (eight) {
            const Moment mm = moment8(m.at(i), cls, numel, device, "exp_avgs"), vv = moment8(v.at(i), cls, numel, device, "exp_avg_sqs");
            if (!mm.is_signed || vv.is_signed) value_error("the first moment is signed, the second is not");
            r.exp_avg = mm.codes->data_ptr();
            r.exp_avg_sq = vv.codes->data_ptr();
            r.exp_avg_exponents = (uint8_t*)mm.exps->data_ptr();
            r.exp_avg_sq_exponents = (uint8_t*)vv.exps->data_ptr();
            const Each keys(ko, n, "keys");
            r.round_key = keys.low32(i);
        } else {
            for (int k = 0; k < 2; ++k) {
                PyObject* o = (k ? v : m).at(i);
                if (!THPVariable_Check(o)) value_error("moments are float32 tensors, or all of them Moment8");
                const at::Tensor& x = THPVariable_Unpack(o);
                if (x.scalar_type() != at::kFloat || x.numel() != numel || !x.is_contiguous() || x.device() != device)
                    value_error("moments are contiguous float32 tensors of the parameter's size on its device, or all of them Moment8");
                (k ? r.exp_avg_sq : r.exp_avg) = x.data_ptr();
            }
        }
        if (bf16) {
            const at::Tensor& x = tensor(PySequence_Fast_GET_ITEM(rseq.p, i), "residuals");
            if (x.scalar_type() != at::kShort || x.numel() != numel || !x.is_contiguous() || x.device() != device)
                value_error("a residual is a contiguous int16 tensor of the parameter's size on its device");
            r.residual = (int16_t*)x.data_ptr();
        }
        const long long step = steps.whole(i);
        if (step < 1 || step > INT32_MAX) value_error("steps count from 1");
        r.param = pt.data_ptr();
        r.numel = numel;
        r.step = (int32_t)step;
        r.lr = lr.number(i);
        r.weight_decay = wd.number(i);
        if (numel) {
            written.push_back((uintptr_t)r.param);
            written.push_back((uintptr_t)r.exp_avg);
            written.push_back((uintptr_t)r.exp_avg_sq);
        }
        out[i] = r;
    }
    std::sort(written.begin(), written.end());
    if (std::adjacent_find(written.begin(), written.end()) != written.end()) value_error("a tensor is in the lists twice");
    return Py_BuildValue("NiiN", bytes.give(), bf16 ? FDGS_TYPE_BF16 : FDGS_TYPE_F32, eight ? 8 : 32, hold.give());
}

// moment8_records(moments, values, keys | None, Moment8) -> (records, value type)
PyObject* moment8_records(PyObject* a) {
    PyObject *mo, *vo, *ko, *cls;
    if (!PyArg_ParseTuple(a, "OOOO", &mo, &vo, &ko, &cls)) throw Raised();
    List m(mo), v(vo);
    const Py_ssize_t n = m.size();
    if (n == 0 || v.size() != n) value_error("a tensor of values is needed for each moment");
    const Each keys(ko, n, "keys");
    const at::Tensor& first = tensor(v.at(0), "values");
    const at::ScalarType type = first.scalar_type();
    if (type != at::kFloat && type != at::kBFloat16) value_error("the values of 8-bit moments are float32 or bfloat16");
    on_gpu(first);
    Ref bytes(PyBytes_FromStringAndSize(nullptr, n * (Py_ssize_t)sizeof(fdgs_moment8_tensor)));
    fdgs_moment8_tensor* out = (fdgs_moment8_tensor*)PyBytes_AS_STRING(bytes.p);
    for (Py_ssize_t i = 0; i < n; ++i) {
        const at::Tensor& t = tensor(v.at(i), "values");
        if (t.scalar_type() != type || t.device() != first.device() || !t.is_contiguous())
            value_error("the values of 8-bit moments are contiguous tensors of one type on one device");
        const Moment x = moment8(m.at(i), cls, t.numel(), t.device(), "moments");
        fdgs_moment8_tensor r;
        memset(&r, 0, sizeof(r));
        r.codes = (uint8_t*)x.codes->data_ptr();
        r.exponents = (uint8_t*)x.exps->data_ptr();
        r.value = t.data_ptr();
        r.numel = t.numel();
        r.is_signed = x.is_signed;
        r.round_key = ko == Py_None ? 0u : keys.low32(i);
        out[i] = r;
    }
    return Py_BuildValue("Ni", bytes.give(), type == at::kBFloat16 ? FDGS_TYPE_BF16 : FDGS_TYPE_F32);
}

template <PyObject* (*F)(PyObject*)>
PyObject* guarded(PyObject*, PyObject* args) {
    try {
        return F(args);
    } catch (const Raised&) {
    } catch (const Refused& r) {
        PyErr_SetString(r.type, r.what.c_str());
    } catch (const std::bad_alloc&) {
        PyErr_NoMemory();
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

PyMethodDef methods[] = {
    {"adamw_records", guarded<adamw_records>, METH_VARARGS, "the records of fdgs_adamw_step for lists of tensors"},
    {"moment8_records", guarded<moment8_records>, METH_VARARGS, "the records of fdgs_moment8_pack / unpack for lists of tensors"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "argument records of libfdgs's list calls", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
