// fdgs._host: the calls over lists of tensors from the lists on, and the table lookup with its autograd function.
//
// A step over 200 tensors looks at 1400 tensors' types, sizes, layouts, devices and addresses.  From Python each look
// costs 0.1 to 0.4 us, 5 to 7 us a tensor, several times what the GPU needs for the step; here the whole list costs
// 0.1 to 0.2 us a tensor.  Every check raises the Python exception that a caller sees.
// The lookup of one token takes the GPU 4 us; its checks, output and call take 12 from Python, its training pass 130.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <algorithm>
#include <cstring>
#include <memory>
#include <stdexcept>
#include <string>
#include <unordered_set>
#include <vector>
#include "fdgs.h"

namespace {

// (A standard exception, so that one that leaves a backward pass is autograd's to report.)
struct Refused : std::exception {
    PyObject* type;
    std::string text;
    Refused(PyObject* t, std::string s) : type(t), text(std::move(s)) {}
    const char* what() const noexcept override { return text.c_str(); }
};
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

// The memory that a call writes, and what it reads beside: a piece that is written and another one that overlaps it would be touched by
// workgroups that do not wait for each other.  The pieces of a list of tensors often lie in the list's order, so that the lists only need
// merging (a step over 211 tensors with 8-bit moments looks at 1266 pieces).
struct Touched {
    struct Piece { uintptr_t at, end; size_t rows; };                    // rows: 0, or 1 + its place in that list
    struct Rows { size_t row, step; };                                   // only rows of `row` bytes, `step` apart, are read of a piece
    const int written, lists;                                            // the first `written` lists are written
    const size_t n;
    std::unique_ptr<Piece[]> pieces;                                     // [lists][n]
    size_t count[8] = {};
    std::vector<Rows> rows;
    Touched(int w, int r, size_t each) : written(w), lists(w + r), n(each), pieces(new Piece[(w + r) * each]) {}
    void add(int list, const void* p, size_t bytes, size_t in_rows = 0) {
        if (bytes) pieces[list * n + count[list]++] = {(uintptr_t)p, (uintptr_t)p + bytes, in_rows};
    }
    void add_rows(int list, const void* p, size_t number, size_t row, size_t step) {
        rows.push_back({row, step});
        add(list, p, (number - 1) * step + row, rows.size());
    }
    bool meet(const Piece& w, const Piece& o) const {
        if (o.at >= w.end || w.at >= o.end || o.rows == 0) return o.at < w.end && w.at < o.end;
        // the first row that ends behind w's beginning: does it begin before w's end?
        const Rows r = rows[o.rows - 1];
        const size_t k = w.at < o.at + r.row ? 0 : (w.at - o.at - r.row) / r.step + 1;
        return o.at + k * r.step < std::min(w.end, o.end);
    }
    void check() {
        for (int l = 0; l < lists; ++l) {
            Piece *first = &pieces[l * n], *last = first + count[l];
            const auto less = [](const Piece& a, const Piece& b) { return a.at < b.at; };
            if (!std::is_sorted(first, last, less)) std::sort(first, last, less);
        }
        const Piece none = {UINTPTR_MAX, UINTPTR_MAX, 0}, *head[8], *stop[8];
        uintptr_t next[8], end_written = 0, end = 0;
        for (int l = 0; l < lists; ++l) {
            head[l] = &pieces[l * n];
            stop[l] = head[l] + count[l];
            next[l] = count[l] ? head[l]->at : none.at;
        }
        for (bool apart = true; apart;) {
            int l = 0;                               // the list that goes on, and where another one does
            uintptr_t limit = none.at;
            for (int k = 1; k < lists; ++k) {
                limit = std::min(limit, std::max(next[k], next[l]));
                l = next[k] < next[l] ? k : l;
            }
            if (next[l] == none.at) return;
            const Piece* p = head[l];
            do {
                apart = p->at >= (l < written ? end : end_written);
                end = std::max(end, p->end);
                if (l < written) end_written = std::max(end_written, p->end);
            } while (apart && ++p != stop[l] && p->at <= limit);
            head[l] = p;
            next[l] = p != stop[l] ? p->at : none.at;
        }
        for (int l = 0; l < written; ++l)            // two pieces' spans overlap: also what lies in them?
            for (size_t i = 0; i < count[l]; ++i)
                for (int k = l; k < lists; ++k)
                    for (size_t j = k == l ? i + 1 : 0; j < count[k]; ++j)
                        if (meet(pieces[l * n + i], pieces[k * n + j]))
                            value_error(k < written ? "a tensor is in the lists twice, or two of them overlap" : "what a call reads and what it writes must not overlap");
    }
};

std::string name_of(const at::Tensor& t) { return std::string("torch.") + (t.scalar_type() == at::kFloat ? "float32" : t.scalar_type() == at::kBFloat16 ? "bfloat16" : c10::toString(t.scalar_type())); }

// In memory as it reads: elements one after another, and not a view whose negation is still to be done.
bool plain(const at::Tensor& t) { return t.is_contiguous() && !t.is_neg(); }

// Whether element i of the one is element i of the other, both contiguous: the shapes are equal, or one of them is flat.
bool same_order(at::IntArrayRef a, at::IntArrayRef b) { return a.size() <= 1 || b.size() <= 1 || a == b; }

struct Moment { const at::Tensor *codes, *exps; bool is_signed; };

bool is_moment(PyObject* o, PyObject* cls) { return (PyObject*)Py_TYPE(o) == cls || PyObject_IsInstance(o, cls) == 1; }

// of a tensor `like`: its parameter, or its values
Moment moment8(PyObject* o, PyObject* cls, const at::Tensor& like, const std::string& what) {
    const int64_t numel = like.numel();
    if (!is_moment(o, cls)) value_error(what + ": an 8-bit moment is an adamw.Moment8; do not mix moments in 8 and in 32 bits");
    const at::Tensor &c = tensor(PyTuple_GET_ITEM(o, 0), "codes"), &e = tensor(PyTuple_GET_ITEM(o, 1), "exponents");
    const int truth = PyObject_IsTrue(PyTuple_GET_ITEM(o, 2));
    if (truth < 0) throw Raised();
    if (c.scalar_type() != at::kByte || e.scalar_type() != at::kByte || !plain(c) || !plain(e))
        value_error(what + ": codes and exponents are contiguous uint8 tensors");
    if (c.numel() != numel || e.numel() != (numel + FDGS_MOMENT8_BLOCK - 1) / FDGS_MOMENT8_BLOCK)
        value_error(what + ": one code per element, one exponent per " + std::to_string(FDGS_MOMENT8_BLOCK) + " elements");
    if (!same_order(c.sizes(), like.sizes())) value_error(what + ": codes have the shape of the tensor they belong to, or are flat");
    if (c.device() != like.device() || e.device() != like.device()) value_error(what + ": every tensor of a call is on one device");
    return {&c, &e, truth != 0};
}

// Written in place: a graph that has saved the tensor is to notice, as after torch's own operations.
void changed(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void on_gpu(const at::Tensor& t) {
    if (!t.is_cuda()) throw Refused{PyExc_RuntimeError, "libfdgs kernels run on the GPU only; got a tensor on " + t.device().str()};
}

using at::Tensor;

// The library that fdgs._lib has loaded (its functions' addresses), and that module: where its PROFILE is set every call
// goes through its call_address(), which brackets it with events.
struct Library {
    int (*fwd)(const fdgs_embedding_fwd_args*, void*) = nullptr;
    size_t (*ws)(int64_t, int32_t, int32_t, int32_t) = nullptr;
    int (*bwd)(const fdgs_embedding_bwd_args*, void*) = nullptr;
    int (*adamw)(const fdgs_adamw_args*, void*) = nullptr;
    int (*unpack8)(const fdgs_moment8_args*, void*) = nullptr;
    int (*pack8)(const fdgs_moment8_args*, void*) = nullptr;
    const char* (*strerror)(int) = nullptr;
    size_t (*adamw_ws)(int32_t) = nullptr;
    size_t (*moment8_ws)(int32_t) = nullptr;
    size_t (*sort_ws)(int64_t) = nullptr;
    PyObject* module = nullptr;
} library;

template <class Args>
void launch(const char* name, int (*fn)(const Args*, void*), const Args& a, const at::Device& device) {
    const c10::DeviceGuard guard(device);
    {
        const PyGILState_STATE gil = PyGILState_Ensure();
        PyObject* on = PyObject_GetAttrString(library.module, "PROFILE");
        const bool profiled = on && on != Py_None;
        Py_XDECREF(on);
        PyObject* r = nullptr;
        if (profiled) r = PyObject_CallMethod(library.module, "call_address", "sK", name, (unsigned long long)(uintptr_t)&a);
        const bool failed = profiled && !r;
        Py_XDECREF(r);
        python_error raised;
        if (failed) raised.persist();
        PyGILState_Release(gil);
        if (failed) throw std::move(raised);
        if (profiled) return;
    }
    const int rc = fn(&a, (void*)c10::hip::getCurrentHIPStream(device.index()).stream());
    if (rc != FDGS_OK) throw std::runtime_error(std::string(name) + ": " + library.strerror(rc) + " (" + std::to_string(rc) + ")");
}

// adamw_step(params, grads, exp_avgs, exp_avg_sqs, residuals | None, steps, lr, weight_decay, keys | None, Moment8,
//            beta1, beta2, eps)
PyObject* adamw_step(PyObject* a) {
    PyObject *po, *go, *mo, *vo, *ro, *so, *lo, *wo, *ko, *cls;
    double beta1, beta2, eps;
    if (!PyArg_ParseTuple(a, "OOOOOOOOOOddd", &po, &go, &mo, &vo, &ro, &so, &lo, &wo, &ko, &cls, &beta1, &beta2, &eps)) throw Raised();
    List p(po), g(go), m(mo), v(vo);
    const Py_ssize_t n = p.size();
    if (g.size() != n || m.size() != n || v.size() != n) value_error("params, grads and moments have to be lists of the same length");
    if (n == 0) Py_RETURN_NONE;
    const Each steps(so, n, "steps"), lr(lo, n, "lr"), wd(wo, n, "weight_decay");
    const at::Tensor& first = tensor(p.at(0), "params");
    const at::ScalarType type = first.scalar_type();
    const at::Device device = first.device();
    const bool bf16 = type == at::kBFloat16;
    if (!bf16 && type != at::kFloat) value_error("adamw_step takes float32 and bfloat16 parameters, not " + name_of(first));
    on_gpu(first);
    const c10::DeviceGuard guard(device);
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None)
        throw Refused{PyExc_RuntimeError, "adamw_step reads its step counts on the host and cannot be captured into a graph"};
    Ref rseq(ro == Py_None ? PyTuple_New(0) : PySequence_Fast(ro, "residuals: a list of tensors is needed"));
    if (bf16 && PySequence_Fast_GET_SIZE(rseq.p) != n) value_error("bfloat16 parameters need residuals: an int16 tensor for each");
    const bool eight = is_moment(m.at(0), cls);
    if (eight && (ko == Py_None || !(PyList_Check(ko) || PyTuple_Check(ko)) || PySequence_Fast_GET_SIZE(ko) != n))
        value_error("8-bit moments need keys: a number for each tensor, others at every step");
    std::vector<Tensor> hold;                        // copies of gradients, kept until the kernels are on the stream
    std::vector<fdgs_adamw_tensor> out(n);
    const int P = 0, M = 1, V = 2, LOW = 3, ME = bf16 ? 4 : 3, VE = ME + 1, G = eight ? VE + 1 : ME;    // the gradients behind what is written
    Touched touched(G, 1, n);
    for (Py_ssize_t i = 0; i < n; ++i) {
        const at::Tensor &pt = tensor(p.at(i), "params"), &gt = tensor(g.at(i), "grads");
        const int64_t numel = pt.numel();
        const at::IntArrayRef shape = pt.sizes();
        fdgs_adamw_tensor r;
        memset(&r, 0, sizeof(r));
        if (pt.scalar_type() != type || gt.scalar_type() != type)
            value_error("parameters and gradients of one step have one type: " + name_of(first) + ", " + name_of(pt) + " and " + name_of(gt) + " given");
        if (gt.sizes() != shape || !plain(pt)) value_error("a parameter has to be contiguous, and its gradient of its size and shape");
        if (pt.device() != device || gt.device() != device) value_error("every tensor of a call is on one device");
        r.grad = gt.data_ptr();
        if (!plain(gt)) {
            // rows that are contiguous runs a constant distance apart are read in place
            int64_t len = 1;
            bool rows = !gt.is_neg() && gt.dim() >= 2 && gt.size(0) > 0 && gt.stride(0) > 0;
            for (int64_t d = gt.dim() - 1; rows && d >= 1; --d) {
                if (gt.size(d) != 1 && gt.stride(d) != len) rows = false;
                len *= gt.size(d);
            }
            if (rows && len > 0 && gt.stride(0) >= len && len <= INT32_MAX) {
                r.grad_row_len = (int32_t)len;
                r.grad_row_stride = gt.stride(0);
                const size_t size = bf16 ? 2 : 4;
                touched.add_rows(G, r.grad, gt.size(0), len * size, gt.stride(0) * size);
            } else {
                hold.push_back(gt.detach().resolve_neg().contiguous());
                r.grad = hold.back().data_ptr();
            }
        } else {
            touched.add(G, r.grad, numel * (bf16 ? 2 : 4));
        }
        if (eight) {
            const Moment mm = moment8(m.at(i), cls, pt, "exp_avgs"), vv = moment8(v.at(i), cls, pt, "exp_avg_sqs");
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
                if (x.scalar_type() != at::kFloat || x.numel() != numel || !plain(x) || x.device() != device || !same_order(x.sizes(), shape))
                    value_error("moments are contiguous float32 tensors of the parameter's shape (or flat) on its device, or all of them Moment8");
                (k ? r.exp_avg_sq : r.exp_avg) = x.data_ptr();
            }
        }
        if (bf16) {
            const at::Tensor& x = tensor(PySequence_Fast_GET_ITEM(rseq.p, i), "residuals");
            if (x.scalar_type() != at::kShort || x.numel() != numel || !plain(x) || x.device() != device || !same_order(x.sizes(), shape))
                value_error("a residual is a contiguous int16 tensor of the parameter's shape (or flat) on its device");
            r.residual = (int16_t*)x.data_ptr();
        }
        const long long step = steps.whole(i);
        if (step < 1 || step > INT32_MAX) value_error("steps count from 1");
        r.param = pt.data_ptr();
        r.numel = numel;
        r.step = (int32_t)step;
        r.lr = lr.number(i);
        r.weight_decay = wd.number(i);
        touched.add(P, r.param, numel * (bf16 ? 2 : 4));
        touched.add(M, r.exp_avg, numel * (eight ? 1 : 4));
        touched.add(V, r.exp_avg_sq, numel * (eight ? 1 : 4));
        if (bf16) touched.add(LOW, r.residual, numel * 2);
        if (eight) {
            const int64_t blocks = (numel + FDGS_MOMENT8_BLOCK - 1) / FDGS_MOMENT8_BLOCK;
            touched.add(ME, r.exp_avg_exponents, blocks);
            touched.add(VE, r.exp_avg_sq_exponents, blocks);
        }
        out[i] = r;
    }
    touched.check();
    fdgs_adamw_args args;
    memset(&args, 0, sizeof(args));
    args.num_tensors = (int32_t)n;
    args.param_type = bf16 ? FDGS_TYPE_BF16 : FDGS_TYPE_F32;
    args.state_bits = eight ? 8 : 32;
    args.beta1 = beta1;
    args.beta2 = beta2;
    args.eps = eps;
    args.tensors = out.data();
    args.workspace_bytes = library.adamw_ws(args.num_tensors);
    const Tensor workspace = args.workspace_bytes ? at::empty({(int64_t)args.workspace_bytes}, first.options().dtype(at::kByte).requires_grad(false)) : Tensor();
    args.workspace = args.workspace_bytes ? workspace.data_ptr() : nullptr;
    launch("fdgs_adamw_step", library.adamw, args, device);
    for (Py_ssize_t i = 0; i < n; ++i) changed(THPVariable_Unpack(p.at(i)));     // the state is the optimizer's own
    Py_RETURN_NONE;
}

// moment8(pack, moments, values, keys | None, Moment8): values -> moments (to the nearest without keys), or back
PyObject* moment8_convert(PyObject* a) {
    PyObject *mo, *vo, *ko, *cls;
    int pack;
    if (!PyArg_ParseTuple(a, "pOOOO", &pack, &mo, &vo, &ko, &cls)) throw Raised();
    List m(mo), v(vo);
    const Py_ssize_t n = m.size();
    if (n == 0 || v.size() != n) value_error("a tensor of values is needed for each moment");
    const Each keys(ko, n, "keys");
    const at::Tensor& first = tensor(v.at(0), "values");
    const at::ScalarType type = first.scalar_type();
    if (type != at::kFloat && type != at::kBFloat16) value_error("the values of 8-bit moments are float32 or bfloat16");
    on_gpu(first);
    std::vector<fdgs_moment8_tensor> out(n);
    const int V = pack ? 2 : 0, C = pack ? 0 : 1, E = C + 1;             // values, codes, exponents: what is written first
    Touched touched(pack ? 2 : 1, pack ? 1 : 2, n);
    for (Py_ssize_t i = 0; i < n; ++i) {
        const at::Tensor& t = tensor(v.at(i), "values");
        if (t.scalar_type() != type || t.device() != first.device() || !plain(t))
            value_error("the values of 8-bit moments are contiguous tensors of one type on one device");
        const Moment x = moment8(m.at(i), cls, t, "moments");
        fdgs_moment8_tensor r;
        memset(&r, 0, sizeof(r));
        r.codes = (uint8_t*)x.codes->data_ptr();
        r.exponents = (uint8_t*)x.exps->data_ptr();
        r.value = t.data_ptr();
        r.numel = t.numel();
        r.is_signed = x.is_signed;
        r.round_key = ko == Py_None ? 0u : keys.low32(i);
        touched.add(V, r.value, r.numel * t.element_size());
        touched.add(C, r.codes, r.numel);
        touched.add(E, r.exponents, (r.numel + FDGS_MOMENT8_BLOCK - 1) / FDGS_MOMENT8_BLOCK);
        out[i] = r;
    }
    touched.check();
    fdgs_moment8_args args;
    memset(&args, 0, sizeof(args));
    args.num_tensors = (int32_t)n;
    args.value_type = type == at::kBFloat16 ? FDGS_TYPE_BF16 : FDGS_TYPE_F32;
    args.nearest = ko == Py_None;
    args.tensors = out.data();
    const c10::DeviceGuard guard(first.device());
    args.workspace_bytes = library.moment8_ws(args.num_tensors);
    const Tensor workspace = args.workspace_bytes ? at::empty({(int64_t)args.workspace_bytes}, first.options().dtype(at::kByte)) : Tensor();
    args.workspace = args.workspace_bytes ? workspace.data_ptr() : nullptr;
    launch(pack ? "fdgs_moment8_pack" : "fdgs_moment8_unpack", pack ? library.pack8 : library.unpack8, args, first.device());
    for (Py_ssize_t i = 0; i < n && !pack; ++i) changed(THPVariable_Unpack(v.at(i)));
    Py_RETURN_NONE;
}

// ---- the table lookup ----
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int type_of(const Tensor& t, const char* what) {
    switch (t.scalar_type()) {
        case at::kFloat: return FDGS_TYPE_F32;
        case at::kBFloat16: return FDGS_TYPE_BF16;
        case at::kHalf: return FDGS_TYPE_F16;
        default: value_error(std::string(what) + " is float32, bfloat16 or float16");
    }
}

Tensor ids_of(const Tensor& ids, const at::Device& device) {
    if (ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong) value_error("ids are int32 or int64");
    if (ids.device() != device) value_error("ids and table have to be on one device");
    return (ids.is_neg() ? ids.resolve_neg() : ids).contiguous();
}

// t [lead..., row...] with rows that are contiguous runs a constant, not negative distance apart: t itself where it is
// laid out so, else a copy.
Tensor rows_of(const Tensor& t0, int64_t lead, int64_t& width, int64_t& stride) {
    const Tensor t = t0.is_neg() ? t0.resolve_neg() : t0;
    width = 1;
    for (int64_t d = lead; d < t.dim(); ++d) width *= t.size(d);
    stride = width;
    if (t.is_contiguous()) return t;
    int64_t run = 1;
    bool ok = true;
    for (int64_t d = t.dim() - 1; ok && d >= lead; --d) {
        ok = t.size(d) == 1 || t.stride(d) == run;
        run *= t.size(d);
    }
    int64_t step = -1, span = 0;                     // of the leading dimensions, those of one element left out
    for (int64_t d = lead - 1; ok && d >= 0; --d) {
        if (t.size(d) == 1) continue;
        if (step < 0) step = t.stride(d);
        else ok = t.stride(d) == span;
        span = t.stride(d) * t.size(d);
    }
    if (!ok) return t.contiguous();
    stride = step < 0 ? width : step;
    return t;
}

// What leaves here carries no tangent, so a tensor that has one is refused.
void no_tangent(const Tensor& t, const char* what) {
    if (t._fw_grad(/*level=*/0).defined()) throw Refused{PyExc_NotImplementedError, std::string(what) + " has a forward-mode derivative, which embedding() does not carry on"};
}

// sorted: where it is given, it is set to the tokens by row, which spare the gradient its sort (undefined where there is
// nothing to sort).
Tensor lookup(const Tensor& ids0, const Tensor& table0, double scale, int64_t padding, Tensor* sorted = nullptr) {
    const int type = type_of(table0, "the table");
    no_tangent(table0, "the table");
    const Tensor ids = ids_of(ids0, table0.device());
    int64_t width, stride;
    const Tensor table = rows_of(table0, 1, width, stride);
    if (table.size(0) > INT32_MAX || width > INT32_MAX) value_error("the table has at most 2^31 - 1 rows and columns");
    std::vector<int64_t> shape(ids.sizes().begin(), ids.sizes().end());
    shape.insert(shape.end(), table.sizes().begin() + 1, table.sizes().end());
    Tensor out = at::empty(shape, table.options());
    fdgs_embedding_fwd_args a;
    memset(&a, 0, sizeof(a));
    a.num_tokens = ids.numel();
    a.num_rows = (int32_t)table.size(0);
    a.dim = (int32_t)width;
    a.type = type;
    a.id_bytes = (int32_t)ids.element_size();
    a.ids = ids.data_ptr();
    a.table = table.data_ptr();
    a.table_row_stride = stride;
    a.padding_id = padding;
    a.out = out.data_ptr();
    a.scale = (float)scale;
    Tensor workspace;
    if (sorted && a.num_tokens > FDGS_EMBEDDING_FEW && a.num_tokens <= FDGS_EMBEDDING_MAX_TOKENS && a.num_rows > 0 && width > 0) {
        const auto bytes = table.options().dtype(at::kByte).requires_grad(false);
        *sorted = at::empty({8 * a.num_tokens}, bytes);
        a.workspace_bytes = library.sort_ws(a.num_tokens);
        if (a.workspace_bytes) workspace = at::empty({(int64_t)a.workspace_bytes}, bytes);
        a.sorted = sorted->data_ptr();
        a.workspace = a.workspace_bytes ? workspace.data_ptr() : nullptr;
    }
    launch("fdgs_embedding_fwd", library.fwd, a, table.device());
    return out;
}

Tensor table_grad(const Tensor& grad_out0, const Tensor& ids0, int64_t rows, double scale, int64_t padding, const Tensor& sorted = Tensor()) {
    no_tangent(grad_out0, "grad_out");
    on_gpu(grad_out0);
    const int type = type_of(grad_out0, "grad_out");
    const Tensor ids = ids_of(ids0, grad_out0.device());
    int64_t lead = ids.dim();
    if (grad_out0.dim() <= lead || grad_out0.sizes().slice(0, lead) != ids.sizes()) value_error("grad_out has to be [*ids.shape, ...]");
    if (rows < 0 || rows > INT32_MAX) value_error("num_rows is between 0 and 2^31 - 1");
    if (sorted.defined() && sorted.numel() != 8 * ids.numel()) value_error("ids have another size than in the lookup");
    std::vector<int64_t> shape{rows};
    shape.insert(shape.end(), grad_out0.sizes().begin() + lead, grad_out0.sizes().end());
    Tensor view = grad_out0;
    if (lead == 0) {
        view = grad_out0.unsqueeze(0);
        lead = 1;
    }
    int64_t width, stride;
    const Tensor g = rows_of(view, lead, width, stride);
    if (width > INT32_MAX) value_error("a row has at most 2^31 - 1 columns");
    Tensor out = at::empty(shape, g.options());
    if (rows == 0 || width == 0) return out;
    fdgs_embedding_bwd_args a;
    memset(&a, 0, sizeof(a));
    const size_t bytes = library.ws(ids.numel(), (int32_t)rows, (int32_t)width, type);
    const Tensor workspace = at::empty({(int64_t)bytes}, g.options().dtype(at::kByte));
    a.num_tokens = ids.numel();
    a.num_rows = (int32_t)rows;
    a.dim = (int32_t)width;
    a.type = type;
    a.id_bytes = (int32_t)ids.element_size();
    a.ids = ids.data_ptr();
    a.grad_out = g.data_ptr();
    a.grad_out_row_stride = stride;
    a.padding_id = padding;
    a.grad_table = out.data_ptr();
    a.scale = (float)scale;
    a.sorted = sorted.defined() ? sorted.data_ptr() : nullptr;
    a.workspace = workspace.data_ptr();
    a.workspace_bytes = bytes;
    launch("fdgs_embedding_bwd", library.bwd, a, g.device());
    return out;
}

// The lookup is linear in the table and its gradient linear in grad_out, each the other's transpose: two functions that
// are each other's backward pass, to any order.
struct Lookup : torch::autograd::Function<Lookup> {
    static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& ids, double scale, int64_t padding);
    static variable_list backward(AutogradContext* ctx, variable_list grads);
};
struct Sorted { Tensor pairs; };                      // not one of a function's inputs; undefined: not sorted yet
struct TableGrad : torch::autograd::Function<TableGrad> {
    static Tensor forward(AutogradContext* ctx, const Tensor& grad_out, const Tensor& ids, const Sorted& sorted, int64_t rows, double scale, int64_t padding);
    static variable_list backward(AutogradContext* ctx, variable_list grads);
};

Tensor Lookup::forward(AutogradContext* ctx, const Tensor& table, const Tensor& ids, double scale, int64_t padding) {
    Tensor sorted;
    const Tensor out = lookup(ids, table, scale, padding, &sorted);
    ctx->save_for_backward({ids, sorted});
    ctx->saved_data["rows"] = table.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return out;
}
variable_list Lookup::backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &ids = saved[0], &sorted = saved[1];
    const int64_t rows = ctx->saved_data["rows"].toInt(), padding = ctx->saved_data["padding"].toInt();
    const double scale = ctx->saved_data["scale"].toDouble();
    const bool graph = at::GradMode::is_enabled() && grads[0].requires_grad();
    return {graph ? TableGrad::apply(grads[0], ids, Sorted{sorted}, rows, scale, padding) : table_grad(grads[0], ids, rows, scale, padding, sorted),
            Tensor(), Tensor(), Tensor()};
}
Tensor TableGrad::forward(AutogradContext* ctx, const Tensor& grad_out, const Tensor& ids, const Sorted& sorted, int64_t rows, double scale, int64_t padding) {
    ctx->save_for_backward({ids});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return table_grad(grad_out, ids, rows, scale, padding, sorted.pairs);
}
variable_list TableGrad::backward(AutogradContext* ctx, variable_list grads) {
    const Tensor ids = ctx->get_saved_variables()[0];
    const int64_t padding = ctx->saved_data["padding"].toInt();
    const double scale = ctx->saved_data["scale"].toDouble();
    const bool graph = at::GradMode::is_enabled() && grads[0].requires_grad();
    return {graph ? Lookup::apply(grads[0], ids, scale, padding) : lookup(ids, grads[0], scale, padding), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
}

int64_t padding_of(PyObject* o) {
    if (o == Py_None) return -1;
    Ref n(PyNumber_Index(o));
    const long long v = PyLong_AsLongLong(n.p);
    if (v == -1 && PyErr_Occurred()) throw Raised();
    if (v < 0) value_error("padding_id is a row of the table; negative ids are padding always");
    return v;
}

// A backward pass that is captured while a graph of the same leaf made on another stream lives waits for that stream, from
// autograd's own thread, where the error that the capture makes of it ends the process.  Refused here, where it can be: the
// leaves that the table was made of are looked up, while a capture runs.
void capture_alone(const Tensor& table) {
    const c10::DeviceGuard guard(table.device());
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    const auto stream = c10::hip::getCurrentHIPStream(table.device().index());
    std::vector<torch::autograd::Node*> next;
    std::unordered_set<torch::autograd::Node*> seen;
    const auto of_leaf = table.is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(table) : nullptr;
    if (of_leaf) next.push_back(of_leaf.get());
    if (!table.is_leaf()) next.push_back(table.grad_fn().get());
    while (!next.empty()) {
        torch::autograd::Node* node = next.back();
        next.pop_back();
        if (!seen.insert(node).second) continue;
        if (dynamic_cast<torch::autograd::AccumulateGrad*>(node)) {
            const auto made_on = node->stream();
            if (!made_on.has_value() || made_on->id() != stream.id())
                throw Refused{PyExc_RuntimeError, "embedding: an autograd graph of this table from outside the capture is alive; delete "
                                                  "its outputs before capturing a pass that wants gradients"};
        }
        for (const auto& e : node->next_edges())
            if (e.function) next.push_back(e.function.get());
    }
}

// A tensor here would lose its gradient without a word.
double scale_of(PyObject* o) {
    if (THPVariable_Check(o)) throw Refused{PyExc_TypeError, "scale is a number, not a tensor: it gets no gradient"};
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised();
    return v;
}

// embedding(ids, table, scale, padding_id | None)
PyObject* embedding(PyObject* a) {
    PyObject *io, *to, *so, *po;
    if (!PyArg_ParseTuple(a, "OOOO", &io, &to, &so, &po)) throw Raised();
    const double scale = scale_of(so);
    const Tensor &ids = tensor(io, "ids"), &table = tensor(to, "the table");
    if (table.dim() < 2) value_error("the table is [rows, ...] in float32, bfloat16 or float16");
    type_of(table, "the table");
    if (!table.is_cuda()) no_tangent(table, "the table");                // (lookup() looks at the others)
    on_gpu(table);
    const int64_t padding = padding_of(po);
    Tensor out;
    if (table.requires_grad() && at::GradMode::is_enabled()) {
        ids_of(ids, table.device());                 // refused here, as the type that a caller expects
        capture_alone(table);
        out = Lookup::apply(table, ids, scale, padding);
    } else {
        out = lookup(ids, table, scale, padding);
    }
    return THPVariable_Wrap(std::move(out));
}

// embedding_grad(grad_out, ids, num_rows, scale, padding_id | None)
PyObject* embedding_grad(PyObject* a) {
    PyObject *go, *io, *so, *po;
    long long rows;
    if (!PyArg_ParseTuple(a, "OOLOO", &go, &io, &rows, &so, &po)) throw Raised();
    const double scale = scale_of(so);
    const Tensor &g = tensor(go, "grad_out"), &ids = tensor(io, "ids");
    return THPVariable_Wrap(table_grad(g, ids, rows, scale, padding_of(po)));
}

// rows_layout(tensor, lead) -> (read in place, width, stride): what rows_of() makes of a tensor
PyObject* rows_layout(PyObject* a) {
    PyObject* o;
    long long lead;
    if (!PyArg_ParseTuple(a, "OL", &o, &lead)) throw Raised();
    const Tensor& t = tensor(o, "tensor");
    int64_t width, stride;
    const Tensor r = rows_of(t, lead, width, stride);
    return Py_BuildValue("NLL", PyBool_FromLong(r.is_same(t)), (long long)width, (long long)stride);
}

// bind(module, addresses of fdgs_embedding_fwd, _bwd_workspace_bytes, _bwd, fdgs_adamw_step, fdgs_moment8_unpack, _pack,
// fdgs_strerror, fdgs_adamw_workspace_bytes, fdgs_moment8_workspace_bytes, fdgs_embedding_sort_workspace_bytes)
PyObject* bind(PyObject* a) {
    unsigned long long fwd, ws, bwd, adamw, unpack, pack, err, adamw_ws, moment8_ws, sort_ws;
    PyObject* module;
    if (!PyArg_ParseTuple(a, "OKKKKKKKKKK", &module, &fwd, &ws, &bwd, &adamw, &unpack, &pack, &err, &adamw_ws, &moment8_ws, &sort_ws)) throw Raised();
    Py_INCREF(module);
    Py_XDECREF(library.module);
    library.module = module;
    library.fwd = (decltype(library.fwd))(uintptr_t)fwd;
    library.ws = (decltype(library.ws))(uintptr_t)ws;
    library.bwd = (decltype(library.bwd))(uintptr_t)bwd;
    library.adamw = (decltype(library.adamw))(uintptr_t)adamw;
    library.unpack8 = (decltype(library.unpack8))(uintptr_t)unpack;
    library.pack8 = (decltype(library.pack8))(uintptr_t)pack;
    library.strerror = (decltype(library.strerror))(uintptr_t)err;
    library.adamw_ws = (decltype(library.adamw_ws))(uintptr_t)adamw_ws;
    library.moment8_ws = (decltype(library.moment8_ws))(uintptr_t)moment8_ws;
    library.sort_ws = (decltype(library.sort_ws))(uintptr_t)sort_ws;
    Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*)>
PyObject* guarded(PyObject*, PyObject* args) {
    try {
        return F(args);
    } catch (const Raised&) {
    } catch (const Refused& r) {
        PyErr_SetString(r.type, r.what());
    } catch (python_error& e) {                      // out of a hook that autograd has called: it stays what it is
        e.restore();
    } catch (const std::bad_alloc&) {
        PyErr_NoMemory();
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

PyMethodDef methods[] = {
    {"adamw_step", guarded<adamw_step>, METH_VARARGS, "fdgs_adamw_step for lists of tensors"},
    {"moment8", guarded<moment8_convert>, METH_VARARGS, "fdgs_moment8_pack / unpack for lists of tensors"},
    {"embedding", guarded<embedding>, METH_VARARGS, "the table lookup, with its gradient where the table wants one"},
    {"embedding_grad", guarded<embedding_grad>, METH_VARARGS, "the gradient of the table alone"},
    {"rows_layout", guarded<rows_layout>, METH_VARARGS, "how the rows of a tensor are read"},
    {"bind", guarded<bind>, METH_VARARGS, "the library's entry points"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "host work of libfdgs's calls over lists of tensors and tables", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
