// The Python package's calls in native code: `nuvec_amd._native`.
//
// A decode step is launch-bound: its kernels take 3 to 20 us each, and the argument checks, descriptors and allocations of
// one call took 12 to 17 us in Python (a one-row product of W[1024,4096]: 16.7 us per call, of which the kernel is 3.4).  Here
// the same work is done on the tensors' own C++ objects, a block's layers in one call.
//
// Every function takes the plain case alone: operands on the bound device, dense, of one element type, of matching shapes, and
// layers whose methods are the package's own.  Whatever else it meets (and whatever the library refuses) it declines by returning
// None, and the caller's Python path, which holds every conversion and the reference's messages, does the call.  The operands of
// every product of a block are looked at before the first is launched; where the library itself refuses a later one, what ran
// before it has written intermediate tensors that are dropped.
//
// The interpreter lock is released while a call allocates and launches, as ctypes and torch's own operators release it.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ExpandUtils.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/core/Tensor.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>

#include <atomic>
#include <vector>

#include "nuvec_hip.h"

namespace {

using at::Tensor;

// ── reading Python objects ──────────────────────────────────────────────────────────────────────────────────────────
struct Names {
    PyObject *mode, *group_size, *bits, *weight, *scales, *biases, *bias, *quant, *global_scale;
    PyObject *gate_proj, *up_proj, *down_proj, *gate_up_proj, *geglu;
    PyObject *keys, *values, *table, *interleaved, *axes, *down, *up;
    PyObject *gate, *switch_mlp, *experts_per_token, *norm_topk_prob, *gate_up_paired, *activation, *alpha, *limit;
} names;

std::atomic<uint64_t> ready_devices{0};  // devices nvq_init has answered for (ops._init)

struct Ref {
    PyObject *p;
    explicit Ref(PyObject *o) : p(o) {}
    Ref(const Ref &) = delete;
    ~Ref() { Py_XDECREF(p); }
};

bool declined() {
    PyErr_Clear();
    return false;
}

// A class of `layers` and the methods of it that a call here stands in for.  An object is plain if it is of that very class
// (a subclass may have others), the class still holds the functions it was defined with, and the object has none of its own.
struct Kind {
    PyTypeObject *type = nullptr;
    std::vector<std::pair<PyObject *, PyObject *>> methods;  // name, function

    bool plain(PyObject *o) const {
        if (type == nullptr || Py_TYPE(o) != type) return false;
        PyObject **own = _PyObject_GetDictPtr(o);
        for (const auto &m : methods) {
            if (PyDict_GetItemWithError(type->tp_dict, m.first) != m.second) return declined();
            if (own != nullptr && *own != nullptr && PyDict_GetItemWithError(*own, m.first) != nullptr) return false;
        }
        return true;
    }
};
Kind linear_kind, projection_kind, switch_glu_kind, moe_kind;

bool read_int(PyObject *o, PyObject *name, int32_t &v) {
    Ref a(PyObject_GetAttr(o, name));
    if (a.p == nullptr || !PyLong_Check(a.p)) return declined();
    const long n = PyLong_AsLong(a.p);
    if (n == -1 && PyErr_Occurred()) return declined();
    v = (int32_t)n;
    return true;
}

bool read_quant(PyObject *o, nvq_quant &q) {
    return read_int(o, names.mode, q.mode) && read_int(o, names.group_size, q.group_size) && read_int(o, names.bits, q.bits);
}

bool read_float(PyObject *o, PyObject *name, float &v) {
    Ref a(PyObject_GetAttr(o, name));
    if (a.p == nullptr) return declined();
    const double d = PyFloat_AsDouble(a.p);
    if (d == -1.0 && PyErr_Occurred()) return declined();
    v = (float)d;
    return true;
}

bool read_truth(PyObject *o, PyObject *name, bool &v) {
    Ref a(PyObject_GetAttr(o, name));
    const int t = a.p == nullptr ? -1 : PyObject_IsTrue(a.p);
    if (t < 0) return declined();
    v = t != 0;
    return true;
}

// A tensor, or none at all for None.
bool as_tensor(PyObject *o, Tensor &t) {
    if (o == Py_None) return true;
    if (!THPVariable_Check(o)) return false;
    t = THPVariable_Unpack(o);
    return true;
}
bool read_tensor(PyObject *o, PyObject *name, Tensor &t) {
    Ref a(PyObject_GetAttr(o, name));
    return a.p == nullptr ? declined() : as_tensor(a.p, t);
}

// ── operands ────────────────────────────────────────────────────────────────────────────────────────────────────────
int32_t code_of(at::ScalarType t) {
    switch (t) {
    case at::kHalf: return NVQ_F16;
    case at::kBFloat16: return NVQ_BF16;
    case at::kFloat: return NVQ_F32;
    default: return -1;
    }
}

bool is_word(at::ScalarType t) { return t == at::kUInt32 || t == at::kInt; }

const void *ptr(const Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }

// Whether `t` lies densely on the device that the library is bound to and that is current.
struct Place {
    c10::Device device;
    explicit Place(const Tensor &x) : device(x.defined() ? x.device() : c10::Device(at::kCPU)) {}
    bool usable() const {
        return device.is_cuda() && device.index() >= 0 && device.index() < 64 && (ready_devices >> device.index() & 1) != 0 &&
               c10::hip::current_device() == device.index();
    }
    bool holds(const Tensor &t) const { return t.device() == device && t.is_contiguous(); }
    void *stream() const { return c10::hip::getCurrentHIPStream(device.index()).stream(); }
    Tensor empty(at::IntArrayRef sizes, at::ScalarType type) const {
        return at::detail::empty_cuda(sizes, type, device, std::nullopt);
    }
};

struct Packed {
    Tensor w, s, b;
    nvq_quant q;

    // Codes, scales and biases of `dims` dimensions that go together and with activations of `type` (ops._check_groups,
    // ops._quantized_columns); `columns`: the values of a packed row.
    bool fits(const Place &at, at::ScalarType type, int64_t dims, int64_t &columns) const {
        if (!w.defined() || !s.defined() || !is_word(w.scalar_type()) || w.dim() != dims || s.dim() != dims || !at.holds(w) || !at.holds(s))
            return false;
        if (q.mode == NVQ_AFFINE) {
            if (!b.defined() || s.scalar_type() != type || b.scalar_type() != type || !at.holds(b) || b.sizes() != s.sizes()) return false;
        } else if (b.defined() || s.scalar_type() != at::kByte) {
            return false;
        }
        for (int64_t i = 0; i + 1 < dims; i++)
            if (w.size(i) != s.size(i)) return false;
        columns = s.size(dims - 1) * q.group_size;
        return columns > 0 && w.size(dims - 1) * 32 == columns * q.bits;
    }
};

bool bias_fits(const Tensor &bias, const Place &at, at::ScalarType type, int64_t n) {
    return !bias.defined() || (bias.scalar_type() == type && bias.dim() == 1 && bias.size(0) == n && at.holds(bias));
}

using Sizes = c10::SmallVector<int64_t, 6>;
Sizes with_last(at::IntArrayRef sizes, int64_t last) {
    Sizes s(sizes.begin(), sizes.end());
    s.back() = last;
    return s;
}

// ── the calls ───────────────────────────────────────────────────────────────────────────────────────────────────────
struct Flags {
    bool transpose = true, row_exact = false, rows = false, scratch = true;
};

// ops.quantized_matmul of one weight matrix.
bool product(const Tensor &x, const Packed &p, const Tensor &bias, Flags f, Tensor &out) {
    const Place at(x);
    if (!at.usable() || x.dim() < 2 || !x.is_contiguous() || x.numel() == 0) return false;
    const int32_t code = code_of(x.scalar_type());
    int64_t columns;
    if (code < 0 || !p.fits(at, x.scalar_type(), 2, columns)) return false;
    const int64_t rows = p.w.size(0), inner = f.transpose ? columns : rows, outer = f.transpose ? rows : columns;
    if (x.size(-1) != inner || outer == 0 || !bias_fits(bias, at, x.scalar_type(), outer)) return false;
    nvq_qmm_desc d{};
    d.quant = p.q, d.dtype = code, d.transpose = f.transpose, d.row_exact = f.row_exact, d.rows = f.rows;
    d.m = x.numel() / inner, d.n = outer, d.k = inner, d.item_rows = x.size(-2);
    const size_t need = f.scratch ? nvq_quantized_matmul_workspace_bytes(&d) : 0;
    Tensor workspace, y = at.empty(with_last(x.sizes(), outer), x.scalar_type());
    if (need > 0) workspace = at.empty({(int64_t)need}, at::kByte);
    const int32_t rc = nvq_quantized_linear(&d, ptr(x), ptr(p.w), ptr(p.s), ptr(p.b), ptr(bias), y.mutable_data_ptr(),
                                            need > 0 ? workspace.mutable_data_ptr() : nullptr, at.stream());
    if (rc != NVQ_OK) return false;
    out = std::move(y);
    return true;
}

nvq_qmm_desc gated_desc(const Tensor &x, int32_t code, const nvq_quant &q, int64_t n) {
    nvq_qmm_desc d{};
    d.quant = q, d.dtype = code, d.transpose = 1;
    d.m = x.numel() / x.size(-1), d.n = n, d.k = x.size(-1), d.item_rows = x.dim() > 1 ? x.size(-2) : 1;
    return d;
}

// The kernel of several gated rows that nvq_quantized_matmul_glu_several_takes names, and its workspace.
struct Several {
    int32_t kernel = 0;
    size_t need = 0;
};

// ops.quantized_matmul_glu, or (`several`) ops.quantized_matmul_glu_grouped or ops.quantized_matmul_glu_rows.  `asked`: what the
// question gave for a pair of these sizes, which costs as much as a launch.
bool product_glu(const Tensor &x, const Packed &p, const Tensor &bias, int32_t activation, float alpha, float limit, bool several,
                 const Several *asked, Tensor &out) {
    const Place at(x);
    if (!at.usable() || x.dim() < 1 || !x.is_contiguous() || x.numel() == 0) return false;
    const int32_t code = code_of(x.scalar_type());
    int64_t columns;
    if (code < 0 || !p.fits(at, x.scalar_type(), 2, columns) || x.size(-1) != columns) return false;
    const int64_t n = p.w.size(0);
    if (n == 0 || n % 128 != 0 || !bias_fits(bias, at, x.scalar_type(), n)) return false;
    const nvq_qmm_desc d = gated_desc(x, code, p.q, n);
    Several to;
    if (several && asked != nullptr) to = *asked;
    else if (several) to.kernel = nvq_quantized_matmul_glu_several_takes(&d, &to.need);
    if (several && to.kernel == 0) return false;
    const bool grouped = to.kernel == 1;
    const size_t need = to.need;
    Tensor workspace, y = at.empty(with_last(x.sizes(), n / 2), x.scalar_type());
    if (need > 0) workspace = at.empty({(int64_t)need}, at::kByte);
    const int32_t rc = grouped   ? nvq_quantized_matmul_glu_grouped(&d, activation, alpha, limit, ptr(x), ptr(p.w), ptr(p.s), ptr(p.b), ptr(bias),
                                                                    y.mutable_data_ptr(), at.stream())
                       : several ? nvq_quantized_matmul_glu_rows(&d, activation, alpha, limit, ptr(x), ptr(p.w), ptr(p.s), ptr(p.b), ptr(bias),
                                                               y.mutable_data_ptr(), need > 0 ? workspace.mutable_data_ptr() : nullptr, at.stream())
                               : nvq_quantized_matmul_glu(&d, activation, alpha, limit, ptr(x), ptr(p.w), ptr(p.s), ptr(p.b), ptr(bias),
                                                          y.mutable_data_ptr(), at.stream());
    if (rc != NVQ_OK) return false;
    out = std::move(y);
    return true;
}

struct Activation {
    int32_t code = NVQ_GLU_SWIGLU;
    float alpha = 0.0f, limit = 0.0f;
};

// ops.glu of two dense tensors, without biases.
bool gated(const Tensor &gate, const Tensor &up, int32_t activation, Tensor &out) {
    const Place at(gate);
    const int64_t hidden = gate.size(-1);
    nvq_glu_desc d{code_of(gate.scalar_type()), activation, 0.0f, 0.0f, gate.numel() / hidden, hidden, hidden, hidden, 0};
    Tensor y = at.empty(gate.sizes(), gate.scalar_type());
    if (nvq_glu(&d, ptr(gate), ptr(up), nullptr, nullptr, nullptr, y.mutable_data_ptr(), at.stream()) != NVQ_OK) return false;
    out = std::move(y);
    return true;
}

// ── mixture of experts ──────────────────────────────────────────────────────────────────────────────────────────────
struct Projection {  // layers.SwitchProjection: a packed weight and perhaps a bias per expert
    Packed p;
    Tensor bias;
    int64_t columns = 0, rows = 0;

    bool fits(const Place &at, at::ScalarType type, int64_t experts) {
        if (!p.fits(at, type, 3, columns) || p.w.size(0) != experts) return false;
        rows = p.w.size(1);
        return rows > 0 && (!bias.defined() || (bias.scalar_type() == type && bias.dim() == 2 && bias.size(0) == experts &&
                                                bias.size(1) == rows && at.holds(bias)));
    }
};

// The pairs of a pass: which row of x and which expert each takes, in the order they run.
struct Pairs {
    int64_t count, experts;
    const uint32_t *expert;       // of each pair, in order
    const int32_t *offsets;       // sorted by expert: where each expert's pairs start; NULL: any order
};

// One projection of all pairs (ops.gather_qmm, ops.gather_qmm_grouped): pair z takes row `from[z]` of x [x_rows, columns] and
// writes row `to[z]` (NULL: z).
bool project(const Place &at, const Tensor &x, int64_t x_rows, const Projection &w, const Pairs &pairs, const uint32_t *from, const uint32_t *to,
             bool with_bias, Tensor &out) {
    const nvq_gather_desc d{w.p.q, code_of(x.scalar_type()), 1, 0, 1, 1, w.rows, w.columns, pairs.count, x_rows, pairs.experts};
    Tensor y = at.empty({pairs.count, w.rows}, x.scalar_type());
    if (nvq_gather_qmm_expert_bias(&d, ptr(x), ptr(w.p.w), ptr(w.p.s), ptr(w.p.b), nullptr, from, pairs.expert, pairs.offsets, to,
                                   with_bias ? ptr(w.bias) : nullptr, y.mutable_data_ptr(), nullptr, at.stream()) != NVQ_OK)
        return false;
    out = std::move(y);
    return true;
}

struct Experts {  // layers.SwitchGlu
    Projection gate, up, down, both;
    bool fused = false, paired = false;
    Activation act;
};

// The pairs' gated hidden states (layers.SwitchGlu.forward up to the down projection).
bool hidden_states(const Place &at, const Tensor &x, int64_t x_rows, Experts &e, const Pairs &pairs, const uint32_t *tokens, Tensor &out) {
    const at::ScalarType type = x.scalar_type();
    const int64_t hidden = e.down.columns;
    if (e.fused && e.paired) {
        const nvq_gather_desc d{e.both.p.q, code_of(type), 1, 0, 1, 1, e.both.rows, e.both.columns, pairs.count, x_rows, pairs.experts};
        Tensor y = at.empty({pairs.count, hidden}, type);
        if (nvq_gather_qmm_glu(&d, e.act.code, e.act.alpha, e.act.limit, ptr(x), ptr(e.both.p.w), ptr(e.both.p.s), ptr(e.both.p.b), tokens,
                               pairs.expert, pairs.offsets, ptr(e.both.bias), y.mutable_data_ptr(), at.stream()) == NVQ_OK) {
            out = std::move(y);
            return true;
        }
    }
    // products without their biases, then biases and activation in one pass
    Tensor gate, up;
    int64_t stride = hidden;
    const char *second;
    if (e.fused && !e.paired) {
        if (!project(at, x, x_rows, e.both, pairs, tokens, nullptr, false, gate)) return false;
        stride = 2 * hidden;
        second = (const char *)ptr(gate) + hidden * gate.element_size();
    } else {
        if (!project(at, x, x_rows, e.gate, pairs, tokens, nullptr, false, gate) || !project(at, x, x_rows, e.up, pairs, tokens, nullptr, false, up))
            return false;
        second = (const char *)ptr(up);
    }
    const bool biased = e.gate.bias.defined();
    const nvq_glu_desc d{code_of(type), e.act.code, e.act.alpha, e.act.limit, pairs.count, hidden, stride, stride, biased ? pairs.experts : 0};
    Tensor y = at.empty({pairs.count, hidden}, type);
    if (nvq_glu(&d, ptr(gate), second, ptr(e.gate.bias), ptr(e.up.bias), biased ? (const int32_t *)pairs.expert : nullptr, y.mutable_data_ptr(),
                at.stream()) != NVQ_OK)
        return false;
    out = std::move(y);
    return true;
}

// layers.SwitchGlu._ordered.
bool pairs_ordered(const Experts &e, int32_t code, int64_t tokens, int64_t choices, int64_t experts) {
    if (tokens * choices >= 64) return true;
    const int64_t size = e.up.rows * e.up.columns;
    auto rule = [&](const Projection &w, int64_t values) { return nvq_moe_ordered(&w.p.q, code, tokens, (int32_t)choices, experts, values, 0) != 0; };
    if (!rule(e.up, 3 * size)) return false;
    const Projection *taken[3];
    int count = 0;
    for (const Projection *w : {&e.gate, &e.up, &e.down}) {
        const nvq_gather_desc d{w->p.q, code, 1, 0, 1, 1, w->rows, w->columns, tokens * choices, tokens * choices, experts};
        if (nvq_gather_sorted_takes(&d)) taken[count++] = w;
    }
    for (int i = 0; i < count; i++)
        if (!rule(*taken[i], count * size)) return false;
    return count > 0;
}

// layers.MoeMlp.forward.
bool moe(const Tensor &x, const Tensor &router, int64_t k, bool normalize, Experts &e, Tensor &out) {
    const Place at(x);
    if (!at.usable() || x.dim() != 3 || x.numel() == 0 || !x.is_contiguous()) return false;
    const at::ScalarType type = x.scalar_type();
    const int32_t code = code_of(type);
    if (code < 0 || !router.defined() || router.scalar_type() != type || router.dim() != 2 || !at.holds(router) || router.size(1) != x.size(2))
        return false;
    const int64_t rows = x.size(0) * x.size(1), dims = x.size(2), experts = router.size(0);
    if (k < 1 || k > experts || k >= 32 || dims > INT32_MAX || experts > 1024 || rows > INT32_MAX / k) return false;
    if (!e.gate.fits(at, type, experts) || !e.up.fits(at, type, experts) || !e.down.fits(at, type, experts)) return false;
    const int64_t hidden = e.down.columns;
    if (e.gate.columns != dims || e.up.columns != dims || e.gate.rows != hidden || e.up.rows != hidden ||
        e.gate.bias.defined() != e.up.bias.defined())
        return false;
    if (e.fused && (!e.both.fits(at, type, experts) || e.both.columns != dims || e.both.rows != 2 * hidden ||
                    e.both.bias.defined() != e.gate.bias.defined() || (e.paired && hidden % 64 != 0)))
        return false;

    const int64_t pairs = rows * k;
    void *stream = at.stream();
    // choices, tokens and numbers of the pairs; for ordered pairs the order, its inverse, sorted experts and tokens, the offsets
    const bool ordered = pairs_ordered(e, code, rows, k, experts);
    Tensor index = at.empty({pairs * (ordered ? 7 : 3) + (ordered ? experts : 0)}, at::kInt), scores = at.empty({rows, k}, type);
    uint32_t *chosen = (uint32_t *)index.mutable_data_ptr(), *tokens = chosen + pairs, *identity = tokens + pairs;
    if (nvq_moe_router(code, ptr(x), ptr(router), rows, (int32_t)dims, (int32_t)experts, (int32_t)k, normalize, chosen, scores.mutable_data_ptr(),
                       tokens, identity, stream) != NVQ_OK)
        return false;
    Pairs p{pairs, experts, chosen, nullptr};
    const uint32_t *to = nullptr;
    Tensor workspace, h, y;
    if (ordered) {
        uint32_t *order = identity + pairs, *restore = order + pairs, *sorted = restore + pairs, *sorted_tokens = sorted + pairs;
        int32_t *offsets = (int32_t *)(sorted_tokens + pairs);
        const size_t need = nvq_moe_order_workspace_bytes(pairs, (int32_t)experts);
        if (need > 0) workspace = at.empty({(int64_t)need}, at::kByte);
        if (nvq_moe_order_tokens(chosen, pairs, (int32_t)experts, (int32_t)k, order, restore, sorted, offsets, sorted_tokens,
                                 need > 0 ? workspace.mutable_data_ptr() : nullptr, stream) != NVQ_OK)
            return false;
        p.expert = sorted, p.offsets = offsets;
        tokens = sorted_tokens, to = order;
    }
    if (!hidden_states(at, x, rows, e, p, tokens, h) || e.down.rows == 0) return false;
    Tensor sum = at.empty({x.size(0), x.size(1), e.down.rows}, type);
    if (!ordered) {  // (few tokens: the down products with their sum)
        const nvq_gather_desc d{e.down.p.q, code, 1, 0, 0, 1, e.down.rows, hidden, pairs, pairs, experts};
        if (nvq_gather_qmm_sum_takes(&d, (int32_t)k) &&
            nvq_gather_qmm_sum(&d, ptr(h), ptr(e.down.p.w), ptr(e.down.p.s), ptr(e.down.p.b), nullptr, identity, chosen, ptr(e.down.bias), ptr(scores),
                               (int32_t)k, sum.mutable_data_ptr(), stream) == NVQ_OK) {
            out = std::move(sum);
            return true;
        }
    }
    if (!project(at, h, pairs, e.down, p, identity, to, true, y)) return false;
    if (nvq_weighted_sum(code, ptr(y), ptr(scores), rows, (int32_t)k, e.down.rows, sum.mutable_data_ptr(), stream) != NVQ_OK) return false;
    out = std::move(sum);
    return true;
}

// ── layers ──────────────────────────────────────────────────────────────────────────────────────────────────────────
struct Linear {
    Packed p;
    Tensor bias;
};
bool read_linear(PyObject *o, Linear &l) {
    if (!linear_kind.plain(o)) return false;
    if (!read_tensor(o, names.weight, l.p.w) || !read_tensor(o, names.scales, l.p.s) || !read_tensor(o, names.biases, l.p.b) ||
        !read_tensor(o, names.bias, l.bias))
        return false;
    Ref q(PyObject_GetAttr(o, names.quant));
    return q.p == nullptr ? declined() : read_quant(q.p, l.p.q);
}
bool read_linear(PyObject *o, PyObject *name, Linear &l) {
    Ref a(PyObject_GetAttr(o, name));
    return a.p == nullptr ? declined() : read_linear(a.p, l);
}

PyObject *none() { Py_RETURN_NONE; }

// A refusal inside torch (no memory left) is Python's exception, as it is where Python allocates.
template <typename F>
PyObject *guarded(F &&f) {
    try {
        return f();
    } catch (...) {  // (torch.OutOfMemoryError among them)
        torch::translate_exception_to_python(std::current_exception());
        return nullptr;
    }
}

// `f`, which touches no Python object, without the interpreter lock.
struct Unlocked {
    PyThreadState *state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
};
template <typename F>
bool unlocked(F &&f) {
    const Unlocked here;
    return f();
}

PyObject *wrap(bool done, Tensor &y) { return done ? THPVariable_Wrap(std::move(y)) : none(); }

// linear(layer, x)
PyObject *py_linear(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        Tensor x, y;
        Linear l;
        if (n != 2 || !as_tensor(args[1], x) || !read_linear(args[0], l)) return none();
        return wrap(unlocked([&] { return product(x, l.p, l.bias, Flags(), y); }), y);
    });
}

// quantized_matmul(x, weight, scales, biases, quant, transpose, row_exact, rows, scratch, bias)
PyObject *py_quantized_matmul(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        Tensor x, bias, y;
        Packed p;
        if (n != 10 || !as_tensor(args[0], x) || !as_tensor(args[1], p.w) || !as_tensor(args[2], p.s) || !as_tensor(args[3], p.b) ||
            !read_quant(args[4], p.q) || !as_tensor(args[9], bias))
            return none();
        int flag[4];
        for (int i = 0; i < 4; i++)
            if ((flag[i] = PyObject_IsTrue(args[5 + i])) < 0) return nullptr;
        const Flags f{flag[0] != 0, flag[1] != 0, flag[2] != 0, flag[3] != 0};
        return wrap(unlocked([&] { return product(x, p, bias, f, y); }), y);
    });
}

// Whether `l` takes rows of `inner` values of `type` (the rest of `product`'s checks is x's).
bool linear_fits(const Linear &l, const Place &at, at::ScalarType type, int64_t inner) {
    int64_t columns;
    return l.p.fits(at, type, 2, columns) && columns == inner && bias_fits(l.bias, at, type, l.p.w.size(0));
}

// mlp(block, x): layers.Mlp.forward
PyObject *py_mlp(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        Tensor x, hidden, y;
        Linear down, gate, up, fused;
        if (n != 2 || !as_tensor(args[1], x) || !x.defined() || x.dim() < 1 || x.numel() == 0) return none();
        Ref geglu(PyObject_GetAttr(args[0], names.geglu)), both(PyObject_GetAttr(args[0], names.gate_up_proj));
        if (geglu.p == nullptr || both.p == nullptr || !read_linear(args[0], names.down_proj, down) ||
            !read_linear(args[0], names.gate_proj, gate)) {
            PyErr_Clear();
            return none();
        }
        const int truth = PyObject_IsTrue(geglu.p);
        if (truth < 0) return nullptr;
        const int32_t activation = truth ? NVQ_GLU_GEGLU : NVQ_GLU_SWIGLU;
        const int64_t rows = x.numel() / x.size(-1), most = gate.p.q.mode == NVQ_AFFINE ? 2 : 4;  // (layers.Mlp.forward says why)
        const Place at(x);
        const at::ScalarType type = x.scalar_type();
        if (!linear_fits(gate, at, type, x.size(-1)) || !linear_fits(down, at, type, gate.p.w.size(0))) return none();
        const bool several = rows > most;
        bool paired = both.p != Py_None;
        Several asked;
        if (paired && several) {  // (what the projections' sizes say already: the pair is not read where it would be refused)
            const nvq_qmm_desc d = gated_desc(x, code_of(type), gate.p.q, 2 * gate.p.w.size(0));
            asked.kernel = nvq_quantized_matmul_glu_several_takes(&d, &asked.need);
            paired = asked.kernel != 0;
        }
        if (paired) {
            const bool fits = read_linear(both.p, fused) && linear_fits(fused, at, type, x.size(-1)) && fused.p.w.size(0) == 2 * gate.p.w.size(0);
            if (!fits && !several) return none();
            if (fits) {
                const nvq_quant &q = gate.p.q, &r = fused.p.q;
                const bool same = q.mode == r.mode && q.group_size == r.group_size && q.bits == r.bits;
                const bool done = unlocked([&] {
                    return product_glu(x, fused.p, fused.bias, activation, 0.0f, 0.0f, several, same ? &asked : nullptr, hidden) && product(hidden, down.p, down.bias, Flags(), y);
                });
                if (hidden.defined()) return wrap(done, y);
            }
        }
        if (!read_linear(args[0], names.up_proj, up) || !linear_fits(up, at, type, x.size(-1)) || up.p.w.size(0) != gate.p.w.size(0)) return none();
        const bool done = unlocked([&] {
            Tensor g, u;
            return product(x, gate.p, gate.bias, Flags(), g) && product(x, up.p, up.bias, Flags(), u) && gated(g, u, activation, hidden) &&
                   product(hidden, down.p, down.bias, Flags(), y);
        });
        return wrap(done, y);
    });
}

bool read_projection(PyObject *o, PyObject *name, Projection &j) {
    Ref a(PyObject_GetAttr(o, name));
    if (a.p == nullptr) return declined();
    if (!projection_kind.plain(a.p)) return false;
    Tensor global_scale;
    if (!read_tensor(a.p, names.weight, j.p.w) || !read_tensor(a.p, names.scales, j.p.s) || !read_tensor(a.p, names.biases, j.p.b) ||
        !read_tensor(a.p, names.bias, j.bias) || !read_tensor(a.p, names.global_scale, global_scale) || global_scale.defined())
        return false;
    Ref q(PyObject_GetAttr(a.p, names.quant));
    return q.p == nullptr ? declined() : read_quant(q.p, j.p.q);
}

// moe(block, x): layers.MoeMlp.forward
PyObject *py_moe(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        Tensor x, router, y;
        int32_t k;
        bool normalize;
        Experts e;
        if (n != 2 || !moe_kind.plain(args[0]) || !as_tensor(args[1], x) || !read_tensor(args[0], names.gate, router) || !read_int(args[0], names.experts_per_token, k) ||
            !read_truth(args[0], names.norm_topk_prob, normalize))
            return none();
        Ref glu(PyObject_GetAttr(args[0], names.switch_mlp));
        if (glu.p == nullptr || !switch_glu_kind.plain(glu.p)) {
            PyErr_Clear();
            return none();
        }
        Ref both(PyObject_GetAttr(glu.p, names.gate_up_proj)), activation(PyObject_GetAttr(glu.p, names.activation));
        if (both.p == nullptr || activation.p == nullptr || !PyUnicode_Check(activation.p)) {
            PyErr_Clear();
            return none();
        }
        e.fused = both.p != Py_None;
        if (PyUnicode_CompareWithASCIIString(activation.p, "swiglu") == 0) e.act.code = NVQ_GLU_SWIGLU;
        else if (PyUnicode_CompareWithASCIIString(activation.p, "swiglu_oai") == 0) e.act.code = NVQ_GLU_SWIGLU_OAI;
        else if (PyUnicode_CompareWithASCIIString(activation.p, "geglu") == 0) e.act.code = NVQ_GLU_GEGLU;
        else return none();
        if (!read_projection(glu.p, names.gate_proj, e.gate) || !read_projection(glu.p, names.up_proj, e.up) ||
            !read_projection(glu.p, names.down_proj, e.down) || (e.fused && !read_projection(glu.p, names.gate_up_proj, e.both)) ||
            !read_truth(glu.p, names.gate_up_paired, e.paired) || !read_float(glu.p, names.alpha, e.act.alpha) ||
            !read_float(glu.p, names.limit, e.act.limit))
            return none();
        return wrap(unlocked([&] { return moe(x, router, k, normalize, e, y); }), y);
    });
}

// quantize(w, quant): (packed, scales, biases)
PyObject *py_quantize(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        Tensor w;
        nvq_quant q;
        if (n != 2 || !as_tensor(args[0], w) || !read_quant(args[1], q)) return none();
        const Place at(w);
        if (!at.usable() || w.dim() < 2 || w.numel() == 0 || !w.is_contiguous() || code_of(w.scalar_type()) < 0) return none();
        const int64_t cols = w.size(-1);
        if (q.group_size <= 0 || cols % q.group_size != 0) return none();
        const bool affine = q.mode == NVQ_AFFINE;
        const Sizes groups = with_last(w.sizes(), cols / q.group_size);
        Tensor packed, scales, biases;
        const bool done = unlocked([&] {
            packed = at.empty(with_last(w.sizes(), cols * q.bits / 32), at::kUInt32);
            scales = at.empty(groups, affine ? w.scalar_type() : at::kByte);
            if (affine) biases = at.empty(groups, w.scalar_type());
            return nvq_quantize(&q, code_of(w.scalar_type()), ptr(w), w.numel() / cols, cols, packed.mutable_data_ptr(), scales.mutable_data_ptr(),
                                affine ? biases.mutable_data_ptr() : nullptr, at.stream()) == NVQ_OK;
        });
        if (!done) return none();
        Ref p(THPVariable_Wrap(std::move(packed))), s(THPVariable_Wrap(std::move(scales)));
        Ref b(affine ? THPVariable_Wrap(std::move(biases)) : none());
        return p.p && s.p && b.p ? PyTuple_Pack(3, p.p, s.p, b.p) : nullptr;
    });
}

// The type a packed table gives its rows: the scales' for affine codes, else bfloat16 (ops.dequantize).
at::ScalarType table_type(const Packed &p) { return p.q.mode == NVQ_AFFINE && p.s.defined() ? p.s.scalar_type() : at::kBFloat16; }

bool is_dtype(PyObject *o, at::ScalarType &t) {
    if (!THPDtype_Check(o)) return false;
    t = reinterpret_cast<THPDtype *>(o)->scalar_type;
    return true;
}

// dequantize(weight, scales, biases, quant, dtype or None)
PyObject *py_dequantize(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        Packed p;
        if (n != 5 || !as_tensor(args[0], p.w) || !as_tensor(args[1], p.s) || !as_tensor(args[2], p.b) || !read_quant(args[3], p.q)) return none();
        const Place at(p.w);
        at::ScalarType type = table_type(p), asked = type;
        if (args[4] != Py_None && !is_dtype(args[4], asked)) return none();
        if (p.q.mode != NVQ_AFFINE) type = asked;
        int64_t columns;
        if (!at.usable() || code_of(type) < 0 || asked != type || p.w.dim() < 2 || p.w.numel() == 0 || !p.fits(at, type, p.w.dim(), columns))
            return none();
        Tensor y;
        const bool done = unlocked([&] {
            y = at.empty(with_last(p.w.sizes(), columns), type);
            return nvq_dequantize(&p.q, code_of(type), ptr(p.w), ptr(p.s), ptr(p.b), y.numel() / columns, columns, y.mutable_data_ptr(),
                                  at.stream()) == NVQ_OK;
        });
        return wrap(done, y);
    });
}

// embedding(weight, scales, biases, quant, ids)
PyObject *py_embedding(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        Packed p;
        Tensor ids;
        if (n != 5 || !as_tensor(args[0], p.w) || !as_tensor(args[1], p.s) || !as_tensor(args[2], p.b) || !read_quant(args[3], p.q) ||
            !as_tensor(args[4], ids))
            return none();
        const Place at(p.w);
        const at::ScalarType type = table_type(p);
        int64_t columns;
        if (!at.usable() || code_of(type) < 0 || !ids.defined() || !is_word(ids.scalar_type()) || !at.holds(ids) || ids.numel() == 0 ||
            !p.fits(at, type, 2, columns))
            return none();
        Sizes sizes(ids.sizes().begin(), ids.sizes().end());
        sizes.push_back(columns);
        Tensor y;
        const bool done = unlocked([&] {
            y = at.empty(sizes, type);
            return nvq_dequantize_rows(&p.q, code_of(type), ptr(p.w), ptr(p.s), ptr(p.b), p.w.size(0), columns, (const uint32_t *)ptr(ids),
                                       ids.numel(), y.mutable_data_ptr(), at.stream()) == NVQ_OK;
        });
        return wrap(done, y);
    });
}

// attention(q, k weight, scales, biases, v weight, scales, biases, quant, scale, sinks, causal[, several float32 rows too])
// (ops.quantized_attention, ops.quantized_attention_fits for one query row per head; ops.quantized_attention_prompt)
PyObject *py_attention(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        Tensor q, sinks;
        Packed k, v;
        if ((n != 11 && n != 12) || !as_tensor(args[0], q) || !as_tensor(args[1], k.w) || !as_tensor(args[2], k.s) || !as_tensor(args[3], k.b) ||
            !as_tensor(args[4], v.w) || !as_tensor(args[5], v.s) || !as_tensor(args[6], v.b) || !read_quant(args[7], k.q) ||
            !as_tensor(args[9], sinks))
            return none();
        v.q = k.q;
        const double scale = PyFloat_AsDouble(args[8]);
        if (scale == -1.0 && PyErr_Occurred()) {
            PyErr_Clear();
            return none();
        }
        const Place at(q);
        int64_t dim, same;
        if (!at.usable() || q.dim() != 4 || q.numel() == 0 || !q.is_contiguous() || k.q.mode != NVQ_AFFINE) return none();
        const at::ScalarType type = q.scalar_type();
        const int32_t code = code_of(type);
        if (code < 0 || !k.fits(at, type, 4, dim) || !v.fits(at, type, 4, same) || dim != q.size(3) || same != dim ||
            k.w.sizes() != v.w.sizes() || k.w.size(0) != q.size(0) || k.w.size(1) == 0 || k.w.size(2) == 0 ||
            !bias_fits(sinks, at, type, q.size(1)))
            return none();
        const nvq_attention_desc d{code, k.q.bits, k.q.group_size, (int32_t)dim, q.size(0), q.size(1), k.w.size(1), k.w.size(2), (float)scale};
        const bool several = q.size(2) > 1;
        // (ops.quantized_attention_fits: one query row takes caches of unsigned words)
        if (!several && (k.w.scalar_type() != at::kUInt32 || v.w.scalar_type() != at::kUInt32)) return none();
        const int causal = PyObject_IsTrue(args[10]), single_too = n == 12 ? PyObject_IsTrue(args[11]) : 0;
        if (causal < 0 || single_too < 0) return nullptr;
        const bool single = several && code == NVQ_F32;
        if (single && !single_too) return none();
        const nvq_attention_prompt_desc prompt{d, q.size(2), causal};
        Tensor y;
        const bool done = unlocked([&] {
            const size_t need = single    ? nvq_quantized_attention_prompt_f32_workspace_bytes(&prompt)
                                : several ? nvq_quantized_attention_prompt_workspace_bytes(&prompt)
                                          : nvq_quantized_attention_workspace_bytes(&d);
            if (several && !single && need == 0) return false;
            y = at.empty(q.sizes(), type);
            Tensor workspace;
            if (need > 0) workspace = at.empty({(int64_t)need}, at::kByte);
            void *scratch = need > 0 ? workspace.mutable_data_ptr() : nullptr;
            if (single)
                return nvq_quantized_attention_prompt_f32(&prompt, ptr(q), ptr(k.w), ptr(k.s), ptr(k.b), ptr(v.w), ptr(v.s), ptr(v.b), ptr(sinks),
                                                          y.mutable_data_ptr(), scratch, at.stream()) == NVQ_OK;
            return (several ? nvq_quantized_attention_prompt(&prompt, ptr(q), ptr(k.w), ptr(k.s), ptr(k.b), ptr(v.w), ptr(v.s), ptr(v.b), ptr(sinks),
                                                             y.mutable_data_ptr(), scratch, at.stream())
                            : nvq_quantized_attention(&d, ptr(q), ptr(k.w), ptr(k.s), ptr(k.b), ptr(v.w), ptr(v.s), ptr(v.b), ptr(sinks),
                                                      y.mutable_data_ptr(), scratch, at.stream())) == NVQ_OK;
        });
        return wrap(done, y);
    });
}

// ── heads and the paged cache (paged.py) ────────────────────────────────────────────────────────────────────────────
// A rotation's table of angles, or none at all; nothing here is looked up of a class, so any object with the attributes will do.
struct Angles {
    Tensor table;
    bool interleaved = false;
    nvq_rotary_axes axes{};  // count 0: none; else one more than the largest of the pairs'
    int64_t pairs = -1;      // that have an axis
    int32_t dims() const { return table.defined() ? (int32_t)(2 * table.size(1)) : 0; }
    int64_t rows() const { return table.defined() ? table.size(0) : 0; }
    bool fits(const Place &at, int64_t dim, int64_t least = 1) const {  // least: pairs
        return !table.defined() || (table.scalar_type() == at::kFloat && table.dim() == 3 && table.size(2) == 2 && table.size(0) > 0 && table.size(1) >= least &&
                                    2 * table.size(1) <= dim && at.holds(table));
    }
};
bool read_axes(PyObject *o, Angles &a) {
    Ref axes(PyObject_GetAttr(o, names.axes));
    if (axes.p == nullptr) PyErr_Clear();  // (an object without them)
    if (axes.p == nullptr || axes.p == Py_None) return true;
    if (!PyTuple_CheckExact(axes.p) || PyTuple_GET_SIZE(axes.p) > 256) return false;
    a.pairs = PyTuple_GET_SIZE(axes.p);
    for (int64_t i = 0; i < a.pairs; i++) {
        PyObject *v = PyTuple_GET_ITEM(axes.p, i);
        const long axis = PyLong_Check(v) ? PyLong_AsLong(v) : -1;
        if (PyErr_Occurred()) return declined();
        if (axis < 0 || axis > 3) return false;
        a.axes.of_pairs[i / 16] |= (uint32_t)axis << 2 * (i % 16);
        if (axis >= a.axes.count) a.axes.count = (int32_t)axis + 1;
    }
    return true;
}
bool read_angles(PyObject *o, Angles &a) {
    return o == Py_None || (read_tensor(o, names.table, a.table) && a.table.defined() && read_truth(o, names.interleaved, a.interleaved) && read_axes(o, a));
}
// The axes for positions of `count` of them.
bool axes_fit(const Angles &a, int64_t count, nvq_rotary_axes &axes) {
    axes = a.axes, axes.count = (int32_t)count;
    return a.table.defined() && a.pairs == a.table.size(1) && count >= a.axes.count && count <= 4;
}

bool weight_fits(const Tensor &w, const Place &at, at::ScalarType type, int64_t dim) {
    return !w.defined() || (w.scalar_type() == type && w.dim() == 1 && w.size(0) == dim && at.holds(w));
}

bool is_index(const Tensor &t, const Place &at, int64_t n) { return t.defined() && t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && at.holds(t); }

// Heads [batch, heads, length, dim] with consecutive values, on the device.
bool is_heads(const Tensor &x, const Place &at, at::ScalarType type) {
    return x.defined() && x.dim() == 4 && x.numel() > 0 && x.device() == at.device && x.scalar_type() == type && x.stride(3) == 1 && x.size(3) <= 512;
}

// Rows that share their memory: never written.
bool is_expanded(const Tensor &y) {
    for (int64_t i = 0; i < y.dim(); i++)
        if (y.size(i) > 1 && y.stride(i) == 0) return true;
    return false;
}

// Operands of one call (queries and keys, or one alone) rotated into dense outputs with consecutive values, or `out` of the first.
bool rotate(const Place &at, const Tensor *xs, const Tensor *weights, int count, const Angles &angles, const Tensor &offsets, int64_t offset, double eps,
            Tensor *ys) {
    const Tensor &x = xs[0];
    nvq_head_rope_desc d{};
    d.dtype = code_of(x.scalar_type()), d.head_dim = (int32_t)x.size(3), d.rotary_dims = angles.dims(), d.interleaved = angles.interleaved;
    d.table_rows = angles.rows(), d.batch = x.size(0), d.length = x.size(2), d.eps = eps;
    nvq_rotary_axes axes;
    const bool several = offsets.defined() && offsets.dim() == 3;
    if (several) {
        if (!axes_fit(angles, offsets.size(0), axes) || offsets.scalar_type() != at::kInt || !at.holds(offsets) || offsets.size(1) != d.batch ||
            offsets.size(2) != d.length)
            return false;
    } else if (offsets.defined()) {
        d.per_position = offsets.dim() == 2;
        if (offsets.scalar_type() != at::kInt || !at.holds(offsets) || offsets.dim() < 1 || offsets.dim() > 2 || offsets.size(0) != d.batch ||
            (d.per_position && offsets.size(1) != d.length))
            return false;
    } else {
        d.offset = offset;
        if (angles.table.defined() && (offset < 0 || offset + d.length > d.table_rows)) return false;
    }
    for (int i = 0; i < count; i++) {
        if (!ys[i].defined()) {
            // (the strides' order is x's; one of overlapping rows may put another dimension innermost)
            const auto strides = at::infer_dense_strides(xs[i].sizes(), xs[i].strides());
            ys[i] = strides[3] == 1 || xs[i].size(3) == 1 ? at::detail::empty_strided_cuda(xs[i].sizes(), strides, xs[i].scalar_type(), at.device)
                                                          : at.empty(xs[i].sizes(), xs[i].scalar_type());
        } else if (!is_heads(ys[i], at, x.scalar_type()) || ys[i].sizes() != xs[i].sizes() || is_expanded(ys[i])) {
            return false;
        }
        d.heads[i] = xs[i].size(1);
        for (int k = 0; k < 3; k++) d.x_strides[i][k] = xs[i].stride(k), d.y_strides[i][k] = ys[i].stride(k);
    }
    const bool two = count == 2;
    if (several)
        return nvq_head_norm_rope_axes(&d, &axes, (const float *)ptr(angles.table), (const int32_t *)ptr(offsets), ptr(xs[0]), ptr(weights[0]),
                                       ys[0].mutable_data_ptr(), two ? ptr(xs[1]) : nullptr, two ? ptr(weights[1]) : nullptr,
                                       two ? ys[1].mutable_data_ptr() : nullptr, at.stream()) == NVQ_OK;
    return nvq_head_norm_rope(&d, (const float *)ptr(angles.table), (const int32_t *)ptr(offsets), ptr(xs[0]), ptr(weights[0]), ys[0].mutable_data_ptr(),
                              two ? ptr(xs[1]) : nullptr, two ? ptr(weights[1]) : nullptr, two ? ys[1].mutable_data_ptr() : nullptr,
                              at.stream()) == NVQ_OK;
}

// An offset: a tensor, or an int.
bool read_offset(PyObject *o, Tensor &offsets, int64_t &offset) {
    if (THPVariable_Check(o)) return as_tensor(o, offsets);
    if (!PyLong_Check(o)) return false;
    offset = PyLong_AsLongLong(o);
    return offset != -1 || !PyErr_Occurred() || declined();
}

// rope(x, rotation, offset, out or None)
PyObject *py_rope(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        Tensor x, y, offsets;
        const Tensor no_weight;
        Angles angles;
        int64_t offset = 0;
        if (n != 4 || !as_tensor(args[0], x) || !read_angles(args[1], angles) || !angles.table.defined() || !read_offset(args[2], offsets, offset) ||
            !as_tensor(args[3], y))
            return none();
        const Place at(x);
        if (!at.usable() || code_of(x.scalar_type()) < 0 || !is_heads(x, at, x.scalar_type()) || !angles.fits(at, x.size(3))) return none();
        return wrap(unlocked([&] { return rotate(at, &x, &no_weight, 1, angles, offsets, offset, 0.0, &y); }), y);
    });
}

// head_norm_rope(q, k, q weight, k weight, rotation or None, offset, eps)
PyObject *py_head_norm_rope(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        Tensor xs[2], ys[2], weights[2], offsets;
        Angles angles;
        int64_t offset = 0;
        if (n != 7 || !as_tensor(args[0], xs[0]) || !as_tensor(args[1], xs[1]) || !as_tensor(args[2], weights[0]) || !as_tensor(args[3], weights[1]) ||
            !read_angles(args[4], angles) || !read_offset(args[5], offsets, offset))
            return none();
        const double eps = PyFloat_AsDouble(args[6]);
        if (eps == -1.0 && PyErr_Occurred()) return declined(), none();
        const Place at(xs[0]);
        if (!at.usable() || code_of(xs[0].scalar_type()) < 0) return none();
        const at::ScalarType type = xs[0].scalar_type();
        for (int i = 0; i < 2; i++)
            if (!is_heads(xs[i], at, type) || !weight_fits(weights[i], at, type, xs[0].size(3))) return none();
        if (xs[1].size(0) != xs[0].size(0) || xs[1].size(2) != xs[0].size(2) || xs[1].size(3) != xs[0].size(3) || !angles.fits(at, xs[0].size(3))) return none();
        if (!unlocked([&] { return rotate(at, xs, weights, 2, angles, offsets, offset, eps, ys); })) return none();
        Ref q(THPVariable_Wrap(std::move(ys[0]))), k(THPVariable_Wrap(std::move(ys[1])));
        return q.p && k.p ? PyTuple_Pack(2, q.p, k.p) : nullptr;
    });
}

struct Paged {
    Packed k, v;
    Tensor table;  // of pages
    nvq_paged_desc d{};

    bool fits(const Place &at, at::ScalarType type) {
        int64_t dim, same;
        const auto apart = [](const Tensor &t) { return t.dim() == 2 && (t.numel() == 0 || (t.stride(1) == 1 && t.stride(0) >= t.size(1))); };
        if (code_of(type) < 0 || k.q.mode != NVQ_AFFINE || k.q.bits != v.q.bits || k.q.group_size != v.q.group_size || v.q.mode != NVQ_AFFINE ||
            !k.fits(at, type, 4, dim) || !v.fits(at, type, 4, same) || k.w.sizes() != v.w.sizes() || !table.defined() || table.scalar_type() != at::kInt ||
            table.device() != at.device || !apart(table) || k.w.numel() == 0)
            return false;
        d = nvq_paged_desc{code_of(type), k.q.bits, k.q.group_size, (int32_t)dim, k.w.size(0), k.w.size(2), k.w.size(1), table.size(0), table.size(1),
                           std::max(table.stride(0), table.size(1))};
        return true;
    }
};
bool read_pages(PyObject *o, PyObject *name, Packed &p) {
    Ref a(PyObject_GetAttr(o, name));
    if (a.p == nullptr) return declined();
    Ref q(PyObject_GetAttr(a.p, names.quant));
    return q.p == nullptr ? declined() : read_quant(q.p, p.q) && read_tensor(a.p, names.weight, p.w) && read_tensor(a.p, names.scales, p.s) && read_tensor(a.p, names.biases, p.b);
}
bool read_paged(PyObject *cache, PyObject *table, Paged &p) { return read_pages(cache, names.keys, p.k) && read_pages(cache, names.values, p.v) && as_tensor(table, p.table); }

// Rows [tokens, heads, dim] with consecutive values.
bool is_rows(const Tensor &x, const Place &at, at::ScalarType type, int64_t tokens, int64_t dim) {
    return x.defined() && x.dim() == 3 && x.numel() > 0 && x.device() == at.device && x.scalar_type() == type && x.size(0) == tokens && x.size(2) == dim &&
           x.stride(2) == 1;
}

// append_paged(cache, k, v, page table, positions, sequences, rotation, k weight, q, q weight, eps, rotary positions): the queries, or True without any
PyObject *py_append_paged(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        Paged p;
        Angles angles;
        Tensor k, v, positions, sequences, k_weight, q, q_weight, rotary, y;
        if (n != 12 || !as_tensor(args[11], rotary) || !as_tensor(args[1], k) || !as_tensor(args[2], v) || !read_paged(args[0], args[3], p) || !as_tensor(args[4], positions) ||
            !as_tensor(args[5], sequences) || !read_angles(args[6], angles) || !as_tensor(args[7], k_weight) || !as_tensor(args[8], q) ||
            !as_tensor(args[9], q_weight))
            return none();
        const double eps = PyFloat_AsDouble(args[10]);
        if (eps == -1.0 && PyErr_Occurred()) return declined(), none();
        const Place at(k);
        if (!at.usable() || k.dim() != 3) return none();
        const at::ScalarType type = k.scalar_type();
        const int64_t tokens = k.size(0), dim = k.size(2);
        if (!p.fits(at, type) || p.d.head_dim != dim || !is_rows(k, at, type, tokens, dim) || !is_rows(v, at, type, tokens, dim) ||
            k.size(1) != p.d.key_heads || v.size(1) != p.d.key_heads || !is_index(positions, at, tokens) ||
            (sequences.defined() ? !is_index(sequences, at, tokens) : p.d.sequences != tokens) || !angles.fits(at, dim, 0) ||
            !weight_fits(k_weight, at, type, dim) || (q.defined() && (!is_rows(q, at, type, tokens, dim) || !weight_fits(q_weight, at, type, dim))))
            return none();
        nvq_paged_append_desc d{};
        d.cache = p.d, d.tokens = tokens, d.rotary_dims = angles.dims(), d.interleaved = angles.interleaved, d.table_rows = angles.rows(), d.eps = eps;
        d.query_heads = q.defined() ? q.size(1) : 0;
        for (int i = 0; i < 2; i++) {
            d.k_strides[i] = k.stride(i), d.v_strides[i] = v.stride(i);
            if (q.defined()) d.q_strides[i] = q.stride(i);
        }
        nvq_rotary_axes axes{1, {}};
        if (rotary.defined()) {
            const bool one = rotary.dim() == 1;
            if (!angles.table.defined() || (one ? !is_index(rotary, at, tokens) : rotary.dim() != 2 || !axes_fit(angles, rotary.size(0), axes) ||
                                                                                      rotary.scalar_type() != at::kInt || rotary.size(1) != tokens || !at.holds(rotary)))
                return none();
        }
        const bool done = unlocked([&] {
            if (q.defined()) y = at.empty(q.sizes(), type);
            if (rotary.defined())
                return nvq_append_paged_axes(&d, &axes, (const int32_t *)ptr(p.table), (const int32_t *)ptr(sequences), (const int32_t *)ptr(positions),
                                             (const int32_t *)ptr(rotary), (const float *)ptr(angles.table), ptr(q), q.defined() ? ptr(q_weight) : nullptr,
                                             q.defined() ? y.mutable_data_ptr() : nullptr, ptr(k), ptr(k_weight), ptr(v), (uint32_t *)p.k.w.mutable_data_ptr(),
                                             p.k.s.mutable_data_ptr(), p.k.b.mutable_data_ptr(), (uint32_t *)p.v.w.mutable_data_ptr(),
                                             p.v.s.mutable_data_ptr(), p.v.b.mutable_data_ptr(), at.stream()) == NVQ_OK;
            return nvq_append_paged(&d, (const int32_t *)ptr(p.table), (const int32_t *)ptr(sequences), (const int32_t *)ptr(positions),
                                    (const float *)ptr(angles.table), ptr(q), q.defined() ? ptr(q_weight) : nullptr,
                                    q.defined() ? y.mutable_data_ptr() : nullptr, ptr(k), ptr(k_weight), ptr(v), (uint32_t *)p.k.w.mutable_data_ptr(),
                                    p.k.s.mutable_data_ptr(), p.k.b.mutable_data_ptr(), (uint32_t *)p.v.w.mutable_data_ptr(), p.v.s.mutable_data_ptr(),
                                    p.v.b.mutable_data_ptr(), at.stream()) == NVQ_OK;
        });
        if (done && !q.defined()) Py_RETURN_TRUE;
        return wrap(done, y);
    });
}

// read_paged(cache, page table, positions, sequences)
PyObject *py_read_paged(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        Paged p;
        Tensor positions, sequences, keys, values;
        if (n != 4 || !read_paged(args[0], args[1], p) || !as_tensor(args[2], positions) || !as_tensor(args[3], sequences) || !p.k.s.defined()) return none();
        const Place at(p.k.w);
        const at::ScalarType type = p.k.s.scalar_type();
        if (!at.usable() || !p.fits(at, type) || !positions.defined() || positions.dim() != 1 || positions.size(0) == 0) return none();
        const int64_t tokens = positions.size(0);
        if (!is_index(positions, at, tokens) || (sequences.defined() ? !is_index(sequences, at, tokens) : p.d.sequences != tokens)) return none();
        const bool done = unlocked([&] {
            keys = at.empty({tokens, p.d.key_heads, p.d.head_dim}, type), values = at.empty({tokens, p.d.key_heads, p.d.head_dim}, type);
            return nvq_read_paged(&p.d, tokens, (const int32_t *)ptr(p.table), (const int32_t *)ptr(sequences), (const int32_t *)ptr(positions),
                                  (const uint32_t *)ptr(p.k.w), ptr(p.k.s), ptr(p.k.b), (const uint32_t *)ptr(p.v.w), ptr(p.v.s), ptr(p.v.b),
                                  keys.mutable_data_ptr(), values.mutable_data_ptr(), at.stream()) == NVQ_OK;
        });
        if (!done) return none();
        Ref k(THPVariable_Wrap(std::move(keys))), v(THPVariable_Wrap(std::move(values)));
        return k.p && v.p ? PyTuple_Pack(2, k.p, v.p) : nullptr;
    });
}

// paged_attention(q, cache, page table, lengths, scale, query starts, max queries or None, sinks, causal, window, out or None)
PyObject *py_paged_attention(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        Paged p;
        Tensor q, lengths, starts, sinks, y;
        if (n != 11 || !as_tensor(args[0], q) || !read_paged(args[1], args[2], p) || !as_tensor(args[3], lengths) || !as_tensor(args[5], starts) ||
            !as_tensor(args[7], sinks) || !as_tensor(args[10], y) || !PyLong_Check(args[9]))
            return none();
        const double scale = PyFloat_AsDouble(args[4]);
        if (scale == -1.0 && PyErr_Occurred()) return declined(), none();
        const int64_t window = PyLong_AsLongLong(args[9]);
        int64_t most = args[6] == Py_None ? INT64_MAX : PyLong_Check(args[6]) ? PyLong_AsLongLong(args[6]) : -1;
        if (PyErr_Occurred()) return declined(), none();
        const int causal = PyObject_IsTrue(args[8]);
        if (causal < 0) return nullptr;
        const Place at(q);
        if (!at.usable() || q.dim() != 3 || window < 0 || most < 0) return none();
        const at::ScalarType type = q.scalar_type();
        const int64_t rows = q.size(0), heads = q.size(1), dim = q.size(2);
        if (!p.fits(at, type) || p.d.head_dim != dim || !is_rows(q, at, type, rows, dim) || !is_index(lengths, at, p.d.sequences) ||
            (starts.defined() ? !is_index(starts, at, p.d.sequences + 1) : p.d.sequences != rows) || !bias_fits(sinks, at, type, heads) ||
            (y.defined() && (!is_rows(y, at, type, rows, dim) || y.size(1) != heads || is_expanded(y))))
            return none();
        nvq_paged_attention_desc d{};
        d.cache = p.d, d.rows = rows, d.query_heads = heads, d.max_queries = !starts.defined() ? 1 : most < 1 ? 1 : most < rows ? most : rows;
        d.window = window, d.causal = causal, d.scale = (float)scale;
        const bool done = unlocked([&] {
            if (!y.defined()) y = at.empty(q.sizes(), type);
            for (int i = 0; i < 2; i++) d.q_strides[i] = q.stride(i), d.out_strides[i] = y.stride(i);
            const size_t need = nvq_paged_attention_workspace_bytes(&d);
            Tensor workspace;
            if (need > 0) workspace = at.empty({(int64_t)need}, at::kByte);
            return nvq_paged_attention(&d, ptr(q), (const uint32_t *)ptr(p.k.w), ptr(p.k.s), ptr(p.k.b), (const uint32_t *)ptr(p.v.w), ptr(p.v.s),
                                       ptr(p.v.b), (const int32_t *)ptr(p.table), (const int32_t *)ptr(lengths), (const int32_t *)ptr(starts), ptr(sinks),
                                       y.mutable_data_ptr(), need > 0 ? workspace.mutable_data_ptr() : nullptr, at.stream()) == NVQ_OK;
        });
        return wrap(done, y);
    });
}

// Starts of sequences.
bool is_starts(const Tensor &t, const Place &at) { return t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) > 0 && at.holds(t); }

// prompt_attention(q, k, v, scale, query starts, key starts, sinks, causal, window, out or None)
PyObject *py_prompt_attention(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        Tensor q, k, v, starts, key_starts, sinks, y;
        if (n != 10 || !as_tensor(args[0], q) || !as_tensor(args[1], k) || !as_tensor(args[2], v) || !as_tensor(args[4], starts) || !as_tensor(args[5], key_starts) ||
            !as_tensor(args[6], sinks) || !as_tensor(args[9], y) || !PyLong_Check(args[8]))
            return none();
        const double scale = PyFloat_AsDouble(args[3]);
        if (scale == -1.0 && PyErr_Occurred()) return declined(), none();
        const int64_t window = PyLong_AsLongLong(args[8]);
        if (PyErr_Occurred()) return declined(), none();
        const int causal = PyObject_IsTrue(args[7]);
        if (causal < 0) return nullptr;
        const Place at(q);
        if (!at.usable() || q.dim() != 3 || !k.defined() || k.dim() != 3 || !v.defined() || window < 0) return none();
        const at::ScalarType type = q.scalar_type();
        const int64_t rows = q.size(0), heads = q.size(1), dim = q.size(2), keys = k.size(0);
        const int64_t sequences = starts.defined() && starts.dim() == 1 ? starts.size(0) - 1 : 1;
        if (code_of(type) < 0 || !is_rows(q, at, type, rows, dim) || !is_rows(k, at, type, keys, dim) || !is_rows(v, at, type, keys, dim) || v.size(1) != k.size(1) ||
            (starts.defined() && !is_starts(starts, at)) ||
            (key_starts.defined() ? !is_starts(key_starts, at) || key_starts.size(0) != sequences + 1 : sequences != 1 && keys != rows) ||
            !bias_fits(sinks, at, type, heads) || (y.defined() && (!is_rows(y, at, type, rows, dim) || y.size(1) != heads || is_expanded(y))))
            return none();
        nvq_prompt_attention_desc d{};
        d.dtype = code_of(type), d.head_dim = (int32_t)dim, d.rows = rows, d.keys = keys, d.query_heads = heads, d.key_heads = k.size(1), d.sequences = sequences;
        d.window = window, d.causal = causal, d.scale = (float)scale;
        const bool done = unlocked([&] {
            if (!y.defined()) y = at.empty(q.sizes(), type);
            for (int i = 0; i < 2; i++)
                d.q_strides[i] = q.stride(i), d.k_strides[i] = k.stride(i), d.v_strides[i] = v.stride(i), d.out_strides[i] = y.stride(i);
            const size_t need = nvq_prompt_attention_workspace_bytes(&d);
            Tensor workspace;
            if (need > 0) workspace = at.empty({(int64_t)need}, at::kByte);
            return nvq_prompt_attention(&d, ptr(q), ptr(k), ptr(v), (const int32_t *)ptr(starts), (const int32_t *)ptr(key_starts), ptr(sinks),
                                        y.mutable_data_ptr(), need > 0 ? workspace.mutable_data_ptr() : nullptr, at.stream()) == NVQ_OK;
        });
        return wrap(done, y);
    });
}

// ── adapters and the choice of experts ──────────────────────────────────────────────────────────────────────────────
// apply_adapters(y, x, adapters, ids, out or None)
PyObject *py_apply_adapters(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        Tensor x, y, ids, down, up, scales, out;
        if (n != 5 || !as_tensor(args[0], y) || !as_tensor(args[1], x) || !read_tensor(args[2], names.down, down) || !read_tensor(args[2], names.up, up) ||
            !read_tensor(args[2], names.scales, scales) || !as_tensor(args[3], ids) || !as_tensor(args[4], out))
            return none();
        const Place at(x);
        if (!at.usable() || !y.defined() || !ids.defined() || !down.defined() || !up.defined()) return none();
        const at::ScalarType type = x.scalar_type();
        const int64_t dims = x.dim();
        if (code_of(type) < 0 || dims < 1 || x.numel() == 0 || y.numel() == 0 || !at.holds(x) || !at.holds(y) || y.scalar_type() != type || y.dim() != dims ||
            down.dim() != 3 || up.dim() != 3 || down.scalar_type() != type || up.scalar_type() != type || !at.holds(down) || !at.holds(up) ||
            down.numel() == 0 || up.numel() == 0)
            return none();
        const int64_t inputs = x.size(dims - 1), outputs = y.size(dims - 1), rows = x.numel() / inputs, count = down.size(0), rank = down.size(1);
        if (down.size(2) != inputs || up.size(0) != count || up.size(1) != outputs || up.size(2) != rank || rank > INT32_MAX ||
            ids.scalar_type() != at::kInt || !at.holds(ids) || ids.sizes() != x.sizes().slice(0, dims - 1) || ids.sizes() != y.sizes().slice(0, dims - 1) ||
            (scales.defined() && (scales.scalar_type() != at::kFloat || scales.dim() != 1 || scales.size(0) != count || !at.holds(scales))) ||
            (out.defined() && (out.scalar_type() != type || !at.holds(out) || out.sizes() != y.sizes())))
            return none();
        const nvq_adapters_desc d{code_of(type), (int32_t)rank, rows, inputs, outputs, count, inputs, outputs, outputs};
        const bool done = unlocked([&] {
            if (!out.defined()) out = at.empty(y.sizes(), type);
            const size_t need = nvq_apply_adapters_workspace_bytes(&d);
            Tensor workspace;
            if (need > 0) workspace = at.empty({(int64_t)need}, at::kByte);
            return nvq_apply_adapters(&d, ptr(x), ptr(down), ptr(up), (const float *)ptr(scales), (const int32_t *)ptr(ids), ptr(y), out.mutable_data_ptr(),
                                      need > 0 ? workspace.mutable_data_ptr() : nullptr, at.stream()) == NVQ_OK;
        });
        return wrap(done, out);
    });
}

bool read_count(PyObject *o, int32_t otherwise, int32_t &v) {
    if (o == Py_None) return v = otherwise, true;
    if (!PyLong_Check(o)) return false;
    const long n = PyLong_AsLong(o);
    if (n == -1 && PyErr_Occurred()) return declined();
    return n >= 0 && n <= 1024 ? (v = (int32_t)n, true) : false;
}

// moe_select(logits, k, sigmoid or None, bias, groups, top groups, group best, normalize, scale)
PyObject *py_moe_select(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        Tensor logits, bias, experts, weights;
        nvq_moe_select_desc d{};
        if (n != 9 || !as_tensor(args[0], logits) || !read_count(args[1], 0, d.k) || !PyBool_Check(args[2]) || !as_tensor(args[3], bias) ||
            !read_count(args[4], 0, d.groups) || !read_count(args[5], d.groups, d.top_groups) || !read_count(args[6], bias.defined() ? 2 : 1, d.group_best))
            return none();
        const int normalize = PyObject_IsTrue(args[7]);
        if (normalize < 0) return nullptr;
        d.scale = PyFloat_AsDouble(args[8]);
        if (d.scale == -1.0 && PyErr_Occurred()) return declined(), none();
        const Place at(logits);
        if (!at.usable() || code_of(logits.scalar_type()) < 0 || logits.dim() < 1 || logits.numel() == 0 || !at.holds(logits) || d.k < 1) return none();
        const int64_t e = logits.size(logits.dim() - 1);
        if (e > 1024 || (bias.defined() && (bias.scalar_type() != at::kFloat || bias.dim() != 1 || bias.size(0) != e || !at.holds(bias)))) return none();
        d.dtype = code_of(logits.scalar_type()), d.scores = args[2] == Py_True ? NVQ_SCORES_SIGMOID : NVQ_SCORES_SOFTMAX, d.experts = (int32_t)e;
        d.normalize = normalize;
        if (nvq_moe_select(&d, nullptr, nullptr, nullptr, nullptr, nullptr) != NVQ_OK) return none();  // (the sizes)
        d.rows = logits.numel() / e;
        const bool done = unlocked([&] {
            std::vector<int64_t> sizes = logits.sizes().vec();
            sizes.back() = d.k;
            experts = at.empty(sizes, at::kInt), weights = at.empty(sizes, logits.scalar_type());
            return nvq_moe_select(&d, ptr(logits), (const float *)ptr(bias), (int32_t *)experts.mutable_data_ptr(), weights.mutable_data_ptr(), at.stream()) ==
                   NVQ_OK;
        });
        if (!done) return none();
        Ref i(THPVariable_Wrap(std::move(experts))), w(THPVariable_Wrap(std::move(weights)));
        return i.p && w.p ? PyTuple_Pack(2, i.p, w.p) : nullptr;
    });
}

// register((type, {name: function}), ...): QuantizedLinear, SwitchProjection, SwitchGlu and MoeMlp with their own methods
PyObject *py_register(PyObject *, PyObject *const *args, Py_ssize_t n) {
    Kind *const kinds[] = {&linear_kind, &projection_kind, &switch_glu_kind, &moe_kind};
    PyObject *types[4], *methods[4];
    for (Py_ssize_t i = 0; i < 4; i++) {
        if (n != 4 || !PyArg_ParseTuple(args[i], "O!O!", &PyType_Type, &types[i], &PyDict_Type, &methods[i])) {
            PyErr_SetString(PyExc_TypeError, "register: four pairs of a class and its methods");
            return nullptr;
        }
    }
    for (Py_ssize_t i = 0; i < 4; i++) {
        Py_INCREF(types[i]), Py_INCREF(methods[i]);  // (kept until the process ends, with the names and functions they hold)
        kinds[i]->methods.clear();
        PyObject *name, *function;
        for (Py_ssize_t at = 0; PyDict_Next(methods[i], &at, &name, &function);) kinds[i]->methods.emplace_back(name, function);
        kinds[i]->type = (PyTypeObject *)types[i];
    }
    return none();
}

// ready(index): nvq_init has answered for the device
PyObject *py_ready(PyObject *, PyObject *index) {
    const long i = PyLong_AsLong(index);
    if (i == -1 && PyErr_Occurred()) return nullptr;
    if (i >= 0 && i < 64) ready_devices |= 1ull << i;
    return none();
}

#define NVQ_FAST(f) (PyCFunction)(void (*)(void)) f, METH_FASTCALL
PyMethodDef methods[] = {
    {"register", NVQ_FAST(py_register), nullptr},
    {"ready", py_ready, METH_O, nullptr},
    {"linear", NVQ_FAST(py_linear), nullptr},
    {"quantized_matmul", NVQ_FAST(py_quantized_matmul), nullptr},
    {"mlp", NVQ_FAST(py_mlp), nullptr},
    {"moe", NVQ_FAST(py_moe), nullptr},
    {"quantize", NVQ_FAST(py_quantize), nullptr},
    {"dequantize", NVQ_FAST(py_dequantize), nullptr},
    {"embedding", NVQ_FAST(py_embedding), nullptr},
    {"attention", NVQ_FAST(py_attention), nullptr},
    {"rope", NVQ_FAST(py_rope), nullptr},
    {"head_norm_rope", NVQ_FAST(py_head_norm_rope), nullptr},
    {"append_paged", NVQ_FAST(py_append_paged), nullptr},
    {"read_paged", NVQ_FAST(py_read_paged), nullptr},
    {"paged_attention", NVQ_FAST(py_paged_attention), nullptr},
    {"prompt_attention", NVQ_FAST(py_prompt_attention), nullptr},
    {"apply_adapters", NVQ_FAST(py_apply_adapters), nullptr},
    {"moe_select", NVQ_FAST(py_moe_select), nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject *PyInit__native(void) {
    struct { PyObject **at; const char *text; } all[] = {
        {&names.mode, "mode"}, {&names.group_size, "group_size"}, {&names.bits, "bits"}, {&names.weight, "weight"},
        {&names.scales, "scales"}, {&names.biases, "biases"}, {&names.bias, "bias"}, {&names.quant, "quant"},
        {&names.global_scale, "global_scale"}, {&names.gate_proj, "gate_proj"}, {&names.up_proj, "up_proj"},
        {&names.down_proj, "down_proj"}, {&names.gate_up_proj, "gate_up_proj"}, {&names.geglu, "geglu"},
        {&names.gate, "gate"}, {&names.switch_mlp, "switch_mlp"}, {&names.experts_per_token, "experts_per_token"},
        {&names.norm_topk_prob, "norm_topk_prob"}, {&names.gate_up_paired, "gate_up_paired"}, {&names.activation, "activation"},
        {&names.alpha, "alpha"}, {&names.limit, "limit"}, {&names.keys, "keys"}, {&names.values, "values"},
        {&names.table, "table"}, {&names.interleaved, "interleaved"}, {&names.axes, "axes"}, {&names.down, "down"}, {&names.up, "up"},
    };
    for (auto &n : all) {
        *n.at = PyUnicode_InternFromString(n.text);
        if (*n.at == nullptr) return nullptr;
    }
    return PyModule_Create(&module);
}
