// uhm_torch.cpp -- the Python entry points of include/uh_model_ops.h on torch tensors (module _uhm_torch; ops.py holds their
// signatures and documentation).
//
// Native because of its cost: a list of 300 gradients takes 4 launches (12 us on the device), and reading the attributes of 300 tensors
// through the interpreter took 150 us; one 8-bit product for a single pair takes 10 us and its checks took 15.
// Every function checks its arguments, allocates outputs and workspace from torch's allocator, and enqueues on the current stream of the
// tensors' device.  Nothing is kept between calls.
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <c10/util/SmallVector.h>
#include <algorithm>
#include <deque>
#include <numeric>
#include <string>
#include <vector>
#include "../../include/uh_model_ops.h"

namespace {

using at::Tensor;
using std::string;
using std::vector;

PyObject* error_class = nullptr;

[[noreturn]] void fail(const string& what) {
    PyErr_SetString(error_class, what.c_str());
    throw py::error_already_set();
}

void check(int code, const char* what) {
    if (code) fail(string(what) + " failed: " + uhm_error_string(code) + " (code " + std::to_string(code) + ")");
}

string shape_of(const Tensor& t) {
    string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + (t.dim() == 1 ? ",)" : ")");
}

int dtype_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return UHM_F32;
        case at::kBFloat16: return UHM_BF16;
        case at::kHalf: return UHM_F16;
        default: return -1;
    }
}

string type_name(at::ScalarType t) { return py::str(py::cast(t)); }

bool on_device(PyObject* o) {
    if (!THPVariable_Check(o)) return false;
    const Tensor& t = THPVariable_Unpack(o);
    return t.is_cuda() && t.layout() == at::kStrided;
}
[[noreturn]] void not_on_device(PyObject* o, const string& name) {
    fail(name + " must be a dense tensor on the HIP device (got " +
         (THPVariable_Check(o) ? THPVariable_Unpack(o).device().str() : string(Py_TYPE(o)->tp_name)) + "); there is no CPU fallback");
}
const Tensor& tensor(const py::object& o, const char* name) {
    if (!on_device(o.ptr())) not_on_device(o.ptr(), name);
    return THPVariable_Unpack(o.ptr());
}

// A call records nothing for autograd, backward or forward: inputs that ask for that are refused rather than cut off in silence.
void no_tangent(const Tensor& t, const char* name) {
    if (t._fw_grad(/*level=*/0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
        fail(string(name) + " has no gradient: pass the primal of a tensor that carries a forward-mode tangent");
}
void no_gradient(const Tensor& t, const char* name) {
    if (!t.unsafeGetTensorImpl()->autograd_meta()) return;             // (lists of gradients: nothing to ask)
    if (t.requires_grad() && at::GradMode::is_enabled())
        fail(string(name) + " has no gradient: pass detached tensors or call it under torch.no_grad()");
    no_tangent(t, name);
}
// what an optimizer updates in place: leaves may ask for a gradient
void no_gradient_but_of_leaves(const Tensor& t, const char* name) {
    if (t.is_leaf()) no_tangent(t, name);
    else no_gradient(t, name);
}

// values as memory holds them (a lazy negation is carried out)
Tensor plain(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
// ... and without gaps, in whatever order
Tensor dense(const Tensor& t) {
    const Tensor p = plain(t);
    return p.is_non_overlapping_and_dense() ? p : p.contiguous();
}

void written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

struct Call {                                        // the device as the current one, its current stream
    c10::DeviceGuard guard;
    hipStream_t stream;
    at::TensorOptions options;
    explicit Call(at::Device d) : guard(d), stream(c10::hip::getCurrentHIPStream(d.index()).stream()), options(at::TensorOptions().device(d)) {}
    Tensor bytes(size_t n) const { return n ? at::empty({(int64_t)n}, options.dtype(at::kByte)) : Tensor(); }
    Tensor scalar() const { return at::empty({}, options.dtype(at::kFloat)); }
};
void* at_of(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// ---- lists ------------------------------------------------------------------------------------------------------------------
// The tensors stay those of the Python objects (references are not counted again: a list of 300 is read in 6 us), except where a
// copy takes the place of one.
struct List {
    py::object seq;
    vector<const Tensor*> t;
    std::deque<Tensor> copies;
    at::Device device = at::kCPU;
    void replace(size_t i, Tensor by) {
        copies.push_back(std::move(by));
        t[i] = &copies.back();
    }
    // copies in place of what does not fill its memory in some order
    void make_dense() {
        for (size_t i = 0; i < t.size(); ++i)
            if (t[i]->is_neg() || !t[i]->is_non_overlapping_and_dense()) replace(i, dense(*t[i]));
    }
};

List take_list(const py::object& given, const char* name, bool only_f32) {
    List l;
    PyObject* fast = PySequence_Fast(given.ptr(), "a list of tensors is needed");
    if (!fast) throw py::error_already_set();
    l.seq = py::reinterpret_steal<py::object>(fast);
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(fast);
    if (n == 0) fail(string(name) + ": at least one tensor is needed");
    if (n > 0x7fffffff) fail(string(name) + ": too many tensors");
    l.t.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject* o = PySequence_Fast_GET_ITEM(fast, i);
        if (!on_device(o)) not_on_device(o, name);
        const Tensor& t = THPVariable_Unpack(o);
        if (i == 0) l.device = t.device();
        const int d = dtype_of(t);
        if (d < 0 || (only_f32 && d != UHM_F32))
            fail(string(name) + ": " + type_name(t.scalar_type()) + " is not supported (" + (only_f32 ? "float32" : "float32, bfloat16, float16") + ")");
        if (t.device() != l.device) fail(string(name) + ": tensors on several devices (" + l.device.str() + ", " + t.device().str() + ")");
        l.t.push_back(&t);
    }
    return l;
}

struct Described {                                   // a list as the C entry points take it
    vector<const void*> p;
    vector<long long> numel;
    vector<int> dtype;
    explicit Described(const List& l) {
        p.reserve(l.t.size()); numel.reserve(l.t.size()); dtype.reserve(l.t.size());
        for (const Tensor* t : l.t) {
            p.push_back(t->data_ptr());
            numel.push_back(t->numel());
            dtype.push_back(dtype_of(*t));
        }
    }
    int count() const { return (int)p.size(); }
};
vector<const void*> pointers(const List& l) {
    vector<const void*> p;
    p.reserve(l.t.size());
    for (const Tensor* t : l.t) p.push_back(t->data_ptr());
    return p;
}

double clip_value(double clip, const char* name) {
    if (!(clip > 0.0)) fail(string(name) + ": clip_norm must be > 0 (got " + std::to_string(clip) + ")");
    return clip;
}

Tensor given_norm(const py::object& o, at::Device device, const char* name) {
    if (o.is_none()) return Tensor();
    const Tensor& t = tensor(o, "use_norm");
    no_gradient(t, name);
    if (t.scalar_type() != at::kFloat || t.numel() != 1 || t.device() != device) fail(string(name) + ": use_norm must be one float32 value on " + device.str());
    return plain(t);
}

Tensor global_norm(const py::object& tensors) {
    List l = take_list(tensors, "tensors", false);
    for (const Tensor* t : l.t) no_gradient(*t, "global_norm");
    const Call call(l.device);
    l.make_dense();
    const Described d(l);
    const size_t nbytes = uhm_multi_workspace_bytes(d.count());
    const Tensor norm = call.scalar(), ws = call.bytes(nbytes);
    check(uhm_global_norm(d.p.data(), d.numel.data(), d.dtype.data(), d.count(), (float*)norm.data_ptr(), ws.data_ptr(), nbytes, call.stream), "uhm_global_norm");
    return norm;
}

Tensor clip(const Call& call, const Described& d, const vector<const void*>& out, double clip_norm, const Tensor& use_norm, const char* name) {
    const size_t nbytes = use_norm.defined() ? 0 : uhm_multi_workspace_bytes(d.count());
    const Tensor norm = call.scalar(), ws = call.bytes(nbytes);
    check(uhm_clip_by_global_norm(d.p.data(), (void* const*)out.data(), d.numel.data(), d.dtype.data(), d.count(), (float)clip_norm, (const float*)at_of(use_norm),
                                  (float*)norm.data_ptr(), at_of(ws), nbytes, call.stream), name);
    return norm;
}

// Tensors like those of the list.  Allocating one costs 0.7 us, as much as 3 MB of clipping: small ones get their memory from one
// allocation together (each on 256 bytes; it is held until the last of them is gone), so that no more than SMALL bytes of a tensor are.
vector<Tensor> empty_like(const Call& call, const List& l) {
    constexpr size_t SMALL = 256 << 10, ALIGN = 256;
    auto room = [&](const Tensor& t) { return (t.nbytes() + ALIGN - 1) / ALIGN * ALIGN; };
    size_t shared = 0;
    for (const Tensor* t : l.t)
        if (t->nbytes() <= SMALL) shared += room(*t);
    const Tensor all = at::empty({(int64_t)shared}, call.options.dtype(at::kByte));
    vector<Tensor> out;
    out.reserve(l.t.size());
    size_t at = 0;
    for (const Tensor* t : l.t) {
        if (t->nbytes() > SMALL) {
            out.push_back(at::empty_strided(t->sizes(), t->strides(), call.options.dtype(t->scalar_type())));
            continue;
        }
        Tensor o = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), t->dtype());
        o.unsafeGetTensorImpl()->set_sizes_and_strides(t->sizes(), t->strides(), (int64_t)(at / t->element_size()));
        out.push_back(std::move(o));
        at += room(*t);
    }
    return out;
}

py::tuple clip_by_global_norm(const py::object& tensors, double clip_norm, const py::object& use) {
    const char* name = "clip_by_global_norm";
    clip_value(clip_norm, name);
    List l = take_list(tensors, "tensors", false);
    const Tensor use_norm = given_norm(use, l.device, name);
    for (const Tensor* t : l.t) no_gradient(*t, name);
    const Call call(l.device);
    l.make_dense();
    const vector<Tensor> out = empty_like(call, l);
    vector<const void*> p;
    p.reserve(out.size());
    for (const Tensor& t : out) p.push_back(t.data_ptr());
    const Tensor norm = clip(call, Described(l), p, clip_norm, use_norm, name);
    py::list given_back(out.size());
    for (size_t i = 0; i < out.size(); ++i) given_back[i] = py::cast(out[i]);
    return py::make_tuple(given_back, norm);
}

// ---- views that are written in place ------------------------------------------------------------------------------------------
// A view is the bytes base + sum_k stride_k i_k + (0 .. width - 1), 0 <= i_k < size_k.  Whether two views share a byte is whether a sum of
// terms c x, lo <= x <= hi, reaches an interval.
struct Term { int64_t c, lo, hi; };                  // c > 0
using Terms = c10::SmallVector<Term, 8>;             // (300 slices of one tensor are 45000 pairs)

struct Sum {
    Terms t;                                         // largest c first, each c once
    c10::SmallVector<int64_t, 9> low, high;          // of the terms from k on
    int budget = 1 << 16;                            // steps of the search; past them the views count as sharing

    explicit Sum(Terms terms) {
        std::sort(terms.begin(), terms.end(), [](const Term& a, const Term& b) { return a.c > b.c; });
        for (const Term& x : terms) {
            if (!t.empty() && t.back().c == x.c) { t.back().lo += x.lo; t.back().hi += x.hi; }
            else t.push_back(x);
        }
        low.assign(t.size() + 1, 0);
        high.assign(t.size() + 1, 0);
        for (size_t k = t.size(); k-- > 0;) {
            low[k] = low[k + 1] + t[k].c * t[k].lo;
            high[k] = high[k + 1] + t[k].c * t[k].hi;
        }
    }
    static int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }      // b > 0

    bool search(size_t k, int64_t from, int64_t to) {
        if (k == t.size()) return from <= 0 && 0 <= to;
        const int64_t c = t[k].c, first = std::max(t[k].lo, -floor_div(high[k + 1] - from, c)), last = std::min(t[k].hi, floor_div(to - low[k + 1], c));
        for (int64_t x = first; x <= last; ++x)
            if (--budget < 0 || search(k + 1, from - c * x, to - c * x)) return true;
        return false;
    }
    bool reaches(int64_t from, int64_t to) {
        // the terms up to k add up to a multiple of their common divisor, the others to something in [low, high]: rows and columns of one
        // larger tensor are told apart here
        int64_t g = 0;
        for (size_t k = 0; k < t.size(); ++k) {
            g = std::gcd(g, t[k].c);
            if (floor_div(to - low[k + 1], g) * g < from - high[k + 1]) return false;
        }
        return search(0, from, to);
    }
};

struct View {
    uintptr_t base, end;
    int64_t width, row = 0, rows = 0, within;        // the largest stride, the bytes it spans, and those that the rest spans
    c10::SmallVector<std::pair<int64_t, int64_t>, 4> dims;             // stride in bytes, size - 1
    bool copied;                                     // clipped in a copy: the native check sees the copy
    explicit View(const Tensor& v)
        : base((uintptr_t)v.data_ptr()), end(base + v.element_size()), width(v.element_size()), copied(v.is_neg() || !v.is_non_overlapping_and_dense()) {
        for (int64_t i = 0; i < v.dim(); ++i) {
            const int64_t stride = v.stride(i) * width, last = v.size(i) - 1;
            if (last < 1 || stride == 0) continue;                      // (an expanded dimension adds no bytes)
            dims.push_back({stride, last});
            end += stride * last;
            if (stride > row) { row = stride; rows = stride * last; }
        }
        within = (int64_t)(end - base) - rows;
    }
    bool shares(const View& o) const {
        if (base >= o.end || o.base >= end) return false;
        const int64_t gap = (int64_t)(o.base - base);
        if (row && row == o.row && gap >= 0 && gap % row >= within && gap % row + o.within <= row) return false;      // other columns of the same rows
        Terms terms;
        for (const auto& d : dims) terms.push_back({d.first, 0, d.second});
        for (const auto& d : o.dims) terms.push_back({d.first, -d.second, 0});
        return Sum(std::move(terms)).reaches(gap - (width - 1), gap + (o.width - 1));
    }
    bool shares_with_itself() const {                // two indexes, apart first in dimension k, for one byte
        for (size_t k = 0; k < dims.size(); ++k) {
            Terms terms = {{dims[k].first, 1, dims[k].second}};
            for (size_t j = k + 1; j < dims.size(); ++j) terms.push_back({dims[j].first, -dims[j].second, dims[j].second});
            if (Sum(std::move(terms)).reaches(-(width - 1), width - 1)) return true;
        }
        return false;
    }
};

// whether memory of a view that is clipped in a copy is given twice (among tensors without gaps the native call checks that)
bool shares_elements(const vector<const Tensor*>& ts) {
    if (std::none_of(ts.begin(), ts.end(), [](const Tensor* t) { return t->is_neg() || !t->is_non_overlapping_and_dense(); })) return false;
    vector<View> v;
    v.reserve(ts.size());
    for (const Tensor* t : ts)
        if (t->numel()) v.emplace_back(*t);
    std::sort(v.begin(), v.end(), [](const View& a, const View& b) { return a.base < b.base; });
    for (size_t i = 0; i < v.size(); ++i) {
        if (v[i].copied && v[i].shares_with_itself()) return true;
        for (size_t j = i + 1; j < v.size() && v[j].base < v[i].end; ++j)
            if ((v[i].copied || v[j].copied) && v[i].shares(v[j])) return true;
    }
    return false;
}

Tensor clip_by_global_norm_(const py::object& tensors, double clip_norm, const py::object& use) {
    const char* name = "clip_by_global_norm_";
    clip_value(clip_norm, name);
    List l = take_list(tensors, "tensors", false);
    const vector<const Tensor*> given = l.t;
    const Tensor use_norm = given_norm(use, l.device, name);
    for (const Tensor* t : given) {
        no_gradient(*t, name);
        for (int64_t i = 0; i < t->dim() && t->numel(); ++i)            // slices of something larger: clipped in a copy
            if (t->stride(i) == 0 && t->size(i) > 1) fail(string(name) + ": an expanded tensor cannot be written in place");
    }
    vector<const Tensor*> memory = given;
    if (use_norm.defined()) memory.push_back(&use_norm);
    if (shares_elements(memory)) fail(string(name) + ": the same elements are given twice (views that overlap)");
    const Call call(l.device);
    l.make_dense();
    const Tensor norm = clip(call, Described(l), pointers(l), clip_norm, use_norm, name);
    at::NoGradGuard no_grad;
    for (size_t i = 0; i < given.size(); ++i) {
        if (given[i] != l.t[i]) given[i]->copy_(*l.t[i]);
        else written(*given[i]);
    }
    return norm;
}

// whether two tensors of one shape hold their elements in the same order
bool laid_out_alike(const Tensor& a, const Tensor& b) {
    for (int64_t i = 0; i < a.dim(); ++i)
        if (a.size(i) > 1 && a.stride(i) != b.stride(i)) return false;
    return true;
}

Tensor adam_clip_update_(const py::object& params, const py::object& grads, const py::object& exp_avgs, const py::object& exp_avg_sqs, double lr,
                         double beta1, double beta2, double eps, long long step, double clip_norm, const py::object& use, bool skip_nonfinite) {
    const char* name = "adam_clip_update_";
    clip_value(clip_norm, name);
    const List p = take_list(params, "params", true), m = take_list(exp_avgs, "exp_avgs", true), v = take_list(exp_avg_sqs, "exp_avg_sqs", true);
    List g = take_list(grads, "grads", false);
    const size_t n = p.t.size();
    if (g.t.size() != n || m.t.size() != n || v.t.size() != n)
        fail(string(name) + ": lists of " + std::to_string(n) + ", " + std::to_string(g.t.size()) + ", " + std::to_string(m.t.size()) + " and " +
             std::to_string(v.t.size()) + " tensors");
    if (g.device != p.device || m.device != p.device || v.device != p.device) fail(string(name) + ": lists on several devices");
    const Tensor use_norm = given_norm(use, p.device, name);
    const Call call(p.device);
    vector<size_t> reordered;                                          // gradients that a copy takes the place of
    for (size_t i = 0; i < n; ++i) {
        const Tensor &pi = *p.t[i], &gi = *g.t[i], &mi = *m.t[i], &vi = *v.t[i];
        no_gradient_but_of_leaves(pi, name);
        for (const Tensor* t : {&gi, &mi, &vi}) no_gradient(*t, name);
        if (pi.sizes() != gi.sizes() || pi.sizes() != mi.sizes() || pi.sizes() != vi.sizes())
            fail(string(name) + ": shapes " + shape_of(pi) + ", " + shape_of(gi) + ", " + shape_of(mi) + ", " + shape_of(vi));
        if (!pi.is_non_overlapping_and_dense() || !laid_out_alike(pi, mi) || !laid_out_alike(pi, vi) || pi.is_neg() || mi.is_neg() || vi.is_neg())
            fail(string(name) + ": params and moments must be dense and laid out alike");
        if (gi.is_neg() || !laid_out_alike(pi, gi)) reordered.push_back(i);
    }
    for (size_t i : reordered) {                                       // the native check sees the copies
        const View gi(*g.t[i]);
        for (const List* l : {&p, &m, &v})
            for (const Tensor* t : l->t)
                if (g.t[i]->numel() && t->numel() && gi.shares(View(*t))) fail(string(name) + ": a gradient shares elements with params or moments");
    }
    for (size_t i : reordered) {                                       // a gradient in another order
        Tensor same = at::empty_strided(p.t[i]->sizes(), p.t[i]->strides(), g.t[i]->options().requires_grad(false));
        at::NoGradGuard no_grad;
        same.copy_(*g.t[i]);
        g.replace(i, same);
    }
    const Described d(g);
    vector<const void*> pp = pointers(p), pm = pointers(m), pv = pointers(v);
    const size_t nbytes = use_norm.defined() ? 0 : uhm_multi_workspace_bytes(d.count());
    const Tensor norm = call.scalar(), ws = call.bytes(nbytes);
    check(uhm_adam_clip_update((float* const*)pp.data(), d.p.data(), (float* const*)pm.data(), (float* const*)pv.data(), d.numel.data(), d.dtype.data(),
                               d.count(), lr, beta1, beta2, eps, step, (float)clip_norm, skip_nonfinite ? UHM_SKIP_NONFINITE : 0,
                               (const float*)at_of(use_norm), (float*)norm.data_ptr(), at_of(ws), nbytes, call.stream), name);
    for (const List* l : {&p, &m, &v})
        for (const Tensor* t : l->t) written(*t);
    return norm;
}

// ---- 8-bit rows ---------------------------------------------------------------------------------------------------------------
int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

struct Rows {                                        // x [..., K] as rows of contiguous elements that do not overlap
    Tensor t;                                        // 2-D
    int64_t rows, K, ld;
};

Rows rows_of(const Tensor& given, const char* name) {
    if (given.dim() < 1 || given.size(-1) < 1) fail(string(name) + " must be [..., K] with K >= 1 (got " + shape_of(given) + ")");
    Rows r;
    r.K = given.size(-1);
    r.rows = given.numel() / r.K;
    r.t = plain(given);
    if (r.t.dim() != 2) r.t = r.t.reshape({r.rows, r.K});
    if (r.rows && ((r.t.stride(1) != 1 && r.K > 1) || (r.rows > 1 && r.t.stride(0) < r.K))) r.t = r.t.contiguous();
    r.ld = std::max(r.t.stride(0), r.K);             // (a single row may carry any stride)
    return r;
}

// rows as uhm_int8_matmul takes them: aligned, each readable up to the next multiple of 16.  quantize_rows gives such rows; others are copied
Rows int8_rows(const Tensor& given, const char* name) {
    if (given.scalar_type() != at::kChar) fail(string(name) + " must be int8 (got " + type_name(given.scalar_type()) + ")");
    Rows r = rows_of(given, name);
    if (r.rows == 1) r.ld = round_up(r.K, 16);
    const int64_t behind = (int64_t)r.t.storage().nbytes() - r.t.storage_offset();
    if (r.rows && (r.ld % 16 || r.ld > (1 << 23) || (uintptr_t)r.t.data_ptr() % 16 || behind < (r.rows - 1) * r.ld + round_up(r.K, 16))) {
        r.ld = round_up(r.K, 128);
        const Tensor copy = at::zeros({r.rows, r.ld}, r.t.options()).narrow(1, 0, r.K);
        copy.copy_(r.t);
        r.t = copy;
    }
    return r;
}

Tensor values(const py::object& o, int64_t count, at::Device device, const char* name) {
    const Tensor& t = tensor(o, name);
    if (t.scalar_type() != at::kFloat) fail(string(name) + " must be float32 (got " + type_name(t.scalar_type()) + ")");
    if (t.numel() != count || t.device() != device) fail(string(name) + " must hold " + std::to_string(count) + " values on " + device.str());
    return plain(t).contiguous();
}

struct Weight {
    Rows w;
    Tensor scale, bias;
};
Weight weight_of(const py::object& weight, const py::object& scale, const py::object& bias, int64_t K, at::Device device, const char* name) {
    Weight r;
    const Tensor& t = tensor(weight, "weight");
    r.w = int8_rows(t, "weight");
    if (t.dim() != 2 || r.w.K != K || t.device() != device)
        fail("weight must be int8 [N, " + std::to_string(K) + "] on " + device.str() + " (got " + shape_of(t) + " on " + t.device().str() + ")");
    r.scale = values(scale, r.w.rows, device, "weight_scale");
    no_gradient(r.scale, name);
    if (!bias.is_none()) {
        r.bias = values(bias, r.w.rows, device, "bias");
        no_gradient(r.bias, name);
    }
    return r;
}

vector<int64_t> with_last(const Tensor& x, int64_t last) {
    vector<int64_t> s(x.sizes().begin(), x.sizes().end());
    s.back() = last;
    return s;
}

Rows float_rows(const py::object& x, int* dtype, const char* name) {
    const Tensor& t = tensor(x, "x");
    *dtype = dtype_of(t);
    Rows r = rows_of(t, "x");
    if (*dtype < 0) fail("x: " + type_name(t.scalar_type()) + " is not supported (float32, bfloat16, float16)");
    no_gradient(t, name);
    return r;
}

py::tuple quantize_rows(const py::object& x) {
    int dtype;
    const Rows r = float_rows(x, &dtype, "quantize_rows");
    const Tensor& given = THPVariable_Unpack(x.ptr());
    const Call call(given.device());
    const int64_t ld = round_up(r.K, 128);                            // rows start on 128 bytes
    vector<int64_t> lead(given.sizes().begin(), given.sizes().end() - 1);
    const Tensor q = at::empty(with_last(given, ld), call.options.dtype(at::kChar)), scale = at::empty(lead, call.options.dtype(at::kFloat));
    check(uhm_quantize_rows(r.t.data_ptr(), dtype, r.ld, (int8_t*)q.data_ptr(), ld, (float*)scale.data_ptr(), r.rows, r.K, call.stream), "uhm_quantize_rows");
    return py::make_tuple(q.narrow(-1, 0, r.K), scale);
}

Tensor int8_matmul(const py::object& x, const py::object& x_scale, const py::object& weight, const py::object& weight_scale, const py::object& bias,
                   bool relu, const py::object& out_dtype) {
    const char* name = "int8_matmul";
    at::ScalarType type = at::kFloat;
    if (THPDtype_Check(out_dtype.ptr())) type = reinterpret_cast<THPDtype*>(out_dtype.ptr())->scalar_type;
    if (!THPDtype_Check(out_dtype.ptr()) || (type != at::kFloat && type != at::kBFloat16 && type != at::kHalf))
        fail("int8_matmul: out_dtype " + string(py::str(out_dtype)) + " is not supported (float32, bfloat16, float16)");
    const Tensor& given = tensor(x, "x");
    const Rows a = int8_rows(given, "x");
    const Tensor scale = values(x_scale, a.rows, given.device(), "x_scale");
    no_gradient(scale, name);
    const Weight w = weight_of(weight, weight_scale, bias, a.K, given.device(), name);
    const Call call(given.device());
    const Tensor out = at::empty(with_last(given, w.w.rows), call.options.dtype(type));
    const size_t nbytes = uhm_int8_matmul_workspace_bytes(a.rows, w.w.rows, a.K);
    const Tensor ws = call.bytes(nbytes);
    check(uhm_int8_matmul((const int8_t*)a.t.data_ptr(), a.ld, (const float*)scale.data_ptr(), (const int8_t*)w.w.t.data_ptr(), w.w.ld,
                          (const float*)w.scale.data_ptr(), (const float*)at_of(w.bias), out.data_ptr(), dtype_of(out), a.rows, w.w.rows, a.K,
                          relu ? UHM_RELU : 0, at_of(ws), nbytes, call.stream), "uhm_int8_matmul");
    return out;
}

Tensor int8_linear(const py::object& x, const py::object& weight, const py::object& weight_scale, const py::object& bias, bool relu) {
    const char* name = "int8_linear";
    int dtype;
    const Rows r = float_rows(x, &dtype, name);
    const Tensor& given = THPVariable_Unpack(x.ptr());
    const Weight w = weight_of(weight, weight_scale, bias, r.K, given.device(), name);
    const Call call(given.device());
    const Tensor out = at::empty(with_last(given, w.w.rows), call.options.dtype(given.scalar_type()));
    const size_t nbytes = uhm_int8_linear_workspace_bytes(r.rows, w.w.rows, r.K);
    const Tensor ws = call.bytes(nbytes);
    check(uhm_int8_linear(r.t.data_ptr(), dtype, r.ld, (const int8_t*)w.w.t.data_ptr(), w.w.ld, (const float*)w.scale.data_ptr(), (const float*)at_of(w.bias),
                          out.data_ptr(), r.rows, w.w.rows, r.K, relu ? UHM_RELU : 0, at_of(ws), nbytes, call.stream), "uhm_int8_linear");
    return out;
}

}  // namespace

PYBIND11_MODULE(_uhm_torch, m) {
    m.def("abi_version", [] { return uhm_abi_version(); });
    m.def("set_error", [](py::object cls) { error_class = cls.release().ptr(); });
    m.def("global_norm", torch::wrap_pybind_function(&global_norm));
    m.def("clip_by_global_norm", torch::wrap_pybind_function(&clip_by_global_norm));
    m.def("clip_by_global_norm_", torch::wrap_pybind_function(&clip_by_global_norm_));
    m.def("adam_clip_update_", torch::wrap_pybind_function(&adam_clip_update_));
    m.def("quantize_rows", torch::wrap_pybind_function(&quantize_rows));
    m.def("int8_matmul", torch::wrap_pybind_function(&int8_matmul));
    m.def("int8_linear", torch::wrap_pybind_function(&int8_linear));
}
