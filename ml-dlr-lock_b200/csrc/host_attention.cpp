// Host side of the attention operators, native because a decode step calls them for every layer and the kernels of a small
// batch take 3 us: checks, outputs and argument structs cost 20 to 40 us per call in Python (197 us for a training step with
// its Python autograd function), about 6 here with the launch.
//
//   bind(addresses)          the C-ABI functions to call, in the order of Library
//   paged_plan(...), qk_norm_rope(...), qk_norm_rope_append(...), paged_attention(...)
//
// The operators take the arguments of their namesakes in dlr_lock_b200/attention.py, in its order, and return what those
// return (tuples), or the C-ABI's code as an int where that is not 0, or None for anything that they do not take as it is:
// arguments that are wrong, tensors that are not laid out as the kernels read them, tensors of another device than the
// current one.  The caller then names what is wrong, or brings the arguments into shape and calls again.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cmath>
#include <cstring>
#include <limits>
#include <optional>

#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include "dlr_b200.h"

namespace {

struct Library {
    decltype(&dlrb200_paged_plan) paged_plan;
    decltype(&dlrb200_qk_norm_rope) norm_rope;
    decltype(&dlrb200_qk_norm_rope_backward) norm_rope_backward;
    decltype(&dlrb200_qk_norm_rope_backward_workspace_bytes) norm_rope_backward_workspace;
    decltype(&dlrb200_paged_attention) paged_attention;
    decltype(&dlrb200_paged_attention_workspace_bytes) paged_attention_workspace;
    decltype(&dlrb200_strerror) strerror;
} g_lib;
bool g_bound = false;

PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long a[7];
    if (!PyArg_ParseTuple(args, "KKKKKKK", a, a + 1, a + 2, a + 3, a + 4, a + 5, a + 6)) return nullptr;
    static_assert(sizeof(Library) == sizeof(a), "one address per function");
    std::memcpy(&g_lib, a, sizeof(a));
    g_bound = true;
    Py_RETURN_NONE;
}

constexpr int64_t kMostInt = std::numeric_limits<int>::max(), kMostRows = int64_t(1) << 30;

// The tensor behind an argument; null for anything else.
const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

bool plain(const at::Tensor& t, int device) {
    return t.is_cuda() && t.get_device() == device && t.layout() == at::kStrided && t.has_storage() && !t.is_neg();
}

// int32 and contiguous
bool ints(const at::Tensor& t, int device) { return plain(t, device) && t.scalar_type() == at::kInt && t.is_contiguous(); }

bool aligned(const at::Tensor& t, uintptr_t to) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % to == 0; }

// The device of a tensor if it is the current one, else -1.
int device_of(const at::Tensor* t) {
    if (!g_bound || !t || !t->is_cuda()) return -1;
    const int device = t->get_device();
    return c10::cuda::current_device() == device ? device : -1;
}

void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(c10::DeviceIndex(device)).stream(); }

int* as_ints(const at::Tensor& t) { return static_cast<int*>(t.data_ptr()); }

// Whether one carries a tangent of forward-mode differentiation, which no_grad leaves on.
bool has_tangent(std::initializer_list<const at::Tensor*> tensors) {
    for (const at::Tensor* t : tensors)
        if (t && t->defined() && t->_fw_grad(0).defined()) return true;
    return false;
}

bool wants_grad(std::initializer_list<const at::Tensor*> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const at::Tensor* t : tensors)
        if (t && t->defined() && t->requires_grad()) return true;
    return false;
}

// Result of a call: the outputs, or the code.
PyObject* result(int code, std::initializer_list<at::Tensor> outputs, bool tuple) {
    if (code != DLRB200_OK) return PyLong_FromLong(code);
    if (!tuple) return THPVariable_Wrap(*outputs.begin());
    PyObject* const t = PyTuple_New(Py_ssize_t(outputs.size()));
    if (!t) return nullptr;
    Py_ssize_t i = 0;
    for (const at::Tensor& o : outputs) {
        PyObject* const item = THPVariable_Wrap(o);
        if (!item) {
            Py_DECREF(t);
            return nullptr;
        }
        PyTuple_SET_ITEM(t, i++, item);
    }
    return t;
}

bool integer(PyObject* o, int64_t* v) {
    if (!PyLong_CheckExact(o)) return false;
    int overflow = 0;
    *v = PyLong_AsLongLongAndOverflow(o, &overflow);
    return overflow == 0;
}

bool real(PyObject* o, double* v) {
    if (PyFloat_Check(o)) *v = PyFloat_AS_DOUBLE(o);
    else if (int64_t i; integer(o, &i)) *v = double(i);
    else return false;
    return true;
}

// The truth of a flag; false with Python's error set where it has none.
bool flag(PyObject* o, bool* v) {
    const int is = PyObject_IsTrue(o);
    *v = is == 1;
    return is >= 0;
}

// (a dimension of one has any stride)
int64_t step_of(const at::Tensor& t, int64_t i) { return t.size(i) == 1 ? 0 : t.stride(i); }

// ---- plan ------------------------------------------------------------------------------------------------------------------
// (lengths, new_tokens, block_table, free_pages, n_free, page_size, width, rows, finished, in_place)
PyObject* paged_plan(PyObject*, PyObject* const* o, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 10) Py_RETURN_NONE;
    bool in_place;
    if (!flag(o[9], &in_place)) return nullptr;
    const at::Tensor *lengths = tensor(o[0]), *fresh = tensor(o[1]), *table = tensor(o[2]), *pages = tensor(o[3]), *count = tensor(o[4]);
    const at::Tensor* finished = o[8] == Py_None ? nullptr : tensor(o[8]);
    if (!lengths || !fresh || !table || !pages || !count || (o[8] != Py_None && !finished)) Py_RETURN_NONE;
    const int device = device_of(lengths);
    if (device < 0 || !ints(*lengths, device) || !ints(*fresh, device) || !ints(*pages, device) || !ints(*count, device) ||
        !plain(*table, device) || table->scalar_type() != at::kInt)
        Py_RETURN_NONE;
    if (lengths->dim() != 1 || fresh->dim() != 1 || table->dim() != 2 || pages->dim() != 1 || count->dim() != 1) Py_RETURN_NONE;
    const int64_t n = lengths->size(0), columns = table->size(1);
    if (fresh->size(0) != n || table->size(0) != n || count->size(0) != 1 || n > DLRB200_MAX_PLAN_REQUESTS || columns > kMostInt) Py_RETURN_NONE;
    if (table->numel() > 0 && (table->stride(1) != 1 || (n > 1 && table->stride(0) < columns))) Py_RETURN_NONE;
    if (finished && (!plain(*finished, device) || !finished->is_contiguous() || finished->dim() != 1 || finished->size(0) != n ||
                     (finished->scalar_type() != at::kBool && finished->scalar_type() != at::kByte)))
        Py_RETURN_NONE;
    int64_t page_size, width = 0, rows = 0;
    if (!integer(o[5], &page_size) || page_size < 16 || page_size > kMostInt || (page_size & (page_size - 1)) ||
        pages->size(0) > kMostInt / page_size)
        Py_RETURN_NONE;
    if (o[6] != Py_None) {
        if (!integer(o[6], &width) || width < 1 || width > kMostInt || width * n > kMostRows) Py_RETURN_NONE;
        if (o[7] != Py_None && (!integer(o[7], &rows) || rows != width * n)) Py_RETURN_NONE;
        rows = width * n;
    } else if (!integer(o[7], &rows) || rows < 0 || rows > kMostRows) {
        Py_RETURN_NONE;
    }
    at::Tensor slots, positions, starts, lengths_out, count_out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const at::Tensor all = at::empty({2 * rows + 2 * n + 2}, lengths->options());
        // vectors over parts of it, made directly (a narrow() costs 0.4 us, five of them a quarter of the call)
        auto part = [&](int64_t first, int64_t size) {
            at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
            t.unsafeGetTensorImpl()->set_storage_offset(first);
            t.unsafeGetTensorImpl()->set_sizes_contiguous({size});
            return t;
        };
        slots = part(0, rows);
        positions = part(rows, rows);
        starts = part(2 * rows, n + 1);
        lengths_out = in_place ? *lengths : part(2 * rows + n + 1, n);
        count_out = in_place ? *count : part(2 * rows + 2 * n + 1, 1);
    }
    dlrb200_plan_step s{};
    s.lengths = as_ints(*lengths), s.new_tokens = as_ints(*fresh);
    s.finished = finished ? static_cast<const unsigned char*>(finished->const_data_ptr()) : nullptr;
    s.block_table = as_ints(*table), s.table_stride = table->stride(0), s.free_pages = as_ints(*pages), s.n_free = as_ints(*count);
    s.slots = as_ints(slots), s.positions = as_ints(positions), s.starts = as_ints(starts);
    s.lengths_out = as_ints(lengths_out), s.n_free_out = as_ints(count_out);
    s.requests = int(n), s.columns = int(columns), s.pages = int(pages->size(0)), s.page_size = int(page_size);
    s.width = int(width), s.rows = int(rows);
    return result(g_lib.paged_plan(&s, stream_of(device)), {slots, positions, starts, lengths_out, count_out}, true);
    END_HANDLE_TH_ERRORS
}

// ---- norm and rotation -----------------------------------------------------------------------------------------------------
// A (..., heads, dim) tensor as (tokens, heads, dim), where it lies.
struct Rows {
    void* data;
    int64_t tokens, token, head;
};

bool rows_of(const at::Tensor& t, Rows* r) {
    const int64_t n = t.dim();
    if (n < 2 || (t.stride(n - 1) != 1 && t.size(n - 1) > 1)) return false;
    r->data = t.data_ptr();
    r->head = step_of(t, n - 2);
    r->tokens = 1;
    r->token = 0;
    if (t.numel() == 0) {                    // (no strides to agree on)
        r->tokens = r->head = 0;
        return true;
    }
    for (int64_t i = n - 3; i >= 0; --i) {
        if (t.size(i) == 1) continue;
        if (r->tokens == 1) r->token = t.stride(i);
        else if (t.stride(i) != r->token * r->tokens) return false;
        r->tokens *= t.size(i);
    }
    return r->token % 4 == 0 && r->head % 4 == 0 && aligned(t, 8);
}

bool same_leading(const at::Tensor& a, const at::Tensor& b, int64_t n) {
    for (int64_t i = 0; i < n; ++i)
        if (a.size(i) != b.size(i)) return false;
    return true;
}

// What the forward and the backward have in common.
struct Heads {
    at::Tensor q, k, q_weight, k_weight, cos, sin, positions;     // undefined: no weight
    int device = -1, type = 0;
    int64_t dim = 0, half = 0;
    Rows q_rows, k_rows;
    double eps = 0;
    bool interleaved = false, weights_f32 = false;

    bool check() {
        device = device_of(&q);
        if (device < 0 || !plain(q, device) || !plain(k, device) || !plain(cos, device) || !plain(sin, device) || !plain(positions, device))
            return false;
        const auto t = q.scalar_type();
        if ((t != at::kBFloat16 && t != at::kHalf) || k.scalar_type() != t) return false;
        type = t == at::kHalf ? DLRB200_F16 : DLRB200_BF16;
        const int64_t n = q.dim();
        if (n < 2 || k.dim() != n || !same_leading(q, k, n - 2) || q.size(n - 1) != k.size(n - 1)) return false;
        dim = q.size(n - 1);
        if (dim % 8 || dim <= 0 || dim > 256 || q.size(n - 2) < 1 || k.size(n - 2) < 1 || q.size(n - 2) > kMostInt || k.size(n - 2) > kMostInt)
            return false;
        if (!rows_of(q, &q_rows) || !rows_of(k, &k_rows)) return false;
        if (cos.dim() != 2 || sin.dim() != 2 || cos.size(0) != sin.size(0) || cos.size(1) != sin.size(1) || cos.scalar_type() != at::kFloat ||
            sin.scalar_type() != at::kFloat || !cos.is_contiguous() || !sin.is_contiguous() || !aligned(cos, 16) || !aligned(sin, 16))
            return false;
        half = cos.size(1);
        if (half % 4 || 2 * half > dim || cos.size(0) > kMostInt) return false;
        if ((positions.scalar_type() != at::kInt && positions.scalar_type() != at::kLong) || positions.dim() != n - 2 ||
            !same_leading(positions, q, n - 2))
            return false;
        const at::Tensor* given[2] = {&q_weight, &k_weight};
        at::ScalarType type_of_weights = at::kFloat;
        bool any = false;
        for (const at::Tensor* w : given) {
            if (!w->defined()) continue;
            if (!plain(*w, device) || w->dim() != 1 || w->size(0) != dim || !w->is_contiguous() || !aligned(*w, 16)) return false;
            if (w->scalar_type() != t && w->scalar_type() != at::kFloat) return false;
            if (any && w->scalar_type() != type_of_weights) return false;
            type_of_weights = w->scalar_type();
            any = true;
        }
        weights_f32 = any && type_of_weights == at::kFloat;
        if (wants_grad({&cos, &sin}) || has_tangent({&q, &k, &q_weight, &k_weight, &cos, &sin})) return false;
        // (the host framework's positions are those of one row, expanded over the batch)
        if (!positions.is_contiguous()) {
            at::AutoDispatchBelowADInplaceOrView below;
            positions = positions.contiguous();
        }
        return true;
    }

    dlrb200_norm_rope_args args() const {
        dlrb200_norm_rope_args a{};
        a.q = q_rows.data, a.q_token = q_rows.token, a.q_head = q_rows.head;
        a.k = k_rows.data, a.k_token = k_rows.token, a.k_head = k_rows.head;
        a.q_weight = q_weight.defined() ? q_weight.data_ptr() : nullptr;
        a.k_weight = k_weight.defined() ? k_weight.data_ptr() : nullptr;
        a.cos = static_cast<const float*>(cos.data_ptr()), a.sin = static_cast<const float*>(sin.data_ptr());
        a.positions = positions.data_ptr(), a.tokens = q_rows.tokens;
        a.q_heads = int(q.size(q.dim() - 2)), a.k_heads = int(k.size(k.dim() - 2));
        a.dim = int(dim), a.half = int(half), a.table_rows = int(cos.size(0)), a.type = type;
        a.weights_f32 = weights_f32, a.positions_64 = positions.scalar_type() == at::kLong, a.interleaved = interleaved;
        a.eps = float(eps);
        return a;
    }
};

void succeed(int code, const char* what) {
    TORCH_CHECK(code == DLRB200_OK, what, ": ", g_lib.strerror(code));
}

// q_out and k_out
std::pair<at::Tensor, at::Tensor> turned(const Heads& h) {
    at::AutoDispatchBelowADInplaceOrView below;
    at::Tensor q_out = at::empty(h.q.sizes(), h.q.options()), k_out = at::empty(h.k.sizes(), h.k.options());
    dlrb200_norm_rope_args a = h.args();
    a.q_out = q_out.data_ptr(), a.k_out = k_out.data_ptr();
    succeed(g_lib.norm_rope(&a, stream_of(h.device)), "dlrb200_qk_norm_rope");
    return {q_out, k_out};
}

struct NormRope : torch::autograd::Function<NormRope> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k,
                                                  const std::optional<at::Tensor>& q_weight, const std::optional<at::Tensor>& k_weight,
                                                  const Heads* h) {
        auto out = turned(*h);
        // without a norm the gradient does not depend on the input
        ctx->save_for_backward({q_weight ? q : at::Tensor(), k_weight ? k : at::Tensor(), q_weight.value_or(at::Tensor()),
                                k_weight.value_or(at::Tensor()), h->cos, h->sin, h->positions});
        ctx->saved_data["eps"] = h->eps;
        ctx->saved_data["interleaved"] = h->interleaved;
        return {out.first, out.second};
    }

    // What was saved may have gone through hooks: other layouts are brought back, anything else is refused.
    static void check_saved(int device, const at::Tensor (&grads)[2], at::Tensor* q, at::Tensor* k, at::Tensor* q_weight, at::Tensor* k_weight,
                            at::Tensor* cos, at::Tensor* sin, at::Tensor* positions) {
        const int64_t n = grads[0].dim(), dim = grads[0].size(n - 1);
        const auto type = grads[0].scalar_type();
        const auto back = [&](at::Tensor* t, bool as_given) {
            TORCH_CHECK(t->is_cuda() && t->get_device() == device && t->layout() == at::kStrided && t->has_storage() && as_given,
                        "qk_norm_rope: a saved tensor came back on another device, or with another type or shape");
            *t = t->resolve_neg().contiguous();
            if (!aligned(*t, 16)) *t = t->clone(at::MemoryFormat::Contiguous);
        };
        for (int i = 0; i < 2; ++i) {
            at::Tensor *const x = i ? k : q, *const w = i ? k_weight : q_weight;
            if (x->defined() && (!plain(*x, device) || x->scalar_type() != type || x->sizes() != grads[i].sizes() || !fits(*x)))
                back(x, x->scalar_type() == type && x->sizes() == grads[i].sizes());
            if (w->defined()) back(w, (w->scalar_type() == type || w->scalar_type() == at::kFloat) && w->dim() == 1 && w->size(0) == dim);
        }
        back(cos, cos->scalar_type() == at::kFloat && cos->dim() == 2 && cos->size(1) % 4 == 0 && 2 * cos->size(1) <= dim);
        back(sin, sin->scalar_type() == at::kFloat && sin->sizes() == cos->sizes());
        back(positions, (positions->scalar_type() == at::kInt || positions->scalar_type() == at::kLong) &&
                            positions->sizes() == grads[0].sizes().slice(0, size_t(n - 2)));
        TORCH_CHECK(!q_weight->defined() || !k_weight->defined() || q_weight->scalar_type() == k_weight->scalar_type(),
                    "qk_norm_rope: the saved weights came back with two types");
    }

    static bool fits(const at::Tensor& t) {
        Rows r;
        return rows_of(t, &r);
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        at::Tensor q = saved[0], k = saved[1], q_weight = saved[2], k_weight = saved[3], cos = saved[4], sin = saved[5], positions = saved[6];
        bool twice = false;
        torch::autograd::variable_list out(5);
        {
            for (const at::Tensor& t : grads) twice = twice || (at::GradMode::is_enabled() && t.requires_grad());
            for (const at::Tensor& t : saved) twice = twice || (at::GradMode::is_enabled() && t.defined() && t.requires_grad());
            at::AutoDispatchBelowAutograd below;
            const c10::DeviceGuard guard(grads[0].device());
            const int device = grads[0].get_device();
            Rows g[2], x[2] = {};
            at::Tensor kept[2];
            for (int i = 0; i < 2; ++i) {
                kept[i] = grads[i].resolve_neg();
                if (!rows_of(kept[i], &g[i])) {
                    kept[i] = kept[i].clone(at::MemoryFormat::Contiguous);
                    TORCH_CHECK(rows_of(kept[i], &g[i]), "qk_norm_rope: gradients of unexpected shape");
                }
            }
            check_saved(device, kept, &q, &k, &q_weight, &k_weight, &cos, &sin, &positions);
            if (q.defined()) TORCH_CHECK(rows_of(q, &x[0]), "qk_norm_rope: saved queries of unexpected layout");
            if (k.defined()) TORCH_CHECK(rows_of(k, &x[1]), "qk_norm_rope: saved keys of unexpected layout");
            for (int i = 0; i < 2; ++i) out[i] = at::empty(kept[i].sizes(), kept[i].options().memory_format(at::MemoryFormat::Contiguous));
            dlrb200_norm_rope_grad_args a{};
            at::Tensor workspace;
            const int64_t n = kept[0].dim(), dim = kept[0].size(n - 1);
            for (int i = 0; i < 2; ++i) {
                const at::Tensor& w = i ? k_weight : q_weight;
                if (!w.defined()) continue;
                out[2 + i] = at::empty(w.sizes(), w.options());
                (i ? a.k_weight : a.q_weight) = w.data_ptr();
                (i ? a.dk_weight : a.dq_weight) = out[2 + i].data_ptr();
                a.weights_f32 = w.scalar_type() == at::kFloat;
                if (workspace.defined()) continue;
                a.workspace_bytes = g_lib.norm_rope_backward_workspace(int(dim));
                workspace = at::empty({int64_t(a.workspace_bytes)}, w.options().dtype(at::kByte));
                a.workspace = workspace.data_ptr();
            }
            a.q = x[0].data, a.q_token = x[0].token, a.q_head = x[0].head;
            a.k = x[1].data, a.k_token = x[1].token, a.k_head = x[1].head;
            a.q_grad = g[0].data, a.qg_token = g[0].token, a.qg_head = g[0].head;
            a.k_grad = g[1].data, a.kg_token = g[1].token, a.kg_head = g[1].head;
            a.cos = static_cast<const float*>(cos.data_ptr()), a.sin = static_cast<const float*>(sin.data_ptr());
            a.positions = positions.data_ptr(), a.dq = out[0].data_ptr(), a.dk = out[1].data_ptr();
            a.tokens = g[0].tokens, a.q_heads = int(kept[0].size(n - 2)), a.k_heads = int(kept[1].size(n - 2));
            a.dim = int(dim), a.half = int(cos.size(1)), a.table_rows = int(cos.size(0));
            a.type = kept[0].scalar_type() == at::kHalf ? DLRB200_F16 : DLRB200_BF16;
            a.positions_64 = positions.scalar_type() == at::kLong, a.interleaved = ctx->saved_data["interleaved"].toBool();
            a.eps = float(ctx->saved_data["eps"].toDouble());
            succeed(g_lib.norm_rope_backward(&a, stream_of(device)), "dlrb200_qk_norm_rope_backward");
        }
        if (twice) {                         // a graph of the gradient was asked for: there is none, and using it says so
            torch::autograd::variable_list some;
            for (at::Tensor& t : out)
                if (t.defined()) some.push_back(t.requires_grad_(true));
            auto error = std::make_shared<torch::autograd::DelayedError>("qk_norm_rope can be differentiated once only", int64_t(some.size()));
            some = (*error)(std::move(some));
            size_t i = 0;
            for (at::Tensor& t : out)
                if (t.defined()) t = some[i++];
        }
        return out;
    }
};

bool heads_from(PyObject* const* o, Heads* h) {
    const at::Tensor *q = tensor(o[0]), *k = tensor(o[1]), *cos = tensor(o[4]), *sin = tensor(o[5]), *positions = tensor(o[6]);
    if (!q || !k || !cos || !sin || !positions) return false;
    for (int i = 2; i < 4; ++i) {
        if (o[i] == Py_None) continue;
        const at::Tensor* const w = tensor(o[i]);
        if (!w) return false;
        (i == 2 ? h->q_weight : h->k_weight) = *w;
    }
    h->q = *q, h->k = *k, h->cos = *cos, h->sin = *sin, h->positions = *positions;
    return true;
}

// (q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
PyObject* qk_norm_rope(PyObject*, PyObject* const* o, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    Heads h;
    if (n_args != 9 || !heads_from(o, &h) || !real(o[7], &h.eps)) Py_RETURN_NONE;
    if (!flag(o[8], &h.interleaved)) return nullptr;
    if (!h.check()) Py_RETURN_NONE;
    if (!wants_grad({&h.q, &h.k, &h.q_weight, &h.k_weight})) {
        auto out = turned(h);
        return result(DLRB200_OK, {out.first, out.second}, true);
    }
    const auto given = [](const at::Tensor& w) { return w.defined() ? std::optional<at::Tensor>(w) : std::nullopt; };
    auto out = NormRope::apply(h.q, h.k, given(h.q_weight), given(h.k_weight), static_cast<const Heads*>(&h));
    return result(DLRB200_OK, {out[0], out[1]}, true);
    END_HANDLE_TH_ERRORS
}

struct Cache {
    void* data;
    int64_t page, head, slot;
};

// a (pages, heads, page tokens, dim) cache like `like`, strides multiples of `multiple` elements
bool cache_of(const at::Tensor& t, int device, at::ScalarType type, int64_t heads, int64_t dim, int64_t multiple, Cache* c) {
    if (!plain(t, device) || t.scalar_type() != type || t.dim() != 4 || t.size(1) != heads || t.size(3) != dim) return false;
    const int64_t page = t.size(2);
    if (page < 16 || page > kMostInt || (page & (page - 1)) || t.size(0) > kMostInt / page) return false;
    *c = {t.data_ptr(), step_of(t, 0), step_of(t, 1), t.stride(2)};
    return t.numel() == 0 || (t.stride(3) == 1 && c->page % multiple == 0 && c->head % multiple == 0 && c->slot % multiple == 0 &&
                              aligned(t, uintptr_t(2 * multiple)));
}

// An expanded cache, of which slots lie in one place: nothing to write to.
bool expanded(const at::Tensor& t) {
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.size(i) > 1 && t.stride(i) == 0) return t.numel() > 0;
    return false;
}

// (q, k, q_weight, k_weight, cos, sin, positions, v, slots, k_cache, v_cache, eps, interleaved, return_keys)
PyObject* qk_norm_rope_append(PyObject*, PyObject* const* o, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    Heads h;
    if (n_args != 14 || !heads_from(o, &h) || !real(o[11], &h.eps)) Py_RETURN_NONE;
    const at::Tensor *v = tensor(o[7]), *slots = tensor(o[8]), *k_cache = tensor(o[9]), *v_cache = tensor(o[10]);
    if (!v || !slots || !k_cache || !v_cache) Py_RETURN_NONE;
    bool keys;
    if (!flag(o[12], &h.interleaved) || !flag(o[13], &keys)) return nullptr;
    if (!h.check() || wants_grad({&h.q, &h.k, v, &h.q_weight, &h.k_weight, k_cache, v_cache}) || has_tangent({v, k_cache, v_cache})) Py_RETURN_NONE;
    Rows v_rows;
    Cache kc, vc;
    const int64_t n = h.q.dim(), kv_heads = h.k.size(n - 2);
    if (!plain(*v, h.device) || v->scalar_type() != h.k.scalar_type() || v->sizes() != h.k.sizes() || !rows_of(*v, &v_rows)) Py_RETURN_NONE;
    if (!ints(*slots, h.device) || slots->dim() != n - 2 || !same_leading(*slots, h.q, n - 2)) Py_RETURN_NONE;
    if (!cache_of(*k_cache, h.device, h.q.scalar_type(), kv_heads, h.dim, 4, &kc) || !cache_of(*v_cache, h.device, h.q.scalar_type(), kv_heads, h.dim, 4, &vc) ||
        k_cache->sizes() != v_cache->sizes() || expanded(*k_cache) || expanded(*v_cache))
        Py_RETURN_NONE;
    at::Tensor q_out, k_out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        q_out = at::empty(h.q.sizes(), h.q.options());
        if (keys) k_out = at::empty(h.k.sizes(), h.k.options());
    }
    dlrb200_norm_rope_args a = h.args();
    a.v = v_rows.data, a.v_token = v_rows.token, a.v_head = v_rows.head;
    a.q_out = q_out.data_ptr(), a.k_out = keys ? k_out.data_ptr() : nullptr, a.slots = as_ints(*slots);
    a.k_cache = kc.data, a.kc_page = kc.page, a.kc_head = kc.head, a.kc_slot = kc.slot;
    a.v_cache = vc.data, a.vc_page = vc.page, a.vc_head = vc.head, a.vc_slot = vc.slot;
    a.pages = int(k_cache->size(0)), a.page_size = int(k_cache->size(2));
    const int code = g_lib.norm_rope(&a, stream_of(h.device));
    return keys ? result(code, {q_out, k_out}, true) : result(code, {q_out}, false);
    END_HANDLE_TH_ERRORS
}

// ---- attention -------------------------------------------------------------------------------------------------------------
// (q, k_cache, v_cache, block_table, lengths, scale)
PyObject* paged_attention(PyObject*, PyObject* const* o, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 6) Py_RETURN_NONE;
    const at::Tensor *q = tensor(o[0]), *k_cache = tensor(o[1]), *v_cache = tensor(o[2]), *table = tensor(o[3]), *lengths = tensor(o[4]);
    if (!q || !k_cache || !v_cache || !table || !lengths) Py_RETURN_NONE;
    const int device = device_of(q);
    if (device < 0 || !plain(*q, device) || q->dim() != 3 || k_cache->dim() != 4 || wants_grad({q, k_cache, v_cache}) ||
        has_tangent({q, k_cache, v_cache}))
        Py_RETURN_NONE;
    const auto type = q->scalar_type();
    const int64_t n = q->size(0), heads = q->size(1), dim = q->size(2), kv_heads = k_cache->size(1);
    if ((type != at::kBFloat16 && type != at::kHalf) || (dim != 64 && dim != 96 && dim != 128 && dim != 256) || kv_heads < 1 || heads < 1 ||
        heads % kv_heads || n > kMostInt / heads)
        Py_RETURN_NONE;
    if (q->numel() > 0 && (q->stride(2) != 1 || step_of(*q, 0) % 2 || step_of(*q, 1) % 2 || !aligned(*q, 4))) Py_RETURN_NONE;
    Cache kc, vc;
    if (!cache_of(*k_cache, device, type, kv_heads, dim, 8, &kc) || !cache_of(*v_cache, device, type, kv_heads, dim, 8, &vc) ||
        k_cache->sizes() != v_cache->sizes())
        Py_RETURN_NONE;
    if (!ints(*lengths, device) || lengths->dim() != 1 || lengths->size(0) != n) Py_RETURN_NONE;
    if (!plain(*table, device) || table->scalar_type() != at::kInt || table->dim() != 2 || table->size(0) != n ||
        (table->numel() > 0 && table->stride(1) != 1) || table->size(1) > (1 << 30) / k_cache->size(2))
        Py_RETURN_NONE;
    double scale = 1.0 / std::sqrt(double(dim));
    if (o[5] != Py_None && !real(o[5], &scale)) Py_RETURN_NONE;
    at::Tensor out, workspace;
    const size_t bytes = g_lib.paged_attention_workspace(int(heads), int(kv_heads), int(dim));
    {
        at::AutoDispatchBelowADInplaceOrView below;
        out = at::empty({n, heads, dim}, q->options());
        workspace = at::empty({int64_t(bytes)}, lengths->options().dtype(at::kByte));
    }
    dlrb200_paged_attention_args a{};
    a.q = q->data_ptr(), a.q_request = step_of(*q, 0), a.q_head = step_of(*q, 1);
    a.k_cache = kc.data, a.kc_page = kc.page, a.kc_head = kc.head, a.kc_slot = kc.slot;
    a.v_cache = vc.data, a.vc_page = vc.page, a.vc_head = vc.head, a.vc_slot = vc.slot;
    a.block_table = as_ints(*table), a.table_stride = table->stride(0), a.lengths = as_ints(*lengths);
    a.out = out.data_ptr(), a.workspace = workspace.data_ptr(), a.workspace_bytes = bytes;
    a.requests = int(n), a.heads = int(heads), a.kv_heads = int(kv_heads), a.dim = int(dim), a.columns = int(table->size(1));
    a.pages = int(k_cache->size(0)), a.page_size = int(k_cache->size(2)), a.type = type == at::kHalf ? DLRB200_F16 : DLRB200_BF16;
    a.scale = float(scale);
    return result(g_lib.paged_attention(&a, stream_of(device)), {out}, false);
    END_HANDLE_TH_ERRORS
}

}  // namespace

PyMethodDef kAttentionMethods[] = {{"bind", bind, METH_VARARGS, nullptr},
                                   {"paged_plan", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paged_plan)), METH_FASTCALL, nullptr},
                                   {"qk_norm_rope", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(qk_norm_rope)), METH_FASTCALL, nullptr},
                                   {"qk_norm_rope_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(qk_norm_rope_append)),
                                    METH_FASTCALL, nullptr},
                                   {"paged_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paged_attention)), METH_FASTCALL,
                                    nullptr},
                                   {nullptr, nullptr, 0, nullptr}};
