// ternainfer_amd._native: the host path of one library call as one native function -- checks, output tensors, current
// stream, launch(es).  In Python (ctypes) that path costs 13 - 16 us a call, several times what a decode-sized launch
// takes on the device; here 2 - 3 us.  PyTorch stays what it is elsewhere in the package: the owner of device memory
// and streams.  The library is the one _lib.py loads; init() binds its entry points by name.
//
// Every function checks shapes and element counts before anything is enqueued (the C ABI takes pointers on trust) and
// raises ValueError, or TypeError where an argument is no tensor; the tensors' types and devices are the caller's business
// where linear.py does not state otherwise.  What follows the checks -- allocations, copies, launches, which may wait for the
// device -- runs without the interpreter's lock, as the same calls do from Python.
#include <dlfcn.h>

#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <ATen/EmptyTensor.h>
#include <ATen/hip/impl/HIPCachingAllocatorMasqueradingAsCUDA.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <cstdarg>
#include <optional>
#include <vector>

#include "../../include/ternaspmm.h"

namespace {

#define TERNA_ENTRY_POINTS(X)                                                                                          \
    X(bitlinear_TernaSpMM)                                                                                             \
    X(bitlinear_TernaSpMM_bf16)                                                                                        \
    X(bitlinear_TernaSpMM_bf16_decode)                                                                                 \
    X(bitlinear_TernaSpMM_bf16_prefill)                                                                                \
    X(bitlinear_TernaSpMM_packed_ws)                                                                                   \
    X(bitlinear_TernaSpMM_bf16_packed_ws)                                                                              \
    X(bitlinear_TernaSpMM_quant)                                                                                       \
    X(bitlinear_TernaSpMM_quant_packed)                                                                                \
    X(ternaspmm_quant_rows_linear)                                                                                     \
    X(ternaspmm_quant_rows_linear_packed)                                                                              \
    X(ternaspmm_qkv_rope_linear)                                                                                       \
    X(ternaspmm_prefill_attention_rows)                                                                                \
    X(ternaspmm_gate_linear)                                                                                           \
    X(ternaspmm_residual_linear)                                                                                       \
    X(ternaspmm_quant_input)                                                                                           \
    X(ternaspmm_rmsnorm_quant)                                                                                         \
    X(ternaspmm_rmsnorm_quant_ahead)                                                                                   \
    X(ternaspmm_relu2_mul_rmsnorm_quant)                                                                               \
    X(ternaspmm_relu2_mul_rmsnorm_quant_ahead)                                                                         \
    X(ternaspmm_fused_linear)                                                                                          \
    X(ternaspmm_quant_from_stats)                                                                                      \
    X(ternaspmm_rope_kv_store)                                                                                         \
    X(ternaspmm_prefill_attention)                                                                                     \
    X(ternaspmm_rope_decode_attention)                                                                                 \
    X(ternaspmm_rope_decode_attention_stats)                                                                           \
    X(ternaspmm_step_attention)                                                                                        \
    X(ternaspmm_step_attention_merge)                                                                                  \
    X(ternaspmm_attention_partial_bytes)                                                                               \
    X(ternaspmm_attention_workspace_bytes)                                                                             \
    X(ternaspmm_attention_merge)                                                                                       \
    X(ternaspmm_attention_merge_rmsnorm_quant)                                                                         \
    X(ternaspmm_row_stats_count)                                                                                       \
    X(ternaspmm_step_inputs)                                                                                           \
    X(ternaspmm_prompt_inputs)                                                                                         \
    X(ternaspmm_decode_step_bytes)                                                                                     \
    X(ternaspmm_decode_step)                                                                                           \
    X(ternaspmm_rotary)                                                                                                \
    X(ternaspmm_kv4_store)                                                                                             \
    X(ternaspmm_kv4_rows)                                                                                              \
    X(ternaspmm_kv4_workspace_bytes)                                                                                   \
    X(ternaspmm_kv4_attention)                                                                                         \
    X(ternaspmm_kv4_step)                                                                                              \
    X(ternaspmm_token_logprobs_workspace_bytes)                                                                        \
    X(ternaspmm_token_logprobs)                                                                                        \
    X(ternaspmm_draft_tree)                                                                                            \
    X(ternaspmm_tree_attention_workspace_bytes)                                                                        \
    X(ternaspmm_tree_attention)                                                                                        \
    X(ternaspmm_tree_accept_workspace_bytes)                                                                           \
    X(ternaspmm_tree_accept)                                                                                           \
    X(ternaspmm_cache_move)                                                                                            \
    X(ternaspmm_int8_bytes)                                                                                            \
    X(ternaspmm_int8_quantise)                                                                                         \
    X(ternaspmm_int8_pack)                                                                                             \
    X(ternaspmm_int8_linear_workspace_bytes)                                                                           \
    X(ternaspmm_int8_linear)
struct Library {
#define X(name) decltype(&::name) name = nullptr;
    TERNA_ENTRY_POINTS(X)
#undef X
} lib;

struct Refused : std::exception {};            // a Python error is set

// From its construction to end() other Python threads run: no Python object is touched and nothing refused in between.
class Unlocked {
    PyThreadState* state = PyEval_SaveThread();

public:
    Unlocked() = default;
    Unlocked(const Unlocked&) = delete;
    ~Unlocked() { end(); }
    void end()
    {
        if (state != nullptr) PyEval_RestoreThread(state);
        state = nullptr;
    }
};

// an argument that is a tensor
const at::Tensor& tensor(PyObject* o)
{
    if (!THPVariable_CheckExact(o) && !THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "expected a torch.Tensor, got %s", Py_TYPE(o)->tp_name);
        throw Refused();
    }
    return THPVariable_Unpack(o);
}
// ... or None
const at::Tensor* optional(PyObject* o) { return o == Py_None ? nullptr : &tensor(o); }

[[noreturn]] void refuse(const char* format, ...)
{
    va_list args;
    va_start(args, format);
    PyErr_FormatV(PyExc_ValueError, format, args);
    va_end(args);
    throw Refused();
}

long long integer(PyObject* o)
{
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Refused();
    return v;
}
int integer32(PyObject* o)
{
    const long long v = integer(o);
    if (v < INT32_MIN || v > INT32_MAX) refuse("integer argument %lld out of range", v);
    return static_cast<int>(v);
}
float real(PyObject* o)
{
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Refused();
    return static_cast<float>(v);
}

bool truth(PyObject* o)
{
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Refused();                // (a tensor of several elements has none)
    return v != 0;
}

template <typename T = void>
T* data(const at::Tensor* t) { return t == nullptr ? nullptr : static_cast<T*>(t->data_ptr()); }

void check_matrix(const char* who, const at::Tensor& x)
{
    if (x.dim() != 2) refuse("%s: expected a [M, K] tensor, got %d dimensions", who, static_cast<int>(x.dim()));
    if (x.size(0) > INT32_MAX || x.size(1) > INT32_MAX) refuse("%s: tensor too large", who);
}
void check_numel(const char* who, const char* name, const at::Tensor* t, int64_t want)
{
    if (t != nullptr && t->numel() != want)
        refuse("%s: %s has %lld elements, expected %lld", who, name, static_cast<long long>(t->numel()), static_cast<long long>(want));
}
void check_weight(const char* who, const at::Tensor& packed, const at::Tensor& ws, int ws_num, int64_t n, int64_t k)
{
    if (static_cast<int64_t>(packed.numel() * packed.element_size()) < n * k / 4 || ws.numel() < ws_num)
        refuse("%s: packed weight or weight scales too small for this shape", who);
}

// The caching allocator under the device name that torch's Python side uses.
c10::Allocator* device_allocator() { return c10::hip::HIPCachingAllocatorMasqueradingAsCUDA::get(); }

// A device tensor straight from the caching allocator: torch's dispatcher costs more than the allocation (1.2 against 0.6 us).
at::Tensor make(at::IntArrayRef shape, at::ScalarType type, const at::Tensor& like)
{
    if (like.is_cuda() && like.device().index() == c10::hip::current_device())
        return at::Tensor(at::detail::empty_generic(shape, device_allocator(), c10::DispatchKeySet(c10::DispatchKey::CUDA), type, std::nullopt));
    return at::empty(shape, at::TensorOptions(type).device(like.device()));
}
// Several int64 results in one allocation (a tensor more is 0.15 us, an allocation 0.6).
struct Longs {
    at::Tensor all;
    int64_t used = 0;

    Longs(int64_t count, const at::Tensor& like) : all(make({count}, at::kLong, like)) {}
    at::Tensor take(at::IntArrayRef shape)
    {
        at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
        t.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
        t.unsafeGetTensorImpl()->set_storage_offset(used);
        used += t.numel();
        return t;
    }
};
terna_stream stream() { return c10::hip::getCurrentHIPStream().stream(); }

// int8 rows and their bf16 scales, for the length of one call: (rows [m][k], scales [m]) on the current device
struct QuantRows {
    c10::DataPtr held;
    int8_t* q;
    terna_bf16* s;
};
QuantRows make_quant_rows(int64_t m, int64_t k)
{
    QuantRows r{device_allocator()->allocate(m * k + 2 * m), nullptr, nullptr};     // k is even: the scales are aligned
    r.q = static_cast<int8_t*>(r.held.get());
    r.s = reinterpret_cast<terna_bf16*>(r.q + m * k);
    return r;
}

// Results: the end of an unlocked stretch.
PyObject* none(Unlocked& unlocked)
{
    unlocked.end();
    Py_RETURN_NONE;
}
PyObject* wrap(at::Tensor t, Unlocked& unlocked)
{
    unlocked.end();
    return THPVariable_Wrap(std::move(t));
}
PyObject* wrap_or_none(at::Tensor t) { return t.defined() ? THPVariable_Wrap(std::move(t)) : Py_NewRef(Py_None); }
template <typename... Ts>
PyObject* pack(Unlocked& unlocked, Ts&&... items)
{
    unlocked.end();
    PyObject* tuple = PyTuple_New(sizeof...(items));
    Py_ssize_t i = 0;
    (PyTuple_SET_ITEM(tuple, i++, wrap_or_none(std::forward<Ts>(items))), ...);
    return tuple;
}

// A module's activations: bf16 rows on the current device.  False: something the native path does not take (another type, an
// empty batch ...), linear.py goes on.
bool bf16_rows(const at::Tensor& x, int64_t* m, int64_t* k)
{
    if (!x.is_cuda() || x.scalar_type() != at::kBFloat16 || x.dim() < 1) return false;
    *k = x.size(-1);
    if (*k < 64 || x.numel() == 0 || x.device().index() != c10::hip::current_device()) return false;
    *m = x.numel() / *k;
    return *m <= INT32_MAX && *k <= INT32_MAX;
}
at::Tensor make_output(const at::Tensor& x, int64_t n)
{
    at::DimVector shape(x.sizes());
    shape.back() = n;
    return make(shape, at::kBFloat16, x);
}
void check_format(const char* who, const at::Tensor& bitmap, int64_t n, int64_t k)
{
    if (bitmap.numel() * 64 != n * k)
        refuse("%s: the weight's bitmap does not belong to a [%lld, %lld] matrix", who, static_cast<long long>(n), static_cast<long long>(k));
}

#define TERNA_FUNCTION(name, count)                                                                                    \
    PyObject* name##_body(PyObject* const* a);                                                                         \
    PyObject* name(PyObject*, PyObject* const* a, Py_ssize_t n)                                                        \
    {                                                                                                                  \
        HANDLE_TH_ERRORS                                                                                               \
        if (n != (count)) {                                                                                            \
            PyErr_Format(PyExc_TypeError, #name ": %d arguments expected", (count));                                   \
            return nullptr;                                                                                            \
        }                                                                                                              \
        try {                                                                                                          \
            return name##_body(a);                                                                                     \
        } catch (const Refused&) {                                                                                     \
            return nullptr;                                                                                            \
        }                                                                                                              \
        END_HANDLE_TH_ERRORS                                                                                           \
    }                                                                                                                  \
    PyObject* name##_body(PyObject* const* a)

// (x, packed | None, bitmap, tile offsets, median offsets, signs, ws, ws_num, out_features, workspace | None): SpBitLinear -- quantise
// the rows, then the int8 linear on the repacked weight or on the reference format.  None: x is not for this path.
TERNA_FUNCTION(bit_linear, 10)
{
    const at::Tensor &x = tensor(a[0]), &bitmap = tensor(a[2]), &offsets = tensor(a[3]), &median = tensor(a[4]), &signs = tensor(a[5]), &ws = tensor(a[6]);
    const at::Tensor *packed = optional(a[1]), *workspace = optional(a[9]);
    const int ws_num = integer32(a[7]);
    const int64_t n = integer32(a[8]);
    int64_t m, k;
    if (!bf16_rows(x, &m, &k) || k > 8192) Py_RETURN_NONE;
    if (packed != nullptr) check_weight("SpBitLinear", *packed, ws, ws_num, n, k);
    else check_format("SpBitLinear", bitmap, n, k);
    Unlocked unlocked;
    const at::Tensor rows = x.contiguous();
    at::Tensor out = make_output(x, n);
    const terna_stream st = stream();
    if (m <= 8) {                       // a few rows: both steps in one launch
        const int done = packed != nullptr ? lib.bitlinear_TernaSpMM_quant_packed(data<terna_bf16>(&rows), data(packed), data<terna_bf16>(&out),
                                                                                  data<terna_bf16>(&ws), ws_num, m, n, k, st)
                                           : lib.bitlinear_TernaSpMM_quant(data<terna_bf16>(&rows), data<uint64_t>(&bitmap), data<int>(&offsets),
                                                                           data<uint16_t>(&median), data<uint32_t>(&signs), data<terna_bf16>(&out),
                                                                           data<terna_bf16>(&ws), ws_num, m, n, k, st);
        if (done) return wrap(std::move(out), unlocked);
    }
    {                                   // ... or of more rows, where one round of workgroups covers the matrix
        const int done = packed != nullptr ? lib.ternaspmm_quant_rows_linear_packed(data<terna_bf16>(&rows), data(packed), data<terna_bf16>(&out),
                                                                                    data<terna_bf16>(&ws), ws_num, m, n, k, st)
                                           : lib.ternaspmm_quant_rows_linear(data<terna_bf16>(&rows), data<uint64_t>(&bitmap), data<int>(&offsets),
                                                                             data<uint16_t>(&median), data<uint32_t>(&signs), data<terna_bf16>(&out),
                                                                             data<terna_bf16>(&ws), ws_num, m, n, k, st);
        if (done) return wrap(std::move(out), unlocked);
    }
    QuantRows q = make_quant_rows(m, k);
    if (lib.ternaspmm_quant_input(data<terna_bf16>(&rows), q.q, q.s, m, k, st) != 0) return none(unlocked);
    if (packed != nullptr)
        lib.bitlinear_TernaSpMM_packed_ws(q.q, data(packed), data<terna_bf16>(&out), q.s, data<terna_bf16>(&ws), ws_num, m, n, k, 0,
                                          data(workspace), workspace != nullptr ? workspace->numel() : 0, st);
    else
        lib.bitlinear_TernaSpMM(q.q, data<uint64_t>(&bitmap), data<int>(&offsets), data<uint16_t>(&median), data<uint32_t>(&signs),
                                data<terna_bf16>(&out), q.s, data<terna_bf16>(&ws), ws_num, m, n, k, 7, data<int32_t>(workspace), st);
    return wrap(std::move(out), unlocked);
}

// (x, bitmap, tile offsets, median offsets, signs, scale, ws_num, out_features, route 0 auto / 1 decode / 2 prefill)
TERNA_FUNCTION(bit_linear_bf16, 9)
{
    const at::Tensor &x = tensor(a[0]), &bitmap = tensor(a[1]), &offsets = tensor(a[2]), &median = tensor(a[3]), &signs = tensor(a[4]), &scale = tensor(a[5]);
    const int ws_num = integer32(a[6]), route = integer32(a[8]);
    const int64_t n = integer32(a[7]);
    int64_t m, k;
    if (!bf16_rows(x, &m, &k)) Py_RETURN_NONE;
    check_format("TernaInfer_linear_bf16", bitmap, n, k);
    Unlocked unlocked;
    const at::Tensor rows = x.contiguous();
    at::Tensor out = make_output(x, n);
    const auto fn = route == 1 ? lib.bitlinear_TernaSpMM_bf16_decode : route == 2 ? lib.bitlinear_TernaSpMM_bf16_prefill : lib.bitlinear_TernaSpMM_bf16;
    fn(data<terna_bf16>(&rows), data<uint64_t>(&bitmap), data<int>(&offsets), data<uint16_t>(&median), data<uint32_t>(&signs),
       data<terna_bf16>(&out), data<float>(&scale), ws_num, m, n, k, 1, nullptr, stream());
    return wrap(std::move(out), unlocked);
}

// (x bf16 [..., K]) -> (int8 [..., K], bf16 [..., 1]), or None
TERNA_FUNCTION(quant_input, 1)
{
    const at::Tensor& x = tensor(a[0]);
    int64_t m, k;
    if (!bf16_rows(x, &m, &k)) Py_RETURN_NONE;
    Unlocked unlocked;
    const at::Tensor rows = x.contiguous();
    at::DimVector shape(x.sizes());
    at::Tensor q = make(shape, at::kChar, x);
    shape.back() = 1;
    at::Tensor s = make(shape, at::kBFloat16, x);
    if (lib.ternaspmm_quant_input(data<terna_bf16>(&rows), data<int8_t>(&q), data<terna_bf16>(&s), m, k, stream()) != 0) return none(unlocked);
    return pack(unlocked, std::move(q), std::move(s));
}

// (x int8 [M, K], s, packed, ws, ws_num, out_features, workspace | None), the weights' scales by the rule of M (route 0) or the decode rule (2)
PyObject* linear_packed_by(PyObject* const* a, int route)
{
    const char* who = "TernaInfer_linear_packed";
    const at::Tensor &x = tensor(a[0]), &s = tensor(a[1]), &packed = tensor(a[2]), &ws = tensor(a[3]);
    const at::Tensor* workspace = optional(a[6]);
    const int ws_num = integer32(a[4]);
    const int64_t n = integer32(a[5]);
    check_matrix(who, x);
    const int64_t m = x.size(0), k = x.size(1);
    check_numel(who, "s", &s, m);
    check_weight(who, packed, ws, ws_num, n, k);
    Unlocked unlocked;
    const at::Tensor rows = x.contiguous(), scales = s.contiguous();
    at::Tensor out = make({m, n}, at::kBFloat16, x);
    lib.bitlinear_TernaSpMM_packed_ws(data<int8_t>(&rows), data(&packed), data<terna_bf16>(&out), data<terna_bf16>(&scales), data<terna_bf16>(&ws),
                                      ws_num, m, n, k, route, data(workspace), workspace != nullptr ? workspace->numel() : 0, stream());
    return wrap(std::move(out), unlocked);
}
TERNA_FUNCTION(linear_packed, 7) { return linear_packed_by(a, 0); }
TERNA_FUNCTION(linear_packed_decode_rule, 7) { return linear_packed_by(a, 2); }

// (x bf16 [M, K], packed, scale fp32, ws_num, out_features, workspace | None)
TERNA_FUNCTION(linear_bf16_packed, 6)
{
    const char* who = "bf16 linear on a packed weight";
    const at::Tensor &x = tensor(a[0]), &packed = tensor(a[1]), &scale = tensor(a[2]);
    const at::Tensor* workspace = optional(a[5]);
    const int ws_num = integer32(a[3]);
    const int64_t n = integer32(a[4]);
    check_matrix(who, x);
    const int64_t m = x.size(0), k = x.size(1);
    check_weight(who, packed, scale, ws_num, n, k);
    Unlocked unlocked;
    const at::Tensor rows = x.contiguous();
    at::Tensor out = make({m, n}, at::kBFloat16, x);
    lib.bitlinear_TernaSpMM_bf16_packed_ws(data<terna_bf16>(&rows), data(&packed), data<terna_bf16>(&out), data<float>(&scale), ws_num, m, n, k, 0,
                                           data(workspace), workspace != nullptr ? workspace->numel() : 0, stream());
    return wrap(std::move(out), unlocked);
}

// (x, weight, eps, residual | None, quant) -> (xq, s, h) or (y, None, h)
TERNA_FUNCTION(rmsnorm_quant, 5)
{
    const char* who = "rmsnorm_quant";
    const at::Tensor &x = tensor(a[0]), &weight = tensor(a[1]);
    const at::Tensor* residual = optional(a[3]);
    const float eps = real(a[2]);
    check_matrix(who, x);
    const int64_t m = x.size(0), k = x.size(1);
    check_numel(who, "residual", residual, m * k);
    check_numel(who, "weight", &weight, k);
    const bool quant = PyObject_IsTrue(a[4]);
    Unlocked unlocked;
    const at::Tensor rows = x.contiguous();
    at::Tensor added, h = rows, q, s;
    if (residual != nullptr) {
        added = residual->contiguous();
        h = make({m, k}, at::kBFloat16, x);
    }
    q = make({m, k}, quant ? at::kChar : at::kBFloat16, x);
    if (quant) s = make({m}, at::kBFloat16, x);
    lib.ternaspmm_rmsnorm_quant(data<terna_bf16>(&rows), residual != nullptr ? data<terna_bf16>(&added) : nullptr,
                                residual != nullptr ? data<terna_bf16>(&h) : nullptr, data<terna_bf16>(&weight), eps,
                                quant ? nullptr : data<terna_bf16>(&q), quant ? data<int8_t>(&q) : nullptr, quant ? data<terna_bf16>(&s) : nullptr, m, k,
                                stream());
    return pack(unlocked, std::move(q), std::move(s), std::move(h));             // (x itself where it is neither added to nor copied)
}

// (x13, weight, eps, quant) -> (xq, s) or (y, None)
TERNA_FUNCTION(relu2_mul_rmsnorm_quant, 4)
{
    const char* who = "relu2_mul_rmsnorm_quant";
    const at::Tensor &x = tensor(a[0]), &weight = tensor(a[1]);
    const float eps = real(a[2]);
    check_matrix(who, x);
    const int64_t m = x.size(0), f = x.size(1) / 2;
    check_numel(who, "weight", &weight, f);
    const bool quant = PyObject_IsTrue(a[3]);
    Unlocked unlocked;
    const at::Tensor rows = x.contiguous();
    at::Tensor q = make({m, f}, quant ? at::kChar : at::kBFloat16, x), s;
    if (quant) s = make({m}, at::kBFloat16, x);
    lib.ternaspmm_relu2_mul_rmsnorm_quant(data<terna_bf16>(&rows), data<terna_bf16>(&weight), eps, quant ? nullptr : data<terna_bf16>(&q),
                                          quant ? data<int8_t>(&q) : nullptr, quant ? data<terna_bf16>(&s) : nullptr, m, f, stream());
    return pack(unlocked, std::move(q), std::move(s));
}

void check_stats(const char* who, const at::Tensor& stats, int64_t m)
{
    if (stats.scalar_type() != at::kFloat || stats.dim() != 3 || stats.size(0) != m || stats.size(2) != 2 || !stats.is_contiguous())
        refuse("%s: stats must be a contiguous fp32 [M, count, 2] tensor", who);
}

// (h, stats, norm_weight, eps) -> (xq, s)
TERNA_FUNCTION(quant_from_stats, 4)
{
    const char* who = "quant_from_stats";
    const at::Tensor &h = tensor(a[0]), &stats = tensor(a[1]), &weight = tensor(a[2]);
    const float eps = real(a[3]);
    check_matrix(who, h);
    const int64_t m = h.size(0), k = h.size(1);
    check_numel(who, "norm_weight", &weight, k);
    check_stats(who, stats, m);
    Unlocked unlocked;
    const at::Tensor rows = h.contiguous();
    at::Tensor q = make({m, k}, at::kChar, h), s = make({m}, at::kBFloat16, h);
    const int rc = lib.ternaspmm_quant_from_stats(data<terna_bf16>(&rows), data<float>(&stats), stats.size(1), data<terna_bf16>(&weight), eps,
                                                  data<int8_t>(&q), data<terna_bf16>(&s), m, k, stream());
    unlocked.end();
    if (rc != 0) refuse("%s: unsupported shape M=%d K=%d", who, static_cast<int>(m), static_cast<int>(k));
    return pack(unlocked, std::move(q), std::move(s));
}

// (x, norm_weight | None, eps, packed, ws, ws_num, out_features, in_features, stats | None, attention splits (0: none), head_dim,
//  quantised | None, epilogue, residual | None, next_norm_weight | None, want_raw, publish) -> the five tensors of
// linear.fused_linear, or None where the library does not take the combination
PyObject* chained_linear(const char* who, bool own_stats, PyObject* const* a)
{
    const at::Tensor &x = tensor(a[0]), &packed = tensor(a[3]), &ws = tensor(a[4]);
    const at::Tensor *weight = optional(a[1]), *stats = optional(a[8]), *quantised = optional(a[11]), *residual = optional(a[13]), *next_weight = optional(a[14]);
    const int64_t n = integer32(a[6]), k = integer32(a[7]);
    ternaspmm_fused_linear_desc d{};
    d.eps = real(a[2]);
    d.ws_num = integer32(a[5]);
    d.attention_splits = integer32(a[9]);
    d.head_dim = integer32(a[10]);
    d.epilogue = integer32(a[12]);
    at::Tensor rows = x, scales, stream_in, out, stats_out, raw, xq, s;
    int64_t m = 1;
    if (d.attention_splits > 0) {
        d.prologue = TERNASPMM_PROLOGUE_ATTENTION;
    } else {
        check_matrix(who, x);
        m = x.size(0);
        if (x.size(1) != k) refuse("%s: expected a [M, %lld] tensor", who, static_cast<long long>(k));
        if (quantised != nullptr) {
            d.prologue = TERNASPMM_PROLOGUE_QUANTISED;
            check_numel(who, "s", quantised, m);
            if (x.scalar_type() != at::kChar || quantised->scalar_type() != at::kBFloat16)
                refuse("%s: quantised activations are int8 with bf16 scales", who);
        } else {
            d.prologue = stats == nullptr ? TERNASPMM_PROLOGUE_NORM : own_stats ? TERNASPMM_PROLOGUE_OWN_STATS : TERNASPMM_PROLOGUE_STATS;
            check_numel(who, "norm_weight", weight, k);
        }
    }
    check_weight(who, packed, ws, d.ws_num, n, k);
    d.M = m, d.N = n, d.K = k;
    d.packed = data(&packed), d.ws = data<terna_bf16>(&ws), d.norm_weight = data<terna_bf16>(weight);
    if (stats != nullptr) {
        check_stats(who, *stats, m);
        d.stats_in = data<float>(stats), d.stats_count = stats->size(1);
    }
    const int64_t columns = d.epilogue == TERNASPMM_EPILOGUE_GATE ? n / 2 : n;
    if (d.epilogue != TERNASPMM_EPILOGUE_STORE && (next_weight == nullptr || next_weight->numel() != columns))
        refuse("%s: a producing epilogue needs the next norm's weights", who);
    if (d.epilogue == TERNASPMM_EPILOGUE_RESIDUAL) {
        if (residual == nullptr || residual->numel() != m * n || residual->scalar_type() != at::kBFloat16)
            refuse("%s: the residual epilogue needs a bf16 [M, N] stream", who);
    }
    const bool want_raw = d.epilogue == TERNASPMM_EPILOGUE_RESIDUAL && PyObject_IsTrue(a[15]), publish = PyObject_IsTrue(a[16]);

    Unlocked unlocked;
    if (d.attention_splits <= 0) rows = x.contiguous();
    d.x = data(&rows);
    if (d.prologue == TERNASPMM_PROLOGUE_QUANTISED) {
        scales = quantised->contiguous();
        d.s_in = data<terna_bf16>(&scales);
    }
    if (d.epilogue == TERNASPMM_EPILOGUE_RESIDUAL) {
        stream_in = residual->contiguous();
        d.residual = data<terna_bf16>(&stream_in);
    }
    if (want_raw) {
        raw = make({m, n}, at::kBFloat16, packed);
        d.raw_out = data<terna_bf16>(&raw);
    }
    out = make({m, columns}, at::kBFloat16, packed);
    d.out = data<terna_bf16>(&out);
    if (d.epilogue != TERNASPMM_EPILOGUE_STORE) {
        stats_out = make({m, columns / 16, 2}, at::kFloat, packed);
        d.next_norm_weight = data<terna_bf16>(next_weight), d.stats_out = data<float>(&stats_out);
    }
    if (publish) {
        xq = make({m, k}, at::kChar, packed), s = make({m}, at::kBFloat16, packed);
        d.xq_out = data<int8_t>(&xq), d.s_out = data<terna_bf16>(&s);
    }
    if (lib.ternaspmm_fused_linear(&d, stream()) < 0) return none(unlocked);
    return pack(unlocked, std::move(out), std::move(stats_out), std::move(raw), std::move(xq), std::move(s));
}

TERNA_FUNCTION(fused_linear, 17) { return chained_linear("fused_linear", false, a); }
// The same where `stats` are the rows' own (TERNASPMM_PROLOGUE_OWN_STATS).
TERNA_FUNCTION(fused_linear_own_stats, 17) { return chained_linear("fused_linear_own_stats", true, a); }

// What the attention entry points read beside a block's new rows, checked against these and each other.
struct AttentionArgs {
    const at::Tensor &cos, &sin, &pos, &ck, &cv;
    int64_t heads, head_dim, batch, kv, slots, t;
    float scale;
    int adjacent;
    bool each;                     // every sequence has its own positions

    // a: cos, sin, pos, cache_k, cache_v, heads, head_dim, scale, adjacent; qkv is [new_rows = B * T, columns = (H + 2 KV) D]
    AttentionArgs(const char* who, PyObject* const* a, int64_t new_rows, int64_t columns)
        : cos(tensor(a[0])), sin(tensor(a[1])), pos(tensor(a[2])), ck(tensor(a[3])), cv(tensor(a[4])), heads(integer32(a[5])),
          head_dim(integer32(a[6])), scale(real(a[7])), adjacent(integer32(a[8]))
    {
        if (ck.dim() != 4 || ck.sizes() != cv.sizes() || ck.size(0) < 1 || ck.size(3) != head_dim || !ck.is_contiguous() || !cv.is_contiguous())
            refuse("%s: the caches are contiguous [B, KV, S, D] tensors of one shape", who);
        batch = ck.size(0), kv = ck.size(1), slots = ck.size(2), t = new_rows / batch;
        if (t < 1 || new_rows != batch * t || columns != (heads + 2 * kv) * head_dim)
            refuse("%s: qkv does not have the shape of its caches", who);
        each = pos.dim() == 2;
        const int64_t rows = each ? batch * t : t;
        if (pos.scalar_type() != at::kLong || pos.numel() != rows || !pos.is_contiguous())
            refuse("%s: positions are a contiguous int64 [T] or [B, T] tensor", who);
        if (cos.numel() < rows * (head_dim / 2) || sin.numel() != cos.numel() || cos.scalar_type() != at::kFloat || sin.scalar_type() != at::kFloat ||
            !cos.is_contiguous() || !sin.is_contiguous())
            refuse("%s: cos / sin are contiguous fp32 rows of D / 2, one per position", who);
    }
};
// the leading arguments of those entry points
#define TERNA_ATTENTION_INPUTS(qkv, g)                                                                                 \
    qkv, data<float>(&(g).cos), data<float>(&(g).sin), data<long long>(&(g).pos), (g).each

// the new rows of an attention call
const at::Tensor& new_rows(const char* who, PyObject* o)
{
    const at::Tensor& qkv = tensor(o);
    check_matrix(who, qkv);
    if (!qkv.is_contiguous()) refuse("%s: qkv is a contiguous tensor", who);
    return qkv;
}

// (qkv, the nine of AttentionArgs, attention): RoPE and cache write of T new tokens per sequence, and with `attention` the multi-token
// attention -> bf16 [B * T, H D]; without it the rotated q [B, H, T, D]
TERNA_FUNCTION(prompt_attention, 11)
{
    const char* who = "prompt_attention";
    const at::Tensor& qkv = new_rows(who, a[0]);
    const AttentionArgs g(who, a + 1, qkv.size(0), qkv.size(1));
    const bool attention = PyObject_IsTrue(a[10]);
    Unlocked unlocked;
    at::Tensor q = make({g.batch, g.heads, g.t, g.head_dim}, at::kBFloat16, qkv);
    const terna_stream st = stream();
    lib.ternaspmm_rope_kv_store(TERNA_ATTENTION_INPUTS(data<terna_bf16>(&qkv), g), data<terna_bf16>(&q), data<terna_bf16>(&g.ck), data<terna_bf16>(&g.cv), g.batch, g.t, g.heads,
                                g.kv, g.head_dim, g.slots, g.adjacent, st);
    if (!attention) return wrap(std::move(q), unlocked);
    at::Tensor o = make({g.batch * g.t, g.heads * g.head_dim}, at::kBFloat16, qkv);
    lib.ternaspmm_prefill_attention(data<terna_bf16>(&q), data<terna_bf16>(&g.ck), data<terna_bf16>(&g.cv), data<long long>(&g.pos), g.each,
                                    data<terna_bf16>(&o), g.batch, g.t, g.heads, g.kv, g.head_dim, g.slots, g.scale, st);
    return wrap(std::move(o), unlocked);
}

// (qkv, the nine of AttentionArgs, workspace | None, norm_weight | None, partial | None, splits): RoPE, cache write and attention of one new
// token per sequence -> (out bf16 [B, H D], None); with the norm's weights (out, its partial statistics [B, H, 2]); with a
// buffer for partial results these are all that is written -> None
TERNA_FUNCTION(decode_attention, 14)
{
    const char* who = "decode_attention";
    const at::Tensor& qkv = new_rows(who, a[0]);
    const AttentionArgs g(who, a + 1, qkv.size(0), qkv.size(1));
    const at::Tensor *workspace = optional(a[10]), *weight = optional(a[11]), *partial = optional(a[12]);
    if (g.t != 1) refuse("%s: one new token per sequence", who);
    const terna_stream st = stream();
    terna_bf16 *ck = data<terna_bf16>(&g.ck), *cv = data<terna_bf16>(&g.cv);
    if (partial != nullptr) {
        const long long need = lib.ternaspmm_attention_partial_bytes(g.batch, g.heads, g.head_dim);
        if (need < 0 || static_cast<long long>(partial->numel() * partial->element_size()) < need) refuse("%s: the partial buffer is too small", who);
        const int splits = integer32(a[13]);
        Unlocked unlocked;
        const int left = lib.ternaspmm_step_attention(TERNA_ATTENTION_INPUTS(data<terna_bf16>(&qkv), g), ck, cv, data<float>(partial), splits, g.batch, g.heads, g.kv,
                                                      g.head_dim, g.slots, g.scale, g.adjacent, nullptr, nullptr, nullptr, 0, st);
        if (left != 0) {
            unlocked.end();
            refuse("%s: one to eight splits, 65536 of all heads", who);
        }
        return none(unlocked);
    }
    check_numel(who, "norm_weight", weight, g.heads * g.head_dim);
    if (weight == nullptr && workspace != nullptr &&
        static_cast<long long>(workspace->numel() * workspace->element_size()) < lib.ternaspmm_attention_workspace_bytes(g.batch, g.heads, g.head_dim))
        refuse("%s: the workspace is too small", who);
    Unlocked unlocked;
    at::Tensor o = make({g.batch, g.heads * g.head_dim}, at::kBFloat16, qkv), stats;
    if (weight != nullptr) {
        stats = make({g.batch, g.heads, 2}, at::kFloat, qkv);
        const int left = lib.ternaspmm_rope_decode_attention_stats(TERNA_ATTENTION_INPUTS(data<terna_bf16>(&qkv), g), ck, cv, data<terna_bf16>(&o), g.batch, g.heads, g.kv,
                                                                   g.head_dim, g.slots, g.scale, g.adjacent, data<terna_bf16>(weight), data<float>(&stats), st);
        unlocked.end();
        if (left != g.heads) refuse("%s: ternaspmm_rope_decode_attention_stats refused the launch", who);
    } else {
        lib.ternaspmm_rope_decode_attention(TERNA_ATTENTION_INPUTS(data<terna_bf16>(&qkv), g), ck, cv, data<terna_bf16>(&o), g.batch, g.heads, g.kv, g.head_dim, g.slots, g.scale,
                                            g.adjacent, data(workspace), st);
    }
    return pack(unlocked, std::move(o), std::move(stats));
}

// A ternary matrix of a block as four arguments: packed, ws, ws_num, out_features.
struct BlockLinear {
    const at::Tensor &packed, &ws;
    int ws_num;
    int64_t n;
    BlockLinear(const char* who, PyObject* const* a, int64_t k) : packed(tensor(a[0])), ws(tensor(a[1])), ws_num(integer32(a[2])), n(integer32(a[3]))
    {
        check_weight(who, packed, ws, ws_num, n, k);
    }
};

// (x, pending | None, cos, sin, pos, cache_k, cache_v, heads, head_dim, scale, adjacent, eps, attention workspace | (partial results, splits) | None, linear workspace | None,
//  attention_norm, attn_sub_norm, ffn_norm, ffn_sub_norm, wqkv [4], wo [4], w13 [4], w2 [4], interleaved w13 | None) -> (stream, pending; None where the stream has it): a whole block on int8
// activations with its norms as launches of their own (prompt pass, decode steps of many sequences): the nine launches and nothing
// else.  Called one by one from Python they cost 53 us of host time, more than they take on the device up to a hundred tokens.
TERNA_FUNCTION(block, 35)
{
    const char* who = "block";
    const at::Tensor& x = tensor(a[0]);
    const at::Tensor *pending = optional(a[1]), *attn_work = nullptr, *partial = nullptr, *work = optional(a[13]), *interleaved = optional(a[34]);
    int splits = 1;
    if (PyTuple_Check(a[12])) {
        if (PyTuple_GET_SIZE(a[12]) != 2) refuse("%s: (partial results, splits)", who);
        partial = &tensor(PyTuple_GET_ITEM(a[12], 0));
        splits = integer32(PyTuple_GET_ITEM(a[12], 1));
    } else {
        attn_work = optional(a[12]);
    }
    const at::Tensor *norm[4] = {&tensor(a[14]), &tensor(a[15]), &tensor(a[16]), &tensor(a[17])};
    const int64_t heads = integer32(a[7]), head_dim = integer32(a[8]);
    const float eps = real(a[11]);
    check_matrix(who, x);
    const int64_t m = x.size(0), dim = x.size(1), wide = heads * head_dim;
    const BlockLinear qkv_w(who, a + 18, dim), o_w(who, a + 22, wide), gate_w(who, a + 26, dim), down_w(who, a + 30, gate_w.n / 2);
    const int64_t ffn = gate_w.n / 2;
    if (interleaved != nullptr) check_weight(who, *interleaved, gate_w.ws, gate_w.ws_num, gate_w.n, dim);
    check_numel(who, "pending", pending, m * dim);
    check_numel(who, "attention_norm", norm[0], dim);
    check_numel(who, "attn_sub_norm", norm[1], wide);
    check_numel(who, "ffn_norm", norm[2], dim);
    check_numel(who, "ffn_sub_norm", norm[3], ffn);
    if (!x.is_contiguous() || (pending != nullptr && !pending->is_contiguous()) || x.scalar_type() != at::kBFloat16 || o_w.n != dim || down_w.n != dim)
        refuse("%s: the stream is a contiguous bf16 [M, dim] tensor, and the O and down projections return to it", who);

    const AttentionArgs g(who, a + 2, m, qkv_w.n);
    if (g.t == 1 && attn_work != nullptr && static_cast<long long>(attn_work->numel() * attn_work->element_size()) <
                                                lib.ternaspmm_attention_workspace_bytes(g.batch, heads, head_dim))
        refuse("%s: the attention workspace is too small", who);
    if (partial != nullptr && (g.t != 1 || splits < 1 || splits > 8 || g.batch * heads * splits > 65536 ||
                               static_cast<long long>(partial->numel() * partial->element_size()) < lib.ternaspmm_attention_partial_bytes(g.batch, heads, head_dim)))
        refuse("%s: split attention takes one new token, one to eight splits and a buffer that holds their results", who);

    Unlocked unlocked;
    // scratch of this call, in one piece: int8 rows and scales; then qkv, rotated queries, attention output and its projection,
    // in whose place the gate and up outputs go
    auto up = [](int64_t bytes) { return (bytes + 255) & ~int64_t{255}; };
    const int64_t q_bytes = up(m * std::max(std::max(dim, wide), ffn)), s_bytes = up(2 * m), qkv_bytes = up(2 * m * qkv_w.n), wide_bytes = up(2 * m * wide);
    const int64_t attn_bytes = qkv_bytes + 2 * wide_bytes + up(2 * m * dim);
    const c10::DataPtr held = device_allocator()->allocate(q_bytes + s_bytes + std::max(attn_bytes, up(2 * m * gate_w.n)));
    char* at_byte = static_cast<char*>(held.get());
    int8_t* xq = reinterpret_cast<int8_t*>(at_byte);
    terna_bf16* s = reinterpret_cast<terna_bf16*>(at_byte + q_bytes);
    auto rows = [&](int64_t offset) { return reinterpret_cast<terna_bf16*>(at_byte + q_bytes + s_bytes + offset); };
    terna_bf16 *qkv = rows(0), *q = rows(qkv_bytes), *o = rows(qkv_bytes + wide_bytes), *attn = rows(qkv_bytes + 2 * wide_bytes), *x13 = rows(0);

    at::Tensor mid = make({m, dim}, at::kBFloat16, x), out = make({m, dim}, at::kBFloat16, x), first;
    if (pending != nullptr) first = make({m, dim}, at::kBFloat16, x);
    const auto next = [](const BlockLinear& w, int64_t k) { return ternaspmm_next_linear{data(&w.packed), static_cast<int>(w.n), static_cast<int>(k), 0}; };
    const ternaspmm_next_linear next_qkv = next(qkv_w, dim), next_o = next(o_w, wide), next_down = next(down_w, ffn);
    ternaspmm_next_linear next_gate = next(gate_w, dim);
    if (interleaved != nullptr) next_gate.packed = data(interleaved), next_gate.gate = 1;
    const terna_bf16* in = data<terna_bf16>(&x);
    const terna_stream st = stream();
    terna_bf16 *ck = data<terna_bf16>(&g.ck), *cv = data<terna_bf16>(&g.cv);
    auto linear = [&](const BlockLinear& w, int64_t k, terna_bf16* to) {
        lib.bitlinear_TernaSpMM_packed_ws(xq, data(&w.packed), to, s, data<terna_bf16>(&w.ws), w.ws_num, m, w.n, k, 0, data(work),
                                          work != nullptr ? work->numel() : 0, st);
    };
    lib.ternaspmm_rmsnorm_quant_ahead(in, data<terna_bf16>(pending), pending != nullptr ? data<terna_bf16>(&first) : nullptr, data<terna_bf16>(norm[0]), eps, nullptr,
                                      xq, s, m, dim, &next_qkv, st);
    if (pending != nullptr) in = data<terna_bf16>(&first);
    // RoPE and the cache write in the projection's epilogue, for the attention that reads its rows
    const bool rows_in_place =
        g.t > 1 && g.adjacent && head_dim == 128 && heads == 4 * g.kv &&
        lib.ternaspmm_qkv_rope_linear(xq, data(&qkv_w.packed), qkv, s, data<terna_bf16>(&qkv_w.ws), qkv_w.ws_num, m, qkv_w.n, dim, data<float>(&g.cos),
                                      data<float>(&g.sin), data<long long>(&g.pos), g.each, ck, cv, g.t, heads, g.kv, head_dim, g.slots, st);
    if (!rows_in_place) linear(qkv_w, dim, qkv);
    if (rows_in_place) {
        if (!lib.ternaspmm_prefill_attention_rows(qkv, qkv_w.n, ck, cv, data<long long>(&g.pos), g.each, o, g.batch, g.t, heads, g.kv, head_dim, g.slots,
                                                  g.scale, st)) {
            unlocked.end();
            refuse("%s: the attention over the projection's rows refused the launch", who);
        }
    } else if (g.t > 1) {
        lib.ternaspmm_rope_kv_store(TERNA_ATTENTION_INPUTS(qkv, g), q, ck, cv, g.batch, g.t, heads, g.kv, head_dim, g.slots, g.adjacent, st);
        lib.ternaspmm_prefill_attention(q, ck, cv, data<long long>(&g.pos), g.each, o, g.batch, g.t, heads, g.kv, head_dim, g.slots, g.scale, st);
    } else if (partial != nullptr) {
        lib.ternaspmm_step_attention(TERNA_ATTENTION_INPUTS(qkv, g), ck, cv, data<float>(partial), splits, g.batch, heads, g.kv, head_dim, g.slots, g.scale, g.adjacent,
                                     nullptr, nullptr, nullptr, 0, st);
    } else {
        lib.ternaspmm_rope_decode_attention(TERNA_ATTENTION_INPUTS(qkv, g), ck, cv, o, g.batch, heads, g.kv, head_dim, g.slots, g.scale, g.adjacent,
                                            data(attn_work), st);
    }
    // the stream's sums in the epilogues of the projections that return to it, where these have one (elsewhere in the norm that follows)
    auto add_linear = [&](const BlockLinear& w, int64_t k, const terna_bf16* stream_in, terna_bf16* to) {
        return lib.ternaspmm_residual_linear(xq, data(&w.packed), to, s, data<terna_bf16>(&w.ws), w.ws_num, stream_in, m, w.n, k, data(work),
                                             work != nullptr ? work->numel() : 0, st) == 1;
    };
    if (partial == nullptr || lib.ternaspmm_step_attention_merge(data<float>(partial), splits, data<terna_bf16>(norm[1]), eps, nullptr, xq, s, g.batch, heads,
                                                                 head_dim, &next_o, st) != 0) {
        if (partial != nullptr) lib.ternaspmm_attention_merge(data<float>(partial), splits, o, g.batch, heads, head_dim, st);
        lib.ternaspmm_rmsnorm_quant_ahead(o, nullptr, nullptr, data<terna_bf16>(norm[1]), eps, nullptr, xq, s, m, wide, &next_o, st);
    }
    if (add_linear(o_w, wide, in, data<terna_bf16>(&mid))) {
        lib.ternaspmm_rmsnorm_quant_ahead(data<terna_bf16>(&mid), nullptr, nullptr, data<terna_bf16>(norm[2]), eps, nullptr, xq, s, m, dim, &next_gate, st);
    } else {
        linear(o_w, wide, attn);
        lib.ternaspmm_rmsnorm_quant_ahead(in, attn, data<terna_bf16>(&mid), data<terna_bf16>(norm[2]), eps, nullptr, xq, s, m, dim, &next_gate, st);
    }
    if (interleaved != nullptr && lib.ternaspmm_gate_linear(xq, data(interleaved), x13, s, data<terna_bf16>(&gate_w.ws), gate_w.ws_num, m, gate_w.n, dim, st)) {
        lib.ternaspmm_rmsnorm_quant_ahead(x13, nullptr, nullptr, data<terna_bf16>(norm[3]), eps, nullptr, xq, s, m, ffn, &next_down, st);
    } else {
        linear(gate_w, dim, x13);
        lib.ternaspmm_relu2_mul_rmsnorm_quant_ahead(x13, data<terna_bf16>(norm[3]), eps, nullptr, xq, s, m, ffn, &next_down, st);
    }
    if (add_linear(down_w, ffn, data<terna_bf16>(&mid), data<terna_bf16>(&out))) return pack(unlocked, std::move(out), at::Tensor());
    linear(down_w, ffn, data<terna_bf16>(&out));
    return pack(unlocked, std::move(mid), std::move(out));
}

// (packed, out_features, in_features, gate) | None: the linear behind a launch
ternaspmm_next_linear next_linear(const char* who, PyObject* o)
{
    if (o == Py_None) return ternaspmm_next_linear{};
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) refuse("%s: the next linear is (packed, out_features, in_features, gate)", who);
    const at::Tensor& packed = tensor(PyTuple_GET_ITEM(o, 0));
    const int n = integer32(PyTuple_GET_ITEM(o, 1)), k = integer32(PyTuple_GET_ITEM(o, 2));
    if (n < 1 || k < 1 || static_cast<int64_t>(packed.numel() * packed.element_size()) < static_cast<int64_t>(n) * k / 4)
        refuse("%s: the next linear's weight is too small", who);
    return ternaspmm_next_linear{data(&packed), n, k, PyObject_IsTrue(PyTuple_GET_ITEM(o, 3))};
}

PyObject* merge_norm_quant(const char* who, bool any_splits, const ternaspmm_next_linear& next, PyObject* const* a)
{
    const at::Tensor &partial = tensor(a[0]), &weight = tensor(a[4]);
    const int splits = integer32(a[1]), heads = integer32(a[2]), head_dim = integer32(a[3]), sequences = integer32(a[6]);
    const float eps = real(a[5]);
    const int64_t k = static_cast<int64_t>(heads) * head_dim;
    const long long held = partial.numel() * partial.element_size(), need = lib.ternaspmm_attention_partial_bytes(sequences, heads, head_dim);
    if (sequences < 1 || need < 0 || held < need) refuse("partial buffer of %lld bytes does not hold %d sequences", held, sequences);
    if (weight.numel() != k || weight.scalar_type() != at::kBFloat16) refuse("%s: the norm weight is a bf16 vector of heads * head_dim elements", who);
    const bool want_output = PyObject_IsTrue(a[7]);
    Unlocked unlocked;
    at::Tensor q = make({sequences, k}, at::kChar, partial), s = make({sequences}, at::kBFloat16, partial), o;
    if (want_output) o = make({sequences, k}, at::kBFloat16, partial);
    terna_bf16* const o_out = o.defined() ? data<terna_bf16>(&o) : nullptr;
    if ((any_splits ? lib.ternaspmm_step_attention_merge(data<float>(&partial), splits, data<terna_bf16>(&weight), eps, o_out, data<int8_t>(&q), data<terna_bf16>(&s),
                                                         sequences, heads, head_dim, &next, stream())
                    : lib.ternaspmm_attention_merge_rmsnorm_quant(data<float>(&partial), splits, data<terna_bf16>(&weight), eps, o_out, data<int8_t>(&q),
                                                                  data<terna_bf16>(&s), sequences, heads, head_dim, stream())) != 0)
        return none(unlocked);
    return pack(unlocked, std::move(q), std::move(s), std::move(o));
}

// (partial, splits, heads, head_dim, norm_weight, eps, sequences, want_output) -> (xq, s, o | None), or None
TERNA_FUNCTION(attention_merge_rmsnorm_quant, 8) { return merge_norm_quant("attention_merge_rmsnorm_quant", false, ternaspmm_next_linear{}, a); }
// (..., next linear | None): the same for any split count up to eight
TERNA_FUNCTION(step_attention_merge, 9) { return merge_norm_quant("step_attention_merge", true, next_linear("step_attention_merge", a[8]), a); }

// (tokens, pos, embedding, rope_table, norm_weight) -> (x, stats, rope [2, B, half]); tokens / pos contiguous int64 vectors
TERNA_FUNCTION(step_inputs, 5)
{
    const char* who = "step_inputs";
    const at::Tensor &tokens = tensor(a[0]), &pos = tensor(a[1]), &embedding = tensor(a[2]), &table = tensor(a[3]), &weight = tensor(a[4]);
    check_matrix(who, embedding);
    const int64_t b = tokens.numel(), v = embedding.size(0), k = embedding.size(1);
    if (table.dim() != 3 || table.size(1) != 2 || tokens.scalar_type() != at::kLong || pos.scalar_type() != at::kLong || (pos.numel() != 1 && pos.numel() != b) ||
        table.scalar_type() != at::kFloat || embedding.scalar_type() != at::kBFloat16 || !embedding.is_contiguous() || !table.is_contiguous())
        refuse("%s: tokens / pos int64, embedding bf16 [V, K] and rope_table fp32 [S, 2, half] contiguous", who);
    check_numel(who, "norm_weight", &weight, k);
    const int count = lib.ternaspmm_row_stats_count(k);
    if (count < 1) refuse("%s: unsupported K=%d", who, static_cast<int>(k));
    Unlocked unlocked;
    const at::Tensor ids = tokens.contiguous(), at_slot = pos.contiguous();         // (copies only where a caller passed a strided view)
    const int64_t slots = table.size(0), half = table.size(2);
    at::Tensor x = make({b, k}, at::kBFloat16, embedding), stats = make({b, count, 2}, at::kFloat, embedding), rope = make({2, b, half}, at::kFloat, embedding);
    const int left = lib.ternaspmm_step_inputs(data<long long>(&ids), data<long long>(&at_slot), pos.numel() == b && b > 1, data<terna_bf16>(&embedding), v, k,
                                               data<float>(&table), slots, half, data<terna_bf16>(&weight), data<terna_bf16>(&x), data<float>(&stats),
                                               data<float>(&rope), b, stream());
    unlocked.end();
    if (left != count)
        refuse("%s: the library refused the launch (B=%d V=%d K=%d S=%d half=%d)", who, static_cast<int>(b), static_cast<int>(v), static_cast<int>(k),
               static_cast<int>(slots), static_cast<int>(half));
    return pack(unlocked, std::move(x), std::move(stats), std::move(rope));
}

// (tokens, pos, embedding, rope_table) -> (x, rope [2, positions, half]): int64 tokens [B, T] and positions of T or B T elements
TERNA_FUNCTION(prompt_inputs, 4)
{
    const char* who = "prompt_inputs";
    const at::Tensor &tokens = tensor(a[0]), &pos = tensor(a[1]), &embedding = tensor(a[2]), &table = tensor(a[3]);
    check_matrix(who, embedding);
    const int64_t m = tokens.numel(), v = embedding.size(0), k = embedding.size(1), rows = pos.numel();
    if (tokens.dim() != 2 || m < 1 || m > INT32_MAX || (rows != m && rows != tokens.size(1)))
        refuse("%s: tokens [B, T] and positions of T or B * T elements", who);
    if (table.dim() != 3 || table.size(1) != 2 || tokens.scalar_type() != at::kLong || pos.scalar_type() != at::kLong || table.scalar_type() != at::kFloat ||
        embedding.scalar_type() != at::kBFloat16 || !embedding.is_contiguous() || !table.is_contiguous())
        refuse("%s: tokens / pos int64, embedding bf16 [V, K] and rope_table fp32 [S, 2, half] contiguous", who);
    Unlocked unlocked;
    const at::Tensor ids = tokens.contiguous(), at_slot = pos.contiguous();
    const int64_t slots = table.size(0), half = table.size(2);
    at::Tensor x = make({m, k}, at::kBFloat16, embedding), rope = make({2, rows, half}, at::kFloat, embedding);
    const int rc = lib.ternaspmm_prompt_inputs(data<long long>(&ids), data<long long>(&at_slot), rows, data<terna_bf16>(&embedding), v, k, data<float>(&table), slots,
                                               half, data<terna_bf16>(&x), data<float>(&rope), m, stream());
    unlocked.end();
    if (rc != 0)
        refuse("%s: the library refused the launch (M=%d V=%d K=%d S=%d half=%d)", who, static_cast<int>(m), static_cast<int>(v), static_cast<int>(k),
               static_cast<int>(slots), static_cast<int>(half));
    return pack(unlocked, std::move(x), std::move(rope));
}

// (tokens, pos, embedding, rope_table, heads, head_dim, scale, eps, splits, blocks) -> the residual stream behind the last block, bf16 [B, dim],
// or None where the step is not one for this launch (the launches it stands for have the checks that raise).  blocks: a sequence of tuples (wqkv, ws, ws_num, out_features, wo [4], interleaved
// w13 [4], w2 [4], attention_norm, attn_sub_norm, ffn_norm, ffn_sub_norm, cache_k, cache_v).
TERNA_FUNCTION(decode_step, 10)
{
    const char* who = "decode_step";
    const at::Tensor &tokens = tensor(a[0]), &pos = tensor(a[1]), &embedding = tensor(a[2]), &table = tensor(a[3]);
    check_matrix(who, embedding);
    const int64_t b = tokens.numel(), v = embedding.size(0), dim = embedding.size(1);
    const int64_t heads = integer32(a[4]), head_dim = integer32(a[5]), wide = heads * head_dim;
    if (table.dim() != 3 || table.size(1) != 2 || 2 * table.size(2) != head_dim || tokens.scalar_type() != at::kLong || pos.scalar_type() != at::kLong ||
        (pos.numel() != 1 && pos.numel() != b) || table.scalar_type() != at::kFloat || embedding.scalar_type() != at::kBFloat16 || !embedding.is_contiguous() ||
        !table.is_contiguous() || !embedding.is_cuda())
        Py_RETURN_NONE;
    if (!PyTuple_Check(a[9]) && !PyList_Check(a[9])) refuse("%s: blocks is a list", who);
    const Py_ssize_t layers = PySequence_Fast_GET_SIZE(a[9]);
    if (b < 1 || b > 64 || layers < 1 || layers > 1024) Py_RETURN_NONE;
    ternaspmm_step_desc d{};
    d.layers = layers, d.M = b, d.dim = dim, d.heads = heads, d.head_dim = head_dim, d.slots = table.size(0);
    d.splits = integer32(a[8]), d.per_sequence = pos.numel() == b && b > 1, d.vocab = v;
    d.scale = real(a[6]), d.eps = real(a[7]);
    std::vector<ternaspmm_step_block> blocks(layers);
    for (Py_ssize_t n = 0; n < layers; ++n) {
        PyObject* item = PySequence_Fast_GET_ITEM(a[9], n);
        if (!PyTuple_Check(item) || PyTuple_GET_SIZE(item) != 22) refuse("%s: a block is a tuple of 22", who);
        PyObject* const* p = reinterpret_cast<PyTupleObject*>(item)->ob_item;
        const int64_t qkv_n = integer32(p[3]), gate_n = integer32(p[11]), ffn = gate_n / 2;
        const BlockLinear qkv_w(who, p, dim), o_w(who, p + 4, wide), gate_w(who, p + 8, dim), down_w(who, p + 12, ffn);
        const at::Tensor* norm[4] = {&tensor(p[16]), &tensor(p[17]), &tensor(p[18]), &tensor(p[19])};
        const int64_t want[4] = {dim, wide, dim, ffn};
        for (int i = 0; i < 4; ++i)
            if (norm[i]->numel() != want[i] || norm[i]->scalar_type() != at::kBFloat16 || !norm[i]->is_contiguous()) Py_RETURN_NONE;
        const at::Tensor &ck = tensor(p[20]), &cv = tensor(p[21]);
        if (ck.dim() != 4 || ck.sizes() != cv.sizes() || ck.size(0) != b || ck.size(2) != d.slots || ck.size(3) != head_dim || !ck.is_contiguous() ||
            !cv.is_contiguous() || ck.scalar_type() != at::kBFloat16 || cv.scalar_type() != at::kBFloat16)
            Py_RETURN_NONE;
        const int kv = ck.size(1);
        if (o_w.n != dim || down_w.n != dim || qkv_n != (heads + 2 * kv) * head_dim) Py_RETURN_NONE;
        if (n == 0) {
            d.kv_heads = kv, d.ffn = ffn, d.ws_num_qkv = qkv_w.ws_num, d.ws_num_o = o_w.ws_num, d.ws_num_down = down_w.ws_num;
        } else if (d.kv_heads != kv || d.ffn != ffn || d.ws_num_qkv != qkv_w.ws_num || d.ws_num_o != o_w.ws_num || d.ws_num_down != down_w.ws_num) {
            Py_RETURN_NONE;                      // blocks of different shapes
        }
        if (gate_w.ws_num != 2 || ffn * 2 != gate_n) Py_RETURN_NONE;
        blocks[n] = ternaspmm_step_block{data(&qkv_w.packed), data(&o_w.packed), data(&gate_w.packed), data(&down_w.packed),
                                         data<terna_bf16>(&qkv_w.ws), data<terna_bf16>(&o_w.ws), data<terna_bf16>(&gate_w.ws), data<terna_bf16>(&down_w.ws),
                                         data<terna_bf16>(norm[0]), data<terna_bf16>(norm[1]), data<terna_bf16>(norm[2]), data<terna_bf16>(norm[3]),
                                         data<terna_bf16>(&ck), data<terna_bf16>(&cv)};
    }
    const long long bytes = lib.ternaspmm_decode_step_bytes(&d);
    if (bytes < 0) Py_RETURN_NONE;
    Unlocked unlocked;
    const at::Tensor ids = tokens.contiguous(), at_slot = pos.contiguous();
    at::Tensor x = make({b, dim}, at::kBFloat16, embedding);
    const c10::DataPtr scratch = device_allocator()->allocate(bytes);
    if (lib.ternaspmm_decode_step(&d, blocks.data(), data<long long>(&ids), data<long long>(&at_slot), data<terna_bf16>(&embedding), data<float>(&table), scratch.get(),
                                  data<terna_bf16>(&x), stream()) != 0)
        return none(unlocked);
    return wrap(std::move(x), unlocked);
}

// ---- long contexts: rotary positions, the 4-bit cache, log probabilities.  These take tensors of any device: the current one is changed for the call.
using Guard = std::optional<c10::DeviceGuard>;
void on_device_of(Guard& guard, const at::Tensor& x)
{
    if (x.device().index() != c10::hip::current_device()) guard.emplace(x.device());
}
void check_device(const char* who, const char* name, const at::Tensor& t, const at::Tensor& with)
{
    if (!t.is_cuda() || t.device() != with.device()) refuse("%s: %s has to be on the GPU, with the other tensors", who, name);
}

// int64 positions [T], or [B, T]: of every sequence its own
struct Positions {
    at::Tensor pos;
    int each;

    Positions(const char* who, PyObject* o, const at::Tensor& with, int64_t batch, int64_t tokens) : pos(tensor(o)), each(pos.dim() == 2)
    {
        if (pos.scalar_type() != at::kLong || !(each ? pos.size(0) == batch && pos.size(1) == tokens : pos.dim() == 1 && pos.size(0) == tokens))
            refuse("%s: positions are int64 [T] or [B, T] with B = %lld, T = %lld", who, static_cast<long long>(batch), static_cast<long long>(tokens));
        check_device(who, "pos", pos, with);
        pos = pos.contiguous();
    }
    const long long* data() const { return reinterpret_cast<const long long*>(pos.const_data_ptr<int64_t>()); }
};

struct Frequencies {
    at::Tensor held;

    Frequencies(const char* who, PyObject* o, const at::Tensor& with, int64_t dim) : held(tensor(o))
    {
        if (held.scalar_type() != at::kDouble || held.dim() != 1 || held.size(0) < 1 || 2 * held.size(0) > dim)
            refuse("%s: inv_freq is a float64 vector of 1 to %lld elements", who, static_cast<long long>(dim / 2));
        check_device(who, "inv_freq", held, with);
        held = held.contiguous();
    }
    const double* data() const { return held.const_data_ptr<double>(); }
    int pairs() const { return static_cast<int>(held.size(0)); }
};

// bytes from a tensor's first element to behind its last
int64_t byte_extent(const at::Tensor& t)
{
    int64_t last = 0;
    for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
    return (last + 1) * static_cast<int64_t>(t.element_size());
}
// whether two indexes may name the same element
bool overlaps_itself(const at::Tensor& t)
{
    std::vector<std::pair<int64_t, int64_t>> dims;             // (stride, size)
    for (int64_t d = 0; d < t.dim(); ++d)
        if (t.size(d) > 1) dims.emplace_back(t.stride(d), t.size(d));
    std::sort(dims.begin(), dims.end());
    int64_t extent = 1;
    for (const auto& [stride, size] : dims) {
        if (stride < extent) return true;
        extent = stride * (size - 1) + extent;
    }
    return false;
}
bool aligned16(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0; }

// (x [B, T, H, D], pos, inv_freq, amplitude, adjacent, out | None) -> out
TERNA_FUNCTION(rotary_embed, 6)
{
    const char* who = "rotary_embed";
    const at::Tensor& x = tensor(a[0]);
    const at::Tensor* given = optional(a[5]);
    const double amplitude = PyFloat_AsDouble(a[3]);
    if (amplitude == -1.0 && PyErr_Occurred()) throw Refused();
    const bool adjacent = truth(a[4]);
    if (x.dim() != 4 || (x.scalar_type() != at::kBFloat16 && x.scalar_type() != at::kFloat)) refuse("%s: x is a bfloat16 or float32 [B, T, H, D] tensor", who);
    check_device(who, "x", x, x);
    const int64_t b = x.size(0), t = x.size(1), h = x.size(2), d = x.size(3);
    if (d > 1024 || h > 65535 || b * t > 1 << 30) refuse("%s: at most 65535 heads of 1024 dimensions and 2^30 tokens", who);
    if (d < 2) refuse("%s: heads have two dimensions at least", who);
    const Positions pos(who, a[1], x, b, t);
    const Frequencies frequency(who, a[2], x, d);
    if (given != nullptr) {
        if (given->scalar_type() != x.scalar_type() || given->sizes() != x.sizes()) refuse("%s: out has another shape or type than x", who);
        check_device(who, "out", *given, x);
        const char *p = static_cast<const char*>(x.const_data_ptr()), *q = static_cast<const char*>(given->const_data_ptr());
        const bool same = p == q && x.strides() == given->strides();
        if (x.numel() != 0 && (overlaps_itself(*given) || given->stride(3) != 1 || (!same && p < q + byte_extent(*given) && q < p + byte_extent(x))))
            refuse("%s: out is x itself, or rows of their own, its last dimension contiguous", who);
    }
    Guard guard;
    on_device_of(guard, x);
    Unlocked unlocked;
    // (a last dimension of other strides: a copy, which an out that is x is not written through, but its own memory)
    const at::Tensor rows = x.stride(3) == 1 ? x : x.contiguous();
    at::Tensor out = given != nullptr ? *given : make(x.sizes(), x.scalar_type(), x);
    if (x.numel() == 0) return wrap(std::move(out), unlocked);
    const long long in_strides[3] = {rows.stride(0), rows.stride(1), rows.stride(2)}, out_strides[3] = {out.stride(0), out.stride(1), out.stride(2)};
    const int rc = lib.ternaspmm_rotary(rows.const_data_ptr(), in_strides, out.mutable_data_ptr(), out_strides, x.scalar_type() == at::kFloat, pos.data(), pos.each,
                                        frequency.data(), frequency.pairs(), amplitude, b, t, h, d, adjacent, stream());
    unlocked.end();
    if (rc != 0) refuse("%s: more tokens than a launch has room for: fewer than 2^24, or than 2^24 groups of several", who);
    return THPVariable_Wrap(std::move(out));
}

// k, k_scale, v, v_scale from a[0 .. 3]
struct Kv4 {
    ternaspmm_kv4 c;
    int64_t batch, kv, slots, dim;

    Kv4(const char* who, PyObject* const* a)
    {
        const at::Tensor *t[4] = {&tensor(a[0]), &tensor(a[1]), &tensor(a[2]), &tensor(a[3])};
        if (t[0]->dim() != 4) refuse("%s: the cache's codes are uint8 [B, KV, S, D / 2]", who);
        batch = t[0]->size(0), kv = t[0]->size(1), slots = t[0]->size(2), dim = 2 * t[0]->size(3);
        if ((dim != 64 && dim != 128) || kv < 1 || kv > 4096 || slots < 1 || slots > 1 << 25)
            refuse("%s: a cache has heads of 64 or 128 dimensions and 1 to 2^25 slots", who);
        for (int i = 0; i < 4; ++i) {
            const std::array<int64_t, 4> want{batch, kv, slots, i & 1 ? dim / 32 : dim / 2};
            if (t[i]->scalar_type() != at::kByte || t[i]->sizes() != at::IntArrayRef(want) || !t[i]->is_contiguous() || (reinterpret_cast<uintptr_t>(t[i]->const_data_ptr()) & (i & 1 ? 3 : 15)) != 0)
                refuse("%s: the cache is contiguous uint8: codes [B, KV, S, D / 2] from a multiple of 16 bytes on, scales [B, KV, S, D / 32] from one of 4", who);
            check_device(who, "the cache", *t[i], *t[0]);
        }
        c = ternaspmm_kv4{data<uint8_t>(t[0]), data<uint8_t>(t[1]), data<uint8_t>(t[2]), data<uint8_t>(t[3])};
    }
};

// rows of a fused projection: bf16 [B * T, (H + 2 KV) D]
at::Tensor projection_rows(const char* who, const at::Tensor& x, const at::Tensor& codes, const Kv4& cache, int64_t heads, int64_t* tokens)
{
    if (x.dim() != 2 || x.scalar_type() != at::kBFloat16 || heads < 1 || heads > 4096 || heads % cache.kv != 0 || x.size(1) != (heads + 2 * cache.kv) * cache.dim)
        refuse("%s: xqkv is bfloat16 [B * T, (H + 2 KV) D] with H a multiple of KV", who);
    check_device(who, "xqkv", x, codes);
    if (cache.batch < 1 ? x.size(0) != 0 : x.size(0) % cache.batch != 0) refuse("%s: %lld rows for %lld sequences", who, static_cast<long long>(x.size(0)), static_cast<long long>(cache.batch));
    *tokens = cache.batch < 1 ? 0 : x.size(0) / cache.batch;
    if (x.size(0) * heads > 1 << 28 || x.size(0) > 1 << 24) refuse("%s: too many rows", who);
    return x.stride(1) == 1 && x.stride(0) >= x.size(1) && x.stride(0) % 8 == 0 && aligned16(x) ? x : x.clone(at::MemoryFormat::Contiguous);
}
// the scale of the scores: None for dim ** -0.5
std::optional<float> scale_or_none(PyObject* o) { return o == Py_None ? std::nullopt : std::optional<float>(real(o)); }
float scale_of(const std::optional<float>& given, int64_t dim) { return given ? *given : static_cast<float>(std::pow(static_cast<double>(dim), -0.5)); }
c10::DataPtr kv4_workspace(int64_t b, int64_t t, int64_t h, const Kv4& cache)
{
    const long long bytes = lib.ternaspmm_kv4_workspace_bytes(b, t, h, cache.kv, cache.dim, cache.slots);
    return bytes > 0 ? device_allocator()->allocate(bytes) : c10::DataPtr();
}

// (xqkv, pos, inv_freq, amplitude, k, k_scale, v, v_scale, heads, adjacent) -> q [B, H, T, D]
TERNA_FUNCTION(kv4_store, 10)
{
    const char* who = "kv4_store";
    const at::Tensor &x = tensor(a[0]), &codes = tensor(a[4]);
    const double amplitude = PyFloat_AsDouble(a[3]);
    if (amplitude == -1.0 && PyErr_Occurred()) throw Refused();
    const int64_t heads = integer32(a[8]);
    const bool adjacent = truth(a[9]);
    const Kv4 cache(who, a + 4);
    check_device(who, "the cache", codes, codes);
    Guard guard;
    on_device_of(guard, codes);
    int64_t t;
    const at::Tensor rows = projection_rows(who, x, codes, cache, heads, &t);
    const Positions pos(who, a[1], codes, cache.batch, t);
    const Frequencies frequency(who, a[2], codes, cache.dim);
    Unlocked unlocked;
    at::Tensor q = make({cache.batch, heads, t, cache.dim}, at::kBFloat16, codes);
    if (q.numel() == 0) return wrap(std::move(q), unlocked);
    const int rc = lib.ternaspmm_kv4_store(data<terna_bf16>(&rows), rows.stride(0), pos.data(), pos.each, frequency.data(), frequency.pairs(), amplitude, data<terna_bf16>(&q),
                                           &cache.c, cache.batch, t, heads, cache.kv, cache.dim, cache.slots, adjacent, stream());
    unlocked.end();
    if (rc != 0) refuse("%s: the library refused the launch", who);
    return THPVariable_Wrap(std::move(q));
}

// (k, k_scale, v, v_scale, pos) -> (keys, values) bf16 [B, T, KV, D]
TERNA_FUNCTION(kv4_rows, 5)
{
    const char* who = "kv4_rows";
    const at::Tensor &codes = tensor(a[0]), &at_slot = tensor(a[4]);
    const Kv4 cache(who, a);
    check_device(who, "the cache", codes, codes);
    if (at_slot.dim() < 1) refuse("%s: positions are int64 [T] or [B, T]", who);
    Guard guard;
    on_device_of(guard, codes);
    const int64_t t = at_slot.size(-1);
    const Positions pos(who, a[4], codes, cache.batch, t);
    if (cache.batch * t * cache.kv > 1 << 28 || cache.batch * t > 1 << 24) refuse("%s: too many rows", who);
    Unlocked unlocked;
    at::Tensor k = make({cache.batch, t, cache.kv, cache.dim}, at::kBFloat16, codes), v = make({cache.batch, t, cache.kv, cache.dim}, at::kBFloat16, codes);
    const int rc = k.numel() == 0 ? 0
                                  : lib.ternaspmm_kv4_rows(&cache.c, pos.data(), pos.each, data<terna_bf16>(&k), data<terna_bf16>(&v), cache.batch, t, cache.kv, cache.dim,
                                                           cache.slots, stream());
    unlocked.end();
    if (rc != 0) refuse("%s: the library refused the launch", who);
    return pack(unlocked, std::move(k), std::move(v));
}

// (q [B, H, T, D], pos, k, k_scale, v, v_scale, scale | None) -> [B * T, H * D]
TERNA_FUNCTION(kv4_attention, 7)
{
    const char* who = "kv4_attention";
    const at::Tensor &q = tensor(a[0]), &codes = tensor(a[2]);
    const std::optional<float> given_scale = scale_or_none(a[6]);
    const Kv4 cache(who, a + 2);
    const float scale = scale_of(given_scale, cache.dim);
    check_device(who, "the cache", codes, codes);
    if (q.dim() != 4 || q.scalar_type() != at::kBFloat16 || q.size(0) != cache.batch || q.size(3) != cache.dim || q.size(1) < 1 || q.size(1) > 4096 || q.size(1) % cache.kv != 0)
        refuse("%s: q is bfloat16 [B, H, T, D] with the cache's B and D and H a multiple of its KV", who);
    check_device(who, "q", q, codes);
    const int64_t h = q.size(1), t = q.size(2);
    if (cache.batch * t * h > 1 << 28 || cache.batch * t > 1 << 24) refuse("%s: too many rows", who);
    Guard guard;
    on_device_of(guard, codes);
    const Positions pos(who, a[1], codes, cache.batch, t);
    const at::Tensor rows = q.is_contiguous() && aligned16(q) ? q : q.clone(at::MemoryFormat::Contiguous);
    Unlocked unlocked;
    at::Tensor out = make({cache.batch * t, h * cache.dim}, at::kBFloat16, codes);
    if (out.numel() == 0) return wrap(std::move(out), unlocked);
    const c10::DataPtr work = kv4_workspace(cache.batch, t, h, cache);
    const int rc = lib.ternaspmm_kv4_attention(data<terna_bf16>(&rows), &cache.c, pos.data(), pos.each, data<terna_bf16>(&out), work.get(), cache.batch, t, h, cache.kv, cache.dim,
                                               cache.slots, scale, stream());
    unlocked.end();
    if (rc != 0) refuse("%s: the library refused the launch", who);
    return THPVariable_Wrap(std::move(out));
}

// (xqkv, pos, inv_freq, amplitude, k, k_scale, v, v_scale, heads, adjacent, scale | None) -> [B, H * D]
TERNA_FUNCTION(kv4_step, 11)
{
    const char* who = "kv4_step";
    const at::Tensor &x = tensor(a[0]), &codes = tensor(a[4]);
    const double amplitude = PyFloat_AsDouble(a[3]);
    if (amplitude == -1.0 && PyErr_Occurred()) throw Refused();
    const int64_t heads = integer32(a[8]);
    const bool adjacent = truth(a[9]);
    const std::optional<float> given_scale = scale_or_none(a[10]);
    const Kv4 cache(who, a + 4);
    const float scale = scale_of(given_scale, cache.dim);
    check_device(who, "the cache", codes, codes);
    Guard guard;
    on_device_of(guard, codes);
    int64_t t;
    const at::Tensor rows = projection_rows(who, x, codes, cache, heads, &t);
    if (cache.batch > 0 && t != 1) refuse("%s: one new token per sequence", who);
    const Positions pos(who, a[1], codes, cache.batch, 1);
    const Frequencies frequency(who, a[2], codes, cache.dim);
    Unlocked unlocked;
    at::Tensor out = make({cache.batch, heads * cache.dim}, at::kBFloat16, codes);
    if (out.numel() == 0) return wrap(std::move(out), unlocked);
    const c10::DataPtr work = kv4_workspace(cache.batch, 1, heads, cache);
    const int rc = lib.ternaspmm_kv4_step(data<terna_bf16>(&rows), rows.stride(0), pos.data(), pos.each, frequency.data(), frequency.pairs(), amplitude, &cache.c,
                                          data<terna_bf16>(&out), work.get(), cache.batch, heads, cache.kv, cache.dim, cache.slots, scale, adjacent, stream());
    unlocked.end();
    if (rc != 0) refuse("%s: the library refused the launch", who);
    return THPVariable_Wrap(std::move(out));
}

// (logits [M, V], targets | None, top) -> (logprob | None, entropy, top_ids | None, top_logprobs | None)
TERNA_FUNCTION(token_logprobs, 3)
{
    const char* who = "token_logprobs";
    const at::Tensor& logits = tensor(a[0]);
    const at::Tensor* targets = optional(a[1]);
    const int top = integer32(a[2]);
    if (logits.dim() != 2 || (logits.scalar_type() != at::kBFloat16 && logits.scalar_type() != at::kFloat)) refuse("%s: logits are bfloat16 or float32 [M, V]", who);
    check_device(who, "logits", logits, logits);
    const int64_t m = logits.size(0), v = logits.size(1);
    if (v < 1 || v > 1 << 19 || m >= 1 << 24) refuse("%s: 1 to 2^19 logits in fewer than 2^24 rows", who);
    if (top < 0 || top > 64 || top > v) refuse("%s: top is 0 to 64 and at most V", who);
    if (targets != nullptr) {
        if (targets->scalar_type() != at::kLong || targets->dim() != 1 || targets->size(0) != m) refuse("%s: targets are int64 [M]", who);
        check_device(who, "targets", *targets, logits);
    }
    Guard guard;
    on_device_of(guard, logits);
    Unlocked unlocked;
    const at::Tensor rows = v == 1 || logits.stride(1) == 1 ? logits : logits.contiguous();
    at::Tensor wanted, logprob, entropy = make({m}, at::kFloat, logits), ids, values;
    if (targets != nullptr) {
        wanted = targets->contiguous();
        logprob = make({m}, at::kFloat, logits);
    }
    if (top > 0) {
        ids = make({m, top}, at::kLong, logits);
        values = make({m, top}, at::kFloat, logits);
    }
    int rc = 0;
    if (m > 0) {
        const long long bytes = lib.ternaspmm_token_logprobs_workspace_bytes(m, v, logits.scalar_type() == at::kFloat, top);
        const c10::DataPtr work = bytes > 0 ? device_allocator()->allocate(bytes) : c10::DataPtr();
        rc = lib.ternaspmm_token_logprobs(rows.const_data_ptr(), rows.stride(0), logits.scalar_type() == at::kFloat, targets != nullptr ? data<long long>(&wanted) : nullptr,
                                          targets != nullptr ? data<float>(&logprob) : nullptr, data<float>(&entropy), top > 0 ? data<long long>(&ids) : nullptr,
                                          top > 0 ? data<float>(&values) : nullptr, top, work.get(), m, v, stream());
    }
    unlocked.end();
    if (rc != 0) refuse("%s: the library refused the launch", who);
    return pack(unlocked, std::move(logprob), std::move(entropy), std::move(ids), std::move(values));
}

// ---- drafted tokens, 8-bit projections: tensors of any device here too
const long long* longs(const at::Tensor& t) { return reinterpret_cast<const long long*>(t.const_data_ptr<int64_t>()); }
long long* mutable_longs(at::Tensor& t) { return reinterpret_cast<long long*>(t.mutable_data_ptr<int64_t>()); }

constexpr int64_t kMaxNodes = 512;
// int64 [B, T] of a tree's nodes, contiguous
at::Tensor nodes_of(const char* who, const char* name, PyObject* o)
{
    const at::Tensor& t = tensor(o);
    if (t.scalar_type() != at::kLong || t.dim() != 2 || t.size(1) > kMaxNodes || t.size(0) > 65535) refuse("%s: %s is int64 [B, T], of at most 65535 sequences of 512 nodes", who, name);
    check_device(who, name, t, t);
    return t;
}
// int64 [B]
void check_each(const char* who, const char* name, const at::Tensor& t, int64_t batch, const at::Tensor& with)
{
    if (t.scalar_type() != at::kLong || t.dim() != 1 || t.size(0) != batch) refuse("%s: %s is int64 [B] with B = %lld", who, name, static_cast<long long>(batch));
    check_device(who, name, t, with);
}

// (parents) -> (mask [B, T, W], depth [B, T])
TERNA_FUNCTION(draft_tree, 1)
{
    const char* who = "draft_tree";
    const at::Tensor parents = nodes_of(who, "parents", a[0]);
    const int64_t b = parents.size(0), t = parents.size(1);
    Guard guard;
    on_device_of(guard, parents);
    Unlocked unlocked;
    const at::Tensor rows = parents.contiguous();
    Longs results(b * t * ((t + 63) / 64 + 1), parents);
    at::Tensor mask = results.take({b, t, (t + 63) / 64}), depth = results.take({b, t});
    const int rc = depth.numel() == 0 ? 0 : lib.ternaspmm_draft_tree(longs(rows), mutable_longs(mask), mutable_longs(depth), b, t, stream());
    unlocked.end();
    if (rc != 0) refuse("%s: the library refused the launch", who);
    return pack(unlocked, std::move(mask), std::move(depth));
}

// (q [B, H, T, D], k, v [B, KV, S, D], start [B], mask [T, W] | [B, T, W], scale | None) -> [B * T, H * D]
TERNA_FUNCTION(tree_attention, 6)
{
    const char* who = "tree_attention";
    const at::Tensor &q = tensor(a[0]), &k = tensor(a[1]), &v = tensor(a[2]), &start = tensor(a[3]), &mask = tensor(a[4]);
    const std::optional<float> given_scale = scale_or_none(a[5]);
    if (k.dim() != 4 || v.dim() != 4 || k.scalar_type() != at::kBFloat16 || v.scalar_type() != at::kBFloat16 || k.sizes() != v.sizes())
        refuse("%s: the cache's keys and values are bfloat16 [B, KV, S, D]", who);
    check_device(who, "the cache", k, k);
    check_device(who, "the cache", v, k);
    const int64_t b = k.size(0), kv = k.size(1), s = k.size(2), d = k.size(3);
    if ((d != 64 && d != 128) || kv < 1 || s < 1 || s > 1 << 25) refuse("%s: a cache has heads of 64 or 128 dimensions and 1 to 2^25 slots", who);
    for (const at::Tensor* t : {&k, &v})
        if (t->stride(3) != 1 || (t->stride(0) & 7) || (t->stride(1) & 7) || (t->stride(2) & 7) || t->stride(2) >= 1 << 24 || !aligned16(*t))
            refuse("%s: the cache's rows are contiguous, each from a multiple of 16 bytes on, slots fewer than 2^24 elements apart", who);
    if (q.dim() != 4 || q.scalar_type() != at::kBFloat16 || q.size(0) != b || q.size(3) != d || q.size(1) < 1 || q.size(1) > 4096 || q.size(1) % kv != 0)
        refuse("%s: q is bfloat16 [B, H, T, D] with the cache's B and D and H a multiple of its KV", who);
    check_device(who, "q", q, k);
    const int64_t h = q.size(1), t = q.size(2), words = (t + 63) / 64;
    if (t > kMaxNodes || b * t * h > 1 << 28) refuse("%s: at most 512 nodes a tree, 2^28 rows of all heads", who);
    check_each(who, "start", start, b, k);
    const bool each = mask.dim() == 3;
    if (mask.scalar_type() != at::kLong || (!each && mask.dim() != 2) || (each && mask.size(0) != b) || mask.size(-2) != t || mask.size(-1) != words)
        refuse("%s: mask is int64 [T, W] or [B, T, W] with W = (T + 63) / 64", who);
    check_device(who, "mask", mask, k);
    const float scale = scale_of(given_scale, d);
    if (!std::isfinite(scale * static_cast<float>(M_LOG2E))) refuse("%s: a scale that is not finite, in powers of two", who);
    Guard guard;
    on_device_of(guard, k);
    Unlocked unlocked;
    at::Tensor out = make({b * t, h * d}, at::kBFloat16, k);
    if (out.numel() == 0) return wrap(std::move(out), unlocked);
    const at::Tensor rows = q.stride(3) == 1 && !(q.stride(0) & 7) && !(q.stride(1) & 7) && !(q.stride(2) & 7) && aligned16(q) ? q : q.clone(at::MemoryFormat::Contiguous);
    const at::Tensor starts = start.contiguous(), masks = mask.contiguous();
    const long long q_strides[3] = {rows.stride(0), rows.stride(1), rows.stride(2)}, k_strides[3] = {k.stride(0), k.stride(1), k.stride(2)},
                    v_strides[3] = {v.stride(0), v.stride(1), v.stride(2)};
    const long long bytes = lib.ternaspmm_tree_attention_workspace_bytes(b, t, h, kv, d, s);
    const c10::DataPtr work = bytes > 0 ? device_allocator()->allocate(bytes) : c10::DataPtr();
    const int rc = lib.ternaspmm_tree_attention(data<terna_bf16>(&rows), q_strides, data<terna_bf16>(&k), k_strides, data<terna_bf16>(&v), v_strides, longs(starts), longs(masks), each,
                                                data<terna_bf16>(&out), work.get(), b, t, h, kv, d, s, scale, stream());
    unlocked.end();
    if (rc != 0) refuse("%s: the library refused the launch", who);
    return THPVariable_Wrap(std::move(out));
}

// (logits [B, T, V], tokens, parents) -> (path [B, T], count [B], next [B])
TERNA_FUNCTION(tree_accept, 3)
{
    const char* who = "tree_accept";
    const at::Tensor& logits = tensor(a[0]);
    const at::Tensor tokens = nodes_of(who, "tokens", a[1]), parents = nodes_of(who, "parents", a[2]);
    if (logits.dim() != 3 || (logits.scalar_type() != at::kBFloat16 && logits.scalar_type() != at::kFloat)) refuse("%s: logits are bfloat16 or float32 [B, T, V]", who);
    check_device(who, "logits", logits, logits);
    const int64_t b = logits.size(0), t = logits.size(1), v = logits.size(2);
    if (t < 1 || v < 1 || v > 1 << 19) refuse("%s: 1 to 512 nodes, 1 to 2^19 logits", who);
    for (const at::Tensor* x : {&tokens, &parents})
        if (x->size(0) != b || x->size(1) != t) refuse("%s: tokens and parents are [B, T] as the logits' rows", who);
    check_device(who, "tokens", tokens, logits);
    check_device(who, "parents", parents, logits);
    Guard guard;
    on_device_of(guard, logits);
    Unlocked unlocked;
    const bool fp32 = logits.scalar_type() == at::kFloat;
    const int64_t work = b == 0 ? 0 : std::max(0ll, static_cast<long long>(lib.ternaspmm_tree_accept_workspace_bytes(b, t, v, fp32)));      // (no more than 2048 parts, or one a node)
    Longs results(b * (t + 2) + work / 8, logits);
    at::Tensor path = results.take({b, t}), count = results.take({b}), next = results.take({b});
    int rc = 0;
    if (b > 0) {
        const at::Tensor rows = (v == 1 || logits.stride(2) == 1) && (b == 1 || t == 1 || logits.stride(0) == t * logits.stride(1)) ? logits : logits.contiguous();
        const at::Tensor drafted = tokens.contiguous(), of = parents.contiguous();
        rc = lib.ternaspmm_tree_accept(rows.const_data_ptr(), t == 1 ? rows.stride(0) : rows.stride(1), fp32, longs(drafted), longs(of), mutable_longs(path), mutable_longs(count),
                                       mutable_longs(next), work == 0 ? nullptr : results.all.mutable_data_ptr<int64_t>() + results.used, b, t, v, stream());
    }
    unlocked.end();
    if (rc != 0) refuse("%s: the library refused the launch", who);
    return pack(unlocked, std::move(path), std::move(count), std::move(next));
}

// ([cache [B, heads, S, ...] ...], start [B], path [B, T], count [B])
TERNA_FUNCTION(cache_move, 4)
{
    const char* who = "cache_move";
    const at::Tensor path = nodes_of(who, "path", a[2]);
    const at::Tensor &start = tensor(a[1]), &count = tensor(a[3]);
    const int64_t b = path.size(0), t = path.size(1);
    check_each(who, "start", start, b, path);
    check_each(who, "count", count, b, path);
    if (!PyTuple_Check(a[0]) && !PyList_Check(a[0])) refuse("%s: caches is a list of tensors", who);
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(a[0]);
    std::vector<ternaspmm_cache_rows> caches(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
        const at::Tensor& c = tensor(PySequence_Fast_GET_ITEM(a[0], i));
        if (c.dim() != 4 || c.size(0) != b || c.size(1) > 65535 || c.size(2) > INT32_MAX || c.size(3) > 1 << 20) refuse("%s: a cache is [B, heads, S, D] with the path's B", who);
        check_device(who, "a cache", c, path);
        const bool empty = c.numel() == 0 || c.size(2) == 1;               // (of one slot nothing moves, whatever its stride)
        if (!empty && !c.is_contiguous() && ((c.size(3) > 1 && c.stride(3) != 1) || overlaps_itself(c) || c.stride(2) < c.size(3))) refuse("%s: a cache's rows are contiguous and apart from each other", who);
        const long long size = c.element_size();
        caches[i] = ternaspmm_cache_rows{empty ? nullptr : c.mutable_data_ptr(), c.stride(0) * size, c.stride(1) * size, c.stride(2) * size, static_cast<int>(c.size(1)),
                                         static_cast<int>(c.size(2)), static_cast<int>(c.size(3) * size)};
    }
    caches.erase(std::remove_if(caches.begin(), caches.end(), [](const ternaspmm_cache_rows& c) { return c.rows == nullptr; }), caches.end());
    size_t places = 16;
    while (places < 4 * caches.size()) places *= 2;
    std::vector<const void*> seen(places, nullptr);
    for (const ternaspmm_cache_rows& c : caches) {
        size_t at = (reinterpret_cast<uintptr_t>(c.rows) * 0x9e3779b97f4a7c15ull >> 32) & (places - 1);
        for (; seen[at] != nullptr; at = (at + 1) & (places - 1))
            if (seen[at] == c.rows) refuse("%s: a cache is given twice", who);
        seen[at] = c.rows;
    }
    Guard guard;
    on_device_of(guard, path);
    Unlocked unlocked;
    const at::Tensor starts = start.contiguous(), lines = path.contiguous(), counts = count.contiguous();
    const int rc = caches.empty() || path.numel() == 0 ? 0 : lib.ternaspmm_cache_move(caches.data(), static_cast<int>(caches.size()), longs(starts), longs(lines), longs(counts), b, t, stream());
    unlocked.end();
    if (rc != 0) refuse("%s: the library refused the launch", who);
    Py_RETURN_NONE;
}

constexpr int64_t kInt8MaxRows = 1 << 28, kInt8MaxK = 131056;
// rows [R, K] of a type that the kernels read
void check_int8_rows(const char* who, const at::Tensor& x)
{
    check_device(who, "the rows", x, x);
    if (x.dim() != 2 || x.size(1) < 1 || x.size(1) > kInt8MaxK || x.size(0) > kInt8MaxRows) refuse("%s: rows [R, K] of 1 to 131056 columns, at most 2^28 of them", who);
}
at::Tensor rows_in_order(const at::Tensor& x) { return (x.size(1) == 1 || x.stride(1) == 1) && x.stride(0) >= 0 ? x : x.contiguous(); }

// (x [R, K] bf16 | fp32) -> (packed, scale [R])
TERNA_FUNCTION(int8_quantise, 1)
{
    const char* who = "quantise_rows";
    const at::Tensor& x = tensor(a[0]);
    if (x.scalar_type() != at::kBFloat16 && x.scalar_type() != at::kFloat) refuse("%s: rows are bfloat16 or float32", who);
    check_int8_rows(who, x);
    const int64_t r = x.size(0), k = x.size(1);
    Guard guard;
    on_device_of(guard, x);
    Unlocked unlocked;
    const at::Tensor rows = rows_in_order(x);
    at::Tensor packed = make({r == 0 ? 0 : lib.ternaspmm_int8_bytes(r, k)}, at::kByte, x), scale = make({r}, at::kFloat, x);
    const int rc = r == 0 ? 0
                          : lib.ternaspmm_int8_quantise(rows.const_data_ptr(), rows.stride(0), x.scalar_type() == at::kFloat, packed.mutable_data_ptr(), data<float>(&scale), r, k, stream());
    unlocked.end();
    if (rc != 0) refuse("%s: the library refused the launch", who);
    return pack(unlocked, std::move(packed), std::move(scale));
}

// (q int8 [R, K]) -> packed
TERNA_FUNCTION(int8_pack, 1)
{
    const char* who = "int8_rows";
    const at::Tensor& x = tensor(a[0]);
    if (x.scalar_type() != at::kChar) refuse("%s: rows are int8", who);
    check_int8_rows(who, x);
    const int64_t r = x.size(0), k = x.size(1);
    Guard guard;
    on_device_of(guard, x);
    Unlocked unlocked;
    const at::Tensor rows = rows_in_order(x);
    at::Tensor packed = make({r == 0 ? 0 : lib.ternaspmm_int8_bytes(r, k)}, at::kByte, x);
    const int rc = r == 0 ? 0 : lib.ternaspmm_int8_pack(rows.const_data_ptr(), rows.stride(0), packed.mutable_data_ptr(), r, k, stream());
    unlocked.end();
    if (rc != 0) refuse("%s: the library refused the launch", who);
    return THPVariable_Wrap(std::move(packed));
}

// packed rows and their scales, of R rows and K columns
struct Int8Side {
    at::Tensor packed, scale;

    Int8Side(const char* who, PyObject* p, PyObject* s, int64_t r, int64_t k, const at::Tensor& with) : packed(tensor(p)), scale(tensor(s))
    {
        check_device(who, "packed rows", packed, with);
        check_device(who, "scales", scale, with);
        if (r < 0 || r > kInt8MaxRows || k < 1 || k > kInt8MaxK || packed.scalar_type() != at::kByte || !packed.is_contiguous() || !aligned16(packed) ||
            packed.numel() != (r == 0 ? 0 : lib.ternaspmm_int8_bytes(r, k)) || scale.scalar_type() != at::kFloat || scale.dim() != 1 || scale.size(0) != r)
            refuse("%s: packed rows of another size, or scales that are not float32, one a row", who);
        scale = scale.contiguous();
    }
};

// (x | packed, x_scale | None, M, w packed, w_scale, N, K, float32) -> [M, N]
TERNA_FUNCTION(int8_linear, 8)
{
    const char* who = "int8_linear";
    const at::Tensor& x = tensor(a[0]);
    const bool given = a[1] != Py_None, fp32 = truth(a[7]);
    const int64_t n = integer(a[5]), k = integer(a[6]);
    check_device(who, "x", x, x);
    const Int8Side w(who, a[3], a[4], n, k, x);
    int64_t m = integer(a[2]);
    if (!given) {
        if (x.scalar_type() != at::kBFloat16 && x.scalar_type() != at::kFloat) refuse("%s: x is bfloat16 or float32 [M, K], or rows in 8 bits", who);
        check_int8_rows(who, x);
        if (x.size(1) != k) refuse("%s: x has %lld columns, the weights %lld", who, static_cast<long long>(x.size(1)), static_cast<long long>(k));
        m = x.size(0);
    }
    std::optional<Int8Side> rows8;
    Guard guard;
    on_device_of(guard, x);
    if (given) rows8.emplace(who, a[0], a[1], m, k, x);
    Unlocked unlocked;
    at::Tensor out = make({m, n}, fp32 ? at::kFloat : at::kBFloat16, x);
    if (out.numel() == 0) return wrap(std::move(out), unlocked);
    c10::DataPtr held;
    const void* packed = given ? rows8->packed.const_data_ptr() : nullptr;
    const float* scale = given ? rows8->scale.const_data_ptr<float>() : nullptr;
    int rc = 0;
    if (!given) {
        const at::Tensor rows = rows_in_order(x);
        const long long bytes = lib.ternaspmm_int8_bytes(m, k);
        held = device_allocator()->allocate(bytes + 4 * m);
        packed = held.get();
        float* const scales = reinterpret_cast<float*>(static_cast<uint8_t*>(held.get()) + bytes);
        scale = scales;
        rc = lib.ternaspmm_int8_quantise(rows.const_data_ptr(), rows.stride(0), x.scalar_type() == at::kFloat, held.get(), scales, m, k, stream());
    }
    const long long sums = lib.ternaspmm_int8_linear_workspace_bytes(m, n, k);
    const c10::DataPtr work = sums > 0 ? device_allocator()->allocate(sums) : c10::DataPtr();
    if (rc == 0) rc = lib.ternaspmm_int8_linear(packed, scale, w.packed.const_data_ptr(), w.scale.const_data_ptr<float>(), out.mutable_data_ptr(), fp32, work.get(), m, n, k, stream());
    unlocked.end();
    if (rc != 0) refuse("%s: the library refused the launch", who);
    return THPVariable_Wrap(std::move(out));
}

// (path of libternaspmm.so)
TERNA_FUNCTION(init, 1)
{
    const char* path = PyUnicode_AsUTF8(a[0]);
    if (path == nullptr) throw Refused();
    void* handle = dlopen(path, RTLD_NOW | RTLD_LOCAL);
    if (handle == nullptr) {
        PyErr_SetString(PyExc_ImportError, dlerror());
        throw Refused();
    }
#define X(name)                                                                                                        \
    if ((lib.name = reinterpret_cast<decltype(&::name)>(dlsym(handle, #name))) == nullptr) {                             \
        PyErr_SetString(PyExc_ImportError, "libternaspmm.so does not export " #name);                                  \
        throw Refused();                                                                                               \
    }
    TERNA_ENTRY_POINTS(X)
#undef X
    Py_RETURN_NONE;
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(init), METHOD(bit_linear), METHOD(bit_linear_bf16), METHOD(quant_input), METHOD(linear_packed), METHOD(linear_packed_decode_rule),
                         METHOD(linear_bf16_packed), METHOD(rmsnorm_quant), METHOD(relu2_mul_rmsnorm_quant), METHOD(quant_from_stats),
                         METHOD(fused_linear), METHOD(fused_linear_own_stats), METHOD(prompt_attention), METHOD(decode_attention), METHOD(block),
                         METHOD(attention_merge_rmsnorm_quant), METHOD(step_attention_merge), METHOD(step_inputs), METHOD(prompt_inputs), METHOD(decode_step),
                         METHOD(rotary_embed), METHOD(kv4_store), METHOD(kv4_rows), METHOD(kv4_attention), METHOD(kv4_step), METHOD(token_logprobs),
                         METHOD(draft_tree), METHOD(tree_attention), METHOD(tree_accept), METHOD(cache_move), METHOD(int8_quantise), METHOD(int8_pack), METHOD(int8_linear),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native() { return PyModule_Create(&module); }
