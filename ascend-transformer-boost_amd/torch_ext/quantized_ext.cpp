// The calls behind quantized.py: takes torch tensors apart, allocates results and workspaces from torch's allocator, and
// launches through the C ABI (atbmi_kernels.h) on torch's current stream of the tensors' device. A decode step's operators
// run for a few microseconds, as long as an interpreter takes to look at their arguments, so that is done here.
//
// Each function returns None, having done nothing, for arguments that are not what its operator takes: quantized.py then
// says what is wrong with them. It raises ValueError for what the C ABI refuses and RuntimeError for a failed launch.
// Arguments are positional; optional ones are None.
#include <algorithm>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include "atbmi_kernels.h"

namespace {
using at::Tensor;
using c10::ScalarType;

constexpr int INVALID_PARAM = 1; // the C ABI's code for arguments that it refuses

// The arguments of a call. `ok` ends false when one is not what it should be.
struct Args {
    PyObject *const *items;
    bool ok = true;

    bool Given(int i) const { return items[i] != Py_None; }
    const Tensor *Get(int i)
    {
        if (!THPVariable_Check(items[i])) {
            ok = false;
            return nullptr;
        }
        const Tensor &t = THPVariable_Unpack(items[i]);
        if (t.layout() != c10::kStrided) {
            ok = false;
            return nullptr;
        }
        return &t;
    }
    int64_t Int(int i)
    {
        const int64_t v = PyLong_Check(items[i]) ? PyLong_AsLongLong(items[i]) : -1;
        if (!PyLong_Check(items[i]) || (v == -1 && PyErr_Occurred())) {
            PyErr_Clear();
            ok = false;
        }
        return v;
    }
    float Float(int i)
    {
        const double v = PyFloat_AsDouble(items[i]);
        if (v == -1.0 && PyErr_Occurred()) {
            PyErr_Clear();
            ok = false;
        }
        return static_cast<float>(v);
    }
};

bool IsModelType(ScalarType t)
{
    return t == ScalarType::Half || t == ScalarType::BFloat16;
}

int32_t Code(ScalarType t)
{
    return t == ScalarType::BFloat16 ? ATBMI_BF16 : ATBMI_F16;
}

// What every tensor is held against: type, sizes, device.
bool Is(const Tensor *t, ScalarType type, at::IntArrayRef sizes, c10::Device device)
{
    return t != nullptr && t->scalar_type() == type && t->sizes() == sizes && t->device() == device;
}

bool IsWhole(const Tensor *t, ScalarType type, at::IntArrayRef sizes, c10::Device device)
{
    return Is(t, type, sizes, device) && t->is_contiguous();
}

// Row stride of a matrix whose rows have no gaps; below 0 if they have.
int64_t RowStride(const Tensor &t)
{
    if (t.size(1) > 1 && t.stride(1) != 1) {
        return -1;
    }
    return t.size(0) > 1 ? t.stride(0) : t.size(1);
}

// Token stride of [tokens, heads, channels] whose tokens have no gaps; below 0 if they have.
int64_t TokenStride(const Tensor &t)
{
    if ((t.size(2) > 1 && t.stride(2) != 1) || (t.size(1) > 1 && t.stride(1) != t.size(2))) {
        return -1;
    }
    return t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2);
}

void *Stream(c10::Device device)
{
    return c10::hip::getCurrentHIPStream(device.index()).stream();
}

Tensor Empty(at::IntArrayRef sizes, ScalarType type, c10::Device device)
{
    return at::empty(sizes, c10::TensorOptions().dtype(type).device(device));
}

// Address of a tensor's first value, null for no tensor. It raises for a tensor without memory of its own (torch.vmap's, a
// FakeTensor), so it is asked for in front of Unlocked and of anything that is done on the device.
template <typename T = void> T *At(const Tensor *t)
{
    return t != nullptr ? static_cast<T *>(t->data_ptr()) : nullptr;
}

// The C ABI is called without the interpreter's lock: a launch may wait for room in the device's queue.
template <typename F> int Unlocked(F call)
{
    struct Released {
        PyThreadState *const state = PyEval_SaveThread();
        ~Released() { PyEval_RestoreThread(state); } // (by an exception's way out as well)
    } const released;
    return call();
}

PyObject *Failed(int rc)
{
    return PyErr_Format(rc == INVALID_PARAM ? PyExc_ValueError : PyExc_RuntimeError, "%s", atbmi_last_error());
}

bool Count(Py_ssize_t have, Py_ssize_t want)
{
    if (have != want) {
        PyErr_Format(PyExc_TypeError, "%zd arguments, %zd expected", have, want);
    }
    return have == want;
}

// x, gamma, residual, epsilon, out, scale, residualOut
PyObject *RmsNormQuant(PyObject *, PyObject *const *items, Py_ssize_t count)
{
    HANDLE_TH_ERRORS
    if (!Count(count, 7)) {
        return nullptr;
    }
    Args a{items};
    const Tensor *x = a.Get(0), *gamma = a.Get(1);
    const float epsilon = a.Float(3);
    if (!a.ok || !x->is_cuda() || x->dim() != 2 || !IsModelType(x->scalar_type()) || x->size(1) == 0) {
        Py_RETURN_NONE;
    }
    const ScalarType type = x->scalar_type();
    const c10::Device device = x->device();
    const int64_t rows = x->size(0), dim = x->size(1);
    const int64_t xStride = RowStride(*x);
    if (xStride < 0 || !IsWhole(gamma, type, {dim}, device)) {
        Py_RETURN_NONE;
    }
    int64_t rStride = 0;
    const Tensor *residual = nullptr;
    if (a.Given(2)) {
        residual = a.Get(2);
        if (!Is(residual, type, x->sizes(), device) || (rStride = RowStride(*residual)) < 0) {
            Py_RETURN_NONE;
        }
    } else if (a.Given(6)) {
        Py_RETURN_NONE;
    }
    if ((a.Given(4) && !IsWhole(a.Get(4), ScalarType::Char, x->sizes(), device)) ||
        (a.Given(5) && !IsWhole(a.Get(5), ScalarType::Float, {rows}, device)) ||
        (a.Given(6) && !IsWhole(a.Get(6), type, x->sizes(), device))) {
        Py_RETURN_NONE;
    }
    const void *xAt = At(x), *rAt = At(residual), *gammaAt = At(gamma);
    const c10::DeviceGuard guard(device);
    Tensor out = a.Given(4) ? *a.Get(4) : Empty({rows, dim}, ScalarType::Char, device);
    Tensor scale = a.Given(5) ? *a.Get(5) : Empty({rows}, ScalarType::Float, device);
    Tensor sum = a.Given(6) ? *a.Get(6) : (residual ? Empty({rows, dim}, type, device) : *x);
    int8_t *outAt = At<int8_t>(&out);
    float *scaleAt = At<float>(&scale);
    void *sumAt = residual ? At(&sum) : nullptr;
    void *stream = Stream(device);
    const int rc = rows == 0 ? 0 : Unlocked([&] {
        return atbmi_rms_norm_quant(xAt, rAt, gammaAt, outAt, scaleAt, sumAt, rows, dim, xStride, rStride, Code(type), epsilon,
                                    stream);
    });
    if (rc != 0) {
        return Failed(rc);
    }
    PyObject *got = PyTuple_New(3);
    if (got == nullptr) {
        return nullptr;
    }
    auto give = [&](int i, int from, const Tensor &t) { // the very object that was handed in, where one was
        PyObject *object = from >= 0 ? items[from] : nullptr;
        Py_XINCREF(object);
        PyTuple_SET_ITEM(got, i, object ? object : THPVariable_Wrap(t));
    };
    give(0, a.Given(4) ? 4 : -1, out);
    give(1, a.Given(5) ? 5 : -1, scale);
    give(2, a.Given(6) ? 6 : (residual ? -1 : 0), sum);
    return got;
    END_HANDLE_TH_ERRORS
}

// x, weight, xScale, weightScale, bias, outDtype, out
PyObject *LinearInt8(PyObject *, PyObject *const *items, Py_ssize_t count)
{
    HANDLE_TH_ERRORS
    if (!Count(count, 7)) {
        return nullptr;
    }
    Args a{items};
    const Tensor *x = a.Get(0), *w = a.Get(1), *xScale = a.Get(2), *wScale = a.Get(3);
    if (!a.ok || !x->is_cuda() || x->dim() != 2 || w->dim() != 2) {
        Py_RETURN_NONE;
    }
    const c10::Device device = x->device();
    const int64_t m = x->size(0), k = x->size(1), n = w->size(0);
    const int64_t xStride = RowStride(*x), wStride = RowStride(*w);
    const Tensor *bias = a.Given(4) ? a.Get(4) : nullptr;
    if (!Is(x, ScalarType::Char, {m, k}, device) || !Is(w, ScalarType::Char, {n, k}, device) || xStride < 0 || wStride < 0 ||
        !IsWhole(xScale, ScalarType::Float, {m}, device) || !IsWhole(wScale, ScalarType::Float, {n}, device) ||
        (a.Given(4) && !IsWhole(bias, ScalarType::Float, {n}, device)) || (a.Given(5) && !THPDtype_Check(items[5])) ||
        (!a.Given(5) && !a.Given(6))) {
        Py_RETURN_NONE;
    }
    const Tensor *given = a.Given(6) ? a.Get(6) : nullptr;
    if (!a.ok) {
        Py_RETURN_NONE;
    }
    const ScalarType type = a.Given(5) ? reinterpret_cast<THPDtype *>(items[5])->scalar_type : given->scalar_type();
    if (!IsModelType(type) || (given && (!Is(given, type, {m, n}, device) || RowStride(*given) < 0))) {
        Py_RETURN_NONE;
    }
    const int8_t *xAt = At<int8_t>(x), *wAt = At<int8_t>(w);
    const float *xScaleAt = At<float>(xScale), *wScaleAt = At<float>(wScale), *biasAt = At<float>(bias);
    const c10::DeviceGuard guard(device);
    Tensor out = given ? *given : Empty({m, n}, type, device);
    if (m != 0 && n != 0) {
        uint64_t need = 0;
        int rc = atbmi_linear_int8_workspace_size(m, n, k, &need);
        if (rc != 0) {
            return Failed(rc);
        }
        Tensor workspace;
        if (need > 0) {
            workspace = Empty({static_cast<int64_t>(need)}, ScalarType::Byte, device);
        }
        void *outAt = At(&out), *at = need > 0 ? At(&workspace) : nullptr;
        const int64_t outStride = RowStride(out);
        void *stream = Stream(device);
        rc = Unlocked([&] {
            return atbmi_linear_int8(xAt, wAt, xScaleAt, wScaleAt, biasAt, outAt, m, n, k, xStride, wStride, outStride, Code(type),
                                     at, need, stream);
        });
        if (rc != 0) {
            return Failed(rc);
        }
    }
    if (given) {
        Py_INCREF(items[6]);
        return items[6];
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// The cache's four tensors, from argument `at` on.
struct Cache {
    const Tensor *kc = nullptr, *vc = nullptr, *kp = nullptr, *vp = nullptr;
    ScalarType type = ScalarType::Undefined;
    c10::Device device{c10::kCPU};
    int64_t blocks = 0, heads = 0, block = 0, half = 0;
    uint8_t *keys = nullptr, *values = nullptr; // where they lie: see At
    void *keyParams = nullptr, *valueParams = nullptr;

    bool Read(Args &a, int at)
    {
        kc = a.Get(at), vc = a.Get(at + 1), kp = a.Get(at + 2), vp = a.Get(at + 3);
        if (!a.ok || !kc->is_cuda() || kc->dim() != 4 || !IsModelType(kp->scalar_type())) {
            return false;
        }
        type = kp->scalar_type();
        device = kc->device();
        blocks = kc->size(0), heads = kc->size(1), block = kc->size(2), half = kc->size(3);
        return IsWhole(kc, ScalarType::Byte, kc->sizes(), device) &&
               IsWhole(vc, ScalarType::Byte, {blocks, heads, half, block}, device) &&
               IsWhole(kp, type, {blocks, heads, block, 2}, device) && IsWhole(vp, type, {blocks, heads, block, 2}, device);
    }
    void Locate()
    {
        keys = At<uint8_t>(kc), values = At<uint8_t>(vc), keyParams = At(kp), valueParams = At(vp);
    }
};

// key, value, keyCache, valueCache, keyParams, valueParams, slotMapping -> True
PyObject *ReshapeAndCacheInt4(PyObject *, PyObject *const *items, Py_ssize_t count)
{
    HANDLE_TH_ERRORS
    if (!Count(count, 7)) {
        return nullptr;
    }
    Args a{items};
    Cache c;
    const Tensor *key = a.Get(0), *value = a.Get(1), *slots = a.Get(6);
    if (!c.Read(a, 2) || key->dim() != 3) {
        Py_RETURN_NONE;
    }
    const int64_t tokens = key->size(0), d = 2 * c.half;
    if (!Is(key, c.type, {tokens, c.heads, d}, c.device) || !Is(value, c.type, {tokens, c.heads, d}, c.device) ||
        !IsWhole(slots, ScalarType::Int, {tokens}, c.device) || TokenStride(*key) < 0 || TokenStride(*value) < 0) {
        Py_RETURN_NONE;
    }
    if (tokens != 0) {
        c.Locate();
        const void *keyAt = At(key), *valueAt = At(value);
        const int32_t *slotsAt = At<int32_t>(slots);
        const int64_t keyStride = TokenStride(*key), valueStride = TokenStride(*value);
        const c10::DeviceGuard guard(c.device);
        void *stream = Stream(c.device);
        const int rc = Unlocked([&] {
            return atbmi_reshape_and_cache_int4(keyAt, valueAt, c.keys, c.values, c.keyParams, c.valueParams, slotsAt, tokens,
                                                c.heads, d, c.block, c.blocks, keyStride, valueStride, Code(c.type), stream);
        });
        if (rc != 0) {
            return Failed(rc);
        }
    }
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// keyCache, valueCache, keyParams, valueParams, blockTables, seqLens, totalRows, seqStarts, maxSeqLen, key, value
PyObject *PagedCacheLoadInt4(PyObject *, PyObject *const *items, Py_ssize_t count)
{
    HANDLE_TH_ERRORS
    if (!Count(count, 11)) {
        return nullptr;
    }
    Args a{items};
    Cache c;
    const Tensor *tables = a.Get(4), *lens = a.Get(5), *starts = a.Given(7) ? a.Get(7) : nullptr;
    const int64_t rows = a.Int(6);
    if (!c.Read(a, 0) || tables->dim() != 2 || rows < 0) {
        Py_RETURN_NONE;
    }
    const int64_t batch = tables->size(0), reach = tables->size(1), d = 2 * c.half;
    const int64_t longest = a.Given(8) ? a.Int(8) : reach * c.block;
    if (!a.ok || !IsWhole(tables, ScalarType::Int, {batch, reach}, c.device) ||
        !IsWhole(lens, ScalarType::Int, {batch}, c.device) ||
        (starts && !IsWhole(starts, ScalarType::Int, {batch}, c.device)) ||
        (a.Given(9) && !IsWhole(a.Get(9), c.type, {rows, c.heads, d}, c.device)) ||
        (a.Given(10) && !IsWhole(a.Get(10), c.type, {rows, c.heads, d}, c.device))) {
        Py_RETURN_NONE;
    }
    c.Locate();
    const int32_t *tablesAt = At<int32_t>(tables), *lensAt = At<int32_t>(lens), *startsAt = At<int32_t>(starts);
    const c10::DeviceGuard guard(c.device);
    Tensor key = a.Given(9) ? *a.Get(9) : Empty({rows, c.heads, d}, c.type, c.device);
    Tensor value = a.Given(10) ? *a.Get(10) : Empty({rows, c.heads, d}, c.type, c.device);
    if (batch != 0 && reach != 0 && rows != 0) {
        void *keyAt = At(&key), *valueAt = At(&value);
        void *stream = Stream(c.device);
        const int rc = Unlocked([&] {
            return atbmi_paged_cache_load_int4(c.keys, c.values, c.keyParams, c.valueParams, tablesAt, lensAt, startsAt, keyAt,
                                               valueAt, batch, reach, c.heads, d, c.block, c.blocks, rows, longest, Code(c.type),
                                               stream);
        });
        if (rc != 0) {
            return Failed(rc);
        }
    }
    PyObject *got = PyTuple_New(2);
    if (got == nullptr) {
        return nullptr;
    }
    for (int i = 0; i < 2; ++i) {
        PyObject *object = a.Given(9 + i) ? items[9 + i] : nullptr;
        Py_XINCREF(object);
        PyTuple_SET_ITEM(got, i, object ? object : THPVariable_Wrap(i == 0 ? key : value));
    }
    return got;
    END_HANDLE_TH_ERRORS
}

// query, keyCache, valueCache, keyParams, valueParams, blockTables, contextLens, qkScale, queryTokens, mask, out, workspace
PyObject *PagedAttentionInt4(PyObject *, PyObject *const *items, Py_ssize_t count)
{
    HANDLE_TH_ERRORS
    if (!Count(count, 12)) {
        return nullptr;
    }
    Args a{items};
    Cache c;
    const Tensor *query = a.Get(0), *tables = a.Get(5), *lens = a.Get(6);
    const float scale = a.Float(7);
    const int64_t tokens = a.Int(8);
    constexpr int64_t MOST = 0x7fffffff;
    if (!c.Read(a, 1) || query->dim() != 3 || tables->dim() != 2 || tokens < 1 || tokens > MOST) {
        Py_RETURN_NONE;
    }
    const int64_t batch = tables->size(0), reach = tables->size(1), heads = query->size(1), d = 2 * c.half;
    if (std::max({batch, reach, heads, c.heads, c.block, c.blocks, d}) > MOST || // (the C ABI's fields have 32 bits)
        !IsWhole(query, c.type, {batch * tokens, heads, d}, c.device) ||
        !IsWhole(tables, ScalarType::Int, {batch, reach}, c.device) || !IsWhole(lens, ScalarType::Int, {batch}, c.device) ||
        (a.Given(10) && !IsWhole(a.Get(10), c.type, query->sizes(), c.device)) ||
        (a.Given(11) && !IsWhole(a.Get(11), ScalarType::Byte, {a.Get(11) ? a.Get(11)->numel() : 0}, c.device))) {
        Py_RETURN_NONE;
    }
    AtbmiPaInt4Call call{};
    if (a.Given(9)) {
        const Tensor *mask = a.Get(9);
        if (!a.ok || mask->dim() != 4 || !Is(mask, c.type, mask->sizes(), c.device) || mask->size(3) < 1 ||
            mask->size(3) > MOST || (mask->size(3) > 1 && mask->stride(3) != 1)) {
            Py_RETURN_NONE;
        }
        const int64_t want[3] = {batch, heads, tokens};
        int64_t *const strides[3] = {&call.maskSeqStride, &call.maskHeadStride, &call.maskRowStride};
        for (int i = 0; i < 3; ++i) {
            if (mask->size(i) != 1 && mask->size(i) != want[i]) {
                Py_RETURN_NONE;
            }
            *strides[i] = mask->size(i) > 1 ? mask->stride(i) : 0;
        }
        call.mask = At(mask);
        call.maskLen = static_cast<int32_t>(mask->size(3));
    }
    c.Locate();
    call.query = At(query);
    call.keyCache = c.keys;
    call.valueCache = c.values;
    call.keyParams = c.keyParams;
    call.valueParams = c.valueParams;
    call.blockTables = At<int32_t>(tables);
    call.contextLens = At<int32_t>(lens);
    const c10::DeviceGuard guard(c.device);
    Tensor out = a.Given(10) ? *a.Get(10) : Empty(query->sizes(), c.type, c.device);
    if (batch != 0) {
        call.dtype = Code(c.type);
        call.numHeads = static_cast<int32_t>(heads);
        call.numKvHeads = static_cast<int32_t>(c.heads);
        call.headDim = static_cast<int32_t>(d);
        call.blockSize = static_cast<int32_t>(c.block);
        call.numBlocks = static_cast<int32_t>(c.blocks);
        call.maxBlocksPerSeq = static_cast<int32_t>(reach);
        call.batch = static_cast<int32_t>(batch);
        call.queryTokens = static_cast<int32_t>(tokens);
        call.qkScale = scale;
        call.out = At(&out);
        uint64_t need = 0;
        int rc = atbmi_pa_int4_workspace_size(&call, &need);
        if (rc != 0) {
            return Failed(rc);
        }
        Tensor workspace;
        if (a.Given(11)) {
            workspace = *a.Get(11);
        } else if (need > 0) {
            workspace = Empty({static_cast<int64_t>(need)}, ScalarType::Byte, c.device);
        }
        const uint64_t size = workspace.defined() ? static_cast<uint64_t>(workspace.numel()) : 0;
        void *at = size > 0 ? At(&workspace) : nullptr;
        void *stream = Stream(c.device);
        rc = Unlocked([&] { return atbmi_pa_int4_decode(&call, at, size, stream); });
        if (rc != 0) {
            return Failed(rc);
        }
    }
    if (a.Given(10)) {
        Py_INCREF(items[10]);
        return items[10];
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

#define ATBMI_METHOD(name, function)                                                                                      \
    {                                                                                                                      \
        name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(function)), METH_FASTCALL, nullptr                \
    }
PyMethodDef METHODS[] = {ATBMI_METHOD("rms_norm_quant", RmsNormQuant),
                         ATBMI_METHOD("linear_int8", LinearInt8),
                         ATBMI_METHOD("reshape_and_cache_int4", ReshapeAndCacheInt4),
                         ATBMI_METHOD("paged_cache_load_int4", PagedCacheLoadInt4),
                         ATBMI_METHOD("paged_attention_int4", PagedAttentionInt4),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef MODULE = {PyModuleDef_HEAD_INIT, "quantized_ext", nullptr, -1, METHODS, nullptr, nullptr, nullptr, nullptr};
} // namespace

PyMODINIT_FUNC PyInit_quantized_ext()
{
    return PyModule_Create(&MODULE);
}
