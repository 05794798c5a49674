// The 4-bit cache's operators as a CPython extension over the C ABI: checks of the tensors,
// outputs and workspaces, then one call of libpagedkv.so.  pagedcore_b200/int4.py documents
// them and is how they are called.
//
// Why compiled: a decode layer of one sequence is 4 us on the GPU, and the same checks with
// their allocations and a ctypes call of 26 arguments took 15 us of Python.
//
// Nothing is thrown out of an entry point: a refusal is a ValueError, whatever libtorch throws
// a RuntimeError.

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>
#include <optional>
#include <string>
#include <utility>

#include "pagedkv.h"

namespace {

constexpr int64_t kQueryHeads = PKV_QUERY_HEADS, kKvHeads = PKV_KV_HEADS, kDim = PKV_HEAD_DIM;
constexpr int64_t kRow = kQueryHeads * kDim;  // values of a query row
constexpr int64_t kBlockTokens = PKV_BLOCK_TOKENS;
constexpr int64_t kMost = INT32_MAX - (1 << 16);  // rows and list entries: the C ABI's int32, and a step of a row loop

struct Refusal {
    std::string message;
};

[[noreturn]] void refuse(std::string message) { throw Refusal{std::move(message)}; }

struct PythonError {};  // already set

std::string on_device(int index) { return " on cuda:" + std::to_string(index); }

// -- arguments -----------------------------------------------------------------------
const at::Tensor &tensor_of(PyObject *object, const char *name) {
    if (!THPVariable_Check(object)) {
        PyErr_Format(PyExc_TypeError, "%s must be a tensor", name);
        throw PythonError{};
    }
    return THPVariable_Unpack(object);
}

// A tensor or, for None, null.
const at::Tensor *maybe(PyObject *object, const char *name) {
    return object == Py_None ? nullptr : &tensor_of(object, name);
}

int64_t int_of(PyObject *object) {
    const long long value = PyLong_AsLongLong(object);
    if (value == -1 && PyErr_Occurred()) throw PythonError{};
    return value;
}

int32_t int32_of(PyObject *object, const char *name) {
    const int64_t value = int_of(object);
    if (value < INT32_MIN || value > kMost) refuse(std::string(name) + " must be at most " + std::to_string(kMost) + ", not " + std::to_string(value));
    return static_cast<int32_t>(value);
}

void fits(const char *name, int64_t count) {
    if (count > kMost) refuse(std::string(name) + " must be at most " + std::to_string(kMost) + ", not " + std::to_string(count));
}

struct Cache {
    void *storage;
    int32_t layers;
    int32_t blocks;
    int index;  // CUDA device
};

Cache cache_of(PyObject *object) {
    const at::Tensor &storage = tensor_of(object, "storage");
    if (storage.dim() != 3 || storage.size(2) != PKV_INT4_BLOCK_BYTES || storage.scalar_type() != at::kByte ||
        !storage.is_contiguous()) {
        refuse("a 4-bit cache is contiguous uint8 [layers, blocks, 4608]");
    }
    if (storage.size(0) < 1 || storage.size(1) < 1) refuse("a 4-bit cache needs at least one layer and one block");
    fits("layers", storage.size(0));
    fits("blocks", storage.size(1));
    if (!storage.is_cuda()) refuse("4-bit operators need CUDA tensors");
    return {storage.data_ptr(), static_cast<int32_t>(storage.size(0)), static_cast<int32_t>(storage.size(1)),
            storage.get_device()};
}

// Address of `count` or more int32 values on the device.
int32_t *int_list(const at::Tensor &tensor, const char *name, int64_t count, int index) {
    fits(name, count);
    if (tensor.scalar_type() != at::kInt || tensor.numel() < count || !tensor.is_cuda() || tensor.get_device() != index ||
        !tensor.is_contiguous()) {
        refuse(std::string(name) + " must hold " + std::to_string(count) + " contiguous int32 values" + on_device(index));
    }
    return static_cast<int32_t *>(tensor.data_ptr());
}

int32_t *int_list(PyObject *object, const char *name, int64_t count, int index) {
    return int_list(tensor_of(object, name), name, count, index);
}

bool here(const at::Tensor &tensor, int index) { return tensor.is_cuda() && tensor.get_device() == index; }

const void *rope_of(const at::Tensor &table, int index) {
    if (table.scalar_type() != at::kHalf || !here(table, index) || table.dim() != 3 || table.size(0) != 2 ||
        table.size(1) != PKV_CONTEXT_LIMIT || table.size(2) != kDim / 2 || !table.is_contiguous()) {
        refuse("rope_table must be contiguous FP16 [2, 2048, 32]" + on_device(index));
    }
    return table.data_ptr();
}

struct Norms {
    const void *query = nullptr;
    const void *key = nullptr;
    double eps = 0;
};

// From three arguments: both weights (or None) and eps.
Norms norms_of(PyObject *const *args, const Cache &cache) {
    if (args[0] == Py_None && args[1] == Py_None) return {};
    Norms norms;
    for (int i = 0; i < 2; ++i) {
        const at::Tensor &weight = tensor_of(args[i], "head norms");
        if (weight.scalar_type() != at::kHalf || !here(weight, cache.index) || weight.dim() != 2 ||
            weight.size(0) != cache.layers || weight.size(1) != kDim || !weight.is_contiguous() ||
            reinterpret_cast<uintptr_t>(weight.data_ptr()) % 16) {
            refuse("head norms must be contiguous, 16-byte aligned FP16 [" + std::to_string(cache.layers) + ", 64]" +
                   on_device(cache.index));
        }
        (i == 0 ? norms.query : norms.key) = weight.data_ptr();
    }
    norms.eps = PyFloat_AsDouble(args[2]);
    if (norms.eps == -1.0 && PyErr_Occurred()) throw PythonError{};
    if (!(norms.eps >= 0)) refuse("eps must not be negative");
    return norms;
}

void half_rows(const at::Tensor &tensor, const char *name, int index) {
    if (tensor.scalar_type() != at::kHalf || !here(tensor, index)) refuse(std::string(name) + " must be FP16" + on_device(index));
}

// -- rows ------------------------------------------------------------------------------
bool aligned(const at::Tensor &tensor) { return reinterpret_cast<uintptr_t>(tensor.data_ptr()) % 16 == 0; }

// Inner [heads, 64] contiguous and rows 16-byte aligned: [..., rows, heads, 64].
bool rows_ok(const at::Tensor &tensor) {
    const auto s = tensor.strides();
    const auto n = s.size();
    return s[n - 1] == 1 && s[n - 2] == kDim && s[0] % 8 == 0 && s[n - 3] % 8 == 0 && aligned(tensor);
}

// A copy in contiguous, 16-byte aligned storage (contiguous() keeps an unaligned tensor).
at::Tensor dense(const at::Tensor &tensor) { return tensor.clone(at::MemoryFormat::Contiguous); }

// A tensor used as it is, or its copy where the kernels cannot take it.
struct Rows {
    const at::Tensor *given;
    at::Tensor copy;

    explicit Rows(const at::Tensor &tensor) : given(&tensor) {}
    const at::Tensor &get() const { return copy.defined() ? copy : *given; }
    void make_dense() { copy = dense(get()); }
    void *data() const { return get().data_ptr(); }
    int64_t stride(int dim) const { return get().stride(dim); }
};

// Row stride of [rows, heads, 64] for the kernels: of one row it may be anything.
int64_t row_stride(const at::Tensor &tensor) { return tensor.size(0) == 1 ? kRow : tensor.stride(0); }

// Query [rows, 32, 64], copied where the kernels cannot take its rows.
void take_query(Rows &query) {
    const at::Tensor &q = query.get();
    const bool ok = q.stride(2) == 1 && q.stride(1) == kDim && aligned(q) &&
                    (q.size(0) == 1 || (q.stride(0) >= kRow && q.stride(0) % 8 == 0));
    if (!ok) query.make_dense();
}

// K and V, copied where they have no common strides that the kernels take.
void take_pair(Rows &key, Rows &value) {
    if (value.get().strides() == key.get().strides() && rows_ok(key.get()) && aligned(value.get())) return;
    key.make_dense();
    value.make_dense();
}

void check_query(const at::Tensor &query, int index, const char *rows, bool fp32) {
    if (query.dim() != 3 || query.size(0) < 1 || query.size(1) != kQueryHeads || query.size(2) != kDim) {
        refuse(std::string("query must be FP16 [") + rows + ", 32, 64] of a nonempty " + rows);
    }
    fits(rows, query.size(0));
    if (fp32 && query.scalar_type() == at::kFloat && here(query, index)) return;
    half_rows(query, "query", index);
}

// The output [rows, 32, 64]: the given one, checked, or a new one.
at::Tensor output(const at::Tensor *out, int64_t rows, int index, const char *what) {
    if (out == nullptr) {
        return at::detail::empty_cuda({rows, kQueryHeads, kDim}, at::kHalf, at::Device(at::kCUDA, index), std::nullopt);
    }
    if (out->dim() != 3 || out->size(0) != rows || out->size(1) != kQueryHeads || out->size(2) != kDim ||
        out->scalar_type() != at::kHalf || !here(*out, index)) {
        refuse("out must be FP16 [" + std::to_string(rows) + ", 32, 64]" + on_device(index));
    }
    if (!rows_ok(*out)) refuse(std::string("out must be FP16 [") + what + ", 32, 64] with contiguous, 16-byte aligned rows");
    if (rows > 1 && out->stride(0) < kRow) refuse("the rows of out overlap");
    return *out;
}

// Whether rows of `a` and of `b`, [..., rows, heads, 64] with contiguous [heads, 64], share memory.
// Exact where the rows of both lie in the same pattern (views of one projection), else by the
// ranges that they span.
bool share(const at::Tensor &a, const at::Tensor &b) {
    const auto reach = [](const at::Tensor &t) {  // bytes from the first to the end of the last
        const int64_t n = t.dim();
        int64_t values = t.size(n - 2) * kDim;
        for (int64_t d = 0; d < n - 2; ++d) values += (t.size(d) - 1) * t.stride(d);
        return static_cast<int64_t>(t.element_size()) * values;
    };
    if (a.numel() == 0 || b.numel() == 0) return false;
    const int64_t apart = static_cast<int64_t>(reinterpret_cast<uintptr_t>(b.data_ptr()) - reinterpret_cast<uintptr_t>(a.data_ptr()));
    if (apart >= reach(a) || -apart >= reach(b)) return false;
    const int64_t n = a.dim();
    const auto pitch = [n](const at::Tensor &t) { return static_cast<int64_t>(t.element_size()) * t.stride(n - 3); };
    bool same = b.dim() == n && pitch(a) == pitch(b) && pitch(a) > 0;
    if (n == 4) {
        const auto layer = [](const at::Tensor &t) { return static_cast<int64_t>(t.element_size()) * t.stride(0); };
        same = same && layer(a) == layer(b) && layer(a) % pitch(a) == 0;
    }
    if (!same) return true;
    const int64_t at = (apart % pitch(a) + pitch(a)) % pitch(a);  // where rows of b begin within those of a
    const auto width = [n](const at::Tensor &t) { return static_cast<int64_t>(t.element_size()) * t.size(n - 2) * kDim; };
    return at < width(a) || at + width(b) > pitch(a);
}

// Whether `rows` lie where `out` is written, other than as the same rows.
bool within(const at::Tensor &rows, const at::Tensor &out) {
    if (rows.data_ptr() == out.data_ptr() && rows.sizes() == out.sizes() && rows.strides() == out.strides() &&
        rows.scalar_type() == out.scalar_type()) {
        return false;
    }
    return share(rows, out);
}

void check_status(int status) {
    if (status == PKV_OK) return;
    const std::string message = pkv_last_error();
    if (status == PKV_VALUE_ERROR) refuse(message);
    PyErr_SetString(PyExc_RuntimeError, message.c_str());
    throw PythonError{};
}

// Runs `call` with the current stream of device `index`, whatever the current device is.  Other
// threads run meanwhile: a launch waits where the stream's queue is full.
template <typename Call>
void launch(int index, Call call) {
    const c10::cuda::OptionalCUDAGuard guard(at::Device(at::kCUDA, index));
    void *const stream = c10::cuda::getCurrentCUDAStream(index).stream();
    PyThreadState *const thread = PyEval_SaveThread();
    const int status = call(stream);  // throws nothing
    PyEval_RestoreThread(thread);
    check_status(status);
}

at::Tensor bytes(int64_t count, int index) {
    return at::detail::empty_cuda({count}, at::kByte, at::Device(at::kCUDA, index), std::nullopt);
}

// -- operators ----------------------------------------------------------------------------
// (storage)
PyObject *check_cache(PyObject *const *args) {
    cache_of(args[0]);
    Py_RETURN_NONE;
}

// (storage, query_norm, key_norm, eps)
PyObject *check_norms(PyObject *const *args) {
    const Cache cache = cache_of(args[0]);
    tensor_of(args[1], "head norms");
    norms_of(args + 1, cache);
    Py_RETURN_NONE;
}

// (rows, out): whether [rows, heads, 64] lie where [rows, 32, 64] are written, other than as the same rows.
PyObject *overlaps(PyObject *const *args) {
    const at::Tensor &rows = tensor_of(args[0], "rows"), &out = tensor_of(args[1], "out");
    if (rows.dim() != 3 || out.dim() != 3) refuse("rows and out must have three dimensions");
    if (rows.numel() == 0 || out.numel() == 0 || !within(rows, out)) Py_RETURN_FALSE;
    Py_RETURN_TRUE;
}

// Whether the rows of [layers, tokens, 32, 64] do not overlap: one of the two dimensions within the other.
bool rows_apart(const at::Tensor &rows) {
    const int64_t layers = rows.size(0), tokens = rows.size(1), over = rows.stride(0), within_ = rows.stride(1);
    if (layers < 2 || tokens < 2) return (layers < 2 || over >= kRow) && (tokens < 2 || within_ >= kRow);
    if (over < within_) return over >= kRow && within_ >= (layers - 1) * over + kRow;
    return within_ >= kRow && over >= (tokens - 1) * within_ + kRow;
}

// (storage, key, value, slots, layer_begin, error_flag, positions, rope_table, query, query_out, query_norm, key_norm, eps)
PyObject *append_kv(PyObject *const *args) {
    const Cache cache = cache_of(args[0]);
    const int index = cache.index;
    Rows key(tensor_of(args[1], "key")), value(tensor_of(args[2], "value"));
    const at::Tensor &k = key.get();
    if (k.dim() != 4 || k.size(2) != kKvHeads || k.size(3) != kDim || value.get().sizes() != k.sizes()) {
        refuse("K and V must share FP16 [layers, tokens, 4, 64]");
    }
    half_rows(k, "key", index);
    half_rows(value.get(), "value", index);
    const int64_t layers = k.size(0), tokens = k.size(1);
    fits("layers", layers);
    const int32_t *const slots = int_list(args[3], "slots", tokens, index);
    const int32_t layer_begin = int32_of(args[4], "layer_begin");
    int32_t *const flag = int_list(args[5], "error_flag", 1, index);
    const at::Tensor *const positions = maybe(args[6], "positions"), *const table = maybe(args[7], "rope_table");
    const at::Tensor *const given = maybe(args[8], "query"), *const out = maybe(args[9], "query_out");
    if ((table == nullptr) != (positions == nullptr) || (given != nullptr && table == nullptr)) {
        refuse("rope_table goes with positions, query with both");
    }
    if (out != nullptr && given == nullptr) refuse("query_out goes with query");
    if ((args[10] != Py_None || args[11] != Py_None) && table == nullptr) refuse("norms go with rope_table");
    const void *const rope = table != nullptr ? rope_of(*table, index) : nullptr;
    const int32_t *const at_positions = table != nullptr ? int_list(*positions, "positions", tokens, index) : nullptr;
    const Norms norms = norms_of(args + 10, cache);
    at::Tensor result, query;
    if (given != nullptr) {
        if (given->dim() != 4 || given->size(0) != layers || given->size(1) != tokens || given->size(2) != kQueryHeads ||
            given->size(3) != kDim) {
            refuse("query must be FP16 [layers, tokens, 32, 64]");
        }
        half_rows(*given, "query", index);
        if (out == nullptr) {
            result = at::detail::empty_cuda(given->sizes(), at::kFloat, at::Device(at::kCUDA, index), std::nullopt);
        } else {
            if (out->sizes() != given->sizes() || !rows_ok(*out) || !rows_apart(*out)) {
                refuse("query_out must be [layers, tokens, 32, 64] with contiguous, 16-byte aligned rows");
            }
            if ((out->scalar_type() != at::kHalf && out->scalar_type() != at::kFloat) || !here(*out, index)) {
                refuse("query_out must be FP16 or FP32" + on_device(index));
            }
            result = *out;
        }
        query = given->numel() != 0 && (!rows_ok(*given) || (out != nullptr && within(*given, *out))) ? dense(*given) : *given;
    }
    if (layers != 0 && tokens != 0) {
        take_pair(key, value);
        if (out != nullptr && (share(key.get(), *out) || share(value.get(), *out))) {  // read while queries are written
            key.make_dense();
            value.make_dense();
        }
        const bool rotates = query.defined();
        launch(index, [&](void *stream) {
            return pkv_int4_append_kv(
                cache.storage, cache.layers, cache.blocks, layer_begin, static_cast<int32_t>(layers), key.data(),
                value.data(), key.stride(0), key.stride(1), slots, at_positions, static_cast<int32_t>(tokens), rope,
                norms.query, norms.key, norms.eps, rotates ? query.data_ptr() : nullptr, rotates ? query.stride(0) : 0,
                rotates ? query.stride(1) : 0, rotates ? result.data_ptr() : nullptr,
                rotates && result.scalar_type() == at::kFloat, rotates ? result.stride(0) : 0,
                rotates ? result.stride(1) : 0, flag, stream);
        });
    }
    if (out != nullptr) return Py_NewRef(args[9]);
    if (!result.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(result));
}

// (storage, layer, blocks, error_flag)
PyObject *read_blocks(PyObject *const *args) {
    const Cache cache = cache_of(args[0]);
    const int32_t layer = int32_of(args[1], "layer");
    const at::Tensor &blocks = tensor_of(args[2], "blocks");
    const int64_t count = blocks.numel();
    const int32_t *const list = int_list(blocks, "blocks", count, cache.index);
    int32_t *const flag = int_list(args[3], "error_flag", 1, cache.index);
    const at::Device device(at::kCUDA, cache.index);
    at::Tensor key = at::detail::empty_cuda({count, kBlockTokens, kKvHeads, kDim}, at::kHalf, device, std::nullopt);
    at::Tensor value = at::detail::empty_cuda({count, kBlockTokens, kKvHeads, kDim}, at::kHalf, device, std::nullopt);
    if (count != 0) {
        launch(cache.index, [&](void *stream) {
            return pkv_int4_read_blocks(cache.storage, cache.layers, cache.blocks, layer, list, static_cast<int32_t>(count),
                                        key.data_ptr(), value.data_ptr(), flag, stream);
        });
    }
    PyObject *const first = THPVariable_Wrap(std::move(key));
    if (first == nullptr) return nullptr;
    PyObject *const second = THPVariable_Wrap(std::move(value));
    if (second == nullptr) {
        Py_DECREF(first);
        return nullptr;
    }
    PyObject *const pair = PyTuple_New(2);
    if (pair == nullptr) {
        Py_DECREF(first);
        Py_DECREF(second);
        return nullptr;
    }
    PyTuple_SET_ITEM(pair, 0, first);
    PyTuple_SET_ITEM(pair, 1, second);
    return pair;
}

// The batch's tables: (lengths, prefix, flat, total_blocks, error_flag) from `args`.
struct Batch {
    int32_t rows, total, grid;
    int32_t *lengths, *prefix, *flat, *flag;
    int64_t workspace_bytes;

    Batch(PyObject *const *args, int64_t count, int index) {
        rows = static_cast<int32_t>(count);
        total = int32_of(args[3], "total_blocks");
        check_status(pkv_int4_decode_plan(index, rows, total, &grid, &workspace_bytes));
        lengths = int_list(args[0], "lengths", count, index);
        prefix = int_list(args[1], "prefix", count + 1, index);
        flat = int_list(args[2], "flat", total, index);
        flag = int_list(args[4], "error_flag", 1, index);
    }
};

// (storage, layer, query, lengths, prefix, flat, total_blocks, error_flag, out)
PyObject *decode_attention(PyObject *const *args) {
    const Cache cache = cache_of(args[0]);
    const int32_t layer = int32_of(args[1], "layer");
    Rows query(tensor_of(args[2], "query"));
    check_query(query.get(), cache.index, "batch", false);
    const int64_t rows = query.get().size(0);
    const at::Tensor *const given = maybe(args[8], "out");
    const Batch batch(args + 3, rows, cache.index);
    at::Tensor out = output(given, rows, cache.index, "batch");
    take_query(query);
    if (given != nullptr && within(query.get(), out)) query.make_dense();
    at::Tensor workspace;
    if (batch.workspace_bytes != 0) workspace = bytes(batch.workspace_bytes, cache.index);
    launch(cache.index, [&](void *stream) {
        return pkv_int4_decode_attention(cache.storage, cache.layers, cache.blocks, layer, query.data(), row_stride(query.get()),
                                         batch.lengths, batch.prefix, batch.flat, batch.rows, batch.total, batch.grid,
                                         out.data_ptr(), row_stride(out), workspace.defined() ? workspace.data_ptr() : nullptr,
                                         batch.workspace_bytes, batch.flag, stream);
    });
    return given != nullptr ? Py_NewRef(args[8]) : THPVariable_Wrap(std::move(out));
}

// (storage, layer, query, key, value, rope_table, lengths, prefix, flat, total_blocks, error_flag, out, query_norm, key_norm, eps)
PyObject *decode_layer(PyObject *const *args) {
    const Cache cache = cache_of(args[0]);
    const int index = cache.index;
    const int32_t layer = int32_of(args[1], "layer");
    Rows query(tensor_of(args[2], "query")), key(tensor_of(args[3], "key")), value(tensor_of(args[4], "value"));
    check_query(query.get(), index, "batch", false);
    const int64_t rows = query.get().size(0);
    for (const auto *fresh : {&key, &value}) {
        const at::Tensor &t = fresh->get();
        if (t.dim() != 3 || t.size(0) != rows || t.size(1) != kKvHeads || t.size(2) != kDim ||
            t.scalar_type() != at::kHalf || !here(t, index)) {
            refuse(std::string(fresh == &key ? "key" : "value") + " must be FP16 [" + std::to_string(rows) + ", 4, 64]" +
                   on_device(index));
        }
    }
    const void *const rope = rope_of(tensor_of(args[5], "rope_table"), index);
    const at::Tensor *const given = maybe(args[11], "out");
    const Batch batch(args + 6, rows, index);
    const Norms norms = norms_of(args + 12, cache);
    at::Tensor out = output(given, rows, index, "batch");
    take_query(query);
    take_pair(key, value);
    if (given != nullptr) {  // an output that lies over the inputs: rows are written while others are still read
        if (within(query.get(), out)) query.make_dense();
        if (within(key.get(), out) || within(value.get(), out)) {
            key.make_dense();
            value.make_dense();
        }
    }
    at::Tensor workspace;
    if (batch.workspace_bytes != 0) workspace = bytes(batch.workspace_bytes, index);
    launch(index, [&](void *stream) {
        return pkv_int4_decode_layer(cache.storage, cache.layers, cache.blocks, layer, query.data(), row_stride(query.get()),
                                     key.data(), value.data(), key.stride(0), rope, norms.query, norms.key, norms.eps,
                                     batch.lengths, batch.prefix, batch.flat, batch.rows, batch.total, batch.grid, 1,
                                     out.data_ptr(), row_stride(out), workspace.defined() ? workspace.data_ptr() : nullptr,
                                     batch.workspace_bytes, batch.flag, stream);
    });
    return given != nullptr ? Py_NewRef(args[11]) : THPVariable_Wrap(std::move(out));
}

// (storage, layer, query, blocks, start, error_flag, out)
PyObject *prefill_attention(PyObject *const *args) {
    const Cache cache = cache_of(args[0]);
    const int32_t layer = int32_of(args[1], "layer");
    Rows query(tensor_of(args[2], "query"));
    check_query(query.get(), cache.index, "tokens", true);
    const int64_t tokens = query.get().size(0);
    const int64_t start = PyLong_CheckExact(args[4]) ? int_of(args[4]) : -1;
    if (start < 0 || start > PKV_CONTEXT_LIMIT || start + tokens > PKV_CONTEXT_LIMIT) {
        refuse("the chunk must hold 1 or more tokens at positions below 2048");
    }
    const int64_t count = (start + tokens + kBlockTokens - 1) / kBlockTokens;
    const int32_t *const list = int_list(args[3], "blocks", count, cache.index);
    int32_t *const flag = int_list(args[5], "error_flag", 1, cache.index);
    const at::Tensor *const given = maybe(args[6], "out");
    at::Tensor out = output(given, tokens, cache.index, "tokens");
    take_query(query);
    if (given != nullptr && within(query.get(), out)) query.make_dense();
    int64_t workspace_bytes = 0;
    check_status(pkv_int4_prefill_plan(cache.index, static_cast<int32_t>(start), static_cast<int32_t>(tokens), &workspace_bytes));
    const at::Tensor workspace = bytes(workspace_bytes, cache.index);
    const at::Tensor &q = query.get();
    launch(cache.index, [&](void *stream) {
        return pkv_int4_prefill_attention(cache.storage, cache.layers, cache.blocks, layer, q.data_ptr(),
                                          q.scalar_type() == at::kFloat, row_stride(q), list, static_cast<int32_t>(start),
                                          static_cast<int32_t>(tokens), out.data_ptr(), row_stride(out),
                                          workspace.data_ptr(), workspace_bytes, flag, stream);
    });
    return given != nullptr ? Py_NewRef(args[6]) : THPVariable_Wrap(std::move(out));
}

// -- module ------------------------------------------------------------------------------
// torch.OutOfMemoryError, as torch's own allocations raise it.
void out_of_memory(const char *message) {
    PyObject *const torch = PyImport_ImportModule("torch");
    PyObject *const type = torch != nullptr ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (type != nullptr) PyErr_SetString(type, message);
    Py_XDECREF(type);
    Py_XDECREF(torch);
}

template <PyObject *(*Operator)(PyObject *const *), Py_ssize_t kArgs>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t count) {
    if (count != kArgs) {
        PyErr_Format(PyExc_TypeError, "takes %zd arguments, not %zd", kArgs, count);
        return nullptr;
    }
    try {
        return Operator(args);
    } catch (const PythonError &) {
    } catch (const Refusal &refusal) {
        PyErr_SetString(PyExc_ValueError, refusal.message.c_str());
    } catch (const c10::OutOfMemoryError &error) {
        out_of_memory(error.what_without_backtrace());
    } catch (const c10::Error &error) {
        PyErr_SetString(PyExc_RuntimeError, error.what_without_backtrace());
    } catch (const std::exception &error) {
        PyErr_SetString(PyExc_RuntimeError, error.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "4-bit operator: unknown C++ exception");
    }
    return nullptr;
}

#define OPERATOR(name, count) \
    {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<name, count>)), METH_FASTCALL, nullptr}

PyMethodDef methods[] = {
    OPERATOR(check_cache, 1),      OPERATOR(check_norms, 4),   OPERATOR(overlaps, 2),
    OPERATOR(append_kv, 13),       OPERATOR(read_blocks, 4),   OPERATOR(decode_attention, 9),
    OPERATOR(decode_layer, 15),    OPERATOR(prefill_attention, 7),
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_int4_ops", "Operators of the 4-bit KV cache.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__int4_ops() {
    PyObject *const created = PyModule_Create(&module);
    if (created == nullptr || PyModule_AddStringConstant(created, "built_for", PKV_BUILT_FOR) == 0) return created;
    Py_DECREF(created);
    return nullptr;
}
