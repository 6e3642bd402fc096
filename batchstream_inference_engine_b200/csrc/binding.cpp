// Python entry points of the bounded-cache and 4-bit operators and of draft verification
// (module _native).
//
// The calls last a few microseconds on the device, and a ctypes call with its checks
// in Python takes 15 to 20 on the host: here the checks, the output and scratch
// tensors and the C ABI call cost about 5.  ops.py documents the functions and gives
// the arguments their defaults; every function takes all of them by position and
// raises RuntimeError as the rest of the package does.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <initializer_list>
#include <map>
#include <optional>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

#include "../../include/batchstream_b200.h"

namespace {

using at::Tensor;
using std::string;

[[noreturn]] void refuse(const string& message) { throw std::runtime_error(message); }

void require(bool condition, const char* name, const char* message) {
  if (!condition) refuse(string(name) + ": " + message);
}

void check(int rc) {
  if (rc != 0) {
    const char* message = bs_last_error();
    refuse(*message != '\0' ? message : "batchstream_b200 call failed with code " + std::to_string(rc));
  }
}

// A Python error is already set.
struct PythonError {};

const Tensor& tensor_of(PyObject* o, const char* name, const char* arg) {
  if (!THPVariable_Check(o)) refuse(string(name) + ": " + arg + " must be a tensor");
  return THPVariable_Unpack(o);
}

std::optional<Tensor> optional_tensor(PyObject* o, const char* name, const char* arg) {
  if (o == Py_None) return std::nullopt;
  return tensor_of(o, name, arg);
}

int64_t int_of(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PythonError();
  return v;
}

double float_of(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PythonError();
  return v;
}

bool bool_of(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw PythonError();
  return v != 0;
}

// The CUDA device that every given tensor is on.
c10::Device cuda_device(const char* name, std::initializer_list<const Tensor*> tensors) {
  std::optional<c10::Device> device;
  for (const Tensor* t : tensors) {
    if (t == nullptr) continue;
    if (!t->is_cuda()) refuse(string(name) + ": every tensor must be a CUDA tensor");
    if (!device) {
      device = t->device();
    } else if (t->device() != *device) {
      refuse(string(name) + ": tensors are on different devices");
    }
  }
  return *device;
}

const Tensor* pointer(const std::optional<Tensor>& t) { return t ? &*t : nullptr; }

int32_t dtype_code(at::ScalarType t) {
  return t == at::kBFloat16 ? BS_BF16 : t == at::kFloat ? BS_F32 : -1;
}

// int32 entries one after the other, at least `count` of them.
Tensor int32_list(const char* name, const char* arg, const Tensor& t, int64_t count) {
  if (t.scalar_type() != at::kInt) refuse(string(name) + ": " + arg + " must be int32");
  if (t.dim() != 1 || t.numel() < count) {
    refuse(string(name) + ": " + arg + " must be one-dimensional with at least " +
           std::to_string(count) + " entries");
  }
  return t.contiguous();
}

// ------------------------------------------------------------------ status words

// The status word of each (device, stream) is a tensor that ops.py keeps and never
// moves; its address is asked for once.
struct StatusWord {
  int device;
  void* stream;
  uint32_t* word;
};
std::vector<StatusWord> g_status;
PyObject* g_status_source = nullptr;

uint32_t* status_word(int device, void* stream) {
  for (const StatusWord& s : g_status) {
    if (s.device == device && s.stream == stream) return s.word;
  }
  if (g_status_source == nullptr) refuse("no status source is set");
  PyObject* got = PyObject_CallFunction(g_status_source, "iK", device,
                                        reinterpret_cast<unsigned long long>(stream));
  if (got == nullptr) throw PythonError();
  const unsigned long long address = PyLong_AsUnsignedLongLong(got);
  Py_DECREF(got);
  if (PyErr_Occurred()) throw PythonError();
  uint32_t* word = reinterpret_cast<uint32_t*>(address);
  g_status.push_back({device, stream, word});
  return word;
}

// The device made current, its current stream and that stream's status word.
struct Launch {
  c10::cuda::OptionalCUDAGuard guard;
  void* stream;
  uint32_t* status;
  explicit Launch(c10::Device device) {
    if (c10::cuda::current_device() != device.index()) guard.set_device(device);
    stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    status = status_word(device.index(), stream);
  }
};

// (bytes, device index): zero bytes for good, whatever the current stream records.  A
// stream of its own fills them, waited for here; the allocator gives a captured stream's
// pool to that stream alone.
PyObject* zeros_apart(PyObject* const* a) {
  const int64_t bytes = int_of(a[0]);
  const auto device = static_cast<c10::DeviceIndex>(int_of(a[1]));
  const c10::cuda::CUDAGuard guard(device);
  const c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
  static std::map<c10::DeviceIndex, cudaStream_t> streams;
  cudaStream_t& stream = streams[device];
  if (stream == nullptr) {
    C10_CUDA_CHECK(cudaStreamCreateWithFlags(&stream, cudaStreamNonBlocking));
  }
  const c10::cuda::CUDAStreamGuard on(c10::cuda::getStreamFromExternal(stream, device));
  const Tensor t = at::empty({bytes}, at::TensorOptions(at::kByte).device(at::kCUDA, device));
  C10_CUDA_CHECK(cudaMemsetAsync(t.data_ptr(), 0, bytes, stream));
  C10_CUDA_CHECK(cudaStreamSynchronize(stream));
  return THPVariable_Wrap(t);
}

// Scratch of one call, from the stream-ordered allocator (inside a capture: from the
// graph's own pool, so two graphs never share it).
Tensor scratch(uint64_t bytes, c10::Device device) {
  if (bytes == 0) return Tensor();
  return at::empty({static_cast<int64_t>(bytes)}, at::TensorOptions(at::kByte).device(device));
}

void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// ------------------------------------------------------------------ window attention

// Bytes of a token and kv head in a 4-bit pool, and head_dim from them.
int64_t int4_row(int64_t head_dim) { return head_dim / 2 + head_dim / 16; }

int64_t int4_head_dim(const char* name, const Tensor& key_pool, const Tensor& value_pool) {
  require(key_pool.dim() == 4 && value_pool.sizes() == key_pool.sizes() &&
              key_pool.scalar_type() == at::kByte && value_pool.scalar_type() == at::kByte,
          name, "4-bit pools must be uint8 [Hkv, NB, bs, 9 * D / 16] of one shape");
  require(key_pool.size(3) > 0 && key_pool.size(3) % 18 == 0, name,
          "4-bit pools must be uint8 [Hkv, NB, bs, 9 * D / 16], D a multiple of 32");
  require(key_pool.is_contiguous() && value_pool.is_contiguous(), name, "pools must be contiguous");
  return key_pool.size(3) / 9 * 16;
}

// What the window attentions and those over 4-bit pools take: [T, H, D] queries over paged
// pools.
struct WindowInputs {
  Tensor query, tables, out;
  bool own_out = false;  // allocated here
  int64_t T, H, D, Hkv, NB, bs, mb;
  int32_t code;
};

// Elements between tokens of [T, H, D] (any stride of a single token will do).
int64_t token_stride(const Tensor& t) { return std::max(t.stride(0), t.size(1) * t.size(2)); }

WindowInputs window_inputs(const char* name, const Tensor& query, const Tensor& key_pool,
                           const Tensor& value_pool, const Tensor& block_tables,
                           const std::optional<Tensor>& out, PyObject* max_blocks, bool int4) {
  if (int4) {
    const int64_t head_dim = int4_head_dim(name, key_pool, value_pool);
    require(query.dim() == 3, name, "query must be [T, H, D]");
    require(query.size(2) == head_dim, name, "query and pools disagree on head_dim");
  } else {
    require(query.dim() == 3 && key_pool.dim() == 4 && value_pool.sizes() == key_pool.sizes(), name,
            "query must be [T, H, D] and the pools [Hkv, NB, bs, D]");
    require(query.scalar_type() == key_pool.scalar_type() &&
                value_pool.scalar_type() == key_pool.scalar_type(),
            name, "query and pools must share a dtype");
    require(key_pool.is_contiguous() && value_pool.is_contiguous(), name,
            "pools must be contiguous");
    require(query.size(2) == key_pool.size(3), name, "query and pools disagree on head_dim");
  }
  require(block_tables.scalar_type() == at::kInt && block_tables.dim() == 2, name,
          "block_tables must be int32 [rows, max_blocks]");
  WindowInputs w;
  w.T = query.size(0);
  w.H = query.size(1);
  w.D = query.size(2);
  w.Hkv = key_pool.size(0);
  w.NB = key_pool.size(1);
  w.bs = key_pool.size(2);
  w.code = dtype_code(query.scalar_type());
  auto heads_together = [&](const Tensor& t) {
    return t.is_contiguous() ||
           (t.stride(2) == 1 && t.stride(1) == w.D && t.stride(0) >= w.H * w.D);
  };
  w.query = heads_together(query) ? query : query.contiguous();
  const bool rows_apart = block_tables.is_contiguous() ||
                          (block_tables.stride(1) == 1 &&
                           block_tables.stride(0) >= block_tables.size(1));
  w.tables = rows_apart ? block_tables : block_tables.contiguous();
  w.mb = max_blocks == Py_None ? block_tables.size(1) : int_of(max_blocks);
  if (out) {
    if (out->sizes() != query.sizes() || out->scalar_type() != query.scalar_type() ||
        !heads_together(*out)) {
      refuse(string(name) + ": out must be [T, H, D] like the query, with contiguous heads, in its "
             "dtype");
    }
    w.out = *out;
  } else {
    w.out = at::empty_like(query, at::MemoryFormat::Contiguous);
    w.own_out = true;
  }
  return w;
}

int64_t table_stride(const Tensor& t) { return std::max(t.stride(0), t.size(1)); }

PyObject* result(const WindowInputs& w, PyObject* out) {
  if (w.own_out) return THPVariable_Wrap(w.out);
  Py_INCREF(out);
  return out;
}

// (query, key_pool, value_pool, block_tables, context_lens, scaling, window, sinks,
//  seq_rows, out, max_blocks_per_seq)
template <bool Int4>
PyObject* attention_batched(PyObject* const* a) {
  const char* name = Int4 ? "int4_attention_batched" : "window_attention_batched";
  const auto workspace_bytes = Int4 ? &bs_int4_attention_batched_workspace_bytes
                                    : &bs_window_attention_batched_workspace_bytes;
  const auto attend = Int4 ? &bs_int4_attention_batched : &bs_window_attention_batched;
  const Tensor& query = tensor_of(a[0], name, "query");
  const Tensor& key_pool = tensor_of(a[1], name, "key_pool");
  const Tensor& value_pool = tensor_of(a[2], name, "value_pool");
  const Tensor& block_tables = tensor_of(a[3], name, "block_tables");
  const Tensor& context_lens = tensor_of(a[4], name, "context_lens");
  const double scaling = float_of(a[5]);
  const int64_t window = int_of(a[6]), sinks = int_of(a[7]);
  const std::optional<Tensor> seq_rows = optional_tensor(a[8], name, "seq_rows");
  const std::optional<Tensor> out = optional_tensor(a[9], name, "out");
  const c10::Device device = cuda_device(name, {&query, &key_pool, &value_pool, &block_tables,
                                                &context_lens, pointer(seq_rows), pointer(out)});
  const WindowInputs w = window_inputs(name, query, key_pool, value_pool, block_tables, out, a[10],
                                       Int4);
  const Tensor lens = int32_list(name, "context_lens", context_lens, w.T);
  const Tensor rows = seq_rows ? int32_list(name, "seq_rows", *seq_rows, w.T) : Tensor();
  const Launch launch(device);
  uint64_t need = 0;
  check(workspace_bytes(w.T, w.H, w.Hkv, w.D, w.bs, w.mb, w.code, window, sinks, &need));
  const Tensor ws = scratch(need, device);
  check(attend(
      w.query.data_ptr(), token_stride(w.query), key_pool.data_ptr(), value_pool.data_ptr(),
      static_cast<const int32_t*>(w.tables.data_ptr()), table_stride(w.tables), w.tables.size(0),
      static_cast<const int32_t*>(address(rows)), static_cast<const int32_t*>(lens.data_ptr()), w.T,
      w.H, w.Hkv, w.D, w.bs, w.NB, w.mb, w.code, scaling, window, sinks, w.out.data_ptr(),
      token_stride(w.out), address(ws), need, launch.status, launch.stream));
  return result(w, a[9]);
}

// (query, key_pool, value_pool, block_tables, cu_q, context_lens, scaling,
//  max_query_len, window, sinks, seq_rows, out, max_blocks_per_seq)
template <bool Int4>
PyObject* prefill_attention(PyObject* const* a) {
  const char* name = Int4 ? "int4_prefill_attention" : "window_prefill_attention";
  const auto workspace_bytes = Int4 ? &bs_int4_prefill_attention_workspace_bytes
                                    : &bs_window_prefill_attention_workspace_bytes;
  const auto attend = Int4 ? &bs_int4_prefill_attention : &bs_window_prefill_attention;
  const Tensor& query = tensor_of(a[0], name, "query");
  const Tensor& key_pool = tensor_of(a[1], name, "key_pool");
  const Tensor& value_pool = tensor_of(a[2], name, "value_pool");
  const Tensor& block_tables = tensor_of(a[3], name, "block_tables");
  const Tensor& cu_q = tensor_of(a[4], name, "cu_q");
  const Tensor& context_lens = tensor_of(a[5], name, "context_lens");
  const double scaling = float_of(a[6]);
  const int64_t max_query_len = int_of(a[7]), window = int_of(a[8]), sinks = int_of(a[9]);
  const std::optional<Tensor> seq_rows = optional_tensor(a[10], name, "seq_rows");
  const std::optional<Tensor> out = optional_tensor(a[11], name, "out");
  const c10::Device device =
      cuda_device(name, {&query, &key_pool, &value_pool, &block_tables, &cu_q, &context_lens,
                         pointer(seq_rows), pointer(out)});
  const WindowInputs w = window_inputs(name, query, key_pool, value_pool, block_tables, out, a[12],
                                       Int4);
  const Tensor lens = int32_list(name, "context_lens", context_lens, 0);
  const int64_t R = lens.numel();
  const Tensor cu = int32_list(name, "cu_q", cu_q, R + 1);
  const Tensor rows = seq_rows ? int32_list(name, "seq_rows", *seq_rows, R) : Tensor();
  const Launch launch(device);
  uint64_t need = 0;
  check(workspace_bytes(w.T, R, max_query_len, w.H, w.Hkv, w.D, w.bs, w.mb, w.code, window, sinks,
                        &need));
  const Tensor ws = scratch(need, device);
  check(attend(
      w.query.data_ptr(), token_stride(w.query), static_cast<const int32_t*>(cu.data_ptr()), R, w.T,
      max_query_len, static_cast<const int32_t*>(lens.data_ptr()),
      static_cast<const int32_t*>(address(rows)), key_pool.data_ptr(), value_pool.data_ptr(),
      static_cast<const int32_t*>(w.tables.data_ptr()), table_stride(w.tables), w.tables.size(0),
      w.mb, w.H, w.Hkv, w.D, w.bs, w.NB, w.code, scaling, window, sinks, w.out.data_ptr(),
      token_stride(w.out), address(ws), need, launch.status, launch.stream));
  return result(w, a[11]);
}

// ------------------------------------------------------------------ rotary, copies

PyObject* pair(const Tensor& x, const Tensor& y) {
  PyObject* first = THPVariable_Wrap(x);
  PyObject* second = first != nullptr ? THPVariable_Wrap(y) : nullptr;
  PyObject* both = second != nullptr ? PyTuple_Pack(2, first, second) : nullptr;
  Py_XDECREF(first);
  Py_XDECREF(second);
  if (both == nullptr) throw PythonError();
  return both;
}

// Whether two tensors' memory overlaps (both with non-negative strides).
bool overlap(const Tensor& a, const Tensor& b) {
  auto span = [](const Tensor& t) {
    const char* begin = static_cast<const char*>(t.data_ptr());
    int64_t last = 0;
    for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
    return std::make_pair(begin, begin + (last + 1) * t.element_size());
  };
  if (a.numel() == 0 || b.numel() == 0) return false;
  const auto x = span(a), y = span(b);
  return x.first < y.second && y.first < x.second;
}

// (qkv, frequencies, positions, slot_mapping, key_pool, value_pool, num_heads,
//  interleaved, amplitude, query_out)
template <bool Int4>
PyObject* append(PyObject* const* a) {
  const char* name = Int4 ? "rotary_append_int4" : "rotary_append";
  const Tensor& qkv = tensor_of(a[0], name, "qkv");
  const Tensor& frequencies = tensor_of(a[1], name, "frequencies");
  const Tensor& positions = tensor_of(a[2], name, "positions");
  const Tensor& slot_mapping = tensor_of(a[3], name, "slot_mapping");
  const Tensor& key_pool = tensor_of(a[4], name, "key_pool");
  const Tensor& value_pool = tensor_of(a[5], name, "value_pool");
  const int64_t H = int_of(a[6]);
  const bool interleaved = bool_of(a[7]);
  const double amplitude = float_of(a[8]);
  const std::optional<Tensor> query_out = optional_tensor(a[9], name, "query_out");
  const c10::Device device = cuda_device(name, {&qkv, &frequencies, &positions, &slot_mapping,
                                                &key_pool, &value_pool, pointer(query_out)});
  int64_t D;
  if (Int4) {
    D = int4_head_dim(name, key_pool, value_pool);
  } else {
    require(key_pool.dim() == 4 && value_pool.sizes() == key_pool.sizes() &&
                value_pool.scalar_type() == key_pool.scalar_type(),
            name, "the pools must be [Hkv, NB, bs, D] of one shape and dtype");
    require(key_pool.is_contiguous() && value_pool.is_contiguous(), name,
            "pools must be contiguous");
    D = key_pool.size(3);
  }
  const int64_t Hkv = key_pool.size(0), T = positions.numel();
  const Tensor pos = int32_list(name, "positions", positions, T);
  const Tensor slots = int32_list(name, "slot_mapping", slot_mapping, T);
  require(frequencies.scalar_type() == at::kDouble && frequencies.dim() == 1, name,
          "frequencies must be one-dimensional float64");
  const Tensor freq = frequencies.contiguous();
  require(qkv.dim() >= 2 && qkv.size(0) >= T, name, "qkv needs a row per position");
  const int64_t width = (H + 2 * Hkv) * D;
  Tensor rows = qkv.dim() == 2 ? qkv : qkv.flatten(1);
  if (rows.size(1) != width) {
    refuse(string(name) + ": qkv rows must hold " + std::to_string(width) + " elements");
  }
  if (rows.stride(1) != 1 || (rows.size(0) > 1 && rows.stride(0) < width)) rows = rows.contiguous();
  Tensor q_out;
  if (query_out) {
    require(query_out->is_contiguous() && query_out->scalar_type() == qkv.scalar_type() &&
                query_out->numel() >= T * H * D,
            name, "query_out must be contiguous [T, heads, head_dim] in the qkv dtype");
    require(!overlap(*query_out, qkv), name, "query_out must not overlap qkv");
    q_out = *query_out;
  } else {
    require(Int4 ? H >= 0 : H > 0, name,
            Int4 ? "num_heads must not be negative" : "num_heads must be positive");
    q_out = at::empty({T, H, D}, qkv.options());
  }
  const Launch launch(device);
  if (Int4) {
    for (const Tensor* pool : {&key_pool, &value_pool}) {
      require(!overlap(*pool, rows) && !overlap(*pool, q_out), name,
              "the pools must not overlap qkv or query_out");
    }
    check(bs_rotary_append_int4(
        rows.data_ptr(), std::max(rows.stride(0), width), dtype_code(qkv.scalar_type()),
        static_cast<const double*>(freq.data_ptr()), 2 * freq.numel(), interleaved ? 1 : 0,
        amplitude, static_cast<const int32_t*>(pos.data_ptr()),
        static_cast<const int32_t*>(slots.data_ptr()), T, H, Hkv, D, q_out.data_ptr(),
        key_pool.data_ptr(), value_pool.data_ptr(), key_pool.size(1), key_pool.size(2),
        launch.status, launch.stream));
    if (!query_out) return THPVariable_Wrap(q_out);
    Py_INCREF(a[9]);
    return a[9];
  }
  check(bs_rotary_append(rows.data_ptr(), std::max(rows.stride(0), width),
                         dtype_code(qkv.scalar_type()),
                         static_cast<const double*>(freq.data_ptr()), 2 * freq.numel(),
                         interleaved ? 1 : 0, amplitude,
                         static_cast<const int32_t*>(pos.data_ptr()),
                         static_cast<const int32_t*>(slots.data_ptr()), T, H, Hkv, D,
                         q_out.data_ptr(), key_pool.data_ptr(), value_pool.data_ptr(),
                         dtype_code(key_pool.scalar_type()), key_pool.size(1), key_pool.size(2),
                         launch.status, launch.stream));
  if (!query_out) return THPVariable_Wrap(q_out);
  Py_INCREF(a[9]);
  return a[9];
}

// (key_pool, value_pool, slot_mapping)
PyObject* read_int4(PyObject* const* a) {
  const char* name = "read_int4";
  const Tensor& key_pool = tensor_of(a[0], name, "key_pool");
  const Tensor& value_pool = tensor_of(a[1], name, "value_pool");
  const Tensor& slot_mapping = tensor_of(a[2], name, "slot_mapping");
  const c10::Device device = cuda_device(name, {&key_pool, &value_pool, &slot_mapping});
  const int64_t D = int4_head_dim(name, key_pool, value_pool), Hkv = key_pool.size(0);
  const int64_t T = slot_mapping.numel();
  const Tensor slots = int32_list(name, "slot_mapping", slot_mapping, T);
  const Launch launch(device);
  const auto options = at::TensorOptions(at::kBFloat16).device(device);
  const Tensor k = at::empty({T, Hkv, D}, options), v = at::empty({T, Hkv, D}, options);
  check(bs_read_int4(key_pool.data_ptr(), value_pool.data_ptr(),
                     static_cast<const int32_t*>(slots.data_ptr()), T, Hkv, key_pool.size(1),
                     key_pool.size(2), D, k.data_ptr(), v.data_ptr(), launch.status,
                     launch.stream));
  return pair(k, v);
}

// (key_pool, value_pool, src, dst).  4-bit pools are copied as pairs of bytes.
PyObject* copy_blocks(PyObject* const* a) {
  const char* name = "copy_blocks";
  const Tensor& key_pool = tensor_of(a[0], name, "key_pool");
  const Tensor& value_pool = tensor_of(a[1], name, "value_pool");
  const Tensor& src = tensor_of(a[2], name, "src");
  const Tensor& dst = tensor_of(a[3], name, "dst");
  const c10::Device device = cuda_device(name, {&key_pool, &value_pool, &src, &dst});
  const int64_t dims = key_pool.dim();
  require((dims == 4 || dims == 5) && value_pool.sizes() == key_pool.sizes() &&
              value_pool.scalar_type() == key_pool.scalar_type(),
          name, "the pools must be [L, Hkv, NB, bs, D] of one shape and dtype");
  require(key_pool.is_contiguous() && value_pool.is_contiguous(), name, "pools must be contiguous");
  require(src.numel() == dst.numel(), name, "src and dst must have one entry per pair");
  const int64_t n = src.numel();
  const Tensor from = int32_list(name, "src", src, n), to = int32_list(name, "dst", dst, n);
  const bool int4 = key_pool.scalar_type() == at::kByte;
  require(!int4 || key_pool.size(dims - 1) % 18 == 0, name,
          "4-bit pools must be uint8 [L, Hkv, NB, bs, 9 * D / 16], D a multiple of 32");
  const Launch launch(device);
  check(bs_copy_blocks(key_pool.data_ptr(), value_pool.data_ptr(),
                       int4 ? BS_BF16 : dtype_code(key_pool.scalar_type()),
                       dims == 5 ? key_pool.size(0) : 1,
                       key_pool.size(dims - 4), key_pool.size(dims - 3), key_pool.size(dims - 2),
                       key_pool.size(dims - 1) / (int4 ? 2 : 1), static_cast<const int32_t*>(from.data_ptr()),
                       static_cast<const int32_t*>(to.data_ptr()), n, launch.status,
                       launch.stream));
  Py_RETURN_NONE;
}

// ------------------------------------------------------------------ drafts

// (logits, draft_tokens, cu_rows, uniforms, temperature, draft_probs)
PyObject* verify_drafts(PyObject* const* a) {
  const char* name = "verify_drafts";
  const Tensor& logits = tensor_of(a[0], name, "logits");
  const Tensor& draft_tokens = tensor_of(a[1], name, "draft_tokens");
  const Tensor& cu_rows = tensor_of(a[2], name, "cu_rows");
  const Tensor& uniforms = tensor_of(a[3], name, "uniforms");
  std::optional<Tensor> temperatures;
  double temperature = 0.0;
  if (THPVariable_Check(a[4])) {
    temperatures = tensor_of(a[4], name, "temperature");
  } else {
    temperature = float_of(a[4]);
  }
  const std::optional<Tensor> draft_probs = optional_tensor(a[5], name, "draft_probs");
  const c10::Device device = cuda_device(name, {&logits, &draft_tokens, &cu_rows, &uniforms,
                                                pointer(temperatures), pointer(draft_probs)});
  require(logits.dim() == 2, name, "logits must be [rows, vocab]");
  const int64_t N = logits.size(0), V = logits.size(1);
  auto rows_of = [&](const Tensor& t) {
    return t.stride(1) == 1 && (N <= 1 || t.stride(0) >= V) ? t : t.contiguous();
  };
  auto floats = [&](const char* arg, const Tensor& t, int64_t count) {
    if (t.scalar_type() != at::kFloat || t.dim() != 1 || t.numel() < count) {
      refuse(string(name) + ": " + arg + " must be one-dimensional float32 with at least " +
             std::to_string(count) + " entries");
    }
    return t.contiguous();
  };
  const Tensor l = rows_of(logits);
  const Tensor tokens = int32_list(name, "draft_tokens", draft_tokens, N);
  const Tensor cu = int32_list(name, "cu_rows", cu_rows, 1);
  const int64_t B = cu.numel() - 1;
  const Tensor u = floats("uniforms", uniforms, N);
  const Tensor temps = temperatures ? floats("temperature", *temperatures, B) : Tensor();
  Tensor probs;
  if (draft_probs) {
    require(draft_probs->dim() == 2 && draft_probs->sizes() == logits.sizes(), name,
            "draft_probs must be [rows, vocab] like the logits");
    probs = rows_of(*draft_probs);
  }
  const Launch launch(device);
  uint64_t need = 0;
  check(bs_verify_drafts_workspace_bytes(N, V, dtype_code(logits.scalar_type()), &need));
  const Tensor ws = scratch(need, device);
  const auto options = at::TensorOptions(at::kInt).device(device);
  const Tensor out = at::empty({N}, options), accepted = at::empty({B}, options);
  check(bs_verify_drafts(
      l.data_ptr(), std::max(l.stride(0), V), dtype_code(logits.scalar_type()), N, V,
      static_cast<const int32_t*>(tokens.data_ptr()), static_cast<const int32_t*>(cu.data_ptr()), B,
      static_cast<const float*>(u.data_ptr()), static_cast<const float*>(address(temps)),
      temperature, address(probs), probs.defined() ? std::max(probs.stride(0), V) : 0,
      probs.defined() ? dtype_code(probs.scalar_type()) : 0, static_cast<int32_t*>(out.data_ptr()),
      static_cast<int32_t*>(accepted.data_ptr()), address(ws), need, launch.status,
      launch.stream));
  return pair(out, accepted);
}

// (callable(device index, stream handle) -> address of the status word)
PyObject* set_status_source(PyObject* const* a) {
  Py_INCREF(a[0]);
  Py_XDECREF(g_status_source);
  g_status_source = a[0];
  g_status.clear();
  Py_RETURN_NONE;
}

// ------------------------------------------------------------------ module

template <PyObject* (*Fn)(PyObject* const*), Py_ssize_t Count>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t count) {
  if (count != Count) {
    PyErr_Format(PyExc_TypeError, "%zd arguments given, %zd expected", count, Count);
    return nullptr;
  }
  try {
    return Fn(args);
  } catch (const PythonError&) {
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

template <PyObject* (*Fn)(PyObject* const*), Py_ssize_t Count>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<Fn, Count>)),
          METH_FASTCALL, nullptr};
}

PyMethodDef g_methods[] = {
    method<attention_batched<false>, 11>("window_attention_batched"),
    method<prefill_attention<false>, 13>("window_prefill_attention"),
    method<append<false>, 10>("rotary_append"),
    method<attention_batched<true>, 11>("int4_attention_batched"),
    method<prefill_attention<true>, 13>("int4_prefill_attention"),
    method<append<true>, 10>("rotary_append_int4"),
    method<read_int4, 3>("read_int4"),
    method<verify_drafts, 6>("verify_drafts"),
    method<copy_blocks, 4>("copy_blocks"),
    method<set_status_source, 1>("set_status_source"),
    method<zeros_apart, 2>("zeros_apart"),
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native() { return PyModule_Create(&g_module); }
