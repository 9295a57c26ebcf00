// SPDX-License-Identifier: MIT
//
// dg_torch.cpp -- the attention operators' calls from Python
// (decode_opt_b200._host, used by decode_opt_b200/attention.py): checks the
// tensors, allocates the outputs, fills the C ABI's argument structs and calls
// it on the tensors' current stream.
//
// Host code only.  The calls of a decode step take the GPU a few microseconds;
// the same checks in Python cost the host 10 to 15.  Arguments come by
// position, None for those that are absent; attention.py documents them.  The
// C ABI's entry points are handed over by bind(), so that there is one copy
// of the library in the process.

#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/TracerMode.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime_api.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <atomic>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <map>
#include <stdexcept>
#include <string>
#include <tuple>
#include <utility>

#include "decode_attention_b200.h"

namespace {

using at::Tensor;

constexpr int64_t kInt32Max = 2147483647;
constexpr int64_t kMostStride = 0x1fffffff;      // elements: below 2^31 bytes for any type
constexpr int64_t kTicketBytes = 1024;           // of the attention workspace: zeroed once

int (*call_tables)(const dg_block_tables*, void*, int) = nullptr;
int (*call_rotary)(const dg_rotary_args*, void*, int) = nullptr;
int (*call_attention)(const dg_attention_args*, void*, int) = nullptr;
unsigned long long (*call_workspace_bytes)() = nullptr;

// An argument that cannot be served: ValueError in Python.
struct Refused {
  std::string what;
};

#if defined(__GNUC__)
__attribute__((format(printf, 2, 3)))
#endif
void need(bool ok, const char* form, ...) {
  if (ok) return;
  char text[512];
  va_list list;
  va_start(list, form);
  std::vsnprintf(text, sizeof(text), form, list);
  va_end(list);
  throw Refused{text};
}

bool given(PyObject* o) { return o != Py_None; }

const Tensor& tensor(PyObject* o, const char* name) {
  need(THPVariable_Check(o), "%s must be a tensor", name);
  return THPVariable_Unpack(o);
}

int64_t whole(PyObject* o, const char* name) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Refused{std::string(name) + " must be an integer"};
  }
  return v;
}

double real(PyObject* o, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Refused{std::string(name) + " must be a number"};
  }
  return v;
}

bool truth(PyObject* o) { return PyObject_IsTrue(o) == 1; }

template <typename P>
P* data(const Tensor& t) {
  return static_cast<P*>(t.data_ptr());
}

// An argument that may be a tensor: not None, nor a truth value (asked first,
// as asking those whether they are tensors takes Python 0.1 us each).
bool some_tensor(PyObject* o) { return o != Py_None && !PyBool_Check(o) && THPVariable_Check(o); }

// An argument, read or written, that wants a derivative, backward or forward,
// where the call has none.
void no_gradient(PyObject* o, const char* call) {
  if (!some_tensor(o)) return;
  const Tensor& t = THPVariable_Unpack(o);
  need(!(t.requires_grad() && c10::GradMode::is_enabled()),
       "%s has no gradient for one of its tensors that wants one: call it under torch.no_grad()", call);
  need(!t._fw_grad(0).defined(), "%s has no forward-mode derivative for one of its tensors: call it on primal ones",
       call);
}

// torch.jit.trace records no calls of this module: their results would be
// constants of the trace.
void no_trace(const char* call) {
  if (at::tracer::impl::is_dispatch_enabled())
    throw std::runtime_error(std::string("torch.jit.trace cannot record ") + call +
                             ": its results would be constants of the trace");
}

// A tensor that a launch has written into: what autograd saved of it is out of
// date.  (Inference tensors have no versions.)
void written(PyObject* o) {
  if (!some_tensor(o)) return;
  const Tensor& t = THPVariable_Unpack(o);
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// An output with a place for each of its values, and none of them in another
// place of `in` (it may be `in` itself).
void apart(const Tensor& out, const Tensor* in, const char* name) {
  need(at::has_internal_overlap(out) != at::MemOverlap::Yes, "%s has several values in one place", name);
  need(in == nullptr || at::get_overlap_status(out, *in) != at::MemOverlapStatus::Partial,
       "%s partly overlaps its input", name);
}

// A contiguous vector of `count` values.
void vector_of(const Tensor& t, const char* name, int64_t count, c10::Device device, at::ScalarType type) {
  need(t.scalar_type() == type && t.dim() == 1 && t.size(0) == count && t.is_contiguous() && t.device() == device,
       "%s must be a contiguous %s tensor of %lld values on %s", name, c10::toString(type),
       static_cast<long long>(count), device.str().c_str());
}

int* status_of(PyObject* o, c10::Device device) {
  if (!given(o)) return nullptr;
  const Tensor& t = tensor(o, "status");
  need(t.scalar_type() == at::kInt && t.numel() >= 1 && t.device() == device, "status must be an int32 tensor on %s",
       device.str().c_str());
  return data<int>(t);
}

// (entries a row, row stride) of a block table.
std::pair<int, int64_t> table_of(const Tensor& t, int64_t batch, c10::Device device) {
  need(t.scalar_type() == at::kInt && t.dim() == 2 && t.device() == device && t.size(0) == batch && t.size(1) >= 1 &&
           t.size(1) <= kInt32Max && (t.stride(1) == 1 || t.size(1) == 1) &&
           (batch == 1 || t.stride(0) >= t.size(1)),
       "block_table must be int32 [%lld, width >= 1] on %s with unit column stride and rows that do not overlap",
       static_cast<long long>(batch), device.str().c_str());
  return {static_cast<int>(t.size(1)), batch > 1 ? t.stride(0) : t.size(1)};
}

// Whether part of the vector lies in one of the rows.
bool in_rows(const int* vector, int64_t count, const int* rows, int64_t batch, int64_t width, int64_t stride) {
  const auto from = reinterpret_cast<uintptr_t>(vector), to = from + 4 * static_cast<uintptr_t>(count);
  const auto first = reinterpret_cast<uintptr_t>(rows), row = 4 * static_cast<uintptr_t>(width);
  const auto step = 4 * static_cast<uintptr_t>(stride);
  const uintptr_t b = from < first + row ? 0 : (from - first - row) / step + 1;    // the first that ends past `from`
  return count > 0 && b < static_cast<uintptr_t>(batch) && first + b * step < to;
}

int type_of(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return DG_TYPE_BF16;
    case at::kHalf: return DG_TYPE_FP16;
    case at::kFloat: return DG_TYPE_FP32;
    case at::kFloat8_e4m3fn:
    case at::kByte: return DG_TYPE_E4M3;
    default: return -1;
  }
}

// [tokens, heads, dim] like `like`; fills (token, head) strides.
int heads_of(const Tensor& t, const char* name, const Tensor& like, long long (&stride)[2]) {
  need(t.dim() == 3 && t.scalar_type() == like.scalar_type() && t.device() == like.device() &&
           t.size(0) == like.size(0) && t.size(2) == like.size(2) && t.size(1) >= 1 && t.size(1) <= kInt32Max &&
           t.stride(2) == 1 && t.stride(0) <= kMostStride && t.stride(1) <= kMostStride,
       "%s must be %s [%lld, heads >= 1, %lld] on %s with unit last stride and strides below 2^29", name,
       c10::toString(like.scalar_type()), static_cast<long long>(like.size(0)), static_cast<long long>(like.size(2)),
       like.device().str().c_str());
  stride[0] = t.stride(0);
  stride[1] = t.stride(1);
  return static_cast<int>(t.size(1));
}

struct Cache {
  int type, page_size, num_pages;
};

Cache cache_of(const Tensor& k, const Tensor& v, int64_t heads, const Tensor& like, long long (&ks)[3],
               long long (&vs)[3]) {
  const int type = type_of(k.scalar_type());
  need((type == DG_TYPE_E4M3 || k.scalar_type() == like.scalar_type()) && v.scalar_type() == k.scalar_type(),
       "both caches must be %s or e4m3 (float8_e4m3fn or uint8)", c10::toString(like.scalar_type()));
  need(k.dim() == 4 && v.sizes() == k.sizes() && k.device() == like.device() && v.device() == like.device() &&
           k.size(2) == heads && k.size(3) == like.size(2) && k.stride(3) == 1 && v.stride(3) == 1 &&
           k.size(0) >= 1 && k.size(0) <= kInt32Max && k.size(1) >= 1 && k.size(1) <= kInt32Max,
       "the caches must be [pages >= 1, page_size >= 1, %lld, %lld] on %s with unit last stride",
       static_cast<long long>(heads), static_cast<long long>(like.size(2)), like.device().str().c_str());
  for (int i = 0; i < 3; ++i) {
    ks[i] = k.stride(i);
    vs[i] = v.stride(i);
  }
  return {type, static_cast<int>(k.size(1)), static_cast<int>(k.size(0))};
}

const float* scale_of(PyObject* o, const char* name, int64_t heads, int cache_type, c10::Device device) {
  if (!given(o)) return nullptr;
  const Tensor& t = tensor(o, name);
  need(cache_type == DG_TYPE_E4M3, "%s goes with an e4m3 cache", name);
  vector_of(t, name, heads, device, at::kFloat);
  return data<float>(t);
}

void check(int rc, const char* call) {
  if (rc != 0) throw std::runtime_error(std::string(call) + " failed: cudaError " + std::to_string(rc));
}

void* stream_of(c10::Device device) { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }

template <typename F>
PyObject* guarded(F body) {
  HANDLE_TH_ERRORS
  try {
    return body();
  } catch (const Refused& r) {
    PyErr_SetString(PyExc_ValueError, r.what.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

#define COUNT(n)                                                                   \
  if (count != (n)) {                                                              \
    PyErr_Format(PyExc_TypeError, "%d arguments, %zd given", (n), count);          \
    return nullptr;                                                                \
  }

// context_lens, new_lens, free_pages, block_table, page_size, num_tokens,
// cursor, out (tuple of the six results, or None), status, pdl_attr
//   -> (seq_lens, query_start, slots, positions, requests, cursor), or None with out
PyObject* build_block_tables(PyObject*, PyObject* const* arg, Py_ssize_t count) {
  COUNT(10)
  return guarded([&]() -> PyObject* {
    no_trace("build_block_tables");
    const Tensor& context = tensor(arg[0], "context_lens");
    const Tensor& fresh = tensor(arg[1], "new_lens");
    const Tensor& free_pages = tensor(arg[2], "free_pages");
    const Tensor& table = tensor(arg[3], "block_table");
    need(context.is_cuda() && context.dim() == 1, "context_lens must be a CUDA vector");
    const c10::Device device = context.device();
    const int64_t batch = context.size(0);
    need(batch >= 1 && batch <= 16384, "batch must be 1 .. 16384");
    vector_of(context, "context_lens", batch, device, at::kInt);
    vector_of(fresh, "new_lens", batch, device, at::kInt);
    need(free_pages.dim() == 1 && free_pages.size(0) <= kInt32Max, "free_pages must be a vector");
    vector_of(free_pages, "free_pages", free_pages.size(0), device, at::kInt);
    const auto [width, table_stride] = table_of(table, batch, device);
    const int64_t page = whole(arg[4], "page_size"), tokens = whole(arg[5], "num_tokens");
    need(page >= 1 && page <= kInt32Max && tokens >= 0 && tokens <= kInt32Max, "page_size >= 1 and num_tokens >= 0");
    dg_block_tables a{};
    a.batch = static_cast<int>(batch);
    a.page_size = static_cast<int>(page);
    a.table_width = width;
    a.num_tokens = static_cast<int>(tokens);
    a.free_count = static_cast<int>(free_pages.size(0));
    a.table_stride = table_stride;
    a.context_lens = data<int>(context);
    a.new_lens = data<int>(fresh);
    a.free_pages = data<int>(free_pages);
    if (given(arg[6])) {
      const Tensor& t = tensor(arg[6], "cursor");
      vector_of(t, "cursor", 1, device, at::kInt);
      a.cursor_in = data<int>(t);
    }
    a.block_table = data<int>(table);
    need(!in_rows(a.free_pages, a.free_count, a.block_table, batch, width, table_stride),
         "free_pages must not be part of block_table");
    a.status = status_of(arg[8], device);
    const c10::cuda::CUDAGuard guard(device);
    Tensor made[6];
    const Tensor* out[6];
    static const char* const names[6] = {"out.seq_lens", "out.query_start", "out.slots",
                                         "out.positions", "out.requests",   "out.cursor"};
    const int64_t sizes[6] = {batch, batch + 1, tokens, tokens, tokens, 1};
    if (given(arg[7])) {
      need(PyTuple_Check(arg[7]) && PyTuple_GET_SIZE(arg[7]) == 6, "out must be six tensors");
      for (int i = 0; i < 6; ++i) {
        out[i] = &tensor(PyTuple_GET_ITEM(arg[7], i), names[i]);
        vector_of(*out[i], names[i], sizes[i], device, i == 2 ? at::kLong : at::kInt);
      }
      need(a.cursor_in == nullptr || data<int>(*out[5]) != a.cursor_in, "out.cursor must not be cursor");
      need(data<int>(*out[0]) != a.context_lens && data<int>(*out[0]) != a.new_lens,
           "out.seq_lens must not be context_lens or new_lens");
    } else {
      // One allocation, each part begun on 16 bytes: six would take the host
      // longer than the kernel takes the GPU.
      int64_t offset[6], total = 0;                // in 4-byte units
      for (int i = 0; i < 6; ++i) {
        offset[i] = total;
        total += ((i == 2 ? 2 : 1) * sizes[i] + 3) / 4 * 4;
      }
      const Tensor whole_part = at::empty({total}, at::TensorOptions().device(device).dtype(at::kInt));
      for (int i = 0; i < 6; ++i) {
        made[i] = at::detail::make_tensor<c10::TensorImpl>(
            c10::Storage(whole_part.storage()), whole_part.key_set(),
            c10::scalarTypeToTypeMeta(i == 2 ? at::kLong : at::kInt));
        made[i].unsafeGetTensorImpl()->set_storage_offset(i == 2 ? offset[i] / 2 : offset[i]);
        made[i].unsafeGetTensorImpl()->set_sizes_contiguous({sizes[i]});
        out[i] = &made[i];
      }
    }
    a.seq_lens = data<int>(*out[0]);
    a.query_start = data<int>(*out[1]);
    a.slots = data<long long>(*out[2]);
    a.positions = data<int>(*out[3]);
    a.requests = data<int>(*out[4]);
    a.cursor_out = data<int>(*out[5]);
    check(call_tables(&a, stream_of(device), truth(arg[9])), "dg_build_block_tables");
    written(arg[3]);
    if (given(arg[7])) {
      for (int i = 0; i < 6; ++i) written(PyTuple_GET_ITEM(arg[7], i));
      Py_RETURN_NONE;
    }
    PyObject* result = PyTuple_New(6);
    for (int i = 0; i < 6; ++i) PyTuple_SET_ITEM(result, i, THPVariable_Wrap(made[i]));
    return result;
  });
}

// q, k, v, positions, slots, k_cache, v_cache, table, axes, words (bytes),
// pairing, inverse, k_scale, v_scale, out_q, out_k, status, pdl_attr
//   -> (q_out, k_out).  q, k: None without; out_q, out_k: a tensor, True to
// make one, None for none.  k_cache None: no cache write.
PyObject* rotary(PyObject*, PyObject* const* arg, Py_ssize_t count) {
  COUNT(18)
  return guarded([&]() -> PyObject* {
    const Tensor* q = given(arg[0]) ? &tensor(arg[0], "q") : nullptr;
    const Tensor* k = given(arg[1]) ? &tensor(arg[1], "k") : nullptr;
    need(q != nullptr || k != nullptr, "q or k must be given");
    const Tensor& x = q != nullptr ? *q : *k;
    const int kind = type_of(x.scalar_type());
    need(x.is_cuda() && x.dim() == 3 && (kind == DG_TYPE_BF16 || kind == DG_TYPE_FP16 || kind == DG_TYPE_FP32),
         "q and k must be bf16, fp16 or fp32 CUDA tensors [tokens, heads, dim]");
    const c10::Device device = x.device();
    const int64_t tokens = x.size(0), dim = x.size(2);
    need(tokens >= 1 && tokens <= kInt32Max && dim >= 2 && dim <= 2048,
         "q and k need at least one token and a dim of 2 .. 2048");
    dg_rotary_args a{};
    a.tokens = static_cast<int>(tokens);
    a.head_dim = static_cast<int>(dim);
    a.type = a.cache_type = kind;
    if (q != nullptr) {
      a.heads = heads_of(*q, "q", x, a.q_stride);
      a.q = q->data_ptr();
    }
    if (k != nullptr) {
      a.kv_heads = heads_of(*k, "k", x, a.k_stride);
      a.k = k->data_ptr();
    }
    const Tensor& table = tensor(arg[7], "table");
    need(table.scalar_type() == at::kFloat && table.dim() == 2 && table.is_contiguous() && table.device() == device,
         "table must be a contiguous fp32 [max_position, rot] tensor on %s", device.str().c_str());
    need(table.size(0) >= 1 && table.size(0) <= kInt32Max && table.size(1) >= 2 && table.size(1) % 2 == 0 &&
             table.size(1) <= dim && table.size(1) <= DG_MAX_ROT,
         "the table's width must be even and at most %lld", static_cast<long long>(dim < DG_MAX_ROT ? dim : DG_MAX_ROT));
    a.max_position = static_cast<int>(table.size(0));
    a.rot = static_cast<int>(table.size(1));
    a.cos_sin = data<float>(table);
    const char* const call =
        given(arg[5]) ? "rotary_append" : "rotary, but for q and k without out_q and out_k,";
    for (int i : {0, 1, 7, 14, 15}) no_gradient(arg[i], call);
    const int64_t axes = whole(arg[8], "axes");
    need(PyBytes_Check(arg[9]) && PyBytes_GET_SIZE(arg[9]) == static_cast<Py_ssize_t>(sizeof(a.axis_of)),
         "words must be the packed axes");
    std::memcpy(a.axis_of, PyBytes_AS_STRING(arg[9]), sizeof(a.axis_of));
    a.pairing = static_cast<int>(whole(arg[10], "pairing"));
    a.inverse = truth(arg[11]);
    const Tensor& positions = tensor(arg[3], "positions");
    const bool wide = positions.scalar_type() == at::kLong;
    need((wide || positions.scalar_type() == at::kInt) && positions.device() == device &&
             (positions.dim() == 1 || positions.dim() == 2) && positions.size(-1) == tokens &&
             (positions.stride(-1) == 1 || tokens == 1),
         "positions must be int32 or int64 [%lld] or [axes, %lld] on %s", static_cast<long long>(tokens),
         static_cast<long long>(tokens), device.str().c_str());
    if (positions.dim() == 2) {
      need(positions.size(0) == axes, "positions has %lld axes, the sections %lld",
           static_cast<long long>(positions.size(0)), static_cast<long long>(axes));
      a.position_stride = axes > 1 ? positions.stride(0) : 0;
    }
    a.positions = positions.data_ptr();
    a.position_64 = wide;
    a.status = status_of(arg[16], device);
    if (given(arg[5])) {
      no_trace("rotary_append");
      need(q != nullptr && k != nullptr, "the cache write takes q, k and v");
      const Tensor& v = tensor(arg[2], "v");
      for (int i : {2, 5, 6, 12, 13}) no_gradient(arg[i], "rotary_append");
      need(kind != DG_TYPE_FP32, "the cache write takes bf16 or fp16");
      need(heads_of(v, "v", x, a.v_stride) == a.kv_heads,
           "k and v must have one shape");
      const Tensor& kc = tensor(arg[5], "k_cache");
      const Tensor& vc = tensor(arg[6], "v_cache");
      const Cache c = cache_of(kc, vc, a.kv_heads, x, a.k_cache_stride,
                               a.v_cache_stride);
      apart(kc, nullptr, "k_cache");
      apart(vc, nullptr, "v_cache");
      const auto overlap = at::get_overlap_status(kc, vc);
      need(overlap != at::MemOverlapStatus::Full && overlap != at::MemOverlapStatus::Partial,
           "k_cache and v_cache must not overlap");
      const Tensor& slots = tensor(arg[4], "slots");
      vector_of(slots, "slots", tokens, device, at::kLong);
      a.v = v.data_ptr();
      a.cache_type = c.type;
      a.page_size = c.page_size;
      a.num_pages = c.num_pages;
      a.k_cache = kc.data_ptr();
      a.v_cache = vc.data_ptr();
      a.slots = data<long long>(slots);
      a.k_scale = scale_of(arg[12], "k_scale", a.kv_heads, c.type, device);
      a.v_scale = scale_of(arg[13], "v_scale", a.kv_heads, c.type, device);
    }
    const c10::cuda::CUDAGuard guard(device);
    Tensor made[2];
    PyObject* result[2] = {Py_None, Py_None};
    for (int i = 0; i < 2; ++i) {
      PyObject* o = arg[14 + i];
      if (!given(o)) continue;
      const Tensor* in = i == 0 ? q : k;
      need(in != nullptr, "out_%s without its input", i == 0 ? "q" : "k");
      const int heads = i == 0 ? a.heads : a.kv_heads;
      const Tensor* out = &made[i];
      if (o == Py_True) {
        made[i] = at::empty({tokens, heads, dim}, at::TensorOptions().device(device).dtype(x.scalar_type()));
      } else {
        out = &tensor(o, i == 0 ? "out_q" : "out_k");
        apart(*out, in, i == 0 ? "out_q" : "out_k");
        result[i] = o;
      }
      auto& stride = i == 0 ? a.q_out_stride : a.k_out_stride;
      need(heads_of(*out, i == 0 ? "out_q" : "out_k", x, stride) == heads,
           "out_%s must have its input's shape", i == 0 ? "q" : "k");
      (i == 0 ? a.q_out : a.k_out) = out->data_ptr();
    }
    check(call_rotary(&a, stream_of(device), truth(arg[17])), "dg_rotary");
    for (int i : {5, 6, 14, 15}) written(arg[i]);
    PyObject* both = PyTuple_New(2);
    for (int i = 0; i < 2; ++i) {
      if (made[i].defined())
        PyTuple_SET_ITEM(both, i, THPVariable_Wrap(made[i]));
      else
        PyTuple_SET_ITEM(both, i, Py_NewRef(result[i]));
    }
    return both;
  });
}

Tensor new_workspace(c10::Device device) {
  Tensor ws = at::empty({static_cast<int64_t>(call_workspace_bytes())},
                        at::TensorOptions().device(device).dtype(at::kByte));
  ws.narrow(0, 0, kTicketBytes).zero_();         // the tickets; the rest is written before it is read
  return ws;
}

// A number for each host thread that asks, never given twice.
int64_t thread_number() {
  static std::atomic<int64_t> next{1};
  thread_local const int64_t mine = next++;
  return mine;
}

// Kept per stream: calls on one stream run one after another.  The per-thread
// default stream's handle names another stream in each host thread.  A captured
// graph may be replayed on any stream, so it gets its own, from its pool.
Tensor stream_workspace(c10::Device device, void* stream) {
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &capture) != cudaSuccess ||
      capture != cudaStreamCaptureStatusNone)
    return new_workspace(device);
  // (never destroyed: the process's end is no time to call the GPU's allocator)
  static auto* kept = new std::map<std::tuple<int, void*, int64_t>, Tensor>();
  Tensor& ws = (*kept)[{device.index(), stream, stream == cudaStreamPerThread ? thread_number() : 0}];
  if (!ws.defined()) ws = new_workspace(device);
  return ws;
}

// q, k_cache, v_cache, block_table, seq_lens, scale, window, softcap, k_scale,
// v_scale, out, return_lse, q_out, q_scales, workspace, status, pdl_attr
//   -> out, or (out, lse)
PyObject* paged_attention(PyObject*, PyObject* const* arg, Py_ssize_t count) {
  COUNT(17)
  return guarded([&]() -> PyObject* {
    no_trace("paged_attention");
    const Tensor& q = tensor(arg[0], "q");
    const Tensor& kc = tensor(arg[1], "k_cache");
    const Tensor& vc = tensor(arg[2], "v_cache");
    const Tensor& table = tensor(arg[3], "block_table");
    const Tensor& lens = tensor(arg[4], "seq_lens");
    const int kind = type_of(q.scalar_type());
    need(q.is_cuda() && q.dim() == 3 && (kind == DG_TYPE_BF16 || kind == DG_TYPE_FP16),
         "q must be a bf16 or fp16 CUDA tensor [batch, heads, dim]");
    for (int i : {0, 1, 2, 8, 9, 10, 12, 13}) no_gradient(arg[i], "paged_attention");
    const c10::Device device = q.device();
    const int64_t batch = q.size(0), heads = q.size(1), dim = q.size(2);
    need(batch >= 1 && batch <= kInt32Max && heads <= kInt32Max && q.stride(2) == 1 && q.stride(0) % 2 == 0 &&
             q.stride(1) % 2 == 0 && reinterpret_cast<uintptr_t>(q.data_ptr()) % 4 == 0,
         "q must be [batch >= 1, heads, dim], 4-byte aligned, with unit last and otherwise even strides");
    need(kc.dim() == 4, "the caches must be [pages, page_size, kv_heads, dim]");
    const int64_t kv_heads = kc.size(2);
    need(kv_heads >= 1 && heads >= 1 && heads % kv_heads == 0, "heads must be a multiple of the cache's heads");
    dg_attention_args a{};
    const Cache c = cache_of(kc, vc, kv_heads, q, a.k_cache_stride,
                             a.v_cache_stride);
    const int unit = c.type == DG_TYPE_E4M3 ? 16 : 8;    // 16 bytes
    need(dim >= 8 && dim <= 256 && dim % unit == 0, "dim must be a multiple of %d, at most 256", unit);
    bool aligned = (reinterpret_cast<uintptr_t>(kc.data_ptr()) | reinterpret_cast<uintptr_t>(vc.data_ptr())) % 16 == 0;
    for (int i = 0; i < 3; ++i) aligned = aligned && (a.k_cache_stride[i] | a.v_cache_stride[i]) % unit == 0;
    need(aligned, "the caches must be 16-byte aligned, strides multiples of 16 bytes");
    const auto [width, table_stride] = table_of(table, batch, device);
    vector_of(lens, "seq_lens", batch, device, at::kInt);
    a.batch = static_cast<int>(batch);
    a.heads = static_cast<int>(heads);
    a.kv_heads = static_cast<int>(kv_heads);
    a.head_dim = static_cast<int>(dim);
    a.page_size = c.page_size;
    a.num_pages = c.num_pages;
    a.table_width = width;
    a.type = kind;
    a.cache_type = c.type;
    a.scale = given(arg[5]) ? static_cast<float>(real(arg[5], "scale"))
                            : static_cast<float>(1.0 / std::sqrt(static_cast<double>(dim)));
    need(!std::isnan(a.scale), "scale must be a number");
    if (given(arg[6])) {
      const int64_t window = whole(arg[6], "window");
      need(window >= 1 && window <= kInt32Max, "window must be at least 1");
      a.window = static_cast<int>(window);
    }
    if (given(arg[7])) {
      const double cap = real(arg[7], "softcap");
      need(cap > 0.0 && static_cast<float>(cap) > 0.0f && std::isfinite(static_cast<float>(cap)),
           "softcap must be positive");
      a.softcap = static_cast<float>(cap);
    }
    a.q = q.data_ptr();
    a.q_stride[0] = q.stride(0);
    a.q_stride[1] = q.stride(1);
    a.k_cache = kc.data_ptr();
    a.v_cache = vc.data_ptr();
    a.block_table = data<int>(table);
    a.table_stride = table_stride;
    a.seq_lens = data<int>(lens);
    a.k_scale = scale_of(arg[8], "k_scale", kv_heads, c.type, device);
    a.v_scale = scale_of(arg[9], "v_scale", kv_heads, c.type, device);
    a.status = status_of(arg[15], device);
    const c10::cuda::CUDAGuard guard(device);
    const auto options = at::TensorOptions().device(device);
    Tensor made, lse;
    if (given(arg[10])) {
      const Tensor& out = tensor(arg[10], "out");
      need(heads_of(out, "out", q, a.out_stride) == heads,
           "out must have q's shape");
      apart(out, nullptr, "out");
      a.out = out.data_ptr();
    }
    if (given(arg[12]) || given(arg[13])) {
      need(given(arg[12]) && given(arg[13]), "q_out and q_scales go together");
      need(kind == DG_TYPE_BF16 && dim % 128 == 0, "the quantised result takes bf16 and dim a multiple of 128");
      const Tensor& bits = tensor(arg[12], "q_out");
      const Tensor& scales = tensor(arg[13], "q_scales");
      const int64_t n = heads * dim;
      need(type_of(bits.scalar_type()) == DG_TYPE_E4M3 && bits.dim() == 2 && bits.size(0) == batch &&
               bits.size(1) == n && bits.is_contiguous() && bits.device() == device,
           "q_out must be uint8 [%lld, %lld], contiguous", static_cast<long long>(batch), static_cast<long long>(n));
      need(scales.scalar_type() == at::kFloat && scales.dim() == 2 && scales.size(0) == batch &&
               scales.size(1) == n / 128 && scales.is_contiguous() && scales.device() == device,
           "q_scales must be fp32 [%lld, %lld], contiguous", static_cast<long long>(batch),
           static_cast<long long>(n / 128));
      a.q_out = bits.data_ptr();
      a.q_scales = data<float>(scales);
    }
    void* stream = stream_of(device);
    Tensor ws;
    if (given(arg[14])) {
      ws = tensor(arg[14], "workspace");
      need(ws.device() == device && ws.is_contiguous() && reinterpret_cast<uintptr_t>(ws.data_ptr()) % 16 == 0 &&
               ws.nbytes() >= call_workspace_bytes(),
           "workspace must come from attention_workspace() on %s", device.str().c_str());
    } else {
      ws = stream_workspace(device, stream);
    }
    a.workspace = ws.data_ptr();
    a.workspace_bytes = ws.nbytes();
    if (a.out == nullptr) {
      made = at::empty({batch, heads, dim}, options.dtype(q.scalar_type()));
      a.out = made.data_ptr();
      a.out_stride[0] = heads * dim;
      a.out_stride[1] = dim;
    }
    if (truth(arg[11])) {
      lse = at::empty({batch, heads}, options.dtype(at::kFloat));
      a.lse = data<float>(lse);
    }
    check(call_attention(&a, stream, truth(arg[16])), "dg_paged_attention");
    for (int i : {10, 12, 13}) written(arg[i]);
    PyObject* out = made.defined() ? THPVariable_Wrap(made) : Py_NewRef(arg[10]);
    if (!lse.defined()) return out;
    PyObject* both = PyTuple_New(2);
    PyTuple_SET_ITEM(both, 0, out);
    PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(lse));
    return both;
  });
}

// Addresses of dg_build_block_tables, dg_rotary, dg_paged_attention,
// dg_attention_workspace_bytes.
PyObject* bind(PyObject*, PyObject* const* arg, Py_ssize_t count) {
  COUNT(4)
  void* p[4];
  for (int i = 0; i < 4; ++i) {
    p[i] = PyLong_AsVoidPtr(arg[i]);
    if (p[i] == nullptr) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind() takes four addresses");
      return nullptr;
    }
  }
  call_tables = reinterpret_cast<int (*)(const dg_block_tables*, void*, int)>(p[0]);
  call_rotary = reinterpret_cast<int (*)(const dg_rotary_args*, void*, int)>(p[1]);
  call_attention = reinterpret_cast<int (*)(const dg_attention_args*, void*, int)>(p[2]);
  call_workspace_bytes = reinterpret_cast<unsigned long long (*)()>(p[3]);
  Py_RETURN_NONE;
}

PyCFunction fast(PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef methods[] = {{"bind", fast(bind), METH_FASTCALL, nullptr},
                         {"build_block_tables", fast(build_block_tables), METH_FASTCALL, nullptr},
                         {"rotary", fast(rotary), METH_FASTCALL, nullptr},
                         {"paged_attention", fast(paged_attention), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// Compiled against the torch and Python that the build names here: the module
// is of no use to others.
PyMODINIT_FUNC PyInit__host(void) {
  PyObject* m = PyModule_Create(&module);
  if (m != nullptr && PyModule_AddStringConstant(m, "built_for", DG_BUILT_FOR) != 0) Py_CLEAR(m);
  return m;
}
