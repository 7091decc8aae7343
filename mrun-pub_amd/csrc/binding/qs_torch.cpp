// The per-call half of the operators around the 4-bit KV cache: argument checks, output allocation,
// current stream and the C entry point in one call from Python.  A decode step makes two of these
// calls a layer, each of a few microseconds on the GPU; in Python the same work takes 10 to 20 us.
//
// The entry points themselves come from libqstore_hip.so as addresses (bind), so this module links
// to torch alone.  Refusals are ValueError for arguments, RuntimeError for the rest.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/InferenceMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <map>
#include <optional>
#include <stdexcept>
#include <string>
#include <utility>

#include "../../../include/qstore_hip.h"

namespace {

struct Refusal : std::runtime_error {  // ValueError
  using std::runtime_error::runtime_error;
};

#define REFUSE(cond, text) \
  do {                     \
    if (cond) throw Refusal(text); \
  } while (0)

struct Entries {
  decltype(&qs_plan_step) plan_step;
  decltype(&qs_rotary) rotary;
  decltype(&qs_kv4_append) append;
  decltype(&qs_kv4_read) read;
  decltype(&qs_kv4_attend) attend;
  decltype(&qs_kv4_attend_workspace_bytes) attend_space;
  decltype(&qs_last_error) last_error;
} entry;

void check(int status, const char* what) {
  if (status == QS_OK) return;
  const std::string text = std::string(what) + ": " + entry.last_error();
  if (status == QS_ERR_INVALID || status == QS_ERR_LIMIT) throw Refusal(text);
  throw std::runtime_error(text);
}

// ---- arguments -------------------------------------------------------------------------------

const at::Tensor& tensor(PyObject* o, const char* name) {
  REFUSE(!THPVariable_Check(o), std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}
int64_t whole(PyObject* o, const char* name) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Refusal(std::string(name) + " must be a whole number");
  }
  return v;
}
double number(PyObject* o, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Refusal(std::string(name) + " must be a number");
  }
  return v;
}

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return QS_F32;
    case at::kBFloat16: return QS_BF16;
    case at::kHalf: return QS_F16;
    case at::kInt: return QS_I32;
    case at::kLong: return QS_I64;
    default: throw Refusal("unsupported dtype");
  }
}
bool activation(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }

// All tensors live on one HIP device.
struct Device {
  int index = -1;
  void add(const at::Tensor& t) {
    REFUSE(!t.is_cuda(), "QStore HIP operators require tensors on a HIP (cuda) device");
    const int i = t.get_device();
    REFUSE(index >= 0 && i != index, "QStore HIP operator tensors must share one device");
    index = i;
  }
  c10::Device place() const { return c10::Device(c10::kCUDA, index); }
  // The default stream is a null handle, which means the current device's: calls run under a guard.
  void* stream() const { return c10::hip::getCurrentHIPStream(index).stream(); }
  at::Tensor empty(at::IntArrayRef size, at::ScalarType type) const {
    return at::detail::empty_cuda(size, type, place(), std::nullopt);
  }
};

// Makes the tensors' device the current one for a call, if it is not already.
struct Here {
  std::optional<c10::DeviceGuard> guard;
  explicit Here(const Device& d) {
    if (c10::hip::current_device() != d.index) guard.emplace(d.place());
  }
};

// A vector over part of a tensor's storage, `offset` in values of its own type.
at::Tensor part_of(const at::Tensor& whole, at::ScalarType type, int64_t offset, int64_t size) {
  auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), at::scalarTypeToTypeMeta(type));
  impl->set_storage_offset(offset);
  impl->set_sizes_contiguous(at::IntArrayRef(&size, 1));
  return at::Tensor(std::move(impl));
}

// Values from one entry of a dimension to the next; a dimension of one has no next, whatever its stride.
int64_t step(const at::Tensor& t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }

at::Tensor vector_of(const at::Tensor& t, at::ScalarType type) {
  if (t.scalar_type() == type && t.is_contiguous()) return t;
  return t.to(type).contiguous();
}
at::Tensor lengths(const at::Tensor& t, int64_t n, const char* name) {
  REFUSE(t.dim() != 1 || t.numel() != n || (t.scalar_type() != at::kInt && t.scalar_type() != at::kLong),
         std::string(name) + " must be an int32 or int64 vector of one length per request");
  return vector_of(t, at::kInt);
}
at::Tensor positions_of(const at::Tensor& t, int64_t tokens) {
  REFUSE(t.dim() != 1 || t.numel() != tokens, "positions must be one per token");
  REFUSE(t.scalar_type() != at::kInt && t.scalar_type() != at::kLong, "positions must be int32 or int64");
  return vector_of(t, at::kInt);
}
at::Tensor slots_of(const at::Tensor& t, int64_t tokens) {
  REFUSE(t.dim() != 1 || t.numel() != tokens || (t.scalar_type() != at::kInt && t.scalar_type() != at::kLong),
         "slots must be an int32 or int64 vector of one slot per token");
  return vector_of(t, at::kLong);
}
void check_tables(const at::Tensor& t, int64_t requests) {
  REFUSE(t.dim() != 2 || t.scalar_type() != at::kInt || t.size(0) != requests,
         "block tables must be int32 [requests, columns]");
  REFUSE(t.numel() && t.size(1) > 1 && t.stride(1) != 1, "block table rows must be contiguous");
}

// [tokens, heads, head_dim] with heads aligned to `values` values, copied if it is not.
at::Tensor heads_of(const at::Tensor& x, const char* name, int64_t tokens, int64_t heads, int64_t head_dim, int values) {
  REFUSE(x.dim() != 3 || x.size(0) != tokens || x.size(2) != head_dim,
         std::string(name) + " must have shape [" + std::to_string(tokens) + ", heads, " + std::to_string(head_dim) + "]");
  REFUSE(heads >= 0 && x.size(1) != heads, std::string(name) + " must have " + std::to_string(heads) + " heads");
  const auto off = [&](const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % (t.element_size() * values); };
  if (x.stride(2) == 1 && step(x, 0) % values == 0 && step(x, 1) % values == 0 && !off(x)) return x;
  at::Tensor y = x.contiguous();
  return off(y) ? y.clone() : y;  // a contiguous view may start off the grid
}

struct Cache {  // a layer of a KV4Cache, as (storage, bases, kv_heads, head_dim, pages, page_size)
  at::Tensor storage;
  PyObject* bases;
  int64_t kv_heads, head_dim, pages, page_size;
  explicit Cache(PyObject* o) {
    REFUSE(!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 6, "not a KV cache");
    storage = tensor(PyTuple_GET_ITEM(o, 0), "cache storage");
    bases = PyTuple_GET_ITEM(o, 1);
    kv_heads = whole(PyTuple_GET_ITEM(o, 2), "kv_heads");
    head_dim = whole(PyTuple_GET_ITEM(o, 3), "head_dim");
    pages = whole(PyTuple_GET_ITEM(o, 4), "pages");
    page_size = whole(PyTuple_GET_ITEM(o, 5), "page_size");
  }
  uint8_t* layer(PyObject* o) const {
    const int64_t i = whole(o, "layer"), n = PyTuple_GET_SIZE(bases);
    REFUSE(i < 0 || i >= n, "layer " + std::to_string(i) + " of a cache of " + std::to_string(n));
    return reinterpret_cast<uint8_t*>(whole(PyTuple_GET_ITEM(bases, i), "layer address"));
  }
};

// A workspace whose first kSyncBytes are zero, for kernels that leave them zero: one a stream, whose
// calls follow one another.  A call that is captured into a graph, which may run beside them, gets
// one of its own, cleared in the graph.
constexpr int64_t kSyncBytes = 32768;
at::Tensor workspace(const Device& device, void* stream, int64_t need) {
  static auto* kept = new std::map<std::pair<int, void*>, at::Tensor>;  // outlives the runtime's end
  const bool capturing = c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None;
  at::Tensor* have = capturing ? nullptr : &(*kept)[{device.index, stream}];
  if (have && have->defined() && have->numel() >= need) return *have;
  at::Tensor fresh = device.empty({need}, at::kByte);
  fresh.narrow(0, 0, kSyncBytes).zero_();
  if (have) *have = fresh;
  return fresh;
}

PyObject* give(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }

// Runs f with C++ exceptions turned into Python's.
template <class F>
PyObject* guarded(F f) {
  try {
    c10::InferenceMode inference(true);
    return f();
  } catch (const Refusal& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}
void count_args(Py_ssize_t n, Py_ssize_t want) { REFUSE(n != want, "wrong number of arguments"); }

// ---- operators -------------------------------------------------------------------------------

// ring, free_state, block_tables, past_lens, new_lens, page_size, tokens
PyObject* plan_step(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count_args(n, 7);
    const at::Tensor &ring = tensor(v[0], "ring"), &state = tensor(v[1], "free_state"), &tables = tensor(v[2], "block_tables");
    REFUSE(ring.dim() != 1 || ring.scalar_type() != at::kInt || !ring.numel() || !ring.is_contiguous(),
           "the ring of free pages must be a contiguous int32 vector");
    REFUSE(state.dim() != 1 || state.numel() != 3 || state.scalar_type() != at::kLong || !state.is_contiguous(),
           "the pool's state must be three int64");
    const at::Tensor& past_in = tensor(v[3], "past_lens");
    const int64_t B = past_in.numel(), T = whole(v[6], "tokens");
    const at::Tensor past = lengths(past_in, B, "past_lens"), fresh = lengths(tensor(v[4], "new_lens"), B, "new_lens");
    check_tables(tables, B);
    REFUSE(T < 0, "tokens must not be negative");
    Device d;
    d.add(ring), d.add(state), d.add(tables), d.add(past), d.add(fresh);
    const Here here(d);
    // one allocation: slots and state in int64, then the rest in int32
    const at::Tensor all = d.empty({T + 3 + T + B + 1}, at::kLong);
    const int64_t words = 2 * (T + 3);
    at::Tensor slots = part_of(all, at::kLong, 0, T), next = part_of(all, at::kLong, T, 3);
    at::Tensor positions = part_of(all, at::kInt, words, T), requests = part_of(all, at::kInt, words + T, T);
    at::Tensor starts = part_of(all, at::kInt, words + 2 * T, B + 1), context = part_of(all, at::kInt, words + 2 * T + B + 1, B);
    check(entry.plan_step(static_cast<int32_t*>(ring.data_ptr()), ring.numel(), static_cast<int64_t*>(state.data_ptr()),
                          static_cast<int64_t*>(next.data_ptr()), static_cast<int32_t*>(tables.data_ptr()), tables.stride(0),
                          tables.size(1), static_cast<int32_t*>(past.data_ptr()), static_cast<int32_t*>(fresh.data_ptr()), B,
                          whole(v[5], "page_size"), T, static_cast<int64_t*>(slots.data_ptr()),
                          static_cast<int32_t*>(positions.data_ptr()), static_cast<int32_t*>(requests.data_ptr()),
                          static_cast<int32_t*>(starts.data_ptr()), static_cast<int32_t*>(context.data_ptr()), d.stream()),
          "qs_plan_step");
    PyObject* out = PyTuple_New(6);
    if (!out) return nullptr;
    at::Tensor* each[6] = {&slots, &positions, &requests, &starts, &context, &next};
    for (int i = 0; i < 6; ++i) PyTuple_SET_ITEM(out, i, give(std::move(*each[i])));
    return out;
  });
}

// x, positions, frequencies (None before a device is known), dim, interleaved, inverse, magnitude, out
PyObject* rotary(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count_args(n, 8);
    at::Tensor x = tensor(v[0], "rotary input");
    REFUSE(x.dim() != 3, "rotary input must have shape [tokens, heads, head_dim]");
    const int64_t T = x.size(0), H = x.size(1), D = x.size(2), dim = whole(v[3], "dim");
    REFUSE(dim > D, "rotary spec turns " + std::to_string(dim) + " values of a head of " + std::to_string(D));
    const int code = code_of(x.scalar_type());
    const at::Tensor pos = positions_of(tensor(v[1], "positions"), T);
    Device d;
    d.add(x), d.add(pos);
    const Here here(d);
    at::Tensor out;
    if (v[7] == Py_None) {
      out = d.empty({T, H, D}, x.scalar_type());
    } else {
      out = tensor(v[7], "rotary output");
      d.add(out);
      REFUSE(out.sizes() != x.sizes() || out.scalar_type() != x.scalar_type() || (D && out.stride(2) != 1),
             "rotary output must have the input's shape and type, with contiguous heads");
    }
    if (x.stride(2) != 1) x = x.contiguous();
    if (T == 0 || H == 0) return give(out);
    const at::Tensor& freq = tensor(v[2], "frequencies");
    d.add(freq);
    check(entry.rotary(x.data_ptr(), code, step(x, 0), step(x, 1), static_cast<int32_t*>(pos.data_ptr()),
                       static_cast<double*>(freq.data_ptr()), (int)dim, PyObject_IsTrue(v[4]), PyObject_IsTrue(v[5]),
                       number(v[6], "magnitude"), out.data_ptr(), step(out, 0), step(out, 1), T, (int)H, (int)D, d.stream()),
          "qs_rotary");
    return give(out);
  });
}

// cache, layer, k, v, slots, q, positions, rotary: None or (dim, interleaved, magnitude), frequencies
PyObject* append(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count_args(n, 9);
    const Cache cache(v[0]);
    at::Tensor k = tensor(v[2], "keys"), val = tensor(v[3], "values"), q;
    const bool has_q = v[5] != Py_None, has_pos = v[6] != Py_None, turns = v[7] != Py_None;
    if (has_q) q = tensor(v[5], "queries");
    REFUSE(val.scalar_type() != k.scalar_type() || (has_q && q.scalar_type() != k.scalar_type()),
           "queries, keys and values must share one type");
    REFUSE(!activation(k.scalar_type()), "keys and values must be float32, bfloat16 or float16");
    REFUSE(k.dim() != 3, "keys must have shape [tokens, heads, head_dim]");
    const int64_t T = k.size(0), D = cache.head_dim;
    k = heads_of(k, "keys", T, cache.kv_heads, D, 4);
    val = heads_of(val, "values", T, cache.kv_heads, D, 4);
    const at::Tensor slots = slots_of(tensor(v[4], "slots"), T);
    uint8_t* base = cache.layer(v[1]);
    Device d;
    d.add(k), d.add(val), d.add(slots), d.add(cache.storage);
    if (has_q) d.add(q);
    const Here here(d);
    at::Tensor pos, freq, out;
    if (has_pos) d.add(tensor(v[6], "positions"));
    REFUSE(turns != has_pos, "rotary positions need both a spec and positions");
    REFUSE(has_q && !turns, "queries are only turned: without rotary positions there is nothing to do for them");
    int64_t dim = 0;
    int interleaved = 0;
    double magnitude = 1.0;
    if (turns) {
      REFUSE(!PyTuple_Check(v[7]) || PyTuple_GET_SIZE(v[7]) != 3, "not a rotary spec");
      dim = whole(PyTuple_GET_ITEM(v[7], 0), "dim");
      REFUSE(dim > D || dim % 8, "the rotated size must be a multiple of 8 up to " + std::to_string(D));
      interleaved = PyObject_IsTrue(PyTuple_GET_ITEM(v[7], 1));
      magnitude = number(PyTuple_GET_ITEM(v[7], 2), "magnitude");
      pos = positions_of(tensor(v[6], "positions"), T);
      freq = tensor(v[8], "frequencies");
      d.add(freq);
    }
    int64_t Hq = 0, ldq_t = 0, ldq_h = 0;
    if (has_q) {
      q = heads_of(q, "queries", T, -1, D, 4);
      Hq = q.size(1), ldq_t = step(q, 0), ldq_h = step(q, 1);
      out = d.empty({T, Hq, D}, q.scalar_type());
    }
    check(entry.append(k.data_ptr(), step(k, 0), step(k, 1), val.data_ptr(), step(val, 0), step(val, 1),
                       code_of(k.scalar_type()), static_cast<int64_t*>(slots.data_ptr()), base, cache.pages, cache.page_size,
                       (int)cache.kv_heads, (int)D, T, has_q ? q.data_ptr() : nullptr, ldq_t, ldq_h, (int)Hq,
                       has_q ? out.data_ptr() : nullptr, turns ? static_cast<int32_t*>(pos.data_ptr()) : nullptr,
                       turns ? static_cast<double*>(freq.data_ptr()) : nullptr, (int)dim, interleaved, magnitude, d.stream()),
          "qs_kv4_append");
    if (!has_q) Py_RETURN_NONE;
    return give(out);
  });
}

// cache, layer, slots, a tensor of the wanted type's code
PyObject* read(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count_args(n, 4);
    const Cache cache(v[0]);
    const at::Tensor& slots_in = tensor(v[2], "slots");
    const int64_t count = slots_in.numel(), code = whole(v[3], "dtype");
    REFUSE(code != QS_F32 && code != QS_BF16 && code != QS_F16, "cache values are read as float32, bfloat16 or float16");
    const at::Tensor slots = slots_of(slots_in, count);
    uint8_t* base = cache.layer(v[1]);
    Device d;
    d.add(slots), d.add(cache.storage);
    const Here here(d);
    const auto type = code == QS_F32 ? at::kFloat : code == QS_BF16 ? at::kBFloat16 : at::kHalf;
    at::Tensor k = d.empty({count, cache.kv_heads, cache.head_dim}, type), val = d.empty({count, cache.kv_heads, cache.head_dim}, type);
    check(entry.read(base, cache.pages, cache.page_size, (int)cache.kv_heads, (int)cache.head_dim,
                     static_cast<int64_t*>(slots.data_ptr()), count, k.data_ptr(), val.data_ptr(), (int)code, d.stream()),
          "qs_kv4_read");
    PyObject* out = PyTuple_New(2);
    if (!out) return nullptr;
    PyTuple_SET_ITEM(out, 0, give(std::move(k)));
    PyTuple_SET_ITEM(out, 1, give(std::move(val)));
    return out;
  });
}

// q, cache, layer, block_tables, query_starts, context_lens, max_query, max_context, scale, window, out
PyObject* attend(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count_args(n, 11);
    at::Tensor q = tensor(v[0], "queries"), out;
    const Cache cache(v[1]);
    REFUSE(q.dim() != 3 || !activation(q.scalar_type()), "queries must be float32, bfloat16 or float16 [tokens, heads, head_dim]");
    const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2);
    REFUSE(D != cache.head_dim || Hq < 1 || Hq % cache.kv_heads,
           "query heads must be a multiple of the cache's KV heads, of its head size");
    const at::Tensor &tables = tensor(v[3], "block_tables"), &starts_in = tensor(v[4], "query_starts"), &ctx_in = tensor(v[5], "context_lens");
    const int64_t B = ctx_in.numel();
    check_tables(tables, B);
    REFUSE(starts_in.dim() != 1 || starts_in.numel() != B + 1 || starts_in.scalar_type() != at::kInt,
           "query_starts must be int32, one more than requests");
    REFUSE(ctx_in.dim() != 1 || ctx_in.scalar_type() != at::kInt, "context_lens must be an int32 vector");
    const int64_t width = tables.size(1), most = width * cache.page_size;
    const int64_t max_query = v[6] == Py_None ? T : whole(v[6], "max_query");
    int64_t max_context = v[7] == Py_None ? most : whole(v[7], "max_context");
    const int64_t window = v[9] == Py_None ? 0 : whole(v[9], "window");
    REFUSE(max_query < 0 || max_context < 0 || (v[9] != Py_None && window < 1),
           "bounds must not be negative and a window holds at least one token");
    if (max_context > most) max_context = most;
    const double scale = v[8] == Py_None ? 1.0 / std::sqrt((double)D) : number(v[8], "scale");
    q = heads_of(q, "queries", T, -1, D, q.scalar_type() == at::kFloat ? 4 : 8);
    const at::Tensor starts = starts_in.contiguous(), ctx = ctx_in.contiguous();
    uint8_t* base = cache.layer(v[2]);
    Device d;
    d.add(q), d.add(cache.storage), d.add(tables), d.add(starts), d.add(ctx);
    const Here here(d);
    if (v[10] == Py_None) {
      out = d.empty({T, Hq, D}, q.scalar_type());
    } else {
      out = tensor(v[10], "attention output");
      d.add(out);
      REFUSE(out.sizes() != q.sizes() || out.scalar_type() != q.scalar_type() || !out.is_contiguous() ||
                 reinterpret_cast<uintptr_t>(out.data_ptr()) % 16,
             "attention output must be contiguous, 16-byte aligned, of the queries' shape and type");
    }
    void* stream = d.stream();
    const int64_t need = (int64_t)entry.attend_space(T, B, (int)cache.kv_heads, (int)Hq, (int)D, cache.page_size, max_query,
                                                     max_context, window);
    at::Tensor space;
    if (need) space = workspace(d, stream, need);
    check(entry.attend(q.data_ptr(), code_of(q.scalar_type()), step(q, 0), step(q, 1), base, cache.pages, cache.page_size,
                       (int)cache.kv_heads, (int)Hq, (int)D, static_cast<int32_t*>(tables.data_ptr()), tables.stride(0), width,
                       static_cast<int32_t*>(starts.data_ptr()), static_cast<int32_t*>(ctx.data_ptr()), B, T, max_query,
                       max_context, (float)scale, window, out.data_ptr(), need ? space.data_ptr() : nullptr, (size_t)need, stream),
          "qs_kv4_attend");
    return give(out);
  });
}

// Addresses of the C entry points, in the order of Entries.
PyObject* bind(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count_args(n, 7);
    void* at[7];
    for (int i = 0; i < 7; ++i) at[i] = reinterpret_cast<void*>(whole(v[i], "address"));
    entry.plan_step = reinterpret_cast<decltype(entry.plan_step)>(at[0]);
    entry.rotary = reinterpret_cast<decltype(entry.rotary)>(at[1]);
    entry.append = reinterpret_cast<decltype(entry.append)>(at[2]);
    entry.read = reinterpret_cast<decltype(entry.read)>(at[3]);
    entry.attend = reinterpret_cast<decltype(entry.attend)>(at[4]);
    entry.attend_space = reinterpret_cast<decltype(entry.attend_space)>(at[5]);
    entry.last_error = reinterpret_cast<decltype(entry.last_error)>(at[6]);
    Py_RETURN_NONE;
  });
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind),  METHOD(plan_step), METHOD(rotary), METHOD(append),
                         METHOD(read), METHOD(attend),    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_qs_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// built_for: the torch whose C++ interface this was compiled against, which no other need have.
PyMODINIT_FUNC PyInit__qs_torch() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "built_for", QS_BUILT_FOR) != 0) Py_CLEAR(m);
  return m;
}
