// qg_paged_torch.cpp -- the torch front end of the paged cache operators: checks tensors, makes
// the ones that a call returns and calls the C-ABI (include/qgemv_b200.h).  Small batches are
// bound by the host: with the same checks in Python a call took 12 us (append), 10 (attend) and 14
// (evict), now 5, 6 and 8, of which the launches are 3, 3 and 5.
//
// A CPython module (qgemv_b200/paged.py and paged8.py are its only users).  It does not link the library: bind()
// is given the addresses of its entry points.  No device code, no computation.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <initializer_list>
#include <optional>

#include "../../include/qgemv_b200.h"

namespace {

struct Entries {
  decltype(&qg_qk_norm_rope_append) append = nullptr;
  decltype(&qg_paged_attn) attn = nullptr;
  decltype(&qg_kv_evict) evict = nullptr;
  decltype(&qg_qk_norm_rope_append8) append8 = nullptr;
  decltype(&qg_kv_read8) read8 = nullptr;
  decltype(&qg_paged_attn8) attn8 = nullptr;
} g_entries;

// What a PagedCache and an AttentionPlan hold: addresses, and the storages that they lie in, so
// that no memory goes back to the allocator while a description of it lives, whatever becomes of
// the caller's tensors.
struct Cache {
  qg_kv_pages pages;
  int index;  // device
  c10::Storage k, v, table;
};
struct Plan {
  Cache cache;
  uint32_t n_q, max_len;
  bool weights;
  void* workspace;
  c10::Storage space;
};
struct Cache8 {
  qg_kv_pages8 pages;
  int index;
  c10::Storage k, v, k_scale, v_scale, table;
};
struct Plan8 {
  Cache8 cache;
  uint32_t n_q, tokens;
  void* workspace;
  c10::Storage space;
};
constexpr char kCache8Name[] = "qgemv_b200.paged8.cache", kPlan8Name[] = "qgemv_b200.paged8.plan";
constexpr char kCacheName[] = "qgemv_b200.paged.cache", kPlanName[] = "qgemv_b200.paged.plan";

template <typename S>
S* held(PyObject* capsule, const char* name) {
  return static_cast<S*>(PyCapsule_GetPointer(capsule, name));
}
template <typename S>
PyObject* hold(const S& value, const char* name) {
  S* copy = new S(value);
  PyObject* capsule = PyCapsule_New(copy, name, [](PyObject* c) {
    delete static_cast<S*>(PyCapsule_GetPointer(c, PyCapsule_GetName(c)));
  });
  if (capsule == nullptr) delete copy;
  return capsule;
}

// A call's arguments in order; the first one that does not fit raises ValueError.
struct Refused {};
[[noreturn]] void refuse(const char* name, const std::string& what) {
  PyErr_SetString(PyExc_ValueError, (std::string(name) + ": " + what).c_str());
  throw Refused();
}
const at::Tensor& tensor_of(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(name, "a tensor is needed");
  return THPVariable_Unpack(o);
}
std::string shape_text(std::initializer_list<int64_t> shape) {
  std::string s = "[";
  for (int64_t n : shape) s += (s.size() > 1 ? ", " : "") + std::to_string(n);
  return s + "]";
}
bool on(const at::Tensor& t, int index) { return t.is_cuda() && t.get_device() == index; }

// Stride from row to row of a [rows, heads, dim] tensor whose rows are contiguous.
uint64_t heads_of(const at::Tensor& t, int64_t rows, int64_t heads, int64_t dim, at::ScalarType type, int index,
                  const char* name) {
  if (t.dim() != 3 || t.size(0) != rows || t.size(1) != heads || t.size(2) != dim || t.scalar_type() != type ||
      !on(t, index)) {
    refuse(name, std::string("a ") + at::toString(type) + " tensor of shape " + shape_text({rows, heads, dim}) +
                     " on cuda:" + std::to_string(index) + " is needed");
  }
  if ((t.stride(2) != 1 && dim > 1) || (t.stride(1) != dim && heads > 1)) {
    refuse(name, "the heads of one row must be contiguous");
  }
  return static_cast<uint64_t>(rows > 1 ? t.stride(0) : heads * dim);
}
void* ints_of(const at::Tensor& t, int64_t n, int index, const char* name) {
  if (t.scalar_type() != at::kInt || t.numel() != n || !t.is_contiguous() || !on(t, index)) {
    refuse(name, "a contiguous int32 tensor of " + std::to_string(n) + " entries on cuda:" + std::to_string(index) +
                     " is needed");
  }
  return t.data_ptr();
}
const int32_t* ints_or_null(PyObject* o, int64_t n, int index, const char* name) {
  return o == Py_None ? nullptr : static_cast<const int32_t*>(ints_of(tensor_of(o, name), n, index, name));
}
float* floats_of(const at::Tensor& t, std::initializer_list<int64_t> shape, int index, const char* name) {
  if (t.scalar_type() != at::kFloat || t.sizes() != at::IntArrayRef(shape) || !t.is_contiguous() || !on(t, index)) {
    refuse(name, "a contiguous float32 tensor of shape " + shape_text(shape) + " on cuda:" + std::to_string(index) +
                     " is needed");
  }
  return static_cast<float*>(t.data_ptr());
}
float* floats_or_null(PyObject* o, std::initializer_list<int64_t> shape, int index, const char* name) {
  return o == Py_None ? nullptr : floats_of(tensor_of(o, name), shape, index, name);
}
int dtype_code(at::ScalarType type, const char* name) {
  switch (type) {
    case at::kFloat: return QG_F32;
    case at::kHalf: return QG_F16;
    case at::kBFloat16: return QG_BF16;
    default: refuse(name, "float32, float16 or bfloat16 is needed");
  }
}
int dtype_of(const at::Tensor& t, const char* name) { return dtype_code(t.scalar_type(), name); }
// A number of slots, heads and the like; one that is none becomes the largest, which the
// library refuses.
uint32_t count_of(PyObject* o) {
  const long long n = PyLong_AsLongLong(o);
  if (n == -1 && PyErr_Occurred() != nullptr) throw Refused();
  return n < 0 || n > 0xffffffffll ? 0xffffffffu : static_cast<uint32_t>(n);
}
float number_of(PyObject* o) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred() != nullptr) throw Refused();
  return static_cast<float>(x);
}

// The device and stream of a call: tensors made in it belong to that stream.  `handle` is a
// cudaStream_t as an int, None for the current stream.
struct Call {
  c10::cuda::CUDAGuard device;
  cudaStream_t stream;
  std::optional<c10::cuda::CUDAStreamGuard> scope;
  Call(int index, PyObject* handle) : device(static_cast<c10::DeviceIndex>(index)) {
    if (handle == Py_None) {
      stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index)).stream();
    } else {
      stream = static_cast<cudaStream_t>(PyLong_AsVoidPtr(handle));
      scope.emplace(c10::cuda::getStreamFromExternal(stream, static_cast<c10::DeviceIndex>(index)));
    }
  }
};

template <typename F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F body) {
  HANDLE_TH_ERRORS
  if (n != want) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  try {
    return body();
  } catch (const Refused&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// bind(append, attn, evict): addresses of the library's entry points
PyObject* py_bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 3, [&]() -> PyObject* {
    g_entries.append = reinterpret_cast<decltype(g_entries.append)>(PyLong_AsVoidPtr(args[0]));
    g_entries.attn = reinterpret_cast<decltype(g_entries.attn)>(PyLong_AsVoidPtr(args[1]));
    g_entries.evict = reinterpret_cast<decltype(g_entries.evict)>(PyLong_AsVoidPtr(args[2]));
    if (PyErr_Occurred() != nullptr) throw Refused();
    Py_RETURN_NONE;
  });
}

// cache(k, v, table) -> (held description, address of its qg_kv_pages)
PyObject* py_cache(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 3, [&]() -> PyObject* {
    const at::Tensor &k = tensor_of(args[0], "k"), &v = tensor_of(args[1], "v"), &table = tensor_of(args[2], "table");
    auto step = [](const at::Tensor& t, int d) { return t.size(d) > 1 ? t.stride(d) : 0; };  // one entry: no step
    bool alike = k.dim() == 4 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type();
    for (int d = 0; alike && d < 4; ++d) alike = step(k, d) == step(v, d);
    if (!alike) refuse("k and v", "two [pages, heads, page size, dim] tensors of one type and layout are needed");
    if (!k.is_cuda() || k.device() != v.device() || k.device() != table.device()) {
      refuse("k, v and table", "have to be on one CUDA device (there is no CPU path)");
    }
    if ((k.scalar_type() != at::kHalf && k.scalar_type() != at::kBFloat16) || (k.size(3) > 1 && k.stride(3) != 1)) {
      refuse("k and v", "float16 or bfloat16 with contiguous dims are needed");
    }
    if (table.scalar_type() != at::kInt || table.dim() != 2 || (table.size(1) > 1 && table.stride(1) != 1)) {
      refuse("table", "an int32 tensor [sequences, pages per sequence] is needed");
    }
    for (int64_t size : {k.size(0), k.size(1), k.size(2), table.size(0), table.size(1), table.stride(0)}) {
      if (size > 0x7fffffff) refuse("k, v and table", "sizes below 2^31 are needed");
    }
    Cache c{};
    c.index = k.get_device();
    c.pages.k = k.data_ptr();
    c.pages.v = v.data_ptr();
    c.pages.dtype = dtype_of(k, "k");
    c.pages.num_pages = static_cast<uint32_t>(k.size(0));
    c.pages.n_kv_heads = static_cast<uint32_t>(k.size(1));
    c.pages.page_size = static_cast<uint32_t>(k.size(2));
    c.pages.head_dim = static_cast<uint32_t>(k.size(3));
    c.pages.page_stride = static_cast<uint64_t>(step(k, 0));
    c.pages.head_stride = static_cast<uint64_t>(step(k, 1));
    c.pages.slot_stride = static_cast<uint64_t>(step(k, 2));
    c.pages.table = static_cast<const int32_t*>(table.data_ptr());
    c.pages.batch = static_cast<uint32_t>(table.size(0));
    c.pages.table_pages = static_cast<uint32_t>(table.size(1));
    c.pages.table_stride = static_cast<uint32_t>(table.size(0) > 1 ? table.stride(0) : table.size(1));
    c.k = k.storage();
    c.v = v.storage();
    c.table = table.storage();
    PyObject* capsule = hold(c, kCacheName);
    if (capsule == nullptr) return nullptr;
    PyObject* at = PyLong_FromVoidPtr(&held<Cache>(capsule, kCacheName)->pages);
    if (at == nullptr) {
      Py_DECREF(capsule);
      return nullptr;
    }
    return Py_BuildValue("(NN)", capsule, at);
  });
}

// plan(cache, n_q_heads, max_len, weights, workspace) -> held plan
PyObject* py_plan(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 5, [&]() -> PyObject* {
    Plan p{};
    const Cache* cache = held<Cache>(args[0], kCacheName);
    if (cache == nullptr) throw Refused();
    p.cache = *cache;
    p.n_q = count_of(args[1]);
    p.max_len = count_of(args[2]);
    p.weights = args[3] == Py_True;
    const at::Tensor& workspace = tensor_of(args[4], "workspace");
    p.workspace = workspace.data_ptr();
    p.space = workspace.storage();
    return hold(p, kPlanName);
  });
}

// append(cache, q, k, v, rope, positions, slots, seqs, q_norm, k_norm, eps, pairs, q_out, stream)
// -> (cudaError_t, q_out)
PyObject* py_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 14, [&]() -> PyObject* {
    const Cache* c = held<Cache>(args[0], kCacheName);
    if (c == nullptr) throw Refused();
    const at::Tensor &q = tensor_of(args[1], "q"), &k = tensor_of(args[2], "k"), &v = tensor_of(args[3], "v");
    if (q.dim() != 3) refuse("q", "a [tokens, heads, dim] tensor is needed");
    const int64_t tokens = q.size(0), heads = q.size(1), dim = c->pages.head_dim, kv = c->pages.n_kv_heads;
    if (tokens > 0x7fffffff || heads > 0xffff) refuse("q", "at most 2^31 - 1 tokens and 65535 heads are taken");
    const at::ScalarType type = q.scalar_type();
    qg_append a{};
    a.dtype = dtype_of(q, "q");
    a.tokens = static_cast<uint32_t>(tokens);
    a.n_q_heads = static_cast<uint32_t>(heads);
    a.q_stride = heads_of(q, tokens, heads, dim, type, c->index, "q");
    a.k_stride = heads_of(k, tokens, kv, dim, type, c->index, "k");
    a.v_stride = heads_of(v, tokens, kv, dim, type, c->index, "v");
    a.q = q.data_ptr();
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.q_norm = floats_or_null(args[8], {dim}, c->index, "q_norm");
    a.k_norm = floats_or_null(args[9], {dim}, c->index, "k_norm");
    a.eps = number_of(args[10]);
    if (args[4] != Py_None) {
      const at::Tensor& rope = tensor_of(args[4], "rope");
      if (rope.dim() != 2 || rope.size(0) > 0x7fffffff || rope.size(1) > 0x7fffffff) refuse("rope", "[rows, rot_dim] is needed");
      a.rope = floats_of(rope, {rope.size(0), rope.size(1)}, c->index, "rope");
      a.rope_rows = static_cast<uint32_t>(rope.size(0));
      a.rot_dim = static_cast<uint32_t>(rope.size(1));
    }
    a.pairs = static_cast<int>(count_of(args[11]));
    a.positions = static_cast<const int32_t*>(ints_of(tensor_of(args[5], "positions"), tokens, c->index, "positions"));
    a.slots = ints_or_null(args[6], tokens, c->index, "slots");
    a.seqs = ints_or_null(args[7], tokens, c->index, "seqs");
    const Call call(c->index, args[13]);
    const at::Tensor q_out = args[12] == Py_None ? at::empty({tokens, heads, dim}, q.options()) : tensor_of(args[12], "q_out");
    a.q_out_stride = heads_of(q_out, tokens, heads, dim, type, c->index, "q_out");
    a.q_out = q_out.data_ptr();
    const cudaError_t e = g_entries.append(&c->pages, &a, call.stream);
    return Py_BuildValue("(iN)", static_cast<int>(e), THPVariable_Wrap(q_out));
  });
}

// attend(plan, q, lens, window, scale, out, lse, return_lse, weight_in, weight_out, stream)
// -> (cudaError_t, out, lse or None)
PyObject* py_attend(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 11, [&]() -> PyObject* {
    const Plan* p = held<Plan>(args[0], kPlanName);
    if (p == nullptr) throw Refused();
    const Cache* c = &p->cache;
    const at::Tensor& q = tensor_of(args[1], "q");
    const int64_t batch = c->pages.batch, heads = p->n_q, dim = c->pages.head_dim, kv = c->pages.n_kv_heads;
    const at::ScalarType type = q.scalar_type();
    qg_attn a{};
    a.dtype = dtype_of(q, "q");
    a.n_q_heads = p->n_q;
    a.max_len = p->max_len;
    a.q_stride = heads_of(q, batch, heads, dim, type, c->index, "q");
    a.q = q.data_ptr();
    a.lens = static_cast<const int32_t*>(ints_of(tensor_of(args[2], "lens"), batch, c->index, "lens"));
    a.window = count_of(args[3]);
    if (a.window == 0xffffffffu) refuse("window", "a number of slots is needed, 0 for all");
    a.scale = number_of(args[4]);
    if (args[9] != Py_None) {
      if (!p->weights) refuse("weight_out", "needs a plan with weights");
      const at::Tensor& w = tensor_of(args[9], "weight_out");
      const int64_t width = w.dim() == 3 ? w.size(2) : 0;
      if (width > 0x7fffffff) refuse("weight_out", "rows of fewer than 2^31 slots are needed");
      a.weight_out = floats_of(w, {batch, kv, width}, c->index, "weight_out");
      a.weight_in = floats_or_null(args[8], {batch, kv, width}, c->index, "weight_in");
      a.weight_stride = static_cast<uint32_t>(width);
    } else if (args[8] != Py_None) {
      refuse("weight_in", "needs weight_out");
    }
    const Call call(c->index, args[10]);
    const at::Tensor out = args[5] == Py_None ? at::empty({batch, heads, dim}, q.options()) : tensor_of(args[5], "out");
    a.out_stride = heads_of(out, batch, heads, dim, type, c->index, "out");
    a.out = out.data_ptr();
    at::Tensor lse;
    if (args[6] != Py_None) {
      lse = tensor_of(args[6], "lse");
    } else if (args[7] == Py_True) {
      lse = at::empty({batch, heads}, q.options().dtype(at::kFloat));
    }
    if (lse.defined()) a.lse = floats_of(lse, {batch, heads}, c->index, "lse");
    const cudaError_t e = g_entries.attn(&c->pages, &a, p->workspace, call.stream);
    PyObject* lse_out = Py_None;
    if (lse.defined()) {
      lse_out = THPVariable_Wrap(lse);
    } else {
      Py_INCREF(Py_None);
    }
    return Py_BuildValue("(iNN)", static_cast<int>(e), THPVariable_Wrap(out), lse_out);
  });
}

// evict(cache, lens, weight, budget, sink, recent, new_table, lens_out, weight_out, kept, stream)
// -> (cudaError_t, kept, lens_out)
PyObject* py_evict(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 11, [&]() -> PyObject* {
    const Cache* c = held<Cache>(args[0], kCacheName);
    if (c == nullptr) throw Refused();
    const int64_t batch = c->pages.batch, kv = c->pages.n_kv_heads;
    const at::Tensor &lens = tensor_of(args[1], "lens"), &weight = tensor_of(args[2], "weight");
    const int64_t width = weight.dim() == 3 ? weight.size(2) : 0;
    if (width > 0x7fffffff) refuse("weight", "rows of fewer than 2^31 slots are needed");
    qg_evict e{};
    e.lens = static_cast<const int32_t*>(ints_of(lens, batch, c->index, "lens"));
    e.weight = floats_of(weight, {batch, kv, width}, c->index, "weight");
    e.max_len = e.weight_stride = static_cast<uint32_t>(width);
    e.budget = count_of(args[3]);
    if (e.budget > 0x7fffffffu) refuse("budget", "a number of slots below 2^31 is needed");  // before it is made room for
    e.sink = count_of(args[4]);
    e.recent = count_of(args[5]);
    const bool elsewhere = args[6] != Py_None;
    if (elsewhere) {
      const at::Tensor& to = tensor_of(args[6], "new_table");
      if (to.scalar_type() != at::kInt || to.dim() != 2 || to.size(0) != batch || !on(to, c->index) ||
          (to.size(1) > 1 && to.stride(1) != 1) || to.size(1) > 0x7fffffff || to.stride(0) > 0x7fffffff) {
        refuse("new_table", "an int32 tensor [sequences, pages per sequence] is needed");
      }
      if (args[8] == Py_None) refuse("new_table", "needs weight_out: a tensor for the new weights, or weight itself");
      e.new_table = static_cast<const int32_t*>(to.data_ptr());
      e.new_table_pages = static_cast<uint32_t>(to.size(1));
      e.new_table_stride = static_cast<uint32_t>(batch > 1 ? to.stride(0) : to.size(1));
    }
    e.weight_out = args[8] == Py_None ? const_cast<float*>(e.weight)
                                      : floats_of(tensor_of(args[8], "weight_out"), {batch, kv, width}, c->index, "weight_out");
    const Call call(c->index, args[10]);
    const at::Tensor lens_out = args[7] != Py_None ? tensor_of(args[7], "lens_out")
                                : elsewhere        ? at::empty({batch}, lens.options())
                                                   : lens;
    e.lens_out = static_cast<int32_t*>(ints_of(lens_out, batch, c->index, "lens_out"));
    const at::Tensor kept = args[9] != Py_None ? tensor_of(args[9], "kept")
                                               : at::empty({batch, kv, static_cast<int64_t>(e.budget)}, lens.options());
    e.kept = static_cast<int32_t*>(ints_of(kept, batch * kv * static_cast<int64_t>(e.budget), c->index, "kept"));
    const cudaError_t err = g_entries.evict(&c->pages, &e, call.stream);
    return Py_BuildValue("(iNN)", static_cast<int>(err), THPVariable_Wrap(kept), THPVariable_Wrap(lens_out));
  });
}

// ---- the 8-bit cache

// bind8(append8, read8, attn8): addresses of the library's entry points
PyObject* py_bind8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 3, [&]() -> PyObject* {
    g_entries.append8 = reinterpret_cast<decltype(g_entries.append8)>(PyLong_AsVoidPtr(args[0]));
    g_entries.read8 = reinterpret_cast<decltype(g_entries.read8)>(PyLong_AsVoidPtr(args[1]));
    g_entries.attn8 = reinterpret_cast<decltype(g_entries.attn8)>(PyLong_AsVoidPtr(args[2]));
    if (PyErr_Occurred() != nullptr) throw Refused();
    Py_RETURN_NONE;
  });
}

// cache8(k, v, k_scale, v_scale, table) -> (held description, address of its qg_kv_pages8, block)
PyObject* py_cache8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 5, [&]() -> PyObject* {
    const at::Tensor &k = tensor_of(args[0], "k"), &v = tensor_of(args[1], "v"), &ks = tensor_of(args[2], "k_scale"),
                     &vs = tensor_of(args[3], "v_scale"), &table = tensor_of(args[4], "table");
    auto step = [](const at::Tensor& t, int d) { return t.size(d) > 1 ? t.stride(d) : 0; };  // one entry: no step
    bool alike = k.dim() == 4 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type();
    for (int d = 0; alike && d < 4; ++d) alike = step(k, d) == step(v, d);
    if (!alike) refuse("k and v", "two [pages, heads, page size, dim] tensors of one type and layout are needed");
    if (!k.is_cuda() || k.device() != v.device() || k.device() != ks.device() || k.device() != vs.device() ||
        k.device() != table.device()) {
      refuse("k, v, their scales and table", "have to be on one CUDA device (there is no CPU path)");
    }
    if (k.scalar_type() != at::kFloat8_e4m3fn || (k.size(3) > 1 && k.stride(3) != 1)) {
      refuse("k and v", "float8_e4m3fn with contiguous dims is needed");
    }
    alike = ks.dim() == 3 && ks.sizes() == vs.sizes() && ks.size(0) == k.size(0) && ks.size(1) == k.size(1) &&
            ks.scalar_type() == at::kFloat && vs.scalar_type() == at::kFloat;
    for (int d = 0; alike && d < 3; ++d) alike = step(ks, d) == step(vs, d);
    if (!alike || (ks.size(2) > 1 && ks.stride(2) != 1)) {
      refuse("k_scale and v_scale", "two float32 tensors [pages, heads, blocks of a page] of one layout, blocks contiguous, are needed");
    }
    if (ks.size(2) == 0 || k.size(2) % ks.size(2) != 0) {
      refuse("k_scale and v_scale", "a page is divided into blocks of as many slots each");
    }
    if (table.scalar_type() != at::kInt || table.dim() != 2 || (table.size(1) > 1 && table.stride(1) != 1)) {
      refuse("table", "an int32 tensor [sequences, pages per sequence] is needed");
    }
    for (int64_t size : {k.size(0), k.size(1), k.size(2), table.size(0), table.size(1), table.stride(0)}) {
      if (size > 0x7fffffff) refuse("k, v and table", "sizes below 2^31 are needed");
    }
    Cache8 c{};
    c.index = k.get_device();
    c.pages.k = k.data_ptr();
    c.pages.v = v.data_ptr();
    c.pages.k_scale = static_cast<float*>(ks.data_ptr());
    c.pages.v_scale = static_cast<float*>(vs.data_ptr());
    c.pages.num_pages = static_cast<uint32_t>(k.size(0));
    c.pages.n_kv_heads = static_cast<uint32_t>(k.size(1));
    c.pages.page_size = static_cast<uint32_t>(k.size(2));
    c.pages.head_dim = static_cast<uint32_t>(k.size(3));
    c.pages.block = static_cast<uint32_t>(k.size(2) / ks.size(2));
    c.pages.page_stride = static_cast<uint64_t>(step(k, 0));
    c.pages.head_stride = static_cast<uint64_t>(step(k, 1));
    c.pages.slot_stride = static_cast<uint64_t>(step(k, 2));
    c.pages.scale_page_stride = static_cast<uint64_t>(step(ks, 0));
    c.pages.scale_head_stride = static_cast<uint64_t>(step(ks, 1));
    c.pages.table = static_cast<const int32_t*>(table.data_ptr());
    c.pages.batch = static_cast<uint32_t>(table.size(0));
    c.pages.table_pages = static_cast<uint32_t>(table.size(1));
    c.pages.table_stride = static_cast<uint32_t>(table.size(0) > 1 ? table.stride(0) : table.size(1));
    c.k = k.storage();
    c.v = v.storage();
    c.k_scale = ks.storage();
    c.v_scale = vs.storage();
    c.table = table.storage();
    const unsigned block = c.pages.block;
    PyObject* capsule = hold(c, kCache8Name);
    if (capsule == nullptr) return nullptr;
    PyObject* at = PyLong_FromVoidPtr(&held<Cache8>(capsule, kCache8Name)->pages);
    if (at == nullptr) {
      Py_DECREF(capsule);
      return nullptr;
    }
    return Py_BuildValue("(NNI)", capsule, at, block);
  });
}

// plan8(cache, n_q_heads, tokens, workspace) -> held plan
PyObject* py_plan8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 4, [&]() -> PyObject* {
    Plan8 p{};
    const Cache8* cache = held<Cache8>(args[0], kCache8Name);
    if (cache == nullptr) throw Refused();
    p.cache = *cache;
    p.n_q = count_of(args[1]);
    p.tokens = count_of(args[2]);
    const at::Tensor& workspace = tensor_of(args[3], "workspace");
    p.workspace = workspace.data_ptr();
    p.space = workspace.storage();
    return hold(p, kPlan8Name);
  });
}

// Offsets of a call of `tokens` rows; without them a row is a sequence's.
const int32_t* offsets_of(PyObject* o, const Cache8* c, int64_t tokens) {
  const int64_t batch = c->pages.batch;
  if (o == Py_None && tokens > batch) refuse("offsets", "rows of a sequence each are at most as many as sequences");
  return ints_or_null(o, batch + 1, c->index, "offsets");
}

// append8(cache, q, k, v, rope, positions, lens, offsets, q_norm, k_norm, eps, pairs, q_out, stream)
// -> (cudaError_t, q_out)
PyObject* py_append8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 14, [&]() -> PyObject* {
    const Cache8* c = held<Cache8>(args[0], kCache8Name);
    if (c == nullptr) throw Refused();
    const at::Tensor &q = tensor_of(args[1], "q"), &k = tensor_of(args[2], "k"), &v = tensor_of(args[3], "v");
    if (q.dim() != 3) refuse("q", "a [tokens, heads, dim] tensor is needed");
    const int64_t tokens = q.size(0), heads = q.size(1), dim = c->pages.head_dim, kv = c->pages.n_kv_heads;
    if (tokens > 0x7fffffff || heads > 0xffff) refuse("q", "at most 2^31 - 1 tokens and 65535 heads are taken");
    const at::ScalarType type = q.scalar_type();
    qg_append8 a{};
    a.dtype = dtype_of(q, "q");
    a.tokens = static_cast<uint32_t>(tokens);
    a.n_q_heads = static_cast<uint32_t>(heads);
    a.q_stride = heads_of(q, tokens, heads, dim, type, c->index, "q");
    a.k_stride = heads_of(k, tokens, kv, dim, type, c->index, "k");
    a.v_stride = heads_of(v, tokens, kv, dim, type, c->index, "v");
    a.q = q.data_ptr();
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.q_norm = floats_or_null(args[8], {dim}, c->index, "q_norm");
    a.k_norm = floats_or_null(args[9], {dim}, c->index, "k_norm");
    a.eps = number_of(args[10]);
    if (args[4] != Py_None) {
      const at::Tensor& rope = tensor_of(args[4], "rope");
      if (rope.dim() != 2 || rope.size(0) > 0x7fffffff || rope.size(1) > 0x7fffffff) refuse("rope", "[rows, rot_dim] is needed");
      a.rope = floats_of(rope, {rope.size(0), rope.size(1)}, c->index, "rope");
      a.rope_rows = static_cast<uint32_t>(rope.size(0));
      a.rot_dim = static_cast<uint32_t>(rope.size(1));
    }
    a.pairs = static_cast<int>(count_of(args[11]));
    a.positions = static_cast<const int32_t*>(ints_of(tensor_of(args[5], "positions"), tokens, c->index, "positions"));
    a.lens = static_cast<const int32_t*>(ints_of(tensor_of(args[6], "lens"), c->pages.batch, c->index, "lens"));
    a.offsets = offsets_of(args[7], c, tokens);
    const Call call(c->index, args[13]);
    const at::Tensor q_out = args[12] == Py_None ? at::empty({tokens, heads, dim}, q.options()) : tensor_of(args[12], "q_out");
    a.q_out_stride = heads_of(q_out, tokens, heads, dim, type, c->index, "q_out");
    a.q_out = q_out.data_ptr();
    const cudaError_t e = g_entries.append8(&c->pages, &a, call.stream);
    return Py_BuildValue("(iN)", static_cast<int>(e), THPVariable_Wrap(q_out));
  });
}

// read8(cache, starts, offsets, tokens, dtype, k_out, v_out, stream) -> (cudaError_t, k_out, v_out)
PyObject* py_read8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject* {
    const Cache8* c = held<Cache8>(args[0], kCache8Name);
    if (c == nullptr) throw Refused();
    const int64_t batch = c->pages.batch, dim = c->pages.head_dim, kv = c->pages.n_kv_heads;
    qg_read8 r{};
    r.starts = static_cast<const int32_t*>(ints_of(tensor_of(args[1], "starts"), batch, c->index, "starts"));
    r.offsets = static_cast<const int32_t*>(ints_of(tensor_of(args[2], "offsets"), batch + 1, c->index, "offsets"));
    r.tokens = count_of(args[3]);
    if (r.tokens > 0x7fffffffu) refuse("tokens", "a number of rows below 2^31 is needed");
    const int64_t tokens = r.tokens;
    if (!THPDtype_Check(args[4])) refuse("dtype", "a torch.dtype is needed");
    const at::ScalarType type = reinterpret_cast<THPDtype*>(args[4])->scalar_type;
    r.dtype = dtype_code(type, "dtype");
    const auto options = at::TensorOptions().dtype(type).device(at::kCUDA, static_cast<c10::DeviceIndex>(c->index));
    const Call call(c->index, args[7]);
    const at::Tensor k = args[5] == Py_None ? at::empty({tokens, kv, dim}, options) : tensor_of(args[5], "k_out");
    const at::Tensor v = args[6] == Py_None ? at::empty({tokens, kv, dim}, options) : tensor_of(args[6], "v_out");
    r.k_stride = heads_of(k, tokens, kv, dim, type, c->index, "k_out");
    r.v_stride = heads_of(v, tokens, kv, dim, type, c->index, "v_out");
    r.k_out = k.data_ptr();
    r.v_out = v.data_ptr();
    const cudaError_t e = g_entries.read8(&c->pages, &r, call.stream);
    return Py_BuildValue("(iNN)", static_cast<int>(e), THPVariable_Wrap(k), THPVariable_Wrap(v));
  });
}

// attend8(plan, q, lens, offsets, window, sink, scale, out, lse, return_lse, stream)
// -> (cudaError_t, out, lse or None)
PyObject* py_attend8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 11, [&]() -> PyObject* {
    const Plan8* p = held<Plan8>(args[0], kPlan8Name);
    if (p == nullptr) throw Refused();
    const Cache8* c = &p->cache;
    const at::Tensor& q = tensor_of(args[1], "q");
    if (q.dim() != 3) refuse("q", "a [tokens, heads, dim] tensor is needed");
    const int64_t tokens = q.size(0), heads = p->n_q, dim = c->pages.head_dim;
    if (tokens > p->tokens) refuse("q", "the plan is for at most " + std::to_string(p->tokens) + " tokens");
    const at::ScalarType type = q.scalar_type();
    qg_attn8 a{};
    a.dtype = dtype_of(q, "q");
    a.tokens = static_cast<uint32_t>(tokens);
    a.n_q_heads = p->n_q;
    a.q_stride = heads_of(q, tokens, heads, dim, type, c->index, "q");
    a.q = q.data_ptr();
    a.lens = static_cast<const int32_t*>(ints_of(tensor_of(args[2], "lens"), c->pages.batch, c->index, "lens"));
    a.offsets = offsets_of(args[3], c, tokens);
    a.window = count_of(args[4]);
    if (a.window == 0xffffffffu) refuse("window", "a number of slots is needed, 0 for all");
    a.sink = count_of(args[5]);
    if (a.sink == 0xffffffffu) refuse("sink", "a number of slots is needed");
    a.scale = number_of(args[6]);
    const Call call(c->index, args[10]);
    const at::Tensor out = args[7] == Py_None ? at::empty({tokens, heads, dim}, q.options()) : tensor_of(args[7], "out");
    a.out_stride = heads_of(out, tokens, heads, dim, type, c->index, "out");
    a.out = out.data_ptr();
    at::Tensor lse;
    if (args[8] != Py_None) {
      lse = tensor_of(args[8], "lse");
    } else if (args[9] == Py_True) {
      lse = at::empty({tokens, heads}, q.options().dtype(at::kFloat));
    }
    if (lse.defined()) a.lse = floats_of(lse, {tokens, heads}, c->index, "lse");
    const cudaError_t e = g_entries.attn8(&c->pages, &a, p->workspace, call.stream);
    PyObject* lse_out = Py_None;
    if (lse.defined()) {
      lse_out = THPVariable_Wrap(lse);
    } else {
      Py_INCREF(Py_None);
    }
    return Py_BuildValue("(iNN)", static_cast<int>(e), THPVariable_Wrap(out), lse_out);
  });
}

#define QG_METHOD(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##name)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {QG_METHOD(bind),   QG_METHOD(cache), QG_METHOD(plan), QG_METHOD(append),
                           QG_METHOD(attend), QG_METHOD(evict), QG_METHOD(bind8), QG_METHOD(cache8), QG_METHOD(plan8),
                           QG_METHOD(append8), QG_METHOD(read8), QG_METHOD(attend8), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "qgemv_paged_torch", nullptr, -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit_qgemv_paged_torch() { return PyModule_Create(&g_module); }
