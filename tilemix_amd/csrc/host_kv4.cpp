// The Python calls of the paged 4-bit cache (tilemix_amd/attention/hip/paged_int4.py), each as one
// native call: checks, outputs and workspace, launch.  Unlike the calls of host.cpp they
// have no second path in Python: what they do not take raises here, before anything is launched.
// What depends on shapes and types is checked before the device, so that it is refused
// on a machine without a GPU as well.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>
#include <pybind11/gil.h>

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/TensorSubclassLikeUtils.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include "host_kv4.h"
#include "tilemix_hip.h"

namespace {

struct Library {
  decltype(&tilemix_kv4_store) store = nullptr;
  decltype(&tilemix_kv4_load) load = nullptr;
  decltype(&tilemix_kv4_attn) attn = nullptr;
  decltype(&tilemix_kv4_attn_workspace) workspace = nullptr;
  decltype(&tilemix_kv4_extend) extend = nullptr;
  decltype(&tilemix_kv4_truncate) truncate = nullptr;
  decltype(&tilemix_last_error) last_error = nullptr;
  PyObject* error = nullptr;  // TileMixLibraryError
} g_lib;

constexpr int kGroup = 32;

// ---- arguments --------------------------------------------------------------------

void count_args(Py_ssize_t n, Py_ssize_t wanted, const char* name) {
  TORCH_CHECK_TYPE(n == wanted, name, "() takes ", wanted, " arguments, got ", n);
  TORCH_CHECK(g_lib.store != nullptr, name, "(): the library is not bound");
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a torch.Tensor, got ", Py_TYPE(o)->tp_name);
  const at::Tensor& t = THPVariable_Unpack(o);
  TORCH_CHECK_TYPE(t.defined() && t.layout() == at::kStrided && !t.is_neg() && !at::isTensorSubclassLike(t), name,
                   " must be a plain strided tensor");
  return t;
}

void check_dtype(const at::Tensor& t, at::ScalarType dtype, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == dtype, name, " must be ", dtype, ", got ", t.scalar_type());
}

int64_t integer(PyObject* o, const char* name, int64_t low, int64_t high) {
  PyObject* const index = PyNumber_Index(o);
  if (index == nullptr) throw python_error();
  int overflow = 0;
  const int64_t v = PyLong_AsLongLongAndOverflow(index, &overflow);
  Py_DECREF(index);
  TORCH_CHECK_VALUE(overflow == 0 && v >= low && v <= high, name, " must be in [", low, ", ", high, "]");
  return v;
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}

// fp16: 0, bf16: 1
int value_type(at::ScalarType dtype, const char* name) {
  TORCH_CHECK_TYPE(dtype == at::kHalf || dtype == at::kBFloat16, name, " must be float16 or bfloat16, got ", dtype);
  return dtype == at::kBFloat16 ? 1 : 0;
}

struct Pool {
  const at::Tensor* t[4];  // K codes and parameters, V codes and parameters
  int pages = 0, heads = 0, page_size = 0, head_dim = 0;
  at::Device device() const { return t[0]->device(); }
};

// Arguments a[0 .. 4]: the four arrays and head_dim.
Pool pool(PyObject* const* a) {
  static const char* const names[4] = {"k_codes", "k_params", "v_codes", "v_params"};
  Pool p;
  for (int i = 0; i < 4; ++i) {
    p.t[i] = &tensor(a[i], names[i]);
    check_dtype(*p.t[i], i % 2 == 0 ? at::kByte : at::kHalf, names[i]);
  }
  p.head_dim = static_cast<int>(integer(a[4], "head_dim", 1, 128));
  const int64_t groups = (p.head_dim + kGroup - 1) / kGroup;
  const at::Tensor& codes = *p.t[0];
  TORCH_CHECK_VALUE(codes.dim() == 4 && codes.size(3) == groups * (kGroup / 2) && codes.size(0) >= 1 &&
                        codes.size(0) <= INT32_MAX && codes.size(1) >= 1 && codes.size(1) <= 65535,
                    "k_codes must be [pages, heads, page_size, ", groups * (kGroup / 2), "] for head_dim ", p.head_dim,
                    ", got ", codes.sizes());
  TORCH_CHECK_VALUE(codes.size(2) >= 16 && codes.size(2) % 16 == 0 && codes.size(2) <= (1 << 24),
                    "page_size must be a positive multiple of 16, got ", codes.size(2));
  TORCH_CHECK_VALUE(codes.size(0) * codes.size(1) <= INT32_MAX / codes.size(2), "a cache has fewer than 2^31 rows, got ",
                    codes.sizes());
  p.pages = static_cast<int>(codes.size(0));
  p.heads = static_cast<int>(codes.size(1));
  p.page_size = static_cast<int>(codes.size(2));
  for (int i = 1; i < 4; ++i) {
    const at::Tensor& t = *p.t[i];
    const bool fits = i == 2 ? t.sizes() == codes.sizes()
                             : t.dim() == 5 && t.size(0) == codes.size(0) && t.size(1) == codes.size(1) &&
                                   t.size(2) == codes.size(2) && t.size(3) == groups && t.size(4) == 2;
    TORCH_CHECK_VALUE(fits, names[i], " does not match k_codes ", codes.sizes(), ": ", t.sizes());
  }
  for (int i = 0; i < 4; ++i) {
    TORCH_CHECK_VALUE(p.t[i]->is_contiguous() &&
                          reinterpret_cast<uintptr_t>(p.t[i]->const_data_ptr()) % (i % 2 == 0 ? 16 : 4) == 0,
                      names[i], " must be contiguous and aligned");
    TORCH_CHECK_VALUE(p.t[i]->device() == codes.device(), "the cache's arrays must share one device");
  }
  return p;
}

void check_device(at::Device device, std::initializer_list<const at::Tensor*> tensors) {
  for (const at::Tensor* t : tensors)
    TORCH_CHECK_VALUE(t == nullptr || t->device() == device, "all tensors must be on ", device, ", got ", t->device());
  TORCH_CHECK(device.is_cuda(), "the 4-bit cache runs on the GPU (HIP); got ", device, " tensors");
}

// A table with unit column stride, and what the kernels index it by.
void check_table(const at::Tensor& t, bool written) {
  check_dtype(t, at::kInt, "block_table");
  TORCH_CHECK_VALUE(t.dim() == 2 && t.size(1) <= INT32_MAX, "block_table must be [sequences, columns], got ", t.sizes());
  if (written)
    TORCH_CHECK_VALUE((t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1)),
                      "block_table must have contiguous rows of its own");
}

void check_vector(const at::Tensor& t, at::ScalarType dtype, const char* name, int64_t size) {
  check_dtype(t, dtype, name);
  TORCH_CHECK_VALUE(t.dim() == 1 && (size < 0 || t.size(0) == size), name, " must be a vector",
                    size < 0 ? std::string() : " of " + std::to_string(size), ", got ", t.sizes());
}

// Whether the rows [n0][n1] of t [n0, n1, d] lie apart (token-major or head-major, with any gaps).
bool rows_apart(const at::Tensor& t) {
  const int64_t n0 = t.size(0), n1 = t.size(1), d = t.size(2);
  const int64_t s0 = n0 > 1 ? t.stride(0) : INT64_MAX, s1 = n1 > 1 ? t.stride(1) : INT64_MAX;
  const int64_t low = std::min(s0, s1), high = std::max(s0, s1), n = s0 < s1 ? n0 : n1;
  return (d <= 1 || t.stride(2) == 1) && low >= d && (high == INT64_MAX || high >= (n - 1) * low + d);
}

at::Tensor unit_stride(const at::Tensor& t) {
  return t.dim() == 0 || t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

// A contiguous tensor of its own in the memory of another, `from` bytes in.
at::Tensor part_of(const at::Tensor& room, at::ScalarType type, int64_t from, c10::IntArrayRef sizes) {
  const auto dtype = c10::scalarTypeToTypeMeta(type);
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(room.storage()), room.key_set(), dtype);
  t.unsafeGetTensorImpl()->set_storage_offset(from / static_cast<int64_t>(dtype.itemsize()));
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return t;
}

void* stream_of(at::Device device) { return c10::hip::getCurrentHIPStream(device.index()).stream(); }

void check_status(int status) {
  if (status == 0) return;
  PyErr_Format(g_lib.error, "libtilemix_hip: %s (status %d)", g_lib.last_error(), status);
  throw python_error();
}

void fill(tilemix_kv4_rows_params& p, const Pool& c) {
  p.k_codes = const_cast<void*>(c.t[0]->const_data_ptr());
  p.k_params = const_cast<void*>(c.t[1]->const_data_ptr());
  p.v_codes = const_cast<void*>(c.t[2]->const_data_ptr());
  p.v_params = const_cast<void*>(c.t[3]->const_data_ptr());
  p.pages = c.pages;
  p.page_size = c.page_size;
  p.heads = c.heads;
  p.head_dim = c.head_dim;
}

}  // namespace

// kv4_bind(the addresses of the six entry points and of tilemix_last_error, the error class)
PyObject* kv4_bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 8) {
    PyErr_SetString(PyExc_TypeError, "kv4_bind() takes seven addresses and an exception class");
    return nullptr;
  }
  void* at[7];
  for (int i = 0; i < 7; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (at[i] == nullptr) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null entry point");
      return nullptr;
    }
  }
  g_lib.store = reinterpret_cast<decltype(g_lib.store)>(at[0]);
  g_lib.load = reinterpret_cast<decltype(g_lib.load)>(at[1]);
  g_lib.attn = reinterpret_cast<decltype(g_lib.attn)>(at[2]);
  g_lib.workspace = reinterpret_cast<decltype(g_lib.workspace)>(at[3]);
  g_lib.extend = reinterpret_cast<decltype(g_lib.extend)>(at[4]);
  g_lib.truncate = reinterpret_cast<decltype(g_lib.truncate)>(at[5]);
  g_lib.last_error = reinterpret_cast<decltype(g_lib.last_error)>(at[6]);
  Py_INCREF(args[7]);
  Py_XDECREF(g_lib.error);
  g_lib.error = args[7];
  Py_RETURN_NONE;
}

// The sizes of the structs that these calls pass, as tilemix_params_size numbers them (4, 5, 6).
PyObject* kv4_built_for(PyObject*, PyObject* const*, Py_ssize_t) {
  return Py_BuildValue("(nnn)", static_cast<Py_ssize_t>(sizeof(tilemix_kv4_rows_params)),
                       static_cast<Py_ssize_t>(sizeof(tilemix_kv4_attn_params)),
                       static_cast<Py_ssize_t>(sizeof(tilemix_kv4_tables_params)));
}

// kv4_check(k_codes, k_params, v_codes, v_params, head_dim): raises where they are no cache.
PyObject* kv4_check(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 5, "kv4_check");
  pool(a);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// kv4_store(k_codes, k_params, v_codes, v_params, head_dim, k, v, slots)
PyObject* kv4_store(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 8, "kv4_store");
  const Pool c = pool(a);
  const at::Tensor &k0 = tensor(a[5], "k"), &v0 = tensor(a[6], "v"), &slots0 = tensor(a[7], "slots");
  tilemix_kv4_rows_params p{};
  p.dtype = value_type(k0.scalar_type(), "k");
  check_dtype(v0, k0.scalar_type(), "v");
  TORCH_CHECK_VALUE(k0.dim() == 3 && k0.size(1) == c.heads && k0.size(2) == c.head_dim, "k must be [tokens, ", c.heads,
                    ", ", c.head_dim, "], got ", k0.sizes());
  TORCH_CHECK_VALUE(v0.sizes() == k0.sizes(), "k and v must have one shape, got ", k0.sizes(), " and ", v0.sizes());
  check_vector(slots0, at::kLong, "slots", k0.size(0));
  check_device(c.device(), {&k0, &v0, &slots0});
  if (k0.size(0) == 0) Py_RETURN_NONE;
  const c10::DeviceGuard guard(c.device());
  const at::Tensor k = unit_stride(k0), v = unit_stride(v0), slots = unit_stride(slots0);
  fill(p, c);
  p.k = const_cast<void*>(k.const_data_ptr());
  p.v = const_cast<void*>(v.const_data_ptr());
  p.slots = static_cast<const int64_t*>(slots.const_data_ptr());
  p.stride_k_token = k.stride(0);
  p.stride_k_head = k.stride(1);
  p.stride_v_token = v.stride(0);
  p.stride_v_head = v.stride(1);
  p.tokens = k.size(0);
  void* const stream = stream_of(c.device());
  int status = 0;
  {
    pybind11::gil_scoped_release no_gil;  // a launch may wait for room in the queue
    status = g_lib.store(&p, stream);
  }
  check_status(status);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// kv4_load(k_codes, k_params, v_codes, v_params, head_dim, block_table, cu_seqlens, num_tokens, dtype): (k, v)
PyObject* kv4_load(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 9, "kv4_load");
  const Pool c = pool(a);
  const at::Tensor &table0 = tensor(a[5], "block_table"), &cu0 = tensor(a[6], "cu_seqlens");
  check_table(table0, false);
  check_vector(cu0, at::kInt, "cu_seqlens", table0.size(0) + 1);
  tilemix_kv4_rows_params p{};
  p.tokens = integer(a[7], "num_tokens", 0, INT32_MAX);
  TORCH_CHECK_TYPE(THPDtype_Check(a[8]), "dtype must be a torch.dtype, got ", Py_TYPE(a[8])->tp_name);
  const at::ScalarType dtype = reinterpret_cast<THPDtype*>(a[8])->scalar_type;
  p.dtype = value_type(dtype, "dtype");
  TORCH_CHECK_VALUE(table0.size(0) >= 1 || p.tokens == 0, "num_tokens ", p.tokens, " without a sequence");
  TORCH_CHECK_VALUE(table0.size(0) <= INT32_MAX, "too many sequences");
  check_device(c.device(), {&table0, &cu0});
  const c10::DeviceGuard guard(c.device());
  const at::Tensor table = unit_stride(table0), cu = unit_stride(cu0);
  // Short sequences: one allocation for both (the host's time for the call 0.6 us less).  Large ones may be freed
  // one by one.
  const auto options = at::TensorOptions().device(c.device());
  const int64_t sizes[3] = {p.tokens, c.heads, c.head_dim};
  const int64_t bytes = (p.tokens * c.heads * c.head_dim * 2 + 15) / 16 * 16;
  at::Tensor k, v;
  if (bytes <= 1 << 20) {
    const at::Tensor room = at::empty({2 * bytes}, options.dtype(at::kByte));
    k = part_of(room, dtype, 0, sizes);
    v = part_of(room, dtype, bytes, sizes);
  } else {
    k = at::empty(sizes, options.dtype(dtype));
    v = at::empty(sizes, options.dtype(dtype));
  }
  if (p.tokens > 0) {
    fill(p, c);
    p.k = k.data_ptr();
    p.v = v.data_ptr();
    p.block_table = static_cast<const int32_t*>(table.const_data_ptr());
    p.cu_seqlens = static_cast<const int32_t*>(cu.const_data_ptr());
    p.stride_k_token = p.stride_v_token = int64_t(c.heads) * c.head_dim;
    p.stride_k_head = p.stride_v_head = c.head_dim;
    p.stride_table = table.stride(0);
    p.batch = static_cast<int32_t>(table.size(0));
    p.table_columns = static_cast<int32_t>(table.size(1));
    void* const stream = stream_of(c.device());
    int status = 0;
    {
      pybind11::gil_scoped_release no_gil;
      status = g_lib.load(&p, stream);
    }
    check_status(status);
  }
  PyObject* const rk = THPVariable_Wrap(std::move(k));
  PyObject* const rv = rk == nullptr ? nullptr : THPVariable_Wrap(std::move(v));
  PyObject* const both = rv == nullptr ? nullptr : PyTuple_Pack(2, rk, rv);
  Py_XDECREF(rk);
  Py_XDECREF(rv);
  return both;
  END_HANDLE_TH_ERRORS
}

// kv4_attention(k_codes, k_params, v_codes, v_params, head_dim, q, block_table, seq_lens, cu_seqlens_q | None,
//               max_seqlen_q, max_seqlen_k, causal, sm_scale | None, out | None): out
PyObject* kv4_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 14, "kv4_attention");
  const Pool c = pool(a);
  const at::Tensor &q0 = tensor(a[5], "q"), &table0 = tensor(a[6], "block_table"), &lens0 = tensor(a[7], "seq_lens");
  const at::Tensor* const cu0 = a[8] == Py_None ? nullptr : &tensor(a[8], "cu_seqlens_q");
  const at::Tensor* const out0 = a[13] == Py_None ? nullptr : &tensor(a[13], "out");
  tilemix_kv4_attn_params p{};
  p.dtype = value_type(q0.scalar_type(), "q");
  TORCH_CHECK_VALUE(q0.dim() == 3 && q0.size(2) == c.head_dim, "q must be [tokens, heads, ", c.head_dim, "], got ",
                    q0.sizes());
  TORCH_CHECK_VALUE(q0.size(1) >= 1 && q0.size(1) % c.heads == 0 && q0.size(1) <= INT32_MAX, "q's ", q0.size(1),
                    " heads must be a multiple of the cache's ", c.heads);
  TORCH_CHECK_VALUE(q0.size(0) <= INT32_MAX, "too many queries");
  check_table(table0, false);
  const int64_t batch = table0.size(0);
  check_vector(lens0, at::kInt, "seq_lens", batch);
  p.max_seqlen_q = static_cast<int32_t>(integer(a[9], "max_seqlen_q", 0, INT32_MAX));
  p.max_seqlen_k = static_cast<int32_t>(integer(a[10], "max_seqlen_k", 0, INT32_MAX));
  if (cu0 != nullptr) {
    check_vector(*cu0, at::kInt, "cu_seqlens_q", batch + 1);
  } else {
    TORCH_CHECK_VALUE(q0.size(0) == batch * p.max_seqlen_q, "without cu_seqlens_q every one of the ", batch,
                      " sequences has max_seqlen_q = ", p.max_seqlen_q, " queries, got ", q0.size(0));
  }
  p.causal = truth(a[11]) ? 1 : 0;
  double scale = 1.0 / std::sqrt(static_cast<double>(c.head_dim));
  if (a[12] != Py_None) {
    scale = PyFloat_AsDouble(a[12]);
    if (scale == -1.0 && PyErr_Occurred()) throw python_error();
  }
  TORCH_CHECK_VALUE(std::isfinite(static_cast<float>(scale)), "sm_scale must be finite in 32 bits, got ", scale);
  p.sm_scale = static_cast<float>(scale);
  if (out0 != nullptr) {
    check_dtype(*out0, q0.scalar_type(), "out");
    TORCH_CHECK_VALUE(out0->sizes() == q0.sizes() && rows_apart(*out0), "out must have q's shape ", q0.sizes(),
                      " and contiguous rows that lie apart, got ", out0->sizes(), " with strides ", out0->strides());
    TORCH_CHECK_VALUE(at::get_overlap_status(*out0, q0) != at::MemOverlapStatus::Partial,
                      "out must be q itself or have memory of its own");
  }
  check_device(c.device(), {&q0, &table0, &lens0, cu0, out0});
  const c10::DeviceGuard guard(c.device());
  const at::Tensor q = unit_stride(q0), table = unit_stride(table0), lens = unit_stride(lens0);
  const at::Tensor cu = cu0 == nullptr ? at::Tensor() : unit_stride(*cu0);
  const auto options = at::TensorOptions().device(c.device());
  at::Tensor out = out0 != nullptr ? *out0 : at::empty(q.sizes(), options.dtype(q.scalar_type()));
  p.q = q.const_data_ptr();
  p.out = out.data_ptr();
  p.k_codes = c.t[0]->const_data_ptr();
  p.k_params = c.t[1]->const_data_ptr();
  p.v_codes = c.t[2]->const_data_ptr();
  p.v_params = c.t[3]->const_data_ptr();
  p.block_table = static_cast<const int32_t*>(table.const_data_ptr());
  p.seq_lens = static_cast<const int32_t*>(lens.const_data_ptr());
  p.cu_seqlens_q = cu0 == nullptr ? nullptr : static_cast<const int32_t*>(cu.const_data_ptr());
  p.stride_q_token = q.stride(0);
  p.stride_q_head = q.stride(1);
  p.stride_o_token = out.stride(0);
  p.stride_o_head = out.stride(1);
  p.stride_table = table.stride(0);
  p.tokens_q = q.size(0);
  p.pages = c.pages;
  p.page_size = c.page_size;
  p.heads_q = static_cast<int32_t>(q.size(1));
  p.heads_k = c.heads;
  p.head_dim = c.head_dim;
  TORCH_CHECK_VALUE(batch <= 65535, "at most 65535 sequences in one call, got ", batch);
  p.batch = static_cast<int32_t>(batch);
  p.table_columns = static_cast<int32_t>(table.size(1));
  p.workspace_bytes = g_lib.workspace(&p);
  if (p.workspace_bytes < 0) check_status(TILEMIX_E_INVALID);
  at::Tensor work;
  if (p.workspace_bytes > 0) {
    work = at::empty({p.workspace_bytes}, options.dtype(at::kByte));
    p.workspace = work.data_ptr();
  }
  void* const stream = stream_of(c.device());
  int status = 0;
  {
    pybind11::gil_scoped_release no_gil;
    status = g_lib.attn(&p, stream);
  }
  check_status(status);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

namespace {

// a[0 .. 6]: block_table, seq_lens, free_pages, free_count, ticket, lens, page_size
at::Device tables(PyObject* const* a, tilemix_kv4_tables_params& p, at::Tensor& lens, int64_t tokens = 0) {
  const at::Tensor &table = tensor(a[0], "block_table"), &seq_lens = tensor(a[1], "seq_lens"),
                   &free_pages = tensor(a[2], "free_pages"), &free_count = tensor(a[3], "free_count"),
                   &ticket = tensor(a[4], "ticket"), &lens0 = tensor(a[5], "the new lengths");
  check_table(table, true);
  const int64_t batch = table.size(0);
  TORCH_CHECK_VALUE(batch <= 4096, "at most 4096 sequences, got ", batch);
  check_vector(seq_lens, at::kInt, "seq_lens", batch);
  check_vector(free_pages, at::kInt, "free_pages", -1);
  check_vector(free_count, at::kInt, "free_count", 1);
  check_vector(ticket, at::kInt, "ticket", 1);
  check_vector(lens0, at::kInt, "the new lengths", batch);
  TORCH_CHECK_VALUE(seq_lens.is_contiguous() && free_pages.is_contiguous() && free_pages.size(0) <= INT32_MAX,
                    "seq_lens and free_pages must be contiguous");
  p.page_size = static_cast<int32_t>(integer(a[6], "page_size", 1, 1 << 24));
  TORCH_CHECK_VALUE(batch > 0 || tokens == 0, "num_tokens ", tokens, " without a sequence");
  check_device(table.device(), {&seq_lens, &free_pages, &free_count, &ticket, &lens0});
  lens = unit_stride(lens0);
  p.block_table = static_cast<int32_t*>(table.data_ptr());
  p.seq_lens = static_cast<int32_t*>(seq_lens.data_ptr());
  p.free_pages = static_cast<int32_t*>(free_pages.data_ptr());
  p.free_count = static_cast<int32_t*>(free_count.data_ptr());
  p.ticket = static_cast<int32_t*>(ticket.data_ptr());
  p.stride_table = table.stride(0);
  p.batch = static_cast<int32_t>(batch);
  p.table_columns = static_cast<int32_t>(table.size(1));
  p.free_capacity = static_cast<int32_t>(free_pages.size(0));
  return table.device();
}

}  // namespace

// kv4_extend(block_table, seq_lens, free_pages, free_count, ticket, new_lens, page_size, num_tokens):
// (slots, positions, cu_seqlens, granted)
PyObject* kv4_extend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 8, "kv4_extend");
  tilemix_kv4_tables_params p{};
  at::Tensor lens;
  const int64_t tokens = integer(a[7], "num_tokens", 0, INT32_MAX);
  const at::Device device = tables(a, p, lens, tokens);
  const c10::DeviceGuard guard(device);
  // One allocation for the four: they are small, live as long as each other, and a second one takes the host a
  // microsecond (a step of 64 sequences, extend and truncate: host 10.7 us with four, 9.2 with one).
  const int64_t length[4] = {tokens, tokens, p.batch + 1, p.batch};
  int64_t from[5] = {0};
  for (int i = 0; i < 4; ++i) from[i + 1] = from[i] + (length[i] * (i < 2 ? 8 : 4) + 15) / 16 * 16;
  const auto options = at::TensorOptions().device(device).dtype(at::kByte);
  const at::Tensor room = p.batch > 0 ? at::empty({from[4]}, options) : at::zeros({from[4]}, options);
  at::Tensor out[4];
  for (int i = 0; i < 4; ++i) out[i] = part_of(room, i < 2 ? at::kLong : at::kInt, from[i], length[i]);
  p.lens = static_cast<const int32_t*>(lens.const_data_ptr());
  p.slots = static_cast<int64_t*>(out[0].data_ptr());
  p.positions = static_cast<int64_t*>(out[1].data_ptr());
  p.cu_seqlens = static_cast<int32_t*>(out[2].data_ptr());
  p.granted = static_cast<int32_t*>(out[3].data_ptr());
  p.tokens = tokens;
  void* const stream = stream_of(device);
  int status = 0;
  {
    pybind11::gil_scoped_release no_gil;
    status = g_lib.extend(&p, stream);
  }
  check_status(status);
  PyObject* const result = PyTuple_New(4);
  if (result == nullptr) return nullptr;
  for (int i = 0; i < 4; ++i) {
    PyObject* const o = THPVariable_Wrap(std::move(out[i]));
    if (o == nullptr) {
      Py_DECREF(result);
      return nullptr;
    }
    PyTuple_SET_ITEM(result, i, o);
  }
  return result;
  END_HANDLE_TH_ERRORS
}

// kv4_truncate(block_table, seq_lens, free_pages, free_count, ticket, lens, page_size)
PyObject* kv4_truncate(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 7, "kv4_truncate");
  tilemix_kv4_tables_params p{};
  at::Tensor lens;
  const at::Device device = tables(a, p, lens);
  const c10::DeviceGuard guard(device);
  p.lens = static_cast<const int32_t*>(lens.const_data_ptr());
  void* const stream = stream_of(device);
  int status = 0;
  {
    pybind11::gil_scoped_release no_gil;
    status = g_lib.truncate(&p, stream);
  }
  check_status(status);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
