// Calls on a paged key-value cache from Python: checks, results and workspace, and the library's one call each, without Python code on the
// way.  Such calls are small: the slots of a step are 3 us of kernel and 4 of host.
#include "ra_host.h"

#include <ATen/EmptyTensor.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/impl/HIPCachingAllocatorMasqueradingAsCUDA.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/ring_attention_hip.h"

namespace {

using at::Tensor;
using namespace ra_host;

struct Library {
  decltype(&ra_page_slots) page_slots;
  decltype(&ra_write_pages) write_pages;
  decltype(&ra_page_means) page_means;
  decltype(&ra_select_pages) select_pages;
  decltype(&ra_select_pages_workspace) select_workspace;
  decltype(&ra_paged_attention) attention;
  decltype(&ra_paged_attention_workspace) attention_workspace;
  decltype(&ra_put_floats) put_floats;
} g_lib;

// init_paged(addresses of the entry points, in the order above)
PyObject* init(PyObject*, PyObject* args) {
  unsigned long long p[8];
  if (!PyArg_ParseTuple(args, "KKKKKKKK", p, p + 1, p + 2, p + 3, p + 4, p + 5, p + 6, p + 7)) return nullptr;
  g_lib = {reinterpret_cast<decltype(&ra_page_slots)>(p[0]),         reinterpret_cast<decltype(&ra_write_pages)>(p[1]),
           reinterpret_cast<decltype(&ra_page_means)>(p[2]),         reinterpret_cast<decltype(&ra_select_pages)>(p[3]),
           reinterpret_cast<decltype(&ra_select_pages_workspace)>(p[4]), reinterpret_cast<decltype(&ra_paged_attention)>(p[5]),
           reinterpret_cast<decltype(&ra_paged_attention_workspace)>(p[6]), reinterpret_cast<decltype(&ra_put_floats)>(p[7])};
  Py_RETURN_NONE;
}

// Memory of the current device and stream, for a call's results and its workspace; without the dispatcher, which takes as long again (a tensor 1.3 us).
c10::Allocator* allocator() { return c10::hip::HIPCachingAllocatorMasqueradingAsCUDA::get(); }
Tensor empty(at::IntArrayRef shape, at::ScalarType dtype) {
  return at::detail::empty_generic(shape, allocator(), c10::DispatchKeySet(c10::DispatchKey::CUDA), dtype, c10::nullopt);
}
// Several small results in one piece of memory, which takes a third of the time; none overlaps another.
struct Results {
  c10::Storage memory;
  int64_t used = 0;
  explicit Results(int64_t bytes) : memory(c10::Storage::use_byte_size_t(), (size_t)bytes, allocator()->allocate((size_t)bytes), allocator(), false) {}
  Tensor take(int64_t n, at::ScalarType dtype) {
    const auto type = c10::scalarTypeToTypeMeta(dtype);
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(memory), c10::DispatchKeySet(c10::DispatchKey::CUDA), type);
    t.unsafeGetTensorImpl()->set_storage_offset(used / (int64_t)type.itemsize());
    t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
    used += n * (int64_t)type.itemsize();
    return t;
  }
};
struct Workspace {
  c10::DataPtr held;
  explicit Workspace(int64_t bytes) {
    if (bytes > 0) held = allocator()->allocate((size_t)bytes);
  }
  void* at() const { return held.get(); }
};

int64_t number_of(PyObject* x, const char* name, int64_t most = INT32_MAX) {
  const int64_t n = THPVariable_Check(x) ? -1 : PyLong_AsLongLong(x);
  if (n == -1 && PyErr_Occurred()) throw python_error();
  TORCH_CHECK_TYPE(!THPVariable_Check(x), name, " must be an int");
  TORCH_CHECK_VALUE(n >= 0 && n <= most, name, " must lie in [0, ", most, "] (got ", n, ")");
  return n;
}

// The call's device: that of its first array, on which all others have to be.
struct Call {
  at::Device device;
  c10::DeviceGuard on;
  explicit Call(const Tensor& t, const char* name) : device(require(t, name)), on(device) {}
  static at::Device require(const Tensor& t, const char* name) {
    TORCH_CHECK(!torch::jit::tracer::isTracing(), "calls on a paged cache cannot be traced");
    TORCH_CHECK(t.is_cuda(), "a paged cache is on the GPU only: ", name, " must live on a HIP device (there is no CPU fallback)");
    return t.device();
  }
  void here(const Tensor& t, const char* name) const {
    TORCH_CHECK_VALUE(t.device() == device, name, " must be on ", device, ", as the other arrays are (it is on ", t.device(), ")");
    TORCH_CHECK_VALUE(t.layout() == at::kStrided, name, " must be a strided tensor");
  }
  void no_grad(const Tensor& t, const char* name) const {
    TORCH_CHECK(!(c10::GradMode::is_enabled() && t.requires_grad()), name, " requires a gradient, and calls on a paged cache have none: use torch.no_grad()");
    TORCH_CHECK(!(c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined()), name,
                " has a tangent of forward-mode differentiation, and calls on a paged cache have no gradient");
  }
};

void changed(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// An int32 array [B] that is read.
Tensor ints(const Call& c, const Tensor& t, const char* name, int64_t B) {
  c.here(t, name);
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == B, name, " must be int32 [", B, "], not ", t.scalar_type(), " ", t.sizes());
  return t.contiguous();
}

// Rows and sizes of a table; page_size and n_pages are the pool's.
ra_page_table table_of(const Call& c, const Tensor& t, int64_t n_pages, int64_t page_size) {
  c.here(t, "block_table");
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 2, "block_table must be int32 [sequences, pages], not ", t.scalar_type(), " ", t.sizes());
  TORCH_CHECK_VALUE(t.size(0) > 0 && t.size(1) > 0, "block_table must have a row and a column at least, not ", t.sizes());
  TORCH_CHECK_VALUE(t.size(1) == 1 || t.stride(1) == 1, "the rows of block_table must be contiguous");
  TORCH_CHECK_VALUE(t.size(0) == 1 || t.stride(0) >= t.size(1), "the rows of block_table must not overlap");
  TORCH_CHECK_VALUE(n_pages > 0 && n_pages <= INT32_MAX && t.size(1) <= INT32_MAX && page_size <= INT32_MAX, "too many pages: ", n_pages, " and a table of ", t.sizes());
  return ra_page_table{t.data_ptr<int32_t>(), t.size(0) == 1 ? t.size(1) : t.stride(0), (int32_t)t.size(1), (int32_t)n_pages, (int32_t)page_size};
}

int64_t stride_of(const Tensor& t, int i) { return t.size(i) == 1 ? 0 : t.stride(i); }
bool aligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

// [pages, page_size, heads, d], in place.
ra_pool pool_of(const Call& c, const Tensor& t, const char* name) {
  c.here(t, name);
  c.no_grad(t, name);
  TORCH_CHECK_VALUE(t.dim() == 4 && (t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf), name,
                    " must be bfloat16 or float16 [pages, page_size, heads, d], not ", t.scalar_type(), " ", t.sizes());
  TORCH_CHECK_VALUE(t.numel() > 0, name, " is empty: ", t.sizes());
  const ra_pool p{t.data_ptr(), stride_of(t, 0), stride_of(t, 1), stride_of(t, 2)};
  TORCH_CHECK_VALUE(t.stride(3) == 1 && aligned(t) && !((p.stride_page | p.stride_token | p.stride_head) & 7), name,
                    " must have a contiguous last dimension, 16-byte alignment and strides of multiples of 8 elements (strides ", t.strides(), ")");
  return p;
}
void check_writable(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(at::has_internal_overlap(t) != at::MemOverlap::Yes, name, " is written to, and elements of it share memory");
}
void check_pair(const Tensor& k, const Tensor& v) {
  TORCH_CHECK_VALUE(k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type(), "k_pages ", k.sizes(), " ", k.scalar_type(), " and v_pages ", v.sizes(), " ",
                    v.scalar_type(), " must be of one shape and type");
}

// [n, heads, d], as the kernels take it: itself or a copy (one that is contiguous, too, where it does not begin on 16 bytes).
Tensor copy_of(const Tensor& t) { return t.clone(at::MemoryFormat::Contiguous); }
Tensor rows(const Tensor& t) {
  const bool ok = t.stride(2) == 1 && aligned(t) && !((stride_of(t, 0) | stride_of(t, 1)) & 7) && stride_of(t, 0) >= 0 && stride_of(t, 1) >= 0 &&
                  t.size(1) * stride_of(t, 1) <= INT32_MAX;
  return ok ? t : copy_of(t);
}

int32_t int32_of(int64_t n, const char* name) {
  TORCH_CHECK_VALUE(n <= INT32_MAX, name, " has 2^31 or more rows");
  return (int32_t)n;
}

// page_slots(block_table, lengths, new_lengths, free_pages, free_state, page_size, num_tokens) -> slots, starts, lengths, free_state
PyObject* page_slots(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 7, "page_slots(block_table, lengths, new_lengths, free_pages, free_state, page_size, num_tokens)");
  const Tensor &table = tensor_of(args[0]), &before = tensor_of(args[1]), &after = tensor_of(args[2]), &ring = tensor_of(args[3]),
               &state = tensor_of(args[4]);
  const int64_t page_size = number_of(args[5], "page_size"), tokens = number_of(args[6], "num_tokens");
  std::vector<Tensor> got;
  {
    pybind11::gil_scoped_release no_gil;  // (allocations may wait for the GPU)
    const Call c(table, "block_table");
    c.here(ring, "free_pages");
    TORCH_CHECK_VALUE(ring.scalar_type() == at::kInt && ring.dim() == 1 && ring.size(0) > 0 && (ring.size(0) == 1 || ring.stride(0) == 1),
                      "free_pages must be int32 [pages], contiguous, not ", ring.scalar_type(), " ", ring.sizes());
    const ra_page_table t = table_of(c, table, ring.size(0), page_size);
    const int64_t B = table.size(0);
    const Tensor x = ints(c, before, "lengths", B), y = ints(c, after, "new_lengths", B), s = ints(c, state, "free_state", 2);
    Results r(8 * tokens + 4 * (2 * B + 3));  // (the widest first)
    got = {r.take(tokens, at::kLong), r.take(B + 1, at::kInt), r.take(B, at::kInt), r.take(2, at::kInt)};
    check("ra_page_slots", g_lib.page_slots(&t, x.data_ptr<int32_t>(), y.data_ptr<int32_t>(), (int32_t)B, ring.data_ptr<int32_t>(), s.data_ptr<int32_t>(),
                                            tokens ? got[0].data_ptr<int64_t>() : nullptr, (int32_t)tokens, got[1].data_ptr<int32_t>(),
                                            got[2].data_ptr<int32_t>(), got[3].data_ptr<int32_t>(), stream(c.device)));
    changed(table);
    changed(ring);
  }
  return tuple_of(std::move(got));
  END_HANDLE_TH_ERRORS
}

// write_pages(k, v, k_pages, v_pages, slots)
PyObject* write_pages(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 5, "write_pages(k, v, k_pages, v_pages, slots)");
  const Tensor &k = tensor_of(args[0]), &v = tensor_of(args[1]), &k_pages = tensor_of(args[2]), &v_pages = tensor_of(args[3]), &slots = tensor_of(args[4]);
  {
    pybind11::gil_scoped_release no_gil;
    const Call c(k_pages, "k_pages");
    const ra_pool kp = pool_of(c, k_pages, "k_pages"), vp = pool_of(c, v_pages, "v_pages");
    check_pair(k_pages, v_pages);
    check_writable(k_pages, "k_pages");
    check_writable(v_pages, "v_pages");
    for (const Tensor* t : {&k, &v}) {
      const char* name = t == &k ? "k" : "v";
      c.here(*t, name);
      c.no_grad(*t, name);
      TORCH_CHECK_VALUE(t->dim() == 3 && t->size(1) == k_pages.size(2) && t->size(2) == k_pages.size(3) && t->sizes() == k.sizes() &&
                            t->scalar_type() == k.scalar_type() && row_dtype(t->scalar_type()) >= 0,
                        "k and v must be [tokens, ", k_pages.size(2), ", ", k_pages.size(3), "] of one of bfloat16, float16 and float32, not ", k.scalar_type(),
                        " ", k.sizes(), " and ", v.scalar_type(), " ", v.sizes());
    }
    c.here(slots, "slots");
    TORCH_CHECK_VALUE(slots.scalar_type() == at::kLong && slots.dim() == 1 && slots.size(0) == k.size(0), "slots must be int64 [", k.size(0), "], not ",
                      slots.scalar_type(), " ", slots.sizes());
    if (k.size(0)) {
      // (a source that lies in a pool itself is read before anything is written)
      auto apart = [&](const Tensor& t) { return t.is_alias_of(k_pages) || t.is_alias_of(v_pages) ? copy_of(t) : rows(t); };
      const Tensor x = apart(k), y = apart(v), s = slots.contiguous();
      check("ra_write_pages", g_lib.write_pages(x.data_ptr(), stride_of(x, 0), stride_of(x, 1), y.data_ptr(), stride_of(y, 0), stride_of(y, 1),
                                                row_dtype(x.scalar_type()), int32_of(x.size(0), "k"), (int32_t)x.size(1), (int32_t)x.size(2), &kp, &vp,
                                                row_dtype(k_pages.scalar_type()), int32_of(k_pages.size(0), "k_pages"), int32_of(k_pages.size(1), "a page"),
                                                s.data_ptr<int64_t>(), stream(c.device)));
      changed(k_pages);
      changed(v_pages);
    }
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// [pages, heads, d] beside a pool of n_pages, in place
void check_means(const Call& c, const Tensor& means, int64_t heads, int64_t d, at::ScalarType type) {
  c.here(means, "means");
  c.no_grad(means, "means");
  TORCH_CHECK_VALUE(means.dim() == 3 && means.size(0) > 0 && means.size(1) == heads && means.size(2) == d && means.scalar_type() == type, "means must be ", type,
                    " [pages, ", heads, ", ", d, "], not ", means.scalar_type(), " ", means.sizes());
  TORCH_CHECK_VALUE(means.stride(2) == 1 && aligned(means) && !((stride_of(means, 0) | stride_of(means, 1)) & 7),
                    "means must have a contiguous last dimension, 16-byte alignment and strides of multiples of 8 elements (strides ", means.strides(), ")");
}

// page_means(k_pages, block_table, lengths, new_lengths, means)
PyObject* page_means(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 5, "page_means(k_pages, block_table, lengths, new_lengths, means)");
  const Tensor &k_pages = tensor_of(args[0]), &table = tensor_of(args[1]), &before = tensor_of(args[2]), &after = tensor_of(args[3]),
               &means = tensor_of(args[4]);
  {
    pybind11::gil_scoped_release no_gil;
    const Call c(k_pages, "k_pages");
    const ra_pool kp = pool_of(c, k_pages, "k_pages");
    const ra_page_table t = table_of(c, table, k_pages.size(0), k_pages.size(1));
    check_means(c, means, k_pages.size(2), k_pages.size(3), k_pages.scalar_type());
    TORCH_CHECK_VALUE(means.size(0) == k_pages.size(0), "means holds ", means.size(0), " pages, k_pages ", k_pages.size(0));
    check_writable(means, "means");
    const Tensor x = ints(c, before, "lengths", table.size(0)), y = ints(c, after, "new_lengths", table.size(0));
    check("ra_page_means", g_lib.page_means(&kp, row_dtype(k_pages.scalar_type()), &t, x.data_ptr<int32_t>(), y.data_ptr<int32_t>(),
                                            int32_of(table.size(0), "block_table"), int32_of(k_pages.size(2), "heads"), int32_of(k_pages.size(3), "d"),
                                            means.data_ptr(), stride_of(means, 0), stride_of(means, 1), stream(c.device)));
    changed(means);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

Tensor queries(const Call& c, const Tensor& q, int64_t B, int64_t heads, int64_t d, at::ScalarType type) {
  c.here(q, "q");
  c.no_grad(q, "q");
  TORCH_CHECK_VALUE(q.dim() == 3 && q.size(0) == B && q.size(1) > 0 && q.size(1) % heads == 0 && q.size(2) == d && q.scalar_type() == type, "q must be ", type,
                    " [", B, ", a multiple of ", heads, ", ", d, "], not ", q.scalar_type(), " ", q.sizes());
  return rows(q);
}

// select_pages(q, means, block_table, lengths, page_size, count, first, last) -> pages
PyObject* select_pages(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 8, "select_pages(q, means, block_table, lengths, page_size, count, first, last)");
  const Tensor &q = tensor_of(args[0]), &means = tensor_of(args[1]), &table = tensor_of(args[2]), &lengths = tensor_of(args[3]);
  const int64_t page_size = number_of(args[4], "page_size"), count = number_of(args[5], "count"), first = number_of(args[6], "first"),
                last = number_of(args[7], "last");
  Tensor pages;
  {
    pybind11::gil_scoped_release no_gil;
    const Call c(q, "q");
    TORCH_CHECK_VALUE(means.dim() == 3 && means.numel() > 0 && (means.scalar_type() == at::kBFloat16 || means.scalar_type() == at::kHalf),
                      "means must be bfloat16 or float16 [pages, heads, d], not ", means.scalar_type(), " ", means.sizes());
    const int64_t H = means.size(1), B = table.dim() ? table.size(0) : 0;
    check_means(c, means, H, means.size(2), means.scalar_type());
    const ra_page_table t = table_of(c, table, means.size(0), page_size);
    const Tensor x = queries(c, q, B, H, means.size(2), means.scalar_type()), y = ints(c, lengths, "lengths", B);
    // (the call's own checks come before anything is allocated)
    TORCH_CHECK_VALUE(count > 0 && first + last <= count, "count must be positive and hold the first and last pages (got ", count, ", ", first, ", ", last, ")");
    TORCH_CHECK_VALUE(B * H * count <= INT32_MAX, "too many pages to choose: ", B, " x ", H, " x ", count);
    pages = empty({B, H, count}, at::kInt);
    const int64_t bytes = t.width > count ? g_lib.select_workspace(&t, (int32_t)B, int32_of(H, "heads")) : 0;
    const Workspace work(bytes);
    check("ra_select_pages", g_lib.select_pages(x.data_ptr(), stride_of(x, 0), stride_of(x, 1), means.data_ptr(), stride_of(means, 0), stride_of(means, 1),
                                                row_dtype(means.scalar_type()), &t, y.data_ptr<int32_t>(), int32_of(B, "block_table"), int32_of(H, "heads"),
                                                int32_of(x.size(1) / H, "q"), int32_of(x.size(2), "d"), (int32_t)count, (int32_t)first, (int32_t)last,
                                                pages.data_ptr<int32_t>(), work.at(), bytes, stream(c.device)));
  }
  return THPVariable_Wrap(std::move(pages));
  END_HANDLE_TH_ERRORS
}

// paged_attention(q, k_pages, v_pages, block_table, lengths, pages or None, slopes or None, window, scale) -> output, logsumexp
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 9, "paged_attention(q, k_pages, v_pages, block_table, lengths, pages, slopes, window, scale)");
  const Tensor &q = tensor_of(args[0]), &k_pages = tensor_of(args[1]), &v_pages = tensor_of(args[2]), &table = tensor_of(args[3]),
               &lengths = tensor_of(args[4]);
  const Tensor chosen = args[5] == Py_None ? Tensor() : tensor_of(args[5]), slopes = args[6] == Py_None ? Tensor() : tensor_of(args[6]);
  const int64_t window = number_of(args[7], "window");
  const double scale = PyFloat_AsDouble(args[8]);
  if (scale == -1.0 && PyErr_Occurred()) throw python_error();
  std::vector<Tensor> got;
  {
    pybind11::gil_scoped_release no_gil;
    const Call c(q, "q");
    ra_paged_params p{};
    p.k = pool_of(c, k_pages, "k_pages");
    p.v = pool_of(c, v_pages, "v_pages");
    check_pair(k_pages, v_pages);
    p.table = table_of(c, table, k_pages.size(0), k_pages.size(1));
    const int64_t B = table.size(0), H = k_pages.size(2), D = k_pages.size(3);
    const at::ScalarType type = k_pages.scalar_type();
    const Tensor x = queries(c, q, B, H, D, type), y = ints(c, lengths, "lengths", B);
    Tensor pages, heads_slopes;
    if (chosen.defined()) {
      c.here(chosen, "pages");
      TORCH_CHECK_VALUE(chosen.scalar_type() == at::kInt && chosen.dim() == 3 && chosen.size(0) == B && chosen.size(1) == H && chosen.size(2) > 0,
                        "pages must be int32 [", B, ", ", H, ", count], not ", chosen.scalar_type(), " ", chosen.sizes());
      pages = chosen.contiguous();
      p.pages = pages.data_ptr<int32_t>();
      p.n_pages_read = int32_of(pages.size(2), "pages");
    }
    if (slopes.defined()) {
      const bool on_host = slopes.is_cpu();
      if (!on_host) c.here(slopes, "slopes");
      c.no_grad(slopes, "slopes");
      TORCH_CHECK_VALUE(slopes.scalar_type() == at::kFloat && slopes.dim() == 1 && slopes.size(0) == x.size(1), "ALiBi slopes must be float32 [", x.size(1),
                        "], one for each query head, not ", slopes.scalar_type(), " ", slopes.sizes());
      heads_slopes = slopes.contiguous();
      if (on_host) {  // (without a copy that waits for the GPU)
        const Tensor there = empty({slopes.size(0)}, at::kFloat);
        check("ra_put_floats", g_lib.put_floats(heads_slopes.data_ptr<float>(), int32_of(slopes.size(0), "slopes"), there.data_ptr<float>(), stream(c.device)));
        heads_slopes = there;
      }
      p.slopes = heads_slopes.data_ptr<float>();
    }
    p.B = int32_of(B, "block_table");
    p.H = int32_of(H, "heads");
    p.group = int32_of(x.size(1) / H, "q");
    p.D = int32_of(D, "d");
    p.dtype = row_dtype(type);
    p.window = (int32_t)window;
    p.sm_scale = (float)scale;
    p.q = x.data_ptr();
    p.q_stride_b = stride_of(x, 0);
    p.q_stride_h = stride_of(x, 1);
    p.lengths = y.data_ptr<int32_t>();
    const int64_t bytes = g_lib.attention_workspace(&p);
    got = {empty({B, x.size(1), D}, type), empty({B, x.size(1)}, at::kFloat)};
    const Workspace work(bytes);
    check("ra_paged_attention", g_lib.attention(&p, got[0].data_ptr(), got[1].data_ptr<float>(), work.at(), bytes, stream(c.device)));
  }
  return tuple_of(std::move(got));
  END_HANDLE_TH_ERRORS
}

PyMethodDef g_methods[] = {{"init_paged", init, METH_VARARGS, nullptr},
                           {"page_slots", (PyCFunction)(void (*)(void))page_slots, METH_FASTCALL, nullptr},
                           {"write_pages", (PyCFunction)(void (*)(void))write_pages, METH_FASTCALL, nullptr},
                           {"page_means", (PyCFunction)(void (*)(void))page_means, METH_FASTCALL, nullptr},
                           {"select_pages", (PyCFunction)(void (*)(void))select_pages, METH_FASTCALL, nullptr},
                           {"paged_attention", (PyCFunction)(void (*)(void))paged_attention, METH_FASTCALL, nullptr},
                           {nullptr, nullptr, 0, nullptr}};

}  // namespace

PyMethodDef* ra_host::paged_methods() { return g_methods; }
