// Python entry points of the paged 4-bit cache (motif_b200/paged.py): argument checks, allocation of
// the outputs and the call of the C ABI in one compiled step.  A decode step's calls are bound by the
// host (each kernel runs for a few microseconds): through ctypes and Python-level checks an attention
// call took 20.3 us, an append 14.6, a gather 12.3 and a reservation 14.3 on the host; here they take
// 7.4, 5.3 (3.5 without the stored values), 4.6 and 5.7, of which the launches themselves are 2 to 5.
#include <cmath>
#include <string>

#include "host.hpp"

namespace {

using namespace mb_host;

constexpr int kUnit = 16;

// A contiguous [n] tensor on dev.
const at::Tensor& vector(const char* name, PyObject* o, int64_t n, c10::Device dev, at::ScalarType type = at::kInt) {
  const at::Tensor& t = on(name, o, dev);
  if (t.scalar_type() != type || t.dim() != 1 || t.size(0) != n || !t.is_contiguous())
    refuse(std::string(name) + " must be a contiguous " + c10::toString(type) + " tensor [" + std::to_string(n) +
           "], got " + kind_of(t));
  return t;
}
const at::Tensor& table(PyObject* o, c10::Device dev, int64_t batch = -1) {
  const at::Tensor& t = on("block_table", o, dev);
  if (t.scalar_type() != at::kInt || t.dim() != 2 || t.stride(1) != 1 || (batch >= 0 && t.size(0) != batch))
    refuse("block_table must be an int32 [B, max_pages] tensor with contiguous rows, got " + kind_of(t));
  return t;
}
const at::Tensor& lengths(PyObject* o) {
  const at::Tensor& t = tensor("lens", o);
  if (!t.is_cuda() || t.dim() != 1) refuse("lens must be a CUDA tensor [B]");
  return t;
}

struct Pool {
  const at::Tensor& t;
  int64_t pages, kv, page_size, dim;
};
Pool pool(PyObject* o) {
  const at::Tensor& t = tensor("pool", o);
  if (!t.is_cuda()) refuse("pool must live on CUDA");
  int64_t dim = 0;
  if (t.dim() == 4)
    for (int64_t d : {32, 64, 128})
      if (motif_b200_kv4_unit_bytes(d) == t.size(3)) dim = d;
  if (t.scalar_type() != at::kByte || !dim || !t.numel() || !t.is_contiguous())
    refuse("pool must be a contiguous uint8 tensor from kv4_pool, got " + kind_of(t));
  return {t, t.size(0), t.size(1), t.size(2) * kUnit, dim};
}

// t with rows that the kernels can read as 16-byte vectors (a copy where they are not).
at::Tensor rows16(const at::Tensor& t) {
  const int64_t step = 16 / t.element_size();
  bool ok = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && t.stride(i) % step == 0;
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// No gradient is dropped without a word: neither a backward one nor a forward-mode tangent.
void no_grad(const at::Tensor& t) {
  if ((t.requires_grad() && at::GradMode::is_enabled()) ||
      (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined()))
    throw Refusal{PyExc_NotImplementedError, "the 4-bit cache is forward-only (no autograd)"};
}

// ------------------------------------------------------------------ the calls
PyObject* reserve(PyObject* const* a) {
  const at::Tensor& lens = lengths(a[0]);
  const c10::Device dev = lens.device();
  const int64_t B = lens.size(0);
  vector("lens", a[0], B, dev);
  const at::Tensor& added = vector("new_lens", a[1], B, dev);
  const at::Tensor& tab = table(a[2], dev, B);
  const at::Tensor& free = on("free_pages", a[3], dev);
  vector("free_pages", a[3], free.numel(), dev);
  const at::Tensor& count = vector("free_count", a[4], 1, dev);
  const int64_t page_size = whole(a[5]), total = whole(a[6]);
  if (total < 0) refuse("total_new must not be negative, got " + std::to_string(total));
  at::Tensor lens_out, count_out, slots;
  if (a[7] != Py_None) lens_out = vector("lens_out", a[7], B, dev);
  if (a[8] != Py_None) count_out = vector("free_count_out", a[8], 1, dev);
  if (a[9] != Py_None) slots = vector("slots", a[9], total, dev);
  {
    const NoGil others;
    const c10::cuda::CUDAGuard guard(dev);
    if (!lens_out.defined()) lens_out = fresh({B}, at::kInt, dev);
    if (!count_out.defined()) count_out = fresh({1}, at::kInt, dev);
    if (!slots.defined()) slots = fresh({total}, at::kInt, dev);
    check("motif_b200_paged_reserve",
          motif_b200_paged_reserve(lens.data_ptr<int>(), added.data_ptr<int>(), tab.data_ptr<int>(), tab.stride(0),
                                   free.data_ptr<int>(), count.data_ptr<int>(), lens_out.data_ptr<int>(),
                                   count_out.data_ptr<int>(), slots.data_ptr<int>(), total, B, tab.size(1),
                                   free.numel(), page_size, stream_of(dev)));
  }
  return tuple({slots, lens_out, count_out});
}

PyObject* release(PyObject* const* a) {
  const at::Tensor& lens = lengths(a[1]);
  const c10::Device dev = lens.device();
  const int64_t B = lens.size(0);
  vector("lens", a[1], B, dev);
  const at::Tensor& done = vector("done", a[0], B, dev, at::kBool);
  const at::Tensor& tab = table(a[2], dev, B);
  const at::Tensor& free = on("free_pages", a[3], dev);
  vector("free_pages", a[3], free.numel(), dev);
  const at::Tensor& count = vector("free_count", a[4], 1, dev);
  const int64_t page_size = whole(a[5]);
  {
    const NoGil others;
    const c10::cuda::CUDAGuard guard(dev);
    check("motif_b200_paged_release",
          motif_b200_paged_release(static_cast<const uint8_t*>(done.data_ptr()), lens.data_ptr<int>(),
                                   tab.data_ptr<int>(), tab.stride(0), free.data_ptr<int>(), count.data_ptr<int>(), B,
                                   tab.size(1), free.numel(), page_size, stream_of(dev)));
  }
  Py_RETURN_NONE;
}

PyObject* append(PyObject* const* a) {
  const Pool p = pool(a[3]);
  const c10::Device dev = p.t.device();
  const at::Tensor &k0 = on("k", a[0], dev), &v0 = on("v", a[1], dev);
  if ((k0.dim() != 3 && k0.dim() != 4) || k0.sizes() != v0.sizes() || k0.size(1) != p.kv || k0.size(-1) != p.dim) {
    const std::string h = std::to_string(p.kv), d = std::to_string(p.dim);
    refuse("k / v must be [N, " + h + ", " + d + "] or [B, " + h + ", T, " + d + "], got " + shape_of(k0) + ", " +
           shape_of(v0));
  }
  if (k0.scalar_type() != v0.scalar_type()) refuse("k / v must share one dtype");
  no_grad(k0);
  no_grad(v0);
  const bool flat = k0.dim() == 3;
  const int64_t B = flat ? 1 : k0.size(0), T = flat ? k0.size(0) : k0.size(2);
  const at::Tensor& slots = vector("slots", a[2], B * T, dev);
  const int dc = dtype_code(k0.scalar_type());
  const int values = PyObject_IsTrue(a[4]);
  if (values < 0) throw Refusal{nullptr, ""};
  at::Tensor ko, vo;
  {
    const NoGil others;
    const c10::cuda::CUDAGuard guard(dev);
    const at::Tensor k = rows16(k0), v = rows16(v0);
    if (values) {
      ko = fresh(k.sizes(), k.scalar_type(), dev);
      vo = fresh(k.sizes(), k.scalar_type(), dev);
    }
    int64_t strides[12] = {0};
    const at::Tensor* ts[4] = {&k, &v, &ko, &vo};
    for (int i = 0; i < (values ? 4 : 2); ++i) {
      strides[3 * i] = flat ? 0 : ts[i]->stride(0);
      strides[3 * i + 1] = ts[i]->stride(1);
      strides[3 * i + 2] = ts[i]->stride(flat ? 0 : 2);
    }
    check("motif_b200_kv4_append",
          motif_b200_kv4_append(k.data_ptr(), v.data_ptr(), slots.data_ptr<int>(), p.t.data_ptr(),
                                values ? ko.data_ptr() : nullptr, values ? vo.data_ptr() : nullptr, strides, B, T, p.kv,
                                p.dim, p.pages, p.page_size, dc, stream_of(dev)));
  }
  if (!values) Py_RETURN_NONE;
  return tuple({ko, vo});
}

PyObject* gather(PyObject* const* a) {
  const Pool p = pool(a[0]);
  const c10::Device dev = p.t.device();
  const at::Tensor& tab = table(a[1], dev);
  const int64_t B = tab.size(0);
  const at::Tensor& lens = vector("lens", a[2], B, dev);
  const int64_t S = whole(a[3]);
  if (S < 0) refuse("max_len must not be negative, got " + std::to_string(S));
  if (!THPDtype_Check(a[4])) refuse("dtype must be a torch.dtype");
  const at::ScalarType type = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
  const int dc = dtype_code(type);
  at::Tensor k, v;
  {
    const NoGil others;
    const c10::cuda::CUDAGuard guard(dev);
    k = fresh({B, p.kv, S, p.dim}, type, dev), v = fresh({B, p.kv, S, p.dim}, type, dev);
    check("motif_b200_kv4_gather",
          motif_b200_kv4_gather(p.t.data_ptr(), tab.data_ptr<int>(), tab.stride(0), lens.data_ptr<int>(), k.data_ptr(),
                                v.data_ptr(), B, p.kv, S, p.dim, p.pages, p.page_size, tab.size(1), dc,
                                stream_of(dev)));
  }
  return tuple({k, v});
}

PyObject* attention(PyObject* const* a) {
  const Pool p = pool(a[1]);
  const c10::Device dev = p.t.device();
  const at::Tensor& q0 = on("q", a[0], dev);
  if (q0.dim() != 4 || q0.size(3) != p.dim)
    refuse("q must be [B, H, T, " + std::to_string(p.dim) + "], got " + shape_of(q0));
  const int64_t B = q0.size(0), H = q0.size(1), T = q0.size(2);
  if (H % p.kv)
    refuse("num_heads " + std::to_string(H) + " must be divisible by num_kv_heads " + std::to_string(p.kv));
  no_grad(q0);
  const int dc = dtype_code(q0.scalar_type());
  const at::Tensor& tab = table(a[2], dev, B);
  const at::Tensor& lens = vector("lens", a[3], B, dev);
  const float* per_head[4];
  const char* names[4] = {"alpha", "beta", "mu", "ssmax"};
  for (int i = 0; i < 4; ++i) {
    const at::Tensor& t = vector(names[i], a[4 + i], H, dev, at::kFloat);
    no_grad(t);
    per_head[i] = t.data_ptr<float>();
  }
  const int* q_lens = a[8] == Py_None ? nullptr : vector("q_lens", a[8], B, dev).data_ptr<int>();
  const double scale = a[9] == Py_None ? 1.0 / std::sqrt((double)p.dim) : number(a[9]), eps = number(a[10]);
  at::Tensor out;
  {
    const NoGil others;
    const c10::cuda::CUDAGuard guard(dev);
    const at::Tensor q = rows16(q0);
    out = fresh(q.sizes(), q.scalar_type(), dev);
    const int64_t bytes = motif_b200_kv4_attention_workspace_bytes(H, p.kv, T, p.dim);
    const c10::DataPtr ws = c10::cuda::CUDACachingAllocator::get()->allocate((size_t)bytes);
    const int64_t strides[6] = {q.stride(0), q.stride(1), q.stride(2), out.stride(0), out.stride(1), out.stride(2)};
    check("motif_b200_kv4_chord_attention",
          motif_b200_kv4_chord_attention(q.data_ptr(), p.t.data_ptr(), tab.data_ptr<int>(), tab.stride(0),
                                         lens.data_ptr<int>(), q_lens, per_head[0], per_head[1], per_head[2],
                                         per_head[3], out.data_ptr(), strides, B, H, p.kv, T, p.dim, p.pages,
                                         p.page_size, tab.size(1), (float)scale, (float)eps, ws.get(), bytes, dc,
                                         stream_of(dev)));
  }
  return wrap(out);
}

PyMethodDef methods[] = {method<reserve, 10>("paged_reserve"), method<release, 6>("paged_release"),
                         method<append, 5>("kv4_append"),      method<gather, 5>("kv4_gather"),
                         method<attention, 11>("kv4_chord_attention"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_host", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__paged_host(void) { return PyModule_Create(&module); }
