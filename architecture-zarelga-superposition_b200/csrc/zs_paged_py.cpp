// Python binding of the paged key-value cache operators: checks the tensors, allocates outputs and
// workspaces from torch's allocator and calls the C ABI on the current stream of their device.
//
// A decode step's calls are a few microseconds of kernel time each.  The same checks written in Python
// around ctypes took 17 us a call besides the launches, these take about 2, so this is the one part of the
// package that is bound through CPython and torch's C++ API; the kernels stay in libzs.so behind include/zs.h.
#include <Python.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/torch.h>

#include <cmath>
#include <sstream>
#include <string>

#include "../../include/zs.h"

namespace {

struct Refused {
  std::string why;
};

template <typename... A>
[[noreturn]] void refuse(const A&... a) {
  std::ostringstream s;
  (s << ... << a);
  throw Refused{s.str()};
}

// An error of a module's class, by default the package's, zs_b200._lib.ZsError.
PyObject* raise(const std::string& why, const char* module = "zs_b200._lib", const char* cls = "ZsError") {
  PyObject* m = PyImport_ImportModule(module);
  if (m == nullptr) return nullptr;
  PyObject* e = PyObject_GetAttrString(m, cls);
  Py_DECREF(m);
  if (e == nullptr) return nullptr;
  PyErr_SetString(e, why.c_str());
  Py_DECREF(e);
  return nullptr;
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(name, " must be a tensor");
  return THPVariable_Unpack(o);
}
// nullptr for None.
const at::Tensor* maybe(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }

long long whole(PyObject* o, const char* name) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(name, " must be a whole number");
  }
  return v;
}
double real(PyObject* o, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(name, " must be a number");
  }
  return v;
}

void* ptr(const at::Tensor* t) { return t == nullptr ? nullptr : t->data_ptr(); }
bool misaligned(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0; }

// All on the device of the first, none asking for a gradient or carrying a tangent.
struct Inputs {
  c10::Device device;
  bool grad;
  explicit Inputs(const at::Tensor& first) : device(first.device()), grad(at::GradMode::is_enabled()) {
    if (!device.is_cuda()) refuse("zs ops run only on CUDA tensors (no CPU fallback); got a tensor on ", device);
    look(first);
  }
  void look(const at::Tensor& t) const {
    if (grad && t.requires_grad())
      refuse("the paged operators have no gradient: call them under torch.no_grad() or on detached tensors");
    if (t._fw_grad(0).defined())
      refuse("the paged operators have no derivative: a tensor carries a forward-mode tangent, which would be lost");
  }
  void add(const at::Tensor* t) const {
    if (t == nullptr) return;
    if (!t->is_cuda()) refuse("zs ops run only on CUDA tensors (no CPU fallback); got a tensor on ", t->device());
    if (t->device() != device) refuse("all tensors must be on one device (got ", device, " and ", t->device(), ")");
    look(*t);
  }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }
};

struct Pages {
  int64_t num, heads, page, hd, stride;
  at::ScalarType dtype;
  int code;
  const at::Tensor &k, &v;
  Pages(const at::Tensor& k_, const at::Tensor& v_) : k(k_), v(v_) {
    dtype = k.scalar_type();
    if (k.dim() != 4 || k.sizes() != v.sizes() || v.scalar_type() != dtype)
      refuse("k_pages and v_pages must be [num_pages, Hkv, page, hd] of one shape and dtype (got ", k.sizes(), " ", dtype,
             ", ", v.sizes(), " ", v.scalar_type(), ")");
    num = k.size(0), heads = k.size(1), page = k.size(2), hd = k.size(3);
    if ((dtype != at::kBFloat16 && dtype != at::kHalf) || (page != 16 && page != 32 && page != 64 && page != 128) ||
        (hd != 64 && hd != 128) || num < 1 || heads < 1)
      refuse("the cache holds bf16 or f16 pages of 16, 32, 64 or 128 tokens of head_dim 64 or 128 (got ", dtype, " ",
             k.sizes(), ")");
    code = dtype == at::kHalf ? ZS_F16 : ZS_BF16;
    const int64_t run = page * hd, whole_page = heads * run;
    stride = num == 1 ? whole_page : k.stride(0);
    for (const at::Tensor* t : {&k, &v})
      if (t->stride(3) != 1 || t->stride(2) != hd || (heads > 1 && t->stride(1) != run) ||
          (num > 1 && t->stride(0) != stride) || stride % 8 || stride < whole_page || misaligned(*t))
        refuse("pages must be 16-byte aligned and packed in their last three dimensions, with one page stride that is a "
               "multiple of 8 (got strides ",
               k.strides(), ", ", v.strides(), ")");
  }
};

void int32_list(const char* name, const at::Tensor& t, int64_t want) {
  if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != want || !t.is_contiguous())
    refuse(name, " must be a contiguous int32 [", want, "] (got ", t.scalar_type(), " ", t.sizes(), ")");
}

struct Tables {
  int64_t n, pages, ld;
  Tables(const at::Tensor& table, const at::Tensor& lens, const at::Tensor* cu) {
    if (table.dim() != 2 || table.scalar_type() != at::kInt || table.size(1) < 1)
      refuse("block_table must be int32 [num_seqs, max_pages] (got ", table.scalar_type(), " ", table.sizes(), ")");
    n = table.size(0), pages = table.size(1);
    if ((pages > 1 && table.stride(1) != 1) || (n > 1 && table.stride(0) < pages))
      refuse("block_table rows must be packed and apart (got strides ", table.strides(), ")");
    ld = std::max(table.stride(0), pages);
    if (n >= int64_t(1) << 31 || pages >= int64_t(1) << 31) refuse("block_table is too large (", table.sizes(), ")");
    int32_list("seq_lens", lens, n);
    if (cu != nullptr) int32_list("cu_seqlens", *cu, n + 1);
  }
};

void check(int rc, const char* what) {
  if (rc != ZS_OK) {
    std::ostringstream s;
    s << what << " failed: " << zs_error_string(rc) << " (zs code " << rc;
    if (rc == ZS_ERR_CUDA) s << ", CUDA error " << zs_last_cuda_error();
    s << ")";
    throw Refused{s.str()};
  }
}

at::Tensor workspace(size_t bytes, const c10::Device& dev) {
  return at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(dev));
}

// append(qkvg, k_pages, v_pages, block_table, seq_lens, n_heads, cu_seqlens, q_weight, k_weight, eps, cos, sin)
PyObject* append(PyObject* const* a) {
  const at::Tensor &k = tensor(a[1], "k_pages"), &v = tensor(a[2], "v_pages");
  at::Tensor x = tensor(a[0], "qkvg");
  const at::Tensor &table = tensor(a[3], "block_table"), &lens = tensor(a[4], "seq_lens");
  const int64_t H = whole(a[5], "n_heads");
  const at::Tensor* cu = maybe(a[6], "cu_seqlens");
  const at::Tensor *wq = maybe(a[7], "q_weight"), *wk = maybe(a[8], "k_weight");
  const double eps = real(a[9], "eps");
  const at::Tensor *cos = maybe(a[10], "cos"), *sin = maybe(a[11], "sin");
  const Inputs in(k);
  const c10::cuda::CUDAGuard on(in.device);   // the library makes that device current
  for (const at::Tensor* t : {&v, (const at::Tensor*)&x, &table, &lens, cu, wq, wk, cos, sin}) in.add(t);
  const Pages p(k, v);
  const Tables tab(table, lens, cu);
  const int64_t width = (H + 2 * p.heads) * p.hd;
  if (x.dim() != 2 || x.scalar_type() != p.dtype || H < 1 || H > x.size(1) || H % p.heads || x.size(1) < width)
    refuse("qkvg must be ", p.dtype, " [T, >= (H + 2 Hkv) hd] with H % Hkv == 0 (got ", x.scalar_type(), " ", x.sizes(),
           ", H=", H, ", Hkv=", p.heads, ", hd=", p.hd, ")");
  const int64_t T = x.size(0);
  if (cu == nullptr && T != tab.n)
    refuse("without cu_seqlens each sequence has one row (got ", T, " rows, ", tab.n, " sequences)");
  if ((wq == nullptr) != (wk == nullptr)) refuse("q_weight and k_weight come together");
  at::Tensor gains[2];
  if (wq != nullptr) {
    const at::Tensor* w[2] = {wq, wk};
    for (int i = 0; i < 2; ++i) {
      if (w[i]->scalar_type() != at::kFloat || w[i]->dim() != 1 || w[i]->size(0) != p.hd)
        refuse("norm weights must be f32 [", p.hd, "] (got ", w[i]->scalar_type(), " ", w[i]->sizes(), ")");
      gains[i] = !w[i]->is_contiguous() || misaligned(*w[i]) ? w[i]->detach().clone(at::MemoryFormat::Contiguous) : *w[i];
    }
  }
  if ((cos == nullptr) != (sin == nullptr)) refuse("cos and sin come together");
  int64_t rows = 0, rot = 0, table_ld = 0;
  at::Tensor turn[2];
  if (cos != nullptr) {
    if (cos->dim() != 2 || cos->sizes() != sin->sizes() || cos->scalar_type() != at::kFloat ||
        sin->scalar_type() != at::kFloat || cos->size(1) > p.hd / 2 || cos->size(0) < 1)
      refuse("cos and sin must be f32 [positions, rot <= ", p.hd / 2, "] of one shape (got ", cos->scalar_type(), " ",
             cos->sizes(), ", ", sin->scalar_type(), " ", sin->sizes(), ")");
    rows = cos->size(0), rot = cos->size(1);
    const bool as_is = cos->strides() == sin->strides() && cos->stride(1) == 1 && cos->stride(0) >= rot;
    turn[0] = as_is ? *cos : cos->contiguous();
    turn[1] = as_is ? *sin : sin->contiguous();
    table_ld = as_is ? cos->stride(0) : rot;
  }
  at::Tensor q = at::empty({T, H, p.hd}, k.options());
  if (T == 0 || tab.n == 0) {
    q.zero_();
    return THPVariable_Wrap(q);
  }
  int64_t ld = x.stride(0);
  if (x.stride(1) != 1 || ld % 8 || misaligned(x) || (T > 1 && ld < width)) {
    x = x.narrow(1, 0, width).clone(at::MemoryFormat::Contiguous);
    ld = width;
  }
  check(zs_paged_append(x.data_ptr(), std::max(ld, width), wq ? gains[0].data_ptr<float>() : nullptr,
                        wk ? gains[1].data_ptr<float>() : nullptr, (float)eps, rot ? turn[0].data_ptr<float>() : nullptr,
                        rot ? turn[1].data_ptr<float>() : nullptr, table_ld, rows, (int)rot, k.data_ptr(), v.data_ptr(),
                        p.stride, p.num, table.data_ptr<int>(), tab.ld, (int)tab.pages, lens.data_ptr<int>(),
                        static_cast<const int*>(ptr(cu)), (int)tab.n, T, (int)H, (int)p.heads, (int)p.hd, (int)p.page,
                        q.data_ptr(), p.code, in.stream()),
        "zs_paged_append");
  return THPVariable_Wrap(q);
}

// attention(q, k_pages, v_pages, block_table, seq_lens, cu_seqlens, window, k_sink, gate, scale, return_lse):
// cu_seqlens None is the decode step
PyObject* attention(PyObject* const* a) {
  const at::Tensor &k = tensor(a[1], "k_pages"), &v = tensor(a[2], "v_pages");
  at::Tensor q = tensor(a[0], "q");
  const at::Tensor &table = tensor(a[3], "block_table"), &lens = tensor(a[4], "seq_lens");
  const at::Tensor* cu = maybe(a[5], "cu_seqlens");
  const bool decode = cu == nullptr;
  const at::Tensor *sink_in = maybe(a[7], "k_sink"), *gate_in = maybe(a[8], "gate");
  const Inputs in(k);
  const c10::cuda::CUDAGuard on(in.device);   // the library makes that device current
  for (const at::Tensor* t : {&v, (const at::Tensor*)&q, &table, &lens, cu, sink_in, gate_in}) in.add(t);
  const Pages p(k, v);
  const Tables tab(table, lens, cu);
  if (q.dim() != 3 || q.scalar_type() != p.dtype || q.size(2) != p.hd || q.size(1) < 1 || q.size(1) % p.heads)
    refuse("q must be ", p.dtype, " [T, H, ", p.hd, "] with H % Hkv == 0 (got ", q.scalar_type(), " ", q.sizes(),
           ", Hkv=", p.heads, ")");
  const int64_t T = q.size(0), H = q.size(1);
  if (decode && T != tab.n) refuse("q has one row per sequence (got ", T, " rows, ", tab.n, " sequences)");
  if (!decode && H / p.heads > 128) refuse("at most 128 query heads share a key head (got H=", H, ", Hkv=", p.heads, ")");
  int64_t window = 0;
  if (a[6] != Py_None) {
    window = whole(a[6], "window");
    if (window <= 0 || window >= int64_t(1) << 31) refuse("window must be None or positive (got ", window, ")");
  }
  double scale = 1.0 / std::sqrt((double)p.hd);
  if (a[9] != Py_None) {
    scale = real(a[9], "scale");
    if (!(scale >= 0.0)) refuse("scale must not be negative (got ", scale, ")");
  }
  at::Tensor sink, gate;
  if (sink_in != nullptr) {
    if (sink_in->dim() != 2 || sink_in->size(0) != H || sink_in->size(1) != p.hd || !sink_in->is_floating_point())
      refuse("k_sink must be a floating-point [", H, ", ", p.hd, "] (got ", sink_in->scalar_type(), " ", sink_in->sizes(), ")");
    sink = *sink_in;
    if (sink.scalar_type() != at::kFloat || !sink.is_contiguous() || misaligned(sink))
      sink = sink.detach().to(at::kFloat, false, true, at::MemoryFormat::Contiguous);
  }
  int64_t ldg = 0;
  if (gate_in != nullptr) {
    if (gate_in->dim() != 2 || gate_in->size(0) != T || gate_in->size(1) != H || gate_in->scalar_type() != p.dtype)
      refuse("gate must be ", p.dtype, " [", T, ", ", H, "] (got ", gate_in->scalar_type(), " ", gate_in->sizes(), ")");
    gate = *gate_in;
    if ((H > 1 && gate.stride(1) != 1) || (T > 1 && gate.stride(0) < H)) gate = gate.contiguous();
    ldg = std::max(gate.stride(0), H);
  }
  at::Tensor o = at::empty({T, H, p.hd}, k.options()), lse;
  const int want_lse = PyObject_IsTrue(a[10]);
  if (want_lse < 0) return nullptr;
  if (want_lse) lse = at::empty({T, H}, k.options().dtype(at::kFloat));
  if (T == 0 || tab.n == 0) {
    o.zero_();
    if (want_lse) lse.fill_(-INFINITY);
  } else {
    const int64_t width = H * p.hd;
    int64_t ld = q.stride(0);
    if (q.stride(2) != 1 || (H > 1 && q.stride(1) != p.hd) || ld % 8 || misaligned(q) || (T > 1 && ld < width)) {
      q = q.clone(at::MemoryFormat::Contiguous);
      ld = width;
    }
    ld = std::max(ld, width);
    float* lse_p = want_lse ? lse.data_ptr<float>() : nullptr;
    const float* sink_p = sink.defined() ? sink.data_ptr<float>() : nullptr;
    const void* gate_p = gate.defined() ? gate.data_ptr() : nullptr;
    const int n = (int)tab.n, m = (int)tab.pages, h = (int)H, hk = (int)p.heads, hd = (int)p.hd, pg = (int)p.page;
    if (decode) {
      const size_t bytes = zs_paged_decode_workspace(n, h, hk, hd);
      const at::Tensor ws = workspace(bytes, in.device);
      check(zs_paged_decode_attention(q.data_ptr(), ld, k.data_ptr(), v.data_ptr(), p.stride, p.num, table.data_ptr<int>(),
                                      tab.ld, m, lens.data_ptr<int>(), n, h, hk, hd, pg, (int)window, (float)scale, sink_p,
                                      gate_p, ldg, o.data_ptr(), lse_p, p.code, ws.data_ptr(), bytes, in.stream()),
            "zs_paged_decode_attention");
    } else {
      const size_t bytes = zs_paged_prompt_workspace(T, n, h, hk, hd, m, pg, (int)window);
      const at::Tensor ws = workspace(bytes, in.device);
      check(zs_paged_prompt_attention(q.data_ptr(), ld, k.data_ptr(), v.data_ptr(), p.stride, p.num, table.data_ptr<int>(),
                                      tab.ld, m, lens.data_ptr<int>(), cu->data_ptr<int>(), n, T, h, hk, hd, pg, (int)window,
                                      (float)scale, sink_p, gate_p, ldg, o.data_ptr(), lse_p, p.code, ws.data_ptr(), bytes,
                                      in.stream()),
            "zs_paged_prompt_attention");
    }
  }
  if (!want_lse) return THPVariable_Wrap(o);
  PyObject* r = PyTuple_New(2);
  if (r == nullptr) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(o));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(lse));
  return r;
}

// pages(op, cache, kv, block_table, seq_lens, ref_count, a, b): op 0 extend, 1 fork, 2 free, 3 compact, 4 copy; cache: the
// address of the zs_kv_cache, which holds the addresses of the four tensors; a, b: its request lists (None where the
// operation has none)
PyObject* pages(PyObject* const* a) {
  const long long op = whole(a[0], "op");
  const auto* cache = reinterpret_cast<const zs_kv_cache*>((uintptr_t)whole(a[1], "cache"));
  const at::Tensor& kv = tensor(a[2], "kv");
  const void* held[4] = {cache->kv, cache->block_table, cache->seq_lens, cache->ref_count};
  for (int i = 0; i < 4; ++i)
    if (tensor(a[2 + i], "the cache's tensors").data_ptr() != held[i])
      refuse("the cache's kv, block_table, seq_lens and ref_count stay where it made them: write into them (copy_) "
             "instead of replacing them");
  const at::Tensor* lists[2] = {maybe(a[6], "requests"), maybe(a[7], "requests")};
  int64_t n = 0;
  for (const at::Tensor* t : lists) {
    if (t == nullptr) continue;
    if (t->scalar_type() != at::kInt || t->dim() != 1 || !t->is_contiguous() || t->device() != kv.device())
      refuse("requests are contiguous int32 [n] tensors on ", kv.device(), " (got ", t->scalar_type(), " ", t->sizes(),
             " on ", t->device(), ")");
    n = t->size(0);
  }
  if (lists[0] && lists[1] && lists[0]->size(0) != lists[1]->size(0)) refuse("request lists must have one length");
  if (op != 3 && n == 0) Py_RETURN_NONE;
  const c10::cuda::CUDAGuard on(kv.device());
  void* stream = c10::cuda::getCurrentCUDAStream(kv.get_device()).stream();
  const int* x = static_cast<const int*>(ptr(lists[0]));
  const int* y = static_cast<const int*>(ptr(lists[1]));
  if (op == 2) {
    check(zs_kv_free(cache, x, n, stream), "zs_kv_free");
    Py_RETURN_NONE;
  }
  const size_t bytes = zs_kv_workspace(cache, n);
  const at::Tensor ws = workspace(bytes, kv.device());
  switch (op) {
    case 0: check(zs_kv_extend(cache, x, y, n, ws.data_ptr(), bytes, stream), "zs_kv_extend"); break;
    case 1: check(zs_kv_fork(cache, x, y, n, ws.data_ptr(), bytes, stream), "zs_kv_fork"); break;
    case 3: check(zs_kv_compact(cache, ws.data_ptr(), bytes, stream), "zs_kv_compact"); break;
    case 4: check(zs_kv_copy_pages(cache, x, y, n, ws.data_ptr(), bytes, stream), "zs_kv_copy_pages"); break;
    default: refuse("no such operation");
  }
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject* const*), int N>
PyObject* call(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
    return nullptr;
  }
  try {
    return F(a);
  } catch (const Refused& r) {
    return raise(r.why);
  } catch (const python_error&) {
    return nullptr;                       // already set
  } catch (const c10::OutOfMemoryError& e) {
    return raise(e.what_without_backtrace(), "torch", "OutOfMemoryError");
  } catch (const std::exception& e) {
    return raise(e.what());
  }
}

PyMethodDef methods[] = {
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&call<append, 12>)), METH_FASTCALL, nullptr},
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&call<attention, 11>)), METH_FASTCALL, nullptr},
    {"pages", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&call<pages, 8>)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_paged", "Paged key-value cache operators (see paged.py).", -1, methods,
                          nullptr, nullptr, nullptr, nullptr};

}  // namespace

// abi: the Python and torch that this was compiled against, which paged.py compares before the first call.
PyMODINIT_FUNC PyInit__paged(void) {
  PyObject* m = PyModule_Create(&module_def);
  if (m != nullptr && PyModule_AddStringConstant(m, "abi", ZS_BINDING_ABI) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
