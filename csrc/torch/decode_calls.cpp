// The decoding operators' way from Python to their launchers for calls that have nothing to convert: a decoding step is a few
// microseconds of GPU time, and checks, allocations and a ctypes call written in Python took 13 to 16 us a call, 75 for a forward and
// backward pass through a Python autograd function. What is here checks the same conditions on the tensors themselves and fills in
// the launcher's record. A call that it does not take as it is (another type, a copy needed, an argument to refuse) returns None before
// anything has been allocated or launched, and the Python wrapper goes on: it converts, refuses with its message, or computes in PyTorch.
#include <Python.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/torch.h>
#include <torch/version.h>

#include "decode_calls.h"

namespace {

using at::Tensor;

// ------------------------------------------------------------------------------------------------ the library
void (*set_device)(int) = nullptr;
int (*rotary_fn)(const RotaryCall*, void*) = nullptr;
int (*write_fn)(const KvCall*, void*) = nullptr;
int (*read_fn)(const KvCall*, void*) = nullptr;
int (*attn_fn)(const CacheAttnCall*, void*) = nullptr;
int (*verify_fn)(const VerifyCall*, void*) = nullptr;
long (*attn_ws)(int, int, int, int, int) = nullptr;
const char* (*last_error)() = nullptr;
PyObject* native_dict = nullptr;   // of torsh_b200._native: the device that the library was last told, and the count of launches
PyObject *key_bound = nullptr, *key_count = nullptr, *native_error = nullptr;

// Makes `device` the library's, where the Python side keeps its own note of that. With the GIL held.
bool bind_device(int device) {
  PyObject* bound = PyDict_GetItem(native_dict, key_bound);
  if (bound && PyLong_AsLong(bound) == device) return true;
  PyObject* now = PyLong_FromLong(device);
  const bool ok = now && PyDict_SetItem(native_dict, key_bound, now) == 0;
  if (ok) set_device(device);
  Py_XDECREF(now);
  return ok;
}
void count_launches(int n) {
  PyObject* was = PyDict_GetItem(native_dict, key_count);
  PyObject* now = PyLong_FromLong((was ? PyLong_AsLong(was) : 0) + n);
  if (now) PyDict_SetItem(native_dict, key_count, now);
  Py_XDECREF(now);
}
[[noreturn]] void raise_set() {   // the Python exception that has been set, also through the autograd engine's threads
  python_error e;
  e.persist();
  throw e;
}
template <typename Call>
void launch(int (*fn)(const Call*, void*), const Call& c, int device, const char* name, int kernels) {
  if (!bind_device(device)) {
    raise_set();
  }
  const int rc = fn(&c, (void*)c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream());
  if (rc != 0) {
    PyErr_Format(native_error, "%s failed (rc=%d): %s", name, rc, last_error());
    raise_set();
  }
  count_launches(kernels);
}

// ------------------------------------------------------------------------------------------------ arguments
bool tensor(PyObject* o, Tensor& t) {
  if (!THPVariable_CheckExact(o)) return false;   // subclasses have ways of their own
  t = THPVariable_Unpack(o);
  return true;
}
bool maybe(PyObject* o, Tensor& t) { return o == Py_None || tensor(o, t); }
bool on(const Tensor& t, int device) { return t.is_cuda() && t.get_device() == device; }
bool plain_dense(const Tensor& t) { return t.layout() == at::kStrided && t.has_storage() && !t.is_neg() && !t.is_conj(); }
// A CUDA tensor of the current device, of a kind that kernels read.
bool here(const Tensor& t, int device) { return on(t, device) && plain_dense(t); }
bool ints(const Tensor& t, int64_t n, int device) {
  return here(t, device) && t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous();
}
bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool rows16(const Tensor& t) {   // [., ., ., D]: every row starts on 16 bytes, and a sequence's rows are not too far apart for 32 bits
  const int64_t n = 16 / t.element_size();
  return t.stride(1) <= 0x7fffffff && t.stride(2) <= 0x7fffffff && t.stride(3) == 1 && aligned(t.const_data_ptr()) && t.stride(0) % n == 0 && t.stride(1) % n == 0 && t.stride(2) % n == 0;
}
int kind_of(at::ScalarType t) { return t == at::kBFloat16 ? 0 : t == at::kChar ? 1 : t == at::kFloat8_e4m3fn ? 2 : -1; }
int row_type(at::ScalarType t) { return t == at::kBFloat16 ? 0 : t == at::kFloat ? 1 : -1; }

// Pages, scales and table that the kernels take as they are.
bool pages_ok(const Tensor& kp, const Tensor& vp, const Tensor& ks, const Tensor& vs, const Tensor& table, int device, int64_t B) {
  if (!here(kp, device) || !here(vp, device) || kp.dim() != 4 || vp.sizes() != kp.sizes() || vp.scalar_type() != kp.scalar_type()) return false;
  const int kind = kind_of(kp.scalar_type());
  const int64_t D = kp.size(3), page = kp.size(2);
  if (kind < 0 || (D != 64 && D != 128) || page <= 0 || page % 16 || !kp.is_contiguous() || !vp.is_contiguous() || !aligned(kp.const_data_ptr()) || !aligned(vp.const_data_ptr()))
    return false;
  for (const Tensor* s : {&ks, &vs}) {
    if (s->defined() != (kind != 0)) return false;
    if (s->defined() && (!here(*s, device) || s->scalar_type() != at::kFloat || s->sizes() != kp.sizes().slice(0, 3) || !s->is_contiguous() || !aligned(s->const_data_ptr())))
      return false;
  }
  // an empty pool or table holds nothing: the formulas in PyTorch say so
  return here(table, device) && kp.numel() > 0 && table.numel() > 0 && table.dim() == 2 && table.size(0) == B && table.scalar_type() == at::kInt && (table.stride(1) == 1 || table.size(1) <= 1);
}
template <typename T>
T* ptr(const Tensor& t) { return t.defined() ? (T*)t.const_data_ptr() : nullptr; }

// Forward-mode derivatives: a tensor that carries a tangent looks like any other, and the kernels would drop it.
bool dual(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad() && at::GradMode::is_enabled(); }
int current() { return c10::cuda::current_device(); }
PyObject* pair(const Tensor& a, const Tensor& b) {
  PyObject* x = THPVariable_Wrap(a);
  PyObject* y = b.defined() ? THPVariable_Wrap(b) : Py_NewRef(Py_None);
  PyObject* r = x && y ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x);
  Py_XDECREF(y);
  return r;
}

// ------------------------------------------------------------------------------------------------ rotary
// One stride over all leading dimensions, columns contiguous; a copy where that is not so.
Tensor flat(const Tensor& x, int64_t& ld, int64_t& lh) {
  if (x.dim() == 4 && x.stride(3) == 1 && (x.size(0) == 1 || x.stride(0) == x.size(1) * x.stride(1))) {
    ld = x.stride(1), lh = x.stride(2);
    return x;
  }
  if (x.dim() == 3 && x.stride(2) == 1) {
    ld = x.stride(0), lh = x.stride(1);
    return x;
  }
  lh = x.size(-1), ld = x.size(-2) * lh;
  return x.contiguous();
}
std::pair<Tensor, Tensor> turn(const Tensor& q, const Tensor& k, const Tensor& pos, const Tensor& freqs, bool interleaved, double magnitude, bool inverse) {
  RotaryCall c{};
  int64_t ld = 0, lh = 0;
  const Tensor qc = flat(q, ld, lh);
  c.ldq = ld, c.lhq = lh;
  Tensor yq = at::empty(q.sizes(), q.options()), kc, yk;
  c.q = qc.const_data_ptr(), c.yq = yq.mutable_data_ptr();
  c.tokens = pos.numel(), c.hq = q.size(-2), c.D = q.size(-1), c.R = 2 * freqs.numel();
  if (k.defined()) {
    kc = flat(k, ld, lh);
    c.ldk = ld, c.lhk = lh, c.hk = k.size(-2);
    yk = at::empty(k.sizes(), k.options());
    c.k = kc.const_data_ptr(), c.yk = yk.mutable_data_ptr();
  }
  c.pos = pos.const_data_ptr<int64_t>(), c.freqs = freqs.const_data_ptr<double>();
  c.half = !interleaved, c.inverse = inverse, c.dtype = row_type(q.scalar_type()), c.magnitude = magnitude;
  launch(rotary_fn, c, q.get_device(), "tb_rotary", 1);
  return {yq, yk};
}
// Gradients that the kernel does not read (batched ones have no memory of their own, dual ones a tangent): the formula in PyTorch. With the GIL held.
Tensor turn_plain(const Tensor& x, const Tensor& pos, const Tensor& freqs, bool interleaved, double magnitude, bool inverse) {
  struct Held {
    PyObject* p;
    Held(PyObject* p) : p(p) {
      if (!p) raise_set();
    }
    ~Held() { Py_DECREF(p); }
  };
  const Held module(PyImport_ImportModule("torsh_b200.ops.rotary")), px(THPVariable_Wrap(x)), pp(THPVariable_Wrap(pos)), pf(THPVariable_Wrap(freqs));
  const Held y(PyObject_CallMethod(module.p, "_rotary_plain", "OOOOdO", px.p, pp.p, pf.p, interleaved ? Py_True : Py_False, magnitude, inverse ? Py_True : Py_False));
  return THPVariable_Unpack(y.p);
}
struct RotaryFn : public torch::autograd::Function<RotaryFn> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, Tensor q, std::optional<Tensor> k, Tensor pos, Tensor freqs, bool interleaved, double magnitude, bool inverse) {
    ctx->save_for_backward({pos, freqs});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["magnitude"] = magnitude;
    ctx->saved_data["inverse"] = inverse;
    auto y = turn(q, k ? *k : Tensor(), pos, freqs, interleaved, magnitude, inverse);
    if (!k) return {y.first};
    return {y.first, y.second};
  }
  // a rotation's gradient is the rotation back, with the same factor; differentiable again
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list dy) {
    const auto saved = ctx->get_saved_variables();
    const bool interleaved = ctx->saved_data["interleaved"].toBool(), inverse = ctx->saved_data["inverse"].toBool();
    const double magnitude = ctx->saved_data["magnitude"].toDouble();
    const PyGILState_STATE gil = PyGILState_Ensure();   // the engine's threads run without it; the launch keeps its notes in Python
    struct Release {
      PyGILState_STATE s;
      ~Release() { PyGILState_Release(s); }
    } release{gil};
    const std::optional<Tensor> dk = dy.size() > 1 ? std::optional<Tensor>(dy[1]) : std::nullopt;
    torch::autograd::variable_list d;
    if (!plain_dense(dy[0]) || dual(dy[0]) || (dk && (!plain_dense(*dk) || dual(*dk)))) {
      for (const Tensor& x : dy) d.push_back(turn_plain(x, saved[0], saved[1], interleaved, magnitude, !inverse));
    } else if (at::GradMode::is_enabled()) {
      d = RotaryFn::apply(dy[0], dk, saved[0], saved[1], interleaved, magnitude, !inverse);
    } else {
      auto y = turn(dy[0], dk ? *dk : Tensor(), saved[0], saved[1], interleaved, magnitude, !inverse);
      d = {y.first, y.second};
    }
    return {d[0], d.size() > 1 ? d[1] : Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// rotary(q, k | None, positions, freqs, interleaved, magnitude)
PyObject* py_rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor q, k, pos, freqs;
  if (n != 6 || !tensor(args[0], q) || !maybe(args[1], k) || !tensor(args[2], pos) || !tensor(args[3], freqs)) Py_RETURN_NONE;
  const int device = current();
  const int64_t dims = q.dim();
  if (!here(q, device) || !here(pos, device) || !here(freqs, device) || dims < 2 || row_type(q.scalar_type()) < 0) Py_RETURN_NONE;
  if (pos.scalar_type() != at::kLong || !pos.is_contiguous() || pos.sizes() != q.sizes().slice(0, dims - 2)) Py_RETURN_NONE;
  if (freqs.scalar_type() != at::kDouble || freqs.dim() != 1 || !freqs.is_contiguous() || 2 * freqs.numel() > std::min<int64_t>(q.size(-1), 512)) Py_RETURN_NONE;
  if (k.defined() && (!here(k, device) || k.scalar_type() != q.scalar_type() || k.dim() != dims || k.size(-1) != q.size(-1) || k.sizes().slice(0, dims - 2) != q.sizes().slice(0, dims - 2)))
    Py_RETURN_NONE;
  if (dual(q) || dual(k) || dual(freqs) || wants_grad(freqs)) Py_RETURN_NONE;   // frequencies that learn: the kernel has no gradient for them
  const int interleaved = PyObject_IsTrue(args[4]);
  const double magnitude = PyFloat_AsDouble(args[5]);
  if (interleaved < 0 || (magnitude == -1.0 && PyErr_Occurred())) return nullptr;
  if (wants_grad(q) || wants_grad(k)) {
    const auto y = RotaryFn::apply(q, k.defined() ? std::optional<Tensor>(k) : std::nullopt, pos, freqs, interleaved != 0, magnitude, false);
    return pair(y[0], y.size() > 1 ? y[1] : Tensor());
  }
  const auto y = turn(q, k, pos, freqs, interleaved != 0, magnitude, false);
  return pair(y.first, y.second);
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------------------------ cache
void fill(KvCall& c, const Tensor& kp, const Tensor& vp, const Tensor& ks, const Tensor& vs, const Tensor& table) {
  c.pages[0] = ptr<void>(kp), c.pages[1] = ptr<void>(vp), c.scales[0] = ptr<float>(ks), c.scales[1] = ptr<float>(vs);
  c.table = ptr<int>(table), c.table_ld = table.stride(0);
  c.page = kp.size(2), c.pages_per_seq = table.size(1), c.num_pages = kp.size(0), c.kind = kind_of(kp.scalar_type());
}

// kv_write(k, v, k_pages, v_pages, page_table, start, counts | None, k_scales | None, v_scales | None) -> True
PyObject* py_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor k, v, kp, vp, table, start, counts, ks, vs;
  if (n != 9 || !tensor(args[0], k) || !tensor(args[1], v) || !tensor(args[2], kp) || !tensor(args[3], vp) || !tensor(args[4], table) || !tensor(args[5], start) ||
      !maybe(args[6], counts) || !maybe(args[7], ks) || !maybe(args[8], vs))
    Py_RETURN_NONE;
  const int device = current();
  if (!here(k, device) || !here(v, device) || k.dim() != 4 || v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type() || row_type(k.scalar_type()) < 0) Py_RETURN_NONE;
  const int64_t B = k.size(0);
  if (!pages_ok(kp, vp, ks, vs, table, device, B) || kp.size(1) != k.size(2) || kp.size(3) != k.size(3) || !rows16(k) || !rows16(v)) Py_RETURN_NONE;
  if (!ints(start, B, device) || (counts.defined() && !ints(counts, B, device)) || wants_grad(k) || wants_grad(v) || dual(k) || dual(v)) Py_RETURN_NONE;
  if (k.numel() == 0) Py_RETURN_TRUE;
  KvCall c{};
  const Tensor* x[2] = {&k, &v};
  for (int z = 0; z < 2; ++z) {
    c.x[z] = ptr<void>(*x[z]);
    for (int i = 0; i < 3; ++i) c.strides[3 * z + i] = x[z]->stride(i);
  }
  fill(c, kp, vp, ks, vs, table);
  c.start = ptr<int>(start), c.counts = ptr<int>(counts);
  c.B = B, c.T = k.size(1), c.H = k.size(2), c.D = k.size(3), c.dtype = row_type(k.scalar_type());
  launch(write_fn, c, device, "tb_kv_write", 1);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// kv_read(k_pages, v_pages, page_table, lengths, max_len, begin | None, k_scales | None, v_scales | None, fp32) -> (k, v)
PyObject* py_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor kp, vp, table, lengths, begin, ks, vs;
  if (n != 9 || !tensor(args[0], kp) || !tensor(args[1], vp) || !tensor(args[2], table) || !tensor(args[3], lengths) || !maybe(args[5], begin) || !maybe(args[6], ks) ||
      !maybe(args[7], vs) || !PyLong_Check(args[4]))
    Py_RETURN_NONE;
  const int device = current();
  const int64_t most = PyLong_AsLongLong(args[4]);
  if (most == -1 && PyErr_Occurred()) return nullptr;
  if (table.dim() != 2 || most < 0 || most > 0x7fffffff) Py_RETURN_NONE;
  const int64_t B = table.size(0);
  if (!pages_ok(kp, vp, ks, vs, table, device, B) || !ints(lengths, B, device) || (begin.defined() && !ints(begin, B, device))) Py_RETURN_NONE;
  if (dual(kp) || dual(vp) || dual(ks) || dual(vs)) Py_RETURN_NONE;
  const bool wide = PyObject_IsTrue(args[8]) == 1;
  const auto options = kp.options().dtype(wide ? at::kFloat : at::kBFloat16);
  Tensor k = at::empty({B, most, kp.size(1), kp.size(3)}, options), v = at::empty({B, most, kp.size(1), kp.size(3)}, options);
  if (k.numel()) {
    KvCall c{};
    c.x[0] = k.mutable_data_ptr(), c.x[1] = v.mutable_data_ptr();
    fill(c, kp, vp, ks, vs, table);
    c.start = ptr<int>(begin), c.counts = ptr<int>(lengths);
    c.B = B, c.T = most, c.H = kp.size(1), c.D = kp.size(3), c.dtype = wide;
    launch(read_fn, c, device, "tb_kv_read", 1);
  }
  return pair(k, v);
  END_HANDLE_TH_ERRORS
}

// kv_attention(q, k_pages, v_pages, page_table, start, tree_mask | None, counts | None, k_scales | None, v_scales | None, scale | None,
//              max_len | None, address of the status word) -> out
PyObject* py_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor q, kp, vp, table, start, mask, counts, ks, vs;
  if (n != 12 || !tensor(args[0], q) || !tensor(args[1], kp) || !tensor(args[2], vp) || !tensor(args[3], table) || !tensor(args[4], start) || !maybe(args[5], mask) ||
      !maybe(args[6], counts) || !maybe(args[7], ks) || !maybe(args[8], vs))
    Py_RETURN_NONE;
  const int device = current();
  if (!here(q, device) || q.dim() != 4 || q.scalar_type() != at::kBFloat16) Py_RETURN_NONE;
  const int64_t B = q.size(0), T = q.size(1), Hq = q.size(2), D = q.size(3);
  if (!pages_ok(kp, vp, ks, vs, table, device, B) || kp.size(3) != D || kp.size(1) == 0 || Hq % kp.size(1) || !rows16(q)) Py_RETURN_NONE;
  if (!ints(start, B, device) || (counts.defined() && !ints(counts, B, device)) || wants_grad(q)) Py_RETURN_NONE;
  if (dual(q) || dual(kp) || dual(vp) || dual(ks) || dual(vs)) Py_RETURN_NONE;
  CacheAttnCall c{};
  if (mask.defined()) {
    const int64_t m = mask.dim();
    if (!here(mask, device) || mask.scalar_type() != at::kBool || (m != 2 && m != 3) || mask.size(m - 1) != T || mask.size(m - 2) != T || (m == 3 && mask.size(0) != B) ||
        mask.stride(m - 1) != 1)
      Py_RETURN_NONE;
    c.mask = ptr<uint8_t>(mask), c.mask_t = mask.stride(m - 2), c.mask_b = m == 3 ? mask.stride(0) : 0;
  }
  c.scale = 1.0 / std::sqrt((double)D);
  if (args[9] != Py_None) {
    c.scale = PyFloat_AsDouble(args[9]);
    if (c.scale == -1.0 && PyErr_Occurred()) return nullptr;
    if (!(c.scale >= 0.0 && c.scale < INFINITY)) Py_RETURN_NONE;
  }
  c.max_len = 0x7fff0000;
  if (args[10] != Py_None) {
    const int64_t most = PyLong_AsLongLong(args[10]);
    if (most == -1 && PyErr_Occurred()) return nullptr;
    if (most < 0) Py_RETURN_NONE;
    c.max_len = std::min<int64_t>(most, c.max_len);
  }
  c.status = (int*)PyLong_AsVoidPtr(args[11]);
  if (!c.status && PyErr_Occurred()) return nullptr;
  if (B > 0x7fffffff || T > 0x7fffffff || Hq > 0x7fffffff || !bind_device(device)) return PyErr_Occurred() ? nullptr : Py_NewRef(Py_None);
  Tensor out = at::empty(q.sizes(), q.options());
  if (out.numel() == 0) return THPVariable_Wrap(out);
  // of this call alone: calls on several streams, or in several captured graphs, never share it
  Tensor ws = at::empty({attn_ws((int)B, (int)T, (int)Hq, (int)kp.size(1), (int)D)}, q.options().dtype(at::kByte));
  c.q = ptr<void>(q), c.qb = q.stride(0), c.qt = q.stride(1), c.qh = q.stride(2);
  c.k_pages = ptr<void>(kp), c.v_pages = ptr<void>(vp), c.k_scales = ptr<float>(ks), c.v_scales = ptr<float>(vs);
  c.table = ptr<int>(table), c.table_ld = table.stride(0), c.start = ptr<int>(start), c.counts = ptr<int>(counts);
  c.out = out.mutable_data_ptr(), c.ws = ws.mutable_data_ptr();
  c.B = B, c.T = T, c.Hq = Hq, c.Hkv = kp.size(1), c.D = D, c.page = kp.size(2), c.pages_per_seq = table.size(1), c.num_pages = kp.size(0);
  c.kind = kind_of(kp.scalar_type());
  launch(attn_fn, c, device, "tb_cache_attention", 0);
  count_launches((int)c.kernels);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------------------------ verification
// verify(probs, tokens, uniforms, draft_probs | None, parents | None, counts | None) -> (accepted, path, next token)
PyObject* py_verify(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor probs, tokens, uniforms, draft, parents, counts;
  if (n != 6 || !tensor(args[0], probs) || !tensor(args[1], tokens) || !tensor(args[2], uniforms) || !maybe(args[3], draft) || !maybe(args[4], parents) || !maybe(args[5], counts))
    Py_RETURN_NONE;
  const int device = current();
  if (!here(probs, device) || probs.dim() != 3 || row_type(probs.scalar_type()) < 0 || probs.stride(2) != 1) Py_RETURN_NONE;
  const int64_t B = probs.size(0), T = probs.size(1), V = probs.size(2);
  if (T < 1 || T > 1024 || V < 1 || V > (1 << 22)) Py_RETURN_NONE;
  for (const Tensor* t : {&tokens, &uniforms})
    if (!here(*t, device) || t->dim() != 2 || t->size(0) != B || t->size(1) != T || !t->is_contiguous()) Py_RETURN_NONE;
  if (tokens.scalar_type() != at::kLong || uniforms.scalar_type() != at::kFloat) Py_RETURN_NONE;
  VerifyCall c{};
  if (draft.defined()) {
    if (parents.defined() || !here(draft, device) || draft.dim() != 3 || draft.size(0) != B || draft.size(1) != T - 1 || draft.size(2) != V || draft.scalar_type() != probs.scalar_type() ||
        draft.stride(2) != 1)
      Py_RETURN_NONE;
    if (T > 1) c.draft = ptr<void>(draft), c.db = draft.stride(0), c.dt = draft.stride(1);
  }
  if (parents.defined()) {
    const int64_t m = parents.dim();
    if (!here(parents, device) || parents.scalar_type() != at::kLong || !parents.is_contiguous() || (m != 1 && m != 2) || parents.size(m - 1) != T || (m == 2 && parents.size(0) != B))
      Py_RETURN_NONE;
    c.parents = ptr<long>(parents), c.parents_ld = m == 2 ? T : 0;
  }
  if (counts.defined() && !ints(counts, B, device)) Py_RETURN_NONE;
  Tensor out = at::empty({B * (T + 2)}, tokens.options());
  c.probs = ptr<void>(probs), c.pb = probs.stride(0), c.pt = probs.stride(1);
  c.tokens = ptr<long>(tokens), c.uniforms = ptr<float>(uniforms), c.counts = ptr<int>(counts), c.out = (long*)out.mutable_data_ptr();
  c.B = B, c.T = T, c.V = V, c.dtype = row_type(probs.scalar_type());
  launch(verify_fn, c, device, "tb_verify_draft", 1);
  PyObject *a = THPVariable_Wrap(out.as_strided({B}, {1}, 0)), *b = THPVariable_Wrap(out.as_strided({B, T}, {T, 1}, 2 * B)), *d = THPVariable_Wrap(out.as_strided({B}, {1}, B));
  PyObject* r = a && b && d ? PyTuple_Pack(3, a, b, d) : nullptr;
  Py_XDECREF(a);
  Py_XDECREF(b);
  Py_XDECREF(d);
  return r;
  END_HANDLE_TH_ERRORS
}

// bind(module torsh_b200._native, addresses of: tb_set_device, tb_last_error, tb_rotary, tb_kv_write, tb_kv_read, tb_cache_attention,
//      tb_cache_attention_workspace, tb_verify_draft, tb_decode_layout)
PyObject* py_bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  constexpr int ADDRESSES = 9;
  if (n != 1 + ADDRESSES || !PyModule_Check(args[0])) {
    PyErr_SetString(PyExc_TypeError, "bind: a module and nine addresses");
    return nullptr;
  }
  void* at[ADDRESSES];
  for (int i = 0; i < ADDRESSES; ++i)
    if (!(at[i] = PyLong_AsVoidPtr(args[i + 1]))) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "bind: null address");
  PyObject* dict = PyModule_GetDict(args[0]);
  PyObject* error = PyDict_GetItemString(dict, "NativeError");
  if (!error) return PyErr_Format(PyExc_ValueError, "bind: no NativeError");
  if (((uint64_t (*)())at[8])() != TB_DECODE_LAYOUT)
    return PyErr_Format(error, "_decode_calls.so and libtorsh_b200_cuda.so have been built with different records: run `python -m torsh_b200._build`");
  key_bound = PyUnicode_InternFromString("_bound_device");
  key_count = PyUnicode_InternFromString("launch_count");
  native_error = Py_NewRef(error);
  native_dict = Py_NewRef(dict);
  set_device = (void (*)(int))at[0];
  last_error = (const char* (*)())at[1];
  rotary_fn = (int (*)(const RotaryCall*, void*))at[2];
  write_fn = (int (*)(const KvCall*, void*))at[3];
  read_fn = (int (*)(const KvCall*, void*))at[4];
  attn_fn = (int (*)(const CacheAttnCall*, void*))at[5];
  attn_ws = (long (*)(int, int, int, int, int))at[6];
  verify_fn = (int (*)(const VerifyCall*, void*))at[7];
  Py_RETURN_NONE;
}

#define TB_METHOD(name, fn, doc) {name, (PyCFunction)(void (*)(void))fn, METH_FASTCALL, doc}
PyMethodDef methods[] = {TB_METHOD("bind", py_bind, "The launchers' addresses; before anything else."),
                         TB_METHOD("rotary", py_rotary, "See torsh_b200.ops.rotary.rotary."),
                         TB_METHOD("kv_write", py_write, "See torsh_b200.ops.kv_cache.kv_cache_write."),
                         TB_METHOD("kv_read", py_read, "See torsh_b200.ops.kv_cache.kv_cache_read."),
                         TB_METHOD("kv_attention", py_attention, "See torsh_b200.ops.kv_cache.kv_cache_attention."),
                         TB_METHOD("verify", py_verify, "See torsh_b200.ops.speculative.verify_draft."),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_decode_calls", "Calls of the decoding operators that need no conversion.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__decode_calls() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) < 0) Py_CLEAR(m);
  return m;
}
