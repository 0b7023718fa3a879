// _mvfp8: the calls of the 8-bit cache (paged_attention_fp8.py) from a plan's
// packed words and one layer's tensors, with the wrappers' checks, the outputs'
// allocation and the launch in native code (host C++ on torch's tensor API, no
// HIP), as _mvtorch does for the other caches (py_torch.cpp). Measured on the
// box's host, us of a call back to back: an append of one token 13.7 in Python,
// a decode 10.6, a gather 9.7, where their kernels take 3 to 6.
//
// Every function returns None where anything differs from the plain case (other
// shapes, types, devices, strides or alignments, subclassed tensors, another
// current device): the wrapper then runs its own path, which copies or raises.
// Otherwise it launches and returns the outputs, or the entry point's status code
// where that is not 0. Nothing is kept between calls.
#include "py_rows.h"

#include <c10/core/impl/DeviceGuardImplInterface.h>

namespace {

decltype(&mv_fp8_kv_cache_write) g_write;
decltype(&mv_fp8_paged_decode) g_decode;
decltype(&mv_fp8_paged_prefill) g_prefill;
decltype(&mv_fp8_gather_kv) g_gather;

// The 8-bit pool of one layer, [nb, hkv, bs, d], on the current device `index`.
bool pool_ok(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& sc, int64_t nb, int64_t hkv, int64_t bs,
             int64_t d, int64_t index) {
  if (!kc.is_cuda() || kc.device().index() != index) return false;
  const auto* guard = c10::impl::getDeviceGuardImpl(kc.device().type());
  return guard->getDevice().index() == index && kc.scalar_type() == at::kFloat8_e4m3fn && caches_ok(kc, vc, kc) &&
         sized(kc, {nb, hkv, bs, d}) && (d == 64 || d == 128) && sc.scalar_type() == at::kFloat &&
         sc.device() == kc.device() && sized(sc, {nb, hkv, 2}) && sc.is_contiguous();
}
bool rows16(const at::Tensor& t, const at::Tensor& pool) {
  return t.device() == pool.device() && (t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16);
}

// write(plan words, query or None, key, value, cos or None, sin or None,
// key_cache, value_cache, kv_scales, block_size, return_key, stream): (query out
// or None, key out or None). Words: items, table, status, max items, positions,
// tokens, block size, blocks, table rows, device.
PyObject* write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 12) return PyErr_Format(PyExc_TypeError, "_mvfp8.write takes 12 arguments");
  const Words w(a[0], 10);
  const bool has_q = a[1] != Py_None, rope = a[4] != Py_None;
  const at::Tensor *q = has_q ? plain(a[1]) : nullptr, *k = plain(a[2]), *v = plain(a[3]),
                   *cos = rope ? plain(a[4]) : nullptr, *sin = rope ? plain(a[5]) : nullptr, *kc = plain(a[6]),
                   *vc = plain(a[7]), *sc = plain(a[8]);
  const int64_t bs = PyLong_AsLongLong(a[9]);
  const int return_key = PyObject_IsTrue(a[10]);
  if (PyErr_Occurred()) return nullptr;
  if (!w.p || (has_q && !q) || !k || !v || (rope && (!cos || !sin)) || (has_q && !rope) || !kc || !vc || !sc ||
      k->dim() != 3 || (q && q->dim() != 3) || (rope && cos->dim() != 2))
    return none();
  const int64_t t = w.i(5), hkv = k->size(1), d = k->size(2);
  Rows rq{}, rk, rv;
  const auto like = [&](const at::Tensor& x) {
    return x.scalar_type() == k->scalar_type() && x.device() == k->device();
  };
  if (t == 0 || bs != w.i(6) || !pool_ok(*kc, *vc, *sc, w.i(7), hkv, bs, d, w.i(9)) || !rows16(*k, *kc) ||
      k->size(0) != t || k->sizes() != v->sizes() || !like(*v) || !aligned_rows(*k, rk) || !aligned_rows(*v, rv))
    return none();
  if (q && (!like(*q) || q->size(0) != t || q->size(2) != d || !aligned_rows(*q, rq))) return none();
  if (rope && (!like(*cos) || !like(*sin) || cos->sizes() != sin->sizes() || cos->size(0) != w.i(8) || cos->size(1) < d ||
               cos->stride(1) != 1 || sin->stride(1) != 1 || cos->stride(0) != sin->stride(0) || cos->stride(0) % 8 ||
               reinterpret_cast<uintptr_t>(cos->data_ptr()) % 16 || reinterpret_cast<uintptr_t>(sin->data_ptr()) % 16))
    return none();
  at::Tensor q_out, k_out;
  const int64_t hq = q ? q->size(1) : 0;
  if (q) q_out = at::empty(q->sizes(), q->options());
  if (return_key) k_out = at::empty(k->sizes(), k->options());
  const int rc = g_write(
      rq.p, rq.st, rq.sh, q ? q_out.data_ptr() : nullptr, hq * d, q ? d : 0, rk.p, rk.st, rk.sh,
      return_key ? k_out.data_ptr() : nullptr, return_key ? hkv * d : 0, return_key ? d : 0, rv.p, rv.st, rv.sh,
      kc->data_ptr(), vc->data_ptr(), sc->data_ptr<float>(), w.ptr<const int32_t>(0), w.ptr<const int32_t>(1),
      w.ptr<const int32_t>(2), static_cast<int32_t>(w.i(3)), rope ? w.ptr<const int64_t>(4) : nullptr,
      rope ? cos->data_ptr() : nullptr, rope ? sin->data_ptr() : nullptr, rope ? cos->stride(0) : 0, w.i(8), t,
      static_cast<int32_t>(hq), static_cast<int32_t>(hkv), static_cast<int32_t>(d), static_cast<int32_t>(bs), w.i(7),
      dtype_code(k->scalar_type()), address(a[11]));
  if (rc) return status(rc);
  PyObject* qo = q ? THPVariable_Wrap(std::move(q_out)) : Py_NewRef(Py_None);
  PyObject* ko = return_key ? THPVariable_Wrap(std::move(k_out)) : Py_NewRef(Py_None);
  PyObject* pair = qo && ko ? PyTuple_Pack(2, qo, ko) : nullptr;
  Py_XDECREF(qo);
  Py_XDECREF(ko);
  return pair;
  END_HANDLE_TH_ERRORS
}

// decode(plan words, query, key_cache, value_cache, kv_scales, block_table,
// kv_len, block_size, stream). Words: as _mvtorch.decode's (the dtype's place
// not used), then the device.
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9) return PyErr_Format(PyExc_TypeError, "_mvfp8.decode takes 9 arguments");
  const Words w(a[0], 18);
  const at::Tensor *q = plain(a[1]), *kc = plain(a[2]), *vc = plain(a[3]), *sc = plain(a[4]), *bt = plain(a[5]),
                   *kv = plain(a[6]);
  if (!w.p || !q || !kc || !vc || !sc || !bt || !kv) return none();
  const int64_t b = w.i(8), hq = w.i(9), hkv = w.i(10), d = w.i(11), bs = w.i(12), nb = w.i(13);
  const int64_t block_size = PyLong_AsLongLong(a[7]);
  if (PyErr_Occurred()) return nullptr;
  Rows rq;
  if (block_size != bs || !pool_ok(*kc, *vc, *sc, nb, hkv, bs, d, w.i(17)) || !rows16(*q, *kc) ||
      !sized(*q, {b, hq, d}) || bt->dim() < 1 || bt->size(0) != b || !sized(*kv, {b}) || b == 0 || !aligned_rows(*q, rq))
    return none();
  at::Tensor out = at::empty({b, hq, d}, q->options());
  const int rc =
      g_decode(rq.p, rq.st, rq.sh, kc->data_ptr(), vc->data_ptr(), sc->data_ptr<float>(), w.ptr<const int32_t>(0),
               w.ptr<const int32_t>(1), w.i(2), static_cast<int32_t>(w.i(3)), static_cast<int32_t>(w.i(4)),
               static_cast<int32_t>(w.i(5)), w.ptr<int32_t>(6), out.data_ptr(), hq * d, d, static_cast<float>(w.f(7)),
               static_cast<int32_t>(b), static_cast<int32_t>(hq), static_cast<int32_t>(hkv), static_cast<int32_t>(d),
               static_cast<int32_t>(bs), nb, dtype_code(q->scalar_type()), w.ptr<void>(15),
               static_cast<size_t>(w.i(16)), address(a[8]));
  return rc ? status(rc) : THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// prefill(plan words, query, key, value, key_cache, value_cache, kv_scales,
// rows of out, block_size, stream). Words: as _mvtorch.prefill's.
PyObject* prefill(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 10) return PyErr_Format(PyExc_TypeError, "_mvfp8.prefill takes 10 arguments");
  const Words w(a[0], 20);
  const at::Tensor *q = plain(a[1]), *k = plain(a[2]), *v = plain(a[3]), *kc = plain(a[4]), *vc = plain(a[5]),
                   *sc = plain(a[6]);
  const int64_t rows = PyLong_AsLongLong(a[7]), block_size = PyLong_AsLongLong(a[8]);
  if (PyErr_Occurred()) return nullptr;
  if (!w.p || !q || !k || !v || !kc || !vc || !sc || q->dim() != 3 || k->dim() != 3) return none();
  const int64_t hq = w.i(11), hkv = w.i(12), d = w.i(13), bs = w.i(14), nb = w.i(15);
  Rows rq, rk, rv;
  if (block_size != bs || !pool_ok(*kc, *vc, *sc, nb, hkv, bs, d, w.i(19)) || !rows16(*q, *kc) || q->size(0) < rows ||
      rows == 0 || q->size(1) != hq || q->size(2) != d || k->sizes() != v->sizes() || k->size(0) < rows ||
      k->size(1) != hkv || k->size(2) != d || dtype_code(q->scalar_type()) != w.i(16) ||
      k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type() || k->device() != q->device() ||
      v->device() != q->device() || !aligned_rows(*q, rq) || !aligned_rows(*k, rk) || !aligned_rows(*v, rv))
    return none();
  at::Tensor out = at::empty({rows, hq, d}, q->options());
  const int rc = g_prefill(
      rq.p, rq.st, rq.sh, rk.p, rk.st, rk.sh, rv.p, rv.st, rv.sh, kc->data_ptr(), vc->data_ptr(), sc->data_ptr<float>(),
      w.ptr<const void>(0), static_cast<int32_t>(w.i(1)), w.i(2), w.ptr<const int64_t>(3), static_cast<int32_t>(w.i(4)),
      w.ptr<const int32_t>(5), static_cast<int32_t>(w.i(6)), static_cast<int32_t>(w.i(7)),
      static_cast<int32_t>(w.i(8)), static_cast<int32_t>(w.i(9)), out.data_ptr(), hq * d, d,
      static_cast<float>(w.f(10)), static_cast<int32_t>(hq), static_cast<int32_t>(hkv), static_cast<int32_t>(d),
      static_cast<int32_t>(bs), nb, static_cast<int32_t>(w.i(16)), w.ptr<void>(17), static_cast<size_t>(w.i(18)),
      address(a[9]));
  return rc ? status(rc) : THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// gather(plan words, key_cache, value_cache, kv_scales, block_size, fp16?,
// stream): (K, V). Words: slots, tokens, block size, blocks, device.
PyObject* gather(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7) return PyErr_Format(PyExc_TypeError, "_mvfp8.gather takes 7 arguments");
  const Words w(a[0], 5);
  const at::Tensor *kc = plain(a[1]), *vc = plain(a[2]), *sc = plain(a[3]);
  const int64_t bs = PyLong_AsLongLong(a[4]);
  const int half = PyObject_IsTrue(a[5]);
  if (PyErr_Occurred()) return nullptr;
  if (!w.p || !kc || !vc || !sc || kc->dim() != 4) return none();
  const int64_t t = w.i(1), hkv = kc->size(1), d = kc->size(3);
  if (t == 0 || bs != w.i(2) || !pool_ok(*kc, *vc, *sc, w.i(3), hkv, bs, d, w.i(4))) return none();
  const auto options = kc->options().dtype(half ? at::kHalf : at::kBFloat16);
  at::Tensor k = at::empty({t, hkv, d}, options), v = at::empty({t, hkv, d}, options);
  const int rc = g_gather(kc->data_ptr(), vc->data_ptr(), sc->data_ptr<float>(), w.ptr<const int64_t>(0), t,
                          k.data_ptr(), v.data_ptr(), static_cast<int32_t>(hkv), static_cast<int32_t>(d),
                          static_cast<int32_t>(bs), w.i(3), half ? MV_DTYPE_F16 : MV_DTYPE_BF16, address(a[6]));
  if (rc) return status(rc);
  PyObject* ko = THPVariable_Wrap(std::move(k));
  PyObject* vo = THPVariable_Wrap(std::move(v));
  PyObject* pair = ko && vo ? PyTuple_Pack(2, ko, vo) : nullptr;
  Py_XDECREF(ko);
  Py_XDECREF(vo);
  return pair;
  END_HANDLE_TH_ERRORS
}

// bind(write, decode, prefill, gather): the entry points' addresses in the
// loaded libmvattn.so.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 4) return PyErr_Format(PyExc_TypeError, "_mvfp8.bind takes 4 addresses");
  void* p[4];
  for (int k = 0; k < 4; ++k) {
    p[k] = PyLong_AsVoidPtr(a[k]);
    if (PyErr_Occurred()) return nullptr;
    if (!p[k]) return PyErr_Format(PyExc_ValueError, "_mvfp8.bind: null address");
  }
  g_write = reinterpret_cast<decltype(g_write)>(p[0]);
  g_decode = reinterpret_cast<decltype(g_decode)>(p[1]);
  g_prefill = reinterpret_cast<decltype(g_prefill)>(p[2]);
  g_gather = reinterpret_cast<decltype(g_gather)>(p[3]);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", FASTCALL(bind), "bind the entry points"},
    {"write", FASTCALL(write), "mv_fp8_kv_cache_write of one layer"},
    {"decode", FASTCALL(decode), "mv_fp8_paged_decode of one layer"},
    {"prefill", FASTCALL(prefill), "mv_fp8_paged_prefill of one layer"},
    {"gather", FASTCALL(gather), "mv_fp8_gather_kv of one layer"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mvfp8", "calls of the 8-bit cache of libmvattn", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

// (ABI: the header this module was built against)
PyMODINIT_FUNC PyInit__mvfp8(void) {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddIntConstant(m, "ABI", MVATTN_ABI_VERSION) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
