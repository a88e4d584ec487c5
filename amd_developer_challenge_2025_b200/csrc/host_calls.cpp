// The per-call host work of the Python entry points, as a CPython module: the checks of the five (or two) tensors, the
// current stream, and the call of the C ABI. The operator is called in tight loops on problems that run for a few
// microseconds; the same checks and the argument conversion of a ctypes call took 12 to 15 us in Python and take about
// one here. Every call is checked in full, nothing is remembered between calls.
//
// A function returns True (or its results) when the kernel has been launched. It returns False, having done nothing, for anything but
// the plain case (a check that fails, tensors that are not plain CUDA tensors on the current device, a workspace that
// does not exist yet, a code other than 0 from the library): the caller then goes through the checks in Python, which
// raise the error or handle the case.

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "b200_fp8_mm.h"
#include "b200_mla_cache.h"
#include "b200_mla_consumers.h"

namespace {

decltype(&b200_fp8_mm_strided) g_strided = nullptr;
decltype(&b200_fp8_mm_grouped) g_grouped = nullptr;
decltype(&b200_mla_rope) g_rope = nullptr;
decltype(&b200_mla_div_softmax) g_softmax = nullptr;
decltype(&b200_mla_cache_append) g_append = nullptr;
decltype(&b200_mla_cache_attend) g_attend = nullptr;
decltype(&b200_mla_cache_attend_workspace_bytes) g_attend_workspace = nullptr;
decltype(&b200_mla_cache_evict) g_evict = nullptr;
decltype(&b200_mla_cache_evict_workspace_bytes) g_evict_workspace = nullptr;

constexpr int64_t kScaleBlock = 128;

// The library's call without the GIL: a launch can block while the device's queue is full. (The caller holds the
// tensors; everything the call needs has been read out of them before.)
template <typename F, typename... Args>
bool launched(F fn, Args... args) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = fn(args...);
  Py_END_ALLOW_THREADS
  return rc == 0;
}

const at::Tensor* plain_tensor(PyObject* o) {
  return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr;
}

// A strided CUDA tensor of the given type and rank on device `dev`.
bool is_cuda(const at::Tensor& t, c10::ScalarType type, int64_t rank, c10::DeviceIndex dev) {
  return t.is_cuda() && t.layout() == c10::kStrided && t.scalar_type() == type && t.dim() == rank && t.get_device() == dev;
}

bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

bool fits_int(int64_t v) { return v >= 0 && v <= 0x7fffffff; }

// The entry of `dict` for `key` (consumed), as a tensor; null when there is none.
const at::Tensor* lookup(PyObject* dict, PyObject* key) {
  if (key == nullptr) return nullptr;
  PyObject* v = PyDict_GetItemWithError(dict, key);  // borrowed
  Py_DECREF(key);
  return v != nullptr ? plain_tensor(v) : nullptr;
}

// fp8_mm(a, b, a_scale, b_scale, c, n_phase, workspaces, status[, address of the forced b200_fp8_mm_plan or 0])
bool run_fp8_mm(PyObject* const* args) {
  const at::Tensor *a = plain_tensor(args[0]), *b = plain_tensor(args[1]), *as = plain_tensor(args[2]),
                   *bs = plain_tensor(args[3]), *c = plain_tensor(args[4]);
  if (!a || !b || !as || !bs || !c || !PyIndex_Check(args[5])) return false;
  const c10::DeviceIndex dev = c10::cuda::current_device();
  if (!is_cuda(*a, at::kFloat8_e4m3fn, 2, dev) || !is_cuda(*b, at::kFloat8_e4m3fn, 2, dev) ||
      !is_cuda(*as, at::kFloat, 2, dev) || !is_cuda(*bs, at::kFloat, 2, dev) || !is_cuda(*c, at::kBFloat16, 2, dev))
    return false;
  const Py_ssize_t phase = PyNumber_AsSsize_t(args[5], nullptr);
  if (phase < 0 || phase >= kScaleBlock) return false;
  const auto* plan = static_cast<const b200_fp8_mm_plan*>(args[8] != nullptr ? PyLong_AsVoidPtr(args[8]) : nullptr);
  if (PyErr_Occurred()) return false;
  const int64_t m = a->size(0), k = a->size(1), n = b->size(0);
  if (m <= 0 || n <= 0 || k <= 0 || !fits_int(m) || !fits_int(n) || !fits_int(k) || k % kScaleBlock != 0) return false;
  const int64_t kb = k / kScaleBlock, nb = (n + phase + kScaleBlock - 1) / kScaleBlock;
  if (b->size(1) != k || c->size(0) != m || c->size(1) != n || as->size(0) != m || as->size(1) != kb ||
      bs->size(0) != nb || bs->size(1) != kb)
    return false;
  const int64_t a0 = a->stride(0), a1 = a->stride(1), b0 = b->stride(0), b1 = b->stride(1);
  const bool a_k = a1 == 1 && a0 >= k, b_k = b1 == 1 && b0 >= k;
  if (!a_k && !(a0 == 1 && a1 >= m)) return false;
  if (!b_k && !(b0 == 1 && b1 >= n)) return false;
  if ((a_k ? a0 : a1) % 16 != 0 || (b_k ? b0 : b1) % 16 != 0 || !aligned16(*a) || !aligned16(*b)) return false;
  if (c->stride(1) != 1) return false;
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  const at::Tensor* st = lookup(args[7], PyLong_FromLong(dev));
  if (st == nullptr) return false;
  const at::Tensor* ws = lookup(args[6], Py_BuildValue("(iK)", static_cast<int>(dev),
                                                       static_cast<unsigned long long>(reinterpret_cast<uintptr_t>(stream))));
  return launched(g_strided, a->data_ptr(), b->data_ptr(), static_cast<const float*>(as->data_ptr()),
                   static_cast<const float*>(bs->data_ptr()), c->data_ptr(), static_cast<int>(m), static_cast<int>(n),
                   static_cast<int>(k), a0, a1, b0, b1, as->stride(0), as->stride(1), bs->stride(0), bs->stride(1),
                   c->stride(0), static_cast<int>(phase), ws ? ws->data_ptr() : nullptr,
                   ws ? static_cast<size_t>(ws->numel()) : 0, static_cast<int*>(st->data_ptr()), stream,
                  plan);
}

// fp8_mm_grouped(a, b, a_scale, b_scale, c, m_valid or None, status)
bool run_grouped(PyObject* const* args) {
  const at::Tensor *a = plain_tensor(args[0]), *b = plain_tensor(args[1]), *as = plain_tensor(args[2]),
                   *bs = plain_tensor(args[3]), *c = plain_tensor(args[4]);
  if (!a || !b || !as || !bs || !c) return false;
  const c10::DeviceIndex dev = c10::cuda::current_device();
  if (!is_cuda(*a, at::kFloat8_e4m3fn, 3, dev) || !is_cuda(*b, at::kFloat8_e4m3fn, 3, dev) ||
      !is_cuda(*as, at::kFloat, 3, dev) || !is_cuda(*bs, at::kFloat, 3, dev) || !is_cuda(*c, at::kBFloat16, 3, dev))
    return false;
  const int64_t g = a->size(0), m = a->size(1), k = a->size(2), n = b->size(1);
  if (g <= 0 || m <= 0 || n <= 0 || k <= 0 || !fits_int(g) || !fits_int(m) || !fits_int(n) || !fits_int(k) ||
      k % kScaleBlock != 0)
    return false;
  const int64_t kb = k / kScaleBlock, nb = (n + kScaleBlock - 1) / kScaleBlock;
  if (b->size(0) != g || b->size(2) != k || c->size(0) != g || c->size(1) != m || c->size(2) != n || as->size(0) != g ||
      as->size(1) != m || as->size(2) != kb || bs->size(0) != g || bs->size(1) != nb || bs->size(2) != kb)
    return false;
  if (a->stride(2) != 1 || b->stride(2) != 1 || c->stride(2) != 1) return false;
  if (a->stride(1) % 16 != 0 || a->stride(0) % 16 != 0 || b->stride(1) % 16 != 0 || b->stride(0) % 16 != 0 ||
      !aligned16(*a) || !aligned16(*b))
    return false;
  const int* rows = nullptr;
  if (args[5] != Py_None) {
    const at::Tensor* mv = plain_tensor(args[5]);
    if (!mv || !is_cuda(*mv, at::kInt, 1, dev) || mv->size(0) != g || !mv->is_contiguous()) return false;
    rows = static_cast<const int*>(mv->data_ptr());
  }
  const at::Tensor* st = lookup(args[6], PyLong_FromLong(dev));
  if (st == nullptr) return false;
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  return launched(g_grouped, a->data_ptr(), b->data_ptr(), static_cast<const float*>(as->data_ptr()),
                   static_cast<const float*>(bs->data_ptr()), c->data_ptr(), static_cast<int>(g), static_cast<int>(m),
                   static_cast<int>(n), static_cast<int>(k), a->stride(1), a->stride(0), b->stride(1), b->stride(0),
                   as->stride(0), as->stride(1), as->stride(2), bs->stride(0), bs->stride(1), bs->stride(2), c->stride(1),
                   c->stride(0), rows, static_cast<int*>(st->data_ptr()),
                   stream, static_cast<const b200_fp8_mm_plan*>(nullptr));
}

// Reads `count` Python ints; false when one is none or does not fit `limit`.
bool ints(PyObject* const* args, int count, long long limit, long long* out) {
  for (int i = 0; i < count; ++i) {
    if (!PyLong_CheckExact(args[i])) return false;
    int overflow = 0;
    out[i] = PyLong_AsLongLongAndOverflow(args[i], &overflow);  // (beyond 64 bits the value itself would read as -1)
    if (overflow != 0 || out[i] > limit || out[i] < -limit) return false;
  }
  return true;
}

// Whether the elements off + [0, span1] + [0, span2] + [0, row) lie inside the bf16 tensor's storage (spans of either sign).
bool inside(const at::Tensor& t, long long off, long long span1, long long span2, long long row) {
  const long long first = off + (span1 < 0 ? span1 : 0) + (span2 < 0 ? span2 : 0);
  const long long last = off + (span1 > 0 ? span1 : 0) + (span2 > 0 ? span2 : 0) + row - 1;
  return t.storage_offset() + first >= 0 && t.storage_offset() + last < static_cast<long long>(t.storage().nbytes() / 2);
}

// mla_decode(x, y, pos, xoff, yoff, d0, d1, d2, xs1, xs2, ys1, ys2)
bool run_rope(PyObject* const* args) {
  const at::Tensor *x = plain_tensor(args[0]), *y = plain_tensor(args[1]);
  long long v[10];
  // (40 bits: the products below stay inside 64 bits once d0, d1 and d2 are known to fit 20)
  if (!x || !y || !ints(args + 2, 10, 1ll << 40, v)) return false;
  const long long pos = v[0], xoff = v[1], yoff = v[2], d0 = v[3], d1 = v[4], d2 = v[5], xs1 = v[6], xs2 = v[7],
                  ys1 = v[8], ys2 = v[9];
  const c10::DeviceIndex dev = c10::cuda::current_device();
  if (!x->is_cuda() || !y->is_cuda() || x->get_device() != dev || y->get_device() != dev ||
      x->layout() != c10::kStrided || y->layout() != c10::kStrided || x->scalar_type() != at::kBFloat16 ||
      y->scalar_type() != at::kBFloat16)
    return false;
  if (d0 <= 0 || d1 <= 0 || d2 <= 0 || d2 % 2 != 0 || d0 > (1 << 20) || d1 > (1 << 20) || d2 > (1 << 20) ||
      pos > 0x7fffffff || pos < -0x7fffffff || xoff < 0 || yoff < 0)
    return false;
  if (!inside(*x, xoff, (d0 - 1) * xs1, (d1 - 1) * xs2, d2) || !inside(*y, yoff, (d0 - 1) * ys1, (d1 - 1) * ys2, d2)) return false;
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  return launched(g_rope, static_cast<char*>(x->data_ptr()) + 2 * xoff, static_cast<char*>(y->data_ptr()) + 2 * yoff,
                static_cast<int>(pos), static_cast<int>(d0), static_cast<int>(d1), static_cast<int>(d2), xs1, xs2, ys1,
                ys2, stream);
}

// div_softmax(qk, bs, nh, sl, dnope, drope)
bool run_softmax(PyObject* const* args) {
  const at::Tensor* t = plain_tensor(args[0]);
  long long v[5];
  if (!t || !ints(args + 1, 5, 1 << 20, v)) return false;
  const c10::DeviceIndex dev = c10::cuda::current_device();
  if (!t->is_cuda() || t->get_device() != dev || t->layout() != c10::kStrided || t->scalar_type() != at::kBFloat16 ||
      !t->is_contiguous())
    return false;
  if (v[0] <= 0 || v[1] <= 0 || v[2] <= 0 || t->numel() != v[0] * v[1] * v[2]) return false;
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  return launched(g_softmax, t->data_ptr(), static_cast<int>(v[0]), static_cast<int>(v[1]), static_cast<int>(v[2]),
                   static_cast<int>(v[3]), static_cast<int>(v[4]), stream);
}

// ---- Operators around a paged latent cache: the checks of mla_cache.py

// No two elements share an address.
bool distinct(const at::Tensor& t) {
  int64_t need = 1;
  bool used[3] = {};
  for (int64_t round = 0; round < t.dim(); ++round) {
    int64_t best = -1;
    for (int64_t i = 0; i < t.dim(); ++i)
      if (!used[i] && (best < 0 || t.stride(i) < t.stride(best))) best = i;
    used[best] = true;
    if (t.size(best) <= 1) continue;
    if (t.stride(best) < need) return false;
    need += t.stride(best) * (t.size(best) - 1);
  }
  return true;
}

// The bytes from the first to behind the last element do not meet. (Where they do, Python looks closer.)
bool apart(const at::Tensor& a, const at::Tensor& b) {
  auto end = [](const at::Tensor& t) {
    int64_t n = 1;
    for (int64_t i = 0; i < t.dim(); ++i) n += t.stride(i) * (t.size(i) - 1);
    return static_cast<const char*>(t.data_ptr()) + n * static_cast<int64_t>(t.element_size());
  };
  return end(a) <= static_cast<const char*>(b.data_ptr()) || end(b) <= static_cast<const char*>(a.data_ptr());
}

bool same(const at::Tensor& a, const at::Tensor& b) {
  return a.data_ptr() == b.data_ptr() && a.sizes() == b.sizes() && a.strides() == b.strides();
}

struct CacheCall {
  b200_mla_cache c;
  const at::Tensor* cache;
  int64_t batch, capacity, d;
  c10::DeviceIndex dev;
};

bool cache_call(PyObject* cache_arg, PyObject* table_arg, PyObject* lens_arg, long long dv, CacheCall* out) {
  const at::Tensor *cache = plain_tensor(cache_arg), *table = plain_tensor(table_arg), *lens = plain_tensor(lens_arg);
  if (!cache || !table || !lens) return false;
  const c10::DeviceIndex dev = c10::cuda::current_device();
  const auto type = cache->scalar_type();
  if ((type != at::kBFloat16 && type != at::kHalf) || !is_cuda(*cache, type, 3, dev) || !is_cuda(*table, at::kInt, 2, dev) ||
      !is_cuda(*lens, at::kInt, 1, dev))
    return false;
  const int64_t pages = cache->size(0), ps = cache->size(1), d = cache->size(2), batch = table->size(0), per = table->size(1);
  if (dv < 128 || dv > 512 || dv % 128 != 0 || d < dv || d > 576 || d % 64 != 0 || pages <= 0 || ps <= 0 || !fits_int(pages) || !fits_int(ps))
    return false;
  if (cache->stride(2) != 1 || cache->stride(0) % 8 != 0 || cache->stride(1) % 8 != 0 || cache->stride(0) < d || cache->stride(1) < d ||
      !aligned16(*cache))
    return false;
  if (per <= 0 || table->stride(1) != 1 || batch <= 0 || batch >= 65536 || lens->size(0) != batch || (batch > 1 && lens->stride(0) != 1) ||
      per > (1 << 30) / ps)
    return false;
  out->c = b200_mla_cache{cache->data_ptr(), static_cast<const int*>(table->data_ptr()), static_cast<const int*>(lens->data_ptr()),
                          type == at::kBFloat16 ? B200_MLA_CACHE_BF16 : B200_MLA_CACHE_FP16, static_cast<int>(pages), static_cast<int>(ps),
                          static_cast<int>(dv), static_cast<int>(d - dv), static_cast<int>(batch), static_cast<int>(per),
                          cache->stride(0), cache->stride(1), table->stride(0)};
  out->cache = cache;
  out->batch = batch;
  out->capacity = per * ps;
  out->d = d;
  out->dev = dev;
  return true;
}

// A value per slot of every sequence.
bool slots(const at::Tensor* t, c10::ScalarType type, const CacheCall& k) {
  return t && is_cuda(*t, type, 2, k.dev) && t->size(0) == k.batch && t->size(1) >= k.capacity && t->stride(1) == 1;
}

bool head_rows(const at::Tensor* t, const CacheCall& k, int64_t width) {
  return t && is_cuda(*t, k.cache->scalar_type(), 3, k.dev) && t->size(0) == k.batch && t->size(1) > 0 && t->size(2) == width && t->stride(2) == 1;
}

bool number(PyObject* o, double* out) {
  if (!PyFloat_CheckExact(o) && !PyLong_CheckExact(o)) return false;
  *out = PyFloat_AsDouble(o);
  return std::isfinite(*out) && !PyErr_Occurred();
}

// mla_cache_append(row, position, cache, block_table, lens, dv, theta, q, q_out, score, slot_position), the last four maybe None
bool run_append(PyObject* const* args) {
  CacheCall k;
  long long dv;
  double theta;
  if (!ints(args + 5, 1, 1 << 20, &dv) || !number(args[6], &theta) || theta <= 0 || !cache_call(args[2], args[3], args[4], dv, &k)) return false;
  const at::Tensor *row = plain_tensor(args[0]), *position = plain_tensor(args[1]);
  if (!row || !position || !is_cuda(*row, k.cache->scalar_type(), 2, k.dev) || row->size(0) != k.batch || row->size(1) != k.d || row->stride(1) != 1 ||
      !is_cuda(*position, at::kInt, 1, k.dev) || position->size(0) != k.batch || (k.batch > 1 && position->stride(0) != 1))
    return false;
  if (!distinct(*k.cache) || !apart(*row, *k.cache)) return false;
  const at::Tensor *q = nullptr, *q_out = nullptr, *score = nullptr, *at_slot = nullptr;
  if (args[7] != Py_None) {
    q = plain_tensor(args[7]);
    q_out = args[8] != Py_None ? plain_tensor(args[8]) : q;
    if (!head_rows(q, k, k.d) || !head_rows(q_out, k, k.d) || q->size(1) != q_out->size(1) || q->size(1) > (1 << 20) || !distinct(*q_out) ||
        !(same(*q, *q_out) || apart(*q, *q_out)) || !apart(*q_out, *row) || !apart(*q_out, *k.cache) || !apart(*q, *k.cache))
      return false;
  } else if (args[8] != Py_None) {
    return false;
  }
  if (args[9] != Py_None && (!slots(score = plain_tensor(args[9]), at::kFloat, k) || !distinct(*score))) return false;
  if (args[10] != Py_None && (!slots(at_slot = plain_tensor(args[10]), at::kInt, k) || !distinct(*at_slot))) return false;
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(k.dev).stream();
  return launched(g_append, static_cast<const b200_mla_cache*>(&k.c), row->data_ptr(), static_cast<long long>(row->stride(0)),
                  static_cast<const int*>(position->data_ptr()), theta, q ? q->data_ptr() : nullptr, q ? static_cast<long long>(q->stride(0)) : 0,
                  q ? static_cast<long long>(q->stride(1)) : 0, q_out ? q_out->data_ptr() : nullptr,
                  q_out ? static_cast<long long>(q_out->stride(0)) : 0, q_out ? static_cast<long long>(q_out->stride(1)) : 0,
                  q ? static_cast<int>(q->size(1)) : 0, score ? static_cast<float*>(score->data_ptr()) : nullptr,
                  score ? static_cast<long long>(score->stride(0)) : 0, at_slot ? static_cast<int*>(at_slot->data_ptr()) : nullptr,
                  at_slot ? static_cast<long long>(at_slot->stride(0)) : 0, stream);
}

// mla_cache_attend(q, cache, block_table, lens, dv, scale, out, score, score_out, max_len, return_lse, status); out, score, score_out and
// max_len maybe None. Returns out, or (out, lse).
PyObject* run_attend(PyObject* const* args) {
  CacheCall k;
  long long dv, most;
  double scale;
  if (!ints(args + 4, 1, 1 << 20, &dv) || !number(args[5], &scale) || !cache_call(args[1], args[2], args[3], dv, &k)) return nullptr;
  const at::Tensor* q = plain_tensor(args[0]);
  if (!head_rows(q, k, k.d) || q->size(1) > (1 << 16) || !aligned16(*q)) return nullptr;
  for (int i = 0; i < 2; ++i)
    if (q->size(i) > 1 && (q->stride(i) % 8 != 0 || q->stride(i) < k.d)) return nullptr;
  most = k.capacity;
  if (args[9] != Py_None && (!ints(args + 9, 1, 1ll << 40, &most) || most <= 0)) return nullptr;
  if (most > k.capacity) most = k.capacity;
  if (args[10] != Py_True && args[10] != Py_False) return nullptr;
  at::Tensor out, lse;
  if (args[6] != Py_None) {
    const at::Tensor* given = plain_tensor(args[6]);
    if (!head_rows(given, k, dv) || given->size(1) != q->size(1) || !distinct(*given) || !apart(*given, *q) || !apart(*given, *k.cache)) return nullptr;
    out = *given;
  }
  const at::Tensor *score = nullptr, *score_out = nullptr;
  if (args[7] != Py_None) {
    score = plain_tensor(args[7]);
    score_out = args[8] != Py_None ? plain_tensor(args[8]) : score;
    if (!slots(score, at::kFloat, k) || !slots(score_out, at::kFloat, k) || !distinct(*score_out) || !(same(*score, *score_out) || apart(*score, *score_out)))
      return nullptr;
  } else if (args[8] != Py_None) {
    return nullptr;
  }
  const at::Tensor* st = lookup(args[11], PyLong_FromLong(k.dev));
  if (st == nullptr) return nullptr;
  const int heads = static_cast<int>(q->size(1));
  // All of torch's allocator on the current stream, as in Python.
  if (!out.defined()) out = at::empty({k.batch, heads, dv}, q->options());
  if (args[10] == Py_True) lse = at::empty({k.batch, heads}, q->options().dtype(at::kFloat));
  const size_t bytes = g_attend_workspace(static_cast<int>(k.batch), heads, static_cast<int>(dv), static_cast<int>(k.d - dv), static_cast<int>(most), score != nullptr);
  const at::Tensor ws = at::empty({static_cast<int64_t>(bytes)}, q->options().dtype(at::kByte));
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(k.dev).stream();
  if (!launched(g_attend, static_cast<const b200_mla_cache*>(&k.c), q->data_ptr(), static_cast<long long>(q->stride(0)), static_cast<long long>(q->stride(1)),
                heads, static_cast<float>(scale), out.data_ptr(), static_cast<long long>(out.stride(0)), static_cast<long long>(out.stride(1)),
                lse.defined() ? static_cast<float*>(lse.data_ptr()) : nullptr, score ? static_cast<const float*>(score->data_ptr()) : nullptr,
                score ? static_cast<long long>(score->stride(0)) : 0, score ? static_cast<float*>(score_out->data_ptr()) : nullptr,
                score ? static_cast<long long>(score_out->stride(0)) : 0, static_cast<int>(most), ws.data_ptr(), bytes,
                static_cast<int*>(st->data_ptr()), stream))
    return nullptr;
  PyObject* o = THPVariable_Wrap(out);
  if (o == nullptr || !lse.defined()) return o;
  PyObject* l = THPVariable_Wrap(lse);
  if (l == nullptr) {
    Py_DECREF(o);
    return nullptr;
  }
  PyObject* both = PyTuple_Pack(2, o, l);
  Py_DECREF(o);
  Py_DECREF(l);
  return both;
}

// mla_cache_evict(cache, block_table, lens, score, slot_position, budget, recent, lens_out, score_out, position_out)
bool run_evict(PyObject* const* args) {
  CacheCall k;
  long long v[2];
  if (!ints(args + 5, 2, 0x7fffffff, v) || v[0] <= 0 || v[1] < 0 || v[1] > v[0] || !cache_call(args[0], args[1], args[2], 128, &k)) return false;
  const at::Tensor *lens = plain_tensor(args[2]), *score = plain_tensor(args[3]), *at_slot = plain_tensor(args[4]), *lens_out = plain_tensor(args[7]),
                   *score_out = plain_tensor(args[8]), *at_out = plain_tensor(args[9]);
  if (!lens_out || !is_cuda(*lens_out, at::kInt, 1, k.dev) || lens_out->size(0) != k.batch || (k.batch > 1 && lens_out->stride(0) != 1)) return false;
  if (!slots(score, at::kFloat, k) || !slots(score_out, at::kFloat, k) || !slots(at_slot, at::kInt, k) || !slots(at_out, at::kInt, k)) return false;
  if (!distinct(*k.cache) || !distinct(*score_out) || !distinct(*at_out)) return false;
  if (!(same(*lens, *lens_out) || apart(*lens, *lens_out)) || !(same(*score, *score_out) || apart(*score, *score_out)) ||
      !(same(*at_slot, *at_out) || apart(*at_slot, *at_out)))
    return false;
  const size_t bytes = g_evict_workspace(static_cast<int>(k.batch), static_cast<int>(k.capacity), static_cast<int>(v[0]));
  const at::Tensor ws = at::empty({static_cast<int64_t>(bytes)}, score->options().dtype(at::kByte));
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(k.dev).stream();
  return launched(g_evict, static_cast<const b200_mla_cache*>(&k.c), static_cast<const float*>(score->data_ptr()), static_cast<long long>(score->stride(0)),
                  static_cast<const int*>(at_slot->data_ptr()), static_cast<long long>(at_slot->stride(0)), static_cast<int>(v[0]),
                  static_cast<int>(v[1]), static_cast<int*>(lens_out->data_ptr()), static_cast<float*>(score_out->data_ptr()),
                  static_cast<long long>(score_out->stride(0)), static_cast<int*>(at_out->data_ptr()), static_cast<long long>(at_out->stride(0)),
                  ws.data_ptr(), bytes, stream);
}

// A C++ exception (a tensor without storage, a device that is gone) is "not the plain case" too.
// The last `Optional` of the N arguments may be left out (null).
template <bool (*F)(PyObject* const*), Py_ssize_t N, Py_ssize_t Optional = 0>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  bool done = false;
  if (nargs <= N && nargs >= N - Optional) {
    PyObject* all[N] = {};
    for (Py_ssize_t i = 0; i < nargs; ++i) all[i] = args[i];
    try {
      done = F(all);
    } catch (...) {
      done = false;
    }
    if (PyErr_Occurred()) {
      PyErr_Clear();
      done = false;
    }
  }
  return PyBool_FromLong(done);
}

// The same for a function that returns its results, or null.
template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
PyObject* results(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  PyObject* found = nullptr;
  if (nargs == N) {
    try {
      found = F(args);
    } catch (...) {
      found = nullptr;
    }
    if (PyErr_Occurred()) {
      PyErr_Clear();
      Py_CLEAR(found);
    }
  }
  if (found != nullptr) return found;
  Py_RETURN_FALSE;
}

// bind_cache(append, attend, attend_workspace_bytes, evict, evict_workspace_bytes): addresses of the loaded library's functions.
PyObject* bind_cache(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  void* f[5];
  if (nargs != 5) {
    PyErr_SetString(PyExc_TypeError, "bind_cache takes five addresses");
    return nullptr;
  }
  for (int i = 0; i < 5; ++i) {
    f[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  g_append = reinterpret_cast<decltype(g_append)>(f[0]);
  g_attend = reinterpret_cast<decltype(g_attend)>(f[1]);
  g_attend_workspace = reinterpret_cast<decltype(g_attend_workspace)>(f[2]);
  g_evict = reinterpret_cast<decltype(g_evict)>(f[3]);
  g_evict_workspace = reinterpret_cast<decltype(g_evict_workspace)>(f[4]);
  Py_RETURN_NONE;
}

// bind(strided, grouped, rope, softmax): addresses of the loaded library's functions.
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  void* f[4];
  if (nargs != 4) {
    PyErr_SetString(PyExc_TypeError, "bind takes four addresses");
    return nullptr;
  }
  for (int i = 0; i < 4; ++i) {
    f[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  g_strided = reinterpret_cast<decltype(g_strided)>(f[0]);
  g_grouped = reinterpret_cast<decltype(g_grouped)>(f[1]);
  g_rope = reinterpret_cast<decltype(g_rope)>(f[2]);
  g_softmax = reinterpret_cast<decltype(g_softmax)>(f[3]);
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F));
}

PyMethodDef methods[] = {
    {"bind", fast<bind>(), METH_FASTCALL, nullptr},
    {"fp8_mm", fast<entry<run_fp8_mm, 9, 1>>(), METH_FASTCALL, nullptr},
    {"fp8_mm_grouped", fast<entry<run_grouped, 7>>(), METH_FASTCALL, nullptr},
    {"mla_decode", fast<entry<run_rope, 12>>(), METH_FASTCALL, nullptr},
    {"div_softmax", fast<entry<run_softmax, 6>>(), METH_FASTCALL, nullptr},
    {"bind_cache", fast<bind_cache>(), METH_FASTCALL, nullptr},
    {"mla_cache_append", fast<entry<run_append, 11>>(), METH_FASTCALL, nullptr},
    {"mla_cache_attend", fast<results<run_attend, 12>>(), METH_FASTCALL, nullptr},
    {"mla_cache_evict", fast<entry<run_evict, 10>>(), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
