// Host side of the per-layer ops: argument checks and launches without
// Python in between.
//
// store_kvcache, paged_decode_attention, paged_prefill_attention and
// prompt_attention run once per layer and step, build_step_metadata once per
// step; checked in Python and bound through ctypes, a call costs
// the host more than the kernels of a small step take.  These functions do the
// same checks on the tensors themselves and call the C ABI (one layer's store
// and decode, B = 1, 1800 tokens: 41.8 us a step in Python, 16.1 here, where
// the GPU needs 14; a 3001-token store 13.0 and 4.9 us; a prefill reads its
// outcome from pinned memory instead of through a concatenation and a copy,
// 18 us less).  They only take calls that they can prove good: anything else
// (another device than the current one, a tensor subclass, no workspace yet, a
// contract violation, an error status) returns None, and the caller's Python
// path handles it, with its messages.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/Functions.h>
#include <ATen/core/Tensor.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>

#include "prism_kv.h"

namespace {

constexpr int kMaxDevices = 64;
bool g_ready[kMaxDevices];  // the library's code objects are loaded (written and read under the GIL)

// A plain tensor with storage, or null.  Subclasses and wrappers (fake,
// functional, vmapped) go to the Python path.
const at::Tensor* tensor(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.defined() && t.has_storage() && t.layout() == at::kStrided ? &t : nullptr;
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return PRISM_DTYPE_F32;
    case at::kBFloat16: return PRISM_DTYPE_BF16;
    case at::kHalf: return PRISM_DTYPE_F16;
    case at::kFloat8_e4m3fn: return PRISM_DTYPE_FP8_E4M3FN;
    default: return -1;
  }
}

// Every tensor on one device, which is ready and current.
template <typename... T>
bool on_current_device(int& device, const at::Tensor* first, const T*... rest) {
  if (!first->is_cuda()) return false;
  device = first->get_device();
  if (device < 0 || device >= kMaxDevices || !g_ready[device]) return false;
  return ((rest == nullptr || (rest->is_cuda() && rest->get_device() == device)) && ...) &&
         c10::hip::current_device() == device;
}

bool scale_pair(const at::Tensor& cache, const at::Tensor* ks, const at::Tensor* vs) {
  if (ks == nullptr) return true;
  const auto want = cache.sizes().slice(0, cache.dim() - 1);
  return cache.scalar_type() == at::kFloat8_e4m3fn && ks->sizes() == want && vs->sizes() == want &&
         ks->scalar_type() == at::kFloat && vs->scalar_type() == at::kFloat;
}

// An optional pair of arguments: both None, or both tensors.
bool optional_pair(PyObject* a, PyObject* b, const at::Tensor*& ta, const at::Tensor*& tb) {
  ta = tb = nullptr;
  if (a == Py_None && b == Py_None) return true;
  ta = tensor(a);
  tb = tensor(b);
  return ta != nullptr && tb != nullptr;
}

// The value at (device, stream) of a dict, borrowed, or null.
PyObject* by_stream(PyObject* dict, int device, void* stream) {
  PyObject* key = Py_BuildValue("(iK)", device, static_cast<unsigned long long>(reinterpret_cast<uintptr_t>(stream)));
  if (key == nullptr) return nullptr;
  PyObject* found = PyDict_CheckExact(dict) ? PyDict_GetItem(dict, key) : nullptr;
  Py_DECREF(key);
  return found;
}

bool capturing() { return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None; }

// The kernels enqueued on this stream by the call; Python's device context is
// not needed since the tensors are on the current device.
void* current_stream(int device) { return c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(device)).stream(); }

// The GIL is released over allocations and launches, which may wait (for memory,
// for room in a full queue): other Python threads run meanwhile, as they do
// under the ctypes calls.  The arguments stay alive, their caller holds them;
// what is found elsewhere (a stream's workspace) has to be held here.
class WithoutGil {
 public:
  WithoutGil() : state_(PyEval_SaveThread()) {}
  ~WithoutGil() { PyEval_RestoreThread(state_); }
  WithoutGil(const WithoutGil&) = delete;
  WithoutGil& operator=(const WithoutGil&) = delete;

 private:
  PyThreadState* state_;
};

// mark_ready(device): prism_preload has run there.
PyObject* mark_ready(PyObject*, PyObject* arg) {
  const long device = PyLong_AsLong(arg);
  if (device == -1 && PyErr_Occurred()) return nullptr;
  if (device >= 0 && device < kMaxDevices) g_ready[device] = true;
  Py_RETURN_NONE;
}

// store(key, value, k_cache, v_cache, slot_mapping, k_scale, v_scale) -> True or None
PyObject* store(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7) Py_RETURN_NONE;
  const at::Tensor *key = tensor(args[0]), *value = tensor(args[1]), *kc = tensor(args[2]), *vc = tensor(args[3]),
                   *slots = tensor(args[4]), *ks, *vs;
  if (!key || !value || !kc || !vc || !slots || !optional_pair(args[5], args[6], ks, vs)) Py_RETURN_NONE;
  int device;
  if (!on_current_device(device, key, value, kc, vc, slots, ks, vs)) Py_RETURN_NONE;
  if (key->dim() != 3 || key->sizes() != value->sizes() || (kc->dim() != 3 && kc->dim() != 4) ||
      kc->sizes() != vc->sizes() || kc->scalar_type() != vc->scalar_type())
    Py_RETURN_NONE;
  const int64_t tokens = key->size(0), heads = key->size(1), dim = key->size(2);
  if (tokens <= 0 || heads <= 0 || dim <= 0 || heads > INT32_MAX || dim > INT32_MAX || kc->size(-2) != heads ||
      kc->size(-1) != dim || slots->dim() != 1 || slots->numel() != tokens || slots->scalar_type() != at::kInt ||
      !slots->is_contiguous() || !scale_pair(*kc, ks, vs))
    Py_RETURN_NONE;
  const int in = dtype_code(key->scalar_type()), out = dtype_code(kc->scalar_type());
  if (in < 0 || in == PRISM_DTYPE_FP8_E4M3FN || value->scalar_type() != key->scalar_type() || out < 0 ||
      key->stride(2) != 1 || value->stride(2) != 1 || key->stride(1) != dim || value->stride(1) != dim ||
      !kc->is_contiguous() || !vc->is_contiguous() || (ks && (!ks->is_contiguous() || !vs->is_contiguous())))
    Py_RETURN_NONE;
  const int64_t kst[3] = {key->stride(0), key->stride(1), key->stride(2)};
  const int64_t vst[3] = {value->stride(0), value->stride(1), value->stride(2)};
  int rc;
  {
    WithoutGil released;
    rc = prism_kv_store(key->data_ptr(), value->data_ptr(), in, kst, vst, kc->data_ptr(), vc->data_ptr(), out,
                        ks ? static_cast<float*>(ks->data_ptr()) : nullptr,
                        vs ? static_cast<float*>(vs->data_ptr()) : nullptr,
                        static_cast<const int32_t*>(slots->data_ptr()), tokens, static_cast<int>(heads),
                        static_cast<int>(dim), kc->numel() / (heads * dim), current_stream(device));
  }
  if (rc != PRISM_OK) Py_RETURN_NONE;
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// rows: 0 for leading dimensions of one entry, which may hold any number there.
struct Strides {
  int64_t v[4];
  explicit Strides(const at::Tensor* t, bool rows = false) : v{0, 0, 0, 0} {
    if (t != nullptr)
      for (int64_t i = 0; i < t->dim() && i < 4; ++i) v[i] = rows && i + 1 < t->dim() && t->size(i) == 1 ? 0 : t->stride(i);
  }
};

// Every row of the last dimension is contiguous and starts on 16 bytes.
bool aligned_rows(const at::Tensor& t) {
  const int64_t unit = 16 / static_cast<int64_t>(t.element_size()), last = t.dim() - 1;
  if (t.stride(last) != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0) return false;
  for (int64_t i = 0; i < last; ++i)
    if (t.size(i) != 1 && t.stride(i) % unit != 0) return false;
  return true;
}

bool records_gradients(const at::Tensor* q, const at::Tensor* k, const at::Tensor* v) {
  return c10::GradMode::is_enabled() && (q->requires_grad() || k->requires_grad() || v->requires_grad());
}

bool int32_vector(const at::Tensor& t) { return t.dim() == 1 && t.scalar_type() == at::kInt && t.is_contiguous(); }

// A paged decode's arguments, checked: decode's of eleven (from args[0]).
struct DecodeCall {
  const at::Tensor *q, *kc, *vc, *bt, *ctx, *max_ctx, *ks, *vs;
  double scale;
  int device, qd, cd;
  int64_t batch, heads, dim, blocks, page, kv_heads, width;
  void* stream;
  int64_t need;       // workspace bytes
  at::Tensor ws_own;  // the workspace: the stream's, held over the launch (another thread may put a larger one in
                      // its place), or a captured call's from the graph's pool
  void* ws;
};

bool check_decode(PyObject* const* args, DecodeCall& d) {
  d.q = tensor(args[0]), d.kc = tensor(args[1]), d.vc = tensor(args[2]), d.bt = tensor(args[3]);
  d.ctx = tensor(args[4]), d.max_ctx = tensor(args[8]);
  if (!d.q || !d.kc || !d.vc || !d.bt || !d.ctx || !d.max_ctx || !optional_pair(args[6], args[7], d.ks, d.vs)) return false;
  if (!PyFloat_CheckExact(args[5]) || !PyLong_CheckExact(args[9])) return false;
  d.scale = PyFloat_AS_DOUBLE(args[5]);
  int overflow = 0;
  const long block_n = PyLong_AsLongAndOverflow(args[9], &overflow);
  if (overflow || block_n <= 0 || (block_n & (block_n - 1))) return false;
  const at::Tensor &q = *d.q, &kc = *d.kc;
  if (!on_current_device(d.device, d.q, d.kc, d.vc, d.bt, d.ctx, d.max_ctx, d.ks, d.vs)) return false;
  if (q.dim() != 3 || kc.dim() != 4 || kc.sizes() != d.vc->sizes() || kc.scalar_type() != d.vc->scalar_type() ||
      d.bt->dim() != 2 || d.ctx->dim() != 1 || d.bt->scalar_type() != at::kInt || d.ctx->scalar_type() != at::kInt ||
      !d.ctx->is_contiguous() || d.max_ctx->numel() != 1 || d.max_ctx->scalar_type() != at::kInt ||
      !scale_pair(kc, d.ks, d.vs))
    return false;
  d.batch = q.size(0), d.heads = q.size(1), d.dim = q.size(2);
  d.blocks = kc.size(0), d.page = kc.size(1), d.kv_heads = kc.size(2), d.width = d.bt->size(1);
  d.qd = dtype_code(q.scalar_type()), d.cd = dtype_code(kc.scalar_type());
  if (d.qd < 0 || d.qd == PRISM_DTYPE_FP8_E4M3FN || d.cd < 0 || d.batch <= 0 || d.heads <= 0 || d.dim <= 0 ||
      d.dim > 256 || kc.size(3) != d.dim || d.page <= 0 || d.kv_heads <= 0 || d.heads % d.kv_heads != 0 ||
      d.bt->size(0) < d.batch || d.ctx->size(0) < d.batch || kc.stride(3) != 1 || d.batch > INT32_MAX ||
      d.heads > INT32_MAX || d.page > INT32_MAX || d.width > INT32_MAX)
    return false;
  d.stream = current_stream(d.device);
  d.need = prism_paged_decode_workspace_bytes(static_cast<int>(d.batch), static_cast<int>(d.heads),
                                              static_cast<int>(d.kv_heads), static_cast<int>(d.dim),
                                              static_cast<int>(d.page), static_cast<int>(d.width), d.cd);
  d.ws = nullptr;
  if (d.need > 0) {
    if (capturing()) {
      WithoutGil released;
      d.ws_own = at::empty({d.need}, q.options().dtype(at::kByte));
    } else {
      PyObject* found = by_stream(args[10], d.device, d.stream);
      const at::Tensor* ws = found ? tensor(found) : nullptr;
      if (ws == nullptr || ws->numel() < d.need) return false;
      d.ws_own = *ws;
    }
    d.ws = d.ws_own.data_ptr();
  }
  return true;
}

const float* scales(const at::Tensor* t) { return t ? static_cast<const float*>(t->data_ptr()) : nullptr; }

// decode(q, k_cache, v_cache, block_tables, context_lens, scale, k_scale, v_scale, max_context_len, block_n,
//        workspaces) -> output or None
PyObject* decode(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  DecodeCall d;
  if (n != 11 || !check_decode(args, d)) Py_RETURN_NONE;
  at::Tensor out;
  int rc;
  {
    WithoutGil released;
    out = at::empty_like(*d.q);
    const Strides sq(d.q), sk(d.kc), sv(d.vc), sks(d.ks), svs(d.vs), sbt(d.bt), so(&out);
    rc = prism_paged_decode(
        d.q->data_ptr(), d.qd, sq.v, d.kc->data_ptr(), d.vc->data_ptr(), d.cd, sk.v, sv.v, scales(d.ks), scales(d.vs),
        sks.v, svs.v, static_cast<const int32_t*>(d.bt->data_ptr()), sbt.v, static_cast<const int32_t*>(d.ctx->data_ptr()),
        static_cast<const int32_t*>(d.max_ctx->data_ptr()), out.data_ptr(), so.v, static_cast<int>(d.batch),
        static_cast<int>(d.heads), static_cast<int>(d.kv_heads), static_cast<int>(d.dim), static_cast<int>(d.page),
        d.blocks, static_cast<int>(d.width), static_cast<float>(d.scale), d.ws, d.need, d.stream);
  }
  if (rc != PRISM_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// step(decode's eleven, key, value, slot_mapping) -> output or None: the store
// of the step's rows, then the decode
PyObject* step(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  DecodeCall d;
  if (n != 14 || !check_decode(args, d)) Py_RETURN_NONE;
  const at::Tensor *key = tensor(args[11]), *value = tensor(args[12]), *slots = tensor(args[13]);
  int device;
  if (!key || !value || !slots || !on_current_device(device, key, value, slots) || device != d.device) Py_RETURN_NONE;
  if (key->dim() != 3 || key->sizes() != value->sizes() || key->size(0) != d.batch || key->size(1) != d.kv_heads ||
      key->size(2) != d.dim || slots->dim() != 1 || slots->numel() != d.batch || slots->scalar_type() != at::kInt ||
      !slots->is_contiguous() || key->scalar_type() != d.q->scalar_type() ||
      value->scalar_type() != d.q->scalar_type() || key->stride(2) != 1 || value->stride(2) != 1 ||
      key->stride(1) != d.dim || value->stride(1) != d.dim || !d.kc->is_contiguous() || !d.vc->is_contiguous() ||
      (d.ks && (!d.ks->is_contiguous() || !d.vs->is_contiguous())))
    Py_RETURN_NONE;
  at::Tensor out;
  int rc;
  {
    WithoutGil released;
    out = at::empty_like(*d.q);
    const Strides skey(key), sval(value), sq(d.q), sk(d.kc), sv(d.vc), sks(d.ks), svs(d.vs), sbt(d.bt), so(&out);
    rc = prism_paged_decode_step(
        key->data_ptr(), value->data_ptr(), skey.v, sval.v, static_cast<const int32_t*>(slots->data_ptr()),
        d.q->data_ptr(), d.qd, sq.v, d.kc->data_ptr(), d.vc->data_ptr(), d.cd, sk.v, sv.v,
        const_cast<float*>(scales(d.ks)), const_cast<float*>(scales(d.vs)), sks.v, svs.v,
        static_cast<const int32_t*>(d.bt->data_ptr()), sbt.v, static_cast<const int32_t*>(d.ctx->data_ptr()),
        static_cast<const int32_t*>(d.max_ctx->data_ptr()), out.data_ptr(), so.v, static_cast<int>(d.batch),
        static_cast<int>(d.heads), static_cast<int>(d.kv_heads), static_cast<int>(d.dim), static_cast<int>(d.page),
        d.blocks, static_cast<int>(d.width), static_cast<float>(d.scale), d.ws, d.need, d.stream);
  }
  if (rc != PRISM_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// Waits until the word is set; false where the stream is done, or has failed,
// without that.
bool outcome_known(const int32_t* word, void* stream) {
  while (true) {
    for (int i = 0; i < 2000; ++i) {
      if (__atomic_load_n(word, __ATOMIC_ACQUIRE) != 0) return true;
      __builtin_ia32_pause();
    }
    if (hipStreamQuery(static_cast<hipStream_t>(stream)) != hipErrorNotReady) return __atomic_load_n(word, __ATOMIC_ACQUIRE) != 0;
    (void)hipGetLastError();  // (not ready: no error for the next launch's check to find)
  }
}

// prefill(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens_q, num_heads, num_kv_heads, scale, k_scale,
//         v_scale, buffers) -> (out, first bad sequence, first row, end row) or None
//
// buffers: this thread's {(device, stream): (status int32[1] on the device,
// pinned int32[4])}; status holds INT32_MAX between calls.  Waits for the
// outcome: over FP8 caches with the stream, over 16-bit ones for the word that
// the launch's check sets.
PyObject* prefill(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 12) Py_RETURN_NONE;
  const at::Tensor *q = tensor(args[0]), *kc = tensor(args[1]), *vc = tensor(args[2]), *bt = tensor(args[3]),
                   *ctx = tensor(args[4]), *cu = tensor(args[5]), *ks, *vs;
  if (!q || !kc || !vc || !bt || !ctx || !cu || !optional_pair(args[9], args[10], ks, vs)) Py_RETURN_NONE;
  if (!PyLong_CheckExact(args[6]) || !PyLong_CheckExact(args[7]) || !PyFloat_CheckExact(args[8])) Py_RETURN_NONE;
  int over1 = 0, over2 = 0;
  const long heads = PyLong_AsLongAndOverflow(args[6], &over1), kv_heads = PyLong_AsLongAndOverflow(args[7], &over2);
  const double scale = PyFloat_AS_DOUBLE(args[8]);
  int device;
  if (over1 || over2 || !on_current_device(device, q, kc, vc, bt, ctx, cu, ks, vs) || capturing()) Py_RETURN_NONE;
  if (q->dim() != 3 || kc->dim() != 4 || kc->sizes() != vc->sizes() || bt->dim() != 2 ||
      (kc->scalar_type() != at::kFloat8_e4m3fn && kc->scalar_type() != q->scalar_type()) ||
      vc->scalar_type() != kc->scalar_type() || !scale_pair(*kc, ks, vs) ||
      bt->scalar_type() != at::kInt || ctx->scalar_type() != at::kInt || cu->scalar_type() != at::kInt ||
      ctx->dim() != 1 || cu->dim() != 1 || !ctx->is_contiguous() || !cu->is_contiguous())
    Py_RETURN_NONE;
  const int64_t total = q->size(0), dim = q->size(2), batch = ctx->numel();
  const int qd = dtype_code(q->scalar_type());
  if ((qd != PRISM_DTYPE_BF16 && qd != PRISM_DTYPE_F16) || total <= 0 || total > INT32_MAX || batch <= 0 ||
      batch > INT32_MAX || heads <= 0 || kv_heads <= 0 || heads > INT32_MAX || heads % kv_heads != 0 ||
      q->size(1) != heads || q->stride(2) != 1 || kc->size(2) != kv_heads || kc->size(3) != dim ||
      kc->size(0) > INT32_MAX || kc->size(1) > INT32_MAX || bt->size(1) > INT32_MAX || cu->numel() < batch + 1 ||
      bt->size(0) < batch)
    Py_RETURN_NONE;
  const bool sixteen = kc->scalar_type() == q->scalar_type();
  if (sixteen && records_gradients(q, kc, vc)) Py_RETURN_NONE;
  if (sixteen ? (dim != 64 && dim != 128) || !aligned_rows(*q) : dim != 128) Py_RETURN_NONE;
  void* stream = current_stream(device);
  PyObject* found = by_stream(args[11], device, stream);
  if (found == nullptr || !PyTuple_CheckExact(found) || PyTuple_GET_SIZE(found) != 2) Py_RETURN_NONE;
  const at::Tensor *status = tensor(PyTuple_GET_ITEM(found, 0)), *report = tensor(PyTuple_GET_ITEM(found, 1));
  if (!status || !report) Py_RETURN_NONE;
  const int page = static_cast<int>(kc->size(1)), width = static_cast<int>(bt->size(1));
  const int64_t need =
      sixteen ? prism_paged_prefill_16bit_workspace_bytes(static_cast<int>(batch), static_cast<int>(total), static_cast<int>(heads),
                                                          static_cast<int>(kv_heads), static_cast<int>(dim), page, width)
              : prism_paged_prefill_workspace_bytes(static_cast<int>(batch), static_cast<int>(total),
                                                    static_cast<int>(heads), static_cast<int>(kv_heads), page, width);
  at::Tensor out, ws;
  int32_t* words = static_cast<int32_t*>(report->data_ptr());
  words[0] = words[3] = 0;  // (the thread's previous call on this stream has its outcome: nothing writes them any more)
  int rc;
  {
    WithoutGil released;
    out = at::empty(q->sizes(), q->options());
    if (need > 0) ws = at::empty({need}, q->options().dtype(at::kByte));
    const Strides sq(q, sixteen), sk(kc), sv(vc), sks(ks), svs(vs), sbt(bt), so(&out);
    rc = prism_paged_prefill_ws(
        q->data_ptr(), qd, sq.v, kc->data_ptr(), vc->data_ptr(), dtype_code(kc->scalar_type()), sk.v, sv.v, scales(ks),
        scales(vs), sks.v, svs.v, static_cast<const int32_t*>(bt->data_ptr()), sbt.v,
        static_cast<const int32_t*>(ctx->data_ptr()), static_cast<const int32_t*>(cu->data_ptr()), out.data_ptr(), so.v,
        static_cast<int>(batch), static_cast<int>(total), static_cast<int>(heads), static_cast<int>(kv_heads),
        static_cast<int>(dim), page, static_cast<int>(kc->size(0)), width, static_cast<float>(scale),
        static_cast<int32_t*>(status->data_ptr()), need > 0 ? ws.data_ptr() : nullptr, need, words, stream);
    if (rc == PRISM_OK && (!sixteen || !outcome_known(words + 3, stream) || *static_cast<volatile int32_t*>(words) != 0))
      C10_HIP_CHECK(hipStreamSynchronize(static_cast<hipStream_t>(stream)));
  }
  const volatile int32_t* r = words;
  if (rc != PRISM_OK || (sixteen && r[3] == 0)) Py_RETURN_NONE;
  const int row0 = r[1], row1 = r[2];
  const int bad = r[0] == 0 ? INT32_MAX : status->item<int32_t>();
  PyObject* wrapped = THPVariable_Wrap(std::move(out));
  if (wrapped == nullptr) return nullptr;
  return Py_BuildValue("(Niii)", wrapped, bad, row0, row1);
  END_HANDLE_TH_ERRORS
}

// prompt(q, k, v, cu_seqlens_q, cu_seqlens_k or None, num_heads, num_kv_heads, scale) -> output or None
PyObject* prompt(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) Py_RETURN_NONE;
  const bool same = args[4] == Py_None;
  const at::Tensor *q = tensor(args[0]), *k = tensor(args[1]), *v = tensor(args[2]), *cq = tensor(args[3]),
                   *ck = same ? cq : tensor(args[4]);
  if (!q || !k || !v || !cq || !ck || !PyLong_CheckExact(args[5]) || !PyLong_CheckExact(args[6]) || !PyFloat_CheckExact(args[7]))
    Py_RETURN_NONE;
  int over1 = 0, over2 = 0;
  const long heads = PyLong_AsLongAndOverflow(args[5], &over1), kv_heads = PyLong_AsLongAndOverflow(args[6], &over2);
  int device;
  if (over1 || over2 || !on_current_device(device, q, k, v, cq, ck) || records_gradients(q, k, v)) Py_RETURN_NONE;
  const int type = dtype_code(q->scalar_type());
  if (q->dim() != 3 || k->dim() != 3 || k->sizes() != v->sizes() || (type != PRISM_DTYPE_BF16 && type != PRISM_DTYPE_F16) ||
      k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type() || !int32_vector(*cq) || !int32_vector(*ck))
    Py_RETURN_NONE;
  const int64_t total_q = q->size(0), total_k = k->size(0), dim = q->size(2), batch = cq->numel() - 1;
  if (heads <= 0 || kv_heads <= 0 || heads > INT32_MAX || heads % kv_heads != 0 || q->size(1) != heads || k->size(1) != kv_heads ||
      k->size(2) != dim || (dim != 64 && dim != 128) || total_q <= 0 || total_q > (1 << 29) || total_k <= 0 || total_k > (1 << 29) ||
      batch < 0 || batch > INT32_MAX || ck->numel() != cq->numel() || (same && total_k != total_q) || !aligned_rows(*q) ||
      !aligned_rows(*k) || !aligned_rows(*v))
    Py_RETURN_NONE;
  void* stream = current_stream(device);
  const int64_t need = prism_prompt_attention_workspace_bytes(static_cast<int>(batch), static_cast<int>(total_q),
                                                              static_cast<int>(total_k), static_cast<int>(heads),
                                                              static_cast<int>(kv_heads), static_cast<int>(dim));
  at::Tensor out, ws;
  int rc;
  {
    WithoutGil released;
    out = at::empty(q->sizes(), q->options());
    if (need > 0) ws = at::empty({need}, q->options().dtype(at::kByte));
    const Strides sq(q, true), sk(k, true), sv(v, true), so(&out);
    rc = prism_prompt_attention(q->data_ptr(), sq.v, k->data_ptr(), sk.v, v->data_ptr(), sv.v, type,
                                static_cast<const int32_t*>(cq->data_ptr()), static_cast<const int32_t*>(ck->data_ptr()),
                                out.data_ptr(), so.v, static_cast<int>(batch), static_cast<int>(total_q),
                                static_cast<int>(total_k), static_cast<int>(heads), static_cast<int>(kv_heads),
                                static_cast<int>(dim), static_cast<float>(PyFloat_AS_DOUBLE(args[7])),
                                need > 0 ? ws.data_ptr() : nullptr, need, stream);
  }
  if (rc != PRISM_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// A tensor of `sizes` (contiguous) at an offset of int32 storage.
at::Tensor int32_view(const at::Tensor& base, int64_t offset, at::IntArrayRef sizes) {
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(base.storage()), base.key_set(), base.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(offset);
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return t;
}

// step_metadata(block_tables, cached_lens, query_lens, block_size, num_tokens, free_blocks or None, free_start or None)
// -> (packed, slot_mapping, positions, cu_seqlens_q, context_lens, max_context_len, next_free, first_misfit,
//     block_tables) or None
PyObject* step_metadata(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7) Py_RETURN_NONE;
  const at::Tensor *bt = tensor(args[0]), *cached = tensor(args[1]), *fresh = tensor(args[2]),
                   *free = args[5] == Py_None ? nullptr : tensor(args[5]), *start = args[6] == Py_None ? nullptr : tensor(args[6]);
  if (!bt || !cached || !fresh || (!free && args[5] != Py_None) || (!start && args[6] != Py_None) || !PyLong_CheckExact(args[3]) ||
      !PyLong_CheckExact(args[4]))
    Py_RETURN_NONE;
  int over1 = 0, over2 = 0;
  const long page = PyLong_AsLongAndOverflow(args[3], &over1), tokens = PyLong_AsLongAndOverflow(args[4], &over2);
  int device;
  if (over1 || over2 || page <= 0 || page > INT32_MAX || tokens < 0 || tokens > (1 << 30) ||
      !on_current_device(device, bt, cached, fresh, free, start))
    Py_RETURN_NONE;
  if (bt->dim() != 2 || bt->scalar_type() != at::kInt || !int32_vector(*cached) || !int32_vector(*fresh) ||
      (free && !int32_vector(*free)) || (start && (start->scalar_type() != at::kInt || start->numel() != 1)))
    Py_RETURN_NONE;
  const int64_t batch = bt->size(0), width = bt->size(1);
  if (cached->numel() != batch || fresh->numel() != batch || batch > 8192 || width > INT32_MAX ||
      (free && free->numel() > INT32_MAX))
    Py_RETURN_NONE;
  void* stream = current_stream(device);
  const int64_t words = prism_step_metadata_words(static_cast<int>(batch), static_cast<int>(width), static_cast<int>(tokens));
  at::Tensor packed;
  int rc;
  {
    WithoutGil released;
    packed = at::empty({words}, bt->options());
    const Strides sbt(bt);
    rc = prism_step_metadata(static_cast<const int32_t*>(bt->data_ptr()), sbt.v, static_cast<const int32_t*>(cached->data_ptr()),
                             static_cast<const int32_t*>(fresh->data_ptr()),
                             free ? static_cast<const int32_t*>(free->data_ptr()) : nullptr,
                             free ? static_cast<int>(free->numel()) : 0,
                             start ? static_cast<const int32_t*>(start->data_ptr()) : nullptr, static_cast<int>(batch),
                             static_cast<int>(width), static_cast<int>(page), static_cast<int>(tokens),
                             static_cast<int32_t*>(packed.data_ptr()), stream);
  }
  if (rc != PRISM_OK) Py_RETURN_NONE;
  const int64_t padded = (tokens + 3) / 4 * 4, cu = 2 * padded, ctx = cu + batch + 1, tail = ctx + batch;
  const int64_t tables = cu + (2 * batch + 4 + 3) / 4 * 4;
  at::Tensor views[9] = {packed, int32_view(packed, 0, {tokens}), int32_view(packed, padded, {tokens}),
                         int32_view(packed, cu, {batch + 1}), int32_view(packed, ctx, {batch}), int32_view(packed, tail, {}),
                         int32_view(packed, tail + 1, {}), int32_view(packed, tail + 2, {}),
                         int32_view(packed, tables, {batch, width})};
  PyObject* result = PyTuple_New(9);
  if (result == nullptr) return nullptr;
  for (int i = 0; i < 9; ++i) {
    PyObject* item = THPVariable_Wrap(std::move(views[i]));
    if (item == nullptr) {
      Py_DECREF(result);
      return nullptr;
    }
    PyTuple_SET_ITEM(result, i, item);
  }
  return result;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"mark_ready", mark_ready, METH_O, nullptr},
    {"store", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(store)), METH_FASTCALL, nullptr},
    {"decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(decode)), METH_FASTCALL, nullptr},
    {"step", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(step)), METH_FASTCALL, nullptr},
    {"prompt", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(prompt)), METH_FASTCALL, nullptr},
    {"step_metadata", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(step_metadata)), METH_FASTCALL, nullptr},
    {"prefill", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(prefill)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host_ops() { return PyModule_Create(&module); }
