// Native call path of the operators a generation calls per layer and step
// (attention, the QKV producer, the slab pack): the Python extension
// heatkv_amd._op_call.
//
// A small launch runs 6-8 us on the device, but checking eight tensors, reading
// the knobs and marshalling about thirty arguments cost the Python operator
// 15-16 us per call, so calls on early scales ran at the host's pace.  Here the
// same checks read the tensors in C++ (nothing is remembered from one call for
// the next), the outputs are allocated and the library is called: 16.4 -> 6.1 us
// per call of 16 tokens (B=2, 16 heads), back to back; a whole layer's ten small
// scales at B=1 966 -> 837 us.
//
// Only calls that the Python operator would take as they are: every function
// returns None, having launched nothing, when anything asks for more (an
// error to raise, an input to convert, a knob that is set, a HIP graph being
// captured, a tensor subclass, a torch mode or transform, the stream's first
// call, which makes its workspace), and the caller runs the operator's Python
// body, which stays the one place that defines what is refused and why.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstring>
#include <string>
#include <type_traits>

#include "heatkv.h"

namespace {

constexpr int64_t kD = 128;

// The library's entry points (addresses from the handle that _lib.load()
// opened) and the Python dicts that hold the environment, the per-stream
// workspaces and the checked devices.
struct State {
  decltype(&hkv_segmented_attention) attention = nullptr;
  decltype(&hkv_segmented_attention_split) attention_split = nullptr;
  decltype(&hkv_segmented_attention_split_bytes) split_bytes = nullptr;
  decltype(&hkv_segmented_attention_item_shape) item_shape = nullptr;
  decltype(&hkv_qkv_produce) produce = nullptr;
  decltype(&hkv_pack_segments) pack = nullptr;
  decltype(&hkv_paged_tables) paged_tables = nullptr;
  decltype(&hkv_paged_append) paged_append = nullptr;
  decltype(&hkv_paged_attention) paged_attention = nullptr;
  decltype(&hkv_paged_attention_workspace_bytes) paged_workspace = nullptr;
  PyObject* env = nullptr;
  PyObject* knobs = nullptr;  // tuple of the environment keys that change a launch
  PyObject* workspaces = nullptr;
  PyObject* devices = nullptr;
  PyObject* paged_counters = nullptr;  // the paged attention's, per (device, stream)
  PyObject* plan_queries = nullptr;  // attribute names of a work plan
  PyObject* plan_shape = nullptr;
  bool ready = false;
} g;

struct Ref {  // a new reference
  PyObject* p;
  explicit Ref(PyObject* o) : p(o) {}
  ~Ref() { Py_XDECREF(p); }
  Ref(const Ref&) = delete;
  Ref& operator=(const Ref&) = delete;
};

int32_t code_of(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return HKV_DTYPE_F16;
    case at::kBFloat16: return HKV_DTYPE_BF16;
    case at::kFloat: return HKV_DTYPE_F32;
    default: return 0;
  }
}

// A plain strided tensor of the GPU: a torch.Tensor or Parameter that no
// subclass, transform, conjugate / negative view or fake mode stands behind.
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  const c10::DispatchKeySet rest =
      t.key_set() - c10::autograd_dispatch_keyset_with_ADInplaceOrView - c10::autocast_dispatch_keyset;
  return rest == c10::DispatchKeySet(c10::DispatchKey::CUDA) ? &t : nullptr;
}

bool dense(const at::Tensor& t, int64_t dim) { return t.dim() == dim && t.is_contiguous(); }
bool aligned(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

// No mode or transform that would see the operator's torch calls.
bool no_modes() {
  if (at::impl::torch_function_mode_enabled()) return false;
  const c10::DispatchKeySet usual =
      c10::DispatchKeySet({c10::DispatchKey::BackendSelect, c10::DispatchKey::ADInplaceOrView});
  return (c10::impl::tls_local_dispatch_key_set().included_ - usual).empty();
}

// The current device, gfx950 as already checked, with its current stream not
// under capture; -1 otherwise.
int current_device(void** stream) {
  const c10::DeviceIndex dev = c10::hip::current_device();
  Ref index(PyLong_FromLong(dev));
  if (PyDict_GetItem(g.devices, index.p) != Py_True) return -1;
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None) return -1;
  *stream = c10::hip::getCurrentHIPStream(dev).stream();
  return dev;
}

bool knobs_set() {
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(g.knobs); ++i)
    if (PyDict_GetItem(g.env, PyTuple_GET_ITEM(g.knobs, i)) != nullptr) return true;
  return false;
}

bool flag(PyObject* o, bool* v) {
  *v = o == Py_True;
  return o == Py_True || o == Py_False;
}

bool number(PyObject* o, double* v) {
  if (!PyFloat_CheckExact(o)) return false;
  *v = PyFloat_AS_DOUBLE(o);
  return true;
}

bool whole(PyObject* o, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  *v = PyLong_AsLongLongAndOverflow(o, &overflow);
  return overflow == 0;
}

// Whether `plan` (None: no plan) is what segmented_attention_plan made for
// items of `queries`, batch B and length L on `dev`; its tensor in *out.
bool plan_fits(PyObject* plan, int32_t queries, int64_t B, int64_t L, int dev, const at::Tensor** out) {
  *out = nullptr;
  if (plan == Py_None) return true;
  const at::Tensor* t = plain(plan);
  if (t == nullptr || t->scalar_type() != at::kInt || !dense(*t, 2) || t->size(1) != 8 || t->size(0) == 0 ||
      t->get_device() != dev)
    return false;
  Ref have(PyObject_GetAttr(plan, g.plan_queries)), shape(PyObject_GetAttr(plan, g.plan_shape));
  int64_t q = 0, b = 0, l = 0;
  if (have.p == nullptr || shape.p == nullptr) {
    PyErr_Clear();
    return false;
  }
  *out = t;
  return whole(have.p, &q) && q == queries && PyTuple_CheckExact(shape.p) && PyTuple_GET_SIZE(shape.p) == 2 &&
         whole(PyTuple_GET_ITEM(shape.p, 0), &b) && whole(PyTuple_GET_ITEM(shape.p, 1), &l) && b == B && l == L;
}

// Where an all-fp32 call is better split (_split_values_pays in
// real_pruning_fused_attention.py, which holds the figures; `split_from` and
// `split_slab` are its two limits).
bool split_values_pays(int64_t B, int64_t H, int64_t L, int64_t cap, int64_t split_from, int64_t split_slab, int dev) {
  const int64_t pairs = B * H, rows = pairs * L;
  int64_t limit = split_slab;
  if (rows >= split_from) limit = std::max((L > 256 ? 8 : 4) * rows, split_slab / 4);
  if (B * cap > limit) return false;
  if (rows < 8192 || pairs <= 64) return true;
  int32_t cus = 0;  // the staged kernel's resident workgroups
  if (g.item_shape(HKV_DTYPE_F32, HKV_DTYPE_F32, HKV_DTYPE_F32, 1, 0, 0, dev, &cus) < 0) return false;
  return pairs * ((L + 127) / 128) > cus;
}

// attention(q, persisted_k, persisted_v, segment_starts, segment_ends,
// segment_counts, current_k, current_v, softmax_scale, softmax_mode,
// return_lse, out_dtype, work_plan, k_split_rows, split_values_rows,
// split_values_slab_rows)
PyObject* attention_call(PyObject* const* args, Py_ssize_t n) {
  if (!g.ready || n != 16 || !no_modes() || knobs_set()) Py_RETURN_NONE;
  const at::Tensor* t[8];
  for (int i = 0; i < 8; ++i)
    if ((t[i] = plain(args[i])) == nullptr) Py_RETURN_NONE;
  const at::Tensor &q = *t[0], &pk = *t[1], &pv = *t[2], &st = *t[3], &en = *t[4], &ct = *t[5], &ck = *t[6],
                   &cv = *t[7];
  double scale = 0;
  int64_t split_from = 0, split_slab = 0;
  bool with_lse = false, k_split = false;
  if (!number(args[8], &scale) || !flag(args[10], &with_lse) || !flag(args[13], &k_split) ||
      !whole(args[14], &split_from) || !whole(args[15], &split_slab))
    Py_RETURN_NONE;
  const char* mode = PyUnicode_CheckExact(args[9]) ? PyUnicode_AsUTF8(args[9]) : nullptr;
  if (mode == nullptr || (std::strcmp(mode, "exp") != 0 && std::strcmp(mode, "exp2") != 0)) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  at::ScalarType out_type = q.scalar_type();
  if (args[11] != Py_None) {
    if (!THPDtype_Check(args[11])) Py_RETURN_NONE;
    out_type = reinterpret_cast<THPDtype*>(args[11])->scalar_type;
  }
  void* stream = nullptr;
  const int dev = current_device(&stream);
  if (dev < 0) Py_RETURN_NONE;
  for (const at::Tensor* x : t)
    if (x->get_device() != dev) Py_RETURN_NONE;

  if (!dense(q, 4) || !dense(ck, 4) || !dense(cv, 4) || !dense(pk, 3) || !dense(pv, 3) || !dense(st, 2) ||
      !dense(en, 2) || !dense(ct, 1))
    Py_RETURN_NONE;
  const int64_t B = q.size(0), H = q.size(1), L = q.size(2), cap = pk.size(1), S = st.size(1);
  if (ck.sizes() != q.sizes() || cv.sizes() != q.sizes() || q.size(3) != kD || L <= 0 || B <= 0 || H <= 0 ||
      pk.sizes() != pv.sizes() || pk.size(0) != B || pk.size(2) != kD || st.sizes() != en.sizes() ||
      st.size(0) != H || ct.size(0) != H || B > 0x7fffffff || H > 0x7fffffff || L > 0x7fffffff || S > 0x7fffffff)
    Py_RETURN_NONE;
  const int32_t qc = code_of(q.scalar_type()), kc = code_of(ck.scalar_type()), vc = code_of(cv.scalar_type()),
                oc = code_of(out_type);
  if (qc == 0 || kc != qc || vc == 0 || oc == 0 || pk.scalar_type() != ck.scalar_type() ||
      pv.scalar_type() != cv.scalar_type() || st.scalar_type() != at::kInt || en.scalar_type() != at::kInt ||
      ct.scalar_type() != at::kInt)
    Py_RETURN_NONE;
  // fp32 q and k at the default dot modes: K (and V) as split rows, made by the
  // call itself unless the caller has them
  const bool rows32 = qc == HKV_DTYPE_F32 && vc != HKV_DTYPE_F32;
  if (k_split && !rows32) Py_RETURN_NONE;
  const bool split_v =
      qc == HKV_DTYPE_F32 && vc == HKV_DTYPE_F32 && split_values_pays(B, H, L, cap, split_from, split_slab, dev);
  const bool splits = (rows32 && !k_split) || split_v;
  if (splits && (!aligned(ck) || !aligned(pk) || (split_v && (!aligned(cv) || !aligned(pv))))) Py_RETURN_NONE;
  const int32_t queries = rows32 ? g.item_shape(qc, HKV_DTYPE_SPLIT_ROWS, vc, 1, 0, 0, 0, nullptr) : 128;
  const at::Tensor* plan = nullptr;
  if (!plan_fits(args[12], queries, B, L, dev, &plan)) Py_RETURN_NONE;

  Ref index(PyLong_FromLong(dev)), handle(PyLong_FromVoidPtr(stream));
  Ref key(PyTuple_Pack(2, index.p, handle.p));
  PyObject* const ws_obj = key.p != nullptr ? PyDict_GetItem(g.workspaces, key.p) : nullptr;
  if (ws_obj == nullptr || !THPVariable_Check(ws_obj)) Py_RETURN_NONE;
  const at::Tensor ws = THPVariable_Unpack(ws_obj);

  const auto options = q.options().requires_grad(false);
  int64_t need = 0;
  if (splits && (need = g.split_bytes(static_cast<int32_t>(B), static_cast<int32_t>(H), static_cast<int32_t>(L), cap,
                                      vc)) < 0)
    Py_RETURN_NONE;
  at::Tensor out = at::empty({B, L, H * kD}, options.dtype(out_type));
  at::Tensor lse, scratch;
  if (with_lse) lse = at::empty({B, H, L}, options.dtype(at::kFloat));
  if (splits) scratch = at::empty({need}, options.dtype(at::kByte));
  const int32_t* const plan_p = plan != nullptr ? static_cast<const int32_t*>(plan->data_ptr()) : nullptr;
  const int32_t units = plan != nullptr ? static_cast<int32_t>(plan->size(0)) : 0;
  float* const lse_p = with_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
  const int32_t k_code = k_split ? HKV_DTYPE_SPLIT_ROWS : kc, exp2 = mode[3] != 0 ? 1 : 0;
  const int32_t b = static_cast<int32_t>(B), h = static_cast<int32_t>(H), l = static_cast<int32_t>(L),
                s = static_cast<int32_t>(S), d = static_cast<int32_t>(kD);
  const int32_t *sp = static_cast<const int32_t*>(st.data_ptr()), *ep = static_cast<const int32_t*>(en.data_ptr()),
                *cp = static_cast<const int32_t*>(ct.data_ptr());
  const float fscale = static_cast<float>(scale);
  int32_t code;
  Py_BEGIN_ALLOW_THREADS
  if (splits)
    code = g.attention_split(q.data_ptr(), pk.data_ptr(), pv.data_ptr(), sp, ep, cp, ck.data_ptr(), cv.data_ptr(),
                             out.data_ptr(), lse_p, b, h, l, cap, s, d, qc, k_code, vc, oc, fscale, exp2, 0, 0,
                             plan_p, units, ws.data_ptr(), ws.numel(), nullptr, nullptr, nullptr, 0, nullptr,
                             scratch.data_ptr(), need, stream);
  else
    code = g.attention(q.data_ptr(), pk.data_ptr(), pv.data_ptr(), sp, ep, cp, ck.data_ptr(), cv.data_ptr(),
                       out.data_ptr(), lse_p, b, h, l, cap, s, d, qc, k_code, vc, oc, fscale, exp2, 0, 0, plan_p,
                       units, ws.data_ptr(), ws.numel(), stream);
  Py_END_ALLOW_THREADS
  if (code != HKV_OK) Py_RETURN_NONE;  // refused: the Python body repeats the call and raises
  if (!with_lse) return THPVariable_Wrap(std::move(out));
  Ref o(THPVariable_Wrap(std::move(out))), e(THPVariable_Wrap(std::move(lse)));
  return o.p != nullptr && e.p != nullptr ? PyTuple_Pack(2, o.p, e.p) : nullptr;
}

// produce(qkv, num_heads, scale_mul, rope_table, rope_start_row, normalize,
// eps, qk_dtype, append, k_split_rows)
PyObject* produce_call(PyObject* const* args, Py_ssize_t n) {
  if (!g.ready || n != 10 || !no_modes()) Py_RETURN_NONE;
  const at::Tensor* qkv = plain(args[0]);
  int64_t H = 0, start = 0;
  bool normalize = false, k_split = false;
  double eps = 0;
  if (qkv == nullptr || !whole(args[1], &H) || !whole(args[4], &start) || !flag(args[5], &normalize) ||
      !number(args[6], &eps) || !THPDtype_Check(args[7]) || !flag(args[9], &k_split))
    Py_RETURN_NONE;
  void* stream = nullptr;
  const int dev = current_device(&stream);
  if (dev < 0 || qkv->get_device() != dev || !qkv->is_contiguous()) Py_RETURN_NONE;
  if (H <= 0 || H > 0x7fffffff) Py_RETURN_NONE;
  const bool whole_rows = qkv->dim() == 3 && qkv->size(2) == 3 * H * kD;
  const bool parts = qkv->dim() == 5 && qkv->size(2) == 3 && qkv->size(3) == H && qkv->size(4) == kD;
  if (!whole_rows && !parts) Py_RETURN_NONE;
  const int64_t B = qkv->size(0), L = qkv->size(1);
  const at::ScalarType qk = reinterpret_cast<THPDtype*>(args[7])->scalar_type;
  const int32_t ic = code_of(qkv->scalar_type()), oc = code_of(qk);
  if (B <= 0 || L <= 0 || B > 0x7fffffff || L > 0x7fffffff || ic == 0 || oc == 0 ||
      (k_split && oc != HKV_DTYPE_F32))
    Py_RETURN_NONE;
  const float *sm = nullptr, *rope = nullptr;
  int64_t rope_rows = 0;
  if (args[2] != Py_None) {
    const at::Tensor* t = plain(args[2]);
    if (t == nullptr || t->get_device() != dev || t->scalar_type() != at::kFloat || !t->is_contiguous() ||
        t->numel() != H)
      Py_RETURN_NONE;
    sm = static_cast<const float*>(t->data_ptr());
  }
  if (args[3] != Py_None) {
    const at::Tensor* t = plain(args[3]);
    if (t == nullptr || t->get_device() != dev || t->scalar_type() != at::kFloat || !dense(*t, 3) ||
        t->size(0) != 2 || t->size(2) != kD / 2)
      Py_RETURN_NONE;
    rope = static_cast<const float*>(t->data_ptr());
    rope_rows = t->size(1);
  }
  const at::Tensor *slab_k = nullptr, *slab_v = nullptr, *offsets = nullptr;
  if (args[8] != Py_None) {
    if (!PyTuple_CheckExact(args[8]) || PyTuple_GET_SIZE(args[8]) != 3) Py_RETURN_NONE;
    slab_k = plain(PyTuple_GET_ITEM(args[8], 0));
    slab_v = plain(PyTuple_GET_ITEM(args[8], 1));
    offsets = plain(PyTuple_GET_ITEM(args[8], 2));
    if (slab_k == nullptr || slab_v == nullptr || offsets == nullptr || slab_k->get_device() != dev ||
        slab_v->get_device() != dev || offsets->get_device() != dev || !dense(*slab_k, 3) || !dense(*slab_v, 3) ||
        slab_k->sizes() != slab_v->sizes() || slab_k->size(0) != B || slab_k->size(2) != kD ||
        slab_k->scalar_type() != qk || slab_v->scalar_type() != qkv->scalar_type() ||
        offsets->scalar_type() != at::kInt || !offsets->is_contiguous() || offsets->numel() != H)
      Py_RETURN_NONE;
  }
  const auto options = qkv->options().requires_grad(false);
  at::Tensor q = at::empty({B, H, L, kD}, options.dtype(qk)), k = at::empty({B, H, L, kD}, options.dtype(qk)),
             v = at::empty({B, H, L, kD}, options);
  int32_t code;
  Py_BEGIN_ALLOW_THREADS
  code = g.produce(qkv->data_ptr(), 3 * H * kD, nullptr, nullptr, sm, rope, rope_rows, start, q.data_ptr(),
                   k.data_ptr(), v.data_ptr(), slab_k != nullptr ? slab_k->data_ptr() : nullptr,
                   slab_v != nullptr ? slab_v->data_ptr() : nullptr,
                   offsets != nullptr ? static_cast<const int32_t*>(offsets->data_ptr()) : nullptr,
                   slab_k != nullptr ? slab_k->size(1) : 0, static_cast<int32_t>(B), static_cast<int32_t>(H),
                   static_cast<int32_t>(L), static_cast<int32_t>(kD), ic, oc, k_split ? HKV_DTYPE_SPLIT_ROWS : oc,
                   ic, normalize ? 1 : 0, static_cast<float>(eps), stream);
  Py_END_ALLOW_THREADS
  if (code != HKV_OK) Py_RETURN_NONE;
  Ref a(THPVariable_Wrap(std::move(q))), b(THPVariable_Wrap(std::move(k))), c(THPVariable_Wrap(std::move(v)));
  return a.p != nullptr && b.p != nullptr && c.p != nullptr ? PyTuple_Pack(3, a.p, b.p, c.p) : nullptr;
}

// pack(dst_k, dst_v, src_k, src_v, dst_starts, src_starts, lengths, max_length,
// block_t): True when the copy was launched
PyObject* pack_call(PyObject* const* args, Py_ssize_t n) {
  int64_t longest = 0, block = 0;
  if (!g.ready || n != 9 || !no_modes() || !whole(args[7], &longest) || !whole(args[8], &block)) Py_RETURN_NONE;
  const at::Tensor* t[7];
  for (int i = 0; i < 7; ++i)
    if ((t[i] = plain(args[i])) == nullptr) Py_RETURN_NONE;
  const at::Tensor &dk = *t[0], &dv = *t[1], &sk = *t[2], &sv = *t[3], &ds = *t[4], &ss = *t[5], &ln = *t[6];
  void* stream = nullptr;
  const int dev = current_device(&stream);
  if (dev < 0) Py_RETURN_NONE;
  for (const at::Tensor* x : t)
    if (x->get_device() != dev) Py_RETURN_NONE;
  if (!dense(dk, 3) || !dense(dv, 3) || !dense(sk, 3) || !dense(sv, 3) || dk.sizes() != dv.sizes() ||
      sk.sizes() != sv.sizes() || dk.size(0) != sk.size(0) || dk.size(2) != sk.size(2) || dk.size(2) > kD ||
      dk.numel() == 0 || sk.numel() == 0 || sk.scalar_type() != dk.scalar_type() ||
      sv.scalar_type() != dv.scalar_type() || dk.size(0) > 0x7fffffff)
    Py_RETURN_NONE;
  const int64_t items = ln.numel();
  for (const at::Tensor* x : {&ds, &ss, &ln})
    if (x->scalar_type() != at::kLong || !x->is_contiguous() || x->numel() != items) Py_RETURN_NONE;
  if (items <= 0 || items > 0x7fffffff || longest <= 0 || longest > 0x7fffffff || block <= 0 || block > 0x7fffffff)
    Py_RETURN_NONE;
  const int64_t limit = (longest + block - 1) / block * block;
  int32_t code;
  Py_BEGIN_ALLOW_THREADS
  code = g.pack(sk.data_ptr(), sv.data_ptr(), dk.data_ptr(), dv.data_ptr(), sk.stride(0), dk.stride(0), sk.size(1),
                dk.size(1), static_cast<int32_t>(dk.size(0)), static_cast<int32_t>(dk.size(2)),
                static_cast<int32_t>(dk.element_size()), static_cast<int32_t>(dv.element_size()),
                static_cast<const int64_t*>(ds.data_ptr()), static_cast<const int64_t*>(ss.data_ptr()),
                static_cast<const int64_t*>(ln.data_ptr()), static_cast<int32_t>(items),
                static_cast<int32_t>(limit < 0x7fffffff ? limit : 0x7fffffff), stream);
  Py_END_ALLOW_THREADS
  if (code != HKV_OK) Py_RETURN_NONE;
  Py_RETURN_TRUE;
}

// ------------------------------------------------------------- paged cache

// int32 vector of n elements on dev.
bool ints(const at::Tensor& t, int64_t n, int dev) {
  return t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous() && t.get_device() == dev;
}

// A block table [R, M] with rows side by side or further apart.
bool table_rows(const at::Tensor& t, int dev) {
  return t.scalar_type() == at::kInt && t.dim() == 2 && t.get_device() == dev && t.size(0) <= 4096 &&
         t.size(1) <= 0x7fffffff && (t.size(1) <= 1 || t.stride(1) == 1) &&
         (t.size(0) <= 1 || t.stride(0) >= t.size(1));
}

bool power_of_two(int64_t v) { return v > 0 && v <= (1 << 20) && (v & (v - 1)) == 0; }

bool wants_grad(const at::Tensor& t) { return t.requires_grad() && c10::GradMode::is_enabled(); }

// Two caches [blocks, kv_heads, block, dim] of one 16-bit type on dev.
bool caches(const at::Tensor& k, const at::Tensor& v, int dev) {
  if (k.dim() != 4 || v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type() || k.get_device() != dev ||
      v.get_device() != dev || (k.scalar_type() != at::kHalf && k.scalar_type() != at::kBFloat16))
    return false;
  return k.size(0) > 0 && k.size(0) <= 0x7fffffff && k.size(1) > 0 && k.size(1) <= 1024 && power_of_two(k.size(2)) &&
         (k.size(3) == 64 || k.size(3) == 128) && k.stride(3) == 1 && v.stride(3) == 1 && !wants_grad(k) &&
         !wants_grad(v);
}

const int32_t* i32(const at::Tensor& t) { return static_cast<const int32_t*>(t.data_ptr()); }

PyObject* tuple_of(std::initializer_list<at::Tensor> tensors) {
  PyObject* out = PyTuple_New(static_cast<Py_ssize_t>(tensors.size()));
  Py_ssize_t i = 0;
  for (const at::Tensor& t : tensors) {
    PyObject* o = out != nullptr ? THPVariable_Wrap(t) : nullptr;
    if (o == nullptr) {
      Py_XDECREF(out);
      return nullptr;
    }
    PyTuple_SET_ITEM(out, i++, o);
  }
  return out;
}

// Elements [offset, offset + n) of a one-dimensional tensor, sharing its storage
// (0.1 us where a dispatched view takes 1 and an allocation of its own 0.9).
at::Tensor piece(const at::Tensor& base, int64_t offset, int64_t n) {
  auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(base.storage()),
                                                   c10::DispatchKeySet(c10::DispatchKey::CUDA), base.dtype());
  impl->set_storage_offset(base.storage_offset() + offset);
  impl->set_sizes_contiguous({n});
  return at::Tensor(std::move(impl));
}

// paged_tables(block_tables, lengths, new_counts, free_blocks, free_range,
// num_tokens, block_size, window, sinks, in_place): (slot_map, query_starts, lengths,
// free_range, status)
PyObject* paged_tables_call(PyObject* const* args, Py_ssize_t n) {
  if (!g.ready || n != 10 || !no_modes()) Py_RETURN_NONE;
  const at::Tensor* t[5];
  for (int i = 0; i < 5; ++i)
    if ((t[i] = plain(args[i])) == nullptr) Py_RETURN_NONE;
  const at::Tensor &tables = *t[0], &lengths = *t[1], &counts = *t[2], &ring = *t[3], &range = *t[4];
  int64_t tokens, block, window, sinks;
  bool in_place;
  void* stream = nullptr;
  const int dev = current_device(&stream);
  if (dev < 0 || !whole(args[5], &tokens) || !whole(args[6], &block) || !whole(args[7], &window) ||
      !whole(args[8], &sinks) || !flag(args[9], &in_place) || !table_rows(tables, dev) || ring.dim() != 1)
    Py_RETURN_NONE;
  const int64_t R = tables.size(0), N = ring.size(0);
  if (!ints(lengths, R, dev) || !ints(counts, R, dev) || !ints(ring, N, dev) || !ints(range, 2, dev) || tokens < 0 ||
      tokens > 0x7fffffff || N > 0x7fffffff || !power_of_two(block) || window < 0 || window > 0x7fffffff || sinks < 0 ||
      sinks > 0x7fffffff)
    Py_RETURN_NONE;
  const auto options = lengths.options();
  at::Tensor slots = at::empty({tokens}, options.dtype(at::kLong));
  at::Tensor small = at::empty({2 * R + 6}, options);
  at::Tensor starts = piece(small, 0, R + 1), status = piece(small, R + 1, 3);
  at::Tensor range_out = in_place ? range : piece(small, R + 4, 2);
  at::Tensor lengths_out = in_place ? lengths : piece(small, R + 6, R);
  int32_t code;
  Py_BEGIN_ALLOW_THREADS
  code = g.paged_tables(static_cast<int32_t*>(tables.data_ptr()), tables.stride(0), i32(lengths), i32(counts),
                        static_cast<int32_t*>(ring.data_ptr()), i32(range), static_cast<int32_t>(R),
                        static_cast<int32_t>(tables.size(1)), static_cast<int32_t>(N), static_cast<int32_t>(tokens),
                        static_cast<int32_t>(block), static_cast<int32_t>(window), static_cast<int32_t>(sinks),
                        static_cast<int64_t*>(slots.data_ptr()), static_cast<int32_t*>(starts.data_ptr()),
                        static_cast<int32_t*>(lengths_out.data_ptr()), static_cast<int32_t*>(range_out.data_ptr()),
                        static_cast<int32_t*>(status.data_ptr()), stream);
  Py_END_ALLOW_THREADS
  if (code != HKV_OK) Py_RETURN_NONE;
  at::Tensor first = piece(small, R + 1, 1);
  if (!in_place) return tuple_of({slots, starts, lengths_out, range_out, first});
  Ref a(THPVariable_Wrap(slots)), b(THPVariable_Wrap(starts)), c(THPVariable_Wrap(first));
  if (a.p == nullptr || b.p == nullptr || c.p == nullptr) return nullptr;
  return PyTuple_Pack(5, a.p, b.p, args[1], args[4], c.p);
}

// paged_append(k, v, k_cache, v_cache, slot_map): True when the copy was launched
PyObject* paged_append_call(PyObject* const* args, Py_ssize_t n) {
  if (!g.ready || n != 5 || !no_modes()) Py_RETURN_NONE;
  const at::Tensor* t[5];
  for (int i = 0; i < 5; ++i)
    if ((t[i] = plain(args[i])) == nullptr) Py_RETURN_NONE;
  const at::Tensor &k = *t[0], &v = *t[1], &kc = *t[2], &vc = *t[3], &slots = *t[4];
  void* stream = nullptr;
  const int dev = current_device(&stream);
  if (dev < 0 || !caches(kc, vc, dev) || k.dim() != 3 || v.sizes() != k.sizes() || k.size(0) > 0x7fffffff ||
      k.size(1) != kc.size(1) || k.size(2) != kc.size(3) || k.scalar_type() != kc.scalar_type() ||
      v.scalar_type() != kc.scalar_type() || k.get_device() != dev || v.get_device() != dev || k.stride(2) != 1 ||
      v.stride(2) != 1 || wants_grad(k) || wants_grad(v) || slots.scalar_type() != at::kLong || slots.dim() != 1 ||
      slots.size(0) != k.size(0) || !slots.is_contiguous() || slots.get_device() != dev)
    Py_RETURN_NONE;
  int32_t code;
  Py_BEGIN_ALLOW_THREADS
  code = g.paged_append(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), v.stride(0), v.stride(1), kc.data_ptr(),
                        vc.data_ptr(), kc.stride(0), kc.stride(1), kc.stride(2), vc.stride(0), vc.stride(1),
                        vc.stride(2), static_cast<const int64_t*>(slots.data_ptr()),
                        static_cast<int32_t>(kc.size(0)), static_cast<int32_t>(k.size(0)),
                        static_cast<int32_t>(kc.size(1)), static_cast<int32_t>(kc.size(3)),
                        static_cast<int32_t>(kc.size(2)), stream);
  Py_END_ALLOW_THREADS
  if (code != HKV_OK) Py_RETURN_NONE;
  Py_RETURN_TRUE;
}

// paged_attention(q, k_cache, v_cache, prefix_blocks, prefix_length,
// block_tables, lengths, query_starts, softmax_scale, window, sinks, causal,
// out, return_lse): out, or (out, lse)
PyObject* paged_attention_call(PyObject* const* args, Py_ssize_t n) {
  if (!g.ready || n != 14 || !no_modes()) Py_RETURN_NONE;
  const int at_index[6] = {0, 1, 2, 5, 6, 7};
  const at::Tensor* t[6];
  for (int i = 0; i < 6; ++i)
    if ((t[i] = plain(args[at_index[i]])) == nullptr) Py_RETURN_NONE;
  const at::Tensor &q = *t[0], &kc = *t[1], &vc = *t[2], &tables = *t[3], &lengths = *t[4], &starts = *t[5];
  int64_t prefix, window, sinks;
  double scale;
  bool causal, with_lse;
  void* stream = nullptr;
  const int dev = current_device(&stream);
  if (dev < 0 || !whole(args[4], &prefix) || !number(args[8], &scale) || !whole(args[9], &window) ||
      !whole(args[10], &sinks) || !flag(args[11], &causal) || !flag(args[13], &with_lse) || !caches(kc, vc, dev) ||
      !table_rows(tables, dev))
    Py_RETURN_NONE;
  const at::Tensor* pb = nullptr;
  if (args[3] != Py_None) {
    if ((pb = plain(args[3])) == nullptr || pb->dim() != 1 || !ints(*pb, pb->size(0), dev)) Py_RETURN_NONE;
  }
  const int64_t hk = kc.size(1), block = kc.size(2), D = kc.size(3), R = tables.size(0), M = tables.size(1);
  if (prefix < 0 || prefix > 0x7fffffff || (prefix > 0 && (pb == nullptr || prefix > pb->size(0) * block)) ||
      window < 0 || window > 0x7fffffff || sinks < 0 || sinks > 0x7fffffff || q.dim() != 3 || q.size(2) != D ||
      q.scalar_type() != kc.scalar_type() || q.get_device() != dev || q.size(0) > 0x7fffffff || q.size(1) <= 0 ||
      q.size(1) > 1024 || q.size(1) % hk != 0 || q.stride(2) != 1 || ((q.stride(0) | q.stride(1)) & 7) != 0 ||
      wants_grad(q) || !ints(lengths, R, dev) || !ints(starts, R + 1, dev))
    Py_RETURN_NONE;
  for (const at::Tensor* x : {&kc, &vc})
    if (!aligned(*x) || ((x->stride(0) | x->stride(1) | x->stride(2)) & 7) != 0) Py_RETURN_NONE;
  if (!aligned(q)) Py_RETURN_NONE;
  const int64_t T = q.size(0), H = q.size(1);
  at::Tensor out;
  const bool fill = args[12] == Py_None;
  if (!fill) {
    const at::Tensor* o = plain(args[12]);
    if (o == nullptr || o->dim() != 2 || o->size(0) != T || o->size(1) != H * D ||
        o->scalar_type() != q.scalar_type() || o->get_device() != dev || !o->is_contiguous() || !aligned(*o))
      Py_RETURN_NONE;
    out = *o;
  }
  const int32_t i_t = static_cast<int32_t>(T), i_r = static_cast<int32_t>(R), i_h = static_cast<int32_t>(H),
                i_hk = static_cast<int32_t>(hk), i_d = static_cast<int32_t>(D), i_m = static_cast<int32_t>(M),
                i_b = static_cast<int32_t>(block), i_p = static_cast<int32_t>(prefix),
                i_w = static_cast<int32_t>(window), i_s = static_cast<int32_t>(sinks);
  const int64_t need = g.paged_workspace(i_t, i_r, i_h, i_hk, i_d, i_m, i_b, i_p, i_w, i_s, causal ? 1 : 0);
  if (need < 0) Py_RETURN_NONE;
  at::Tensor counters;
  if (need > 0) {
    Ref index(PyLong_FromLong(dev)), handle(PyLong_FromVoidPtr(stream));
    Ref key(PyTuple_Pack(2, index.p, handle.p));
    PyObject* const o = key.p != nullptr ? PyDict_GetItem(g.paged_counters, key.p) : nullptr;
    if (o == nullptr || !THPVariable_Check(o)) Py_RETURN_NONE;
    counters = THPVariable_Unpack(o);
  }
  const auto options = q.options().requires_grad(false);
  at::Tensor lse, workspace;
  if (fill) out = at::empty({T, H * D}, options);
  if (with_lse) lse = at::empty({H, T}, options.dtype(at::kFloat));
  if (need > 0) workspace = at::empty({need}, options.dtype(at::kByte));
  int32_t code;
  Py_BEGIN_ALLOW_THREADS
  code = g.paged_attention(q.data_ptr(), q.stride(0), q.stride(1), kc.data_ptr(), vc.data_ptr(), kc.stride(0),
                           kc.stride(1), kc.stride(2), vc.stride(0), vc.stride(1), vc.stride(2), i32(tables),
                           tables.stride(0), i32(lengths), i32(starts), prefix > 0 ? i32(*pb) : nullptr, i_p,
                           out.data_ptr(), with_lse ? static_cast<float*>(lse.data_ptr()) : nullptr, i_t, i_r, i_m,
                           static_cast<int32_t>(kc.size(0)), i_h, i_hk, i_d, i_b, i_w, i_s, causal ? 1 : 0,
                           code_of(q.scalar_type()), static_cast<float>(scale), fill ? 1 : 0,
                           need > 0 ? workspace.data_ptr() : nullptr, need,
                           need > 0 ? counters.data_ptr() : nullptr, stream);
  Py_END_ALLOW_THREADS
  if (code != HKV_OK) Py_RETURN_NONE;
  if (!fill) {
    if (!with_lse) {
      Py_INCREF(args[12]);
      return args[12];
    }
    Ref l(THPVariable_Wrap(lse));
    return l.p != nullptr ? PyTuple_Pack(2, args[12], l.p) : nullptr;
  }
  return with_lse ? tuple_of({out, lse}) : THPVariable_Wrap(out);
}

// torch's exceptions (out of memory among them) end at this boundary: the
// Python body then runs and meets them itself.
template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t n) {
  try {
    return F(args, n);
  } catch (const std::exception&) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

// A prototype as compiled here: return and argument types, i int32, l int64,
// f float, p pointer.
template <typename T>
constexpr char type_code() {
  if (std::is_pointer<T>::value) return 'p';
  if (std::is_same<T, float>::value) return 'f';
  return sizeof(T) == 8 ? 'l' : 'i';
}
template <typename R, typename... A>
std::string prototype(R (*)(A...)) {
  return {type_code<R>(), type_code<A>()...};
}

// prototypes(): those of init's entry points, in its order.
PyObject* prototypes(PyObject*, PyObject*) {
  const std::string p[10] = {prototype(g.attention),    prototype(g.attention_split), prototype(g.split_bytes),
                             prototype(g.item_shape),   prototype(g.produce),         prototype(g.pack),
                             prototype(g.paged_tables), prototype(g.paged_append),    prototype(g.paged_attention),
                             prototype(g.paged_workspace)};
  return Py_BuildValue("(ssssssssss)", p[0].c_str(), p[1].c_str(), p[2].c_str(), p[3].c_str(), p[4].c_str(),
                       p[5].c_str(), p[6].c_str(), p[7].c_str(), p[8].c_str(), p[9].c_str());
}

// init(addresses, env, knobs, workspaces, devices, paged_counters)
PyObject* init(PyObject*, PyObject* args) {
  unsigned long long a[10];
  PyObject *env, *knobs, *workspaces, *devices, *counters;
  if (!PyArg_ParseTuple(args, "(KKKKKKKKKK)O!O!O!O!O!", a, a + 1, a + 2, a + 3, a + 4, a + 5, a + 6, a + 7, a + 8,
                        a + 9, &PyDict_Type, &env, &PyTuple_Type, &knobs, &PyDict_Type, &workspaces, &PyDict_Type,
                        &devices, &PyDict_Type, &counters))
    return nullptr;
  if (!g.ready) {
    g.attention = reinterpret_cast<decltype(g.attention)>(a[0]);
    g.attention_split = reinterpret_cast<decltype(g.attention_split)>(a[1]);
    g.split_bytes = reinterpret_cast<decltype(g.split_bytes)>(a[2]);
    g.item_shape = reinterpret_cast<decltype(g.item_shape)>(a[3]);
    g.produce = reinterpret_cast<decltype(g.produce)>(a[4]);
    g.pack = reinterpret_cast<decltype(g.pack)>(a[5]);
    g.paged_tables = reinterpret_cast<decltype(g.paged_tables)>(a[6]);
    g.paged_append = reinterpret_cast<decltype(g.paged_append)>(a[7]);
    g.paged_attention = reinterpret_cast<decltype(g.paged_attention)>(a[8]);
    g.paged_workspace = reinterpret_cast<decltype(g.paged_workspace)>(a[9]);
    for (PyObject* o : {env, knobs, workspaces, devices, counters}) Py_INCREF(o);
    g.env = env;
    g.knobs = knobs;
    g.workspaces = workspaces;
    g.devices = devices;
    g.paged_counters = counters;
    g.plan_queries = PyUnicode_InternFromString("hkv_queries_per_item");
    g.plan_shape = PyUnicode_InternFromString("hkv_plan_shape");
    g.ready = g.plan_queries != nullptr && g.plan_shape != nullptr;
  }
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<attention_call>)),
     METH_FASTCALL, "The attention operator's launch, or None"},
    {"produce", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<produce_call>)), METH_FASTCALL,
     "The QKV producer's launch, or None"},
    {"pack", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<pack_call>)), METH_FASTCALL,
     "The slab pack's launch, or None"},
    {"paged_tables", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<paged_tables_call>)),
     METH_FASTCALL, "The paged tables' launch, or None"},
    {"paged_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<paged_append_call>)),
     METH_FASTCALL, "The paged append's launch, or None"},
    {"paged_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<paged_attention_call>)),
     METH_FASTCALL, "The paged attention's launch, or None"},
    {"prototypes", prototypes, METH_NOARGS, "The entry points' prototypes as compiled, in init's order"},
    {"init", init, METH_VARARGS, "init(addresses, env, knobs, workspaces, devices, paged_counters)"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_op_call", "Native call path of the operators", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__op_call() { return PyModule_Create(&module); }
