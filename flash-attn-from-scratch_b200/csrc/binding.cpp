// binding.cpp — the Python calls of the serving operators, as a CPython extension over the C ABI.
//
// A decode step makes several small calls per layer, and their checks cost more than their
// kernels when Python makes them attribute by attribute.  Here a tensor's pointer, shape,
// strides, type and device come from torch's DLPack exchange functions (a capsule of C function
// pointers, so nothing is linked to torch), are checked, and go to the C ABI.  The functions
// raise what the Python layer raises (LKInputError, LKError), and return None where a tensor's
// layout is not one that the kernels read: the Python layer then copies and calls again.
#define PY_SSIZE_T_CLEAN
#include <ATen/dlpack.h>
#include <Python.h>

#include <cstdint>
#include <cstring>
#include <map>
#include <utility>

#include "../../include/llm_kernels_b200.h"

namespace {

const DLPackExchangeAPI* g_api = nullptr;
PyObject* g_tensor = nullptr;     // torch.Tensor
PyObject* g_empty_like = nullptr;
PyObject* g_new_lse = nullptr;    // (q, shape) -> fp32 tensor
PyObject* g_capturing = nullptr;  // (device index) -> bool: of the current stream there
PyObject* g_zeros = nullptr;      // (device index, bytes) -> uint8 tensor
PyObject* g_input_error = nullptr;
PyObject* g_call_error = nullptr;  // (name, status, detail) -> exception

struct Fail {};

[[noreturn]] void refuse(const char* msg) {
  PyErr_SetString(g_input_error, msg);
  throw Fail{};
}
inline void require(bool ok, const char* msg) {
  if (!ok) refuse(msg);
}

struct Tensor : DLTensor {
  PyObject* obj = nullptr;
  int64_t size(int i) const { return shape[i]; }
  // A dim of one element has no stride of its own.
  int64_t stride(int i) const { return shape[i] == 1 ? 0 : strides[i]; }
  bool is(int code, int bits) const { return dtype.code == code && dtype.bits == bits && dtype.lanes == 1; }
  bool half() const { return is(kDLFloat, 16) || is(kDLBfloat, 16); }
  bool index() const { return is(kDLInt, 32) || is(kDLInt, 64); }
  int code() const {
    return dtype.code == kDLBfloat ? LK_BF16
           : dtype.code == kDLFloat ? (dtype.bits == 16 ? LK_F16 : LK_F32)
                                    : (dtype.bits == 32 ? LK_I32 : LK_I64);
  }
  bool same_type(const Tensor& o) const { return dtype.code == o.dtype.code && dtype.bits == o.dtype.bits; }
  uint8_t* ptr() const { return static_cast<uint8_t*>(data) + byte_offset; }
  bool flat(int i) const { return stride(i) == 1 || shape[i] == 1; }
};

Tensor tensor(PyObject* o, const char* msg) {
  if (!PyObject_TypeCheck(o, reinterpret_cast<PyTypeObject*>(g_tensor))) refuse(msg);
  Tensor t;
  if (g_api->dltensor_from_py_object_no_sync(o, &t)) throw Fail{};
  t.obj = o;
  return t;
}
void on_cuda(const char* msg, const Tensor& t) { require(t.device.device_type == kDLCUDA, msg); }
void same_device(const Tensor& a, const Tensor& b) {
  require(a.device.device_type == b.device.device_type && a.device.device_id == b.device.device_id,
          "all inputs must be on the same device");
}

void check(const char* name, int status) {
  if (status == LK_OK) return;
  PyObject* e = PyObject_CallFunction(g_call_error, "sii", name, status, status == LK_ERR_CUDA ? lk_last_cuda_error() : 0);
  if (e) PyErr_SetObject(reinterpret_cast<PyObject*>(Py_TYPE(e)), e);
  Py_XDECREF(e);
  throw Fail{};
}

bool flag(PyObject* o) {
  const int yes = PyObject_IsTrue(o);
  if (yes < 0) throw Fail{};
  return yes != 0;
}

void* stream_on(const Tensor& t) {
  check("lk_set_device", lk_set_device(t.device.device_id));  // for the default stream, which names none
  void* s = nullptr;
  if (g_api->current_work_stream(kDLCUDA, t.device.device_id, &s)) throw Fail{};
  return s;
}

// A reference that is dropped unless it is handed out.
struct Ref {
  PyObject* o;
  explicit Ref(PyObject* x) : o(x) {
    if (!x) throw Fail{};
  }
  ~Ref() { Py_XDECREF(o); }
  PyObject* give() { return std::exchange(o, nullptr); }
  Ref(const Ref&) = delete;
};

PyObject* like(PyObject* t) { return PyObject_CallOneArg(g_empty_like, t); }

// Positions, table and axes of the rotation, in the order of the C entry points.
struct Angles {
  const void* positions = nullptr;
  int pos_type = 0;
  int64_t pos_strides[3] = {0, 0, 0};
  const float* table = nullptr;
  int64_t rows = 0, pairs = 0, axes = 0;
  int64_t sections[4] = {0, 0, 0, 0};
};

// lead: the tokens' shape, of one or two dims.  Returns false where positions would have to be
// broadcast first.
bool angles(Angles& a, PyObject* positions, PyObject* table, PyObject* sections, const int64_t* lead, int nlead, int64_t D,
            const Tensor& dev) {
  const Tensor p = tensor(positions, "positions must be an int32 / int64 tensor");
  require(p.index(), "positions must be an int32 / int64 tensor");
  const Tensor t = tensor(table, "cos_sin must be a contiguous fp32 [positions, pairs, 2] tensor");
  require(t.is(kDLFloat, 32) && t.ndim == 3 && t.size(2) == 2 && t.flat(2) && (t.size(1) == 1 || t.strides[1] == 2) &&
              (t.size(0) == 1 || t.strides[0] == 2 * t.size(1)),
          "cos_sin must be a contiguous fp32 [positions, pairs, 2] tensor");
  on_cuda("inputs must be CUDA tensors (this library has no CPU path)", p);
  same_device(p, dev);
  same_device(t, dev);
  a.rows = t.size(0), a.pairs = t.size(1);
  require(a.rows > 0 && a.pairs > 0 && 2 * a.pairs <= D, "cos_sin turns more values than a head has, or has no row");
  int first = 0;
  if (sections == Py_None) {
    a.axes = 1;
    bool same = p.ndim == nlead;
    for (int i = 0; same && i < nlead; ++i) same = p.size(i) == lead[i];
    if (!same) return false;
  } else {
    const char* msg = "sections must be 1 to 4 counts of pairs whose sum is cos_sin's";
    require(PyTuple_Check(sections), msg);
    a.axes = PyTuple_GET_SIZE(sections);
    require(a.axes >= 1 && a.axes <= 4, msg);
    int64_t sum = 0;
    for (int i = 0; i < a.axes; ++i) {
      PyObject* s = PyTuple_GET_ITEM(sections, i);
      require(PyLong_Check(s), msg);
      a.sections[i] = PyLong_AsLongLong(s);
      if (a.sections[i] == -1 && PyErr_Occurred()) PyErr_Clear();
      require(a.sections[i] >= 0 && a.sections[i] <= a.pairs, msg);
      sum += a.sections[i];
    }
    require(sum == a.pairs, msg);
    bool same = p.ndim == nlead + 1 && p.size(0) == a.axes;
    for (int i = 0; same && i < nlead; ++i) same = p.size(1 + i) == lead[i];
    require(same, "with sections, positions must be [axes, tokens...]");
    a.pos_strides[0] = p.stride(0);
    first = 1;
  }
  if (nlead == 2) a.pos_strides[1] = p.stride(first);
  a.pos_strides[2] = p.stride(first + nlead - 1);
  a.positions = p.ptr();
  a.pos_type = p.code();
  a.table = reinterpret_cast<const float*>(t.ptr());
  return true;
}

template <class F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const Fail&) {
    return nullptr;
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "llm_kernels: a C++ exception in a call");
    return nullptr;
  }
}

bool count(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
  return false;
}

// rotary(q, k, positions, cos_sin, sections, interleaved, inverse) -> (q', k'); q or k may be None
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!count(n, 7)) return nullptr;
  return guarded([&]() -> PyObject* {
    Tensor x[2];
    bool have[2];
    for (int i = 0; i < 2; ++i)
      if ((have[i] = a[i] != Py_None)) x[i] = tensor(a[i], "q and k must be tensors");
    const Tensor& q = have[0] ? x[0] : x[1];
    require(have[0] || have[1], "q and k must be tensors");
    require(q.half(), "q must be an fp16 / bf16 tensor");
    require(q.ndim == 3 || q.ndim == 4, "q must be [S, H, D] or [B, S, H, D]");
    const int nd = q.ndim;
    on_cuda("rotary_embed: inputs must be CUDA tensors (this library has no CPU path)", q);
    if (have[0] && have[1]) {
      bool same = x[1].same_type(q) && x[1].ndim == nd && x[1].size(nd - 1) == q.size(nd - 1);
      for (int i = 0; same && i < nd - 2; ++i) same = x[1].size(i) == q.size(i);
      require(same, "k must have q's dtype, tokens and head dim");
      same_device(x[1], q);
    }
    const int64_t D = q.size(nd - 1);
    const bool interleaved = flag(a[5]), inverse = flag(a[6]);
    Angles g;
    if (!angles(g, a[2], a[3], a[4], q.shape, nd - 2, D, q)) Py_RETURN_NONE;
    for (int i = 0; i < 2; ++i)
      if (have[i] && !x[i].flat(nd - 1)) Py_RETURN_NONE;
    PyObject* none = Py_None;
    Ref out[2] = {Ref(have[0] ? like(a[0]) : Py_NewRef(none)), Ref(have[1] ? like(a[1]) : Py_NewRef(none))};
    int64_t strides[12] = {0}, heads[2] = {0, 0};
    void* ptrs[4] = {nullptr, nullptr, nullptr, nullptr};
    for (int i = 0; i < 2; ++i) {
      if (!have[i]) continue;
      const Tensor y = tensor(out[i].o, "");
      if (!y.flat(nd - 1)) refuse("q and k must have a contiguous last dim");
      heads[i] = x[i].size(nd - 2);
      ptrs[2 * i] = x[i].ptr(), ptrs[2 * i + 1] = y.ptr();
      int64_t* st = strides + 6 * i;
      st[0] = nd == 4 ? x[i].stride(0) : 0, st[1] = x[i].stride(nd - 3), st[2] = x[i].stride(nd - 2);
      st[3] = nd == 4 ? y.stride(0) : 0, st[4] = y.stride(nd - 3), st[5] = y.stride(nd - 2);
    }
    check("lk_rotary_embed",
          lk_rotary_embed(ptrs[0], ptrs[1], ptrs[2], ptrs[3], strides, q.code(), nd == 4 ? q.size(0) : 1, q.size(nd - 3),
                          heads[0], heads[1], D, g.positions, g.pos_type, g.pos_strides, g.table, g.rows, g.pairs, g.axes,
                          g.sections, interleaved, inverse, stream_on(q)));
    PyObject* r = PyTuple_New(2);
    if (!r) throw Fail{};
    PyTuple_SET_ITEM(r, 0, out[0].give());
    PyTuple_SET_ITEM(r, 1, out[1].give());
    return r;
  });
}

// Strides of a cache: one page, row or head has none of its own (a positive one for the kernels).
void cache_strides(const Tensor& c, int64_t* st) {
  for (int i = 0; i < 3; ++i) st[i] = c.shape[i] == 1 ? 64 : c.strides[i];
}

void check_caches(const Tensor& k, const Tensor& v, const Tensor& like) {
  bool same = k.ndim == 4 && v.ndim == 4;
  for (int i = 0; same && i < 4; ++i) same = k.size(i) == v.size(i);
  require(same, "k_cache and v_cache must be [num_pages, page_size, H_kv, D], of one shape");
  require(k.same_type(like) && v.same_type(like), "the caches must have the dtype of the tokens");
  require(k.flat(3) && v.flat(3), "the caches' last dim must be contiguous");
  require(k.size(0) > 0 && k.size(1) > 0, "the caches must have a page, and a page a row");
}

// append(k, v, k_cache, v_cache, slots, q, positions, cos_sin, sections, interleaved, q_out) -> q'
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!count(n, 11)) return nullptr;
  return guarded([&]() -> PyObject* {
    const char* kv = "k and v must be fp16 / bf16 [T, H_kv, D], of one shape and dtype";
    const Tensor k = tensor(a[0], kv), v = tensor(a[1], kv);
    require(k.ndim == 3 && k.half() && v.ndim == 3 && v.same_type(k) && v.size(0) == k.size(0) && v.size(1) == k.size(1) &&
                v.size(2) == k.size(2),
            kv);
    const char* caches = "k_cache and v_cache must be [num_pages, page_size, H_kv, D], of one shape";
    const Tensor kc = tensor(a[2], caches), vc = tensor(a[3], caches);
    check_caches(kc, vc, k);
    const int64_t T = k.size(0), Hk = k.size(1), D = k.size(2);
    require(kc.size(2) == Hk && kc.size(3) == D, "the caches' H_kv and D must be those of k");
    const Tensor slots = tensor(a[4], "slots must be int32 / int64 [T]");
    require(slots.index() && slots.ndim == 1 && slots.size(0) == T, "slots must be int32 / int64 [T]");
    require((a[6] == Py_None) == (a[7] == Py_None), "positions and cos_sin go together");
    require(a[5] != Py_None || a[10] == Py_None, "q_out needs q");
    on_cuda("paged_kv_append: inputs must be CUDA tensors (this library has no CPU path)", k);
    same_device(v, k), same_device(kc, k), same_device(vc, k), same_device(slots, k);
    Tensor q, qo;
    const bool with_q = a[5] != Py_None;
    if (with_q) {
      require(a[7] != Py_None, "q is passed to be rotated: positions and cos_sin are needed");
      q = tensor(a[5], "q must be [T, H, D] with k's dtype and device");
      require(q.ndim == 3 && q.same_type(k) && q.size(0) == T && q.size(2) == D && q.device.device_type == k.device.device_type &&
                  q.device.device_id == k.device.device_id,
              "q must be [T, H, D] with k's dtype and device");
      if (a[10] != Py_None) {
        const char* msg = "q_out must match q, both with a contiguous last dim";
        qo = tensor(a[10], msg);
        require(qo.ndim == 3 && qo.same_type(q) && qo.size(0) == T && qo.size(1) == q.size(1) && qo.size(2) == D && qo.flat(2) &&
                    q.flat(2) && qo.device.device_type == q.device.device_type && qo.device.device_id == q.device.device_id,
                msg);
      }
    }
    const bool interleaved = flag(a[9]);
    Angles g;
    if (a[7] != Py_None && !angles(g, a[6], a[7], a[8], k.shape, 1, D, k)) Py_RETURN_FALSE;
    if (!k.flat(2) || !v.flat(2) || !(slots.stride(0) == 1 || T <= 1) || (with_q && !q.flat(2))) Py_RETURN_FALSE;
    PyObject* none = Py_None;
    Ref out(!with_q ? Py_NewRef(none) : a[10] != Py_None ? Py_NewRef(a[10]) : like(a[5]));
    if (with_q && a[10] == Py_None) qo = tensor(out.o, "");
    int64_t st[14] = {0};
    if (with_q) st[0] = q.stride(0), st[1] = q.stride(1), st[2] = qo.stride(0), st[3] = qo.stride(1);
    st[4] = k.stride(0), st[5] = k.stride(1), st[6] = v.stride(0), st[7] = v.stride(1);
    cache_strides(kc, st + 8);
    cache_strides(vc, st + 11);
    check("lk_paged_kv_append",
          lk_paged_kv_append(with_q ? q.ptr() : nullptr, with_q ? qo.ptr() : nullptr, k.ptr(), v.ptr(), kc.ptr(), vc.ptr(), st,
                             k.code(), T, with_q ? q.size(1) : 0, Hk, D, kc.size(0), kc.size(1), slots.ptr(), slots.code(),
                             g.positions, g.pos_type, g.pos_strides, g.table, g.rows, g.pairs, g.axes, g.sections,
                             interleaved, stream_on(k)));
    return out.give();
  });
}

// (device, stream) -> workspace: the partial sums of sequences whose keys are shared among blocks,
// and the counters of their joins, which every call leaves at zero.  Calls on one stream follow one
// another, so they share it.
struct Workspace {
  PyObject* tensor;
  uint8_t* ptr;
  int64_t bytes;
};
std::map<std::pair<int, void*>, Workspace>& workspaces() {
  static auto* m = new std::map<std::pair<int, void*>, Workspace>;
  return *m;
}

// attention(q, k_cache, v_cache, prefix_pages, prefix_length, block_table, lengths, scale, out, return_lse)
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (!count(n_args, 10)) return nullptr;
  return guarded([&]() -> PyObject* {
    const char* qm = "q must be fp16 / bf16 [B, H, D] or [B, n, H, D]";
    const Tensor q = tensor(a[0], qm);
    require(q.half() && (q.ndim == 3 || q.ndim == 4), qm);
    const bool single = q.ndim == 3;
    const int nd = q.ndim;
    const int64_t B = q.size(0), n = single ? 1 : q.size(1), H = q.size(nd - 2), D = q.size(nd - 1);
    const char* cm = "k_cache and v_cache must be [num_pages, page_size, H_kv, D], of one shape";
    const Tensor kc = tensor(a[1], cm), vc = tensor(a[2], cm);
    check_caches(kc, vc, q);
    const int64_t Hk = kc.size(2);
    require(kc.size(3) == D, "the caches' D must be q's");
    require(Hk > 0 && H % Hk == 0, "H_kv must divide H");
    require(D % 8 == 0 && 8 <= D && D <= 128, "head dim must be a multiple of 8 up to 128");
    const Tensor table = tensor(a[5], "block_table must be int32 [B, pages]");
    require(table.is(kDLInt, 32) && table.ndim == 2 && table.size(0) == B, "block_table must be int32 [B, pages]");
    const Tensor lengths = tensor(a[6], "lengths must be int32 [B]");
    require(lengths.is(kDLInt, 32) && lengths.ndim == 1 && lengths.size(0) == B, "lengths must be int32 [B]");
    on_cuda("paged attention: inputs must be CUDA tensors (this library has no CPU path)", q);
    same_device(kc, q), same_device(vc, q), same_device(table, q), same_device(lengths, q);
    int64_t st[12];
    cache_strides(kc, st + 6);
    cache_strides(vc, st + 9);
    bool rows16 = reinterpret_cast<uintptr_t>(kc.ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(vc.ptr()) % 16 == 0;
    for (int i = 6; i < 12; ++i) rows16 = rows16 && st[i] % 8 == 0;
    require(rows16, "the caches' rows must start on 16 bytes");
    float scale = 0.f;  // the C ABI's default: D^-0.5
    if (a[7] != Py_None) {
      const double s = PyFloat_AsDouble(a[7]);
      if (s == -1.0 && PyErr_Occurred()) throw Fail{};
      scale = (float)s;
      require(scale > 0.f && scale < __FLT_MAX__, "softmax_scale must be positive and finite");
    }
    int64_t prefix = 0;
    Tensor pages;
    bool copy = false;
    if (a[3] != Py_None) {
      pages = tensor(a[3], "prefix_pages must be int32 [pages]");
      require(pages.is(kDLInt, 32) && pages.ndim == 1, "prefix_pages must be int32 [pages]");
      require(PyLong_Check(a[4]), "prefix_length must be an int >= 0");
      prefix = PyLong_AsLongLong(a[4]);
      if (prefix == -1 && PyErr_Occurred()) PyErr_Clear();
      require(prefix >= 0, "prefix_length must be an int >= 0");
      require(prefix / kc.size(1) + (prefix % kc.size(1) != 0) <= pages.size(0), "prefix_pages holds fewer than prefix_length keys");
      same_device(pages, q);
      copy = copy || !(pages.stride(0) == 1 || pages.size(0) <= 1);
    }
    auto strides_of = [&](const Tensor& t, int64_t* s) {  // (sequence, token, head); whether the kernels take them
      s[0] = t.stride(0), s[1] = single ? 0 : t.stride(1), s[2] = t.stride(nd - 2);
      return t.flat(nd - 1) && s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0 && reinterpret_cast<uintptr_t>(t.ptr()) % 16 == 0;
    };
    copy = copy || !strides_of(q, st) || !(table.stride(1) == 1 || table.size(1) <= 1) || !(lengths.stride(0) == 1 || B <= 1);
    Tensor o;
    if (a[8] != Py_None) {
      const char* om = "out must match q's shape, dtype and device";
      o = tensor(a[8], om);
      bool same = o.ndim == nd && o.same_type(q) && o.device.device_type == q.device.device_type &&
                  o.device.device_id == q.device.device_id;
      for (int i = 0; same && i < nd; ++i) same = o.size(i) == q.size(i);
      require(same, om);
      copy = copy || !strides_of(o, st + 3);
    }
    if (copy) Py_RETURN_NONE;
    Ref out(a[8] != Py_None ? Py_NewRef(a[8]) : like(a[0]));
    if (a[8] == Py_None) {
      o = tensor(out.o, "");
      if (!strides_of(o, st + 3)) refuse("q must have rows on 16 bytes");
    }
    const bool want_lse = flag(a[9]);
    PyObject* none = Py_None;
    Ref lse(want_lse ? PyObject_CallOneArg(g_new_lse, a[0]) : Py_NewRef(none));
    if (B > 0 && n > 0 && H > 0) {
      void* stream = stream_on(q);
      const int64_t need = lk_paged_attention_workspace_bytes(B, n, H, Hk, D, prefix);
      bool capturing = false;
      if (stream) {  // the legacy default stream cannot be captured
        Ref device(PyLong_FromLong(q.device.device_id));
        Ref yes(PyObject_CallOneArg(g_capturing, device.o));
        capturing = yes.o == Py_True;
      }
      Workspace ws{};
      PyObject* own = nullptr;
      if (capturing) {
        // A graph may be replayed beside this stream's other work: it keeps a workspace of its own.
        own = PyObject_CallFunction(g_zeros, "iL", (int)q.device.device_id, (long long)need);
        if (!own) throw Fail{};
        Ref hold(own);
        ws.ptr = tensor(own, "").ptr(), ws.bytes = need;
        hold.give();
      } else {
        Workspace& held = workspaces()[{(int)q.device.device_id, stream}];
        if (held.bytes < need) {
          PyObject* t = PyObject_CallFunction(g_zeros, "iL", (int)q.device.device_id, (long long)need);
          if (!t) throw Fail{};
          Py_XDECREF(held.tensor);
          held = Workspace{t, tensor(t, "").ptr(), need};
        }
        ws = held;
      }
      Ref own_ref(own ? own : Py_NewRef(none));
      float* lse_ptr = want_lse ? reinterpret_cast<float*>(tensor(lse.o, "").ptr()) : nullptr;
      const int32_t *tp = reinterpret_cast<const int32_t*>(table.ptr()), *lp = reinterpret_cast<const int32_t*>(lengths.ptr());
      if (prefix > 0)
        check("lk_shared_prefix_attention",
              lk_shared_prefix_attention(q.ptr(), kc.ptr(), vc.ptr(), reinterpret_cast<const int32_t*>(pages.ptr()), prefix, tp,
                                         table.stride(0), table.size(1), lp, o.ptr(), lse_ptr, st, q.code(), B, n, H, Hk, D,
                                         kc.size(0), kc.size(1), scale, ws.ptr, ws.bytes, stream));
      else
        check("lk_paged_attention",
              lk_paged_attention(q.ptr(), kc.ptr(), vc.ptr(), tp, table.stride(0), table.size(1), lp, o.ptr(), lse_ptr, st,
                                 q.code(), B, n, H, Hk, D, kc.size(0), kc.size(1), scale, ws.ptr, ws.bytes, stream));
    }
    if (!want_lse) return out.give();
    PyObject* r = PyTuple_New(2);
    if (!r) throw Fail{};
    PyTuple_SET_ITEM(r, 0, out.give());
    PyTuple_SET_ITEM(r, 1, lse.give());
    return r;
  });
}

// Drops the workspaces: after a device failure their counters are not to be trusted.
PyObject* drop_workspaces(PyObject*, PyObject*) {
  for (auto& w : workspaces()) Py_XDECREF(w.second.tensor);
  workspaces().clear();
  Py_RETURN_NONE;
}

// setup(torch.Tensor, empty_like, new_lse, capturing, zeros, LKInputError, call_error)
PyObject* setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!count(n, 7)) return nullptr;
  const char* no_api = "llm_kernels: this torch has no usable DLPack exchange functions";
  PyObject* capsule = PyObject_GetAttrString(a[0], "__dlpack_c_exchange_api__");
  if (!capsule) {
    PyErr_SetString(PyExc_ImportError, no_api);
    return nullptr;
  }
  const auto* api = static_cast<const DLPackExchangeAPI*>(PyCapsule_GetPointer(capsule, "dlpack_exchange_api"));
  Py_DECREF(capsule);  // the type holds it
  if (!api) return nullptr;
  if (api->header.version.major != DLPACK_MAJOR_VERSION || !api->dltensor_from_py_object_no_sync || !api->current_work_stream) {
    PyErr_SetString(PyExc_ImportError, no_api);
    return nullptr;
  }
  PyObject** to[] = {&g_tensor, &g_empty_like, &g_new_lse, &g_capturing, &g_zeros, &g_input_error, &g_call_error};
  for (int i = 0; i < 7; ++i) Py_XSETREF(*to[i], Py_NewRef(a[i]));
  g_api = api;
  Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f))
PyMethodDef methods[] = {
    {"setup", FAST(setup), METH_FASTCALL, nullptr},
    {"rotary", FAST(rotary), METH_FASTCALL, nullptr},
    {"append", FAST(append), METH_FASTCALL, nullptr},
    {"attention", FAST(attention), METH_FASTCALL, nullptr},
    {"drop_workspaces", drop_workspaces, METH_NOARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&module); }
