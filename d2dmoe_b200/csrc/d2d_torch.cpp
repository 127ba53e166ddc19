// Native host path of the module forwards: one call from Python per layer call.
//
// A layer call launches two to four kernels that take 20 to 100 us together; prepared in Python
// (attribute walks, argument checks, thirty ctypes conversions: 55 to 60 us) every call below about
// 10k tokens would be bound by the host.  Here the facts that do not change between
// calls (weight addresses, shapes, packed copies) are kept in a plan, and a call only checks that
// the plan still describes the module, allocates the outputs and enters the C ABI.
//
// The plan never serves stale weights: each of its links names the dictionary slot a parameter, a
// sub-module or a packed image sits in, and a call compares what is in the slot now (object, storage
// address, version counter) with what the plan was made from.  A mismatch returns None and the caller
// makes a new plan.  (Writes past the version counter are announced by emptying the image's slot.)
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/CachingHostAllocator.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <memory>
#include <vector>

#include "../../include/d2dmoe.h"

namespace {

struct Link {
  PyObject* dict;      // slot holder; null: roots[root]
  int root;
  PyObject* key;
  PyObject* obj;       // what the slot held when the plan was made
  const void* data;    // tensors: storage address and version counter
  int64_t version;
  bool tensor;
};

struct Plan {
  std::vector<Link> links;
  at::Tensor hold[2];                  // packed router / experts images
  PyObject* marks[2] = {};             // behind the kernels that wrote them (capsules of a Mark), or null
  std::vector<cudaStream_t> users;     // other streams that have waited for those
  const void *wa = nullptr, *wb = nullptr, *rp = nullptr;
  const void *w1 = nullptr, *b1 = nullptr, *wup = nullptr, *w2 = nullptr, *ep = nullptr;
  const void* last_bias = nullptr;
  int64_t d = 0, R = 0, E = 0, H = 0, act = 0;
  at::ScalarType dtype = at::kFloat;
  c10::Device device = c10::Device(c10::kCUDA, 0);
  ~Plan() {
    for (PyObject* m : marks) Py_XDECREF(m);
    for (Link& l : links) {
      Py_XDECREF(l.dict);
      Py_XDECREF(l.key);
      Py_XDECREF(l.obj);
    }
  }
};

constexpr const char* kPlan = "d2dmoe_b200.plan";

void plan_free(PyObject* cap) { delete static_cast<Plan*>(PyCapsule_GetPointer(cap, kPlan)); }

const at::Tensor* tensor_of(PyObject* o) {
  return o != nullptr && THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr;
}

const void* ptr_of(PyObject* o) {
  const at::Tensor* t = tensor_of(o);
  return t ? t->data_ptr() : nullptr;
}

bool still_valid(const Plan& p, PyObject* const* roots) {
  for (const Link& l : p.links) {
    PyObject* now = PyDict_GetItemWithError(l.dict ? l.dict : roots[l.root], l.key);   // borrowed
    if (now != l.obj) return false;
    if (l.tensor) {
      const at::Tensor& t = THPVariable_Unpack(now);
      if (t.data_ptr() != l.data || t._version() != l.version) return false;
    }
  }
  return !PyErr_Occurred();
}

bool capturing(cudaStream_t s) {
  cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
  C10_CUDA_CHECK(cudaStreamIsCapturing(s, &st));
  return st != cudaStreamCaptureStatusNone;
}

// The point of a stream behind the kernels that wrote a packed image.
struct Mark {
  cudaEvent_t event = nullptr;
  cudaStream_t stream = nullptr;
};
constexpr const char* kMark = "d2dmoe_b200.mark";
void mark_free(PyObject* cap) {
  Mark* m = static_cast<Mark*>(PyCapsule_GetPointer(cap, kMark));
  cudaEventDestroy(m->event);
  delete m;
}

// mark(device index) -> Mark of the current stream, or None while it captures (a graph's event means
// nothing outside it)
PyObject* mark(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n == 1, "mark(device index)");
  const auto dev = (c10::DeviceIndex)PyLong_AsLong(a[0]);
  if (PyErr_Occurred()) return nullptr;
  c10::cuda::CUDAGuard guard(dev);
  auto m = std::make_unique<Mark>();
  m->stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  if (capturing(m->stream)) Py_RETURN_NONE;
  C10_CUDA_CHECK(cudaEventCreateWithFlags(&m->event, cudaEventDisableTiming));
  const cudaError_t err = cudaEventRecord(m->event, m->stream);
  if (err != cudaSuccess) cudaEventDestroy(m->event);
  C10_CUDA_CHECK(err);
  return PyCapsule_New(m.release(), kMark, mark_free);
  END_HANDLE_TH_ERRORS
}

// Before `s` reads the image: it comes behind the kernels that wrote it, and the allocator learns that
// `s` uses it.  (A capture cannot depend on work outside it; it starts behind that.)
void wait_for(const Mark* m, const at::Tensor& image, c10::cuda::CUDAStream s) {
  if (s.stream() == m->stream) return;
  C10_CUDA_CHECK(cudaStreamWaitEvent(s.stream(), m->event, 0));
  c10::cuda::CUDACachingAllocator::recordStream(image.storage().data_ptr(), s);
}

// wait_mark(mark, image): the current stream may read the image
PyObject* wait_mark(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const at::Tensor* t = n == 2 ? tensor_of(a[1]) : nullptr;
  TORCH_CHECK(t, "wait_mark(mark, image)");
  const Mark* m = static_cast<const Mark*>(PyCapsule_GetPointer(a[0], kMark));
  if (!m) return nullptr;
  c10::cuda::CUDAGuard guard(t->device());
  const auto s = c10::cuda::getCurrentCUDAStream(t->device().index());
  if (s.stream() != m->stream && !capturing(s.stream())) wait_for(m, *t, s);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

void use_on(Plan& p, c10::cuda::CUDAStream s) {
  const Mark* m[2];
  bool other = false;
  for (int i = 0; i < 2; ++i) {
    m[i] = p.marks[i] ? static_cast<const Mark*>(PyCapsule_GetPointer(p.marks[i], kMark)) : nullptr;
    other |= m[i] && m[i]->stream != s.stream();
  }
  if (!other) return;
  for (cudaStream_t u : p.users)
    if (u == s.stream()) return;
  if (capturing(s.stream())) return;
  for (int i = 0; i < 2; ++i)
    if (m[i]) wait_for(m[i], p.hold[i], s);
  if (p.users.size() >= 16) p.users.clear();
  p.users.push_back(s.stream());
}

// make_plan(links, (wa, wb, router_packed, mark), (w1, b1, w_up, w2, experts_packed, mark), last_bias,
//           act, modules, parameters, attributes)
//   links: sequence of (holder, key); holder = a dict, or 0 / 1 / 2 for the module's own _modules /
//   _parameters / __dict__, which run_layer receives with every call (the plan does not refer to its
//   module)
PyObject* make_plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) {
    PyErr_SetString(PyExc_TypeError, "make_plan takes 8 arguments");
    return nullptr;
  }
  auto p = std::make_unique<Plan>();
  PyObject* const roots[3] = {a[5], a[6], a[7]};
  PyObject* seq = PySequence_Fast(a[0], "links");
  if (!seq) return nullptr;
  for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(seq); ++i) {
    PyObject* it = PySequence_Fast_GET_ITEM(seq, i);
    PyObject* holder = PyTuple_GetItem(it, 0);
    PyObject* key = PyTuple_GetItem(it, 1);
    if (!holder || !key) {
      Py_DECREF(seq);
      return nullptr;
    }
    Link l = {};
    if (PyLong_Check(holder)) {
      l.root = (int)PyLong_AsLong(holder);
      TORCH_CHECK(l.root >= 0 && l.root < 3, "link holder");
    } else {
      Py_INCREF(holder);
      l.dict = holder;
    }
    Py_INCREF(key);
    l.key = key;
    PyObject* now = PyDict_GetItemWithError(l.dict ? l.dict : roots[l.root], key);
    Py_XINCREF(now);
    l.obj = now;
    if (const at::Tensor* t = tensor_of(now)) {
      l.tensor = true;
      l.data = t->data_ptr();
      l.version = t->_version();
    }
    p->links.push_back(l);
  }
  Py_DECREF(seq);
  PyObject *r = a[1], *e = a[2];
  if (r != Py_None) {
    const at::Tensor* wa = tensor_of(PyTuple_GetItem(r, 0));
    TORCH_CHECK(wa, "router weight");
    p->wa = wa->data_ptr();
    p->wb = ptr_of(PyTuple_GetItem(r, 1));
    p->R = wa->size(0);
    if (const at::Tensor* t = tensor_of(PyTuple_GetItem(r, 2))) {
      p->hold[0] = *t;
      p->rp = t->data_ptr();
      if (PyObject* m = PyTuple_GetItem(r, 3); m && m != Py_None) p->marks[0] = Py_NewRef(m);
    }
  }
  const at::Tensor* w1 = tensor_of(PyTuple_GetItem(e, 0));
  TORCH_CHECK(w1 && w1->dim() == 3 && w1->is_cuda(), "expert weights");
  p->w1 = w1->data_ptr();
  p->b1 = ptr_of(PyTuple_GetItem(e, 1));
  p->wup = ptr_of(PyTuple_GetItem(e, 2));
  p->w2 = ptr_of(PyTuple_GetItem(e, 3));
  if (const at::Tensor* t = tensor_of(PyTuple_GetItem(e, 4))) {
    p->hold[1] = *t;
    p->ep = t->data_ptr();
    if (PyObject* m = PyTuple_GetItem(e, 5); m && m != Py_None) p->marks[1] = Py_NewRef(m);
  }
  p->E = w1->size(0);
  p->d = w1->size(1);
  p->H = w1->size(2);
  p->dtype = w1->scalar_type();
  p->device = w1->device();
  p->last_bias = ptr_of(a[3]);
  p->act = PyLong_AsLong(a[4]);
  if (PyErr_Occurred()) return nullptr;
  return PyCapsule_New(p.release(), kPlan, plan_free);
  END_HANDLE_TH_ERRORS
}

// buffers of one call: ops.Workspace of (tokens, experts, device), from a cache of the module's
struct Buffers {
  void *mask, *idx, *off, *ws, *status;
  size_t ws_bytes;
};

PyObject* s_get;      // "raw"

// keep: a list that holds on to it, or null
bool buffers_of(PyObject* cache, const Plan& p, int64_t N, Buffers* b, PyObject* keep = nullptr) {
  // the cache is a dictionary (tokens, experts, device index) -> Workspace with a miss handler, which
  // allocates on the current stream
  PyObject* key = Py_BuildValue("(LLi)", (long long)N, (long long)p.E, (int)p.device.index());
  if (!key) return false;
  PyObject* w = PyDict_GetItemWithError(cache, key);       // borrowed
  PyObject* made = nullptr;
  if (!w && !PyErr_Occurred()) w = made = PyObject_GetItem(cache, key);   // __missing__ allocates
  Py_DECREF(key);
  if (!w) return false;
  PyObject* raw = keep && PyList_Append(keep, w) != 0
                      ? nullptr
                      : PyObject_GetAttr(w, s_get);         // bytes: five addresses and a size
  Py_XDECREF(made);                                         // the cache keeps it
  if (!raw) return false;
  const bool ok = PyBytes_Check(raw) && PyBytes_GET_SIZE(raw) == 48;
  if (ok) {
    uint64_t v[6];
    memcpy(v, PyBytes_AS_STRING(raw), 48);
    *b = {(void*)v[0], (void*)v[1], (void*)v[2], (void*)v[3], (void*)v[4], (size_t)v[5]};
  } else {
    PyErr_SetString(PyExc_TypeError, "workspace addresses");
  }
  Py_DECREF(raw);
  return ok;
}

// run_layer(plan, modules, parameters, attributes, workspaces, x, rule, k, tau, residual, scores, norm,
//           capture)
//   -> (out, routing[, norms]) | status code (int) | None: the plan is stale | False: it is as the module
//   is, but this call takes the general path
// rule: D2D_RULE_*; k / tau as that rule reads them (MAX: threshold 1 - tau).
// scores: None or [.., E] of x's dtype.  norm: None or (kind, gamma, beta|None, eps, gamma_offset):
// x + layer(norm(x)).  capture: None or (norm layer, ord), with D2D_RULE_ALL.
PyObject* run_layer(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 13) {
    PyErr_SetString(PyExc_TypeError, "run_layer takes 13 arguments");
    return nullptr;
  }
  Plan* p = static_cast<Plan*>(PyCapsule_GetPointer(a[0], kPlan));
  if (!p) return nullptr;
  if (!still_valid(*p, a + 1)) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
  }
  const at::Tensor* xp = tensor_of(a[5]);
  if (!xp || !xp->is_cuda() || xp->scalar_type() != p->dtype || xp->device() != p->device ||
      xp->dim() < 1 || xp->size(-1) != p->d || xp->numel() == 0)
    Py_RETURN_FALSE;
  const at::Tensor x = xp->contiguous();
  const int64_t N = x.numel() / p->d;
  const int rule = (int)PyLong_AsLong(a[6]);
  const int k = (int)PyLong_AsLong(a[7]);
  const bool reads_tau = rule == D2D_RULE_MAX || rule == D2D_RULE_DYNK;
  const double tau = reads_tau ? PyFloat_AsDouble(a[8]) : 0.0;
  const int residual = PyObject_IsTrue(a[9]);
  if (PyErr_Occurred()) return nullptr;
  const float mult = (float)(1.0 - tau);
  const bool ranked = rule == D2D_RULE_TOPK || rule == D2D_RULE_DYNK;
  at::Tensor scores, scratch;
  const bool given = a[10] != Py_None;
  if (given) {
    const at::Tensor* sp = tensor_of(a[10]);
    if (!sp || !sp->is_cuda() || sp->scalar_type() != p->dtype || sp->device() != p->device ||
        sp->numel() != N * p->E)
      Py_RETURN_FALSE;
    scores = sp->contiguous();
  } else if (!p->wa && rule != D2D_RULE_ALL) {
    Py_RETURN_FALSE;
  }
  c10::cuda::CUDAGuard guard(p->device);
  const auto cur = c10::cuda::getCurrentCUDAStream(p->device.index());
  const auto stream = (d2d_stream_t)cur.stream();
  Buffers b;
  if (!buffers_of(a[4], *p, N, &b)) return nullptr;
  use_on(*p, cur);
  const int dt = p->dtype == at::kBFloat16 ? D2D_BF16 : D2D_F32;
  const auto opts = x.options();
  at::Tensor out = at::detail::empty_cuda(x.sizes(), opts);
  c10::SmallVector<int64_t, 5> rs(x.sizes().begin(), x.sizes().end());
  rs.back() = p->E;
  at::Tensor rt = at::detail::empty_cuda(rs, opts);
  if (ranked && !given) scratch = at::detail::empty_cuda({N, p->E}, opts);
  const void* xin = x.data_ptr();
  const void* lb = p->last_bias;
  int res = residual ? 1 : 0, rc = D2D_OK;
  at::Tensor xn, norms;
  int norm_layer = 0, norm_ord = 0;
  if (a[12] != Py_None) {
    norm_layer = (int)PyLong_AsLong(PyTuple_GetItem(a[12], 0));
    norm_ord = (int)PyLong_AsLong(PyTuple_GetItem(a[12], 1));
    if (PyErr_Occurred()) return nullptr;
    norms = at::detail::empty_cuda({p->E, N}, opts);
  }
  if (a[11] != Py_None) {
    PyObject* nm = a[11];
    xn = at::detail::empty_cuda(x.sizes(), opts);
    const long kind = PyLong_AsLong(PyTuple_GetItem(nm, 0));
    const double eps = PyFloat_AsDouble(PyTuple_GetItem(nm, 3));
    const double goff = PyFloat_AsDouble(PyTuple_GetItem(nm, 4));
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor* gt = tensor_of(PyTuple_GetItem(nm, 1));
    const at::Tensor* bt = tensor_of(PyTuple_GetItem(nm, 2));
    const auto fits = [&](const at::Tensor* t) {
      return t->numel() == p->d && t->scalar_type() == p->dtype && t->device() == p->device;
    };
    TORCH_CHECK(gt && fits(gt) && (!bt || fits(bt)), "norm parameters: ", p->d,
                " values of x's dtype, on its device");
    const at::Tensor g = gt->contiguous(), bb = bt ? bt->contiguous() : at::Tensor();
    rc = d2d_prenorm_init(xin, g.data_ptr(), bt ? bb.data_ptr() : nullptr, (float)eps, (int)kind,
                          (float)goff, lb, xn.data_ptr(), out.data_ptr(), N, (int)p->d, dt, stream);
    xin = xn.data_ptr();
    lb = nullptr;
    res = D2D_OUT_PREINITIALISED;
  }
  if (rc == D2D_OK)
    rc = d2d_moe_forward_rule(
        xin, given ? nullptr : p->wa, given ? nullptr : p->wb, given ? nullptr : p->rp,
        given ? scores.data_ptr() : nullptr, scratch.defined() ? scratch.data_ptr() : nullptr, rule,
        k, (float)tau, mult, p->w1, p->b1, p->wup, p->w2, p->ep, lb, res, out.data_ptr(),
        (uint32_t*)b.mask, (int32_t*)b.idx, (int32_t*)b.off, N, (int)p->d, (int)p->R, (int)p->E,
        (int)p->H, (int)p->act, dt, b.ws, b.ws_bytes, (int*)b.status, rt.data_ptr(),
        norms.defined() ? norms.data_ptr() : nullptr, norm_layer, norm_ord, stream);
  if (rc != D2D_OK) return PyLong_FromLong(rc);
  const bool has_norms = norms.defined();
  PyObject* res_t = PyTuple_New(has_norms ? 3 : 2);
  if (!res_t) return nullptr;
  PyTuple_SET_ITEM(res_t, 0, THPVariable_Wrap(std::move(out)));
  PyTuple_SET_ITEM(res_t, 1, THPVariable_Wrap(std::move(rt)));
  if (has_norms) PyTuple_SET_ITEM(res_t, 2, THPVariable_Wrap(std::move(norms)));
  return res_t;
  END_HANDLE_TH_ERRORS
}

// ---- host-buffer pipeline -------------------------------------------------------
// Two staging buffers for slices of x, three for slices of the output; the events say when the
// stream that last used one is done with it (never recorded: at once).
constexpr int kIn = 2, kOut = 3;
struct HostPipe {
  int device = 0;
  cudaEvent_t in_full[kIn] = {}, in_free[kIn] = {}, out_full[kOut] = {}, out_free[kOut] = {},
              caller = nullptr;
  unsigned long long n = 0;            // slices so far, over all calls
  std::vector<cudaEvent_t*> all() {
    std::vector<cudaEvent_t*> v = {&caller};
    for (auto& e : in_full) v.push_back(&e);
    for (auto& e : in_free) v.push_back(&e);
    for (auto& e : out_full) v.push_back(&e);
    for (auto& e : out_free) v.push_back(&e);
    return v;
  }
};
constexpr const char* kPipe = "d2dmoe_b200.host_pipe";
void pipe_free(PyObject* cap) {
  auto* h = static_cast<HostPipe*>(PyCapsule_GetPointer(cap, kPipe));
  for (cudaEvent_t* e : h->all())
    if (*e) cudaEventDestroy(*e);
  delete h;
}

PyObject* make_pipe(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n == 1, "make_pipe(device index)");
  auto h = std::make_unique<HostPipe>();
  h->device = (int)PyLong_AsLong(a[0]);
  if (PyErr_Occurred()) return nullptr;
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)h->device);
  for (cudaEvent_t* e : h->all())
    C10_CUDA_CHECK(cudaEventCreateWithFlags(e, cudaEventDisableTiming));
  return PyCapsule_New(h.release(), kPipe, pipe_free);
  END_HANDLE_TH_ERRORS
}

// run_host(plan, modules, parameters, attributes, workspaces, pipe, x_host, out_host,
//          staging (kIn + kOut tensors), (stream in, stream run, stream out), slices, rule, k, tau,
//          residual, sync)
//   -> True | status code (int) | None / False as run_layer
// Slice i's copy in, the kernels of slice i - 1 and the copy out of slice i - 2 overlap.  (Issued from
// Python it takes 70 us of host time per slice, more than a slice's copies.)
PyObject* run_host(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n == 16, "run_host takes 16 arguments");
  Plan* p = static_cast<Plan*>(PyCapsule_GetPointer(a[0], kPlan));
  HostPipe* h = static_cast<HostPipe*>(PyCapsule_GetPointer(a[5], kPipe));
  if (!p || !h) return nullptr;
  if (!still_valid(*p, a + 1)) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
  }
  const at::Tensor *xh = tensor_of(a[6]), *oh = tensor_of(a[7]);
  if (!xh || !oh || xh->scalar_type() != p->dtype || oh->scalar_type() != p->dtype ||
      !xh->is_contiguous() || !oh->is_contiguous() || !oh->is_cpu() || xh->sizes() != oh->sizes() ||
      xh->dim() < 2 || xh->size(-1) != p->d || xh->numel() == 0 || h->device != p->device.index())
    Py_RETURN_FALSE;
  void* stage[kIn + kOut];
  for (int i = 0; i < kIn + kOut; ++i) stage[i] = const_cast<void*>(ptr_of(PyTuple_GetItem(a[8], i)));
  cudaStream_t st[3];
  for (int i = 0; i < 3; ++i) st[i] = (cudaStream_t)PyLong_AsVoidPtr(PyTuple_GetItem(a[9], i));
  const int64_t slices = PyLong_AsLongLong(a[10]);
  const int rule = (int)PyLong_AsLong(a[11]), k = (int)PyLong_AsLong(a[12]);
  const bool reads_tau = rule == D2D_RULE_MAX || rule == D2D_RULE_DYNK;
  const double tau = reads_tau ? PyFloat_AsDouble(a[13]) : 0.0;
  const int residual = PyObject_IsTrue(a[14]), sync = PyObject_IsTrue(a[15]);
  if (PyErr_Occurred()) return nullptr;
  if ((rule != D2D_RULE_ALL && !p->wa) || (rule != D2D_RULE_ALL && rule != D2D_RULE_MAX))
    Py_RETURN_FALSE;
  c10::cuda::CUDAGuard guard(p->device);
  const cudaStream_t cur = c10::cuda::getCurrentCUDAStream(p->device.index()).stream();
  if (sync) {                          // what the caller's stream has queued comes first
    C10_CUDA_CHECK(cudaEventRecord(h->caller, cur));
    for (cudaStream_t s : st) C10_CUDA_CHECK(cudaStreamWaitEvent(s, h->caller, 0));
  }
  const int dt = p->dtype == at::kBFloat16 ? D2D_BF16 : D2D_F32;
  const int64_t B = xh->size(0), per = xh->numel() / B;      // values of one batch entry
  // `workspaces` is the pipeline's own: allocated and used on the stream of the kernels alone, whatever
  // the caller's stream is doing, so that one that leaves the cache is reused in stream order
  const auto run = c10::cuda::getStreamFromExternal(st[1], p->device.index());
  std::vector<Buffers> bufs((size_t)slices);
  THPObjectPtr keep(PyList_New(0));
  if (!keep) return nullptr;
  {
    c10::cuda::CUDAStreamGuard on_run(run);
    for (int64_t i = 0; i < slices; ++i)
      if (!buffers_of(a[4], *p, (B * (i + 1) / slices - B * i / slices) * per / p->d, &bufs[i],
                      keep))
        return nullptr;
  }
  use_on(*p, run);
  // pinned blocks that their owner drops are not handed out again before these copies are done (memory
  // of another origin is none of the allocator's)
  const std::pair<const at::Tensor*, cudaStream_t> used[2] = {{xh, st[0]}, {oh, st[2]}};
  for (const auto& u : used)
    at::getHostAllocator(at::kCUDA)->record_event(
        u.first->data_ptr(), u.first->storage().data_ptr().get_context(),
        c10::cuda::getStreamFromExternal(u.second, p->device.index()).unwrap());
  const size_t es = xh->element_size();
  const char* src = static_cast<const char*>(xh->data_ptr());
  char* dst = static_cast<char*>(oh->data_ptr());
  int rc = D2D_OK;
  for (int64_t i = 0; i < slices && rc == D2D_OK; ++i, ++h->n) {
    const int64_t lo = B * i / slices, hi = B * (i + 1) / slices, N = (hi - lo) * per / p->d;
    const int b = (int)(h->n % kIn), o = (int)(h->n % kOut);
    const size_t bytes = (size_t)((hi - lo) * per) * es, at = (size_t)(lo * per) * es;
    const Buffers& buf = bufs[i];
    C10_CUDA_CHECK(cudaStreamWaitEvent(st[0], h->in_free[b], 0));
    C10_CUDA_CHECK(cudaMemcpyAsync(stage[b], src + at, bytes, cudaMemcpyHostToDevice, st[0]));
    C10_CUDA_CHECK(cudaEventRecord(h->in_full[b], st[0]));
    C10_CUDA_CHECK(cudaStreamWaitEvent(st[1], h->in_full[b], 0));
    C10_CUDA_CHECK(cudaStreamWaitEvent(st[1], h->out_free[o], 0));
    rc = d2d_moe_forward_rule(stage[b], p->wa, p->wb, p->rp, nullptr, nullptr, rule, k, (float)tau,
                              (float)(1.0 - tau), p->w1, p->b1, p->wup, p->w2, p->ep, p->last_bias,
                              residual ? 1 : 0, stage[kIn + o], (uint32_t*)buf.mask,
                              (int32_t*)buf.idx, (int32_t*)buf.off, N, (int)p->d, (int)p->R,
                              (int)p->E, (int)p->H, (int)p->act, dt, buf.ws, buf.ws_bytes,
                              (int*)buf.status, nullptr, nullptr, 0, 0, (d2d_stream_t)st[1]);
    C10_CUDA_CHECK(cudaEventRecord(h->in_free[b], st[1]));
    C10_CUDA_CHECK(cudaEventRecord(h->out_full[o], st[1]));
    C10_CUDA_CHECK(cudaStreamWaitEvent(st[2], h->out_full[o], 0));
    C10_CUDA_CHECK(cudaMemcpyAsync(dst + at, stage[kIn + o], bytes, cudaMemcpyDeviceToHost, st[2]));
    C10_CUDA_CHECK(cudaEventRecord(h->out_free[o], st[2]));
  }
  if (sync) {                          // the last copy out is behind everything else
    cudaError_t err;
    Py_BEGIN_ALLOW_THREADS
    err = cudaStreamSynchronize(st[2]);
    Py_END_ALLOW_THREADS
    C10_CUDA_CHECK(err);
  }
  if (rc != D2D_OK) return PyLong_FromLong(rc);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// ---- norm, routing and weighted experts -------------------------------------------
// One call from Python per operator: arguments are checked, outputs and workspaces allocated on the current stream, the C
// ABI entered.  Each returns its outputs, or the status code (int) of a refused call.

// a tensor argument, which must be on the GPU (and on that of `like`) and without a forward-mode tangent, which the result
// would lose; None: null
const at::Tensor* given(PyObject* o, const char* name, const at::Tensor* like = nullptr) {
  if (o == Py_None) return nullptr;
  const at::Tensor* t = tensor_of(o);
  TORCH_CHECK_TYPE(t, name, " must be a tensor");
  TORCH_CHECK(t->is_cuda(), "d2dmoe_b200 runs on CUDA tensors only (there is no CPU path)");
  TORCH_CHECK_VALUE(!like || t->device() == like->device(), "tensors of one call live on different devices: ",
                    like->device(), " and ", t->device(), " (", name, ")");
  TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(/*level=*/0).defined(), "d2dmoe_b200's operators have no forward-mode derivative (",
                              name, " has a tangent)");
  return t;
}

const at::Tensor& needed(PyObject* o, const char* name, const at::Tensor* like = nullptr) {
  const at::Tensor* t = given(o, name, like);
  TORCH_CHECK_TYPE(t, name, " must be a tensor");
  return *t;
}

int dtype_of(const at::Tensor& t) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16,
                   "d2dmoe_b200 supports float32 and bfloat16, got ", t.scalar_type());
  return t.scalar_type() == at::kBFloat16 ? D2D_BF16 : D2D_F32;
}

void of_type(const at::Tensor& t, at::ScalarType s, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == s, name, " must be ", s, ", got ", t.scalar_type());
}

// [.., d] as rows: a matrix whose rows lie apart by any stride stays as it is, all else that is not contiguous is copied
struct Rows {
  at::Tensor t;
  int64_t n, stride;
};
Rows rows_of(const at::Tensor& t) {
  const int64_t d = t.size(-1);
  if (t.dim() == 2 && (t.stride(1) == 1 || d == 1) && !t.is_contiguous()) return {t, t.size(0), t.stride(0)};
  return {t.contiguous(), d > 0 ? t.numel() / d : 0, d};
}

// the stream, with the tensors' device current
struct On {
  c10::cuda::CUDAGuard guard;
  d2d_stream_t stream;
  explicit On(const at::Tensor& t)
      : guard(t.device()), stream((d2d_stream_t)c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};

void* data_or_null(const at::Tensor* t) { return t && t->defined() ? t->data_ptr() : nullptr; }

PyObject* wrap(at::Tensor t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(t));
}
PyObject* wrap_all(std::initializer_list<at::Tensor> ts) {
  PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
  if (!r) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor& t : ts) {
    PyObject* o = wrap(t);
    if (!o) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

at::Tensor param_of(const at::Tensor* t, const char* name, int64_t d, at::ScalarType x, at::ScalarType* type) {
  if (!t) return {};
  TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == d, name, " must have ", d, " values");
  TORCH_CHECK_TYPE(t->scalar_type() == at::kFloat || t->scalar_type() == x, name,
                   " must be float32 or of x's dtype, got ", t->scalar_type());
  TORCH_CHECK_TYPE(*type == at::ScalarType::Undefined || *type == t->scalar_type(),
                   "weight and bias must be of one dtype");
  *type = t->scalar_type();
  return t->contiguous();
}
int param_code(at::ScalarType t, int x) {
  return t == at::ScalarType::Undefined ? x : t == at::kFloat ? D2D_F32 : D2D_BF16;
}

// The operators themselves, without Python (autograd's threads call them too): status code, outputs by reference.
// (Tensors without rows have no address; arguments are checked all the same.)
void* address(const at::Tensor& t) {
  static double none;
  return t.numel() ? t.data_ptr() : &none;
}

struct NormHow {
  double eps, offset;
  int kind;
};

int norm_forward(const at::Tensor& xt, const at::Tensor* wt, const at::Tensor* bt, const NormHow& h, bool stats,
                 at::Tensor* y, at::Tensor* mean, at::Tensor* rstd) {
  const int dt = dtype_of(xt);
  TORCH_CHECK_VALUE(xt.dim() >= 1 && xt.size(-1) > 0, "x must have rows of one value or more");
  const int64_t d = xt.size(-1);
  at::ScalarType pt = at::ScalarType::Undefined;
  const at::Tensor w = param_of(wt, "weight", d, xt.scalar_type(), &pt);
  const at::Tensor b = param_of(bt, "bias", d, xt.scalar_type(), &pt);
  if (d > D2D_NORM_MAX_D) return D2D_ERR_UNSUPPORTED;
  On on(xt);
  const Rows x = rows_of(xt);
  *y = at::detail::empty_cuda(xt.sizes(), xt.options());
  if (stats) {
    const auto f32 = xt.options().dtype(at::kFloat);
    if (h.kind == D2D_NORM_LAYER) *mean = at::detail::empty_cuda({x.n}, f32);
    *rstd = at::detail::empty_cuda({x.n}, f32);
  }
  return d2d_layer_norm(address(x.t), x.stride, data_or_null(&w), data_or_null(&b), (float)h.eps, h.kind,
                        (float)h.offset, address(*y), x.n ? (float*)data_or_null(mean) : nullptr,
                        x.n ? (float*)data_or_null(rstd) : nullptr, x.n, (int)d, dt, param_code(pt, dt), on.stream);
}

int norm_backward(const at::Tensor& gt, const at::Tensor& xt, const at::Tensor* wt, const at::Tensor* mean,
                  const at::Tensor& rstd, const NormHow& h, const bool (&want)[3], at::Tensor* dx, at::Tensor* dw,
                  at::Tensor* db) {
  const int dt = dtype_of(xt);
  of_type(gt, xt.scalar_type(), "dy");
  TORCH_CHECK_VALUE(xt.dim() >= 1 && xt.size(-1) > 0, "x must have rows of one value or more");
  TORCH_CHECK_VALUE(gt.sizes() == xt.sizes(), "dy must have the shape of x");
  const int64_t d = xt.size(-1);
  at::ScalarType pt = at::ScalarType::Undefined;
  const at::Tensor w = param_of(wt, "weight", d, xt.scalar_type(), &pt);
  if (d > D2D_NORM_MAX_D) return D2D_ERR_UNSUPPORTED;
  On on(xt);
  const Rows x = rows_of(xt), g = rows_of(gt);
  for (const at::Tensor* t : {mean, &rstd})
    if (t) {
      of_type(*t, at::kFloat, "statistics");
      TORCH_CHECK_VALUE(t->numel() == x.n && t->is_contiguous(), "mean and rstd must be contiguous, one value a row");
    }
  TORCH_CHECK_VALUE(h.kind != D2D_NORM_LAYER || mean, "mean is missing");
  const auto po = xt.options().dtype(pt == at::ScalarType::Undefined ? xt.scalar_type() : pt);
  if (want[0]) *dx = at::detail::empty_cuda(xt.sizes(), xt.options());
  if (want[1]) *dw = at::detail::empty_cuda({d}, po);
  if (want[2]) *db = at::detail::empty_cuda({d}, po);
  at::Tensor ws;
  size_t bytes = 0;
  if (want[1] || want[2]) {
    const int rc = d2d_layer_norm_workspace_bytes(x.n, (int)d, &bytes);
    if (rc != D2D_OK) return rc;
    ws = at::detail::empty_cuda({(int64_t)std::max<size_t>(bytes, 16)}, xt.options().dtype(at::kByte));
  }
  return d2d_layer_norm_backward(address(g.t), g.stride, address(x.t), x.stride, data_or_null(&w), h.kind,
                                 (float)h.offset, mean ? (const float*)address(*mean) : nullptr,
                                 (const float*)address(rstd), x.n ? data_or_null(dx) : nullptr, data_or_null(dw),
                                 data_or_null(db), x.n, (int)d, dt, param_code(pt, dt), data_or_null(&ws), bytes,
                                 on.stream);
}

struct RouteHow {
  int64_t k, scores, groups, top;
  bool renormalise;
  double scale;
};

int route_forward(const at::Tensor& lt, const at::Tensor* bt, const RouteHow& h, const at::Tensor* mask, bool dense,
                  at::Tensor* w, at::Tensor* e, at::Tensor* rt) {
  const int dt = dtype_of(lt);
  TORCH_CHECK_VALUE(lt.dim() >= 1 && lt.size(-1) > 0, "logits must have one expert or more");
  const int64_t E = lt.size(-1), N = lt.numel() / E;
  if (E > (1 << 20)) return D2D_ERR_UNSUPPORTED;
  if (h.k < 0 || h.k > E || h.groups < 0 || h.groups > E || h.top < 0 || h.top > E) return D2D_ERR_BAD_ARG;
  On on(lt);
  at::Tensor bias;
  if (bt) {
    of_type(*bt, at::kFloat, "bias");
    TORCH_CHECK_VALUE(bt->dim() == 1 && bt->size(0) == E, "bias must have ", E, " values");
    bias = bt->contiguous();
  }
  if (mask)
    TORCH_CHECK_VALUE(mask->is_contiguous() && mask->element_size() == 4 && mask->numel() >= N * ((E + 31) / 32),
                      "mask bits: room for [tokens, ceil(experts / 32)] words");
  const at::Tensor logits = lt.contiguous();
  c10::SmallVector<int64_t, 5> shape(lt.sizes().begin(), lt.sizes().end());
  shape.back() = h.k;
  *w = at::detail::empty_cuda(shape, lt.options().dtype(at::kFloat));
  *e = at::detail::empty_cuda(shape, lt.options().dtype(at::kInt));
  if (dense) *rt = at::detail::empty_cuda(lt.sizes(), lt.options());
  return d2d_route(address(logits), (const float*)data_or_null(&bias), (int)h.scores, (int)h.k, (int)h.groups,
                   (int)h.top, h.renormalise, (float)h.scale, (int32_t*)address(*e), (float*)address(*w),
                   (uint32_t*)data_or_null(mask), data_or_null(rt), N, (int)E, dt, on.stream);
}

int route_gradient(const at::Tensor& gt, const at::Tensor& lt, const at::Tensor& et, const at::Tensor& wt,
                   const RouteHow& h, at::Tensor* out) {
  const int dt = dtype_of(lt);
  of_type(gt, at::kFloat, "dweights");
  of_type(wt, at::kFloat, "weights");
  of_type(et, at::kInt, "experts");
  TORCH_CHECK_VALUE(lt.dim() >= 1 && lt.size(-1) > 0, "logits must have one expert or more");
  const int64_t E = lt.size(-1), N = lt.numel() / E;
  TORCH_CHECK_VALUE(et.dim() == lt.dim() && et.sizes().slice(0, et.dim() - 1) == lt.sizes().slice(0, lt.dim() - 1) &&
                        wt.sizes() == et.sizes() && gt.sizes() == et.sizes(),
                    "experts, weights and dweights must be [.., k] for logits [.., experts]");
  const int64_t k = et.size(-1);
  if (E > (1 << 20) || k > E) return k > E ? D2D_ERR_BAD_ARG : D2D_ERR_UNSUPPORTED;
  On on(lt);
  const at::Tensor logits = lt.contiguous(), e = et.contiguous(), w = wt.contiguous(), g = gt.contiguous();
  *out = at::detail::empty_cuda(lt.sizes(), lt.options());
  return d2d_route_backward(address(logits), (const int32_t*)address(e), (const float*)address(w),
                            (const float*)address(g), (int)h.scores, h.renormalise, (float)h.scale, address(*out), N,
                            (int)E, (int)k, dt, on.stream);
}

// ---- the same under autograd ----------------------------------------------------------
// First derivatives only: where the gradients' own graph is asked for, differentiating it says so, whatever the incoming
// gradient is made of (the second derivative in the operator's own input would be left out without a word).
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

variable_list once(variable_list grads, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  for (at::Tensor& g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  auto error = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " has first derivatives only",
                                                               (int64_t)grads.size());
  return (*error)(std::move(grads));
}

struct NormFunction : torch::autograd::Function<NormFunction> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const std::optional<at::Tensor>& w,
                            const std::optional<at::Tensor>& b, const NormHow& h) {
    at::Tensor y, mean, rstd;
    const int rc = norm_forward(x, w ? &*w : nullptr, b ? &*b : nullptr, h, true, &y, &mean, &rstd);
    TORCH_CHECK(rc == D2D_OK, "d2d_layer_norm: ", d2d_strerror(rc));
    ctx->save_for_backward({x, w ? *w : at::Tensor(), mean, rstd});
    ctx->saved_data["how"] = std::vector<double>{h.eps, h.offset, (double)h.kind, b ? 1.0 : 0.0};
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list s = ctx->get_saved_variables();
    const auto how = ctx->saved_data["how"].toDoubleVector();
    const NormHow h = {how[0], how[1], (int)how[2]};
    const bool weight = s[1].defined(), bias = how[3] != 0.0;      // (only tensors that are there are counted)
    const bool want[3] = {ctx->needs_input_grad(0), weight && ctx->needs_input_grad(1),
                          bias && ctx->needs_input_grad(weight ? 2 : 1)};
    variable_list out(4);
    if (!g[0].defined()) return out;
    const int rc = norm_backward(g[0], s[0], s[1].defined() ? &s[1] : nullptr, s[2].defined() ? &s[2] : nullptr, s[3], h,
                                 want, &out[0], &out[1], &out[2]);
    TORCH_CHECK(rc == D2D_OK, "d2d_layer_norm_backward: ", d2d_strerror(rc));
    return once(std::move(out), "layer_norm");
  }
};

struct RouteFunction : torch::autograd::Function<RouteFunction> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, const std::optional<at::Tensor>& bias,
                               const RouteHow& h) {
    at::Tensor w, e, rt;
    const int rc = route_forward(logits, bias ? &*bias : nullptr, h, nullptr, false, &w, &e, &rt);
    TORCH_CHECK(rc == D2D_OK, "d2d_route: ", d2d_strerror(rc));
    ctx->save_for_backward({logits, e, w});
    ctx->mark_non_differentiable({e});
    ctx->set_materialize_grads(false);
    ctx->saved_data["scores"] = h.scores;
    ctx->saved_data["renormalise"] = h.renormalise;
    ctx->saved_data["scale"] = h.scale;
    return {w, e};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(3);
    if (!g[0].defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    RouteHow h = {};
    h.scores = ctx->saved_data["scores"].toInt();
    h.renormalise = ctx->saved_data["renormalise"].toBool();
    h.scale = ctx->saved_data["scale"].toDouble();
    const int rc = route_gradient(g[0], s[0], s[1], s[2], h, &out[0]);
    TORCH_CHECK(rc == D2D_OK, "d2d_route_backward: ", d2d_strerror(rc));
    return once(std::move(out), "route_tokens");
  }
};

std::optional<at::Tensor> optional(const at::Tensor* t) { return t ? std::optional<at::Tensor>(*t) : std::nullopt; }

// ---- calls from Python ------------------------------------------------------------------
// layer_norm(x, weight | None, bias | None, eps, kind, weight offset, statistics wanted) -> (y, mean | None, rstd | None)
PyObject* layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 7, "layer_norm takes 7 arguments");
  const at::Tensor& x = needed(a[0], "x");
  const at::Tensor *w = given(a[1], "weight", &x), *b = given(a[2], "bias", &x);
  NormHow h = {PyFloat_AsDouble(a[3]), PyFloat_AsDouble(a[5]), (int)PyLong_AsLong(a[4])};
  const int stats = PyObject_IsTrue(a[6]);
  if (PyErr_Occurred()) return nullptr;
  at::Tensor y, mean, rstd;
  const int rc = norm_forward(x, w, b, h, stats, &y, &mean, &rstd);
  if (rc != D2D_OK) return PyLong_FromLong(rc);
  return wrap_all({y, mean, rstd});
  END_HANDLE_TH_ERRORS
}

// layer_norm_autograd(x, weight | None, bias | None, eps, kind, weight offset) -> y
PyObject* layer_norm_autograd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 6, "layer_norm_autograd takes 6 arguments");
  const at::Tensor& x = needed(a[0], "x");
  const at::Tensor *w = given(a[1], "weight", &x), *b = given(a[2], "bias", &x);
  NormHow h = {PyFloat_AsDouble(a[3]), PyFloat_AsDouble(a[5]), (int)PyLong_AsLong(a[4])};
  if (PyErr_Occurred()) return nullptr;
  // refusals by status code come before autograd
  if (x.dim() >= 1 && x.size(-1) > D2D_NORM_MAX_D) return PyLong_FromLong(D2D_ERR_UNSUPPORTED);
  if (!(h.eps >= 0.0)) return PyLong_FromLong(D2D_ERR_BAD_ARG);
  return wrap(NormFunction::apply(x, optional(w), optional(b), h));
  END_HANDLE_TH_ERRORS
}

// layer_norm_backward(dy, x, weight | None, mean | None, rstd, kind, weight offset, dx, dweight, dbias wanted)
//   -> (dx, dweight, dbias), None where not wanted; without a weight the gradients are of x's dtype
PyObject* layer_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 10, "layer_norm_backward takes 10 arguments");
  const at::Tensor& x = needed(a[1], "x");
  const at::Tensor& g = needed(a[0], "dy", &x);
  const at::Tensor *w = given(a[2], "weight", &x), *mean = given(a[3], "mean", &x);
  const at::Tensor& rstd = needed(a[4], "rstd", &x);
  NormHow h = {0.0, PyFloat_AsDouble(a[6]), (int)PyLong_AsLong(a[5])};
  const bool want[3] = {PyObject_IsTrue(a[7]) == 1, PyObject_IsTrue(a[8]) == 1, PyObject_IsTrue(a[9]) == 1};
  if (PyErr_Occurred()) return nullptr;
  at::Tensor dx, dw, db;
  const int rc = norm_backward(g, x, w, mean, rstd, h, want, &dx, &dw, &db);
  if (rc != D2D_OK) return PyLong_FromLong(rc);
  return wrap_all({dx, dw, db});
  END_HANDLE_TH_ERRORS
}

// from a[1] on: k, scores, bias | None, groups, top_groups, renormalise, scale
bool route_how(PyObject* const* a, const at::Tensor& logits, RouteHow* h, const at::Tensor** bias) {
  *bias = given(a[3], "bias", &logits);
  *h = {PyLong_AsLong(a[1]), PyLong_AsLong(a[2]),           PyLong_AsLong(a[4]),
        PyLong_AsLong(a[5]), PyObject_IsTrue(a[6]) == 1, PyFloat_AsDouble(a[7])};
  return !PyErr_Occurred();
}

// route(logits [.., E], k, scores, bias | None, groups, top_groups, renormalise, scale, mask bits | None, dense wanted)
//   -> (weights, experts, routing tensor | None)
PyObject* route(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 10, "route takes 10 arguments");
  const at::Tensor& logits = needed(a[0], "logits");
  RouteHow h;
  const at::Tensor* bias;
  if (!route_how(a, logits, &h, &bias)) return nullptr;
  const at::Tensor* mask = given(a[8], "mask bits", &logits);
  const int dense = PyObject_IsTrue(a[9]);
  if (PyErr_Occurred()) return nullptr;
  at::Tensor w, e, rt;
  const int rc = route_forward(logits, bias, h, mask, dense, &w, &e, &rt);
  if (rc != D2D_OK) return PyLong_FromLong(rc);
  return wrap_all({w, e, rt});
  END_HANDLE_TH_ERRORS
}

// route_autograd(logits, k, scores, bias | None, groups, top_groups, renormalise, scale) -> (weights, experts)
PyObject* route_autograd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 8, "route_autograd takes 8 arguments");
  const at::Tensor& logits = needed(a[0], "logits");
  RouteHow h;
  const at::Tensor* bias;
  if (!route_how(a, logits, &h, &bias)) return nullptr;
  // refusals by status code come before autograd: the same call for no tokens
  if (logits.dim() >= 1 && logits.size(-1) > 0) {
    int none = 0;
    const auto small = [](int64_t v) { return (int)std::min<int64_t>(std::max<int64_t>(v, -1), 1 << 21); };
    const int rc = d2d_route(&none, nullptr, (int)h.scores, small(h.k), small(h.groups), small(h.top), h.renormalise,
                             (float)h.scale, &none, (float*)&none, nullptr, nullptr, 0, small(logits.size(-1)),
                             dtype_of(logits), nullptr);
    if (rc != D2D_OK) return PyLong_FromLong(rc);
  }
  const variable_list r = RouteFunction::apply(logits, optional(bias), h);
  return wrap_all({r[0], r[1]});
  END_HANDLE_TH_ERRORS
}

// route_backward(dweights, logits, experts, weights, scores, renormalise, scale) -> dlogits
PyObject* route_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 7, "route_backward takes 7 arguments");
  const at::Tensor& logits = needed(a[1], "logits");
  const at::Tensor& g = needed(a[0], "dweights", &logits);
  const at::Tensor& e = needed(a[2], "experts", &logits);
  const at::Tensor& w = needed(a[3], "weights", &logits);
  RouteHow h = {};
  h.scores = PyLong_AsLong(a[4]);
  h.renormalise = PyObject_IsTrue(a[5]) == 1;
  h.scale = PyFloat_AsDouble(a[6]);
  if (PyErr_Occurred()) return nullptr;
  at::Tensor out;
  const int rc = route_gradient(g, logits, e, w, h, &out);
  if (rc != D2D_OK) return PyLong_FromLong(rc);
  return wrap(out);
  END_HANDLE_TH_ERRORS
}

// What both calls of the weighted experts share: weights as addresses and sizes.
struct ExpertWeights {
  const void *w1, *b1, *up, *w2, *packed;
  int64_t E, d, H;
  int act;
  at::ScalarType dtype;
};

PyObject* run_weighted_experts(const ExpertWeights& m, const at::Tensor& xt, const at::Tensor& et, const at::Tensor& wt,
                               const at::Tensor* bias, bool residual, const at::Tensor* status) {
  const int dt = dtype_of(xt);
  of_type(xt, m.dtype, "x");
  of_type(et, at::kInt, "experts");
  of_type(wt, at::kFloat, "weights");
  TORCH_CHECK_VALUE(xt.dim() >= 1 && xt.size(-1) == m.d, "x must be [.., ", m.d, "]");
  const int64_t N = xt.numel() / m.d;
  TORCH_CHECK_VALUE(et.dim() == xt.dim() && et.sizes().slice(0, et.dim() - 1) == xt.sizes().slice(0, xt.dim() - 1) &&
                        wt.sizes() == et.sizes(),
                    "experts and weights must be [.., k] for x [.., d]");
  const int64_t k = et.size(-1);
  if (bias) {
    of_type(*bias, xt.scalar_type(), "last_bias");
    TORCH_CHECK_VALUE(bias->numel() == m.d && bias->is_contiguous(), "last_bias must have ", m.d, " values");
  }
  if (status) {
    of_type(*status, at::kInt, "status");
    TORCH_CHECK_VALUE(status->numel() > 0, "status must have one value");
  }
  if (k < 1 || k > m.E) return PyLong_FromLong(D2D_ERR_BAD_ARG);
  On on(xt);
  const auto aligned = [](at::Tensor t) {      // (views may start anywhere)
    return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 ? t : t.clone();
  };
  const at::Tensor x = aligned(xt.contiguous()), e = et.contiguous(), w = wt.contiguous();
  const at::Tensor lb = bias ? aligned(*bias) : at::Tensor();
  at::Tensor out = at::detail::empty_cuda(xt.sizes(), xt.options().requires_grad(c10::nullopt)), ws;
  size_t bytes = 0;
  int rc = d2d_experts_weighted_workspace_bytes(N, (int)m.d, (int)m.E, (int)m.H, (int)k, m.up != nullptr,
                                                m.packed != nullptr, dt, &bytes);
  if (rc != D2D_OK) return PyLong_FromLong(rc);
  if (N > 0) {
    ws = at::detail::empty_cuda({(int64_t)bytes}, xt.options().dtype(at::kByte));
    rc = d2d_experts_weighted(x.data_ptr(), (const int32_t*)e.data_ptr(), (const float*)w.data_ptr(), m.w1, m.b1, m.up,
                              m.w2, m.packed, data_or_null(&lb), residual, out.data_ptr(), N, (int)m.d, (int)m.E,
                              (int)m.H, (int)k, m.act, dt, ws.data_ptr(), bytes, (int*)data_or_null(status), on.stream);
  }
  if (rc != D2D_OK) return PyLong_FromLong(rc);
  return wrap(out);
}

// experts_weighted(x [.., d], experts [.., k], weights [.., k], w1, b1 | None, w_up | None, w2, packed | None,
//                  last bias | None, residual, act, status | None) -> out
PyObject* experts_weighted(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 12, "experts_weighted takes 12 arguments");
  const at::Tensor& xt = needed(a[0], "x");
  const at::Tensor& et = needed(a[1], "experts", &xt);
  const at::Tensor& wt = needed(a[2], "weights", &xt);
  const at::Tensor& w1 = needed(a[3], "w1", &xt);
  const at::Tensor* b1 = given(a[4], "b1", &xt);
  const at::Tensor* up = given(a[5], "w_up", &xt);
  const at::Tensor& w2 = needed(a[6], "w2", &xt);
  const at::Tensor* packed = given(a[7], "packed weights", &xt);
  const at::Tensor* bias = given(a[8], "last_bias", &xt);
  const int residual = PyObject_IsTrue(a[9]);
  const int act = (int)PyLong_AsLong(a[10]);
  const at::Tensor* status = given(a[11], "status", &xt);
  if (PyErr_Occurred()) return nullptr;
  const int dt = dtype_of(xt);
  TORCH_CHECK_VALUE(w1.dim() == 3 && w1.numel() > 0, "w1 must be [experts, d, expert width]");
  const int64_t E = w1.size(0), d = w1.size(1), H = w1.size(2);
  const auto weight = [&](const at::Tensor& t, const char* name, at::IntArrayRef shape) {
    of_type(t, xt.scalar_type(), name);
    TORCH_CHECK_VALUE(t.sizes() == shape && t.is_contiguous(), name, " must be contiguous, of shape ", shape);
  };
  weight(w1, "w1", {E, d, H});
  weight(w2, "w2", {E, H, d});
  if (b1) weight(*b1, "b1", {E, H});
  if (up) weight(*up, "w_up", {E, d, H});
  if (packed) {
    size_t most = 0;
    const int rc = d2d_prepack_experts_bytes((int)d, (int)E, (int)H, up != nullptr, dt, &most);
    TORCH_CHECK_VALUE(rc == D2D_OK && most > 0 && packed->is_contiguous() && packed->nbytes() >= most,
                      "packed weights are not those of this shape");
  }
  const ExpertWeights m = {w1.data_ptr(), data_or_null(b1), data_or_null(up), w2.data_ptr(), data_or_null(packed),
                           E, d, H, act, w1.scalar_type()};
  return run_weighted_experts(m, xt, et, wt, bias, residual, status);
  END_HANDLE_TH_ERRORS
}

// run_weighted(plan, modules, parameters, attributes, x, experts, weights, last bias | None, residual, status)
//   -> out | status code (int) | None: the plan is stale.  The plan's module is the experts'.
PyObject* run_weighted(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 10, "run_weighted takes 10 arguments");
  Plan* p = static_cast<Plan*>(PyCapsule_GetPointer(a[0], kPlan));
  if (!p) return nullptr;
  if (!still_valid(*p, a + 1)) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
  }
  const at::Tensor& xt = needed(a[4], "x");
  TORCH_CHECK_VALUE(xt.device() == p->device, "tensors of one call live on different devices: ", p->device, " and ",
                    xt.device(), " (x)");
  const at::Tensor& et = needed(a[5], "experts", &xt);
  const at::Tensor& wt = needed(a[6], "weights", &xt);
  const at::Tensor* bias = given(a[7], "last_bias", &xt);
  const int residual = PyObject_IsTrue(a[8]);
  const at::Tensor* status = given(a[9], "status", &xt);
  if (PyErr_Occurred()) return nullptr;
  const auto cur = c10::cuda::getCurrentCUDAStream(p->device.index());
  use_on(*p, cur);
  // (the word is the module's: it may be gone before this call has run)
  if (status) c10::cuda::CUDACachingAllocator::recordStream(status->storage().data_ptr(), cur);
  const ExpertWeights m = {p->w1, p->b1, p->wup, p->w2, p->ep, p->E, p->d, p->H, (int)p->act, p->dtype};
  return run_weighted_experts(m, xt, et, wt, bias, residual, status);
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"layer_norm", (PyCFunction)(void (*)(void))layer_norm, METH_FASTCALL, nullptr},
    {"layer_norm_autograd", (PyCFunction)(void (*)(void))layer_norm_autograd, METH_FASTCALL, nullptr},
    {"route_autograd", (PyCFunction)(void (*)(void))route_autograd, METH_FASTCALL, nullptr},
    {"layer_norm_backward", (PyCFunction)(void (*)(void))layer_norm_backward, METH_FASTCALL, nullptr},
    {"route", (PyCFunction)(void (*)(void))route, METH_FASTCALL, nullptr},
    {"route_backward", (PyCFunction)(void (*)(void))route_backward, METH_FASTCALL, nullptr},
    {"experts_weighted", (PyCFunction)(void (*)(void))experts_weighted, METH_FASTCALL, nullptr},
    {"run_weighted", (PyCFunction)(void (*)(void))run_weighted, METH_FASTCALL, nullptr},
    {"mark", (PyCFunction)(void (*)(void))mark, METH_FASTCALL, nullptr},
    {"wait_mark", (PyCFunction)(void (*)(void))wait_mark, METH_FASTCALL, nullptr},
    {"make_pipe", (PyCFunction)(void (*)(void))make_pipe, METH_FASTCALL, nullptr},
    {"run_host", (PyCFunction)(void (*)(void))run_host, METH_FASTCALL, nullptr},
    {"make_plan", (PyCFunction)(void (*)(void))make_plan, METH_FASTCALL, nullptr},
    {"run_layer", (PyCFunction)(void (*)(void))run_layer, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_d2d_torch", nullptr, -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__d2d_torch(void) {
  s_get = PyUnicode_InternFromString("raw");
  return PyModule_Create(&kModule);
}
