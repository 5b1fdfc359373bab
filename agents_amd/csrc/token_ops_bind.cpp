// Host side of the token operators (agents_amd/ops.py: categorical_log_prob .. layer_norm_backward) as
// a CPython module: checks of arguments, output tensors, strides, scratch and the call of the C ABI.
// A call of these operators on a small input is bound by this code, not by its kernels: in Python it
// took 15 .. 45 us on the MI355X host, here 5 .. 20 us.
// The C entries are called through addresses that agents_amd/_lib.py passes to init(): the module needs
// no link against libagents_amd.so and follows the library that the package loaded.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <array>
#include <initializer_list>
#include <sstream>
#include <vector>

#include "agents_amd.h"

namespace {

struct Entries {
  decltype(&aa_categorical_workspace_bytes) cat_bytes = nullptr;
  decltype(&aa_categorical_log_prob) cat = nullptr;
  decltype(&aa_categorical_log_prob_backward) cat_backward = nullptr;
  decltype(&aa_clip_tensors_workspace_bytes) clip_bytes = nullptr;
  decltype(&aa_clip_tensors) clip = nullptr;
  decltype(&aa_layer_norm_forward) norm = nullptr;
  decltype(&aa_layer_norm_backward_workspace_bytes) norm_bytes = nullptr;
  decltype(&aa_layer_norm_backward) norm_backward = nullptr;
} lib;
PyObject* raw_stream = nullptr;   // device index -> hipStream_t of torch's current stream, as an int
PyObject* lib_error = nullptr;    // agents_amd._lib.AgentsAmdError

// an error already described to Python
struct Raised {};

template <typename... A>
[[noreturn]] void raise(PyObject* type, const A&... parts) {
  std::ostringstream s;
  (void)std::initializer_list<int>{(s << parts, 0)...};
  PyErr_SetString(type, s.str().c_str());
  throw Raised{};
}
template <typename... A>
[[noreturn]] void refuse(const A&... parts) {
  raise(PyExc_ValueError, parts...);
}

void check(int rc, const char* what) {
  if (rc == 0) return;
  const char* text = rc == -22   ? "AA_ERR_INVALID (bad argument)"
                     : rc == -34 ? "AA_ERR_RANGE (size / workspace)"
                     : rc == -5  ? "AA_ERR_LAUNCH (HIP launch failure)"
                                 : nullptr;
  if (text != nullptr) raise(lib_error, what, " failed: ", text);
  raise(lib_error, what, " failed: ", rc);
}

// ---- arguments ------------------------------------------------------------------------------
const at::Tensor* tensor(PyObject* o, const char* what, const char* name) {
  if (o == Py_None) return nullptr;
  if (!THPVariable_Check(o))
    raise(PyExc_TypeError, what, ": ", name, " must be a tensor, got ", Py_TYPE(o)->tp_name);
  return &THPVariable_Unpack(o);
}
const at::Tensor& tensor_given(PyObject* o, const char* what, const char* name) {
  const at::Tensor* t = tensor(o, what, name);
  if (t == nullptr) raise(PyExc_TypeError, what, ": ", name, " must be a tensor, got None");
  return *t;
}
double number(PyObject* o, const char* what, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    raise(PyExc_TypeError, what, ": ", name, " must be a number, got ", Py_TYPE(o)->tp_name);
  }
  return v;
}
int64_t whole(PyObject* o, const char* what, const char* name) {
  PyObject* i = PyNumber_Index(o);
  const long long v = i != nullptr ? PyLong_AsLongLong(i) : -1;
  Py_XDECREF(i);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    raise(PyExc_TypeError, what, ": ", name, " must be a whole number, got ", Py_TYPE(o)->tp_name);
  }
  return v;
}

int type_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return AA_DT_F32;
    case at::kBFloat16: return AA_DT_BF16;
    case at::kHalf: return AA_DT_F16;
    default: return -1;
  }
}

// The last check of a call, behind all that look at types, shapes and layouts: those hold for host tensors
// as well, so that their refusals are tested without a device.
void on_device(std::initializer_list<const at::Tensor*> ts) {
  const at::Tensor* first = nullptr;
  for (const at::Tensor* t : ts) {
    if (t == nullptr || !t->defined()) continue;
    if (!t->is_cuda())
      raise(lib_error,
            "agents_amd kernels need device tensors (torch 'cuda' = HIP on ROCm); got a ",
            t->device().str(), " tensor.  There is no CPU fallback on the product path.");
    if (first == nullptr) first = t;
    if (t->device() != first->device())
      refuse("tensors on ", first->device().str(), " and ", t->device().str());
  }
}

// ---- memory: what a result may share with the other tensors of a call -----------------------------
// A tensor as runs of `width` bytes, one for every choice of multiples of its axes' strides.
struct Runs {
  struct Axis {
    int64_t stride, size;          // bytes, multiples
  };
  uintptr_t begin = 0;
  int64_t width = 0, reach = 0;    // bytes of a run; from the first run's begin to the last one's
  bool twice = false;              // an axis of stride 0
  c10::SmallVector<Axis, 6> axes;
  explicit Runs(const at::Tensor& t) {
    if (t.numel() == 0) return;    // (width 0: meets nothing)
    begin = (uintptr_t)t.data_ptr();
    width = t.element_size();
    int64_t last = t.dim();
    if (last > 0 && t.stride(-1) == 1) width *= t.size(--last);
    for (int64_t i = 0; i < last; ++i) {
      if (t.size(i) == 1) continue;
      const int64_t stride = t.stride(i) * t.element_size();
      if (stride == 0) {
        twice = true;
        continue;
      }
      axes.push_back({stride, t.size(i)});
      reach += stride * (t.size(i) - 1);
    }
  }
};

// Whether two tensors share a byte: whether a run of b starts less than a run's length before or behind one
// of a.  The distance of two starts is a sum of multiples of the strides; the largest stride is chosen
// first, and only those multiples from which the smaller ones can still come near 0.  Axes nested in each
// other leave two or three of them an axis.  A search past `budget` steps (strides that do not nest, in
// tensors that reach over each other) counts as shared.
struct Meeting {
  struct Step {
    int64_t stride, lo, hi, rest_lo, rest_hi;    // multiples lo .. hi; what the steps behind it add
  };
  c10::SmallVector<Step, 12> steps;
  int64_t below, above;            // a distance d is too near for below < d < above
  bool itself;                     // one tensor: a run does not meet itself
  int budget = 1 << 15;

  Meeting(const Runs& a, const Runs& b, bool itself_) : below(-b.width), above(a.width), itself(itself_) {
    for (const Runs::Axis& x : a.axes) add(x.stride, 1 - x.size, 0);
    for (const Runs::Axis& x : b.axes) add(x.stride, 0, x.size - 1);
    std::sort(steps.begin(), steps.end(), [](const Step& p, const Step& q) { return p.stride > q.stride; });
    int64_t lo = 0, hi = 0;
    for (size_t i = steps.size(); i-- > 0;) {
      steps[i].rest_lo = lo;
      steps[i].rest_hi = hi;
      lo += steps[i].stride * steps[i].lo;
      hi += steps[i].stride * steps[i].hi;
    }
  }
  void add(int64_t stride, int64_t lo, int64_t hi) {
    for (Step& s : steps)
      if (s.stride == stride) {
        s.lo += lo;
        s.hi += hi;
        return;
      }
    steps.push_back({stride, lo, hi, 0, 0});
  }
  static int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }
  bool search(size_t at, int64_t d, bool zero) {
    if (--budget < 0) return true;
    if (at == steps.size()) return below < d && d < above && !(itself && zero);
    const Step& s = steps[at];
    const int64_t lo = std::max(s.lo, floor_div(below - d - s.rest_hi, s.stride) + 1);
    const int64_t hi = std::min(s.hi, -floor_div(d + s.rest_lo - above, s.stride) - 1);
    for (int64_t m = lo; m <= hi; ++m)
      if (search(at + 1, d + m * s.stride, zero && m == 0)) return true;
    return false;
  }
};

bool meet(const Runs& a, const Runs& b) {
  if (a.width == 0 || b.width == 0) return false;
  const int64_t d = (int64_t)(b.begin - a.begin);
  if (d >= a.reach + a.width || -d >= b.reach + b.width) return false;
  return Meeting(a, b, false).search(0, d, false);
}

// a result's memory: no element twice, and what it reads either element for element in the same place or
// elsewhere
void apart(const at::Tensor& out, const at::Tensor& in, const char* name, const char* what) {
  const Runs o(out);
  if (o.width == 0) return;
  // (in one tensor two equal strides would cancel in the difference: they hold an element twice)
  bool twice = o.twice;
  for (size_t i = 1; i < o.axes.size(); ++i)
    for (size_t j = 0; j < i; ++j) twice = twice || o.axes[i].stride == o.axes[j].stride;
  if (twice || (!out.is_contiguous() && Meeting(o, o, true).search(0, 0, true)))
    refuse(what, ": ", name, " must not hold an element twice (strides ", out.strides(), ")");
  bool same = out.data_ptr() == in.data_ptr();
  for (int64_t i = 0; same && i < out.dim(); ++i)
    same = out.size(i) == 1 || out.stride(i) == in.stride(i);
  if (!same && meet(o, Runs(in))) refuse(what, ": ", name, " overlaps an input without being it");
}

// a result's memory against what it must not touch at all
void disjoint(const at::Tensor& out, std::initializer_list<const at::Tensor*> others, const char* name,
              const char* what) {
  const Runs r(out);
  for (const at::Tensor* o : others)
    if (o != nullptr && o->defined() && meet(r, Runs(*o)))
      refuse(what, ": ", name, " overlaps another tensor of the call");
}

// ---- rows: the leading axes folded to (outer, inner) ------------------------------------------
struct Fold {
  int64_t outer = 0, inner = 0;
};

// stride of the row index when the axes from .. to - 1 of t fold to one
bool one_stride(const at::Tensor& t, int64_t from, int64_t to, int64_t* out) {
  int64_t stride = 0, rows = 0;
  for (int64_t i = to - 1; i >= from; --i) {
    const int64_t size = t.size(i);
    if (size == 1) continue;
    if (rows == 0) {
      stride = t.stride(i);
      rows = size;
    } else if (t.stride(i) == stride * rows) {
      rows *= size;
    } else {
      return false;
    }
  }
  *out = stride;
  return true;
}

// One stride where every tensor allows it, else two: the leading axes are cut where both sides fold in
// every tensor (a [B, T - 1] slice of [B, T] rows: before the last).  Returns `inner`.
template <size_t N>
int64_t fold_rows(int64_t lead, const std::array<const at::Tensor*, N>& ts, std::array<Fold, N>& f,
                  const char* what) {
  for (int64_t cut = lead; cut == lead || cut > 0; --cut) {
    bool all = true;
    int64_t inner = 1;
    for (size_t i = 0; i < N && all; ++i) {
      f[i] = Fold{};
      if (ts[i] == nullptr) continue;
      all = one_stride(*ts[i], 0, cut, &f[i].outer) && one_stride(*ts[i], cut, lead, &f[i].inner);
      inner = 1;
      for (int64_t j = cut; j < lead; ++j) inner *= ts[i]->size(j);
    }
    if (all) return inner;
  }
  std::ostringstream s;
  for (size_t i = 0; i < N; ++i)
    if (ts[i] != nullptr) s << " " << ts[i]->strides();
  refuse(what, ": leading axes with strides", s.str(),
         " do not fold to the same two axes; pass contiguous tensors");
}

int64_t rows_of(const at::Tensor& t) {
  int64_t n = 1;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) n *= t.size(i);
  return n;
}

// a contiguous tensor of t's sizes, its rows folded with `inner`
Fold own_fold(const at::Tensor& t, int64_t inner) {
  const int64_t width = t.size(-1);
  return inner == 1 ? Fold{width, 0} : Fold{inner * width, width};
}

bool last_contiguous(const at::Tensor& t) {
  return t.size(-1) <= 1 || t.stride(-1) == 1;
}

// sizes of t without its last axis, `more` appended
c10::SmallVector<int64_t, 6> lead_of(const at::Tensor& t, int64_t more = -1) {
  c10::SmallVector<int64_t, 6> s(t.sizes().begin(), t.sizes().end() - 1);
  if (more >= 0) s.push_back(more);
  return s;
}

// Scratch of ONE call from torch's allocator: calls on several streams and captured graphs that
// replay beside each other never meet in it (a captured call's stays with its graph's pool).
at::Tensor scratch(int64_t bytes, const at::Tensor& like) {
  return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : at::Tensor();
}
void* data(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* data(const at::Tensor* t) { return t != nullptr ? t->data_ptr() : nullptr; }

// the current device is the tensors' for the launch; the stream is torch's current one there
struct OnDevice {
  c10::DeviceGuard guard;
  void* stream;
  explicit OnDevice(const at::Tensor& t) : guard(t.device()), stream(nullptr) {
    PyObject* i = PyLong_FromLong(t.get_device());
    PyObject* s = i != nullptr ? PyObject_CallFunctionObjArgs(raw_stream, i, nullptr) : nullptr;
    Py_XDECREF(i);
    if (s == nullptr) throw Raised{};
    stream = PyLong_AsVoidPtr(s);
    Py_DECREF(s);
    if (stream == nullptr && PyErr_Occurred()) throw Raised{};
  }
};

// other Python threads run while a launch waits for room in the stream's queue
struct Unlocked {
  PyThreadState* s = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(s); }
};
template <typename F, typename... A>
int unlocked(F entry, A... args) {
  Unlocked u;
  return entry(args...);
}

at::TensorOptions f32(const at::Tensor& like) { return like.options().dtype(at::kFloat); }

// Results as pieces of one allocation (as networks keep their gradients), each on a cache line of its
// own: an allocation of each took 0.8 us a tensor, most of a call on small inputs.
struct Pieces {
  at::Tensor flat;
  int64_t at = 0;
  static int64_t room(int64_t n, int64_t width) {
    const int64_t line = 128 / width;
    return (n + line - 1) / line * line;
  }
  Pieces(int64_t total, const at::TensorOptions& options) : flat(at::empty({total}, options)) {}
  at::Tensor take(at::IntArrayRef sizes) {
    auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(flat.storage()), flat.key_set(),
                                                     flat.dtype());
    impl->set_storage_offset(at);
    impl->set_sizes_contiguous(sizes);
    at += room(impl->numel(), flat.element_size());
    return at::Tensor(std::move(impl));
  }
};

PyObject* wrap(const at::Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  PyObject* o = THPVariable_Wrap(t);
  if (o == nullptr) throw Raised{};
  return o;
}

// a tuple that owns its items; nothing leaks when one of them cannot be made
template <size_t N>
PyObject* tuple_of(const std::array<at::Tensor, N>& ts) {
  PyObject* out = PyTuple_New(N);
  if (out == nullptr) throw Raised{};
  for (size_t i = 0; i < N; ++i) {
    try {
      PyTuple_SET_ITEM(out, i, wrap(ts[i]));
    } catch (...) {
      Py_DECREF(out);
      throw;
    }
  }
  return out;
}

void count(Py_ssize_t got, Py_ssize_t want, const char* what) {
  if (got != want) raise(PyExc_TypeError, what, " takes ", want, " arguments, got ", got);
}

#define AA_BIND_BEGIN HANDLE_TH_ERRORS try {
#define AA_BIND_END             \
  }                             \
  catch (const Raised&) {       \
    return nullptr;             \
  }                             \
  END_HANDLE_TH_ERRORS

// ---- categorical ------------------------------------------------------------------------------
struct Categorical {
  const at::Tensor* logits;
  const at::Tensor* actions;
  at::Tensor mask;             // expanded to the logits' shape
  aa_categorical_desc d;
};

Categorical categorical_args(PyObject* logits, PyObject* actions, PyObject* mask, PyObject* temperature,
                             PyObject* first_action, PyObject* padding, const char* what) {
  Categorical c;
  const at::Tensor& x = tensor_given(logits, what, "logits");
  c.logits = &x;
  c.actions = tensor(actions, what, "actions");
  const at::Tensor* m = tensor(mask, what, "mask");
  const int dtype = type_code(x);
  if (x.dim() < 1 || dtype < 0)
    refuse(what, ": logits must be a float32 / bfloat16 / float16 [.., actions] tensor, got ",
           x.scalar_type(), " ", x.sizes());
  const int64_t vocab = x.size(-1);
  if (vocab < 1) refuse(what, ": no actions");
  if (!last_contiguous(x)) refuse(what, ": the last axis of logits must be contiguous");
  const double t = number(temperature, what, "temperature");
  if (!(t >= 1e-30 && t <= 1e30))
    refuse(what, ": temperature must be positive (1e-30 .. 1e30), got ", t);
  if (c.actions != nullptr) {
    const auto at = c.actions->scalar_type();
    if (at != at::kInt && at != at::kLong)
      refuse(what, ": actions must be int32 or int64, got ", at);
    if (c.actions->sizes() != x.sizes().slice(0, x.dim() - 1))
      refuse(what, ": actions ", c.actions->sizes(), " for logits ", x.sizes());
  }
  if (m != nullptr) {
    const auto mt = m->scalar_type();
    if (mt != at::kBool && mt != at::kByte && mt != at::kInt)
      refuse(what, ": mask must be bool, uint8 or int32, got ", mt);
    if (m->sizes() == x.sizes()) {
      c.mask = *m;
    } else {
      bool ok = m->dim() >= 1 && m->dim() <= x.dim() && m->size(-1) == vocab;
      for (int64_t i = 2; ok && i <= m->dim(); ++i)
        ok = m->size(-i) == 1 || m->size(-i) == x.size(-i);
      if (!ok) refuse(what, ": mask ", m->sizes(), " for logits ", x.sizes());
      c.mask = m->expand(x.sizes());
    }
    if (!last_contiguous(c.mask)) refuse(what, ": the last axis of mask must be contiguous");
  }
  aa_categorical_desc& d = c.d;
  d = aa_categorical_desc{};
  d.rows = rows_of(x);
  d.vocab = vocab;
  d.logits = x.data_ptr();
  d.actions = data(c.actions);
  d.first_action = whole(first_action, what, "first_action");
  d.mask = data(c.mask);
  d.dtype = dtype;
  d.action_bytes = c.actions != nullptr ? (int32_t)c.actions->element_size() : 4;
  d.mask_bytes = c.mask.defined() ? (int32_t)c.mask.element_size() : 1;
  d.temperature = (float)t;
  d.no_padding = padding != Py_True;
  return c;
}

// the strides of everything the call reads and of what it writes (`out`, nullable)
Fold categorical_fold(Categorical& c, const at::Tensor* out, const char* what) {
  const std::array<const at::Tensor*, 4> ts = {
      c.logits, c.actions, c.mask.defined() ? &c.mask : nullptr, out};
  std::array<Fold, 4> f;
  c.d.inner = c.d.rows > 0 ? fold_rows(c.logits->dim() - 1, ts, f, what) : 1;
  c.d.x_outer = f[0].outer; c.d.x_inner = f[0].inner;
  c.d.a_outer = f[1].outer; c.d.a_inner = f[1].inner;
  c.d.k_outer = f[2].outer; c.d.k_inner = f[2].inner;
  return f[3];
}

// (logits, actions, mask, temperature, top_k, first_action, padding)
//   -> (log_prob, entropy, top_ids, top_log_prob, stats)
PyObject* py_categorical(PyObject*, PyObject* const* a, Py_ssize_t n) {
  AA_BIND_BEGIN
  const char* what = "categorical_log_prob";
  count(n, 7, what);
  Categorical c = categorical_args(a[0], a[1], a[2], a[3], a[5], a[6], what);
  int64_t k = whole(a[4], what, "top_k");
  if (k < 0 || k > AA_CATEGORICAL_MAX_TOP)
    refuse(what, ": top_k must be 0..", AA_CATEGORICAL_MAX_TOP, ", got ", k);
  if (k > c.d.vocab) k = c.d.vocab;
  categorical_fold(c, nullptr, what);
  const at::Tensor& x = *c.logits;
  on_device({&x, c.actions, &c.mask});
  const auto lead = lead_of(x);
  at::Tensor log_prob, ids, top;
  const int64_t rows = c.d.rows;
  Pieces pieces((c.actions != nullptr ? 2 : 1) * Pieces::room(rows, 4) + Pieces::room(2 * rows, 4) +
                    Pieces::room(k * rows, 4), f32(x));
  if (c.actions != nullptr) log_prob = pieces.take(lead);
  const at::Tensor entropy = pieces.take(lead), stats = pieces.take(lead_of(x, 2));
  if (k > 0) {
    ids = at::empty(lead_of(x, k), x.options().dtype(at::kLong));
    top = pieces.take(lead_of(x, k));
  }
  if (c.d.rows > 0) {
    c.d.top_k = (int32_t)k;
    c.d.log_prob = (float*)data(log_prob);
    c.d.entropy = (float*)data(entropy);
    c.d.stats = (float*)data(stats);
    c.d.top_ids = (int64_t*)data(ids);
    c.d.top_log_prob = (float*)data(top);
    const int64_t need = lib.cat_bytes(&c.d);
    const at::Tensor ws = scratch(need, x);
    OnDevice on(x);
    check(unlocked(lib.cat, &c.d, data(ws), need, on.stream), "aa_categorical_log_prob");
  }
  return tuple_of<5>({log_prob, entropy, ids, top, stats});
  AA_BIND_END
}

// (logits, actions, entropy, stats, dlog_prob, dentropy, mask, temperature, first_action, padding, out)
//   -> dlogits
PyObject* py_categorical_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  AA_BIND_BEGIN
  const char* what = "categorical_log_prob_backward";
  count(n, 11, what);
  Categorical c = categorical_args(a[0], a[1], a[6], a[7], a[8], a[9], what);
  const at::Tensor& x = *c.logits;
  const auto lead = lead_of(x);
  const at::Tensor& entropy = tensor_given(a[2], what, "forward.entropy");
  const at::Tensor& stats = tensor_given(a[3], what, "forward.stats");
  if (a[4] == Py_None && a[5] == Py_None) refuse(what, ": needs dlog_prob or dentropy");
  if (a[4] != Py_None && c.actions == nullptr) refuse(what, ": dlog_prob needs actions");
  at::Tensor g[2];
  for (int i = 0; i < 2; ++i) {
    const char* name = i == 0 ? "dlog_prob" : "dentropy";
    const at::Tensor* t = tensor(a[4 + i], what, name);
    if (t == nullptr) continue;
    if (t->scalar_type() != at::kFloat || t->sizes() != at::IntArrayRef(lead))
      refuse(what, ": ", name, " must be float32 ", at::IntArrayRef(lead), ", got ",
             t->scalar_type(), " ", t->sizes());
    g[i] = t->contiguous();
  }
  const auto lead2 = lead_of(x, 2);
  if (entropy.sizes() != at::IntArrayRef(lead) || entropy.scalar_type() != at::kFloat ||
      !entropy.is_contiguous())
    refuse(what, ": forward.entropy is not of these logits");
  if (stats.sizes() != at::IntArrayRef(lead2) || stats.scalar_type() != at::kFloat ||
      !stats.is_contiguous())
    refuse(what, ": forward.stats is not of these logits");
  at::Tensor out;
  const at::Tensor* const o = tensor(a[10], what, "out");
  if (o != nullptr) {
    if (o->scalar_type() != x.scalar_type() || o->sizes() != x.sizes() || !last_contiguous(*o))
      refuse(what, ": out must be ", x.scalar_type(), " ", x.sizes(),
             " with a contiguous last axis");
    apart(*o, x, "out", what);
    disjoint(*o, {&entropy, &stats, c.actions, &c.mask, &g[0], &g[1]}, "out", what);
    out = *o;
  }
  Fold f = categorical_fold(c, o, what);
  on_device({&x, c.actions, &c.mask, &entropy, &stats, &g[0], &g[1], &out});
  if (!out.defined()) {
    out = at::empty(x.sizes(), x.options());
    f = own_fold(x, c.d.inner);
  }
  if (c.d.rows > 0) {
    c.d.entropy = (float*)data(entropy);
    c.d.stats = (float*)data(stats);
    OnDevice on(x);
    check(unlocked(lib.cat_backward, &c.d, (const float*)data(g[0]), (const float*)data(g[1]),
                   data(out), f.outer, f.inner, on.stream),
          "aa_categorical_log_prob_backward");
  }
  return wrap(out);
  AA_BIND_END
}

// ---- clipping ---------------------------------------------------------------------------------
// items of a sequence of tensors; `hold`, a tuple of the call's own, keeps them while they are used (the
// caller's list may change meanwhile: a number's conversion is Python code, a launch lets other threads run)
std::vector<const at::Tensor*> tensors(PyObject* o, PyObject** hold, const char* what,
                                       const char* name) {
  *hold = PySequence_Tuple(o);
  if (*hold == nullptr) throw Raised{};
  const Py_ssize_t n = PyTuple_GET_SIZE(*hold);
  std::vector<const at::Tensor*> ts((size_t)n);
  for (Py_ssize_t i = 0; i < n; ++i)
    ts[i] = &tensor_given(PyTuple_GET_ITEM(*hold, i), what, name);
  return ts;
}

// results of a list: none overlaps another, and none an input other than its own
void clip_apart(const std::vector<const void*>& src, const std::vector<void*>& dst,
                const std::vector<int64_t>& sizes, int64_t width, const char* what) {
  struct Range {
    uintptr_t begin, end;
    size_t of;
  };
  std::vector<Range> outs;
  outs.reserve(dst.size());
  for (size_t i = 0; i < dst.size(); ++i) {
    const uintptr_t b = (uintptr_t)dst[i];
    if (sizes[i] > 0) outs.push_back({b, b + (uintptr_t)(sizes[i] * width), i});
  }
  std::sort(outs.begin(), outs.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
  for (size_t i = 1; i < outs.size(); ++i)
    if (outs[i].begin < outs[i - 1].end) refuse(what, ": tensors of out overlap");
  for (size_t i = 0; i < src.size(); ++i) {
    const uintptr_t b = (uintptr_t)src[i], e = b + (uintptr_t)(sizes[i] * width);
    if (b == e) continue;
    // the first result that ends behind the input's begin
    auto at = std::partition_point(outs.begin(), outs.end(),
                                   [&](const Range& r) { return r.end <= b; });
    if (at != outs.end() && at->begin < e && !(at->of == i && at->begin == b))
      refuse(what, ": a tensor of out overlaps an input that is not its own");
    if (at != outs.end() && at->of == i && at + 1 != outs.end() && (at + 1)->begin < e)
      refuse(what, ": a tensor of out overlaps an input that is not its own");
  }
}

struct Held {
  PyObject* o = nullptr;
  ~Held() { Py_XDECREF(o); }
};

// (tensors, clip_norm, each, scale, out, name) -> (clipped, norm)
PyObject* py_clip(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  AA_BIND_BEGIN
  count(nargs, 6, "clip");
  const char* what = PyUnicode_AsUTF8(a[5]);
  if (what == nullptr) throw Raised{};
  Held hold, hold_out;
  const std::vector<const at::Tensor*> ts = tensors(a[0], &hold.o, what, "tensors");
  const double clip = number(a[1], what, "clip_norm");
  const bool each = a[2] == Py_True, scale = a[3] == Py_True;
  const size_t n = ts.size();
  if (n == 0) refuse(what, ": no tensors");
  if (n > 0x7fffffff) refuse(what, ": too many tensors");
  if (scale && !(clip > 0)) refuse(what, ": clip_norm must be positive, got ", clip);
  const at::Tensor& t0 = *ts[0];
  const int dtype = type_code(t0);
  if (dtype < 0)
    refuse(what, ": tensors must be float32 / bfloat16 / float16, got ", t0.scalar_type());
  std::vector<const void*> src(n);
  std::vector<void*> dst(scale ? n : 0);
  std::vector<int64_t> sizes(n);
  for (size_t i = 0; i < n; ++i) {
    const at::Tensor& t = *ts[i];
    if (t.scalar_type() != t0.scalar_type() || !t.is_contiguous())
      refuse(what, ": tensors must be contiguous and of one type, got ", t.scalar_type(), " ",
             t.sizes(), " strides ", t.strides(), " beside ", t0.scalar_type());
    src[i] = t.data_ptr();
    sizes[i] = t.numel();
  }
  std::vector<const at::Tensor*> os;
  if (scale && a[4] != Py_None) {
    os = tensors(a[4], &hold_out.o, what, "out");
    if (os.size() != n) refuse(what, ": out must mirror the tensors");
    for (size_t i = 0; i < n; ++i) {
      const at::Tensor& o = *os[i];
      if (o.scalar_type() != t0.scalar_type() || o.sizes() != ts[i]->sizes() || !o.is_contiguous())
        refuse(what, ": out must mirror the tensors");
      dst[i] = o.data_ptr();
    }
    clip_apart(src, dst, sizes, t0.element_size(), what);
  }
  for (size_t i = 0; i < n; ++i) on_device({&t0, ts[i], os.empty() ? nullptr : os[i]});
  PyObject* out = nullptr;     // owned; released on every way out but the last
  Held out_guard;
  // The scratch, some kilobytes of sums, lies behind the clipped tensors (an allocation less); the norm is
  // one of its own, so that a program that keeps the norm of every step keeps no more than that.
  const int64_t need = lib.clip_bytes(sizes.data(), (int32_t)n);
  at::Tensor sums;
  void* ws = nullptr;
  if (!os.empty()) {
    out = out_guard.o = PySequence_List(hold_out.o);
    if (out == nullptr) throw Raised{};
  } else if (scale) {
    int64_t total = 0;
    const int64_t width = t0.element_size();
    for (size_t i = 0; i < n; ++i) total += Pieces::room(sizes[i], width);
    Pieces pieces(total + (need + width - 1) / width, t0.options());
    ws = static_cast<char*>(pieces.flat.data_ptr()) + total * width;
    out = out_guard.o = PyList_New((Py_ssize_t)n);
    if (out == nullptr) throw Raised{};
    for (size_t i = 0; i < n; ++i) {
      const at::Tensor o = pieces.take(ts[i]->sizes());
      dst[i] = o.data_ptr();
      PyList_SET_ITEM(out, (Py_ssize_t)i, wrap(o));
    }
  } else {
    out = out_guard.o = Py_None;
    Py_INCREF(out);
  }
  if (ws == nullptr) {
    sums = scratch(need, t0);
    ws = data(sums);
  }
  const at::Tensor norm = each ? at::empty({(int64_t)n}, f32(t0)) : at::empty({}, f32(t0));
  {
    OnDevice on(t0);
    check(unlocked(lib.clip, src.data(), scale ? dst.data() : nullptr, sizes.data(), (int32_t)n,
                   dtype, clip, (int32_t)each, (float*)norm.data_ptr(), ws, need, on.stream),
          "aa_clip_tensors");
  }
  Held wrapped;
  wrapped.o = wrap(norm);
  PyObject* r = PyTuple_Pack(2, out, wrapped.o);
  if (r == nullptr) throw Raised{};
  return r;
  AA_BIND_END
}

// ---- layer normalisation -----------------------------------------------------------------------
void norm_rows(const at::Tensor& t, const char* name, const at::Tensor& x, const char* what) {
  if (t.scalar_type() != x.scalar_type() || t.sizes() != x.sizes() || !last_contiguous(t))
    refuse(what, ": ", name, " must be ", x.scalar_type(), " ", x.sizes(),
           " with a contiguous last axis, got ", t.scalar_type(), " ", t.sizes(), " strides ",
           t.strides());
}

void norm_weight(const at::Tensor* w, const char* name, const at::Tensor& x, const char* what) {
  if (w == nullptr) return;
  if (w->scalar_type() != at::kFloat || w->dim() != 1 || w->size(0) != x.size(-1) ||
      !w->is_contiguous())
    refuse(what, ": ", name, " must be contiguous float32 [", x.size(-1), "], got ",
           w->scalar_type(), " ", w->sizes());
}

void norm_stats(const at::Tensor& s, const at::Tensor& x, const char* what) {
  const auto want = lead_of(x, 2);
  if (s.sizes() != at::IntArrayRef(want) || s.scalar_type() != at::kFloat || !s.is_contiguous())
    refuse(what, ": stats must be contiguous float32 ", at::IntArrayRef(want));
}

const at::Tensor& norm_input(PyObject* o, const char* what) {
  const at::Tensor& x = tensor_given(o, what, "x");
  if (x.dim() < 1 || type_code(x) < 0 || x.size(-1) < 1)
    refuse(what, ": x must be a float32 / bfloat16 / float16 [.., n] tensor, got ", x.scalar_type(),
           " ", x.sizes());
  norm_rows(x, "x", x, what);
  return x;
}

// (x, gamma, beta, epsilon, out, stats) -> (y, stats)
PyObject* py_layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  AA_BIND_BEGIN
  const char* what = "layer_norm_forward";
  count(n, 6, what);
  const at::Tensor& x = norm_input(a[0], what);
  const at::Tensor* gamma = tensor(a[1], what, "gamma");
  const at::Tensor* beta = tensor(a[2], what, "beta");
  norm_weight(gamma, "gamma", x, what);
  norm_weight(beta, "beta", x, what);
  const double epsilon = number(a[3], what, "epsilon");
  if (!(epsilon >= 0)) refuse(what, ": epsilon must not be negative, got ", epsilon);
  at::Tensor y, stats;
  const at::Tensor* const out = tensor(a[4], what, "out");
  if (out != nullptr) {
    norm_rows(*out, "out", x, what);
    apart(*out, x, "out", what);
    disjoint(*out, {gamma, beta}, "out", what);
    y = *out;
  }
  if (const at::Tensor* s = tensor(a[5], what, "stats")) {
    norm_stats(*s, x, what);
    disjoint(*s, {&x, &y, gamma, beta}, "stats", what);
    stats = *s;
  }
  const int64_t rows = rows_of(x);
  // (results of the call's own are contiguous: they fold as x does)
  std::array<Fold, 2> f;
  const int64_t inner = rows > 0 ? fold_rows<2>(x.dim() - 1, {&x, out}, f, what) : 1;
  on_device({&x, gamma, beta, &y, &stats});
  if (!y.defined()) {
    y = at::empty(x.sizes(), x.options());
    f[1] = own_fold(x, inner);
  }
  if (!stats.defined()) stats = at::empty(lead_of(x, 2), f32(x));
  if (rows > 0) {
    aa_layer_norm_desc d{};
    d.inner = inner;
    d.rows = rows;
    d.width = x.size(-1);
    d.x = x.data_ptr(); d.x_outer = f[0].outer; d.x_inner = f[0].inner;
    d.y = y.data_ptr(); d.y_outer = f[1].outer; d.y_inner = f[1].inner;
    d.gamma = (const float*)data(gamma);
    d.beta = (const float*)data(beta);
    d.stats = (float*)data(stats);
    d.epsilon = (float)epsilon;
    d.dtype = type_code(x);
    OnDevice on(x);
    check(unlocked(lib.norm, &d, on.stream), "aa_layer_norm_forward");
  }
  return tuple_of<2>({y, stats});
  AA_BIND_END
}

// (dy, x, gamma, stats, dx, dgamma, dbeta, mask_act code, param_grads, input_grad)
//   -> (dx, dgamma, dbeta)
PyObject* py_layer_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  AA_BIND_BEGIN
  const char* what = "layer_norm_backward";
  count(n, 10, what);
  const at::Tensor& x = norm_input(a[1], what);
  const at::Tensor& dy = tensor_given(a[0], what, "dy");
  const at::Tensor* gamma = tensor(a[2], what, "gamma");
  const at::Tensor& stats = tensor_given(a[3], what, "stats");
  norm_rows(dy, "dy", x, what);
  norm_weight(gamma, "gamma", x, what);
  norm_stats(stats, x, what);
  const bool params = a[8] == Py_True, input = a[9] == Py_True;
  if (!params && !input) refuse(what, ": nothing to compute");
  at::Tensor dx, dgamma, dbeta;
  const at::Tensor* const dx_out = input ? tensor(a[4], what, "dx") : nullptr;
  if (dx_out != nullptr) {
    norm_rows(*dx_out, "dx", x, what);
    apart(*dx_out, x, "dx", what);
    apart(*dx_out, dy, "dx", what);
    disjoint(*dx_out, {gamma, &stats}, "dx", what);
    dx = *dx_out;
  }
  if (params) {
    const at::Tensor* g = tensor(a[5], what, "dgamma");
    const at::Tensor* b = tensor(a[6], what, "dbeta");
    norm_weight(g, "dgamma", x, what);
    norm_weight(b, "dbeta", x, what);
    if (g != nullptr) disjoint(*g, {b, &dx, &x, &dy, gamma, &stats}, "dgamma", what);
    if (b != nullptr) disjoint(*b, {&dx, &x, &dy, gamma, &stats}, "dbeta", what);
    if (g != nullptr) dgamma = *g;
    if (b != nullptr) dbeta = *b;
  }
  const int32_t mask_act = (int32_t)whole(a[7], what, "mask_act");
  const int64_t rows = rows_of(x);
  std::array<Fold, 3> f;
  const int64_t inner = rows > 0 ? fold_rows<3>(x.dim() - 1, {&x, &dy, dx_out}, f, what) : 1;
  on_device({&x, &dy, gamma, &stats, &dx, &dgamma, &dbeta});
  if (input && !dx.defined()) {
    dx = at::empty(x.sizes(), x.options());
    f[2] = own_fold(x, inner);
  }
  if (params && (!dgamma.defined() || !dbeta.defined())) {
    Pieces pieces((!dgamma.defined() + !dbeta.defined()) * Pieces::room(x.size(-1), 4), f32(x));
    if (!dgamma.defined()) dgamma = pieces.take({x.size(-1)});
    if (!dbeta.defined()) dbeta = pieces.take({x.size(-1)});
  }
  if (rows == 0) {
    if (params) {
      dgamma.zero_();
      dbeta.zero_();
    }
  } else {
    aa_layer_norm_desc d{};
    d.inner = inner;
    d.rows = rows;
    d.width = x.size(-1);
    d.x = x.data_ptr(); d.x_outer = f[0].outer; d.x_inner = f[0].inner;
    d.dy = dy.data_ptr(); d.dy_outer = f[1].outer; d.dy_inner = f[1].inner;
    d.dx = data(dx); d.dx_outer = f[2].outer; d.dx_inner = f[2].inner;
    d.gamma = (const float*)data(gamma);
    d.stats = (float*)data(stats);
    d.dgamma = (float*)data(dgamma);
    d.dbeta = (float*)data(dbeta);
    d.dtype = type_code(x);
    d.mask_act = mask_act;
    const int64_t need = lib.norm_bytes(&d);
    const at::Tensor ws = scratch(need, x);
    OnDevice on(x);
    check(unlocked(lib.norm_backward, &d, data(ws), need, on.stream), "aa_layer_norm_backward");
  }
  return tuple_of<3>({dx, dgamma, dbeta});
  AA_BIND_END
}

// (addresses of the eight C entries in the order of `Entries`, raw_stream, error class)
PyObject* py_init(PyObject*, PyObject* const* a, Py_ssize_t n) {
  AA_BIND_BEGIN
  count(n, 3, "init");
  if (!PyTuple_Check(a[0]) || PyTuple_GET_SIZE(a[0]) != 8)
    raise(PyExc_TypeError, "init needs eight addresses");
  void* p[8];
  for (int i = 0; i < 8; ++i) {
    p[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(a[0], i));
    if (p[i] == nullptr) raise(PyExc_ValueError, "init needs eight addresses");
  }
  lib.cat_bytes = (decltype(lib.cat_bytes))p[0];
  lib.cat = (decltype(lib.cat))p[1];
  lib.cat_backward = (decltype(lib.cat_backward))p[2];
  lib.clip_bytes = (decltype(lib.clip_bytes))p[3];
  lib.clip = (decltype(lib.clip))p[4];
  lib.norm = (decltype(lib.norm))p[5];
  lib.norm_bytes = (decltype(lib.norm_bytes))p[6];
  lib.norm_backward = (decltype(lib.norm_backward))p[7];
  Py_INCREF(a[1]);
  Py_XSETREF(raw_stream, a[1]);
  Py_INCREF(a[2]);
  Py_XSETREF(lib_error, a[2]);
  Py_RETURN_NONE;
  AA_BIND_END
}

#define AA_METHOD(name, fn) {name, (PyCFunction)(void (*)(void))fn, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {AA_METHOD("init", py_init),
                         AA_METHOD("categorical_log_prob", py_categorical),
                         AA_METHOD("categorical_log_prob_backward", py_categorical_backward),
                         AA_METHOD("clip", py_clip),
                         AA_METHOD("layer_norm_forward", py_layer_norm),
                         AA_METHOD("layer_norm_backward", py_layer_norm_backward),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_token_ops", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__token_ops() { return PyModule_Create(&module); }
