// Host side of the serving operators' device implementations: what op_reg's handler and launch.py do for a call (checks, results,
// scratch, strides, stream, the C entry), for the calls whose arguments are as the kernels take them.  Host only: no kernel
// is built here, and the entries are those of the loaded kernel library, handed in by bind().
//
// A step of a serving loop makes several calls of a few microseconds each, and the interpreter takes longer for one than the
// GPU (rope_kv_append of 64 tokens: 4 us of device time, 16 us a call from Python).  Every function here returns None
// for a call that it does not take -- another device than the current one, operands that need a copy, anything that breaks
// the contract, an entry that reports an error -- and the caller goes on in Python, which copies, or raises with
// its message.  So the contract stays where it is (contract.py), and the tests here only have to be as strict.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <optional>

#include "../../include/turbine_mi355.h"

namespace {

using at::Tensor;

struct Entries {
  decltype(&mi355_rope) rope = nullptr;
  decltype(&mi355_rope_kv_append) append = nullptr;
  decltype(&mi355_paged_batch_layout) layout = nullptr;
  decltype(&mi355_flash_attn_varlen_fwd) varlen = nullptr;
  decltype(&mi355_flash_attn_varlen_workspace_bytes) varlen_bytes = nullptr;
  decltype(&mi355_paged_tree_attn) tree = nullptr;
  decltype(&mi355_paged_tree_default_splits) tree_splits = nullptr;
  decltype(&mi355_verify_draft) verify = nullptr;
  decltype(&mi355_verify_draft_workspace_bytes) verify_bytes = nullptr;
  decltype(&mi355_last_error) last_error = nullptr;
} entry;

// ---- arguments -------------------------------------------------------------------------------------------------------

struct NotTaken {};
void want(bool ok) {
  if (!ok) throw NotTaken{};
}
const Tensor& tensor(PyObject* o) {
  want(THPVariable_Check(o));
  return THPVariable_Unpack(o);
}
bool flag(PyObject* o) {
  want(PyBool_Check(o));
  return o == Py_True;
}
int64_t whole(PyObject* o) {
  want(PyLong_CheckExact(o));
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw NotTaken{};
  }
  return v;
}
double number(PyObject* o) {
  want(PyFloat_CheckExact(o));
  return PyFloat_AS_DOUBLE(o);
}

// Memory that is what the tensor stands for.  (Below the dispatcher every tensor is; the rotation is also called above it,
// with lazily negated ones, zeros without memory, and the wrappers of torch.func and of tensor subclasses.)
bool is_plain(const Tensor& t) {
  static const c10::DispatchKeySet odd({c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::Batched,
                                        c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize, c10::DispatchKey::Python});
  return t.layout() == at::kStrided && t.has_storage() && !t.key_set().has_any(odd);
}
// All on one device, the current one: the caller of the kernel needs no guard then.
template <typename... Ts>
void on_current(const Tensor& first, const Ts&... rest) {
  const c10::Device dev = first.device();
  auto plain = [&](const Tensor& t) { return t.device() == dev && is_plain(t); };
  want(dev.is_cuda() && dev.index() == c10::hip::current_device() && plain(first) && (plain(rest) && ...));
}
void* current_stream(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

int half_code(const Tensor& t) {
  if (t.scalar_type() == at::kHalf) return MI355_F16;
  want(t.scalar_type() == at::kBFloat16);
  return MI355_BF16;
}
bool is_vector(const Tensor& t, at::ScalarType type, int64_t n) {
  return t.dim() == 1 && t.size(0) == n && t.scalar_type() == type && t.is_contiguous();
}
bool is_matrix(const Tensor& t, at::ScalarType type, int64_t n, int64_t m) {
  return t.dim() == 2 && t.size(0) == n && t.size(1) == m && t.scalar_type() == type && t.is_contiguous();
}
bool page_ok(int64_t p) { return p == 16 || p == 32 || p == 64 || p == 128 || p == 256; }
void caches(const Tensor& k, const Tensor& v) {
  want(k.dim() == 4 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() && k.is_contiguous() && v.is_contiguous());
  want(k.size(3) == 128 && page_ok(k.size(1)) && k.size(0) > 0 && k.size(2) > 0);
}
struct Strides {
  int64_t v[2];  // {token, head}
};
// [tokens, heads, 128] rows that the attention kernels read in place (launch._row_strides)
Strides rows(const Tensor& t) {
  Strides s{{t.size(0) == 1 ? 128 : t.stride(0), t.size(1) == 1 ? 0 : t.stride(1)}};
  want(t.stride(2) == 1 && ((uintptr_t)t.data_ptr() & 15) == 0 && s.v[0] >= 128 && s.v[0] < (1 << 24) && ((s.v[0] | s.v[1]) & 7) == 0);
  return s;
}
float default_scale(double s) { return (float)(s <= 0 ? 1 / std::sqrt(128.0) : s); }
Tensor fresh(at::IntArrayRef size, const Tensor& like, at::ScalarType type) { return at::empty(size, like.options().dtype(type)); }

// ---- the operators ---------------------------------------------------------------------------------------------------

void check_angles(const Tensor& pos, const Tensor& freq, int64_t tokens, int64_t D) {
  want(is_vector(pos, at::kInt, tokens) && freq.dim() == 1 && freq.is_contiguous());
  want(freq.scalar_type() == at::kDouble || freq.scalar_type() == at::kFloat);
  const int64_t R = 2 * freq.size(0);
  want(R > 0 && R <= D && R <= 1024);
}

void check_rope(const Tensor& x, const Tensor& pos, const Tensor& freq) {
  on_current(x, pos, freq);
  want(x.dim() == 3 && (x.scalar_type() == at::kFloat || x.scalar_type() == at::kHalf || x.scalar_type() == at::kBFloat16));
  const int64_t T = x.size(0), H = x.size(1), D = x.size(2);
  want(T > 0 && T < (1 << 24) && H > 0 && H <= 65535 && D > 0 && D <= 65536 && H * D <= (1 << 30) && x.stride(2) == 1);
  check_angles(pos, freq, T, D);
}

Tensor rope(const Tensor& x, const Tensor& pos, const Tensor& freq, bool inter, bool inverse, double scale) {
  check_rope(x, pos, freq);
  Tensor out = fresh(x.sizes(), x, x.scalar_type());
  const int64_t xs[2] = {x.stride(0), x.stride(1)}, os[2] = {out.stride(0), out.stride(1)};
  want(entry.rope(x.data_ptr(), out.data_ptr(), (const int32_t*)pos.data_ptr(), freq.data_ptr(), freq.scalar_type() == at::kDouble, x.size(0),
                  x.size(1), x.size(2), 2 * freq.size(0), xs, os, inter, inverse, (float)scale,
                  x.scalar_type() == at::kFloat ? MI355_F32 : half_code(x), current_stream(x)) == 0);
  return out;
}

// The op itself, for what the functions here do not take: the lock is taken on the way.
Tensor rope_by_dispatcher(const Tensor& x, const Tensor& pos, const Tensor& freq, bool inter, bool inverse, double scale) {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("mi355::rope", "").typed<Tensor(const Tensor&, const Tensor&, const Tensor&, bool, bool, double)>();
  return op.call(x, pos, freq, inter, inverse, scale);
}

// A leaf's gradient goes on to its accumulator, on the stream that was current when the accumulator was made.  It lives as long
// as a graph of the leaf does: with an eager one alive that is the default stream, which cannot wait for a stream under capture, and
// the engine's attempt may end the process.  Refused here, before it.
void refuse_capture_beside_eager_graph() {
  const auto node = torch::autograd::get_current_node();
  if (!node || node->num_outputs() == 0) return;
  auto* leaf = dynamic_cast<torch::autograd::AccumulateGrad*>(node->next_edge(0).function.get());
  if (!leaf || c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const auto stream = leaf->stream();
  TORCH_CHECK(!stream || stream->id() != 0, "rope: a backward pass under capture while a graph of the same leaf, made on the default stream, is alive; "
              "delete that graph (its outputs) before the capture, or make it on another stream");
}

// The gradient as a node of the engine's own kind: its backward pass takes no interpreter lock (a forward and backward pass of a
// small x: 98 us with the node in Python).  Same formula and same saved tensors as ops._RopeGrad.  Gradients that are to be
// differentiated, have a tangent, are no plain tensors or meet a dispatch mode go through the op, and so does what a function
// here does not take.
struct RopeGrad : torch::autograd::Function<RopeGrad> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& pos, const Tensor& freq, bool inter, bool inverse,
                        double scale) {
    ctx->save_for_backward({pos, freq});
    ctx->saved_data["inter"] = inter;
    ctx->saved_data["inverse"] = inverse;
    ctx->saved_data["scale"] = scale;
    return rope(x, pos, freq, inter, inverse, scale);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    refuse_capture_beside_eager_graph();
    const auto saved = ctx->get_saved_variables();
    const bool inter = ctx->saved_data["inter"].toBool(), inverse = !ctx->saved_data["inverse"].toBool();
    const double scale = ctx->saved_data["scale"].toDouble();
    Tensor g = grads[0], dx;
    if (!(at::GradMode::is_enabled() && g.requires_grad()) && !g._fw_grad(0).defined() && is_plain(g) && !c10::impl::TorchDispatchModeTLS::any_modes_set()) {
      if (g.stride(2) != 1) g = g.contiguous();
      try {
        dx = rope(g, saved[0], saved[1], inter, inverse, scale);  // (saved-tensor hooks may have put anything in their place)
      } catch (NotTaken&) {
      }
    }
    if (!dx.defined()) dx = rope_by_dispatcher(g, saved[0], saved[1], inter, inverse, scale);
    return {dx, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor append(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& pos, const Tensor& freq, const Tensor& kc, const Tensor& vc,
              const Tensor& slots, bool inter, double scale) {
  on_current(q, k, v, pos, freq, kc, vc, slots);
  const int code = half_code(q);
  want(q.dim() == 3 && k.dim() == 3 && v.sizes() == k.sizes() && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type() &&
       kc.scalar_type() == q.scalar_type());
  caches(kc, vc);
  const int64_t T = q.size(0), hq = q.size(1), hkv = k.size(1);
  want(q.size(2) == 128 && k.size(2) == 128 && k.size(0) == T && T > 0 && T < (1 << 24) && hq > 0 && hq <= 65535 && hkv == kc.size(2) && hkv <= 65535);
  want(q.stride(2) == 1 && k.stride(2) == 1 && v.stride(2) == 1 && is_vector(slots, at::kLong, T));
  check_angles(pos, freq, T, 128);
  Tensor out = fresh(q.sizes(), q, q.scalar_type());
  const int64_t qs[2] = {q.stride(0), q.stride(1)}, ks[2] = {k.stride(0), k.stride(1)}, vs[2] = {v.stride(0), v.stride(1)};
  want(entry.append(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), kc.data_ptr(), vc.data_ptr(), (const int32_t*)pos.data_ptr(),
                    freq.data_ptr(), freq.scalar_type() == at::kDouble, (const int64_t*)slots.data_ptr(), T, hq, hkv, 128, 2 * freq.size(0),
                    kc.size(0) * kc.size(1), qs, ks, vs, inter, (float)scale, code, current_stream(q)) == 0);
  return out;
}

std::array<Tensor, 6> layout(const Tensor& table, const Tensor& ctx, const Tensor& add, const Tensor& free, int64_t page, int64_t T) {
  on_current(table, ctx, add, free);
  want(table.dim() == 2 && table.size(0) > 0 && table.size(1) > 0);
  const int64_t S = table.size(0), W = table.size(1);
  want(S <= 65535 && W <= (1 << 22) && is_matrix(table, at::kInt, S, W) && is_vector(ctx, at::kInt, S) && is_vector(add, at::kInt, S));
  want(free.dim() == 1 && free.size(0) <= (1 << 30) && is_vector(free, at::kInt, free.size(0)) && page_ok(page) && T >= 1 && T <= (1 << 30));
  std::array<Tensor, 6> r = {fresh({S}, table, at::kInt), fresh({S + 1}, table, at::kInt), fresh({T}, table, at::kInt),
                             fresh({T}, table, at::kInt), fresh({T}, table, at::kLong),    fresh({1}, table, at::kInt)};
  auto i32 = [](const Tensor& t) { return (int32_t*)t.data_ptr(); };
  want(entry.layout(i32(table), i32(ctx), i32(add), free.size(0) ? i32(free) : nullptr, free.size(0), S, W, page, T, i32(r[0]), i32(r[1]), i32(r[2]),
                    i32(r[3]), (int64_t*)r[4].data_ptr(), i32(r[5]), current_stream(table)) == 0);
  return r;
}

Tensor varlen(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cq, const Tensor& ck, bool causal, double scale) {
  on_current(q, k, v, cq, ck);
  const int code = half_code(q);
  want(q.dim() == 3 && k.dim() == 3 && v.sizes() == k.sizes() && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type());
  const int64_t Tq = q.size(0), H = q.size(1), Tk = k.size(0), Hkv = k.size(1);
  want(q.size(2) == 128 && k.size(2) == 128 && Hkv > 0 && H > 0 && H <= 65535 && H % Hkv == 0);
  want(Tq > 0 && Tq <= (1 << 24) && Tk > 0 && Tk <= (1 << 24) && Tq * (H / Hkv) <= (1 << 30));
  want(cq.dim() == 1 && cq.size(0) >= 2 && cq.size(0) <= 65536 && is_vector(cq, at::kInt, cq.size(0)) && is_vector(ck, at::kInt, cq.size(0)));
  const Strides qs = rows(q), ks = rows(k), vs = rows(v);
  const int64_t S = cq.size(0) - 1, bytes = entry.varlen_bytes(S, Tq, Tk, H, Hkv, causal);
  Tensor out = fresh(q.sizes(), q, q.scalar_type()), ws;
  if (bytes) ws = fresh({bytes}, q, at::kByte);
  const Strides os = rows(out);
  want(entry.varlen(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), (const int32_t*)cq.data_ptr(), (const int32_t*)ck.data_ptr(), S, Tq, Tk,
                    H, Hkv, 128, qs.v, ks.v, vs.v, os.v, default_scale(scale), causal, 1, code, bytes ? ws.data_ptr() : nullptr, bytes,
                    current_stream(q)) == 0);
  return out;
}

Tensor tree(const Tensor& q, const Tensor& kc, const Tensor& vc, const Tensor& table, const Tensor& lens, const Tensor& parents, double scale,
            int64_t splits) {
  on_current(q, kc, vc, table, lens, parents);
  const int code = half_code(q);
  want(q.dim() == 4 && q.is_contiguous() && kc.scalar_type() == q.scalar_type());
  caches(kc, vc);
  const int64_t S = q.size(0), N = q.size(1), hq = q.size(2), hkv = kc.size(2);
  want(S > 0 && q.size(3) == 128 && hq > 0 && hq % hkv == 0 && hq / hkv <= 128 && N >= 1 && N <= 64 && splits <= 1024);
  want(table.dim() == 2 && table.size(1) > 0 && is_matrix(table, at::kInt, S, table.size(1)) && is_vector(lens, at::kInt, S) &&
       is_matrix(parents, at::kInt, S, N));
  if (splits <= 0) splits = entry.tree_splits(S, N, hq, hkv, kc.size(1), table.size(1));
  Tensor out = fresh(q.sizes(), q, q.scalar_type()), acc, ml;
  if (splits > 1) {
    acc = fresh({S, N, hq, splits, 128}, q, at::kFloat);
    ml = fresh({S, N, hq, splits, 2}, q, at::kFloat);
  }
  auto i32 = [](const Tensor& t) { return (const int32_t*)t.data_ptr(); };
  want(entry.tree(q.data_ptr(), kc.data_ptr(), vc.data_ptr(), i32(table), i32(lens), i32(parents), out.data_ptr(),
                  splits > 1 ? (float*)acc.data_ptr() : nullptr, splits > 1 ? (float*)ml.data_ptr() : nullptr, S, N, hq, hkv, 128, kc.size(1),
                  table.size(1), kc.size(0), splits, default_scale(scale), code, current_stream(q)) == 0);
  return out;
}

std::array<Tensor, 3> verify(const Tensor& target, const Tensor* draft, const Tensor& tokens, const Tensor& parents, const Tensor& uniforms) {
  on_current(target, tokens, parents, uniforms, draft ? *draft : target);
  want(target.dim() == 3 && target.scalar_type() == at::kFloat && target.is_contiguous());
  const int64_t S = target.size(0), N = target.size(1), V = target.size(2);
  want(S >= 1 && S <= 65535 && N >= 1 && N <= 64 && V >= 1 && V <= (1 << 24));
  want(!draft || (draft->scalar_type() == at::kFloat && draft->sizes() == target.sizes() && draft->is_contiguous()));
  want(is_matrix(tokens, at::kInt, S, N) && is_matrix(parents, at::kInt, S, N) && is_matrix(uniforms, at::kFloat, S, N));
  const int64_t bytes = entry.verify_bytes(S, N, V);
  std::array<Tensor, 3> r = {fresh({S, N}, tokens, at::kInt), fresh({S}, tokens, at::kInt), fresh({S}, tokens, at::kInt)};
  Tensor ws = fresh({bytes}, tokens, at::kByte);
  auto i32 = [](const Tensor& t) { return (int32_t*)t.data_ptr(); };
  want(entry.verify((const float*)target.data_ptr(), draft ? (const float*)draft->data_ptr() : nullptr, i32(tokens), i32(parents),
                    (const float*)uniforms.data_ptr(), i32(r[0]), i32(r[1]), i32(r[2]), S, N, V, ws.data_ptr(), bytes,
                    current_stream(target)) == 0);
  return r;
}

// ---- the interpreter's side ------------------------------------------------------------------------------------------

PyObject* wrapped(Tensor t) { return THPVariable_Wrap(std::move(t)); }
template <size_t N>
PyObject* wrapped(std::array<Tensor, N> ts) {
  PyObject* r = PyTuple_New(N);
  for (size_t i = 0; r && i < N; i++) {
    PyObject* t = THPVariable_Wrap(std::move(ts[i]));
    if (!t) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i, t);
  }
  return r;
}

struct Unlocked {  // runs without the interpreter lock: an allocation or a launch may wait for the GPU
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// The call's result, None if it is not taken.  `f` reads its arguments and returns what computes the result without the lock.
template <typename F>
PyObject* taken(Py_ssize_t given, Py_ssize_t wanted, F&& f) {
  HANDLE_TH_ERRORS
  if (given == wanted && entry.rope) {
    try {
      auto compute = f();
      decltype(compute()) r;
      {
        Unlocked unlocked;
        r = compute();
      }
      return wrapped(std::move(r));
    } catch (NotTaken&) {
    }
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

using Args = PyObject* const*;

PyObject* py_rope(PyObject*, Args a, Py_ssize_t n) {
  return taken(n, 6, [&] {
    const Tensor &x = tensor(a[0]), &pos = tensor(a[1]), &freq = tensor(a[2]);
    const bool inter = flag(a[3]), inverse = flag(a[4]);
    const double scale = number(a[5]);
    return [=, &x, &pos, &freq] { return rope(x, pos, freq, inter, inverse, scale); };
  });
}
PyObject* py_rope_grad(PyObject*, Args a, Py_ssize_t n) {
  return taken(n, 6, [&] {
    const Tensor &x = tensor(a[0]), &pos = tensor(a[1]), &freq = tensor(a[2]);
    const bool inter = flag(a[3]), inverse = flag(a[4]);
    const double scale = number(a[5]);
    return [=, &x, &pos, &freq] {
      check_rope(x, pos, freq);  // before anything is recorded
      return RopeGrad::apply(x, pos, freq, inter, inverse, scale);
    };
  });
}
PyObject* py_append(PyObject*, Args a, Py_ssize_t n) {
  return taken(n, 10, [&] {
    const Tensor* t[8];
    for (int i = 0; i < 8; i++) t[i] = &tensor(a[i]);
    const bool inter = flag(a[8]);
    const double scale = number(a[9]);
    return [=] { return append(*t[0], *t[1], *t[2], *t[3], *t[4], *t[5], *t[6], *t[7], inter, scale); };
  });
}
PyObject* py_layout(PyObject*, Args a, Py_ssize_t n) {
  return taken(n, 6, [&] {
    const Tensor* t[4];
    for (int i = 0; i < 4; i++) t[i] = &tensor(a[i]);
    const int64_t page = whole(a[4]), T = whole(a[5]);
    return [=] { return layout(*t[0], *t[1], *t[2], *t[3], page, T); };
  });
}
PyObject* py_varlen(PyObject*, Args a, Py_ssize_t n) {
  return taken(n, 7, [&] {
    const Tensor* t[5];
    for (int i = 0; i < 5; i++) t[i] = &tensor(a[i]);
    const bool causal = flag(a[5]);
    const double scale = number(a[6]);
    return [=] { return varlen(*t[0], *t[1], *t[2], *t[3], *t[4], causal, scale); };
  });
}
PyObject* py_tree(PyObject*, Args a, Py_ssize_t n) {
  return taken(n, 8, [&] {
    const Tensor* t[6];
    for (int i = 0; i < 6; i++) t[i] = &tensor(a[i]);
    const double scale = number(a[6]);
    const int64_t splits = whole(a[7]);
    return [=] { return tree(*t[0], *t[1], *t[2], *t[3], *t[4], *t[5], scale, splits); };
  });
}
PyObject* py_verify(PyObject*, Args a, Py_ssize_t n) {
  return taken(n, 5, [&] {
    const Tensor *target = &tensor(a[0]), *draft = a[1] == Py_None ? nullptr : &tensor(a[1]);
    const Tensor *tokens = &tensor(a[2]), *parents = &tensor(a[3]), *u = &tensor(a[4]);
    return [=] { return verify(*target, draft, *tokens, *parents, *u); };
  });
}

// bind(address, ...): the entries of the kernel library, in the order of _lib._HOST_ENTRIES
PyObject* py_bind(PyObject*, Args a, Py_ssize_t n) {
  void* at[10];
  if (n != 10) {
    PyErr_SetString(PyExc_TypeError, "bind() takes 10 addresses");
    return nullptr;
  }
  for (int i = 0; i < 10; i++) {
    at[i] = PyLong_AsVoidPtr(a[i]);
    if (!at[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind(): null address");
      return nullptr;
    }
  }
  entry.append = (decltype(entry.append))at[1];
  entry.layout = (decltype(entry.layout))at[2];
  entry.varlen = (decltype(entry.varlen))at[3];
  entry.varlen_bytes = (decltype(entry.varlen_bytes))at[4];
  entry.tree = (decltype(entry.tree))at[5];
  entry.tree_splits = (decltype(entry.tree_splits))at[6];
  entry.verify = (decltype(entry.verify))at[7];
  entry.verify_bytes = (decltype(entry.verify_bytes))at[8];
  entry.last_error = (decltype(entry.last_error))at[9];
  entry.rope = (decltype(entry.rope))at[0];
  Py_RETURN_NONE;
}

#define FAST(f) (PyCFunction)(void (*)(void)) f, METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"bind", FAST(py_bind)},
                         {"rope", FAST(py_rope)},
                         {"rope_grad", FAST(py_rope_grad)},
                         {"rope_kv_append", FAST(py_append)},
                         {"paged_batch_layout", FAST(py_layout)},
                         {"flash_attn_varlen_fwd", FAST(py_varlen)},
                         {"paged_tree_attn", FAST(py_tree)},
                         {"verify_draft", FAST(py_verify)},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "mi355_host_ops", "Host side of the serving operators (see host_ops.cpp).", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_mi355_host_ops() { return PyModule_Create(&module); }
