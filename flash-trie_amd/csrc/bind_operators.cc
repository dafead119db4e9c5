// bind_operators.cc -- the model head's operators in the `flashtrie` Python
// module, on torch tensors (the module itself needs no torch: it is imported
// by the first call).  Outputs and workspaces come from torch's allocator;
// launches go to the current stream of the tensors' device, so that a call
// is ordered, freed and captured as torch's own operators are.
#include "bind_operators.h"

#include <dlfcn.h>

#include <cstring>
#include <initializer_list>
#include <string>

#include "../../include/flashtrie_amd.h"
#include "marisa.h"

namespace py = pybind11;

namespace {

[[noreturn]] void fail_type(const std::string& call, const std::string& what) {
  throw py::type_error(call + ": " + what);
}
[[noreturn]] void fail_value(const std::string& call, const std::string& what) {
  throw py::value_error(call + ": " + what);
}

// torch brings a HIP runtime of its own.  Imported first, it is this module's
// too; imported after this module, there are two, and neither knows the
// other's streams.
bool shares_runtime(const py::module_& torch) {
  const std::string init = py::cast<std::string>(torch.attr("__file__"));
  const std::string lib = init.substr(0, init.find_last_of('/') + 1) + "lib/libc10_hip.so";
  void* h = dlopen(lib.c_str(), RTLD_LAZY | RTLD_NOLOAD);
  if (!h) return true;  // a torch without GPUs: its tensors are refused
  const void* theirs = dlsym(h, "hipGetDevice");
  dlclose(h);
  return !theirs || theirs == ft_hip_runtime();
}

// What the calls use of torch, looked up once.
struct Torch {
  py::object tensor, dtypes[3], int32, uint8, raw_stream, current_stream, grad_enabled, written;
  PyObject *get_device, *dtype, *shape, *stride, *data_ptr, *new_empty, *contiguous, *requires_grad;
};

const Torch& torch() {
  // (made under the GIL and kept until the process ends; an import may let
  // another thread in, which then makes its own)
  static const Torch* t = nullptr;
  if (!t) {
    py::module_ m = py::module_::import("torch");
    if (!shares_runtime(m))
      throw marisa::Exception(MARISA_STATE_ERROR,
                              "torch was imported after flashtrie and runs on a HIP runtime of "
                              "its own: import torch first");
    auto* n = new Torch();
    n->tensor = m.attr("Tensor");
    n->dtypes[FT_F32] = m.attr("float32");
    n->dtypes[FT_F16] = m.attr("float16");
    n->dtypes[FT_BF16] = m.attr("bfloat16");
    n->int32 = m.attr("int32");
    n->uint8 = m.attr("uint8");
    // the stream's handle without an object for it, where torch has that
    n->raw_stream = py::getattr(m.attr("_C"), "_cuda_getCurrentRawStream", py::none());
    n->current_stream = m.attr("cuda").attr("current_stream");
    n->grad_enabled = m.attr("is_grad_enabled");
    n->written = m.attr("autograd").attr("graph").attr("increment_version");
    n->get_device = PyUnicode_InternFromString("get_device");
    n->dtype = PyUnicode_InternFromString("dtype");
    n->shape = PyUnicode_InternFromString("shape");
    n->stride = PyUnicode_InternFromString("stride");
    n->data_ptr = PyUnicode_InternFromString("data_ptr");
    n->new_empty = PyUnicode_InternFromString("new_empty");
    n->contiguous = PyUnicode_InternFromString("contiguous");
    n->requires_grad = PyUnicode_InternFromString("requires_grad");
    t = n;
  }
  return *t;
}

py::object call0(py::handle self, PyObject* name) {
  PyObject* args[1] = {self.ptr()};
  PyObject* r = PyObject_VectorcallMethod(name, args, 1 | PY_VECTORCALL_ARGUMENTS_OFFSET, nullptr);
  if (!r) throw py::error_already_set();
  return py::reinterpret_steal<py::object>(r);
}
py::object attr(py::handle self, PyObject* name) {
  PyObject* r = PyObject_GetAttr(self.ptr(), name);
  if (!r) throw py::error_already_set();
  return py::reinterpret_steal<py::object>(r);
}

constexpr int kMaxDims = 3;

struct Tensor {
  py::object obj;  // kept alive during the call
  int ndim = 0;
  int64_t size[kMaxDims], step[kMaxDims];
  void* data = nullptr;
};

// A tensor argument: `dims` dimensions on device `device` (-1: any GPU, which
// is then set), of a type in `types`.
struct Reader {
  std::string call;
  int device = -1;

  Tensor read(py::handle h, const char* name, int dims, int* dtype = nullptr) {
    const Torch& t = torch();
    Tensor r;
    const int is = PyObject_IsInstance(h.ptr(), t.tensor.ptr());
    if (is < 0) throw py::error_already_set();
    if (!is) fail_type(call, std::string(name) + " must be a torch tensor");
    r.obj = py::reinterpret_borrow<py::object>(h);
    fill(r, name, dims);
    const py::object dt = attr(h, t.dtype);
    if (dtype) {
      *dtype = -1;
      for (int i = 0; i < 3; ++i)
        if (dt.is(t.dtypes[i])) *dtype = i;
      if (*dtype < 0)
        fail_type(call, std::string(name) + " must be float32, float16 or bfloat16");
    }
    return r;
  }

  // rows of any stride, elements next to each other
  Tensor rows(py::handle h, const char* name, int dims, int* dtype) {
    Tensor r = read(h, name, dims, dtype);
    if (r.size[dims - 1] > 1 && r.step[dims - 1] != 1)
      fail_value(call, std::string(name) + " must be contiguous in its last dimension");
    return r;
  }

  // a small array of `dt`, made contiguous if it is not
  Tensor array(py::handle h, const char* name, const py::object& dt, const char* dt_name,
               std::initializer_list<int64_t> size) {
    const Torch& t = torch();
    Tensor r = read(h, name, (int)size.size());
    if (!attr(r.obj, t.dtype).is(dt)) fail_type(call, std::string(name) + " must be " + dt_name);
    int i = 0;
    for (int64_t n : size) {
      if (r.size[i] != n)
        fail_value(call, std::string(name) + " has size " + std::to_string(r.size[i]) +
                             " in dimension " + std::to_string(i) + ", not " + std::to_string(n));
      ++i;
    }
    int64_t want = 1;
    bool dense = true;
    for (i = r.ndim - 1; i >= 0; --i) {
      dense = dense && (r.size[i] <= 1 || r.step[i] == want);
      want *= r.size[i];
    }
    if (!dense) {
      r.obj = call0(r.obj, t.contiguous);
      r.data = (void*)PyLong_AsUnsignedLongLong(call0(r.obj, t.data_ptr).ptr());
    }
    return r;
  }

 private:
  void fill(Tensor& r, const char* name, int dims) {
    const Torch& t = torch();
    const py::object shape = attr(r.obj, t.shape);
    r.ndim = (int)PyTuple_GET_SIZE(shape.ptr());
    if (r.ndim != dims)
      fail_value(call, std::string(name) + " must have " + std::to_string(dims) +
                           " dimensions, not " + std::to_string(r.ndim));
    const py::object step = call0(r.obj, t.stride);
    for (int i = 0; i < r.ndim; ++i) {
      r.size[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(shape.ptr(), i));
      r.step[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(step.ptr(), i));
    }
    const long d = PyLong_AsLong(call0(r.obj, t.get_device).ptr());
    if (PyErr_Occurred()) throw py::error_already_set();
    if (d < 0) fail_value(call, std::string(name) + " must be on the GPU");
    if (device < 0) device = (int)d;
    if (d != device) fail_value(call, std::string(name) + " is on another device");
    r.data = (void*)PyLong_AsUnsignedLongLong(call0(r.obj, t.data_ptr).ptr());
    if (PyErr_Occurred()) throw py::error_already_set();
  }
};

// like.new_empty(size, dtype=dtype)
Tensor make(const Tensor& like, std::initializer_list<int64_t> size, const py::object& dtype) {
  const Torch& t = torch();
  Tensor r;
  py::tuple shape(size.size());
  int i = 0;
  for (int64_t n : size) {
    PyTuple_SET_ITEM(shape.ptr(), i, PyLong_FromLongLong(n));
    r.size[i++] = n;
  }
  r.ndim = i;
  int64_t want = 1;
  for (i = r.ndim - 1; i >= 0; --i) {
    r.step[i] = want;
    want *= r.size[i];
  }
  static PyObject* names = PyTuple_Pack(1, t.dtype);
  PyObject* args[3] = {like.obj.ptr(), shape.ptr(), dtype.ptr()};
  PyObject* o = PyObject_VectorcallMethod(t.new_empty, args, 2 | PY_VECTORCALL_ARGUMENTS_OFFSET, names);
  if (!o) throw py::error_already_set();
  r.obj = py::reinterpret_steal<py::object>(o);
  r.data = (void*)PyLong_AsUnsignedLongLong(call0(r.obj, t.data_ptr).ptr());
  return r;
}

void* stream_of(int device) {
  const Torch& t = torch();
  const py::object h = t.raw_stream.is_none()
                           ? py::object(t.current_stream(device).attr("cuda_stream"))
                           : py::object(t.raw_stream(device));
  void* s = (void*)PyLong_AsUnsignedLongLong(h.ptr());
  if (PyErr_Occurred()) throw py::error_already_set();
  return s;
}

void check(int rc, const char* call) {
  if (rc == FT_OK) return;
  const char* d = ft_last_error();
  std::string msg = d && *d ? std::string(d) : std::string(call) + ": " + ft_strerror(rc);
  if (rc == FT_E_ARG) throw py::value_error(msg);
  throw marisa::Exception(rc == FT_E_LIMIT    ? MARISA_SIZE_ERROR
                          : rc == FT_E_NOMEM ? MARISA_MEMORY_ERROR
                                             : MARISA_STATE_ERROR,
                          msg);
}

// Runs a call with a workspace of torch's; the allocator hands its memory on
// only to work that follows on the stream.
template <typename A>
void launch(const A& a, int device, const Tensor& like, const char* call,
            size_t (*size)(const A*), int (*fn)(const A*, void*, size_t, void*)) {
  const size_t n = size(&a);
  Tensor ws;
  if (n) ws = make(like, {(int64_t)n}, torch().uint8);
  check(fn(&a, ws.data, n, stream_of(device)), call);
}

uint32_t u32(int64_t v) { return v > 0xFFFFFFFFll ? 0xFFFFFFFFu : (uint32_t)v; }

py::object adapter_logits(py::object x, py::object weight, py::object down, py::object up,
                          py::object adapter, py::object scale, py::object out_dtype,
                          py::object out) {
  const Torch& t = torch();
  Reader in{"adapter_logits"};
  int dt, d;
  const Tensor tx = in.rows(x, "x", 2, &dt);
  const auto same = [&](py::handle h, const char* name, int dims) {
    const Tensor r = in.rows(h, name, dims, &d);
    if (d != dt) fail_type(in.call, std::string(name) + " must be of x's type");
    return r;
  };
  const Tensor tw = same(weight, "weight", 2), td = same(down, "down", 3), tu = same(up, "up", 3);
  const int64_t T = tx.size[0], H = tx.size[1], V = tw.size[0], G = td.size[0], r = td.size[1];
  if (tw.size[1] != H) fail_value(in.call, "weight and x differ in their hidden size");
  if (td.size[2] != H) fail_value(in.call, "down and x differ in their hidden size");
  if (tu.size[0] != G || tu.size[1] != V || tu.size[2] != r)
    fail_value(in.call, "up must be [adapters, vocab, rank] of down and weight");
  const Tensor ta = in.array(adapter, "adapter", t.int32, "int32", {T});
  const Tensor ts = in.array(scale, "scale", t.dtypes[FT_F32], "float32", {G});
  Tensor to;
  int odt = dt;
  if (!out.is_none()) {
    to = in.rows(out, "out", 2, &odt);
    if (to.size[0] != T || to.size[1] != V) fail_value(in.call, "out must be [rows, vocab]");
    if (!out_dtype.is_none() && !out_dtype.is(t.dtypes[odt]))
      fail_type(in.call, "out is not of out_dtype");
    // (as torch's own out= do: no gradient passes the call)
    if (attr(to.obj, t.requires_grad).is(py::bool_(true)) && py::cast<bool>(t.grad_enabled()))
      fail_value(in.call, "out requires a gradient, which the call does not have");
  } else {
    if (!out_dtype.is_none()) {
      odt = -1;
      for (int i = 0; i < 3; ++i)
        if (out_dtype.is(t.dtypes[i])) odt = i;
    }
    if (odt != FT_F32 && odt != dt)
      fail_type(in.call, "out_dtype must be float32 or the inputs' type");
    to = make(tx, {T, V}, t.dtypes[odt]);
  }
  ft_adapter_logits_args a{};
  a.device = in.device;
  a.dtype = dt;
  a.out_dtype = odt;
  a.rows = (uint64_t)T;
  a.hidden = u32(H);
  a.vocab = u32(V);
  a.adapters = u32(G);
  a.rank = u32(r);
  a.x = tx.data;
  a.x_stride = tx.step[0];
  a.weight = tw.data;
  a.weight_stride = tw.step[0];
  a.down = td.data;
  a.up = tu.data;
  for (int i = 0; i < 2; ++i) {
    a.down_stride[i] = td.step[i];
    a.up_stride[i] = tu.step[i];
  }
  a.adapter = (const int32_t*)ta.data;
  a.scale = (const float*)ts.data;
  a.out = to.data;
  a.out_stride = to.step[0];
  if (!out.is_none()) t.written(to.obj);  // for autograd: its values change
  launch(a, in.device, tx, "adapter_logits", ft_adapter_logits_workspace, ft_adapter_logits);
  return to.obj;
}

py::tuple propose(py::object logits, int64_t topk) {
  const Torch& t = torch();
  Reader in{"propose"};
  ft_propose_args a{};
  const Tensor x = in.rows(logits, "logits", 3, &a.dtype);
  if (topk < 1 || topk > x.size[2]) fail_value(in.call, "topk must be from 1 to vocab");
  const Tensor ids = make(x, {x.size[0], x.size[1], topk}, t.int32);
  const Tensor lp = make(x, {x.size[0], x.size[1], topk}, t.dtypes[FT_F32]);
  a.device = in.device;
  a.batch = (uint64_t)x.size[0];
  a.steps = (uint64_t)x.size[1];
  a.vocab = u32(x.size[2]);
  a.topk = u32(topk);
  a.logits = x.data;
  a.stride[0] = x.step[0];
  a.stride[1] = x.step[1];
  a.ids = (int32_t*)ids.data;
  a.logp = (float*)lp.data;
  launch(a, in.device, x, "propose", ft_propose_workspace, ft_propose);
  return py::make_tuple(ids.obj, lp.obj);
}

// What both losses read and make.
struct Keys {
  Tensor logits, tokens, lengths, loss, logp, dlogits;
  int64_t R, C;
};

Keys read_keys(Reader& in, py::handle logits, py::handle tokens, py::handle lengths, bool grad,
               ft_keys& k) {
  const Torch& t = torch();
  Keys q;
  q.logits = in.rows(logits, "logits", 3, &k.dtype);
  const int64_t R = q.R = q.logits.size[0], S = q.logits.size[1], V = q.logits.size[2];
  const Tensor shape = in.read(tokens, "tokens", 3);
  const int64_t C = q.C = shape.size[1];
  q.tokens = in.array(tokens, "tokens", t.int32, "int32", {R, C, S});
  q.lengths = in.array(lengths, "lengths", t.int32, "int32", {R, C});
  q.loss = make(q.logits, {}, t.dtypes[FT_F32]);
  q.logp = make(q.logits, {R, C, S}, t.dtypes[FT_F32]);
  if (grad) q.dlogits = make(q.logits, {R, S, V}, t.dtypes[k.dtype]);
  k.device = in.device;
  k.batch = (uint64_t)R;
  k.steps = (uint64_t)S;
  k.vocab = u32(V);
  k.keys = u32(C);
  k.logits = q.logits.data;
  k.tokens = (const int32_t*)q.tokens.data;
  k.lengths = (const int32_t*)q.lengths.data;
  k.logp = (float*)q.logp.data;
  k.loss = (float*)q.loss.data;
  k.dlogits = grad ? q.dlogits.data : nullptr;
  for (int i = 0; i < 2; ++i) {
    k.stride[i] = q.logits.step[i];
    k.dstride[i] = grad ? q.dlogits.step[i] : 0;
  }
  return q;
}

py::tuple results(const Keys& q, bool grad) {
  return py::make_tuple(q.loss.obj, q.logp.obj, grad ? q.dlogits.obj : py::none());
}

py::tuple policy_loss(py::object logits, py::object tokens, py::object lengths,
                      py::object old_logp, py::object advantage, py::object weight,
                      double clip_low, double clip_high, double kl_coef, py::object ref_logp,
                      bool grad) {
  const Torch& t = torch();
  Reader in{"policy_loss"};
  ft_policy_loss_args a{};
  const Keys q = read_keys(in, logits, tokens, lengths, grad, a.k);
  const py::object& f32 = t.dtypes[FT_F32];
  const int64_t S = q.logits.size[1];
  const Tensor old = in.array(old_logp, "old_logp", f32, "float32", {q.R, q.C, S});
  const Tensor adv = in.array(advantage, "advantage", f32, "float32", {q.R, q.C});
  const Tensor w = in.array(weight, "weight", f32, "float32", {q.R, q.C});
  Tensor ref;
  if (!ref_logp.is_none()) ref = in.array(ref_logp, "ref_logp", f32, "float32", {q.R, q.C, S});
  else if (kl_coef != 0.0) fail_value(in.call, "kl_coef needs ref_logp");
  a.old_logp = (const float*)old.data;
  a.ref_logp = (const float*)ref.data;
  a.advantage = (const float*)adv.data;
  a.weight = (const float*)w.data;
  a.clip_low = (float)clip_low;
  a.clip_high = (float)clip_high;
  a.kl_coef = (float)kl_coef;
  launch(a, in.device, q.logits, "policy_loss", ft_policy_loss_workspace, ft_policy_loss);
  return results(q, grad);
}

py::tuple preference_loss(py::object logits, py::object tokens, py::object lengths,
                          py::object pairs, py::object ref_logp, py::object weight, double beta,
                          double smoothing, bool grad) {
  const Torch& t = torch();
  Reader in{"preference_loss"};
  ft_preference_loss_args a{};
  const Keys q = read_keys(in, logits, tokens, lengths, grad, a.k);
  const py::object& f32 = t.dtypes[FT_F32];
  const int64_t P = in.read(pairs, "pairs", 2).size[0];
  const Tensor pr = in.array(pairs, "pairs", t.int32, "int32", {P, 2});
  const Tensor ref = in.array(ref_logp, "ref_logp", f32, "float32", {q.R, q.C});
  const Tensor w = in.array(weight, "weight", f32, "float32", {P});
  a.pairs = (uint64_t)P;
  a.pair = (const int32_t*)pr.data;
  a.ref_logp = (const float*)ref.data;
  a.weight = (const float*)w.data;
  a.beta = (float)beta;
  a.smoothing = (float)smoothing;
  launch(a, in.device, q.logits, "preference_loss", ft_preference_loss_workspace,
         ft_preference_loss);
  return results(q, grad);
}

}  // namespace

void bind_operators(py::module_& m) {
  m.def("adapter_logits", &adapter_logits, py::arg("x"), py::arg("weight"), py::arg("down"),
        py::arg("up"), py::arg("adapter"), py::arg("scale"), py::arg("out_dtype") = py::none(),
        py::arg("out") = py::none(),
        "Logits [rows, vocab] of x [rows, hidden] under a shared weight [vocab, hidden], each row "
        "with its request's low-rank adapter: x weight^T + scale[g] (x down[g]^T) up[g]^T with "
        "down [adapters, rank, hidden], up [adapters, vocab, rank] and g = adapter[row] (int32, "
        "negative: none).  float16 or bfloat16 tensors on the GPU; sums in 32 bits; out_dtype is "
        "the inputs' type or float32.");
  m.def("propose", &propose, py::arg("logits"), py::arg("topk"),
        "(ids, logp) [batch, steps, topk] of logits [batch, steps, vocab]: each row's topk "
        "largest logits (ties: the lowest ids) in ascending token order, as the search takes "
        "them, int32, and their float32 log-softmax scores.");
  m.def("policy_loss", &policy_loss, py::arg("logits"), py::arg("tokens"), py::arg("lengths"),
        py::arg("old_logp"), py::arg("advantage"), py::arg("weight"), py::arg("clip_low") = 0.2,
        py::arg("clip_high") = 0.2, py::arg("kl_coef") = 0.0, py::arg("ref_logp") = py::none(),
        py::arg("grad") = true,
        "(loss, logp, dlogits): the clipped policy loss, with a KL term to ref_logp, of the keys "
        "tokens [batch, keys, steps] (int32; lengths [batch, keys]) that logits [batch, steps, "
        "vocab] score; advantage and weight [batch, keys]; logp [batch, keys, steps] are the "
        "tokens' log-probabilities; dlogits is the loss's gradient (None without grad).");
  m.def("preference_loss", &preference_loss, py::arg("logits"), py::arg("tokens"),
        py::arg("lengths"), py::arg("pairs"), py::arg("ref_logp"), py::arg("weight"),
        py::arg("beta") = 0.1, py::arg("smoothing") = 0.0, py::arg("grad") = true,
        "(loss, logp, dlogits): the loss of pairs [n, 2] (int32 indexes into batch * keys: the "
        "preferred key, the other) on their log-probability ratios to ref_logp [batch, keys]; "
        "weight [n]; the rest as in policy_loss.");
}
