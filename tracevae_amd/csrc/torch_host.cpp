// Host side of operators whose cost in Python would be several times that of their kernels: an
// autograd node for the scaled embedding (a node written in Python needs the interpreter's lock in
// autograd's own thread: 30 us of a 90 us forward + backward) and the addresses of many tensors at
// once (150 parameters: 60 us as Python loops, 5 here).  The kernels are reached through the C-ABI, by
// the addresses that `bind` is given, so that both sides use the same build of the library.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>
#include <unordered_set>
#include <vector>

#include "../../include/tracevae_hip.h"

namespace {

struct {
  decltype(&tv_last_error) last_error;
  decltype(&tv_scaled_embedding_fwd) fwd;
  decltype(&tv_scaled_embedding_bwd) bwd;
  decltype(&tv_scaled_embedding_bwd_workspace_bytes) bwd_bytes;
  decltype(&tv_adamw_step) adamw_step;
} lib;
PyObject *library_error, *memory_error;           // hip.HipLibraryError, torch.OutOfMemoryError

struct LibraryError : std::runtime_error {        // becomes hip.HipLibraryError
  using std::runtime_error::runtime_error;
};
struct Mismatch : std::runtime_error {            // becomes TypeError
  using std::runtime_error::runtime_error;
};

void check(int rc, const char *name) {
  if (rc != TV_OK) throw LibraryError(std::string(name) + " failed (" + std::to_string(rc) + "): " + lib.last_error());
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return TV_DTYPE_F32;
    case at::kBFloat16: return TV_DTYPE_BF16;
    case at::kHalf: return TV_DTYPE_F16;
    default: return -1;
  }
}
at::ScalarType dtype_of(int64_t code) {
  return code == TV_DTYPE_F32 ? at::kFloat : code == TV_DTYPE_BF16 ? at::kBFloat16 : at::kHalf;
}

void *stream_of(const at::Tensor &t) {
  return (void *)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

bool capturing(hipStream_t stream) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (stream == nullptr) return false;            // (the default stream cannot be captured)
  if (hipStreamIsCapturing(stream, &status) != hipSuccess) {
    (void)hipGetLastError();
    return false;
  }
  return status == hipStreamCaptureStatusActive;
}
bool capturing(const c10::Stream &s) { return capturing(c10::hip::HIPStreamMasqueradingAsCUDA(s).stream()); }

// Autograd runs a node on the stream on which it was made and lets that stream wait for the node before it.
// In a captured backward pass a node from outside the capture - the accumulator of a leaf that an eager
// graph still holds - ties an eager stream to the capture, which ends the process: refused here, before
// the engine gets there.
void refuse_nodes_outside_capture(const c10::Stream &current) {
  if (!capturing(current)) return;
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  const auto *exec = torch::autograd::get_current_graph_task_exec_info();
  std::vector<torch::autograd::Node *> todo{node.get()};
  std::unordered_set<torch::autograd::Node *> seen;
  while (!todo.empty()) {
    torch::autograd::Node *at = todo.back();
    todo.pop_back();
    for (const auto &edge : at->next_edges()) {
      torch::autograd::Node *next = edge.function.get();
      if (!next || !seen.insert(next).second) continue;
      if (exec && !exec->empty()) {               // (of autograd.grad: the nodes that it needs)
        const auto it = exec->find(next);
        if (it == exec->end() || !it->second.should_execute()) continue;
      }
      const auto stream = next->stream();
      if (stream && *stream != current && !capturing(*stream))
        throw LibraryError("scaled_embedding: this backward pass is being captured, but " + next->name() +
                           " of a tensor it leads to belongs to an eager graph that is still alive: drop that "
                           "graph's outputs before the capture");
      todo.push_back(next);
    }
  }
}

// A lookup hands on no tangent: a result without one would read as a derivative of zero.
void refuse_tangent(const at::Tensor &t, const char *what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), "scaled_embedding: ", what,
                              " carries a tangent, forward mode is not implemented");
}

// What a view or a tensor without memory stands for, in memory: a sign that is pending (the imaginary part of a
// conjugate), autograd's zeros, whose address is null.
at::Tensor in_memory(const at::Tensor &t) {
  return t._is_zerotensor() ? t.clone() : t.is_neg() ? t.resolve_neg() : t;
}

// (behind the checks of scaled_embedding below: a [tokens, dim] table with contiguous rows, contiguous
// int64 ids on its device, types that go together)
at::Tensor lookup(const at::Tensor &weight, const at::Tensor &ids, double scale, int64_t padding_id, int64_t out_code) {
  const c10::DeviceGuard guard(weight.device());
  const int64_t tokens = weight.size(0), dim = weight.size(1), rows = ids.numel();
  at::DimVector shape(ids.sizes());
  shape.push_back(dim);
  at::Tensor out = at::empty(shape, weight.options().dtype(dtype_of(out_code)).requires_grad(false));
  check(lib.fwd(rows, dim, tokens, dtype_code(weight.scalar_type()), (int)out_code, weight.const_data_ptr(),
                tokens > 1 ? weight.stride(0) : dim, ids.const_data_ptr<int64_t>(), padding_id, (float)scale,
                out.mutable_data_ptr(), dim, stream_of(weight)),
        "tv_scaled_embedding_fwd");
  return out;
}

class ScaledEmbedding : public torch::autograd::Function<ScaledEmbedding> {
 public:
  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &weight,
                            const at::Tensor &ids, double scale, int64_t padding_id, int64_t out_code) {
    const int64_t tokens = weight.size(0), dim = weight.size(1);
    const at::Tensor out = lookup(weight, ids, scale, padding_id, out_code);
    ctx->save_for_backward({ids});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["sizes"] = std::vector<int64_t>{tokens, dim, (int64_t)dtype_code(weight.scalar_type()),
                                                    out_code, padding_id};
    return out;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                 torch::autograd::variable_list grads) {
    const at::Tensor ids = ctx->get_saved_variables()[0];
    const double scale = ctx->saved_data["scale"].toDouble();
    const auto sizes = ctx->saved_data["sizes"].toIntVector();
    const int64_t tokens = sizes[0], dim = sizes[1], rows = ids.numel();
    const c10::DeviceGuard guard(ids.device());
    // (autograd's engine hands over nothing else; a node that is called by hand may)
    if (grads[0].device() != ids.device() || grads[0].layout() != at::kStrided ||
        grads[0].scalar_type() != dtype_of(sizes[3]))
      throw Mismatch(std::string("the gradient of the rows must be a dense tensor of their type (") +
                     c10::toString(dtype_of(sizes[3])) + ") on " + ids.device().str() + ", got " +
                     c10::toString(grads[0].scalar_type()) + " on " + grads[0].device().str());
    refuse_tangent(grads[0], "the gradient of the rows");
    refuse_nodes_outside_capture(
        c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(ids.device().index()).unwrap());
    at::Tensor dw;
    {
      const at::AutoGradMode no_grad(false);
      at::Tensor dout = in_memory(grads[0]).reshape({rows, dim});
      const bool rows_apart = rows <= 1 || dout.stride(0) >= dim, dense_rows = dim <= 1 || dout.stride(1) == 1;
      if (!rows_apart || !dense_rows) dout = dout.contiguous();
      dw = at::empty({tokens, dim}, dout.options().dtype(dtype_of(sizes[2])));
      // (a buffer of this call: a captured graph has it to itself)
      const int64_t bytes = lib.bwd_bytes(rows, dim, tokens);
      at::Tensor ws = at::empty({bytes}, dout.options().dtype(at::kByte));
      check(lib.bwd(rows, dim, tokens, (int)sizes[2], (int)sizes[3], ids.const_data_ptr<int64_t>(), sizes[4],
                    (float)scale, dout.const_data_ptr(), rows > 1 ? dout.stride(0) : dim, dw.mutable_data_ptr(),
                    ws.mutable_data_ptr(), bytes, stream_of(ids)),
            "tv_scaled_embedding_bwd");
    }
    if (at::GradMode::is_enabled() && grads[0].requires_grad()) {
      // no second derivative: differentiating the result again is an error, as in the other operators
      auto error = std::make_shared<torch::autograd::DelayedError>(
          "trying to differentiate scaled_embedding twice: its gradient is once differentiable", 1);
      dw.set_requires_grad(true);
      dw = (*error)({dw})[0];
    }
    return {dw, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// ---------------------------------------------------------------------------------------
bool address_of(PyObject *o, void **to) {
  *to = PyLong_AsVoidPtr(o);
  return *to != nullptr || !PyErr_Occurred();
}

PyObject *bind(PyObject *, PyObject *const *args, Py_ssize_t n) {
  void *a[5];
  if (n != 7) {
    PyErr_SetString(PyExc_TypeError, "bind takes five addresses and two exception classes");
    return nullptr;
  }
  for (int i = 0; i < 5; ++i)
    if (!address_of(args[i], &a[i])) return nullptr;
  lib.last_error = (decltype(lib.last_error))a[0];
  lib.fwd = (decltype(lib.fwd))a[1];
  lib.bwd = (decltype(lib.bwd))a[2];
  lib.bwd_bytes = (decltype(lib.bwd_bytes))a[3];
  lib.adamw_step = (decltype(lib.adamw_step))a[4];
  Py_INCREF(args[5]);
  Py_INCREF(args[6]);
  library_error = args[5];
  memory_error = args[6];
  Py_RETURN_NONE;
}

template <typename F> PyObject *guarded(F f) {
  try {
    return f();
  } catch (const LibraryError &e) {
    PyErr_SetString(library_error, e.what());
  } catch (const Mismatch &e) {
    PyErr_SetString(PyExc_TypeError, e.what());
  } catch (const std::invalid_argument &e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const python_error &) {
    // (set already)
  } catch (const c10::NotImplementedError &e) {
    PyErr_SetString(PyExc_NotImplementedError, e.what_without_backtrace());
  } catch (const c10::OutOfMemoryError &e) {
    PyErr_SetString(memory_error, e.what());
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// scaled_embedding(weight, ids, scale, padding_idx or None, out_dtype or None)
PyObject *scaled_embedding(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != 5 || !THPVariable_Check(args[0]) || !THPVariable_Check(args[1]) ||
      !(args[4] == Py_None || THPDtype_Check(args[4]))) {
    PyErr_SetString(PyExc_TypeError, "scaled_embedding(weight, ids, scale, padding_idx, out_dtype): two tensors, "
                                     "a number, a number or None, a torch.dtype or None");
    return nullptr;
  }
  const double scale = PyFloat_AsDouble(args[2]);
  const int64_t padding = args[3] == Py_None ? -1 : PyLong_AsLongLong(args[3]);
  if (PyErr_Occurred()) return nullptr;
  return guarded([&]() -> PyObject * {
    at::Tensor weight = THPVariable_Unpack(args[0]), ids = THPVariable_Unpack(args[1]);
    if (!weight.is_cuda() || ids.device() != weight.device())
      throw LibraryError("weight is on " + weight.device().str() + ", ids on " + ids.device().str() +
                         ": the accelerated path runs on the GPU only (there is no CPU fallback)");
    const at::ScalarType in = weight.scalar_type();
    const at::ScalarType to = args[4] == Py_None ? in : reinterpret_cast<THPDtype *>(args[4])->scalar_type;
    if (dtype_code(in) < 0 || dtype_code(to) < 0 || (to != in && in != at::kFloat))
      throw Mismatch(std::string("a table of ") + c10::toString(in) + " does not give rows of " + c10::toString(to));
    if (ids.scalar_type() != at::kLong)
      throw Mismatch(std::string("ids must be torch.int64, got ") + c10::toString(ids.scalar_type()));
    if (weight.layout() != at::kStrided || ids.layout() != at::kStrided) throw Mismatch("weight and ids are dense");
    if (weight.dim() != 2 || weight.numel() == 0) throw std::invalid_argument("weight must be [tokens, dim]");
    refuse_tangent(weight, "weight");
    at::Tensor out;
    {
      struct Released {                           // (also when an exception passes)
        PyThreadState *state = PyEval_SaveThread();
        ~Released() { PyEval_RestoreThread(state); }
      } released;
      weight = in_memory(weight);
      if (!weight.is_contiguous() && (weight.stride(1) != 1 || weight.stride(0) < weight.size(1)))
        weight = weight.contiguous();
      ids = in_memory(ids).contiguous();
      out = at::GradMode::is_enabled() && weight.requires_grad()
                ? ScaledEmbedding::apply(weight, ids, scale, padding, dtype_code(to))
                : lookup(weight, ids, scale, padding, dtype_code(to));
    }
    return THPVariable_Wrap(out);
  });
}

// adamw_step(params, grads or None, dtypes, sizes, planned, addresses, plan_host, plan_device, bits,
// moment1, moment2, scale1, scale2, master, control, clip, norm, seed, guard, guard_kind, guard_host,
// workspace, workspace_bytes, stream, device): tv_adamw_step with the gradients' addresses.  dtypes (int), sizes
// and planned (int64: the parameters' addresses in the plan) are arrays of the optimizer, addresses is
// its int64 scratch.  False: a parameter is not where the plan has it, nothing was done.  None: the step was
// captured, with the plan's address.
PyObject *adamw_step(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != 25 || !PyList_Check(args[0]) || !(args[1] == Py_None || PyList_Check(args[1]))) {
    PyErr_SetString(PyExc_TypeError, "adamw_step takes a list of parameters, a list of gradients or None, and 23 more");
    return nullptr;
  }
  void *a[25] = {};
  double clip = 0.0;
  for (int i = 2; i < 25; ++i) {
    if (i == 15) clip = PyFloat_AsDouble(args[i]);
    else if (i == 17) a[i] = (void *)(intptr_t)PyLong_AsUnsignedLongLongMask(args[i]);     // the seed
    else if (args[i] != Py_None) a[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  const int *dtypes = (const int *)a[2];
  const int64_t *sizes = (const int64_t *)a[3], *planned = (const int64_t *)a[4];
  const void **grad_at = (const void **)a[5];
  PyObject *params = args[0], *grads = args[1] == Py_None ? nullptr : args[1];
  const Py_ssize_t count = PyList_GET_SIZE(params);
  const at::Device device(at::kCUDA, (at::DeviceIndex)(intptr_t)a[24]);
  const int64_t planned_count = ((const int64_t *)a[6])[1];        // (head of the plan: magic, count)
  if (count != planned_count) {
    PyErr_Format(PyExc_ValueError, "%zd parameters, but the optimizer was made for %lld", count, (long long)planned_count);
    return nullptr;
  }
  if (grads && PyList_GET_SIZE(grads) != count) {
    PyErr_Format(PyExc_ValueError, "%zd gradients for %zd parameters", PyList_GET_SIZE(grads), count);
    return nullptr;
  }
  return guarded([&]() -> PyObject * {
    std::vector<at::Tensor> kept;                 // contiguous copies, until the launch
    bool moved = false;
    for (Py_ssize_t i = 0; i < count; ++i) {
      PyObject *po = PyList_GET_ITEM(params, i), *go = grads ? PyList_GET_ITEM(grads, i) : Py_None;
      if (!THPVariable_Check(po) || (go != Py_None && !THPVariable_Check(go)))
        throw Mismatch("parameters and gradients are tensors");
      const at::Tensor &p = THPVariable_Unpack(po);
      if (p.numel() != sizes[i] || dtype_code(p.scalar_type()) != dtypes[i] || p.device() != device ||
          !p.is_contiguous() || p.is_neg())
        throw Mismatch("parameter " + std::to_string(i) +
                       " no longer has the size, type, device or layout that the optimizer was made for");
      moved |= (int64_t)p.const_data_ptr() != planned[i];
      at::Tensor g;
      if (!grads) g = p.grad();
      else if (go != Py_None) g = THPVariable_Unpack(go);
      if (!g.defined()) {
        grad_at[i] = nullptr;
        continue;
      }
      if (g.layout() != at::kStrided || g.scalar_type() != p.scalar_type() || g.device() != p.device() ||
          g.sizes() != p.sizes())
        throw Mismatch("gradient " + std::to_string(i) + " must be a dense tensor of the parameter's type (" +
                       c10::toString(p.scalar_type()) + "), shape and device, got " +
                       c10::toString(g.scalar_type()) + " on " + g.device().str());
      if (!g.is_contiguous() || g.is_neg() || g._is_zerotensor()) {
        g = in_memory(g.detach()).contiguous();
        kept.push_back(g);
      }
      grad_at[i] = g.const_data_ptr();
    }
    if (moved) Py_RETURN_FALSE;
    check(lib.adamw_step(a[6], a[7], grad_at, (int)(intptr_t)a[8], a[9], a[10], (float *)a[11], (float *)a[12],
                         (float *)a[13], a[14], clip, (double *)a[16], (int64_t)(intptr_t)a[17],
                         (const float *)a[18], (int)(intptr_t)a[19], (float *)a[20], a[21],
                         (int64_t)(intptr_t)a[22], a[23]),
          "tv_adamw_step");
    for (Py_ssize_t i = 0; i < count; ++i) {      // written by a kernel
      const at::Tensor &p = THPVariable_Unpack(PyList_GET_ITEM(params, i));
      if (!p.is_inference()) p.unsafeGetTensorImpl()->bump_version();
    }
    if (capturing((hipStream_t)a[23])) Py_RETURN_NONE;
    Py_RETURN_TRUE;
  });
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, nullptr},
    {"scaled_embedding", (PyCFunction)(void (*)(void))scaled_embedding, METH_FASTCALL, nullptr},
    {"adamw_step", (PyCFunction)(void (*)(void))adamw_step, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_host(void) { return PyModule_Create(&module); }
