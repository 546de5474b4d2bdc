// Host side of the operators whose calls are short next to what Python adds to them: embedding lookup, label log
// probabilities, gradient norm and clipping.  Arguments, workspaces and the autograd nodes live here, in C++ (a backward
// that runs in the engine's thread without the interpreter); the arithmetic is libgsplat_mi355x's, whose entry points are
// looked up in the library that the package has loaded.  A lookup of one id with its gradient took 101 us with a Python
// autograd node over ctypes (an empty one takes 41) and takes 46 here, of which torch's engine has 40.
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/extension.h>

#include <atomic>
#include <unordered_set>

#include "../../include/gsplat_mi355x.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Library {
  decltype(&gs_error_string) error_string = nullptr;
  decltype(&gs_embedding_fwd) embedding_fwd = nullptr;
  decltype(&gs_embedding_bwd_workspace_bytes) embedding_bwd_workspace_bytes = nullptr;
  decltype(&gs_embedding_bwd) embedding_bwd = nullptr;
  decltype(&gs_label_log_probs_workspace_bytes) label_workspace_bytes = nullptr;
  decltype(&gs_label_log_probs_fwd) label_fwd = nullptr;
  decltype(&gs_label_log_probs_bwd) label_bwd = nullptr;
  decltype(&gs_grad_norm_workspace_bytes) grad_workspace_bytes = nullptr;
  decltype(&gs_grad_norm) grad_norm = nullptr;
  decltype(&gs_grad_clip) grad_clip = nullptr;
} L;

template <typename F> void find(void* handle, const char* name, F& f) {
  f = reinterpret_cast<F>(dlsym(handle, name));
  if (!f) throw std::runtime_error(std::string(name) + " is missing in the native library");
}

void load(const std::string& path) {
  void* h = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);  // the package has loaded it: the same library
  if (!h) throw std::runtime_error(dlerror());
  find(h, "gs_error_string", L.error_string);
  find(h, "gs_embedding_fwd", L.embedding_fwd);
  find(h, "gs_embedding_bwd_workspace_bytes", L.embedding_bwd_workspace_bytes);
  find(h, "gs_embedding_bwd", L.embedding_bwd);
  find(h, "gs_label_log_probs_workspace_bytes", L.label_workspace_bytes);
  find(h, "gs_label_log_probs_fwd", L.label_fwd);
  find(h, "gs_label_log_probs_bwd", L.label_bwd);
  find(h, "gs_grad_norm_workspace_bytes", L.grad_workspace_bytes);
  find(h, "gs_grad_norm", L.grad_norm);
  find(h, "gs_grad_clip", L.grad_clip);
}

void check(int status, const char* what) {
  TORCH_CHECK(status == 0, what, " failed with status ", status, ": ", L.error_string(status));
}

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return GS_DTYPE_F32;
    case at::kBFloat16: return GS_DTYPE_BF16;
    case at::kHalf: return GS_DTYPE_F16;
    default: TORCH_CHECK_TYPE(false, "gsplat (MI355X build): float32, bfloat16 or float16 expected, got ", t.scalar_type());
  }
}

int index_bytes(const Tensor& t) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt,
                   "gsplat (MI355X build): int64 or int32 expected, got ", t.scalar_type());
  return t.scalar_type() == at::kLong ? 8 : 4;
}

void require_gpu(const Tensor& t, const Tensor& first) {
  TORCH_CHECK(t.is_cuda(), "gsplat (MI355X build): tensors must live on a HIP device; this build has no CPU path (got a "
                           "tensor on ", t.device(), ").");
  TORCH_CHECK(t.device() == first.device(), "gsplat (MI355X build): tensors on different devices: ", first.device(), " vs ",
              t.device());
}

// the tensor's device is the current one, and its current stream is at hand
struct Launch {
  c10::DeviceGuard guard;
  void* stream;
  explicit Launch(const Tensor& t) : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};

// The package's timing brackets (gsplat._backend.timed) around the launch of a backward, which has no Python around it.
std::atomic<bool> timing{false};
PyObject* timed = nullptr;  // the class while timing is on; read and written with the interpreter's lock

void set_timed(const pybind11::object& cls) {
  PyObject* const before = timed;
  timed = cls.is_none() ? nullptr : cls.inc_ref().ptr();
  timing = timed != nullptr;
  Py_XDECREF(before);
}

class Bracket {
  PyObject* guard = nullptr;

 public:
  Bracket(const char* name, const Tensor& t) {
    if (!timing.load(std::memory_order_relaxed)) return;
    const pybind11::gil_scoped_acquire lock;
    if (!timed) return;
    auto g = pybind11::reinterpret_borrow<pybind11::object>(timed)(name, t.device());
    g.attr("__enter__")();
    guard = g.release().ptr();
  }
  Bracket(const Bracket&) = delete;
  Bracket& operator=(const Bracket&) = delete;
  ~Bracket() {
    if (!guard) return;
    const pybind11::gil_scoped_acquire lock;
    const auto g = pybind11::reinterpret_steal<pybind11::object>(guard);
    try {
      g.attr("__exit__")(pybind11::none(), pybind11::none(), pybind11::none());
    } catch (pybind11::error_already_set& e) {
      e.discard_as_unraisable("gsplat timing");
    }
  }
};

Tensor bytes(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte)); }

// dense rows with their elements next to each other, in memory as they are (a lazily negated view is not)
Tensor rows_of(const Tensor& t) { return (t.size(1) <= 1 || t.stride(1) == 1) && !t.is_neg() ? t : t.resolve_neg().contiguous(); }

// A gradient that nothing can be differentiated through again: a second backward reaches an error, not a zero.
Tensor once(const Tensor& v, const char* what) {
  auto fail = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " cannot be differentiated twice", 1);
  return (*fail)({v.detach().requires_grad_(true)})[0];
}

// Called by a backward before it launches anything.  While a graph captures the backward, a leaf further down whose gradient
// would be accumulated on another stream (an eager graph of that leaf, still alive, has made the node that does it) would
// pull that stream into the capture, which ends the process: an error instead.  Where the gradient is only handed out, the
// engine still makes the node's stream wait, which the default stream must not do during a capture.
void check_capture(const Tensor& grad) {
  const auto current = torch::autograd::get_current_node();
  auto* const node = current.get();
  if (!node || c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const c10::impl::VirtualGuardImpl streams(grad.device().type());
  const auto here = streams.getStream(grad.device()), unnamed = streams.getDefaultStream(grad.device());
  const auto* tasks = torch::autograd::get_current_graph_task_exec_info();  // of torch.autograd.grad: what it needs
  std::unordered_set<torch::autograd::Node*> seen{node};
  std::vector<torch::autograd::Node*> left{node};
  while (!left.empty()) {
    auto* const at = left.back();
    left.pop_back();
    for (const auto& edge : at->next_edges()) {
      auto* const next = edge.function.get();
      if (!next || !seen.insert(next).second) continue;
      if (tasks && !tasks->empty()) {
        const auto it = tasks->find(next);
        if (it == tasks->end() || !it->second.should_execute()) continue;
      }
      left.push_back(next);
      if (!dynamic_cast<torch::autograd::AccumulateGrad*>(next)) continue;
      const bool kept = !tasks || tasks->empty() || tasks->at(next).needed_;  // else it is handed out, not accumulated
      const auto there = next->stream();
      TORCH_CHECK(!there || *there == here || (!kept && *there != unnamed),
                  "gsplat (MI355X build): this backward is being captured while an eager graph of the same leaf, made on "
                  "another stream, is alive: delete its outputs before the capture");
    }
  }
}

// ---------------------------------------------------------------------------------------------------------- embedding
struct EmbeddingLookup : torch::autograd::Function<EmbeddingLookup> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& ids, double scale) {
    const int64_t V = table.size(0), D = table.size(1), n = ids.numel();
    const Tensor flat = ids.contiguous(), rows = rows_of(table);
    auto shape = ids.sizes().vec();
    shape.push_back(D);
    Tensor out = at::empty(shape, table.options());
    Launch on(table);
    check(L.embedding_fwd(n, V, D, dtype_code(table), rows.data_ptr(), rows.stride(0), flat.data_ptr(), index_bytes(flat),
                          (float)scale, out.data_ptr(), on.stream), "gs_embedding_fwd");
    ctx->save_for_backward({flat});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["rows"] = V;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_capture(grads[0]);
    const Tensor flat = ctx->get_saved_variables()[0];
    const double scale = ctx->saved_data["scale"].toDouble();
    const int64_t V = ctx->saved_data["rows"].toInt(), n = flat.numel(), D = grads[0].size(-1);
    const Tensor v = rows_of(grads[0].reshape({n, D}));
    Tensor v_table = at::empty({V, D}, v.options());
    const int64_t nbytes = L.embedding_bwd_workspace_bytes(n, V, D);
    const Tensor ws = nbytes ? bytes(nbytes, v) : Tensor();
    Launch on(v);
    const Bracket bracket("gs_embedding_bwd", v);
    check(L.embedding_bwd(n, V, D, dtype_code(v), flat.data_ptr(), index_bytes(flat), v.data_ptr(), v.stride(0), (float)scale,
                          nbytes ? ws.data_ptr() : nullptr, nbytes, v_table.data_ptr(), on.stream), "gs_embedding_bwd");
    if (at::GradMode::is_enabled() && grads[0].requires_grad()) v_table = once(v_table, "embedding_lookup");
    return {v_table, Tensor(), Tensor()};
  }
};

Tensor embedding_lookup(const Tensor& table, const Tensor& ids, double scale) {
  dtype_code(table);
  index_bytes(ids);
  TORCH_CHECK_VALUE(table.dim() == 2, "table must be [V,D], got ", table.sizes());
  require_gpu(table, table);
  require_gpu(ids, table);
  return EmbeddingLookup::apply(table, ids, scale);
}

// ------------------------------------------------------------------------------------------------------------- labels
struct LabelLogProbs : torch::autograd::Function<LabelLogProbs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& labels, int64_t top_k) {
    const int64_t rows = logits.size(0), K = logits.size(1);
    TORCH_CHECK_VALUE(K <= GS_LABEL_CLASSES_MAX, "at most ", GS_LABEL_CLASSES_MAX, " classes, got ", K);
    const Tensor x = rows_of(logits), y = labels.contiguous();
    const auto f32 = logits.options().dtype(at::kFloat);
    Tensor log_prob = at::empty({rows}, f32), entropy = at::empty({rows}, f32), stats = at::empty({rows, 2}, f32);
    Tensor top = at::empty({rows, top_k}, f32), top_idx = at::empty({rows, top_k}, f32.dtype(at::kLong));
    const int64_t nbytes = L.label_workspace_bytes(rows, (int32_t)K, (int32_t)top_k);
    const Tensor ws = nbytes ? bytes(nbytes, logits) : Tensor();
    Launch on(logits);
    check(L.label_fwd(rows, (int32_t)K, dtype_code(x), (int32_t)top_k, x.data_ptr(), x.stride(0), y.data_ptr(),
                      index_bytes(y), nbytes ? ws.data_ptr() : nullptr, nbytes, log_prob.data_ptr<float>(),
                      entropy.data_ptr<float>(), stats.data_ptr<float>(), top.data_ptr<float>(), top_idx.data_ptr<int64_t>(),
                      on.stream), "gs_label_log_probs_fwd");
    ctx->save_for_backward({x, y, stats, entropy, top_idx});
    ctx->mark_non_differentiable({top_idx});
    ctx->set_materialize_grads(false);
    return {log_prob, entropy, top, top_idx};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    check_capture(saved[0]);
    const Tensor &x = saved[0], &y = saved[1], &stats = saved[2], &entropy = saved[3], &top_idx = saved[4];
    const int64_t rows = x.size(0), K = x.size(1), top_k = top_idx.size(1);
    Tensor g[3];
    for (int i = 0; i < 3; ++i)
      if (grads[i].defined() && (i < 2 || top_k > 0)) g[i] = grads[i].to(at::kFloat).resolve_neg().contiguous();
    if (!g[0].defined() && !g[1].defined() && !g[2].defined()) return {Tensor(), Tensor(), Tensor()};
    Tensor v = at::empty({rows, K}, x.options());
    auto ptr = [](const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; };
    Launch on(x);
    const Bracket bracket("gs_label_log_probs_bwd", x);
    check(L.label_bwd(rows, (int32_t)K, dtype_code(x), (int32_t)top_k, x.data_ptr(), x.stride(0), y.data_ptr(),
                      index_bytes(y), stats.data_ptr<float>(), entropy.data_ptr<float>(), top_idx.data_ptr<int64_t>(),
                      ptr(g[0]), ptr(g[1]), ptr(g[2]), v.data_ptr(), on.stream), "gs_label_log_probs_bwd");
    if (at::GradMode::is_enabled()) v = once(v, "label_log_probs");
    return {v, Tensor(), Tensor()};
  }
};

variable_list label_log_probs(const Tensor& logits, const Tensor& labels, int64_t top_k) {
  dtype_code(logits);
  index_bytes(labels);
  // (the kernels read a label for each row: not left to Python's assertions, which can be switched off)
  TORCH_CHECK_VALUE(logits.dim() >= 1 && labels.sizes() == logits.sizes().slice(0, logits.dim() - 1), "labels must be ",
                    logits.sizes(), " without the last dimension, got ", labels.sizes());
  require_gpu(logits, logits);
  require_gpu(labels, logits);
  const bool flat = logits.dim() == 2;
  const Tensor x = flat ? logits : logits.reshape({labels.numel(), logits.size(-1)});
  auto res = LabelLogProbs::apply(x, flat ? labels : labels.reshape({-1}), top_k);
  if (!flat)
    for (auto& t : res) {
      auto shape = labels.sizes().vec();
      if (t.dim() == 2) shape.push_back(top_k);
      t = t.reshape(shape);
    }
  return res;
}

// ---------------------------------------------------------------------------------------------------------- gradients
std::vector<Tensor> checked(const std::vector<Tensor>& grads) {
  std::vector<Tensor> raw;
  raw.reserve(grads.size());
  for (const Tensor& g : grads) {
    TORCH_CHECK_TYPE(g.layout() == at::kStrided, "gsplat (MI355X build): dense gradients expected, got a sparse one");
    dtype_code(g);
    require_gpu(g, grads[0]);
    // values that fill their memory, in whatever order of dimensions, are taken as they lie
    raw.push_back(g.is_non_overlapping_and_dense() && !g.is_neg() ? g : g.resolve_neg().contiguous());
  }
  return raw;
}

struct Tables {
  std::vector<const void*> src;
  std::vector<void*> dst;
  std::vector<int64_t> numel;
  std::vector<int32_t> dtype;
  Tables(const std::vector<Tensor>& from, const std::vector<Tensor>& to) {
    const size_t n = from.size();
    src.reserve(n); dst.reserve(n); numel.reserve(n); dtype.reserve(n);
    for (size_t i = 0; i < n; ++i) {
      src.push_back(from[i].data_ptr());
      dst.push_back(to[i].data_ptr());
      numel.push_back(from[i].numel());
      dtype.push_back(dtype_code(from[i]));
    }
  }
};

Tensor grad_norm(const std::vector<Tensor>& grads) {
  TORCH_CHECK_VALUE(!grads.empty(), "no gradients given");
  const at::NoGradGuard no_grad;
  const auto src = checked(grads);
  const int32_t n = (int32_t)src.size();
  const int64_t nbytes = L.grad_workspace_bytes(n);
  Tensor norm = at::empty({}, src[0].options().dtype(at::kFloat)), ws = bytes(nbytes, src[0]);
  const Tables t(src, src);
  Launch on(src[0]);
  check(L.grad_norm(n, t.src.data(), t.numel.data(), t.dtype.data(), ws.data_ptr(), nbytes, norm.data_ptr<float>(), on.stream),
        "gs_grad_norm");
  return norm;
}

// Tensors like the given ones.  The small ones share one allocation, 512 bytes apart as separate ones would be: 62 of them
// take 14 us of the host's time instead of 40.
std::vector<Tensor> outputs(const std::vector<Tensor>& like) {
  constexpr int64_t SMALL = 256 << 10, ALIGN = 512;
  const at::AutoDispatchBelowADInplaceOrView direct;
  std::vector<Tensor> out;
  out.reserve(like.size());
  int64_t total = 0;
  for (const Tensor& t : like) total += (int64_t)t.nbytes() <= SMALL ? ((int64_t)t.nbytes() + ALIGN - 1) / ALIGN * ALIGN : 0;
  const Tensor pool = total ? bytes(total, like[0]) : Tensor();
  int64_t at = 0;
  for (const Tensor& t : like) {
    if ((int64_t)t.nbytes() > SMALL || t.numel() == 0) {
      out.push_back(at::empty_like(t));
      continue;
    }
    out.push_back(at::detail::make_tensor<c10::TensorImpl>(c10::Storage(pool.storage()), pool.key_set(), t.dtype()));
    c10::TensorImpl* impl = out.back().unsafeGetTensorImpl();
    impl->set_sizes_and_strides(t.sizes(), t.strides(), at / (int64_t)t.element_size());
    at += ((int64_t)t.nbytes() + ALIGN - 1) / ALIGN * ALIGN;
  }
  return out;
}

std::pair<std::vector<Tensor>, Tensor> clip(const std::vector<Tensor>& grads, double max_norm, double eps, bool inplace) {
  TORCH_CHECK_VALUE(!grads.empty(), "no gradients given");
  const at::NoGradGuard no_grad;
  if (inplace)
    for (const Tensor& g : grads)
      for (int64_t d = 0; g.layout() == at::kStrided && d < g.dim(); ++d)
        TORCH_CHECK_VALUE(g.stride(d) != 0 || g.size(d) <= 1,
                          "a gradient whose values share memory (an expanded one) cannot be scaled in place");
  const auto src = checked(grads);
  const std::vector<Tensor> dst = inplace ? std::vector<Tensor>() : outputs(src);
  const auto& to = inplace ? src : dst;
  const int32_t n = (int32_t)src.size();
  const int64_t nbytes = L.grad_workspace_bytes(n);
  Tensor norm = at::empty({}, src[0].options().dtype(at::kFloat)), ws = bytes(nbytes, src[0]);
  const Tables t(src, to);
  {
    Launch on(src[0]);
    check(L.grad_clip(n, t.src.data(), t.dst.data(), t.numel.data(), t.dtype.data(), (float)max_norm, (float)eps,
                      ws.data_ptr(), nbytes, norm.data_ptr<float>(), on.stream), "gs_grad_clip");
  }
  if (!inplace) return {dst, norm};
  for (size_t i = 0; i < src.size(); ++i) {
    if (!src[i].is_same(grads[i])) grads[i].copy_(src[i]);
    else if (!grads[i].is_inference()) torch::autograd::impl::bump_version(grads[i]);  // written behind autograd's back
  }
  return {grads, norm};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  const auto free = pybind11::call_guard<pybind11::gil_scoped_release>();
  m.def("load", &load);
  m.def("set_timed", &set_timed);
  m.def("embedding_lookup", &embedding_lookup, free);
  m.def("label_log_probs", &label_log_probs, free);
  m.def("grad_norm", &grad_norm, free);
  m.def("clip", &clip, free);
}
