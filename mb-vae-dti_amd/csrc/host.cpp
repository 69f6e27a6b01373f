// Host side of the operators whose calls are short next to what Python spends on one: argument checks, allocation, autograd nodes and
// the call of the C entry points.  Everything else of the package binds the library with ctypes; a training call of a few hundred rows
// spends 5-20 us on the GPU, and its backward, which autograd runs in a thread of its own, 60 us in Python and 8 us here.
// The entry points are handed over as addresses, so that this module runs whichever build of the library the package has loaded.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <c10/hip/HIPStream.h>
#include <c10/core/DeviceGuard.h>
#include <atomic>
#include <cmath>
#include <limits>
#include <map>
#include <string>

typedef struct ihipStream_t* mbvae_stream_t;
namespace py = pybind11;

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ------------------------------------------------------------------------------------------------ the library
struct Library {
  int (*gated_norm_fwd)(const void*, int64_t, const void*, int64_t, const void*, int64_t, const uint8_t*, float, const void*, const void*, const void*,
                        const void*, const void*, void*, void*, float*, int64_t, int64_t, int, float, int, int, mbvae_stream_t);
  int64_t (*gated_norm_bwd_workspace)(int64_t, int64_t, int);
  int (*gated_norm_bwd)(const void*, int64_t, const void*, int64_t, const void*, int64_t, const uint8_t*, float, const void*, const void*, const void*,
                        const void*, const float*, const void*, int64_t, const void*, int64_t, void*, void*, void*, void*, void*, void*, void*, void*,
                        int64_t, int64_t, int, float, int, int, void*, int64_t, mbvae_stream_t);
  int (*embedding_fwd)(const void*, int, const void*, void*, int64_t, int64_t, int64_t, float, int, mbvae_stream_t);
  int64_t (*embedding_bwd_workspace)(int64_t, int64_t, int64_t, int);
  int (*embedding_bwd)(const void*, int, const void*, int64_t, void*, int64_t, int64_t, int64_t, float, int, void*, int64_t, mbvae_stream_t);
  int64_t (*grad_clip_workspace)(int64_t);
  int (*grad_clip)(const void* const*, void* const*, const int64_t*, const int32_t*, int64_t, double, double, float*, void*, int64_t, mbvae_stream_t);
} lib;

// While the package notes kernel calls (_lib.PROFILE), every call of an entry point is bracketed as its ctypes calls are: bracket(name) notes
// the start and returns what notes the end.  Never freed: threads of autograd may outlast the interpreter.
std::atomic<bool> profiling{false};
py::object* bracket = nullptr;

void bind(const std::map<std::string, uintptr_t>& entries, py::object noted) {
  bracket = new py::object(std::move(noted));
#define BIND(name) lib.name = reinterpret_cast<decltype(lib.name)>(entries.at("mbvae_" #name))
  BIND(gated_norm_fwd);
  BIND(gated_norm_bwd_workspace);
  BIND(gated_norm_bwd);
  BIND(embedding_fwd);
  BIND(embedding_bwd_workspace);
  BIND(embedding_bwd);
  BIND(grad_clip_workspace);
  BIND(grad_clip);
#undef BIND
}

void succeeded(int status, const char* entry) {
  TORCH_CHECK(status == 0, entry, " failed: ",
              status == -1 ? "invalid argument" : status == -2 ? "unsupported shape" : status == -3 ? "kernel launch failure" : "unknown status");
}

// Calls an entry point; raises on failure.
template <typename F>
void entry(const char* name, F call) {
  if (!profiling.load(std::memory_order_relaxed)) return succeeded(call(), name);
  const auto with_gil = [&](auto f) {                        // (autograd's threads do not hold it)
    py::gil_scoped_acquire gil;
    f();
  };
  PyObject* end = nullptr;
  with_gil([&] { end = (*bracket)(name).release().ptr(); });
  const int status = call();
  with_gil([&] { py::reinterpret_steal<py::object>(end)(status); });
  succeeded(status, name);
}

// ------------------------------------------------------------------------------------------------ operands
int type_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: return -1;
  }
}
std::string name_of(at::ScalarType t) {
  const int code = type_code(t);
  return code == 0 ? "float32" : code == 1 ? "bfloat16" : code == 2 ? "float16" : c10::toString(t);
}
int id_code(at::ScalarType t) {
  switch (t) {
    case at::kChar: return 1;
    case at::kShort: return 2;
    case at::kByte: return 3;
    case at::kInt: return 4;
    case at::kLong: return 8;
    default: return -1;
  }
}

bool present(const OptTensor& t) { return t.has_value() && t->defined(); }
Tensor or_none(const OptTensor& t) { return present(t) ? *t : Tensor(); }
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out_ptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
mbvae_stream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
Tensor bytes_on(const Tensor& t, int64_t n) { return at::empty({n}, t.options().dtype(at::kByte).requires_grad(false)); }
Tensor contiguous_like(const Tensor& t) { return at::empty(t.sizes(), t.options().requires_grad(false)); }

// n elements of a flat buffer from `at` on, as a tensor of its own (the gradients of a block's vectors share one allocation: asking the
// allocator for each of them took longer than the kernel that writes them).
Tensor part_of(const Tensor& flat, int64_t at, int64_t n) {
  auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(flat.storage()), flat.key_set(), flat.dtype());
  impl->set_storage_offset(at);
  impl->set_sizes_contiguous({n});
  return Tensor(std::move(impl));
}

// A tangent would be lost without a word: the kernels know nothing of it.  (There are none outside a dual level; asking hundreds of views for
// theirs took 12 us.)
bool tangents_possible() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }
void check_no_tangent(const Tensor& t, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), what, " has no forward-mode derivative (an operand carries a tangent)");
}
void check_typed(const Tensor& t, const char* what, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.layout() == at::kStrided && type_code(t.scalar_type()) >= 0, what, ": ", name,
              ": expected a dense float32, bfloat16 or float16 tensor on the GPU (got ", name_of(t.scalar_type()), " on ", t.device(),
              "); the HIP path has no CPU fallback");
  if (tangents_possible()) check_no_tangent(t, what);
}
void check_same(const Tensor& t, const Tensor& as, const char* what, const char* name) {
  check_typed(t, what, name);
  TORCH_CHECK_VALUE(t.scalar_type() == as.scalar_type(), what, ": ", name, ": expected ", name_of(as.scalar_type()), ", got ", name_of(t.scalar_type()));
  TORCH_CHECK_VALUE(t.device() == as.device(), what, ": ", name, ": expected a tensor on ", as.device(), ", got one on ", t.device());
}

// A tensor as rows of D contiguous elements: a view where the layout allows one, a copy otherwise.  (The imaginary part of a conjugate
// holds its values with the other sign and a mark, which kernels do not see.)
struct Rows {
  Tensor t;
  int64_t ld = 0;
  Rows() {}
  Rows(const Tensor& x, int64_t D) {
    if (!x.defined()) return;
    t = x.resolve_neg();
    if (t.dim() != 2) t = t.reshape({-1, D});
    if (D > 1 && t.size(0) > 0 && t.stride(1) != 1) t = t.contiguous();
    ld = t.size(0) > 1 ? t.stride(0) : D;
  }
};

// A backward of these nodes cannot be differentiated again: its results say so when that is tried.
variable_list differentiable_once(variable_list grads, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& t : grads)                                    // (what the kernels wrote has no history of its own to hang the error on)
    if (t.defined()) t = t.detach().requires_grad_(true);
  auto refuse = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " cannot be differentiated twice", grads.size());
  return (*refuse)(std::move(grads));
}

// ------------------------------------------------------------------------------------------------ embedding
Tensor embedding_raw(const Tensor& ids, const Tensor& weight, double scale) {
  auto sizes = ids.sizes().vec();
  sizes.push_back(weight.size(1));
  Tensor y = at::empty(sizes, weight.options().requires_grad(false));
  const c10::DeviceGuard guard(weight.device());
  entry("mbvae_embedding_fwd", [&] {
    return lib.embedding_fwd(ids.const_data_ptr(), id_code(ids.scalar_type()), weight.const_data_ptr(), y.mutable_data_ptr(), ids.numel(),
                             weight.size(0), weight.size(1), (float)scale, type_code(weight.scalar_type()), stream_of(weight));
  });
  return y;
}

struct Embedding : torch::autograd::Function<Embedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& ids, double scale) {
    ctx->save_for_backward({ids});
    ctx->saved_data["vocab"] = weight.size(0);
    ctx->saved_data["scale"] = scale;
    return embedding_raw(ids, weight, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor& dy = grads[0];
    const Tensor ids = ctx->get_saved_variables()[0];
    const int64_t vocab = ctx->saved_data["vocab"].toInt(), rows = ids.numel(), D = dy.size(-1);
    check_typed(dy, "embedding", "gradient");
    Tensor dw = at::empty({vocab, D}, dy.options().requires_grad(false));
    if (vocab > 0 && D > 0) {
      const Rows d(dy, D);
      const c10::DeviceGuard guard(dy.device());
      const Tensor ws = bytes_on(dy, lib.embedding_bwd_workspace(rows, vocab, D, type_code(dy.scalar_type())));
      entry("mbvae_embedding_bwd", [&] {
        return lib.embedding_bwd(ids.const_data_ptr(), id_code(ids.scalar_type()), d.t.const_data_ptr(), d.ld, dw.mutable_data_ptr(), rows, vocab, D,
                                 (float)ctx->saved_data["scale"].toDouble(), type_code(dy.scalar_type()), ws.mutable_data_ptr(), ws.numel(),
                                 stream_of(dy));
      });
    }
    return differentiable_once({dw, Tensor(), Tensor()}, "embedding");
  }
};

Tensor embedding(const Tensor& ids, const Tensor& weight, double scale) {
  check_typed(weight, "embedding", "weight");
  TORCH_CHECK(id_code(ids.scalar_type()) > 0 && ids.device() == weight.device() && ids.layout() == at::kStrided,
              "embedding: expected dense integer ids on ", weight.device(), " (got ", ids.scalar_type(), " on ", ids.device(),
              "); the HIP path has no CPU fallback");
  TORCH_CHECK_VALUE(weight.dim() == 2, "embedding: weight must be [V, D], got shape ", weight.sizes());
  TORCH_CHECK_VALUE(ids.numel() < ((int64_t)1 << 31) && weight.size(0) < ((int64_t)1 << 31) && weight.size(1) <= ((int64_t)1 << 23),
                    "embedding: at most 2^31 - 1 ids, 2^31 - 1 table rows and 2^23 columns");
  const Tensor i = ids.contiguous(), w = weight.resolve_neg().contiguous();
  if (at::GradMode::is_enabled() && w.requires_grad()) return Embedding::apply(w, i, scale);
  return embedding_raw(i, w, scale);
}

// ------------------------------------------------------------------------------------------------ gated residual norm
struct GatedArgs {
  double keep_scale, eps;
  bool rms;
};

Tensor stats_for(const Tensor& x, int64_t rows) { return at::empty({rows, 4}, x.options().dtype(at::kFloat).requires_grad(false)); }

int param_code(const Tensor& post_g, const Tensor& scale, const Tensor& pre_g) {
  const Tensor& p = post_g.defined() ? post_g : scale.defined() ? scale : pre_g;
  return p.defined() ? type_code(p.scalar_type()) : 0;
}

std::tuple<Tensor, Tensor> gated_norm_raw(const Tensor& x, const Tensor& u, const Tensor& z, const Tensor& keep, const Tensor& post_g,
                                          const Tensor& post_b, const Tensor& scale, const Tensor& pre_g, const Tensor& pre_b, const GatedArgs& a,
                                          Tensor* stats) {
  const int64_t D = x.size(-1);
  const Rows xr(x, D), ur(u, D), zr(z, D);
  const int64_t rows = xr.t.size(0);
  Tensor y = contiguous_like(x), n = pre_g.defined() ? contiguous_like(x) : Tensor();
  if (stats) *stats = stats_for(x, rows);
  const c10::DeviceGuard guard(x.device());
  entry("mbvae_gated_norm_fwd", [&] {
    return lib.gated_norm_fwd(ptr(xr.t), xr.ld, ptr(ur.t), ur.ld, ptr(zr.t), zr.ld, (const uint8_t*)ptr(keep), (float)a.keep_scale, ptr(post_g),
                               ptr(post_b), ptr(scale), ptr(pre_g), ptr(pre_b), out_ptr(y), out_ptr(n), stats ? stats->data_ptr<float>() : nullptr, rows,
                               D, a.rms, (float)a.eps, type_code(x.scalar_type()), param_code(post_g, scale, pre_g), stream_of(x));
  });
  return {y, n};
}

// Nothing but the inputs and two statistics per norm and row are kept: the backward forms y again from what it reads anyway.
struct GatedNorm : torch::autograd::Function<GatedNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& u, const OptTensor& z, const OptTensor& post_g,
                               const OptTensor& post_b, const OptTensor& scale, const OptTensor& pre_g, const OptTensor& pre_b, const OptTensor& keep,
                               const GatedArgs& a) {
    Tensor stats;
    auto [y, n] = gated_norm_raw(x, or_none(u), or_none(z), or_none(keep), or_none(post_g), or_none(post_b), or_none(scale), or_none(pre_g),
                                 or_none(pre_b), a, &stats);
    ctx->save_for_backward({x, or_none(u), or_none(z), or_none(post_g), or_none(post_b), or_none(scale), or_none(pre_g), or_none(pre_b), or_none(keep), stats});
    ctx->saved_data["keep_scale"] = a.keep_scale;
    ctx->saved_data["eps"] = a.eps;
    ctx->saved_data["rms"] = a.rms;
    ctx->set_materialize_grads(false);
    return n.defined() ? variable_list{y, n} : variable_list{y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0], &u = s[1], &z = s[2], &post_g = s[3], &post_b = s[4], &scale = s[5], &pre_g = s[6], &pre_b = s[7], &keep = s[8], &stats = s[9];
    const Tensor dy = grads[0], dn = grads.size() > 1 ? grads[1] : Tensor();
    variable_list out(10);
    if (!dy.defined() && !dn.defined()) return out;
    const int64_t D = x.size(-1);
    for (const Tensor& d : {dy, dn})
      if (d.defined()) check_same(d, x, "gated_residual_norm", "gradient");
    const Rows xr(x, D), ur(u, D), zr(z, D), dyr(dy, D), dnr(dn, D);
    const int64_t rows = xr.t.size(0);
    const Tensor* of[8] = {&x, &u, &z, &post_g, &post_b, &scale, &pre_g, &pre_b};
    int vectors = 0;
    bool wanted[8];
    for (int i = 0, edge = 0; i < 8; ++i) {                   // (operands that are absent have no edge)
      wanted[i] = of[i]->defined() && ctx->needs_input_grad(edge++);
      if (wanted[i] && i < 3) out[i] = contiguous_like(x);
      vectors += wanted[i] && i >= 3;
    }
    if (vectors) {
      const Tensor& any = post_g.defined() ? post_g : scale.defined() ? scale : pre_g;
      const int64_t piece = 16 / (int64_t)any.element_size(), step = (D + piece - 1) / piece * piece;      // (each begins at 16 bytes)
      const Tensor flat = at::empty({vectors * step}, any.options().requires_grad(false));
      for (int i = 3, k = 0; i < 8; ++i)
        if (wanted[i]) out[i] = part_of(flat, step * k++, D);
    }
    const int code = type_code(x.scalar_type());
    const c10::DeviceGuard guard(x.device());
    const Tensor ws = bytes_on(x, lib.gated_norm_bwd_workspace(rows, D, code));
    entry("mbvae_gated_norm_bwd", [&] {
      return lib.gated_norm_bwd(ptr(xr.t), xr.ld, ptr(ur.t), ur.ld, ptr(zr.t), zr.ld, (const uint8_t*)ptr(keep),
                                 (float)ctx->saved_data["keep_scale"].toDouble(), ptr(post_g), ptr(post_b), ptr(scale), ptr(pre_g),
                                 stats.data_ptr<float>(), ptr(dyr.t), dyr.ld, ptr(dnr.t), dnr.ld, out_ptr(out[0]), out_ptr(out[1]), out_ptr(out[2]),
                                 out_ptr(out[5]), out_ptr(out[3]), out_ptr(out[4]), out_ptr(out[6]), out_ptr(out[7]), rows, D,
                                 ctx->saved_data["rms"].toBool(), (float)ctx->saved_data["eps"].toDouble(), code, param_code(post_g, scale, pre_g),
                                 ws.mutable_data_ptr(), ws.numel(), stream_of(x));
    });
    return differentiable_once(std::move(out), "gated_residual_norm");
  }
};

std::tuple<Tensor, OptTensor> gated_residual_norm(const Tensor& x, const OptTensor& u, const OptTensor& z, const OptTensor& keep, double keep_scale,
                                                  const OptTensor& post_g, const OptTensor& post_b, const OptTensor& scale, const OptTensor& pre_g,
                                                  const OptTensor& pre_b, bool rms, double eps) {
  const char* what = "gated_residual_norm";
  check_typed(x, what, "x");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= 8192, what, ": the last dimension must hold 1 to 8192 values, got shape ", x.sizes());
  TORCH_CHECK_VALUE(eps >= 0, what, ": eps must not be negative");
  const int64_t D = x.size(-1);
  const auto like_x = [&](const OptTensor& t, const char* name) {
    if (!present(t)) return;
    check_same(*t, x, what, name);
    TORCH_CHECK_VALUE(t->sizes() == x.sizes(), what, ": ", name, " must have x's shape ", x.sizes(), ", got ", t->sizes());
  };
  like_x(u, "u");
  like_x(z, "z");
  OptTensor mask;
  if (present(keep)) {
    TORCH_CHECK_VALUE(keep->sizes() == x.sizes() && (keep->scalar_type() == at::kByte || keep->scalar_type() == at::kBool) && keep->device() == x.device(),
                      what, ": keep must be a uint8 or bool mask of x's shape on x's device");
    mask = keep->contiguous();
  }
  const Tensor* first = nullptr;
  const auto param = [&](const OptTensor& t, const char* name) -> OptTensor {
    if (!present(t)) return std::nullopt;
    check_typed(*t, what, name);
    if (first) check_same(*t, *first, what, name);
    TORCH_CHECK_VALUE(t->device() == x.device(), what, ": ", name, ": expected a tensor on ", x.device(), ", got one on ", t->device());
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == D, what, ": ", name, " must have shape [", D, "], got ", t->sizes());
    first = &*t;
    return t->resolve_neg().contiguous();
  };
  const OptTensor pg = param(post_g, "post gamma"), pb = param(post_b, "post beta"), sc = param(scale, "res_scale"), ng = param(pre_g, "pre gamma"),
                  nb = param(pre_b, "pre beta");
  TORCH_CHECK_VALUE((pg || !pb) && (ng || !nb), what, ": a norm needs its gamma");
  const GatedArgs a{keep_scale, eps, rms};
  if (at::GradMode::is_enabled()) {
    bool wanted = x.requires_grad();
    for (const OptTensor* t : {&u, &z, &pg, &pb, &sc, &ng, &nb}) wanted = wanted || (present(*t) && (*t)->requires_grad());
    if (wanted) {
      variable_list out = GatedNorm::apply(x, u, z, pg, pb, sc, ng, nb, mask, a);
      return {out[0], out.size() > 1 ? OptTensor(out[1]) : std::nullopt};
    }
  }
  auto [y, n] = gated_norm_raw(x, or_none(u), or_none(z), or_none(mask), or_none(pg), or_none(pb), or_none(sc), or_none(ng), or_none(nb), a, nullptr);
  return {y, n.defined() ? OptTensor(n) : std::nullopt};
}

// ------------------------------------------------------------------------------------------------ gradient norm and clipping
// Whether grad_clip takes these gradients (what it refuses with an error).
bool grad_clip_takes(const std::vector<Tensor>& grads) {
  const bool tangents = tangents_possible();
  for (const Tensor& g : grads)
    if (!g.is_cuda() || g.device() != grads[0].device() || g.layout() != at::kStrided || type_code(g.scalar_type()) < 0 || g.requires_grad() ||
        !g.has_storage() || g.unsafeGetTensorImpl()->is_python_dispatch() || (tangents && g._fw_grad(0).defined()) || !(g.is_contiguous() || g.is_non_overlapping_and_dense()))
      return false;
  return true;
}

// max_norm < 0: the norm alone.  out empty: in place.
Tensor grad_clip(const std::vector<Tensor>& grads, const std::vector<Tensor>& out, double max_norm, double p) {
  const char* what = "gradient norm";
  TORCH_CHECK_VALUE(p == 1 || p == 2 || p == std::numeric_limits<double>::infinity(), what, ": norm_type is 1, 2 or infinity, got ", p);
  const size_t count = grads.size();
  const bool write = max_norm >= 0, apart = write && !out.empty(), tangents = tangents_possible();
  std::vector<const void*> src(count);
  std::vector<void*> dst(write ? count : 0);
  std::vector<int64_t> numel(count);
  std::vector<int32_t> types(count);
  const auto device = grads[0].device();
  for (size_t i = 0; i < count; ++i) {
    const Tensor& g = grads[i];
    TORCH_CHECK(g.is_cuda() && g.device() == device, what, ": all gradients must be on one GPU; the HIP path has no CPU fallback");
    types[i] = type_code(g.scalar_type());
    TORCH_CHECK(types[i] >= 0 && g.layout() == at::kStrided, what, ": expected dense float32, bfloat16 or float16 gradients, got ", g.scalar_type());
    if (tangents) check_no_tangent(g, what);
    TORCH_CHECK_VALUE(!g.requires_grad(), what, ": expected gradients (p.grad), got a tensor that requires gradients itself");
    TORCH_CHECK_VALUE(g.is_contiguous() || g.is_non_overlapping_and_dense(), what, ": a gradient must fill its memory densely, got strides ", g.strides(),
                      " for shape ", g.sizes());
    numel[i] = g.numel();
    src[i] = write && !apart ? dst[i] = g.mutable_data_ptr() : g.const_data_ptr();
    if (apart) {
      const Tensor& o = out[i];
      TORCH_CHECK_VALUE(o.scalar_type() == g.scalar_type() && o.device() == device && o.sizes() == g.sizes() &&
                            (numel[i] <= 1 || o.strides() == g.strides()) && o.layout() == at::kStrided && !o.requires_grad(),
                        what, ": an output must have its gradient's type, shape, strides and device");
      TORCH_CHECK_VALUE(o.is_neg() == g.is_neg(), what, ": an output must hold its values with the sign its gradient does");
      if (tangents) check_no_tangent(o, what);
      dst[i] = o.mutable_data_ptr();
    }
  }
  if (write)
    for (const Tensor& t : apart ? out : grads)
      TORCH_CHECK(!t.is_inference() || c10::InferenceMode::is_enabled(), what, ": an inference tensor may not be written outside inference mode");
  Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat));
  const Tensor ws = bytes_on(grads[0], lib.grad_clip_workspace((int64_t)count));
  const c10::DeviceGuard guard(device);
  entry("mbvae_grad_clip", [&] {
    return lib.grad_clip(src.data(), write ? dst.data() : nullptr, numel.data(), types.data(), (int64_t)count, p, max_norm, norm.data_ptr<float>(),
                          ws.mutable_data_ptr(), ws.numel(), stream_of(grads[0]));
  });
  if (write)                                                 // (behind the call: one that is refused has written nothing)
    for (const Tensor& t : apart ? out : grads) t.unsafeGetTensorImpl()->bump_version();
  return norm;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("profile", [](bool on) { profiling = on; });
  m.def("embedding", &embedding);
  m.def("gated_residual_norm", &gated_residual_norm);
  m.def("grad_clip", &grad_clip);
  m.def("grad_clip_takes", &grad_clip_takes);
}
