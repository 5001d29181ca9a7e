// native_mixers.cpp — the host path of the gated delta rule and of causal attention: argument
// checks, output and scratch allocation, the launches through libkdecay.so's C ABI,
// and the autograd node of the scan.
//
// Scratch comes from torch's allocator on the current stream, one allocation per
// call: no two calls share it, on any stream, thread or captured graph.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/torch.h>

#include <array>

#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>

#include "kattn.h"
#include "kdecay.h"
#include "kdelta.h"

namespace py = pybind11;
using at::Tensor;

namespace {

int code_of(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return KDECAY_F32;
    case at::kBFloat16: return KDECAY_BF16;
    case at::kHalf: return KDECAY_F16;
    default:
      TORCH_CHECK_TYPE(false, "kilat_amd: ", name, " dtype ", t.scalar_type(), " is not float32/bfloat16/float16");
  }
}

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == 0, "kilat_amd: ", what, " failed (code ", rc, "): ", kdecay_last_error_string());
}

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void require_hip(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), "kilat_amd: ", name, " is on ", t.device(), "; the kilat_amd kernels run on HIP devices only");
}

// q, k [B, Hq or Hk, N, Dk] and v [B, Hv, N, Dv], one type and device.
void check_qkv(const Tensor& q, const Tensor& k, const Tensor& v) {
  code_of(q, "q");
  TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                   "kilat_amd: q, k and v must have one dtype, got ", q.scalar_type(), ", ", k.scalar_type(), " and ",
                   v.scalar_type());
  TORCH_CHECK_VALUE(k.device() == q.device() && v.device() == q.device(), "kilat_amd: q, k and v must be on one device");
}

void check_float(const Tensor& t, const Tensor& q, const char* name) {
  TORCH_CHECK_TYPE(t.is_floating_point(), "kilat_amd: ", name, " must be a floating point tensor");
  TORCH_CHECK_VALUE(t.device() == q.device(), "kilat_amd: ", name, " must be on q's device");
}

// `t` as float32 (recorded by autograd where it converts).
Tensor as_float(const Tensor& t) { return t.to(at::kFloat).resolve_neg(); }

// Whether the kernels read (and write) `t` as it lies: channels adjacent, every row aligned to
// 16 bytes.  For head dims that are multiples of 8.
bool rows_ok(const Tensor& t) {
  if (reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 || t.stride(3) != 1) return false;
  for (int64_t k = 0; k < 3; ++k)
    if (t.size(k) > 1 && t.stride(k) * t.element_size() % 16) return false;
  return true;
}

// `t` as the kernels read it, its memory holding its values.  (A contiguous tensor off the
// alignment is its own contiguous().)
Tensor as_rows(const Tensor& t) {
  const Tensor r = t.resolve_neg();
  return rows_ok(r) ? r : r.clone(at::MemoryFormat::Contiguous);
}

// A new tensor of `like`'s shape and, as far as the kernels write it, its layout.
Tensor new_like(const Tensor& like) {
  Tensor r = at::empty_like(like);
  if (!rows_ok(r)) r = at::empty(like.sizes(), like.options());
  return r;
}

// Channels (of dimension `dim`) padded with zeros to a multiple of 8.
Tensor pad8(const Tensor& t, int64_t dim) {
  const int64_t n = t.size(dim);
  if (n % 8 == 0) return t;
  std::vector<int64_t> pad(2 * (t.dim() - dim), 0);
  pad.back() = 8 - n % 8;
  return at::constant_pad_nd(t, pad, 0);
}

// cu_seqlens, or an undefined tensor.
Tensor check_cu(const std::optional<Tensor>& cu, const Tensor& q) {
  if (!cu.has_value() || !cu->defined()) return Tensor();
  TORCH_CHECK_TYPE(cu->scalar_type() == at::kInt || cu->scalar_type() == at::kLong,
                   "kilat_amd: cu_seqlens must be int32 or int64");
  TORCH_CHECK_VALUE(cu->dim() == 1 && cu->numel() >= 2, "kilat_amd: cu_seqlens must be [sequences + 1], got shape ",
                    cu->sizes());
  TORCH_CHECK_VALUE(cu->device() == q.device(), "kilat_amd: cu_seqlens must be on q's device");
  TORCH_CHECK_VALUE(q.size(0) == 1, "kilat_amd: a packed batch (cu_seqlens) has B=1, got B=", q.size(0));
  TORCH_CHECK_VALUE(q.size(2) <= 0x7fffffff, "kilat_amd: a packed batch has at most 2^31 - 1 rows");
  return *cu;
}

Tensor as_cu(const Tensor& cu) { return cu.defined() ? cu.to(at::kInt).contiguous() : cu; }

bool grad_wanted(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t->defined() && ((at::GradMode::is_enabled() && t->requires_grad()) || t->_fw_grad(0).defined())) return true;
  return false;
}

Tensor optional(const std::optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }
const void* cptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; }

void copy_strides(int64_t* to, const Tensor& t) {
  for (int64_t k = 0; k < t.dim(); ++k) to[k] = k < 3 && t.size(k) == 1 ? 0 : t.stride(k);
}

std::array<int64_t, 4> strides(const Tensor& t) {
  std::array<int64_t, 4> r;
  copy_strides(r.data(), t);
  return r;
}

// ---------------------------------------------------------------------------
// gated_delta_scan
// ---------------------------------------------------------------------------
kdelta_problem problem(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta,
                       const Tensor& cu, const Tensor& init, double scale) {
  kdelta_problem p = {};
  p.q = q.const_data_ptr(), p.k = k.const_data_ptr(), p.v = v.const_data_ptr();
  p.g = static_cast<const float*>(g.const_data_ptr()), p.beta = static_cast<const float*>(beta.const_data_ptr());
  p.cu_seqlens = static_cast<const int32_t*>(cptr(cu));
  p.init = static_cast<const float*>(cptr(init));
  copy_strides(p.q_strides, q), copy_strides(p.k_strides, k), copy_strides(p.v_strides, v);
  copy_strides(p.g_strides, g), copy_strides(p.beta_strides, beta);
  p.B = v.size(0), p.Hk = k.size(1), p.H = v.size(1), p.N = v.size(2), p.Dk = k.size(3), p.Dv = v.size(3);
  p.sequences = cu.defined() ? cu.numel() - 1 : p.B;
  p.scale = static_cast<float>(scale);
  p.dtype = code_of(q, "q");
  return p;
}

Tensor bytes_on(const Tensor& like, size_t n) {
  return at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte));
}

struct Scanned {
  Tensor o, final, saved;
};

Scanned delta_forward(const kdelta_problem& p, const Tensor& v, bool want_final, bool save) {
  const c10::DeviceGuard guard(v.device());
  const auto f32 = v.options().dtype(at::kFloat);
  Scanned r;
  r.o = new_like(v);
  if (want_final) r.final = at::empty({p.sequences, p.H, p.Dk, p.Dv}, f32);
  if (save) r.saved = at::empty({static_cast<int64_t>(kdelta_scan_saved_floats(&p))}, f32);
  const size_t n = kdelta_scan_workspace_bytes(&p);
  const Tensor ws = bytes_on(v, n);
  check_rc(kdelta_scan_fwd(&p, r.o.data_ptr(), strides(r.o).data(), fptr(r.final), save && r.saved.numel() ? fptr(r.saved) : nullptr,
                           ws.data_ptr(), n, stream_of(v)),
           "kdelta_scan_fwd");
  return r;
}

// Inputs as the kernels read them; outputs o and the final state.
struct DeltaNode : torch::autograd::Function<DeltaNode> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k,
                                                const Tensor& v, const Tensor& g, const Tensor& beta,
                                                const std::optional<Tensor>& init, const std::optional<Tensor>& cu,
                                                double scale) {
    const kdelta_problem p = problem(q, k, v, g, beta, optional(cu), optional(init), scale);
    const Scanned r = delta_forward(p, v, true, true);
    ctx->set_materialize_grads(false);
    ctx->saved_data["scale"] = scale;
    ctx->save_for_backward({q, k, v, g, beta, optional(init), optional(cu), r.saved});
    return {r.o, r.final};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &g = saved[3], &beta = saved[4], &init = saved[5],
                 &cu = saved[6], &states = saved[7];
    const kdelta_problem p = problem(q, k, v, g, beta, cu, init, ctx->saved_data["scale"].toDouble());
    const c10::DeviceGuard guard(v.device());
    const Tensor d_o = grads[0].defined() ? as_rows(grads[0].to(v.scalar_type())) : at::zeros_like(v);
    const Tensor d_final = grads[1].defined() ? grads[1].to(at::kFloat).resolve_neg().contiguous() : Tensor();
    const auto f32 = v.options().dtype(at::kFloat);
    const Tensor dq = new_like(q), dk = new_like(k), dv = new_like(v);
    const Tensor dg = at::empty({p.B, p.H, p.N}, f32), dbeta = at::empty({p.B, p.H, p.N}, f32);
    const Tensor d_init = init.defined() ? at::empty(init.sizes(), f32) : Tensor();
    const size_t n = kdelta_scan_bwd_workspace_bytes(&p);
    const Tensor ws = bytes_on(v, n);
    check_rc(kdelta_scan_bwd(&p, d_o.const_data_ptr(), strides(d_o).data(), fptr(d_final), fptr(states), dq.data_ptr(),
                             strides(dq).data(), dk.data_ptr(), strides(dk).data(), dv.data_ptr(), strides(dv).data(),
                             fptr(dg), fptr(dbeta), fptr(d_init), ws.data_ptr(), n, stream_of(v)),
             "kdelta_scan_bwd");
    return {dq, dk, dv, dg, dbeta, d_init, Tensor(), Tensor()};
  }
};

// A tensor made under inference_mode cannot be saved for a backward.
Tensor saveable(const Tensor& t) { return t.defined() && t.is_inference() ? t.clone() : t; }

py::object delta_scan(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& g_in,
                      const Tensor& beta_in, std::optional<double> scale_in, const std::optional<Tensor>& init_in,
                      bool want_final, const std::optional<Tensor>& cu_in) {
  check_qkv(q_in, k_in, v_in);
  TORCH_CHECK_VALUE(q_in.dim() == 4 && k_in.dim() == 4 && v_in.dim() == 4,
                    "kilat_amd: q, k and v must be [B,H,N,D], got shapes ", q_in.sizes(), ", ", k_in.sizes(), " and ",
                    v_in.sizes());
  TORCH_CHECK_VALUE(q_in.sizes() == k_in.sizes(), "kilat_amd: q and k must have one shape, got ", q_in.sizes(), " and ",
                    k_in.sizes());
  TORCH_CHECK_VALUE(v_in.size(0) == k_in.size(0) && v_in.size(2) == k_in.size(2),
                    "kilat_amd: v must have k's batch and rows, got ", v_in.sizes(), " and ", k_in.sizes());
  const int64_t B = v_in.size(0), Hk = k_in.size(1), H = v_in.size(1), N = v_in.size(2), Dk = k_in.size(3),
                Dv = v_in.size(3);
  TORCH_CHECK_VALUE(Hk >= 1 && H >= 1 && H % Hk == 0, "kilat_amd: v's heads (", H, ") must be a multiple of k's (", Hk, ")");
  TORCH_CHECK_VALUE(Dk >= 1 && Dk <= KDELTA_MAX_DK && Dv >= 1 && Dv <= KDELTA_MAX_DV, "kilat_amd: head dims of k (", Dk,
                    ") and v (", Dv, ") must be 1..", KDELTA_MAX_DK, " and 1..", KDELTA_MAX_DV);
  for (const Tensor* t : {&g_in, &beta_in})
    TORCH_CHECK_VALUE(t->dim() == 3 && t->size(0) == B && t->size(1) == H && t->size(2) == N, "kilat_amd: ",
                      t == &g_in ? "g" : "beta", " must be [B,H,N]=", at::IntArrayRef({B, H, N}), ", got ", t->sizes());
  check_float(g_in, q_in, "g"), check_float(beta_in, q_in, "beta");
  Tensor cu = check_cu(cu_in, q_in), init = optional(init_in);
  if (init.defined()) {
    const int64_t S = cu.defined() ? cu.numel() - 1 : B;
    TORCH_CHECK_VALUE(init.dim() == 4 && init.size(0) == S && init.size(1) == H && init.size(2) == Dk && init.size(3) == Dv,
                      "kilat_amd: initial_state must be ", at::IntArrayRef({S, H, Dk, Dv}), ", got ", init.sizes());
    check_float(init, q_in, "initial_state");
  }
  require_hip(q_in, "q");
  cu = as_cu(cu);
  const double scale = scale_in.has_value() ? *scale_in : 1.0 / std::sqrt(static_cast<double>(Dk));
  Tensor q = as_rows(pad8(q_in, 3)), k = as_rows(pad8(k_in, 3)), v = as_rows(pad8(v_in, 3));
  Tensor g = as_float(g_in), beta = as_float(beta_in);
  if (init.defined()) init = pad8(pad8(as_float(init), 3), 2).contiguous();
  Tensor o, final;
  {
    py::gil_scoped_release nogil;
    if (grad_wanted({&q, &k, &v, &g, &beta, &init})) {
      q = saveable(q), k = saveable(k), v = saveable(v), g = saveable(g), beta = saveable(beta), init = saveable(init);
      const auto opt = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
      const auto r = DeltaNode::apply(q, k, v, g, beta, opt(init), opt(saveable(cu)), scale);
      o = r[0], final = r[1];
    } else {
      at::AutoDispatchBelowADInplaceOrView below;  // new buffers only: nothing to record
      const Scanned r = delta_forward(problem(q, k, v, g, beta, cu, init, scale), v, want_final, false);
      o = r.o, final = r.final;
    }
    if (Dv % 8) o = at::empty_like(v_in).copy_(o.narrow(3, 0, Dv));
    if (want_final && (Dk % 8 || Dv % 8)) final = final.narrow(2, 0, Dk).narrow(3, 0, Dv).contiguous();
  }
  return want_final ? py::object(py::make_tuple(o, final)) : py::cast(o);
}

// ---------------------------------------------------------------------------
// gated_delta_step
// ---------------------------------------------------------------------------
std::pair<uintptr_t, uintptr_t> extent(const Tensor& t) {  // of a contiguous tensor
  const uintptr_t p = reinterpret_cast<uintptr_t>(t.const_data_ptr());
  return {p, p + t.numel() * t.element_size()};
}

bool meets(const Tensor& a, const Tensor& b) {
  const auto [x, y] = extent(a);
  const auto [z, w] = extent(b);
  return x < w && z < y;
}

py::object delta_step(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& g_in,
                      const Tensor& beta_in, const Tensor& state_in, std::optional<double> scale_in,
                      const py::object& out_o, const py::object& new_o, std::optional<at::ScalarType> out_dtype) {
  at::NoGradGuard no_grad;
  check_qkv(q_in, k_in, v_in);
  TORCH_CHECK_VALUE(state_in.dim() == 4, "kilat_amd: state must be [B,H,Dk,Dv], got ", state_in.sizes());
  const int64_t B = state_in.size(0), H = state_in.size(1), Dk = state_in.size(2), Dv = state_in.size(3);
  TORCH_CHECK_VALUE(q_in.dim() == 3 && q_in.size(0) == B && q_in.size(2) == Dk && q_in.sizes() == k_in.sizes(),
                    "kilat_amd: q and k must be [B,Hk,Dk] with B=", B, ", Dk=", Dk, ", got ", q_in.sizes(), " and ",
                    k_in.sizes());
  const int64_t Hk = k_in.size(1);
  TORCH_CHECK_VALUE(Hk >= 1 && H >= 1 && H % Hk == 0, "kilat_amd: v's heads (", H, ") must be a multiple of k's (", Hk, ")");
  TORCH_CHECK_VALUE(v_in.dim() == 3 && v_in.size(0) == B && v_in.size(1) == H && v_in.size(2) == Dv,
                    "kilat_amd: v must be [B,H,Dv]=", at::IntArrayRef({B, H, Dv}), ", got ", v_in.sizes());
  TORCH_CHECK_VALUE(Dk >= 1 && Dk <= KDELTA_MAX_DK && Dv >= 1 && Dv <= KDELTA_MAX_DV, "kilat_amd: head dims of k (", Dk,
                    ") and v (", Dv, ") must be 1..", KDELTA_MAX_DK, " and 1..", KDELTA_MAX_DV);
  for (const Tensor* t : {&g_in, &beta_in})
    TORCH_CHECK_VALUE(t->dim() == 2 && t->size(0) == B && t->size(1) == H, "kilat_amd: ", t == &g_in ? "g" : "beta",
                      " must be [B,H]=", at::IntArrayRef({B, H}), ", got ", t->sizes());
  check_float(g_in, q_in, "g"), check_float(beta_in, q_in, "beta"), check_float(state_in, q_in, "state");
  require_hip(q_in, "q");
  const Tensor q = q_in.resolve_neg().contiguous(), k = k_in.resolve_neg().contiguous(),
               v = v_in.resolve_neg().contiguous();
  const Tensor g = as_float(g_in).contiguous(), beta = as_float(beta_in).contiguous();
  const Tensor state = as_float(state_in).contiguous();
  const c10::DeviceGuard guard(q.device());
  Tensor next, out;
  if (!new_o.is_none()) {
    next = new_o.cast<Tensor>();
    TORCH_CHECK_VALUE(next.scalar_type() == at::kFloat && next.is_contiguous() && next.sizes() == state_in.sizes() &&
                          next.device() == q.device() && !next.is_neg(),
                      "kilat_amd: new_state must be a contiguous float32 ", state_in.sizes(), " tensor on q's device");
  } else {
    next = at::empty(state_in.sizes(), state.options());
  }
  if (!out_o.is_none()) {
    out = out_o.cast<Tensor>();
    TORCH_CHECK_VALUE(out.is_contiguous() && out.sizes() == v_in.sizes() && out.device() == q.device() && !out.is_neg(),
                      "kilat_amd: out must be a contiguous ", v_in.sizes(), " tensor on q's device");
  } else {
    out = at::empty(v_in.sizes(), v.options().dtype(out_dtype.value_or(v.scalar_type())));
  }
  TORCH_CHECK_TYPE(out.scalar_type() == v.scalar_type() || out.scalar_type() == at::kFloat,
                   "kilat_amd: out dtype must be v's dtype or float32");
  // Outputs in memory that other workgroups still read: through new buffers.  The state
  // itself is not: each workgroup reads what it then writes.
  const bool same = next.const_data_ptr() == state.const_data_ptr();
  bool next_apart = same || !meets(next, state), out_apart = !meets(out, state) && !meets(out, next);
  for (const Tensor* t : {&q, &k, &v, &g, &beta}) next_apart = next_apart && !meets(next, *t), out_apart = out_apart && !meets(out, *t);
  const Tensor next_k = next_apart ? next : at::empty_like(next), out_k = out_apart ? out : at::empty_like(out);
  const double scale = scale_in.has_value() ? *scale_in : 1.0 / std::sqrt(static_cast<double>(Dk));
  {
    py::gil_scoped_release nogil;
    check_rc(kdelta_step(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), code_of(q, "q"),
                         static_cast<const float*>(g.const_data_ptr()), static_cast<const float*>(beta.const_data_ptr()),
                         static_cast<const float*>(state.const_data_ptr()), fptr(next_k), out_k.data_ptr(),
                         code_of(out, "out"), B, Hk, H, Dk, Dv, static_cast<float>(scale), stream_of(q)),
             "kdelta_step");
    if (!next_apart) next.copy_(next_k);
    if (!out_apart) out.copy_(out_k);
  }
  return py::make_tuple(out_o.is_none() ? py::cast(out) : out_o, new_o.is_none() ? py::cast(next) : new_o);
}

// ---------------------------------------------------------------------------
// causal_attention
// ---------------------------------------------------------------------------
Tensor attention(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, std::optional<double> scale_in,
                 const std::optional<Tensor>& cu_in) {
  check_qkv(q_in, k_in, v_in);
  TORCH_CHECK_VALUE(q_in.dim() == 4 && k_in.dim() == 4 && v_in.dim() == 4,
                    "kilat_amd: q, k and v must be [B,H,N,D], got shapes ", q_in.sizes(), ", ", k_in.sizes(), " and ",
                    v_in.sizes());
  const int64_t B = q_in.size(0), H = q_in.size(1), N = q_in.size(2), Dk = q_in.size(3), Hk = k_in.size(1),
                Dv = v_in.size(3);
  TORCH_CHECK_VALUE(k_in.size(0) == B && v_in.size(0) == B && k_in.size(2) == N && v_in.size(2) == N &&
                        k_in.size(3) == Dk && v_in.size(1) == Hk,
                    "kilat_amd: k and v must be [B,Hk,N,Dk] and [B,Hk,N,Dv] for q ", q_in.sizes(), ", got ", k_in.sizes(),
                    " and ", v_in.sizes());
  TORCH_CHECK_VALUE(Hk >= 1 && H >= 1 && H % Hk == 0, "kilat_amd: q's heads (", H, ") must be a multiple of k's (", Hk, ")");
  TORCH_CHECK_VALUE(Dk >= 1 && Dk <= KATTN_MAX_DK && Dv >= 1 && Dv <= KATTN_MAX_DV, "kilat_amd: head dims of k (", Dk,
                    ") and v (", Dv, ") must be 1..", KATTN_MAX_DK, " and 1..", KATTN_MAX_DV);
  const Tensor cu_any = check_cu(cu_in, q_in);
  require_hip(q_in, "q");
  TORCH_CHECK(!grad_wanted({&q_in, &k_in, &v_in}),
              "kilat_amd: causal_attention has no backward; call it under torch.no_grad()");
  at::AutoDispatchBelowADInplaceOrView below;  // new buffers only: nothing to record
  const Tensor q = as_rows(pad8(q_in, 3)), k = as_rows(pad8(k_in, 3)), v = as_rows(pad8(v_in, 3)), cu = as_cu(cu_any);
  const c10::DeviceGuard guard(q.device());
  // Laid out like q: rows of all heads together where q's are.
  const bool tokens = H > 1 && N > 1 && q_in.stride(1) < q_in.stride(2);
  const auto empty = [&](int64_t D) {
    return tokens ? at::empty({B, N, H, D}, q.options()).transpose(1, 2) : at::empty({B, H, N, D}, q.options());
  };
  const Tensor o = empty(v.size(3));
  kattn_problem p = {};
  p.q = q.const_data_ptr(), p.k = k.const_data_ptr(), p.v = v.const_data_ptr();
  p.cu_seqlens = static_cast<const int32_t*>(cptr(cu));
  copy_strides(p.q_strides, q), copy_strides(p.k_strides, k), copy_strides(p.v_strides, v);
  p.B = B, p.Hk = Hk, p.H = H, p.N = N, p.Dk = q.size(3), p.Dv = v.size(3);
  p.sequences = cu.defined() ? cu.numel() - 1 : B;
  p.scale = static_cast<float>(scale_in.has_value() ? *scale_in : 1.0 / std::sqrt(static_cast<double>(Dk)));
  p.dtype = code_of(q, "q");
  check_rc(kattn_fwd(&p, o.data_ptr(), strides(o).data(), stream_of(q)), "kattn_fwd");
  if (Dv % 8) return empty(Dv).copy_(o.narrow(3, 0, Dv));
  return o;
}

}  // namespace

void bind_mixers(py::module_& m) {
  m.def("gated_delta_scan", &delta_scan);
  m.def("gated_delta_step", &delta_step);
  m.def("causal_attention", &attention, py::call_guard<py::gil_scoped_release>());
}
