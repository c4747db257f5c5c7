// genie_tk._C — thin PyTorch binding over the C ABI in include/genie_tk.h.
//
// Mirrors the operator surface of the reference extension
// (kernels/bindings.cpp:69-101: triangle_mul_outgoing/incoming,
// triangle_attention_starting/ending, layernorm, fused_layernorm_linear) and
// adds the fused module entry points used by the modules' _forward_cuda.
// Tensors are checked, made contiguous, and every launch goes to the caller's
// current HIP stream; scratch comes from torch's caching allocator.
#include <c10/hip/HIPStream.h>
#include <ATen/MemoryOverlap.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <algorithm>
#include <array>
#include <functional>
#include <limits>
#include <utility>
#include <vector>

#include "../../include/genie_tk.h"

namespace {

int gtk_dtype_of(const at::Tensor& t, const char* what) {
  if (t.scalar_type() == at::kFloat) return GTK_F32;
  if (t.scalar_type() == at::kBFloat16) return GTK_BF16;
  TORCH_CHECK(false, "genie_tk._C: ", what, " must be float32 or bfloat16, got ", t.scalar_type());
  return -1;
}

void check_rc(int rc) { TORCH_CHECK(rc == GTK_OK, "genie_tk._C: ", gtk_last_error()); }

void* cur_stream(const at::Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

void check_gpu(const at::Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda(), what, " must be CUDA tensor");
}

// Every tensor whose data pointer reaches a kernel must live on the device the
// kernels run on (the device of the main input): a host or foreign-device
// pointer would be dereferenced by the GPU.
void check_on(const at::Tensor& t, const at::Tensor& like, const char* what) {
  if (!t.defined()) return;
  TORCH_CHECK(t.device() == like.device(), "genie_tk._C: ", what, " is on ", t.device(),
              " but the input is on ", like.device());
}
void check_on(const c10::optional<at::Tensor>& t, const at::Tensor& like, const char* what) {
  if (t.has_value()) check_on(*t, like, what);
}
void check_all_on(const std::vector<at::Tensor>& ts, const at::Tensor& like, const char* what) {
  for (const auto& t : ts) check_on(t, like, what);
}

at::Tensor f32c(const at::Tensor& t) { return t.to(at::kFloat).contiguous(); }

at::Tensor workspace(const at::Tensor& like, size_t bytes) {
  return at::empty({(int64_t)std::max<size_t>(bytes, 1)}, like.options().dtype(at::kByte));
}

// ---------------------------------------------------------------------------
// Reference operator surface
// ---------------------------------------------------------------------------
at::Tensor layernorm(const at::Tensor& x, const at::Tensor& gamma, const at::Tensor& beta,
                     double eps) {
  check_gpu(x, "x");
  check_on(gamma, x, "gamma");
  check_on(beta, x, "beta");
  const at::DeviceGuard guard(x.device());
  TORCH_CHECK(x.dim() >= 1, "x must have at least one dimension");
  auto xc = x.contiguous();
  const int64_t d = xc.size(-1);
  const int64_t rows = d ? xc.numel() / d : 0;
  auto g = f32c(gamma), b = f32c(beta);
  TORCH_CHECK(g.numel() == d && b.numel() == d, "gamma/beta must have ", d, " elements");
  auto y = at::empty_like(xc);
  check_rc(gtk_layernorm(xc.data_ptr(), y.data_ptr(), g.data_ptr<float>(), b.data_ptr<float>(),
                         rows, d, (float)eps, gtk_dtype_of(xc, "x"), cur_stream(xc)));
  return y;
}

// LayerNorm + Linear over the last dimension of x; weight [D_IN, D_OUT]
// (layout GTK_W_IN_OUT, the reference's operator) or [D_OUT, D_IN]
// (GTK_W_OUT_IN, nn.Linear.weight).
static at::Tensor layernorm_linear_impl(const at::Tensor& x, const at::Tensor& gamma,
                                        const at::Tensor& beta, const at::Tensor& weight,
                                        const c10::optional<at::Tensor>& bias, double eps,
                                        int layout) {
  check_gpu(x, "x");
  check_on(weight, x, "weight");
  check_on(gamma, x, "gamma");
  check_on(beta, x, "beta");
  check_on(bias, x, "bias");
  const at::DeviceGuard guard(x.device());
  auto xc = x.contiguous();
  const int64_t d_in = xc.size(-1);
  const int in_dim = layout == GTK_W_IN_OUT ? 0 : 1;
  TORCH_CHECK(weight.dim() == 2 && weight.size(in_dim) == d_in,
              layout == GTK_W_IN_OUT ? "weight must be [D_IN, D_OUT]" : "weight must be [D_OUT, D_IN]");
  const int64_t d_out = weight.size(1 - in_dim);
  const int64_t rows = d_in ? xc.numel() / d_in : 0;
  auto g = f32c(gamma), b = f32c(beta);
  TORCH_CHECK(g.numel() == d_in && b.numel() == d_in, "gamma/beta must have ", d_in, " elements");
  auto w = weight.contiguous();
  at::Tensor bb;
  if (bias.has_value()) {
    bb = f32c(*bias);
    TORCH_CHECK(bb.numel() == d_out, "bias must have ", d_out, " elements");
  }
  auto sizes = xc.sizes().vec();
  sizes.back() = d_out;
  auto y = at::empty(sizes, xc.options());
  const int dt = gtk_dtype_of(xc, "x");
  auto ws = workspace(xc, gtk_fused_layernorm_linear_workspace_size(d_in, d_out, dt));
  check_rc(gtk_layernorm_linear(xc.data_ptr(), y.data_ptr(), g.data_ptr<float>(),
                                b.data_ptr<float>(), w.data_ptr(), gtk_dtype_of(w, "weight"), layout,
                                bias.has_value() ? bb.data_ptr<float>() : nullptr, rows, d_in, d_out,
                                (float)eps, dt, ws.data_ptr(), ws.numel(), cur_stream(xc)));
  return y;
}

at::Tensor fused_layernorm_linear(const at::Tensor& x, const at::Tensor& gamma,
                                  const at::Tensor& beta, const at::Tensor& weight,
                                  const c10::optional<at::Tensor>& bias, double eps) {
  return layernorm_linear_impl(x, gamma, beta, weight, bias, eps, GTK_W_IN_OUT);
}

at::Tensor layernorm_linear(const at::Tensor& x, const at::Tensor& gamma, const at::Tensor& beta,
                            const at::Tensor& weight, const c10::optional<at::Tensor>& bias,
                            double eps) {
  return layernorm_linear_impl(x, gamma, beta, weight, bias, eps, GTK_W_OUT_IN);
}

at::Tensor triangle_mul_raw(const at::Tensor& a, const at::Tensor& b, const at::Tensor& mask,
                            bool outgoing) {
  check_gpu(a, "a");
  check_on(b, a, "b");
  check_on(mask, a, "mask");
  const at::DeviceGuard guard(a.device());
  TORCH_CHECK(a.dim() == 4 && a.sizes() == b.sizes() && a.size(1) == a.size(2),
              "a and b must both be [B, N, N, C]");
  TORCH_CHECK(a.scalar_type() == b.scalar_type(), "a and b must have the same dtype");
  TORCH_CHECK(mask.numel() == a.size(0) * a.size(1) * a.size(2), "mask must be [B, N, N]");
  auto ac = a.contiguous(), bc = b.contiguous();
  const int64_t B = ac.size(0), N = ac.size(1), C = ac.size(3);
  const int dt = gtk_dtype_of(ac, "a");
  auto x = at::empty_like(ac);
  auto ws = workspace(ac, gtk_triangle_mul_workspace_size(B, N, C, dt));
  auto fn = outgoing ? gtk_triangle_mul_outgoing : gtk_triangle_mul_incoming;
  check_rc(fn(ac.data_ptr(), bc.data_ptr(), nullptr, x.data_ptr(), B, N, C, dt, ws.data_ptr(),
              ws.numel(), cur_stream(ac)));
  return x;
}

at::Tensor triangle_mul_outgoing(const at::Tensor& a, const at::Tensor& b, const at::Tensor& mask) {
  return triangle_mul_raw(a, b, mask, true);
}
at::Tensor triangle_mul_incoming(const at::Tensor& a, const at::Tensor& b, const at::Tensor& mask) {
  return triangle_mul_raw(a, b, mask, false);
}

at::Tensor triangle_attention_raw(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                  const at::Tensor& bias, const at::Tensor& mask, double scale,
                                  bool starting) {
  check_gpu(q, "q");
  check_on(k, q, "k");
  check_on(v, q, "v");
  check_on(bias, q, "bias");
  check_on(mask, q, "mask");
  const at::DeviceGuard guard(q.device());
  TORCH_CHECK(q.dim() == 5 && q.sizes() == k.sizes() && q.sizes() == v.sizes() &&
                  q.size(2) == q.size(3),
              "q, k, v must be [B, H, N, N, D]");
  TORCH_CHECK(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(),
              "q, k, v must have the same dtype");
  const int64_t B = q.size(0), H = q.size(1), N = q.size(2), D = q.size(4);
  TORCH_CHECK(bias.numel() == B * H * N * N, "bias must be [B, H, N, N]");
  TORCH_CHECK(mask.numel() == B * N * N, "mask must be [B, N, N]");
  auto qc = q.contiguous(), kc = k.contiguous(), vc = v.contiguous();
  auto bc = f32c(bias), mc = f32c(mask);
  const int dt = gtk_dtype_of(qc, "q");
  auto out = at::empty({B, N, N, H * D}, qc.options());
  auto ws = workspace(qc, gtk_triangle_attention_workspace_size(B, H, N, D, dt));
  auto fn = starting ? gtk_triangle_attention_starting : gtk_triangle_attention_ending;
  check_rc(fn(qc.data_ptr(), kc.data_ptr(), vc.data_ptr(), bc.data_ptr<float>(),
              mc.data_ptr<float>(), (float)scale, out.data_ptr(), B, H, N, D, dt, ws.data_ptr(),
              ws.numel(), cur_stream(qc)));
  return out;
}

at::Tensor triangle_attention_starting(const at::Tensor& q, const at::Tensor& k,
                                       const at::Tensor& v, const at::Tensor& bias,
                                       const at::Tensor& mask, double scale) {
  return triangle_attention_raw(q, k, v, bias, mask, scale, true);
}
at::Tensor triangle_attention_ending(const at::Tensor& q, const at::Tensor& k,
                                     const at::Tensor& v, const at::Tensor& bias,
                                     const at::Tensor& mask, double scale) {
  return triangle_attention_raw(q, k, v, bias, mask, scale, false);
}

// ---------------------------------------------------------------------------
// Fused module forwards
// ---------------------------------------------------------------------------
int common_param_dtype(std::vector<at::Tensor>& ps) {
  bool all_bf16 = true;
  for (auto& p : ps)
    if (p.defined() && p.scalar_type() != at::kBFloat16) all_bf16 = false;
  for (auto& p : ps)
    if (p.defined()) p = (all_bf16 ? p : p.to(at::kFloat)).contiguous();
  return all_bf16 ? GTK_BF16 : GTK_F32;
}

const void* ptr_or_null(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// Parameter gradients as views of one fp32 buffer, each starting 16-byte
// aligned (one allocation; the caller casts them with one conversion of the
// buffer, which follows the views in out).  Zero for an empty input, on which
// the C functions do nothing.
void flat_grads(std::vector<at::Tensor>& out, const at::Tensor& like,
                const std::vector<std::vector<int64_t>>& shapes, float** const* gs) {
  auto numel = [](const std::vector<int64_t>& s) {
    int64_t n = 1;
    for (auto d : s) n *= d;
    return n;
  };
  int64_t total = 0;
  for (auto& s : shapes) total += (numel(s) + 3) / 4 * 4;
  const auto opts = like.options().dtype(at::kFloat);
  auto flat = like.numel() == 0 ? at::zeros({total}, opts) : at::empty({total}, opts);
  int64_t o = 0;
  for (size_t i = 0; i < shapes.size(); ++i) {
    const int64_t n = numel(shapes[i]);
    auto t = flat.narrow(0, o, n).view(shapes[i]);
    *gs[i] = t.data_ptr<float>();
    out.push_back(t);
    o += (n + 3) / 4 * 4;
  }
  out.push_back(flat);
}

// params: ln_in_w, ln_in_b, a_p_w, a_p_b, a_g_w, a_g_b, b_p_w, b_p_b, b_g_w, b_g_b,
//         g_w, g_b, ln_out_w, ln_out_b, z_w, z_b
at::Tensor tri_mul_pack(std::vector<at::Tensor> ps, int64_t c_z, int64_t c, bool fp32) {
  TORCH_CHECK(ps.size() == 16, "tri_mul_pack expects 16 parameter tensors");
  check_gpu(ps[2], "weights");
  check_all_on(ps, ps[2], "a parameter");
  const at::DeviceGuard guard(ps[2].device());
  gtk_tri_mul_weights w;
  w.dtype = common_param_dtype(ps);
  const void** slots[16] = {&w.ln_in_w, &w.ln_in_b, &w.a_p_w, &w.a_p_b, &w.a_g_w, &w.a_g_b,
                            &w.b_p_w,   &w.b_p_b,   &w.b_g_w, &w.b_g_b, &w.g_w,   &w.g_b,
                            &w.ln_out_w, &w.ln_out_b, &w.z_w, &w.z_b};
  for (int i = 0; i < 16; ++i) *slots[i] = ptr_or_null(ps[i]);
  const int dt = fp32 ? GTK_F32 : GTK_BF16;
  const size_t bytes = gtk_tri_mul_packed_size(c_z, c, dt);
  TORCH_CHECK(bytes > 0, "genie_tk._C: tri_mul shape c_z=", c_z, " c=", c, " unsupported");
  auto packed = workspace(ps[2], bytes);
  check_rc(gtk_tri_mul_pack(&w, c_z, c, dt, packed.data_ptr(), packed.numel(), cur_stream(ps[2])));
  return packed;
}

// Backward of tri_mul_forward (update only): returns [dz, then the gradients of
// the 16 parameters in tri_mul_pack's order (fp32 views of one buffer), then
// that buffer].
std::vector<at::Tensor> tri_mul_backward(const at::Tensor& z, const c10::optional<at::Tensor>& mask,
                                         const at::Tensor& dy, std::vector<at::Tensor> ps,
                                         int64_t c_z, int64_t c, bool outgoing, double eps_in,
                                         double eps_out) {
  TORCH_CHECK(ps.size() == 16, "tri_mul_backward expects 16 parameter tensors");
  check_gpu(z, "z");
  check_on(mask, z, "mask");
  check_on(dy, z, "dy");
  check_all_on(ps, z, "a parameter");
  const at::DeviceGuard guard(z.device());
  TORCH_CHECK(z.dim() == 4 && z.size(1) == z.size(2) && z.size(3) == c_z, "z must be [B, N, N, c_z]");
  TORCH_CHECK(dy.sizes() == z.sizes() && dy.scalar_type() == z.scalar_type(),
              "dy must match z in shape and dtype");
  auto zc = z.contiguous();
  auto dyc = dy.contiguous();
  const int64_t B = zc.size(0), N = zc.size(1);
  at::Tensor mc;
  if (mask.has_value()) {
    TORCH_CHECK(mask->numel() == B * N * N, "mask must be [B, N, N]");
    mc = f32c(*mask);
  }
  gtk_tri_mul_weights w;
  w.dtype = common_param_dtype(ps);
  const void** slots[16] = {&w.ln_in_w, &w.ln_in_b, &w.a_p_w, &w.a_p_b, &w.a_g_w, &w.a_g_b,
                            &w.b_p_w,   &w.b_p_b,   &w.b_g_w, &w.b_g_b, &w.g_w,   &w.g_b,
                            &w.ln_out_w, &w.ln_out_b, &w.z_w, &w.z_b};
  std::vector<at::Tensor> pc(16);
  for (int i = 0; i < 16; ++i) {
    if (ps[i].defined()) pc[i] = ps[i].contiguous();
    *slots[i] = ptr_or_null(pc[i]);
  }
  const int dt = gtk_dtype_of(zc, "z");
  std::vector<at::Tensor> out;
  out.push_back(at::empty_like(zc));
  gtk_tri_mul_grads g;
  float** gs[16] = {&g.ln_in_w, &g.ln_in_b, &g.a_p_w, &g.a_p_b, &g.a_g_w, &g.a_g_b, &g.b_p_w,
                    &g.b_p_b,   &g.b_g_w,   &g.b_g_b, &g.g_w,   &g.g_b,   &g.ln_out_w,
                    &g.ln_out_b, &g.z_w,    &g.z_b};
  flat_grads(out, zc,
             {{c_z}, {c_z}, {c, c_z}, {c}, {c, c_z}, {c}, {c, c_z}, {c}, {c, c_z}, {c}, {c_z, c_z}, {c_z},
              {c}, {c}, {c_z, c}, {c_z}},
             gs);
  const size_t bytes = gtk_tri_mul_backward_workspace_size(B, N, c_z, c, dt);
  TORCH_CHECK(bytes > 0, "genie_tk._C: tri_mul backward shape c_z=", c_z, " c=", c, " unsupported");
  auto ws = workspace(zc, bytes);
  check_rc(gtk_tri_mul_backward(zc.data_ptr(), mask.has_value() ? mc.data_ptr<float>() : nullptr,
                                dyc.data_ptr(), &w, out[0].data_ptr(), &g, B, N, c_z, c,
                                outgoing ? 1 : 0, (float)eps_in, (float)eps_out, dt, ws.data_ptr(),
                                ws.numel(), cur_stream(zc)));
  return out;
}

// Backward of tri_attn_forward (update only): returns [dx, then the gradients of
// the 10 parameters in tri_attn_pack's order (fp32 views of one buffer), then
// that buffer].
// `entry` is the C function: gtk_tri_attn_backward (four heads of 32) or
// gtk_tri_attn_backward_heads (every head shape of the forward kernels), whose
// workspace is that of four heads of 32.
std::vector<at::Tensor> tri_attn_backward_with(decltype(&gtk_tri_attn_backward) entry, const at::Tensor& x,
                                               const c10::optional<at::Tensor>& mask, const at::Tensor& dy,
                                               std::vector<at::Tensor> ps, int64_t c_in, int64_t c_h, int64_t H,
                                               bool starting, double eps) {
  TORCH_CHECK(ps.size() == 10, "tri_attn_backward expects 10 parameter tensors");
  check_gpu(x, "x");
  check_on(mask, x, "mask");
  check_on(dy, x, "dy");
  check_all_on(ps, x, "a parameter");
  const at::DeviceGuard guard(x.device());
  TORCH_CHECK(x.dim() == 4 && x.size(1) == x.size(2) && x.size(3) == c_in, "x must be [B, N, N, c_in]");
  TORCH_CHECK(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type(),
              "dy must match x in shape and dtype");
  auto xc = x.contiguous();
  auto dyc = dy.contiguous();
  const int64_t B = xc.size(0), N = xc.size(1);
  at::Tensor mc;
  if (mask.has_value()) {
    TORCH_CHECK(mask->numel() == B * N * N, "mask must be [B, N, N]");
    mc = f32c(*mask);
  }
  gtk_tri_attn_weights w;
  w.dtype = common_param_dtype(ps);
  const void** slots[10] = {&w.ln_w, &w.ln_b, &w.tri_w, &w.q_w, &w.k_w,
                            &w.v_w,  &w.g_w,  &w.g_b,   &w.o_w, &w.o_b};
  for (int i = 0; i < 10; ++i) *slots[i] = ptr_or_null(ps[i]);
  const int dt = gtk_dtype_of(xc, "x");
  std::vector<at::Tensor> out;
  out.push_back(at::empty_like(xc));
  gtk_tri_attn_grads g;
  float** gs[10] = {&g.ln_w, &g.ln_b, &g.tri_w, &g.q_w, &g.k_w, &g.v_w, &g.g_w, &g.g_b, &g.o_w, &g.o_b};
  flat_grads(out, xc,
             {{c_in}, {c_in}, {H, c_in}, {c_h, c_in}, {c_h, c_in}, {c_h, c_in}, {c_h, c_in}, {c_h},
              {c_in, c_h}, {c_in}},
             gs);
  const bool heads = entry == &gtk_tri_attn_backward_heads;
  const size_t bytes = gtk_tri_attn_backward_workspace_size(B, N, c_in, heads ? 128 : c_h, heads ? 4 : H, dt);
  TORCH_CHECK(bytes > 0, "genie_tk._C: tri_attn backward shape c_in=", c_in, " c_h=", c_h, " H=", H,
              " unsupported");
  auto ws = workspace(xc, bytes);
  check_rc(entry(xc.data_ptr(), mask.has_value() ? mc.data_ptr<float>() : nullptr, dyc.data_ptr(), &w,
                 out[0].data_ptr(), &g, B, N, c_in, c_h, H, starting ? 1 : 0, (float)eps, dt, ws.data_ptr(),
                 ws.numel(), cur_stream(xc)));
  return out;
}

std::vector<at::Tensor> tri_attn_backward(const at::Tensor& x, const c10::optional<at::Tensor>& mask,
                                          const at::Tensor& dy, std::vector<at::Tensor> ps,
                                          int64_t c_in, int64_t c_h, int64_t H, bool starting,
                                          double eps) {
  return tri_attn_backward_with(&gtk_tri_attn_backward, x, mask, dy, std::move(ps), c_in, c_h, H, starting, eps);
}

std::vector<at::Tensor> tri_attn_backward_heads(const at::Tensor& x, const c10::optional<at::Tensor>& mask,
                                                const at::Tensor& dy, std::vector<at::Tensor> ps,
                                                int64_t c_in, int64_t c_h, int64_t H, bool starting,
                                                double eps) {
  return tri_attn_backward_with(&gtk_tri_attn_backward_heads, x, mask, dy, std::move(ps), c_in, c_h, H, starting,
                                eps);
}

// chunk_rows > 0: the memory-bounded mode (output rows that many at a time)
at::Tensor tri_mul_forward(const at::Tensor& z, const c10::optional<at::Tensor>& mask,
                           const at::Tensor& packed, int64_t c_z, int64_t c, bool outgoing,
                           bool residual, double eps_in, double eps_out, int64_t chunk_rows) {
  check_gpu(z, "z");
  check_on(mask, z, "mask");
  check_on(packed, z, "packed");
  const at::DeviceGuard guard(z.device());
  TORCH_CHECK(z.dim() == 4 && z.size(1) == z.size(2) && z.size(3) == c_z, "z must be [B, N, N, c_z]");
  auto zc = z.contiguous();
  const int64_t B = zc.size(0), N = zc.size(1);
  at::Tensor mc;
  if (mask.has_value()) {
    TORCH_CHECK(mask->numel() == B * N * N, "mask must be [B, N, N]");
    mc = f32c(*mask);
  }
  const int dt = gtk_dtype_of(zc, "z");
  auto out = at::empty_like(zc);
  TORCH_CHECK(chunk_rows >= 0, "tri_mul_forward: chunk_rows must be >= 0");
  auto ws = workspace(zc, gtk_tri_mul_workspace_size_chunked(B, N, c_z, c, dt, chunk_rows));
  check_rc(gtk_tri_mul_forward_chunked(
      zc.data_ptr(), mask.has_value() ? mc.data_ptr<float>() : nullptr, out.data_ptr(),
      packed.data_ptr(), B, N, c_z, c, outgoing ? 1 : 0, residual ? 1 : 0, (float)eps_in,
      (float)eps_out, dt, chunk_rows, ws.data_ptr(), ws.numel(), cur_stream(zc)));
  return out;
}

// The fp8 a/b storage experiment (bf16 z; packed from tri_mul_pack(fp32=False)).
at::Tensor tri_mul_forward_fp8ab(const at::Tensor& z, const c10::optional<at::Tensor>& mask,
                                 const at::Tensor& packed, int64_t c_z, int64_t c, bool outgoing,
                                 bool residual, double eps_in, double eps_out) {
  check_gpu(z, "z");
  check_on(mask, z, "mask");
  check_on(packed, z, "packed");
  const at::DeviceGuard guard(z.device());
  TORCH_CHECK(z.dim() == 4 && z.size(1) == z.size(2) && z.size(3) == c_z, "z must be [B, N, N, c_z]");
  TORCH_CHECK(z.scalar_type() == at::kBFloat16, "tri_mul_forward_fp8ab: bf16 only");
  auto zc = z.contiguous();
  const int64_t B = zc.size(0), N = zc.size(1);
  at::Tensor mc;
  if (mask.has_value()) {
    TORCH_CHECK(mask->numel() == B * N * N, "mask must be [B, N, N]");
    mc = f32c(*mask);
  }
  auto out = at::empty_like(zc);
  const size_t bytes = gtk_tri_mul_fp8ab_workspace_size(B, N, c_z, c);
  TORCH_CHECK(bytes > 0, "tri_mul_forward_fp8ab: shape unsupported");
  auto ws = workspace(zc, bytes);
  check_rc(gtk_tri_mul_forward_fp8ab(zc.data_ptr(), mask.has_value() ? mc.data_ptr<float>() : nullptr,
                                     out.data_ptr(), packed.data_ptr(), B, N, c_z, c, outgoing ? 1 : 0,
                                     residual ? 1 : 0, (float)eps_in, (float)eps_out, ws.data_ptr(),
                                     ws.numel(), cur_stream(zc)));
  return out;
}

// a, b: uint8 [P, Np, Np] (fp8 E4M3 bytes) -> bf16 [P, Np, Np]
at::Tensor tri_mul_contract_fp8(const at::Tensor& a, const at::Tensor& b) {
  check_gpu(a, "a");
  check_on(b, a, "b");
  const at::DeviceGuard guard(a.device());
  TORCH_CHECK(a.scalar_type() == at::kByte && b.scalar_type() == at::kByte, "a, b must be uint8");
  TORCH_CHECK(a.dim() == 3 && a.size(1) == a.size(2) && a.sizes() == b.sizes(), "a, b must be [P, Np, Np]");
  auto ac = a.contiguous(), bc = b.contiguous();
  auto x = at::empty(ac.sizes(), ac.options().dtype(at::kBFloat16));
  check_rc(gtk_tri_mul_contract_fp8(ac.data_ptr(), bc.data_ptr(), x.data_ptr(), ac.size(0), ac.size(1),
                                    cur_stream(ac)));
  return x;
}

// params: ln_w, ln_b, w1, b1, w2, b2 (PairTransition: layer_norm, linear_1, linear_2)
// fp32: pack for the fp32 forward (else bf16)
at::Tensor pair_transition_pack(std::vector<at::Tensor> ps, int64_t c, int64_t n, bool fp32) {
  TORCH_CHECK(ps.size() == 6, "pair_transition_pack expects 6 parameter tensors");
  check_gpu(ps[2], "weights");
  check_all_on(ps, ps[2], "a parameter");
  const at::DeviceGuard guard(ps[2].device());
  gtk_pair_transition_weights w;
  w.dtype = common_param_dtype(ps);
  const void** slots[6] = {&w.ln_w, &w.ln_b, &w.w1, &w.b1, &w.w2, &w.b2};
  for (int i = 0; i < 6; ++i) *slots[i] = ptr_or_null(ps[i]);
  const int dt = fp32 ? GTK_F32 : GTK_BF16;
  const size_t bytes = gtk_pair_transition_packed_size(c, n, dt);
  TORCH_CHECK(bytes > 0, "genie_tk._C: pair_transition shape c=", c, " n=", n, " unsupported");
  auto packed = workspace(ps[2], bytes);
  check_rc(gtk_pair_transition_pack(&w, c, n, dt, packed.data_ptr(), packed.numel(),
                                    cur_stream(ps[2])));
  return packed;
}

// p: [..., c] bf16; mask: [...] (rows of p) or None
at::Tensor pair_transition_forward(const at::Tensor& p, const c10::optional<at::Tensor>& mask,
                                   const at::Tensor& packed, int64_t c, int64_t n, bool residual,
                                   double eps) {
  check_gpu(p, "p");
  check_on(mask, p, "mask");
  check_on(packed, p, "packed");
  const at::DeviceGuard guard(p.device());
  TORCH_CHECK(p.dim() >= 1 && p.size(-1) == c, "p must be [..., c]");
  auto pc = p.contiguous();
  const int dt = gtk_dtype_of(pc, "p");
  const int64_t rows = pc.numel() / c;
  at::Tensor mc;
  if (mask.has_value()) {
    TORCH_CHECK(mask->numel() == rows, "mask must have one value per row of p");
    mc = f32c(*mask);
  }
  auto out = at::empty_like(pc);
  check_rc(gtk_pair_transition_forward(pc.data_ptr(), mask.has_value() ? mc.data_ptr<float>() : nullptr,
                                       out.data_ptr(), packed.data_ptr(), rows, c, n,
                                       residual ? 1 : 0, (float)eps, dt, cur_stream(pc)));
  return out;
}

// Backward of pair_transition_forward (no residual, no mask): returns [dp,
// then the gradients of ln_w, ln_b, w1, b1, w2, b2 (fp32 views of one
// buffer), then that buffer].
std::vector<at::Tensor> pair_transition_backward(const at::Tensor& p, const at::Tensor& dy,
                                                 std::vector<at::Tensor> ps, int64_t c, int64_t n,
                                                 double eps) {
  TORCH_CHECK(ps.size() == 6, "pair_transition_backward expects 6 parameter tensors");
  check_gpu(p, "p");
  check_on(dy, p, "dy");
  check_all_on(ps, p, "a parameter");
  const at::DeviceGuard guard(p.device());
  TORCH_CHECK(p.dim() >= 1 && p.size(-1) == c, "p must be [..., c]");
  TORCH_CHECK(dy.sizes() == p.sizes() && dy.scalar_type() == p.scalar_type(),
              "dy must match p in shape and dtype");
  auto pc = p.contiguous();
  auto dyc = dy.contiguous();
  const int64_t rows = pc.numel() / c;
  gtk_pair_transition_weights w;
  w.dtype = common_param_dtype(ps);
  const void** slots[6] = {&w.ln_w, &w.ln_b, &w.w1, &w.b1, &w.w2, &w.b2};
  std::vector<at::Tensor> prm(6);
  for (int i = 0; i < 6; ++i) {
    if (ps[i].defined()) prm[i] = ps[i].contiguous();
    *slots[i] = ptr_or_null(prm[i]);
  }
  const int dt = gtk_dtype_of(pc, "p");
  std::vector<at::Tensor> out;
  out.push_back(at::empty_like(pc));
  gtk_pair_transition_grads g;
  float** gs[6] = {&g.ln_w, &g.ln_b, &g.w1, &g.b1, &g.w2, &g.b2};
  const int64_t hid = c * n;
  flat_grads(out, pc, {{c}, {c}, {hid, c}, {hid}, {c, hid}, {c}}, gs);
  const size_t bytes = gtk_pair_transition_backward_workspace_size(rows, c, n, dt);
  TORCH_CHECK(bytes > 0, "genie_tk._C: pair_transition backward shape c=", c, " n=", n, " unsupported");
  auto ws = workspace(pc, bytes);
  check_rc(gtk_pair_transition_backward(pc.data_ptr(), dyc.data_ptr(), &w, out[0].data_ptr(), &g,
                                        rows, c, n, (float)eps, dt, ws.data_ptr(), ws.numel(),
                                        cur_stream(pc)));
  return out;
}

// params: ln_w, ln_b, tri_w, q_w, k_w, v_w, g_w, g_b, o_w, o_b
at::Tensor tri_attn_pack(std::vector<at::Tensor> ps, int64_t c_in, int64_t c_h, int64_t H,
                         bool fp32) {
  TORCH_CHECK(ps.size() == 10, "tri_attn_pack expects 10 parameter tensors");
  check_gpu(ps[3], "weights");
  check_all_on(ps, ps[3], "a parameter");
  const at::DeviceGuard guard(ps[3].device());
  gtk_tri_attn_weights w;
  w.dtype = common_param_dtype(ps);
  const void** slots[10] = {&w.ln_w, &w.ln_b, &w.tri_w, &w.q_w, &w.k_w,
                            &w.v_w,  &w.g_w,  &w.g_b,   &w.o_w, &w.o_b};
  for (int i = 0; i < 10; ++i) *slots[i] = ptr_or_null(ps[i]);
  const int dt = fp32 ? GTK_F32 : GTK_BF16;
  const size_t bytes = gtk_tri_attn_packed_size(c_in, c_h, H, dt);
  TORCH_CHECK(bytes > 0, "genie_tk._C: tri_attn shape c_in=", c_in, " c_h=", c_h, " H=", H,
              " unsupported");
  auto packed = workspace(ps[3], bytes);
  check_rc(gtk_tri_attn_pack(&w, c_in, c_h, H, dt, packed.data_ptr(), packed.numel(),
                             cur_stream(ps[3])));
  return packed;
}

at::Tensor tri_attn_forward(const at::Tensor& x, const c10::optional<at::Tensor>& mask,
                            const at::Tensor& packed, int64_t c_in, int64_t c_h, int64_t H,
                            bool starting, bool residual, double eps, int64_t chunk_rows,
                            double inf) {
  check_gpu(x, "x");
  check_on(mask, x, "mask");
  check_on(packed, x, "packed");
  const at::DeviceGuard guard(x.device());
  TORCH_CHECK(x.dim() == 4 && x.size(1) == x.size(2) && x.size(3) == c_in, "x must be [B, N, N, c_in]");
  auto xc = x.contiguous();
  const int64_t B = xc.size(0), N = xc.size(1);
  at::Tensor mc;
  if (mask.has_value()) {
    TORCH_CHECK(mask->numel() == B * N * N, "mask must be [B, N, N]");
    mc = f32c(*mask);
  }
  const int dt = gtk_dtype_of(xc, "x");
  auto out = at::empty_like(xc);
  auto ws = workspace(xc, gtk_tri_attn_workspace_size_chunked(B, N, c_in, c_h, H, chunk_rows, dt));
  check_rc(gtk_tri_attn_forward_chunked(
      xc.data_ptr(), mask.has_value() ? mc.data_ptr<float>() : nullptr, out.data_ptr(),
      packed.data_ptr(), B, N, c_in, c_h, H, starting ? 1 : 0, residual ? 1 : 0, (float)eps,
      (float)inf, chunk_rows, dt, ws.data_ptr(), ws.numel(), cur_stream(xc)));
  return out;
}

// ---------------------------------------------------------------------------
// LayerNorm as training uses it
// ---------------------------------------------------------------------------
// x as rows of its last dimension, one stride apart and contiguous inside: x
// itself where its strides allow it, else a contiguous copy.
at::Tensor as_rows(const at::Tensor& x, int64_t* stride) {
  const int64_t d = x.size(-1);
  *stride = d;
  if (x.is_contiguous()) return x;
  bool ok = d == 1 || x.stride(-1) == 1;
  int64_t step = -1, expect = -1;  // of the row index, from the innermost leading dimension outwards
  for (int64_t k = x.dim() - 2; ok && k >= 0; --k) {
    if (x.size(k) == 1) continue;
    if (step < 0)
      step = x.stride(k);
    else
      ok = x.stride(k) == expect;
    expect = x.stride(k) * x.size(k);
  }
  if (!ok || x.numel() == 0) return x.contiguous();
  if (step >= 0) *stride = step;
  return x;
}

void check_ln(const at::Tensor& x, const c10::optional<at::Tensor>& p, const char* what) {
  if (!p.has_value()) return;
  check_on(*p, x, what);
  TORCH_CHECK(p->dim() == 1 && p->size(0) == x.size(-1), what, " must be [", x.size(-1), "]");
  gtk_dtype_of(*p, what);
}

at::Tensor layer_norm_forward(const at::Tensor& x, const c10::optional<at::Tensor>& weight,
                              const c10::optional<at::Tensor>& bias, double eps) {
  check_gpu(x, "x");
  TORCH_CHECK(x.dim() >= 1, "x must have at least one dimension");
  check_ln(x, weight, "weight");
  check_ln(x, bias, "bias");
  const at::DeviceGuard guard(x.device());
  const int dt = gtk_dtype_of(x, "x");
  const int64_t d = x.size(-1);
  int64_t stride;
  auto xc = as_rows(x, &stride);
  // one type for both parameters
  const bool mixed = weight.has_value() && bias.has_value() && weight->scalar_type() != bias->scalar_type();
  at::Tensor w, b;
  if (weight.has_value()) w = mixed ? f32c(*weight) : weight->contiguous();
  if (bias.has_value()) b = mixed ? f32c(*bias) : bias->contiguous();
  const int pdt = w.defined() ? gtk_dtype_of(w, "weight") : b.defined() ? gtk_dtype_of(b, "bias") : GTK_F32;
  auto y = at::empty(x.sizes(), x.options());
  check_rc(gtk_layer_norm_forward(xc.data_ptr(), stride, y.data_ptr(), ptr_or_null(w), ptr_or_null(b), pdt,
                                  d ? x.numel() / d : 0, d, (float)eps, dt, cur_stream(x)));
  return y;
}

// {dx, dweight, dbias}, the ones not asked for undefined; dweight and dbias in
// the weight's type (fp32 without a weight).
std::array<at::Tensor, 3> ln_backward(const at::Tensor& x, const at::Tensor& dy,
                                      const c10::optional<at::Tensor>& weight, double eps, bool need_x,
                                      bool need_weight, bool need_bias) {
  check_gpu(x, "x");
  TORCH_CHECK(x.dim() >= 1, "x must have at least one dimension");
  check_on(dy, x, "dy");
  check_ln(x, weight, "weight");
  TORCH_CHECK(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type(),
              "dy must match x in shape and dtype");
  const at::DeviceGuard guard(x.device());
  const int dt = gtk_dtype_of(x, "x");
  const int64_t d = x.size(-1), rows = d ? x.numel() / d : 0;
  int64_t xs, ds;
  auto xc = as_rows(x, &xs), dyc = as_rows(dy, &ds);
  at::Tensor w;
  if (weight.has_value()) w = weight->contiguous();
  const auto popts = w.defined() ? w.options() : x.options().dtype(at::kFloat);
  std::array<at::Tensor, 3> out;
  if (need_x) out[0] = at::empty(x.sizes(), x.options());
  if (need_weight) out[1] = at::empty({d}, popts);
  if (need_bias) out[2] = at::empty({d}, popts);
  auto ptr = [&](int k) { return out[k].defined() ? out[k].data_ptr() : nullptr; };
  auto ws = workspace(x, gtk_layer_norm_backward_workspace_size(rows, d, dt));
  check_rc(gtk_layer_norm_backward(xc.data_ptr(), xs, dyc.data_ptr(), ds, ptr_or_null(w),
                                   w.defined() ? gtk_dtype_of(w, "weight") : GTK_F32, ptr(0), ptr(1), ptr(2), rows, d,
                                   (float)eps, dt, ws.data_ptr(), ws.numel(), cur_stream(x)));
  return out;
}

std::vector<c10::optional<at::Tensor>> layer_norm_backward(const at::Tensor& x, const at::Tensor& dy,
                                                           const c10::optional<at::Tensor>& weight, double eps,
                                                           bool need_x, bool need_weight, bool need_bias) {
  std::vector<c10::optional<at::Tensor>> out(3);
  auto g = ln_backward(x, dy, weight, eps, need_x, need_weight, need_bias);
  for (int k = 0; k < 3; ++k)
    if (g[k].defined()) out[k] = g[k];
  return out;
}

// What a backward pass returns under create_graph: differentiating it again is an
// error that names the operator.
void once_differentiable(torch::autograd::variable_list& out, const char* what) {
  if (!at::GradMode::is_enabled()) return;
  torch::autograd::variable_list some;
  for (const auto& t : out)
    if (t.defined()) some.push_back(t.detach().requires_grad_(true));
  if (some.empty()) return;
  torch::autograd::DelayedError error(
      std::string(what) + "'s backward is once_differentiable: a second derivative is not implemented",
      (int)some.size());
  const auto guarded = error.apply(std::move(some));
  size_t k = 0;
  for (auto& t : out)
    if (t.defined()) t = guarded[k++];
}

// layer_norm_forward under autograd.  A node of C++: a training pass over 4096
// rows of 128 takes 71 us of host time with it, 87 with a Python one.  Only x and
// the weight are saved: the backward computes the rows' statistics again.
struct LayerNormFn : public torch::autograd::Function<LayerNormFn> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x,
                            const c10::optional<at::Tensor>& weight, const c10::optional<at::Tensor>& bias,
                            double eps) {
    ctx->save_for_backward({x, weight.has_value() ? *weight : at::Tensor()});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["bias_dtype"] = (int64_t)(bias.has_value() ? bias->scalar_type() : at::kFloat);
    return layer_norm_forward(x, weight, bias, eps);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor& x = saved[0];
    c10::optional<at::Tensor> weight;
    if (saved[1].defined()) weight = saved[1];
    const auto bias_dtype = (at::ScalarType)ctx->saved_data["bias_dtype"].toInt();
    const bool need_x = ctx->needs_input_grad(0), need_w = weight.has_value() && ctx->needs_input_grad(1);
    // the edges of absent parameters are not counted
    const bool need_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(weight.has_value() ? 2 : 1);
    std::array<at::Tensor, 3> g;
    {
      at::NoGradGuard no_grad;
      const auto weight_dtype = weight.has_value() ? weight->scalar_type() : at::kFloat;
      // parameters of two types: both in fp32, each rounded once to its own
      if (need_b && weight.has_value() && weight_dtype != bias_dtype) weight = weight->to(at::kFloat);
      g = ln_backward(x, grads[0], weight, ctx->saved_data["eps"].toDouble(), need_x, need_w, need_b);
      if (need_w) g[1] = g[1].to(weight_dtype);
      if (need_b) g[2] = g[2].to(bias_dtype);
    }
    torch::autograd::variable_list out{g[0], g[1], g[2], at::Tensor()};
    once_differentiable(out, "layer_norm");
    return out;
  }
};

// Without `strict`, None where an input carries a forward-mode tangent, which
// the kernels do not propagate (a dual tensor need not require a gradient).
c10::optional<at::Tensor> layer_norm(const at::Tensor& x, const c10::optional<at::Tensor>& weight,
                                     const c10::optional<at::Tensor>& bias, double eps, bool strict) {
  auto dual = [](const at::Tensor& t) { return t._fw_grad(/*level=*/0).defined(); };
  if (dual(x) || (weight.has_value() && dual(*weight)) || (bias.has_value() && dual(*bias))) {
    TORCH_CHECK_NOT_IMPLEMENTED(!strict, "genie_tk._C: layer_norm has no forward-mode derivative");
    return c10::nullopt;
  }
  const bool grad = at::GradMode::is_enabled() &&
                    (x.requires_grad() || (weight.has_value() && weight->requires_grad()) ||
                     (bias.has_value() && bias->requires_grad()));
  return grad ? LayerNormFn::apply(x, weight, bias, eps) : layer_norm_forward(x, weight, bias, eps);
}

// ---------------------------------------------------------------------------
// Dropout with a counter-based generator
// ---------------------------------------------------------------------------
// What fixes a mask: the view of x, the share that is dropped and the key.
struct DropoutMask {
  int64_t outer, shared, inner;
  double p;
  uint64_t seed, offset;
};

at::Tensor dropout_forward(const at::Tensor& x, const at::Tensor& residual, at::ScalarType out_type,
                           const at::Tensor& seed_device, const DropoutMask& k) {
  const at::DeviceGuard guard(x.device());
  const auto xc = x.contiguous(), rc = residual.defined() ? residual.contiguous() : residual;
  auto out = at::empty(x.sizes(), x.options().dtype(out_type));
  check_rc(gtk_dropout(xc.data_ptr(), gtk_dtype_of(xc, "x"), ptr_or_null(rc),
                       rc.defined() ? gtk_dtype_of(rc, "residual") : GTK_F32, out.data_ptr(),
                       gtk_dtype_of(out, "the output"), k.outer, k.shared, k.inner, k.p, k.seed,
                       (const uint64_t*)ptr_or_null(seed_device), k.offset, cur_stream(x)));
  return out;
}

using MaybeTensor = c10::optional<at::Tensor>;
at::Tensor or_undefined(const MaybeTensor& t) { return t.value_or(at::Tensor()); }

at::Tensor dropout_or_grad(const at::Tensor& x, const MaybeTensor& residual, at::ScalarType out_type,
                           const MaybeTensor& seed_device, const DropoutMask& k);

// Linear in x and in the residual: dL/dx is the same call on dL/dout, of which
// any number of derivatives may be taken.  Nothing is saved but the key.
struct DropoutFn : public torch::autograd::Function<DropoutFn> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const MaybeTensor& residual,
                            int64_t out_type, const MaybeTensor& seed_device, const DropoutMask& k) {
    ctx->save_for_backward({or_undefined(seed_device)});
    ctx->saved_data["key"] = std::vector<int64_t>{k.outer, k.shared, k.inner, (int64_t)k.seed, (int64_t)k.offset,
                                                  (int64_t)x.scalar_type()};
    ctx->saved_data["p"] = k.p;
    ctx->saved_data["has_residual"] = residual.has_value();
    ctx->saved_data["residual_type"] = (int64_t)(residual.has_value() ? residual->scalar_type() : at::kFloat);
    return dropout_forward(x, or_undefined(residual), (at::ScalarType)out_type, or_undefined(seed_device), k);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const at::Tensor& dy = grads[0];
    const auto v = ctx->saved_data["key"].toIntVector();
    const DropoutMask k{v[0], v[1], v[2], ctx->saved_data["p"].toDouble(), (uint64_t)v[3], (uint64_t)v[4]};
    const auto seed = ctx->get_saved_variables()[0];
    torch::autograd::variable_list out(5);
    if (ctx->needs_input_grad(0))
      out[0] = dropout_or_grad(dy, c10::nullopt, (at::ScalarType)v[5],
                               seed.defined() ? MaybeTensor(seed) : c10::nullopt, k);
    // an absent residual has no edge to ask about
    const bool residual = ctx->saved_data["has_residual"].toBool();
    if (residual && ctx->needs_input_grad(1))
      out[1] = dy.to((at::ScalarType)ctx->saved_data["residual_type"].toInt());
    return out;
  }
};

at::Tensor dropout_or_grad(const at::Tensor& x, const MaybeTensor& residual, at::ScalarType out_type,
                           const MaybeTensor& seed_device, const DropoutMask& k) {
  const bool grad =
      at::GradMode::is_enabled() && (x.requires_grad() || (residual.has_value() && residual->requires_grad()));
  return grad ? DropoutFn::apply(x, residual, (int64_t)out_type, seed_device, k)
              : dropout_forward(x, or_undefined(residual), out_type, or_undefined(seed_device), k);
}

// x seen as [outer, size of shared_dim, inner] (no shared_dim: one decision a
// value).  Without `strict`, None where an input has a forward-mode tangent.
c10::optional<at::Tensor> dropout(const at::Tensor& x, double p, uint64_t seed, uint64_t offset,
                                  c10::optional<int64_t> shared_dim, const c10::optional<at::Tensor>& residual,
                                  const c10::optional<at::Tensor>& seed_device, bool strict) {
  check_gpu(x, "x");
  check_on(residual, x, "residual");
  check_on(seed_device, x, "seed");
  TORCH_CHECK(p >= 0.0 && p <= 1.0, "dropout probability has to be between 0 and 1, but got ", p);
  TORCH_CHECK(!residual.has_value() || residual->sizes() == x.sizes(), "genie_tk._C: residual must have x's shape");
  TORCH_CHECK(!seed_device.has_value() || (seed_device->numel() == 1 && seed_device->scalar_type() == at::kLong),
              "genie_tk._C: a seed tensor is one int64 value");
  if (x._fw_grad(0).defined() || (residual.has_value() && residual->_fw_grad(0).defined())) {
    TORCH_CHECK_NOT_IMPLEMENTED(!strict, "genie_tk._C: dropout has no forward-mode derivative");
    return c10::nullopt;
  }
  DropoutMask k{1, 1, x.numel(), p, seed, offset};
  if (shared_dim.has_value()) {
    const int64_t dim = at::maybe_wrap_dim(*shared_dim, x.dim());
    k.inner = 1;
    for (int64_t i = 0; i < x.dim(); ++i) (i < dim ? k.outer : i == dim ? k.shared : k.inner) *= x.size(i);
  }
  return dropout_or_grad(x, residual, residual.has_value() ? residual->scalar_type() : x.scalar_type(), seed_device, k);
}

// ---------------------------------------------------------------------------
// Group norm with an activation, channels last
// ---------------------------------------------------------------------------
// Checked arguments: x [B, ..., C] as rows, the mask as floats, one type for both
// parameters.
struct GroupNormArgs {
  int64_t B, P, C, groups, stride;
  int dtype, param_dtype;
  at::Tensor x, mask, weight, bias;

  GroupNormArgs(const at::Tensor& in, int64_t groups_, const at::Tensor& w, const at::Tensor& b, const at::Tensor& m)
      : groups(groups_) {
    check_gpu(in, "x");
    TORCH_CHECK(in.dim() >= 2, "x must be [B, ..., C]");
    C = in.size(-1);
    B = in.size(0);
    P = 1;
    for (int64_t k = 1; k < in.dim() - 1; ++k) P *= in.size(k);
    TORCH_CHECK(groups >= 1 && C >= 1 && C % groups == 0, "genie_tk._C: ", C, " channels in ", groups, " groups");
    dtype = gtk_dtype_of(in, "x");
    c10::optional<at::Tensor> ow, ob;
    if (w.defined()) ow = w;
    if (b.defined()) ob = b;
    check_ln(in, ow, "weight");
    check_ln(in, ob, "bias");
    check_on(m, in, "mask");
    const bool mixed = w.defined() && b.defined() && w.scalar_type() != b.scalar_type();
    if (w.defined()) weight = mixed ? f32c(w) : w.contiguous();
    if (b.defined()) bias = mixed ? f32c(b) : b.contiguous();
    param_dtype = weight.defined() ? gtk_dtype_of(weight, "weight")
                  : bias.defined() ? gtk_dtype_of(bias, "bias")
                                   : GTK_F32;
    if (m.defined()) {
      TORCH_CHECK(m.sizes() == in.sizes().slice(0, in.dim() - 1), "mask must be x's shape without its channels");
      // what is not 0 stays so
      mask = f32c(m.scalar_type() == at::kDouble ? m.ne(0) : m);
    }
    x = as_rows(in, &stride);
  }
  const float* mask_ptr() const { return mask.defined() ? mask.data_ptr<float>() : nullptr; }
};

// {y, stats}
std::array<at::Tensor, 2> gn_forward(const at::Tensor& x, int64_t groups, const at::Tensor& weight,
                                     const at::Tensor& bias, double eps, int64_t act, const at::Tensor& mask) {
  const at::DeviceGuard guard(x.device());
  const GroupNormArgs a(x, groups, weight, bias, mask);
  auto y = at::empty(x.sizes(), x.options());
  auto stats = at::empty({a.B, groups, 4}, x.options().dtype(at::kFloat));
  if (a.B && a.P) {
    at::Tensor ws;
    const size_t need = gtk_group_norm_workspace_size(a.B, a.P, a.C, groups, a.dtype);
    if (need) ws = workspace(x, need);
    check_rc(gtk_group_norm_forward(a.x.data_ptr(), a.stride, a.mask_ptr(), y.data_ptr(), stats.data_ptr<float>(),
                                    ptr_or_null(a.weight), ptr_or_null(a.bias), a.param_dtype, a.B, a.P, a.C, groups,
                                    (float)eps, (int)act, a.dtype, need ? ws.data_ptr() : nullptr, need,
                                    cur_stream(x)));
  }
  return {y, stats};
}

// {dx, dweight, dbias}, the ones not asked for undefined; dweight and dbias in
// their parameters' types (fp32 without).
std::array<at::Tensor, 3> gn_backward(const at::Tensor& x, const at::Tensor& dy, const at::Tensor& stats,
                                      int64_t groups, const at::Tensor& weight, const at::Tensor& bias, int64_t act,
                                      const at::Tensor& mask, std::array<bool, 3> need) {
  const at::DeviceGuard guard(x.device());
  const GroupNormArgs a(x, groups, weight, bias, mask);
  check_on(dy, x, "dy");
  check_on(stats, x, "stats");
  TORCH_CHECK(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type(), "dy must match x in shape and dtype");
  TORCH_CHECK(stats.scalar_type() == at::kFloat && stats.is_contiguous() && stats.numel() == a.B * groups * 4,
              "stats are those that the forward pass returned");
  int64_t ds;
  const auto dyc = as_rows(dy, &ds);
  const auto popts = x.options().dtype(a.param_dtype == GTK_F32 ? at::kFloat : at::kBFloat16);
  std::array<at::Tensor, 3> out;
  if (need[0]) out[0] = at::empty(x.sizes(), x.options());
  for (int k = 1; k < 3; ++k)
    if (need[k]) out[k] = at::empty({a.C}, popts);
  if (a.P) {
    at::Tensor ws;
    const size_t bytes = gtk_group_norm_backward_workspace_size(a.B, a.P, a.C, groups, a.dtype);
    if (bytes) ws = workspace(x, bytes);
    auto ptr = [&](int k) { return out[k].defined() ? out[k].data_ptr() : nullptr; };
    check_rc(gtk_group_norm_backward(a.x.data_ptr(), a.stride, a.mask_ptr(), dyc.data_ptr(), ds,
                                     stats.data_ptr<float>(), ptr_or_null(a.weight), ptr_or_null(a.bias),
                                     a.param_dtype, ptr(0), ptr(1), ptr(2), a.B, a.P, a.C, groups, (int)act, a.dtype,
                                     bytes ? ws.data_ptr() : nullptr, bytes, cur_stream(x)));
  } else {
    for (int k = 1; k < 3; ++k)
      if (need[k]) out[k].zero_();
  }
  // parameters of two types were taken in fp32
  if (out[1].defined() && weight.defined()) out[1] = out[1].to(weight.scalar_type());
  if (out[2].defined() && bias.defined()) out[2] = out[2].to(bias.scalar_type());
  return out;
}

std::vector<at::Tensor> group_norm_forward(const at::Tensor& x, int64_t groups, const c10::optional<at::Tensor>& weight,
                                           const c10::optional<at::Tensor>& bias, double eps, int64_t act,
                                           const c10::optional<at::Tensor>& mask) {
  const auto r = gn_forward(x, groups, or_undefined(weight), or_undefined(bias), eps, act, or_undefined(mask));
  return {r[0], r[1]};
}

std::vector<c10::optional<at::Tensor>> group_norm_backward(const at::Tensor& x, const at::Tensor& dy,
                                                           const at::Tensor& stats, int64_t groups,
                                                           const c10::optional<at::Tensor>& weight,
                                                           const c10::optional<at::Tensor>& bias, int64_t act,
                                                           const c10::optional<at::Tensor>& mask, bool need_x,
                                                           bool need_weight, bool need_bias) {
  const auto g = gn_backward(x, dy, stats, groups, or_undefined(weight), or_undefined(bias), act, or_undefined(mask),
                             {need_x, need_weight, need_bias});
  std::vector<c10::optional<at::Tensor>> out(3);
  for (int k = 0; k < 3; ++k)
    if (g[k].defined()) out[k] = g[k];
  return out;
}

struct GroupNormFn : public torch::autograd::Function<GroupNormFn> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const MaybeTensor& weight,
                            const MaybeTensor& bias, int64_t groups, double eps, int64_t act,
                            const MaybeTensor& mask) {
    const auto w = or_undefined(weight), b = or_undefined(bias), m = or_undefined(mask);
    const auto r = gn_forward(x, groups, w, b, eps, act, m);
    ctx->save_for_backward({x, w, b, m, r[1]});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["act"] = act;
    return r[0];
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    torch::autograd::variable_list out(7);
    {
      at::NoGradGuard no_grad;
      // the edges of absent parameters are not counted
      const bool has_w = saved[1].defined(), has_b = saved[2].defined();
      const auto g = gn_backward(saved[0], grads[0], saved[4], ctx->saved_data["groups"].toInt(), saved[1], saved[2],
                                 ctx->saved_data["act"].toInt(), saved[3],
                                 {ctx->needs_input_grad(0), has_w && ctx->needs_input_grad(1),
                                  has_b && ctx->needs_input_grad(has_w ? 2 : 1)});
      for (int k = 0; k < 3; ++k) out[k] = g[k];
    }
    once_differentiable(out, "group_norm");
    return out;
  }
};

// Without `strict`, None where an input has a forward-mode tangent.
c10::optional<at::Tensor> group_norm(const at::Tensor& x, int64_t groups, const c10::optional<at::Tensor>& weight,
                                     const c10::optional<at::Tensor>& bias, double eps, int64_t act,
                                     const c10::optional<at::Tensor>& mask, bool strict) {
  bool grad = false;
  auto dual = [&](const at::Tensor& t) {
    grad = grad || t.requires_grad();
    return t._fw_grad(/*level=*/0).defined();
  };
  bool any = dual(x);
  if (weight.has_value()) any = dual(*weight) || any;
  if (bias.has_value()) any = dual(*bias) || any;
  if (any) {
    TORCH_CHECK_NOT_IMPLEMENTED(!strict, "genie_tk._C: group_norm has no forward-mode derivative");
    return c10::nullopt;
  }
  if (grad && at::GradMode::is_enabled()) return GroupNormFn::apply(x, weight, bias, groups, eps, act, mask);
  return gn_forward(x, groups, or_undefined(weight), or_undefined(bias), eps, act, or_undefined(mask))[0];
}

// ---------------------------------------------------------------------------
// Global gradient norm and clipping
// ---------------------------------------------------------------------------
// Gradients as the C functions take them.  The tensors are those of a Python
// sequence, or with `grads_of` their .grad (ones without are passed over), and
// are not copied: a net has hundreds of small ones, and the host time of a call
// is theirs.
struct GradList {
  std::vector<const at::Tensor*> t;
  std::vector<void*> data;
  std::vector<int64_t> numel;
  std::vector<int> dtype;
  py::object items;  // holds the tensors

  // What the kernels take: bf16 or fp32, strided, on one GPU.  Otherwise false
  // without `strict`, and an error with it.
  bool collect(const py::handle& seq, bool grads_of, bool strict) {
    items = py::reinterpret_steal<py::object>(PySequence_Fast(seq.ptr(), "expected a sequence of tensors"));
    if (!items) throw py::error_already_set();
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(items.ptr());
    PyObject** it = PySequence_Fast_ITEMS(items.ptr());
    t.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
      TORCH_CHECK_TYPE(THPVariable_Check(it[i]), "genie_tk._C: item ", i, " is not a tensor");
      const at::Tensor* v = &THPVariable_Unpack(it[i]);
      if (grads_of) v = &v->grad();
      if (v->defined()) t.push_back(v);
    }
    for (const auto* v : t) {
      const bool ok = v->is_cuda() && v->layout() == at::kStrided && v->device() == t[0]->device() &&
                      (v->scalar_type() == at::kFloat || v->scalar_type() == at::kBFloat16);
      if (ok) continue;
      if (!strict) return false;
      check_gpu(*v, "gradients");
      TORCH_CHECK(v->layout() == at::kStrided, "genie_tk._C: a gradient is not a dense tensor");
      check_on(*v, *t[0], "a gradient");
      gtk_dtype_of(*v, "a gradient");
    }
    data.reserve(t.size());
    numel.reserve(t.size());
    dtype.reserve(t.size());
    return true;
  }
  void add(const at::Tensor& v) {
    data.push_back(v.data_ptr());
    numel.push_back(v.numel());
    dtype.push_back(v.scalar_type() == at::kFloat ? GTK_F32 : GTK_BF16);
  }
  gtk_tensor_list list() const { return {(int64_t)data.size(), data.data(), numel.data(), dtype.data()}; }
};

int norm_kind(double p) {
  if (p == 2.0) return GTK_NORM_2;
  if (p == 1.0) return GTK_NORM_1;
  TORCH_CHECK(p == std::numeric_limits<double>::infinity(), "genie_tk._C: norm_type must be 1, 2 or inf, got ", p);
  return GTK_NORM_INF;
}

// The norm of the tensors; without `strict`, None where a tensor is not one for
// the kernels.
c10::optional<at::Tensor> grad_norm(const py::handle& tensors, double p, bool strict) {
  const at::NoGradGuard no_grad;
  GradList l;
  const int kind = norm_kind(p);
  if (!l.collect(tensors, false, strict)) return c10::nullopt;
  TORCH_CHECK(!l.t.empty(), "grad_norm expects at least one tensor");
  const at::Tensor& like = *l.t[0];
  const at::DeviceGuard guard(like.device());
  std::vector<at::Tensor> copies;  // alive until the launch is enqueued
  for (const auto* t : l.t) {
    // the order of the values does not matter: a tensor that fills its memory
    // is taken as it lies, any other is copied
    if (t->is_contiguous() || t->is_non_overlapping_and_dense()) {
      l.add(*t);
    } else {
      copies.push_back(t->contiguous());
      l.add(copies.back());
    }
  }
  const auto g = l.list();
  auto norm = at::empty({}, like.options().dtype(at::kFloat));
  auto ws = workspace(like, gtk_grad_norm_workspace_size(&g));
  check_rc(gtk_grad_norm(&g, kind, norm.data_ptr<float>(), ws.data_ptr(), ws.numel(), cur_stream(like)));
  return norm;
}

// Whether two strided tensors share a byte.  A value of a tensor lies at its
// address + the sum of i_k stride_k, so they do if the distance of their addresses
// is a sum of c_s s over the distinct strides s (1 for the bytes of a value), each
// c_s in a range that the sizes give.  Searched from the largest stride down: what
// the smaller ones can still reach leaves few c_s to try where strides nest, as
// slices' do.  Past 2^16 tries the answer is yes.
bool share_memory(const at::Tensor& a, const at::Tensor& b) {
  struct Axis {
    int64_t stride, lo, hi;
  };
  std::vector<Axis> axes;
  auto add = [&](int64_t stride, int64_t lo, int64_t hi) {
    for (auto& x : axes)
      if (x.stride == stride) {
        x.lo += lo;
        x.hi += hi;
        return;
      }
    if (stride) axes.push_back({stride, lo, hi});
  };
  const int64_t ea = a.element_size(), eb = b.element_size();
  for (int64_t k = 0; k < a.dim(); ++k) add(a.stride(k) * ea, 0, a.size(k) - 1);
  for (int64_t k = 0; k < b.dim(); ++k) add(b.stride(k) * eb, 1 - b.size(k), 0);
  add(1, 0, ea - 1);
  add(1, 1 - eb, 0);
  std::sort(axes.begin(), axes.end(), [](const Axis& x, const Axis& y) { return x.stride > y.stride; });
  std::vector<int64_t> low(axes.size() + 1, 0), high(axes.size() + 1, 0);  // of the sum from axis k on
  for (size_t k = axes.size(); k-- > 0;) {
    low[k] = low[k + 1] + axes[k].lo * axes[k].stride;
    high[k] = high[k + 1] + axes[k].hi * axes[k].stride;
  }
  int tries = 1 << 16;
  std::function<bool(size_t, int64_t)> reach = [&](size_t k, int64_t to) {
    if (to < low[k] || to > high[k]) return false;
    if (k == axes.size()) return true;
    const Axis& x = axes[k];
    // the first c that the rest can complete
    const int64_t need = to - high[k + 1];
    int64_t c = std::max(x.lo, need >= 0 ? (need + x.stride - 1) / x.stride : -(-need / x.stride));
    for (; c <= x.hi && c * x.stride <= to - low[k + 1]; ++c)
      if (--tries < 0 || reach(k + 1, to - c * x.stride)) return true;
    return false;
  };
  return reach(0, (const char*)b.data_ptr() - (const char*)a.data_ptr());
}

// No written tensor may overlap another tensor of the call.  The C functions see
// to that for those that they are given; here, for those that are clipped on
// copies (`copied`).
void check_apart(const GradList& l, const GradList* lo, const std::vector<bool>& copied) {
  struct Piece {
    const char *begin, *end;
    const at::Tensor* t;
    size_t index;
    bool written;
  };
  std::vector<Piece> pieces;
  auto add = [&](const at::Tensor& t, size_t i, bool written) {
    if (t.numel() == 0) return;
    int64_t last = 0;
    for (int64_t k = 0; k < t.dim(); ++k) last += (t.size(k) - 1) * t.stride(k);
    const char* p = (const char*)t.data_ptr();
    pieces.push_back({p, p + (last + 1) * t.element_size(), &t, i, written});
  };
  for (size_t i = 0; i < l.t.size(); ++i) {
    add(*l.t[i], i, !lo);
    if (lo) add(*lo->t[i], i, true);
  }
  std::sort(pieces.begin(), pieces.end(), [](const Piece& a, const Piece& b) { return a.begin < b.begin; });
  std::vector<const Piece*> open;  // those that reach past the current one's begin
  for (const auto& p : pieces) {
    size_t kept = 0;
    for (const Piece* q : open)
      if (q->end > p.begin) open[kept++] = q;
    open.resize(kept);
    for (const Piece* q : open) {
      // a tensor and its own output: the copy is whole before anything is written
      if (q->index == p.index || !(p.written || q->written) || !(copied[p.index] || copied[q->index])) continue;
      TORCH_CHECK(!share_memory(*p.t, *q->t),
                  "genie_tk._C: a tensor that is written overlaps another (or is given twice)");
    }
    open.push_back(&p);
  }
}

// Clips l into lo (in place without it).  norm: given, or undefined: computed,
// and returned.
at::Tensor clip_list(GradList& l, GradList* lo, double max_norm, double p, at::Tensor norm) {
  const at::NoGradGuard no_grad;  // of the copies: a gradient may require one itself
  const at::Tensor& like = *l.t[0];
  const bool given = norm.defined();
  const int kind = given ? GTK_NORM_2 : norm_kind(p);
  const at::DeviceGuard guard(like.device());
  // Tensors that are no run of memory in the other's order are clipped on
  // copies, which are copied back at the end.
  std::vector<std::pair<at::Tensor, at::Tensor>> back;
  std::vector<at::Tensor> copies;
  std::vector<bool> copied(l.t.size(), false);
  for (size_t i = 0; i < l.t.size(); ++i) {
    const at::Tensor &t = *l.t[i], &o = lo ? *lo->t[i] : t;
    TORCH_CHECK(!lo || o.sizes() == t.sizes(), "genie_tk._C: output ", i, " has another shape");
    if ((t.is_contiguous() && o.is_contiguous()) ||
        (t.strides() == o.strides() && t.is_non_overlapping_and_dense())) {
      l.add(t);
      if (lo) lo->add(o);
      continue;
    }
    at::assert_no_internal_overlap(o);
    copied[i] = true;
    copies.push_back(t.contiguous());
    l.add(copies.back());
    if (lo) {
      back.emplace_back(o, at::empty(o.sizes(), o.options().memory_format(at::MemoryFormat::Contiguous)));
      lo->add(back.back().second);
    } else {
      back.emplace_back(o, copies.back());
    }
  }
  if (!copies.empty()) check_apart(l, lo, copied);
  const auto g = l.list(), go = lo ? lo->list() : gtk_tensor_list{};
  const gtk_tensor_list* out = lo ? &go : nullptr;
  void* st = cur_stream(like);
  if (given) {
    check_rc(gtk_grad_clip_with_norm(&g, out, max_norm, norm.data_ptr<float>(), st));
  } else {
    norm = at::empty({}, like.options().dtype(at::kFloat));
    auto ws = workspace(like, gtk_grad_norm_workspace_size(&g));
    check_rc(gtk_grad_clip(&g, out, kind, max_norm, norm.data_ptr<float>(), ws.data_ptr(), ws.numel(), st));
  }
  for (auto& b : back) b.first.copy_(b.second);
  // written behind autograd's back
  for (const auto* t : lo ? lo->t : l.t)
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  return norm;
}

c10::optional<at::Tensor> grad_clip(const py::handle& tensors, const py::handle& outs, double max_norm, double p,
                                    bool strict) {
  GradList l, lo;
  norm_kind(p);
  if (!l.collect(tensors, false, strict)) return c10::nullopt;
  TORCH_CHECK(!l.t.empty(), "grad_clip expects at least one tensor");
  if (outs.is_none()) return clip_list(l, nullptr, max_norm, p, at::Tensor());
  if (!lo.collect(outs, false, strict)) return c10::nullopt;
  TORCH_CHECK(lo.t.size() == l.t.size(), "genie_tk._C: ", lo.t.size(), " outputs for ", l.t.size(), " gradients");
  check_on(*lo.t[0], *l.t[0], "an output");
  return clip_list(l, &lo, max_norm, p, at::Tensor());
}

// grad_clip in place on the gradients of `parameters`: the norm, or None where
// there is no gradient or one that is not for the kernels.
c10::optional<at::Tensor> grad_clip_parameters(const py::handle& parameters, double max_norm, double p) {
  GradList l;
  norm_kind(p);
  if (!l.collect(parameters, true, false) || l.t.empty()) return c10::nullopt;
  return clip_list(l, nullptr, max_norm, p, at::Tensor());
}

void grad_clip_with_norm(const py::handle& tensors, const py::handle& outs, double max_norm, const at::Tensor& norm) {
  GradList l, lo;
  l.collect(tensors, false, true);
  TORCH_CHECK(!l.t.empty(), "grad_clip_with_norm expects at least one tensor");
  check_on(norm, *l.t[0], "norm");
  TORCH_CHECK(norm.numel() == 1 && norm.scalar_type() == at::kFloat, "norm must be one float32 value");
  if (outs.is_none()) {
    clip_list(l, nullptr, max_norm, 2.0, norm);
    return;
  }
  lo.collect(outs, false, true);
  TORCH_CHECK(lo.t.size() == l.t.size(), "genie_tk._C: ", lo.t.size(), " outputs for ", l.t.size(), " gradients");
  check_on(*lo.t[0], *l.t[0], "an output");
  clip_list(l, &lo, max_norm, 2.0, norm);
}

py::dict timing_report() {
  std::vector<char> buf(1 << 16);
  check_rc(gtk_timing_report(buf.data(), buf.size()));
  py::dict out;
  const char* p = buf.data();
  while (*p) {
    char name[128];
    int n = 0, used = 0;
    double total = 0, mn = 0, mx = 0;
    if (sscanf(p, "%127s %d %lf %lf %lf%n", name, &n, &total, &mn, &mx, &used) != 5) break;
    out[py::str(name)] = py::make_tuple(n, total, mn, mx);
    p += used;
    while (*p == '\n') ++p;
  }
  return out;
}

}  // namespace

PYBIND11_MODULE(_C, m) {
  m.doc() = "genie_tk._C: gfx950 HIP kernels for the pair-representation hot path";
  m.def("triangle_mul_outgoing", &triangle_mul_outgoing, "Triangle contraction, outgoing edges",
        py::arg("a"), py::arg("b"), py::arg("mask"));
  m.def("triangle_mul_incoming", &triangle_mul_incoming, "Triangle contraction, incoming edges",
        py::arg("a"), py::arg("b"), py::arg("mask"));
  m.def("triangle_attention_starting", &triangle_attention_starting,
        "Triangle attention core, starting node", py::arg("q"), py::arg("k"), py::arg("v"),
        py::arg("bias"), py::arg("mask"), py::arg("scale"));
  m.def("triangle_attention_ending", &triangle_attention_ending,
        "Triangle attention core, ending node", py::arg("q"), py::arg("k"), py::arg("v"),
        py::arg("bias"), py::arg("mask"), py::arg("scale"));
  m.def("layernorm", &layernorm, "LayerNorm forward", py::arg("x"), py::arg("gamma"),
        py::arg("beta"), py::arg("eps") = 1e-5);
  m.def("fused_layernorm_linear", &fused_layernorm_linear, "LayerNorm + Linear forward",
        py::arg("x"), py::arg("gamma"), py::arg("beta"), py::arg("weight"),
        py::arg("bias") = py::none(), py::arg("eps") = 1e-5);
  m.def("layernorm_linear", &layernorm_linear,
        "LayerNorm + Linear forward with an nn.Linear-layout weight [D_OUT, D_IN]", py::arg("x"),
        py::arg("gamma"), py::arg("beta"), py::arg("weight"), py::arg("bias") = py::none(),
        py::arg("eps") = 1e-5);
  m.def("tri_mul_pack", &tri_mul_pack, "Pack TriangleMultiplicativeUpdate parameters",
        py::arg("params"), py::arg("c_z"), py::arg("c"), py::arg("fp32"));
  m.def("tri_mul_forward", &tri_mul_forward, "Fused TriangleMultiplicativeUpdate forward",
        py::arg("z"), py::arg("mask"), py::arg("packed"), py::arg("c_z"), py::arg("c"),
        py::arg("outgoing"), py::arg("residual") = false, py::arg("eps_in") = 1e-5,
        py::arg("eps_out") = 1e-5, py::arg("chunk_rows") = 0);
  m.def("tri_mul_forward_fp8ab", &tri_mul_forward_fp8ab,
        "TriangleMultiplicativeUpdate forward with a and b stored in fp8 E4M3 (experiment)",
        py::arg("z"), py::arg("mask"), py::arg("packed"), py::arg("c_z"), py::arg("c"),
        py::arg("outgoing"), py::arg("residual") = false, py::arg("eps_in") = 1e-5,
        py::arg("eps_out") = 1e-5);
  m.def("tri_mul_contract_fp8", &tri_mul_contract_fp8,
        "x[p] = a[p] . b[p]^T over fp8 E4M3 planes, bf16 out (experiment)", py::arg("a"), py::arg("b"));
  m.def("tri_mul_backward", &tri_mul_backward,
        "TriangleMultiplicativeUpdate backward: [dz, 16 parameter gradients (fp32), their buffer]",
        py::arg("z"), py::arg("mask"), py::arg("dy"), py::arg("params"), py::arg("c_z"),
        py::arg("c"), py::arg("outgoing"), py::arg("eps_in") = 1e-5, py::arg("eps_out") = 1e-5);
  m.def("tri_attn_backward", &tri_attn_backward,
        "TriangleAttention backward: [dx, 10 parameter gradients (fp32), their buffer]", py::arg("x"),
        py::arg("mask"), py::arg("dy"), py::arg("params"), py::arg("c_in"), py::arg("c_h"),
        py::arg("no_heads"), py::arg("starting"), py::arg("eps") = 1e-5);
  m.def("tri_attn_backward_heads", &tri_attn_backward_heads,
        "tri_attn_backward for every head shape of the forward kernels", py::arg("x"), py::arg("mask"),
        py::arg("dy"), py::arg("params"), py::arg("c_in"), py::arg("c_h"), py::arg("no_heads"),
        py::arg("starting"), py::arg("eps") = 1e-5);
  m.def("pair_transition_pack", &pair_transition_pack, "Pack PairTransition parameters",
        py::arg("params"), py::arg("c"), py::arg("n"), py::arg("fp32") = false);
  m.def("pair_transition_forward", &pair_transition_forward,
        "Fused PairTransition forward: (residual ? p : 0) + transition(p), times mask",
        py::arg("p"), py::arg("mask"), py::arg("packed"), py::arg("c"), py::arg("n"),
        py::arg("residual") = false, py::arg("eps") = 1e-5);
  m.def("pair_transition_backward", &pair_transition_backward,
        "PairTransition backward: [dp, 6 parameter gradients (fp32), their buffer]", py::arg("p"), py::arg("dy"),
        py::arg("params"), py::arg("c"), py::arg("n"), py::arg("eps") = 1e-5);
  m.def("tri_attn_pack", &tri_attn_pack, "Pack TriangleAttention parameters", py::arg("params"),
        py::arg("c_in"), py::arg("c_h"), py::arg("no_heads"), py::arg("fp32"));
  m.def("tri_attn_forward", &tri_attn_forward, "Fused TriangleAttention forward", py::arg("x"),
        py::arg("mask"), py::arg("packed"), py::arg("c_in"), py::arg("c_h"), py::arg("no_heads"),
        py::arg("starting"), py::arg("residual") = false, py::arg("eps") = 1e-5,
        py::arg("chunk_rows") = 0, py::arg("inf") = 1e9);
  m.def("layer_norm", &layer_norm,
        "layer_norm_forward under autograd (differentiable once, in reverse mode).  Without strict, None where an "
        "input has a forward-mode tangent",
        py::arg("x"), py::arg("weight") = py::none(), py::arg("bias") = py::none(), py::arg("eps") = 1e-5,
        py::arg("strict") = true);
  m.def("layer_norm_forward", &layer_norm_forward,
        "LayerNorm over the last dimension, optional affine in either parameter type", py::arg("x"),
        py::arg("weight") = py::none(), py::arg("bias") = py::none(), py::arg("eps") = 1e-5);
  m.def("layer_norm_backward", &layer_norm_backward,
        "layer_norm_forward's backward: [dx, dweight, dbias], None where not needed", py::arg("x"), py::arg("dy"),
        py::arg("weight") = py::none(), py::arg("eps") = 1e-5, py::arg("need_x") = true,
        py::arg("need_weight") = true, py::arg("need_bias") = true);
  m.def("dropout", &dropout,
        "residual + dropout(x) with the mask of a counter-based generator (shared along shared_dim), under autograd.  "
        "Without strict, None where an input has a forward-mode tangent",
        py::arg("x"), py::arg("p"), py::arg("seed"), py::arg("offset") = 0, py::arg("shared_dim") = py::none(),
        py::arg("residual") = py::none(), py::arg("seed_device") = py::none(), py::arg("strict") = true);
  m.def("group_norm", &group_norm,
        "group_norm_forward under autograd (differentiable once, in reverse mode).  Without strict, None where an "
        "input has a forward-mode tangent",
        py::arg("x"), py::arg("groups"), py::arg("weight") = py::none(), py::arg("bias") = py::none(),
        py::arg("eps") = 1e-5, py::arg("activation") = 0, py::arg("mask") = py::none(), py::arg("strict") = true);
  m.def("group_norm_forward", &group_norm_forward,
        "Group norm over channels-last x [B, ..., C] with an activation (0 none, 1 silu, 2 gelu): [y, stats]",
        py::arg("x"), py::arg("groups"), py::arg("weight") = py::none(), py::arg("bias") = py::none(),
        py::arg("eps") = 1e-5, py::arg("activation") = 0, py::arg("mask") = py::none());
  m.def("group_norm_backward", &group_norm_backward,
        "group_norm_forward's backward: [dx, dweight, dbias], None where not needed", py::arg("x"), py::arg("dy"),
        py::arg("stats"), py::arg("groups"), py::arg("weight") = py::none(), py::arg("bias") = py::none(),
        py::arg("activation") = 0, py::arg("mask") = py::none(), py::arg("need_x") = true,
        py::arg("need_weight") = true, py::arg("need_bias") = true);
  m.def("grad_norm", &grad_norm,
        "Norm over every value of the tensors (fp32 scalar; norm_type 1, 2 or inf).  Without strict, None where a "
        "tensor is not bf16 or fp32 on one GPU",
        py::arg("tensors"), py::arg("norm_type") = 2.0, py::arg("strict") = true);
  m.def("grad_clip", &grad_clip, "Clip the tensors by their global norm into outs (None: in place); the norm",
        py::arg("tensors"), py::arg("outs"), py::arg("max_norm"), py::arg("norm_type") = 2.0, py::arg("strict") = true);
  m.def("grad_clip_parameters", &grad_clip_parameters,
        "grad_clip in place on the parameters' gradients; None where there is none, or one not for the kernels",
        py::arg("parameters"), py::arg("max_norm"), py::arg("norm_type") = 2.0);
  m.def("grad_clip_with_norm", &grad_clip_with_norm, "grad_clip by a given norm (one float32 value on the GPU)",
        py::arg("tensors"), py::arg("outs"), py::arg("max_norm"), py::arg("norm"));
  m.def("version", []() { return gtk_version(); });
  m.def("timing_enable", [](bool on) { check_rc(gtk_timing_enable(on ? 1 : 0)); },
        "Record HIP events around every kernel launch (per-kernel timing)", py::arg("on"));
  m.def("timing_report", &timing_report,
        "Wait for recorded kernels; {name: (count, total_ms, min_ms, max_ms)}; clears records");
}
