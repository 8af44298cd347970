// torch_ext.cpp - thin torch binding of the krsi_b200 C ABI.
//
// Registers the operator names and schemas the reference registers through
// torch.library.triton_op (library/rmsnorm.py:86-103, library/geglu.py:85-101,
// library/relpos_attention.py:175-195), so that torch.compile(fullgraph=True) traces them
// as opaque ops.  The binding owns allocation (outputs and workspaces come from the torch
// caching allocator on the input's device), passes the current CUDA stream, and turns a
// nonzero krsi_status into a Python RuntimeError.  No synchronisation, so the ops can be
// captured in CUDA graphs.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "../../include/krsi_b200.h"

namespace {

int krsi_dtype_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return KRSI_F32;
    case at::kBFloat16: return KRSI_BF16;
    case at::kHalf: return KRSI_F16;
    default: TORCH_CHECK(false, "krsi: unsupported dtype ", t.scalar_type());
  }
  return -1;
}

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == KRSI_OK, what, " failed: ", krsi_error_string(rc), " (status ", rc, ")");
}

void check_cuda(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), "krsi: ", name, " must be a CUDA tensor");
}

at::Tensor workspace(const at::Tensor& like, size_t bytes) {
  return at::empty({(int64_t)std::max<size_t>(bytes, 16)}, like.options().dtype(at::kByte));
}

// ---------------------------------------------------------------- RMSNorm
std::tuple<at::Tensor, at::Tensor> rmsnorm_fwd(const at::Tensor& x2d_in, const at::Tensor& w_in, double eps) {
  check_cuda(x2d_in, "x2d");
  check_cuda(w_in, "w");
  TORCH_CHECK(x2d_in.dim() == 2, "rmsnorm: x2d must be 2-D, got ", x2d_in.dim(), "-D");
  TORCH_CHECK(w_in.dim() == 1 && w_in.size(0) == x2d_in.size(1), "rmsnorm: w must be [", x2d_in.size(1), "]");
  c10::cuda::CUDAGuard guard(x2d_in.device());
  auto x2d = x2d_in.contiguous();
  auto w = w_in.contiguous();
  auto y = at::empty_like(x2d);
  auto rstd = at::empty({x2d.size(0)}, x2d.options().dtype(at::kFloat));
  check_rc(krsi_rmsnorm_fwd(x2d.data_ptr(), w.data_ptr(), y.data_ptr(), rstd.data_ptr<float>(), x2d.size(0),
                            x2d.size(1), (float)eps, krsi_dtype_of(x2d), krsi_dtype_of(w),
                            at::cuda::getCurrentCUDAStream()),
           "krsi_rmsnorm_fwd");
  return {y, rstd};
}

std::tuple<at::Tensor, at::Tensor> rmsnorm_bwd(const at::Tensor& g_in, const at::Tensor& x2d_in,
                                               const at::Tensor& w_in, const at::Tensor& rstd_in) {
  check_cuda(g_in, "g");
  check_cuda(x2d_in, "x2d");
  TORCH_CHECK(x2d_in.dim() == 2 && g_in.sizes() == x2d_in.sizes(), "rmsnorm_bwd: g must match x2d");
  TORCH_CHECK(rstd_in.scalar_type() == at::kFloat && rstd_in.numel() == x2d_in.size(0), "rmsnorm_bwd: bad rstd");
  c10::cuda::CUDAGuard guard(x2d_in.device());
  auto x2d = x2d_in.contiguous();
  auto g = g_in.to(x2d.scalar_type()).contiguous();
  auto w = w_in.contiguous();
  auto rstd = rstd_in.contiguous();
  auto dx = at::empty_like(x2d);
  auto dw = at::empty_like(w);
  size_t ws = 0;
  check_rc(krsi_rmsnorm_bwd_workspace_size(x2d.size(0), x2d.size(1), &ws), "krsi_rmsnorm_bwd_workspace_size");
  auto wsp = workspace(x2d, ws);
  check_rc(krsi_rmsnorm_bwd(g.data_ptr(), x2d.data_ptr(), w.data_ptr(), rstd.data_ptr<float>(), dx.data_ptr(),
                            dw.data_ptr(), wsp.data_ptr(), (size_t)wsp.numel(), x2d.size(0), x2d.size(1),
                            krsi_dtype_of(x2d), krsi_dtype_of(w), at::cuda::getCurrentCUDAStream()),
           "krsi_rmsnorm_bwd");
  return {dx, dw};
}

std::tuple<at::Tensor, at::Tensor> rmsnorm_bwd_add(const at::Tensor& g_in, const at::Tensor& x2d_in,
                                                   const at::Tensor& w_in, const at::Tensor& rstd_in,
                                                   const at::Tensor& gadd_in) {
  check_cuda(g_in, "g");
  check_cuda(x2d_in, "x2d");
  check_cuda(gadd_in, "gadd");
  TORCH_CHECK(x2d_in.dim() == 2 && g_in.sizes() == x2d_in.sizes() && gadd_in.sizes() == x2d_in.sizes(),
              "rmsnorm_bwd_add: g and gadd must match x2d");
  TORCH_CHECK(rstd_in.scalar_type() == at::kFloat && rstd_in.numel() == x2d_in.size(0), "rmsnorm_bwd_add: bad rstd");
  c10::cuda::CUDAGuard guard(x2d_in.device());
  auto x2d = x2d_in.contiguous();
  auto g = g_in.to(x2d.scalar_type()).contiguous();
  auto gadd = gadd_in.to(x2d.scalar_type()).contiguous();
  auto w = w_in.contiguous();
  auto rstd = rstd_in.contiguous();
  auto dx = at::empty_like(x2d);
  auto dw = at::empty_like(w);
  size_t ws = 0;
  check_rc(krsi_rmsnorm_bwd_workspace_size(x2d.size(0), x2d.size(1), &ws), "krsi_rmsnorm_bwd_workspace_size");
  auto wsp = workspace(x2d, ws);
  check_rc(krsi_rmsnorm_bwd_add(g.data_ptr(), x2d.data_ptr(), w.data_ptr(), rstd.data_ptr<float>(), gadd.data_ptr(),
                                dx.data_ptr(), dw.data_ptr(), wsp.data_ptr(), (size_t)wsp.numel(), x2d.size(0),
                                x2d.size(1), krsi_dtype_of(x2d), krsi_dtype_of(w), at::cuda::getCurrentCUDAStream()),
           "krsi_rmsnorm_bwd_add");
  return {dx, dw};
}

// ---------------------------------------------------------------- GEGLU
at::Tensor geglu_fwd(const at::Tensor& u_in) {
  check_cuda(u_in, "u");
  TORCH_CHECK(u_in.dim() == 2 && u_in.size(1) % 2 == 0, "geglu: u must be [rows, 2F]");
  c10::cuda::CUDAGuard guard(u_in.device());
  auto u = u_in.contiguous();
  const int64_t F = u.size(1) / 2;
  auto out = at::empty({u.size(0), F}, u.options());
  check_rc(krsi_geglu_fwd(u.data_ptr(), out.data_ptr(), u.size(0), F, krsi_dtype_of(u),
                          at::cuda::getCurrentCUDAStream()),
           "krsi_geglu_fwd");
  return out;
}

at::Tensor geglu_bwd(const at::Tensor& g_in, const at::Tensor& u_in) {
  check_cuda(g_in, "g");
  check_cuda(u_in, "u");
  TORCH_CHECK(u_in.dim() == 2 && u_in.size(1) % 2 == 0, "geglu_bwd: u must be [rows, 2F]");
  TORCH_CHECK(g_in.dim() == 2 && g_in.size(0) == u_in.size(0) && g_in.size(1) * 2 == u_in.size(1),
              "geglu_bwd: g must be [rows, F]");
  c10::cuda::CUDAGuard guard(u_in.device());
  auto u = u_in.contiguous();
  auto g = g_in.to(u.scalar_type()).contiguous();
  auto du = at::empty_like(u);
  check_rc(krsi_geglu_bwd(g.data_ptr(), u.data_ptr(), du.data_ptr(), u.size(0), u.size(1) / 2, krsi_dtype_of(u),
                          at::cuda::getCurrentCUDAStream()),
           "krsi_geglu_bwd");
  return du;
}

// ---------------------------------------------------------------- projection + GEGLU
std::tuple<at::Tensor, at::Tensor> linear_geglu_fwd(const at::Tensor& x_in, const at::Tensor& w_in) {
  check_cuda(x_in, "x2d");
  check_cuda(w_in, "w");
  TORCH_CHECK(x_in.dim() == 2, "linear_geglu: x2d must be 2-D, got ", x_in.dim(), "-D");
  TORCH_CHECK(w_in.dim() == 2 && w_in.size(1) == x_in.size(1) && w_in.size(0) % 2 == 0,
              "linear_geglu: w must be [2F, ", x_in.size(1), "]");
  TORCH_CHECK(x_in.scalar_type() == w_in.scalar_type(), "linear_geglu: x2d and w must have one dtype");
  c10::cuda::CUDAGuard guard(x_in.device());
  auto x = x_in.contiguous();
  auto w = w_in.contiguous();
  const int64_t F = w.size(0) / 2;
  auto u = at::empty({x.size(0), 2 * F}, x.options());
  auto out = at::empty({x.size(0), F}, x.options());
  check_rc(krsi_linear_geglu_fwd(x.data_ptr(), w.data_ptr(), u.data_ptr(), out.data_ptr(), x.size(0), x.size(1), F,
                                 krsi_dtype_of(x), at::cuda::getCurrentCUDAStream()),
           "krsi_linear_geglu_fwd");
  return {u, out};
}

at::Tensor linear_geglu_bwd(const at::Tensor& dy_in, const at::Tensor& w_in, const at::Tensor& u_in) {
  check_cuda(dy_in, "dy");
  check_cuda(w_in, "w");
  check_cuda(u_in, "u");
  TORCH_CHECK(dy_in.dim() == 2 && w_in.dim() == 2 && u_in.dim() == 2, "linear_geglu_bwd: 2-D tensors expected");
  TORCH_CHECK(w_in.size(0) == dy_in.size(1), "linear_geglu_bwd: w must be [", dy_in.size(1), ", F]");
  TORCH_CHECK(u_in.size(0) == dy_in.size(0) && u_in.size(1) == 2 * w_in.size(1),
              "linear_geglu_bwd: u must be [", dy_in.size(0), ", ", 2 * w_in.size(1), "]");
  TORCH_CHECK(dy_in.scalar_type() == w_in.scalar_type() && u_in.scalar_type() == w_in.scalar_type(),
              "linear_geglu_bwd: dy, w and u must have one dtype");
  c10::cuda::CUDAGuard guard(dy_in.device());
  auto dy = dy_in.contiguous();
  auto w = w_in.contiguous();
  auto u = u_in.contiguous();
  auto du = at::empty_like(u);
  check_rc(krsi_linear_geglu_bwd(dy.data_ptr(), w.data_ptr(), u.data_ptr(), du.data_ptr(), dy.size(0), dy.size(1),
                                 w.size(1), krsi_dtype_of(dy), at::cuda::getCurrentCUDAStream()),
           "krsi_linear_geglu_bwd");
  return du;
}

// ---------------------------------------------------------------- relpos attention
void check_attn_shapes(const at::Tensor& qkv, const at::Tensor& pd, int64_t B, int64_t S, int64_t H, int64_t D) {
  TORCH_CHECK(B >= 0 && S >= 0 && H > 0 && D > 0, "relpos_attention: bad B/S/H/D");
  TORCH_CHECK(qkv.dim() == 2 && qkv.size(0) == B * S && qkv.size(1) == 3 * H * D,
              "relpos_attention: qkv must be [B*S, 3*H*D] = [", B * S, ", ", 3 * H * D, "], got ", qkv.sizes());
  TORCH_CHECK(pd.dim() == 2 && pd.size(0) == H && pd.size(1) == std::max<int64_t>(2 * S - 1, 0),
              "relpos_attention: pd must be [H, 2S-1] = [", H, ", ", 2 * S - 1, "], got ", pd.sizes());
}

// qkv may be a row-strided view (the reference reads it in place with stride(0)); the
// kernels need unit column stride and a row stride that is a multiple of 8 elements.
at::Tensor qkv_view(const at::Tensor& qkv) {
  if (qkv.stride(1) == 1 && qkv.stride(0) % 8 == 0 && qkv.stride(0) >= qkv.size(1) &&
      (reinterpret_cast<uintptr_t>(qkv.data_ptr()) & 15u) == 0)
    return qkv;
  return qkv.contiguous();
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> relpos_attn_fwd(const at::Tensor& qkv_in, const at::Tensor& pd_in,
                                                               int64_t B, int64_t S, int64_t H, int64_t D,
                                                               double scale) {
  check_cuda(qkv_in, "qkv");
  check_cuda(pd_in, "pd");
  check_attn_shapes(qkv_in, pd_in, B, S, H, D);
  c10::cuda::CUDAGuard guard(qkv_in.device());
  auto qkv = qkv_view(qkv_in);
  auto pd = pd_in.to(at::kFloat).contiguous();
  auto out = at::empty({B * S, H * D}, qkv.options().memory_format(at::MemoryFormat::Contiguous));
  auto out32 = at::empty({B * S, H * D}, qkv.options().dtype(at::kFloat));
  auto lse = at::empty({B * H, S}, qkv.options().dtype(at::kFloat));
  check_rc(krsi_relpos_attn_fwd(qkv.data_ptr(), qkv.stride(0), pd.data_ptr<float>(), out.data_ptr(),
                                out32.data_ptr<float>(), lse.data_ptr<float>(), B, S, H, D, (float)scale,
                                krsi_dtype_of(qkv), at::cuda::getCurrentCUDAStream()),
           "krsi_relpos_attn_fwd");
  return {out, out32, lse};
}

std::tuple<at::Tensor, at::Tensor> relpos_attn_bwd(const at::Tensor& dout_in, const at::Tensor& qkv_in,
                                                   const at::Tensor& pd_in, const at::Tensor& out32_in,
                                                   const at::Tensor& lse_in, int64_t B, int64_t S, int64_t H,
                                                   int64_t D, double scale) {
  check_cuda(dout_in, "dout");
  check_cuda(qkv_in, "qkv");
  check_attn_shapes(qkv_in, pd_in, B, S, H, D);
  TORCH_CHECK(dout_in.numel() == B * S * H * D, "relpos_attn_bwd: dout must have B*S*H*D elements");
  TORCH_CHECK(out32_in.scalar_type() == at::kFloat && out32_in.numel() == B * S * H * D, "relpos_attn_bwd: bad out32");
  TORCH_CHECK(lse_in.scalar_type() == at::kFloat && lse_in.numel() == B * H * S, "relpos_attn_bwd: bad lse");
  c10::cuda::CUDAGuard guard(qkv_in.device());
  auto qkv = qkv_view(qkv_in);
  auto dout = dout_in.to(qkv.scalar_type()).contiguous();
  auto pd = pd_in.to(at::kFloat).contiguous();
  auto out32 = out32_in.contiguous();
  auto lse = lse_in.contiguous();
  auto dqkv = at::empty({B * S, 3 * H * D}, qkv.options().memory_format(at::MemoryFormat::Contiguous));
  auto dpd = at::empty({H, std::max<int64_t>(2 * S - 1, 0)}, qkv.options().dtype(at::kFloat));
  size_t ws = 0;
  check_rc(krsi_relpos_attn_bwd_workspace_size(B, S, H, D, &ws), "krsi_relpos_attn_bwd_workspace_size");
  auto wsp = workspace(qkv, ws);
  check_rc(krsi_relpos_attn_bwd(dout.data_ptr(), qkv.data_ptr(), qkv.stride(0), pd.data_ptr<float>(),
                                out32.data_ptr<float>(), lse.data_ptr<float>(), dqkv.data_ptr(), dqkv.stride(0),
                                dpd.data_ptr<float>(), wsp.data_ptr(), (size_t)wsp.numel(), B, S, H, D,
                                (float)scale, krsi_dtype_of(qkv), at::cuda::getCurrentCUDAStream()),
           "krsi_relpos_attn_bwd");
  return {dqkv, dpd};
}

// ---------------------------------------------------------------- T5 bucketed relative position
at::Tensor t5_bias_fwd(const at::Tensor& table_in, int64_t S, int64_t num_buckets, int64_t max_distance,
                       bool bidirectional) {
  check_cuda(table_in, "table");
  TORCH_CHECK(table_in.dim() == 2 && table_in.size(0) == num_buckets, "t5_bias: table must be [num_buckets, H]");
  TORCH_CHECK(S >= 0, "t5_bias: S must be >= 0");
  c10::cuda::CUDAGuard guard(table_in.device());
  auto table = table_in.contiguous();
  auto pd = at::empty({table.size(1), std::max<int64_t>(2 * S - 1, 0)}, table.options().dtype(at::kFloat));
  check_rc(krsi_t5_bias_fwd(table.data_ptr(), pd.data_ptr<float>(), S, table.size(1), (int)num_buckets,
                            (int)max_distance, bidirectional ? 1 : 0, krsi_dtype_of(table),
                            at::cuda::getCurrentCUDAStream()),
           "krsi_t5_bias_fwd");
  return pd;
}

at::Tensor t5_bias_bwd(const at::Tensor& dpd_in, const at::Tensor& table, int64_t S, int64_t num_buckets,
                       int64_t max_distance, bool bidirectional) {
  check_cuda(dpd_in, "dpd");
  TORCH_CHECK(table.dim() == 2 && table.size(0) == num_buckets, "t5_bias_bwd: table must be [num_buckets, H]");
  TORCH_CHECK(dpd_in.dim() == 2 && dpd_in.size(0) == table.size(1) && dpd_in.size(1) == std::max<int64_t>(2 * S - 1, 0),
              "t5_bias_bwd: dpd must be [H, 2S-1]");
  c10::cuda::CUDAGuard guard(dpd_in.device());
  auto dpd = dpd_in.to(at::kFloat).contiguous();
  auto dtable = at::empty(table.sizes(), table.options().memory_format(at::MemoryFormat::Contiguous));
  check_rc(krsi_t5_bias_bwd(dpd.data_ptr<float>(), dtable.data_ptr(), S, table.size(1), (int)num_buckets,
                            (int)max_distance, bidirectional ? 1 : 0, krsi_dtype_of(table),
                            at::cuda::getCurrentCUDAStream()),
           "krsi_t5_bias_bwd");
  return dtable;
}

// ---------------------------------------------------------------- embedding
int token_bits_of(const at::Tensor& t, const char* what) {
  TORCH_CHECK(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt, what, " must be int32 or int64, got ",
              t.scalar_type());
  return t.scalar_type() == at::kLong ? 64 : 32;
}

void check_same_device(const at::Tensor& a, const at::Tensor& b, const char* what) {
  TORCH_CHECK(a.device() == b.device(), what, ": tensors on different devices (", a.device(), " and ", b.device(), ")");
}

// padding_idx is its registered gradient's: the lookup itself treats that token like any other.
at::Tensor embedding_fwd(const at::Tensor& tokens_in, const at::Tensor& table_in, double scale, int64_t /*padding_idx*/) {
  check_cuda(tokens_in, "tokens");
  check_cuda(table_in, "table");
  check_same_device(tokens_in, table_in, "embedding");
  TORCH_CHECK(table_in.dim() == 2 && table_in.size(0) > 0 && table_in.size(1) > 0, "embedding: table must be [V, d]");
  const int bits = token_bits_of(tokens_in, "embedding: tokens");
  c10::cuda::CUDAGuard guard(table_in.device());
  auto tokens = tokens_in.contiguous();
  auto table = table_in.contiguous();
  auto sizes = tokens.sizes().vec();
  sizes.push_back(table.size(1));
  auto out = at::empty(sizes, table.options());
  check_rc(krsi_embedding_fwd(tokens.data_ptr(), bits, table.data_ptr(), out.data_ptr(), tokens.numel(), table.size(0),
                              table.size(1), (float)scale, krsi_dtype_of(table), at::cuda::getCurrentCUDAStream()),
           "krsi_embedding_fwd");
  return out;
}

// The gradient of a table of V rows in g's type.  It needs nothing of the table itself, so the autograd node does
// not keep it: a table that is changed in place between forward and backward is none of its business.
at::Tensor embedding_grad(const at::Tensor& g_in, const at::Tensor& tokens_in, int64_t V, double scale,
                          int64_t padding_idx) {
  check_cuda(g_in, "g");
  check_cuda(tokens_in, "tokens");
  check_same_device(g_in, tokens_in, "embedding_grad");
  TORCH_CHECK(g_in.dim() > 0 && g_in.size(-1) > 0 && g_in.numel() == tokens_in.numel() * g_in.size(-1),
              "embedding_grad: g must be [*tokens.shape, d]");
  TORCH_CHECK(V > 0 && padding_idx >= -1 && padding_idx < V, "embedding_grad: padding_idx out of range");
  const int bits = token_bits_of(tokens_in, "embedding_grad: tokens");
  c10::cuda::CUDAGuard guard(g_in.device());
  auto tokens = tokens_in.contiguous();
  auto g = g_in.contiguous();
  const int64_t n = tokens.numel(), d = g.size(-1);
  auto dtable = at::empty({V, d}, g.options());
  size_t ws = 0;
  check_rc(krsi_embedding_bwd_workspace_size(n, V, d, &ws), "krsi_embedding_bwd_workspace_size");
  auto wsp = workspace(g, ws);
  check_rc(krsi_embedding_bwd(tokens.data_ptr(), bits, g.data_ptr(), dtable.data_ptr(), wsp.data_ptr(),
                              (size_t)wsp.numel(), n, V, d, (float)scale, padding_idx, krsi_dtype_of(g),
                              at::cuda::getCurrentCUDAStream()),
           "krsi_embedding_bwd");
  return dtable;
}

// The same for a table at hand, whose shape and type the gradient takes.
at::Tensor embedding_bwd(const at::Tensor& g_in, const at::Tensor& tokens_in, const at::Tensor& table, double scale,
                         int64_t padding_idx) {
  check_cuda(table, "table");
  check_same_device(g_in, table, "embedding_bwd");
  TORCH_CHECK(table.dim() == 2 && g_in.dim() > 0 && g_in.size(-1) == table.size(1) &&
                  g_in.numel() == tokens_in.numel() * table.size(1),
              "embedding_bwd: g must be [*tokens.shape, d]");
  return embedding_grad(g_in.to(table.scalar_type()), tokens_in, table.size(0), scale, padding_idx);
}

// ---------------------------------------------------------------- GEGLU with an 8-bit checkpoint
// (out, q, exponents): the checkpoint is empty unless it is to be kept.
std::tuple<at::Tensor, at::Tensor, at::Tensor> geglu_q8_fwd(const at::Tensor& u_in, bool keep) {
  check_cuda(u_in, "u");
  TORCH_CHECK(u_in.dim() == 2 && u_in.size(1) % 2 == 0, "geglu_q8: u must be [rows, 2F]");
  c10::cuda::CUDAGuard guard(u_in.device());
  auto u = u_in.contiguous();
  const int64_t rows = u.size(0), F = u.size(1) / 2;
  auto out = at::empty({rows, F}, u.options());
  auto q = at::empty({keep ? rows : 0, 2 * F}, u.options().dtype(at::kChar));
  auto ex = at::empty({keep ? rows : 0, (F + 31) / 32, 2}, u.options().dtype(at::kByte));
  check_rc(krsi_geglu_q8_fwd(u.data_ptr(), out.data_ptr(), keep ? q.data_ptr() : nullptr,
                             keep ? ex.data_ptr() : nullptr, rows, F, krsi_dtype_of(u),
                             at::cuda::getCurrentCUDAStream()),
           "krsi_geglu_q8_fwd");
  return {out, q, ex};
}

// (du, out): out is GEGLU of the checkpoint's values, empty unless asked for.
std::tuple<at::Tensor, at::Tensor> geglu_q8_bwd(const at::Tensor& g_in, const at::Tensor& q, const at::Tensor& ex,
                                                bool want_out) {
  check_cuda(g_in, "g");
  check_cuda(q, "q");
  check_cuda(ex, "exponents");
  TORCH_CHECK(q.dim() == 2 && q.size(1) % 2 == 0 && q.scalar_type() == at::kChar && q.is_contiguous(),
              "geglu_q8_bwd: q must be a contiguous int8 [rows, 2F]");
  const int64_t rows = q.size(0), F = q.size(1) / 2;
  TORCH_CHECK(g_in.dim() == 2 && g_in.size(0) == rows && g_in.size(1) == F, "geglu_q8_bwd: g must be [rows, F]");
  TORCH_CHECK(ex.scalar_type() == at::kByte && ex.is_contiguous() && ex.numel() == rows * ((F + 31) / 32) * 2,
              "geglu_q8_bwd: exponents must be a contiguous uint8 [rows, ceil(F / 32), 2]");
  check_same_device(g_in, q, "geglu_q8_bwd");
  check_same_device(ex, q, "geglu_q8_bwd");
  c10::cuda::CUDAGuard guard(q.device());
  auto g = g_in.contiguous();
  auto du = at::empty({rows, 2 * F}, g.options());
  auto out = at::empty({want_out ? rows : 0, F}, g.options());
  check_rc(krsi_geglu_q8_bwd(g.data_ptr(), q.data_ptr(), ex.data_ptr(), du.data_ptr(),
                             want_out ? out.data_ptr() : nullptr, rows, F, krsi_dtype_of(g),
                             at::cuda::getCurrentCUDAStream()),
           "krsi_geglu_q8_bwd");
  return {du, out};
}

// ---------------------------------------------------------------- vocabulary cross entropy
// The operands as the kernels take them, and a workspace of the mode's size.
struct CeCall {
  at::Tensor x, w, targets, ws;
  int bits, dtype;
  int64_t N, V, K;
};
int ce_mode(int kind, bool want_dx, bool want_dw) {
  if (!want_dx && !want_dw) return 0;
  return kind + (want_dx ? 0 : KRSI_CE_NO_DX) + (want_dw ? 0 : KRSI_CE_NO_DW);
}
CeCall ce_call(const at::Tensor& x_in, const at::Tensor& w_in, const at::Tensor& targets_in, int mode) {
  check_cuda(x_in, "x2d");
  check_cuda(w_in, "w");
  check_cuda(targets_in, "targets");
  check_same_device(x_in, w_in, "linear_cross_entropy");
  check_same_device(x_in, targets_in, "linear_cross_entropy");
  TORCH_CHECK(x_in.dim() == 2, "linear_cross_entropy: x2d must be 2-D, got ", x_in.dim(), "-D");
  TORCH_CHECK(w_in.dim() == 2 && w_in.size(0) > 0 && w_in.size(1) == x_in.size(1),
              "linear_cross_entropy: w must be [V, ", x_in.size(1), "]");
  TORCH_CHECK(x_in.scalar_type() == w_in.scalar_type(), "linear_cross_entropy: x2d and w must have one dtype");
  TORCH_CHECK(targets_in.dim() == 1 && targets_in.size(0) == x_in.size(0), "linear_cross_entropy: targets must be [",
              x_in.size(0), "]");
  const int bits = token_bits_of(targets_in, "linear_cross_entropy: targets");
  // 16-byte aligned operands: a view that starts elsewhere is copied
  auto aligned = [](const at::Tensor& t) {
    auto c = t.contiguous();
    return (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15u) == 0 ? c : c.clone();
  };
  CeCall c{aligned(x_in), aligned(w_in), targets_in.contiguous(), {}, bits, krsi_dtype_of(x_in),
           x_in.size(0), w_in.size(0), x_in.size(1)};
  size_t ws = 0;
  check_rc(krsi_linear_ce_workspace_size(c.N, c.V, c.K, mode, &ws), "krsi_linear_ce_workspace_size");
  c.ws = workspace(c.x, ws);
  return c;
}

// (loss rows, loss, row weight, stats, dx, dw): stats is for linear_ce_grad; the gradients are fp32, of the sum
// of the losses and without `scale`, or empty.  reduction 0 none, 1 mean, 2 sum.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> linear_ce_fwd(
    const at::Tensor& x_in, const at::Tensor& w_in, const at::Tensor& targets_in, double scale, int64_t ignore_index,
    double z_loss, int64_t reduction, bool want_dx, bool want_dw) {
  TORCH_CHECK(x_in.is_cuda(), "krsi: x2d must be a CUDA tensor");
  c10::cuda::CUDAGuard guard(x_in.device());
  const CeCall c = ce_call(x_in, w_in, targets_in, ce_mode(1, want_dx, want_dw));
  auto f32 = c.x.options().dtype(at::kFloat);
  auto loss = at::empty({c.N}, f32);
  // (tensors of their own: the weight is saved, and a caller may change the loss in place)
  auto total = reduction != 0 ? at::empty({}, f32) : at::empty({0}, f32);
  auto weight = at::empty({reduction != 0 ? 1 : 0}, f32);
  auto stats = at::empty({c.N, 2}, f32);
  auto dx = at::empty({want_dx ? c.N : 0, c.K}, f32);
  auto dw = at::empty({want_dw ? c.V : 0, c.K}, f32);
  check_rc(krsi_linear_ce_fwd(c.x.data_ptr(), c.w.data_ptr(), c.targets.data_ptr(), c.bits, loss.data_ptr<float>(),
                              reduction != 0 ? total.data_ptr<float>() : nullptr,
                              reduction != 0 ? weight.data_ptr<float>() : nullptr, stats.data_ptr<float>(),
                              want_dx ? dx.data_ptr<float>() : nullptr, want_dw ? dw.data_ptr<float>() : nullptr,
                              c.ws.data_ptr(), (size_t)c.ws.numel(), c.N, c.V, c.K, (float)scale, ignore_index,
                              (float)z_loss, reduction == 1, c.dtype, at::cuda::getCurrentCUDAStream()),
           "krsi_linear_ce_fwd");
  return {loss, total, weight, stats, dx, dw};
}

// Gradients in x2d's dtype for g, the upstream gradient of each row's loss ([N], or one for all), times
// weight (one value, or empty); stats: linear_ce_fwd's.
std::tuple<at::Tensor, at::Tensor> linear_ce_grad(const at::Tensor& g_in, const at::Tensor& weight_in,
                                                  const at::Tensor& stats, const at::Tensor& x_in,
                                                  const at::Tensor& w_in,
                                                  const at::Tensor& targets_in, double scale, int64_t ignore_index,
                                                  double z_loss, bool want_dx, bool want_dw) {
  TORCH_CHECK(x_in.is_cuda(), "krsi: x2d must be a CUDA tensor");
  c10::cuda::CUDAGuard guard(x_in.device());
  const CeCall c = ce_call(x_in, w_in, targets_in, ce_mode(2, want_dx, want_dw));
  TORCH_CHECK(g_in.numel() == c.N || g_in.numel() == 1, "linear_ce_grad: g must have ", c.N, " values or one");
  TORCH_CHECK(weight_in.numel() <= 1, "linear_ce_grad: weight must be one value or empty");
  TORCH_CHECK(stats.scalar_type() == at::kFloat && stats.is_contiguous() && stats.numel() == 2 * c.N,
              "linear_ce_grad: stats must be linear_ce_fwd's");
  check_cuda(g_in, "g");
  check_same_device(g_in, x_in, "linear_ce_grad");
  check_same_device(stats, x_in, "linear_ce_grad");
  auto g = g_in.to(at::kFloat).contiguous();
  auto weight = weight_in.to(at::kFloat).contiguous();
  auto dx = at::empty({want_dx ? c.N : 0, c.K}, c.x.options());
  auto dw = at::empty({want_dw ? c.V : 0, c.K}, c.x.options());
  if (!want_dx && !want_dw) return {dx, dw};
  check_rc(krsi_linear_ce_grad(c.x.data_ptr(), c.w.data_ptr(), c.targets.data_ptr(), c.bits, g.data_ptr<float>(),
                               g.numel() == 1 ? 0 : 1, weight.numel() == 1 ? weight.data_ptr<float>() : nullptr,
                               stats.data_ptr<float>(), want_dx ? dx.data_ptr() : nullptr,
                               want_dw ? dw.data_ptr() : nullptr, c.ws.data_ptr(), (size_t)c.ws.numel(), c.N, c.V,
                               c.K, (float)scale, ignore_index, (float)z_loss, c.dtype,
                               at::cuda::getCurrentCUDAStream()),
           "krsi_linear_ce_grad");
  return {dx, dw};
}

// scale * g * weight * grad in `like`'s dtype (g, weight: one value each).
at::Tensor linear_ce_finish(const at::Tensor& grad, const at::Tensor& g_in, const at::Tensor& weight, double scale,
                            const at::Tensor& like) {
  check_cuda(grad, "grad");
  check_cuda(g_in, "g");
  check_cuda(weight, "weight");
  TORCH_CHECK(grad.scalar_type() == at::kFloat && grad.is_contiguous(), "linear_ce_finish: grad must be contiguous fp32");
  TORCH_CHECK(g_in.numel() == 1 && weight.numel() == 1 && weight.scalar_type() == at::kFloat,
              "linear_ce_finish: g and weight must be one value each");
  c10::cuda::CUDAGuard guard(grad.device());
  auto g = g_in.to(at::kFloat);
  auto out = at::empty(grad.sizes(), grad.options().dtype(like.scalar_type()));
  check_rc(krsi_linear_ce_finish(grad.data_ptr<float>(), g.data_ptr<float>(), weight.data_ptr<float>(), out.data_ptr(),
                                 grad.numel(), (float)scale, krsi_dtype_of(like), at::cuda::getCurrentCUDAStream()),
           "krsi_linear_ce_finish");
  return out;
}

// ---------------------------------------------------------------- eager autograd
// Autograd nodes of the vocabulary operators and the 8-bit checkpoint, in C++: at small sizes a pass is
// bound by the host, and a Python autograd.Function costs it some 25 us more a step than these do (5,003 tokens
// looked up and summed: 89.6 us against 62).  (Compiled graphs use the *_fwd operators with the gradients registered in _ext.py.)
// They call the operators through the dispatcher, below autograd: dispatch modes and fake tensors see them there.
#define KRSI_OP(NAME)                                                                                    \
  ([]() -> const auto& {                                                                                 \
    static const auto handle =                                                                           \
        c10::Dispatcher::singleton().findSchemaOrThrow("krsi::" #NAME, "").typed<decltype(NAME)>();      \
    return handle;                                                                                       \
  }())
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A gradient of the gradient is not built: it would come back as zero, so it is refused.
void check_once(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, ": the backward has no gradient of its own (create_graph)");
}

// Nor is a forward-mode derivative: a dual tensor's tangent would be dropped, with a derivative of zero, on the way
// below the autograd keys.
void check_no_tangent(std::initializer_list<const at::Tensor*> inputs, const char* what) {
  for (const at::Tensor* t : inputs)
    TORCH_CHECK(!t->_fw_grad(/*level=*/0).defined(), what, ": forward-mode differentiation is not supported");
}

struct EmbeddingNode : public torch::autograd::Function<EmbeddingNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& tokens, const at::Tensor& table, double scale,
                            int64_t padding_idx) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({tokens});
    ctx->saved_data["rows"] = table.dim() > 0 ? table.size(0) : 0;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding_idx"] = padding_idx;
    return KRSI_OP(embedding_fwd).call(tokens, table, scale, padding_idx);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_once("embedding");
    const auto saved = ctx->get_saved_variables();
    at::AutoDispatchBelowADInplaceOrView below;
    return {at::Tensor(),
            KRSI_OP(embedding_grad)
                .call(g[0], saved[0], ctx->saved_data["rows"].toInt(), ctx->saved_data["scale"].toDouble(),
                      ctx->saved_data["padding_idx"].toInt()),
            at::Tensor(), at::Tensor()};
  }
};
at::Tensor embedding_autograd(const at::Tensor& tokens, const at::Tensor& table, double scale, int64_t padding_idx) {
  check_no_tangent({&table}, "embedding");
  if (at::GradMode::is_enabled() && table.requires_grad())
    return EmbeddingNode::apply(tokens, table, scale, padding_idx);
  at::AutoDispatchBelowADInplaceOrView below;
  return KRSI_OP(embedding_fwd).call(tokens, table, scale, padding_idx);
}

struct GegluQ8Node : public torch::autograd::Function<GegluQ8Node> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& u) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [out, q, ex] = KRSI_OP(geglu_q8_fwd).call(u, true);
    ctx->save_for_backward({q, ex});
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_once("geglu_q8");
    const auto saved = ctx->get_saved_variables();
    at::AutoDispatchBelowADInplaceOrView below;
    return {std::get<0>(KRSI_OP(geglu_q8_bwd).call(g[0], saved[0], saved[1], false))};
  }
};
at::Tensor geglu_q8_autograd(const at::Tensor& u) {
  check_no_tangent({&u}, "geglu_q8");
  if (at::GradMode::is_enabled() && u.requires_grad()) return GegluQ8Node::apply(u);
  at::AutoDispatchBelowADInplaceOrView below;
  return std::get<0>(KRSI_OP(geglu_q8_fwd).call(u, false));
}
at::Tensor geglu_q8_plain(const at::Tensor& u) { return std::get<0>(geglu_q8_fwd(u, false)); }

// keep: form the gradients in the forward (saved in fp32) instead of saving the operands.
at::Tensor linear_ce_plain(const at::Tensor& x, const at::Tensor& w, const at::Tensor& targets, double scale,
                           int64_t ignore_index, double z_loss, int64_t reduction, bool /*keep*/) {
  auto [loss, total, weight, stats, dx, dw] =
      KRSI_OP(linear_ce_fwd).call(x, w, targets, scale, ignore_index, z_loss, reduction, false, false);
  return reduction != 0 ? total : loss;
}
struct LinearCeNode : public torch::autograd::Function<LinearCeNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const at::Tensor& targets,
                            double scale, int64_t ignore_index, double z_loss, int64_t reduction, bool keep) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [loss, total, weight, stats, dx, dw] =
        KRSI_OP(linear_ce_fwd).call(x, w, targets, scale, ignore_index, z_loss, reduction, keep && x.requires_grad(),
                                    keep && w.requires_grad());
    if (keep) ctx->save_for_backward({weight, dx, dw, at::empty({0}, x.options())});   // (the gradients' type)
    else ctx->save_for_backward({weight, stats, x, w, targets});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->saved_data["z_loss"] = z_loss;
    ctx->saved_data["keep"] = keep;
    return reduction != 0 ? total : loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_once("linear_cross_entropy");
    const auto saved = ctx->get_saved_variables();
    const double scale = ctx->saved_data["scale"].toDouble();
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    at::AutoDispatchBelowADInplaceOrView below;
    at::Tensor dx, dw;
    if (ctx->saved_data["keep"].toBool()) {
      if (need_x) dx = KRSI_OP(linear_ce_finish).call(saved[1], g[0], saved[0], scale, saved[3]);
      if (need_w) dw = KRSI_OP(linear_ce_finish).call(saved[2], g[0], saved[0], scale, saved[3]);
    } else {
      std::tie(dx, dw) = KRSI_OP(linear_ce_grad)
                             .call(g[0], saved[0], saved[1], saved[2], saved[3], saved[4], scale,
                                   ctx->saved_data["ignore_index"].toInt(), ctx->saved_data["z_loss"].toDouble(),
                                   need_x, need_w);
      if (!need_x) dx = at::Tensor();
      if (!need_w) dw = at::Tensor();
    }
    return {dx, dw, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};
at::Tensor linear_ce_autograd(const at::Tensor& x, const at::Tensor& w, const at::Tensor& targets, double scale,
                              int64_t ignore_index, double z_loss, int64_t reduction, bool keep) {
  check_no_tangent({&x, &w}, "linear_cross_entropy");
  if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad()))
    return LinearCeNode::apply(x, w, targets, scale, ignore_index, z_loss, reduction, keep);
  at::AutoDispatchBelowADInplaceOrView below;
  return linear_ce_plain(x, w, targets, scale, ignore_index, z_loss, reduction, keep);
}

}  // namespace

TORCH_LIBRARY(krsi, m) {
  m.def("rmsnorm_fwd(Tensor x2d, Tensor w, float eps) -> (Tensor, Tensor)");
  m.def("rmsnorm_bwd(Tensor g, Tensor x2d, Tensor w, Tensor rstd) -> (Tensor, Tensor)");
  m.def("rmsnorm_bwd_add(Tensor g, Tensor x2d, Tensor w, Tensor rstd, Tensor gadd) -> (Tensor, Tensor)");
  m.def("geglu_fwd(Tensor u) -> Tensor");
  m.def("geglu_bwd(Tensor g, Tensor u) -> Tensor");
  m.def("linear_geglu_fwd(Tensor x2d, Tensor w) -> (Tensor, Tensor)");
  m.def("linear_geglu_bwd(Tensor dy, Tensor w, Tensor u) -> Tensor");
  m.def("relpos_attn_fwd(Tensor qkv, Tensor pd, int B, int S, int H, int D, float scale) -> (Tensor, Tensor, Tensor)");
  m.def("relpos_attn_bwd(Tensor dout, Tensor qkv, Tensor pd, Tensor out32, Tensor lse, int B, int S, int H, int D, "
        "float scale) -> (Tensor, Tensor)");
  m.def("t5_bias_fwd(Tensor table, int S, int num_buckets, int max_distance, bool bidirectional) -> Tensor");
  m.def("t5_bias_bwd(Tensor dpd, Tensor table, int S, int num_buckets, int max_distance, bool bidirectional) -> Tensor");
  m.def("embedding_fwd(Tensor tokens, Tensor table, float scale, int padding_idx) -> Tensor");
  m.def("embedding_bwd(Tensor g, Tensor tokens, Tensor table, float scale, int padding_idx) -> Tensor");
  m.def("embedding_grad(Tensor g, Tensor tokens, SymInt rows, float scale, int padding_idx) -> Tensor");
  m.def("embedding(Tensor tokens, Tensor table, float scale, int padding_idx) -> Tensor");
  m.def("geglu_q8(Tensor u) -> Tensor");
  m.def("linear_ce(Tensor x2d, Tensor w, Tensor targets, float scale, int ignore_index, float z_loss, int reduction, "
        "bool keep) -> Tensor");
  m.def("linear_ce_fwd(Tensor x2d, Tensor w, Tensor targets, float scale, int ignore_index, float z_loss, "
        "int reduction, bool want_dx, bool want_dw) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("linear_ce_grad(Tensor g, Tensor weight, Tensor stats, Tensor x2d, Tensor w, Tensor targets, float scale, "
        "int ignore_index, float z_loss, bool want_dx, bool want_dw) -> (Tensor, Tensor)");
  m.def("linear_ce_finish(Tensor grad, Tensor g, Tensor weight, float scale, Tensor like) -> Tensor");
  m.def("geglu_q8_fwd(Tensor u, bool keep) -> (Tensor, Tensor, Tensor)");
  m.def("geglu_q8_bwd(Tensor g, Tensor q, Tensor exponents, bool want_out) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(krsi, CUDA, m) {
  m.impl("rmsnorm_fwd", &rmsnorm_fwd);
  m.impl("rmsnorm_bwd", &rmsnorm_bwd);
  m.impl("rmsnorm_bwd_add", &rmsnorm_bwd_add);
  m.impl("geglu_fwd", &geglu_fwd);
  m.impl("geglu_bwd", &geglu_bwd);
  m.impl("linear_geglu_fwd", &linear_geglu_fwd);
  m.impl("linear_geglu_bwd", &linear_geglu_bwd);
  m.impl("relpos_attn_fwd", &relpos_attn_fwd);
  m.impl("relpos_attn_bwd", &relpos_attn_bwd);
  m.impl("t5_bias_fwd", &t5_bias_fwd);
  m.impl("t5_bias_bwd", &t5_bias_bwd);
  m.impl("embedding_fwd", &embedding_fwd);
  m.impl("embedding_bwd", &embedding_bwd);
  m.impl("embedding_grad", &embedding_grad);
  m.impl("embedding", &embedding_fwd);
  m.impl("geglu_q8", &geglu_q8_plain);
  m.impl("linear_ce", &linear_ce_plain);
  m.impl("linear_ce_fwd", &linear_ce_fwd);
  m.impl("linear_ce_grad", &linear_ce_grad);
  m.impl("linear_ce_finish", &linear_ce_finish);
  m.impl("geglu_q8_fwd", &geglu_q8_fwd);
  m.impl("geglu_q8_bwd", &geglu_q8_bwd);
}

TORCH_LIBRARY_IMPL(krsi, AutogradCUDA, m) {
  m.impl("embedding", &embedding_autograd);
  m.impl("geglu_q8", &geglu_q8_autograd);
  m.impl("linear_ce", &linear_ce_autograd);
}
