// torch_ext.cpp - thin torch binding of the krsi_b200 C ABI.
//
// Registers the operator names and schemas the reference registers through
// torch.library.triton_op (library/rmsnorm.py:86-103, library/geglu.py:85-101,
// library/relpos_attention.py:175-195), so that torch.compile(fullgraph=True) traces them
// as opaque ops.  The binding owns allocation (outputs and workspaces come from the torch
// caching allocator on the input's device), passes the current CUDA stream, and turns a
// nonzero krsi_status into a Python RuntimeError.  No synchronisation, so the ops can be
// captured in CUDA graphs.
#include <torch/csrc/python_headers.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/library.h>

#include <algorithm>
#include <vector>

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

// ---------------------------------------------------------------- residual addition and RMSNorm
// Contiguous, and rows of whole 16 bytes on 16 bytes: a view that starts elsewhere is copied, so that the bits of a
// result do not depend on where an operand lies.
at::Tensor packed(const at::Tensor& t) {
  auto c = t.contiguous();
  const bool whole = c.dim() > 0 && c.size(-1) * c.element_size() % 16 == 0;
  return whole && (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15u) != 0 ? c.clone() : c;
}
// The arguments of the entry points below.
struct NormCall {
  at::Tensor x, res, w;
};
NormCall norm_call(const at::Tensor& x_in, const c10::optional<at::Tensor>& res_in, const at::Tensor& w_in,
                   const char* what) {
  check_cuda(x_in, "x2d");
  check_cuda(w_in, "w");
  check_same_device(x_in, w_in, what);
  TORCH_CHECK(x_in.dim() == 2, what, ": x2d must be 2-D, got ", x_in.dim(), "-D");
  TORCH_CHECK(w_in.dim() == 1 && w_in.size(0) == x_in.size(1), what, ": w must be [", x_in.size(1), "]");
  NormCall c{packed(x_in), {}, packed(w_in)};
  if (res_in.has_value() && res_in->defined()) {
    check_cuda(*res_in, "res");
    check_same_device(x_in, *res_in, what);
    TORCH_CHECK(res_in->sizes() == x_in.sizes() && res_in->scalar_type() == x_in.scalar_type(), what,
                ": res must have x2d's shape and dtype");
    c.res = packed(*res_in);
  }
  return c;
}

// (y, z, rstd): z is empty where there is no res (it is x2d then).
std::tuple<at::Tensor, at::Tensor, at::Tensor> add_rmsnorm_fwd(const at::Tensor& x_in,
                                                               const c10::optional<at::Tensor>& res_in,
                                                               const at::Tensor& w_in, double eps) {
  TORCH_CHECK(x_in.is_cuda(), "krsi: x2d must be a CUDA tensor");
  c10::cuda::CUDAGuard guard(x_in.device());
  const NormCall c = norm_call(x_in, res_in, w_in, "add_rmsnorm");
  const int64_t rows = c.x.size(0), n = c.x.size(1);
  auto y = at::empty({rows, n}, c.x.options());
  auto z = at::empty({c.res.defined() ? rows : 0, n}, c.x.options());
  auto rstd = at::empty({rows}, c.x.options().dtype(at::kFloat));
  check_rc(krsi_add_rmsnorm_fwd(c.x.data_ptr(), c.res.defined() ? c.res.data_ptr() : nullptr, c.w.data_ptr(),
                                c.res.defined() ? z.data_ptr() : nullptr, y.data_ptr(), rstd.data_ptr<float>(), rows, n,
                                (float)eps, krsi_dtype_of(c.x), krsi_dtype_of(c.w), at::cuda::getCurrentCUDAStream()),
           "krsi_add_rmsnorm_fwd");
  return {y, z, rstd};
}

// (dz, dw) for the gradients of y and z, either of which may be missing (dw is then empty, or z's is not added).
std::tuple<at::Tensor, at::Tensor> add_rmsnorm_bwd(const c10::optional<at::Tensor>& gy,
                                                   const c10::optional<at::Tensor>& gz, const at::Tensor& z,
                                                   const at::Tensor& w, const at::Tensor& rstd) {
  check_cuda(z, "z");
  const bool have_z = gz.has_value() && gz->defined();
  TORCH_CHECK(z.dim() == 2 && w.dim() == 1 && w.size(0) == z.size(1), "add_rmsnorm_bwd: z must be [rows, n] and w [n]");
  TORCH_CHECK(rstd.scalar_type() == at::kFloat && rstd.numel() == z.size(0), "add_rmsnorm_bwd: bad rstd");
  TORCH_CHECK(!have_z || gz->sizes() == z.sizes(), "add_rmsnorm_bwd: gz must match z");
  c10::cuda::CUDAGuard guard(z.device());
  if (!gy.has_value() || !gy->defined()) {   // contiguous like the kernel's, whatever gz's and z's strides
    auto dz = at::empty(z.sizes(), z.options());
    if (have_z) dz.copy_(*gz);
    else dz.zero_();
    return {dz, at::zeros(w.sizes(), w.options())};
  }
  TORCH_CHECK(gy->sizes() == z.sizes(), "add_rmsnorm_bwd: gy must match z");
  auto zc = packed(z), wc = packed(w), rc = rstd.contiguous();
  auto g = packed(gy->to(z.scalar_type()));
  at::Tensor g2 = have_z ? packed(gz->to(z.scalar_type())) : at::Tensor();
  for (const at::Tensor* t : {&g, &wc, &rc}) check_same_device(z, *t, "add_rmsnorm_bwd");
  if (have_z) check_same_device(z, g2, "add_rmsnorm_bwd");
  const int64_t rows = zc.size(0), n = zc.size(1);
  auto dz = at::empty({rows, n}, zc.options());
  auto dw = at::empty({n}, wc.options());
  size_t ws = 0;
  check_rc(krsi_add_rmsnorm_bwd_workspace_size(rows, n, &ws), "krsi_add_rmsnorm_bwd_workspace_size");
  auto wsp = workspace(zc, ws);
  check_rc(krsi_add_rmsnorm_bwd(g.data_ptr(), have_z ? g2.data_ptr() : nullptr, zc.data_ptr(), wc.data_ptr(),
                                rc.data_ptr<float>(), dz.data_ptr(), dw.data_ptr(), wsp.data_ptr(),
                                (size_t)wsp.numel(), rows, n, krsi_dtype_of(zc), krsi_dtype_of(wc),
                                at::cuda::getCurrentCUDAStream()),
           "krsi_add_rmsnorm_bwd");
  return {dz, dw};
}

// Rows of 8-bit values, each row padded to whole 16 bytes (what a TMA copy of them needs).
at::Tensor empty_q8(int64_t rows, int64_t n, const at::Tensor& like) {
  auto q = at::empty({rows, (n + 15) / 16 * 16}, like.options().dtype(at::kFloat8_e4m3fn));
  return q.size(1) == n ? q : q.narrow(1, 0, n);
}

// (q, scale, z): z is empty where there is no res.
std::tuple<at::Tensor, at::Tensor, at::Tensor> add_rmsnorm_q8(const at::Tensor& x_in,
                                                              const c10::optional<at::Tensor>& res_in,
                                                              const at::Tensor& w_in, double eps) {
  TORCH_CHECK(x_in.is_cuda(), "krsi: x2d must be a CUDA tensor");
  c10::cuda::CUDAGuard guard(x_in.device());
  const NormCall c = norm_call(x_in, res_in, w_in, "add_rmsnorm_q8");
  const int64_t rows = c.x.size(0), n = c.x.size(1);
  auto q = empty_q8(rows, n, c.x);
  auto z = at::empty({c.res.defined() ? rows : 0, n}, c.x.options());
  auto scale = at::empty({rows}, c.x.options().dtype(at::kFloat));
  check_rc(krsi_add_rmsnorm_q8_fwd(c.x.data_ptr(), c.res.defined() ? c.res.data_ptr() : nullptr, c.w.data_ptr(),
                                   c.res.defined() ? z.data_ptr() : nullptr, q.data_ptr(), (n + 15) / 16 * 16,
                                   scale.data_ptr<float>(), rows, n, (float)eps, krsi_dtype_of(c.x), krsi_dtype_of(c.w),
                                   at::cuda::getCurrentCUDAStream()),
           "krsi_add_rmsnorm_q8_fwd");
  return {q, scale, z};
}

std::tuple<at::Tensor, at::Tensor> quantise_rows(const at::Tensor& x_in) {
  check_cuda(x_in, "x2d");
  TORCH_CHECK(x_in.dim() == 2, "quantise: x2d must be 2-D, got ", x_in.dim(), "-D");
  c10::cuda::CUDAGuard guard(x_in.device());
  auto x = packed(x_in);
  const int64_t rows = x.size(0), n = x.size(1);
  auto q = empty_q8(rows, n, x);
  auto scale = at::empty({rows}, x.options().dtype(at::kFloat));
  check_rc(krsi_quantise_rows(x.data_ptr(), q.data_ptr(), (n + 15) / 16 * 16, scale.data_ptr<float>(), rows, n,
                              krsi_dtype_of(x), at::cuda::getCurrentCUDAStream()),
           "krsi_quantise_rows");
  return {q, scale};
}

// ---------------------------------------------------------------- product in 8 bits
at::Tensor linear_q8(const at::Tensor& q_in, const at::Tensor& scale_in, const at::Tensor& wq_in,
                     const at::Tensor& wscale_in, at::ScalarType out_dtype) {
  check_cuda(q_in, "q");
  for (const at::Tensor* t : {&scale_in, &wq_in, &wscale_in}) check_same_device(q_in, *t, "linear_q8");
  TORCH_CHECK(q_in.dim() == 2 && wq_in.dim() == 2 && q_in.size(1) == wq_in.size(1) && q_in.size(1) > 0 &&
                  wq_in.size(0) > 0,
              "linear_q8: q must be [rows, K] and wq [M, K], got ", q_in.sizes(), " and ", wq_in.sizes());
  TORCH_CHECK(q_in.scalar_type() == at::kFloat8_e4m3fn && wq_in.scalar_type() == at::kFloat8_e4m3fn,
              "linear_q8: q and wq must be float8_e4m3fn");
  TORCH_CHECK(scale_in.scalar_type() == at::kFloat && scale_in.dim() == 1 && scale_in.size(0) == q_in.size(0),
              "linear_q8: scale must be float32 [", q_in.size(0), "]");
  TORCH_CHECK(wscale_in.scalar_type() == at::kFloat && wscale_in.dim() == 1 && wscale_in.size(0) == wq_in.size(0),
              "linear_q8: wscale must be float32 [", wq_in.size(0), "]");
  c10::cuda::CUDAGuard guard(q_in.device());
  const int64_t K = q_in.size(1), pitch = (K + 15) / 16 * 16;
  // rows on 16 bytes; others are copied
  auto rows_of = [&](const at::Tensor& t, int64_t* stride) {
    const bool one = t.size(0) <= 1;
    if (t.stride(1) == 1 && (one || (t.stride(0) >= K && t.stride(0) % 16 == 0)) &&
        (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0) {
      *stride = one ? pitch : t.stride(0);
      return t;
    }
    auto c = empty_q8(t.size(0), K, t);
    c.copy_(t);
    *stride = pitch;
    return c;
  };
  int64_t qs = 0, ws = 0;
  auto q = rows_of(q_in, &qs), wq = rows_of(wq_in, &ws);
  auto scale = scale_in.contiguous(), wscale = wscale_in.contiguous();
  auto out = at::empty({q.size(0), wq.size(0)}, q.options().dtype(out_dtype));
  check_rc(krsi_linear_q8(q.data_ptr(), qs, scale.data_ptr<float>(), wq.data_ptr(), ws, wscale.data_ptr<float>(),
                          out.data_ptr(), q.size(0), K, wq.size(0), krsi_dtype_of(out),
                          at::cuda::getCurrentCUDAStream()),
           "krsi_linear_q8");
  return out;
}

// ---------------------------------------------------------------- AdamW
// One step for every tensor, in place; returns the norm of all gradients (empty where max_norm is 0).  masters and
// exponents: a tensor for each parameter, one without elements where it has none, or an empty list.  random_m: of the 8-bit
// states, m's codes at random too.
at::Tensor adamw_step(at::TensorList params, at::TensorList grads, at::TensorList exp_avgs, at::TensorList exp_avg_sqs,
                      at::TensorList masters, at::TensorList exponents, const at::Tensor& step,
                      const c10::optional<at::Tensor>& lr_tensor, double lr, double beta1, double beta2, double eps,
                      double weight_decay, double max_norm, bool random_m) {
  const size_t count = params.size();
  TORCH_CHECK(grads.size() == count && exp_avgs.size() == count && exp_avg_sqs.size() == count,
              "adamw_step: as many grads, exp_avgs and exp_avg_sqs as params are needed");
  TORCH_CHECK(masters.empty() || masters.size() == count, "adamw_step: as many masters as params are needed, or none");
  TORCH_CHECK(exponents.empty() || exponents.size() == count,
              "adamw_step: as many exponents as params are needed, or none");
  TORCH_CHECK(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, "adamw_step: betas must be in [0, 1)");
  TORCH_CHECK(eps >= 0 && max_norm >= 0, "adamw_step: eps and max_norm must not be negative");
  check_cuda(step, "step");
  TORCH_CHECK(step.scalar_type() == at::kLong && step.numel() == 1, "adamw_step: step must be one int64");
  const bool device_lr = lr_tensor.has_value() && lr_tensor->defined();
  if (device_lr)
    TORCH_CHECK(lr_tensor->scalar_type() == at::kFloat && lr_tensor->numel() == 1 &&
                    lr_tensor->device() == step.device(),
                "adamw_step: a tensor lr must be one float32 on the step's device");
  c10::cuda::CUDAGuard guard(step.device());
  std::vector<krsi_adamw_tensor> table(count);
  std::vector<at::Tensor> copies;   // gradients that were not contiguous, until the launch
  std::vector<std::pair<uintptr_t, uintptr_t>> spans;   // no tensor may be updated twice
  spans.reserve(count);
  auto own = [&](const at::Tensor& t, const at::Tensor& p, at::ScalarType type, const char* what) {
    TORCH_CHECK(t.device() == step.device() && t.scalar_type() == type && t.numel() == p.numel() && t.is_contiguous(),
                "adamw_step: ", what, " must be contiguous ", type, " of the parameter's size on the step's device");
  };
  for (size_t i = 0; i < count; ++i) {
    const at::Tensor& p = params[i];
    TORCH_CHECK(p.device() == step.device(), "adamw_step: parameters and step must be on one CUDA device");
    TORCH_CHECK(p.is_contiguous(), "adamw_step: parameters must be contiguous");
    TORCH_CHECK(grads[i].layout() == at::kStrided, "adamw_step: gradients must be dense");
    TORCH_CHECK(grads[i].device() == p.device() && grads[i].sizes() == p.sizes(),
                "adamw_step: a gradient must have its parameter's shape and device");
    krsi_adamw_tensor& t = table[i];
    t = krsi_adamw_tensor{};
    t.n = p.numel();
    t.p_dtype = krsi_dtype_of(p);
    t.g_dtype = krsi_dtype_of(grads[i]);
    TORCH_CHECK(t.g_dtype == t.p_dtype || t.g_dtype == KRSI_F32,
                "adamw_step: a gradient must have its parameter's dtype or float32");
    const bool q8 = exp_avgs[i].scalar_type() == at::kFloat8_e4m3fn;
    t.state_bits = !q8 ? 32 : random_m ? 8 + KRSI_ADAMW_RANDOM_M : 8;
    own(exp_avgs[i], p, q8 ? at::kFloat8_e4m3fn : at::kFloat, "exp_avgs");
    own(exp_avg_sqs[i], p, q8 ? at::kFloat8_e4m3fn : at::kFloat, "exp_avg_sqs");
    t.p = p.data_ptr();
    t.m = exp_avgs[i].data_ptr();
    t.v = exp_avg_sqs[i].data_ptr();
    if (grads[i].is_contiguous()) {
      t.g = grads[i].data_ptr();
    } else {
      copies.push_back(grads[i].contiguous());
      t.g = copies.back().data_ptr();
    }
    if (!masters.empty() && masters[i].numel() > 0) {
      TORCH_CHECK(p.scalar_type() != at::kFloat, "adamw_step: a float32 parameter has no master");
      own(masters[i], p, at::kFloat, "masters");
      t.master = masters[i].data_ptr<float>();
    } else {
      TORCH_CHECK(masters.empty() || t.n == 0 || p.scalar_type() == at::kFloat || masters[i].dim() == 1,
                  "adamw_step: masters must have their parameters' size, or no elements");
    }
    if (q8 && t.n > 0) {
      TORCH_CHECK(!exponents.empty(), "adamw_step: 8-bit states need exponents");
      const at::Tensor& e = exponents[i];
      TORCH_CHECK(e.device() == step.device() && e.scalar_type() == at::kByte && e.is_contiguous() &&
                      e.numel() == 2 * ((t.n + 255) / 256),
                  "adamw_step: exponents must be contiguous uint8 [ceil(n / 256), 2]");
      t.exponents = e.data_ptr<uint8_t>();
    }
    if (t.n > 0) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(t.p);
      spans.emplace_back(at, at + (uintptr_t)p.nbytes());
    }
  }
  if (!std::is_sorted(spans.begin(), spans.end())) std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    TORCH_CHECK(spans[i].first >= spans[i - 1].second, "adamw_step: two parameters share memory");
  auto norm = at::empty(max_norm > 0 ? at::IntArrayRef{} : at::IntArrayRef{0}, step.options().dtype(at::kFloat));
  size_t ws = 0;
  check_rc(krsi_adamw_workspace_size((int64_t)count, &ws), "krsi_adamw_workspace_size");
  auto wsp = workspace(step, ws);
  check_rc(krsi_adamw_step(table.data(), (int64_t)count, step.data_ptr<int64_t>(),
                           device_lr ? lr_tensor->data_ptr<float>() : nullptr, lr, beta1, beta2, eps, weight_decay,
                           max_norm, max_norm > 0 ? norm.data_ptr<float>() : nullptr, wsp.data_ptr(),
                           (size_t)wsp.numel(), at::cuda::getCurrentCUDAStream()),
           "krsi_adamw_step");
  // what was written counts as changed in place (a graph that still needs the old values is told so)
  auto bump = [](at::TensorList l) {
    for (const at::Tensor& t : l)
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  };
  for (const at::TensorList& l : {params, exp_avgs, exp_avg_sqs, masters, exponents}) bump(l);
  if (!step.is_inference()) step.unsafeGetTensorImpl()->bump_version();
  return norm;
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

// (y, z): z is x2d itself where there is no res.
std::tuple<at::Tensor, at::Tensor> add_rmsnorm_plain(const at::Tensor& x, const c10::optional<at::Tensor>& res,
                                                     const at::Tensor& w, double eps) {
  auto [y, z, rstd] = KRSI_OP(add_rmsnorm_fwd).call(x, res, w, eps);
  return {y, res.has_value() && res->defined() ? z : x.alias()};
}
struct AddRmsnormNode : public torch::autograd::Function<AddRmsnormNode> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const c10::optional<at::Tensor>& res,
                               const at::Tensor& w, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [y, z, rstd] = KRSI_OP(add_rmsnorm_fwd).call(x, res, w, eps);
    const bool add = res.has_value() && res->defined();
    if (!add) z = x;
    ctx->save_for_backward({z, w, rstd});
    ctx->saved_data["add"] = add;
    ctx->set_materialize_grads(false);
    return {y, z};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_once("add_rmsnorm");
    const auto saved = ctx->get_saved_variables();
    const bool add = ctx->saved_data["add"].toBool();
    if (!g[0].defined()) return {g[1], add ? g[1] : at::Tensor(), at::Tensor(), at::Tensor()};   // (z's alone, or none)
    at::AutoDispatchBelowADInplaceOrView below;
    auto opt = [](const at::Tensor& t) { return t.defined() ? c10::optional<at::Tensor>(t) : c10::nullopt; };
    auto [dz, dw] = KRSI_OP(add_rmsnorm_bwd).call(g[0], opt(g[1]), saved[0], saved[1], saved[2]);
    return {dz, add ? dz : at::Tensor(), dw, at::Tensor()};
  }
};
std::tuple<at::Tensor, at::Tensor> add_rmsnorm_autograd(const at::Tensor& x, const c10::optional<at::Tensor>& res,
                                                        const at::Tensor& w, double eps) {
  const bool add = res.has_value() && res->defined();
  check_no_tangent({&x, &w}, "add_rmsnorm");
  if (add) check_no_tangent({&*res}, "add_rmsnorm");
  if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || (add && res->requires_grad()))) {
    auto out = AddRmsnormNode::apply(x, res, w, eps);
    return {out[0], out[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return add_rmsnorm_plain(x, res, w, eps);
}

// 8 bits carry no gradient: where one would be asked for, it is refused rather than lost.
void check_no_grad(std::initializer_list<const at::Tensor*> inputs, const char* what) {
  check_no_tangent(inputs, what);
  if (!at::GradMode::is_enabled()) return;
  for (const at::Tensor* t : inputs)
    TORCH_CHECK(!t->requires_grad(), what, ": has no gradient; call it under torch.no_grad()");
}
std::tuple<at::Tensor, at::Tensor, at::Tensor> add_rmsnorm_q8_autograd(const at::Tensor& x,
                                                                       const c10::optional<at::Tensor>& res,
                                                                       const at::Tensor& w, double eps) {
  check_no_grad({&x, &w}, "add_rmsnorm_q8");
  if (res.has_value() && res->defined()) check_no_grad({&*res}, "add_rmsnorm_q8");
  at::AutoDispatchBelowADInplaceOrView below;
  return KRSI_OP(add_rmsnorm_q8).call(x, res, w, eps);
}
std::tuple<at::Tensor, at::Tensor> quantise_rows_autograd(const at::Tensor& x) {
  check_no_grad({&x}, "quantise");
  at::AutoDispatchBelowADInplaceOrView below;
  return KRSI_OP(quantise_rows).call(x);
}
at::Tensor linear_q8_autograd(const at::Tensor& q, const at::Tensor& scale, const at::Tensor& wq,
                              const at::Tensor& wscale, at::ScalarType out_dtype) {
  check_no_grad({&q, &scale, &wq, &wscale}, "linear_q8");
  at::AutoDispatchBelowADInplaceOrView below;
  return KRSI_OP(linear_q8).call(q, scale, wq, wscale, out_dtype);
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
  m.def("add_rmsnorm(Tensor x2d, Tensor? res, Tensor w, float eps) -> (Tensor, Tensor)");
  m.def("add_rmsnorm_fwd(Tensor x2d, Tensor? res, Tensor w, float eps) -> (Tensor, Tensor, Tensor)");
  m.def("add_rmsnorm_bwd(Tensor? gy, Tensor? gz, Tensor z, Tensor w, Tensor rstd) -> (Tensor, Tensor)");
  m.def("add_rmsnorm_q8(Tensor x2d, Tensor? res, Tensor w, float eps) -> (Tensor, Tensor, Tensor)");
  m.def("quantise_rows(Tensor x2d) -> (Tensor, Tensor)");
  m.def("linear_q8(Tensor q, Tensor scale, Tensor wq, Tensor wscale, ScalarType out_dtype) -> Tensor");
  m.def("adamw_step(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] exp_avgs, Tensor(c!)[] exp_avg_sqs, "
        "Tensor(d!)[] masters, Tensor(e!)[] exponents, Tensor(f!) step, Tensor? lr_tensor, float lr, float beta1, "
        "float beta2, float eps, float weight_decay, float max_norm, bool random_m=False) -> Tensor");
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
  m.impl("add_rmsnorm", &add_rmsnorm_plain);
  m.impl("add_rmsnorm_fwd", &add_rmsnorm_fwd);
  m.impl("add_rmsnorm_bwd", &add_rmsnorm_bwd);
  m.impl("add_rmsnorm_q8", &add_rmsnorm_q8);
  m.impl("quantise_rows", &quantise_rows);
  m.impl("linear_q8", &linear_q8);
  m.impl("adamw_step", &adamw_step);
}

// ---------------------------------------------------------------- Python lists
// adamw_step from Python lists as they are.  An operator's list arguments are boxed and unboxed tensor by tensor on the
// way, which for a model's lists is most of a step's time on the host (0.5 us a tensor; this takes a quarter).  What
// only the dispatcher can see to, a mode that is on or a tensor that is not torch's own, is left to the operator: the
// answer is then NotImplemented.
namespace {

bool unpack(PyObject* list, std::vector<at::Tensor>& out) {
  if (!PyList_CheckExact(list) && !PyTuple_CheckExact(list)) return false;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(list);
  PyObject** items = PySequence_Fast_ITEMS(list);
  out.reserve(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (!THPVariable_CheckExact(items[i])) return false;
    out.push_back(THPVariable_Unpack(items[i]));
  }
  return true;
}

PyObject* py_adamw_step(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 14 && nargs != 15)
    return PyErr_Format(PyExc_TypeError, "adamw_step: 14 or 15 arguments expected, got %zd", nargs);
  const bool modes = c10::impl::TorchDispatchModeTLS::any_modes_set() ||
                     at::impl::PythonTorchFunctionTLS::stack_len() > 0;
  std::vector<at::Tensor> lists[6];
  bool ok = !modes && THPVariable_CheckExact(args[6]) && (args[7] == Py_None || THPVariable_CheckExact(args[7]));
  for (int k = 0; ok && k < 6; ++k) ok = unpack(args[k], lists[k]);
  // (the operator's own refusals where there is no CUDA tensor)
  ok = ok && THPVariable_Unpack(args[6]).is_cuda();
  for (int k = 0; ok && k < 4; ++k)
    for (const at::Tensor& t : lists[k]) ok = ok && t.is_cuda();
  if (!ok) Py_RETURN_NOTIMPLEMENTED;
  double number[6];
  for (int k = 0; k < 6; ++k) {
    number[k] = PyFloat_AsDouble(args[8 + k]);
    if (number[k] == -1.0 && PyErr_Occurred()) return nullptr;
  }
  const int random_m = nargs == 15 ? PyObject_IsTrue(args[14]) : 0;
  if (random_m < 0) return nullptr;
  const at::Tensor step = THPVariable_Unpack(args[6]);
  const c10::optional<at::Tensor> lr =
      args[7] == Py_None ? c10::nullopt : c10::optional<at::Tensor>(THPVariable_Unpack(args[7]));
  at::Tensor norm;
  {
    pybind11::gil_scoped_release release;
    at::AutoDispatchBelowADInplaceOrView below;
    norm = adamw_step(lists[0], lists[1], lists[2], lists[3], lists[4], lists[5], step, lr, number[0], number[1],
                      number[2], number[3], number[4], number[5], random_m != 0);
  }
  return THPVariable_Wrap(std::move(norm));
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"adamw_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&py_adamw_step)),
                          METH_FASTCALL, "torch.ops.krsi.adamw_step on Python lists, or NotImplemented"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_krsi_torch", nullptr, -1, methods};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__krsi_torch() { return PyModule_Create(&module); }

TORCH_LIBRARY_IMPL(krsi, AutogradCUDA, m) {
  m.impl("embedding", &embedding_autograd);
  m.impl("geglu_q8", &geglu_q8_autograd);
  m.impl("linear_ce", &linear_ce_autograd);
  m.impl("add_rmsnorm", &add_rmsnorm_autograd);
  m.impl("add_rmsnorm_q8", &add_rmsnorm_q8_autograd);
  m.impl("quantise_rows", &quantise_rows_autograd);
  m.impl("linear_q8", &linear_q8_autograd);
  m.impl("adamw_step", torch::CppFunction::makeFallthrough());   // an update is no part of a graph
}
