// PyTorch-ROCm bindings for the LuminaAI-AMD HIP kernels (gfx950).
// Host-side code only; kernels live in the *.hip translation units and are
// reached through extern "C" launchers taking hipStream_t.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <c10/hip/HIPStream.h>
#include <c10/core/DeviceGuard.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <optional>
#include <tuple>
#include <utility>
#include <vector>

namespace {

hipStream_t cur_stream() {
  return c10::hip::getCurrentHIPStream().stream();
}

void check_hip(hipError_t e, const char* what) {
  TORCH_CHECK(e == hipSuccess, what, " failed: ", hipGetErrorString(e));
}

bool is_bf16(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16; }

void check_dtype(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat,
              name, " must be bf16 or fp32, got ", t.scalar_type());
}

}  // namespace

// ---- launchers from the .hip TUs ----------------------------------------
extern "C" {
hipError_t lumina_attn_fwd(const void*, const void*, const void*, void*, void*, int, int, int, int, int, int, float, hipStream_t);
hipError_t lumina_attn_delta(const void*, const void*, void*, int64_t, int, int, int, hipStream_t);
hipError_t lumina_attn_bwd(const void*, const void*, const void*, const void*, const void*, const void*, void*, void*, void*, int, int, int, int, int, int, float, hipStream_t);
hipError_t lumina_rmsnorm_fwd_bf16(const void*, const void*, void*, float*, int64_t, int, float, hipStream_t);
hipError_t lumina_rmsnorm_fwd_f32(const void*, const void*, void*, float*, int64_t, int, float, hipStream_t);
hipError_t lumina_rmsnorm_bwd_bf16(const void*, const void*, const void*, const float*, void*, float*, int64_t, int, hipStream_t);
hipError_t lumina_rmsnorm_bwd_f32(const void*, const void*, const void*, const float*, void*, float*, int64_t, int, hipStream_t);
hipError_t lumina_rope_bf16(const void*, const void*, void*, void*, const float*, const float*, const int*, int64_t, int, int, int, int, int, int, hipStream_t);
hipError_t lumina_rope_f32(const void*, const void*, void*, void*, const float*, const float*, const int*, int64_t, int, int, int, int, int, int, hipStream_t);
hipError_t lumina_swiglu_fwd_bf16(const void*, const void*, void*, int64_t, int, int64_t, int64_t, hipStream_t);
hipError_t lumina_swiglu_fwd_f32(const void*, const void*, void*, int64_t, int, int64_t, int64_t, hipStream_t);
hipError_t lumina_swiglu_bwd_bf16(const void*, const void*, const void*, void*, void*, int64_t, int, int64_t, int64_t, hipStream_t);
hipError_t lumina_swiglu_bwd_f32(const void*, const void*, const void*, void*, void*, int64_t, int, int64_t, int64_t, hipStream_t);
hipError_t lumina_ce_fwd_bf16(const void*, const int32_t*, const float*, float*, float*, int64_t, int, int, hipStream_t);
hipError_t lumina_ce_fwd_f32(const void*, const int32_t*, const float*, float*, float*, int64_t, int, int, hipStream_t);
hipError_t lumina_ce_bwd_bf16(const void*, const int32_t*, const float*, const float*, const float*, const float*, void*, int64_t, int, int, hipStream_t);
hipError_t lumina_ce_bwd_f32(const void*, const int32_t*, const float*, const float*, const float*, const float*, void*, int64_t, int, int, hipStream_t);
hipError_t lumina_l2norm_sq_bf16(const void*, int64_t, float*, hipStream_t);
hipError_t lumina_l2norm_sq_f32(const void*, int64_t, float*, hipStream_t);
hipError_t lumina_adamw_step(float*, const void*, int, float*, float*, void*, int, int64_t, float, float, float, float, float, float, float, const float*, float, float, hipStream_t);
void launch_grouped_gemm_nt(const void*, const void*, void*, int, int, int, int, int64_t, int64_t, int64_t, hipStream_t);
void launch_gg8p(const void*, const void*, void*, int, int, int, int, int, int64_t, int64_t, int64_t, int, hipStream_t);
hipError_t lumina_mx_quant_rows(const void*, void*, void*, int64_t, int, int, hipStream_t);
hipError_t lumina_mx_quant_cols(const void*, void*, void*, void*, int, int, int, int, hipStream_t);
hipError_t lumina_gg_mx_nt(const void*, const void*, const void*, const void*, void*, int, int, int, int, int64_t, int64_t, int64_t, hipStream_t);
void launch_grouped_gemm_nt_v2(const void*, const void*, void*, int, int, int, int, int64_t, int64_t, int64_t, int, hipStream_t);
void launch_grouped_gemm_nt_v3(const void*, const void*, void*, int, int, int, int, int64_t, int64_t, int64_t, hipStream_t);
void launch_grouped_gemm_nt_v4(const void*, const void*, void*, int, int, int, int, int64_t, int64_t, int64_t, hipStream_t);
hipError_t lumina_gemv(const void*, const void*, void*, int, int64_t, int, hipStream_t);
hipError_t lumina_dec_gemv(const void*, const void*, const void*, const void*, void*, int, int, float, int, hipStream_t);
hipError_t lumina_dec_rope_cache(const void*, void*, void*, void*, const float*, const float*, const int*, int, int, int, hipStream_t);
hipError_t lumina_dec_attn(const void*, const void*, const void*, void*, const int*, int, int, int, int, float, hipStream_t);
hipError_t lumina_dec_advance(int*, hipStream_t);
hipError_t lumina_gg8t_nt(const void*, const void*, void*, int, int, int, int, int64_t, int64_t, int64_t, int, hipStream_t);
hipError_t lumina_dec_rmsnorm(const void*, const void*, void*, int, float, hipStream_t);
hipError_t lumina_dec_topk(const void*, int*, float*, int, int, float, hipStream_t);
hipError_t lumina_dec_router(const void*, const void*, const void*, void*, int*, float*, int, int, int, float, float, hipStream_t);
hipError_t lumina_dec_gemv_moe(const void*, const void*, const void*, void*, const int*, const float*, int, int64_t, int, int, int, hipStream_t);
hipError_t lumina_moe_gather_rows(const void*, const int64_t*, const bool*, void*, int64_t, int, int, hipStream_t);
hipError_t lumina_moe_dispatch_bwd(const void*, const int64_t*, void*, int64_t, int, int, int64_t, int, hipStream_t);
hipError_t lumina_moe_combine_fwd(const void*, const float*, const int64_t*, void*, int64_t, int, int, int64_t, int, hipStream_t);
hipError_t lumina_moe_combine_bwd_y(const void*, const float*, const int64_t*, const int64_t*, const bool*, void*, int64_t, int64_t, int, int, hipStream_t);
hipError_t lumina_moe_combine_bwd_w(const void*, const void*, const int64_t*, float*, int64_t, int, int, int64_t, int, hipStream_t);
hipError_t lumina_packed_attn_fwd(const void*, const void*, const void*, void*, void*, float*, const int*, int*, const int64_t*, int, int, int, int, int, int, float, hipStream_t);
hipError_t lumina_packed_attn_bwd(const void*, const void*, const void*, const void*, const void*, const void*, const float*, float*, void*, void*, void*, float*, int, const int*, int*, const int64_t*, int, int, int, int, int, int, float, hipStream_t);
hipError_t lumina_pack_rows(const void* const*, void* const*, const int64_t*, const int*, int, int64_t, int, hipStream_t);
hipError_t lumina_paged_attn(const void*, const void*, const void*, void*, const int*, const int*, float*, float*, int*, int*, const int64_t*, int64_t, int, int, int, int, int, int, int, int, int, int, float, hipStream_t);
hipError_t lumina_paged_append(const void*, const void*, void*, void*, const int*, const int*, const int*, const int64_t*, int64_t, int64_t, int, int, int, int, int, int, int, hipStream_t);
hipError_t lumina_copy_pages(void* const*, int, const int64_t*, const int64_t*, int, int64_t, const int*, const int*, int64_t, hipStream_t);
hipError_t lumina_logprob_fwd(const void*, int, const void*, int, float*, float*, float*, float*, int64_t*, int64_t, int, int64_t, int, int64_t, hipStream_t);
hipError_t lumina_logprob_bwd(const void*, int, const void*, int, const float*, const float*, const float*, const float*, void*, int64_t, int, int64_t, int64_t, hipStream_t);
}

// ---- RMSNorm -------------------------------------------------------------
std::tuple<at::Tensor, at::Tensor> rmsnorm_fwd(const at::Tensor& x,
                                               const at::Tensor& w,
                                               double eps, bool save_inv) {
  TORCH_CHECK(x.is_contiguous() && w.is_contiguous());
  check_dtype(x, "x");
  TORCH_CHECK(x.scalar_type() == w.scalar_type(), "x/w dtype mismatch");
  const int H = (int)x.size(-1);
  const int64_t N = x.numel() / H;
  auto y = at::empty_like(x);
  auto inv = save_inv
      ? at::empty({N}, x.options().dtype(at::kFloat))
      : at::Tensor();
  float* invp = save_inv ? inv.data_ptr<float>() : nullptr;
  if (is_bf16(x))
    check_hip(lumina_rmsnorm_fwd_bf16(x.data_ptr(), w.data_ptr(), y.data_ptr(),
                                      invp, N, H, (float)eps, cur_stream()),
              "rmsnorm_fwd_bf16");
  else
    check_hip(lumina_rmsnorm_fwd_f32(x.data_ptr(), w.data_ptr(), y.data_ptr(),
                                     invp, N, H, (float)eps, cur_stream()),
              "rmsnorm_fwd_f32");
  return {y, inv};
}

std::tuple<at::Tensor, at::Tensor> rmsnorm_bwd(const at::Tensor& gy,
                                               const at::Tensor& x,
                                               const at::Tensor& w,
                                               const at::Tensor& inv) {
  TORCH_CHECK(gy.is_contiguous() && x.is_contiguous() && w.is_contiguous());
  const int H = (int)x.size(-1);
  const int64_t N = x.numel() / H;
  auto dx = at::empty_like(x);
  auto dw = at::zeros({H}, x.options().dtype(at::kFloat));
  if (is_bf16(x))
    check_hip(lumina_rmsnorm_bwd_bf16(gy.data_ptr(), x.data_ptr(), w.data_ptr(),
                                      inv.data_ptr<float>(), dx.data_ptr(),
                                      dw.data_ptr<float>(), N, H, cur_stream()),
              "rmsnorm_bwd_bf16");
  else
    check_hip(lumina_rmsnorm_bwd_f32(gy.data_ptr(), x.data_ptr(), w.data_ptr(),
                                     inv.data_ptr<float>(), dx.data_ptr(),
                                     dw.data_ptr<float>(), N, H, cur_stream()),
              "rmsnorm_bwd_f32");
  return {dx, dw};
}

// ---- RoPE ----------------------------------------------------------------
// q: [B, S, Hq, D], k: [B, S, Hk, D] contiguous; cos/sin: [S_cache, D/2] fp32.
std::tuple<at::Tensor, at::Tensor> rope_fwd(const at::Tensor& q,
                                            const at::Tensor& k,
                                            const at::Tensor& cos_t,
                                            const at::Tensor& sin_t,
                                            const std::optional<at::Tensor>& pos,
                                            int64_t pos_offset, bool conj) {
  TORCH_CHECK(q.is_contiguous() && k.is_contiguous());
  TORCH_CHECK(cos_t.is_contiguous() && sin_t.is_contiguous());
  TORCH_CHECK(cos_t.scalar_type() == at::kFloat && sin_t.scalar_type() == at::kFloat);
  check_dtype(q, "q");
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4);
  const int64_t B = q.size(0);
  const int S = (int)q.size(1), Hq = (int)q.size(2), Hk = (int)k.size(2);
  const int D = (int)q.size(3);
  TORCH_CHECK(k.size(0) == B && k.size(1) == S && k.size(3) == D);
  TORCH_CHECK(cos_t.size(1) == D / 2);
  const int* posp = nullptr;
  if (pos.has_value()) {
    TORCH_CHECK(pos->scalar_type() == at::kInt && pos->is_contiguous());
    TORCH_CHECK(pos->numel() == B * S);
    posp = pos->data_ptr<int>();
  }
  auto oq = at::empty_like(q);
  auto ok = at::empty_like(k);
  if (is_bf16(q))
    check_hip(lumina_rope_bf16(q.data_ptr(), k.data_ptr(), oq.data_ptr(),
                               ok.data_ptr(), cos_t.data_ptr<float>(),
                               sin_t.data_ptr<float>(), posp, B, S, Hq, Hk, D,
                               (int)pos_offset, conj ? 1 : 0, cur_stream()),
              "rope_bf16");
  else
    check_hip(lumina_rope_f32(q.data_ptr(), k.data_ptr(), oq.data_ptr(),
                              ok.data_ptr(), cos_t.data_ptr<float>(),
                              sin_t.data_ptr<float>(), posp, B, S, Hq, Hk, D,
                              (int)pos_offset, conj ? 1 : 0, cur_stream()),
              "rope_f32");
  return {oq, ok};
}

// ---- SwiGLU ---------------------------------------------------------------
// g, u: [rows, I] views into the fused gate_up output (row stride may exceed I).
at::Tensor swiglu_fwd(const at::Tensor& g, const at::Tensor& u) {
  check_dtype(g, "gate");
  TORCH_CHECK(g.dim() == 2 && u.dim() == 2 && g.sizes() == u.sizes());
  TORCH_CHECK(g.stride(1) == 1 && u.stride(1) == 1, "inner dim must be contiguous");
  const int64_t rows = g.size(0);
  const int I = (int)g.size(1);
  auto y = at::empty({rows, I}, g.options());
  auto fn = is_bf16(g) ? lumina_swiglu_fwd_bf16 : lumina_swiglu_fwd_f32;
  check_hip(fn(g.data_ptr(), u.data_ptr(), y.data_ptr(), rows, I,
               g.stride(0), u.stride(0), cur_stream()), "swiglu_fwd");
  return y;
}

std::tuple<at::Tensor, at::Tensor> swiglu_bwd(const at::Tensor& dy,
                                              const at::Tensor& g,
                                              const at::Tensor& u) {
  TORCH_CHECK(dy.is_contiguous());
  TORCH_CHECK(g.stride(1) == 1 && u.stride(1) == 1);
  const int64_t rows = g.size(0);
  const int I = (int)g.size(1);
  // dg/du are allocated as one fused [rows, 2I] buffer when g/u share storage
  // layout, so the caller can feed the downstream GEMM one contiguous tensor.
  at::Tensor dg, du;
  bool fused = (g.stride(0) == 2 * I && u.stride(0) == 2 * I &&
                u.data_ptr() == (char*)g.data_ptr() + I * g.element_size());
  if (fused) {
    auto dgu = at::empty({rows, 2 * I}, g.options());
    dg = dgu.narrow(1, 0, I);
    du = dgu.narrow(1, I, I);
  } else {
    dg = at::empty({rows, I}, g.options());
    du = at::empty({rows, I}, u.options());
  }
  auto fn = is_bf16(g) ? lumina_swiglu_bwd_bf16 : lumina_swiglu_bwd_f32;
  check_hip(fn(dy.data_ptr(), g.data_ptr(), u.data_ptr(), dg.data_ptr(),
               du.data_ptr(), rows, I,
               fused ? 2 * I : I, fused ? 2 * I : I, cur_stream()),
            "swiglu_bwd");
  return {dg, du};
}

at::Tensor swiglu_bwd_fused(const at::Tensor& dy, const at::Tensor& gu) {
  // dy [rows, I], gu [rows, 2I] contiguous -> dgu [rows, 2I].  Taking the
  // FUSED projection output directly keeps autograd away from narrow()
  // slices: the two narrow-backwards cost a zero-fill + two slice copies
  // + a buffer add on [rows, 2I] (measured 6% of the b1 training step).
  TORCH_CHECK(dy.is_contiguous() && gu.is_contiguous());
  TORCH_CHECK(gu.dim() == 2 && dy.dim() == 2);
  const int64_t rows = gu.size(0);
  const int I = (int)(gu.size(1) / 2);
  TORCH_CHECK(dy.size(0) == rows && dy.size(1) == I);
  auto dgu = at::empty_like(gu);
  auto fn = is_bf16(gu) ? lumina_swiglu_bwd_bf16 : lumina_swiglu_bwd_f32;
  const char* g = (const char*)gu.data_ptr();
  char* dg = (char*)dgu.data_ptr();
  const int64_t ib = (int64_t)I * gu.element_size();
  check_hip(fn(dy.data_ptr(), g, g + ib, dg, dg + ib, rows, I,
               2 * (int64_t)I, 2 * (int64_t)I, cur_stream()),
            "swiglu_bwd_fused");
  return dgu;
}

// ---- fused CE ------------------------------------------------------------
std::tuple<at::Tensor, at::Tensor> ce_fwd(const at::Tensor& logits,
                                          const at::Tensor& labels,
                                          const std::optional<at::Tensor>& weights,
                                          int64_t ignore_index) {
  TORCH_CHECK(logits.is_contiguous() && logits.dim() == 2);
  TORCH_CHECK(labels.scalar_type() == at::kInt && labels.is_contiguous());
  check_dtype(logits, "logits");
  const int64_t N = logits.size(0);
  const int V = (int)logits.size(1);
  const float* wp = nullptr;
  if (weights.has_value()) {
    TORCH_CHECK(weights->scalar_type() == at::kFloat && weights->is_contiguous());
    wp = weights->data_ptr<float>();
  }
  auto lse = at::empty({N}, logits.options().dtype(at::kFloat));
  auto stats = at::zeros({4}, logits.options().dtype(at::kFloat));
  auto fn = is_bf16(logits) ? lumina_ce_fwd_bf16 : lumina_ce_fwd_f32;
  check_hip(fn(logits.data_ptr(), labels.data_ptr<int>(), wp,
               lse.data_ptr<float>(), stats.data_ptr<float>(), N, V,
               (int)ignore_index, cur_stream()), "ce_fwd");
  return {lse, stats};
}

at::Tensor ce_bwd(const at::Tensor& logits, const at::Tensor& labels,
                  const std::optional<at::Tensor>& weights,
                  const at::Tensor& lse, const at::Tensor& stats,
                  const at::Tensor& gscale, int64_t ignore_index) {
  const int64_t N = logits.size(0);
  const int V = (int)logits.size(1);
  const float* wp = weights.has_value() ? weights->data_ptr<float>() : nullptr;
  auto dlogits = at::empty_like(logits);
  auto fn = is_bf16(logits) ? lumina_ce_bwd_bf16 : lumina_ce_bwd_f32;
  check_hip(fn(logits.data_ptr(), labels.data_ptr<int>(), wp,
               lse.data_ptr<float>(), stats.data_ptr<float>(),
               gscale.data_ptr<float>(), dlogits.data_ptr(), N, V,
               (int)ignore_index, cur_stream()), "ce_bwd");
  return dlogits;
}

// ---- optimizer -----------------------------------------------------------
at::Tensor l2norm_sq(const at::Tensor& x) {
  TORCH_CHECK(x.is_contiguous());
  check_dtype(x, "x");
  auto out = at::zeros({1}, x.options().dtype(at::kFloat));
  auto fn = is_bf16(x) ? lumina_l2norm_sq_bf16 : lumina_l2norm_sq_f32;
  check_hip(fn(x.data_ptr(), x.numel(), out.data_ptr<float>(), cur_stream()),
            "l2norm_sq");
  return out;
}

void adamw_step(at::Tensor& master, const at::Tensor& grad, at::Tensor& m,
                at::Tensor& v, const std::optional<at::Tensor>& w_out,
                double lr, double beta1, double beta2, double eps, double wd,
                int64_t step, const std::optional<at::Tensor>& gnorm_sq,
                double max_norm, double grad_scale) {
  TORCH_CHECK(master.scalar_type() == at::kFloat && master.is_contiguous());
  TORCH_CHECK(m.scalar_type() == at::kFloat && v.scalar_type() == at::kFloat);
  check_dtype(grad, "grad");
  const int64_t n = master.numel();
  TORCH_CHECK(grad.numel() == n && m.numel() == n && v.numel() == n);
  void* wp = nullptr;
  int w_bf16 = 1;
  if (w_out.has_value()) {
    TORCH_CHECK(w_out->numel() == n && w_out->is_contiguous());
    wp = w_out->data_ptr();
    w_bf16 = is_bf16(*w_out) ? 1 : 0;
  }
  const float* np = gnorm_sq.has_value() ? gnorm_sq->data_ptr<float>() : nullptr;
  const float bias1 = 1.0f / (1.0f - (float)std::pow(beta1, (double)step));
  const float bias2 = 1.0f / (1.0f - (float)std::pow(beta2, (double)step));
  check_hip(lumina_adamw_step(master.data_ptr<float>(), grad.data_ptr(),
                              is_bf16(grad) ? 1 : 0, m.data_ptr<float>(),
                              v.data_ptr<float>(), wp, w_bf16, n, (float)lr,
                              (float)beta1, (float)beta2, (float)eps, (float)wd,
                              bias1, bias2, np, (float)max_norm,
                              (float)grad_scale, cur_stream()),
            "adamw_step");
}

// ---- fused MoE dispatch/combine gathers ----------------------------------
at::Tensor moe_gather_rows(const at::Tensor& x, const at::Tensor& src_tok,
                           const at::Tensor& fill) {
  TORCH_CHECK(x.is_contiguous() && x.dim() == 2);
  const int64_t n_slots = src_tok.numel();
  auto buf = at::empty({n_slots, x.size(1)}, x.options());
  check_hip(lumina_moe_gather_rows(x.data_ptr(), src_tok.data_ptr<int64_t>(),
                                   fill.data_ptr<bool>(), buf.data_ptr(),
                                   n_slots, (int)x.size(1),
                                   is_bf16(x) ? 1 : 0, cur_stream()),
            "moe_gather_rows");
  return buf;
}

at::Tensor moe_dispatch_bwd(const at::Tensor& gbuf, const at::Tensor& slot_tm,
                            int64_t k) {
  TORCH_CHECK(gbuf.is_contiguous() && gbuf.dim() == 2);
  const int64_t n_tok = slot_tm.numel() / k;
  auto gx = at::empty({n_tok, gbuf.size(1)}, gbuf.options());
  check_hip(lumina_moe_dispatch_bwd(gbuf.data_ptr(),
                                    slot_tm.data_ptr<int64_t>(),
                                    gx.data_ptr(), n_tok, (int)k,
                                    (int)gbuf.size(1), gbuf.size(0),
                                    is_bf16(gbuf) ? 1 : 0, cur_stream()),
            "moe_dispatch_bwd");
  return gx;
}

at::Tensor moe_combine_fwd(const at::Tensor& y, const at::Tensor& w_tm,
                           const at::Tensor& slot_tm, int64_t k) {
  TORCH_CHECK(y.is_contiguous() && y.dim() == 2);
  TORCH_CHECK(w_tm.scalar_type() == at::kFloat);
  const int64_t n_tok = slot_tm.numel() / k;
  auto out = at::empty({n_tok, y.size(1)}, y.options());
  check_hip(lumina_moe_combine_fwd(y.data_ptr(), w_tm.data_ptr<float>(),
                                   slot_tm.data_ptr<int64_t>(),
                                   out.data_ptr(), n_tok, (int)k,
                                   (int)y.size(1), y.size(0),
                                   is_bf16(y) ? 1 : 0, cur_stream()),
            "moe_combine_fwd");
  return out;
}

at::Tensor moe_combine_bwd_y(const at::Tensor& gout, const at::Tensor& w_tm,
                             const at::Tensor& inv, const at::Tensor& src_tok,
                             const at::Tensor& fill) {
  TORCH_CHECK(gout.is_contiguous() && gout.dim() == 2);
  const int64_t n_slots = inv.numel();
  auto gy = at::empty({n_slots, gout.size(1)}, gout.options());
  check_hip(lumina_moe_combine_bwd_y(
                gout.data_ptr(), w_tm.data_ptr<float>(),
                inv.data_ptr<int64_t>(), src_tok.data_ptr<int64_t>(),
                fill.data_ptr<bool>(), gy.data_ptr(), n_slots,
                w_tm.numel(), (int)gout.size(1), is_bf16(gout) ? 1 : 0,
                cur_stream()),
            "moe_combine_bwd_y");
  return gy;
}

at::Tensor moe_combine_bwd_w(const at::Tensor& gout, const at::Tensor& y,
                             const at::Tensor& slot_tm, int64_t k) {
  TORCH_CHECK(gout.is_contiguous() && y.is_contiguous());
  const int64_t n_flat = slot_tm.numel();
  auto gw = at::empty({n_flat}, gout.options().dtype(at::kFloat));
  check_hip(lumina_moe_combine_bwd_w(
                gout.data_ptr(), y.data_ptr(), slot_tm.data_ptr<int64_t>(),
                gw.data_ptr<float>(), n_flat, (int)k, (int)gout.size(1),
                y.size(0), is_bf16(gout) ? 1 : 0, cur_stream()),
            "moe_combine_bwd_w");
  return gw;
}

// ---- grouped NT GEMM -----------------------------------------------------
at::Tensor grouped_gemm_nt(const at::Tensor& A, const at::Tensor& B) {
  // out[e] = A[e] @ B[e]^T : A [E,M,K], B [E,N,K] -> out [E,M,N]
  TORCH_CHECK(A.is_contiguous() && B.is_contiguous(),
              "grouped_gemm_nt needs contiguous operands");
  TORCH_CHECK(is_bf16(A) && is_bf16(B), "grouped_gemm_nt is bf16-only");
  TORCH_CHECK(A.dim() == 3 && B.dim() == 3 && A.size(0) == B.size(0)
              && A.size(2) == B.size(2), "shape mismatch");
  const int E = (int)A.size(0), M = (int)A.size(1);
  const int K = (int)A.size(2), N = (int)B.size(1);
  auto O = at::empty({E, M, N}, A.options());
  launch_grouped_gemm_nt(A.data_ptr(), B.data_ptr(), O.data_ptr(),
                         E, M, N, K, (int64_t)M * K, (int64_t)N * K,
                         (int64_t)M * N, cur_stream());
  check_hip(hipGetLastError(), "grouped_gemm_nt");
  return O;
}

at::Tensor grouped_gemm_nt_v2(const at::Tensor& A, const at::Tensor& B,
                              int64_t swz_mode) {
  TORCH_CHECK(A.is_contiguous() && B.is_contiguous());
  TORCH_CHECK(is_bf16(A) && is_bf16(B));
  TORCH_CHECK(A.dim() == 3 && B.dim() == 3 && A.size(2) == B.size(2));
  TORCH_CHECK(A.size(2) % 64 == 0, "v2 kernel requires K % 64 == 0");
  const int E = (int)A.size(0), M = (int)A.size(1);
  const int K = (int)A.size(2), N = (int)B.size(1);
  auto O = at::empty({E, M, N}, A.options());
  launch_grouped_gemm_nt_v2(A.data_ptr(), B.data_ptr(), O.data_ptr(),
                            E, M, N, K, (int64_t)M * K, (int64_t)N * K,
                            (int64_t)M * N, (int)swz_mode, cur_stream());
  check_hip(hipGetLastError(), "grouped_gemm_nt_v2");
  return O;
}

at::Tensor grouped_gemm_nt_v3(const at::Tensor& A, const at::Tensor& B) {
  TORCH_CHECK(A.is_contiguous() && B.is_contiguous());
  TORCH_CHECK(is_bf16(A) && is_bf16(B));
  TORCH_CHECK(A.dim() == 3 && B.dim() == 3 && A.size(2) == B.size(2));
  TORCH_CHECK(A.size(2) % 64 == 0, "v3 kernel requires K % 64 == 0");
  const int E = (int)A.size(0), M = (int)A.size(1);
  const int K = (int)A.size(2), N = (int)B.size(1);
  auto O = at::empty({E, M, N}, A.options());
  launch_grouped_gemm_nt_v3(A.data_ptr(), B.data_ptr(), O.data_ptr(),
                            E, M, N, K, (int64_t)M * K, (int64_t)N * K,
                            (int64_t)M * N, cur_stream());
  check_hip(hipGetLastError(), "grouped_gemm_nt_v3");
  return O;
}

at::Tensor grouped_gemm_nt_v4(const at::Tensor& A, const at::Tensor& B) {
  TORCH_CHECK(A.is_contiguous() && B.is_contiguous());
  TORCH_CHECK(is_bf16(A) && is_bf16(B));
  TORCH_CHECK(A.dim() == 3 && B.dim() == 3 && A.size(2) == B.size(2));
  TORCH_CHECK(A.size(2) % 64 == 0, "v4 kernel requires K % 64 == 0");
  const int E = (int)A.size(0), M = (int)A.size(1);
  const int K = (int)A.size(2), N = (int)B.size(1);
  auto O = at::empty({E, M, N}, A.options());
  launch_grouped_gemm_nt_v4(A.data_ptr(), B.data_ptr(), O.data_ptr(),
                            E, M, N, K, (int64_t)M * K, (int64_t)N * K,
                            (int64_t)M * N, cur_stream());
  check_hip(hipGetLastError(), "grouped_gemm_nt_v4");
  return O;
}

// ---- causal GQA flash attention ------------------------------------------
// q,k,v: [B,H|HKV,S,DP] bf16 contiguous, DP % 32 == 0 (pad channels zero).
std::tuple<at::Tensor, at::Tensor> attn_fwd(const at::Tensor& q,
                                            const at::Tensor& k,
                                            const at::Tensor& v,
                                            double scale) {
  TORCH_CHECK(q.is_contiguous() && k.is_contiguous() && v.is_contiguous());
  TORCH_CHECK(is_bf16(q) && is_bf16(k) && is_bf16(v));
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4);
  const int B = (int)q.size(0), H = (int)q.size(1);
  const int S = (int)q.size(2), DP = (int)q.size(3);
  const int HKV = (int)k.size(1);
  TORCH_CHECK(DP % 32 == 0 && (DP == 64 || DP == 128 || DP == 160),
              "unsupported padded head dim ", DP);
  TORCH_CHECK(H % HKV == 0 && k.size(2) == S && v.size(1) == HKV);
  const int SP = (S + 127) / 128 * 128;
  auto o = at::empty_like(q);
  auto lse2 = at::empty({B, H, SP}, q.options().dtype(at::kFloat));
  check_hip(lumina_attn_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(),
                            o.data_ptr(), lse2.data_ptr(), B, H, HKV, S, SP,
                            DP, (float)scale, cur_stream()),
            "attn_fwd");
  return {o, lse2};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> attn_bwd(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
    const at::Tensor& o, const at::Tensor& do_, const at::Tensor& lse2,
    double scale) {
  TORCH_CHECK(q.is_contiguous() && k.is_contiguous() && v.is_contiguous() &&
              o.is_contiguous() && do_.is_contiguous() && lse2.is_contiguous());
  TORCH_CHECK(is_bf16(do_) && lse2.scalar_type() == at::kFloat);
  const int B = (int)q.size(0), H = (int)q.size(1);
  const int S = (int)q.size(2), DP = (int)q.size(3);
  const int HKV = (int)k.size(1);
  const int SP = (S + 127) / 128 * 128;
  TORCH_CHECK(lse2.size(2) == SP);
  auto delta = at::empty({B, H, SP}, q.options().dtype(at::kFloat));
  check_hip(lumina_attn_delta(do_.data_ptr(), o.data_ptr(), delta.data_ptr(),
                              (int64_t)B * H * S, S, SP, DP, cur_stream()),
            "attn_delta");
  auto dq = at::empty_like(q);
  auto dk = at::empty_like(k);
  auto dv = at::empty_like(v);
  check_hip(lumina_attn_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(),
                            do_.data_ptr(), lse2.data_ptr(), delta.data_ptr(),
                            dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                            B, H, HKV, S, SP, DP, (float)scale, cur_stream()),
            "attn_bwd");
  return {dq, dk, dv};
}

// deep-pipelined 256^2 grouped GEMM (gemm8p.hip)
// nt: out[e] = A[e] @ B[e]^T, A [E,M,K], B [E,N,K]; K % 32 == 0
// nn: out[e] = A[e] @ B[e],   A [E,M,K], B [E,Kb,N]; K % 32, Kb <= K
//     (A zero-padded along K up to a multiple of 32; B rows clamped)
at::Tensor gg8t_nt(const at::Tensor& A, const at::Tensor& B, int64_t pf2) {
  TORCH_CHECK(A.is_contiguous() && B.is_contiguous());
  TORCH_CHECK(is_bf16(A) && is_bf16(B));
  TORCH_CHECK(A.dim() == 3 && B.dim() == 3 && A.size(2) == B.size(2));
  TORCH_CHECK(A.size(2) % 64 == 0, "gg8t requires K % 64 == 0");
  const int E = (int)A.size(0), M = (int)A.size(1);
  const int K = (int)A.size(2), N = (int)B.size(1);
  auto O = at::empty({E, M, N}, A.options());
  check_hip(lumina_gg8t_nt(A.data_ptr(), B.data_ptr(), O.data_ptr(), E, M,
                           N, K, (int64_t)M * K, (int64_t)N * K,
                           (int64_t)M * N, (int)pf2, cur_stream()),
            "gg8t_nt");
  return O;
}

at::Tensor gg8p_nt(const at::Tensor& A, const at::Tensor& B) {
  TORCH_CHECK(A.is_contiguous() && B.is_contiguous());
  TORCH_CHECK(is_bf16(A) && is_bf16(B));
  TORCH_CHECK(A.dim() == 3 && B.dim() == 3 && A.size(2) == B.size(2));
  TORCH_CHECK(A.size(2) % 32 == 0, "gg8p requires K % 32 == 0");
  const int E = (int)A.size(0), M = (int)A.size(1);
  const int K = (int)A.size(2), N = (int)B.size(1);
  auto O = at::empty({E, M, N}, A.options());
  launch_gg8p(A.data_ptr(), B.data_ptr(), O.data_ptr(), E, M, N, K, K,
              (int64_t)M * K, (int64_t)N * K, (int64_t)M * N, 0,
              cur_stream());
  check_hip(hipGetLastError(), "gg8p_nt");
  return O;
}

at::Tensor gg8p_nn(const at::Tensor& A, const at::Tensor& B) {
  TORCH_CHECK(A.is_contiguous() && B.is_contiguous());
  TORCH_CHECK(is_bf16(A) && is_bf16(B));
  TORCH_CHECK(A.dim() == 3 && B.dim() == 3);
  const int E = (int)A.size(0), M = (int)A.size(1);
  const int K = (int)A.size(2), Kb = (int)B.size(1), N = (int)B.size(2);
  TORCH_CHECK(K % 32 == 0, "gg8p requires (padded) K % 32 == 0");
  TORCH_CHECK(Kb <= K && K - Kb < 32, "K must be Kb padded up to 32");
  TORCH_CHECK(N % 8 == 0, "gg8p_nn requires N % 8 == 0");
  auto O = at::empty({E, M, N}, A.options());
  launch_gg8p(A.data_ptr(), B.data_ptr(), O.data_ptr(), E, M, N, K, Kb,
              (int64_t)M * K, (int64_t)Kb * N, (int64_t)M * N, 1,
              cur_stream());
  check_hip(hipGetLastError(), "gg8p_nn");
  return O;
}

// ---- MX-fp8 rowwise path (mxfp8.hip) -------------------------------------
std::tuple<at::Tensor, at::Tensor> mx_quant_rows(const at::Tensor& x,
                                                 int64_t kp) {
  TORCH_CHECK(x.is_contiguous() && is_bf16(x));
  const int K = (int)x.size(-1);
  const int Kp = (int)(kp > 0 ? kp : (K + 127) / 128 * 128);
  TORCH_CHECK(Kp % 128 == 0 && Kp >= K);
  const int64_t R = x.numel() / K;
  auto sizes = x.sizes().vec();
  sizes.back() = Kp;
  auto q = at::empty(sizes, x.options().dtype(at::kByte));
  auto ssz = x.sizes().vec();
  ssz.pop_back();
  auto s = at::empty(ssz, x.options().dtype(at::kByte));
  check_hip(lumina_mx_quant_rows(x.data_ptr(), q.data_ptr(), s.data_ptr(),
                                 R, K, Kp, cur_stream()),
            "mx_quant_rows");
  return {q, s};
}

std::tuple<at::Tensor, at::Tensor> mx_quant_cols(const at::Tensor& w,
                                                 int64_t kp) {
  // w [K, N] or batched [E, K, N] -> transposed quant [.., N, Kp]
  TORCH_CHECK(w.is_contiguous() && is_bf16(w));
  TORCH_CHECK(w.dim() == 2 || w.dim() == 3);
  const int E = w.dim() == 3 ? (int)w.size(0) : 1;
  const int K = (int)w.size(-2), N = (int)w.size(-1);
  const int Kp = (int)(kp > 0 ? kp : (K + 127) / 128 * 128);
  TORCH_CHECK(Kp % 128 == 0 && Kp >= K);
  auto q = w.dim() == 3
      ? at::empty({E, N, Kp}, w.options().dtype(at::kByte))
      : at::empty({N, Kp}, w.options().dtype(at::kByte));
  auto s = w.dim() == 3
      ? at::empty({E, N}, w.options().dtype(at::kByte))
      : at::empty({N}, w.options().dtype(at::kByte));
  auto ws = at::empty({(int64_t)E * N}, w.options().dtype(at::kFloat));
  check_hip(lumina_mx_quant_cols(w.data_ptr(), q.data_ptr(), s.data_ptr(),
                                 ws.data_ptr(), E, K, N, Kp, cur_stream()),
            "mx_quant_cols");
  return {q, s};
}

at::Tensor gg_mx_nt(const at::Tensor& Aq, const at::Tensor& As,
                    const at::Tensor& Bq, const at::Tensor& Bs) {
  TORCH_CHECK(Aq.is_contiguous() && Bq.is_contiguous());
  TORCH_CHECK(Aq.scalar_type() == at::kByte && Bq.scalar_type() == at::kByte);
  TORCH_CHECK(Aq.dim() == 3 && Bq.dim() == 3 && Aq.size(2) == Bq.size(2));
  TORCH_CHECK(Aq.size(2) % 128 == 0, "MX GEMM needs padded K % 128 == 0");
  const int E = (int)Aq.size(0), M = (int)Aq.size(1);
  const int K = (int)Aq.size(2), N = (int)Bq.size(1);
  TORCH_CHECK(As.numel() == (int64_t)E * M && Bs.numel() == (int64_t)E * N);
  auto O = at::empty({E, M, N},
                     Aq.options().dtype(at::kBFloat16));
  check_hip(lumina_gg_mx_nt(Aq.data_ptr(), Bq.data_ptr(), As.data_ptr(),
                            Bs.data_ptr(), O.data_ptr(), E, M, N, K,
                            (int64_t)M * K, (int64_t)N * K, (int64_t)M * N,
                            cur_stream()),
            "gg_mx_nt");
  return O;
}

// ---- fused batch-1 decode kernels (decode.hip) ---------------------------
void dec_gemv(const at::Tensor& W, const at::Tensor& x,
              const std::optional<at::Tensor>& wn,
              const std::optional<at::Tensor>& resid, at::Tensor& y,
              double eps, int64_t flags) {
  const int K = (int)x.numel();
  const int N = (int)y.numel();
  check_hip(lumina_dec_gemv(W.data_ptr(), x.data_ptr(),
                            wn ? wn->data_ptr() : nullptr,
                            resid ? resid->data_ptr() : nullptr,
                            y.data_ptr(), N, K, (float)eps, (int)flags,
                            cur_stream()),
            "dec_gemv");
}

void dec_rope_cache(const at::Tensor& qkv, at::Tensor& q_out, at::Tensor& kc,
                    at::Tensor& vc, const at::Tensor& cost,
                    const at::Tensor& sint, const at::Tensor& pos_dev,
                    int64_t H, int64_t HKV, int64_t D) {
  check_hip(lumina_dec_rope_cache(qkv.data_ptr(), q_out.data_ptr(),
                                  kc.data_ptr(), vc.data_ptr(),
                                  cost.data_ptr<float>(),
                                  sint.data_ptr<float>(),
                                  pos_dev.data_ptr<int>(), (int)H, (int)HKV,
                                  (int)D, cur_stream()),
            "dec_rope_cache");
}

void dec_attn(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc,
              at::Tensor& out, const at::Tensor& pos_dev, int64_t H,
              int64_t HKV, int64_t D, double scale) {
  const int cap = (int)kc.size(0);
  check_hip(lumina_dec_attn(q.data_ptr(), kc.data_ptr(), vc.data_ptr(),
                            out.data_ptr(), pos_dev.data_ptr<int>(), cap,
                            (int)H, (int)HKV, (int)D, (float)scale,
                            cur_stream()),
            "dec_attn");
}

void dec_advance(const at::Tensor& pos_dev) {
  check_hip(lumina_dec_advance(pos_dev.data_ptr<int>(), cur_stream()),
            "dec_advance");
}

void dec_rmsnorm(const at::Tensor& x, const at::Tensor& wn, at::Tensor& out,
                 double eps) {
  check_hip(lumina_dec_rmsnorm(x.data_ptr(), wn.data_ptr(), out.data_ptr(),
                               (int)x.numel(), (float)eps, cur_stream()),
            "dec_rmsnorm");
}

void dec_router(const at::Tensor& x, const at::Tensor& wn,
                const at::Tensor& Wg, at::Tensor& xhat, at::Tensor& eidx,
                at::Tensor& ew, int64_t k, double temp, double eps) {
  check_hip(lumina_dec_router(x.data_ptr(), wn.data_ptr(), Wg.data_ptr(),
                              xhat.data_ptr(), eidx.data_ptr<int>(),
                              ew.data_ptr<float>(), (int)x.numel(),
                              (int)Wg.size(0), (int)k, (float)temp,
                              (float)eps, cur_stream()),
            "dec_router");
}

void dec_topk(const at::Tensor& logits, at::Tensor& eidx, at::Tensor& ew,
              int64_t k, double temp) {
  check_hip(lumina_dec_topk(logits.data_ptr(), eidx.data_ptr<int>(),
                            ew.data_ptr<float>(), (int)logits.numel(),
                            (int)k, (float)temp, cur_stream()),
            "dec_topk");
}

void dec_gemv_moe(const at::Tensor& W, const at::Tensor& x,
                  const std::optional<at::Tensor>& resid, at::Tensor& y,
                  const at::Tensor& eidx, const at::Tensor& ew,
                  int64_t slot, int64_t flags) {
  // W: [E, N(or 2N), K] contiguous; rows per expert from y/x sizes
  const int K = (int)x.numel();
  const int N = (int)y.numel();
  const int64_t estride = W.size(1) * W.size(2);
  check_hip(lumina_dec_gemv_moe(W.data_ptr(), x.data_ptr(),
                                resid ? resid->data_ptr() : nullptr,
                                y.data_ptr(), eidx.data_ptr<int>(),
                                ew.data_ptr<float>(), (int)slot, estride,
                                N, K, (int)flags, cur_stream()),
            "dec_gemv_moe");
}

at::Tensor gemv(const at::Tensor& x, const at::Tensor& w) {
  // y[N] = w[N,K] @ x[K]
  TORCH_CHECK(x.is_contiguous() && w.is_contiguous());
  TORCH_CHECK(x.dim() == 1 && w.dim() == 2 && w.size(1) == x.numel());
  TORCH_CHECK(x.scalar_type() == w.scalar_type());
  auto y = at::empty({w.size(0)}, x.options());
  check_hip(lumina_gemv(w.data_ptr(), x.data_ptr(), y.data_ptr(),
                        (int)w.size(0), x.numel(), is_bf16(x) ? 1 : 0,
                        cur_stream()),
            "gemv");
  return y;
}

// ---- paged cache -----------------------------------------------------------
namespace {

void check_same_device(const at::Tensor& t, const at::Tensor& first,
                       const char* name) {
  TORCH_CHECK_VALUE(t.device() == first.device(), name, " is on ", t.device(),
                    ", not on ", first.device());
}

// Whether two elements of t may share memory (an expanded tensor, or strides
// that step over less than they span): what is written there is not defined.
bool overlaps(const at::Tensor& t) {
  if (t.is_non_overlapping_and_dense()) return false;
  std::vector<std::pair<int64_t, int64_t>> dims;     // stride, size
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1) dims.emplace_back(t.stride(i), t.size(i));
  std::sort(dims.begin(), dims.end());
  int64_t extent = 1;
  for (const auto& [stride, size] : dims) {
    if (stride < extent) return t.numel() > 0;
    extent += stride * (size - 1);
  }
  return false;
}

// t is written in place: autograd refuses a backward pass that saved it before.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Pages [P, HKV, page, W]; returns log2(page).
int check_pages(const at::Tensor& t, const at::Tensor& like, const char* name,
                int64_t heads, int64_t dim) {
  TORCH_CHECK_VALUE(t.dim() == 4, name, " must be [pages, kv_heads, page, width]");
  check_same_device(t, like, name);
  TORCH_CHECK_TYPE(t.scalar_type() == like.scalar_type(), name, " is ",
                   t.scalar_type(), ", not ", like.scalar_type());
  const int64_t page = t.size(2), W = t.size(3);
  TORCH_CHECK_VALUE(t.size(1) == heads, name, " has ", t.size(1),
                    " heads, not ", heads);
  TORCH_CHECK_VALUE(page >= 16 && page <= 4096 && (page & (page - 1)) == 0,
                    "page size must be a power of two from 16 to 4096, got ",
                    page);
  TORCH_CHECK_VALUE(W % 8 == 0 && W >= dim && W < dim + 8, name,
                    " must be head_dim rounded up to a multiple of 8 wide "
                    "(head_dim ", dim, ", got ", W, ")");
  TORCH_CHECK_VALUE(t.stride(3) == 1 && t.stride(2) % 8 == 0 &&
                    t.stride(1) % 8 == 0 && t.stride(0) % 8 == 0 &&
                    (uintptr_t)t.data_ptr() % 16 == 0,
                    name, " rows must be contiguous and 16-byte aligned");
  TORCH_CHECK_VALUE(t.size(0) <= INT32_MAX, name, " has too many pages");
  int shift = 0;
  while ((1ll << shift) < page) ++shift;
  return shift;
}

void check_int32(const at::Tensor& t, const at::Tensor& like, int64_t dims,
                 const char* name) {
  check_same_device(t, like, name);
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt, name, " must be int32, got ",
                   t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() == dims && (t.numel() == 0 ||
                    t.size(dims - 1) == 1 || t.stride(dims - 1) == 1), name, " must be a ", dims,
                    "-dimensional tensor with contiguous rows");
}

}  // namespace

at::Tensor paged_attn(const at::Tensor& q_, const at::Tensor& kp,
                      const at::Tensor& vp, const at::Tensor& table,
                      const at::Tensor& lens, double scale) {
  TORCH_CHECK_VALUE(q_.dim() == 3, "q must be [batch, heads, head_dim]");
  TORCH_CHECK_TYPE(is_bf16(q_), "paged_attention on the GPU takes bf16, got ",
                   q_.scalar_type());
  TORCH_CHECK(!(at::GradMode::is_enabled() &&
                (q_.requires_grad() || kp.requires_grad() ||
                 vp.requires_grad())),
              "paged_attention has no gradient: call it under torch.no_grad()");
  const c10::DeviceGuard guard(q_.device());
  const at::Tensor q = q_.stride(2) == 1 || q_.size(2) == 1
      ? q_ : q_.contiguous();
  const int64_t B = q.size(0), H = q.size(1), D = q.size(2);
  TORCH_CHECK_VALUE(kp.dim() == 4 && kp.sizes() == vp.sizes(),
                    "k_pages and v_pages must be [pages, kv_heads, page, "
                    "width], of one shape");
  const int64_t HKV = kp.size(1);
  TORCH_CHECK_VALUE(D >= 1 && D <= 192, "head_dim must be 1 to 192, got ", D);
  TORCH_CHECK_VALUE(HKV > 0 && H > 0 && H % HKV == 0, "heads (", H,
                    ") must be a multiple of kv_heads (", HKV, ")");
  TORCH_CHECK_VALUE(scale > -1e30 && scale < 1e30, "scale must be between -1e30 "
                    "and 1e30, got ", scale);
  const int shift = check_pages(kp, q, "k_pages", HKV, D);
  check_pages(vp, q, "v_pages", HKV, D);
  check_int32(table, q, 2, "block_table");
  check_int32(lens, q, 1, "seq_lens");
  TORCH_CHECK_VALUE(table.size(0) == B && lens.size(0) == B,
                    "block_table and seq_lens need a row for each of the ", B,
                    " sequences");
  const int64_t M = table.size(1), cap = M << shift;
  TORCH_CHECK_VALUE(cap < (1 << 29), "a row of block_table holds ", cap,
                    " tokens: fewer than 2^29 are supported");
  auto o = at::empty({B, H, D}, q.options());
  if (B == 0) return o;
  if (cap == 0 || kp.size(0) == 0) return o.zero_();
  // Workgroups wanted for all chunks together: 512 (two of the three that a unit
  // holds), until a chunk has 1024 tokens, then up to 4096 of them, as far as the
  // table has room for that much; the kernel sets the chunks' length by it. 512 /
  // 768 / 1024 at first: 8 rows of up to 4096 tokens 16.3 / 16.4 / 19.8 us, 64 of
  // 1000 44.7 / 52.4 / 50.8, one of 30000 28 / 30 / 32 (32:8 heads x 128). 1024 /
  // 2048 / 4096 for long ones: 64 rows of up to 32690 tokens 802 / 767 / 754.
  const int64_t R = HKV * ((H / HKV + 15) / 16), steps = (cap + 127) / 128;
  TORCH_CHECK_VALUE(B * steps <= (1 << 24), "block_table holds ", B * cap,
                    " tokens: up to 2^31 are supported");
  const int64_t few = std::max<int64_t>(1, 512 / R);
  const int64_t many = std::max(few, std::min(4096 / R, B * steps / 8));
  const int64_t chunks = std::min(many + B + 1, B * steps + B);
  at::Tensor ws, where, plan;
  float* part = nullptr;
  float* ml = nullptr;
  int* wh = nullptr;
  if (steps > 1) {
    ws = at::empty({chunks * H * (D + 2)}, q.options().dtype(at::kFloat));
    ml = ws.data_ptr<float>();
    part = ml + chunks * H * 2;
    where = at::empty({B, 2}, lens.options());
    wh = where.data_ptr<int>();
  }
  if (B > 128) plan = at::empty({4 + 2 * chunks}, lens.options());
  const int64_t strides[9] = {q.stride(0), q.stride(1), kp.stride(0),
                              kp.stride(1), kp.stride(2), vp.stride(0),
                              vp.stride(1), vp.stride(2), table.stride(0)};
  check_hip(lumina_paged_attn(q.data_ptr(), kp.data_ptr(), vp.data_ptr(),
                              o.data_ptr(), table.data_ptr<int>(),
                              lens.data_ptr<int>(), part, ml, wh,
                              plan.defined() ? plan.data_ptr<int>() : nullptr,
                              strides,
                              kp.size(0), (int)B, (int)H, (int)HKV, (int)D,
                              (int)kp.size(3), shift, (int)M, (int)few, (int)many,
                              (int)chunks, (float)scale, cur_stream()),
            "paged_attention");
  return o;
}

void paged_append(const at::Tensor& k_, const at::Tensor& v_,
                  const at::Tensor& kp, const at::Tensor& vp,
                  const at::Tensor& table, const at::Tensor& pos,
                  const std::optional<at::Tensor>& ids) {
  TORCH_CHECK_VALUE(k_.dim() == 3 && v_.sizes() == k_.sizes(),
                    "k and v must be [tokens, kv_heads, head_dim]");
  TORCH_CHECK_TYPE(k_.scalar_type() == at::kBFloat16 ||
                   k_.scalar_type() == at::kHalf ||
                   k_.scalar_type() == at::kFloat,
                   "k must be bf16, fp16 or fp32, got ", k_.scalar_type());
  check_same_device(v_, k_, "v");
  TORCH_CHECK_TYPE(v_.scalar_type() == k_.scalar_type(), "v is ",
                   v_.scalar_type(), ", not ", k_.scalar_type());
  const c10::DeviceGuard guard(k_.device());
  const int64_t T = k_.size(0), HKV = k_.size(1), D = k_.size(2);
  const at::Tensor k = k_.stride(2) == 1 || D == 1 ? k_ : k_.contiguous();
  const at::Tensor v = v_.stride(2) == 1 || D == 1 ? v_ : v_.contiguous();
  TORCH_CHECK_VALUE(HKV > 0 && D > 0, "k has no heads or no channels");
  TORCH_CHECK_VALUE(kp.sizes() == vp.sizes(),
                    "k_pages and v_pages must be of one shape");
  const int shift = check_pages(kp, k, "k_pages", HKV, D);
  check_pages(vp, k, "v_pages", HKV, D);
  TORCH_CHECK_VALUE(!overlaps(kp) && !overlaps(vp) &&
                    (kp.numel() == 0 || kp.data_ptr() != vp.data_ptr()),
                    "the pages' memory overlaps");
  check_int32(table, k, 2, "block_table");
  check_int32(pos, k, 1, "positions");
  TORCH_CHECK_VALUE(pos.size(0) == T, "positions has ", pos.size(0),
                    " entries for ", T, " tokens");
  if (ids.has_value()) {
    check_int32(*ids, k, 1, "seq_ids");
    TORCH_CHECK_VALUE(ids->size(0) == T, "seq_ids has ", ids->size(0),
                      " entries for ", T, " tokens");
  } else {
    TORCH_CHECK_VALUE(table.size(0) == T, "without seq_ids there is one token "
                      "for each sequence: ", T, " tokens, ", table.size(0),
                      " sequences");
  }
  if (T == 0) return;
  const int64_t strides[11] = {k.stride(0), k.stride(1), v.stride(0),
                               v.stride(1), kp.stride(0), kp.stride(1),
                               kp.stride(2), vp.stride(0), vp.stride(1),
                               vp.stride(2), table.stride(0)};
  check_hip(lumina_paged_append(k.data_ptr(), v.data_ptr(), kp.data_ptr(),
                                vp.data_ptr(), table.data_ptr<int>(),
                                pos.data_ptr<int>(),
                                ids.has_value() ? ids->data_ptr<int>()
                                                : nullptr,
                                strides, kp.size(0), T, (int)table.size(0),
                                (int)HKV, (int)D, (int)kp.size(3), shift,
                                (int)table.size(1), (int)k.element_size(),
                                cur_stream()),
            "paged_kv_append");
  written(kp);
  written(vp);
}

void copy_pages(const std::vector<at::Tensor>& pools,
                const std::vector<int64_t>& src,
                const std::vector<int64_t>& dst) {
  TORCH_CHECK_VALUE(src.size() == dst.size(), "src names ", src.size(),
                    " pages, dst ", dst.size());
  TORCH_CHECK_VALUE(!pools.empty(), "no pool was given");
  std::vector<int64_t> s(src), d(dst);
  std::sort(s.begin(), s.end());
  std::sort(d.begin(), d.end());
  for (size_t i = 1; i < d.size(); ++i)
    TORCH_CHECK_VALUE(d[i] != d[i - 1], "page ", d[i], " is written twice");
  for (int64_t p : d)
    TORCH_CHECK_VALUE(!std::binary_search(s.begin(), s.end(), p), "page ", p,
                      " is both read and written");
  for (const auto& t : pools) {
    TORCH_CHECK_VALUE(t.dim() >= 3, "a pool must be [layers, pages, ...]");
    check_same_device(t, pools[0], "pool");
    TORCH_CHECK_VALUE(t.size(0) > 0 && t.size(1) > 0 && t.numel() > 0,
                      "a pool is empty");
    int64_t span = 1;
    bool contiguous = true;
    for (int64_t i = t.dim() - 1; i >= 2; --i) {
      contiguous = contiguous && (t.size(i) == 1 || t.stride(i) == span);
      span *= t.size(i);
    }
    TORCH_CHECK_VALUE(contiguous, "a pool's pages must be contiguous");
    TORCH_CHECK_VALUE(!overlaps(t), "a pool's memory overlaps");
    TORCH_CHECK_VALUE(t.size(1) <= INT32_MAX, "a pool has too many pages");
    if (!d.empty())
      TORCH_CHECK_VALUE(s.front() >= 0 && d.front() >= 0 &&
                        s.back() < t.size(1) && d.back() < t.size(1),
                        "page numbers must be in 0 to ", t.size(1) - 1);
  }
  if (d.empty()) return;
  const std::vector<int> si(src.begin(), src.end()), di(dst.begin(), dst.end());
  const c10::DeviceGuard guard(pools[0].device());
  auto page_bytes = [](const at::Tensor& t) {
    return (int64_t)(t.numel() / (t.size(0) * t.size(1)) * t.element_size());
  };
  for (size_t i = 0; i < pools.size();) {
    // two pools of the same size (keys and values) share a launch
    const bool two = i + 1 < pools.size() &&
        pools[i].size(0) == pools[i + 1].size(0) &&
        page_bytes(pools[i]) == page_bytes(pools[i + 1]);
    void* ptr[2];
    int64_t layer[2], page[2];
    const int n = two ? 2 : 1;
    for (int j = 0; j < n; ++j) {
      const auto& t = pools[i + j];
      ptr[j] = t.data_ptr();
      layer[j] = t.stride(0) * t.element_size();
      page[j] = t.stride(1) * t.element_size();
    }
    check_hip(lumina_copy_pages(ptr, n, layer, page, (int)pools[i].size(0),
                                page_bytes(pools[i]), si.data(), di.data(),
                                (int64_t)si.size(), cur_stream()),
              "copy_pages");
    for (int j = 0; j < n; ++j) written(pools[i + j]);
    i += n;
  }
}

// ---- token log probabilities -------------------------------------------------
namespace {
int logit_dtype(const at::Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return 0;
  if (t.scalar_type() == at::kHalf) return 1;
  TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat,
                   "logits must be bf16, fp16 or fp32, got ", t.scalar_type());
  return 2;
}
}  // namespace

// logits [N, V] with contiguous rows. stat [N, 2] (row maximum, log2 of the sum)
// is what the gradient needs; undefined where want_stat is false.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>
logprob_fwd(const at::Tensor& x, const at::Tensor& tok, int64_t k,
            int64_t ignore, bool want_stat) {
  TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) > 0 &&
                    (x.stride(1) == 1 || x.size(1) == 1),
                    "logits must be [rows, vocab] with contiguous rows");
  const int dtype = logit_dtype(x);
  check_same_device(tok, x, "tokens");
  TORCH_CHECK_TYPE(tok.scalar_type() == at::kLong ||
                   tok.scalar_type() == at::kInt,
                   "tokens must be int64 or int32, got ", tok.scalar_type());
  const int64_t N = x.size(0), V = x.size(1);
  TORCH_CHECK_VALUE(tok.dim() == 1 && tok.size(0) == N && tok.is_contiguous(),
                    "tokens must hold one token for each of the ", N, " rows");
  TORCH_CHECK_VALUE(V <= (1 << 30) && N <= INT32_MAX,
                    "logits of ", N, " x ", V, " are not supported");
  TORCH_CHECK_VALUE(k >= 0 && k <= 64 && k <= V, "top_k must be 0 to 64 and at "
                    "most the vocabulary's ", V, ", got ", k);
  const c10::DeviceGuard guard(x.device());
  const auto f32 = x.options().dtype(at::kFloat);
  auto lp = at::empty({N}, f32), ent = at::empty({N}, f32);
  at::Tensor stat;
  if (want_stat) stat = at::empty({N, 2}, f32);
  auto tl = at::empty({N, k}, f32);
  auto ti = at::empty({N, k}, x.options().dtype(at::kLong));
  if (N > 0)
    check_hip(lumina_logprob_fwd(x.data_ptr(), dtype, tok.data_ptr(),
                                 tok.scalar_type() == at::kLong,
                                 lp.data_ptr<float>(), ent.data_ptr<float>(),
                                 want_stat ? stat.data_ptr<float>() : nullptr,
                                 tl.data_ptr<float>(), ti.data_ptr<int64_t>(),
                                 N, (int)V, x.stride(0), (int)k, ignore,
                                 cur_stream()), "token_logprobs");
  return {lp, ent, tl, ti, stat};
}

at::Tensor logprob_bwd(const at::Tensor& x, const at::Tensor& tok,
                       const at::Tensor& stat, const at::Tensor& ent,
                       const std::optional<at::Tensor>& g_lp,
                       const std::optional<at::Tensor>& g_ent,
                       int64_t ignore) {
  const int dtype = logit_dtype(x);
  const int64_t N = x.size(0), V = x.size(1);
  const c10::DeviceGuard guard(x.device());
  auto grad = [&](const std::optional<at::Tensor>& g) -> const float* {
    if (!g.has_value()) return nullptr;
    TORCH_CHECK_VALUE(g->scalar_type() == at::kFloat && g->is_contiguous() &&
                      g->numel() == N && g->device() == x.device(),
                      "a gradient must be fp32 and contiguous, one for each row");
    return g->data_ptr<float>();
  };
  auto dx = at::empty({N, V}, x.options());
  if (N > 0)
    check_hip(lumina_logprob_bwd(x.data_ptr(), dtype, tok.data_ptr(),
                                 tok.scalar_type() == at::kLong,
                                 stat.data_ptr<float>(),
                                 ent.data_ptr<float>(), grad(g_lp),
                                 grad(g_ent), dx.data_ptr(), N, (int)V,
                                 x.stride(0), ignore, cur_stream()),
              "token_logprobs gradient");
  return dx;
}

namespace {

// Gradients that cannot be differentiated again: doing so raises. Small calls are
// bound by the host, so these operators' gradients are recorded here and not by
// Python functions (a row of log probabilities and its gradient: 56 us of
// host time for 96, packed attention of 64 tokens 73 for 125).
torch::autograd::variable_list once(
    torch::autograd::variable_list grads,
    const torch::autograd::variable_list& inputs) {
  if (!at::GradMode::is_enabled()) return grads;
  torch::autograd::variable_list in;
  for (const auto& g : grads)
    if (g.defined()) in.push_back(g.detach().requires_grad_(true));
  in.insert(in.end(), inputs.begin(), inputs.end());   // leads back to them
  const auto fn = std::make_shared<torch::autograd::DelayedError>(
      "this gradient can be taken once only", (int)in.size());
  const auto out = (*fn)(std::move(in));
  size_t i = 0;
  for (auto& g : grads)
    if (g.defined()) g = out[i++];
  return grads;
}

class LogprobFn : public torch::autograd::Function<LogprobFn> {
 public:
  static torch::autograd::variable_list forward(
      torch::autograd::AutogradContext* ctx, const at::Tensor& x,
      const at::Tensor& tok, int64_t k, int64_t ignore) {
    const auto [lp, ent, tl, ti, stat] = logprob_fwd(x, tok, k, ignore, true);
    ctx->save_for_backward({x, tok, stat, ent});
    ctx->saved_data["ignore"] = ignore;
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({tl, ti});
    return {lp, ent, tl, ti};
  }

  static torch::autograd::variable_list backward(
      torch::autograd::AutogradContext* ctx,
      torch::autograd::variable_list g) {
    at::Tensor dx;
    const auto s = ctx->get_saved_variables();
    if (g[0].defined() || g[1].defined()) {
      const at::NoGradGuard no_grad;
      auto grad = [](const at::Tensor& t) {
        return t.defined() ? std::optional<at::Tensor>(t.contiguous())
                           : std::nullopt;
      };
      dx = logprob_bwd(s[0], s[1], s[2], s[3], grad(g[0]), grad(g[1]),
                       ctx->saved_data["ignore"].toInt());
    }
    auto out = once({dx}, {s[0]});
    return {out[0], at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

}  // namespace

// logits [N, V] with contiguous rows, tokens [N] -> logprobs, entropy,
// alternatives and their ids
std::vector<at::Tensor> token_logprobs(const at::Tensor& x,
                                       const at::Tensor& tok, int64_t k,
                                       int64_t ignore) {
  if (at::GradMode::is_enabled() && x.requires_grad())
    return LogprobFn::apply(x, tok, k, ignore);
  const auto r = logprob_fwd(x, tok, k, ignore, false);
  return {std::get<0>(r), std::get<1>(r), std::get<2>(r), std::get<3>(r)};
}

// ---- packed attention ------------------------------------------------------
namespace {
// Rows as the kernels take them: whole aligned 16-byte pieces, and tokens no
// further apart than a tile's 32-bit offsets reach.
bool aligned_rows(const at::Tensor& t) {
  return t.size(2) % 8 == 0 && t.stride(2) == 1 && t.stride(0) % 8 == 0 &&
         t.stride(1) % 8 == 0 && t.stride(0) >= 0 &&
         t.stride(0) <= (1 << 23) && (uintptr_t)t.data_ptr() % 16 == 0;
}

// Room for the blocks of more than 64 sequences (packed_list_kernel).
at::Tensor block_list(const at::Tensor& cu, int64_t T) {
  const int64_t B = cu.size(0) - 1;
  if (B <= 64) return at::Tensor();
  return at::empty({4 * (T / 128 + B + 2)}, cu.options());
}

// Those that are not become copies of head_dim rounded up to 8, zero past it;
// all of them if one has to change its width.
std::vector<at::Tensor> align_rows(std::vector<at::Tensor> ts) {
  const int64_t T = ts[0].size(0), D = ts[0].size(2), W = (D + 7) / 8 * 8;
  const void* src[3];
  void* dst[3];
  int64_t strides[6];
  int heads[3], n = 0;
  std::vector<at::Tensor> keep;
  for (auto& t : ts) {
    if (T == 0 || aligned_rows(t)) continue;
    const at::Tensor s = t.stride(2) == 1 || D == 1 ? t : t.contiguous();
    keep.push_back(s);
    t = at::empty({T, s.size(1), W}, s.options());
    src[n] = s.data_ptr();
    dst[n] = t.data_ptr();
    strides[2 * n] = s.stride(0);
    strides[2 * n + 1] = s.stride(1);
    heads[n++] = (int)s.size(1);
  }
  if (n > 0)
    check_hip(lumina_pack_rows(src, dst, strides, heads, n, T, (int)D,
                               cur_stream()), "flash_attention_packed");
  return ts;
}
}  // namespace

// -> (o, rest, lse2, q, k, v) for packed_attn_bwd: rest is what rounding o left
// over, q, k and v are as the kernels read them. rest and lse2 are empty where
// want_lse is false.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor,
           at::Tensor>
packed_attn_fwd(const at::Tensor& q_, const at::Tensor& k_,
                const at::Tensor& v_, const at::Tensor& cu, double scale,
                bool want_lse) {
  TORCH_CHECK_VALUE(q_.dim() == 3 && k_.dim() == 3 && v_.sizes() == k_.sizes(),
                    "q must be [tokens, heads, head_dim], k and v [tokens, "
                    "kv_heads, head_dim]");
  TORCH_CHECK_TYPE(is_bf16(q_), "flash_attention_packed on the GPU takes bf16, "
                   "got ", q_.scalar_type());
  for (const auto* t : {&k_, &v_}) {
    check_same_device(*t, q_, "k or v");
    TORCH_CHECK_TYPE(t->scalar_type() == q_.scalar_type(), "k or v is ",
                     t->scalar_type(), ", not ", q_.scalar_type());
  }
  const int64_t T = q_.size(0), H = q_.size(1), D = q_.size(2);
  const int64_t HKV = k_.size(1);
  TORCH_CHECK_VALUE(k_.size(0) == T && k_.size(2) == D,
                    "q, k and v need the same tokens and head_dim");
  TORCH_CHECK_VALUE(D >= 1 && D <= 192, "head_dim must be 1 to 192, got ", D);
  TORCH_CHECK_VALUE(HKV > 0 && H > 0 && H % HKV == 0, "heads (", H,
                    ") must be a multiple of kv_heads (", HKV, ")");
  TORCH_CHECK_VALUE(T <= (1 << 30), "at most 2^30 tokens, got ", T);
  check_int32(cu, q_, 1, "cu_seqlens");
  TORCH_CHECK_VALUE(cu.size(0) >= 1, "cu_seqlens needs one entry more than "
                    "there are sequences");
  // one workgroup lists their blocks
  TORCH_CHECK_VALUE(cu.size(0) <= 65537, "at most 65536 sequences, got ",
                    cu.size(0) - 1);
  TORCH_CHECK_VALUE(scale > 1e-30 && scale < 1e30, "scale must be positive "
                    "(1e-30 to 1e30), got ", scale);
  const c10::DeviceGuard guard(q_.device());
  const auto in = align_rows({q_, k_, v_});
  const auto &q = in[0], &k = in[1], &v = in[2];
  auto o = at::empty({T, H, D}, q.options());
  auto lse = at::empty({want_lse ? H : 0, T}, q.options().dtype(at::kFloat));
  auto rest = at::empty({want_lse ? T : 0, H, q.size(2)}, q.options());
  if (T == 0) return {o, rest, lse, q, k, v};
  const at::Tensor list = block_list(cu, T);
  const int64_t strides[8] = {q.stride(0), q.stride(1), k.stride(0),
                              k.stride(1), v.stride(0), v.stride(1), 0, 0};
  check_hip(lumina_packed_attn_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                   o.data_ptr(),
                                   want_lse ? rest.data_ptr() : nullptr,
                                   want_lse ? lse.data_ptr<float>() : nullptr,
                                   cu.data_ptr<int>(),
                                   list.defined() ? list.data_ptr<int>()
                                                  : nullptr, strides, (int)T,
                                   (int)cu.size(0) - 1, (int)H, (int)HKV,
                                   (int)q.size(2), (int)D, (float)scale,
                                   cur_stream()),
            "flash_attention_packed");
  return {o, rest, lse, q, k, v};
}

// Takes the gradient of o, and what packed_attn_fwd returned.
std::tuple<at::Tensor, at::Tensor, at::Tensor> packed_attn_bwd(
    const at::Tensor& go_, const at::Tensor& o, const at::Tensor& rest,
    const at::Tensor& lse, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
    const at::Tensor& cu, double scale) {
  TORCH_CHECK_VALUE(go_.sizes() == o.sizes() && go_.device() == o.device(),
                    "the gradient must be of the result's shape and device");
  TORCH_CHECK_TYPE(is_bf16(go_), "the gradient must be bf16");
  const c10::DeviceGuard guard(q.device());
  const int64_t T = o.size(0), H = o.size(1), D = o.size(2), HKV = k.size(1);
  auto dq = at::empty({T, H, D}, q.options());
  auto dk = at::empty({T, HKV, D}, q.options());
  auto dv = at::empty({T, HKV, D}, q.options());
  if (T == 0) return {dq, dk, dv};
  const auto go = align_rows({go_})[0];
  auto delta = at::empty({H, T}, lse.options());
  // dK / dV: a workgroup goes over the queries of its 128 keys for all heads of
  // the group. The causal half of all (query, key, head) pairs is spread over 256
  // units, and the longest workgroup alone takes more than its share while
  // T * HKV < 65536; twice that levels the rest. Below it the group's heads are
  // split, at the price of fp32 results that are written and read once more.
  // 8192 tokens: 8 kv heads x 4 x 128, 1 / 2 / 4 parts: 625 / 574 / 661 us;
  // 4 kv heads x 3 x 159, 1 / 3 parts: 343 / 257 us.
  const int64_t G = H / HKV;
  int64_t splits = 1;
  while (splits < G && (G % splits != 0 || splits * HKV * T < 131072)) ++splits;
  at::Tensor part;
  if (splits > 1) part = at::empty({2, splits, T, HKV, (D + 3) / 4 * 4}, lse.options());
  const at::Tensor list = block_list(cu, T);
  const int64_t strides[8] = {q.stride(0), q.stride(1), k.stride(0),
                              k.stride(1), v.stride(0), v.stride(1),
                              go.stride(0), go.stride(1)};
  check_hip(lumina_packed_attn_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                   o.data_ptr(), rest.data_ptr(),
                                   go.data_ptr(),
                                   lse.data_ptr<float>(),
                                   delta.data_ptr<float>(), dq.data_ptr(),
                                   dk.data_ptr(), dv.data_ptr(),
                                   splits > 1 ? part.data_ptr<float>()
                                              : nullptr, (int)splits,
                                   cu.data_ptr<int>(),
                                   list.defined() ? list.data_ptr<int>()
                                                  : nullptr, strides, (int)T,
                                   (int)cu.size(0) - 1, (int)H, (int)HKV,
                                   (int)q.size(2), (int)D, (float)scale,
                                   cur_stream()),
            "flash_attention_packed gradient");
  return {dq, dk, dv};
}

namespace {

class PackedAttnFn : public torch::autograd::Function<PackedAttnFn> {
 public:
  static at::Tensor forward(torch::autograd::AutogradContext* ctx,
                            const at::Tensor& q, const at::Tensor& k,
                            const at::Tensor& v, const at::Tensor& cu,
                            double scale) {
    // rows that start between 16 bytes were copied: the copies are kept
    const auto [o, rest, lse, qr, kr, vr] =
        packed_attn_fwd(q, k, v, cu, scale, true);
    ctx->save_for_backward({qr, kr, vr, o, rest, lse, cu});
    ctx->saved_data["scale"] = scale;
    return o;
  }

  static torch::autograd::variable_list backward(
      torch::autograd::AutogradContext* ctx,
      torch::autograd::variable_list g) {
    const auto s = ctx->get_saved_variables();
    at::Tensor dq, dk, dv;
    {
      const at::NoGradGuard no_grad;
      std::tie(dq, dk, dv) =
          packed_attn_bwd(g[0], s[3], s[4], s[5], s[0], s[1], s[2], s[6],
                          ctx->saved_data["scale"].toDouble());
    }
    auto out = once({dq, dk, dv}, {s[0], s[1], s[2]});
    return {out[0], out[1], out[2], at::Tensor(), at::Tensor()};
  }
};

}  // namespace

at::Tensor packed_attn(const at::Tensor& q, const at::Tensor& k,
                       const at::Tensor& v, const at::Tensor& cu,
                       double scale) {
  if (at::GradMode::is_enabled() &&
      (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return PackedAttnFn::apply(q, k, v, cu, scale);
  return std::get<0>(packed_attn_fwd(q, k, v, cu, scale, false));
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, mod) {
  mod.def("attn_fwd", &attn_fwd,
          "causal GQA flash attention forward -> (O, LSE2) (gfx950)");
  mod.def("attn_bwd", &attn_bwd,
          "causal GQA flash attention backward -> (dQ, dK, dV) (gfx950)");
  mod.def("gemv", &gemv, "batch-1 decode GEMV y = W @ x (gfx950)");
  mod.def("dec_gemv", &dec_gemv,
          "fused decode GEMV (norm/residual/swiglu epilogues, nt loads)");
  mod.def("dec_rope_cache", &dec_rope_cache,
          "decode RoPE + KV-cache append at the device cursor");
  mod.def("dec_attn", &dec_attn, "single-token GQA attention over the cache");
  mod.def("dec_advance", &dec_advance, "advance the decode cursor");
  mod.def("swiglu_bwd_fused", &swiglu_bwd_fused,
          "swiglu backward into one fused [rows, 2I] grad buffer");
  mod.def("dec_rmsnorm", &dec_rmsnorm, "decode rmsnorm -> xhat buffer");
  mod.def("dec_router", &dec_router,
          "fused decode MoE router: rmsnorm + gate GEMV + top-k");
  mod.def("dec_topk", &dec_topk,
          "decode router: softmax/temp top-k, renormalized, on device");
  mod.def("dec_gemv_moe", &dec_gemv_moe,
          "expert-indirect decode GEMV (weight = W + eidx[slot]*estride)");
  mod.def("mx_quant_rows", &mx_quant_rows,
          "rowwise e8m0 fp8 quantization, K zero-padded (gfx950)");
  mod.def("mx_quant_cols", &mx_quant_cols,
          "columnwise e8m0 fp8 quantization + transpose (gfx950)");
  mod.def("gg_mx_nt", &gg_mx_nt,
          "grouped MX-fp8 GEMM A.B^T at the ~5PF fp8 MFMA rate (gfx950)");
  mod.def("gg8t_nt", &gg8t_nt,
          "8-phase-template grouped NT GEMM (256^2, BK64, 16x16x32)");
  mod.def("gg8p_nt", &gg8p_nt,
          "256^2 pipelined grouped GEMM, A.B^T (gfx950)");
  mod.def("gg8p_nn", &gg8p_nn,
          "256^2 pipelined grouped GEMM, A.B with K-major B (gfx950)");
  mod.def("grouped_gemm_nt_v4", &grouped_gemm_nt_v4,
          "2-buffer raw-barrier counted-vmcnt variant (K%64==0)");
  mod.def("grouped_gemm_nt_v3", &grouped_gemm_nt_v3,
          "3-buffer counted-vmcnt variant (K%64==0)");
  mod.def("grouped_gemm_nt", &grouped_gemm_nt,
          "grouped expert GEMM out[e]=A[e]@B[e]^T, bf16 MFMA (gfx950)");
  mod.def("grouped_gemm_nt_v2", &grouped_gemm_nt_v2,
          "32x32 MFMA variant (K%64==0), swizzle-mode knob");
  mod.def("moe_gather_rows", &moe_gather_rows, "MoE dispatch gather (gfx950)");
  mod.def("moe_dispatch_bwd", &moe_dispatch_bwd, "MoE dispatch backward");
  mod.def("moe_combine_fwd", &moe_combine_fwd, "MoE weighted combine");
  mod.def("moe_combine_bwd_y", &moe_combine_bwd_y, "MoE combine backward (y)");
  mod.def("moe_combine_bwd_w", &moe_combine_bwd_w, "MoE combine backward (w)");
  mod.def("rmsnorm_fwd", &rmsnorm_fwd, "RMSNorm forward (gfx950)");
  mod.def("rmsnorm_bwd", &rmsnorm_bwd, "RMSNorm backward (gfx950)");
  mod.def("rope_fwd", &rope_fwd, "RoPE q/k rotation (gfx950)");
  mod.def("swiglu_fwd", &swiglu_fwd, "SwiGLU forward (gfx950)");
  mod.def("swiglu_bwd", &swiglu_bwd, "SwiGLU backward (gfx950)");
  mod.def("ce_fwd", &ce_fwd, "fused CE+accuracy forward (gfx950)");
  mod.def("ce_bwd", &ce_bwd, "fused CE backward (gfx950)");
  mod.def("l2norm_sq", &l2norm_sq, "flat L2 norm squared (gfx950)");
  mod.def("adamw_step", &adamw_step, "fused clip+AdamW on flat buffers (gfx950)");
  mod.def("packed_attn", &packed_attn,
          "packed causal attention, with its gradient");
  mod.def("paged_attn", &paged_attn, "single-token attention over pages");
  mod.def("paged_append", &paged_append, "append keys and values to pages");
  mod.def("copy_pages", &copy_pages, "copy pages within pools");
  mod.def("token_logprobs", &token_logprobs,
          "token log probabilities and entropy, with their gradient");
}
