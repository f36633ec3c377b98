// Torch bindings of the norm, the e4m3 products and the clipped optimizer steps
// (rmsnorm.hip, fp8.hip, optim.hip). Everything runs on the current stream of
// the tensors' own device; scratch memory is torch's, taken for each call, so
// that neither streams nor captured graphs share any.

#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <optional>
#include <unordered_set>
#include <vector>

using torch::Tensor;
using OptTensor = std::optional<Tensor>;

extern "C" {
void al_rms_fwd(int type, int wtype, const void* x, long x_stride, const void* res,
                long res_stride, const void* w, void* y, void* total, float* rstd, void* q,
                void* scale, int out, long rows, int dim, int pitch, int scale_stride, float eps,
                void* stream);
int al_rms_bwd_parts(int type, long rows, int dim);
void al_rms_bwd(int type, int wtype, const void* s, long s_stride, const void* dy,
                const void* dsum, const void* w, const float* rstd, void* dx, float* part,
                void* dw, int parts, long rows, int dim, void* stream);
void al_col_sum(const double* part, void* out, int type, int parts, int dim, void* stream);
void al_quant_rows(int type, int kind, const void* x, long row_stride, long col_stride, void* q,
                   void* scale, long rows, int dim, int pitch, int scale_stride, void* stream);
void al_quant_tile(int type, int kind, int tile, const void* x, long row_stride, int rows,
                   int cols, void* q, void* scale, int pitch, int scale_stride, void* qt,
                   void* scale_t, int pitch_t, int scale_t_stride, double* part, void* stream);
int al_fp8_gemm_splits(int kind, int out_type, int m, int n, int blocks);
void al_fp8_gemm(int kind, const void* a, const void* sa, long lda, int sa_stride, const void* b,
                 const void* sb, long ldb, int sb_stride, int b_tile, int m, int n, int blocks,
                 const void* bias, int bias_type, void* out, int out_type, float* split_out,
                 int splits, void* stream);
void al_fp8_few_rows(int kind, int type, const void* x, long x_stride, int dim, const void* b,
                     const void* sb, long ldb, int sb_stride, int b_tile, int m, int n, int blocks,
                     const void* bias, int bias_type, void* out, void* stream);
int al_norm_batch_bytes();
void al_norm_batch_clear(void* batch);
int al_norm_batch_add(void* batch, void* p, long n);
int al_norm_blocks(const void* batch);
void al_sq_sum(int type, const void* batch, double* part, void* stream);
void al_norm_factor(const double* part, int parts, float max_norm, const float* max_dev,
                    float* out, void* stream);
void al_scale_by_factor(int type, const void* batch, const float* norm_factor, void* stream);
void al_sgd_step_multi_clip(const void* table, int nchunks, float lr, float momentum, float wd,
                            const float* hyper, const float* norm_factor, int zero_grad,
                            void* stream);
void al_sgd_step_clip(float* p, const float* g, float* buf, float lr, float momentum, float wd,
                      const float* hyper, long n, void* shadow, const float* norm_factor,
                      void* stream);
void al_adam_step_clip(float* p, const float* g, float* m, float* v, float lr, float b1, float b2,
                       float eps, float wd, float bc1, float bc2, long n,
                       const float* norm_factor, void* stream);
}

namespace {

constexpr long kBlock = 128;    // values that share a scale
constexpr long kFewRows = 16;   // the most rows that need no quantised copy

void* cur_stream() { return (void*)c10::hip::getCurrentHIPStream().stream(); }

void check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  TORCH_CHECK(e == hipSuccess, what, ": ", hipGetErrorString(e));
}

int type_of(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case torch::kBFloat16: return 0;
    case torch::kFloat16: return 1;
    case torch::kFloat32: return 2;
    default: TORCH_CHECK_TYPE(false, name, " must be bfloat16, float16 or float32, got ", t.scalar_type());
  }
}

// a matrix with its last axis dense, on x's device
void check_rows(const Tensor& t, const char* name, const Tensor& x) {
  TORCH_CHECK(t.is_cuda() && t.device() == x.device(), name, " must be on ", x.device());
  TORCH_CHECK(t.dim() == 2, name, " must have two axes");
  TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == 1, name, " must be dense along its last axis");
  TORCH_CHECK(t.size(1) <= INT_MAX - kBlock, name, " has too long rows");
}

long row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
long blocks_of(long n) { return (n + kBlock - 1) / kBlock; }

// A tensor on like's device, from the allocator without a dispatch: calls as short as
// these feel the difference (one row's norm to e4m3 5.1 us instead of 5.7).
Tensor fresh(torch::IntArrayRef shape, torch::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(shape, type, like.device(), std::nullopt);
}

// storage of e4m3 codes: rows of whole blocks
Tensor new_codes(const Tensor& like, long rows, long cols) {
  return fresh({rows, blocks_of(cols) * kBlock}, torch::kFloat8_e4m3fn, like);
}
// storage of scales: rows of whole fours, since the products read them four at a time
Tensor new_scales(const Tensor& like, long rows, long cols, long kind) {
  return fresh({rows, (blocks_of(cols) + 3) / 4 * 4}, kind == 0 ? torch::kFloat8_e8m0fnu : torch::kFloat32, like);
}

const Tensor& value(const OptTensor& t) { return *t; }

void check_norm(const Tensor& x, const Tensor& w, const OptTensor& res, double eps) {
  type_of(x, "input");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, "the norm needs a last axis of at least one value");
  // a row's places are counted in 32 bits, up to a whole sweep of a workgroup behind its end
  TORCH_CHECK_VALUE(x.size(-1) <= 1 << 30, "the last axis is too long: ", x.size(-1), " values, at most 2^30");
  TORCH_CHECK_VALUE(w.dim() == 1 && w.size(0) == x.size(-1), "weight has shape ", w.sizes(), ", not [",
                    x.size(-1), "]");
  TORCH_CHECK_TYPE(w.scalar_type() == torch::kFloat32 || w.scalar_type() == x.scalar_type(),
                   "weight must be float32 or ", x.scalar_type(), ", got ", w.scalar_type());
  TORCH_CHECK_VALUE(w.device() == x.device(), "weight is on ", w.device(), ", the input on ", x.device());
  if (res) {
    TORCH_CHECK_VALUE(value(res).sizes() == x.sizes() && value(res).scalar_type() == x.scalar_type(),
                      "residual must have the input's shape and type: ", value(res).sizes(), " ",
                      value(res).scalar_type(), ", not ", x.sizes(), " ", x.scalar_type());
    TORCH_CHECK_VALUE(value(res).device() == x.device(), "residual is on ", value(res).device(),
                      ", the input on ", x.device());
  }
  TORCH_CHECK_VALUE((float)eps > 0, "eps must be positive, got ", eps);
}

// (rows, last axis) with a dense last axis; a view wherever there is one
Tensor as_rows(const Tensor& t) {
  if (!t.numel()) {  // what is empty counts as dense, whatever its strides
    long rows = 1;
    for (int64_t i = 0; i + 1 < t.dim(); ++i) rows *= t.size(i);
    return fresh({rows, t.size(-1)}, t.scalar_type(), t);
  }
  if (t.dim() == 2 && (t.stride(1) == 1 || t.size(1) == 1)) return t;
  const Tensor r = t.reshape({-1, t.size(-1)});
  return r.size(1) == 1 || r.stride(1) == 1 ? r : r.contiguous();
}

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

// A dual tensor (forward-mode differentiation) need not ask for a gradient: its output
// without a tangent would read as a derivative of zero.
void no_tangent(const char* name, const Tensor& x, const OptTensor& y = std::nullopt,
                const OptTensor& z = std::nullopt) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  const auto dual = [](const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); };
  TORCH_CHECK_NOT_IMPLEMENTED(!dual(x) && !(y && dual(*y)) && !(z && dual(*z)), name,
                              " has no forward-mode derivative");
}

// A gradient that has none of its own though what it depends on asks for one (`asked`):
// where it is to be differentiable, differentiating it raises.
Tensor once(const Tensor& grad, bool asked, const char* name) {
  if (!grad.defined() || !asked || !torch::GradMode::is_enabled()) return grad;
  auto stop = std::make_shared<torch::autograd::DelayedError>(
      std::string(name) + " is differentiable once: its backward pass has no gradient", 1);
  return (*stop)({grad.detach().requires_grad_()})[0];
}

struct NormOut {
  Tensor y, total, rstd;
};

// rows of a checked input, as outputs of the given shape; rstd only where it is asked for
NormOut norm_rows(const Tensor& x, const Tensor& w, const OptTensor& res, double eps, bool need_rstd,
                  torch::IntArrayRef shape) {
  const long rows = x.size(0), dim = x.size(1);
  NormOut o;
  o.y = fresh(shape, x.scalar_type(), x);
  if (res) o.total = fresh(shape, x.scalar_type(), x);
  if (need_rstd) o.rstd = fresh({rows}, torch::kFloat32, x);
  if (rows) {
    al_rms_fwd(type_of(x, "input"), type_of(w, "weight"), x.data_ptr(), row_stride(x),
               res ? value(res).data_ptr() : nullptr, res ? row_stride(value(res)) : 0, w.data_ptr(),
               o.y.data_ptr(), res ? o.total.data_ptr() : nullptr,
               need_rstd ? o.rstd.data_ptr<float>() : nullptr, nullptr, nullptr, 0, rows, (int)dim, 0, 0,
               (float)eps, cur_stream());
    check_launch("rms_norm");
  }
  return o;
}

// (dx, dw): dw is undefined where it is not asked for
std::pair<Tensor, Tensor> norm_rows_bwd(const Tensor& s, const Tensor& w, const Tensor& rstd,
                                        const Tensor& dy, const Tensor& dsum, bool need_dw) {
  const long rows = s.size(0), dim = s.size(1);
  Tensor dx = fresh({rows, dim}, s.scalar_type(), s), dw, part;
  if (need_dw) dw = rows ? fresh({dim}, w.scalar_type(), w) : torch::zeros({dim}, w.options());
  if (!rows) return {dx, dw};
  const int parts = al_rms_bwd_parts(type_of(s, "input"), rows, (int)dim);
  if (need_dw) part = fresh({parts, dim}, torch::kFloat32, s);
  al_rms_bwd(type_of(s, "input"), type_of(w, "weight"), s.data_ptr(), row_stride(s), dy.data_ptr(),
             dsum.defined() ? dsum.data_ptr() : nullptr, w.data_ptr(), rstd.data_ptr<float>(),
             dx.data_ptr(), need_dw ? part.data_ptr<float>() : nullptr,
             need_dw ? dw.data_ptr() : nullptr, parts, rows, (int)dim, cur_stream());
  check_launch("rms_norm backward");
  return {dx, dw};
}

enum : int64_t { kResidual = 1, kRowsAsk = 2, kWeightAsks = 4 };

struct RmsNorm : public torch::autograd::Function<RmsNorm> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x,
                                                const Tensor& w, const OptTensor& res, double eps) {
    ctx->set_materialize_grads(false);
    c10::OptionalDeviceGuard guard(x.device());
    const Tensor rows = as_rows(x);
    const NormOut o = norm_rows(rows, w, res ? OptTensor(as_rows(*res)) : res, eps, true, x.sizes());
    // the sum as it goes out, not a view of it: a change in place is noticed
    ctx->save_for_backward({res ? o.total : rows, w, o.rstd});
    // which inputs ask for a gradient, whichever of them a backward pass is for
    const bool rows_ask = wants_grad(x) || (res && wants_grad(*res));
    ctx->saved_data["what"] = (res ? kResidual : 0) | (rows_ask ? kRowsAsk : 0) | (wants_grad(w) ? kWeightAsks : 0);
    if (!res) return {o.y};
    return {o.y, o.total};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor total = as_rows(saved[0]), &w = saved[1], &rstd = saved[2];
    const int64_t what = ctx->saved_data["what"].toInt();
    const bool res = what & kResidual;
    const bool need_w = ctx->needs_input_grad(1);
    Tensor dy = grads[0], dsum = res ? grads[1] : Tensor();
    c10::OptionalDeviceGuard guard(total.device());
    Tensor dx, dw;
    if (!dy.defined()) {  // only the sum was used
      dx = dsum;
      if (need_w) dw = torch::zeros_like(w);
    } else {
      const auto shape = dy.sizes().vec();
      dy = dy.reshape(total.sizes()).contiguous();
      if (dsum.defined()) dsum = dsum.reshape(total.sizes()).contiguous();
      std::tie(dx, dw) = norm_rows_bwd(total, w, rstd, dy, dsum, need_w);
      dx = dx.view(shape);
    }
    const bool need_x = ctx->needs_input_grad(0), need_r = res && ctx->needs_input_grad(2);
    if (grads[0].defined()) {  // otherwise dx is the sum's gradient itself
      const bool outer = wants_grad(grads[0]) || (res && wants_grad(grads[1]));
      dx = once(dx, outer || what & (kRowsAsk | kWeightAsks), "rms_norm");
      dw = once(dw, outer || what & kRowsAsk, "rms_norm");
    }
    return {need_x ? dx : Tensor(), dw, need_r ? dx : Tensor(), Tensor()};
  }
};

// y, or y and the stored sum where there is a residual
std::vector<Tensor> rms_norm(const Tensor& x, const Tensor& w_in, const OptTensor& res, double eps) {
  check_norm(x, w_in, res, eps);
  no_tangent("rms_norm", x, w_in, res);
  const Tensor w = w_in.contiguous();
  if (torch::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || (res && wants_grad(*res))))
    return RmsNorm::apply(x, w, res, eps);
  c10::OptionalDeviceGuard guard(x.device());
  const NormOut o = norm_rows(as_rows(x), w, res ? OptTensor(as_rows(*res)) : res, eps, false, x.sizes());
  if (!res) return {o.y};
  return {o.y, o.total};
}

// (codes, scales, stored sum)
std::vector<Tensor> rms_norm_quant(const Tensor& x_in, const Tensor& w_in, const OptTensor& res_in,
                                   double eps, long kind) {
  check_norm(x_in, w_in, res_in, eps);
  no_tangent("rms_norm_fp8", x_in, w_in, res_in);
  TORCH_CHECK(!torch::GradMode::is_enabled() ||
                  !(wants_grad(x_in) || wants_grad(w_in) || (res_in && wants_grad(*res_in))),
              "rms_norm_fp8 has no gradient: use rms_norm and fp8_linear to train, or torch.no_grad()");
  c10::OptionalDeviceGuard guard(x_in.device());
  const Tensor x = as_rows(x_in), w = w_in.contiguous();
  const OptTensor res = res_in ? OptTensor(as_rows(*res_in)) : res_in;
  const long rows = x.size(0), dim = x.size(1);
  Tensor q = new_codes(x, rows, dim), scale = new_scales(x, rows, dim, kind);
  Tensor total = res ? fresh({rows, dim}, x.scalar_type(), x) : x;
  if (rows) {
    al_rms_fwd(type_of(x, "input"), type_of(w, "weight"), x.data_ptr(), row_stride(x),
               res ? value(res).data_ptr() : nullptr, res ? row_stride(value(res)) : 0, w.data_ptr(),
               nullptr, res ? total.data_ptr() : nullptr, nullptr, q.data_ptr(), scale.data_ptr(),
               kind == 0 ? 1 : 2, rows, (int)dim, (int)q.size(1), (int)scale.size(1), (float)eps,
               cur_stream());
    check_launch("rms_norm_fp8");
  }
  return {q, scale, res ? total.view(x_in.sizes()) : total};
}

// (codes, scales) of 1x128 blocks; any strides
std::vector<Tensor> fp8_quant_rows(const Tensor& x, long kind) {
  const int type = type_of(x, "input");
  TORCH_CHECK(x.is_cuda() && x.dim() == 2, "input must be a matrix on the GPU");
  c10::OptionalDeviceGuard guard(x.device());
  const long rows = x.size(0), dim = x.size(1);
  TORCH_CHECK(dim <= INT_MAX - kBlock, "input has too long rows");
  Tensor q = new_codes(x, rows, dim), scale = new_scales(x, rows, dim, kind);
  if (rows && dim) {
    al_quant_rows(type, (int)kind, x.data_ptr(), x.stride(0), dim > 1 ? x.stride(1) : 1, q.data_ptr(),
                  scale.data_ptr(), rows, (int)dim, (int)q.size(1), (int)scale.size(1), cur_stream());
    check_launch("quantize_fp8");
  }
  return {q, scale};
}

// (codes, scales, transposed codes, transposed scales, column sums), each empty
// where it is not asked for
std::vector<Tensor> fp8_quant_tile(const Tensor& x, long kind, bool tile, bool plain, bool transposed,
                                   std::optional<torch::ScalarType> sums) {
  const int type = type_of(x, "input");
  check_rows(x, "input", x);
  c10::OptionalDeviceGuard guard(x.device());
  const long rows = x.size(0), cols = x.size(1);
  TORCH_CHECK_VALUE(rows <= INT_MAX - kBlock && blocks_of(rows) * blocks_of(cols) <= INT_MAX - 1024,
                    "a matrix of ", rows, " x ", cols, " is too large");
  Tensor none = fresh({0}, torch::kFloat32, x);
  Tensor q = none, scale = none, qt = none, scale_t = none, part, sum = none;
  if (plain) {
    q = new_codes(x, rows, cols);
    scale = new_scales(x, tile ? blocks_of(rows) : rows, cols, kind);
  }
  if (transposed) {
    qt = new_codes(x, cols, rows);
    scale_t = new_scales(x, tile ? blocks_of(cols) : cols, rows, kind);
  }
  if (sums) sum = fresh({cols}, *sums, x);
  if (!rows || !cols) {
    if (sums) sum.zero_();
    return {q, scale, qt, scale_t, sum};
  }
  if (sums) part = fresh({blocks_of(rows), cols}, torch::kFloat64, x);
  al_quant_tile(type, (int)kind, tile, x.data_ptr(), row_stride(x), (int)rows, (int)cols,
                plain ? q.data_ptr() : nullptr, plain ? scale.data_ptr() : nullptr,
                plain ? (int)q.size(1) : 0, plain ? (int)scale.size(1) : 0,
                transposed ? qt.data_ptr() : nullptr, transposed ? scale_t.data_ptr() : nullptr,
                transposed ? (int)qt.size(1) : 0, transposed ? (int)scale_t.size(1) : 0,
                sums ? part.data_ptr<double>() : nullptr, cur_stream());
  if (sums)
    al_col_sum(part.data_ptr<double>(), sum.data_ptr(), type_of(sum, "sum"), (int)part.size(0),
               (int)cols, cur_stream());
  check_launch("quantize_fp8");
  return {q, scale, qt, scale_t, sum};
}

int kind_of(const Tensor& scale) { return scale.scalar_type() == torch::kFloat8_e8m0fnu ? 0 : 1; }

void check_codes(const Tensor& q, const Tensor& s, long rows, long cols, bool tile, const char* name) {
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == torch::kFloat8_e4m3fn && q.dim() == 2 &&
                  q.is_contiguous() && q.size(0) == rows && q.size(1) == blocks_of(cols) * kBlock &&
                  (uintptr_t)q.data_ptr() % 16 == 0, name, " codes are not laid out as blocks");
  TORCH_CHECK(s.device() == q.device() && s.is_contiguous() && s.dim() == 2 &&
                  (s.scalar_type() == torch::kFloat32 || s.scalar_type() == torch::kFloat8_e8m0fnu) &&
                  s.size(0) == (tile ? blocks_of(rows) : rows) && s.size(1) >= blocks_of(cols) &&
                  s.size(1) % 4 == 0 && (uintptr_t)s.data_ptr() % (kind_of(s) ? 16 : 4) == 0,
              name, " scales are not laid out as blocks");
  // a workgroup addresses its 256 rows with 32 bits
  TORCH_CHECK(rows <= INT_MAX && cols <= (1 << 23), name, " matrix has too many rows or too long ones");
}

void check_bias(const OptTensor& bias, long n, const Tensor& like) {
  if (!bias) return;
  type_of(value(bias), "bias");
  TORCH_CHECK_VALUE(value(bias).device() == like.device() && value(bias).dim() == 1 && value(bias).size(0) == n &&
                  value(bias).is_contiguous(),
              "bias must be a dense vector of one value for each output column, on the operands' device");
}

// [m, n], or that in the given shape: outputs of a differentiable function are no
// views, so that they may be changed in place
Tensor fp8_gemm_as(const Tensor& a, const Tensor& sa, const Tensor& b, const Tensor& sb, bool b_tile,
                   long m, long n, long k, const OptTensor& bias, torch::ScalarType out_type,
                   torch::IntArrayRef shape) {
  check_codes(a, sa, m, k, false, "left operand's");
  check_codes(b, sb, n, k, b_tile, "right operand's");
  TORCH_CHECK(a.device() == b.device(), "operands must be on one device");
  TORCH_CHECK(kind_of(sa) == kind_of(sb), "operands must have scales of one type");
  check_bias(bias, n, a);
  // tiles are counted in 32 bits, and a launch has at most 2^32 threads
  TORCH_CHECK_VALUE((m + 63) / 64 * ((n + 63) / 64) <= (1 << 23), "a product of ", m, " x ", n, " is too large");
  c10::OptionalDeviceGuard guard(a.device());
  Tensor out = fresh(shape, out_type, a);
  const int ot = type_of(out, "output"), blocks = (int)blocks_of(k);
  if (!m || !n) return out;
  if (!k) {  // sums of nothing
    out.zero_();
    if (bias) out.view({m, n}).add_(value(bias));
    return out;
  }
  const int splits = al_fp8_gemm_splits(kind_of(sa), ot, (int)m, (int)n, blocks);
  Tensor split;
  if (splits > 1) split = fresh({splits, m, n}, torch::kFloat32, a);
  al_fp8_gemm(kind_of(sa), a.data_ptr(), sa.data_ptr(), a.size(1), (int)sa.size(1), b.data_ptr(),
              sb.data_ptr(), b.size(1), (int)sb.size(1), b_tile, (int)m, (int)n, blocks,
              bias ? value(bias).data_ptr() : nullptr, bias ? type_of(value(bias), "bias") : 0,
              out.data_ptr(), ot, splits > 1 ? split.data_ptr<float>() : nullptr, splits, cur_stream());
  check_launch("fp8_matmul");
  return out;
}
Tensor fp8_gemm(const Tensor& a, const Tensor& sa, const Tensor& b, const Tensor& sb, bool b_tile,
                long m, long n, long k, const OptTensor& bias, torch::ScalarType out_type) {
  return fp8_gemm_as(a, sa, b, sb, b_tile, m, n, k, bias, out_type, {m, n});
}

// x [m <= 16, k] in its own type times the blocks of b
Tensor fp8_few_rows(const Tensor& x, const Tensor& b, const Tensor& sb, bool b_tile, long n,
                    const OptTensor& bias) {
  const int type = type_of(x, "input");
  check_rows(x, "input", b);
  const long m = x.size(0), k = x.size(1);
  check_codes(b, sb, n, k, b_tile, "weight's");
  TORCH_CHECK(m <= 16, "at most 16 rows");
  check_bias(bias, n, x);
  c10::OptionalDeviceGuard guard(x.device());
  Tensor out = fresh({m, n}, x.scalar_type(), x);
  TORCH_CHECK_VALUE(k > 0, "x needs a last axis of at least one value");
  TORCH_CHECK_VALUE(n < 1 << 29, "a weight of ", n, " rows is too large");  // 2^32 threads
  if (!m || !n) return out;
  al_fp8_few_rows(kind_of(sb), type, x.data_ptr(), row_stride(x), (int)k, b.data_ptr(), sb.data_ptr(),
                  b.size(1), (int)sb.size(1), b_tile, (int)m, (int)n, (int)blocks_of(k),
                  bias ? value(bias).data_ptr() : nullptr, bias ? type_of(value(bias), "bias") : 0,
                  out.data_ptr(), cur_stream());
  check_launch("fp8_linear");
  return out;
}

// y = Q(x) Q(w)^T + b,  dx = Q(dy) Q(w),  dw = Q(dy^T) Q(x^T)^T: each operand in
// blocks along its product's contraction. The weight's tiles are the same for both
// of its products.
struct Fp8Linear : public torch::autograd::Function<Fp8Linear> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& w,
                        const OptTensor& bias, long kind, bool need_x, bool need_w) {
    c10::OptionalDeviceGuard guard(x.device());
    const Tensor rows = as_rows(x), wr = as_rows(w);
    const long m = rows.size(0), k = rows.size(1), n = wr.size(0);
    const auto xq = fp8_quant_tile(rows, kind, false, true, need_w, std::nullopt);
    const auto wq = fp8_quant_tile(wr, kind, true, true, need_x, std::nullopt);
    ctx->save_for_backward({xq[2], xq[3], wq[2], wq[3]});
    ctx->saved_data["k"] = k;
    ctx->saved_data["kind"] = kind;
    ctx->saved_data["asks"] = (need_x ? kRowsAsk : 0) | (need_w ? kWeightAsks : 0);
    ctx->saved_data["w"] = (int64_t)w.scalar_type();
    ctx->saved_data["x"] = (int64_t)x.scalar_type();
    ctx->saved_data["bias"] = bias ? (int64_t)value(bias).scalar_type() : -1;
    auto shape = x.sizes().vec();
    shape.back() = n;
    return fp8_gemm_as(xq[0], xq[1], wq[0], wq[1], true, m, n, k, bias, x.scalar_type(), shape);
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    const long k = ctx->saved_data["k"].toInt(), kind = ctx->saved_data["kind"].toInt();
    const int64_t bias = ctx->saved_data["bias"].toInt();
    const bool need_b = bias >= 0 && ctx->needs_input_grad(2);
    c10::OptionalDeviceGuard guard(grads[0].device());
    const Tensor dy = as_rows(grads[0]);
    const long m = dy.size(0), n = dy.size(1);
    const auto dq = fp8_quant_tile(dy, kind, false, need_x, need_w,
                                   need_b ? std::optional((torch::ScalarType)bias) : std::nullopt);
    Tensor dx, dw;
    if (need_x) {
      auto shape = grads[0].sizes().vec();
      shape.back() = k;
      dx = fp8_gemm(dq[0], dq[1], saved[2], saved[3], true, m, k, n, std::nullopt,
                    (torch::ScalarType)ctx->saved_data["x"].toInt()).view(shape);
    }
    if (need_w)
      dw = fp8_gemm(dq[2], dq[3], saved[0], saved[1], false, n, k, m, std::nullopt,
                    (torch::ScalarType)ctx->saved_data["w"].toInt());
    const bool outer = wants_grad(grads[0]);
    const int64_t asks = ctx->saved_data["asks"].toInt();
    return {once(dx, outer || asks & kWeightAsks, "fp8_linear"), once(dw, outer || asks & kRowsAsk, "fp8_linear"),
            need_b ? once(dq[4], outer, "fp8_linear") : Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

void check_linear(const Tensor& x, long n, long k, const OptTensor& bias, const Tensor& like) {
  type_of(x, "x");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, "x needs a last axis of at least one value");
  TORCH_CHECK_VALUE(x.size(-1) == k, "the operands' rows are ", x.size(-1), " and ", k, " values long");
  TORCH_CHECK_VALUE(x.device() == like.device(), "the operands are on ", x.device(), " and ", like.device());
  check_bias(bias, n, like);
}

// x times a weight, quantised here
Tensor fp8_linear(const Tensor& x, const Tensor& w, const OptTensor& bias_in, long kind) {
  type_of(w, "weight");
  TORCH_CHECK_TYPE(w.dim() == 2, "weight must be a matrix");
  const OptTensor bias = bias_in ? OptTensor(bias_in->contiguous()) : bias_in;
  check_linear(x, w.size(0), w.size(1), bias, w);
  no_tangent("fp8_linear", x, w, bias);
  TORCH_CHECK_VALUE(x.is_cuda(), "x must be on the GPU");
  const bool grad = torch::GradMode::is_enabled();
  const bool need_x = grad && x.requires_grad(), need_w = grad && w.requires_grad();
  if (need_x || need_w || (grad && bias && bias->requires_grad()))
    return Fp8Linear::apply(x, w, bias, kind, need_x, need_w);
  c10::OptionalDeviceGuard guard(x.device());
  const Tensor rows = as_rows(x);
  const auto xq = fp8_quant_rows(rows, kind);
  const auto wq = fp8_quant_tile(as_rows(w), kind, true, true, false, std::nullopt);
  auto shape = x.sizes().vec();
  shape.back() = w.size(0);
  return fp8_gemm(xq[0], xq[1], wq[0], wq[1], true, rows.size(0), w.size(0), w.size(1), bias,
                  x.scalar_type()).view(shape);
}

// x times a weight that is kept in blocks
Tensor fp8_linear_kept(const Tensor& x, const Tensor& b, const Tensor& sb, bool b_tile, long n, long k,
                       const OptTensor& bias_in) {
  const OptTensor bias = bias_in ? OptTensor(bias_in->contiguous()) : bias_in;
  check_linear(x, n, k, bias, b);
  no_tangent("fp8_linear", x, bias);
  TORCH_CHECK(!torch::GradMode::is_enabled() || !(x.requires_grad() || (bias && bias->requires_grad())),
              "a weight kept in Fp8Blocks has no gradient: pass the weight itself to train, or use "
              "torch.no_grad()");
  c10::OptionalDeviceGuard guard(x.device());
  const Tensor rows = as_rows(x);
  auto shape = x.sizes().vec();
  shape.back() = n;
  if (rows.size(0) <= kFewRows) return fp8_few_rows(rows, b, sb, b_tile, n, bias).view(shape);
  const auto xq = fp8_quant_rows(rows, kind_of(sb));
  return fp8_gemm(xq[0], xq[1], b, sb, b_tile, rows.size(0), n, k, bias, x.scalar_type()).view(shape);
}

// Batches of tensors of one type for the kernels that take many at once.
struct Batches {
  std::vector<std::vector<char>> batch;
  std::vector<int> type;
  void add(const Tensor& t) {
    const int ty = type_of(t, "gradient");
    if (!t.numel()) return;
    for (size_t i = 0; i < batch.size(); ++i)
      if (type[i] == ty && al_norm_batch_add(batch[i].data(), t.data_ptr(), t.numel())) return;
    batch.emplace_back(al_norm_batch_bytes());
    type.push_back(ty);
    al_norm_batch_clear(batch.back().data());
    al_norm_batch_add(batch.back().data(), t.data_ptr(), t.numel());
  }
};

// what the values of a tensor occupy, without gaps and each once, in any order
bool dense(const Tensor& t) { return t.is_non_overlapping_and_dense(); }

// each tensor once, however often it is listed
std::vector<Tensor> distinct(const std::vector<Tensor>& tensors) {
  std::vector<Tensor> kept;
  std::unordered_set<const void*> seen;
  seen.reserve(tensors.size() * 2);
  for (const Tensor& t : tensors)
    if (t.defined() && seen.insert(t.unsafeGetTensorImpl()).second) kept.push_back(t);
  return kept;
}

std::vector<Tensor> grads_of(const std::vector<Tensor>& params) {
  std::vector<Tensor> grads;
  grads.reserve(params.size());
  for (const Tensor& p : params) grads.push_back(p.grad());
  return distinct(grads);
}

// [norm, factor] of distinct tensors, in `to` where it is given; max_dev, where given,
// holds the bound on the device
Tensor norm_factor(const std::vector<Tensor>& grads, double max_norm, const OptTensor& max_dev,
                   const OptTensor& to) {
  const Tensor& first = grads[0];
  c10::OptionalDeviceGuard guard(first.device());
  Batches all;
  std::vector<Tensor> kept;  // copies of what is not dense
  for (const Tensor& g : grads) {
    TORCH_CHECK_VALUE(g.is_cuda() && g.device() == first.device(), "gradients are on ", first.device(),
                      " and ", g.device());
    TORCH_CHECK_TYPE(g.layout() == torch::kStrided, "sparse gradients have no norm here");
    if (dense(g)) { all.add(g); continue; }
    kept.push_back(g.contiguous());
    all.add(kept.back());
  }
  int parts = 0;
  for (auto& b : all.batch) parts += al_norm_blocks(b.data());
  Tensor part = fresh({std::max(parts, 1)}, torch::kFloat64, first);
  if (to)
    TORCH_CHECK(value(to).device() == first.device() && value(to).numel() == 2 && value(to).is_contiguous() &&
                    value(to).scalar_type() == torch::kFloat32, "norm and factor");
  Tensor out = to ? value(to) : fresh({2}, torch::kFloat32, first);
  int at = 0;
  for (size_t i = 0; i < all.batch.size(); ++i) {
    al_sq_sum(all.type[i], all.batch[i].data(), part.data_ptr<double>() + at, cur_stream());
    at += al_norm_blocks(all.batch[i].data());
  }
  al_norm_factor(part.data_ptr<double>(), parts, (float)max_norm,
                 max_dev ? value(max_dev).data_ptr<float>() : nullptr, out.data_ptr<float>(), cur_stream());
  check_launch("grad_norm");
  return out;
}

Tensor grad_norm_factor(const std::vector<Tensor>& tensors, double max_norm, const OptTensor& max_dev) {
  return norm_factor(distinct(tensors), max_norm, max_dev, std::nullopt);
}

Tensor params_norm_factor(const std::vector<Tensor>& params, double max_norm, const OptTensor& max_dev,
                          const OptTensor& to) {
  return norm_factor(grads_of(params), max_norm, max_dev, to);
}

// the parameters' gradients times the factor, in place
void scale_grads(const std::vector<Tensor>& params, const Tensor& norm_factor) {
  TORCH_CHECK(norm_factor.is_cuda() && norm_factor.numel() == 2 && norm_factor.scalar_type() == torch::kFloat32 &&
                  norm_factor.is_contiguous(), "norm and factor");
  c10::OptionalDeviceGuard guard(norm_factor.device());
  Batches all;
  std::vector<std::pair<Tensor, Tensor>> copies;
  std::vector<std::pair<uintptr_t, uintptr_t>> spans;
  const std::vector<Tensor> grads = grads_of(params);
  for (const Tensor& g : grads) {
    TORCH_CHECK(g.is_cuda() && g.device() == norm_factor.device(), "gradients must be on one GPU");
    TORCH_CHECK(at::has_internal_overlap(g) != at::MemOverlap::Yes,
                "a gradient whose values share memory cannot be scaled in place");
    Tensor at = g;
    if (!dense(g)) {
      copies.emplace_back(g, g.contiguous());
      at = copies.back().second;
    } else if (g.numel()) {
      const uintptr_t p = (uintptr_t)g.data_ptr();
      spans.emplace_back(p, p + g.numel() * g.element_size());
    }
    all.add(at);
  }
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    TORCH_CHECK(spans[i].first >= spans[i - 1].second, "gradients that share memory cannot be scaled in place");
  for (size_t i = 0; i < all.batch.size(); ++i)
    al_scale_by_factor(all.type[i], all.batch[i].data(), norm_factor.data_ptr<float>(), cur_stream());
  check_launch("clip_grad_norm_");
  for (auto& c : copies) c.first.copy_(c.second);
  for (const Tensor& g : grads) g.unsafeGetTensorImpl()->bump_version();
}

// whether the multi-tensor step can take all of these parameters
bool sgd_fusable(const std::vector<Tensor>& params) {
  for (const Tensor& p : params) {
    const Tensor& g = p.grad();
    if (!p.is_cuda() || p.scalar_type() != torch::kFloat32 || !p.is_contiguous() || !g.defined() ||
        g.scalar_type() != torch::kFloat32 || !g.is_contiguous() || g.device() != p.device())
      return false;
  }
  return true;
}

// what an update reads and writes beside a parameter, value for value
void check_state(const Tensor& p, const Tensor& t, const char* name, torch::ScalarType type = torch::kFloat32) {
  TORCH_CHECK_VALUE(t.scalar_type() == type && t.is_contiguous() && t.numel() == p.numel() && t.device() == p.device(),
                    name, " must be a dense ", type, " tensor like its parameter: ", t.sizes(), " ", t.scalar_type(),
                    " on ", t.device(), ", the parameter is ", p.sizes(), " on ", p.device());
}

// five words a parameter: the addresses of its values, gradient, momentum and bf16
// copy (0: none), and its length
py::bytes sgd_addresses(const std::vector<Tensor>& params, const std::vector<OptTensor>& bufs,
                        const std::vector<OptTensor>& shadows) {
  TORCH_CHECK(bufs.size() == params.size() && shadows.size() == params.size(), "one of each a parameter");
  std::vector<int64_t> words;
  words.reserve(params.size() * 5);
  for (size_t i = 0; i < params.size(); ++i) {
    if (bufs[i]) check_state(params[i], *bufs[i], "momentum_buffer");
    if (shadows[i]) check_state(params[i], *shadows[i], "the bf16 copy", torch::kBFloat16);
    words.push_back((int64_t)params[i].data_ptr());
    words.push_back((int64_t)params[i].grad().data_ptr());
    words.push_back(bufs[i] ? (int64_t)bufs[i]->data_ptr() : 0);
    words.push_back(shadows[i] ? (int64_t)shadows[i]->data_ptr() : 0);
    words.push_back(params[i].numel());
  }
  return py::bytes((const char*)words.data(), words.size() * 8);
}

const float* hyper_of(const OptTensor& h) {
  if (!h) return nullptr;
  TORCH_CHECK(value(h).is_cuda() && value(h).numel() >= 3 && value(h).scalar_type() == torch::kFloat32, "hyper");
  return value(h).data_ptr<float>();
}

const float* factor_of(const Tensor& f) {
  TORCH_CHECK(f.is_cuda() && f.numel() == 2 && f.scalar_type() == torch::kFloat32 && f.is_contiguous(),
              "norm and factor must be two floats on the GPU");
  return f.data_ptr<float>();
}

void sgd_step_multi_clip(const Tensor& table, int64_t nchunks, double lr, double momentum, double wd,
                         const OptTensor& hyper, const Tensor& norm_factor, bool zero_grad) {
  TORCH_CHECK(table.is_cuda() && table.scalar_type() == torch::kInt64 && table.is_contiguous(), "chunk table");
  c10::OptionalDeviceGuard guard(table.device());
  al_sgd_step_multi_clip(table.data_ptr<int64_t>(), (int)nchunks, (float)lr, (float)momentum, (float)wd,
                         hyper_of(hyper), factor_of(norm_factor), zero_grad, cur_stream());
  check_launch("SGD step");
}

void check_update(const Tensor& p, const Tensor& g, const char* what) {
  TORCH_CHECK(p.is_cuda() && p.scalar_type() == torch::kFloat32 && p.is_contiguous() &&
                  g.scalar_type() == torch::kFloat32 && g.is_contiguous() && g.numel() == p.numel() &&
                  g.device() == p.device(), what, ": float32 parameters and gradients, dense");
}

void sgd_step_clip(Tensor& p, const Tensor& g, Tensor& buf, double lr, double momentum, double wd,
                   const OptTensor& hyper, Tensor& shadow, const Tensor& norm_factor) {
  check_update(p, g, "SGD step");
  if (!p.numel()) return;
  if (buf.numel()) check_state(p, buf, "momentum_buffer");
  if (shadow.numel()) check_state(p, shadow, "the bf16 copy", torch::kBFloat16);
  c10::OptionalDeviceGuard guard(p.device());
  al_sgd_step_clip(p.data_ptr<float>(), g.data_ptr<float>(), buf.numel() ? buf.data_ptr<float>() : nullptr,
                   (float)lr, buf.numel() ? (float)momentum : 0.f, (float)wd, hyper_of(hyper), p.numel(),
                   shadow.numel() ? shadow.data_ptr() : nullptr, factor_of(norm_factor), cur_stream());
  check_launch("SGD step");
}

void adam_step_clip(Tensor& p, const Tensor& g, Tensor& m, Tensor& v, double lr, double b1, double b2,
                    double eps, double wd, double bc1, double bc2, const Tensor& norm_factor) {
  check_update(p, g, "Adam step");
  if (!p.numel()) return;
  check_state(p, m, "exp_avg");
  check_state(p, v, "exp_avg_sq");
  c10::OptionalDeviceGuard guard(p.device());
  al_adam_step_clip(p.data_ptr<float>(), g.data_ptr<float>(), m.data_ptr<float>(), v.data_ptr<float>(),
                    (float)lr, (float)b1, (float)b2, (float)eps, (float)wd, (float)bc1, (float)bc2, p.numel(),
                    factor_of(norm_factor), cur_stream());
  check_launch("Adam step");
}

}  // namespace

void register_head_ops(py::module_& m) {
  m.def("rms_norm", &rms_norm);
  m.def("rms_norm_quant", &rms_norm_quant);
  m.def("fp8_quant_rows", &fp8_quant_rows);
  m.def("fp8_quant_tile", &fp8_quant_tile);
  m.def("fp8_gemm", &fp8_gemm);
  m.def("fp8_linear", &fp8_linear);
  m.def("fp8_linear_kept", &fp8_linear_kept);
  m.def("grad_norm_factor", &grad_norm_factor);
  m.def("params_norm_factor", &params_norm_factor);
  m.def("scale_grads", &scale_grads);
  m.def("sgd_fusable", &sgd_fusable);
  m.def("sgd_addresses", &sgd_addresses);
  m.def("sgd_step_multi_clip", &sgd_step_multi_clip);
  m.def("sgd_step_clip", &sgd_step_clip);
  m.def("adam_step_clip", &adam_step_clip);
}
