// Argument checks, torch operators and Python bindings of the attention operators:
// masked attention (forward, backward, mask plans) and the per-head norm with
// rotation.  Every launch is on the caller's current stream of the tensors'
// device; workspaces come from the caching allocator on that stream.
//
// They are operators of torch's dispatcher (namespace bitscom_b200), so that traces, fake tensors
// and function transforms see them; the bindings call them through it, which costs
// less than a call through torch.ops.
#include "ops/attention_ops.h"

#include <ATen/cuda/CUDAContext.h>
#include <c10/core/InferenceMode.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>
#include <torch/library.h>

#include "kernels/attention.h"
#include "kernels/qk_norm_rotary.h"

namespace bitscom_b200 {
namespace {

using OptTensor = c10::optional<at::Tensor>;

DType float_type(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return kF32;
    case at::kBFloat16: return kBF16;
    case at::kHalf: return kF16;
    default:
      TORCH_CHECK_TYPE(false, "bitscom: ", name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
  }
}

bool has(const OptTensor& t) { return t && t->defined(); }

void same_device(const at::Tensor& t, const at::Tensor& like, const char* name) {
  TORCH_CHECK_VALUE(t.device() == like.device(), "bitscom: ", name, " is on ", t.device(), ", expected ", like.device());
}

int int_bytes(const at::Tensor& t, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, "bitscom: ", name,
                   " must be int32 or int64, got ", t.scalar_type());
  return t.scalar_type() == at::kLong ? 8 : 4;
}

// The operators have no forward-mode derivative: a tangent is refused, not dropped.
void no_tangents(std::initializer_list<OptTensor> tensors) {
  for (const auto& t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!has(t) || !t->_fw_grad(0).defined(),
                                "bitscom: the attention operators have no forward-mode derivative");
}

cudaStream_t stream_of(const at::Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------

// Whether the tensor-core kernels take these tensors (other forms: attention_simt.cu).
bool for_tensor_cores(const at::Tensor& q) {
  return q.scalar_type() != at::kFloat && q.size(3) % 8 == 0 && q.size(3) <= 128;
}

// A [B, H, S, D] tensor as the kernels read it: copied when its last dimension
// is not contiguous, and for the tensor maps of the tensor-core kernels also
// when a row does not start on a 16-byte boundary or a dimension is expanded.
at::Tensor rows_of(const at::Tensor& t) {
  bool fits = t.stride(3) == 1 || t.size(3) <= 1;
  if (fits && for_tensor_cores(t)) {
    fits = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    for (int i = 0; i < 3; ++i) fits = fits && (t.size(i) <= 1 || (t.stride(i) % 8 == 0 && t.stride(i) > 0));
  }
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}

// Strides of dimensions of one entry are never used, and may be anything: a tensor map wants them to be legal.
AttnTensor view_of(const at::Tensor& t) {
  const int64_t any = (t.size(3) + 7) / 8 * 8;
  const auto stride = [&](int i) { return t.size(i) <= 1 ? any : t.stride(i); };
  return {t.data_ptr(), stride(0), stride(1), stride(2)};
}

// New [B, H, S, D] tensor laid out [B, S, H, D], the order in which projections leave and take it.
at::Tensor tokens_first(const at::Tensor& like) {
  return at::empty({like.size(0), like.size(2), like.size(1), like.size(3)}, like.options()).transpose(1, 2);
}

void check_qkv(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v) {
  TORCH_CHECK_VALUE(q.is_cuda() && k.is_cuda() && v.is_cuda(), "bitscom: q, k and v must be CUDA tensors");
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && v.dim() == 4,
                    "bitscom: q, k and v must be [batch, heads, length, head size]");
  float_type(q, "q");
  TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                   "bitscom: q, k and v must have one dtype, got ", q.scalar_type(), ", ", k.scalar_type(), " and ",
                   v.scalar_type());
  same_device(k, q, "k");
  same_device(v, q, "v");
  TORCH_CHECK_VALUE(k.sizes() == v.sizes(), "bitscom: k and v must have one shape, got ", k.sizes(), " and ", v.sizes());
  TORCH_CHECK_VALUE(k.size(0) == q.size(0) && k.size(3) == q.size(3), "bitscom: q ", q.sizes(), " and k ", k.sizes(),
                    " must agree in batch and head size");
  TORCH_CHECK_VALUE(k.size(1) > 0 && q.size(1) % k.size(1) == 0, "bitscom: ", q.size(1),
                    " query heads are not a multiple of ", k.size(1), " key heads");
  TORCH_CHECK_VALUE(q.size(3) >= 1 && q.size(3) <= 256, "bitscom: head size must be 1 to 256, got ", q.size(3));
  TORCH_CHECK_VALUE(q.size(0) <= 65535 && q.size(1) <= 65535, "bitscom: at most 65535 batch entries and heads");
  TORCH_CHECK_VALUE(q.size(2) < (1 << 30) && k.size(2) < (1 << 30), "bitscom: lengths must be below 2^30");
}

// As the kernels read them, which is one after another.
OptTensor slopes_of(const OptTensor& t) { return has(t) ? OptTensor(t->contiguous()) : OptTensor(); }

// The kernels read a plan 16 bytes at a time.
OptTensor plan_of(const OptTensor& t) {
  return has(t) && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 != 0 ? OptTensor(t->clone()) : t;
}

// The tensors have to outlive the launch: `plan` and `slopes` are from plan_of() and slopes_of().
AttnParams params_of(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const OptTensor& plan,
                     const OptTensor& slopes, bool causal, double scale, double cap) {
  AttnParams p{};
  p.q = view_of(q);
  p.k = view_of(k);
  p.v = view_of(v);
  p.b = static_cast<int>(q.size(0));
  p.hq = static_cast<int>(q.size(1));
  p.hk = static_cast<int>(k.size(1));
  p.sq = static_cast<int>(q.size(2));
  p.sk = static_cast<int>(k.size(2));
  p.d = static_cast<int>(q.size(3));
  p.causal = causal;
  p.scale = static_cast<float>(scale);
  p.cap = static_cast<float>(cap);
  p.splits = 1;
  p.dt = float_type(q, "q");
  if (has(slopes)) {
    same_device(*slopes, q, "slopes");
    TORCH_CHECK_TYPE(slopes->scalar_type() == at::kFloat, "bitscom: slopes must be float32");
    TORCH_CHECK_VALUE(slopes->dim() == 1 && slopes->size(0) == q.size(1),
                      "bitscom: slopes must be a vector of one value for each of the ", q.size(1), " query heads");
    p.slopes = slopes->data_ptr<float>();
  }
  if (has(plan)) {
    same_device(*plan, q, "mask");
    TORCH_CHECK_VALUE(plan->scalar_type() == at::kInt && plan->is_contiguous() &&
                          plan->numel() == PlanView::words(p.b, p.sq, p.sk),
                      "bitscom: the mask was built for other sizes");
    p.plan = PlanView::of(plan->data_ptr<int>(), p.b, p.sq, p.sk);
  }
  return p;
}

at::Tensor attention_plan(const OptTensor& documents, const OptTensor& prefix, bool causal, int64_t batch, int64_t q_len,
                          int64_t k_len) {
  const at::Tensor& like = has(documents) ? *documents : *prefix;
  TORCH_CHECK_VALUE(like.is_cuda(), "bitscom: documents and prefix must be CUDA tensors");
  TORCH_CHECK_VALUE(batch >= 0 && batch <= 65535 && q_len >= 0 && k_len >= 0 && q_len < (1 << 30) && k_len < (1 << 30),
                    "bitscom: batch must be at most 65535, lengths below 2^30");
  int ids_bytes = 4, prefix_bytes = 4;
  if (has(documents)) {
    ids_bytes = int_bytes(*documents, "documents");
    TORCH_CHECK_VALUE(documents->dim() == 2 && documents->size(0) == batch && documents->size(1) == k_len,
                      "bitscom: documents must be [", batch, ", ", k_len, "] (batch, key length), got ",
                      documents->sizes());
  }
  if (has(prefix)) {
    prefix_bytes = int_bytes(*prefix, "prefix");
    same_device(*prefix, like, "prefix");
    TORCH_CHECK_VALUE(causal, "bitscom: a prefix needs a causal mask");
    TORCH_CHECK_VALUE(prefix->dim() == 1 && prefix->size(0) == batch, "bitscom: prefix must be [", batch, "], got ",
                      prefix->sizes());
  }
  c10::cuda::CUDAGuard g(like.device());
  const at::Tensor pre = has(prefix) ? prefix->contiguous() : at::Tensor();
  c10::InferenceMode normal(false);  // a plan made in inference mode serves training too
  auto plan = at::empty({PlanView::words(batch, q_len, k_len)}, like.options().dtype(at::kInt));
  if (plan.numel() == 0) return plan;
  launch::attention_plan(has(documents) ? documents->data_ptr() : nullptr, ids_bytes,
                         has(documents) ? documents->stride(0) : 0, has(documents) ? documents->stride(1) : 0,
                         pre.defined() ? pre.data_ptr() : nullptr, prefix_bytes, causal, static_cast<int>(batch),
                         static_cast<int>(q_len), static_cast<int>(k_len),
                         PlanView::of(plan.data_ptr<int>(), batch, q_len, k_len), stream_of(like));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return plan;
}

// Returns (out, log-sums, out's rounding); the last two only for the backward pass, the last one empty where
// it is not kept.
std::tuple<at::Tensor, at::Tensor, at::Tensor> run_forward(const at::Tensor& q_in, const at::Tensor& k_in,
                                                           const at::Tensor& v_in, const OptTensor& plan_in,
                                                           const OptTensor& slopes_in, bool causal, double scale,
                                                           double cap, bool want_sums) {
  check_qkv(q_in, k_in, v_in);
  c10::cuda::CUDAGuard g(q_in.device());
  const auto q = rows_of(q_in), k = rows_of(k_in), v = rows_of(v_in);
  const OptTensor plan = plan_of(plan_in), slopes = slopes_of(slopes_in);
  AttnParams p = params_of(q, k, v, plan, slopes, causal, scale, cap);
  auto out = tokens_first(q);
  at::Tensor lse, lo;
  const auto f32 = q.options().dtype(at::kFloat);
  if (want_sums) {
    lse = at::empty({q.size(0), q.size(1), q.size(2)}, f32);
    lo = for_tensor_cores(q) ? tokens_first(q) : at::empty({0}, q.options());
  }
  if (out.numel() == 0) return {out, lse, lo};
  if (p.sk == 0) {
    out.zero_();
    if (want_sums) lse.fill_(std::numeric_limits<float>::infinity());
    return {out, lse, lo};
  }
  p.o = view_of(out);
  p.lse = want_sums ? lse.data_ptr<float>() : nullptr;
  if (for_tensor_cores(q)) {
    if (want_sums) p.lo = view_of(lo);
    launch::attention_tc_splits(p, at::cuda::getCurrentDeviceProperties()->multiProcessorCount, &p.splits, &p.split_tiles);
    at::Tensor part_o, part_lse;
    if (p.splits > 1) {
      part_o = at::empty({p.splits, q.size(0), q.size(1), q.size(2), q.size(3)}, f32);
      part_lse = at::empty({p.splits, q.size(0), q.size(1), q.size(2)}, f32);
      p.part_o = part_o.data_ptr<float>();
      p.part_lse = part_lse.data_ptr<float>();
    }
    C10_CUDA_CHECK(launch::attention_tc_forward(p, stream_of(q)));
  } else {
    launch::attention_simt_forward(p, stream_of(q));
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  return {out, lse, lo};
}

at::Tensor attention_forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const OptTensor& plan,
                             const OptTensor& slopes, bool causal, double scale, double cap) {
  return std::get<0>(run_forward(q, k, v, plan, slopes, causal, scale, cap, false));
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> attention_forward_sums(const at::Tensor& q, const at::Tensor& k,
                                                                      const at::Tensor& v, const OptTensor& plan,
                                                                      const OptTensor& slopes, bool causal,
                                                                      double scale, double cap) {
  return run_forward(q, k, v, plan, slopes, causal, scale, cap, true);
}

// What autograd hands back need not lie as it was saved (hooks that move saved tensors): out, low, sums and plan are
// copied where their place does not fit.
std::tuple<at::Tensor, at::Tensor, at::Tensor> attention_backward(
    const at::Tensor& dout_in, const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in,
    const at::Tensor& out_in, const at::Tensor& lse_in, const at::Tensor& lo_in, const OptTensor& plan_in,
    const OptTensor& slopes_in, bool causal, double scale, double cap) {
  check_qkv(q_in, k_in, v_in);
  same_device(dout_in, q_in, "the output's gradient");
  same_device(out_in, q_in, "the output");
  same_device(lse_in, q_in, "the log-sums");
  same_device(lo_in, q_in, "the output's rounding");
  c10::cuda::CUDAGuard g(q_in.device());
  const auto q = rows_of(q_in), k = rows_of(k_in), v = rows_of(v_in);
  TORCH_CHECK_VALUE(dout_in.sizes() == q.sizes(), "bitscom: the output's gradient must be ", q.sizes());
  TORCH_CHECK_VALUE(out_in.sizes() == q.sizes() && out_in.scalar_type() == q.scalar_type() &&
                        lse_in.scalar_type() == at::kFloat && lse_in.sizes() == q.sizes().slice(0, 3),
                    "bitscom: the output and its log-sums are not of these queries");
  const auto dout = rows_of(dout_in.to(q.scalar_type())), out = rows_of(out_in);
  const auto lse = lse_in.contiguous();
  auto dq = tokens_first(q), dk = tokens_first(k), dv = tokens_first(v);
  if (q.numel() == 0 || k.numel() == 0) {
    dq.zero_();
    dk.zero_();
    dv.zero_();
    return {dq, dk, dv};
  }
  const OptTensor plan = plan_of(plan_in), slopes = slopes_of(slopes_in);
  AttnParams p = params_of(q, k, v, plan, slopes, causal, scale, cap);
  p.o = view_of(out);
  p.dout = view_of(dout);
  p.dq = view_of(dq);
  p.dk = view_of(dk);
  p.dv = view_of(dv);
  p.lse = lse.data_ptr<float>();
  if (for_tensor_cores(q)) {
    TORCH_CHECK_VALUE(lo_in.sizes() == out.sizes() && lo_in.scalar_type() == out.scalar_type(),
                      "bitscom: the forward pass kept no rounding of its output");
    auto lo = rows_of(lo_in);
    if (lo.strides() != out.strides()) lo = at::empty_strided(out.sizes(), out.strides(), out.options()).copy_(lo);
    p.lo = view_of(lo);
    const int64_t tiles = (q.size(2) + kAttnTile - 1) / kAttnTile;
    auto stats = at::empty({q.size(0), q.size(1), tiles, 2, kAttnTile}, lse.options());
    p.stats = stats.data_ptr<float>();
    C10_CUDA_CHECK(launch::attention_tc_backward(p, stream_of(q)));
  } else {
    auto delta = at::empty_like(lse);
    p.delta = delta.data_ptr<float>();
    launch::attention_simt_backward(p, stream_of(q));
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  return {dq, dk, dv};
}

// ---------------------------------------------------------------------------
// Norm of queries and keys with rotation
// ---------------------------------------------------------------------------

RotaryTensor heads_of(const at::Tensor& t) {
  return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2), static_cast<int>(t.size(2))};
}

at::Tensor gains_of(const OptTensor& w, const at::Tensor& like, const char* name) {
  if (!has(w)) return {};
  same_device(*w, like, name);
  float_type(*w, name);
  TORCH_CHECK_VALUE(w->dim() == 1 && w->size(0) == like.size(3), "bitscom: ", name, " must be [", like.size(3), "], got ",
                    w->sizes());
  return w->to(at::kFloat).contiguous();
}

struct RotaryCall {
  at::Tensor q, k, wq, wk, freq;
  RotaryParams p{};
};

RotaryCall rotary_call(const at::Tensor& q, const at::Tensor& k, const at::Tensor& freq, const OptTensor& wq,
                       const OptTensor& wk, const OptTensor& positions, double eps, bool interleaved) {
  TORCH_CHECK_VALUE(q.is_cuda() && k.is_cuda(), "bitscom: q and k must be CUDA tensors");
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4, "bitscom: q and k must be [batch, length, heads, head size]");
  RotaryCall c;
  c.p.dt = float_type(q, "q");
  TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type(), "bitscom: q and k must have one dtype, got ", q.scalar_type(),
                   " and ", k.scalar_type());
  same_device(k, q, "k");
  TORCH_CHECK_VALUE(q.size(0) == k.size(0) && q.size(1) == k.size(1) && q.size(3) == k.size(3), "bitscom: q ", q.sizes(),
                    " and k ", k.sizes(), " must agree in batch, length and head size");
  const int64_t d = q.size(3);
  TORCH_CHECK_VALUE(d >= 1 && d <= launch::kRotaryMaxDim, "bitscom: head size must be 1 to ", launch::kRotaryMaxDim,
                    ", got ", d);
  TORCH_CHECK_VALUE(q.size(0) * q.size(1) < (int64_t(1) << 31), "bitscom: at most 2^31 - 1 tokens");
  TORCH_CHECK_VALUE(q.size(2) + k.size(2) <= 65535, "bitscom: at most 65535 heads");
  same_device(freq, q, "frequencies");
  TORCH_CHECK_TYPE(freq.is_floating_point(), "bitscom: frequencies must be floating point");
  TORCH_CHECK_VALUE(freq.dim() == 1 && 2 * freq.size(0) <= d, "bitscom: frequencies must be a vector of at most ", d / 2,
                    " values, got ", freq.sizes());
  c.q = q.stride(3) == 1 || d == 1 ? q : q.contiguous();
  c.k = k.stride(3) == 1 || d == 1 ? k : k.contiguous();
  c.wq = gains_of(wq, q, "q_weight");
  c.wk = gains_of(wk, k, "k_weight");
  c.freq = freq.to(at::kDouble).contiguous();
  RotaryParams& p = c.p;
  p.q = heads_of(c.q);
  p.k = heads_of(c.k);
  p.wq = c.wq.defined() ? c.wq.data_ptr<float>() : nullptr;
  p.wk = c.wk.defined() ? c.wk.data_ptr<float>() : nullptr;
  p.freq = c.freq.data_ptr<double>();
  if (has(positions)) {
    same_device(*positions, q, "positions");
    p.pos_bytes = int_bytes(*positions, "positions");
    const bool row = positions->dim() == 1;
    TORCH_CHECK_VALUE((row || positions->dim() == 2) && positions->size(-1) == q.size(1) &&
                          (row || positions->size(0) == q.size(0)),
                      "bitscom: positions must be [", q.size(1), "] or [", q.size(0), ", ", q.size(1), "], got ",
                      positions->sizes());
    p.positions = positions->data_ptr();
    p.pos_sb = row ? 0 : positions->stride(0);
    p.pos_ss = positions->stride(-1);
  }
  p.tokens = q.size(0) * q.size(1);
  p.s = static_cast<unsigned>(q.size(1));
  p.d = static_cast<int>(d);
  p.rotated = static_cast<int>(2 * freq.size(0));
  p.interleaved = interleaved;
  p.eps = static_cast<float>(eps);
  return c;
}

std::tuple<at::Tensor, at::Tensor> rotary_forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& freq,
                                                  const OptTensor& wq, const OptTensor& wk, const OptTensor& positions,
                                                  double eps, bool interleaved) {
  RotaryCall c = rotary_call(q, k, freq, wq, wk, positions, eps, interleaved);
  c10::cuda::CUDAGuard g(q.device());
  auto oq = at::empty(q.sizes(), q.options()), ok = at::empty(k.sizes(), k.options());
  c.p.oq = heads_of(oq);
  c.p.ok = heads_of(ok);
  launch::qk_norm_rotary_forward(c.p, at::cuda::getCurrentDeviceProperties()->multiProcessorCount, stream_of(q));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {oq, ok};
}

// Returns (dq, dk, dw [2, D] fp32, empty when not wanted).
std::tuple<at::Tensor, at::Tensor, at::Tensor> rotary_backward(const at::Tensor& gq_in, const at::Tensor& gk_in,
                                                               const at::Tensor& q, const at::Tensor& k,
                                                               const at::Tensor& freq, const OptTensor& wq,
                                                               const OptTensor& wk, const OptTensor& positions,
                                                               double eps, bool interleaved, bool want_dw) {
  RotaryCall c = rotary_call(q, k, freq, wq, wk, positions, eps, interleaved);
  c10::cuda::CUDAGuard g(q.device());
  same_device(gq_in, q, "the gradient of q");
  same_device(gk_in, q, "the gradient of k");
  TORCH_CHECK_VALUE(gq_in.sizes() == q.sizes() && gk_in.sizes() == k.sizes(), "bitscom: gradients must be ", q.sizes(),
                    " and ", k.sizes());
  const auto fit = [&](const at::Tensor& t) {
    auto x = t.to(q.scalar_type());
    return x.stride(3) == 1 || x.size(3) == 1 ? x : x.contiguous();
  };
  const auto gq = fit(gq_in), gk = fit(gk_in);
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  auto dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options());
  c.p.oq = heads_of(dq);
  c.p.ok = heads_of(dk);
  c.p.gq = heads_of(gq);
  c.p.gk = heads_of(gk);
  at::Tensor partial;
  const auto f32 = q.options().dtype(at::kFloat);
  at::Tensor dw = at::empty({0}, f32);
  if (want_dw) {
    if (c.p.tokens == 0) {
      dw = at::zeros({2, q.size(3)}, f32);
    } else {
      dw = at::empty({2, q.size(3)}, f32);
      partial = at::empty({launch::qk_norm_rotary_blocks(c.p, sms), 2, q.size(3)}, f32);
      c.p.partial = partial.data_ptr<float>();
    }
  }
  launch::qk_norm_rotary_backward(c.p, sms, want_dw ? dw.data_ptr<float>() : nullptr, stream_of(q));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {dq, dk, dw};
}

// ---------------------------------------------------------------------------
// The operators below autograd, as the nodes and bindings call them.
// ---------------------------------------------------------------------------
template <auto Impl, const char* Name>
struct Op;
template <typename R, typename... A, R (*Impl)(A...), const char* Name>
struct Op<Impl, Name> {
  static R call(A... a) {
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow(Name, "").template typed<R(A...)>();
    return op.call(std::forward<A>(a)...);
  }
};
constexpr char kPlan[] = "bitscom_b200::attention_plan", kForward[] = "bitscom_b200::attention_forward",
               kForwardSums[] = "bitscom_b200::attention_forward_sums", kBackward[] = "bitscom_b200::attention_backward",
               kRotary[] = "bitscom_b200::rotary_forward", kRotaryBackward[] = "bitscom_b200::rotary_backward";
using PlanOp = Op<&attention_plan, kPlan>;
using ForwardOp = Op<&attention_forward, kForward>;
using ForwardSumsOp = Op<&attention_forward_sums, kForwardSums>;
using BackwardOp = Op<&attention_backward, kBackward>;
using RotaryOp = Op<&rotary_forward, kRotary>;
using RotaryBackwardOp = Op<&rotary_backward, kRotaryBackward>;

// ---------------------------------------------------------------------------
// Autograd nodes, in C++: a training call of small tensors is bound by the host.
// ---------------------------------------------------------------------------
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

at::Tensor or_undefined(const OptTensor& t) { return has(t) ? *t : at::Tensor(); }
OptTensor if_defined(const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

// Passes gradients on that cannot be differentiated again: the operators have no second derivative.
struct Once : public torch::autograd::Function<Once> {
  static variable_list forward(AutogradContext*, variable_list grads_and_sources, int64_t grads) {
    variable_list out;
    for (int64_t i = 0; i < grads; ++i) out.push_back(grads_and_sources[i].defined() ? grads_and_sources[i].clone() : at::Tensor());
    return out;
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "bitscom: the attention operators are differentiable once only");
  }
};

variable_list once(variable_list grads, const variable_list& sources) {
  if (!at::GradMode::is_enabled()) return grads;
  const auto n = static_cast<int64_t>(grads.size());
  variable_list all = std::move(grads);
  for (auto& t : all)
    if (!t.defined()) t = at::empty({0}, sources[0].options());
  all.insert(all.end(), sources.begin(), sources.end());
  return Once::apply(all, n);
}

struct Attention : public torch::autograd::Function<Attention> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                            const OptTensor& plan, const OptTensor& slopes, bool causal, double scale, double cap) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [out, lse, lo] = ForwardSumsOp::call(q, k, v, plan, slopes, causal, scale, cap);
    ctx->save_for_backward({q, k, v, out, lse, lo, or_undefined(plan), or_undefined(slopes)});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["cap"] = cap;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    variable_list d;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      auto [dq, dk, dv] = BackwardOp::call(g[0], s[0], s[1], s[2], s[3], s[4], s[5], if_defined(s[6]), if_defined(s[7]),
                                    ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble(),
                                    ctx->saved_data["cap"].toDouble());
      d = {dq, dk, dv};
    }
    d = once(std::move(d), {s[0], s[1], s[2], g[0]});
    return {d[0], d[1], d[2], at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

at::Tensor attention_autograd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const OptTensor& plan,
                              const OptTensor& slopes, bool causal, double scale, double cap) {
  no_tangents({q, k, v, slopes});
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return Attention::apply(q, k, v, plan, slopes, causal, scale, cap);
  at::AutoDispatchBelowADInplaceOrView below;
  return ForwardOp::call(q, k, v, plan, slopes, causal, scale, cap);
}

struct QkNormRotary : public torch::autograd::Function<QkNormRotary> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& freq,
                               const OptTensor& wq, const OptTensor& wk, const OptTensor& positions, double eps,
                               bool interleaved) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [oq, ok] = RotaryOp::call(q, k, freq, wq, wk, positions, eps, interleaved);
    ctx->save_for_backward({q, k, freq, or_undefined(wq), or_undefined(wk), or_undefined(positions)});
    ctx->saved_data["want_q"] = has(wq) && wq->requires_grad();
    ctx->saved_data["want_k"] = has(wk) && wk->requires_grad();
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    return {oq, ok};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    const bool want_q = ctx->saved_data["want_q"].toBool(), want_k = ctx->saved_data["want_k"].toBool();
    variable_list d;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      auto [dq, dk, dw] = RotaryBackwardOp::call(g[0], g[1], s[0], s[1], s[2], if_defined(s[3]), if_defined(s[4]), if_defined(s[5]),
                                    ctx->saved_data["eps"].toDouble(), ctx->saved_data["interleaved"].toBool(),
                                    want_q || want_k);
      d = {dq, dk, want_q ? dw.select(0, 0).to(s[3].scalar_type()) : at::Tensor(),
           want_k ? dw.select(0, 1).to(s[4].scalar_type()) : at::Tensor()};
    }
    variable_list sources = {s[0], s[1], g[0], g[1]};
    for (const auto& w : {s[3], s[4]})
      if (w.defined()) sources.push_back(w);
    const variable_list r = once(d, sources);
    return {r[0], r[1], at::Tensor(), want_q ? r[2] : at::Tensor(), want_k ? r[3] : at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

std::tuple<at::Tensor, at::Tensor> rotary_autograd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& freq,
                                                   const OptTensor& wq, const OptTensor& wk, const OptTensor& positions,
                                                   double eps, bool interleaved) {
  no_tangents({q, k, freq, wq, wk});
  const auto wants = [](const OptTensor& t) { return has(t) && t->requires_grad(); };
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || wants(wq) || wants(wk))) {
    auto out = QkNormRotary::apply(q, k, freq, wq, wk, positions, eps, interleaved);
    return {out[0], out[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return RotaryOp::call(q, k, freq, wq, wk, positions, eps, interleaved);
}

}  // namespace

TORCH_LIBRARY(bitscom_b200, m) {
  m.def("attention_plan(Tensor? documents, Tensor? prefix, bool causal, int batch, int q_len, int k_len) -> Tensor");
  m.def(
      "attention_forward(Tensor q, Tensor k, Tensor v, Tensor? plan, Tensor? slopes, bool causal, float scale, "
      "float cap) -> Tensor");
  m.def(
      "attention_forward_sums(Tensor q, Tensor k, Tensor v, Tensor? plan, Tensor? slopes, bool causal, float scale, "
      "float cap) -> (Tensor out, Tensor sums, Tensor low)");
  m.def(
      "attention_backward(Tensor grad, Tensor q, Tensor k, Tensor v, Tensor out, Tensor sums, Tensor low, Tensor? plan, "
      "Tensor? slopes, bool causal, float scale, float cap) -> (Tensor, Tensor, Tensor)");
  m.def(
      "rotary_forward(Tensor q, Tensor k, Tensor frequencies, Tensor? q_weight, Tensor? k_weight, Tensor? positions, "
      "float eps, bool interleaved) -> (Tensor, Tensor)");
  m.def(
      "rotary_backward(Tensor grad_q, Tensor grad_k, Tensor q, Tensor k, Tensor frequencies, Tensor? q_weight, "
      "Tensor? k_weight, Tensor? positions, float eps, bool interleaved, bool want_gains) -> (Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(bitscom_b200, CUDA, m) {
  m.impl("attention_plan", &attention_plan);
  m.impl("attention_forward", &attention_forward);
  m.impl("attention_forward_sums", &attention_forward_sums);
  m.impl("attention_backward", &attention_backward);
  m.impl("rotary_forward", &rotary_forward);
  m.impl("rotary_backward", &rotary_backward);
}

TORCH_LIBRARY_IMPL(bitscom_b200, Autograd, m) {
  m.impl("attention_forward", &attention_autograd);
  m.impl("rotary_forward", &rotary_autograd);
}

void register_attention_bindings(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("attention_plan", &PlanOp::call, py::arg("documents"), py::arg("prefix"), py::arg("causal"), py::arg("batch"),
        py::arg("q_len"), py::arg("k_len"));
  m.def("attention_forward", &ForwardOp::call, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("plan"),
        py::arg("slopes"), py::arg("causal"), py::arg("scale"), py::arg("cap"));
  m.def("rotary_forward", &RotaryOp::call, py::arg("q"), py::arg("k"), py::arg("frequencies"), py::arg("q_weight"),
        py::arg("k_weight"), py::arg("positions"), py::arg("eps"), py::arg("interleaved"));
  m.def("attention_status", [](bool reset) { return launch::attention_status(reset); }, py::arg("reset") = false,
        "1 once a wait of a tensor-core attention kernel on the current device ran out, else 0 (waits for the device).");
  m.def("attention_wait_limit", &launch::attention_wait_limit, py::arg("clocks"),
        "Sets how many clocks a wait inside a tensor-core attention kernel may last before the kernel gives up (0: the "
        "wait for scores always runs out, for tests of that path); returns the limit before.");
}

}  // namespace bitscom_b200
