// torch <-> kernel adapter of the recurrent-decoder operators: linear attention (prompts and single
// tokens), residual add + RMSNorm + E4M3 rows, logit rules.
#include <cmath>

#include "bind_util.h"
#include "linear_attn.h"
#include "logit_rules.h"
#include "norm_fp8.h"

using namespace air_bind;

namespace {

const int* int_row(const optional<Tensor>& t, int64_t n, const Tensor& as, const char* what) {
  if (!t.has_value()) return nullptr;
  same_device(*t, as, what);
  TORCH_CHECK(t->scalar_type() == at::kInt && t->is_contiguous() && t->numel() == n, what, " must be int32 [", str(n), "]");
  return t->data_ptr<int>();
}
const float* float_row(const optional<Tensor>& t, int64_t n, const Tensor& as, const char* what) {
  if (!t.has_value()) return nullptr;
  same_device(*t, as, what);
  TORCH_CHECK(t->scalar_type() == at::kFloat && t->is_contiguous() && t->numel() == n, what, " must be float32 [", str(n), "]");
  return t->data_ptr<float>();
}

// Operands that prompts and single tokens share. `op` names the caller in messages.
air::LinAttnArgs lin_args(const char* op, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& decay,
                          const optional<Tensor>& state, double scale, Tensor& out, Tensor& err) {
  TORCH_CHECK(q.is_cuda(), op, ": q must be a CUDA tensor");
  const Tensor* rows[4] = {&q, &k, &v, &out};
  const char* names[4] = {"q", "k", "v", "out"};
  for (int i = 0; i < 4; ++i) {
    same_device(*rows[i], q, names[i]);
    TORCH_CHECK(rows[i]->dim() == 3, op, ": ", names[i], " must be [tokens, heads, dim]");
    TORCH_CHECK(rows[i]->scalar_type() == q.scalar_type(), op, ": q, k, v and out must have one type");
    TORCH_CHECK(rows[i]->size(2) <= 1 || rows[i]->stride(2) == 1, op, ": the last dimension of ", names[i], " must be contiguous");
    TORCH_CHECK(rows[i]->size(0) == q.size(0), op, ": ", names[i], " has ", str(rows[i]->size(0)), " tokens, q ", str(q.size(0)));
  }
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kFloat, op, ": bfloat16 or float32 q, k, v");
  TORCH_CHECK(q.size(0) < (1ll << 31), op, ": too many tokens");
  same_device(decay, q, "log_decay");
  same_device(err, q, "err");
  TORCH_CHECK(err.scalar_type() == at::kInt && err.numel() >= 1, op, ": err must be int32");
  TORCH_CHECK(decay.scalar_type() == at::kFloat && (decay.dim() == 1 || decay.dim() == 2), op,
              ": log_decay must be float32 [heads] or [tokens, heads]");
  const int64_t H = decay.size(-1);
  TORCH_CHECK(H >= 1 && (H == 1 || decay.stride(-1) == 1), op, ": the heads of log_decay must be contiguous");
  TORCH_CHECK(decay.dim() == 1 || decay.size(0) == q.size(0), op, ": log_decay [tokens, heads] has ", str(decay.size(0)),
              " tokens, q ", str(q.size(0)));
  air::LinAttnArgs a{};
  const int64_t dk = q.size(2), dv = v.size(2);
  TORCH_CHECK(k.size(2) == dk, op, ": q and k must have one head size");
  TORCH_CHECK(dk >= 1 && dk <= 256 && dv >= 1 && dv <= 1024, op, ": head sizes up to 256 (q, k) and 1024 (v)");
  int* div[3] = {&a.q_div, &a.k_div, &a.v_div};
  for (int i = 0; i < 3; ++i) {
    TORCH_CHECK(rows[i]->size(1) >= 1 && H % rows[i]->size(1) == 0, op, ": the heads of ", names[i],
                " must divide the ", str(H), " heads of log_decay");
    *div[i] = (int)(H / rows[i]->size(1));
  }
  TORCH_CHECK(out.size(1) == H && out.size(2) == dv, op, ": out must be [tokens, ", str(H), ", ", str(dv), "]");
  distinct_rows(out, op, "out");
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.out = out.data_ptr();
  a.qs_t = q.stride(0), a.qs_h = q.stride(1);
  a.ks_t = k.stride(0), a.ks_h = k.stride(1);
  a.vs_t = v.stride(0), a.vs_h = v.stride(1);
  a.os_t = out.stride(0), a.os_h = out.stride(1);
  a.decay = decay.data_ptr<float>();
  a.decay_t = decay.dim() == 2 ? decay.stride(0) : 0;
  if (state.has_value()) {
    same_device(*state, q, "state");
    TORCH_CHECK(state->scalar_type() == at::kFloat && state->dim() == 4 && state->is_contiguous() && state->size(1) == H &&
                    state->size(2) == dv && state->size(3) == dk,
                op, ": state must be contiguous float32 [rows, ", str(H), ", ", str(dv), ", ", str(dk), "]");
    a.state = state->data_ptr<float>();
    a.S = state->size(0);
  }
  a.T = (int)q.size(0);
  a.H = (int)H;
  a.dk = (int)dk;
  a.dv = (int)dv;
  a.scale = (float)scale;
  a.err = err.data_ptr<int>();
  return a;
}

Tensor rows_or_new(const char* op, const optional<Tensor>& out, const Tensor& q, const Tensor& v, const Tensor& decay) {
  TORCH_CHECK(q.dim() == 3 && v.dim() == 3 && decay.dim() >= 1, op, ": q and v must be [tokens, heads, dim], log_decay [.., heads]");
  return or_new(out, {q.size(0), decay.size(-1), v.size(2)}, q, q.scalar_type());
}

// Packed prompts. cu [N + 1] int32 token offsets (none: one sequence of all tokens).
Tensor linear_attention(Tensor q, Tensor k, Tensor v, Tensor decay, optional<Tensor> state, optional<Tensor> cu,
                        optional<Tensor> slots, optional<Tensor> has_state, optional<double> scale_, optional<Tensor> out_,
                        Tensor err) {
  Tensor out = rows_or_new("linear_attention", out_, q, v, decay);
  const double scale = scale_.has_value() ? *scale_ : 1.0 / std::sqrt((double)q.size(2));
  air::LinAttnArgs a = lin_args("linear_attention", q, k, v, decay, state, scale, out, err);
  const c10::cuda::CUDAGuard guard(q.device());
  int64_t N = 1;
  a.whole = 1;
  if (cu.has_value()) {
    TORCH_CHECK(cu->numel() >= 1, "linear_attention: cu_seqlens must be int32 [sequences + 1]");
    N = cu->numel() - 1;
    a.cu = int_row(cu, N + 1, q, "cu_seqlens");
  }
  TORCH_CHECK(N < (1ll << 31) / a.H, "linear_attention: too many sequences");
  TORCH_CHECK(state.has_value() || (!slots.has_value() && !has_state.has_value()),
              "linear_attention: slots and has_state go with a state");
  a.N = (int)N;
  a.slots = int_row(slots, N, q, "slots");
  a.has_state = int_row(has_state, N, q, "has_state");
  TORCH_CHECK(!a.state || a.slots || N <= a.S, "linear_attention: ", str(N), " sequences, ", str(a.S), " state rows");
  if (N == 0) return out;
  const bool f32 = q.scalar_type() == at::kFloat;
  auto st = at::cuda::getCurrentCUDAStream();
  if (air::linear_blocks_supported(a, f32) && air::linear_blocks_worth(a)) {
    const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
    // scratch of the split over the length, from the allocator's pool of this stream
    Tensor ws;
    const int64_t n = air::linear_blocks_workspace(a, sms);
    if (n) ws = at::empty({n}, q.options().dtype(at::kFloat));
    const char* e = air::launch_linear_blocks(a, n ? ws.data_ptr<float>() : nullptr, sms, st);
    TORCH_CHECK(e == nullptr, e ? e : "");
  } else {
    air::launch_linear_scan(a, f32, st);
  }
  post("linear_attention");
  return out;
}

// One new token per sequence: row n of q, k and v belongs to state row slots[n] (none: n).
Tensor linear_attention_step(Tensor q, Tensor k, Tensor v, Tensor decay, Tensor state, optional<Tensor> slots,
                             optional<double> scale_, optional<Tensor> out_, Tensor err) {
  Tensor out = rows_or_new("linear_attention_step", out_, q, v, decay);
  const double scale = scale_.has_value() ? *scale_ : 1.0 / std::sqrt((double)q.size(2));
  air::LinAttnArgs a = lin_args("linear_attention_step", q, k, v, decay, state, scale, out, err);
  const c10::cuda::CUDAGuard guard(q.device());
  a.N = a.T;
  a.has_state_all = 1;
  a.zero_pad = 1;
  TORCH_CHECK((int64_t)a.N < (1ll << 31) / a.H, "linear_attention_step: too many rows");
  a.slots = int_row(slots, a.N, q, "slots");
  TORCH_CHECK(a.slots || a.N <= a.S, "linear_attention_step: ", str(a.N), " rows, ", str(a.S), " state rows");
  if (a.N == 0) return out;
  const bool f32 = q.scalar_type() == at::kFloat;
  auto st = at::cuda::getCurrentCUDAStream();
  if (air::linear_step_supported(a, f32)) air::launch_linear_step(a, f32, st);
  else air::launch_linear_scan(a, f32, st);
  post("linear_attention_step");
  return out;
}

bool aligned(const Tensor& t, int64_t bytes, bool rows = true) {
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % bytes == 0 && (!rows || t.stride(0) * t.element_size() % bytes == 0);
}

std::tuple<Tensor, Tensor> add_rmsnorm_fp8(Tensor x, optional<Tensor> y, Tensor w, double eps, double w_offset,
                                           optional<Tensor> resid, optional<Tensor> xq_, optional<Tensor> xs_,
                                           optional<Tensor> out_bf16) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.scalar_type() == at::kFloat && x.stride(1) == 1,
              "add_rmsnorm_fp8: x must be a CUDA float32 [tokens, dim] with contiguous rows");
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t T = x.size(0), K = x.size(1);
  TORCH_CHECK(K % 8 == 0 && K >= 8 && K <= air::kAddNormMaxK, "add_rmsnorm_fp8: dim must be a multiple of 8 up to ",
              str(air::kAddNormMaxK));
  auto rows = [&](const Tensor& t, const char* what) {
    same_device(t, x, what);
    TORCH_CHECK(t.dim() == 2 && t.size(0) == T && t.size(1) == K && t.stride(1) == 1, "add_rmsnorm_fp8: ", what,
                " must be [", str(T), ", ", str(K), "] with contiguous rows");
    TORCH_CHECK(aligned(t, 16, T > 1), "add_rmsnorm_fp8: the rows of ", what, " must be 16-byte aligned");
  };
  rows(x, "x");
  air::AddNormF8Args a{};
  a.x = x.data_ptr<float>();
  a.ldx = x.stride(0);
  if (y.has_value()) {
    rows(*y, "y");
    TORCH_CHECK(y->scalar_type() == at::kBFloat16 || y->scalar_type() == at::kFloat, "add_rmsnorm_fp8: y bfloat16 or float32");
    a.y = y->data_ptr();
    a.y_bf16 = y->scalar_type() == at::kBFloat16;
    a.ldy = y->stride(0);
  }
  same_device(w, x, "w");
  TORCH_CHECK(w.scalar_type() == at::kFloat && w.is_contiguous() && w.numel() == K && aligned(w, 16, false),
              "add_rmsnorm_fp8: w must be float32 [", str(K), "], 16-byte aligned");
  a.w = w.data_ptr<float>();
  if (resid.has_value()) {
    rows(*resid, "resid_out");
    TORCH_CHECK(resid->scalar_type() == at::kFloat, "add_rmsnorm_fp8: resid_out float32");
    distinct_rows(*resid, "add_rmsnorm_fp8", "resid_out");
    a.resid = resid->data_ptr<float>();
    a.ldr = resid->stride(0);
  }
  if (out_bf16.has_value()) {
    rows(*out_bf16, "out_bf16");
    TORCH_CHECK(out_bf16->scalar_type() == at::kBFloat16, "add_rmsnorm_fp8: out_bf16 bfloat16");
    distinct_rows(*out_bf16, "add_rmsnorm_fp8", "out_bf16");
    a.out_bf16 = out_bf16->data_ptr();
    a.ldo = out_bf16->stride(0);
  }
  Tensor xq = or_new(xq_, {T, K}, x, at::kByte), xs = or_new(xs_, {T}, x, at::kFloat);
  same_device(xq, x, "xq");
  same_device(xs, x, "xs");
  TORCH_CHECK(xq.element_size() == 1 && xq.is_contiguous() && xq.numel() == T * K && aligned(xq, 8, false),
              "add_rmsnorm_fp8: xq must be contiguous bytes [", str(T), ", ", str(K), "]");
  TORCH_CHECK(xs.scalar_type() == at::kFloat && xs.is_contiguous() && xs.numel() == T, "add_rmsnorm_fp8: xs float32 [", str(T), "]");
  a.xq = reinterpret_cast<uint8_t*>(xq.data_ptr());
  a.xs = xs.data_ptr<float>();
  a.w_offset = (float)w_offset;
  a.eps = (float)eps;
  TORCH_CHECK(T < (1ll << 31), "add_rmsnorm_fp8: too many rows");
  a.T = (int)T;
  a.K = (int)K;
  const char* e = air::launch_add_rmsnorm_fp8(a, at::cuda::getCurrentCUDAStream());
  TORCH_CHECK(e == nullptr, e ? e : "");
  post("add_rmsnorm_fp8");
  return {xq, xs};
}

void logit_rules(Tensor logits, Tensor out, optional<Tensor> counts, optional<Tensor> count_row,
                 optional<Tensor> repetition, optional<Tensor> frequency, optional<Tensor> presence,
                 optional<Tensor> bias_ptr, optional<Tensor> bias_ids, optional<Tensor> bias_vals,
                 optional<Tensor> mask, Tensor err) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && (logits.size(1) <= 1 || logits.stride(1) == 1),
              "logit_rules: logits must be a CUDA [rows, vocab] with contiguous rows");
  TORCH_CHECK(logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kBFloat16,
              "logit_rules: float32 or bfloat16 logits");
  const c10::cuda::CUDAGuard guard(logits.device());
  const int64_t B = logits.size(0), V = logits.size(1);
  same_device(out, logits, "out");
  TORCH_CHECK(out.scalar_type() == at::kFloat && out.sizes() == logits.sizes() && (V <= 1 || out.stride(1) == 1),
              "logit_rules: out must be float32 [rows, vocab] with contiguous rows");
  distinct_rows(out, "logit_rules", "out");
  TORCH_CHECK(B <= 65535 && V < (1ll << 31) - 4096, "logit_rules: at most 65535 rows");
  same_device(err, logits, "err");
  TORCH_CHECK(err.scalar_type() == at::kInt && err.numel() >= 1, "logit_rules: err must be int32");
  air::LogitRulesArgs a{};
  a.logits = logits.data_ptr();
  a.bf16 = logits.scalar_type() == at::kBFloat16;
  a.ld_in = logits.stride(0);
  a.out = out.data_ptr<float>();
  a.ld_out = out.stride(0);
  a.B = (int)B;
  a.V = (int)V;
  if (counts.has_value()) {
    same_device(*counts, logits, "counts");
    TORCH_CHECK(counts->scalar_type() == at::kByte && counts->dim() == 2 && counts->is_contiguous() && counts->size(1) == V,
                "logit_rules: counts must be contiguous uint8 [rows, ", str(V), "]");
    a.counts = counts->data_ptr<uint8_t>();
    a.S = counts->size(0);
    a.count_row = int_row(count_row, B, logits, "count_row");
    TORCH_CHECK(a.count_row || B <= a.S, "logit_rules: ", str(B), " rows, ", str(a.S), " rows of counts");
  }
  TORCH_CHECK(counts.has_value() || (!repetition.has_value() && !frequency.has_value() && !presence.has_value() &&
                                     !count_row.has_value()),
              "logit_rules: penalties need counts");
  a.repetition = float_row(repetition, B, logits, "repetition");
  a.frequency = float_row(frequency, B, logits, "frequency");
  a.presence = float_row(presence, B, logits, "presence");
  TORCH_CHECK(bias_ptr.has_value() == bias_ids.has_value() && bias_ptr.has_value() == bias_vals.has_value(),
              "logit_rules: a bias is (ptr, ids, values)");
  if (bias_ptr.has_value()) {
    a.bias_ptr = int_row(bias_ptr, B + 1, logits, "bias ptr");
    a.n_bias = bias_ids->numel();
    a.bias_ids = int_row(bias_ids, a.n_bias, logits, "bias ids");
    a.bias_vals = float_row(bias_vals, a.n_bias, logits, "bias values");
  }
  if (mask.has_value()) {
    same_device(*mask, logits, "mask");
    TORCH_CHECK(mask->scalar_type() == at::kInt && mask->is_contiguous() && mask->numel() == B * ((V + 31) / 32),
                "logit_rules: mask must be contiguous int32 [", str(B), ", ", str((V + 31) / 32), "]");
    a.mask = reinterpret_cast<const uint32_t*>(mask->data_ptr<int>());
  }
  a.err = err.data_ptr<int>();
  air::launch_logit_rules(a, at::cuda::getCurrentCUDAStream());
  post("logit_rules");
}

}  // namespace

void register_recurrent(pybind11::module_& m) {
  m.def("linear_attention", &linear_attention);
  m.def("linear_attention_step", &linear_attention_step);
  m.def("add_rmsnorm_fp8", &add_rmsnorm_fp8);
  m.def("logit_rules", &logit_rules);
}
