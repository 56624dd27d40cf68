// torch <-> kernel adapter of the state-space decoder's operators: causal convolution and selective scan (prompts and
// single tokens), block norm, token log probabilities. Shapes, types, strides and aliasing are checked before devices,
// so every refusal but that of a wrong device is the same for CPU tensors.
#include "bind_util.h"
#include "state_space.h"

using namespace air_bind;

namespace {

// What a call was given, for the checks that concern all operands.
struct Operands {
  struct Operand {
    const Tensor* t;
    const char* what;
  };
  const char* op;
  Operand all[16];
  int n = 0;

  explicit Operands(const char* name) : op(name) {}
  void add(const Tensor& t, const char* what) { all[n++] = {&t, what}; }

  // [rows, cols] bf16 or f32 with contiguous rows (`type`: the type it must have)
  void rows(const Tensor& t, const char* what, int64_t n, int64_t d, c10::optional<at::ScalarType> type = c10::nullopt) {
    TORCH_CHECK(t.dim() == 2 && t.size(0) == n && t.size(1) == d, op, ": ", what, " must be [", str(n), ", ", str(d), "]");
    TORCH_CHECK(d <= 1 || t.stride(1) == 1, op, ": the rows of ", what, " must be contiguous");
    type_is(t, what, type);
    add(t, what);
  }
  void type_is(const Tensor& t, const char* what, c10::optional<at::ScalarType> type) {
    const auto is = t.scalar_type();
    TORCH_CHECK(type.has_value() ? is == *type : is == at::kBFloat16 || is == at::kFloat, op, ": ", what, " must be ",
                type.has_value() ? toString(*type) : "BFloat16 or Float");
  }
  const float* floats(const Tensor& t, const char* what, at::IntArrayRef shape) {
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.is_contiguous() && t.sizes() == shape, op, ": ", what,
                " must be contiguous float32 of ", str(shape[0]), shape.size() > 1 ? " x " + str(shape[1]) : std::string(),
                " values");
    add(t, what);
    return t.data_ptr<float>();
  }
  const float* floats(const optional<Tensor>& t, const char* what, at::IntArrayRef shape) {
    return t.has_value() ? floats(*t, what, shape) : nullptr;
  }
  const int* ints(const optional<Tensor>& t, const char* what, int64_t n) {
    if (!t.has_value()) return nullptr;
    TORCH_CHECK(t->scalar_type() == at::kInt && t->is_contiguous() && t->dim() == 1 && t->numel() == n, op, ": ", what,
                " must be contiguous int32 [", str(n), "]");
    add(*t, what);
    return t->data_ptr<int>();
  }
  int* error_word(const Tensor& t) {
    TORCH_CHECK(t.scalar_type() == at::kInt && t.numel() >= 1, op, ": err must be int32");
    add(t, "err");
    return t.data_ptr<int>();
  }

  // First and last byte of a tensor's elements.
  static std::pair<uintptr_t, uintptr_t> span(const Tensor& t) {
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    const uintptr_t p = reinterpret_cast<uintptr_t>(t.data_ptr());
    return {p, p + (last + 1) * t.element_size()};
  }
  // Two operands that meet in memory: not if their spans are apart, nor if both are rows of one stride at columns that
  // do not meet (two parts of one projection's rows).
  static bool meet(const Tensor& a, const Tensor& b) {
    if (a.numel() == 0 || b.numel() == 0) return false;
    const auto sa = span(a), sb = span(b);
    if (sa.second <= sb.first || sb.second <= sa.first) return false;
    if (a.dim() != 2 || b.dim() != 2) return true;
    const int64_t ra = a.stride(0) * a.element_size(), rb = b.stride(0) * b.element_size();
    const int64_t wa = a.size(1) * a.element_size(), wb = b.size(1) * b.element_size();
    if (ra != rb || ra < wa || ra < wb) return true;
    const int64_t off = (int64_t)(sb.first > sa.first ? sb.first - sa.first : ra - (sa.first - sb.first) % ra) % ra;
    return off < wa || off + wb > ra;          // b's columns start inside a's, or reach a's next row
  }
  // `t` is written: nothing else may lie in it, but for `same`, which may be the same memory element by element.
  void written(const Tensor& t, const char* what, const Tensor* same = nullptr) const {
    for (int i = 0; i < n; ++i) {
      const Tensor& o = *all[i].t;
      if (&o == &t) continue;
      if (same && &o == same && t.data_ptr() == o.data_ptr() && t.strides() == o.strides() && t.scalar_type() == o.scalar_type()) continue;
      TORCH_CHECK(!meet(t, o), op, ": ", what, " shares memory with ", all[i].what);
    }
  }
  void on_device() const {
    TORCH_CHECK(all[0].t->is_cuda(), op, ": ", all[0].what, " must be a CUDA tensor");
    const auto device = all[0].t->device();
    for (int i = 1; i < n; ++i) TORCH_CHECK(all[i].t->device() == device, op, ": ", all[i].what, " must be on the device of ", all[0].what);
  }
};

bool aligned(const Tensor& t, int64_t bytes) {
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % bytes) return false;
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) * t.element_size() % bytes) return false;
  return true;
}

// A new output, made on the first operand's device before the devices are checked.
Tensor output(const optional<Tensor>& out, at::IntArrayRef sizes, const Tensor& as, at::ScalarType type) {
  return out.has_value() ? *out : at::empty(sizes, as.options().dtype(type));
}

constexpr int64_t kMaxTokens = (1ll << 31) - 4096;   // room for the tokens that blocks look ahead

// Sequences of a prompt call (step = 0) or one token each (step = 1).
air::SeqArgs sequences(Operands& c, int64_t T, int64_t S, bool has_pool, const optional<Tensor>& cu, const optional<Tensor>& slots,
                       const optional<Tensor>& has_state, const Tensor& err, int step) {
  TORCH_CHECK(T < kMaxTokens, c.op, ": too many tokens");
  air::SeqArgs s{};
  int64_t N = step ? T : 1;
  if (cu.has_value()) {
    TORCH_CHECK(cu->numel() >= 1, c.op, ": cu_seqlens must be int32 [sequences + 1]");
    N = cu->numel() - 1;
    s.cu = c.ints(cu, "cu_seqlens", N + 1);
  }
  TORCH_CHECK(has_pool || (!slots.has_value() && !has_state.has_value()), c.op, ": slots and has_state go with a state");
  s.slots = c.ints(slots, "slots", N);
  s.has_state = c.ints(has_state, "has_state", N);
  s.has_state_all = step;
  s.step = step;
  s.S = S;
  s.N = (int)N;
  s.T = (int)T;
  TORCH_CHECK(!has_pool || s.slots || N <= S, c.op, ": ", str(N), " sequences, ", str(S), " state rows");
  s.err = c.error_word(err);
  return s;
}

Tensor conv(const char* op, const Tensor& x, const Tensor& w, const optional<Tensor>& bias, const optional<Tensor>& state,
            const optional<Tensor>& cu, const optional<Tensor>& slots, const optional<Tensor>& has_state, bool silu,
            const optional<Tensor>& out_, const Tensor& err, int step) {
  TORCH_CHECK(x.dim() == 2 && w.dim() == 2, op, ": x must be [tokens, channels], w [channels, taps]");
  const int64_t T = x.size(0), D = x.size(1), W = w.size(1);
  TORCH_CHECK(W >= 2 && W <= 4, op, ": 2 to 4 taps, not ", str(W));
  TORCH_CHECK(D >= 1 && D < (1ll << 31) - 4096, op, ": at least one channel");
  Operands c(op);
  c.rows(x, "x", T, D);
  air::ConvArgs a{};
  a.w = c.floats(w, "w", {D, W});
  a.bias = c.floats(bias, "bias", {D});
  if (state.has_value()) {
    TORCH_CHECK(state->dim() == 3 && state->is_contiguous() && state->scalar_type() == x.scalar_type() && state->size(1) == W - 1 &&
                    state->size(2) == D, op, ": state must be contiguous [rows, ", str(W - 1), ", ", str(D), "] of x's type");
    c.add(*state, "state");
    a.state = state->data_ptr();
  }
  a.seq = sequences(c, T, state.has_value() ? state->size(0) : 0, state.has_value(), cu, slots, has_state, err, step);
  Tensor out = output(out_, {T, D}, x, x.scalar_type());
  c.rows(out, "out", T, D, x.scalar_type());
  distinct_rows(out, op, "out");
  c.written(out, "out");
  if (state.has_value()) c.written(*state, "state");
  c.on_device();
  const c10::cuda::CUDAGuard guard(x.device());
  a.x = x.data_ptr();
  a.out = out.data_ptr();
  a.xs = x.stride(0);
  a.os = out.stride(0);
  a.D = (int)D;
  a.W = (int)W;
  a.silu = silu;
  // a thread's taps start at a multiple of vec W floats: w need only start at 16 bytes
  int vec = reinterpret_cast<uintptr_t>(a.w) % 16 ? 1 : x.scalar_type() == at::kFloat ? 4 : 8;
  auto rows = [&](const Tensor& t) {
    while (vec > 1 && (D % vec || !aligned(t, vec * t.element_size()))) vec /= 2;
  };
  rows(x);
  rows(out);
  if (state.has_value()) rows(*state);
  const char* e = air::launch_causal_conv(a, x.scalar_type() == at::kFloat, vec, at::cuda::getCurrentCUDAStream());
  TORCH_CHECK(e == nullptr, e ? e : "");
  post(op);
  return out;
}

Tensor causal_conv(Tensor x, Tensor w, optional<Tensor> bias, optional<Tensor> state, optional<Tensor> cu, optional<Tensor> slots,
                   optional<Tensor> has_state, bool silu, optional<Tensor> out, Tensor err) {
  return conv("causal_conv", x, w, bias, state, cu, slots, has_state, silu, out, err, 0);
}
Tensor causal_conv_step(Tensor x, Tensor w, Tensor state, optional<Tensor> bias, optional<Tensor> slots, bool silu,
                        optional<Tensor> out, Tensor err) {
  return conv("causal_conv_step", x, w, bias, state, c10::nullopt, slots, c10::nullopt, silu, out, err, 1);
}

Tensor scan(const char* op, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B_, const Tensor& C_,
            const optional<Tensor>& skip, const optional<Tensor>& z, const optional<Tensor>& dt_bias, bool softplus,
            const optional<Tensor>& state, const optional<Tensor>& cu, const optional<Tensor>& slots,
            const optional<Tensor>& has_state, const optional<Tensor>& out_, const Tensor& err, int step) {
  TORCH_CHECK(x.dim() == 2 && A.dim() == 2, op, ": x must be [tokens, channels], A [channels, states]");
  const int64_t T = x.size(0), D = x.size(1), N = A.size(1);
  TORCH_CHECK(N >= 1 && N <= air::kScanMaxStates, op, ": 1 to ", str(air::kScanMaxStates), " states, not ", str(N));
  TORCH_CHECK(D >= 1 && D < (1ll << 31) - 4096, op, ": at least one channel");
  Operands c(op);
  const auto type = x.scalar_type();
  c.rows(x, "x", T, D);
  c.rows(dt, "dt", T, D, type);
  if (z.has_value()) c.rows(*z, "z", T, D, type);
  air::ScanArgs a{};
  a.A = c.floats(A, "A", {D, N});
  a.skip = c.floats(skip, "D", {D});
  a.dt_bias = c.floats(dt_bias, "dt_bias", {D});
  const Tensor B = B_.dim() == 2 ? B_.unsqueeze(1) : B_, C = C_.dim() == 2 ? C_.unsqueeze(1) : C_;
  const std::pair<const Tensor*, const char*> bc[2] = {{&B, "B"}, {&C, "C"}};
  for (const auto& o : bc) {
    const Tensor& t = *o.first;
    TORCH_CHECK(t.dim() == 3 && t.size(0) == T && t.size(2) == N && t.size(1) >= 1 && D % t.size(1) == 0 && t.size(1) == B.size(1),
                op, ": B and C must be [", str(T), ", ", str(N), "] or [", str(T), ", groups, ", str(N), "] with groups that divide ",
                str(D), " channels");
    TORCH_CHECK(N <= 1 || t.stride(2) == 1, op, ": the states of ", o.second, " must be contiguous");
    c.type_is(t, o.second, type);
    c.add(t, o.second);
  }
  if (state.has_value()) {
    TORCH_CHECK(state->dim() == 3 && state->is_contiguous() && state->scalar_type() == at::kFloat && state->size(1) == D &&
                    state->size(2) == N, op, ": state must be contiguous float32 [rows, ", str(D), ", ", str(N), "]");
    c.add(*state, "state");
    a.state = state->data_ptr<float>();
  }
  a.seq = sequences(c, T, state.has_value() ? state->size(0) : 0, state.has_value(), cu, slots, has_state, err, step);
  Tensor out = output(out_, {T, D}, x, type);
  c.rows(out, "out", T, D, type);
  distinct_rows(out, op, "out");
  c.written(out, "out");
  if (state.has_value()) c.written(*state, "state");
  c.on_device();
  const c10::cuda::CUDAGuard guard(x.device());
  a.x = x.data_ptr();
  a.dt = dt.data_ptr();
  a.z = z.has_value() ? z->data_ptr() : nullptr;
  a.B = B.data_ptr();
  a.C = C.data_ptr();
  a.out = out.data_ptr();
  a.xs = x.stride(0);
  a.ds = dt.stride(0);
  a.zs = z.has_value() ? z->stride(0) : 0;
  a.os = out.stride(0);
  a.bs_t = B.stride(0), a.bs_g = B.stride(1);
  a.cs_t = C.stride(0), a.cs_g = C.stride(1);
  a.D = (int)D;
  a.G = (int)B.size(1);
  a.N = (int)N;
  a.softplus = softplus;
  TORCH_CHECK(a.seq.N <= (1ll << 31) / (D / 4 + 1), op, ": too many sequences");
  const bool f32 = type == at::kFloat;
  auto st = at::cuda::getCurrentCUDAStream();
  if (!step && air::scan_tiles_worth(a)) {
    const air::ScanPlan p = air::scan_plan(a, at::cuda::getCurrentDeviceProperties()->multiProcessorCount);
    Tensor ws;                                     // from the allocator's pool of this stream
    if (p.floats) ws = at::empty({p.floats}, x.options().dtype(at::kFloat));
    const char* e = air::launch_scan_tiles(a, p, p.floats ? ws.data_ptr<float>() : nullptr, f32, st);
    TORCH_CHECK(e == nullptr, e ? e : "");
  } else {
    air::launch_scan_tokens(a, f32, st);
  }
  post(op);
  return out;
}

Tensor selective_scan(Tensor x, Tensor dt, Tensor A, Tensor B, Tensor C, optional<Tensor> skip, optional<Tensor> z,
                      optional<Tensor> dt_bias, bool softplus, optional<Tensor> state, optional<Tensor> cu, optional<Tensor> slots,
                      optional<Tensor> has_state, optional<Tensor> out, Tensor err) {
  return scan("selective_scan", x, dt, A, B, C, skip, z, dt_bias, softplus, state, cu, slots, has_state, out, err, 0);
}
Tensor selective_scan_step(Tensor x, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor state, optional<Tensor> skip,
                           optional<Tensor> z, optional<Tensor> dt_bias, bool softplus, optional<Tensor> slots,
                           optional<Tensor> out, Tensor err) {
  return scan("selective_scan_step", x, dt, A, B, C, skip, z, dt_bias, softplus, state, c10::nullopt, slots, c10::nullopt, out, err, 1);
}

// act: 0 SiLU, 1 sigmoid, 2 the gate itself. `new_out`: out is made here, in bf16.
std::tuple<optional<Tensor>, optional<Tensor>> block_norm(Tensor y, optional<Tensor> w, double eps, optional<Tensor> resid,
                                                          optional<Tensor> post_w, optional<Tensor> gate, int64_t act, double scale,
                                                          optional<Tensor> scale_row, double w_offset, optional<Tensor> out,
                                                          bool new_out, optional<Tensor> resid_out) {
  const char* op = "block_norm";
  TORCH_CHECK(y.dim() == 2, op, ": y must be [tokens, dim]");
  const int64_t T = y.size(0), K = y.size(1);
  TORCH_CHECK(K >= 1 && K <= air::kBlockNormMaxK, op, ": 1 to ", str(air::kBlockNormMaxK), " columns, not ", str(K));
  TORCH_CHECK(T < (1ll << 31), op, ": too many rows");
  Operands c(op);
  c.rows(y, "y", T, K);
  air::BlockNormArgs a{};
  a.w = c.floats(w, "weight", {K});
  a.post = c.floats(post_w, "post_weight", {K});
  a.scale_row = c.floats(scale_row, "scale", {K});
  int vec = 4;
  auto four = [&](const Tensor& t) {
    while (vec > 1 && (K % vec || !aligned(t, vec * t.element_size()))) vec /= 2;
  };
  for (const auto* t : {&w, &post_w, &scale_row})
    if (t->has_value()) four(**t);
  four(y);
  if (resid.has_value()) {
    c.rows(*resid, "residual", T, K);
    a.resid = resid->data_ptr();
    a.ldr = resid->stride(0);
    a.r_bf16 = resid->scalar_type() == at::kBFloat16;
    four(*resid);
  }
  if (gate.has_value()) {
    if (gate->dim() == 1) {
      TORCH_CHECK(gate->size(0) == K && (K <= 1 || gate->stride(0) == 1), op, ": gate must be [", str(K), "] or [", str(T), ", ",
                  str(K), "] with contiguous rows");
      c.type_is(*gate, "gate", y.scalar_type());
      c.add(*gate, "gate");
    } else {
      c.rows(*gate, "gate", T, K, y.scalar_type());
      a.ldg = gate->stride(0);
    }
    a.gate = gate->data_ptr();
    four(*gate);
  }
  if (resid_out.has_value()) {
    c.rows(*resid_out, "resid_out", T, K, resid.has_value() ? c10::make_optional(resid->scalar_type()) : c10::nullopt);
    distinct_rows(*resid_out, op, "resid_out");
    a.resid_out = resid_out->data_ptr();
    a.ldro = resid_out->stride(0);
    a.r_bf16 = resid_out->scalar_type() == at::kBFloat16;
    four(*resid_out);
  }
  if (new_out) out = at::empty({T, K}, y.options().dtype(at::kBFloat16));
  if (out.has_value()) {
    c.rows(*out, "out", T, K);
    distinct_rows(*out, op, "out");
    a.out = out->data_ptr();
    a.ldo = out->stride(0);
    a.o_bf16 = out->scalar_type() == at::kBFloat16;
    four(*out);
    c.written(*out, "out");
  }
  if (resid_out.has_value()) c.written(*resid_out, "resid_out", resid.has_value() ? &*resid : nullptr);
  c.on_device();
  const c10::cuda::CUDAGuard guard(y.device());
  a.y = y.data_ptr();
  a.ldy = y.stride(0);
  a.y_bf16 = y.scalar_type() == at::kBFloat16;
  a.scale = (float)scale;
  a.w_offset = (float)w_offset;
  a.eps = (float)eps;
  a.act = (int)act;
  a.T = (int)T;
  a.K = (int)K;
  const char* e = air::launch_block_norm(a, vec, at::cuda::getCurrentCUDAStream());
  TORCH_CHECK(e == nullptr, e ? e : "");
  post(op);
  return {out, resid_out};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> token_logprobs(Tensor logits, optional<Tensor> tokens, int64_t k, Tensor err) {
  const char* op = "token_logprobs";
  TORCH_CHECK(logits.dim() == 2, op, ": logits must be [tokens, vocabulary]");
  const int64_t T = logits.size(0), V = logits.size(1);
  TORCH_CHECK(V >= 1 && V < kMaxTokens && T < (1ll << 31) / 64, op, ": a vocabulary of at least one token, at most 33554431 rows");
  TORCH_CHECK(k >= 0 && k <= air::kLogprobMaxTop, op, ": 0 to ", str(air::kLogprobMaxTop), " alternatives, not ", str(k));
  Operands c(op);
  c.rows(logits, "logits", T, V);
  air::TokenLogprobArgs a{};
  a.tokens = c.ints(tokens, "tokens", T);
  a.err = c.error_word(err);
  c.on_device();
  const c10::cuda::CUDAGuard guard(logits.device());
  const auto f = logits.options().dtype(at::kFloat);
  Tensor lp = at::empty({T}, f), ent = at::empty({T}, f), top = at::empty({T, k}, f), ids = at::empty({T, k}, f.dtype(at::kInt));
  a.logits = logits.data_ptr();
  a.ld = logits.stride(0);
  a.logprob = lp.data_ptr<float>();
  a.entropy = ent.data_ptr<float>();
  a.top_lp = top.data_ptr<float>();
  a.top_id = ids.data_ptr<int>();
  a.T = (int)T;
  a.V = (int)V;
  a.k = (int)k;
  air::launch_token_logprobs(a, logits.scalar_type() == at::kFloat, at::cuda::getCurrentCUDAStream());
  post(op);
  return {lp, ent, top, ids};
}

}  // namespace

void register_state_space(pybind11::module_& m) {
  m.def("causal_conv", &causal_conv);
  m.def("causal_conv_step", &causal_conv_step);
  m.def("selective_scan", &selective_scan);
  m.def("selective_scan_step", &selective_scan_step);
  m.def("block_norm", &block_norm);
  m.def("token_logprobs", &token_logprobs);
}
