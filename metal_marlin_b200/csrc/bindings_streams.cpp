// torch.ops.mmb200.{causal_conv, ssm, sink_decode}: checks and argument packing of the operators that keep a sequence going at constant cost
// per token.  Checks that concern shapes and types raise ValueError and come before the one that asks for a GPU, so they can be
// exercised without one.
#include <climits>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>
#include <torch/torch.h>

#include "api_ext.h"

namespace {

using torch::Tensor;
using OptT = c10::optional<Tensor>;

constexpr int64_t kMaxRows = 1 << 30;        // the kernels count rows, sequences, channels and tiles of them in 32 bits: room for the last tile's end
constexpr int64_t kMaxGrid = 65535;          // rows of a single-token call

inline cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }
inline bool given(const OptT& t) { return t.has_value() && t->defined(); }
inline void check(int err, const char* what) {
  TORCH_CHECK(err == 0, what, " failed: ", cudaGetErrorString((cudaError_t)err), " (", err, ")");
}
inline int elt_type(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    default: TORCH_CHECK_VALUE(false, name, " must be bf16, fp16 or fp32");
  }
  return -1;
}
inline void check_2d(const Tensor& t, int64_t rows, int64_t cols, const Tensor& on, const char* name) {
  TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == rows && t.size(1) == cols, name, " must have the shape [", rows, ", ", cols, "]");
  TORCH_CHECK_VALUE(t.stride(1) == 1 || cols <= 1, name, " must have unit stride along its last axis");
  TORCH_CHECK_VALUE(t.device() == on.device(), name, " must be on the device of x");
}
inline const float* opt_f32(const OptT& t, int64_t n, const Tensor& on, const char* name) {
  if (!given(t)) return nullptr;
  TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat && t->is_contiguous() && t->numel() == n, name, " must be contiguous fp32 of ", n, " values");
  TORCH_CHECK_VALUE(t->device() == on.device(), name, " must be on the device of the activations");
  return t->data_ptr<float>();
}

inline void check_tokens(const Tensor& x) {
  TORCH_CHECK_VALUE(x.dim() == 2, "x must be [tokens, channels]");
  TORCH_CHECK_VALUE(x.size(0) <= kMaxRows && x.size(1) <= kMaxRows, "at most ", kMaxRows, " rows and channels, got ", x.size(0), " and ", x.size(1));
}

// State pool [rows, c, n], rows / fresh / cu_seqlens of a call over the activation rows of x.
template <typename P>
void fill_sequences(P& p, const Tensor& x, const OptT& state, int64_t c, int64_t n, const OptT& rows, const OptT& fresh, const OptT& cu) {
  int64_t S = x.size(0);
  if (given(cu)) {
    TORCH_CHECK_VALUE(cu->scalar_type() == at::kInt && cu->dim() == 1 && cu->numel() >= 1 && cu->numel() <= kMaxRows && cu->is_contiguous() &&
                          cu->device() == x.device(),
                      "cu_seqlens must be a contiguous int32 vector on the device of x");
    S = cu->numel() - 1;
    p.cu_seqlens = cu->data_ptr<int>();
  } else {
    TORCH_CHECK_VALUE(S <= kMaxGrid, "a single-token step takes at most ", kMaxGrid, " rows, got ", S);
  }
  if (given(state)) {
    TORCH_CHECK_VALUE(state->scalar_type() == at::kFloat && state->is_contiguous() && state->dim() == 3 && state->size(1) == c && state->size(2) == n,
                      "state must be a contiguous fp32 pool [rows, ", c, ", ", n, "]");
    TORCH_CHECK_VALUE(state->device() == x.device(), "state must be on the device of x");
    TORCH_CHECK_VALUE(state->size(0) <= INT_MAX, "state has too many rows");
    p.state = state->data_ptr<float>();
    p.pool_rows = (int)state->size(0);
  } else {
    TORCH_CHECK_VALUE(given(cu), "a single-token step needs a state pool");
    TORCH_CHECK_VALUE(!given(rows), "rows name places of a state pool: pass state too");
  }
  if (given(rows)) {
    TORCH_CHECK_VALUE(rows->scalar_type() == at::kLong && rows->dim() == 1 && rows->numel() == S && rows->is_contiguous() && rows->device() == x.device(),
                      "rows must be a contiguous int64 vector with one entry per sequence (", S, ") on the device of x");
    p.rows = (const long long*)rows->data_ptr<int64_t>();
  } else if (given(state)) {
    TORCH_CHECK_VALUE(p.pool_rows >= S, "without rows, sequence i owns row i of state: it needs ", S, " rows");
  }
  if (given(fresh)) {
    TORCH_CHECK_VALUE((fresh->scalar_type() == at::kBool || fresh->scalar_type() == at::kByte) && fresh->dim() == 1 && fresh->numel() == S &&
                          fresh->is_contiguous() && fresh->device() == x.device(),
                      "fresh must be a contiguous bool or uint8 vector with one entry per sequence (", S, ") on the device of x");
    p.fresh = (const unsigned char*)fresh->data_ptr();
  }
  p.T = (int)x.size(0);
  p.S = (int)S;
}

void causal_conv(const Tensor& x, const Tensor& w, const OptT& bias, Tensor out, const OptT& state, const OptT& rows, const OptT& fresh,
                 const OptT& cu_seqlens, int64_t act, bool zero_dead) {
  check_tokens(x);
  const int64_t T = x.size(0), C = x.size(1);
  check_2d(x, T, C, x, "x");
  TORCH_CHECK_VALUE(w.dim() == 2 && w.size(0) == C && w.size(1) >= 2 && w.size(1) <= 8 && w.is_contiguous(), "w must be contiguous [", C, ", 2 .. 8]");
  TORCH_CHECK_VALUE(w.device() == x.device(), "w must be on the device of x");
  check_2d(out, T, C, x, "out");
  TORCH_CHECK_VALUE(act == 0 || act == 1, "act must be 0 (none) or 1 (SiLU)");
  MmbCausalConvParams p{};
  p.x = x.data_ptr();
  p.w = w.data_ptr();
  p.out = out.data_ptr();
  p.xt = elt_type(x, "x");
  p.wt = elt_type(w, "w");
  p.ot = elt_type(out, "out");
  if (given(bias)) {
    TORCH_CHECK_VALUE(bias->numel() == C && bias->is_contiguous() && bias->scalar_type() == w.scalar_type() && bias->device() == x.device(),
                      "bias must hold ", C, " values of w's type on the device of x");
    p.bias = bias->data_ptr();
  }
  p.ldx = x.stride(0);
  p.ldo = out.stride(0);
  p.K = (int)w.size(1);
  p.act = (int)act;
  p.zero_dead = zero_dead ? 1 : 0;
  fill_sequences(p, x, state, C, p.K - 1, rows, fresh, cu_seqlens);
  p.C = (int)C;
  TORCH_CHECK(x.is_cuda(), "causal_conv needs CUDA tensors");
  c10::cuda::CUDAGuard guard(x.device());
  p.status = mmb_status_word(x.device().index());
  check(p.cu_seqlens ? mmb_causal_conv(&p, cur_stream()) : mmb_causal_conv_step(&p, cur_stream()), "causal_conv");
}

void ssm(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const OptT& D, const OptT& z, const OptT& dt_bias,
         Tensor out, const OptT& state, const OptT& rows, const OptT& fresh, const OptT& cu_seqlens, bool softplus, bool zero_dead) {
  check_tokens(x);
  const int64_t T = x.size(0), Di = x.size(1);
  check_2d(x, T, Di, x, "x");
  check_2d(dt, T, Di, x, "dt");
  TORCH_CHECK_VALUE(A.dim() == 2 && A.size(0) == Di && A.size(1) >= 1 && A.size(1) <= 128 && A.scalar_type() == at::kFloat && A.is_contiguous() &&
                        A.device() == x.device(),
                    "A must be contiguous fp32 [", Di, ", 1 .. 128] on the device of x");
  const int64_t N = A.size(1);
  check_2d(B, T, N, x, "Bm");
  check_2d(C, T, N, x, "Cm");
  TORCH_CHECK_VALUE(B.scalar_type() == C.scalar_type(), "Bm and Cm must have one type");
  check_2d(out, T, Di, x, "out");
  MmbSsmParams p{};
  p.x = x.data_ptr();
  p.dt = dt.data_ptr();
  p.B = B.data_ptr();
  p.C = C.data_ptr();
  p.out = out.data_ptr();
  p.xt = elt_type(x, "x");
  p.dtt = elt_type(dt, "dt");
  p.bt = elt_type(B, "Bm");
  p.ot = elt_type(out, "out");
  if (given(z)) {
    check_2d(*z, T, Di, x, "z");
    p.z = z->data_ptr();
    p.zt = elt_type(*z, "z");
    p.ldz = z->stride(0);
  }
  p.A = A.data_ptr<float>();
  p.Dskip = opt_f32(D, Di, x, "D");
  p.dt_bias = opt_f32(dt_bias, Di, x, "dt_bias");
  p.ldx = x.stride(0);
  p.lddt = dt.stride(0);
  p.ldb = B.stride(0);
  p.ldc = C.stride(0);
  p.ldo = out.stride(0);
  p.N = (int)N;
  p.softplus = softplus ? 1 : 0;
  p.zero_dead = zero_dead ? 1 : 0;
  fill_sequences(p, x, state, Di, N, rows, fresh, cu_seqlens);
  p.D = (int)Di;
  TORCH_CHECK(x.is_cuda(), "ssm needs CUDA tensors");
  c10::cuda::CUDAGuard guard(x.device());
  p.status = mmb_status_word(x.device().index());
  check(p.cu_seqlens ? mmb_ssm_scan(&p, cur_stream()) : mmb_ssm_step(&p, cur_stream()), "ssm");
}

void sink_decode(const Tensor& q, const Tensor& k, const Tensor& v, const OptT& k_scale, const OptT& v_scale, const Tensor& block_tables,
                 const Tensor& ctx_lens, Tensor out, int64_t Hq, int64_t Hkv, int64_t D, int64_t block_size, double scale, int64_t window, int64_t sinks,
                 int64_t fmt, int64_t splits) {
  const int64_t B = ctx_lens.numel();
  TORCH_CHECK_VALUE(window >= 1 && window <= INT_MAX && sinks >= 0 && sinks <= INT_MAX, "sinks need a window of at least one token");
  TORCH_CHECK_VALUE(D == 64 || D == 128 || D == 256, "attention with sinks takes head sizes 64, 128 and 256, got ", D);
  TORCH_CHECK_VALUE(Hkv >= 1 && Hq >= 1 && Hq % Hkv == 0 && Hq <= INT_MAX, "query heads must be a multiple of KV heads");
  TORCH_CHECK_VALUE(block_size >= 1 && block_size <= INT_MAX, "block_size must be positive");
  TORCH_CHECK_VALUE(splits >= 0 && splits <= 8, "attention with sinks takes 1 to 8 splits, got ", splits);
  TORCH_CHECK_VALUE(q.scalar_type() == at::kBFloat16 && out.scalar_type() == at::kBFloat16, "q and out must be bf16");
  TORCH_CHECK_VALUE(q.is_contiguous() && q.numel() == B * Hq * D, "q must be contiguous with ", B * Hq * D, " values");
  TORCH_CHECK_VALUE(out.is_contiguous() && out.numel() == B * Hq * D, "out must be contiguous with ", B * Hq * D, " values");
  TORCH_CHECK_VALUE(block_tables.dim() == 2 && block_tables.size(0) == B && block_tables.scalar_type() == at::kInt && block_tables.is_contiguous() &&
                        ctx_lens.scalar_type() == at::kInt && ctx_lens.is_contiguous(),
                    "block_tables [B, blocks] and ctx_lens [B] must be contiguous int32");
  TORCH_CHECK_VALUE(B <= kMaxGrid, "attention with sinks takes at most ", kMaxGrid, " rows, got ", B);
  TORCH_CHECK_VALUE(block_tables.size(1) <= kMaxRows / block_size, "block_tables reaches more than ", kMaxRows, " tokens");
  TORCH_CHECK_VALUE(fmt >= -1 && fmt <= 3, "unknown cache format");
  const int64_t row = fmt >= 2 ? D / 2 : D;
  TORCH_CHECK_VALUE(k.scalar_type() == (fmt < 0 ? at::kBFloat16 : at::kByte) && v.scalar_type() == k.scalar_type(), "K and V pools have another type");
  TORCH_CHECK_VALUE(k.is_contiguous() && v.is_contiguous() && k.numel() == v.numel() && k.numel() % (Hkv * row) == 0,
                    "K and V pools must be contiguous [slots, ", Hkv, ", ", row, "]");
  MmbSinkDecodeParams p{};
  p.n_slots = k.numel() / (Hkv * row);
  TORCH_CHECK_VALUE(p.n_slots <= INT_MAX, "the pools have too many slots");
  if (fmt >= 0) {
    p.k_scale = opt_f32(k_scale, p.n_slots * Hkv, q, "k_scale");
    p.v_scale = opt_f32(v_scale, p.n_slots * Hkv, q, "v_scale");
    TORCH_CHECK_VALUE(given(k_scale) && given(v_scale), "a quantized pool has row scales");
  }
  for (const Tensor* t : {&k, &v, &block_tables, &ctx_lens, (const Tensor*)&out})
    TORCH_CHECK_VALUE(t->device() == q.device(), "all tensors must be on the device of q");
  for (const Tensor* t : {&q, &k, &v, (const Tensor*)&out})
    TORCH_CHECK_VALUE(reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0, "q, out and the pools must be 16-byte aligned");
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.block_tables = block_tables.data_ptr<int>();
  p.ctx_lens = ctx_lens.data_ptr<int>();
  p.out = out.data_ptr();
  p.B = (int)B;
  p.Hq = (int)Hq;
  p.Hkv = (int)Hkv;
  p.D = (int)D;
  p.block_size = (int)block_size;
  p.max_blocks = (int)block_tables.size(1);
  p.fmt = (int)fmt;
  p.window = (int)window;
  p.sinks = (int)sinks;
  p.scale = (float)scale;
  p.splits = (int)splits;
  TORCH_CHECK(q.is_cuda(), "sink_decode needs CUDA tensors");
  c10::cuda::CUDAGuard guard(q.device());
  p.status = mmb_status_word(q.device().index());
  check(mmb_sink_decode(&p, cur_stream()), "sink_decode");
}

// The same with an output that is made here: one call from Python instead of two.
Tensor causal_conv_new(const Tensor& x, const Tensor& w, const OptT& bias, const OptT& state, const OptT& rows, const OptT& fresh,
                       const OptT& cu_seqlens, int64_t act, c10::optional<at::ScalarType> out_dtype) {
  Tensor out = at::empty(x.sizes(), x.options().dtype(out_dtype.value_or(x.scalar_type())));
  causal_conv(x, w, bias, out, state, rows, fresh, cu_seqlens, act, true);
  return out;
}
Tensor ssm_new(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const OptT& D, const OptT& z, const OptT& dt_bias,
               const OptT& state, const OptT& rows, const OptT& fresh, const OptT& cu_seqlens, bool softplus, c10::optional<at::ScalarType> out_dtype) {
  Tensor out = at::empty(x.sizes(), x.options().dtype(out_dtype.value_or(x.scalar_type())));
  ssm(x, dt, A, B, C, D, z, dt_bias, out, state, rows, fresh, cu_seqlens, softplus, true);
  return out;
}
Tensor sink_decode_new(const Tensor& q, const Tensor& k, const Tensor& v, const OptT& k_scale, const OptT& v_scale, const Tensor& block_tables,
                       const Tensor& ctx_lens, int64_t Hq, int64_t Hkv, int64_t D, int64_t block_size, double scale, int64_t window, int64_t sinks,
                       int64_t fmt) {
  Tensor out = at::empty({ctx_lens.numel(), Hq, D}, q.options());
  sink_decode(q, k, v, k_scale, v_scale, block_tables, ctx_lens, out, Hq, Hkv, D, block_size, scale, window, sinks, fmt, 0);
  return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(mmb200, m) {
  m.def("causal_conv_new", &causal_conv_new);
  m.def("ssm_new", &ssm_new);
  m.def("sink_decode_new", &sink_decode_new);
  m.def("causal_conv", &causal_conv);
  m.def("ssm", &ssm);
  m.def("sink_decode", &sink_decode);
}
