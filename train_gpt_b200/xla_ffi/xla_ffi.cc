// XLA FFI handlers over the C ABI of libtrain_gpt_b200.so: what train-gpt's JAX code binds with
// jax.ffi.register_ffi_target / jax.ffi.ffi_call in place of jax.nn.scaled_matmul (fp8.py:70-76),
// the XLA quantisation fusions (fp8.py:39-47) and the Pallas norm (kernels.py:87-97).
//
// One handler per kernel entry point of include/train_gpt_b200.h; each is a thin adapter from
// XLA's buffers to one C call, on the stream XLA hands over.  Nothing here allocates: scratch and
// workspace arrive as extra result buffers that XLA plans, the status word as a result buffer
// the handler zeroes itself.
//
// Build (needs the XLA FFI headers that ship with jaxlib; see build.py next to this file):
//   g++ -O2 -std=c++17 -shared -fPIC -I$(python -c 'import jax.ffi; print(jax.ffi.include_dir())')
//       -I<repo>/include -I/usr/local/cuda/include xla_ffi.cc -L<repo>/train_gpt_b200
//       -ltrain_gpt_b200 -lcudart -o libtg_xla.so
#include <cuda_runtime_api.h>

#include <cstdint>
#include <string>

#include "train_gpt_b200.h"
#include "xla/ffi/api/ffi.h"

namespace ffi = xla::ffi;

namespace {

using Stream = ffi::PlatformStream<cudaStream_t>;
using BF16 = ffi::Buffer<ffi::BF16>;
using F8 = ffi::Buffer<ffi::F8E4M3FN>;
using F32 = ffi::Buffer<ffi::F32>;
using S32 = ffi::Buffer<ffi::S32>;
using U8 = ffi::Buffer<ffi::U8>;
using U32 = ffi::Buffer<ffi::U32>;
using RBF16 = ffi::ResultBuffer<ffi::BF16>;
using RF8 = ffi::ResultBuffer<ffi::F8E4M3FN>;
using RF32 = ffi::ResultBuffer<ffi::F32>;
using RS32 = ffi::ResultBuffer<ffi::S32>;
using RU8 = ffi::ResultBuffer<ffi::U8>;
using RU32 = ffi::ResultBuffer<ffi::U32>;

ffi::Error Check(int rc, const char* what) {
  if (rc == TG_OK) return ffi::Error::Success();
  const std::string msg = std::string(what) + " returned " + std::to_string(rc) +
                          (rc == TG_ERR_CUDA ? std::string(": ") + tg_last_cuda_error() : std::string());
  return ffi::Error(rc == TG_ERR_CUDA ? ffi::ErrorCode::kInternal : ffi::ErrorCode::kInvalidArgument, msg);
}

// rows x cols of a buffer whose last axis is the feature axis (leading axes are flattened,
// as fp8.py:65 and kernels.py:60-62 do)
template <typename B>
void RowsCols(const B& x, int64_t* rows, int64_t* cols) {
  auto d = x.dimensions();
  *cols = d.size() ? d.back() : 1;
  *rows = *cols ? static_cast<int64_t>(x.element_count()) / *cols : 0;
}

// ---- quantisers (fp8.py:39-47) ----------------------------------------------------------------

ffi::Error QuantizeRowwise(cudaStream_t s, BF16 x, RF8 q, RF32 scales) {
  int64_t rows, cols;
  RowsCols(x, &rows, &cols);
  return Check(tg_quantize_rowwise(x.untyped_data(), q->untyped_data(), scales->typed_data(), rows, cols, s),
               "tg_quantize_rowwise");
}

ffi::Error QuantizeColwise(cudaStream_t s, BF16 x, RF8 q, RF32 scales) {
  auto d = x.dimensions();
  if (d.size() != 2) return ffi::Error(ffi::ErrorCode::kInvalidArgument, "TgQuantizeColwise takes a 2-D operand");
  return Check(tg_quantize_colwise(x.untyped_data(), q->untyped_data(), scales->typed_data(), d[0], d[1], s),
               "tg_quantize_colwise");
}

ffi::Error QuantizeRowcol(cudaStream_t s, BF16 x, RF8 q_row, RF32 s_row, RF8 q_col, RF32 s_col) {
  auto d = x.dimensions();
  if (d.size() != 2) return ffi::Error(ffi::ErrorCode::kInvalidArgument, "TgQuantizeRowcol takes a 2-D operand");
  return Check(tg_quantize_rowcol(x.untyped_data(), q_row->untyped_data(), s_row->typed_data(), q_col->untyped_data(),
                                  s_col->typed_data(), d[0], d[1], s),
               "tg_quantize_rowcol");
}

// Both forms go into columns [col0, col0 + cols) of wider matrices that several calls fill side by side (the
// gradients of q, k and v for the one dgrad GEMM that contracts over all of them and the one wgrad GEMM that
// produces all three weight gradients).  XLA has no strided results: the four wide matrices come in as operands
// and go out as results aliased to them (input_output_aliases={1: 0, 2: 1, 3: 2, 4: 3} on the JAX side), so
// every call writes its slices in place.
ffi::Error QuantizeRowcolInto(cudaStream_t s, BF16 x, F8 wide_q_in, F32 wide_s_in, F8 wide_qc_in, F32 wide_sc_in, RF8 wide_q,
                              RF32 wide_s, RF8 wide_qc, RF32 wide_sc, int64_t col0) {
  auto d = x.dimensions();
  auto wq = wide_q->dimensions();
  auto ws = wide_s->dimensions();
  auto wqc = wide_qc->dimensions();
  auto wsc = wide_sc->dimensions();
  if (d.size() != 2 || wq.size() != 2 || ws.size() != 2 || wqc.size() != 2 || wsc.size() != 2 || wq[0] != d[0] ||
      ws[0] != d[0] || wqc[0] != d[0] || wsc[0] != (d[0] + 127) / 128 || col0 < 0 || col0 % 128 != 0 ||
      col0 + d[1] > wq[1] || (col0 + d[1]) / 128 > ws[1] || col0 + d[1] > wqc[1] || col0 + d[1] > wsc[1])
    return ffi::Error(ffi::ErrorCode::kInvalidArgument, "TgQuantizeRowcolInto: the slice does not fit the wide matrices");
  if (wide_q_in.untyped_data() != wide_q->untyped_data() || wide_s_in.untyped_data() != wide_s->untyped_data() ||
      wide_qc_in.untyped_data() != wide_qc->untyped_data() || wide_sc_in.untyped_data() != wide_sc->untyped_data())
    return ffi::Error(ffi::ErrorCode::kInvalidArgument, "TgQuantizeRowcolInto: declare input_output_aliases={1: 0, 2: 1, 3: 2, 4: 3}");
  return Check(tg_quantize_rowcol_ld(x.untyped_data(), static_cast<uint8_t*>(wide_q->untyped_data()) + col0, wq[1],
                                     wide_s->typed_data() + col0 / 128, ws[1],
                                     static_cast<uint8_t*>(wide_qc->untyped_data()) + col0, wqc[1],
                                     wide_sc->typed_data() + col0, wsc[1], d[0], d[1], s),
               "tg_quantize_rowcol_ld");
}

// act: TG_ACT_RELU2 / TG_ACT_GELU
ffi::Error ActQuantizeRowcol(cudaStream_t s, BF16 x, RF8 q_row, RF32 s_row, RF8 q_col, RF32 s_col, int32_t act) {
  auto d = x.dimensions();
  if (d.size() != 2) return ffi::Error(ffi::ErrorCode::kInvalidArgument, "TgActQuantizeRowcol takes a 2-D operand");
  return Check(tg_act_quantize_rowcol(x.untyped_data(), nullptr, act, q_row->untyped_data(), s_row->typed_data(),
                                      q_col->untyped_data(), s_col->typed_data(), d[0], d[1], s),
               "tg_act_quantize_rowcol");
}

// act: TG_ACT_RELU2_BWD / TG_ACT_GELU_BWD; gate = the gradient arriving at the activation's output
ffi::Error ActQuantizeRowcolBwd(cudaStream_t s, BF16 x, BF16 gate, RF8 q_row, RF32 s_row, RF8 q_col, RF32 s_col,
                                int32_t act) {
  auto d = x.dimensions();
  if (d.size() != 2) return ffi::Error(ffi::ErrorCode::kInvalidArgument, "TgActQuantizeRowcolBwd takes 2-D operands");
  return Check(tg_act_quantize_rowcol(x.untyped_data(), gate.untyped_data(), act, q_row->untyped_data(),
                                      s_row->typed_data(), q_col->untyped_data(), s_col->typed_data(), d[0], d[1], s),
               "tg_act_quantize_rowcol");
}

ffi::Error QuantizeBlock128(cudaStream_t s, BF16 x, RF8 q, RF32 scales) {
  auto d = x.dimensions();
  if (d.size() != 2) return ffi::Error(ffi::ErrorCode::kInvalidArgument, "TgQuantizeBlock128 takes a 2-D operand");
  return Check(tg_quantize_block128(x.untyped_data(), q->untyped_data(), scales->typed_data(), d[0], d[1], s),
               "tg_quantize_block128");
}

// ---- RMSNorm (kernels.py:30-33, 44-99, 104-118) -------------------------------------------------

ffi::Error RmsnormFwd(cudaStream_t s, BF16 x, BF16 gamma, RBF16 y, RF32 rnorm, float eps, int32_t mode) {
  int64_t rows, cols;
  RowsCols(x, &rows, &cols);
  return Check(tg_rmsnorm_fwd(x.untyped_data(), gamma.untyped_data(), eps, y->untyped_data(), rnorm->typed_data(), rows,
                              cols, mode, s),
               "tg_rmsnorm_fwd");
}

ffi::Error RmsnormQuantFwd(cudaStream_t s, BF16 x, BF16 gamma, RF8 q, RF32 scales, RBF16 y, RF32 rnorm, float eps,
                           int32_t mode) {
  int64_t rows, cols;
  RowsCols(x, &rows, &cols);
  return Check(tg_rmsnorm_quant_fwd(x.untyped_data(), gamma.untyped_data(), eps, q->untyped_data(), scales->typed_data(),
                                    y->untyped_data(), rnorm->typed_data(), rows, cols, mode, s),
               "tg_rmsnorm_quant_fwd");
}

// the residual add folded into the norm that follows it (model.py:68 / :72 then :76-77); rows of at most 2048
ffi::Error AddRmsnormQuantFwd(cudaStream_t s, BF16 x, BF16 res, BF16 gamma, RBF16 sum, RF8 q, RF32 scales, RBF16 y, RF32 rnorm,
                              float eps, int32_t mode) {
  int64_t rows, cols;
  RowsCols(x, &rows, &cols);
  return Check(tg_add_rmsnorm_quant_fwd(x.untyped_data(), res.untyped_data(), gamma.untyped_data(), eps, sum->untyped_data(),
                                        q->untyped_data(), scales->typed_data(), y->untyped_data(), rnorm->typed_data(), rows,
                                        cols, mode, s),
               "tg_add_rmsnorm_quant_fwd");
}

// scratch: a result buffer of tg_rmsnorm_bwd_scratch_bytes(rows, cols) bytes that XLA plans
ffi::Error RmsnormBwd(cudaStream_t s, BF16 x, BF16 gamma, BF16 g, RBF16 dx, RBF16 dgamma, RU8 scratch, float eps) {
  int64_t rows, cols;
  RowsCols(x, &rows, &cols);
  if (static_cast<int64_t>(scratch->element_count()) < tg_rmsnorm_bwd_scratch_bytes(rows, cols))
    return ffi::Error(ffi::ErrorCode::kInvalidArgument, "TgRmsnormBwd: scratch result smaller than tg_rmsnorm_bwd_scratch_bytes");
  return Check(tg_rmsnorm_bwd(x.untyped_data(), gamma.untyped_data(), g.untyped_data(), eps, dx->untyped_data(),
                              dgamma->untyped_data(), scratch->untyped_data(), rows, cols, s),
               "tg_rmsnorm_bwd");
}

// the backward with the skip path's gradient added in the same pass; rows of at most 2048
ffi::Error RmsnormBwdAdd(cudaStream_t s, BF16 x, BF16 gamma, BF16 g, BF16 addend, RBF16 dx, RBF16 dgamma, RU8 scratch, float eps) {
  int64_t rows, cols;
  RowsCols(x, &rows, &cols);
  if (static_cast<int64_t>(scratch->element_count()) < tg_rmsnorm_bwd_scratch_bytes(rows, cols))
    return ffi::Error(ffi::ErrorCode::kInvalidArgument, "TgRmsnormBwdAdd: scratch result smaller than tg_rmsnorm_bwd_scratch_bytes");
  return Check(tg_rmsnorm_bwd_add(x.untyped_data(), gamma.untyped_data(), g.untyped_data(), addend.untyped_data(), eps,
                                  dx->untyped_data(), dgamma->untyped_data(), scratch->untyped_data(), rows, cols, s),
               "tg_rmsnorm_bwd_add");
}

// the same backward with the scratch inside the library (fixed 4 MiB array; see the header)
ffi::Error RmsnormBwdStatic(cudaStream_t s, BF16 x, BF16 gamma, BF16 g, RBF16 dx, RBF16 dgamma, float eps) {
  int64_t rows, cols;
  RowsCols(x, &rows, &cols);
  return Check(tg_rmsnorm_bwd_static(x.untyped_data(), gamma.untyped_data(), g.untyped_data(), eps, dx->untyped_data(),
                                     dgamma->untyped_data(), rows, cols, s),
               "tg_rmsnorm_bwd_static");
}

// ---- capped-logit cross-entropy (model.py:97, losses.py:8-12) -------------------------------------

// logits (rows, ld) with ld a multiple of 8 >= vocab (pad on the JAX side for a ragged vocabulary)
ffi::Error SoftcapCeFwd(cudaStream_t s, BF16 logits, S32 targets, RBF16 tanh_out, RF32 lse, RF32 nll, float cap,
                        int64_t vocab) {
  int64_t rows, ld;
  RowsCols(logits, &rows, &ld);
  return Check(tg_softcap_ce_fwd(logits.untyped_data(), targets.typed_data(), cap, tanh_out->untyped_data(),
                                 lse->typed_data(), nll->typed_data(), rows, vocab, ld, ld, s),
               "tg_softcap_ce_fwd");
}

// dlogits may alias tanh_in (declare input_output_aliases={0: 0} on the JAX side)
ffi::Error SoftcapCeBwd(cudaStream_t s, BF16 tanh_in, S32 targets, F32 lse, F32 gscale, RBF16 dlogits, float cap,
                        int64_t vocab) {
  int64_t rows, ld;
  RowsCols(tanh_in, &rows, &ld);
  return Check(tg_softcap_ce_bwd(tanh_in.untyped_data(), targets.typed_data(), lse.typed_data(), gscale.typed_data(), cap,
                                 dlogits->untyped_data(), rows, vocab, ld, ld, s),
               "tg_softcap_ce_bwd");
}

// whether each of these buffers has n elements
template <typename... B>
bool Have(int64_t n, const B&... b) {
  return ((static_cast<int64_t>(b.element_count()) == n) && ...);
}
ffi::Error Mismatch(const char* what) { return ffi::Error(ffi::ErrorCode::kInvalidArgument, what); }

// ---- the junction of blocks with a norm on both sides (no counterpart) -----------------------------

bool HaveGate(int32_t kind, int64_t rows, int64_t cols, const BF16& gate) {
  return kind == TG_GATE_NONE || (kind == TG_GATE_CHANNEL && Have(cols, gate)) || (kind == TG_GATE_TOKEN && Have(rows, gate));
}

// gate_kind: TG_GATE_NONE (pass any bf16 buffer), TG_GATE_CHANNEL (cols,) or TG_GATE_TOKEN (rows,)
ffi::Error SandwichNormFwd(cudaStream_t s, BF16 x, BF16 branch, BF16 post, BF16 pre, BF16 gate, RBF16 x_new, RBF16 h, int32_t gate_kind,
                           float residual_scale, float eps) {
  int64_t rows, cols;
  RowsCols(x, &rows, &cols);
  if (!Have(rows * cols, branch, *x_new, *h) || !Have(cols, post, pre) || !HaveGate(gate_kind, rows, cols, gate))
    return Mismatch("TgSandwichNormFwd: branch, x_new and h must be like x, post and pre (cols,), gate (cols,) or (rows,) as gate_kind says");
  return Check(tg_sandwich_norm_fwd(x.untyped_data(), branch.untyped_data(), post.untyped_data(), pre.untyped_data(), gate.untyped_data(), gate_kind,
                                    residual_scale, eps, x_new->untyped_data(), h->untyped_data(), nullptr, nullptr, rows, cols, s),
               "tg_sandwich_norm_fwd");
}

ffi::Error SandwichNormQuantFwd(cudaStream_t s, BF16 x, BF16 branch, BF16 post, BF16 pre, BF16 gate, RBF16 x_new, RBF16 h, RF8 q, RF32 scales,
                                int32_t gate_kind, float residual_scale, float eps) {
  int64_t rows, cols;
  RowsCols(x, &rows, &cols);
  if (!Have(rows * cols, branch, *x_new, *h, *q) || !Have(cols, post, pre) || !HaveGate(gate_kind, rows, cols, gate) || !Have(rows * (cols / 128), *scales))
    return Mismatch("TgSandwichNormQuantFwd: branch, x_new, h and q must be like x, scales (rows, cols / 128), post and pre (cols,), gate (cols,) or (rows,) as gate_kind says");
  return Check(tg_sandwich_norm_fwd(x.untyped_data(), branch.untyped_data(), post.untyped_data(), pre.untyped_data(), gate.untyped_data(), gate_kind,
                                    residual_scale, eps, x_new->untyped_data(), h->untyped_data(), q->untyped_data(), scales->typed_data(), rows,
                                    cols, s),
               "tg_sandwich_norm_fwd");
}

// dgate has the gate's shape; scratch: tg_sandwich_norm_bwd_scratch_bytes(rows, cols) bytes that XLA plans
ffi::Error SandwichNormBwd(cudaStream_t s, BF16 x_new, BF16 branch, BF16 post, BF16 pre, BF16 gate, BF16 g_new, BF16 g_h, RBF16 dx, RBF16 dbranch,
                           RBF16 dpost, RBF16 dpre, RBF16 dgate, RU8 scratch, int32_t gate_kind, float residual_scale, float eps) {
  int64_t rows, cols;
  RowsCols(x_new, &rows, &cols);
  if (!Have(rows * cols, branch, g_new, g_h, *dx, *dbranch) || !Have(cols, post, pre, *dpost, *dpre) || !HaveGate(gate_kind, rows, cols, gate) ||
      !HaveGate(gate_kind, rows, cols, *dgate))
    return Mismatch("TgSandwichNormBwd: branch, gradients, dx and dbranch must be like x_new, post, pre and theirs (cols,), gate and dgate (cols,) or (rows,) as gate_kind says");
  if (static_cast<int64_t>(scratch->element_count()) < tg_sandwich_norm_bwd_scratch_bytes(rows, cols))
    return ffi::Error(ffi::ErrorCode::kInvalidArgument, "TgSandwichNormBwd: scratch result smaller than tg_sandwich_norm_bwd_scratch_bytes");
  return Check(tg_sandwich_norm_bwd(x_new.untyped_data(), branch.untyped_data(), post.untyped_data(), pre.untyped_data(), gate.untyped_data(), gate_kind,
                                    residual_scale, eps, g_new.untyped_data(), g_h.untyped_data(), dx->untyped_data(), dbranch->untyped_data(),
                                    dpost->untyped_data(), dpre->untyped_data(), dgate->untyped_data(), scratch->untyped_data(), rows, cols, s),
               "tg_sandwich_norm_bwd");
}

// ---- distillation from a teacher's top logits (no counterpart) --------------------------------------

// ids, logp (rows, k), log_rest (rows,)
ffi::Error TopLogits(cudaStream_t s, BF16 logits, RS32 ids, RF32 logp, RF32 log_rest, float cap, float temperature) {
  int64_t rows, vocab;
  RowsCols(logits, &rows, &vocab);
  auto d = ids->dimensions();
  const int64_t k = d.size() ? d.back() : 0;
  if (k > TG_TOP_LOGITS_MAX || !Have(rows * k, *ids, *logp) || !Have(rows, *log_rest))
    return Mismatch("TgTopLogits: ids and logp must be (rows, k), log_rest (rows,)");
  return Check(tg_top_logits(logits.untyped_data(), cap, temperature, ids->typed_data(), logp->typed_data(), log_rest->typed_data(), rows, vocab, vocab,
                             static_cast<int>(k), s),
               "tg_top_logits");
}

// The rows' losses and the gradient of their mean from one read of the logits: a custom_vjp's forward rule, whose backward rule
// multiplies by the cotangent.  targets of -1 where there are none.
ffi::Error SoftcapDistill(cudaStream_t s, BF16 logits, S32 ids, F32 logp, F32 log_rest, S32 targets, RF32 row_loss, RBF16 dlogits, float cap,
                          float temperature, float weight) {
  tg_distill_args a = {};
  RowsCols(logits, &a.rows, &a.vocab);
  auto d = ids.dimensions();
  const int64_t k = d.size() ? d.back() : 0;
  if (k > TG_TOP_LOGITS_MAX || !Have(a.rows * k, ids, logp) || !Have(a.rows, log_rest, targets, *row_loss) || !Have(a.rows * a.vocab, *dlogits))
    return Mismatch("TgSoftcapDistill: ids and logp must be (rows, k), log_rest, targets and row_loss (rows,), dlogits like logits");
  a.logits = logits.untyped_data(); a.ids = ids.untyped_data(); a.logp = logp.typed_data(); a.log_rest = log_rest.typed_data();
  a.targets = targets.untyped_data(); a.cap = cap; a.temperature = temperature; a.weight = weight;
  a.dlogits = dlogits->untyped_data(); a.row_loss = row_loss->typed_data();
  a.ld = a.vocab; a.k = static_cast<int>(k);
  return Check(tg_softcap_distill(&a, s), "tg_softcap_distill");
}

// ---- rotary positions, the gated feed-forward, dropout (no counterpart) -----------------------------

// q (batch, tokens, heads, dim), k (batch, tokens, kv_heads, dim), contiguous; positions (batch, tokens)
bool QkArgs(const BF16& q, const BF16& k, const BF16& q_scale, const BF16& k_scale, const S32& positions, bool norm, tg_qk_args* a) {
  auto d = q.dimensions();
  auto e = k.dimensions();
  if (d.size() != 4 || e.size() != 4 || d[0] != e[0] || d[1] != e[1] || d[3] != e[3]) return false;
  if (!Have(d[0] * d[1], positions) || (norm && !Have(d[3], q_scale, k_scale))) return false;
  for (int64_t n : {d[2], e[2], d[3]})
    if (n > 65536) return false;
  a->batch = d[0]; a->tokens = d[1]; a->heads = static_cast<int>(d[2]); a->kv_heads = static_cast<int>(e[2]); a->dim = static_cast<int>(d[3]);
  int64_t* strides[4] = {a->q_stride, a->g_q_stride, a->k_stride, a->g_k_stride};
  for (int i = 0; i < 4; ++i) {
    const int64_t heads = i < 2 ? d[2] : e[2];
    strides[i][0] = d[1] * heads * d[3]; strides[i][1] = heads * d[3]; strides[i][2] = d[3];
  }
  a->q = q.untyped_data(); a->k = k.untyped_data();
  if (norm) { a->q_scale = q_scale.untyped_data(); a->k_scale = k_scale.untyped_data(); }
  a->positions = positions.untyped_data(); a->positions_stride[0] = d[1]; a->positions_stride[1] = 1;
  return true;
}

// norm 0: the rotation alone (pass any bf16 buffers for the scales)
ffi::Error QkNormRopeFwd(cudaStream_t s, BF16 q, BF16 k, BF16 q_scale, BF16 k_scale, S32 positions, RBF16 q_out, RBF16 k_out, int32_t norm, float eps,
                         double theta, int32_t rotary_dim, int32_t interleaved) {
  tg_qk_args a = {};
  if (!QkArgs(q, k, q_scale, k_scale, positions, norm != 0, &a) || !Have(static_cast<int64_t>(q.element_count()), *q_out) ||
      !Have(static_cast<int64_t>(k.element_count()), *k_out))
    return Mismatch("TgQkNormRopeFwd: q and k must be (batch, tokens, heads, dim) of one batch, tokens and dim, the results like them, scales (dim,), positions (batch, tokens)");
  a.eps = eps; a.theta = theta; a.rotary_dim = rotary_dim; a.interleaved = interleaved;
  a.q_out = q_out->untyped_data(); a.k_out = k_out->untyped_data();
  return Check(tg_qk_norm_rope_fwd(&a, s), "tg_qk_norm_rope_fwd");
}

// scratch: tg_qk_norm_rope_bwd_scratch_bytes bytes that XLA plans; dq_scale and dk_scale are left alone with norm 0
ffi::Error QkNormRopeBwd(cudaStream_t s, BF16 q, BF16 k, BF16 q_scale, BF16 k_scale, S32 positions, BF16 g_q, BF16 g_k, RBF16 dq, RBF16 dk, RBF16 dq_scale,
                         RBF16 dk_scale, RU8 scratch, int32_t norm, float eps, double theta, int32_t rotary_dim, int32_t interleaved) {
  tg_qk_args a = {};
  if (!QkArgs(q, k, q_scale, k_scale, positions, norm != 0, &a) || !Have(static_cast<int64_t>(q.element_count()), g_q, *dq) ||
      !Have(static_cast<int64_t>(k.element_count()), g_k, *dk) || (norm != 0 && !Have(a.dim, *dq_scale, *dk_scale)))
    return Mismatch("TgQkNormRopeBwd: gradients and results must be like q and k, scales and their gradients (dim,), positions (batch, tokens)");
  a.eps = eps; a.theta = theta; a.rotary_dim = rotary_dim; a.interleaved = interleaved;
  if (static_cast<int64_t>(scratch->element_count()) < tg_qk_norm_rope_bwd_scratch_bytes(&a))
    return Mismatch("TgQkNormRopeBwd: scratch result smaller than tg_qk_norm_rope_bwd_scratch_bytes");
  a.g_q = g_q.untyped_data(); a.g_k = g_k.untyped_data();
  a.q_out = dq->untyped_data(); a.k_out = dk->untyped_data();
  a.dq_scale = dq_scale->untyped_data(); a.dk_scale = dk_scale->untyped_data(); a.scratch = scratch->untyped_data();
  return Check(tg_qk_norm_rope_bwd(&a, s), "tg_qk_norm_rope_bwd");
}

// what both directions of the gated feed-forward are called with; `inner` values per row in h or its gradient
bool GatedArgs(cudaStream_t s, const BF16& x, const BF16& w_gate, const BF16& w_up, int64_t outer, RU32& status, tg_gated_args* a) {
  RowsCols(x, &a->rows, &a->cols);
  auto d = w_gate.dimensions();
  if (d.size() != 2 || d[0] != a->cols || !Have(d[0] * d[1], w_up) || outer != a->rows * d[1] || !Have(1, *status)) return false;
  a->inner = d[1];
  a->ldx = a->cols; a->ld_gate = a->ld_up = a->inner;
  a->x = x.untyped_data(); a->w_gate = w_gate.untyped_data(); a->w_up = w_up.untyped_data();
  a->status = status->typed_data();
  return cudaMemsetAsync(a->status, 0, sizeof(uint32_t), s) == cudaSuccess;
}

// saved_gate, saved_up: 2 rows inner bytes each, exponents tg_gated_linear_exponent_bytes (a custom_vjp's residuals); status (1,)
ffi::Error GatedLinearFwd(cudaStream_t s, BF16 x, BF16 w_gate, BF16 w_up, RBF16 h, RU8 saved_gate, RU8 saved_up, RU8 exponents, RU32 status, int32_t act) {
  tg_gated_args a = {};
  if (!GatedArgs(s, x, w_gate, w_up, static_cast<int64_t>(h->element_count()), status, &a) || !Have(2 * a.rows * a.inner, *saved_gate, *saved_up) ||
      static_cast<int64_t>(exponents->element_count()) < tg_gated_linear_exponent_bytes(a.rows, a.inner))
    return Mismatch("TgGatedLinearFwd: weights must be (cols, inner), h (rows, inner), saved results 2 rows inner bytes, exponents tg_gated_linear_exponent_bytes, status (1,)");
  a.act = act; a.h = h->untyped_data();
  a.saved_gate = saved_gate->untyped_data(); a.saved_up = saved_up->untyped_data(); a.saved_exponents = exponents->typed_data();
  return Check(tg_gated_linear_fwd(&a, s), "tg_gated_linear_fwd");
}

ffi::Error GatedLinearBwd(cudaStream_t s, BF16 x, BF16 w_gate, BF16 w_up, U8 saved_gate, U8 saved_up, U8 exponents, BF16 g, RBF16 dx, RBF16 dw_gate,
                          RBF16 dw_up, RU8 scratch, RU32 status, int32_t act) {
  tg_gated_args a = {};
  if (!GatedArgs(s, x, w_gate, w_up, static_cast<int64_t>(g.element_count()), status, &a) || !Have(2 * a.rows * a.inner, saved_gate, saved_up) ||
      !Have(a.rows * a.cols, *dx) || !Have(a.cols * a.inner, *dw_gate, *dw_up) ||
      static_cast<int64_t>(exponents.element_count()) < tg_gated_linear_exponent_bytes(a.rows, a.inner))
    return Mismatch("TgGatedLinearBwd: g must be (rows, inner), results like x and the weights, saved buffers as TgGatedLinearFwd's");
  a.act = act; a.g = g.untyped_data();
  a.saved_gate = saved_gate.untyped_data(); a.saved_up = saved_up.untyped_data(); a.saved_exponents = exponents.typed_data();
  a.dx = dx->untyped_data(); a.dw_gate = dw_gate->untyped_data(); a.dw_up = dw_up->untyped_data(); a.scratch = scratch->untyped_data();
  a.scratch_bytes = static_cast<int64_t>(scratch->element_count());
  if (a.scratch_bytes < tg_gated_linear_bwd_scratch_bytes(&a)) return Mismatch("TgGatedLinearBwd: scratch result smaller than tg_gated_linear_bwd_scratch_bytes");
  return Check(tg_gated_linear_bwd(&a, s), "tg_gated_linear_bwd");
}

// seed: two words, low and high (a JAX PRNG key is that); site: site bits of the attribute.  TgDropout without a residual is its own backward rule.
ffi::Error Dropout(cudaStream_t s, BF16 x, U32 seed, RBF16 y, double p, int32_t site) {
  const int64_t n = static_cast<int64_t>(x.element_count());
  if (!Have(2, seed) || !Have(n, *y)) return Mismatch("TgDropout: seed must be two words, y like x");
  return Check(tg_dropout(x.untyped_data(), nullptr, p, static_cast<const int64_t*>(seed.untyped_data()), static_cast<uint32_t>(site), y->untyped_data(), n, s),
               "tg_dropout");
}
ffi::Error DropoutAdd(cudaStream_t s, BF16 x, BF16 residual, U32 seed, RBF16 y, double p, int32_t site) {
  const int64_t n = static_cast<int64_t>(x.element_count());
  if (!Have(2, seed) || !Have(n, residual, *y)) return Mismatch("TgDropoutAdd: seed must be two words, residual and y like x");
  return Check(tg_dropout(x.untyped_data(), residual.untyped_data(), p, static_cast<const int64_t*>(seed.untyped_data()), static_cast<uint32_t>(site),
                          y->untyped_data(), n, s),
               "tg_dropout");
}

// ---- optimiser (train.py:114-123, 132-134) --------------------------------------------------------

ffi::Error SumsqBf16(cudaStream_t s, BF16 x, RF32 out, RU8 scratch) {
  if (static_cast<int64_t>(scratch->element_count()) < tg_sumsq_scratch_bytes())
    return ffi::Error(ffi::ErrorCode::kInvalidArgument, "TgSumsqBf16: scratch result smaller than tg_sumsq_scratch_bytes");
  return Check(tg_sumsq_bf16(x.untyped_data(), static_cast<int64_t>(x.element_count()), out->typed_data(),
                             scratch->untyped_data(), s),
               "tg_sumsq_bf16");
}

// p, m, v are updated in place: bind with input_output_aliases={0: 0, 2: 1, 3: 2}
ffi::Error AdamwBf16(cudaStream_t s, BF16 p, BF16 g, BF16 m, BF16 v, S32 step, F32 gscale, RBF16 p_out, RBF16 m_out,
                     RBF16 v_out, float lr, float b1, float b2, float eps, float weight_decay) {
  if (p_out->untyped_data() != p.untyped_data() || m_out->untyped_data() != m.untyped_data() ||
      v_out->untyped_data() != v.untyped_data())
    return ffi::Error(ffi::ErrorCode::kInvalidArgument, "TgAdamwBf16 updates in place: alias p, m, v to the results");
  return Check(tg_adamw_bf16(p_out->untyped_data(), g.untyped_data(), m_out->untyped_data(), v_out->untyped_data(),
                             static_cast<int64_t>(p.element_count()), lr, b1, b2, eps, weight_decay, step.typed_data(),
                             gscale.typed_data(), s),
               "tg_adamw_bf16");
}

// ---- block-scaled GEMM (fp8.py:70-78 and the FP8 form of fp8.py:96-97) ------------------------------

// Common tail: zero the status word, attach the workspace XLA planned (may be empty), launch.
ffi::Error LaunchGemm(cudaStream_t s, tg_gemm_args* g, RU32& status, RU8& workspace) {
  if (cudaMemsetAsync(status->typed_data(), 0, sizeof(uint32_t), s) != cudaSuccess)
    return ffi::Error(ffi::ErrorCode::kInternal, "cudaMemsetAsync(status) failed");
  g->status = status->typed_data();
  const int64_t need = tg_gemm_workspace_bytes(g);
  if (need > 0 && static_cast<int64_t>(workspace->element_count()) >= need) {
    g->workspace = workspace->untyped_data();
    g->workspace_bytes = static_cast<int64_t>(workspace->element_count());
  }
  return Check(tg_gemm_fp8_blockscaled(g, s), "tg_gemm_fp8_blockscaled");
}

// y = x W.  a (M, K) row-wise quantised, sa (M, K/128); b (K, N) as stored (no b.T), sb (K/128, N) for
// weight_gran 1 [the reference's granularity] or (K/128, N/128) for weight_gran 128.
ffi::Error GemmFwd(cudaStream_t s, F8 a, F32 sa, F8 b, F32 sb, RBF16 y, RU32 status, RU8 workspace, int32_t weight_gran) {
  const int64_t M = a.dimensions()[0], K = a.dimensions()[1], N = b.dimensions()[1];
  tg_gemm_args g = {};
  g.a = a.untyped_data(); g.lda = K; g.a_major = TG_MAJOR_K;
  g.b = b.untyped_data(); g.ldb = N; g.b_major = TG_MAJOR_MN;
  g.sa = sa.typed_data(); g.sa_stride_m = sa.dimensions()[1]; g.sa_stride_kb = 1;
  g.sb = sb.typed_data(); g.sb_stride_n = 1; g.sb_stride_kb = sb.dimensions()[1]; g.sb_gran_n = weight_gran;
  g.d = y->untyped_data(); g.ldd = N; g.out_dtype = TG_OUT_BF16;
  g.M = M; g.N = N; g.K = K;
  return LaunchGemm(s, &g, status, workspace);
}

// dx = g W^T (contracts N).  g (M, N) row-wise quantised, sg (M, N/128); w (K, N) quantised along N:
// sw (K, N/128) for weight_gran 1, or the forward's (K/128, N/128) tiles for weight_gran 128.
ffi::Error GemmDgrad(cudaStream_t s, F8 gq, F32 sg, F8 w, F32 sw, RBF16 dx, RU32 status, RU8 workspace,
                     int32_t weight_gran) {
  const int64_t M = gq.dimensions()[0], N = gq.dimensions()[1], K = w.dimensions()[0];
  tg_gemm_args g = {};
  g.a = gq.untyped_data(); g.lda = N; g.a_major = TG_MAJOR_K;
  g.b = w.untyped_data(); g.ldb = N; g.b_major = TG_MAJOR_K;
  g.sa = sg.typed_data(); g.sa_stride_m = sg.dimensions()[1]; g.sa_stride_kb = 1;
  g.sb = sw.typed_data(); g.sb_stride_n = sw.dimensions()[1]; g.sb_stride_kb = 1; g.sb_gran_n = weight_gran;
  g.d = dx->untyped_data(); g.ldd = K; g.out_dtype = TG_OUT_BF16;
  g.M = M; g.N = K; g.K = N;
  return LaunchGemm(s, &g, status, workspace);
}

// dW = x^T g (contracts the tokens).  x (T, K) and g (T, N) column-wise quantised (128 tokens x 1):
// sx (ceil(T/128), K), sg (ceil(T/128), N) for grad_gran 1 or (ceil(T/128), N/128) for grad_gran 128.
ffi::Error GemmWgrad(cudaStream_t s, F8 xq, F32 sx, F8 gq, F32 sg, RBF16 dw, RU32 status, RU8 workspace,
                     int32_t grad_gran) {
  const int64_t T = xq.dimensions()[0], K = xq.dimensions()[1], N = gq.dimensions()[1];
  tg_gemm_args g = {};
  g.a = xq.untyped_data(); g.lda = K; g.a_major = TG_MAJOR_MN;
  g.b = gq.untyped_data(); g.ldb = N; g.b_major = TG_MAJOR_MN;
  g.sa = sx.typed_data(); g.sa_stride_m = 1; g.sa_stride_kb = K;
  g.sb = sg.typed_data(); g.sb_stride_n = 1; g.sb_stride_kb = sg.dimensions()[1]; g.sb_gran_n = grad_gran;
  g.d = dw->untyped_data(); g.ldd = N; g.out_dtype = TG_OUT_BF16;
  g.M = K; g.N = N; g.K = T;
  return LaunchGemm(s, &g, status, workspace);
}

}  // namespace

#define TG_QUANT_BINDING ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Ret<F8>().Ret<F32>()

XLA_FFI_DEFINE_HANDLER_SYMBOL(TgQuantizeRowwise, QuantizeRowwise, TG_QUANT_BINDING);
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgQuantizeColwise, QuantizeColwise, TG_QUANT_BINDING);
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgQuantizeBlock128, QuantizeBlock128, TG_QUANT_BINDING);
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgQuantizeRowcol, QuantizeRowcol,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Ret<F8>().Ret<F32>().Ret<F8>().Ret<F32>());
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgQuantizeRowcolInto, QuantizeRowcolInto,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Arg<F8>().Arg<F32>().Arg<F8>().Arg<F32>()
                                  .Ret<F8>().Ret<F32>().Ret<F8>().Ret<F32>().Attr<int64_t>("col0"));
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgActQuantizeRowcol, ActQuantizeRowcol,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Ret<F8>().Ret<F32>().Ret<F8>().Ret<F32>()
                                  .Attr<int32_t>("act"));
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgActQuantizeRowcolBwd, ActQuantizeRowcolBwd,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Arg<BF16>().Ret<F8>().Ret<F32>().Ret<F8>().Ret<F32>()
                                  .Attr<int32_t>("act"));
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgRmsnormFwd, RmsnormFwd,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Arg<BF16>().Ret<BF16>().Ret<F32>()
                                  .Attr<float>("eps").Attr<int32_t>("mode"));
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgRmsnormQuantFwd, RmsnormQuantFwd,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Arg<BF16>().Ret<F8>().Ret<F32>().Ret<BF16>().Ret<F32>()
                                  .Attr<float>("eps").Attr<int32_t>("mode"));
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgAddRmsnormQuantFwd, AddRmsnormQuantFwd,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Arg<BF16>().Arg<BF16>().Ret<BF16>().Ret<F8>().Ret<F32>()
                                  .Ret<BF16>().Ret<F32>().Attr<float>("eps").Attr<int32_t>("mode"));
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgRmsnormBwdAdd, RmsnormBwdAdd,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Arg<BF16>().Arg<BF16>().Arg<BF16>().Ret<BF16>().Ret<BF16>()
                                  .Ret<U8>().Attr<float>("eps"));
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgRmsnormBwd, RmsnormBwd,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Arg<BF16>().Arg<BF16>().Ret<BF16>().Ret<BF16>().Ret<U8>()
                                  .Attr<float>("eps"));
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgRmsnormBwdStatic, RmsnormBwdStatic,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Arg<BF16>().Arg<BF16>().Ret<BF16>().Ret<BF16>()
                                  .Attr<float>("eps"));
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgSoftcapCeFwd, SoftcapCeFwd,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Arg<S32>().Ret<BF16>().Ret<F32>().Ret<F32>()
                                  .Attr<float>("cap").Attr<int64_t>("vocab"));
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgSoftcapCeBwd, SoftcapCeBwd,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Arg<S32>().Arg<F32>().Arg<F32>().Ret<BF16>()
                                  .Attr<float>("cap").Attr<int64_t>("vocab"));
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgSumsqBf16, SumsqBf16, ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Ret<F32>().Ret<U8>());
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgAdamwBf16, AdamwBf16,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Arg<BF16>().Arg<BF16>().Arg<BF16>().Arg<S32>().Arg<F32>()
                                  .Ret<BF16>().Ret<BF16>().Ret<BF16>()
                                  .Attr<float>("lr").Attr<float>("b1").Attr<float>("b2").Attr<float>("eps")
                                  .Attr<float>("weight_decay"));

#define TG_GEMM_BINDING(attr) \
  ffi::Ffi::Bind().Ctx<Stream>().Arg<F8>().Arg<F32>().Arg<F8>().Arg<F32>().Ret<BF16>().Ret<U32>().Ret<U8>().Attr<int32_t>(attr)

XLA_FFI_DEFINE_HANDLER_SYMBOL(TgGemmFwd, GemmFwd, TG_GEMM_BINDING("weight_gran"));
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgGemmDgrad, GemmDgrad, TG_GEMM_BINDING("weight_gran"));
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgGemmWgrad, GemmWgrad, TG_GEMM_BINDING("grad_gran"));
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgSandwichNormFwd, SandwichNormFwd,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Arg<BF16>().Arg<BF16>().Arg<BF16>().Arg<BF16>().Ret<BF16>().Ret<BF16>()
                                  .Attr<int32_t>("gate_kind").Attr<float>("residual_scale").Attr<float>("eps"));
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgSandwichNormQuantFwd, SandwichNormQuantFwd,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Arg<BF16>().Arg<BF16>().Arg<BF16>().Arg<BF16>().Ret<BF16>().Ret<BF16>()
                                  .Ret<F8>().Ret<F32>().Attr<int32_t>("gate_kind").Attr<float>("residual_scale").Attr<float>("eps"));
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgSandwichNormBwd, SandwichNormBwd,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Arg<BF16>().Arg<BF16>().Arg<BF16>().Arg<BF16>().Arg<BF16>().Arg<BF16>()
                                  .Ret<BF16>().Ret<BF16>().Ret<BF16>().Ret<BF16>().Ret<BF16>().Ret<U8>()
                                  .Attr<int32_t>("gate_kind").Attr<float>("residual_scale").Attr<float>("eps"));
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgTopLogits, TopLogits,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Ret<S32>().Ret<F32>().Ret<F32>().Attr<float>("cap")
                                  .Attr<float>("temperature"));
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgSoftcapDistill, SoftcapDistill,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Arg<S32>().Arg<F32>().Arg<F32>().Arg<S32>().Ret<F32>().Ret<BF16>()
                                  .Attr<float>("cap").Attr<float>("temperature").Attr<float>("weight"));
#define TG_QK_ATTRS Attr<int32_t>("norm").Attr<float>("eps").Attr<double>("theta").Attr<int32_t>("rotary_dim").Attr<int32_t>("interleaved")

XLA_FFI_DEFINE_HANDLER_SYMBOL(TgQkNormRopeFwd, QkNormRopeFwd,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Arg<BF16>().Arg<BF16>().Arg<BF16>().Arg<S32>().Ret<BF16>().Ret<BF16>().TG_QK_ATTRS);
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgQkNormRopeBwd, QkNormRopeBwd,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Arg<BF16>().Arg<BF16>().Arg<BF16>().Arg<S32>().Arg<BF16>().Arg<BF16>()
                                  .Ret<BF16>().Ret<BF16>().Ret<BF16>().Ret<BF16>().Ret<U8>().TG_QK_ATTRS);
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgGatedLinearFwd, GatedLinearFwd,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Arg<BF16>().Arg<BF16>().Ret<BF16>().Ret<U8>().Ret<U8>().Ret<U8>().Ret<U32>()
                                  .Attr<int32_t>("act"));
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgGatedLinearBwd, GatedLinearBwd,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Arg<BF16>().Arg<BF16>().Arg<U8>().Arg<U8>().Arg<U8>().Arg<BF16>()
                                  .Ret<BF16>().Ret<BF16>().Ret<BF16>().Ret<U8>().Ret<U32>().Attr<int32_t>("act"));
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgDropout, Dropout,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Arg<U32>().Ret<BF16>().Attr<double>("p").Attr<int32_t>("site"));
XLA_FFI_DEFINE_HANDLER_SYMBOL(TgDropoutAdd, DropoutAdd,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<BF16>().Arg<BF16>().Arg<U32>().Ret<BF16>().Attr<double>("p").Attr<int32_t>("site"));
