/*
 * stew_step.h -- C ABI of the layer kernels around the NF4 projections in the packed-token
 * QLoRA step (same library and conventions as stew_nf4.h: device pointers, sizes in elements,
 * `void* stream` = cudaStream_t, int status, no allocation, no host synchronisation).
 *
 * They stand in for the reference's Triton kernels of the same Qwen2 layer:
 *   nf4b_rmsnorm_fwd (delta == NULL) <- solution/rmsnorm.py:19-34  _rms_fwd
 *   nf4b_rmsnorm_fwd (delta given)   <- solution/rmsnorm.py:152-168 _add_rms_fwd
 *   nf4b_rmsnorm_bwd (dsum NULL/set) <- solution/rmsnorm.py:36-50 _rms_bwd, :171-190 _add_rms_bwd
 *   nf4b_rope_qk                     <- solution/rope.py:24-52 rope_kernel (forward, and INVERSE
 *                                       for the backward) applied to q and k in one launch
 *   nf4b_swiglu_fwd / _bwd           <- solution/swiglu.py:15-40
 *   nf4b_ce_fwd / _bwd               <- solution/head_loss.py (loss, then softmax - onehot)
 *   nf4b_attn_fwd / _bwd             <- the per-row SDPA of solution/unpad.py:177-219
 * Activations are fp16, row-major (attention: fp16 or bf16, strided).
 */
#ifndef STEW_STEP_H
#define STEW_STEP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* y[r] = fp16(w * fp16(s[r] * rstd[r])), rstd[r] = 1/sqrt(mean(s[r]^2) + eps), where
 * s = x (delta == NULL) or s = fp16(x + delta), then also written to `sum` (the residual
 * stream).  x, delta, sum, y: fp16 [rows, hidden]; w: fp32 [hidden]; rstd: fp32 [rows].
 * hidden must be a multiple of 256 and at most 4096.  */
int nf4b_rmsnorm_fwd(const void* x, const void* delta, const float* w, float eps, void* sum,
                     void* y, float* rstd, int64_t rows, int64_t hidden, void* stream);

/* dx = rstd * (w*dy - xn * mean(w*dy*xn)) (+ dsum), xn = x * rstd: the input gradient of
 * nf4b_rmsnorm_fwd (x = the normalised input s); with the fused add, dsum is the gradient
 * arriving at `sum`, and dx is the gradient of both x and delta.  */
int nf4b_rmsnorm_bwd(const void* dy, const void* x, const float* w, const float* rstd,
                     const void* dsum, void* dx, int64_t rows, int64_t hidden, void* stream);

/* Rotary embedding (rotate-half convention, fp32 math) on q [tokens, q_heads, head_dim] and
 * k [tokens, k_heads, head_dim] with cos/sin fp32 [tokens, head_dim]:
 *   out[i] = x[i] cos[i] - x[i+d] sin[i],   out[i+d] = x[i+d] cos[i+d] + x[i] sin[i+d],
 * d = head_dim/2; inverse != 0 applies the transposed rotation (the backward).
 * head_dim must be a multiple of 16; either tensor may be skipped with 0 heads.  */
int nf4b_rope_qk(const void* q, const void* k, const float* cos_t, const float* sin_t, void* q_out,
                 void* k_out, int64_t tokens, int32_t q_heads, int32_t k_heads, int32_t head_dim,
                 int32_t inverse, void* stream);

/* m = fp16(gate * sigmoid(gate) * up), fp32 inside (the reference's SwiGLU kernel,
 * solution/swiglu.py:16-23), n elements (a multiple of 8).  */
int nf4b_swiglu_fwd(const void* gate, const void* up, void* out, int64_t n, void* stream);

/* dup = fp16(dout * gate * sig), dgate = fp16(dout * up * sig * (1 + gate * (1 - sig))),
 * sig = sigmoid(gate), fp32 inside (solution/swiglu.py:26-37).  */
int nf4b_swiglu_bwd(const void* dout, const void* gate, const void* up, void* dgate, void* dup,
                    int64_t n, void* stream);

/* Next-token cross-entropy of the LM head over fp16 logits [rows, vocab] (vocab a multiple of
 * 8, rows 16-byte aligned) with int64 labels [rows] -- the reference's fused head loss
 * (solution/head_loss.py: per-row loss, then the gradient softmax - onehot in place):
 *   nf4b_ce_fwd: loss[r] = logsumexp(logits[r]) - logits[r, labels[r]] (fp32; 0 where the
 *                label is outside [0, vocab), e.g. -100), lse[r] = logsumexp(logits[r]);
 *   nf4b_ce_bwd: logits[r, j] <- fp16(g * (exp(logits[r, j] - lse[r]) - [j == labels[r]])) in
 *                place, g = *gscale (device fp32), zero rows for ignored labels.  */
int nf4b_ce_fwd(const void* logits, const int64_t* labels, float* loss, float* lse, int64_t rows,
                int64_t vocab, void* stream);
int nf4b_ce_bwd(void* logits, const int64_t* labels, const float* lse, const float* gscale,
                int64_t rows, int64_t vocab, void* stream);

/* Attention over packed token rows.  q [tokens, heads, head_dim] and k, v [tokens, kv_heads,
 * head_dim] (fp16 or bf16) hold `rows` sequences one after the other: sequence b is tokens
 * [cu[b], cu[b+1]) (device int32 [rows + 1], cu[0] = 0, ascending, cu[rows] <= tokens; an empty
 * sequence is allowed).  Inside a sequence token i sees the tokens j with
 * i - left <= j <= i + right; a negative bound is no bound ((-1, 0) is causal attention).  Query
 * head h reads key/value head h / (heads / kv_heads).  With s_ij = scale q_i.k_j:
 *   p_ij = exp(s_ij) / sum_j exp(s_ij),   o_i = sum_j p_ij v_j,   lse_i = log sum_j exp(s_ij)
 * head_dim: a multiple of 8, at most 128.  The last dimension is contiguous; token and head
 * strides (in elements) are multiples of 8 and at least head_dim, pointers are 16-byte aligned.
 * cu is read on the device: values outside [0, tokens] are clamped there.  */
typedef struct nf4b_attn {
  const void* q;
  const void* k;
  const void* v;
  const int32_t* cu;
  int64_t tokens;
  int64_t q_stride, q_head_stride;
  int64_t k_stride, k_head_stride;
  int64_t v_stride, v_head_stride;
  int32_t rows, heads, kv_heads, head_dim;
  int32_t dtype;         /* NF4B_F16 or NF4B_BF16 */
  int32_t left, right;
  float scale;           /* > 0, below 2^127 */
} nf4b_attn;

/* out [tokens, heads, head_dim] contiguous, of q's type; lse fp32 [heads, tokens] (natural log);
 * rest (NULL: not wanted): what out's rounding left of the output, again in q's type, for the
 * backward's do.o.  Tokens at and behind cu[rows] get zeros (lse -inf).  */
int nf4b_attn_fwd(const nf4b_attn* a, void* out, void* rest, float* lse, void* stream);

/* Gradients from dout, out, rest (contiguous, as nf4b_attn_fwd wrote them; rest may be NULL: do.o is
 * then taken from the rounded output, whose error all of a row's ds share) and lse:
 *   dv_j = sum_i p_ij do_i,   ds_ij = p_ij (do_i.v_j - do_i.o_i),
 *   dq_i = scale sum_j ds_ij k_j,   dk_j = scale sum_i ds_ij q_i,
 * k's and v's summed over the query heads that share them.  The probabilities are recomputed
 * from lse; every sum is taken in a fixed order (the same bits on every run).  dout, dq
 * [tokens, heads, head_dim] and dk, dv [tokens, kv_heads, head_dim] are contiguous, of q's type;
 * tokens at and behind cu[rows] get zeros.  work: nf4b_attn_bwd_work_bytes(a) bytes of device
 * scratch, 16-byte aligned, of any content; -1 for a call that would be refused.  */
int64_t nf4b_attn_bwd_work_bytes(const nf4b_attn* a);
int nf4b_attn_bwd(const nf4b_attn* a, const void* out, const void* rest, const float* lse, const void* dout,
                  void* dq, void* dk, void* dv, void* work, int64_t work_bytes, void* stream);

/* Reads (and with reset != 0 clears) the device-side flag the attention kernels set when a pipeline
 * wait ran out of time (the kernel then ends early instead of hanging, with NaN in the output rows
 * that it did not finish).  0 = no timeout since the last reset.  Synchronous.  */
int nf4b_attn_error_flag(int* value, int reset);

/* One gradient of a list: src and dst hold `numel` contiguous values of `dtype` (NF4B_F16,
 * NF4B_BF16 or NF4B_F32; the element's own alignment is enough).  dst == src scales in place;
 * dst == NULL reads it for the norm only.  numel 0 is allowed (pointers may then be NULL).  */
typedef struct nf4b_grad {
  const void* src;
  void* dst;
  int64_t numel;
  int32_t dtype;
  int32_t reserved;
} nf4b_grad;

/* Global 2-norm of a list of gradients and clipping to max_norm (>= 0, or infinity):
 *   *norm = || src / *divisor ||_2 over all n gradients (device fp32; divisor: device fp32, NULL = 1)
 *   dst   = src * (1 / *divisor) * min(1, max_norm / (*norm + 1e-6))
 * The squares are summed in 64 bits in a fixed order (16-bit values' exact squares in pairs, rounded to
 * fp32, before that).  A norm that is infinite gives zeros (NaN
 * where src is infinite), a NaN norm gives NaN everywhere.  An in-place list under the limit with
 * no divisor is not written.  No dst may overlap another gradient's src or dst.  `grads` is a host
 * array, read before the call returns.  work: nf4b_clip_grads_work_bytes(n) bytes of device
 * scratch, 8-byte aligned, of any content.  */
int64_t nf4b_clip_grads_work_bytes(int32_t n);
int nf4b_clip_grads(const nf4b_grad* grads, int32_t n, float max_norm, const float* divisor, float* norm,
                    void* work, int64_t work_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* STEW_STEP_H */
