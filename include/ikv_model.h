/*
 * ikv_model.h — C-ABI of the ops around the KV-cache path that a whole
 * Qwen3 step needs on the MI355X (gfx950): the projections (mul_mat), the
 * token-embedding gather, the elementwise ops of the FFN and residuals, the
 * greedy sampler, and the synthetic weight initialiser of the benchmarks.
 *
 * These replace the reference's CPU / CUDA ops of the same names
 * (src/backends/cpu_backend.cpp:259-332, 386-424, 636-703;
 * src/kernels/cuda/kernel_f32.cu:94-205, 515-630; src/sampler.cpp:42-65) so
 * that the scheduler keeps a whole Qwen3 graph on the HIP backend instead of
 * copying weights to the CPU every step (src/scheduler.cpp:67-69).
 * Conventions as in ikv.h: device pointers unless a name ends in _host,
 * stream as void*, 0 / negative errno / positive hipError_t, F32 row-major
 * with the reference Tensor layout (dims[0] innermost).
 */
#ifndef IKV_MODEL_H
#define IKV_MODEL_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---------------------------------------------------------------------
 * mul_mat: out[m][n] = sum_k x[m][k] * w[n][k]   (w: [n_out][k] rows, the
 * ggml [K, N] weight of CPUBackend::compute_mul_mat,
 * src/backends/cpu_backend.cpp:386-424; x: [m][k]; out: [m][n_out]).
 * m == 1 (decode) runs a hand-written streaming GEMV. 2 <= m <= 64 with
 * n_out % 16 == 0, k % 1024 == 0 and 16-byte aligned w and x runs a
 * hand-written F32 MFMA kernel. Other m > 1 with n_out % 64 == 0,
 * k % 64 == 0, k < 2^22 and 16-byte aligned w and x run the tiled F32 MFMA GEMM of
 * ikv_gemm_nt_f32 or, for products large enough, the same product on bf16
 * MFMA with every float split into three exact bf16 pieces (F32 inputs,
 * sums and results; no farther from a 64-bit product than the F32 MFMA
 * kernel: an output tile whose operands hold an infinity, a NaN or bits below
 * bf16's smallest, 2^-133, is formed on F32 MFMA), with K split over several
 * workgroups when the tiles would leave compute units idle: such a call needs
 * a split-K workspace of its device and stream, which the first one allocates
 * (8 MiB + 16 KiB, kept until exit; so make it outside HIP graph capture;
 * -ENOMEM after 64 device-stream pairs). A product that only the bf16 plan
 * splits does without where none can be had, its sums then in the unsplit
 * order. Any other shape runs one wavefront per output (m <= 65535, else
 * -ENOTSUP). Every path is deterministic: a fixed summation order per output
 * for given n_out, k and m.
 * residual: NULL, or [m][n_out] added to the result (out may equal
 * residual).
 * ------------------------------------------------------------------- */
int ikv_mul_mat_f32(const float *w, const float *x, float *out, int64_t n_out, int64_t k,
                    int64_t m, const float *residual, void *stream);

/* The hand-written MFMA GEMM of mul_mat for prompts (the same product,
 * CPUBackend::compute_mul_mat, src/backends/cpu_backend.cpp:386-424), for
 * any m >= 1: n_out % 64 == 0, k % 64 == 0, k < 2^22, 16-byte aligned w and x (else
 * -ENOTSUP / -EINVAL, nothing launched). Deterministic (a fixed summation
 * order per output); never splits K, so it allocates nothing. residual as
 * for mul_mat. */
int ikv_gemm_nt_f32(const float *w, const float *x, float *out, int64_t n_out, int64_t k,
                    int64_t m, const float *residual, void *stream);

/* Three projections of one input in one launch (the q, k, v projections of
 * a Qwen3 layer, src/models/Qwen3.cpp:56-58), m == 1:
 * out_i = w_i · x' for i = 0, 1, 2 with w_i [n_i][k], where x' = x, or, when
 * norm_w is not NULL, x' = ikv_rms_norm_f32(x, norm_w, eps) (the layer's
 * attn_norm folded in; k % 1024 == 0 and 16-byte aligned operands, else
 * -ENOTSUP). */
int ikv_gemv3_f32(const float *w0, const float *w1, const float *w2, const float *x, float *out0,
                  float *out1, float *out2, int64_t n0, int64_t n1, int64_t n2, int64_t k,
                  const float *norm_w, float eps, void *stream);

/* SwiGLU FFN input, m == 1: out[n] = (w_up[n] · x') * silu(w_gate[n] · x') —
 * mul_mat(ffn_gate), mul_mat(ffn_up), silu, mul of Qwen3Model::build_graph
 * (src/models/Qwen3.cpp:103-113) in one launch; silu(g) = g / (1 + exp(-g))
 * (src/backends/cpu_backend.cpp:660-673). x' as for ikv_gemv3_f32 (ffn_norm
 * folded in when norm_w is not NULL). */
int ikv_gemv_swiglu_f32(const float *w_gate, const float *w_up, const float *x, float *out,
                        int64_t n_out, int64_t k, const float *norm_w, float eps, void *stream);

/* ---------------------------------------------------------------------
 * get_rows: out[i][:] = table[ids[i]][:] for i < n_ids, rows of row_len
 * floats (CPUBackend::compute_get_rows, src/backends/cpu_backend.cpp:
 * 259-332; the token embedding). An id outside [0, n_rows) does not fault:
 * its output row is zeros and IKV_STATUS_TOKEN (include/ikv.h) is raised in
 * *status (device int, if non-NULL).
 * ------------------------------------------------------------------- */
int ikv_get_rows_f32(const float *table, const int32_t *ids, float *out, int64_t n_ids,
                     int64_t row_len, int64_t n_rows, int *status, void *stream);

/* Elementwise over n floats (src/backends/cpu_backend.cpp:636-703):
 * add: out = a + b; mul: out = a * b; silu: out = x / (1 + exp(-x)).
 * out may equal an input. */
int ikv_add_f32(const float *a, const float *b, float *out, int64_t n, void *stream);
int ikv_mul_f32(const float *a, const float *b, float *out, int64_t n, void *stream);
int ikv_silu_f32(const float *x, float *out, int64_t n, void *stream);
/* out = up * silu(gate): the SILU node and the MUL that consumes it
 * (src/models/Qwen3.cpp:107-112) in one pass, bitwise equal to the two ops.
 * out may equal gate or up. */
int ikv_silu_mul_f32(const float *gate, const float *up, float *out, int64_t n, void *stream);

/* ---------------------------------------------------------------------
 * Greedy sampling on the device (sample_greedy, src/sampler.cpp:42-65):
 * *token = the index of the largest of logits[0, n); ties go to the lowest
 * index. A NaN or +inf logit, or all logits -inf, writes *token = -1 (the
 * reference returns invalid_argument). n must be in [1, 2^31). token is a
 * device int32; token_mirror, if not NULL, receives the same value and may
 * be pinned host memory (hipHostMalloc), so that the host reads the token
 * once the stream has passed this launch, with no copy of its own.
 * ------------------------------------------------------------------- */
int ikv_argmax_f32(const float *logits, int64_t n, int32_t *token, int32_t *token_mirror,
                   void *stream);

/* The same sampler over up to 64 workgroups (no counterpart in the reference:
 * its sampler runs on the host). workspace: device memory of at least
 * ikv_argmax_workspace_bytes() bytes, 256-byte aligned, zero-filled once
 * before its first use; each call leaves it as it expects to find it, so it
 * is reused call after call. Calls sharing a workspace must not overlap
 * (one stream). Returns -EINVAL for a missing, small or misaligned
 * workspace. The result equals ikv_argmax_f32's. */
size_t ikv_argmax_workspace_bytes(void);
int ikv_argmax_ws_f32(const float *logits, int64_t n, int32_t *token, int32_t *token_mirror,
                      void *workspace, size_t workspace_bytes, void *stream);

/* ---------------------------------------------------------------------
 * Rules on each row of logits [n_rows][n_vocab] ahead of the samplers (the
 * reference has none, src/sampler.cpp:42-65): penalties for the tokens of the row's
 * history, biases, and a mask of the tokens that a grammar allows. For a token
 * that the row's history holds, and holds c times behind the prompt,
 *     x = x > 0 ? x / repetition : x * repetition
 *     x = x - frequency * c - presence   (where c > 0)
 * then x = x + bias, then x = -inf where the mask does not allow the token; in F32,
 * other tokens' bits unchanged. out may equal logits (and overlaps it in no other
 * way). Each part is left out where its array is NULL:
 *   history        [n_rows][history_stride] token ids: the prompt's, then the
 *                  generated ones; n_history [n_rows] of them (NULL: all), the
 *                  first n_prompt [n_rows] (NULL: none) from the prompt
 *   repetition, presence, frequency  [n_rows] (NULL: 1, 0, 0); computed with as
 *                  they stand, whatever they are
 *   bias_tokens, bias_values  [n_rows][bias_stride], n_bias [n_rows] of them (NULL:
 *                  all); of several for one token the last one counts
 *   masks          [n_masks][(n_vocab + 31) / 32] words, token t bit t % 32 of word
 *                  t / 32, 1: allowed; mask_of [n_rows] says which (NULL: mask 0),
 *                  a negative one: none
 * All arrays are device memory, read by the kernel, so a captured call serves
 * growing histories. An id outside [0, n_vocab) is skipped and raises
 * IKV_STATUS_TOKEN in *status; an n_history or n_bias outside its list raises
 * IKV_STATUS_POSITION and is taken for 0, a mask_of past the last mask raises it and
 * allows no token. A row that allows none is all -inf, which the samplers answer
 * with token -1.
 * -EINVAL: no rules, a negative stride, values or masks missing; -EOVERFLOW:
 * n_vocab or a stride past 2^30, n_rows past 2^21, n_rows * ceil(n_vocab / 4096)
 * past 2^23 - 1.
 * ------------------------------------------------------------------- */
typedef struct ikv_logit_rules {
    const int32_t *history;
    int64_t history_stride;
    const int32_t *n_history;
    const int32_t *n_prompt;
    const float *repetition;
    const float *presence;
    const float *frequency;
    const int32_t *bias_tokens;
    const float *bias_values;
    int64_t bias_stride;
    const int32_t *n_bias;
    const uint32_t *masks;
    int64_t n_masks;
    const int32_t *mask_of;
} ikv_logit_rules;

int ikv_adjust_logits_f32(const float *logits, float *out, const ikv_logit_rules *rules,
                          int64_t n_rows, int64_t n_vocab, int32_t *status, void *stream);

/* ---------------------------------------------------------------------
 * Sampling of each row of logits [n_rows][n_vocab] from a given uniform number
 * u[row] in [0, 1) (the reference samples greedily, src/sampler.cpp:42-65).
 * With y_i = (x_i - max) / temperature and w_i = exp(y_i), tokens in the order
 * of descending x_i, ties by index:
 *   top_k   keeps the first top_k tokens (<= 0 or > n_vocab: all);
 *   top_p   of them the shortest start whose mass is at least top_p times
 *           theirs (>= 1: all; one token at least);
 *   min_p   of it the tokens with y_i >= ln(min_p) (<= 0: all; one at least).
 * token[row] is the first token of the order whose running mass exceeds u times
 * the kept mass; logprob[row], if logprob is not NULL, is the logarithm of its
 * share of the kept mass. temperature <= 0 is greedy: the first of the largest
 * logits, logprob 0. -inf logits are never drawn. A NaN or +inf logit, all
 * logits -inf, a NaN parameter or a temperature of +inf give token -1 and a
 * NaN logprob. u is brought into [0, 1 - 2^-24]. temperature, top_k, top_p,
 * min_p [n_rows] may each be NULL: 1, all, 1, 0. Parameters are device memory.
 * The masses are summed exactly in integers of 2^-44 of the heaviest token's
 * (n_vocab = 151936; 62 bits less those of n_vocab, 51 at most), so equal calls
 * give equal results. Each weight is rounded to such an integer: a token below half
 * of one weighs nothing and is never drawn, and where u is next to 1 and the tail is
 * long (1 - 2^-24 and thousands of tokens of 2^-36) another token of the tail than
 * by exact masses may be.
 * workspace: device memory of ikv_sample_workspace_bytes(n_rows, n_vocab)
 * bytes, 16-byte aligned (else -EINVAL); nothing is expected in it or left in
 * it, and it is enough for fewer rows. Launches that share it must be ordered.
 * -EOVERFLOW: n_vocab past 2^30 or n_rows past 2^21.
 * ------------------------------------------------------------------- */
size_t ikv_sample_workspace_bytes(int64_t n_rows, int64_t n_vocab);
int ikv_sample_f32(const float *logits, const float *u, const float *temperature,
                   const int32_t *top_k, const float *top_p, const float *min_p, int64_t n_rows,
                   int64_t n_vocab, int32_t *token, float *logprob, void *workspace,
                   size_t workspace_bytes, void *stream);

/* ---------------------------------------------------------------------
 * Host helper: the benchmarks' synthetic weights. out_host[i] =
 * std * N(0,1) sample number (offset + i) of the stream `seed`:
 * splitmix64 outputs 2j+1 and 2j+2 of the seed give the uniforms of
 * Box-Muller pair j (u1 = (z1 >> 11 + 1) 2^-53, u2 = (z2 >> 11) 2^-53,
 * r = sqrt(-2 ln u1), normals r cos(2 pi u2), r sin(2 pi u2)), times std,
 * computed in double and rounded once to float. Any split of [0, n) over calls gives the
 * same values. Uses up to `threads` host threads (<= 1: the calling thread).
 * ------------------------------------------------------------------- */
int ikv_synth_normal_f32(uint64_t seed, uint64_t offset, size_t n, double std, float *out_host,
                         int threads);

#ifdef __cplusplus
}
#endif

#endif /* IKV_MODEL_H */
