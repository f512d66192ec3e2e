/* C ABI of attention over packed sequences and over a shared prefix (libechosparse_hip.so, gfx950).
 *
 * The conventions of echosparse_hip.h: caller-owned device pointers, the HIP stream to enqueue on, an es_status in
 * return and a message in es_last_error_string(); nothing allocates or synchronises, no state is kept between calls.
 * Entry points that take token tensors (const void* / void*) read and write bf16; each has a twin with the suffix _f16
 * and the same arguments for fp16. The reference has no counterpart of these operators.
 *
 * Layouts (row-major; token tensors and the workspace aligned to 16 bytes):
 *   q, out, dout, dq   (Tq, H, D)      D = 64 or 128, H a multiple of Hk: query head h reads kv head h / (H / Hk)
 *   k, v, dk, dv       (Tk, Hk, D)
 *   lse                (Tq, H) float32, natural logarithm, -inf for rows that see no key
 *   cu_q, cu_k         (B + 1) int32: sequence b holds rows cu[b] .. cu[b + 1] - 1, cu[0] taken as 0; values are clamped to
 *                      the tensor and must not decrease. NULL: B sequences of Tq / B (Tk / B) rows each.
 *   bias               (num_buckets, H) float32, NULL: none; buckets (2 * R + 1) int32 in 0 .. num_buckets - 1 (clamped)
 * Query i of a sequence with nq queries and nk keys has position i + nk - nq. It sees every key, with causal != 0 those up
 * to its position; its score against key j is scale * q.k + bias[buckets[clamp(j - position, -R, R) + R]][h].
 * Rows that see no key get out = 0 and lse = -inf and give no gradient. Rows behind the last sequence are such rows;
 * key rows behind it get zero gradients, and their values are never used.
 * Scores are float32 and must stay below 2^22 in magnitude. (H / Hk) * (2 * R + 1) is at most ES_PACKED_BIAS_ROWS. Bias
 * values are finite or -inf (which masks); finite ones beyond +-ES_PACKED_BIAS_MAX count as that, and their dbias is 0. Calls
 * of about 2^24 / Hk sequences and more are refused.
 */
#pragma once
#include "echosparse_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define ES_PACKED_BIAS_ROWS 784
#define ES_PACKED_BIAS_MAX 131072.0f

/* Forward. workspace: es_packed_fwd_workspace bytes (0: none needed; NULL / 0 is then accepted), for batches of few query
 * rows against many keys, whose keys are cut into ranges that run side by side and are merged in a fixed order. (Without cu_k
 * the lengths are known, and a call that cuts nothing takes NULL / 0 where one of the same sizes with cu_k does not.) */
size_t es_packed_fwd_workspace(int B, int Tq, int Tk, int H, int Hk, int D);
int es_packed_fwd(const void* q, const void* k, const void* v, const int* cu_q, const int* cu_k, const float* bias,
                  const int* buckets, int num_buckets, int R, void* out, float* lse, void* workspace,
                  size_t workspace_bytes, int B, int Tq, int Tk, int H, int Hk, int D, int causal, float scale,
                  hipStream_t stream);
int es_packed_fwd_f16(const void* q, const void* k, const void* v, const int* cu_q, const int* cu_k, const float* bias,
                      const int* buckets, int num_buckets, int R, void* out, float* lse, void* workspace,
                      size_t workspace_bytes, int B, int Tq, int Tk, int H, int Hk, int D, int causal, float scale,
                      hipStream_t stream);

/* Backward of the same call from its out and lse; dbias (num_buckets, H) float32 with bias, NULL without. No atomics on
 * global memory: the same inputs give the same bits. workspace: es_packed_bwd_workspace bytes. */
size_t es_packed_bwd_workspace(int B, int Tq, int Tk, int H, int Hk, int D, int R, int with_bias, int causal);
int es_packed_bwd(const void* q, const void* k, const void* v, const void* dout, const void* out, const float* lse,
                  const int* cu_q, const int* cu_k, const float* bias, const int* buckets, int num_buckets, int R, void* dq,
                  void* dk, void* dv, float* dbias, void* workspace, size_t workspace_bytes, int B, int Tq, int Tk, int H,
                  int Hk, int D, int causal, float scale, hipStream_t stream);
int es_packed_bwd_f16(const void* q, const void* k, const void* v, const void* dout, const void* out, const float* lse,
                      const int* cu_q, const int* cu_k, const float* bias, const int* buckets, int num_buckets, int R,
                      void* dq, void* dk, void* dv, float* dbias, void* workspace, size_t workspace_bytes, int B, int Tq,
                      int Tk, int H, int Hk, int D, int causal, float scale, hipStream_t stream);

/* n query rows of each of B sequences, q / out (B, n, H, D), lse (B, n, H): every row sees all P rows of k_prefix /
 * v_prefix (P, Hk, D); row i of sequence b also sees rows 0 .. lens[b] - n + i of its own cache k[b] / v[b] (B, S, Hk, D),
 * lens[b] (clamped to 0 .. S) counting the n rows' own keys. One softmax over both. Cache rows from lens[b] on are not used.
 * workspace: es_shared_prefix_workspace bytes. */
size_t es_shared_prefix_workspace(int B, int n, int P, int S, int H, int Hk, int D);
int es_shared_prefix_fwd(const void* q, const void* k_prefix, const void* v_prefix, const void* k, const void* v,
                         const int* lens, void* out, float* lse, void* workspace, size_t workspace_bytes, int B, int n,
                         int P, int S, int H, int Hk, int D, float scale, hipStream_t stream);
int es_shared_prefix_fwd_f16(const void* q, const void* k_prefix, const void* v_prefix, const void* k, const void* v,
                             const int* lens, void* out, float* lse, void* workspace, size_t workspace_bytes, int B, int n,
                             int P, int S, int H, int Hk, int D, float scale, hipStream_t stream);

#ifdef __cplusplus
}
#endif
