/* C ABI of norms with position rotation, of paged caches in 16 or 4 bits, and of attention over them (libechosparse_hip.so,
 * gfx950).
 *
 * The conventions of packed_hip.h: caller-owned device pointers, the HIP stream to enqueue on, an es_status in return and a
 * message in es_last_error_string(); nothing allocates or synchronises, no state is kept between calls. Entry points that take
 * token tensors (const void* / void*) read and write bf16; each has a twin with the suffix _f16 and the same arguments for fp16.
 * The reference has no counterpart of these operators.
 *
 * Layouts (row-major; tensors aligned to 16 bytes, strides multiples of 8 values):
 *   q (T, H, D), k, v (T, Hk, D)   D = 64 or 128, H a multiple of Hk; *_stride: values between two tokens' rows (heads are D apart)
 *   q_weight, k_weight (D)          of the norm; the token type, or float32 with weight_f32 != 0; both NULL: no norm
 *   table (P, R / 2, 2) float32     cosine and sine of each position and pair, R a multiple of 16 up to D; NULL (R = 0): no
 *                                   rotation. halves == 0: pair i is channels 2 i and 2 i + 1, otherwise i and i + R / 2.
 *                                   Positions past the last row take that row's angles, negative ones the first row's.
 *   pages (B, max_pages) int32      page numbers of a sequence; lens (B) int32: its tokens with the new ones (below 0: 0)
 *   cu (B + 1) int32                running counts of new tokens as in packed_hip.h; NULL: T / B each
 *   cache, 16 bits                  k_pages, v_pages: (num_pages, Hk, page_size, D) with the strides page_stride, head_stride and
 *                                   row_stride (values) that both have
 *   cache, 4 bits                   k_codes, v_codes (num_pages, Hk, page_size, D / 2), k_scales, v_scales (num_pages, Hk,
 *                                   page_size, D / 32), contiguous: 32 channels share the power of two s = 2^(scale - 127), the
 *                                   smallest with max |x| <= 7 s (held to 2^-120 .. 2^120, fp16 2^-13 .. 2^13); bit 3 of a code
 *                                   is the sign, bits 0 to 2 number the magnitudes 0 0.5 1 1.5 2 3 4 6 times s. The nearest, ties
 *                                   to the even code. Channel 2 i is in the low half of byte i.
 * page_size is a power of two from 16 to 4096. Token i of n new ones of sequence b has position p = lens[b] - n + i and is held in
 * row p % page_size of page pages[b][p / page_size]. Tokens of negative positions, past the table of pages, or whose page number
 * is outside 0 .. num_pages - 1 are neither written nor read.
 */
#pragma once
#include "echosparse_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* q_out (T, H, D), k_out (T, Hk, D), contiguous: x / sqrt(mean x^2 + eps) * weight of each head's row, rotated. positions (T)
 * int32; NULL: row t has position t % L. q or k may be NULL (with H or Hk 0 and their weight NULL). */
int es_norm_rotate(const void* q, const void* k, const void* q_weight, const void* k_weight, const float* table,
                   const int* positions, void* q_out, void* k_out, int T, int L, int H, int Hk, int D, int R, int P, int halves,
                   int weight_f32, double eps, long long q_stride, long long k_stride, hipStream_t stream);
int es_norm_rotate_f16(const void* q, const void* k, const void* q_weight, const void* k_weight, const float* table,
                       const int* positions, void* q_out, void* k_out, int T, int L, int H, int Hk, int D, int R, int P,
                       int halves, int weight_f32, double eps, long long q_stride, long long k_stride, hipStream_t stream);

/* Its backward, from the same inputs and the gradients of both outputs (contiguous): dq (T, H, D), dk (T, Hk, D) contiguous,
 * dq_weight and dk_weight (D) in the weights' type. Sums have a fixed order. workspace: es_norm_rotate_workspace bytes (0 without
 * a norm; NULL is then accepted). */
size_t es_norm_rotate_workspace(int T, int H, int Hk, int D);
int es_norm_rotate_bwd(const void* q, const void* k, const void* dq_out, const void* dk_out, const void* q_weight,
                       const void* k_weight, const float* table, const int* positions, void* dq, void* dk, void* dq_weight,
                       void* dk_weight, void* workspace, size_t workspace_bytes, int T, int L, int H, int Hk, int D, int R, int P,
                       int halves, int weight_f32, double eps, long long q_stride, long long k_stride, hipStream_t stream);
int es_norm_rotate_bwd_f16(const void* q, const void* k, const void* dq_out, const void* dk_out, const void* q_weight,
                           const void* k_weight, const float* table, const int* positions, void* dq, void* dk, void* dq_weight,
                           void* dk_weight, void* workspace, size_t workspace_bytes, int T, int L, int H, int Hk, int D, int R,
                           int P, int halves, int weight_f32, double eps, long long q_stride, long long k_stride,
                           hipStream_t stream);

/* New tokens into the cache: k normed (k_weight) and rotated, v as it is; with q (T, H, D) also q_out (T, H, D) contiguous, q
 * normed and rotated at the same positions (q NULL, H 0: none). q_out rows of tokens without a position (behind the last
 * sequence, or negative) are zeros. What two tokens of a call are held in at once is not defined. */
int es_append_paged(const void* q, const void* k, const void* v, const void* q_weight, const void* k_weight, const float* table,
                    const int* pages, const int* lens, const int* cu, void* q_out, void* k_pages, void* v_pages, int B, int T,
                    int max_pages, int num_pages, int page_size, int H, int Hk, int D, int R, int P, int halves, int weight_f32,
                    double eps, long long q_stride, long long k_stride, long long v_stride, long long page_stride,
                    long long head_stride, long long row_stride, hipStream_t stream);
int es_append_paged_f16(const void* q, const void* k, const void* v, const void* q_weight, const void* k_weight,
                        const float* table, const int* pages, const int* lens, const int* cu, void* q_out, void* k_pages,
                        void* v_pages, int B, int T, int max_pages, int num_pages, int page_size, int H, int Hk, int D, int R,
                        int P, int halves, int weight_f32, double eps, long long q_stride, long long k_stride, long long v_stride,
                        long long page_stride, long long head_stride, long long row_stride, hipStream_t stream);
/* The same into a cache of 4 bits: k is normed and rotated in 64 bits, rounded to float32 and held as the nearest values, so
 * that a key's code follows from the formula alone. Values must be finite. */
int es_append_paged4(const void* q, const void* k, const void* v, const void* q_weight, const void* k_weight, const float* table,
                     const int* pages, const int* lens, const int* cu, void* q_out, uint8_t* k_codes, uint8_t* k_scales,
                     uint8_t* v_codes, uint8_t* v_scales, int B, int T, int max_pages, int num_pages, int page_size, int H,
                     int Hk, int D, int R, int P, int halves, int weight_f32, double eps, long long q_stride, long long k_stride,
                     long long v_stride, hipStream_t stream);
int es_append_paged4_f16(const void* q, const void* k, const void* v, const void* q_weight, const void* k_weight,
                         const float* table, const int* pages, const int* lens, const int* cu, void* q_out, uint8_t* k_codes,
                         uint8_t* k_scales, uint8_t* v_codes, uint8_t* v_scales, int B, int T, int max_pages, int num_pages,
                         int page_size, int H, int Hk, int D, int R, int P, int halves, int weight_f32, double eps,
                         long long q_stride, long long k_stride, long long v_stride, hipStream_t stream);

/* k, v (T, Hk, D) contiguous: what the cache holds of the tokens that cu and lens name (the last cu[b + 1] - cu[b] of sequence
 * b); zeros for tokens that it does not hold. */
int es_paged_rows(const void* k_pages, const void* v_pages, const int* pages, const int* lens, const int* cu, void* k, void* v,
                  int B, int T, int max_pages, int num_pages, int page_size, int Hk, int D, long long page_stride,
                  long long head_stride, long long row_stride, hipStream_t stream);
int es_paged_rows_f16(const void* k_pages, const void* v_pages, const int* pages, const int* lens, const int* cu, void* k,
                      void* v, int B, int T, int max_pages, int num_pages, int page_size, int Hk, int D, long long page_stride,
                      long long head_stride, long long row_stride, hipStream_t stream);
int es_paged_rows4(const uint8_t* k_codes, const uint8_t* k_scales, const uint8_t* v_codes, const uint8_t* v_scales,
                   const int* pages, const int* lens, const int* cu, void* k, void* v, int B, int T, int max_pages,
                   int num_pages, int page_size, int Hk, int D, hipStream_t stream);
int es_paged_rows4_f16(const uint8_t* k_codes, const uint8_t* k_scales, const uint8_t* v_codes, const uint8_t* v_scales,
                       const int* pages, const int* lens, const int* cu, void* k, void* v, int B, int T, int max_pages,
                       int num_pages, int page_size, int Hk, int D, hipStream_t stream);

/* Attention of new tokens q (Tq, H, D) over the cache: token i of n new ones of sequence b sees all its lens[b] keys, with causal
 * != 0 those up to its own position; out (Tq, H, D), lse (Tq, H) float32 as in packed_hip.h. Keys of pages that the cache does not
 * have are left out. Rows that see no key, and rows behind the last sequence, get out = 0 and lse = -inf. Values of the keys in
 * use must be finite (of a cache of 4 bits within the token type), scores below 2^22 in magnitude.
 * workspace: es_paged_workspace bytes (0: none needed; NULL / 0 is then accepted); bits: 16 or 4. */
size_t es_paged_workspace(int B, int Tq, int max_pages, int page_size, int H, int Hk, int D, int bits);
int es_paged_fwd(const void* q, const void* k_pages, const void* v_pages, const int* pages, const int* lens, const int* cu,
                 void* out, float* lse, void* workspace, size_t workspace_bytes, int B, int Tq, int max_pages, int num_pages,
                 int page_size, int H, int Hk, int D, int causal, float scale, long long page_stride, long long head_stride,
                 long long row_stride, hipStream_t stream);
int es_paged_fwd_f16(const void* q, const void* k_pages, const void* v_pages, const int* pages, const int* lens, const int* cu,
                     void* out, float* lse, void* workspace, size_t workspace_bytes, int B, int Tq, int max_pages,
                     int num_pages, int page_size, int H, int Hk, int D, int causal, float scale, long long page_stride,
                     long long head_stride, long long row_stride, hipStream_t stream);
int es_paged4_fwd(const void* q, const uint8_t* k_codes, const uint8_t* k_scales, const uint8_t* v_codes,
                  const uint8_t* v_scales, const int* pages, const int* lens, const int* cu, void* out, float* lse,
                  void* workspace, size_t workspace_bytes, int B, int Tq, int max_pages, int num_pages, int page_size, int H,
                  int Hk, int D, int causal, float scale, hipStream_t stream);
int es_paged4_fwd_f16(const void* q, const uint8_t* k_codes, const uint8_t* k_scales, const uint8_t* v_codes,
                      const uint8_t* v_scales, const int* pages, const int* lens, const int* cu, void* out, float* lse,
                      void* workspace, size_t workspace_bytes, int B, int Tq, int max_pages, int num_pages, int page_size,
                      int H, int Hk, int D, int causal, float scale, hipStream_t stream);

#ifdef __cplusplus
}
#endif
