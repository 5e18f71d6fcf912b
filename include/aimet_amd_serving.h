/*
 * aimet_amd_serving.h -- C ABI of libaimet_amd.so, second part: running what calibrated encodings describe.  Linear layers
 * on packed 4-bit weights, a key/value cache held in 8 bits, and the attention that reads it.
 *
 * The conventions are those of aimet_amd.h: device pointers, work enqueued on `stream` without synchronising, ahq_status
 * codes with ahq_last_error(), no allocation inside the library.
 */
#ifndef AIMET_AMD_SERVING_H
#define AIMET_AMD_SERVING_H

#include "aimet_amd.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---------------------------------------------------------------- packed 4-bit linear layers -----------------------
 * Inference on the codes a calibrated 4-bit weight quantizer describes (AT/nn/fake_quant.py's QuantizedLinear with the
 * weight's encoding applied on the fly instead of a quantize-dequantized copy; no kernel of the reference does this).
 *
 *   y[m][j] = sum_g scale[j][g] * ( sum_{k in group g} x[m][k] * (code[j][k] - qmin + zero[j][g] + zero_const) ) + bias[j]
 *
 * ahq_int4_pack lays out the codes of an [n][k] weight (row-major bytes, each in [qmin, qmin + 15]; only the low four
 * bits of code - qmin are kept) as ahq_int4_linear reads them, ahq_int4_packed_bytes(n, k) bytes (0: bad shape; n is
 * at most 2^28, k at most 2^20).
 * ahq_int4_linear: x is [m][k] of `dtype` with rows ldx elements apart, y [m][n] with rows ldy apart, both dense along
 * the row; m is at most 2^20, and the result at most 2^22 blocks of 64 x 256 (float32 32 x 128) values.  bias: n values of
 * `dtype`, or NULL.  Products and sums are float32 with exact factors; y is rounded once.
 */
typedef struct {
    int64_t n, k;        /* output and input channels */
    int64_t group;       /* columns that share a scale: a multiple of 32 that divides k, or k */
    const void* packed;  /* ahq_int4_pack's output; like scale and zero 16-byte aligned */
    const float* scale;  /* [ceil(n / 16)][k / group][16]: channel 16 i + j at [i][.][j]; padding: any finite value */
    const int8_t* zero;  /* same shape, or NULL for zero_const alone */
    float zero_const;
} ahq_int4_weight;

size_t ahq_int4_packed_bytes(int64_t n, int64_t k);
int ahq_int4_pack(const int8_t* codes, int64_t n, int64_t k, int32_t qmin, void* packed, void* stream);
int ahq_int4_linear(const ahq_int4_weight* w, int32_t dtype, const void* x, int64_t m, int64_t ldx, const void* bias,
                    void* y, int64_t ldy, void* stream);

/* ---------------------------------------------------------------- 8-bit key/value cache ----------------------------
 * A cache of keys and values as codes in [-127, 127] with the largest magnitude (`amax`, float) of every block of
 * `block` tokens (16, 32 or 64) of a sequence and head: a code stands for code * amax / 127 (the symmetric grid of
 * the 8-bit quantizers without its lowest code).  head_dim: 64, 128 or 256; capacity: tokens per sequence, a
 * multiple of 64.  All arrays are the caller's; a new cache has code bytes 128 (the code 0; a byte holds code + 128) and
 * maxima 0.
 *   k_codes [batch][heads][capacity / 64][4][head_dim / 64][4][16][16]: [.][s][u][c][4 g + r][e] is token 16 g + 4 s + r of
 *           the tile of 64, channel 64 u + 16 c + e
 *   v_codes [batch][heads][capacity / 64][head_dim / 16][4][16][16]: [.][u][c][i][e] is token 16 c + e, channel 16 u + i
 *           (both 16-byte aligned)
 *   k_amax, v_amax [batch][heads][capacity / block]
 */
typedef struct {
    int32_t batch, heads, capacity, head_dim, block;
    uint8_t *k_codes, *v_codes;
    float *k_amax, *v_amax;
} ahq_kv_cache;

/* Keys and values to store: [batch][heads][tokens][head_dim] of `dtype`, dense along head_dim, with strides in elements
 * for keys [0] and values [1].  Token t of sequence b goes to position start[b] + t, for t < counts[b]; start / counts
 * are device arrays of `batch` entries, or NULL for start_all / count_all everywhere.  Positions outside [0, capacity)
 * are not written; counts are limited to [0, tokens]. */
typedef struct {
    int32_t dtype, tokens;
    const void *k, *v;
    int64_t stride_batch[2], stride_head[2], stride_token[2];
    const int32_t *start, *counts;
    int32_t start_all, count_all;
} ahq_kv_tokens;

/* Queries [batch][query_heads][queries][head_dim] and their answers, strides in elements, dense along head_dim.  Query
 * head j reads cache head j / (query_heads / heads).  Sequence b holds lengths[b] tokens (limited to [0, capacity]) and
 * its first counts[b] queries are the last ones of them: query t stands at position lengths[b] - counts[b] + t and sees
 * the tokens up to its own.  queries * query_heads / heads is below 2^20.  Queries behind counts[b], and those that see
 * nothing, are answered with zeros.  scale multiplies the scores. */
typedef struct {
    int32_t dtype, query_heads, queries;
    const void* q;
    void* out;
    int64_t q_stride_batch, q_stride_head, q_stride_query, out_stride_batch, out_stride_head, out_stride_query;
    const int32_t *lengths, *counts;
    int32_t length_all, count_all;
    float scale;
} ahq_kv_queries;

/* Stores tokens: a block's amax is that of the new finite magnitudes, and no less than what it was where the first new token
 * is not the block's first (tokens at and behind `start`, of an earlier call, have their part in it although they are
 * overwritten or discarded), codes are rint(127 x / amax) half to even (exact; infinities saturate, NaN and everything in a
 * block of zeros is 0), and the codes of a block's tokens in front of `start` become rint(code * old amax / new amax) where
 * it grew.  No code behind the last new token is written; such tokens count as discarded, and the block's amax need not be
 * theirs.  Two calls for the same block have to be ordered. */
int ahq_kv_append(const ahq_kv_cache* cache, const ahq_kv_tokens* x, void* stream);

/* The first `length` tokens' values as [batch][heads][length][head_dim] of `dtype`, keys and values (16-byte aligned). */
int ahq_kv_dequantize(const ahq_kv_cache* cache, int32_t dtype, int32_t length, void* k, void* v, void* stream);

/* softmax(scale * q k^T) v over the cache.  Codes are exact in both products, 16-bit queries as well (bfloat16
 * down to 2^-30 of a row's largest value); float32 queries have 22 bits, those far below a row's largest value fewer;
 * probabilities 22 bits for queries of every type, sums are float32.  Blocks whose values are all below 2^-72 of the largest
 * one that the call's queries see of their sequence and head count as up to that.  The workspace (0 bytes where the token
 * axis is not split) depends on the shapes and on whether the lengths are a device array, not on their values. */
size_t ahq_kv_attend_workspace_bytes(const ahq_kv_cache* cache, const ahq_kv_queries* q);
int ahq_kv_attend(const ahq_kv_cache* cache, const ahq_kv_queries* q, void* workspace, size_t workspace_bytes,
                  void* stream);

#ifdef __cplusplus
}
#endif
#endif /* AIMET_AMD_SERVING_H */
