/* cgvec_q4.h - C ABI of the 4-bit scan: a corpus kept as 4-bit codes with one scale per group of elements, and the dot
 * products of one or a few queries with every row.
 *
 *   value of element k of row r = scale[r][k / group] * (code[r][k] - 8),  code 0..15
 *   score[m][r]                 = sum over k of query[m][k] * value[r][k]
 *
 * It stands beside the int8 scan (cgvec_i8.h): half its bytes per element, scales that follow each group of a row instead of the
 * fixed range [-1, 1], and queries that are NOT quantised (f32: 24 bits of an element, or an absolute 2^-39 of the query's largest; fp16
 * and bf16: all bits of an element down to 2^-28 of the largest; sums in f32). The
 * reference quantises to 4 bits (optimization.rs:248-262) but scans 8-bit data only (:76-82).
 * A single query is bound by the bytes of the corpus: dim / 2 + 2 * ceil(dim / group) per row.
 * Same status / error convention as cgvec.h. No CPU fallback: creating a handle without a GPU fails.
 *
 * Threading: calls on one handle may come from several threads; those that add rows run alone. cgv_q4_scores_dev only enqueues.
 * A HIP graph that captured cgv_q4_scores_dev keeps the addresses of that moment, and a replay scores the rows that were there at
 * the capture: where rows added later move the corpus, the handle keeps what it left until it is destroyed (cgv_q4_reserve
 * beforehand keeps the corpus in place). */
#ifndef CGVEC_Q4_H
#define CGVEC_Q4_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct cgv_q4_index cgv_q4_index;

/* dim in 1..=8192; group 32, 64 or 128 elements (the last group of a row may be shorter); scale_dtype CGV_DTYPE_FP16 (scales
 * up to 65504, 11 bits) or CGV_DTYPE_BF16 (the range of f32, 8 bits). */
int cgv_q4_create(uint32_t dim, uint32_t group, int scale_dtype, int device_id, cgv_q4_index** out);
int cgv_q4_destroy(cgv_q4_index* h);
int cgv_q4_reserve(cgv_q4_index* h, uint64_t n_rows);
uint64_t cgv_q4_count(const cgv_q4_index* h);

/* Append n f32 rows, quantised on the device: scale = the group's largest magnitude / 7 rounded to the scale type, code = the
 * nearest integer of element / scale (ties to even) held to -8..7, plus 8. A group whose scale rounds to zero is stored as
 * zeros. NaN / Inf in a row: CGV_ERR_NONFINITE; a scale beyond the scale type: CGV_ERR_INVALID_ARG; nothing is added then.
 * rows_host is HOST memory; rows_dev is DEVICE memory, read on `stream`. Both return when the rows are in place. */
int cgv_q4_add_f32(cgv_q4_index* h, const float* rows_host, uint64_t n);
int cgv_q4_add_f32_dev(cgv_q4_index* h, const float* rows_dev, uint64_t n, void* stream);

/* Append n rows that are already quantised: codes [n][ceil(dim/2)] bytes, two codes per byte, low nibble first (the layout of
 * cgv_quantize_u4_f32; an odd last nibble is ignored), scales [n][ceil(dim/group)] in the handle's scale type. NaN / Inf scale:
 * CGV_ERR_NONFINITE, nothing is added. */
int cgv_q4_add_codes(cgv_q4_index* h, const uint8_t* codes_host, const uint16_t* scales_host, uint64_t n);
int cgv_q4_add_codes_dev(cgv_q4_index* h, const uint8_t* codes_dev, const uint16_t* scales_dev, uint64_t n, void* stream);

/* Row `id` as f32 values (HOST). CGV_ERR_OUT_OF_RANGE beyond the last row. */
int cgv_q4_get_row_f32(cgv_q4_index* h, uint64_t id, float* out_host);

/* Scores of m queries against the first n_rows rows: out [m][n_rows] f32; more than cgv_q4_count: CGV_ERR_OUT_OF_RANGE (rows that
 * another thread adds between the two calls do not matter). A query with a NaN or Inf gets NaN for every row. A score is Inf only
 * if it is itself beyond f32 (rows with bf16 scales of 2^94 and more cost a launch more: their sums may need 64 bits).
 * _f32: HOST queries [m][dim] and output, returns when done. _dev: DEVICE queries of type query_dtype (CGV_DTYPE_F32 / BF16 /
 * FP16), contiguous [m][dim]; enqueued on `stream`, no synchronisation, nothing allocated. m == 0 or n_rows == 0: nothing is
 * written. The workspace (DEVICE, cgv_q4_scores_workspace bytes, 0 for one query of ordinary size; aligned to 256) belongs to one
 * call until its work on the stream is done. */
int cgv_q4_scores_f32(cgv_q4_index* h, const float* queries_host, uint32_t m, uint64_t n_rows, float* out_host);
size_t cgv_q4_scores_workspace(const cgv_q4_index* h, int query_dtype, uint32_t m);
int cgv_q4_scores_dev(cgv_q4_index* h, const void* queries_dev, int query_dtype, uint32_t m, uint64_t n_rows, float* out_dev,
                      void* workspace_dev, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* CGVEC_Q4_H */
