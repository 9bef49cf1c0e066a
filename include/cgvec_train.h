/* cgvec_train.h - C ABI of what trains the rows and queries an index serves: rows of a table by id with their gradient, and the
 * softmax losses of queries against ALL rows of a corpus with theirs.
 *
 * All buffers are DEVICE memory of `device_id`, rows are contiguous in their elements, dtype is CGV_DTYPE_F32, CGV_DTYPE_BF16 or
 * CGV_DTYPE_FP16; sums are f32, each output is rounded once (what the losses' gradients round on their way stands with them). Every
 * call only enqueues on `stream` (a hipStream_t; NULL is HIP's default stream): it allocates nothing, waits for nothing, can be captured into a HIP graph, and the thread's current device is
 * left as it was. Results do not depend on the order in which workgroups run: the same call gives the same bits.
 * A workspace belongs to ONE call at a time: calls that may overlap (two streams, two captured graphs) need one each. Its size
 * comes from the *_workspace function beside the call; it needs no initial contents, an alignment of 256 bytes, and may be reused
 * as soon as the call's work on the stream is done.
 * Same status / error convention as cgvec.h. No CPU fallback. */
#ifndef CGVEC_TRAIN_H
#define CGVEC_TRAIN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* out[i] = scale * table[ids[i]], i < n_ids: the rows behind the ids of a search, or the tokens' rows of an embedding table.
 * table [n_rows] rows of dim elements, row_stride elements apart (>= dim); out [n_ids][dim], contiguous. An id outside
 * [0, n_rows) - the padding (UINT64_MAX) of a short search result among them - gives a row of zeros.
 * n_rows and n_ids below 2^31, dim in 1..=8192. */
int cgv_lookup_rows_dev(int device_id, const void* table_dev, int dtype, uint64_t n_rows, uint32_t dim, uint64_t row_stride,
                        const int64_t* ids_dev, uint64_t n_ids, float scale, void* out_dev, void* stream);

/* The table's gradient: dtable[r] = scale * (sum of dout[i] over the i with ids[i] == r, in f32), rounded to dtype. EVERY row of
 * dtable [n_rows][dim] is written; rows that no id names become zero; ids outside [0, n_rows) take no part.
 * A row's summands are added in the order of the input, those of an id with many of them in pieces: more than 256 ids are sorted
 * first, stably - up to 2048 by one workgroup, else by radix. */
size_t cgv_lookup_grad_workspace(uint64_t n_ids, uint64_t n_rows, uint32_t dim);
int cgv_lookup_grad_dev(int device_id, const void* dout_dev, int dtype, const int64_t* ids_dev, uint64_t n_ids, uint64_t n_rows,
                        uint32_t dim, float scale, void* dtable_dev, void* workspace_dev, size_t workspace_bytes, void* stream);

/* Softmax losses of b queries against ALL n_rows rows of a corpus. With s[i][j] = scale * <queries[i], rows[j]>, lse[i] =
 * log(sum over j of exp(s[i][j])) and weights p[i][0..k) on the listed rows ids[i][0..k),
 *     loss[i] = sum over t of p[i][t] * (log p[i][t] - s[i][ids[i][t]] + lse[i])
 * teacher_scores NULL: the entries with an id in [0, n_rows) share the weight equally; k = 1 is the cross entropy with label ids[i].
 * Otherwise p[i] = softmax over the entries of teacher_scale * teacher_scores[i], i.e. loss[i] is the divergence KL(p || softmax(s))
 * of the student's scores from the teacher's on its list - what a search returns goes in as it is: entries whose id is outside
 * [0, n_rows) or whose score is -Inf have weight 0 (its padding is both). An id may be listed twice: its weights add up.
 * A query without an entry of positive weight takes no part: loss 0, no gradient, its values are not read into any other result.
 * NaN or Inf in a query, in a corpus row or in a teacher's score makes the losses they enter NaN (or Inf; a corpus row whose Inf gives a
 * query of 16 bits a score of -Inf has no weight there).
 *
 * The b x n_rows scores are never stored: the corpus is scored in tiles and only a running maximum and sum per query are kept; the
 * gradient scores it again, piece by piece.
 * queries [b] rows of dim elements, query_stride elements apart; rows likewise; both of type dtype. ids [b][k] int64,
 * teacher_scores [b][k] f32, loss [b] f32. saved [b * (k + 2)] f64 carries what the gradient needs (the softmax sums, the scores of
 * the listed rows). b in 0..=2^24, k in 1..=256, n_rows in 1..2^31 - 1, dim in 1..=8192.
 * The gradient's workspace holds the scores' gradient of one piece of the corpus in 16 bits (f32: three times that): 512 MiB, or
 * 16384 rows of the corpus for very many queries; f32 rows, and rows whose dim is no multiple of 8, also a copy of the piece; fp16
 * queries a second copy. */
size_t cgv_corpus_loss_workspace(uint64_t b, uint64_t n_rows, uint32_t dim, uint32_t k, int dtype);
int cgv_corpus_loss_dev(int device_id, const void* queries_dev, uint64_t query_stride, const void* rows_dev, uint64_t row_stride, int dtype,
                        uint64_t b, uint64_t n_rows, uint32_t dim, const int64_t* ids_dev, const float* teacher_scores_dev, uint32_t k,
                        float scale, float teacher_scale, float* loss_dev, double* saved_dev, void* workspace_dev, size_t workspace_bytes,
                        void* stream);

/* Gradients of sum over i of dloss[i] * loss[i] in the queries and in the corpus rows (either may be NULL: it is not computed), from
 * the same arguments and the `saved` of the forward call: dqueries [b][dim] and drows [n_rows][dim], contiguous, of type dtype;
 * every row of them is written.
 * The scores' gradient G, softmax minus weight times dloss and scale, is what both products read. f32: it keeps 24 bits. 16-bit types: up to
 * 32 queries it keeps two parts of the type; above, an entry is rounded to the type once (fp16: at a power of two of its query's own),
 * half a step at most. What that leaves of the listed rows' entries, the largest, is always added to dqueries. It is added to drows in
 * small problems (b * k <= 1024, ceil(dim / 256) * ceil(n_rows / 256) < 128 for n_rows of a piece) and in large ones (b * n_rows * dim
 * >= 2^36, k <= n_rows / 1024), where it takes a twentieth of the time or less; drows between them are off by up to half a step of each
 * entry besides their own rounding (bf16: some 0.0023 of the norm, their own rounding alone 0.0017). */
size_t cgv_corpus_loss_grad_workspace(uint64_t b, uint64_t n_rows, uint32_t dim, uint32_t k, int dtype);
int cgv_corpus_loss_grad_dev(int device_id, const void* queries_dev, uint64_t query_stride, const void* rows_dev, uint64_t row_stride,
                             int dtype, uint64_t b, uint64_t n_rows, uint32_t dim, const int64_t* ids_dev, const float* teacher_scores_dev,
                             uint32_t k, float scale, float teacher_scale, const double* saved_dev, const float* dloss_dev,
                             void* dqueries_dev, void* drows_dev, void* workspace_dev, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* CGVEC_TRAIN_H */
