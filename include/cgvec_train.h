/* cgvec_train.h - C ABI of what trains the rows and queries an index serves: rows of a table by id with their gradient, and the
 * softmax losses of queries against ALL rows of a corpus with theirs.
 *
 * All buffers are DEVICE memory of `device_id`, rows are contiguous in their elements, dtype is CGV_DTYPE_F32, CGV_DTYPE_BF16 or
 * CGV_DTYPE_FP16; sums are f32, each output is rounded once. Every call only enqueues on `stream` (a hipStream_t; NULL is HIP's
 * default stream): it allocates nothing, waits for nothing, can be captured into a HIP graph, and the thread's current device is
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
 * Ids are sorted (a stable radix sort), a row's summands are added in a fixed order. */
size_t cgv_lookup_grad_workspace(uint64_t n_ids, uint64_t n_rows, uint32_t dim);
int cgv_lookup_grad_dev(int device_id, const void* dout_dev, int dtype, const int64_t* ids_dev, uint64_t n_ids, uint64_t n_rows,
                        uint32_t dim, float scale, void* dtable_dev, void* workspace_dev, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* CGVEC_TRAIN_H */
