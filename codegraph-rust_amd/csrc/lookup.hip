// lookup.hip - rows of a table by id, scaled, and the table's gradient (include/cgvec_train.h).
//
// Gradient: out of n incoming rows every table row r gets the sum of those whose id is r. A thread owns 16 bytes of one table
// row and adds up its summands, so that each row is written exactly once and no atomics touch a float; for that the positions
// are sorted by id first (stable, so that a row's summands come in the order of the input).
//   few ids (<= DIRECT_IDS): a workgroup owns some table rows, looks through all ids itself, and there is one launch;
//   more: (id, position) sorted, by one workgroup up to SMALL_SORT of them, else by radix, 11 bits at most a pass; a run's ends are
//   noted per row; rows whose run is longer than `longer` positions are first summed in pieces of that many by separate waves (a
//   frequent token would otherwise keep one thread busy).
// Bound by the bytes of the incoming rows and of the whole table gradient. 65 536 ids, 100 k x 768 f32: forward 61 us (402 MB, 6.6 TB/s), rows
// of the gradient 100 us (508 MB, 5.1 TB/s), pieces of long runs 18 us, sorting 33 us; 10 240 rows of 768 bf16: 8 us.
#include <type_traits>

#include "../../include/cgvec_train.h"
#include "ops_common.h"
#include "sort_ids.h"

using namespace cgv_ops;

namespace {

// Without sorting a row's summands come one after another. 10 k x 384 fp16, ids at random / all the same: 250 ids 10 / 99 us, sorted 22 / 21;
// 500 ids 10 / 195, sorted 21 / 22
constexpr uint32_t DIRECT_IDS = 256;
constexpr uint32_t FLIGHT = 4;

// ---- a vector of a row: V elements, 16 bytes where rows are so aligned, else 8, 4 or one element -----------------------------
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <int BYTES>
struct Words { typedef u32x4 type; };
template <>
struct Words<8> { typedef u32x2 type; };
template <>
struct Words<4> { typedef uint32_t type; };
template <>
struct Words<2> { typedef uint16_t type; };
__device__ inline uint32_t word(u32x4 v, int i) { return v[i]; }
__device__ inline uint32_t word(u32x2 v, int i) { return v[i & 1]; }
__device__ inline uint32_t word(uint32_t v, int) { return v; }
__device__ inline uint32_t word(uint16_t v, int) { return v; }
__device__ inline void set_word(u32x4& v, int i, uint32_t x) { v[i] = x; }
__device__ inline void set_word(u32x2& v, int i, uint32_t x) { v[i & 1] = x; }
__device__ inline void set_word(uint32_t& v, int, uint32_t x) { v = x; }
__device__ inline void set_word(uint16_t& v, int, uint32_t x) { v = (uint16_t)x; }

template <int DT, int V>
struct Vec {
    static constexpr int ES = DT == cgv::DT_F32 ? 4 : 2, N = V * ES < 4 ? 1 : V * ES / 4;   // words
    typedef typename Words<V * ES>::type Raw;
    float v[V];
    __device__ void zero() {
        for (int i = 0; i < V; ++i) v[i] = 0.0f;
    }
    __device__ void load(const void* p, uint64_t at) {   // at: in elements, a multiple of V
        const Raw r = *(const Raw*)((const char*)p + at * ES);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (DT == cgv::DT_F32) v[i] = __uint_as_float(word(r, i));
            else v[i] = half_to_f32<DT>((uint16_t)(word(r, i / 2) >> (16 * (i & 1))));
        }
    }
    // ONCE: past the caches
    template <bool ONCE>
    __device__ void store(void* p, uint64_t at) const {
        Raw r;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (DT == cgv::DT_F32) set_word(r, i, __float_as_uint(v[i]));
            else set_word(r, i, f32_to_half<DT>(v[2 * i]) | (V > 1 ? (uint32_t)f32_to_half<DT>(v[(2 * i + 1) % V]) << 16 : 0u));
        }
        Raw* o = (Raw*)((char*)p + at * ES);
        if (ONCE) __builtin_nontemporal_store(r, o);
        else *o = r;
    }
    __device__ void add(const Vec& o) {
        for (int i = 0; i < V; ++i) v[i] += o.v[i];
    }
    __device__ void mul(float s) {
        for (int i = 0; i < V; ++i) v[i] *= s;
    }
};

// ---- forward ----------------------------------------------------------------------------------------------------------------
// one thread per vector of the output; VPR vectors a row
template <int DT, int V, bool ONCE>
__global__ __launch_bounds__(256) void lookup_kernel(const void* __restrict__ table, uint64_t n_rows, uint32_t vpr, uint64_t row_stride,
                                                     const int64_t* __restrict__ ids, uint64_t n_ids, float scale, void* __restrict__ out) {
    const uint64_t base = wide_block() * 256;
    const uint64_t row0 = base / vpr;                       // the same for the whole workgroup
    const uint32_t in = (uint32_t)(base % vpr) + threadIdx.x;
    const uint64_t row = row0 + in / vpr;
    if (row >= n_ids) return;
    const uint32_t col = in % vpr;
    const int64_t id = ids[row];
    Vec<DT, V> v;
    if (id >= 0 && (uint64_t)id < n_rows) {
        v.load(table, (uint64_t)id * row_stride + (uint64_t)col * V);
        v.mul(scale);
    } else {
        v.zero();
    }
    v.template store<ONCE>(out, (row * vpr + col) * V);
}

// ---- gradient, few ids ------------------------------------------------------------------------------------------------------
template <int DT, int V, bool ONCE>
__global__ __launch_bounds__(256) void grad_direct_kernel(const void* __restrict__ dout, const int64_t* __restrict__ ids, uint32_t n_ids,
                                                          uint64_t n_rows, uint32_t vpr, uint32_t rows_per_block, float scale,
                                                          void* __restrict__ dtable) {
    __shared__ uint32_t mine[DIRECT_IDS], at[DIRECT_IDS];   // the ids that name a row of this workgroup: row - row0, and their place
    __shared__ uint32_t found;
    const uint64_t row0 = wide_block() * rows_per_block;
    if (row0 >= n_rows) return;
    const uint32_t rows = (uint32_t)min((uint64_t)rows_per_block, n_rows - row0);
    if (threadIdx.x < 64) {   // one wave: the list keeps the order of the input
        uint32_t base = 0;
        for (uint32_t a = 0; a < n_ids; a += 64) {
            const uint32_t i = a + threadIdx.x;
            const int64_t id = i < n_ids ? ids[i] : -1;
            const bool in = id >= (int64_t)row0 && id < (int64_t)(row0 + rows);
            const uint64_t m = __ballot(in);
            if (in) {
                const uint32_t k = base + __popcll(m & ((1ull << threadIdx.x) - 1));
                mine[k] = (uint32_t)(id - (int64_t)row0);
                at[k] = i;
            }
            base += __popcll(m);
        }
        if (threadIdx.x == 0) found = base;
    }
    __syncthreads();
    const uint32_t nf = found;
    for (uint32_t t = threadIdx.x; t < rows * vpr; t += 256) {
        const uint32_t r = t / vpr, col = t % vpr;
        Vec<DT, V> acc, v;
        acc.zero();
        for (uint32_t k = 0; k < nf; ++k)
            if (mine[k] == r) {
                v.load(dout, ((uint64_t)at[k] * vpr + col) * V);
                acc.add(v);
            }
        acc.mul(scale);
        acc.template store<ONCE>(dtable, ((row0 + r) * vpr + col) * V);
    }
}

// ---- gradient, sorted (sort_ids.h) ------------------------------------------------------------------------------------------
// runs[r] = where the positions of row r begin (low word) and end (high word)
__global__ __launch_bounds__(256) void runs_kernel(const uint32_t* __restrict__ keys, uint32_t n, uint32_t n_rows, uint32_t* __restrict__ runs) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const uint32_t k = keys[i];
    if (k >= n_rows) return;
    if (i == 0 || keys[i - 1] != k) runs[2 * (uint64_t)k] = i;
    if (i + 1 == n || keys[i + 1] != k) runs[2 * (uint64_t)k + 1] = i + 1;
}

template <int DT, int V>
__device__ inline void sum_positions(Vec<DT, V>& acc, const void* dout, const uint32_t* pos, uint32_t lo, uint32_t hi, uint32_t vpr, uint32_t col) {
    uint32_t k = lo;
    for (; k + FLIGHT <= hi; k += FLIGHT) {     // that many rows on their way at a time
        Vec<DT, V> v[FLIGHT];
#pragma unroll
        for (uint32_t j = 0; j < FLIGHT; ++j) v[j].load(dout, ((uint64_t)pos[k + j] * vpr + col) * V);
#pragma unroll
        for (uint32_t j = 0; j < FLIGHT; ++j) acc.add(v[j]);
    }
    for (; k < hi; ++k) {
        Vec<DT, V> v;
        v.load(dout, ((uint64_t)pos[k] * vpr + col) * V);
        acc.add(v);
    }
}

// piece c of `longer` sorted positions: a longer run crosses an end of every piece it touches, so a piece has at most two
// such runs - the one of its first position (slot 2 c) and the one of its last (slot 2 c + 1)
template <int DT, int V>
__global__ __launch_bounds__(64) void pieces_kernel(const void* __restrict__ dout, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos,
                                                    const uint64_t* __restrict__ runs, uint32_t n, uint32_t n_rows, uint32_t longer, uint32_t vpr,
                                                    float* __restrict__ partial) {
    const uint32_t c = blockIdx.x, lo = c * longer, hi = min(lo + longer, n);
    const uint32_t col = blockIdx.y * 64 + threadIdx.x;
    if (col >= vpr) return;
    const uint32_t first = keys[lo], last = keys[hi - 1];
    for (int side = 0; side < 2; ++side) {
        const uint32_t k = side ? last : first;
        if (k >= n_rows || (side && last == first)) continue;
        const uint32_t b = (uint32_t)runs[k], e = (uint32_t)(runs[k] >> 32);
        if (e - b <= longer) continue;
        Vec<DT, V> acc;
        acc.zero();
        sum_positions<DT, V>(acc, dout, pos, max(lo, b), min(hi, e), vpr, col);
        for (int i = 0; i < V; ++i) partial[(((uint64_t)c * 2 + side) * vpr + col) * V + i] = acc.v[i];
    }
}

template <int DT, int V, bool ONCE>
__global__ __launch_bounds__(256) void grad_rows_kernel(const void* __restrict__ dout, const uint32_t* __restrict__ pos,
                                                        const uint64_t* __restrict__ runs, uint64_t n_rows, uint32_t longer, uint32_t vpr,
                                                        const float* __restrict__ partial, float scale, void* __restrict__ dtable) {
    const uint64_t base = wide_block() * 256;
    const uint64_t row0 = base / vpr;
    const uint32_t in = (uint32_t)(base % vpr) + threadIdx.x;
    const uint64_t row = row0 + in / vpr;
    if (row >= n_rows) return;
    const uint32_t col = in % vpr;
    const uint32_t b = (uint32_t)runs[row], e = (uint32_t)(runs[row] >> 32);
    Vec<DT, V> acc;
    acc.zero();
    if (e - b <= longer) {
        sum_positions<DT, V>(acc, dout, pos, b, e, vpr, col);
    } else {
        // the piece in which the run begins has it in slot 1, unless it begins there too; the others in slot 0
        uint32_t c = b / longer;
        const uint32_t last = (e - 1) / longer;
        constexpr int W = V < 4 ? V : 4, H = V / W;        // partial sums are f32: two vectors for eight elements
        Vec<cgv::DT_F32, W> t[FLIGHT][H];
        auto add = [&](uint32_t count) {
#pragma unroll
            for (uint32_t j = 0; j < FLIGHT; ++j)
                if (j < count)
#pragma unroll
                    for (int h = 0; h < H; ++h)
                        t[j][h].load(partial, (((uint64_t)(c + j) * 2 + ((c + j) * longer < b ? 1 : 0)) * vpr + col) * V + h * W);
#pragma unroll
            for (uint32_t j = 0; j < FLIGHT; ++j)
                if (j < count)
#pragma unroll
                    for (int i = 0; i < V; ++i) acc.v[i] += t[j][i / W].v[i % W];
            c += count;
        };
        while (c + FLIGHT <= last + 1) add(FLIGHT);
        if (c <= last) add(last + 1 - c);
    }
    acc.mul(scale);
    acc.template store<ONCE>(dtable, (row * vpr + col) * V);
}

// ---- host -------------------------------------------------------------------------------------------------------------------

struct GradPlan {
    SortPlan sort;
    uint32_t longer = 0;
    uint64_t off_runs, off_partial, bytes = 0;
    GradPlan(uint64_t n, uint64_t n_rows, uint32_t dim) : sort(n > DIRECT_IDS ? n : 0, n_rows) {
        if (n <= DIRECT_IDS) return;
        // a run is summed by one thread up to `longer` positions, and pieces of a longer one by one thread again: an eighth
        // of the root of n keeps both chains short (100 k ids into 20 k x 1024 fp16: 106 us with half the root, 78 with an eighth)
        longer = 32;
        while ((uint64_t)longer * longer * 64 < n) longer *= 2;
        const uint64_t pieces = (n + longer - 1) / longer;
        bytes = sort.bytes;
        off_runs = bytes, bytes += up256(n_rows * 8);
        off_partial = bytes, bytes += up256(pieces * 2 * dim * 4);
    }
};

// elements of a vector: the most that 16 bytes hold and every row's start and length allow
uint32_t vector_elems(uint32_t dim, int dtype, uint64_t stride, const void* a, const void* b) {
    const uint32_t es = esize(dtype);
    uint32_t v = 16 / es;
    while (v > 1 && ((uint64_t)dim % v || stride % v || ((uintptr_t)a | (uintptr_t)b) % (v * es))) v /= 2;
    return v;
}

// Results larger than this are stored past the caches, which could not hold them for a reader anyway (gradient of 100 k x 768 f32 by 65 536
// ids: 187 -> 115 us; 200 MB of looked-up rows: 60 -> 44 us)
constexpr uint64_t ONCE_BYTES = 64ull << 20;

template <class F>
int by_vector(int dtype, uint32_t v, F&& f) {
    return by_dtype(dtype, [&](auto t) {
        if (v == 1) return f(t, std::integral_constant<int, 1>());
        if (v == 2) return f(t, std::integral_constant<int, 2>());
        if (decltype(t)::value == cgv::DT_F32 || v == 4) return f(t, std::integral_constant<int, 4>());
        return f(t, std::integral_constant<int, decltype(t)::value == cgv::DT_F32 ? 4 : 8>());
    });
}

int check_common(int dtype, uint64_t n_rows, uint32_t dim, uint64_t n_ids, float scale) {
    if (dtype != CGV_DTYPE_F32 && dtype != CGV_DTYPE_BF16 && dtype != CGV_DTYPE_FP16) return fail(CGV_ERR_INVALID_ARG, "dtype must be f32, bf16 or fp16");
    if (dim == 0 || dim > 8192) return fail(CGV_ERR_INVALID_ARG, "dim must be in 1..=8192");
    if (n_rows >= (1ull << 31) || n_ids >= (1ull << 31)) return fail(CGV_ERR_INVALID_ARG, "n_rows and n_ids must be below 2^31");
    if (!(fabsf(scale) < INFINITY)) return fail(CGV_ERR_NONFINITE, "scale is not finite");
    return CGV_OK;
}

template <int DT, int V>
int launch_lookup(const void* table, uint64_t n_rows, uint32_t dim, uint64_t stride, const int64_t* ids, uint64_t n_ids, float scale, void* out,
                  hipStream_t s) {
    const uint32_t vpr = dim / V;
    const uint64_t blocks = (n_ids * vpr + 255) / 256;
    if (blocks > MOST_BLOCKS) return fail(CGV_ERR_INVALID_ARG, "too many elements for one call");
    auto kern = n_ids * dim * (DT == cgv::DT_F32 ? 4 : 2) > ONCE_BYTES ? lookup_kernel<DT, V, true> : lookup_kernel<DT, V, false>;
    hipLaunchKernelGGL(kern, wide_grid(blocks), dim3(256), 0, s, table, n_rows, vpr, stride, ids, n_ids, scale, out);
    OPCHK(hipGetLastError());
    return CGV_OK;
}

template <int DT, int V>
int launch_grad(const void* dout, const int64_t* ids, uint64_t n_ids, uint64_t n_rows, uint32_t dim, float scale, void* dtable, char* ws,
                const GradPlan& pl, hipStream_t s) {
    const uint32_t vpr = dim / V;
    const uint64_t blocks = (n_rows * vpr + 255) / 256;
    if (blocks > MOST_BLOCKS) return fail(CGV_ERR_INVALID_ARG, "too many elements for one call");
    const bool once = n_rows * dim * (DT == cgv::DT_F32 ? 4 : 2) > ONCE_BYTES;
    if (!pl.sort.passes) {
        const uint32_t rpb = std::max<uint32_t>(1, 1024 / vpr);      // four vectors a thread
        auto kern = once ? grad_direct_kernel<DT, V, true> : grad_direct_kernel<DT, V, false>;
        hipLaunchKernelGGL(kern, wide_grid((n_rows + rpb - 1) / rpb), dim3(256), 0, s, dout, ids, (uint32_t)n_ids, n_rows,
                           vpr, rpb, scale, dtable);
        OPCHK(hipGetLastError());
        return CGV_OK;
    }
    uint64_t* runs = (uint64_t*)(ws + pl.off_runs);
    const uint32_t *keys, *pos;
    if (const int rc = sort_ids(pl.sort, ids, n_ids, n_rows, ws, runs, &keys, &pos, s)) return rc;
    float* partial = (float*)(ws + pl.off_partial);
    const uint32_t n = (uint32_t)n_ids;
    hipLaunchKernelGGL(runs_kernel, dim3((n + 255) / 256), dim3(256), 0, s, keys, n, (uint32_t)n_rows, (uint32_t*)runs);
    OPCHK(hipGetLastError());
    hipLaunchKernelGGL((pieces_kernel<DT, V>), dim3((n + pl.longer - 1) / pl.longer, (vpr + 63) / 64), dim3(64), 0, s, dout, keys, pos,
                       (const uint64_t*)runs, n, (uint32_t)n_rows, pl.longer, vpr, partial);
    OPCHK(hipGetLastError());
    auto kern = once ? grad_rows_kernel<DT, V, true> : grad_rows_kernel<DT, V, false>;
    hipLaunchKernelGGL(kern, wide_grid(blocks), dim3(256), 0, s, dout, pos, (const uint64_t*)runs, n_rows, pl.longer, vpr,
                       (const float*)partial, scale, dtable);
    OPCHK(hipGetLastError());
    return CGV_OK;
}

}  // namespace

extern "C" {

int cgv_lookup_rows_dev(int device_id, const void* table_dev, int dtype, uint64_t n_rows, uint32_t dim, uint64_t row_stride,
                        const int64_t* ids_dev, uint64_t n_ids, float scale, void* out_dev, void* stream) {
    return guarded([&]() -> int {
        int rc = check_common(dtype, n_rows, dim, n_ids, scale);
        if (rc) return rc;
        if (row_stride < dim) return fail(CGV_ERR_INVALID_ARG, "row_stride is smaller than dim");
        if (n_ids == 0) return CGV_OK;
        if (!ids_dev || !out_dev || (n_rows && !table_dev)) return fail(CGV_ERR_INVALID_ARG, "NULL argument");
        if ((rc = need_gpu(device_id))) return rc;
        DeviceScope dev(device_id);
        OPCHK(dev.enter());
        return by_vector(dtype, vector_elems(dim, dtype, row_stride, table_dev, out_dev), [&](auto t, auto v) {
            return launch_lookup<decltype(t)::value, decltype(v)::value>(table_dev, n_rows, dim, row_stride, ids_dev, n_ids, scale, out_dev,
                                                                         (hipStream_t)stream);
        });
    });
}

size_t cgv_lookup_grad_workspace(uint64_t n_ids, uint64_t n_rows, uint32_t dim) {
    if (n_rows >= (1ull << 31) || n_ids >= (1ull << 31) || dim == 0 || dim > 8192 || n_rows == 0) return 0;
    return (size_t)GradPlan(n_ids, n_rows, dim).bytes;
}

int cgv_lookup_grad_dev(int device_id, const void* dout_dev, int dtype, const int64_t* ids_dev, uint64_t n_ids, uint64_t n_rows,
                        uint32_t dim, float scale, void* dtable_dev, void* workspace_dev, size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        int rc = check_common(dtype, n_rows, dim, n_ids, scale);
        if (rc) return rc;
        if (n_rows == 0) return CGV_OK;
        if (!dtable_dev || (n_ids && (!dout_dev || !ids_dev))) return fail(CGV_ERR_INVALID_ARG, "NULL argument");
        const GradPlan pl(n_ids, n_rows, dim);
        if (workspace_bytes < pl.bytes || (pl.bytes && !workspace_dev)) return fail(CGV_ERR_INVALID_ARG, "the workspace is smaller than cgv_lookup_grad_workspace says");
        if ((uintptr_t)workspace_dev % 256 && pl.bytes) return fail(CGV_ERR_INVALID_ARG, "the workspace must be aligned to 256 bytes");
        if ((rc = need_gpu(device_id))) return rc;
        DeviceScope dev(device_id);
        OPCHK(dev.enter());
        return by_vector(dtype, vector_elems(dim, dtype, dim, dout_dev, dtable_dev), [&](auto t, auto v) {
            return launch_grad<decltype(t)::value, decltype(v)::value>(dout_dev, ids_dev, n_ids, n_rows, dim, scale, dtable_dev, (char*)workspace_dev, pl,
                                                                       (hipStream_t)stream);
        });
    });
}

}  // extern "C"
