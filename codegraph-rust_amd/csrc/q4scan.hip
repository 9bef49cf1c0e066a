// q4scan.hip - scores of a few queries against a corpus in 4 bits with group scales (include/cgvec_q4.h).
//
// Layout in HBM. 16 rows form a tile, 128 elements of them a chunk of 1 KiB; lane l = c * 16 + r of a wave owns 16 bytes of
// it: row r, and in dword t the eight elements t * 32 + c * 8 + 0..7. One 16-byte load per lane thus reads a whole chunk as
// one linear kilobyte, and dword t of the 64 lanes is a 16 x 32 piece of the tile whose 32 columns lie in ONE group.
// Inside a dword element 2p sits in nibble p and element 2p + 1 in nibble p + 4, so that one shift and one mask give the
// two elements of a pair in the two halves of a register.
// The scales of a tile's chunk are [16 rows][128 / group] behind each other.
#include <mutex>
#include <type_traits>

#include "../../include/cgvec_q4.h"
#include "ops_common.h"

using namespace cgv_ops;

namespace {

constexpr uint32_t CHUNK = 128;           // elements of a chunk
constexpr uint32_t CHUNK_BYTES = 1024;    // of 16 rows

struct Layout {
    uint32_t dim, group, ng, kc, gpc;     // groups per row, chunks per row, groups per chunk
    __host__ __device__ uint64_t tile_codes(uint64_t tile) const { return tile * kc * CHUNK_BYTES; }
    __host__ __device__ uint64_t tile_scales(uint64_t tile) const { return tile * kc * gpc * 16; }
    // dword of elements e .. e + 7 (e a multiple of 8) of row r
    __host__ __device__ uint64_t dword(uint64_t row, uint32_t e) const {
        const uint32_t in = e % CHUNK;
        return (tile_codes(row / 16) + (uint64_t)(e / CHUNK) * CHUNK_BYTES) / 4 + ((in % 32) / 8 * 16 + row % 16) * 4 + in / 32;
    }
    __host__ __device__ uint64_t scale(uint64_t row, uint32_t g) const {
        return tile_scales(row / 16) + ((uint64_t)(g / gpc) * 16 + row % 16) * gpc + g % gpc;
    }
};

constexpr uint32_t BAD_NONFINITE = 1, BAD_RANGE = 2;

__device__ inline uint32_t pair_bits(uint32_t c0, uint32_t c1, uint32_t p) { return c0 << (4 * p) | c1 << (16 + 4 * p); }

// one wave per row: 64 lanes x 2 elements = one chunk per step
template <int SDT>
__global__ __launch_bounds__(256) void q4_quantise_kernel(const float* __restrict__ rows, uint64_t n, uint64_t row0, Layout L,
                                                          uint32_t* __restrict__ codes, uint16_t* __restrict__ scales,
                                                          uint32_t* __restrict__ bad) {
    const int lane = threadIdx.x & 63;
    const uint64_t i = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= n) return;
    const float* x = rows + i * L.dim;
    for (uint32_t k = 0; k < L.kc; ++k) {
        const uint32_t e = k * CHUNK + lane * 2;
        const float v0 = e < L.dim ? x[e] : 0.0f, v1 = e + 1 < L.dim ? x[e + 1] : 0.0f;
        if (!(fabsf(v0) < INFINITY) || !(fabsf(v1) < INFINITY)) atomicOr(bad, BAD_NONFINITE);
        float a = fmaxf(fabsf(v0), fabsf(v1));
        for (uint32_t o = 1; o < L.group / 2; o <<= 1) a = fmaxf(a, __shfl_xor(a, (int)o));
        const uint16_t sb = f32_to_half<SDT>(a / 7.0f);
        const float s = half_to_f32<SDT>(sb);
        if (!(s < INFINITY)) atomicOr(bad, BAD_RANGE);
        const uint32_t g = e / L.group;
        if (lane % (L.group / 2) == 0) scales[L.scale(row0 + i, g)] = g < L.ng ? sb : (uint16_t)0;
        const int q0 = s > 0.0f ? (int)fminf(fmaxf(rintf(v0 / s), -8.0f), 7.0f) : 0;
        const int q1 = s > 0.0f ? (int)fminf(fmaxf(rintf(v1 / s), -8.0f), 7.0f) : 0;
        uint32_t w = pair_bits((uint32_t)(q0 + 8), (uint32_t)(q1 + 8), lane & 3);
        w |= __shfl_xor(w, 1);
        w |= __shfl_xor(w, 2);
        if ((lane & 3) == 0) codes[L.dword(row0 + i, e)] = w;
    }
}

template <int SDT>
__global__ __launch_bounds__(256) void q4_pack_kernel(const uint8_t* __restrict__ src, const uint16_t* __restrict__ src_scales,
                                                      uint64_t n, uint64_t row0, Layout L, uint32_t* __restrict__ codes,
                                                      uint16_t* __restrict__ scales, uint32_t* __restrict__ bad) {
    const int lane = threadIdx.x & 63;
    const uint64_t i = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= n) return;
    const uint32_t rb = (L.dim + 1) / 2;
    for (uint32_t k = 0; k < L.kc; ++k) {
        const uint32_t e = k * CHUNK + lane * 2;
        const uint32_t b = e < L.dim ? src[i * rb + e / 2] : 0x88u;
        uint32_t w = pair_bits(b & 15u, e + 1 < L.dim ? b >> 4 : 8u, lane & 3);
        w |= __shfl_xor(w, 1);
        w |= __shfl_xor(w, 2);
        if ((lane & 3) == 0) codes[L.dword(row0 + i, e)] = w;
    }
    for (uint32_t g = lane; g < L.kc * L.gpc; g += 64) {
        const uint16_t s = g < L.ng ? src_scales[i * L.ng + g] : (uint16_t)0;
        if (!(fabsf(half_to_f32<SDT>(s)) < INFINITY)) atomicOr(bad, BAD_NONFINITE);
        scales[L.scale(row0 + i, g)] = s;
    }
}

template <int SDT>
__global__ void q4_get_row_kernel(const uint32_t* __restrict__ codes, const uint16_t* __restrict__ scales, uint64_t row, Layout L,
                                  float* __restrict__ out) {
    for (uint32_t e = threadIdx.x; e < L.dim; e += blockDim.x) {
        const uint32_t w = codes[L.dword(row, e & ~7u)], j = e & 7u;
        const int c = (int)((w >> (4 * (j >> 1) + 16 * (j & 1u))) & 15u);
        out[e] = half_to_f32<SDT>(scales[L.scale(row, e / L.group)]) * (float)(c - 8);
    }
}

// scores of MB queries (from q0): a wave per tile, its lane (c, r) sums the elements c * 8 .. + 7 of every 32 of row r in f32,
// the four lanes of a row are added at the end. Queries stand in LDS as f32, padded with zeros to whole chunks.
template <int MB, int QDT, int SDT>
__global__ __launch_bounds__(256) void q4_scores_kernel(const uint4* __restrict__ codes, const uint16_t* __restrict__ scales,
                                                        const void* __restrict__ queries, uint64_t n, Layout L, uint32_t m,
                                                        float* __restrict__ out) {
    extern __shared__ float xs[];   // [MB][kc * CHUNK]
    const uint32_t kp = L.kc * CHUNK;
    for (uint32_t i = threadIdx.x; i < MB * kp; i += 256) {
        const uint32_t q = i / kp, e = i % kp;
        const float v = (q < m && e < L.dim) ? load_elem<QDT>(queries, (uint64_t)q * L.dim + e) : 0.0f;
        xs[i] = fabsf(v) < INFINITY ? v : NAN;
    }
    __syncthreads();
    const uint32_t lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
    const uint64_t tiles = (n + 15) / 16;
    for (uint64_t tile = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6); tile < tiles; tile += (uint64_t)gridDim.x * 4) {
        float acc[MB];
        for (int q = 0; q < MB; ++q) acc[q] = 0.0f;
        const uint4* cp = codes + L.tile_codes(tile) / 16 + lane;
        const uint16_t* sp = scales + L.tile_scales(tile) + r * L.gpc;
        for (uint32_t k = 0; k < L.kc; ++k) {
            const uint4 v = cp[(uint64_t)k * 64];
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const float s = half_to_f32<SDT>(sp[(uint64_t)k * 16 * L.gpc + (uint32_t)t * 32 / L.group]);
                float part[MB];
                for (int q = 0; q < MB; ++q) part[q] = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float cv = (float)((int)((w[t] >> (4 * (j >> 1) + 16 * (j & 1))) & 15u) - 8);
#pragma unroll
                    for (int q = 0; q < MB; ++q) part[q] = fmaf(xs[q * kp + k * CHUNK + t * 32 + c * 8 + j], cv, part[q]);
                }
#pragma unroll
                for (int q = 0; q < MB; ++q) acc[q] = fmaf(s, part[q], acc[q]);
            }
        }
#pragma unroll
        for (int q = 0; q < MB; ++q) {
            acc[q] += __shfl_xor(acc[q], 16);
            acc[q] += __shfl_xor(acc[q], 32);
            const uint64_t row = tile * 16 + r;
            if (c == 0 && (uint32_t)q < m && row < n) out[(uint64_t)q * n + row] = acc[q];
        }
    }
}

}  // namespace

struct cgv_q4_index {
    int device = 0, sdt = CGV_DTYPE_FP16;
    Layout L{};
    uint64_t n = 0, cap = 0;        // rows; cap a multiple of 16
    uint32_t* codes = nullptr;
    uint16_t* scales = nullptr;
    void* stage = nullptr;          // host forms: rows, queries, scores
    size_t stage_bytes = 0;
    uint32_t* bad = nullptr;
    hipStream_t stream = nullptr;
    mutable std::mutex mu;
};

namespace {

int ensure_stage(cgv_q4_index* h, size_t bytes) {
    if (bytes <= h->stage_bytes) return CGV_OK;
    OPCHK(hipStreamSynchronize(h->stream));
    if (h->stage) (void)hipFree(h->stage);
    h->stage = nullptr;
    h->stage_bytes = 0;
    OPCHK(hipMalloc(&h->stage, bytes));
    h->stage_bytes = bytes;
    return CGV_OK;
}

int grow(cgv_q4_index* h, uint64_t rows, bool exact) {
    if (rows <= h->cap) return CGV_OK;
    uint64_t want = exact ? rows : std::max<uint64_t>(rows, h->cap + h->cap / 2);
    want = (std::max<uint64_t>(want, 1024) + 15) / 16 * 16;
    uint32_t* c = nullptr;
    uint16_t* s = nullptr;
    const uint64_t cb = h->L.tile_codes(want / 16), sb = h->L.tile_scales(want / 16) * 2;
    OPCHK(hipMalloc((void**)&c, cb));
    hipError_t e = hipMalloc((void**)&s, sb);
    const uint64_t used = (h->n + 15) / 16;
    if (e == hipSuccess && used) e = hipMemcpyAsync(c, h->codes, h->L.tile_codes(used), hipMemcpyDeviceToDevice, h->stream);
    if (e == hipSuccess && used) e = hipMemcpyAsync(s, h->scales, h->L.tile_scales(used) * 2, hipMemcpyDeviceToDevice, h->stream);
    // scores enqueued on other streams may still read the old buffers
    if (e == hipSuccess) e = hipDeviceSynchronize();
    if (e != hipSuccess) {
        (void)hipGetLastError();
        (void)hipFree(c);
        if (s) (void)hipFree(s);
        return fail(e == hipErrorOutOfMemory ? CGV_ERR_OOM : CGV_ERR_HIP, std::string("growing the 4-bit corpus: ") + hipGetErrorString(e));
    }
    if (h->codes) (void)hipFree(h->codes);
    if (h->scales) (void)hipFree(h->scales);
    h->codes = c;
    h->scales = s;
    h->cap = want;
    return CGV_OK;
}

int refuse_capture(hipStream_t s, const char* what) {
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    OPCHK(hipStreamIsCapturing(s, &st));
    if (st != hipStreamCaptureStatusNone)
        return fail(CGV_ERR_INVALID_ARG, std::string(what) + " waits for the stream: it cannot be captured into a graph");
    return CGV_OK;
}

// reads the flags of the rows just written; they count from here on
int commit(cgv_q4_index* h, uint64_t n, hipStream_t s) {
    uint32_t bad = 0;
    OPCHK(hipMemcpyAsync(&bad, h->bad, 4, hipMemcpyDeviceToHost, s));
    OPCHK(hipStreamSynchronize(s));
    if (bad & BAD_NONFINITE) return fail(CGV_ERR_NONFINITE, "NaN or Inf in the rows or scales: not applied");
    if (bad & BAD_RANGE) return fail(CGV_ERR_INVALID_ARG, "a group's scale is beyond the scale type: not applied");
    h->n += n;
    return CGV_OK;
}

unsigned row_blocks(uint64_t n) { return (unsigned)((n + 3) / 4); }
constexpr uint64_t ROWS_PER_LAUNCH = 1ull << 22;

int quantise_rows(cgv_q4_index* h, const float* rows, uint64_t n, uint64_t at, hipStream_t s) {
    for (uint64_t a = 0; a < n; a += ROWS_PER_LAUNCH) {
        const uint64_t c = std::min<uint64_t>(ROWS_PER_LAUNCH, n - a);
        auto k = h->sdt == CGV_DTYPE_FP16 ? q4_quantise_kernel<cgv::DT_FP16> : q4_quantise_kernel<cgv::DT_BF16>;
        hipLaunchKernelGGL(k, dim3(row_blocks(c)), dim3(256), 0, s, rows + a * h->L.dim, c, at + a, h->L, h->codes, h->scales, h->bad);
        OPCHK(hipGetLastError());
    }
    return CGV_OK;
}

int pack_rows(cgv_q4_index* h, const uint8_t* codes, const uint16_t* scales, uint64_t n, uint64_t at, hipStream_t s) {
    const uint64_t rb = (h->L.dim + 1) / 2;
    for (uint64_t a = 0; a < n; a += ROWS_PER_LAUNCH) {
        const uint64_t c = std::min<uint64_t>(ROWS_PER_LAUNCH, n - a);
        auto k = h->sdt == CGV_DTYPE_FP16 ? q4_pack_kernel<cgv::DT_FP16> : q4_pack_kernel<cgv::DT_BF16>;
        hipLaunchKernelGGL(k, dim3(row_blocks(c)), dim3(256), 0, s, codes + a * rb, scales + a * h->L.ng, c, at + a, h->L, h->codes,
                           h->scales, h->bad);
        OPCHK(hipGetLastError());
    }
    return CGV_OK;
}

int begin_add(cgv_q4_index* h, uint64_t n) {
    if (n > (1ull << 40) || h->n + n > (1ull << 40)) return fail(CGV_ERR_INVALID_ARG, "too many rows");
    return grow(h, h->n + n, false);
}

template <int MB, int QDT, int SDT>
int launch_scores(const cgv_q4_index* h, const void* q, uint32_t m, float* out, hipStream_t s) {
    const uint64_t tiles = (h->n + 15) / 16;
    const unsigned blocks = (unsigned)std::min<uint64_t>((tiles + 3) / 4, 2048);
    hipLaunchKernelGGL((q4_scores_kernel<MB, QDT, SDT>), dim3(blocks), dim3(256), (size_t)MB * h->L.kc * CHUNK * 4, s,
                       (const uint4*)h->codes, (const uint16_t*)h->scales, q, h->n, h->L, m, out);
    OPCHK(hipGetLastError());
    return CGV_OK;
}

template <int QDT, int SDT>
int scores_typed(const cgv_q4_index* h, const void* q, uint32_t m, float* out, hipStream_t s) {
    for (uint32_t a = 0; a < m;) {
        const uint32_t c = std::min<uint32_t>(4, m - a);
        const char* qa = (const char*)q + (uint64_t)a * h->L.dim * (QDT == cgv::DT_F32 ? 4 : 2);
        float* oa = out + (uint64_t)a * h->n;
        const int rc = c == 1 ? launch_scores<1, QDT, SDT>(h, qa, c, oa, s) : launch_scores<4, QDT, SDT>(h, qa, c, oa, s);
        if (rc) return rc;
        a += c;
    }
    return CGV_OK;
}

int scores_on(const cgv_q4_index* h, const void* q, int qdt, uint32_t m, float* out, hipStream_t s) {
    return by_dtype(qdt, [&](auto t) {
        constexpr int Q = decltype(t)::value;
        return h->sdt == CGV_DTYPE_FP16 ? scores_typed<Q, cgv::DT_FP16>(h, q, m, out, s) : scores_typed<Q, cgv::DT_BF16>(h, q, m, out, s);
    });
}

}  // namespace

extern "C" {

int cgv_q4_create(uint32_t dim, uint32_t group, int scale_dtype, int device_id, cgv_q4_index** out) {
    return guarded([&]() -> int {
        if (!out) return fail(CGV_ERR_INVALID_ARG, "out is NULL");
        *out = nullptr;
        if (dim == 0 || dim > 8192) return fail(CGV_ERR_INVALID_ARG, "dim must be in 1..=8192");
        if (group != 32 && group != 64 && group != 128) return fail(CGV_ERR_INVALID_ARG, "group must be 32, 64 or 128");
        if (scale_dtype != CGV_DTYPE_FP16 && scale_dtype != CGV_DTYPE_BF16) return fail(CGV_ERR_INVALID_ARG, "scale_dtype must be fp16 or bf16");
        const int rc = need_gpu(device_id);
        if (rc) return rc;
        DeviceScope dev(device_id);
        OPCHK(dev.enter());
        cgv_q4_index* h = new cgv_q4_index();
        h->device = device_id;
        h->sdt = scale_dtype;
        h->L.dim = dim;
        h->L.group = group;
        h->L.ng = (dim + group - 1) / group;
        h->L.kc = (dim + CHUNK - 1) / CHUNK;
        h->L.gpc = CHUNK / group;
        hipError_t e = hipStreamCreateWithFlags(&h->stream, hipStreamNonBlocking);
        if (e == hipSuccess) e = hipMalloc((void**)&h->bad, 4);
        if (e != hipSuccess) {
            (void)hipGetLastError();
            const std::string m = hipGetErrorString(e);
            cgv_q4_destroy(h);
            return fail(CGV_ERR_HIP, "cgv_q4_create: " + m);
        }
        *out = h;
        return CGV_OK;
    });
}

int cgv_q4_destroy(cgv_q4_index* h) {
    if (!h) return CGV_OK;
    DeviceScope dev(h->device);
    (void)dev.enter();
    if (h->stream) (void)hipStreamSynchronize(h->stream);
    void* bufs[] = {h->codes, h->scales, h->stage, h->bad};
    for (void* p : bufs)
        if (p) (void)hipFree(p);   // waits for the device: scores in flight on any stream have ended
    if (h->stream) (void)hipStreamDestroy(h->stream);
    delete h;
    return CGV_OK;
}

int cgv_q4_reserve(cgv_q4_index* h, uint64_t n_rows) {
    return guarded([&]() -> int {
        if (!h) return fail(CGV_ERR_INVALID_ARG, "handle is NULL");
        if (n_rows > (1ull << 40)) return fail(CGV_ERR_INVALID_ARG, "too many rows");
        std::lock_guard<std::mutex> lk(h->mu);
        DeviceScope dev(h->device);
        OPCHK(dev.enter());
        return grow(h, n_rows, true);
    });
}

uint64_t cgv_q4_count(const cgv_q4_index* h) {
    if (!h) return 0;
    std::lock_guard<std::mutex> lk(h->mu);
    return h->n;
}

int cgv_q4_add_f32(cgv_q4_index* h, const float* rows_host, uint64_t n) {
    return guarded([&]() -> int {
        if (!h) return fail(CGV_ERR_INVALID_ARG, "handle is NULL");
        if (n == 0) return CGV_OK;
        if (!rows_host) return fail(CGV_ERR_INVALID_ARG, "rows is NULL");
        std::lock_guard<std::mutex> lk(h->mu);
        DeviceScope dev(h->device);
        OPCHK(dev.enter());
        int rc = begin_add(h, n);
        if (rc) return rc;
        OPCHK(hipMemsetAsync(h->bad, 0, 4, h->stream));
        const uint64_t chunk = std::max<uint64_t>(1, (256ull << 20) / ((uint64_t)h->L.dim * 4));
        if ((rc = ensure_stage(h, std::min(chunk, n) * h->L.dim * 4))) return rc;
        for (uint64_t a = 0; a < n; a += chunk) {
            const uint64_t c = std::min<uint64_t>(chunk, n - a);
            OPCHK(hipMemcpyAsync(h->stage, rows_host + a * h->L.dim, c * h->L.dim * 4, hipMemcpyHostToDevice, h->stream));
            if ((rc = quantise_rows(h, (const float*)h->stage, c, h->n + a, h->stream))) return rc;
            OPCHK(hipStreamSynchronize(h->stream));
        }
        return commit(h, n, h->stream);
    });
}

int cgv_q4_add_f32_dev(cgv_q4_index* h, const float* rows_dev, uint64_t n, void* stream) {
    return guarded([&]() -> int {
        if (!h) return fail(CGV_ERR_INVALID_ARG, "handle is NULL");
        if (n == 0) return CGV_OK;
        if (!rows_dev) return fail(CGV_ERR_INVALID_ARG, "rows is NULL");
        std::lock_guard<std::mutex> lk(h->mu);
        DeviceScope dev(h->device);
        OPCHK(dev.enter());
        const hipStream_t s = (hipStream_t)stream;
        int rc = refuse_capture(s, "cgv_q4_add_f32_dev");
        if (!rc) rc = begin_add(h, n);
        if (rc) return rc;
        OPCHK(hipMemsetAsync(h->bad, 0, 4, s));
        if ((rc = quantise_rows(h, rows_dev, n, h->n, s))) return rc;
        return commit(h, n, s);
    });
}

int cgv_q4_add_codes(cgv_q4_index* h, const uint8_t* codes_host, const uint16_t* scales_host, uint64_t n) {
    return guarded([&]() -> int {
        if (!h) return fail(CGV_ERR_INVALID_ARG, "handle is NULL");
        if (n == 0) return CGV_OK;
        if (!codes_host || !scales_host) return fail(CGV_ERR_INVALID_ARG, "codes or scales is NULL");
        std::lock_guard<std::mutex> lk(h->mu);
        DeviceScope dev(h->device);
        OPCHK(dev.enter());
        int rc = begin_add(h, n);
        if (rc) return rc;
        OPCHK(hipMemsetAsync(h->bad, 0, 4, h->stream));
        const uint64_t rb = (h->L.dim + 1) / 2, sb = (uint64_t)h->L.ng * 2, rb16 = (rb + 15) / 16 * 16;
        const uint64_t chunk = std::max<uint64_t>(1, (256ull << 20) / (rb16 + sb));
        const uint64_t most = std::min(chunk, n), soff = (most * rb + 15) / 16 * 16;
        if ((rc = ensure_stage(h, soff + most * sb))) return rc;
        for (uint64_t a = 0; a < n; a += chunk) {
            const uint64_t c = std::min<uint64_t>(chunk, n - a);
            char* st = (char*)h->stage;
            OPCHK(hipMemcpyAsync(st, codes_host + a * rb, c * rb, hipMemcpyHostToDevice, h->stream));
            OPCHK(hipMemcpyAsync(st + soff, scales_host + a * h->L.ng, c * sb, hipMemcpyHostToDevice, h->stream));
            if ((rc = pack_rows(h, (const uint8_t*)st, (const uint16_t*)(st + soff), c, h->n + a, h->stream))) return rc;
            OPCHK(hipStreamSynchronize(h->stream));
        }
        return commit(h, n, h->stream);
    });
}

int cgv_q4_add_codes_dev(cgv_q4_index* h, const uint8_t* codes_dev, const uint16_t* scales_dev, uint64_t n, void* stream) {
    return guarded([&]() -> int {
        if (!h) return fail(CGV_ERR_INVALID_ARG, "handle is NULL");
        if (n == 0) return CGV_OK;
        if (!codes_dev || !scales_dev) return fail(CGV_ERR_INVALID_ARG, "codes or scales is NULL");
        std::lock_guard<std::mutex> lk(h->mu);
        DeviceScope dev(h->device);
        OPCHK(dev.enter());
        const hipStream_t s = (hipStream_t)stream;
        int rc = refuse_capture(s, "cgv_q4_add_codes_dev");
        if (!rc) rc = begin_add(h, n);
        if (rc) return rc;
        OPCHK(hipMemsetAsync(h->bad, 0, 4, s));
        if ((rc = pack_rows(h, codes_dev, scales_dev, n, h->n, s))) return rc;
        return commit(h, n, s);
    });
}

int cgv_q4_get_row_f32(cgv_q4_index* h, uint64_t id, float* out_host) {
    return guarded([&]() -> int {
        if (!h || !out_host) return fail(CGV_ERR_INVALID_ARG, "NULL argument");
        std::lock_guard<std::mutex> lk(h->mu);
        if (id >= h->n) return fail(CGV_ERR_OUT_OF_RANGE, "row id out of range");
        DeviceScope dev(h->device);
        OPCHK(dev.enter());
        const int rc = ensure_stage(h, (size_t)h->L.dim * 4);
        if (rc) return rc;
        auto k = h->sdt == CGV_DTYPE_FP16 ? q4_get_row_kernel<cgv::DT_FP16> : q4_get_row_kernel<cgv::DT_BF16>;
        hipLaunchKernelGGL(k, dim3(1), dim3(256), 0, h->stream, (const uint32_t*)h->codes, (const uint16_t*)h->scales, id, h->L,
                           (float*)h->stage);
        OPCHK(hipGetLastError());
        OPCHK(hipMemcpyAsync(out_host, h->stage, (size_t)h->L.dim * 4, hipMemcpyDeviceToHost, h->stream));
        OPCHK(hipStreamSynchronize(h->stream));
        return CGV_OK;
    });
}

int cgv_q4_scores_f32(cgv_q4_index* h, const float* queries_host, uint32_t m, float* out_host) {
    return guarded([&]() -> int {
        if (!h) return fail(CGV_ERR_INVALID_ARG, "handle is NULL");
        std::lock_guard<std::mutex> lk(h->mu);
        if (m == 0 || h->n == 0) return CGV_OK;
        if (!queries_host || !out_host) return fail(CGV_ERR_INVALID_ARG, "NULL argument");
        DeviceScope dev(h->device);
        OPCHK(dev.enter());
        // queries in pieces whose scores fit the staging buffer
        const uint64_t per = std::max<uint64_t>(1, std::min<uint64_t>(m, (512ull << 20) / (h->n * 4)));
        const size_t qb = ((size_t)per * h->L.dim * 4 + 255) / 256 * 256;
        int rc = ensure_stage(h, qb + per * h->n * 4);
        if (rc) return rc;
        float* dq = (float*)h->stage;
        float* ds = (float*)((char*)h->stage + qb);
        for (uint64_t a = 0; a < m; a += per) {
            const uint32_t c = (uint32_t)std::min<uint64_t>(per, m - a);
            OPCHK(hipMemcpyAsync(dq, queries_host + a * h->L.dim, (size_t)c * h->L.dim * 4, hipMemcpyHostToDevice, h->stream));
            if ((rc = scores_on(h, dq, CGV_DTYPE_F32, c, ds, h->stream))) return rc;
            OPCHK(hipMemcpyAsync(out_host + a * h->n, ds, (size_t)c * h->n * 4, hipMemcpyDeviceToHost, h->stream));
            OPCHK(hipStreamSynchronize(h->stream));
        }
        return CGV_OK;
    });
}

int cgv_q4_scores_dev(cgv_q4_index* h, const void* queries_dev, int query_dtype, uint32_t m, float* out_dev, void* stream) {
    return guarded([&]() -> int {
        if (!h) return fail(CGV_ERR_INVALID_ARG, "handle is NULL");
        if (query_dtype != CGV_DTYPE_F32 && query_dtype != CGV_DTYPE_BF16 && query_dtype != CGV_DTYPE_FP16)
            return fail(CGV_ERR_INVALID_ARG, "dtype must be f32, bf16 or fp16");
        std::lock_guard<std::mutex> lk(h->mu);
        if (m == 0 || h->n == 0) return CGV_OK;
        if (!queries_dev || !out_dev) return fail(CGV_ERR_INVALID_ARG, "NULL argument");
        DeviceScope dev(h->device);
        OPCHK(dev.enter());
        return scores_on(h, queries_dev, query_dtype, m, out_dev, (hipStream_t)stream);
    });
}

}  // extern "C"
