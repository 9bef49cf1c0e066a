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

// ---- scores -----------------------------------------------------------------------------------------------------------------
// One v_mfma_f32_16x16x32_f16 takes 32 columns of a 16-row tile against 16 rows of query data: codes become f16 integers -8..7
// (exact), so the only roundings are those of the query's parts and of the f32 sums. An f32 query is three f16 parts (11 bits
// each: all 24), a 16-bit query one. Parts are taken of the query scaled by a power of two to a largest magnitude of
// 2^14 .. 2^15, so that f16's range does not matter: an element keeps an absolute 2^-39 of the query's largest. A query's rows of the
// product depend on nothing but itself, so the 13 rows that a single f32 query leaves unused cost nothing and hold anything.
// A group's products are scaled and added in f32 (its scale differs from row to row of the corpus: one value per lane).
//
// Bound by the codes' way from HBM: a wave streams its tiles' chunks with the next ones already in flight. Per 8 codes a lane
// spends 11 instructions on unpacking, 4 FMAs per 32 columns on scales of group 32.
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct ScoreArgs {
    const uint4* codes;
    const uint16_t* scales;
    const void* queries;
    float* out;
    uint64_t n;
    Layout L;
    uint32_t m;            // queries of this launch
    int qdt;
};

__device__ inline float load_query(const void* q, int dt, uint64_t i) {
    return dt == CGV_DTYPE_F32 ? load_elem<cgv::DT_F32>(q, i) : dt == CGV_DTYPE_BF16 ? load_elem<cgv::DT_BF16>(q, i) : load_elem<cgv::DT_FP16>(q, i);
}

// eight codes of a dword as f16 integers -8..7: 0x6400 | c is 1024 + c
__device__ inline f16x8 unpack(uint32_t w) {
    const f16x2 off = {(_Float16)-1032.0f, (_Float16)-1032.0f};
    f16x2 p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = __builtin_bit_cast(f16x2, ((w >> (4 * i)) & 0x000f000fu) | 0x64006400u) + off;
    f16x8 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = p[i][0], v[2 * i + 1] = p[i][1];
    return v;
}

template <int GPC>
struct ScalePiece;   // the scales of one row's groups in a chunk
template <>
struct ScalePiece<1> { typedef uint16_t type; };
template <>
struct ScalePiece<2> { typedef uint32_t type; };
template <>
struct ScalePiece<4> { typedef uint2 type; };
__device__ inline uint16_t piece_at(uint16_t v, int) { return v; }
__device__ inline uint16_t piece_at(uint32_t v, int i) { return (uint16_t)(v >> (16 * i)); }
__device__ inline uint16_t piece_at(uint2 v, int i) { return (uint16_t)((i < 2 ? v.x : v.y) >> (16 * (i & 1))); }

// PARTS f16 parts of a query (3: f32 queries, 4 queries a 16-row operand; 1: 16 queries), MT such operands, NT tiles at a time
template <int PARTS, int SDT, int GPC, int MT, int NT>
__global__ __launch_bounds__(256) void q4_scores_kernel(ScoreArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr uint32_t QPT = PARTS == 3 ? 4 : 16;      // queries of an operand
    typedef typename ScalePiece<GPC>::type SP;
    const uint32_t lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4, wave = threadIdx.x >> 6;
    const uint32_t kc = a.L.kc, rows = a.m * PARTS, kp = kc * CHUNK;
    _Float16* xs = (_Float16*)smem;                    // [kp / 32][rows][32]
    int* expo = (int*)(smem + (uint64_t)rows * kp * 2);

    // this wave's tiles, and the first chunks on their way before anything else
    const uint64_t units = ((a.n + 15) / 16 + NT - 1) / NT, waves = (uint64_t)gridDim.x * 4, w = (uint64_t)blockIdx.x * 4 + wave;
    const uint64_t u0 = units * w / waves, u1 = units * (w + 1) / waves;
    const uint64_t tiles = (a.n + 15) / 16;
    struct Chunk {
        uint4 v[NT];
        SP s[NT];
    };
    uint64_t lu = u0;          // the load side's unit and chunk
    uint32_t lk = 0;
    auto load = [&](Chunk& ch) {
        if (lu < u1) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const uint64_t tile = min(lu * NT + t, tiles - 1);
                ch.v[t] = a.codes[(tile * kc + lk) * 64 + lane];
                ch.s[t] = *(const SP*)(a.scales + ((tile * kc + lk) * 16 + r) * GPC);
            }
            if (++lk == kc) lk = 0, ++lu;
        }
    };
    constexpr int DEPTH = 4;
    Chunk ring[DEPTH];
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) load(ring[i]);

    // queries into LDS: a wave per query
    for (uint32_t q = wave; q < a.m; q += 4) {
        const uint64_t base = (uint64_t)q * a.L.dim;
        float mx = 0.0f;
        bool bad = false;
        for (uint32_t e = lane; e < a.L.dim; e += 64) {
            const float v = fabsf(load_query(a.queries, a.qdt, base + e));
            bad |= !(v < INFINITY);
            mx = fmaxf(mx, v);
        }
        for (int o = 32; o; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
        bad = __ballot(bad) != 0;
        const int ex = mx > 0.0f && !bad ? 14 - ilogbf(mx) : 0;
        if (lane == 0) expo[q] = -ex;
        for (uint32_t e = lane; e < kp; e += 64) {
            float v = e < a.L.dim ? ldexpf(load_query(a.queries, a.qdt, base + e), ex) : 0.0f;
            if (bad) v = NAN;
            _Float16* x = xs + ((uint64_t)(e / 32) * rows + q * PARTS) * 32 + e % 32;
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                const _Float16 h = (_Float16)v;
                x[p * 32] = h;
                v -= (float)h;
            }
        }
    }
    __syncthreads();

    // LDS row of this lane for each operand: row r is part r & 3 of query r >> 2 (three parts), or query r
    uint32_t xrow[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const uint32_t q = mt * QPT + (PARTS == 3 ? r >> 2 : r), p = PARTS == 3 ? min(r & 3u, 2u) : 0u;
        xrow[mt] = (min(q, a.m - 1) * PARTS + p) * 32 + c * 8;
    }
    f32x4 acc[NT][MT];
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    auto chunk = [&](const Chunk& ch, uint32_t k) {
        f32x4 d[NT][MT];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const bool starts = t % (4 / GPC) == 0, ends = t % (4 / GPC) == 4 / GPC - 1;
            f16x8 x[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) x[mt] = *(const f16x8*)(xs + (uint64_t)(k * 4 + t) * rows * 32 + xrow[mt]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const uint32_t w4 = t == 0 ? ch.v[nt].x : t == 1 ? ch.v[nt].y : t == 2 ? ch.v[nt].z : ch.v[nt].w;
                const f16x8 wv = unpack(w4);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) d[nt][mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[mt], wv, starts ? zero : d[nt][mt], 0, 0, 0);
                if (ends) {
                    const float s = half_to_f32<SDT>(piece_at(ch.s[nt], t / (4 / GPC)));
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[nt][mt][i] = fmaf(s, d[nt][mt][i], acc[nt][mt][i]);
                }
            }
        }
    };
    uint32_t k = 0;
    for (uint64_t u = u0; u < u1;) {
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) {
            if (u < u1) {
                if (k == 0) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) acc[nt][mt] = zero;
                }
                chunk(ring[i], k);
                load(ring[i]);
                if (++k == kc) {
                    k = 0;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const uint64_t row = (u * NT + nt) * 16 + r;
                        if (row < a.n) {
#pragma unroll
                            for (int mt = 0; mt < MT; ++mt) {
                                if (PARTS == 3) {
                                    const uint32_t q = mt * 4 + c;
                                    if (q < a.m) a.out[(uint64_t)q * a.n + row] = ldexpf(acc[nt][mt][2] + acc[nt][mt][1] + acc[nt][mt][0], expo[q]);
                                } else {
#pragma unroll
                                    for (int x = 0; x < 4; ++x) {
                                        const uint32_t q = mt * 16 + c * 4 + x;
                                        if (q < a.m) a.out[(uint64_t)q * a.n + row] = ldexpf(acc[nt][mt][x], expo[q]);
                                    }
                                }
                            }
                        }
                    }
                    ++u;
                }
            }
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

constexpr size_t LDS_MAX = 160 * 1024;

template <int PARTS, int SDT, int GPC, int MT, int NT>
int launch_scores(const cgv_q4_index* h, const ScoreArgs& a, hipStream_t s) {
    const size_t lds = (size_t)a.m * PARTS * h->L.kc * CHUNK * 2 + a.m * 4;
    const uint64_t units = ((h->n + 15) / 16 + NT - 1) / NT;
    const uint64_t per_cu = std::min<uint64_t>(4, LDS_MAX / lds);     // workgroups of four waves that a CU holds
    const unsigned blocks = (unsigned)std::min<uint64_t>((units + 3) / 4, 256 * per_cu);
    void (*kern)(ScoreArgs) = q4_scores_kernel<PARTS, SDT, GPC, MT, NT>;
    OPCHK(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)LDS_MAX));
    hipLaunchKernelGGL(kern, dim3(blocks), dim3(256), lds, s, a);
    OPCHK(hipGetLastError());
    return CGV_OK;
}

template <int PARTS, int SDT, int GPC>
int launch_by_queries(const cgv_q4_index* h, const ScoreArgs& a, hipStream_t s) {
    constexpr uint32_t QPT = PARTS == 3 ? 4 : 16;
    return a.m <= QPT ? launch_scores<PARTS, SDT, GPC, 1, 1>(h, a, s) : a.m <= 2 * QPT ? launch_scores<PARTS, SDT, GPC, 2, 2>(h, a, s)
                                                                                       : launch_scores<PARTS, SDT, GPC, 4, 2>(h, a, s);
}

template <int PARTS, int SDT>
int launch_by_group(const cgv_q4_index* h, const ScoreArgs& a, hipStream_t s) {
    return h->L.gpc == 1 ? launch_by_queries<PARTS, SDT, 1>(h, a, s) : h->L.gpc == 2 ? launch_by_queries<PARTS, SDT, 2>(h, a, s)
                                                                                     : launch_by_queries<PARTS, SDT, 4>(h, a, s);
}

int scores_on(const cgv_q4_index* h, const void* q, int qdt, uint32_t m, float* out, hipStream_t s) {
    const uint32_t parts = qdt == CGV_DTYPE_F32 ? 3 : 1;
    const size_t per_query = (size_t)parts * h->L.kc * CHUNK * 2 + 4;
    const uint32_t most = std::min<uint32_t>(parts == 3 ? 16 : 64, (uint32_t)(LDS_MAX / per_query));   // at least 3 (dim 8192, f32)
    for (uint32_t i = 0; i < m; i += most) {
        ScoreArgs a{(const uint4*)h->codes, h->scales, (const char*)q + (uint64_t)i * h->L.dim * esize(qdt), out + (uint64_t)i * h->n, h->n, h->L,
                    std::min(most, m - i), qdt};
        const bool f16 = h->sdt == CGV_DTYPE_FP16;
        const int rc = parts == 3 ? (f16 ? launch_by_group<3, cgv::DT_FP16>(h, a, s) : launch_by_group<3, cgv::DT_BF16>(h, a, s))
                                  : (f16 ? launch_by_group<1, cgv::DT_FP16>(h, a, s) : launch_by_group<1, cgv::DT_BF16>(h, a, s));
        if (rc) return rc;
    }
    return CGV_OK;
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
