// q4scan.hip - scores of a few queries against a corpus in 4 bits with group scales (include/cgvec_q4.h).
//
// Layout in HBM. 16 rows form a tile, 128 elements of them a chunk of 1 KiB; lane l = c * 16 + r of a wave owns 16 bytes of
// it: row r, and in dword t the eight elements t * 32 + c * 8 + 0..7. One 16-byte load per lane thus reads a whole chunk as
// one linear kilobyte, and dword t of the 64 lanes is a 16 x 32 piece of the tile whose 32 columns lie in ONE group.
// Inside a dword element 2p sits in nibble p and element 2p + 1 in nibble p + 4, so that one shift and one mask give the
// two elements of a pair in the two halves of a register.
// The scales of a tile's chunk are [16 rows][128 / group] behind each other.
#include <limits.h>

#include <mutex>
#include <type_traits>
#include <vector>

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

constexpr uint32_t BAD_NONFINITE = 1, BAD_RANGE = 2, HAS_LARGE = 4;
// below this no group's sum times its scale, nor the sum of a row's 256 groups, leaves f32's range on its way (codes times queries: 2^25 a group)
constexpr float LARGE_SCALE = 0x1p94f;

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
    bool large = false;
    for (uint32_t k = 0; k < L.kc; ++k) {
        const uint32_t e = k * CHUNK + lane * 2;
        const float v0 = e < L.dim ? x[e] : 0.0f, v1 = e + 1 < L.dim ? x[e + 1] : 0.0f;
        if (!(fabsf(v0) < INFINITY) || !(fabsf(v1) < INFINITY)) atomicOr(bad, BAD_NONFINITE);
        float a = fmaxf(fabsf(v0), fabsf(v1));
        for (uint32_t o = 1; o < L.group / 2; o <<= 1) a = fmaxf(a, __shfl_xor(a, (int)o));
        const uint16_t sb = f32_to_half<SDT>(a / 7.0f);
        const float s = half_to_f32<SDT>(sb);
        if (!(s < INFINITY)) atomicOr(bad, BAD_RANGE);
        large |= s >= LARGE_SCALE;
        const uint32_t g = e / L.group;
        if (lane % (L.group / 2) == 0) scales[L.scale(row0 + i, g)] = g < L.ng ? sb : (uint16_t)0;
        const int q0 = s > 0.0f ? (int)fminf(fmaxf(rintf(v0 / s), -8.0f), 7.0f) : 0;
        const int q1 = s > 0.0f ? (int)fminf(fmaxf(rintf(v1 / s), -8.0f), 7.0f) : 0;
        uint32_t w = pair_bits((uint32_t)(q0 + 8), (uint32_t)(q1 + 8), lane & 3);
        w |= __shfl_xor(w, 1);
        w |= __shfl_xor(w, 2);
        if ((lane & 3) == 0) codes[L.dword(row0 + i, e)] = w;
    }
    if (__any(large) && lane == 0) atomicOr(bad, HAS_LARGE);
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
    bool large = false;
    for (uint32_t g = lane; g < L.kc * L.gpc; g += 64) {
        const uint16_t s = g < L.ng ? src_scales[i * L.ng + g] : (uint16_t)0;
        const float v = fabsf(half_to_f32<SDT>(s));
        if (!(v < INFINITY)) atomicOr(bad, BAD_NONFINITE);
        large |= v >= LARGE_SCALE;
        scales[L.scale(row0 + i, g)] = s;
    }
    if (__any(large) && lane == 0) atomicOr(bad, HAS_LARGE);
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
// A matrix instruction takes 32 columns of a 16-row tile (B operand: a lane holds 8 codes of one row) against 16 rows of query
// data (A operand); rows of the result depend on nothing but their own row of A, so rows that a few queries leave unused cost
// nothing and hold anything.
//   f32 queries: fixed point. A query is scaled by a power of two to integers below 2^38 in magnitude (an element keeps 24
//     bits, or an absolute 2^-39 of the query's largest) and split into five signed bytes; v_mfma_i32_16x16x32_i8 adds byte x code
//     exactly. A code's byte is 16 (c - 8): two masks and a shift make eight of them. Three queries of five rows an operand.
//   16-bit queries: one f16 row per query (scaled to 2^14 .. 2^15, so that bf16's range fits), 16 queries an operand;
//     codes become f16 integers -8..7 by 0x6400 | c = 1024 + c and one packed multiply-add; v_mfma_f32_16x16x32_f16.
// A group's sum is multiplied by its scale - one value per lane, its row's - and added up in f32.
//
// Bound by the codes' way from HBM, if the vector instructions per KiB stay below its time: a CU's share of 6 TB/s is a KiB per
// 105 cycles, its four SIMDs spend 4 cycles on a vector instruction: 105 of them per KiB and SIMD is the limit. The same sums
// with codes turned to f32 and fmaf (8 + 8 instructions for 8 codes) ran at 3.5 TB/s. One f32 query over 1M x 768 in groups of 64: 68.5 us,
// 6.0 TB/s of codes and scales; 16 bf16 queries over 300 k x 1536 in groups of 128: 51 us and 5 us for the queries' image, 5.0 TB/s.
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct ScoreArgs {
    const u32x4* codes;
    const uint16_t* scales;
    const void* queries;
    float* out;
    uint64_t n;
    Layout L;
    uint32_t m;            // queries of this launch
    int qdt;
    const char* image;     // the queries as the kernel wants them in LDS, or NULL: every workgroup makes them itself
};

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

__device__ inline float load_query(const void* q, int dt, uint64_t i) {
    return dt == CGV_DTYPE_F32 ? load_elem<cgv::DT_F32>(q, i) : dt == CGV_DTYPE_BF16 ? load_elem<cgv::DT_BF16>(q, i) : load_elem<cgv::DT_FP16>(q, i);
}

// f32 queries
struct Fixed {
    static constexpr uint32_t QPT = 3, ROWS = 5;      // queries of an operand, LDS rows of a query (byte 0 is the lowest)
    static constexpr uint32_t ROW_BYTES = 32;         // of 32 columns
    typedef i32x4 Acc;
    typedef long Frag;
    static __device__ Frag weights(uint32_t w) {
        const uint32_t lo = ((w << 4) & 0xf0f0f0f0u) ^ 0x80808080u, hi = (w & 0xf0f0f0f0u) ^ 0x80808080u;   // nibbles 0 2 4 6, 1 3 5 7
        return (long)((uint64_t)hi << 32 | lo);
    }
    static __device__ Acc mma(Frag x, Frag w, Acc c) { return __builtin_amdgcn_mfma_i32_16x16x32_i8(x, w, c, 0, 0, 0); }
    // operand row r: rows 4 q .. 4 q + 3 are bytes 1 .. 4 of query q, row 12 + q is its byte 0
    static __device__ uint32_t query_of(uint32_t r) { return r < 12 ? r >> 2 : min(r - 12, 2u); }
    static __device__ uint32_t part_of(uint32_t r) { return r < 12 ? (r & 3) + 1 : 0u; }
    static __device__ int unit(float mx) { return mx > 0.0f ? 37 - ilogbf(mx) : 0; }
    static constexpr int SCORE_SHIFT = -4;             // the codes are 16 times too large
    static __device__ void stage(char* xs, uint32_t rows, uint32_t q, uint32_t e, float v) {
        // v is below 2^38: its bits from 2^16 up and its rest are exact integers of 23 and 17 bits
        const float t = rintf(v * 0x1p-16f);
        int low = (int)rintf(v - t * 65536.0f), top = (int)t;
        int d[5];
        d[0] = (signed char)(low & 255);
        low = (low - d[0]) >> 8;
        d[1] = (signed char)(low & 255);
        top += (low - d[1]) >> 8;
#pragma unroll
        for (int p = 2; p < 5; ++p) {
            d[p] = (signed char)(top & 255);
            top = (top - d[p]) >> 8;
        }
        // element 2 p lies in nibble p, 2 p + 1 in nibble p + 4: their bytes come out in the order 0 4 1 5 2 6 3 7
        char* x = xs + ((e / 32) * rows + q * ROWS) * ROW_BYTES + (e % 32 & ~7u) + ((0x75316420u >> (4 * (e & 7u))) & 7u);
#pragma unroll
        for (int p = 0; p < 5; ++p) x[p * ROW_BYTES] = (char)d[p];
    }
    template <int MT>
    static __device__ void store(const ScoreArgs& a, const f32x4 (&acc)[MT], uint64_t row, uint32_t lane, const int* expo) {
        const uint32_t r = lane & 15, c = lane >> 4;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const float e0 = __shfl(acc[mt][0], 48 + r), e1 = __shfl(acc[mt][1], 48 + r), e2 = __shfl(acc[mt][2], 48 + r);
            const float low = c == 0 ? e0 : c == 1 ? e1 : e2;
            const float v = fmaf(fmaf(fmaf(fmaf(low, 0x1p-8f, acc[mt][0]), 0x1p-8f, acc[mt][1]), 0x1p-8f, acc[mt][2]), 0x1p-8f, acc[mt][3]);
            const uint32_t q = mt * 3 + c;
            if (c < 3 && q < a.m && row < a.n) a.out[(uint64_t)q * a.n + row] = expo[q] == INT_MIN ? NAN : ldexpf(v, expo[q] + 32);
        }
    }
};

// bf16 and fp16 queries
struct Half {
    static constexpr uint32_t QPT = 16, ROWS = 1, ROW_BYTES = 64;
    typedef f32x4 Acc;
    typedef f16x8 Frag;
    static __device__ Frag weights(uint32_t w) {
        // 1024 + c from the low four bits of a half, 1024 + 16 c from the next four
        const f16x2 one = {(_Float16)1.0f, (_Float16)1.0f}, m1032 = {(_Float16)-1032.0f, (_Float16)-1032.0f};
        const f16x2 x16 = {(_Float16)0.0625f, (_Float16)0.0625f}, m72 = {(_Float16)-72.0f, (_Float16)-72.0f};
        const uint32_t w8 = w >> 8;
        f16x2 p[4];
        p[0] = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (w & 0x000f000fu) | 0x64006400u), one, m1032);
        p[1] = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (w & 0x00f000f0u) | 0x64006400u), x16, m72);
        p[2] = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (w8 & 0x000f000fu) | 0x64006400u), one, m1032);
        p[3] = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (w8 & 0x00f000f0u) | 0x64006400u), x16, m72);
        Frag v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[2 * i] = p[i][0], v[2 * i + 1] = p[i][1];
        return v;
    }
    static __device__ Acc mma(Frag x, Frag w, Acc c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, w, c, 0, 0, 0); }
    static __device__ uint32_t query_of(uint32_t r) { return r; }
    static __device__ uint32_t part_of(uint32_t) { return 0; }
    static __device__ int unit(float mx) { return mx > 0.0f ? 14 - ilogbf(mx) : 0; }
    static constexpr int SCORE_SHIFT = 0;
    static __device__ void stage(char* xs, uint32_t rows, uint32_t q, uint32_t e, float v) {
        ((_Float16*)(xs + ((e / 32) * rows + q) * ROW_BYTES))[e % 32] = (_Float16)v;
    }
    template <int MT>
    static __device__ void store(const ScoreArgs& a, const f32x4 (&acc)[MT], uint64_t row, uint32_t lane, const int* expo) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const uint32_t q = mt * 16 + (lane >> 4) * 4 + x;
                if (q < a.m && row < a.n) a.out[(uint64_t)q * a.n + row] = expo[q] == INT_MIN ? NAN : ldexpf(acc[mt][x], expo[q]);
            }
    }
};

// all queries into their places in LDS, by a workgroup: largest magnitudes first (as bits: NaN
// and Inf win), then the parts. A thread has four elements on their way at a time
template <class P, uint32_t THREADS>
__device__ inline void stage_queries(const ScoreArgs& a, char* xs, uint32_t rows, int* expo, uint32_t* top) {
    const uint32_t kp = a.L.kc * CHUNK, total = a.m * kp;
    for (uint32_t q = threadIdx.x; q < a.m; q += THREADS) top[q] = 0;
    __syncthreads();
    constexpr uint32_t BATCH = 4;
    for (int pass = 0; pass < 2; ++pass) {
        for (uint32_t i0 = 0; i0 < total; i0 += THREADS * BATCH) {
            float v[BATCH];
#pragma unroll
            for (uint32_t j = 0; j < BATCH; ++j) {
                const uint32_t i = i0 + j * THREADS + threadIdx.x, q = i / kp, e = i - q * kp;
                v[j] = i < total && e < a.L.dim ? load_query(a.queries, a.qdt, (uint64_t)q * a.L.dim + e) : 0.0f;
            }
#pragma unroll
            for (uint32_t j = 0; j < BATCH; ++j) {
                const uint32_t i = i0 + j * THREADS + threadIdx.x, q = i / kp, e = i - q * kp;   // kp: a multiple of 128, a wave has one query
                if (i >= total) continue;
                if (pass == 0) {
                    uint32_t bits = __float_as_uint(fabsf(v[j]));
                    for (int o = 32; o; o >>= 1) bits = max(bits, (uint32_t)__shfl_xor((int)bits, o));
                    if ((threadIdx.x & 63) == 0) atomicMax(&top[q], bits);
                } else {
                    const uint32_t t = top[q];
                    const bool bad = t >= 0x7f800000u;
                    const int ex = bad ? 0 : P::unit(__uint_as_float(t));
                    P::stage(xs, rows, q, e, bad ? 0.0f : ldexpf(v[j], ex));
                    if (e == 0) expo[q] = bad ? INT_MIN : P::SCORE_SHIFT - ex;
                }
            }
        }
        __syncthreads();
    }
}

// a workgroup per query: the image of what the kernel below wants in LDS. A query stays in registers between the two steps
template <class P>
__global__ __launch_bounds__(1024) void q4_image_kernel(ScoreArgs a, char* image) {
    __shared__ uint32_t tops[16];
    const uint32_t rows = a.m * P::ROWS, kp = a.L.kc * CHUNK, q = blockIdx.x;
    float v[8];                                        // dim is at most 8192
    uint32_t bits = 0;
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
        const uint32_t e = j * 1024 + threadIdx.x;
        v[j] = e < a.L.dim ? load_query(a.queries, a.qdt, (uint64_t)q * a.L.dim + e) : 0.0f;
        bits = max(bits, __float_as_uint(fabsf(v[j])));
    }
    for (int o = 32; o; o >>= 1) bits = max(bits, (uint32_t)__shfl_xor((int)bits, o));
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = bits;
    __syncthreads();
    for (int x = 0; x < 16; ++x) bits = max(bits, tops[x]);
    const bool bad = bits >= 0x7f800000u;
    const int ex = bad ? 0 : P::unit(__uint_as_float(bits));
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
        const uint32_t e = j * 1024 + threadIdx.x;
        if (e < kp) P::stage(image, rows, q, e, bad ? 0.0f : ldexpf(v[j], ex));
    }
    if (threadIdx.x == 0) ((int*)(image + (uint64_t)(kp / 32) * rows * P::ROW_BYTES))[q] = bad ? INT_MIN : P::SCORE_SHIFT - ex;
}

// MT operands of queries, NT tiles at a time
template <class P, int SDT, int GPC, int MT, int NT, bool ONCE, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void q4_scores_kernel(ScoreArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    typedef typename ScalePiece<GPC>::type SP;
    const uint32_t lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4, wave = threadIdx.x >> 6;
    const uint32_t kc = a.L.kc, rows = a.m * P::ROWS, kp = kc * CHUNK;
    char* xs = smem;                                   // [kp / 32][rows][32 columns]
    int* expo = (int*)(smem + (uint64_t)(kp / 32) * rows * P::ROW_BYTES);

    // this wave takes every `waves`-th unit of tiles (all waves together read one stretch of the corpus at a time); its first
    // chunks are on their way before anything else
    const uint64_t tiles = (a.n + 15) / 16, units = (tiles + NT - 1) / NT;
    const uint64_t waves = (uint64_t)gridDim.x * WAVES, w = (uint64_t)wave * gridDim.x + blockIdx.x;
    struct Chunk {
        u32x4 v[NT];
        SP s[NT];
    };
    uint64_t lu = w;           // the load side's unit and chunk
    uint32_t lk = 0;
    auto load = [&](Chunk& ch) {
        if (lu < units) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const uint64_t tile = min(lu * NT + t, tiles - 1);
                const u32x4* src = &a.codes[(tile * kc + lk) * 64 + lane];
                ch.v[t] = ONCE ? __builtin_nontemporal_load(src) : *src;
                ch.s[t] = *(const SP*)(a.scales + ((tile * kc + lk) * 16 + r) * GPC);
            }
            if (++lk == kc) lk = 0, lu += waves;
        }
    };
    constexpr int DEPTH = 4;
    Chunk ring[DEPTH];
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) load(ring[i]);

    if (a.image) {
        const uint4* src = (const uint4*)a.image;
        const uint32_t pieces = (kp / 32) * rows * P::ROW_BYTES / 16;
        for (uint32_t i = threadIdx.x; i < pieces; i += 64 * WAVES) ((uint4*)xs)[i] = src[i];
        for (uint32_t i = threadIdx.x; i < a.m; i += 64 * WAVES) expo[i] = ((const int*)(src + pieces))[i];
    } else {
        stage_queries<P, 64 * WAVES>(a, xs, rows, expo, (uint32_t*)expo + a.m);
    }
    __syncthreads();

    uint32_t xrow[MT];                                 // this lane's piece of each operand, in bytes from a step's first row
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
        xrow[mt] = (min(mt * P::QPT + P::query_of(r), a.m - 1) * P::ROWS + P::part_of(r)) * P::ROW_BYTES + c * (P::ROW_BYTES / 4);
    f32x4 acc[NT][MT];
    const f32x4 fzero = {0.0f, 0.0f, 0.0f, 0.0f};
    const typename P::Acc zero = {0, 0, 0, 0};
    auto chunk = [&](const Chunk& ch, uint32_t k) {
        typename P::Acc d[NT][MT];
        const char* xk = xs + k * 4 * rows * P::ROW_BYTES;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const bool starts = t % (4 / GPC) == 0, ends = t % (4 / GPC) == 4 / GPC - 1;
            typename P::Frag x[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) x[mt] = *(const typename P::Frag*)(xk + t * rows * P::ROW_BYTES + xrow[mt]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const typename P::Frag wv = P::weights(ch.v[nt][t]);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) d[nt][mt] = P::mma(x[mt], wv, starts ? zero : d[nt][mt]);
                if (ends) {
                    const float s = half_to_f32<SDT>(piece_at(ch.s[nt], t / (4 / GPC)));
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[nt][mt][i] = fmaf(s, (float)d[nt][mt][i], acc[nt][mt][i]);
                }
            }
        }
    };
    uint32_t k = 0;
    for (uint64_t u = w; u < units;) {
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) {
            if (u < units) {
                if (k == 0) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) acc[nt][mt] = fzero;
                }
                chunk(ring[i], k);
                load(ring[i]);
                if (++k == kc) {
                    k = 0;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) P::template store<MT>(a, acc[nt], (u * NT + nt) * 16 + r, lane, expo);
                    u += waves;
                }
            }
        }
    }
}

// Rows with scales of 2^94 and more (bf16): group sums are formed at the size that the queries have on the matrix cores, and can leave f32's
// range where the score itself does not. Such results are Inf or NaN; a thread each computes them again in 64 bits. A launch of its own, and
// only for an index that has such rows: nothing else pays for it
__global__ __launch_bounds__(256) void q4_again_kernel(ScoreArgs a) {
    const uint64_t t = wide_block() * 256 + threadIdx.x;
    if (t >= a.m * a.n || fabsf(a.out[t]) < INFINITY) return;
    const uint64_t q = t / a.n, row = t - q * a.n;
    double sum = 0.0;
    bool bad = false;
    for (uint32_t e = 0; e < a.L.dim; e += 8) {
        const uint32_t w = ((const uint32_t*)a.codes)[a.L.dword(row, e)];
        double part = 0.0;
        for (uint32_t j = 0; j < 8 && e + j < a.L.dim; ++j) {
            const float x = load_query(a.queries, a.qdt, q * a.L.dim + e + j);
            bad |= !(fabsf(x) < INFINITY);
            part = fma((double)x, (double)((int)((w >> (4 * (j >> 1) + 16 * (j & 1u))) & 15u) - 8), part);
        }
        sum = fma((double)half_to_f32<cgv::DT_BF16>(a.scales[a.L.scale(row, e / a.L.group)]), part, sum);
    }
    a.out[t] = bad ? NAN : (float)sum;
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
    bool large = false;             // rows with scales of LARGE_SCALE or more (bf16)
    bool captured = false;          // a graph may hold the addresses of codes and scales
    std::vector<void*> retired;     // such buffers that a larger corpus has left: kept for the graph's replays
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
    if (h->captured) h->retired.reserve(h->retired.size() + 2);
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
    for (void* p : {(void*)h->codes, (void*)h->scales}) {
        if (p && h->captured) h->retired.push_back(p);      // room for both was made beforehand
        else if (p) (void)hipFree(p);
    }
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
    h->large |= (bad & HAS_LARGE) != 0;
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

template <class P>
size_t query_bytes(const cgv_q4_index* h) { return (size_t)(h->L.kc * CHUNK / 32) * P::ROWS * P::ROW_BYTES + 8; }

template <class P, int SDT, int GPC, int MT, int NT, bool ONCE = false>
int launch_scores(const cgv_q4_index* h, const ScoreArgs& a, hipStream_t s) {
    constexpr int WAVES = 8;
    const size_t lds = a.m * query_bytes<P>(h);
    const uint64_t units = ((a.n + 15) / 16 + NT - 1) / NT;
    const uint64_t per_cu = std::min<uint64_t>(2, LDS_MAX / lds);     // workgroups of a CU
    const unsigned blocks = (unsigned)std::min<uint64_t>((units + WAVES - 1) / WAVES, 256 * per_cu);
    void (*kern)(ScoreArgs) = q4_scores_kernel<P, SDT, GPC, MT, NT, ONCE, WAVES>;
    static LdsLimit limit;
    OPCHK(limit.raise((const void*)kern, h->device, (int)LDS_MAX));
    hipLaunchKernelGGL(kern, dim3(blocks), dim3(64 * WAVES), lds, s, a);
    OPCHK(hipGetLastError());
    return CGV_OK;
}

template <class P, int SDT, int GPC>
int launch_by_queries(const cgv_q4_index* h, const ScoreArgs& a, hipStream_t s) {
    // one operand of queries: two tiles at a time where every wave gets two such pairs, so that there is always one to work on
    // (one query, 1M x 768: 87 -> 70 us), single tiles below, where the number of waves counts (10 k x 384: 6.0 -> 5.1 us)
    // Codes that the 256 MiB last-level cache cannot hold until the next call are read past it (1M x 768: 78 -> 69 us), smaller ones
    // stay there (250 k x 768, the same corpus again: 25 -> 21 us)
    if (a.m <= P::QPT) {
        if (a.n < 16ull * 4 * 4096) return launch_scores<P, SDT, GPC, 1, 1>(h, a, s);
        return h->L.tile_codes((a.n + 15) / 16) > (256ull << 20) ? launch_scores<P, SDT, GPC, 1, 2, true>(h, a, s)
                                                                   : launch_scores<P, SDT, GPC, 1, 2>(h, a, s);
    }
    return a.m <= 2 * P::QPT ? launch_scores<P, SDT, GPC, 2, 2>(h, a, s)
                                                                                         : launch_scores<P, SDT, GPC, 4, 2>(h, a, s);
}

template <class P, int SDT>
int launch_by_group(const cgv_q4_index* h, const ScoreArgs& a, hipStream_t s) {
    return h->L.gpc == 1 ? launch_by_queries<P, SDT, 1>(h, a, s) : h->L.gpc == 2 ? launch_by_queries<P, SDT, 2>(h, a, s)
                                                                                 : launch_by_queries<P, SDT, 4>(h, a, s);
}

template <class P>
uint32_t queries_per_launch(const cgv_q4_index* h) { return std::min<uint32_t>(4 * P::QPT, (uint32_t)(LDS_MAX / query_bytes<P>(h))); }   // 3 at least

// one workgroup's way through 8192 elements is about 4 us, hidden behind the first codes; a launch more costs as much
constexpr uint32_t STAGE_IN_PLACE = 8192;

template <class P>
size_t image_bytes(const cgv_q4_index* h, uint32_t m) {
    const uint32_t most = std::min(m, queries_per_launch<P>(h));
    return (uint64_t)most * h->L.kc * CHUNK <= STAGE_IN_PLACE ? 0 : most * query_bytes<P>(h);
}

template <class P>
int scores_by(const cgv_q4_index* h, const void* q, int qdt, uint32_t m, uint64_t n, float* out, char* ws, hipStream_t s) {
    const uint32_t most = queries_per_launch<P>(h);
    for (uint32_t i = 0; i < m; i += most) {
        ScoreArgs a{(const u32x4*)h->codes, h->scales, (const char*)q + (uint64_t)i * h->L.dim * esize(qdt), out + (uint64_t)i * n, n, h->L,
                    std::min(most, m - i), qdt, nullptr};
        if ((uint64_t)a.m * h->L.kc * CHUNK > STAGE_IN_PLACE) {
            hipLaunchKernelGGL((q4_image_kernel<P>), dim3(a.m), dim3(1024), 0, s, a, ws);
            OPCHK(hipGetLastError());
            a.image = ws;
        }
        const int rc = h->sdt == CGV_DTYPE_FP16 ? launch_by_group<P, cgv::DT_FP16>(h, a, s) : launch_by_group<P, cgv::DT_BF16>(h, a, s);
        if (rc) return rc;
        if (h->large) {
            hipLaunchKernelGGL(q4_again_kernel, wide_grid((a.m * a.n + 255) / 256), dim3(256), 0, s, a);
            OPCHK(hipGetLastError());
        }
    }
    return CGV_OK;
}

size_t scores_workspace(const cgv_q4_index* h, int qdt, uint32_t m) {
    return qdt == CGV_DTYPE_F32 ? image_bytes<Fixed>(h, m) : image_bytes<Half>(h, m);
}

int scores_on(const cgv_q4_index* h, const void* q, int qdt, uint32_t m, uint64_t n, float* out, char* ws, hipStream_t s) {
    return qdt == CGV_DTYPE_F32 ? scores_by<Fixed>(h, q, qdt, m, n, out, ws, s) : scores_by<Half>(h, q, qdt, m, n, out, ws, s);
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
    for (void* p : h->retired) (void)hipFree(p);
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

int cgv_q4_scores_f32(cgv_q4_index* h, const float* queries_host, uint32_t m, uint64_t n_rows, float* out_host) {
    return guarded([&]() -> int {
        if (!h) return fail(CGV_ERR_INVALID_ARG, "handle is NULL");
        std::lock_guard<std::mutex> lk(h->mu);
        if (n_rows > h->n) return fail(CGV_ERR_OUT_OF_RANGE, "n_rows is beyond the last row");
        if (m == 0 || n_rows == 0) return CGV_OK;
        if (!queries_host || !out_host) return fail(CGV_ERR_INVALID_ARG, "NULL argument");
        DeviceScope dev(h->device);
        OPCHK(dev.enter());
        // queries in pieces whose scores fit the staging buffer
        const uint64_t per = std::max<uint64_t>(1, std::min<uint64_t>(m, (512ull << 20) / (n_rows * 4)));
        const size_t qb = ((size_t)per * h->L.dim * 4 + 255) / 256 * 256, sb = (per * n_rows * 4 + 255) / 256 * 256;
        int rc = ensure_stage(h, qb + sb + scores_workspace(h, CGV_DTYPE_F32, (uint32_t)per));
        if (rc) return rc;
        float* dq = (float*)h->stage;
        float* ds = (float*)((char*)h->stage + qb);
        for (uint64_t a = 0; a < m; a += per) {
            const uint32_t c = (uint32_t)std::min<uint64_t>(per, m - a);
            OPCHK(hipMemcpyAsync(dq, queries_host + a * h->L.dim, (size_t)c * h->L.dim * 4, hipMemcpyHostToDevice, h->stream));
            if ((rc = scores_on(h, dq, CGV_DTYPE_F32, c, n_rows, ds, (char*)h->stage + qb + sb, h->stream))) return rc;
            OPCHK(hipMemcpyAsync(out_host + a * n_rows, ds, (size_t)c * n_rows * 4, hipMemcpyDeviceToHost, h->stream));
            OPCHK(hipStreamSynchronize(h->stream));
        }
        return CGV_OK;
    });
}

size_t cgv_q4_scores_workspace(const cgv_q4_index* h, int query_dtype, uint32_t m) { return h && m ? scores_workspace(h, query_dtype, m) : 0; }

int cgv_q4_scores_dev(cgv_q4_index* h, const void* queries_dev, int query_dtype, uint32_t m, uint64_t n_rows, float* out_dev, void* workspace_dev,
                      size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        if (!h) return fail(CGV_ERR_INVALID_ARG, "handle is NULL");
        if (query_dtype != CGV_DTYPE_F32 && query_dtype != CGV_DTYPE_BF16 && query_dtype != CGV_DTYPE_FP16)
            return fail(CGV_ERR_INVALID_ARG, "dtype must be f32, bf16 or fp16");
        std::lock_guard<std::mutex> lk(h->mu);
        if (n_rows > h->n) return fail(CGV_ERR_OUT_OF_RANGE, "n_rows is beyond the last row");
        if (m == 0 || n_rows == 0) return CGV_OK;
        if (!queries_dev || !out_dev) return fail(CGV_ERR_INVALID_ARG, "NULL argument");
        const size_t need = scores_workspace(h, query_dtype, m);
        if (workspace_bytes < need || (need && !workspace_dev)) return fail(CGV_ERR_INVALID_ARG, "the workspace is smaller than cgv_q4_scores_workspace says");
        if (need && (uintptr_t)workspace_dev % 256) return fail(CGV_ERR_INVALID_ARG, "the workspace must be aligned to 256 bytes");
        DeviceScope dev(h->device);
        OPCHK(dev.enter());
        if (!h->captured) {
            hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
            OPCHK(hipStreamIsCapturing((hipStream_t)stream, &st));
            h->captured = st != hipStreamCaptureStatusNone;
        }
        return scores_on(h, queries_dev, query_dtype, m, n_rows, out_dev, (char*)workspace_dev, (hipStream_t)stream);
    });
}

}  // extern "C"
