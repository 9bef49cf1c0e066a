// softmax.hip - softmax losses of queries against all rows of a corpus and their gradients (include/cgvec_train.h).
//
// forward   queries into a padded copy, scores of the listed rows; scores of the whole corpus tile by tile, keeping a maximum and a
//           sum of exp per query; loss.
// backward  per piece of the corpus: G = c (exp(s - lse) - p) in 16 bits (three planes for f32), dQ += G R in f32 partial sums,
//           dR = G^T Q; then dQ's partial sums are added and rounded.
// Four products of 2 b n dim operations (the scores twice: keeping them would be the matrix that is not to be stored). 1024 queries x
// 1M x 768 bf16, loss and both gradients: 5.90 ms = 1.07 PFLOP/s; 256 x 1M x 1536 fp16, loss alone: 0.79 ms = 1.0 PFLOP/s, 3.9 TB/s.
//
// Two things keep a small loss and a small gradient exact where exp(s - lse) is close to 1. The heaviest listed row (the anchor) is
// left out of the sum over the corpus: tail = lse - s_anchor = log(1 + sum of the others' exp(s - s_anchor)) then comes from log1p
// and not from the difference of two large numbers, and the anchor's 1 - exp(s - lse) is -expm1(-tail). And the listed rows' entries
// of G, softmax minus weight, are computed in f32 from the saved scores and put into G as differences, before any rounding.
//
// For 16-bit inputs G is rounded to their type, which is what the matrix cores multiply their rows with. Over many entries these roundings
// average out; the listed entries', the largest and often alone in their rows, are made good in dQ and dR. Up to
// TWINS queries leave half of a tile's columns empty: there what the rounding leaves of G is stored and multiplied too (3 queries x 326 x
// 123 bf16: 0.0029 without, 0.0018 with).
// fp16: each query's entries of G are scaled by a power of two of its own, which brings its largest to 2^13 .. 2^14 (what is 2^-27 of that still has
// all its digits); dQ is scaled back in f32. Factors of other queries do not matter then (60 queries x 300 k x 64, factors 1 and 10^-6: dQ of the
// latter is off by 0.00026 of its norm, with one power for all by 1.9). dR sums over queries: it takes them from a copy that is scaled the
// other way round, so that all products carry the same power, the largest that keeps every query in range.
#include <float.h>
#include <limits.h>

#include <type_traits>

#include "../../include/cgvec_train.h"
#include "kernels_gemm.h"
#include "ops_common.h"
#include "sort_ids.h"

using namespace cgv_ops;
using namespace cgv_gemm;

namespace {

constexpr double LOG2E = 1.4426950408889634, LN2 = 0.6931471805599453;
constexpr uint32_t MAX_K = 256, NONE = 0xffffffffu, TWINS = 32;
// The listed entries are the largest of a row of the corpus' gradient, and often alone in it: what 16 bits leave of them is added there too
// (1024 queries x 125 k x 768 bf16, lists of ten: 0.0023 of the norm off without, 0.0017 with, which is the result's own rounding). Up to
// this many of them, all queries together, every small tile looks through; in large problems they are sorted by groups of rows, up to seven small
// launches, and make up one more product of their tiles. That takes a twentieth of the time or less from so many products of elements on and
// with lists so short beside the corpus; elsewhere the entries' rounding stays (0.0023 as well). 1024 x 65 536 x 768, half as many products, and
// lists of 16: loss and gradients 464 us without, 511 with; lists of 64, one row in 1024: 529 and 601, of 256: 781 and 967; 600 x 4000 x 256
// and lists of two: 60 and 84
constexpr uint32_t LOOKED_THROUGH = 1024, LISTED_ONE_IN = 1024, GROUP_BITS = 5;
constexpr double SORTED_FROM = 0x1p36;
constexpr uint32_t CUS = 256;                                  // workgroups of one per CU that fill the card
// of G, and of copied corpus rows. Each piece costs a round over dQ's partial sums (1024 x 500 k x 768, gradient: 3.05 ms with 128 MiB, 2.99 with
// 512, 2.97 with 1024); the corpus' gradient needs some 256 tiles a piece, however many queries there are
constexpr uint64_t PIECE_BYTES = 512ull << 20, PIECE_ROWS = 16384;
constexpr uint64_t CACHE = 256ull << 20;                       // the last-level cache

// ---- weights of a query's list (WEIGHTS; else only its ids and the anchor): one wave, entry j at lane j % 64, slot j / 64 -----
struct List {
    uint32_t id[4];       // NONE: weight 0
    double logp[4], p[4];
    uint32_t anchor;      // index of the first heaviest entry
    bool has;
};
__device__ inline float wave_max(float v) {
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
template <class T>
__device__ inline T wave_sum(T v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
template <bool WEIGHTS = true>
__device__ inline List read_list(const int64_t* ids, const float* ts, uint64_t i, uint32_t k, uint64_t n_rows, float tscale, int lane) {
    List l;
    float raw[4], mx = -INFINITY;
    bool any = false;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const uint32_t j = s * 64 + lane;
        l.id[s] = NONE;
        raw[s] = -INFINITY;
        if (j < k) {
            const int64_t id = ids[i * k + j];
            const float v = ts ? ts[i * k + j] : 0.0f;
            if (id >= 0 && (uint64_t)id < n_rows && v != -INFINITY) {
                l.id[s] = (uint32_t)id;
                raw[s] = v;
                any = true;
            }
        }
        // a negative factor turns the order round; the list's weights are few: 64 bits
        mx = fmaxf(mx, l.id[s] == NONE ? -INFINITY : tscale < 0.0f ? -raw[s] : raw[s]);
    }
    l.has = __ballot(any) != 0;
    mx = wave_max(mx);
    const double top = tscale < 0.0f ? -(double)mx : (double)mx;
    double z = 0.0;
    uint32_t first = NONE;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        if (WEIGHTS) {
            l.logp[s] = l.id[s] == NONE ? 0.0 : (raw[s] - top) * (double)(ts ? tscale : 0.0f);
            l.p[s] = l.id[s] == NONE ? 0.0 : exp(l.logp[s]);
            z += l.p[s];
        }
        const uint64_t eq = __ballot(l.id[s] != NONE && (double)raw[s] == top);
        if (first == NONE && eq) first = s * 64 + __ffsll((unsigned long long)eq) - 1;
    }
    if (first == NONE)
        for (int s = 0; s < 4; ++s) {       // only NaN scores: any listed row will do, the loss is NaN
            const uint64_t some = __ballot(l.id[s] != NONE);
            if (first == NONE && some) first = s * 64 + __ffsll((unsigned long long)some) - 1;
        }
    l.anchor = first;
    if (!WEIGHTS) return l;
    z = wave_sum(z);
    const double lz = log(z);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        if (l.id[s] != NONE) {
            l.p[s] /= z;
            l.logp[s] -= lz;
            if (l.p[s] == 0.0) l.id[s] = NONE;      // underflow: no weight, and no 0 * inf below
        }
    }
    return l;
}
template <class T>
__device__ inline T pick(const T (&v)[4], uint32_t j) {     // entry j of the list, for every lane
    const T x = j < 64 ? v[0] : j < 128 ? v[1] : j < 192 ? v[2] : v[3];
    return __shfl(x, (int)(j & 63u));
}

// a row of the padded copy: 16-bit types as they are, f32 as three planes; zeros beyond dim, and altogether if !src. fp16: the largest finite
// magnitude that the thread has seen
template <int DT>
__device__ inline float copy_row(const void* src, uint64_t at, uint32_t dim, uint32_t dp, uint16_t* dst, uint64_t plane, uint32_t t0, uint32_t step) {
    float most = 0.0f;
    for (uint32_t e = t0; e < dp; e += step) {
        if (DT == cgv::DT_F32) {
            uint16_t p[3] = {0, 0, 0};
            if (src && e < dim) split3(((const float*)src)[at + e], p);
            for (int x = 0; x < 3; ++x) dst[x * plane + e] = p[x];
        } else {
            const uint16_t v = src && e < dim ? ((const uint16_t*)src)[at + e] : (uint16_t)0;
            dst[e] = v;
            const float a = DT == cgv::DT_FP16 ? fabsf(half_to_f32<DT>(v)) : 0.0f;
            if (a < INFINITY) most = fmaxf(most, a);
        }
    }
    return most;
}

struct Piece {              // corpus rows [n0, n0 + c) on their way into the padded copy
    const void* rows;
    uint64_t stride, n0, plane;
    uint16_t* dst;
    uint32_t c, dim, dp;
};
// a workgroup of 256 threads, each with eight elements of a row
template <int DT>
__device__ inline void copy_piece_block(const Piece& P, uint64_t block) {
    const void* rows = P.rows;
    const uint64_t stride = P.stride, n0 = P.n0, plane = P.plane;
    const uint32_t c = P.c, dim = P.dim, dp = P.dp;
    uint16_t* dst = P.dst;
    const uint32_t per = dp / 8;
    const uint64_t t = block * 256 + threadIdx.x;
    const uint64_t row = t / per;
    if (row >= c) return;
    const uint32_t e = (uint32_t)(t - row * per) * 8;
    const uint64_t at = (n0 + row) * stride + e;
    uint16_t* o = dst + row * dp + e;
    if (DT == cgv::DT_F32) {
        const float* src = (const float*)rows + at;
        float v[8];
        if (e + 8 <= dim && ((uintptr_t)src & 15) == 0) {
            const float4 x = *(const float4*)src, y = *(const float4*)(src + 4);
            v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
        } else {
            for (int j = 0; j < 8; ++j) v[j] = e + j < dim ? src[j] : 0.0f;
        }
        uint16_t p[8][3];
#pragma unroll
        for (int j = 0; j < 8; ++j) split3(v[j], p[j]);
#pragma unroll
        for (int x = 0; x < 3; ++x) {
            uint32_t w[4];
            for (int j = 0; j < 4; ++j) w[j] = p[2 * j][x] | (uint32_t)p[2 * j + 1][x] << 16;
            *(uint4*)(o + x * plane) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    } else {
        const uint16_t* src = (const uint16_t*)rows + at;
        uint32_t w[4];
        for (int j = 0; j < 4; ++j)
            w[j] = (e + 2 * j < dim ? src[2 * j] : 0u) | (uint32_t)(e + 2 * j + 1 < dim ? src[2 * j + 1] : 0u) << 16;
        *(uint4*)o = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
template <int DT>
__global__ __launch_bounds__(256) void copy_rows_kernel(Piece P) { copy_piece_block<DT>(P, blockIdx.x); }

struct Problem {
    const void *queries, *rows;
    uint64_t q_stride, r_stride, n_rows;
    const int64_t* ids;
    const float* tscores;
    double* saved;            // [b][k + 2]: lse, tail, scores of the list
    uint32_t b, bp, dim, dp, k;
    float scale, tscale;
    uint16_t* qws;            // [planes][bp][dp]
    int device;
    uint32_t twin;            // backward: query i also stands at twin + i; 0: it does not
};

// (the first piece of the corpus is copied by further workgroups of the same launch)
template <int DT>
__global__ __launch_bounds__(256) void forward_prep_kernel(Problem P, uint32_t* __restrict__ anchor, Piece first) {
    const uint32_t lists = (P.k + 15) / 16;            // workgroups of a query
    const uint64_t block = wide_block(), listing = (uint64_t)P.bp * lists;
    if (block >= listing) return copy_piece_block<DT>(first, block - listing);
    const uint32_t i = (uint32_t)(block / lists), list = (uint32_t)(block % lists), wave = threadIdx.x >> 6;
    const int lane = threadIdx.x & 63;
    const uint64_t plane = (uint64_t)P.bp * P.dp;
    uint16_t* dst = P.qws + (uint64_t)i * P.dp;
    if (i >= P.b) {
        if (list) return;
        copy_row<DT>(nullptr, 0, P.dim, P.dp, dst, plane, threadIdx.x, 256);
        if (threadIdx.x == 0) anchor[i] = NONE;
        return;
    }
    const List l = read_list<false>(P.ids, P.tscores, i, P.k, P.n_rows, P.tscale, lane);
    if (!list) copy_row<DT>(l.has ? P.queries : nullptr, (uint64_t)i * P.q_stride, P.dim, P.dp, dst, plane, threadIdx.x, 256);
    // the listed rows' scores in 64 bits - a small loss and its gradient are as exact as the anchor's score -, four rows a wave
    double* sv = P.saved + (uint64_t)i * (P.k + 2);
    const uint32_t j0 = list * 16 + wave;
    if (j0 < P.k) {
        uint64_t at[4];                                // an entry without a row reads row 0, and nobody its score
        double s[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const uint32_t id = j0 + 4 * x < P.k ? pick(l.id, j0 + 4 * x) : NONE;
            at[x] = id == NONE ? 0 : (uint64_t)id * P.r_stride;
        }
        for (uint32_t e0 = 0; e0 < P.dim; e0 += 256) { // 20 loads on their way at a time
            float q[4], r[4][4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const uint32_t e = e0 + y * 64 + lane, ec = min(e, P.dim - 1);
                q[y] = load_elem<DT>(P.queries, (uint64_t)i * P.q_stride + ec);
#pragma unroll
                for (int x = 0; x < 4; ++x) r[y][x] = load_elem<DT>(P.rows, at[x] + ec);
                if (e >= P.dim) q[y] = r[y][0] = r[y][1] = r[y][2] = r[y][3] = 0.0f;
            }
#pragma unroll
            for (int y = 0; y < 4; ++y)
#pragma unroll
                for (int x = 0; x < 4; ++x) s[x] = fma((double)q[y], (double)r[y][x], s[x]);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const double v = wave_sum(s[x]) * (double)P.scale;
            if (lane == 0 && j0 + 4 * x < P.k) sv[2 + j0 + 4 * x] = v;
        }
    }
    if (list || wave) return;
    const uint32_t a = l.has ? pick(l.id, l.anchor) : NONE;
    if (lane == 0) anchor[i] = a;
}

// one wave per query: the corpus' partial maxima and sums, the loss
__global__ __launch_bounds__(256) void loss_kernel(Problem P, const float2* __restrict__ part, uint32_t parts, float* __restrict__ loss) {
    const uint32_t i = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (i >= P.b) return;
    const List l = read_list(P.ids, P.tscores, i, P.k, P.n_rows, P.tscale, lane);
    double* sv = P.saved + (uint64_t)i * (P.k + 2);
    if (!l.has) {
        if (lane == 0) loss[i] = 0.0f, sv[0] = 0.0, sv[1] = 0.0;
        return;
    }
    float m = -INFINITY;
    double s = 0.0;           // maxima are integers (or infinite): the factors are exact
    for (uint32_t p = lane; p < parts; p += 64) {
        const float2 v = part[(uint64_t)p * P.bp + i];
        const float nm = fmaxf(m, v.x), base = nm == -INFINITY ? 0.0f : nm;
        s = s * (double)exp2f(m - base) + (double)v.y * (double)exp2f(v.x - base);
        m = nm;
    }
    const float top = wave_max(m), base = top == -INFINITY ? 0.0f : top;
    s = wave_sum(s * (double)exp2f(m - base));
    const double sa = sv[2 + l.anchor];
    const double rest = (double)base * LN2 - sa + log(s);       // log of (the others' sum / the anchor's term)
    const double tail = rest > 40.0 ? rest : log1p(exp(rest));
    double sum = 0.0;
#pragma unroll
    for (int x = 0; x < 4; ++x)
        if (l.id[x] != NONE) sum += l.p[x] * (l.logp[x] + (sa - sv[2 + x * 64 + lane]) + tail);
    sum = wave_sum(sum);
    if (lane == 0) {
        loss[i] = (float)sum;
        sv[0] = sa + tail;
        sv[1] = tail;
    }
}

// fp16: the power of two for a query's entries of G, of which the largest is |c| * most: to 2^13 .. 2^14, as far as c itself stays in range
__device__ inline int g_power(float c, double most) {
    const double x = fabs((double)c * most);
    return x > 0.0 && x < (double)INFINITY ? max(min(min(13 - ilogb(x), 110 - ilogbf(c)), 120), -126) : 0;
}

// per place of a query, [bp] each
struct Places {
    float2* lse2;             // log2 of the softmax sum: its f32 and what that leaves
    float* coef;              // factor of G, times 2^power
    uint32_t* has;            // has a list
    int *power, *room;        // fp16; room: what power and the power of the query's copy for dR can add up to, INT_MAX: anything
};

// factor and log2 of the softmax sum per query; entries of G on the listed rows; the padded copy of the queries
template <int DT>
__global__ __launch_bounds__(256) void backward_prep_kernel(Problem P, const float* __restrict__ dloss, Places at, uint32_t* __restrict__ ent_id,
                                                            float* __restrict__ ent_val, Piece first_piece) {
    const uint64_t block = wide_block();
    if (block >= P.bp) return copy_piece_block<DT>(first_piece, block - P.bp);
    __shared__ uint32_t ids[MAX_K];
    __shared__ double ps[MAX_K], vs[4];
    __shared__ float qs[4];
    const uint32_t place = (uint32_t)block, i = P.twin && place >= P.twin ? place - P.twin : place, wave = threadIdx.x >> 6;
    const int lane = threadIdx.x & 63;
    const uint64_t plane = (uint64_t)P.bp * P.dp;
    uint16_t* dst = P.qws + (uint64_t)place * P.dp;
    if (i >= P.b) {
        copy_row<DT>(nullptr, 0, P.dim, P.dp, dst, plane, threadIdx.x, 256);
        if (threadIdx.x == 0) at.coef[place] = 0.0f, at.lse2[place] = make_float2(0.0f, 0.0f), at.has[place] = 0, at.power[place] = 0, at.room[place] = INT_MAX;
        if (P.twin && threadIdx.x < P.k) ent_id[(uint64_t)place * P.k + threadIdx.x] = NONE;
        return;
    }
    const List l = read_list(P.ids, P.tscores, i, P.k, P.n_rows, P.tscale, lane);
    float most_q = copy_row<DT>(l.has ? P.queries : nullptr, (uint64_t)i * P.q_stride, P.dim, P.dp, dst, plane, threadIdx.x, 256);
    const double* sv = P.saved + (uint64_t)i * (P.k + 2);
    const float c = l.has ? dloss[i] * P.scale : 0.0f;
    if (wave == 0)
        for (int x = 0; x < 4; ++x) {
            ids[x * 64 + lane] = l.id[x];
            ps[x * 64 + lane] = l.p[x];
        }
    __syncthreads();
    const uint32_t j = threadIdx.x, id = j < P.k ? ids[j] : NONE;
    const uint32_t aid = l.has ? ids[l.anchor] : NONE;
    bool first = id != NONE;
    double same = 0.0, other = 0.0;
    for (uint32_t x = 0; first && x < P.k; ++x) {
        if (ids[x] == id) {
            if (x < j) first = false;
            same += ps[x];
        } else {
            other += ps[x];
        }
    }
    double v = 0.0;
    if (first) v = id == aid ? expm1(-sv[1]) + other : exp(sv[2 + j] - sv[0]) - same;
    int power = 0;
    if constexpr (DT == cgv::DT_FP16) {
        // rows outside the list have a softmax value of 1 - exp(-tail) at most, the heaviest listed row having the rest
        double most = fabs(v);
        for (int o = 32; o; o >>= 1) most = fmax(most, __shfl_xor(most, o));
        most_q = wave_max(most_q);
        if (lane == 0) vs[wave] = most, qs[wave] = most_q;
        __syncthreads();
        most = fmax(fmax(fmax(vs[0], vs[1]), fmax(vs[2], vs[3])), l.has ? -expm1(-sv[1]) : 0.0);
        most_q = fmaxf(fmaxf(qs[0], qs[1]), fmaxf(qs[2], qs[3]));
        power = g_power(c, most);
        const double x = fabs((double)c * most);
        if (threadIdx.x == 0) {
            at.power[place] = power;
            at.room[place] = x > 0.0 && x < (double)INFINITY && most_q > 0.0f ? power + 15 - ilogbf(most_q) : INT_MAX;
        }
    }
    if (threadIdx.x == 0) {
        at.coef[place] = ldexpf(c, power);
        const double l2 = l.has ? sv[0] * LOG2E : 0.0;
        at.lse2[place] = make_float2((float)l2, (float)(l2 - (double)(float)l2));
        at.has[place] = l.has;
    }
    if (j >= P.k) return;
    ent_id[(uint64_t)place * P.k + j] = first ? id : NONE;
    ent_val[(uint64_t)place * P.k + j] = (float)ldexp(v * c, power);
}

// fp16: the queries' copy for dR, and the factor that takes the common power back. Few workgroups, each of which looks for that power itself
__global__ __launch_bounds__(256) void scaled_queries_kernel(Problem P, Places at, uint16_t* __restrict__ dst, float* __restrict__ unscale) {
    __shared__ int low[4];
    int common = INT_MAX;
    for (uint32_t i = threadIdx.x; i < P.bp; i += 256) common = min(common, at.room[i]);
    for (int o = 32; o; o >>= 1) common = min(common, __shfl_xor(common, o));
    if ((threadIdx.x & 63) == 0) low[threadIdx.x >> 6] = common;
    __syncthreads();
    common = min(min(low[0], low[1]), min(low[2], low[3]));
    common = common == INT_MAX ? 0 : min(common, 120);
    if (blockIdx.x == 0 && threadIdx.x == 0) *unscale = ldexpf(1.0f, -common);
    const uint32_t per = P.dp / 8;
    const uint64_t total = (uint64_t)P.bp * per;
    for (uint64_t t = (uint64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (uint64_t)gridDim.x * 256) {
        const uint32_t place = (uint32_t)(t / per);
        // a query without a gradient, or with one that is not finite, stays as it is
        const int shift = at.room[place] == INT_MAX ? 0 : common - at.power[place];
        const uint4 in = ((const uint4*)P.qws)[t];
        const uint32_t w[4] = {in.x, in.y, in.z, in.w};
        uint32_t o[4];
#pragma unroll
        for (int x = 0; x < 4; ++x)
            o[x] = f32_to_half<cgv::DT_FP16>(ldexpf(half_to_f32<cgv::DT_FP16>((uint16_t)w[x]), shift)) |
                   (uint32_t)f32_to_half<cgv::DT_FP16>(ldexpf(half_to_f32<cgv::DT_FP16>((uint16_t)(w[x] >> 16)), shift)) << 16;
        ((uint4*)dst)[t] = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

// 16-bit inputs, more than TWINS queries: the listed entries of G are its largest, and often all alike, so that their roundings do not average
// out. What 16 bits leave of them is added to dQ here (812 queries x 115 k x 64 fp16, lists of two: 0.00032 of its norm against 64 bits
// without, 0.00021 with, which is the result's own rounding)
struct Listed {
    const uint32_t* id;
    const float* val;
    uint32_t k;               // entries of a query, 0: not needed
    const void* rows;
    uint64_t stride;
};
// dQ: the shares' partial sums, added in a fixed order and rounded once. 64 threads a stretch of 256 elements, four groups of shares
template <int DT>
__global__ __launch_bounds__(256) void finish_dq_kernel(const float* __restrict__ part, uint32_t splits, uint64_t share, uint32_t b, uint32_t twin,
                                                        uint32_t dim, uint32_t dp,
                                                        const uint32_t* __restrict__ has, const int* __restrict__ power, void* __restrict__ dq, Listed l) {
    __shared__ float4 sum[4][64];
    const uint32_t stretches = (dim + 255) / 256;
    const uint64_t i = wide_block() / stretches;
    const uint32_t first = (uint32_t)(wide_block() % stretches) * 256, t = threadIdx.x & 63, group = threadIdx.x >> 6, e = first + t * 4;
    if (i >= b) return;
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (e < dp)
#pragma unroll 4
        for (uint32_t x = group; x < splits; x += 4) {
            const float4 v = *(const float4*)(part + x * share + i * dp + e);
            s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
            if (twin) {
                const float4 w = *(const float4*)(part + x * share + (i + twin) * dp + e);
                s = make_float4(s.x + w.x, s.y + w.y, s.z + w.z, s.w + w.w);
            }
        }
    sum[group][t] = s;
    __syncthreads();
    const uint32_t o = threadIdx.x, at = first + o;
    if (at >= dim) return;
    float v = 0.0f;
    for (int x = 0; x < 4; ++x) v += ((const float*)sum[x])[o];
    if (DT != cgv::DT_F32 && l.k) {
#pragma unroll 4
        for (uint32_t j = 0; j < l.k; ++j) {
            const uint32_t id = l.id[i * l.k + j];
            const float rest = rest16<DT>(l.val[i * l.k + j]), r = load_elem<DT>(l.rows, (id == NONE ? 0 : (uint64_t)id) * l.stride + at);
            if (id != NONE) v = fmaf(rest, r, v);
        }
    }
    if (DT == cgv::DT_FP16) v = ldexpf(v, -power[i]);
    store_elem<DT>(dq, i * dim + at, has[i] ? v : 0.0f);
}

// where the sorted entries of each group of corpus rows start, from group `first` on
__global__ __launch_bounds__(256) void starts_kernel(const uint32_t* __restrict__ keys, uint32_t n, uint32_t first, uint32_t groups, uint32_t* __restrict__ start) {
    const uint32_t g = blockIdx.x * 256 + threadIdx.x;
    if (g > groups) return;
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (keys[mid] < first + g) lo = mid + 1;
        else hi = mid;
    }
    start[g] = lo;
}

template <int DT>
__global__ void zero_kernel(void* p, uint64_t total) {
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (uint64_t)gridDim.x * blockDim.x) store_elem<DT>(p, i, 0.0f);
}

// ---- host -------------------------------------------------------------------------------------------------------------------

typedef Shape<64, 64, 2, 2> S64x64;
typedef Shape<64, 64, 2, 2, 3> S64x64f;      // f32
template <int DT>
using Small = std::conditional_t<DT == cgv::DT_F32, S64x64f, S64x64>;
typedef Shape<256, 64, 4, 1> S64;
typedef Shape<256, 128, 4, 2> S128;
typedef Shape<256, 192, 4, 2> S192;
typedef Shape<256, 256, 2, 4> S256;

uint64_t up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

struct Plan {
    uint32_t b, bp, dim, dp, k, planes, bm;               // bm: corpus rows of a tile of the scores
    uint32_t bn, columns, bn2, off;                       // the batch: `columns` tiles of bn queries, and from query `off` on one of bn2 (0: none)
    bool copy;                     // corpus rows go through a padded copy
    bool scaled;                   // fp16: dR takes the queries from a copy of their own
    uint64_t n, piece_f, piece_b;  // corpus rows of a piece, forward and backward
    uint32_t parts;                // (maximum, sum) pairs of a query, all pieces together
    struct Shares { uint32_t s1, s2; };                   // shares of the long axis, for the columns of bn and for that of bn2
    uint32_t dqn, dq_columns, dq_splits;                  // dQ: tiles of dqn queries, shares of the corpus
    SortPlan sort{0, 0};                                  // dR: of the listed entries, if they are sorted
    Plan(uint64_t b_, uint64_t n_, uint32_t dim_, uint32_t k_, int dtype) : b((uint32_t)b_), dim(dim_), k(k_), n(n_) {
        bp = (uint32_t)up(std::max<uint64_t>(b_, 1), 64);
        dp = (uint32_t)up(dim_, 64);
        planes = dtype == CGV_DTYPE_F32 ? 3 : 1;
        copy = dtype == CGV_DTYPE_F32 || dim % 8 != 0;
        scaled = dtype == CGV_DTYPE_FP16;
        // the tile width whose padded batch takes the least time. Narrower tiles read LDS more often per product: 768 queries over 200 k x 768
        // (bf16, loss and both gradients) take 1.19 ms with tiles of 256, 1.22 with 192, 1.28 with 128, 1.63 with 64. Against that stands the
        // padding: 576 queries take 0.84 ms with 192, 0.93 with 256, 0.92 with 128
        // The scores' last column may be narrower than the others (loss of 320 queries as 192 + 128: 130 us, as 2 x 192: 163 us). Not so dQ's:
        // columns with different shares of the corpus do not read it together (300 queries x 300 k x 1000: 339 us, with equal columns 304 us)
        double least = 1e30;
        for (int i = 0; i < 4; ++i) {
            const double t = (bp + WIDTH[i] - 1) / WIDTH[i] * cost(WIDTH[i]);
            if (t < least) least = t, bn = WIDTH[i], bn2 = 0;
        }
        dqn = bn;
        for (int i = 0; i < 2; ++i)
            for (int j = i + 1; j < 3; ++j) {
                const uint32_t w = WIDTH[i];
                if (bp <= WIDTH[j]) continue;
                const double t = (bp - WIDTH[j] + w - 1) / w * cost(w) + cost(WIDTH[j]);
                if (t < 0.97 * least) least = t, bn = w, bn2 = WIDTH[j];
            }
        bm = 256;
        // few tiles: small ones on more CUs, with more stages on the way. Loss and gradients of 256 queries x 768 with small and with large tiles,
        // bf16: 107 and 122 us at 20 k rows, 157 and 148 at 25 k; f32: 316 and 371 us at 20 k, 473 and 484 at 30 k
        if ((n_ + 255) / 256 * ((bp - bn2 + bn - 1) / bn + (bn2 > 0)) < (planes == 3 ? CUS / 2 : CUS * 3 / 8)) bm = bn = dqn = 64, bn2 = 0;
        columns = (bp - bn2 + bn - 1) / bn;
        off = bn2 ? columns * bn : bp;
        const uint64_t rows = up(n_, 256);
        const uint64_t by_copy = copy ? std::max<uint64_t>(256, PIECE_BYTES / ((uint64_t)dp * 2 * planes) / 256 * 256) : rows;
        const uint64_t by_g = std::max<uint64_t>(PIECE_ROWS, PIECE_BYTES / ((uint64_t)bp * 2 * planes) / 256 * 256);
        piece_f = std::min(rows, by_copy);
        piece_b = std::min(rows, std::min(by_copy, by_g));
        if (piece_b < rows && piece_b > 256 * CUS / 4) piece_b = piece_b / (256 * CUS / 4) * (256 * CUS / 4);
        const uint64_t last = n - (pieces_f() - 1) * piece_f;
        parts = (uint32_t)((pieces_f() - 1) * slots(score_shares((uint32_t)(piece_f / bm))) + slots(score_shares((uint32_t)((last + bm - 1) / bm))));
        dq_columns = (bp + dqn - 1) / dqn;
        dq_splits = std::max<uint32_t>(1, std::min<uint32_t>((uint32_t)(piece_b / BK), CUS / ((dp + bm - 1) / bm * dq_columns)));
        const uint64_t entries = b_ * k_;
        if (planes == 1 && !twin() && entries < 1ull << 31 && n >= (uint64_t)LISTED_ONE_IN * k_ && (double)b_ * n * dim >= SORTED_FROM)
            sort = SortPlan(entries, n, GROUP_BITS);
    }
    // the corpus' gradient of a piece of c rows: large tiles if they are enough to occupy half the card (256 queries x 20 k x 768 bf16, both
    // gradients: 72 us, in small ones 81)
    bool large_dr(uint64_t c) const { return (uint64_t)((dim + 255) / 256) * ((c + 255) / 256) >= CUS / 2; }
    static constexpr uint32_t WIDTH[4] = {256, 192, 128, 64};
    static double cost(uint32_t w) { return w / (w == 256 ? 1.0 : w == 192 ? 0.98 : w == 128 ? 0.93 : 0.73); }
    static uint32_t wave_rows(uint32_t bm, uint32_t bn) { return bm == 64 ? S64x64::WM : bn == 256 ? S256::WM : S64::WM; }
    uint32_t slots(Shares s) const { return std::max(s.s1 * wave_rows(bm, bn), bn2 ? s.s2 * wave_rows(bm, bn2) : 0u); }
    // shares of `tm` rows of tiles that occupy the card and end together, no more than the same time needs
    Shares score_shares(uint32_t tm) const {
        Shares s{std::max<uint32_t>(1, std::min(tm, CUS / columns)), 0};
        if (bn2) {
            double least = 1e30;
            s = {1, 1};
            for (uint32_t s1 = 1; s1 * columns < CUS; ++s1) {
                const uint32_t s2 = CUS - s1 * columns;
                const double t = std::max((tm + s1 - 1) / s1 * cost(bn), (tm + s2 - 1) / s2 * cost(bn2));
                if (t < least) least = t, s = {std::min(tm, s1), std::min(tm, s2)};
            }
            const uint32_t each = (tm + s.s2 - 1) / s.s2;
            s.s2 = (tm + each - 1) / each;
        }
        const uint32_t each = (tm + s.s1 - 1) / s.s1;
        s.s1 = (tm + each - 1) / each;
        return s;
    }
    uint64_t pieces_f() const { return (n + piece_f - 1) / piece_f; }
    uint64_t q_bytes() const { return up((uint64_t)planes * bp * dp * 2, 256); }
    uint64_t r_bytes(uint64_t piece) const { return copy ? up((uint64_t)planes * piece * dp * 2, 256) : 0; }
    // forward workspace
    uint64_t f_anchor() const { return q_bytes(); }
    uint64_t f_part() const { return f_anchor() + up((uint64_t)bp * 4, 256); }
    uint64_t f_rows() const { return f_part() + up((uint64_t)parts * bp * 8, 256); }
    uint64_t f_bytes() const { return f_rows() + r_bytes(piece_f); }
    // backward workspace
    uint64_t b_places() const { return q_bytes(); }                     // Places, and the factor of dR
    uint64_t b_ent() const { return b_places() + up((uint64_t)bp * 24 + 4, 256); }
    uint32_t twin() const { return planes == 1 && b <= TWINS ? TWINS : 0; }
    uint64_t b_g() const { return b_ent() + up((uint64_t)bp * k * 8, 256); }
    uint64_t b_part() const { return b_g() + up((uint64_t)planes * bp * piece_b * 2, 256); }
    uint64_t b_rows() const { return b_part() + up((uint64_t)dq_splits * bp * dp * 4, 256); }
    uint64_t b_scaled() const { return b_rows() + r_bytes(piece_b); }
    uint64_t b_sort() const { return b_scaled() + (scaled ? q_bytes() : 0); }
    uint64_t b_start() const { return b_sort() + sort.bytes; }
    uint64_t b_bytes() const { return b_start() + (sort.passes ? up(((piece_b >> GROUP_BITS) + 1) * 4, 256) : 0); }
};

void set_segments(Args& a, int dtype, bool small) {
    if (dtype != CGV_DTYPE_F32 || small) {       // small tiles: all planes are in a stage
        a.nseg = 1;
        a.sa[0] = a.sb[0] = 0;
        return;
    }
    static const uint32_t x[6] = {2, 0, 1, 1, 0, 0}, y[6] = {0, 2, 1, 0, 1, 0};   // the smallest products first
    a.nseg = 6;
    for (int i = 0; i < 6; ++i) a.sa[i] = x[i], a.sb[i] = y[i];
}

template <int DT, class S, bool TA, bool TB, int EPI>
int launch_gemm(const Args& a, int device, hipStream_t s) {
    constexpr int bytes = S::lds_bytes(EPI != EPI_DR);
    if (a.blocks == 0) return CGV_OK;
    void (*kern)(const Args) = gemm_kernel<DT, S, TA, TB, EPI>;
    static LdsLimit limit;
    OPCHK(limit.raise((const void*)kern, device, bytes));
    hipLaunchKernelGGL(kern, dim3(a.blocks), dim3(S::THREADS), bytes, s, a);
    OPCHK(hipGetLastError());
    return CGV_OK;
}
template <int DT>
int launch_gradients(const Args& q, const Args& r, int device, hipStream_t s) {
    typedef Small<DT> S;
    constexpr int bytes = S::lds_bytes(true);
    void (*kern)(const Args, const Args) = gradients_kernel<DT, S>;
    static LdsLimit limit;
    OPCHK(limit.raise((const void*)kern, device, bytes));
    hipLaunchKernelGGL(kern, dim3(q.blocks + r.blocks), dim3(S::THREADS), bytes, s, q, r);
    OPCHK(hipGetLastError());
    return CGV_OK;
}
template <int DT, class S, class T, bool TA, bool TB, int EPI>
int launch_mixed(const Args& a, const Args& b, int device, hipStream_t s) {
    constexpr int bytes = std::max(S::lds_bytes(true), T::lds_bytes(true));
    void (*kern)(const Args, const Args) = mixed_kernel<DT, S, T, TA, TB, EPI>;
    static LdsLimit limit;
    OPCHK(limit.raise((const void*)kern, device, bytes));
    hipLaunchKernelGGL(kern, dim3(a.blocks + b.blocks), dim3(S::THREADS), bytes, s, a, b);
    OPCHK(hipGetLastError());
    return CGV_OK;
}
template <int DT, bool TA, bool TB, int EPI>
int launch_by_width(const Args& a, uint32_t bm, uint32_t bn, int device, hipStream_t s) {
    if (bm == 64) return launch_gemm<DT, Small<DT>, TA, TB, EPI>(a, device, s);
    if (bn == 64) return launch_gemm<DT, S64, TA, TB, EPI>(a, device, s);
    if (bn == 128) return launch_gemm<DT, S128, TA, TB, EPI>(a, device, s);
    if (bn == 192) return launch_gemm<DT, S192, TA, TB, EPI>(a, device, s);
    return launch_gemm<DT, S256, TA, TB, EPI>(a, device, s);
}
// scores: the arguments `a` of all columns, and their shares
template <int DT, int EPI>
int launch_scores(const Plan& pl, Args a, Plan::Shares sh, int device, hipStream_t s) {
    a.tn = pl.columns;
    a.splits = sh.s1;
    a.blocks = a.tn * a.splits;
    // The loss with one column of tiles reads every row once: past the caches, if they could not hold the rows for the next call (256 queries x
    // 400 k x 768 bf16: 180 -> 166 us). Not so for G, whose rows the gradients read again (gradients of the same: 672 us, past the caches 695)
    if constexpr (EPI == EPI_LSE && DT != cgv::DT_F32) {
        if (pl.columns == 1 && !pl.bn2 && pl.bm == 256 && a.m_valid * a.a.pitch > CACHE) {
            if (pl.bn == 64) return launch_gemm<DT, Once<S64>, false, false, EPI>(a, device, s);
            if (pl.bn == 128) return launch_gemm<DT, Once<S128>, false, false, EPI>(a, device, s);
            if (pl.bn == 192) return launch_gemm<DT, Once<S192>, false, false, EPI>(a, device, s);
            return launch_gemm<DT, Once<S256>, false, false, EPI>(a, device, s);
        }
    }
    if (!pl.bn2) return launch_by_width<DT, false, false, EPI>(a, pl.bm, pl.bn, device, s);
    Args b = a;                        // the last column
    b.tn = 1;
    b.splits = b.blocks = sh.s2;
    b.b.p += pl.off * b.b.pitch;
    b.b.limit -= pl.off;
    b.n_valid -= pl.off;
    b.n_pad -= pl.off;
    if (EPI == EPI_LSE) {
        b.anchor += pl.off;
        b.part += pl.off;
    } else {
        b.coef += pl.off;
        b.lse2 += pl.off;
        b.ent_id += (uint64_t)pl.off * b.ent_k;
        b.ent_val += (uint64_t)pl.off * b.ent_k;
        b.out += pl.off * b.out_pitch;
    }
    a.n_valid = a.n_pad = pl.off;
    if (pl.bn2 == 192) return launch_mixed<DT, S256, S192, false, false, EPI>(a, b, device, s);
    return pl.bn == 256 ? launch_mixed<DT, S256, S128, false, false, EPI>(a, b, device, s) : launch_mixed<DT, S192, S128, false, false, EPI>(a, b, device, s);
}

// scores of the corpus rows [n0, n0 + c) against all queries
Args score_args(const Plan& pl, const Problem& P, int dtype, const char* rows, uint64_t pitch, uint64_t plane, uint32_t c) {
    Args a{};
    a.a = {rows, pitch, plane, c};
    a.b = {(const char*)P.qws, (uint64_t)pl.dp * 2, (uint64_t)pl.bp * pl.dp * 2, pl.bp};
    set_segments(a, dtype, pl.bm == 64);
    a.ksteps = pl.dp / BK;
    a.kvalid = pl.copy ? pl.dp : pl.dim;
    a.tm = (c + pl.bm - 1) / pl.bm;
    a.scale2 = (float)(P.scale * LOG2E);
    if (a.scale2 == 0.0f) a.scale2 = FLT_TRUE_MIN;     // -inf times it is to stay -inf
    a.m_valid = c;
    a.n_valid = pl.b;
    a.n_pad = a.part_ld = pl.bp;
    return a;
}

Piece piece_of(const Plan& pl, const Problem& P, uint64_t n0, uint64_t most, char* dst) {
    return {P.rows, P.r_stride, n0, most * pl.dp, (uint16_t*)dst, pl.copy ? (uint32_t)std::min<uint64_t>(most, pl.n - n0) : 0u, pl.dim, pl.dp};
}
uint32_t copy_blocks(const Piece& p) { return (uint32_t)(((uint64_t)p.c * (p.dp / 8) + 255) / 256); }

template <int DT>
int copy_piece(const Piece& p, hipStream_t s) {
    hipLaunchKernelGGL((copy_rows_kernel<DT>), dim3(copy_blocks(p)), dim3(256), 0, s, p);
    OPCHK(hipGetLastError());
    return CGV_OK;
}

template <int DT>
int forward(const Plan& pl, Problem P, int dtype, float* loss, char* ws, hipStream_t s) {
    P.qws = (uint16_t*)ws;
    uint32_t* anchor = (uint32_t*)(ws + pl.f_anchor());
    float2* part = (float2*)(ws + pl.f_part());
    const Piece first = piece_of(pl, P, 0, pl.piece_f, ws + pl.f_rows());
    hipLaunchKernelGGL((forward_prep_kernel<DT>), wide_grid((uint64_t)pl.bp * ((pl.k + 15) / 16) + copy_blocks(first)), dim3(256), 0, s, P, anchor, first);
    OPCHK(hipGetLastError());
    uint32_t parts = 0;
    for (uint64_t n0 = 0; n0 < pl.n; n0 += pl.piece_f) {
        const uint32_t c = (uint32_t)std::min<uint64_t>(pl.piece_f, pl.n - n0);
        const char* rows = (const char*)P.rows + n0 * P.r_stride * 2;
        uint64_t pitch = P.r_stride * 2, plane = 0;
        if (pl.copy) {
            const int rc = n0 ? copy_piece<DT>(piece_of(pl, P, n0, pl.piece_f, ws + pl.f_rows()), s) : CGV_OK;
            if (rc) return rc;
            rows = ws + pl.f_rows();
            pitch = (uint64_t)pl.dp * 2;
            plane = pl.piece_f * pitch;
        }
        Args a = score_args(pl, P, dtype, rows, pitch, plane, c);
        a.row0 = n0;
        a.anchor = anchor;
        a.part = part + (uint64_t)parts * pl.bp;
        const Plan::Shares sh = pl.score_shares(a.tm);
        a.slots = pl.slots(sh);
        parts += a.slots;
        const int rc = launch_scores<DT, EPI_LSE>(pl, a, sh, P.device, s);
        if (rc) return rc;
    }
    hipLaunchKernelGGL(loss_kernel, dim3((pl.b + 3) / 4), dim3(256), 0, s, P, (const float2*)part, parts, loss);
    OPCHK(hipGetLastError());
    return CGV_OK;
}

template <int DT>
int backward(const Plan& pl, Problem P, int dtype, const float* dloss, void* dq, void* dr, char* ws, hipStream_t s) {
    P.qws = (uint16_t*)ws;
    Places at;
    at.lse2 = (float2*)(ws + pl.b_places());
    at.coef = (float*)(at.lse2 + pl.bp);
    at.has = (uint32_t*)(at.coef + pl.bp);
    at.power = (int*)(at.has + pl.bp);
    at.room = at.power + pl.bp;
    float* unscale = (float*)(at.room + pl.bp);
    uint32_t* ent_id = (uint32_t*)(ws + pl.b_ent());
    float* ent_val = (float*)(ent_id + (uint64_t)pl.bp * pl.k);
    P.twin = pl.twin();
    char* G = ws + pl.b_g();
    float* part = (float*)(ws + pl.b_part());
    const uint64_t g_pitch = pl.piece_b * 2, g_plane = (uint64_t)pl.bp * g_pitch;
    const Piece first = piece_of(pl, P, 0, pl.piece_b, ws + pl.b_rows());
    hipLaunchKernelGGL((backward_prep_kernel<DT>), wide_grid((uint64_t)pl.bp + copy_blocks(first)), dim3(256), 0, s, P, dloss, at, ent_id, ent_val, first);
    OPCHK(hipGetLastError());
    if (DT == cgv::DT_FP16 && dr) {
        const uint64_t blocks = ((uint64_t)pl.bp * (pl.dp / 8) + 255) / 256;
        hipLaunchKernelGGL(scaled_queries_kernel, dim3((unsigned)std::min<uint64_t>(blocks, CUS)), dim3(256), 0, s, P, at, (uint16_t*)(ws + pl.b_scaled()), unscale);
        OPCHK(hipGetLastError());
    }
    const uint32_t *keys, *pos = nullptr;
    uint32_t* start = nullptr;
    if (dr && pl.sort.passes) {
        if (const int rc = sort_ids(pl.sort, P.ids, (uint64_t)pl.b * pl.k, pl.n, ws + pl.b_sort(), nullptr, &keys, &pos, s)) return rc;
        start = (uint32_t*)(ws + pl.b_start());
    }
    for (uint64_t n0 = 0; n0 < pl.n; n0 += pl.piece_b) {
        const uint32_t c = (uint32_t)std::min<uint64_t>(pl.piece_b, pl.n - n0);
        const char* rows = (const char*)P.rows + n0 * P.r_stride * 2;
        uint64_t pitch = P.r_stride * 2, plane = 0;
        int rc;
        if (pl.copy) {
            if (n0 && (rc = copy_piece<DT>(piece_of(pl, P, n0, pl.piece_b, ws + pl.b_rows()), s))) return rc;
            rows = ws + pl.b_rows();
            pitch = (uint64_t)pl.dp * 2;
            plane = pl.piece_b * pitch;
        }
        Args a = score_args(pl, P, dtype, rows, pitch, plane, c);
        a.coef = at.coef;
        a.lse2 = at.lse2;
        if (P.twin) a.n_valid = pl.bp;
        a.twin = P.twin;
        a.row0 = n0;
        a.ent_id = ent_id;
        a.ent_val = ent_val;
        a.ent_k = pl.k;
        a.out = G;
        a.out_pitch = g_pitch;
        a.out_plane = g_plane;
        if ((rc = launch_scores<DT, EPI_G>(pl, a, pl.score_shares(a.tm), P.device, s))) return rc;
        const bool big = dr && pl.large_dr(c), together = dq && dr && !big && pl.bm == 64;      // small tiles: both gradients share a launch
        Args d{}, e{};
        if (dq) {
            d.a = {rows, pitch, plane, pl.copy ? pl.dp : pl.dim};
            d.b = {G, g_pitch, g_plane, pl.bp};
            set_segments(d, dtype, pl.bm == 64);
            d.ksteps = (c + BK - 1) / BK;
            d.kvalid = c;
            d.tm = (pl.dp + pl.bm - 1) / pl.bm;
            d.tn = pl.dq_columns;
            d.splits = pl.dq_splits;
            d.blocks = d.tm * d.tn * d.splits;
            d.m_valid = pl.dp;
            d.n_valid = P.twin ? pl.bp : pl.b;
            d.part_ld = pl.dp;
            d.out = (char*)part;
            d.out_plane = (uint64_t)pl.bp * pl.dp * 4;
            d.accumulate = n0 > 0;
        }
        if (start) {
            const uint32_t groups = (c + (1u << GROUP_BITS) - 1) >> GROUP_BITS;
            hipLaunchKernelGGL(starts_kernel, dim3(groups / 256 + 1), dim3(256), 0, s, keys, pl.b * pl.k, (uint32_t)(n0 >> GROUP_BITS), groups, start);
            OPCHK(hipGetLastError());
            e.ent_start = start;
            e.ent_pos = pos;
            e.ent_groups = groups;
        }
        if (dr) {
            e.a = {DT == cgv::DT_FP16 ? ws + pl.b_scaled() : (const char*)P.qws, (uint64_t)pl.dp * 2, (uint64_t)pl.bp * pl.dp * 2, pl.dp};
            e.b = {G, g_pitch, g_plane, (uint32_t)pl.piece_b};
            e.ksteps = pl.bp / BK;
            e.kvalid = pl.bp;
            set_segments(e, dtype, !big);
            const uint32_t side = big ? 256 : 64;
            e.tm = (pl.dim + side - 1) / side;
            e.tn = (c + side - 1) / side;
            e.splits = 1;
            e.blocks = (uint32_t)std::min<uint64_t>((uint64_t)e.tm * e.tn, CUS);
            e.m_valid = pl.dim;
            e.n_valid = c;
            e.out = (char*)dr + n0 * pl.dim * esize(dtype);
            e.out_pitch = (uint64_t)pl.dim * esize(dtype);
            e.vec_out = e.out_pitch % 16 == 0 && (uintptr_t)dr % 16 == 0;
            e.unscale = DT == cgv::DT_FP16 ? unscale : nullptr;
            e.row0 = n0;
            e.ent_id = ent_id;
            e.ent_val = ent_val;
            e.ent_k = pl.k;
            e.ent_n = big || start || P.twin || DT == cgv::DT_F32 || (uint64_t)pl.b * pl.k > LOOKED_THROUGH ? 0 : pl.b * pl.k;
        }
        if (together) {
            if ((rc = launch_gradients<DT>(d, e, P.device, s))) return rc;
            continue;
        }
        if (dq && (rc = launch_by_width<DT, true, false, EPI_DQ>(d, pl.bm, pl.dqn, P.device, s))) return rc;
        if (dr && (rc = big ? launch_gemm<DT, S256, true, true, EPI_DR>(e, P.device, s) : launch_gemm<DT, Small<DT>, true, true, EPI_DR>(e, P.device, s))) return rc;
    }
    if (dq) {
        hipLaunchKernelGGL((finish_dq_kernel<DT>), wide_grid((uint64_t)pl.b * ((pl.dim + 255) / 256)), dim3(256), 0, s, (const float*)part, pl.dq_splits, (uint64_t)pl.bp * pl.dp,
                           pl.b, P.twin, pl.dim, pl.dp, (const uint32_t*)at.has, (const int*)at.power, dq, Listed{ent_id, ent_val, P.twin ? 0 : pl.k, P.rows, P.r_stride});
        OPCHK(hipGetLastError());
    }
    return CGV_OK;
}

bool sizes_ok(uint64_t b, uint64_t n_rows, uint32_t dim, uint32_t k, int dtype) {
    return b <= (1ull << 24) && n_rows >= 1 && n_rows < (1ull << 31) - 1 && dim >= 1 && dim <= 8192 && k >= 1 && k <= MAX_K &&
           (dtype == CGV_DTYPE_F32 || dtype == CGV_DTYPE_BF16 || dtype == CGV_DTYPE_FP16);
}

int check_loss(const void* q, uint64_t qs, const void* r, uint64_t rs, int dtype, uint64_t b, uint64_t n, uint32_t dim, const int64_t* ids, uint32_t k,
               float scale, float tscale, const void* saved) {
    if (dtype != CGV_DTYPE_F32 && dtype != CGV_DTYPE_BF16 && dtype != CGV_DTYPE_FP16) return fail(CGV_ERR_INVALID_ARG, "dtype must be f32, bf16 or fp16");
    if (!sizes_ok(b, n, dim, k, dtype)) return fail(CGV_ERR_INVALID_ARG, "b must be at most 2^24, n_rows in 1..2^31 - 1, dim in 1..=8192, k in 1..=256");
    if (qs < dim || rs < dim) return fail(CGV_ERR_INVALID_ARG, "a stride is smaller than dim");
    if (!(fabsf(scale) < INFINITY) || !(fabsf(tscale) < INFINITY)) return fail(CGV_ERR_NONFINITE, "scale is not finite");
    if (!r || (b && (!q || !ids || !saved))) return fail(CGV_ERR_INVALID_ARG, "NULL argument");
    if (dtype != CGV_DTYPE_F32 && dim % 8 == 0 && ((uintptr_t)r % 16 || rs % 8 || rs > (1u << 22)))
        return fail(CGV_ERR_INVALID_ARG, "rows of 16-bit elements with dim a multiple of 8 are read in place: they must start on 16-byte addresses, at "
                                         "most 2^22 elements apart");
    return CGV_OK;
}

}  // namespace

extern "C" {

size_t cgv_corpus_loss_workspace(uint64_t b, uint64_t n_rows, uint32_t dim, uint32_t k, int dtype) {
    if (!sizes_ok(b, n_rows, dim, k, dtype) || b == 0) return 0;
    return (size_t)Plan(b, n_rows, dim, k, dtype).f_bytes();
}

size_t cgv_corpus_loss_grad_workspace(uint64_t b, uint64_t n_rows, uint32_t dim, uint32_t k, int dtype) {
    if (!sizes_ok(b, n_rows, dim, k, dtype) || b == 0) return 0;
    return (size_t)Plan(b, n_rows, dim, k, dtype).b_bytes();
}

int cgv_corpus_loss_dev(int device_id, const void* queries_dev, uint64_t query_stride, const void* rows_dev, uint64_t row_stride, int dtype, uint64_t b,
                        uint64_t n_rows, uint32_t dim, const int64_t* ids_dev, const float* teacher_scores_dev, uint32_t k, float scale,
                        float teacher_scale, float* loss_dev, double* saved_dev, void* workspace_dev, size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        int rc = check_loss(queries_dev, query_stride, rows_dev, row_stride, dtype, b, n_rows, dim, ids_dev, k, scale, teacher_scale, saved_dev);
        if (rc) return rc;
        if (b == 0) return CGV_OK;
        if (!loss_dev) return fail(CGV_ERR_INVALID_ARG, "NULL argument");
        const Plan pl(b, n_rows, dim, k, dtype);
        if (!workspace_dev || workspace_bytes < pl.f_bytes()) return fail(CGV_ERR_INVALID_ARG, "the workspace is smaller than cgv_corpus_loss_workspace says");
        if ((uintptr_t)workspace_dev % 256) return fail(CGV_ERR_INVALID_ARG, "the workspace must be aligned to 256 bytes");
        if ((rc = need_gpu(device_id))) return rc;
        DeviceScope dev(device_id);
        OPCHK(dev.enter());
        const Problem P{queries_dev, rows_dev, query_stride, row_stride, n_rows, ids_dev, teacher_scores_dev, saved_dev,
                        pl.b, pl.bp, dim, pl.dp, k, scale, teacher_scale, nullptr, device_id, 0};
        return by_dtype(dtype, [&](auto t) { return forward<decltype(t)::value>(pl, P, dtype, loss_dev, (char*)workspace_dev, (hipStream_t)stream); });
    });
}

int cgv_corpus_loss_grad_dev(int device_id, const void* queries_dev, uint64_t query_stride, const void* rows_dev, uint64_t row_stride, int dtype,
                             uint64_t b, uint64_t n_rows, uint32_t dim, const int64_t* ids_dev, const float* teacher_scores_dev, uint32_t k,
                             float scale, float teacher_scale, const double* saved_dev, const float* dloss_dev, void* dqueries_dev, void* drows_dev,
                             void* workspace_dev, size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        int rc = check_loss(queries_dev, query_stride, rows_dev, row_stride, dtype, b, n_rows, dim, ids_dev, k, scale, teacher_scale, saved_dev);
        if (rc) return rc;
        if (!dqueries_dev && !drows_dev) return CGV_OK;
        if (b && !dloss_dev) return fail(CGV_ERR_INVALID_ARG, "NULL argument");
        const Plan pl(b, n_rows, dim, k, dtype);
        if (b && (!workspace_dev || workspace_bytes < pl.b_bytes()))
            return fail(CGV_ERR_INVALID_ARG, "the workspace is smaller than cgv_corpus_loss_grad_workspace says");
        if (b && (uintptr_t)workspace_dev % 256) return fail(CGV_ERR_INVALID_ARG, "the workspace must be aligned to 256 bytes");
        if ((rc = need_gpu(device_id))) return rc;
        DeviceScope dev(device_id);
        OPCHK(dev.enter());
        const hipStream_t s = (hipStream_t)stream;
        const Problem P{queries_dev, rows_dev, query_stride, row_stride, n_rows, ids_dev, teacher_scores_dev, const_cast<double*>(saved_dev),
                        pl.b, pl.bp, dim, pl.dp, k, scale, teacher_scale, nullptr, device_id, 0};
        return by_dtype(dtype, [&](auto t) -> int {
            constexpr int DT = decltype(t)::value;
            if (b == 0) {
                if (drows_dev) {
                    hipLaunchKernelGGL((zero_kernel<DT>), dim3(1024), dim3(256), 0, s, drows_dev, n_rows * dim);
                    OPCHK(hipGetLastError());
                }
                return CGV_OK;
            }
            return backward<DT>(pl, P, dtype, dloss_dev, dqueries_dev, drows_dev, (char*)workspace_dev, s);
        });
    });
}

}  // extern "C"
