// kernels_gemm.h - the matrix products behind the softmax losses (softmax.hip): one persistent MFMA loop, three products, four
// epilogues. Written from the formulas: with S = c Q R^T, G = dL/dS * c,
//     scores   M = corpus rows, N = queries,     K = elements   -> running maximum and sum of exp per query, or a piece of G
//     dQ       M = elements,    N = queries,     K = corpus     -> f32 partial sums, one slot per share of the corpus
//     dR       M = elements,    N = corpus rows, K = queries    -> rows of the corpus' gradient
// An operand lies in memory either with K contiguous ("rows") or with M or N contiguous ("columns", TA / TB): R is read by rows
// for the scores and by columns for dQ, G [query][corpus] by rows for dQ and by columns for dR. Columns are turned into
// fragments by ds_read_b64_tr_b16: of 16 lanes, lane 4 j + a supplies the elements 4 a .. 4 a + 3 of k-row j and lane i receives
// element i of the k-rows 0 .. 3.
//
// C layout of v_mfma_f32_32x32x16: a lane holds ONE column n = lane & 31 and 16 rows m = (r & 3) + 8 (r >> 2) + 4 (lane >> 5).
// With queries as N the softmax statistics of a query stay in its lane; four consecutive m are four neighbours in memory of G
// [query][corpus], dQ and dR.
//
// f32 inputs are three bf16 planes x = h + m + l (8 bits each, exact); a product is the six plane products of weight 2^0 .. 2^-16
// (the three left out are below 2^-24 of it), added in f32 from the smallest up, or the five small ones in a sum of their own: six passes
// of bf16 MFMA run at 2.5 / 6 = 0.42 PFLOP/s, the f32 MFMA at 0.16.
//
// Workgroup tiles of 256 corpus rows x 256 queries, eight waves of 128 x 64: 128 accumulators leave room for two waves a SIMD and two sets
// of fragments. Stages of 64 elements of K (128 bytes of a row: shorter pieces load at less than half the rate) go from memory to LDS
// directly; a wave issues its loads one at a time between matrix instructions, as a burst behind the barrier they held the wave up
// (scores of 1024 x 125 k x 768 bf16: 198 us, spread 177). One barrier a stage. Bound by the matrix cores at the clock that they
// leave (bf16, same sizes, 197 GFLOP each): scores 170 us with their exponentials, dQ 163 us, dR 186 us (200 with the listed entries of 1024 lists
// of ten) and G 199 us with 192 and 256 MB of results; matrix pipes busy 0.65, 0.70, 0.62 (0.56) and 0.54 of the time at 1.5 .. 1.8 GHz. What is left of the scores' time are the
// exponentials, a sixth of it, which nothing runs beside: both waves of a SIMD reach them at the same barrier, and two workgroups of
// 128 x 128 on a CU, which would not, load twice as much (scores 252 us, dQ 253 us).
#pragma once
#include <type_traits>

#include "common.h"
#include "ops_common.h"

namespace cgv_gemm {

typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr uint32_t BK = 64;                 // elements of K a stage: 128 bytes of a row
constexpr int MAX_SEG = 6;

template <int DT>
__device__ inline f32x16 mma(s16x8 a, s16x8 b, f32x16 c) {
    if constexpr (DT == cgv::DT_FP16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
}

// three bf16 planes of an f32, largest first
__device__ inline void split3(float x, uint16_t (&p)[3]) {
    p[0] = cgv::f32_to_bf16_rne(x);
    const float r = x - cgv::bf16_to_f32(p[0]);
    p[1] = cgv::f32_to_bf16_rne(r);
    p[2] = cgv::f32_to_bf16_rne(r - cgv::bf16_to_f32(p[1]));
}

struct Operand {
    const char* p;          // plane 0, element (0, 0)
    uint64_t pitch, plane;  // bytes from row to row in memory, from plane to plane
    uint32_t limit;         // rows form: rows that exist; columns form: elements of a row (a multiple of 8). Beyond: clamped
};

enum Epilogue { EPI_LSE, EPI_G, EPI_DQ, EPI_DR };

struct Args {
    Operand a, b;
    uint32_t nseg, sa[MAX_SEG], sb[MAX_SEG];      // plane pairs
    uint32_t ksteps, kvalid;                      // stages of 64; elements of K that `a` holds
    uint32_t tm, tn;                              // tiles of M and N
    uint32_t splits, blocks;                      // shares of the long axis; workgroups
    // epilogues
    float scale2;                                 // LSE, G: scores in units of log 2 = accumulator * scale2, not zero
    uint32_t m_valid, n_valid;                    // rows / columns of the result that exist
    uint32_t n_pad;                               // LSE, G: columns that have a place in part / out, n_valid rounded up to 64
    uint64_t row0;                                // LSE, G: corpus row of m = 0; DR: of n = 0
    const uint32_t* anchor;                       // LSE: [n] corpus row left out of the sum, 0xffffffff for none
    float2* part;                                 // LSE: [slots][part_ld] (maximum, sum), slots at least splits * WM
    uint32_t slots;
    uint32_t part_ld;
    const float* coef;                            // G: [n] factor
    const float2* lse2;                           // G: [n] log2 of the softmax sum, its f32 and what that leaves
    uint32_t twin;                                // G: from this column on, what 16 bits leave of the entries of the column `twin` before; 0: none
    const uint32_t* ent_id;                       // G, DR: [n][ent_k] corpus rows whose entries are given, 0xffffffff for none
    const float* ent_val;                         // G: [n][ent_k] those entries
    uint32_t ent_k, ent_n;                        // DR, small tiles: ent_n of them, all queries together, whose rounding is made good; 0: none
    const uint32_t *ent_start, *ent_pos;          // DR, or by corpus row: where those of each 32 rows from row0 on start, [ent_groups + 1], and their places; NULL: none
    uint32_t ent_groups;
    char* out;                                    // G, DR, DQ
    uint64_t out_pitch, out_plane;                // bytes
    uint32_t accumulate, vec_out;                 // DQ: add to what is there; DR: 16-byte stores possible
    const float* unscale;                         // DR: [1] factor of the result; NULL: 1
};

// PL planes of an operand in a stage: 3 for f32 where tiles are small - each plane is then loaded once and not once per product
template <int BM_, int BN_, int WM_, int WN_, int PL_ = 1>
struct Shape {
    static constexpr int PL = PL_;
    static constexpr bool ONCE = false;           // A is read past the caches
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NW = WM_ * WN_, THREADS = 64 * NW;
    static constexpr int TM = BM / WM, TN = BN / WN, MB = TM / 32, NB = TN / 32;
    static constexpr int A_BYTES = BM * 128, B_BYTES = BN * 128, STAGE = PL * (A_BYTES + B_BYTES);
    // stages in LDS: as many as fit, six at most; all but one of them are loading or waiting
    static constexpr int STAGES = 160 * 1024 / STAGE < 6 ? 160 * 1024 / STAGE : 6;
    // where only two fit, the operand that comes from HBM has three places and loads two stages ahead; the other, which the workgroups
    // share through L2, has two
    static constexpr bool UNEVEN = STAGES == 2;
    static constexpr int lds_bytes(bool long_a) { return STAGES * STAGE + (UNEVEN ? long_a ? A_BYTES : B_BYTES : 0); }
};

template <class S>
struct Once : S {
    static constexpr bool ONCE = true;
};

// swizzle of a row's eight 16-byte pieces: 16 consecutive rows put the same piece at 16 different places of the 256 bytes that the
// 64 banks hold (row & 7 instead repeats after eight: half of the reads' cycles were conflicts)
__device__ inline uint32_t row_swz(uint32_t row) { return (row >> 1) & 7u; }

// swizzle of the 32-byte segments of k-row k in the columns form: four k-rows of one read lie in different banks
template <int W>
__device__ inline uint32_t seg_swz(uint32_t k) {
    return W >= 128 ? (k & 3u) << 1 : ((k >> 1) & 1u) << 1;
}

// where a lane's 16-byte pieces of a W-row (or W-column) stage come from
template <bool T, int W, int NW>
struct Loader {
    static constexpr int I = W / 8 / NW;          // 1-KiB instructions of a wave
    static_assert(!T || 1024 % (W * 2) == 0, "columns form: an instruction loads whole k-rows");
    uint32_t voff[I];
    // first = first row / column of the tile; elems: elements of K that exist from the stage's first on, 64 but for the last stage.
    // Rows form: the missing ones are read as the row's last eight (the other operand holds zeros there); columns form: as the last k-row
    __device__ void place(const Operand& o, uint32_t first, int wave, int lane, uint32_t elems) {
#pragma unroll
        for (int i = 0; i < I; ++i) {
            const uint32_t u = (uint32_t)(wave * I + i);
            if (!T) {
                const uint32_t row = u * 8 + (lane >> 3), chunk = (uint32_t)(lane & 7) ^ row_swz(row);
                voff[i] = (min(first + row, o.limit - 1) - first) * (uint32_t)o.pitch + min(chunk * 8, elems - 8) * 2;
            } else {
                constexpr uint32_t RB = W * 2, LPR = RB / 16;           // bytes of a k-row, lanes of one
                const uint32_t k = u * (1024 / RB) + lane / LPR, c = lane % LPR;
                const uint32_t seg = (c >> 1) ^ seg_swz<W>(k), col = seg * 16 + (c & 1) * 8;
                voff[i] = min(k, elems - 1) * (uint32_t)o.pitch + (min(first + col, o.limit - 8) - first) * 2;
            }
        }
    }
    template <int AUX>
    __device__ void issue_one(int i, const char* base, uint32_t soff, char* lds, int wave) const {
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0x7fffffff, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(lds + (wave * I + i) * 1024), 16, voff[i], soff, 0, AUX);
    }
    template <int AUX>
    __device__ void issue(const char* base, uint32_t soff, char* lds, int wave) const {
#pragma unroll
        for (int i = 0; i < I; ++i) issue_one<AUX>(i, base, soff, lds, wave);
    }
};

// Four rows of a column form's piece, turned. The `restrict` here is for the compiler's waits alone: in front of a transposing read about which
// it knows nothing it waits for every load into LDS on its way (dQ of 1024 x 125 k x 768 bf16: 416 us with those waits, 194 without them). That the
// piece has landed is what the stage's own wait and barrier see to
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
__device__ __forceinline__ s16x4 read_turned(lds_s16x4* __restrict__ p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16(p); }

// fragment of 32 rows (or columns) starting at `at` of a stage, 16 elements of K from kk * 16
template <bool T, int W>
__device__ inline s16x8 fragment(const char* lds, uint32_t at, int kk, int lane) {
    if (!T) {
        const uint32_t row = at + (lane & 31);
        return *(const s16x8*)(lds + row * 128 + (((uint32_t)(kk * 2 + (lane >> 5)) ^ row_swz(lane & 31)) << 4));
    }
    constexpr uint32_t RB = W * 2;
    const uint32_t k = (uint32_t)kk * 16 + (lane >> 5) * 8 + ((lane & 15) >> 2);
    const uint32_t seg = at / 16 + ((lane >> 4) & 1);
    const char* p = lds + k * RB + ((seg ^ seg_swz<W>(k)) << 5) + (lane & 3) * 8;
    const s16x4 lo = read_turned((lds_s16x4*)p), hi = read_turned((lds_s16x4*)(p + 4 * RB));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// two f32 -> two 16-bit values in a word (f32: the largest plane)
template <int DT>
__device__ inline uint32_t pair(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    if constexpr (DT == cgv::DT_FP16) {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), f16x2));
    } else {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
    }
}
// what 16 bits leave of a value
template <int DT>
__device__ inline float rest16(float v) { return v - cgv_ops::half_to_f32<DT>(cgv_ops::f32_to_half<DT>(v)); }
// A lane's rows (x & 3) + 8 (x >> 2) + 4 (lane >> 5), x < 8, of its column in 16 bits -> the column's rows 8 (lane >> 5) + 0 .. 7, which are
// neighbours in memory: the lanes l and l + 32 trade halves. f32: the largest plane, and v keeps what it leaves
template <int DT>
__device__ inline uint4 sixteen(float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = pair<DT>(v[2 * i], v[2 * i + 1]);
        if (DT == cgv::DT_F32) v[2 * i] -= __uint_as_float(w[i] << 16), v[2 * i + 1] -= __uint_as_float(w[i] & 0xffff0000u);
    }
    const auto x = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false), y = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    return make_uint4(x[0], y[0], x[1], y[1]);
}

__device__ inline const char* uniform(const char* p) {
    const uint64_t v = (uint64_t)p;
    return (const char*)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

// tile `i` of workgroup `id`: consecutive tiles run on one XCD (the hardware deals workgroups to the 8 XCDs in turn)
__device__ inline uint32_t unit_of(uint32_t id, uint32_t blocks) {
    const uint32_t x = id & 7u, per = blocks >> 3, extra = blocks & 7u;
    return x * per + min(x, extra) + (id >> 3);
}

#if defined(__HIP_DEVICE_COMPILE__)   // the host pass only needs the launch stubs
template <int DT, class S, bool TA, bool TB, int EPI>
__device__ __forceinline__ void work(const Args& g, uint32_t block) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    constexpr bool UNEVEN = S::UNEVEN, LONG_A = EPI != EPI_DR;
    constexpr int NST = S::STAGES, NSA = UNEVEN && LONG_A ? 3 : NST, NSB = UNEVEN && !LONG_A ? 3 : NST;   // places of A and B
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave % S::WM, wn = wave / S::WM;
    const uint32_t unit = unit_of(block, g.blocks);

    // ---- this workgroup's tiles: LSE and G keep a query tile and walk the corpus; dR walks (element tile, corpus tile); dQ has one
    uint32_t mt, nt, k0 = 0, ksteps = g.ksteps, tiles, split = 0;
    if (EPI == EPI_LSE || EPI == EPI_G) {
        nt = unit % g.tn;
        split = unit / g.tn;
        mt = split;
        tiles = split < g.tm ? (g.tm - split + g.splits - 1) / g.splits : 0;
    } else if (EPI == EPI_DQ) {
        mt = unit % g.tm;
        nt = unit / g.tm % g.tn;
        split = unit / (g.tm * g.tn);
        k0 = (uint32_t)((uint64_t)g.ksteps * split / g.splits);
        ksteps = (uint32_t)((uint64_t)g.ksteps * (split + 1) / g.splits) - k0;
        tiles = 1;
    } else {
        const uint32_t all = g.tm * g.tn;
        mt = nt = 0;
        tiles = unit < all ? (all - unit + g.blocks - 1) / g.blocks : 0;
    }
    auto tile_at = [&](uint32_t i) {
        if (EPI == EPI_LSE || EPI == EPI_G) {
            mt = split + i * g.splits;
        } else if (EPI == EPI_DR) {
            const uint32_t t = unit + i * g.blocks;
            mt = t % g.tm;
            nt = t / g.tm;
        }
    };

    Loader<TA, S::BM, S::NW> la;
    Loader<TB, S::BN, S::NW> lb;
    const char *abase = nullptr, *bbase = nullptr;    // of the tile, plane 0, k = k0
    auto enter = [&](uint32_t i) {
        tile_at(i);
        lb.place(g.b, nt * S::BN, wave, lane, 64);
        abase = g.a.p + (TA ? (uint64_t)mt * S::BM * 2 : (uint64_t)mt * S::BM * g.a.pitch);
        bbase = g.b.p + (TB ? (uint64_t)nt * S::BN * 2 : (uint64_t)nt * S::BN * g.b.pitch);
    };
    // The load side runs ahead of the products, across plane pairs and tiles. prepare() finds out where the next stage comes from: the
    // next 64 elements of the same run of stages, but for a run's ends. Behind the last stage the last one is loaded again: nobody
    // reads it, and the number of loads on the way is always the same.
    uint32_t li = 0, lseg = 0, left = 0;              // tile and plane pair of the next run; stages left in this one
    const char *pa = nullptr, *pb = nullptr;
    uint32_t sa = 0, sb = 0;
    bool clamped = false, part = false;               // the run's last stage is a partial one: is, is still to come
    const uint64_t step_a = TA ? (uint64_t)BK * g.a.pitch : 0, step_b = TB ? (uint64_t)BK * g.b.pitch : 0;
    auto advance = [&]() {
        if (TA) pa += step_a;
        else sa += BK * 2;
        if (TB) pb += step_b;
        else sb += BK * 2;
    };
    const uint32_t rest = (uint32_t)(g.kvalid % BK);
    const bool ends_part = EPI != EPI_DR && rest && (k0 + ksteps) * (uint64_t)BK > g.kvalid;
    auto new_run = [&]() {
        if (part) {
            advance();
            la.place(g.a, mt * S::BM, wave, lane, rest);
            clamped = true;
            part = false;
            return;
        }
        if (li == tiles) return;
        if (lseg == 0) enter(li);
        const uint32_t full = ends_part ? ksteps - 1 : ksteps;
        if (lseg == 0 || clamped) la.place(g.a, mt * S::BM, wave, lane, full ? BK : rest);
        clamped = full == 0;
        part = ends_part && full;
        pa = abase + g.sa[lseg] * g.a.plane + k0 * step_a;
        pb = bbase + g.sb[lseg] * g.b.plane + k0 * step_b;
        sa = TA ? 0 : k0 * BK * 2;
        sb = TB ? 0 : k0 * BK * 2;
        left = full ? full - 1 : 0;
        if (++lseg == g.nseg) lseg = 0, ++li;
    };
    auto prepare = [&]() {
        if (left) {
            --left;
            advance();
        } else {
            new_run();
        }
        // all of this is the same for every lane; said here, because the compiler loses sight of it
        left = __builtin_amdgcn_readfirstlane(left);
        sa = __builtin_amdgcn_readfirstlane(sa);
        sb = __builtin_amdgcn_readfirstlane(sb);
        pa = uniform(pa);
        pb = uniform(pb);
    };
    char *const smem_a = smem, *const smem_b = smem + NSA * S::PL * S::A_BYTES;
    constexpr int AUX = S::ONCE ? 2 : 0;              // of A's loads: nontemporal
    auto issue_a = [&](const Loader<TA, S::BM, S::NW>& l, const char* base, uint32_t off, int slot) {
#pragma unroll
        for (int p = 0; p < S::PL; ++p) l.template issue<AUX>(base + p * g.a.plane, off, smem_a + (slot * S::PL + p) * S::A_BYTES, wave);
    };
    auto issue_b = [&](const Loader<TB, S::BN, S::NW>& l, const char* base, uint32_t off, int slot) {
#pragma unroll
        for (int p = 0; p < S::PL; ++p) l.template issue<0>(base + p * g.b.plane, off, smem_b + (slot * S::PL + p) * S::B_BYTES, wave);
    };
    // UNEVEN: the short operand's stage before the prepared one, still to be loaded (a short B is the same query tile all the time)
    Loader<TA, S::BM, S::NW> wla;
    const char* wp = nullptr;
    uint32_t ws = 0;
    auto keep = [&]() {
        if constexpr (UNEVEN) {
            if (LONG_A) wp = pb, ws = sb;
            else wla = la, wp = pa, ws = sa;
        }
    };
    constexpr int IA = Loader<TA, S::BM, S::NW>::I, IB = Loader<TB, S::BN, S::NW>::I, SHORT = LONG_A ? IB : IA;
    // load q of those that follow when the places (a, b) become free: of the prepared stage, UNEVEN: the short operand's kept stage first
    auto issue_one = [&](int q, int a, int b) {
        if constexpr (UNEVEN) {
            if (q < SHORT) {
                if (LONG_A) lb.template issue_one<0>(q, wp, ws, smem_b + b * S::B_BYTES, wave);
                else wla.template issue_one<AUX>(q, wp, ws, smem_a + a * S::A_BYTES, wave);
            } else {
                if (LONG_A) la.template issue_one<AUX>(q - SHORT, pa, sa, smem_a + a * S::A_BYTES, wave);
                else lb.template issue_one<0>(q - SHORT, pb, sb, smem_b + b * S::B_BYTES, wave);
            }
        } else {
            if (q < IA) la.template issue_one<AUX>(q, pa, sa, smem_a + a * S::A_BYTES, wave);
            else lb.template issue_one<0>(q - IA, pb, sb, smem_b + b * S::B_BYTES, wave);
        }
    };
    auto issue = [&](int a, int b) {
        issue_a(la, pa, sa, a);
        issue_b(lb, pb, sb, b);
    };

    float g_coef[S::NB];                              // G: of the lane's queries
    float2 g_lse[S::NB];
    if (EPI == EPI_G)
        for (int nb = 0; nb < S::NB; ++nb) {
            const uint32_t q = nt * S::BN + wn * S::TN + nb * 32 + (lane & 31);
            g_coef[nb] = q < g.n_valid ? g.coef[q] : 0.0f;
            g_lse[nb] = q < g.n_valid ? g.lse2[q] : make_float2(0.0f, 0.0f);
        }
    // LSE: per query of the lane, over the corpus rows of the lane: maximum, sum, and what the sum's additions lost. Where scores are alike all
    // additions round the same way, and a query's share may be the whole corpus: a chain of single exponentials was off by 1.4e-3 of the sum (33 000
    // queries, 300 k equal rows). So a tile's are added up apart (16 a block, then the blocks), and adding a tile to the rest loses nothing. The
    // maximum is rounded up to an integer: moving to a new one multiplies by a power of two, which is exact however often it happens
    float run_m[S::NB], run_s[S::NB], run_r[S::NB];
    if (EPI == EPI_LSE)
        for (int nb = 0; nb < S::NB; ++nb) run_m[nb] = -INFINITY, run_s[nb] = run_r[nb] = 0.0f;

    // A small wave tile has few products per read: it keeps the fragments of two whole stages and reads the next one while it
    // multiplies this one; a large one keeps those of two times 16 elements of K
    constexpr bool SMALL = S::MB * S::NB <= 2 && S::PL == 1;
    constexpr int SETS = SMALL ? 4 : 1, FA = S::PL * S::MB, FB = S::PL * S::NB;
    s16x8 fa0[SETS][FA], fb0[SETS][FB], fa1[SETS][FA], fb1[SETS][FB];
    f32x16 acc[S::MB][S::NB], low[S::PL == 3 ? S::MB : 1][S::PL == 3 ? S::NB : 1];   // three planes: the five small products have their own sum
    auto read = [&](s16x8(&fa)[FA], s16x8(&fb)[FB], int a, int b, int kk) {
#pragma unroll
        for (int p = 0; p < S::PL; ++p) {
#pragma unroll
            for (int nb = 0; nb < S::NB; ++nb)
                fb[p * S::NB + nb] = fragment<TB, S::BN>(smem_b + (b * S::PL + p) * S::B_BYTES, (uint32_t)(wn * S::TN + nb * 32), kk, lane);
#pragma unroll
            for (int mb = 0; mb < S::MB; ++mb)
                fa[p * S::MB + mb] = fragment<TA, S::BM>(smem_a + (a * S::PL + p) * S::A_BYTES, (uint32_t)(wm * S::TM + mb * 32), kk, lane);
        }
    };
    // the fragments that are read in gap x of a phase, the first in gap `from`
    auto read_at = [&](int x, int from, s16x8(&fa)[FA], s16x8(&fb)[FB], int a, int b, int kk) {
        constexpr int N = FA + FB, P = S::MB * S::NB;
#pragma unroll
        for (int f = 0; f < N; ++f) {
            if (x != from + f * (P - 1 - from) / N) continue;
            if (f == 0 || (f > 1 && f <= FB)) {
                const int nb = f ? f - 1 : 0;
                fb[nb] = fragment<TB, S::BN>(smem_b + b * S::B_BYTES, (uint32_t)(wn * S::TN + nb * 32), kk, lane);
            } else {
                const int mb = f == 1 ? 0 : f - FB;
                fa[mb] = fragment<TA, S::BM>(smem_a + a * S::A_BYTES, (uint32_t)(wm * S::TM + mb * 32), kk, lane);
            }
        }
    };
    auto products = [&](s16x8(&fa)[FA], s16x8(&fb)[FB]) {
        if constexpr (S::PL == 3) {
            constexpr int x[6] = {2, 0, 0, 1, 1, 0}, y[6] = {0, 2, 0, 1, 0, 1};
#pragma unroll
            for (int i = 0; i < 6; ++i)
#pragma unroll
                for (int mb = 0; mb < S::MB; ++mb)
#pragma unroll
                    for (int nb = 0; nb < S::NB; ++nb) {
                        f32x16& c = x[i] + y[i] ? low[mb][nb] : acc[mb][nb];
                        c = mma<DT>(fa[x[i] * S::MB + mb], fb[y[i] * S::NB + nb], c);
                    }
        } else {
#pragma unroll
            for (int mb = 0; mb < S::MB; ++mb)
#pragma unroll
                for (int nb = 0; nb < S::NB; ++nb) acc[mb][nb] = mma<DT>(fa[mb], fb[nb], acc[mb][nb]);
        }
    };
    constexpr bool PLACED = !SMALL && S::NW == 8;
    constexpr int LOADS = S::PL * (IA + IB);                                  // of a stage
    constexpr int FIRST = UNEVEN ? SHORT : (LOADS + 2) / 3;                   // of those that follow right behind the stage's change
    constexpr int WAIT = UNEVEN ? IA + IB - SHORT : (NST - 2) * LOADS;        // of what lies behind the next stage
    // dR: the results of a whole wave tile are at least STORED stores (16 bytes a lane is the widest there is). They count like loads and in
    // turn with them; the first stage behind them needs only what was issued before them, and so does not wait for them (1024 x 125 k x
    // 768 bf16: 235 -> 219 us; G, with the same, gains nothing)
    constexpr int STORED = EPI == EPI_DR && DT != cgv::DT_F32 && UNEVEN ? 2 * S::MB * S::NB : 0;
    bool stored = false;
    auto stage_ready = [&]() {
        // this wave's part of the next stage has landed, its reads of this one are done
        if (STORED && stored) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(WAIT + STORED) : "memory");
        else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(WAIT) : "memory");
        stored = false;
        __builtin_amdgcn_s_barrier();                                 // everybody's: the next stage can be read, this one overwritten
        asm volatile("" ::: "memory");
    };

    constexpr int PRODUCTS = S::MB * S::NB * (S::PL == 3 ? 6 : 1), READS = FA * (TA ? 2 : 1) + FB * (TB ? 2 : 1);
    // the order of a phase: behind each of the first matrix instructions come a few reads of the next fragments, then the loads
    auto interleave = [&](int loads) {
        constexpr int each = PRODUCTS > 2 ? (READS + PRODUCTS - 3) / (PRODUCTS - 2) : READS;
        const int per = (loads + PRODUCTS - 1) / PRODUCTS;
#pragma unroll
        for (int x = 0; x < PRODUCTS; ++x) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, each, 0);
            if (per == 1) __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
            if (per == 2) __builtin_amdgcn_sched_group_barrier(0x010, 2, 0);
            if (per > 2) __builtin_amdgcn_sched_group_barrier(0x010, 5, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };

    if (!ksteps) tiles = EPI == EPI_DQ ? tiles : 0;
    int buf = 0, bufb = 0;                            // places of the stage at work; when it is done the next loads go there
    auto after = [](int x, int n) { return n == 2 ? x ^ 1 : x + 1 == n ? 0 : x + 1; };
    auto read_stage = [&](s16x8(&fa)[SETS][FA], s16x8(&fb)[SETS][FB], int slot) {
#pragma unroll
        for (int kk = 0; kk < SETS; ++kk) read(fa[kk], fb[kk], slot, slot, kk);
    };
    // small wave tiles: a stage's products while the next stage's fragments are read
    auto step = [&](s16x8(&ca)[SETS][FA], s16x8(&cb)[SETS][FB], s16x8(&na)[SETS][FA], s16x8(&nb)[SETS][FB]) {
        __builtin_amdgcn_sched_barrier(0);
        prepare();
        stage_ready();
        const int next = after(buf, NST);
        read_stage(na, nb, next);
        issue(buf, buf);
        buf = next;
#pragma unroll
        for (int kk = 0; kk < SETS; ++kk) products(ca[kk], cb[kk]);
        __builtin_amdgcn_sched_barrier(0);
    };
    if (tiles && ksteps) {
        if constexpr (UNEVEN) {
            prepare();
            issue_a(la, pa, sa, 0);
            issue_b(lb, pb, sb, 0);
            prepare();
            if (LONG_A) issue_a(la, pa, sa, 1);
            else issue_b(lb, pb, sb, 1);
            keep();
            prepare();
            stage_ready();
            for (int q = 0; q < SHORT; ++q) issue_one(q, NSA - 1, NSB - 1);
        } else {
            for (int x = 0; x < NST - 1; ++x) {
                prepare();
                issue(x, x);
            }
            prepare();
            stage_ready();
            if (PLACED)
                for (int q = 0; q < FIRST; ++q) issue_one(q, NST - 1, NST - 1);
            else
                issue(NST - 1, NST - 1);
        }
        read_stage(fa0, fb0, 0);
    }
    // Large wave tiles: products one by one, and between them what is issued beside them. The compiler moves matrix instructions as it likes,
    // so that empty asm statements tie each to its place: behind one that has its result, before one that has an operand of the next
    auto phase = [&](s16x8(&fa)[FA], s16x8(&fb)[FB], auto&& gap) {
        constexpr auto col = [](int x) { return x / S::NB % 2 ? S::NB - 1 - x % S::NB : x % S::NB; };   // neighbours share an operand
#pragma unroll
        for (int x = 0; x < S::MB * S::NB; ++x) {
            f32x16& c = acc[x / S::NB][col(x)];
            c = mma<DT>(fa[x / S::NB], fb[col(x)], c);
            asm volatile("" : "+v"(c)::"memory");
            gap(x);
            if (x + 1 < S::MB * S::NB) {
                if ((x + 1) / S::NB != x / S::NB) asm volatile("" : "+v"(fa[(x + 1) / S::NB])::"memory");
                else asm volatile("" : "+v"(fb[col(x + 1)])::"memory");
            }
        }
    };
    // loads q .. q + n - 1 spread over the gaps of a phase, behind the fragments' reads
    auto loads_at = [&](int x, int q, int n, int a, int b) {
        constexpr int P = S::MB * S::NB, from = P >= 8 ? 3 : P >= 6 ? 2 : 1;
#pragma unroll
        for (int d = 0; d < n; ++d)
            if (x == from + d * (P - from) / n) issue_one(q + d, a, b);
    };
    auto placed_step = [&]() {
        constexpr int P0 = (LOADS - FIRST + 1) / 2, P1 = LOADS - FIRST - P0;
        const int fra = buf ? buf - 1 : NSA - 1, frb = bufb ? bufb - 1 : NSB - 1;        // places that the stage before has left
        phase(fa0[0], fb0[0], [&](int x) {
            read_at(x, 0, fa1[0], fb1[0], buf, bufb, 1);
            loads_at(x, FIRST, P0, fra, frb);
        });
        phase(fa1[0], fb1[0], [&](int x) {
            read_at(x, 0, fa0[0], fb0[0], buf, bufb, 2);
            loads_at(x, FIRST + P0, P1, fra, frb);
        });
        phase(fa0[0], fb0[0], [&](int x) {
            read_at(x, 0, fa1[0], fb1[0], buf, bufb, 3);
        });
        keep();
        prepare();
        const int a = after(buf, NSA), b = after(bufb, NSB);
        // the stage changes behind the first product of its last 16 elements, whose fragments have been read
        phase(fa1[0], fb1[0], [&](int x) {
            if (x == 0) stage_ready();
            read_at(x, 1, fa0[0], fb0[0], a, b, 0);
            loads_at(x, 0, FIRST, buf, bufb);
        });
        buf = a;
        bufb = b;
    };
    // four waves, one a SIMD: the same in the compiler's order, which suits them better (64 queries x 200 k x 768, loss: 82 us, placed 120)
    auto ordered_step = [&]() {
        __builtin_amdgcn_sched_barrier(0);
        read(fa1[0], fb1[0], buf, bufb, 1);
        products(fa0[0], fb0[0]);
        interleave(0);
        read(fa0[0], fb0[0], buf, bufb, 2);
        products(fa1[0], fb1[0]);
        interleave(0);
        read(fa1[0], fb1[0], buf, bufb, 3);
        products(fa0[0], fb0[0]);
        interleave(0);
        prepare();
        stage_ready();
        const int next = after(buf, NST);
        read(fa0[0], fb0[0], next, next, 0);
        issue(buf, bufb);
        buf = bufb = next;
        products(fa1[0], fb1[0]);
        interleave(LOADS);
    };
    uint32_t nmt = mt, nnt = nt;
    for (uint32_t i = 0; i < tiles; ++i) {
        // (mt, nt) belong to the load side, which may already be in the next tile
        if (EPI == EPI_LSE || EPI == EPI_G) {
            nmt = split + i * g.splits;
        } else if (EPI == EPI_DR) {
            const uint32_t t = unit + i * g.blocks;
            nmt = t % g.tm;
            nnt = t / g.tm;
        }
        const uint32_t my_mt = nmt, my_nt = nnt, stages = g.nseg * ksteps;
        uint32_t l0 = 0, l1 = 0;                      // DR: listed entries of the wave's corpus rows, asked for long before they are needed
        if (EPI == EPI_DR && DT != cgv::DT_F32 && g.ent_start) {
            const auto* start = (const __attribute__((address_space(4))) uint32_t*)g.ent_start;
            const uint32_t at = (my_nt * S::BN + wn * S::TN) / 32;
            l0 = start[min(at, g.ent_groups)];
            l1 = start[min(at + S::TN / 32, g.ent_groups)];
        }
#pragma unroll
        for (int mb = 0; mb < S::MB; ++mb)
#pragma unroll
            for (int nb = 0; nb < S::NB; ++nb)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    acc[mb][nb][r] = 0.0f;
                    if (S::PL == 3) low[mb][nb][r] = 0.0f;
                }
        if constexpr (SMALL) {
            uint32_t s = 0;
            for (; s + 2 <= stages; s += 2) {
                step(fa0, fb0, fa1, fb1);
                step(fa1, fb1, fa0, fb0);
            }
            if (s < stages) {
                step(fa0, fb0, fa1, fb1);
#pragma unroll
                for (int kk = 0; kk < SETS; ++kk) {
#pragma unroll
                    for (int mb = 0; mb < S::MB; ++mb) fa0[kk][mb] = fa1[kk][mb];
#pragma unroll
                    for (int nb = 0; nb < S::NB; ++nb) fb0[kk][nb] = fb1[kk][nb];
                }
            }
        } else {
            for (uint32_t s = 0; s < stages; ++s) {
                if constexpr (PLACED) placed_step();
                else ordered_step();
            }
            if constexpr (S::PL == 3) {
#pragma unroll
                for (int mb = 0; mb < S::MB; ++mb)
#pragma unroll
                    for (int nb = 0; nb < S::NB; ++nb) acc[mb][nb] += low[mb][nb];
            }
        }

        // ---- epilogue of the tile
        const uint32_t m0 = my_mt * S::BM + wm * S::TM, n0 = my_nt * S::BN + wn * S::TN;
        const uint32_t half4 = (uint32_t)(lane >> 5) * 4;
        if (EPI == EPI_LSE) {
            const bool edge = m0 + S::TM > g.m_valid;
#pragma unroll
            for (int nb = 0; nb < S::NB; ++nb) {
                const uint32_t q = n0 + nb * 32 + (lane & 31);
                // corpus row that this query leaves out, as a row of the wave's part of the tile
                const uint32_t skip = q < g.n_valid ? g.anchor[q] - (uint32_t)(g.row0 + m0) : 0xffffffffu;
                const bool any = __ballot(skip < (uint32_t)S::TM) != 0;
                if (edge || any) {                     // rows beyond the corpus, the row left out: a score of -inf (scale2 is not zero)
                    const float none = g.scale2 > 0.0f ? -INFINITY : INFINITY;
#pragma unroll
                    for (int mb = 0; mb < S::MB; ++mb)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const uint32_t m = mb * 32 + (r & 3) + 8 * (r >> 2) + half4;
                            if (m == skip || m0 + m >= g.m_valid) acc[mb][nb][r] = none;
                        }
                }
                float ext = acc[0][nb][0];
                if (g.scale2 >= 0.0f) {
#pragma unroll
                    for (int mb = 0; mb < S::MB; ++mb)
#pragma unroll
                        for (int r = 0; r < 16; ++r) ext = fmaxf(ext, acc[mb][nb][r]);
                } else {
#pragma unroll
                    for (int mb = 0; mb < S::MB; ++mb)
#pragma unroll
                        for (int r = 0; r < 16; ++r) ext = fminf(ext, acc[mb][nb][r]);
                }
                const float nm = fmaxf(run_m[nb], ceilf(ext * g.scale2)), base = nm == -INFINITY ? 0.0f : nm;
                const float f = __builtin_amdgcn_exp2f(run_m[nb] - base), before = run_s[nb] * f;
                float sum[S::MB];                      // of the tile: a lane's 16 rows of a block
#pragma unroll
                for (int mb = 0; mb < S::MB; ++mb) {
                    sum[mb] = 0.0f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) sum[mb] += __builtin_amdgcn_exp2f(fmaf(acc[mb][nb][r], g.scale2, -base));
                    if (mb) sum[0] += sum[mb];
                }
                const float s = before + sum[0], b = s - before;
                run_m[nb] = nm;
                run_s[nb] = s;
                run_r[nb] = fmaf(run_r[nb], f, (before - (s - b)) + (sum[0] - b));
            }
        } else if (EPI == EPI_G) {
            auto store = [&](auto at_edge) {
#pragma unroll
                for (int nb = 0; nb < S::NB; ++nb) {
                    const uint32_t q = n0 + nb * 32 + (lane & 31);
                    char* const o = g.out + q * g.out_pitch + (uint64_t)(m0 + (lane >> 5) * 8) * 2;
#pragma unroll
                    for (int mb = 0; mb < S::MB; ++mb)
#pragma unroll
                        for (int p = 0; p < 2; ++p) {
                            float v[8];
#pragma unroll
                            for (int x = 0; x < 8; ++x) {
                                const float t = fmaf(acc[mb][nb][p * 8 + x], g.scale2, -g_lse[nb].x);
                                // the second part of the logarithm is below the roundings of 16 bits
                                v[x] = g_coef[nb] * __builtin_amdgcn_exp2f(DT == cgv::DT_F32 ? t - g_lse[nb].y : t);
                                const uint32_t m = m0 + mb * 32 + p * 16 + (x & 3) + 8 * (x >> 2) + half4;
                                if (g_coef[nb] == 0.0f || (decltype(at_edge)::value && m >= g.m_valid)) v[x] = 0.0f;
                                if (DT != cgv::DT_F32 && g.twin && q >= g.twin) v[x] = rest16<DT>(v[x]);
                            }
#pragma unroll
                            for (uint32_t plane = 0; plane < (DT == cgv::DT_F32 ? 3u : 1u); ++plane) {
                                const uint4 w = sixteen<DT>(v);
                                if (q < g.n_pad) *(uint4*)(o + plane * g.out_plane + (mb * 32 + p * 16) * 2) = w;
                            }
                        }
                }
            };
            if (m0 + S::TM > g.m_valid) store(std::true_type());
            else store(std::false_type());
        } else if (EPI == EPI_DQ) {
            float* out = (float*)(g.out + split * g.out_plane);
#pragma unroll
            for (int nb = 0; nb < S::NB; ++nb) {
                const uint32_t q = n0 + nb * 32 + (lane & 31);
#pragma unroll
                for (int mb = 0; mb < S::MB; ++mb)
#pragma unroll
                    for (int r4 = 0; r4 < 4; ++r4) {
                        const uint32_t m = m0 + mb * 32 + r4 * 8 + half4;
                        if (q < g.n_valid && m < g.m_valid) {
                            float4* p = (float4*)(out + (uint64_t)q * g.part_ld + m);
                            float4 v = make_float4(acc[mb][nb][r4 * 4], acc[mb][nb][r4 * 4 + 1], acc[mb][nb][r4 * 4 + 2], acc[mb][nb][r4 * 4 + 3]);
                            if (g.accumulate) {
                                const float4 o = *p;
                                v = make_float4(v.x + o.x, v.y + o.y, v.z + o.z, v.w + o.w);
                            }
                            *p = v;
                        }
                    }
            }
        } else {   // EPI_DR
            const float u = g.unscale ? *g.unscale : 1.0f;
            stored = g.vec_out && m0 + S::TM <= g.m_valid && n0 + S::TN <= g.n_valid;
            if (DT != cgv::DT_F32 && S::MB == 1 && g.ent_n) {
                // what 16 bits leave of the listed entries of G, in the order of the list: eight times 64 of them looked through at a time
                constexpr uint32_t AT_ONCE = 8;
                for (uint32_t e0 = 0; e0 < g.ent_n; e0 += 64 * AT_ONCE) {
                    uint32_t at[AT_ONCE];
#pragma unroll
                    for (uint32_t x = 0; x < AT_ONCE; ++x) {
                        const uint32_t e = e0 + x * 64 + lane;
                        at[x] = e < g.ent_n ? g.ent_id[e] - (uint32_t)(g.row0 + n0) : 0xffffffffu;       // column of the wave tile, or beyond it
                    }
#pragma unroll
                    for (uint32_t x = 0; x < AT_ONCE; ++x)
                        for (uint64_t hits = __ballot(at[x] < (uint32_t)S::TN); hits; hits &= hits - 1) {
                            const int l = __ffsll((unsigned long long)hits) - 1;
                            const uint32_t e = e0 + x * 64 + l, c = __builtin_amdgcn_readlane(at[x], l);
                            const float rest = rest16<DT>(g.ent_val[e]), mine = (uint32_t)(lane & 31) == (c & 31u) ? rest : 0.0f;
                            const char* row = g.a.p + (uint64_t)(e / g.ent_k) * g.a.pitch;
#pragma unroll
                            for (int mb = 0; mb < S::MB; ++mb)
#pragma unroll
                                for (int r4 = 0; r4 < 4; ++r4) {
                                    const uint2 w = *(const uint2*)(row + min(m0 + mb * 32 + r4 * 8 + half4, g.a.limit - 4) * 2);
                                    const float q[4] = {cgv_ops::half_to_f32<DT>((uint16_t)w.x), cgv_ops::half_to_f32<DT>((uint16_t)(w.x >> 16)),
                                                        cgv_ops::half_to_f32<DT>((uint16_t)w.y), cgv_ops::half_to_f32<DT>((uint16_t)(w.y >> 16))};
#pragma unroll
                                    for (int nb = 0; nb < S::NB; ++nb)
                                        if (nb == (int)(c / 32))
#pragma unroll
                                            for (int y = 0; y < 4; ++y) acc[mb][nb][r4 * 4 + y] = fmaf(mine, q[y], acc[mb][nb][r4 * 4 + y]);
                                }
                        }
                }
            }
            if constexpr (DT != cgv::DT_F32) {
                // the same with entries sorted by corpus row: 16 of them are K of one more product, queries' rows times what is left of each in its column
                for (uint32_t l = l0; l < l1; l += 16) {
                    uint32_t query = 0, word = 0xffff0000u;           // of entry l + (lane & 15): its query; column of the wave tile, and what is left
                    if (l + (lane & 15) < l1) {
                        const uint32_t e = g.ent_pos[l + (lane & 15)], c = g.ent_id[e] - (uint32_t)(g.row0 + n0);
                        query = e / g.ent_k;
                        if (c < (uint32_t)S::TN) word = c << 16 | cgv_ops::f32_to_half<DT>(rest16<DT>(g.ent_val[e]));
                    }
                    s16x8 fb[S::NB];
                    uint64_t from[8];
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        const int of = (lane >> 5) * 8 + x;
                        const uint32_t w = __shfl(word, of);
                        from[x] = (uint64_t)__shfl(query, of) * g.a.pitch;
#pragma unroll
                        for (int nb = 0; nb < S::NB; ++nb) fb[nb][x] = (short)(w >> 16 == (uint32_t)(nb * 32 + (lane & 31)) ? w & 0xffffu : 0u);
                    }
#pragma unroll
                    for (int mb = 0; mb < S::MB; ++mb) {
                        const char* q = g.a.p + min(m0 + mb * 32 + (lane & 31), g.a.limit - 1) * 2;
                        s16x8 fa;
#pragma unroll
                        for (int x = 0; x < 8; ++x) fa[x] = *(const short*)(q + from[x]);
#pragma unroll
                        for (int nb = 0; nb < S::NB; ++nb) acc[mb][nb] = mma<DT>(fa, fb[nb], acc[mb][nb]);
                    }
                }
            }
#pragma unroll
            for (int nb = 0; nb < S::NB; ++nb) {
                const uint32_t row = n0 + nb * 32 + (lane & 31);
                if (DT != cgv::DT_F32 && g.vec_out) {
                    char* const o = g.out + row * g.out_pitch;
#pragma unroll
                    for (int mb = 0; mb < S::MB; ++mb)
#pragma unroll
                        for (int p = 0; p < 2; ++p) {
                            float v[8];
#pragma unroll
                            for (int x = 0; x < 8; ++x) v[x] = acc[mb][nb][p * 8 + x] * u;
                            const uint4 w = sixteen<DT>(v);
                            const uint32_t m = m0 + mb * 32 + p * 16 + (lane >> 5) * 8;
                            if (row < g.n_valid && m < g.m_valid) *(uint4*)(o + m * 2) = w;      // m_valid: a multiple of 8
                        }
                } else {
#pragma unroll
                    for (int mb = 0; mb < S::MB; ++mb)
#pragma unroll
                        for (int r4 = 0; r4 < 4; ++r4) {
                            const uint32_t m = m0 + mb * 32 + r4 * 8 + half4;
                            if (row < g.n_valid && m < g.m_valid) {
                                char* p = g.out + row * g.out_pitch;
                                float v[4];
                                for (int x = 0; x < 4; ++x) v[x] = acc[mb][nb][r4 * 4 + x] * u;
                                if (DT == cgv::DT_F32 && g.vec_out) {
                                    *(float4*)(p + m * 4) = make_float4(v[0], v[1], v[2], v[3]);
                                } else {
                                    for (int x = 0; x < 4; ++x)
                                        if (m + x < g.m_valid) {
                                            if (DT == cgv::DT_F32) ((float*)p)[m + x] = v[x];
                                            else ((uint16_t*)p)[m + x] = DT == cgv::DT_FP16 ? cgv::f32_to_f16_rne(v[x]) : cgv::f32_to_bf16_rne(v[x]);
                                        }
                                }
                            }
                        }
                }
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // nothing may land in LDS behind the workgroup's end
    if (EPI == EPI_LSE) {
        const uint32_t n0 = nt * S::BN + wn * S::TN;
#pragma unroll
        for (int nb = 0; nb < S::NB; ++nb) {
            const float mine = run_s[nb] + run_r[nb], om = __shfl_xor(run_m[nb], 32), os = __shfl_xor(mine, 32);
            const float nm = fmaxf(run_m[nb], om), base = nm == -INFINITY ? 0.0f : nm;
            const float s = mine * __builtin_amdgcn_exp2f(run_m[nb] - base) + os * __builtin_amdgcn_exp2f(om - base);
            const uint32_t q = n0 + nb * 32 + (lane & 31);
            const uint32_t own = split * S::WM + wm;
            if (lane < 32 && q < g.n_pad) {
                g.part[(uint64_t)own * g.part_ld + q] = make_float2(nm, s);
                for (uint32_t x = own + g.splits * S::WM; x < g.slots; x += g.splits * S::WM)      // other columns have more
                    g.part[(uint64_t)x * g.part_ld + q] = make_float2(-INFINITY, 0.0f);
            }
        }
    }
    if (EPI == EPI_G) {
        // the listed rows' entries, computed apart, take the place of what this workgroup has stored for them: every wave's stores are done
        __syncthreads();
        const uint32_t n0 = nt * S::BN, queries = min((uint32_t)S::BN, g.n_valid - n0);
        const uint32_t* ids = g.ent_id + (uint64_t)n0 * g.ent_k;
        const float* vals = g.ent_val + (uint64_t)n0 * g.ent_k;
        for (uint32_t t0 = threadIdx.x; t0 < queries * g.ent_k; t0 += 8 * S::THREADS) {
            uint32_t id[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) id[x] = t0 + x * S::THREADS < queries * g.ent_k ? ids[t0 + x * S::THREADS] : 0xffffffffu;
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                const uint64_t m = (uint64_t)id[x] - g.row0;                // none: beyond every piece; earlier pieces: wraps round
                if (m >= g.m_valid || (uint32_t)m / S::BM % g.splits != split) continue;
                const uint32_t t = t0 + x * S::THREADS;
                uint16_t* o = (uint16_t*)(g.out + (n0 + t / g.ent_k) * g.out_pitch) + m;
                const float v = vals[t];
                if (DT == cgv::DT_F32) {
                    uint16_t p[3];
                    split3(v, p);
                    for (int i = 0; i < 3; ++i) o[i * (g.out_plane / 2)] = p[i];
                } else {
                    *o = cgv_ops::f32_to_half<DT>(g.twin && n0 + t / g.ent_k >= g.twin ? rest16<DT>(v) : v);
                }
            }
        }
    }
}
#endif

template <int DT, class S, bool TA, bool TB, int EPI>
static __global__ __launch_bounds__(S::THREADS) void gemm_kernel(const Args g) {
#if defined(__HIP_DEVICE_COMPILE__)
    work<DT, S, TA, TB, EPI>(g, blockIdx.x);
#endif
}

// columns of two widths: `a` with tiles of shape S, `b` with tiles of shape T
template <int DT, class S, class T, bool TA, bool TB, int EPI>
static __global__ __launch_bounds__(S::THREADS) void mixed_kernel(const Args a, const Args b) {
#if defined(__HIP_DEVICE_COMPILE__)
    static_assert(S::THREADS == T::THREADS, "one workgroup size");
    if (blockIdx.x < a.blocks) work<DT, S, TA, TB, EPI>(a, blockIdx.x);
    else work<DT, T, TA, TB, EPI>(b, blockIdx.x - a.blocks);
#endif
}

// dQ and dR, which share nothing but their input, in one launch
template <int DT, class S>
static __global__ __launch_bounds__(S::THREADS) void gradients_kernel(const Args q, const Args r) {
#if defined(__HIP_DEVICE_COMPILE__)
    if (blockIdx.x < q.blocks) work<DT, S, true, false, EPI_DQ>(q, blockIdx.x);
    else work<DT, S, true, true, EPI_DR>(r, blockIdx.x - q.blocks);
#endif
}

}  // namespace cgv_gemm
