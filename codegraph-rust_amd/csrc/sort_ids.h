// sort_ids.h - (id, position) sorted by id, stably: what lookup.hip sums a table's gradient by, and softmax.hip finds the listed rows by (there
// by groups of ids: 2^down ids have one key). By one workgroup up to SMALL_SORT ids; more by radix, 11 bits at most a pass, three launches each. Ids outside [0, n_rows) come last.
#pragma once
#include "ops_common.h"

namespace cgv_ops {
namespace {

// One workgroup's sort against the radix passes, six launches: 1000 ids 23 and 30 us, 2000 ids 30 and 31, 4000 ids 46 and 33
constexpr uint32_t SMALL_SORT = 2048;
constexpr uint32_t SORT_THREADS = 256, SORT_STEPS = 4, SORT_BLOCK = SORT_THREADS * SORT_STEPS;   // elements of a workgroup
constexpr uint32_t MAX_DIGIT = 11;

// strangers go behind the last row
__device__ inline uint32_t key_of(int64_t id, uint32_t n_rows, uint32_t down) {
    return id >= 0 && id < (int64_t)n_rows ? (uint32_t)id >> down : (n_rows + (1u << down) - 1) >> down;
}

struct SortPass {
    const int64_t* ids;             // first pass: keys come from here
    const uint32_t *keys, *pos;     // later passes
    uint32_t *keys_out, *pos_out;
    uint32_t *hist, *total;         // [bins][blocks], [bins]
    uint32_t n, n_rows, down, blocks, shift, bits;
    __device__ uint32_t key(uint32_t i) const { return ids ? key_of(ids[i], n_rows, down) : keys[i]; }
    __device__ uint32_t digit(uint32_t k) const { return (k >> shift) & ((1u << bits) - 1u); }
};

// counts of a workgroup's digits; the first pass clears the rows' run ends on the way, with further workgroups for many rows
// (gradient of 1M x 64 bf16 by 1000 ids: 164 us with the one workgroup of the ids alone, 59 with 245)
__global__ __launch_bounds__(SORT_THREADS) void sort_count_kernel(SortPass p, uint64_t* __restrict__ runs) {
    if (runs)
        for (uint64_t i = (uint64_t)blockIdx.x * SORT_THREADS + threadIdx.x; i < p.n_rows; i += (uint64_t)gridDim.x * SORT_THREADS) runs[i] = 0;
    if (blockIdx.x >= p.blocks) return;
    __shared__ uint32_t h[1u << MAX_DIGIT];
    const uint32_t bins = 1u << p.bits;
    for (uint32_t i = threadIdx.x; i < bins; i += SORT_THREADS) h[i] = 0;
    __syncthreads();
    const uint32_t lo = blockIdx.x * SORT_BLOCK;
    for (uint32_t s = 0; s < SORT_STEPS; ++s) {
        const uint32_t i = lo + s * SORT_THREADS + threadIdx.x;
        if (i < p.n) atomicAdd(&h[p.digit(p.key(i))], 1u);
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < bins; i += SORT_THREADS) p.hist[(uint64_t)i * p.blocks + blockIdx.x] = h[i];
}

// one wave per digit: where each workgroup's elements of that digit start among those of the digit
__global__ __launch_bounds__(256) void sort_scan_kernel(SortPass p) {
    const uint32_t bin = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (bin >= (1u << p.bits)) return;
    uint32_t* h = p.hist + (uint64_t)bin * p.blocks;
    uint32_t carry = 0;
    for (uint32_t a = 0; a < p.blocks; a += 64) {
        const uint32_t v = a + lane < p.blocks ? h[a + lane] : 0u;
        uint32_t s = v;
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t t = __shfl_up(s, o);
            if ((int)lane >= o) s += t;
        }
        if (a + lane < p.blocks) h[a + lane] = carry + s - v;
        carry += __shfl(s, 63);
    }
    if (lane == 0) p.total[bin] = carry;
}

__global__ __launch_bounds__(SORT_THREADS) void sort_scatter_kernel(SortPass p) {
    constexpr uint32_t W = SORT_THREADS / 64;
    __shared__ uint32_t next[W][1u << MAX_DIGIT];     // where the wave's next element of a digit goes
    __shared__ uint32_t part[SORT_THREADS];
    const uint32_t bins = 1u << p.bits, tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
    for (uint32_t i = tid; i < W * bins; i += SORT_THREADS) next[i / bins][i % bins] = 0;
    __syncthreads();
    const uint32_t lo = blockIdx.x * SORT_BLOCK + w * (SORT_STEPS * 64);
    uint32_t k[SORT_STEPS];
#pragma unroll
    for (uint32_t s = 0; s < SORT_STEPS; ++s) {
        const uint32_t i = lo + s * 64 + lane;
        k[s] = i < p.n ? p.key(i) : 0u;
        if (i < p.n) atomicAdd(&next[w][p.digit(k[s])], 1u);
    }
    // totals of the digits -> where each digit starts: every thread sums its stretch, the stretches are scanned
    const uint32_t per = (bins + SORT_THREADS - 1) / SORT_THREADS, b0 = tid * per;
    uint32_t sum = 0;
    for (uint32_t j = 0; j < per; ++j)
        if (b0 + j < bins) sum += p.total[b0 + j];
    part[tid] = sum;
    __syncthreads();
    for (uint32_t o = 1; o < SORT_THREADS; o <<= 1) {
        const uint32_t t = tid >= o ? part[tid - o] : 0u;
        __syncthreads();
        part[tid] += t;
        __syncthreads();
    }
    uint32_t start = part[tid] - sum;
    for (uint32_t j = 0; j < per; ++j) {
        const uint32_t b = b0 + j;
        if (b >= bins) break;
        uint32_t at = start + p.hist[(uint64_t)b * p.blocks + blockIdx.x];
        start += p.total[b];
        for (uint32_t x = 0; x < W; ++x) {
            const uint32_t c = next[x][b];
            next[x][b] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t s = 0; s < SORT_STEPS; ++s) {
        const uint32_t i = lo + s * 64 + lane;
        const bool on = i < p.n;
        const uint32_t d = p.digit(k[s]);
        uint64_t same = __ballot(on);
        for (uint32_t b = 0; b < p.bits; ++b) {
            const bool bit = (d >> b) & 1u;
            const uint64_t m = __ballot(bit);
            same &= bit ? m : ~m;
        }
        const uint32_t before = __popcll(same & ((1ull << lane) - 1));
        uint32_t to = 0;
        if (on) to = ((volatile uint32_t*)next[w])[d] + before;
        __builtin_amdgcn_wave_barrier();
        if (on && before == 0) ((volatile uint32_t*)next[w])[d] = to + (uint32_t)__popcll(same);
        __builtin_amdgcn_wave_barrier();
        if (on) {
            p.keys_out[to] = k[s];
            p.pos_out[to] = p.ids ? i : p.pos[i];
        }
    }
}

// up to SMALL_SORT ids: one workgroup sorts (key, position) in its LDS, in the order of a bitonic network - positions differ, so the order is
// the stable one -, and the others clear the rows' run ends
__global__ __launch_bounds__(1024) void sort_small_kernel(const int64_t* __restrict__ ids, uint32_t n, uint32_t n_rows, uint32_t down, uint32_t* __restrict__ keys,
                                                          uint32_t* __restrict__ pos, uint64_t* __restrict__ runs) {
    if (blockIdx.x) {
        for (uint64_t i = (uint64_t)(blockIdx.x - 1) * 1024 + threadIdx.x; i < n_rows; i += (uint64_t)(gridDim.x - 1) * 1024) runs[i] = 0;
        return;
    }
    __shared__ uint64_t a[SMALL_SORT];
    uint32_t size = 2;
    while (size < n) size *= 2;
    for (uint32_t i = threadIdx.x; i < size; i += 1024) {
        const uint32_t key = key_of(i < n ? ids[i] : -1, n_rows, down);
        a[i] = i < n ? (uint64_t)key << 32 | i : ~0ull;
    }
    for (uint32_t k = 2; k <= size; k *= 2)
        for (uint32_t j = k / 2; j; j /= 2) {
            __syncthreads();
            for (uint32_t t = threadIdx.x; t < size / 2; t += 1024) {
                const uint32_t lo = t / j * 2 * j + t % j, hi = lo + j;
                const uint64_t x = a[lo], y = a[hi];
                if ((x > y) == ((lo & k) == 0)) a[lo] = y, a[hi] = x;
            }
        }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += 1024) {
        keys[i] = (uint32_t)(a[i] >> 32);
        pos[i] = (uint32_t)a[i];
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------------

inline uint64_t up256(uint64_t b) { return (b + 255) / 256 * 256; }

struct SortPlan {             // where things lie in a workspace; n = 0: nothing to sort
    uint32_t passes = 0, bits = 0, blocks = 0, down;
    uint64_t off_keys[2], off_pos[2], off_hist, off_total, bytes = 0;
    SortPlan(uint64_t n, uint64_t n_rows, uint32_t down_ = 0) : down(down_) {
        if (!n) return;
        const uint64_t stranger = (n_rows + (1ull << down) - 1) >> down;      // the largest key
        uint32_t need = 1;
        while (need < 32 && (stranger >> need)) ++need;
        passes = (need + MAX_DIGIT - 1) / MAX_DIGIT;
        bits = (need + passes - 1) / passes;
        blocks = (uint32_t)((n + SORT_BLOCK - 1) / SORT_BLOCK);
        for (int i = 0; i < 2; ++i) {
            off_keys[i] = bytes, bytes += up256(n * 4);
            off_pos[i] = bytes, bytes += up256(n * 4);
        }
        off_hist = bytes, bytes += up256(((uint64_t)blocks << MAX_DIGIT) * 4);      // the same for every n_rows
        off_total = bytes, bytes += up256(4ull << MAX_DIGIT);
    }
};

// n ids, n and n_rows below 2^31, into *keys and *pos (of the workspace); runs, if not NULL: [n_rows], cleared on the way
inline int sort_ids(const SortPlan& pl, const int64_t* ids, uint64_t n, uint64_t n_rows, char* ws, uint64_t* runs, const uint32_t** keys,
                    const uint32_t** pos, hipStream_t s) {
    const uint32_t last = n <= SMALL_SORT ? 0 : (pl.passes - 1) & 1;
    const uint64_t clearing = runs ? (n_rows + 4095) / 4096 : 0;
    if (n <= SMALL_SORT) {
        hipLaunchKernelGGL(sort_small_kernel, dim3(1 + (unsigned)std::min<uint64_t>(clearing, 1024)), dim3(1024), 0, s, ids, (uint32_t)n,
                           (uint32_t)n_rows, pl.down, (uint32_t*)(ws + pl.off_keys[0]), (uint32_t*)(ws + pl.off_pos[0]), runs);
        OPCHK(hipGetLastError());
    }
    for (uint32_t i = 0; i < pl.passes && n > SMALL_SORT; ++i) {
        SortPass p{};
        p.ids = i == 0 ? ids : nullptr;
        p.keys = (const uint32_t*)(ws + pl.off_keys[(i + 1) & 1]);
        p.pos = (const uint32_t*)(ws + pl.off_pos[(i + 1) & 1]);
        p.keys_out = (uint32_t*)(ws + pl.off_keys[i & 1]);
        p.pos_out = (uint32_t*)(ws + pl.off_pos[i & 1]);
        p.hist = (uint32_t*)(ws + pl.off_hist);
        p.total = (uint32_t*)(ws + pl.off_total);
        p.n = (uint32_t)n;
        p.n_rows = (uint32_t)n_rows;
        p.down = pl.down;
        p.blocks = pl.blocks;
        p.shift = i * pl.bits;
        p.bits = pl.bits;
        const uint32_t more = i == 0 ? (uint32_t)std::min<uint64_t>(clearing, 2048) : 0;
        hipLaunchKernelGGL(sort_count_kernel, dim3(std::max(pl.blocks, more)), dim3(SORT_THREADS), 0, s, p, i == 0 ? runs : (uint64_t*)nullptr);
        OPCHK(hipGetLastError());
        hipLaunchKernelGGL(sort_scan_kernel, dim3(((1u << pl.bits) + 3) / 4), dim3(256), 0, s, p);
        OPCHK(hipGetLastError());
        hipLaunchKernelGGL(sort_scatter_kernel, dim3(pl.blocks), dim3(SORT_THREADS), 0, s, p);
        OPCHK(hipGetLastError());
    }
    *keys = (const uint32_t*)(ws + pl.off_keys[last]);
    *pos = (const uint32_t*)(ws + pl.off_pos[last]);
    return CGV_OK;
}

}  // namespace
}  // namespace cgv_ops
