// Query tiles of packed prompts, found on the device from the cumulated lengths.
#pragma once

#include "kernels.h"

namespace gkv {

// Prompt b of rows cu[b] .. cu[b + 1] takes tile numbers floor(cu[b] / T) + b + (0 .. ceil(len / T) - 1):
// ceil(len / T) <= floor(cu[b + 1] / T) + 1 - floor(cu[b] / T), so the ranges of the prompts do not
// meet, and a tile finds its prompt by searching the increasing function floor(cu[b] / T) + b, with no
// sum over the prompts before it.  At most one number per prompt is left over.
struct PromptTile {
    int64_t row0;  // first row of the prompt
    int len, tile;
};

// One more than the largest tile number.
inline int64_t prompt_tile_bound(const PromptArgs& a, int tile_rows) { return a.total / tile_rows + a.batch; }

// Tiles of a prompt, none where its range is bad.
template <int T>
__device__ __forceinline__ int tiles_of(int begin, int end, int total) {
    return begin >= 0 && end >= begin && end <= total ? (end - begin) / T + ((end - begin) % T != 0) : 0;
}

// The prompt of tile number x by going over all of them: where bad ranges have led the search astray.
template <int T>
__device__ __noinline__ int prompt_of_tile(const int32_t* cu, int batch, int total, int x) {
    const int lane = threadIdx.x & 31;
    for (int base = 0; base < batch; base += 32) {
        const int b = base + lane;
        bool mine = false;
        if (b < batch) {
            const int begin = __ldg(cu + b), n = tiles_of<T>(begin, __ldg(cu + b + 1), total);
            mine = n > 0 && x >= begin / T + b && x - (begin / T + b) < n;
        }
        const unsigned found = __ballot_sync(~0u, mine);
        if (found) return base + __ffs(found) - 1;
    }
    return -1;
}

// Every thread of a warp calls it with the same x; false where no tile has that number.  The search is exact where
// the ranges are good.  Next to a bad one (left out) it may end anywhere; but where it ends at a good prompt whose first
// number and the next prompt's enclose x, x is this prompt's or nobody's: good prompts that follow one another
// without overlap have their numbers in order.  Only otherwise are all prompts gone over.
template <int T>
__device__ __forceinline__ bool find_prompt_tile(const PromptArgs& a, int x, PromptTile& out) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = a.batch;  // the last b in [lo, lo + n) whose first tile number is at most x
    while (n > 1) {
        const int step = (n + 31) / 32;
        const int b = lo + lane * step;
        const bool le = lane * step < n && __ldg(a.cu + b) / T + b <= x;
        const int last = 31 - __clz(__ballot_sync(~0u, le) | 1u);
        const int at = last * step;
        lo += at;
        n = min(step, n - at);
    }
    int begin = __ldg(a.cu + lo), end = __ldg(a.cu + lo + 1);
    const bool good = begin >= 0 && end >= begin && end <= a.total;
    if (!good || (lo > 0 && x < begin / T + lo) || (lo + 1 < a.batch && x > end / T + lo)) {
        lo = prompt_of_tile<T>(a.cu, a.batch, a.total, x);
        if (lo < 0) return false;
        begin = __ldg(a.cu + lo), end = __ldg(a.cu + lo + 1);
    }
    out.row0 = begin;
    out.len = end - begin;
    out.tile = x - (begin / T + lo);
    return out.tile >= 0 && out.tile < tiles_of<T>(begin, end, a.total);
}

// The tiles of up to kListed prompts in descending order of their keys: first every prompt's last tile
// that is as far from its start as any, then the next nearer ones.  With the prompts sorted by tile count,
// c_0 >= c_1 >= ..., c_k tiles deep the first k + 1 of them still have one: levels c_{k+1} .. c_k - 1 hold
// (k + 1) (c_k - c_{k+1}) tiles, so a tile number finds its k by a search over their sums.
// Ranking a batch takes a block batch^2 / threads comparisons, once where blocks go from tile to tile (on the tensor
// cores).  Listed against prompt by prompt there, 28 heads and 4 heads, us: prompts of 1 to 2000 tokens (median 100)
// 256: 321 / 343 and 62 / 72, 512: 788 / 846 and 136 / 148, 1024: 1538 / 1575 and 257 / 241; prompts of 16 tokens, which need
// no order, 256: 162 / 161 and 34 / 30, 512: 321 / 315 and 64 / 53, 1024: 647 / 619 and 133 / 98.
constexpr int kListed = 512;
struct PromptList {
    int count[kListed];        // tiles of each prompt (none where its range is bad)
    int sorted[kListed + 1];   // in descending order, then 0
    int before[kListed + 1];   // tiles of the levels above c_k
    unsigned short order[kListed];
};
// Three steps, a block barrier behind each of the first two.
template <int T>
__device__ __forceinline__ void count_prompt_tiles(const PromptArgs& a, PromptList& l, int thread, int threads) {
    for (int b = thread; b < a.batch; b += threads) {
        const int begin = __ldg(a.cu + b), end = __ldg(a.cu + b + 1);
        l.count[b] = tiles_of<T>(begin, end, a.total);
    }
}
__device__ __forceinline__ void sort_prompts(const PromptArgs& a, PromptList& l, int thread, int threads) {
    for (int b = thread; b < a.batch; b += threads) {
        const int c = l.count[b];
        int rank = 0;
        for (int o = 0; o < a.batch; ++o) {
            const int x = l.count[o];
            rank += x > c || (x == c && o < b);
        }
        l.sorted[rank] = c;
        l.order[rank] = static_cast<unsigned short>(b);
    }
    if (thread == 0) l.sorted[a.batch] = 0;
}
// By one warp; returns the number of tiles.  Sums stop at kTileLimit, above every tile number of a grid: prompts
// that overlap (each range good by itself, the order of the rows not) may have more tiles than 32 bits count.
constexpr int kTileLimit = 1 << 26;
__device__ __forceinline__ int sum_prompt_levels(const PromptArgs& a, PromptList& l) {
    const int lane = threadIdx.x & 31;
    int sum = 0;
    for (int base = 0; base < a.batch; base += 32) {
        const int k = base + lane;
        const int n = k < a.batch ? static_cast<int>(min(static_cast<int64_t>(k + 1) * (l.sorted[k] - l.sorted[k + 1]), int64_t{kTileLimit})) : 0;
        int inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(~0u, inc, o);
            if (lane >= o) inc = min(inc + y, kTileLimit);
        }
        const int up = __shfl_up_sync(~0u, inc, 1);
        if (k < a.batch) l.before[k] = min(sum + (lane ? up : 0), kTileLimit);
        sum = min(sum + __shfl_sync(~0u, inc, 31), kTileLimit);
    }
    __syncwarp();
    return sum;
}
__device__ __forceinline__ void listed_prompt_tile(const PromptArgs& a, const PromptList& l, int tile, PromptTile& out) {
    int lo = 0, hi = a.batch;  // the last k with before[k] <= tile: those with as many tiles as the next hold none
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (l.before[mid] <= tile) lo = mid;
        else hi = mid;
    }
    const int in = tile - l.before[lo], level = in / (lo + 1);
    const int b = l.order[in - level * (lo + 1)];
    const int begin = __ldg(a.cu + b), end = __ldg(a.cu + b + 1);
    out.row0 = begin;
    out.len = end - begin;
    out.tile = l.sorted[lo] - 1 - level;
}

// Looks every prompt's range over, whether or not a tile of it is ever searched for.
__device__ __forceinline__ void check_prompts(const PromptArgs& a, int first, int step) {
    for (int b = first; b < a.batch; b += step) {
        const int begin = __ldg(a.cu + b), end = __ldg(a.cu + b + 1);
        if (begin < 0 || end < begin || end > a.total) atomicOr(a.err, kErrBadStep);
    }
}

}  // namespace gkv
