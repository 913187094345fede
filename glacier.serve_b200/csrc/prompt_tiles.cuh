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

// Every thread of a warp calls it with the same x; false where no tile has that number.
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
    const int begin = __ldg(a.cu + lo), end = __ldg(a.cu + lo + 1);
    if (begin < 0 || end < begin || end > a.total) return false;
    out.row0 = begin;
    out.len = end - begin;
    out.tile = x - (begin / T + lo);
    return out.tile >= 0 && static_cast<int64_t>(out.tile) * T < out.len;
}

// The same with the tile counts of all prompts listed first, by one warp: before[b] = tiles of the
// prompts before b (before[batch] = all of them, returned).  A prompt whose range is bad has none.
template <int T>
__device__ __forceinline__ int list_prompt_tiles(const PromptArgs& a, int* before) {
    const int lane = threadIdx.x & 31;
    int sum = 0;
    for (int base = 0; base < a.batch; base += 32) {
        const int b = base + lane;
        int n = 0;
        if (b < a.batch) {
            const int begin = __ldg(a.cu + b), end = __ldg(a.cu + b + 1);
            if (begin >= 0 && end >= begin && end <= a.total) n = (end - begin + T - 1) / T;
        }
        int inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(~0u, inc, o);
            if (lane >= o) inc += y;
        }
        if (b < a.batch) before[b] = sum + inc - n;
        sum += __shfl_sync(~0u, inc, 31);
    }
    if (lane == 0) before[a.batch] = sum;
    __syncwarp();
    return sum;
}
template <int T>
__device__ __forceinline__ bool listed_prompt_tile(const PromptArgs& a, const int* before, int tile, PromptTile& out) {
    int lo = 0, hi = a.batch;  // the last prompt with before[b] <= tile: those behind it without tiles share its end
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (before[mid] <= tile) lo = mid;
        else hi = mid;
    }
    const int begin = __ldg(a.cu + lo), end = __ldg(a.cu + lo + 1);
    out.row0 = begin;
    out.len = end - begin;
    out.tile = tile - before[lo];
    return true;
}

// Looks every prompt's range over, whether or not a tile of it is ever searched for.
__device__ __forceinline__ void check_prompts(const PromptArgs& a, int first, int step) {
    for (int b = first; b < a.batch; b += step) {
        const int begin = __ldg(a.cu + b), end = __ldg(a.cu + b + 1);
        if (begin < 0 || end < begin || end > a.total) atomicOr(a.err, kErrBadStep);
    }
}

}  // namespace gkv
