// Device helpers shared by the kernels of the paged cache: packed rows, their owners, pages.
#pragma once

#include <math.h>

#include "common.hip.h"
#include "paged.h"

namespace cactus_hip {

// Softmax weights are rounded to binary16 before they meet the values.  They are held as exp2(score - maximum + LIFT) against a
// maximum that may be up to LAG behind (the output is rescaled only when it has fallen further behind), so the largest is
// 2^(LAG + LIFT) at most and binary16's full 2^-11 reaches down to 2^-25 of the largest weight, a step of 2^-35 below that.
// Without the lift, weights of 2^-24 of the largest were a single step, and 8000 of them beside a first token that takes
// nearly everything were off by half.  The factor leaves with the division by their sum.
constexpr float LAG = 4.0f, LIFT = 11.0f;

struct Rows {
    int first, count;
};

// Rows of sequence b.  cu is device data that nobody checked: whatever it holds, the rows stay inside [0, tokens).
__device__ __forceinline__ Rows rows_of(const int32_t* __restrict__ cu, int b, int tokens) {
    if (!cu) return Rows{b, 1};
    const int lo = min(max(cu[b], 0), tokens), hi = min(max(cu[b + 1], lo), tokens);
    return Rows{lo, hi - lo};
}

// The last b in [0, batch) with begin(b) <= w, for begin not decreasing and begin(0) <= w: 64 candidates at a time, one per
// lane, so 256 sequences take two dependent loads instead of eight.  All 64 lanes of the wave call it.
template <class Begin>
__device__ __forceinline__ int owner_of(int w, int batch, Begin begin) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = batch;
    while (n > 1) {
        const int step = (n + 63) >> 6;
        const int at = lane * step;
        const bool reached = at < n && begin(lo + at) <= w;
        const int c = max(__popcll(__ballot(reached)), 1) - 1;
        lo += c * step;
        n = min(step, n - c * step);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// Work of a ragged batch without its lengths on the host: sequence b owns the work slots floor(cu[b] * per / size) + extra * b
// up to the next sequence's first one.  That is at least floor(rows * per / size) + extra slots for its rows * per items: with
// extra 1 enough for pieces of `size` items that start at the sequence's first item (ceil), with extra 2 for pieces cut at
// multiples of `size` of some other origin.  The launch takes floor(tokens * per / size) + extra * batch slots.
__device__ __forceinline__ int slot_begin(const int32_t* __restrict__ cu, int b, int tokens, int per, int size, int extra) {
    const int at = cu ? min(max(cu[b], 0), tokens) : b;
    return (int)((long long)at * per / size) + extra * b;
}

// Page of tokens page_size * i .. of sequence b, or -1.
__device__ __forceinline__ int page_of(const PagedCache& c, int b, int i) {
    if (i < 0 || i >= c.table_width) return -1;
    const int p = c.tables[(size_t)b * c.table_width + i];
    return p >= 0 && p < c.num_pages ? p : -1;
}

// A page's scale as every kernel takes it: what is not positive and finite (append makes no such scale) is zero.
__device__ __forceinline__ float page_scale(float s) { return s > 0.0f && s < INFINITY ? s : 0.0f; }

// Tokens of sequence b that its table can hold.  The lengths are device data that nobody checked: between 0 and 2^30, positions
// and their differences stay in an int.
__device__ __forceinline__ int context_of(const PagedAttnArgs& a, int b) {
    return min(max(a.contexts[b], 0), a.c.table_width << a.c.page_shift);
}

// The key tiles that rows at positions first .. last see: `sinks` tiles from key 0, then tile `first` and on.
struct TilePlan {
    int sinks, first, tiles;
};
__device__ __forceinline__ TilePlan plan_tiles(int pos_first, int pos_last, int window, int sink, int size) {
    TilePlan p;
    const int all = pos_last < 0 ? 0 : pos_last / size + 1;
    const int low = window ? pos_first - window : 0;
    p.first = low > 0 ? low / size : 0;
    p.sinks = min(p.first, window ? (sink + size - 1) / size : 0);
    p.tiles = p.sinks + max(all - p.first, 0);
    return p;
}

}  // namespace cactus_hip
