// What the kernels of the attention behind a shared prefix have in common: their arguments, and how the sequences' own keys are split.
#pragma once

#include <algorithm>
#include <atomic>

#include "mx4.cuh"
#include "stream_common.cuh"
#include "warp_mma.cuh"

namespace mps {

struct AttendArgs {
    const uint16_t* q;
    const uint16_t* k;                 // the cache's pages
    const uint16_t* v;
    uint16_t* out;
    float* lse;
    const int32_t* tables;
    const int32_t* lengths;
    const int32_t* prefix_table;
    float* prefix_o;                   // [split][key head][row][dim], and the same of (m, l)
    float2* prefix_ml;
    float* own_o;                      // [item][key head][query head of the group][dim]
    float2* own_ml;
    int64_t q_token, q_head, k_page, k_slot, k_head, v_page, v_slot, v_head;      // strides
    int32_t* plan;                     // [0]: stretches of the prefix; from [1] on: the stretches of own keys before each sequence's first, and after the last's
    int64_t table_columns, most_own, page_mask;
    int32_t prefix, pages, page_shift, batch, kv_heads, group;
    int32_t wide_tiles;                // CTAs for a stretch of the prefix and a key head
    int32_t most_splits, own_items;    // places for stretches: of the prefix, of own keys
    int32_t own_ctas;                  // where the host has settled who does what; else -1
    int32_t q_factor;                  // 1, -1 or 0: what queries are multiplied by, exactly
    float scale_log2;                  // positive
    uint32_t* workspace;               // word 0 records a wait that ran out
};

template <bool BF16>
__device__ __forceinline__ uint32_t times_zero(uint32_t pair) {      // 0, or NaN for what is not finite
    uint32_t r;
    if (BF16) asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(pair), "r"(0u));
    else asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(pair), "r"(0u));
    return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t query_pair(uint32_t pair, int factor) {
    return factor == 1 ? pair : factor == -1 ? pair ^ 0x80008000u : times_zero<BF16>(pair);
}

// How the work is split.  The prefix is cut into stretches that a CTA has for up to 256 rows of a key head; the other CTAs have the sequences' own keys, cut into stretches of
// a length that is the same for all.  How long sequences are is known on the GPU only, so every CTA finds the split for itself, from the lengths: of all numbers
// of stretches of the prefix that leave a CTA for the sequences, the one with which the slower side is soonest done.  What a side takes, in cycles, from
// measurements at 1.9 GHz: a CTA that has a part of the prefix, its start and end and 128 keys for 256 rows or for 128; one that has sequences, its start and a
// byte.  What counts is how one side stands to the other: side by side both are slower (3750 cycles, 27 bytes a cycle), in the same ratio.  With 3750 and 50, 128 sequences behind
// 32768 with up to 1024 own keys each took 161 us, with these and with 3750 and 40 118 to 121.  Heads of 64 and F16 share them (a key's cycles are rounded down to a whole number).
constexpr int kPrefixKeys = 128, kPrefixRows = 128;
constexpr int kPrefixStart = 9000, kPrefixPaired = 3000, kPrefixSingle = 1800, kOwnStart = 6000, kOwnBytesPerCycle = 50;
constexpr int kOwnWarps = 14;              // that have own keys, of a CTA
constexpr int kOwnLeast = 64;              // keys of a stretch, at least
constexpr int kFewColumns = 8;             // query heads of a key head that go together

struct AttendSplit { int splits, step, own_ctas, own_step; };      // of the prefix: stretches, and tiles of one; of own keys: CTAs, and keys of a stretch

// Of a CTA that has so many tiles of the prefix's keys (up to 2^23).
__host__ __device__ constexpr int64_t prefix_cycles(int tiles, int tile_cycles) { return kPrefixStart + (int64_t)tiles * tile_cycles; }

// Keys of a stretch, a multiple of 64: so many own keys in all in so many places.  No sequence is longer than 2^30, however many there are of them.
__host__ __device__ constexpr int own_stretch(int64_t keys, int64_t places) {
    const int64_t step = ((keys + places - 1) / places + 63) / 64 * 64;
    return step < kOwnLeast ? kOwnLeast : step > MPS_MOST_KEYS ? (int)MPS_MOST_KEYS : (int)step;
}

// Lengths are at most 2^30.
__device__ __forceinline__ int own_length(const AttendArgs& p, int b) { return min(max(p.lengths[b], 0), (int)p.most_own); }

__device__ __forceinline__ int64_t warp_total(int64_t v) {
#pragma unroll
    for (int x = 16; x; x >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, x);
    return v;
}
// By a whole warp, the same in every lane.  With T own keys in all, B sequences and P places beyond B, stretches of at least T / P are at most T / (T / P) + B.
template <int DIM>
__device__ __forceinline__ AttendSplit split_work(const AttendArgs& p, int ctas) {
    const int lane = threadIdx.x & 31, units = p.kv_heads * p.wide_tiles, tiles = (p.prefix + kPrefixKeys - 1) / kPrefixKeys;
    const int heads = p.kv_heads * ((p.group + kFewColumns - 1) / kFewColumns);
    int64_t keys = 0;
    if (p.own_items) {
        for (int b = lane; b < p.batch; b += 32) keys += own_length(p, b);
        keys = warp_total(keys);
    }
    AttendSplit r = {0, 0, ctas, kOwnLeast};
    if (tiles && p.own_ctas >= 0) {
        r = {1, tiles, p.own_ctas, kOwnLeast};
    } else if (tiles) {
        const int tile_cycles = (p.batch * p.group + kPrefixRows - 1) / kPrefixRows > 1 ? kPrefixPaired : kPrefixSingle;
        const float own_cycles = (float)keys * (float)heads * (float)(DIM * 4 / kOwnBytesPerCycle);
        int64_t best = INT64_MAX;
        int best_splits = 1;
        for (int s = lane + 1; s <= p.most_splits; s += 32) {
            const int left = ctas - units * s;
            if (keys && left < 1) break;
            const float own = keys ? kOwnStart + own_cycles / (float)left : 0.f;
            const int64_t cost = max(prefix_cycles((tiles + s - 1) / s, tile_cycles), (int64_t)fminf(own, 1e18f));
            if (cost < best) { best = cost; best_splits = s; }
        }
#pragma unroll
        for (int x = 16; x; x >>= 1) {
            const int64_t cost = __shfl_xor_sync(0xFFFFFFFFu, best, x);
            const int s = __shfl_xor_sync(0xFFFFFFFFu, best_splits, x);
            if (cost < best || (cost == best && s < best_splits)) { best = cost; best_splits = s; }
        }
        r.step = (tiles + best_splits - 1) / best_splits;
        r.splits = (tiles + r.step - 1) / r.step;
        r.own_ctas = ctas - units * r.splits;
    }
    if (p.own_items) {
        // four stretches for each of the warps that have them
        const int64_t places = min((int64_t)(p.own_items - p.batch), max((int64_t)1, ((int64_t)r.own_ctas * (4 * kOwnWarps) + heads - 1) / heads));
        r.own_step = own_stretch(keys, places);
    }
    return r;
}

// The numbers of stretches before each sequence's first, for who joins them; by a whole warp.
__device__ __forceinline__ void write_plan(const AttendArgs& p, const AttendSplit& split) {
    const int lane = threadIdx.x & 31;
    int before = 0;
    if (lane == 0) p.plan[0] = split.splits;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
        const int b = b0 + lane, count = p.own_items && b < p.batch ? (own_length(p, b) + split.own_step - 1) / split.own_step : 0;
        int behind = count;
#pragma unroll
        for (int x = 1; x < 32; x *= 2) {
            const int v = __shfl_up_sync(0xFFFFFFFFu, behind, x);
            if (lane >= x) behind += v;
        }
        if (b < p.batch) p.plan[1 + b] = before + behind - count;
        before += __shfl_sync(0xFFFFFFFFu, behind, 31);
    }
    if (lane == 0) p.plan[1 + p.batch] = before;
}

// Stretches in the order of their numbers, by a whole warp: 32 sequences at a time.
struct OwnFinder {
    int step, first_sequence, before;      // stretches of the sequences before first_sequence
    int sequence, first, last;             // what was found: keys first to last - 1; sequence -1: none
    __device__ __forceinline__ void find(const AttendArgs& p, int item) {
        const int lane = threadIdx.x & 31;
        for (; first_sequence < p.batch; first_sequence += 32) {
            const int b = first_sequence + lane, length = b < p.batch ? own_length(p, b) : 0, count = (length + step - 1) / step;
            int behind = count;
#pragma unroll
            for (int x = 1; x < 32; x *= 2) {
                const int v = __shfl_up_sync(0xFFFFFFFFu, behind, x);
                if (lane >= x) behind += v;
            }
            const int all = __shfl_sync(0xFFFFFFFFu, behind, 31), number = item - before - (behind - count);
            const uint32_t here = __ballot_sync(0xFFFFFFFFu, number >= 0 && number < count);
            if (here) {
                const int from = __ffs(here) - 1;
                sequence = first_sequence + from;
                first = __shfl_sync(0xFFFFFFFFu, number, from) * step;
                last = min(first + step, __shfl_sync(0xFFFFFFFFu, length, from));
                return;
            }
            before += all;
        }
        sequence = -1;
    }
};

}  // namespace mps
