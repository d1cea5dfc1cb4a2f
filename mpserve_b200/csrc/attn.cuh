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
    int64_t table_columns, most_own, prefix, prefix_step, own_items, page_mask;
    int32_t pages, page_shift, prefix_splits, prefix_units, batch, kv_heads, group;
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

// A sequence's own keys are cut into stretches of a length that is the same for all, such that no more come of it than there are places for: with
// T keys in all, B sequences and P places, stretches of at least T / (P - B) are at most T / (T / (P - B)) + B.  How long sequences are is known on the
// GPU only, so whoever works on stretches finds them for itself, from the lengths.  Lengths are at most 2^30.
constexpr int kOwnLeast = 128;         // keys of a stretch, at least

__device__ __forceinline__ int own_length(const AttendArgs& p, int b) { return min(max(p.lengths[b], 0), (int)p.most_own); }

__device__ __forceinline__ int64_t warp_total(int64_t v) {
#pragma unroll
    for (int x = 16; x; x >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, x);
    return v;
}
// By a whole warp.
__device__ __forceinline__ int own_step(const AttendArgs& p) {
    int64_t total = 0;
    for (int b = threadIdx.x & 31; b < p.batch; b += 32) total += own_length(p, b);
    total = warp_total(total);
    const int64_t places = p.own_items - p.batch;
    return (int)max((int64_t)kOwnLeast, ((total + places - 1) / places + 63) / 64 * 64);
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

struct OwnItems { int first, count; };
// The stretches of a sequence, by a whole warp.
__device__ __forceinline__ OwnItems own_items(const AttendArgs& p, int sequence) {
    if (p.own_items == 0) return {0, 0};
    const int step = own_step(p);
    int64_t before = 0;
    for (int b = threadIdx.x & 31; b < sequence; b += 32) before += (own_length(p, b) + step - 1) / step;
    return {(int)warp_total(before), (own_length(p, sequence) + step - 1) / step};
}

}  // namespace mps
