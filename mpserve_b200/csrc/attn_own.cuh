// The sequences' own tokens: keys on the rows of the products.
//
// A warp has a stretch of one sequence's keys for one key head, 16 keys at a time, through a ring of its own.  Logits are computed as K q^T, 16 keys by 8 query
// heads, and the result as V^T P^T, so that the eight columns are the query heads that share the key head, and none of the tensor cores' rows idles.
// Bound: memory.  A CTA's rings are 224 KB, and a warp's stretches follow one another without a gap: the next one's first keys are asked for while the last ones of this are
// multiplied.
#pragma once

#include "attn.cuh"

namespace mps {

// Weights are 2^(logit - m), rounded to the cache's type before they multiply the values.  In F16 m is so many powers of two below the largest logit: weights are at most
// 2^15, and the small ones keep their digits down to 2^-29 of the largest.
constexpr float kOwnLift = 15.f;

template <int DIM>
struct FewShape {
    static constexpr int kRow = DIM * 2, kBlock = 16 * kRow, kStage = 2 * kBlock;      // 16 keys, then their values
    static constexpr int kStages = 256 / DIM;                                          // 16 KB a warp
    static constexpr int kRing = kStages * kStage;
    static constexpr int kSmem = kOwnWarps * kRing;
};

// 16-byte piece `piece` of row `row`: rows of 256 (128) bytes, pieces XORed with the row, so that eight rows' pieces lie in different banks.
template <int DIM>
__device__ __forceinline__ uint32_t few_place(int row, int piece) { return row * (DIM * 2) + ((piece ^ (row & 7)) << 4); }

struct FewBlock {
    int unit, sequence;      // unit: (stretch, eight query heads, key head); -1: none
    int keys;                // of 16, and kFirst, kLast: the block is the first, the last of its stretch
    static constexpr int kFirst = 32, kLast = 64;
};

// Every workers-th unit is this warp's.  `ring`: its shared memory.
template <int DIM, bool BF16>
__device__ __forceinline__ void attend_own(const AttendArgs& p, int own_step, uint32_t ring, int worker, int workers) {
    using S = FewShape<DIM>;
    constexpr int kPieces = DIM / 8;       // of a row
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int column_tiles = (p.group + kFewColumns - 1) / kFewColumns, per_item = p.kv_heads * column_tiles, units = p.own_items * per_item;
    OwnFinder find;
    find.step = own_step;
    find.first_sequence = find.before = find.first = find.last = 0;
    find.sequence = 0;

    // the block after those that were asked for, and its page: looked up a turn before it is needed
    int next_unit = worker - workers, next_key = 0, page = 0, slot = 0;
    FewBlock next;
    const auto look_ahead = [&]() {
        if (find.sequence >= 0 && next_key >= find.last) {
            next_unit += workers;
            if (next_unit < units) find.find(p, next_unit / per_item);
            else find.sequence = -1;
            next_key = find.first;
        }
        next.unit = -1;
        if (find.sequence < 0) return;
        next.unit = next_unit;
        next.sequence = find.sequence;
        page = p.tables[find.sequence * p.table_columns + (next_key >> p.page_shift)];
        slot = next_key & (int)p.page_mask;
        next.keys = min(16, find.last - next_key) | (next_key == find.first ? FewBlock::kFirst : 0);
        next_key += 16;
        if (next_key >= find.last) next.keys |= FewBlock::kLast;
    };
    const auto ask = [&](int stage) {
        if (next.unit >= 0) {
            if ((uint32_t)page >= (uint32_t)p.pages) { next.keys &= ~31; page = 0; }
            const int keys = next.keys & 31, kv_head = next.unit % per_item % p.kv_heads;
            const uint16_t* k = p.k + (int64_t)page * p.k_page + slot * p.k_slot + kv_head * p.k_head + lane % kPieces * 8;
            const uint16_t* v = p.v + (int64_t)page * p.v_page + slot * p.v_slot + kv_head * p.v_head + lane % kPieces * 8;
            const uint32_t to = ring + stage * S::kStage;
#pragma unroll
            for (int i = 0; i < kPieces / 2; ++i) {
                const int row = i * (32 / kPieces) + lane / kPieces;
                const bool there = row < keys;      // others become zeros: a value that is not there must not be a NaN, which 0 does not multiply away
                cp_async_16_or_zero(to + few_place<DIM>(row, lane % kPieces), there ? k + row * p.k_slot : p.k, there);
                cp_async_16_or_zero(to + S::kBlock + few_place<DIM>(row, lane % kPieces), there ? v + row * p.v_slot : p.v, there);
            }
        }
        cp_async_commit();
    };

    FewBlock blocks[S::kStages];      // that were asked for, the oldest first
    look_ahead();
#pragma unroll
    for (int s = 0; s < S::kStages - 1; ++s) {
        ask(s);
        blocks[s] = next;
        look_ahead();
    }
    uint32_t q[DIM / 16][2];
    float m[2], l[2], o[DIM / 16][4];
    int stage = 0;
    while (blocks[0].unit >= 0) {
        ask(stage == 0 ? S::kStages - 1 : stage - 1);
        blocks[S::kStages - 1] = next;
        look_ahead();
        const FewBlock now = blocks[0];
        const int keys = now.keys & 31;
        if (now.keys & FewBlock::kFirst) {
            const int in_item = now.unit % per_item, head = in_item % p.kv_heads * p.group + in_item / p.kv_heads * kFewColumns;
            const bool live = in_item / p.kv_heads * kFewColumns + g < p.group;
            const uint16_t* query = p.q + now.sequence * p.q_token + (head + (live ? g : 0)) * p.q_head + 2 * t;
#pragma unroll
            for (int d = 0; d < DIM / 16; ++d) {
                const uint32_t* at = reinterpret_cast<const uint32_t*>(query + d * 16);
                q[d][0] = live ? query_pair<BF16>(at[0], p.q_factor) : 0u;
                q[d][1] = live ? query_pair<BF16>(at[4], p.q_factor) : 0u;
                o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
            }
            m[0] = m[1] = -INFINITY;
            l[0] = l[1] = 0.f;
        }
        cp_async_wait<S::kStages - 1>();
        __syncwarp();
        const uint32_t at = ring + stage * S::kStage;
        // K q^T
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < DIM / 16; ++d) {
            uint32_t a[4];
            load_matrices(a, at + few_place<DIM>(lane & 15, 2 * d + (lane >> 4)));
            multiply<BF16>(s, a, q[d][0], q[d][1]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = g + 8 * (i >> 1) < keys ? s[i] * p.scale_log2 : -INFINITY;
        float up[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float top = fmaxf(s[i], s[i + 2]);
#pragma unroll
            for (int x = 4; x < 32; x *= 2) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
            if (!BF16) top = __fadd_ru(top, -kOwnLift);      // not below, however far FP32's numbers lie apart
            top = fmaxf(top, m[i]);
            const float base = top == -INFINITY ? 0.f : top;
            up[i] = exp2f(m[i] - base);
            m[i] = top;
            s[i] = exp2f(s[i] - base);
            s[i + 2] = exp2f(s[i + 2] - base);
            l[i] = fmaf(l[i], up[i], s[i] + s[i + 2]);
        }
        const uint32_t p0 = transpose8(pack_pair<BF16>(s[0], s[1])), p1 = transpose8(pack_pair<BF16>(s[2], s[3]));
        // V^T P^T
#pragma unroll
        for (int d = 0; d < DIM / 16; ++d) {
            uint32_t a[4];
            load_matrices_transposed(a, at + S::kBlock + few_place<DIM>((lane & 7) + ((lane >> 4) << 3), 2 * d + ((lane >> 3) & 1)));
#pragma unroll
            for (int i = 0; i < 4; ++i) o[d][i] *= up[i & 1];
            multiply<BF16>(o[d], a, p0, p1);
        }
        __syncwarp();
        if (now.keys & FewBlock::kLast) {
            const int in_item = now.unit % per_item, first = in_item / p.kv_heads * kFewColumns;
            const int64_t part = ((int64_t)(now.unit / per_item) * p.kv_heads + in_item % p.kv_heads) * p.group + first;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int x = 4; x < 32; x *= 2) l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], x);
                const int c = 2 * t + i;
                if (first + c < p.group) {
                    if (g == 0) p.own_ml[part + c] = make_float2(m[i], l[i]);
                    float* to = p.own_o + (part + c) * DIM + g;
#pragma unroll
                    for (int d = 0; d < DIM / 16; ++d) {
                        to[d * 16] = o[d][i];
                        to[d * 16 + 8] = o[d][i + 2];
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i + 1 < S::kStages; ++i) blocks[i] = blocks[i + 1];
        if (++stage == S::kStages) stage = 0;
    }
    cp_async_wait<0>();
}

}  // namespace mps
