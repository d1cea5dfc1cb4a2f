// The shared prefix: 128 queries of a key head at a time on the tensor cores.
//
// A query of the batch is a row: row b * group + g of key head h is query head h * group + g of sequence b.  A CTA has one stretch of the prefix for up to 256 rows, in
// two groups of four warps; keys and values come 128 at a time into a ring in shared memory, page by page as tiled copies.
//   S = Q K^T   128 x 128 in tensor memory, operands from shared memory;
//   P = 2^(S - m) in the cache's type, which takes S's place: a thread has a row, so that maxima and sums need no other thread;
//   O += P V    128 x dim in tensor memory, P from there.
// While one group makes its P, the tensor cores work for the other.  With more than 128 rows each group has 128 of them and both use the same keys; with no more
// (or for the last 128 of an odd number of such tiles) the groups take the stretch's tiles of keys in turn, and add their results up at the end.
//
// O is scaled anew only where a row's largest logit has grown by more than 2^kRescale since it last was; what m a part refers to does not matter when parts are
// joined.  P is rounded to 16 bits, as the tensor cores take it: a relative 2^-8 (BF16) or 2^-11 (F16) of every weight by itself, no more than what the result is rounded by.
// Sums are of P as it was before.  BF16 has FP32's range, and m is the largest logit: P is at most 2^8.  F16 has numbers down to 2^-14, and below that steps of 2^-24: there m is
// 2^12 below the largest logit, P at most 2^15, a weight keeps its 2^-11 down to 2^-26 of the stretch's largest and is off by 2^-37 of that beyond.  (With m the largest
// logit itself, keys behind one that weighed e^17 as much and had no value gave a result 44 % off: 2^-24.5 became 2^-24.)
// Bounds: for many rows the softmax.  A period of 128 keys by 256 rows takes 3750 cycles: 2560 of a row's softmax (500 to fetch it, 290 for its maximum, the rest for
// exponentials, sums and packing; 128 x 128 exponentials are 1024 of a scheduler's at the nominal rate) and 690 of two hand-overs, where the products are 2048 for both groups.
// 128 sequences behind 32768 keys with none of their own take 84 to 88 us (32 query heads, 8 key heads of 128).  For few rows the memory.
#pragma once

#include <cuda.h>

#include "attn_own.cuh"
#include "mx4_tensor.cuh"

namespace mps {

constexpr int kAttendThreads = 512;
// In powers of two.  Of BF16 with a kRescale of 0, scaling with every larger maximum, 128 sequences behind 32768 keys took 88.7 us instead of 83.4; F16 takes 86.4, and
// with a kRescale of 8 and nothing to keep small weights' digits took 84.2.
template <bool BF16> constexpr float kLift = BF16 ? 0.f : 12.f;
template <bool BF16> constexpr float kRescale = BF16 ? 8.f : 3.f;
// Logits are scaled and have m taken off in one rounding, m being a rounded number: it may lie so far from the largest logit as FP32's rounding goes, and beyond 2^28 (F16) or
// 2^31 (BF16) that is past the type's range, either way.  Rows whose largest is beyond this are scaled, rounded, first, as m was.  (To look for them costs 128 sequences behind
// 32768 with up to 1024 own keys each 2 of 118 us.)
constexpr float kWide = 1048576.f;

template <int DIM>
struct PrefixShape {
    static constexpr int kHalf = kPrefixKeys * 128, kHalves = DIM / 64;      // 64 columns of a tile, rows of 128 bytes
    static constexpr int kStage = kHalves * kHalf, kStages = DIM == 128 ? 5 : 12;
    static constexpr int kRing = 2 * kStage;                                  // behind two tiles of queries
    static constexpr int kBars = kRing + kStages * kStage;
    static_assert(FewShape<DIM>::kSmem <= kBars, "the sequences' own keys take the same place in the CTAs that have them");
    static constexpr int kSmem = kBars + (2 * kStages + 7) * 8 + 32;
    static constexpr int kColumns = 512;                                      // S, S, O, O
    static_assert(kSmem <= 232448, "shared memory");
};
struct PrefixMaps { CUtensorMap k, v; };

// A box: 64 columns of neighbouring slots of one page.  A page outside the cache gives zeros.
__device__ __forceinline__ void page_box(uint32_t dst, const CUtensorMap* map, int column, int slot, int head, int page, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(column), "r"(slot), "r"(head), "r"(page), "r"(bar) : "memory");
}
// The larger; NaN where there is one.
__device__ __forceinline__ float max2(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// 2^x, off by 2^-22 of itself: far below what P is rounded by.  (Results below 2^-126 become 0.)
__device__ __forceinline__ float fast_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Logits of 32 keys from `key` on: minus infinity for keys behind the stretch's last, and for those of pages outside the cache.
__device__ __forceinline__ void leave_gaps(const AttendArgs& p, int key, int key_end, uint32_t (&v)[32]) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const int first = key + b * 16;
        const int keys = first < key_end && (uint32_t)p.prefix_table[first >> p.page_shift] < (uint32_t)p.pages ? min(key_end - first, 16) : 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) v[b * 16 + i] = i < keys ? v[b * 16 + i] : 0xFF800000u;
    }
}

// Warps of a CTA that has a part of the prefix: 0 to 3 and 4 to 7 a group's rows, 8 multiplies, 9 copies (the others complete groups of four).  Of one that has the sequences'
// own keys: 0 to 13, each for itself.
template <int DIM, bool BF16>
__global__ void __launch_bounds__(kAttendThreads, 1) attend_kernel(const AttendArgs p, const __grid_constant__ PrefixMaps maps) {
    using S = PrefixShape<DIM>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = smem_u32(smem), ring = base + S::kRing, bar0 = base + S::kBars;
    AttendSplit& shared_split = *reinterpret_cast<AttendSplit*>(smem + S::kSmem - 32);
    uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(smem + S::kSmem - 16);
    volatile uint32_t& failed = *reinterpret_cast<volatile uint32_t*>(smem + S::kSmem - 12);
    volatile uint32_t& absent = *reinterpret_cast<volatile uint32_t*>(smem + S::kSmem - 8);      // pages of this stretch lie outside the cache
    const auto full = [&](int s) { return bar0 + 8u * s; };
    const auto empty = [&](int s) { return bar0 + 8u * (S::kStages + s); };
    const auto s_full = [&](int g) { return bar0 + 8u * (2 * S::kStages + g); };
    const auto p_ready = [&](int g, int half) { return bar0 + 8u * (2 * S::kStages + 2 + 2 * g + half); };      // of 64 keys
    const uint32_t done = bar0 + 8u * (2 * S::kStages + 6);

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        for (int g = 0; g < 2; ++g) { mbar_init(s_full(g), 1); mbar_init(p_ready(g, 0), 4); mbar_init(p_ready(g, 1), 4); }
        mbar_init(done, 1);
        failed = 0u;
        absent = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8 && p.prefix) tmem_alloc<1>(smem_u32(&tmem_slot), S::kColumns);
    if (warp == 9 && lane == 0 && p.prefix) { prefetch_map(&maps.k); prefetch_map(&maps.v); }
    griddep_wait();
    griddep_launch();
    if (warp == 0) {
        const AttendSplit split = split_work<DIM>(p, (int)gridDim.x);
        if (lane == 0) shared_split = split;
    }
    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    const AttendSplit split = shared_split;
    const int prefix_ctas = p.kv_heads * p.wide_tiles * split.splits;
    if (blockIdx.x == gridDim.x - 1 && warp == 15) write_plan(p, split);      // it has own keys, and this warp none of them
    const uint32_t tmem = p.prefix ? __shfl_sync(0xFFFFFFFFu, tmem_slot, 0) : 0u;
    if ((int)blockIdx.x >= prefix_ctas) {
        if (p.own_items && warp < kOwnWarps)
            attend_own<DIM, BF16>(p, split.own_step, base + warp * FewShape<DIM>::kRing, ((int)blockIdx.x - prefix_ctas) * kOwnWarps + warp, split.own_ctas * kOwnWarps);
        __syncthreads();
        if (warp == 8 && p.prefix) tmem_free<1>(tmem, S::kColumns);
        return;
    }

    const int rows = p.batch * p.group, row_tiles = (rows + kPrefixRows - 1) / kPrefixRows, pairs = row_tiles / 2;
    const int x = blockIdx.x % p.wide_tiles, kv_head = blockIdx.x / p.wide_tiles % p.kv_heads, stretch = blockIdx.x / p.wide_tiles / p.kv_heads;
    const bool paired = x < pairs;             // else the groups take the keys in turn
    const int key0 = stretch * split.step * kPrefixKeys, key_end = min(p.prefix, key0 + split.step * kPrefixKeys);
    const int tiles = (key_end - key0 + kPrefixKeys - 1) / kPrefixKeys;
    int asked = 0;                             // tiles that this warp has asked for
    const uint32_t s_at = tmem, o_at = tmem + 256;      // and 128 columns on for the second group

    // tiles come as K0, K1, V0, K2, V1, ...: number in that order
    const auto key_number = [&](int j) { return j == 0 ? 0 : 2 * j - 1; };
    const auto value_number = [&](int j) { return j + 1 < tiles ? 2 * j + 2 : 2 * tiles - 1; };

    // What the softmax warps and the multiplying one wait for: the queries in shared memory, and (from warps 10 and 11) whether pages are absent.
    const auto prepared = [&]() { asm volatile("bar.sync 1, 352;" ::: "memory"); };

    // a row's 128 logits want more registers than a 512th of them: the other warps give up theirs (256 x 192 + 128 x 64 + 128 x 64 = 512 x 128)
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == 10 || warp == 11) {
            const int first = key0 >> p.page_shift, last = (key_end - 1) >> p.page_shift;
            for (int i = first + threadIdx.x - 320; i <= last; i += 64)
                if ((uint32_t)p.prefix_table[i] >= (uint32_t)p.pages) absent = 1u;
            prepared();
        } else if (warp == 9) {
            const int box = (int)min(p.page_mask + 1, (int64_t)kPrefixKeys), boxes = kPrefixKeys / box;
            // this lane's box of a tile: its page (the one behind the last, which gives zeros, for one outside), or -1
            const auto page_of = [&](int j) {
                const int key = key0 + j * kPrefixKeys + lane * box;
                if (j >= tiles || lane >= boxes || key >= key_end) return -1;
                const int page = p.prefix_table[key >> p.page_shift];
                return (uint32_t)page < (uint32_t)p.pages ? page : p.pages;
            };
            int ahead = page_of(0), keys = -1, values = -1, n = 0;
            bool ok = true;
            for (; n < 2 * tiles; ++n) {
                const bool is_key = n == 0 || ((n & 1) && (n + 1) / 2 < tiles);
                const int j = n == 0 ? 0 : is_key ? (n + 1) / 2 : n & 1 ? tiles - 1 : n / 2 - 1, s = n % S::kStages;
                if (is_key) {
                    values = keys;
                    keys = ahead;
                    ahead = page_of(j + 1);
                } else if (n == 2 * tiles - 1) {
                    values = keys;
                }
                const int page = is_key ? keys : values;
                if (n >= S::kStages && !(ok = warp_wait(empty(s), (uint32_t)(n / S::kStages - 1) & 1u, &failed))) break;
                const uint32_t live = __popc(__ballot_sync(0xFFFFFFFFu, page >= 0));
                if (lane == 0) mbar_expect_tx(full(s), live * box * 128 * S::kHalves);
                __syncwarp();
                if (page >= 0) {
                    const int slot = (key0 + j * kPrefixKeys + lane * box) & (int)p.page_mask;
#pragma unroll
                    for (int h = 0; h < S::kHalves; ++h)
                        page_box(ring + s * S::kStage + h * S::kHalf + lane * box * 128, is_key ? &maps.k : &maps.v, h * 64, slot, kv_head, page, full(s));
                }
                __syncwarp();
            }
            asked = n;
        } else if (warp == 8) {
            prepared();
            tensor_fence_after();
            const uint32_t lead = elect_one();
            const uint32_t qk = half_instruction(BF16, kPrefixKeys, false), pv = half_instruction(BF16, DIM, true);
            bool ok = true;
            const auto arrived = [&](int n) { ok = ok && warp_wait(full(n % S::kStages), (uint32_t)(n / S::kStages) & 1u, &failed); };
            const auto logits = [&](int g, int j) {
                const uint32_t q = base + (paired ? g : 0) * S::kStage, k = ring + key_number(j) % S::kStages * S::kStage;
#pragma unroll
                for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i)      // 32 bytes on: two in the descriptors' unit
                        half_multiply(lead, s_at + g * 128, operand_desc(q + h * S::kHalf) + 2 * i, operand_desc(k + h * S::kHalf) + 2 * i, qk, h + i ? 1u : 0u);
                tensor_commit(lead, s_full(g));
            };
            // half by half, as the weights come
            const auto results = [&](int g, int j, int turn) {
                const uint32_t v = ring + value_number(j) % S::kStages * S::kStage;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    ok = ok && warp_wait(p_ready(g, half), (uint32_t)turn & 1u, &failed);
                    if (!ok) return;
                    tensor_fence_after();
#pragma unroll
                    for (int i = half * 4; i < half * 4 + 4; ++i)      // 16 keys on: two groups of eight rows
                        half_multiply_kept(lead, o_at + g * 128, s_at + g * 128 + i * 8, wide_operand_desc(v, S::kHalf) + i * (2048 >> 4), pv, i || turn ? 1u : 0u);
                }
            };
            // values behind the prefix's last are what the page holds, which may be NaN: rows of zeros instead
            const auto values = [&](int j) {
                arrived(value_number(j));
                const int valid = min(kPrefixKeys, key_end - key0 - j * kPrefixKeys);
                if (ok && valid < kPrefixKeys) {
                    uint8_t* v = smem + S::kRing + value_number(j) % S::kStages * S::kStage;
#pragma unroll
                    for (int h = 0; h < S::kHalves; ++h)
                        for (int i = valid * 8 + lane; i < kPrefixKeys * 8; i += 32) *reinterpret_cast<uint4*>(v + h * S::kHalf + i * 16) = make_uint4(0u, 0u, 0u, 0u);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
            };
            arrived(0);
            if (ok) {
                logits(0, 0);
                if (paired) logits(1, 0);
                tensor_commit(lead, empty(0));
            }
            if (!paired && tiles > 1) {
                arrived(key_number(1));
                if (ok) {
                    logits(1, 1);
                    tensor_commit(lead, empty(key_number(1) % S::kStages));
                }
            }
            for (int j = 0; j < tiles && ok; ++j) {
                values(j);
                if (paired) {
                    if (j + 1 < tiles) arrived(key_number(j + 1));
                    for (int g = 0; g < 2 && ok; ++g) {
                        results(g, j, j);
                        if (!ok) break;
                        if (g) tensor_commit(lead, empty(value_number(j) % S::kStages));
                        if (j + 1 < tiles) {
                            logits(g, j + 1);
                            if (g) tensor_commit(lead, empty(key_number(j + 1) % S::kStages));
                        }
                    }
                } else {
                    results(j & 1, j, j >> 1);
                    if (!ok) break;
                    tensor_commit(lead, empty(value_number(j) % S::kStages));
                    if (j + 2 < tiles) {
                        arrived(key_number(j + 2));
                        if (!ok) break;
                        logits(j & 1, j + 2);
                        tensor_commit(lead, empty(key_number(j + 2) % S::kStages));
                    }
                }
            }
            tensor_commit(lead, done);
            warp_wait(done, 0, &failed);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
        // the queries, as the tensor cores read them: 16-byte pieces XORed with the row; eight at a time under way
        constexpr int kAhead = DIM / 16, kRowStep = 256 / (DIM / 8);      // pieces of a tile by 256 threads, and how many rows on the next one is
        for (int tile = 0; tile < (paired ? 2 : 1); ++tile) {
            uint4 v[kAhead];
            const int r0 = threadIdx.x / (DIM / 8), piece = threadIdx.x % (DIM / 8), row0 = (x * 2 + tile) * kPrefixRows + r0;
            int sequence = row0 / p.group, in_group = row0 % p.group;
            const int sequences = kRowStep / p.group, others = kRowStep % p.group;
            const uint16_t* q = p.q + (int64_t)kv_head * p.group * p.q_head + piece * 8;
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                v[i] = make_uint4(0u, 0u, 0u, 0u);
                if (sequence < p.batch) v[i] = *reinterpret_cast<const uint4*>(q + sequence * p.q_token + in_group * p.q_head);
                sequence += sequences;
                in_group += others;
                if (in_group >= p.group) { in_group -= p.group; ++sequence; }
            }
            uint8_t* to = smem + tile * S::kStage + piece / 8 * S::kHalf + r0 * 128 + (((piece & 7) ^ (r0 & 7)) << 4);      // the rows' steps are multiples of eight
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                *reinterpret_cast<uint4*>(to + i * kRowStep * 128) = make_uint4(query_pair<BF16>(v[i].x, p.q_factor), query_pair<BF16>(v[i].y, p.q_factor),
                                                                               query_pair<BF16>(v[i].z, p.q_factor), query_pair<BF16>(v[i].w, p.q_factor));
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // the tensor core reads what was written here
        prepared();
        const int g = warp >> 2, row = (x * 2 + (paired ? g : 0)) * kPrefixRows + (warp & 3) * 32 + lane;
        const bool some = row - lane < rows;         // of the warp's rows are queries
        const uint32_t mine = (uint32_t)(warp & 3) << 21, s_mine = s_at + g * 128 + mine, o_mine = o_at + g * 128 + mine;
        const int turns = paired ? tiles : (tiles - g + 1) / 2;
        float m = -INFINITY;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        bool ok = true;
        for (int turn = 0; turn < turns; ++turn) {
            ok = warp_wait(s_full(g), (uint32_t)turn & 1u, &failed);
            if (!ok) break;
            tensor_fence_after();
            if (some) {
                const int j = paired ? turn : 2 * turn + g, key = key0 + j * kPrefixKeys;
                uint32_t s[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ask32(s_mine + c * 32, s[c]);
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_arrived(s[c]);
                if (key_end - key < kPrefixKeys || absent) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) leave_gaps(p, key + c * 32, key_end, s[c]);
                }
                float top[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) top[i] = __uint_as_float(s[0][i]);
#pragma unroll
                for (int i = 8; i < kPrefixKeys; ++i) top[i & 7] = max2(top[i & 7], __uint_as_float(s[i >> 5][i & 31]));
                float factor = p.scale_log2, high = max2(max2(max2(top[0], top[1]), max2(top[2], top[3])), max2(max2(top[4], top[5]), max2(top[6], top[7]))) * factor;
                if (const bool wide = fabsf(high) > kWide; __any_sync(0xFFFFFFFFu, wide)) {
                    const float now = wide ? factor : 1.f;      // a row's arithmetic does not go by its neighbours
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int i = 0; i < 32; ++i) s[c][i] = __float_as_uint(__uint_as_float(s[c][i]) * now);
                    factor = wide ? 1.f : factor;
                }
                if (!BF16) high = __fadd_ru(high, -kLift<BF16>);      // not below the logit less the lift, and the sum not above, however far FP32's numbers lie apart
                if (turn == 0) {
                    m = high;
                } else if (const bool grown = !(high <= __fadd_rd(m, kRescale<BF16>)); __any_sync(0xFFFFFFFFu, grown)) {
                    // rows that have not keep their scale: what a row gets does not go by its neighbours
                    const float next = grown ? max2(m, high) : m, up = grown ? fast_exp2(m - (next == -INFINITY ? 0.f : next)) : 1.f;
                    m = next;
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[i] *= up;
#pragma unroll 1
                    for (int c = 0; c < DIM / 16; ++c) {
                        float o[16];
                        tmem_load16(o_mine + c * 16, o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] *= up;
                        tmem_store16(o_mine + c * 16, o);
                    }
                }
                const float from = m == -INFINITY ? 0.f : m;
                // the tensor cores multiply the first half's weights while the second's are made
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t w[32];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        // nothing waits for what was begun right before it: two warps a scheduler do not hide that
                        float e[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) e[i] = fmaf(__uint_as_float(s[half * 2 + c][i]), factor, -from);
#pragma unroll
                        for (int i = 0; i < 32; ++i) e[i] = fast_exp2(e[i]);
#pragma unroll
                        for (int i = 0; i < 32; ++i) sum[i & 3] += e[i];
#pragma unroll
                        for (int i = 0; i < 16; ++i) w[c * 16 + i] = pack_pair<BF16>(e[2 * i], e[2 * i + 1]);
                    }
                    tmem_store32(s_mine + half * 32, w);
                    tmem_stored();
                    tensor_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_ready(g, half));
                }
            } else if (lane == 0) {
                mbar_arrive(p_ready(g, 0));
                mbar_arrive(p_ready(g, 1));
            }
        }
        ok = ok && warp_wait(done, 0, &failed);
        tensor_fence_after();
        const float total = (sum[0] + sum[1]) + (sum[2] + sum[3]);
        if (!paired) {
            float2* turn_ml = reinterpret_cast<float2*>(smem + S::kRing + 65536);      // of both groups; behind what the rows pass through below
            turn_ml[threadIdx.x] = make_float2(m, total);
            asm volatile("bar.sync 2, 256;" ::: "memory");
        }
        if (ok && some) {
            // By way of the ring, whose tiles have been multiplied: straight from the registers every store would touch 32 rows.  There: 32 rows of 32 columns,
            // pieces XORed with the row.
            const uint32_t rows_at = ring + warp * (32 * 128);
            const int64_t part = ((int64_t)stretch * p.kv_heads + kv_head) * rows + row, first_part = part - lane;
            const auto store = [&](int column, const auto& o) {
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(rows_at + lane * 128 + ((i ^ (lane & 7)) << 4)), "r"(o[4 * i]), "r"(o[4 * i + 1]),
                                 "r"(o[4 * i + 2]), "r"(o[4 * i + 3]) : "memory");
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int r = i * 4 + (lane >> 3), piece = lane & 7;
                    uint4 v;
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                                 : "r"(rows_at + r * 128 + ((piece ^ (r & 7)) << 4)) : "memory");
                    if (row - lane + r < rows) *reinterpret_cast<uint4*>(p.prefix_o + (first_part + r) * DIM + column + piece * 4) = v;
                }
            };
            if (paired) {
                uint32_t o[DIM / 32][32];
#pragma unroll
                for (int c = 0; c < DIM / 32; ++c) tmem_ask32(o_mine + c * 32, o[c]);
#pragma unroll
                for (int c = 0; c < DIM / 32; ++c) {
                    tmem_arrived(o[c]);
                    store(c * 32, o[c]);
                }
                if (row < rows) p.prefix_ml[part] = make_float2(m, total);
            } else {
                // both groups' sums of the same rows become one, each group half of the columns: half as many parts to write and to join (with two, 32 sequences
                // behind 8192 wrote 11.5 MB of them)
                const float2* turn_ml = reinterpret_cast<const float2*>(smem + S::kRing + 65536);
                const float2 first = turn_ml[threadIdx.x & 127], second = turn_ml[128 + (threadIdx.x & 127)];
                const float high = max2(first.x, second.x), from = high == -INFINITY ? 0.f : high, f0 = fast_exp2(first.x - from), f1 = fast_exp2(second.x - from);
                const uint32_t o_half = o_at + mine + g * (DIM / 2);
                uint32_t o0[DIM / 64][32], o1[DIM / 64][32];
#pragma unroll
                for (int c = 0; c < DIM / 64; ++c) {
                    tmem_ask32(o_half + c * 32, o0[c]);
                    tmem_ask32(o_half + 128 + c * 32, o1[c]);
                }
#pragma unroll
                for (int c = 0; c < DIM / 64; ++c) {
                    tmem_arrived(o0[c]);
                    tmem_arrived(o1[c]);
#pragma unroll
                    for (int i = 0; i < 32; ++i)      // of one tile the second group has had none, and nothing is in its sums
                        o0[c][i] = __float_as_uint(fmaf(__uint_as_float(o0[c][i]), f0, tiles > 1 ? __uint_as_float(o1[c][i]) * f1 : 0.f));
                    store(g * (DIM / 2) + c * 32, o0[c]);
                }
                if (g == 0 && row < rows) p.prefix_ml[part] = make_float2(high, fmaf(first.y, f0, second.y * f1));
            }
        }
    }
    __syncwarp();
    tensor_fence_before();
    __syncthreads();      // what was copied has been multiplied, unless a wait ran out
    tensor_fence_after();
    if (failed) {
        // no copy may come after this CTA is gone
        for (int i = max(0, asked - S::kStages); i < asked; ++i) mbar_wait(full(i % S::kStages), (uint32_t)(i / S::kStages) & 1u, kMx4SpinLimit);
        if (threadIdx.x == 0) atomicExch(p.workspace, 1u);
        __syncthreads();
    }
    if (warp == 8) tmem_free<1>(tmem, S::kColumns);
}

}  // namespace mps
