// The shared prefix: 128 queries of a key head at a time on the tensor cores.
//
// A query of the batch is a row: row b * group + g of key head h is query head h * group + g of sequence b.  A CTA has one stretch of the prefix for up to 256 rows, in
// two groups of four warps; keys and values come 128 at a time into a ring in shared memory, page by page as tiled copies.
//   S = Q K^T   128 x 64 in tensor memory, operands from shared memory;
//   P = 2^(S - m) in the cache's type, which takes S's place: a thread has a row, so that maxima and sums need no other thread;
//   O += P V    128 x dim in tensor memory, P from there.
// A group has two places for S, for the halves of a tile of 128 keys: the next S is there when a P is done, and nobody waits for the tensor cores, which work for
// the other half and the other group meanwhile.  (With one place of 128 keys a group's steps are a chain, softmax, P V, Q K^T, of 4100 cycles.)  With more than 128 rows each
// group has 128 of them and both use the same keys; with no more (or for the last 128 of an odd number of such tiles) the groups take the stretch's tiles of
// keys in turn, and their results are two parts.
//
// O is scaled anew only where a row's largest logit has grown by more than 2^8 since it last was: P is then at most 2^8, which is far from the end of
// either type's range, and what m a part refers to does not matter when parts are joined.  P is rounded to 16 bits, as the tensor cores take it: a relative
// 2^-8 (BF16) of every weight by itself, below what the result is rounded by.  Sums are of P as it was before.
// Bounds: for many rows the tensor cores and the exponentials alike (128 x 128 logits are 1024 cycles of each per group at the nominal rates), for few the memory.
#pragma once

#include <cuda.h>

#include "attn_own.cuh"
#include "mx4_tensor.cuh"

namespace mps {

constexpr int kAttendThreads = 512;
constexpr float kRescale = 8.f;      // in powers of two

template <int DIM>
struct PrefixShape {
    static constexpr int kHalf = kPrefixKeys * 128, kHalves = DIM / 64;      // 64 columns of a tile, rows of 128 bytes
    static constexpr int kStage = kHalves * kHalf, kStages = DIM == 128 ? 5 : 12;
    static constexpr int kRing = 2 * kStage;                                  // behind two tiles of queries
    static constexpr int kBars = kRing + kStages * kStage;
    static_assert(FewShape<DIM>::kSmem <= kBars, "the sequences' own keys take the same place in the CTAs that have them");
    static constexpr int kSmem = kBars + (2 * kStages + 11) * 8 + 32;
    static constexpr int kColumns = 512;                                      // S, S, O, O
    static_assert(kSmem <= 232448, "shared memory");
};
struct PrefixMaps { CUtensorMap k, v; };

// A box: 64 columns of neighbouring slots of one page.  A page outside the cache gives zeros.
__device__ __forceinline__ void page_box(uint32_t dst, const CUtensorMap* map, int column, int slot, int head, int page, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(column), "r"(slot), "r"(head), "r"(page), "r"(bar) : "memory");
}
// The largest of three; NaN where there is one.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// 2^x, off by 2^-22 of itself: far below what P is rounded by.  (Results below 2^-126 become 0.)
__device__ __forceinline__ float fast_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// The same by multiplications and additions, for a part of the exponentials, so that the unit that makes them is not alone with them: x is a whole number and a
// rest of half at most, whose power is the polynomial that has 2^x's values at the zeros of Chebyshev's polynomial of degree six on [-1/2, 1/2] (off by
// 2^-22); the whole number is added to the exponent.  Below 2^-126 it stays there.
__device__ __forceinline__ float2 poly_exp2(float2 x) {
    const auto both = [](float c) { return make_float2(c, c); };
    x = make_float2(max3(x.x, -126.f, -126.f), max3(x.y, -126.f, -126.f));
    const float2 one = both(1.f), shifted = fma2(x, one, both(12582912.f)), whole = fma2(shifted, one, both(-12582912.f));      // 1.5 2^23: rounds to whole numbers
    const float2 f = fma2(whole, both(-1.f), x);
    float2 r = fma2(f, both(0.0013390863314270973f), both(0.009676031768321991f));
    r = fma2(f, r, both(0.055503569543361664f));
    r = fma2(f, r, both(0.2402210682630539f));
    r = fma2(f, r, both(0.6931471824645996f));
    r = fma2(f, r, both(1.0000001192092896f));
    return make_float2(__uint_as_float(__float_as_uint(r.x) + (__float_as_uint(shifted.x) << 23)), __uint_as_float(__float_as_uint(r.y) + (__float_as_uint(shifted.y) << 23)));
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
    const auto s_full = [&](int g, int h) { return bar0 + 8u * (2 * S::kStages + 2 * g + h); };                // of 64 keys
    const auto p_ready = [&](int g, int h) { return bar0 + 8u * (2 * S::kStages + 4 + 2 * g + h); };
    const auto added = [&](int g) { return bar0 + 8u * (2 * S::kStages + 8 + g); };                            // P V to the result
    const uint32_t done = bar0 + 8u * (2 * S::kStages + 10);

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        for (int g = 0; g < 2; ++g) {
            for (int h = 0; h < 2; ++h) { mbar_init(s_full(g, h), 1); mbar_init(p_ready(g, h), 4); }
            mbar_init(added(g), 1);
        }
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

    // What the softmax warps and the multiplying one wait for: the queries in shared memory, and whether pages are absent.
    const auto prepared = [&]() { asm volatile("bar.sync 1, 288;" ::: "memory"); };

    // a row's 128 logits want more registers than a 512th of them: the other warps give up theirs (256 x 192 + 128 x 64 + 128 x 64 = 512 x 128)
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == 9) {
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
            const uint32_t qk = half_instruction(BF16, kPrefixKeys / 2, false), pv = half_instruction(BF16, DIM, true);
            bool ok = true;
            const auto arrived = [&](int n) { ok = ok && warp_wait(full(n % S::kStages), (uint32_t)(n / S::kStages) & 1u, &failed); };
            // of half a tile's keys
            const auto logits = [&](int g, int j, int h) {
                const uint32_t q = base + (paired ? g : 0) * S::kStage, k = ring + key_number(j) % S::kStages * S::kStage + h * (S::kHalf / 2);
#pragma unroll
                for (int c = 0; c < S::kHalves; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i)      // 32 bytes on: two in the descriptors' unit
                        half_multiply(lead, s_at + g * 128 + h * 64, operand_desc(q + c * S::kHalf) + 2 * i, operand_desc(k + c * S::kHalf) + 2 * i, qk, c + i ? 1u : 0u);
                tensor_commit(lead, s_full(g, h));
            };
            const auto results = [&](int g, int j, int h, int turn) {
                ok = ok && warp_wait(p_ready(g, h), (uint32_t)turn & 1u, &failed);
                if (!ok) return;
                tensor_fence_after();
                const uint32_t v = ring + value_number(j) % S::kStages * S::kStage + h * (S::kHalf / 2);
#pragma unroll
                for (int i = 0; i < kPrefixKeys / 32; ++i)      // 16 keys on: two groups of eight rows
                    half_multiply_kept(lead, o_at + g * 128, s_at + g * 128 + h * 64 + i * 8, wide_operand_desc(v, S::kHalf) + i * (2048 >> 4), pv, i + h || turn ? 1u : 0u);
                tensor_commit(lead, added(g));
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
                for (int h = 0; h < 2; ++h) {
                    logits(0, 0, h);
                    if (paired) logits(1, 0, h);
                }
                tensor_commit(lead, empty(0));
            }
            if (!paired && tiles > 1) {
                arrived(key_number(1));
                if (ok) {
                    for (int h = 0; h < 2; ++h) logits(1, 1, h);
                    tensor_commit(lead, empty(key_number(1) % S::kStages));
                }
            }
            // what takes the place of a P that has been multiplied comes right after it
            for (int j = 0; j < tiles && ok; ++j) {
                const int next = paired ? j + 1 : j + 2, first = paired ? 0 : j & 1, last = paired ? 1 : j & 1;
                values(j);
                if (next < tiles) arrived(key_number(next));
                for (int h = 0; h < 2 && ok; ++h) {
                    for (int g = first; g <= last && ok; ++g) {
                        results(g, j, h, paired ? j : j >> 1);
                        if (ok && next < tiles) logits(g, next, h);
                    }
                }
                if (!ok) break;
                tensor_commit(lead, empty(value_number(j) % S::kStages));
                if (next < tiles) tensor_commit(lead, empty(key_number(next) % S::kStages));
            }
            tensor_commit(lead, done);
            warp_wait(done, 0, &failed);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
        // the queries, as the tensor cores read them: 16-byte pieces XORed with the row; eight at a time under way
        constexpr int kAhead = DIM / 16;      // pieces of a row by 256 threads
        for (int tile = 0; tile < (paired ? 2 : 1); ++tile) {
            uint4 v[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int r = (i * 256 + threadIdx.x) / (DIM / 8), piece = threadIdx.x % (DIM / 8), row = (x * 2 + tile) * kPrefixRows + r;
                v[i] = make_uint4(0u, 0u, 0u, 0u);
                if (row < rows) v[i] = *reinterpret_cast<const uint4*>(p.q + (int64_t)(row / p.group) * p.q_token + (int64_t)(kv_head * p.group + row % p.group) * p.q_head + piece * 8);
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int r = (i * 256 + threadIdx.x) / (DIM / 8), piece = threadIdx.x % (DIM / 8);
                *reinterpret_cast<uint4*>(smem + tile * S::kStage + piece / 8 * S::kHalf + r * 128 + (((piece & 7) ^ (r & 7)) << 4)) =
                    make_uint4(query_pair<BF16>(v[i].x, p.q_factor), query_pair<BF16>(v[i].y, p.q_factor), query_pair<BF16>(v[i].z, p.q_factor),
                               query_pair<BF16>(v[i].w, p.q_factor));
            }
        }
        {
            const int first = key0 >> p.page_shift, last = (key_end - 1) >> p.page_shift;
            for (int i = first + threadIdx.x; i <= last; i += 256)
                if ((uint32_t)p.prefix_table[i] >= (uint32_t)p.pages) absent = 1u;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // the tensor core reads what was written here
        prepared();
        const int g = warp >> 2, row = (x * 2 + (paired ? g : 0)) * kPrefixRows + (warp & 3) * 32 + lane;
        const bool some = row - lane < rows;         // of the warp's rows are queries
        const uint32_t mine = (uint32_t)(warp & 3) << 21, s_mine = s_at + g * 128 + mine, o_mine = o_at + g * 128 + mine;
        const int turns = paired ? tiles : (tiles - g + 1) / 2;
        float m = -INFINITY;
        float2 sum = make_float2(0.f, 0.f);
        bool ok = true;
        uint32_t s[2][32];
        bool asked_for = false;      // this half's logits, while the last one's weights were made
#pragma unroll 1
        for (int step = 0; step < 2 * turns; ++step) {
            const int h = step & 1, turn = step >> 1;
            if (!some) {
                ok = warp_wait(s_full(g, h), (uint32_t)turn & 1u, &failed);
                if (!ok) break;
                if (lane == 0) mbar_arrive(p_ready(g, h));
                continue;
            }
            if (!asked_for) {
                ok = warp_wait(s_full(g, h), (uint32_t)turn & 1u, &failed);
                if (!ok) break;
                tensor_fence_after();
                tmem_ask32(s_mine + h * 64, s[0]);
                tmem_ask32(s_mine + h * 64 + 32, s[1]);
            }
            const int key = key0 + (paired ? turn : 2 * turn + g) * kPrefixKeys + h * 64;
            tmem_arrived(s[0]);
            tmem_arrived(s[1]);
            if (key_end - key < 64 || absent) {
                leave_gaps(p, key, key_end, s[0]);
                leave_gaps(p, key + 32, key_end, s[1]);
            }
            float top[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                top[k] = max3(__uint_as_float(s[0][k]), __uint_as_float(s[1][k]), __uint_as_float(s[0][k + 4]));
                top[k] = max3(top[k], __uint_as_float(s[1][k + 4]), __uint_as_float(s[0][k + 8]));
                top[k] = max3(top[k], __uint_as_float(s[1][k + 8]), __uint_as_float(s[0][k + 12]));
                top[k] = max3(top[k], __uint_as_float(s[1][k + 12]), __uint_as_float(s[0][k + 16]));
                top[k] = max3(top[k], __uint_as_float(s[1][k + 16]), __uint_as_float(s[0][k + 20]));
                top[k] = max3(top[k], __uint_as_float(s[1][k + 20]), __uint_as_float(s[0][k + 24]));
                top[k] = max3(top[k], __uint_as_float(s[1][k + 24]), __uint_as_float(s[0][k + 28]));
                top[k] = max3(top[k], __uint_as_float(s[1][k + 28]), __uint_as_float(s[1][k + 28]));
            }
            const float high = max3(max3(top[0], top[1], top[2]), top[3], top[3]) * p.scale_log2;
            if (step == 0) {
                m = high;
            } else if (const bool grown = !(high <= m + kRescale); __any_sync(0xFFFFFFFFu, grown)) {
                // the last half's weights may still be on their way into the result
                ok = warp_wait(added(g), (uint32_t)(step - 1) & 1u, &failed);
                if (!ok) break;
                tensor_fence_after();
                // rows that have not keep their scale: what a row gets does not go by its neighbours
                const float next = grown ? max3(m, high, high) : m, up = grown ? fast_exp2(m - (next == -INFINITY ? 0.f : next)) : 1.f;
                m = next;
                sum.x *= up;
                sum.y *= up;
#pragma unroll 1
                for (int c = 0; c < DIM / 32; ++c) {
                    uint32_t o[32];
                    tmem_ask32(o_mine + c * 32, o);
                    tmem_arrived(o);
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * up);
                    tmem_store32(o_mine + c * 32, o);
                }
            }
            const float from = m == -INFINITY ? 0.f : m;
            const float2 scale2 = make_float2(p.scale_log2, p.scale_log2), from2 = make_float2(-from, -from), one2 = make_float2(1.f, 1.f);
            uint32_t w[32];
            const int next = step + 1;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float2 e = fma2(make_float2(__uint_as_float(s[c][2 * i]), __uint_as_float(s[c][2 * i + 1])), scale2, from2);
                    if (i % 3 == 2) {
                        e = poly_exp2(e);
                    } else {
                        e.x = fast_exp2(e.x);
                        e.y = fast_exp2(e.y);
                    }
                    sum = fma2(e, one2, sum);
                    w[c * 16 + i] = pack_pair<BF16>(e.x, e.y);
                }
                if (c == 0) {
                    asked_for = next < 2 * turns && __all_sync(0xFFFFFFFFu, mbar_try_wait(s_full(g, next & 1), (uint32_t)(next >> 1) & 1u));
                    tensor_fence_after();
                }
                if (asked_for) tmem_ask32(s_mine + (next & 1) * 64 + c * 32, s[c]);
            }
            tmem_store32(s_mine + h * 64, w);
            tmem_stored();
            tensor_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_ready(g, h));
        }
        ok = ok && warp_wait(done, 0, &failed);
        tensor_fence_after();
        if (ok && some) {
            const int64_t part = ((int64_t)(paired ? stretch : 2 * stretch + g) * p.kv_heads + kv_head) * rows + row;
            // by way of the ring, whose tiles have been multiplied: straight from the registers every store would touch 32 rows
            const uint32_t rows_at = ring + warp * (32 * 128);      // 32 rows of 32 columns, pieces XORed with the row
            const int64_t first_part = part - lane;
#pragma unroll
            for (int c = 0; c < DIM / 32; ++c) {
                uint32_t o[32];
                tmem_ask32(o_mine + c * 32, o);
                tmem_arrived(o);
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(rows_at + lane * 128 + ((i ^ (lane & 7)) << 4)), "r"(turns ? o[4 * i] : 0u),
                                 "r"(turns ? o[4 * i + 1] : 0u), "r"(turns ? o[4 * i + 2] : 0u), "r"(turns ? o[4 * i + 3] : 0u) : "memory");
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int r = i * 4 + (lane >> 3), piece = lane & 7;
                    uint4 v;
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                                 : "r"(rows_at + r * 128 + ((piece ^ (r & 7)) << 4)) : "memory");
                    if (row - lane + r < rows) *reinterpret_cast<uint4*>(p.prefix_o + (first_part + r) * DIM + c * 32 + piece * 4) = v;
                }
            }
            if (row < rows) p.prefix_ml[part] = make_float2(m, sum.x + sum.y);
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
