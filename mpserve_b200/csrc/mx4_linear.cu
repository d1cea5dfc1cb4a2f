// Products of MXFP4 matrices: out[t, r] = sum_k x[t, k] w[r, k], and the gated pair act(x Wg) * (x Wu).
#include "mx4.cuh"
#include "mx4_tensor.cuh"
#include "stream_common.cuh"

namespace mps {

int launched(const char* what);

// ---- what the kernels share -------------------------------------------------------------------------

constexpr int kMx4MostSms = 192;               // CTAs of a launch are at most the SMs
constexpr uint32_t kMx4SpinLimit = 1u << 20;
constexpr int kMx4SmemMost = 232448;           // 227 KB

// Workspace: word 0 records a wait that ran out; from byte 4096 on, counters; then partial sums.
constexpr int64_t kMx4CounterBytes = 4096, kMx4PartialOffset = 4096 + kMx4CounterBytes;
constexpr int64_t kMx4PartialFloats = 128 * 256;   // most of one CTA's accumulator, features x tokens
constexpr int64_t kMx4WorkspaceBytes = kMx4PartialOffset + 2 * kMx4MostSms * kMx4PartialFloats * 4;

struct ProductArgs {
    const uint8_t* x;        // tiles
    const uint8_t* w;
    const uint8_t* w_up;
    void* out;
    uint32_t* workspace;
    int64_t out_stride;
    int64_t tokens;
    int32_t rows;            // of the weight: features
    int32_t chunks;          // tiles of a row
    int32_t row_tiles, token_tiles;
    int32_t out_dtype, activation;
    bool x_follows;          // x is written by the kernel before, which this one may overlap
};

// Both activations are g / (1 + exp(-t)): SiLU with t = g, and GELU's tanh form since (1 + tanh z) / 2 = 1 / (1 + exp(-2 z)).  The
// exponential is CUDA's accurate one; the quotient's two units in the last place are far below what the result is rounded to.
__device__ __forceinline__ float act(float g, int which) {
    const float t = which == MPS_SILU ? g : 1.5957691216057308f * g * fmaf(0.044715f * g, g, 1.f);
    return __fdividef(g, 1.f + expf(-t));
}

// A wait that gives up when another one has.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile uint32_t* failed) {
#pragma unroll 1
    for (uint32_t i = 0; i < kMx4SpinLimit; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 63u) == 63u && *failed) return false;
    }
    *failed = 1u;
    return false;
}

// The same for a whole warp: the same answer in every lane.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile uint32_t* failed) {
    return __all_sync(0xFFFFFFFFu, bar_wait(bar, parity, failed));
}

// ---- few tokens: weights on the accumulator's lanes -------------------------------------------------
//
// One CTA per SM streams weight tiles through a ring in shared memory, 17 KB a bulk copy; TOKENS tokens (16 to 128) are the
// product's narrow side.  The work is cut evenly into runs of (tile of the output, tile of K) pairs, a run per CTA, so that
// every SM reads the same number of bytes whatever the sizes; a tile of the output that several CTAs have parts of is summed by
// whichever of them ends last, always in the same order.  Nothing waits for another CTA.
//
// Warps: 0 copies, 1 multiplies, 2 to 5 take the accumulator over, two of which take turns.
template <int TOKENS, bool GATED>
struct StreamShape {
    static constexpr int kWeights = GATED ? 2 : 1;
    static constexpr int kXBytes = kMx4ScaleBytes + TOKENS * kMx4RowBytes;
    static constexpr int kStageBytes = kWeights * kMx4TileBytes + kXBytes;
    static constexpr int kStages = (kMx4SmemMost - 2048) / kStageBytes < 12 ? (kMx4SmemMost - 2048) / kStageBytes : 12;
    static constexpr int kSmem = kStages * kStageBytes + 2048;
    static constexpr int kAcc = TOKENS * kWeights;              // columns of one accumulator
    static constexpr int kScaleColumns = 8 * kWeights + 8;      // of one stage
    static constexpr int kBuffers = kAcc <= 128 ? 2 : 1;        // accumulators that take turns
    static constexpr int kScaleBase = kBuffers * kAcc;
    static constexpr int kColumns = 512;
    static_assert(kScaleBase + kStages * kScaleColumns <= kColumns, "tensor memory");
    static_assert(kStageBytes % 1024 == 0, "the swizzle counts from multiples of 1024 bytes");
    static_assert(kAcc * 128 <= kMx4PartialFloats, "partial sums");
};
constexpr int kStreamThreads = 192;

struct StreamRun { int64_t first, last; };   // units [first, last) of a CTA
__device__ __forceinline__ StreamRun run_of(int64_t units, int cta, int ctas) {
    return {units * cta / ctas, units * (cta + 1) / ctas};
}
// The CTA that has unit u: the largest c with units * c / ctas <= u.
__device__ __forceinline__ int cta_of(int64_t units, int64_t u, int ctas) { return (int)(((u + 1) * ctas - 1) / units); }

// Sixteen tokens of one feature, `up` too where the pair is gated: into the output.
template <bool GATED>
__device__ __forceinline__ void finish16(const ProductArgs& p, int row_tile, int quarter, int lane, int64_t token0, float (&v)[16], float (&up)[16]) {
    const int feature = row_tile * kMx4Rows + quarter * 32 + lane;
    if (GATED) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = act(v[i], p.activation) * up[i];
    }
    if (GATED && p.out_dtype == MPS_MX4) {
        // the warp's 32 features are one block of every token
        const int first = row_tile * kMx4Rows + quarter * 32, chunks = (int)mx4_chunks(p.rows);
        const int chunk = first / kMx4Cols, block = (first % kMx4Cols) / kMx4Block;
        // the last tile's second half may lie beyond the last feature and is filled up with zeros
        const bool fill = row_tile == p.row_tiles - 1 && (row_tile & 1) == 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int64_t t = token0 + i;
            if (t >= p.tokens) break;
            const float f = feature < p.rows ? v[i] : 0.f;
            const uint32_t byte = mx4_scale_byte(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(f) & 0x7FFFFFFFu));
            const float q[8] = {byte == 255u ? 0.f : f * mx4_inverse_scale(byte), 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            uint32_t code = mx4_codes8(q) & 15u;
            code |= __shfl_xor_sync(0xFFFFFFFFu, code, 1) << 4;    // right in the even lanes, then in every fourth, then in every eighth
            code |= __shfl_xor_sync(0xFFFFFFFFu, code, 2) << 8;
            code |= __shfl_xor_sync(0xFFFFFFFFu, code, 4) << 16;
            uint8_t* tile = static_cast<uint8_t*>(p.out) + mx4_tile_offset(t / kMx4Rows, chunk, chunks);
            const int row = (int)(t % kMx4Rows);
            if ((lane & 7) == 0) *reinterpret_cast<uint32_t*>(tile + mx4_code_offset(row, block) + (lane >> 3) * 4) = code;
            if (lane == 0) tile[mx4_scale_offset(row, block >> 2) + (block & 3)] = (uint8_t)byte;
            if (fill) {
                if ((lane & 7) == 0) *reinterpret_cast<uint32_t*>(tile + mx4_code_offset(row, block + 4) + (lane >> 3) * 4) = 0u;
                if (lane == 0) tile[mx4_scale_offset(row, 1) + (block & 3)] = 0u;
            }
        }
        return;
    }
    if (feature >= p.rows) return;
    uint16_t* out = static_cast<uint16_t*>(p.out) + feature;
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (token0 + i < p.tokens) out[(token0 + i) * p.out_stride] = (uint16_t)pack2(v[i], 0.f, p.out_dtype);
}

template <int TOKENS, bool GATED>
__global__ void __launch_bounds__(kStreamThreads, 1)
mx4_stream_kernel(const ProductArgs p) {
    using S = StreamShape<TOKENS, GATED>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * S::kStages + 5];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile uint32_t failed;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t bar0 = smem_u32(bars);
    const auto full = [&](int s) { return bar0 + 8u * s; };
    const auto empty = [&](int s) { return bar0 + 8u * (S::kStages + s); };
    const auto acc_full = [&](int b) { return bar0 + 8u * (2 * S::kStages + b); };
    const auto acc_empty = [&](int b) { return bar0 + 8u * (2 * S::kStages + 2 + b); };
    const uint32_t drained = bar0 + 8u * (2 * S::kStages + 4);

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(acc_full(b), 1); mbar_init(acc_empty(b), 4); }
        mbar_init(drained, 1);
        failed = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc<1>(smem_u32(&tmem_slot), S::kColumns);
    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    constexpr uint32_t tmem = 0;       // all columns were asked for: the allocation begins at the first

    const int chunks = p.chunks;
    const int64_t units = (int64_t)p.row_tiles * p.token_tiles * chunks;
    const StreamRun run = run_of(units, blockIdx.x, gridDim.x);

    if (warp == 0) {
        if (lane == 0) {
            const int64_t count = run.last - run.first;
            const auto weights = [&](int64_t i) {      // of the run's i-th unit, into its stage
                const int64_t u = run.first + i, tile = u / chunks;
                const int s = (int)(i % S::kStages), k = (int)(u - tile * chunks);
                const int64_t at = mx4_tile_offset(tile / p.token_tiles, k, chunks);
                const uint32_t to = ring + s * S::kStageBytes;
                mbar_expect_tx(full(s), S::kStageBytes);
                bulk_g2s(to, p.w + at, kMx4TileBytes, full(s));
                if (GATED) bulk_g2s(to + kMx4TileBytes, p.w_up + at, kMx4TileBytes, full(s));
            };
            const auto activations = [&](int64_t i) {
                const int64_t u = run.first + i, tile = u / chunks;
                const int s = (int)(i % S::kStages), k = (int)(u - tile * chunks);
                bulk_g2s(ring + s * S::kStageBytes + S::kWeights * kMx4TileBytes, p.x + mx4_tile_offset(tile % p.token_tiles, k, chunks),
                         S::kXBytes, full(s));
            };
            // weights do not depend on the kernel before: the first of them are on their way while it still runs
            const int64_t ahead = p.x_follows ? (count < S::kStages ? count : S::kStages) : 0;
            for (int64_t i = 0; i < ahead; ++i) weights(i);
            if (p.x_follows) asm volatile("griddepcontrol.wait;" ::: "memory");
            for (int64_t i = 0; i < ahead; ++i) activations(i);
            int64_t i = ahead;
            for (; i < count; ++i) {
                if (i >= S::kStages && !bar_wait(empty(i % S::kStages), (uint32_t)(i / S::kStages - 1) & 1u, &failed)) break;
                weights(i);
                activations(i);
            }
            // no copy and no arrival may come after this CTA is gone
            for (int64_t j = i > S::kStages ? i - S::kStages : 0; j < i; ++j) {
                const uint32_t parity = (uint32_t)(j / S::kStages) & 1u;
                if (!bar_wait(empty(j % S::kStages), parity, &failed)) mbar_wait(full(j % S::kStages), parity, kMx4SpinLimit);
            }
        }
    } else if (warp == 1) {
        const uint32_t lead = elect_one();
        int s = 0, segment = 0;
        uint32_t parity = 0;
        for (int64_t u = run.first; u < run.last; ++segment) {
            const int64_t tile = u / chunks;
            const int64_t end = (tile + 1) * chunks < run.last ? (tile + 1) * chunks : run.last;
            const int b = segment % S::kBuffers;
            if (segment >= S::kBuffers && !warp_wait(acc_empty(b), (uint32_t)(segment / S::kBuffers - 1) & 1u, &failed)) break;
            tensor_fence_after();
            uint32_t add = 0u;
            for (; u < end; ++u) {
                if (!warp_wait(full(s), parity, &failed)) break;
                tensor_fence_after();
                const uint32_t stage = ring + s * S::kStageBytes, x = stage + S::kWeights * kMx4TileBytes;
                const uint32_t sf = tmem + S::kScaleBase + s * S::kScaleColumns, sfx = sf + 8 * S::kWeights;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int w = 0; w < S::kWeights; ++w) copy_scales<1>(lead, sf + w * 8 + h * 4, scale_desc(stage + w * kMx4TileBytes) + 32 * h);
                    copy_scales<1>(lead, sfx + h * 4, scale_desc(x) + 32 * h);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {      // 32 bytes on: two in the descriptors' unit
#pragma unroll
                    for (int w = 0; w < S::kWeights; ++w)
                        mx4_multiply<1>(lead, tmem + b * S::kAcc + w * TOKENS, operand_desc(stage + w * kMx4TileBytes + kMx4ScaleBytes) + 2 * j,
                                        operand_desc(x + kMx4ScaleBytes) + 2 * j, mx4_instruction(128, TOKENS, (j & 1) * 2),
                                        sf + w * 8 + (j >> 1) * 4, sfx + (j >> 1) * 4, j ? 1u : add);
                }
                tensor_commit(lead, empty(s));
                add = 1u;
                if (++s == S::kStages) { s = 0; parity ^= 1u; }
            }
            if (u < end) break;
            tensor_commit(lead, acc_full(b));
        }
        tensor_commit(lead, drained);
        warp_wait(drained, 0, &failed);
    } else {
        const int quarter = warp & 3;
        uint32_t* counters = p.workspace + 4096 / 4;
        float* partials = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(p.workspace) + kMx4PartialOffset);
        int segment = 0;
        for (int64_t u = run.first; u < run.last; ++segment) {
            const int64_t tile = u / chunks, from = tile * chunks, to = from + chunks;
            const int64_t end = to < run.last ? to : run.last;
            const int b = segment % S::kBuffers;
            if (!warp_wait(acc_full(b), (uint32_t)(segment / S::kBuffers) & 1u, &failed)) break;
            __syncwarp();
            tensor_fence_after();
            const int row_tile = (int)(tile / p.token_tiles);
            const int64_t token0 = (tile % p.token_tiles) * TOKENS;
            const uint32_t acc = tmem + b * S::kAcc + ((uint32_t)quarter << 21);
            const bool whole = u == from && end == to;
            constexpr int64_t kSlot = (int64_t)S::kAcc * 128;
            float* mine = partials + (2 * (int64_t)blockIdx.x + (segment ? 1 : 0)) * kSlot + quarter * 32 + lane;
            float v[16], up[16];
#pragma unroll 1
            for (int c = 0; c < TOKENS; c += 16) {
                if (token0 + c >= p.tokens) break;
                __syncwarp();
                tmem_load16(acc + c, v);
                if (GATED) tmem_load16(acc + TOKENS + c, up);
                if (whole) {
                    finish16<GATED>(p, row_tile, quarter, lane, token0 + c, v, up);
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        __stcg(mine + (c + i) * 128, v[i]);
                        if (GATED) __stcg(mine + (TOKENS + c + i) * 128, up[i]);
                    }
                }
            }
            tensor_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty(b));
            if (!whole) {
                // every warp's 32 features are counted by themselves, so that no barrier is needed
                const int c0 = cta_of(units, from, gridDim.x), c1 = cta_of(units, to - 1, gridDim.x);
                uint32_t before = 0u;
                __threadfence();
                __syncwarp();
                if (lane == 0) before = atomicAdd(&counters[c0 * 4 + quarter], 1u);
                before = __shfl_sync(0xFFFFFFFFu, before, 0);
                if (before == (uint32_t)(c1 - c0)) {
                    __threadfence();
                    if (lane == 0) counters[c0 * 4 + quarter] = 0u;
                    // c0's part is its last segment, the others' their first; c0 has only one segment where its run begins inside the tile
                    const int64_t at0 = 2 * (int64_t)c0 + (run_of(units, c0, gridDim.x).first / chunks == tile ? 0 : 1);
#pragma unroll 1
                    for (int c = 0; c < TOKENS; c += 16) {
                        if (token0 + c >= p.tokens) break;
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = up[i] = 0.f;
                        for (int g = c0; g <= c1; ++g) {
                            const float* from_g = partials + (g == c0 ? at0 : 2 * (int64_t)g) * kSlot + quarter * 32 + lane;
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                v[i] += __ldcg(from_g + (c + i) * 128);
                                if (GATED) up[i] += __ldcg(from_g + (TOKENS + c + i) * 128);
                            }
                        }
                        finish16<GATED>(p, row_tile, quarter, lane, token0 + c, v, up);
                    }
                }
            }
            u = end;
        }
    }
    __syncwarp();
    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    if (threadIdx.x == 0 && failed) atomicExch(p.workspace, 1u);
    if (warp == 1) tmem_free<1>(tmem_slot, S::kColumns);
}

// ---- many tokens: tokens on the accumulator's lanes ------------------------------------------------
//
// A pair of CTAs on neighbouring SMs works on 256 tokens x 256 features (with a gate: 128 features of both weights): each holds
// 128 tokens and half of the features in shared memory, and one instruction multiplies what both hold, so that a byte of shared memory
// feeds twice the work that it would feed one CTA.  A thread of the epilogue has one token and neighbouring features in its
// registers: an MXFP4 block needs no exchange with other threads, and rows go out in whole sectors.  The accumulator takes all
// but the scales' columns of the tensor memory, so it is read into registers as a whole (some 300 cycles) and multiplied into again
// while it is converted and stored.
//
// Warps: 0 copies, 1 multiplies (first CTA) or hands on the arrival of the copies (second), 2 to 9 take the accumulator over, two
// on each quarter of the lanes, one on each half of the columns.
struct WideShape {
    static constexpr int kCodes = kMx4Rows * kMx4RowBytes;
    static constexpr int kWeightScales = kMx4TileBytes;                     // of a stage: tokens, the weights' scales, their codes
    static constexpr int kWeightCodes = kWeightScales + 2 * kMx4ScaleBytes;
    static constexpr int kStageBytes = kWeightCodes + kCodes;
    static constexpr int kStages = 6;
    static constexpr int kStageRows = kStages * kStageBytes;                // eight warps' rows on their way out, 2 KB each
    static constexpr int kBars = kStageRows + 8 * 2048;
    static constexpr int kSmem = kBars + (2 * kStages + 3) * 8 + 16;
    static constexpr int kScaleBase = 256, kScaleColumns = 24, kColumns = 512;
    static_assert(kScaleBase + kStages * kScaleColumns <= kColumns, "tensor memory");
    static_assert(kStageBytes % 1024 == 0 && kWeightCodes % 1024 == 0, "the swizzle counts from multiples of 1024 bytes");
    static_assert(kSmem <= kMx4SmemMost, "shared memory");
};
constexpr int kWideThreads = 320;

struct WideTile { int token, feature; };      // in units of a pair's tile
__device__ __forceinline__ WideTile wide_tile(int64_t tile, int token_tiles) {
    return {(int)(tile % token_tiles), (int)(tile / token_tiles)};
}

// 32 neighbouring values of one token, as a block.
__device__ __forceinline__ uint4 block_codes(const float* v, uint32_t& byte) {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < 32; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    byte = mx4_scale_byte(m);
    const float inverse = mx4_inverse_scale(byte);
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = byte == 255u ? 0.f : v[j * 8 + i] * inverse;
        w[j] = mx4_codes8(q);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// A warp's 32 tokens x 32 features, a token per lane, go out by way of 2 KB of shared memory: written straight from the registers every
// instruction would touch 32 rows with 16 bytes each.  `w`: 32 values in pairs; rows below `tokens`, columns below `valid` are stored.
__device__ __forceinline__ void store_rows(uint32_t buffer, int lane, const uint32_t* w, uint16_t* out, int64_t stride, int64_t tokens, int valid,
                                           bool even) {
    // a row is four pieces of 16 bytes; two rows share the banks, so the pieces change places with every second row
    const auto place = [&](int row, int piece) { return buffer + row * 64 + ((piece ^ ((row >> 1) & 3)) << 4); };
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 4; ++c)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(place(lane, c)), "r"(w[4 * c]), "r"(w[4 * c + 1]), "r"(w[4 * c + 2]),
                     "r"(w[4 * c + 3]) : "memory");
    __syncwarp();
    if (even && valid >= 32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = i * 8 + (lane >> 2), c = lane & 3;
            uint4 v;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(place(row, c)));
            if (row < tokens) *reinterpret_cast<uint4*>(out + row * stride + c * 8) = v;
        }
    } else {
        const int rows = tokens < 32 ? (int)tokens : 32;
        for (int row = 0; row < rows; ++row) {
            uint16_t v;
            asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(place(row, lane >> 3) + (lane & 7) * 2));
            if (lane < valid) out[row * stride + lane] = v;
        }
    }
}

template <bool GATED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kWideThreads, 1)
mx4_wide_kernel(const ProductArgs p, const bool even) {
    using S = WideShape;
    extern __shared__ __align__(1024) uint8_t ring_bytes[];      // all of the shared memory: rings begin at multiples of 1024
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank();
    const uint32_t ring = smem_u32(ring_bytes), bar0 = ring + S::kBars;
    uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(ring_bytes + S::kSmem - 16);
    volatile uint32_t& failed = *reinterpret_cast<volatile uint32_t*>(ring_bytes + S::kSmem - 12);
    const auto full = [&](int s) { return bar0 + 8u * s; };                       // this CTA's copies have come; in the first CTA, the second's too
    const auto empty = [&](int s) { return bar0 + 8u * (S::kStages + s); };
    const uint32_t acc_full = bar0 + 8u * (2 * S::kStages), acc_empty = acc_full + 8u, drained = acc_full + 16u;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) { mbar_init(full(s), rank == 0 ? 2 : 1); mbar_init(empty(s), 1); }
        mbar_init(acc_full, 1);
        mbar_init(acc_empty, 16);
        mbar_init(drained, 1);
        failed = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc<2>(smem_u32(&tmem_slot), S::kColumns);
    tensor_fence_before();
    __syncthreads();
    cluster_sync();
    tensor_fence_after();
    constexpr uint32_t tmem = 0;       // all columns were asked for: the allocation begins at the first

    const int chunks = p.chunks, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int feature_tiles = GATED ? p.row_tiles : (p.row_tiles + 1) / 2;
    const int64_t tiles = (int64_t)p.token_tiles * feature_tiles;
    const int last_token_tile = (int)((p.tokens - 1) / kMx4Rows);

    if (warp == 0) {
        if (lane == 0) {
            int64_t i = 0;
            bool ok = true;
            if (p.x_follows) asm volatile("griddepcontrol.wait;" ::: "memory");
            for (int64_t tile = pair; tile < tiles && ok; tile += pairs) {
                const WideTile t = wide_tile(tile, p.token_tiles);
                // what lies beyond the last tile of 128 is multiplied as the last and not stored
                const uint8_t* x = p.x + mx4_tile_offset(min(2 * t.token + rank, last_token_tile), 0, chunks);
                const uint8_t* w0 = GATED ? p.w + mx4_tile_offset(t.feature, 0, chunks) : p.w + mx4_tile_offset(2 * t.feature, 0, chunks);
                const uint8_t* w1 = GATED ? p.w_up + mx4_tile_offset(t.feature, 0, chunks)
                                          : p.w + mx4_tile_offset(min(2 * t.feature + 1, p.row_tiles - 1), 0, chunks);
                for (int k = 0; k < chunks; ++k, ++i) {
                    const int s = (int)(i % S::kStages);
                    if (i >= S::kStages && !bar_wait(empty(s), (uint32_t)(i / S::kStages - 1) & 1u, &failed)) { ok = false; break; }
                    const uint32_t to = ring + s * S::kStageBytes;
                    const int64_t at = (int64_t)k * kMx4TileBytes;
                    mbar_expect_tx(full(s), S::kStageBytes);
                    bulk_g2s(to, x + at, kMx4TileBytes, full(s));
                    bulk_g2s(to + S::kWeightScales, w0 + at, kMx4ScaleBytes, full(s));
                    bulk_g2s(to + S::kWeightScales + kMx4ScaleBytes, w1 + at, kMx4ScaleBytes, full(s));
                    bulk_g2s(to + S::kWeightCodes, (rank ? w1 : w0) + at + kMx4ScaleBytes, S::kCodes, full(s));
                }
            }
            for (int64_t j = i > S::kStages ? i - S::kStages : 0; j < i; ++j) {
                const uint32_t parity = (uint32_t)(j / S::kStages) & 1u;
                if (!bar_wait(empty(j % S::kStages), parity, &failed)) mbar_wait(full(j % S::kStages), parity, kMx4SpinLimit);
            }
        }
    } else if (warp == 1) {
        if (rank == 1) {
            const int64_t units = (tiles - pair + pairs - 1) / pairs * chunks;
            if (lane == 0) {
                for (int64_t i = 0; i < units; ++i) {
                    if (!bar_wait(full(i % S::kStages), (uint32_t)(i / S::kStages) & 1u, &failed)) break;
                    arrive_at_first(full(i % S::kStages));
                }
                bar_wait(drained, 0, &failed);
            }
        } else {
            const uint32_t lead = elect_one();
            int s = 0;
            uint32_t parity = 0, round = 0;
            bool ok = true;
            for (int64_t tile = pair; tile < tiles && ok; tile += pairs, ++round) {
                if (round && !warp_wait(acc_empty, (round - 1) & 1u, &failed)) break;
                for (int k = 0; k < chunks; ++k) {
                    if (!warp_wait(full(s), parity, &failed)) { ok = false; break; }
                    tensor_fence_after();
                    const uint32_t stage = ring + s * S::kStageBytes;
                    const uint32_t sfx = tmem + S::kScaleBase + s * S::kScaleColumns, sfw = sfx + 8;
                    const uint64_t x = scale_desc(stage), w = scale_desc(stage + S::kWeightScales);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {      // 512 bytes on: 32 in the descriptors' unit
                        copy_scales<2>(lead, sfx + h * 4, x + 32 * h);
                        copy_scales<2>(lead, sfw + h * 8, w + 32 * h);
                        copy_scales<2>(lead, sfw + h * 8 + 4, w + 64 + 32 * h);
                    }
                    const uint64_t a = operand_desc(stage + kMx4ScaleBytes), b = operand_desc(stage + S::kWeightCodes);
#pragma unroll
                    for (int j = 0; j < 4; ++j)      // 32 bytes on: two in the descriptors' unit
                        mx4_multiply<2>(lead, tmem, a + 2 * j, b + 2 * j, mx4_instruction(256, 256, (j & 1) * 2), sfx + (j >> 1) * 4,
                                        sfw + (j >> 1) * 8, k || j ? 1u : 0u);
                    tensor_commit_pair(lead, empty(s));
                    if (++s == S::kStages) { s = 0; parity ^= 1u; }
                }
                if (ok) tensor_commit_pair(lead, acc_full);
            }
            tensor_commit_pair(lead, drained);
            warp_wait(drained, 0, &failed);
        }
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        uint32_t round = 0;
        for (int64_t tile = pair; tile < tiles; tile += pairs, ++round) {
            if (!warp_wait(acc_full, round & 1u, &failed)) break;
            __syncwarp();
            tensor_fence_after();
            const WideTile t = wide_tile(tile, p.token_tiles);
            const int64_t token0 = ((int64_t)2 * t.token + rank) * kMx4Rows + quarter * 32, tokens = p.tokens - token0;   // this warp's
            const uint32_t acc = tmem + ((uint32_t)quarter << 21), buffer = ring + S::kStageRows + (warp - 2) * 2048;
            uint16_t* rows = static_cast<uint16_t*>(p.out) + token0 * p.out_stride;
            const auto release = [&] {
                tensor_fence_before();
                __syncwarp();
                if (lane == 0) arrive_at_first(acc_empty);
            };
            if (GATED) {
                float g[64], u[64];
#pragma unroll
                for (int c = 0; c < 64; c += 32) {
                    tmem_load32(acc + half * 64 + c, g + c);
                    tmem_load32(acc + 128 + half * 64 + c, u + c);
                }
                release();
                const int first = t.feature * kMx4Rows + half * 64, valid = p.rows - first;
#pragma unroll
                for (int i = 0; i < 64; ++i) g[i] = i < valid ? act(g[i], p.activation) * u[i] : 0.f;
                if (p.out_dtype == MPS_MX4) {
                    const int64_t token = token0 + lane;
                    if (token < p.tokens) {
                        const int out_chunks = (int)mx4_chunks(p.rows), row = (int)(token % kMx4Rows), part = t.feature & 1;
                        uint8_t* to = static_cast<uint8_t*>(p.out) + mx4_tile_offset(token / kMx4Rows, t.feature >> 1, out_chunks);
                        uint32_t b0, b1;
                        *reinterpret_cast<uint4*>(to + mx4_code_offset(row, part * 4 + half * 2)) = block_codes(g, b0);
                        *reinterpret_cast<uint4*>(to + mx4_code_offset(row, part * 4 + half * 2 + 1)) = block_codes(g + 32, b1);
                        *reinterpret_cast<uint16_t*>(to + mx4_scale_offset(row, part) + half * 2) = (uint16_t)(b0 | b1 << 8);
                        if (t.feature == p.row_tiles - 1 && part == 0) {      // fill up the last tile
                            *reinterpret_cast<uint4*>(to + mx4_code_offset(row, 4 + half * 2)) = make_uint4(0u, 0u, 0u, 0u);
                            *reinterpret_cast<uint4*>(to + mx4_code_offset(row, 5 + half * 2)) = make_uint4(0u, 0u, 0u, 0u);
                            *reinterpret_cast<uint16_t*>(to + mx4_scale_offset(row, 1) + half * 2) = 0;
                        }
                    }
                } else {
                    uint32_t w[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) w[i] = pack2(g[2 * i], g[2 * i + 1], p.out_dtype);
#pragma unroll
                    for (int c = 0; c < 64; c += 32) store_rows(buffer, lane, w + c / 2, rows + first + c, p.out_stride, tokens, valid - c, even);
                }
            } else {
                uint32_t w[64];
#pragma unroll
                for (int c = 0; c < 128; c += 32) {
                    float v[32];
                    tmem_load32(acc + half * 128 + c, v);
#pragma unroll
                    for (int i = 0; i < 16; ++i) w[c / 2 + i] = pack2(v[2 * i], v[2 * i + 1], p.out_dtype);
                }
                release();
#pragma unroll
                for (int c = 0; c < 128; c += 32) {
                    const int first = t.feature * 256 + half * 128 + c;
                    store_rows(buffer, lane, w + c / 2, rows + first, p.out_stride, tokens, p.rows - first, even);
                }
            }
        }
    }
    __syncwarp();
    tensor_fence_before();
    __syncthreads();
    cluster_sync();      // what the pair's instructions read and write is there until both are done
    tensor_fence_after();
    if (threadIdx.x == 0 && failed) atomicExch(p.workspace, 1u);
    if (warp == 1) tmem_free<2>(tmem_slot, S::kColumns);
}

template <typename Kernel, typename... More>
static int launch_product(Kernel kernel, int smem, int threads, int ctas, cudaStream_t st, const ProductArgs& p, More... more) {
    MPS_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)ctas);
    config.blockDim = dim3((unsigned)threads);
    config.dynamicSmemBytes = (size_t)smem;
    config.stream = st;
    cudaLaunchAttribute overlap;
    overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    overlap.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &overlap;
    config.numAttrs = p.x_follows ? 1 : 0;
    MPS_CUDA_TRY(cudaLaunchKernelEx(&config, kernel, p, more...));
    return MPS_OK;
}

template <int TOKENS, bool GATED>
static int launch_stream(ProductArgs p, int sms, cudaStream_t st) {
    using S = StreamShape<TOKENS, GATED>;
    p.token_tiles = (int)((p.tokens + TOKENS - 1) / TOKENS);
    const int64_t units = (int64_t)p.row_tiles * p.token_tiles * p.chunks;
    return launch_product(mx4_stream_kernel<TOKENS, GATED>, S::kSmem, kStreamThreads, (int)(units < sms ? units : sms), st, p);
}

template <bool GATED>
static int launch_wide(ProductArgs p, int sms, cudaStream_t st) {
    p.token_tiles = (int)((p.tokens + 255) / 256);
    const int64_t tiles = (int64_t)p.token_tiles * (GATED ? p.row_tiles : (p.row_tiles + 1) / 2);
    const int pairs = (int)(tiles < sms / 2 ? tiles : sms / 2);
    const bool even = p.out_dtype != MPS_MX4 && p.out_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15u) == 0;
    return launch_product(mx4_wide_kernel<GATED>, WideShape::kSmem, kWideThreads, 2 * pairs, st, p, even);
}


static int sm_count(int* sms) {
    int dev = 0;
    MPS_CUDA_TRY(cudaGetDevice(&dev));
    MPS_CUDA_TRY(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev));
    if (*sms > kMx4MostSms) *sms = kMx4MostSms;
    return MPS_OK;
}

}  // namespace mps

using namespace mps;

extern "C" {

int64_t mps_mx4_workspace_bytes(void) { return kMx4WorkspaceBytes; }

int mps_mx4_product(const mps_mx4_linear* args, void* workspace, int64_t workspace_bytes, void* stream) {
    if (!args) { set_error("mps_mx4_product: null arguments"); return MPS_ERR_INVALID; }
    const mps_mx4_linear& a = *args;
    if (a.tokens < 0 || a.tokens > kMx4MostRows || a.rows <= 0 || a.rows > kMx4MostCols || a.cols <= 0 || a.cols > kMx4MostCols) {
        set_error("mps_mx4_product: tokens must be in [0, %lld], rows and cols in [1, %lld]", (long long)kMx4MostRows, (long long)kMx4MostCols);
        return MPS_ERR_INVALID;
    }
    if (a.out_dtype != MPS_BF16 && a.out_dtype != MPS_F16 && !(a.out_dtype == MPS_MX4 && a.w_up)) {
        set_error("mps_mx4_product: the output is BF16 or F16, or MXFP4 where the product is gated");
        return MPS_ERR_INVALID;
    }
    if (a.x_dtype != MPS_MX4 && !mx4_dtype_ok(a.x_dtype)) { set_error("mps_mx4_product: unknown dtype %d", (int)a.x_dtype); return MPS_ERR_INVALID; }
    if (a.w_up && a.activation != MPS_SILU && a.activation != MPS_GELU_TANH) { set_error("mps_mx4_product: unknown activation %d", (int)a.activation); return MPS_ERR_INVALID; }
    if (a.tokens == 0) return MPS_OK;
    if (!workspace || workspace_bytes < kMx4WorkspaceBytes) { set_error("workspace missing or too small"); return MPS_ERR_WORKSPACE; }
    const void* tiles = a.x_dtype == MPS_MX4 ? a.x : a.x_tiles;
    if (!a.x || !tiles || !a.w || !a.out) { set_error("mps_mx4_product: null pointer"); return MPS_ERR_INVALID; }
    if (((reinterpret_cast<uintptr_t>(tiles) | reinterpret_cast<uintptr_t>(a.w) | reinterpret_cast<uintptr_t>(a.w_up) |
          (a.out_dtype == MPS_MX4 ? reinterpret_cast<uintptr_t>(a.out) : 0)) & 15u) || (reinterpret_cast<uintptr_t>(workspace) & 255u)) {
        set_error("mps_mx4_product: tiles must be 16-byte aligned, the workspace 256");
        return MPS_ERR_INVALID;
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int sms = 0, rc = sm_count(&sms);
    if (rc) return rc;
    if (a.x_dtype != MPS_MX4) {
        rc = mps_mx4_quantize(a.x, a.x_dtype, a.tokens, a.cols, a.x_stride, a.x_tiles, stream);
        if (rc) return rc;
    }
    ProductArgs p = {};
    p.x = static_cast<const uint8_t*>(tiles);
    p.w = static_cast<const uint8_t*>(a.w);
    p.w_up = static_cast<const uint8_t*>(a.w_up);
    p.out = a.out;
    p.workspace = static_cast<uint32_t*>(workspace);
    p.out_stride = a.out_stride;
    p.tokens = a.tokens;
    p.rows = (int32_t)a.rows;
    p.chunks = (int32_t)mx4_chunks(a.cols);
    p.row_tiles = (int32_t)mx4_row_tiles(a.rows);
    p.out_dtype = a.out_dtype;
    p.activation = a.activation;
    p.x_follows = a.x_dtype != MPS_MX4;
    if (a.tokens > 128) return a.w_up ? launch_wide<true>(p, sms, st) : launch_wide<false>(p, sms, st);
    if (a.w_up) {
        if (a.tokens <= 16) return launch_stream<16, true>(p, sms, st);
        if (a.tokens <= 32) return launch_stream<32, true>(p, sms, st);
        if (a.tokens <= 64) return launch_stream<64, true>(p, sms, st);
        return launch_stream<128, true>(p, sms, st);
    }
    if (a.tokens <= 16) return launch_stream<16, false>(p, sms, st);
    if (a.tokens <= 32) return launch_stream<32, false>(p, sms, st);
    if (a.tokens <= 64) return launch_stream<64, false>(p, sms, st);
    return launch_stream<128, false>(p, sms, st);
}

int mps_mx4_status(void* workspace, int64_t workspace_bytes, void* stream, int32_t* timed_out) {
    if (!timed_out || !workspace || workspace_bytes < kMx4WorkspaceBytes) { set_error("mps_mx4_status: bad argument"); return MPS_ERR_INVALID; }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    uint32_t flag = 0;
    MPS_CUDA_TRY(cudaMemcpyAsync(&flag, workspace, sizeof(flag), cudaMemcpyDeviceToHost, st));
    MPS_CUDA_TRY(cudaStreamSynchronize(st));
    if (flag) MPS_CUDA_TRY(cudaMemsetAsync(workspace, 0, (size_t)kMx4PartialOffset, st));
    *timed_out = flag ? 1 : 0;
    return MPS_OK;
}

}  // extern "C"
