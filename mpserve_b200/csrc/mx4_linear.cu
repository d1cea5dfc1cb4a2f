// Products of MXFP4 matrices: out[t, r] = sum_k x[t, k] w[r, k], and the gated pair act(x Wg) * (x Wu).
#include "mx4.cuh"
#include "mx4_tensor.cuh"
#include "stream_common.cuh"

#include <atomic>

namespace mps {

// ---- what the kernels share -------------------------------------------------------------------------

constexpr int kMx4SmemMost = 232448;           // 227 KB

constexpr int64_t kMx4WorkspaceBytes = 256;    // word 0 records a wait that ran out

struct ProductArgs {
    const uint8_t* x;        // tiles, or (stream kernel with QUANTIZE) the tokens as they came
    const uint8_t* w;
    const uint8_t* w_up;
    void* out;
    uint32_t* workspace;
    int64_t out_stride, x_stride;
    int64_t tokens;
    int32_t rows, cols;      // of the weight
    int32_t chunks;          // tiles of a row
    int32_t row_tiles, token_tiles, parts;
    int32_t x_dtype, out_dtype, activation;
    bool x_vec;
    bool even;               // rows of an output that is not MXFP4 begin at multiples of 16 bytes
    bool half_values;        // an FP32 output takes F16's values where F16 has them
    bool early;              // the kernel before writes no weight: weights may be read before it is done
};

// Both activations are g / (1 + exp(-t)): SiLU with t = g, and GELU's tanh form since (1 + tanh z) / 2 = 1 / (1 + exp(-2 z)).  CUDA's fast exponential (off by
// 2 + 1.17 |t| units in the last place) and quotient (by 2) are far below what the result is rounded to, 16 bits or 4; with the accurate ones the
// gated epilogue of 256 tokens took 10000 cycles, as long as the multiplications of 4096 columns.
__device__ __forceinline__ float act(float g, bool silu) {
    const float t = silu ? g : 1.5957691216057308f * g * fmaf(0.044715f * g, g, 1.f);
    return __fdividef(g, 1.f + __expf(-t));
}

// What F16 holds of a value, and the value itself where that would be an infinity: F16's precision with FP32's range.
__device__ __forceinline__ float half_value(float v) {
    const float h = __half2float(__float2half_rn(v));
    return isinf(h) ? v : h;
}

// ---- few tokens: weights on the accumulator's lanes -------------------------------------------------
//
// A CTA streams the weight tiles of 128 features through a ring in shared memory, 17 KB a bulk copy; TOKENS tokens (16 to 128) are the
// product's narrow side.  Two CTAs share an SM, and a cluster of up to four shares the columns of one tile of the output, as many as
// fill the GPU: then every SM has some 200 KB under way, and all end together.  The parts of a tile meet in the cluster's shared memory,
// where every CTA adds up a share of the tokens, always in the same order.  Up to 32 tokens (16 with a gate) each sends its parts to where they are
// added, as they come out of the accumulator, and a barrier there counts them: nothing but that barrier is waited for (1 token through 14336 x 4096
// 7.4 us).  More would take stages from the ring; they take its place, and the adding CTA fetches them between two barriers of the whole cluster
// (1 token 7.9 us that way; 64 tokens through 4096 x 14336 9.8 us, sent 10.2).
//
// Warps: 0 copies, 1 multiplies, the next four or eight take the accumulator over, one or two on each quarter of its lanes (four launch a little
// sooner, 1 token 7.4 us and with eight 7.6; eight are done sooner where there are more tokens, the gated pair for 64 17.4 us and with four 18.4); all of them add the
// parts up.  With QUANTIZE, one more for every stage of the ring quantises the tokens' columns on their way into it, instead of a kernel before this one.
template <int TOKENS, bool GATED>
struct StreamShape {
    static constexpr int kWeights = GATED ? 2 : 1;
    static constexpr int kTakeOver = TOKENS <= 16 ? 4 : 8, kWarps = 2 + kTakeOver;
    static constexpr int kXBytes = kMx4ScaleBytes + TOKENS * kMx4RowBytes;
    static constexpr int kStageBytes = kWeights * kMx4TileBytes + kXBytes;
    static constexpr int kMost = 115712 - 1024;                 // of an SM's 228 KB, for two CTAs and the KB that each costs
    static constexpr int kAcc = TOKENS * kWeights;              // columns of the accumulator
    static constexpr bool kSend = kAcc <= 32;
    static constexpr int kStages = (kMost - (kSend ? kAcc * 512 : 0)) / kStageBytes;
    static constexpr int kReceived = kStages * kStageBytes;     // where the parts of this CTA's tokens come in
    static constexpr int kBars = kReceived + (kSend ? kAcc * 512 : 0);
    static constexpr int kSmem = kBars + (2 * kStages + 3) * 8 + 16;
    static constexpr int kScaleColumns = 8 * kWeights + 8;      // of one stage
    static constexpr int kUsed = kAcc + kStages * kScaleColumns;
    static constexpr int kColumns = kUsed <= 128 ? 128 : 256;   // an allocation is a power of two
    static_assert(kUsed <= kColumns, "tensor memory");
    static_assert(kStageBytes % 1024 == 0, "the swizzle counts from multiples of 1024 bytes");
    static_assert(kAcc * 128 * 4 <= kReceived, "a part of the accumulator takes the ring's place");
};
// Tokens that the kernel quantises itself.  us, inside | by a kernel before it: 14336 x 4096, 1 token 7.7 | 8.8, 8: 9.2 | 9.6, 9: 9.9 | 9.6, 16: 12.3 | 9.7
// (1024 x 4096 3.1 | 4.7, 3.9 | 5.2, 4.2 | 5.2, 5.3 | 5.3); and a launch and a buffer less for the host.
constexpr int kMostQuantizedInside = MPS_MX4_TOKENS_INSIDE;
static_assert(kMostQuantizedInside <= 16, "the kernel that quantises has 16 tokens");
constexpr int kMostParts = 4;                  // CTAs of a cluster

// One token of a tile's 128 features, four neighbouring ones a lane (`up` too where the pair is gated), into the output.
template <bool GATED>
__device__ __forceinline__ void finish(const ProductArgs& p, int row_tile, int lane, int64_t token, float4 v, float4 up) {
    const int first = row_tile * kMx4Rows + lane * 4, valid = p.rows - first;
    float f[4] = {v.x, v.y, v.z, v.w};
    if (GATED) {
        const float u[4] = {up.x, up.y, up.z, up.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = i < valid ? act(f[i], p.activation == MPS_SILU) * u[i] : 0.f;
    }
    if (GATED && p.out_dtype == MPS_MX4) {
        // eight lanes hold a block
        uint32_t m = 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max(m, __float_as_uint(f[i]) & 0x7FFFFFFFu);
#pragma unroll
        for (int o = 1; o < 8; o *= 2) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        const uint32_t byte = mx4_scale_byte(m);
        const float inverse = mx4_inverse_scale(byte);
        float q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = i < 4 && byte != 255u ? f[i & 3] * inverse : 0.f;
        const int part = row_tile & 1, block = part * 4 + (lane >> 3), row = (int)(token % kMx4Rows);
        uint8_t* tile = static_cast<uint8_t*>(p.out) + mx4_tile_offset(token / kMx4Rows, row_tile >> 1, mx4_chunks(p.rows));
        *reinterpret_cast<uint16_t*>(tile + mx4_code_offset(row, block) + (lane & 7) * 2) = (uint16_t)mx4_codes8(q);
        if ((lane & 7) == 0) tile[mx4_scale_offset(row, part) + (lane >> 3)] = (uint8_t)byte;
        if (row_tile == p.row_tiles - 1 && part == 0) {
            // the second half of the last tile lies beyond the last feature and is filled up with zeros
            *reinterpret_cast<uint16_t*>(tile + mx4_code_offset(row, block + 4) + (lane & 7) * 2) = 0;
            if (lane == 0) *reinterpret_cast<uint32_t*>(tile + mx4_scale_offset(row, 1)) = 0u;
        }
        return;
    }
    if (!GATED && p.out_dtype == MPS_F32) {
        float* out = static_cast<float*>(p.out) + token * p.out_stride + first;
        if (p.half_values) {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = half_value(f[i]);
        }
        if (valid >= 4 && p.even) {
            *reinterpret_cast<float4*>(out) = make_float4(f[0], f[1], f[2], f[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) if (i < valid) out[i] = f[i];
        }
        return;
    }
    uint16_t* out = static_cast<uint16_t*>(p.out) + token * p.out_stride + first;
    const uint2 w = make_uint2(pack2(f[0], f[1], p.out_dtype), pack2(f[2], f[3], p.out_dtype));
    if (valid >= 4 && p.even) {
        *reinterpret_cast<uint2*>(out) = w;
    } else {
        if (valid > 0) out[0] = (uint16_t)w.x;
        if (valid > 1) out[1] = (uint16_t)(w.x >> 16);
        if (valid > 2) out[2] = (uint16_t)w.y;
        if (valid > 3) out[3] = (uint16_t)(w.y >> 16);
    }
}

template <int TOKENS, bool GATED, bool QUANTIZE>
__global__ void __launch_bounds__((StreamShape<TOKENS, GATED>::kWarps + (QUANTIZE ? StreamShape<TOKENS, GATED>::kStages : 0)) * 32, 2)
mx4_stream_kernel(const ProductArgs p) {
    using S = StreamShape<TOKENS, GATED>;
    extern __shared__ __align__(1024) uint8_t ring_bytes[];      // all of the shared memory: rings begin at multiples of 1024
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t ring = smem_u32(ring_bytes), bar0 = ring + S::kBars;
    uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(ring_bytes + S::kSmem - 16);
    volatile uint32_t& failed = *reinterpret_cast<volatile uint32_t*>(ring_bytes + S::kSmem - 12);
    const auto full = [&](int s) { return bar0 + 8u * s; };
    const auto empty = [&](int s) { return bar0 + 8u * (S::kStages + s); };
    const uint32_t acc_full = bar0 + 8u * (2 * S::kStages), drained = acc_full + 8u, received = acc_full + 16u;

    // this CTA's tile of the output, and its share of the columns
    const int part = blockIdx.x % p.parts, chunks = p.chunks;
    const int64_t tile = blockIdx.x / p.parts;
    const int row_tile = (int)(tile / p.token_tiles);
    const int64_t token0 = (tile % p.token_tiles) * TOKENS;
    const int tokens = (int)min((int64_t)TOKENS, p.tokens - token0);
    const int k0 = (int)((int64_t)chunks * part / p.parts), k1 = (int)((int64_t)chunks * (part + 1) / p.parts);
    const bool send = S::kSend && p.parts > 1;
    const int shares = (tokens + p.parts - 1) / p.parts;        // tokens of a part: every parts-th, from its own number on

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) { mbar_init(full(s), QUANTIZE ? 2 : 1); mbar_init(empty(s), 1); }
        mbar_init(acc_full, 1);
        mbar_init(drained, 1);
        mbar_init(received, 1);
        failed = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (send) mbar_expect_tx(received, (uint32_t)((tokens - part + p.parts - 1) / p.parts * p.parts * S::kWeights * 512));
    }
    if (warp == 1) tmem_alloc<1>(smem_u32(&tmem_slot), S::kColumns);
    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    if (send) cluster_arrive();      // `received` can be sent to
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, tmem_slot, 0);

    if (warp == 0) {
        if (lane == 0) {
            const uint8_t* w = p.w + mx4_tile_offset(row_tile, 0, chunks);
            const uint8_t* w_up = GATED ? p.w_up + mx4_tile_offset(row_tile, 0, chunks) : nullptr;
            const uint8_t* x = QUANTIZE ? nullptr : p.x + mx4_tile_offset(tile % p.token_tiles, 0, chunks);
            const auto weights = [&](int k, int s) {
                const uint32_t to = ring + s * S::kStageBytes;
                mbar_expect_tx(full(s), S::kStageBytes - (QUANTIZE ? S::kXBytes : 0));
                bulk_g2s(to, w + (int64_t)k * kMx4TileBytes, kMx4TileBytes, full(s));
                if (GATED) bulk_g2s(to + kMx4TileBytes, w_up + (int64_t)k * kMx4TileBytes, kMx4TileBytes, full(s));
            };
            const auto activations = [&](int k, int s) {
                if (!QUANTIZE) bulk_g2s(ring + s * S::kStageBytes + S::kWeights * kMx4TileBytes, x + (int64_t)k * kMx4TileBytes, S::kXBytes, full(s));
            };
            // weights that the kernel before does not write are on their way while it still runs
            const int ahead = p.early ? min(k1 - k0, S::kStages) : 0;
            for (int i = 0; i < ahead; ++i) weights(k0 + i, i);
            griddep_wait();
            for (int i = 0; i < ahead; ++i) activations(k0 + i, i);
            griddep_launch();
            int k = k0 + ahead;
            for (; k < k1; ++k) {
                const int i = k - k0, s = i % S::kStages;
                if (i >= S::kStages && !bar_wait(empty(s), (uint32_t)(i / S::kStages - 1) & 1u, &failed)) break;
                weights(k, s);
                activations(k, s);
            }
            // no copy and no arrival may come after this CTA is gone
            for (int i = max(0, k - k0 - S::kStages); i < k - k0; ++i) {
                const uint32_t parity = (uint32_t)(i / S::kStages) & 1u;
                if (!bar_wait(empty(i % S::kStages), parity, &failed)) mbar_wait(full(i % S::kStages), parity, kMx4SpinLimit);
            }
        }
    } else if (warp == 1) {
        const uint32_t lead = elect_one();
        int s = 0;
        uint32_t parity = 0, add = 0;
        bool ok = true;
        for (int k = k0; k < k1; ++k) {
            ok = warp_wait(full(s), parity, &failed);
            if (!ok) break;
            tensor_fence_after();
            const uint32_t stage = ring + s * S::kStageBytes, x = stage + S::kWeights * kMx4TileBytes;
            const uint32_t sf = tmem + S::kAcc + s * S::kScaleColumns, sfx = sf + 8 * S::kWeights;
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
                    mx4_multiply<1>(lead, tmem + w * TOKENS, operand_desc(stage + w * kMx4TileBytes + kMx4ScaleBytes) + 2 * j,
                                    operand_desc(x + kMx4ScaleBytes) + 2 * j, mx4_instruction(128, TOKENS, (j & 1) * 2),
                                    sf + w * 8 + (j >> 1) * 4, sfx + (j >> 1) * 4, j ? 1u : add);
            }
            tensor_commit(lead, empty(s));
            add = 1u;
            if (++s == S::kStages) { s = 0; parity ^= 1u; }
        }
        if (ok) tensor_commit(lead, acc_full);
        tensor_commit(lead, drained);
        warp_wait(drained, 0, &failed);
    } else if (warp < S::kWarps) {
        // the accumulator, token by token, to where the parts meet, or to where the ring was: what that held has been multiplied
        const int feature = (warp & 3) * 32 + lane;
        const uint32_t acc = tmem + ((uint32_t)(warp & 3) << 21);
        const bool ok = warp_wait(acc_full, 0, &failed);
        tensor_fence_after();
        if (send) cluster_wait();
        if (ok) {
#pragma unroll 1
            for (int c = ((warp - 2) >> 2) * 16; c < S::kAcc; c += S::kTakeOver * 4) {
                const int w = c / TOKENS, t0 = c % TOKENS;
                if (t0 >= tokens) continue;
                float v[16];
                tmem_load16(acc + c, v);
                if (send) {
                    const uint32_t to = ring + S::kReceived + ((w * p.parts + part) * shares * 128 + feature) * 4;
                    const int shift = __ffs(p.parts) - 1;      // parts are a power of two
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int t = t0 + i, owner = t & (p.parts - 1);
                        if (t < tokens) send_to(peer_address(to + (t >> shift) * 512, owner), peer_address(received, owner), v[i]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) asm volatile("st.shared.f32 [%0], %1;" ::"r"(ring + ((c + i) * 128 + feature) * 4), "f"(v[i]) : "memory");
                }
            }
        }
    } else {
        // Each has one stage, and so sees every phase of its barriers: a wait for a parity is right only for who has seen the phase before.
        const int rows = tokens, s = warp - S::kWarps;
        uint8_t* to = ring_bytes + s * S::kStageBytes + S::kWeights * kMx4TileBytes;
        griddep_wait();
        for (int i = s; i < k1 - k0; i += S::kStages) {
            const int64_t c = (int64_t)(k0 + i) * kMx4Cols + lane * 8, left = p.cols - c;
            const bool simple = p.x_vec && p.x_dtype != MPS_F32 && (int64_t)(k0 + i + 1) * kMx4Cols <= p.cols;
            bool ok = true;
            for (int r = 0; r < rows; r += 4) {
                Raw8 raw[4];
                if (simple) {       // no branch between the loads, so that they are under way together
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        raw[j].a = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.x) + (token0 + min(r + j, rows - 1)) * p.x_stride + c);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        raw[j] = load_raw8(p.x, p.x_dtype, (token0 + r + j) * p.x_stride + c, r + j >= rows ? 0 : left > 8 ? 8 : (int)left, p.x_vec);
                }
                if (r == 0 && i >= S::kStages) ok = warp_wait(empty(s), (uint32_t)(i / S::kStages - 1) & 1u, &failed);
                if (!ok) break;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (r + j >= rows) break;
                    float v[8];
                    unpack8(raw[j], p.x_dtype, v);
                    mx4_store_row(to, r + j, lane, v);
                }
            }
            if (!ok) break;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // the tensor core reads what was written here
            __syncwarp();
            if (lane == 0) mbar_arrive(full(s));
        }
    }
    __syncwarp();
    tensor_fence_before();
    // The parts meet: every warp of the cluster takes a token in turn.  (The code is short on purpose: it runs once, and what it costs is to fetch it.)
    const int warps = blockDim.x >> 5;
    if (send) {
        if (warp < 2 || warp >= S::kWarps) cluster_wait();      // the other warps have
        cluster_arrive();
        if (warp_wait<true>(received, 0, &failed)) {
#pragma unroll 1
            for (int i = warp; i * p.parts + part < tokens; i += warps) {
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f), up = v;
#pragma unroll
                for (int g = 0; g < kMostParts; ++g) {
                    if (g < p.parts) {
                        const uint8_t* from = ring_bytes + S::kReceived + ((g * shares + i) * 128 + lane * 4) * 4;
                        add4(v, *reinterpret_cast<const float4*>(from));
                        if (GATED) add4(up, *reinterpret_cast<const float4*>(from + p.parts * shares * 512));
                    }
                }
                finish<GATED>(p, row_tile, lane, token0 + i * p.parts + part, v, up);
            }
        }
        __syncwarp();
        cluster_wait();      // nobody leaves before all have sent: they long have
    } else {
        if (p.parts > 1) cluster_sync(); else __syncthreads();
        if (!failed) {
#pragma unroll 1
            for (int c = warp * p.parts + part; c < tokens; c += warps * p.parts) {
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f), up = v;
#pragma unroll
                for (int g = 0; g < kMostParts; ++g) {
                    if (g < p.parts) {
                        const uint32_t from = p.parts > 1 ? peer_address(ring + c * 512 + lane * 16, g) : ring + c * 512 + lane * 16;
                        add4(v, load_peer(from));
                        if (GATED) add4(up, load_peer(from + TOKENS * 512));
                    }
                }
                finish<GATED>(p, row_tile, lane, token0 + c, v, up);
            }
        }
        __syncwarp();
        if (p.parts > 1) cluster_sync();       // nobody leaves while his part is read
    }
    __syncthreads();
    tensor_fence_after();
    if (threadIdx.x == 0 && failed) atomicExch(p.workspace, 1u);
    if (warp == 1) tmem_free<1>(tmem, S::kColumns);
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
// The copies of both CTAs count at the first one's barrier, whose thread issues the multiplications, so they are tiled copies: a tile is 17 rows of 1 KB,
// the scales the first, and box and coordinates say which are wanted.  (With untiled copies, which count at their own CTA's barriers, the second
// CTA has to hand every stage on with a release at cluster scope: 4096 x 4096 x 14336 took 164 us that way, and takes 98.5.)
//
// Warps: 0 copies, 1 multiplies (first CTA only), 2 to 9 take the accumulator over, two
// on each quarter of the lanes, one on each half of the columns.
struct WideMaps { CUtensorMap x, w_scales, w_codes, up_scales, up_codes; };
constexpr int kMx4MapRow = 1024, kMx4TileMapRows = kMx4TileBytes / kMx4MapRow;

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
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 32; i += 2) m = max_abs3(m, v[i], v[i + 1]);
    byte = mx4_scale_byte(__float_as_uint(m) & 0x7FFFFFFFu);
    const float inverse = mx4_inverse_scale(byte);
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = v[j * 8 + i] * inverse;      // of a NaN block, whatever it gives: its codes say nothing
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

// OUT32: an FP32 output, of a product that is not gated.  Its rows go out as rows of twice as many 16-bit halves.
template <bool GATED, bool OUT32>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kWideThreads, 1)
mx4_wide_kernel(const ProductArgs p, const __grid_constant__ WideMaps maps) {
    using S = WideShape;
    extern __shared__ __align__(1024) uint8_t ring_bytes[];      // all of the shared memory: rings begin at multiples of 1024
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank();
    const uint32_t ring = smem_u32(ring_bytes), bar0 = ring + S::kBars;
    uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(ring_bytes + S::kSmem - 16);
    volatile uint32_t& failed = *reinterpret_cast<volatile uint32_t*>(ring_bytes + S::kSmem - 12);
    const auto full = [&](int s) { return bar0 + 8u * s; };                       // both CTAs' copies have come; the first CTA's
    const auto empty = [&](int s) { return bar0 + 8u * (S::kStages + s); };
    const uint32_t acc_full = bar0 + 8u * (2 * S::kStages), acc_empty = acc_full + 8u, drained = acc_full + 16u;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        mbar_init(acc_full, 1);
        mbar_init(acc_empty, 16);
        mbar_init(drained, 1);
        failed = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc<2>(smem_u32(&tmem_slot), S::kColumns);
    tensor_fence_before();
    __syncthreads();
    cluster_arrive();      // barriers can be arrived at from the other CTA
    cluster_wait();
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
            prefetch_map(&maps.x);
            prefetch_map(&maps.w_scales);
            prefetch_map(GATED && rank ? &maps.up_codes : &maps.w_codes);
            if (GATED) prefetch_map(&maps.up_scales);
            griddep_wait();
            griddep_launch();
            for (int64_t tile = pair; tile < tiles && ok; tile += pairs) {
                const WideTile t = wide_tile(tile, p.token_tiles);
                // what lies beyond the last tile of 128 is multiplied as the last and not stored
                const auto row_of = [&](int64_t row_tile) { return (int)(row_tile * chunks * kMx4TileMapRows); };
                const int x = row_of(min(2 * t.token + rank, last_token_tile));
                const int w0 = row_of(GATED ? t.feature : 2 * t.feature), w1 = row_of(GATED ? t.feature : min(2 * t.feature + 1, p.row_tiles - 1));
                const CUtensorMap* scales1 = GATED ? &maps.up_scales : &maps.w_scales;
                const CUtensorMap* codes = GATED && rank ? &maps.up_codes : &maps.w_codes;
                for (int k = 0; k < chunks; ++k, ++i) {
                    const int s = (int)(i % S::kStages);
                    if (i >= S::kStages && !bar_wait<true>(empty(s), (uint32_t)(i / S::kStages - 1) & 1u, &failed)) { ok = false; break; }
                    const uint32_t to = ring + s * S::kStageBytes, bar = peer_address(full(s), 0);
                    const int at = k * kMx4TileMapRows;
                    if (rank == 0) mbar_expect_tx(full(s), 2 * S::kStageBytes);
                    tiled_g2s_pair(to, &maps.x, x + at, bar);
                    tiled_g2s_pair(to + S::kWeightScales, &maps.w_scales, w0 + at, bar);
                    tiled_g2s_pair(to + S::kWeightScales + kMx4ScaleBytes, scales1, w1 + at, bar);
                    tiled_g2s_pair(to + S::kWeightCodes, codes, (rank ? w1 : w0) + at + 1, bar);
                }
            }
            // Copies that nobody multiplied come all the same, before this CTA is gone.  (The second CTA's count at the other's barrier: its own is never
            // arrived at, and the wait there lasts for its 1024 polls, 4 ms, a thousand times what a copy takes.)
            for (int64_t j = i > S::kStages ? i - S::kStages : 0; j < i; ++j) {
                const uint32_t parity = (uint32_t)(j / S::kStages) & 1u;
                if (!bar_wait<true>(empty(j % S::kStages), parity, &failed)) mbar_wait(full(j % S::kStages), rank ? 0u : parity, rank ? 1024u : kMx4SpinLimit);
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t lead = elect_one();
            int s = 0;
            uint32_t parity = 0, round = 0;
            bool ok = true;
            for (int64_t tile = pair; tile < tiles && ok; tile += pairs, ++round) {
                if (round && !warp_wait<true>(acc_empty, (round - 1) & 1u, &failed)) break;
                for (int k = 0; k < chunks; ++k) {
                    if (!warp_wait<true>(full(s), parity, &failed)) { ok = false; break; }
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
            tensor_commit_pair<1>(lead, drained);      // the second CTA leaves when the first does; a wait of its own would have to outlast the kernel
            warp_wait(drained, 0, &failed);
        }
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        uint32_t round = 0;
        for (int64_t tile = pair; tile < tiles; tile += pairs, ++round) {
            if (!warp_wait<true>(acc_full, round & 1u, &failed)) break;
            __syncwarp();
            tensor_fence_after();
            const WideTile t = wide_tile(tile, p.token_tiles);
            const int64_t token0 = ((int64_t)2 * t.token + rank) * kMx4Rows + quarter * 32, tokens = p.tokens - token0;   // this warp's
            const uint32_t acc = tmem + ((uint32_t)quarter << 21), buffer = ring + S::kStageRows + (warp - 2) * 2048;
            uint16_t* rows = static_cast<uint16_t*>(p.out) + token0 * p.out_stride * (OUT32 ? 2 : 1);
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
                for (int i = 0; i < 64; ++i) g[i] = act(g[i], p.activation == MPS_SILU) * u[i];
                if (valid < 64) {
#pragma unroll
                    for (int i = 0; i < 64; ++i) if (i >= valid) g[i] = 0.f;
                }
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
                    for (int c = 0; c < 64; c += 32) store_rows(buffer, lane, w + c / 2, rows + first + c, p.out_stride, tokens, valid - c, p.even);
                }
            } else if (OUT32) {
                float v[128];
#pragma unroll
                for (int c = 0; c < 128; c += 32) tmem_load32(acc + half * 128 + c, v + c);
                release();
                if (p.half_values) {
#pragma unroll
                    for (int i = 0; i < 128; ++i) v[i] = half_value(v[i]);
                }
#pragma unroll
                for (int c = 0; c < 128; c += 16) {
                    const int first = t.feature * 256 + half * 128 + c;
                    store_rows(buffer, lane, reinterpret_cast<const uint32_t*>(v + c), rows + 2 * (int64_t)first, 2 * p.out_stride, tokens, 2 * (p.rows - first), p.even);
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
                    store_rows(buffer, lane, w + c / 2, rows + first, p.out_stride, tokens, p.rows - first, p.even);
                }
            }
        }
    }
    __syncwarp();
    tensor_fence_before();
    __syncthreads();
    cluster_sync();      // what the pair's instructions read and write, and the barriers that one arrives at in the other, are there until both are done
    tensor_fence_after();
    if (threadIdx.x == 0 && failed) atomicExch(p.workspace, 1u);
    if (warp == 1) tmem_free<2>(tmem_slot, S::kColumns);
}

// Every launch may begin while the kernel before it in its stream ends: what it reads of it, and all it writes, comes after griddep_wait.
// What is set once per kernel and device is remembered in `ready`, a bit a device.
template <typename... Args>
static int launch_product(void (*kernel)(Args...), std::atomic<uint64_t>& ready, const Device& d, int smem, int threads, int ctas, int cluster,
                          cudaStream_t st, const Args&... args) {
    if (!(ready.load(std::memory_order_relaxed) >> d.ordinal & 1)) {
        MPS_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        MPS_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
        ready.fetch_or(uint64_t(1) << d.ordinal, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)ctas);
    config.blockDim = dim3((unsigned)threads);
    config.dynamicSmemBytes = (size_t)smem;
    config.stream = st;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = (unsigned)cluster;
    attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = cluster > 1 ? 2 : 1;
    MPS_CUDA_TRY(cudaLaunchKernelEx(&config, kernel, args...));
    return MPS_OK;
}

// CTAs that share a tile's columns: a power of two (three took longer than two: 384 tokens, 14336 x 4096, 26 us against 19 for 512), at most what fills
// every SM with two.
static int parts_of(int64_t tiles, int chunks, int sms) {
    int parts = 1;
    while (parts < kMostParts && 2 * parts * tiles <= 2 * sms && 2 * parts <= chunks) parts *= 2;
    return parts;
}

template <int TOKENS, bool GATED, bool QUANTIZE = false>
static int launch_stream(ProductArgs p, const Device& d, cudaStream_t st) {
    using S = StreamShape<TOKENS, GATED>;
    static std::atomic<uint64_t> ready{0};
    p.token_tiles = (int)((p.tokens + TOKENS - 1) / TOKENS);
    const int64_t tiles = (int64_t)p.row_tiles * p.token_tiles;
    if (tiles * kMostParts > 0x7FFFFFFF) { set_error("mps_mx4_product: output too large"); return MPS_ERR_INVALID; }
    p.parts = parts_of(tiles, p.chunks, d.sms);
    return launch_product(mx4_stream_kernel<TOKENS, GATED, QUANTIZE>, ready, d, S::kSmem, (S::kWarps + (QUANTIZE ? S::kStages : 0)) * 32,
                          (int)tiles * p.parts, p.parts, st, p);
}

// Whether 128 tokens a tile with the weights on the lanes take less time than 256 with the tokens on the lanes, by an estimate of both: so much for a launch,
// a tile of K and a further round of CTAs.  It is there to be compared, not to be read: where a cluster adds parts up the streaming kernel takes up to
// 1.6 times as long.  Measured, stream | wide, us: 14336 x 4096, 128 tokens 12.0 | 12.1, 160: 14.1 | 12.1, 384: 24.3 | 18.8, 512: 25.8 | 18.9; 4096 x 14336,
// 128: 12.1 | 25.0, 512: 19.0 | 25.3, 1024: 29.9 | 26.1; 4096 x 4096, 256: 10.0 | 10.6, 1024: 13.2 | 11.3; 517 x 1000, 1024: 7.4 | 9.2.  It takes the shorter
// one at each of these.
static bool stream_pays(const ProductArgs& p, int sms) {
    const int64_t tiles = (int64_t)p.row_tiles * ((p.tokens + 127) / 128), wide = (int64_t)((p.row_tiles + 1) / 2) * ((p.tokens + 255) / 256);
    const int parts = parts_of(tiles, p.chunks, sms);
    const int64_t waves = (tiles * parts + 2 * sms - 1) / (2 * sms), rounds = (wide + sms / 2 - 1) / (sms / 2);
    return 4.2 + (double)waves * 0.54 * ((p.chunks + parts - 1) / parts) + 2.5 * (double)(waves - 1) < 5.5 + (double)rounds * 0.39 * p.chunks;
}

// Tiles as rows of 1 KB, `box` of them a copy.
using EncodeTiled = decltype(&cuTensorMapEncodeTiled);
static int tile_map(CUtensorMap& map, EncodeTiled encode, const void* tiles, int64_t row_tiles, int chunks, int box) {
    const cuuint64_t size[2] = {kMx4MapRow / 4, (cuuint64_t)(row_tiles * chunks * kMx4TileMapRows)}, stride[1] = {kMx4MapRow};
    const cuuint32_t boxes[2] = {kMx4MapRow / 4, (cuuint32_t)box}, steps[2] = {1, 1};
    if (size[1] > 0x7FFFFFFFu) { set_error("mps_mx4_product: matrix too large"); return MPS_ERR_INVALID; }
    const CUresult r = encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(tiles), size, stride, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? MPS_OK : cuda_fail(static_cast<cudaError_t>(r), "cuTensorMapEncodeTiled");      // the two count their errors alike
}
int tensor_map_encoder(EncodeTiled& encode) {
    static std::atomic<EncodeTiled> known{nullptr};
    encode = known.load(std::memory_order_relaxed);
    if (!encode) {
        void* entry = nullptr;
        cudaDriverEntryPointQueryResult found;
        MPS_CUDA_TRY(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &entry, 12000, cudaEnableDefault, &found));
        if (found != cudaDriverEntryPointSuccess || !entry) { set_error("the driver has no cuTensorMapEncodeTiled"); return MPS_ERR_UNSUPPORTED; }
        encode = reinterpret_cast<EncodeTiled>(entry);
        known.store(encode, std::memory_order_relaxed);
    }
    return MPS_OK;
}
static int wide_maps(WideMaps& m, const ProductArgs& p) {
    EncodeTiled encode;
    const int found = tensor_map_encoder(encode);
    if (found) return found;
    int rc = tile_map(m.x, encode, p.x, mx4_row_tiles(p.tokens), p.chunks, kMx4TileMapRows);
    if (!rc) rc = tile_map(m.w_scales, encode, p.w, p.row_tiles, p.chunks, 1);
    if (!rc) rc = tile_map(m.w_codes, encode, p.w, p.row_tiles, p.chunks, kMx4TileMapRows - 1);
    if (!rc && p.w_up) rc = tile_map(m.up_scales, encode, p.w_up, p.row_tiles, p.chunks, 1);
    if (!rc && p.w_up) rc = tile_map(m.up_codes, encode, p.w_up, p.row_tiles, p.chunks, kMx4TileMapRows - 1);
    return rc;
}

template <bool GATED, bool OUT32 = false>
static int launch_wide(ProductArgs p, const Device& d, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};
    WideMaps maps = {};
    const int rc = wide_maps(maps, p);
    if (rc) return rc;
    p.token_tiles = (int)((p.tokens + 255) / 256);
    const int64_t tiles = (int64_t)p.token_tiles * (GATED ? p.row_tiles : (p.row_tiles + 1) / 2);
    const int pairs = (int)(tiles < d.sms / 2 ? tiles : d.sms / 2);
    return launch_product(mx4_wide_kernel<GATED, OUT32>, ready, d, WideShape::kSmem, kWideThreads, 2 * pairs, 1, st, p, maps);
}

// `half_values`: of an FP32 output (ProductArgs).
static int product(const mps_mx4_linear& a, bool half_values, void* workspace, int64_t workspace_bytes, void* stream) {
    if (a.tokens < 0 || a.tokens > kMx4MostRows || a.rows <= 0 || a.rows > kMx4MostCols || a.cols <= 0 || a.cols > kMx4MostCols) {
        set_error("mps_mx4_product: tokens must be in [0, %lld], rows and cols in [1, %lld]", (long long)kMx4MostRows, (long long)kMx4MostCols);
        return MPS_ERR_INVALID;
    }
    if (a.out_dtype != MPS_BF16 && a.out_dtype != MPS_F16 && a.out_dtype != (a.w_up ? MPS_MX4 : MPS_F32)) {
        set_error("mps_mx4_product: the output is BF16 or F16, or MXFP4 where the product is gated and FP32 where it is not");
        return MPS_ERR_INVALID;
    }
    if (a.x_dtype != MPS_MX4 && !mx4_dtype_ok(a.x_dtype)) { set_error("mps_mx4_product: unknown dtype %d", (int)a.x_dtype); return MPS_ERR_INVALID; }
    if (a.w_up && a.activation != MPS_SILU && a.activation != MPS_GELU_TANH) { set_error("mps_mx4_product: unknown activation %d", (int)a.activation); return MPS_ERR_INVALID; }
    if (a.tokens == 0) return MPS_OK;
    if (!workspace || workspace_bytes < kMx4WorkspaceBytes) { set_error("workspace missing or too small"); return MPS_ERR_WORKSPACE; }
    if (!a.x || !a.w || !a.out) { set_error("mps_mx4_product: null pointer"); return MPS_ERR_INVALID; }
    const bool quantized = a.x_dtype == MPS_MX4, inside = !quantized && a.tokens <= kMostQuantizedInside;
    const void* tiles = a.x;
    if (!quantized && !inside) {
        // not in the workspace: of two threads on one stream, one's tokens could come between the other's two kernels
        tiles = a.x_tiles;
        if (!tiles) { set_error("mps_mx4_product: x_tiles missing"); return MPS_ERR_WORKSPACE; }
    }
    if (((reinterpret_cast<uintptr_t>(inside ? nullptr : tiles) | reinterpret_cast<uintptr_t>(a.w) | reinterpret_cast<uintptr_t>(a.w_up) |
          (a.out_dtype == MPS_MX4 ? reinterpret_cast<uintptr_t>(a.out) : 0)) & 15u) || (reinterpret_cast<uintptr_t>(workspace) & 255u)) {
        set_error("mps_mx4_product: tiles must be 16-byte aligned, the workspace 256");
        return MPS_ERR_INVALID;
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    Device d;
    int rc = current_device(d);
    if (rc) return rc;
    if (!quantized && !inside) {
        rc = mps_mx4_quantize(a.x, a.x_dtype, a.tokens, a.cols, a.x_stride, const_cast<void*>(tiles), stream);
        if (rc) return rc;
    }
    ProductArgs p = {};
    p.x = static_cast<const uint8_t*>(tiles);
    p.w = static_cast<const uint8_t*>(a.w);
    p.w_up = static_cast<const uint8_t*>(a.w_up);
    p.out = a.out;
    p.workspace = static_cast<uint32_t*>(workspace);
    p.out_stride = a.out_stride;
    p.x_stride = a.x_stride;
    p.tokens = a.tokens;
    p.rows = (int32_t)a.rows;
    p.cols = (int32_t)a.cols;
    p.chunks = (int32_t)mx4_chunks(a.cols);
    p.row_tiles = (int32_t)mx4_row_tiles(a.rows);
    p.x_dtype = a.x_dtype;
    p.out_dtype = a.out_dtype;
    p.activation = a.activation;
    p.x_vec = inside && mx4_vec_ok(a.x, a.x_stride, a.x_dtype);
    p.even = a.out_dtype != MPS_MX4 && a.out_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15u) == 0;
    p.half_values = half_values;
    p.early = (!quantized && !inside) || a.weights_ready;
    if (a.w_up) {
        if (inside) return launch_stream<16, true, true>(p, d, st);
        if (a.tokens <= 16) return launch_stream<16, true>(p, d, st);
        if (a.tokens <= 32) return launch_stream<32, true>(p, d, st);
        if (a.tokens <= 64) return launch_stream<64, true>(p, d, st);
        return launch_wide<true>(p, d, st);
    }
    if (inside) return launch_stream<16, false, true>(p, d, st);
    if (a.tokens <= 16) return launch_stream<16, false>(p, d, st);
    if (a.tokens <= 32) return launch_stream<32, false>(p, d, st);
    if (a.tokens <= 64) return launch_stream<64, false>(p, d, st);
    if (stream_pays(p, d.sms)) return launch_stream<128, false>(p, d, st);
    return a.out_dtype == MPS_F32 ? launch_wide<false, true>(p, d, st) : launch_wide<false>(p, d, st);
}

}  // namespace mps

using namespace mps;

extern "C" {

int64_t mps_mx4_workspace_bytes(void) { return kMx4WorkspaceBytes; }

int mps_mx4_product(const mps_mx4_linear* args, void* workspace, int64_t workspace_bytes, void* stream) {
    if (!args) { set_error("mps_mx4_product: null arguments"); return MPS_ERR_INVALID; }
    return product(*args, false, workspace, workspace_bytes, stream);
}

int64_t mps_mx4_mlp_scratch_bytes(int64_t tokens, int64_t hidden, int64_t inter) {
    const int64_t x = mps_mx4_bytes(tokens, hidden), a = mps_mx4_bytes(tokens, inter), y = tokens * hidden;
    if (x < 0 || a < 0) return -1;
    return a + (x + y * 2 > y * 4 ? x + y * 2 : y * 4);      // x and a are multiples of 256
}

int mps_mx4_gated_mlp(const mps_mx4_mlp* block, const void* h, int32_t h_dtype, int64_t h_stride, int64_t tokens, void* h_out, int64_t h_out_stride,
                      void* n_out, int32_t n_dtype, void* scratch, int64_t scratch_bytes, void* workspace, int64_t workspace_bytes, void* stream) {
    // whatever would be refused on the way is refused here, before the first kernel
    const auto refuse = [](const char* why) { set_error("mps_mx4_gated_mlp: %s", why); return MPS_ERR_INVALID; };
    if (!block || !block->gate_proj || !block->up_proj || !block->down_proj || !block->pre_weight) return refuse("null argument");
    if (block->hidden > kMx4MostNormCols) return refuse("hidden out of a norm's range");
    if (!mx4_dtype_ok(h_dtype) || !mx4_dtype_ok(block->pre_dtype) || (block->gate && !mx4_dtype_ok(block->gate_dtype)) ||
        ((block->post_weight || block->next_weight) && !mx4_dtype_ok(block->weight_dtype)) || (block->next_weight && n_dtype != MPS_MX4 && !mx4_dtype_ok(n_dtype)))
        return refuse("unknown dtype");
    if (block->activation != MPS_SILU && block->activation != MPS_GELU_TANH) return refuse("unknown activation");
    if ((reinterpret_cast<uintptr_t>(block->gate_proj) | reinterpret_cast<uintptr_t>(block->up_proj) | reinterpret_cast<uintptr_t>(block->down_proj) |
         (n_dtype == MPS_MX4 ? reinterpret_cast<uintptr_t>(n_out) : 0)) & 15u) return refuse("tiles must be 16-byte aligned");
    const int64_t need = mps_mx4_mlp_scratch_bytes(tokens, block->hidden, block->inter);
    if (need < 0) { set_error("mps_mx4_gated_mlp: sizes out of range"); return MPS_ERR_INVALID; }
    if (tokens == 0) return MPS_OK;
    if (!h || !h_out || (block->next_weight && !n_out)) return refuse("null pointer");
    if (tokens > kMx4MostNormRows) return refuse("more tokens than a norm has rows");
    if (!scratch || scratch_bytes < need || (reinterpret_cast<uintptr_t>(scratch) & 255u)) { set_error("mps_mx4_gated_mlp: scratch missing, too small or unaligned"); return MPS_ERR_WORKSPACE; }
    if (!workspace || workspace_bytes < kMx4WorkspaceBytes || (reinterpret_cast<uintptr_t>(workspace) & 255u)) { set_error("mps_mx4_gated_mlp: workspace missing, too small or unaligned"); return MPS_ERR_WORKSPACE; }
    // The block's result is held in 16 bits, as mps_mx4_product would give it to mps_mx4_norm_rows: 2048 tokens of an 8B layer take 169 us, in FP32
    // 175 (512 tokens 62.5 and 63.1, fewer the same).  Of a stream in F16 it is F16's value, but in FP32 (180 us): what lies beyond 65504 would be an infinity,
    // and its row NaN behind the norm, where the stream is in range.
    const bool half = h_dtype == MPS_F16 && !block->wide_result;
    const int32_t y_dtype = h_dtype == MPS_F16 || block->wide_result ? MPS_F32 : MPS_BF16;
    uint8_t* a = static_cast<uint8_t*>(scratch);
    uint8_t* x = a + mps_mx4_bytes(tokens, block->inter);
    uint8_t* y = y_dtype == MPS_F32 ? x : x + mps_mx4_bytes(tokens, block->hidden);      // x has been multiplied when y comes

    mps_mx4_norm norm = {};
    norm.h = h;
    norm.next_weight = block->pre_weight;
    norm.n_out = x;
    norm.rows = tokens;
    norm.cols = block->hidden;
    norm.h_stride = h_stride;
    norm.h_dtype = h_dtype;
    norm.n_dtype = MPS_MX4;
    norm.weight_dtype = block->pre_dtype;
    norm.eps = block->eps;
    norm.residual_scale = 1.f;
    int rc = mps_mx4_norm_rows(&norm, stream);
    if (rc) return rc;

    mps_mx4_linear gated = {};
    gated.x = x;
    gated.w = block->gate_proj;
    gated.w_up = block->up_proj;
    gated.out = a;
    gated.tokens = tokens;
    gated.cols = block->hidden;
    gated.rows = block->inter;
    gated.x_dtype = gated.out_dtype = MPS_MX4;
    gated.activation = block->activation;
    gated.weights_ready = 1;          // the kernel before each of the two is this block's own
    rc = product(gated, false, workspace, workspace_bytes, stream);
    if (rc) return rc;

    mps_mx4_linear down = gated;
    down.x = a;
    down.w = block->down_proj;
    down.w_up = nullptr;
    down.out = y;
    down.cols = block->inter;
    down.rows = down.out_stride = block->hidden;
    down.out_dtype = y_dtype;
    rc = product(down, half, workspace, workspace_bytes, stream);
    if (rc) return rc;

    norm.y = y;
    norm.post_weight = block->post_weight;
    norm.gate = block->gate;
    norm.next_weight = block->next_weight;
    norm.h_out = h_out;
    norm.n_out = block->next_weight ? n_out : nullptr;
    norm.y_stride = norm.n_stride = block->hidden;
    norm.h_out_stride = h_out_stride;
    norm.gate_row_stride = block->gate_row_stride;
    norm.gate_col_stride = block->gate_col_stride;
    norm.y_dtype = y_dtype;
    norm.n_dtype = n_dtype;
    norm.gate_dtype = block->gate_dtype;
    norm.weight_dtype = block->weight_dtype;
    norm.residual_scale = block->residual_scale;
    return mps_mx4_norm_rows(&norm, stream);
}

int mps_mx4_status(void* workspace, int64_t workspace_bytes, void* stream, int32_t* timed_out) {
    if (!timed_out || !workspace || workspace_bytes < kMx4WorkspaceBytes) { set_error("mps_mx4_status: bad argument"); return MPS_ERR_INVALID; }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    uint32_t flag = 0;
    MPS_CUDA_TRY(cudaMemcpyAsync(&flag, workspace, sizeof(flag), cudaMemcpyDeviceToHost, st));
    MPS_CUDA_TRY(cudaStreamSynchronize(st));
    if (flag) MPS_CUDA_TRY(cudaMemsetAsync(workspace, 0, sizeof(flag), st));
    *timed_out = flag ? 1 : 0;
    return MPS_OK;
}

}  // extern "C"
