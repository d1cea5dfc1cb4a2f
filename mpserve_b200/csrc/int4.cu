// Products of a few tokens with INT4 weights: out[t, r] = sum_k x[t, k] (q[r, k] - z[r, k / group]) s[r, k / group].
//
// q is a 4-bit code, z a 4-bit zero point and s a 16-bit scale that a group of 32, 64 or 128 neighbouring columns of a row share.  A code minus its zero
// point is a whole number of at most 15, exact in BF16 and F16, so the tensor cores multiply those by the tokens as they came, a group's products are summed in
// FP32, and the scale multiplies that sum, in FP32: nothing is rounded before the output.
//
// In memory a weight is an array of tiles of 128 rows x 128 columns, row of tiles after row of tiles, each in one piece, so that one bulk copy brings it: 8 KB of
// codes, then a word for every row and group, the scale in its low half and the zero point in its high one.  Codes are in sixteen blocks of 16 rows x 64 columns (two
// for the first 16 rows, two for the next ...), and a block has 16 bytes for every lane of a warp: lane 4 g + t has rows g and g + 8; its word s the columns
// k = 16 s + 4 t and the three after: codes of (g, k), (g + 8, k), (g, k + 2), (g + 8, k + 2) in the four nibbles of the low half, their right neighbours in those
// of the high half.  A mask and a shift give a pair of codes in the two halves of a register, an OR makes them 128 + q in BF16 (1024 + q in
// F16), and one subtraction of 128 + z takes both to q - z: four registers that are a lane's share of 16 rows x 16 columns in tensor memory.  What fills a tile up
// has codes, zero points and scales of 0.
#include "mx4.cuh"
#include "mx4_tensor.cuh"
#include "stream_common.cuh"
#include "warp_mma.cuh"

#include <algorithm>
#include <atomic>

namespace mps {

constexpr int kInt4Rows = 128, kInt4Cols = 128, kInt4CodeBytes = kInt4Rows * kInt4Cols / 2;
constexpr int64_t kInt4MostRows = int64_t(1) << 27, kInt4MostCols = int64_t(1) << 24;

__host__ __device__ constexpr int int4_tile_bytes(int group) { return kInt4CodeBytes + kInt4Rows * (kInt4Cols / group) * 4; }
__host__ __device__ inline int64_t int4_chunks(int64_t cols) { return (cols + kInt4Cols - 1) / kInt4Cols; }
__host__ __device__ inline int64_t int4_row_tiles(int64_t rows) { return (rows + kInt4Rows - 1) / kInt4Rows; }
// In a tile: the word of a row and one of its groups, after the codes; sixteen rows' words of a group lie together.
__host__ __device__ inline int int4_scale_word(int row, int group, int groups) { return (row / 16 * groups + group) * 16 + row % 16; }
static bool int4_size_ok(int64_t rows, int64_t cols, int32_t group) {
    return rows >= 0 && rows <= kInt4MostRows && cols > 0 && cols <= kInt4MostCols && (group == 32 || group == 64 || group == 128);
}

// Row and column, within a tile, of the first code of nibble `i` (0 to 3) of code word `w`.
__device__ __forceinline__ int int4_row(int w, int i) { return (w >> 8) * 16 + ((w >> 4) & 7) + 8 * (i & 1); }
__device__ __forceinline__ int int4_column(int w, int i) {
    const int s = w & 3, t = (w >> 2) & 3, block = (w >> 7) & 1;
    return block * 64 + 16 * s + 4 * t + (i & 2);
}

// ---- laid out once, and back --------------------------------------------------------------------------

struct Int4Parts {
    const uint8_t* codes;      // a code a byte
    const uint16_t* scales;
    const uint8_t* zeros;      // or null: 8
    int64_t rows, cols;
    int32_t group;
};

// A CTA a tile at a time.
__global__ void __launch_bounds__(256) int4_pack_kernel(const Int4Parts p, uint8_t* __restrict__ data) {
    griddep_wait();
    griddep_launch();
    const int64_t chunks = int4_chunks(p.cols), tiles = int4_row_tiles(p.rows) * chunks, groups = (p.cols + p.group - 1) / p.group;
    const int in_tile = kInt4Cols / p.group;
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int64_t row0 = tile / chunks * kInt4Rows, col0 = tile % chunks * kInt4Cols;
        uint32_t* out = reinterpret_cast<uint32_t*>(data + tile * int4_tile_bytes(p.group));
        for (int w = threadIdx.x; w < kInt4CodeBytes / 4; w += blockDim.x) {
            uint32_t word = 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t row = row0 + int4_row(w, i);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int64_t col = col0 + int4_column(w, i) + j, g = col / p.group;
                    uint32_t code = 0u;
                    if (row < p.rows && g < groups) code = col < p.cols ? p.codes[row * p.cols + col] : p.zeros ? p.zeros[row * groups + g] : 8u;      // q - z = 0
                    word |= (code & 15u) << (4 * i + 16 * j);
                }
            }
            out[w] = word;
        }
        for (int w = threadIdx.x; w < kInt4Rows * in_tile; w += blockDim.x) {
            const int64_t row = row0 + w % kInt4Rows, g = col0 / p.group + w / kInt4Rows;
            uint32_t word = 0u;
            if (row < p.rows && g < groups) word = p.scales[row * groups + g] | (p.zeros ? (uint32_t)p.zeros[row * groups + g] & 15u : 8u) << 16;
            out[kInt4CodeBytes / 4 + int4_scale_word(w % kInt4Rows, w / kInt4Rows, in_tile)] = word;
        }
    }
}

__device__ __forceinline__ float int4_scale(uint32_t word, bool bf16) {
    return bf16 ? __uint_as_float(word << 16) : __half2float(__ushort_as_half((uint16_t)word));
}

__global__ void __launch_bounds__(256) int4_values_kernel(const uint8_t* __restrict__ data, int64_t rows, int64_t cols, int32_t group, int scale_bf16, int dtype,
                                                          void* __restrict__ out) {
    griddep_wait();
    griddep_launch();
    const int64_t chunks = int4_chunks(cols), tiles = int4_row_tiles(rows) * chunks;
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int64_t row0 = tile / chunks * kInt4Rows, col0 = tile % chunks * kInt4Cols;
        const uint32_t* in = reinterpret_cast<const uint32_t*>(data + tile * int4_tile_bytes(group));
        for (int w = threadIdx.x; w < kInt4CodeBytes / 4; w += blockDim.x) {
            const uint32_t word = in[w];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = int4_row(w, i), c = int4_column(w, i);
                if (row0 + r >= rows) continue;
                const uint32_t sz = in[kInt4CodeBytes / 4 + int4_scale_word(r, c / group, kInt4Cols / group)];
                const float scale = int4_scale(sz, scale_bf16);
                const int zero = (int)(sz >> 16);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if (col0 + c + j >= cols) continue;
                    const float v = (float)((int)((word >> (4 * i + 16 * j)) & 15u) - zero) * scale;      // exact: 5 bits times 11
                    const int64_t at = (row0 + r) * cols + col0 + c + j;
                    if (dtype == MPS_F32) static_cast<float*>(out)[at] = v;
                    else static_cast<uint16_t*>(out)[at] = (uint16_t)pack2(v, 0.f, dtype);
                }
            }
        }
    }
}

// ---- products -------------------------------------------------------------------------------------------
//
// Two kernels.  In both a CTA has 128 features for up to TOKENS tokens, and a share of the columns: a cluster of up to eight shares a row of tiles, as many as fill the
// GPU, and adds its CTAs' sums up in shared memory, always in the same order.  Two tiles and their columns of the tokens come at a time into a ring of some 200 KB, as
// one copy each: how many copies an SM has to start counts, not their bytes (31 MB in copies of 4.25 KB take 18.5 to 22.6 us, of 8.5 KB 12.4, of 17 KB 8.3, as
// plain loads 8.3).
constexpr int kInt4Workers = 8, kInt4Adders = 4, kInt4Threads = (2 + kInt4Workers + kInt4Adders) * 32;
constexpr int kInt4StageTiles = 2;
constexpr int kInt4Buffers = 4, kInt4Sums = 4, kInt4MostParts = 8;
constexpr int kInt4Smem = 227 << 10;
// Up to 16 tokens codes stay in registers (1, 8 and 16 tokens through 14336 x 4096: 10.6, 10.7 and 13.3 us); more tokens there want as many registers again and took 30 us
// for 17 to 32, where the other kernel takes 16 for 33 and 17 for 64.
constexpr int kInt4FewTokens = 16;

struct Int4Args {
    const uint8_t* w;
    void* out;
    int64_t out_stride, tokens, rows;
    int32_t chunks, parts, token_tiles;
    int32_t out_dtype;
    bool whole;              // columns are a multiple of 64: the tokens' map has a third dimension, columns by 64
    bool scale_bf16;
    bool even;               // rows of the output begin at multiples of 8 bytes
    uint32_t* workspace;     // word 0 records a wait that ran out
};

template <int TOKENS, int GROUP>
struct Int4Tensor {
    static constexpr int kGroups = kInt4Cols / GROUP, kTile = int4_tile_bytes(GROUP);
    static constexpr int kX = kInt4StageTiles * TOKENS * kInt4Cols * 2;              // by 64 columns
    static constexpr int kStage = (kX + kInt4StageTiles * kTile + 1023) / 1024 * 1024;      // the tokens, then the tiles
    static constexpr int kStages = (kInt4Smem - 1024) / kStage;
    static constexpr int kBars = kStages * kStage;
    static constexpr int kSmem = kBars + (2 * kStages + 2 * kInt4Buffers + 2 * kInt4Sums + 1) * 8 + 16;
    static constexpr int kSumColumns = kInt4Buffers * 64, kColumns = 512;            // tensor memory: left operands, then accumulators
    static_assert(kSumColumns + kInt4Sums * TOKENS <= kColumns, "tensor memory");
    static_assert(kSmem <= kInt4Smem && kX % 1024 == 0, "shared memory");
    static_assert(TOKENS * kInt4Rows * 4 <= kStages * kStage, "sums take the ring's place");
};

template <bool BF16>
__device__ __forceinline__ uint32_t subtract2(uint32_t a, uint32_t b) {
    uint32_t r;
    if (BF16) asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// What codes are masked and completed with.  From registers: an instruction takes one of the two as it is, and the compiler, which knows both, would make two
// instructions of one (one token through 14336 x 4096 took 12.5 us that way).
template <bool BF16>
struct Int4Masks {
    uint32_t mask, magic;
    __device__ __forceinline__ Int4Masks() {
        asm volatile("mov.b32 %0, 0x000F000F;" : "=r"(mask));
        asm volatile("mov.b32 %0, %1;" : "=r"(magic) : "n"(BF16 ? 0x43004300 : 0x64006400));
    }
    // Two codes, nibble i of both halves of `w`, minus their zero point: `zero` is 128 + z in BF16 (1024 + z in F16), twice.
    __device__ __forceinline__ uint32_t pair(uint32_t w, int i, uint32_t zero) const {
        uint32_t r;
        asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w >> (4 * i)), "r"(mask), "r"(magic));      // and, or
        return subtract2<BF16>(r, zero);
    }
    __device__ __forceinline__ uint32_t zero(uint32_t word) const { return __byte_perm(word, 0u, 0x3232) | magic; }
};
// Sixteen lanes of tensor memory x 64 columns: lane 4 g + t has, of every eight columns, 2 t and 2 t + 1 of lanes g (two words) and g + 8.
__device__ __forceinline__ void tmem_store_fragments(uint32_t tmem, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x256b.x8.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
          "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
          "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
          "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(tmem) : "memory");
}

// The sums of a cluster's CTAs, [token][row] at the start of each one's shared memory, into the output: every parts-th token is this CTA's, a warp has 128 rows of
// one at a time.  All threads take part; nobody leaves while his sums are read.
__device__ __forceinline__ void finish_tile(const Int4Args& p, uint32_t sums, int64_t row_tile, int64_t token0, int tokens, int part, int warp, int lane, int warps, bool failed) {
    if (p.parts > 1) cluster_sync(); else __syncthreads();
    if (!failed) {
        const int64_t feature = row_tile * kInt4Rows + lane * 4;
        for (int t = part + warp * p.parts; t < tokens; t += warps * p.parts) {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int g = 0; g < kInt4MostParts; ++g) {
                const uint32_t at = sums + t * (kInt4Rows * 4) + lane * 16;
                if (g < p.parts) add4(v, load_peer(p.parts > 1 ? peer_address(at, g) : at));
            }
            uint16_t* to = static_cast<uint16_t*>(p.out) + (token0 + t) * p.out_stride + feature;
            const uint32_t lo = pack2(v.x, v.y, p.out_dtype), hi = pack2(v.z, v.w, p.out_dtype);
            if (p.even && feature + 4 <= p.rows) {
                *reinterpret_cast<uint2*>(to) = make_uint2(lo, hi);
            } else {
                if (feature < p.rows) to[0] = (uint16_t)lo;
                if (feature + 1 < p.rows) to[1] = (uint16_t)(lo >> 16);
                if (feature + 2 < p.rows) to[2] = (uint16_t)hi;
                if (feature + 3 < p.rows) to[3] = (uint16_t)(hi >> 16);
            }
        }
    }
    __syncwarp();
    if (p.parts > 1) cluster_sync();
}

// ... unless a wait ran out: no copy may come after the CTA is gone, or while sums take the ring's place.
template <int STAGES, typename Full>
__device__ __forceinline__ void copies_end(int asked, Full full) {
    for (int i = max(0, asked - STAGES); i < asked; ++i) mbar_wait(full(i % STAGES), (uint32_t)(i / STAGES) & 1u, kMx4SpinLimit);
    __syncthreads();
}

// Columns of TOKENS tokens, from column 64 `block` on, 64 a row, zeros beyond both.
template <int TOKENS>
__device__ __forceinline__ void token_boxes(uint32_t dst, const CUtensorMap* map, int block, int token, bool whole, uint32_t bar) {
    if (whole) {
        asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                     ::"r"(dst), "l"(map), "r"(0), "r"(token), "r"(block), "r"(bar) : "memory");
    } else {
#pragma unroll
        for (int h = 0; h < kInt4StageTiles * 2; ++h)
            asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                         ::"r"(dst + h * (TOKENS * 128)), "l"(map), "r"((block + h) * 64), "r"(token), "r"(bar) : "memory");
    }
}

// ---- up to 16 tokens: codes stay in registers -----------------------------------------------------------
//
// Sixteen warps, four sets of four that take tiles in turn, a warp 32 rows: a code word becomes the left operand of an m16n8k16 where it is, and a group's products
// are multiplied by its scale in registers.  Bound: memory; taking codes apart (11 instructions for eight codes, seven of them on a pipe that takes two a
// cycle) some 220 cycles an SM for 8.5 KB, the products of eight tokens 130.
constexpr int kFewSets = 4, kFewSetWarps = 4, kFewWarps = kFewSets * kFewSetWarps, kFewThreads = (2 + kFewWarps) * 32;
template <int TOKENS, int GROUP>
struct Int4Few {
    static constexpr int kGroups = kInt4Cols / GROUP, kTile = int4_tile_bytes(GROUP);
    static constexpr int kX = kInt4StageTiles * TOKENS * kInt4Cols * 2;
    static constexpr int kStage = (kX + kInt4StageTiles * kTile + 1023) / 1024 * 1024;
    static constexpr int kStages = (kInt4Smem - 1024) / kStage;
    static constexpr int kBars = kStages * kStage;
    static constexpr int kSmem = kBars + 2 * kStages * 8 + 16;
    static_assert(kSmem <= kInt4Smem && kX % 1024 == 0, "shared memory");
    static_assert(kFewSets % kInt4StageTiles == 0 && kStages >= kFewSets / kInt4StageTiles, "a set's tiles are in the same place of their stages");
    static_assert(kFewSets * TOKENS * kInt4Rows * 4 <= kBars, "sums take the ring's place");
};

__device__ __forceinline__ int few_token(int column) { return column < 4 ? 2 * column : 2 * column - 7; }      // of eight

template <int TOKENS, int GROUP, bool BF16>
__global__ void __launch_bounds__(kFewThreads, 1) int4_few_kernel(const Int4Args p, const __grid_constant__ CUtensorMap x_map) {
    using S = Int4Few<TOKENS, GROUP>;
    constexpr int kTiles = TOKENS / 8;
    extern __shared__ __align__(1024) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = smem_u32(smem), bar0 = base + S::kBars;
    volatile uint32_t& failed = *reinterpret_cast<volatile uint32_t*>(smem + S::kSmem - 12);
    const auto full = [&](int s) { return bar0 + 8u * s; };
    const auto empty = [&](int s) { return bar0 + 8u * (S::kStages + s); };
    const int part = blockIdx.x % p.parts;
    const int64_t at = blockIdx.x / p.parts, token0 = at % p.token_tiles * TOKENS, row_tile = at / p.token_tiles;
    const int tokens = (int)min((int64_t)TOKENS, p.tokens - token0);
    const int k0 = (int)((int64_t)p.chunks * part / p.parts), count = (int)((int64_t)p.chunks * (part + 1) / p.parts) - k0;      // this CTA's tiles
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) { mbar_init(full(s), 2); mbar_init(empty(s), kInt4StageTiles * kFewSetWarps); }
        failed = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    griddep_wait();
    griddep_launch();
    float acc[2][kTiles][4];      // of two times 16 rows
    int asked = 0;      // stages that this thread has filled
    if (warp < 2) {
        if (lane == 0) {
            const uint8_t* w = p.w + (row_tile * p.chunks + k0) * S::kTile;
            int i = 0;
            for (; i * kInt4StageTiles < count; ++i) {
                const int s = i % S::kStages, tile = i * kInt4StageTiles;
                if (i >= S::kStages && !bar_wait(empty(s), (uint32_t)(i / S::kStages - 1) & 1u, &failed)) break;
                const uint32_t to = base + s * S::kStage;
                if (warp == 0) {
                    const uint32_t bytes = min(kInt4StageTiles, count - tile) * S::kTile;
                    mbar_expect_tx(full(s), bytes);
                    bulk_g2s(to + S::kX, w + (int64_t)tile * S::kTile, bytes, full(s));
                } else {
                    mbar_expect_tx(full(s), S::kX);
                    token_boxes<TOKENS>(to, &x_map, (k0 + tile) * 2, (int)token0, p.whole, full(s));
                }
            }
            asked = i;
        }
    } else {
        const int quarter = (warp - 2) % kFewSetWarps, set = (warp - 2) / kFewSetWarps, g = lane >> 2, t = lane & 3;
        const Int4Masks<BF16> masks;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int n = 0; n < kTiles; ++n) { acc[h][n][0] = acc[h][n][1] = acc[h][n][2] = acc[h][n][3] = 0.f; }
        // Four columns of a token, 16 k + 4 t on: piece 2 k + t / 2 of its row's eight, XORed with the row.  Column g of a product is token few_token(g): four rows of
        // which half a warp reads at once then have their pieces in different banks.
        int x_at[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x_at[k] = few_token(g) * 128 + (((2 * k + (t >> 1)) ^ few_token(g)) << 4) + (t & 1) * 8;
        int s = set / kInt4StageTiles;
        uint32_t parity = 0;
        for (int i = set; i < count; i += kFewSets) {
            if (!warp_wait(full(s), parity, &failed)) break;
            const uint8_t* x = smem + s * S::kStage + set % kInt4StageTiles * (TOKENS * kInt4Cols * 2);
            const uint8_t* tile = smem + s * S::kStage + S::kX + set % kInt4StageTiles * S::kTile;
            const uint4* codes = reinterpret_cast<const uint4*>(tile + quarter * 2048) + lane;
            const uint32_t* words = reinterpret_cast<const uint32_t*>(tile + kInt4CodeBytes) + quarter * (S::kGroups * 32) + g;
            uint2 b[kTiles][8];
#pragma unroll
            for (int n = 0; n < kTiles; ++n)
#pragma unroll
                for (int k = 0; k < 8; ++k) b[n][k] = *reinterpret_cast<const uint2*>(x + x_at[k & 3] + (k >> 2) * (TOKENS * 128) + n * 1024);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint4 w[2] = {codes[h * 64], codes[h * 64 + 32]};
                uint32_t lo[S::kGroups], hi[S::kGroups];
#pragma unroll
                for (int j = 0; j < S::kGroups; ++j) {
                    lo[j] = words[(h * S::kGroups + j) * 16];
                    hi[j] = words[(h * S::kGroups + j) * 16 + 8];
                }
                // products of 64 columns (32 in groups of 32) do not wait for those of the next
                constexpr int kParts = GROUP == 32 ? 4 : 2;
                float sums[kTiles][kParts][4];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int j = k * 16 / GROUP, c = k * kParts / 8;
                    const uint32_t zlo = masks.zero(lo[j]), zhi = masks.zero(hi[j]);
                    const uint4& v4 = w[k >> 2];
                    const uint32_t v = (k & 3) == 0 ? v4.x : (k & 3) == 1 ? v4.y : (k & 3) == 2 ? v4.z : v4.w;
                    const uint32_t a[4] = {masks.pair(v, 0, zlo), masks.pair(v, 1, zhi), masks.pair(v, 2, zlo), masks.pair(v, 3, zhi)};
#pragma unroll
                    for (int n = 0; n < kTiles; ++n) {
                        const uint2 y = b[n][k];
                        if (k * kParts % 8 == 0) multiply_first<BF16>(sums[n][c], a, y.x, y.y);
                        else multiply<BF16>(sums[n][c], a, y.x, y.y);
                    }
                }
                if (h == 1) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(empty(s));
                }
#pragma unroll
                for (int j = 0; j < S::kGroups; ++j) {
                    const float slo = int4_scale(lo[j], p.scale_bf16), shi = int4_scale(hi[j], p.scale_bf16);
#pragma unroll
                    for (int n = 0; n < kTiles; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float sum = GROUP == 128 ? sums[n][0][e] + sums[n][1][e] : sums[n][j][e];
                            acc[h][n][e] = fmaf(e < 2 ? slo : shi, sum, acc[h][n][e]);
                        }
                }
            }
            s += kFewSets / kInt4StageTiles;
            if (s >= S::kStages) { s -= S::kStages; parity ^= 1u; }
        }
    }
    __syncwarp();
    __syncthreads();      // whatever the ring held has been used ...
    if (failed) copies_end<S::kStages>(asked, full);
    if (warp >= 2) {
        // the sets' sums beside one another, then added
        float* sums = reinterpret_cast<float*>(smem) + (warp - 2) / kFewSetWarps * (TOKENS * kInt4Rows) + (warp - 2) % kFewSetWarps * 32 + (lane >> 2);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int n = 0; n < kTiles; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) sums[(n * 8 + few_token(2 * (lane & 3) + (e & 1))) * kInt4Rows + h * 16 + (e >> 1) * 8] = acc[h][n][e];
    }
    __syncthreads();
    float* sums = reinterpret_cast<float*>(smem);
    for (int i = threadIdx.x; i < tokens * kInt4Rows; i += kFewThreads) {
        float v = sums[i];
#pragma unroll
        for (int set = 1; set < kFewSets; ++set) v += sums[set * (TOKENS * kInt4Rows) + i];
        sums[i] = v;
    }
    finish_tile(p, base, row_tile, token0, tokens, part, warp, lane, kFewThreads / 32, failed != 0u);
    if (threadIdx.x == 0 && failed) atomicExch(p.workspace, 1u);
}

// ---- more tokens: codes go to tensor memory ---------------------------------------------------------------
//
// Warps:
//   0 copies;  1 multiplies: features (left operand, tensor memory) by tokens (right operand, shared memory), a group of columns into an accumulator of its own;
//   2 to 9 take codes apart and store them in tensor memory, four warps a tile, 32 rows each: two tiles at a time, since what one takes is mostly waits in a row;
//   10 to 13 add the groups' accumulators up, times their scales: a thread has a feature, its tokens are in registers.
// Bound: handing over.  16 columns by 64 tokens take the tensor core 33 cycles, a tile 260; each of the tile's groups waits some 150 for codes, products or sums of the other side.
template <int TOKENS, int GROUP, bool BF16>
__global__ void __launch_bounds__(kInt4Threads, 1) int4_tensor_kernel(const Int4Args p, const __grid_constant__ CUtensorMap x_map) {
    using S = Int4Tensor<TOKENS, GROUP>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = smem_u32(smem), bar0 = base + S::kBars;
    uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(smem + S::kSmem - 16);
    volatile uint32_t& failed = *reinterpret_cast<volatile uint32_t*>(smem + S::kSmem - 12);
    const auto full = [&](int s) { return bar0 + 8u * s; };                                     // a tile and its tokens have come
    const auto empty = [&](int s) { return bar0 + 8u * (S::kStages + s); };
    const auto ready = [&](int b) { return bar0 + 8u * (2 * S::kStages + b); };                 // a tile is in tensor memory
    const auto used = [&](int b) { return bar0 + 8u * (2 * S::kStages + kInt4Buffers + b); };
    const auto summed = [&](int d) { return bar0 + 8u * (2 * S::kStages + 2 * kInt4Buffers + d); };      // a group's accumulator
    const auto taken = [&](int d) { return bar0 + 8u * (2 * S::kStages + 2 * kInt4Buffers + kInt4Sums + d); };
    const uint32_t drained = bar0 + 8u * (2 * S::kStages + 2 * kInt4Buffers + 2 * kInt4Sums);

    const int part = blockIdx.x % p.parts;
    const int64_t at = blockIdx.x / p.parts, token0 = at % p.token_tiles * TOKENS, row_tile = at / p.token_tiles;
    const int tokens = (int)min((int64_t)TOKENS, p.tokens - token0);
    const int k0 = (int)((int64_t)p.chunks * part / p.parts), count = (int)((int64_t)p.chunks * (part + 1) / p.parts) - k0;      // this CTA's tiles

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), kInt4StageTiles * (kInt4Workers / 2 + kInt4Adders + 1)); }
        for (int b = 0; b < kInt4Buffers; ++b) { mbar_init(ready(b), kInt4Workers / 2); mbar_init(used(b), 1); }
        for (int d = 0; d < kInt4Sums; ++d) { mbar_init(summed(d), 1); mbar_init(taken(d), kInt4Adders); }
        mbar_init(drained, 1);
        failed = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc<1>(smem_u32(&tmem_slot), S::kColumns);
    if (warp == 0 && lane == 0) prefetch_map(&x_map);
    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, tmem_slot, 0);
    griddep_wait();
    griddep_launch();

    float acc[TOKENS];      // of the adding warps
    int asked = 0;          // stages that this thread has filled
    if (warp == 0) {
        if (lane == 0) {
            const uint8_t* w = p.w + (row_tile * p.chunks + k0) * S::kTile;
            int i = 0;
            for (; i * kInt4StageTiles < count; ++i) {
                const int s = i % S::kStages, tile = i * kInt4StageTiles;
                if (i >= S::kStages && !bar_wait(empty(s), (uint32_t)(i / S::kStages - 1) & 1u, &failed)) break;
                const uint32_t to = base + s * S::kStage, bytes = min(kInt4StageTiles, count - tile) * S::kTile;
                mbar_expect_tx(full(s), S::kX + bytes);
                bulk_g2s(to + S::kX, w + (int64_t)tile * S::kTile, bytes, full(s));
                token_boxes<TOKENS>(to, &x_map, (k0 + tile) * 2, (int)token0, p.whole, full(s));
            }
            asked = i;
        }
    } else if (warp == 1) {
        const uint32_t lead = elect_one(), instruction = half_instruction(BF16, TOKENS, false);
        bool ok = true;
        int n = 0;      // groups so far
        for (int i = 0; i < count && ok; ++i) {
            const int b = i % kInt4Buffers, stage = i / kInt4StageTiles, s = stage % S::kStages;
            // of a tile that is in tensor memory the tokens have come, too: those who put it there have seen it.  A sum's first place is free from the start: the phase
            // before the first counts as over.
            ok = warp_wait2(ready(b), (uint32_t)(i / kInt4Buffers) & 1u, taken(n % kInt4Sums), (uint32_t)(n / kInt4Sums - 1) & 1u, &failed);
            if (!ok) break;
            const uint32_t x = base + s * S::kStage + i % kInt4StageTiles * (TOKENS * kInt4Cols * 2);
#pragma unroll
            for (int g = 0; g < S::kGroups; ++g, ++n) {
                const int d = n % kInt4Sums;
                if (g) ok = ok && warp_wait(taken(d), (uint32_t)(n / kInt4Sums - 1) & 1u, &failed);
                if (!ok) break;
                tensor_fence_after();
#pragma unroll
                for (int k = g * (GROUP / 16); k < (g + 1) * (GROUP / 16); ++k)      // 16 columns: eight of tensor memory, 32 bytes of a token's row
                    half_multiply_kept(lead, tmem + S::kSumColumns + d * TOKENS, tmem + b * 64 + k * 8, operand_desc(x + k / 4 * (TOKENS * 128)) + 2 * (k & 3), instruction,
                                       k > g * (GROUP / 16) ? 1u : 0u);
                tensor_commit(lead, summed(d));
            }
            if (ok) {
                tensor_commit(lead, used(b));
                tensor_commit(lead, empty(s));
            }
        }
        tensor_commit(lead, drained);
        warp_wait(drained, 0, &failed);
    } else if (warp < 2 + kInt4Workers) {
        // a quarter of tensor memory's lanes: sixteen rows, and sixteen more
        const int quarter = warp & 3, g = lane >> 2;
        const Int4Masks<BF16> masks;
        for (int i = warp >= 6; i < count; i += 2) {
            const int b = i % kInt4Buffers, stage = i / kInt4StageTiles, s = stage % S::kStages;
            if (!warp_wait2(full(s), (uint32_t)(stage / S::kStages) & 1u, used(b), (uint32_t)(i / kInt4Buffers - 1) & 1u, &failed)) break;
            tensor_fence_after();
            const uint8_t* tile = smem + s * S::kStage + S::kX + i % kInt4StageTiles * S::kTile;
            const uint4* codes = reinterpret_cast<const uint4*>(tile + quarter * 2048) + lane;
            const uint4 w[4] = {codes[0], codes[32], codes[64], codes[96]};
            const uint32_t* words = reinterpret_cast<const uint32_t*>(tile + kInt4CodeBytes) + quarter * (S::kGroups * 32) + g;
            uint32_t zeros[2][S::kGroups][2];      // of rows g and g + 8
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < S::kGroups; ++j) {
                    zeros[h][j][0] = masks.zero(words[(h * S::kGroups + j) * 16]);
                    zeros[h][j][1] = masks.zero(words[(h * S::kGroups + j) * 16 + 8]);
                }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t r[32];
#pragma unroll
                for (int k = 0; k < 8; ++k) {      // 16 columns of the product
                    const uint4& v4 = w[h * 2 + (k >> 2)];
                    const uint32_t v = (k & 3) == 0 ? v4.x : (k & 3) == 1 ? v4.y : (k & 3) == 2 ? v4.z : v4.w;
                    const uint32_t(&z)[2] = zeros[h][k * 16 / GROUP];
                    r[4 * k] = masks.pair(v, 0, z[0]);
                    r[4 * k + 1] = masks.pair(v, 2, z[0]);
                    r[4 * k + 2] = masks.pair(v, 1, z[1]);
                    r[4 * k + 3] = masks.pair(v, 3, z[1]);
                }
                tmem_store_fragments(tmem + ((uint32_t)(quarter * 32 + h * 16) << 16) + b * 64, r);
            }
            tmem_stored();
            tensor_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(ready(b));
                mbar_arrive(empty(s));
            }
        }
    } else {
        const int quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + S::kSumColumns;
#pragma unroll
        for (int t = 0; t < TOKENS; ++t) acc[t] = 0.f;
        bool ok = true;
        int n = 0;
        for (int i = 0; i < count && ok; ++i) {
            const int stage = i / kInt4StageTiles, s = stage % S::kStages;
            ok = warp_wait2(full(s), (uint32_t)(stage / S::kStages) & 1u, summed(n % kInt4Sums), (uint32_t)(n / kInt4Sums) & 1u, &failed);
            if (!ok) break;
            const uint32_t* words = reinterpret_cast<const uint32_t*>(smem + s * S::kStage + S::kX + i % kInt4StageTiles * S::kTile + kInt4CodeBytes);
            float scale[S::kGroups];
#pragma unroll
            for (int g = 0; g < S::kGroups; ++g) scale[g] = int4_scale(words[int4_scale_word(row, g, S::kGroups)], p.scale_bf16);
#pragma unroll
            for (int g = 0; g < S::kGroups; ++g, ++n) {
                const int d = n % kInt4Sums;
                if (g) ok = ok && warp_wait(summed(d), (uint32_t)(n / kInt4Sums) & 1u, &failed);
                if (!ok) break;
                tensor_fence_after();
                constexpr int kStep = 32;
#pragma unroll
                for (int c = 0; c < TOKENS; c += kStep) {
                    if (c < tokens) {
                        float v[kStep];
                        tmem_load32(from + d * TOKENS + c, v);
                        const float2 s2 = make_float2(scale[g], scale[g]);
#pragma unroll
                        for (int t = 0; t < kStep; t += 2) {
                            const float2 sum = fma2(s2, make_float2(v[t], v[t + 1]), make_float2(acc[c + t], acc[c + t + 1]));
                            acc[c + t] = sum.x;
                            acc[c + t + 1] = sum.y;
                        }
                    }
                }
                tensor_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(taken(d));
            }
            if (lane == 0 && ok) mbar_arrive(empty(s));
        }
    }
    __syncwarp();
    tensor_fence_before();
    __syncthreads();      // whatever the ring held has been used ...
    if (failed) copies_end<S::kStages>(asked, full);
    if (warp >= 2 + kInt4Workers) {
        float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int t = 0; t < TOKENS; ++t)
            if (t < tokens) sums[t * kInt4Rows + (warp & 3) * 32 + lane] = acc[t];
    }
    finish_tile(p, base, row_tile, token0, tokens, part, warp, lane, kInt4Threads / 32, failed != 0u);
    __syncthreads();
    tensor_fence_after();
    if (threadIdx.x == 0 && failed) atomicExch(p.workspace, 1u);
    if (warp == 1) tmem_free<1>(tmem, S::kColumns);
}

using EncodeTiled = decltype(&cuTensorMapEncodeTiled);
// The tokens as boxes of 64 columns x `box` rows (x as many 64 columns as a stage has, where the columns are a multiple of 64); rows begin at multiples of 16 bytes.
static int token_map(CUtensorMap& map, const void* x, int64_t tokens, int64_t cols, int64_t stride, bool bf16, int box) {
    EncodeTiled encode;
    const int rc = tensor_map_encoder(encode);
    if (rc) return rc;
    const bool whole = cols % 64 == 0;
    const cuuint64_t row = (cuuint64_t)(tokens > 1 ? stride : (cols + 7) / 8 * 8) * 2;
    const cuuint64_t size[3] = {whole ? 64 : (cuuint64_t)cols, (cuuint64_t)tokens, (cuuint64_t)(cols / 64)}, pitch[2] = {row, 128};
    const cuuint32_t boxes[3] = {64, (cuuint32_t)box, kInt4StageTiles * 2}, step[3] = {1, 1, 1};
    const CUresult r = encode(&map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, whole ? 3 : 2, const_cast<void*>(x), size, pitch, boxes, step,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? MPS_OK : cuda_fail(static_cast<cudaError_t>(r), "cuTensorMapEncodeTiled");      // the two count their errors alike
}

struct Int4Tokens { const void* x; int64_t cols, stride; };

template <int TOKENS, typename Kernel>
static int launch_kernel(const char* what, Kernel kernel, int smem, int threads, std::atomic<uint64_t>& ready, Int4Args p, const Int4Tokens& x, bool bf16, const Device& d,
                         cudaStream_t st) {
    if (!(ready.load(std::memory_order_acquire) >> (d.ordinal & 63) & 1)) {
        MPS_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        ready.fetch_or(uint64_t(1) << (d.ordinal & 63), std::memory_order_release);
    }
    CUtensorMap map;
    const int rc = token_map(map, x.x, p.tokens, x.cols, x.stride, bf16, TOKENS);
    if (rc) return rc;
    p.whole = x.cols % 64 == 0;
    p.token_tiles = (int)((p.tokens + TOKENS - 1) / TOKENS);
    const int64_t tiles = int4_row_tiles(p.rows) * p.token_tiles;
    p.parts = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(kInt4MostParts, p.chunks), d.sms / tiles));
    if (tiles * p.parts > 0x7FFFFFFF) { set_error("mps_int4_product: too many tiles for one launch"); return MPS_ERR_INVALID; }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned int)(tiles * p.parts));
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = st;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = (unsigned int)p.parts;
    attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&config, kernel, p, map);
    return e == cudaSuccess ? MPS_OK : cuda_fail(e, what);
}
template <int TOKENS, int GROUP, bool BF16>
static int launch_group(const Int4Args& p, const Int4Tokens& x, const Device& d, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};
    if constexpr (TOKENS <= kInt4FewTokens)
        return launch_kernel<TOKENS>("int4_few_kernel", int4_few_kernel<TOKENS, GROUP, BF16>, Int4Few<TOKENS, GROUP>::kSmem, kFewThreads, ready, p, x, BF16, d, st);
    else
        return launch_kernel<TOKENS>("int4_tensor_kernel", int4_tensor_kernel<TOKENS, GROUP, BF16>, Int4Tensor<TOKENS, GROUP>::kSmem, kInt4Threads, ready, p, x, BF16, d, st);
}
template <int TOKENS, bool BF16>
static int launch_tokens(const Int4Args& p, const Int4Tokens& x, int group, const Device& d, cudaStream_t st) {
    return group == 128 ? launch_group<TOKENS, 128, BF16>(p, x, d, st) : group == 64 ? launch_group<TOKENS, 64, BF16>(p, x, d, st)
                                                                                     : launch_group<TOKENS, 32, BF16>(p, x, d, st);
}
template <bool BF16>
static int launch_product(const Int4Args& p, const Int4Tokens& x, int group, const Device& d, cudaStream_t st) {
    return p.tokens <= 8 ? launch_tokens<8, BF16>(p, x, group, d, st) : p.tokens <= kInt4FewTokens ? launch_tokens<16, BF16>(p, x, group, d, st)
                                                                           : launch_tokens<64, BF16>(p, x, group, d, st);
}

// Tokens whose rows do not begin at multiples of 16 bytes, as tiled copies want them, or lie over one another: copied into rows that do.
__global__ void __launch_bounds__(256) int4_align_kernel(const uint16_t* __restrict__ x, int64_t stride, int64_t tokens, int32_t cols, int32_t wide, uint16_t* __restrict__ out) {
    griddep_wait();
    griddep_launch();
    const int64_t all = tokens * wide, step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += step) {
        const int64_t token = i / wide, col = i - token * wide;
        out[i] = col < cols ? x[token * stride + col] : (uint16_t)0;
    }
}

}  // namespace mps

using namespace mps;

extern "C" int64_t mps_int4_bytes(int64_t rows, int64_t cols, int32_t group) {
    return int4_size_ok(rows, cols, group) ? int4_row_tiles(rows) * int4_chunks(cols) * int4_tile_bytes(group) : -1;
}

extern "C" int mps_int4_pack(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int64_t rows, int64_t cols, int32_t group, void* data,
                             void* stream) {
    if (!int4_size_ok(rows, cols, group)) { set_error("mps_int4_pack: rows, cols or group out of range"); return MPS_ERR_INVALID; }
    if (rows == 0) return MPS_OK;
    if (!codes || !scales || !data) { set_error("mps_int4_pack: null pointer"); return MPS_ERR_INVALID; }
    if (reinterpret_cast<uintptr_t>(data) & 15u) { set_error("mps_int4_pack: unaligned data"); return MPS_ERR_INVALID; }
    const int64_t tiles = int4_row_tiles(rows) * int4_chunks(cols);
    return launch_overlapping("int4_pack_kernel", int4_pack_kernel, (unsigned int)std::min(tiles, int64_t(1) << 20), dim3(256),
                              static_cast<cudaStream_t>(stream), Int4Parts{codes, scales, zeros, rows, cols, group}, static_cast<uint8_t*>(data));
}

extern "C" int mps_int4_dequantize(const void* data, int64_t rows, int64_t cols, int32_t group, int32_t scale_dtype, int32_t dtype, void* out, void* stream) {
    if (!int4_size_ok(rows, cols, group)) { set_error("mps_int4_dequantize: rows, cols or group out of range"); return MPS_ERR_INVALID; }
    if ((scale_dtype != MPS_BF16 && scale_dtype != MPS_F16) || !mx4_dtype_ok(dtype)) { set_error("mps_int4_dequantize: unknown dtype"); return MPS_ERR_INVALID; }
    if (rows == 0) return MPS_OK;
    if (!data || !out) { set_error("mps_int4_dequantize: null pointer"); return MPS_ERR_INVALID; }
    if (reinterpret_cast<uintptr_t>(data) & 15u) { set_error("mps_int4_dequantize: unaligned data"); return MPS_ERR_INVALID; }
    const int64_t tiles = int4_row_tiles(rows) * int4_chunks(cols);
    return launch_overlapping("int4_values_kernel", int4_values_kernel, (unsigned int)std::min(tiles, int64_t(1) << 20), dim3(256),
                              static_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(data), rows, cols, group, (int)(scale_dtype == MPS_BF16), (int)dtype, out);
}

extern "C" int mps_int4_product(const mps_int4_linear* args, void* workspace, int64_t workspace_bytes, void* stream) {
    if (!args) { set_error("mps_int4_product: null arguments"); return MPS_ERR_INVALID; }
    const mps_int4_linear& a = *args;
    if (a.rows <= 0 || !int4_size_ok(a.rows, a.cols, a.group)) { set_error("mps_int4_product: rows, cols or group out of range"); return MPS_ERR_INVALID; }
    if (a.tokens < 0 || a.tokens > MPS_INT4_MOST_TOKENS) { set_error("mps_int4_product: tokens must be in [0, %d]", (int)MPS_INT4_MOST_TOKENS); return MPS_ERR_INVALID; }
    if ((a.x_dtype != MPS_BF16 && a.x_dtype != MPS_F16) || (a.out_dtype != MPS_BF16 && a.out_dtype != MPS_F16) ||
        (a.scale_dtype != MPS_BF16 && a.scale_dtype != MPS_F16)) {
        set_error("mps_int4_product: dtypes are BF16 or F16");
        return MPS_ERR_INVALID;
    }
    if (a.tokens == 0) return MPS_OK;
    if (!a.x || !a.w || !a.out) { set_error("mps_int4_product: null pointer"); return MPS_ERR_INVALID; }
    if (reinterpret_cast<uintptr_t>(a.w) & 15u) { set_error("mps_int4_product: unaligned weight"); return MPS_ERR_INVALID; }
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) || workspace_bytes < mps_mx4_workspace_bytes()) {
        set_error("mps_int4_product: workspace missing, unaligned or too small");
        return MPS_ERR_WORKSPACE;
    }
    Device d;
    const int rc = current_device(d);
    if (rc) return rc;
    Int4Args p = {};
    p.workspace = static_cast<uint32_t*>(workspace);
    p.w = static_cast<const uint8_t*>(a.w);
    p.out = a.out;
    p.out_stride = a.out_stride;
    p.tokens = a.tokens;
    p.rows = a.rows;
    p.chunks = (int32_t)int4_chunks(a.cols);
    p.out_dtype = a.out_dtype;
    p.scale_bf16 = a.scale_dtype == MPS_BF16;
    p.even = reinterpret_cast<uintptr_t>(a.out) % 8 == 0 && a.out_stride % 4 == 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    Int4Tokens x = {a.x, a.cols, a.x_stride};
    if (reinterpret_cast<uintptr_t>(a.x) % 16 || (a.tokens > 1 && (a.x_stride % 8 || a.x_stride < a.cols))) {
        if (!a.x_rows || reinterpret_cast<uintptr_t>(a.x_rows) % 16) { set_error("mps_int4_product: x_rows missing or unaligned"); return MPS_ERR_WORKSPACE; }
        const int64_t wide = (a.cols + 7) / 8 * 8;
        const int rc2 = launch_overlapping("int4_align_kernel", int4_align_kernel, (unsigned int)std::min((a.tokens * wide + 255) / 256, int64_t(1) << 16), dim3(256), st,
                                           static_cast<const uint16_t*>(a.x), a.x_stride, a.tokens, (int32_t)a.cols, (int32_t)wide, static_cast<uint16_t*>(a.x_rows));
        if (rc2) return rc2;
        x.x = a.x_rows;
        x.stride = wide;
    }
    return a.x_dtype == MPS_BF16 ? launch_product<true>(p, x, a.group, d, st) : launch_product<false>(p, x, a.group, d, st);
}
