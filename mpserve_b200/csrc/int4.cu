// Products of a few tokens with INT4 weights: out[t, r] = sum_k x[t, k] (q[r, k] - z[r, k / group]) s[r, k / group].
//
// q is a 4-bit code, z a 4-bit zero point and s a 16-bit scale that a group of 32, 64 or 128 neighbouring columns of a row share.  A code minus its zero
// point is a whole number of at most 15, exact in BF16 and F16, so the tensor cores multiply those by the tokens as they came, a group's products are summed in
// FP32, and the scale multiplies that sum, in FP32: nothing is rounded before the output.
//
// In memory a weight is an array of blocks of 16 rows x 64 columns, 512 bytes each, row of blocks after row of blocks, then a word for every group and
// row, 16 rows together.  A block holds for every lane of a warp the 16 bytes that make its left operands of four m16n8k16 multiplications: lane 4 g + t
// has rows g and g + 8; its word s the columns k = 32 (s / 2) + 8 t + 4 (s % 2) and the three after: codes of (g, k), (g + 8, k), (g, k + 2), (g + 8, k + 2) in
// the four nibbles of the low half, their right neighbours in those of the high half.  A mask and a shift give a pair of codes in the two halves of a register,
// an OR makes them 128 + q in BF16 (1024 + q in F16), and one subtraction of 128 + z takes both to q - z.  The order of columns is that in
// which a lane reads 16 bytes of a token at a time.  Columns are filled up to a multiple of 64 and of the group with codes that equal their zero
// point, rows to a multiple of 16 with a scale of 0.
#include "mx4.cuh"
#include "stream_common.cuh"
#include "warp_mma.cuh"

namespace mps {

constexpr int kInt4Rows = 16, kInt4Cols = 64, kInt4BlockBytes = 512;
constexpr int64_t kInt4MostRows = int64_t(1) << 27, kInt4MostCols = int64_t(1) << 24;

struct Int4Shape {
    int64_t row_tiles;
    int32_t blocks;      // of a row of blocks
    int32_t groups;      // with those that fill up
    __host__ __device__ int64_t codes_bytes() const { return row_tiles * blocks * kInt4BlockBytes; }
    __host__ __device__ int64_t bytes() const { return codes_bytes() + row_tiles * groups * kInt4Rows * 4; }
};
static __host__ __device__ inline Int4Shape int4_shape(int64_t rows, int64_t cols, int32_t group) {
    const int unit = group > kInt4Cols ? group : kInt4Cols;
    const int64_t wide = (cols + unit - 1) / unit * unit;
    return {(rows + kInt4Rows - 1) / kInt4Rows, (int32_t)(wide / kInt4Cols), (int32_t)(wide / group)};
}
static bool int4_size_ok(int64_t rows, int64_t cols, int32_t group) {
    return rows >= 0 && rows <= kInt4MostRows && cols > 0 && cols <= kInt4MostCols && (group == 32 || group == 64 || group == 128);
}

// Column, within a block, of the first code of nibble `i` (0 to 3) of word s of lane 4 g + t.
__device__ __forceinline__ int int4_column(int t, int s, int i) { return 32 * (s >> 1) + 8 * t + 4 * (s & 1) + (i & 2); }

// ---- laid out once, and back --------------------------------------------------------------------------

struct Int4Parts {
    const uint8_t* codes;      // a code a byte
    const uint16_t* scales;
    const uint8_t* zeros;      // or null: 8
    int64_t rows, cols;
    int32_t group;
};

__global__ void __launch_bounds__(256) int4_pack_kernel(const Int4Parts p, uint8_t* __restrict__ data) {
    griddep_wait();
    griddep_launch();
    const Int4Shape shape = int4_shape(p.rows, p.cols, p.group);
    const int64_t groups = (p.cols + p.group - 1) / p.group, words = shape.codes_bytes() / 4, step = (int64_t)gridDim.x * blockDim.x;
    uint32_t* out = reinterpret_cast<uint32_t*>(data);
    for (int64_t w = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; w < words; w += step) {
        const int64_t block = w >> 7, tile = block / shape.blocks;
        const int64_t first = (block - tile * shape.blocks) * kInt4Cols;
        const int lane = (int)(w >> 2) & 31, s = (int)w & 3;
        uint32_t word = 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t row = tile * kInt4Rows + (lane >> 2) + 8 * (i & 1);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int64_t col = first + int4_column(lane & 3, s, i) + j, g = col / p.group;
                uint32_t code = 0u;
                if (row < p.rows) {
                    if (col < p.cols) code = p.codes[row * p.cols + col];
                    else if (g < groups) code = p.zeros ? p.zeros[row * groups + g] : 8u;
                }
                word |= (code & 15u) << (4 * i + 16 * j);
            }
        }
        out[w] = word;
    }
    const int64_t scales = shape.row_tiles * shape.groups * kInt4Rows;
    for (int64_t w = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; w < scales; w += step) {
        const int64_t g = (w >> 4) % shape.groups, row = (w >> 4) / shape.groups * kInt4Rows + (w & 15);
        uint32_t word = 0u;
        if (row < p.rows && g < groups) word = p.scales[row * groups + g] | (p.zeros ? (uint32_t)p.zeros[row * groups + g] & 15u : 8u) << 16;
        out[words + w] = word;
    }
}

__device__ __forceinline__ float int4_scale(uint32_t word, bool bf16) {
    return bf16 ? __uint_as_float(word << 16) : __half2float(__ushort_as_half((uint16_t)word));
}

// A thread a word: eight values.
__global__ void __launch_bounds__(256) int4_values_kernel(const uint8_t* __restrict__ data, int64_t rows, int64_t cols, int32_t group, int scale_bf16, int dtype,
                                                          void* __restrict__ out) {
    griddep_wait();
    griddep_launch();
    const Int4Shape shape = int4_shape(rows, cols, group);
    const int64_t words = shape.codes_bytes() / 4, step = (int64_t)gridDim.x * blockDim.x;
    const uint32_t* in = reinterpret_cast<const uint32_t*>(data);
    for (int64_t w = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; w < words; w += step) {
        const int64_t block = w >> 7, tile = block / shape.blocks;
        const int64_t first = (block - tile * shape.blocks) * kInt4Cols;
        const int lane = (int)(w >> 2) & 31, s = (int)w & 3;
        const uint32_t word = in[w];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = (lane >> 2) + 8 * (i & 1);
            const int64_t row = tile * kInt4Rows + r;
            const int64_t col = first + int4_column(lane & 3, s, i);
            if (row >= rows) continue;
            const uint32_t sz = in[words + (tile * shape.groups + col / group) * kInt4Rows + r];
            const float scale = int4_scale(sz, scale_bf16);
            const int zero = (int)(sz >> 16);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if (col + j >= cols) continue;
                const float v = (float)((int)((word >> (4 * i + 16 * j)) & 15u) - zero) * scale;      // exact: 5 bits times 11
                const int64_t at = row * cols + col + j;
                if (dtype == MPS_F32) static_cast<float*>(out)[at] = v;
                else static_cast<uint16_t*>(out)[at] = (uint16_t)pack2(v, 0.f, dtype);
            }
        }
    }
}

// ---- products -------------------------------------------------------------------------------------------

struct Int4Args {
    const void* x;
    const uint8_t* w;
    void* out;
    int64_t x_stride, out_stride, tokens;
    int64_t rows;
    int32_t cols, group, blocks, groups;
    int32_t out_dtype;
    bool scale_bf16, x_vec;
};

template <bool BF16>
__device__ __forceinline__ uint32_t subtract2(uint32_t a, uint32_t b) {
    uint32_t r;
    if (BF16) asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Two codes, nibble i of both halves of `w`, minus their zero point: `zero` is 128 + z in BF16 (1024 + z in F16), twice.
template <bool BF16>
__device__ __forceinline__ uint32_t int4_pair(uint32_t w, int i, uint32_t zero) {
    return subtract2<BF16>(((w >> (4 * i)) & 0x000F000Fu) | (BF16 ? 0x43004300u : 0x64006400u), zero);
}
template <bool BF16>
__device__ __forceinline__ uint32_t int4_zero(uint32_t word) {
    const uint32_t z = word >> 16;
    return (z | z << 16) | (BF16 ? 0x43004300u : 0x64006400u);
}

// A CTA of eight warps has 16 features; the warps share their columns, a group (64 columns at least) in turn.
constexpr int kInt4Warps = 8;

template <int TILES, bool BF16>
__global__ void __launch_bounds__(kInt4Warps * 32) int4_few_kernel(const Int4Args p) {
    __shared__ float parts[kInt4Warps][TILES * 8][kInt4Rows + 1];
    griddep_wait();
    griddep_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t tile = blockIdx.x, token0 = (int64_t)blockIdx.y * (TILES * 8);
    const int tokens = (int)min((int64_t)(TILES * 8), p.tokens - token0);
    const uint4* codes = reinterpret_cast<const uint4*>(p.w + tile * p.blocks * kInt4BlockBytes) + lane;
    const uint32_t* scales = reinterpret_cast<const uint32_t*>(p.w + (int64_t)gridDim.x * p.blocks * kInt4BlockBytes) + tile * p.groups * kInt4Rows;
    const uint16_t* x = static_cast<const uint16_t*>(p.x) + token0 * p.x_stride;
    const int unit = max(p.group, kInt4Cols), units = p.blocks * kInt4Cols / unit;

    float acc[TILES][4];
#pragma unroll
    for (int n = 0; n < TILES; ++n) { acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f; }
    for (int u = warp; u < units; u += kInt4Warps) {
        // a unit is one group of 128 (two blocks), one of 64, or two of 32 (half a block each)
        float part[TILES][4];
        uint32_t lo = 0u, hi = 0u;
#pragma unroll 1
        for (int h = 0; h < unit / 32; ++h) {
            const int k = u * unit + h * 32;
            if ((k & (p.group - 1)) == 0) {
                lo = scales[(k / p.group) * kInt4Rows + g];
                hi = scales[(k / p.group) * kInt4Rows + g + 8];
#pragma unroll
                for (int n = 0; n < TILES; ++n) { part[n][0] = part[n][1] = part[n][2] = part[n][3] = 0.f; }
            }
            const uint2 w = reinterpret_cast<const uint2*>(codes + (k >> 6) * 32)[(k >> 5) & 1];
            const uint32_t zlo = int4_zero<BF16>(lo), zhi = int4_zero<BF16>(hi);
            uint32_t a[2][4];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const uint32_t v = s ? w.y : w.x;
                a[s][0] = int4_pair<BF16>(v, 0, zlo);
                a[s][1] = int4_pair<BF16>(v, 1, zhi);
                a[s][2] = int4_pair<BF16>(v, 2, zlo);
                a[s][3] = int4_pair<BF16>(v, 3, zhi);
            }
#pragma unroll
            for (int n = 0; n < TILES; ++n) {
                const int token = n * 8 + g;
                const Raw8 b = load_raw8(x, MPS_BF16, token * p.x_stride + k + 8 * t, token < tokens ? p.cols - (k + 8 * t) : 0, p.x_vec);
                multiply<BF16>(part[n], a[0], b.a.x, b.a.y);
                multiply<BF16>(part[n], a[1], b.a.z, b.a.w);
            }
            if (((k + 32) & (p.group - 1)) == 0) {
                const float slo = int4_scale(lo, p.scale_bf16), shi = int4_scale(hi, p.scale_bf16);
#pragma unroll
                for (int n = 0; n < TILES; ++n) {
                    acc[n][0] = fmaf(slo, part[n][0], acc[n][0]);
                    acc[n][1] = fmaf(slo, part[n][1], acc[n][1]);
                    acc[n][2] = fmaf(shi, part[n][2], acc[n][2]);
                    acc[n][3] = fmaf(shi, part[n][3], acc[n][3]);
                }
            }
        }
    }
#pragma unroll
    for (int n = 0; n < TILES; ++n) {
        parts[warp][n * 8 + 2 * t][g] = acc[n][0];
        parts[warp][n * 8 + 2 * t + 1][g] = acc[n][1];
        parts[warp][n * 8 + 2 * t][g + 8] = acc[n][2];
        parts[warp][n * 8 + 2 * t + 1][g + 8] = acc[n][3];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < tokens * kInt4Rows; i += kInt4Warps * 32) {
        const int token = i / kInt4Rows, r = i % kInt4Rows;
        const int64_t row = tile * kInt4Rows + r;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kInt4Warps; ++w) v += parts[w][token][r];
        if (row < p.rows) static_cast<uint16_t*>(p.out)[(token0 + token) * p.out_stride + row] = (uint16_t)pack2(v, 0.f, p.out_dtype);
    }
}

template <int TILES>
static int launch_few(const Int4Args& p, bool bf16, cudaStream_t st) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned int)((p.rows + kInt4Rows - 1) / kInt4Rows), (unsigned int)((p.tokens + TILES * 8 - 1) / (TILES * 8)));
    config.blockDim = dim3(kInt4Warps * 32);
    config.stream = st;
    cudaLaunchAttribute overlap;
    overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    overlap.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &overlap;
    config.numAttrs = 1;
    const cudaError_t e = bf16 ? cudaLaunchKernelEx(&config, int4_few_kernel<TILES, true>, p) : cudaLaunchKernelEx(&config, int4_few_kernel<TILES, false>, p);
    return e == cudaSuccess ? MPS_OK : cuda_fail(e, "int4_few_kernel");
}

}  // namespace mps

using namespace mps;

extern "C" int64_t mps_int4_bytes(int64_t rows, int64_t cols, int32_t group) {
    return int4_size_ok(rows, cols, group) ? int4_shape(rows, cols, group).bytes() : -1;
}

extern "C" int mps_int4_pack(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int64_t rows, int64_t cols, int32_t group, void* data,
                             void* stream) {
    if (!int4_size_ok(rows, cols, group)) { set_error("mps_int4_pack: rows, cols or group out of range"); return MPS_ERR_INVALID; }
    if (rows == 0) return MPS_OK;
    if (!codes || !scales || !data) { set_error("mps_int4_pack: null pointer"); return MPS_ERR_INVALID; }
    if (reinterpret_cast<uintptr_t>(data) & 15u) { set_error("mps_int4_pack: unaligned data"); return MPS_ERR_INVALID; }
    const int64_t words = int4_shape(rows, cols, group).codes_bytes() / 4;
    return launch_overlapping("int4_pack_kernel", int4_pack_kernel, (unsigned int)min((words + 255) / 256, int64_t(1) << 20), dim3(256),
                              static_cast<cudaStream_t>(stream), Int4Parts{codes, scales, zeros, rows, cols, group}, static_cast<uint8_t*>(data));
}

extern "C" int mps_int4_dequantize(const void* data, int64_t rows, int64_t cols, int32_t group, int32_t scale_dtype, int32_t dtype, void* out, void* stream) {
    if (!int4_size_ok(rows, cols, group)) { set_error("mps_int4_dequantize: rows, cols or group out of range"); return MPS_ERR_INVALID; }
    if ((scale_dtype != MPS_BF16 && scale_dtype != MPS_F16) || !mx4_dtype_ok(dtype)) { set_error("mps_int4_dequantize: unknown dtype"); return MPS_ERR_INVALID; }
    if (rows == 0) return MPS_OK;
    if (!data || !out) { set_error("mps_int4_dequantize: null pointer"); return MPS_ERR_INVALID; }
    if (reinterpret_cast<uintptr_t>(data) & 15u) { set_error("mps_int4_dequantize: unaligned data"); return MPS_ERR_INVALID; }
    const int64_t words = int4_shape(rows, cols, group).codes_bytes() / 4;
    return launch_overlapping("int4_values_kernel", int4_values_kernel, (unsigned int)min((words + 255) / 256, int64_t(1) << 20), dim3(256),
                              static_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(data), rows, cols, group, (int)(scale_dtype == MPS_BF16), (int)dtype, out);
}

extern "C" int mps_int4_product(const mps_int4_linear* args, void* stream) {
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
    const Int4Shape shape = int4_shape(a.rows, a.cols, a.group);
    Int4Args p;
    p.x = a.x;
    p.w = static_cast<const uint8_t*>(a.w);
    p.out = a.out;
    p.x_stride = a.x_stride;
    p.out_stride = a.out_stride;
    p.tokens = a.tokens;
    p.rows = a.rows;
    p.cols = (int32_t)a.cols;
    p.group = a.group;
    p.blocks = shape.blocks;
    p.groups = shape.groups;
    p.out_dtype = a.out_dtype;
    p.scale_bf16 = a.scale_dtype == MPS_BF16;
    p.x_vec = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && (a.x_stride % 8 == 0 || a.tokens == 1);
    const bool bf16 = a.x_dtype == MPS_BF16;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a.tokens <= 8) return launch_few<1>(p, bf16, st);
    if (a.tokens <= 16) return launch_few<2>(p, bf16, st);
    if (a.tokens <= 32) return launch_few<4>(p, bf16, st);
    return launch_few<8>(p, bf16, st);
}
