// MXFP4 quantisation and the ways back: matrix <-> tiles, checkpoint parts <-> tiles.
//
// Bounds: memory.  Quantising a BF16 matrix reads 2 bytes and writes 0.53 per element; a warp takes four neighbouring pieces of 256 columns, of one row
// or of several, so that a lane has four 16-byte loads under way, and the codes of a piece leave as one 128-byte line.  14336 x 4096 BF16 in 28 us,
// 5.3 TB/s, and back in 27 us, 5.5 TB/s.
#include "mx4.cuh"

#include <atomic>

namespace mps {

constexpr int kConvertThreads = 256;
constexpr int kConvertPieces = 4;   // of a warp

// Where a warp's pieces are.  Of a row of at least four they are neighbours in it; SHORT rows have fewer, and a warp takes those of several rows (385667 x 128
// BF16 59 us, one row a warp 88; 14336 x 4096 28 us, counted as short ones are 36).
template <bool SHORT>
struct Pieces {
    int64_t rows, row, tile;
    int chunks, chunk, in_tile;
    __device__ __forceinline__ Pieces(int64_t rows_, int chunks_) : rows(rows_), chunks(chunks_) {
        const int64_t warp = ((int64_t)blockIdx.x * kConvertThreads + threadIdx.x) >> 5;
        const int of_row = SHORT ? chunks : (chunks + kConvertPieces - 1) / kConvertPieces;
        const int64_t at = SHORT ? warp * kConvertPieces : warp;
        row = at / of_row;
        chunk = (int)(at - row * of_row) * (SHORT ? 1 : kConvertPieces);
        place();
    }
    __device__ __forceinline__ void place() {
        tile = mx4_tile_offset(row / kMx4Rows, chunk, chunks);
        in_tile = (int)(row % kMx4Rows);
    }
    __device__ __forceinline__ void next() {
        ++chunk;
        tile += kMx4TileBytes;
        if (SHORT && chunk == chunks) { chunk = 0; ++row; place(); }
    }
    __device__ __forceinline__ bool beyond() const { return row >= rows; }                               // once, at the start
    __device__ __forceinline__ bool any() const { return SHORT ? row < rows : chunk < chunks; }
};

// The largest magnitude's bits, as FP32, of eight values as they were loaded: BF16 compares as it is, two at a time.
template <int DTYPE>
__device__ __forceinline__ uint32_t raw_max_bits(const Raw8& r, const float (&v)[8]) {
    if (DTYPE != MPS_BF16) return max_bits8(v);
    const uint32_t a = __vmaxu2(__vmaxu2(r.a.x & 0x7FFF7FFFu, r.a.y & 0x7FFF7FFFu), __vmaxu2(r.a.z & 0x7FFF7FFFu, r.a.w & 0x7FFF7FFFu));
    return max(a & 0xFFFF0000u, a << 16);
}

template <int DTYPE, bool SHORT>
__global__ void __launch_bounds__(kConvertThreads)
mx4_quantize_kernel(const void* __restrict__ x, int64_t rows, int64_t cols, int64_t row_stride, bool vec, int chunks, uint8_t* __restrict__ out) {
    griddep_wait();
    griddep_launch();
    const int lane = threadIdx.x & 31;
    const Pieces<SHORT> first(rows, chunks);
    if (first.beyond()) return;
    Raw8 raw[kConvertPieces];
    Pieces<SHORT> at = first;
#pragma unroll
    for (int i = 0; i < kConvertPieces; ++i, at.next()) {
        const int64_t c = (int64_t)at.chunk * kMx4Cols + lane * 8, left = !SHORT || at.any() ? cols - c : 0;
        raw[i] = load_raw8(x, DTYPE, at.row * row_stride + c, left > 8 ? 8 : (int)left, vec);
    }
    at = first;
#pragma unroll
    for (int i = 0; i < kConvertPieces; ++i, at.next()) {
        if (!at.any()) break;
        float v[8];
        unpack8(raw[i], DTYPE, v);
        mx4_store_row(out + at.tile, at.in_tile, lane, v, raw_max_bits<DTYPE>(raw[i], v));
    }
}

template <int DTYPE, bool SHORT>
__global__ void __launch_bounds__(kConvertThreads)
mx4_dequantize_kernel(const uint8_t* __restrict__ q, int64_t rows, int64_t cols, int chunks, bool vec, void* __restrict__ out) {
    __shared__ __align__(16) float buffers[kConvertThreads / 32][256];
    griddep_wait();
    griddep_launch();
    const int lane = threadIdx.x & 31;
    const Pieces<SHORT> first(rows, chunks);
    if (first.beyond()) return;
    uint32_t codes[kConvertPieces], scale[kConvertPieces];
    Pieces<SHORT> at = first;
#pragma unroll
    for (int i = 0; i < kConvertPieces; ++i, at.next()) {
        codes[i] = scale[i] = 0u;
        if (at.any()) {
            const uint8_t* tile = q + at.tile;
            codes[i] = *reinterpret_cast<const uint32_t*>(tile + mx4_code_offset(at.in_tile, lane >> 2) + (lane & 3) * 4);
            scale[i] = tile[mx4_scale_offset(at.in_tile, lane >> 4) + ((lane >> 2) & 3)];
        }
    }
    at = first;
#pragma unroll
    for (int i = 0; i < kConvertPieces; ++i, at.next()) {
        if (!at.any()) break;
        const int64_t c = (int64_t)at.chunk * kMx4Cols, left = cols - c;
        const float s = mx4_scale(scale[i]);
        float v[8];
        mx4_values8(codes[i], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= s;
        if (vec && left >= kMx4Cols) store8(out, DTYPE, at.row * cols + c + lane * 8, 8, true, v);
        else if (vec && left % 8 == 0) store8(out, DTYPE, at.row * cols + c + lane * 8, lane * 8 < left ? 8 : 0, true, v);
        else store_span(out, DTYPE, at.row * cols + c, left > kMx4Cols ? kMx4Cols : (int)left, buffers[threadIdx.x >> 5], lane, v);
    }
}

// Checkpoint parts: codes [rows, ceil(cols / 2)], two a byte with the even column low, and scales [rows, ceil(cols / 32)].  What lies
// beyond the last column in them is not taken over.
template <bool SHORT>
__global__ void __launch_bounds__(kConvertThreads)
mx4_pack_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t rows, int64_t cols, int chunks, uint8_t* __restrict__ out) {
    griddep_wait();
    griddep_launch();
    const int lane = threadIdx.x & 31;
    const int64_t row_bytes = (cols + 1) / 2, blocks = (cols + kMx4Block - 1) / kMx4Block;
    Pieces<SHORT> at(rows, chunks);
    if (at.beyond()) return;
#pragma unroll
    for (int i = 0; i < kConvertPieces; ++i, at.next()) {
        if (!at.any()) break;
        uint8_t* tile = out + at.tile;
        const int64_t c = (int64_t)at.chunk * kMx4Cols + lane * 8;
        uint32_t word = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + 2 * j < cols) {
                uint32_t b = codes[at.row * row_bytes + c / 2 + j];
                if (c + 2 * j + 1 >= cols) b &= 15u;
                word |= b << (8 * j);
            }
        *reinterpret_cast<uint32_t*>(tile + mx4_code_offset(at.in_tile, lane >> 2) + (lane & 3) * 4) = word;
        if (lane < 8) {
            const int64_t block = (int64_t)at.chunk * 8 + lane;
            tile[mx4_scale_offset(at.in_tile, lane >> 2) + (lane & 3)] = block < blocks ? scales[at.row * blocks + block] : (uint8_t)0;
        }
    }
}

template <bool SHORT>
__global__ void __launch_bounds__(kConvertThreads)
mx4_unpack_kernel(const uint8_t* __restrict__ q, int64_t rows, int64_t cols, int chunks, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    griddep_wait();
    griddep_launch();
    const int lane = threadIdx.x & 31;
    const int64_t row_bytes = (cols + 1) / 2, blocks = (cols + kMx4Block - 1) / kMx4Block;
    Pieces<SHORT> at(rows, chunks);
    if (at.beyond()) return;
#pragma unroll
    for (int i = 0; i < kConvertPieces; ++i, at.next()) {
        if (!at.any()) break;
        const uint8_t* tile = q + at.tile;
        const int64_t c = (int64_t)at.chunk * kMx4Cols + lane * 8, block = (int64_t)at.chunk * 8 + lane;
        const uint32_t word = *reinterpret_cast<const uint32_t*>(tile + mx4_code_offset(at.in_tile, lane >> 2) + (lane & 3) * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + 2 * j < cols) codes[at.row * row_bytes + c / 2 + j] = (uint8_t)(word >> (8 * j));
        if (lane < 8 && block < blocks) scales[at.row * blocks + block] = tile[mx4_scale_offset(at.in_tile, lane >> 2) + (lane & 3)];
    }
}

struct ConvertGrid { int chunks; bool few; unsigned int ctas; };

static int convert_grid(const char* who, int64_t rows, int64_t cols, ConvertGrid& g) {
    if (rows < 0 || rows > kMx4MostRows || cols <= 0 || cols > kMx4MostCols) {
        set_error("%s: rows must be in [0, %lld], cols in [1, %lld]", who, (long long)kMx4MostRows, (long long)kMx4MostCols);
        return MPS_ERR_INVALID;
    }
    g.chunks = (int)mx4_chunks(cols);
    g.few = g.chunks < kConvertPieces;
    const int64_t warps = g.few ? (rows * g.chunks + kConvertPieces - 1) / kConvertPieces : rows * ((g.chunks + kConvertPieces - 1) / kConvertPieces);
    const int64_t ctas = (warps + kConvertThreads / 32 - 1) / (kConvertThreads / 32);
    if (ctas > 0x7FFFFFFFLL) { set_error("%s: matrix too large", who); return MPS_ERR_INVALID; }
    g.ctas = (unsigned int)ctas;
    return MPS_OK;
}

// The current device, its SMs counted once.
int current_device(Device& d) {
    static std::atomic<int> sms[64];
    MPS_CUDA_TRY(cudaGetDevice(&d.ordinal));
    if (d.ordinal < 0 || d.ordinal >= 64) { set_error("device ordinal %d out of range", d.ordinal); return MPS_ERR_UNSUPPORTED; }
    d.sms = sms[d.ordinal].load(std::memory_order_relaxed);
    if (d.sms == 0) {
        MPS_CUDA_TRY(cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, d.ordinal));
        sms[d.ordinal].store(d.sms, std::memory_order_relaxed);
    }
    return MPS_OK;
}

}  // namespace mps

using namespace mps;

extern "C" {

int64_t mps_mx4_bytes(int64_t rows, int64_t cols) {
    if (rows < 0 || rows > kMx4MostRows || cols <= 0 || cols > kMx4MostCols) return -1;
    return mx4_row_tiles(rows) * mx4_chunks(cols) * kMx4TileBytes;
}

int mps_mx4_quantize(const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t row_stride, void* tiles, void* stream) {
    ConvertGrid g;
    int rc = convert_grid("mps_mx4_quantize", rows, cols, g);
    if (rc) return rc;
    if (!mx4_dtype_ok(dtype)) { set_error("mps_mx4_quantize: unknown dtype %d", (int)dtype); return MPS_ERR_INVALID; }
    if (rows == 0) return MPS_OK;
    if (!x || !tiles || (reinterpret_cast<uintptr_t>(tiles) & 15u)) { set_error("mps_mx4_quantize: null or unaligned pointer"); return MPS_ERR_INVALID; }
    const auto kernel = g.few ? (dtype == MPS_BF16 ? mx4_quantize_kernel<MPS_BF16, true> : dtype == MPS_F16 ? mx4_quantize_kernel<MPS_F16, true> : mx4_quantize_kernel<MPS_F32, true>)
                              : (dtype == MPS_BF16 ? mx4_quantize_kernel<MPS_BF16, false> : dtype == MPS_F16 ? mx4_quantize_kernel<MPS_F16, false> : mx4_quantize_kernel<MPS_F32, false>);
    return launch_overlapping("mx4_quantize_kernel", kernel, g.ctas, kConvertThreads, static_cast<cudaStream_t>(stream), x, rows, cols, row_stride,
                              mx4_vec_ok(x, row_stride, dtype), g.chunks, static_cast<uint8_t*>(tiles));
}

int mps_mx4_dequantize(const void* tiles, int64_t rows, int64_t cols, int32_t dtype, void* out, void* stream) {
    ConvertGrid g;
    int rc = convert_grid("mps_mx4_dequantize", rows, cols, g);
    if (rc) return rc;
    if (!mx4_dtype_ok(dtype)) { set_error("mps_mx4_dequantize: unknown dtype %d", (int)dtype); return MPS_ERR_INVALID; }
    if (rows == 0) return MPS_OK;
    if (!tiles || !out || (reinterpret_cast<uintptr_t>(tiles) & 15u)) { set_error("mps_mx4_dequantize: null or unaligned pointer"); return MPS_ERR_INVALID; }
    const auto kernel = g.few ? (dtype == MPS_BF16 ? mx4_dequantize_kernel<MPS_BF16, true> : dtype == MPS_F16 ? mx4_dequantize_kernel<MPS_F16, true> : mx4_dequantize_kernel<MPS_F32, true>)
                              : (dtype == MPS_BF16 ? mx4_dequantize_kernel<MPS_BF16, false> : dtype == MPS_F16 ? mx4_dequantize_kernel<MPS_F16, false> : mx4_dequantize_kernel<MPS_F32, false>);
    return launch_overlapping("mx4_dequantize_kernel", kernel, g.ctas, kConvertThreads, static_cast<cudaStream_t>(stream),
                              static_cast<const uint8_t*>(tiles), rows, cols, g.chunks, mx4_vec_ok(out, cols, dtype), out);
}

int mps_mx4_pack(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t cols, void* tiles, void* stream) {
    ConvertGrid g;
    int rc = convert_grid("mps_mx4_pack", rows, cols, g);
    if (rc || rows == 0) return rc;
    if (!codes || !scales || !tiles || (reinterpret_cast<uintptr_t>(tiles) & 15u)) { set_error("mps_mx4_pack: null or unaligned pointer"); return MPS_ERR_INVALID; }
    return launch_overlapping("mx4_pack_kernel", g.few ? mx4_pack_kernel<true> : mx4_pack_kernel<false>, g.ctas, kConvertThreads, static_cast<cudaStream_t>(stream), codes, scales, rows, cols,
                              g.chunks, static_cast<uint8_t*>(tiles));
}

int mps_mx4_unpack(const void* tiles, int64_t rows, int64_t cols, uint8_t* codes, uint8_t* scales, void* stream) {
    ConvertGrid g;
    int rc = convert_grid("mps_mx4_unpack", rows, cols, g);
    if (rc || rows == 0) return rc;
    if (!tiles || !codes || !scales || (reinterpret_cast<uintptr_t>(tiles) & 15u)) { set_error("mps_mx4_unpack: null or unaligned pointer"); return MPS_ERR_INVALID; }
    return launch_overlapping("mx4_unpack_kernel", g.few ? mx4_unpack_kernel<true> : mx4_unpack_kernel<false>, g.ctas, kConvertThreads, static_cast<cudaStream_t>(stream),
                              static_cast<const uint8_t*>(tiles), rows, cols, g.chunks, codes, scales);
}

}  // extern "C"
