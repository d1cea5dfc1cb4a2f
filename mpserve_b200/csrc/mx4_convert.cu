// MXFP4 quantisation and the ways back: matrix <-> tiles, checkpoint parts <-> tiles.
//
// Bounds: memory.  Quantising a BF16 matrix reads 2 bytes and writes 0.53 per element; a warp takes one row of up to four
// tiles, so that a lane has four 16-byte loads under way, and each tile row leaves as one 128-byte line.
#include "mx4.cuh"

#include <atomic>

namespace mps {

constexpr int kConvertThreads = 256;
constexpr int kConvertChunks = 4;   // tiles that a warp takes of a row

struct ConvertPlace { int64_t row; int64_t chunk0; };

static __device__ __forceinline__ bool convert_place(int64_t rows, int segments, ConvertPlace& p) {
    const int64_t unit = ((int64_t)blockIdx.x * kConvertThreads + threadIdx.x) >> 5;
    p.row = unit / segments;
    p.chunk0 = (unit - p.row * segments) * kConvertChunks;
    return p.row < rows;
}

// The largest magnitude's bits, as FP32, of eight values as they were loaded: BF16 compares as it is, two at a time.
template <int DTYPE>
__device__ __forceinline__ uint32_t raw_max_bits(const Raw8& r, const float (&v)[8]) {
    if (DTYPE != MPS_BF16) return max_bits8(v);
    const uint32_t a = __vmaxu2(__vmaxu2(r.a.x & 0x7FFF7FFFu, r.a.y & 0x7FFF7FFFu), __vmaxu2(r.a.z & 0x7FFF7FFFu, r.a.w & 0x7FFF7FFFu));
    return max(a & 0xFFFF0000u, a << 16);
}

template <int DTYPE>
__global__ void __launch_bounds__(kConvertThreads)
mx4_quantize_kernel(const void* __restrict__ x, int64_t rows, int64_t cols, int64_t row_stride, bool vec, int chunks, int segments,
                    uint8_t* __restrict__ out) {
    griddep_wait();
    griddep_launch();
    ConvertPlace p;
    if (!convert_place(rows, segments, p)) return;
    const int lane = threadIdx.x & 31, row = (int)(p.row % kMx4Rows);
    Raw8 raw[kConvertChunks];
#pragma unroll
    for (int i = 0; i < kConvertChunks; ++i) {
        const int64_t c = (p.chunk0 + i) * kMx4Cols + lane * 8, left = cols - c;
        raw[i] = load_raw8(x, DTYPE, p.row * row_stride + c, left > 8 ? 8 : (int)left, vec);
    }
    uint8_t* tile = out + mx4_tile_offset(p.row / kMx4Rows, p.chunk0, chunks);
#pragma unroll
    for (int i = 0; i < kConvertChunks; ++i, tile += kMx4TileBytes) {
        if (p.chunk0 + i >= chunks) break;
        float v[8];
        unpack8(raw[i], DTYPE, v);
        mx4_store_row(tile, row, lane, v, raw_max_bits<DTYPE>(raw[i], v));
    }
}

template <int DTYPE>
__global__ void __launch_bounds__(kConvertThreads)
mx4_dequantize_kernel(const uint8_t* __restrict__ q, int64_t rows, int64_t cols, int chunks, int segments, bool vec, void* __restrict__ out) {
    __shared__ __align__(16) float buffers[kConvertThreads / 32][256];
    griddep_wait();
    griddep_launch();
    ConvertPlace p;
    if (!convert_place(rows, segments, p)) return;
    const int lane = threadIdx.x & 31, row = (int)(p.row % kMx4Rows);
    const uint8_t* tile = q + mx4_tile_offset(p.row / kMx4Rows, p.chunk0, chunks);
    uint32_t codes[kConvertChunks], scale[kConvertChunks];
#pragma unroll
    for (int i = 0; i < kConvertChunks; ++i) {
        codes[i] = scale[i] = 0u;
        if (p.chunk0 + i < chunks) {
            codes[i] = *reinterpret_cast<const uint32_t*>(tile + i * kMx4TileBytes + mx4_code_offset(row, lane >> 2) + (lane & 3) * 4);
            scale[i] = tile[i * kMx4TileBytes + mx4_scale_offset(row, lane >> 4) + ((lane >> 2) & 3)];
        }
    }
#pragma unroll
    for (int i = 0; i < kConvertChunks; ++i) {
        if (p.chunk0 + i >= chunks) break;
        const int64_t c = (p.chunk0 + i) * kMx4Cols, left = cols - c;
        const float s = mx4_scale(scale[i]);
        float v[8];
        mx4_values8(codes[i], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= s;
        if (vec && left >= kMx4Cols) store8(out, DTYPE, p.row * cols + c + lane * 8, 8, true, v);
        else store_span(out, DTYPE, p.row * cols + c, left > kMx4Cols ? kMx4Cols : (int)left, buffers[threadIdx.x >> 5], lane, v);
    }
}

// Checkpoint parts: codes [rows, ceil(cols / 2)], two a byte with the even column low, and scales [rows, ceil(cols / 32)].  What lies
// beyond the last column in them is not taken over.
__global__ void __launch_bounds__(kConvertThreads)
mx4_pack_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t rows, int64_t cols, int chunks,
                int segments, uint8_t* __restrict__ out) {
    griddep_wait();
    griddep_launch();
    ConvertPlace p;
    if (!convert_place(rows, segments, p)) return;
    const int lane = threadIdx.x & 31, row = (int)(p.row % kMx4Rows);
    const int64_t row_bytes = (cols + 1) / 2, blocks = (cols + kMx4Block - 1) / kMx4Block;
#pragma unroll
    for (int i = 0; i < kConvertChunks; ++i) {
        const int64_t chunk = p.chunk0 + i;
        if (chunk >= chunks) break;
        uint8_t* tile = out + mx4_tile_offset(p.row / kMx4Rows, chunk, chunks);
        const int64_t c = chunk * kMx4Cols + lane * 8;
        uint32_t word = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + 2 * j < cols) {
                uint32_t b = codes[p.row * row_bytes + c / 2 + j];
                if (c + 2 * j + 1 >= cols) b &= 15u;
                word |= b << (8 * j);
            }
        *reinterpret_cast<uint32_t*>(tile + mx4_code_offset(row, lane >> 2) + (lane & 3) * 4) = word;
        if (lane < 8) {
            const int64_t block = chunk * 8 + lane;
            tile[mx4_scale_offset(row, lane >> 2) + (lane & 3)] = block < blocks ? scales[p.row * blocks + block] : (uint8_t)0;
        }
    }
}

__global__ void __launch_bounds__(kConvertThreads)
mx4_unpack_kernel(const uint8_t* __restrict__ q, int64_t rows, int64_t cols, int chunks, int segments, uint8_t* __restrict__ codes,
                  uint8_t* __restrict__ scales) {
    griddep_wait();
    griddep_launch();
    ConvertPlace p;
    if (!convert_place(rows, segments, p)) return;
    const int lane = threadIdx.x & 31, row = (int)(p.row % kMx4Rows);
    const int64_t row_bytes = (cols + 1) / 2, blocks = (cols + kMx4Block - 1) / kMx4Block;
#pragma unroll
    for (int i = 0; i < kConvertChunks; ++i) {
        const int64_t chunk = p.chunk0 + i;
        if (chunk >= chunks) break;
        const uint8_t* tile = q + mx4_tile_offset(p.row / kMx4Rows, chunk, chunks);
        const int64_t c = chunk * kMx4Cols + lane * 8;
        const uint32_t word = *reinterpret_cast<const uint32_t*>(tile + mx4_code_offset(row, lane >> 2) + (lane & 3) * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + 2 * j < cols) codes[p.row * row_bytes + c / 2 + j] = (uint8_t)(word >> (8 * j));
        if (lane < 8 && chunk * 8 + lane < blocks)
            scales[p.row * blocks + chunk * 8 + lane] = tile[mx4_scale_offset(row, lane >> 2) + (lane & 3)];
    }
}

struct ConvertGrid { int chunks, segments; unsigned int ctas; };

static int convert_grid(const char* who, int64_t rows, int64_t cols, ConvertGrid& g) {
    if (rows < 0 || rows > kMx4MostRows || cols <= 0 || cols > kMx4MostCols) {
        set_error("%s: rows must be in [0, %lld], cols in [1, %lld]", who, (long long)kMx4MostRows, (long long)kMx4MostCols);
        return MPS_ERR_INVALID;
    }
    g.chunks = (int)mx4_chunks(cols);
    g.segments = (g.chunks + kConvertChunks - 1) / kConvertChunks;
    const int64_t per_cta = kConvertThreads / 32, ctas = (rows * g.segments + per_cta - 1) / per_cta;
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
    const auto kernel = dtype == MPS_BF16 ? mx4_quantize_kernel<MPS_BF16> : dtype == MPS_F16 ? mx4_quantize_kernel<MPS_F16> : mx4_quantize_kernel<MPS_F32>;
    return launch_overlapping("mx4_quantize_kernel", kernel, g.ctas, kConvertThreads, static_cast<cudaStream_t>(stream), x, rows, cols, row_stride,
                              mx4_vec_ok(x, row_stride, dtype), g.chunks, g.segments, static_cast<uint8_t*>(tiles));
}

int mps_mx4_dequantize(const void* tiles, int64_t rows, int64_t cols, int32_t dtype, void* out, void* stream) {
    ConvertGrid g;
    int rc = convert_grid("mps_mx4_dequantize", rows, cols, g);
    if (rc) return rc;
    if (!mx4_dtype_ok(dtype)) { set_error("mps_mx4_dequantize: unknown dtype %d", (int)dtype); return MPS_ERR_INVALID; }
    if (rows == 0) return MPS_OK;
    if (!tiles || !out || (reinterpret_cast<uintptr_t>(tiles) & 15u)) { set_error("mps_mx4_dequantize: null or unaligned pointer"); return MPS_ERR_INVALID; }
    const auto kernel = dtype == MPS_BF16 ? mx4_dequantize_kernel<MPS_BF16> : dtype == MPS_F16 ? mx4_dequantize_kernel<MPS_F16> : mx4_dequantize_kernel<MPS_F32>;
    return launch_overlapping("mx4_dequantize_kernel", kernel, g.ctas, kConvertThreads, static_cast<cudaStream_t>(stream),
                              static_cast<const uint8_t*>(tiles), rows, cols, g.chunks, g.segments, mx4_vec_ok(out, cols, dtype), out);
}

int mps_mx4_pack(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t cols, void* tiles, void* stream) {
    ConvertGrid g;
    int rc = convert_grid("mps_mx4_pack", rows, cols, g);
    if (rc || rows == 0) return rc;
    if (!codes || !scales || !tiles || (reinterpret_cast<uintptr_t>(tiles) & 15u)) { set_error("mps_mx4_pack: null or unaligned pointer"); return MPS_ERR_INVALID; }
    return launch_overlapping("mx4_pack_kernel", mx4_pack_kernel, g.ctas, kConvertThreads, static_cast<cudaStream_t>(stream), codes, scales, rows, cols,
                              g.chunks, g.segments, static_cast<uint8_t*>(tiles));
}

int mps_mx4_unpack(const void* tiles, int64_t rows, int64_t cols, uint8_t* codes, uint8_t* scales, void* stream) {
    ConvertGrid g;
    int rc = convert_grid("mps_mx4_unpack", rows, cols, g);
    if (rc || rows == 0) return rc;
    if (!tiles || !codes || !scales || (reinterpret_cast<uintptr_t>(tiles) & 15u)) { set_error("mps_mx4_unpack: null or unaligned pointer"); return MPS_ERR_INVALID; }
    return launch_overlapping("mx4_unpack_kernel", mx4_unpack_kernel, g.ctas, kConvertThreads, static_cast<cudaStream_t>(stream),
                              static_cast<const uint8_t*>(tiles), rows, cols, g.chunks, g.segments, codes, scales);
}

}  // extern "C"
