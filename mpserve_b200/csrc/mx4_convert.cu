// MXFP4 quantisation and the ways back: matrix <-> tiles, checkpoint parts <-> tiles.
//
// Bounds: memory, and instructions nearly as much.  Quantising a BF16 matrix reads 2 bytes and writes 0.53 per element; a warp takes four neighbouring
// pieces of 256 columns, of one row or of several, so that a lane has 64 bytes under way, and the codes of a piece leave as one 128-byte line.
// Long 16-bit rows that begin at multiples of 32 bytes have kernels of their own with sixteen columns a lane, half a block, which need half the instructions
// (14336 x 4096 BF16 23.3 us, 6.4 TB/s, with eight columns a lane 28; and back 24.6 us, 6.0 TB/s, with eight 27).
#include "mx4.cuh"

#include <atomic>

namespace mps {

constexpr int kConvertThreads = 256;
constexpr int kConvertPieces = 4;   // of a warp

// Where a warp's pieces are.  Of a row of at least four they are neighbours in it; SHORT rows have fewer, and a warp takes those of several rows (385667 x 128
// BF16 59 us, one row a warp 96; 14336 x 4096 28 us, counted as short ones are 36).
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

// Long rows of a 16-bit type: at least four pieces, a multiple of 16 columns, every row at a multiple of 32 bytes.  A lane has sixteen columns, a warp two
// neighbouring tiles at a time.  (FP32, 64 bytes a lane, takes longer this way than with eight columns a lane: 3000 x 5008 12.1 us against 11.7, and back
// 25 against 18.)
struct LongPlace {
    int64_t row;
    int chunk, column;                   // this lane's tile in the first step, and its column
    int64_t tile;
    int codes, scale;                    // this lane's codes and its block's scale in a tile
};
static __device__ __forceinline__ LongPlace long_place(int chunks) {
    const int64_t warp = ((int64_t)blockIdx.x * kConvertThreads + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31, of_row = (chunks + kConvertPieces - 1) / kConvertPieces;
    LongPlace p;
    p.row = warp / of_row;
    p.chunk = (int)(warp - p.row * of_row) * kConvertPieces + (lane >> 4);
    p.column = p.chunk * kMx4Cols + (lane & 15) * 16;
    p.tile = mx4_tile_offset(p.row / kMx4Rows, p.chunk, chunks);
    const int in_tile = (int)(p.row % kMx4Rows), block = (lane & 15) >> 1;
    p.codes = mx4_code_offset(in_tile, block) + (lane & 1) * 8;
    p.scale = mx4_scale_offset(in_tile, block >> 2) + (block & 3);
    return p;
}

template <int DTYPE>
__global__ void __launch_bounds__(kConvertThreads)
mx4_quantize_long_kernel(const void* __restrict__ x, int64_t rows, int cols, int64_t row_stride, int chunks, uint8_t* __restrict__ out) {
    constexpr int kSteps = kConvertPieces / 2;
    griddep_wait();
    griddep_launch();
    const LongPlace p = long_place(chunks);
    if (p.row >= rows) return;
    Raw8 raw[kSteps];      // sixteen 16-bit values each
    const uint16_t* from = static_cast<const uint16_t*>(x) + p.row * row_stride + p.column;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        raw[i].a = raw[i].b = make_uint4(0u, 0u, 0u, 0u);
        if (p.column + i * 2 * kMx4Cols < cols) raw[i] = load_wide8(reinterpret_cast<const float*>(from + i * 2 * kMx4Cols));
    }
    uint8_t* tile = out + p.tile;
#pragma unroll
    for (int i = 0; i < kSteps; ++i, tile += 2 * kMx4TileBytes) {
        Pairs a, b;
        unpack8(raw[i], DTYPE, a.each());
        raw[i].a = raw[i].b;
        unpack8(raw[i], DTYPE, b.each());
        uint32_t m = max(max_bits8(a.each()), max_bits8(b.each()));
        m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
        const uint32_t byte = mx4_scale_byte(m);
        const float inverse = mx4_inverse_scale(byte);
        a = times(a, inverse);
        b = times(b, inverse);
        if (p.chunk + 2 * i < chunks) {            // all lanes take part in every step's exchange
            *reinterpret_cast<uint2*>(tile + p.codes) = make_uint2(mx4_codes8(a.each()), mx4_codes8(b.each()));
            if (!(threadIdx.x & 1)) tile[p.scale] = (uint8_t)byte;
        }
    }
}

template <int DTYPE>
__global__ void __launch_bounds__(kConvertThreads)
mx4_dequantize_long_kernel(const uint8_t* __restrict__ q, int64_t rows, int cols, int chunks, void* __restrict__ out) {
    constexpr int kSteps = kConvertPieces / 2;
    griddep_wait();
    griddep_launch();
    const LongPlace p = long_place(chunks);
    if (p.row >= rows) return;
    uint2 codes[kSteps];
    uint32_t byte[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        codes[i] = make_uint2(0u, 0u);
        byte[i] = 0u;
        if (p.column + i * 2 * kMx4Cols < cols) {
            const uint8_t* tile = q + p.tile + i * 2 * kMx4TileBytes;
            codes[i] = *reinterpret_cast<const uint2*>(tile + p.codes);
            byte[i] = tile[p.scale];
        }
    }
    const int64_t to = p.row * cols + p.column;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        if (p.column + i * 2 * kMx4Cols >= cols) break;
        Pairs a, b;
        mx4_values8(codes[i].x, a.each());
        mx4_values8(codes[i].y, b.each());
        const float s = mx4_scale(byte[i]);
        a = times(a, s);
        b = times(b, s);
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            w[j] = pack2(a.p[j].x, a.p[j].y, DTYPE);
            w[4 + j] = pack2(b.p[j].x, b.p[j].y, DTYPE);
        }
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(static_cast<uint16_t*>(out) + to + i * 2 * kMx4Cols),
                     "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
    }
}

// Checkpoint parts: codes [rows, ceil(cols / 2)], two a byte with the even column low, and scales [rows, ceil(cols / 32)].  What lies
// beyond the last column in them is not taken over.  Byte by byte, since their rows begin anywhere: 14336 x 4096 37 us, and back 33 us (62 MB, 9.5 us at the
// rate of HBM), once for a weight when it is loaded.
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

static bool long_ok(const void* p, int64_t row_stride, int64_t cols, int dtype) {
    return dtype != MPS_F32 && cols % 16 == 0 && reinterpret_cast<uintptr_t>(p) % 32 == 0 && row_stride % 16 == 0;
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
    if (!g.few && long_ok(x, row_stride, cols, dtype)) {
        const auto kernel = dtype == MPS_BF16 ? mx4_quantize_long_kernel<MPS_BF16> : mx4_quantize_long_kernel<MPS_F16>;
        return launch_overlapping("mx4_quantize_long_kernel", kernel, g.ctas, kConvertThreads, static_cast<cudaStream_t>(stream), x, rows, (int)cols, row_stride,
                                  g.chunks, static_cast<uint8_t*>(tiles));
    }
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
    if (!g.few && long_ok(out, cols, cols, dtype)) {
        const auto kernel = dtype == MPS_BF16 ? mx4_dequantize_long_kernel<MPS_BF16> : mx4_dequantize_long_kernel<MPS_F16>;
        return launch_overlapping("mx4_dequantize_long_kernel", kernel, g.ctas, kConvertThreads, static_cast<cudaStream_t>(stream),
                                  static_cast<const uint8_t*>(tiles), rows, (int)cols, g.chunks, out);
    }
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
