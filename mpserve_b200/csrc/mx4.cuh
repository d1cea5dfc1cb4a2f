// MXFP4 as this library holds it, and the device code that its kernels share.
//
// A value is an E2M1 code (sign, two exponent bits, one mantissa bit: 0, .5, 1, 1.5, 2, 3, 4, 6) times a scale, a power of two in a
// byte (E8M0: 2^(byte - 127), 255 is NaN) that 32 neighbouring columns of a row share.  For a block with largest magnitude a
// the scale is 2^(floor(log2 a) - 2), which puts a into [4, 8); codes are rounded to nearest, halfway to the even code, and
// what is above 6 becomes 6.  A block that holds an infinity or a NaN gets the scale 255: all its values are NaN.
//
// In memory a matrix is a row-major array of tiles of 128 rows x 256 columns.  A tile is 17408 bytes in one piece: first the scales
// of its two halves of 128 columns, 512 bytes each, row r at 16 (r % 32) + 4 (r / 32), four bytes for its four blocks; then
// the codes, 128 bytes a row, the even column in the low half of a byte, the row's eight 16-byte pieces at their place XOR
// (row % 8).  That is what the tensor cores read from shared memory, so one bulk copy brings a tile and nothing is laid out again:
// a weight streams from HBM in pieces of 17 KB, 4.25 bits an element.  Columns are filled up to a multiple of 256 with zero
// codes of the least scale; rows beyond the last are never read as values (they are what the memory holds).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mps_common.cuh"

namespace mps {

constexpr int kMx4Rows = 128, kMx4Cols = 256, kMx4Block = 32;
constexpr int kMx4ScaleBytes = 1024, kMx4RowBytes = 128;
constexpr int kMx4TileBytes = kMx4ScaleBytes + kMx4Rows * kMx4RowBytes;

__host__ __device__ inline int64_t mx4_row_tiles(int64_t rows) { return (rows + kMx4Rows - 1) / kMx4Rows; }
__host__ __device__ inline int64_t mx4_chunks(int64_t cols) { return (cols + kMx4Cols - 1) / kMx4Cols; }
// Every offset of a tile is 64 bits wide: a matrix may hold more than 2^32 bytes.
__host__ __device__ inline int64_t mx4_tile_offset(int64_t row_tile, int64_t chunk, int64_t chunks) {
    return (row_tile * chunks + chunk) * kMx4TileBytes;
}
// Inside a tile: the scale word (four blocks) of a row in half `half`, and 16-byte piece `piece` of its codes.
__host__ __device__ inline int mx4_scale_offset(int row, int half) { return half * 512 + (row & 31) * 16 + (row >> 5) * 4; }
__host__ __device__ inline int mx4_code_offset(int row, int piece) {
    return kMx4ScaleBytes + row * kMx4RowBytes + ((piece ^ (row & 7)) << 4);
}

// ---- values of the tensors that come in and go out -------------------------------------------------

// Eight neighbouring elements as they were loaded: 16 bytes of a 16-bit type, or 32 of FP32.
struct Raw8 { uint4 a, b; };

// 32 bytes at a time: as two halves, each would touch every second 16 bytes of a warp's kilobyte.  (Stored as two halves all the same: as one, rows of
// 4096 FP32 beside BF16 took 68 us where they take 64, rows of FP32 alone 41 and 43.)
__device__ __forceinline__ Raw8 load_wide8(const float* p) {
    Raw8 r;
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r.a.x), "=r"(r.a.y), "=r"(r.a.z), "=r"(r.a.w), "=r"(r.b.x), "=r"(r.b.y), "=r"(r.b.z), "=r"(r.b.w) : "l"(p));
    return r;
}

// `vec`: the address is aligned to the eight elements (host rule on pointer and stride, mx4_vec_ok).  Elements from `valid` on are zero.
__device__ __forceinline__ Raw8 load_raw8(const void* __restrict__ base, int dtype, int64_t at, int valid, bool vec) {
    Raw8 r;
    r.a = make_uint4(0u, 0u, 0u, 0u);
    r.b = r.a;
    if (valid <= 0) return r;
    if (dtype == MPS_F32) {
        const float* p = static_cast<const float*>(base) + at;
        if (vec && valid >= 8) {
            r = load_wide8(p);
        } else {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = i < valid ? __float_as_uint(p[i]) : 0u;
            r.a = make_uint4(w[0], w[1], w[2], w[3]);
            r.b = make_uint4(w[4], w[5], w[6], w[7]);
        }
    } else {
        const uint16_t* p = static_cast<const uint16_t*>(base) + at;
        if (vec && valid >= 8) {
            r.a = *reinterpret_cast<const uint4*>(p);
        } else {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = i < valid ? (uint32_t)p[i] : 0u;
            r.a = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
        }
    }
    return r;
}

__device__ __forceinline__ void unpack8(const Raw8& r, int dtype, float (&v)[8]) {
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
    if (dtype == MPS_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
    } else if (dtype == MPS_BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}

// Two values in a 16-bit type, rounded to nearest even.
__device__ __forceinline__ uint32_t pack2(float lo, float hi, int dtype) {
    if (dtype == MPS_BF16) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&t);
    }
    const __half2 t = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&t);
}

__device__ __forceinline__ void store8(void* __restrict__ base, int dtype, int64_t at, int valid, bool vec, const float (&v)[8]) {
    if (valid <= 0) return;
    if (dtype == MPS_F32) {
        float* p = static_cast<float*>(base) + at;
        if (vec && valid >= 8) {
            *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) if (i < valid) p[i] = v[i];
        }
        return;
    }
    uint16_t* p = static_cast<uint16_t*>(base) + at;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack2(v[2 * i], v[2 * i + 1], dtype);
    if (vec && valid >= 8) {
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) if (i < valid) p[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
    }
}

// A warp's 256 neighbouring values, eight a lane, into a row that begins anywhere: by way of 1 KB of shared memory, so that neighbouring
// lanes store neighbouring elements.  (Stored by the lanes that hold them, every instruction would touch 32 pieces: 2047 x 1337 FP32 took 14 us
// that way.)  All 32 lanes take part; elements from `valid` on, counted from the warp's first, are not stored.
__device__ __forceinline__ void store_span(void* __restrict__ base, int dtype, int64_t at, int valid, float* __restrict__ buffer, int lane, const float (&v)[8]) {
    __syncwarp();
    reinterpret_cast<float4*>(buffer)[2 * lane] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(buffer)[2 * lane + 1] = make_float4(v[4], v[5], v[6], v[7]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int e = i * 32 + lane;
        if (e >= valid) break;
        if (dtype == MPS_F32) static_cast<float*>(base)[at + e] = buffer[e];
        else static_cast<uint16_t*>(base)[at + e] = (uint16_t)pack2(buffer[e], 0.f, dtype);
    }
}

// And the other way: a warp's 256 neighbouring values of a row that begins anywhere, every 32nd a lane as they are loaded; then, as values, eight
// neighbouring ones a lane.
__device__ __forceinline__ void load_spread(const void* __restrict__ base, int dtype, int64_t at, int valid, int lane, uint32_t (&w)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int e = i * 32 + lane;
        w[i] = 0u;
        if (e < valid) w[i] = dtype == MPS_F32 ? static_cast<const uint32_t*>(base)[at + e] : (uint32_t)static_cast<const uint16_t*>(base)[at + e];
    }
}
__device__ __forceinline__ void gather_spread(const uint32_t (&w)[8], int dtype, float* __restrict__ buffer, int lane, float (&v)[8]) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i)
        buffer[i * 32 + lane] = dtype == MPS_F32 ? __uint_as_float(w[i]) : dtype == MPS_BF16 ? __uint_as_float(w[i] << 16)
                                                                                            : __half2float(__ushort_as_half((uint16_t)w[i]));
    __syncwarp();
    const float4 a = reinterpret_cast<const float4*>(buffer)[2 * lane], b = reinterpret_cast<const float4*>(buffer)[2 * lane + 1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

// ---- codes ------------------------------------------------------------------------------------------

// Scale byte of a block whose largest magnitude has these bits.  An exponent field of e stands for 2^(e - 127), so the byte of
// 2^(e - 127 - 2) is e - 2; subnormal maxima and zero (e = 0) get the least scale.
__device__ __forceinline__ uint32_t mx4_scale_byte(uint32_t max_bits) {
    const uint32_t e = max_bits >> 23;
    return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
// 1 / scale, always a normal number: 2^(127 - byte).  (The NaN scale gets 0 here: its codes are zeros.)
__device__ __forceinline__ float mx4_inverse_scale(uint32_t byte) { return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ float mx4_scale(uint32_t byte) {
    return byte == 255u ? __uint_as_float(0x7FFFFFFFu) : __uint_as_float(byte ? byte << 23 : 0x00400000u);
}

// Eight values, already divided by their scale, as eight codes, the first in the lowest bits.
__device__ __forceinline__ uint32_t mx4_codes8(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// The other way: eight codes as values without their scale.
__device__ __forceinline__ void mx4_values8(uint32_t codes, float (&v)[8]) {
    uint32_t h[4];
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(codes));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

// The largest of eight magnitudes, as bits; NaN where there is one.
__device__ __forceinline__ float max_abs3(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ uint32_t max_bits8(const float (&v)[8]) {
    return __float_as_uint(max_abs3(max_abs3(max_abs3(v[0], v[1], v[2]), v[3], v[4]), max_abs3(v[5], v[6], v[7]), 0.f)) & 0x7FFFFFFFu;
}

// Two FP32 values at a time.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(r)) : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<uint64_t&>(r))
        : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)), "l"(reinterpret_cast<const uint64_t&>(c)));
    return r;
}
struct Pairs {       // eight values
    float2 p[4];
    __device__ __forceinline__ float (&each())[8] { return reinterpret_cast<float(&)[8]>(p); }
};
__device__ __forceinline__ Pairs times(const Pairs& a, const Pairs& b) {
    Pairs r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.p[i] = mul2(a.p[i], b.p[i]);
    return r;
}
__device__ __forceinline__ Pairs times(const Pairs& a, float b) {
    Pairs r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.p[i] = mul2(a.p[i], make_float2(b, b));
    return r;
}

// A warp quantises and stores one row of a tile: lane l holds columns 8 l to 8 l + 7 (zeros beyond the matrix), `m` the bits of the largest of
// its magnitudes.  Four lanes share a block; 128 bytes of codes go out in one piece.  All 32 lanes take part.
__device__ __forceinline__ void mx4_store_row(uint8_t* __restrict__ tile, int row, int lane, const float (&v)[8], uint32_t m) {
    m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
    m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
    const uint32_t byte = mx4_scale_byte(m);
    const float inverse = mx4_inverse_scale(byte);
    Pairs q = times(reinterpret_cast<const Pairs&>(v), inverse);      // of a NaN block, whatever it gives: its codes say nothing
    *reinterpret_cast<uint32_t*>(tile + mx4_code_offset(row, lane >> 2) + (lane & 3) * 4) = mx4_codes8(q.each());
    if ((lane & 3) == 0) tile[mx4_scale_offset(row, lane >> 4) + ((lane >> 2) & 3)] = (uint8_t)byte;
}
__device__ __forceinline__ void mx4_store_row(uint8_t* __restrict__ tile, int row, int lane, const float (&v)[8]) {
    mx4_store_row(tile, row, lane, v, max_bits8(v));
}

// The kernels of these operators may be launched while the kernel before them in the stream ends.  A kernel waits for that one before it reads what
// others write and before it writes anything, and only then lets the next begin: so whatever begins early can rely on all but
// the kernel right before it being done.
__device__ __forceinline__ void griddep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void griddep_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

inline bool mx4_dtype_ok(int dtype) { return dtype == MPS_BF16 || dtype == MPS_F16 || dtype == MPS_F32; }
inline int64_t mx4_dtype_bytes(int dtype) { return dtype == MPS_F32 ? 4 : 2; }
inline bool mx4_vec_ok(const void* p, int64_t row_stride, int dtype) {
    const int64_t bytes = 8 * mx4_dtype_bytes(dtype);
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && row_stride % 8 == 0;
}
// Row and column counts that every entry point accepts: tile counts and launch grids stay within 31 bits.
constexpr int64_t kMx4MostRows = int64_t(1) << 31, kMx4MostCols = int64_t(1) << 24;
// And the norms: a CTA a row, 512 threads x 8 steps x 8 columns.
constexpr int64_t kMx4MostNormRows = 0x7FFFFFFF, kMx4MostNormCols = 32768;

struct Device { int ordinal, sms; };
int current_device(Device& d);

// A launch that may overlap the end of the kernel before it.
template <typename... Params, typename... Args>
inline int launch_overlapping(const char* what, void (*kernel)(Params...), unsigned int ctas, dim3 threads, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(ctas);
    config.blockDim = threads;
    config.stream = st;
    cudaLaunchAttribute overlap;
    overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    overlap.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &overlap;
    config.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&config, kernel, args...);
    return e == cudaSuccess ? MPS_OK : cuda_fail(e, what);
}

}  // namespace mps
