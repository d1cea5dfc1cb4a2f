// The norms before and after a block, with the block's gate and the residual stream, in one pass.
//
//   t  = y * rsqrt(mean(y^2) + eps) * post_weight      (t = y without post_weight)
//   h' = residual_scale * h + gate * t                 (h' = h without y)
//   n  = h' * rsqrt(mean(h'^2) + eps) * next_weight    (in a 16-bit type, FP32, or quantised to MXFP4)
//
// One CTA has one row in registers, eight neighbouring columns per lane and step, so that y and h are read once and the two means
// cost two barriers.  All arithmetic is in FP32; h' is normalised as it was before it is rounded to the stream's type.  Four lanes
// hold an MXFP4 block and a warp a whole row of a tile, so the quantised form needs nothing but shuffles.
// Bounds: memory, and for a few rows the two barriers and the launch.
#include "mx4.cuh"

namespace mps {

constexpr int kNormMostThreads = 512;
constexpr int kNormMostCols = 32768;    // 512 threads x 8 steps x 8 columns

struct NormArgs {
    mps_mx4_norm a;
    float inv_cols;
    int groups;      // groups of eight columns, those that fill up the last tile included where n is quantised
    bool vec_y, vec_h, vec_post, vec_gate, vec_next, vec_h_out, vec_n;
};

// Sum over the CTA, the same in every thread.  `slot` is not used by another sum without a barrier in between.
static __device__ __forceinline__ float row_sum(float v, float* slot) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (warps == 1) return v;
    if (lane == 0) slot[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < warps ? slot[lane] : 0.f;
#pragma unroll
    for (int o = 8; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return __shfl_sync(0xFFFFFFFFu, v, 0);
}

template <int STEPS>
__global__ void __launch_bounds__(kNormMostThreads)
mx4_norm_kernel(const NormArgs p) {
    __shared__ float slots[2][16];
    __shared__ __align__(16) float buffers[kNormMostThreads / 32][256];
    float* buffer = buffers[threadIdx.x >> 5];
    const int lane = threadIdx.x & 31;
    griddep_wait();
    griddep_launch();
    const mps_mx4_norm& a = p.a;
    const int64_t row = blockIdx.x;
    const int cols = (int)a.cols;
    Raw8 ry[STEPS], rh[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int c = (s * blockDim.x + threadIdx.x) * 8, valid = min(cols - c, 8);
        if (a.y) ry[s] = load_raw8(a.y, a.y_dtype, row * a.y_stride + c, valid, p.vec_y);
        rh[s] = load_raw8(a.h, a.h_dtype, row * a.h_stride + c, valid, p.vec_h);
    }
    float v[STEPS][8];
    float sum = 0.f;
    if (a.y) {
        float r = 1.f;
        if (a.post_weight) {
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                float y[8];
                unpack8(ry[s], a.y_dtype, y);
#pragma unroll
                for (int i = 0; i < 8; ++i) sum = fmaf(y[i], y[i], sum);
            }
            r = 1.f / sqrtf(fmaf(row_sum(sum, slots[0]), p.inv_cols, a.eps));
        }
        sum = 0.f;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int c = (s * blockDim.x + threadIdx.x) * 8, valid = min(cols - c, 8), span = c - lane * 8;    // the warp's first
            float y[8], h[8], w[8];
            unpack8(ry[s], a.y_dtype, y);
            unpack8(rh[s], a.h_dtype, h);
            if (a.post_weight) {
                unpack8(load_raw8(a.post_weight, a.weight_dtype, c, valid, p.vec_post), a.weight_dtype, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] *= r * w[i];
            }
            if (a.gate) {
                if (a.gate_col_stride) {
                    unpack8(load_raw8(a.gate, a.gate_dtype, row * a.gate_row_stride + c, valid, p.vec_gate), a.gate_dtype, w);
                } else {
                    unpack8(load_raw8(a.gate, a.gate_dtype, row * a.gate_row_stride, 1, false), a.gate_dtype, w);
#pragma unroll
                    for (int i = 1; i < 8; ++i) w[i] = w[0];
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] *= w[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[s][i] = i < valid ? fmaf(a.residual_scale, h[i], y[i]) : 0.f;
                sum = fmaf(v[s][i], v[s][i], sum);
            }
            if (p.vec_h_out) store8(a.h_out, a.h_dtype, row * a.h_out_stride + c, valid, true, v[s]);
            else store_span(a.h_out, a.h_dtype, row * a.h_out_stride + span, cols - span, buffer, lane, v[s]);
        }
        if (!a.n_out) return;
    } else {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            unpack8(rh[s], a.h_dtype, v[s]);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fmaf(v[s][i], v[s][i], sum);
        }
    }
    const float r = 1.f / sqrtf(fmaf(row_sum(sum, slots[1]), p.inv_cols, a.eps));
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int g = s * blockDim.x + threadIdx.x, c = g * 8, valid = min(cols - c, 8), span = c - lane * 8;
        if ((g & ~31) >= p.groups) break;     // whole warps: a tile's row is one warp's
        float w[8];
        unpack8(load_raw8(a.next_weight, a.weight_dtype, c, valid, p.vec_next), a.weight_dtype, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = i < valid ? v[s][i] * r * w[i] : 0.f;
        if (a.n_dtype == MPS_MX4) {
            const int chunks = (int)mx4_chunks(cols);
            mx4_store_row(static_cast<uint8_t*>(a.n_out) + mx4_tile_offset(row / kMx4Rows, c / kMx4Cols, chunks),
                          (int)(row % kMx4Rows), lane, w);
        } else {
            if (p.vec_n) store8(a.n_out, a.n_dtype, row * a.n_stride + c, valid, true, w);
            else store_span(a.n_out, a.n_dtype, row * a.n_stride + span, cols - span, buffer, lane, w);
        }
    }
}

}  // namespace mps

using namespace mps;

extern "C" int mps_mx4_norm_rows(const mps_mx4_norm* args, void* stream) {
    if (!args) { set_error("mps_mx4_norm_rows: null arguments"); return MPS_ERR_INVALID; }
    NormArgs p;
    p.a = *args;
    const mps_mx4_norm& a = p.a;
    if (a.rows < 0 || a.rows > 0x7FFFFFFFLL || a.cols <= 0 || a.cols > kNormMostCols) {
        set_error("mps_mx4_norm_rows: rows must be below 2^31, cols in [1, %d]", kNormMostCols);
        return MPS_ERR_INVALID;
    }
    if (!mx4_dtype_ok(a.h_dtype) || (a.y && !mx4_dtype_ok(a.y_dtype)) || (a.gate && !mx4_dtype_ok(a.gate_dtype)) ||
        ((a.post_weight || a.next_weight) && !mx4_dtype_ok(a.weight_dtype)) || (a.n_out && a.n_dtype != MPS_MX4 && !mx4_dtype_ok(a.n_dtype))) {
        set_error("mps_mx4_norm_rows: unknown dtype");
        return MPS_ERR_INVALID;
    }
    if (a.rows == 0) return MPS_OK;
    if (!a.h || (a.y && !a.h_out) || (a.n_out != nullptr) != (a.next_weight != nullptr) || (!a.y && !a.n_out)) {
        set_error("mps_mx4_norm_rows: missing pointer");
        return MPS_ERR_INVALID;
    }
    if (a.n_out && a.n_dtype == MPS_MX4 && (reinterpret_cast<uintptr_t>(a.n_out) & 15u)) { set_error("mps_mx4_norm_rows: unaligned tiles"); return MPS_ERR_INVALID; }
    p.inv_cols = (float)(1.0 / (double)a.cols);
    p.groups = a.n_out && a.n_dtype == MPS_MX4 ? (int)mx4_chunks(a.cols) * 32 : (int)((a.cols + 7) / 8);
    p.vec_y = a.y && mx4_vec_ok(a.y, a.y_stride, a.y_dtype);
    p.vec_h = mx4_vec_ok(a.h, a.h_stride, a.h_dtype);
    p.vec_post = a.post_weight && mx4_vec_ok(a.post_weight, 0, a.weight_dtype);
    p.vec_next = a.next_weight && mx4_vec_ok(a.next_weight, 0, a.weight_dtype);
    p.vec_gate = a.gate && mx4_vec_ok(a.gate, a.gate_row_stride, a.gate_dtype);
    p.vec_h_out = a.h_out && mx4_vec_ok(a.h_out, a.h_out_stride, a.h_dtype);
    p.vec_n = a.n_out && a.n_dtype != MPS_MX4 && mx4_vec_ok(a.n_out, a.n_stride, a.n_dtype);
    int steps = 1;
    while ((p.groups + steps - 1) / steps > kNormMostThreads) steps *= 2;
    const int threads = ((p.groups + steps - 1) / steps + 31) / 32 * 32;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const unsigned int rows = (unsigned int)a.rows;
    switch (steps) {
        case 1: return launch_overlapping("mx4_norm_kernel", mx4_norm_kernel<1>, rows, threads, st, p);
        case 2: return launch_overlapping("mx4_norm_kernel", mx4_norm_kernel<2>, rows, threads, st, p);
        case 4: return launch_overlapping("mx4_norm_kernel", mx4_norm_kernel<4>, rows, threads, st, p);
        default: return launch_overlapping("mx4_norm_kernel", mx4_norm_kernel<8>, rows, threads, st, p);
    }
}
