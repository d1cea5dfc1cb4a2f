// The norms before and after a block, with the block's gate and the residual stream, in one pass.
//
//   t  = y * rsqrt(mean(y^2) + eps) * post_weight      (t = y without post_weight)
//   h' = residual_scale * h + gate * t                 (h' = h without y)
//   n  = h' * rsqrt(mean(h'^2) + eps) * next_weight    (in a 16-bit type, FP32, or quantised to MXFP4)
//
// A CTA has one row in registers (several short ones), eight neighbouring columns per lane and step, so that y and h are read once and the two
// means cost two barriers.  All arithmetic is in FP32; h' is normalised as it was before it is rounded to the stream's type.  Four lanes
// hold an MXFP4 block and a warp a whole row of a tile, so the quantised form needs nothing but shuffles.
// Bounds: memory, and for a few rows the two barriers and the launch.  Weights and gate are asked for before the barrier that they wait behind,
// not after it: each would add a trip to the L2 to every row.
#include "mx4.cuh"

namespace mps {

constexpr int kNormThreads = 256, kNormMostThreads = 512;
constexpr int64_t kNormManyRows = 512;

struct NormArgs {
    mps_mx4_norm a;
    float inv_cols;
    int groups;      // groups of eight columns, those that fill up the last tile included where n is quantised
    bool vec_y, vec_h, vec_post, vec_gate, vec_next, vec_h_out, vec_n;
};

// Eight neighbouring elements of a 16-bit type at a multiple of 16 bytes, or zeros.
static __device__ __forceinline__ Raw8 load_half8(const void* __restrict__ base, int64_t at, int valid) {
    Raw8 r;
    r.a = valid > 0 ? *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at) : make_uint4(0u, 0u, 0u, 0u);
    r.b = r.a;
    return r;
}

// Eight columns of an operand.  VEC: columns are a multiple of 8 and every row begins at a multiple of 16 bytes; else any row, `vec` telling whether
// this operand's do.  WIDE: FP32 (or, without VEC, whatever its dtype says).
template <bool VEC, bool WIDE>
struct Eight {
    uint32_t w[8];
    __device__ __forceinline__ void load(const void* __restrict__ base, int dtype, int64_t row, int column, int cols, bool vec, int lane) {
        const int valid = min(cols - column, 8);
        if (VEC || vec) {
            const Raw8 r = VEC && !WIDE ? load_half8(base, row + column, valid) : load_raw8(base, VEC ? MPS_F32 : dtype, row + column, VEC && valid > 0 ? 8 : valid, true);
            w[0] = r.a.x; w[1] = r.a.y; w[2] = r.a.z; w[3] = r.a.w;
            if (WIDE) { w[4] = r.b.x; w[5] = r.b.y; w[6] = r.b.z; w[7] = r.b.w; }
        } else {
            load_spread(base, dtype, row + column - lane * 8, cols - column + lane * 8, lane, w);
        }
    }
    // Once, before the first use: without VEC the words become the FP32 values of this lane's columns.
    __device__ __forceinline__ void settle(int dtype, bool vec, float* buffer, int lane) {
        if (VEC) return;
        float v[8];
        if (vec) {
            Raw8 r;
            r.a = make_uint4(w[0], w[1], w[2], w[3]);
            r.b = make_uint4(w[4], w[5], w[6], w[7]);
            unpack8(r, dtype, v);
        } else {
            gather_spread(w, dtype, buffer, lane, v);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[i]);
    }
    __device__ __forceinline__ void values(int dtype, Pairs& v) const {
        Raw8 r;
        r.a = make_uint4(w[0], w[1], w[2], w[3]);
        r.b = WIDE ? make_uint4(w[4], w[5], w[6], w[7]) : r.a;
        unpack8(r, WIDE ? MPS_F32 : dtype == MPS_BF16 ? MPS_BF16 : MPS_F16, v.each());
    }
};

// Sum over a row's threads (whole warps), the same in each of them.  `slot`, a word a warp, is not used by another sum without a barrier in between.
static __device__ __forceinline__ float row_sum(float v, float* slot) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31, first = threadIdx.y * warps;
    if (warps == 1) return v;
    if (lane == 0) slot[first + (threadIdx.x >> 5)] = v;
    __syncthreads();
    v = lane < warps ? slot[first + lane] : 0.f;
#pragma unroll
    for (int o = 8; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return __shfl_sync(0xFFFFFFFFu, v, 0);
}

// JOIN: there is a y.
template <int STEPS, bool VEC, bool JOIN, bool WIDE_Y, bool WIDE_H, bool WIDE_W>
__global__ void __launch_bounds__(kNormMostThreads)
mx4_norm_kernel(const NormArgs p) {
    __shared__ float slots[2][16];
    __shared__ __align__(16) float buffers[VEC ? 1 : kNormMostThreads / 32][256];
    constexpr bool kAhead = STEPS <= (JOIN ? 2 : 4);      // with more, the registers are for y and h
    griddep_wait();
    griddep_launch();
    const mps_mx4_norm& a = p.a;
    const int per_row = blockDim.x, place = threadIdx.x, warp = (threadIdx.y * blockDim.x + threadIdx.x) >> 5;
    float* buffer = buffers[VEC ? 0 : warp];
    const int lane = threadIdx.x & 31, cols = (int)a.cols;
    const int64_t own_row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    const bool live = own_row < a.rows;                    // whole warps; the last CTA may have rows too many, which repeat the last and store nothing
    const int64_t row = live ? own_row : a.rows - 1;
    const auto column = [&](int s) { return (s * per_row + place) * 8; };
    Eight<VEC, WIDE_Y> ry[STEPS];
    Eight<VEC, WIDE_H> rh[STEPS];
    Eight<VEC, WIDE_W> post[STEPS], gate[STEPS], next[STEPS];
    const auto load_post = [&](int s) { if (JOIN && a.post_weight) post[s].load(a.post_weight, a.weight_dtype, 0, column(s), cols, p.vec_post, lane); };
    const auto load_gate = [&](int s) {
        if (JOIN && a.gate && a.gate_col_stride) gate[s].load(a.gate, a.gate_dtype, row * a.gate_row_stride, column(s), cols, p.vec_gate, lane);
    };
    const auto load_next = [&](int s) { if (a.next_weight) next[s].load(a.next_weight, a.weight_dtype, 0, column(s), cols, p.vec_next, lane); };
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        if (JOIN) ry[s].load(a.y, a.y_dtype, row * a.y_stride, column(s), cols, p.vec_y, lane);
        rh[s].load(a.h, a.h_dtype, row * a.h_stride, column(s), cols, p.vec_h, lane);
    }
    if (kAhead) {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            load_post(s);
            load_gate(s);
            if (!JOIN) load_next(s);
        }
    }
    if (!VEC) {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            if (JOIN) ry[s].settle(a.y_dtype, p.vec_y, buffer, lane);
            rh[s].settle(a.h_dtype, p.vec_h, buffer, lane);
        }
    }
    // Columns beyond the last are zeros all through.
    Pairs v[STEPS];
    float2 sum = make_float2(0.f, 0.f);
    if (JOIN) {
        float row_gate = 1.f;      // one gate for the row
        if (a.gate && !a.gate_col_stride) {
            float w[8];
            unpack8(load_raw8(a.gate, a.gate_dtype, row * a.gate_row_stride, 1, false), a.gate_dtype, w);
            row_gate = w[0];
        }
        float r = 1.f;
        if (a.post_weight) {
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                Pairs y;
                ry[s].values(a.y_dtype, y);
#pragma unroll
                for (int i = 0; i < 4; ++i) sum = fma2(y.p[i], y.p[i], sum);
            }
            r = rsqrtf(fmaf(row_sum(sum.x + sum.y, slots[0]), p.inv_cols, a.eps));
        }
        sum = make_float2(0.f, 0.f);
        const float scale = r * row_gate;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            Pairs y, h, w;
            ry[s].values(a.y_dtype, y);
            rh[s].values(a.h_dtype, h);
            if (a.post_weight) {
                if (!kAhead) load_post(s);
                post[s].settle(a.weight_dtype, p.vec_post, buffer, lane);
                post[s].values(a.weight_dtype, w);
                y = times(y, times(w, scale));
            } else {
                y = times(y, scale);
            }
            if (a.gate && a.gate_col_stride) {
                if (!kAhead) load_gate(s);
                gate[s].settle(a.gate_dtype, p.vec_gate, buffer, lane);
                gate[s].values(a.gate_dtype, w);
                y = times(y, w);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[s].p[i] = fma2(make_float2(a.residual_scale, a.residual_scale), h.p[i], y.p[i]);
                sum = fma2(v[s].p[i], v[s].p[i], sum);
            }
            if (!live) continue;
            if (VEC || p.vec_h_out) {
                store8(a.h_out, a.h_dtype, row * a.h_out_stride + column(s), cols - column(s), true, v[s].each());
            } else {
                const int first = column(s) - lane * 8;      // the warp's
                store_span(a.h_out, a.h_dtype, row * a.h_out_stride + first, cols - first, buffer, lane, v[s].each());
            }
        }
        if (!a.n_out) return;
        if (kAhead) {      // on their way during the second sum
#pragma unroll
            for (int s = 0; s < STEPS; ++s) load_next(s);
        }
    } else {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            rh[s].values(a.h_dtype, v[s]);
#pragma unroll
            for (int i = 0; i < 4; ++i) sum = fma2(v[s].p[i], v[s].p[i], sum);
        }
    }
    const float r = rsqrtf(fmaf(row_sum(sum.x + sum.y, slots[1]), p.inv_cols, a.eps));
    if (!live) return;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int g = s * per_row + place;
        if ((g & ~31) >= p.groups) break;     // whole warps: a tile's row is one warp's
        Pairs w;
        if (!kAhead) load_next(s);
        next[s].settle(a.weight_dtype, p.vec_next, buffer, lane);
        next[s].values(a.weight_dtype, w);
        w = times(times(v[s], r), w);
        if (a.n_dtype == MPS_MX4) {
            const int chunks = (int)mx4_chunks(cols);
            mx4_store_row(static_cast<uint8_t*>(a.n_out) + mx4_tile_offset(row / kMx4Rows, g >> 5, chunks), (int)(row % kMx4Rows), lane, w.each());
        } else if (VEC || p.vec_n) {
            store8(a.n_out, a.n_dtype, row * a.n_stride + g * 8, cols - g * 8, true, w.each());
        } else {
            const int first = (g - lane) * 8;
            store_span(a.n_out, a.n_dtype, row * a.n_stride + first, cols - first, buffer, lane, w.each());
        }
    }
}

template <int STEPS>
static int launch_norm(const NormArgs& p, bool vec, bool wide_w, int per_row, cudaStream_t st) {
    const mps_mx4_norm& a = p.a;
    // short rows share a CTA
    const int rows_per_cta = per_row >= kNormThreads ? 1 : kNormThreads / per_row;
    const bool wide_y = a.y && a.y_dtype == MPS_F32, wide_h = a.h_dtype == MPS_F32;
    void (*kernel)(NormArgs) = a.y ? mx4_norm_kernel<STEPS, false, true, true, true, true> : mx4_norm_kernel<STEPS, false, false, true, true, true>;
    if (vec && a.y) {
        static void (*const fast[8])(NormArgs) = {
            mx4_norm_kernel<STEPS, true, true, false, false, false>, mx4_norm_kernel<STEPS, true, true, false, false, true>,
            mx4_norm_kernel<STEPS, true, true, false, true, false>,  mx4_norm_kernel<STEPS, true, true, false, true, true>,
            mx4_norm_kernel<STEPS, true, true, true, false, false>,  mx4_norm_kernel<STEPS, true, true, true, false, true>,
            mx4_norm_kernel<STEPS, true, true, true, true, false>,   mx4_norm_kernel<STEPS, true, true, true, true, true>};
        kernel = fast[wide_y * 4 + wide_h * 2 + wide_w];
    } else if (vec) {
        static void (*const fast[4])(NormArgs) = {
            mx4_norm_kernel<STEPS, true, false, false, false, false>, mx4_norm_kernel<STEPS, true, false, false, false, true>,
            mx4_norm_kernel<STEPS, true, false, false, true, false>,  mx4_norm_kernel<STEPS, true, false, false, true, true>};
        kernel = fast[wide_h * 2 + wide_w];
    }
    return launch_overlapping("mx4_norm_kernel", kernel, (unsigned int)((a.rows + rows_per_cta - 1) / rows_per_cta), dim3(per_row, rows_per_cta), st, p);
}

}  // namespace mps

using namespace mps;

extern "C" int mps_mx4_norm_rows(const mps_mx4_norm* args, void* stream) {
    if (!args) { set_error("mps_mx4_norm_rows: null arguments"); return MPS_ERR_INVALID; }
    NormArgs p;
    p.a = *args;
    const mps_mx4_norm& a = p.a;
    if (a.rows < 0 || a.rows > kMx4MostNormRows || a.cols <= 0 || a.cols > kMx4MostNormCols) {
        set_error("mps_mx4_norm_rows: rows must be below 2^31, cols in [1, %d]", (int)kMx4MostNormCols);
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
    // the weights, and a gate that has columns, share a width in the kernels for aligned rows; FP32 weights beside a 16-bit gate, or the reverse, go the way of
    // unaligned ones (8191 x 4096 BF16 111 and 118 us, of one width 62 and 63): as many kernels again would serve a mixture that a caller can avoid
    const bool column_gate = a.y && a.gate && a.gate_col_stride, weights = a.next_weight || (a.y && a.post_weight);
    const bool wide_w = weights ? a.weight_dtype == MPS_F32 : column_gate && a.gate_dtype == MPS_F32;
    const bool vec = a.cols % 8 == 0 && p.vec_h && (!a.y || (p.vec_y && p.vec_h_out)) && (!a.n_out || a.n_dtype == MPS_MX4 || p.vec_n) &&
                     (!a.y || !a.post_weight || p.vec_post) && (!a.next_weight || p.vec_next) &&
                     (!column_gate || (p.vec_gate && (a.gate_dtype == MPS_F32) == wide_w));
    // 256 threads for a row where there are many rows (8191 x 4096 beside FP32: 64 us, with 512 75 us), without a y 128 (8191 x 4096 FP32, quantised: 27 us,
    // with 256 30 us), 512 where a few wait for their own length (64 x 4096: 2.4 us, with 256 2.7 us) or where 256 would hold 32 columns each and more
    // (2048 x 14336: 50 us, with 256 73 us), one warp for short rows (20000 x 512: 17 us, with 64 threads 19 us)
    const int many = a.y || p.groups > 512 ? kNormThreads : kNormThreads / 2;
    const int most = a.rows < kNormManyRows ? kNormMostThreads : p.groups <= 64 ? 32 : p.groups <= 4 * kNormThreads ? many : kNormMostThreads;
    int steps = 1;
    while ((p.groups + steps - 1) / steps > most) steps *= 2;
    const int per_row = ((p.groups + steps - 1) / steps + 31) / 32 * 32;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (steps) {
        case 1: return launch_norm<1>(p, vec, wide_w, per_row, st);
        case 2: return launch_norm<2>(p, vec, wide_w, per_row, st);
        case 4: return launch_norm<4>(p, vec, wide_w, per_row, st);
        default: return launch_norm<8>(p, vec, wide_w, per_row, st);
    }
}
