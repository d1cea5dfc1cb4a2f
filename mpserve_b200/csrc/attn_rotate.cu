// Norms of queries and keys for each head with the position rotation, and the way of a step's keys and values into the paged cache, in one pass.
//
//   y = x * rsqrt(mean(x^2) + eps) * weight                     (y = x without weight), over a head's `dim` values
//   (y_a, y_b) -> scale * (y_a cos u - y_b sin u, y_b cos u + y_a sin u)    for each pair j of the first `rotated` values, u = position[axis_j] f_j
//
// A pair is (j, j + rotated / 2), or neighbours (2 j, 2 j + 1).  An angle of a far position has more revolutions than FP32 has digits: position times
// frequency, in revolutions, is an FP64 product, whose whole part is dropped in FP64; what is left is below half a revolution and its sine and cosine
// are FP32's.  All other arithmetic is FP32, rounded once to the output's type.
//
// A CTA has one token: its first threads make the token's cosines and sines, once for all heads, while every thread's share of the heads is on its way; a
// share is eight neighbouring values, so that four to 32 lanes have a head, and neighbours' halves of a pair change lanes by shuffles.  Bounds: memory,
// for a few tokens the launch.
#include <initializer_list>

#include "mx4.cuh"

namespace mps {

constexpr int kHeadMostDim = 256;

struct RotateArgs {
    mps_head_rotate a;
    float inv_dim;
    int page_shift;
    int64_t slots;       // of the cache
};

struct HeadPlace {
    const void* in;
    void* out;           // null: nowhere
    int64_t in_at, out_at;
    const void* weight;
    bool turned;         // not a value
};

// Head h of a token, queries first, then keys, then values.
__device__ __forceinline__ HeadPlace head_place(const RotateArgs& p, int64_t token, int h, int64_t page, int64_t offset) {
    const mps_head_rotate& a = p.a;
    HeadPlace r;
    r.turned = true;
    if (h < a.q_heads) {
        r.in = a.q; r.in_at = token * a.q_token_stride + (int64_t)h * a.q_head_stride;
        r.out = a.q_out; r.out_at = (token * a.q_heads + h) * a.dim;
        r.weight = a.q_weight;
        return r;
    }
    h -= a.q_heads;
    const bool key = h < a.kv_heads;
    if (!key) h -= a.kv_heads;
    r.turned = key;
    r.weight = key ? a.k_weight : nullptr;
    r.in = key ? a.k : a.v;
    r.in_at = key ? token * a.k_token_stride + (int64_t)h * a.k_head_stride : token * a.v_token_stride + (int64_t)h * a.v_head_stride;
    if (!a.slots) {
        r.out = a.k_out; r.out_at = (token * a.kv_heads + h) * a.dim;
    } else {
        r.out = page < 0 ? nullptr : key ? a.k_out : a.v_out;
        r.out_at = key ? page * a.k_page_stride + offset * a.k_slot_stride + (int64_t)h * a.k_cache_head_stride
                       : page * a.v_page_stride + offset * a.v_slot_stride + (int64_t)h * a.v_cache_head_stride;
    }
    return r;
}

// The token's cosines and sines, times the rotation's scale, by the CTA's threads.
__device__ __forceinline__ void token_angles(const RotateArgs& p, int64_t token, float* cosines, float* sines) {
    const mps_head_rotate& a = p.a;
    for (int j = threadIdx.x; j < a.rotated / 2; j += blockDim.x) {
        const int64_t at = (a.axis ? (int64_t)a.axis[j] * a.tokens : 0) + token;
        const double position = a.wide_positions ? (double)static_cast<const int64_t*>(a.positions)[at] : (double)static_cast<const int32_t*>(a.positions)[at];
        const double turns = position * a.turns[j];
        float s, c;
        sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
        cosines[j] = c * a.scale;
        sines[j] = s * a.scale;
    }
}

__device__ __forceinline__ void token_slot(const RotateArgs& p, int64_t token, int64_t& page, int64_t& offset) {
    page = -1;
    offset = 0;
    if (p.a.slots) {
        const int64_t slot = p.a.slots[token];
        if (slot >= 0 && slot < p.slots) {
            page = slot >> p.page_shift;
            offset = slot & ((int64_t(1) << p.page_shift) - 1);
        }
    }
}

// Rows of whole eights, aligned.  LANES (a power of two) have a head; STEPS heads a thread; WIDE: FP32.
template <int LANES, int STEPS, bool WIDE>
__global__ void __launch_bounds__(STEPS == 1 ? 1024 : 512) rotate_kernel(const RotateArgs p) {
    __shared__ __align__(16) float cosines[kHeadMostDim / 2], sines[kHeadMostDim / 2];
    griddep_wait();
    griddep_launch();
    const mps_head_rotate& a = p.a;
    const int64_t token = blockIdx.x;
    const int u = threadIdx.x % LANES, units = a.dim / 8, per_pass = blockDim.x / LANES, heads = a.q_heads + (a.v ? 2 : 1) * a.kv_heads;
    const uint32_t mates = LANES == 32 ? 0xFFFFFFFFu : ((1u << (LANES & 31)) - 1u) << (threadIdx.x & 31 & ~(LANES - 1));      // the lanes of a head
    const int dtype = WIDE ? MPS_F32 : a.dtype == MPS_BF16 ? MPS_BF16 : MPS_F16;
    int64_t page, offset;
    token_slot(p, token, page, offset);
    const auto valid = [&](int h) { return h < heads && u < units ? 8 : 0; };
    const auto gain = [&](int h) {
        const void* weight = h < a.q_heads ? a.q_weight : h < a.q_heads + a.kv_heads ? a.k_weight : nullptr;
        return load_raw8(weight, a.weight_dtype, u * 8, weight ? valid(h) : 0, true);
    };
    uint4 raw[STEPS][WIDE ? 2 : 1];
    Raw8 first_gain;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int h = s * per_pass + threadIdx.x / LANES;
        const HeadPlace place = head_place(p, token, min(h, heads - 1), page, offset);
        const Raw8 r = load_raw8(place.in, WIDE ? MPS_F32 : MPS_BF16, place.in_at + u * 8, valid(h), true);
        raw[s][0] = r.a;
        if (WIDE) raw[s][WIDE ? 1 : 0] = r.b;
        if (s == 0) first_gain = gain(h);
    }
    token_angles(p, token, cosines, sines);
    __syncthreads();
    // this lane's pairs: those of a unit of the first halves, or (half as many) of neighbours
    const int half = a.rotated / 16, place_of = a.interleaved ? u * 4 : (u < half ? u : u - half) * 8;
    const int partner = u < half ? u + half : u - half;
    const bool turned = u * 8 < a.rotated;
    float c[8], s8[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int at = turned ? place_of + (a.interleaved ? i >> 1 : i) : 0;
        c[i] = cosines[at];
        s8[i] = sines[at];
        if (a.interleaved ? !(i & 1) : u < half) s8[i] = -s8[i];
    }
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int h = s * per_pass + threadIdx.x / LANES;      // the same for the lanes of a head
        if (h >= heads) break;
        float v[8];
        Raw8 r;
        r.a = raw[s][0];
        r.b = raw[s][WIDE ? 1 : 0];
        unpack8(r, dtype, v);
        const HeadPlace place = head_place(p, token, h, page, offset);
        if (place.weight) {
            float w[8], sum = 0.f;
            unpack8(s == 0 ? first_gain : gain(h), a.weight_dtype, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fmaf(v[i], v[i], sum);
#pragma unroll
            for (int o = LANES / 2; o; o >>= 1) sum += __shfl_xor_sync(mates, sum, o);
            const float rms = rsqrtf(fmaf(sum, p.inv_dim, a.eps));
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = v[i] * rms * w[i];
        }
        if (place.turned) {
            float other[8];
            if (a.interleaved) {
#pragma unroll
                for (int i = 0; i < 8; ++i) other[i] = v[i ^ 1];
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) other[i] = __shfl_sync(mates, v[i], partner, LANES);
            }
            if (turned) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = fmaf(other[i], s8[i], v[i] * c[i]);
            }
        }
        if (place.out) store8(place.out, dtype, place.out_at + u * 8, valid(h), true, v);
    }
}

// Any dim, any alignment: a warp has a head, value by value, by way of shared memory.
constexpr int kRotateAnyWarps = 8;
__global__ void __launch_bounds__(kRotateAnyWarps * 32) rotate_any_kernel(const RotateArgs p) {
    __shared__ float cosines[kHeadMostDim / 2], sines[kHeadMostDim / 2], values[kRotateAnyWarps][kHeadMostDim];
    griddep_wait();
    griddep_launch();
    const mps_head_rotate& a = p.a;
    const int64_t token = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, heads = a.q_heads + (a.v ? 2 : 1) * a.kv_heads, pairs = a.rotated / 2;
    int64_t page, offset;
    token_slot(p, token, page, offset);
    token_angles(p, token, cosines, sines);
    __syncthreads();
    for (int h = warp; h < heads; h += kRotateAnyWarps) {
        const HeadPlace place = head_place(p, token, h, page, offset);
        if (!place.out) continue;
        float sum = 0.f, r = 1.f;
        for (int i = lane; i < a.dim; i += 32) {
            float v[8];
            unpack8(load_raw8(place.in, a.dtype, place.in_at + i, 1, false), a.dtype, v);
            values[warp][i] = v[0];
            sum = fmaf(v[0], v[0], sum);
        }
        if (place.weight) {
#pragma unroll
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
            r = rsqrtf(fmaf(sum, p.inv_dim, a.eps));
            for (int i = lane; i < a.dim; i += 32) {
                float w[8];
                unpack8(load_raw8(place.weight, a.weight_dtype, i, 1, false), a.weight_dtype, w);
                values[warp][i] = values[warp][i] * r * w[0];
            }
        }
        __syncwarp();
        for (int i = lane; i < a.dim; i += 32) {
            float v[8] = {values[warp][i]};
            if (place.turned && i < a.rotated) {
                const int j = a.interleaved ? i >> 1 : i < pairs ? i : i - pairs;
                const bool first = a.interleaved ? !(i & 1) : i < pairs;
                const float other = values[warp][a.interleaved ? i ^ 1 : first ? i + pairs : j];
                v[0] = fmaf(first ? -other : other, sines[j], v[0] * cosines[j]);
            }
            store8(place.out, a.dtype, place.out_at + i, 1, false, v);
        }
        __syncwarp();
    }
}

template <int LANES>
static int launch_rotate(const RotateArgs& p, cudaStream_t st) {
    const int heads = p.a.q_heads + (p.a.v ? 2 : 1) * p.a.kv_heads;
    // few tokens: every head at once; many: 256 threads, which leave the SM room for other tokens
    const int all = (heads * LANES + 31) / 32 * 32, most = p.a.tokens <= 148 ? 1024 : 256;
    int steps = 1;
    while (steps < 4 && (all + steps - 1) / steps > most) ++steps;
    const int threads = ((heads + steps - 1) / steps * LANES + 31) / 32 * 32;
    if (threads > (steps == 1 ? 1024 : 512)) return launch_overlapping("rotate_any_kernel", rotate_any_kernel, (unsigned int)p.a.tokens, dim3(kRotateAnyWarps * 32), st, p);
    const unsigned int ctas = (unsigned int)p.a.tokens;
    if (p.a.dtype == MPS_F32) {
        static void (*const kernels[4])(RotateArgs) = {rotate_kernel<LANES, 1, true>, rotate_kernel<LANES, 2, true>, rotate_kernel<LANES, 3, true>,
                                                       rotate_kernel<LANES, 4, true>};
        return launch_overlapping("rotate_kernel", kernels[steps - 1], ctas, dim3(threads), st, p);
    }
    static void (*const kernels[4])(RotateArgs) = {rotate_kernel<LANES, 1, false>, rotate_kernel<LANES, 2, false>, rotate_kernel<LANES, 3, false>,
                                                   rotate_kernel<LANES, 4, false>};
    return launch_overlapping("rotate_kernel", kernels[steps - 1], ctas, dim3(threads), st, p);
}

}  // namespace mps

using namespace mps;

extern "C" int mps_head_rotate_rows(const mps_head_rotate* args, void* stream) {
    if (!args) { set_error("mps_head_rotate_rows: null arguments"); return MPS_ERR_INVALID; }
    RotateArgs p;
    p.a = *args;
    const mps_head_rotate& a = p.a;
    if (a.tokens < 0 || a.tokens > 0x7FFFFFFF || a.q_heads < 0 || a.kv_heads < 0 || a.q_heads > MPS_MOST_HEADS || a.kv_heads > MPS_MOST_HEADS ||
        a.q_heads + a.kv_heads == 0) {
        set_error("mps_head_rotate_rows: tokens must be below 2^31, heads at most %d", (int)MPS_MOST_HEADS);
        return MPS_ERR_INVALID;
    }
    if (a.dim <= 0 || a.dim > kHeadMostDim || a.rotated < 0 || a.rotated > a.dim || (a.rotated & 1)) {
        set_error("mps_head_rotate_rows: dim must be in [1, %d], rotated even and at most dim", kHeadMostDim);
        return MPS_ERR_INVALID;
    }
    if (!mx4_dtype_ok(a.dtype) || ((a.q_weight || a.k_weight) && !mx4_dtype_ok(a.weight_dtype))) { set_error("mps_head_rotate_rows: unknown dtype"); return MPS_ERR_INVALID; }
    if (a.tokens == 0) return MPS_OK;
    const bool append = a.slots != nullptr;
    if ((a.q_heads && (!a.q || !a.q_out)) || (a.kv_heads && (!a.k || !a.k_out)) || (append && a.kv_heads && (!a.v || !a.v_out)) || (!append && a.v) ||
        (a.rotated && (!a.positions || !a.turns))) {
        set_error("mps_head_rotate_rows: missing pointer");
        return MPS_ERR_INVALID;
    }
    if (append && (a.pages < 0 || a.page_size <= 0 || (a.page_size & (a.page_size - 1)))) {
        set_error("mps_head_rotate_rows: the size of a page must be a power of two");
        return MPS_ERR_INVALID;
    }
    p.inv_dim = (float)(1.0 / (double)a.dim);
    p.page_shift = append ? __builtin_ctzll((unsigned long long)a.page_size) : 0;
    p.slots = append ? a.pages * a.page_size : 0;
    // every head begins at a multiple of eight values, by pointer and strides
    const int64_t unit = 8 * mx4_dtype_bytes(a.dtype);
    const auto even = [&](const void* q, std::initializer_list<int64_t> strides) {
        bool ok = reinterpret_cast<uintptr_t>(q) % unit == 0;
        for (const int64_t s : strides) ok = ok && s % 8 == 0;
        return ok;
    };
    const auto weight_even = [&](const void* q) { return reinterpret_cast<uintptr_t>(q) % (8 * mx4_dtype_bytes(a.weight_dtype)) == 0; };
    const bool vec = a.dim % 8 == 0 && a.rotated % (a.interleaved ? 8 : 16) == 0 && even(a.q, {a.q_token_stride, a.q_head_stride}) &&
                     even(a.k, {a.k_token_stride, a.k_head_stride}) && even(a.q_out, {}) && weight_even(a.q_weight) && weight_even(a.k_weight) &&
                     (append ? even(a.v, {a.v_token_stride, a.v_head_stride}) && even(a.k_out, {a.k_page_stride, a.k_slot_stride, a.k_cache_head_stride}) &&
                                   even(a.v_out, {a.v_page_stride, a.v_slot_stride, a.v_cache_head_stride})
                             : even(a.k_out, {}));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!vec) return launch_overlapping("rotate_any_kernel", rotate_any_kernel, (unsigned int)a.tokens, dim3(kRotateAnyWarps * 32), st, p);
    if (a.dim <= 32) return launch_rotate<4>(p, st);
    if (a.dim <= 64) return launch_rotate<8>(p, st);
    if (a.dim <= 128) return launch_rotate<16>(p, st);
    return launch_rotate<32>(p, st);
}
