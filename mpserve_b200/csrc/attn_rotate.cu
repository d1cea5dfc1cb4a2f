// Norms of queries and keys for each head with the position rotation, and the way of a step's keys and values into the paged cache, in one pass.
//
//   y = x * rsqrt(mean(x^2) + eps) * weight                     (y = x without weight), over a head's `dim` values
//   (y_a, y_b) -> scale * (y_a cos u - y_b sin u, y_b cos u + y_a sin u)    for each pair j of the first `rotated` values, u = position[axis_j] f_j
//
// A pair is (j, j + rotated / 2), or neighbours (2 j, 2 j + 1).  An angle of a far position has more revolutions than FP32 has digits: position times
// frequency, in revolutions, is an FP64 product, whose whole part is dropped in FP64; what is left is below half a revolution and its sine and cosine
// are FP32's.  (The frequency in revolutions and the product are off by 2^-51 of the whole angle together.)  All other arithmetic is FP32, rounded once to the output's type.
//
// Eight values of a head are a lane's, four and the four that they are paired with, so that four to 32 lanes have a head and a pair never changes lanes.  With few
// tokens a CTA has one, all heads at once or, of 1024 to 2048 lanes, in three or four steps, and its first threads make the token's cosines and sines while the heads are
// on their way; with many a warp has one, makes them for itself and goes through the heads with four of them on their way, without a barrier.  Bounds: memory, for a few tokens the launch.
#include <initializer_list>

#include "mx4.cuh"

namespace mps {

constexpr int kHeadMostDim = 256;
// Up to six a SM a token has a CTA: 32 query and 8 key heads of 128 take 2.5 us for 148 tokens and 4.6 for 400, with a warp a token 5.5 and 7.4; 2048 tokens take 16.5 that
// way and 13.3 with a warp each.
constexpr int64_t kRotateFewTokens = 888;

struct RotateArgs {
    mps_head_rotate a;
    float inv_dim;
    int page_shift;
    int64_t slots;       // of the cache
};

struct HeadPlace {
    const void* in;
    void* out;           // null: nowhere
    int64_t in_at, out_at, out_stride;      // out_stride: of the next head of its kind
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
        r.out = a.q_out; r.out_at = (token * a.q_heads + h) * a.dim; r.out_stride = a.dim;
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
        r.out = a.k_out; r.out_at = (token * a.kv_heads + h) * a.dim; r.out_stride = a.dim;
    } else {
        r.out = page < 0 ? nullptr : key ? a.k_out : a.v_out;
        r.out_stride = key ? a.k_cache_head_stride : a.v_cache_head_stride;
        r.out_at = key ? page * a.k_page_stride + offset * a.k_slot_stride + (int64_t)h * a.k_cache_head_stride
                       : page * a.v_page_stride + offset * a.v_slot_stride + (int64_t)h * a.v_cache_head_stride;
    }
    return r;
}

// Cosine and sine of a token's pair j, times the rotation's scale.
__device__ __forceinline__ void pair_angle(const mps_head_rotate& a, int64_t token, int j, float& cosine, float& sine) {
    const int64_t at = (a.axis ? (int64_t)a.axis[j] * a.tokens : 0) + token;
    const double position = a.wide_positions ? (double)static_cast<const int64_t*>(a.positions)[at] : (double)static_cast<const int32_t*>(a.positions)[at];
    const double turns = position * a.turns[j];
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    cosine = c * a.scale;
    sine = s * a.scale;
}
// Those of all its pairs, by the CTA's threads.
__device__ __forceinline__ void token_angles(const RotateArgs& p, int64_t token, float* cosines, float* sines) {
    for (int j = threadIdx.x; j < p.a.rotated / 2; j += blockDim.x) pair_angle(p.a, token, j, cosines[j], sines[j]);
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

// Which eight values of a head are lane u's: a to a + 3 and b to b + 3; their pairs, where they are turned, are 4 u to 4 u + 3.
struct RotateLane {
    int a, b;
    bool live, turned;
    __device__ __forceinline__ RotateLane(const mps_head_rotate& r, int u) {
        live = u < r.dim / 8;
        turned = u < r.rotated / 8;
        const bool halves = turned && !r.interleaved;
        a = halves ? 4 * u : 8 * u;
        b = halves ? r.rotated / 2 + 4 * u : 8 * u + 4;
    }
};
template <bool WIDE>
struct RotateRaw {       // as they were loaded
    uint4 a, b;          // of a 16-bit type the first two words each
    __device__ __forceinline__ void load(const void* base, int64_t at, const RotateLane& l) {
        if (WIDE) {
            const float* p = static_cast<const float*>(base) + at;
            a = *reinterpret_cast<const uint4*>(p + l.a);
            b = *reinterpret_cast<const uint4*>(p + l.b);
        } else {
            const uint16_t* p = static_cast<const uint16_t*>(base) + at;
            const uint2 x = *reinterpret_cast<const uint2*>(p + l.a), y = *reinterpret_cast<const uint2*>(p + l.b);
            a.x = x.x; a.y = x.y; b.x = y.x; b.y = y.y;
        }
    }
    __device__ __forceinline__ void values(int dtype, Pairs& v) const {
        Raw8 r;
        r.a = WIDE ? a : make_uint4(a.x, a.y, b.x, b.y);
        r.b = WIDE ? b : r.a;
        unpack8(r, WIDE ? MPS_F32 : dtype == MPS_BF16 ? MPS_BF16 : MPS_F16, v.each());
    }
    static __device__ __forceinline__ void store(void* base, int dtype, int64_t at, const RotateLane& l, const Pairs& v) {
        if (WIDE) {
            float* p = static_cast<float*>(base) + at;
            *reinterpret_cast<float4*>(p + l.a) = make_float4(v.p[0].x, v.p[0].y, v.p[1].x, v.p[1].y);
            *reinterpret_cast<float4*>(p + l.b) = make_float4(v.p[2].x, v.p[2].y, v.p[3].x, v.p[3].y);
        } else {
            uint16_t* p = static_cast<uint16_t*>(base) + at;
            *reinterpret_cast<uint2*>(p + l.a) = make_uint2(pack2(v.p[0].x, v.p[0].y, dtype), pack2(v.p[1].x, v.p[1].y, dtype));
            *reinterpret_cast<uint2*>(p + l.b) = make_uint2(pack2(v.p[2].x, v.p[2].y, dtype), pack2(v.p[3].x, v.p[3].y, dtype));
        }
    }
};
// A norm's weight at a lane's places.
__device__ __forceinline__ void rotate_gain(const mps_head_rotate& r, const void* weight, const RotateLane& l, Pairs& v) {
    if (!weight || !l.live) return;
    if (r.weight_dtype == MPS_F32) {
        RotateRaw<true> raw;
        raw.load(weight, 0, l);
        raw.values(MPS_F32, v);
    } else {
        RotateRaw<false> raw;
        raw.load(weight, 0, l);
        raw.values(r.weight_dtype, v);
    }
}
// A lane's values, normalised (all LANES of the head, `mates`, together) and turned.
template <int LANES>
__device__ __forceinline__ void rotate8(const RotateArgs& p, Pairs& v, bool normed, const Pairs& gain, bool turned, const float (&c)[4], const float (&s)[4], uint32_t mates) {
    if (normed) {
        float2 two = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 4; ++i) two = fma2(v.p[i], v.p[i], two);
        float sum = two.x + two.y;
#pragma unroll
        for (int o = LANES / 2; o; o >>= 1) sum += __shfl_xor_sync(mates, sum, o);
        v = times(times(v, rsqrtf(fmaf(sum, p.inv_dim, p.a.eps))), gain);
    }
    if (!turned) return;
    if (p.a.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v.p[i] = fma2(make_float2(v.p[i].y, v.p[i].x), make_float2(-s[i], s[i]), mul2(v.p[i], make_float2(c[i], c[i])));
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float2 x = v.p[i], y = v.p[i + 2], c2 = make_float2(c[2 * i], c[2 * i + 1]), s2 = make_float2(s[2 * i], s[2 * i + 1]);
            v.p[i] = fma2(y, make_float2(-s2.x, -s2.y), mul2(x, c2));
            v.p[i + 2] = fma2(x, s2, mul2(y, c2));
        }
    }
}

// Few tokens.  LANES (a power of two) have a head; STEPS heads a thread; WIDE: FP32.
template <int LANES, int STEPS, bool WIDE>
__global__ void __launch_bounds__(STEPS == 1 ? 1024 : 512) rotate_kernel(const RotateArgs p) {
    __shared__ __align__(16) float cosines[kHeadMostDim / 2], sines[kHeadMostDim / 2];
    griddep_wait();
    griddep_launch();
    const mps_head_rotate& a = p.a;
    const int64_t token = blockIdx.x;
    const int u = threadIdx.x % LANES, per_pass = blockDim.x / LANES, heads = a.q_heads + (a.v ? 2 : 1) * a.kv_heads;
    const uint32_t mates = LANES == 32 ? 0xFFFFFFFFu : ((1u << (LANES & 31)) - 1u) << (threadIdx.x & 31 & ~(LANES - 1));      // the lanes of a head
    const RotateLane lane(a, u);
    int64_t page, offset;
    token_slot(p, token, page, offset);
    RotateRaw<WIDE> raw[STEPS];
    Pairs gain[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int h = s * per_pass + threadIdx.x / LANES;
        raw[s].a = raw[s].b = make_uint4(0u, 0u, 0u, 0u);
        if (h < heads) {
            const HeadPlace place = head_place(p, token, h, page, offset);
            if (lane.live) raw[s].load(place.in, place.in_at, lane);
            rotate_gain(a, place.weight, lane, gain[s]);
        }
    }
    token_angles(p, token, cosines, sines);
    __syncthreads();
    float c[4], sn[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int j = lane.turned ? 4 * u + i : 0;
        c[i] = cosines[j];
        sn[i] = sines[j];
    }
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int h = s * per_pass + threadIdx.x / LANES;      // the same for the lanes of a head
        if (h >= heads) break;
        const HeadPlace place = head_place(p, token, h, page, offset);
        Pairs v;
        raw[s].values(a.dtype, v);
        rotate8<LANES>(p, v, place.weight != nullptr, gain[s], place.turned && lane.turned, c, sn, mates);
        if (place.out && lane.live) RotateRaw<WIDE>::store(place.out, a.dtype, place.out_at, lane, v);
    }
}

// Many tokens: `share` warps have one.
constexpr int kRotateAhead = 4, kRotateWarps = 4;
template <int LANES, bool WIDE>
__global__ void __launch_bounds__(kRotateWarps * 32) rotate_many_kernel(const RotateArgs p, const int share) {
    griddep_wait();
    griddep_launch();
    const mps_head_rotate& a = p.a;
    const int64_t worker = (int64_t)blockIdx.x * kRotateWarps + (threadIdx.x >> 5), token = worker / share;
    if (token >= a.tokens) return;
    constexpr int kHeads = 32 / LANES;
    const int l = threadIdx.x & 31, u = l % LANES, first = (int)(worker % share) * kHeads + l / LANES, step = share * kHeads;
    const uint32_t mates = LANES == 32 ? 0xFFFFFFFFu : ((1u << (LANES & 31)) - 1u) << (l & ~(LANES - 1));      // the lanes of a head
    const RotateLane lane(a, u);
    int64_t page, offset;
    token_slot(p, token, page, offset);
    float c[4], s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (lane.turned) pair_angle(a, token, 4 * u + i, c[i], s[i]);
    // heads of one kind; h0: the first one's number among all
    const auto go = [&](int h0, int heads, int64_t in_stride) {
        if (first >= heads) return;
        const HeadPlace place = head_place(p, token, h0 + first, page, offset);
        Pairs gain;
        rotate_gain(a, place.weight, lane, gain);
        const bool turned = place.turned && lane.turned;
        const int64_t in_step = in_stride * step, out_step = place.out_stride * step;
        RotateRaw<WIDE> raw[kRotateAhead];
        int64_t in = place.in_at, out = place.out_at;
#pragma unroll
        for (int i = 0; i < kRotateAhead; ++i) {
            raw[i].a = raw[i].b = make_uint4(0u, 0u, 0u, 0u);
            if (first + i * step < heads && lane.live) raw[i].load(place.in, in, lane);
            in += in_step;
        }
        for (int h = first; h < heads; h += kRotateAhead * step) {
#pragma unroll
            for (int i = 0; i < kRotateAhead; ++i) {
                if (h + i * step >= heads) break;      // the same for the lanes of a head
                Pairs v;
                raw[i].values(a.dtype, v);
                if (h + (i + kRotateAhead) * step < heads && lane.live) raw[i].load(place.in, in, lane);
                in += in_step;
                rotate8<LANES>(p, v, place.weight != nullptr, gain, turned, c, s, mates);
                if (place.out && lane.live) RotateRaw<WIDE>::store(place.out, a.dtype, out, lane, v);
                out += out_step;
            }
        }
    };
    go(0, a.q_heads, a.q_head_stride);
    go(a.q_heads, a.kv_heads, a.k_head_stride);
    if (a.v) go(a.q_heads + a.kv_heads, a.kv_heads, a.v_head_stride);
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
    const auto threads = [&](int steps) { return ((heads + steps - 1) / steps * LANES + 31) / 32 * 32; };
    // Every head at once, where a CTA has the threads; in three or four steps, where 512 threads have that many (two steps of those would be 1024 threads' one).  64 query and
    // 8 key heads of 128 in three steps take 3.5 us for a token, 7.0 for 400 and 11.3 for 888; in two of 1024 threads 3.2, 8.2 and 15.5; with warps a token 3.2, 8.4 and 11.2.
    int steps = 1;
    if (threads(1) > 1024) steps = threads(3) <= 512 ? 3 : threads(4) <= 512 ? 4 : 0;
    if (p.a.tokens > kRotateFewTokens || !steps) {
        // as many warps for a token as there are places for on the GPU, and passes for
        const int passes = (heads * LANES + 31) / 32;
        int share = 1;
        while (share < passes && p.a.tokens * share < 4096) share *= 2;
        const int64_t ctas = (p.a.tokens * share + kRotateWarps - 1) / kRotateWarps;
        if (ctas > 0x7FFFFFFF) { set_error("mps_head_rotate_rows: too many tokens"); return MPS_ERR_INVALID; }
        return p.a.dtype == MPS_F32 ? launch_overlapping("rotate_many_kernel", rotate_many_kernel<LANES, true>, (unsigned int)ctas, dim3(kRotateWarps * 32), st, p, share)
                                    : launch_overlapping("rotate_many_kernel", rotate_many_kernel<LANES, false>, (unsigned int)ctas, dim3(kRotateWarps * 32), st, p, share);
    }
    const unsigned int ctas = (unsigned int)p.a.tokens;
    const dim3 block((unsigned int)threads(steps));
    if (p.a.dtype == MPS_F32)
        return launch_overlapping("rotate_kernel", steps == 1 ? rotate_kernel<LANES, 1, true> : steps == 3 ? rotate_kernel<LANES, 3, true> : rotate_kernel<LANES, 4, true>, ctas, block, st, p);
    return launch_overlapping("rotate_kernel", steps == 1 ? rotate_kernel<LANES, 1, false> : steps == 3 ? rotate_kernel<LANES, 3, false> : rotate_kernel<LANES, 4, false>, ctas, block, st, p);
}

}  // namespace mps

using namespace mps;

extern "C" int mps_head_rotate_rows(const mps_head_rotate* args, void* stream) {
    if (!args) { set_error("mps_head_rotate_rows: null arguments"); return MPS_ERR_INVALID; }
    RotateArgs p;
    p.a = *args;
    mps_head_rotate& own = p.a;
    const mps_head_rotate& a = p.a;
    // strides of dimensions of one mean nothing
    if (a.tokens == 1) own.q_token_stride = own.k_token_stride = own.v_token_stride = 0;
    if (a.q_heads == 1) own.q_head_stride = 0;
    if (a.kv_heads == 1) own.k_head_stride = own.v_head_stride = own.k_cache_head_stride = own.v_cache_head_stride = 0;
    if (a.pages == 1) own.k_page_stride = own.v_page_stride = 0;
    if (a.page_size == 1) own.k_slot_stride = own.v_slot_stride = 0;
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
    // fours of every head begin at multiples of four values, by pointer and strides
    const auto even = [](const void* q, int dtype, std::initializer_list<int64_t> strides) {
        bool ok = reinterpret_cast<uintptr_t>(q) % (4 * mx4_dtype_bytes(dtype)) == 0;
        for (const int64_t s : strides) ok = ok && s % 4 == 0;
        return ok;
    };
    const bool vec = a.dim % 8 == 0 && a.rotated % 8 == 0 && even(a.q, a.dtype, {a.q_token_stride, a.q_head_stride}) &&
                     even(a.k, a.dtype, {a.k_token_stride, a.k_head_stride}) && even(a.q_out, a.dtype, {}) && even(a.q_weight, a.weight_dtype, {}) &&
                     even(a.k_weight, a.weight_dtype, {}) &&
                     (append ? even(a.v, a.dtype, {a.v_token_stride, a.v_head_stride}) &&
                                   even(a.k_out, a.dtype, {a.k_page_stride, a.k_slot_stride, a.k_cache_head_stride}) &&
                                   even(a.v_out, a.dtype, {a.v_page_stride, a.v_slot_stride, a.v_cache_head_stride})
                             : even(a.k_out, a.dtype, {}));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!vec) return launch_overlapping("rotate_any_kernel", rotate_any_kernel, (unsigned int)a.tokens, dim3(kRotateAnyWarps * 32), st, p);
    if (a.dim <= 32) return launch_rotate<4>(p, st);
    if (a.dim <= 64) return launch_rotate<8>(p, st);
    if (a.dim <= 128) return launch_rotate<16>(p, st);
    return launch_rotate<32>(p, st);
}
