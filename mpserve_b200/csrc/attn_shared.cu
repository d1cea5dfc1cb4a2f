// Attention of a batch of single tokens that share a prefix: every sequence's query attends to the prefix, which all have in common, and to tokens of its own.
//
//   out = sum_k softmax_k(scale q . key_k) value_k      over the prefix's keys and those of the sequence's own table
//
// Both lie in one paged cache.  A part of the keys gives, for a query, a number m near the largest logit, l = sum_k 2^(logit_k - m) and o = sum_k 2^(logit_k - m) value_k (logits
// in units of log 2); parts join as
//   M = max m_i,  out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i
// whatever the keys were split into, so that the prefix is read once for many queries and every sequence's own keys once, each in as many parts as fill the GPU.
#include "attn_prefix.cuh"

namespace mps {

// ---- the parts of a query joined -----------------------------------------------------------------------
//
// A warp has a head of a sequence, its lanes the columns, eight parts at a time under way; with few heads eight warps share one's parts.  (One after the
// other, a warp to a head, the parts of four sequences behind 1024 took 43 us.)
constexpr int kJoinWarps = 8, kJoinAhead = 8;
// A call of 4 sequences of 32 heads takes 14.6 us with eight warps a head and 16.3 with one, of 16 sequences 17.5 and 17.8, of 32 sequences 35.2 and 32.4, of 64 55 and 47.
constexpr int64_t kJoinFewHeads = 512;
template <int DIM, bool BF16, int SHARE>
__global__ void __launch_bounds__(kJoinWarps * 32) attend_join_kernel(const AttendArgs p) {
    constexpr int kColumns = DIM / 32, kHeads = kJoinWarps / SHARE;
    __shared__ float ms[kJoinWarps], ls[kJoinWarps], os[SHARE == 1 ? 1 : kJoinWarps][DIM];
    griddep_wait();
    griddep_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q_heads = p.kv_heads * p.group, tiles = (q_heads + kHeads - 1) / kHeads;
    const int sequence = blockIdx.x / tiles, head = blockIdx.x % tiles * kHeads + warp / SHARE, share = warp % SHARE;
    const int splits = p.plan[0], own_before = p.plan[1 + sequence], own_count = p.plan[2 + sequence] - own_before;
    if (SHARE == 1 && head >= q_heads) return;
    const int kv_head = head / p.group, in_group = head % p.group;
    const int64_t rows = (int64_t)p.batch * p.group, row = (int64_t)sequence * p.group + in_group;
    const int count = splits + own_count;
    const int64_t prefix_step = p.kv_heads * rows, prefix_first = kv_head * rows + row, own_step = (int64_t)p.kv_heads * p.group;
    const int64_t own_first = ((int64_t)own_before * p.kv_heads + kv_head) * p.group + in_group;
    float top = -INFINITY, sum = 0.f, out[kColumns];
#pragma unroll
    for (int c = 0; c < kColumns; ++c) out[c] = 0.f;
    for (int first = share; first < count; first += kJoinAhead * SHARE) {
        float2 ml[kJoinAhead];
        float o[kJoinAhead][kColumns];
#pragma unroll
        for (int j = 0; j < kJoinAhead; ++j) {
            const int i = first + j * SHARE;
            const bool prefix = i < splits, there = i < count;
            const int64_t at = prefix ? prefix_first + i * prefix_step : own_first + (i - splits) * own_step;
            ml[j] = there ? (prefix ? p.prefix_ml : p.own_ml)[at] : make_float2(-INFINITY, 0.f);
            const float* from = (prefix ? p.prefix_o : p.own_o) + at * DIM + lane * kColumns;
            if (kColumns == 4) {
                const float4 v = there ? *reinterpret_cast<const float4*>(from) : make_float4(0.f, 0.f, 0.f, 0.f);
                o[j][0] = v.x; o[j][1] = v.y; o[j][kColumns - 2] = v.z; o[j][kColumns - 1] = v.w;
            } else {
                const float2 v = there ? *reinterpret_cast<const float2*>(from) : make_float2(0.f, 0.f);
                o[j][0] = v.x; o[j][1] = v.y;
            }
        }
        float high = top;
#pragma unroll
        for (int j = 0; j < kJoinAhead; ++j) high = fmaxf(high, ml[j].x);
        const float base = high == -INFINITY ? 0.f : high, up = exp2f(top - base);
        top = high;
        sum *= up;
#pragma unroll
        for (int c = 0; c < kColumns; ++c) out[c] *= up;
#pragma unroll
        for (int j = 0; j < kJoinAhead; ++j) {
            const float w = exp2f(ml[j].x - base);
            sum = fmaf(ml[j].y, w, sum);
#pragma unroll
            for (int c = 0; c < kColumns; ++c) out[c] = fmaf(o[j][c], w, out[c]);
        }
    }
    if (SHARE > 1) {
#pragma unroll
        for (int c = 0; c < kColumns; ++c) os[warp][lane * kColumns + c] = out[c];
        if (lane == 0) { ms[warp] = top; ls[warp] = sum; }
        __syncthreads();
        if (share || head >= q_heads) return;
#pragma unroll
        for (int w = 1; w < SHARE; ++w) top = fmaxf(top, ms[warp + w]);
        const float base = top == -INFINITY ? 0.f : top;
        sum = 0.f;
#pragma unroll
        for (int c = 0; c < kColumns; ++c) out[c] = 0.f;
#pragma unroll
        for (int w = 0; w < SHARE; ++w) {
            const float f = exp2f(ms[warp + w] - base);
            sum = fmaf(ls[warp + w], f, sum);
#pragma unroll
            for (int c = 0; c < kColumns; ++c) out[c] = fmaf(os[SHARE == 1 ? 0 : warp + w][lane * kColumns + c], f, out[c]);
        }
    }
    const float inverse = sum == 0.f ? 0.f : 1.f / sum;      // a query with nothing to attend to gets zeros
    uint16_t* to = p.out + ((int64_t)sequence * q_heads + head) * DIM + lane * kColumns;
#pragma unroll
    for (int c = 0; c < kColumns; c += 2) *reinterpret_cast<uint32_t*>(to + c) = pack_pair<BF16>(out[c] * inverse, out[c + 1] * inverse);
    if (p.lse && lane == 0) p.lse[(int64_t)sequence * q_heads + head] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

// ---- host side -------------------------------------------------------------------------------------------

struct AttendPlan {
    int wide_tiles;               // CTAs for a stretch of the prefix and a key head
    int most_splits;              // stretches of the prefix, at most
    int own_ctas;                 // -1: the GPU settles it
    int64_t ctas;
    int64_t own_items;            // stretches of own keys, at most
    int64_t floats(int64_t rows, int64_t kv_heads, int64_t group, int64_t dim) const {      // of the scratch, behind its first part
        return (most_splits * kv_heads * rows + own_items * kv_heads * group) * (dim + 2);
    }
};
static int64_t plan_words(int64_t batch) { return (batch + 2 + 3) / 4 * 4; }
static AttendPlan attend_plan(const mps_prefix_attend& a, int sms) {
    AttendPlan plan = {};
    const int64_t group = a.q_heads / a.kv_heads, rows = a.batch * group, row_tiles = (rows + kPrefixRows - 1) / kPrefixRows;
    const int64_t most = a.table_columns * a.page_size, heads = a.kv_heads * ((group + kFewColumns - 1) / kFewColumns);
    plan.wide_tiles = (int)((row_tiles + 1) / 2);
    plan.own_ctas = -1;
    plan.ctas = sms;
    if (a.prefix_length > 0) {
        // a CTA an SM, one of them at least for the sequences, as long as there are tiles of keys
        const int64_t units = plan.wide_tiles * (int64_t)a.kv_heads, tiles = (a.prefix_length + kPrefixKeys - 1) / kPrefixKeys;
        if (units + (most > 0) > sms) {
            // More than there are SMs for already: the sequences get a CTA an SM behind them.  1200 sequences (32 query, 8 key heads of 128) behind 300 keys with up to 100 of
            // their own take 128 us, with a CTA for every second SM 149, for every fourth 224, with two an SM 141; behind 2048 with up to 512 319, 421, 687 and 323; 4096 behind
            // 8192 with up to 100 865, 855, 1096 and 874.
            plan.most_splits = 1;
            plan.own_ctas = most > 0 ? sms : 0;
            plan.ctas = units + plan.own_ctas;
        } else {
            plan.most_splits = (int)std::min<int64_t>(tiles, (sms - (most > 0)) / units);
        }
    }
    if (most > 0) {
        const int64_t extra = std::min<int64_t>((4 * kOwnWarps * (int64_t)sms + heads - 1) / heads, a.batch * ((most + kOwnLeast - 1) / kOwnLeast));
        plan.own_items = a.batch + extra;
    }
    return plan;
}

static int check_attend(const mps_prefix_attend& a) {
    if (a.batch < 0 || a.batch > MPS_MOST_SEQUENCES || a.q_heads <= 0 || a.kv_heads <= 0 || a.q_heads > MPS_MOST_HEADS || a.q_heads % a.kv_heads) {
        set_error("mps_prefix_attend_tokens: batch must be in [0, %d], query heads a multiple of the key heads and at most %d", (int)MPS_MOST_SEQUENCES, (int)MPS_MOST_HEADS);
        return MPS_ERR_INVALID;
    }
    if (a.dim != 64 && a.dim != 128) { set_error("mps_prefix_attend_tokens: dim must be 64 or 128"); return MPS_ERR_INVALID; }
    if (a.dtype != MPS_BF16 && a.dtype != MPS_F16) { set_error("mps_prefix_attend_tokens: dtype must be BF16 or F16"); return MPS_ERR_INVALID; }
    if (a.pages < 0 || a.pages > 0x7FFFFFFF || a.page_size < 16 || a.page_size > 1 << 20 || (a.page_size & (a.page_size - 1))) {
        set_error("mps_prefix_attend_tokens: the size of a page must be a power of two from 16 to 2^20, pages below 2^31");
        return MPS_ERR_INVALID;
    }
    if (a.table_columns < 0 || a.table_columns > MPS_MOST_KEYS / a.page_size || a.prefix_length < 0 || a.prefix_length > MPS_MOST_KEYS) {
        set_error("mps_prefix_attend_tokens: a table and the prefix may have at most %lld keys", (long long)MPS_MOST_KEYS);
        return MPS_ERR_INVALID;
    }
    return MPS_OK;
}

using EncodeTiled = decltype(&cuTensorMapEncodeTiled);
static int page_map(CUtensorMap& map, EncodeTiled encode, const void* pages, const mps_prefix_attend& a, int64_t slot, int64_t head, int64_t page) {
    const cuuint64_t size[4] = {(cuuint64_t)a.dim, (cuuint64_t)a.page_size, (cuuint64_t)a.kv_heads, (cuuint64_t)a.pages};
    // of a dimension of one the stride is never used, but may not be 0
    const auto bytes = [&](int64_t stride) { return (cuuint64_t)(stride ? stride : a.dim) * 2; };
    const cuuint64_t stride[3] = {bytes(slot), bytes(head), bytes(page)};
    const cuuint32_t box[4] = {64, (cuuint32_t)std::min(a.page_size, (int64_t)kPrefixKeys), 1, 1}, step[4] = {1, 1, 1, 1};
    const CUresult r = encode(&map, a.dtype == MPS_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(pages), size, stride, box, step,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? MPS_OK : cuda_fail(static_cast<cudaError_t>(r), "cuTensorMapEncodeTiled");      // the two count their errors alike
}
static int page_maps(PrefixMaps& maps, const mps_prefix_attend& a) {
    EncodeTiled encode;
    const int found = tensor_map_encoder(encode);
    if (found) return found;
    const int rc = page_map(maps.k, encode, a.k_pages, a, a.k_slot_stride, a.k_head_stride, a.k_page_stride);
    return rc ? rc : page_map(maps.v, encode, a.v_pages, a, a.v_slot_stride, a.v_head_stride, a.v_page_stride);
}

template <int DIM, bool BF16>
static int attend(const AttendArgs& p, const mps_prefix_attend& a, unsigned int ctas, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};
    Device d;
    int rc = current_device(d);
    if (rc) return rc;
    if (!(ready.load(std::memory_order_acquire) >> (d.ordinal & 63) & 1)) {
        MPS_CUDA_TRY(cudaFuncSetAttribute(attend_kernel<DIM, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, PrefixShape<DIM>::kSmem));
        ready.fetch_or(uint64_t(1) << (d.ordinal & 63), std::memory_order_release);
    }
    PrefixMaps maps = {};
    if (p.prefix) rc = page_maps(maps, a);
    if (!rc) rc = launch_overlapping_smem("attend_kernel", attend_kernel<DIM, BF16>, ctas, dim3(kAttendThreads), PrefixShape<DIM>::kSmem, st, p, maps);
    if (rc) return rc;
    const int64_t q_heads = (int64_t)p.kv_heads * p.group;
    if (a.batch * q_heads <= kJoinFewHeads)
        return launch_overlapping("attend_join_kernel", attend_join_kernel<DIM, BF16, kJoinWarps>, (unsigned int)(a.batch * q_heads), dim3(kJoinWarps * 32), st, p);
    return launch_overlapping("attend_join_kernel", attend_join_kernel<DIM, BF16, 1>, (unsigned int)(a.batch * ((q_heads + kJoinWarps - 1) / kJoinWarps)), dim3(kJoinWarps * 32), st, p);
}

}  // namespace mps

using namespace mps;

extern "C" int64_t mps_prefix_attend_scratch_bytes(const mps_prefix_attend* args) {
    if (!args || check_attend(*args)) return -1;
    Device d;
    if (current_device(d)) return -1;
    const int64_t group = args->q_heads / args->kv_heads;
    return attend_plan(*args, d.sms).floats(args->batch * group, args->kv_heads, group, args->dim) * 4 + plan_words(args->batch) * 4;
}

extern "C" int mps_prefix_attend_tokens(const mps_prefix_attend* args, void* scratch, int64_t scratch_bytes, void* workspace, int64_t workspace_bytes,
                                        void* stream) {
    if (!args) { set_error("mps_prefix_attend_tokens: null arguments"); return MPS_ERR_INVALID; }
    mps_prefix_attend a = *args;
    int rc = check_attend(a);
    if (rc) return rc;
    if (a.batch == 0) return MPS_OK;
    if (a.pages == 0) a.prefix_length = a.table_columns = 0;      // no key is there
    // strides of dimensions of one mean nothing
    if (a.batch == 1) a.q_token_stride = 0;
    if (a.q_heads == 1) a.q_head_stride = 0;
    if (a.kv_heads == 1) a.k_head_stride = a.v_head_stride = 0;
    if (a.pages == 1) a.k_page_stride = a.v_page_stride = 0;
    if (!a.q || !a.out || (a.pages && (!a.k_pages || !a.v_pages)) || (a.table_columns && (!a.tables || !a.lengths)) || (a.prefix_length && !a.prefix_table)) {
        set_error("mps_prefix_attend_tokens: missing pointer");
        return MPS_ERR_INVALID;
    }
    if (((reinterpret_cast<uintptr_t>(a.k_pages) | reinterpret_cast<uintptr_t>(a.v_pages)) & 15u) || (a.k_page_stride | a.k_slot_stride | a.k_head_stride) % 8 ||
        (a.v_page_stride | a.v_slot_stride | a.v_head_stride) % 8) {
        set_error("mps_prefix_attend_tokens: pages must be 16-byte aligned, their strides multiples of 8 elements");
        return MPS_ERR_INVALID;
    }
    if ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out)) & 15u || (a.q_token_stride | a.q_head_stride) % 8) {
        set_error("mps_prefix_attend_tokens: queries must be 16-byte aligned, their strides multiples of 8 elements");
        return MPS_ERR_INVALID;
    }
    Device d;
    rc = current_device(d);
    if (rc) return rc;
    AttendArgs p = {};
    const int64_t group = a.q_heads / a.kv_heads, rows = a.batch * group;
    const AttendPlan plan = attend_plan(a, d.sms);
    if (!scratch || (reinterpret_cast<uintptr_t>(scratch) & 15u) || scratch_bytes < plan.floats(rows, a.kv_heads, group, a.dim) * 4 + plan_words(a.batch) * 4) {
        set_error("mps_prefix_attend_tokens: scratch missing, unaligned or too small");
        return MPS_ERR_WORKSPACE;
    }
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) || workspace_bytes < mps_mx4_workspace_bytes()) {
        set_error("mps_prefix_attend_tokens: workspace missing, unaligned or too small");
        return MPS_ERR_WORKSPACE;
    }
    p.workspace = static_cast<uint32_t*>(workspace);
    p.q = static_cast<const uint16_t*>(a.q);
    p.k = static_cast<const uint16_t*>(a.k_pages);
    p.v = static_cast<const uint16_t*>(a.v_pages);
    p.out = static_cast<uint16_t*>(a.out);
    p.lse = a.lse;
    p.tables = a.tables;
    p.lengths = a.lengths;
    p.prefix_table = a.prefix_table;
    p.q_token = a.q_token_stride; p.q_head = a.q_head_stride;
    p.k_page = a.k_page_stride; p.k_slot = a.k_slot_stride; p.k_head = a.k_head_stride;
    p.v_page = a.v_page_stride; p.v_slot = a.v_slot_stride; p.v_head = a.v_head_stride;
    p.table_columns = a.table_columns;
    p.most_own = a.table_columns * a.page_size;
    p.prefix = (int32_t)a.prefix_length;
    p.wide_tiles = plan.wide_tiles;
    p.most_splits = plan.most_splits;
    p.own_items = (int32_t)plan.own_items;
    p.own_ctas = plan.own_ctas;
    p.pages = (int32_t)a.pages;
    p.page_shift = __builtin_ctzll((unsigned long long)a.page_size);
    p.page_mask = a.page_size - 1;
    p.batch = (int32_t)a.batch;
    p.kv_heads = a.kv_heads;
    p.group = (int32_t)group;
    // a negative scale is the queries' sign, one of 0 makes them zeros: what multiplies the logits is positive, and the largest stays the largest
    p.q_factor = a.scale > 0.f ? 1 : a.scale < 0.f ? -1 : a.scale == 0.f ? 0 : 1;
    p.scale_log2 = a.scale == 0.f ? 1.f : fabsf(a.scale) * 1.4426950408889634f;
    const int64_t prefix_parts = plan.most_splits * a.kv_heads * rows, own_parts = plan.own_items * a.kv_heads * group;
    p.plan = static_cast<int32_t*>(scratch);
    p.prefix_o = static_cast<float*>(scratch) + plan_words(a.batch);
    p.own_o = p.prefix_o + prefix_parts * a.dim;
    p.prefix_ml = reinterpret_cast<float2*>(p.own_o + own_parts * a.dim);
    p.own_ml = p.prefix_ml + prefix_parts;
    if (plan.ctas > 0x7FFFFFFF || plan.own_items * a.kv_heads * ((group + kFewColumns - 1) / kFewColumns) > 0x7FFFFFFF) {
        set_error("mps_prefix_attend_tokens: too much work for one launch");
        return MPS_ERR_INVALID;
    }
    const unsigned int ctas = (unsigned int)plan.ctas;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a.dim == 64) return a.dtype == MPS_BF16 ? attend<64, true>(p, a, ctas, st) : attend<64, false>(p, a, ctas, st);
    return a.dtype == MPS_BF16 ? attend<128, true>(p, a, ctas, st) : attend<128, false>(p, a, ctas, st);
}
