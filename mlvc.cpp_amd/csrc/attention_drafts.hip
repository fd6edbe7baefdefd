// Attention of each stream's last tokens (drafts that form a tree, or one
// token) on its paged, quantised context, under a window.
//
//   out_i = sum_{j in V(i)} softmax_j(scale q_i . k_j) v_j
//
// V(i) holds the context's places j with place_i - j < window or j < sinks, and
// the drafts of i's mask, at places past + depth, by the same rule. depth is the
// number of other drafts that a draft sees.

#include "attention.hpp"

#include <algorithm>

namespace mlvc_hip {
namespace {

constexpr int kStep = 32;     // tokens of a step
constexpr int kMostDrafts = 64;

struct DraftArgs {
    const std::uint8_t* k;
    const std::uint8_t* v;
    const float* k_scale;
    const float* v_scale;
    const std::uint16_t* q;
    std::uint16_t* out;
    std::int64_t q_stride, out_stride;
    const std::int32_t* starts;
    const unsigned long long* seen;
    const std::int32_t* table;
    const std::int32_t* lengths;
    int table_stride, pages, page, heads, q_heads, group, dim, longest, longest_q, q_tokens, streams, window, sinks;
    float scale2;
};

// A stream's context. Its steps: those that hold sinks, then those from the
// window's first token on.
struct View {
    int start, drafts, queries;  // first row of q; drafts in the cache; rows that are computed
    int past, length;            // place of the first draft; tokens in the cache
    int sinks, sink_steps, skipped, steps;
    __device__ View(const DraftArgs& a, int stream) : View(a, a.starts[stream], a.starts[stream + 1], a.lengths[stream]) {}
    __device__ View(const DraftArgs& a, int begin, int end, int tokens)
    {
        const std::int64_t held = static_cast<std::int64_t>(a.table_stride) * a.page;
        start = min(max(begin, 0), a.q_tokens);
        drafts = max(end - begin, 0);
        queries = min(min(drafts, a.longest_q), a.q_tokens - start);
        tokens = max(tokens, 0);
        past = tokens - drafts;
        length = static_cast<int>(min(static_cast<std::int64_t>(min(tokens, a.longest)), held));
        const int first = a.window ? max(past - a.window + 1, 0) / kStep : 0;
        sinks = a.window ? min(a.sinks, length) : 0;
        sink_steps = (sinks + kStep - 1) / kStep;
        const int all = (length + kStep - 1) / kStep;
        skipped = max(min(first, all) - sink_steps, 0);
        steps = all - skipped;
    }
    // First token of a step.
    __device__ int token(int step) const { return (step < sink_steps ? step : step + skipped) * kStep; }
};

// What a draft sees.
struct Sight {
    int from = 0, sinks = 0, past = 0;  // context from `from` on, and before `sinks`
    unsigned long long drafts = 0;
    __device__ bool operator()(int j) const
    {
        return j < past ? j >= from || j < sinks : j - past < kMostDrafts && (drafts >> (j - past) & 1);
    }
};

// Masks and depths of a stream's drafts, one a lane.
__device__ __forceinline__ unsigned long long mask_of(const DraftArgs& a, const View& w, int draft)
{
    const unsigned long long there = w.drafts < 64 ? (1ull << w.drafts) - 1 : ~0ull;
    if (!a.seen || w.start + draft >= a.q_tokens || draft >= w.drafts) return there & (2ull << draft) - 1;
    return a.seen[w.start + draft] & there;
}
__device__ __forceinline__ int depth_of(unsigned long long mask, int draft) { return __popcll(mask & ~(1ull << draft)); }

// Row of token j of a stream's context, or -1 where its page is not in the cache.
__device__ __forceinline__ std::int64_t token_row(const DraftArgs& a, int stream, int head, int j)
{
    const int page = a.table[static_cast<std::int64_t>(stream) * a.table_stride + j / a.page];
    return page < 0 || page >= a.pages ? -1 : (static_cast<std::int64_t>(page) * a.heads + head) * a.page + j % a.page;
}

// Any head size: one wave for a draft and a query head, 64 tokens at a time,
// one token a lane for the scores and one value column a lane for the sum.
template <int KIND>
__global__ __launch_bounds__(64) void drafts_any_kernel(DraftArgs a)
{
    __shared__ float qs[kMaxHeadDim], ps[64];
    __shared__ long long at[64];
    const int lane = threadIdx.x, head = blockIdx.x % a.q_heads, rest = blockIdx.x / a.q_heads;
    const int draft = rest % a.longest_q, stream = rest / a.longest_q;
    const View w(a, stream);
    if (draft >= w.queries) return;
    Sight sight;
    {
        const unsigned long long mine = mask_of(a, w, lane), mask = __shfl(mine, draft);
        const int depth = depth_of(mine, lane), depth_i = __shfl(depth, draft);
        sight.past = w.past;
        sight.from = a.window ? max(w.past + depth_i - a.window + 1, 0) : 0;
        sight.sinks = w.sinks;
        sight.drafts = mask & __ballot(!a.window || depth_i - depth < a.window || w.past + depth < a.sinks);
    }
    constexpr int kColumns = kMaxHeadDim / 64;
    auto value = [&](const std::uint8_t* x, long long row, int d) {
        if constexpr (KIND == MLVC_KV_F16) return h2f(reinterpret_cast<const std::uint16_t*>(x)[row * a.dim + d]);
        else return from_byte(KIND, x[row * a.dim + d]);
    };
    const std::int64_t token = w.start + draft;
    const std::uint16_t* q = a.q + token * a.q_stride + static_cast<std::int64_t>(head) * a.dim;
    for (int d = lane; d < a.dim; d += 64) qs[d] = h2f(q[d]) * a.scale2;
    __syncthreads();
    float acc[kColumns] = {}, m = -INFINITY, l = 0.0f;
    for (int step = 0; step < w.steps; step += 2) {
        const int mine = step + lane / kStep, j = mine < w.steps ? w.token(mine) + lane % kStep : w.length;
        const long long row = j < w.length && sight(j) ? token_row(a, stream, head / a.group, j) : -1;
        float s = -INFINITY;
        if (row >= 0) {
            s = 0.0f;
            for (int d = 0; d < a.dim; ++d) s = fmaf(qs[d], value(a.k, row, d), s);
            if constexpr (KIND != MLVC_KV_F16) s *= a.k_scale[row];
        }
        const float top = fmaxf(m, group_max<64>(s)), base = top == -INFINITY ? 0.0f : top;
        float p = __builtin_amdgcn_exp2f(s - base);
        const float keep = __builtin_amdgcn_exp2f(m - base);
        m = top;
        l = l * keep + group_sum<64>(p);
        if constexpr (KIND != MLVC_KV_F16) p = row < 0 ? 0.0f : p * a.v_scale[row];
        ps[lane] = p;
        at[lane] = row;
        __syncthreads();
#pragma unroll
        for (int c = 0; c < kColumns; ++c) {
            const int d = c * 64 + lane;
            if (d >= a.dim) break;
            float sum = acc[c] * keep;
            for (int i = 0; i < 64; ++i)
                if (at[i] >= 0) sum = fmaf(ps[i], value(a.v, at[i], d), sum);
            acc[c] = sum;
        }
        __syncthreads();
    }
    if constexpr (KIND == MLVC_KV_F16) {
        for (int c = 0; c < kColumns; ++c) {
            const int d = c * 64 + lane;
            if (d >= a.dim || is_finite(acc[c])) continue;
            OddValues odd;
            for (int step = 0; step < w.steps; ++step)
                for (int j = w.token(step), i = 0; i < kStep && j < w.length; ++i, ++j) {
                    const std::int64_t row = sight(j) ? token_row(a, stream, head / a.group, j) : -1;
                    if (row >= 0) odd.add(reinterpret_cast<const std::uint16_t*>(a.v)[row * a.dim + d]);
                }
            acc[c] = odd.sum(acc[c]);
        }
    }
    const float r = l == 0.0f ? 0.0f : 1.0f / l;
    std::uint16_t* out = a.out + token * a.out_stride + static_cast<std::int64_t>(head) * a.dim;
#pragma unroll
    for (int c = 0; c < kColumns; ++c)
        if (c * 64 + lane < a.dim) out[c * 64 + lane] = f2h(opaque(acc[c] * r));
}

void check_desc(const mlvc_hip_attention_drafts_desc* d, const char* op)
{
    require(d != nullptr, op, "no descriptor");
    check_cache(d->cache, op);
    require(d->streams >= 0 && d->longest >= 0 && d->table_stride >= 0 && d->q_tokens >= 0, op, "negative size");
    require(d->longest_q >= 1 && d->longest_q <= kMostDrafts, op, "longest_q must be 1..64");
    require(d->window >= 0 && d->sinks >= 0, op, "window and sinks must not be negative");
    require(d->q_heads >= 1 && d->q_heads <= 65535 && d->q_heads % d->cache->heads == 0, op,
            "q_heads must be a multiple of the cache's heads, 1..65535");
    require(std::isfinite(d->scale), op, "scale must be finite");
}

void attention_drafts(const mlvc_hip_attention_drafts_desc* d, hipStream_t s)
{
    const char* op = "attention_drafts";
    check_desc(d, op);
    const std::int64_t row = static_cast<std::int64_t>(d->q_heads) * d->cache->head_dim;
    require(d->q_stride >= row && d->out_stride >= row, op, "a stride is shorter than a row of heads");
    if (d->streams == 0 || d->q_tokens == 0) return;
    require(d->q && d->out && d->starts && d->lengths && (d->table || d->table_stride == 0), op, "null tensor");
    require(aligned2(d->q) && aligned2(d->out), op, "a tensor is not aligned to its FP16 values");
    require(aligned_to<8>(d->seen) && aligned_to<4>(d->starts) && aligned_to<4>(d->lengths) && aligned_to<4>(d->table), op,
            "seen, starts, lengths or table is not aligned to its values");
    const std::int64_t grid = static_cast<std::int64_t>(d->streams) * d->longest_q * d->q_heads;
    require(launchable(grid, 64), op, "too many streams, heads and drafts in one call");

    const mlvc_hip_kv_cache* c = d->cache;
    DraftArgs a{};
    a.k = static_cast<const std::uint8_t*>(c->k), a.v = static_cast<const std::uint8_t*>(c->v);
    a.k_scale = c->k_scale, a.v_scale = c->v_scale;
    a.q = static_cast<const std::uint16_t*>(d->q), a.out = static_cast<std::uint16_t*>(d->out);
    a.q_stride = d->q_stride, a.out_stride = d->out_stride;
    a.starts = d->starts, a.seen = reinterpret_cast<const unsigned long long*>(d->seen), a.table = d->table, a.lengths = d->lengths;
    a.table_stride = d->table_stride, a.pages = c->pages, a.page = c->page_size, a.heads = c->heads;
    a.q_heads = d->q_heads, a.group = d->q_heads / c->heads, a.dim = c->head_dim;
    a.longest = c->pages ? d->longest : 0, a.longest_q = d->longest_q, a.q_tokens = d->q_tokens, a.streams = d->streams;
    a.window = d->window, a.sinks = d->sinks;
    a.scale2 = d->scale * 1.4426950408889634f;
    const unsigned n = static_cast<unsigned>(grid);
    if (c->kind == MLVC_KV_F16) drafts_any_kernel<MLVC_KV_F16><<<n, 64, 0, s>>>(a);
    else if (c->kind == MLVC_KV_E4M3) drafts_any_kernel<MLVC_KV_E4M3><<<n, 64, 0, s>>>(a);
    else drafts_any_kernel<MLVC_KV_INT8><<<n, 64, 0, s>>>(a);
    check(hipGetLastError(), "attention_drafts launch");
}

}  // namespace
}  // namespace mlvc_hip

using namespace mlvc_hip;

extern "C" {

size_t mlvc_hip_attention_drafts_workspace_bytes(const mlvc_hip_attention_drafts_desc* desc)
{
    guard([&] { check_desc(desc, "attention_drafts"); });
    return 0;
}

int mlvc_hip_attention_drafts(const mlvc_hip_attention_drafts_desc* desc, mlvc_hip_stream s)
{
    return guard([&] { attention_drafts(desc, to_stream(s)); });
}

}  // extern "C"
