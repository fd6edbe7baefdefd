// Attention of one query per stream on its paged, quantised context.
//
// The context is split over workgroups; each leaves the FP32 state of its
// part, (m, l, o) of the running softmax, in the workspace, and a second kernel
// joins the parts in their order:
//
//   m = max_s m_s,  l = sum_s l_s 2^(m_s - m),  out = sum_s o_s 2^(m_s - m) / l
//
// Scores are in powers of two (scaled by log2(e)). A context of one part
// writes its output itself.

#include "attention.hpp"

#include <algorithm>

namespace mlvc_hip {
namespace {

struct TokenArgs {
    const std::uint8_t* k;
    const std::uint8_t* v;
    const float* k_scale;
    const float* v_scale;
    const std::uint16_t* q;
    std::uint16_t* out;
    std::int64_t q_stride, out_stride;
    const std::int32_t* table;
    const std::int32_t* lengths;
    float* part;   // [streams][q_heads][splits][dim]
    float2* state; // [streams][q_heads][splits]: m, l
    int table_stride, pages, page, heads, q_heads, group, dim, longest, chunk, splits, streams;
    float scale2;
};

__device__ __forceinline__ int context(const TokenArgs& a, int stream)
{
    const std::int64_t held = static_cast<std::int64_t>(a.table_stride) * a.page;
    return static_cast<int>(min(static_cast<std::int64_t>(min(max(a.lengths[stream], 0), a.longest)), held));
}

// Any head size: one wave for a part of one query head's context, 64 tokens
// at a time, one token a lane for the scores and one value column a lane for
// the sum.
template <int KIND>
__global__ __launch_bounds__(64) void token_any_kernel(TokenArgs a)
{
    __shared__ float qs[kMaxHeadDim], ps[64];
    __shared__ long long at[64];
    const int lane = threadIdx.x, split = blockIdx.x % a.splits, rest = blockIdx.x / a.splits;
    const int head = rest % a.q_heads, stream = rest / a.q_heads;
    const int n = context(a, stream), first = split * a.chunk, last = min(n, first + a.chunk);
    const std::uint16_t* q = a.q + stream * a.q_stride + static_cast<std::int64_t>(head) * a.dim;
    for (int d = lane; d < a.dim; d += 64) qs[d] = h2f(q[d]) * a.scale2;
    __syncthreads();
    constexpr int kColumns = kMaxHeadDim / 64;
    float acc[kColumns] = {}, m = -INFINITY, l = 0.0f;
    auto value = [&](const std::uint8_t* x, long long row, int d) {
        if constexpr (KIND == MLVC_KV_F16) return h2f(reinterpret_cast<const std::uint16_t*>(x)[row * a.dim + d]);
        else return from_byte(KIND, x[row * a.dim + d]);
    };
    for (int j0 = first; j0 < last; j0 += 64) {
        const int j = j0 + lane;
        long long row = -1;
        if (j < last) {
            const int page = a.table[static_cast<std::int64_t>(stream) * a.table_stride + j / a.page];
            if (page >= 0 && page < a.pages) row = (static_cast<long long>(page) * a.heads + head / a.group) * a.page + j % a.page;
        }
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
        const int count = min(64, last - j0);
#pragma unroll
        for (int c = 0; c < kColumns; ++c) {
            const int d = c * 64 + lane;
            if (d >= a.dim) break;
            float sum = acc[c] * keep;
            for (int i = 0; i < count; ++i)
                if (at[i] >= 0) sum = fmaf(ps[i], value(a.v, at[i], d), sum);
            acc[c] = sum;
        }
        __syncthreads();
    }
    if (a.splits == 1) {
        const float r = l == 0.0f ? 0.0f : 1.0f / l;
        std::uint16_t* out = a.out + stream * a.out_stride + static_cast<std::int64_t>(head) * a.dim;
#pragma unroll
        for (int c = 0; c < kColumns; ++c)
            if (c * 64 + lane < a.dim) out[c * 64 + lane] = f2h(opaque(acc[c] * r));
        return;
    }
    const std::int64_t slot = (static_cast<std::int64_t>(stream) * a.q_heads + head) * a.splits + split;
#pragma unroll
    for (int c = 0; c < kColumns; ++c)
        if (c * 64 + lane < a.dim) a.part[slot * a.dim + c * 64 + lane] = acc[c];
    if (lane == 0) a.state[slot] = make_float2(m, l);
}

// One workgroup for a query head of a stream.
__global__ __launch_bounds__(64) void token_join_kernel(TokenArgs a)
{
    const int lane = threadIdx.x, head = blockIdx.x % a.q_heads, stream = blockIdx.x / a.q_heads;
    const int parts = min(a.splits, (context(a, stream) + a.chunk - 1) / a.chunk);
    const std::int64_t slot = static_cast<std::int64_t>(blockIdx.x) * a.splits;
    float m = -INFINITY;
    for (int i = lane; i < parts; i += 64) m = fmaxf(m, a.state[slot + i].x);
    m = group_max<64>(m);
    if (m == -INFINITY) m = 0.0f;
    float l = 0.0f;
    for (int i = lane; i < parts; i += 64) {
        const float2 st = a.state[slot + i];
        l += st.y * __builtin_amdgcn_exp2f(st.x - m);
    }
    l = group_sum<64>(l);
    const float r = l == 0.0f ? 0.0f : 1.0f / l;
    std::uint16_t* out = a.out + stream * a.out_stride + static_cast<std::int64_t>(head) * a.dim;
    for (int d = lane; d < a.dim; d += 64) {
        float sum = 0.0f;
        for (int i = 0; i < parts; ++i)
            sum = fmaf(a.part[(slot + i) * a.dim + d], __builtin_amdgcn_exp2f(a.state[slot + i].x - m), sum);
        out[d] = f2h(opaque(sum * r));
    }
}

struct Plan {
    int chunk, splits;
    size_t part_bytes, bytes;
};

// Tokens of a part and parts of a context, from the sizes the host knows.
Plan plan(const mlvc_hip_attention_token_desc* d)
{
    Plan p{};
    p.chunk = 256;
    p.splits = std::max(1, (d->longest + p.chunk - 1) / p.chunk);
    if (p.splits > 1) {
        const size_t slots = static_cast<size_t>(d->streams) * d->q_heads * p.splits;
        p.part_bytes = slots * d->cache->head_dim * sizeof(float);
        p.bytes = p.part_bytes + slots * sizeof(float2);
    }
    return p;
}

void check_desc(const mlvc_hip_attention_token_desc* d, const char* op)
{
    require(d != nullptr, op, "no descriptor");
    check_cache(d->cache, op);
    require(d->streams >= 0 && d->longest >= 0 && d->table_stride >= 0, op, "negative size");
    require(d->q_heads >= 1 && d->q_heads <= 65535 && d->q_heads % d->cache->heads == 0, op,
            "q_heads must be a multiple of the cache's heads, 1..65535");
    require(std::isfinite(d->scale), op, "scale must be finite");
}

void attention_token(const mlvc_hip_attention_token_desc* d, hipStream_t s)
{
    const char* op = "attention_token";
    check_desc(d, op);
    const std::int64_t row = static_cast<std::int64_t>(d->q_heads) * d->cache->head_dim;
    require(d->q_stride >= row && d->out_stride >= row, op, "a stride is shorter than a row of heads");
    if (d->streams == 0) return;
    require(d->q && d->out && d->lengths && (d->table || d->table_stride == 0), op, "null tensor");
    require(aligned2(d->q) && aligned2(d->out), op, "a tensor is not aligned to its FP16 values");
    const Plan p = plan(d);
    require(p.bytes == 0 || (d->workspace && d->workspace_bytes >= p.bytes && aligned16(d->workspace)), op,
            "the workspace is missing, too small or not 16-byte aligned");
    const std::int64_t heads = static_cast<std::int64_t>(d->streams) * d->q_heads;
    require(heads * p.splits <= INT_MAX, op, "too many streams, heads and parts in one call");

    const mlvc_hip_kv_cache* c = d->cache;
    TokenArgs a{};
    a.k = static_cast<const std::uint8_t*>(c->k), a.v = static_cast<const std::uint8_t*>(c->v);
    a.k_scale = c->k_scale, a.v_scale = c->v_scale;
    a.q = static_cast<const std::uint16_t*>(d->q), a.out = static_cast<std::uint16_t*>(d->out);
    a.q_stride = d->q_stride, a.out_stride = d->out_stride;
    a.table = d->table, a.lengths = d->lengths;
    a.part = static_cast<float*>(d->workspace);
    a.state = reinterpret_cast<float2*>(static_cast<char*>(d->workspace) + p.part_bytes);
    a.table_stride = d->table_stride, a.pages = c->pages, a.page = c->page_size, a.heads = c->heads;
    a.q_heads = d->q_heads, a.group = d->q_heads / c->heads, a.dim = c->head_dim;
    a.longest = d->longest, a.chunk = p.chunk, a.splits = p.splits, a.streams = d->streams;
    a.scale2 = d->scale * 1.4426950408889634f;
    const unsigned grid = static_cast<unsigned>(heads * p.splits);
    if (c->kind == MLVC_KV_F16) token_any_kernel<MLVC_KV_F16><<<grid, 64, 0, s>>>(a);
    else if (c->kind == MLVC_KV_E4M3) token_any_kernel<MLVC_KV_E4M3><<<grid, 64, 0, s>>>(a);
    else token_any_kernel<MLVC_KV_INT8><<<grid, 64, 0, s>>>(a);
    check(hipGetLastError(), "attention_token launch");
    if (p.splits > 1) {
        token_join_kernel<<<static_cast<unsigned>(heads), 64, 0, s>>>(a);
        check(hipGetLastError(), "attention_token join launch");
    }
}

}  // namespace
}  // namespace mlvc_hip

using namespace mlvc_hip;

extern "C" {

size_t mlvc_hip_attention_token_workspace_bytes(const mlvc_hip_attention_token_desc* desc)
{
    size_t bytes = 0;
    guard([&] {
        check_desc(desc, "attention_token");
        bytes = plan(desc).bytes;
    });
    return bytes;
}

int mlvc_hip_attention_token(const mlvc_hip_attention_token_desc* desc, mlvc_hip_stream s)
{
    return guard([&] { attention_token(desc, to_stream(s)); });
}

}  // extern "C"
