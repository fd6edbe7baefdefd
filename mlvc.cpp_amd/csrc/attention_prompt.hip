// Attention of packed sequences (one pass over the keys with the running
// maximum and sum of the softmax).
//
//   m' = max(m, max_j s_j),  l' = l e^(m - m') + sum_j e^(s_j - m'),
//   o' = o e^(m - m') + sum_j e^(s_j - m') v_j,   out = o / l
//
// in powers of two: s is scaled by log2(e), so each exponential is one
// v_exp_f32.

#include "attention.hpp"

namespace mlvc_hip {
namespace {

struct PromptArgs {
    const std::uint16_t* q;
    const std::uint16_t* k;
    const std::uint16_t* v;
    std::uint16_t* out;
    std::int64_t q_stride, k_stride, v_stride, out_stride;
    const std::int32_t* q_starts;
    const std::int32_t* k_starts;
    int sequences, q_heads, group, dim, q_tokens, k_tokens, longest_q, causal;
    float scale2;  // scale log2(e)
};

// Rows [first, first + count) of a sequence, cut to the tensor.
struct Span {
    int first, count;
};
__device__ __forceinline__ Span span(const std::int32_t* starts, int n, int tokens)
{
    const int a = min(max(starts[n], 0), tokens), b = min(max(starts[n + 1], a), tokens);
    return {a, b - a};
}

// Any head size and alignment: one wave for a query of a head, 64 keys at a
// time, one key a lane for the scores and one value column a lane for the sum.
__global__ __launch_bounds__(64) void prompt_any_kernel(PromptArgs a)
{
    __shared__ float qs[kMaxHeadDim], ps[64];
    const int lane = threadIdx.x, token = blockIdx.x, head = blockIdx.y;
    int lo = 0, hi = a.sequences;  // the last sequence that starts at or before the token
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.q_starts[mid] <= token) lo = mid;
        else hi = mid;
    }
    const Span sq = span(a.q_starts, lo, a.q_tokens), sk = span(a.k_starts, lo, a.k_tokens);
    const int i = token - sq.first;
    if (i < 0 || i >= sq.count || i >= a.longest_q) return;
    const int seen = a.causal ? min(sk.count, max(0, sk.count - sq.count + i + 1)) : sk.count;
    const std::uint16_t* q = a.q + token * a.q_stride + static_cast<std::int64_t>(head) * a.dim;
    for (int d = lane; d < a.dim; d += 64) qs[d] = h2f(q[d]) * a.scale2;
    __syncthreads();
    const std::int64_t column = static_cast<std::int64_t>(head / a.group) * a.dim;
    constexpr int kColumns = kMaxHeadDim / 64;
    float acc[kColumns] = {}, m = -INFINITY, l = 0.0f;
    for (int j0 = 0; j0 < seen; j0 += 64) {
        float s = -INFINITY;
        if (j0 + lane < seen) {
            const std::uint16_t* k = a.k + static_cast<std::int64_t>(sk.first + j0 + lane) * a.k_stride + column;
            s = 0.0f;
            for (int d = 0; d < a.dim; ++d) s = fmaf(qs[d], h2f(k[d]), s);
        }
        const float top = fmaxf(m, group_max<64>(s)), base = top == -INFINITY ? 0.0f : top;
        const float p = __builtin_amdgcn_exp2f(s - base), keep = __builtin_amdgcn_exp2f(m - base);
        m = top;
        l = l * keep + group_sum<64>(p);
        ps[lane] = p;
        __syncthreads();
        const int n = min(64, seen - j0);
        const std::uint16_t* v = a.v + static_cast<std::int64_t>(sk.first + j0) * a.v_stride + column;
#pragma unroll
        for (int c = 0; c < kColumns; ++c) {
            const int d = c * 64 + lane;
            if (d >= a.dim) break;
            float sum = acc[c] * keep;
            for (int j = 0; j < n; ++j) sum = fmaf(ps[j], h2f(v[j * a.v_stride + d]), sum);
            acc[c] = sum;
        }
        __syncthreads();
    }
    const float r = l == 0.0f ? 0.0f : 1.0f / l;
    std::uint16_t* out = a.out + token * a.out_stride + static_cast<std::int64_t>(head) * a.dim;
#pragma unroll
    for (int c = 0; c < kColumns; ++c)
        if (c * 64 + lane < a.dim) out[c * 64 + lane] = f2h(opaque(acc[c] * r));
}

void attention_prompt(const mlvc_hip_attention_prompt_desc* d, hipStream_t s)
{
    const char* op = "attention_prompt";
    require(d != nullptr, op, "no descriptor");
    require(d->sequences >= 0 && d->q_tokens >= 0 && d->k_tokens >= 0 && d->longest_q >= 0, op, "negative size");
    require(d->head_dim >= 1 && d->head_dim <= kMaxHeadDim, op, "head_dim must be 1..512");
    require(d->kv_heads >= 1 && d->q_heads >= 1 && d->q_heads <= 65535 && d->q_heads % d->kv_heads == 0, op,
            "q_heads must be a multiple of kv_heads, 1..65535");
    require(std::isfinite(d->scale), op, "scale must be finite");
    const std::int64_t q_row = static_cast<std::int64_t>(d->q_heads) * d->head_dim,
                       k_row = static_cast<std::int64_t>(d->kv_heads) * d->head_dim;
    require(d->q_stride >= q_row && d->out_stride >= q_row && d->k_stride >= k_row && d->v_stride >= k_row, op,
            "a stride is shorter than a row of heads");
    if (d->sequences == 0 || d->q_tokens == 0 || d->longest_q == 0) return;
    require(d->q && d->out && d->q_starts && d->k_starts && (d->k_tokens == 0 || (d->k && d->v)), op, "null tensor");
    for (const void* p : {d->q, d->k, d->v, static_cast<const void*>(d->out)})
        require(aligned2(p), op, "a tensor is not aligned to its FP16 values");

    PromptArgs a{};
    a.q = static_cast<const std::uint16_t*>(d->q);
    a.k = static_cast<const std::uint16_t*>(d->k);
    a.v = static_cast<const std::uint16_t*>(d->v);
    a.out = static_cast<std::uint16_t*>(d->out);
    a.q_stride = d->q_stride, a.k_stride = d->k_stride, a.v_stride = d->v_stride, a.out_stride = d->out_stride;
    a.q_starts = d->q_starts, a.k_starts = d->k_starts;
    a.sequences = d->sequences, a.q_heads = d->q_heads, a.group = d->q_heads / d->kv_heads, a.dim = d->head_dim;
    a.q_tokens = d->q_tokens, a.k_tokens = d->k_tokens, a.longest_q = d->longest_q, a.causal = d->causal != 0;
    a.scale2 = d->scale * 1.4426950408889634f;
    prompt_any_kernel<<<dim3(static_cast<unsigned>(d->q_tokens), static_cast<unsigned>(d->q_heads)), 64, 0, s>>>(a);
    check(hipGetLastError(), "attention_prompt launch");
}

}  // namespace
}  // namespace mlvc_hip

using namespace mlvc_hip;

extern "C" int mlvc_hip_attention_prompt(const mlvc_hip_attention_prompt_desc* desc, mlvc_hip_stream s)
{
    return guard([&] { attention_prompt(desc, to_stream(s)); });
}
