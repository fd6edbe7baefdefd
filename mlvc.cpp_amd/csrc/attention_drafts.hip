// Attention of each stream's last tokens (drafts that form a tree, or one
// token) on its paged, quantised context, under a window.
//
//   out_i = sum_{j in V(i)} softmax_j(scale q_i . k_j) v_j
//
// V(i) holds the context's places j with place_i - j < window or j < sinks, and
// the drafts of i's mask, at places past + depth, by the same rule. depth is the
// number of other drafts that a draft sees.

#include "attention_cache.hpp"

#include <algorithm>

namespace mlvc_hip {
namespace {

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
    float* part;    // [heads][rows][2 shares + streams][dim], a row for each draft and query head of a group
    float2* state;  // [heads][rows][2 shares + streams]: base, l
    int shares;     // workgroups of a key head and a block of rows that the GPU holds at once; 0: a context goes to one workgroup
    int blocks;     // of rows
    bool spare;     // small shares behind the large ones
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
        steps = queries > 0 ? all - skipped : 0;
    }
    // First token of a step.
    __device__ int token(int step) const { return (step < sink_steps ? step : step + skipped) * kStep; }
};

// What a draft sees.
struct Sight {
    int from, sinks, past;  // context from `from` on, and before `sinks`
    unsigned long long drafts;
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

// ------------------------------------------------------------ matrix cores

// Calls fn(stream, first, last, whole, place) for each piece of a context, steps
// [first, last), that workgroup `share` of a key head and block of rows takes;
// place: the piece's among a row's parts, when it is not the whole context.
template <class F>
__device__ __forceinline__ void each_piece(const DraftArgs& a, int share, F&& fn)
{
    const int lane = threadIdx.x & 63;
    auto steps = [&](int b) { return b + lane < a.streams ? View(a, b + lane).steps : 0; };
    int block = 0, n = steps(0), upto = wave_scan(n);
    int total = __builtin_amdgcn_readlane(upto, 63);
    for (int b = 64; b < a.streams; b += 64) total += wave_sum(steps(b));
    total = __builtin_amdgcn_readfirstlane(total);
    const Shares shares(a.shares, total, a.spare);
    if (share >= 2 * shares.count || (share >= shares.count && shares.large == total)) return;
    int at = __builtin_amdgcn_readfirstlane(shares.first(share));
    const int end = __builtin_amdgcn_readfirstlane(shares.first(share + 1));
    if (at >= end) return;
    auto next_block = [&] {
        const int before = __builtin_amdgcn_readlane(upto, 63);
        block += 64;
        n = steps(block);
        upto = before + wave_scan(n);
    };
    unsigned long long past;
    while (!(past = __ballot(upto > at))) next_block();  // at < total: some stream holds it
    int i = __builtin_ctzll(past);
    for (;;) {
        const int stop = __builtin_amdgcn_readlane(upto, i), start = stop - __builtin_amdgcn_readlane(n, i), to = min(end, stop);
        if (to > at) fn(block + i, at - start, to - start, to - at == stop - start, share + block + i);
        at = max(at, to);
        if (at >= end) return;
        if (++i == 64) next_block(), i = 0;
    }
}

// Sums of FP16 values that a draft sees in steps [first, last), four columns from
// d on, one of which met an infinity or NaN.
__device__ __forceinline__ void decide_odd(const DraftArgs& a, const View& w, const Sight& sight, int stream, int head, int first, int last, int d,
                                           floatx4& sums)
{
    OddValues odd[4];
    for (int step = first; step < last; ++step)
        for (int i = 0, j = w.token(step); i < kStep && j < w.length; ++i, ++j) {
            const std::int64_t row = sight(j) ? token_row(a, stream, head, j) : -1;
            if (row < 0) continue;
#pragma unroll
            for (int r = 0; r < 4; ++r) odd[r].add(reinterpret_cast<const std::uint16_t*>(a.v)[row * a.dim + d + r]);
        }
#pragma unroll
    for (int r = 0; r < 4; ++r) sums[r] = odd[r].sum(sums[r]);
}

// Heads of D values. The rows of a key head are its drafts times the query heads
// that share it; a workgroup takes NB blocks of 16 of them, and a part of one
// stream's context; its waves take consecutive runs of the part, 32 tokens a
// step, and join through LDS at the end. Every row of the cache is read and
// unpacked once for all rows of the workgroup.
//
// Per step, with 16x16x32 products: S^T = K Q^T (two tiles of 16 tokens as rows,
// queries as columns), so a lane's 8 scores belong to one query, and rounded to
// halves they are the B operand of O^T += V^T P^T as they stand. The cache is
// read straight into registers: K rows are A operands as they lie, and V is
// transposed by its conversion to halves.
//
// Scales are applied to scores and weights, not to values: s = (q . k) scale_k,
// and the weight of a row of V is w = 2^(s - base) scale_v. The base is common to
// the weights and their sum: it follows the largest s + log2(scale_v), kLift below
// it, and scale_v counts as 2^-40 at least there (a zero row's is 0; others' are
// 2^-33 and more), so that the sum stays below 2^(15 + 40) a token. Weights are
// rounded to FP16, the type the matrix cores take beside V: by 2^-11 of
// themselves, as the output is, or by 2^-37 of the largest where they are
// subnormal.
//
// A step whose tokens all rows see needs no masks. In the others, those of the
// drafts, of the window's edge and of missing pages, what some of the rows do
// not see must not reach them: infinities and NaN of V are zeroed (a weight of
// zero times one of them is NaN); a quantised row that has one shows it by its
// scale, and the FP16 sums that met one are decided by a second look.
template <int KIND_, int D_, int NB_, int WAVES_, int OCC_>
struct DraftCfg {
    static constexpr int KIND = KIND_, D = D_, NB = NB_, WAVES = WAVES_, OCC = OCC_;
    static constexpr int BYTES = KIND == MLVC_KV_F16 ? 2 : 1;
    static constexpr int KL = D * BYTES / 64;          // 16-byte loads of a lane for a tile of K
    static constexpr int VW = D * BYTES / 64;          // words of a lane for a row of V
    static constexpr int PER = 4 / BYTES;              // values of a word
    static constexpr int DT = D / 16;                  // tiles of O^T
    static constexpr int KS = D / 32;                  // products of a score
    static constexpr int ROWS = NB * 16;
    static constexpr size_t JOINT = (WAVES * 16 * D + 2 * WAVES * 16) * sizeof(float), QUERIES = NB > 1 ? KS * NB * 1024 : 0;
    static constexpr size_t LDS = JOINT > QUERIES ? JOINT : QUERIES;
};

template <class C>
__device__ __forceinline__ void draft_piece(const DraftArgs& a, char* lds, Sight* sights, int* odd_met, int head, int block, int stream, const View& w,
                                            int first, int last, bool whole, int place)
{
    constexpr int D = C::D, KIND = C::KIND, NB = C::NB, KS = C::KS, WAVES = C::WAVES;
    constexpr float kBase0 = -3.402823466e38f;
    // Opaque, so that what follows from it is not kept in registers from piece to piece.
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const int rows = w.queries * a.group, row0 = block * C::ROWS, mine = min(C::ROWS, rows - row0);
    if (mine <= 0) return;

    const int from = first + (last - first) * wave / WAVES, to = first + (last - first) * (wave + 1) / WAVES;
    typedef const __attribute__((address_space(4))) std::int32_t* scalar_table;
    const scalar_table table = (scalar_table)(a.table + static_cast<std::int64_t>(stream) * a.table_stride);

    // Rows of the two tiles (16 tokens each, in one page) of a step, row 0 for a
    // tile that is not there.
    std::int64_t row[2];
    bool there[2];
    auto locate = [&](int j) {
        int at = static_cast<int>(static_cast<unsigned>(j) / static_cast<unsigned>(a.page)), in_page = j - at * a.page;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            int page = -1;
            if (j + 16 * t < w.length) page = table[at];
            there[t] = page >= 0 && page < a.pages;
            row[t] = there[t] ? (static_cast<std::int64_t>(page) * a.heads + head) * a.page + in_page : 0;
            in_page += 16;
            if (in_page == a.page) in_page = 0, ++at;
        }
    };
    u32x4 k[2][C::KL];
    std::uint32_t v[8][C::VW];
    floatx4 ks[2], vs[2];
    auto fetch_k = [&] {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const std::uint8_t* p = a.k + row[t] * (D * C::BYTES);
            const std::uint32_t at = col * (D * C::BYTES) + 16 * g;
#pragma unroll
            for (int i = 0; i < C::KL; ++i) k[t][i] = *reinterpret_cast<const u32x4*>(p + at + 64 * i);
            if constexpr (KIND != MLVC_KV_F16) {
                ks[t] = *reinterpret_cast<const floatx4*>(a.k_scale + row[t] + 4 * g);
                vs[t] = *reinterpret_cast<const floatx4*>(a.v_scale + row[t] + 4 * g);
            }
        }
    };
    auto fetch_v = [&] {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const std::uint8_t* p = a.v + row[t] * (D * C::BYTES);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const std::uint8_t* at = p + (4 * g + e) * (D * C::BYTES) + col * (4 * C::VW);
                if constexpr (C::VW == 4) {
                    const u32x4 x = *reinterpret_cast<const u32x4*>(at);
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[4 * t + e][i] = x[i];
                } else if constexpr (C::VW == 2) {
                    const u32x2 x = *reinterpret_cast<const u32x2*>(at);
                    v[4 * t + e][0] = x[0], v[4 * t + e][1] = x[1];
                } else {
                    v[4 * t + e][0] = *reinterpret_cast<const std::uint32_t*>(at);
                }
            }
        }
    };
    if (from < to) {
        locate(w.token(from));
        fetch_k();
        fetch_v();
    }

    // Queries as B operands, in registers or, shared by the waves, in LDS; rows past the last are zeros.
    auto query = [&](int b, int ks_, int lane_) {
        const int r = b * 16 + (lane_ & 15), g_ = lane_ >> 4;
        const int d = C::BYTES == 1 ? (ks_ >> 1) * 64 + 16 * g_ + 8 * (ks_ & 1) : ks_ * 32 + 8 * g_;
        const int at = row0 + min(r, mine - 1), draft = static_cast<int>(static_cast<unsigned>(at) / static_cast<unsigned>(a.group));
        const u32x4 x = *reinterpret_cast<const u32x4*>(a.q + (w.start + draft) * a.q_stride + static_cast<std::int64_t>(head * a.group + at - draft * a.group) * D + d);
        return r < mine ? x : u32x4{0, 0, 0, 0};
    };
    u32x4* const queries = reinterpret_cast<u32x4*>(lds);  // [KS][NB][64]
    half8 q[KS];
    if constexpr (NB == 1) {
#pragma unroll
        for (int i = 0; i < KS; ++i) q[i] = __builtin_bit_cast(half8, query(0, i, lane));
    } else {
        for (int i = threadIdx.x; i < KS * NB * 64; i += WAVES * 64) queries[i] = query(i >> 6 & (NB - 1), i >> 6 >> (NB == 4 ? 2 : 1), i & 63);
    }
    if (wave == 0) {
        const unsigned long long mask = mask_of(a, w, lane);
        const int depth = depth_of(mask, lane);
        Sight s;
        s.past = w.past, s.sinks = w.sinks;
        s.from = a.window ? max(w.past + depth - a.window + 1, 0) : 0;
        s.drafts = mask;
        if (a.window && a.window < kMostDrafts)
            for (int e = 0; e < kMostDrafts; ++e) {
                const int other = __builtin_amdgcn_readlane(depth, e);
                if (depth - other >= a.window && w.past + other >= a.sinks) s.drafts &= ~(1ull << e);
            }
        sights[lane] = s;
        if (lane == 0) *odd_met = 0;
    }
    int draft[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) draft[b] = static_cast<int>(static_cast<unsigned>(row0 + min(b * 16 + col, mine - 1)) / static_cast<unsigned>(a.group));
    __syncthreads();
    // Context that all drafts see, from here to `past`.
    const int clear_from = a.window ? max(w.past + min(w.drafts, kMostDrafts) - a.window, 0) : 0;

    floatx4 acc[NB][C::DT];
    float base[NB], l[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        base[b] = kBase0, l[b] = 0.0f;
#pragma unroll
        for (int i = 0; i < C::DT; ++i) acc[b][i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    bool met = false;
    // K of the next step is asked for as soon as this step's has been used, V
    // likewise, so a wave always has about a step of the cache in flight.
    for (int step = from; step < to; ++step) {
#pragma clang fp contract(off)  // a score less the base: of the score as it was when the base was taken
        const int j = w.token(step);
        floatx4 dot[NB][2];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            half8 kf[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                if constexpr (C::BYTES == 2) kf[t] = __builtin_bit_cast(half8, k[t][s]);
                else kf[t] = eight<KIND>(k[t][s >> 1][2 * (s & 1)], k[t][s >> 1][2 * (s & 1) + 1]);
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                half8 qf;
                if constexpr (NB == 1) qf = q[s];
                else qf = __builtin_bit_cast(half8, queries[(s * NB + b) * 64 + lane]);
#pragma unroll
                for (int t = 0; t < 2; ++t) dot[b][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[t], qf, s ? dot[b][t] : floatx4{}, 0, 0, 0);
            }
        }
        float factor[8], scale[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            factor[e] = KIND == MLVC_KV_F16 ? a.scale2 : ks[e >> 2][e & 3] * a.scale2;
            scale[e] = KIND == MLVC_KV_F16 ? 1.0f : __builtin_elementwise_maximum(vs[e >> 2][e & 3], 0x1p-40f);
        }
        const bool masked = j + kStep > w.past || !there[0] || !there[1] || (j < clear_from && j + kStep > w.sinks);
        const bool here[2] = {there[0], there[1]};
        if (step + 1 < to) {
            locate(w.token(step + 1));
            fetch_k();
        }
        if (masked) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool gone = !here[e >> 2] || j + 16 * (e >> 2) + 4 * g + (e & 3) >= w.length;
                if constexpr (KIND == MLVC_KV_F16) {
#pragma unroll
                    for (int i = 0; i < C::VW; ++i) {
                        const std::uint32_t x = v[e][i], odd = ((x & 0x7c00u) == 0x7c00u ? 0xffffu : 0u) | ((x & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u);
                        met |= !gone && odd;
                        v[e][i] = gone ? 0u : x & ~odd;
                    }
                } else {
                    if (gone) scale[e] = 1.0f;
#pragma unroll
                    for (int i = 0; i < C::VW; ++i) v[e][i] = gone || scale[e] != scale[e] ? 0u : v[e][i];
                }
            }
        }
        half8 weights[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float x[8], p[8], wt[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = dot[b][e >> 2][e & 3] * factor[e];
            unsigned unseen = 0;
            if (masked) {
                const Sight sight = sights[draft[b]];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int at = j + 16 * (e >> 2) + 4 * g + (e & 3);
                    if (!here[e >> 2] || at >= w.length || !sight(at)) unseen |= 1u << e, x[e] = -INFINITY;
                }
            }
            auto weigh = [&] {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    p[e] = __builtin_amdgcn_exp2f(x[e] - base[b]);
                    wt[e] = KIND == MLVC_KV_F16 ? p[e] : p[e] * scale[e];
                }
                if (KIND != MLVC_KV_F16 && masked) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (unseen >> e & 1) wt[e] = 0.0f;
                }
            };
            weigh();
            float top = fmaxf(wt[0], wt[1]);
#pragma unroll
            for (int e = 2; e < 8; ++e) top = fmaxf(top, wt[e]);
            if (__any(top > 0x1p15f)) {
                top = -INFINITY;
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, KIND == MLVC_KV_F16 ? x[e] : x[e] + __builtin_amdgcn_logf(scale[e]));
                const float now = fmaxf(base[b], lifted(column_max(top))), keep = __builtin_amdgcn_exp2f(base[b] - now);
                l[b] *= keep;
#pragma unroll
                for (int i = 0; i < C::DT; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[b][i][r] *= keep;
                base[b] = now;
                weigh();
            }
            float sum[2] = {p[0] + p[1], p[2] + p[3]};
            sum[0] += p[4] + p[5], sum[1] += p[6] + p[7];
            l[b] += sum[0] + sum[1];
#pragma unroll
            for (int e = 0; e < 8; ++e) weights[b][e] = static_cast<_Float16>(wt[e]);
        }
#pragma unroll
        for (int i = 0; i < C::VW; ++i) {
            std::uint32_t pair[4][C::PER];
#pragma unroll
            for (int e = 0; e < 4; ++e) columns<KIND>(v[2 * e][i], v[2 * e + 1][i], pair[e]);
#pragma unroll
            for (int c = 0; c < C::PER; ++c) {
                const half8 vf = __builtin_bit_cast(half8, u32x4{pair[0][c], pair[1][c], pair[2][c], pair[3][c]});
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    floatx4& o = acc[b][i * C::PER + c];
                    o = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, weights[b], o, 0, 0, 0);
                }
            }
        }
        if (step + 1 < to) fetch_v();
    }
    if (KIND == MLVC_KV_F16 && met) *odd_met = 1;

    // Join the waves, 16 rows at a time. A lane holds, of its column's row, the values (4 g + r) * DT + i.
    float* const joint = reinterpret_cast<float*>(lds);
    float* const st = joint + WAVES * 16 * D;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        if (b * 16 >= mine) break;
        __syncthreads();
        const float total_l = column_sum(l[b]);
        float* o = joint + (wave * 16 + col) * D;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < C::DT; i += 4)
                *reinterpret_cast<floatx4*>(o + (4 * g + r) * C::DT + i) = floatx4{acc[b][i][r], acc[b][i + 1][r], acc[b][i + 2][r], acc[b][i + 3][r]};
        if (g == 0) st[wave * 16 + col] = base[b], st[(WAVES + wave) * 16 + col] = total_l;
        __syncthreads();
        for (int i = threadIdx.x; i < min(16, mine - b * 16) * (D / 4); i += WAVES * 64) {
            const int r = i / (D / 4), d = i % (D / 4) * 4, at = row0 + b * 16 + r;
            float top = kBase0, total = 0.0f;
#pragma unroll
            for (int n = 0; n < WAVES; ++n) top = fmaxf(top, st[n * 16 + r]);
            floatx4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int n = 0; n < WAVES; ++n) {
                const float f = __builtin_amdgcn_exp2f(st[n * 16 + r] - top);
                total += st[(WAVES + n) * 16 + r] * f;
                const floatx4 x = *reinterpret_cast<const floatx4*>(joint + (n * 16 + r) * D + d);
#pragma unroll
                for (int c = 0; c < 4; ++c) sum[c] = fmaf(x[c], f, sum[c]);
            }
            const int of = static_cast<int>(static_cast<unsigned>(at) / static_cast<unsigned>(a.group));
            if constexpr (KIND == MLVC_KV_F16)
                if (*odd_met || !is_finite(sum[0]) || !is_finite(sum[1]) || !is_finite(sum[2]) || !is_finite(sum[3]))
                    decide_odd(a, w, sights[of], stream, head, first, last, d, sum);
            if (whole) {
                const float f = total == 0.0f ? 0.0f : 1.0f / total;
                *reinterpret_cast<uint2*>(a.out + (w.start + of) * a.out_stride + static_cast<std::int64_t>(head * a.group + at - of * a.group) * D + d) =
                    make_uint2(pack_rounded(sum[0] * f, sum[1] * f), pack_rounded(sum[2] * f, sum[3] * f));
            } else {
                const std::int64_t slot = (static_cast<std::int64_t>(head) * a.longest_q * a.group + at) * (2 * a.shares + a.streams) + place;
                *reinterpret_cast<floatx4*>(a.part + slot * D + d) = sum;
                if (d == 0) a.state[slot] = make_float2(top, total);
            }
        }
    }
}

// Workgroups of neighbouring numbers take the same tokens of different key
// heads, which lie side by side in a page; those of the blocks of one head's
// rows run on one XCD, whose L2 they share, one after the other.
template <class C, bool SHARES>
__global__ __launch_bounds__(C::WAVES * 64, C::OCC) void drafts_kernel(DraftArgs a)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ Sight sights[kMostDrafts];
    __shared__ int odd_met;
    const int turn = blockIdx.x / kXcds, block = turn % a.blocks, item = a.blocks == 1 ? blockIdx.x : turn / a.blocks * kXcds + blockIdx.x % kXcds;
    const int head = item % a.heads, rest = item / a.heads;
    if constexpr (SHARES)
        each_piece(a, rest, [&](int stream, int first, int last, bool whole, int place) {
            draft_piece<C>(a, lds, sights, &odd_met, head, block, stream, View(a, stream), first, last, whole, place);
            __syncthreads();  // before the next piece's queries and states
        });
    else if (rest < a.streams) {
        const View w(a, rest);
        draft_piece<C>(a, lds, sights, &odd_met, head, block, rest, w, 0, w.steps, true, 0);
    }
}

// Puts the parts of ROWS rows of a stream and key head together: LANES threads
// hold a part's row, four values each, and GROUPS of them take every GROUPS-th
// part, each with a base of its own; they are put together in LDS.
template <int LANES, int ROWS, int GROUPS>
__global__ __launch_bounds__(LANES* ROWS* GROUPS) void drafts_join_kernel(DraftArgs a, int row_blocks)
{
    __shared__ floatx4 sums[GROUPS][ROWS][LANES];
    __shared__ float2 states[GROUPS][ROWS];
    constexpr float kBase0 = -3.402823466e38f;
    const int lane = threadIdx.x & 63, row_block = blockIdx.x % row_blocks, rest = blockIdx.x / row_blocks, head = rest % a.heads, stream = rest / a.heads;
    const int at = threadIdx.x % LANES, r = threadIdx.x / LANES % ROWS, group = threadIdx.x / (LANES * ROWS);
    const View w(a, stream);
    const int row = row_block * ROWS + r, rows = w.queries * a.group;
    if (row_block * ROWS >= rows) return;
    int total = 0, start = 0;
    for (int b = 0; b < a.streams; b += 64) {
        const int mine = b + lane < a.streams ? View(a, b + lane).steps : 0;
        if (b + lane < stream) start += mine;
        total += mine;
    }
    total = wave_sum(total), start = wave_sum(start);
    const Shares shares(a.shares, total, a.spare);
    const int first = w.steps ? shares.holder(start) : 0, parts = w.steps ? shares.holder(start + w.steps - 1) - first + 1 : 0;
    if (parts == 1) return;  // written by the share that holds it
    const std::int64_t slot = (static_cast<std::int64_t>(head) * a.longest_q * a.group + row) * (2 * a.shares + a.streams) + first + stream;
    const int d = at * 4;
    float base = kBase0, l = 0.0f;
    floatx4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    if (row < rows) {
#pragma unroll 4
        for (int i = group; i < parts; i += GROUPS) {
            const floatx4 v = *reinterpret_cast<const floatx4*>(a.part + (slot + i) * a.dim + d);
            const float2 st = a.state[slot + i];
            const float now = fmaxf(base, st.x), old = __builtin_amdgcn_exp2f(base - now), f = __builtin_amdgcn_exp2f(st.x - now);
            base = now;
            l = l * old + st.y * f;
#pragma unroll
            for (int c = 0; c < 4; ++c) sum[c] = sum[c] * old + v[c] * f;
        }
    }
    sums[group][r][at] = sum;
    if (at == 0) states[group][r] = make_float2(base, l);
    __syncthreads();
    if (group != 0 || row >= rows) return;
    float top = kBase0;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) top = fmaxf(top, states[i][r].x);
    l = 0.0f;
    sum = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
        const float2 st = states[i][r];
        const float f = __builtin_amdgcn_exp2f(st.x - top);
        l += st.y * f;
#pragma unroll
        for (int c = 0; c < 4; ++c) sum[c] = fmaf(sums[i][r][at][c], f, sum[c]);
    }
    // A part that is infinite, with however small a weight.
    if (!is_finite(sum[0]) || !is_finite(sum[1]) || !is_finite(sum[2]) || !is_finite(sum[3])) {
        floatx4 odd = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int i = 0; i < parts; ++i) {
            const floatx4 v = *reinterpret_cast<const floatx4*>(a.part + (slot + i) * a.dim + d);
#pragma unroll
            for (int c = 0; c < 4; ++c) odd[c] += is_finite(v[c]) ? 0.0f : v[c];
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) sum[c] = is_finite(sum[c]) ? sum[c] : odd[c];
    }
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
    const int of = static_cast<int>(static_cast<unsigned>(row) / static_cast<unsigned>(a.group));
    *reinterpret_cast<uint2*>(a.out + (w.start + of) * a.out_stride + static_cast<std::int64_t>(head * a.group + row - of * a.group) * a.dim + d) =
        make_uint2(pack_rounded(sum[0] * f, sum[1] * f), pack_rounded(sum[2] * f, sum[3] * f));
}

// How a call is laid out; from what the host knows.
struct Plan {
    int nb, blocks, shares;
    bool fast, spare;
    std::int64_t row_count;  // rows of all key heads
    size_t part_bytes, bytes;
};

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

// Whether a context goes to one workgroup, without a cut.
bool whole(std::int64_t longest, std::int64_t workgroups)
{
    const std::int64_t cus = conv::cu_count();
    return longest <= 1024 || (longest <= 2048 && 2 * workgroups >= cus) || (longest <= 4096 && workgroups >= 3 * cus);
}

Plan plan(const mlvc_hip_attention_drafts_desc* d)
{
    Plan p{};
    const mlvc_hip_kv_cache* c = d->cache;
    const std::int64_t rows = static_cast<std::int64_t>(d->longest_q) * (d->q_heads / c->heads), blocks = (rows + 15) / 16;
    p.row_count = rows * c->heads;
    p.fast = c->head_dim == 64 || c->head_dim == 128;
    p.nb = blocks <= 1 ? 1 : blocks == 2 ? 2 : 4;
    p.blocks = static_cast<int>((blocks + p.nb - 1) / p.nb);
    p.spare = p.nb == 1;
    if (!p.fast) return p;
    // Tokens that a stream's drafts see at most, and those beside them in their steps.
    std::int64_t longest = d->longest;
    if (d->window) longest = std::min(longest, static_cast<std::int64_t>(d->window) + kMostDrafts + std::min(d->sinks, d->longest) + 2 * kStep);
    if (longest <= 1024) return p;
    const std::int64_t of_stream = static_cast<std::int64_t>(c->heads) * p.blocks;
    const int shares = static_cast<int>(std::max<std::int64_t>(1, (p.nb == 1 ? 3 : 1) * conv::cu_count() / of_stream));
    const size_t slots = (2 * static_cast<size_t>(shares) + d->streams) * p.row_count;
    p.part_bytes = slots * c->head_dim * sizeof(float);
    // Asked for whether this call cuts or not, so that what is enough for a
    // batch is enough for a smaller one.
    p.bytes = p.part_bytes + slots * sizeof(float2);
    if (!whole(longest, d->streams * of_stream)) p.shares = shares;
    return p;
}

template <class C, bool SHARES>
void launch_drafts(const DraftArgs& a, unsigned grid, hipStream_t s)
{
    drafts_kernel<C, SHARES><<<grid, C::WAVES * 64, C::LDS, s>>>(a);
}

template <int KIND, int D>
void launch_drafts(const DraftArgs& a, int nb, unsigned grid, hipStream_t s)
{
    if (a.shares) {
        if (nb == 1) launch_drafts<DraftCfg<KIND, D, 1, 4, 3>, true>(a, grid, s);
        else if (nb == 2) launch_drafts<DraftCfg<KIND, D, 2, 8, 2>, true>(a, grid, s);
        else launch_drafts<DraftCfg<KIND, D, 4, D == 64 ? 8 : 4, D == 64 ? 2 : 1>, true>(a, grid, s);
    } else {
        if (nb == 1) launch_drafts<DraftCfg<KIND, D, 1, 8, 2>, false>(a, grid, s);
        else if (nb == 2) launch_drafts<DraftCfg<KIND, D, 2, 8, 2>, false>(a, grid, s);
        else launch_drafts<DraftCfg<KIND, D, 4, D == 64 ? 8 : 4, D == 64 ? 2 : 1>, false>(a, grid, s);
    }
}

template <int KIND>
void launch_drafts(const DraftArgs& a, const Plan& p, bool fast, unsigned grid, hipStream_t s)
{
    if (!fast) drafts_any_kernel<KIND><<<grid, 64, 0, s>>>(a);
    else if (a.dim == 64) launch_drafts<KIND, 64>(a, p.nb, grid, s);
    else launch_drafts<KIND, 128>(a, p.nb, grid, s);
}

template <int LANES>
void launch_join(const DraftArgs& a, hipStream_t s)
{
    // A row for 256 threads where there are few, eight rows where there are many.
    const int rows = a.longest_q * a.group;
    const std::int64_t all = static_cast<std::int64_t>(rows) * a.heads * a.streams;
    if (all > 4096) {
        const int blocks = (rows + 7) / 8;
        drafts_join_kernel<LANES, 8, 1><<<static_cast<unsigned>(static_cast<std::int64_t>(blocks) * a.heads * a.streams), LANES * 8, 0, s>>>(a, blocks);
    } else {
        drafts_join_kernel<LANES, 1, 256 / LANES><<<static_cast<unsigned>(all), 256, 0, s>>>(a, rows);
    }
    check(hipGetLastError(), "attention_drafts join launch");
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
    Plan p = plan(d);
    const bool fast = p.fast && vector_rows(d->q, d->q_stride) && vector_rows(d->out, d->out_stride);
    if (!fast) p.shares = 0;
    const std::int64_t all_rows = static_cast<std::int64_t>(d->streams) * p.row_count;
    std::int64_t grid = all_rows;
    if (fast) {
        const std::int64_t items = static_cast<std::int64_t>(d->cache->heads) * (p.shares ? (p.spare ? 2 : 1) * p.shares : d->streams);
        grid = p.blocks == 1 ? items : (items + kXcds - 1) / kXcds * kXcds * p.blocks;
    }
    require(launchable(grid, fast ? 512 : 64) && launchable(all_rows, 256) &&
                static_cast<std::int64_t>(d->streams) * (d->longest / kStep + 2) <= INT_MAX, op,
            "too many streams, heads and drafts in one call");
    require(p.bytes == 0 || (d->workspace && d->workspace_bytes >= p.bytes && aligned16(d->workspace)), op,
            "the workspace is missing, too small or not 16-byte aligned");

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
    a.part = static_cast<float*>(d->workspace);
    a.state = reinterpret_cast<float2*>(static_cast<char*>(d->workspace) + p.part_bytes);
    a.shares = p.shares, a.blocks = p.blocks, a.spare = p.spare;
    const unsigned n = static_cast<unsigned>(grid);
    if (c->kind == MLVC_KV_F16) launch_drafts<MLVC_KV_F16>(a, p, fast, n, s);
    else if (c->kind == MLVC_KV_E4M3) launch_drafts<MLVC_KV_E4M3>(a, p, fast, n, s);
    else launch_drafts<MLVC_KV_INT8>(a, p, fast, n, s);
    check(hipGetLastError(), "attention_drafts launch");
    if (!p.shares) return;
    if (a.dim == 64) launch_join<16>(a, s);
    else launch_join<32>(a, s);
}

}  // namespace
}  // namespace mlvc_hip

using namespace mlvc_hip;

extern "C" {

size_t mlvc_hip_attention_drafts_workspace_bytes(const mlvc_hip_attention_drafts_desc* desc)
{
    size_t bytes = 0;
    guard([&] {
        check_desc(desc, "attention_drafts");
        bytes = plan(desc).bytes;
    });
    return bytes;
}

int mlvc_hip_attention_drafts(const mlvc_hip_attention_drafts_desc* desc, mlvc_hip_stream s)
{
    return guard([&] { attention_drafts(desc, to_stream(s)); });
}

}  // extern "C"
