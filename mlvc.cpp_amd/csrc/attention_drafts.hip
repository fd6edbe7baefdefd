// Attention of each stream's last tokens (drafts that form a tree, or one
// token) on its paged, quantised context, under a window.
//
//   out_i = sum_{j in V(i)} softmax_j(scale q_i . k_j) v_j
//
// V(i) holds the context's places j with place_i - j < window or j < sinks, and
// the drafts of i's mask, at places past + depth, by the same rule. depth is the
// number of other drafts that a draft sees.
//
// Bound by the bytes of the cache while a key head has few rows (drafts times the
// query heads that share it): 64 streams of one token under a window of 4080, 32
// query heads on 8 of 128, E4M3, 0.51 GB in 111 us or 4.6 TB/s. From 64 rows on
// by what is computed for a cached row, its unpacking and the softmax: 64 streams
// of 16 drafts on up to 8160 tokens, INT8, 0.57 GB and 69 GFLOP in 170 us, vector
// units busy 50% of the time and matrix cores 20%, the rest waits for LDS and for
// products that follow from each other; 64 of 64 drafts 275 GFLOP in 462 us. One
// token under a window of 920 is a launch and the latency of four steps, 9.0 us.

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
    const std::int32_t* placed;  // drafts of a stream in the cache; any array where all are
    int all_placed;              // INT_MAX: all are; 0
    int table_stride, pages, page, heads, q_heads, group, dim, longest, longest_q, q_tokens, streams, window, sinks;
    float scale2;
    float* part;    // [heads][rows][places][dim], a row for each draft and query head of a group
    float2* state;  // [heads][rows][places]: base, l
    int places;     // of a row's parts: shares and streams
    int shares;     // workgroups of a key head and a block of rows that the GPU holds at once; 0: a context goes to one workgroup
    int blocks;     // of rows
    bool spare;     // small shares behind the large ones
};

// The first place that a token at `place` sees under a window.
__device__ __forceinline__ int first_seen(int place, int window) { return place >= window ? place - window + 1 : 0; }

// A stream's context. Its steps: those that hold sinks, then those from the
// window's first token on.
struct View {
    int start, drafts, queries;  // first row of q; drafts in the cache; rows that are computed
    int past, length;            // place of the first draft; tokens in the cache
    int sinks, sink_steps, skipped, steps;
    __device__ View(const DraftArgs& a, int stream)
    {
        const int begin = a.starts[stream], end = a.starts[stream + 1];
        const int placed = max(a.placed[stream], a.all_placed);  // no branch: the four are asked for together
        int tokens = a.lengths[stream];
        const std::int64_t held = static_cast<std::int64_t>(a.table_stride) * a.page;
        start = min(max(begin, 0), a.q_tokens);
        drafts = min(max(end - begin, 0), placed);
        queries = min(min(drafts, a.longest_q), a.q_tokens - start);
        tokens = max(tokens, 0);
        past = tokens - drafts;
        length = static_cast<int>(min(static_cast<std::int64_t>(min(tokens, a.longest)), held));
        const int first = a.window ? first_seen(past, a.window) / kStep : 0;
        sinks = a.window ? min(a.sinks, length) : 0;
        sink_steps = steps_for(sinks);
        const int all = steps_for(length);
        skipped = max(min(first, all) - sink_steps, 0);
        steps = queries > 0 ? all - skipped : 0;
    }
    // First token of a step.
    __device__ int token(int step) const { return (step < sink_steps ? step : step + skipped) * kStep; }
    // Whether all drafts see all of the step at token j, if its tiles are there: context before the drafts and the
    // cut (clear_to), from the window's edge on (clear_from) or among the sinks.
    __device__ bool clear(int j, int clear_from, int clear_to) const { return clear_to - j >= kStep && (j >= clear_from || sinks - j >= kStep); }
};

// What a draft sees.
struct Sight {
    int from, sinks, past;  // context from `from` on, and before `sinks`
    unsigned long long drafts;
    __device__ bool operator()(int j) const
    {
        return j < past ? j >= from || j < sinks : j - past < kMostDrafts && (drafts >> (j - past) & 1);
    }
    // Of the 32 tokens from j on, one a bit; those before `length` that are there.
    __device__ __forceinline__ unsigned step(int j, int length, bool here0, bool here1) const
    {
        auto below = [&](int end) { return end <= j ? 0u : end - j >= 32 ? ~0u : (1u << (end - j)) - 1; };
        const unsigned context = (~below(from) | below(sinks)) & below(past);
        const unsigned long long later = past - j >= 64 ? 0 : past >= j ? drafts << (past - j) : j - past >= 64 ? 0 : drafts >> (j - past);
        return (context | (static_cast<unsigned>(later) & ~below(past))) & below(length) & (here0 ? ~0u : 0xffff0000u) & (here1 ? ~0u : 0xffffu);
    }
};

// Largest score and logarithm of its row's scale of a lane's N, for the base. FP32
// numbers of 2^28 and more are 32 and more apart: there a sum that falls so far below
// the exact one that the weight, 2^(score - sum) scale, would not fit FP16 gives way to
// the score, which is above the exact one (scales of 2^15 and more do not come from
// FP16 rows).
template <int KIND, int N>
__device__ __forceinline__ float largest(const float (&x)[N], const float (&scale)[N])
{
#pragma clang fp contract(off) reassociate(off)
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, KIND == MLVC_KV_F16 ? x[i] : x[i] + __builtin_amdgcn_logf(scale[i]));
    if constexpr (KIND != MLVC_KV_F16)
        if (__builtin_expect(__any(fabsf(top) >= 0x1p28f && is_finite(top)), false)) {
            top = -INFINITY;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float log = __builtin_amdgcn_logf(scale[i]), sum = x[i] + log;
                top = fmaxf(top, x[i] - sum + log > kMost ? x[i] : sum);
            }
        }
    return top;
}

// Masks and depths of a stream's drafts, one a lane.
__device__ __forceinline__ unsigned long long mask_of(const DraftArgs& a, const View& w, int draft)
{
    const int count = min(w.drafts, a.longest_q);  // those behind are seen by none
    const unsigned long long there = count < 64 ? (1ull << count) - 1 : ~0ull;
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

// Heads of more than 256 values and cached rows that are no whole 16-byte pieces
// (8-bit heads of 8, 24, 40, ...): one wave for a piece of a context and a draft's query head, 64
// tokens at a time, one token a lane for the scores and one value column a lane
// for the sum.
template <int KIND>
__global__ __launch_bounds__(64) void drafts_any_kernel(DraftArgs a)
{
    __shared__ float qs[kMaxHeadDim], ps[64];
    __shared__ long long at[64];
    const int rows = a.longest_q * a.group, row_of_head = blockIdx.x % rows, draft = row_of_head / a.group;
    const int lane = threadIdx.x, rest = blockIdx.x / rows, kv_head = rest % a.heads, head = kv_head * a.group + row_of_head - draft * a.group;
    constexpr int kColumns = kMaxHeadDim / 64;
    constexpr float kBase0 = -3.402823466e38f;
    auto value = [&](const std::uint8_t* x, long long row, int d) {
        if constexpr (KIND == MLVC_KV_F16) return h2f(reinterpret_cast<const std::uint16_t*>(x)[row * a.dim + d]);
        else return from_byte(KIND, x[row * a.dim + d]);
    };
    auto piece = [&](int stream, int first, int last, bool whole, int place) {
        const View w(a, stream);
        if (draft >= w.queries) return;
        Sight sight;
        {
            const unsigned long long mine = mask_of(a, w, lane), mask = __shfl(mine, draft);
            const int depth = depth_of(mine, lane), depth_i = __shfl(depth, draft);
            sight.past = w.past;
            sight.from = a.window ? first_seen(w.past + depth_i, a.window) : 0;
            sight.sinks = w.sinks;
            sight.drafts = mask & __ballot(!a.window || depth_i - depth < a.window || w.past + depth < a.sinks);
        }
        const std::int64_t token = w.start + draft;
        const std::uint16_t* q = a.q + token * a.q_stride + static_cast<std::int64_t>(head) * a.dim;
        for (int d = lane; d < a.dim; d += 64) qs[d] = h2f(q[d]) * a.scale2;
        __syncthreads();
        float acc[kColumns] = {}, m = -INFINITY, l = 0.0f;
        for (int step = first; step < last; step += 2) {
            const int mine = step + lane / kStep, j = mine < last ? w.token(mine) + lane % kStep : w.length;
            const long long row = j < w.length && sight(j) ? token_row(a, stream, kv_head, j) : -1;
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
                for (int step = first; step < last; ++step)
                    for (int j = w.token(step), i = 0; i < kStep && j < w.length; ++i, ++j) {
                        const std::int64_t row = sight(j) ? token_row(a, stream, kv_head, j) : -1;
                        if (row >= 0) odd.add(reinterpret_cast<const std::uint16_t*>(a.v)[row * a.dim + d]);
                    }
                acc[c] = odd.sum(acc[c]);
            }
        }
        if (whole) {
            const float r = l == 0.0f ? 0.0f : 1.0f / l;
            std::uint16_t* out = a.out + token * a.out_stride + static_cast<std::int64_t>(head) * a.dim;
#pragma unroll
            for (int c = 0; c < kColumns; ++c)
                if (c * 64 + lane < a.dim) out[c * 64 + lane] = f2h(opaque(acc[c] * r));
            return;
        }
        const std::int64_t slot = (static_cast<std::int64_t>(kv_head) * rows + row_of_head) * a.places + place;
#pragma unroll
        for (int c = 0; c < kColumns; ++c)
            if (c * 64 + lane < a.dim) a.part[slot * a.dim + c * 64 + lane] = acc[c];
        if (lane == 0) a.state[slot] = make_float2(m == -INFINITY ? kBase0 : m, l);
        __syncthreads();  // before the next piece's query
    };
    const int item = rest / a.heads;
    if (a.shares) each_piece(a, item, piece);
    else piece(item, 0, View(a, item).steps, true, 0);
}

// ------------------------------------------------------------ matrix cores

// Rows of the cache of a stream's tiles of 16 tokens (each in one page), those of
// 64 tiles at a time, one a lane: the table is read once for 32 steps, and no
// step waits for it.
struct Tiles {
    const DraftArgs& a;
    const View& w;
    int stream, head, first = -64;
    std::int64_t mine = -1;
    __device__ Tiles(const DraftArgs& a_, const View& w_, int stream_, int head_) : a(a_), w(w_), stream(stream_), head(head_) {}
    // Of the tiles of a step, from its first token on; -1 for one that is not there.
    __device__ __forceinline__ void find(int token, std::int64_t* row)
    {
        const int tile = token / 16;
        if (static_cast<unsigned>(tile - first) >= 64u) {
            first = tile;
            const int ahead = 16 * static_cast<int>(threadIdx.x & 63);
            mine = ahead < w.length - token ? token_row(a, stream, head, token + ahead) : -1;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int lane = tile + t - first;
            row[t] = static_cast<std::int64_t>(static_cast<unsigned long long>(static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(mine >> 32), lane))) << 32 |
                                               static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(mine), lane)));
        }
    }
};

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
// An RNE narrowing of a weight that is kept as two halves, as attention of single
// tokens has it, would double the products of V, which here are many.
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
    static_assert(NB <= 2);
    static constexpr size_t LDS = (WAVES * 16 * D + 2 * WAVES * 16) * sizeof(float);
    static_assert(NB == 1 || KS * NB * 1024 <= LDS);
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
    // Rows of the two tiles of a step, row 0 for a tile that is not there.
    Tiles tiles(a, w, stream, head);
    std::int64_t row[2];
    bool there[2];
    auto locate = [&](int j) {
        tiles.find(j, row);
#pragma unroll
        for (int t = 0; t < 2; ++t) there[t] = row[t] >= 0, row[t] = there[t] ? row[t] : 0;
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
        for (int i = threadIdx.x; i < KS * NB * 64; i += WAVES * 64) queries[i] = query(i >> 6 & 1, i >> 7, i & 63);
    }
    if (wave == 0) {
        const unsigned long long mask = mask_of(a, w, lane);
        const int depth = depth_of(mask, lane);
        Sight s;
        s.past = w.past, s.sinks = w.sinks;
        s.from = a.window ? first_seen(w.past + depth, a.window) : 0;
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
    // Context that all drafts see.
    const int clear_to = min(w.past, w.length), clear_from = a.window ? max(w.past + min(w.drafts, kMostDrafts) - a.window, 0) : 0;

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
        const bool masked = !there[0] || !there[1] || !w.clear(j, clear_from, clear_to);
        const bool here[2] = {there[0], there[1]};
        // The last step asks for itself again: so that there are always as many loads,
        // and the wait for K leaves V on its way.
        locate(w.token(min(step + 1, to - 1)));
        fetch_k();
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
            unsigned see = ~0u;
            if (masked) {
                see = sights[draft[b]].step(j, w.length, here[0], here[1]) >> 4 * g;
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = see >> (16 * (e >> 2) + (e & 3)) & 1 ? x[e] : -INFINITY;
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
                        wt[e] = see >> (16 * (e >> 2) + (e & 3)) & 1 ? wt[e] : 0.0f;
                }
            };
            weigh();
            float top = fmaxf(wt[0], wt[1]);
#pragma unroll
            for (int e = 2; e < 8; ++e) top = fmaxf(top, wt[e]);
            if (__any(top > 0x1p15f)) {
                const float now = fmaxf(base[b], lifted(column_max(largest<KIND>(x, scale)))), keep = __builtin_amdgcn_exp2f(base[b] - now);
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
        fetch_v();
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
                const std::int64_t slot = (static_cast<std::int64_t>(head) * a.longest_q * a.group + at) * a.places + place;
                *reinterpret_cast<floatx4*>(a.part + slot * D + d) = sum;
                if (d == 0) a.state[slot] = make_float2(top, total);
            }
        }
    }
}

// More rows than 32: RG x KG waves take RG * 32 rows. The KG groups of waves take
// every KG-th step of the part, and put their states together at the end. The
// waves of a group unpack the step's rows of the cache to halves in LDS, once for
// all of them, while the next step's are on their way to registers; each wave
// holds 32 rows as columns of S^T = K Q^T (32x32x16 products, keys as rows), so
// that a lane's scores all belong to one row, and rounded to halves they are the
// B operand of O^T += V^T P^T as they stand. 16-byte pieces of a row are permuted
// in LDS against bank conflicts; V is read transposing. 8-bit steps are asked for
// two ahead, FP16 ones, twice as large, one ahead. Three workgroups a CU instead of
// two, on one buffer and one step ahead, spill with heads of 128 and took 107
// instead of 111 us at 64 streams of 16 drafts, heads of 64.
//
// PAD: heads of up to D values, with zeros behind them in LDS, and rows of q and
// out of any alignment; the cache's rows are whole 16-byte pieces. us of a call,
// and of one wave for each row, value by value, as other rows are taken:
//   1 x 16 on 65280, E4M3, 32 / 8 heads of 96     67.8   8720
//                                    of 256        149  31900
//   64 x 16 on 16 to 8160, INT8, heads of 96       181  17400
//   16 x 64 on 920 to 3001, FP16, 16 heads of 96  62.8   4050
//   1 x 1, a window of 920, INT8, heads of 96     24.9    272
// Heads of more than 128 leave one wave a SIMD, of up to 512 registers, with steps
// one ahead (two ahead spill twice as many registers).
template <int KIND_, int D_, int RG_, int KG_, bool PAD_ = false>
struct TileCfg {
    static constexpr int KIND = KIND_, D = D_, RG = RG_, KG = KG_, WAVES = RG * KG, ROWS = RG * 32, OCC = D > 128 ? 1 : 2;
    static constexpr bool PAD = PAD_;
    static constexpr int BYTES = KIND == MLVC_KV_F16 ? 2 : 1;
    static constexpr int TILE = kStep * D;                     // halves of K or V of a step
    static constexpr int LOADS = 2 * kStep * D * BYTES / 1024; // of a wave, for K and V of a step
    static constexpr int MINE = (LOADS + RG - 1) / RG;         // of each wave of a group
    static constexpr int DEPTH = KIND == MLVC_KV_F16 || D > 128 ? 1 : 2;  // steps on their way
    static constexpr int WORDS = D / 8 + 1;                    // 16-byte words of a lane's state
    static constexpr size_t TILES = KG * 2 * 2 * TILE * 2, SCALES = KG * 2 * 2 * kStep * sizeof(float),
                            JOINT = static_cast<size_t>(KG - 1) * WORDS * RG * 64 * 16;
    static constexpr size_t LDS = TILES + SCALES > JOINT ? TILES + SCALES : JOINT;
    // Place of a 16-byte piece of row t, so that 16 rows of one piece (a K read) fall
    // on all 64 banks, 4 rows of 4 pieces (a V read) do too, and the pieces that
    // eight lanes write at once on 32 of them: every one of a row of halves, every
    // other one of unpacked bytes (in the order of the pieces those took 10% of the
    // cycles at 64 streams of 16 drafts).
    __host__ __device__ static constexpr int place(int piece, int t)
    {
        if (BYTES == 2) return piece ^ (D >= 128 ? 4 * (t & 3) + (t >> 2 & 3) : 4 * (t >> 1 & 1) + (t >> 2 & 3));
        const int evens_first = (piece >> 1) + (piece & 1) * (D / 16);
        return evens_first ^ (D >= 128 ? 2 * (t & 3) + (t >> 2 & 1) + 8 * (t >> 3 & 1) : 2 * (t >> 1 & 1) + (t >> 2 & 1) + 4 * ((t >> 3 ^ t) & 1));
    }
};

template <class C>
__device__ __forceinline__ void tile_piece(const DraftArgs& a, char* lds, Sight* sights, int* odd_met, int head, int block, int stream, const View& w,
                                           int first, int last, bool whole, int place)
{
    constexpr int D = C::D, KIND = C::KIND, RG = C::RG, KG = C::KG, KS = D / 16, DT = D / 32, RB = D * C::BYTES;
    const int dim = C::PAD ? a.dim : D;
    constexpr float kBase0 = -3.402823466e38f;
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rg = wave % RG, kg = wave / RG, column = lane & 31, hi = lane >> 5;
    const int rows = w.queries * a.group, row0 = block * C::ROWS, mine = min(C::ROWS, rows - row0);
    if (mine <= 0) return;
    std::uint16_t* const tiles = reinterpret_cast<std::uint16_t*>(lds) + kg * 4 * C::TILE;      // [buffer][K, V][TILE]
    float* const scales = reinterpret_cast<float*>(lds + C::TILES) + kg * 4 * kStep;            // [buffer][scale_k, scale_v][kStep]

    // A step that is on its way: its first token, whether its tiles are there, its rows as they lie in the cache.
    struct Coming {
        int j = 0;
        bool there[2] = {false, false};
        u32x4 raw[C::MINE];
        float scale = 0.0f;
    };
    Tiles table(a, w, stream, head);
    Coming coming[C::DEPTH];
    auto fetch = [&](int step, Coming& c) {
        std::int64_t row[2];
        c.j = w.token(step);
        table.find(c.j, row);
#pragma unroll
        for (int t = 0; t < 2; ++t) c.there[t] = row[t] >= 0, row[t] = c.there[t] ? row[t] : 0;
#pragma unroll
        for (int i = 0; i < C::MINE; ++i) {
            const int n = rg + i * RG;
            if (C::LOADS % RG != 0 && n >= C::LOADS) continue;
            const bool is_v = n >= C::LOADS / 2;
            const int byte = (n - (is_v ? C::LOADS / 2 : 0)) * 1024, t = byte / RB / 16;
            if constexpr (C::PAD) {  // the first piece again where there is none
                const int at = byte - t * 16 * RB + lane * 16, r = at / RB, inside = at - r * RB, rb = dim * C::BYTES;
                c.raw[i] = *reinterpret_cast<const u32x4*>((is_v ? a.v : a.k) + (t ? row[1] : row[0]) * rb + r * rb + (inside < rb ? inside : 0));
            } else {
                c.raw[i] = *reinterpret_cast<const u32x4*>((is_v ? a.v : a.k) + (t ? row[1] : row[0]) * RB + (byte - t * 16 * RB) + lane * 16);
            }
        }
        if constexpr (KIND != MLVC_KV_F16) c.scale = (hi ? a.v_scale : a.k_scale)[(lane & 16 ? row[1] : row[0]) + (lane & 15)];
    };
    // Always as many loads, the last step's again past the end: so that the wait
    // for a step leaves the next one's on their way.
    if (first < last)
#pragma unroll
        for (int i = 0; i < C::DEPTH; ++i) fetch(min(first + i * KG + kg, last - 1), coming[i]);

    if (wave == 0) {
        const unsigned long long mask = mask_of(a, w, lane);
        const int depth = depth_of(mask, lane);
        Sight s;
        s.past = w.past, s.sinks = w.sinks;
        s.from = a.window ? first_seen(w.past + depth, a.window) : 0;
        s.drafts = mask;
        if (a.window && a.window < kMostDrafts)
            for (int e = 0; e < kMostDrafts; ++e) {
                const int other = __builtin_amdgcn_readlane(depth, e);
                if (depth - other >= a.window && w.past + other >= a.sinks) s.drafts &= ~(1ull << e);
            }
        sights[lane] = s;
        if (lane == 0) *odd_met = 0;
    }
    // This lane's row: of a draft and a query head.
    const int at_row = row0 + min(rg * 32 + column, mine - 1), draft = static_cast<int>(static_cast<unsigned>(at_row) / static_cast<unsigned>(a.group));
    const bool has_rows = rg * 32 < mine, my_row = rg * 32 + column < mine;
    const std::int64_t token = w.start + draft, at_head = static_cast<std::int64_t>(head * a.group + at_row - draft * a.group) * dim;
    half8 q[KS];
    {
        const std::uint16_t* x = a.q + token * a.q_stride + at_head + hi * 8;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            if constexpr (C::PAD) {
                q[i] = half8{};
                if (i * 16 + hi * 8 >= dim) continue;
#pragma unroll
                for (int e = 0; e < 8; ++e) q[i][e] = __builtin_bit_cast(_Float16, x[i * 16 + e]);
            } else {
                q[i] = __builtin_bit_cast(half8, *reinterpret_cast<const u32x4*>(x + i * 16));
            }
        }
    }
    const int clear_to = min(w.past, w.length), clear_from = a.window ? max(w.past + min(w.drafts, kMostDrafts) - a.window, 0) : 0;

    // Places of this lane's pieces: of K, pieces 2 ks + hi of row lane & 31; of V,
    // the transposing read of 16 lanes takes 4 halves of each of 4 rows (4 hi + 8 e
    // + 0..3 of a 16-row step) a lane and returns one column's four.
    int kat[KS], vat[DT][2];
#pragma unroll
    for (int i = 0; i < KS; ++i) kat[i] = column * D + C::place(2 * i + hi, column) * 8;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = 8 * e + 4 * hi + ((lane & 15) >> 2);
            vat[dt][e] = r * D + C::place(4 * dt + 2 * (lane >> 4 & 1) + (lane >> 1 & 1), r) * 8 + (lane & 1) * 4;
        }
    floatx16 acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[dt][r] = 0.0f;
    float base = kBase0, l = 0.0f;
    bool met = false;
    __syncthreads();
    const Sight sight = sights[draft];

    // The step that came in, as halves in LDS; what rows that do not see it must
    // not meet is zeroed.
    auto unpack = [&](const Coming& c, int buffer, bool masked) {
        std::uint16_t* const tile = tiles + buffer * 2 * C::TILE;
#pragma unroll
        for (int i = 0; i < C::MINE; ++i) {
            const int n = rg + i * RG;
            if (C::LOADS % RG != 0 && n >= C::LOADS) continue;
            const bool is_v = n >= C::LOADS / 2;
            const int byte = (n - (is_v ? C::LOADS / 2 : 0)) * 1024 + lane * 16, r = byte / RB, piece = byte % RB / 16 * (2 / C::BYTES);
            std::uint16_t* const to = tile + (is_v ? C::TILE : 0) + r * D;
            const bool gone = masked && is_v && (!(r & 16 ? c.there[1] : c.there[0]) || c.j + r >= w.length);
            auto put = [&](int at, u32x4 x) {
                if (C::PAD && at * 8 >= dim) x = u32x4{0, 0, 0, 0};
                if (masked && is_v) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const std::uint32_t odd = KIND == MLVC_KV_INT8 ? 0u : ((x[e] & 0x7c00u) == 0x7c00u ? 0xffffu : 0u) | ((x[e] & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u);
                        if (KIND == MLVC_KV_F16) met |= !gone && odd;
                        x[e] = gone ? 0u : x[e] & ~odd;
                    }
                }
                *reinterpret_cast<u32x4*>(to + C::place(at, r) * 8) = x;
            };
            if constexpr (KIND == MLVC_KV_F16) {
                put(piece, c.raw[i]);
            } else {
                put(piece, __builtin_bit_cast(u32x4, eight<KIND>(c.raw[i][0], c.raw[i][1])));
                put(piece + 1, __builtin_bit_cast(u32x4, eight<KIND>(c.raw[i][2], c.raw[i][3])));
            }
        }
        if (KIND != MLVC_KV_F16 && rg == 0)
            scales[buffer * 2 * kStep + lane] = hi ? __builtin_elementwise_maximum(c.scale, 0x1p-40f) : c.scale * a.scale2;
    };
    auto compute = [&](int buffer, int j, bool masked, bool here0, bool here1) {
#pragma clang fp contract(off)  // a score less the base: of the score as it was when the base was taken
        const std::uint16_t* const tile_k = tiles + buffer * 2 * C::TILE;
        const std::uint16_t* const tile_v = tile_k + C::TILE;
        floatx16 s;
#pragma unroll
        for (int i = 0; i < KS; ++i) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const half8*>(tile_k + kat[i]), q[i], i ? s : floatx16{}, 0, 0, 0);
        float x[16], scale[16], p[16], wt[16];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            floatx4 f = {a.scale2, a.scale2, a.scale2, a.scale2}, t = {1.0f, 1.0f, 1.0f, 1.0f};
            if constexpr (KIND != MLVC_KV_F16) {
                f = *reinterpret_cast<const floatx4*>(scales + buffer * 2 * kStep + 8 * g + 4 * hi);
                t = *reinterpret_cast<const floatx4*>(scales + buffer * 2 * kStep + kStep + 8 * g + 4 * hi);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * g + e] = s[4 * g + e] * f[e], scale[4 * g + e] = t[e];
        }
        if (masked) {
            const unsigned see = sight.step(j, w.length, here0, here1) >> 4 * hi;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const bool seen = see >> (8 * (r >> 2) + (r & 3)) & 1;
                x[r] = seen ? x[r] : -INFINITY, scale[r] = seen ? scale[r] : 1.0f;
            }
        }
        auto weigh = [&] {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                p[r] = __builtin_amdgcn_exp2f(x[r] - base);
                wt[r] = KIND == MLVC_KV_F16 ? p[r] : p[r] * scale[r];
            }
        };
        weigh();
        float top = wt[0];
#pragma unroll
        for (int r = 1; r < 15; r += 2) top = fmaxf(fmaxf(top, wt[r]), wt[r + 1]);
        top = fmaxf(top, wt[15]);
        if (__any(top > 0x1p15f)) {
            const float now = fmaxf(base, lifted(both_max(largest<KIND>(x, scale)))), keep = __builtin_amdgcn_exp2f(base - now);
            l *= keep;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[dt][r] *= keep;
            base = now;
            weigh();
        }
        float sum[4] = {};
        half8 weights[2];
#pragma unroll
        for (int r = 0; r < 16; ++r) sum[r & 3] += p[r], weights[r >> 3][r & 7] = static_cast<_Float16>(wt[r]);
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                typedef short s16x4 __attribute__((ext_vector_type(4)));
                u32x2 v[2];
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    v[e] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                         (__attribute__((address_space(3))) s16x4*)(tile_v + vat[dt][e] + h * 16 * D)));
                acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, u32x4{v[0][0], v[0][1], v[1][0], v[1][1]}), weights[h], acc[dt], 0, 0, 0);
            }
    };
    const int turns = (last - first + KG - 1) / KG;
    auto take_turn = [&](int turn, Coming& c) {
        const int step = first + turn * KG + kg, buffer = turn & 1, j = c.j;
        const bool here0 = c.there[0], here1 = c.there[1];
        const bool masked = !here0 || !here1 || !w.clear(j, clear_from, clear_to);
        unpack(c, buffer, masked);
        fetch(min(step + C::DEPTH * KG, last - 1), c);
        __syncthreads();
        if (step < last && has_rows) compute(buffer, j, masked, here0, here1);
    };
    for (int turn = 0; turn < turns; turn += C::DEPTH) {
        take_turn(turn, coming[0]);
        if constexpr (C::DEPTH > 1)
            if (turn + 1 < turns) take_turn(turn + 1, coming[1]);
    }
    if (KIND == MLVC_KV_F16 && met) *odd_met = 1;

    // The other groups hand their states to the first, lane by lane.
    __syncthreads();
    l = both_sum(l);
    if constexpr (KG > 1) {
        floatx4* const states = reinterpret_cast<floatx4*>(lds) + rg * 64 + lane;
        if (kg > 0 && has_rows) {
            floatx4* const to = states + (kg - 1) * C::WORDS * RG * 64;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    to[(dt * 4 + g) * RG * 64] = floatx4{acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]};
            to[DT * 4 * RG * 64] = floatx4{base, l, 0.0f, 0.0f};
        }
        __syncthreads();
        if (kg > 0 || !has_rows) return;
#pragma unroll
        for (int n = 0; n < KG - 1; ++n) {
            const floatx4* const from = states + n * C::WORDS * RG * 64;
            const floatx4 st = from[DT * 4 * RG * 64];
            const float now = fmaxf(base, st[0]), old = __builtin_amdgcn_exp2f(base - now), f = __builtin_amdgcn_exp2f(st[0] - now);
            base = now;
            l = l * old + st[1] * f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const floatx4 v = from[(dt * 4 + g) * RG * 64];
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[dt][4 * g + e] = acc[dt][4 * g + e] * old + v[e] * f;
                }
        }
    }
    if (!my_row) return;
    if constexpr (KIND == MLVC_KV_F16) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                floatx4 v = {acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]};
                if (C::PAD && dt * 32 + 8 * g >= dim) continue;
                if (*odd_met || !is_finite(v[0]) || !is_finite(v[1]) || !is_finite(v[2]) || !is_finite(v[3])) {
                    decide_odd(a, w, sight, stream, head, first, last, dt * 32 + 8 * g + 4 * hi, v);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[dt][4 * g + e] = v[e];
                }
            }
    }
    if (whole) {
        const float f = l == 0.0f ? 0.0f : 1.0f / l;
        std::uint16_t* const out = a.out + token * a.out_stride + at_head + 4 * hi;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                if constexpr (C::PAD) {
                    if (dt * 32 + 8 * g >= dim) continue;
#pragma unroll
                    for (int e = 0; e < 4; ++e) out[dt * 32 + 8 * g + e] = f2h(opaque(acc[dt][4 * g + e] * f));
                } else {
                    *reinterpret_cast<uint2*>(out + dt * 32 + 8 * g) = make_uint2(pack_rounded(acc[dt][4 * g] * f, acc[dt][4 * g + 1] * f),
                                                                                  pack_rounded(acc[dt][4 * g + 2] * f, acc[dt][4 * g + 3] * f));
                }
    } else {
        const std::int64_t slot = (static_cast<std::int64_t>(head) * a.longest_q * a.group + at_row) * a.places + place;
        float* const part = a.part + slot * dim + 4 * hi;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                if (!C::PAD || dt * 32 + 8 * g < dim) *reinterpret_cast<floatx4*>(part + dt * 32 + 8 * g) = floatx4{acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]};
        if (hi == 0) a.state[slot] = make_float2(base, l);
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
    auto take = [&](int stream, const View& w, int first, int last, bool whole, int place) {
        if constexpr (requires { C::NB; }) draft_piece<C>(a, lds, sights, &odd_met, head, block, stream, w, first, last, whole, place);
        else tile_piece<C>(a, lds, sights, &odd_met, head, block, stream, w, first, last, whole, place);
    };
    if constexpr (SHARES)
        each_piece(a, rest, [&](int stream, int first, int last, bool whole, int place) {
            take(stream, View(a, stream), first, last, whole, place);
            __syncthreads();  // before the next piece's queries and states
        });
    else if (rest < a.streams) {
        const View w(a, rest);
        take(rest, w, 0, w.steps, true, 0);
    }
}

// Puts the parts of a stream's and key head's rows together, ROWS at a time:
// LANES threads hold a part's row, four values each, and GROUPS of them take every
// GROUPS-th part, each with a base of its own; they are put together in LDS.
// `turns` workgroups take a stream's and key head's rows by turns. ANY: heads of
// any size, rows of any alignment.
template <int LANES, int ROWS, int GROUPS, bool ANY = false>
__global__ __launch_bounds__(LANES* ROWS* GROUPS) void drafts_join_kernel(DraftArgs a, int turns)
{
    __shared__ floatx4 sums[GROUPS][ROWS][LANES];
    __shared__ float2 states[GROUPS][ROWS];
    constexpr float kBase0 = -3.402823466e38f;
    const int lane = threadIdx.x & 63, rest = blockIdx.x / turns, head = rest % a.heads, stream = rest / a.heads;
    const int at = threadIdx.x % LANES, r = threadIdx.x / LANES % ROWS, group = threadIdx.x / (LANES * ROWS);
    const View w(a, stream);
    const int rows = w.queries * a.group;
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
    for (int row0 = blockIdx.x % turns * ROWS; row0 < rows; row0 += turns * ROWS)
        for (int d = at * 4; d < (ANY ? a.dim : LANES * 4); d += LANES * 4) {
            const int row = min(row0 + r, rows - 1);
            const std::int64_t slot = (static_cast<std::int64_t>(head) * a.longest_q * a.group + row) * a.places + first + stream;
            float base = kBase0, l = 0.0f;
            floatx4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
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
            if constexpr (GROUPS > 1) {
                __syncthreads();  // the last rows' sums are read
                sums[group][r][at] = sum;
                if (at == 0) states[group][r] = make_float2(base, l);
                __syncthreads();
                if (group != 0) continue;
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
            if (row0 + r >= rows) continue;
            const float f = l == 0.0f ? 0.0f : 1.0f / l;
            const int of = static_cast<int>(static_cast<unsigned>(row) / static_cast<unsigned>(a.group));
            std::uint16_t* const out = a.out + (w.start + of) * a.out_stride + static_cast<std::int64_t>(head * a.group + row - of * a.group) * a.dim + d;
            if constexpr (ANY) {
#pragma unroll
                for (int c = 0; c < 4; ++c) out[c] = f2h(opaque(sum[c] * f));
            } else {
                *reinterpret_cast<uint2*>(out) = make_uint2(pack_rounded(sum[0] * f, sum[1] * f), pack_rounded(sum[2] * f, sum[3] * f));
            }
        }
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

// Workgroups: rows of one, and how many fit a CU.
enum Shape { kOne8, kOne4, kTwo4, kTile21, kTile22, kTile41, kTile42, kPad, kAny };
constexpr int kRows[] = {16, 16, 32, 64, 64, 128, 128, 64, 1}, kPerCu[] = {1, 3, 2, 4, 2, 2, 1, 2, 16};

// Parts of a call for each CU, at most: those of its workgroups' rows, twice where
// there are small shares behind the large ones.
constexpr int kParts = 256;
constexpr bool enough_parts()
{
    for (int i = kOne8; i <= kAny; ++i)
        if (kRows[i] * kPerCu[i] * (i == kOne4 ? 2 : 1) > kParts) return false;
    return true;
}
static_assert(enough_parts());

// How a call is laid out; from what the host knows.
struct Plan {
    Shape shape;
    int blocks, shares;
    std::int64_t row_count;  // rows of all key heads
    size_t part_bytes, bytes;
};

// Contexts of few steps go to one workgroup each, whole: by 8 waves for 16 rows
// while there are no more workgroups than CUs, then to workgroups of as many rows
// as still let all of them run at once. Others are cut into shares: for 16 rows
// while a wave has few steps, as more rows take longer to start and to join; else
// for as many as let each cached row be unpacked for all rows of a head, or for
// two workgroups of them. Shapes with more rows than 32 unpack into LDS; a CU
// holds four of two waves, which leave the most independent of each other, where
// there are enough contexts for the parts they leave not to count. us, E4M3 or
// INT8, 32 / 8 heads of 128 where not said otherwise, the one taken marked *:
//   whole                            One8  One4  Two4  Tile22
//     1 x 16 drafts, 920 tokens, 16 / 4 of 64
//                                    9.6*        14.1  19.6
//     1 x 64, 920                    14.7*       20.2  26.8
//     8 x 16, 500 to 2000            20.7*       28.8  48.7
//     16 x 16, 200 to 1000           26.7        20.4* 28.4
//     32 x 16, 500 to 2000           67.6        38.6* 50.2
//     64 x 16, 200 to 1000           96.4        48.7  38.3*
//   shares                           One4  Two4  Tile21 Tile22 Tile41 Tile42
//     1 x 16, 4000                   17.5* 17.9         20.8
//     1 x 8, 65280                   45.9  40.4* 45.4   42.8
//     1 x 16, 65280                  77.8  50.3  53.8   51.6*  64.6   68.8
//     64 x 8, 16 to 8160             165   141*  142    151    197    242
//     64 x 16, 16 to 8160            256   192   172*   179    226    263
//     16 x 64, 920 to 3001, 16 / 16 of 64, FP16
//                                    58.6  51.9  43.9   39.9*  46.1   49.9
//     8 x 32, 4000 to 8160, FP16     151   90.1  75.0   70.9   73.9   67.2*
//     1 x 64, 65280                  223   128   130    132    123*   129
//     64 x 64, 64 to 8160            906   599   524    563    476*   537
// `vectors`: rows of q and out on 16 bytes. Other rows and heads are padded, or
// take a wave a row.
Plan plan(const mlvc_hip_attention_drafts_desc* d, bool vectors)
{
    Plan p{};
    const mlvc_hip_kv_cache* c = d->cache;
    const std::int64_t rows = static_cast<std::int64_t>(d->longest_q) * (d->q_heads / c->heads), cus = conv::cu_count();
    p.row_count = rows * c->heads;
    const bool fast = vectors && (c->head_dim == 64 || c->head_dim == 128);
    const bool any = c->head_dim > 256 || c->head_dim * (c->kind == MLVC_KV_F16 ? 2 : 1) % 16 != 0;  // cached rows off 16 bytes
    // Tokens that a stream's drafts see at most, and those beside them in their steps.
    std::int64_t longest = d->longest;
    if (d->window) longest = std::min(longest, static_cast<std::int64_t>(d->window) + d->longest_q + std::min(d->sinks, d->longest) + 2 * kStep);
    auto workgroups = [&](Shape shape) { return (rows + kRows[shape] - 1) / kRows[shape] * c->heads * d->streams; };
    auto take = [&](Shape shape) { p.shape = shape, p.blocks = static_cast<int>((rows + kRows[shape] - 1) / kRows[shape]); };
    take(any                                                          ? kAny
         : !fast                                                      ? kPad
         : workgroups(kOne4) <= cus                                   ? kOne8
         : rows <= 16                                                 ? kOne4
         : rows <= 32 || workgroups(kTwo4) <= 2 * cus                 ? kTwo4
         : rows <= 64 || workgroups(kTile22) <= 4 * cus               ? kTile22
                                                                      : kTile41);
    if (longest <= 1024) return p;
    // Parts: each share leaves one a row, and one for each context that begins in
    // it. Asked for whether this call cuts or not and for the shape that leaves the
    // most, so that what is enough for a batch is enough for a smaller one.
    const size_t slots = kParts * static_cast<size_t>(cus) + (d->streams + 2) * static_cast<size_t>(p.row_count);
    p.part_bytes = slots * c->head_dim * sizeof(float);
    p.bytes = p.part_bytes + slots * sizeof(float2);
    const std::int64_t whole = workgroups(p.shape);
    if (!any ? (longest <= 2048 && 2 * whole >= cus) || (longest <= 4096 && whole >= 3 * cus) : whole >= kPerCu[kAny] * cus) return p;
    const bool bytes = c->kind != MLVC_KV_F16, many = static_cast<std::int64_t>(c->heads) * d->streams >= cus;
    take(any                                                             ? kAny
         : !fast                                                         ? kPad
         : rows <= 16 || workgroups(kOne4) * (longest / kStep) <= 48 * cus ? kOne4
         : rows <= 32                                                    ? kTwo4
         : rows <= 64                                                    ? (bytes && many ? kTile21 : kTile22)
                                                                         : (bytes ? kTile41 : kTile42));
    p.shares = static_cast<int>(std::max<std::int64_t>(1, kPerCu[p.shape] * cus / (static_cast<std::int64_t>(c->heads) * p.blocks)));
    return p;
}

template <class C>
void launch_drafts(const DraftArgs& a, unsigned grid, hipStream_t s)
{
    if (a.shares) drafts_kernel<C, true><<<grid, C::WAVES * 64, C::LDS, s>>>(a);
    else drafts_kernel<C, false><<<grid, C::WAVES * 64, C::LDS, s>>>(a);
}

template <int KIND, int D>
void launch_drafts(const DraftArgs& a, Shape shape, unsigned grid, hipStream_t s)
{
    switch (shape) {
    case kOne8: return launch_drafts<DraftCfg<KIND, D, 1, 8, 2>>(a, grid, s);
    case kOne4: return launch_drafts<DraftCfg<KIND, D, 1, 4, 3>>(a, grid, s);
    case kTwo4: return launch_drafts<DraftCfg<KIND, D, 2, 4, 2>>(a, grid, s);
    case kTile21: return launch_drafts<TileCfg<KIND, D, 2, 1>>(a, grid, s);
    case kTile22: return launch_drafts<TileCfg<KIND, D, 2, 2>>(a, grid, s);
    case kTile41: return launch_drafts<TileCfg<KIND, D, 4, 1>>(a, grid, s);
    case kTile42: return launch_drafts<TileCfg<KIND, D, 4, 2>>(a, grid, s);
    case kPad:
    case kAny: break;
    }
}

template <int KIND>
void launch_drafts(const DraftArgs& a, const Plan& p, unsigned grid, hipStream_t s)
{
    if (p.shape == kAny) drafts_any_kernel<KIND><<<grid, 64, 0, s>>>(a);
    else if (p.shape == kPad) a.dim <= 128 ? launch_drafts<TileCfg<KIND, 128, 2, 2, true>>(a, grid, s) : launch_drafts<TileCfg<KIND, 256, 2, 1, true>>(a, grid, s);
    else if (a.dim == 64) launch_drafts<KIND, 64>(a, p.shape, grid, s);
    else launch_drafts<KIND, 128>(a, p.shape, grid, s);
}

template <int LANES>
void launch_join(const DraftArgs& a, bool any, hipStream_t s)
{
    // A row for 256 threads where there are few; else eight at a time, by no more
    // workgroups than find where the parts lie in one turn of the GPU.
    const int rows = a.longest_q * a.group;
    const std::int64_t of_head = static_cast<std::int64_t>(a.heads) * a.streams;
    if (any || rows * of_head > 4096) {
        const int turns = static_cast<int>(std::max<std::int64_t>(1, std::min<std::int64_t>((rows + 7) / 8, 8 * conv::cu_count() / of_head)));
        const unsigned grid = static_cast<unsigned>(turns * of_head);
        if (any) drafts_join_kernel<LANES, 8, 1, true><<<grid, LANES * 8, 0, s>>>(a, turns);
        else drafts_join_kernel<LANES, 8, 1><<<grid, LANES * 8, 0, s>>>(a, turns);
    } else {
        drafts_join_kernel<LANES, 1, 256 / LANES><<<static_cast<unsigned>(rows * of_head), 256, 0, s>>>(a, rows);
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
    require(aligned_to<8>(d->seen) && aligned_to<4>(d->starts) && aligned_to<4>(d->lengths) && aligned_to<4>(d->table) && aligned_to<4>(d->placed), op,
            "seen, starts, lengths, table or placed is not aligned to its values");
    const Plan p = plan(d, vector_rows(d->q, d->q_stride) && vector_rows(d->out, d->out_stride));
    const std::int64_t all_rows = static_cast<std::int64_t>(d->streams) * p.row_count;
    const std::int64_t items = static_cast<std::int64_t>(d->cache->heads) * (p.shares ? (p.shape == kOne4 ? 2 : 1) * p.shares : d->streams);
    const std::int64_t grid = p.blocks == 1 || p.shape == kAny ? items * p.blocks : (items + kXcds - 1) / kXcds * kXcds * p.blocks;
    require(launchable(grid, 512) && launchable(all_rows, 256) &&
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
    a.placed = d->placed ? d->placed : d->lengths, a.all_placed = d->placed ? 0 : INT_MAX;
    a.table_stride = d->table_stride, a.pages = c->pages, a.page = c->page_size, a.heads = c->heads;
    a.q_heads = d->q_heads, a.group = d->q_heads / c->heads, a.dim = c->head_dim;
    a.longest = c->pages ? d->longest : 0, a.longest_q = d->longest_q, a.q_tokens = d->q_tokens, a.streams = d->streams;
    a.window = d->window, a.sinks = d->sinks;
    a.scale2 = d->scale * 1.4426950408889634f;
    a.part = static_cast<float*>(d->workspace);
    a.state = reinterpret_cast<float2*>(static_cast<char*>(d->workspace) + p.part_bytes);
    a.shares = p.shares, a.blocks = p.blocks, a.spare = p.shape == kOne4;
    a.places = (a.spare ? 2 : 1) * a.shares + a.streams;
    const unsigned n = static_cast<unsigned>(grid);
    if (c->kind == MLVC_KV_F16) launch_drafts<MLVC_KV_F16>(a, p, n, s);
    else if (c->kind == MLVC_KV_E4M3) launch_drafts<MLVC_KV_E4M3>(a, p, n, s);
    else launch_drafts<MLVC_KV_INT8>(a, p, n, s);
    check(hipGetLastError(), "attention_drafts launch");
    if (!p.shares) return;
    if (a.dim == 64) launch_join<16>(a, p.shape >= kPad, s);
    else launch_join<32>(a, p.shape >= kPad, s);
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
        bytes = plan(desc, true).bytes;  // the same for any rows
    });
    return bytes;
}

int mlvc_hip_attention_drafts(const mlvc_hip_attention_drafts_desc* desc, mlvc_hip_stream s)
{
    return guard([&] { attention_drafts(desc, to_stream(s)); });
}

}  // extern "C"
