// Attention of one query per stream on its paged, quantised context.
//
// Short contexts, and longer ones of large batches, go to one workgroup a stream
// and key head, which writes the output itself. The others are dealt evenly: the contexts
// of all streams, in steps of 32 tokens, are laid end to end and cut into one
// share for each workgroup the GPU holds at once, so ragged batches leave no CU
// idle and a single long stream fills them all. A workgroup finds its share from
// the lengths, and leaves the FP32 state (m, l, o) of the running softmax for
// each stream that does not lie in its share whole. A second kernel joins a
// stream's parts in their order:
//
//   m = max_s m_s,  l = sum_s l_s 2^(m_s - m),  out = sum_s o_s 2^(m_s - m) / l
//
// Scores are in powers of two (scaled by log2(e)).

#include "attention.hpp"

#include <algorithm>

namespace mlvc_hip {
namespace {

constexpr int kStep = 32;  // tokens of a step

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
    float* part;    // [q_heads][2 shares + streams][dim]
    float2* state;  // [q_heads][2 shares + streams]: m, l
    int table_stride, pages, page, heads, q_heads, group, dim, longest, streams;
    int shares;     // workgroups of a key head that the GPU holds at once; 0: a context goes to one workgroup
    unsigned long long tiles;  // 2^32 / (page / 16), rounded up: a tile's page by a product, for tiles below 2^32 / (page / 16)
    float scale2;
};

__device__ __forceinline__ int context(const TokenArgs& a, int stream)
{
    const std::int64_t held = static_cast<std::int64_t>(a.table_stride) * a.page;
    return static_cast<int>(min(static_cast<std::int64_t>(min(max(a.lengths[stream], 0), a.longest)), held));
}

__device__ __forceinline__ int steps_of(const TokenArgs& a, int stream)
{
    return stream < a.streams ? (context(a, stream) + kStep - 1) / kStep : 0;
}

__device__ __forceinline__ int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }

// The shares of a key head's steps: `shares` large ones, all on the GPU at
// once, cover five sixths of them, and as many small ones cover the rest,
// for the workgroups that are done first (their rates differ by a tenth
// either way). Few steps are not cut below kLeast, in one row of shares.
struct Shares {
    static constexpr int kLeast = 8;
    int total, large, count;  // steps; of them in the first `count` shares; the others are `count` more, or none
    __device__ Shares(const TokenArgs& a, int total_) : total(total_)
    {
        const bool few = total < 6 * kLeast * a.shares;
        count = few ? max(1, min(a.shares, total / kLeast)) : a.shares;
        large = few ? total : total - total / 6;
    }
    // First step of share i of n that cut `steps` evenly: i * steps / n without
    // a 64-bit product (n is a few workgroups a CU).
    __device__ static int cut(int i, int n, int steps)
    {
        const unsigned whole = static_cast<unsigned>(steps) / static_cast<unsigned>(n), rest = static_cast<unsigned>(steps) - whole * n;
        return static_cast<int>(i * whole + i * rest / static_cast<unsigned>(n));
    }
    // The share that holds a step: an estimate that is off by at most one.
    __device__ static int holds(int step, int n, int steps)
    {
        int i = min(static_cast<int>(static_cast<float>(step) * static_cast<float>(n) / static_cast<float>(steps)), n - 1);
        if (cut(i, n, steps) > step) --i;
        else if (cut(i + 1, n, steps) <= step) ++i;
        return i;
    }
    // First step of a share, and the share that holds a step.
    __device__ int first(int share) const
    {
        return share <= count ? cut(share, count, large) : large + cut(min(share - count, count), count, total - large);
    }
    __device__ int holder(int step) const
    {
        return step < large ? holds(step, count, large) : count + holds(step - large, count, total - large);
    }
};

// Calls fn(stream, first, last, whole, slot) for each piece [first, last) of a
// context that workgroup `share` of a key head takes; slot: the piece's place
// among a query head's parts, when it is not the whole context.
template <class F>
__device__ __forceinline__ void each_piece(const TokenArgs& a, int share, F&& fn)
{
    const int lane = threadIdx.x & 63;
    // 64 streams at a time, one a lane: tokens, and steps up to its end.
    auto tokens = [&](int b) { return b + lane < a.streams ? context(a, b + lane) : 0; };
    auto steps = [](int n) { return (n + kStep - 1) / kStep; };
    int block = 0, n = tokens(0), upto = wave_scan(steps(n));
    int total = __builtin_amdgcn_readlane(upto, 63);
    for (int b = 64; b < a.streams; b += 64) total += wave_sum(steps(tokens(b)));
    total = __builtin_amdgcn_readfirstlane(total);
    const Shares shares(a, total);
    if (share >= 2 * shares.count || (share >= shares.count && shares.large == total)) return;
    int at = __builtin_amdgcn_readfirstlane(shares.first(share));
    const int end = __builtin_amdgcn_readfirstlane(shares.first(share + 1));
    if (at >= end) return;
    auto next_block = [&] {
        const int before = __builtin_amdgcn_readlane(upto, 63);
        block += 64;
        n = tokens(block);
        upto = before + wave_scan(steps(n));
    };
    unsigned long long past;
    while (!(past = __ballot(upto > at))) next_block();  // at < total: some stream holds it
    int i = __builtin_ctzll(past);
    for (;;) {
        const int mine = __builtin_amdgcn_readlane(n, i), stop = __builtin_amdgcn_readlane(upto, i), start = stop - steps(mine);
        const int to = min(end, stop);
        if (to > at) fn(block + i, (at - start) * kStep, min(mine, (to - start) * kStep), to - at == stop - start, share + block + i);
        at = max(at, to);
        if (at >= end) return;
        if (++i == 64) next_block(), i = 0;
    }
}

// Row of token j of a stream's context, or -1 where its page is not in the cache.
__device__ __forceinline__ std::int64_t token_row(const TokenArgs& a, int stream, int head, int j)
{
    const int page = a.table[static_cast<std::int64_t>(stream) * a.table_stride + j / a.page];
    return page < 0 || page >= a.pages ? -1 : (static_cast<std::int64_t>(page) * a.heads + head) * a.page + j % a.page;
}

// Sums of FP16 values of tokens [first, last), N columns from d on, one of which came out as infinite or NaN.
template <int N, typename T>
__device__ __forceinline__ void decide_odd(const TokenArgs& a, int stream, int head, int first, int last, int d, T& sums)
{
    OddValues odd[N];
    for (int j = first; j < last; ++j) {
        const std::int64_t row = token_row(a, stream, head, j);
        if (row < 0) continue;
#pragma unroll
        for (int r = 0; r < N; ++r) odd[r].add(reinterpret_cast<const std::uint16_t*>(a.v)[row * a.dim + d + r]);
    }
#pragma unroll
    for (int r = 0; r < N; ++r) sums[r] = odd[r].sum(sums[r]);
}

// Any head size: one wave for a piece of one query head's context, 64 tokens
// at a time, one token a lane for the scores and one value column a lane for
// the sum.
template <int KIND>
__global__ __launch_bounds__(64) void token_any_kernel(TokenArgs a)
{
    __shared__ float qs[kMaxHeadDim], ps[64];
    __shared__ long long at[64];
    const int lane = threadIdx.x, head = blockIdx.x % a.q_heads, rest = blockIdx.x / a.q_heads;
    constexpr int kColumns = kMaxHeadDim / 64;
    auto value = [&](const std::uint8_t* x, long long row, int d) {
        if constexpr (KIND == MLVC_KV_F16) return h2f(reinterpret_cast<const std::uint16_t*>(x)[row * a.dim + d]);
        else return from_byte(KIND, x[row * a.dim + d]);
    };
    auto piece = [&](int stream, int first, int last, bool whole, int place) {
        const std::uint16_t* q = a.q + stream * a.q_stride + static_cast<std::int64_t>(head) * a.dim;
        for (int d = lane; d < a.dim; d += 64) qs[d] = h2f(q[d]) * a.scale2;
        __syncthreads();
        float acc[kColumns] = {}, m = -INFINITY, l = 0.0f;
        for (int j0 = first; j0 < last; j0 += 64) {
            const int j = j0 + lane;
            const long long row = j < last ? token_row(a, stream, head / a.group, j) : -1;
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
        if constexpr (KIND == MLVC_KV_F16) {
#pragma unroll
            for (int c = 0; c < kColumns; ++c) {
                float sum[1] = {acc[c]};
                if (c * 64 + lane < a.dim && !is_finite(sum[0])) decide_odd<1>(a, stream, head / a.group, first, last, c * 64 + lane, sum);
                acc[c] = sum[0];
            }
        }
        if (whole) {
            const float r = l == 0.0f ? 0.0f : 1.0f / l;
            std::uint16_t* out = a.out + stream * a.out_stride + static_cast<std::int64_t>(head) * a.dim;
#pragma unroll
            for (int c = 0; c < kColumns; ++c)
                if (c * 64 + lane < a.dim) out[c * 64 + lane] = f2h(opaque(acc[c] * r));
            return;
        }
        const std::int64_t slot = static_cast<std::int64_t>(head) * (2 * a.shares + a.streams) + place;
#pragma unroll
        for (int c = 0; c < kColumns; ++c)
            if (c * 64 + lane < a.dim) a.part[slot * a.dim + c * 64 + lane] = acc[c];
        if (lane == 0) a.state[slot] = make_float2(m, l);
    };
    if (a.shares == 0) piece(rest, 0, context(a, rest), true, 0);
    else each_piece(a, rest, piece);
}

// ------------------------------------------------------------ matrix cores

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

// Largest of a value over the four lanes of a column (16 apart).
__device__ __forceinline__ float column_max(float x) { return fmaxf(fmaxf(x, __shfl_xor(x, 16)), fmaxf(__shfl_xor(x, 32), __shfl_xor(x, 48))); }
__device__ __forceinline__ float column_sum(float x)
{
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// The half of bits 0x6480 ^ q is 1152 + q for a signed byte q: the byte under
// an exponent of 1024, its sign bit flipped.
__device__ __forceinline__ std::uint32_t minus_1152(std::uint32_t pair)
{
    const half2_t bias = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
    return __builtin_bit_cast(std::uint32_t, __builtin_bit_cast(half2_t, pair) + bias);
}

// Halves of the E4M3 bytes 0, 1 (2, 3) of a word.
template <bool UPPER>
__device__ __forceinline__ std::uint32_t e4m3_pair(std::uint32_t w)
{
    return __builtin_bit_cast(std::uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w), 1.0f, UPPER));
}

// Eight consecutive 8-bit values as halves.
template <int KIND>
__device__ __forceinline__ half8 eight(std::uint32_t w0, std::uint32_t w1)
{
    if constexpr (KIND == MLVC_KV_INT8) {
        constexpr std::uint32_t kUpper = 0x64646464u;
        const std::uint32_t a = w0 ^ 0x80808080u, b = w1 ^ 0x80808080u;
        return __builtin_bit_cast(half8, u32x4{minus_1152(__builtin_amdgcn_perm(kUpper, a, 0x04010400u)), minus_1152(__builtin_amdgcn_perm(kUpper, a, 0x04030402u)),
                                               minus_1152(__builtin_amdgcn_perm(kUpper, b, 0x04010400u)), minus_1152(__builtin_amdgcn_perm(kUpper, b, 0x04030402u))});
    } else {
        return __builtin_bit_cast(half8, u32x4{e4m3_pair<false>(w0), e4m3_pair<true>(w0), e4m3_pair<false>(w1), e4m3_pair<true>(w1)});
    }
}

// A word of each of two rows -> for each of its columns, the pair of halves.
template <int KIND>
__device__ __forceinline__ void columns(std::uint32_t a, std::uint32_t b, std::uint32_t* out)
{
    if constexpr (KIND == MLVC_KV_INT8) {
        out[0] = minus_1152(__builtin_amdgcn_perm(b, a, 0x0c040c00u) ^ 0x64806480u);
        out[1] = minus_1152(__builtin_amdgcn_perm(b, a, 0x0c050c01u) ^ 0x64806480u);
        out[2] = minus_1152(__builtin_amdgcn_perm(b, a, 0x0c060c02u) ^ 0x64806480u);
        out[3] = minus_1152(__builtin_amdgcn_perm(b, a, 0x0c070c03u) ^ 0x64806480u);
    } else if constexpr (KIND == MLVC_KV_E4M3) {
        const std::uint32_t a0 = e4m3_pair<false>(a), a1 = e4m3_pair<true>(a), b0 = e4m3_pair<false>(b), b1 = e4m3_pair<true>(b);
        out[0] = __builtin_amdgcn_perm(b0, a0, 0x05040100u), out[1] = __builtin_amdgcn_perm(b0, a0, 0x07060302u);
        out[2] = __builtin_amdgcn_perm(b1, a1, 0x05040100u), out[3] = __builtin_amdgcn_perm(b1, a1, 0x07060302u);
    } else {
        out[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
        out[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    }
}

// Heads of D values. A workgroup takes up to 16 query heads that share a key
// head, and a part of one stream's context; its waves take consecutive runs
// of the part, 32 tokens a step, and join through LDS at the end.
//
// Per step, with 16x16x32 products: S^T = K Q^T (two tiles of 16 tokens as
// rows, query heads as columns), so a lane's 8 scores belong to one query, and
// rounded to halves they are the B operand of O^T += V^T P^T as they stand. The
// cache is read straight into registers, each row once: K rows are A operands
// as they lie (16 bytes a lane; which value of the head stands where in a
// product does not matter as long as Q agrees), and V is transposed by the
// conversion to halves, which takes one column of two rows at a time.
//
// Scales are applied to scores and weights, not to values: s = (q . k) scale_k,
// and the weight of a row of V is 2^(s - m + log2(scale_v) - mw) with a running
// base mw of its own on top of m, so weights keep FP16's precision whatever the
// scales, and the logarithm its bits whatever the scores. It is -inf while all
// values seen are zero (scale 0).
// They go in as two halves, w and the rounding's remainder: the products are
// few next to the bytes. A weight is off by 2^-22 of itself or, as both halves
// end at 2^-24 and the largest weight is given as 2^12 at least (kLift), by
// 2^-37 of the largest: 2^-21 of the values in a context of 65536.
//
// Bound by the bytes of the cache: 64 streams of 1 to 8160 tokens, 32 query
// heads on 8 of 128, INT8, 0.55 GB in 111 us or 5.0 TB/s; one stream of 65280
// in E4M3, 138 MB in 34.1 us, of them 6 for the launches and the join; 16
// streams of 920 to 3001 tokens, 16 heads of 64, FP16, 128 MB in 30.5 us. A
// context of one workgroup is bound by the latency of its few steps: 920 tokens
// 8.4 us, of them 4 for an empty launch.
template <int KIND_, int D_, int WAVES_, int OCC_>
struct TokenCfg {
    static constexpr int KIND = KIND_, D = D_, WAVES = WAVES_, OCC = OCC_;
    static constexpr int BYTES = KIND == MLVC_KV_F16 ? 2 : 1;
    static constexpr int KL = D * BYTES / 64;          // 16-byte loads of a lane for a tile of K
    static constexpr int VW = D * BYTES / 64;          // words of a lane for a row of V
    static constexpr int PER = 4 / BYTES;              // values of a word
    static constexpr int DT = D / 16;                  // tiles of O^T
};

template <class C, bool SHARES>
__device__ __forceinline__ void token_piece(const TokenArgs& a, float* joint, int head, int block, int stream, int first, int last,
                                            bool whole, int place_of_part)
{
    constexpr int D = C::D, KIND = C::KIND;
    // Opaque, so that what follows from it is not kept in registers from piece to piece.
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const int mine = min(16, a.group - block * 16), q_head = head * a.group + block * 16;

    constexpr int KS = D / 32;
    half8 q[KS];
    {
        const std::uint16_t* row = a.q + stream * a.q_stride + static_cast<std::int64_t>(q_head + min(col, mine - 1)) * D;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int d = C::BYTES == 1 ? (ks >> 1) * 64 + 16 * g + 8 * (ks & 1) : ks * 32 + 8 * g;
            const u32x4 v = *reinterpret_cast<const u32x4*>(row + d);
            q[ks] = __builtin_bit_cast(half8, col < mine ? v : u32x4{0, 0, 0, 0});
        }
    }

    // A share's piece is cut into a run of steps for each wave. A whole context
    // is dealt step by step, so that a wave's first step does not depend on the
    // length: its rows are asked for while the length is still on its way.
    const int steps = (max(last - first, 0) + kStep - 1) / kStep;
    constexpr int kStride = SHARES ? kStep : C::WAVES * kStep;
    const int from = first + (SHARES ? steps * wave / C::WAVES : wave) * kStep;
    const int to = SHARES ? min(last, first + steps * (wave + 1) / C::WAVES * kStep) : last;
    typedef const __attribute__((address_space(4))) std::int32_t* scalar_table;
    const scalar_table table = (scalar_table)(a.table + static_cast<std::int64_t>(stream) * a.table_stride);

    // Rows of the two tiles (16 tokens each, in one page) of a step, row 0 for a
    // tile that is not there.
    std::int64_t row[2];
    bool there[2];
    int page_at = SHARES ? from / a.page : 0, place = from - page_at * a.page;
    auto locate = [&](int j) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            int page = -1, in_page;
            if constexpr (SHARES) {
                if (j + 16 * t < to) page = table[page_at];
                in_page = place;
                place += 16;
                if (place == a.page) place = 0, ++page_at;
            } else {
                const unsigned tile = static_cast<unsigned>(j >> 4) + t;
                const int at = static_cast<int>(tile * a.tiles >> 32);
                if (at < a.table_stride) page = table[at];
                in_page = j + 16 * t - at * a.page;
            }
            there[t] = page >= 0 && page < a.pages;
            row[t] = there[t] ? (static_cast<std::int64_t>(page) * a.heads + head) * a.page + in_page : 0;
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
    auto fetch_v = [&](const std::int64_t* row) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const std::uint8_t* p = a.v + row[t] * (D * C::BYTES);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const std::uint8_t* at = p + (4 * g + e) * (D * C::BYTES) + col * (4 * C::VW);
                if constexpr (C::VW == 4) {
                    const u32x4 w = *reinterpret_cast<const u32x4*>(at);
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[4 * t + e][i] = w[i];
                } else if constexpr (C::VW == 2) {
                    const u32x2 w = *reinterpret_cast<const u32x2*>(at);
                    v[4 * t + e][0] = w[0], v[4 * t + e][1] = w[1];
                } else {
                    v[4 * t + e][0] = *reinterpret_cast<const std::uint32_t*>(at);
                }
            }
        }
    };

    floatx4 acc[C::DT];
#pragma unroll
    for (int i = 0; i < C::DT; ++i) acc[i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, mw = -INFINITY, l = 0.0f;

    if (SHARES ? from < to : a.pages > 0) {
        locate(from);
        fetch_k();
        fetch_v(row);
    }
    // K of the next step is asked for as soon as this step's has been used, V
    // likewise, so a wave always has about a step of the cache in flight.
    for (int j = from; j < to; j += kStride) {
#pragma clang fp contract(off)  // a score less the base: of the score as it was when the base was taken
        floatx4 dot[2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                half8 kf;
                if constexpr (C::BYTES == 2) kf = __builtin_bit_cast(half8, k[t][s]);
                else kf = eight<KIND>(k[t][s >> 1][2 * (s & 1)], k[t][s >> 1][2 * (s & 1) + 1]);
                dot[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[s], s ? dot[t] : floatx4{}, 0, 0, 0);
            }
        float x[8], y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = dot[e >> 2][e & 3] * a.scale2;
            if constexpr (KIND != MLVC_KV_F16) {
                x[e] *= ks[e >> 2][e & 3];
                y[e] = __builtin_amdgcn_logf(vs[e >> 2][e & 3]);
            }
        }
        const bool ragged = j + kStep > to || !there[0] || !there[1];
        const bool seen[2] = {there[0], there[1]};
        if (j + kStride < to) {
            locate(j + kStride);
            fetch_k();
        }
        if (ragged) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (!seen[e >> 2] || j + 16 * (e >> 2) + 4 * g + (e & 3) >= to) {
                    // Not seen: weight zero, and a value that is finite whatever lies there.
                    x[e] = -INFINITY, y[e] = 0.0f;
#pragma unroll
                    for (int w = 0; w < C::VW; ++w) v[e][w] = 0;
                }
        }
        auto rescale = [&](float keep) {
#pragma unroll
            for (int i = 0; i < C::DT; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[i][r] *= keep;
        };
        float top = x[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) top = __builtin_elementwise_maximum(top, x[e]);
        if (__any(top - m > kMost)) {
            const float now = fmaxf(m, lifted(column_max(top))), keep = __builtin_amdgcn_exp2f(m - (now == -INFINITY ? 0.0f : now));
            l *= keep;
            if constexpr (KIND == MLVC_KV_F16) rescale(keep);
            else if (m != -INFINITY) mw += m - now;
            m = now;
        }
        const float base = m == -INFINITY ? 0.0f : m;
        float basew = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] -= base;
        if constexpr (KIND != MLVC_KV_F16) {
            float topw = -INFINITY;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                y[e] += x[e];
                topw = __builtin_elementwise_maximum(topw, y[e]);
            }
            if (__any(topw - mw > kMost)) {
                const float now = fmaxf(mw, lifted(column_max(topw)));
                rescale(__builtin_amdgcn_exp2f(mw - (now == -INFINITY ? 0.0f : now)));
                mw = now;
            }
            if (mw != -INFINITY) basew = mw;
        }
        half8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float p = __builtin_amdgcn_exp2f(x[e]);
            l += p;
            const float w = KIND == MLVC_KV_F16 ? p : __builtin_amdgcn_exp2f(y[e] - basew);
            hi[e] = static_cast<_Float16>(w);
            lo[e] = static_cast<_Float16>(w - static_cast<float>(hi[e]));
        }
#pragma unroll
        for (int w = 0; w < C::VW; ++w) {
            std::uint32_t pair[4][C::PER];
#pragma unroll
            for (int i = 0; i < 4; ++i) columns<KIND>(v[2 * i][w], v[2 * i + 1][w], pair[i]);
#pragma unroll
            for (int i = 0; i < C::PER; ++i) {
                const half8 vf = __builtin_bit_cast(half8, u32x4{pair[0][i], pair[1][i], pair[2][i], pair[3][i]});
                floatx4& o = acc[w * C::PER + i];
                o = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, hi, o, 0, 0, 0);
                o = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, lo, o, 0, 0, 0);
            }
        }
        if (j + kStride < to) fetch_v(row);
    }
    l = column_sum(l);

    // Join the waves. A lane holds, of its column's head, the values (4 g + r) * DT + i.
    float* const st = joint + C::WAVES * mine * D;
    if (col < mine) {
        float* o = joint + (wave * mine + col) * D;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < C::DT; i += 4)
                *reinterpret_cast<floatx4*>(o + (4 * g + r) * C::DT + i) = floatx4{acc[i][r], acc[i + 1][r], acc[i + 2][r], acc[i + 3][r]};
        if (g == 0) st[wave * 16 + col] = m, st[(C::WAVES + wave) * 16 + col] = l, st[(2 * C::WAVES + wave) * 16 + col] = mw;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < mine * (D / 4); i += C::WAVES * 64) {
        const int h = i / (D / 4), d = i % (D / 4) * 4;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < C::WAVES; ++w) top = fmaxf(top, st[w * 16 + h]);
        const float base = top == -INFINITY ? 0.0f : top;
        float total = 0.0f;
        floatx4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < C::WAVES; ++w) {
            float f = __builtin_amdgcn_exp2f(st[w * 16 + h] - base);
            total += st[(C::WAVES + w) * 16 + h] * f;
            if constexpr (KIND != MLVC_KV_F16) f *= __builtin_amdgcn_exp2f(st[(2 * C::WAVES + w) * 16 + h]);
            const floatx4 v = *reinterpret_cast<const floatx4*>(joint + (w * mine + h) * D + d);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = fmaf(v[r], f, o[r]);
        }
        if constexpr (KIND == MLVC_KV_F16)
            if (!is_finite(o[0]) || !is_finite(o[1]) || !is_finite(o[2]) || !is_finite(o[3])) decide_odd<4>(a, stream, head, first, last, d, o);
        if (whole) {
            const float f = total == 0.0f ? 0.0f : 1.0f / total;
            *reinterpret_cast<uint2*>(a.out + stream * a.out_stride + static_cast<std::int64_t>(q_head + h) * D + d) =
                make_uint2(pack_rounded(o[0] * f, o[1] * f), pack_rounded(o[2] * f, o[3] * f));
        } else {
            const std::int64_t slot = static_cast<std::int64_t>(q_head + h) * (2 * a.shares + a.streams) + place_of_part;
            *reinterpret_cast<floatx4*>(a.part + slot * D + d) = o;
            if (d == 0) a.state[slot] = make_float2(top, total);
        }
    }
}

// Workgroups of neighbouring numbers take the same tokens of different key
// heads, which lie side by side in a page.
template <class C, bool SHARES>
__global__ __launch_bounds__(C::WAVES * 64, C::OCC) void token_kernel(TokenArgs a)
{
    extern __shared__ float joint[];  // [WAVES][heads here][D], then [WAVES][16] of m, l and mw
    const int blocks = (a.group + 15) / 16, per = a.heads * blocks;
    const int which = blockIdx.x % per, rest = blockIdx.x / per, head = which / blocks, block = which % blocks;
    if constexpr (SHARES)
        each_piece(a, rest, [&](int stream, int first, int last, bool whole, int place) {
            token_piece<C, true>(a, joint, head, block, stream, first, last, whole, place);
            __syncthreads();  // before the next piece's states
        });
    else token_piece<C, false>(a, joint, head, block, rest, 0, context(a, rest), true, 0);
}

// One workgroup for a query head of a stream. LANES threads hold a part's row,
// four values each, and the others take every (THREADS / LANES)-th part, each
// with a running maximum of its own; they are put together in LDS.
template <int LANES, int THREADS>
__global__ __launch_bounds__(THREADS) void token_join_kernel(TokenArgs a)
{
    constexpr int kGroups = THREADS / LANES;
    __shared__ floatx4 sums[kGroups][LANES];
    __shared__ float2 states[kGroups];
    const int lane = threadIdx.x & 63, head = blockIdx.x % a.q_heads, stream = blockIdx.x / a.q_heads;
    const int group = threadIdx.x / LANES, at = threadIdx.x % LANES;
    int total = 0, start = 0;
    for (int b = 0; b < a.streams; b += 64) {
        const int mine = steps_of(a, b + lane);
        if (b + lane < stream) start += mine;
        total += mine;
    }
    total = wave_sum(total), start = wave_sum(start);
    const int steps = steps_of(a, stream);
    const Shares shares(a, total);
    const int first = steps ? shares.holder(start) : 0, parts = steps ? shares.holder(start + steps - 1) - first + 1 : 0;
    if (parts == 1) return;  // written by the share that holds it
    const std::int64_t slot = static_cast<std::int64_t>(head) * (2 * a.shares + a.streams) + first + stream;
    for (int d = at * 4; d - at * 4 < a.dim; d += LANES * 4) {
        float m = -INFINITY, l = 0.0f;
        floatx4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
        if (d < a.dim) {
#pragma unroll 4
            for (int i = group; i < parts; i += kGroups) {
                const floatx4 v = *reinterpret_cast<const floatx4*>(a.part + (slot + i) * a.dim + d);
                const float2 st = a.state[slot + i];
                const float now = fmaxf(m, st.x), base = now == -INFINITY ? 0.0f : now;
                const float old = __builtin_amdgcn_exp2f(m - base), f = __builtin_amdgcn_exp2f(st.x - base);
                m = now;
                l = l * old + st.y * f;
#pragma unroll
                for (int r = 0; r < 4; ++r) sum[r] = sum[r] * old + v[r] * f;
            }
        }
        sums[group][at] = sum;
        if (at == 0) states[group] = make_float2(m, l);
        __syncthreads();
        if (group == 0 && d < a.dim) {
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < kGroups; ++i) top = fmaxf(top, states[i].x);
            if (top == -INFINITY) top = 0.0f;
            l = 0.0f;
            sum = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < kGroups; ++i) {
                const float2 st = states[i];
                const float f = __builtin_amdgcn_exp2f(st.x - top);
                l += st.y * f;
#pragma unroll
                for (int r = 0; r < 4; ++r) sum[r] = fmaf(sums[i][at][r], f, sum[r]);
            }
            // A part that is infinite, with however small a weight.
            if (!is_finite(sum[0]) || !is_finite(sum[1]) || !is_finite(sum[2]) || !is_finite(sum[3])) {
                floatx4 odd = {0.0f, 0.0f, 0.0f, 0.0f};
                for (int i = 0; i < parts; ++i) {
                    const floatx4 v = *reinterpret_cast<const floatx4*>(a.part + (slot + i) * a.dim + d);
#pragma unroll
                    for (int r = 0; r < 4; ++r) odd[r] += is_finite(v[r]) ? 0.0f : v[r];
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) sum[r] = is_finite(sum[r]) ? sum[r] : odd[r];
            }
            const float f = l == 0.0f ? 0.0f : 1.0f / l;
            std::uint16_t* out = a.out + stream * a.out_stride + static_cast<std::int64_t>(head) * a.dim + d;
#pragma unroll
            for (int r = 0; r < 4; ++r) out[r] = f2h(opaque(sum[r] * f));
        }
        __syncthreads();
    }
}

struct Plan {
    int shares;
    size_t part_bytes, bytes;
};

// Whether a context goes to one workgroup of eight waves, without a cut. Up to
// 1024 tokens it is done before a second kernel would start; longer ones are
// not cut where enough workgroups keep the GPU busy through the longest: half
// one a CU up to 2048 tokens, three a CU up to 4096. The lengths themselves are
// on the device: a batch of very different ones, which a cut would even out,
// and the shortest of the contexts that are cut lose by the rule. us, whole /
// cut, the one taken marked *:
//   1 x 920, 4 heads of 64, INT8      8.7*/ 10.2
//   200 x 512..1024, 8 of 128, INT8  75.7*/ 83.9    (1600 workgroups)
//   16 x 1..1300, 4 of 64, E4M3       9.7 / 12.5*   (64)
//   16 x 1000..2000, 4 of 64, FP16   15.4 / 13.5*   (64)
//   16 x 1000..2000, 8 of 128, INT8  20.6*/ 19.7    (128)
//   64 x 1000..2000, 4 of 64, FP16   19.5*/ 24.2    (256)
//   48 x 1..2000, 8 of 128, INT8     32.6*/ 29.6    (384)
//   64 x 1..2000, 8 of 128, INT8     41.0*/ 37.7    (512)
//   64 x 1000..2000, 8 of 128, INT8  46.8*/ 49.6    (512)
//   200 x 1..4080, 8 of 128, INT8     174*/ 177     (1600)
//   200 x 1..4080, 4 of 64, E4M3     56.7*/ 57.3    (800)
//   64 x 2040..4080, 4 of 64, FP16   40.8 / 45.5*   (256)
//   64 x 1..4080, 8 of 128, INT8     71.9 / 62.1*   (512)
//   200 x 4080..8160, 4 of 64, FP16   239 / 227*    (800)
bool whole(int longest, std::int64_t workgroups)
{
    const std::int64_t cus = conv::cu_count();
    return longest <= 1024 || (longest <= 2048 && 2 * workgroups >= cus) || (longest <= 4096 && workgroups >= 3 * cus);
}

Plan plan(const mlvc_hip_attention_token_desc* d)
{
    Plan p{};
    if (d->longest <= 1024) return p;
    // Three workgroups of four waves fit a CU (up to 168 registers).
    const int group = d->q_heads / d->cache->heads, of_stream = d->cache->heads * ((group + 15) / 16);
    const int shares = std::max(1, 3 * conv::cu_count() / of_stream);
    const size_t slots = (2 * static_cast<size_t>(shares) + d->streams) * d->q_heads;
    p.part_bytes = slots * d->cache->head_dim * sizeof(float);
    // Asked for whether this call cuts or not, so that what is enough for a
    // batch is enough for a smaller one.
    p.bytes = p.part_bytes + slots * sizeof(float2);
    if (!whole(d->longest, static_cast<std::int64_t>(d->streams) * of_stream)) p.shares = shares;
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

template <class C, bool SHARES>
void launch_token(const TokenArgs& a, unsigned grid, hipStream_t s)
{
    const int most = std::min(a.group, 16);
    const size_t lds = (static_cast<size_t>(C::WAVES) * most * C::D + 3 * C::WAVES * 16) * sizeof(float);
    token_kernel<C, SHARES><<<grid, C::WAVES * 64, lds, s>>>(a);
}

template <int KIND>
void launch_token(const TokenArgs& a, unsigned grid, hipStream_t s)
{
    if (a.shares) {
        if (a.dim == 64) launch_token<TokenCfg<KIND, 64, 4, 3>, true>(a, grid, s);
        else launch_token<TokenCfg<KIND, 128, 4, 3>, true>(a, grid, s);
    } else {
        if (a.dim == 64) launch_token<TokenCfg<KIND, 64, 8, 2>, false>(a, grid, s);
        else launch_token<TokenCfg<KIND, 128, 8, 2>, false>(a, grid, s);
    }
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
    const bool fast = (d->cache->head_dim == 64 || d->cache->head_dim == 128) && vector_rows(d->q, d->q_stride) && vector_rows(d->out, d->out_stride);
    // Workgroups of the first kernel, and of the one that joins.
    const int group = d->q_heads / d->cache->heads;
    const std::int64_t grid = static_cast<std::int64_t>(fast ? d->cache->heads * ((group + 15) / 16) : d->q_heads) * (p.shares ? 2 * p.shares : d->streams);
    require(launchable(grid, fast && !p.shares ? 512 : 256) && (!p.shares || launchable(heads, 256)) &&
                static_cast<std::int64_t>(d->streams) * (d->longest / kStep + 1) <= INT_MAX, op,
            "too many streams, heads and tokens in one call");

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
    a.q_heads = d->q_heads, a.group = group, a.dim = c->head_dim;
    a.longest = c->pages ? d->longest : 0, a.streams = d->streams;
    a.shares = p.shares;
    a.tiles = ((1ull << 32) + c->page_size / 16 - 1) / (c->page_size / 16);
    a.scale2 = d->scale * 1.4426950408889634f;
    const unsigned n = static_cast<unsigned>(grid);
    if (fast && c->kind == MLVC_KV_F16) launch_token<MLVC_KV_F16>(a, n, s);
    else if (fast && c->kind == MLVC_KV_E4M3) launch_token<MLVC_KV_E4M3>(a, n, s);
    else if (fast) launch_token<MLVC_KV_INT8>(a, n, s);
    else if (c->kind == MLVC_KV_F16) token_any_kernel<MLVC_KV_F16><<<n, 64, 0, s>>>(a);
    else if (c->kind == MLVC_KV_E4M3) token_any_kernel<MLVC_KV_E4M3><<<n, 64, 0, s>>>(a);
    else token_any_kernel<MLVC_KV_INT8><<<n, 64, 0, s>>>(a);
    check(hipGetLastError(), "attention_token launch");
    if (p.shares) {
        const unsigned n = static_cast<unsigned>(heads);
        // A stream of few parts is put together by one wave instead of four: 200
        // streams of up to 8160 tokens 225.6 us instead of 230, 64 of up to 4080
        // 62.1 instead of 64.0; 16 of up to 3001 the same.
        const bool few = 2 * p.shares <= 8 * d->streams;
        if (few && a.dim <= 64) token_join_kernel<16, 64><<<n, 64, 0, s>>>(a);
        else if (few) token_join_kernel<32, 64><<<n, 64, 0, s>>>(a);
        else if (a.dim <= 64) token_join_kernel<16, 256><<<n, 256, 0, s>>>(a);
        else token_join_kernel<32, 256><<<n, 256, 0, s>>>(a);
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
