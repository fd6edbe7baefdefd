// Attention of packed sequences (one pass over the keys with the running
// maximum and sum of the softmax).
//
//   m' = max(m, max_j s_j),  l' = l e^(m - m') + sum_j e^(s_j - m'),
//   o' = o e^(m - m') + sum_j e^(s_j - m') v_j,   out = o / l
//
// in powers of two: s is scaled by log2(e), so each exponential is one
// v_exp_f32.

#include "attention.hpp"

#include <algorithm>
#include <type_traits>

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
    int sequences, q_heads, group, dim, q_tokens, k_tokens, longest_q, causal, negate, cus;
    float scale2;  // |scale| log2(e); negate: scale is negative
};

// Rows [first, first + count) of a sequence, cut to the tensor.
struct Span {
    int first, count;
};
__device__ __forceinline__ Span span(int start, int end, int tokens)
{
    const int a = min(max(start, 0), tokens), b = min(max(end, a), tokens);
    return {a, b - a};
}
__device__ __forceinline__ Span span(const std::int32_t* starts, int n, int tokens) { return span(starts[n], starts[n + 1], tokens); }

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
    for (int d = lane; d < a.dim; d += 64) qs[d] = h2f(q[d]) * (a.negate ? -a.scale2 : a.scale2);
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
#pragma unroll
    for (int c = 0; c < kColumns; ++c) {
        const int d = c * 64 + lane;
        if (d >= a.dim || is_finite(acc[c])) continue;
        OddValues odd;
        for (int j = 0; j < seen; ++j) odd.add(a.v[static_cast<std::int64_t>(sk.first + j) * a.v_stride + column + d]);
        acc[c] = odd.sum(acc[c]);
    }
    const float r = l == 0.0f ? 0.0f : 1.0f / l;
    std::uint16_t* out = a.out + token * a.out_stride + static_cast<std::int64_t>(head) * a.dim;
#pragma unroll
    for (int c = 0; c < kColumns; ++c)
        if (c * 64 + lane < a.dim) out[c * 64 + lane] = f2h(opaque(acc[c] * r));
}

// ------------------------------------------------------------ matrix cores

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

constexpr int kRawBufferFlags = 0x00020000;
constexpr int kProducts = 0x8, kReads = 0x100;  // instruction groups of sched_group_barrier: MFMA, LDS reads

__device__ __forceinline__ std::uint32_t uniform(std::uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }

// 16 bytes a lane from `at` bytes into a raw buffer to LDS, lane after lane;
// out of the buffer's range, zeros. In assembly because the compiler lets every
// LDS read that follows the builtin wait for it: here the tile that is read and
// the one being filled are never the same, and the caller waits (vmcnt) and
// synchronises before it turns to the next. The compiler does not see that this
// is a load, so the wait states that the hardware leaves to it stand here too:
// one after a scalar write of m0, five after a vector write of the buffer's
// scalar registers (lanes made uniform just before); s_nop N makes N + 1. All
// five instead of the one cost 1% at 8160 tokens, 16 heads of 64, and nothing
// at heads of 128.
__device__ __forceinline__ void lds_dma16(u32x4 buffer, std::uint32_t to, std::uint32_t at)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(at), "s"(buffer) : "memory", "m0");
}
__device__ __forceinline__ std::uint32_t lds_address(const void* p)
{
    return static_cast<std::uint32_t>(reinterpret_cast<std::uintptr_t>((__attribute__((address_space(3))) const void*)p));
}

// Maximum (sum) of a lane's value and that of the lane 32 away, in both.
__device__ __forceinline__ float both_max(float x)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float both_sum(float x)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Heads of D values, rows on 16 bytes. A workgroup of RG x KG waves takes
// RG * 32 queries of a head. A wave holds 32 of them as columns of S^T = K Q^T
// (32x32x16 products, keys as rows), so that
//   * a lane's scores all belong to one query: the softmax needs one exchange,
//     between the two lanes of a column;
//   * the accumulator registers of S^T, rounded to FP16, are the B operand of
//     O^T += V^T P^T as they stand (the 16 keys of a step are taken in the order
//     the registers hold them), so weights never leave the lane.
// The KG groups of waves take every KG-th tile of KEYS keys and are put together
// in LDS at the end: more waves where there are too few queries to fill the GPU.
//
// Tiles are staged by LDS DMA, double-buffered, 16-byte pieces of a row
// permuted (piece ^ f(row)) so that both reads are free of bank conflicts: K
// rows by 16 bytes, V by the transposing read. Rows past a sequence's end are
// out of the buffer's range and read as zeros.
//
// The base of the weights lies 12 powers of two below a score and moves only
// when one passes it by 15 (FP16 and the FP32 sums hold weights up to 2^15), so
// the accumulators are seldom rescaled. Weights are rounded to FP16, the type
// the matrix cores take beside V: by 2^-11 of themselves, as the output is, or
// by 2^-37 of the largest where they are subnormal. Their sum is of FP32 values.
template <int D_, int RG_, int KG_, int KEYS_, int OCC_>
struct PromptCfg {
    static constexpr int D = D_, RG = RG_, KG = KG_, KEYS = KEYS_, OCC = OCC_;
    static constexpr int WAVES = RG * KG;
    // Several workgroups on a CU: long ones are put beside short ones.
    static constexpr bool PAIRED = KG == 1 && OCC * 4 / WAVES > 1;
    static constexpr int ROWS = RG * 32;             // queries of a workgroup
    static constexpr int PIECES = D / 8;             // 16-byte pieces of a row
    static constexpr int DMA_ROWS = 64 / PIECES;     // rows of a DMA instruction
    static constexpr int DMA = KEYS / DMA_ROWS;      // instructions of a tile
    static constexpr int TILE = KEYS * D;            // halves
    static constexpr int TILES = KG * 2 * 2 * TILE;  // two buffers of K and V
    static constexpr size_t LDS = TILES * 2 + 2 * WAVES * sizeof(int);
    // Piece p of row t is kept at place p ^ swizzle(t): 16 rows of one piece
    // (a K read) fall on all 64 banks, and so do 4 rows of 4 pieces (a V read).
    __host__ __device__ static constexpr int swizzle(int t)
    {
        return D == 128 ? 4 * (t & 3) + (t >> 2 & 3) : 4 * (t >> 1 & 1) + (t >> 2 & 3);
    }
};

// The rank-th tile of queries; false past the last, and for one that is not
// there. By the number of keys a tile may see, most first: tile t of sequence n
// has level base_n + t, in ROWS keys, and the tiles above a level are counted
// for 64 levels at a time, one a lane (up to 64 sequences, one a lane too).
// That takes 0.3 us. When it came, 8 ragged sequences (1 to 2040 tokens, 16 heads
// of 128) took 57 us instead of 64.5 (54 now), and where tiles just fit the CUs,
// ones that are not there take no CU's turn: one sequence of 2000 and three of 100
// tokens 37.7 instead of 52, of 300 and 20 tokens 9.4 instead of 13.5. More
// sequences follow one another, each with its last tile first, 64 at a time.
// by_turns: sequence after sequence within a tile number.
template <class C>
__device__ __forceinline__ bool choose(const PromptArgs& a, int rank, int tiles, bool by_turns, int& n, int& tile, Span& sq, Span& sk)
{
    constexpr int ROWS = C::ROWS;
    if (by_turns) {
        n = rank % a.sequences;
        tile = tiles - 1 - rank / a.sequences;
        const int qa = a.q_starts[n], qb = a.q_starts[n + 1], ka = a.k_starts[n], kb = a.k_starts[n + 1];
        asm volatile("" ::"s"(qa), "s"(qb), "s"(ka), "s"(kb));
        sq = span(qa, qb, a.q_tokens), sk = span(ka, kb, a.k_tokens);
        return tile >= 0 && tile * ROWS < min(sq.count, a.longest_q);
    }
    const int lane = threadIdx.x & 63;
    if (a.sequences > 64) {
        auto ends = [&](int i) {
            return i < a.sequences ? make_int4(a.q_starts[i], a.q_starts[i + 1], a.k_starts[i], a.k_starts[i + 1]) : make_int4(0, 0, 0, 0);
        };
        int before = 0;
        int4 next = ends(lane);
        for (int b = 0; b < a.sequences; b += 64) {
            const Span q = span(next.x, next.y, a.q_tokens), k = span(next.z, next.w, a.k_tokens);
            next = ends(b + 64 + lane);
            const int count = (min(q.count, a.longest_q) + ROWS - 1) / ROWS, upto = before + wave_scan(count);
            const unsigned long long past = __ballot(upto > rank);
            before = __builtin_amdgcn_readlane(upto, 63);
            if (!past) continue;
            const int i = __builtin_ctzll(past);
            n = b + i;
            tile = __builtin_amdgcn_readlane(upto, i) - 1 - rank;
            sq = {__builtin_amdgcn_readlane(q.first, i), __builtin_amdgcn_readlane(q.count, i)};
            sk = {__builtin_amdgcn_readlane(k.first, i), __builtin_amdgcn_readlane(k.count, i)};
            return true;
        }
        return false;
    }
    Span q = {0, 0}, k = {0, 0};
    if (lane < a.sequences) q = span(a.q_starts, lane, a.q_tokens), k = span(a.k_starts, lane, a.k_tokens);
    const int count = (min(q.count, a.longest_q) + ROWS - 1) / ROWS;
    const int base = (a.causal ? max(k.count - q.count, 0) : k.count) / ROWS;
    int level = 0, above = 0;
    for (int width = (a.k_tokens / ROWS + tiles + 64) / 64;; width = (width + 63) / 64) {
        const int top = level + (lane + 1) * width - 1;
        above = 0;
        for (int s = 0; s < a.sequences; ++s) {
            const int c = __builtin_amdgcn_readlane(count, s), b = __builtin_amdgcn_readlane(base, s);
            above += min(max(b + c - 1 - top, 0), c);
        }
        const int at = __builtin_ctzll(__ballot(above <= rank) | 1ull << 63);
        level += at * width;
        above = __builtin_amdgcn_readlane(above, at);
        if (width == 1) break;
    }
    const bool has = static_cast<unsigned>(level - base) < static_cast<unsigned>(count);
    const unsigned long long all = __ballot(has);
    const int before = __builtin_amdgcn_mbcnt_hi(static_cast<unsigned>(all >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<unsigned>(all), 0));
    const unsigned long long mine = __ballot(has && above + before == rank);
    if (!mine) return false;
    n = __builtin_ctzll(mine);
    tile = level - __builtin_amdgcn_readlane(base, n);
    sq = {__builtin_amdgcn_readlane(q.first, n), __builtin_amdgcn_readlane(q.count, n)};
    sk = {__builtin_amdgcn_readlane(k.first, n), __builtin_amdgcn_readlane(k.count, n)};
    return true;
}

template <class C>
__global__ __launch_bounds__(C::WAVES * 64, C::OCC) void prompt_kernel(PromptArgs a, int tiles, bool by_turns)
{
    constexpr int D = C::D, KS = D / 16, DT = D / 32, kKeys = C::KEYS, TT = kKeys / 32;
    extern __shared__ __attribute__((aligned(16))) std::uint16_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row_group = wave % C::RG, key_group = wave / C::RG, column = lane & 31, hi = lane >> 5;

    // Workgroup i runs on XCD i % 8, its (i / 8)-th there: with a multiple of 8
    // heads an XCD keeps the same heads, of all sequences, so their keys stay
    // in its L2. Tiles of queries go in the order of their keys, most first. An
    // XCD's first workgroups take a CU each and the next ones join them in the
    // same order, so those come in the opposite one: the longest beside the
    // shortest.
    // All arguments at once: each would be asked for where it is first used, one
    // latency after another (0.2 to 0.7 us of a small call).
    asm volatile("" ::"s"(a.q), "s"(a.k), "s"(a.v), "s"(a.out), "s"(a.q_stride), "s"(a.k_stride), "s"(a.v_stride), "s"(a.out_stride),
                 "s"(a.q_starts), "s"(a.k_starts), "s"(a.sequences), "s"(a.q_heads), "s"(a.scale2), "s"(a.cus));
    int head, n, tile;
    Span sq, sk;
    {
        unsigned i = blockIdx.x / kXcds;
        if constexpr (C::PAIRED) {
            const unsigned cus = a.cus / kXcds, joined = min(2 * cus, gridDim.x / kXcds);
            if (i >= cus && i < joined) i = cus + joined - 1 - i;
        }
        int rank;
        if (a.q_heads % kXcds == 0) {
            const int per = a.q_heads / kXcds;
            head = blockIdx.x % kXcds * per + i % per;
            rank = i / per;
        } else {
            i = i * kXcds + blockIdx.x % kXcds;
            head = i % a.q_heads;
            rank = i / a.q_heads;
        }
        if (!choose<C>(a, rank, tiles, by_turns, n, tile, sq, sk)) return;
    }
    const int q0 = tile * C::ROWS, nq = min(sq.count, a.longest_q);
    const int behind = sk.count - sq.count;  // keys before the first query
    const int last = min(q0 + C::ROWS, nq) - 1;
    const int keys = a.causal ? max(0, min(sk.count, behind + last + 1)) : sk.count;  // seen by any query here
    const int steps = (keys + kKeys - 1) / kKeys;

    // This wave's queries, as B fragments.
    const int w0 = q0 + row_group * 32, i_query = w0 + column, at_query = min(i_query, nq - 1);
    half8 q[KS];
    {
        const std::uint16_t* row = a.q + (sq.first + at_query) * a.q_stride + static_cast<std::int64_t>(head) * D + hi * 8;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            u32x4 v = *reinterpret_cast<const u32x4*>(row + ks * 16);
            if (a.negate)
                for (int e = 0; e < 4; ++e) v[e] ^= 0x80008000u;
            q[ks] = __builtin_bit_cast(half8, v);
        }
    }
    const int seen = a.causal ? max(0, min(sk.count, behind + at_query + 1)) : sk.count;  // keys this lane's query sees
    // Tiles that every query of the workgroup sees whole, and keys that any of this wave's sees.
    const int clear = (a.causal ? max(0, min(sk.count, behind + q0 + 1)) : sk.count) / kKeys;
    const int any = w0 >= nq ? 0 : a.causal ? max(0, min(sk.count, behind + min(w0 + 32, nq))) : sk.count;

    const std::int64_t kv = static_cast<std::int64_t>(head / a.group) * D;
    const std::uint16_t* const k0 = a.k + sk.first * a.k_stride + kv;
    const std::uint16_t* const v0 = a.v + sk.first * a.v_stride + kv;
    // A tile's DMA instructions are dealt to the waves of its group.
    const int first_row = row_group * C::DMA_ROWS + lane / C::PIECES;
    auto stage = [&](const std::uint16_t* x, std::int64_t stride, int step, std::uint32_t to) {
        const std::uint32_t stride2 = static_cast<std::uint32_t>(stride) * 2u;
        const std::uint64_t p = reinterpret_cast<std::uint64_t>(x + static_cast<std::int64_t>(step) * kKeys * stride);
        const int rows = min(kKeys, sk.count - step * kKeys);
        const u32x4 r = {uniform(static_cast<std::uint32_t>(p)), uniform(static_cast<std::uint32_t>(p >> 32)) & 0xffffu,
                         uniform((rows - 1) * stride2 + 2u * D), kRawBufferFlags};
#pragma unroll
        for (int i = 0; i < (C::DMA + C::RG - 1) / C::RG; ++i) {
            if (C::DMA % C::RG != 0 && row_group + i * C::RG >= C::DMA) continue;
            const int t = first_row + i * C::RG * C::DMA_ROWS;
            lds_dma16(r, to + (row_group + i * C::RG) * 1024, t * stride2 + ((lane % C::PIECES) ^ C::swizzle(t)) * 16u);
        }
    };
    // Places of this lane's pieces: of K, pieces 2 ks + hi of row lane & 31; of
    // V, the transposing read of 16 lanes takes 4 halves of each of 4 rows
    // (4 hi + 8 e + 0..3 of a 16-row step) a lane and returns one column's four.
    int kat[KS], vat[DT][2];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kat[ks] = column * D + ((2 * ks + hi) ^ C::swizzle(column)) * 8;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int row = 8 * e + 4 * hi + ((lane & 15) >> 2);
            vat[dt][e] = row * D + ((4 * dt + 2 * (lane >> 4 & 1) + (lane >> 1 & 1)) ^ C::swizzle(row)) * 8 + (lane & 1) * 4;
        }
    auto value_fragment = [&](const std::uint16_t* tile_v, int step, int dt) {
        u32x2 v[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
            v[e] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                 (__attribute__((address_space(3))) s16x4*)(tile_v + vat[dt][e] + step * 16 * D)));
        return u32x4{v[0][0], v[0][1], v[1][0], v[1][1]};
    };

    floatx16 acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[dt][r] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    bool coarse = false;

    auto compute = [&](int step, const std::uint16_t* tile_k, const std::uint16_t* tile_v, auto masked, auto cleaned) {
        constexpr bool MASKED = decltype(masked)::value, CLEANED = decltype(cleaned)::value;
        const int j0 = step * kKeys;
        // Eight K fragments are read ahead of the products, then one for each
        // fragment used: an LDS read takes as long as four products.
        floatx16 s[TT];
        half8 kf[TT * KS];
#pragma unroll
        for (int i = 0; i < TT * KS; ++i) kf[i] = *reinterpret_cast<const half8*>(tile_k + kat[i / TT] + i % TT * 32 * D);
#pragma unroll
        for (int i = 0; i < TT * KS; ++i)
            s[i % TT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[i], q[i / TT], i >= TT ? s[i % TT] : floatx16{}, 0, 0, 0);
        constexpr int kAhead = TT * KS < 8 ? TT * KS : 8;
        __builtin_amdgcn_sched_group_barrier(kReads, kAhead, 0);
#pragma unroll
        for (int i = 0; i < TT * KS - kAhead; ++i) {
            __builtin_amdgcn_sched_group_barrier(kProducts, 1, 0);
            __builtin_amdgcn_sched_group_barrier(kReads, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(kProducts, kAhead, 0);
        // The first step's V fragments come in under the softmax.
        u32x4 vf[2][DT];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) vf[0][dt] = value_fragment(tile_v, 0, dt);
        __builtin_amdgcn_sched_barrier(0);
        half8 p[2 * TT];
        {
            if constexpr (MASKED) {
#pragma unroll
                for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (j0 + tt * 32 + 8 * (r >> 2) + 4 * hi + (r & 3) >= seen) s[tt][r] = -INFINITY;
            }
            // The NaN-propagating maximum of three is one instruction; a score that
            // is NaN leaves the maximum where it was, and its query becomes NaN.
            float tops[TT];
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
                tops[tt] = s[tt][0];
#pragma unroll
                for (int r = 1; r < 15; r += 2)
                    tops[tt] = __builtin_elementwise_maximum(__builtin_elementwise_maximum(tops[tt], s[tt][r]), s[tt][r + 1]);
            }
            float top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(tops[0], s[0][15]),
                                                      __builtin_elementwise_maximum(tops[TT - 1], s[TT - 1][15]));
            top = both_max(top) * a.scale2;
            if (__any(top - m > kMost)) {
                const float now = fmaxf(m, lifted(top)), keep = __builtin_amdgcn_exp2f(m - (now == -INFINITY ? 0.0f : now));
                m = now;
                coarse = __any(fabsf(m) >= kCoarse && m != -INFINITY);
                l *= keep;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[dt][r] *= keep;
            }
            float base = m == -INFINITY ? 0.0f : m, factor = a.scale2;
            if (coarse) {
                // One rounding of s factor - base would be of another number than the
                // score that the base was taken from, by up to half a unit of its last
                // place, and here that is a power of two. (The test costs 1% at 8160
                // tokens.)
#pragma unroll
                for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[tt][r] = opaque(s[tt][r] * factor) - base;
                base = 0.0f, factor = 1.0f;
            }
            // Plain additions: the dot-product instructions share the matrix cores'
            // pipe, and take 26 cycles instead of 5 beside another wave's products.
            float sum[2 * TT] = {};
#pragma unroll
            for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    const float x = __builtin_amdgcn_exp2f(fmaf(s[tt][r], factor, -base)),
                                y = __builtin_amdgcn_exp2f(fmaf(s[tt][r + 1], factor, -base));
                    const half2_t w = {static_cast<_Float16>(x), static_cast<_Float16>(y)};
                    sum[2 * tt] += x;
                    sum[2 * tt + 1] += y;
                    p[tt * 2 + (r >> 3)][r & 7] = w[0];
                    p[tt * 2 + (r >> 3)][(r & 7) + 1] = w[1];
                }
            l += sum[0] + sum[1];
            if constexpr (TT == 2) l += sum[2] + sum[3];
        }
#pragma unroll
        for (int st = 0; st < 2 * TT; ++st)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                u32x4 v = vf[st & 1][dt];
                if (st < 2 * TT - 1) vf[st & 1 ^ 1][dt] = value_fragment(tile_v, st + 1, dt);
                if constexpr (CLEANED) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        v[e] &= ~(((v[e] & 0x7c00u) == 0x7c00u ? 0xffffu : 0u) | ((v[e] & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u));
                }
                acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, v), p[st], acc[dt], 0, 0, 0);
                if constexpr (!CLEANED) __builtin_amdgcn_sched_barrier(0);
            }
    };

    // This group's buffers: K and V of one tile, then of the next.
    std::uint16_t* const tiles_of_group = lds + key_group * 4 * C::TILE;
    const std::uint32_t to = uniform(lds_address(tiles_of_group));
    auto stage_both = [&](int step, int buffer) {
        stage(k0, a.k_stride, step, to + buffer * C::TILE * 4);
        stage(v0, a.v_stride, step, to + buffer * C::TILE * 4 + C::TILE * 2);
    };
    if (key_group < steps) stage_both(key_group, 0);
    // Whether the pieces of V that this wave staged hold an infinity or NaN.
    auto any_odd = [&](const std::uint16_t* tile_v) {
        typedef std::uint16_t u16x2 __attribute__((ext_vector_type(2)));
        u16x2 top = {0, 0};
#pragma unroll
        for (int i = 0; i < (C::DMA + C::RG - 1) / C::RG; ++i) {
            if (C::DMA % C::RG != 0 && row_group + i * C::RG >= C::DMA) continue;
            const u32x4 v = *reinterpret_cast<const u32x4*>(tile_v + (row_group + i * C::RG) * 512 + lane * 8);
#pragma unroll
            for (int e = 0; e < 4; ++e) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, v[e] & 0x7fff7fffu));
        }
        return __any(max(top[0], top[1]) >= 0x7c00u) != 0;
    };
    int* const flags = reinterpret_cast<int*>(lds + C::TILES);  // [2][WAVES]
    auto arrived = [&](auto&& after) {
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's DMA of the tile
        after();
        __syncthreads();
    };
    auto turn = [&](int step, int buffer, auto masked, auto cleaned) {
        if (step + C::KG < steps) stage_both(step + C::KG, buffer ^ 1);
        const std::uint16_t* const tile = tiles_of_group + buffer * 2 * C::TILE;
        if (!masked || step * kKeys < any) compute(step, tile, tile + C::TILE, masked, cleaned);
    };
    // All groups take as many turns; `any` is at most `steps` tiles. First the
    // tiles that are seen whole; then those with masked keys, whose values get
    // the weight 0, while all of them are finite; then, cleaned of infinities and
    // NaN, the rest.
    int round = 0, buffer = 0;
    for (; (round + 1) * C::KG <= clear; ++round, buffer ^= 1) {
        arrived([] {});
        turn(round * C::KG + key_group, buffer, std::false_type{}, std::false_type{});
    }
    for (; round * C::KG < steps; ++round, buffer ^= 1) {
        const int step = round * C::KG + key_group;
        arrived([&] { flags[buffer * C::WAVES + wave] = step < steps && any_odd(tiles_of_group + (2 * buffer + 1) * C::TILE); });
        if (__any(flags[buffer * C::WAVES + lane % C::WAVES])) break;
        turn(step, buffer, std::true_type{}, std::false_type{});
    }
    const int cleaned_from = round * C::KG * kKeys;
    for (; round * C::KG < steps; ++round, buffer ^= 1) {
        arrived([] {});
        turn(round * C::KG + key_group, buffer, std::true_type{}, std::true_type{});
    }

    if constexpr (C::KG > 1) {
        // The other groups hand their states to the first, lane by lane.
        constexpr int kWords = DT * 4 + 1, kLanes = C::RG * 64;
        static_assert(sizeof(floatx4) * kWords * kLanes * (C::KG - 1) <= C::LDS);
        floatx4* const states = reinterpret_cast<floatx4*>(lds) + row_group * 64 + lane;
        __syncthreads();
        if (key_group > 0) {
            floatx4* const to_state = states + (key_group - 1) * kWords * kLanes;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    to_state[(dt * 4 + g) * kLanes] = floatx4{acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]};
            to_state[DT * 4 * kLanes] = floatx4{m, l, 0.0f, 0.0f};
        }
        __syncthreads();
        if (key_group > 0) return;
#pragma unroll
        for (int k = 0; k < C::KG - 1; ++k) {
            const floatx4* const from = states + k * kWords * kLanes;
            const floatx4 st = from[DT * 4 * kLanes];
            const float now = fmaxf(m, st[0]), base = now == -INFINITY ? 0.0f : now;
            const float mine = __builtin_amdgcn_exp2f(m - base), other = __builtin_amdgcn_exp2f(st[0] - base);
            m = now;
            l = l * mine + st[1] * other;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const floatx4 v = from[(dt * 4 + g) * kLanes];
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[dt][4 * g + e] = acc[dt][4 * g + e] * mine + v[e] * other;
                }
        }
    }

    // A query that sees an infinity or NaN gets it, however small the weight: the
    // first place of each in a column decides, before the query's end or not. They
    // are looked for where values were cleaned, and from the first key on where a
    // sum shows that it met one (8160 tokens, 16 heads of 128, an infinity at the
    // first key: 1.25 ms instead of 0.27; a sum that is finite costs its test).
    bool odd = false;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) odd |= !is_finite(acc[dt][r]);
    odd = __any(odd) != 0;
    if (odd || cleaned_from < keys) {
        constexpr int PER = D / 64;  // columns of a lane
        int first[3][PER];
        for (int kind = 0; kind < 3; ++kind)
            for (int c = 0; c < PER; ++c) first[kind][c] = INT_MAX;
#pragma unroll 4
        for (int j = odd ? 0 : cleaned_from; j < keys; ++j) {
            const std::uint16_t* const row = v0 + j * a.v_stride + lane * PER;
            std::uint32_t v;
            if constexpr (PER == 2) v = *reinterpret_cast<const std::uint32_t*>(row);
            else v = *row;
#pragma unroll
            for (int c = 0; c < PER; ++c) {
                const unsigned kind = OddValues::of(static_cast<std::uint16_t>(v >> 16 * c));
#pragma unroll
                for (int k = 0; k < 3; ++k)
                    if (kind == 1u << k) first[k][c] = min(first[k][c], j);
            }
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int holder = (dt * 32 + 8 * (r >> 2) + 4 * hi + (r & 3)) / PER;
                OddValues seen_here;
#pragma unroll
                for (int k = 0; k < 3; ++k)
                    if (__shfl(first[k][(r & 3) % PER], holder) < seen) seen_here.seen |= 1u << k;
                acc[dt][r] = seen_here.sum(acc[dt][r]);
            }
    }

    const float sum = both_sum(l), r = sum == 0.0f ? 0.0f : 1.0f / sum;
    if (i_query >= nq) return;
    std::uint16_t* out = a.out + (sq.first + i_query) * a.out_stride + static_cast<std::int64_t>(head) * D + 4 * hi;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<uint2*>(out + dt * 32 + 8 * g) =
                make_uint2(pack_rounded(acc[dt][4 * g] * r, acc[dt][4 * g + 1] * r),
                           pack_rounded(acc[dt][4 * g + 2] * r, acc[dt][4 * g + 3] * r));
}

template <class C>
void launch_prompt(const PromptArgs& a, hipStream_t s)
{
    const int tiles = (a.longest_q + C::ROWS - 1) / C::ROWS;
    // Tiles, at most, from what the host knows; a multiple of the XCDs' number.
    // Many sequences go by turns where they fit a tile each or nearly all have as
    // many tiles as the longest: a workgroup then finds its tile without reading
    // past other sequences. us, by turns / one after the other: 1000 of one query,
    // 16 heads of 64, 71 / 104, on 100 keys 115 / 154; 300 of 20 27 / 30; 200 of one
    // query on 900 keys, heads of 128, 205 / 205; 70 of 200 59.8 / 63.3; one of 4080
    // and 99 of 100 193 / 113; 200 of 30 to 240, heads of 64, 60 / 50.
    const std::int64_t by_longest = static_cast<std::int64_t>(tiles) * a.sequences, full = a.q_tokens / C::ROWS;
    const bool by_turns = a.sequences == 1 || (a.sequences > 64 && (tiles == 1 || by_longest <= full + a.sequences * 3LL / 4));
    const std::int64_t most = by_turns ? by_longest : std::min(by_longest, full + a.sequences);
    const std::int64_t grid = (most * a.q_heads + kXcds - 1) / kXcds * kXcds;
    require(launchable(grid, C::WAVES * 64), "attention_prompt", "too many sequences, heads and queries in one call");
    prompt_kernel<C><<<static_cast<unsigned>(grid), C::WAVES * 64, C::LDS, s>>>(a, tiles, by_turns);
}

// Workgroups of 128 queries, two a CU, read each key tile once for 128 queries
// and balance well; they need two of them for every CU. Fewer queries are
// given more waves by key groups, at first beside as many queries, then fewer:
// 96 where those workgroups just fit the CUs, so that they all take part.
// Tiles of 32 keys leave LDS for two buffers of four or eight groups; eight
// groups take longer to start than they save on up to 512 keys.
// us, the same work by the alternatives (16 query heads, causal):
//   heads of 128               (4,1)  (4,2)  (2,4)  (1,4)  (8,1)
//     10 on 1500                31.3   24.7   20.0   17.7   39.4
//     240                       10.9   11.9   10.5    9.1   14.9
//     920                       22.9   20.8   17.5   20.6   28.8
//     2040                      44.0   36.9   37.2   57.8   56.5
//     4080                      93.3   84.1    112    173    109
//     1..2040 packed            54.0   66.6   96.4    144   62.6
//     4 x 2040                  83.7    101    145    235   86.7
//     8160                       289    295    377    589    277
//   heads of 64                (4,1)  (4,2)  (4,3)  (3,4)  (2,4)  (1,4)  (1,8)
//     10 on 1500                22.1   18.2   17.4   14.7   12.9   11.5   11.6
//     240                        8.0    8.2    9.4    8.6    7.4    6.5    7.6
//     920                       15.9   14.3   14.4   13.0   10.9   14.6   15.7
//     1400                      22.0   18.8   19.1   17.0   16.0   23.5   25.2
//     2040                      29.7   24.8   23.8   23.4   22.7   35.8   37.9
//     700 and 600, not causal   14.2   13.1   13.4   12.8   19.3   23.4   25.9
//     920 on 4600, 460 on 3001  60.5   47.6   44.1   38.9   49.6   65.2   61.9
//     4080                      58.6   51.9   52.7   62.5   64.9    105    105
//     1..2040 packed            36.2   41.4   46.5   54.9   63.1   97.8    106
//     8160                       172    182    178    193    215    343    326
// 256 queries a workgroup halve the key traffic again, which pays where a
// sequence is long enough for its last, partly seen tiles not to count.
template <int D>
void launch_prompt(const PromptArgs& a, hipStream_t s)
{
    const std::int64_t cus = conv::cu_count();
    auto workgroups = [&](int queries) {  // at most, from what the host knows
        const std::int64_t by_longest = static_cast<std::int64_t>((a.longest_q + queries - 1) / queries) * a.sequences;
        return a.q_heads * std::min(by_longest, static_cast<std::int64_t>(a.q_tokens / queries) + a.sequences);
    };
    if (workgroups(32) <= cus) {
        if constexpr (D == 128) launch_prompt<PromptCfg<D, 1, 4, 32, 2>>(a, s);
        else if (a.k_tokens > 512LL * a.sequences) launch_prompt<PromptCfg<64, 1, 8, 32, 2>>(a, s);
        else launch_prompt<PromptCfg<64, 1, 4, 64, 2>>(a, s);
    }
    else if (workgroups(64) <= cus) launch_prompt<PromptCfg<D, 2, 4, D == 64 ? 64 : 32, 2>>(a, s);
    else if (D == 64 && workgroups(96) <= cus) launch_prompt<PromptCfg<64, 3, 4, 64, 3>>(a, s);
    else if (D == 64 && workgroups(128) <= cus) launch_prompt<PromptCfg<64, 4, 3, 64, 3>>(a, s);
    else if (workgroups(128) <= 2 * cus) launch_prompt<PromptCfg<D, 4, 2, 64, 2>>(a, s);
    else if (D == 128 && a.longest_q >= 4096 && workgroups(128) >= 4 * cus && static_cast<std::int64_t>(a.longest_q) * a.sequences <= 2 * static_cast<std::int64_t>(a.q_tokens))
        launch_prompt<PromptCfg<128, 8, 1, 64, 2>>(a, s);
    else launch_prompt<PromptCfg<D, 4, 1, 64, D == 64 ? 3 : 2>>(a, s);
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
    a.q_tokens = d->q_tokens, a.k_tokens = d->k_tokens, a.longest_q = std::min(d->longest_q, d->q_tokens), a.causal = d->causal != 0;
    a.cus = conv::cu_count();
    a.scale2 = std::fabs(d->scale) * 1.4426950408889634f, a.negate = d->scale < 0.0f;
    // The matrix-core kernel addresses a tile's rows by 32-bit byte offsets,
    // and scales masked scores (-inf) by the factor, which must not be 0.
    constexpr std::int64_t kFarthest = std::int64_t{1} << 23;
    const bool rows = vector_rows(d->q, d->q_stride) && vector_rows(d->out, d->out_stride) && vector_rows(d->k, d->k_stride) &&
                      vector_rows(d->v, d->v_stride) && d->k_stride < kFarthest && d->v_stride < kFarthest && a.scale2 > 1e-30f;
    if (rows && d->head_dim == 128) launch_prompt<128>(a, s);
    else if (rows && d->head_dim == 64) launch_prompt<64>(a, s);
    else {
        require(launchable(d->q_tokens, 64), op, "too many sequences, heads and queries in one call");
        prompt_any_kernel<<<dim3(static_cast<unsigned>(d->q_tokens), static_cast<unsigned>(d->q_heads)), 64, 0, s>>>(a);
    }
    check(hipGetLastError(), "attention_prompt launch");
}

}  // namespace
}  // namespace mlvc_hip

using namespace mlvc_hip;

extern "C" int mlvc_hip_attention_prompt(const mlvc_hip_attention_prompt_desc* desc, mlvc_hip_stream s)
{
    return guard([&] { attention_prompt(desc, to_stream(s)); });
}
