// Attention of packed sequences (one pass over the keys with the running
// maximum and sum of the softmax).
//
//   m' = max(m, max_j s_j),  l' = l e^(m - m') + sum_j e^(s_j - m'),
//   o' = o e^(m - m') + sum_j e^(s_j - m') v_j,   out = o / l
//
// in powers of two: s is scaled by log2(e), so each exponential is one
// v_exp_f32.

#include "attention.hpp"

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
    int sequences, q_heads, group, dim, q_tokens, k_tokens, longest_q, causal, negate;
    float scale2;  // |scale| log2(e); negate: scale is negative
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
constexpr int kKeys = 64;          // keys of a tile
constexpr int kProducts = 0x8, kReads = 0x100;  // instruction groups of sched_group_barrier: MFMA, LDS reads
constexpr float kSlack = 8.0f;     // how far, in powers of two, a score may pass the running maximum before it moves

__device__ __forceinline__ std::uint32_t uniform(std::uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }

// 16 bytes a lane from `at` bytes into a raw buffer to LDS, lane after lane;
// out of the buffer's range, zeros. In assembly because the compiler lets every
// LDS read that follows the builtin wait for it: here the tile that is read and
// the one being filled are never the same, and the caller waits (vmcnt) and
// synchronises before it turns to the next.
__device__ __forceinline__ void lds_dma16(u32x4 buffer, std::uint32_t to, std::uint32_t at)
{
    asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(at), "s"(buffer) : "memory", "m0");
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

// Heads of D values, rows on 16 bytes. A workgroup of WAVES waves takes
// WAVES * QT * 32 queries of a head; a wave holds QT * 32 of them as columns
// of S^T = K Q^T (32x32x16 products, keys as rows), so that
//   * a lane's scores all belong to one query: the softmax needs one exchange,
//     between the two lanes of a column;
//   * the accumulator registers of S^T, rounded to FP16, are the B operand of
//     O^T += V^T P^T as they stand (the 16 keys of a step are taken in the order
//     the registers hold them), so weights never leave the lane.
// Tiles of 64 keys are staged by LDS DMA, double-buffered, 16-byte pieces of a
// row permuted (piece ^ f(row)) so that both reads are free of bank conflicts:
// K rows by 16 bytes, V by the transposing read. Rows past a sequence's end are
// out of the buffer's range and read as zeros.
//
// The running maximum moves only when a score passes it by 2^8 (weights up to
// 2^8 lose nothing in FP16 or in the FP32 sums), so the accumulators are seldom
// rescaled. Weights are rounded to FP16, the type the matrix cores take beside
// V: one rounding of 2^-11 each, no more than the output's own.
template <int D_, int WAVES_, int QT_>
struct PromptCfg {
    static constexpr int D = D_, WAVES = WAVES_, QT = QT_;
    static constexpr int ROWS = WAVES * QT * 32;     // queries of a workgroup
    static constexpr int PIECES = D / 8;             // 16-byte pieces of a row
    static constexpr int DMA_ROWS = 64 / PIECES;     // rows of a DMA instruction
    static constexpr int DMA = kKeys / DMA_ROWS;     // instructions of a tile
    static constexpr int TILE = kKeys * D;           // halves
    static constexpr size_t LDS = 4 * TILE * 2;      // K and V, two buffers
    // Piece p of row t is kept at place p ^ swizzle(t): 16 rows of one piece
    // (a K read) fall on all 64 banks, and so do 4 rows of 4 pieces (a V read).
    __host__ __device__ static constexpr int swizzle(int t)
    {
        return D == 128 ? 4 * (t & 3) + (t >> 2 & 3) : 4 * (t >> 1 & 1) + (t >> 2 & 3);
    }
};

template <class C>
__global__ __launch_bounds__(C::WAVES * 64, 2) void prompt_kernel(PromptArgs a, int tiles)
{
    constexpr int D = C::D, QT = C::QT, KS = D / 16, DT = D / 32;
    extern __shared__ __attribute__((aligned(16))) std::uint16_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int column = lane & 31, hi = lane >> 5;

    // Workgroup i runs on XCD i % 8: with a multiple of 8 heads an XCD keeps the
    // same heads, of all sequences, so their keys stay in its L2. The last
    // tiles of the queries, which see most keys, go first.
    int head, n, tile;
    if (a.q_heads % kXcds == 0) {
        const int per = a.q_heads / kXcds, i = blockIdx.x / kXcds, j = i / per;
        head = blockIdx.x % kXcds * per + i % per;
        n = j % a.sequences;
        tile = tiles - 1 - j / a.sequences;
    } else {
        const int j = blockIdx.x / a.q_heads;
        head = blockIdx.x % a.q_heads;
        n = j % a.sequences;
        tile = tiles - 1 - j / a.sequences;
    }
    const Span sq = span(a.q_starts, n, a.q_tokens), sk = span(a.k_starts, n, a.k_tokens);
    const int q0 = tile * C::ROWS, nq = min(sq.count, a.longest_q);
    if (q0 >= nq) return;
    const int behind = sk.count - sq.count;  // keys before the first query
    const int last = min(q0 + C::ROWS, nq) - 1;
    const int keys = a.causal ? max(0, min(sk.count, behind + last + 1)) : sk.count;  // seen by any query here
    const int steps = (keys + kKeys - 1) / kKeys;

    // This wave's queries, as B fragments.
    const int w0 = q0 + wave * QT * 32;
    half8 q[QT][KS];
    int seen[QT];  // keys this lane's query sees
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const int i = w0 + qt * 32 + column, at = min(i, nq - 1);
        const std::uint16_t* row = a.q + (sq.first + at) * a.q_stride + static_cast<std::int64_t>(head) * D + hi * 8;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            u32x4 v = *reinterpret_cast<const u32x4*>(row + ks * 16);
            if (a.negate)
                for (int e = 0; e < 4; ++e) v[e] ^= 0x80008000u;
            q[qt][ks] = __builtin_bit_cast(half8, v);
        }
        seen[qt] = a.causal ? max(0, min(sk.count, behind + at + 1)) : sk.count;
    }
    // Tiles that every query of the workgroup sees whole, and keys that any of this wave's sees.
    const int clear = (a.causal ? max(0, min(sk.count, behind + q0 + 1)) : sk.count) / kKeys;
    const int any = w0 >= nq ? 0 : a.causal ? max(0, min(sk.count, behind + min(w0 + QT * 32, nq))) : sk.count;

    const std::int64_t kv = static_cast<std::int64_t>(head / a.group) * D;
    const std::uint16_t* const k0 = a.k + sk.first * a.k_stride + kv;
    const std::uint16_t* const v0 = a.v + sk.first * a.v_stride + kv;
    const int drow = lane / C::PIECES, first_row = wave * C::DMA_ROWS + drow;
    const int piece = (lane % C::PIECES) ^ C::swizzle(first_row);  // the same for all of this lane's rows
    static_assert(C::DMA_ROWS * C::WAVES % 16 == 0 && C::DMA % C::WAVES == 0);
    auto stage = [&](const std::uint16_t* x, std::int64_t stride, int step, std::uint32_t to) {
        const std::uint32_t stride2 = static_cast<std::uint32_t>(stride) * 2u;
        const std::uint64_t p = reinterpret_cast<std::uint64_t>(x + static_cast<std::int64_t>(step) * kKeys * stride);
        const int rows = min(kKeys, sk.count - step * kKeys);
        const u32x4 r = {uniform(static_cast<std::uint32_t>(p)), uniform(static_cast<std::uint32_t>(p >> 32)) & 0xffffu,
                         uniform((rows - 1) * stride2 + 2u * D), kRawBufferFlags};
        const std::uint32_t at = first_row * stride2 + piece * 16u;
#pragma unroll
        for (int i = 0; i < C::DMA / C::WAVES; ++i)
            lds_dma16(r, to + (wave + i * C::WAVES) * 1024, at + i * C::WAVES * C::DMA_ROWS * stride2);
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

    floatx16 acc[QT][DT];
    float m[QT], l[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        m[qt] = -INFINITY, l[qt] = 0.0f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[qt][dt][r] = 0.0f;
    }

    auto compute = [&](int step, const std::uint16_t* tile_k, const std::uint16_t* tile_v, auto masked) {
        constexpr bool MASKED = decltype(masked)::value;
        const int j0 = step * kKeys;
        // Eight K fragments are read ahead of the products, then one for each
        // fragment used: an LDS read takes as long as four products.
        floatx16 s[QT][2];
        half8 kf[2 * KS];
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i) kf[i] = *reinterpret_cast<const half8*>(tile_k + kat[i >> 1] + (i & 1) * 32 * D);
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i)
#pragma unroll
            for (int qt = 0; qt < QT; ++qt)
                s[qt][i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[i], q[qt][i >> 1], i > 1 ? s[qt][i & 1] : floatx16{}, 0, 0, 0);
        __builtin_amdgcn_sched_group_barrier(kReads, 8, 0);
#pragma unroll
        for (int i = 0; i < 2 * KS - 8; ++i) {
            __builtin_amdgcn_sched_group_barrier(kProducts, QT, 0);
            __builtin_amdgcn_sched_group_barrier(kReads, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(kProducts, 8 * QT, 0);
        // The first step's V fragments come in under the softmax.
        u32x4 vf[2][DT];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) vf[0][dt] = value_fragment(tile_v, 0, dt);
        __builtin_amdgcn_sched_barrier(0);
        half8 p[QT][4];
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
            if constexpr (MASKED) {
#pragma unroll
                for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (j0 + tt * 32 + 8 * (r >> 2) + 4 * hi + (r & 3) >= seen[qt]) s[qt][tt][r] = -INFINITY;
            }
            // The NaN-propagating maximum of three is one instruction; a score that
            // is NaN leaves the maximum where it was, and its query becomes NaN.
            float top = __builtin_elementwise_maximum(s[qt][0][0], s[qt][1][0]);
#pragma unroll
            for (int r = 1; r < 16; ++r)
                top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top, s[qt][0][r]), s[qt][1][r]);
            top = both_max(top) * a.scale2;
            if (__any(top > m[qt] + kSlack)) {
                const float now = fmaxf(m[qt], top), keep = __builtin_amdgcn_exp2f(m[qt] - (now == -INFINITY ? 0.0f : now));
                m[qt] = now;
                l[qt] *= keep;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[qt][dt][r] *= keep;
            }
            const float base = m[qt] == -INFINITY ? 0.0f : m[qt];
            const half2_t ones = {static_cast<_Float16>(1.0f), static_cast<_Float16>(1.0f)};
            float sum[2] = {0.0f, 0.0f};
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    const float x = __builtin_amdgcn_exp2f(fmaf(s[qt][tt][r], a.scale2, -base)),
                                y = __builtin_amdgcn_exp2f(fmaf(s[qt][tt][r + 1], a.scale2, -base));
                    const half2_t w = {static_cast<_Float16>(x), static_cast<_Float16>(y)};
                    sum[tt] = __builtin_amdgcn_fdot2(w, ones, sum[tt], false);
                    p[qt][tt * 2 + (r >> 3)][r & 7] = w[0];
                    p[qt][tt * 2 + (r >> 3)][(r & 7) + 1] = w[1];
                }
            l[qt] += sum[0] + sum[1];
        }
        std::uint32_t odd = 0;
#pragma unroll
        for (int st = 0; st < 4; ++st)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                u32x4 v = vf[st & 1][dt];
                if (st < 3) vf[st & 1 ^ 1][dt] = value_fragment(tile_v, st + 1, dt);
                if constexpr (MASKED) {
                    // Values whose weight may be zero must be finite: 0 * inf is NaN.
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const std::uint32_t lo = (v[e] & 0x7c00u) == 0x7c00u ? 0xffffu : 0u,
                                            up = (v[e] & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u;
                        odd |= lo | up;
                        v[e] &= ~(lo | up);
                    }
                }
#pragma unroll
                for (int qt = 0; qt < QT; ++qt)
                    acc[qt][dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, v), p[qt][st], acc[qt][dt], 0, 0, 0);
                if constexpr (!MASKED) __builtin_amdgcn_sched_barrier(0);
            }
        if constexpr (MASKED) {
            // What was left out above: a query that sees an infinity or NaN gets
            // it. Counted by products of 0 / 1 matrices, once for +inf and NaN,
            // once for -inf and NaN.
            if (__any(odd != 0)) {
#pragma unroll
                for (int qt = 0; qt < QT; ++qt)
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
                        for (int sign = 0; sign < 2; ++sign) {
                            floatx16 count = {};
                            for (int st = 0; st < 4; ++st) {
                                const u32x4 vf = value_fragment(tile_v, st, dt);
                                half8 is, sees;
#pragma unroll
                                for (int e = 0; e < 8; ++e) {
                                    const std::uint32_t v = vf[e >> 1] >> (16 * (e & 1)) & 0xffffu;
                                    const bool bad = (v & 0x7fffu) > 0x7c00u || v == (sign ? 0xfc00u : 0x7c00u);
                                    is[e] = static_cast<_Float16>(bad ? 1.0f : 0.0f);
                                    const int j = j0 + st * 16 + 8 * (e >> 2) + 4 * hi + (e & 3);
                                    sees[e] = static_cast<_Float16>(j < seen[qt] ? 1.0f : 0.0f);
                                }
                                count = __builtin_amdgcn_mfma_f32_32x32x16_f16(is, sees, count, 0, 0, 0);
                            }
#pragma unroll
                            for (int r = 0; r < 16; ++r)
                                if (count[r] > 0.0f) acc[qt][dt][r] += sign ? -INFINITY : INFINITY;
                        }
            }
        }
    };

    std::uint16_t* const tile_k = lds;
    std::uint16_t* const tile_v = lds + 2 * C::TILE;
    const std::uint32_t to_k = uniform(lds_address(tile_k)), to_v = uniform(lds_address(tile_v));
    if (steps > 0) {
        stage(k0, a.k_stride, 0, to_k);
        stage(v0, a.v_stride, 0, to_v);
    }
    auto turn = [&](int step, auto masked) {
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's DMA of the tile
        __syncthreads();
        const int now = step & 1, next = now ^ 1;
        if (step + 1 < steps) {
            stage(k0, a.k_stride, step + 1, to_k + next * C::TILE * 2);
            stage(v0, a.v_stride, step + 1, to_v + next * C::TILE * 2);
        }
        if (!masked || step * kKeys < any) compute(step, tile_k + now * C::TILE, tile_v + now * C::TILE, masked);
    };
    int step = 0;
    for (; step < clear; ++step) turn(step, std::false_type{});
    for (; step < steps; ++step) turn(step, std::true_type{});

#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const int i = w0 + qt * 32 + column;
        const float sum = both_sum(l[qt]), r = sum == 0.0f ? 0.0f : 1.0f / sum;
        if (i >= nq) continue;
        std::uint16_t* out = a.out + (sq.first + i) * a.out_stride + static_cast<std::int64_t>(head) * D + 4 * hi;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<uint2*>(out + dt * 32 + 8 * g) =
                    make_uint2(pack_rounded(acc[qt][dt][4 * g] * r, acc[qt][dt][4 * g + 1] * r),
                               pack_rounded(acc[qt][dt][4 * g + 2] * r, acc[qt][dt][4 * g + 3] * r));
    }
}

template <class C>
void launch_prompt(const PromptArgs& a, hipStream_t s)
{
    const int tiles = (a.longest_q + C::ROWS - 1) / C::ROWS;
    const std::int64_t grid = static_cast<std::int64_t>(tiles) * a.q_heads * a.sequences;
    require(grid <= INT_MAX, "attention_prompt", "too many sequences, heads and queries in one call");
    prompt_kernel<C><<<static_cast<unsigned>(grid), C::WAVES * 64, C::LDS, s>>>(a, tiles);
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
    a.scale2 = std::fabs(d->scale) * 1.4426950408889634f, a.negate = d->scale < 0.0f;
    // The matrix-core kernel addresses a tile's rows by 32-bit byte offsets,
    // and scales masked scores (-inf) by the factor, which must not be 0.
    constexpr std::int64_t kFarthest = std::int64_t{1} << 23;
    const bool rows = vector_rows(d->q, d->q_stride) && vector_rows(d->out, d->out_stride) && vector_rows(d->k, d->k_stride) &&
                      vector_rows(d->v, d->v_stride) && d->k_stride < kFarthest && d->v_stride < kFarthest && a.scale2 > 1e-30f;
    // 256 queries a workgroup read the keys half as often as 128, and one
    // such workgroup a CU is as many waves; 8160 tokens, 16 heads of 128: 283
    // against 301 us. They need work for every CU twice over, and sequences of
    // like length (packed 1..2040: 68 against 67 us).
    const std::int64_t large = static_cast<std::int64_t>(d->q_tokens) / 256 * d->q_heads;
    const bool even = static_cast<std::int64_t>(d->longest_q) * d->sequences <= 2 * static_cast<std::int64_t>(d->q_tokens);
    const bool eight = even && large >= 2 * conv::cu_count() - d->q_heads;
    if (rows && d->head_dim == 128) eight ? launch_prompt<PromptCfg<128, 8, 1>>(a, s) : launch_prompt<PromptCfg<128, 4, 1>>(a, s);
    else if (rows && d->head_dim == 64) eight ? launch_prompt<PromptCfg<64, 8, 1>>(a, s) : launch_prompt<PromptCfg<64, 4, 1>>(a, s);
    else
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
