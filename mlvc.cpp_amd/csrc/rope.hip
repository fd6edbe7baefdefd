// Norm of queries and keys per head and their rotation by position, one pass.
//
//   x' = x rsqrt(mean(x^2) + eps) w,  (a, b) -> (a c - b s, b c + a s)
//
// Bound by memory: a row of head_dim halves is read and written once. The
// cosines and sines belong to a token and are shared by its heads, so a
// workgroup computes those of its tokens into LDS first. A phase p f is
// reduced to one turn in FP64 (four operations for each of rot_dim / 2
// frequencies of a token): in FP32 the product alone is 4e-3 radians off at
// position 65536.

#include "attention.hpp"

#include <algorithm>

namespace mlvc_hip {
namespace {

constexpr int kBlock = 256;

struct RopeArgs {
    const std::uint16_t* in[2];   // q, k
    std::uint16_t* out[2];
    const std::uint16_t* weight[2];
    std::int64_t in_stride[2], out_stride[2];
    int heads[2];
    const std::int32_t* positions;
    const double* freqs;
    int tokens, dim, rot;
    float eps, inv_dim, rot_scale;
    int pairs;  // adjacent pairs (rope_any_kernel)
};

// (m cos, m sin) of position p at frequency f.
__device__ __forceinline__ float2 turn(std::int32_t p, double f, float m)
{
    const double turns = static_cast<double>(p) * (f * 0.15915494309189535);
    const float part = static_cast<float>(turns - __builtin_rint(turns));
    float s, c;
    sincospif(2.0f * part, &s, &c);
    return make_float2(m * c, m * s);
}

// Heads of at most 8 * LANES values, a multiple of 8: LANES lanes hold a row, 8
// values each, and a wave holds 64 / LANES rows. A lane has both values of its
// pairs: 8 adjacent values where pairs are adjacent, else 4 of the first half
// of the rotated part and their 4 partners (8 adjacent ones past that part).
// A row is worked on while the next one is on its way, and a workgroup takes
// every gridDim.x-th token, so that the GPU reads and writes one narrow stretch
// at a time. At 8160 tokens of 32 + 8 heads of 128, 64 values of each rotated,
// 167 MB in and out: 33.6 us, 5.0 TB/s, a copy's rate (neighbouring tokens to a
// workgroup 34.7; two rows on their way 34.5, three 35.6); 4080 tokens 14.8 us.
// Stores past the caches take 27.3 us alone, but the attention that reads the
// result next then takes longer by as much or more (4 sequences of 1020 tokens,
// both kernels: 74.8 us, 71.5 with plain stores), so the result stays in the
// caches.
template <int LANES, bool PAIRS>
__global__ __launch_bounds__(kBlock) void rope_rows_kernel(RopeArgs a)
{
    extern __shared__ float2 table[];  // [per][rot / 2]
    const int t0 = blockIdx.x, every = gridDim.x, nt = (a.tokens - t0 + every - 1) / every, half = a.rot >> 1;
    const int lane = threadIdx.x % LANES, heads = a.heads[0] + a.heads[1];
    const bool mine = lane * 8 < a.dim, turned = lane * 8 < a.rot;
    // First values of the lane's two runs of 4; those of lane 0 past the row.
    const int d0 = !mine ? 0 : PAIRS || !turned ? lane * 8 : lane * 4, d1 = !mine || PAIRS || !turned ? d0 + 4 : half + d0;

    constexpr int kStep = kBlock / LANES;
    const int step_t = kStep / heads, step_h = kStep % heads;
    struct Row {
        int t, h;
    };
    struct Eight {
        uint2 lo, hi;
    };
    auto further = [&](Row r) {
        r.h += step_h, r.t += step_t;
        if (r.h >= heads) r.h -= heads, ++r.t;
        return r;
    };
    // Queries or keys, lane by lane: a choice of two values, where an index
    // into the arguments would be a load from memory.
    auto of = [&](Row r, auto q, auto k) { return r.h >= a.heads[0] ? k : q; };
    auto place = [&](int t, Row r, auto q, auto k, std::int64_t q_stride, std::int64_t k_stride) {
        return of(r, q, k) + (t0 + static_cast<std::int64_t>(t) * every) * of(r, q_stride, k_stride) + (r.h - of(r, 0, a.heads[0])) * a.dim;
    };
    auto load = [&](const std::uint16_t* p) {
        if constexpr (PAIRS) {
            const u32x4 v = *reinterpret_cast<const u32x4*>(p + d0);
            return Eight{make_uint2(v[0], v[1]), make_uint2(v[2], v[3])};
        } else {
            return Eight{*reinterpret_cast<const uint2*>(p + d0), *reinterpret_cast<const uint2*>(p + d1)};
        }
    };
    // Past the last token, that one again: without a branch the loads stay in flight.
    auto fetch = [&](Row r) { return load(place(min(r.t, nt - 1), r, a.in[0], a.in[1], a.in_stride[0], a.in_stride[1])); };
    const int group = threadIdx.x / LANES;
    Row now{group / heads, group % heads};
    Eight raw = fetch(now);

    for (int i = threadIdx.x; i < nt * half; i += kBlock) {
        const int t = i / half;
        table[i] = turn(a.positions[t0 + static_cast<std::int64_t>(t) * every], a.freqs[i - t * half], a.rot_scale);
    }
    const bool normed[2] = {a.weight[0] != nullptr, a.weight[1] != nullptr};
    const Eight w[2] = {normed[0] ? load(a.weight[0]) : Eight{}, normed[1] ? load(a.weight[1]) : Eight{}};
    __syncthreads();

    auto widen = [](const Eight& v, float* x) {
        x[0] = lo_f16(v.lo.x), x[1] = hi_f16(v.lo.x), x[2] = lo_f16(v.lo.y), x[3] = hi_f16(v.lo.y);
        x[4] = lo_f16(v.hi.x), x[5] = hi_f16(v.hi.x), x[6] = lo_f16(v.hi.y), x[7] = hi_f16(v.hi.y);
    };
    for (Row next; now.t < nt; now = next) {
        float x[8];
        widen(raw, x);
        next = further(now);
        raw = fetch(next);
        if (normed[0] || normed[1]) {
            float sum = 0.0f, f[8];
            if (!mine)
                for (int i = 0; i < 8; ++i) x[i] = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
            const float r = rsqrtf(fmaf(group_sum<LANES>(sum), a.inv_dim, a.eps));
            const Eight wide = {make_uint2(of(now, w[0].lo.x, w[1].lo.x), of(now, w[0].lo.y, w[1].lo.y)),
                                make_uint2(of(now, w[0].hi.x, w[1].hi.x), of(now, w[0].hi.y, w[1].hi.y))};
            widen(wide, f);
            if (of(now, normed[0], normed[1])) {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = x[i] * r * f[i];
            }
        }
        if (turned) {
            const float2* cs = table + now.t * half + lane * 4;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float& p = x[PAIRS ? 2 * i : i];
                float& q = x[PAIRS ? 2 * i + 1 : i + 4];
                if (PAIRS && lane * 8 + 2 * i >= a.rot) continue;  // adjacent pairs may end inside a lane
                const float2 c = cs[i];
                const float y = p * c.x - q * c.y;
                q = q * c.x + p * c.y;
                p = y;
            }
        }
        if (!mine) continue;
        const uint2 lo = make_uint2(pack_rounded(x[0], x[1]), pack_rounded(x[2], x[3])),
                    hi = make_uint2(pack_rounded(x[4], x[5]), pack_rounded(x[6], x[7]));
        std::uint16_t* out = place(now.t, now, a.out[0], a.out[1], a.out_stride[0], a.out_stride[1]);
        if constexpr (PAIRS) {
            *reinterpret_cast<u32x4*>(out + d0) = u32x4{lo.x, lo.y, hi.x, hi.y};
        } else {
            *reinterpret_cast<uint2*>(out + d0) = lo;
            *reinterpret_cast<uint2*>(out + d1) = hi;
        }
    }
}

// Any head size, any alignment, pairs anywhere: one wave a row, through LDS.
__global__ __launch_bounds__(kBlock) void rope_any_kernel(RopeArgs a)
{
    __shared__ float lines[kBlock / 64][kMaxHeadDim];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, heads = a.heads[0] + a.heads[1], half = a.rot >> 1;
    const std::int64_t rows = static_cast<std::int64_t>(a.tokens) * heads;
    float* const x = lines[wave];
    for (std::int64_t base = blockIdx.x * static_cast<std::int64_t>(kBlock / 64); base < rows;
         base += gridDim.x * static_cast<std::int64_t>(kBlock / 64)) {
        const std::int64_t row = base + wave;
        const bool real = row < rows;
        const std::int64_t t = real ? row / heads : 0;
        const int h = real ? static_cast<int>(row - t * heads) : 0, of = h >= a.heads[0];
        const std::int64_t at = static_cast<std::int64_t>(h - (of ? a.heads[0] : 0)) * a.dim;
        const std::uint16_t* in = a.in[of] + t * a.in_stride[of] + at;
        float sum = 0.0f;
        if (real)
            for (int d = lane; d < a.dim; d += 64) {
                const float v = h2f(in[d]);
                sum = fmaf(v, v, sum);
                x[d] = v;
            }
        sum = group_sum<64>(sum);
        if (real && a.weight[of]) {
            const float r = rsqrtf(fmaf(sum, a.inv_dim, a.eps));
            for (int d = lane; d < a.dim; d += 64) x[d] = x[d] * r * h2f(a.weight[of][d]);
        }
        __syncthreads();
        if (real) {
            std::uint16_t* out = a.out[of] + t * a.out_stride[of] + at;
            const std::int32_t p = a.rot ? a.positions[t] : 0;
            for (int d = lane; d < a.dim; d += 64) {
                float y = x[d];
                if (d < a.rot) {
                    const bool second = a.pairs ? (d & 1) : d >= half;
                    const int i = a.pairs ? d >> 1 : (second ? d - half : d);
                    const int mate = a.pairs ? d ^ 1 : (second ? d - half : d + half);
                    const float2 c = turn(p, a.freqs[i], a.rot_scale);
                    y = second ? y * c.x + x[mate] * c.y : y * c.x - x[mate] * c.y;
                }
                out[d] = f2h(opaque(y));
            }
        }
        __syncthreads();
    }
}

template <int LANES>
void launch_rows(const RopeArgs& a, bool pairs, hipStream_t s)
{
    // As many workgroups as the GPU holds at once, so that one's launch and
    // first loads are paid once; up to kMost tokens each, and their tables.
    constexpr int kMost = 4;
    const int held = 8 * conv::cu_count(), grid = std::max(std::min(a.tokens, held), (a.tokens - 1) / kMost + 1);
    const size_t lds = static_cast<size_t>((a.tokens - 1) / grid + 1) * (a.rot / 2) * sizeof(float2);
    if (pairs) rope_rows_kernel<LANES, true><<<grid, kBlock, lds, s>>>(a);
    else rope_rows_kernel<LANES, false><<<grid, kBlock, lds, s>>>(a);
}

void qk_norm_rope(const mlvc_hip_qk_norm_rope_desc* d, hipStream_t s)
{
    const char* op = "qk_norm_rope";
    require(d != nullptr, op, "no descriptor");
    require(d->tokens >= 0, op, "negative token count");
    require(launchable(d->tokens / 4 + 1, kBlock), op, "too many tokens in one call");
    require(d->head_dim >= 1 && d->head_dim <= kMaxHeadDim, op, "head_dim must be 1..512");
    require(d->q_heads >= 0 && d->k_heads >= 0 && d->q_heads <= 65536 && d->k_heads <= 65536 && d->q_heads + d->k_heads > 0,
            op, "head counts must be 0..65536 and not both 0");
    require(d->rot_dim >= 0 && d->rot_dim % 2 == 0 && d->rot_dim <= d->head_dim, op, "rot_dim must be even and 0..head_dim");
    require(d->eps >= 0.0f && std::isfinite(d->eps), op, "eps must be finite and not negative");
    require(std::isfinite(d->rot_scale), op, "rot_scale must be finite");
    const std::int64_t q_row = static_cast<std::int64_t>(d->q_heads) * d->head_dim,
                       k_row = static_cast<std::int64_t>(d->k_heads) * d->head_dim;
    require(d->q_stride >= q_row && d->q_out_stride >= q_row && d->k_stride >= k_row && d->k_out_stride >= k_row, op,
            "a stride is shorter than a row of heads");
    if (d->tokens == 0) return;
    require((!d->q_heads || (d->q && d->q_out)) && (!d->k_heads || (d->k && d->k_out)), op, "null tensor");
    require(!d->rot_dim || (d->positions && d->freqs), op, "positions and freqs are needed to rotate");
    for (const void* p : {d->q, d->k, static_cast<const void*>(d->q_out), static_cast<const void*>(d->k_out), d->q_weight, d->k_weight})
        require(aligned2(p), op, "a tensor is not aligned to its FP16 values");

    RopeArgs a{};
    a.in[0] = static_cast<const std::uint16_t*>(d->q);
    a.in[1] = static_cast<const std::uint16_t*>(d->k);
    a.out[0] = static_cast<std::uint16_t*>(d->q_out);
    a.out[1] = static_cast<std::uint16_t*>(d->k_out);
    a.weight[0] = static_cast<const std::uint16_t*>(d->q_weight);
    a.weight[1] = static_cast<const std::uint16_t*>(d->k_weight);
    a.in_stride[0] = d->q_stride, a.in_stride[1] = d->k_stride;
    a.out_stride[0] = d->q_out_stride, a.out_stride[1] = d->k_out_stride;
    a.heads[0] = d->q_heads, a.heads[1] = d->k_heads;
    a.positions = d->positions, a.freqs = d->freqs;
    a.tokens = d->tokens, a.dim = d->head_dim, a.rot = d->rot_dim;
    a.eps = d->eps, a.inv_dim = 1.0f / static_cast<float>(d->head_dim), a.rot_scale = d->rot_scale;

    bool rows = d->head_dim % 8 == 0 && d->head_dim > 32 && d->head_dim <= 256 && (d->interleaved || d->rot_dim % 8 == 0) &&
                aligned16(d->q_weight) && aligned16(d->k_weight);
    if (d->q_heads) rows = rows && vector_rows(d->q, d->q_stride) && vector_rows(d->q_out, d->q_out_stride);
    if (d->k_heads) rows = rows && vector_rows(d->k, d->k_stride) && vector_rows(d->k_out, d->k_out_stride);
    if (rows) {
        if (d->head_dim <= 64) launch_rows<8>(a, d->interleaved != 0, s);
        else if (d->head_dim <= 128) launch_rows<16>(a, d->interleaved != 0, s);
        else launch_rows<32>(a, d->interleaved != 0, s);
    } else {
        a.pairs = d->interleaved != 0;
        const std::int64_t blocks = (static_cast<std::int64_t>(d->tokens) * (d->q_heads + d->k_heads) + 3) / 4;
        rope_any_kernel<<<static_cast<unsigned>(blocks < (1 << 20) ? blocks : (1 << 20)), kBlock, 0, s>>>(a);
    }
    check(hipGetLastError(), "qk_norm_rope launch");
}

void rope_frequencies(int rot_dim, double base, int scaling, double factor, double trained, double* freqs, float* rot_scale)
{
    const char* op = "rope_frequencies";
    require(rot_dim >= 0 && rot_dim % 2 == 0 && rot_dim <= kMaxHeadDim, op, "rot_dim must be even and 0..512");
    require((freqs || rot_dim == 0) && rot_scale, op, "null result");
    require(base > 0.0 && std::isfinite(base), op, "base must be positive");
    require(factor >= 1.0 && std::isfinite(factor), op, "factor must be at least 1");
    require(scaling >= MLVC_ROPE_PLAIN && scaling <= MLVC_ROPE_BANDS, op, "unknown scaling");
    require(scaling != MLVC_ROPE_BANDS || (trained >= 1.0 && std::isfinite(trained)), op, "trained must be at least 1");
    const double pi2 = 6.283185307179586476925;
    if (scaling == MLVC_ROPE_BASE && rot_dim > 2) base *= std::pow(factor, static_cast<double>(rot_dim) / (rot_dim - 2));
    for (int i = 0; i < rot_dim / 2; ++i) {
        double f = std::pow(base, -2.0 * i / rot_dim);
        if (scaling == MLVC_ROPE_LINEAR) f /= factor;
        if (scaling == MLVC_ROPE_BANDS) {
            const double kept = std::fmin(1.0, std::fmax(0.0, (trained * f / pi2 - 1.0) / 31.0));
            f = f * kept + f / factor * (1.0 - kept);
        }
        freqs[i] = f;
    }
    *rot_scale = scaling == MLVC_ROPE_BANDS ? static_cast<float>(0.1 * std::log(factor) + 1.0) : 1.0f;
}

}  // namespace
}  // namespace mlvc_hip

using namespace mlvc_hip;

extern "C" {

int mlvc_hip_qk_norm_rope(const mlvc_hip_qk_norm_rope_desc* desc, mlvc_hip_stream s)
{
    return guard([&] { qk_norm_rope(desc, to_stream(s)); });
}

int mlvc_hip_rope_frequencies(int rot_dim, double base, int scaling, double factor, double trained, double* freqs_host,
                              float* rot_scale)
{
    return guard([&] { rope_frequencies(rot_dim, base, scaling, factor, trained, freqs_host, rot_scale); });
}

}  // extern "C"
