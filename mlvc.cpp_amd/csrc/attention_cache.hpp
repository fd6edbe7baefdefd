// Shared parts of the kernels that read the paged cache on the matrix cores:
// cached bytes as halves, and contexts dealt evenly over workgroups.
#pragma once

#include "attention.hpp"

namespace mlvc_hip {

constexpr int kStep = 32;  // tokens of a step

// Steps of so many tokens; a context may have 2^31 - 1.
__device__ __forceinline__ int steps_for(int tokens) { return tokens / kStep + (tokens % kStep != 0); }

__device__ __forceinline__ int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }

// The shares of a key head's steps: `shares` large ones, all on the GPU at
// once, cover five sixths of them, and as many small ones cover the rest,
// for the workgroups that are done first (their rates differ by a tenth
// either way). Few steps are not cut below kLeast, in one row of shares; nor
// are any without `spare`.
struct Shares {
    static constexpr int kLeast = 8;
    int total, large, count;  // steps; of them in the first `count` shares; the others are `count` more, or none
    __device__ Shares(int shares, int total_, bool spare = true) : total(total_)
    {
        const bool few = !spare || total < 6 * kLeast * shares;
        count = few ? max(1, min(shares, total / kLeast)) : shares;
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

}  // namespace mlvc_hip
