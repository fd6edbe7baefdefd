// Shared parts of the attention kernels: argument checks, wave reductions and
// the rows of the paged cache.
#pragma once

#include "common.hpp"
#include "mlvc_hip_device.h"

#include <climits>
#include <cmath>
#include <cstdint>
#include <string>

namespace mlvc_hip {

inline void require(bool ok, const char* op, const char* what)
{
    if (!ok) throw std::runtime_error(std::string(op) + ": " + what);
}

template <int BYTES>
bool aligned_to(const void* p) { return (reinterpret_cast<std::uintptr_t>(p) & (BYTES - 1u)) == 0; }
inline bool aligned16(const void* p) { return aligned_to<16>(p); }
inline bool aligned2(const void* p) { return aligned_to<2>(p); }

// 16-byte aligned rows of halves.
inline bool vector_rows(const void* p, std::int64_t stride) { return aligned16(p) && stride % 8 == 0; }

constexpr int kMaxHeadDim = 512;

// A launch counts its threads in 32 bits along an axis.
inline bool launchable(std::int64_t workgroups, int threads) { return workgroups <= UINT_MAX / threads; }

// Checks a cache descriptor; `op` names the caller in the message.
void check_cache(const mlvc_hip_kv_cache* cache, const char* op);

// Opaque to the optimiser: keeps the narrowing of an FP32 result a rounding
// of its own.
__device__ __forceinline__ float opaque(float x)
{
    asm("" : "+v"(x));
    return x;
}

__device__ __forceinline__ std::uint32_t pack_rounded(float a, float b) { return pack_f16(opaque(a), opaque(b)); }

// Value of the lane O away, where the values already agree between lanes 2 O
// away (or O is half the group). Within 16 lanes by the adders' own lane
// exchange, without a trip through LDS.
template <int O, int LANES, typename T>
__device__ __forceinline__ T across(T x)
{
    constexpr int kSwap1 = 0xB1, kSwap2 = 0x4E, kRotate = 0x120, kMirror8 = 0x141;
    constexpr int kHow = O == 1 ? kSwap1 : O == 2 ? kSwap2 : LANES == 8 ? kMirror8 : kRotate + O;
    if constexpr (O >= 16) return __shfl_xor(x, O);
    else return __builtin_bit_cast(T, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), kHow, 0xf, 0xf, true));
}

// Reductions over groups of LANES adjacent lanes; every lane gets the result.
template <int LANES, int O = LANES / 2>
__device__ __forceinline__ float group_sum(float x)
{
    x += across<O, LANES>(x);
    if constexpr (O > 1) return group_sum<LANES, O / 2>(x);
    else return x;
}

template <int LANES, int O = LANES / 2>
__device__ __forceinline__ float group_max(float x)
{
    x = fmaxf(x, across<O, LANES>(x));
    if constexpr (O > 1) return group_max<LANES, O / 2>(x);
    else return x;
}

template <int LANES, int O = LANES / 2>
__device__ __forceinline__ std::uint32_t group_max(std::uint32_t x)
{
    x = max(x, across<O, LANES>(x));
    if constexpr (O > 1) return group_max<LANES, O / 2>(x);
    else return x;
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

// Weights go to the matrix cores in FP16, as 2^(score - m) with a base m of the
// running softmax that lies kLift powers of two below a score: FP16's numbers
// end at 2^-24, so with the largest weight at 2^12 or more one of 2^-26 of it
// keeps all its bits, and what is lost below is 2^-37 of it. The base follows
// once a score is kMost above it; FP16 ends at 2^16.
constexpr float kLift = 12.0f, kMost = 15.0f;

// The base for a largest score. From kCoarse on FP32's scores are too coarse to
// lie 12 below one another, and the score itself is the base.
constexpr float kCoarse = 0x1p22f;
__device__ __forceinline__ float lifted(float top) { return fabsf(top) < kCoarse ? top - kLift : top; }

__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) < INFINITY; }

// The infinities and NaN among the values of a sum with weights above 0. In
// numbers of few bits a weight may be 0, and its product with one of them NaN:
// every sum that holds one ends as infinite or NaN and is then decided by these.
struct OddValues {
    unsigned seen = 0;
    // 1: +inf, 2: -inf, 4: NaN, 0: neither.
    __device__ static unsigned of(std::uint16_t v) { return (v & 0x7c00u) != 0x7c00u ? 0u : (v & 0x3ffu) ? 4u : (v & 0x8000u) ? 2u : 1u; }
    __device__ void add(std::uint16_t v) { seen |= of(v); }
    __device__ float sum(float otherwise) const
    {
        return seen == 0 ? otherwise : seen == 1 ? INFINITY : seen == 2 ? -INFINITY : __builtin_nanf("");
    }
};

// Sum over this lane and those before it: rows of 16 lanes by shifts, then
// each row's total to the rows after it.
__device__ __forceinline__ int wave_scan(int x)
{
    constexpr int kShift = 0x110, kLast15 = 0x142, kLast31 = 0x143;
    x += __builtin_amdgcn_update_dpp(0, x, kShift + 1, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, kShift + 2, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, kShift + 4, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, kShift + 8, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, kLast15, 0xa, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, kLast31, 0xc, 0xf, false);
    return x;
}

// 8-bit values of a cached row, widened. INT8 is two's complement.
__device__ __forceinline__ float from_byte(int kind, std::uint8_t b)
{
    if (kind == MLVC_KV_INT8) return static_cast<float>(static_cast<std::int8_t>(b));
    return __builtin_amdgcn_cvt_f32_fp8(b, 0);
}

}  // namespace mlvc_hip
