// The 4-bit cache's number format and the checks its operators share.
#ifndef ATBMI_INT4_COMMON_H
#define ATBMI_INT4_COMMON_H
#include <type_traits>
#include "atbmi_common.h"

namespace atbmi {
namespace int4kv {

template <bool BF16> __device__ __forceinline__ float Widen(uint16_t bits)
{
    return BF16 ? Bf16ToFloat(bits) : HalfBitsToFloat(bits);
}
template <bool BF16> __device__ __forceinline__ uint16_t Narrow(float v)
{
    return BF16 ? FloatToBf16(v) : FloatToHalfBits(v);
}

// Two values in one word, the first in its low half (one instruction for bf16).
template <bool BF16> __device__ __forceinline__ uint32_t NarrowPair(float a, float b)
{
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    if constexpr (BF16) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
    } else {
        return static_cast<uint32_t>(FloatToHalfBits(a)) | (static_cast<uint32_t>(FloatToHalfBits(b)) << 16);
    }
}

// A row's parameter word: scale in the low half, middle in the high half.
template <bool BF16> __device__ __forceinline__ float ScaleOf(uint32_t word)
{
    return Widen<BF16>(static_cast<uint16_t>(word));
}
template <bool BF16> __device__ __forceinline__ float MidOf(uint32_t word)
{
    return Widen<BF16>(static_cast<uint16_t>(word >> 16));
}

struct RowParams {
    float inv; // 1 / scale, 0 where the scale is 0
    float mid;
    uint32_t word;
};

// scale = (hi - lo) / 15 and middle = (hi + lo) / 2, rounded to the 16-bit type: the codes are taken against the
// rounded values, so that rounding them costs at most 15 / 2 half steps of the scale's type at the row's ends and
// nothing in between. The halves keep the sums within fp32 for the largest bf16 values. A bf16 scale below the
// smallest normal number has no reciprocal in fp32 and counts as 0 (fp16 scales always have one).
template <bool BF16> __device__ __forceinline__ RowParams ParamsOf(float hi, float lo, bool bad)
{
    RowParams p;
    const uint32_t both = NarrowPair<BF16>((0.5f * hi - 0.5f * lo) * (2.0f / 15.0f), 0.5f * hi + 0.5f * lo);
    uint16_t scale = static_cast<uint16_t>(both);
    uint16_t mid = static_cast<uint16_t>(both >> 16);
    if (BF16 && (scale & 0x7f80u) == 0) {
        scale = 0;
    }
    if (bad) {
        scale = mid = BF16 ? 0x7fc0u : 0x7e00u; // NaN
    }
    const float s = Widen<BF16>(scale);
    p.inv = (bad || s == 0.0f) ? 0.0f : __builtin_amdgcn_rcpf(s); // (within an ulp: see Codes8)
    p.mid = bad ? 0.0f : Widen<BF16>(mid);
    p.word = static_cast<uint32_t>(scale) | (static_cast<uint32_t>(mid) << 16);
    return p;
}

// Codes of eight values, the first in the lowest four bits: rint((x - mid) / scale + 7.5) in 0 .. 15; 8 where the scale is
// 0 or the row is not finite (x is then ignored). All three numbers have few bits, so whole quotients, which the half makes
// ties, are common, and ties go to the even code. Sums with 96 are rounded to 2^-17 and sums with 1.5 2^23 to whole numbers,
// which the lowest bits then are: the first makes a tie of every quotient that is one (the product with a reciprocal that
// is a little off is within 2^-19 of it), at the price that places within 2^-18 of the middle between two codes count as
// ties as well; the second rounds to the even code.
__device__ __forceinline__ uint32_t Codes8(const float (&x)[8], float mid, float inv)
{
    constexpr float SNAP = 96.0f, MAGIC = 12582912.0f;
    uint32_t codes = 0, extra = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float place = __builtin_fmaf(x[i] - mid, inv, SNAP + 7.5f);
        const float q = __builtin_amdgcn_fmed3f(place, SNAP, SNAP + 15.0f) + (MAGIC - SNAP);
        codes += __float_as_uint(q) << (4 * i);
        extra += 0x4b400000u << (4 * i); // the bits of MAGIC
    }
    return inv == 0.0f ? 0x88888888u : codes - extra;
}

inline int CheckCache(const char *who, int32_t dtype, int64_t numKvHeads, int64_t headDim, int64_t blockSize,
                      int64_t numBlocks)
{
    if (dtype != ATBMI_F16 && dtype != ATBMI_BF16) {
        return Fail(ERR_INVALID_PARAM, "%s: the model's type is fp16 or bf16, got %d", who, dtype);
    }
    if (headDim != 64 && headDim != 128 && headDim != 256) {
        return Fail(ERR_INVALID_PARAM, "%s: head size %lld (64, 128 and 256 are built)", who, (long long)headDim);
    }
    if (numKvHeads <= 0 || numKvHeads > (1 << 20)) {
        return Fail(ERR_INVALID_PARAM, "%s: %lld KV heads", who, (long long)numKvHeads);
    }
    if (blockSize <= 0 || blockSize % 16 != 0 || blockSize > 1024) {
        return Fail(ERR_INVALID_PARAM, "%s: blocks of %lld tokens (a multiple of 16 up to 1024 is needed)", who,
                    (long long)blockSize);
    }
    if (numBlocks <= 0 || numBlocks > 0x7fffffffLL / blockSize) {
        return Fail(ERR_INVALID_PARAM, "%s: %lld blocks of %lld tokens (slots are 32-bit numbers)", who,
                    (long long)numBlocks, (long long)blockSize);
    }
    return OK;
}

// A launch has fewer than 2^32 threads along each dimension of its grid.
inline bool FitsLaunch(int64_t workgroups, int64_t threads)
{
    return workgroups <= 0xffffffffLL / threads;
}

// Compile-time values from run-time ones.
template <typename F> void WithFlag(bool flag, F &&next)
{
    if (flag) {
        next(std::true_type{});
    } else {
        next(std::false_type{});
    }
}
template <typename F> void WithHeadDim(int64_t headDim, F &&next)
{
    if (headDim == 64) {
        next(std::integral_constant<int, 64>{});
    } else if (headDim == 128) {
        next(std::integral_constant<int, 128>{});
    } else {
        next(std::integral_constant<int, 256>{});
    }
}

} // namespace int4kv
} // namespace atbmi
#endif
