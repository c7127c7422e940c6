// RMS norm with the residual's addition and an 8-bit output with a scale for each row (atbmi_rms_norm_quant).
//
//   s = round(x + residual);  y = s gamma rsqrt(mean s^2 + eps);  scale = max|y| / 127;  q = rint(y / scale)
//
// The factor rsqrt(..) is one number a row and drops out of y / scale = 127 s gamma / max|s gamma|, so one reduction
// over the row, of s^2 (sum) and |s gamma| (maximum) together, gives everything: a row is read once, held in registers
// and written once. HBM bounds long calls (7 bytes a value with a residual), latency short ones.
#include "pa_internal.h"
#include "int4_common.h"

namespace atbmi {
namespace normq {

using int4kv::Narrow;
using int4kv::Widen;
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

constexpr int THREADS = 256;
constexpr int WAVES = THREADS / WAVE;

struct Args {
    const uint16_t *x;
    const uint16_t *residual; // null: none
    const uint16_t *gamma;
    int8_t *out;
    float *scale;
    uint16_t *residualOut; // null: not stored
    int64_t xStride;
    int64_t rStride;
    int32_t dim;
    float eps;
};

// Sum of `a` and maximum of `b` and of `c` over the workgroup, in a fixed order.
__device__ __forceinline__ void Reduce(float &a, float &b, float &c, float (*lds)[3])
{
#pragma unroll
    for (int step = 1; step < WAVE; step *= 2) {
        a += __shfl_xor(a, step);
        b = fmaxf(b, __shfl_xor(b, step));
        c = fmaxf(c, __shfl_xor(c, step));
    }
    const int wave = threadIdx.x / WAVE;
    __syncthreads(); // (what an earlier reduction left has been read)
    if ((threadIdx.x & (WAVE - 1)) == 0) {
        lds[wave][0] = a;
        lds[wave][1] = b;
        lds[wave][2] = c;
    }
    __syncthreads();
    a = b = c = 0.0f;
    for (int w = 0; w < static_cast<int>(blockDim.x) / WAVE; ++w) {
        a += lds[w][0];
        b = fmaxf(b, lds[w][1]);
        c = fmaxf(c, lds[w][2]);
    }
}

struct RowFactors {
    float pre;   // multiplies s before gamma (PreOf)
    float step;  // 127 / max|s gamma pre|
    float scale; // what goes to Args::scale
    bool bad;
};

// Power of two that a row is multiplied by before its squares and products are taken: 1 but for rows of finite values
// that leave fp32's range on the way (bf16 values past 1e19, whose squares are infinite, or below 2^-50, whose squares
// lose bits or vanish). Such a row is taken a second time. (The factor for small rows keeps eps pre^2 finite.)
__device__ __forceinline__ float PreOf(float sumSq, float maxSg, float maxS, float eps)
{
    if (!__builtin_isfinite(maxS) || maxS == 0.0f || sumSq != sumSq) {
        return 1.0f;
    }
    if (__builtin_isinf(sumSq) || __builtin_isinf(maxSg)) {
        return __builtin_ldexpf(1.0f, -min(__builtin_amdgcn_frexp_expf(maxS), 126));
    }
    if (maxS < 0x1p-50f) {
        return eps > 0.0f ? 0x1p63f : 0x1p126f;
    }
    return 1.0f;
}

// From the sum of squares and max|s gamma| of a row multiplied by `pre`.
__device__ __forceinline__ RowFactors FactorsOf(float sumSq, float maxSg, int dim, float eps, float pre)
{
    RowFactors f;
    f.pre = pre;
    f.bad = !__builtin_isfinite(sumSq) || !__builtin_isfinite(maxSg);
    const float rstd = rsqrtf(sumSq / static_cast<float>(dim) + eps * pre * pre);
    const bool none = !(maxSg >= 0x1p-118f); // (127 / maxSg stays finite)
    f.scale = f.bad ? __builtin_nanf("") : (none ? 0.0f : maxSg * rstd * (1.0f / 127.0f));
    f.step = (f.bad || none) ? 0.0f : 127.0f / maxSg;
    return f;
}

__device__ __forceinline__ int Code(float sg, float step)
{
    const float q = rintf(sg * step);
    return static_cast<int>(fminf(fmaxf(q, -127.0f), 127.0f));
}

// Any dimension, stride and alignment: three passes over the row, element by element (the row stays in L2).
template <bool BF16> __global__ __launch_bounds__(THREADS) void NormPlainKernel(const Args a)
{
    __shared__ float lds[WAVES][3];
    const int64_t row = blockIdx.x;
    const uint16_t *x = a.x + row * a.xStride;
    const uint16_t *r = a.residual ? a.residual + row * a.rStride : nullptr;
    uint16_t *ro = a.residualOut ? a.residualOut + row * a.dim : nullptr;
    // (residualOut may be the residual itself: it is written in the last pass only, by the thread that reads the value)
    auto value = [&](int i) {
        const float v = Widen<BF16>(x[i]);
        return r ? Widen<BF16>(Narrow<BF16>(v + Widen<BF16>(r[i]))) : v;
    };
    auto pass = [&](float pre, float &sumSq, float &maxSg, float &maxS) {
        sumSq = maxSg = maxS = 0.0f;
        for (int i = threadIdx.x; i < a.dim; i += THREADS) {
            const float s = value(i) * pre;
            sumSq += s * s;
            const float sg = fabsf(s * Widen<BF16>(a.gamma[i]));
            maxSg = fmaxf(maxSg, sg == sg ? sg : INFINITY); // (a maximum alone would pass over a NaN in gamma)
            maxS = fmaxf(maxS, fabsf(s));
        }
        Reduce(sumSq, maxSg, maxS, lds);
    };
    float sumSq, maxSg, maxS;
    pass(1.0f, sumSq, maxSg, maxS);
    const float pre = PreOf(sumSq, maxSg, maxS, a.eps);
    if (pre != 1.0f) {
        pass(pre, sumSq, maxSg, maxS);
    }
    const RowFactors f = FactorsOf(sumSq, maxSg, a.dim, a.eps, pre);
    for (int i = threadIdx.x; i < a.dim; i += THREADS) {
        const float s = value(i);
        a.out[row * a.dim + i] = f.bad ? 0 : static_cast<int8_t>(Code(s * f.pre * Widen<BF16>(a.gamma[i]), f.step));
        if (ro) {
            ro[i] = Narrow<BF16>(s);
        }
    }
    if (threadIdx.x == 0) {
        a.scale[row] = f.scale;
    }
}

} // namespace normq
} // namespace atbmi

using namespace atbmi;

extern "C" int atbmi_rms_norm_quant(const void *x, const void *residual, const void *gamma, int8_t *out, float *scale,
                                    void *residualOut, int64_t rows, int64_t dim, int64_t xRowStride,
                                    int64_t residualRowStride, int32_t dtype, float epsilon, void *stream)
{
    if (dtype != ATBMI_F16 && dtype != ATBMI_BF16) {
        return Fail(ERR_INVALID_PARAM, "rms_norm_quant: the input is fp16 or bf16, got %d", dtype);
    }
    if (rows < 0 || rows > 0x7fffffffLL || dim <= 0 || dim > 65536 || xRowStride < dim ||
        (residual && residualRowStride < dim) || !(epsilon >= 0.0f) || !__builtin_isfinite(epsilon)) {
        return Fail(ERR_INVALID_PARAM, "rms_norm_quant: %lld rows of %lld values (strides %lld, %lld), epsilon %g",
                    (long long)rows, (long long)dim, (long long)xRowStride, (long long)residualRowStride, epsilon);
    }
    if (rows == 0) {
        return OK;
    }
    if (!x || !gamma || !out || !scale) {
        return Fail(ERR_INVALID_PARAM, "rms_norm_quant: x, gamma, out and scale must be non-null");
    }
    if ((residualOut == x && xRowStride != dim) || (residual && residualOut == residual && residualRowStride != dim)) {
        return Fail(ERR_INVALID_PARAM, "rms_norm_quant: residualOut may be an input only where that has no gaps");
    }
    normq::Args a{};
    a.x = static_cast<const uint16_t *>(x);
    a.residual = static_cast<const uint16_t *>(residual);
    a.gamma = static_cast<const uint16_t *>(gamma);
    a.out = out;
    a.scale = scale;
    a.residualOut = static_cast<uint16_t *>(residualOut);
    a.xStride = xRowStride;
    a.rStride = residual ? residualRowStride : 0;
    a.dim = static_cast<int32_t>(dim);
    a.eps = epsilon;
    hipStream_t s = static_cast<hipStream_t>(stream);
    int4kv::WithFlag(dtype == ATBMI_BF16, [&](auto bf16) {
        normq::NormPlainKernel<decltype(bf16)::value><<<static_cast<unsigned>(rows), normq::THREADS, 0, s>>>(a);
    });
    ATBMI_HIP_CHECK(hipGetLastError());
    return OK;
}
