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
using int4kv::NarrowPair;
using int4kv::Widen;
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

constexpr int THREADS = 256;
constexpr int WAVES = THREADS / WAVE;
constexpr int MOST_THREADS = 1024;

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

constexpr float LEAST = 0x1p-118f; // (127 / LEAST is finite)

// Power of two that a row is multiplied by before its squares and products are taken: 1 but for rows of finite values that
// leave fp32's range on the way: bf16 values past 1e19, whose squares are infinite, or below 2^-50, whose squares lose bits
// or vanish, and products with gamma past either end. Such a row is taken a second time, its largest value brought between
// a half and one. With a large eps it is brought up only as far as eps pre^2 stays finite: its squares are then lost in
// eps, where they would be lost in any case.
__device__ __forceinline__ float PreOf(float sumSq, float maxSg, float maxS, float eps)
{
    if (!__builtin_isfinite(maxS) || maxS == 0.0f || sumSq != sumSq) {
        return 1.0f;
    }
    if (__builtin_isfinite(sumSq) && __builtin_isfinite(maxSg) && maxS >= 0x1p-50f && maxSg >= LEAST && eps < 0x1p126f) {
        return 1.0f;
    }
    int power = min(-__builtin_amdgcn_frexp_expf(maxS), 126);
    if (eps > 0.0f) {
        power = min(power, (126 - __builtin_amdgcn_frexp_expf(eps)) >> 1);
    }
    return __builtin_ldexpf(1.0f, power);
}

// From the sum of squares and max|s gamma| of a row multiplied by `pre`.
__device__ __forceinline__ RowFactors FactorsOf(float sumSq, float maxSg, int dim, float eps, float pre)
{
    RowFactors f;
    f.pre = pre;
    f.bad = !__builtin_isfinite(sumSq) || !__builtin_isfinite(maxSg);
    const float rstd = rsqrtf(sumSq / static_cast<float>(dim) + eps * pre * pre);
    const bool none = !(maxSg >= LEAST);
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

// Rows in 16-byte pieces, NV of them to a thread: a row is read once and stays in registers (rounded to the model's type,
// as it is stored) between the reduction and the codes. gamma stays as well, but for the longest rows, which read it twice.
template <bool BF16, bool RES, int NV> __global__ __launch_bounds__(MOST_THREADS) void NormRowKernel(const Args a)
{
    __shared__ float lds[MOST_THREADS / WAVE][3];
    const int64_t row = blockIdx.x;
    const int pieces = a.dim / 8;
    const int T = blockDim.x;
    const u32x4 *x = reinterpret_cast<const u32x4 *>(a.x + row * a.xStride);
    const u32x4 *r = reinterpret_cast<const u32x4 *>(a.residual + row * a.rStride);
    const u32x4 *gamma = reinterpret_cast<const u32x4 *>(a.gamma);
    constexpr bool HOLD = NV < 8;
    u32x4 s[NV], held[HOLD ? NV : 1];
    auto gammaOf = [&](int v) __attribute__((always_inline)) {
        return HOLD ? held[HOLD ? v : 0] : gamma[min(static_cast<int>(threadIdx.x) + v * T, pieces - 1)];
    };
    u32x4 add[RES ? NV : 1];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int at = min(static_cast<int>(threadIdx.x) + v * T, pieces - 1); // (a row's last piece again: not counted)
        s[v] = __builtin_nontemporal_load(x + at);
        if constexpr (RES) {
            add[v] = __builtin_nontemporal_load(r + at);
        }
    }
    if constexpr (HOLD) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            held[v] = gamma[min(static_cast<int>(threadIdx.x) + v * T, pieces - 1)];
        }
    }
    u32x4 *ro = reinterpret_cast<u32x4 *>(a.residualOut + row * a.dim);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        if constexpr (RES) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[v][i] = NarrowPair<BF16>(
                    Widen<BF16>(static_cast<uint16_t>(s[v][i])) + Widen<BF16>(static_cast<uint16_t>(add[v][i])),
                    Widen<BF16>(static_cast<uint16_t>(s[v][i] >> 16)) + Widen<BF16>(static_cast<uint16_t>(add[v][i] >> 16)));
            }
        }
        const int at = static_cast<int>(threadIdx.x) + v * T;
        if (at < pieces && a.residualOut) {
            ro[at] = s[v];
        }
    }
    auto pass = [&](float pre, float &sumSq, float &maxSg, float &maxS) __attribute__((always_inline)) {
        sumSq = maxSg = maxS = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (static_cast<int>(threadIdx.x) + v * T < pieces) {
                const u32x4 gm = gammaOf(v);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float one = Widen<BF16>(static_cast<uint16_t>(s[v][i / 2] >> (i % 2 * 16))) * pre;
                    const float sg = fabsf(one * Widen<BF16>(static_cast<uint16_t>(gm[i / 2] >> (i % 2 * 16))));
                    sumSq += one * one;
                    maxSg = fmaxf(maxSg, sg == sg ? sg : INFINITY); // (a maximum alone would pass over a NaN in gamma)
                    maxS = fmaxf(maxS, fabsf(one));
                }
            }
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
    u32x2 *out = reinterpret_cast<u32x2 *>(a.out + row * a.dim);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const u32x4 gm = gammaOf(v);
        u32x2 codes = {0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float sg = Widen<BF16>(static_cast<uint16_t>(s[v][i / 2] >> (i % 2 * 16))) * f.pre *
                             Widen<BF16>(static_cast<uint16_t>(gm[i / 2] >> (i % 2 * 16)));
            codes[i / 4] |= (static_cast<uint32_t>(f.bad ? 0 : Code(sg, f.step)) & 255u) << (i % 4 * 8);
        }
        const int at = static_cast<int>(threadIdx.x) + v * T;
        if (at < pieces) {
            out[at] = codes;
        }
    }
    if (threadIdx.x == 0) {
        a.scale[row] = f.scale;
    }
}

bool Aligned(const void *p, unsigned bytes)
{
    return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
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
    const bool pieces = dim % 8 == 0 && xRowStride % 8 == 0 && a.rStride % 8 == 0 && normq::Aligned(x, 16) &&
                        normq::Aligned(residual, 16) && normq::Aligned(gamma, 16) && normq::Aligned(residualOut, 16) &&
                        normq::Aligned(out, 8);
    // Threads a row. Few rows leave CUs idle, so each gets a thread for every piece. Many rows fill the chip with small
    // workgroups of up to four pieces a thread (8191 x 8192 with a residual: 72 us, 6.5 TB/s), larger ones only where a row
    // has more.
    int64_t most = rows < 2LL * DeviceComputeUnits() ? normq::MOST_THREADS : normq::THREADS;
    while (most < normq::MOST_THREADS && dim / 8 > most * 4) {
        most *= 2;
    }
    int nv = 1;
    while (nv < 8 && dim / 8 > most * nv) {
        nv *= 2;
    }
    const int64_t threads = ((dim / 8 + nv - 1) / nv + WAVE - 1) / WAVE * WAVE;
    // (a workgroup for each row: more rows than one launch has room for go in several)
    constexpr int64_t LAUNCH_ROWS = 1 << 21;
    static_assert(LAUNCH_ROWS * normq::MOST_THREADS < (1LL << 32), "threads of a launch");
    for (int64_t left = rows; left > 0; left -= LAUNCH_ROWS) {
        const dim3 grid(static_cast<unsigned>(left < LAUNCH_ROWS ? left : LAUNCH_ROWS)), block(static_cast<unsigned>(threads));
        int4kv::WithFlag(dtype == ATBMI_BF16, [&](auto bf16) {
            constexpr bool BF16 = decltype(bf16)::value;
            if (!pieces) {
                normq::NormPlainKernel<BF16><<<grid, normq::THREADS, 0, s>>>(a);
                return;
            }
            int4kv::WithFlag(residual != nullptr, [&](auto res) {
                constexpr bool RES = decltype(res)::value;
                switch (nv) {
                case 1: normq::NormRowKernel<BF16, RES, 1><<<grid, block, 0, s>>>(a); break;
                case 2: normq::NormRowKernel<BF16, RES, 2><<<grid, block, 0, s>>>(a); break;
                case 4: normq::NormRowKernel<BF16, RES, 4><<<grid, block, 0, s>>>(a); break;
                default: normq::NormRowKernel<BF16, RES, 8><<<grid, block, 0, s>>>(a); break;
                }
            });
        });
        ATBMI_HIP_CHECK(hipGetLastError());
        a.x += LAUNCH_ROWS * a.xStride;
        a.residual = a.residual ? a.residual + LAUNCH_ROWS * a.rStride : nullptr;
        a.residualOut = a.residualOut ? a.residualOut + LAUNCH_ROWS * dim : nullptr;
        a.out += LAUNCH_ROWS * dim;
        a.scale += LAUNCH_ROWS;
    }
    return OK;
}
