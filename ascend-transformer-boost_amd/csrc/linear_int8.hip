// Product of 8-bit integers with a scale for each token and output channel (atbmi_linear_int8):
//   out[i][j] = xScale[i] wScale[j] sum_k x[i][k] w[j][k] + bias[j],  the sum exact in 32-bit integers.
//
// v_mfma_i32_16x16x64_i8 with the weights as the A operand and the activations as B: lane (c = lane % 16, kg = lane /
// 16) supplies the 16 contraction values 16 kg .. 16 kg + 15 of weight row c and of token c and receives the sums of
// output channels 4 kg .. 4 kg + 3 of token c, four neighbours of one output row.
#include "pa_internal.h"
#include "int4_common.h"

namespace atbmi {
namespace lin8 {

typedef int i32x4 __attribute__((ext_vector_type(4)));

struct Args {
    const int8_t *x;
    const int8_t *w;
    const float *xScale;
    const float *wScale;
    const float *bias; // null: none
    uint16_t *out;
    int64_t xStride;
    int64_t wStride;
    int64_t outStride;
    int32_t m, n, k;
    int32_t bf16;
};

__device__ __forceinline__ uint16_t Rounded(const Args &a, float v)
{
    return a.bf16 ? FloatToBf16(v) : FloatToHalfBits(v);
}

// Sixteen values from an address of any alignment; those at or past `valid` count as zero.
__device__ __forceinline__ i32x4 Load16Any(const int8_t *p, int valid)
{
    i32x4 v = {0, 0, 0, 0};
    if (valid >= 16) {
        __builtin_memcpy(&v, p, 16);
    } else if (valid > 0) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int byte = i < valid ? static_cast<uint8_t>(p[i]) : 0;
            v[i / 4] |= byte << (8 * (i % 4));
        }
    }
    return v;
}

// Any size, stride and alignment: a wave computes 16 output channels x 64 tokens straight from global memory.
constexpr int PLAIN_THREADS = 256;
__global__ __launch_bounds__(PLAIN_THREADS) void LinearPlainKernel(const Args a)
{
    const int lane = threadIdx.x & (WAVE - 1);
    const int wave = threadIdx.x / WAVE;
    const int c = lane & 15;
    const int kg = lane >> 4;
    const int n0 = (blockIdx.x * (PLAIN_THREADS / WAVE) + wave) * 16;
    const int m0 = blockIdx.y * 64;
    if (n0 >= a.n) {
        return;
    }
    const int8_t *w = a.w + static_cast<int64_t>(min(n0 + c, a.n - 1)) * a.wStride;
    const int8_t *x[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        x[t] = a.x + static_cast<int64_t>(min(m0 + 16 * t + c, a.m - 1)) * a.xStride;
    }
    i32x4 acc[4] = {};
    for (int k0 = 16 * kg; k0 - 16 * kg < a.k; k0 += 64) {
        const i32x4 wv = Load16Any(w + k0, a.k - k0);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv, Load16Any(x[t] + k0, a.k - k0), acc[t], 0, 0, 0);
        }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int i = m0 + 16 * t + c;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int j = n0 + 4 * kg + e;
            if (i < a.m && j < a.n) {
                const float v = static_cast<float>(acc[t][e]) * (a.xScale[i] * a.wScale[j]) + (a.bias ? a.bias[j] : 0.0f);
                a.out[static_cast<int64_t>(i) * a.outStride + j] = Rounded(a, v);
            }
        }
    }
}

int Check(int64_t m, int64_t n, int64_t k)
{
    if (m < 0 || n < 0 || k <= 0 || k > 131071 || m > 0x7fffff00LL || n > 0x7fffff00LL) {
        return Fail(ERR_INVALID_PARAM, "linear_int8: [%lld, %lld] by [%lld, %lld]: the contraction must be 1 .. 131071",
                    (long long)m, (long long)k, (long long)n, (long long)k);
    }
    return OK;
}

} // namespace lin8
} // namespace atbmi

using namespace atbmi;

extern "C" int atbmi_linear_int8_workspace_size(int64_t m, int64_t n, int64_t k, uint64_t *bytes)
{
    if (!bytes) {
        return Fail(ERR_INVALID_PARAM, "linear_int8_workspace_size: null result pointer");
    }
    if (int rc = lin8::Check(m, n, k)) {
        return rc;
    }
    *bytes = 0;
    return OK;
}

extern "C" int atbmi_linear_int8(const int8_t *x, const int8_t *w, const float *xScale, const float *wScale,
                                 const float *bias, void *out, int64_t m, int64_t n, int64_t k, int64_t xRowStride,
                                 int64_t wRowStride, int64_t outRowStride, int32_t outDtype, void *workspace,
                                 uint64_t workspaceBytes, void *stream)
{
    if (int rc = lin8::Check(m, n, k)) {
        return rc;
    }
    if (outDtype != ATBMI_F16 && outDtype != ATBMI_BF16) {
        return Fail(ERR_INVALID_PARAM, "linear_int8: the output is fp16 or bf16, got %d", outDtype);
    }
    if (xRowStride < k || wRowStride < k || outRowStride < n) {
        return Fail(ERR_INVALID_PARAM, "linear_int8: row strides %lld, %lld, %lld of rows of %lld, %lld, %lld",
                    (long long)xRowStride, (long long)wRowStride, (long long)outRowStride, (long long)k, (long long)k,
                    (long long)n);
    }
    if (m == 0 || n == 0) {
        return OK;
    }
    if (!x || !w || !xScale || !wScale || !out) {
        return Fail(ERR_INVALID_PARAM, "linear_int8: every tensor but bias must be non-null");
    }
    (void)workspace;
    (void)workspaceBytes;
    lin8::Args a{};
    a.x = x;
    a.w = w;
    a.xScale = xScale;
    a.wScale = wScale;
    a.bias = bias;
    a.out = static_cast<uint16_t *>(out);
    a.xStride = xRowStride;
    a.wStride = wRowStride;
    a.outStride = outRowStride;
    a.m = static_cast<int32_t>(m);
    a.n = static_cast<int32_t>(n);
    a.k = static_cast<int32_t>(k);
    a.bf16 = outDtype == ATBMI_BF16;
    if ((m + 63) / 64 > 65535) {
        return Fail(ERR_INVALID_PARAM, "linear_int8: %lld tokens are more than one launch takes", (long long)m);
    }
    const dim3 grid(static_cast<unsigned>((n + 63) / 64), static_cast<unsigned>((m + 63) / 64));
    lin8::LinearPlainKernel<<<grid, lin8::PLAIN_THREADS, 0, static_cast<hipStream_t>(stream)>>>(a);
    ATBMI_HIP_CHECK(hipGetLastError());
    return OK;
}
