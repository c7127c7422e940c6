// Product of 8-bit integers with a scale for each token and output channel (atbmi_linear_int8):
//   out[i][j] = xScale[i] wScale[j] sum_k x[i][k] w[j][k] + bias[j],  the sum exact in 32-bit integers.
//
// v_mfma_i32_16x16x64_i8 with the weights as the A operand and the activations as B: lane (c = lane % 16, kg = lane /
// 16) supplies the 16 contraction values 16 kg .. 16 kg + 15 of weight row c and of token c and receives the sums of
// output channels 4 kg .. 4 kg + 3 of token c, four neighbours of one output row.
#include <algorithm>
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

// Four neighbouring sums of token m, channels n .. n + 3, scaled and rounded.
__device__ __forceinline__ void StoreOut(const Args &a, int m, int n, i32x4 sum)
{
    typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
    const float xs = a.xScale[m];
    uint16_t *dst = a.out + static_cast<int64_t>(m) * a.outStride + n;
    if (n + 4 <= a.n) {
        uint16_t v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = Rounded(a, __builtin_fmaf(static_cast<float>(sum[e]), xs * a.wScale[n + e], a.bias ? a.bias[n + e] : 0.0f));
        }
        if ((reinterpret_cast<uintptr_t>(dst) & 7) == 0) {
            *reinterpret_cast<u32x2 *>(dst) = u32x2{static_cast<uint32_t>(v[0]) | (static_cast<uint32_t>(v[1]) << 16),
                                                    static_cast<uint32_t>(v[2]) | (static_cast<uint32_t>(v[3]) << 16)};
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                dst[e] = v[e];
            }
        }
    } else {
        for (int e = 0; n + e < a.n; ++e) {
            dst[e] = Rounded(a, __builtin_fmaf(static_cast<float>(sum[e]), xs * a.wScale[n + e], a.bias ? a.bias[n + e] : 0.0f));
        }
    }
}

__device__ __forceinline__ void StorePartial(const Args &a, int32_t *dst, int n, i32x4 sum)
{
    if (n + 4 <= a.n && (a.n & 3) == 0) {
        *reinterpret_cast<i32x4 *>(dst) = sum;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (n + e < a.n) {
                dst[e] = sum[e];
            }
        }
    }
}

// ---- tiles: TN output channels x TM tokens a workgroup
//
// Both operands go through LDS in stages of 128 contraction values, two stages in turn: while one is multiplied the
// next is on its way. A row of a stage is 128 bytes, eight 16-byte chunks, chunk p of row r at place p ^ (r % 8): the 16
// rows that a fragment read touches side by side then lie in different banks. Where rows start on 16-byte boundaries
// the stage moves from memory to LDS without registers (global_load_lds_dwordx4, a wave instruction moves eight rows: its
// lane l writes place l % 8 of row l / 8, so it reads chunk (l % 8) ^ (l / 8)); rows of any other alignment, and the last
// stage where the contraction ends inside it, go through registers with what lies past the end set to zero.
// A workgroup is WN x WM waves, each with TN / WN channels x TM / WM tokens in its accumulators.
__device__ __forceinline__ void RowsToLds(const int8_t *base, uint32_t offset, uint32_t ldsAt)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(ldsAt), "v"(offset), "s"(base)
                 : "memory", "m0");
}

struct Split {
    int32_t *partial; // [splits][m][n]; null: the tile is the whole contraction and writes the output
    int32_t kPer;     // contraction values a split, a multiple of 128
};

template <int TN, int TM, int WN, int WM, bool VEC>
__global__ __launch_bounds__(WN *WM *WAVE) void LinearTileKernel(const Args a, const Split sp, int tilesN, int tilesM)
{
    constexpr int THREADS = WN * WM * WAVE;
    constexpr int NI = TN / WN / 16, MI = TM / WM / 16;
    constexpr int STAGE = (TN + TM) * 128;
    constexpr int MOVES = STAGE / (THREADS * 16); // 16-byte pieces a thread moves per stage
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int lane = threadIdx.x & (WAVE - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int c = lane & 15;
    const int kg = lane >> 4;
    const int wn = wave / WM, wm = wave % WM;

    // ---- which tile. Workgroups go to the eight XCDs in turn; each XCD gets a contiguous part of the tile list, in which
    // four rows of token tiles are walked side by side, so that what its CUs work on at a time shares rows in its L2.
    const int tiles = tilesN * tilesM;
    int t = blockIdx.x;
    {
        const int per = tiles / 8, over = tiles % 8;
        const int xcd = t % 8, at = t / 8;
        t = xcd * per + min(xcd, over) + at;
    }
    constexpr int BAND = 4;
    const int band = t / (BAND * tilesN);
    const int bandRows = min(BAND, tilesM - band * BAND);
    const int inBand = t - band * BAND * tilesN;
    const int m0 = (band * BAND + inBand % bandRows) * TM;
    const int n0 = inBand / bandRows * TN;
    const int kBegin = blockIdx.y * sp.kPer;
    const int kEnd = min(a.k, kBegin + sp.kPer);

    // ---- the pieces this thread moves: piece i covers rows 8 (wave + waves i) .. + 7 of the stage (weights, then tokens)
    const int8_t *wBase = a.w + static_cast<int64_t>(n0) * a.wStride;
    const int8_t *xBase = a.x + static_cast<int64_t>(m0) * a.xStride;
    uint32_t at[MOVES]; // offset of the piece's source from its matrix' first row of the tile, at contraction value 0
#pragma unroll
    for (int i = 0; i < MOVES; ++i) {
        const int row = 8 * (wave + WN * WM * i) + lane / 8;
        const int chunk = (lane % 8) ^ (lane / 8);
        const bool isW = 8 * (WN * WM) * i < TN; // (TN is a multiple of the rows all waves move at once)
        const int r = isW ? min(row, a.n - 1 - n0) : min(row - TN, a.m - 1 - m0);
        at[i] = static_cast<uint32_t>(r) * static_cast<uint32_t>(isW ? a.wStride : a.xStride) + 16 * chunk;
    }
    auto ldsOf = [&](int buffer, int i) { return static_cast<uint32_t>(buffer * STAGE + (wave + WN * WM * i) * 1024); };
    i32x4 held[VEC ? 1 : MOVES];
    auto loadAny = [&](int i, int k0) {
        const bool isW = 8 * (WN * WM) * i < TN;
        return Load16Any((isW ? wBase : xBase) + at[i] + k0, kEnd - k0 - 16 * ((lane % 8) ^ (lane / 8)));
    };
    auto storeAny = [&](int buffer, int i, i32x4 v) {
        *reinterpret_cast<i32x4 *>(lds + ldsOf(buffer, i) + lane * 16) = v;
    };
    auto request = [&](int buffer, int k0) {
        if constexpr (VEC) {
            if (k0 + 128 <= kEnd) {
#pragma unroll
                for (int i = 0; i < MOVES; ++i) {
                    const bool isW = 8 * (WN * WM) * i < TN;
                    RowsToLds((isW ? wBase : xBase) + k0, at[i], ldsOf(buffer, i));
                }
            } else {
#pragma unroll
                for (int i = 0; i < MOVES; ++i) {
                    storeAny(buffer, i, loadAny(i, k0));
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < MOVES; ++i) {
                held[i] = loadAny(i, k0);
            }
        }
    };
    auto arrive = [&](int buffer) {
        if constexpr (!VEC) {
#pragma unroll
            for (int i = 0; i < MOVES; ++i) {
                storeAny(buffer, i, held[i]);
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };

    i32x4 acc[NI][MI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
#pragma unroll
        for (int j = 0; j < MI; ++j) {
            acc[i][j] = i32x4{0, 0, 0, 0};
        }
    }
    request(0, kBegin);
    arrive(0);
    int buffer = 0;
    for (int k0 = kBegin; k0 < kEnd; k0 += 128, buffer ^= 1) {
        const bool more = k0 + 128 < kEnd;
        if (more) {
            request(buffer ^ 1, k0 + 128);
        }
        const unsigned char *wt = lds + buffer * STAGE + (wn * (TN / WN) + c) * 128;
        const unsigned char *xt = lds + buffer * STAGE + (TN + wm * (TM / WM) + c) * 128;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int place = ((4 * half + kg) ^ (c & 7)) * 16;
            i32x4 wf[NI], xf[MI];
#pragma unroll
            for (int j = 0; j < MI; ++j) {
                xf[j] = *reinterpret_cast<const i32x4 *>(xt + j * 2048 + place);
            }
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                wf[i] = *reinterpret_cast<const i32x4 *>(wt + i * 2048 + place);
            }
#pragma unroll
            for (int i = 0; i < NI; ++i) {
#pragma unroll
                for (int j = 0; j < MI; ++j) {
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[i], xf[j], acc[i][j], 0, 0, 0);
                }
            }
        }
        if (more) {
            arrive(buffer ^ 1);
        }
    }

    // ---- a lane holds four neighbouring channels of one token
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int n = n0 + wn * (TN / WN) + 16 * i + 4 * kg;
#pragma unroll
        for (int j = 0; j < MI; ++j) {
            const int m = m0 + wm * (TM / WM) + 16 * j + c;
            if (m < a.m) {
                if (sp.partial) {
                    StorePartial(a, sp.partial + (static_cast<int64_t>(blockIdx.y) * a.m + m) * a.n + n, n, acc[i][j]);
                } else {
                    StoreOut(a, m, n, acc[i][j]);
                }
            }
        }
    }
}

// ---- few tokens: the weights stream from memory once, straight into the matrix instructions
//
// A workgroup of eight waves takes 16 CT channels and all tokens (16 MT of them, fewer are padded by repeating the last);
// the waves take the 128-value chunks of the contraction in turn and join their integer sums in LDS. What is read of the
// activations comes from L2, MT / CT times the weights' bytes.
constexpr int SKINNY_WAVES = 8;
template <int MT, int CT, bool VEC>
__global__ __launch_bounds__(SKINNY_WAVES *WAVE) void LinearSkinnyKernel(const Args a, const Split sp)
{
    __shared__ i32x4 joined[SKINNY_WAVES][CT * MT][WAVE];
    const int lane = threadIdx.x & (WAVE - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int c = lane & 15;
    const int kg = lane >> 4;
    const int n0 = blockIdx.x * 16 * CT;
    const int m0 = blockIdx.z * 16 * MT;
    const int kBegin = blockIdx.y * sp.kPer;
    const int kEnd = min(a.k, kBegin + sp.kPer);
    const int8_t *w[CT];
    const int8_t *x[MT];
#pragma unroll
    for (int i = 0; i < CT; ++i) {
        w[i] = a.w + static_cast<int64_t>(min(n0 + 16 * i + c, a.n - 1)) * a.wStride + 16 * kg;
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        x[j] = a.x + static_cast<int64_t>(min(m0 + 16 * j + c, a.m - 1)) * a.xStride + 16 * kg;
    }
    i32x4 acc[CT][MT];
#pragma unroll
    for (int i = 0; i < CT; ++i) {
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            acc[i][j] = i32x4{0, 0, 0, 0};
        }
    }
    auto step = [&](int k, auto load) {
        i32x4 wf[2][CT], xf[2][MT];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int i = 0; i < CT; ++i) {
                wf[half][i] = load(w[i] + k + 64 * half, kEnd - k - 64 * half - 16 * kg);
            }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                xf[half][j] = load(x[j] + k + 64 * half, kEnd - k - 64 * half - 16 * kg);
            }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int i = 0; i < CT; ++i) {
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[half][i], xf[half][j], acc[i][j], 0, 0, 0);
                }
            }
        }
    };
    int k = kBegin + 128 * wave;
    for (; k + 128 <= kEnd; k += 128 * SKINNY_WAVES) {
        step(k, [](const int8_t *p, int) {
            if constexpr (VEC) {
                return *reinterpret_cast<const i32x4 *>(p);
            } else {
                i32x4 v;
                __builtin_memcpy(&v, p, 16);
                return v;
            }
        });
    }
    if (k < kEnd) {
        step(k, [](const int8_t *p, int valid) { return Load16Any(p, valid); });
    }
#pragma unroll
    for (int i = 0; i < CT; ++i) {
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            joined[wave][i * MT + j][lane] = acc[i][j];
        }
    }
    __syncthreads();
    for (int f = wave; f < CT * MT; f += SKINNY_WAVES) {
        i32x4 sum = joined[0][f][lane];
#pragma unroll
        for (int v = 1; v < SKINNY_WAVES; ++v) {
            sum += joined[v][f][lane];
        }
        const int n = n0 + 16 * (f / MT) + 4 * kg;
        const int m = m0 + 16 * (f % MT) + c;
        if (m < a.m) {
            if (sp.partial) {
                StorePartial(a, sp.partial + (static_cast<int64_t>(blockIdx.y) * a.m + m) * a.n + n, n, sum);
            } else {
                StoreOut(a, m, n, sum);
            }
        }
    }
}

// Adds the integer partial sums of a split contraction and writes the output; a thread takes four neighbours of a row.
constexpr int JOIN_THREADS = 256;
__global__ __launch_bounds__(JOIN_THREADS) void LinearJoinKernel(const Args a, const Split sp, int splits)
{
    const int64_t quads = (a.n + 3) / 4;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * JOIN_THREADS + threadIdx.x;
    if (at >= quads * a.m) {
        return;
    }
    const int m = static_cast<int>(at / quads);
    const int n = static_cast<int>(at - m * quads) * 4;
    i32x4 sum = {0, 0, 0, 0};
    for (int s = 0; s < splits; ++s) {
        const int32_t *p = sp.partial + (static_cast<int64_t>(s) * a.m + m) * a.n + n;
        if ((a.n & 3) == 0) {
            sum += *reinterpret_cast<const i32x4 *>(p);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sum[e] += n + e < a.n ? p[e] : 0;
            }
        }
    }
    StoreOut(a, m, n, sum);
}

// ---- which kernel, tile and split
enum Kind { SKINNY, TILE_128, TILE_256 };
struct Plan {
    Kind kind = SKINNY;
    int mt = 1;       // SKINNY: 16-token tiles of a workgroup
    int ct = 1;       // SKINNY: 16-channel tiles of a workgroup
    int splits = 1;
    int kPer = 0;
    uint64_t bytes = 0;
};

Plan PlanOf(int64_t m, int64_t n, int64_t k)
{
    Plan p;
    const int64_t cus = DeviceComputeUnits();
    const int64_t chunks = (k + 127) / 128;
    int64_t groups, most; // workgroups without a split, and how many splits the contraction is worth
    if (m <= 64) {
        p.kind = SKINNY;
        p.mt = m <= 16 ? 1 : (m <= 32 ? 2 : 4);
        p.ct = (n + 31) / 32 >= cus ? 2 : 1;
        groups = (n + 16 * p.ct - 1) / (16 * p.ct);
        most = chunks / (2 * SKINNY_WAVES);
    } else {
        const int64_t big = ((n + 255) / 256) * ((m + 255) / 256);
        p.kind = big >= cus ? TILE_256 : TILE_128;
        groups = p.kind == TILE_256 ? big : ((n + 127) / 128) * ((m + 127) / 128);
        most = chunks / 4;
    }
    int64_t splits = std::max<int64_t>(1, std::min<int64_t>(cus / std::max<int64_t>(groups, 1), most));
    const int64_t per = (chunks + splits - 1) / splits;
    splits = (chunks + per - 1) / per;
    p.splits = static_cast<int>(splits);
    p.kPer = static_cast<int>(per * 128);
    p.bytes = splits > 1 ? static_cast<uint64_t>(splits) * m * n * sizeof(int32_t) : 0;
    return p;
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
    *bytes = lin8::PlanOf(m, n, k).bytes;
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
    if (xRowStride > (1 << 23) || wRowStride > (1 << 23)) { // (a tile's rows are addressed with 32-bit offsets)
        return Fail(ERR_INVALID_PARAM, "linear_int8: row strides %lld, %lld are past 2^23", (long long)xRowStride,
                    (long long)wRowStride);
    }
    if (m == 0 || n == 0) {
        return OK;
    }
    if (!x || !w || !xScale || !wScale || !out) {
        return Fail(ERR_INVALID_PARAM, "linear_int8: every tensor but bias must be non-null");
    }
    const lin8::Plan plan = lin8::PlanOf(m, n, k);
    if (plan.bytes > 0 && (!workspace || workspaceBytes < plan.bytes || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0)) {
        return Fail(ERR_INVALID_PARAM, "linear_int8: workspace of %llu bytes at %p, %llu on a 16-byte boundary needed",
                    (unsigned long long)workspaceBytes, workspace, (unsigned long long)plan.bytes);
    }
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
    lin8::Split split{plan.splits > 1 ? static_cast<int32_t *>(workspace) : nullptr, plan.kPer};
    const bool vec = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15) == 0 && xRowStride % 16 == 0 &&
                     wRowStride % 16 == 0 && k % 16 == 0;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const unsigned splits = static_cast<unsigned>(plan.splits);
    int rc = OK;
    int4kv::WithFlag(vec, [&](auto v) {
        constexpr bool VEC = decltype(v)::value;
        if (plan.kind == lin8::SKINNY) {
            auto launch = [&](auto mt, auto ct) {
                const dim3 grid(static_cast<unsigned>((n + 16 * plan.ct - 1) / (16 * plan.ct)), splits,
                                static_cast<unsigned>((m + 16 * plan.mt - 1) / (16 * plan.mt)));
                lin8::LinearSkinnyKernel<decltype(mt)::value, decltype(ct)::value, VEC>
                    <<<grid, lin8::SKINNY_WAVES * WAVE, 0, s>>>(a, split);
            };
            auto withCt = [&](auto mt) {
                if (plan.ct == 2) {
                    launch(mt, std::integral_constant<int, 2>{});
                } else {
                    launch(mt, std::integral_constant<int, 1>{});
                }
            };
            if (plan.mt == 1) {
                withCt(std::integral_constant<int, 1>{});
            } else if (plan.mt == 2) {
                withCt(std::integral_constant<int, 2>{});
            } else {
                withCt(std::integral_constant<int, 4>{});
            }
            return;
        }
        auto launch = [&](auto kernel, int tile, int threads) {
            const int64_t tilesN = (n + tile - 1) / tile, tilesM = (m + tile - 1) / tile;
            const int ldsBytes = 2 * 2 * tile * 128;
            if (tilesN * tilesM > 0x7fffffffLL) {
                rc = Fail(ERR_INVALID_PARAM, "linear_int8: %lld tiles", (long long)(tilesN * tilesM));
                return;
            }
            rc = ConfigureKernelLds(reinterpret_cast<const void *>(kernel), ldsBytes);
            if (rc == OK) {
                kernel<<<dim3(static_cast<unsigned>(tilesN * tilesM), splits), threads, ldsBytes, s>>>(
                    a, split, static_cast<int>(tilesN), static_cast<int>(tilesM));
            }
        };
        if (plan.kind == lin8::TILE_256) {
            launch(lin8::LinearTileKernel<256, 256, 2, 4, VEC>, 256, 512);
        } else {
            launch(lin8::LinearTileKernel<128, 128, 2, 2, VEC>, 128, 256);
        }
    });
    if (rc != OK) {
        return rc;
    }
    ATBMI_HIP_CHECK(hipGetLastError());
    if (plan.splits > 1) {
        const int64_t threads = (n + 3) / 4 * m;
        const int64_t groups = (threads + lin8::JOIN_THREADS - 1) / lin8::JOIN_THREADS;
        lin8::LinearJoinKernel<<<static_cast<unsigned>(groups), lin8::JOIN_THREADS, 0, s>>>(a, split, plan.splits);
        ATBMI_HIP_CHECK(hipGetLastError());
    }
    return OK;
}
