// The 4-bit KV cache: the write that quantises key and value rows into it and the gather that gives them back
// (atbmi_reshape_and_cache_int4, atbmi_paged_cache_load_int4). The layout is described in atbmi_kernels.h; a row of
// D channels is D codes of 4 bits, a scale and a middle value.
//
// Both move a few bytes per value and compute next to nothing: HBM bounds them on long calls and the launch on short
// ones. In both kernels a lane owns eight channels of a row (16 bytes in the model's type, 4 bytes of codes), D / 8
// lanes a row, so that rows of the model's type move in 16-byte pieces.
#include <algorithm>
#include "pa_internal.h"
#include "int4_common.h"

namespace atbmi {
namespace int4kv {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x2 __attribute__((ext_vector_type(2)));

constexpr int MOVE_THREADS = 256;

struct WriteArgs {
    const uint16_t *key;
    const uint16_t *value;
    uint8_t *keyCache;
    uint8_t *valueCache;
    uint32_t *keyParams; // (scale, middle) as one word
    uint32_t *valueParams;
    const int32_t *slots;
    int64_t numRows; // tokens x heads
    int64_t numSlots;
    int64_t keyTokenStride;
    int64_t valueTokenStride;
    int32_t G;
    int32_t blockSize;
};

template <int CTRL> __device__ __forceinline__ s16x2 Moved(s16x2 x)
{
    return __builtin_bit_cast(s16x2, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}

// 16-bit floats as integers of the same order and back (two at a time): the bits below the sign are turned over where it is
// set. NaN with a sign lie below -infinity, those without one above infinity.
__device__ __forceinline__ s16x2 Ordered(s16x2 x)
{
    return x ^ ((x >> 15) & 0x7fff);
}
__device__ __forceinline__ s16x2 Ordered(uint32_t word)
{
    return Ordered(__builtin_bit_cast(s16x2, word));
}

// Largest and smallest value of a row that LPR lanes hold, eight values each (w: as they are read), as 16-bit floats in the
// low and high half. Both are found on integers, two values to an instruction, the minimum as the maximum of the
// complements in the other half of a word: the kernel for many tokens was bound by its arithmetic, 208 instructions for
// eight values, half of them for this.
template <int LPR> __device__ __forceinline__ uint32_t SpanOf(const u32x4 w)
{
    s16x2 hi = Ordered(w[0]), lo = hi;
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        const s16x2 v = Ordered(w[i]);
        hi = __builtin_elementwise_max(hi, v);
        lo = __builtin_elementwise_min(lo, v);
    }
    lo = ~lo;
    s16x2 span = __builtin_elementwise_max(s16x2{hi[0], lo[0]}, s16x2{hi[1], lo[1]}); // maximum, ~minimum
    span = __builtin_elementwise_max(span, Moved<0xb1>(span));  // lanes 1, 0, 3, 2 of four
    span = __builtin_elementwise_max(span, Moved<0x4e>(span));  // lanes 2, 3, 0, 1
    span = __builtin_elementwise_max(span, Moved<0x141>(span)); // eight lanes in reverse
    if constexpr (LPR >= 16) {
        span = __builtin_elementwise_max(span, Moved<0x140>(span)); // sixteen lanes in reverse
    }
    if constexpr (LPR == 32) {
        span = __builtin_elementwise_max(span, __builtin_bit_cast(s16x2, __shfl_xor(__builtin_bit_cast(int, span), 16)));
    }
    span[1] = ~span[1];
    return __builtin_bit_cast(uint32_t, Ordered(span));
}

template <bool BF16> __device__ __forceinline__ RowParams ParamsOfSpan(uint32_t span)
{
    constexpr uint32_t INF = BF16 ? 0x7f80u : 0x7c00u;
    const bool bad = (span & 0x7fffu) >= INF || ((span >> 16) & 0x7fffu) >= INF; // an infinity or NaN somewhere in the row
    return ParamsOf<BF16>(Widen<BF16>(static_cast<uint16_t>(span)), Widen<BF16>(static_cast<uint16_t>(span >> 16)), bad);
}

// The parameters that lane LANE of four neighbouring ones holds.
template <int LANE> __device__ __forceinline__ void FromQuad(const RowParams &p, float &mid, float &inv, uint32_t &word)
{
    mid = __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(p.mid), LANE * 0x55, 0xf, 0xf, true));
    inv = __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(p.inv), LANE * 0x55, 0xf, 0xf, true));
    word = static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(p.word), LANE * 0x55, 0xf, 0xf, true));
}

// The lane's eight values against the row's parameters.
template <bool BF16> __device__ __forceinline__ uint32_t CodesOf(const u32x4 w, float mid, float inv)
{
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = Widen<BF16>(static_cast<uint16_t>(w[i]));
        x[2 * i + 1] = Widen<BF16>(static_cast<uint16_t>(w[i] >> 16));
    }
    return Codes8(x, mid, inv);
}

// One row (token, head) to D / 8 lanes; blockIdx.y: 0 keys, 1 values.
template <int D, bool BF16, bool VEC>
__global__ __launch_bounds__(MOVE_THREADS) void WriteKernel(const WriteArgs a)
{
    constexpr int LPR = D / 8; // lanes a row
    const bool isValue = blockIdx.y != 0;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (MOVE_THREADS / LPR) + threadIdx.x / LPR;
    const int l = threadIdx.x % LPR;
    const bool live = row < a.numRows;
    const int64_t token = live ? row / a.G : 0;
    const int g = live ? static_cast<int>(row - token * a.G) : 0;
    const int64_t slot = live ? a.slots[token] : -1;
    const uint16_t *src = isValue ? a.value + token * a.valueTokenStride : a.key + token * a.keyTokenStride;
    src += g * D + l * 8;
    u32x4 w;
    if constexpr (VEC) {
        w = *reinterpret_cast<const u32x4 *>(src);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = src[2 * i] | (static_cast<uint32_t>(src[2 * i + 1]) << 16);
        }
    }
    const RowParams params = ParamsOfSpan<BF16>(SpanOf<LPR>(w));
    const uint32_t codes = CodesOf<BF16>(w, params.mid, params.inv);
    if (slot < 0 || slot >= a.numSlots) {
        return; // (after the last cross-lane step)
    }
    const int64_t block = static_cast<int32_t>(slot) / a.blockSize;
    const int at = static_cast<int>(slot - block * a.blockSize);
    const int64_t head = block * a.G + g;
    if (isValue) {
        uint8_t *dst = a.valueCache + (head * (D / 2) + l * 4) * a.blockSize + at;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            dst[static_cast<int64_t>(i) * a.blockSize] = static_cast<uint8_t>(codes >> (8 * i));
        }
    } else {
        *reinterpret_cast<uint32_t *>(a.keyCache + (head * a.blockSize + at) * (D / 2) + l * 4) = codes;
    }
    if (l == 0) {
        (isValue ? a.valueParams : a.keyParams)[head * a.blockSize + at] = params.word;
    }
}

// The same for many tokens: a workgroup takes 64 tokens of one head, a wave 16 of them. Value codes lie token after token in
// the cache, so they are turned in LDS: a wave then stores 64 neighbouring tokens' bytes of one channel pair at a time,
// which the memory takes as one piece where the tokens' slots follow each other (as a prompt's do) and byte by byte where
// they do not. (2048 new tokens of 5 sequences with 8 heads of 128 channels: 40 -> 16 us, against bytes stored from
// the lanes of the row; one token a call of 512 sequences: 7 us in rows, 11 us in tiles, so that fewer than 1024 go in rows.)
constexpr int TILE_TOKENS = 64;
constexpr int TILE_FROM = 1024;
template <int D, bool BF16, bool VEC>
__global__ __launch_bounds__(MOVE_THREADS) void WriteTileKernel(const WriteArgs a)
{
    constexpr int LPR = D / 8;
    constexpr int ROWS = WAVE / LPR;    // rows a wave works on at once
    constexpr int STEPS = 16 / ROWS;
    constexpr int PITCH = TILE_TOKENS + 4;
    __shared__ uint8_t turned[D / 2][PITCH];
    __shared__ uint32_t params[TILE_TOKENS];
    const bool isValue = blockIdx.y != 0;
    const int64_t tile = blockIdx.x / a.G;
    const int g = static_cast<int>(blockIdx.x - tile * a.G);
    const int lane = threadIdx.x & (WAVE - 1);
    const int wave = threadIdx.x / WAVE;
    const int l = lane % LPR;
    const int64_t token0 = tile * TILE_TOKENS;
    const int tokens = static_cast<int>(min(static_cast<int64_t>(TILE_TOKENS), a.numRows / a.G - token0));
    const uint16_t *src = (isValue ? a.value : a.key) + g * D + l * 8;
    const int64_t stride = isValue ? a.valueTokenStride : a.keyTokenStride;
    u32x4 w[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const uint16_t *from = src + (token0 + min(wave * 16 + s * ROWS + lane / LPR, tokens - 1)) * stride;
        if constexpr (VEC) {
            w[s] = *reinterpret_cast<const u32x4 *>(from);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[s][i] = from[2 * i] | (static_cast<uint32_t>(from[2 * i + 1]) << 16);
            }
        }
    }
    // The parameters of four rows at a time: each of four neighbouring lanes works out those of one, and gives them to the
    // other three.
    float mid[STEPS], inv[STEPS];
    uint32_t word[STEPS];
#pragma unroll
    for (int s0 = 0; s0 < STEPS; s0 += 4) {
        uint32_t span = SpanOf<LPR>(w[s0]);
#pragma unroll
        for (int s = 1; s < 4 && s0 + s < STEPS; ++s) {
            const uint32_t other = SpanOf<LPR>(w[s0 + s]);
            span = lane % 4 == s ? other : span;
        }
        const RowParams p = ParamsOfSpan<BF16>(span);
        FromQuad<0>(p, mid[s0], inv[s0], word[s0]);
        FromQuad<1>(p, mid[s0 + 1], inv[s0 + 1], word[s0 + 1]);
        if constexpr (STEPS > 2) {
            FromQuad<2>(p, mid[s0 + 2], inv[s0 + 2], word[s0 + 2]);
            FromQuad<3>(p, mid[s0 + 3], inv[s0 + 3], word[s0 + 3]);
        }
    }
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int t = wave * 16 + s * ROWS + lane / LPR; // (past the last token: the last one again, not stored)
        const uint32_t codes = CodesOf<BF16>(w[s], mid[s], inv[s]);
        if (isValue) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                turned[4 * l + i][t] = static_cast<uint8_t>(codes >> (8 * i));
            }
            if (l == 0) {
                params[t] = word[s];
            }
        } else if (t < tokens) {
            const int64_t slot = a.slots[token0 + t];
            if (slot >= 0 && slot < a.numSlots) {
                const int32_t block = static_cast<int32_t>(slot) / a.blockSize;
                const int64_t at = (static_cast<int64_t>(block) * a.G + g) * a.blockSize + (static_cast<int32_t>(slot) - block * a.blockSize);
                *reinterpret_cast<uint32_t *>(a.keyCache + at * (D / 2) + l * 4) = codes;
                if (l == 0) {
                    a.keyParams[at] = word[s];
                }
            }
        }
    }
    if (!isValue) { // (the same for the whole workgroup)
        return;
    }
    __syncthreads();
    const int64_t slot = lane < tokens ? a.slots[token0 + lane] : -1;
    if (slot < 0 || slot >= a.numSlots) {
        return;
    }
    const int64_t block = static_cast<int32_t>(slot) / a.blockSize;
    const int at = static_cast<int>(slot - block * a.blockSize);
    const int64_t head = block * a.G + g;
    uint8_t *dst = a.valueCache + head * (D / 2) * a.blockSize + at;
    for (int pair = wave; pair < D / 2; pair += MOVE_THREADS / WAVE) {
        dst[static_cast<int64_t>(pair) * a.blockSize] = turned[pair][lane];
    }
    if (wave == 0) {
        a.valueParams[head * a.blockSize + at] = params[lane];
    }
}

struct LoadArgs {
    const uint8_t *keyCache;
    const uint8_t *valueCache;
    const uint32_t *keyParams;
    const uint32_t *valueParams;
    const int32_t *tables;
    const int32_t *lens;
    const int32_t *starts;
    uint16_t *key;
    uint16_t *value;
    int64_t outRows;
    int32_t maxBlocksPerSeq;
    int32_t blockSize;
    int32_t numBlocks;
    int32_t G;
    int32_t maxSeqLen;
};

// Sum of the lengths (those below zero count as none) of the sequences before b, by one wave.
__device__ __forceinline__ int64_t RowsBefore(const int32_t *lens, int b, int lane)
{
    int64_t sum = 0;
    for (int i = lane; i < b; i += WAVE) {
        sum += max(lens[i], 0);
    }
#pragma unroll
    for (int step = 1; step < WAVE; step *= 2) {
        sum += __shfl_xor(sum, step);
    }
    return sum;
}

// Eight codes (4 bytes) of one row to eight values of the model's type.
template <bool BF16> __device__ __forceinline__ u32x4 Expand(uint32_t codes, float scale, float mid)
{
    u32x4 out;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float even = __builtin_fmaf(static_cast<float>((codes >> (8 * i)) & 15u) - 7.5f, scale, mid);
        const float odd = __builtin_fmaf(static_cast<float>((codes >> (8 * i + 4)) & 15u) - 7.5f, scale, mid);
        out[i] = NarrowPair<BF16>(even, odd);
    }
    return out;
}

// A wave takes the keys or the values of 16 x (64 / (D / 8)) positions of one sequence and head, counted from the 16-token
// group that holds the sequence's first one: lane (l, grp) owns channels 8 l .. 8 l + 7 of the 16 positions of its group,
// which lie in one block. Everything is asked for before the first row is stored. Value codes lie token after token, so the
// lane reads four 16-byte runs (its four channel pairs) and turns them by 4 x 4 byte transpositions; no shared memory. One
// wave a workgroup: a short prefix is spread over as many CUs as it has pieces. Tables reach further than most sequences
// go, but a workgroup that finds nothing is cheap: with fewer, each going on with later pieces, the longest sequences came
// last (16 sequences with 65000 rows 79 us, 90 with at most 32 workgroups a CU).
template <int D, bool BF16>
__global__ __launch_bounds__(WAVE) void LoadKernel(const LoadArgs a)
{
    constexpr int LPR = D / 8;
    constexpr int GROUPS = WAVE / LPR;
    const int lane = threadIdx.x;
    const bool isValue = (blockIdx.x & 1) != 0;
    const int b = blockIdx.y;
    const int g = blockIdx.z;
    const int l = lane % LPR;
    const int start = a.starts ? a.starts[b] : 0;
    const int len = min(a.lens[b], a.maxSeqLen);
    const int64_t pos0 = (static_cast<int64_t>(start) & ~15LL) + (static_cast<int64_t>(blockIdx.x / 2) * GROUPS + lane / LPR) * 16;
    const int64_t end = static_cast<int64_t>(start) + len;
    if (__ballot(pos0 < end) == 0) {
        return; // (before the sum below, which all lanes take part in)
    }
    const int64_t rowsBefore = RowsBefore(a.lens, b, lane);
    if (pos0 >= end) {
        return;
    }
    if (pos0 < 0 || pos0 >= static_cast<int64_t>(a.maxBlocksPerSeq) * a.blockSize) { // (that is below 2^30)
        return;
    }
    const int tableAt = static_cast<int>(pos0) / a.blockSize;
    const int block = a.tables[static_cast<int64_t>(b) * a.maxBlocksPerSeq + tableAt];
    if (block < 0 || block >= a.numBlocks) {
        return;
    }
    const int at = static_cast<int>(pos0) - tableAt * a.blockSize;
    const int64_t head = static_cast<int64_t>(block) * a.G + g;
    const int64_t firstRow = rowsBefore + pos0 - start; // row of the group's first position (below the sequence's own
                                                        // first row where the group begins in front of it)
    const u32x4 *params = reinterpret_cast<const u32x4 *>((isValue ? a.valueParams : a.keyParams) + head * a.blockSize + at);
    u32x4 param[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        param[q] = params[q];
    }
    uint32_t codes[16];
    if (isValue) {
        const uint8_t *vc = a.valueCache + (head * (D / 2) + l * 4) * a.blockSize + at;
        u32x4 pairs[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            pairs[i] = *reinterpret_cast<const u32x4 *>(vc + static_cast<int64_t>(i) * a.blockSize);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            // tokens 4 q .. 4 q + 3: byte t of pairs[i][q] is pair i of token 4 q + t
            const uint32_t lo01 = __builtin_amdgcn_perm(pairs[1][q], pairs[0][q], 0x05010400u); // t0: p0 p1, t1: p0 p1
            const uint32_t lo23 = __builtin_amdgcn_perm(pairs[3][q], pairs[2][q], 0x05010400u);
            const uint32_t hi01 = __builtin_amdgcn_perm(pairs[1][q], pairs[0][q], 0x07030602u);
            const uint32_t hi23 = __builtin_amdgcn_perm(pairs[3][q], pairs[2][q], 0x07030602u);
            codes[4 * q] = __builtin_amdgcn_perm(lo23, lo01, 0x05040100u);
            codes[4 * q + 1] = __builtin_amdgcn_perm(lo23, lo01, 0x07060302u);
            codes[4 * q + 2] = __builtin_amdgcn_perm(hi23, hi01, 0x05040100u);
            codes[4 * q + 3] = __builtin_amdgcn_perm(hi23, hi01, 0x07060302u);
        }
    } else {
        const uint8_t *kc = a.keyCache + (head * a.blockSize + at) * (D / 2) + l * 4;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            codes[j] = *reinterpret_cast<const uint32_t *>(kc + j * (D / 2));
        }
    }
    u32x4 *out = reinterpret_cast<u32x4 *>((isValue ? a.value : a.key) + (firstRow * a.G + g) * D + l * 8);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        if (pos0 + j >= start && pos0 + j < end && firstRow + j < a.outRows) {
            const uint32_t word = param[j / 4][j % 4];
            out[static_cast<int64_t>(j) * a.G * (D / 8)] = Expand<BF16>(codes[j], ScaleOf<BF16>(word), MidOf<BF16>(word));
        }
    }
}

bool Aligned16(const void *p)
{
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}

} // namespace int4kv
} // namespace atbmi

using namespace atbmi;

extern "C" int atbmi_reshape_and_cache_int4(const void *key, const void *value, uint8_t *keyCache, uint8_t *valueCache,
                                            void *keyParams, void *valueParams, const int32_t *slotMapping,
                                            int64_t numTokens, int64_t numKvHeads, int64_t headDim, int64_t blockSize,
                                            int64_t numBlocks, int64_t keyTokenStride, int64_t valueTokenStride,
                                            int32_t dtype, void *stream)
{
    if (int rc = int4kv::CheckCache("reshape_and_cache_int4", dtype, numKvHeads, headDim, blockSize, numBlocks)) {
        return rc;
    }
    if (numTokens < 0 || numTokens > 0x7fffffffLL || keyTokenStride < numKvHeads * headDim || valueTokenStride < numKvHeads * headDim) {
        return Fail(ERR_INVALID_PARAM, "reshape_and_cache_int4: %lld tokens with strides %lld and %lld (rows of %lld)",
                    (long long)numTokens, (long long)keyTokenStride, (long long)valueTokenStride,
                    (long long)(numKvHeads * headDim));
    }
    if (numTokens == 0) {
        return OK;
    }
    if (!key || !value || !keyCache || !valueCache || !keyParams || !valueParams || !slotMapping) {
        return Fail(ERR_INVALID_PARAM, "reshape_and_cache_int4: every tensor must be non-null");
    }
    if (!int4kv::Aligned16(keyCache) || !int4kv::Aligned16(valueCache) || !int4kv::Aligned16(keyParams) ||
        !int4kv::Aligned16(valueParams)) {
        return Fail(ERR_INVALID_PARAM, "reshape_and_cache_int4: the caches and params must start on 16-byte boundaries");
    }
    int4kv::WriteArgs a{};
    a.key = static_cast<const uint16_t *>(key);
    a.value = static_cast<const uint16_t *>(value);
    a.keyCache = keyCache;
    a.valueCache = valueCache;
    a.keyParams = static_cast<uint32_t *>(keyParams);
    a.valueParams = static_cast<uint32_t *>(valueParams);
    a.slots = slotMapping;
    a.numRows = numTokens * numKvHeads;
    a.numSlots = numBlocks * blockSize;
    a.keyTokenStride = keyTokenStride;
    a.valueTokenStride = valueTokenStride;
    a.G = static_cast<int32_t>(numKvHeads);
    a.blockSize = static_cast<int32_t>(blockSize);
    const bool vec = int4kv::Aligned16(key) && int4kv::Aligned16(value) && keyTokenStride % 8 == 0 && valueTokenStride % 8 == 0;
    const bool tiles = numTokens >= int4kv::TILE_FROM;
    const int64_t rowsPerWg = int4kv::MOVE_THREADS / (headDim / 8);
    const int64_t groups = tiles ? (numTokens + int4kv::TILE_TOKENS - 1) / int4kv::TILE_TOKENS * numKvHeads
                                 : (a.numRows + rowsPerWg - 1) / rowsPerWg;
    if (!int4kv::FitsLaunch(groups, int4kv::MOVE_THREADS)) {
        return Fail(ERR_INVALID_PARAM, "reshape_and_cache_int4: %lld rows are more than one launch takes",
                    (long long)a.numRows);
    }
    const dim3 grid(static_cast<unsigned>(groups), 2);
    hipStream_t s = static_cast<hipStream_t>(stream);
    int4kv::WithHeadDim(headDim, [&](auto d) {
        int4kv::WithFlag(dtype == ATBMI_BF16, [&](auto bf16) {
            int4kv::WithFlag(vec, [&](auto v) {
                constexpr int D = decltype(d)::value;
                constexpr bool BF16 = decltype(bf16)::value, VEC = decltype(v)::value;
                if (tiles) {
                    int4kv::WriteTileKernel<D, BF16, VEC><<<grid, int4kv::MOVE_THREADS, 0, s>>>(a);
                } else {
                    int4kv::WriteKernel<D, BF16, VEC><<<grid, int4kv::MOVE_THREADS, 0, s>>>(a);
                }
            });
        });
    });
    ATBMI_HIP_CHECK(hipGetLastError());
    return OK;
}

extern "C" int atbmi_paged_cache_load_int4(const uint8_t *keyCache, const uint8_t *valueCache, const void *keyParams,
                                           const void *valueParams, const int32_t *blockTables, const int32_t *seqLens,
                                           const int32_t *seqStarts, void *key, void *value, int64_t batch,
                                           int64_t maxBlocksPerSeq, int64_t numKvHeads, int64_t headDim,
                                           int64_t blockSize, int64_t numBlocks, int64_t outRows, int64_t maxSeqLen,
                                           int32_t dtype, void *stream)
{
    if (int rc = int4kv::CheckCache("paged_cache_load_int4", dtype, numKvHeads, headDim, blockSize, numBlocks)) {
        return rc;
    }
    if (batch < 0 || maxBlocksPerSeq <= 0 || maxBlocksPerSeq > ((1LL << 30) - 1) / blockSize || outRows < 0 || maxSeqLen < 0) {
        return Fail(ERR_INVALID_PARAM, "paged_cache_load_int4: batch %lld, %lld blocks a sequence, %lld rows, length %lld",
                    (long long)batch, (long long)maxBlocksPerSeq, (long long)outRows, (long long)maxSeqLen);
    }
    if (batch == 0 || outRows == 0 || maxSeqLen == 0) {
        return OK;
    }
    if (!keyCache || !valueCache || !keyParams || !valueParams || !blockTables || !seqLens || !key || !value) {
        return Fail(ERR_INVALID_PARAM, "paged_cache_load_int4: every tensor but seqStarts must be non-null");
    }
    for (const void *p : {static_cast<const void *>(keyCache), static_cast<const void *>(valueCache), keyParams, valueParams,
                          static_cast<const void *>(key), static_cast<const void *>(value)}) {
        if (!int4kv::Aligned16(p)) {
            return Fail(ERR_INVALID_PARAM, "paged_cache_load_int4: caches, params, key and value must start on 16-byte "
                                           "boundaries");
        }
    }
    // (no sequence is longer than the table's reach, and tokens past the output's rows have no place to go)
    const int64_t longest = std::min({maxSeqLen, maxBlocksPerSeq * blockSize, outRows});
    const int64_t perWg = 16LL * (WAVE / (headDim / 8));
    const int64_t chunks = (longest + 15 + perWg - 1) / perWg; // (a sequence may begin 15 places into its first group)
    if (batch > 65535 || numKvHeads > 65535 || !int4kv::FitsLaunch(2 * chunks, WAVE)) {
        return Fail(ERR_INVALID_PARAM, "paged_cache_load_int4: %lld sequences of %lld tokens with %lld heads are more than one "
                                       "launch takes", (long long)batch, (long long)longest, (long long)numKvHeads);
    }
    int4kv::LoadArgs a{};
    a.keyCache = keyCache;
    a.valueCache = valueCache;
    a.keyParams = static_cast<const uint32_t *>(keyParams);
    a.valueParams = static_cast<const uint32_t *>(valueParams);
    a.tables = blockTables;
    a.lens = seqLens;
    a.starts = seqStarts;
    a.key = static_cast<uint16_t *>(key);
    a.value = static_cast<uint16_t *>(value);
    a.outRows = outRows;
    a.maxBlocksPerSeq = static_cast<int32_t>(maxBlocksPerSeq);
    a.blockSize = static_cast<int32_t>(blockSize);
    a.numBlocks = static_cast<int32_t>(numBlocks);
    a.G = static_cast<int32_t>(numKvHeads);
    a.maxSeqLen = static_cast<int32_t>(longest);
    const dim3 grid(static_cast<unsigned>(2 * chunks), static_cast<unsigned>(batch), static_cast<unsigned>(numKvHeads));
    hipStream_t s = static_cast<hipStream_t>(stream);
    int4kv::WithHeadDim(headDim, [&](auto d) {
        int4kv::WithFlag(dtype == ATBMI_BF16, [&](auto bf16) {
            int4kv::LoadKernel<decltype(d)::value, decltype(bf16)::value><<<grid, WAVE, 0, s>>>(a);
        });
    });
    ATBMI_HIP_CHECK(hipGetLastError());
    return OK;
}
