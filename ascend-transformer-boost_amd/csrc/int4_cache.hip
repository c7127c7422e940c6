// The 4-bit KV cache: the write that quantises key and value rows into it and the gather that gives them back
// (atbmi_reshape_and_cache_int4, atbmi_paged_cache_load_int4). The layout is described in atbmi_kernels.h; a row of
// D channels is D codes of 4 bits, a scale and a middle value.
//
// Both move a few bytes per value and compute next to nothing: HBM bounds them on long calls and the launch on short
// ones. In both kernels a lane owns eight channels of a row (16 bytes in the model's type, 4 bytes of codes), D / 8
// lanes a row, so that rows of the model's type move in 16-byte pieces.
#include "pa_internal.h"
#include "int4_common.h"

namespace atbmi {
namespace int4kv {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

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
    float x[8];
    if constexpr (VEC) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(src);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = Widen<BF16>(static_cast<uint16_t>(w[i]));
            x[2 * i + 1] = Widen<BF16>(static_cast<uint16_t>(w[i] >> 16));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = Widen<BF16>(src[i]);
        }
    }
    float hi = x[0], lo = x[0];
    bool finite = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        hi = fmaxf(hi, x[i]);
        lo = fminf(lo, x[i]);
        finite = finite && __builtin_isfinite(x[i]);
    }
    float bad = finite ? 0.0f : 1.0f;
#pragma unroll
    for (int step = 1; step < LPR; step *= 2) {
        hi = fmaxf(hi, __shfl_xor(hi, step));
        lo = fminf(lo, __shfl_xor(lo, step));
        bad = fmaxf(bad, __shfl_xor(bad, step));
    }
    if (slot < 0 || slot >= a.numSlots) {
        return; // (after the last cross-lane step)
    }
    const RowParams p = ParamsOf<BF16>(hi, lo, bad != 0.0f);
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        codes |= CodeOf(x[i], p) << (4 * i);
    }
    const int64_t block = slot / a.blockSize;
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
        (isValue ? a.valueParams : a.keyParams)[head * a.blockSize + at] = p.word;
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
        out[i] = static_cast<uint32_t>(Narrow<BF16>(even)) | (static_cast<uint32_t>(Narrow<BF16>(odd)) << 16);
    }
    return out;
}

// A wave takes 16 x (64 / (D / 8)) positions of one sequence and head, counted from the 16-token group that holds the
// sequence's first one: lane (l, grp) owns channels 8 l .. 8 l + 7 of the 16 positions of its group, which lie in one
// block. Value codes lie token after token, so the lane reads four 16-byte runs (its four channel pairs) and turns
// them by 4 x 4 byte transpositions; no shared memory.
template <int D, bool BF16>
__global__ __launch_bounds__(MOVE_THREADS) void LoadKernel(const LoadArgs a)
{
    constexpr int LPR = D / 8;
    constexpr int GROUPS = WAVE / LPR;
    const int lane = threadIdx.x & (WAVE - 1);
    const int wave = threadIdx.x / WAVE;
    const int b = blockIdx.y;
    const int g = blockIdx.z;
    const int l = lane % LPR;
    const int start = a.starts ? max(a.starts[b], 0) : 0;
    const int len = min(a.lens[b], a.maxSeqLen);
    const int64_t pos0 = (static_cast<int64_t>(start) & ~15LL) +
                         ((static_cast<int64_t>(blockIdx.x) * (MOVE_THREADS / WAVE) + wave) * GROUPS + lane / LPR) * 16;
    const int64_t end = static_cast<int64_t>(start) + len;
    const int64_t rowsBefore = RowsBefore(a.lens, b, lane);
    if (pos0 >= end) {
        return;
    }
    const int64_t tableAt = pos0 / a.blockSize;
    if (tableAt >= a.maxBlocksPerSeq) {
        return;
    }
    const int block = a.tables[static_cast<int64_t>(b) * a.maxBlocksPerSeq + tableAt];
    if (block < 0 || block >= a.numBlocks) {
        return;
    }
    const int at = static_cast<int>(pos0 - tableAt * a.blockSize);
    const int64_t head = static_cast<int64_t>(block) * a.G + g;
    const int64_t firstRow = rowsBefore + pos0 - start; // row of the group's first position (below the sequence's own
                                                        // first row where the group begins in front of it)
    const uint8_t *kc = a.keyCache + (head * a.blockSize + at) * (D / 2) + l * 4;
    const uint32_t *kp = a.keyParams + head * a.blockSize + at;
    const uint32_t *vp = a.valueParams + head * a.blockSize + at;
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
        const uint32_t codes[4] = {
            __builtin_amdgcn_perm(lo23, lo01, 0x05040100u), __builtin_amdgcn_perm(lo23, lo01, 0x07060302u),
            __builtin_amdgcn_perm(hi23, hi01, 0x05040100u), __builtin_amdgcn_perm(hi23, hi01, 0x07060302u)};
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int j = 4 * q + t;
            const int64_t row = firstRow + j;
            if (pos0 + j >= start && pos0 + j < end && row < a.outRows) {
                const int64_t dst = (row * a.G + g) * D + l * 8;
                const uint32_t kw = kp[j];
                const uint32_t vw = vp[j];
                const uint32_t kcodes = *reinterpret_cast<const uint32_t *>(kc + static_cast<int64_t>(j) * (D / 2));
                *reinterpret_cast<u32x4 *>(a.key + dst) = Expand<BF16>(kcodes, ScaleOf<BF16>(kw), MidOf<BF16>(kw));
                *reinterpret_cast<u32x4 *>(a.value + dst) = Expand<BF16>(codes[t], ScaleOf<BF16>(vw), MidOf<BF16>(vw));
            }
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
    if (numTokens < 0 || keyTokenStride < numKvHeads * headDim || valueTokenStride < numKvHeads * headDim) {
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
    const int64_t rowsPerWg = int4kv::MOVE_THREADS / (headDim / 8);
    const int64_t groups = (a.numRows + rowsPerWg - 1) / rowsPerWg;
    if (groups > 0x7fffffffLL) {
        return Fail(ERR_INVALID_PARAM, "reshape_and_cache_int4: %lld rows are more than one launch takes",
                    (long long)a.numRows);
    }
    const dim3 grid(static_cast<unsigned>(groups), 2);
    hipStream_t s = static_cast<hipStream_t>(stream);
    int4kv::WithHeadDim(headDim, [&](auto d) {
        int4kv::WithFlag(dtype == ATBMI_BF16, [&](auto bf16) {
            int4kv::WithFlag(vec, [&](auto v) {
                int4kv::WriteKernel<decltype(d)::value, decltype(bf16)::value, decltype(v)::value>
                    <<<grid, int4kv::MOVE_THREADS, 0, s>>>(a);
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
    if (batch < 0 || maxBlocksPerSeq <= 0 || maxBlocksPerSeq * blockSize >= (1LL << 30) || outRows < 0 || maxSeqLen < 0) {
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
    // (no sequence is longer than the table's reach)
    const int64_t longest = maxSeqLen < maxBlocksPerSeq * blockSize ? maxSeqLen : maxBlocksPerSeq * blockSize;
    const int64_t perWg = 16LL * (int4kv::MOVE_THREADS / (headDim / 8));
    const int64_t chunks = (longest + 15 + perWg - 1) / perWg; // (a sequence may begin 15 places into its first group)
    if (batch > 65535 || numKvHeads > 65535) {
        return Fail(ERR_INVALID_PARAM, "paged_cache_load_int4: %lld sequences with %lld heads are more than one launch takes",
                    (long long)batch, (long long)numKvHeads);
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
    const dim3 grid(static_cast<unsigned>(chunks), static_cast<unsigned>(batch), static_cast<unsigned>(numKvHeads));
    hipStream_t s = static_cast<hipStream_t>(stream);
    int4kv::WithHeadDim(headDim, [&](auto d) {
        int4kv::WithFlag(dtype == ATBMI_BF16, [&](auto bf16) {
            int4kv::LoadKernel<decltype(d)::value, decltype(bf16)::value><<<grid, int4kv::MOVE_THREADS, 0, s>>>(a);
        });
    });
    ATBMI_HIP_CHECK(hipGetLastError());
    return OK;
}
