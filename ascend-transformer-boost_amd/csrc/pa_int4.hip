// Decode attention over the 4-bit cache (atbmi_pa_int4_decode) for gfx950.
//
// Mathematics, per KV head and query column (a column: one query token and one of the query heads of the KV head). A
// cached row is scale (code - 7.5) + mid, so with u = codes (0 .. 15)
//   q . k_t   = ks_t (q . u_t - 7.5 sum q) + km_t sum q
//   sum w v   = sum_t (w_t vs_t) (u_t - 7.5) + sum_t w_t vm_t
// and both contractions run on the codes themselves: the scales meet the scores and the weights, one number a token
// instead of one a channel. Codes become operands of the matrix instructions with a shift and an and-or for two of
// them: 0x4180 | u << 3 is the bf16 number 16 + u, and u alone is the fp16 number u 2^-24, both exact; the constants
// (23.5 sum q; 23.5 sum of the rounded weights) are taken off in fp32 afterwards, against sums of exactly the values
// that were multiplied. (0x4300 | u = 128 + u needs a shift less in eight values, but a long context's output is a
// small difference of sums that carry the offset: at 5000 tokens of fp16 the error against 64 bits was 3.3e-4 with 128,
// of which 2.1e-4 are the output's own rounding.)
//
// Layout of v_mfma_f32_16x16x32_{bf16,f16}: lane (c = lane % 16, kg = lane / 16) supplies contraction values 8 kg ..
// 8 kg + 7 of row c (A) / column c (B) and receives D[4 kg + e][c], e = 0 .. 3. The order of the contraction is free as
// long as both operands share it:
//   scores   A = codes of 16 tokens, B = the query columns. Lane kg holds channels [kg D / 4, (kg + 1) D / 4) of its
//            token: D / 8 bytes side by side; nibble x and x + 4 of a word share an operand register, so the query is
//            permuted the same way. Row m of block st is token 16 (m / 4) + 4 st + m % 4 of the 64-token tile, which
//            leaves lane (c, kg) with the scores of tokens 16 kg .. 16 kg + 15 of column c.
//   values   O^T = V^T P^T: A = value codes, which lie token after token (16 tokens of a channel pair are 16 bytes: a
//            lane's tokens 16 kg .. + 15), B = the lane's own 16 weights. Nothing passes through LDS.
// Running maximum and sums are fp32. The maximum a column is scaled by moves only when a score exceeds it by more
// than 2^8 (in the exponent: 8): weights up to 256 are as exact as weights up to 1, and the accumulators are rescaled
// a few times a context instead of every tile.
//
// Work: the 64-token tiles of all sequences, back to back, are cut into equal ranges (an empty sequence counts as one
// tile); a workgroup of four waves takes one range of one KV head and 16 columns, its waves every fourth tile, and
// joins the waves' sums in LDS at the end of each sequence. A sequence inside one range is written at once; of one that
// was cut, the parts go to fp32 partial rows (range r: part 2 r + 1 if the sequence begins in the range, else 2 r) and
// PaInt4MergeKernel joins them. Lengths are read on the device: every workgroup adds them up for itself.
#include <algorithm>
#include "pa_internal.h"
#include "int4_common.h"

namespace atbmi {
namespace int4kv {

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int TW = 64;          // tokens a tile
constexpr int HT = 16;          // columns a workgroup
constexpr int PA_WAVES = 4;
constexpr int PA_THREADS = PA_WAVES * WAVE;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float STEP_UP = 8.0f; // how far (log2) a score may exceed the reference before that moves

struct PaInt4Args {
    const uint16_t *q;
    const uint8_t *kc;
    const uint8_t *vc;
    const uint32_t *kp;
    const uint32_t *vp;
    const int32_t *tables;
    const int32_t *lens;
    const uint16_t *mask;
    uint16_t *out;
    float *partO; // [2 ranges][pairs][16][D], relative to partM
    float *partM; // [2 ranges][pairs][16], log2
    float *partL;
    int64_t maskSeqStride;
    int64_t maskHeadStride;
    int64_t maskRowStride;
    int32_t maskLen;
    int32_t H;
    int32_t G;
    int32_t group; // H / G
    int32_t tokens; // query tokens a sequence
    int32_t colTiles;
    int32_t batch;
    int32_t maxBlocksPerSeq;
    int32_t blockSize;
    int32_t groupsPerBlock; // blockSize / 16
    uint32_t groupsMagic;   // ceil(2^32 / groupsPerBlock): x / groupsPerBlock for x * groupsPerBlock < 2^32 (0 for 1)
    int32_t numBlocks;
    int32_t ranges;
    float scale2; // qkScale log2(e)
};

__device__ __forceinline__ int ContextLen(const PaInt4Args &a, int b)
{
    return min(max(a.lens[b], 0), a.maxBlocksPerSeq * a.blockSize);
}
__device__ __forceinline__ int TilesOf(int len)
{
    return max(1, (len + TW - 1) / TW);
}

__device__ __forceinline__ int WaveSum(int v)
{
#pragma unroll
    for (int step = 1; step < WAVE; step *= 2) {
        v += __shfl_xor(v, step);
    }
    return v;
}

// Ranges that get work: none shorter than a tile for each wave.
__device__ __forceinline__ int LiveRanges(int ranges, int tiles)
{
    return min(ranges, (tiles + PA_WAVES - 1) / PA_WAVES);
}
__device__ __forceinline__ int RangeBegin(int r, int tiles, int live)
{
    return static_cast<int>(static_cast<int64_t>(tiles) * r / live);
}

__device__ __forceinline__ float QuadMax(float x)
{
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float QuadSum(float x)
{
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

template <bool BF16> __device__ __forceinline__ f32x4 Mfma(u32x4 a, u32x4 b, f32x4 c)
{
    if constexpr (BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
}

// Nibbles x and x + 4 (x = 0 .. 3) of a word as four operand registers.
template <bool BF16> __device__ __forceinline__ u32x4 Spread(uint32_t w)
{
    if constexpr (BF16) {
        constexpr uint32_t M = 0x00780078u, ONE = 0x41804180u;
        return u32x4{((w << 3) & M) | ONE, ((w >> 1) & M) | ONE, ((w >> 5) & M) | ONE, ((w >> 9) & M) | ONE};
    } else {
        constexpr uint32_t M = 0x000f000fu;
        return u32x4{w & M, (w >> 4) & M, (w >> 8) & M, (w >> 12) & M};
    }
}

__device__ __forceinline__ uint32_t PackBf16(float a, float b)
{
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}

template <int D, bool BF16, bool MASK>
__global__ __launch_bounds__(PA_THREADS, D == 256 ? 1 : 2) void PaInt4Kernel(const PaInt4Args a)
{
    constexpr int KW = D / 32; // 32-bit words of a token's codes a lane holds = matrix instructions a 16-token block
    constexpr int CT = D / 32; // tiles of 16 channel pairs
    constexpr int PITCH = D + 4;
    // what the operands stand for beyond u - 7.5, and the factor of u
    constexpr float K_OFFSET = BF16 ? 23.5f : 7.5f;
    constexpr float K_FACTOR = BF16 ? 1.0f : 16777216.0f;
    __shared__ float ldsO[PA_WAVES][HT][PITCH];
    __shared__ float ldsM[PA_WAVES][HT];
    __shared__ float ldsL[PA_WAVES][HT];

    const int lane = threadIdx.x & (WAVE - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int c = lane & 15;
    const int kg = lane >> 4;
    const int pairs = a.G * a.colTiles;
    const int range = blockIdx.x / pairs;
    const int pair = blockIdx.x % pairs;
    const int g = pair / a.colTiles;
    const int ct = pair % a.colTiles;

    // ---- where the range begins
    int tiles = 0;
    for (int b = lane; b < a.batch; b += WAVE) {
        tiles += TilesOf(ContextLen(a, b));
    }
    tiles = WaveSum(tiles);
    const int live = LiveRanges(a.ranges, tiles);
    if (range >= live) {
        return;
    }
    const int begin = RangeBegin(range, tiles, live);
    const int end = RangeBegin(range + 1, tiles, live);
    int seq = 0, before = 0; // the sequence that holds tile `begin`, tiles of the sequences before it
    for (int b0 = 0;; b0 += WAVE) {
        const int mine = b0 + lane < a.batch ? TilesOf(ContextLen(a, b0 + lane)) : 0;
        int upTo = mine;
#pragma unroll
        for (int step = 1; step < WAVE; step *= 2) {
            const int other = __shfl_up(upTo, step);
            upTo += lane >= step ? other : 0;
        }
        const uint64_t past = __ballot(before + upTo > begin);
        if (past != 0) { // (begin < tiles: some sequence holds it)
            const int at = __builtin_ctzll(past);
            seq = b0 + at;
            before += __shfl(upTo - mine, at);
            break;
        }
        before += __shfl(upTo, WAVE - 1);
    }
    seq = __builtin_amdgcn_readfirstlane(seq);
    before = __builtin_amdgcn_readfirstlane(before);

    const int columns = a.group * a.tokens;
    const int col = min(ct * HT + c, columns - 1); // (lanes past the last column repeat it; nothing of theirs is stored)
    const int qTok = col / a.group;
    const int qHead = g * a.group + col % a.group;
    const int liveCols = min(HT, columns - ct * HT);

    for (int at = begin; at < end;) {
        const int len = ContextLen(a, seq);
        const int seqTiles = TilesOf(len);
        const int tBegin = at - before;
        const int tEnd = min(seqTiles, end - before);
        const int32_t *table = a.tables + static_cast<int64_t>(seq) * a.maxBlocksPerSeq;

        // ---- the query columns, permuted as Spread orders the codes, and their sums
        u32x4 q[KW];
        float sumQ = 0.0f;
        const uint16_t *qRow = a.q + (static_cast<int64_t>(seq) * a.tokens + qTok) * a.H * D + static_cast<int64_t>(qHead) * D + kg * (D / 4);
#pragma unroll
        for (int i = 0; i < KW; ++i) {
            const u32x4 w = *reinterpret_cast<const u32x4 *>(qRow + 8 * i);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sumQ += Widen<BF16>(static_cast<uint16_t>(w[e])) + Widen<BF16>(static_cast<uint16_t>(w[e] >> 16));
            }
            q[i] = u32x4{__builtin_amdgcn_perm(w[2], w[0], 0x05040100u), __builtin_amdgcn_perm(w[2], w[0], 0x07060302u),
                         __builtin_amdgcn_perm(w[3], w[1], 0x05040100u), __builtin_amdgcn_perm(w[3], w[1], 0x07060302u)};
        }
        sumQ = QuadSum(sumQ);
        const float midQ = sumQ * a.scale2;
        const float offQ = -K_OFFSET * sumQ * a.scale2;
        const float facQ = K_FACTOR * a.scale2;
        const int seen = len - a.tokens + 1 + qTok; // positions this column sees
        const int allSee = len - a.tokens + 1;      // positions every column sees
        const uint16_t *maskRow = MASK ? a.mask + seq * a.maskSeqStride + qHead * a.maskHeadStride + qTok * a.maskRowStride : nullptr;

        f32x4 acc[CT][2]; // [..][0]: even channels of the pairs, [1]: odd ones
        f32x4 ones = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < CT; ++i) {
            acc[i][0] = acc[i][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        float top = -INFINITY; // the reference (log2)
        float total = 0.0f;    // of the lane's own tokens
        float mids = 0.0f;

        for (int t = tBegin + wave; t < tEnd; t += PA_WAVES) {
            const int t0 = t * TW;
            // ---- block of a 16-token group of the tile; `ok` is false where the id is none
            auto blockOf = [&](int grp, int &place, bool &ok) {
                const uint32_t x = static_cast<uint32_t>(t0 / 16 + grp);
                const uint32_t at16 = a.groupsMagic ? __umulhi(x, a.groupsMagic) : x;
                place = static_cast<int>(x - at16 * a.groupsPerBlock) * 16;
                const int id = table[min(static_cast<int>(at16), a.maxBlocksPerSeq - 1)];
                ok = id >= 0 && id < a.numBlocks;
                return static_cast<int64_t>(ok ? id : 0) * a.G + g;
            };
            int kPlace, vPlace;
            bool kOk, vOk;
            const int64_t kHead = blockOf(c >> 2, kPlace, kOk);
            const int64_t vHead = blockOf(kg, vPlace, vOk);
            // ---- codes
            uint32_t kw[4][KW];
#pragma unroll
            for (int st = 0; st < 4; ++st) {
                const uint8_t *at8 = a.kc + (kHead * a.blockSize + kPlace + 4 * st + (c & 3)) * (D / 2) + kg * (D / 8);
                __builtin_memcpy(kw[st], __builtin_assume_aligned(at8, D / 8 < 16 ? 8 : 16), D / 8);
            }
            u32x4 vw[CT];
#pragma unroll
            for (int i = 0; i < CT; ++i) {
                vw[i] = *reinterpret_cast<const u32x4 *>(a.vc + (vHead * (D / 2) + 16 * i + c) * a.blockSize + vPlace);
            }
            u32x4 kpw[4], vpw[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                kpw[i] = reinterpret_cast<const u32x4 *>(a.kp + vHead * a.blockSize + vPlace)[i];
                vpw[i] = reinterpret_cast<const u32x4 *>(a.vp + vHead * a.blockSize + vPlace)[i];
            }
            // ---- scores of tokens t0 + 16 kg + j, in log2 units
            float s[16];
#pragma unroll
            for (int st = 0; st < 4; ++st) {
                f32x4 dot = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < KW; ++i) {
                    dot = Mfma<BF16>(Spread<BF16>(kw[st][i]), q[i], dot);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t word = kpw[st][e];
                    s[4 * st + e] = __builtin_fmaf(ScaleOf<BF16>(word), __builtin_fmaf(dot[e], facQ, offQ), MidOf<BF16>(word) * midQ);
                }
            }
            const int first = t0 + 16 * kg;
            if constexpr (MASK) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float m = Widen<BF16>(maskRow[min(first + j, a.maskLen - 1)]);
                    // (the lowest finite value leaves fp32 when it is turned into log2 units: it stays finite here, so that
                    // a row of nothing else is the mean of its values; NaN stays NaN)
                    float v = __builtin_fmaf(m, LOG2E, s[j]);
                    v = v < -3.0e38f ? -3.0e38f : v;
                    s[j] = (m == -INFINITY || first + j >= a.maskLen) ? -INFINITY : v;
                }
            }
            if (t0 + TW > allSee || __ballot(!vOk) != 0) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    s[j] = vOk && first + j < seen ? s[j] : -INFINITY;
                }
            }
            // ---- weights
            float most = s[0];
#pragma unroll
            for (int j = 1; j < 16; ++j) {
                most = fmaxf(most, s[j]);
            }
            if (__ballot(most > top + STEP_UP || (top == -INFINITY && most > -INFINITY)) != 0) {
                const float newTop = fmaxf(top, QuadMax(most));
                const float keep = top == -INFINITY ? 0.0f : exp2f(top - newTop);
                top = newTop;
                total *= keep;
                mids *= keep;
                ones *= keep;
#pragma unroll
                for (int i = 0; i < CT; ++i) {
                    acc[i][0] *= keep;
                    acc[i][1] *= keep;
                }
            }
            const float base = top == -INFINITY ? 0.0f : top;
            float pv[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float p = __builtin_amdgcn_exp2f(s[j] - base);
                const uint32_t word = vpw[j / 4][j % 4];
                total += p;
                // (a hidden token's params may hold anything: 0 times them must be 0)
                const bool none = s[j] == -INFINITY;
                pv[j] = none ? 0.0f : p * ScaleOf<BF16>(word);
                mids += none ? 0.0f : p * MidOf<BF16>(word);
            }
            // ---- values. The weights (times the value scale) are rounded to bf16, which has fp32's range whatever the
            // scales are: an error of at most 2^-8 each for bf16 models, whose output is rounded as coarsely; for fp16
            // models the remainder is multiplied as well (2^-16 left).
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                u32x4 pw, pr;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int j = 8 * h + 4 * (e / 2) + e % 2; // tokens j and j + 2 share a register, as Spread leaves them
                    pw[e] = PackBf16(pv[j], pv[j + 2]);
                    if constexpr (!BF16) {
                        pr[e] = PackBf16(pv[j] - __uint_as_float(pw[e] << 16), pv[j + 2] - __uint_as_float(pw[e] & 0xffff0000u));
                    }
                }
                constexpr uint32_t ONE = 0x3f803f80u;
                const u32x4 one = {ONE, ONE, ONE, ONE};
                ones = Mfma<true>(one, pw, ones);
                if constexpr (!BF16) {
                    ones = Mfma<true>(one, pr, ones);
                }
#pragma unroll
                for (int i = 0; i < CT; ++i) {
                    const uint32_t w0 = vw[i][2 * h], w1 = vw[i][2 * h + 1];
                    const u32x4 a0 = Spread<true>(w0), a1 = Spread<true>(w1); // low, high half of tokens 0, 2; of 1, 3
                    const u32x4 even = {a0[0], a0[2], a1[0], a1[2]};
                    const u32x4 odd = {a0[1], a0[3], a1[1], a1[3]};
                    acc[i][0] = Mfma<true>(even, pw, acc[i][0]);
                    acc[i][1] = Mfma<true>(odd, pw, acc[i][1]);
                    if constexpr (!BF16) {
                        acc[i][0] = Mfma<true>(even, pr, acc[i][0]);
                        acc[i][1] = Mfma<true>(odd, pr, acc[i][1]);
                    }
                }
            }
        }

        // ---- join the waves
        total = QuadSum(total);
        mids = QuadSum(mids);
        const int busy = min(PA_WAVES, tEnd - tBegin);
        __syncthreads(); // (the rows of the sequence before have been read)
        if (kg == 0) {
            ldsM[wave][c] = top;
        }
        __syncthreads();
        float joint = -INFINITY;
        for (int w = 0; w < busy; ++w) {
            joint = fmaxf(joint, ldsM[w][c]);
        }
        const float f = top == -INFINITY ? 0.0f : exp2f(top - joint);
        if (wave < busy) {
            if (kg == 0) {
                ldsL[wave][c] = total * f;
            }
            const float rest = mids - 23.5f * ones[0];
#pragma unroll
            for (int i = 0; i < CT; ++i) {
                float *to = &ldsO[wave][c][32 * i + 8 * kg];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    to[2 * e] = top == -INFINITY ? 0.0f : (acc[i][0][e] + rest) * f;
                    to[2 * e + 1] = top == -INFINITY ? 0.0f : (acc[i][1][e] + rest) * f;
                }
            }
        }
        __syncthreads();
        const bool whole = tBegin == 0 && tEnd == seqTiles;
        const int64_t part = static_cast<int64_t>(2 * range + (tBegin == 0 ? 1 : 0)) * pairs + pair;
        for (int i = threadIdx.x; i < liveCols * (D / 4); i += PA_THREADS) {
            const int n = i / (D / 4);
            const int d = i % (D / 4) * 4;
            f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
            float l = 0.0f;
            for (int w = 0; w < busy; ++w) {
                o += *reinterpret_cast<const f32x4 *>(&ldsO[w][n][d]);
                l += ldsL[w][n];
            }
            if (whole) {
                const float inv = l > 0.0f ? 1.0f / l : (l == l ? 0.0f : l); // nothing seen: zeros; NaN stays
                const int cc = ct * HT + n;
                uint16_t *dst = a.out + ((static_cast<int64_t>(seq) * a.tokens + cc / a.group) * a.H + g * a.group + cc % a.group) * D + d;
                u32x2 w;
                w[0] = static_cast<uint32_t>(Narrow<BF16>(o[0] * inv)) | (static_cast<uint32_t>(Narrow<BF16>(o[1] * inv)) << 16);
                w[1] = static_cast<uint32_t>(Narrow<BF16>(o[2] * inv)) | (static_cast<uint32_t>(Narrow<BF16>(o[3] * inv)) << 16);
                *reinterpret_cast<u32x2 *>(dst) = w;
            } else {
                *reinterpret_cast<f32x4 *>(a.partO + (part * HT + n) * D + d) = o;
                if (d == 0) {
                    a.partL[part * HT + n] = l;
                }
            }
        }
        if (!whole && threadIdx.x < liveCols) {
            float m = -INFINITY;
            for (int w = 0; w < busy; ++w) {
                m = fmaxf(m, ldsM[w][threadIdx.x]);
            }
            a.partM[part * HT + threadIdx.x] = m;
        }
        before += seqTiles;
        at = before;
        ++seq;
    }
}

// Joins the parts of a sequence that was cut: out = sum 2^(M_p - M) O_p / sum 2^(M_p - M) L_p. A workgroup takes one
// sequence and one pair; a thread four channels of a column.
template <int D, bool BF16> __global__ __launch_bounds__(PA_THREADS) void PaInt4MergeKernel(const PaInt4Args a)
{
    const int lane = threadIdx.x & (WAVE - 1);
    const int pairs = a.G * a.colTiles;
    const int seq = blockIdx.x / pairs;
    const int pair = blockIdx.x % pairs;
    const int g = pair / a.colTiles;
    const int ct = pair % a.colTiles;
    int tiles = 0, before = 0;
    for (int b = lane; b < a.batch; b += WAVE) {
        const int mine = TilesOf(ContextLen(a, b));
        tiles += mine;
        before += b < seq ? mine : 0;
    }
    tiles = WaveSum(tiles);
    before = WaveSum(before);
    const int live = LiveRanges(a.ranges, tiles);
    const int last = before + TilesOf(ContextLen(a, seq)) - 1;
    auto rangeOf = [&](int tile) { // the range r with begin(r) <= tile < begin(r + 1)
        return static_cast<int>(((static_cast<int64_t>(tile) + 1) * live - 1) / tiles);
    };
    const int r0 = rangeOf(before);
    const int r1 = rangeOf(last);
    if (r0 == r1) {
        return;
    }
    const int columns = a.group * a.tokens;
    const int liveCols = min(HT, columns - ct * HT);
    // (the part that begins the sequence is its range's second kind, the others are the first)
    auto partOf = [&](int r) { return static_cast<int64_t>(2 * r + (r == r0 ? 1 : 0)) * pairs + pair; };
    for (int i = threadIdx.x; i < liveCols * (D / 4); i += PA_THREADS) {
        const int n = i / (D / 4);
        const int d = i % (D / 4) * 4;
        float top = -INFINITY;
        for (int r = r0; r <= r1; ++r) {
            top = fmaxf(top, a.partM[partOf(r) * HT + n]);
        }
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        float l = 0.0f;
        for (int r = r0; r <= r1; ++r) {
            const int64_t at = partOf(r) * HT + n;
            const float m = a.partM[at];
            const float w = m == -INFINITY ? 0.0f : exp2f(m - top);
            l += w * a.partL[at];
            o += w * *reinterpret_cast<const f32x4 *>(a.partO + at * D + d);
        }
        const float inv = l > 0.0f ? 1.0f / l : (l == l ? 0.0f : l);
        const int cc = ct * HT + n;
        uint16_t *dst = a.out + ((static_cast<int64_t>(seq) * a.tokens + cc / a.group) * a.H + g * a.group + cc % a.group) * D + d;
        u32x2 w;
        w[0] = static_cast<uint32_t>(Narrow<BF16>(o[0] * inv)) | (static_cast<uint32_t>(Narrow<BF16>(o[1] * inv)) << 16);
        w[1] = static_cast<uint32_t>(Narrow<BF16>(o[2] * inv)) | (static_cast<uint32_t>(Narrow<BF16>(o[3] * inv)) << 16);
        *reinterpret_cast<u32x2 *>(dst) = w;
    }
}

int CheckCall(const AtbmiPaInt4Call *c)
{
    if (!c) {
        return Fail(ERR_INVALID_PARAM, "pa_int4: null call");
    }
    if (int rc = CheckCache("pa_int4", c->dtype, c->numKvHeads, c->headDim, c->blockSize, c->numBlocks)) {
        return rc;
    }
    if (c->numHeads <= 0 || c->numHeads % c->numKvHeads != 0 || c->numHeads > (1 << 20)) {
        return Fail(ERR_INVALID_PARAM, "pa_int4: %d heads over %d KV heads", c->numHeads, c->numKvHeads);
    }
    if (c->batch < 0 || c->queryTokens < 1 || c->queryTokens > 64 || c->maxBlocksPerSeq <= 0 ||
        static_cast<int64_t>(c->maxBlocksPerSeq) * c->blockSize >= (1LL << 30) || c->reserved != 0) {
        return Fail(ERR_INVALID_PARAM, "pa_int4: batch %d, %d query tokens, %d blocks a sequence, reserved %d", c->batch,
                    c->queryTokens, c->maxBlocksPerSeq, c->reserved);
    }
    // (tiles of all sequences are counted in 32 bits)
    const int64_t mostTiles = (static_cast<int64_t>(c->maxBlocksPerSeq) * c->blockSize + TW - 1) / TW;
    if (mostTiles * c->batch > 0x7fffffffLL) {
        return Fail(ERR_INVALID_PARAM, "pa_int4: %d sequences of up to %lld tokens are more than one call takes", c->batch,
                    (long long)mostTiles * TW);
    }
    if (!(c->qkScale > 0.0f) || !__builtin_isfinite(c->qkScale)) {
        return Fail(ERR_INVALID_PARAM, "pa_int4: qkScale %g", c->qkScale);
    }
    if (c->mask && (c->maskLen <= 0 || c->maskSeqStride < 0 || c->maskHeadStride < 0 || c->maskRowStride < 0)) {
        return Fail(ERR_INVALID_PARAM, "pa_int4: a mask of %d positions with strides %lld, %lld, %lld", c->maskLen,
                    (long long)c->maskSeqStride, (long long)c->maskHeadStride, (long long)c->maskRowStride);
    }
    return OK;
}

struct PaInt4Shape {
    int colTiles = 1;
    int64_t pairs = 1;
    int64_t ranges = 1;
    bool merge = false; // some sequence may be cut
    uint64_t partO = 0, partM = 0, partL = 0, bytes = 0;
};

PaInt4Shape ShapeOf(const AtbmiPaInt4Call *c)
{
    PaInt4Shape s;
    const int64_t columns = static_cast<int64_t>(c->numHeads / c->numKvHeads) * c->queryTokens;
    s.colTiles = static_cast<int>((columns + HT - 1) / HT);
    s.pairs = s.colTiles * static_cast<int64_t>(c->numKvHeads);
    const int64_t mostTiles = (static_cast<int64_t>(c->maxBlocksPerSeq) * c->blockSize + TW - 1) / TW;
    const int64_t perCu = c->headDim == 256 ? 1 : 2; // workgroups a CU holds at once (registers)
    s.ranges = std::max<int64_t>(1, DeviceComputeUnits() * perCu / s.pairs);
    s.ranges = std::min<int64_t>(s.ranges, std::max<int64_t>(1, (mostTiles * c->batch + PA_WAVES - 1) / PA_WAVES));
    s.merge = s.ranges > 1 && mostTiles > 1;
    if (s.merge) {
        const uint64_t rows = static_cast<uint64_t>(2 * s.ranges * s.pairs) * HT;
        auto align = [](uint64_t v) { return (v + 255) / 256 * 256; };
        s.partM = align(rows * c->headDim * sizeof(float));
        s.partL = s.partM + align(rows * sizeof(float));
        s.bytes = s.partL + rows * sizeof(float);
    }
    return s;
}

} // namespace int4kv
} // namespace atbmi

using namespace atbmi;

extern "C" int atbmi_pa_int4_workspace_size(const AtbmiPaInt4Call *call, uint64_t *bytes)
{
    if (!bytes) {
        return Fail(ERR_INVALID_PARAM, "pa_int4_workspace_size: null result pointer");
    }
    if (int rc = int4kv::CheckCall(call)) {
        return rc;
    }
    *bytes = int4kv::ShapeOf(call).bytes;
    return OK;
}

extern "C" int atbmi_pa_int4_decode(const AtbmiPaInt4Call *call, void *workspace, uint64_t workspaceBytes, void *stream)
{
    if (int rc = int4kv::CheckCall(call)) {
        return rc;
    }
    if (call->batch == 0) {
        return OK;
    }
    if (!call->query || !call->keyCache || !call->valueCache || !call->keyParams || !call->valueParams ||
        !call->blockTables || !call->contextLens || !call->out) {
        return Fail(ERR_INVALID_PARAM, "pa_int4: every tensor but the mask must be non-null");
    }
    for (const void *p : {call->query, static_cast<const void *>(call->keyCache), static_cast<const void *>(call->valueCache),
                          call->keyParams, call->valueParams, static_cast<const void *>(call->out)}) {
        if ((reinterpret_cast<uintptr_t>(p) & 15) != 0) {
            return Fail(ERR_INVALID_PARAM, "pa_int4: query, caches, params and out must start on 16-byte boundaries");
        }
    }
    const int4kv::PaInt4Shape shape = int4kv::ShapeOf(call);
    if (shape.bytes > 0 && (!workspace || workspaceBytes < shape.bytes)) {
        return Fail(ERR_INVALID_PARAM, "pa_int4: workspace of %llu bytes, %llu needed", (unsigned long long)workspaceBytes,
                    (unsigned long long)shape.bytes);
    }
    if ((reinterpret_cast<uintptr_t>(workspace) & 15) != 0) {
        return Fail(ERR_INVALID_PARAM, "pa_int4: the workspace must start on a 16-byte boundary");
    }
    const int64_t grid = shape.ranges * shape.pairs;
    const int64_t mergeGrid = shape.pairs * call->batch;
    if (grid > 0x7fffffffLL || mergeGrid > 0x7fffffffLL) {
        return Fail(ERR_INVALID_PARAM, "pa_int4: %lld workgroups", (long long)std::max(grid, mergeGrid));
    }
    int4kv::PaInt4Args a{};
    a.q = static_cast<const uint16_t *>(call->query);
    a.kc = call->keyCache;
    a.vc = call->valueCache;
    a.kp = static_cast<const uint32_t *>(call->keyParams);
    a.vp = static_cast<const uint32_t *>(call->valueParams);
    a.tables = call->blockTables;
    a.lens = call->contextLens;
    a.mask = static_cast<const uint16_t *>(call->mask);
    a.out = static_cast<uint16_t *>(call->out);
    if (shape.bytes > 0) {
        unsigned char *ws = static_cast<unsigned char *>(workspace);
        a.partO = reinterpret_cast<float *>(ws + shape.partO);
        a.partM = reinterpret_cast<float *>(ws + shape.partM);
        a.partL = reinterpret_cast<float *>(ws + shape.partL);
    }
    a.maskSeqStride = call->maskSeqStride;
    a.maskHeadStride = call->maskHeadStride;
    a.maskRowStride = call->maskRowStride;
    a.maskLen = call->maskLen;
    a.H = call->numHeads;
    a.G = call->numKvHeads;
    a.group = call->numHeads / call->numKvHeads;
    a.tokens = call->queryTokens;
    a.colTiles = shape.colTiles;
    a.batch = call->batch;
    a.maxBlocksPerSeq = call->maxBlocksPerSeq;
    a.blockSize = call->blockSize;
    a.groupsPerBlock = call->blockSize / 16;
    a.groupsMagic = a.groupsPerBlock == 1 ? 0 : static_cast<uint32_t>(((1ULL << 32) + a.groupsPerBlock - 1) / a.groupsPerBlock);
    a.numBlocks = call->numBlocks;
    a.ranges = static_cast<int32_t>(shape.ranges);
    a.scale2 = call->qkScale * int4kv::LOG2E;
    hipStream_t s = static_cast<hipStream_t>(stream);
    int rc = OK;
    int4kv::WithHeadDim(call->headDim, [&](auto d) {
        int4kv::WithFlag(call->dtype == ATBMI_BF16, [&](auto bf16) {
            constexpr int D = decltype(d)::value;
            constexpr bool BF16 = decltype(bf16)::value;
            int4kv::WithFlag(call->mask != nullptr, [&](auto mask) {
                int4kv::PaInt4Kernel<D, BF16, decltype(mask)::value>
                    <<<static_cast<unsigned>(grid), int4kv::PA_THREADS, 0, s>>>(a);
            });
            if (hipError_t e = hipGetLastError(); e != hipSuccess) {
                rc = Fail(ERR_RT_FAIL, "pa_int4: launch failed: %s", hipGetErrorString(e));
            } else if (shape.merge) {
                int4kv::PaInt4MergeKernel<D, BF16><<<static_cast<unsigned>(mergeGrid), int4kv::PA_THREADS, 0, s>>>(a);
            }
        });
    });
    if (rc != OK) {
        return rc;
    }
    ATBMI_HIP_CHECK(hipGetLastError());
    return OK;
}
