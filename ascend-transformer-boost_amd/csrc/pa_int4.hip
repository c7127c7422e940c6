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
//            lane's tokens 16 kg .. + 15), B = the lane's own 16 weights. With 16 columns the weights stay in the lane
//            that has the scores; with fewer, scores and weights pass through LDS once so that no lane computes the
//            softmax of a repeated column (batch of 64, 4 columns, 1024 to 4096 tokens: 49.5 -> 47.8 us).
// Running maximum and sums are fp32. The maximum a column is scaled by moves only when a score exceeds it by more
// than 2^8 (in the exponent: 8): weights up to 256 are as exact as weights up to 1, and the accumulators are rescaled
// a few times a context instead of every tile.
//
// Work: the 64-token tiles of all sequences, back to back, each sequence behind START units that stand for what it costs
// beyond its tiles, are cut into equal ranges (an empty sequence has one tile); a workgroup of four waves takes one range of one KV head and 16 columns, its waves every fourth tile, and
// joins the waves' sums in LDS at the end of each sequence. A sequence inside one range is written at once; of one that
// was cut, the parts go to fp32 partial rows (range r: part 2 r + 1 if the sequence begins in the range, else 2 r) and
// PaInt4MergeKernel joins them. Lengths are read on the device: every workgroup adds them up for itself.
#include <algorithm>
#include "pa_internal.h"
#include "int4_common.h"

// (the lambdas of the kernel hold its registers: called, they would move them to memory)
#define ATBMI_INLINE __attribute__((always_inline))

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
constexpr int MERGE_MOST_THREADS = 1024;
constexpr float LOG2E = 1.4426950408889634f;
constexpr int START = 8;        // see UnitsOf
constexpr int WHOLE_TILES = 16; // see ShapeOf
constexpr float STEP_UP = 8.0f; // how far (log2) a score may exceed the reference before that moves
// bf16 values may lie so high that the sums leave fp32: weights of up to 2^8 times scales of up to 2^125.1 times operands of up
// to 31, over up to 2^30 tokens, come to 2^168. Columns whose sums are not below FAR are not stored; the range's part of that
// sequence goes through once more for them, with its weights brought down by 2^DOWN, which their total shares. (Below FAR, 2^31
// parts may be added up. The others are stored the first time only: `out` may be the query, which is then no longer there. All
// this costs ordinary rows 0.6 us of 47.4 with a batch of 64 and of 43.8 with four query tokens, 1 % with 64 or 256 channels.)
constexpr float FAR = 0x1p96f;
constexpr float DOWN = 48.0f;

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
    int32_t maskVec; // every mask row starts on a 16-byte boundary
    int32_t H;
    int32_t G;
    int32_t group; // H / G
    int32_t tokens; // query tokens a sequence
    int32_t colTiles;
    int32_t batch;
    int32_t maxBlocksPerSeq;
    int32_t blockSize;
    int32_t tilesPerBlock;  // blockSize / 64, 0 where that is no whole number
    uint32_t tilesMagic;    // as groupsMagic, for tilesPerBlock
    int32_t groupsPerBlock; // blockSize / 16
    uint32_t groupsMagic;   // ceil(2^32 / groupsPerBlock): x / groupsPerBlock for x * groupsPerBlock < 2^32 (0 for 1)
    int32_t numBlocks;
    int32_t whole;          // 1: range r is sequence r, nothing is cut
    int32_t ranges;
    float scale2; // qkScale log2(e)
};

__device__ __forceinline__ int ContextLen(const PaInt4Args &a, int b)
{
    return min(max(a.lens[b], 0), a.maxBlocksPerSeq * a.blockSize);
}
// The same through the scalar cache, for a sequence that all lanes agree on: not counted with the tiles on their way.
template <typename T> __device__ __forceinline__ const __attribute__((address_space(4))) T *Scalar(const T *p)
{
    return reinterpret_cast<const __attribute__((address_space(4))) T *>(reinterpret_cast<uintptr_t>(p));
}
__device__ __forceinline__ int UniformLen(const PaInt4Args &a, int b)
{
    return min(max(Scalar(a.lens)[b], 0), a.maxBlocksPerSeq * a.blockSize);
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
    return __builtin_amdgcn_readfirstlane(v);
}

// What is cut into ranges: the tiles of a sequence behind START units that stand for none. They are what a sequence costs
// a workgroup beyond its tiles (its first tiles are waited for, its sums are joined), so that equal ranges take equally
// long. (19 sequences of 256 .. 32768 with 16 columns: 49.2 us with 2, 46.8 with 4, 43.9 with 8, 44.0 with 11; 64 sequences
// of 1024 .. 4096 with 4 columns: 49.1, 48.6, 47.8 and 47.7.)
__device__ __forceinline__ int UnitsOf(int len)
{
    return TilesOf(len) + START;
}
// Ranges that get work: none shorter than a tile for each wave.
__device__ __forceinline__ int LiveRanges(int ranges, int units)
{
    return min(ranges, (units + PA_WAVES - 1) / PA_WAVES);
}
__device__ __forceinline__ int RangeBegin(int r, int units, int live)
{
    return static_cast<int>(static_cast<int64_t>(units) * r / live);
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
        // (one instruction for the and and the or wants its constants in registers: two literals would make two of it)
        uint32_t m = 0x00780078u, one = 0x41804180u;
        asm("" : "+s"(m), "+v"(one));
        return u32x4{((w << 3) & m) | one, ((w >> 1) & m) | one, ((w >> 5) & m) | one, ((w >> 9) & m) | one};
    } else {
        constexpr uint32_t M = 0x000f000fu;
        return u32x4{w & M, (w >> 4) & M, (w >> 8) & M, (w >> 12) & M};
    }
}

__device__ __forceinline__ uint32_t LdsAddress(const void *p)
{
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void *)p));
}

__device__ __forceinline__ uint32_t PackBf16(float a, float b)
{
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}

// 16 bytes (4 bytes) a lane to LDS at ldsAt + 16 (4) x lane, from an address of its own or from an offset to the wave's;
// read once, so not to displace anything. Value codes in long blocks are left in the L2 a while (Kept): a 64-token tile takes
// half of each 128-byte line of theirs, and the wave that takes the other half comes about the same time (fp16, batch of 128 with
// 2048 .. 8192 tokens: 156 -> 149 us, and slower again with the keys kept as well; with 64 and 256 channels 3 % slower).
__device__ __forceinline__ void ToLds16(const void *from, uint32_t ldsAt)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"s"(ldsAt), "v"(from) : "memory", "m0");
}
__device__ __forceinline__ void ToLds4(const void *from, uint32_t ldsAt)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off nt" ::"s"(ldsAt), "v"(from) : "memory", "m0");
}
__device__ __forceinline__ void ToLds16(const void *base, uint32_t offset, uint32_t ldsAt)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(ldsAt), "v"(offset), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void ToLds4(const void *base, uint32_t offset, uint32_t ldsAt)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2 nt" ::"s"(ldsAt), "v"(offset), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void ToLds16Kept(const void *base, uint32_t offset, uint32_t ldsAt)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(ldsAt), "v"(offset), "s"(base) : "memory", "m0");
}
// Orders a wave's LDS writes before its own later reads and the other way round: a wave's LDS instructions execute in
// order, only the compiler has to keep them.
__device__ __forceinline__ void WaveSync()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A wave's tile in LDS: key codes token after token (rows of D / 2 bytes), value codes in blocks of 16 channel pairs by 64
// tokens (rows of 64 bytes), the params of the 64 keys, those of the values. The 16-byte pieces of a row are permuted by an
// exclusive or so that the rows the matrix instruction reads side by side lie in different banks.
template <int D> struct TileLayout {
    static constexpr int KEYS = TW * D / 2, VALUES = TW * D / 2;
    static constexpr int PARAMS = KEYS + VALUES;
    static constexpr int BYTES = PARAMS + 2 * TW * 4;
    static constexpr int PIECES = D / 32;           // 16-byte pieces of a key row
    static constexpr int KEY_MOVES = KEYS / 1024;
    static constexpr int KEY_ROWS = 1024 / (D / 2); // tokens an instruction moves
    static constexpr int MOVES = KEY_MOVES + VALUES / 1024 + 2;
    static constexpr int SLOTS = 2;                 // tiles of a wave that are in LDS or on their way
    // what the place of a piece is its index xor-ed with, for token `row` of 16-token group `grp`: the lanes of a read hold
    // four neighbouring rows of four groups
    static __device__ __forceinline__ int KeyTwist(int row, int grp)
    {
        return D == 64 ? (grp & 1) : (D == 128 ? ((row / 2 + grp) & 3) : ((row & 3) | ((grp & 1) << 2)));
    }
    static constexpr int RING = PA_WAVES * SLOTS * BYTES;
    static constexpr int PITCH = D + 4;
    static constexpr int JOIN_COLS = 4; // columns whose sums the waves join at a time
    static constexpr int JOIN = PA_WAVES * JOIN_COLS * PITCH * 4;
    static constexpr int MASKS = PA_WAVES * 2048; // a tile's mask values for each wave, in the place of the joined sums
    static constexpr int LDS = RING + (JOIN > MASKS ? JOIN : MASKS);
};

// NC: columns that the softmax is computed for, 4, 8 or 16. The matrix instruction gives 16 columns' scores, 16 of a column
// to a lane; with fewer columns most lanes would work on repetitions. The live scores then pass through LDS (the place of
// the tile's keys, which have been read) so that every lane has NC scores of one live column, and the weights come back
// the same way in the matrix instruction's layout.
template <int D, bool BF16, bool MASK, int NC>
__global__ __launch_bounds__(PA_THREADS, D == 256 ? 1 : 2) void PaInt4Kernel(const PaInt4Args a)
{
    using L = TileLayout<D>;
    constexpr int KW = D / 32; // 32-bit words of a token's codes a lane holds = matrix instructions a 16-token block
    constexpr int CT = D / 32; // tiles of 16 channel pairs
    constexpr int PER = WAVE / NC; // lanes that hold a column's scores
    constexpr int WP = D == 64 ? 128 : 144; // bytes between the columns of the weights that pass through LDS
    // what the operands stand for beyond u - 7.5, and the factor of u
    constexpr float K_OFFSET = BF16 ? 23.5f : 7.5f;
    constexpr float K_FACTOR = BF16 ? 1.0f : 16777216.0f;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[]; // a ring of tiles for each wave, then sums or masks
    __shared__ float ldsM[PA_WAVES][HT];
    __shared__ float ldsL[PA_WAVES][HT];
    __shared__ bool ldsFar[HT];

    const int lane = threadIdx.x & (WAVE - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int c = lane & 15;
    const int kg = lane >> 4;
    const int pairs = a.G * a.colTiles;
    const int range = blockIdx.x / pairs;
    const int pair = blockIdx.x % pairs;
    const int g = pair % a.G; // (the column tiles of a head are G workgroups apart: with 8 heads on the same XCD and its L2)
    const int ct = pair / a.G;

    // ---- where the range begins
    int begin = 0, end = 1; // (of a whole sequence: any, it ends after the first)
    int seq = range, before = 0; // the sequence that holds unit `begin`, units of the sequences before it
    if (a.whole == 0) {
        int units = 0;
        for (int b = lane; b < a.batch; b += WAVE) {
            units += UnitsOf(ContextLen(a, b));
        }
        units = WaveSum(units);
        const int live = LiveRanges(a.ranges, units);
        if (range >= live) {
            return;
        }
        begin = RangeBegin(range, units, live);
        end = RangeBegin(range + 1, units, live);
        for (int b0 = 0;; b0 += WAVE) {
            const int own = b0 + lane < a.batch ? UnitsOf(ContextLen(a, b0 + lane)) : 0;
            int upTo = own;
#pragma unroll
            for (int step = 1; step < WAVE; step *= 2) {
                const int other = __shfl_up(upTo, step);
                upTo += lane >= step ? other : 0;
            }
            const uint64_t past = __ballot(before + upTo > begin);
            if (past != 0) { // (begin < units: some sequence holds it)
                const int at = __builtin_ctzll(past);
                seq = b0 + at;
                before += __shfl(upTo - own, at);
                break;
            }
            before += __shfl(upTo, WAVE - 1);
        }
    }
    seq = __builtin_amdgcn_readfirstlane(seq);
    before = __builtin_amdgcn_readfirstlane(before);

    const int columns = a.group * a.tokens;
    const int liveCols = min(HT, columns - ct * HT);
    auto columnOf = [&](int n) { return min(ct * HT + n, columns - 1); }; // (past the last one: the last again, not stored)
    const int col = columnOf(c);             // of the matrix instruction's lane
    const int sl = NC == 16 ? c : lane / PER; // the column whose scores the lane works on, and the first of its NC tokens
    const int tok0 = NC == 16 ? 16 * kg : lane % PER * NC;
    const int sCol = columnOf(sl);
    unsigned char *mine = lds + wave * L::SLOTS * L::BYTES;
    const uint32_t mineAt = LdsAddress(mine);
    float *const sums = reinterpret_cast<float *>(lds + L::RING); // [waves][JOIN_COLS][PITCH]
    unsigned char *const masks = lds + L::RING + wave * 2048;     // [NC][64] (MASK only)
    const uint32_t maskAt = LdsAddress(masks);

    // where a lane reads in a tile that lies in one block: offsets from the tile's first key, value and param
    uint32_t keyAt[L::KEY_MOVES];
#pragma unroll
    for (int i = 0; i < L::KEY_MOVES; ++i) {
        const int token = L::KEY_ROWS * i + lane / L::PIECES;
        keyAt[i] = token * (D / 2) + ((lane % L::PIECES) ^ L::KeyTwist(token % 16, token / 16)) * 16;
    }
    const int vGrp = (lane % 4) ^ (lane / 8 % 4);
    const uint32_t valueAt = lane / 4 * a.blockSize + 16 * vGrp;
    const int64_t headBytes = static_cast<int64_t>(a.blockSize) * (D / 2);
    float down = 0.0f; // by how much the references lie above the scores that they are taken from (bf16 only: see DOWN)

    for (;;) {
        const int len = UniformLen(a, seq);
        const int tBegin = max(max(begin - before, 0) - START, 0);
        const int tEnd = a.whole != 0 ? TilesOf(len) : max(min(end - before, UnitsOf(len)) - START, tBegin);
        // (block ids are read through the scalar cache: not counted with the tiles on their way)
        const auto *table = Scalar(a.tables + static_cast<int64_t>(seq) * a.maxBlocksPerSeq);

        // ---- asks for tile t; returns which of its four 16-token groups lie in blocks that exist, as bits
        auto request = [&](int t, int slot) ATBMI_INLINE -> uint32_t {
            const uint32_t to = mineAt + slot * L::BYTES;
            if (a.tilesPerBlock > 0) { // a block holds whole tiles
                const uint32_t at = a.tilesMagic ? static_cast<uint32_t>((static_cast<uint64_t>(t) * a.tilesMagic) >> 32) : t;
                const int id = table[min(static_cast<int>(at), a.maxBlocksPerSeq - 1)];
                const bool ok = id >= 0 && id < a.numBlocks;
                const int64_t head = static_cast<int64_t>(ok ? id : 0) * a.G + g;
                const int place = (t - static_cast<int>(at) * a.tilesPerBlock) * TW;
                const uint8_t *k = a.kc + head * headBytes + place * (D / 2);
                const uint8_t *v = a.vc + head * headBytes + place;
#pragma unroll
                for (int i = 0; i < L::KEY_MOVES; ++i) {
                    ToLds16(k, keyAt[i], to + i * 1024);
                }
#pragma unroll
                for (int i = 0; i < CT; ++i) {
                    if constexpr (D == 128) {
                        ToLds16Kept(v + i * 16 * a.blockSize, valueAt, to + L::KEYS + i * 1024);
                    } else {
                        ToLds16(v + i * 16 * a.blockSize, valueAt, to + L::KEYS + i * 1024);
                    }
                }
                const int64_t param = head * a.blockSize + place;
                ToLds4(a.kp + param, 4 * lane, to + L::PARAMS);
                ToLds4(a.vp + param, 4 * lane, to + L::PARAMS + TW * 4);
                return ok ? 15u : 0u;
            }
            uint32_t there = 0;
            int64_t first[4]; // of a group: its block's head
            int place[4];     // and its first token within the block
#pragma unroll
            for (int grp = 0; grp < 4; ++grp) {
                const uint32_t x = static_cast<uint32_t>(t * (TW / 16) + grp);
                const uint32_t at16 = a.groupsMagic ? static_cast<uint32_t>((static_cast<uint64_t>(x) * a.groupsMagic) >> 32) : x;
                const int id = table[min(static_cast<int>(at16), a.maxBlocksPerSeq - 1)];
                const bool ok = id >= 0 && id < a.numBlocks;
                there |= ok ? 1u << grp : 0u;
                first[grp] = static_cast<int64_t>(ok ? id : 0) * a.G + g;
                place[grp] = static_cast<int>(x - at16 * a.groupsPerBlock) * 16;
            }
            auto headOf = [&](int grp) ATBMI_INLINE { // (a lane's own choice of four values of the wave)
                const int64_t lo = grp == 0 ? first[0] : int64_t(first[1]), hi = grp == 2 ? first[2] : int64_t(first[3]);
                return grp < 2 ? lo : int64_t(hi);
            };
            auto placeOf = [&](int grp) ATBMI_INLINE {
                const int lo = grp == 0 ? place[0] : int(place[1]), hi = grp == 2 ? place[2] : int(place[3]);
                return grp < 2 ? lo : int(hi);
            };
#pragma unroll
            for (int i = 0; i < L::KEY_MOVES; ++i) {
                const int token = L::KEY_ROWS * i + lane / L::PIECES;
                const int grp = token / 16;
                const int64_t head = L::KEY_ROWS <= 16 ? first[L::KEY_ROWS * i / 16 % 4] : headOf(grp);
                const int in = L::KEY_ROWS <= 16 ? place[L::KEY_ROWS * i / 16 % 4] : placeOf(grp);
                ToLds16(a.kc + head * headBytes + in * (D / 2) + (keyAt[i] - 16 * grp * (D / 2)), to + i * 1024);
            }
            const uint8_t *v = a.vc + headOf(vGrp) * headBytes + placeOf(vGrp) + (valueAt - 16 * vGrp);
#pragma unroll
            for (int i = 0; i < CT; ++i) {
                ToLds16(v + static_cast<int64_t>(16 * i) * a.blockSize, to + L::KEYS + i * 1024);
            }
            const int64_t param = headOf(kg) * a.blockSize + placeOf(kg) + c;
            ToLds4(a.kp + param, to + L::PARAMS);
            ToLds4(a.vp + param, to + L::PARAMS + TW * 4);
            return there;
        };

        // ---- the query columns, permuted as Spread orders the codes, and their sums
        u32x4 q[KW];
        float sumQ = 0.0f;
        const uint16_t *qRow = a.q + ((static_cast<int64_t>(seq) * a.tokens + col / a.group) * a.H + g * a.group + col % a.group) * D + kg * (D / 4);
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
        if constexpr (NC < 16) {
            sumQ = __shfl(sumQ, sl);
        }
        const float midQ = sumQ * a.scale2;
        const float offQ = -K_OFFSET * sumQ * a.scale2;
        const float facQ = K_FACTOR * a.scale2;
        const int seen = len - a.tokens + 1 + sCol / a.group; // positions the lane's column sees
        const int allSee = len - a.tokens + 1;                // positions every column sees
        auto maskRowOf = [&](int column) ATBMI_INLINE {
            return a.mask + seq * a.maskSeqStride + (g * a.group + column % a.group) * a.maskHeadStride +
                   column / a.group * a.maskRowStride;
        };

        f32x4 acc[CT][2]; // [..][0]: even channels of the pairs, [1]: odd ones
        f32x4 ones = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < CT; ++i) {
            acc[i][0] = acc[i][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        float top = -INFINITY; // the reference (log2) of the lane's column
        float total = 0.0f;    // of the lane's own tokens
        float mids = 0.0f;

        // Mask values. Rows on 16-byte boundaries come through LDS, asked for a tile ahead (eight lanes a column); others, and
        // those of a sequence's first tile and of the one in which the mask ends, are read where they are used.
        bool maskThere = false;
        auto maskAhead = [&](int t) ATBMI_INLINE { return a.maskVec != 0 && (t + 1) * TW <= a.maskLen; };
        auto requestMask = [&](int t) ATBMI_INLINE {
#pragma unroll
            for (int i = 0; i < (NC + 7) / 8; ++i) {
                if (NC >= 8 || lane < 8 * NC) {
                    ToLds16(maskRowOf(columnOf(lane / 8 + 8 * i)) + t * TW + lane % 8 * 8, maskAt + i * 1024);
                }
            }
        };

        uint32_t there[L::SLOTS];
#pragma unroll
        for (int i = 0; i < L::SLOTS; ++i) {
            const int t = tBegin + wave + i * PA_WAVES;
            there[i] = t < tEnd ? request(t, i) : 0;
        }

        // (HIDDEN: some token of the tile may be hidden from some column)
        auto tile = [&](int t, int slot, auto hidden) ATBMI_INLINE {
            constexpr bool HIDDEN = MASK || decltype(hidden)::value;
            unsigned char *from = mine + slot * L::BYTES;
            const int first = t * TW + tok0;
            float bias[MASK ? NC : 1];
            if constexpr (MASK) {
                const uint16_t *row = maskRowOf(sCol);
#pragma unroll
                for (int j = 0; j < NC; ++j) {
                    const uint16_t m = maskThere ? *reinterpret_cast<const uint16_t *>(masks + sl * 128 + (tok0 + j) * 2)
                                                 : row[min(first + j, a.maskLen - 1)];
                    bias[j] = first + j < a.maskLen ? Widen<BF16>(m) : -INFINITY;
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                maskThere = t + PA_WAVES < tEnd && maskAhead(t + PA_WAVES);
                if (maskThere) {
                    requestMask(t + PA_WAVES);
                }
            }
            // ---- q . u of 16 tokens a column to a lane: tokens 16 kg + 4 st + e
            f32x4 dot[4];
#pragma unroll
            for (int st = 0; st < 4; ++st) {
                const int row = 4 * st + (c & 3), grp = c >> 2;
                uint32_t kw[KW];
                const unsigned char *kr = from + (16 * grp + row) * (D / 2);
                const int twist = L::KeyTwist(row, grp);
                if constexpr (D == 64) {
                    __builtin_memcpy(kw, __builtin_assume_aligned(kr + ((kg / 2) ^ twist) * 16 + (kg % 2) * 8, 8), 8);
                } else {
#pragma unroll
                    for (int i = 0; i < D / 128; ++i) {
                        __builtin_memcpy(kw + 4 * i, __builtin_assume_aligned(kr + ((D / 128 * kg + i) ^ twist) * 16, 16), 16);
                    }
                }
                dot[st] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < KW; ++i) {
                    dot[st] = Mfma<BF16>(Spread<BF16>(kw[i]), q[i], dot[st]);
                }
            }
            // ---- the lane's scores, in log2 units
            float s[NC];
            if constexpr (NC == 16) {
#pragma unroll
                for (int j = 0; j < NC; ++j) {
                    s[j] = dot[j / 4][j % 4];
                }
            } else {
                WaveSync();
                if (c < NC) {
#pragma unroll
                    for (int st = 0; st < 4; ++st) {
                        *reinterpret_cast<f32x4 *>(from + c * 256 + 64 * kg + 16 * st) = dot[st];
                    }
                }
                WaveSync();
#pragma unroll
                for (int j = 0; j < NC; j += 4) {
                    const f32x4 x = *reinterpret_cast<const f32x4 *>(from + sl * 256 + (tok0 + j) * 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[j + e] = x[e];
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < NC; j += 4) {
                const u32x4 word = *reinterpret_cast<const u32x4 *>(from + L::PARAMS + (tok0 + j) * 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[j + e] = __builtin_fmaf(ScaleOf<BF16>(word[e]), __builtin_fmaf(s[j + e], facQ, offQ), MidOf<BF16>(word[e]) * midQ);
                }
            }
            if constexpr (MASK) {
                // The largest bf16 values leave fp32 when they are turned into log2 units. From LARGE on they grow by half
                // instead (a tile that has any takes that branch): still apart by far more than scores are, and in the same
                // order, and a row of nothing but the lowest value is the mean of its values.
                constexpr float LARGE = 0x1p126f;
                bool large = false;
                if constexpr (BF16) {
#pragma unroll
                    for (int j = 0; j < NC; ++j) {
                        large |= fabsf(bias[j]) > LARGE && bias[j] != -INFINITY;
                    }
                }
                if (BF16 && __ballot(large) != 0) {
#pragma unroll
                    for (int j = 0; j < NC; ++j) {
                        const bool slow = fabsf(bias[j]) > LARGE;
                        const float from = slow ? __builtin_copysignf(LARGE * (LOG2E - 0.5f), bias[j]) : 0.0f;
                        const float v = __builtin_fmaf(bias[j], slow ? 0.5f : LOG2E, s[j] + from);
                        s[j] = bias[j] == -INFINITY ? -INFINITY : v;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < NC; ++j) {
                        const float v = __builtin_fmaf(bias[j], LOG2E, s[j]);
                        s[j] = bias[j] == -INFINITY ? -INFINITY : v;
                    }
                }
            }
            if constexpr (HIDDEN) {
                const uint32_t ok4 = there[slot];
#pragma unroll
                for (int j = 0; j < NC; ++j) {
                    const bool ok = ((ok4 >> (NC == 16 ? kg : (tok0 + j) / 16)) & 1) != 0;
                    s[j] = ok && first + j < seen ? s[j] : -INFINITY;
                }
            }
            // ---- weights
            float most = s[0];
#pragma unroll
            for (int j = 1; j < NC; ++j) {
                most = fmaxf(most, s[j]);
            }
            if (__ballot(most > top + (STEP_UP - down) || (top == -INFINITY && most > -INFINITY)) != 0) {
                float newTop = most;
#pragma unroll
                for (int step = NC == 16 ? 16 : 1; step < (NC == 16 ? WAVE : PER); step *= 2) {
                    newTop = fmaxf(newTop, __shfl_xor(newTop, step));
                }
                newTop = fmaxf(top, newTop + down);
                float keep = top == -INFINITY ? 0.0f : exp2f(top - newTop);
                top = newTop;
                total *= keep;
                mids *= keep;
                if constexpr (NC < 16) {
                    keep = __shfl(keep, c % NC * PER);
                }
                ones *= keep;
#pragma unroll
                for (int i = 0; i < CT; ++i) {
                    acc[i][0] *= keep;
                    acc[i][1] *= keep;
                }
            }
            const float base = top == -INFINITY ? 0.0f : top;
            float pv[NC];
#pragma unroll
            for (int j4 = 0; j4 < NC; j4 += 4) {
                const u32x4 vpw = *reinterpret_cast<const u32x4 *>(from + L::PARAMS + TW * 4 + (tok0 + j4) * 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int j = j4 + e;
                    const float p = __builtin_amdgcn_exp2f(s[j] - base);
                    total += p;
                    // (a hidden token's params may hold anything: 0 times them must be 0)
                    const uint32_t word = HIDDEN && s[j] == -INFINITY ? 0u : vpw[e];
                    pv[j] = p * ScaleOf<BF16>(word);
                    mids = __builtin_fmaf(p, MidOf<BF16>(word), mids);
                }
            }
            // ---- values. The weights (times the value scale) are rounded to bf16, which has fp32's range whatever the
            // scales are: an error of at most 2^-8 each for bf16 models, whose output is rounded as coarsely; for fp16
            // models the remainder is multiplied as well (2^-16 left). Tokens j and j + 2 share a register, as Spread
            // leaves them.
            u32x4 pw[2], pr[2]; // tokens 16 kg + 8 h .. + 7
            uint32_t packed[NC / 2], rest[NC / 2];
#pragma unroll
            for (int e = 0; e < NC / 2; ++e) {
                const int j = 4 * (e / 2) + e % 2;
                packed[e] = PackBf16(pv[j], pv[j + 2]);
                if constexpr (!BF16) {
                    rest[e] = PackBf16(pv[j] - __uint_as_float(packed[e] << 16), pv[j + 2] - __uint_as_float(packed[e] & 0xffff0000u));
                }
            }
            if constexpr (NC == 16) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    pw[e / 4][e % 4] = packed[e];
                    if constexpr (!BF16) {
                        pr[e / 4][e % 4] = rest[e];
                    }
                }
            } else {
                // (rows of WP bytes a column, 16 more than they hold where there is room; the scores have been read)
                WaveSync();
#pragma unroll
                for (int e = 0; e < NC / 2; e += 2) {
                    *reinterpret_cast<u32x2 *>(from + sl * WP + tok0 * 2 + e * 4) = u32x2{packed[e], packed[e + 1]};
                    if constexpr (!BF16) {
                        *reinterpret_cast<u32x2 *>(from + (NC + sl) * WP + tok0 * 2 + e * 4) = u32x2{rest[e], rest[e + 1]};
                    }
                }
                WaveSync();
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    pw[h] = *reinterpret_cast<const u32x4 *>(from + c % NC * WP + 32 * kg + 16 * h);
                    if constexpr (!BF16) {
                        pr[h] = *reinterpret_cast<const u32x4 *>(from + (NC + c % NC) * WP + 32 * kg + 16 * h);
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                constexpr uint32_t ONE = 0x3f803f80u;
                const u32x4 one = {ONE, ONE, ONE, ONE};
                ones = Mfma<true>(one, pw[h], ones);
                if constexpr (!BF16) {
                    ones = Mfma<true>(one, pr[h], ones);
                }
            }
#pragma unroll
            for (int i = 0; i < CT; ++i) {
                const u32x4 vw = *reinterpret_cast<const u32x4 *>(from + L::KEYS + i * 1024 + c * 64 + 16 * (kg ^ (c / 2 % 4)));
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const u32x4 a0 = Spread<true>(vw[2 * h]), a1 = Spread<true>(vw[2 * h + 1]);
                    const u32x4 even = {a0[0], a0[2], a1[0], a1[2]}; // low half, then high half, of tokens 0, 2 and 1, 3
                    const u32x4 odd = {a0[1], a0[3], a1[1], a1[3]};
                    acc[i][0] = Mfma<true>(even, pw[h], acc[i][0]);
                    acc[i][1] = Mfma<true>(odd, pw[h], acc[i][1]);
                    if constexpr (!BF16) {
                        acc[i][0] = Mfma<true>(even, pr[h], acc[i][0]);
                        acc[i][1] = Mfma<true>(odd, pr[h], acc[i][1]);
                    }
                }
            }
        };

        // ---- tiles. A slot is waited for by the number of loads that were asked for behind it (mask values are asked for
        // in front of the tile that is the last behind).
        for (int t = tBegin + wave; t < tEnd; t += L::SLOTS * PA_WAVES) {
#pragma unroll
            for (int i = 0; i < L::SLOTS; ++i) {
                const int now = t + i * PA_WAVES;
                if (now < tEnd) {
                    if (now + (L::SLOTS - 1) * PA_WAVES < tEnd) {
                        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((L::SLOTS - 1) * L::MOVES) : "memory");
                    } else {
                        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                    }
                    if (!MASK && (now + 1) * TW <= allSee && there[i] == 15u) {
                        tile(now, i, std::false_type{});
                    } else {
                        tile(now, i, std::true_type{});
                    }
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // the slot has been read
                    const int later = now + L::SLOTS * PA_WAVES;
                    if (later < tEnd) {
                        there[i] = request(later, i);
                    }
                }
            }
        }

        // ---- join the waves, four columns at a time
        if (tEnd > tBegin) {
            if constexpr (NC == 16) {
                total = QuadSum(total);
                mids = QuadSum(mids);
            } else {
#pragma unroll
                for (int step = 1; step < PER; step *= 2) {
                    total += __shfl_xor(total, step);
                    mids += __shfl_xor(mids, step);
                }
                total = __shfl(total, c % NC * PER);
                mids = __shfl(mids, c % NC * PER);
                top = __shfl(top, c % NC * PER);
            }
            __syncthreads(); // (mask values in the place of the sums, and the maxima of the sequence before, have been read)
            if (kg == 0) {
                ldsM[wave][c] = top;
            }
            __syncthreads();
            float joint = -INFINITY;
#pragma unroll
            for (int w = 0; w < PA_WAVES; ++w) {
                joint = fmaxf(joint, ldsM[w][c]);
            }
            const bool none = top == -INFINITY;
            const float f = none ? 0.0f : exp2f(top - joint);
            if (kg == 0) {
                ldsL[wave][c] = total * f;
            }
            const float rest = mids - 23.5f * ones[0];
            const bool whole = tBegin == 0 && tEnd == TilesOf(len);
            const int64_t part = static_cast<int64_t>(2 * range + (tBegin == 0 ? 1 : 0)) * pairs + pair;
            for (int n0 = 0; n0 < liveCols; n0 += L::JOIN_COLS) {
                if (c / L::JOIN_COLS == n0 / L::JOIN_COLS) {
                    float *to = sums + (wave * L::JOIN_COLS + c % L::JOIN_COLS) * L::PITCH + 8 * kg;
#pragma unroll
                    for (int i = 0; i < CT; ++i) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            to[32 * i + 2 * e] = none ? 0.0f : (acc[i][0][e] + rest) * f;
                            to[32 * i + 2 * e + 1] = none ? 0.0f : (acc[i][1][e] + rest) * f;
                        }
                    }
                }
                __syncthreads();
                const int n = n0 + static_cast<int>(threadIdx.x) / (D / 4);
                if (static_cast<int>(threadIdx.x) < L::JOIN_COLS * (D / 4) && n < liveCols) {
                    const int d = static_cast<int>(threadIdx.x) % (D / 4) * 4;
                    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
                    float l = 0.0f;
#pragma unroll
                    for (int w = 0; w < PA_WAVES; ++w) {
                        o += *reinterpret_cast<const f32x4 *>(sums + (w * L::JOIN_COLS + n - n0) * L::PITCH + d);
                        l += ldsL[w][n];
                    }
                    bool store = true;
                    if constexpr (BF16) {
                        if (down == 0.0f) { // (the D / 4 lanes of a column agree)
                            const uint64_t far = __ballot(!(fabsf(o[0]) < FAR) || !(fabsf(o[1]) < FAR) || !(fabsf(o[2]) < FAR) ||
                                                          !(fabsf(o[3]) < FAR));
                            constexpr uint64_t COLUMN = D == 256 ? ~0ull : (1ull << (D / 4 % 64)) - 1;
                            store = ((far >> (lane & ~(D / 4 - 1))) & COLUMN) == 0;
                            ldsFar[n] = !store;
                        } else {
                            store = ldsFar[n];
                        }
                    }
                    if (!store) {
                    } else if (whole) {
                        const float inv = l > 0.0f ? 1.0f / l : (l == l ? 0.0f : l); // nothing seen: zeros; NaN stays
                        const int cc = ct * HT + n;
                        uint16_t *dst = a.out + ((static_cast<int64_t>(seq) * a.tokens + cc / a.group) * a.H + g * a.group + cc % a.group) * D + d;
                        u32x2 w;
                        w[0] = NarrowPair<BF16>(o[0] * inv, o[1] * inv);
                        w[1] = NarrowPair<BF16>(o[2] * inv, o[3] * inv);
                        *reinterpret_cast<u32x2 *>(dst) = w;
                    } else {
                        *reinterpret_cast<f32x4 *>(a.partO + (part * HT + n) * D + d) = o;
                        if (d == 0) {
                            float m = -INFINITY;
#pragma unroll
                            for (int w = 0; w < PA_WAVES; ++w) {
                                m = fmaxf(m, ldsM[w][n]);
                            }
                            a.partL[part * HT + n] = l;
                            a.partM[part * HT + n] = m;
                        }
                    }
                }
                __syncthreads();
            }
            // (stores are counted with loads: the next sequence's tiles are waited for by the number behind them)
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if constexpr (BF16) {
                if (down == 0.0f && __ballot(lane < liveCols && ldsFar[lane & (HT - 1)]) != 0) {
                    down = DOWN;
                    continue;
                }
            }
        }
        before += UnitsOf(len);
        if (before >= end) {
            return;
        }
        ++seq;
        down = 0.0f;
    }
}

// Joins the parts of a sequence that was cut: out = sum 2^(M_p - M) O_p / sum 2^(M_p - M) L_p. A workgroup takes one
// sequence and one pair. D / 4 lanes hold a column, four channels each, and look at that many parts at a time together for
// the maxima and sums. Waves beyond those that the columns need share out the parts. (One sequence of 32768 tokens, 64
// parts a head: 36 us when each thread walked all parts of its channels.)
template <int D, bool BF16> __global__ __launch_bounds__(MERGE_MOST_THREADS) void PaInt4MergeKernel(const PaInt4Args a)
{
    constexpr int LANES = D / 4;          // lanes a column
    constexpr int COLS = WAVE / LANES;    // columns a wave
    __shared__ f32x4 shared[MERGE_MOST_THREADS];
    const int lane = threadIdx.x & (WAVE - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int pairs = a.G * a.colTiles;
    const int seq = blockIdx.x / pairs;
    const int pair = blockIdx.x % pairs;
    const int g = pair % a.G;
    const int ct = pair / a.G;
    int units = 0, before = 0;
    for (int b = lane; b < a.batch; b += WAVE) {
        const int own = UnitsOf(ContextLen(a, b));
        units += own;
        before += b < seq ? own : 0;
    }
    units = WaveSum(units);
    before = WaveSum(before);
    const int live = LiveRanges(a.ranges, units);
    auto rangeOf = [&](int unit) { // the range r with begin(r) <= unit < begin(r + 1)
        return static_cast<int>(((static_cast<int64_t>(unit) + 1) * live - 1) / units);
    };
    const int r0 = rangeOf(before + START); // (of the sequence's first tile)
    const int parts = rangeOf(before + UnitsOf(ContextLen(a, seq)) - 1) - r0 + 1;
    if (parts == 1) {
        return;
    }
    const int liveCols = min(HT, a.group * a.tokens - ct * HT);
    const int waves = blockDim.x / WAVE;
    const int colWaves = min((liveCols + COLS - 1) / COLS, waves); // waves that the columns are spread over
    const int slices = waves / colWaves;
    const int slice = wave / colWaves;
    const int q = lane % LANES;
    // (the part that begins the sequence is its range's second kind, the others are the first)
    auto rowOf = [&](int p, int n) { return (static_cast<int64_t>(2 * (r0 + p) + (p == 0 ? 1 : 0)) * pairs + pair) * HT + n; };
    for (int n0 = wave % colWaves * COLS; n0 < liveCols; n0 += colWaves * COLS) { // (as often for every slice)
        const int n = min(n0 + lane / LANES, liveCols - 1);
        float top = -INFINITY;
        for (int p = q; p < parts; p += LANES) {
            top = fmaxf(top, a.partM[rowOf(p, n)]);
        }
#pragma unroll
        for (int step = 1; step < LANES; step *= 2) {
            top = fmaxf(top, __shfl_xor(top, step));
        }
        auto weightOf = [&](int p) {
            const float m = a.partM[rowOf(p, n)];
            return m == -INFINITY ? 0.0f : exp2f(m - top);
        };
        float l = 0.0f;
        for (int p = q; p < parts; p += LANES) {
            l += weightOf(p) * a.partL[rowOf(p, n)];
        }
#pragma unroll
        for (int step = 1; step < LANES; step *= 2) {
            l += __shfl_xor(l, step);
        }
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        if (slice < slices) { // (waves that do not make up a whole slice hold nothing)
#pragma unroll 4
            for (int p = slice; p < parts; p += slices) {
                o += weightOf(p) * *reinterpret_cast<const f32x4 *>(a.partO + rowOf(p, n) * D + 4 * q);
            }
        }
        if (slices > 1) {
            shared[threadIdx.x] = o;
            __syncthreads();
            for (int s = 1; s < slices && slice == 0; ++s) {
                o += shared[threadIdx.x + s * colWaves * WAVE];
            }
            __syncthreads();
        }
        if (slice == 0 && n0 + lane / LANES < liveCols) {
            const float inv = l > 0.0f ? 1.0f / l : (l == l ? 0.0f : l);
            const int cc = ct * HT + n;
            uint16_t *dst = a.out + ((static_cast<int64_t>(seq) * a.tokens + cc / a.group) * a.H + g * a.group + cc % a.group) * D + 4 * q;
            u32x2 w;
            w[0] = NarrowPair<BF16>(o[0] * inv, o[1] * inv);
            w[1] = NarrowPair<BF16>(o[2] * inv, o[3] * inv);
            *reinterpret_cast<u32x2 *>(dst) = w;
        }
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
    if ((mostTiles + START) * c->batch > 0x7fffffffLL) {
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
    bool whole = false; // a workgroup takes whole sequences
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
    s.ranges = std::min<int64_t>(s.ranges, std::max<int64_t>(1, ((mostTiles + START) * c->batch + PA_WAVES - 1) / PA_WAVES));
    // Whole sequences to a workgroup need no second kernel and no search for where a range begins, and leave the balance to
    // the order in which workgroups end: taken where no sequence can be long, and up to twice that where there is a
    // workgroup for every CU. (32 query heads over 8 of 128 channels, lengths n / 4 .. n. 1 sequence of 512: 11.1 us cut,
    // 7.7 whole; 1 of 1024: 12.0, 10.9; 64 up to 1024: 25.3, 18.3; 64 up to 2048: 33.1, 27.7; but 1 of 2048: 13.1, 17.9;
    // 4 up to 4096: 15.9, 30.6; 64 up to 8192: 90, 104.)
    s.whole = mostTiles <= WHOLE_TILES || (mostTiles <= 2 * WHOLE_TILES && s.pairs * c->batch >= DeviceComputeUnits());
    if (s.whole) {
        s.ranges = c->batch;
    }
    s.merge = s.ranges > 1 && !s.whole;
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
    // (many ranges a sequence: many parts to join for each)
    const int mergeThreads = shape.ranges > 4 * static_cast<int64_t>(call->batch) ? int4kv::MERGE_MOST_THREADS : 256;
    if (!int4kv::FitsLaunch(grid, int4kv::PA_THREADS) || (shape.merge && !int4kv::FitsLaunch(mergeGrid, mergeThreads))) {
        return Fail(ERR_INVALID_PARAM, "pa_int4: %d sequences with %lld groups of 16 query rows are more than one launch takes",
                    call->batch, (long long)shape.pairs);
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
    a.maskVec = ((reinterpret_cast<uintptr_t>(call->mask) & 15) == 0 &&
                 ((call->maskSeqStride | call->maskHeadStride | call->maskRowStride) & 7) == 0) ? 1 : 0;
    a.H = call->numHeads;
    a.G = call->numKvHeads;
    a.group = call->numHeads / call->numKvHeads;
    a.tokens = call->queryTokens;
    a.colTiles = shape.colTiles;
    a.batch = call->batch;
    a.maxBlocksPerSeq = call->maxBlocksPerSeq;
    a.blockSize = call->blockSize;
    auto magic = [](int32_t d) { return d <= 1 ? 0 : static_cast<uint32_t>(((1ULL << 32) + d - 1) / d); };
    a.tilesPerBlock = call->blockSize % int4kv::TW == 0 ? call->blockSize / int4kv::TW : 0;
    a.tilesMagic = magic(a.tilesPerBlock);
    a.groupsPerBlock = call->blockSize / 16;
    a.groupsMagic = magic(a.groupsPerBlock);
    a.numBlocks = call->numBlocks;
    a.whole = shape.whole ? 1 : 0;
    a.ranges = static_cast<int32_t>(shape.ranges);
    a.scale2 = call->qkScale * int4kv::LOG2E;
    hipStream_t s = static_cast<hipStream_t>(stream);
    int rc = OK;
    int4kv::WithHeadDim(call->headDim, [&](auto d) {
        int4kv::WithFlag(call->dtype == ATBMI_BF16, [&](auto bf16) {
            constexpr int D = decltype(d)::value;
            constexpr bool BF16 = decltype(bf16)::value;
            auto launch = [&](auto mask, auto nc) {
                auto kernel = int4kv::PaInt4Kernel<D, BF16, decltype(mask)::value, decltype(nc)::value>;
                constexpr int LDS = int4kv::TileLayout<D>::LDS;
                rc = ConfigureKernelLds(reinterpret_cast<const void *>(kernel), LDS);
                if (rc == OK) {
                    kernel<<<static_cast<unsigned>(grid), int4kv::PA_THREADS, LDS, s>>>(a);
                }
            };
            int4kv::WithFlag(call->mask != nullptr, [&](auto mask) {
                const int columns = a.group * a.tokens;
                if (columns <= 4) {
                    launch(mask, std::integral_constant<int, 4>{});
                } else if (columns <= 8) {
                    launch(mask, std::integral_constant<int, 8>{});
                } else {
                    launch(mask, std::integral_constant<int, 16>{});
                }
            });
            if (rc != OK) {
                return;
            }
            if (hipError_t e = hipGetLastError(); e != hipSuccess) {
                rc = Fail(ERR_RT_FAIL, "pa_int4: launch failed: %s", hipGetErrorString(e));
            } else if (shape.merge) {
                int4kv::PaInt4MergeKernel<D, BF16><<<static_cast<unsigned>(mergeGrid), mergeThreads, 0, s>>>(a);
            }
        });
    });
    if (rc != OK) {
        return rc;
    }
    ATBMI_HIP_CHECK(hipGetLastError());
    return OK;
}
