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

// Sixteen values from an address of any alignment, those at or past `valid` zero; the row they end is `row` values long.
// Where the row ends inside them (or in front of them) its last sixteen are read instead and shifted, so that every lane
// makes one load and no branch stands between the loads of a stage.
__device__ __forceinline__ i32x4 Load16Any(const int8_t *p, int valid, int row)
{
    i32x4 v = {0, 0, 0, 0};
    if (row >= 16) { // (the same for all)
        const int missing = min(max(16 - valid, 0), 16);
        unsigned __int128 wide;
        __builtin_memcpy(&wide, p + min(valid - 16, 0), 16);
        wide = missing < 16 ? wide >> (8 * missing) : 0;
        __builtin_memcpy(&v, &wide, 16);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int byte = i < valid ? static_cast<uint8_t>(p[i]) : 0;
            v[i / 4] |= byte << (8 * (i % 4));
        }
    }
    return v;
}

__device__ __forceinline__ float Scaled(const Args &a, int32_t sum, float xs, int n)
{
    return __builtin_fmaf(static_cast<float>(sum), xs * a.wScale[n], a.bias ? a.bias[n] : 0.0f);
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
            v[e] = Rounded(a, Scaled(a, sum[e], xs, n + e));
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
            dst[e] = Rounded(a, Scaled(a, sum[e], xs, n + e));
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

// LDS holds rows of 64 contraction values, 16 of them (1024 bytes) a block that one wave instruction fills: 16-byte piece p
// of row r lies at place p ^ (r / 2 % 4), so that the rows a fragment read touches side by side (lanes c = 0 .. 15 read
// piece kg of rows c) lie in different banks. Lane l of the instruction writes place l % 4 of row l / 4, so it reads piece
// PieceOf(l) of it.
__device__ __forceinline__ int PieceOf(int lane)
{
    return (lane % 4) ^ (lane / 8 % 4);
}
__device__ __forceinline__ int FragmentAt(int c, int kg) // of the fragment's block
{
    return c * 64 + 16 * (kg ^ (c / 2 % 4));
}

// 16 bytes a lane from base + offset to LDS address ldsAt + 16 x lane (base and ldsAt the same for the whole wave).
__device__ __forceinline__ void RowsToLds(const int8_t *base, uint32_t offset, uint32_t ldsAt)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(ldsAt), "v"(offset), "s"(base)
                 : "memory", "m0");
}

// Orders the LDS writes of a wave before its own later reads (and the reads before later writes): a wave's LDS
// instructions execute in order, so only the compiler has to keep them.
__device__ __forceinline__ void WaveSync()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

struct Split {
    int32_t *partial; // [splits][m][n]; null: the tile is the whole contraction and writes the output
    int32_t kPer;     // contraction values a split, a multiple of 128
};

// Which tile a workgroup takes. Workgroups go to the eight XCDs in turn; each XCD gets a contiguous part of the tile list,
// in which four rows of token tiles are walked side by side, so that what its CUs work on at a time shares rows in its L2.
template <int TN, int TM> __device__ __forceinline__ void TileOf(int tilesN, int tilesM, int &n0, int &m0)
{
    constexpr int BAND = 4;
    const int tiles = tilesN * tilesM;
    const int per = tiles / 8, over = tiles % 8;
    const int xcd = blockIdx.x % 8;
    const int t = xcd * per + min(xcd, over) + blockIdx.x / 8;
    const int band = t / (BAND * tilesN);
    const int bandRows = min(BAND, tilesM - band * BAND);
    const int inBand = t - band * BAND * tilesN;
    m0 = (band * BAND + inBand % bandRows) * TM;
    n0 = inBand / bandRows * TN;
}

// The scales (and bias) of a tile travel in registers while the products run and are laid into LDS behind them, so that the
// stores wait for memory once at most: read where they are used they cost 25 us of the 130 that a 256 x 256 x 8192 tile
// takes.
template <int TN, int TM, int THREADS> struct TileScales {
    static constexpr int N = (TN + THREADS - 1) / THREADS, M = (TM + THREADS - 1) / THREADS;
    static constexpr int BYTES = (2 * TN + TM) * 4;
    float w[N], b[N], x[M];
    __device__ __forceinline__ void Load(const Args &a, int n0, int m0)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int n = min(n0 + static_cast<int>(threadIdx.x) + i * THREADS, a.n - 1);
            w[i] = a.wScale[n];
            b[i] = a.bias ? a.bias[n] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < M; ++i) {
            x[i] = a.xScale[min(m0 + static_cast<int>(threadIdx.x) + i * THREADS, a.m - 1)];
        }
    }
    __device__ __forceinline__ void Store(float *lds) const // [TN] channel scales, [TN] bias, [TM] token scales
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int n = static_cast<int>(threadIdx.x) + i * THREADS;
            if (n < TN) {
                lds[n] = w[i];
                lds[TN + n] = b[i];
            }
        }
#pragma unroll
        for (int i = 0; i < M; ++i) {
            const int m = static_cast<int>(threadIdx.x) + i * THREADS;
            if (m < TM) {
                lds[2 * TN + m] = x[i];
            }
        }
    }
};

// Stores a wave's accumulators, channels nAt .. and tokens mAt .. of the tile at (n0, m0). A lane holds four neighbouring
// channels of one token: the wave turns 16 tokens at a time in LDS of its own (16 rows of 16 NI + 4 words) so that its
// stores run along the channels.
template <int TN, int NI, int MI>
__device__ __forceinline__ void StoreTile(const Args &a, const Split &sp, int32_t *turn, const float *scales,
                                          const i32x4 (&acc)[NI][MI], int n0, int m0, int nAt, int mAt, int lane)
{
    typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    constexpr int PITCH = 16 * NI + 4, QUADS = 4 * NI;
    const int c = lane & 15, kg = lane >> 4;
    const bool even = ((reinterpret_cast<uintptr_t>(a.out) | (2 * a.outStride)) & 7) == 0; // quads on 8-byte boundaries
    auto flush = [&](int j) {
#pragma unroll 2
        for (int at = lane; at < 16 * QUADS; at += WAVE) {
            const int mt = mAt + 16 * j + at / QUADS, nt = nAt + at % QUADS * 4;
            const int m = m0 + mt, n = n0 + nt;
            const i32x4 sum = *reinterpret_cast<const i32x4 *>(turn + at / QUADS * PITCH + at % QUADS * 4);
            if (m >= a.m || n >= a.n) {
                continue;
            }
            if (sp.partial) {
                StorePartial(a, sp.partial + (static_cast<int64_t>(blockIdx.y) * a.m + m) * a.n + n, n, sum);
                continue;
            }
            const f32x4 ws = *reinterpret_cast<const f32x4 *>(scales + nt);
            const f32x4 bias = *reinterpret_cast<const f32x4 *>(scales + TN + nt);
            const float xs = scales[2 * TN + mt];
            uint16_t v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = Rounded(a, __builtin_fmaf(static_cast<float>(sum[e]), xs * ws[e], bias[e]));
            }
            uint16_t *dst = a.out + static_cast<int64_t>(m) * a.outStride + n;
            if (even && n + 4 <= a.n) {
                *reinterpret_cast<u32x2 *>(dst) = u32x2{static_cast<uint32_t>(v[0]) | (static_cast<uint32_t>(v[1]) << 16),
                                                        static_cast<uint32_t>(v[2]) | (static_cast<uint32_t>(v[3]) << 16)};
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (n + e < a.n) {
                        dst[e] = v[e];
                    }
                }
            }
        }
    };
#pragma unroll
    for (int j = 0; j < MI; ++j) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            *reinterpret_cast<i32x4 *>(turn + c * PITCH + 16 * i + 4 * kg) = acc[i][j];
        }
        WaveSync();
        flush(j);
        WaveSync();
    }
}

// ---- rows of any alignment: 128 channels x 128 tokens a workgroup of four waves, 64 x 64 each
//
// Stages of 128 values pass through registers into one of two LDS buffers while the stage before is multiplied; what lies
// past the end of the contraction is set to zero on the way. Chunk p of row r (of 128 bytes) lies at place p ^ (r % 8).
constexpr int ANY_TILE = 128;
constexpr int ANY_WAVES = 4;
constexpr int ANY_STAGE = 2 * ANY_TILE * 128;
__global__ __launch_bounds__(ANY_WAVES *WAVE, 2) void LinearAnyKernel(const Args a, const Split sp, int tilesN, int tilesM)
{
    constexpr int NI = 4, MI = 4;
    constexpr int MOVES = ANY_STAGE / (ANY_WAVES * 1024);
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int lane = threadIdx.x & (WAVE - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int c = lane & 15;
    const int kg = lane >> 4;
    const int wn = wave / 2, wm = wave % 2;
    int m0, n0;
    TileOf<ANY_TILE, ANY_TILE>(tilesN, tilesM, n0, m0);
    const int kBegin = blockIdx.y * sp.kPer;
    const int kEnd = min(a.k, kBegin + sp.kPer);
    const int8_t *wBase = a.w + static_cast<int64_t>(n0) * a.wStride;
    const int8_t *xBase = a.x + static_cast<int64_t>(m0) * a.xStride;
    const int chunk16 = 16 * ((lane % 8) ^ (lane / 8));
    uint32_t at[MOVES]; // piece i of a wave: rows 8 (wave + 4 i) .. + 7 of the stage (weights, then tokens)
#pragma unroll
    for (int i = 0; i < MOVES; ++i) {
        const int row = 8 * (wave + ANY_WAVES * i) + lane / 8;
        const bool isW = 8 * ANY_WAVES * i < ANY_TILE;
        const int r = isW ? min(row, a.n - 1 - n0) : min(row - ANY_TILE, a.m - 1 - m0);
        at[i] = static_cast<uint32_t>(r) * static_cast<uint32_t>(isW ? a.wStride : a.xStride) + chunk16;
    }
    i32x4 held[MOVES];
    auto request = [&](int k0) {
        if (k0 + 128 <= kEnd) { // (all loads of a stage on their way together: with the end checked for each they are not)
#pragma unroll
            for (int i = 0; i < MOVES; ++i) {
                __builtin_memcpy(&held[i], (8 * ANY_WAVES * i < ANY_TILE ? wBase : xBase) + at[i] + k0, 16);
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < MOVES; ++i) {
            held[i] = Load16Any((8 * ANY_WAVES * i < ANY_TILE ? wBase : xBase) + at[i] + k0, kEnd - k0 - chunk16, kEnd);
        }
    };
    auto arrive = [&](int buffer) {
#pragma unroll
        for (int i = 0; i < MOVES; ++i) {
            *reinterpret_cast<i32x4 *>(lds + buffer * ANY_STAGE + (wave + ANY_WAVES * i) * 1024 + lane * 16) = held[i];
        }
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
    TileScales<ANY_TILE, ANY_TILE, ANY_WAVES * WAVE> scales;
    scales.Load(a, n0, m0);
    request(kBegin);
    arrive(0);
    int buffer = 0;
    for (int k0 = kBegin; k0 < kEnd; k0 += 128, buffer ^= 1) {
        const bool more = k0 + 128 < kEnd;
        if (more) {
            request(k0 + 128);
        }
        const unsigned char *wt = lds + buffer * ANY_STAGE + (wn * 64 + c) * 128;
        const unsigned char *xt = lds + buffer * ANY_STAGE + (ANY_TILE + wm * 64 + c) * 128;
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
            arrive(buffer ^ 1); // (all waves were done with that buffer when they met last)
        }
    }
    __syncthreads(); // (every wave is done with the stages)
    constexpr int TURN = ANY_WAVES * 16 * (16 * NI + 4) * 4;
    static_assert(TURN + TileScales<ANY_TILE, ANY_TILE, ANY_WAVES * WAVE>::BYTES <= 2 * ANY_STAGE, "this fits the stages");
    scales.Store(reinterpret_cast<float *>(lds + TURN));
    __syncthreads();
    StoreTile<ANY_TILE, NI, MI>(a, sp, reinterpret_cast<int32_t *>(lds) + wave * 16 * (16 * NI + 4),
                                reinterpret_cast<const float *>(lds + TURN), acc, n0, m0, wn * 64, wm * 64, lane);
}

// ---- tiles of aligned rows: TN channels x TM tokens a workgroup of eight waves (WN x WM of them)
//
// Stages of 64 KS values (KS times TN + TM rows of 64 bytes) in a ring of RING, asked for RING - 1 stages ahead and moved
// from memory to LDS without registers, a block of 16 rows with an instruction. A wave alternates between reading a stage's operands into registers (and asking for a later stage) and
// multiplying them, with a barrier after each; the waves of the second half (one on each SIMD, like those of the first) run
// one phase behind, so that on every SIMD one wave multiplies while the other reads. What the phases need of each other,
// counted in barriers (the first half reads stage s in interval 2 s and multiplies it in 2 s + 1, the second half one
// later): a wave waits for its own part of stage s + 1 while it reads stage s, so the stage is whole in interval 2 s + 2;
// stage s + RING - 1 overwrites stage s - 1, which both halves have read by the end of interval 2 s - 1.
constexpr int RING_WAVES = 8;
template <int TN, int TM, int KS, int RING> constexpr int RingLds()
{
    return RING * KS * (TN + TM) * 64;
}
template <int TN, int TM, int WN, int WM, int KS, int RING>
__global__ __launch_bounds__(RING_WAVES *WAVE, 2) void LinearRingKernel(const Args a, const Split sp, int tilesN, int tilesM)
{
    static_assert(WN * WM == RING_WAVES && (TN + TM) % (16 * RING_WAVES) == 0 && TN % 16 == 0, "shape");
    constexpr int NI = TN / WN / 16, MI = TM / WM / 16;
    constexpr int PART = (TN + TM) * 64;
    constexpr int STAGE = KS * PART;
    constexpr int ROWS = (TN + TM) / (16 * RING_WAVES); // instructions a wave moves 64 values with
    constexpr int MOVES = KS * ROWS;
    constexpr int AHEAD = RING - 1;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int lane = threadIdx.x & (WAVE - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int c = lane & 15;
    const int kg = lane >> 4;
    const int wm = wave % WM, wn = wave / WM;
    const bool second = wave >= RING_WAVES / 2;
    int m0, n0;
    TileOf<TN, TM>(tilesN, tilesM, n0, m0);
    const int kBegin = blockIdx.y * sp.kPer;
    const int kEnd = min(a.k, kBegin + sp.kPer);
    const int8_t *wBase = a.w + static_cast<int64_t>(n0) * a.wStride;
    const int8_t *xBase = a.x + static_cast<int64_t>(m0) * a.xStride;
    const int chunk16 = 16 * PieceOf(lane);
    const int8_t *base[ROWS];
    uint32_t at[ROWS]; // instruction i of a wave: rows 16 (wave + 8 i) .. + 15 (weights, then tokens)
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int first = 16 * (wave + RING_WAVES * i);
        const bool isW = first < TN;
        const int row = first + lane / 4;
        const int r = isW ? min(row, a.n - 1 - n0) : min(row - TN, a.m - 1 - m0);
        base[i] = isW ? wBase : xBase;
        at[i] = static_cast<uint32_t>(r) * static_cast<uint32_t>(isW ? a.wStride : a.xStride) + chunk16;
    }
    const int stages = (kEnd - kBegin + 64 * KS - 1) / (64 * KS);
    auto request = [&](int s, int slot) {
        const int k0 = kBegin + 64 * KS * s;
        if (k0 + 64 * KS <= kEnd) {
#pragma unroll
            for (int part = 0; part < KS; ++part) {
#pragma unroll
                for (int i = 0; i < ROWS; ++i) {
                    RowsToLds(base[i] + k0 + 64 * part, at[i],
                              static_cast<uint32_t>(slot * STAGE + part * PART + (wave + RING_WAVES * i) * 1024));
                }
            }
        } else { // the contraction ends inside the stage
#pragma unroll
            for (int part = 0; part < KS; ++part) {
#pragma unroll
                for (int i = 0; i < ROWS; ++i) {
                    *reinterpret_cast<i32x4 *>(lds + slot * STAGE + part * PART + (wave + RING_WAVES * i) * 1024 + lane * 16) =
                        Load16Any(base[i] + k0 + 64 * part + at[i], kEnd - k0 - 64 * part - chunk16, kEnd);
                }
            }
        }
    };
    auto barrier = [] {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    i32x4 acc[NI][MI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
#pragma unroll
        for (int j = 0; j < MI; ++j) {
            acc[i][j] = i32x4{0, 0, 0, 0};
        }
    }
    TileScales<TN, TM, RING_WAVES * WAVE> scales;
    scales.Load(a, n0, m0);
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) {
        if (s < stages) {
            request(s, s);
        }
    }
    if (stages > AHEAD) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((AHEAD - 1) * MOVES) : "memory"); // stage 0
    } else {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    }
    barrier();
    if (second) {
        barrier();
    }
    const unsigned char *wt = lds + wn * (TN / WN) * 64 + FragmentAt(c, kg);
    const unsigned char *xt = lds + (TN + wm * (TM / WM)) * 64 + FragmentAt(c, kg);
    int slot = 0;
    for (int s = 0; s < stages; ++s) {
        // ---- read
        i32x4 wf[KS][NI], xf[KS][MI];
#pragma unroll
        for (int part = 0; part < KS; ++part) {
#pragma unroll
            for (int j = 0; j < MI; ++j) {
                xf[part][j] = *reinterpret_cast<const i32x4 *>(xt + slot * STAGE + part * PART + j * 1024);
            }
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                wf[part][i] = *reinterpret_cast<const i32x4 *>(wt + slot * STAGE + part * PART + i * 1024);
            }
        }
        const int ahead = slot == 0 ? RING - 1 : slot - 1; // slot of stage s + AHEAD
        if (s + AHEAD < stages) {
            request(s + AHEAD, ahead);
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((AHEAD - 1) * MOVES) : "memory"); // stage s + 1
        } else {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        }
        barrier();
        // ---- multiply
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int part = 0; part < KS; ++part) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
#pragma unroll
                for (int j = 0; j < MI; ++j) {
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[part][i], xf[part][j], acc[i][j], 0, 0, 0);
                }
            }
        }
        __builtin_amdgcn_s_setprio(0);
        barrier();
        slot = slot + 1 == RING ? 0 : slot + 1;
    }
    if (!second) {
        barrier();
    }
    constexpr int TURN = RING_WAVES * 16 * (16 * NI + 4) * 4;
    static_assert(TURN + TileScales<TN, TM, RING_WAVES * WAVE>::BYTES <= RING * STAGE, "this fits the ring");
    scales.Store(reinterpret_cast<float *>(lds + TURN));
    __syncthreads();
    StoreTile<TN, NI, MI>(a, sp, reinterpret_cast<int32_t *>(lds) + wave * 16 * (16 * NI + 4),
                          reinterpret_cast<const float *>(lds + TURN), acc, n0, m0, wn * (TN / WN), wm * (TM / WM), lane);
}

// ---- few tokens: the weights stream from memory once
//
// A workgroup of eight waves takes 16 CT channels and all tokens (16 MT of them; fewer are padded by repeating the last).
// The waves take the 128-value chunks of the contraction in turn, each through LDS of its own (RING chunks of rows of 128
// bytes, eight an instruction, piece p of row r at place p ^ (r % 8): whole cache lines from memory, which is what bounds
// this kernel; with 64-byte rows 64 x 6144 x 4096 took 13.8 us instead of 11.1, its weights from HBM), and join their
// integer sums at the end: no barrier in between. What is read of the activations comes from L2, MT / CT times the
// weights' bytes. (Straight into registers in the matrix instruction's layout, 16 neighbouring lanes read 16 bytes of 16
// rows each: 64 tokens by 6144 channels by 4096 took 24 us that way.)
constexpr int SKINNY_WAVES = 8;
template <int MT, int CT> constexpr int SkinnyRing()
{
    return MT + CT <= 3 ? 3 : (MT + CT <= 5 ? 2 : 1);
}
template <int MT, int CT> constexpr int SkinnyLds()
{
    return SKINNY_WAVES * SkinnyRing<MT, CT>() * (MT + CT) * 2048;
}
template <int N> __device__ __forceinline__ void WaitLoads()
{
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

template <int MT, int CT, bool VEC>
__global__ __launch_bounds__(SKINNY_WAVES *WAVE, 1) void LinearSkinnyKernel(const Args a, const Split sp)
{
    constexpr int RING = SkinnyRing<MT, CT>();
    constexpr int MOVES = 2 * (MT + CT); // instructions a chunk
    constexpr int CHUNK = MOVES * 1024;
    static_assert(SKINNY_WAVES * CT * MT * 1024 <= SkinnyLds<MT, CT>(), "the joined sums fit the rings");
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int lane = threadIdx.x & (WAVE - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int c = lane & 15;
    const int kg = lane >> 4;
    const int n0 = blockIdx.x * 16 * CT;
    const int kBegin = blockIdx.y * sp.kPer;
    const int kEnd = min(a.k, kBegin + sp.kPer);
    const int8_t *wBase = a.w + static_cast<int64_t>(n0) * a.wStride;
    const int8_t *xBase = a.x;
    unsigned char *mine = lds + wave * RING * CHUNK;
    const int chunk16 = 16 * ((lane % 8) ^ (lane / 8));
    uint32_t at[MOVES]; // instruction i: rows 8 i .. + 7 (weights, then tokens)
#pragma unroll
    for (int i = 0; i < MOVES; ++i) {
        const bool isW = i < 2 * CT;
        const int row = 8 * (isW ? i : i - 2 * CT) + lane / 8;
        const int r = isW ? min(row, a.n - 1 - n0) : min(row, a.m - 1);
        at[i] = static_cast<uint32_t>(r) * static_cast<uint32_t>(isW ? a.wStride : a.xStride) + chunk16;
    }
    i32x4 acc[CT][MT];
#pragma unroll
    for (int i = 0; i < CT; ++i) {
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            acc[i][j] = i32x4{0, 0, 0, 0};
        }
    }
    const int full = (kEnd - kBegin) / 128;
    // Every workgroup begins at another chunk: rows are often a power of two long, and workgroups that walk them in step
    // would all be at the few memory channels that hold one part of every row.
    const int begin = full > 0 ? static_cast<int>(blockIdx.x * 5u % static_cast<unsigned>(full)) : 0;
    auto chunkAt = [&](int t) { // the wave's t-th chunk
        const int i = begin + wave + t * SKINNY_WAVES; // (below 2 full)
        return kBegin + 128 * (i >= full ? i - full : i);
    };
    auto request = [&](int slot, int k) {
#pragma unroll
        for (int i = 0; i < MOVES; ++i) {
            const int8_t *from = (i < 2 * CT ? wBase : xBase) + k;
            if constexpr (VEC) {
                RowsToLds(from, at[i], static_cast<uint32_t>((wave * RING + slot) * CHUNK + i * 1024));
            } else {
                i32x4 v;
                __builtin_memcpy(&v, from + at[i], 16);
                *reinterpret_cast<i32x4 *>(mine + slot * CHUNK + i * 1024 + lane * 16) = v;
            }
        }
    };
    i32x4 wf[2][CT], xf[2][MT];
    auto fetch = [&](int slot) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const unsigned char *from = mine + slot * CHUNK + c * 128 + 16 * ((4 * half + kg) ^ (c & 7));
#pragma unroll
            for (int i = 0; i < CT; ++i) {
                wf[half][i] = *reinterpret_cast<const i32x4 *>(from + i * 2048);
            }
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                xf[half][j] = *reinterpret_cast<const i32x4 *>(from + (CT + j) * 2048);
            }
        }
    };
    auto multiply = [&]() {
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
    const int count = full > wave ? (full - wave + SKINNY_WAVES - 1) / SKINNY_WAVES : 0;
#pragma unroll
    for (int t = 0; t < RING; ++t) {
        if (t < count) {
            request(t, chunkAt(t));
        }
    }
    int slot = 0;
    for (int t = 0; t < count; ++t) {
        if (VEC) {
            // (the loads of the RING - 1 chunks behind this one may still be on their way)
            if (t + RING <= count) {
                WaitLoads<(RING - 1) * MOVES>();
            } else {
                WaitLoads<0>();
            }
        } else {
            WaveSync();
        }
        fetch(slot);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // in registers: the slot is free
        if (t + RING < count) {
            request(slot, chunkAt(t + RING));
        }
        multiply();
        slot = slot + 1 == RING ? 0 : slot + 1;
    }
    if (kBegin + 128 * full < kEnd && wave == full % SKINNY_WAVES) { // the contraction ends inside a chunk
        const int k = kBegin + 128 * full;
#pragma unroll
        for (int i = 0; i < MOVES; ++i) {
            *reinterpret_cast<i32x4 *>(mine + i * 1024 + lane * 16) =
                Load16Any((i < 2 * CT ? wBase : xBase) + k + at[i], kEnd - k - chunk16, kEnd);
        }
        WaveSync();
        fetch(0);
        multiply();
    }
    __syncthreads();
    i32x4 *joined = reinterpret_cast<i32x4 *>(lds); // [waves][CT MT][64]
#pragma unroll
    for (int i = 0; i < CT; ++i) {
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            joined[(wave * CT * MT + i * MT + j) * WAVE + lane] = acc[i][j];
        }
    }
    __syncthreads();
    for (int f = wave; f < CT * MT; f += SKINNY_WAVES) {
        i32x4 sum = joined[f * WAVE + lane];
#pragma unroll
        for (int v = 1; v < SKINNY_WAVES; ++v) {
            sum += joined[(v * CT * MT + f) * WAVE + lane];
        }
        const int n = n0 + 16 * (f / MT) + 4 * kg;
        const int m = 16 * (f % MT) + c;
        if (m < a.m && n < a.n) {
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

// The cheapest by measured times (us, MI355X). A workgroup of any kind fills a CU, so a kernel costs the rounds that its
// workgroups make on the CUs times what one takes for its part kPer of the contraction:
//   256 x 256   5 + 0.0137 kPer     (32 x 32 tiles of 8192, four rounds: 459; 24 x 8 tiles of 4096, one round: 62)
//   128 x 128   3 + 0.0061 kPer     (48 x 4 tiles of 4096, one round: 28; 48 x 16, three rounds: 78)
//   few tokens  2.5 + rounds kPer x {0.0011, 0.0013, 0.0014} (one channel tile and 16, 32, 64 tokens),
//               {0.0013, 0.0015, 0.0019} (two)   (64 x 6144 x 4096, one round: 11; 64 x 10240 x 8192, two: 33, for
//               which 128 x 128 tiles in three parts, 25, are taken; all with weights from HBM)
// and splitting the contraction 4 us and 0.2 a part for the kernel that joins the parts and their bytes at 4 TB/s (128 x 6144 x 4096:
// 29 whole, 18 in four parts; 512 x 6144 x 4096: 28 whole, 43 in two).
Plan PlanOf(int64_t m, int64_t n, int64_t k)
{
    const int64_t cus = DeviceComputeUnits();
    const int64_t chunks = (k + 127) / 128;
    Plan best;
    double bestCost = 0.0;
    auto offer = [&](Plan p, int64_t groups, double start, double perValue, int64_t mostSplits) {
        for (int64_t s = 1; s <= std::max<int64_t>(1, std::min<int64_t>(mostSplits, 16)); ++s) {
            const int64_t per = (chunks + s - 1) / s;
            const int64_t splits = (chunks + per - 1) / per;
            const double rounds = static_cast<double>((groups * splits + cus - 1) / cus);
            double cost = p.kind == SKINNY ? start + rounds * perValue * 128.0 * per : rounds * (start + perValue * 128.0 * per);
            if (splits > 1) {
                cost += 4.0 + 0.2 * splits + static_cast<double>(splits) * m * n * 8.0 / 4.0e6;
            }
            if (best.kPer == 0 || cost < bestCost) {
                bestCost = cost;
                best = p;
                best.splits = static_cast<int>(splits);
                best.kPer = static_cast<int>(per * 128);
            }
        }
    };
    auto tiles = [&](int64_t size) { return ((n + size - 1) / size) * ((m + size - 1) / size); };
    if (m <= 64) {
        Plan p;
        p.kind = SKINNY;
        p.mt = m <= 16 ? 1 : (m <= 32 ? 2 : 4);
        const double cost[2][3] = {{0.0011, 0.0013, 0.0014}, {0.0013, 0.0015, 0.0019}};
        for (p.ct = 1; p.ct <= 2; ++p.ct) {
            offer(p, (n + 16 * p.ct - 1) / (16 * p.ct), 2.5, cost[p.ct - 1][p.mt == 4 ? 2 : p.mt - 1], chunks / SKINNY_WAVES);
        }
    }
    Plan p;
    p.kind = TILE_128;
    offer(p, tiles(128), 3.0, 0.0061, chunks / 4);
    p.kind = TILE_256;
    offer(p, tiles(256), 5.0, 0.0137, 1);
    best.bytes = best.splits > 1 ? static_cast<uint64_t>(best.splits) * m * n * sizeof(int32_t) : 0;
    return best;
}

int Check(int64_t m, int64_t n, int64_t k)
{
    if (m < 0 || n < 0 || k <= 0 || k > 131071 || m > 0x7fffff00LL || n > 0x7fffff00LL) {
        return Fail(ERR_INVALID_PARAM, "linear_int8: [%lld, %lld] by [%lld, %lld]: the contraction must be 1 .. 131071",
                    (long long)m, (long long)k, (long long)n, (long long)k);
    }
    return OK;
}

int TooLarge(int64_t m, int64_t n)
{
    return Fail(ERR_INVALID_PARAM, "linear_int8: %lld tokens by %lld channels are more than one launch takes", (long long)m,
                (long long)n);
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
                const dim3 grid(static_cast<unsigned>((n + 16 * plan.ct - 1) / (16 * plan.ct)), splits);
                constexpr int MT = decltype(mt)::value, CT = decltype(ct)::value;
                if (!int4kv::FitsLaunch(grid.x, lin8::SKINNY_WAVES * WAVE)) {
                    rc = lin8::TooLarge(m, n);
                    return;
                }
                auto kernel = lin8::LinearSkinnyKernel<MT, CT, VEC>;
                rc = ConfigureKernelLds(reinterpret_cast<const void *>(kernel), lin8::SkinnyLds<MT, CT>());
                if (rc == OK) {
                    kernel<<<grid, lin8::SKINNY_WAVES * WAVE, lin8::SkinnyLds<MT, CT>(), s>>>(a, split);
                }
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
        auto launch = [&](auto kernel, int tn, int tm, int threads, int ldsBytes) {
            const int64_t tilesN = (n + tn - 1) / tn, tilesM = (m + tm - 1) / tm;
            if (!int4kv::FitsLaunch(tilesN * tilesM, threads)) {
                rc = lin8::TooLarge(m, n);
                return;
            }
            rc = ConfigureKernelLds(reinterpret_cast<const void *>(kernel), ldsBytes);
            if (rc == OK) {
                kernel<<<dim3(static_cast<unsigned>(tilesN * tilesM), splits), threads, ldsBytes, s>>>(
                    a, split, static_cast<int>(tilesN), static_cast<int>(tilesM));
            }
        };
        if (!VEC) { // (every tile plan can be served by this one: the split is of the contraction)
            launch(lin8::LinearAnyKernel, lin8::ANY_TILE, lin8::ANY_TILE, lin8::ANY_WAVES * WAVE, 2 * lin8::ANY_STAGE);
        } else if (plan.kind == lin8::TILE_256) {
            launch(lin8::LinearRingKernel<256, 256, 2, 4, 1, 5>, 256, 256, lin8::RING_WAVES * WAVE, lin8::RingLds<256, 256, 1, 5>());
        } else {
            launch(lin8::LinearRingKernel<128, 128, 2, 4, 2, 5>, 128, 128, lin8::RING_WAVES * WAVE, lin8::RingLds<128, 128, 2, 5>());
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
