// Softmax cross entropy of rows against every row of an embedding table, without keeping the scores.
//
//   z_nv = scale x_n . t_v + b_v,   lse_n = log sum_v exp z_nv,   loss_n = lse_n - z_n,target(n)
//   G_nv = grad_n scale (exp(z_nv - lse_n) - [v = target(n)]),   dx = G t,   dt = G' x
//
// The scores are never stored: the forward pass keeps a running maximum and sum per row while the table goes by, the
// backward pass computes the scores again, once for dx (rows stay, the table goes by) and once for dt (table rows stay,
// x goes by).  The three passes are one kernel: a wave OWNS 32 or 64 rows of one operand, held in registers as the
// B operand of the matrix instruction, and the other operand STREAMS through LDS in tiles that the four waves of the
// block share.  S = stream owner' has the owner's row in the lane and the stream's rows in the registers, so the
// running sums need no exchange between lanes, and exp(S) is, as it lies, the B operand of the second product
// (contracted over the stream's rows, 8 of 16 per half wave); the A operand of that product is the same LDS tile read
// through the transposing LDS load, so that a lane ends up with groups of four columns of its own row.  A tile is laid out in 16-byte chunks whose place is exchanged by the row
// (`swizzle`), which keeps both kinds of read free of bank conflicts.
//
// float32 rows are split into three bfloat16 planes (8 + 8 + 8 bits of the mantissa) and a product of them is the six
// plane products that matter, about 2^-24 of |x||t| off: six bfloat16 instructions take 3/8 of the time of the float32
// ones that they replace.  bfloat16 rows are used as they are; for them the probabilities are rounded to bfloat16 (one
// half step in 2^8, after the 1 at the target has been taken off) on their way into the second product.  Everything
// else, and all sums, are in 32 bits.
//
// Few owners (or a long stream) leave compute units idle, so the stream is cut into `splits` that run side by side and
// leave partial sums in the workspace, which a second kernel joins in a fixed order: no atomics, a call gives the same
// bits every time.
#include <math.h>

#include <type_traits>

#include "dense.h"

namespace recsdk {

typedef short Short4 __attribute__((ext_vector_type(4)));
typedef BF16 Bf16x8 __attribute__((ext_vector_type(8)));
typedef float Float16 __attribute__((ext_vector_type(16)));

constexpr float kMaskedBelow = -1e30f;   // an item_bias at or below this takes the item out
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFloor = -3e38f;         // running maximum before the first item
constexpr float kSlack = 10.0f;          // the running maximum may lag by a factor of 2^10
constexpr int kLossThreads = 256;
constexpr int kLossMaxDim = 256;
constexpr int kLossMaxStride = 1 << 22;   // elements; 128 rows of a tile stay within 32-bit offsets

enum LossPass { kLossForward = 0, kLossDx = 1, kLossDt = 2 };

struct LossArgs {
    const void* own;        // the operand that stays
    const void* stream;     // the operand that goes by
    int64_t ownStride;      // elements between rows
    int64_t streamStride;
    int32_t owners;         // rows
    int32_t streams;
    int32_t dim;
    const int64_t* target;  // [rows of x]
    const float* bias;      // [items] or NULL
    const float* lse;       // backward: [rows of x], +inf where a row takes no gradient
    const float* grad;      // backward: [rows of x]
    float scale;
    int32_t splits;         // pieces of the stream
    int32_t tilesPerSplit;
    float2* norm;           // forward: [split parts][owners] (maximum, sum), base 2
    float* part;            // backward: [split parts][owners][partDim] partial sums, or NULL
    int32_t partDim;        // dim rounded up to whole fours
    void* out;              // dt pass without parts: [owners][dim] in the operands' type
};

__device__ __forceinline__ float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }

// Keeps what is derived from v next to its use: the compiler would move the comparisons' operands out of the loop and
// hold them in registers for a branch that is hardly ever taken.
__device__ __forceinline__ void pin(int& v) { asm volatile("" : "+v"(v)); }

// The row of a 32-row piece that the matrix instruction has as row m: 16 x + 4 a + b -> 16 x + 4 b + a.  Its own inverse.
__device__ __forceinline__ constexpr int tile_row(int m) { return (m & ~15) | ((m & 3) << 2) | ((m >> 2) & 3); }

// v = p0 + p1 + p2 up to 2^-24 |v|
__device__ __forceinline__ void split3(float v, BF16& p0, BF16& p1, BF16& p2)
{
    p0 = (BF16)v;
    const float r = v - (float)p0;
    p1 = (BF16)r;
    p2 = (BF16)(r - (float)p1);
}

// One product of 32 x 16 by 16 x 32 for operands of P planes, the small terms first.
template <int P>
__device__ __forceinline__ Float16 product(const Bf16x8 (&a)[P], const Bf16x8 (&b)[P], Float16 c)
{
    if constexpr (P == 3) {
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[2], b[0], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[2], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[1], b[1], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[1], b[0], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[1], c, 0, 0, 0);
    }
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[0], c, 0, 0, 0);
}

// Eight columns of a row as they come from memory.  `at` is the first of them, `cols` how many the row has from there on
// (none, or whole 16-byte pieces); what is not loaded keeps its value.
template <int P>
struct RowChunk;
template <>
struct RowChunk<1> {
    static constexpr int kBytes = 16;
    Word4 v;
    __device__ __forceinline__ void load(const char* at, int cols)
    {
        if (cols > 0) {
            v = *reinterpret_cast<const Word4*>(at);
        }
    }
    __device__ __forceinline__ void clear() { v = Word4{0, 0, 0, 0}; }
    __device__ __forceinline__ void negate() { v ^= Word4{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u}; }
    __device__ __forceinline__ void planes(Bf16x8 (&p)[1]) const { __builtin_memcpy(&p[0], &v, 16); }
};
template <>
struct RowChunk<3> {
    static constexpr int kBytes = 32;
    Float4 v[2];
    __device__ __forceinline__ void load(const char* at, int cols)
    {
        if (cols > 0) {
            v[0] = *reinterpret_cast<const Float4*>(at);
        }
        if (cols > 4) {
            v[1] = *reinterpret_cast<const Float4*>(at + 16);
        }
    }
    __device__ __forceinline__ void clear() { v[0] = v[1] = Float4{0, 0, 0, 0}; }
    __device__ __forceinline__ void negate()
    {
        v[0] = -v[0];
        v[1] = -v[1];
    }
    __device__ __forceinline__ void planes(Bf16x8 (&p)[3]) const
    {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            BF16 a, b, c;
            split3(v[j / 4][j % 4], a, b, c);
            p[0][j] = a;
            p[1][j] = b;
            p[2][j] = c;
        }
    }
};

// Columns d .. d + 3 of a row, as far as it has them.
template <typename T>
__device__ __forceinline__ void store_columns(T* row, int d, int dim, bool fours, Float4 v)
{
    typedef T T4 __attribute__((ext_vector_type(4)));
    if (fours) {
        if (d < dim) {
            *reinterpret_cast<T4*>(row + d) = T4{from_float<T>(v[0]), from_float<T>(v[1]), from_float<T>(v[2]), from_float<T>(v[3])};
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (d + j < dim) {
                row[d + j] = from_float<T>(v[j]);
            }
        }
    }
}

// P: planes per operand (1 bfloat16, 3 float32); DP: columns rounded up to 32, 64, 128 or 256; RW: rows a wave owns;
// OW: owning waves of the block: 4, or fewer: then 4 / OW waves own the same rows and share out the stream's rows.
template <int P, int DP, int RW, int OW, int PASS>
struct LossTile {
    static constexpr int kColBlocks = RW / 32;
    static constexpr int kSteps = DP / 16;
    static constexpr int kChunks = DP / 8;
    static constexpr int kStreamWaves = 4 / OW;
    // rows of a tile: enough for every thread to move whole chunks, 32 for each wave that shares the stream, and no
    // more than what two buffers of LDS and the registers between memory and LDS hold
    static constexpr int kRows = OW < 4 ? 32 * kStreamWaves : (P == 3 && DP > 32) || (DP == 256 && PASS != kLossForward) ? 32 : 64;
    static constexpr int kLoads = kRows * kChunks / kLossThreads;   // chunks per thread and tile
    static constexpr int kRow = DP + 8;                             // elements from row to row
    static constexpr int kPlane = kRows * kRow;
    static constexpr int kBuffers = P * kPlane * 2 * 2 > 147456 ? 1 : 2;
    static_assert(kLoads >= 1 && kLoads * kLossThreads == kRows * kChunks, "whole chunks per thread");
    static_assert(P * kPlane * 2 * kBuffers <= 147456, "the tiles fit LDS");
};

//
// SHIFT: scores are shifted by a value per item (item_bias, or minus infinity past the end of the table).  A kernel without
// it takes the last, partial tile with it in a loop of its own: one loop with both forms in it made the compiler move the
// accumulators from registers to registers in every round.
template <int P, int DP, int RW, int OW, int PASS, bool SHIFT, int OCC>
__global__ __launch_bounds__(kLossThreads, OCC) void k_softmax_tiles(LossArgs a)
{
    using L = LossTile<P, DP, RW, OW, PASS>;
    constexpr int CB = L::kColBlocks;
    constexpr int KS = L::kSteps;
    constexpr int DB = DP / 32;
    constexpr int TR = L::kRows;
    constexpr int CH = L::kChunks;
    constexpr int NB = L::kBuffers;
    __shared__ __attribute__((aligned(16))) BF16 tile[NB][P * L::kPlane];
    // per stream row, in the order of the matrix rows: forward, dx: bias (base 2); dt: log2 |grad scale| - lse (base 2)
    __shared__ __attribute__((aligned(16))) float auxA[NB][TR];
    constexpr bool kDt = PASS == kLossDt;
    __shared__ __attribute__((aligned(16))) float auxG[kDt ? NB : 1][kDt ? TR : 1];     // dt: |grad scale|
    __shared__ __attribute__((aligned(16))) int32_t auxT[kDt ? NB : 1][kDt ? TR : 1];   // dt: target
    constexpr bool kMasks = SHIFT || kDt;
    __shared__ uint32_t deadBits[2][kMasks ? TR / 32 : 1];                   // a bit per stream row that takes no part
    __shared__ uint32_t minusBits[kDt ? NB : 1][kDt ? TR / 32 : 1];          // dt: a bit per row whose grad * scale is negative

    const int wave = threadIdx.x / kWave;
    const int lane = lane_id();
    const int col = lane & 31;
    const int half = lane >> 5;
    const int split = (int)(blockIdx.x % (unsigned)a.splits);
    const int ownBlock = (int)(blockIdx.x / (unsigned)a.splits);
    const int ownBase = (ownBlock * OW + wave % OW) * RW;
    const int streamWave = wave / OW;
    const int tiles = (a.streams + TR - 1) / TR;
    const int t0 = split * a.tilesPerSplit;
    const int t1 = min(t0 + a.tilesPerSplit, tiles);   // t0 < t1: no split is empty
    // the forward pass bounds scores by the largest product, so there a negative scale goes into the owner's rows
    const bool turned = PASS == kLossForward && a.scale < 0.0f;
    const float c2 = (turned ? -a.scale : a.scale) * kLog2e;
    const bool biased = a.bias != nullptr;
    constexpr int kElement = P == 1 ? 2 : 4;

    // ---- the rows this wave owns ----
    Bf16x8 own[CB][KS][P];
    int32_t ownTarget[CB];   // forward, dx
    float ownShift[CB];      // dx: lse (base 2); dt: bias (base 2)
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
        const int n = ownBase + cb * 32 + col;
        bool live = n < a.owners;
        ownTarget[cb] = -1;
        ownShift[cb] = 0.0f;
        if constexpr (PASS == kLossDx) {
            ownShift[cb] = live ? a.lse[n] * kLog2e : INFINITY;
            live = live && ownShift[cb] != INFINITY;
            ownTarget[cb] = live ? (int32_t)a.target[n] : -1;
        }
        if constexpr (PASS == kLossDt) {
            if (biased) {
                const float b = live ? a.bias[n] : -INFINITY;
                live = b > kMaskedBelow;
                ownShift[cb] = live ? b * kLog2e : -INFINITY;
            }
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            RowChunk<P> r;
            r.clear();   // rows past the end, padding positions and free slots may hold anything
            if (live) {
                const int c = (ks * 2 + half) * 8;
                r.load(static_cast<const char*>(a.own) + (n * a.ownStride * kElement + c * kElement), a.dim - c);
            }
            if (turned) {
                r.negate();
            }
            r.planes(own[cb][ks]);
        }
    }

    // ---- the stream's tiles: memory -> registers (one tile ahead) -> LDS ----
    // A thread moves chunk `chunk` of rows chunkRow, chunkRow + kStep, ...: one 32-bit offset per thread for the whole run
    constexpr int kStep = kLossThreads / CH;
    const int chunk = threadIdx.x % CH;
    const int chunkRow = threadIdx.x / CH;
    const int chunkCols = a.dim - chunk * 8;
    const int64_t strideBytes = a.streamStride * kElement;
    const uint32_t chunkAt = (uint32_t)(chunkRow * strideBytes + chunk * RowChunk<P>::kBytes);
    RowChunk<P> staged[L::kLoads];
#pragma unroll
    for (int q = 0; q < L::kLoads; ++q) {
        staged[q].clear();
    }
    auto fetch = [&](int t) {
        const char* base = static_cast<const char*>(a.stream) + (int64_t)t * TR * strideBytes;
        if ((t + 1) * (int64_t)TR <= a.streams) {
#pragma unroll
            for (int q = 0; q < L::kLoads; ++q) {
                staged[q].load(base + q * kStep * strideBytes + chunkAt, chunkCols);
            }
        } else {   // rows past the end: the last one instead
            const int last = a.streams - 1 - t * TR;
#pragma unroll
            for (int q = 0; q < L::kLoads; ++q) {
                const int r = min(q * kStep + chunkRow, last);
                staged[q].load(base + (int64_t)r * strideBytes + chunk * RowChunk<P>::kBytes, chunkCols);
            }
        }
    };
    // What goes with a stream row: one thread per row, two tiles ahead, so that by the time a tile is placed it is known
    // which of its rows take no part and have to be zero (0 times whatever lies there must be 0).
    // The loads are issued ahead of the compute and looked at behind it (aux_mark).
    struct Aux {
        float a;
        float g;
        int64_t t;
        bool dead;
        bool minus;
    };
    auto aux_load = [&](int t) {
        Aux x = {0.0f, 0.0f, -1, true, false};
        if constexpr (kMasks) {
            const int64_t row = (int64_t)t * TR + threadIdx.x;
            if (threadIdx.x < TR && t < t1 && row < a.streams) {
                x.dead = false;
                if constexpr (kDt) {
                    x.a = a.lse[row];
                    x.g = a.grad[row];
                    x.t = a.target[row];
                } else if (biased) {
                    x.a = a.bias[row];
                }
            }
        }
        return x;
    };
    auto aux_mark = [&](Aux& x, int t) {
        if constexpr (kMasks) {
            if constexpr (kDt) {
                x.dead = x.dead || x.a == INFINITY;   // a NaN stays one
                const float g = x.dead ? 0.0f : x.g * a.scale;
                x.minus = g < 0.0f;
                x.g = fabsf(g);
                x.a = x.dead ? -INFINITY : log2f(x.g) - x.a * kLog2e;
                x.t = x.dead ? -1 : x.t;
            } else {
                x.dead = x.dead || x.a <= kMaskedBelow;
                x.a = x.dead ? -INFINITY : x.a * kLog2e;
            }
            const unsigned long long dead = __ballot(x.dead);
            if (threadIdx.x < TR && (lane & 31) == 0) {
                deadBits[t & 1][threadIdx.x / 32] = (uint32_t)(dead >> (lane & 32));
            }
        }
    };
    auto place = [&](int buf, int t, const Aux& x) {
        if constexpr (kMasks) {
            uint32_t any = 0;
#pragma unroll
            for (int w = 0; w < TR / 32; ++w) {
                any |= deadBits[t & 1][w];
            }
            if (__builtin_amdgcn_readfirstlane(any) != 0) {
#pragma unroll
                for (int q = 0; q < L::kLoads; ++q) {
                    const int r = q * kStep + chunkRow;
                    if ((deadBits[t & 1][r / 32] >> (r % 32)) & 1) {
                        staged[q].clear();
                    }
                }
            }
            const unsigned long long minus = __ballot(x.minus);
            if (threadIdx.x < TR) {
                const int at = (threadIdx.x & ~31) | tile_row(threadIdx.x & 31);
                auxA[buf][at] = x.a;
                if constexpr (kDt) {
                    auxG[buf][at] = x.g;
                    auxT[buf][at] = (int32_t)x.t;
                    if ((lane & 31) == 0) {
                        minusBits[buf][threadIdx.x / 32] = (uint32_t)(minus >> (lane & 32));
                    }
                }
            }
        } else if ((t + 1) * (int64_t)TR > a.streams) {
#pragma unroll
            for (int q = 0; q < L::kLoads; ++q) {
                if (t * TR + q * kStep + chunkRow >= a.streams) {
                    staged[q].clear();
                }
            }
            if (threadIdx.x < TR) {
                auxA[buf][(threadIdx.x & ~31) | tile_row(threadIdx.x & 31)] = t * TR + (int)threadIdx.x < a.streams ? 0.0f : -INFINITY;
            }
        }
#pragma unroll
        for (int q = 0; q < L::kLoads; ++q) {
            Bf16x8 p[P];
            staged[q].planes(p);
#pragma unroll
            for (int k = 0; k < P; ++k) {
                *reinterpret_cast<Bf16x8*>(&tile[buf][k * L::kPlane + (q * kStep + chunkRow) * L::kRow + chunk * 8]) = p[k];
            }
        }
    };

    float top[CB];
    float sum[CB];
    Float16 acc[PASS == kLossForward ? 1 : CB][PASS == kLossForward ? 1 : DB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
        top[cb] = kFloor;
        sum[cb] = 0.0f;
        if constexpr (PASS != kLossForward) {
#pragma unroll
            for (int db = 0; db < DB; ++db) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    acc[cb][db][i] = 0.0f;
                }
            }
        }
    }

    // ---- one 32-row piece of a tile ----
    auto piece = [&](auto shiftedC, int buf, int r0, int rowBase) {
        constexpr bool shifted = decltype(shiftedC)::value;
        const BF16* rowAt = &tile[buf][(r0 + tile_row(col)) * L::kRow + half * 8];
        Float16 s[CB];
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[cb][i] = 0.0f;
            }
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            Bf16x8 x[P];
#pragma unroll
            for (int k = 0; k < P; ++k) {
                x[k] = *reinterpret_cast<const Bf16x8*>(rowAt + k * L::kPlane + ks * 16);
            }
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) {
                s[cb] = product<P>(x, own[cb][ks], s[cb]);
            }
        }
        // register i of a lane holds matrix row 8 (i / 4) + 4 half + i % 4, owner row ownBase + cb * 32 + col
        if constexpr (PASS == kLossForward) {
            float b[16];
            float most = 0.0f;   // largest shift
            if constexpr (shifted) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const Float4 v = *reinterpret_cast<const Float4*>(&auxA[buf][r0 + 8 * q + 4 * half]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        b[4 * q + j] = v[j];
                    }
                }
                most = b[0];
#pragma unroll
                for (int i = 1; i < 16; ++i) {
                    most = fmaxf(most, b[i]);
                }
            }
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) {
                // The maximum follows only when it has fallen behind by 2^kSlack (the sums have room for that), so what is
                // asked of every score is a bound: the largest product (c2 is not negative) plus the largest shift.
                float high = s[cb][0];
#pragma unroll
                for (int i = 1; i < 16; ++i) {
                    high = fmaxf(high, s[cb][i]);
                }
                if (__any(__builtin_fmaf(high, c2, most) > top[cb] + kSlack)) {
                    float now = top[cb];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        now = fmaxf(now, shifted ? __builtin_fmaf(s[cb][i], c2, b[i]) : s[cb][i] * c2);
                    }
                    sum[cb] *= exp2_fast(top[cb] - now);
                    top[cb] = now;
                }
                float add = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    add += exp2_fast(__builtin_fmaf(s[cb][i], c2, shifted ? b[i] - top[cb] : -top[cb]));
                }
                sum[cb] += add;
            }
        } else {
            Bf16x8 g[CB][2][P];
            if constexpr (PASS == kLossDx) {
                float b[16];
                if constexpr (shifted) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const Float4 v = *reinterpret_cast<const Float4*>(&auxA[buf][r0 + 8 * q + 4 * half]);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            b[4 * q + j] = v[j];
                        }
                    }
                }
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) {
                    const float shift = -ownShift[cb];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        s[cb][i] = exp2_fast(__builtin_fmaf(s[cb][i], c2, shifted ? b[i] + shift : shift));
                    }
                    int d = ownTarget[cb] - rowBase;
                    if (__any((unsigned)d < 32u)) {
                        d -= half;   // tile_row of a matrix row with 4 half in it
                        pin(d);
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            s[cb][i] -= d == tile_row(8 * (i / 4) + i % 4) ? 1.0f : 0.0f;
                        }
                    }
                }
            } else {
                // |grad scale| is in the exponent; its sign, and the 1 at the target, are rarely asked for
                float shift[16];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const Float4 v = *reinterpret_cast<const Float4*>(&auxA[buf][r0 + 8 * q + 4 * half]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        shift[4 * q + j] = v[j];
                    }
                }
                const bool hit = __any((unsigned)(auxT[buf][r0 + col] - ownBase) < (unsigned)RW);
                const uint32_t minus = __builtin_amdgcn_readfirstlane(minusBits[buf][r0 / 32]);
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        s[cb][i] = exp2_fast(__builtin_fmaf(s[cb][i], c2, shifted ? shift[i] + ownShift[cb] : shift[i]));
                    }
                    if (hit) {
                        int mine = ownBase + cb * 32 + col;
                        pin(mine);
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int m = r0 + 8 * (i / 4) + 4 * half + i % 4;
                            s[cb][i] -= auxT[buf][m] == mine ? auxG[buf][m] : 0.0f;
                        }
                    }
                    if (minus != 0) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            s[cb][i] = ((minus >> tile_row(8 * (i / 4) + i % 4)) >> half) & 1 ? -s[cb][i] : s[cb][i];
                        }
                    }
                }
            }
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if constexpr (P == 1) {
                        g[cb][i / 8][0][i % 8] = (BF16)s[cb][i];
                    } else {
                        BF16 x, y, z;
                        split3(s[cb][i], x, y, z);
                        g[cb][i / 8][0][i % 8] = x;
                        g[cb][i / 8][1][i % 8] = y;
                        g[cb][i / 8][2][i % 8] = z;
                    }
                }
            }
            // second product: contracted over the piece's rows, in the order in which the registers hold them
            const BF16* columnAt = &tile[buf][(r0 + 4 * ((lane & 15) >> 2) + half) * L::kRow + ((lane >> 4) & 1) * 16 + (lane & 3) * 4];
#pragma unroll
            for (int db = 0; db < DB; ++db) {
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                    Bf16x8 w[P];
#pragma unroll
                    for (int k = 0; k < P; ++k) {
                        Short4 v[2];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const BF16* p = columnAt + k * L::kPlane + (16 * kk + 2 * j) * L::kRow + db * 32;
                            v[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                (__attribute__((address_space(3))) Short4*)(const_cast<BF16*>(p)));
                        }
                        __builtin_memcpy(&w[k], v, 16);
                    }
#pragma unroll
                    for (int cb = 0; cb < CB; ++cb) {
                        acc[cb][db] = product<P>(w, g[cb][kk], acc[cb][db]);
                    }
                }
            }
        }
    };

    Aux next = aux_load(t0);   // of the tile that is placed next
    auto sweep = [&](auto shiftedC, int from, int to) {
#pragma unroll 1
        for (int t = from; t < to; ++t) {
            const int buf = NB == 2 ? (t - t0) & 1 : 0;
            const bool more = t + 1 < t1;
            Aux after = aux_load(t + 2);
            if (more) {
                fetch(t + 1);
            }
            // no condition around the pieces: a wave without rows of its own, or rows past the stream's end, compute zeros
#pragma unroll 1
            for (int k = 0; k < TR / 32 / L::kStreamWaves; ++k) {
                const int r0 = (k * L::kStreamWaves + streamWave) * 32;
                piece(shiftedC, buf, r0, t * TR + r0);
            }
            if (NB == 1) {
                __syncthreads();
            }
            if (more) {
                place(NB == 2 ? buf ^ 1 : 0, t + 1, next);
            }
            aux_mark(after, t + 2);
            next = after;
            __syncthreads();
        }
    };
    if (t0 < t1) {
        Aux second = aux_load(t0 + 1);
        fetch(t0);
        aux_mark(next, t0);
        aux_mark(second, t0 + 1);
        __syncthreads();
        place(0, t0, next);
        next = second;
        __syncthreads();
        if constexpr (SHIFT || kDt) {
            sweep(std::integral_constant<bool, SHIFT>{}, t0, t1);
        } else {
            const int whole = max(t0, min(t1, a.streams / TR));
            sweep(std::false_type{}, t0, whole);
            sweep(std::true_type{}, whole, t1);
        }
    }
    if (ownBase >= a.owners) {
        return;
    }

    const int64_t partRow = (int64_t)(split * L::kStreamWaves + streamWave) * a.owners;
    if constexpr (PASS == kLossForward) {
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
            const float otherTop = __shfl_xor(top[cb], 32, kWave);
            const float otherSum = __shfl_xor(sum[cb], 32, kWave);
            const float now = fmaxf(top[cb], otherTop);
            const float all = sum[cb] * exp2_fast(top[cb] - now) + otherSum * exp2_fast(otherTop - now);
            const int n = ownBase + cb * 32 + col;
            if (half == 0 && n < a.owners) {
                a.norm[partRow + n] = make_float2(now, all);
            }
        }
    } else {
        const bool fours = a.dim % 4 == 0;   // then every group of four columns is whole and aligned
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
            const int n = ownBase + cb * 32 + col;
            if (n >= a.owners) {
                continue;
            }
#pragma unroll
            for (int q = 0; q < DB * 4; ++q) {
                const int d = q * 8 + 4 * half;
                const Float4 v = {acc[cb][q / 4][q % 4 * 4], acc[cb][q / 4][q % 4 * 4 + 1], acc[cb][q / 4][q % 4 * 4 + 2],
                                  acc[cb][q / 4][q % 4 * 4 + 3]};
                if (a.part != nullptr) {
                    store_columns(a.part + (partRow + n) * a.partDim, d, a.partDim, true, v);
                } else if constexpr (P == 1) {
                    store_columns(static_cast<BF16*>(a.out) + (int64_t)n * a.dim, d, a.dim, fours, v);
                } else {
                    store_columns(static_cast<float*>(a.out) + (int64_t)n * a.dim, d, a.dim, fours, v);
                }
            }
        }
    }
}

// Joins the parts of the running sums and takes the target's score off.  TEAM threads per row of x: a wave, or the block
// where there are few rows, each with many parts.
template <typename T, int TEAM>
__global__ __launch_bounds__(kBlock) void k_softmax_loss_join(const float2* __restrict__ norm, int parts, int rows, int items,
                                                              int dim, const T* __restrict__ x, int64_t xStride,
                                                              const T* __restrict__ table, int64_t tableStride,
                                                              const int64_t* __restrict__ target, const float* __restrict__ bias,
                                                              float scale, float* __restrict__ loss, float* __restrict__ lse)
{
    constexpr int kWaves = TEAM / kWave;
    __shared__ float joined[kWaves][2];
    const int n = blockIdx.x * (kBlock / TEAM) + threadIdx.x / TEAM;
    const int lane = threadIdx.x % TEAM;
    if (n >= rows) {
        return;
    }
    const int64_t t = target[n];
    const bool inside = t >= 0 && t < items;
    const float b = inside && bias != nullptr ? bias[t] : 0.0f;
    if (!inside || b <= kMaskedBelow) {
        // no target: no loss; a target that is taken out: infinite; neither gives a gradient
        if (lane == 0) {
            loss[n] = inside ? INFINITY : 0.0f;
            lse[n] = INFINITY;
        }
        return;   // the whole team
    }
    float dot = 0.0f;
    for (int d = lane; d < dim && lane < kWave; d += kWave) {
        dot = __builtin_fmaf((float)x[n * xStride + d], (float)table[t * tableStride + d], dot);
    }
    float top = kFloor;
    float sum = 0.0f;
#pragma unroll 4
    for (int p = lane; p < parts; p += TEAM) {
        const float2 v = norm[(int64_t)p * rows + n];
        const float now = fmaxf(top, v.x);
        sum = sum * exp2_fast(top - now) + v.y * exp2_fast(v.x - now);
        top = now;
    }
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) {
        const float otherTop = __shfl_xor(top, d, kWave);
        const float otherSum = __shfl_xor(sum, d, kWave);
        const float now = fmaxf(top, otherTop);
        sum = sum * exp2_fast(top - now) + otherSum * exp2_fast(otherTop - now);
        top = now;
        dot += __shfl_xor(dot, d, kWave);
    }
    if constexpr (kWaves > 1) {
        if (lane % kWave == 0) {
            joined[lane / kWave][0] = top;
            joined[lane / kWave][1] = sum;
        }
        __syncthreads();
#pragma unroll
        for (int w = 1; w < kWaves; ++w) {
            const float now = fmaxf(top, joined[w][0]);
            sum = sum * exp2_fast(top - now) + joined[w][1] * exp2_fast(joined[w][0] - now);
            top = now;
        }
    }
    if (lane == 0) {
        const float l = __builtin_fmaf(top, kLn2, logf(sum));
        loss[n] = l - __builtin_fmaf(dot, scale, b);
        lse[n] = l;
    }
}

// out = factor(row) * sum of the parts, in the operands' type.  Four columns per thread, 32 threads side by side; the WAYS
// groups of 32 in a block take every WAYS-th part each and are joined in their order, so that few values with many parts
// (few rows against a long table) still have many loads in flight.
template <typename T, int WAYS>
__global__ __launch_bounds__(kBlock) void k_softmax_grad_join(const float* __restrict__ part, int parts, int64_t count, int dim,
                                                              int partDim, const float* __restrict__ lse,
                                                              const float* __restrict__ grad, float scale, T* __restrict__ out)
{
    constexpr int kWide = kBlock / WAYS;
    __shared__ Float4 sums[WAYS > 1 ? WAYS : 1][WAYS > 1 ? kWide : 1];
    const int way = threadIdx.x / kWide;
    const int at = threadIdx.x % kWide;
    const int64_t i = ((int64_t)blockIdx.x * kWide + at) * 4;
    Float4 s = 0.0f;
    if (i < count) {
#pragma unroll 8
        for (int p = way; p < parts; p += WAYS) {
            s += *reinterpret_cast<const Float4*>(part + p * count + i);
        }
    }
    if constexpr (WAYS > 1) {
        sums[way][at] = s;
        __syncthreads();
        if (way != 0) {
            return;
        }
#pragma unroll
        for (int w = 1; w < WAYS; ++w) {
            s += sums[w][at];
        }
    }
    if (i >= count) {
        return;
    }
    const int64_t n = i / partDim;
    float factor = 1.0f;
    if (grad != nullptr) {
        factor = grad[n] * scale;
        if (lse[n] == INFINITY) {   // takes no gradient, whatever grad holds
            s = 0.0f;
            factor = 0.0f;
        }
    }
    store_columns(out + n * dim, (int)(i - n * partDim), dim, dim % 4 == 0, s * factor);
}

// Rows of `dim` elements at any stride -> rows of `padded` elements (whole 16-byte pieces), the rest zero.  32 threads take
// a row's pieces.
template <typename T>
__global__ __launch_bounds__(kBlock) void k_pad_rows(const T* __restrict__ src, int64_t stride, int64_t rows, int dim, int padded,
                                                     T* __restrict__ dst)
{
    constexpr int kPer = 16 / sizeof(T);
    const int64_t r = (int64_t)blockIdx.x * (kBlock / 32) + threadIdx.x / 32;
    if (r >= rows) {
        return;
    }
    for (int c = threadIdx.x % 32 * kPer; c < padded; c += 32 * kPer) {
        Pack<T, kPer> v;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            v.v[e] = c + e < dim ? src[r * stride + c + e] : from_float<T>(0.0f);
        }
        *reinterpret_cast<Pack<T, kPer>*>(dst + r * padded + c) = v;
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------

// Blocks that a compute unit holds at once, by the registers and LDS of the tile kernels.
static int resident_blocks(int planes, int dp, int pass)
{
    if (pass == kLossForward) {
        return planes == 1 ? (dp <= 64 ? 4 : dp == 128 ? 3 : 1) : dp == 32 ? 4 : dp == 64 ? 3 : dp == 128 ? 2 : 1;
    }
    return planes == 1 ? (dp == 32 ? 3 : 2) : dp == 32 ? 4 : dp <= 128 ? 2 : 1;
}
constexpr int kComputeUnits = 256;

// What one pass launches.
struct PassPlan {
    int rowsPerWave;
    int ownWaves;
    int tileRows;
    int64_t blocks;
    int splits;
    int tilesPerSplit;
    int parts;   // splits times the waves that share a block's stream
};

static int padded_dim(int dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// Rows a wave owns where there are many: 64 (every LDS read feeds two matrix instructions) while two waves per SIMD fit the
// registers, else 32; two waves matter more (128 columns, 2048 x 1 M, dx: 1.17 ms with 32 rows, 1.27 with 64 and one wave).
static constexpr int wide_rows(int planes, int dp, int pass)
{
    return planes == 1 && (dp < 128 || pass == kLossForward) ? 64 : 32;
}

static int tile_rows(int planes, int dp, int ownWaves, int pass)
{
    return ownWaves < 4 ? 32 * (4 / ownWaves) : (planes == 3 && dp > 32) || (dp == 256 && pass != kLossForward) ? 32 : 64;
}

static PassPlan plan_pass(int planes, int dim, int64_t owners, int64_t streams, int pass)
{
    const int dp = padded_dim(dim);
    PassPlan p{};
    p.rowsPerWave = wide_rows(planes, dp, pass);
    p.ownWaves = 4;
    if (pass != kLossDt) {
        if (owners <= 128) {
            p.rowsPerWave = 32;
        }
        if (owners <= 32) {
            // all waves would own padding but one: they share the stream instead
            p.ownWaves = planes == 3 && dp == 256 ? 2 : 1;
        }
    }
    p.tileRows = tile_rows(planes, dp, p.ownWaves, pass);
    p.blocks = cdiv(owners, (int64_t)p.rowsPerWave * p.ownWaves);
    const int64_t tiles = cdiv(streams, p.tileRows);
    int64_t splits = (int64_t)kComputeUnits * resident_blocks(planes, dp, pass) / p.blocks;
    splits = splits < 1 ? 1 : splits > tiles ? tiles : splits;
    p.tilesPerSplit = (int)cdiv(tiles, splits);
    p.splits = (int)cdiv(tiles, p.tilesPerSplit);
    p.parts = p.splits * (4 / p.ownWaves);
    return p;
}

struct LossPlan {
    int planes;
    int bytes;           // of an element
    int padded;          // columns of padded copies
    bool padX;           // rows that are no whole 16-byte pieces are copied into padded ones first
    bool padTable;
    PassPlan forward, dx, dt;
    int64_t atX, atTable, atParts;   // offsets into the workspace
    int64_t forwardBytes, backwardBytes;
};

static int64_t round256(int64_t v) { return (v + 255) / 256 * 256; }

static LossPlan plan_loss(int64_t rows, int64_t items, int32_t dim, int32_t dtype, int64_t x_stride, int64_t table_stride)
{
    LossPlan p{};
    p.planes = dtype == RECSDK_DT_F32 ? 3 : 1;
    p.bytes = float_bytes(dtype);
    const int piece = 16 / p.bytes;
    p.padded = (int)(cdiv(dim, piece) * piece);
    p.padX = dim % piece != 0 || x_stride % piece != 0;
    p.padTable = dim % piece != 0 || table_stride % piece != 0;
    p.forward = plan_pass(p.planes, dim, rows, items, kLossForward);
    p.dx = plan_pass(p.planes, dim, rows, items, kLossDx);
    p.dt = plan_pass(p.planes, dim, items, rows, kLossDt);
    p.atX = 0;
    p.atTable = round256(p.atX + (p.padX ? rows * p.padded * p.bytes : 0));
    p.atParts = round256(p.atTable + (p.padTable ? items * p.padded * p.bytes : 0));
    const int64_t norm = (int64_t)p.forward.parts * rows * (int64_t)sizeof(float2);
    const int64_t pitch = cdiv(dim, 4) * 4 * (int64_t)sizeof(float);
    const int64_t dx = (int64_t)p.dx.parts * rows * pitch;
    const int64_t dt = p.dt.parts > 1 ? (int64_t)p.dt.parts * items * pitch : 0;
    p.forwardBytes = round256(p.atParts + norm);
    p.backwardBytes = round256(p.atParts + (dx > dt ? dx : dt));   // the two passes run one after the other
    return p;
}

template <int P, int DP, int RW, int OW, int PASS, bool SHIFT, int OCC>
static int launch_tiles(const LossArgs& a, const PassPlan& p, hipStream_t stream)
{
    const char* name = PASS == kLossForward ? "k_softmax_forward" : PASS == kLossDx ? "k_softmax_dx" : "k_softmax_dt";
    RECSDK_LAUNCH_AS(name, (k_softmax_tiles<P, DP, RW, OW, PASS, SHIFT, OCC>), dim3((unsigned)(p.blocks * p.splits)),
                     dim3(kLossThreads), stream, a);
    return RECSDK_OK;
}

template <int P, int DP, int PASS>
static int launch_width(const LossArgs& a, const PassPlan& p, hipStream_t stream)
{
    constexpr int kOcc = PASS == kLossForward ? (DP == 256 ? 1 : 2) : (P == 3 && DP == 256) ? 1 : 2;
    constexpr int kWide = wide_rows(P, DP, PASS);
    if constexpr (PASS != kLossDt) {
        constexpr int kNarrow = P == 3 && DP == 256 ? 2 : 1;
        if (p.ownWaves == kNarrow) {
            constexpr int kNarrowOcc = DP >= 128 || (P == 3 && DP == 64) ? 1 : 2;
            return launch_tiles<P, DP, 32, kNarrow, PASS, true, kNarrowOcc>(a, p, stream);
        }
        if constexpr (kWide == 64) {
            if (p.rowsPerWave == 32) {
                return launch_tiles<P, DP, 32, 4, PASS, true, 2>(a, p, stream);
            }
        }
    }
    return a.bias != nullptr ? launch_tiles<P, DP, kWide, 4, PASS, true, kOcc>(a, p, stream)
                             : launch_tiles<P, DP, kWide, 4, PASS, false, kOcc>(a, p, stream);
}

template <int PASS>
static int launch_pass(int planes, LossArgs a, const PassPlan& p, hipStream_t stream)
{
    a.splits = p.splits;
    a.tilesPerSplit = p.tilesPerSplit;
    const int dp = padded_dim(a.dim);
    if (planes == 1) {
        switch (dp) {
            case 32:
                return launch_width<1, 32, PASS>(a, p, stream);
            case 64:
                return launch_width<1, 64, PASS>(a, p, stream);
            case 128:
                return launch_width<1, 128, PASS>(a, p, stream);
            default:
                return launch_width<1, 256, PASS>(a, p, stream);
        }
    }
    switch (dp) {
        case 32:
            return launch_width<3, 32, PASS>(a, p, stream);
        case 64:
            return launch_width<3, 64, PASS>(a, p, stream);
        case 128:
            return launch_width<3, 128, PASS>(a, p, stream);
        default:
            return launch_width<3, 256, PASS>(a, p, stream);
    }
}

static int check_loss(const char* name, int64_t rows, int64_t items, int32_t dim, int32_t dtype, int64_t x_stride,
                      int64_t table_stride)
{
    if (dtype != RECSDK_DT_F32 && dtype != RECSDK_DT_BF16) {
        set_error("%s: rows must be fp32 or bf16", name);
        return RECSDK_EINVAL;
    }
    if (dim < 1 || dim > kLossMaxDim) {
        set_error("%s: dim must lie in [1, %d]", name, kLossMaxDim);
        return RECSDK_EINVAL;
    }
    if (rows < 0 || rows >= (int64_t(1) << 30) || items < 1 || items >= (int64_t(1) << 30)) {
        set_error("%s: rows must lie in [0, 2^30) and items in [1, 2^30)", name);
        return RECSDK_EINVAL;
    }
    if (x_stride < dim || table_stride < dim) {
        set_error("%s: rows overlap (stride < dim)", name);
        return RECSDK_EINVAL;
    }
    if (x_stride > kLossMaxStride || table_stride > kLossMaxStride) {
        set_error("%s: rows are more than %d elements apart", name, kLossMaxStride);
        return RECSDK_EINVAL;
    }
    return RECSDK_OK;
}

// The operands as the tile kernels read them: whole 16-byte pieces; others are copied into padded rows.
template <typename T>
static int pad_operand(const void*& p, int64_t& stride, int64_t rows, int dim, int padded, void* to, hipStream_t stream)
{
    const int64_t grid = cdiv(rows, kBlock / 32);
    RECSDK_LAUNCH_AS("k_pad_rows", (k_pad_rows<T>), dim3((unsigned)grid), dim3(kBlock), stream, static_cast<const T*>(p), stride,
                     rows, dim, padded, static_cast<T*>(to));
    p = to;
    stride = padded;
    return RECSDK_OK;
}

template <typename T, int WAYS>
static int launch_grad_join(const float* part, int parts, int64_t rows, int dim, const float* lse, const float* grad,
                            float scale, void* out, hipStream_t stream)
{
    const int partDim = (int)cdiv(dim, 4) * 4;
    const int64_t grid = cdiv(rows * partDim, (int64_t)kBlock / WAYS * 4);
    RECSDK_REQUIRE(grid < (int64_t(1) << 31), RECSDK_EINVAL, "softmax loss: table too large for one launch");
    RECSDK_LAUNCH_AS("k_softmax_grad_join", (k_softmax_grad_join<T, WAYS>), dim3((unsigned)grid), dim3(kBlock), stream, part,
                     parts, rows * partDim, dim, partDim, lse, grad, scale, static_cast<T*>(out));
    return RECSDK_OK;
}

template <typename T>
static int join_grad(const float* part, int parts, int64_t rows, int dim, const float* lse, const float* grad, float scale,
                     void* out, hipStream_t stream)
{
    // eight ways where there are parts for all of them
    return parts >= 8 ? launch_grad_join<T, 8>(part, parts, rows, dim, lse, grad, scale, out, stream)
                      : launch_grad_join<T, 1>(part, parts, rows, dim, lse, grad, scale, out, stream);
}

struct LossOperands {
    const void* x;
    const void* table;
    int64_t xStride;
    int64_t tableStride;
};

template <typename T>
static int pad_operands(const LossPlan& plan, LossOperands& o, int64_t rows, int64_t items, int dim, char* workspace,
                        hipStream_t stream)
{
    if (plan.padX) {
        const int rc = pad_operand<T>(o.x, o.xStride, rows, dim, plan.padded, workspace + plan.atX, stream);
        if (rc != RECSDK_OK) {
            return rc;
        }
    }
    if (plan.padTable) {
        return pad_operand<T>(o.table, o.tableStride, items, dim, plan.padded, workspace + plan.atTable, stream);
    }
    return RECSDK_OK;
}

template <typename T>
static int run_forward(const LossPlan& plan, LossOperands o, int64_t rows, int64_t items, int dim, const int64_t* target,
                       const float* bias, float scale, float* loss, float* lse, char* workspace, hipStream_t stream)
{
    const LossOperands given = o;
    int rc = pad_operands<T>(plan, o, rows, items, dim, workspace, stream);
    if (rc != RECSDK_OK) {
        return rc;
    }
    LossArgs a{};
    a.own = o.x;
    a.ownStride = o.xStride;
    a.stream = o.table;
    a.streamStride = o.tableStride;
    a.owners = (int32_t)rows;
    a.streams = (int32_t)items;
    a.dim = dim;
    a.target = target;
    a.bias = bias;
    a.scale = scale;
    a.norm = reinterpret_cast<float2*>(workspace + plan.atParts);
    rc = launch_pass<kLossForward>(plan.planes, a, plan.forward, stream);
    if (rc != RECSDK_OK) {
        return rc;
    }
    const T* x = static_cast<const T*>(given.x);
    const T* table = static_cast<const T*>(given.table);
    if (plan.forward.parts >= 4 * kWave) {
        RECSDK_LAUNCH_AS("k_softmax_loss_join", (k_softmax_loss_join<T, kBlock>), dim3((unsigned)rows), dim3(kBlock), stream,
                         a.norm, plan.forward.parts, (int)rows, (int)items, dim, x, given.xStride, table, given.tableStride,
                         target, bias, scale, loss, lse);
    } else {
        RECSDK_LAUNCH_AS("k_softmax_loss_join", (k_softmax_loss_join<T, kWave>), dim3((unsigned)cdiv(rows, kBlock / kWave)),
                         dim3(kBlock), stream, a.norm, plan.forward.parts, (int)rows, (int)items, dim, x, given.xStride, table,
                         given.tableStride, target, bias, scale, loss, lse);
    }
    return RECSDK_OK;
}

template <typename T>
static int run_backward(const LossPlan& plan, LossOperands o, int64_t rows, int64_t items, int dim, const int64_t* target,
                        const float* bias, float scale, const float* lse, const float* grad, void* dx, void* dtable,
                        char* workspace, hipStream_t stream)
{
    int rc = pad_operands<T>(plan, o, rows, items, dim, workspace, stream);
    if (rc != RECSDK_OK) {
        return rc;
    }
    LossArgs a{};
    a.dim = dim;
    a.target = target;
    a.bias = bias;
    a.lse = lse;
    a.grad = grad;
    a.scale = scale;
    a.partDim = (int)cdiv(dim, 4) * 4;
    float* part = reinterpret_cast<float*>(workspace + plan.atParts);
    if (dx != nullptr) {
        a.own = o.x;
        a.ownStride = o.xStride;
        a.stream = o.table;
        a.streamStride = o.tableStride;
        a.owners = (int32_t)rows;
        a.streams = (int32_t)items;
        a.part = part;
        rc = launch_pass<kLossDx>(plan.planes, a, plan.dx, stream);
        if (rc != RECSDK_OK) {
            return rc;
        }
        rc = join_grad<T>(part, plan.dx.parts, rows, dim, lse, grad, scale, dx, stream);
        if (rc != RECSDK_OK) {
            return rc;
        }
    }
    if (dtable != nullptr) {
        a.own = o.table;
        a.ownStride = o.tableStride;
        a.stream = o.x;
        a.streamStride = o.xStride;
        a.owners = (int32_t)items;
        a.streams = (int32_t)rows;
        a.part = plan.dt.parts > 1 ? part : nullptr;
        a.out = dtable;
        rc = launch_pass<kLossDt>(plan.planes, a, plan.dt, stream);
        if (rc != RECSDK_OK) {
            return rc;
        }
        if (a.part != nullptr) {
            return join_grad<T>(part, plan.dt.parts, items, dim, nullptr, nullptr, scale, dtable, stream);
        }
    }
    return RECSDK_OK;
}

}  // namespace recsdk

extern "C" int recsdk_softmax_loss_workspace(int64_t rows, int64_t items, int32_t dim, int32_t dtype, int64_t x_stride,
                                             int64_t table_stride, int64_t* h_forward_bytes, int64_t* h_backward_bytes)
{
    using namespace recsdk;
    RECSDK_REQUIRE(h_forward_bytes != nullptr && h_backward_bytes != nullptr, RECSDK_ENULL,
                   "recsdk_softmax_loss_workspace: NULL argument");
    const int rc = check_loss("recsdk_softmax_loss_workspace", rows, items, dim, dtype, x_stride, table_stride);
    if (rc != RECSDK_OK) {
        return rc;
    }
    *h_forward_bytes = 0;
    *h_backward_bytes = 0;
    if (rows > 0) {
        const LossPlan p = plan_loss(rows, items, dim, dtype, x_stride, table_stride);
        *h_forward_bytes = p.forwardBytes;
        *h_backward_bytes = p.backwardBytes;
    }
    return RECSDK_OK;
}

extern "C" int recsdk_softmax_loss_forward(const void* d_x, int64_t rows, int64_t x_stride, const void* d_table, int64_t items,
                                           int64_t table_stride, int32_t dim, int32_t dtype, const int64_t* d_target,
                                           const float* d_item_bias, float scale, float* d_loss, float* d_lse, void* d_workspace,
                                           int64_t workspace_bytes, void* stream)
{
    using namespace recsdk;
    const int rc = check_loss("recsdk_softmax_loss_forward", rows, items, dim, dtype, x_stride, table_stride);
    if (rc != RECSDK_OK) {
        return rc;
    }
    if (rows == 0) {
        return RECSDK_OK;
    }
    RECSDK_REQUIRE(d_x != nullptr && d_table != nullptr && d_target != nullptr && d_loss != nullptr && d_lse != nullptr,
                   RECSDK_ENULL, "recsdk_softmax_loss_forward: NULL argument");
    RECSDK_REQUIRE(aligned16(d_x) && aligned16(d_table) && aligned16(d_workspace), RECSDK_EINVAL,
                   "recsdk_softmax_loss_forward: x, table and workspace must be 16-byte aligned");
    const LossPlan p = plan_loss(rows, items, dim, dtype, x_stride, table_stride);
    RECSDK_REQUIRE(d_workspace != nullptr && workspace_bytes >= p.forwardBytes, RECSDK_ECAPACITY,
                   "recsdk_softmax_loss_forward: the workspace is smaller than recsdk_softmax_loss_workspace says");
    const LossOperands o = {d_x, d_table, x_stride, table_stride};
    char* ws = static_cast<char*>(d_workspace);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == RECSDK_DT_F32
               ? run_forward<float>(p, o, rows, items, dim, d_target, d_item_bias, scale, d_loss, d_lse, ws, s)
               : run_forward<BF16>(p, o, rows, items, dim, d_target, d_item_bias, scale, d_loss, d_lse, ws, s);
}

extern "C" int recsdk_softmax_loss_backward(const float* d_grad_loss, const void* d_x, int64_t rows, int64_t x_stride,
                                            const void* d_table, int64_t items, int64_t table_stride, int32_t dim, int32_t dtype,
                                            const int64_t* d_target, const float* d_item_bias, float scale, const float* d_lse,
                                            void* d_dx, void* d_dtable, void* d_workspace, int64_t workspace_bytes, void* stream)
{
    using namespace recsdk;
    const int rc = check_loss("recsdk_softmax_loss_backward", rows, items, dim, dtype, x_stride, table_stride);
    if (rc != RECSDK_OK) {
        return rc;
    }
    if (d_dx == nullptr && d_dtable == nullptr) {
        return RECSDK_OK;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (rows == 0) {
        if (d_dtable != nullptr) {
            RECSDK_REQUIRE(aligned16(d_dtable), RECSDK_EINVAL, "recsdk_softmax_loss_backward: dtable must be 16-byte aligned");
            return dtype == RECSDK_DT_F32
                       ? join_grad<float>(nullptr, 0, items, dim, nullptr, nullptr, scale, d_dtable, s)
                       : join_grad<BF16>(nullptr, 0, items, dim, nullptr, nullptr, scale, d_dtable, s);
        }
        return RECSDK_OK;
    }
    RECSDK_REQUIRE(d_grad_loss != nullptr && d_x != nullptr && d_table != nullptr && d_target != nullptr && d_lse != nullptr,
                   RECSDK_ENULL, "recsdk_softmax_loss_backward: NULL argument");
    RECSDK_REQUIRE(aligned16(d_x) && aligned16(d_table) && aligned16(d_workspace) && aligned16(d_dx) && aligned16(d_dtable),
                   RECSDK_EINVAL, "recsdk_softmax_loss_backward: x, table, dx, dtable and workspace must be 16-byte aligned");
    const LossPlan p = plan_loss(rows, items, dim, dtype, x_stride, table_stride);
    RECSDK_REQUIRE(d_workspace != nullptr && workspace_bytes >= p.backwardBytes, RECSDK_ECAPACITY,
                   "recsdk_softmax_loss_backward: the workspace is smaller than recsdk_softmax_loss_workspace says");
    const LossOperands o = {d_x, d_table, x_stride, table_stride};
    char* ws = static_cast<char*>(d_workspace);
    return dtype == RECSDK_DT_F32 ? run_backward<float>(p, o, rows, items, dim, d_target, d_item_bias, scale, d_lse, d_grad_loss,
                                                        d_dx, d_dtable, ws, s)
                                  : run_backward<BF16>(p, o, rows, items, dim, d_target, d_item_bias, scale, d_lse, d_grad_loss,
                                                       d_dx, d_dtable, ws, s);
}
