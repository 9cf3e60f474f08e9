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
// through the transposing LDS load, so that a lane ends up with groups of four columns of its own row.  A tile's rows
// start 16 bytes further apart than they are long, and matrix row m of a piece is tile row `tile_row`(m): the 16 rows of 16
// bytes that one clock of the first product's reads touches, and the 4 rows of 64 bytes of the transposing ones (4 rows
// apart in the tile), then fall on different banks, and every read is one base register and a constant.
//
// bfloat16 rows are used as they are; for them the probabilities are rounded to bfloat16 (one half step in 2^8, after the 1
// at the target has been taken off) on their way into the second product.  Everything else, and all sums, are in 32 bits.
//
// float32 operands of a product are split into planes of 16 bits, and the product into plane products on the matrix
// instructions of those, whose rate is 16 times that of the float32 ones:
//   P = 2  two float16 planes, 11 + 11 bits of the mantissa, three products (high x high, and the two crossed ones): off by
//          about 3 half steps of 2^-22 of |x||t|.  float16 has few exponents, so values are scaled by powers of two first: x
//          and table by their largest finite value (rows that take no part left out; k_abs_max), which leaves what is
//          below 2^-40 of that; exp(S) in the dx pass by 2^15, its largest value being 1; in the dt pass by an exponent
//          of each item's own that follows the item's largest value as the forward pass's maximum does, so that an item
//          with nothing but small probabilities keeps their precision.
//   P = 3  three bfloat16 planes (8 + 8 + 8 bits), six products, all of float32's exponents: for up to 32 rows, where the
//          time goes into reading the table and a pass over it for its largest value would double that.
//
// Few owners (or a long stream) leave compute units idle, so the stream is cut into `splits` that run side by side and
// leave partial sums in the workspace, which a second kernel joins in a fixed order: no atomics, a call gives the same
// bits every time.
#ifndef RECSDK_CSRC_SOFTMAX_TILES_H
#define RECSDK_CSRC_SOFTMAX_TILES_H

#include <math.h>

#include <type_traits>

#include "dense.h"

namespace recsdk {

constexpr float kMaskedBelow = -1e30f;   // an item_bias at or below this takes the item out
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFloor = -3e38f;         // running maximum before the first item
constexpr float kSlack = 10.0f;          // the running maximum may lag by a factor of 2^10
constexpr float kLift = 15.0f;           // P = 2: exponent that probabilities are raised by, or held below
constexpr float kLiftStart = 100.0f;     // P = 2, dt: before an item's first value
constexpr int kAbsMaxParts = 256;        // blocks per operand of k_abs_max
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
    int32_t whole;          // blocks of owners, the first ones, that take the whole stream (dt: and write their result)
    int32_t splits;         // pieces of the stream for the others
    int32_t tilesPerSplit;
    float2* norm;           // forward: [split parts][owners] (maximum, sum), base 2
    float* part;            // backward: [split parts][owners past the whole blocks][partDim] partial sums
    int32_t partDim;        // dim rounded up to whole fours
    void* out;              // dt: [owners][dim] in the operands' type, by the whole blocks
    int32_t tail;           // the table's rows end inside a 16-byte piece (and are no padded copies)
    const float* ownMax;    // P = 2: [kAbsMaxParts] largest values of the operands' rows
    const float* streamMax;
};

#ifdef __HIPCC__
__device__ __forceinline__ float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }
#endif

// ---- shapes, for kernels and host alike ------------------------------------------------------------------------------

// Columns that a kernel works with: the next multiple of 32.
constexpr int loss_width(int dim) { return (dim + 31) / 32 * 32; }

// Rows a wave owns where there are many: 64 (every LDS read feeds two matrix instructions) while two waves per SIMD fit the
// registers, else 32; two waves matter more (128 columns, 2048 x 1 M, dx: 1.17 ms with 32 rows, 1.27 with 64 and one wave).
constexpr int wide_rows(int planes, int dp, int pass) { return planes == 1 && (dp <= 96 || pass == kLossForward) ? 64 : 32; }

// Waves that own rows of their own where there are at most 32 rows: all would own padding but one, so they share the stream
// instead (all four, unless two such tiles do not fit LDS).
constexpr int narrow_waves(int planes, int dp) { return planes == 3 && dp > 64 ? 2 : 1; }

// Rows of a tile: 32 for each wave that shares the stream; else 64, or 32 where two buffers of LDS, or the registers between
// memory and LDS, would be too many.
constexpr int tile_rows(int planes, int dp, int ownWaves, int pass)
{
    if (ownWaves < 4) {
        return 32 * (4 / ownWaves);
    }
    return planes == 1 ? (dp > 160 && pass != kLossForward ? 32 : 64) : planes == 2 ? (dp > 64 ? 32 : 64) : dp > 32 ? 32 : 64;
}

// Few rows: one buffer of LDS where a compute unit then holds two blocks, with twice the loads in flight (1 x 1 M x 64 float32,
// forward: 79 us with two buffers, 56 with one; 8 x 400000 x 160 bfloat16: 35 and 28).
constexpr bool single_buffer(int planes, int dp, int ownWaves, int pass)
{
    return ownWaves < 4 && (planes == 3 || (dp > 128 && (pass == kLossForward || dp <= 160)));
}

// Waves per SIMD that the registers have to leave room for.
constexpr int loss_waves(int planes, int dp, int ownWaves, int pass)
{
    if (ownWaves < 4) {
        return planes == 3 ? (dp > 128 ? 1 : 2) : pass == kLossForward || dp <= 160 ? 2 : 1;
    }
    if (pass == kLossForward) {
        return planes == 1 && dp > 224 ? 1 : 2;
    }
    return planes == 1 ? 2 : planes == 2 ? (dp <= 160 ? 2 : 1) : (dp <= 128 ? 2 : 1);
}

// Blocks that a compute unit holds at once, by the registers and LDS of the kernels.
constexpr int resident_blocks(int planes, int dp, int pass, int rowsPerWave)
{
    if (pass != kLossForward && rowsPerWave < wide_rows(planes, dp, pass)) {
        return dp <= 64 ? 3 : 2;
    }
    if (pass == kLossForward) {
        return planes == 1   ? (dp <= 64 ? 4 : dp <= 128 ? 3 : dp <= 224 ? 2 : 1)
               : planes == 2 ? (dp <= 64 ? 4 : dp <= 128 ? 3 : 2)
                             : (dp <= 32 ? 4 : dp <= 128 ? 2 : 1);
    }
    return planes == 1   ? (dp <= 32 ? 3 : 2)
           : planes == 2 ? (dp <= 32 ? 4 : dp <= 64 ? 3 : dp <= 160 ? 2 : 1)
                         : (dp <= 32 ? 4 : dp <= 128 ? 2 : 1);
}

// Whether a stream row's shift of the scores goes into the first product's accumulators, read from LDS, instead of being added
// to each score afterwards.  bfloat16 with item_bias, forward, 8192 x 200003 x 64: 433 us added, 398 folded (4096 x 50000 x 256:
// 144 and 156).  The backward passes wait for those reads about as long as for the addition (4096 x 50000 x 192, dt: 221 and
// 226; 128 columns: 158 and 168), but where they are short of registers it holds 16 fewer (dt, 96 columns: 256 and 231;
// 224: 296 and 240; 256: 457 and 382; dx, 256: 280 and 233).  float32 adds: its products are scaled by the operands' largest
// values, where a shift might not fit.
constexpr bool folds_shift(int planes, int dp, int pass)
{
    return planes == 1 && (pass == kLossForward ? dp <= 224 : pass == kLossDx ? dp > 224 : dp == 96 || dp > 128);
}

// What one pass launches.
struct PassPlan {
    int rowsPerWave;
    int ownWaves;
    int64_t blocks;
    int64_t whole;   // the first of them take the whole stream; the others are cut into `splits`
    int splits;
    int tilesPerSplit;
    int parts;   // splits times the waves that share a block's stream
};

// Defined in softmax_{bf16,f32}_{forward,backward}.hip: kernels of one type and direction each.
int launch_bf16_forward(const LossArgs& a, const PassPlan& p, hipStream_t stream);
int launch_f32_forward(int planes, const LossArgs& a, const PassPlan& p, hipStream_t stream);
int launch_bf16_backward(int pass, const LossArgs& a, const PassPlan& p, hipStream_t stream);
int launch_f32_backward(int pass, int planes, const LossArgs& a, const PassPlan& p, hipStream_t stream);

#ifdef RECSDK_SOFTMAX_KERNELS

typedef short Short4 __attribute__((ext_vector_type(4)));
typedef int32_t Int4 __attribute__((ext_vector_type(4)));
typedef float Float16 __attribute__((ext_vector_type(16)));

// 16-bit elements of the planes
template <int P>
struct PlaneOf {
    using T = BF16;
};
template <>
struct PlaneOf<2> {
    using T = F16;
};
template <int P>
using Plane = typename PlaneOf<P>::T;
template <int P>
using Frag = Plane<P> __attribute__((ext_vector_type(8)));   // a lane's share of a matrix operand

// Keeps what is derived from v next to its use: the compiler would move the comparisons' operands out of the loop and
// hold them in registers for a branch that is hardly ever taken.
__device__ __forceinline__ void pin(int& v) { asm volatile("" : "+v"(v)); }

// The row of a 32-row piece that the matrix instruction has as row m: 16 x + 4 a + b -> 16 x + 4 b + a.  Its own inverse.
__device__ __forceinline__ constexpr int tile_row(int m) { return (m & ~15) | ((m & 3) << 2) | ((m >> 2) & 3); }

// v as the sum of its planes: 2^-22 |v| off (P = 2, v in float16's range), 2^-24 |v| (P = 3)
template <int P>
__device__ __forceinline__ void split_planes(float v, int j, Frag<P> (&p)[P])
{
#pragma unroll
    for (int k = 0; k < P; ++k) {
        const Plane<P> high = (Plane<P>)v;
        p[k][j] = high;
        if (k + 1 < P) {
            v -= (float)high;
        }
    }
}

__device__ __forceinline__ Float16 multiply(Frag<1> a, Frag<1> b, Float16 c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ Float16 multiply(Frag<2> a, Frag<2> b, Float16 c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// One product of 32 x 16 by 16 x 32 for operands of P planes, the small terms first.
template <int P>
__device__ __forceinline__ Float16 product(const Frag<P> (&a)[P], const Frag<P> (&b)[P], Float16 c)
{
    if constexpr (P == 3) {
        c = multiply(a[2], b[0], c);
        c = multiply(a[0], b[2], c);
        c = multiply(a[1], b[1], c);
    }
    if constexpr (P > 1) {
        c = multiply(a[1], b[0], c);
        c = multiply(a[0], b[1], c);
    }
    return multiply(a[0], b[0], c);
}

// By value: `c ? a[i] : a[j]` of array elements would choose between addresses, and keep the array in memory.
template <typename V>
__device__ __forceinline__ V choose(bool c, V a, V b)
{
    return c ? a : b;
}

// Eight columns of a row as they come from memory.  `at` is the first of them, `cols` how many the row has from there on;
// what is not loaded keeps its value.  Pieces of 16 bytes are loaded whole: where the row ends inside one, `at` lies `back`(cols)
// columns further back, so that the piece ends where the row does, and `settle` moves the columns to their places.  (Rows have
// eight columns at least, so what lies further back is the row's own.)  Rows may start on any element.
template <int P>
struct RowChunk {
    static constexpr int kBytes = 32;
    static constexpr int kPiece = 4;   // columns
    typedef float Piece __attribute__((ext_vector_type(4), aligned(4)));
    Float4 v[2];
    __device__ __forceinline__ void load(const char* at, int cols)
    {
        if (cols > 0) {
            v[0] = *reinterpret_cast<const Piece*>(at);
        }
        if (cols > 4) {
            v[1] = *reinterpret_cast<const Piece*>(at + 16);
        }
    }
    __device__ __forceinline__ void settle(int back)
    {
        const bool two = (back & 2) != 0;
        const bool one = (back & 1) != 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j / 4][j % 4] = choose(two, j + 2 < 8 ? v[(j + 2) / 4 % 2][(j + 2) % 4] : 0.0f, v[j / 4][j % 4]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j / 4][j % 4] = choose(one, j + 1 < 8 ? v[(j + 1) / 4 % 2][(j + 1) % 4] : 0.0f, v[j / 4][j % 4]);
        }
    }
    __device__ __forceinline__ void clear() { v[0] = v[1] = Float4{0, 0, 0, 0}; }
    __device__ __forceinline__ void negate()
    {
        v[0] = -v[0];
        v[1] = -v[1];
    }
    __device__ __forceinline__ void planes(Frag<P> (&p)[P], float scale) const
    {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            split_planes<P>(P == 2 ? v[j / 4][j % 4] * scale : v[j / 4][j % 4], j, p);
        }
    }
};
template <>
struct RowChunk<1> {
    static constexpr int kBytes = 16;
    static constexpr int kPiece = 8;
    typedef uint32_t Piece __attribute__((ext_vector_type(4), aligned(2)));
    Word4 v;
    __device__ __forceinline__ void load(const char* at, int cols)
    {
        if (cols > 0) {
            v = *reinterpret_cast<const Piece*>(at);
        }
    }
    __device__ __forceinline__ void settle(int back)
    {
        const bool four = (back & 4) != 0;
        const bool two = (back & 2) != 0;
        const bool one = (back & 1) != 0;
        v = Word4{choose(four, v[2], v[0]), choose(four, v[3], v[1]), choose(four, 0u, v[2]), choose(four, 0u, v[3])};
        v = Word4{choose(two, v[1], v[0]), choose(two, v[2], v[1]), choose(two, v[3], v[2]), choose(two, 0u, v[3])};
        v = Word4{choose(one, v[0] >> 16 | v[1] << 16, v[0]), choose(one, v[1] >> 16 | v[2] << 16, v[1]),
                  choose(one, v[2] >> 16 | v[3] << 16, v[2]), choose(one, v[3] >> 16, v[3])};
    }
    __device__ __forceinline__ void clear() { v = Word4{0, 0, 0, 0}; }
    __device__ __forceinline__ void negate() { v ^= Word4{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u}; }
    __device__ __forceinline__ void planes(Frag<1> (&p)[1], float) const { __builtin_memcpy(&p[0], &v, 16); }
};

template <int P>
__device__ __forceinline__ int back(int cols)
{
    return cols > 0 && cols < 8 ? -cols & (RowChunk<P>::kPiece - 1) : 0;
}

__device__ __forceinline__ float wave_max(float v)
{
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) {
        v = fmaxf(v, __shfl_xor(v, d, kWave));
    }
    return v;
}

// The power of two that brings values of up to `most` into [2^14, 2^15); 1 for nothing but zeros.
__device__ __forceinline__ float plane_scale(float most)
{
    const int e = max((int)(__float_as_uint(most) >> 23) - 127, -100);
    return most > 0.0f ? __uint_as_float((uint32_t)(127 + 14 - e) << 23) : 1.0f;
}

// P: planes per operand (1 bfloat16, 2 or 3 float32); DP: columns (loss_width); RW: rows a wave owns; OW: owning waves of
// the block: 4, or fewer: then 4 / OW waves own the same rows and share out the stream's rows.
template <int P, int DP, int RW, int OW, int PASS>
struct LossTile {
    static constexpr int kColBlocks = RW / 32;
    static constexpr int kSteps = DP / 16;
    // threads that move a row, 8 columns each
    static constexpr int kRowThreads = DP <= 32 ? 4 : DP <= 64 ? 8 : DP <= 128 ? 16 : 32;
    static constexpr int kStreamWaves = 4 / OW;
    static constexpr int kRows = tile_rows(P, DP, OW, PASS);
    static constexpr int kLoads = kRows * kRowThreads / kLossThreads;   // chunks per thread and tile
    static constexpr int kRow = DP + 8;                                 // elements from row to row
    static constexpr int kPlane = kRows * kRow;
    static constexpr int kBuffers = P * kPlane * 2 * 2 > 147456 || single_buffer(P, DP, OW, PASS) ? 1 : 2;
    static_assert(kLoads >= 1 && kLoads * kLossThreads == kRows * kRowThreads, "whole chunks per thread");
    static_assert(P * kPlane * 2 * kBuffers <= 147456, "the tiles fit LDS");
};

// SHIFT: scores are shifted by a value per item (item_bias, or minus infinity past the end of the table).  A kernel without
// it takes the last, partial tile with it in a loop of its own: one loop with both forms in it made the compiler move the
// accumulators from registers to registers in every round.
template <int P, int DP, int RW, int OW, int PASS, bool SHIFT>
__global__ __launch_bounds__(kLossThreads, loss_waves(P, DP, OW, PASS)) void k_softmax_tiles(LossArgs a)
{
    using L = LossTile<P, DP, RW, OW, PASS>;
    constexpr int CB = L::kColBlocks;
    constexpr int KS = L::kSteps;
    constexpr int DB = DP / 32;
    constexpr int TR = L::kRows;
    constexpr int CH = L::kRowThreads;
    using E = Plane<P>;
    constexpr int NB = L::kBuffers;
    __shared__ __attribute__((aligned(16))) E tile[NB][P * L::kPlane];
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
    const bool cut = (int)blockIdx.x >= a.whole;
    const int split = cut ? (int)((blockIdx.x - a.whole) % (unsigned)a.splits) : 0;
    const int ownBlock = cut ? a.whole + (int)((blockIdx.x - a.whole) / (unsigned)a.splits) : (int)blockIdx.x;
    const int ownBase = (ownBlock * OW + wave % OW) * RW;
    const int streamWave = wave / OW;
    const int tiles = (a.streams + TR - 1) / TR;
    const int t0 = split * a.tilesPerSplit;
    const int t1 = cut ? min(t0 + a.tilesPerSplit, tiles) : tiles;   // t0 < t1: no split is empty
    const bool biased = a.bias != nullptr;
    // the forward pass bounds scores by the largest product, so there a negative scale goes into the owner's rows
    const bool turned = PASS == kLossForward && a.scale < 0.0f;
    // a shift is divided by the scale and goes into the product as what that adds to; without a scale, rows of zeros take its
    // place
    constexpr bool kFold = folds_shift(P, DP, PASS);
    const bool still = kFold && a.scale == 0.0f;
    float c2 = (still ? 1.0f : turned ? -a.scale : a.scale) * kLog2e;
    const float fold = kFold ? 1.0f / c2 : 1.0f;
    const float gone = kFold && c2 < 0.0f ? INFINITY : -INFINITY;   // the shift of a row that takes no part
    constexpr int kElement = P == 1 ? 2 : 4;
    float ownMost = 0.0f;
    float streamMost = 0.0f;
    if constexpr (P == 2) {
        static_assert(kAbsMaxParts == kLossThreads, "one part per thread");
        ownMost = a.ownMax[threadIdx.x];
        streamMost = a.streamMax[threadIdx.x];
    }

    // ---- the rows this wave owns, as they come from memory: looked at once the first tile's loads are under way ----
    int32_t ownTarget[CB];   // dx
    float ownShift[CB];      // dx: lse; dt: bias
    RowChunk<P> ownRaw[CB][KS];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
        const int64_t n = min(ownBase + cb * 32 + col, a.owners - 1);
        ownTarget[cb] = -1;
        ownShift[cb] = 0.0f;
        if constexpr (PASS == kLossDx) {
            ownShift[cb] = a.lse[n];
            ownTarget[cb] = (int32_t)a.target[n];
        }
        if (kDt && SHIFT) {
            ownShift[cb] = a.bias[n];
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            int c = (ks * 2 + half) * 8;
            const int cols = a.dim - c;
            if (kDt && a.tail != 0) {
                c -= back<P>(cols);
            }
            ownRaw[cb][ks].clear();
            ownRaw[cb][ks].load(static_cast<const char*>(a.own) + (n * a.ownStride * kElement + c * kElement), cols);
        }
    }

    // ---- the stream's tiles: memory -> registers (one tile ahead) -> LDS ----
    // A thread moves chunk `chunk` of rows chunkRow, chunkRow + kStep, ...: one 32-bit offset per thread for the whole run
    constexpr int kStep = kLossThreads / CH;
    const int chunk = threadIdx.x % CH;
    const int chunkRow = threadIdx.x / CH;
    const int chunkCols = a.dim - chunk * 8;
    const int64_t strideBytes = a.streamStride * kElement;
    const int chunkBack = !kDt && a.tail != 0 ? back<P>(chunkCols) : 0;
    const int chunkByte = chunk * RowChunk<P>::kBytes - chunkBack * kElement;
    const uint32_t chunkAt = (uint32_t)(chunkRow * strideBytes + chunkByte);
    float ownScale = 1.0f;
    float streamScale = 1.0f;
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
                staged[q].load(base + (int64_t)r * strideBytes + chunkByte, chunkCols);
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
                if constexpr (SHIFT) {
                    x.a = kFold ? x.a * fold : x.a;
                }
                x.t = x.dead ? -1 : x.t;
            } else {
                x.dead = x.dead || x.a <= kMaskedBelow;
                x.a = x.dead ? gone : x.a * (kLog2e * fold);
            }
            const unsigned long long dead = __ballot(x.dead);
            if (threadIdx.x < TR && (lane & 31) == 0) {
                deadBits[t & 1][threadIdx.x / 32] = (uint32_t)(dead >> (lane & 32));
            }
        }
    };
    auto place = [&](int buf, int t, const Aux& x) {
        if (!kDt && a.tail != 0) {
#pragma unroll
            for (int q = 0; q < L::kLoads; ++q) {
                staged[q].settle(chunkBack);
            }
        }
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
                const int at = (threadIdx.x & ~31) | tile_row(threadIdx.x & 31);
                auxA[buf][at] = t * TR + (int)threadIdx.x < a.streams ? 0.0f : gone;
            }
        }
#pragma unroll
        for (int q = 0; q < L::kLoads; ++q) {
            Frag<P> p[P];
            staged[q].planes(p, streamScale);
            if (CH * 8 > DP && chunk * 8 >= DP) {
                continue;   // more threads per row than it has chunks
            }
#pragma unroll
            for (int k = 0; k < P; ++k) {
                *reinterpret_cast<Frag<P>*>(&tile[buf][k * L::kPlane + (q * kStep + chunkRow) * L::kRow + chunk * 8]) = p[k];
            }
        }
    };

    // ---- the first tile's loads, then the scales and the owners' planes ----
    Aux next = aux_load(t0);   // of the tile that is placed next
    Aux second = aux_load(t0 + 1);
    fetch(t0);
    if constexpr (P == 2) {
        float* largest = &auxA[0][0];   // free until the first tile is placed
        const float o = wave_max(ownMost);
        const float s = wave_max(streamMost);
        if (lane == 0) {
            largest[wave] = o;
            largest[4 + wave] = s;
        }
        __syncthreads();
        ownScale = plane_scale(fmaxf(fmaxf(largest[0], largest[1]), fmaxf(largest[2], largest[3])));
        streamScale = plane_scale(fmaxf(fmaxf(largest[4], largest[5]), fmaxf(largest[6], largest[7])));
        __syncthreads();
        c2 = c2 / ownScale / streamScale;
    }
    Frag<P> own[CB][KS][P];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
        bool live = ownBase + cb * 32 + col < a.owners;
        if constexpr (PASS == kLossDx) {
            live = live && ownShift[cb] != INFINITY;
            ownShift[cb] = live ? ownShift[cb] * kLog2e : INFINITY;
            ownTarget[cb] = live ? ownTarget[cb] : -1;
        }
        if (kDt && SHIFT) {
            live = live && ownShift[cb] > kMaskedBelow;
            ownShift[cb] = live ? ownShift[cb] * kLog2e : -INFINITY;
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            if (kDt && a.tail != 0) {
                ownRaw[cb][ks].settle(back<P>(a.dim - (ks * 2 + half) * 8));
            }
            if (!live || still) {
                ownRaw[cb][ks].clear();   // rows past the end, padding positions and free slots may hold anything
            }
            if (turned) {
                ownRaw[cb][ks].negate();
            }
            ownRaw[cb][ks].planes(own[cb][ks], ownScale);
        }
    }

    float top[CB];
    float sum[CB];
    float lift[CB];   // dt, P = 2: exponent that the item's values are raised by
    Float16 acc[PASS == kLossForward ? 1 : CB][PASS == kLossForward ? 1 : DB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
        top[cb] = kFloor;
        sum[cb] = 0.0f;
        lift[cb] = P == 2 && kDt ? kLiftStart : 0.0f;
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

    // ---- one 32-row piece of a tile: its scores, and what becomes of them ----
    auto shifts = [&](float (&b)[16], int buf, int row0) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const Float4 v = *reinterpret_cast<const Float4*>(&auxA[buf][row0 + 8 * q + 4 * half]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                b[4 * q + j] = v[j];
            }
        }
    };
    auto score = [&](auto shiftedC, Float16 (&s)[CB], int buf, int r0) {
        constexpr bool shifted = decltype(shiftedC)::value;
        const E* rowAt = &tile[buf][(r0 + tile_row(col)) * L::kRow + half * 8];
        constexpr bool folded = shifted && kFold;
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
            float b[16];
            if constexpr (folded) {
                int row0 = r0;
                pin(row0);   // loads of its own for each: copies would take an instruction per score
                shifts(b, buf, row0);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[cb][i] = folded ? b[i] : 0.0f;
            }
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            Frag<P> x[P];
#pragma unroll
            for (int k = 0; k < P; ++k) {
                x[k] = *reinterpret_cast<const Frag<P>*>(rowAt + k * L::kPlane + ks * 16);
            }
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) {
                s[cb] = product<P>(x, own[cb][ks], s[cb]);
            }
        }
    };
    auto use = [&](auto shiftedC, Float16 (&s)[CB], int buf, int r0, int rowBase) {
        constexpr bool shifted = decltype(shiftedC)::value;
        constexpr bool folded = shifted && kFold;
        // register i of a lane holds matrix row 8 (i / 4) + 4 half + i % 4, owner row ownBase + cb * 32 + col
        if constexpr (PASS == kLossForward) {
            float b[16];
            float most = 0.0f;   // largest shift
            constexpr bool add = shifted && !folded;
            if constexpr (add) {
                shifts(b, buf, r0);
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
                        now = fmaxf(now, add ? __builtin_fmaf(s[cb][i], c2, b[i]) : s[cb][i] * c2);
                    }
                    sum[cb] *= exp2_fast(top[cb] - now);
                    top[cb] = now;
                }
                float more = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    more += exp2_fast(__builtin_fmaf(s[cb][i], c2, add ? b[i] - top[cb] : -top[cb]));
                }
                sum[cb] += more;
            }
        } else {
            Frag<P> g[CB][2][P];
            bool hit = false;   // the piece holds a target of the wave's rows
            if constexpr (PASS == kLossDx) {
                float b[16];
                constexpr bool add = shifted && !folded;
                if constexpr (add) {
                    shifts(b, buf, r0);
                }
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) {
                    const float shift = (P == 2 ? kLift : 0.0f) - ownShift[cb];
                    constexpr float kOne = P == 2 ? 32768.0f : 1.0f;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        s[cb][i] = exp2_fast(__builtin_fmaf(s[cb][i], c2, add ? b[i] + shift : shift));
                    }
                    int d = ownTarget[cb] - rowBase;
                    if (__any((unsigned)d < 32u)) {
                        hit = true;
                        d -= half;   // tile_row of a matrix row with 4 half in it
                        pin(d);
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            s[cb][i] -= d == tile_row(8 * (i / 4) + i % 4) ? kOne : 0.0f;
                        }
                    }
                }
            } else {
                // |grad scale| is in the exponent; its sign, and the 1 at the target, are rarely asked for
                float shift[16];
                if constexpr (!folded) {
                    shifts(shift, buf, r0);
                }
                hit = __any((unsigned)(auxT[buf][r0 + col] - ownBase) < (unsigned)RW);
                // four rows' targets and |grad scale|, all loaded: a load of what a comparison asks for would wait for it
                struct Hits {
                    Int4 t;
                    Float4 g;
                };
                auto hits = [&](int row) {
                    return Hits{*reinterpret_cast<const Int4*>(&auxT[buf][r0 + row + 4 * half]),
                                *reinterpret_cast<const Float4*>(&auxG[buf][r0 + row + 4 * half])};
                };
                const uint32_t minus = __builtin_amdgcn_readfirstlane(minusBits[buf][r0 / 32]);
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) {
                    float high = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        if constexpr (folded) {
                            s[cb][i] = __builtin_fmaf(s[cb][i], c2, ownShift[cb]);
                        } else {
                            s[cb][i] = __builtin_fmaf(s[cb][i], c2,
                                                      shifted || P == 2 ? shift[i] + (ownShift[cb] + lift[cb]) : shift[i]);
                        }
                        high = fmaxf(high, s[cb][i]);
                    }
                    if constexpr (P == 2) {
                        if (hit) {   // the 1 at the target is the largest there is
                            int mine = ownBase + cb * 32 + col;
                            pin(mine);
                            float largest = 0.0f;
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                const Hits h = hits(8 * q);
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    largest = fmaxf(largest, h.t[j] == mine ? h.g[j] : 0.0f);
                                }
                            }
                            high = fmaxf(high, log2f(largest) + lift[cb]);
                        }
                        // Follows the item's largest value down, half of float16's reach at a time (2 bits at a time cost 4 %
                        // of the pass), but not below a target's, which is the largest but for another row's |grad|: what is
                        // left out beside the largest is 2^-40 of a target's value, 2^-32 of others.  A half wave holds half
                        // of the item's scores and of its columns' sums: both have to follow alike.
                        if (__any(high > kLift)) {
                            high = fmaxf(high, __shfl_xor(high, 32, kWave));
                            const float down = high > kLift ? ceilf(high - (hit ? kLift : kLift / 2)) : 0.0f;
                            const float factor = exp2_fast(-down);
                            lift[cb] -= down;
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                s[cb][i] -= down;
                            }
#pragma unroll
                            for (int db = 0; db < DB; ++db) {
#pragma unroll
                                for (int i = 0; i < 16; ++i) {
                                    acc[cb][db][i] *= factor;
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        s[cb][i] = exp2_fast(s[cb][i]);
                    }
                    if (hit) {
                        int mine = ownBase + cb * 32 + col;
                        pin(mine);
                        const float raise = P == 2 ? exp2_fast(lift[cb]) : 1.0f;
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const Hits h = hits(8 * q);
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                s[cb][4 * q + j] -= h.t[j] == mine ? h.g[j] * raise : 0.0f;
                            }
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
            // Second product: contracted over the piece's rows, in the order in which the registers hold them.  bfloat16: where the
            // piece holds a target, whose value is nearly the whole gradient of its row, a second round adds what the rounding
            // of the values has left, so that most gradients are off by their own rounding alone.  (A loop, not a branch with
            // the product in it a second time: that made the compiler keep the accumulators twice.)
            const int rowOf = r0 + 4 * ((lane & 15) >> 2) + half;
            const E* columnAt = &tile[buf][rowOf * L::kRow + ((lane >> 4) & 1) * 16 + (lane & 3) * 4];
            bool again = P == 1 && hit;
#pragma unroll 1
            while (true) {
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        split_planes<P>(s[cb][i], i % 8, g[cb][i / 8]);
                    }
                }
#pragma unroll
                for (int db = 0; db < DB; ++db) {
#pragma unroll
                    for (int kk = 0; kk < 2; ++kk) {
                        Frag<P> w[P];
#pragma unroll
                        for (int k = 0; k < P; ++k) {
                            Short4 v[2];
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const E* p = columnAt + k * L::kPlane + (16 * kk + 2 * j) * L::kRow + db * 32;
                                v[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                    (__attribute__((address_space(3))) Short4*)(const_cast<E*>(p)));
                            }
                            __builtin_memcpy(&w[k], v, 16);
                        }
#pragma unroll
                        for (int cb = 0; cb < CB; ++cb) {
                            acc[cb][db] = product<P>(w, g[cb][kk], acc[cb][db]);
                        }
                    }
                }
                if (!again) {
                    break;
                }
                again = false;
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        s[cb][i] -= (float)(E)s[cb][i];
                    }
                }
            }
        }
    };

    // Both pieces' scores first: the second's products run beside the first's exponentials (2048 x 1 M x 128 bfloat16: dx 990 and
    // 953 us, dt 1126 and 1067).  Where a piece's scores take 32 registers, or float32's planes many (2048 x 100 k x 64, dx: 175
    // and 191 us), there is no room for two.
    constexpr bool kPaired = P == 1 && PASS != kLossForward && TR == 64 && OW == 4 && RW == 32 && DP <= 128;
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
            if constexpr (kPaired) {
                Float16 s0[CB];
                Float16 s1[CB];
                score(shiftedC, s0, buf, 0);
                score(shiftedC, s1, buf, 32);
                use(shiftedC, s0, buf, 0, t * TR);
                use(shiftedC, s1, buf, 32, t * TR + 32);
            } else {
#pragma unroll 1
                for (int k = 0; k < TR / 32 / L::kStreamWaves; ++k) {
                    const int r0 = (k * L::kStreamWaves + streamWave) * 32;
                    Float16 s[CB];
                    score(shiftedC, s, buf, r0);
                    use(shiftedC, s, buf, r0, t * TR + r0);
                }
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
    if (ownBase >= a.owners) {
        return;
    }

    const int cutBase = a.whole * (OW * RW);   // the first owner of a cut block
    const int64_t partRow = (int64_t)(split * L::kStreamWaves + streamWave) * (a.owners - cutBase) - cutBase;
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
            // what P = 2 has scaled by: the streaming operand, and the probabilities
            const float down = P != 2 ? 1.0f : exp2_fast(kDt ? -lift[cb] : -kLift) / streamScale;
#pragma unroll
            for (int q = 0; q < DB * 4; ++q) {
                const int d = q * 8 + 4 * half;
                Float4 v = {acc[cb][q / 4][q % 4 * 4], acc[cb][q / 4][q % 4 * 4 + 1], acc[cb][q / 4][q % 4 * 4 + 2],
                            acc[cb][q / 4][q % 4 * 4 + 3]};
                if (P == 2) {
                    v *= down;
                }
                if (cut) {
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

template <int P, int DP, int RW, int OW, int PASS, bool SHIFT>
int launch_tiles(const LossArgs& a, const PassPlan& p, hipStream_t stream)
{
    const char* name = PASS == kLossForward ? "k_softmax_forward" : PASS == kLossDx ? "k_softmax_dx" : "k_softmax_dt";
    const int64_t grid = p.whole + (p.blocks - p.whole) * p.splits;
    RECSDK_LAUNCH_AS(name, (k_softmax_tiles<P, DP, RW, OW, PASS, SHIFT>), dim3((unsigned)grid), dim3(kLossThreads), stream, a);
    return RECSDK_OK;
}

template <int P, int DP, int PASS>
int launch_width(const LossArgs& a, const PassPlan& p, hipStream_t stream)
{
    constexpr int kWide = wide_rows(P, DP, PASS);
    if constexpr (PASS != kLossDt && P != 2) {
        if (p.ownWaves < 4) {
            return launch_tiles<P, DP, 32, narrow_waves(P, DP), PASS, true>(a, p, stream);
        }
    }
    if constexpr (kWide == 64) {
        if (p.rowsPerWave == 32) {
            if constexpr (PASS == kLossDt) {   // a shift is an item's own there, and costs nothing to do without
                return a.bias != nullptr ? launch_tiles<P, DP, 32, 4, PASS, true>(a, p, stream)
                                         : launch_tiles<P, DP, 32, 4, PASS, false>(a, p, stream);
            }
            return launch_tiles<P, DP, 32, 4, PASS, true>(a, p, stream);
        }
    }
    if constexpr (P != 3 || PASS == kLossDt) {
        return a.bias != nullptr ? launch_tiles<P, DP, kWide, 4, PASS, true>(a, p, stream)
                                 : launch_tiles<P, DP, kWide, 4, PASS, false>(a, p, stream);
    }
    set_error("softmax loss: no kernel for this shape");
    return RECSDK_EINVAL;
}

template <int P, int PASS>
int launch_pass(const LossArgs& a, const PassPlan& p, hipStream_t stream)
{
    switch (loss_width(a.dim)) {
        case 32:
            return launch_width<P, 32, PASS>(a, p, stream);
        case 64:
            return launch_width<P, 64, PASS>(a, p, stream);
        case 96:
            return launch_width<P, 96, PASS>(a, p, stream);
        case 128:
            return launch_width<P, 128, PASS>(a, p, stream);
        case 160:
            return launch_width<P, 160, PASS>(a, p, stream);
        case 192:
            return launch_width<P, 192, PASS>(a, p, stream);
        case 224:
            return launch_width<P, 224, PASS>(a, p, stream);
        default:
            return launch_width<P, 256, PASS>(a, p, stream);
    }
}

#endif  // RECSDK_SOFTMAX_KERNELS

}  // namespace recsdk

#endif
