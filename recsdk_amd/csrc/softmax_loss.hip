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
// running sums need no exchange between lanes, and exp(S) is, as it lies, the A operand of the second product
// (contracted over the stream's rows, 8 of 16 per half wave); the B operand of that product is the same LDS tile read
// through the transposing LDS load.  A tile is laid out in 16-byte chunks whose place is exchanged by the row
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

struct Yes {
    static constexpr bool value = true;
};
struct No {
    static constexpr bool value = false;
};

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
    float* part;            // backward: [split parts][owners][dim] partial sums, or NULL
    void* out;              // dt pass without parts: [owners][dim] in the operands' type
};

__device__ __forceinline__ float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }

// Where chunk c (16 bytes) of tile row r lies within the row: the 16 rows that one access of the first product
// touches, and the 4 rows by 4 chunks that one of the transposing loads touches, then fall on different banks.
template <int CHUNKS>
__device__ __forceinline__ int swizzle(int r, int c)
{
    if constexpr (CHUNKS >= 16) {
        return c ^ (((r & 3) << 2) | ((r >> 2) & 3));
    } else if constexpr (CHUNKS == 8) {
        return c ^ ((((r >> 1) & 1) << 2) | ((r >> 2) & 3));
    } else {
        return c ^ ((r >> 2) & 3);
    }
}

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

// Eight columns of a row as they come from memory.
template <int P>
struct RowChunk;
template <>
struct RowChunk<1> {
    Word4 v;
    __device__ __forceinline__ void load(const void* base, int64_t row, int64_t stride, int c, int dim)
    {
        v = Word4{0, 0, 0, 0};
        if (c * 8 < dim) {
            v = *reinterpret_cast<const Word4*>(static_cast<const BF16*>(base) + row * stride + c * 8);
        }
    }
    __device__ __forceinline__ void clear() { v = Word4{0, 0, 0, 0}; }
    __device__ __forceinline__ void planes(Bf16x8 (&p)[1]) const { __builtin_memcpy(&p[0], &v, 16); }
};
template <>
struct RowChunk<3> {
    Float4 v[2];
    __device__ __forceinline__ void load(const void* base, int64_t row, int64_t stride, int c, int dim)
    {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            v[h] = Float4{0, 0, 0, 0};
            if (c * 8 + h * 4 < dim) {
                v[h] = *reinterpret_cast<const Float4*>(static_cast<const float*>(base) + row * stride + c * 8 + h * 4);
            }
        }
    }
    __device__ __forceinline__ void clear() { v[0] = v[1] = Float4{0, 0, 0, 0}; }
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
    static constexpr int kPlane = kRows * DP;                       // elements
    static constexpr int kBuffers = P * kPlane * 2 * 2 > 131072 ? 1 : 2;
    static_assert(kLoads >= 1 && kLoads * kLossThreads == kRows * kChunks, "whole chunks per thread");
    static_assert(P * kPlane * 2 * kBuffers <= 131072, "the tiles fit LDS");
};

template <int P, int DP, int RW, int OW, int PASS, int OCC>
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
    __shared__ __attribute__((aligned(16))) float auxA[NB][TR];                               // forward, dx: bias (base 2); dt: lse (base 2)
    __shared__ __attribute__((aligned(16))) float auxG[PASS == kLossDt ? NB : 1][PASS == kLossDt ? TR : 1];   // dt: grad * scale
    __shared__ int32_t auxT[PASS == kLossDt ? NB : 1][PASS == kLossDt ? TR : 1]; // dt: target

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
    const int t1 = min(t0 + a.tilesPerSplit, tiles);
    const float c2 = a.scale * kLog2e;
    const bool biased = a.bias != nullptr;

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
            if (live) {
                r.load(a.own, n, a.ownStride, ks * 2 + half, a.dim);
            } else {
                r.clear();   // rows past the end, padding positions and free slots may hold anything
            }
            r.planes(own[cb][ks]);
        }
    }

    // ---- the stream's tiles: memory -> registers (one tile ahead) -> LDS ----
    RowChunk<P> staged[L::kLoads];
    float stagedA = 0.0f;
    float stagedG = 0.0f;
    int32_t stagedT = -1;
    bool stagedLive[L::kLoads];
    auto fetch = [&](int t) {
#pragma unroll
        for (int q = 0; q < L::kLoads; ++q) {
            const int i = q * kLossThreads + threadIdx.x;
            const int64_t row = (int64_t)t * TR + i / CH;
            const int64_t at = row < a.streams ? row : a.streams - 1;
            bool live = row < a.streams;
            if constexpr (PASS == kLossDt) {
                live = live && a.lse[at] != INFINITY;
            } else if (biased) {
                live = live && a.bias[at] > kMaskedBelow;
            }
            stagedLive[q] = live;
            staged[q].load(a.stream, at, a.streamStride, i % CH, a.dim);
        }
        if (threadIdx.x < TR) {
            const int64_t row = (int64_t)t * TR + threadIdx.x;
            if constexpr (PASS == kLossDt) {
                const float l = row < a.streams ? a.lse[row] : INFINITY;
                const bool live = l != INFINITY;   // a NaN stays one
                stagedA = live ? l * kLog2e : INFINITY;
                stagedG = live ? a.grad[row] * a.scale : 0.0f;
                stagedT = live ? (int32_t)a.target[row] : -1;
            } else {
                const float b = row >= a.streams ? -INFINITY : biased ? a.bias[row] : 0.0f;
                stagedA = b > kMaskedBelow ? b * kLog2e : -INFINITY;
            }
        }
    };
    auto place = [&](int buf) {
#pragma unroll
        for (int q = 0; q < L::kLoads; ++q) {
            const int i = q * kLossThreads + threadIdx.x;
            const int r = i / CH;
            const int c = swizzle<CH>(r, i % CH);
            if (!stagedLive[q]) {
                staged[q].clear();   // 0 times whatever lies there must be 0
            }
            Bf16x8 p[P];
            staged[q].planes(p);
#pragma unroll
            for (int k = 0; k < P; ++k) {
                *reinterpret_cast<Bf16x8*>(&tile[buf][k * L::kPlane + r * DP + c * 8]) = p[k];
            }
        }
        if (threadIdx.x < TR) {
            auxA[buf][threadIdx.x] = stagedA;
            if constexpr (PASS == kLossDt) {
                auxG[buf][threadIdx.x] = stagedG;
                auxT[buf][threadIdx.x] = stagedT;
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
        const BF16* base = tile[buf];
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
            const int r = r0 + col;
            const int c = swizzle<CH>(r, ks * 2 + half);
#pragma unroll
            for (int k = 0; k < P; ++k) {
                x[k] = *reinterpret_cast<const Bf16x8*>(base + k * L::kPlane + r * DP + c * 8);
            }
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) {
                s[cb] = product<P>(x, own[cb][ks], s[cb]);
            }
        }
        // register i of a lane holds stream row r0 + 8 (i / 4) + 4 half + i % 4, owner row ownBase + cb * 32 + col
        if constexpr (PASS == kLossForward) {
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
                float most = -INFINITY;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[cb][i] = shifted ? __builtin_fmaf(s[cb][i], c2, b[i]) : s[cb][i] * c2;
                    most = fmaxf(most, s[cb][i]);
                }
                // the maximum follows only when it has fallen far behind: sums up to 2^kSlack per item fit easily
                if (__any(most > top[cb] + kSlack)) {
                    const float now = fmaxf(top[cb], most);
                    sum[cb] *= exp2_fast(top[cb] - now);
                    top[cb] = now;
                }
                float add = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    add += exp2_fast(s[cb][i] - top[cb]);
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
                    const int d = ownTarget[cb] - rowBase;
                    if (__any(d >= 0 && d < 32)) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            s[cb][i] -= d == 8 * (i / 4) + 4 * half + i % 4 ? 1.0f : 0.0f;
                        }
                    }
                }
            } else {
                float shift[16];
                float gr[16];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const Float4 v = *reinterpret_cast<const Float4*>(&auxA[buf][r0 + 8 * q + 4 * half]);
                    const Float4 w = *reinterpret_cast<const Float4*>(&auxG[buf][r0 + 8 * q + 4 * half]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        shift[4 * q + j] = -v[j];
                        gr[4 * q + j] = w[j];
                    }
                }
                const int mine = auxT[buf][r0 + col] - ownBase;
                const bool hit = __any(mine >= 0 && mine < RW);
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        s[cb][i] = exp2_fast(__builtin_fmaf(s[cb][i], c2, shifted ? shift[i] + ownShift[cb] : shift[i]));
                    }
                    if (hit) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int d = auxT[buf][r0 + 8 * (i / 4) + 4 * half + i % 4] - ownBase;
                            s[cb][i] -= d == cb * 32 + col ? 1.0f : 0.0f;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        s[cb][i] *= gr[i];
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
            const int quad = (lane & 15) >> 2;
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
                            const int r = r0 + 16 * kk + 8 * j + 4 * half + quad;
                            const int c = swizzle<CH>(r, db * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1));
                            const BF16* p = base + k * L::kPlane + r * DP + c * 8 + (lane & 1) * 4;
                            v[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                (__attribute__((address_space(3))) Short4*)(const_cast<BF16*>(p)));
                        }
                        __builtin_memcpy(&w[k], v, 16);
                    }
#pragma unroll
                    for (int cb = 0; cb < CB; ++cb) {
                        acc[cb][db] = product<P>(g[cb][kk], w, acc[cb][db]);
                    }
                }
            }
        }
    };

    auto compute = [&](int buf, int t) {
        const int rows = min(TR, a.streams - t * TR);
        if (biased || (PASS != kLossDt && rows < TR)) {
#pragma unroll 1
            for (int r0 = streamWave * 32; r0 < rows; r0 += 32 * L::kStreamWaves) {
                piece(Yes{}, buf, r0, t * TR + r0);
            }
        } else {
#pragma unroll 1
            for (int r0 = streamWave * 32; r0 < rows; r0 += 32 * L::kStreamWaves) {
                piece(No{}, buf, r0, t * TR + r0);
            }
        }
    };

    const bool idle = ownBase >= a.owners;   // the wave owns nothing, but keeps the barriers and moves its share
    if (t0 < t1) {
        fetch(t0);
        place(0);
        __syncthreads();
        for (int t = t0; t < t1; ++t) {
            const int buf = NB == 2 ? (t - t0) & 1 : 0;
            if (t + 1 < t1) {
                fetch(t + 1);
            }
            if (!idle) {
                compute(buf, t);
            }
            if (NB == 1) {
                __syncthreads();
            }
            if (t + 1 < t1) {
                place(NB == 2 ? buf ^ 1 : 0);
            }
            __syncthreads();
        }
    }
    if (idle) {
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
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int n = ownBase + cb * 32 + 8 * (i / 4) + 4 * half + i % 4;
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                    const int d = db * 32 + col;
                    if (n < a.owners && d < a.dim) {
                        if (a.part != nullptr) {
                            a.part[(partRow + n) * a.dim + d] = acc[cb][db][i];
                        } else if constexpr (P == 1) {
                            static_cast<BF16*>(a.out)[(int64_t)n * a.dim + d] = (BF16)acc[cb][db][i];
                        } else {
                            static_cast<float*>(a.out)[(int64_t)n * a.dim + d] = acc[cb][db][i];
                        }
                    }
                }
            }
        }
    }
}

// Joins the parts of the running sums and takes the target's score off: one wave per row of x.
template <typename T>
__global__ __launch_bounds__(kBlock) void k_softmax_loss_join(const float2* __restrict__ norm, int parts, int rows, int items,
                                                              int dim, const T* __restrict__ x, int64_t xStride,
                                                              const T* __restrict__ table, int64_t tableStride,
                                                              const int64_t* __restrict__ target, const float* __restrict__ bias,
                                                              float scale, float* __restrict__ loss, float* __restrict__ lse)
{
    const int n = blockIdx.x * (kBlock / kWave) + threadIdx.x / kWave;
    const int lane = lane_id();
    if (n >= rows) {
        return;
    }
    const int64_t t = target[n];
    if (t < 0 || t >= items) {   // no target: no loss, no gradient
        if (lane == 0) {
            loss[n] = 0.0f;
            lse[n] = INFINITY;
        }
        return;
    }
    const float b = bias != nullptr ? bias[t] : 0.0f;
    if (b <= kMaskedBelow) {   // the target cannot be had: infinite loss, no gradient
        if (lane == 0) {
            loss[n] = INFINITY;
            lse[n] = INFINITY;
        }
        return;
    }
    float top = kFloor;
    float sum = 0.0f;
    for (int p = lane; p < parts; p += kWave) {
        const float2 v = norm[(int64_t)p * rows + n];
        const float now = fmaxf(top, v.x);
        sum = sum * exp2_fast(top - now) + v.y * exp2_fast(v.x - now);
        top = now;
    }
    float dot = 0.0f;
    for (int d = lane; d < dim; d += kWave) {
        dot = __builtin_fmaf((float)x[n * xStride + d], (float)table[t * tableStride + d], dot);
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
    if (lane == 0) {
        const float l = __builtin_fmaf(top, kLn2, logf(sum));
        loss[n] = l - __builtin_fmaf(dot, scale, b);
        lse[n] = l;
    }
}

// out = factor(row) * sum of the parts, in their order, in the operands' type.
template <typename T>
__global__ __launch_bounds__(kBlock) void k_softmax_grad_join(const float* __restrict__ part, int parts, int64_t count, int dim,
                                                              const float* __restrict__ lse, const float* __restrict__ grad,
                                                              float scale, T* __restrict__ out)
{
    const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (i >= count) {
        return;
    }
    float s = 0.0f;
#pragma unroll 8
    for (int p = 0; p < parts; ++p) {
        s += part[p * count + i];
    }
    if (grad != nullptr) {
        const int64_t n = i / dim;
        s = lse[n] != INFINITY ? s * (grad[n] * scale) : 0.0f;
    }
    out[i] = from_float<T>(s);
}

// Rows of `dim` elements at any stride -> rows of `padded` elements, the rest zero.
template <typename T>
__global__ __launch_bounds__(kBlock) void k_pad_rows(const T* __restrict__ src, int64_t stride, int64_t rows, int dim, int padded,
                                                     T* __restrict__ dst)
{
    const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    const int64_t r = i / padded;
    const int c = (int)(i - r * padded);
    if (r < rows) {
        dst[i] = c < dim ? src[r * stride + c] : from_float<T>(0.0f);
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------

constexpr int kLossResident = 512;   // blocks the card holds at once (two per compute unit)

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

static int tile_rows(int planes, int dp, int ownWaves, int pass)
{
    return ownWaves < 4 ? 32 * (4 / ownWaves) : (planes == 3 && dp > 32) || (dp == 256 && pass != kLossForward) ? 32 : 64;
}

static PassPlan plan_pass(int planes, int dim, int64_t owners, int64_t streams, int pass)
{
    const int dp = padded_dim(dim);
    PassPlan p{};
    p.rowsPerWave = planes == 3 || (dp == 256 && pass != kLossForward) ? 32 : 64;
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
    int64_t splits = kLossResident / p.blocks;
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
    const int64_t dx = (int64_t)p.dx.parts * rows * dim * (int64_t)sizeof(float);
    const int64_t dt = p.dt.parts > 1 ? (int64_t)p.dt.parts * items * dim * (int64_t)sizeof(float) : 0;
    p.forwardBytes = round256(p.atParts + norm);
    p.backwardBytes = round256(p.atParts + (dx > dt ? dx : dt));   // the two passes run one after the other
    return p;
}

template <int P, int DP, int RW, int OW, int PASS, int OCC>
static int launch_tiles(const LossArgs& a, const PassPlan& p, hipStream_t stream)
{
    const char* name = PASS == kLossForward ? "k_softmax_forward" : PASS == kLossDx ? "k_softmax_dx" : "k_softmax_dt";
    RECSDK_LAUNCH_AS(name, (k_softmax_tiles<P, DP, RW, OW, PASS, OCC>), dim3((unsigned)(p.blocks * p.splits)), dim3(kLossThreads),
                     stream, a);
    return RECSDK_OK;
}

template <int P, int DP, int PASS>
static int launch_width(const LossArgs& a, const PassPlan& p, hipStream_t stream)
{
    constexpr int kOcc = P == 3 && DP == 256 ? 1 : 2;
    if constexpr (PASS != kLossDt) {
        constexpr int kNarrow = P == 3 && DP == 256 ? 2 : 1;
        if (p.ownWaves == kNarrow) {
            constexpr int kNarrowOcc = DP == 256 || (P == 3 && DP == 128) ? 1 : 2;
            return launch_tiles<P, DP, 32, kNarrow, PASS, kNarrowOcc>(a, p, stream);
        }
    }
    if constexpr (P == 1 && (DP < 256 || PASS == kLossForward)) {
        if (p.rowsPerWave == 64) {
            return launch_tiles<P, DP, 64, 4, PASS, kOcc>(a, p, stream);
        }
    }
    if constexpr (PASS != kLossDt || P == 3 || DP == 256) {
        return launch_tiles<P, DP, 32, 4, PASS, kOcc>(a, p, stream);
    }
    set_error("softmax loss: no kernel for this shape");
    return RECSDK_EINVAL;
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
    return RECSDK_OK;
}

// The operands as the tile kernels read them: whole 16-byte pieces; others are copied into padded rows.
template <typename T>
static int pad_operand(const void*& p, int64_t& stride, int64_t rows, int dim, int padded, void* to, hipStream_t stream)
{
    const int64_t grid = cdiv(rows * padded, kBlock);
    RECSDK_REQUIRE(grid < (int64_t(1) << 31), RECSDK_EINVAL, "softmax loss: table too large for rows that need padding");
    RECSDK_LAUNCH_AS("k_pad_rows", (k_pad_rows<T>), dim3((unsigned)grid), dim3(kBlock), stream, static_cast<const T*>(p), stride,
                     rows, dim, padded, static_cast<T*>(to));
    p = to;
    stride = padded;
    return RECSDK_OK;
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
    RECSDK_LAUNCH_AS("k_softmax_loss_join", (k_softmax_loss_join<T>), dim3((unsigned)cdiv(rows, kBlock / kWave)), dim3(kBlock),
                     stream, a.norm, plan.forward.parts, (int)rows, (int)items, dim, static_cast<const T*>(given.x),
                     given.xStride, static_cast<const T*>(given.table), given.tableStride, target, bias, scale, loss, lse);
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
        RECSDK_LAUNCH_AS("k_softmax_grad_join", (k_softmax_grad_join<T>), dim3((unsigned)cdiv(rows * dim, kBlock)), dim3(kBlock),
                         stream, part, plan.dx.parts, rows * dim, dim, lse, grad, scale, static_cast<T*>(dx));
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
            RECSDK_LAUNCH_AS("k_softmax_grad_join", (k_softmax_grad_join<T>), dim3((unsigned)cdiv(items * dim, kBlock)),
                             dim3(kBlock), stream, part, plan.dt.parts, items * dim, dim, nullptr, nullptr, scale,
                             static_cast<T*>(dtable));
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
            const int64_t n = items * dim;
            RECSDK_REQUIRE(cdiv(n, kBlock) < (int64_t(1) << 31), RECSDK_EINVAL,
                           "recsdk_softmax_loss_backward: table too large for one launch");
            if (dtype == RECSDK_DT_F32) {
                RECSDK_LAUNCH_AS("k_softmax_grad_join", (k_softmax_grad_join<float>), dim3((unsigned)cdiv(n, kBlock)), dim3(kBlock),
                                 s, nullptr, 0, n, dim, nullptr, nullptr, scale, static_cast<float*>(d_dtable));
            } else {
                RECSDK_LAUNCH_AS("k_softmax_grad_join", (k_softmax_grad_join<BF16>), dim3((unsigned)cdiv(n, kBlock)), dim3(kBlock),
                                 s, nullptr, 0, n, dim, nullptr, nullptr, scale, static_cast<BF16*>(d_dtable));
            }
        }
        return RECSDK_OK;
    }
    RECSDK_REQUIRE(d_grad_loss != nullptr && d_x != nullptr && d_table != nullptr && d_target != nullptr && d_lse != nullptr,
                   RECSDK_ENULL, "recsdk_softmax_loss_backward: NULL argument");
    RECSDK_REQUIRE(aligned16(d_x) && aligned16(d_table) && aligned16(d_workspace), RECSDK_EINVAL,
                   "recsdk_softmax_loss_backward: x, table and workspace must be 16-byte aligned");
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
