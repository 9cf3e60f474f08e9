// Layer norm over the columns of a row, forward and backward.
//
//   forward    mean = sum x / D,  var = sum (x - mean)^2 / D,  rstd = 1 / sqrt(var + eps),  hat = (x - mean) rstd
//              y = hat weight + bias
//   backward   g = dy weight;  dx = rstd (g - sum g / D - hat sum (g hat) / D);  dweight = sum_rows dy hat;  dbias = sum_rows dy
//
// Rows are held in registers between their one read and their one write: a team of G threads per row, every thread K
// packs of 16 bytes, the variance from the differences and not from the squares.  A team walks rows at a fixed stride,
// keeps its columns of weight and bias in registers and has the next rows' loads in flight while it reduces the present
// ones (R rows side by side where a row is one pack per thread).  In the backward pass the same threads sum their columns
// of dweight and dbias over the team's rows; the teams of a block are joined in LDS, the blocks' sums go to the workspace
// and a second kernel adds them in the order of the blocks: no atomics, so a call gives the same bits every time.  All
// sums are held in 32 bits; every result is rounded once.
// Rows that do not start on 16-byte borders (an odd width) would move element by element, with an eighth of the bytes per
// instruction; contiguous ones are staged instead: a block copies a span of whole rows, 16 KB of them, through LDS along the
// 16-byte borders and works on elements there (30011 x 1001 fp16 forward: 50 -> 31 us).
// What bounds it: the row traffic (read x, write y; read dy and x, write dx).
#include <math.h>

#include "dense.h"

namespace recsdk {

constexpr int kNormBlocks = 1024;       // blocks of the backward pass at most: each leaves 2 D sums in the workspace
constexpr int kNormRowBlocks = 512;     // of them, where a block holds few rows' worth of registers
constexpr int kNormForwardBlocks = 2048;
constexpr int kNormSpanBlocks = 2048;
constexpr int kNormWideBlocks = 65536;  // a launch holds fewer than 2^32 threads
constexpr int kSpanBytes = 16384;       // rows that a block stages at once
constexpr int kSpanLoads = kSpanBytes / 16 / kBlock;
constexpr int kSpanRows = kBlock;       // at most: one thread fetches a row's statistics
constexpr int kReduceCols = 64;         // columns per block of the joining kernel
constexpr int kReduceWaves = 16;

struct NormRows {
    const void* x;
    int64_t stride;     // elements between rows of x
    int64_t rows;
    int32_t dim;
    const void* weight; // NULL: 1
    const void* bias;   // NULL: 0
    float eps;
    float* mean;
    float* rstd;
    void* y;            // forward; rows are dim elements apart
    const void* grad;   // backward; rows are dim elements apart
    void* dx;
    float* part;        // [blocks][2][dim]
};

// Sums over the G threads of a team.  G > 64: the team is the block, `smem` holds N floats per wave.
template <int G, int N>
__device__ __forceinline__ void team_sum(float (&v)[N], float* smem)
{
#pragma unroll
    for (int n = 0; n < N; ++n) {
        v[n] = group_sum<(G < kWave ? G : kWave)>(v[n]);
    }
    if constexpr (G > kWave) {
        constexpr int kWaves = G / kWave;
        const int w = threadIdx.x / kWave;
        __syncthreads();   // the previous sums have been read
        if (lane_id() == 0) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                smem[N * w + n] = v[n];
            }
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) {
            v[n] = 0.0f;
#pragma unroll
            for (int k = 0; k < kWaves; ++k) {
                v[n] += smem[N * k + n];
            }
        }
    }
}

template <typename W>
__device__ __forceinline__ float param(const void* p, int64_t c, float none)
{
    return p != nullptr ? (float)static_cast<const W*>(p)[c] : none;
}

// A thread's values of weight or bias: pack k holds E of them (E = 1, or a whole aligned piece) from column first + k step on;
// 0 past the row's end.  The loads are made at a clamped column, so that none of them waits behind a branch for another.
template <typename W, int E, int K>
__device__ __forceinline__ void params(const void* p, int first, int step, int dim, float none, float (&out)[K][E])
{
    if (p == nullptr) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                out[k][e] = first + k * step < dim ? none : 0.0f;
            }
        }
        return;
    }
    const W* w = static_cast<const W*>(p);
    constexpr int kPer = E * sizeof(W) >= 16 ? 16 / (int)sizeof(W) : E;
    Pack<W, kPer> v[K][E / kPer];
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int q = 0; q < E / kPer; ++q) {
            v[k][q] = load_pack<W, kPer>(w + min(first + k * step, dim - E) + q * kPer);
        }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            out[k][e] = first + k * step < dim ? (float)v[k][e / kPer].v[e % kPer] : 0.0f;
        }
    }
}

// The block's column sums: its teams' joined in LDS (`joined`: kTeams * G * K * E floats; one team: unused), then written.
template <int E, int G, int K, int TEAMS>
__device__ __forceinline__ void leave_parts(const NormRows& a, float* joined, const float (&dw)[K][E], const float (&db)[K][E])
{
    constexpr int kCols = G * K * E;
    const int team = threadIdx.x / G;
    float* part = a.part + (int64_t)blockIdx.x * 2 * a.dim;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if constexpr (TEAMS > 1) {
            __syncthreads();
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int c = (k * G + (int)threadIdx.x % G) * E + e;
                if (c < a.dim) {
                    (TEAMS > 1 ? joined[team * kCols + c] : part[which * a.dim + c]) = which == 0 ? dw[k][e] : db[k][e];
                }
            }
        }
        if constexpr (TEAMS > 1) {
            __syncthreads();
            for (int c = threadIdx.x; c < a.dim; c += TEAMS * G) {
                float sum = 0.0f;
#pragma unroll
                for (int t = 0; t < TEAMS; ++t) {
                    sum += joined[t * kCols + c];
                }
                part[which * a.dim + c] = sum;
            }
        }
    }
}

// Rows that a team has in work at once.
template <int G, int K, bool BACK>
constexpr int kNormRows = G > kWave ? 1 : K == 1 ? (BACK ? 2 : 4) : K == 2 && !BACK ? 2 : 1;

template <typename T, typename W, int E, int G, int K>
__global__ __launch_bounds__(G > kBlock ? G : kBlock) void k_layer_norm(NormRows a)
{
    constexpr int R = kNormRows<G, K, false>;
    constexpr int kTeams = G > kBlock ? 1 : kBlock / G;
    __shared__ float smem[G > kWave ? R * G / kWave : 1];
    const int64_t step = (int64_t)gridDim.x * (R * kTeams);
    int64_t row = (int64_t)blockIdx.x * (R * kTeams) + threadIdx.x / G;
    if (row >= a.rows) {
        return;   // the whole team
    }
    const T* x = static_cast<const T*>(a.x);
    T* y = static_cast<T*>(a.y);
    const int dim = a.dim;
    const int first = threadIdx.x % G * E;   // pack k starts at column first + k G E
    float wt[K][E];
    float bs[K][E];
    params<W, E, K>(a.weight, first, G * E, dim, 1.0f, wt);
    params<W, E, K>(a.bias, first, G * E, dim, 0.0f, bs);
    const float inv = 1.0f / (float)dim;
    Pack<T, E> next[R][K];
    auto fetch = [&](int64_t r) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int64_t at = r + i * kTeams;
            if (at < a.rows) {
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const int c = first + k * G * E;
                    if (c < dim) {
                        next[i][k] = load_pack<T, E>(x + at * a.stride + c);
                    }
                }
            }
        }
    };
    fetch(row);
    for (; row < a.rows; row += step) {
        float v[R][K][E];
        float mean[R];
        float rstd[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            mean[i] = 0.0f;
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    v[i][k][e] = first + k * G * E < dim ? (float)next[i][k].v[e] : 0.0f;
                    mean[i] += v[i][k][e];
                }
            }
        }
        fetch(row + step);
        team_sum<G>(mean, smem);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            mean[i] *= inv;
            rstd[i] = 0.0f;
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    v[i][k][e] = first + k * G * E < dim ? v[i][k][e] - mean[i] : 0.0f;
                    rstd[i] = __builtin_fmaf(v[i][k][e], v[i][k][e], rstd[i]);
                }
            }
        }
        team_sum<G>(rstd, smem);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int64_t r = row + i * kTeams;
            if (r >= a.rows) {
                break;
            }
            rstd[i] = 1.0f / sqrtf(rstd[i] * inv + a.eps);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                Pack<T, E> out;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    out.v[e] = from_float<T>(__builtin_fmaf(v[i][k][e] * rstd[i], wt[k][e], bs[k][e]));
                }
                if (first + k * G * E < dim) {
                    store_pack<T, E>(y + r * dim + first + k * G * E, out);
                }
            }
            if (threadIdx.x % G == 0 && a.mean != nullptr) {
                a.mean[r] = mean[i];
                a.rstd[r] = rstd[i];
            }
        }
    }
}

template <typename T, typename W, int E, int G, int K>
__global__ __launch_bounds__(G > kBlock ? G : kBlock) void k_layer_norm_backward(NormRows a)
{
    constexpr int R = kNormRows<G, K, true>;
    constexpr int kThreads = G > kBlock ? G : kBlock;
    constexpr int kTeams = kThreads / G;
    constexpr int kCols = G * K * E;   // columns a team covers
    // the teams' column sums, joined at the end (one team per block: nothing to join)
    __shared__ float joined[kTeams > 1 ? kTeams * kCols : 1];
    static_assert(kTeams == 1 || kTeams * kCols <= 8192, "the teams' sums fit the LDS array");
    __shared__ float smem[G > kWave ? 2 * R * G / kWave : 1];
    const int team = threadIdx.x / G;
    const int64_t step = (int64_t)gridDim.x * (R * kTeams);
    const int dim = a.dim;
    const float inv = 1.0f / (float)dim;
    const T* x = static_cast<const T*>(a.x);
    const T* dy = static_cast<const T*>(a.grad);
    T* dx = static_cast<T*>(a.dx);
    int64_t row = (int64_t)blockIdx.x * (R * kTeams) + team;
    const int first = threadIdx.x % G * E;   // pack k starts at column first + k G E
    float wt[K][E];
    float dw[K][E];
    float db[K][E];
    params<W, E, K>(a.weight, first, G * E, dim, 1.0f, wt);
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            dw[k][e] = 0.0f;
            db[k][e] = 0.0f;
        }
    }
    Pack<T, E> nx[R][K];
    Pack<T, E> ng[R][K];
    float nmean[R];
    float nrstd[R];
    auto fetch = [&](int64_t from) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int64_t r = from + i * kTeams;
            if (r < a.rows) {
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const int c = first + k * G * E;
                    if (c < dim) {
                        nx[i][k] = load_pack<T, E>(x + r * a.stride + c);
                        ng[i][k] = load_pack<T, E>(dy + r * dim + c);
                    }
                }
                nmean[i] = a.mean[r];
                nrstd[i] = a.rstd[r];
            }
        }
    };
    fetch(row);
    for (; row < a.rows; row += step) {
        float hat[R][K][E];
        float g[R][K][E];
        float s[2 * R];
        float rstd[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const bool here = row + i * kTeams < a.rows;
            rstd[i] = nrstd[i];
            s[2 * i] = 0.0f;
            s[2 * i + 1] = 0.0f;
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const bool in = first + k * G * E < dim && (R == 1 || here);
                    hat[i][k][e] = in ? ((float)nx[i][k].v[e] - nmean[i]) * rstd[i] : 0.0f;
                    const float d = in ? (float)ng[i][k].v[e] : 0.0f;
                    dw[k][e] = __builtin_fmaf(d, hat[i][k][e], dw[k][e]);
                    db[k][e] += d;
                    g[i][k][e] = d * wt[k][e];
                    s[2 * i] += g[i][k][e];
                    s[2 * i + 1] = __builtin_fmaf(g[i][k][e], hat[i][k][e], s[2 * i + 1]);
                }
            }
        }
        fetch(row + step);
        if (dx != nullptr) {
            team_sum<G>(s, smem);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int64_t r = row + i * kTeams;
                if (r >= a.rows) {
                    break;
                }
                const float s0 = s[2 * i] * inv;
                const float s1 = s[2 * i + 1] * inv;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    Pack<T, E> out;
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        out.v[e] = from_float<T>(rstd[i] * (g[i][k][e] - s0 - hat[i][k][e] * s1));
                    }
                    if (first + k * G * E < dim) {
                        store_pack<T, E>(dx + r * dim + first + k * G * E, out);
                    }
                }
            }
        }
    }
    if (a.part != nullptr) {
        leave_parts<E, G, K, kTeams>(a, joined, dw, db);
    }
}

// ---- staged rows ------------------------------------------------------------------------------------------------------
// A span of contiguous rows on its way between memory and LDS.  It starts `lead` elements behind a 16-byte border and moves
// in pieces along those borders: reads take whole pieces also where a neighbouring span has part of one, writes do not;
// what is left, pieces that reach past the buffer (reads) or the span (writes), is a few elements, one thread each.
template <typename T>
struct Span {
    static constexpr int kPer = 16 / sizeof(T);
    const T* origin;   // the border at or before the first element
    int before;        // elements of the buffer, from origin on, as far as a span can reach: [before, behind)
    int behind;
    int lead;
    int count;         // elements of the span
    __device__ __forceinline__ Span(const T* buffer, int64_t total, int64_t from, int n)
    {
        lead = (int)(reinterpret_cast<uintptr_t>(buffer + from) % 16 / sizeof(T));
        origin = buffer + from - lead;
        before = from < lead ? lead - (int)from : 0;
        behind = (int)min(total - from + lead, (int64_t)kSpanBytes);
        count = n;
    }
    __device__ __forceinline__ int pieces() const { return (lead + count + kPer - 1) / kPer; }
    __device__ __forceinline__ bool whole(int piece) const
    {
        return piece * kPer >= before && piece * kPer + kPer <= behind;
    }
    __device__ __forceinline__ void load(Word4 (&r)[kSpanLoads]) const
    {
#pragma unroll
        for (int q = 0; q < kSpanLoads; ++q) {
            const int i = q * kBlock + threadIdx.x;
            if (i < pieces() && whole(i)) {
                r[q] = *reinterpret_cast<const Word4*>(origin + i * kPer);
            }
        }
    }
    __device__ __forceinline__ void place(const Word4 (&r)[kSpanLoads], T* lds) const
    {
#pragma unroll
        for (int q = 0; q < kSpanLoads; ++q) {
            const int i = q * kBlock + threadIdx.x;
            if (i < pieces() && whole(i)) {
                *reinterpret_cast<Word4*>(lds + i * kPer) = r[q];
            }
        }
        edges([&](int piece) { return !whole(piece); }, [&](int e) { lds[e] = origin[e]; });
    }
    // from LDS (laid out like `place` leaves it) to the same place of another buffer
    __device__ __forceinline__ void store(const T* lds, T* to) const
    {
#pragma unroll
        for (int q = 0; q < kSpanLoads; ++q) {
            const int i = q * kBlock + threadIdx.x;
            if (i < pieces() && i * kPer >= lead && i * kPer + kPer <= lead + count) {
                __builtin_nontemporal_store(*reinterpret_cast<const Word4*>(lds + i * kPer),
                                            reinterpret_cast<Word4*>(to - lead + i * kPer));
            }
        }
        edges([&](int piece) { return piece * kPer < lead || piece * kPer + kPer > lead + count; },
              [&](int e) { to[e - lead] = lds[e]; });
    }
    // The span's elements in its first and in its last piece, where those ask for it: one thread each.
    template <typename Asks, typename Move>
    __device__ __forceinline__ void edges(Asks asks, Move move) const
    {
        const int last = pieces() - 1;
        const int piece = threadIdx.x < kPer ? 0 : last;
        const int e = piece * kPer + (int)threadIdx.x % kPer;
        if (threadIdx.x < 2 * kPer && (threadIdx.x < kPer || last > 0) && e >= lead && e < lead + count && asks(piece)) {
            move(e);
        }
    }
};

// The span's rows lie in LDS; a team takes every kTeams-th of them, a thread columns lane, lane + G, ...
template <typename T, typename W, int G, int K>
__global__ __launch_bounds__(kBlock) void k_layer_norm_staged(NormRows a, int spanRows)
{
    constexpr int kTeams = kBlock / G;
    constexpr int R = G > kWave || K > 8 ? 1 : 2;   // rows that a team has in work at once
    __shared__ __attribute__((aligned(16))) T lds[kSpanBytes / sizeof(T)];
    __shared__ float smem[G > kWave ? R * G / kWave : 1];
    const int dim = a.dim;
    const int lane = threadIdx.x % G;
    const int64_t total = a.rows * dim;
    float wt[K][1];
    float bs[K][1];
    params<W, 1, K>(a.weight, lane, G, dim, 1.0f, wt);
    params<W, 1, K>(a.bias, lane, G, dim, 0.0f, bs);
    const float inv = 1.0f / (float)dim;
    Word4 raw[kSpanLoads];
    const int64_t step = (int64_t)gridDim.x * spanRows;
    int64_t row0 = (int64_t)blockIdx.x * spanRows;
    auto span = [&](int64_t r0) {
        return Span<T>(static_cast<const T*>(a.x), total, r0 * dim, (int)min((int64_t)spanRows, a.rows - r0) * dim);
    };
    if (row0 < a.rows) {
        span(row0).load(raw);
    }
    for (; row0 < a.rows; row0 += step) {
        const Span<T> here = span(row0);
        const int rows = (int)min((int64_t)spanRows, a.rows - row0);
        here.place(raw, lds);
        __syncthreads();
        if (row0 + step < a.rows) {
            span(row0 + step).load(raw);
        }
        for (int r0 = threadIdx.x / G; r0 < rows; r0 += R * kTeams) {
            float v[R][K];
            float mean[R];
            float rstd[R];
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const T* at = lds + here.lead + min(r0 + i * kTeams, rows - 1) * dim;
                mean[i] = 0.0f;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const float e = (float)at[min(k * G + lane, dim - 1)];
                    v[i][k] = k * G + lane < dim ? e : 0.0f;
                    mean[i] += v[i][k];
                }
            }
            team_sum<G>(mean, smem);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                mean[i] *= inv;
                rstd[i] = 0.0f;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    v[i][k] = k * G + lane < dim ? v[i][k] - mean[i] : 0.0f;
                    rstd[i] = __builtin_fmaf(v[i][k], v[i][k], rstd[i]);
                }
            }
            team_sum<G>(rstd, smem);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int r = r0 + i * kTeams;
                if (r >= rows) {
                    break;
                }
                T* at = lds + here.lead + r * dim;
                rstd[i] = 1.0f / sqrtf(rstd[i] * inv + a.eps);
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if (k * G + lane < dim) {
                        at[k * G + lane] = from_float<T>(__builtin_fmaf(v[i][k] * rstd[i], wt[k][0], bs[k][0]));
                    }
                }
                if (lane == 0 && a.mean != nullptr) {
                    a.mean[row0 + r] = mean[i];
                    a.rstd[row0 + r] = rstd[i];
                }
            }
        }
        __syncthreads();
        here.store(lds, static_cast<T*>(a.y) + row0 * dim);
        __syncthreads();
    }
}

template <typename T, typename W, int G, int K>
__global__ __launch_bounds__(kBlock) void k_layer_norm_backward_staged(NormRows a, int spanRows)
{
    constexpr int kTeams = kBlock / G;
    constexpr int R = G > kWave || K > 8 ? 1 : 2;
    __shared__ __attribute__((aligned(16))) T lds[2][kSpanBytes / sizeof(T)];
    __shared__ float stats[2][kSpanRows];
    __shared__ float smem[G > kWave ? 2 * R * G / kWave : 1];
    static_assert(kTeams == 1 || kTeams * G * K * sizeof(float) <= 2 * kSpanBytes, "the teams' sums fit the span's LDS");
    const int dim = a.dim;
    const int lane = threadIdx.x % G;
    const int64_t total = a.rows * dim;
    float wt[K][1];
    float dw[K][1];
    float db[K][1];
    params<W, 1, K>(a.weight, lane, G, dim, 1.0f, wt);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        dw[k][0] = 0.0f;
        db[k][0] = 0.0f;
    }
    const float inv = 1.0f / (float)dim;
    Word4 rawX[kSpanLoads];
    Word4 rawG[kSpanLoads];
    const int64_t step = (int64_t)gridDim.x * spanRows;
    int64_t row0 = (int64_t)blockIdx.x * spanRows;
    auto span = [&](const void* p, int64_t r0) {
        return Span<T>(static_cast<const T*>(p), total, r0 * dim, (int)min((int64_t)spanRows, a.rows - r0) * dim);
    };
    float rawMean = 0.0f;
    float rawRstd = 0.0f;
    auto fetch = [&](int64_t r0) {
        span(a.x, r0).load(rawX);
        span(a.grad, r0).load(rawG);
        const int64_t r = min(r0 + (int)threadIdx.x, a.rows - 1);
        rawMean = a.mean[r];
        rawRstd = a.rstd[r];
    };
    if (row0 < a.rows) {
        fetch(row0);
    }
    for (; row0 < a.rows; row0 += step) {
        const Span<T> sx = span(a.x, row0);
        const Span<T> sg = span(a.grad, row0);
        const int rows = (int)min((int64_t)spanRows, a.rows - row0);
        sx.place(rawX, lds[0]);
        sg.place(rawG, lds[1]);
        stats[0][threadIdx.x] = rawMean;
        stats[1][threadIdx.x] = rawRstd;
        __syncthreads();
        if (row0 + step < a.rows) {
            fetch(row0 + step);
        }
        for (int r0 = threadIdx.x / G; r0 < rows; r0 += R * kTeams) {
            float hat[R][K];
            float g[R][K];
            float s[2 * R];
            float rstd[R];
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const bool here = r0 + i * kTeams < rows;
                const int r = here ? r0 + i * kTeams : r0;
                const T* x = lds[0] + sx.lead + r * dim;
                const T* dy = lds[1] + sg.lead + r * dim;
                const float mean = stats[0][r];
                rstd[i] = stats[1][r];
                s[2 * i] = 0.0f;
                s[2 * i + 1] = 0.0f;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const bool in = k * G + lane < dim && here;
                    const int c = min(k * G + lane, dim - 1);
                    const float ex = (float)x[c];
                    const float eg = (float)dy[c];
                    hat[i][k] = in ? (ex - mean) * rstd[i] : 0.0f;
                    const float d = in ? eg : 0.0f;
                    dw[k][0] = __builtin_fmaf(d, hat[i][k], dw[k][0]);
                    db[k][0] += d;
                    g[i][k] = d * wt[k][0];
                    s[2 * i] += g[i][k];
                    s[2 * i + 1] = __builtin_fmaf(g[i][k], hat[i][k], s[2 * i + 1]);
                }
            }
            if (a.dx != nullptr) {
                team_sum<G>(s, smem);
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    if (r0 + i * kTeams >= rows) {
                        break;
                    }
                    T* dy = lds[1] + sg.lead + (r0 + i * kTeams) * dim;
                    const float s0 = s[2 * i] * inv;
                    const float s1 = s[2 * i + 1] * inv;
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        if (k * G + lane < dim) {
                            dy[k * G + lane] = from_float<T>(rstd[i] * (g[i][k] - s0 - hat[i][k] * s1));
                        }
                    }
                }
            }
        }
        __syncthreads();
        if (a.dx != nullptr) {
            sg.store(lds[1], static_cast<T*>(a.dx) + row0 * dim);
            __syncthreads();
        }
    }
    if (a.part != nullptr) {
        leave_parts<1, G, K, kTeams>(a, reinterpret_cast<float*>(&lds[0][0]), dw, db);
    }
}

// Rows too wide for registers: the block walks its row three times (mean, variance, result), from L2 after the first.
template <typename T, typename W>
__global__ __launch_bounds__(1024) void k_layer_norm_wide(NormRows a)
{
    __shared__ float smem[32];
    const float inv = 1.0f / (float)a.dim;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + row * a.stride;
        T* y = static_cast<T*>(a.y) + row * a.dim;
        float sum[1] = {0.0f};
        for (int c = threadIdx.x; c < a.dim; c += 1024) {
            sum[0] += (float)x[c];
        }
        team_sum<1024>(sum, smem);
        const float mean = sum[0] * inv;
        sum[0] = 0.0f;
        for (int c = threadIdx.x; c < a.dim; c += 1024) {
            const float d = (float)x[c] - mean;
            sum[0] = __builtin_fmaf(d, d, sum[0]);
        }
        team_sum<1024>(sum, smem);
        const float rstd = 1.0f / sqrtf(sum[0] * inv + a.eps);
        for (int c = threadIdx.x; c < a.dim; c += 1024) {
            y[c] = from_float<T>(__builtin_fmaf(((float)x[c] - mean) * rstd, param<W>(a.weight, c, 1.0f),
                                                param<W>(a.bias, c, 0.0f)));
        }
        if (threadIdx.x == 0 && a.mean != nullptr) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
    }
}

template <typename T, typename W>
__global__ __launch_bounds__(1024) void k_layer_norm_wide_dx(NormRows a)
{
    __shared__ float smem[32];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + row * a.stride;
        const T* dy = static_cast<const T*>(a.grad) + row * a.dim;
        T* dx = static_cast<T*>(a.dx) + row * a.dim;
        const float mean = a.mean[row];
        const float rstd = a.rstd[row];
        float s[2] = {0.0f, 0.0f};
        for (int c = threadIdx.x; c < a.dim; c += 1024) {
            const float g = (float)dy[c] * param<W>(a.weight, c, 1.0f);
            s[0] += g;
            s[1] = __builtin_fmaf(g, ((float)x[c] - mean) * rstd, s[1]);
        }
        team_sum<1024>(s, smem);
        const float s0 = s[0] / (float)a.dim;
        const float s1 = s[1] / (float)a.dim;
        for (int c = threadIdx.x; c < a.dim; c += 1024) {
            const float g = (float)dy[c] * param<W>(a.weight, c, 1.0f);
            dx[c] = from_float<T>(rstd * (g - s0 - ((float)x[c] - mean) * rstd * s1));
        }
    }
}

// dweight and dbias of wide rows: one column per thread, blockIdx.y takes every gridDim.y-th row.
template <typename T>
__global__ __launch_bounds__(kBlock) void k_layer_norm_wide_params(NormRows a)
{
    const int c = blockIdx.x * kBlock + threadIdx.x;
    if (c >= a.dim) {
        return;
    }
    float dw = 0.0f;
    float db = 0.0f;
    for (int64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
        const float d = (float)static_cast<const T*>(a.grad)[r * a.dim + c];
        const float hat = ((float)static_cast<const T*>(a.x)[r * a.stride + c] - a.mean[r]) * a.rstd[r];
        dw = __builtin_fmaf(d, hat, dw);
        db += d;
    }
    float* part = a.part + (int64_t)blockIdx.y * 2 * a.dim;
    part[c] = dw;
    part[a.dim + c] = db;
}

// dweight / dbias = sums of the blocks' parts, in the order of the blocks inside each of the kReduceWaves strides.
template <typename W>
__global__ __launch_bounds__(kWave* kReduceWaves) void k_layer_norm_join(const float* __restrict__ part, int blocks, int dim,
                                                                         W* __restrict__ dweight, W* __restrict__ dbias)
{
    __shared__ float sums[kReduceWaves][kReduceCols];
    const int wave = threadIdx.x / kWave;
    const int c = blockIdx.x * kReduceCols + lane_id();
    float s = 0.0f;
    if (c < 2 * dim) {
#pragma unroll 8
        for (int b = wave; b < blocks; b += kReduceWaves) {
            s += part[(int64_t)b * 2 * dim + c];
        }
    }
    sums[wave][lane_id()] = s;
    __syncthreads();
    if (wave == 0 && c < 2 * dim) {
        s = 0.0f;
#pragma unroll
        for (int w = 0; w < kReduceWaves; ++w) {
            s += sums[w][lane_id()];
        }
        W* out = c < dim ? dweight : dbias;
        if (out != nullptr) {
            out[c < dim ? c : c - dim] = from_float<W>(s);
        }
    }
}

// How a row is cut.  kWhole: packs of 16 bytes, every row on their borders; kStaged: contiguous rows that are not (every buffer's
// first row equally far behind a border); kSingle: element by element, for rows with gaps that are not; kWide: rows past what
// those hold in registers or LDS.
enum NormCut { kWhole, kStaged, kSingle, kWide };

template <typename T>
static NormCut norm_cut(const NormRows& a)
{
    constexpr int kPer = 16 / (int)sizeof(T);
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.x) % 16;
    bool alike = at % sizeof(T) == 0;
    for (const void* p : {static_cast<const void*>(a.y), a.grad, static_cast<const void*>(a.dx)}) {
        alike = alike && (p == nullptr || reinterpret_cast<uintptr_t>(p) % 16 == at);
    }
    if (alike && at == 0 && a.dim % kPer == 0 && a.stride % kPer == 0 && aligned16(a.weight) && aligned16(a.bias)) {
        return a.dim <= 2048 * kPer ? kWhole : kWide;
    }
    // a span and the elements between it and the borders at its ends
    if (alike && (a.stride == a.dim || a.rows == 1) && ((int64_t)a.dim + 2 * kPer) * (int)sizeof(T) <= kSpanBytes) {
        return kStaged;
    }
    return a.dim <= 4096 ? kSingle : kWide;
}

static int norm_backward_blocks(int64_t rows, int rowsPerBlock, int most)
{
    const int64_t want = cdiv(rows, rowsPerBlock);
    return (int)(want < most ? want : most);
}

template <typename T, typename W, int E, int G, int K, bool BACK>
static int launch_norm(const NormRows& a, int* blocks, hipStream_t stream)
{
    constexpr int kThreads = G > kBlock ? G : kBlock;
    constexpr int kRows = kThreads / G * kNormRows<G, K, BACK>;
    *blocks = norm_backward_blocks(a.rows, kRows, BACK ? kNormRowBlocks : kNormForwardBlocks);
    if constexpr (BACK) {
        RECSDK_LAUNCH_AS("k_layer_norm_backward", (k_layer_norm_backward<T, W, E, G, K>), dim3((unsigned)*blocks), dim3(kThreads),
                         stream, a);
    } else {
        RECSDK_LAUNCH_AS("k_layer_norm", (k_layer_norm<T, W, E, G, K>), dim3((unsigned)*blocks), dim3(kThreads), stream, a);
    }
    return RECSDK_OK;
}

// 16 to 32 values per thread at most: the backward pass keeps five values per column and has to stay within the registers
// of a block of 512 threads.
template <typename T, typename W, bool BACK>
static int launch_whole(const NormRows& a, int* blocks, hipStream_t stream)
{
    constexpr int E = 16 / (int)sizeof(T);
    const int packs = a.dim / E;
    if (packs <= 4) {
        return launch_norm<T, W, E, 4, 1, BACK>(a, blocks, stream);
    }
    if (packs <= 8) {
        return launch_norm<T, W, E, 8, 1, BACK>(a, blocks, stream);
    }
    if (packs <= 16) {
        return launch_norm<T, W, E, 16, 1, BACK>(a, blocks, stream);
    }
    if (packs <= 32) {
        return launch_norm<T, W, E, 32, 1, BACK>(a, blocks, stream);
    }
    if (packs <= 64) {
        return launch_norm<T, W, E, 64, 1, BACK>(a, blocks, stream);
    }
    if (packs <= 128) {
        return launch_norm<T, W, E, 64, 2, BACK>(a, blocks, stream);
    }
    if (packs <= 256) {
        return launch_norm<T, W, E, 64, 4, BACK>(a, blocks, stream);
    }
    if (packs <= 1024) {
        return launch_norm<T, W, E, 256, 4, BACK>(a, blocks, stream);
    }
    return launch_norm<T, W, E, 512, 4, BACK>(a, blocks, stream);
}

template <typename T, typename W, int G, int K, bool BACK>
static int launch_spans(const NormRows& a, int* blocks, hipStream_t stream)
{
    constexpr int kPer = 16 / (int)sizeof(T);
    const int fit = (kSpanBytes / (int)sizeof(T) - 2 * kPer) / a.dim;
    const int spanRows = fit < kSpanRows ? fit : kSpanRows;
    *blocks = norm_backward_blocks(a.rows, spanRows, BACK ? kNormBlocks : kNormSpanBlocks);
    if constexpr (BACK) {
        RECSDK_LAUNCH_AS("k_layer_norm_backward", (k_layer_norm_backward_staged<T, W, G, K>), dim3((unsigned)*blocks), dim3(kBlock),
                         stream, a, spanRows);
    } else {
        RECSDK_LAUNCH_AS("k_layer_norm", (k_layer_norm_staged<T, W, G, K>), dim3((unsigned)*blocks), dim3(kBlock), stream, a,
                         spanRows);
    }
    return RECSDK_OK;
}

template <typename T, typename W, bool BACK>
static int launch_staged(const NormRows& a, int* blocks, hipStream_t stream)
{
    if (a.dim <= 16) {
        return launch_spans<T, W, 4, 4, BACK>(a, blocks, stream);
    }
    if (a.dim <= 64) {
        return launch_spans<T, W, 16, 4, BACK>(a, blocks, stream);
    }
    if (a.dim <= 128) {
        return launch_spans<T, W, 16, 8, BACK>(a, blocks, stream);
    }
    if (a.dim <= 256) {
        return launch_spans<T, W, 32, 8, BACK>(a, blocks, stream);
    }
    if (a.dim <= 512) {
        return launch_spans<T, W, 64, 8, BACK>(a, blocks, stream);
    }
    if (a.dim <= 1024) {
        return launch_spans<T, W, 64, 16, BACK>(a, blocks, stream);
    }
    if (a.dim <= 4096) {
        return launch_spans<T, W, 256, 16, BACK>(a, blocks, stream);
    }
    return launch_spans<T, W, 256, 32, BACK>(a, blocks, stream);
}

template <typename T, typename W, bool BACK>
static int launch_wide(const NormRows& a, int* blocks, hipStream_t stream)
{
    const dim3 grid((unsigned)(a.rows < kNormWideBlocks ? a.rows : kNormWideBlocks));
    if constexpr (BACK) {
        if (a.dx != nullptr) {
            RECSDK_LAUNCH_AS("k_layer_norm_wide_dx", (k_layer_norm_wide_dx<T, W>), grid, dim3(1024), stream, a);
        }
        if (a.part != nullptr) {
            *blocks = norm_backward_blocks(a.rows, 16, kNormBlocks);
            RECSDK_LAUNCH_AS("k_layer_norm_wide_params", (k_layer_norm_wide_params<T>),
                             dim3((unsigned)cdiv(a.dim, kBlock), (unsigned)*blocks), dim3(kBlock), stream, a);
        }
    } else {
        RECSDK_LAUNCH_AS("k_layer_norm_wide", (k_layer_norm_wide<T, W>), grid, dim3(1024), stream, a);
    }
    return RECSDK_OK;
}

template <typename T, typename W, bool BACK>
static int launch_rows(const NormRows& a, int* blocks, hipStream_t stream)
{
    switch (norm_cut<T>(a)) {
        case kWhole:
            return launch_whole<T, W, BACK>(a, blocks, stream);
        case kStaged:
            return launch_staged<T, W, BACK>(a, blocks, stream);
        case kSingle:
            return a.dim <= 256    ? launch_norm<T, W, 1, 64, 4, BACK>(a, blocks, stream)
                   : a.dim <= 1024 ? launch_norm<T, W, 1, 64, 16, BACK>(a, blocks, stream)
                                   : launch_norm<T, W, 1, 256, 16, BACK>(a, blocks, stream);
        default:
            return launch_wide<T, W, BACK>(a, blocks, stream);
    }
}

template <typename T, typename W, bool BACK>
static int run_norm_typed(const NormRows& a, void* dweight, void* dbias, hipStream_t stream)
{
    int blocks = 0;
    if (a.rows > 0) {
        const int rc = launch_rows<T, W, BACK>(a, &blocks, stream);
        if (rc != RECSDK_OK) {
            return rc;
        }
    }
    if (BACK && (dweight != nullptr || dbias != nullptr)) {
        RECSDK_LAUNCH_AS("k_layer_norm_join", (k_layer_norm_join<W>), dim3((unsigned)cdiv(2 * (int64_t)a.dim, kReduceCols)),
                         dim3(kWave * kReduceWaves), stream, a.part, blocks, a.dim, static_cast<W*>(dweight),
                         static_cast<W*>(dbias));
    }
    return RECSDK_OK;
}

template <bool BACK>
static int run_norm(const NormRows& a, int32_t dtype, int32_t w_dtype, void* dweight, void* dbias, hipStream_t stream)
{
    if (dtype == RECSDK_DT_F32) {
        return run_norm_typed<float, float, BACK>(a, dweight, dbias, stream);
    }
    if (dtype == RECSDK_DT_F16) {
        return w_dtype == RECSDK_DT_F32 ? run_norm_typed<F16, float, BACK>(a, dweight, dbias, stream)
                                        : run_norm_typed<F16, F16, BACK>(a, dweight, dbias, stream);
    }
    return w_dtype == RECSDK_DT_F32 ? run_norm_typed<BF16, float, BACK>(a, dweight, dbias, stream)
                                    : run_norm_typed<BF16, BF16, BACK>(a, dweight, dbias, stream);
}

static int check_norm(const char* name, int64_t rows, int32_t dim, int64_t x_stride, int32_t dtype, int32_t w_dtype)
{
    if (float_bytes(dtype) == 0) {
        set_error("%s: dtype must be fp32, fp16 or bf16", name);
        return RECSDK_EINVAL;
    }
    if (w_dtype != RECSDK_DT_F32 && w_dtype != dtype) {
        set_error("%s: weight and bias must be fp32 or of the rows' type", name);
        return RECSDK_EINVAL;
    }
    if (dim < 1 || dim >= (1 << 30) || rows < 0 || rows >= (int64_t(1) << 31)) {
        set_error("%s: dim must lie in [1, 2^30) and rows in [0, 2^31)", name);
        return RECSDK_EINVAL;
    }
    if (x_stride < dim) {
        set_error("%s: rows of x overlap (x_stride < dim)", name);
        return RECSDK_EINVAL;
    }
    return RECSDK_OK;
}

}  // namespace recsdk

extern "C" int recsdk_layer_norm_forward(const void* d_x, int64_t rows, int32_t dim, int64_t x_stride, int32_t dtype,
                                         const void* d_weight, const void* d_bias, int32_t w_dtype, float eps, void* d_y,
                                         float* d_mean, float* d_rstd, void* stream)
{
    using namespace recsdk;
    const int rc = check_norm("recsdk_layer_norm_forward", rows, dim, x_stride, dtype, w_dtype);
    if (rc != RECSDK_OK) {
        return rc;
    }
    RECSDK_REQUIRE(eps >= 0.0f, RECSDK_EINVAL, "recsdk_layer_norm_forward: eps must not be negative");
    RECSDK_REQUIRE((d_mean == nullptr) == (d_rstd == nullptr), RECSDK_EINVAL,
                   "recsdk_layer_norm_forward: mean and rstd are given together or not at all");
    if (rows == 0) {
        return RECSDK_OK;
    }
    RECSDK_REQUIRE(d_x != nullptr && d_y != nullptr, RECSDK_ENULL, "recsdk_layer_norm_forward: NULL argument");
    NormRows a{};
    a.x = d_x;
    a.stride = x_stride;
    a.rows = rows;
    a.dim = dim;
    a.weight = d_weight;
    a.bias = d_bias;
    a.eps = eps;
    a.mean = d_mean;
    a.rstd = d_rstd;
    a.y = d_y;
    return run_norm<false>(a, dtype, w_dtype, nullptr, nullptr, static_cast<hipStream_t>(stream));
}

extern "C" int recsdk_layer_norm_workspace(int64_t rows, int32_t dim, int64_t* h_bytes)
{
    using namespace recsdk;
    RECSDK_REQUIRE(h_bytes != nullptr, RECSDK_ENULL, "recsdk_layer_norm_workspace: NULL argument");
    RECSDK_REQUIRE(rows >= 0 && dim >= 1 && dim < (1 << 30), RECSDK_EINVAL, "recsdk_layer_norm_workspace: bad sizes");
    *h_bytes = (int64_t)norm_backward_blocks(rows, 1, kNormBlocks) * 2 * dim * (int64_t)sizeof(float);
    return RECSDK_OK;
}

extern "C" int recsdk_layer_norm_backward(const void* d_grad, const void* d_x, int64_t rows, int32_t dim, int64_t x_stride,
                                          int32_t dtype, const void* d_weight, int32_t w_dtype, const float* d_mean,
                                          const float* d_rstd, void* d_dx, void* d_dweight, void* d_dbias,
                                          void* d_workspace, int64_t workspace_bytes, void* stream)
{
    using namespace recsdk;
    const int rc = check_norm("recsdk_layer_norm_backward", rows, dim, x_stride, dtype, w_dtype);
    if (rc != RECSDK_OK) {
        return rc;
    }
    const bool params = d_dweight != nullptr || d_dbias != nullptr;
    RECSDK_REQUIRE(rows == 0 || (d_grad != nullptr && d_x != nullptr && d_mean != nullptr && d_rstd != nullptr), RECSDK_ENULL,
                   "recsdk_layer_norm_backward: NULL argument");
    if (params && rows > 0) {
        int64_t need = 0;
        recsdk_layer_norm_workspace(rows, dim, &need);
        RECSDK_REQUIRE(d_workspace != nullptr && workspace_bytes >= need, RECSDK_ECAPACITY,
                       "recsdk_layer_norm_backward: the workspace is smaller than recsdk_layer_norm_workspace says");
        RECSDK_REQUIRE(aligned16(d_workspace), RECSDK_EINVAL, "recsdk_layer_norm_backward: the workspace must be 16-byte aligned");
    }
    if (!params && (d_dx == nullptr || rows == 0)) {
        return RECSDK_OK;
    }
    NormRows a{};
    a.x = d_x;
    a.stride = x_stride;
    a.rows = rows;
    a.dim = dim;
    a.weight = d_weight;
    a.mean = const_cast<float*>(d_mean);
    a.rstd = const_cast<float*>(d_rstd);
    a.grad = d_grad;
    a.dx = d_dx;
    a.part = params ? static_cast<float*>(d_workspace) : nullptr;
    return run_norm<true>(a, dtype, w_dtype, d_dweight, d_dbias, static_cast<hipStream_t>(stream));
}
