// Layer norm over the columns of a row, forward and backward.
//
//   forward    mean = sum x / D,  var = sum (x - mean)^2 / D,  rstd = 1 / sqrt(var + eps),  hat = (x - mean) rstd
//              y = hat weight + bias
//   backward   g = dy weight;  dx = rstd (g - sum g / D - hat sum (g hat) / D);  dweight = sum_rows dy hat;  dbias = sum_rows dy
//
// Rows are held in registers between their one read and their one write: a team of G threads per row, every thread K
// packs of E columns (16 bytes where the rows are aligned to that, single elements where they are not), the variance
// from the differences and not from the squares.  A team walks rows at a fixed stride, keeps its columns of weight and
// bias in registers and has the next row's loads in flight while it reduces the present one.  In the backward pass the
// same threads sum their columns of dweight and dbias over the team's rows; the teams of a block are joined in LDS, the
// blocks' sums go to the workspace and a second kernel adds them in the order of the blocks: no atomics, so a call
// gives the same bits every time.  All sums are held in 32 bits; every result is rounded once.
// What bounds it: the row traffic (read x, write y; read dy and x, write dx).
#include <math.h>

#include "dense.h"

namespace recsdk {

constexpr int kNormBlocks = 512;        // blocks of the backward pass at most: each leaves 2 D sums in the workspace
constexpr int kNormForwardBlocks = 2048;
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

// Sum over the G threads of a team.  G > 64: the team is the block, `smem` holds two floats per wave.
template <int G>
__device__ __forceinline__ void team_sum2(float& a, float& b, float* smem)
{
#pragma unroll
    for (int d = (G < kWave ? G : kWave) / 2; d > 0; d >>= 1) {
        a += __shfl_xor(a, d, kWave);
        b += __shfl_xor(b, d, kWave);
    }
    if constexpr (G > kWave) {
        constexpr int kWaves = G / kWave;
        const int w = threadIdx.x / kWave;
        __syncthreads();   // the previous sums have been read
        if (lane_id() == 0) {
            smem[2 * w] = a;
            smem[2 * w + 1] = b;
        }
        __syncthreads();
        a = 0;
        b = 0;
#pragma unroll
        for (int k = 0; k < kWaves; ++k) {
            a += smem[2 * k];
            b += smem[2 * k + 1];
        }
    }
}

template <typename W>
__device__ __forceinline__ float param(const void* p, int64_t c, float none)
{
    return p != nullptr ? (float)static_cast<const W*>(p)[c] : none;
}

template <typename T, typename W, int E, int G, int K>
__global__ __launch_bounds__(G > kBlock ? G : kBlock) void k_layer_norm(NormRows a)
{
    constexpr int kTeams = G > kBlock ? 1 : kBlock / G;
    __shared__ float smem[2 * (G > kWave ? G / kWave : 1)];
    const int lane = threadIdx.x % G;
    const int64_t teams = (int64_t)gridDim.x * kTeams;
    int64_t row = (int64_t)blockIdx.x * kTeams + threadIdx.x / G;
    if (G <= kWave && row >= a.rows) {
        return;
    }
    const int dim = a.dim;
    float wt[K][E];
    float bs[K][E];
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int c = (k * G + lane) * E + e;
            wt[k][e] = c < dim ? param<W>(a.weight, c, 1.0f) : 0.0f;
            bs[k][e] = c < dim ? param<W>(a.bias, c, 0.0f) : 0.0f;
        }
    }
    const T* x = static_cast<const T*>(a.x);
    T* y = static_cast<T*>(a.y);
    const float inv = 1.0f / (float)dim;
    Pack<T, E> next[K];
    auto fetch = [&](int64_t r) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * G + lane) * E;
            if (c < dim) {
                next[k] = load_pack<T, E>(x + r * a.stride + c);
            }
        }
    };
    if (row < a.rows) {
        fetch(row);
    }
    for (; row < a.rows; row += teams) {
        float v[K][E];
        float sum = 0.0f;
        float none = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const bool in = (k * G + lane) * E < dim;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                v[k][e] = in ? (float)next[k].v[e] : 0.0f;
                sum += v[k][e];
            }
        }
        if (row + teams < a.rows) {
            fetch(row + teams);
        }
        team_sum2<G>(sum, none, smem);
        const float mean = sum * inv;
        float sq = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const bool in = (k * G + lane) * E < dim;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                v[k][e] = in ? v[k][e] - mean : 0.0f;
                sq = __builtin_fmaf(v[k][e], v[k][e], sq);
            }
        }
        team_sum2<G>(sq, none, smem);
        const float rstd = 1.0f / sqrtf(sq * inv + a.eps);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * G + lane) * E;
            if (c < dim) {
                Pack<T, E> out;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    out.v[e] = from_float<T>(__builtin_fmaf(v[k][e] * rstd, wt[k][e], bs[k][e]));
                }
                store_pack<T, E>(y + row * dim + c, out);
            }
        }
        if (lane == 0 && a.mean != nullptr) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
    }
}

template <typename T, typename W, int E, int G, int K>
__global__ __launch_bounds__(G > kBlock ? G : kBlock) void k_layer_norm_backward(NormRows a)
{
    constexpr int kThreads = G > kBlock ? G : kBlock;
    constexpr int kTeams = kThreads / G;
    constexpr int kCols = G * K * E;   // columns a team covers
    // the teams' column sums, joined at the end (one team per block: nothing to join)
    __shared__ float joined[kTeams > 1 ? (kTeams * kCols > 8192 ? 8192 : kTeams * kCols) : 1];
    __shared__ float smem[2 * (G > kWave ? G / kWave : 1)];
    const int lane = threadIdx.x % G;
    const int team = threadIdx.x / G;
    const int64_t teams = (int64_t)gridDim.x * kTeams;
    const int dim = a.dim;
    const float inv = 1.0f / (float)dim;
    const T* x = static_cast<const T*>(a.x);
    const T* dy = static_cast<const T*>(a.grad);
    T* dx = static_cast<T*>(a.dx);
    float wt[K][E];
    float dw[K][E];
    float db[K][E];
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int c = (k * G + lane) * E + e;
            wt[k][e] = c < dim ? param<W>(a.weight, c, 1.0f) : 0.0f;
            dw[k][e] = 0.0f;
            db[k][e] = 0.0f;
        }
    }
    Pack<T, E> nx[K];
    Pack<T, E> ng[K];
    float nmean = 0.0f;
    float nrstd = 0.0f;
    auto fetch = [&](int64_t r) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * G + lane) * E;
            if (c < dim) {
                nx[k] = load_pack<T, E>(x + r * a.stride + c);
                ng[k] = load_pack<T, E>(dy + r * dim + c);
            }
        }
        nmean = a.mean[r];
        nrstd = a.rstd[r];
    };
    int64_t row = (int64_t)blockIdx.x * kTeams + team;
    if (row < a.rows) {
        fetch(row);
    }
    for (; row < a.rows; row += teams) {
        float hat[K][E];
        float g[K][E];
        const float rstd = nrstd;
        float s0 = 0.0f;
        float s1 = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const bool in = (k * G + lane) * E < dim;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                hat[k][e] = in ? ((float)nx[k].v[e] - nmean) * rstd : 0.0f;
                const float d = in ? (float)ng[k].v[e] : 0.0f;
                dw[k][e] = __builtin_fmaf(d, hat[k][e], dw[k][e]);
                db[k][e] += d;
                g[k][e] = d * wt[k][e];
                s0 += g[k][e];
                s1 = __builtin_fmaf(g[k][e], hat[k][e], s1);
            }
        }
        if (row + teams < a.rows) {
            fetch(row + teams);
        }
        if (dx != nullptr) {
            team_sum2<G>(s0, s1, smem);
            s0 *= inv;
            s1 *= inv;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int c = (k * G + lane) * E;
                if (c < dim) {
                    Pack<T, E> out;
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        out.v[e] = from_float<T>(rstd * (g[k][e] - s0 - hat[k][e] * s1));
                    }
                    store_pack<T, E>(dx + row * dim + c, out);
                }
            }
        }
    }
    if (a.part == nullptr) {
        return;
    }
    float* part = a.part + (int64_t)blockIdx.x * 2 * dim;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if constexpr (kTeams == 1) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int c = (k * G + lane) * E + e;
                    if (c < dim) {
                        part[which * dim + c] = which == 0 ? dw[k][e] : db[k][e];
                    }
                }
            }
        } else {
            static_assert(kTeams * kCols <= 8192, "the teams' sums fit the LDS array");
            __syncthreads();
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    joined[team * kCols + (k * G + lane) * E + e] = which == 0 ? dw[k][e] : db[k][e];
                }
            }
            __syncthreads();
            for (int c = threadIdx.x; c < dim; c += kThreads) {
                float s = 0.0f;
#pragma unroll
                for (int t = 0; t < kTeams; ++t) {
                    s += joined[t * kCols + c];
                }
                part[which * dim + c] = s;
            }
        }
    }
}

// Rows too wide for registers: the block walks its row three times (mean, variance, result), from L2 after the first.
template <typename T, typename W>
__global__ __launch_bounds__(1024) void k_layer_norm_wide(NormRows a)
{
    __shared__ float smem[32];
    const T* x = static_cast<const T*>(a.x) + (int64_t)blockIdx.x * a.stride;
    T* y = static_cast<T*>(a.y) + (int64_t)blockIdx.x * a.dim;
    const float inv = 1.0f / (float)a.dim;
    float sum = 0.0f;
    float none = 0.0f;
    for (int c = threadIdx.x; c < a.dim; c += 1024) {
        sum += (float)x[c];
    }
    team_sum2<1024>(sum, none, smem);
    const float mean = sum * inv;
    float sq = 0.0f;
    for (int c = threadIdx.x; c < a.dim; c += 1024) {
        const float d = (float)x[c] - mean;
        sq = __builtin_fmaf(d, d, sq);
    }
    team_sum2<1024>(sq, none, smem);
    const float rstd = 1.0f / sqrtf(sq * inv + a.eps);
    for (int c = threadIdx.x; c < a.dim; c += 1024) {
        y[c] = from_float<T>(__builtin_fmaf(((float)x[c] - mean) * rstd, param<W>(a.weight, c, 1.0f),
                                            param<W>(a.bias, c, 0.0f)));
    }
    if (threadIdx.x == 0 && a.mean != nullptr) {
        a.mean[blockIdx.x] = mean;
        a.rstd[blockIdx.x] = rstd;
    }
}

template <typename T, typename W>
__global__ __launch_bounds__(1024) void k_layer_norm_wide_dx(NormRows a)
{
    __shared__ float smem[32];
    const T* x = static_cast<const T*>(a.x) + (int64_t)blockIdx.x * a.stride;
    const T* dy = static_cast<const T*>(a.grad) + (int64_t)blockIdx.x * a.dim;
    T* dx = static_cast<T*>(a.dx) + (int64_t)blockIdx.x * a.dim;
    const float mean = a.mean[blockIdx.x];
    const float rstd = a.rstd[blockIdx.x];
    float s0 = 0.0f;
    float s1 = 0.0f;
    for (int c = threadIdx.x; c < a.dim; c += 1024) {
        const float g = (float)dy[c] * param<W>(a.weight, c, 1.0f);
        s0 += g;
        s1 = __builtin_fmaf(g, ((float)x[c] - mean) * rstd, s1);
    }
    team_sum2<1024>(s0, s1, smem);
    s0 /= (float)a.dim;
    s1 /= (float)a.dim;
    for (int c = threadIdx.x; c < a.dim; c += 1024) {
        const float g = (float)dy[c] * param<W>(a.weight, c, 1.0f);
        dx[c] = from_float<T>(rstd * (g - s0 - ((float)x[c] - mean) * rstd * s1));
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

// What a row takes: threads per team and packs per thread, for packs of E elements; 0 threads = too wide.
struct NormShape {
    int team;
    int packs;
};

static NormShape norm_shape(int dim, int e)
{
    const int packs = (int)cdiv(dim, e);
    const int most = e == 1 ? 16 : 4;   // packs per thread: 16 to 32 values
    if (packs <= 8) {
        return {8, 1};
    }
    if (packs <= 16) {
        return {16, 1};
    }
    if (packs <= 32) {
        return {32, 1};
    }
    for (int k = 1; k <= most; k *= 2) {
        if (packs <= 64 * k) {
            return {64, k};
        }
    }
    if (packs <= 256 * most) {
        return {256, most};
    }
    if (packs <= 1024 * most) {
        return {1024, most};
    }
    return {0, 0};
}

// Elements per access: whole 16 bytes where every row of every buffer starts on such a border.
template <typename T>
static int norm_pack(const NormRows& a)
{
    const int e = 16 / (int)sizeof(T);
    const bool ok = a.dim % e == 0 && a.stride % e == 0 && aligned16(a.x) && aligned16(a.y) && aligned16(a.grad) &&
                    aligned16(a.dx);
    return ok ? e : 1;
}

static int norm_backward_blocks(int64_t rows, int teamsPerBlock)
{
    const int64_t want = cdiv(rows, teamsPerBlock);
    return (int)(want < kNormBlocks ? want : kNormBlocks);
}

template <typename T, typename W, int E, int G, int K, bool BACK>
static int launch_norm(const NormRows& a, int* blocks, hipStream_t stream)
{
    constexpr int kThreads = G > kBlock ? G : kBlock;
    constexpr int kTeams = kThreads / G;
    if constexpr (BACK) {
        *blocks = norm_backward_blocks(a.rows, kTeams);
        RECSDK_LAUNCH_AS("k_layer_norm_backward", (k_layer_norm_backward<T, W, E, G, K>), dim3((unsigned)*blocks), dim3(kThreads),
                         stream, a);
    } else {
        const int64_t want = cdiv(a.rows, kTeams);
        *blocks = (int)(want < kNormForwardBlocks ? want : kNormForwardBlocks);
        RECSDK_LAUNCH_AS("k_layer_norm", (k_layer_norm<T, W, E, G, K>), dim3((unsigned)*blocks), dim3(kThreads), stream, a);
    }
    return RECSDK_OK;
}

template <typename T, typename W, int E, bool BACK>
static int dispatch_norm(const NormRows& a, int* blocks, hipStream_t stream)
{
    const NormShape s = norm_shape(a.dim, E);
    constexpr int kMost = E == 1 ? 16 : 4;
    switch (s.team) {
        case 8:
            return launch_norm<T, W, E, 8, 1, BACK>(a, blocks, stream);
        case 16:
            return launch_norm<T, W, E, 16, 1, BACK>(a, blocks, stream);
        case 32:
            return launch_norm<T, W, E, 32, 1, BACK>(a, blocks, stream);
        case 64:
            if (s.packs == 1) {
                return launch_norm<T, W, E, 64, 1, BACK>(a, blocks, stream);
            }
            if (s.packs == 2) {
                return launch_norm<T, W, E, 64, 2, BACK>(a, blocks, stream);
            }
            if (s.packs == 4) {
                return launch_norm<T, W, E, 64, 4, BACK>(a, blocks, stream);
            }
            if constexpr (E == 1) {
                if (s.packs == 8) {
                    return launch_norm<T, W, E, 64, 8, BACK>(a, blocks, stream);
                }
                return launch_norm<T, W, E, 64, 16, BACK>(a, blocks, stream);
            }
            break;
        case 256:
            return launch_norm<T, W, E, 256, kMost, BACK>(a, blocks, stream);
        case 1024:
            return launch_norm<T, W, E, 1024, kMost, BACK>(a, blocks, stream);
        default:
            break;
    }
    if constexpr (BACK) {
        if (a.dx != nullptr) {
            RECSDK_LAUNCH_AS("k_layer_norm_wide_dx", (k_layer_norm_wide_dx<T, W>), dim3((unsigned)a.rows), dim3(1024), stream, a);
        }
        if (a.part != nullptr) {
            *blocks = norm_backward_blocks(a.rows, 16);
            RECSDK_LAUNCH_AS("k_layer_norm_wide_params", (k_layer_norm_wide_params<T>),
                             dim3((unsigned)cdiv(a.dim, kBlock), (unsigned)*blocks), dim3(kBlock), stream, a);
        }
    } else {
        RECSDK_LAUNCH_AS("k_layer_norm_wide", (k_layer_norm_wide<T, W>), dim3((unsigned)a.rows), dim3(1024), stream, a);
    }
    return RECSDK_OK;
}

template <typename T, typename W, bool BACK>
static int run_norm_typed(const NormRows& a, void* dweight, void* dbias, hipStream_t stream)
{
    int blocks = 0;
    if (a.rows > 0) {
        const int rc = norm_pack<T>(a) == 1 ? dispatch_norm<T, W, 1, BACK>(a, &blocks, stream)
                                            : dispatch_norm<T, W, 16 / (int)sizeof(T), BACK>(a, &blocks, stream);
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
    if (dim < 1 || rows < 0 || rows >= (int64_t(1) << 31)) {
        set_error("%s: dim must be at least 1 and rows below 2^31", name);
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
    RECSDK_REQUIRE(rows >= 0 && dim >= 1, RECSDK_EINVAL, "recsdk_layer_norm_workspace: bad sizes");
    *h_bytes = (int64_t)norm_backward_blocks(rows, 1) * 2 * dim * (int64_t)sizeof(float);
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
