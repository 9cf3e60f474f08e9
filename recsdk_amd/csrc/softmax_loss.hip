// The softmax loss's entry points and the kernels around the tile kernels (softmax_tiles.h, where the method stands): joins of
// partial results, padded copies, largest values.
#include <algorithm>

#include "softmax_tiles.h"

namespace recsdk {

constexpr int kFewRows = 32;
constexpr int kAbsMaxThreads = 1024;
constexpr int kDirectDim = 8;
constexpr int kDirectRows = 4096;
constexpr int64_t kMostBlocks = 65536;   // of the kernels here, which walk what is more: a launch holds fewer than 2^32 threads

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
    const int lane = threadIdx.x % TEAM;
    for (int64_t n = (int64_t)blockIdx.x * (kBlock / TEAM) + threadIdx.x / TEAM; n < rows;
         n += (int64_t)gridDim.x * (kBlock / TEAM)) {
        const int64_t t = target[n];
        const bool inside = t >= 0 && t < items;
        const float b = inside && bias != nullptr ? bias[t] : 0.0f;
        if (!inside || b <= kMaskedBelow) {
            // no target: no loss; a target that is taken out: infinite; neither gives a gradient
            if (lane == 0) {
                loss[n] = inside ? INFINITY : 0.0f;
                lse[n] = INFINITY;
            }
            continue;   // the whole team
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
            __syncthreads();   // the previous row's have been read
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
    for (int64_t block = blockIdx.x; block * kWide * 4 < count; block += gridDim.x) {
        const int64_t i = (block * kWide + at) * 4;
        Float4 s = 0.0f;
        if (i < count) {
#pragma unroll 8
            for (int p = way; p < parts; p += WAYS) {
                s += *reinterpret_cast<const Float4*>(part + p * count + i);
            }
        }
        if constexpr (WAYS > 1) {
            __syncthreads();   // the previous block's sums have been read
            sums[way][at] = s;
            __syncthreads();
            if (way != 0) {
                continue;
            }
#pragma unroll
            for (int w = 1; w < WAYS; ++w) {
                s += sums[w][at];
            }
        }
        if (i >= count) {
            continue;
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
}

// Rows of `dim` elements at any stride -> rows of `padded` elements (whole 16-byte pieces), the rest zero.  32 threads take
// a row's pieces; the first blocks take x's rows, the others the table's, in one launch (301 x 30011 x 201: 5 us less).
template <typename T>
struct PadRows {
    const T* src;
    int64_t stride;
    int64_t rows;
    T* dst;
    int64_t blocks;   // 0: as they are
};

template <typename T>
__global__ __launch_bounds__(kBlock) void k_pad_rows(PadRows<T> x, PadRows<T> table, int dim, int padded)
{
    constexpr int kPer = 16 / sizeof(T);
    const bool second = blockIdx.x >= x.blocks;
    const PadRows<T> p = second ? table : x;
    const int64_t first = blockIdx.x - (second ? x.blocks : 0);
    for (int64_t r = first * (kBlock / 32) + threadIdx.x / 32; r < p.rows; r += p.blocks * (kBlock / 32)) {
        for (int c = threadIdx.x % 32 * kPer; c < padded; c += 32 * kPer) {
            Pack<T, kPer> v;
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                v.v[e] = c + e < dim ? p.src[r * p.stride + c + e] : from_float<T>(0.0f);
            }
            *reinterpret_cast<Pack<T, kPer>*>(p.dst + r * padded + c) = v;
        }
    }
}

// Largest finite |value| of x (the first kAbsMaxParts blocks) and of the table, a part per block.  Rows that take no part are
// left out: they may hold anything.  32 threads per row, 16 bytes each.
__global__ __launch_bounds__(kAbsMaxThreads) void k_abs_max(const float* __restrict__ x, int64_t xStride, int rows,
                                                    const float* __restrict__ table, int64_t tableStride, int items, int dim,
                                                    const int64_t* __restrict__ target, const float* __restrict__ bias,
                                                    float* __restrict__ parts)
{
    __shared__ float sums[kAbsMaxThreads / kWave];
    constexpr int kStep = kAbsMaxParts * (kAbsMaxThreads / 32);
    constexpr int kFlight = 4;   // rows whose loads are in flight at once
    typedef float Unaligned __attribute__((ext_vector_type(4), aligned(4)));
    const bool second = blockIdx.x >= kAbsMaxParts;
    const float* base = second ? table : x;
    const int64_t stride = second ? tableStride : xStride;
    const int count = second ? items : rows;
    float most = 0.0f;
    for (int r0 = blockIdx.x % kAbsMaxParts * (kAbsMaxThreads / 32) + threadIdx.x / 32; r0 < count; r0 += kFlight * kStep) {
        for (int at = threadIdx.x % 32 * 4; at < dim; at += 128) {
            const int c = dim < 4 ? at : min(at, dim - 4);   // a row's last four columns, where it ends inside a piece
            Float4 v[kFlight];
            bool live[kFlight];
#pragma unroll
            for (int q = 0; q < kFlight; ++q) {
                const int64_t r = min((int64_t)r0 + (int64_t)q * kStep, (int64_t)count - 1);
                v[q] = *reinterpret_cast<const Unaligned*>(base + r * stride + c);
                live[q] = second ? bias == nullptr || bias[r] > kMaskedBelow : (uint64_t)target[r] < (uint64_t)items;
            }
#pragma unroll
            for (int q = 0; q < kFlight; ++q) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float m = fabsf(v[q][j]);
                    most = live[q] && m < INFINITY ? fmaxf(most, m) : most;   // not a NaN either
                }
            }
        }
    }
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) {
        most = fmaxf(most, __shfl_xor(most, d, kWave));
    }
    if (lane_id() == 0) {
        sums[threadIdx.x / kWave] = most;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 1; w < kAbsMaxThreads / kWave; ++w) {
            most = fmaxf(most, sums[w]);
        }
        parts[blockIdx.x] = most;
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------

constexpr int kComputeUnits = 256;
constexpr int kSplitTiles = 3;   // tiles of a split at least: what a block does before its first takes about as long
constexpr int kPieceRows = 320;  // dt: stream rows that a piece's start and its partial sums' way through memory take as long as

static PassPlan plan_pass(int planes, int dim, int64_t owners, int64_t streams, int pass)
{
    const int dp = loss_width(dim);
    PassPlan p{};
    p.rowsPerWave = wide_rows(planes, dp, pass);
    p.ownWaves = 4;
    // Smaller blocks where there are few: a wave's 32 rows instead of 64 (bfloat16 x 64, dx, 300 x 30000: 21 us with 64 rows, 18
    // with 32; 8192 x 200003: 504 and 532; dt, 300 x 30000: 17 and 11, 2000 x 100000: 84 and 72, 8000 x 60000: 171 and 175;
    // x 96, 4000 x 130000: 219 and 235).
    if (owners <= (pass == kLossForward ? 128 : pass == kLossDx ? 1024 : streams <= 2048 ? 131072 : 32768)) {
        p.rowsPerWave = 32;
    }
    if (pass != kLossDt && owners <= kFewRows) {
        p.ownWaves = narrow_waves(planes, dp);
    }
    p.blocks = cdiv(owners, (int64_t)p.rowsPerWave * p.ownWaves);
    const int tileRows = tile_rows(planes, dp, p.ownWaves, pass);
    const int64_t tiles = cdiv(streams, tileRows);
    const int64_t resident = (int64_t)kComputeUnits * resident_blocks(planes, dp, pass, p.rowsPerWave);
    const int64_t most = tiles < kSplitTiles ? 1 : tiles / kSplitTiles;
    int64_t splits = std::clamp(resident / p.blocks, (int64_t)1, most);
    if (pass == kLossDt && splits == 1) {
        // Nothing to split for, but the blocks of the last round, which are fewer than the compute units hold, are cut into up
        // to 8 pieces where that ends the round sooner (8192 x 200003 x 64 bf16, 782 blocks on 512 places: 631 us uncut, 571
        // in 2 pieces, 527 in 5, 535 in 9).
        const int64_t last = p.blocks % resident;
        int64_t least = tiles + kSplitTiles;
        for (int64_t k = 2; k <= std::min(most, (int64_t)8); ++k) {
            const int64_t time = cdiv(last * k, resident) * (cdiv(tiles, k) + cdiv(kPieceRows, tileRows));
            if (time < least) {
                least = time;
                splits = k;
            }
        }
        p.whole = splits > 1 ? p.blocks - last : p.blocks;
    }
    p.tilesPerSplit = (int)cdiv(tiles, splits);
    p.splits = (int)cdiv(tiles, p.tilesPerSplit);
    p.parts = p.splits * (4 / p.ownWaves);
    return p;
}

// dt: items whose partial sums are joined, the last ones
static int64_t cut_items(const PassPlan& p, int64_t items)
{
    return std::max(items - p.whole * p.rowsPerWave * p.ownWaves, (int64_t)0);
}

struct LossPlan {
    int planes;
    int bytes;           // of an element
    int padded;          // columns of padded copies
    bool padX;           // rows that are copied into padded ones first
    bool padTable;
    bool tail;           // the table's rows, not copied, end inside a 16-byte piece
    PassPlan forward, dx, dt;
    int64_t atX, atTable, atMax, atParts;   // offsets into the workspace
    int64_t forwardBytes, backwardBytes;
};

static int64_t round256(int64_t v) { return (v + 255) / 256 * 256; }

// The table's rows of eight columns and more are read as they lie, on whatever border they start, for up to kDirectRows rows of x:
// then the copy takes longer than moving the columns to their places in every tile (1 x 228899 x 203 float32, forward: 149 us with
// a padded copy, 79 without; 1000 x 100000 x 201 bfloat16: 82 and 67; 4000 x 50000 x 201: 108 and 109, with dx 304 and 312, dt
// 259 and 247).  x, whose rows every split and every block of items reads again, is always copied (301 x 30011 x 201 bfloat16,
// forward: 28 us read off the borders, 24 with the copy).
static LossPlan plan_loss(int64_t rows, int64_t items, int32_t dim, int32_t dtype, int64_t x_stride, int64_t table_stride)
{
    LossPlan p{};
    p.planes = dtype == RECSDK_DT_BF16 ? 1 : rows <= kFewRows ? 3 : 2;
    p.bytes = float_bytes(dtype);
    const int piece = 16 / p.bytes;
    p.padded = (int)(cdiv(dim, piece) * piece);
    p.padX = dim % piece != 0 || x_stride % piece != 0 || x_stride > kLossMaxStride;
    p.padTable = dim % piece != 0 || table_stride % piece != 0 || table_stride > kLossMaxStride;
    if (rows <= kDirectRows && (dim >= kDirectDim || dim % piece == 0) && table_stride <= kLossMaxStride) {
        p.padTable = false;
    }
    p.tail = !p.padTable && dim % piece != 0;
    p.forward = plan_pass(p.planes, dim, rows, items, kLossForward);
    p.dx = plan_pass(p.planes, dim, rows, items, kLossDx);
    p.dt = plan_pass(p.planes, dim, items, rows, kLossDt);
    p.atX = 0;
    p.atTable = round256(p.atX + (p.padX ? rows * p.padded * p.bytes : 0));
    p.atMax = round256(p.atTable + (p.padTable ? items * p.padded * p.bytes : 0));
    p.atParts = round256(p.atMax + (p.planes == 2 ? 2 * kAbsMaxParts * (int64_t)sizeof(float) : 0));
    const int64_t norm = (int64_t)p.forward.parts * rows * (int64_t)sizeof(float2);
    const int64_t pitch = cdiv(dim, 4) * 4 * (int64_t)sizeof(float);
    const int64_t dx = (int64_t)p.dx.parts * rows * pitch;
    const int64_t dt = (int64_t)p.dt.parts * cut_items(p.dt, items) * pitch;
    p.forwardBytes = round256(p.atParts + norm);
    p.backwardBytes = round256(p.atParts + (dx > dt ? dx : dt));   // the two passes run one after the other
    return p;
}

static int launch_loss_pass(int pass, int planes, LossArgs a, const PassPlan& p, hipStream_t stream)
{
    a.whole = (int32_t)p.whole;
    a.splits = p.splits;
    a.tilesPerSplit = p.tilesPerSplit;
    if (pass == kLossForward) {
        return planes == 1 ? launch_bf16_forward(a, p, stream) : launch_f32_forward(planes, a, p, stream);
    }
    return planes == 1 ? launch_bf16_backward(pass, a, p, stream) : launch_f32_backward(pass, planes, a, p, stream);
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

template <typename T, int WAYS>
static int launch_grad_join(const float* part, int parts, int64_t rows, int dim, const float* lse, const float* grad,
                            float scale, void* out, hipStream_t stream)
{
    const int partDim = (int)cdiv(dim, 4) * 4;
    const int64_t grid = std::min(cdiv(rows * partDim, (int64_t)kBlock / WAYS * 4), kMostBlocks);
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

// item_bias / scale is what the bfloat16 kernels work with (folds_shift)
static int check_scale(const char* name, int32_t dtype, const float* bias, float scale)
{
    const float size = scale < 0.0f ? -scale : scale;
    if (!(size < INFINITY) || (dtype == RECSDK_DT_BF16 && bias != nullptr && size != 0.0f && size < 0x1p-40f)) {
        set_error("%s: scale must be finite, and 0 or at least 2^-40 for bf16 rows with item_bias", name);
        return RECSDK_EINVAL;
    }
    return RECSDK_OK;
}

// The operands as the tile kernels read them: whole 16-byte pieces; others are copied into padded rows.
template <typename T>
static int pad_operands(const LossPlan& plan, LossOperands& o, int64_t rows, int64_t items, int dim, char* workspace,
                        hipStream_t stream)
{
    auto padding = [&](bool wanted, const void*& src, int64_t& stride, int64_t count, int64_t at) {
        PadRows<T> p{};
        if (wanted) {
            p = {static_cast<const T*>(src), stride, count, reinterpret_cast<T*>(workspace + at),
                 std::min(cdiv(count, kBlock / 32), kMostBlocks)};
            src = p.dst;
            stride = plan.padded;
        }
        return p;
    };
    const PadRows<T> x = padding(plan.padX, o.x, o.xStride, rows, plan.atX);
    const PadRows<T> table = padding(plan.padTable, o.table, o.tableStride, items, plan.atTable);
    if (x.blocks + table.blocks > 0) {
        RECSDK_LAUNCH_AS("k_pad_rows", (k_pad_rows<T>), dim3((unsigned)(x.blocks + table.blocks)), dim3(kBlock), stream, x, table,
                         dim, plan.padded);
    }
    return RECSDK_OK;
}

// The operands' largest values, where the planes are float16.
static int find_largest(const LossPlan& plan, const LossOperands& o, int64_t rows, int64_t items, int dim, const int64_t* target,
                        const float* bias, char* workspace, hipStream_t stream)
{
    if (plan.planes == 2) {
        RECSDK_LAUNCH_AS("k_abs_max", k_abs_max, dim3(2 * kAbsMaxParts), dim3(kAbsMaxThreads), stream,
                         static_cast<const float*>(o.x), o.xStride, (int)rows, static_cast<const float*>(o.table), o.tableStride,
                         (int)items, dim, target, bias, reinterpret_cast<float*>(workspace + plan.atMax));
    }
    return RECSDK_OK;
}

template <typename T>
static int run_forward(const LossPlan& plan, LossOperands o, int64_t rows, int64_t items, int dim, const int64_t* target,
                       const float* bias, float scale, float* loss, float* lse, char* workspace, hipStream_t stream)
{
    const LossOperands given = o;
    int rc = pad_operands<T>(plan, o, rows, items, dim, workspace, stream);
    if (rc == RECSDK_OK) {
        rc = find_largest(plan, o, rows, items, dim, target, bias, workspace, stream);
    }
    if (rc != RECSDK_OK) {
        return rc;
    }
    const float* xMax = reinterpret_cast<const float*>(workspace + plan.atMax);
    const float* tableMax = xMax + kAbsMaxParts;
    LossArgs a{};
    a.own = o.x;
    a.ownStride = o.xStride;
    a.stream = o.table;
    a.streamStride = o.tableStride;
    a.owners = (int32_t)rows;
    a.streams = (int32_t)items;
    a.dim = dim;
    a.tail = plan.tail;
    a.target = target;
    a.bias = bias;
    a.scale = scale;
    a.ownMax = xMax;
    a.streamMax = tableMax;
    a.norm = reinterpret_cast<float2*>(workspace + plan.atParts);
    rc = launch_loss_pass(kLossForward, plan.planes, a, plan.forward, stream);
    if (rc != RECSDK_OK) {
        return rc;
    }
    const T* x = static_cast<const T*>(given.x);
    const T* table = static_cast<const T*>(given.table);
    // a block per row where a wave would walk more than four rounds of parts
    const bool whole = plan.forward.parts >= 4 * kWave;
    const dim3 grid((unsigned)std::min(whole ? rows : cdiv(rows, kBlock / kWave), kMostBlocks));
    if (whole) {
        RECSDK_LAUNCH_AS("k_softmax_loss_join", (k_softmax_loss_join<T, kBlock>), grid, dim3(kBlock), stream, a.norm,
                         plan.forward.parts, (int)rows, (int)items, dim, x, given.xStride, table, given.tableStride, target, bias,
                         scale, loss, lse);
    } else {
        RECSDK_LAUNCH_AS("k_softmax_loss_join", (k_softmax_loss_join<T, kWave>), grid, dim3(kBlock), stream, a.norm,
                         plan.forward.parts, (int)rows, (int)items, dim, x, given.xStride, table, given.tableStride, target, bias,
                         scale, loss, lse);
    }
    return RECSDK_OK;
}

template <typename T>
static int run_backward(const LossPlan& plan, LossOperands o, int64_t rows, int64_t items, int dim, const int64_t* target,
                        const float* bias, float scale, const float* lse, const float* grad, void* dx, void* dtable,
                        char* workspace, hipStream_t stream)
{
    int rc = pad_operands<T>(plan, o, rows, items, dim, workspace, stream);
    if (rc == RECSDK_OK) {
        rc = find_largest(plan, o, rows, items, dim, target, bias, workspace, stream);
    }
    if (rc != RECSDK_OK) {
        return rc;
    }
    const float* xMax = reinterpret_cast<const float*>(workspace + plan.atMax);
    const float* tableMax = xMax + kAbsMaxParts;
    LossArgs a{};
    a.dim = dim;
    a.tail = plan.tail;
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
        a.ownMax = xMax;
        a.streamMax = tableMax;
        a.part = part;
        rc = launch_loss_pass(kLossDx, plan.planes, a, plan.dx, stream);
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
        a.ownMax = tableMax;
        a.streamMax = xMax;
        a.part = part;
        a.out = dtable;
        rc = launch_loss_pass(kLossDt, plan.planes, a, plan.dt, stream);
        if (rc != RECSDK_OK) {
            return rc;
        }
        const int64_t cut = cut_items(plan.dt, items);
        if (cut > 0) {
            return join_grad<T>(part, plan.dt.parts, cut, dim, nullptr, nullptr, scale,
                                static_cast<T*>(dtable) + (items - cut) * dim, stream);
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
    int rc = check_loss("recsdk_softmax_loss_forward", rows, items, dim, dtype, x_stride, table_stride);
    rc = rc == RECSDK_OK ? check_scale("recsdk_softmax_loss_forward", dtype, d_item_bias, scale) : rc;
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
    int rc = check_loss("recsdk_softmax_loss_backward", rows, items, dim, dtype, x_stride, table_stride);
    rc = rc == RECSDK_OK ? check_scale("recsdk_softmax_loss_backward", dtype, d_item_bias, scale) : rc;
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
