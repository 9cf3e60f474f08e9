// Dropout whose mask is stored nowhere: the forward and the backward pass draw it again from a counter.
//
// Element e takes 16 random bits, number e % 8 of the eight that the block with counter (e / 8, offset) under the key
// `seed` holds, and is kept where they are below `below` = round(65536 (1 - p)); kept elements are multiplied by
// 65536 / below, so that the expectation is exact for the probability that 16 bits can hold.  The generator is
// Philox-4x32 with ten rounds (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011):
// a block is a function of its counter alone, so any launch shape, a slice of the tensor or the backward pass get the
// same mask.
//
// What bounds it: one read and one write per element, and one block of the generator (20 products of 32 bits) for
// eight elements.  Sixteen bits per element rather than 32 halve the generator's share.
#include <math.h>

#include "dense.h"

namespace recsdk {

struct Philox {
    uint32_t w[4];
};

__device__ __forceinline__ Philox philox(uint64_t block, uint64_t offset, uint64_t seed)
{
    uint32_t c0 = (uint32_t)block;
    uint32_t c1 = (uint32_t)(block >> 32);
    uint32_t c2 = (uint32_t)offset;
    uint32_t c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed;
    uint32_t k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u;
        const uint64_t b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)b;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}

constexpr int kDropItems = 2;   // pieces of 16 bytes per thread

__device__ __forceinline__ uint32_t neighbour(uint32_t v)   // the value of lane ^ 1
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true);
}

// Two pieces of 16 bytes for each generator block that a thread draws: eight 16-bit elements are one piece, eight float32
// ones two.  The pieces of a wave lie side by side in either case, so that an access covers whole cache lines: of the float32
// elements, a thread holds piece `lane` of its wave's first and second 64, which belong to block lane / 2 of the first and
// of the second 32, and neighbouring lanes (each has drawn one of the two) exchange halves.
// 218 M float32 elements: 327 us with a 32-byte stretch per thread, 297 us so (5.9 TB/s; a copy 6.0).
template <typename T>
__global__ __launch_bounds__(kBlock) void k_dropout(const T* __restrict__ x, T* __restrict__ y, int64_t n, uint32_t below,
                                                    float factor, uint64_t seed, uint64_t offset,
                                                    const int64_t* __restrict__ step)
{
    constexpr int kPer = 16 / sizeof(T);         // elements of a piece
    constexpr int kPieces = 8 / kPer;            // pieces per generator block
    constexpr int kBlocks = kDropItems / kPieces;   // generator blocks per thread
    if (step != nullptr) {
        offset += (uint64_t)*step;
    }
    const int lane = lane_id();
    // pieces of this wave: 64 at a time
    const int64_t wave = ((int64_t)blockIdx.x * (kBlock / kWave) + threadIdx.x / kWave) * (kWave * kDropItems);
    auto element = [&](int q) { return (wave + q * kWave + lane) * kPer; };
    Pack<T, kPer> v[kDropItems];
#pragma unroll
    for (int q = 0; q < kDropItems; ++q) {
        const int64_t e = element(q);
        if (e + kPer <= n) {
            v[q] = load_pack<T, kPer>(x + e);
        } else {
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                v[q].v[j] = e + j < n ? x[e + j] : from_float<T>(0.0f);
            }
        }
    }
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
        uint32_t bits[kPieces][kPer / 2];   // two elements per word
        if constexpr (kPieces == 1) {
            const Philox r = philox((uint64_t)(wave + b * kWave + lane), offset, seed);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                bits[0][w] = r.w[w];
            }
        } else {
            const bool odd = (lane & 1) != 0;
            const Philox r = philox((uint64_t)(wave / 2 + b * kWave + lane / 2 + (odd ? 32 : 0)), offset, seed);
            // the even lane's block is of the first 64 pieces: its first half stays, its second goes to the odd lane
            const uint32_t from0 = neighbour(odd ? r.w[0] : r.w[2]);
            const uint32_t from1 = neighbour(odd ? r.w[1] : r.w[3]);
            bits[0][0] = odd ? from0 : r.w[0];
            bits[0][1] = odd ? from1 : r.w[1];
            bits[1][0] = odd ? r.w[2] : from0;
            bits[1][1] = odd ? r.w[3] : from1;
        }
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
            const int q = b * kPieces + p;
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const uint32_t h = (j & 1) != 0 ? bits[p][j / 2] >> 16 : bits[p][j / 2] & 0xffffu;
                T& t = v[q].v[j];
                // chosen, not multiplied by zero: a dropped NaN or infinity is gone
                t = h < below ? from_float<T>((float)t * factor) : from_float<T>(0.0f);
            }
            const int64_t e = element(q);
            if (e + kPer <= n) {
                store_pack<T, kPer>(y + e, v[q]);
            } else {
#pragma unroll
                for (int j = 0; j < kPer; ++j) {
                    if (e + j < n) {
                        y[e + j] = v[q].v[j];
                    }
                }
            }
        }
    }
}

// The same for buffers that are not 16-byte aligned: a generator block per thread, element by element.
template <typename T>
__global__ __launch_bounds__(kBlock) void k_dropout_single(const T* __restrict__ x, T* __restrict__ y, int64_t n, uint32_t below,
                                                           float factor, uint64_t seed, uint64_t offset,
                                                           const int64_t* __restrict__ step)
{
    if (step != nullptr) {
        offset += (uint64_t)*step;
    }
    const int64_t block = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    const Philox r = philox((uint64_t)block, offset, seed);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int64_t e = block * 8 + j;
        if (e < n) {
            const uint32_t h = (j & 1) != 0 ? r.w[j / 2] >> 16 : r.w[j / 2] & 0xffffu;
            y[e] = h < below ? from_float<T>((float)x[e] * factor) : from_float<T>(0.0f);
        }
    }
}

template <typename T>
static int launch_dropout(const void* x, void* y, int64_t n, uint32_t below, float factor, uint64_t seed, uint64_t offset,
                          const int64_t* step, hipStream_t stream)
{
    const bool whole = aligned16(x) && aligned16(y);
    const int64_t grid = whole ? cdiv(n, (int64_t)kBlock * kDropItems * (16 / (int)sizeof(T))) : cdiv(cdiv(n, 8), kBlock);
    RECSDK_REQUIRE(grid * kBlock < (int64_t(1) << 32), RECSDK_EINVAL, "recsdk_dropout: too large for one launch");
    const T* px = static_cast<const T*>(x);
    T* py = static_cast<T*>(y);
    if (whole) {
        RECSDK_LAUNCH_AS("k_dropout", (k_dropout<T>), dim3((unsigned)grid), dim3(kBlock), stream, px, py, n, below, factor, seed,
                         offset, step);
    } else {
        RECSDK_LAUNCH_AS("k_dropout", (k_dropout_single<T>), dim3((unsigned)grid), dim3(kBlock), stream, px, py, n, below, factor,
                         seed, offset, step);
    }
    return RECSDK_OK;
}

}  // namespace recsdk

extern "C" int recsdk_dropout(const void* d_x, int64_t n, int32_t dtype, double p, uint64_t seed, uint64_t offset,
                              const int64_t* d_step, void* d_y, void* stream)
{
    using namespace recsdk;
    RECSDK_REQUIRE(float_bytes(dtype) != 0, RECSDK_EINVAL, "recsdk_dropout: dtype must be fp32, fp16 or bf16");
    RECSDK_REQUIRE(p >= 0.0 && p <= 1.0, RECSDK_EINVAL, "recsdk_dropout: p must lie in [0, 1]");
    RECSDK_REQUIRE(n >= 0, RECSDK_EINVAL, "recsdk_dropout: n must not be negative");
    if (n == 0) {
        return RECSDK_OK;
    }
    RECSDK_REQUIRE(d_x != nullptr && d_y != nullptr, RECSDK_ENULL, "recsdk_dropout: NULL argument");
    RECSDK_REQUIRE(reinterpret_cast<uintptr_t>(d_x) % float_bytes(dtype) == 0 &&
                       reinterpret_cast<uintptr_t>(d_y) % float_bytes(dtype) == 0,
                   RECSDK_EINVAL, "recsdk_dropout: buffers must be aligned to their elements");
    const uint32_t below = (uint32_t)nearbyint(65536.0 * (1.0 - p));   // 0: everything is dropped
    const float factor = below != 0 ? (float)(65536.0 / below) : 0.0f;
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case RECSDK_DT_F32:
            return launch_dropout<float>(d_x, d_y, n, below, factor, seed, offset, d_step, s);
        case RECSDK_DT_F16:
            return launch_dropout<F16>(d_x, d_y, n, below, factor, seed, offset, d_step, s);
        default:
            return launch_dropout<BF16>(d_x, d_y, n, below, factor, seed, offset, d_step, s);
    }
}
