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

constexpr int kDropItems = 2;   // generator blocks (of eight elements) per thread

// VEC: the buffers are 16-byte aligned, so that eight elements move in one or two accesses.
template <typename T, bool VEC>
__global__ __launch_bounds__(kBlock) void k_dropout(const T* __restrict__ x, T* __restrict__ y, int64_t n, uint32_t below,
                                                    float factor, uint64_t seed, uint64_t offset,
                                                    const int64_t* __restrict__ step)
{
    constexpr int kPer = 16 / sizeof(T);      // elements of a 16-byte access
    constexpr int kAcc = 8 / kPer;            // accesses for eight elements
    if (step != nullptr) {
        offset += (uint64_t)*step;
    }
    const int64_t first = (int64_t)blockIdx.x * (kBlock * kDropItems) + threadIdx.x;
    Pack<T, kPer> v[kDropItems][kAcc];
#pragma unroll
    for (int k = 0; k < kDropItems; ++k) {
        const int64_t e = (first + k * kBlock) * 8;
        if (VEC && e + 8 <= n) {
#pragma unroll
            for (int q = 0; q < kAcc; ++q) {
                v[k][q] = load_pack<T, kPer>(x + e + q * kPer);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (e + j < n) {
                    v[k][j / kPer].v[j % kPer] = x[e + j];
                }
            }
        }
    }
#pragma unroll
    for (int k = 0; k < kDropItems; ++k) {
        const int64_t block = first + k * kBlock;
        const int64_t e = block * 8;
        if (e >= n) {
            return;
        }
        const Philox r = philox((uint64_t)block, offset, seed);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t bits = (j & 1) != 0 ? r.w[j / 2] >> 16 : r.w[j / 2] & 0xffffu;
            T& t = v[k][j / kPer].v[j % kPer];
            // chosen, not multiplied by zero: a dropped NaN or infinity is gone
            t = bits < below ? from_float<T>((float)t * factor) : from_float<T>(0.0f);
        }
        if (VEC && e + 8 <= n) {
#pragma unroll
            for (int q = 0; q < kAcc; ++q) {
                store_pack<T, kPer>(y + e + q * kPer, v[k][q]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (e + j < n) {
                    y[e + j] = v[k][j / kPer].v[j % kPer];
                }
            }
        }
    }
}

template <typename T>
static int launch_dropout(const void* x, void* y, int64_t n, uint32_t below, float factor, uint64_t seed, uint64_t offset,
                          const int64_t* step, hipStream_t stream)
{
    const int64_t grid = cdiv(cdiv(n, 8), (int64_t)kBlock * kDropItems);
    RECSDK_REQUIRE(grid < (int64_t(1) << 31), RECSDK_EINVAL, "recsdk_dropout: too large for one launch");
    const T* px = static_cast<const T*>(x);
    T* py = static_cast<T*>(y);
    if (aligned16(x) && aligned16(y)) {
        RECSDK_LAUNCH_AS("k_dropout", (k_dropout<T, true>), dim3((unsigned)grid), dim3(kBlock), stream, px, py, n, below,
                         factor, seed, offset, step);
    } else {
        RECSDK_LAUNCH_AS("k_dropout", (k_dropout<T, false>), dim3((unsigned)grid), dim3(kBlock), stream, px, py, n, below,
                         factor, seed, offset, step);
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
