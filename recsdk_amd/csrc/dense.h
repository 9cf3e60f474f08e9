// Element types and small helpers shared by the dense kernels (dropout.hip, norm.hip, softmax_loss.hip).
#ifndef RECSDK_CSRC_DENSE_H
#define RECSDK_CSRC_DENSE_H

#include "common.h"

namespace recsdk {

typedef uint32_t Word4 __attribute__((ext_vector_type(4)));   // 16 bytes as one lane moves them
typedef float Float4 __attribute__((ext_vector_type(4)));

// Bytes of a floating element type, 0 for anything else.
inline int float_bytes(int32_t dtype)
{
    return dtype == RECSDK_DT_F32 ? 4 : (dtype == RECSDK_DT_F16 || dtype == RECSDK_DT_BF16) ? 2 : 0;
}

inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

#ifdef __HIPCC__

using F16 = _Float16;
using BF16 = __bf16;

// Rounds to nearest even, as every store of a result does.
template <typename T>
__device__ __forceinline__ T from_float(float v)
{
    return (T)v;
}

// E elements of type T as they come from memory: one 16-byte access where E * sizeof(T) is 16, else element by element.
template <typename T, int E>
struct Pack {
    T v[E];
};

template <typename T, int E>
__device__ __forceinline__ Pack<T, E> load_pack(const T* p)
{
    Pack<T, E> r;
    if constexpr (E * sizeof(T) == 16) {
        const Word4 w = *reinterpret_cast<const Word4*>(p);
        __builtin_memcpy(&r, &w, 16);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            r.v[e] = p[e];
        }
    }
    return r;
}

// Streamed past the caches: results are written once and read by a later kernel.
template <typename T, int E>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, E>& r)
{
    if constexpr (E * sizeof(T) == 16) {
        Word4 w;
        __builtin_memcpy(&w, &r, 16);
        __builtin_nontemporal_store(w, reinterpret_cast<Word4*>(p));
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            p[e] = r.v[e];
        }
    }
}

// Columns d .. d + 3 of a row, as far as it has them.
template <typename T>
__device__ __forceinline__ void store_columns(T* row, int d, int dim, bool fours, Float4 v)
{
    typedef T T4 __attribute__((ext_vector_type(4)));
    if (fours) {
        if (d < dim) {
            *reinterpret_cast<T4*>(row + d) =
                T4{from_float<T>(v[0]), from_float<T>(v[1]), from_float<T>(v[2]), from_float<T>(v[3])};
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

// v + the same of the lane D away (D a power of two; groups of 2 D lanes end up with one value when the smaller steps were
// taken before).  Within 16 lanes by data-parallel moves, across them by the row swaps: no trip through LDS, whose latency
// a short row's two reductions would wait for ten times.
template <int D>
__device__ __forceinline__ float add_across(float v)
{
    if constexpr (D < 16) {
        // quad permutations 1 0 3 2 and 2 3 0 1, then mirrors of 8 and of 16 lanes
        constexpr int kCtrl = D == 1 ? 0xB1 : D == 2 ? 0x4E : D == 4 ? 0x141 : 0x140;
        return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kCtrl, 0xf, 0xf, true));
    } else if constexpr (D == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        return __uint_as_float(r[0]) + __uint_as_float(r[1]);
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        return __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
}

// Sum over aligned groups of G <= 64 lanes, in every lane of them.
template <int G>
__device__ __forceinline__ float group_sum(float v)
{
    if constexpr (G > 1) {
        v = add_across<1>(v);
    }
    if constexpr (G > 2) {
        v = add_across<2>(v);
    }
    if constexpr (G > 4) {
        v = add_across<4>(v);
    }
    if constexpr (G > 8) {
        v = add_across<8>(v);
    }
    if constexpr (G > 16) {
        v = add_across<16>(v);
    }
    if constexpr (G > 32) {
        v = add_across<32>(v);
    }
    return v;
}

#endif  // __HIPCC__

}  // namespace recsdk

#endif
