// Shared by the training kernels (train_norm.hip, train_loss.hip, optim.hip): activation types, wide loads at
// any element alignment, sums over groups of lanes.
#pragma once
#include "az_common.h"

namespace az {

constexpr int64_t MOST_BLOCKS = 0xFFFFFF;      // workgroups of 256 threads: a launch has fewer than 2^32 threads

// A load or store of 16 bytes needs only the element's own alignment: the hardware takes unaligned global accesses
// in one instruction.  So rows of any length and tensors at any offset run through the same wide path.
template <typename T> struct Pack;
#define AZ_PACK(T, N)                                                     \
    template <> struct Pack<T> {                                          \
        static constexpr int V = N;                                       \
        typedef T raw __attribute__((ext_vector_type(N)));                \
        typedef raw loose __attribute__((aligned(sizeof(T))));            \
        typedef float f32 __attribute__((ext_vector_type(N)));            \
    }
AZ_PACK(float, 4);
AZ_PACK(__bf16, 8);
AZ_PACK(_Float16, 8);
#undef AZ_PACK

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4_loose __attribute__((aligned(4)));

// `left` values from p on (the rest zero), widened to float.
template <typename T>
__device__ inline typename Pack<T>::f32 load_pack(const T* p, int left) {
    typename Pack<T>::f32 v;
    if (left >= Pack<T>::V) {
        v = __builtin_convertvector(*(const typename Pack<T>::loose*)p, typename Pack<T>::f32);
    } else {
#pragma unroll
        for (int i = 0; i < Pack<T>::V; ++i) v[i] = i < left ? (float)p[i] : 0.f;
    }
    return v;
}

// Rounds to nearest even, once.
template <typename T>
__device__ inline void store_pack(T* p, typename Pack<T>::f32 v, int left) {
    if (left >= Pack<T>::V) {
        *(typename Pack<T>::loose*)p = __builtin_convertvector(v, typename Pack<T>::raw);
    } else {
#pragma unroll
        for (int i = 0; i < Pack<T>::V; ++i)
            if (i < left) p[i] = (T)v[i];
    }
}

// Sum over L neighbouring lanes (L = 4, 8, 16, 32 or 64), the result in all of them.  Inside 16 lanes the partner's value
// comes through the DPP operand of an add (quad permutes, then mirrors of 8 and 16: the halves are uniform by then).
template <int L>
__device__ inline float lane_sum(float v) {
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, true));   // lane ^ 1
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, true));   // lane ^ 2
    if (L >= 8) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xF, 0xF, true));
    if (L >= 16) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xF, 0xF, true));
    if (L >= 32) v += __shfl_xor(v, 16);
    if (L >= 64) v += __shfl_xor(v, 32);
    return v;
}

template <int L>
__device__ inline float lane_max(float v) {
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, true)));
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, true)));
    if (L >= 8) v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xF, 0xF, true)));
    if (L >= 16) v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xF, 0xF, true)));
    if (L >= 32) v = fmaxf(v, __shfl_xor(v, 16));
    if (L >= 64) v = fmaxf(v, __shfl_xor(v, 32));
    return v;
}

}  // namespace az
