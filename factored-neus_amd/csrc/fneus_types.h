// Element types of the operators that take fp32, bf16 and fp16 tensors (norm_kernels.hip, linear_kernels.hip, muon_kernels.hip):
// conversions, and 16-byte chunks that may start at any element.  Global loads and stores of this target need no alignment beyond the
// element's, so a row of odd length or stride takes the same wide accesses as an aligned one (the chunk types say aligned(element)).
#pragma once
#include "fneus_common.h"

namespace fneus {

enum { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };

typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x8_u __attribute__((ext_vector_type(8), aligned(2)));
typedef _Float16 f16x8_u __attribute__((ext_vector_type(8), aligned(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

template <class T> struct Chunk;
template <> struct Chunk<float> { typedef f32x4_u type; static constexpr int N = 4; };
template <> struct Chunk<__bf16> { typedef bf16x8_u type; static constexpr int N = 8; };
template <> struct Chunk<_Float16> { typedef f16x8_u type; static constexpr int N = 8; };

// N values at p, of which the first `valid` exist (the others: 0)
template <class T>
FN_DEV void load_chunk(const T* p, int valid, float (&v)[Chunk<T>::N]) {
    constexpr int N = Chunk<T>::N;
    if (valid >= N) {
        const typename Chunk<T>::type c = *reinterpret_cast<const typename Chunk<T>::type*>(p);
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = (float)c[k];
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = k < valid ? (float)p[k] : 0.0f;
    }
}

template <class T>
FN_DEV void store_chunk(T* p, int valid, const float (&v)[Chunk<T>::N]) {
    constexpr int N = Chunk<T>::N;
    if (valid >= N) {
        typename Chunk<T>::type c;
#pragma unroll
        for (int k = 0; k < N; ++k) c[k] = (T)v[k];
        *reinterpret_cast<typename Chunk<T>::type*>(p) = c;
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (k < valid) p[k] = (T)v[k];
    }
}

// sum over the 16 lanes of a DPP row, in every lane (quad permutes, half mirror, mirror: no LDS traffic)
FN_DEV float row16_sum(float v) {
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, true));
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x4E, 0xF, 0xF, true));
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x141, 0xF, 0xF, true));
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x140, 0xF, 0xF, true));
    return v;
}

FN_DEV float wave_sum(float v) {
    v = row16_sum(v);
    v += __shfl_xor(v, 16, 64);
    v += __shfl_xor(v, 32, 64);
    return v;
}

}  // namespace fneus
