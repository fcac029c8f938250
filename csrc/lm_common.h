// Shared device helpers of the operators around the language-model head
// (distill.hip, adapters.hip, logits.hip).  Wavefront 64, gfx950.
#pragma once

#include <hip/hip_runtime.h>

#define DEVINL __device__ __forceinline__

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// Eight neighbouring elements at ANY element alignment: rows of an odd vocabulary start at
// every 2-byte offset.  The typedef lowers the alignment and the compiler emits one wide load
// (the amdhsa target allows unaligned vector memory access).
template <typename T> struct Vec8;
template <> struct Vec8<bf16_t> {
    typedef bf16_t type __attribute__((ext_vector_type(8), aligned(2)));
};
template <> struct Vec8<f16_t> {
    typedef f16_t type __attribute__((ext_vector_type(8), aligned(2)));
};
template <> struct Vec8<float> {
    typedef float type __attribute__((ext_vector_type(8), aligned(4)));
};

template <typename T> DEVINL void load8(const T* p, float (&out)[8]) {
    const auto v = *(const typename Vec8<T>::type*)p;
#pragma unroll
    for (int j = 0; j < 8; ++j) out[j] = (float)v[j];
}

template <typename T> DEVINL void store8(T* p, const float (&in)[8]) {
    typename Vec8<T>::type v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (T)in[j];
    *(typename Vec8<T>::type*)p = v;
}

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

DEVINL float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }   // v_exp_f32, 1 ulp
DEVINL float neg_inf() { return -__builtin_huge_valf(); }

// Index tensors come as int32 or int64.
DEVINL long load_index(const void* p, long i, bool wide) {
    return wide ? ((const long*)p)[i] : (long)((const int*)p)[i];
}

// Floating tensors whose type is known at run time only (short lists, not the streams).
enum { LM_BF16 = 0, LM_F16 = 1, LM_F32 = 2 };
DEVINL float load_float(const void* p, long i, int type) {
    if (type == LM_BF16) return (float)((const bf16_t*)p)[i];
    if (type == LM_F16) return (float)((const f16_t*)p)[i];
    return ((const float*)p)[i];
}

// sums[at] += x of a wave's lanes that have one, lane by lane where `at` is the same: a list's
// repeated indices are added in the list's order.  Every lane of the wave has to be there.
DEVINL void add_in_order(bool has, int at, float x, float* sums) {
    unsigned long long left = __ballot(has);
    while (left) {
        const int slot = __builtin_amdgcn_readlane(at, __ffsll(left) - 1);
        unsigned long long same = __ballot(has && at == slot);
        left &= ~same;
        float s = sums[slot];
        for (; same; same &= same - 1)
            s += __int_as_float(
                __builtin_amdgcn_readlane(__float_as_int(x), __ffsll(same) - 1));
        sums[slot] = s;                 // the same from every lane
    }
}
// LDS that one lane of the wave wrote and another reads, or the other way round.
DEVINL void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
}

DEVINL float wave_max(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
    return v;
}
DEVINL float wave_sum(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}
