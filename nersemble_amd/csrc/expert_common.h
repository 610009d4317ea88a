// expert_common.h -- what the routed-experts kernels share: element types, division by a run-time constant, the checks of a
// plan's numbers.  (expert_route.hip: choice and plan; expert_linear.hip: products; expert_combine.hip: the weighted join.)
#pragma once
#include "nsx_common.h"

namespace nsx {

typedef __bf16 bf16_t;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Elem;
template <> struct Elem<half_t> { typedef half_t x8 __attribute__((ext_vector_type(8))); typedef half_t x4 __attribute__((ext_vector_type(4))); };
template <> struct Elem<bf16_t> { typedef bf16_t x8 __attribute__((ext_vector_type(8))); typedef bf16_t x4 __attribute__((ext_vector_type(4))); };
template <> struct Elem<float> { typedef float x8 __attribute__((ext_vector_type(8), aligned(16))); typedef float x4 __attribute__((ext_vector_type(4))); };

// n / d for 0 <= n < 2^31 by one high multiplication (the quotient's error of the rounded-up reciprocal is below 1 / d).
struct FastDiv {
    uint32_t mul, shift;
    __device__ __forceinline__ int operator()(int n) const { return (int)((__umulhi(mul, (uint32_t)n) + (uint32_t)n) >> shift); }
};
inline FastDiv fast_div(int d) {
    uint32_t l = 0;
    while ((1u << l) < (uint32_t)d) ++l;
    return FastDiv{(uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << l) - (uint64_t)d)) / (uint64_t)d + 1), l};
}

// Segment [a, b) of expert e, whatever the offsets hold: inside [0, R] and not reversed.
__device__ __forceinline__ void segment(const int32_t* __restrict__ offsets, int e, int R, int& a, int& b) {
    a = min(max(offsets[e], 0), R);
    b = min(max(offsets[e + 1], a), R);
}

__device__ __forceinline__ void wave_lds_fence() {
    // LDS operations of one wave complete in order: only the compiler has to keep them in it
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// expert_combine.hip: out [T][n] (dtype: 16 bits) = sum over a row's choices of y [R][n], which lies in 32 bits
int expert_join_f32(const float* y, int64_t R, int n, const int32_t* positions, int64_t T, int top_k, void* out, int dtype, hipStream_t st);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace nsx
