// Element types of the sequence operators (gated scan, dropout, shared-prefix attention): fp32 arithmetic on fp32 / bf16 / fp16
// storage, four neighbouring elements per access where alignment allows it.
#pragma once
#include "common.h"

namespace hpmn {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Quad;
template <> struct Quad<float> { typedef v4f type; };
template <> struct Quad<bf16_t> { typedef bf16x4 type; };
template <> struct Quad<f16_t> { typedef f16x4 type; };
template <typename T> using quad_t = typename Quad<T>::type;
// the same in memory, aligned to an element: one access all the same (global memory takes any alignment; across cache lines it costs
// a second one)
template <typename T> struct LooseQuad { typedef quad_t<T> type __attribute__((aligned(sizeof(T)))); };
template <typename T> using loose_quad_t = typename LooseQuad<T>::type;

// Four elements from p on (VEC: one access), or the n in 1..4 valid ones of them (!VEC: scalar accesses; the rest repeat the last
// valid one).  Unconditional in every lane: a load under a condition is waited for where the paths meet.
template <typename T, bool VEC>
__device__ __forceinline__ quad_t<T> load_quad(const T *p, int n) {
    if constexpr (VEC) {
        return *reinterpret_cast<const loose_quad_t<T> *>(p);
    } else {
        quad_t<T> q;
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = p[min(i, n - 1)];
        return q;
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_quad(T *p, v4f x, int n) {
    if constexpr (VEC) {
        *reinterpret_cast<loose_quad_t<T> *>(p) = __builtin_convertvector(x, quad_t<T>);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) p[i] = (T)x[i];
    }
}

// a = sigmoid(z) = 1 / (1 + e) and u = 1 - a = e / (1 + e) with e = exp(-z), each relative to ITSELF (1 - a as a difference has no digits
// left from z = 17 on): a few roundings and the exponent's, about |z| 2^-24, in whichever of the two is small.  e is capped at 2^120, where a has long stopped mattering beside u = 1 (and
// inf * 0 would be NaN); the cap is the minimum that keeps a NaN.  Six instructions, two of them on the transcendental unit.
__device__ __forceinline__ void gate_pair(float z, float &a, float &u) {
    const float e = __builtin_amdgcn_exp2f(__builtin_elementwise_minimum(NEG_LOG2E * z, 120.0f));
    a = __builtin_amdgcn_rcpf(1.0f + e);
    u = e * a;
}

inline bool is_aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
inline size_t elem_size(int dtype) { return dtype == HPMN_F32 ? 4 : 2; }

}  // namespace hpmn
