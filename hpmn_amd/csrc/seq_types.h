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

// Four elements at p (VEC: one aligned access) or the n < 4 valid ones of them (!VEC: scalar accesses, zero behind).
template <typename T, bool VEC>
__device__ __forceinline__ quad_t<T> load_quad(const T *p, int n) {
    if constexpr (VEC) {
        return *reinterpret_cast<const quad_t<T> *>(p);
    } else {
        quad_t<T> q;
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = i < n ? p[i] : (T)0.f;
        return q;
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_quad(T *p, v4f x, int n) {
    if constexpr (VEC) {
        *reinterpret_cast<quad_t<T> *>(p) = __builtin_convertvector(x, quad_t<T>);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) p[i] = (T)x[i];
    }
}

// a = sigmoid(z) and u = 1 - a = sigmoid(-z), both to a relative rounding or two: e = exp(-|z|) <= 1 never overflows, and the
// smaller of the two is e / (1 + e) instead of a difference (1 - a in fp32 has no digits left from z = 17 on).
__device__ __forceinline__ void gate_pair(float z, float &a, float &u) {
    const float e = __builtin_amdgcn_exp2f(NEG_LOG2E * fabsf(z));
    const float big = __builtin_amdgcn_rcpf(1.0f + e), small = e * big;
    const bool pos = z >= 0.f;
    a = pos ? big : small;
    u = pos ? small : big;
}

inline bool is_aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
inline size_t elem_size(int dtype) { return dtype == HPMN_F32 ? 4 : 2; }

}  // namespace hpmn
