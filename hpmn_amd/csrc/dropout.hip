// Dropout from a counter-based generator (include/hpmn_hip.h, hpmn_dropout): y = keep * x / p (+ residual), the keep decisions
// recomputed in the backward instead of stored.
//
// Memory-bound: 16 bytes per access.  A decision has to cost less than moving its element: one splitmix64 word (two 64-bit
// products) decides four elements by 16 bits each -- the probability is quantised to 2^-16 and the scale made exact for it, a
// word per element or 32 bits each would put the generator above the memory time for 16-bit types.  The mask goes by the
// logical element index alone, so strides, alignment and launch shape do not change it.  65536 x 1024 bf16: with residual 403 MB in
// 72.4 us, 5.6 TB/s; without 268 MB in 44.7 us, 6.0 TB/s; 128 x 200 fp32 2.4 us, a launch.
#include "seq_types.h"

namespace hpmn {

__device__ __forceinline__ uint64_t mix64(uint64_t x) {
    x = (x ^ (x >> 30)) * 0xBF58476D1CE4E5B9ull;
    x = (x ^ (x >> 27)) * 0x94D049BB133111EBull;
    return x ^ (x >> 31);
}

struct Words {
    uint64_t base;                           // mix(seed) + golden * (offset + 1)
    __device__ __forceinline__ Words(const HpmnDropout &a) {
        const uint64_t seed = a.rng ? a.rng[0] : a.seed, offset = a.offset + (a.rng ? a.rng[1] : 0);
        base = mix64(seed) + 0x9E3779B97F4A7C15ull * (offset + 1);
    }
    __device__ __forceinline__ uint64_t operator()(uint64_t k) const { return mix64(base + 0x9E3779B97F4A7C15ull * k); }
};

// One word's four elements; a dropped element is zero whatever it holds.
template <bool RES>
__device__ __forceinline__ v4f apply_word(uint64_t w, unsigned thr, float scale, v4f x, v4f r) {
    const unsigned lo = (unsigned)w, hi = (unsigned)(w >> 32);
    const unsigned f[4] = {lo & 0xFFFFu, lo >> 16, hi & 0xFFFFu, hi >> 16};
    v4f y;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        y[i] = f[i] < thr ? x[i] * scale : 0.f;
        if (RES) y[i] += r[i];
    }
    return y;
}

// Any row strides, any alignment: a thread per word, scalar accesses.
template <typename T>
__global__ __launch_bounds__(256) void dropout_words_kernel(const HpmnDropout a, unsigned thr, float scale) {
    const long k = (long)blockIdx.x * 256 + threadIdx.x, n = a.N * a.C;
    if (4 * k >= n) return;
    const uint64_t w = Words(a)((uint64_t)k);
    for (int j = 0; j < 4 && 4 * k + j < n; ++j) {
        const long r = (4 * k + j) / a.C, c = (4 * k + j) % a.C;
        float y = ((unsigned)(w >> (16 * j)) & 0xFFFFu) < thr ? (float)((const T *)a.x)[r * a.x_s + c] * scale : 0.f;
        if (a.residual) y += (float)((const T *)a.residual)[r * a.r_s + c];
        ((T *)a.y)[r * a.y_s + c] = (T)y;
    }
}

// A vector of E = 16 bytes' worth of elements per thread (four of them per thread: 122 against 119 us on 65536 x 1024 bf16 with
// residual, forward + backward, and too few workgroups for small tensors).  DENSE: the tensor is one run of N * C elements.
// !DENSE: rows of C elements, C and the row strides multiples of E.
template <typename T, bool DENSE, bool RES>
__global__ __launch_bounds__(256) void dropout_vec_kernel(const HpmnDropout a, unsigned thr, float scale, unsigned vecs_per_row) {
    constexpr int E = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(E)));
    const T *x = (const T *)a.x, *res = (const T *)a.residual;
    T *y = (T *)a.y;
    const Words words(a);
    const long n = a.N * a.C, nv = n / E, v = (long)blockIdx.x * 256 + threadIdx.x;
    if (v < nv) {
        long ix = v * E, ir = ix, iy = ix;
        if (!DENSE) {
            const unsigned row = (unsigned)v / vecs_per_row, c = ((unsigned)v - row * vecs_per_row) * E;       // (nv < 2^32)
            ix = row * a.x_s + c;
            ir = row * a.r_s + c;
            iy = row * a.y_s + c;
        }
        const vec xv = *(const vec *)(x + ix);
        vec rv = {}, out;
        if (RES) rv = *(const vec *)(res + ir);
#pragma unroll
        for (int h = 0; h < E / 4; ++h) {
            v4f xx, rr;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                xx[i] = (float)xv[4 * h + i];
                rr[i] = (float)rv[4 * h + i];
            }
            const v4f o = apply_word<RES>(words((uint64_t)v * (E / 4) + h), thr, scale, xx, rr);
#pragma unroll
            for (int i = 0; i < 4; ++i) out[4 * h + i] = (T)o[i];
        }
        *(vec *)(y + iy) = out;
    }
    if (DENSE && blockIdx.x == 0) {                          // the run's last, incomplete vector
        const long i = nv * E + threadIdx.x;
        if (i < n) {
            const uint64_t w = words((uint64_t)(i / 4));
            float o = ((unsigned)(w >> (16 * (i % 4))) & 0xFFFFu) < thr ? (float)x[i] * scale : 0.f;
            if (RES) o += (float)res[i];
            y[i] = (T)o;
        }
    }
}

template <typename T>
static void dropout_type(const HpmnDropout &a, unsigned thr, float scale, hipStream_t st) {
    constexpr int E = 16 / sizeof(T);
    const long n = a.N * a.C, nv = n / E;
    const bool res = a.residual != nullptr;
    const bool dense = (a.N == 1 || (a.x_s == a.C && a.y_s == a.C && (!res || a.r_s == a.C)));
    const bool wide = is_aligned(a.x, 16) && is_aligned(a.y, 16) && is_aligned(a.residual, 16) && nv >= 1;
    const bool rows = a.C % E == 0 && a.x_s % E == 0 && a.y_s % E == 0 && (!res || a.r_s % E == 0) && nv < (1l << 32) - 1;
    if (wide && (dense || rows)) {
        const unsigned vpr = (unsigned)(dense ? 1 : a.C / E);
        const dim3 grid((unsigned)((nv + 255) / 256));
        if (dense && res) hipLaunchKernelGGL((dropout_vec_kernel<T, true, true>), grid, dim3(256), 0, st, a, thr, scale, vpr);
        else if (dense) hipLaunchKernelGGL((dropout_vec_kernel<T, true, false>), grid, dim3(256), 0, st, a, thr, scale, vpr);
        else if (res) hipLaunchKernelGGL((dropout_vec_kernel<T, false, true>), grid, dim3(256), 0, st, a, thr, scale, vpr);
        else hipLaunchKernelGGL((dropout_vec_kernel<T, false, false>), grid, dim3(256), 0, st, a, thr, scale, vpr);
        return;
    }
    const long words = (n + 3) / 4;
    hipLaunchKernelGGL(dropout_words_kernel<T>, dim3((unsigned)((words + 255) / 256)), dim3(256), 0, st, a, thr, scale);
}

int dropout_launch(const HpmnDropout &a, unsigned thr, hipStream_t st) {
    const float scale = 65536.0f / (float)thr;
    if (a.dtype == HPMN_F32) dropout_type<float>(a, thr, scale, st);
    else if (a.dtype == HPMN_BF16) dropout_type<bf16_t>(a, thr, scale, st);
    else dropout_type<f16_t>(a, thr, scale, st);
    return check_launch();
}

}  // namespace hpmn
