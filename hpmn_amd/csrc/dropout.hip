// Dropout from a counter-based generator (include/hpmn_hip.h, hpmn_dropout): one splitmix64 word decides four elements, so the
// mask is recomputed in the backward instead of being stored.
//
// First form: a thread per word, scalar accesses.
#include "seq_types.h"

namespace hpmn {

__device__ __forceinline__ uint64_t mix64(uint64_t x) {
    x = (x ^ (x >> 30)) * 0xBF58476D1CE4E5B9ull;
    x = (x ^ (x >> 27)) * 0x94D049BB133111EBull;
    return x ^ (x >> 31);
}

template <typename T>
__global__ __launch_bounds__(256) void dropout_words_kernel(const HpmnDropout a, unsigned thr, float scale) {
    const long k = (long)blockIdx.x * 256 + threadIdx.x, n = a.N * a.C;
    if (4 * k >= n) return;
    const uint64_t seed = a.rng ? a.rng[0] : a.seed, offset = a.offset + (a.rng ? a.rng[1] : 0);
    const uint64_t w = mix64(mix64(seed) + 0x9E3779B97F4A7C15ull * (offset + (uint64_t)k + 1));
    for (int j = 0; j < 4 && 4 * k + j < n; ++j) {
        const long r = (4 * k + j) / a.C, c = (4 * k + j) % a.C;
        float y = ((unsigned)(w >> (16 * j)) & 0xFFFFu) < thr ? (float)((const T *)a.x)[r * a.x_s + c] * scale : 0.f;
        if (a.residual) y += (float)((const T *)a.residual)[r * a.r_s + c];
        ((T *)a.y)[r * a.y_s + c] = (T)y;
    }
}

int dropout_launch(const HpmnDropout &a, unsigned thr, hipStream_t st) {
    const float scale = 65536.0f / (float)thr;
    const long words = (a.N * a.C + 3) / 4;
    const dim3 grid((unsigned)((words + 255) / 256));
    if (a.dtype == HPMN_F32) hipLaunchKernelGGL(dropout_words_kernel<float>, grid, dim3(256), 0, st, a, thr, scale);
    else if (a.dtype == HPMN_BF16) hipLaunchKernelGGL(dropout_words_kernel<bf16_t>, grid, dim3(256), 0, st, a, thr, scale);
    else hipLaunchKernelGGL(dropout_words_kernel<f16_t>, grid, dim3(256), 0, st, a, thr, scale);
    return check_launch();
}

}  // namespace hpmn
