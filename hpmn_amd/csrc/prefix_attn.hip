// Attention of a batch that shares a long prefix (include/hpmn_hip.h, hpmn_prefix_attn).
//
// First form: one wave per (row, query token, head), 64 keys at a time: a lane per key for the scores, a lane per dimension for
// the output, one pass with the running maximum and sum.
#include "seq_types.h"

namespace hpmn {

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

template <typename T>
__global__ __launch_bounds__(64) void prefix_attn_rows_kernel(const HpmnPrefixAttn a) {
    __shared__ float qs[128], ps[64];
    const long row = blockIdx.x;                                // (b * Lq + i) * Hq + h
    const int lane = threadIdx.x, h = row % a.Hq, i = (row / a.Hq) % a.Lq, kv = h / (a.Hq / a.Hkv);
    const long b = row / a.Hq / a.Lq;
    const T *q = (const T *)a.q + b * a.q_sb + i * a.q_sl + h * a.q_sh;
    for (int d = lane; d < 128; d += 64) qs[d] = d < a.D ? (float)q[d] * a.scale : 0.f;
    wave_sync();
    const int plen = a.prefix_len ? min(max(*a.prefix_len, 0), a.P) : a.P;
    const int slen = a.suffix_len ? min(max(a.suffix_len[b], 0), a.S) : a.S;
    float m = -INFINITY, l = 0.f, o[2] = {0.f, 0.f};
    for (int part = 0; part < 2; ++part) {
        const int n = part == 0 ? plen : min(max(slen - a.Lq + 1 + i, 0), slen);
        const T *K = part == 0 ? (const T *)a.k_pre + kv * a.kp_sh : (const T *)a.k_suf + b * a.ks_sb + kv * a.ks_sh;
        const T *V = part == 0 ? (const T *)a.v_pre + kv * a.vp_sh : (const T *)a.v_suf + b * a.vs_sb + kv * a.vs_sh;
        const long kst = part == 0 ? a.kp_st : a.ks_st, vst = part == 0 ? a.vp_st : a.vs_st;
        for (int j0 = 0; j0 < n; j0 += 64) {
            float s = -INFINITY;
            if (j0 + lane < n) {
                s = 0.f;
                for (int d = 0; d < a.D; ++d) s = fmaf(qs[d], (float)K[(j0 + lane) * kst + d], s);
            }
            const float mn = fmaxf(m, wave_max(s));
            const float keep = m == -INFINITY ? 0.f : __expf(m - mn);
            const float p = (j0 + lane < n && mn > -INFINITY) ? __expf(s - mn) : 0.f;
            l = l * keep + wave_sum(p);
            m = mn;
            ps[lane] = p;
            wave_sync();
            for (int r = 0; r < 2; ++r) {
                const int d = lane + 64 * r;
                float acc = o[r] * keep;
                if (d < a.D)
                    for (int j = 0; j < min(64, n - j0); ++j) acc = fmaf(ps[j], (float)V[(j0 + j) * vst + d], acc);
                o[r] = acc;
            }
            wave_sync();
        }
    }
    const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);          // (a NaN sum stays one)
    T *out = (T *)a.out + b * a.o_sb + i * a.o_sl + h * a.o_sh;
    for (int r = 0; r < 2; ++r)
        if (lane + 64 * r < a.D) out[lane + 64 * r] = (T)(o[r] * inv);
    if (a.lse && lane == 0) a.lse[row] = l == 0.f ? -INFINITY : m + __logf(l);
}

size_t prefix_attn_workspace_bytes(const HpmnPrefixAttn &) { return 0; }

int prefix_attn_launch(const HpmnPrefixAttn &a, hipStream_t st) {
    const dim3 grid((unsigned)((long)a.B * a.Lq * a.Hq));
    if (a.dtype == HPMN_F32) hipLaunchKernelGGL(prefix_attn_rows_kernel<float>, grid, dim3(64), 0, st, a);
    else if (a.dtype == HPMN_BF16) hipLaunchKernelGGL(prefix_attn_rows_kernel<bf16_t>, grid, dim3(64), 0, st, a);
    else hipLaunchKernelGGL(prefix_attn_rows_kernel<f16_t>, grid, dim3(64), 0, st, a);
    return check_launch();
}

}  // namespace hpmn
