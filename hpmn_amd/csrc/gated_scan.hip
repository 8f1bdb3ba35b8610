// Gated linear recurrence (include/hpmn_hip.h): h_t = a_t h_{t-1} + (1 - a_t) v_t with a = sigmoid(z), forward, backward and
// the one-event step.
//
// First form: one lane per (sequence, channel), the time loop serial in it.
#include "seq_types.h"

namespace hpmn {

constexpr int TILE = HPMN_GATED_SCAN_TILE;

template <typename T>
__global__ __launch_bounds__(64) void gated_scan_fwd_kernel(const HpmnGatedScan a) {
    const int nc = (a.C + 63) / 64;
    const long b = blockIdx.x / nc;
    const int c = (blockIdx.x % nc) * 64 + threadIdx.x;
    if (c >= a.C) return;
    const T *z = (const T *)a.z + b * a.z_sb + c, *v = (const T *)a.v + b * a.v_sb + c;
    const int begin = a.begin ? a.begin[b] : 0;
    const int tiles = (a.T + TILE - 1) / TILE;
    float h = a.h0 ? a.h0[b * a.h0_sb + c] : 0.f;
    for (int t = 0; t < a.T; ++t) {
        if (a.saved && t % TILE == 0) a.saved[(b * tiles + t / TILE) * a.C + c] = h;
        if (t >= begin) {
            float ag, ug;
            gate_pair((float)z[t * a.z_st], ag, ug);
            h = fmaf(ag, h, ug * (float)v[t * a.v_st]);
        }
        if (a.y && (t + 1) % a.period == 0) ((T *)a.y)[b * a.y_sb + ((t + 1) / a.period - 1) * a.y_st + c] = (T)h;
    }
    if (a.h_last) a.h_last[b * a.C + c] = h;
}

template <typename T>
__global__ __launch_bounds__(64) void gated_scan_bwd_kernel(const HpmnGatedScanBwd a) {
    __shared__ float hs[TILE][64];           // the states in front of every step of a tile (a column per lane)
    const int nc = (a.C + 63) / 64;
    const long b = blockIdx.x / nc;
    const int lane = threadIdx.x, c = (blockIdx.x % nc) * 64 + lane;
    if (c >= a.C) return;
    const T *z = (const T *)a.z + b * a.z_sb + c, *v = (const T *)a.v + b * a.v_sb + c;
    const int begin = a.begin ? a.begin[b] : 0;
    const int tiles = (a.T + TILE - 1) / TILE;
    float G = a.d_h_last ? a.d_h_last[b * a.C + c] : 0.f;
    for (int k = tiles - 1; k >= 0; --k) {
        const int t0 = k * TILE, n = min(TILE, a.T - t0);
        float h = a.saved[(b * tiles + k) * a.C + c];
        for (int i = 0; i < n; ++i) {
            hs[i][lane] = h;
            if (t0 + i >= begin) {
                float ag, ug;
                gate_pair((float)z[(t0 + i) * a.z_st], ag, ug);
                h = fmaf(ag, h, ug * (float)v[(t0 + i) * a.v_st]);
            }
        }
        for (int i = n - 1; i >= 0; --i) {
            const long t = t0 + i;
            if (a.d_y && (t + 1) % a.period == 0)
                G += (float)((const T *)a.d_y)[b * a.dy_sb + ((t + 1) / a.period - 1) * a.dy_st + c];
            float dz = 0.f, dv = 0.f;
            if (t >= begin) {
                float ag, ug;
                gate_pair((float)z[t * a.z_st], ag, ug);
                dv = ug * G;
                dz = ag * dv * (hs[i][lane] - (float)v[t * a.v_st]);
                G *= ag;
            }
            ((T *)a.d_z)[b * a.dz_sb + t * a.dz_st + c] = (T)dz;
            ((T *)a.d_v)[b * a.dv_sb + t * a.dv_st + c] = (T)dv;
        }
    }
    if (a.d_h0) a.d_h0[b * a.C + c] = G;
}

__device__ __forceinline__ long step_user(const HpmnGatedStep &a, int b) {
    if (!a.user) return b;
    return (a.flags & HPMN_STEP_USER_I64) ? (long)((const int64_t *)a.user)[b] : (long)((const int32_t *)a.user)[b];
}

// One wave per row.  With HPMN_STEP_COMMIT and a user list, the FIRST row that names a user carries out all rows of that user,
// in row order; the others find an earlier row with their user and leave.
template <typename T>
__global__ __launch_bounds__(64) void gated_step_kernel(const HpmnGatedStep a) {
    const int b = blockIdx.x, lane = threadIdx.x;
    const long u = step_user(a, b);
    const bool ordered = (a.flags & HPMN_STEP_COMMIT) && a.user;
    if (u < 0 || u >= a.n_users) {
        if (a.y)
            for (int c = lane; c < a.C; c += 64) ((T *)a.y)[b * a.y_s + c] = (T)__builtin_nanf("");
        return;
    }
    if (ordered) {
        bool earlier = false;
        for (int j = lane; j < b; j += 64) earlier |= step_user(a, j) == u;
        if (__any(earlier)) return;
    }
    for (int c0 = 0; c0 < a.C; c0 += 64) {
        const int c = c0 + lane;
        const bool on = c < a.C;
        float h = on ? a.state[u * a.state_s + c] : 0.f;
        for (int j = b; j < (ordered ? a.B : b + 1); ++j) {
            if (j > b && step_user(a, j) != u) continue;
            if (!on) continue;
            float ag, ug;
            gate_pair((float)((const T *)a.z)[j * a.z_s + c], ag, ug);
            h = fmaf(ag, h, ug * (float)((const T *)a.v)[j * a.v_s + c]);
            if (a.y) ((T *)a.y)[j * a.y_s + c] = (T)h;
        }
        if (on && (a.flags & HPMN_STEP_COMMIT)) a.state[u * a.state_s + c] = h;
    }
}

size_t gated_scan_workspace_bytes(int, int, int) { return 0; }

int gated_scan_fwd_launch(const HpmnGatedScan &a, hipStream_t st) {
    const dim3 grid((unsigned)((long)a.B * ((a.C + 63) / 64)));
    if (a.dtype == HPMN_F32) hipLaunchKernelGGL(gated_scan_fwd_kernel<float>, grid, dim3(64), 0, st, a);
    else if (a.dtype == HPMN_BF16) hipLaunchKernelGGL(gated_scan_fwd_kernel<bf16_t>, grid, dim3(64), 0, st, a);
    else hipLaunchKernelGGL(gated_scan_fwd_kernel<f16_t>, grid, dim3(64), 0, st, a);
    return check_launch();
}

int gated_scan_bwd_launch(const HpmnGatedScanBwd &a, hipStream_t st) {
    const dim3 grid((unsigned)((long)a.B * ((a.C + 63) / 64)));
    if (a.dtype == HPMN_F32) hipLaunchKernelGGL(gated_scan_bwd_kernel<float>, grid, dim3(64), 0, st, a);
    else if (a.dtype == HPMN_BF16) hipLaunchKernelGGL(gated_scan_bwd_kernel<bf16_t>, grid, dim3(64), 0, st, a);
    else hipLaunchKernelGGL(gated_scan_bwd_kernel<f16_t>, grid, dim3(64), 0, st, a);
    return check_launch();
}

int gated_step_launch(const HpmnGatedStep &a, hipStream_t st) {
    const dim3 grid((unsigned)a.B);
    if (a.dtype == HPMN_F32) hipLaunchKernelGGL(gated_step_kernel<float>, grid, dim3(64), 0, st, a);
    else if (a.dtype == HPMN_BF16) hipLaunchKernelGGL(gated_step_kernel<bf16_t>, grid, dim3(64), 0, st, a);
    else hipLaunchKernelGGL(gated_step_kernel<f16_t>, grid, dim3(64), 0, st, a);
    return check_launch();
}

}  // namespace hpmn
