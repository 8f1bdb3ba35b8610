// extern "C" entries of the sequence operators (include/hpmn_hip.h, ABI v15): argument validation and dispatch.
#include <algorithm>
#include <initializer_list>

#include "seq_types.h"

namespace hpmn {

bool gated_scan_fits(int B, int T, int C);
size_t gated_scan_workspace_bytes(int B, int T, int C);
int gated_scan_fwd_launch(const HpmnGatedScan &a, hipStream_t st);
int gated_scan_bwd_launch(const HpmnGatedScanBwd &a, hipStream_t st);
int gated_step_launch(const HpmnGatedStep &a, hipStream_t st);
size_t prefix_attn_workspace_bytes(const HpmnPrefixAttn &a);
int prefix_attn_launch(const HpmnPrefixAttn &a, hipStream_t st);
int dropout_launch(const HpmnDropout &a, unsigned threshold, hipStream_t st);

static inline bool known_dtype(int d) { return d == HPMN_F32 || d == HPMN_BF16 || d == HPMN_F16; }
static inline bool aligned_to(const void *p, int dtype) { return is_aligned(p, elem_size(dtype)); }

// Sizes that every index of the attention kernels fits: query rows, keys and work items in 31 bits, head groups whole.
static inline int prefix_attn_sizes(const HpmnPrefixAttn &a) {
    if (a.B < 0 || a.Lq < 0 || a.Hq < 1 || a.Hkv < 1 || a.D < 1 || a.P < 0 || a.S < 0 || a.Hq % a.Hkv != 0 || !known_dtype(a.dtype))
        return HPMN_EINVAL;
    if (a.D > 128 || a.P > (1 << 30) || a.S > (1 << 30)) return HPMN_EUNSUPPORTED;
    if ((double)a.B * a.Lq * a.Hq > (double)(1 << 26)) return HPMN_EUNSUPPORTED;
    return HPMN_OK;
}

// Row strides of the scan: 32 bits (offsets are products of 32-bit numbers in 64 bits); steps: their number plus a tile in 31.
static inline bool scan_rows_ok(int T, std::initializer_list<int64_t> s) {
    if (T > (1 << 30)) return false;
    for (int64_t x : s)
        if (T > 1 && x >= (1l << 31)) return false;
    return true;
}

// What a tensor of up to two strided dimensions over dense rows covers.  Strides in bytes; dimensions of one index or of
// stride zero are left out.
struct Region {
    uintptr_t at;
    int64_t n[2] = {1, 1}, s[2] = {0, 0}, width;             // s[0] >= s[1]
    Region(const void *p, int64_t width_) : at(reinterpret_cast<uintptr_t>(p)), width(p ? width_ : 0) {}
    Region(const void *p, int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t row, int64_t esize) : Region(p, row * esize) {
        if (n0 < 1 || n1 < 1) width = 0;
        const bool first = n0 > 1 && s0 > 0, second = n1 > 1 && s1 > 0;
        int i = 0;
        if (first && !(second && s1 > s0)) { n[i] = n0; s[i++] = s0 * esize; }
        if (second) { n[i] = n1; s[i++] = s1 * esize; }
        if (first && second && s1 > s0) { n[i] = n0; s[i++] = s0 * esize; }
    }
    uintptr_t end() const { return at + (n[0] - 1) * s[0] + (n[1] - 1) * s[1] + width; }
};
static inline Region rows_of(const void *p, int64_t n, int64_t stride, int64_t row, int64_t esize) { return Region(p, n, stride, 1, 0, row, esize); }

static inline int64_t gcd(int64_t a, int64_t b) { return b == 0 ? a : gcd(b, a % b); }

// No byte in common.  Two regions in the same stretch of memory are told apart where they are different columns of rows of one pitch
// (the halves of a projection's gradient), or have the same strides (the first and the last steps of one buffer); anything else there is
// taken for an overlap.
static bool apart(const Region &a, const Region &b) {
    if (a.width == 0 || b.width == 0 || a.end() <= b.at || b.end() <= a.at) return true;
    const int64_t delta = (int64_t)(b.at - a.at);            // (as a signed difference)
    const int64_t pitch = gcd(gcd(a.s[0], a.s[1]), gcd(b.s[0], b.s[1]));
    if (pitch > 0) {
        const int64_t col = (delta % pitch + pitch) % pitch;
        if (col >= a.width && col + b.width <= pitch) return true;
    }
    if (a.s[0] != b.s[0] || a.s[1] != b.s[1] || a.s[0] == 0) return false;
    const int64_t inner = (std::max(a.n[1], b.n[1]) - 1) * a.s[1] + std::max(a.width, b.width);      // dimensions are nested: whole inside a step
    if (a.s[0] < inner || (a.s[1] > 0 && a.s[1] < std::max(a.width, b.width))) return false;
    // row (i of b) - (j of a) along a dimension: only those that bring the two together within a step count
    for (int64_t i = -delta / a.s[0] - 1; i <= -delta / a.s[0] + 1; ++i) {
        if (i <= -a.n[0] || i >= b.n[0]) continue;
        const int64_t d = delta + i * a.s[0];
        const int64_t step = a.s[1] > 0 ? a.s[1] : INT64_MAX / 4, near = -d / step;
        for (int64_t j = near - 1; j <= near + 1; ++j) {
            if (j <= -a.n[1] || j >= b.n[1]) continue;
            const int64_t x = j == 0 ? d : d + j * step;
            if (x < a.width && x > -b.width) return false;
        }
    }
    return true;
}
// Every output apart from every input and from the other outputs.
static bool outputs_apart(std::initializer_list<Region> out, std::initializer_list<Region> in) {
    for (const Region *o = out.begin(); o != out.end(); ++o) {
        for (const Region &i : in)
            if (!apart(*o, i)) return false;
        for (const Region *p = out.begin(); p != o; ++p)
            if (!apart(*o, *p)) return false;
    }
    return true;
}

}  // namespace hpmn

using namespace hpmn;

static inline void drop_stale_hip_error() { (void)hipGetLastError(); }

extern "C" {

size_t hpmn_gated_scan_workspace_bytes(int32_t B, int32_t T, int32_t C) {
    if (B < 1 || T < 1 || C < 1 || !gated_scan_fits(B, T, C)) return 0;
    return gated_scan_workspace_bytes(B, T, C);
}

int hpmn_gated_scan_fwd(const HpmnGatedScan *a, void *stream) {
    drop_stale_hip_error();
    if (!a) return HPMN_EINVAL;
    if (a->B < 0 || a->T < 1 || a->C < 1 || a->period < 1 || a->T % a->period != 0 || !known_dtype(a->dtype)) return HPMN_EINVAL;
    if (a->B == 0) return HPMN_OK;
    if (!a->z || !a->v || !(a->y || a->h_last || a->saved)) return HPMN_EINVAL;
    if (!aligned_to(a->z, a->dtype) || !aligned_to(a->v, a->dtype) || !aligned_to(a->y, a->dtype)) return HPMN_EINVAL;
    if (a->z_sb < 0 || a->z_st < 0 || a->v_sb < 0 || a->v_st < 0 || a->h0_sb < 0 || a->y_sb < 0 || a->y_st < 0) return HPMN_EINVAL;
    if (!gated_scan_fits(a->B, a->T, a->C) || !scan_rows_ok(a->T, {a->z_st, a->v_st, a->y_st})) return HPMN_EUNSUPPORTED;
    const size_t need = gated_scan_workspace_bytes(a->B, a->T, a->C);
    if (need > 0 && (!a->workspace || a->workspace_bytes < need || !is_aligned(a->workspace, 16))) return HPMN_EINVAL;
    const int64_t B = a->B, T = a->T, C = a->C, es = elem_size(a->dtype), tiles = (T + HPMN_GATED_SCAN_TILE - 1) / HPMN_GATED_SCAN_TILE;
    if (!outputs_apart({{a->y, B, a->y_sb, T / a->period, a->y_st, C, es}, {a->h_last, B * C * 4}, {a->saved, B * tiles * C * 4}, {a->workspace, (int64_t)need}},
                       {{a->z, B, a->z_sb, T, a->z_st, C, es}, {a->v, B, a->v_sb, T, a->v_st, C, es}, rows_of(a->h0, B, a->h0_sb, C, 4), {a->begin, B * 4}}))
        return HPMN_EINVAL;
    return gated_scan_fwd_launch(*a, (hipStream_t)stream);
}

int hpmn_gated_scan_bwd(const HpmnGatedScanBwd *a, void *stream) {
    drop_stale_hip_error();
    if (!a) return HPMN_EINVAL;
    if (a->B < 0 || a->T < 1 || a->C < 1 || a->period < 1 || a->T % a->period != 0 || !known_dtype(a->dtype)) return HPMN_EINVAL;
    if (a->B == 0) return HPMN_OK;
    if (!a->z || !a->v || !a->saved || !a->d_z || !a->d_v) return HPMN_EINVAL;
    if (!aligned_to(a->z, a->dtype) || !aligned_to(a->v, a->dtype) || !aligned_to(a->d_y, a->dtype) || !aligned_to(a->d_z, a->dtype) ||
        !aligned_to(a->d_v, a->dtype))
        return HPMN_EINVAL;
    if (a->z_sb < 0 || a->z_st < 0 || a->v_sb < 0 || a->v_st < 0 || a->dy_sb < 0 || a->dy_st < 0 || a->dz_sb < 0 || a->dz_st < 0 ||
        a->dv_sb < 0 || a->dv_st < 0)
        return HPMN_EINVAL;
    if (!gated_scan_fits(a->B, a->T, a->C) || !scan_rows_ok(a->T, {a->z_st, a->v_st, a->dy_st, a->dz_st, a->dv_st})) return HPMN_EUNSUPPORTED;
    const size_t need = gated_scan_workspace_bytes(a->B, a->T, a->C);
    if (need > 0 && (!a->workspace || a->workspace_bytes < need || !is_aligned(a->workspace, 16))) return HPMN_EINVAL;
    const int64_t B = a->B, T = a->T, C = a->C, es = elem_size(a->dtype), tiles = (T + HPMN_GATED_SCAN_TILE - 1) / HPMN_GATED_SCAN_TILE;
    if (!outputs_apart({{a->d_z, B, a->dz_sb, T, a->dz_st, C, es}, {a->d_v, B, a->dv_sb, T, a->dv_st, C, es}, {a->d_h0, B * C * 4}, {a->workspace, (int64_t)need}},
                       {{a->z, B, a->z_sb, T, a->z_st, C, es}, {a->v, B, a->v_sb, T, a->v_st, C, es}, {a->saved, B * tiles * C * 4},
                        {a->d_y, B, a->dy_sb, T / a->period, a->dy_st, C, es}, {a->d_h_last, B * C * 4}, {a->begin, B * 4}}))
        return HPMN_EINVAL;
    return gated_scan_bwd_launch(*a, (hipStream_t)stream);
}

int hpmn_gated_scan_step(const HpmnGatedStep *a, void *stream) {
    drop_stale_hip_error();
    if (!a) return HPMN_EINVAL;
    if (a->B < 0 || a->C < 1 || a->n_users < 0 || !known_dtype(a->dtype)) return HPMN_EINVAL;
    if (a->flags & ~(HPMN_STEP_COMMIT | HPMN_STEP_USER_I64)) return HPMN_EINVAL;
    if (a->B == 0) return HPMN_OK;
    if (!a->z || !a->v || (!a->state && a->n_users > 0) || !(a->y || (a->flags & HPMN_STEP_COMMIT))) return HPMN_EINVAL;
    if (!a->user && a->B != a->n_users) return HPMN_EINVAL;
    if (!aligned_to(a->z, a->dtype) || !aligned_to(a->v, a->dtype) || !aligned_to(a->y, a->dtype)) return HPMN_EINVAL;
    if (a->z_s < 0 || a->v_s < 0 || a->y_s < 0 || a->state_s < a->C) return HPMN_EINVAL;
    if (a->user && (a->flags & HPMN_STEP_COMMIT) && a->B > HPMN_STEP_MAX_INDEXED) return HPMN_EUNSUPPORTED;
    if (a->B >= (1 << 26)) return HPMN_EUNSUPPORTED;             // a launch: below 2^32 threads, 64 a row here
    // y may be z's or v's own rows (an element is read before it is written); a committed state is read and written by row, z and v by event
    const int64_t B = a->B, C = a->C, es = elem_size(a->dtype);
    const Region z = rows_of(a->z, B, a->z_s, C, es), v = rows_of(a->v, B, a->v_s, C, es), y = rows_of(a->y, B, a->y_s, C, es);
    const Region state = rows_of(a->state, a->n_users, a->state_s, C, 4), user(a->user, B * (a->flags & HPMN_STEP_USER_I64 ? 8 : 4));
    const auto itself = [&](const void *p, int64_t stride) { return p == a->y && (B == 1 || stride == a->y_s); };
    if (!apart(y, state) || !apart(y, user) || (!itself(a->z, a->z_s) && !apart(y, z)) || (!itself(a->v, a->v_s) && !apart(y, v))) return HPMN_EINVAL;
    if ((a->flags & HPMN_STEP_COMMIT) && !(apart(state, z) && apart(state, v) && apart(state, user))) return HPMN_EINVAL;
    return gated_step_launch(*a, (hipStream_t)stream);
}

int hpmn_dropout(const HpmnDropout *a, void *stream) {
    drop_stale_hip_error();
    if (!a) return HPMN_EINVAL;
    if (a->N < 0 || a->C < 0 || !known_dtype(a->dtype) || !(a->keep_prob > 0.f && a->keep_prob <= 1.f)) return HPMN_EINVAL;
    if (a->N == 0 || a->C == 0) return HPMN_OK;
    if (!a->x || !a->y) return HPMN_EINVAL;
    if (!aligned_to(a->x, a->dtype) || !aligned_to(a->y, a->dtype) || !aligned_to(a->residual, a->dtype)) return HPMN_EINVAL;
    if (!is_aligned(a->rng, 8)) return HPMN_EINVAL;
    if (a->x_s < 0 || a->r_s < 0 || (a->N > 1 && a->y_s < a->C)) return HPMN_EINVAL;
    if (a->N > ((1l << 34) - 1024) / a->C) return HPMN_EUNSUPPORTED;     // a launch: below 2^32 threads, four elements or more each
    const int64_t es = elem_size(a->dtype);
    const Region y = rows_of(a->y, a->N, a->y_s, a->C, es), x = rows_of(a->x, a->N, a->x_s, a->C, es), r = rows_of(a->residual, a->N, a->r_s, a->C, es);
    const auto itself = [&](const void *p, int64_t stride) { return p == a->y && (a->N == 1 || stride == a->y_s); };
    if ((!itself(a->x, a->x_s) && !apart(y, x)) || (!itself(a->residual, a->r_s) && !apart(y, r)) || !apart(y, Region(a->rng, 16))) return HPMN_EINVAL;
    // floor(p 2^16 + 1/2), as a double: p is a float, so the product is exact
    const double q = (double)a->keep_prob * 65536.0 + 0.5;
    const unsigned thr = q < 1.0 ? 1u : (unsigned)q;
    return dropout_launch(*a, thr > 65536u ? 65536u : thr, (hipStream_t)stream);
}

size_t hpmn_prefix_attn_workspace_bytes(const HpmnPrefixAttn *a) {
    if (!a || prefix_attn_sizes(*a) != HPMN_OK || a->B == 0 || a->Lq == 0) return 0;
    return prefix_attn_workspace_bytes(*a);
}

int hpmn_prefix_attn(const HpmnPrefixAttn *a, void *stream) {
    drop_stale_hip_error();
    if (!a) return HPMN_EINVAL;
    const int rc = prefix_attn_sizes(*a);
    if (rc != HPMN_OK) return rc;
    if (a->B == 0 || a->Lq == 0) return HPMN_OK;
    if (!a->q || !a->out || (a->P > 0 && (!a->k_pre || !a->v_pre)) || (a->S > 0 && (!a->k_suf || !a->v_suf))) return HPMN_EINVAL;
    const void *typed[] = {a->q, a->k_pre, a->v_pre, a->k_suf, a->v_suf, a->out};
    for (const void *p : typed)
        if (!aligned_to(p, a->dtype)) return HPMN_EINVAL;
    if (!is_aligned(a->lse, 4) || !is_aligned(a->prefix_len, 4) || !is_aligned(a->suffix_len, 4)) return HPMN_EINVAL;
    const int64_t strides[] = {a->q_sb, a->q_sl, a->q_sh, a->kp_st, a->kp_sh, a->vp_st, a->vp_sh, a->ks_sb, a->ks_st,
                               a->ks_sh, a->vs_sb, a->vs_st, a->vs_sh, a->o_sb, a->o_sl, a->o_sh};
    for (int64_t s : strides)
        if (s < 0) return HPMN_EINVAL;
    if (!(a->scale - a->scale == 0.f)) return HPMN_EINVAL;                       // infinite or NaN
    const size_t need = prefix_attn_workspace_bytes(*a);
    if (need > 0 && (!a->workspace || a->workspace_bytes < need || !is_aligned(a->workspace, 16))) return HPMN_EINVAL;
    return prefix_attn_launch(*a, (hipStream_t)stream);
}

}  // extern "C"
