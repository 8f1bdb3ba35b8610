// Attention of a batch that shares a long prefix: the kernel, a template over the element type (one translation unit per type
// instantiates it: prefix_attn.hip, prefix_attn_bf16.hip, prefix_attn_f16.hip).
//
// The query rows of one key head -- every (sequence, query token, grouped head) -- are a matrix of M = B Lq Hq / Hkv rows against the
// SAME prefix, so the prefix is a matrix product's operand: a workgroup takes 128 rows (or 64, when there are few) and a range of
// keys, and K and V are read once per 128 rows instead of once per row.  One pass with the running maximum and sum:
//   S^T = K Q^T   a wave: 32 query rows (columns of S^T: one row per lane pair, so maximum and sum are a register reduction and ONE
//                 exchange between the wave's halves), 32 keys at a time on the matrix pipe, Q in registers throughout;
//   O^T += V^T P  P is used where it lies: S^T's accumulator layout is the operand layout of the second product up to an order of
//                 the keys, and V is read in that order (16-bit: transposing LDS reads, four keys x 16 columns per 16 lanes).
// K and V tiles go from global memory to LDS directly, the next tile in flight while this one is used; LDS chunks of 16 bytes are
// permuted by the row number so that neither the reads along a row nor those across sixteen rows meet in a bank.
// Few rows: the waves of a workgroup share out the keys of a tile two by two and join their results in LDS.  The key
// axis is split over workgroups until the chip is full; a second kernel joins the parts (maximum, sum, unnormalised output in fp32).
// A row's own suffix is the same thing with M = Lq Hq / Hkv rows and a key limit per row, in the same launch; a few keys of very many
// sequences are left to the joining kernel.
//
// Bound by the matrix pipe and the VALU together for many rows: 512 x 16 heads over 4 of 128, 32768 keys + 64 own bf16, 137.6 GF:
// 160-168 us + 10 us of joining, 0.82-0.86 PF/s in the first kernel (a library product of 8192^3 1.22).  The matrix pipe is busy in
// 44 % of the cycles, 6.6 other VALU instructions to an MFMA take about as many, and few of the two meet: the alternation gains
// little over the sum.  fp16 the same: 16384 keys 93 us.  fp32 (products of 32 x 32 x 2, 137 TF/s at most): 512 x 16 heads over 4 of
// 128, 8192 keys 353 us, 97 TF/s, the matrix pipe busy in 67 % of the cycles, the rest the exponentials and what the one wave a SIMD
// that 348 registers allow cannot hide; 158 x 16 heads over 8 of 96, 7850 keys 108 us, 71 TF/s, 51 %: its 316 rows a key head fill 384.
// Several query tokens: 512 x 48 tokens x 16 heads of 128 over 512 + 48 keys 301 us + 184 of joining, bound by the parts, 409 MB written
// and read.  Bound by launches and round trips for few: 8 rows of 64 over 1000 keys fp32 7.4 + 3.6 us.
//
// Rounding choices: scores, maxima, sums and outputs are fp32; the probabilities are rounded to the 16-bit type once, as operand of
// the second product: half a step of each, so at most half a step of sum p |v| beside the output's own rounding (reached where many
// equal scores are rounded the same way), and about as much as that rounding where they differ.  The sum that divides stays unrounded,
// so that lse is.  A second operand plane for what is rounded off would be half as many products again.  fp16 probabilities are scaled by
// 2^12 (2^15 at most where the maximum lags): unscaled, everything below 2^-24 of the largest would vanish, which for long prefixes
// is most of them; scaled, what is below 2^-26 of it starts to lose digits and 2^-36 vanishes.
#pragma once
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "seq_types.h"

namespace hpmn {

constexpr int JOIN_KEYS = 8;                 // at most so many suffix keys are the second kernel's

struct AttnPlan {
    int mw_pre, mw_suf;                      // waves along the rows (the other 4 / mw along the keys)
    int rt_pre, rt_suf;                      // row tiles per key head / per sequence and key head
    int splits_pre, splits_suf, per_pre, per_suf;   // key ranges and their length
    int parts;                               // splits_pre + splits_suf
    int keys;                                // suffix keys that the second kernel takes itself (then there are no suffix ranges)
    bool join;                               // a second kernel; else results go straight out
    bool vec;                                // 16-byte accesses: whole 16 bytes in a row, aligned pointers and strides
    bool out_vec;                            // outputs four columns at a time
    int d4;                                  // D rounded up to 4: a row of a part
    long rows;                               // Hkv * M
    long o_at;                               // where the parts' outputs start in the workspace, in floats (behind their m and l)
    unsigned blocks_pre, blocks_suf;
};

AttnPlan attn_plan(const HpmnPrefixAttn &a);
template <typename T> int prefix_attn_type(const HpmnPrefixAttn &a, AttnPlan &p, hipStream_t st);

// Keys per tile and LDS bytes of a configuration.
constexpr int attn_sub(int esize, int mw) { return esize == 2 && mw == 4 ? 2 : 1; }
constexpr int attn_tile(int esize, int mw) { return 4 / mw * 32 * attn_sub(esize, mw); }
constexpr size_t attn_lds(int esize, int dp, int mw) {
    const size_t tiles = (size_t)2 * attn_tile(esize, mw) * dp * esize, join = (size_t)4 * 32 * (dp + 4) * 4 + 4 * 32 * 8;
    return mw == 4 ? 2 * tiles : std::max(2 * tiles, join);
}

typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float v8f __attribute__((ext_vector_type(8)));

template <typename T> struct Frag;
template <> struct Frag<bf16_t> {
    typedef bf16x8 type;
    static __device__ __forceinline__ v16f mma(bf16x8 a, bf16x8 b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Frag<f16_t> {
    typedef f16x8 type;
    static __device__ __forceinline__ v16f mma(f16x8 a, f16x8 b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct Frag<float> { typedef v4f type; };

constexpr float LN2 = 0.69314718055994530942f;

// barrier that orders LDS alone: __syncthreads() would wait for the tile in flight
__device__ __forceinline__ void attn_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Position of 16-byte chunk c of row `row`, CPR chunks to a row: the chunk number is permuted so that one chunk of sixteen
// neighbouring rows (K), and four chunks of four neighbouring rows (V), each cover the 64 banks once.
template <int CPR>
__device__ __forceinline__ int chunk_at(int row, int c) {
    const int f = CPR >= 16 ? ((row & 3) << 2) | ((row >> 2) & 3) : CPR == 8 ? ((row & 2) << 1) | ((row >> 2) & 3) : (row >> 2) & 3;
    return row * CPR + (c ^ f);
}

// x of the lane 32 away (one VALU instruction; a shuffle goes through LDS).  The swap exchanges the upper half of its first operand
// with the lower half of its second; the copy is opaque because with two equal operands the compiler takes the two results for one.
__device__ __forceinline__ float other_half(float x) {
    unsigned a = __builtin_bit_cast(unsigned, x), b = a;
    asm volatile("" : "+v"(b));
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    return __builtin_bit_cast(float, (threadIdx.x & 32) ? r[0] : r[1]);
}

struct AttnKeys {
    const void *K, *V;                       // key head's (and sequence's) first row
    int64_t kst, vst;
    int begin, end;                          // this workgroup's keys, inside the length
    int part;
    bool suffix;
    int b, seen;                             // suffix: its sequence, and suffix_len - Lq + 1: query token i sees seen + i keys
};

// Tiles from global memory to LDS without passing registers: instruction i of wave w fills the 64 chunk slots from i * 256 + w * 64 on,
// slot by slot, so a lane picks the chunk that belongs into its slot.  Lanes of columns behind D load nothing: clear_columns() has put
// zeros there (their Q is zero too, but 0 * what lies there could be NaN).  Row strides below 2^24 elements: a tile's lane offsets
// fit 32 bits.
template <typename T, int DP, int KT>
struct TileLoader {
    static constexpr int EPC = 16 / sizeof(T), CPR = DP / EPC, LD = KT * CPR / 256, ROWS = 256 / CPR;
    static constexpr int ALT = ROWS < 16 ? 2 : 1;            // the permutation goes by the low four row bits: every other instruction's
    int row, col[ALT], w;
    bool wide;                               // every column is there (D == DP)
    bool on[ALT];
    unsigned k_off[ALT], v_off[ALT];
    __device__ __forceinline__ TileLoader(const HpmnPrefixAttn &a, const AttnKeys &src) {
        w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int slot = threadIdx.x;
        row = slot / CPR;
        wide = a.D == DP;
#pragma unroll
        for (int j = 0; j < ALT; ++j) {
            col[j] = (chunk_at<CPR>(row + j * ROWS, slot % CPR) - (row + j * ROWS) * CPR) * EPC;
            on[j] = col[j] < a.D;
            k_off[j] = (unsigned)(row * src.kst + col[j]) * (unsigned)sizeof(T);
            v_off[j] = (unsigned)(row * src.vst + col[j]) * (unsigned)sizeof(T);
        }
    }
    // zeros into the first `bytes` of the LDS, before the first tile
    __device__ __forceinline__ void clear_columns(char *lds, int bytes) const {
        if (wide) return;
        attn_barrier();                      // (the LDS may be in use by the code in front)
        for (int i = threadIdx.x; i < bytes / 16; i += 256) *(u32x4 *)(lds + 16 * i) = u32x4{0, 0, 0, 0};
        attn_barrier();
    }
    // rows k0 .. k0 + KT of `from` (all of them there)
    __device__ __forceinline__ void whole(unsigned lds, const void *from, int64_t stride, const unsigned (&lane_off)[ALT], int k0) const {
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const T *base = (const T *)from + (k0 + i * ROWS) * stride;
            const unsigned at = __builtin_amdgcn_readfirstlane(lds + i * 4096 + w * 1024);
            if (wide) {
                asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(lane_off[i % ALT]), "s"(base) : "memory", "m0");
            } else if (on[i % ALT]) {
                asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(lane_off[i % ALT]), "s"(base) : "memory", "m0");
            }
        }
    }
    // rows behind `end` repeat the last one
    __device__ __forceinline__ void partial(unsigned lds, const void *from, int64_t stride, int k0, int end) const {
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const T *at_row = (const T *)from + min(k0 + row + i * ROWS, end - 1) * stride + col[i % ALT];
            const unsigned at = __builtin_amdgcn_readfirstlane(lds + i * 4096 + w * 1024);
            if (on[i % ALT]) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(at_row) : "memory", "m0");
        }
    }
    __device__ __forceinline__ void load(unsigned lds, const void *from, int64_t stride, const unsigned (&lane_off)[ALT], int k0, int end) const {
        if (k0 + KT <= end) whole(lds, from, stride, lane_off, k0);
        else partial(lds, from, stride, k0, end);
    }
};
// The loads of this wave have arrived, and then those of all.
__device__ __forceinline__ void attn_arrive() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// The whole tile pairs of a prefix range for 128 rows, 16-bit types: the part where the time goes.  A SIMD overlaps the matrix pipe
// with the VALU only where ONE wave's instructions alternate (measured: an MFMA with three fma and an exp behind it 36 cycles, alone
// 32.5; the same work in two waves, each in its own phase: the sum), so every step of 32 keys carries three pipeline stages:
//   step s:  scores of s + 2 (K Q^T),  products of s (V^T P),  and on the VALU the probabilities of s + 1 and the maximum of s + 2.
// The maximum raised at the end of step s scales the probabilities from s + 2 on; the output is rescaled a step later, when
// the products of s + 1 are in it.  Tiles of 64 keys.  K is
// needed a tile before V: after the barrier in front of tile k, K(k + 1) and V(k) are there, and the buffers of K(k) and V(k - 1)
// are free, so two buffers each, one barrier per tile, and a tile's time for the loads.  Tiles go in pairs so that buffers are
// constants and an LDS address is one of NX + DT registers and an immediate.
template <typename T, int DP, int DC>
__device__ __forceinline__ void attend_whole_tiles(const HpmnPrefixAttn &a, char *lds, const AttnKeys &src, int full,
                                                   const typename Frag<T>::type (&qf)[DC / 16], float c, float off, float lazy,
                                                   v16f (&o)[DC / 32], float &m, float &l) {
    constexpr int KT = 64, CPR = DP / 8, NX = DC / 16, DT = DC / 32, BUF = KT * DP * 2;
    typedef typename Frag<T>::type frag;
    typedef __attribute__((address_space(3))) char lds_char;
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    typedef __attribute__((address_space(3))) frag lds_frag;
    const int lane = threadIdx.x & 63, half = lane >> 5, n = lane & 31;
    lds_char *Kt = (lds_char *)lds, *Vt = Kt + 2 * BUF;

    const TileLoader<T, DP, KT> loader(a, src);
    const unsigned lds0 = (unsigned)(uintptr_t)Kt;
    auto load_k = [&](int k) { loader.whole(lds0 + (k & 1) * BUF, src.K, src.kst, loader.k_off, src.begin + k * KT); };
    auto load_v = [&](int k) { loader.whole(lds0 + (2 + (k & 1)) * BUF, src.V, src.vst, loader.v_off, src.begin + k * KT); };

    // LDS addresses: rows 16 and 32 further and the buffer are immediates (they leave the low four row bits, so the permutation, alone)
    const int l16 = lane & 15, vrow = 4 * half + (l16 >> 2), vc = 2 * ((lane >> 4) & 1) + ((l16 & 3) >> 1);
    lds_char *ka[NX], *va[DT][2];
#pragma unroll
    for (int x = 0; x < NX; ++x) ka[x] = Kt + 16 * chunk_at<CPR>(n, 2 * x + half);
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j) va[t][j] = Vt + 16 * chunk_at<CPR>(vrow + 8 * j, 4 * t + vc) + 8 * (l16 & 1);
    auto scores = [&](int buf, int u) {
        v16f s = {};
#pragma unroll
        for (int x = 0; x < NX; ++x) s = Frag<T>::mma(*(const lds_frag *)(ka[x] + buf * BUF + 32 * u * CPR * 16), qf[x], s);
        return s;
    };
    auto top = [&](const v16f &s) {
        float mx = fmaxf(fmaxf(s[0], s[1]), s[2]);
#pragma unroll
        for (int i = 3; i < 15; i += 2) mx = fmaxf(fmaxf(mx, s[i]), s[i + 1]);
        mx = fmaxf(mx, s[15]);
        return fmaxf(mx, other_half(mx)) * c;
    };
    float pending = 1.f;                     // what the output still has to be multiplied with
    auto settle_output = [&](float pending) {
        if (__any(pending != 1.f)) {
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[t][i] *= pending;
        }
    };
    auto raise = [&](float mx) {             // (no branch: it is on the way of the interleaved instructions)
        const float mn = mx > m + lazy ? mx : m;
        pending = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= pending;
    };
    auto probabilities = [&](const v16f &s, frag (&p)[2]) {
        const float mo = off - m;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            v8f e;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                e[i] = __builtin_amdgcn_exp2f(fmaf(s[8 * g + i], c, mo));
                l += e[i];
            }
            p[g] = __builtin_convertvector(e, frag);
        }
    };
    // step (buffer vb, u): s1: scores of the next step, turned into p1; p0: this step's probabilities; leaves the scores of the step
    // after next in s2
    auto step = [&](int vb, int kb, int u, const frag (&p0)[2], const v16f &s1, frag (&p1)[2], v16f &s2, float cap) {
        frag kf[NX], vf[2][DT];
        v16f cur = s1;
        asm volatile("" : "+v"(cur));        // (nothing of this step moves in front of it)
#pragma unroll
        for (int x = 0; x < NX; ++x) kf[x] = *(const lds_frag *)(ka[x] + kb * BUF + 32 * u * CPR * 16);
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                union { s16x4 q[2]; frag f; } v;
                const int at = vb * BUF + (32 * u + 16 * g) * CPR * 16;
                v.q[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(va[t][0] + at));
                v.q[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(va[t][1] + at));
                vf[g][t] = v.f;
            }
        probabilities(cur, p1);
        v16f s = {};
#pragma unroll
        for (int x = 0; x < NX; ++x) s = Frag<T>::mma(kf[x], qf[x], s);
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int t = 0; t < DT; ++t) o[t] = Frag<T>::mma(vf[g][t], p0[g], o[t]);
        s2 = s;
        const float mx = fminf(top(s), cap);     // (cap: whether the step after next exists; no branch)
        const float scale_out = pending;
        raise(mx);
        asm volatile("" : "+v"(p1[0]), "+v"(p1[1]), "+v"(m), "+v"(l));              // (and nothing is left for later)
        // the order: both operand sets from LDS, then an MFMA and a share of the VALU work in turn
        __builtin_amdgcn_sched_group_barrier(0x100, NX, 0);
#pragma unroll
        for (int x = 0; x < NX; ++x) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 4 * DT / NX, 0);
            __builtin_amdgcn_sched_group_barrier(0x400, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);
        }
#pragma unroll
        for (int x = 0; x < 2 * DT; ++x) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x400, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
        }
        settle_output(scale_out);
    };
    loader.clear_columns(lds, 4 * BUF);
    load_k(0);
    load_v(0);
    load_k(1);
    attn_arrive();
    v16f sa = scores(0, 0), sb = scores(0, 1);
    frag pa[2], pb[2];
    raise(top(sa));                                          // (the output is still zero)
    probabilities(sa, pa);
    raise(top(sb));
    for (int k = 0; k < full; k += 2) {
        attn_arrive();                                       // K(k + 1) and V(k) are there; K(k) and V(k - 1) have been read by all
        if (k + 2 < full) load_k(k + 2);
        load_v(k + 1);
        step(0, 1, 0, pa, sb, pb, sa, FLT_MAX);
        step(0, 1, 1, pb, sa, pa, sb, FLT_MAX);
        attn_arrive();
        if (k + 3 < full) load_k(k + 3);
        if (k + 2 < full) load_v(k + 2);
        const float cap = k + 2 < full ? FLT_MAX : -FLT_MAX;
        step(1, 0, 0, pa, sb, pb, sa, cap);
        const float before = l;
        step(1, 0, 1, pb, sa, pa, sb, cap);
        if (k + 2 >= full) l = before;       // (there was no next step whose probabilities could count)
    }
}

template <typename T, int DP, int DC, bool VEC, int MW>
__device__ __forceinline__ void attend(const HpmnPrefixAttn &a, const AttnPlan &p, char *lds, const AttnKeys &src, int kvh, int row0,
                                       int row_end) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int KW = 4 / MW, SUB = attn_sub(sizeof(T), MW), KT = attn_tile(sizeof(T), MW);
    constexpr int EPC = 16 / sizeof(T), CPR = DP / EPC, LD = KT * CPR / 256, DT = DC / 32;
    constexpr bool F16 = std::is_same<T, f16_t>::value;
    // probabilities are taken times 2^OFF, and the maximum may lag by 2^LAZY before the output is rescaled: fp16's largest, 2^15, is met
    constexpr float OFF = F16 ? 12.f : 0.f, LAZY = F16 ? 3.f : 8.f;
    typedef typename Frag<T>::type frag;
    constexpr int BUF = 2 * KT * DP * (int)sizeof(T);    // K and V of a tile; two of them
    char *Kt = lds, *Vt = lds + BUF / 2;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5, n = lane & 31;
    const int mw = w % MW, kw = w / MW;
    const int group = a.Hq / a.Hkv, per_seq = a.Lq * group;
    const int row = row0 + mw * 32 + n;
    const bool active = row0 + mw * 32 < row_end;       // (wave-uniform)
    const int r = min(row, row_end - 1);
    const int in_seq = src.suffix ? r : r % per_seq, b = src.suffix ? src.b : r / per_seq;
    const int tok = in_seq / group, h = kvh * group + in_seq % group;
    const int limit = src.suffix ? min(src.end, max(0, src.seen + tok)) : src.end;

    // Q: column `row` of the first product's second operand, d in the order of the chunks this half of the wave reads
    frag qf[DC / (2 * EPC)];
    {
        const T *q = (const T *)a.q + b * a.q_sb + tok * a.q_sl + h * a.q_sh;
#pragma unroll
        for (int s = 0; s < DC / (2 * EPC); ++s) {
            const int d0 = (2 * s + half) * EPC;
            if constexpr (VEC) {
                const frag x = *(const frag *)(q + (d0 < a.D ? d0 : 0));
#pragma unroll
                for (int e = 0; e < EPC; ++e) qf[s][e] = d0 < a.D ? x[e] : (T)0.f;
            } else {
#pragma unroll
                for (int e = 0; e < EPC; ++e) {
                    const T x = q[min(d0 + e, a.D - 1)];
                    qf[s][e] = d0 + e < a.D ? x : (T)0.f;
                }
            }
        }
        // a negative scale becomes a sign of q, a zero one a zero q: what multiplies the scores is positive
        if (a.scale <= 0.f) {
#pragma unroll
            for (int s = 0; s < DC / (2 * EPC); ++s)
#pragma unroll
                for (int e = 0; e < EPC; ++e) qf[s][e] = a.scale < 0.f ? -qf[s][e] : (T)0.f;
        }
    }
    const float c = a.scale == 0.f ? 1.f : -NEG_LOG2E * fabsf(a.scale);

    // What no 16-byte access can take (VEC false): element by element through registers, the next tile in flight.  This thread's
    // chunks: one column of chunks, rows 256 / CPR apart.
    const int lc = tid % CPR, lrow = tid / CPR;
    u32x4 kr[VEC ? 1 : LD], vr[VEC ? 1 : LD];
    auto fetch = [&](int k0) {
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const int key = min(k0 + lrow + i * (256 / CPR), src.end - 1);
            const T *k = (const T *)src.K + key * src.kst, *v = (const T *)src.V + key * src.vst;
            union { T e[EPC]; u32x4 u; } x, y;
#pragma unroll
            for (int e = 0; e < EPC; ++e) {
                const int d = lc * EPC + e;
                const T ke = k[min(d, a.D - 1)], ve = v[min(d, a.D - 1)];
                x.e[e] = d < a.D ? ke : (T)0.f;
                y.e[e] = d < a.D ? ve : (T)0.f;
            }
            kr[i] = x.u;
            vr[i] = y.u;
        }
    };
    auto stage = [&](int k0, int buf) {
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const int lr = lrow + i * (256 / CPR);
            const bool there = k0 + lr < src.end;            // (zeros, not what lies there: 0 * NaN)
            *(u32x4 *)(Kt + buf + 16 * chunk_at<CPR>(lr, lc)) = there ? kr[i] : u32x4{0, 0, 0, 0};
            *(u32x4 *)(Vt + buf + 16 * chunk_at<CPR>(lr, lc)) = there ? vr[i] : u32x4{0, 0, 0, 0};
        }
    };

    v16f o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = 0.f;
    float m = -FLT_MAX, l = 0.f;

    int start = src.begin;
    if constexpr (!F32 && MW == 4 && VEC) {
        const int full = (src.end - src.begin) / (2 * KT) * 2;
        if (!src.suffix && full > 0) {
            attend_whole_tiles<T, DP, DC>(a, lds, src, full, qf, c, OFF, LAZY, o, m, l);
            start = src.begin + full * KT;
        }
    }
    const TileLoader<T, DP, KT> loader(a, src);
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    auto load = [&](int k0, int buf) {
        loader.load(lds0 + buf, src.K, src.kst, loader.k_off, k0, src.end);
        loader.load(lds0 + buf + BUF / 2, src.V, src.vst, loader.v_off, k0, src.end);
    };
    int buf = 0;
    if (start < src.end) {
        if constexpr (VEC) {
            attn_barrier();                                  // (the LDS may be in use by the code in front)
            loader.clear_columns(lds, 2 * BUF);
            load(start, 0);
        } else {
            fetch(start);
            stage(start, 0);
        }
    }
    for (int k0 = start; k0 < src.end; k0 += KT, buf ^= BUF) {
        // this tile is there, and the last one, whose buffer the next one takes, has been read by all
        if constexpr (VEC) {
            attn_arrive();
            if (k0 + KT < src.end) load(k0 + KT, buf ^ BUF);
            else if (k0 + KT > src.end) {                    // V behind the end: zeros, not repeated rows (0 * inf)
                for (int i = tid; i < (k0 + KT - src.end) * CPR; i += 256)
                    *(u32x4 *)(Vt + buf + 16 * (src.end - k0) * CPR + 16 * i) = u32x4{0, 0, 0, 0};
                attn_barrier();
            }
        } else {
            attn_barrier();
            if (k0 + KT < src.end) fetch(k0 + KT);
        }
        const auto last = [&] {                              // (registers to LDS once this tile has been used)
            if constexpr (!VEC)
                if (k0 + KT < src.end) stage(k0 + KT, buf ^ BUF);
        };
        const int kb = kw * 32 * SUB;
        if (!active || k0 + kb >= src.end) {
            last();
            continue;
        }
        v16f s[SUB];
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[u][i] = 0.f;
#pragma unroll
            for (int x = 0; x < DC / (2 * EPC); ++x) {
                const frag kf = *(const frag *)(Kt + buf + 16 * chunk_at<CPR>(kb + 32 * u + n, 2 * x + half));
                if constexpr (F32) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[u] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[e], qf[x][e], s[u], 0, 0, 0);
                } else {
                    s[u] = Frag<T>::mma(kf, qf[x], s[u]);
                }
            }
        }
        if (src.suffix || k0 + KT > src.end) {
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (k0 + kb + 32 * u + 8 * (i / 4) + 4 * half + i % 4 >= limit) s[u][i] = -INFINITY;
        }
        float mx = s[0][0];
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[u][i]);
        mx = fmaxf(mx, other_half(mx)) * c;
        if (__any(mx > m + LAZY)) {
            const float mn = fmaxf(m, mx), keep = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= keep;
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[t][i] *= keep;
        }
        const float mo = OFF - m;
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[u][i] = __builtin_amdgcn_exp2f(fmaf(s[u][i], c, mo));
                l += s[u][i];
            }
            if constexpr (F32) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int vrow = kb + 32 * u + 8 * (i / 4) + 4 * half + i % 4;
#pragma unroll
                    for (int t = 0; t < DT; ++t) {
                        const int d = 32 * t + n;
                        const float v = *(const float *)(Vt + buf + 16 * chunk_at<CPR>(vrow, d / 4) + 4 * (d % 4));
                        o[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, s[u][i], o[t], 0, 0, 0);
                    }
                }
            } else {
                typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
                const int l16 = lane & 15, vr0 = kb + 32 * u + 4 * half + (l16 >> 2), vc = 2 * ((lane >> 4) & 1) + ((l16 & 3) >> 1);
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    v8f pf;
#pragma unroll
                    for (int i = 0; i < 8; ++i) pf[i] = s[u][8 * g + i];
                    const frag pb = __builtin_convertvector(pf, frag);
#pragma unroll
                    for (int t = 0; t < DT; ++t) {
                        union { s16x4 q[2]; frag f; } x;
                        x.q[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(Vt + buf + 16 * chunk_at<CPR>(vr0 + 16 * g, 4 * t + vc) + 8 * (l16 & 1)));
                        x.q[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(Vt + buf + 16 * chunk_at<CPR>(vr0 + 16 * g + 8, 4 * t + vc) + 8 * (l16 & 1)));
                        o[t] = Frag<T>::mma(x.f, pb, o[t]);
                    }
                }
            }
        }
        last();
    }
    l += __shfl_xor(l, 32);
    m -= OFF;

    // results: quads of four neighbouring d of a row
    float *ml = (float *)a.workspace, *parts = ml + p.o_at;
    const long M = p.rows / a.Hkv;
    auto put_ml = [&](int rr, int bb, int tt, int hh, float mm, float ll) {
        if (p.join) {
            float *at = ml + (src.part * p.rows + kvh * M + (src.suffix ? (long)bb * per_seq : 0) + rr) * 2;
            at[0] = mm;
            at[1] = ll;
        } else if (a.lse) {
            a.lse[((long)bb * a.Lq + tt) * a.Hq + hh] = ll == 0.f ? -INFINITY : (mm + __builtin_amdgcn_logf(ll)) * LN2;
        }
    };
    auto put_quad = [&](int rr, int bb, int tt, int hh, int d, v4f x, float ll) {
        if (d >= a.D) return;
        if (p.join) {
            *(v4f *)(parts + (src.part * p.rows + kvh * M + (src.suffix ? (long)bb * per_seq : 0) + rr) * p.d4 + d) = x;
        } else {
            const float inv = ll == 0.f ? 0.f : 1.0f / ll;
            T *out = (T *)a.out + bb * a.o_sb + tt * a.o_sl + hh * a.o_sh + d;
            if (p.out_vec) store_quad<T, true>(out, x * inv, 4);
            else store_quad<T, false>(out, x * inv, a.D - d);
        }
    };
    if constexpr (KW == 1) {
        if (row >= row_end) return;
        if (half == 0) put_ml(row, b, tok, h, m, l);
        if (l == 0.f && p.join) return;             // (nothing was seen: the second kernel does not look)
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                put_quad(row, b, tok, h, 32 * t + 8 * g + 4 * half, v4f{o[t][4 * g], o[t][4 * g + 1], o[t][4 * g + 2], o[t][4 * g + 3]}, l);
    } else {
        constexpr int RS = DC + 4;                       // a row of the join, in floats
        float *ob = (float *)lds, *mb = ob + 4 * 32 * RS;
        attn_barrier();
        if (active) {
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *(v4f *)(ob + (w * 32 + n) * RS + 32 * t + 8 * g + 4 * half) = v4f{o[t][4 * g], o[t][4 * g + 1], o[t][4 * g + 2], o[t][4 * g + 3]};
            if (half == 0) {
                mb[(w * 32 + n) * 2] = m;
                mb[(w * 32 + n) * 2 + 1] = l;
            }
        }
        attn_barrier();
        for (int i = tid; i < MW * 32 * (DC / 4); i += 256) {
            const int jr = i / (DC / 4), d = i % (DC / 4) * 4, rr = row0 + jr;
            if (rr >= row_end) break;
            float mm = -FLT_MAX, ll = 0.f;
#pragma unroll
            for (int k = 0; k < KW; ++k) mm = fmaxf(mm, mb[((k * MW + jr / 32) * 32 + jr % 32) * 2]);
            v4f x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < KW; ++k) {
                const int at = (k * MW + jr / 32) * 32 + jr % 32;
                const float f = __builtin_amdgcn_exp2f(mb[at * 2] - mm);
                ll += f * mb[at * 2 + 1];
                x += f * *(const v4f *)(ob + at * RS + d);
            }
            const int is = src.suffix ? rr : rr % per_seq, bb = src.suffix ? src.b : rr / per_seq;
            if (d == 0) put_ml(rr, bb, is / group, kvh * group + is % group, mm, ll);
            put_quad(rr, bb, is / group, kvh * group + is % group, d, x, ll);
        }
    }
}

template <typename T, int DP, int DC, bool VEC, int MWP, int MWS>
__global__ __launch_bounds__(256, (sizeof(T) == 4 && (DC == 128 || (DC == 96 && !VEC))) ? 1 : 2) void prefix_attn_kernel(const HpmnPrefixAttn a, const AttnPlan p) {
    extern __shared__ char attn_smem[];
    const int group = a.Hq / a.Hkv;
    AttnKeys k;
    if (blockIdx.x < p.blocks_pre) {
        // the row tiles of one key range on one XCD (workgroups go round the eight): its L2 then holds the range
        const unsigned x = blockIdx.x % 8, j = blockIdx.x / 8;
        const int g = (int)(j / p.rt_pre * 8 + x);
        if (g >= a.Hkv * p.splits_pre) return;
        const int kvh = g / p.splits_pre, split = g % p.splits_pre, rt = (int)(j % p.rt_pre);
        const int len = a.prefix_len ? min(max(*a.prefix_len, 0), a.P) : a.P;
        k.K = (const T *)a.k_pre + kvh * a.kp_sh;
        k.V = (const T *)a.v_pre + kvh * a.vp_sh;
        k.kst = a.kp_st;
        k.vst = a.vp_st;
        k.begin = split * p.per_pre;
        k.end = min(len, k.begin + p.per_pre);
        k.part = split;
        k.suffix = false;
        k.b = k.seen = 0;
        attend<T, DP, DC, VEC, MWP>(a, p, attn_smem, k, kvh, rt * 32 * MWP, a.B * a.Lq * group);
    } else {
        unsigned j = blockIdx.x - p.blocks_pre;
        const int rt = j % p.rt_suf;
        j /= p.rt_suf;
        const int split = j % p.splits_suf;
        j /= p.splits_suf;
        const int kvh = j % a.Hkv, b = j / a.Hkv;
        const int len = a.suffix_len ? min(max(a.suffix_len[b], 0), a.S) : a.S;
        k.K = (const T *)a.k_suf + b * a.ks_sb + kvh * a.ks_sh;
        k.V = (const T *)a.v_suf + b * a.vs_sb + kvh * a.vs_sh;
        k.kst = a.ks_st;
        k.vst = a.vs_st;
        k.begin = split * p.per_suf;
        k.end = min(len, k.begin + p.per_suf);
        k.part = p.splits_pre + split;
        k.suffix = true;
        k.b = b;
        k.seen = len - a.Lq + 1;
        attend<T, DP, DC, VEC, MWS>(a, p, attn_smem, k, kvh, rt * 32 * MWS, a.Lq * group);
    }
}

// Second kernel: joins a row's parts.  Groups of 32 lanes (a quad of the row each, D <= 128) take the parts in turn, BATCH at a
// time; BLOCK: a workgroup of eight groups per row, else a wave of two.  What the parts hold was written by other XCDs, a round trip to
// memory is most of this kernel: a batch's outputs are asked for before its weights are known, and both in one go.
// OWN > 0: the few keys of a short suffix are parts too, of one key each (the score is the maximum, the value the output), OWN to a group,
// grp, grp + GROUPS ...; VEC: their rows and q's in aligned quads.
template <typename T, bool BLOCK, int BATCH, int OWN, bool VEC>
__global__ __launch_bounds__(256) void prefix_attn_join_kernel(const HpmnPrefixAttn a, const AttnPlan p) {
    constexpr int GROUPS = BLOCK ? 8 : 2;
    __shared__ v4f sums[8][32];
    __shared__ float ls[8], ms[8];
    const long R = BLOCK ? (long)blockIdx.x : (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (R >= p.rows) return;                             // (whole waves; BLOCK: never)
    const int lane = threadIdx.x & 63, q = lane & 31, grp = BLOCK ? (int)threadIdx.x >> 5 : lane >> 5;
    const float *ml = (const float *)a.workspace, *parts = ml + p.o_at;
    const int d0 = min(4 * q, p.d4 - 4);
    int kvh, b, tok, h;
    const auto locate = [&] {                            // the row's place (32-bit divisions: all rows are at most 2^26)
        const unsigned group = a.Hq / a.Hkv, per_seq = a.Lq * group, M = a.B * per_seq, row = (unsigned)R, r = row % M, is = r % per_seq;
        kvh = row / M;
        b = r / per_seq;
        tok = is / group;
        h = kvh * group + is % group;
    };
    float m = -FLT_MAX, l = 0.f;
    v4f x = {0.f, 0.f, 0.f, 0.f};
    quad_t<T> qf, kf[OWN ? OWN : 1], vf[OWN ? OWN : 1];
    if constexpr (OWN > 0) {                             // asked for before the parts; what is not to be seen is loaded and not used
        locate();
        const T *Q = (const T *)a.q + b * a.q_sb + tok * a.q_sl + h * a.q_sh;
        const T *K = (const T *)a.k_suf + b * a.ks_sb + kvh * a.ks_sh, *V = (const T *)a.v_suf + b * a.vs_sb + kvh * a.vs_sh;
        qf = load_quad<T, VEC>(Q + d0, a.D - d0);        // (d0 < D; columns behind D: anything)
#pragma unroll
        for (int j = 0; j < OWN; ++j) {
            const int key = min(grp + j * GROUPS, a.S - 1);
            kf[j] = load_quad<T, VEC>(K + key * a.ks_st + d0, a.D - d0);
            vf[j] = load_quad<T, VEC>(V + key * a.vs_st + d0, a.D - d0);
        }
    }
    for (int k0 = grp; k0 < p.parts; k0 += BATCH * GROUPS) {
        v4f o[BATCH];
        const int first = __builtin_amdgcn_readfirstlane(k0);
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {                // (one behind the last part: the last one again, with weight zero)
            o[j] = v4f{0.f, 0.f, 0.f, 0.f};
            if (first + j * GROUPS < p.parts) o[j] = *(const v4f *)(parts + ((long)min(k0 + j * GROUPS, p.parts - 1) * p.rows + R) * p.d4 + d0);
        }
        const int mine = k0 + (q % BATCH) * GROUPS;      // lane q: part q of the batch
        const float *at = ml + ((long)min(mine, p.parts - 1) * p.rows + R) * 2;
        const float mk = at[0], lk = mine < p.parts ? at[1] : 0.f;
        float mn = lk != 0.f ? mk : -FLT_MAX;
#pragma unroll
        for (int d = BATCH / 2; d > 0; d >>= 1) mn = fmaxf(mn, __shfl_xor(mn, d));
        mn = fmaxf(mn, m);
        const float keep = __builtin_amdgcn_exp2f(m - mn), f = lk != 0.f ? __builtin_amdgcn_exp2f(mk - mn) : 0.f;
        float lb = f * lk;
#pragma unroll
        for (int d = BATCH / 2; d > 0; d >>= 1) lb += __shfl_xor(lb, d);
        m = mn;
        l = l * keep + lb;
        x *= keep;
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
            const float fj = __shfl(f, (lane & 32) + j);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] += fj != 0.f ? fj * o[j][i] : 0.f;       // (an empty part was not written)
        }
    }
    if constexpr (OWN > 0) {
        const int len = a.suffix_len ? min(max(a.suffix_len[b], 0), a.S) : a.S, limit = min(len, len - a.Lq + 1 + tok);
        const float c = a.scale == 0.f ? 1.f : -NEG_LOG2E * fabsf(a.scale);
        float sc[OWN], mn = m;
#pragma unroll
        for (int j = 0; j < OWN; ++j) {
            sc[j] = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = a.scale == 0.f ? 0.f : a.scale < 0.f ? -(float)qf[i] : (float)qf[i];
                sc[j] = 4 * q + i < a.D ? fmaf(e, (float)kf[j][i], sc[j]) : sc[j];
            }
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) sc[j] += __shfl_xor(sc[j], d);
            sc[j] *= c;
            if (grp + j * GROUPS < limit) mn = fmaxf(mn, sc[j]);
        }
        const float keep = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= keep;
        x *= keep;
#pragma unroll
        for (int j = 0; j < OWN; ++j) {
            if (grp + j * GROUPS >= limit) break;
            const float f = __builtin_amdgcn_exp2f(sc[j] - mn);
            l += f;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = fmaf(f, (float)vf[j][i], x[i]);
        }
    }
    // the groups' results
    if (BLOCK) {
        sums[grp][q] = x;
        if (q == 0) {
            ls[grp] = l;
            ms[grp] = m;
        }
        __syncthreads();
        if (threadIdx.x >= 32) return;
        for (int g = 0; g < 8; ++g) m = fmaxf(m, ms[g]);
        l = 0.f;
        x = v4f{0.f, 0.f, 0.f, 0.f};
        for (int g = 0; g < 8; ++g) {
            const float f = __builtin_amdgcn_exp2f(ms[g] - m);
            x += f * sums[g][q];
            l += f * ls[g];
        }
    } else {
        const float mo = __shfl_xor(m, 32), lo = __shfl_xor(l, 32), mn = fmaxf(m, mo);
        const float f = __builtin_amdgcn_exp2f(m - mn), fo = __builtin_amdgcn_exp2f(mo - mn);
        l = f * l + fo * lo;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = f * x[i] + fo * __shfl_xor(x[i], 32);
        m = mn;
        if (lane >= 32) return;
    }
    if constexpr (OWN == 0) locate();
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    T *out = (T *)a.out + b * a.o_sb + tok * a.o_sl + h * a.o_sh + 4 * q;
    if (4 * q < a.D) {
        if (p.out_vec) store_quad<T, true>(out, x * inv, 4);
        else store_quad<T, false>(out, x * inv, a.D - 4 * q);
    }
    if (a.lse && q == 0) a.lse[((long)b * a.Lq + tok) * a.Hq + h] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * LN2;
}

template <typename T, bool BLOCK, int BATCH, int OWN, bool VEC>
static void attn_join(const HpmnPrefixAttn &a, const AttnPlan &p, long blocks, hipStream_t st) {
    const dim3 grid((unsigned)blocks);
    if (p.keys > 0) hipLaunchKernelGGL((prefix_attn_join_kernel<T, BLOCK, BATCH, OWN, VEC>), grid, dim3(256), 0, st, a, p);
    else hipLaunchKernelGGL((prefix_attn_join_kernel<T, BLOCK, BATCH, 0, true>), grid, dim3(256), 0, st, a, p);
}

template <typename T, int DP, int DC, bool VEC, int MWP, int MWS>
static int attn_go(const HpmnPrefixAttn &a, const AttnPlan &p, hipStream_t st) {
    const size_t lds = std::max(attn_lds(sizeof(T), DP, MWP), attn_lds(sizeof(T), DP, MWS));
    auto kernel = prefix_attn_kernel<T, DP, DC, VEC, MWP, MWS>;
    if (lds > 64 * 1024) {
        hipError_t e = hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) {
            set_last_hip_error((int)e);
            return HPMN_EHIP;
        }
    }
    hipLaunchKernelGGL(kernel, dim3(p.blocks_pre + p.blocks_suf), dim3(256), lds, st, a, p);
    int rc = check_launch();
    if (rc == HPMN_OK && p.join) {
        const int parts = p.parts + p.keys;
        // a workgroup per row while that makes up to eight a CU or the parts are many; batches that the parts fill (16 where 4 would
        // do: 1600 rows of 19 parts 5.8 -> 7.4 us; 4 where 16 do: 64 rows of 128 parts 4.6 -> 8.9)
        if (p.rows <= 2048 || parts > 64) {
            if (p.parts > 32) attn_join<T, true, 16, 1, VEC>(a, p, p.rows, st);
            else attn_join<T, true, 4, 1, VEC>(a, p, p.rows, st);
        } else if (p.keys <= 2) {
            attn_join<T, false, 8, 1, VEC>(a, p, (p.rows + 3) / 4, st);
        } else {
            attn_join<T, false, 8, JOIN_KEYS / 2, VEC>(a, p, (p.rows + 3) / 4, st);
        }
        rc = check_launch();
    }
    return rc;
}

template <typename T, int DP, int DC, bool VEC>
static int attn_rows(const HpmnPrefixAttn &a, const AttnPlan &p, hipStream_t st) {
    if (p.mw_pre == 4) return p.mw_suf == 4 ? attn_go<T, DP, DC, VEC, 4, 4>(a, p, st) : attn_go<T, DP, DC, VEC, 4, 2>(a, p, st);
    return attn_go<T, DP, DC, VEC, 2, 2>(a, p, st);
}

// Columns: LDS rows of 32, 64 or 128, of which 96 are multiplied for D in 65 .. 96 (fewer registers, so fp32 has two
// waves a SIMD: 158 x 16 heads over 8 of 96, 7850 keys 145 -> 115 us; bf16, 512 x 16 heads over 4 of 96, 8192 keys 60.2 -> 54.1).
template <typename T>
static int attn_width(const HpmnPrefixAttn &a, const AttnPlan &p, hipStream_t st) {
    if (a.D <= 32) return p.vec ? attn_rows<T, 32, 32, true>(a, p, st) : attn_rows<T, 32, 32, false>(a, p, st);
    if (a.D <= 64) return p.vec ? attn_rows<T, 64, 64, true>(a, p, st) : attn_rows<T, 64, 64, false>(a, p, st);
    if (a.D <= 96) return p.vec ? attn_rows<T, 128, 96, true>(a, p, st) : attn_rows<T, 128, 96, false>(a, p, st);
    return p.vec ? attn_rows<T, 128, 128, true>(a, p, st) : attn_rows<T, 128, 128, false>(a, p, st);
}

template <typename T>
int prefix_attn_type(const HpmnPrefixAttn &a, AttnPlan &p, hipStream_t st) {
    constexpr int E = 16 / sizeof(T);
    p.vec = a.D % E == 0;
    for (const void *q : {a.q, a.k_pre, a.v_pre, a.k_suf, a.v_suf}) p.vec = p.vec && is_aligned(q, 16);
    for (int64_t s : {a.q_sb, a.q_sl, a.q_sh, a.kp_st, a.kp_sh, a.vp_st, a.vp_sh, a.ks_sb, a.ks_st, a.ks_sh, a.vs_sb, a.vs_st, a.vs_sh})
        p.vec = p.vec && s % E == 0;
    for (int64_t s : {a.kp_st, a.vp_st, a.ks_st, a.vs_st}) p.vec = p.vec && s < (1l << 24);  // TileLoader: 128 rows in 32 bits of bytes
    p.out_vec = a.D % 4 == 0 && is_aligned(a.out, 4 * sizeof(T));
    for (int64_t s : {a.o_sb, a.o_sl, a.o_sh}) p.out_vec = p.out_vec && s % 4 == 0;
    return attn_width<T>(a, p, st);
}

}  // namespace hpmn
