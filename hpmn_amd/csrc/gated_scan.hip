// Gated linear recurrence (include/hpmn_hip.h): h_t = a_t h_{t-1} + (1 - a_t) v_t with a = sigmoid(z), forward, backward and
// the one-event step.
//
// h -> a h + u v are affine maps, their composition is associative: (A2, B2) o (A1, B1) = (A2 A1, A2 B1 + B2).  A workgroup owns
// one sequence and a block of channels and walks the time axis in tiles of 128 steps held in registers:
//   lane = (4 channels) x (a run of 4 consecutive steps): composes its run, 16-byte accesses in fp32, 8-byte in bf16 / fp16;
//   the runs of a wave are scanned with lane shuffles, the waves of a tile through LDS (one barrier per tile, two buffers);
//   the carried state enters, the run is replayed from it and stored.
// z and v are read once, y is written once, nothing else reaches memory (training: one fp32 row per tile and channel).  Bound
// by memory: the next tile's rows are in flight while this one is composed.  Tiles of 128 steps because that is what one barrier
// pays for at 512 threads (8 waves x 4 runs of 4); runs of 4 because the forward's rows, gates and maps of a run then fit 128
// registers, two workgroups a CU; the backward has about 200 to 230 and one workgroup a CU.
// The backward walks the tiles in reverse.  Its scan G -> a (G + d_y) has the SAME a as the forward's, so one exchange serves
// both: the states are recomputed from the tile's saved first row instead of being stored (a read of z and v, which d_z and d_v
// need anyway, against a write and a read of all states in fp32).
#include <algorithm>

#include "seq_types.h"

namespace hpmn {

constexpr int TILE = HPMN_GATED_SCAN_TILE;
constexpr int RUN = 4;                       // steps per lane and tile
constexpr int MAX_WAVES = 8;                 // TILE = waves * (64 / LPR) * RUN

// barrier that orders LDS alone: __syncthreads() would also wait for the tile's stores to reach memory
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ v4f shfl_up4(v4f x, int d) {
    v4f r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __shfl_up(x[i], d);
    return r;
}
__device__ __forceinline__ v4f shfl_down4(v4f x, int d) {
    v4f r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __shfl_down(x[i], d);
    return r;
}
__device__ __forceinline__ v4f load_state(const float *p, int n) {          // n channels of a dense fp32 row
    v4f r = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < n) r[i] = p[i];
    return r;
}
__device__ __forceinline__ void store_state(float *p, v4f x, int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < n) p[i] = x[i];
}

// Which steps fire (t + 1 a multiple of the period) and the row they fire into, kept without a division per step: q = t / period,
// r = t % period of the step at hand.
struct Firing {
    int q, r;
    __device__ __forceinline__ bool next(int period) {                      // does this step fire?  then on to the next
        const bool fire = r == period - 1;
        q += fire ? 1 : 0;
        r = fire ? 0 : r + 1;
        return fire;
    }
    __device__ __forceinline__ void jump(int dq, int dr, int period) {      // by dq * period + dr steps, |dr| < period
        q += dq;
        r += dr;
        if (r >= period) { r -= period; ++q; }
        if (r < 0) { r += period; --q; }
    }
};

// The decay of many steps.  A gate held at z remembers e^z steps, and what counts then is 1 - a, of which a product of a's rounded
// to fp32 near 1 keeps few digits: at z = 10 the state would settle 10^-3 off, the same way at every step.  So the complement U of
// a product A is carried along, U2 + A2 U1 for two maps, and A is taken from it where it is above one half: rounded once for all the steps.
// States of order one behind 8192 steps with z = 8 / 10 / 12 are off by 7e-6 / 1.4e-5 / 1.5e-5 (products of a: 2.5e-4 / 4.5e-4 /
// 4.7e-4), for 0 to 3 % of a memory-bound pass's time and 1 us of a latency-bound pair.
__device__ __forceinline__ v4f decay(v4f A, v4f U) {
    v4f r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = U[i] < 0.5f ? 1.0f - U[i] : A[i];
    return r;
}

// Row `row` of a [T, ...] operand: row strides fit 32 bits (checked by the entry point), so the offset is ONE 32 x 32 -> 64 bit
// multiply-add; a 64-bit stride takes three, at a quarter of the rate.
template <typename T>
__device__ __forceinline__ T *at_row(T *p, unsigned row, int64_t stride) {
    return p + (uint64_t)row * (uint32_t)stride;
}

// A lane's share of the work: its channels [c, c + n) (n = 0: none, it repeats another lane's loads and stores nothing), and the
// steps [lo, hi) that count.  Where C is no multiple of four the last quad ends at C and computes some of the channels of the one in front
// of it again, to the same values: whole quads at any alignment beat scalar accesses (500 x 1024 x 63 fp32 forward + backward 184 us
// against 305 when it was measured; now 80 / 133 against 80 / 137 for 64 channels.  A bf16 row of 1023 straddles cache lines: 16 x 4096 x
// 1023 125 / 213 against 85 / 150 for 1024).  Loads always go to a row in [lo, hi) (to one valid row if there is none), so that none is
// conditional.
struct Share {
    int c, n, nl, lo, hi;
    __device__ __forceinline__ Share(int C, int T, int first, int begin) {
        nl = min(4, C);
        n = first < C ? nl : 0;
        c = max(0, min(first, C - 4));
        lo = max(0, begin);
        hi = T;
    }
    __device__ __forceinline__ unsigned row(int t) const { return (unsigned)min(max(t, min(lo, hi - 1)), hi - 1); }
    __device__ __forceinline__ bool live(int t) const { return t >= lo && t < hi; }
};

// a, u and v of a run.  Steps that do not count are the identity (a = 1, u = 0, v = 0) whatever was loaded for them.
template <typename T>
__device__ __forceinline__ void gate_run(const Share &sh, bool whole, int t, const quad_t<T> (&zr)[RUN], const quad_t<T> (&vr)[RUN],
                                         v4f (&ag)[RUN], v4f (&ug)[RUN], v4f (&vv)[RUN]) {
#pragma unroll
    for (int s = 0; s < RUN; ++s) {
        ag[s] = __builtin_convertvector(zr[s], v4f);
        vv[s] = __builtin_convertvector(vr[s], v4f);
    }
    if (!whole) {
#pragma unroll
        for (int s = 0; s < RUN; ++s) {
            const bool live = sh.live(t + s);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                ag[s][i] = live ? ag[s][i] : 1e30f;          // sigmoid: exactly 1, and its complement 0
                vv[s][i] = live ? vv[s][i] : 0.f;
            }
        }
    }
#pragma unroll
    for (int s = 0; s < RUN; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float x, y;
            gate_pair(ag[s][i], x, y);
            ag[s][i] = x;
            ug[s][i] = y;
        }
}

// Few sequences, long ones: the time axis is cut into chunks of whole tiles and a first launch composes every chunk to one map
// (A, B) per channel; the main launch then starts each chunk from the maps in front of it (behind it, in the backward).  z and v
// are read a second time, mostly from the caches; no workgroup waits for another.
struct ChunkArgs {
    int T, C, period;
    const void *z, *x;                       // x: v, or d_y in the backward
    int64_t z_sb, z_st, x_sb, x_st;
    const int32_t *begin;
    float *ws;                               // [B][chunks][2][C]
    int chunks, tiles;                       // per sequence, per chunk
};

// Bound by memory latency more than rate (a lane group walks its span alone, loads four steps ahead): 1 x 65536 x 256 bf16 14.3 us
// for 67 MB, 4.7 TB/s; behind it the main kernel finds z and v in the cache, 26.9 us.
template <typename T, int LPR, bool VEC, bool BWD>
__global__ __launch_bounds__(512) void gated_scan_chunk_kernel(const ChunkArgs a) {
    constexpr int TG = 64 / LPR;
    __shared__ v4f agg[MAX_WAVES][2][LPR];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6;
    const int cg = lane % LPR, tg = lane / LPR;
    const int ncb = (a.C + 4 * LPR - 1) / (4 * LPR);
    const int chunk = blockIdx.x % a.chunks, rest = blockIdx.x / a.chunks;
    const long b = rest / ncb;
    if (chunk == (BWD ? 0 : a.chunks - 1)) return;           // nobody starts behind the last (in front of the first) one
    const Share sh(a.C, a.T, ((rest % ncb) * LPR + cg) * 4, a.begin ? a.begin[b] : 0);
    const T *z = (const T *)a.z + b * a.z_sb + sh.c;
    const bool has_x = a.x != nullptr;
    const T *x = has_x ? (const T *)a.x + b * a.x_sb + sh.c : z;
    const long x_st = has_x ? a.x_st : a.z_st;
    const int x_rows = BWD ? a.T / a.period : a.T;
    // a lane group owns a span of a.tiles * RUN consecutive steps here, so that its map is composed without an exchange
    const int span = a.tiles * RUN, t_first = chunk * a.tiles * TILE + (w * TG + tg) * span;
    const v4f one = {1.f, 1.f, 1.f, 1.f}, zero = {0.f, 0.f, 0.f, 0.f};
    v4f A = one, U = zero, Bc = zero;        // of the span so far
    v4f As = one, Us = zero, Bs = zero;      // of its latest SECTION steps: an a rounded near 1 does its damage there only
    constexpr int SECTION = 32;
    quad_t<T> zr[RUN], xr[RUN];
    auto load = [&](int j) {
        const int t = t_first + (BWD ? span - RUN - j : j);
        Firing g = {t / a.period, t % a.period};
#pragma unroll
        for (int s = 0; s < RUN; ++s) {
            zr[s] = load_quad<T, VEC>(at_row(z, sh.row(t + s), a.z_st), sh.nl);
            const unsigned row = BWD ? (unsigned)max(0, min(g.q, x_rows - 1)) : sh.row(t + s);
            xr[s] = load_quad<T, VEC>(at_row(x, row, x_st), sh.nl);
            g.next(a.period);
        }
    };
    load(0);
    for (int j = 0; j < span; j += RUN) {
        const int t = t_first + (BWD ? span - RUN - j : j);
        v4f ag[RUN], ug[RUN], vv[RUN];
        gate_run<T>(sh, false, t, zr, xr, ag, ug, vv);
        if (BWD) {
            Firing g = {t / a.period, t % a.period};
#pragma unroll
            for (int s = 0; s < RUN; ++s) {
                const bool fire = g.next(a.period) && has_x && t + s < sh.hi;
#pragma unroll
                for (int i = 0; i < 4; ++i) vv[s][i] = fire ? (float)xr[s][i] : 0.f;
            }
        }
        load(min(j + RUN, span - RUN));
#pragma unroll
        for (int i = 0; i < RUN; ++i) {
            const int s = BWD ? RUN - 1 - i : i;
            Bs = BWD ? ag[s] * (Bs + vv[s]) : ag[s] * Bs + ug[s] * vv[s];
            Us = ag[s] * Us + ug[s];
            As *= ag[s];
        }
        if ((j + RUN) % SECTION == 0 || j + RUN == span) {
            const v4f D = decay(As, Us);
            Bc = D * Bc + Bs;
            U = D * U + Us;
            A *= D;
            As = one;
            Us = Bs = zero;
        }
    }
#pragma unroll
    for (int d = 1; d < TG; d *= 2) {                        // neighbours in pairs: the earlier map first (the later, in the backward)
        const v4f Ao = BWD ? shfl_down4(A, d * LPR) : shfl_up4(A, d * LPR), Bo = BWD ? shfl_down4(Bc, d * LPR) : shfl_up4(Bc, d * LPR);
        const v4f Uo = BWD ? shfl_down4(U, d * LPR) : shfl_up4(U, d * LPR);
        if (BWD ? tg + d < TG : tg >= d) {
            Bc = A * Bo + Bc;
            U = A * Uo + U;
            A *= Ao;
        }
    }
    if (tg == (BWD ? 0 : TG - 1)) {
        agg[w][0][cg] = decay(A, U);
        agg[w][1][cg] = Bc;
    }
    __syncthreads();
    if (threadIdx.x >= LPR) return;
    A = one;
    Bc = zero;
    for (int i = 0; i < nw; ++i) {
        const int j = BWD ? nw - 1 - i : i;
        Bc = agg[j][0][cg] * Bc + agg[j][1][cg];
        A *= agg[j][0][cg];
    }
    float *out = a.ws + (b * a.chunks + chunk) * 2 * a.C + sh.c;
    store_state(out, A, sh.n);
    store_state(out + a.C, Bc, sh.n);
}

// The state behind chunks first, first + dir, ... (count <= TILE of them) when it is `start` in front: the chunk maps go through the
// same lanes / shuffles / LDS composition as the steps of a tile.
template <int LPR>
__device__ __forceinline__ v4f fold_chunks(const float *ws, int C, int c, int nl, int first, int dir, int count, v4f start,
                                           v4f (&buf)[MAX_WAVES][2][LPR]) {
    constexpr int TG = 64 / LPR;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6, cg = lane % LPR, tg = lane / LPR;
    v4f A = {1.f, 1.f, 1.f, 1.f}, Bc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < RUN; ++s) {
        const int p = (w * TG + tg) * RUN + s;
        if (p >= count) continue;
        const float *m = ws + (long)(first + dir * p) * 2 * C + c;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = m[min(i, nl - 1)];
            Bc[i] = x * Bc[i] + m[C + min(i, nl - 1)];
            A[i] *= x;
        }
    }
#pragma unroll
    for (int d = 1; d < TG; d *= 2) {
        const v4f Ap = shfl_up4(A, d * LPR), Bp = shfl_up4(Bc, d * LPR);
        if (tg >= d) {
            Bc = A * Bp + Bc;
            A *= Ap;
        }
    }
    if (tg == TG - 1) {
        buf[w][0][cg] = A;
        buf[w][1][cg] = Bc;
    }
    lds_barrier();
    for (int i = 0; i < nw; ++i) start = buf[i][0][cg] * start + buf[i][1][cg];
    return start;
}

// Memory-bound: 500 x 1024 x 64 fp32, period 2, 328 MB in 72.2 us, 4.5 TB/s, the waves waiting 41 % of their cycles (a copy reaches
// 4.7, the backward below 5.5: not the memory's limit, but what loads one tile ahead ask of it).  16 x 4096 x 1024 bf16, 403 MB in
// 84.8 us, 4.8 TB/s.  Small calls are a launch and one round trip to memory: 128 x 100 x 32 fp32 5.1 us.
template <typename T, int LPR, bool VEC>
__global__ __launch_bounds__(512) void gated_scan_fwd_kernel(const HpmnGatedScan a, int chunks, int chunk_tiles) {
    constexpr int TG = 64 / LPR;             // runs side by side in a wave
    __shared__ v4f agg[2][MAX_WAVES][2][LPR], maps[MAX_WAVES][2][LPR];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6;
    const int cg = lane % LPR, tg = lane / LPR;
    const int ncb = (a.C + 4 * LPR - 1) / (4 * LPR);
    const int chunk = blockIdx.x % chunks, rest = blockIdx.x / chunks;
    const long b = rest / ncb;
    const Share sh(a.C, a.T, ((rest % ncb) * LPR + cg) * 4, a.begin ? a.begin[b] : 0);
    const int step = nw * TG * RUN;          // steps per tile (TILE, or fewer when the whole sequence fits)
    const int k_first = chunk * chunk_tiles, t_end = min(a.T, (k_first + chunk_tiles) * step);
    const int tiles = (a.T + TILE - 1) / TILE, period = a.period;
    const T *z = (const T *)a.z + b * a.z_sb + sh.c, *v = (const T *)a.v + b * a.v_sb + sh.c;
    T *y = (T *)a.y + b * a.y_sb + sh.c;

    v4f carry = {0.f, 0.f, 0.f, 0.f};
    if (a.h0) carry = load_state(a.h0 + b * a.h0_sb + sh.c, sh.n);
    int t = k_first * step + (w * TG + tg) * RUN;
    Firing f = {t / period, t % period};
    const int dq = step / period, dr = step % period;
    quad_t<T> zr[RUN], vr[RUN];
    auto load = [&](int at) {
#pragma unroll
        for (int s = 0; s < RUN; ++s) {
            zr[s] = load_quad<T, VEC>(at_row(z, sh.row(at + s), a.z_st), sh.nl);
            vr[s] = load_quad<T, VEC>(at_row(v, sh.row(at + s), a.v_st), sh.nl);
        }
    };
    load(t);
    if (chunk > 0)
        carry = fold_chunks<LPR>((const float *)a.workspace + b * chunks * 2 * a.C, a.C, sh.c, sh.nl, 0, 1, chunk, carry, maps);
    for (int k = k_first, t0 = k_first * step; t0 < t_end; ++k, t0 += step) {
        v4f ag[RUN], bv[RUN], vv[RUN];
        gate_run<T>(sh, t0 >= sh.lo && t0 + step <= sh.hi, t, zr, vr, ag, bv, vv);
        v4f A = ag[0], U = bv[0];
#pragma unroll
        for (int s = 1; s < RUN; ++s) {
            U = ag[s] * U + bv[s];
            A *= ag[s];
        }
#pragma unroll
        for (int s = 0; s < RUN; ++s) bv[s] *= vv[s];
        load(t + step);
        v4f Bc = bv[0];
#pragma unroll
        for (int s = 1; s < RUN; ++s) Bc = ag[s] * Bc + bv[s];
#pragma unroll
        for (int d = 1; d < TG; d *= 2) {
            const v4f Ap = shfl_up4(A, d * LPR), Bp = shfl_up4(Bc, d * LPR), Up = shfl_up4(U, d * LPR);
            if (tg >= d) {
                Bc = A * Bp + Bc;
                U = A * Up + U;
                A *= Ap;
            }
        }
        v4f (&buf)[MAX_WAVES][2][LPR] = agg[k & 1];
        if (tg == TG - 1) {
            buf[w][0][cg] = decay(A, U);
            buf[w][1][cg] = Bc;
        }
        const v4f Ae = shfl_up4(A, LPR), Be = shfl_up4(Bc, LPR);
        lds_barrier();
        if (a.saved && threadIdx.x < LPR) store_state(a.saved + (b * tiles + k) * a.C + sh.c, carry, sh.n);
        v4f h = carry;
        for (int i = 0; i < nw; ++i) {
            if (i == w) h = carry;
            carry = buf[i][0][cg] * carry + buf[i][1][cg];
        }
        if (tg > 0) h = Ae * h + Be;
        Firing g = f;
#pragma unroll
        for (int s = 0; s < RUN; ++s) {
            h = ag[s] * h + bv[s];
            const unsigned row = (unsigned)g.q;
            if (g.next(period) && a.y && sh.n > 0 && t + s < sh.hi) store_quad<T, VEC>(at_row(y, row, a.y_st), h, sh.n);
        }
        t += step;
        f.jump(dq, dr, period);
    }
    if (a.h_last && chunk == chunks - 1 && threadIdx.x < LPR) store_state(a.h_last + b * a.C + sh.c, carry, sh.n);
}

// Memory-bound: 500 x 1024 x 64 fp32, period 2, 590 MB in 106.8 us, 5.5 TB/s, behind its forward, which leaves some of z and v in the cache
// (by itself, on inputs that are in no cache, 124 us); 16 x 4096 x 1024 bf16, 671 MB in 149.8 us, 4.5 TB/s (256 workgroups there, one
// a CU, whose waves wait for memory half of their cycles); 128 x 100 x 32 fp32 7.0 us.
template <typename T, int LPR, bool VEC>
__global__ __launch_bounds__(512) void gated_scan_bwd_kernel(const HpmnGatedScanBwd a, int chunks, int chunk_tiles) {
    constexpr int TG = 64 / LPR;
    __shared__ v4f agg[2][MAX_WAVES][3][LPR], maps[MAX_WAVES][2][LPR];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6;
    const int cg = lane % LPR, tg = lane / LPR;
    const int ncb = (a.C + 4 * LPR - 1) / (4 * LPR);
    const int chunk = blockIdx.x % chunks, rest = blockIdx.x / chunks;
    const long b = rest / ncb;
    const Share sh(a.C, a.T, ((rest % ncb) * LPR + cg) * 4, a.begin ? a.begin[b] : 0);
    const int step = nw * TG * RUN;
    const int tiles = (a.T + TILE - 1) / TILE, period = a.period;
    const T *z = (const T *)a.z + b * a.z_sb + sh.c, *v = (const T *)a.v + b * a.v_sb + sh.c;
    // (without d_y its loads go to z, which has at least as many rows, and are not used)
    const bool has_dy = a.d_y != nullptr;
    const T *dy = has_dy ? (const T *)a.d_y + b * a.dy_sb + sh.c : z;
    const long dy_st = has_dy ? a.dy_st : a.z_st;
    const int dy_rows = a.T / period;
    T *dz = (T *)a.d_z + b * a.dz_sb + sh.c, *dv = (T *)a.d_v + b * a.dv_sb + sh.c;

    v4f R = {0.f, 0.f, 0.f, 0.f};            // dL/dh behind the tile
    if (a.d_h_last) R = load_state(a.d_h_last + b * a.C + sh.c, sh.n);
    const int k_first = chunk * chunk_tiles, k_last = min((a.T - 1) / step, k_first + chunk_tiles - 1);
    int t = k_last * step + (w * TG + tg) * RUN;
    Firing f = {t / period, t % period};
    const int dq = step / period, dr = step % period;
    quad_t<T> zr[RUN], vr[RUN], yr[RUN];
    v4f hs;
    auto load = [&](int at, int k, Firing g) {
#pragma unroll
        for (int s = 0; s < RUN; ++s) {
            zr[s] = load_quad<T, VEC>(at_row(z, sh.row(at + s), a.z_st), sh.nl);
            vr[s] = load_quad<T, VEC>(at_row(v, sh.row(at + s), a.v_st), sh.nl);
            yr[s] = load_quad<T, VEC>(at_row(dy, (unsigned)max(0, min(g.q, dy_rows - 1)), dy_st), sh.nl);
            g.next(period);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) hs[i] = a.saved[(b * tiles + max(k, 0)) * a.C + sh.c + min(i, sh.nl - 1)];
    };
    load(t, k_last, f);
    if (chunk < chunks - 1)
        R = fold_chunks<LPR>((const float *)a.workspace + b * chunks * 2 * a.C, a.C, sh.c, sh.nl, chunks - 1, -1, chunks - 1 - chunk, R,
                             maps);
    for (int k = k_last; k >= k_first; --k) {
        const int t0 = k * step;
        v4f ag[RUN], ug[RUN], vv[RUN], dd[RUN];
        const bool whole = t0 >= sh.lo && t0 + step <= sh.hi;
        gate_run<T>(sh, whole, t, zr, vr, ag, ug, vv);
#pragma unroll
        for (int s = 0; s < RUN; ++s) dd[s] = __builtin_convertvector(yr[s], v4f);
        if (!(has_dy && period == 1 && t0 + step <= sh.hi)) {
            Firing g = f;
#pragma unroll
            for (int s = 0; s < RUN; ++s) {
                const bool fire = g.next(period) && has_dy && t + s < sh.hi;
#pragma unroll
                for (int i = 0; i < 4; ++i) dd[s][i] = fire ? dd[s][i] : 0.f;
            }
        }
        const v4f h_tile = hs;
        f.jump(-dq, -dr, period);
        load(t - step, k - 1, f);
        v4f A = ag[0], U = ug[0], Bf = ug[0] * vv[0], Br = ag[RUN - 1] * dd[RUN - 1];
#pragma unroll
        for (int s = 1; s < RUN; ++s) {
            A *= ag[s];
            U = ag[s] * U + ug[s];
            Bf = ag[s] * Bf + ug[s] * vv[s];
            Br = ag[RUN - 1 - s] * (Br + dd[RUN - 1 - s]);
        }
        v4f Af = A, Ar = A;                  // scanned from the front, from the back
#pragma unroll
        for (int d = 1; d < TG; d *= 2) {
            const v4f Ap = shfl_up4(Af, d * LPR), Bp = shfl_up4(Bf, d * LPR), Up = shfl_up4(U, d * LPR);
            const v4f An = shfl_down4(Ar, d * LPR), Bn = shfl_down4(Br, d * LPR);
            if (tg >= d) {
                Bf = Af * Bp + Bf;
                U = Af * Up + U;
                Af *= Ap;
            }
            if (tg + d < TG) {
                Br = Ar * Bn + Br;
                Ar *= An;
            }
        }
        v4f (&buf)[MAX_WAVES][3][LPR] = agg[k & 1];
        if (tg == TG - 1) {
            buf[w][0][cg] = decay(Af, U);
            buf[w][1][cg] = Bf;
        }
        if (tg == 0) buf[w][2][cg] = Br;
        const v4f Ae = shfl_up4(Af, LPR), Be = shfl_up4(Bf, LPR);
        const v4f Ax = shfl_down4(Ar, LPR), Bx = shfl_down4(Br, LPR);
        lds_barrier();
        // (four waves' maps in flight: unrolled further, as the compiler does by itself, they alone take 64 registers, and the
        // fp32 form spills in this loop: 16 x 4096 x 1024 bf16 161 us against 150, 128 x 100 x 32 fp32 7.5 against 6.8)
        v4f h = h_tile, G = R;
#pragma unroll 4
        for (int i = 0; i < w; ++i) h = buf[i][0][cg] * h + buf[i][1][cg];
#pragma unroll 4
        for (int i = nw - 1; i >= 0; --i) {
            if (i == w) G = R;
            R = buf[i][0][cg] * R + buf[i][2][cg];
        }
        if (tg > 0) h = Ae * h + Be;
        if (tg < TG - 1) G = Ax * G + Bx;
#pragma unroll
        for (int s = 0; s < RUN; ++s) {                      // h_{t-1} - v in v's place
            const v4f x = vv[s];
            vv[s] = h - x;
            h = ag[s] * h + ug[s] * x;
        }
#pragma unroll
        for (int s = RUN - 1; s >= 0; --s) {
            G += dd[s];
            v4f gv = ug[s] * G;
            if (!whole) {                                    // steps that do not count: zeros, also where G or h is no number
                const bool live = sh.live(t + s);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    gv[i] = live ? gv[i] : 0.f;
                    vv[s][i] = live ? vv[s][i] : 0.f;
                }
            }
            if (sh.n > 0 && t + s < sh.hi) {
                store_quad<T, VEC>(at_row(dv, (unsigned)(t + s), a.dv_st), gv, sh.n);
                store_quad<T, VEC>(at_row(dz, (unsigned)(t + s), a.dz_st), gv * ag[s] * vv[s], sh.n);
            }
            G = ag[s] * G;
        }
        t -= step;
    }
    if (a.d_h0 && chunk == 0 && threadIdx.x < LPR) store_state(a.d_h0 + b * a.C + sh.c, R, sh.n);
}

__device__ __forceinline__ long step_user(const HpmnGatedStep &a, int b) {
    if (!a.user) return b;
    return (a.flags & HPMN_STEP_USER_I64) ? (long)((const int64_t *)a.user)[b] : (long)((const int32_t *)a.user)[b];
}

// Row j's event on user u's state by one wave; a lane's channels are its own, so the next event of the user sees what this one left.
// Scalar accesses: two dependent round trips (index, then state) are the time, whatever their width.
template <typename T>
__device__ __forceinline__ void step_event(const HpmnGatedStep &a, int lane, int j, long u) {
    for (int c = lane; c < a.C; c += 64) {
        float ag, ug;
        gate_pair((float)((const T *)a.z)[j * a.z_s + c], ag, ug);
        const float old = a.state[u * a.state_s + c], v = (float)((const T *)a.v)[j * a.v_s + c], d = v - old;
        // a state that moves little moves by u (v - h): a rounded near 1 would pull it the same way at every event
        const float h = ug < 0.5f && fabsf(d) < INFINITY ? fmaf(ug, d, old) : fmaf(ag, old, ug * v);
        if (a.y) ((T *)a.y)[j * a.y_s + c] = (T)h;
        if (a.flags & HPMN_STEP_COMMIT) a.state[u * a.state_s + c] = h;
    }
}
template <typename T>
__device__ __forceinline__ void step_unknown(const HpmnGatedStep &a, int lane, int j) {
    if (a.y)
        for (int c = lane; c < a.C; c += 64) ((T *)a.y)[j * a.y_s + c] = (T)__builtin_nanf("");
}

// Rows that do not wait for each other: a wave each.  Bound by its launch and the round trips: one row of 64 fp32 1.4 us, 4096 rows of
// 128 bf16 3.4 us of device time, against the 8 us that the host takes for the call.
template <typename T>
__global__ __launch_bounds__(64) void gated_step_kernel(const HpmnGatedStep a) {
    const int b = blockIdx.x, lane = threadIdx.x;
    const long u = step_user(a, b);
    if (u < 0 || u >= a.n_users) step_unknown<T>(a, lane, b);
    else step_event<T>(a, lane, b, u);
}

// HPMN_STEP_COMMIT with a user list: the FIRST row that names a user carries out all rows of that user, in row order; the others find
// an earlier row with their user and leave.  A wave per row; eight of them read the list together, a part at a time through LDS, and
// compare 512 users before they look at the outcome, which is nothing most of the time.  4096 rows of 128 bf16 8.8 us (a branch
// for every 64 users: 22.5; every wave reading by itself: 18.5; a row at a time: 880).
template <typename T, typename U>
__global__ __launch_bounds__(512) void gated_step_ordered_kernel(const HpmnGatedStep a) {
    constexpr int PART = 2048, LOOK = 8;
    __shared__ U named[PART];
    const int lane = threadIdx.x & 63, b = blockIdx.x * 8 + (threadIdx.x >> 6);
    const U *users = (const U *)a.user, u = users[min(b, a.B - 1)];
    bool done = b >= a.B || u < 0 || (long)u >= a.n_users;
    if (b < a.B && done) step_unknown<T>(a, lane, b);
    for (int j0 = 0; j0 < a.B; j0 += PART) {
        if (j0 > 0) __syncthreads();
        for (int i = threadIdx.x; i < PART; i += 512) named[i] = j0 + i < a.B ? users[j0 + i] : (U)-1;      // (-1: no row's user)
        __syncthreads();
        if (done) continue;
        for (int i = 0; i < min(PART, a.B - j0) && !done; i += 64 * LOOK) {
            uint64_t same[LOOK], any = 0;
#pragma unroll
            for (int k = 0; k < LOOK; ++k) {
                same[k] = __ballot(named[i + 64 * k + lane] == u);
                any |= same[k];
            }
            if (any == 0) continue;
#pragma unroll
            for (int k = 0; k < LOOK; ++k) {
                const int before = b - (j0 + i + 64 * k);    // rows of these in front of this wave's
                if (before > 0 && (before >= 64 ? same[k] : same[k] & ((1ull << before) - 1))) done = true;
                if (!done)
                    for (uint64_t s = same[k]; s; s &= s - 1) step_event<T>(a, lane, j0 + i + 64 * k + __builtin_ctzll(s), (long)u);
            }
        }
    }
}

// Channels per workgroup: 64 (16 lanes per step); narrower layers take 32 or 16 channels and put more steps side by side.
inline int scan_lanes(int C) { return C > 32 ? 16 : C > 16 ? 8 : 4; }
// Waves: a tile of 128 steps, or as many as the whole sequence needs.
inline int scan_waves(int T, int lpr) {
    const int per_wave = 64 / lpr * RUN;
    return std::min(TILE / per_wave, (T + per_wave - 1) / per_wave);
}

struct Cut {
    int chunks, tiles;                       // per sequence, per chunk
};
// Time chunks where whole sequences leave two thirds of the CUs idle and there are at least four tiles to share out: as many as
// fill the CUs once (twice costs more than it hides: the backward has the registers, 202 to 231, for one workgroup per CU), at most
// TILE of them (fold_chunks).  Forward / backward us, cut against whole, fp32, C = 64, device time:
//   8 x 1024: 12 / 15 against 20 / 29;   64 x 4096: 58 / 87 against 79 / 133;   1 x 16384: 15 / 19 against 268 / 406;
//   at the rule's borders: 64 x 512 14.3 / 18.1 against 12.5 / 18.3, 80 x 1024 20 / 30 against 21 / 35;
//   beyond them: 96 x 1024 (two chunks) 28 / 37 against 21 / 38, 8 x 256 (two tiles) 10 / 13 against 7 / 10.
// Up to 32 (16) channels a workgroup has half (a quarter) of the waves, so the CUs are full with twice (four times) as many: 49 x 7701 x
// 10 bf16 20 / 28 against 35 / 48 with 256, 64 x 4096 x 16 fp32 20 / 27 against 27 / 32 when that was measured (24 / 32, 20 / 28 now).
static Cut scan_cut(int B, int T, int C) {
    const int lpr = scan_lanes(C), tiles = (T + TILE - 1) / TILE;
    const long whole = (long)B * ((C + 4 * lpr - 1) / (4 * lpr));
    if (256 / whole < 3 || tiles < 4) return {1, tiles};
    const int want = (int)std::min<long>(std::min(tiles, TILE), 256 * 16 / lpr / whole);
    const int per = (tiles + want - 1) / want;
    return {(tiles + per - 1) / per, per};
}

// A launch has to stay below 2^32 threads, steps and a tile more in 31 bits.
bool gated_scan_fits(int B, int T, int C) {
    if (T > (1 << 30) || C > (1 << 30)) return false;
    const int lpr = scan_lanes(C);
    const Cut cut = scan_cut(B, T, C);
    return (double)B * ((C + 4l * lpr - 1) / (4 * lpr)) * cut.chunks * 64 * scan_waves(T, lpr) < 4294967296.0;
}

size_t gated_scan_workspace_bytes(int B, int T, int C) {
    const Cut cut = scan_cut(B, T, C);
    return cut.chunks > 1 ? (size_t)B * cut.chunks * 2 * C * sizeof(float) : 0;
}

template <typename T, int LPR>
static void scan_fwd_go(const HpmnGatedScan &a, hipStream_t st) {
    const Cut cut = scan_cut(a.B, a.T, a.C);
    const dim3 grid((unsigned)((long)a.B * ((a.C + 4 * LPR - 1) / (4 * LPR)) * cut.chunks)), block(64 * scan_waves(a.T, LPR));
    const bool vec = a.C >= 4;
    if (cut.chunks > 1) {
        const ChunkArgs c = {a.T, a.C, 1, a.z, a.v, a.z_sb, a.z_st, a.v_sb, a.v_st, a.begin, (float *)a.workspace, cut.chunks, cut.tiles};
        if (vec) hipLaunchKernelGGL((gated_scan_chunk_kernel<T, LPR, true, false>), grid, block, 0, st, c);
        else hipLaunchKernelGGL((gated_scan_chunk_kernel<T, LPR, false, false>), grid, block, 0, st, c);
    }
    if (vec) hipLaunchKernelGGL((gated_scan_fwd_kernel<T, LPR, true>), grid, block, 0, st, a, cut.chunks, cut.tiles);
    else hipLaunchKernelGGL((gated_scan_fwd_kernel<T, LPR, false>), grid, block, 0, st, a, cut.chunks, cut.tiles);
}

template <typename T, int LPR>
static void scan_bwd_go(const HpmnGatedScanBwd &a, hipStream_t st) {
    const Cut cut = scan_cut(a.B, a.T, a.C);
    const dim3 grid((unsigned)((long)a.B * ((a.C + 4 * LPR - 1) / (4 * LPR)) * cut.chunks)), block(64 * scan_waves(a.T, LPR));
    const bool vec = a.C >= 4;
    if (cut.chunks > 1) {
        const ChunkArgs c = {a.T, a.C, a.period, a.z, a.d_y, a.z_sb, a.z_st, a.dy_sb, a.dy_st, a.begin, (float *)a.workspace, cut.chunks, cut.tiles};
        if (vec) hipLaunchKernelGGL((gated_scan_chunk_kernel<T, LPR, true, true>), grid, block, 0, st, c);
        else hipLaunchKernelGGL((gated_scan_chunk_kernel<T, LPR, false, true>), grid, block, 0, st, c);
    }
    if (vec) hipLaunchKernelGGL((gated_scan_bwd_kernel<T, LPR, true>), grid, block, 0, st, a, cut.chunks, cut.tiles);
    else hipLaunchKernelGGL((gated_scan_bwd_kernel<T, LPR, false>), grid, block, 0, st, a, cut.chunks, cut.tiles);
}

template <typename T>
static void scan_fwd_type(const HpmnGatedScan &a, hipStream_t st) {
    const int lpr = scan_lanes(a.C);
    if (lpr == 16) scan_fwd_go<T, 16>(a, st);
    else if (lpr == 8) scan_fwd_go<T, 8>(a, st);
    else scan_fwd_go<T, 4>(a, st);
}
template <typename T>
static void scan_bwd_type(const HpmnGatedScanBwd &a, hipStream_t st) {
    const int lpr = scan_lanes(a.C);
    if (lpr == 16) scan_bwd_go<T, 16>(a, st);
    else if (lpr == 8) scan_bwd_go<T, 8>(a, st);
    else scan_bwd_go<T, 4>(a, st);
}

int gated_scan_fwd_launch(const HpmnGatedScan &a, hipStream_t st) {
    if (a.dtype == HPMN_F32) scan_fwd_type<float>(a, st);
    else if (a.dtype == HPMN_BF16) scan_fwd_type<bf16_t>(a, st);
    else scan_fwd_type<f16_t>(a, st);
    return check_launch();
}

int gated_scan_bwd_launch(const HpmnGatedScanBwd &a, hipStream_t st) {
    if (a.dtype == HPMN_F32) scan_bwd_type<float>(a, st);
    else if (a.dtype == HPMN_BF16) scan_bwd_type<bf16_t>(a, st);
    else scan_bwd_type<f16_t>(a, st);
    return check_launch();
}

template <typename T>
static void step_type(const HpmnGatedStep &a, hipStream_t st) {
    const dim3 eighths((unsigned)((a.B + 7) / 8));
    const bool ordered = (a.flags & HPMN_STEP_COMMIT) && a.user;
    if (ordered && (a.flags & HPMN_STEP_USER_I64)) hipLaunchKernelGGL((gated_step_ordered_kernel<T, int64_t>), eighths, dim3(512), 0, st, a);
    else if (ordered) hipLaunchKernelGGL((gated_step_ordered_kernel<T, int32_t>), eighths, dim3(512), 0, st, a);
    else hipLaunchKernelGGL(gated_step_kernel<T>, dim3((unsigned)a.B), dim3(64), 0, st, a);
}

int gated_step_launch(const HpmnGatedStep &a, hipStream_t st) {
    if (a.dtype == HPMN_F32) step_type<float>(a, st);
    else if (a.dtype == HPMN_BF16) step_type<bf16_t>(a, st);
    else step_type<f16_t>(a, st);
    return check_launch();
}

}  // namespace hpmn
