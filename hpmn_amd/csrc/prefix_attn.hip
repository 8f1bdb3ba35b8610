// Attention of a batch that shares a long prefix (include/hpmn_hip.h, hpmn_prefix_attn): how a call is cut up, and the fp32
// instantiation of the kernel in prefix_attn.h.
#include "prefix_attn.h"

namespace hpmn {

extern template int prefix_attn_type<bf16_t>(const HpmnPrefixAttn &a, AttnPlan &p, hipStream_t st);
extern template int prefix_attn_type<f16_t>(const HpmnPrefixAttn &a, AttnPlan &p, hipStream_t st);

// By sizes and type alone.  Rows: 128 per workgroup from 65 on, 64 below (two waves share out the keys; four waves for up to 32 rows,
// 16-bit: 8 rows of 64 over 32768 keys 11.9 against 12.1 us, 4 x 32 heads over 8 of 128 29.1 against 29.7: not kept).
AttnPlan attn_plan(const HpmnPrefixAttn &a) {
    AttnPlan p = {};
    const int esize = (int)elem_size(a.dtype), group = a.Hq / a.Hkv;
    const long M = (long)a.B * a.Lq * group, per_seq = (long)a.Lq * group;
    p.rows = M * a.Hkv;
    p.d4 = (a.D + 3) / 4 * 4;
    p.mw_pre = M > 64 ? 4 : 2;
    p.mw_suf = per_seq > 64 ? 4 : 2;
    p.rt_suf = a.S > 0 ? (int)((per_seq + 32 * p.mw_suf - 1) / (32 * p.mw_suf)) : 0;
    // Few keys of very many sequences: the second kernel's, which asks for them beside the parts.  A workgroup for each costs its
    // start and its own part: 300 x 8 heads of 128 over 4096 keys + 1 45.6 -> 27.6 us, 1000 x 16 heads over 2 of 128, 2048 + 8
    // 75.0 -> 62.8, 64 x 8 heads of 128, 4096 + 1 22.6 -> 18.8; up to 512 of them run beside the prefix's (500 x 1 head of 64,
    // 1000 + 1 11.3 against 11.7, 8 x 8 heads over 1 of 64 12.1 against 12.7).
    long own = (long)a.B * a.Hkv * p.rt_suf;             // (sequence, key head, row tile)s with own keys
    if (a.S <= JOIN_KEYS && own >= 512) {
        p.keys = a.S;
        own = 0;
    }
    auto split = [&](long base, int keys, int tile, long beside, int &splits, int &per) {
        const int tiles = std::max(1, (keys + tile - 1) / tile);
        // Keys: one workgroup per CU, two when each still has 1280 keys (fp32: 320) to work through -- a tile's loads hide behind the
        // other's products, shorter ranges pay more for their start and for the join: 300 x 8 heads of 128, 16384 keys 54 -> 50 us with
        // two, 200 x 8 heads over 2 of 64, 4096 keys 17.5 -> 21.  At most 128 parts to join (fp32, whose ranges cost more: 256):
        // 8 x 8 heads over 1 of 64, 32768 keys 13.8 us against 15.3 with 256 and 15.8 with 64; fp32, 8 rows 20.9 against 16.5 with 256.
        splits = (int)std::max<long>(1, std::min<long>(tiles, 256 / base));
        // Many workgroups of own keys hide beside one of the prefix on a CU: two of the prefix only for so much longer ranges (512 x 16
        // heads over 4 of 128, + 64 own keys: 8192 keys 76.6 us with two, 65.1 with one; 32768 keys 172 against 189).
        if ((long)tiles * tile / splits * 512 >= (esize == 4 ? 320 : 1280) * std::max(512l, beside))
            splits = (int)std::max<long>(1, std::min<long>(tiles, 512 / base));
        splits = std::min(splits, esize == 4 ? 256 : 128);
        per = (tiles + splits - 1) / splits * tile;
        splits = std::max(1, (keys + per - 1) / per);
    };
    // a short prefix and nothing else: one range, no second kernel.  8 x 8 heads over 2 of 64, 512 keys bf16: 9.0 us of device time
    // against 9.1 cut up, and one launch less to wait for; 1024 keys 12.6 against 9.2; 200 x 8 heads over 2 of 64, 256 keys 11.4
    // against 11.0, over 8 of 128 17.5 against 13.5
    const bool whole = a.S == 0 && esize == 2 && (long)a.P * a.D <= (p.mw_pre == 4 ? 256 : 512) * 64;
    p.rt_pre = (int)((M + 32 * p.mw_pre - 1) / (32 * p.mw_pre));
    // (16-bit, many rows: pairs of tiles)
    split((long)p.rt_pre * a.Hkv, a.P, attn_tile(esize, p.mw_pre) * (esize == 2 && p.mw_pre == 4 ? 2 : 1), own, p.splits_pre,
          p.per_pre);
    if (whole) {
        p.splits_pre = 1;
        p.per_pre = std::max(a.P, 1);
    }
    p.blocks_pre = (unsigned)(((long)a.Hkv * p.splits_pre + 7) / 8 * 8 * p.rt_pre);
    if (own > 0) {
        split(own, a.S, attn_tile(esize, p.mw_suf), 0, p.splits_suf, p.per_suf);
        p.blocks_suf = (unsigned)(own * p.splits_suf);
    }
    p.parts = p.splits_pre + p.splits_suf;
    p.join = p.parts > 1 || p.keys > 0;
    p.o_at = ((long)p.parts * p.rows * 2 + 3) / 4 * 4;
    return p;
}

size_t prefix_attn_workspace_bytes(const HpmnPrefixAttn &a) {
    const AttnPlan p = attn_plan(a);
    return p.join ? ((size_t)p.o_at + (size_t)p.parts * p.rows * p.d4) * sizeof(float) : 0;
}

int prefix_attn_launch(const HpmnPrefixAttn &a, hipStream_t st) {
    AttnPlan p = attn_plan(a);
    // a launch has to stay below 2^32 threads
    if ((uint64_t)p.blocks_pre + p.blocks_suf >= (1u << 24) || (p.join && (p.rows + 3) / 4 >= (1l << 24))) return HPMN_EUNSUPPORTED;
    if (a.dtype == HPMN_F32) return prefix_attn_type<float>(a, p, st);
    return a.dtype == HPMN_BF16 ? prefix_attn_type<bf16_t>(a, p, st) : prefix_attn_type<f16_t>(a, p, st);
}

}  // namespace hpmn
