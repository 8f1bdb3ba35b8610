"""Attention of a batch that shares a long prefix (hpmn_prefix_attn): C ABI refusals on the CPU, results against a float64
restatement on the GPU."""
import ctypes as C
import math
import os
import subprocess

import pytest
import torch

from hpmn_amd import _lib, build, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def lib():
    build.build_library()
    return _lib.load()


def _args():
    a = _lib.HpmnPrefixAttn()
    a.B, a.Lq, a.Hq, a.Hkv, a.D, a.dtype, a.P, a.S, a.scale = 2, 1, 4, 2, 64, _lib.HPMN_BF16, 100, 8, 0.125
    a.q = a.k_pre = a.v_pre = a.k_suf = a.v_suf = a.out = 4096
    a.workspace, a.workspace_bytes = 4096, 1 << 40
    return a


@pytest.mark.parametrize("field,value,rc", [("B", -1, -1), ("Lq", -1, -1), ("Hq", 0, -1), ("Hkv", 0, -1), ("Hq", 5, -1), ("D", 0, -1),
                                            ("D", 129, -2), ("P", -1, -1), ("S", -1, -1), ("dtype", 9, -1), ("B", 1 << 26, -2), ("q", None, -1),
                                            ("out", None, -1), ("k_pre", None, -1), ("v_suf", None, -1), ("q", 4097, -1), ("lse", 4098, -1),
                                            ("prefix_len", 4097, -1), ("kp_st", -1, -1), ("o_sh", -64, -1), ("scale", float("inf"), -1),
                                            ("scale", float("nan"), -1), ("P", (1 << 30) + 1, -2), ("B", 0, 0), ("Lq", 0, 0)])
def test_refusals(lib, field, value, rc):
    a = _args()
    setattr(a, field, value)
    assert lib.hpmn_prefix_attn(C.byref(a), None) == rc
    assert lib.hpmn_prefix_attn(None, None) == -1 and lib.hpmn_prefix_attn_workspace_bytes(None) == 0


@pytest.mark.parametrize("sizes", [(2, 1, 4, 2, 64, 100, 8), (1, 1, 1, 1, 128, 1 << 20, 0), (3, 9, 8, 2, 40, 5000, 77), (500, 1, 16, 4, 128, 32768, 64)])
def test_workspace_is_asked_for(lib, sizes):
    a = _args()
    a.B, a.Lq, a.Hq, a.Hkv, a.D, a.P, a.S = sizes
    need = lib.hpmn_prefix_attn_workspace_bytes(C.byref(a))
    if need:
        for ws, n in ((None, need), (4096, need - 1), (4104, need)):
            a.workspace, a.workspace_bytes = ws, n
            assert lib.hpmn_prefix_attn(C.byref(a), None) == -1


@pytest.mark.parametrize("sizes", [(1 << 25, 1, 1, 1, 8, 16, 16), (1, 1, 1 << 24, 1 << 24, 8, 16, 0), (1 << 26, 1, 1, 1, 8, 16, 4)])
def test_more_threads_than_a_launch_has_are_refused(lib, sizes):
    a = _args()
    a.B, a.Lq, a.Hq, a.Hkv, a.D, a.P, a.S = sizes
    assert lib.hpmn_prefix_attn(C.byref(a), None) == -2


def test_struct_layout(tmp_path):
    st = _lib.HpmnPrefixAttn
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "hpmn_hip.h"', 'int main(void){printf("%zu", sizeof(HpmnPrefixAttn));']
    lines += ['printf(" %%zu", offsetof(HpmnPrefixAttn, %s));' % f for f, _ in st._fields_] + ["return 0;}"]
    src = tmp_path / "l.c"
    src.write_text("\n".join(lines))
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "l")])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / "l")], text=True).split()]
    assert got == [C.sizeof(st)] + [getattr(st, f).offset for f, _ in st._fields_]


def test_wrapper_refuses_host_tensors():
    q = torch.zeros(2, 1, 4, 64)
    with pytest.raises(ValueError):
        ops.shared_prefix_attention(q, q[0], q[0])


# ------------------------------------------------------------------------------------------------------------------ oracle
def oracle(q, kp, vp, ks, vs, plen, slen, scale):
    """Row by row in float64: (out, lse, rms) with rms the root mean square of p v, what roundings of p spread over."""
    q, kp, vp = (t.double().cpu() for t in (q, kp, vp))
    B, Lq, Hq, D = q.shape
    S = 0 if ks is None else ks.shape[1]
    if S:
        ks, vs = ks.double().cpu(), vs.double().cpu()
    G = Hq // kp.shape[1]
    plen = kp.shape[0] if plen is None else max(0, min(int(plen), kp.shape[0]))
    out, lse = torch.zeros(B, Lq, Hq, D, dtype=torch.float64), torch.full((B, Lq, Hq), -math.inf, dtype=torch.float64)
    spread = torch.zeros(B, Lq, Hq, D, dtype=torch.float64)
    for b in range(B):
        n = S if slen is None else max(0, min(int(slen[b]), S))
        for i in range(Lq):
            seen = max(0, min(n, n - Lq + 1 + i))
            for h in range(Hq):
                k, v = kp[:plen, h // G], vp[:plen, h // G]
                if S:
                    k, v = torch.cat([k, ks[b, :seen, h // G]]), torch.cat([v, vs[b, :seen, h // G]])
                if len(k) == 0:
                    continue
                s = scale * (k @ q[b, i, h])
                p = torch.softmax(s, 0)
                out[b, i, h], lse[b, i, h] = p @ v, torch.logsumexp(s, 0)
                spread[b, i, h] = p @ v.abs()
    return out, lse, spread


def inputs(B, Lq, Hq, Hkv, D, P, S, dtype, seed=0, sharp=1.5):
    g = torch.Generator().manual_seed(seed)
    f = lambda *s: torch.randn(*s, generator=g).to("cuda", dtype)  # noqa: E731
    q = (sharp * torch.randn(B, Lq, Hq, D, generator=g)).to("cuda", dtype)
    return q, f(P, Hkv, D), f(P, Hkv, D), (f(B, S, Hkv, D) if S else None), (f(B, S, Hkv, D) if S else None)


def check(q, kp, vp, ks=None, vs=None, plen=None, slen=None, scale=None):
    """Tolerances.  16-bit types: out is rounded once (half a step of |out|) and every probability once on its way into the
    second product (half a step of it, so at most half a step of sum p |v|).  Scores: a product of 16-bit values is exact in
    fp32, the sum over D <= 128 rounds by at most 2^-24 * 8 (tree of partial sums in an MFMA chain, D / 16 links) of
    sum |q k| scale <= 40: 2e-5 absolute, which exp turns into a relative 2e-5 of p; twice that with the running rescales.
    fp32: the same without the two storage roundings, with D links of 2^-24 at most: sum |q k| scale 2^-24 sqrt(D) <= 3e-5."""
    dt = q.dtype
    out, lse = ops.shared_prefix_attention(q, kp, vp, ks, vs, prefix_len=plen, suffix_len=slen, scale=scale, want_lse=True)
    assert out.shape == q.shape and out.dtype == dt and lse.shape == q.shape[:3]
    want, wlse, spread = oracle(q, kp, vp, ks, vs, plen, slen, scale if scale is not None else q.shape[-1] ** -0.5)
    half = 0.0 if dt == torch.float32 else torch.finfo(dt).eps / 2
    tol = half * (want.abs() + spread) + 6e-5 * spread + 1e-7
    got = out.double().cpu()
    assert torch.isfinite(got).all()
    over = (got - want).abs() - tol
    assert over.max() <= 0, "off by %.3g, %.3g over" % ((got - want).abs().max(), over.max())
    none = torch.isinf(wlse)
    l = lse.double().cpu()
    assert (l[none] == -math.inf).all() and not out.cpu()[none].any()
    assert ((l - wlse)[~none].abs() <= 6e-5 + 2e-7 * wlse[~none].abs()).all()
    assert torch.equal(ops.shared_prefix_attention(q, kp, vp, ks, vs, prefix_len=plen, suffix_len=slen, scale=scale), out)
    return out, lse


def i32(*v):
    return torch.tensor(v, dtype=torch.int32).cuda()


SIZES = [  # B, Lq, Hq, Hkv, D, P, S
    (1, 1, 1, 1, 64, 1, 0), (1, 1, 1, 1, 32, 0, 1), (2, 1, 2, 1, 128, 31, 3), (3, 1, 4, 2, 64, 64, 0), (5, 1, 3, 3, 40, 65, 17),
    (8, 1, 1, 1, 64, 1000, 0), (33, 1, 4, 1, 64, 257, 65), (1, 1, 8, 8, 128, 4100, 5), (130, 1, 2, 1, 32, 513, 1), (2, 7, 6, 2, 64, 129, 40),
    (3, 33, 4, 2, 96, 300, 33), (1, 40, 5, 1, 72, 50, 200), (4, 2, 1, 1, 1, 10, 4), (2, 1, 2, 2, 17, 100, 9), (70, 3, 2, 1, 128, 700, 10),
    (300, 1, 1, 1, 16, 90, 2), (2, 16, 8, 1, 64, 2000, 100)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("size", SIZES)
def test_against_float64(size, dtype):
    B, Lq, Hq, Hkv, D, P, S = size
    x = inputs(B, Lq, Hq, Hkv, D, P, S, DTYPES[dtype], seed=sum(size))
    check(*x)
    if S:
        n = torch.randint(0, S + 1, (B,), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
        n[0] = 0
        check(*x, slen=n.cuda())
    check(*x, plen=i32(max(0, P - 3)), scale=-0.3 / D ** 0.5)


MANY = [  # a few own keys of very many sequences: joined with the prefix's parts
    (600, 1, 1, 1, 64, 100, 1), (130, 3, 8, 4, 96, 300, 3), (256, 2, 4, 2, 40, 70, 8), (512, 1, 2, 1, 17, 40, 5), (512, 1, 1, 1, 32, 2100, 4),
    (1100, 1, 2, 1, 128, 200, 2), (1030, 1, 4, 1, 24, 90, 7), (2100, 1, 1, 1, 3, 0, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("size", MANY)
def test_few_keys_of_many_sequences(size, dtype):
    B, Lq, Hq, Hkv, D, P, S = size
    q, kp, vp, ks, vs = inputs(*size, DTYPES[dtype], seed=sum(size))
    check(q, kp, vp, ks, vs)
    n = torch.randint(-1, S + 2, (B,), generator=torch.Generator().manual_seed(2), dtype=torch.int32)
    want = check(q, kp, vp, ks, vs, slen=n.cuda(), scale=-0.4 / D ** 0.5)
    for b in range(B):
        for t in (ks, vs):
            t[b, max(0, int(n[b])):] = float("nan")
    got = ops.shared_prefix_attention(q, kp, vp, ks, vs, suffix_len=n.cuda(), scale=-0.4 / D ** 0.5, want_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_few_keys_of_many_sequences_strides(dtype):
    """Head-major storage, one key row for all, odd storage offsets, no scale, a prefix of length zero."""
    dt = DTYPES[dtype]
    q, kp, vp, ks, vs = inputs(300, 1, 4, 2, 64, 150, 4, dt)
    want = check(q, kp, vp, ks, vs)
    major = lambda t: t.transpose(-2, -3).contiguous().transpose(-2, -3)  # noqa: E731
    assert torch.equal(check(q, kp, vp, major(ks), major(vs))[0], want[0])
    flat = torch.empty(2, ks.numel() + 1, device="cuda", dtype=dt)
    ko, vo = flat[0, 1:].view(ks.shape), flat[1, :-1].view(vs.shape)
    ko.copy_(ks)
    vo.copy_(vs)
    check(q, kp, vp, ko, vo)
    check(q, kp, vp, ks[:, :1].expand(300, 4, 2, 64), vs)
    check(q, kp, vp, ks, vs, scale=0.0)
    check(q, kp, vp, ks, vs, plen=i32(0))
    ks[7] = -float("inf")                                              # scores of -inf where q's sign is one: no part
    q[7] = q[7].abs()
    out = ops.shared_prefix_attention(q, kp, vp, ks, vs)
    assert (out[7].double() - ops.shared_prefix_attention(q[7:8], kp, vp)[0].double()).abs().max() <= 4 * max(torch.finfo(dt).eps, 1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_lengths(dtype):
    """Every prefix length around the tile borders; lengths outside the range are clamped; nothing visible gives zeros."""
    x = inputs(3, 2, 2, 1, 64, 140, 70, DTYPES[dtype])
    for p in (0, 1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 140, 141, -5):
        check(*x, plen=i32(p), slen=i32(0, 70, 35))
    for s in ((1, 2, 3), (31, 32, 33), (63, 64, 65), (70, 71, -1)):
        check(*x, plen=i32(20), slen=i32(*s))
    out, lse = check(*x, plen=i32(0), slen=i32(0, 1, 2))
    assert not out[0].any() and not out[1, 0].any() and out[1, 1].any() and out[2].any()
    # no key axis at all
    q, kp, vp, _, _ = x
    out, lse = check(q, kp[:0], vp[:0])
    assert not out.any() and (lse == -math.inf).all()
    assert ops.shared_prefix_attention(q[:0], kp, vp).shape == (0, 2, 2, 64)
    assert ops.shared_prefix_attention(q[:, :0], kp, vp).shape == (3, 0, 2, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("fill", [float("nan"), float("inf"), -float("inf")])
def test_keys_behind_the_lengths_are_not_looked_at(dtype, fill):
    q, kp, vp, ks, vs = inputs(40, 1, 2, 1, 64, 200, 50, DTYPES[dtype])
    plen = i32(77)
    slen = torch.arange(40, dtype=torch.int32).cuda()
    want = check(q, kp, vp, ks, vs, plen, slen)
    for t in (kp, vp):
        t[77:] = fill
    for t in (ks, vs):
        for b in range(40):
            t[b, b:] = fill
    got = ops.shared_prefix_attention(q, kp, vp, ks, vs, prefix_len=plen, suffix_len=slen, want_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("B", [3, 80])
def test_infinite_keys_beside_unused_columns(dtype, B):
    """A key of -inf scores takes no part (its score is -inf), also where the kernel pads the head dimension (40 of 64)."""
    q, kp, vp, _, _ = inputs(B, 1, 1, 1, 40, 300, 0, DTYPES[dtype])
    q = q.abs()
    keep = torch.arange(300, device="cuda") % 7 != 3
    want = check(q, kp[keep].contiguous(), vp[keep].contiguous())
    kp[~keep] = -float("inf")
    out, lse = ops.shared_prefix_attention(q, kp, vp, want_lse=True)
    # the same sums in another order and, for 16-bit types, probabilities of another running maximum: one rounding each
    assert (out.double() - want[0].double()).abs().max() <= 4 * max(torch.finfo(DTYPES[dtype]).eps, 1e-5)
    assert (lse - want[1]).abs().max() < 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_extreme_scores(dtype):
    """Scores far apart and huge alike: one key takes all; equal keys share; a late key overtakes by a lot.  Many small
    probabilities beside one large one still add up (they would vanish below half a step of the type if they were rounded
    to it unscaled: 2^-24 of fp16 against 1)."""
    dt = DTYPES[dtype]
    q, kp, vp, _, _ = inputs(4, 1, 1, 1, 64, 300, 0, dt)
    kp[:] = 0
    kp[250, 0] = q[2, 0, 0]
    check(q, kp, vp, scale=30.0)
    check(q, kp, vp, scale=1e-3)
    kp[:] = kp[:1]
    check(q, kp, vp)
    P = 40000
    q = torch.zeros(1, 1, 1, 32, device="cuda", dtype=dt)
    q[..., 0] = 1
    kp = torch.zeros(P, 1, 32, device="cuda", dtype=dt)
    vp = torch.ones(P, 1, 32, device="cuda", dtype=dt)
    kp[P // 2, 0, 0] = 18.0                                            # every other p is e^-18 = 1.5e-8 of it
    vp[P // 2] = 0
    check(q, kp, vp, scale=1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_strides_and_alignment(dtype):
    """Head-major storage, q / k / v cut out of one buffer, one suffix shared by all rows, odd storage offsets: same numbers."""
    dt = DTYPES[dtype]
    x = inputs(6, 3, 4, 2, 64, 150, 20, dt)
    want = check(*x)
    q, kp, vp, ks, vs = x
    major = lambda t: t.transpose(-2, -3).contiguous().transpose(-2, -3)  # noqa: E731
    assert torch.equal(check(*(major(t) for t in x))[0], want[0])
    kv = torch.stack([kp, vp], 1)                                      # [P, 2, Hkv, D]
    kvs = torch.cat([ks, vs], -1)                                      # [B, S, Hkv, 2 D]
    assert torch.equal(check(q, kv[:, 0], kv[:, 1], kvs[..., :64], kvs[..., 64:])[0], want[0])

    def odd(t):
        flat = torch.empty(t.numel() + 1, device="cuda", dtype=dt)
        flat[1:] = t.reshape(-1)
        return flat[1:].reshape(t.shape)

    got = check(*(odd(t) for t in x))
    assert (got[0].double() - want[0].double()).abs().max() <= torch.finfo(dt).eps * 4 + 6e-5
    check(q, kp, vp, ks[:1].expand(6, 20, 2, 64), vs[:1].expand(6, 20, 2, 64))
    check(q, kp[:1].expand(150, 2, 64), vp)
    kw = torch.zeros(150, 2, 70, device="cuda", dtype=dt)              # rows that no 16-byte access can take
    kw[..., 3:67] = kp
    check(q, kw[..., 3:67], vp, ks, vs)


@pytest.mark.gpu
def test_wrapper_refusals():
    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    q, kp, ks = z(2, 1, 4, 64), z(9, 2, 64), z(2, 5, 2, 64)
    f = ops.shared_prefix_attention
    bad = [lambda: f(q[0], kp, kp), lambda: f(q, kp, kp[:8]), lambda: f(q, kp.half(), kp.half()), lambda: f(q.double(), kp.double(), kp.double()),
           lambda: f(q, kp.cpu(), kp), lambda: f(q, kp, kp, ks), lambda: f(q, kp, kp, ks[:1], ks[:1]), lambda: f(q, kp, kp, ks, ks[:, :4]),
           lambda: f(q[:, :, :3], kp, kp), lambda: f(q[..., :32], kp, kp), lambda: f(q, kp, kp, scale=float("nan")),
           lambda: f(q, kp, kp, prefix_len=torch.zeros(1, device="cuda", dtype=torch.int64)), lambda: f(q, kp, kp, prefix_len=5),
           lambda: f(q, kp, kp, ks, ks, suffix_len=torch.zeros(3, device="cuda", dtype=torch.int32)),
           lambda: f(z(2, 1, 4, 160), z(9, 2, 160), z(9, 2, 160)), lambda: f(q.transpose(2, 3), z(9, 2, 4), z(9, 2, 4)),
           lambda: f(q, kp[:, :0], kp[:, :0]), lambda: f(q, kp[0], kp[0])]
    for i, c in enumerate(bad):
        with pytest.raises((ValueError, AttributeError)):
            c()
            pytest.fail("call %d was accepted" % i)


@pytest.mark.gpu
@pytest.mark.parametrize("B,Lq,D,dtype", [(4, 1, 64, "bf16"), (200, 1, 64, "bf16"), (3, 20, 64, "bf16"), (90, 1, 128, "fp16"), (5, 1, 128, "fp32")])
def test_other_stream_and_captured_graph(B, Lq, D, dtype):
    """The same numbers on a side stream; a replayed graph follows its inputs, its prefix length and its suffix lengths."""
    q, kp, vp, ks, vs = inputs(B, Lq, 4, 2, D, 900, 30, DTYPES[dtype])
    plen, slen = i32(900), torch.full((B,), 30, dtype=torch.int32).cuda()
    f = lambda: ops.shared_prefix_attention(q, kp, vp, ks, vs, prefix_len=plen, suffix_len=slen, want_lse=True)  # noqa: E731
    want = f()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = f()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = f()
    for k in range(3):
        plen.fill_(900 - 333 * k)
        slen.copy_(torch.randint(0, 31, (B,)).to(torch.int32))
        kp[:10] = torch.randn_like(kp[:10])
        want = f()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1]), k


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """A prefix whose rows lie 2^23 elements apart, so that element offsets pass 2^32."""
    P, D = 600, 64
    q, kp, vp, _, _ = inputs(3, 1, 1, 1, D, P, 0, torch.bfloat16)
    store = torch.empty((P - 1) * (1 << 23) + 2 * D, device="cuda", dtype=torch.bfloat16)
    K = torch.as_strided(store, (P, 1, D), (1 << 23, D, 1))
    V = torch.as_strided(store, (P, 1, D), (1 << 23, D, 1), D)
    K.copy_(kp)
    V.copy_(vp)
    assert torch.equal(ops.shared_prefix_attention(q, K, V), ops.shared_prefix_attention(q, kp, vp))


@pytest.mark.gpu
def test_prefix_and_suffix_agree():
    """The same keys as prefix of all rows, as suffix of each row, or cut anywhere between the two."""
    q, kp, vp, _, _ = inputs(5, 1, 4, 2, 64, 96, 0, torch.float32)
    want = check(q, kp, vp)
    for cut in (0, 1, 40, 95):
        ks, vs = (t[None, cut:].expand(5, 96 - cut, 2, 64) for t in (kp, vp))
        got = check(q, kp[:cut], vp[:cut], ks, vs)
        assert (got[0] - want[0]).abs().max() < 2e-6 and (got[1] - want[1]).abs().max() < 2e-6


# ------------------------------------------------------------------------------ many rows: the pipelined whole tiles
def many_rows_check(q, kp, vp, scale, plen=None):
    """q [M, 1, H, D] over H key heads of their own against float64 on the GPU; the tolerances of check()."""
    dt, (M, _, H, D) = q.dtype, q.shape
    p = kp.shape[0] if plen is None else plen
    out, lse = ops.shared_prefix_attention(q, kp, vp, prefix_len=None if plen is None else i32(plen), scale=scale, want_lse=True)
    assert torch.equal(ops.shared_prefix_attention(q, kp, vp, prefix_len=None if plen is None else i32(plen), scale=scale), out)
    half = torch.finfo(dt).eps / 2
    for h0 in range(0, H, 32):
        part = slice(h0, min(H, h0 + 32))
        k = kp[:p, part].double().permute(1, 2, 0).contiguous()
        v = vp[:p, part].double().permute(1, 0, 2).contiguous()
        s = scale * torch.bmm(q[:, 0, part].double().transpose(0, 1).contiguous(), k)
        wlse = torch.logsumexp(s, -1)
        w = torch.exp(s - wlse[..., None])
        want, spread = torch.bmm(w, v), torch.bmm(w, v.abs())
        got = out[:, 0, part].double().transpose(0, 1)
        over = (got - want).abs() - (half * (want.abs() + spread) + 6e-5 * spread + 1e-7)
        assert over.max() <= 0, "heads from %d: off by %.3g, %.3g over" % (h0, (got - want).abs().max(), over.max())
        l = lse[:, 0, part].double().transpose(0, 1)
        assert ((l - wlse).abs() <= 6e-5 + 2e-7 * wlse.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [32, 40, 64, 72, 96, 128])
@pytest.mark.parametrize("P", [356, 421, 640, 1100, 2200])
def test_long_ranges_of_many_rows(P, D, dtype):
    """256 key heads fill the chip, so a range of keys is long: four, six, ten, sixteen and eighteen tiles of 64 in one go, with and
    without a rest; and the same with the prefix cut at the device."""
    dt = DTYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(P + D)
    M = 66 if D >= 96 else 128
    q = (1.5 * torch.randn(M, 1, 256, D, device="cuda", generator=g)).to(dt)
    kp, vp = (torch.randn(P, 256, D, device="cuda", generator=g).to(dt) for _ in range(2))
    many_rows_check(q, kp, vp, D ** -0.5)
    many_rows_check(q, kp, vp, -D ** -0.5, plen=P - 70)
    kp[P - 70:] = float("nan")
    vp[P - 70:] = float("inf")
    want = ops.shared_prefix_attention(q, kp[:P - 70], vp[:P - 70])
    got = ops.shared_prefix_attention(q, kp, vp, prefix_len=i32(P - 70))
    assert (got.double() - want.double()).abs().max() <= 4 * torch.finfo(dt).eps * float(want.double().abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128])
def test_rising_maxima_of_many_rows(D, dtype):
    """The running maximum rises by 1 to 120 (in powers of two) at every step of 32 keys of a range in turn -- the first and
    the second of a tile, across pairs of tiles, in the last one -- once, or at every step, so that it lags, is raised and rescales
    the output late.  Rows see the keys as they rise, as they fall, half as far apart and all alike."""
    dt, P, H, M = DTYPES[dtype], 1100, 256, 72
    g = torch.Generator(device="cuda").manual_seed(D)
    rises = torch.tensor([1.0, 2.5, 4.0, 7.0, 9.0, 20.0, 120.0], device="cuda")
    step = torch.arange(P, device="cuda") // 32                        # 0 .. 34
    level = torch.zeros(P, H, device="cuda")
    for h in range(H):
        r, at = rises[h % 7], h // 7 % 35
        level[:, h] = (step >= at) * r if h < 245 else step * r
    q = torch.zeros(M, 1, H, D, device="cuda", dtype=dt)
    q[:, :, :, 0] = torch.tensor([1.0, -1.0, 0.5, 0.0], device="cuda", dtype=dt).repeat(M // 4)[:, None, None]
    q[0::5, :, :, 0] = 1.0
    kp = torch.zeros(P, H, D, device="cuda", dtype=dt)
    kp[:, :, 0] = (level + 0.5 * torch.randn(P, H, device="cuda", generator=g)).to(dt)
    vp = torch.randn(P, H, D, device="cuda", generator=g).to(dt)
    many_rows_check(q, kp, vp, math.log(2.0))


@pytest.mark.parametrize("sizes,splits", [((8, 1, 1, 1, 64, 1000, 0), True), ((1, 1, 1, 1, 128, 1 << 20, 0), True), ((3, 9, 8, 2, 40, 5000, 77), True),
                                          ((500, 1, 16, 4, 128, 32768, 64), True), ((300, 1, 8, 8, 128, 4096, 1), True),
                                          ((2, 1, 4, 2, 64, 100, 0), False), ((1, 1, 1, 1, 32, 0, 0), False)])
def test_long_prefixes_and_own_keys_are_cut_up(lib, sizes, splits):
    """Where keys are to be shared out a workspace is asked for, and has to be there, large enough and aligned; a short prefix by
    itself needs none."""
    a = _args()
    a.B, a.Lq, a.Hq, a.Hkv, a.D, a.P, a.S = sizes
    need = lib.hpmn_prefix_attn_workspace_bytes(C.byref(a))
    assert (need > 0) == splits
    for ws, n in ((None, need), (4096, need - 1), (4104, need)) if splits else ():
        a.workspace, a.workspace_bytes = ws, n
        assert lib.hpmn_prefix_attn(C.byref(a), None) == -1


@pytest.mark.gpu
def test_refusals_are_value_errors():
    """Every bad argument is refused by name, none by an accident further in."""
    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    q, kp, ks = z(2, 1, 4, 64), z(9, 2, 64), z(2, 5, 2, 64)
    n = lambda *s, dtype=torch.int32: torch.zeros(*s, device="cuda", dtype=dtype)  # noqa: E731
    f = ops.shared_prefix_attention
    for i, call in enumerate([lambda: f(q[0], kp, kp), lambda: f(q, kp, kp[:8]), lambda: f(q, kp.half(), kp.half()),
                              lambda: f(q.double(), kp.double(), kp.double()), lambda: f(q, kp.cpu(), kp), lambda: f(q, kp, kp, ks),
                              lambda: f(q, kp, kp, None, ks), lambda: f(q, kp, kp, ks[:1], ks[:1]), lambda: f(q, kp, kp, ks, ks[:, :4]),
                              lambda: f(q, kp, kp, ks[0], ks[0]), lambda: f(q[:, :, :3], kp, kp), lambda: f(q[..., :32], kp, kp),
                              lambda: f(q, kp, kp, scale=float("nan")), lambda: f(q, kp, kp, scale=float("inf")),
                              lambda: f(q, kp, kp, prefix_len=n(1, dtype=torch.int64)), lambda: f(q, kp, kp, prefix_len=5),
                              lambda: f(q, kp, kp, prefix_len=n(2)), lambda: f(q, kp, kp, ks, ks, suffix_len=n(3)),
                              lambda: f(q, kp, kp, ks, ks, suffix_len=[1, 2]), lambda: f(z(2, 1, 4, 160), z(9, 2, 160), z(9, 2, 160)),
                              lambda: f(q.transpose(2, 3), z(9, 2, 4), z(9, 2, 4)), lambda: f(q, kp[:, :0], kp[:, :0]), lambda: f(q, kp[0], kp[0])]):
        with pytest.raises(ValueError):
            call()
            pytest.fail("call %d was accepted" % i)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(37, 1, 4, 2, 64, 900, 30), (5, 9, 4, 2, 40, 300, 30), (600, 1, 2, 1, 64, 400, 3), (64, 1, 2, 1, 32, 500, 0)])
def test_large_batches_are_cut_up_for_their_workspace(size, monkeypatch):
    """With as little scratch as one sequence needs, and some amounts above: the same results, to the tolerances of check()."""
    B, Lq, Hq, Hkv, D, P, S = size
    x = inputs(*size, torch.bfloat16, seed=sum(size))
    slen = torch.randint(0, S + 1, (B,), generator=torch.Generator().manual_seed(3), dtype=torch.int32).cuda() if S else None
    made, empty = [], torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **k: made.append(empty(*a, **k)) or made[-1])
    check(*x, slen=slen)
    whole = max((t.numel() for t in made if t.dtype == torch.uint8), default=0)
    assert (whole > 0) == (size[-1] > 0)                               # (the short prefix by itself needs none: nothing to cut)
    for most in (0, whole // 5, whole // 2 + 1):
        made.clear()
        monkeypatch.setattr(ops, "_ATTN_WORKSPACE_MOST", most)
        check(*x, slen=slen)
        assert max((t.numel() for t in made if t.dtype == torch.uint8), default=-1) < whole


def test_the_largest_batches_need_more_scratch_than_one_call_takes(lib):
    """What is cut up: 2^25 rows and 2^26 rows of 128 with keys of their own ask for tens of GB."""
    a = _args()
    a.B, a.Lq, a.Hq, a.Hkv, a.D, a.P, a.S = 1 << 19, 4, 16, 4, 128, 512, 48
    assert lib.hpmn_prefix_attn_workspace_bytes(C.byref(a)) > 8 * ops._ATTN_WORKSPACE_MOST
