"""The gated linear recurrence (hpmn_gated_scan_fwd / _bwd / _step): C ABI refusals on the CPU, results against a float64
restatement of the recurrence on the GPU."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

from hpmn_amd import _lib, build, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
TILE = _lib.HPMN_GATED_SCAN_TILE


@pytest.fixture(scope="module")
def lib():
    build.build_library()
    return _lib.load()


# ------------------------------------------------------------------------------------------------------------------ CPU
def test_struct_layouts(tmp_path):
    structs = {"HpmnGatedScan": _lib.HpmnGatedScan, "HpmnGatedScanBwd": _lib.HpmnGatedScanBwd, "HpmnGatedStep": _lib.HpmnGatedStep}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "hpmn_hip.h"', "int main(void){"]
    for name, st in structs.items():
        lines.append('printf("%s %%zu\\n", sizeof(%s));' % (name, name))
        for fname, _ in st._fields_:
            lines.append('printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (name, fname, name, fname))
    lines.append('printf("TILE %d\\nMAXIDX %d\\n", HPMN_GATED_SCAN_TILE, HPMN_STEP_MAX_INDEXED);return 0;}')
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines))
    exe = str(tmp_path / "layout")
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe])
    got = dict(l.split() for l in subprocess.check_output([exe], text=True).splitlines())
    assert int(got["TILE"]) == TILE and int(got["MAXIDX"]) == _lib.HPMN_STEP_MAX_INDEXED
    for name, st in structs.items():
        assert int(got[name]) == C.sizeof(st), name
        for fname, _ in st._fields_:
            assert int(got["%s.%s" % (name, fname)]) == getattr(st, fname).offset, (name, fname)


def _scan_args(cls):
    """A valid-looking descriptor (the pointers are never followed: every call below is refused or empty)."""
    a = cls()
    a.B, a.T, a.C, a.dtype, a.period = 2, 8, 16, _lib.HPMN_F32, 2
    for f in ("z", "v", "y", "h_last", "saved", "d_y", "d_z", "d_v"):
        if hasattr(a, f):
            setattr(a, f, 4096)
    return a


@pytest.mark.parametrize("field,value,rc", [("B", -1, -1), ("T", 0, -1), ("C", 0, -1), ("period", 0, -1), ("period", 3, -1), ("dtype", 3, -1),
                                            ("z", None, -1), ("v", None, -1), ("z", 4098, -1), ("z_st", -4, -1), ("B", 2 ** 30, -2), ("v_st", 2 ** 31, -2), ("T", 2 ** 30 + 2, -2),
                                            ("B", 0, 0)])
def test_scan_refusals(lib, field, value, rc):
    for cls, fn in ((_lib.HpmnGatedScan, lib.hpmn_gated_scan_fwd), (_lib.HpmnGatedScanBwd, lib.hpmn_gated_scan_bwd)):
        a = _scan_args(cls)
        setattr(a, field, value)
        assert fn(C.byref(a), None) == rc, cls.__name__
    assert lib.hpmn_gated_scan_fwd(None, None) == -1 and lib.hpmn_gated_scan_bwd(None, None) == -1
    assert lib.hpmn_gated_scan_workspace_bytes(0, 8, 8) == 0 and lib.hpmn_gated_scan_workspace_bytes(-1, 8, 8) == 0


@pytest.mark.parametrize("B,T,Cc", [(1 << 24, 128, 64), (1 << 26, 1, 16), (1, 2 ** 31 - 1, 1), (1 << 10, 128, 1 << 30), (2 ** 31 - 1, 1, 2 ** 31 - 1)])
def test_more_threads_than_a_launch_has_are_refused(lib, B, T, Cc):
    for cls, fn in ((_lib.HpmnGatedScan, lib.hpmn_gated_scan_fwd), (_lib.HpmnGatedScanBwd, lib.hpmn_gated_scan_bwd)):
        a = _scan_args(cls)
        a.B, a.T, a.C, a.period = B, T, Cc, 1
        assert fn(C.byref(a), None) == -2
    assert lib.hpmn_gated_scan_workspace_bytes(B, T, Cc) == 0
    s = _lib.HpmnGatedStep()
    s.B, s.C, s.z, s.v, s.state, s.y, s.z_s, s.v_s, s.y_s, s.state_s, s.n_users = 1 << 26, 4, 4096, 4096, 4096, 4096, 4, 4, 4, 4, 1 << 26
    assert lib.hpmn_gated_scan_step(C.byref(s), None) == -2


def test_scan_needs_an_output_and_saved_states(lib):
    a = _scan_args(_lib.HpmnGatedScan)
    a.y = a.h_last = a.saved = None
    assert lib.hpmn_gated_scan_fwd(C.byref(a), None) == -1
    b = _scan_args(_lib.HpmnGatedScanBwd)
    b.saved = None
    assert lib.hpmn_gated_scan_bwd(C.byref(b), None) == -1
    # a workspace that is asked for has to be there and large enough
    a = _scan_args(_lib.HpmnGatedScan)
    a.B, a.T, a.C, a.period = 1, 1 << 16, 64, 1
    need = lib.hpmn_gated_scan_workspace_bytes(a.B, a.T, a.C)
    if need:
        assert lib.hpmn_gated_scan_fwd(C.byref(a), None) == -1
        a.workspace, a.workspace_bytes = 4096, need - 1
        assert lib.hpmn_gated_scan_fwd(C.byref(a), None) == -1
        a.workspace, a.workspace_bytes = 4100, need
        assert lib.hpmn_gated_scan_fwd(C.byref(a), None) == -1


@pytest.mark.parametrize("field,value,rc", [("B", -1, -1), ("C", 0, -1), ("dtype", 7, -1), ("flags", 4, -1), ("n_users", -1, -1), ("z", None, -1),
                                            ("state", None, -1), ("state_s", 15, -1), ("v", 4097, -1), ("B", 5000, -2), ("B", 0, 0)])
def test_step_refusals(lib, field, value, rc):
    a = _lib.HpmnGatedStep()
    a.B, a.C, a.dtype, a.flags, a.n_users, a.state_s = 2, 16, _lib.HPMN_BF16, _lib.HPMN_STEP_COMMIT, 9, 16
    a.z = a.v = a.state = a.user = 4096
    setattr(a, field, value)
    assert lib.hpmn_gated_scan_step(C.byref(a), None) == rc
    assert lib.hpmn_gated_scan_step(None, None) == -1
    a = _lib.HpmnGatedStep()
    a.B, a.C, a.n_users, a.state_s, a.z, a.v, a.state = 2, 16, 9, 16, 4096, 4096, 4096
    assert lib.hpmn_gated_scan_step(C.byref(a), None) == -1            # neither committed nor an output
    a.y = 4096
    assert lib.hpmn_gated_scan_step(C.byref(a), None) == -1            # no user list: as many rows as states


def test_wrappers_refuse_host_tensors():
    z = torch.zeros(2, 4, 8)
    with pytest.raises(ValueError):
        ops.gated_scan_fwd(z, z)
    with pytest.raises(ValueError):
        ops.gated_scan_bwd(z, z, None, z)
    with pytest.raises(ValueError):
        ops.gated_scan_step(z[0], z[0], z[0])


# ------------------------------------------------------------------------------------------------------------------ oracle
def oracle(z, v, h0, begin, period, d_y=None, d_h_last=None):
    """The recurrence and its reverse, step by step, in float64 on the CPU."""
    z, v = z.double().cpu().numpy(), v.double().cpu().numpy()
    B, T, Cc = z.shape
    with np.errstate(over="ignore"):
        a, u = 1 / (1 + np.exp(-z)), 1 / (1 + np.exp(z))
    live = np.ones((B, T, 1), bool) if begin is None else (np.arange(T)[None] >= begin.cpu().numpy()[:, None])[..., None]
    a, u, v = np.where(live, a, 1.0), np.where(live, u, 0.0), np.where(live, v, 0.0)
    h = np.zeros((B, T + 1, Cc))
    if h0 is not None:
        h[:, 0] = h0.double().cpu().numpy()
    for t in range(T):
        h[:, t + 1] = a[:, t] * h[:, t] + u[:, t] * v[:, t]
    got = {"y": h[:, period::period], "h_last": h[:, T]}
    if d_y is None and d_h_last is None:
        return got
    d = np.zeros((B, T, Cc))
    if d_y is not None:
        d[:, period - 1::period] = d_y.double().cpu().numpy()
    G = np.zeros((B, Cc)) if d_h_last is None else d_h_last.double().cpu().numpy().copy()
    d_z, d_v = np.zeros((B, T, Cc)), np.zeros((B, T, Cc))
    for t in range(T - 1, -1, -1):
        G = G + d[:, t]
        d_v[:, t] = u[:, t] * G
        d_z[:, t] = G * (h[:, t] - v[:, t]) * a[:, t] * u[:, t]
        G = a[:, t] * G
    got.update(d_z=d_z, d_v=d_v, d_h0=G)
    return got


def close(name, got, want, dtype, size):
    """|got - want| <= storage rounding (half a step of the value) + fp32 error of the computation.  The states are averages of
    values bounded by `size` with weights that sum to at most 1, so errors do not grow along t: every step adds at most four
    fp32 roundings and one exp / reciprocal pair (2 ulp each, and |z| 2^-24 from the scaled exponent, |z| <= 16) and damps what
    came before by its own a.  The damping sum is at most 1 / (1 - a); 2e-5 covers 1 / (1 - a) up to ~50 steps of memory."""
    got = got.double().cpu().numpy()
    assert got.shape == want.shape, name
    assert np.isfinite(got).all(), name
    tol = torch.finfo(dtype).eps / 2 * np.abs(want) * (dtype != torch.float32) + 2e-5 * size + (1e-7 if dtype == torch.float16 else 0)
    bad = np.abs(got - want) - tol
    assert bad.max(initial=-1) <= 0, "%s: off by %.3g beyond %.3g" % (name, np.abs(got - want).max(), size)


def inputs(B, T, Cc, dtype, seed=0, strided=False, dev="cuda"):
    g = torch.Generator().manual_seed(seed)
    z, v = 1 + 1.5 * torch.randn(B, T, Cc, generator=g), torch.tanh(torch.randn(B, T, Cc, generator=g))
    if strided:
        proj = torch.cat([z, v], -1).to(dev, dtype)
        return proj[..., :Cc], proj[..., Cc:]
    return z.to(dev, dtype), v.to(dev, dtype)


def check(z, v, h0, begin, period, seed=1, d_h_last=True, with_dy=True, out=None):
    B, T, Cc = z.shape
    g = torch.Generator().manual_seed(seed)
    d_y = torch.randn(B, T // period, Cc, generator=g).to(z.device, z.dtype) if with_dy else None
    d_h = torch.randn(B, Cc, generator=g).to(z.device) if d_h_last else None
    y, h_last, saved = ops.gated_scan_fwd(z, v, h0=h0, begin=begin, period=period, train=True)
    d_z, d_v, d_h0 = ops.gated_scan_bwd(z, v, saved, d_y, d_h_last=d_h, begin=begin, period=period, out=out)
    want = oracle(z, v, h0, begin, period, d_y, d_h if d_h_last or with_dy else torch.zeros(B, Cc))
    size = max(1.0, float(np.abs(want["y"]).max(initial=0)), float(np.abs(want["h_last"]).max(initial=0)))
    close("y", y, want["y"], z.dtype, size)
    close("h_last", h_last, want["h_last"], torch.float32, size)
    # gradients: G is a sum of d_y with weights below 1 (largest |G| over the case is its scale), times |h - v| <= 2 size
    gsize = max(float(np.abs(want["d_h0"]).max(initial=0)), float(np.abs(want["d_v"]).max(initial=0)), 4.0)
    close("d_v", d_v, want["d_v"], z.dtype, gsize)
    close("d_z", d_z, want["d_z"], z.dtype, 2 * gsize * size)
    close("d_h0", d_h0, want["d_h0"], torch.float32, gsize)
    # inference form: the same numbers
    y2, h2, s2 = ops.gated_scan_fwd(z, v, h0=h0, begin=begin, period=period)
    assert s2 is None and torch.equal(y2, y) and torch.equal(h2, h_last)
    return y, h_last, d_z, d_v, d_h0


SHAPES = [(1, 1, 1, 1), (3, 1, 64, 1), (2, 2, 3, 2), (1, 15, 4, 5), (2, 16, 16, 1), (3, 17, 20, 1), (5, 100, 32, 2), (2, TILE - 1, 37, 1),
          (2, TILE, 64, 2), (3, TILE + 1, 65, 1), (2, 2 * TILE, 100, 4), (4, 517, 100, 1), (1, 1000, 130, 5), (300, 40, 8, 2),
          (1, 5000, 64, 1), (2, 4099, 12, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("shape", SHAPES)
def test_scan_against_float64(shape, dtype):
    B, T, Cc, period = shape
    z, v = inputs(B, T, Cc, DTYPES[dtype], seed=T + Cc)
    check(z, v, None, None, period)
    h0 = torch.randn(B, Cc, generator=torch.Generator().manual_seed(7)).cuda()
    begin = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(8), dtype=torch.int32)
    begin[0] = T if B > 1 else T // 2
    check(z, v, h0, begin.cuda(), period)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("Cc", [64, 37])
def test_strided_inputs_and_outputs(dtype, Cc):
    """Halves of one projection buffer, time-major storage, a row-strided h0, a broadcast gate, gradients into one buffer."""
    B, T = 3, 300
    dt = DTYPES[dtype]
    z, v = inputs(B, T, Cc, dt, strided=True)
    grad = torch.full((B, T, 2 * Cc), 7.0, device="cuda", dtype=dt)
    h0 = torch.randn(B, 2, Cc, device="cuda")[:, 1]
    r = check(z, v, h0, None, 1, out=(grad[..., :Cc], grad[..., Cc:]))
    assert r[2].data_ptr() == grad.data_ptr()
    zc, vc = z.contiguous(), v.contiguous()
    assert all(torch.equal(p, q) for p, q in zip(check(zc, vc, h0.contiguous(), None, 1), r))
    zt, vt = zc.transpose(0, 1).contiguous().transpose(0, 1), vc.transpose(0, 1).contiguous().transpose(0, 1)
    assert all(torch.equal(p, q) for p, q in zip(check(zt, vt, h0, None, 1), r))
    one = zc[:, :1].expand(B, T, Cc)                                   # the same gate at every step: stride 0
    check(one, vc, None, None, 1)
    # storage that starts one element behind an aligned address: same results
    flat = torch.empty(zc.numel() + 1, device="cuda", dtype=dt)
    flat[1:] = zc.reshape(-1)
    odd = flat[1:].reshape(zc.shape)
    y0, h_0, s0 = ops.gated_scan_fwd(zc, vc, train=True)
    y1, h_1, s1 = ops.gated_scan_fwd(odd, vc, train=True)
    assert torch.equal(y0, y1) and torch.equal(h_0, h_1) and torch.equal(s0, s1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_padded_steps_are_not_looked_at(dtype):
    B, T, Cc = 4, 261, 48
    z, v = inputs(B, T, Cc, DTYPES[dtype])
    begin = torch.tensor([T, 130, 0, T + 5], dtype=torch.int32).cuda()
    h0 = torch.randn(B, Cc, device="cuda")
    want = check(z, v, h0, begin, 1)
    for bad in (float("nan"), float("inf"), torch.finfo(DTYPES[dtype]).min):
        z2, v2 = z.clone(), v.clone()
        for b in range(B):
            z2[b, :int(begin[b])] = bad
            v2[b, :int(begin[b])] = bad
        got = check(z2, v2, h0, begin, 1)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    y, h_last, d_z, d_v, d_h0 = want
    assert torch.equal(h_last[0], h0[0]) and not d_z[0].any() and not d_v[0].any()
    assert not d_z[1, :130].any() and not d_v[1, :130].any()


@pytest.mark.gpu
def test_saturated_gates():
    """z = +-inf and +-1e4: the state is kept, or replaced; 1 - a keeps its digits where a rounds to 1."""
    z = torch.tensor([float("inf"), -float("inf"), 1e4, -1e4, 30.0, -30.0]).reshape(1, 6, 1).repeat(1, 1, 4).cuda().contiguous()
    v = torch.arange(1, 7.0).reshape(1, 6, 1).repeat(1, 1, 4).cuda().contiguous()
    h0 = torch.full((1, 4), 0.5).cuda()
    y, h_last, saved = ops.gated_scan_fwd(z, v, h0=h0, train=True)
    assert torch.allclose(y[0, :, 0].cpu(), torch.tensor([0.5, 2, 2, 4, 4, 6.0]), atol=1e-5)
    one = torch.ones(1, 6, 4).cuda()
    d_z, d_v, d_h0 = ops.gated_scan_bwd(z, v, saved, one)
    assert torch.isfinite(d_z).all() and torch.isfinite(d_v).all()
    # step 4 (z = 30): G = 1 (its own d_y; a of step 5 is 1e-13), d_v = 1 - sigmoid(30) = e^-30 to a few ulp of 30 * 2^-24
    assert abs(float(d_v[0, 4, 0]) / np.exp(-30.0) - 1) < 1e-5


@pytest.mark.gpu
def test_gradients_against_differences():
    """Central differences of a float64 loss through the kernel's own forward: step 2^-6 in fp32, so a difference carries
    rounding 2^-24 sqrt(n) / 2^-6 ~ 1e-4 of the loss's scale and curvature (2^-6)^2 / 6 ~ 4e-5 of the third derivative."""
    B, T, Cc = 2, 140, 8
    z, v = inputs(B, T, Cc, torch.float32)
    h0 = torch.randn(B, Cc, generator=torch.Generator().manual_seed(5)).cuda()
    wy, wh = torch.randn(B, T // 2, Cc, generator=torch.Generator().manual_seed(6)).cuda(), torch.randn(B, Cc).cuda()

    def loss(z, v, h0):
        y, h, _ = ops.gated_scan_fwd(z, v, h0=h0, period=2)
        return float((y.double() * wy.double()).sum() + (h.double() * wh.double()).sum())

    _, _, saved = ops.gated_scan_fwd(z, v, h0=h0, period=2, train=True)
    d = ops.gated_scan_bwd(z, v, saved, wy, d_h_last=wh, period=2)
    g = torch.Generator().manual_seed(9)
    for i, x in enumerate((z, v, h0)):
        for _ in range(6):
            at = tuple(int(torch.randint(0, n, (1,), generator=g)) for n in x.shape)
            hi, lo = x.clone(), x.clone()
            hi[at] += 2.0 ** -6
            lo[at] -= 2.0 ** -6
            args = [z, v, h0]
            diff = (loss(*[hi if j == i else t for j, t in enumerate(args)]) - loss(*[lo if j == i else t for j, t in enumerate(args)])) / 2.0 ** -5
            assert abs(diff - float(d[i][at])) < 2e-3 * max(1.0, abs(diff)), (i, at)


@pytest.mark.gpu
def test_missing_gradients_and_empty_calls():
    z, v = inputs(2, 130, 12, torch.float32)
    check(z, v, None, None, 1, d_h_last=False)
    check(z, v, None, None, 1, with_dy=False)
    _, _, saved = ops.gated_scan_fwd(z, v, train=True)
    d_z, d_v, d_h0 = ops.gated_scan_bwd(z, v, saved, None)
    assert not d_z.any() and not d_v.any() and not d_h0.any()
    for shape in ((0, 5, 8), (2, 0, 8), (2, 5, 0)):
        e = torch.empty(*shape, device="cuda")
        h0 = torch.randn(shape[0], shape[2], device="cuda")
        y, h_last, saved = ops.gated_scan_fwd(e, e, h0=h0, train=True)
        assert y.shape == shape and torch.equal(h_last, h0)
        d_h = torch.randn_like(h0)
        d_z, d_v, d_h0 = ops.gated_scan_bwd(e, e, saved, y, d_h_last=d_h)
        assert d_z.shape == shape and torch.equal(d_h0, d_h)
        assert not ops.gated_scan_fwd(e, e)[1].any()


@pytest.mark.gpu
def test_wrapper_refusals():
    z = torch.zeros(2, 6, 8, device="cuda")
    saved = torch.zeros(2, 1, 8, device="cuda")
    bad = [lambda: ops.gated_scan_fwd(z, z[:, :5]), lambda: ops.gated_scan_fwd(z, z.bfloat16()), lambda: ops.gated_scan_fwd(z.double(), z.double()),
           lambda: ops.gated_scan_fwd(z, z, period=4), lambda: ops.gated_scan_fwd(z, z, period=0), lambda: ops.gated_scan_fwd(z, z.cpu()),
           lambda: ops.gated_scan_fwd(z, z, h0=z[:, 0].half()), lambda: ops.gated_scan_fwd(z, z, h0=z[:, 0, :4]),
           lambda: ops.gated_scan_fwd(z, z, begin=torch.zeros(2, device="cuda", dtype=torch.int64)),
           lambda: ops.gated_scan_fwd(z, z, begin=torch.zeros(3, device="cuda", dtype=torch.int32)),
           lambda: ops.gated_scan_fwd(z.transpose(1, 2), z.transpose(1, 2)), lambda: ops.gated_scan_fwd(z[0], z[0]),
           lambda: ops.gated_scan_bwd(z, z, None, z), lambda: ops.gated_scan_bwd(z, z, saved[:1], z), lambda: ops.gated_scan_bwd(z, z, saved, z[:, :3]),
           lambda: ops.gated_scan_bwd(z, z, saved, z, out=(z, z[:, :1].expand(2, 6, 8))),
           lambda: ops.gated_scan_bwd(z, z, saved, z, out=(z.clone(), torch.as_strided(z.clone(), (2, 6, 8), (8, 8, 1)))),
           lambda: ops.gated_scan_bwd(z, z, saved, z, out=(z, z)), lambda: ops.gated_scan_fwd(z, z, begin=[0, 1]), lambda: ops.gated_scan_bwd(z, z, saved, z.half()),
           lambda: ops.gated_scan_step(z[0], z[0], z[0, :5]), lambda: ops.gated_scan_step(z[0], z[0], z[0].half()),
           lambda: ops.gated_scan_step(z[0], z[1], z[0, :1].expand(6, 8)),
           lambda: ops.gated_scan_step(z[0], z[0], z[0], torch.zeros(6, device="cuda")), lambda: ops.gated_scan_step(z, z, z[0])]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail("call %d was accepted" % i)


@pytest.mark.gpu
def test_other_stream_and_captured_graph():
    """The same numbers on a side stream, and from a replayed graph whose inputs change between the replays."""
    z, v = inputs(3, 2000, 64, torch.float32)
    begin = torch.tensor([0, 7, 2000], dtype=torch.int32).cuda()
    d_y = torch.randn(3, 1000, 64, device="cuda")

    def both():
        y, h, saved = ops.gated_scan_fwd(z, v, begin=begin, period=2, train=True)
        return (y, h) + ops.gated_scan_bwd(z, v, saved, d_y, begin=begin, period=2)

    want = both()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = both()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for k in range(3):
        z.copy_(inputs(3, 2000, 64, torch.float32, seed=20 + k)[0])
        want = both()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, held)), k


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Rows whose element offsets pass 2^32: a time-major view with a huge batch stride into one allocation."""
    T, Cc = 300, 64
    far = (1 << 32) + 128
    store = torch.empty(far + T * Cc, device="cuda", dtype=torch.bfloat16)
    near, behind = store[:T * Cc].reshape(T, Cc), store[far:].reshape(T, Cc)
    z, v = inputs(1, T, Cc, torch.bfloat16)
    near.copy_(z[0])
    behind.copy_(z[0])
    both = torch.as_strided(store, (2, T, Cc), (far, Cc, 1))
    y, h, _ = ops.gated_scan_fwd(both, v.expand(2, T, Cc))
    assert torch.equal(y[0], y[1]) and torch.equal(h[0], h[1])
    assert torch.equal(y[0], ops.gated_scan_fwd(z, v)[0][0])


# ------------------------------------------------------------------------------------------------------------- one event
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("B,Cc", [(1, 64), (7, 1), (33, 37), (4096, 20), (5, 512)])
def test_step_against_float64(dtype, B, Cc):
    dt = DTYPES[dtype]
    z, v = (t[:, 0] for t in inputs(B, 1, Cc, dt))
    state = torch.randn(B, Cc, generator=torch.Generator().manual_seed(3)).cuda()
    want = oracle(z[:, None], v[:, None], state, None, 1)
    before = state.clone()
    y = ops.gated_scan_step(z, v, state, commit=False)
    assert torch.equal(state, before)
    size = max(1.0, float(np.abs(want["h_last"]).max()))
    close("y", y, want["h_last"], dt, size)
    y2 = ops.gated_scan_step(z, v, state)
    assert torch.equal(y, y2)
    close("state", state, want["h_last"], torch.float32, size)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [torch.int32, torch.int64])
def test_step_orders_events_of_one_user(width):
    """9000 events over 300 users (three calls' worth of rows): every user's events in row order, equal to one-row calls."""
    B, Cc, U = 9000, 40, 300
    z, v = (t[:, 0] for t in inputs(B, 1, Cc, torch.float32, strided=True))
    user = torch.randint(0, U, (B,), generator=torch.Generator().manual_seed(1)).to("cuda", width)
    state = torch.randn(U, 2, Cc, device="cuda")[:, 0]                 # a strided store
    zc, vc, uc = z.double().cpu().numpy(), v.double().cpu().numpy(), user.cpu().numpy()
    h, ys = state.double().cpu().numpy().copy(), np.zeros((B, Cc))
    for b in range(B):
        a = 1 / (1 + np.exp(-zc[b]))
        ys[b] = h[uc[b]] = a * h[uc[b]] + (1 - a) * vc[b]
    y = ops.gated_scan_step(z, v, state, user)
    close("y", y, ys, torch.float32, 4.0)
    close("state", state, h, torch.float32, 4.0)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [torch.int32, torch.int64])
@pytest.mark.parametrize("B", [1, 7, 9, 64, 511, 513, 2047, 2049, 4096])
def test_step_commits_distinct_users_and_a_late_repeat(width, B):
    """Every user once, then the first row's user again in the last row; an unknown user in between (int64: one whose low half
    is a known user's): equal to the uncommitted step of each row, bit for bit."""
    Cc, U = 70, 5000
    z, v = (t[:, 0] for t in inputs(B, 1, Cc, torch.bfloat16))
    user = torch.randperm(U, generator=torch.Generator().manual_seed(B))[:B].to("cuda", width)
    state = torch.randn(U, Cc, generator=torch.Generator().manual_seed(2)).cuda()
    if B > 8:
        user[-1] = user[0]
        user[5] = -1 if width == torch.int32 else (1 << 32) + int(user[6])
    want, alone = state.clone(), ops.gated_scan_step(z, v, state, user, commit=False)
    y = ops.gated_scan_step(z, v, state, user)
    known = [b for b in range(B) if 0 <= int(user[b]) < U]
    n = len(known) - (1 if B > 8 else 0)
    assert torch.equal(y[known[:n]], alone[known[:n]])
    if B > 8:
        assert torch.isnan(y[5]).all()
        first = ops.gated_scan_step(z[:1].float(), v[:1].float(), want[user[0]][None], commit=False)
        last = ops.gated_scan_step(z[-1:].float(), v[-1:].float(), first, commit=False)
        assert torch.equal(state[user[0]], last[0]) and torch.equal(y[-1], last[0].bfloat16())
    untouched = torch.ones(U, dtype=torch.bool, device="cuda")
    untouched[user[known].long()] = False
    assert torch.equal(state[untouched], want[untouched])


@pytest.mark.gpu
def test_step_reads_only_without_commit_and_skips_unknown_users():
    z, v = (t[:, 0] for t in inputs(6, 1, 16, torch.float32))
    state = torch.randn(3, 16, device="cuda")
    before = state.clone()
    user = torch.tensor([2, 2, 0, -1, 3, 2], device="cuda")
    y = ops.gated_scan_step(z, v, state, user, commit=False)
    assert torch.equal(state, before)
    for b in (0, 1, 2, 5):
        assert torch.equal(y[b], ops.gated_scan_step(z[b:b + 1], v[b:b + 1], state[user[b]:user[b] + 1], commit=False)[0])
    assert torch.isnan(y[3]).all() and torch.isnan(y[4]).all()
    y = ops.gated_scan_step(z, v, state, user)
    assert torch.isnan(y[3:5]).all() and torch.equal(state[1], before[1]) and not torch.equal(state[2], before[2])
    # nothing to do
    assert ops.gated_scan_step(z[:0], v[:0], state, user[:0]).shape == (0, 16)


@pytest.mark.gpu
def test_events_fed_one_by_one_leave_the_scan_state():
    """A store fed event by event holds what the scan over the same events leaves, and its y are the scan's states."""
    z, v = inputs(4, 70, 24, torch.float32)
    y, h_last, _ = ops.gated_scan_fwd(z, v)
    state = torch.zeros(4, 24, device="cuda")
    for t in range(70):
        yt = ops.gated_scan_step(z[:, t], v[:, t], state)
        assert (yt - y[:, t]).abs().max() < 2e-6       # two orders of the same fp32 sums, |state| <= 1
    assert (state - h_last).abs().max() < 2e-6


# ------------------------------------------------------------------------------------------------------ padding, long memory
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("B,T,Cc", [(4, 261, 48), (2, 1500, 37), (3, 40, 2)])
def test_padded_steps_have_zero_gradients_whatever_arrives(B, T, Cc, dtype):
    """d_z and d_v of the steps in front of `begin` are zeros also where d_y there, or the carried state, is infinite or NaN; the
    steps behind do not notice."""
    z, v = inputs(B, T, Cc, DTYPES[dtype])
    begin = torch.tensor([T, T // 2, 0, 130][:B], dtype=torch.int32).clamp(max=T).cuda()
    h0 = torch.randn(B, Cc, generator=torch.Generator().manual_seed(3)).cuda()
    d_y = torch.randn(B, T, Cc, generator=torch.Generator().manual_seed(4)).to("cuda", DTYPES[dtype])
    padded = torch.arange(T, device="cuda")[None] < begin[:, None]
    _, _, saved = ops.gated_scan_fwd(z, v, h0=h0, begin=begin, train=True)
    want = ops.gated_scan_bwd(z, v, saved, d_y, begin=begin)
    for bad in (float("nan"), float("inf"), -float("inf")):
        got = ops.gated_scan_bwd(z, v, saved, torch.where(padded[..., None], bad, d_y.float()).to(d_y.dtype), begin=begin)
        for g, w in zip(got[:2], want[:2]):
            assert not g[padded].any() and torch.equal(g, w), bad
        _, h, s = ops.gated_scan_fwd(z, v, h0=torch.full_like(h0, bad), begin=begin, train=True)
        assert not torch.isfinite(h[0]).any()                          # nothing but padding: the state as it came
        got = ops.gated_scan_bwd(z, v, s, d_y, begin=begin)
        assert not got[0][padded].any() and not got[1][padded].any(), bad


@pytest.mark.gpu
@pytest.mark.parametrize("z0", [6.0, 8.0, 10.0, 12.0])
@pytest.mark.parametrize("B,Cc", [(90, 64), (2, 64), (3, 20), (3, 10), (130, 9)])
def test_long_memory(B, Cc, z0):
    """Gates held near 1: a state remembers e^z steps, and 1 - a is a few parts in 10^5, which a rounded to fp32 near 1 (2^-25) carries
    only to a few digits.  The decay over a wave's 16 or more steps is known to one rounding (2^-25), and the state is rounded once
    (2^-24) when it is taken over them; per 16 steps of memory that adds up to 1.5 2^-24 of the state, over min(T, e^z) steps.  All
    else (gates, the sums of a wave, the replay of four steps) is the constant of close(), 2e-5."""
    T = 8192
    g = torch.Generator().manual_seed(int(z0))
    z = (z0 + 0.25 * torch.rand(B, 1, Cc, generator=g)).expand(B, T, Cc).contiguous().cuda()
    v = (0.5 + 0.5 * torch.rand(B, T, Cc, generator=g)).cuda()         # (one sign: what is lost shows in the mean)
    h0 = torch.rand(B, Cc, generator=g).cuda()
    d_y = (0.5 + 0.5 * torch.rand(B, T // 64, Cc, generator=g)).cuda()
    d_h = torch.rand(B, Cc, generator=g).cuda()
    y, h_last, saved = ops.gated_scan_fwd(z, v, h0=h0, period=64, train=True)
    d_z, d_v, d_h0 = ops.gated_scan_bwd(z, v, saved, d_y, d_h_last=d_h, period=64)
    want = oracle(z, v, h0, None, 64, d_y, d_h)
    tol = 2e-5 + 1.5 * 2.0 ** -24 * min(T, np.exp(z0 + 0.25)) / 16
    for name, got in (("y", y), ("h_last", h_last)):
        off = np.abs(got.double().cpu().numpy() - want[name]).max()
        assert off <= tol, "%s: off by %.3g, %.3g allowed" % (name, off, tol)          # (|h|, |v| <= 1)
    u = 1 / (1 + np.exp(z.double().cpu().numpy()))
    G = want["d_v"] / u
    size = np.abs(G).max()
    for name, got, per in (("d_v", d_v, u), ("d_z", d_z, 2 * u * (1 - u)), ("d_h0", d_h0, 1.0)):
        off = (np.abs(got.double().cpu().numpy() - want[name]) / per).max() / size
        assert off <= tol, "%s: off by %.3g, %.3g allowed" % (name, off, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("z0", [4.0, 8.0, 10.0])
@pytest.mark.parametrize("commit_list", [False, True])
def test_events_of_a_long_memory(z0, commit_list):
    """20000 events into stored states whose gates are held near 1, with and without a user list.  Every event rounds the state once,
    by up to 2^-25 (states in [1/2, 1)), independently: the increments u (v - h) are many such steps.  Over the 1 / (2 u) events whose
    squares add up that is 2^-25 sqrt(1 / 3) sqrt(1 / (2 u)); eight times that for the largest of 256 states, and the gate's own 2e-6
    (|z| 2^-24 and a few roundings, relative to u)."""
    U, Cc, T = 4, 64, 20000
    g = torch.Generator().manual_seed(int(z0))
    z = (z0 + 0.25 * torch.rand(U, Cc, generator=g)).cuda()
    v = (0.5 + 0.5 * torch.rand(T, U, Cc, generator=g)).cuda()
    state = (0.5 + 0.5 * torch.rand(U, Cc, generator=g)).cuda()
    h = state.double().cpu().numpy()
    user = torch.tensor([2, 0, 3, 1], dtype=torch.int32).cuda()
    zd, vd = z.double().cpu().numpy(), v.double().cpu().numpy()
    order = np.argsort(user.cpu().numpy())                             # row of every user
    a, u = 1 / (1 + np.exp(-zd)), 1 / (1 + np.exp(zd))
    for t in range(T):
        ops.gated_scan_step(z, v[t], state, user if commit_list else None)
        h = a[order] * h + u[order] * vd[t][order] if commit_list else a * h + u * vd[t]
    off = np.abs(state.double().cpu().numpy() - h).max()
    tol = 8 * 2.0 ** -25 * np.sqrt(1 / 3) * np.sqrt(1 / (2 * u.min())) + 2e-6
    assert off <= tol, "off by %.3g, %.3g allowed" % (off, tol)


@pytest.mark.gpu
def test_step_on_infinite_states():
    """An infinite state stays what the formula makes of it: infinite while a counts, also where 1 - a is zero."""
    z = torch.tensor([[3.0, float("inf"), 200.0, 0.5, -2.0]]).cuda()
    v = torch.ones(1, 5, device="cuda")
    for bad in (float("inf"), -float("inf")):
        state = torch.full((1, 5), bad, device="cuda")
        y = ops.gated_scan_step(z, v, state)
        assert (y == bad).all() and (state == bad).all()


# ---------------------------------------------------------------------------------------------------------- overlapping memory
def _apart(cls):
    """Descriptors whose operands all lie apart, 1 MiB each."""
    a = cls()
    a.B, a.C, a.dtype = 2, 16, _lib.HPMN_BF16
    for i, f in enumerate(f for f, t in cls._fields_ if t is C.c_void_p):
        setattr(a, f, (i + 1) << 20)
    for f, t in cls._fields_:
        if f.endswith("_st") or f in ("z_s", "v_s", "y_s"):
            setattr(a, f, 16)
        elif f.endswith("_sb"):
            setattr(a, f, 16 * 8 if f != "h0_sb" else 16)
    return a


@pytest.mark.parametrize("field,at", [("y", "z"), ("y", "v"), ("h_last", "h0"), ("saved", "z"), ("y", "begin"), ("y", "h_last"), ("saved", "y")])
def test_forward_outputs_have_memory_of_their_own(lib, field, at):
    a = _apart(_lib.HpmnGatedScan)
    a.T, a.period = 8, 1
    setattr(a, field, getattr(a, at))
    assert lib.hpmn_gated_scan_fwd(C.byref(a), None) == -1


@pytest.mark.parametrize("field,at,by", [("d_z", "z", 0), ("d_z", "v", 0), ("d_v", "z", 16), ("d_v", "d_y", 0), ("d_z", "saved", 64), ("d_v", "d_h_last", 0),
                                         ("d_z", "d_v", 0), ("d_z", "d_v", 16), ("d_v", "d_z", 2 * (2 * 8 * 16) - 2), ("d_h0", "d_h_last", 0), ("d_v", "begin", 0)])
def test_gradients_have_memory_of_their_own(lib, field, at, by):
    a = _apart(_lib.HpmnGatedScanBwd)
    a.T, a.period = 8, 1
    setattr(a, field, getattr(a, at) + by)
    assert lib.hpmn_gated_scan_bwd(C.byref(a), None) == -1


@pytest.mark.parametrize("flags", [_lib.HPMN_STEP_COMMIT, 0])
@pytest.mark.parametrize("field,at,by", [("y", "state", 0), ("y", "user", 0), ("y", "z", 2), ("v", "state", 64), ("z", "state", 0), ("user", "state", 4)])
def test_a_store_has_memory_of_its_own(lib, field, at, by, flags):
    a = _apart(_lib.HpmnGatedStep)
    a.flags, a.n_users, a.state_s = flags, 9, 16
    if not flags and field in ("z", "v", "user"):
        pytest.skip("a store that is only read may be read twice")
    setattr(a, field, getattr(a, at) + by)
    assert lib.hpmn_gated_scan_step(C.byref(a), None) == -1


@pytest.mark.gpu
def test_wrappers_refuse_overlapping_buffers():
    B, T, Cc = 2, 300, 12
    z, v = inputs(B, T, Cc, torch.float32)
    d_y = torch.randn(B, T, Cc, device="cuda")
    _, _, saved = ops.gated_scan_fwd(z, v, train=True)
    want = ops.gated_scan_bwd(z, v, saved, d_y)
    wide = torch.empty(B, T, 3 * Cc, device="cuda")
    long = torch.empty(B, 2 * T, Cc, device="cuda")
    new = lambda: torch.empty_like(z)  # noqa: E731
    for out in ((z, v), (new(), d_y), (d_y, new()), (z, new()), (wide[..., :Cc], wide[..., 1:Cc + 1]), (wide[..., :Cc], wide[..., Cc - 1:2 * Cc - 1]),
                (long[:, :T], long[:, 1:T + 1]), (long[:, :T], long[:, T - 1:-1]), (new(), saved.new_empty(0))):
        with pytest.raises(ValueError):
            ops.gated_scan_bwd(z, v, saved, d_y, out=out)
    # different columns of common rows, the first and the last steps of one buffer, other sequences of it
    both = torch.empty(2 * B, T, Cc, device="cuda")
    for out in ((wide[..., :Cc], wide[..., Cc:2 * Cc]), (wide[..., 2 * Cc:], wide[..., 1:Cc + 1]), (long[:, :T], long[:, T:]), (long[:, T:], long[:, :T]),
                (both[:B], both[B:]), (both[0::2], both[1::2])):
        got = ops.gated_scan_bwd(z, v, saved, d_y, out=out)
        assert all(torch.equal(g, w) for g, w in zip(got, want)) and got[0] is out[0] and got[1] is out[1]
    # inputs and gradients side by side in one buffer
    row = torch.empty(B, T, 5 * Cc, device="cuda")
    for i, t in enumerate((z, v, d_y)):
        row[..., i * Cc:(i + 1) * Cc] = t
    z2, v2, d2, o1, o2 = (row[..., i * Cc:(i + 1) * Cc] for i in range(5))
    assert all(torch.equal(g, w) for g, w in zip(ops.gated_scan_bwd(z2, v2, saved, d2, out=(o1, o2)), want))
    store, user = torch.randn(9, 2 * Cc, device="cuda"), torch.tensor([3, 4], device="cuda")
    for call in (lambda: ops.gated_scan_step(store[:2, :Cc], z[:, 0], store[:, :Cc], user), lambda: ops.gated_scan_step(z[:, 0], store[5:7, 1:Cc + 1], store[:, :Cc], user)):
        with pytest.raises(ValueError):
            call()
    before = store.clone()
    y = ops.gated_scan_step(z[:, 0], store[:2, Cc:], store[:, :Cc], user)              # the other half of the store's rows
    assert torch.equal(y, ops.gated_scan_step(z[:, 0], before[:2, Cc:].clone(), before[:, :Cc].clone(), user))
    ops.gated_scan_step(store[:2, :Cc], z[:, 0], store[:, :Cc], user, commit=False)    # only read


@pytest.mark.gpu
@pytest.mark.parametrize("B,y_s", [(5, 40), (1, 24), (1, 40)])
@pytest.mark.parametrize("over", ["z", "v"])
def test_step_in_place_through_the_c_abi(lib, B, y_s, over):
    """y over z's or v's own rows: the same stride, or a single row, whatever its stride is said to be."""
    Cc = 24
    x = {n: torch.randn(B, 40, generator=torch.Generator().manual_seed(i)).cuda() for i, n in enumerate("zv")}
    state = torch.randn(B, Cc, device="cuda")
    want_state = state.clone()
    want = ops.gated_scan_step(x["z"][:, :Cc].clone(), x["v"][:, :Cc].clone(), want_state)
    a = _lib.HpmnGatedStep()
    a.B, a.C, a.dtype, a.flags, a.n_users, a.state_s, a.z_s, a.v_s, a.y_s = B, Cc, _lib.HPMN_F32, _lib.HPMN_STEP_COMMIT, B, Cc, 40, 40, y_s
    a.z, a.v, a.y, a.state = x["z"].data_ptr(), x["v"].data_ptr(), x[over].data_ptr(), state.data_ptr()
    _lib.check(lib.hpmn_gated_scan_step(C.byref(a), torch.cuda.current_stream().cuda_stream), "hpmn_gated_scan_step")
    assert torch.equal(x[over][:, :Cc], want) and torch.equal(state, want_state)
