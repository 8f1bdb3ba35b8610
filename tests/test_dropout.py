"""Dropout from a counter-based generator (hpmn_dropout): C ABI refusals on the CPU; on the GPU every element against the
definition in numpy's unsigned 64-bit arithmetic."""
import ctypes as C
import math
import os
import subprocess

import numpy as np
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
    a = _lib.HpmnDropout()
    a.N, a.C, a.dtype, a.keep_prob, a.x, a.y, a.x_s, a.y_s = 4, 8, _lib.HPMN_BF16, 0.5, 4096, 4096, 8, 8
    return a


@pytest.mark.parametrize("field,value,rc", [("N", -1, -1), ("C", -1, -1), ("dtype", 3, -1), ("keep_prob", 0.0, -1), ("keep_prob", -0.5, -1),
                                            ("keep_prob", 1.5, -1), ("keep_prob", float("nan"), -1), ("x", None, -1), ("y", None, -1),
                                            ("x", 4097, -1), ("rng", 4100, -1), ("y_s", 7, -1), ("x_s", -8, -1), ("N", 1 << 40, -2),
                                            ("N", 0, 0), ("C", 0, 0)])
def test_refusals(lib, field, value, rc):
    a = _args()
    setattr(a, field, value)
    assert lib.hpmn_dropout(C.byref(a), None) == rc
    assert lib.hpmn_dropout(None, None) == -1


@pytest.mark.parametrize("N,Cc", [(1 << 28, 64), (1 << 34, 1), (1, 1 << 34), (1 << 62, 3)])
def test_more_threads_than_a_launch_has_are_refused(lib, N, Cc):
    a = _args()
    a.N, a.C, a.y_s, a.x_s = N, Cc, Cc, Cc
    assert lib.hpmn_dropout(C.byref(a), None) == -2


def test_struct_layout(tmp_path):
    st = _lib.HpmnDropout
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "hpmn_hip.h"', 'int main(void){printf("%zu", sizeof(HpmnDropout));']
    lines += ['printf(" %%zu", offsetof(HpmnDropout, %s));' % f for f, _ in st._fields_] + ["return 0;}"]
    src = tmp_path / "l.c"
    src.write_text("\n".join(lines))
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "l")])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / "l")], text=True).split()]
    assert got == [C.sizeof(st)] + [getattr(st, f).offset for f, _ in st._fields_]


def test_wrapper_refuses_host_tensors():
    with pytest.raises(ValueError):
        ops.dropout_fwd(torch.zeros(4, 4), 0.5, 1)


def _mix(x):
    x = (x ^ (x >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
    x = (x ^ (x >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
    return x ^ (x >> np.uint64(31))


def oracle_mask(n, keep_prob, seed, offset):
    """0 or 65536 / thr per element, float64."""
    with np.errstate(over="ignore"):
        k = np.arange((n + 3) // 4, dtype=np.uint64) + np.uint64((offset + 1) & 0xFFFFFFFFFFFFFFFF)
        w = _mix(_mix(np.array([seed & 0xFFFFFFFFFFFFFFFF], np.uint64)) + k * np.uint64(0x9E3779B97F4A7C15))
    thr = min(65536, max(1, math.floor(float(np.float32(keep_prob)) * 65536 + 0.5)))
    field = np.stack([(w >> np.uint64(16 * j)) & np.uint64(0xFFFF) for j in range(4)], 1).reshape(-1)[:n]
    return np.where(field < thr, 65536.0 / thr, 0.0)


def test_oracle_words_are_the_published_generator():
    """splitmix64 from state 0 (published reference outputs): the words of offset 0 under a mixed seed of 0."""
    with np.errstate(over="ignore"):
        w = _mix(np.arange(1, 4, dtype=np.uint64) * np.uint64(0x9E3779B97F4A7C15))
    assert [int(x) for x in w] == [0xE220A8397B1DCDAF, 0x6E789E6AA1B965F4, 0x06C45D188009454F]


def test_oracle_mask_is_evenly_spread():
    """Kept fraction within 5 standard deviations, also along each of the four fields and for neighbouring seeds and offsets; the
    masks of neighbouring seeds agree as often as independent ones do."""
    n, p = 1 << 18, 0.9
    masks = [oracle_mask(n, p, s, o) > 0 for s, o in ((1, 0), (2, 0), (3, 1 << 20), (1, n // 4))]
    for m in masks:
        for part in (m, m[0::4], m[1::4], m[2::4], m[3::4]):
            assert abs(part.mean() - p) < 5 * math.sqrt(p * (1 - p) / part.size)
    same = p * p + (1 - p) * (1 - p)
    for m in masks[1:]:
        assert abs((m == masks[0]).mean() - same) < 5 * math.sqrt(same * (1 - same) / n)


def check(x, keep, seed, offset=0, residual=None, rng=None, real=None):
    s, o = real if real else (seed, offset)
    y = ops.dropout_fwd(x, keep, seed, offset=offset, residual=residual, rng=rng)
    assert y.shape == x.shape and y.dtype == x.dtype
    m = oracle_mask(x.numel(), keep, s, o)
    # zero where dropped, whatever x holds there
    x64 = x.double().cpu().numpy().reshape(-1)
    want = np.where(m > 0, x64 * np.where(m > 0, m, 1), 0.0)
    # roundings: the scale and the product in fp32 (2 x 2^-24), the sum (2^-24), the storage type (half a step)
    tol = 3 * 2.0 ** -24 * np.abs(want) + 1e-45
    if residual is not None:
        r = residual.double().cpu().numpy().reshape(-1)
        tol = tol + 2.0 ** -24 * np.abs(want + r)
        want = want + r
    if x.dtype != torch.float32:
        tol = tol + torch.finfo(x.dtype).eps / 2 * np.abs(want) * 1.001 + (3e-8 if x.dtype == torch.float16 else 0)
    got = y.double().cpu().numpy().reshape(-1)
    assert (np.abs(got - want) <= tol).all()
    if residual is None:
        assert ((got == 0) == ((m == 0) | (x64 == 0))).all()
        assert torch.equal(ops.dropout_bwd(x, keep, seed, offset=offset, rng=rng), y)
    return y


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("shape", [(1,), (3,), (8,), (4097,), (1, 7), (128, 200), (33, 37), (5, 3, 24), (129, 1024), (2, 1), (1000, 6)])
def test_against_the_definition(shape, dtype):
    g = torch.Generator().manual_seed(len(shape) + shape[-1])
    x = torch.randn(*shape, generator=g).to("cuda", DTYPES[dtype])
    r = torch.randn(*shape, generator=g).to("cuda", DTYPES[dtype])
    check(x, 0.5, 12345)
    check(x, 0.9, -7, offset=(1 << 40) + 3, residual=r)
    check(x, 0.3, (1 << 64) - 1, offset=(1 << 64) - 2)                 # counters that wrap


@pytest.mark.gpu
def test_keep_probabilities():
    x = torch.randn(64, 96, device="cuda")
    assert torch.equal(ops.dropout_fwd(x, 1.0, 5), x)
    check(x, 1e-9, 5)                                                  # one 65536th is the least
    check(x, 1 - 2.0 ** -17, 5)
    check(x, 2.0 ** -16 * 1.5, 5)
    for bad in (0.0, -1.0, 1.0001, float("nan")):
        with pytest.raises(ValueError):
            ops.dropout_fwd(x, bad, 5)


@pytest.mark.gpu
def test_dropped_elements_hide_what_they_hold():
    x = torch.randn(512, device="cuda").bfloat16()
    y = ops.dropout_fwd(x, 0.5, 3)
    x2 = torch.where(y == 0, torch.full_like(x, float("nan")), x)
    assert torch.equal(ops.dropout_fwd(x2, 0.5, 3), y)
    x2 = torch.where(y == 0, torch.full_like(x, float("inf")), x)
    assert torch.equal(ops.dropout_fwd(x2, 0.5, 3), y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_strides_and_alignment(dtype):
    """Column halves, broadcast rows, permuted tensors, odd storage offsets: the mask goes by the logical index alone."""
    dt = DTYPES[dtype]
    wide = torch.randn(40, 128, device="cuda").to(dt)
    for x in (wide[:, :64], wide[:, 64:], wide[:, 1:65], wide[::2], wide[:1].expand(7, 128), wide.t(), wide[:, :37],
              wide.reshape(4, 10, 128).transpose(0, 1), wide.reshape(-1)[1:4001], wide[:, 5:6]):
        want = ops.dropout_fwd(x.contiguous(), 0.8, 9, offset=2)
        if x.stride(-1) == 1 or x.dim() == 1 or x.shape[-1] == 1:
            r = torch.randn(x.shape, device="cuda").to(dt)
            assert torch.equal(ops.dropout_fwd(x, 0.8, 9, offset=2, residual=r), check(x.contiguous(), 0.8, 9, 2, residual=r))
        assert torch.equal(ops.dropout_fwd(x, 0.8, 9, offset=2), want)
    with pytest.raises(ValueError):
        ops.dropout_fwd(wide, 0.5, 1, residual=wide[:, :64])
    with pytest.raises(ValueError):
        ops.dropout_fwd(wide, 0.5, 1, residual=wide.double())
    with pytest.raises(ValueError):
        ops.dropout_fwd(wide, 0.5, 1, rng=torch.zeros(2, device="cuda"))
    with pytest.raises(ValueError):
        ops.dropout_fwd(torch.zeros((), device="cuda"), 0.5, 1)
    assert ops.dropout_fwd(wide[:0], 0.5, 1).shape == (0, 128) and ops.dropout_fwd(wide[:, :0], 0.5, 1).shape == (40, 0)


@pytest.mark.gpu
def test_in_place_through_the_c_abi(lib):
    x = torch.randn(100, 48, device="cuda")
    want = ops.dropout_fwd(x, 0.5, 77, residual=x)
    a = _lib.HpmnDropout()
    a.N, a.C, a.dtype, a.keep_prob, a.x_s, a.r_s, a.y_s, a.seed = 100, 48, _lib.HPMN_F32, 0.5, 48, 48, 48, 77
    a.x = a.y = a.residual = x.data_ptr()
    _lib.check(lib.hpmn_dropout(C.byref(a), torch.cuda.current_stream().cuda_stream), "hpmn_dropout")
    assert torch.equal(x, want)


@pytest.mark.gpu
def test_captured_graph_draws_anew():
    """A graph reads seed and offset when it runs: the mask follows the tensor between replays; eager calls agree."""
    x = torch.randn(64, 200, device="cuda")
    rng = torch.tensor([42, 0], device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.dropout_fwd(x, 0.5, 0, offset=10, rng=rng)
        d = ops.dropout_bwd(x, 0.5, 0, offset=10, rng=rng)
    seen = []
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, check(x, 0.5, 42, 10 + 3200 * k)) and torch.equal(d, y)
        assert torch.equal(y, check(x, 0.5, 0, 10, rng=rng, real=(42, 10 + 3200 * k)))
        seen.append(y.clone())
        rng[1] += 3200
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


@pytest.mark.gpu
def test_more_than_32_bits_of_elements():
    """Element indices past 2^32: the last rows of a 4.3 G-element tensor against the definition at their own counters."""
    C_ = 1 << 16
    N = (1 << 16) + 8
    x = torch.ones(N, C_, device="cuda", dtype=torch.bfloat16)
    y = ops.dropout_fwd(x, 0.5, 4)
    for row in (0, 1 << 15, N - 1):
        m = oracle_mask(C_, 0.5, 4, row * C_ // 4)
        assert (y[row].double().cpu().numpy() == m).all()


@pytest.mark.parametrize("x,x_s,r,r_s,y,y_s,rng", [(4096, 8, None, 0, 4096, 16, None), (4096, 16, None, 0, 4096, 8, None), (4096, 8, None, 0, 4098, 8, None),
                                                   (4096, 0, None, 0, 4096, 8, None), (4096, 8, 8192, 16, 8192, 8, None), (4096, 8, 8192, 8, 8192 + 46, 8, None),
                                                   (4096, 8, None, 0, 8192, 8, 8192 + 24)])
def test_in_place_is_the_same_rows_or_refused(lib, x, x_s, r, r_s, y, y_s, rng):
    """A row that a thread writes must be no row that another one has yet to read."""
    a = _args()
    a.x, a.x_s, a.residual, a.r_s, a.y, a.y_s, a.rng = x, x_s, r, r_s, y, y_s, rng
    assert lib.hpmn_dropout(C.byref(a), None) == -1


@pytest.mark.gpu
def test_in_place_over_strided_rows_and_beside_other_columns(lib):
    for cols in (slice(0, 48), slice(48, 96)):
        buf = torch.randn(100, 96, device="cuda")
        other = buf[:, :48] if cols.start else buf[:, 48:]
        x, kept = buf[:, cols], other.clone()
        want, beside = ops.dropout_fwd(x, 0.5, 77), ops.dropout_fwd(x, 0.5, 78)
        a = _lib.HpmnDropout()
        a.N, a.C, a.dtype, a.keep_prob, a.x_s, a.y_s = 100, 48, _lib.HPMN_F32, 0.5, 96, 96
        a.x = x.data_ptr()
        for seed, y in ((78, other), (77, x)):
            a.seed, a.y = seed, y.data_ptr()
            _lib.check(lib.hpmn_dropout(C.byref(a), torch.cuda.current_stream().cuda_stream), "hpmn_dropout")
            if seed == 78:
                assert torch.equal(other, beside)
                other.copy_(kept)
        assert torch.equal(x, want) and torch.equal(other, kept)
