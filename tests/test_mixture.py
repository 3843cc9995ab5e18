"""Operators around gated mixtures of kernels (spnc.mixture, include/spnc_hip_rows.h) against their 64-bit definitions."""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest

from conftest import ROOT, compile_spn, oracle_model, quiet
from oracle import mixture as om

HALF = {"float32": 2.0 ** -24, "float64": 2.0 ** -53, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}   # half a step, relative


def _torch():
    import torch
    return torch


def _host(t):
    t = t.detach().cpu()
    return t.double().numpy() if t.is_floating_point() else t.numpy()


def _near(got, want, allowed, what=""):
    """|got - want| <= allowed, the same infinities and NaN."""
    got, want = _host(got), np.asarray(want, dtype=np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    finite = np.isfinite(want)
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)]) and np.isfinite(got[finite]).all(), what
    over = (np.abs(np.where(finite, got, 0.0) - np.where(finite, want, 0.0)) - allowed)[finite]
    assert over.size == 0 or over.max() <= 0, (what, float(over.max()))


# ---- without a GPU --------------------------------------------------------------------------------------------------

def test_header_and_library_agree(native):
    header = open(os.path.join(ROOT, "include", "spnc_hip_rows.h")).read()
    declared = re.findall(r"SPNC_HIP_API[^;(]*?\b(spnc_hip_\w+)\s*\(", header)
    assert len(declared) == 10
    lib = ctypes.CDLL(native.library_path())
    for name in declared:
        assert hasattr(lib, name) and getattr(native._load(), name).argtypes, name


def test_header_is_c(tmp_path):
    src = tmp_path / "c.c"
    src.write_text('#include "spnc_hip_rows.h"\nint main(void){return SPNC_HIP_BFLOAT16 - 3;}\n')
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), "-c", str(src), "-o", str(tmp_path / "c.o")], check=True)


# Known answers of Philox4x32-10: counter and key all zeros, all ones.
PHILOX = [((0, 0, 0), [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]),
          ((2 ** 64 - 1, 2 ** 64 - 1, 2 ** 64 - 1), [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD])]


def test_philox_known_answers(tmp_path):
    src = tmp_path / "p.cpp"
    src.write_text('#include <cstdio>\n#include <cstdlib>\n#include "philox.h"\nint main(int, char** a){ unsigned long long v[3];'
                   'for (int i = 0; i < 3; ++i) v[i] = strtoull(a[i + 1], nullptr, 10);'
                   'auto r = spnc_hip::philox4x32(v[0], v[0] >> 32, v[1], v[1] >> 32, v[2], v[2] >> 32);'
                   'printf("%u %u %u %u", r.w[0], r.w[1], r.w[2], r.w[3]); }\n')
    exe = str(tmp_path / "p")
    subprocess.run(["g++", "-std=c++17", "-Wno-unknown-pragmas", "-I", os.path.join(ROOT, "spn-compiler_amd", "csrc"), str(src), "-o", exe], check=True)
    for (block, offset, seed), want in PHILOX + [((b, o, s), None) for b, o, s in [(5, 0, 1), (2 ** 33 + 7, 9, 2 ** 40 + 3), (1, 2 ** 63, 11)]]:
        got = list(map(int, subprocess.run([exe, str(block), str(offset), str(seed)], capture_output=True, text=True, check=True).stdout.split()))
        assert om.philox(block, offset, seed) == got
        assert want is None or got == want


def test_refusals_before_the_gpu():
    torch = _torch()
    from spnc import mixture as m
    z, i32 = torch.zeros, torch.int32

    def plan(n=2, k=2, experts=3, capacity=4):
        return m.Plan(z(n, k, dtype=i32), z(experts + 1, dtype=i32), z(experts, dtype=i32), capacity)

    cases = [
        (lambda: m.gate(z(3), 1), "shape"), (lambda: m.gate(z(2, 3), 0), "k must be"), (lambda: m.gate(z(2, 3), 4), "k must be"),
        (lambda: m.gate(z(2, 1025), 2), "number of experts"), (lambda: m.gate(z(2, 0), 1), "number of experts"), (lambda: m.gate(z(2, 100), 65), "k must be"),
        (lambda: m.gate(z(2, 3, dtype=i32), 1), "must be float32"), (lambda: m.gate(z(2, 3), 1, over="most"), "over must be"),
        (lambda: m.gate(z(2, 3), 1), "on a GPU"),
        (lambda: m.route(z(2, 2), 3), "int32"), (lambda: m.route(z(4, dtype=i32), 3), "int32"), (lambda: m.route(z(2, 0, dtype=i32), 3), "int32"),
        (lambda: m.route(z(2, 2, dtype=i32), 0), "number of experts"), (lambda: m.route(z(2, 2, dtype=i32), 1025), "number of experts"),
        (lambda: m.route(z(2, 2, dtype=i32), 3, align=0), "align"), (lambda: m.route(z(2, 2, dtype=i32), 1000, align=2 ** 22), "2\\^31"),
        (lambda: m.route(z(2, 2, dtype=i32), 3), "on a GPU"),
        (lambda: m.Plan(z(2, 2), z(4, dtype=i32), z(3, dtype=i32), 4), "position"), (lambda: plan(capacity=2 ** 31), "capacity"),
        (lambda: m.Plan(z(2, 2, dtype=i32), z(3, dtype=i32), z(3, dtype=i32), 4), "one entry more"),
        (lambda: m.dispatch(z(3), plan()), "shape"), (lambda: m.dispatch(z(3, 2), plan()), "for 2 rows"),
        (lambda: m.dispatch(z(2, 2, dtype=torch.complex64), plan()), "not supported"),
        (lambda: m.dispatch(z(2, 2), plan(), out=z(3, 2)), "out must be"), (lambda: m.dispatch(z(2, 2), plan(), out=z(4, 2, dtype=i32)), "out must be"),
        (lambda: m.dispatch(z(2, 2, requires_grad=True), plan(), out=z(4, 2)), "no gradient"), (lambda: m.dispatch(z(2, 2), plan()), "on a GPU"),
        (lambda: m.combine(z(3, 2), plan()), "shape"), (lambda: m.combine(z(4, 2, dtype=i32), plan()), "must be float32"),
        (lambda: m.combine(z(4, 2), plan(), z(2, 3)), "Weights must have shape"), (lambda: m.combine(z(4, 2), plan(), z(2, 2, dtype=torch.float64)), "Weights must be"),
        (lambda: m.combine(z(4, 2), plan(), z(2, 2)), "on a GPU"),
        (lambda: m.combine_log(z(4, 2), plan(), z(2, 2)), "shape"), (lambda: m.combine_log(z(4, dtype=torch.float16), plan(), z(2, 2)), "float32 or float64"),
        (lambda: m.combine_log(z(4), plan(), z(2, 2, dtype=torch.bfloat16)), "Weights must be"), (lambda: m.combine_log(z(4), plan(), z(2, 2)), "on a GPU"),
        (lambda: m.dropout(z(4, dtype=i32), 0.5, 1), "must be float32"), (lambda: m.dropout(z(4), 1.5, 1), "p must be"),
        (lambda: m.dropout(z(4), float("nan"), 1), "p must be"), (lambda: m.dropout(z(4), 0.5, -1), "seed"), (lambda: m.dropout(z(4), 0.5, 2 ** 64), "seed"),
        (lambda: m.dropout(z(4), 0.5, 1, offset=-1), "offset"), (lambda: m.dropout(z(4), 0.5, 1, offset=z(1)), "int64"), (lambda: m.dropout(z(4), 0.5, 1), "on a GPU"),
    ]
    for fn, message in cases:
        with pytest.raises(RuntimeError, match=message):
            fn()


def test_c_entry_points_refuse(native):
    """Every refusal happens before anything reaches the GPU: these run where there is none."""
    lib, big = native._load(), 1 << 31
    p = ctypes.c_void_p(16)   # never read: the calls are refused first

    def refused(rc, message):
        assert rc != 0 and message in lib.spnc_hip_last_error().decode(), lib.spnc_hip_last_error()

    refused(lib.spnc_hip_gate(p, 7, 2, 3, 3, 1, 0, p, p, None), "unknown element type")
    refused(lib.spnc_hip_gate(p, 0, 2, 0, 3, 1, 0, p, p, None), "experts must be")
    refused(lib.spnc_hip_gate(p, 0, 2, 3, 3, 4, 0, p, p, None), "k must be")
    refused(lib.spnc_hip_gate(p, 0, 2, 3, 2, 1, 0, p, p, None), "rows of logits overlap")
    refused(lib.spnc_hip_gate(p, 0, 2, 3, 3, 1, 4, p, p, None), "unknown gate flags")
    refused(lib.spnc_hip_gate(None, 0, 2, 3, 3, 1, 0, p, p, None), "null argument")
    refused(lib.spnc_hip_gate(ctypes.c_void_p(18), 0, 2, 3, 3, 1, 0, p, p, None), "not aligned")
    refused(lib.spnc_hip_gate(p, 0, 2, 3, 1 << 20, 1, 0, p, p, None), "2^20")
    refused(lib.spnc_hip_dropout(ctypes.c_void_p(17), 3, 2, 4, 4, p, 4, 0.5, 0, 0, 0, None, None), "not aligned")
    refused(lib.spnc_hip_route(p, 100000, 3, 1, p, p, p, ctypes.c_void_p(18), 1 << 20, None), "aligned to 4 bytes")
    refused(lib.spnc_hip_gate_backward(None, 0, 2, 3, 3, 1, 1, p, p, p, p, None), "null argument")
    refused(lib.spnc_hip_route(p, 4, 3, 0, p, p, p, None, 0, None), "align")
    refused(lib.spnc_hip_route(p, big, 3, 1, p, p, p, None, 0, None), "too many slots")
    refused(lib.spnc_hip_route(p, 100000, 3, 1, p, p, p, None, 0, None), "the workspace must hold")
    refused(lib.spnc_hip_route(p, 4, 3, 1, p, None, p, None, 0, None), "null argument")
    refused(lib.spnc_hip_dispatch(p, 2, 4, 4, p, 0, 4, None, None, 0, 0, p, None), "k must be")
    refused(lib.spnc_hip_dispatch(p, big, 4, 4, p, 2, 4, None, None, 0, 0, p, None), "too many slots")
    refused(lib.spnc_hip_dispatch(p, 2, 4, 4, p, 2, 4, None, None, 3, 1, p, None), "null argument")
    refused(lib.spnc_hip_dispatch(p, 2, 1 << 31, 1 << 31, p, 2, 4, None, None, 0, 0, p, None), "2 GiB")
    refused(lib.spnc_hip_combine(p, 0, 4, 1 << 62, 1 << 62, p, 2, 2, p, 0, p, None), "2 GiB")
    refused(lib.spnc_hip_combine(p, 0, big, 4, 4, p, 2, 2, p, 0, p, None), "too many rows")
    refused(lib.spnc_hip_combine(p, 0, 4, 4, 4, p, 2, 2, p, 1, p, None), "weights must be float32")
    refused(lib.spnc_hip_combine(ctypes.c_void_p(18), 0, 4, 4, 4, p, 2, 2, p, 0, p, None), "not aligned")
    refused(lib.spnc_hip_combine_backward(p, 0, 4, 4, 4, p, 2, 2, p, 0, p, 4, None, None, 3, p, p, None), "null argument")
    refused(lib.spnc_hip_combine_log(p, 2, 4, p, 2, 2, p, 0, p, p, None), "must be float32 or float64")
    refused(lib.spnc_hip_combine_log(p, 0, 4, p, 2, 2, None, 0, p, p, None), "null argument")
    refused(lib.spnc_hip_combine_log_backward(p, 0, 4, p, 2, 2, 0, p, p, None, 3, p, p, None), "null argument")
    refused(lib.spnc_hip_combine_log_backward(None, 0, 4, p, 2, 2, 0, p, p, p, 3, p, p, None), "null argument")
    refused(lib.spnc_hip_dropout(p, 0, 2, 4, 4, p, 4, 1.5, 0, 0, 0, None, None), "probability")
    refused(lib.spnc_hip_dropout(p, 0, 2, 4, 4, p, 4, float("nan"), 0, 0, 0, None, None), "probability")
    refused(lib.spnc_hip_dropout(p, 0, 2, 4, 3, p, 4, 0.5, 0, 0, 0, None, None), "overlap")
    refused(lib.spnc_hip_dropout(p, 0, 2, 4, 4, p, 4, 0.5, 3, 0, 0, None, None), "unknown dropout mode")
    assert lib.spnc_hip_route_workspace(100000, 0) == 0 and lib.spnc_hip_route_workspace(100000, 70000) == 0
    assert lib.spnc_hip_route_workspace(8192, 10) == 0 and lib.spnc_hip_route_workspace(100000, 10) > 0
    # nothing to do is no error
    assert lib.spnc_hip_gate(None, 0, 0, 3, 3, 1, 0, None, None, None) == 0
    assert lib.spnc_hip_combine(None, 0, 0, 4, 4, None, 0, 2, None, 0, None, None) == 0
    assert lib.spnc_hip_dropout(None, 0, 5, 0, 0, None, 0, 0.5, 0, 0, 0, None, None) == 0


def test_mixture_refuses_kernels_that_do_not_fit_together(native):
    from spnc import synthetic as syn
    from spnc.mixture import Mixture
    a, b = compile_spn(native, syn.c1_spn(), "int32"), compile_spn(native, syn.c2_spn(), "float32")
    try:
        with pytest.raises(RuntimeError, match="agree on the number of features"):
            Mixture([a, b])
        with pytest.raises(RuntimeError, match="number of kernels"):
            Mixture([])
        torch = _torch()
        mix = Mixture([a, a])
        assert (mix.num_features * 4 * mix._align) % a.info()["input_alignment"] == 0
        with pytest.raises(RuntimeError, match="Rows must have shape"):
            mix.log_likelihood(torch.zeros(3, 5, dtype=torch.int32), torch.zeros(3, 2), 1)
        with pytest.raises(RuntimeError, match="Logits must have shape"):
            mix.log_likelihood(torch.zeros(3, 6, dtype=torch.int32), torch.zeros(3, 3), 1)
        with pytest.raises(RuntimeError, match="feature type"):
            mix.log_likelihood(torch.zeros(3, 6), torch.zeros(3, 2), 1)
    finally:
        for k in (a, b):
            os.remove(k.fileName())


# ---- gate -----------------------------------------------------------------------------------------------------------

def _gate_logits(n, experts, dtype, seed, masked=0.2):
    torch = _torch()
    rng = np.random.default_rng(seed)
    z = rng.normal(size=(n, experts)) * 2.0
    z[rng.random(z.shape) < masked] = -np.inf
    if n > 3:
        z[1] = -np.inf                                   # closed altogether
        z[2] = 0.5                                       # all equal
        z[3] = np.finfo(np.float16).min                  # the lowest value of a type, not minus infinity
        z[3, experts // 2] = -1.0
    if n > 4:
        z[4, ::2] = 0.0
        z[4, 1::2] = -0.0                                # equal too
    return torch.tensor(z).to(getattr(torch, dtype))


GATE = [(1, 1, 1), (1, 10, 2), (5, 2, 2), (7, 3, 3), (33, 8, 8), (65, 10, 2), (130, 64, 4), (9, 64, 64), (6, 100, 17), (37, 255, 8), (12, 257, 5),
        (21, 509, 8), (6, 1024, 6), (5, 1000, 64), (513, 17, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float64", "float16", "bfloat16"])
@pytest.mark.parametrize("over,log", [("chosen", True), ("chosen", False), ("all", True), ("all", False)])
def test_gate(native, dtype, over, log):
    """Weights: z - top is rounded once (|z - top| <= 16 in the terms that count), exp within 2 units, a sum of up to 1024
    terms, a quotient or a logarithm: relative (absolute for logarithms) error below (16 + 4 + experts + 4) half steps.
    The lowest value of float16, 65504 below, adds its rounding to a logarithm of that size."""
    torch = _torch()
    from spnc import mixture as m
    u = HALF["float64" if dtype == "float64" else "float32"]
    for n, experts, k in GATE:
        z = _gate_logits(n, experts, dtype, seed=n + experts)
        dev = z.cuda().requires_grad_()
        index, weight = m.gate(dev, k, over=over, log=log)
        want_index, want = om.gate(_host(z), k, over, log)
        assert index.dtype == torch.int32 and np.array_equal(_host(index), want_index), (n, experts, k)
        assert weight.dtype == (torch.float64 if dtype == "float64" else torch.float32)
        bound = (24 + experts) * u * (np.maximum(1.0, np.abs(np.where(np.isfinite(want), want, 0))) if log else np.maximum(np.abs(want), 1e-30))
        _near(weight, want, bound, (n, experts, k))
        grad = torch.randn(n, k, dtype=weight.dtype, generator=torch.Generator().manual_seed(n))
        got, = torch.autograd.grad(weight, dev, grad.cuda())
        want = om.gate_gradient(_host(z), want_index, _host(grad), over, log)
        assert got.dtype == z.dtype
        # a term for each of k slots and their common sum, each with the weights' relative error; then the logits' own type
        scale = np.abs(_host(grad)).sum(axis=1, keepdims=True)
        _near(got, want, (24 + experts + 2 * k) * u * scale + HALF[dtype] * np.abs(want) + (2.0 ** -25 if dtype == "float16" else 0), (n, experts, k))
        assert (_host(got)[~np.isfinite(_host(z))] == 0).all()      # closed experts have no gradient


@pytest.mark.parametrize("over,log", [("chosen", True), ("chosen", False), ("all", True), ("all", False)])
def test_oracles_of_the_gate_agree(over, log):
    z = _gate_logits(40, 12, "float32", seed=2).double().numpy()
    grad = np.random.default_rng(3).normal(size=(40, 5))
    index, weight = om.gate(z, 5, over, log)
    many = om.gate_many(z, 5, over, log, grad)
    assert np.array_equal(index, many[0]) and np.allclose(weight, many[1], rtol=1e-13, atol=1e-13)
    assert np.allclose(om.gate_gradient(z, index, grad, over, log), many[2], rtol=1e-12, atol=1e-13)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float64", "float16", "bfloat16"])
@pytest.mark.parametrize("experts,k", [(3, 2), (10, 2), (33, 1), (64, 4), (67, 4), (96, 20), (130, 8), (256, 4), (509, 8), (511, 3), (512, 6), (1023, 2), (1024, 40)])
def test_gate_of_many_rows(native, dtype, experts, k):
    """From 8192 rows on a row is held by fewer lanes. Tolerances as in test_gate."""
    torch = _torch()
    from spnc import mixture as m
    n, u = 8192 + 61, HALF["float64" if dtype == "float64" else "float32"]
    z = _gate_logits(n, experts, dtype, seed=experts, masked=0.3)
    grad = torch.randn(n, k, dtype=torch.float64 if dtype == "float64" else torch.float32, generator=torch.Generator().manual_seed(n))
    wide = torch.zeros(n, experts + 7, dtype=z.dtype, device="cuda")
    wide[:, 3:experts + 3] = z.cuda()
    for over, log, dev in (("all", True, z.cuda()), ("chosen", False, z.cuda()), ("all", False, wide[:, 3:experts + 3])):
        dev = dev.detach().requires_grad_()
        index, weight = m.gate(dev, k, over=over, log=log)
        got, = torch.autograd.grad(weight, dev, grad.cuda())
        want_index, want, want_grad = om.gate_many(z.double().numpy(), k, over, log, _host(grad))
        assert np.array_equal(_host(index), want_index)
        _near(weight, want, (24 + experts) * u * (np.maximum(1.0, np.abs(np.where(np.isfinite(want), want, 0))) if log else np.maximum(np.abs(want), 1e-30)))
        scale = np.abs(_host(grad)).sum(axis=1, keepdims=True)
        _near(got, want_grad, (24 + experts + 2 * k) * u * scale + HALF[dtype] * np.abs(want_grad) + (2.0 ** -25 if dtype == "float16" else 0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float64", "float16", "bfloat16"])
def test_gate_of_the_types_limits(native, dtype):
    """Masks of the type's lowest value, whole rows of it among them, and its largest: finite logits like others. Weights of 1, 1/2,
    1/7 and 0 within the rounding of one quotient and of exp and a sum of seven, three units each."""
    torch = _torch()
    from spnc import mixture as m
    info = torch.finfo(getattr(torch, dtype))
    z = torch.tensor([[info.min] * 7, [info.min, 0.5, info.min, info.min, 0.5, info.min, info.min], [info.max] + [0.0] * 6, [info.max] * 7,
                      [info.min] * 6 + [-float("inf")], [info.max, info.min] + [-float("inf")] * 5], dtype=torch.float64).to(getattr(torch, dtype))
    u = HALF["float64" if dtype == "float64" else "float32"]
    for repeat in (1, 2000):                          # rows over many lanes and over few
        dev = z.repeat(repeat, 1).cuda().requires_grad_()
        for over in ("chosen", "all"):
            index, weight = m.gate(dev, 2, over=over)
            assert index[:6].tolist() == [[0, 1], [1, 4], [0, 1], [0, 1], [0, 1], [0, 1]]
            half, seventh, sixth = 0.5, 0.5 if over == "chosen" else 1 / 7, 0.5 if over == "chosen" else 1 / 6
            want = np.array([[seventh, seventh], [half, half], [1, 0], [seventh, seventh], [sixth, sixth], [1, 0]])
            _near(weight[-6:], want, 16 * u)
            grad = torch.zeros_like(weight)
            grad[:, 0] = 1.0
            got, = torch.autograd.grad(weight, dev, grad)
            p = np.where(z.double().numpy() == z.double().max(dim=1, keepdim=True).values.numpy(), 1.0, 0.0)
            if over == "chosen":
                p = np.zeros_like(p)
                np.put_along_axis(p, index[:6].cpu().numpy().astype(np.int64), want, axis=1)
            p /= p.sum(axis=1, keepdims=True)
            first = index[:6, 0].cpu().numpy()
            one = np.zeros_like(p)
            one[np.arange(6), first] = 1.0
            _near(got[-6:], p[np.arange(6), first][:, None] * (one - p), 32 * u + 2 * HALF[dtype])
            logs = m.gate(dev, 2, over=over, log=True)[1][-6:]
            _near(logs[[0, 1, 3, 4]], np.log(want[[0, 1, 3, 4]]), 32 * u)


@pytest.mark.gpu
def test_gate_of_nan_and_infinity(native):
    torch = _torch()
    from spnc import mixture as m
    nan, inf = float("nan"), float("inf")
    z = torch.tensor([[1.0, nan, 2.0, nan], [inf, 0.0, 1.0, -inf], [0.0, 1.0, nan, -inf], [-inf, -inf, -inf, 3.0]])
    for dtype in (torch.float32, torch.float64, torch.bfloat16, torch.float16):
        for over in ("chosen", "all"):
            index, weight = m.gate(z.to(dtype).cuda(), 2, over=over)
            assert index.tolist() == [[1, 3], [0, 2], [2, 1], [3, -1]], (dtype, over)
            assert torch.isnan(weight[0]).all() and torch.isnan(weight[2]).all() and weight[3].tolist() == [1.0, 0.0]
            many = m.gate(z.repeat(3000, 1).to(dtype).cuda(), 2, over=over)
            assert torch.equal(many[0], index.repeat(3000, 1)) and torch.equal(many[1].nan_to_num(7.0), weight.repeat(3000, 1).nan_to_num(7.0))


@pytest.mark.gpu
def test_gate_strides_and_empty(native):
    torch = _torch()
    from spnc import mixture as m
    base = torch.randn(40, 24, device="cuda")
    for view in (base[:, 3:14], base[::3, :10], base.t()[:11], base[:, ::2], base[:1].expand(9, 24), base[5:6, 1:8]):
        for over in ("chosen", "all"):
            a, b = m.gate(view, 3, over=over), m.gate(view.contiguous(), 3, over=over)
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
            x, y = view.detach().requires_grad_(), view.contiguous().detach().requires_grad_()
            g = torch.randn(a[1].shape, device="cuda")
            assert torch.equal(torch.autograd.grad(m.gate(x, 3, over=over)[1], x, g)[0], torch.autograd.grad(m.gate(y, 3, over=over)[1], y, g)[0])
            s = torch.autograd.grad(m.gate(x, 3, over=over, log=True)[1].sum(), x)[0]      # a gradient with stride 0
            assert torch.equal(s, torch.autograd.grad(m.gate(x, 3, over=over, log=True)[1], x, torch.ones_like(g))[0])
    empty = torch.empty(0, 5, device="cuda", requires_grad=True)
    index, weight = m.gate(empty, 2)
    assert index.shape == (0, 2) and torch.autograd.grad(weight.sum(), empty)[0].shape == (0, 5)


# ---- routing --------------------------------------------------------------------------------------------------------

def _index(n, k, experts, seed, unrouted=0.1, skew=1.5):
    torch = _torch()
    rng = np.random.default_rng(seed)
    index = np.minimum((experts * rng.random((n, k)) ** skew).astype(np.int32), experts - 1)
    index[rng.random((n, k)) < unrouted] = -1
    if n > 2:
        index[1] = -1
        index[2] = experts          # outside: not routed
    return torch.from_numpy(index)


ROUTE = [(1, 1, 1, 1), (1, 4, 3, 2), (30, 1, 5, 2), (64, 1, 2, 1), (65, 3, 7, 4), (1000, 2, 10, 1), (1023, 1, 1024, 3), (8192, 1, 16, 1), (8193, 1, 64, 1),
         (4099, 8, 33, 16), (70001, 2, 10, 1), (50000, 3, 1000, 7), (300000, 4, 255, 4), (1100000, 1, 2, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("n,k,experts,align", ROUTE)
def test_route(native, n, k, experts, align):
    from spnc import mixture as m
    index = _index(n, k, experts, seed=n)
    plan = m.route(index.cuda(), experts, align=align)
    position, starts, counts = om.route(index.numpy(), experts, align)
    assert plan.capacity == n * k + experts * (align - 1) >= starts[-1]
    assert np.array_equal(_host(plan.counts), counts) and np.array_equal(_host(plan.starts), starts) and np.array_equal(_host(plan.position), position)


@pytest.mark.gpu
def test_route_corner_cases(native):
    torch = _torch()
    from spnc import mixture as m
    plan = m.route(torch.empty(0, 2, dtype=torch.int32, device="cuda"), 3, align=4)
    assert plan.starts.tolist() == [0] * 4 and plan.counts.tolist() == [0] * 3 and plan.capacity == 9
    plan = m.route(torch.full((70000, 1), -5, dtype=torch.int32, device="cuda"), 3)
    assert plan.starts.tolist() == [0] * 4 and (plan.position == -1).all()
    plan = m.route(torch.full((70000, 1), 2, dtype=torch.int32, device="cuda"), 3)
    assert plan.starts.tolist() == [0, 0, 0, 70000] and torch.equal(plan.position.flatten(), torch.arange(70000, dtype=torch.int32, device="cuda"))
    plan = m.route(torch.tensor([[1, 1], [0, 1]], dtype=torch.int32, device="cuda"), 2)      # an expert twice in a row
    assert plan.position.tolist() == [[1, 2], [0, 3]]
    twisted = torch.arange(12, dtype=torch.int32, device="cuda").reshape(3, 4).t() % 5
    assert torch.equal(m.route(twisted, 5).position, m.route(twisted.contiguous(), 5).position)


WIDTHS = [("float32", 1), ("float32", 6), ("float32", 16), ("float32", 100), ("float32", 257), ("bfloat16", 1000), ("bfloat16", 3), ("float16", 10), ("float64", 5),
          ("int8", 7), ("int16", 33), ("int32", 6), ("int64", 4), ("uint8", 64), ("bool", 5), ("bfloat16", 2048)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,width", WIDTHS)
def test_dispatch_and_its_gradient(native, dtype, width):
    """A copy, and the sum of k copies: k - 1 additions of 32 (64) bits, then the type's own rounding."""
    torch = _torch()
    from spnc import mixture as m
    for n, k, experts, align in [(1, 1, 2, 1), (77, 3, 5, 4), (1031, 2, 16, 1), (2100, 2, 7, 1)]:      # from 2048 rows on a wave a row
        index = _index(n, k, experts, seed=width + n)
        plan = m.route(index.cuda(), experts, align=align)
        position, _, _ = om.route(index.numpy(), experts, align)
        gen = torch.Generator().manual_seed(width)
        t = getattr(torch, dtype)
        x = torch.randn(n, width, generator=gen, dtype=torch.float64).mul(50).to(t)
        got = m.dispatch(x.cuda(), plan)
        want = np.zeros((plan.capacity, width)) if t.is_floating_point else None
        assert np.array_equal(_host(got), om.dispatch(_host(x) if want is not None else x.numpy(), position, plan.capacity))
        kept = torch.ones((plan.capacity, width), dtype=t, device="cuda")
        assert m.dispatch(x.cuda(), plan, out=kept) is kept
        used = np.zeros(plan.capacity, dtype=bool)
        used[position[position >= 0]] = True
        assert torch.equal(kept[torch.from_numpy(used).cuda()], got[torch.from_numpy(used).cuda()]) and (kept[torch.from_numpy(~used).cuda()] == 1).all()
        if not t.is_floating_point:
            continue
        leaf = x.cuda().requires_grad_()
        grad = torch.randn(plan.capacity, width, generator=gen, dtype=torch.float64).to(t)
        back, = torch.autograd.grad(m.dispatch(leaf, plan), leaf, grad.cuda())
        want = om.combine(_host(grad), position)
        size = om.combine(np.abs(_host(grad)), position)
        _near(back, want, k * HALF["float64" if dtype == "float64" else "float32"] * size + HALF[dtype] * np.abs(want) * (1 + 1e-3) + (2.0 ** -25 if dtype == "float16" else 0))


@pytest.mark.gpu
def test_dispatch_of_views(native):
    torch = _torch()
    from spnc import mixture as m
    plan = m.route(_index(50, 2, 4, seed=3).cuda(), 4, align=2)
    base = torch.randn(60, 40, device="cuda")
    for view in (base[:50, 1:7], base[10:, 4:20], base[:50, ::3], torch.randn(9, 50, device="cuda").t(), base[:1].expand(50, 40), base[:50, :0]):
        assert torch.equal(m.dispatch(view, plan), m.dispatch(view.contiguous(), plan))
    x = base[:50, 4:20].detach().requires_grad_()
    rows = m.dispatch(x, plan)
    g, = torch.autograd.grad(rows.sum(), x)                                     # a gradient with stride 0: the slots that are routed
    assert torch.equal(g, (plan.position >= 0).sum(dim=1, keepdim=True).float().expand_as(g))


# ---- combination ----------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype,width", [("float32", 1), ("float32", 6), ("float32", 100), ("float32", 257), ("bfloat16", 1000), ("bfloat16", 3), ("float16", 10),
                                         ("float16", 2048), ("float64", 5), ("float64", 64), ("bfloat16", 4096)])
@pytest.mark.parametrize("weight", ["float32", "float64", None])
def test_combine(native, dtype, width, weight):
    """k products and sums of 32 (64) bits, the output's rounding; the weights' gradient is a dot product of `width` terms."""
    torch = _torch()
    from spnc import mixture as m
    if weight == "float64" and dtype != "float64":
        weight = "float32"
    u = HALF["float64" if dtype == "float64" else "float32"]
    tiny = 2.0 ** -25 if dtype == "float16" else 0.0
    for n, k, experts, align in [(1, 1, 2, 1), (1, 4, 9, 1), (77, 3, 5, 4), (531, 8, 16, 1), (40, 11, 6, 1), (2100, 2, 7, 1)]:
        index = _index(n, k, experts, seed=width + n)
        plan = m.route(index.cuda(), experts, align=align)
        position = _host(plan.position)
        gen = torch.Generator().manual_seed(width + k)
        values = torch.randn(plan.capacity, width, generator=gen, dtype=torch.float64).to(getattr(torch, dtype))
        values[~torch.isin(torch.arange(plan.capacity), plan.position.cpu().flatten().long())] = float("nan")     # rows of no segment are not read
        w = None if weight is None else torch.softmax(torch.randn(n, k, generator=gen, dtype=torch.float64), 1).to(getattr(torch, weight))
        v_leaf = values.cuda().requires_grad_()
        w_leaf = None if w is None else w.cuda().requires_grad_()
        out = m.combine(v_leaf, plan, w_leaf)
        clean = np.nan_to_num(_host(values))
        weights = np.ones((n, k)) if w is None else _host(w)
        want = om.combine(clean, position, weights)
        size = om.combine(np.abs(clean), position, weights)
        _near(out, want, 2 * k * u * size + HALF[dtype] * np.abs(want) * (1 + 1e-3) + tiny)
        grad = torch.randn(n, width, generator=gen, dtype=torch.float64).to(values.dtype)
        leaves = (v_leaf,) if w is None else (v_leaf, w_leaf)
        back = torch.autograd.grad(out, leaves, grad.cuda())
        want_v, want_w = om.combine_gradient(clean, position, weights, _host(grad))
        _near(back[0], want_v, 2 * u * np.abs(want_v) + HALF[dtype] * np.abs(want_v) * (1 + 1e-3) + tiny)
        if w is not None:
            _, size = om.combine_gradient(np.abs(clean), position, weights, np.abs(_host(grad)))
            _near(back[1], want_w, (width + 2) * u * size + HALF[weight] * np.abs(want_w))


@pytest.mark.gpu
def test_combine_of_views_and_one_gradient(native):
    torch = _torch()
    from spnc import mixture as m
    plan = m.route(_index(50, 2, 4, seed=3).cuda(), 4, align=2)
    base = torch.randn(plan.capacity, 40, device="cuda")
    weights = torch.rand(50, 2, device="cuda")
    for view in (base[:, 1:7], base[:, 4:20], base[:, ::3], torch.randn(9, plan.capacity, device="cuda").t(), base[:1].expand(plan.capacity, 40)):
        for w in (weights, torch.rand(2, 50, device="cuda").t(), weights[:, :1].expand(50, 2)):
            v, c = view.detach().requires_grad_(), view.contiguous().detach().requires_grad_()
            a, b = m.combine(v, plan, w), m.combine(c, plan, w.contiguous())
            assert torch.equal(a, b)
            g = torch.randn(50, 2 * a.shape[1], device="cuda")[:, 1:a.shape[1] + 1]
            assert torch.equal(torch.autograd.grad(a, v, g)[0], torch.autograd.grad(b, c, g.contiguous())[0])     # the values' gradient alone
    w = weights.clone().requires_grad_()
    both = base.clone().requires_grad_()
    alone, = torch.autograd.grad(m.combine(base, plan, w).sum(), w)                                                # the weights' alone
    assert torch.equal(alone, torch.autograd.grad(m.combine(both, plan, w).sum(), (both, w))[1])
    assert m.combine(base[:, :0], plan, weights).shape == (50, 0)
    one = torch.rand(50, 1, device="cuda").requires_grad_()                                                        # a weight for all slots of a row
    shared, = torch.autograd.grad(m.combine(base, plan, one.expand(50, 2)).sum(), one)
    w = one.detach().expand(50, 2).contiguous().requires_grad_()
    assert torch.equal(shared, torch.autograd.grad(m.combine(base, plan, w).sum(), w)[0].sum(dim=1, keepdim=True))


@pytest.mark.gpu
def test_plans_without_rows(native):
    """A buffer of no rows: everything that comes back is empty sums, nothing is read."""
    torch = _torch()
    from spnc import mixture as m
    i32 = dict(dtype=torch.int32, device="cuda")
    for n in (0, 5):
        plan = m.Plan(torch.full((n, 2), 3, **i32), torch.zeros(4, **i32), torch.zeros(3, **i32), 0)     # positions behind the buffer: not routed
        w = torch.rand(n, 2, device="cuda", requires_grad=True)
        rows = torch.empty(0, 6, device="cuda", requires_grad=True)
        y = m.combine(rows, plan, w)
        assert y.shape == (n, 6) and bool((y == 0).all())
        gr, gw = torch.autograd.grad(y, (rows, w), torch.ones_like(y))
        assert gr.shape == (0, 6) and bool((gw == 0).all()) and gw.shape == (n, 2)
        v = torch.empty(0, device="cuda", requires_grad=True)
        z = m.combine_log(v, plan, w)
        assert z.shape == (n,) and bool((z == -float("inf")).all())
        gv, gw = torch.autograd.grad(z, (v, w), torch.ones_like(z))
        assert gv.shape == (0,) and bool((gw == 0).all())
        assert m.dispatch(torch.rand(n, 6, device="cuda"), plan).shape == (0, 6)


@pytest.mark.gpu
def test_captured_small_calls(native):
    """The serving form of each operator, captured and replayed with new data; a thousand experts need more LDS than a kernel has unasked."""
    torch = _torch()
    from spnc import mixture as m
    z, x, v = torch.randn(3, 1000, device="cuda"), torch.randn(3, 40, device="cuda").bfloat16(), torch.randn(6, device="cuda")

    def step():
        index, w = m.gate(z, 2, log=True)
        plan = m.route(index, 1000)
        return index, plan.position, m.dispatch(x, plan), m.combine(m.dispatch(x, plan), plan, w.exp()), m.combine_log(v, plan, w), m.dropout(x, 0.5, 3)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(3):
        z.normal_(), x.normal_(), v.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, step()))


LOG = [(1, 1, 2, 1), (1, 2, 10, 1), (77, 3, 5, 4), (1031, 2, 16, 1), (300, 8, 9, 1), (130, 11, 6, 2), (70, 64, 100, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("weight", ["float32", "float64"])
def test_combine_log(native, dtype, weight):
    """The result is rounded once at its own size; before that the differences between the terms are, (|difference| <= 64 in
    the terms that count), exp within 2 units, k terms and a logarithm: 64 + k + 8 half steps of a number of order one, and the
    largest term's size decides how many half steps the final sum costs. Shares carry the same relative error."""
    torch = _torch()
    from spnc import mixture as m
    u = HALF[dtype]
    for shift in (0.0, -900.0):
        for n, k, experts, align in LOG:
            rng = np.random.default_rng(n + k)
            index = _index(n, k, experts, seed=n)
            plan = m.route(index.cuda(), experts, align=align)
            position = _host(plan.position)
            values = torch.tensor(shift + 6.0 * rng.normal(size=plan.capacity)).to(getattr(torch, dtype))
            values[torch.from_numpy(rng.random(plan.capacity) < 0.1)] = -float("inf")
            log_weights = torch.log_softmax(torch.tensor(rng.normal(size=(n, k))), 1)
            log_weights[torch.from_numpy(rng.random((n, k)) < 0.1)] = -float("inf")
            log_weights = log_weights.to(getattr(torch, weight))
            # values behind closed slots and in rows of no segment do not matter
            unused = np.ones(plan.capacity, dtype=bool)
            unused[position[(position >= 0) & np.isfinite(_host(log_weights))]] = False
            values[torch.from_numpy(unused)] = float("nan")
            grad = torch.tensor(rng.normal(size=n)).to(values.dtype)
            v, w = values.cuda().requires_grad_(), log_weights.cuda().requires_grad_()
            out = m.combine_log(v, plan, w)
            rounded = _host(log_weights.to(values.dtype))
            want, want_v, want_w = om.combine_log(np.where(unused, 0.0, _host(values)), position, rounded, _host(grad))
            steps = 64 + k + 8
            _near(out, want, u * (steps + 2 * np.abs(np.where(np.isfinite(want), want, 0.0))), (shift, n, k))
            got_v, got_w = torch.autograd.grad(out, (v, w), grad.cuda())
            _near(got_v, want_v, 2 * steps * u * np.abs(want_v) + 1e-300)
            _near(got_w, want_w, (2 * steps * u + HALF[weight]) * np.abs(want_w) + (1e-38 if weight == "float32" else 1e-300))
            assert torch.equal(torch.autograd.grad(m.combine_log(values.cuda(), plan, w), w, grad.cuda())[0], got_w)
            assert torch.equal(torch.autograd.grad(m.combine_log(v, plan, w.detach()), v, grad.cuda())[0], got_v)


@pytest.mark.gpu
def test_combine_log_of_special_values(native):
    torch = _torch()
    from spnc import mixture as m
    nan, inf = float("nan"), float("inf")
    plan = m.Plan(torch.tensor([[0, 1], [2, 3], [4, -1], [-1, -1], [5, 6], [7, 8], [9, 10]], dtype=torch.int32, device="cuda"),
                  torch.tensor([0, 11], dtype=torch.int32, device="cuda"), torch.tensor([11], dtype=torch.int32, device="cuda"), 11)
    values = torch.tensor([-inf, -inf, -inf, -3.0, -5.0, nan, -1.0, nan, -1.0, inf, 0.0], device="cuda", requires_grad=True)
    weights = torch.tensor([[-1.0, -1.0], [-0.5, -0.25], [-2.0, nan], [-1.0, -1.0], [-0.5, -0.5], [-inf, -0.5], [-1.0, -1.0]], device="cuda", requires_grad=True)
    out = m.combine_log(values, plan, weights)
    want = [-inf, -3.25, -7.0, -inf, nan, -1.5, inf]
    assert np.array_equal(_host(out), np.array(want), equal_nan=True)
    gv, gw = torch.autograd.grad(out, (values, weights), torch.ones(7, device="cuda"))
    assert gv[[0, 1, 2, 3, 4, 7, 8]].tolist() == [0, 0, 0, 1, 1, 0, 1] and gw[[0, 1, 2, 3, 5]].tolist() == [[0, 0], [0, 1], [1, 0], [0, 0], [0, 1]]


@pytest.mark.gpu
def test_gradients_against_differences(native):
    """Central differences in 64 bits: the truncation error is of order h^2 = 1e-10, the cancellation 1e-16 / h = 1e-11."""
    torch = _torch()
    from spnc import mixture as m
    rng = np.random.default_rng(11)
    z = torch.tensor(rng.normal(size=(6, 7)), device="cuda")
    values = torch.tensor(rng.normal(size=(12, 5)), device="cuda")
    lls = torch.tensor(rng.normal(size=12) - 4.0, device="cuda")
    x = torch.tensor(rng.normal(size=(6, 5)), device="cuda")
    plan = m.route(m.gate(z, 2)[0], 7)
    w2, w1 = torch.tensor(rng.normal(size=(6, 5)), device="cuda"), torch.tensor(rng.normal(size=6), device="cuda")
    c2 = torch.tensor(rng.normal(size=(12, 5)), device="cuda")

    functions = [(lambda t: (m.combine(values, plan, m.gate(t, 2, over=over)[1]) * w2).sum(), z) for over in ("chosen", "all")]
    functions += [(lambda t: (m.combine_log(lls, plan, m.gate(t, 2, over=over, log=True)[1]) * w1).sum(), z) for over in ("chosen", "all")]
    functions += [(lambda t: (m.combine(t, plan, m.gate(z, 2)[1]) * w2).sum(), values), (lambda t: (m.combine_log(t, plan, m.gate(z, 2, log=True)[1]) * w1).sum(), lls),
                  (lambda t: (m.dispatch(t, plan) * c2).sum(), x), (lambda t: (m.dropout(t, 0.4, 9) * w2).sum(), x)]
    for f, at in functions:
        leaf = at.clone().requires_grad_()
        grad, = torch.autograd.grad(f(leaf), leaf)
        h = 1e-5
        for i in range(0, at.numel(), 3):
            step = torch.zeros(at.numel(), dtype=at.dtype, device="cuda")
            step[i] = h
            up, down = f(at + step.view(at.shape)), f(at - step.view(at.shape))
            assert abs(float((up - down) / (2 * h)) - float(grad.flatten()[i])) <= 1e-8


@pytest.mark.gpu
def test_second_gradients_and_changed_plans_are_errors(native):
    torch = _torch()
    from spnc import mixture as m
    plan = m.route(torch.zeros(4, 1, dtype=torch.int32, device="cuda"), 1)
    x, w, v = torch.randn(4, 3, device="cuda", requires_grad=True), torch.rand(4, 1, device="cuda", requires_grad=True), torch.randn(4, device="cuda", requires_grad=True)
    for f, leaf in ((lambda: m.gate(x, 2, log=True)[1], x), (lambda: m.gate(x, 2, over="all")[1], x), (lambda: m.dispatch(x, plan), x), (lambda: m.combine(x, plan), x),
                    (lambda: m.combine(x, plan, w), w), (lambda: m.combine_log(v, plan, w), v), (lambda: m.dropout(x, 0.1, 3), x)):
        first, = torch.autograd.grad((f() ** 2).sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="cannot be differentiated again"):
            first.sum().backward()
    for f in (lambda: m.dispatch(x, plan), lambda: m.combine(x, plan, w), lambda: m.combine_log(v, plan, w)):
        y = f()
        plan.position.zero_()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
        plan = m.route(torch.zeros(4, 1, dtype=torch.int32, device="cuda"), 1)


# ---- dropout --------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float64", "float16", "bfloat16"])
@pytest.mark.parametrize("marginal", [False, True])
def test_dropout(native, dtype, marginal):
    """One product of the scale rounded to 32 (64) bits, then the type's rounding; the mask has to be equal."""
    torch = _torch()
    from spnc import mixture as m
    t, u = getattr(torch, dtype), HALF["float64" if dtype == "float64" else "float32"]
    for shape, p, seed, offset in [((1,), 0.5, 0, 0), ((), 0.3, 5, 1), ((3,), 0.0, 1, 0), ((37, 16), 0.2, 2 ** 63 + 5, 2 ** 40), ((5, 7, 9), 0.1, 77, 3), ((2, 1001), 1.0, 1, 1),
                                   ((130, 3), 0.9, 123456789, 2 ** 64 - 1), ((64, 8), 0.5, 4, 4), ((0, 5), 0.5, 1, 0), ((3, 0, 2), 0.5, 1, 0)]:
        x = torch.randn(shape, generator=torch.Generator().manual_seed(seed % 1000), dtype=torch.float64).to(t)
        if x.numel() > 20:
            x.view(-1)[::7] = float("inf")
            x.view(-1)[3::11] = float("nan")
        leaf = x.cuda().requires_grad_()
        y = m.dropout(leaf, p, seed, offset=offset, marginal=marginal)
        assert y.shape == x.shape and y.dtype == t
        keep = om.keep(x.numel(), p, seed, offset).reshape(shape)
        scale = 1.0 if marginal else 0.0 if p == 1.0 else 1.0 / (1.0 - p)
        want = np.where(keep, np.where(keep, _host(x), 0.0) * scale, np.nan if marginal else 0.0)
        bound = (2 * u + HALF[dtype] * (1 + 1e-3)) * np.abs(np.where(np.isfinite(want), want, 0.0)) + (2.0 ** -25 if dtype == "float16" else 0)
        _near(y, want, bound)
        device_offset = torch.tensor([offset - 2 ** 64 if offset >= 2 ** 63 else offset], device="cuda")
        again = m.dropout(leaf, p, seed, offset=device_offset, marginal=marginal)
        assert np.array_equal(_host(again), _host(y), equal_nan=True)
        grad = torch.randn(shape, dtype=torch.float64).to(t)
        want = np.where(keep, _host(grad) * scale, 0.0)
        bound = (2 * u + HALF[dtype] * (1 + 1e-3)) * np.abs(want) + (2.0 ** -25 if dtype == "float16" else 0)
        for out in (y, again):
            _near(torch.autograd.grad(out, leaf, grad.cuda())[0], want, bound)


@pytest.mark.gpu
def test_dropout_mask_is_a_function_of_the_position(native):
    torch = _torch()
    from spnc import mixture as m
    base = torch.rand(50, 48, device="cuda") + 1.0
    for view in (base[:, 1:8], base[:, 4:20], base[::2, :12], base[:, ::3], base.t(), base[:1].expand(50, 48), base[:, 5:6]):
        assert torch.equal(m.dropout(view, 0.3, 8), m.dropout(view.contiguous(), 0.3, 8))
    masks = [m.dropout(base.to(t), 0.3, 8) == 0 for t in (torch.float32, torch.float64, torch.float16, torch.bfloat16)]
    assert all(torch.equal(masks[0], x) for x in masks)
    assert torch.equal(torch.isnan(m.dropout(base, 0.3, 8, marginal=True)), masks[0])
    assert torch.equal(m.dropout(base[:10].reshape(-1), 0.3, 8) == 0, masks[0][:10].reshape(-1))
    assert not torch.equal(m.dropout(base, 0.3, 9) == 0, masks[0]) and not torch.equal(m.dropout(base, 0.3, 8, offset=1) == 0, masks[0])
    # a changed offset between the passes is an error, not another mask
    offset, x = torch.zeros(1, dtype=torch.int64, device="cuda"), base.clone().requires_grad_()
    y = m.dropout(x, 0.3, 8, offset=offset)
    offset += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.gpu
def test_dropout_share(native):
    """2^22 draws: five standard deviations of a binomial share, sqrt(p (1 - p) / 2^22) = 2e-4."""
    torch = _torch()
    from spnc import mixture as m
    x = torch.ones(1 << 22, device="cuda")
    for p in (0.05, 0.2, 0.5):
        y = m.dropout(x, p, 31)
        assert abs(float((y == 0).double().mean()) - p) <= 5 * (p * (1 - p) / x.numel()) ** 0.5


# ---- together -------------------------------------------------------------------------------------------------------

def _experts():
    from spnc.structure import Gaussian, Product, Sum
    rng = np.random.default_rng(5)
    out = []
    for _ in range(5):
        parts = [Product(children=[Gaussian(float(rng.normal()), float(rng.uniform(0.4, 1.5)), scope=f) for f in range(6)]) for _ in range(2)]
        out.append(Sum(weights=[0.3, 0.7], children=parts))
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("options", [{}, {"hip-compute-type": "float64"}, {"hip-kernel": "interpreter"}])
def test_mixture_of_kernels(native, options):
    """Kernels within 1e-4 (1e-10 in float64) of their closed form; a log-sum-exp moves no more than its terms do. The gate's log
    weights l have 32 bits here whatever the kernels have: as in test_gate, each is within (24 + 5) 2^-24 max(1, |l|), so the
    result is within the kernels' error plus that of the row's largest |l|. A share exp(t_j - total) moves by twice the terms'
    error relative to itself, the logits' gradient g (r_j - w_j) by that and the weight's: four times, and its own rounding."""
    torch = _torch()
    from oracle import evaluate as ev
    from spnc import mixture as m
    from spnc.hip import HIPCompiler
    spns = _experts()
    with quiet():
        mix = HIPCompiler(**options).compile_mixture(spns, "float32")
    try:
        models = [oracle_model(s, "float32") for s in spns]
        f64 = mix.kernels[0].dataType() == "float64"
        for n in (1, 37, 4001):
            rng = np.random.default_rng(n)
            x = torch.tensor(rng.normal(size=(n, 6)).astype(np.float32), device="cuda")
            x = m.dropout(x, 0.2, 6, offset=n, marginal=True)
            logits = torch.tensor(rng.normal(size=(n, 5)), dtype=torch.float32)
            logits[torch.from_numpy(rng.random((n, 5)) < 0.2)] = -float("inf")
            if n > 1:
                logits[3] = -float("inf")
            leaf = logits.cuda().requires_grad_()
            got = mix.log_likelihood(x, leaf, 2)
            index, log_weights = om.gate(_host(logits), 2, log=True)
            lls = np.stack([ev.ll_closed_f64(mod, x.cpu().numpy(), marginal=True) for mod in models], axis=1)
            position = np.arange(2 * n).reshape(n, 2)
            position[index < 0] = -1
            values = lls[np.arange(n)[:, None], np.maximum(index, 0)].reshape(-1)
            grad = rng.normal(size=n)
            want, _, want_w = om.combine_log(values, position, log_weights, grad)
            terms = (1e-10 if f64 else 1e-4) + 29 * 2.0 ** -24 * np.maximum(1.0, np.abs(np.where(np.isfinite(log_weights), log_weights, 0.0)).max(axis=1))
            _near(got, want, terms + (0.0 if f64 else 2.0 ** -23 * np.abs(np.where(np.isfinite(want), want, 0.0)).astype(np.float64)))
            back, = torch.autograd.grad(got, leaf, torch.tensor(grad, dtype=got.dtype, device="cuda"))
            _near(back, om.gate_gradient(_host(logits), index, want_w, log=True), (4 * terms + 2.0 ** -22)[:, None] * np.abs(grad)[:, None])
        empty = mix.log_likelihood(torch.empty(0, 6, device="cuda"), torch.empty(0, 5, device="cuda"), 2)
        assert empty.shape == (0,)
        with pytest.raises(RuntimeError, match="no gradient with respect to their features"):
            mix.log_likelihood(torch.zeros(1, 6, device="cuda", requires_grad=True), torch.zeros(1, 5, device="cuda"), 2)
    finally:
        for k in mix.kernels:
            os.remove(k.fileName())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["auto", "interpreter"])
def test_mixture_on_several_streams(native, kind):
    """Six segments run beside each other, two of them under one kernel: the same bits as one kernel after the other, call after call
    and from two streams at once."""
    torch = _torch()
    from spnc import mixture as m
    from spnc.hip import HIPCompiler
    with quiet():
        mix = HIPCompiler(**{"hip-kernel": kind}).compile_mixture(_experts(), "float32")
    try:
        mix = m.Mixture(mix.kernels + mix.kernels[:1])
        x, z = torch.randn(30011, 6, device="cuda"), torch.randn(30011, 6, device="cuda")
        index, lw = m.gate(z, 2, log=True)
        each = torch.stack([torch.from_numpy(k.execute(30011, x.cpu().numpy())).cuda() for k in mix.kernels], 1)
        plan = m.Plan(torch.arange(60022, dtype=torch.int32, device="cuda").view(-1, 2), torch.tensor([0, 60022], dtype=torch.int32, device="cuda"),
                      torch.tensor([60022], dtype=torch.int32, device="cuda"), 60022)
        want = m.combine_log(each.gather(1, index.long()).flatten(), plan, lw)
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        got = []
        for call in range(6):
            with torch.cuda.stream(streams[call % 2]):
                got.append(mix.log_likelihood(x, z, 2))
        torch.cuda.synchronize()
        assert all(torch.equal(g, want) for g in got)
    finally:
        for k in mix.kernels[:5]:
            os.remove(k.fileName())


@pytest.mark.gpu
def test_mixture_of_integer_kernels_is_aligned(native):
    """Rows of 6 x 4 bytes: a segment that began at an odd row would not be aligned for the kernel."""
    torch = _torch()
    from spnc import synthetic as syn
    from spnc.hip import HIPCompiler
    from spnc.structure import Categorical, Product
    other = Product(children=[Categorical(p=[.2, .3, .5], scope=i) for i in range(6)])
    with quiet():
        mix = HIPCompiler().compile_mixture([syn.c1_spn(), other, syn.c1_spn()], "int32", supportMarginal=False)
    try:
        x = torch.from_numpy(syn.c1_inputs(501)).cuda()
        index = torch.arange(501, device="cuda") % 3
        logits = torch.full((501, 3), -float("inf"), device="cuda").scatter_(1, index[:, None], 0.0)
        got = mix.log_likelihood(x, logits, 1)
        each = [torch.from_numpy(k.execute(501, x.cpu().numpy())).cuda() for k in mix.kernels]
        want = torch.stack(each, 1).gather(1, index[:, None]).flatten()
        assert torch.equal(got, want)
    finally:
        for k in mix.kernels:
            os.remove(k.fileName())


def _training_step(m, x, logits, expert, grad, offset):
    """dropout -> gate -> route -> dispatch -> experts -> combine, and back to rows, logits and the experts' scales."""
    torch = _torch()
    dropped = m.dropout(x, 0.1, 42, offset=offset)
    index, weight = m.gate(logits, 2, over="all")
    plan = m.route(index, logits.shape[1])
    rows = m.dispatch(dropped, plan)
    y = m.combine(rows * expert, plan, weight)
    return (y, *torch.autograd.grad(y, (x, logits, expert), grad))


@pytest.mark.gpu
def test_captured_training_step_and_other_streams(native):
    """Forward and backward in one graph: every replay on new data, with eager work between, equals the eager result; and so
    does the same step on two streams at once."""
    torch = _torch()
    from spnc import mixture as m
    gen = torch.Generator(device="cuda").manual_seed(1)

    def data():
        return (torch.randn(5000, 96, generator=gen, device="cuda"), torch.randn(5000, 12, generator=gen, device="cuda"),
                torch.rand(10000, 96, generator=gen, device="cuda"), torch.randn(5000, 96, generator=gen, device="cuda"))

    static = [t.requires_grad_(i < 3) for i, t in enumerate(data())]
    offset = torch.zeros(1, dtype=torch.int64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _training_step(m, *static, offset)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = _training_step(m, *static, offset)
    for replay in range(4):
        fresh = data()
        with torch.no_grad():
            for s, f in zip(static, fresh):
                s.copy_(f)
        offset.fill_(replay)
        graph.replay()
        torch.cuda.synchronize()
        eager = _training_step(m, *[f.requires_grad_(i < 3) for i, f in enumerate(fresh)], replay)
        for a, b in zip(captured, eager):
            assert torch.equal(a, b), replay
    sets = [[t.requires_grad_(i < 3) for i, t in enumerate(data())] for _ in range(4)]
    want = [_training_step(m, *s, 7) for s in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i, s in enumerate(sets):
        with torch.cuda.stream(streams[i % 2]):
            got.append(_training_step(m, *s, 7))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
def test_an_error_left_behind_is_not_ours(native):
    """Somebody's failed runtime call (a device that does not exist) leaves its code to be read by the next who asks."""
    torch = _torch()
    from spnc import mixture as m
    z = torch.randn(4, 6, device="cuda")
    want = m.gate(z, 2)
    hip = ctypes.CDLL(os.path.join(os.path.dirname(torch.__file__), "lib", "libamdhip64.so"))      # the runtime both use
    assert hip.hipSetDevice(ctypes.c_int(9999)) != 0 and hip.hipPeekAtLastError() != 0
    got = m.gate(z, 2)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_mixture_refuses_capture(native):
    torch = _torch()
    from spnc.hip import HIPCompiler
    with quiet():
        mix = HIPCompiler().compile_mixture(_experts()[:2], "float32")
    x, z = torch.zeros(8, 6, device="cuda"), torch.zeros(8, 2, device="cuda")
    mix.log_likelihood(x, z, 1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = x + 1.0
        with pytest.raises(RuntimeError, match="graph capture"):
            mix.log_likelihood(x, z, 1)
    graph.replay()
    torch.cuda.synchronize()
    assert bool((y == 1).all())
    for k in mix.kernels:
        os.remove(k.fileName())


@pytest.mark.gpu
def test_rows_past_four_gibibytes(native):
    """Byte offsets past 2^32 in the sorted buffer and in dropout's element count (bf16: 2.2e9 elements)."""
    torch = _torch()
    from spnc import mixture as m
    n, width = 1_100_000, 2048
    x = torch.empty(n, width, dtype=torch.bfloat16, device="cuda")
    x[:] = (torch.arange(n, device="cuda") % 251).to(torch.bfloat16)[:, None]
    index = (torch.arange(n, device="cuda", dtype=torch.int32) % 3)[:, None].contiguous()
    plan = m.route(index, 3)
    rows = m.dispatch(x, plan)
    for at in (0, 1, 366666, 366667, n - 2, n - 1):
        assert bool((rows[plan.position[at, 0]] == at % 251).all())
    back = m.combine(rows, plan, torch.ones(n, 1, device="cuda"))
    assert torch.equal(back, x)
    del back, rows
    y = m.dropout(x, 0.5, 3, marginal=True)
    first = (n - 1) * width
    keep = om.keep(width, 0.5, 3, first=first)
    assert np.array_equal(~torch.isnan(y[-1]).cpu().numpy(), keep)
