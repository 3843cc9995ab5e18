"""Calls of spnc.mixture and of its C-ABI that are out of the ordinary: buffers that are used again or shared, views whose memory does not
hold their values, kinds of derivatives that are not offered, errors of other calls."""
import ctypes
import os
import random
import subprocess

import pytest

from conftest import ROOT, quiet


def _torch():
    import torch
    return torch


@pytest.fixture
def mix(native):
    """Two Gaussian mixtures over six float32 features."""
    from spnc.hip import HIPCompiler
    from spnc.structure import Gaussian, Product, Sum
    spns = [Sum(weights=[0.25, 0.75], children=[Product(children=[Gaussian(0.1 * f - s, 0.5 + 0.2 * p, scope=f) for f in range(6)]) for p in range(2)])
            for s in range(2)]
    with quiet():
        mixture = HIPCompiler().compile_mixture(spns, "float32")
    yield mixture
    for k in mixture.kernels:
        os.remove(k.fileName())


def _plan(rows=4):
    """One expert, slot i in row i."""
    torch = _torch()
    from spnc import mixture as m
    return m.route(torch.zeros(rows, 1, dtype=torch.int32, device="cuda"), 1)


@pytest.mark.gpu
def test_writing_to_out_again_is_seen_by_the_backward_pass(native):
    """Who saved the buffer for a gradient must not compute it from another call's rows."""
    torch = _torch()
    from spnc import mixture as m
    plan, x, buf = _plan(), torch.randn(4, 3, device="cuda"), torch.empty(4, 3, device="cuda")
    w = torch.rand(3, device="cuda", requires_grad=True)
    before = buf._version
    m.dispatch(x, plan, out=buf)
    assert buf._version > before
    (buf * w).sum().backward()
    assert bool(((w.grad - x.sum(dim=0)).abs() <= 8 * 2.0 ** -24 * x.abs().sum(dim=0)).all())      # twice three additions
    y = (buf * w).sum()
    m.dispatch(x + 1.0, plan, out=buf)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():                                   # tensors without a counter
        kept = torch.empty(4, 3, device="cuda")
        assert torch.equal(m.dispatch(x, plan, out=kept), x)
    with pytest.raises(RuntimeError, match="inference"):           # as any write to them from outside
        m.dispatch(x, plan, out=kept)


def _negated(t):
    """A view that holds t with the other sign and torch's flag for it, as autograd makes them of conjugates."""
    torch = _torch()
    view = torch.complex(torch.zeros_like(t), -t).conj().imag
    assert view.is_neg() and torch.equal(view, t)
    return view


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width", [(1, 1), (4, 1), (4, 3)])
def test_negated_views(native, rows, width):
    """As inputs, as weights and as gradients: the same bits as for a tensor of the same numbers."""
    torch = _torch()
    from spnc import mixture as m
    plan = _plan(rows)
    x, one = torch.randn(rows, width, device="cuda"), torch.randn(rows, 1, device="cuda")
    functions = [lambda t: m.gate(t, 1, over="all", log=True)[1], lambda t: m.dispatch(t, plan), lambda t: m.combine(t, plan), lambda t: m.combine(t, plan, one),
                 lambda t: m.dropout(t, 0.3, 5), lambda t: m.dropout(t, 0.3, 5, marginal=True)]
    if width == 1:
        functions += [lambda t: m.combine(one, plan, t), lambda t: m.combine_log(one.flatten(), plan, t), lambda t: m.combine_log(t.flatten(), plan, one)]
    for i, f in enumerate(functions):
        want, got = f(x), f(_negated(x))
        assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0)), i
        leaf = x.clone().requires_grad_()
        out = f(leaf)
        g = torch.randn_like(out)
        want, = torch.autograd.grad(out, leaf, g)
        got, = torch.autograd.grad(f(leaf), leaf, _negated(g))
        assert torch.equal(got, want), i
    # the way they come about: the result as an imaginary part whose conjugate is used
    leaf = x.clone().requires_grad_()
    g = torch.randn(rows, width, dtype=torch.complex64, device="cuda")
    got, = torch.autograd.grad(torch.complex(torch.zeros_like(x), m.combine(leaf, plan)).conj(), leaf, g)
    assert torch.equal(got, -g.imag)
    with pytest.raises(RuntimeError, match="out must be"):
        m.dispatch(x, plan, out=torch._neg_view(torch.empty_like(x)))


@pytest.mark.gpu
def test_kernels_over_negated_views(mix):
    torch = _torch()
    from spnc import mixture as m
    x = torch.randn(40, 6, device="cuda")
    plan = m.route((torch.arange(40, device="cuda", dtype=torch.int32) % 2)[:, None].contiguous(), 2, align=4)
    rows = m.dispatch(x, plan)
    position = plan.position.flatten().long()
    assert torch.equal(mix.execute(torch._neg_view(-rows), plan)[position], mix.execute(rows, plan)[position])


# ---- shared memory --------------------------------------------------------------------------------------------------

def _refused(lib, rc, message):
    text = lib.spnc_hip_last_error().decode()
    assert rc != 0 and message in text, text


def test_dispatch_refuses_to_write_where_it_reads(native):
    """Through the C-ABI, with addresses that nobody reads: the calls are refused first."""
    lib, p = native._load(), ctypes.c_void_p

    def call(rows, out, n=4, row_bytes=16, stride=16, position=1 << 30, capacity=4, starts=1 << 31, counts=1 << 32, clear=0):
        return lib.spnc_hip_dispatch(p(rows), n, row_bytes, stride, p(position), 1, capacity, p(starts), p(counts), 2, clear, p(out), None)

    base = 1 << 20
    for rows, out, more in [(base, base, {}), (base, base + 48, {}), (base + 48, base, {}), (base, base + 63, {}), (base + 16, base, dict(capacity=2)),
                            (base, base + 63, dict(n=2, row_bytes=64, stride=256, capacity=1)),
                            (base, base + 256 - 63, dict(n=2, row_bytes=64, stride=256, capacity=1)),
                            (base, base + 8, dict(stride=0)),                                                      # one row for all
                            (base, 1 << 25, dict(position=(1 << 25) + 63)), (base, 1 << 25, dict(position=(1 << 25) - 15)),
                            (base, 1 << 25, dict(starts=1 << 25, clear=1)), (base, 1 << 25, dict(counts=(1 << 25) + 60, clear=1))]:
        _refused(lib, call(rows, out, **more), "overlaps")


def _overlap_program(tmp_path):
    """The test of the entry points by itself: out, its bytes, and rows' address, number, bytes and stride a line, from standard input."""
    src = tmp_path / "o.hip"
    src.write_text('#include <cstdio>\n#include "row_common.h"\nstd::string& spnc_hip::lastError() { static std::string s; return s; }\n'
                   'int main() { size_t o, l, r, n, b, s; while (scanf("%zu %zu %zu %zu %zu %zu", &o, &l, &r, &n, &b, &s) == 6)'
                   ' putchar(spnc_hip::overlap(reinterpret_cast<void*>(o), l, {reinterpret_cast<void*>(r), n, b, s}) ? \'1\' : \'0\'); }\n')
    exe = str(tmp_path / "o")
    subprocess.run(["/opt/rocm/bin/hipcc", "--offload-arch=gfx950", "-std=c++17", "-Wno-unused-function", "-I", os.path.join(ROOT, "spn-compiler_amd", "csrc"), str(src), "-o", exe],
                   check=True)
    return exe


def test_overlap_of_rows_and_a_buffer(tmp_path):
    """Against sets of bytes: rows that lie around the buffer share nothing with it."""
    rng = random.Random(3)
    cases = [(64 + rng.randrange(60), rng.randrange(20), 64 + rng.randrange(60), rng.randrange(5), rng.randrange(9), rng.randrange(24)) for _ in range(4000)]
    want = ""
    for o, length, r, n, b, s in cases:
        rows = {r + i * s + q for i in range(n) for q in range(b)}
        want += "1" if rows & set(range(o, o + length)) else "0"
    got = subprocess.run([_overlap_program(tmp_path)], input="\n".join(" ".join(map(str, c)) for c in cases), capture_output=True, text=True, check=True).stdout
    assert 400 < want.count("1") < 3600 and got == want


def test_overlap_of_rows_and_rows(tmp_path):
    src = tmp_path / "o.hip"
    src.write_text('#include <cstdio>\n#include "row_common.h"\nstd::string& spnc_hip::lastError() { static std::string s; return s; }\n'
                   'int main() { size_t v[8]; while (scanf("%zu %zu %zu %zu %zu %zu %zu %zu", v, v + 1, v + 2, v + 3, v + 4, v + 5, v + 6, v + 7) == 8)'
                   ' putchar(spnc_hip::overlap({reinterpret_cast<void*>(v[0]), v[1], v[2], v[3]}, {reinterpret_cast<void*>(v[4]), v[5], v[6], v[7]}) ? \'1\' : \'0\'); }\n')
    exe = str(tmp_path / "o")
    subprocess.run(["/opt/rocm/bin/hipcc", "--offload-arch=gfx950", "-std=c++17", "-Wno-unused-function", "-I", os.path.join(ROOT, "spn-compiler_amd", "csrc"), str(src), "-o", exe],
                   check=True)
    rng, cases, want = random.Random(4), [], ""
    for i in range(6000):
        a, b = [(64 + rng.randrange(70), rng.randrange(6), rng.randrange(7), rng.randrange(20)) for _ in range(2)]
        if i % 2:
            b = b[:3] + (a[3],)                                  # equal strides have a formula of their own
        cases.append(a + b)
        x, y = [{at + i * step + q for i in range(n) for q in range(width)} for at, n, width, step in (a, b)]
        want += "1" if x & y else "0"
    got = subprocess.run([exe], input="\n".join(" ".join(map(str, c)) for c in cases), capture_output=True, text=True, check=True).stdout
    assert 600 < want.count("1") < 5400 and got == want


def test_c_entry_points_refuse_to_write_where_they_read(native):
    """Every output on top of every input and of every other output, at the first and at the last byte; addresses that nobody reads."""
    lib = native._load()
    n, k, experts, width, capacity = 6, 2, 4, 8, 12
    slots = n * k
    # name: (pointers in the order of the call: bytes and whether written), the call with their addresses
    calls = {
        "gate": ([(n * experts * 4, 0), (slots * 4, 1), (slots * 4, 1)], lambda z, i, w: lib.spnc_hip_gate(z, 0, n, experts, experts, k, 0, i, w, None)),
        "gate gradient": ([(n * experts * 2, 0), (slots * 4, 0), (slots * 4, 0), (slots * 4, 0), (n * experts * 2, 1)],
                          lambda z, i, w, g, o: lib.spnc_hip_gate_backward(z, 2, n, experts, experts, k, 1, i, w, g, o, None)),
        "route": ([(20000 * 4, 0), (20000 * 4, 1), (20, 1), (16, 1), (lib.spnc_hip_route_workspace(20000, experts), 1)],
                  lambda i, p, s, c, w: lib.spnc_hip_route(i, 20000, experts, 1, p, s, c, w, 1 << 20, None)),
        "dispatch": ([(n * 32, 0), (slots * 4, 0), (20, 0), (16, 0), (capacity * 32, 1)],
                     lambda x, p, s, c, o: lib.spnc_hip_dispatch(x, n, 32, 32, p, k, capacity, s, c, experts, 1, o, None)),
        "combine": ([(capacity * width * 4, 0), (slots * 4, 0), (slots * 4, 0), (n * width * 4, 1)],
                    lambda v, p, w, o: lib.spnc_hip_combine(v, 0, capacity, width, width, p, n, k, w, 0, o, None)),
        "combine gradient": ([(capacity * width * 8, 0), (slots * 4, 0), (slots * 8, 0), (n * width * 8, 0), (20, 0), (16, 0), (capacity * width * 8, 1), (slots * 8, 1)],
                             lambda v, p, w, g, s, c, gv, gw: lib.spnc_hip_combine_backward(v, 1, capacity, width, width, p, n, k, w, 1, g, width, s, c, experts, gv, gw, None)),
        "combine_log": ([(capacity * 8, 0), (slots * 4, 0), (slots * 4, 0), (n * 8, 1), (slots * 8, 1)],
                        lambda v, p, w, o, s: lib.spnc_hip_combine_log(v, 1, capacity, p, n, k, w, 0, o, s, None)),
        "combine_log gradient": ([(slots * 4, 0), (slots * 4, 0), (n * 4, 0), (20, 0), (16, 0), (capacity * 4, 1), (slots * 8, 1)],
                                 lambda h, p, g, s, c, gv, gw: lib.spnc_hip_combine_log_backward(h, 0, capacity, p, n, k, 1, g, s, c, experts, gv, gw, None)),
        "dropout": ([(n * width * 4, 0), (n * width * 4, 1), (8, 0)], lambda x, o, at: lib.spnc_hip_dropout(x, 0, n, width, width, o, width, 0.5, 0, 1, 0, at, None)),
    }
    for name, (sizes, call) in calls.items():
        for out, (out_bytes, written) in enumerate(sizes):
            for other, (bytes_, _) in enumerate(sizes):
                if not written or other == out:
                    continue
                for shift in (8 - out_bytes, 0, bytes_ // 8 * 8 - (8 if bytes_ % 8 == 0 else 0)):
                    if name == "dropout" and other == 0 and shift == 0:
                        continue                                   # in place is allowed
                    addresses = [(1 << 20) * (i + 1) for i in range(len(sizes))]
                    addresses[out] = addresses[other] + shift
                    rc = call(*[ctypes.c_void_p(a) for a in addresses])
                    _refused(lib, rc, name + ": an output overlaps")
    p = ctypes.c_void_p
    _refused(lib, lib.spnc_hip_dropout(p(1 << 20), 0, n, width, 16, p(1 << 20), 24, 0.5, 0, 1, 0, None, None), "overlaps")     # in place, other strides


def test_dispatch_refuses_shared_tensors():
    torch = _torch()
    from spnc import mixture as m
    plan = m.Plan(torch.zeros(4, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 4)
    x = torch.zeros(9, 4)
    ints = torch.zeros(12, dtype=torch.int32)
    for rows, out in [(x[:4], x[:4]), (x[:4], x[3:7]), (x[2:6], x[:4]), (x[:4].t(), x[:4]), (ints[4:8].view(4, 1), ints[5:9].view(4, 1))]:
        with pytest.raises(RuntimeError, match="must not share memory"):
            m.dispatch(rows, plan, out=out)
    shared = m.Plan(ints[:4].view(4, 1), ints[4:6], ints[6:7], 4)
    for out in (ints[3:7].view(4, 1), ints[5:9].view(4, 1), ints[6:10].view(4, 1)):
        with pytest.raises(RuntimeError, match="must not share memory"):
            m.dispatch(torch.zeros(4, 1, dtype=torch.int32), shared, out=out)
    with pytest.raises(RuntimeError, match="on a GPU"):                # beside each other is fine
        m.dispatch(x[:4], plan, out=x[5:9])


@pytest.mark.gpu
def test_dispatch_beside_its_rows(native):
    """Rows that are columns of a wider buffer, and a result that lies between or behind them."""
    torch = _torch()
    from spnc import mixture as m
    base = torch.randn(4, 64, device="cuda")
    want = base[:, :4].clone()
    assert torch.equal(m.dispatch(base[:, :4], _plan(), out=base.view(-1)[32:48].view(4, 4)), want)      # in the first row's free part
    with pytest.raises(RuntimeError, match="overlaps an input"):
        m.dispatch(base[:, :4], _plan(), out=base.view(-1)[52:68].view(4, 4))                            # across the second row's beginning
    with pytest.raises(RuntimeError, match="must not share memory"):
        m.dispatch(base[:, :64], _plan(), out=base)
    assert torch.equal(base[:, :4], want)


@pytest.mark.gpu
def test_dropout_between_its_rows_and_in_place(native):
    """Through the C-ABI: the left half of a buffer's columns into the right half, and onto itself."""
    torch = _torch()
    from spnc import mixture as m
    lib, p = native._load(), ctypes.c_void_p
    base = torch.randn(300, 16, device="cuda")
    want = m.dropout(base[:, :8], 0.4, 9, marginal=True).nan_to_num(7.0)
    stream = p(torch.cuda.current_stream().cuda_stream)
    for out in (base[:, 8:], base[:, :8]):
        assert lib.spnc_hip_dropout(p(base.data_ptr()), 0, 300, 8, 16, p(out.data_ptr()), 16, 0.4, 1, 9, 0, None, stream) == 0
        assert torch.equal(out.nan_to_num(7.0), want)


# ---- derivatives that are not offered -------------------------------------------------------------------------------

def test_kernels_refuse_rows_that_want_a_gradient(mix):
    """In the step-by-step form too, whose rows come out of a differentiable dispatch; without a graph they are rows like others."""
    torch = _torch()
    from spnc import mixture as m
    plan = m.Plan(torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 3)
    x = torch.zeros(3, 6, requires_grad=True)
    for rows in (x, x * 2.0):
        with pytest.raises(RuntimeError, match="no gradient with respect to their features"):
            mix.execute(rows, plan)
        with pytest.raises(RuntimeError, match="no gradient with respect to their features"):
            mix.log_likelihood(rows, torch.zeros(3, 2), 1)
        with pytest.raises(RuntimeError, match="on one GPU"), torch.no_grad():
            mix.execute(rows, plan)
        with pytest.raises(RuntimeError, match="on one GPU"):
            mix.execute(rows.detach(), plan)


@pytest.mark.gpu
def test_kernels_step_by_step(mix):
    torch = _torch()
    from spnc import mixture as m
    x, z = torch.randn(50, 6, device="cuda"), torch.randn(50, 2, device="cuda", requires_grad=True)
    index, log_weights = m.gate(z, 2, log=True)
    plan = m.route(index, 2, align=4)
    got = m.combine_log(mix.execute(m.dispatch(x, plan), plan), plan, log_weights)
    want = mix.log_likelihood(x, z, 2)
    assert torch.equal(got, want)
    assert torch.equal(torch.autograd.grad(got.sum(), z)[0], torch.autograd.grad(want.sum(), z)[0])
    leaf = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient with respect to their features"):
        mix.execute(m.dispatch(leaf, plan), plan)
    with torch.no_grad():
        assert torch.equal(m.combine_log(mix.execute(m.dispatch(leaf, plan), plan), plan, log_weights), want)


def _calls(mix, device):
    """(call, a floating-point tensor it takes) of everything that takes one."""
    torch = _torch()
    from spnc import mixture as m
    i32 = dict(dtype=torch.int32, device=device)
    plan = m.Plan(torch.arange(3, **i32)[:, None], torch.tensor([0, 3, 3], **i32), torch.tensor([3, 0], **i32), 3)
    x, v, w, z = (torch.rand(shape, device=device) for shape in ((3, 6), (3,), (3, 1), (3, 2)))
    return [(lambda t: m.gate(t, 2)[1], z), (lambda t: m.gate(t, 1, over="all", log=True)[1], z), (lambda t: m.dispatch(t, plan), x),
            (lambda t: m.dispatch(t, plan, out=torch.empty_like(x)), x), (lambda t: m.dispatch(x, plan, out=t), x.clone()), (lambda t: m.combine(t, plan), x),
            (lambda t: m.combine(t, plan, w), x), (lambda t: m.combine(x, plan, t), w), (lambda t: m.combine_log(t, plan, w), v), (lambda t: m.combine_log(v, plan, t), w),
            (lambda t: m.dropout(t, 0.5, 1), x), (lambda t: m.dropout(t, 0.5, 1, marginal=True), x), (lambda t: mix.execute(t, plan), x),
            (lambda t: mix.log_likelihood(t, z, 1), x), (lambda t: mix.log_likelihood(x, t, 1), z)]


def test_tangents_and_traces_are_refused(mix):
    """Before anything reaches the GPU; the same calls without a tangent or a trace get as far as the device check."""
    torch = _torch()
    from spnc import mixture as m
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx
    for f, t in _calls(mix, "cpu"):
        with pytest.raises(RuntimeError, match="on (a|one) GPU"):
            f(t)
        with forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="on (a|one) GPU"):
                f(t)
            dual = forward_ad.make_dual(t, torch.ones_like(t))
            for _ in range(2):
                with pytest.raises(RuntimeError, match="no forward-mode derivatives"):
                    f(dual)
            with torch.no_grad(), pytest.raises(RuntimeError, match="no forward-mode derivatives"):       # tangents pass through this
                f(dual)
            with pytest.raises(RuntimeError, match="on (a|one) GPU"):
                f(forward_ad.unpack_dual(dual).primal)
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(f, (t,))
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(f, tracing_mode="real")(t)
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(f, tracing_mode="real", pre_dispatch=True)(t)              # as torch.export records
    index = torch.zeros(3, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(lambda t: m.route(t, 2).position, (index,))
    with pytest.raises(RuntimeError, match="on a GPU"):
        m.route(index, 2)


@pytest.mark.gpu
def test_tangents_of_gradients_are_refused(mix):
    """A backward pass whose incoming gradient has a tangent; wrapped tensors (torch.func) are refused by PyTorch."""
    torch = _torch()
    from torch.autograd import forward_ad
    differentiable = [c for i, c in enumerate(_calls(mix, "cuda")) if i not in (3, 4, 12, 13)]
    for i, (f, t) in enumerate(differentiable):
        leaf = t.clone().requires_grad_()
        out = f(leaf)
        want, = torch.autograd.grad(out, leaf, torch.ones_like(out), retain_graph=True)
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(RuntimeError, match="no forward-mode derivatives"):
                torch.autograd.grad(out, leaf, dual, retain_graph=True)
            got, = torch.autograd.grad(out, leaf, torch.ones_like(out))
        assert torch.equal(got, want), i
        for transform in (lambda: torch.vmap(f)(t[None]), lambda: torch.func.grad(lambda a: f(a).sum())(t), lambda: torch.func.jvp(f, (t,), (torch.ones_like(t),))):
            with pytest.raises(RuntimeError):
                transform()


# ---- errors of other calls ------------------------------------------------------------------------------------------

def _runtime():
    torch = _torch()
    return ctypes.CDLL(os.path.join(os.path.dirname(torch.__file__), "lib", "libamdhip64.so"))        # the runtime both use


@pytest.mark.gpu
def test_c_entry_points_leave_a_foreign_error_to_its_reader(native):
    """A failed call (a device that does not exist) before each entry point: they succeed, and its code can still be read afterwards."""
    torch = _torch()
    from spnc import mixture as m
    lib, p, hip = native._load(), ctypes.c_void_p, _runtime()
    z, x = torch.randn(5, 7, device="cuda"), torch.randn(5, 4, device="cuda")
    index, weight = m.gate(z, 2)
    plan = m.route(index, 7)
    rows, logs, lls = m.dispatch(x, plan), weight.log(), torch.randn(10, device="cuda")
    joined, mixed = m.combine(rows, plan, weight), m.combine_log(lls, plan, logs)
    dropped = m.dropout(x, 0.5, 3)
    outs = [torch.empty_like(t) for t in (index, weight, z, plan.position, plan.starts, plan.counts, rows, joined, rows, weight, mixed, weight, lls, logs, dropped)]
    gi, gw, gz, rp, rs, rc, dr, cj, cv, cw, lm, ls, lv, lw, do = outs
    at = lambda t: p(t.data_ptr())
    stream = p(torch.cuda.current_stream().cuda_stream)
    calls = [lambda: lib.spnc_hip_gate(at(z), 0, 5, 7, 7, 2, 0, at(gi), at(gw), stream),
             lambda: lib.spnc_hip_gate_backward(at(z), 0, 5, 7, 7, 2, 0, at(index), at(weight), at(weight), at(gz), stream),
             lambda: lib.spnc_hip_route(at(index), 10, 7, 1, at(rp), at(rs), at(rc), None, 0, stream),
             lambda: lib.spnc_hip_dispatch(at(x), 5, 16, 16, at(plan.position), 2, 10, at(plan.starts), at(plan.counts), 7, 1, at(dr), stream),
             lambda: lib.spnc_hip_combine(at(rows), 0, 10, 4, 4, at(plan.position), 5, 2, at(weight), 0, at(cj), stream),
             lambda: lib.spnc_hip_combine_backward(at(rows), 0, 10, 4, 4, at(plan.position), 5, 2, at(weight), 0, at(joined), 4, at(plan.starts), at(plan.counts), 7,
                                                   at(cv), at(cw), stream),
             lambda: lib.spnc_hip_combine_log(at(lls), 0, 10, at(plan.position), 5, 2, at(logs), 0, at(lm), at(ls), stream),
             lambda: lib.spnc_hip_combine_log_backward(at(ls), 0, 10, at(plan.position), 5, 2, 0, at(mixed), at(plan.starts), at(plan.counts), 7, at(lv), at(lw), stream),
             lambda: lib.spnc_hip_dropout(at(x), 0, 5, 4, 4, at(do), 4, 0.5, 0, 3, 0, None, stream)]
    torch.cuda.synchronize()
    for call in calls:
        assert hip.hipSetDevice(ctypes.c_int(9999)) != 0
        left = hip.hipPeekAtLastError()
        assert left != 0 and call() == 0
        assert hip.hipGetLastError() == left and hip.hipPeekAtLastError() == 0
    for got, want in ((gi, index), (gw, weight), (rp, plan.position), (rs, plan.starts), (rc, plan.counts), (dr, rows), (cj, joined), (lm, mixed), (do, dropped)):
        assert torch.equal(got, want)


@pytest.mark.gpu
def test_python_calls_tell_of_a_foreign_error(native, capfd):
    """PyTorch raises whatever error it finds at its next launch; the call says where it was found and goes on."""
    torch = _torch()
    from spnc import mixture as m
    z, hip = torch.randn(4, 6, device="cuda"), _runtime()
    want = m.gate(z, 2)
    torch.cuda.synchronize()
    capfd.readouterr()
    assert hip.hipSetDevice(ctypes.c_int(9999)) != 0
    got = m.gate(z, 2)
    assert hip.hipPeekAtLastError() == 0
    assert "left an error behind: invalid device ordinal" in capfd.readouterr().err
    m.gate(z, 2)
    assert "left an error" not in capfd.readouterr().err
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---- limits ---------------------------------------------------------------------------------------------------------

def test_slots_must_be_below_two_to_the_31(native):
    """n * k of exactly 2^31 is refused by everything that takes slots, as the message says; before anything reaches the GPU."""
    lib, p = native._load(), [ctypes.c_void_p(i << 40) for i in range(1, 9)]
    for n, k in ((1 << 31, 1), (1 << 30, 2), (1 << 28, 8), (715827883, 3)):
        _refused(lib, lib.spnc_hip_dispatch(p[0], n, 4, 4, p[1], k, 4, None, None, 0, 0, p[2], None), "n * k must be below 2^31")
        _refused(lib, lib.spnc_hip_combine(p[0], 0, 4, 4, 4, p[1], n, k, p[2], 0, p[3], None), "n * k must be below 2^31")
        _refused(lib, lib.spnc_hip_combine_backward(p[0], 0, 4, 4, 4, p[1], n, k, p[2], 0, p[3], 4, None, None, 0, None, p[4], None), "n * k must be below 2^31")
        _refused(lib, lib.spnc_hip_combine_log(p[0], 0, 4, p[1], n, k, p[2], 0, p[3], None, None), "n * k must be below 2^31")
        _refused(lib, lib.spnc_hip_combine_log_backward(p[0], 0, 4, p[1], n, k, 0, p[2], None, None, 0, None, p[3], None), "n * k must be below 2^31")
    # one fewer is no such error: the capacity is the next check
    for n, k in (((1 << 31) - 1, 1), ((1 << 30) - 1, 2), (715827882, 3)):
        _refused(lib, lib.spnc_hip_dispatch(p[0], n, 4, 4, p[1], k, 1 << 31, None, None, 0, 0, p[2], None), "the capacity must be below 2^31")
