"""Calls of spnc.mixture and of its C-ABI that are out of the ordinary: buffers that are used again or shared, views whose memory does not
hold their values, kinds of derivatives that are not offered, errors of other calls."""
import os

import pytest

from conftest import quiet


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
