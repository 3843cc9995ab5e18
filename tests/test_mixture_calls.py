"""Calls of spnc.mixture and of its C-ABI that are out of the ordinary: buffers that are used again or shared, views whose memory does not
hold their values, kinds of derivatives that are not offered, errors of other calls."""
import pytest


def _torch():
    import torch
    return torch


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
