"""Inputs and output gradients whose rows share memory (stride 0, as expand() and the gradients of sums make them): every result
as with a dense copy."""
import pytest
import torch

from conftest import DT, assert_close_sum

pytestmark = pytest.mark.gpu


def run(x, w, b, dout, checkpoint):
    import causal_conv1d_b200 as cc
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    out = cc.causal_conv1d_fn(*leaves, activation="silu", checkpoint=checkpoint)
    return (out.detach(), *torch.autograd.grad(out, leaves, dout))


def dense(t, channel_last):
    return t.transpose(1, 2).contiguous().transpose(1, 2).clone() if channel_last else t.contiguous().clone()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("channel_last", [False, True])
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
@pytest.mark.parametrize("which,along", [("x", 0), ("x", 1), ("x", 2), ("x", None), ("dout", 0), ("dout", 1), ("dout", 2), ("dout", None)])
def test_expanded(dtype, channel_last, checkpoint, which, along):
    B, D, L = 3, 64, 100
    gen = torch.Generator().manual_seed(3)
    full = {n: torch.randn(B, D, L, generator=gen).to(DT[dtype]).cuda() for n in ("x", "dout")}
    full = {n: dense(t, channel_last) for n, t in full.items()}
    t = full[which]
    for d in range(3) if along is None else [along]:
        t = t.narrow(d, 0, 1).expand(*[(B, D, L)[i] if i == d else -1 for i in range(3)])
    assert t.shape == (B, D, L) and 0 in t.stride()
    w = torch.randn(D, 4, generator=gen).to(DT[dtype]).cuda()
    b = torch.randn(D, generator=gen).to(DT[dtype]).cuda()
    got = run(**{"x": full["x"], "dout": full["dout"], which: t}, w=w, b=b, checkpoint=checkpoint)
    # an x without a contiguous axis is taken as channel-first
    last = channel_last if which == "dout" else t.stride(1) == 1 and t.stride(2) > 1
    want = run(**{"x": full["x"], "dout": full["dout"], which: dense(t, last)}, w=w, b=b, checkpoint=checkpoint)
    # another kernel may serve them: fp32 sums in another order, a 16-bit result at most a step away
    step = torch.finfo(DT[dtype]).eps
    for name, a, c in zip(("out", "dx", "dw", "db"), got, want):
        assert_close_sum(a, c, max(step, 1e-6), name)


@pytest.mark.parametrize("reduce", [lambda o: o.sum(0), lambda o: o.mean(-1), lambda o: o.sum(1)])
def test_gradient_of_a_sum(reduce):
    """out.sum(0) hands back one (dim, seqlen) for all rows of the batch."""
    import causal_conv1d_b200 as cc
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(4, 130, 96, generator=gen).bfloat16().cuda().transpose(1, 2).requires_grad_()
    w = torch.randn(96, 4, generator=gen).bfloat16().cuda().requires_grad_()
    got = torch.autograd.grad(reduce(cc.causal_conv1d_fn(x, w, None)).float().square().sum(), (x, w))
    out = cc.causal_conv1d_fn(x, w, None)
    dout = torch.autograd.grad(reduce(out).float().square().sum(), out, retain_graph=True)[0]
    want = torch.autograd.grad(out, (x, w), dense(dout, True))
    for a, c in zip(got, want):
        assert_close_sum(a, c, 2.0 ** -7)
