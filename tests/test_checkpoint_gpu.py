"""causal_conv1d_fn(..., checkpoint="e4m3"): the kept values bit for bit, the output as without, and the
gradients as those of the convolution of the kept values."""
import pytest
import torch

import oracle
from conftest import DT, TOL, assert_close, assert_close_sum

pytestmark = pytest.mark.gpu


def kept(x, channel_last):
    """x as the checkpoint stands for it, in float64 on the CPU, from the definition."""
    x = x.detach().double().cpu()
    rows = x.mT if channel_last else x
    n = rows.shape[-1]
    g = torch.nn.functional.pad(rows, (0, -n % 32)).unflatten(-1, (-1, 32))
    most = g.abs().amax(-1, keepdim=True)
    # least e with most / 2^e <= 448; e is at least -126
    e = torch.ceil(torch.log2(torch.where(most > 0, most, torch.full_like(most, 448.0)) / 448)).clamp(min=-126)
    v = g / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -30))).clamp(min=-6) - 3)
    v = torch.round(v / step) * step * torch.exp2(e)
    v = v.flatten(-2)[..., :n]
    return v.mT if channel_last else v


def make(B, D, L, dtype, channel_last, seed=0, spread=True):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(B, L, D, generator=gen) if channel_last else torch.randn(B, D, L, generator=gen)
    if spread:        # groups of very different size, zeros, values on the border of a scale
        x = x * torch.exp(2 * torch.randn(x.shape[:-1], generator=gen)).unsqueeze(-1)
        x.view(-1)[::7] = 0
        x.view(-1)[::5] *= 1e-3
        if x.shape[-1] >= 64:
            x[0, 0, :32] = 0
            x[0, 0, 32:64] = 448.0
    x = x.to(dtype).cuda()
    return x.transpose(1, 2) if channel_last else x


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("channel_last,B,D,L", [(False, 2, 3, 333), (False, 2, 5, 1024), (False, 1, 4, 48), (False, 3, 2, 1), (True, 2, 40, 17),
                                                (True, 1, 64, 100), (True, 2, 8, 1), (False, 1, 2, 4112)])
def test_codes_are_the_definitions(dtype, channel_last, B, D, L):
    from causal_conv1d_b200.cpp_functions import causal_conv1d_fwd_e4m3_function
    x = make(B, D, L, DT[dtype], channel_last, seed=L)
    w, b = torch.randn(D, 4, device="cuda"), torch.randn(D, device="cuda")
    out, codes, scales = causal_conv1d_fwd_e4m3_function(x, w, b, None, None, None, True)
    values = codes.view(torch.float8_e4m3fn).double()
    groups = torch.exp2(scales.double() - 127).repeat_interleave(32, -1)[..., : codes.shape[-1]]
    got = (values * groups).cpu()
    want = kept(x, channel_last)
    assert torch.equal(got.mT if channel_last else got, want)
    from causal_conv1d_b200 import causal_conv1d_fn
    assert torch.equal(out, causal_conv1d_fn(x, w, b, activation="silu"))


@pytest.mark.parametrize("activation", ["silu", None])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("channel_last,B,D,L,W", [(False, 2, 72, 333, 4), (False, 2, 40, 2048, 4), (False, 3, 24, 1040, 3), (False, 2, 16, 16, 2),
                                                  (False, 1, 8, 8208, 4), (True, 2, 72, 211, 4), (True, 1, 136, 1000, 2), (False, 2, 8, 1, 4)])
def test_gradients(activation, dtype, channel_last, B, D, L, W):
    """The gradient of the convolution at the kept x: the gates of the backward without a checkpoint."""
    from causal_conv1d_b200 import causal_conv1d_fn
    x = make(B, D, L, DT[dtype], channel_last, seed=D + L, spread=False).requires_grad_()
    w = (torch.rand(D, W, device="cuda") - 0.5).requires_grad_()
    b = (torch.rand(D, device="cuda") - 0.5).requires_grad_()
    out = causal_conv1d_fn(x, w, b, activation=activation, checkpoint="e4m3")
    dout = torch.randn_like(out)
    dx, dw, db = torch.autograd.grad(out, (x, w, b), dout)
    assert dx.stride() == x.stride() or B == 1 or L == 1
    at = kept(x, channel_last).float()       # exact: 4 significant bits
    if channel_last:
        at = at.mT.contiguous().mT
    want = oracle.bwd(at, w, b, dout.float(), activation=activation)
    assert_close(dx, want["dx"].to(DT[dtype]), TOL[DT[dtype]], "dx")
    assert_close_sum(dw, want["dweight"], TOL[DT[dtype]], "dweight")
    assert_close_sum(db, want["dbias"], TOL[DT[dtype]], "dbias")


def test_same_bits_as_the_backward_of_the_kept_x():
    """Read from the codes or restored first, the arithmetic is that of the plain backward."""
    from causal_conv1d_b200 import causal_conv1d_fn
    for channel_last, dtype, L in ((False, torch.bfloat16, 2048), (False, torch.float16, 1040), (False, torch.float32, 100), (True, torch.bfloat16, 300)):
        x = make(2, 64, L, dtype, channel_last, spread=False)
        at = kept(x, channel_last).to(dtype).cuda()
        at = (at.mT.contiguous().mT if channel_last else at.contiguous()).requires_grad_()
        x.requires_grad_()
        w = (torch.rand(64, 4, device="cuda") - 0.5).requires_grad_()
        b = (torch.rand(64, device="cuda") - 0.5).requires_grad_()
        dout = torch.randn_like(x)
        got = torch.autograd.grad(causal_conv1d_fn(x, w, b, activation="silu", checkpoint="e4m3"), (x, w, b), dout)
        want = torch.autograd.grad(causal_conv1d_fn(at, w, b, activation="silu"), (at, w, b), dout)
        for a, c in zip(got, want):
            assert torch.equal(a, c), (channel_last, dtype)


def test_packed_states_and_the_other_layout_of_dout():
    from causal_conv1d_b200 import causal_conv1d_fn
    B, D, L = 2, 64, 150
    x = make(B, D, L, torch.bfloat16, True, spread=False).requires_grad_()
    w, b = (torch.rand(D, 4, device="cuda") - 0.5).requires_grad_(), (torch.rand(D, device="cuda") - 0.5).requires_grad_()
    at = kept(x, True).to(torch.bfloat16).cuda().mT.contiguous().mT.requires_grad_()
    dout = torch.randn(B, D, L, device="cuda").bfloat16()          # channel-first beside a channel-last x
    seq = torch.sort(torch.randint(0, 5, (B, L), device="cuda", dtype=torch.int32), dim=1).values
    got = torch.autograd.grad(causal_conv1d_fn(x, w, b, seq_idx=seq, activation="silu", checkpoint="e4m3"), (x, w, b), dout)
    want = torch.autograd.grad(causal_conv1d_fn(at, w, b, seq_idx=seq, activation="silu"), (at, w, b), dout)
    for a, c in zip(got, want):
        assert torch.equal(a, c)
    init = torch.randn(B, 3, D, device="cuda").bfloat16().transpose(1, 2).requires_grad_()
    dfin = torch.randn(B, D, 3, device="cuda").bfloat16()

    def run(x, **kw):
        out, fin = causal_conv1d_fn(x, w, b, initial_states=init, return_final_states=True, activation="silu", **kw)
        return torch.autograd.grad((out, fin), (x, w, b, init), (dout, dfin))

    for a, c in zip(run(x, checkpoint="e4m3"), run(at)):
        assert torch.equal(a, c)


def test_memory_strides_and_what_is_not_finite():
    from causal_conv1d_b200 import causal_conv1d_fn
    D, L = 32, 128
    wide = torch.randn(2, D, 2 * L, device="cuda").bfloat16()
    x = wide[:, :, 64:64 + L].detach().requires_grad_()      # a window of a wider buffer
    w = torch.rand(D, 4, device="cuda").requires_grad_()
    out = causal_conv1d_fn(x, w, None, activation="silu", checkpoint="e4m3")
    assert all(t.dtype == torch.uint8 or t.numel() < D * L for t in out.grad_fn.saved_tensors if t is not None)
    dx, dw = torch.autograd.grad(out, (x, w), torch.ones_like(out))
    at = kept(x, False).bfloat16().cuda().requires_grad_()
    want = torch.autograd.grad(causal_conv1d_fn(at, w, None, activation="silu"), (at, w), torch.ones_like(out))
    assert torch.equal(dx, want[0]) and torch.equal(dw, want[1])
    bad = torch.zeros(1, D, L, device="cuda").bfloat16()
    bad[0, 3, 40], bad[0, 5, 0] = torch.inf, torch.nan
    bad.requires_grad_()
    dw = torch.autograd.grad(causal_conv1d_fn(bad, w, None, checkpoint="e4m3"), w, torch.ones(1, D, L, device="cuda").bfloat16())[0]
    assert torch.isnan(dw[3]).all() and torch.isnan(dw[5]).all() and torch.isfinite(dw[[0, 1, 2, 4] + list(range(6, D))]).all()
    big = torch.full((1, 8, 64), 65504.0, device="cuda").half().requires_grad_()
    w8 = torch.full((8, 4), 1e-4, device="cuda").requires_grad_()
    dw = torch.autograd.grad(causal_conv1d_fn(big, w8, None, checkpoint="e4m3"), w8, torch.full_like(big, 1e-6))[0]
    assert torch.isfinite(dw).all()


def test_refusals():
    from causal_conv1d_b200 import causal_conv1d_fn
    x = torch.randn(1, 8, 16, device="cuda")
    w = torch.randn(8, 4, device="cuda")
    with pytest.raises(NotImplementedError, match="checkpoint must be None or e4m3"):
        causal_conv1d_fn(x, w, checkpoint="e5m2")
    with pytest.raises(RuntimeError, match="channel last"):
        causal_conv1d_fn(x, w, seq_idx=torch.zeros(1, 16, dtype=torch.int32, device="cuda"), checkpoint="e4m3")
    assert causal_conv1d_fn(torch.empty(0, 8, 16, device="cuda"), w, checkpoint="e4m3").shape == (0, 8, 16)


def test_in_front_of_the_delta_rule():
    """The run a layer makes: convolution with its input in 8 bits, q, k and v out of its output, the delta rule;
    forward and backward against the same in float64."""
    import causal_conv1d_b200 as cc
    import gdr_ref
    B, T, hk, hv, dk, dv = 1, 90, 1, 2, 32, 32
    dim = 2 * hk * dk + hv * dv
    x = make(B, dim, T, torch.bfloat16, True, spread=False).requires_grad_()
    w = (torch.rand(dim, 4, device="cuda") - 0.5).bfloat16().requires_grad_()
    g, beta = (t.requires_grad_() for t in (-torch.rand(B, T, hv, device="cuda"), torch.rand(B, T, hv, device="cuda").bfloat16()))
    dout = torch.randn(B, T, hv, dv, device="cuda").bfloat16()

    def layer(x, w, g, beta, conv, rule):
        q, k, v = conv(x, w).transpose(1, 2).split([hk * dk, hk * dk, hv * dv], -1)
        q, k = (torch.nn.functional.normalize(t.unflatten(-1, (hk, dk)), dim=-1) for t in (q, k))
        return rule(q, k, v.unflatten(-1, (hv, dv)), g, beta)

    def conv64(x, w):
        taps = torch.nn.functional.pad(x, (3, 0))
        y = sum(taps[..., j:j + T] * w[:, j, None] for j in range(4))
        return y * torch.sigmoid(y)

    def rule64(q, k, v, g, beta):
        return gdr_ref.rule(q[0], k[0], v[0], g[0], beta[0], torch.zeros(hv, dk, dv).double(), dk ** -0.5)[0][None]

    out = layer(x, w, g, beta, lambda x, w: cc.causal_conv1d_fn(x, w, activation="silu", checkpoint="e4m3"), cc.gated_delta_rule_fn)
    got = torch.autograd.grad(out, (x, w, g, beta), dout)
    wide = [t.detach().double().cpu().requires_grad_() for t in (x, w, g, beta)]
    ref = layer(*wide, conv64, rule64)
    want = torch.autograd.grad(ref, wide, dout.double().cpu())
    # bf16 between the steps (2^-8 each, about eight of them) and x to 4 significant bits (2^-4) in the
    # convolution's gradients, random signs: compared in the 2-norm
    for a, b, tol, name in [(out, ref, 8 * 2 ** -8, "out"), (got[0], want[0], 2 ** -4 + 8 * 2 ** -8, "dx"), (got[1], want[1], 2 ** -4 + 8 * 2 ** -8, "dw"),
                            (got[2], want[2], 8 * 2 ** -8, "dg"), (got[3], want[3], 8 * 2 ** -8, "dbeta")]:
        a, b = a.detach().double().cpu(), b.detach()
        assert (a - b).norm() <= tol * b.norm(), (name, ((a - b).norm() / b.norm()).item())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("B,D,L,W,form", [(1, 48, 333, 4, "packed"), (2, 176, 40, 3, "states"), (1, 272, 1000, 4, "packed"), (3, 16, 9, 2, "states"),
                                          (2, 64, 1, 4, "plain"), (2, 40, 130, 4, "packed"), (2, 160, 523, 4, "window")])
def test_channel_last_in_its_own_kernels(dtype, B, D, L, W, form):
    """Channel-last rows of whole and broken groups, read from the codes (40 channels: restored first): the bits of
    the plain backward of the kept x."""
    from causal_conv1d_b200 import causal_conv1d_fn
    t = DT[dtype]
    x = make(B, D, L, t, True, seed=L, spread=False).requires_grad_()
    at = kept(x, True).to(t).cuda().mT.contiguous().mT.requires_grad_()
    w, b = (torch.rand(D, W, device="cuda") - 0.5).requires_grad_(), (torch.rand(D, device="cuda") - 0.5).requires_grad_()
    dout = torch.randn(B, L, 2 * D, device="cuda").to(t)[..., :D].mT if form == "window" else torch.randn(B, L, D, device="cuda").to(t).mT
    kw, more = {}, ()
    if form == "packed":
        kw["seq_idx"] = torch.sort(torch.randint(0, 6, (B, L), device="cuda", dtype=torch.int32), dim=1).values
    if form == "states":
        init = torch.randn(B, W - 1, D, device="cuda").to(t).mT.requires_grad_()
        kw["initial_states"], more = init, (init,)
    for x_, checkpoint in ((x, "e4m3"), (at, None)):
        out = causal_conv1d_fn(x_, w, b, activation="silu", checkpoint=checkpoint, **kw)
        grads = torch.autograd.grad(out, (x_, w, b, *more), dout)
        if checkpoint:
            got, first = grads, out
    assert torch.equal(first, causal_conv1d_fn(x, w, b, activation="silu", **kw))
    for a, c in zip(got, grads):
        assert torch.equal(a, c)
