"""gated_delta_rule_fn: outputs and gradients against autograd through the recurrence in float64."""
import pytest
import torch

import gdr_ref
from conftest import DT

pytestmark = pytest.mark.gpu

# fp32 factors enter the gradients' products as two bf16 pieces (what is left out: 2^-17 of a factor;
# three pieces for fp32 inputs) and three or four products follow one another: 8 * 2^-17 = 6e-5 of
# the largest value of a tensor. 16-bit gradients add half a step.
TOL = 6e-5
NAMES = ["dq", "dk", "dv", "dg", "dbeta"]


def expect(q, k, v, g, beta, lens, S0, dout, dfinal, scale):
    """Per sequence (tokens a, a + length of the flattened rows)."""
    leaves = [t.detach().double().cpu().flatten(0, 1).requires_grad_() for t in (q, k, v, g, beta)]
    S0 = S0.detach().double().cpu().requires_grad_()
    outs, last, a = [], [], 0
    for n, length in enumerate(lens):
        o, S = gdr_ref.rule(*(t[a:a + length] for t in leaves), S0[n], scale)
        outs.append(o)
        last.append(S)
        a += length
    out, last = torch.cat(outs), torch.stack(last)
    d = dout.double().cpu().flatten(0, 1)[:a]
    loss = (out * d).sum() + (last * dfinal.double().cpu()).sum()
    grads = torch.autograd.grad(loss, leaves + [S0])
    return out.detach(), last.detach(), grads


def check(lens, hk, hv, dk, dv, dtype, packed, tail=0, seed=0, gdtype=torch.float32, bdtype=None, **kw):
    import causal_conv1d_b200 as cc
    total = sum(lens) + tail
    lead = (1, total) if packed else (len(lens), lens[0])
    q, k, v, g, beta = gdr_ref.inputs(lead, hk, hv, dk, dv, dtype, gdtype, bdtype, seed=seed, **kw)
    gen = torch.Generator().manual_seed(seed + 1)
    S0 = torch.randn(len(lens), hv, dk, dv, generator=gen).cuda()
    dfinal = torch.randn(len(lens), hv, dk, dv, generator=gen).cuda()
    dout = torch.randn(v.shape, generator=gen).to(dtype).cuda()
    cu = None
    if packed:
        cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    leaves = [t.requires_grad_() for t in (q, k, v, g, beta, S0)]
    out, last = cc.gated_delta_rule_fn(*leaves[:5], initial_state=S0, return_final_state=True, cu_seqlens=cu)
    got = torch.autograd.grad((out, last), leaves, (dout, dfinal))
    wout, wlast, want = expect(q, k, v, g, beta, lens, S0, dout, dfinal, dk ** -0.5)
    n = sum(lens)
    gdr_ref.close(out.flatten(0, 1)[:n], wout, TOL, "out", dtype)
    gdr_ref.close(last, wlast, TOL, "final state")
    for name, a, b, leaf in zip(NAMES, got, want, leaves):
        gdr_ref.close(a.flatten(0, 1)[:n], b[:n], TOL, name, leaf.dtype)
        if tail:
            assert not a.flatten(0, 1)[n:].any(), name
    gdr_ref.close(got[5], want[5], TOL, "dinitial_state")
    if tail:
        assert not out.flatten(0, 1)[n:].any()
    return leaves, (out, last), got, (dout, dfinal), cu


def test_one_chunk():
    check([64], 1, 1, 128, 128, torch.bfloat16, False)


def test_three_chunks():
    check([150], 1, 1, 128, 128, torch.bfloat16, False)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("lens,hk,hv,dk,dv,packed,tail", [([1], 1, 1, 128, 128, False, 0), ([65, 65], 2, 4, 64, 128, False, 0),
                                                          ([100, 0, 28, 1, 64], 1, 3, 128, 64, True, 5), ([70], 2, 2, 8, 16, False, 0),
                                                          ([130, 3], 1, 2, 96, 72, True, 0), ([200], 2, 2, 120, 104, True, 60)])
def test_gradients(dtype, lens, hk, hv, dk, dv, packed, tail):
    check(lens, hk, hv, dk, dv, DT[dtype], packed, tail, seed=sum(lens) + dk)


@pytest.mark.parametrize("gdtype,bdtype", [("bf16", "fp32"), ("fp16", "bf16")])
def test_gate_types(gdtype, bdtype):
    check([90], 1, 2, 64, 64, torch.bfloat16, False, gdtype=DT[gdtype], bdtype=DT[bdtype])


def test_slow_decay_long():
    check([700], 1, 1, 128, 128, torch.bfloat16, False, slow=True)


def test_without_states_and_run_twice_the_same_bits():
    import causal_conv1d_b200 as cc
    q, k, v, g, beta = (t.requires_grad_() for t in gdr_ref.inputs((2, 130), 2, 4, 64, 64, torch.bfloat16))
    dout = torch.randn(v.shape, device="cuda").bfloat16()
    runs = []
    for _ in range(2):
        out = cc.gated_delta_rule_fn(q, k, v, g, beta)
        runs.append((out.detach(),) + torch.autograd.grad(out, (q, k, v, g, beta), dout))
    for a, b in zip(*runs):
        assert torch.equal(a, b)
    S0 = torch.zeros(2, 4, 64, 64)
    wout, _, want = expect(q, k, v, g, beta, [130, 130], S0, dout, S0, 64 ** -0.5)
    gdr_ref.close(runs[0][0].flatten(0, 1), wout, TOL, "out", torch.bfloat16)
    for name, a, b, leaf in zip(NAMES, runs[0][1:], want, (q, k, v, g, beta)):
        gdr_ref.close(a.flatten(0, 1), b, TOL, name, leaf.dtype)


def test_gradient_against_differences():
    """Directional derivative of a loss by central differences of the GPU forward in float32."""
    import causal_conv1d_b200 as cc
    leaves = [t.requires_grad_() for t in gdr_ref.inputs((1, 80), 1, 2, 32, 32, torch.float32, seed=3)]
    S0 = torch.randn(1, 2, 32, 32, device="cuda").requires_grad_()
    gen = torch.Generator().manual_seed(9)
    dout = torch.randn(1, 80, 2, 32, generator=gen).cuda()
    dlast = torch.randn(1, 2, 32, 32, generator=gen).cuda()

    def loss(args):
        out, last = cc.gated_delta_rule_fn(*args[:5], initial_state=args[5], return_final_state=True)
        return (out.double() * dout).sum() + (last.double() * dlast).sum()

    args = leaves + [S0]
    grads = torch.autograd.grad(loss(args), args)
    for i, grad in enumerate(grads):
        way = torch.randn(args[i].shape, generator=gen).cuda()
        eps = 2.0 ** -7
        with torch.no_grad():
            up = loss([a + eps * way if j == i else a for j, a in enumerate(args)])
            down = loss([a - eps * way if j == i else a for j, a in enumerate(args)])
        slope = ((up - down) / (2 * eps)).item()
        along = (grad.double() * way).sum().item()
        # third-order term of the difference: eps^2 / 6 times a third derivative of the order of the
        # slope's own scale (the norm of the gradient times that of the direction, over its dimension)
        scale = grad.double().norm().item() * way.double().norm().item() / way.numel() ** 0.5
        assert abs(slope - along) <= 0.02 * max(scale, abs(along)), (i, slope, along, scale)


def test_captured_and_replayed_beside_an_eager_graph():
    """Forward and backward captured into a CUDA graph while an eager graph of other leaves lives."""
    import causal_conv1d_b200 as cc
    leaves = [t.requires_grad_() for t in gdr_ref.inputs((1, 100), 1, 2, 64, 64, torch.bfloat16)]
    dout = torch.randn(leaves[2].shape, device="cuda").bfloat16()
    eager = cc.gated_delta_rule_fn(*leaves)
    want = torch.autograd.grad(eager, leaves, dout, retain_graph=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    static = [t.detach().clone().requires_grad_() for t in leaves]
    with torch.cuda.stream(s):
        torch.autograd.grad(cc.gated_delta_rule_fn(*static), static, dout)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cc.gated_delta_rule_fn(*static)
        grads = torch.autograd.grad(out, static, dout)
    for _ in range(2):
        for t in grads:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        for a, b in zip(grads, want):
            assert torch.equal(a, b)
    torch.autograd.grad(eager, leaves, dout)


def test_strided_slices_of_a_conv_output():
    """q, k, v as slices of one (batch, seqlen, dim) tensor, read in place; an expanded gradient."""
    import causal_conv1d_b200 as cc
    B, T, hk, hv, dk, dv = 2, 77, 2, 4, 64, 32
    x = torch.randn(B, T, 2 * hk * dk + hv * dv, device="cuda").bfloat16().requires_grad_()
    g, beta = (-torch.rand(B, T, hv, device="cuda")), torch.rand(B, T, hv, device="cuda").bfloat16()

    def parts(x):
        q, k, v = x.split([hk * dk, hk * dk, hv * dv], -1)
        return (0.1 * q.unflatten(-1, (hk, dk)), torch.nn.functional.normalize(k.unflatten(-1, (hk, dk)).float(), dim=-1).to(x.dtype),
                v.unflatten(-1, (hv, dv)))

    q, k, v = parts(x)
    out = cc.gated_delta_rule_fn(q, k, v, g, beta)
    out.sum().backward()
    want = expect(q, k, v, g, beta, [T] * B, torch.zeros(B, hv, dk, dv), torch.ones(B, T, hv, dv), torch.zeros(B, hv, dk, dv), dk ** -0.5)
    gdr_ref.close(out.flatten(0, 1), want[0], TOL, "out", torch.bfloat16)
    gdr_ref.close(x.grad[..., 2 * hk * dk:].unflatten(-1, (hv, dv)).flatten(0, 1), want[2][2], TOL, "dv", torch.bfloat16)


@pytest.mark.parametrize("dtype,slow", [("bf16", True), ("fp32", True), ("fp16", False)])
def test_long_sequences_of_few_heads(dtype, slow):
    """Cut into segments that are walked side by side: lengths that end inside, at and just behind a segment."""
    check([2048, 1000, 0, 1, 1985], 1, 2, 64, 32, DT[dtype], True, 7, slow=slow, seed=1)


def test_one_long_row():
    check([2500], 1, 1, 128, 128, torch.bfloat16, False, slow=True, seed=2)


def test_gradients_around_forgotten_states():
    """g = -inf and steep decays inside a chunk: finite gradients, those of the tokens behind as without the past."""
    import causal_conv1d_b200 as cc
    leaves = gdr_ref.inputs((1, 140), 1, 1, 64, 64, torch.float32, seed=5)
    leaves[3][0, 30], leaves[3][0, 100], leaves[3][0, 70:80] = -1000.0, -70.0, -20.0
    leaves = [t.requires_grad_() for t in leaves]
    dout = torch.randn(1, 140, 1, 64, device="cuda")
    got = torch.autograd.grad(cc.gated_delta_rule_fn(*leaves), leaves, dout)
    S0 = torch.zeros(1, 1, 64, 64)
    _, _, want = expect(*leaves, [140], S0, dout, S0, 64 ** -0.5)
    for name, a, b in zip(NAMES, got, want):
        gdr_ref.close(a.flatten(0, 1), b, TOL, name)


def test_empty_batches_and_rows():
    import causal_conv1d_b200 as cc
    for B, T in ((0, 5), (2, 0)):
        leaves = [t.requires_grad_() for t in gdr_ref.inputs((B, T), 1, 2, 32, 32, torch.bfloat16)]
        S0 = torch.randn(B, 2, 32, 32, device="cuda").requires_grad_()
        out, last = cc.gated_delta_rule_fn(*leaves, initial_state=S0, return_final_state=True)
        assert out.shape == (B, T, 2, 32) and torch.equal(last, S0)
        d = torch.randn_like(last)
        got = torch.autograd.grad(last, leaves + [S0], d, allow_unused=True)
        assert torch.equal(got[5], d)


@pytest.mark.parametrize("heads", [2, 160])
def test_no_sequence_at_all(heads):
    """cu_seqlens of one entry: every token is behind the last sequence, zero outputs and gradients."""
    import causal_conv1d_b200 as cc
    T = 200
    leaves = [t.requires_grad_() for t in gdr_ref.inputs((1, T), heads // 2, heads, 32, 32, torch.bfloat16)]
    cu = torch.full((1000,), T, dtype=torch.int32, device="cuda")[:1].zero_()      # what follows the entry is not read
    out, last = cc.gated_delta_rule_fn(*leaves, return_final_state=True, cu_seqlens=cu)
    assert last.shape == (0, heads, 32, 32) and not out.any()
    for d in torch.autograd.grad(out, leaves, torch.ones_like(out)):
        assert not d.any()
    pool = torch.randn(3, heads, 32, 32, device="cuda")
    kept = pool.clone()
    out = cc.gated_delta_rule_varlen_fn(*(t.detach()[0] for t in leaves), cu_seqlens=cu, states=pool)
    assert not out.any() and torch.equal(pool, kept)


def test_what_lies_in_the_workspace_does_not_matter():
    """A long sequence of few heads, 72 columns, after memory full of NaN was given back to the allocator."""
    import causal_conv1d_b200 as cc
    leaves = [t.requires_grad_() for t in gdr_ref.inputs((1, 4000), 1, 2, 96, 72, torch.bfloat16, seed=3, slow=True)]
    S0 = torch.randn(1, 2, 96, 72, device="cuda").requires_grad_()
    first = None
    for fill in (0.0, float("nan"), 1e30):
        junk = [torch.full((1 << 25,), fill, device="cuda") for _ in range(4)]
        del junk
        out, last = cc.gated_delta_rule_fn(*leaves, initial_state=S0, return_final_state=True)
        got = (out, last, *torch.autograd.grad((out, last), leaves + [S0], (torch.ones_like(out), torch.ones_like(last))))
        first = first or got
        for a, b in zip(got, first):
            assert torch.isfinite(a).all() and torch.equal(a, b)
