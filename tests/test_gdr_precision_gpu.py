"""fp32 calls of the gated delta rule keep fp32's precision: bounds below what a lost bf16 piece of a factor leaves."""
import pytest
import torch

import gdr_ref

pytestmark = pytest.mark.gpu


# An fp32 factor is three bf16 pieces; without the third, 2^-17 of it at most and 3e-6 of a tensor's largest value on
# average are lost (in dg, a difference of larger sums, up to 8e-6).  With all three what is left are the sums: the tensor core
# cuts one off at 24 bits after every 16 terms, by 2^-24 of its size on average and always downwards, so n terms cost
# n / 16 * 2^-24.  Four products of dim (or 64) terms follow one another on the way to a gradient: 4 * 4 * 2^-24 for 64,
# twice that for 128, and the sums in registers and the state's own products are given as much again.
@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("dim,T,tol", [(64, 64, 2.0 ** -19), (128, 130, 2.0 ** -18)])
@pytest.mark.parametrize("slow", [False, True])
def test_fp32_calls(seed, dim, T, tol, slow):
    import causal_conv1d_b200 as cc
    leaves = gdr_ref.inputs((1, T), 1, 1, dim, dim, torch.float32, seed=seed, slow=slow)
    gen = torch.Generator().manual_seed(seed + 100)
    S0, dfinal = (torch.randn(1, 1, dim, dim, generator=gen).cuda() for _ in range(2))
    dout = torch.randn(1, T, 1, dim, generator=gen).cuda()
    leaves = [t.requires_grad_() for t in (*leaves, S0)]
    out, last = cc.gated_delta_rule_fn(*leaves[:5], initial_state=S0, return_final_state=True)
    got = (out[0], last[0], *(d[0] for d in torch.autograd.grad((out, last), leaves, (dout, dfinal))))
    wide = [t.detach()[0].double().cpu().requires_grad_() for t in leaves]
    o, S = gdr_ref.rule(*wide, dim ** -0.5)
    want = (o, S, *torch.autograd.grad((o, S), wide, (dout[0].double().cpu(), dfinal[0].double().cpu())))
    for name, a, b in zip(("out", "state", "dq", "dk", "dv", "dg", "dbeta", "dstate"), got, want):
        worst = ((a.detach().double().cpu() - b.detach()).abs().max() / b.abs().max()).item()
        assert worst <= tol, f"{name}: {worst:.2e}"


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,T,tol", [(64, 64, 2.0 ** -19), (128, 130, 2.0 ** -18)])
@pytest.mark.parametrize("slow", [False, True])
def test_fp32_gradients_of_16_bit_calls(seed, dtype, dim, T, tol, slow):
    """dg, dbeta (of fp32 gates) and the first state's gradient are fp32 there too, and inputs of 16 bits are exact: the bounds of
    the fp32 calls.  Two pieces of T - I and of what it is multiplied with in the backward's walks leave 2^-17 of that product."""
    import causal_conv1d_b200 as cc
    leaves = gdr_ref.inputs((1, T), 1, 4, dim, dim, dtype, bdtype=torch.float32, seed=seed, slow=slow)
    gen = torch.Generator().manual_seed(seed + 100)
    S0, dfinal = (torch.randn(1, 4, dim, dim, generator=gen).cuda() for _ in range(2))
    dout = torch.randn(1, T, 4, dim, generator=gen).to(dtype).cuda()
    leaves = [t.requires_grad_() for t in (*leaves, S0)]
    out, last = cc.gated_delta_rule_fn(*leaves[:5], initial_state=S0, return_final_state=True)
    got = torch.autograd.grad((out, last), leaves[3:], (dout, dfinal))
    wide = [t.detach()[0].double().cpu().requires_grad_() for t in leaves]
    o, S = gdr_ref.rule(*wide, dim ** -0.5)
    want = torch.autograd.grad((o, S), wide[3:], (dout[0].double().cpu(), dfinal[0].double().cpu()))
    for name, a, b in zip(("dg", "dbeta", "dstate"), got, want):
        worst = ((a[0].double().cpu() - b).abs().max() / b.abs().max()).item()
        assert worst <= tol, f"{name}: {worst:.2e}"
