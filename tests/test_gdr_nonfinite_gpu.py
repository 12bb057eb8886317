"""Infinities, NaN and overflow in the gated delta rule: which outputs and gradients they reach, and which stay as they are."""
import pytest
import torch

import gdr_ref
from conftest import DT

pytestmark = pytest.mark.gpu


def large_keys(k, at, head, size=1e20):
    """Tokens at .. at + 3 with one direction of length `size`: at 1e20 their products with each other leave float32."""
    k[..., at:at + 4, head, :] = size * k[..., at:at + 1, head, :].clone()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_keys_whose_products_overflow(dtype):
    """k_i.k_j is infinite though k, v and the first product with the state are not."""
    import causal_conv1d_b200 as cc
    q, k, v, g, beta = gdr_ref.inputs((64,), 2, 2, 32, 32, DT[dtype], seed=12)
    cu = torch.tensor([0, 64], dtype=torch.int32).cuda()
    clean = cc.gated_delta_rule_varlen_fn(q, k, v, g, beta, cu_seqlens=cu)
    large_keys(k, 30, 1)
    got = cc.gated_delta_rule_varlen_fn(q, k, v, g, beta, cu_seqlens=cu)
    assert torch.equal(got[:, 0], clean[:, 0]) and torch.equal(got[:30, 1], clean[:30, 1])
    assert not torch.isfinite(got[31:, 1]).any()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_what_a_token_writes_overflows(dtype):
    """Keys of 1e19 over a state of order one: T and R are finite, T R is not, and the tokens before keep their bits."""
    import causal_conv1d_b200 as cc
    q, k, v, g, beta = gdr_ref.inputs((64,), 2, 2, 32, 32, DT[dtype], seed=14, slow=True)
    cu = torch.tensor([0, 64], dtype=torch.int32).cuda()
    first = torch.randn(1, 2, 32, 32, generator=torch.Generator().manual_seed(15)).cuda()
    run = lambda: cc.gated_delta_rule_varlen_fn(q, k, v, g, beta, cu_seqlens=cu, states=first, update_states=False)  # noqa: E731
    clean = run()
    large_keys(k, 30, 1, 1e19)
    got = run()
    assert torch.equal(got[:, 0], clean[:, 0]) and torch.equal(got[:30, 1], clean[:30, 1])
    assert not torch.isfinite(got[32:, 1]).any()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_overflow_passes_from_segment_to_segment(dtype):
    """A long sequence of few heads is walked in segments: the ones behind the overflow know of it, and the last state."""
    import causal_conv1d_b200 as cc
    q, k, v, g, beta = gdr_ref.inputs((4000,), 2, 2, 64, 32, DT[dtype], seed=13, slow=True)
    cu = torch.tensor([0, 4000], dtype=torch.int32).cuda()

    def run(k):
        states = torch.zeros(1, 2, 64, 32, device="cuda")
        return cc.gated_delta_rule_varlen_fn(q, k, v, g, beta, cu_seqlens=cu, states=states), states

    clean, state = run(k)
    large_keys(k, 1000, 1)
    got, last = run(k)
    assert torch.equal(got[:, 0], clean[:, 0]) and torch.equal(got[:1000, 1], clean[:1000, 1]) and torch.equal(last[:, 0], state[:, 0])
    assert not torch.isfinite(got[1001:, 1]).any() and not torch.isfinite(last[:, 1]).any()


NAMES = ["dq", "dk", "dv", "dg", "dbeta"]


def gradients(leaves, S0, cu, dout, dfinal):
    import causal_conv1d_b200 as cc
    every = [t.detach().requires_grad_() for t in (*leaves, S0)]
    out, last = cc.gated_delta_rule_fn(*every[:5], initial_state=every[5], return_final_state=True, cu_seqlens=cu)
    return torch.autograd.grad((out, last), every, (dout, dfinal))


def training(T, hk, hv, dtype, seed, tail_from=None):
    """A sequence of T tokens and one of 20 behind it; tail_from: a padded end without an output's gradient."""
    leaves = gdr_ref.inputs((1, T + 20), hk, hv, 64, 32, DT[dtype], seed=seed, slow=True)
    gen = torch.Generator().manual_seed(seed)
    S0, dfinal = (torch.randn(2, hv, 64, 32, generator=gen).cuda() for _ in range(2))
    dout = torch.randn(1, T + 20, hv, 32, generator=gen).to(DT[dtype]).cuda()
    if tail_from is not None:
        dout[:, tail_from:T] = 0
        dfinal[0] = 0
    return leaves, S0, torch.tensor([0, T, T + 20], dtype=torch.int32).cuda(), dout, dfinal


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype,T,t,tail", [("bf16", 64, 30, False), ("fp32", 200, 64, False), ("fp16", 200, 127, True), ("bf16", 150, 100, True),
                                            ("bf16", 90, 0, False), ("bf16", 2500, 1300, True)])
def test_a_value_that_is_not_finite_leaves_the_gradients_before_it(value, dtype, T, t, tail):
    """v of one token and column.  What the recurrence sends back (dS, dB) is made of q, k, g, beta and the outputs' gradients
    alone, so neither dv nor the first state's gradient depends on v, nor does any gradient of a token before: they are those
    of the run with a finite value there.  From the token on the gradients of q, k, g and beta are NaN.  2500 tokens are
    walked in segments."""
    leaves, *rest = training(T, 1, 2, dtype, T + t, t if tail else None)
    clean = gradients(leaves, *rest)
    leaves[2][0, t, 1, 5] = value
    got = gradients(leaves, *rest)
    for name, a, c in zip(NAMES, got, clean):
        if name == "dv":
            assert torch.equal(a, c)
            continue
        assert torch.equal(a[0, T:], c[0, T:]), f"{name}: another sequence"
        if name in ("dg", "dbeta"):
            assert torch.equal(a[..., 0], c[..., 0]), f"{name}: another head"
            a, c = a[..., 1], c[..., 1]
        # dg is a sum over the chunk's later tokens too, in which the value's part cancels: equal but for its roundings
        # (at most 64 terms of the size of the largest: 64 * 2^-24 = 4e-6)
        gdr_ref.close(a[0, :t], c[0, :t], 4e-6 if name == "dg" else 0, f"{name} before")
        assert torch.isnan(a[0, t:T]).all(), f"{name}: from the token on"
    assert torch.equal(got[5], clean[5])


@pytest.mark.parametrize("dtype,T,t", [("bf16", 64, 30), ("fp32", 200, 100), ("bf16", 2500, 1300)])
def test_overflowed_keys_in_the_backward(dtype, T, t):
    """Keys whose products leave float32: what goes back through them is not finite, where it does not pass them it is
    as it was (dq of the tokens before, the other head, the other sequence)."""
    leaves, *rest = training(T, 2, 2, dtype, T + t + 1)
    clean = gradients(leaves, *rest)
    large_keys(leaves[1], t, 1)
    got = gradients(leaves, *rest)
    for name, a, c in zip(NAMES, got, clean):
        assert torch.equal(a[0, T:], c[0, T:]), f"{name}: another sequence"
        assert torch.equal(a[0, :, 0], c[0, :, 0]), f"{name}: another head"
        if name == "dq":
            assert torch.equal(a[0, :t, 1], c[0, :t, 1])
        else:
            assert not torch.isfinite(a[0, :t, 1]).any(), f"{name} before"
        if name != "dv":
            assert not torch.isfinite(a[0, t + 1:T, 1]).any(), f"{name} behind"
    assert torch.equal(got[5][0, 0], clean[5][0, 0]) and not torch.isfinite(got[5][0, 1]).any()


def test_a_gate_of_minus_infinity_in_the_backward():
    """-inf forgets the state like any gate that takes e^g to 0: finite gradients, the same bits."""
    leaves, *rest = training(150, 1, 2, "bf16", 7)
    leaves[3][0, [0, 30, 64, 100], 1] = -1000.0
    want = gradients(leaves, *rest)
    leaves[3][0, [0, 30, 64, 100], 1] = -torch.inf
    for a, b in zip(gradients(leaves, *rest), want):
        assert torch.isfinite(a).all() and torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_overflowing_products_of_forgotten_tokens(dtype):
    """Two keys of 1e20, the state forgotten in front of both: their product overflows and means nothing."""
    import causal_conv1d_b200 as cc
    q, k, v, g, beta = gdr_ref.inputs((60,), 1, 2, 32, 32, DT[dtype], seed=16, slow=True)
    for t in (5, 40):
        k[t] *= 1e20
        g[t] = -torch.inf
    got = cc.gated_delta_rule_varlen_fn(q, k, v, g, beta, cu_seqlens=torch.tensor([0, 60], dtype=torch.int32).cuda(), scale=1.0)
    want, _ = gdr_ref.rule(*(t.double().cpu() for t in (q, k, v, g, beta)), torch.zeros(2, 32, 32, dtype=torch.float64), 1.0)
    for part in (slice(0, 5), slice(5, 40), slice(40, 60)):
        gdr_ref.close(got[part], want[part], 4e-5, "out", DT[dtype])
