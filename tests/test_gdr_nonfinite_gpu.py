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
