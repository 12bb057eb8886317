"""gated_delta_rule_varlen_fn against the recurrence in float64."""
import pytest
import torch

import gdr_ref
from conftest import DT

pytestmark = pytest.mark.gpu

# The chunked form multiplies with every factor split into bf16 pieces down to 2^-24 (the inputs
# are exact pieces) and adds in fp32: per token sums of 128 terms with unit vectors, and within a
# chunk sums of 64 terms through the triangular inverse, whose entries stay of order one for keys of
# unit length and beta <= 1.  (128 + 2 * 64) * 2^-24 = 1.5e-5 of the largest value.  The 16-bit
# output takes two pieces of the state and of the attention matrix: 2 * 2^-17 = 1.5e-5 more.
TOL = 2e-5
TOL_OUT16 = 4e-5


def expect(q, k, v, g, beta, cu, states, rows, has, scale):
    q, k, v, g, beta = (t.double().cpu() for t in (q, k, v, g, beta))
    states = None if states is None else states.double().cpu().clone()
    hv, dk, dv = v.shape[1], q.shape[2], v.shape[2]
    out = torch.zeros_like(v)
    for n in range(len(cu) - 1):
        a, b = cu[n], cu[n + 1]
        r = -1 if states is None else n if rows is None else int(rows[n])
        r = r if states is not None and 0 <= r < states.shape[0] else -1
        S = torch.zeros(hv, dk, dv, dtype=torch.float64)
        if r >= 0 and (has is None or bool(has[n])):
            S = states[r].clone()
        out[a:b], S = gdr_ref.rule(q[a:b], k[a:b], v[a:b], g[a:b], beta[a:b], S, scale)
        if r >= 0:
            states[r] = S
    return out, states


def check(lens, hk, hv, dk, dv, dtype, tail=0, seed=0, **kw):
    import causal_conv1d_b200 as cc
    total = sum(lens) + tail
    q, k, v, g, beta = gdr_ref.inputs((total,), hk, hv, dk, dv, dtype, seed=seed, **kw)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    n = len(lens)
    gen = torch.Generator().manual_seed(seed + 5)
    states = torch.randn(n + 2, hv, dk, dv, generator=gen).cuda()
    rows = torch.randperm(n + 2, generator=gen)[:n].to(torch.int32)
    if n > 3:
        rows[1], rows[2] = -1, n + 2
    has = torch.rand(n, generator=gen) < 0.6
    want, wstates = expect(q, k, v, g, beta, cu, states, rows, has, dk ** -0.5)
    got = cc.gated_delta_rule_varlen_fn(q, k, v, g, beta, cu_seqlens=torch.tensor(cu, dtype=torch.int32).cuda(), states=states,
                                        state_indices=rows.cuda(), has_initial_state=has.cuda())
    gdr_ref.close(got, want, TOL if dtype == torch.float32 else TOL_OUT16, "out", dtype)
    gdr_ref.close(states, wstates, TOL, "states")
    if tail:
        assert not got[-tail:].any()


def test_one_chunk_one_head():
    check([64], 1, 1, 128, 128, torch.bfloat16)


def test_two_chunks():
    check([128], 1, 1, 128, 128, torch.bfloat16)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("lens,hk,hv,dk,dv,tail", [([1], 1, 1, 128, 128, 0), ([64, 63, 65], 1, 2, 128, 128, 0),
                                                   ([5, 0, 200, 1, 129], 2, 2, 64, 128, 3), ([300], 2, 6, 128, 64, 70),
                                                   ([33, 190], 1, 3, 8, 8, 0), ([100, 28], 2, 2, 96, 72, 1),
                                                   ([0, 0], 1, 1, 32, 32, 9), ([1000], 1, 1, 120, 104, 0)])
def test_varlen(dtype, lens, hk, hv, dk, dv, tail):
    check(lens, hk, hv, dk, dv, DT[dtype], tail, seed=sum(lens) + dv)


def test_many_sequences_more_than_resident():
    check([(37 * i) % 150 for i in range(60)], 2, 4, 64, 64, torch.bfloat16)


def test_slow_decay_long():
    check([3000], 1, 2, 128, 128, torch.bfloat16, slow=True)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("lens", [[4000], [64 * 40, 1, 64 * 17 + 1, 0, 900, 64 * 13 - 1]])
def test_long_sequences_of_few_heads(dtype, lens):
    """Cut into segments that are walked side by side, with states that last through all of them."""
    check(lens, 1, 2, 96, 72, DT[dtype], 3, slow=True, seed=len(lens))
