"""gated_delta_rule_update against the recurrence in float64."""
import pytest
import torch

import gdr_ref
from conftest import DT

pytestmark = pytest.mark.gpu

# Every output is a chain of fp32 dot products of at most 128 terms with vectors of unit length:
# 128 * 2^-24 = 7.6e-6 of the largest state column in the worst order, and a handful of tokens
# whose errors add; sums of random signs stay far below.  16-bit outputs add half a step.
TOL = 2e-5


def run(q, k, v, g, beta, state, idx, scale=None):
    import causal_conv1d_b200 as cc
    return cc.gated_delta_rule_update(q, k, v, g, beta, state, state_indices=idx, scale=scale)


def expect(q, k, v, g, beta, state, idx, scale):
    state = state.double().cpu().clone()
    q, k, v, g, beta = (t.double().cpu() for t in (q, k, v, g, beta))
    out = torch.zeros_like(v)
    for b in range(q.shape[0]):
        r = b if idx is None else int(idx[b])
        if r < 0 or r >= state.shape[0]:
            continue
        out[b], state[r] = gdr_ref.rule(q[b], k[b], v[b], g[b], beta[b], state[r], scale)
    return out, state


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("B,T,hk,hv,dk,dv", [(1, 1, 1, 1, 128, 128), (3, 2, 2, 4, 64, 128), (2, 5, 3, 3, 8, 8), (5, 1, 2, 6, 96, 72),
                                             (40, 1, 4, 16, 128, 128), (90, 3, 4, 8, 120, 56), (2, 0, 1, 1, 16, 16)])
def test_update(dtype, B, T, hk, hv, dk, dv):
    q, k, v, g, beta = gdr_ref.inputs((B, T), hk, hv, dk, dv, DT[dtype], seed=B + T)
    state = torch.randn(B + 3, hv, dk, dv, device="cuda")
    idx = torch.randperm(B + 3)[:B].to(torch.int32)
    if B > 2:
        idx[1] = -1
        idx[2] = B + 3          # not a row: padded
    want, wstate = expect(q, k, v, g, beta, state, idx, dk ** -0.5)
    got = run(q, k, v, g, beta, state, idx.cuda())
    gdr_ref.close(got, want, TOL, "out", DT[dtype])
    gdr_ref.close(state, wstate, TOL, "state")
    touched = {int(i) for i in idx if 0 <= int(i) < B + 3} if T else set()
    for r in range(B + 3):
        if r not in touched:
            assert torch.equal(state[r].double().cpu(), wstate[r])


def test_single_token_form_strides_and_gate_types():
    """Slices of one projection (as the conv's output gives them), a pool with gaps between rows and heads."""
    B, hk, hv, dk, dv = 4, 2, 4, 64, 48
    both = torch.randn(B, hk * dk * 2 + hv * dv + 3, device="cuda", dtype=torch.bfloat16)
    q = both[:, 1:1 + hk * dk].unflatten(1, (hk, dk))
    k = torch.nn.functional.normalize(both[:, 1 + hk * dk:1 + 2 * hk * dk].unflatten(1, (hk, dk)).float(), dim=-1).bfloat16()
    v = both[:, 1 + 2 * hk * dk:1 + 2 * hk * dk + hv * dv].unflatten(1, (hv, dv))
    for gt, bt in ((torch.bfloat16, torch.float32), (torch.float16, torch.float16), (torch.float32, torch.bfloat16)):
        g = (-torch.rand(hv, B, device="cuda")).to(gt).t()
        beta = torch.rand(B, hv, device="cuda").to(bt)
        base = torch.randn(B, hv + 1, dk, dv + 0, device="cuda")
        state = base[:, :hv]
        keep = base.clone()
        want, wstate = expect(*(t.unsqueeze(1) for t in (q, k, v, g, beta)), state, None, 0.5)
        got = run(q, k, v, g, beta, state, None, 0.5)
        assert got.shape == (B, hv, dv)
        gdr_ref.close(got, want[:, 0], TOL, "out", torch.bfloat16)
        gdr_ref.close(state, wstate, TOL, "state")
        assert torch.equal(base[:, hv], keep[:, hv])


def test_forgetting_and_extreme_gates():
    """g = -inf and g = -1000 forget the state exactly; beta = 0 leaves it; a NaN token stays in its row."""
    q, k, v, g, beta = gdr_ref.inputs((4, 1), 1, 1, 32, 32, torch.float32)
    g[0], g[1], beta[2], v[3] = -torch.inf, -1000.0, 0.0, torch.nan
    state = torch.randn(4, 1, 32, 32, device="cuda")
    before = state.clone()
    want, wstate = expect(q, k, v, g, beta, state, None, 1.0)
    got = run(q, k, v, g, beta, state, None, 1.0)
    gdr_ref.close(got[:3], want[:3], TOL, "out")
    gdr_ref.close(state[:3], wstate[:3], TOL, "state")
    assert torch.isnan(got[3]).all() and torch.isnan(state[3]).any() and not torch.isnan(state[:3]).any()
    assert torch.allclose(state[2], before[2] * torch.exp(g[2]), rtol=1e-6)


def test_large_pool_offsets_pass_32_bits():
    """A row whose first element lies beyond 2^32 elements (17 GB into the pool)."""
    rows, hv, dk, dv = 1050, 256, 128, 128
    state = torch.empty(rows, hv, dk, dv, device="cuda")
    idx = torch.tensor([rows - 1], dtype=torch.int32, device="cuda")
    state[rows - 1].normal_()
    q, k, v, g, beta = gdr_ref.inputs((1, 1), 1, hv, dk, dv, torch.bfloat16)
    want, ws = expect(q, k, v, g, beta, state[-1:], None, 1.0)
    got = run(q, k, v, g, beta, state, idx, 1.0)
    gdr_ref.close(got, want, TOL, "out", torch.bfloat16)
    gdr_ref.close(state[-1:], ws, TOL, "state")
    del state
    torch.cuda.empty_cache()


def test_captured_and_replayed():
    q, k, v, g, beta = gdr_ref.inputs((6, 1), 2, 4, 64, 64, torch.bfloat16)
    state = torch.randn(9, 4, 64, 64, device="cuda")
    idx = torch.tensor([3, 0, 8, -1, 5, 1], dtype=torch.int32, device="cuda")
    again = state.clone()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        first = run(q, k, v, g, beta, state, idx)
        torch.cuda.synchronize()
        state.copy_(again)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = run(q, k, v, g, beta, state, idx)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    second = state.clone()
    state.copy_(again)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(state, second)


def test_refusals():
    import causal_conv1d_b200 as cc
    q, k, v, g, beta = gdr_ref.inputs((2, 1), 2, 4, 64, 64, torch.bfloat16)
    state = torch.zeros(2, 4, 64, 64, device="cuda")
    call = lambda **kw: cc.gated_delta_rule_update(**{**dict(q=q, k=k, v=v, g=g, beta=beta, state=state), **kw})  # noqa: E731
    for kw, text in ((dict(state=state.bfloat16()), "float32"), (dict(state=state[:1]), "fewer rows"),
                     (dict(state=state.transpose(2, 3)), "last two"), (dict(q=q.float()), "one dtype"),
                     (dict(v=v[:, :, :3]), "shape"), (dict(state=state.cpu()), "CUDA"), (dict(k=k[..., :32]), "shape"),
                     (dict(state_indices=torch.zeros(2, dtype=torch.int64, device="cuda")), "int32"),
                     (dict(g=g.double()), "float32")):
        with pytest.raises(RuntimeError, match=text):
            call(**kw)
    with pytest.raises(RuntimeError, match="multiples of 8"):
        cc.gated_delta_rule_update(q[..., :60], k[..., :60], v, g, beta, state[:, :, :60].contiguous())
    with pytest.raises(RuntimeError, match="multiple of the number of key heads"):
        cc.gated_delta_rule_update(q, k, v[:, :, :3], g[..., :3], beta[..., :3], state[:, :3].contiguous())


def test_refuses_a_state_whose_rows_are_one_place():
    import causal_conv1d_b200 as cc
    q, k, v, g, beta = gdr_ref.inputs((2, 1), 2, 4, 64, 64, torch.bfloat16)
    shared = torch.zeros(1, 4, 64, 64, device="cuda").expand(2, 4, 64, 64)
    with pytest.raises(RuntimeError, match="expanded"):
        cc.gated_delta_rule_update(q, k, v, g, beta, shared)
    packed, cu = [t[:, 0] for t in (q, k, v, g, beta)], torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="expanded"):
        cc.gated_delta_rule_varlen_fn(*packed, cu_seqlens=cu, states=shared)
    # read only, it is a state that all sequences share
    one = cc.gated_delta_rule_varlen_fn(*packed, cu_seqlens=cu, states=shared, update_states=False)
    own = cc.gated_delta_rule_varlen_fn(*packed, cu_seqlens=cu, states=shared.contiguous(), update_states=False)
    assert torch.equal(one, own)
