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


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_forgetting_inside_chunks(dtype):
    """g = -inf, -1000, -70 and steep runs: exact resets, and tokens behind them as accurate as ever."""
    import causal_conv1d_b200 as cc
    total = 300
    q, k, v, g, beta = gdr_ref.inputs((total,), 1, 2, 64, 64, DT[dtype], seed=4)
    g[5, 0], g[70, 0], g[71, 0], g[130, 1], g[200:216, 1] = -torch.inf, -1000.0, -torch.inf, -70.0, -30.0
    g[64, 1] = -torch.inf
    beta[40:50] = 0
    cu = [0, 300]
    want, _ = expect(q, k, v, g, beta, cu, None, None, None, 1.0)
    got = cc.gated_delta_rule_varlen_fn(q, k, v, g, beta, cu_seqlens=torch.tensor(cu, dtype=torch.int32).cuda(), scale=1.0)
    gdr_ref.close(got, want, TOL if dtype == "fp32" else TOL_OUT16, "out", DT[dtype])


def test_nan_stays_in_its_sequence_and_head():
    import causal_conv1d_b200 as cc
    q, k, v, g, beta = gdr_ref.inputs((200,), 2, 2, 64, 64, torch.bfloat16, seed=6)
    cu = torch.tensor([0, 70, 100, 200], dtype=torch.int32).cuda()
    clean = cc.gated_delta_rule_varlen_fn(q, k, v, g, beta, cu_seqlens=cu)
    v[80, 1, 3] = torch.nan
    k[99, 0, 5] = torch.inf
    got = cc.gated_delta_rule_varlen_fn(q, k, v, g, beta, cu_seqlens=cu)
    assert torch.equal(got[:70], clean[:70]) and torch.equal(got[100:], clean[100:]) and torch.equal(got[70:80], clean[70:80])
    assert torch.isnan(got[80:100, 1, 3]).all() and not torch.isnan(got[70:99, 0]).any()


def test_cu_seqlens_outside_the_tokens_is_clamped():
    """A last entry beyond the tokens, or one below its predecessor, reads and writes nothing outside."""
    import causal_conv1d_b200 as cc
    q, k, v, g, beta = gdr_ref.inputs((100,), 1, 1, 32, 32, torch.bfloat16, seed=8)
    want = cc.gated_delta_rule_varlen_fn(q, k, v, g, beta, cu_seqlens=torch.tensor([0, 40, 100], dtype=torch.int32).cuda())
    got = cc.gated_delta_rule_varlen_fn(q, k, v, g, beta, cu_seqlens=torch.tensor([0, 40, 1000], dtype=torch.int32).cuda())
    assert torch.equal(want, got)


def test_without_states_and_read_only_states():
    import causal_conv1d_b200 as cc
    lens, cu = [90, 30], [0, 90, 120]
    q, k, v, g, beta = gdr_ref.inputs((120,), 2, 2, 64, 32, torch.bfloat16, seed=9)
    cut = torch.tensor(cu).cuda()                       # int64: converted
    states = torch.randn(2, 2, 64, 32, device="cuda")
    before = states.clone()
    got = cc.gated_delta_rule_varlen_fn(q, k, v, g, beta, cu_seqlens=cut, states=states, update_states=False)
    assert torch.equal(states, before)
    gdr_ref.close(got, expect(q, k, v, g, beta, cu, states, None, None, 64 ** -0.5)[0], TOL_OUT16, "out", torch.bfloat16)
    got = cc.gated_delta_rule_varlen_fn(q, k, v, g, beta, cu_seqlens=cut)
    gdr_ref.close(got, expect(q, k, v, g, beta, cu, None, None, None, 64 ** -0.5)[0], TOL_OUT16, "out", torch.bfloat16)


def test_prefill_then_decode_is_the_whole():
    """A prompt in two prefills and single tokens after it, over one pool row: the outputs of one prefill."""
    import causal_conv1d_b200 as cc
    T = 150
    q, k, v, g, beta = gdr_ref.inputs((T,), 2, 4, 128, 64, torch.float32, seed=11)
    pool = torch.zeros(3, 4, 128, 64, device="cuda")
    row = torch.tensor([2], dtype=torch.int32, device="cuda")
    outs, a = [], 0
    for n in (100, 37):
        part = slice(a, a + n)
        outs.append(cc.gated_delta_rule_varlen_fn(q[part], k[part], v[part], g[part], beta[part], cu_seqlens=torch.tensor([0, n], dtype=torch.int32).cuda(),
                                                  states=pool, state_indices=row))
        a += n
    for t in range(a, T):
        outs.append(cc.gated_delta_rule_update(q[t:t + 1], k[t:t + 1], v[t:t + 1], g[t:t + 1], beta[t:t + 1], pool, state_indices=row))
    want, states = expect(q, k, v, g, beta, [0, T], torch.zeros(1, 4, 128, 64), None, None, 128 ** -0.5)
    gdr_ref.close(torch.cat(outs), want, TOL, "out")
    gdr_ref.close(pool[2], states[0], TOL, "state")
    assert not pool[:2].any()


def test_two_graphs_and_a_side_stream():
    """Two captured prefills replayed in turn, and one more on another stream: each with a workspace of its own."""
    import causal_conv1d_b200 as cc
    sets = [gdr_ref.inputs((130,), 1, 2, 64, 64, torch.bfloat16, seed=s) for s in (1, 2)]
    cu = torch.tensor([0, 100, 130], dtype=torch.int32).cuda()
    call = lambda s: cc.gated_delta_rule_varlen_fn(*s, cu_seqlens=cu)  # noqa: E731
    want = [call(s) for s in sets]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(s))
        graphs.append(graph)
    side = torch.cuda.Stream()
    for _ in range(3):
        for graph in graphs:
            graph.replay()
        with torch.cuda.stream(side):
            other = call(sets[0])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(other, want[0])


def test_refusals():
    import causal_conv1d_b200 as cc
    q, k, v, g, beta = gdr_ref.inputs((10,), 1, 2, 32, 32, torch.bfloat16)
    cu = torch.tensor([0, 10], dtype=torch.int32).cuda()
    call = lambda **kw: cc.gated_delta_rule_varlen_fn(**{**dict(q=q, k=k, v=v, g=g, beta=beta, cu_seqlens=cu), **kw})  # noqa: E731
    for kw, text in ((dict(states=torch.zeros(1, 2, 32, 32, device="cuda").half()), "float32"), (dict(states=torch.zeros(0, 2, 32, 32, device="cuda")), "fewer rows"),
                     (dict(cu_seqlens=cu.cpu()), "CUDA"), (dict(v=v.half()), "one dtype"), (dict(g=g[:, :1]), "shape"),
                     (dict(states=torch.zeros(1, 2, 32, 32, device="cuda"), has_initial_state=torch.ones(2, device="cuda")), "one entry per sequence"),
                     (dict(q=q[..., :20], k=k[..., :20]), "multiples of 8")):
        with pytest.raises(RuntimeError, match=text):
            call(**kw)
    q4 = q[None]
    with pytest.raises(RuntimeError, match="one row per sequence"):
        cc.gated_delta_rule_fn(q4, k[None], v[None], g[None], beta[None], initial_state=torch.zeros(2, 2, 32, 32, device="cuda"))
    with pytest.raises(RuntimeError, match="batch of one packed row"):
        cc.gated_delta_rule_fn(q4.repeat(2, 1, 1, 1), k[None].repeat(2, 1, 1, 1), v[None].repeat(2, 1, 1, 1), g[None].repeat(2, 1, 1), beta[None].repeat(2, 1, 1), cu_seqlens=cu)


def test_overflow_stays_behind_its_token():
    """Keys so large that products of gates and keys leave fp32: finite before, not after, no other head."""
    import causal_conv1d_b200 as cc
    q, k, v, g, beta = gdr_ref.inputs((64,), 2, 2, 32, 32, torch.float32, seed=12)
    cu = torch.tensor([0, 64], dtype=torch.int32).cuda()
    clean = cc.gated_delta_rule_varlen_fn(q, k, v, g, beta, cu_seqlens=cu)
    k[30:34, 1] *= 1e19
    got = cc.gated_delta_rule_varlen_fn(q, k, v, g, beta, cu_seqlens=cu)
    assert torch.equal(got[:, 0], clean[:, 0]) and torch.equal(got[:30, 1], clean[:30, 1])
    assert not torch.isfinite(got[40:, 1]).any()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_the_same_bits_every_time(dtype):
    """Nothing a chunk leaves in tensor memory is overwritten while the chunk before still reads its place."""
    import causal_conv1d_b200 as cc
    lens = [64 * 40, 1, 64 * 17 + 1, 0, 900, 64 * 13 - 1]
    q, k, v, g, beta = gdr_ref.inputs((sum(lens),), 1, 2, 96, 72, DT[dtype], seed=6, slow=True)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    first = None
    for _ in range(100):
        states = torch.zeros(len(lens), 2, 96, 72, device="cuda")
        out = cc.gated_delta_rule_varlen_fn(q, k, v, g, beta, cu_seqlens=cu, states=states)
        first = first or (out, states)
        assert torch.equal(out, first[0]) and torch.equal(states, first[1])
