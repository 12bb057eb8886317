"""Where the delta rule's tensors lie: storage offsets, and tokens that no sequence owns."""
import pytest
import torch

import gdr_ref
from conftest import DT

pytestmark = pytest.mark.gpu


def off_by_one(t):
    """The same values, contiguous, one element behind a 16-byte boundary."""
    there = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape)
    assert there.is_contiguous() and there.data_ptr() % 16 == t.element_size()
    return there.copy_(t)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("which", ["q", "k", "v", "g", "beta", "initial_state", "dout", "dfinal_state"])
def test_contiguous_tensors_off_a_16_byte_boundary(which, dtype):
    import causal_conv1d_b200 as cc
    names = ["q", "k", "v", "g", "beta", "initial_state", "dout", "dfinal_state"]
    gen = torch.Generator().manual_seed(1)
    state = lambda: torch.randn(2, 4, 64, 32, generator=gen).cuda()  # noqa: E731
    args = dict(zip(names, (*gdr_ref.inputs((2, 70), 2, 4, 64, 32, DT[dtype]), state(), torch.randn(2, 70, 4, 32, generator=gen).to(DT[dtype]).cuda(), state())))

    def run(a):
        leaves = [a[n].detach().requires_grad_() for n in names[:6]]
        out, last = cc.gated_delta_rule_fn(*leaves, return_final_state=True)
        return (out, last, *torch.autograd.grad((out, last), leaves, (a["dout"], a["dfinal_state"])))

    for a, b in zip(run({**args, which: off_by_one(args[which])}), run(args)):
        assert torch.equal(a, b)


def test_prefill_of_contiguous_tensors_off_a_16_byte_boundary():
    import causal_conv1d_b200 as cc
    args = [t[0] for t in gdr_ref.inputs((1, 70), 2, 4, 64, 32, torch.bfloat16)]
    cu = torch.tensor([0, 70], dtype=torch.int32).cuda()
    want = cc.gated_delta_rule_varlen_fn(*args, cu_seqlens=cu)
    assert torch.equal(cc.gated_delta_rule_varlen_fn(*(off_by_one(t) for t in args), cu_seqlens=cu), want)


def test_gradient_that_is_a_slice_of_a_flat_one():
    """What the backward of torch.cat hands over starts wherever the output lay in the flat tensor."""
    import causal_conv1d_b200 as cc
    leaves = [t.requires_grad_() for t in gdr_ref.inputs((1, 70), 2, 4, 64, 32, torch.bfloat16)]
    flat = torch.randn(1 + 70 * 4 * 32, device="cuda").bfloat16()
    out = cc.gated_delta_rule_fn(*leaves)
    got = torch.autograd.grad(torch.cat([torch.zeros_like(flat[:1]), out.flatten()]), leaves, flat)
    out = cc.gated_delta_rule_fn(*leaves)
    for a, b in zip(got, torch.autograd.grad(out, leaves, flat[1:].clone().view(out.shape))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("heads", [2, 160])
@pytest.mark.parametrize("lens", [[70, 35], [1, 4000], [5, 0, 64], [130]])
def test_tokens_before_the_first_sequence(lens, heads):
    """cu_seqlens that does not start at 0: zero outputs and gradients there, as behind the last sequence; 2 heads of 4000 tokens
    are walked in segments."""
    import causal_conv1d_b200 as cc
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)[1:].cuda()            # lens[0] tokens in front
    begin, end = int(cu[0]), int(cu[-1])
    leaves = [t.requires_grad_() for t in gdr_ref.inputs((1, end + 9), heads // 2, heads, 32, 32, torch.bfloat16)]
    junk = [torch.full((1 << 25,), float("nan"), device="cuda") for _ in range(4)]
    del junk                                                                      # what torch.empty may hand out
    out = cc.gated_delta_rule_fn(*leaves, cu_seqlens=cu)
    grads = torch.autograd.grad(out, leaves, torch.ones_like(out))
    for t in (out, *grads):
        assert not t[:, :begin].any() and not t[:, end:].any()
    part = [t.detach()[:, begin:end].clone().requires_grad_() for t in leaves]
    if end > begin:
        want = cc.gated_delta_rule_fn(*part, cu_seqlens=cu - begin)
        for a, b in zip((out, *grads), (want, *torch.autograd.grad(want, part, torch.ones_like(want)))):
            assert torch.equal(a[:, begin:end], b)
    packed = cc.gated_delta_rule_varlen_fn(*(t.detach()[0] for t in leaves), cu_seqlens=cu)
    assert torch.equal(packed, out[0])


@pytest.mark.parametrize("which", ["q", "k", "v", "g", "beta", "dout"])
@pytest.mark.parametrize("along", [0, 1, 2])
def test_expanded_tensors(which, along):
    """Rows, tokens or heads that share memory (stride 0): read where they lie."""
    import causal_conv1d_b200 as cc
    names = ["q", "k", "v", "g", "beta"]
    args = dict(zip(names, gdr_ref.inputs((2, 70), 2, 4, 64, 32, torch.bfloat16, seed=along)))
    args["dout"] = torch.randn(2, 70, 4, 32, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    t = args[which]
    shared = t.narrow(along, 0, 1).expand(t.shape)

    def run(a):
        leaves = [a[n].detach().requires_grad_() for n in names]
        out = cc.gated_delta_rule_fn(*leaves)
        steps = cc.gated_delta_rule_update(*(x.detach()[:, :5] for x in leaves), torch.zeros(2, 4, 64, 32, device="cuda"))
        return (out, steps, *torch.autograd.grad(out, leaves, a["dout"]))

    for a, b in zip(run({**args, which: shared}), run({**args, which: shared.clone(memory_format=torch.contiguous_format)})):
        assert torch.equal(a, b)
