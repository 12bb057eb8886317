"""The gated delta rule token by token in float64, what the delta-rule tests compare with."""
import torch


def rule(q, k, v, g, beta, S, scale):
    """q, k (T, Hk, K), v (T, Hv, V), g, beta (T, Hv), S (Hv, K, V), all float64 -> out (T, Hv, V), S."""
    group = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(group, 1), k.repeat_interleave(group, 1)
    outs = []
    for t in range(q.shape[0]):
        S = S * torch.exp(g[t])[:, None, None]
        d = beta[t][:, None] * (v[t] - (S * k[t][:, :, None]).sum(1))
        S = S + k[t][:, :, None] * d[:, None, :]
        outs.append(scale * (S * q[t][:, :, None]).sum(1))
    return (torch.stack(outs) if outs else torch.zeros_like(v)), S


def inputs(lead, hk, hv, dk, dv, dtype, gdtype=torch.float32, bdtype=None, seed=0, device="cuda", slow=False):
    """q, k of unit length; decays between 1e-3 and 1 a token."""
    gen = torch.Generator(device="cpu").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    q = torch.nn.functional.normalize(rn(*lead, hk, dk), dim=-1)
    k = torch.nn.functional.normalize(rn(*lead, hk, dk), dim=-1)
    v = rn(*lead, hv, dv)
    g = -torch.exp(3 * rn(*lead, hv) - 3).clamp(max=20.0) * (0.02 if slow else 1.0)
    beta = torch.sigmoid(rn(*lead, hv))
    return (q.to(dtype).to(device), k.to(dtype).to(device), v.to(dtype).to(device), g.to(gdtype).to(device),
            beta.to(bdtype or dtype).to(device))


def close(actual, ref, tol, what, dtype=torch.float32):
    """|a - b| <= tol * max|ref| + half a step of dtype relative to b."""
    a, b = actual.detach().double().cpu(), ref.detach().double().cpu()
    assert a.shape == b.shape, f"{what}: shape {tuple(a.shape)} vs {tuple(b.shape)}"
    if a.numel() == 0:
        return
    assert torch.isfinite(a).all(), f"{what}: not finite"
    allowed = tol * max(1e-3, b.abs().max().item()) + (torch.finfo(dtype).eps / 2) * b.abs() * (1 + 1e-6)
    worst = ((a - b).abs() - allowed).max().item()
    assert worst <= 0, f"{what}: {worst:.3e} beyond the allowed error (max|ref| {b.abs().max().item():.3e})"
