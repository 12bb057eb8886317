"""The workloads by which the gated delta rule and the 8-bit activation checkpoint of the causal
convolution are measured: cases, inputs, a plain PyTorch form, the package's own calls, and a
64-bit statement of what each has to return.

Kinds of case:
  train    gated_delta_rule_fn, forward and backward, (batch, tokens) or packed sequences
  prefill  gated_delta_rule_varlen_fn: packed sequences that continue from a pool of states
  decode   gated_delta_rule_update: a few tokens for each row of a batch, states in a pool
  conv     causal_conv1d_fn with its input kept in 8 bits for the backward pass
"""
import math
import random

import torch
import torch.nn.functional as F

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_CHUNK = 64
_GROUP = 32          # elements that share a scale in the 8-bit checkpoint


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _rule(kind, **kw):
    c = dict(kind=kind, hk=16, hv=16, dk=128, dv=128, dtype="bf16")
    c.update(kw)
    return c


def listed():
    return [
        # a training step's layer: rows of 4096 tokens, values with twice the heads of the keys
        _rule("train", name="train 2x4096 32 heads bf16", batch=2, tokens=4096, nseq=0, state=False, hv=32),
        # documents of many lengths packed into one row, gradients through the carried state
        _rule("train", name="train packed 8000 bf16", batch=1, tokens=8000, nseq=9, state=True),
        # a small model trained in 32 bits, odd length
        _rule("train", name="train 2x501 fp32", batch=2, tokens=501, nseq=0, state=False, hk=4, hv=4, dk=64, dv=64,
              dtype="fp32"),
        # one long prompt: few heads, many chunks
        _rule("prefill", name="prefill 1x32768 bf16", tokens=32768, nseq=1, state=True, hv=32),
        # a serving batch of 16 prompts
        _rule("prefill", name="prefill 16 of 32768 bf16", tokens=32768, nseq=16, state=True, hv=32),
        # a few short prompts in 16-bit floats: latency counts
        _rule("prefill", name="prefill 5 of 333 fp16", tokens=333, nseq=5, state=True, hk=4, hv=8, dk=96, dv=64, dtype="fp16"),
        # one request being answered
        _rule("decode", name="decode 1 bf16", batch=1, tokens=1, rows=2, hv=32),
        # a full batch of requests out of a pool of twice as many states
        _rule("decode", name="decode 256 bf16", batch=256, tokens=1, rows=512, hv=32),
        # drafted tokens checked three at a time
        _rule("decode", name="decode 48x3 fp16", batch=48, tokens=3, rows=64, hv=16, dtype="fp16"),
        # the benchmark's convolution (channel-first) with its input kept in 8 bits
        dict(kind="conv", name="conv 8x5120x2048 bf16", batch=8, dim=5120, tokens=2048, width=4, nseq=0, last=False,
             dtype="bf16"),
        # a channel-last pack of sequences, as in front of the delta rule
        dict(kind="conv", name="conv packed 5376x8192 bf16", batch=1, dim=5376, tokens=8192, width=4, nseq=16, last=True,
             dtype="bf16"),
        # a small convolution in 32 bits, rows of odd length
        dict(kind="conv", name="conv 2x96x333 fp32", batch=2, dim=96, tokens=333, width=3, nseq=0, last=False, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["train", "prefill", "decode", "conv"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    hk = rng.choice([1, 2, 4, 8, 16])
    hv = hk * rng.choice([1, 1, 2, 3] if hk < 16 else [1, 2])
    dk, dv = (rng.choice([32, 64, 80, 96, 128, 128]) for _ in range(2))
    if kind == "train":
        packed = rng.random() < 0.5
        batch = 1 if packed else rng.randint(1, 4)
        most = min(8192, 2 * 4096 * 32 // (hv * batch))
        tokens = _log(rng, 8, most)
        return _rule(kind, batch=batch, tokens=tokens, nseq=rng.randint(1, min(12, tokens)) if packed else 0,
                     state=rng.random() < 0.5, hk=hk, hv=hv, dk=dk, dv=dv, dtype=dtype)
    if kind == "prefill":
        tokens = _log(rng, 16, 32768 if dtype != "fp32" else 16384)
        return _rule(kind, tokens=tokens, nseq=rng.randint(1, min(24, tokens)), state=rng.random() < 0.8, hk=hk, hv=hv,
                     dk=dk, dv=dv, dtype=dtype)
    if kind == "decode":
        batch = _log(rng, 1, 256)
        return _rule(kind, batch=batch, tokens=rng.choice([1, 1, 1, 2, 3, 5]), rows=batch + _log(rng, 1, 256), hk=hk, hv=hv,
                     dk=dk, dv=dv, dtype=dtype)
    last = rng.random() < 0.5
    dim = 8 * _log(rng, 2, 640)
    batch = rng.randint(1, 4)
    tokens = _log(rng, 8, 4096)
    return dict(kind="conv", batch=batch, dim=dim, tokens=tokens, width=rng.choice([2, 3, 4]),
                nseq=rng.randint(1, min(16, tokens)) if last and rng.random() < 0.5 else 0, last=last, dtype=dtype)


def _lengths(case):
    """Lengths of the packed sequences: a spread over more than a factor of ten, one of them 1."""
    total, n = case["tokens"], case["nseq"]
    r = random.Random(1000 * n + total)
    if n == 1:
        return [total]
    w = [math.exp(r.uniform(0, 2.5)) for _ in range(n)]
    lens = [max(1, int((total - 1) * x / sum(w))) for x in w]
    lens[r.randrange(n)] = 1
    while sum(lens) > total:
        lens[lens.index(max(lens))] -= 1
    lens[lens.index(max(lens))] += total - sum(lens)
    return lens


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "conv":
        n, scales = case["batch"] * case["dim"] * case["tokens"], 1 / _GROUP
        # forward: x read, out and the 8-bit copy written; backward: the copy and dout read, dx written
        size = n * (2 * es + 1 + scales) + n * (1 + scales + 2 * es) + 3 * case["dim"] * (case["width"] + 1) * es
        return {"bytes": size + (8 * case["batch"] * case["tokens"] if case["nseq"] else 0), "flops": n * (2 * 3 * case["width"] + 20)}
    hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
    tok = case["tokens"] * case.get("batch", 1)
    qk, vo, gates = tok * hk * dk * es, tok * hv * dv * es, tok * hv * (4 + es)
    one = 4 * hv * dk * dv                     # a state
    flops = 6 * tok * hv * dk * dv             # S^T k, the rank-one update, S^T q
    if case["kind"] == "train":
        n = (case["nseq"] or case["batch"]) * 4 if case["state"] else 0   # the state and its gradient at both ends
        return {"bytes": 2 * (2 * qk + vo + gates) + 2 * vo + n * one, "flops": 3 * flops}
    n = case["batch"] if case["kind"] == "decode" else case["nseq"] if case["state"] else 0
    return {"bytes": 2 * qk + 2 * vo + gates + 2 * n * one, "flops": flops}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _rule_inputs(case, gen, lead, dev):
    """q and k of unit length, gates as a trained layer has them: decays of 1..16 times a small step."""
    dt, hk, hv, dk, dv = _DT[case["dtype"]], case["hk"], case["hv"], case["dk"], case["dv"]
    rn = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    q = F.normalize(rn(*lead, hk, dk), dim=-1).to(dt)
    k = F.normalize(rn(*lead, hk, dk), dim=-1).to(dt)
    v = rn(*lead, hv, dv).to(dt)
    rate = 1 + 15 * torch.rand(hv, generator=gen, device=dev)
    g = -rate * F.softplus(rn(*lead, hv) - 4)
    beta = torch.sigmoid(rn(*lead, hv)).to(dt)
    return dict(q=q, k=k, v=v, g=g, beta=beta)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt, kind = _DT[case["dtype"]], case["kind"]
    s = dict(case=case)
    if kind == "conv":
        B, D, L, W = case["batch"], case["dim"], case["tokens"], case["width"]
        shape = (B, L, D) if case["last"] else (B, D, L)
        x, dout = (torch.randn(*shape, generator=gen, device=dev).to(dt) for _ in range(2))
        if case["last"]:
            x, dout = x.transpose(1, 2), dout.transpose(1, 2)
        s.update(x=x.requires_grad_(), dout=dout)
        s["w"] = (torch.rand(D, W, generator=gen, device=dev) - 0.5).to(dt).requires_grad_()
        s["b"] = (torch.rand(D, generator=gen, device=dev) - 0.5).to(dt).requires_grad_()
        s["seq_idx"] = None
        if case["nseq"]:
            lens = torch.tensor(_lengths(case), device=dev)
            s["seq_idx"] = torch.repeat_interleave(torch.arange(case["nseq"], device=dev, dtype=torch.int32), lens).repeat(B, 1)
        return s
    hv, dk, dv = case["hv"], case["dk"], case["dv"]
    if kind == "decode":
        B, T = case["batch"], case["tokens"]
        s.update(_rule_inputs(case, gen, (B,) if T == 1 else (B, T), dev))
        s["state"] = 0.3 * torch.randn(case["rows"], hv, dk, dv, generator=gen, device=dev)
        s["rows"] = torch.randperm(case["rows"], generator=gen, device=dev)[:B].to(torch.int32)
        return s
    lead = (case["batch"], case["tokens"]) if kind == "train" else (case["tokens"],)
    s.update(_rule_inputs(case, gen, lead, dev))
    n = case["nseq"] or case["batch"]
    s["cu"] = s["lens"] = None
    if case["nseq"]:
        s["lens"] = _lengths(case)
        s["cu"] = torch.tensor([0] + s["lens"], device=dev).cumsum(0).to(torch.int32)
    if kind == "train":
        for name in ("q", "k", "v", "g", "beta"):
            s[name].requires_grad_()
        s["dout"] = torch.randn(*lead, hv, dv, generator=gen, device=dev).to(dt)
        s["state"] = s["dfinal"] = None
        if case["state"]:
            s["state"] = (0.3 * torch.randn(n, hv, dk, dv, generator=gen, device=dev)).requires_grad_()
            s["dfinal"] = 0.3 * torch.randn(n, hv, dk, dv, generator=gen, device=dev)
        return s
    s["state"] = s["rows"] = s["has"] = None
    if case["state"]:
        s["state"] = 0.3 * torch.randn(n + 3, hv, dk, dv, generator=gen, device=dev)
        s["rows"] = torch.randperm(n + 3, generator=gen, device=dev)[:n].to(torch.int32)
        s["has"] = torch.arange(n, device=dev) % 2 == 0
    return s


# ---------------------------------------------------------------------------------------------
# plain forms, in 32 bits
# ---------------------------------------------------------------------------------------------
def _padding(s, dev):
    """Index (sequences, longest) of every token of a pack and which of them exist."""
    lens = torch.tensor(s["lens"], device=dev)
    at = torch.arange(max(s["lens"]), device=dev)
    there = at < lens[:, None]
    return torch.where(there, s["cu"][:-1, None].long() + at, 0), there


def _rule_by_chunks(q, k, v, g, beta, state, scale):
    """The chunked form over (sequences, heads, tokens, ...): within a chunk a triangular solve, from chunk to
    chunk the carried state."""
    n, h, t, dk = q.shape
    dv = v.shape[-1]
    pad = -t % _CHUNK
    if pad:
        q, k, v = (F.pad(x, (0, 0, 0, pad)) for x in (q, k, v))
        g, beta = F.pad(g, (0, pad)), F.pad(beta, (0, pad))
    q, k, v = (x.reshape(n, h, -1, _CHUNK, x.shape[-1]) for x in (q, k, v))
    beta = beta.reshape(n, h, -1, _CHUNK, 1)
    G = g.reshape(n, h, -1, _CHUNK).double().cumsum(-1)
    low = torch.ones(_CHUNK, _CHUNK, device=q.device).tril()
    decay = ((G[..., :, None] - G[..., None, :]).float().masked_fill(low == 0, -math.inf)).exp()
    from_start = G.float().exp().unsqueeze(-1)
    to_end = (G[..., -1:] - G).float().exp().unsqueeze(-1)
    whole = from_start[..., -1:, :]
    lower = (beta * (k @ k.mT) * decay).tril(-1) + torch.eye(_CHUNK, device=q.device)
    solved = torch.linalg.solve_triangular(lower, torch.cat([beta * from_start * k, beta * v], -1), upper=False, unitriangular=True)
    w, u = solved[..., :dk], solved[..., dk:]
    att = (q @ k.mT) * decay * scale
    qs, ke = scale * from_start * q, to_end * k
    outs = []
    for c in range(q.shape[2]):
        new = u[:, :, c] - w[:, :, c] @ state
        outs.append(qs[:, :, c] @ state + att[:, :, c] @ new)
        state = whole[:, :, c] * state + ke[:, :, c].mT @ new
    return torch.stack(outs, 2).reshape(n, h, -1, dv)[:, :, :t], state


def _plain_rule(s, q, k, v, g, beta, state):
    """(batch, tokens, heads, dim) or packed (tokens, heads, dim) -> the same of the output, and the last states."""
    case = s["case"]
    q, k, v, g, beta = (x.float() for x in (q, k, v, g, beta))
    group = case["hv"] // case["hk"]
    if s["lens"] is not None:
        q, k, v, g, beta = (x.reshape(-1, *x.shape[x.dim() - y:]) for x, y in ((q, 2), (k, 2), (v, 2), (g, 1), (beta, 1)))
        at, there = _padding(s, q.device)
        q, k, v, g, beta = (x[at] * there.reshape(*there.shape, *[1] * (x.dim() - 1)) for x in (q, k, v, g, beta))
    q, k = (x.repeat_interleave(group, 2).transpose(1, 2) for x in (q, k))
    out, state = _rule_by_chunks(q, k, v.transpose(1, 2), g.transpose(1, 2), beta.transpose(1, 2), state,
                                 case["dk"] ** -0.5)
    out = out.transpose(1, 2)
    return (out[there] if s["lens"] is not None else out), state


def _plain_decode(s):
    case = s["case"]
    q, k, v, g, beta = (s[n].float() for n in ("q", "k", "v", "g", "beta"))
    group = case["hv"] // case["hk"]
    if case["tokens"] == 1:
        q, k, v, g, beta = (x.unsqueeze(1) for x in (q, k, v, g, beta))
    q, k = (x.repeat_interleave(group, 2) for x in (q, k))
    rows = s["rows"].long()
    state, outs = s["state"][rows], []
    for t in range(case["tokens"]):
        state = state * g[:, t].exp()[..., None, None]
        seen = (state * k[:, t].unsqueeze(-1)).sum(-2)
        new = beta[:, t].unsqueeze(-1) * (v[:, t] - seen)
        state = state + k[:, t].unsqueeze(-1) * new.unsqueeze(-2)
        outs.append((state * q[:, t].unsqueeze(-1)).sum(-2) * case["dk"] ** -0.5)
    s["state"][rows] = state
    out = torch.stack(outs, 1).to(s["q"].dtype)
    return {"out": out[:, 0] if case["tokens"] == 1 else out, "state": s["state"]}


def _in_8_bits(x):
    """x rounded to e4m3 with a power-of-two scale for each 32 neighbours along the last axis; the values that stand there."""
    n = x.shape[-1]
    y = F.pad(x, (0, -n % _GROUP)).unflatten(-1, (-1, _GROUP))
    most = y.abs().amax(-1, keepdim=True)
    frac, power = torch.frexp(most)                      # most = frac * 2^power, frac in [0.5, 1)
    power = torch.where(most > 0, power - 9 + (frac > 448 / 512).int(), 0)
    y = torch.ldexp(torch.ldexp(y, -power).to(torch.float8_e4m3fn).float(), power)
    return y.flatten(-2)[..., :n]


def _conv_parts(case, x, w, b, seq_idx):
    """The taps' inputs (batch, dim, tokens) of each tap, and the sum before the activation."""
    W, L = case["width"], x.shape[-1]
    taps = []
    for j in range(W):
        back = W - 1 - j
        tap = F.pad(x, (back, 0))[..., :L]
        if seq_idx is not None and back:
            tap = tap * (F.pad(seq_idx, (back, 0), value=-1)[:, :L] == seq_idx).unsqueeze(1)
        taps.append(tap)
    return taps, sum(tap * w[:, j, None] for j, tap in enumerate(taps)) + b[:, None]


def _plain_conv(s):
    case, dt = s["case"], s["x"].dtype
    x, dout, w, b = (s[n].detach().float() for n in ("x", "dout", "w", "b"))
    _, y = _conv_parts(case, x, w, b, s["seq_idx"])
    out = (y * torch.sigmoid(y)).to(dt)
    kept = _in_8_bits(x.mT).mT if case["last"] else _in_8_bits(x)
    taps, y = _conv_parts(case, kept, w, b, s["seq_idx"])
    p = torch.sigmoid(y)
    dy = dout * p * (1 + y * (1 - p))
    dx = torch.zeros_like(x)
    L, W = x.shape[-1], case["width"]
    dw = torch.empty_like(w)
    for j in range(W):
        back = W - 1 - j
        d = dy * w[:, j, None]
        if s["seq_idx"] is not None and back:
            d = d * (F.pad(s["seq_idx"], (back, 0), value=-1)[:, :L] == s["seq_idx"]).unsqueeze(1)
        dx += F.pad(d, (0, back))[..., back:]
        dw[:, j] = (taps[j] * dy).sum((0, 2))
    return {"out": out, "dx": dx.to(dt), "dw": dw.to(dt), "db": dy.sum((0, 2)).to(dt)}


def _plain(s):
    case, kind = s["case"], s["case"]["kind"]
    if kind == "conv":
        return _plain_conv(s)
    if kind == "decode":
        return _plain_decode(s)
    n, dev = case["nseq"] or case["batch"], s["q"].device
    shape = (n, case["hv"], case["dk"], case["dv"])
    dt = s["q"].dtype
    if kind == "prefill":
        first = torch.zeros(shape, device=dev)
        if case["state"]:
            first = torch.where(s["has"][:, None, None, None], s["state"][s["rows"].long()], first)
        out, last = _plain_rule(s, *(s[x] for x in ("q", "k", "v", "g", "beta")), first)
        if case["state"]:
            s["state"][s["rows"].long()] = last
        return {"out": out.to(dt), "state": s["state"]}
    wrt = [s[x] for x in ("q", "k", "v", "g", "beta")] + ([s["state"]] if case["state"] else [])
    first = s["state"] if case["state"] else torch.zeros(shape, device=dev)
    out, last = _plain_rule(s, *wrt[:5], first)
    out = out.reshape(s["v"].shape)
    tops, grads = [out], [s["dout"].float()]
    if case["state"]:
        tops, grads = tops + [last], grads + [s["dfinal"]]
    d = torch.autograd.grad(tops, wrt, grads)
    names = ["dq", "dk", "dv", "dg", "dbeta", "dstate"]
    return {"out": out.detach().to(dt), "state": last.detach() if case["state"] else None, **dict(zip(names, d))}


# ---------------------------------------------------------------------------------------------
# the package's own calls
# ---------------------------------------------------------------------------------------------
def _own(s):
    import causal_conv1d_b200 as cc

    case, kind = s["case"], s["case"]["kind"]
    if kind == "conv":
        out = cc.causal_conv1d_fn(s["x"], s["w"], s["b"], seq_idx=s["seq_idx"], activation="silu", checkpoint="e4m3")
        dx, dw, db = torch.autograd.grad(out, (s["x"], s["w"], s["b"]), s["dout"])
        return {"out": out.detach(), "dx": dx, "dw": dw, "db": db}
    q, k, v, g, beta = (s[n] for n in ("q", "k", "v", "g", "beta"))
    if kind == "decode":
        out = cc.gated_delta_rule_update(q, k, v, g, beta, s["state"], state_indices=s["rows"])
        return {"out": out, "state": s["state"]}
    if kind == "prefill":
        out = cc.gated_delta_rule_varlen_fn(q, k, v, g, beta, cu_seqlens=s["cu"], states=s["state"], state_indices=s["rows"],
                                            has_initial_state=s["has"])
        return {"out": out, "state": s["state"]}
    if case["state"]:
        out, last = cc.gated_delta_rule_fn(q, k, v, g, beta, initial_state=s["state"], return_final_state=True,
                                           cu_seqlens=s["cu"])
        d = torch.autograd.grad((out, last), (q, k, v, g, beta, s["state"]), (s["dout"], s["dfinal"]))
    else:
        out, last = cc.gated_delta_rule_fn(q, k, v, g, beta, cu_seqlens=s["cu"]), None
        d = torch.autograd.grad(out, (q, k, v, g, beta), s["dout"])
    names = ["dq", "dk", "dv", "dg", "dbeta", "dstate"]
    return {"out": out.detach(), "state": None if last is None else last.detach(), **dict(zip(names, d))}


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------
# 64 bits, from the definition
# ---------------------------------------------------------------------------------------------
def _token_by_token(q, k, v, g, beta, S, scale):
    """q, k, v, g, beta over (rows, tokens, heads, ...), S (rows, heads, dk, dv): the recurrence itself."""
    outs = []
    for t in range(q.shape[1]):
        S = torch.exp(g[:, t])[..., None, None] * S
        err = beta[:, t, :, None] * (v[:, t] - torch.einsum("nhkv,nhk->nhv", S, k[:, t]))
        S = S + torch.einsum("nhk,nhv->nhkv", k[:, t], err)
        outs.append(scale * torch.einsum("nhkv,nhk->nhv", S, q[:, t]))
    return torch.stack(outs, 1), S


def _one_head_unrolled(q, k, v, g, beta, S, scale):
    """One sequence and head, all tokens at once: what each token writes solves a triangular system over the whole sequence."""
    G = torch.cumsum(g, 0)
    gap = G[:, None] - G[None, :]
    lower = torch.ones_like(gap, dtype=torch.bool).tril()
    fade = torch.where(lower, gap, torch.full_like(gap, -torch.inf)).exp()
    system = torch.eye(len(g), dtype=g.dtype, device=g.device) + torch.tril(beta[:, None] * (k @ k.T) * fade, -1)
    right = beta[:, None] * (v - torch.exp(G)[:, None] * (k @ S))
    wrote = torch.linalg.solve_triangular(system, right, upper=False, unitriangular=True)
    out = scale * (torch.exp(G)[:, None] * (q @ S) + ((q @ k.T) * fade) @ wrote)
    return out, torch.exp(G[-1]) * S + k.T @ (torch.exp(G[-1] - G)[:, None] * wrote)


def _exact_train(s):
    case = s["case"]
    names = ["q", "k", "v", "g", "beta"]
    wide = {n: s[n].detach().double().flatten(0, 1).requires_grad_() for n in names}
    N = case["nseq"] or case["batch"]
    lens = s["lens"] or [case["tokens"]] * N
    S0 = (s["state"].detach().double() if case["state"] else torch.zeros(N, case["hv"], case["dk"], case["dv"], device="cuda").double())
    dout = s["dout"].double().flatten(0, 1)
    out = torch.zeros_like(wide["v"])
    last, dS = torch.zeros_like(S0), torch.zeros_like(S0)
    d = {n: torch.zeros_like(wide[n]) for n in names}
    group, scale, a = case["hv"] // case["hk"], case["dk"] ** -0.5, 0
    for n, length in enumerate(lens):
        for h in range(case["hv"]):
            heads = dict(q=h // group, k=h // group, v=h, g=h, beta=h)
            x = [wide[m][a:a + length, heads[m]].detach().requires_grad_() for m in names] + [S0[n, h].detach().requires_grad_()]
            o, e = _one_head_unrolled(*x, scale)
            tops, back = [o], [dout[a:a + length, h]]
            if case["state"]:
                tops, back = [o, e], back + [s["dfinal"][n, h].double()]
            got = torch.autograd.grad(tops, x, back)
            out.data[a:a + length, h], last[n, h], dS[n, h] = o.detach(), e.detach(), got[5]
            for m, y in zip(names, got):
                d[m][a:a + length, heads[m]] += y
        a += length
    r = {"out": out.detach().reshape(s["v"].shape), "state": last if case["state"] else None}
    r.update({"d" + m: d[m].reshape(s[m].shape) for m in names})
    if case["state"]:
        r["dstate"] = dS
    return r


def _exact_conv(s):
    case = s["case"]
    L, W = case["tokens"], case["width"]
    x, dout, w, b = (s[n].detach().double() for n in ("x", "dout", "w", "b"))
    seq = s["seq_idx"]

    def before(z):
        y = b[:, None].expand_as(z).clone()
        for j in range(W):
            n = W - 1 - j
            same = seq[:, n:] == seq[:, :L - n] if seq is not None else torch.ones(case["batch"], max(0, L - n), device=z.device, dtype=torch.bool)
            y[..., n:] = y[..., n:] + w[:, j, None] * z[..., :max(0, L - n)] * same.unsqueeze(1)
        return y

    y = before(x)
    out = y / (1 + torch.exp(-y))
    # the 8-bit copy: a scale 2^e that is the least with every neighbour within e4m3's largest number, 448
    z = (x.mT if case["last"] else x).contiguous()
    n = z.shape[-1]
    groups = torch.cat([z, z.new_zeros(*z.shape[:-1], -n % _GROUP)], -1).reshape(*z.shape[:-1], -1, _GROUP)
    most = groups.abs().max(-1, keepdim=True).values
    e = torch.ceil(torch.log2(torch.where(most > 0, most, torch.full_like(most, 448.)) / 448))
    at = groups / torch.exp2(e)
    # e4m3: four significant bits down to 2^-6, steps of 2^-9 below; ties to even
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(at.abs().clamp(min=2.0 ** -20))), min=-6) - 3)
    z = (torch.round(at / step) * step * torch.exp2(e)).reshape(*z.shape[:-1], -1)[..., :n]
    kept = z.mT if case["last"] else z
    y = before(kept)
    sg = 1 / (1 + torch.exp(-y))
    dy = dout * (sg + y * sg * (1 - sg))
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for j in range(W):
        m = W - 1 - j
        if m >= L:
            continue
        same = (seq[:, m:] == seq[:, :L - m]).unsqueeze(1) if seq is not None else 1.0
        at = dy[..., m:] * same
        dx[..., :L - m] += w[:, j, None] * at
        dw[:, j] = (kept[..., :L - m] * at).sum((0, 2))
    return {"out": out, "dx": dx, "dw": dw, "db": dy.sum((0, 2))}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "conv":
        return _exact_conv(s)
    if case["kind"] == "train":
        return _exact_train(s)
    group, scale = case["hv"] // case["hk"], case["dk"] ** -0.5
    q, k, v, g, beta = (s[n].double() for n in ("q", "k", "v", "g", "beta"))
    if case["kind"] == "decode":
        if case["tokens"] == 1:
            q, k, v, g, beta = (x[:, None] for x in (q, k, v, g, beta))
        q, k = (x.repeat_interleave(group, 2) for x in (q, k))
        out, last = _token_by_token(q, k, v, g, beta, s["state"][s["rows"].long()].double(), scale)
        state = s["state"].double()
        state[s["rows"].long()] = last
        return {"out": out[:, 0] if case["tokens"] == 1 else out, "state": state}
    q, k = (x.repeat_interleave(group, 1) for x in (q, k))
    outs, a = [], 0
    state = s["state"].double() if case["state"] else None
    for n, length in enumerate(s["lens"]):
        S = torch.zeros(1, case["hv"], case["dk"], case["dv"], dtype=torch.float64, device="cuda")
        if case["state"] and n % 2 == 0:
            S = s["state"][s["rows"][n].long()].double()[None]
        o, S = _token_by_token(*(x[None, a:a + length] for x in (q, k, v, g, beta)), S, scale)
        outs.append(o[0])
        if case["state"]:
            state[s["rows"][n].long()] = S[0]
        a += length
    return {"out": torch.cat(outs), "state": state}
