"""The gated delta rule, the sequence mixer that the convolution's output (q, k and v) goes into:
``gated_delta_rule_fn`` (whole sequences, forward and backward), ``gated_delta_rule_varlen_fn``
(packed prefill over a pool of states) and ``gated_delta_rule_update`` (decode step), the
counterparts of ``causal_conv1d_fn``, ``causal_conv1d_varlen_fn`` and ``causal_conv1d_update``.
The reference has no such operator.

Per sequence and value head, with a state S of (dim_k, dim_v) in float32 and a_t = exp(g_t)::

    S_t = a_t S_{t-1} + k_t (beta_t (v_t - a_t S_{t-1}^T k_t))^T
    o_t = scale * S_t^T q_t

Value head h uses key head h // (heads_v // heads_k).  dim_k and dim_v are multiples of 8 up to 128.
g, the logarithm of the decay, is meant to be at most 0; sums of positive ones above 88 within 64 tokens leave
float32.  A token that is not finite, or whose products leave float32, makes the outputs of itself and those behind it
in its sequence and head NaN, none before.  Gradients: a v that is not finite makes those of q, k, g and beta NaN from
its token on, none before, and leaves those of v and of initial_state; any other tensor (q, k, g, beta, an output's
gradient) that is not finite, and keys whose products overflow, may make all gradients of the sequence and head NaN.
The calls run eagerly: torch.compile leaves a break in its graph at them.  A call takes its workspace from the caching allocator on the current stream, so calls on several streams, and
captured graphs, have one each.
"""
import torch
from torch import Tensor

from causal_conv1d_b200._ext import ext as _ext


def _rows(t: Tensor) -> Tensor:
    """t where the chunked kernels' 16-byte loads can read it, else a dense copy."""
    step = 16 // t.element_size()
    ok = t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(n <= 1 or s % step == 0 for n, s in zip(t.shape[:-1], t.stride()))
    return t if ok else _dense_copy(t)


def _dense_copy(t: Tensor) -> Tensor:
    # (contiguous() returns a contiguous t itself, wherever in its storage that begins)
    return t.clone(memory_format=torch.contiguous_format)


class GatedDeltaRuleFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, initial_state=None, return_final_state=False, cu_seqlens=None, scale=None):
        q, k, v = _rows(q), _rows(k), _rows(v)
        if initial_state is not None:
            dense = initial_state.is_contiguous() and initial_state.data_ptr() % 16 == 0
            initial_state = initial_state if dense else _dense_copy(initial_state)
        if cu_seqlens is not None:
            cu_seqlens = cu_seqlens.to(torch.int32).contiguous()
        scale = q.shape[-1] ** -0.5 if scale is None else scale
        out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
        n = q.shape[0] if cu_seqlens is None else cu_seqlens.shape[0] - 1
        final_state = None
        if return_final_state:
            final_state = torch.empty(n, v.shape[2], q.shape[3], v.shape[3], dtype=torch.float32, device=v.device)
        if initial_state is not None and initial_state.shape[0] != n:
            raise RuntimeError("initial_state must have one row per sequence")
        _ext.gated_delta_rule_fwd(q, k, v, g, beta, cu_seqlens, initial_state, final_state, None, None, out, scale)
        ctx.save_for_backward(q, k, v, g, beta, initial_state, cu_seqlens)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return (out, final_state) if return_final_state else out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dfinal_state=None):
        q, k, v, g, beta, initial_state, cu_seqlens = ctx.saved_tensors
        if dout is None:
            dout = torch.zeros(v.shape, dtype=v.dtype, device=v.device)
        if dfinal_state is not None:
            dfinal_state = dfinal_state.contiguous()
        dq, dk, dv, dg, dbeta = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v, g, beta))
        dinitial_state = None
        if initial_state is not None and ctx.needs_input_grad[5]:
            dinitial_state = torch.empty(initial_state.shape, dtype=torch.float32, device=v.device)
        _ext.gated_delta_rule_bwd(q, k, v, g, beta, cu_seqlens, initial_state, _rows(dout), dfinal_state,
                                  dq, dk, dv, dg, dbeta, dinitial_state, ctx.scale)
        return dq, dk, dv, dg, dbeta, dinitial_state, None, None, None


def gated_delta_rule_fn(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    g: Tensor,
    beta: Tensor,
    initial_state: Tensor | None = None,
    return_final_state: bool = False,
    cu_seqlens: Tensor | None = None,
    scale: float | None = None,
):
    """
    Whole sequences, with gradients for q, k, v, g, beta and initial_state.

    q, k: (batch, seqlen, heads_k, dim_k), contiguous along dim_k (slices of a wider tensor are read in
        place where their rows are 16-byte aligned)
    v: (batch, seqlen, heads_v, dim_v), dtype of q (float32, float16 or bfloat16)
    g, beta: (batch, seqlen, heads_v), float32, float16 or bfloat16; g is the logarithm of the decay
        (-inf: the state is forgotten)
    initial_state: (sequences, heads_v, dim_k, dim_v) float32; zeros when None
    cu_seqlens: (nseq + 1,) int32: the one row of the batch holds nseq packed sequences, sequence s at
        tokens cu_seqlens[s]:cu_seqlens[s+1]; tokens before the first and behind the last one have zero
        outputs and gradients
    scale: factor of the output, dim_k ** -0.5 when None

    out: (batch, seqlen, heads_v, dim_v); with return_final_state also (sequences, heads_v, dim_k, dim_v)

    The backward computes the forward's states again; it needs about 244 KB of workspace for each 64
    tokens of a value head while it runs, whatever dim_k and dim_v are: 1 GB for 8192 tokens of 32 heads. Sums are
    taken in a fixed order.
    """
    return GatedDeltaRuleFn.apply(q, k, v, g, beta, initial_state, return_final_state, cu_seqlens, scale)


def gated_delta_rule_update(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    g: Tensor,
    beta: Tensor,
    state: Tensor,
    state_indices: Tensor | None = None,
    scale: float | None = None,
) -> Tensor:
    """
    Decode step: one token, or a few drafted ones, for each row of a batch. Forward only.

    q, k: (batch, heads_k, dim_k) or (batch, seqlen, heads_k, dim_k)
    v: (batch, heads_v, dim_v) or (batch, seqlen, heads_v, dim_v), dtype of q
    g, beta: (batch, heads_v) or (batch, seqlen, heads_v), float32, float16 or bfloat16;
        g is the logarithm of the decay (-inf: the state is forgotten)
    state: (rows, heads_v, dim_k, dim_v) float32, dense in its last two dimensions; updated in place
    state_indices: (batch,), dtype int32.
        If not None, row state_indices[b] is the state of batch row b; an index that is negative
        or not below the number of rows marks a padded row (zero output, no state touched). No
        two batch rows may name the same state.
    scale: factor of the output, dim_k ** -0.5 when None

    out: (batch, heads_v, dim_v) or (batch, seqlen, heads_v, dim_v)
    """
    return _ext.gated_delta_rule_update(q, k, v, g, beta, state, state_indices,
                                        q.shape[-1] ** -0.5 if scale is None else scale)


def gated_delta_rule_varlen_fn(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    g: Tensor,
    beta: Tensor,
    *,
    cu_seqlens: Tensor,
    states: Tensor | None = None,
    state_indices: Tensor | None = None,
    has_initial_state: Tensor | None = None,
    update_states: bool = True,
    scale: float | None = None,
) -> Tensor:
    """
    Packed variable-length prefill that continues from, and leaves behind, per-sequence states: the
    counterpart of ``causal_conv1d_varlen_fn``. Forward only.

    Parameters:
        q, k: (total_tokens, heads_k, dim_k); sequence s owns rows cu_seqlens[s]:cu_seqlens[s+1]
        v: (total_tokens, heads_v, dim_v), dtype of q
        g, beta: (total_tokens, heads_v), float32, float16 or bfloat16; g: logarithm of the decay
        cu_seqlens: (nseq + 1,) int32, non-decreasing, its last entry at most total_tokens
        states: (rows, heads_v, dim_k, dim_v) float32, dense in its last two dimensions, or None.
            Row r = state_indices[s] (s when state_indices is None) holds sequence s's state. An
            index that is negative or not below the number of rows: the sequence starts from
            zeros and stores nothing. No two sequences may name the same row.
        has_initial_state: (nseq,) bool or None.  Where True (everywhere when None and states is
            given) the sequence starts from its row; elsewhere from zeros.
        update_states: write each sequence's last state back into its row of states (in place).
        scale: factor of the output, dim_k ** -0.5 when None
    Return:
        out: (total_tokens, heads_v, dim_v); tokens before cu_seqlens[0], and at or after cu_seqlens[-1], are zero
    """
    q, k, v, g, beta = (t.unsqueeze(0) for t in (q, k, v, g, beta))
    out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    if state_indices is not None:
        state_indices = state_indices.to(torch.int32).contiguous()
    if has_initial_state is not None:
        has_initial_state = has_initial_state.to(torch.bool).contiguous()
    _ext.gated_delta_rule_fwd(
        _rows(q), _rows(k), _rows(v), g, beta, cu_seqlens.to(torch.int32).contiguous(),
        states, states if update_states else None, state_indices if states is not None else None,
        has_initial_state, out, q.shape[-1] ** -0.5 if scale is None else scale)
    return out.squeeze(0)
