"""The gated delta rule, the sequence mixer that the convolution's output (q, k and v) goes into:
``gated_delta_rule_fn`` (whole sequences, forward and backward), ``gated_delta_rule_varlen_fn``
(packed prefill over a pool of states) and ``gated_delta_rule_update`` (decode step), the
counterparts of ``causal_conv1d_fn``, ``causal_conv1d_varlen_fn`` and ``causal_conv1d_update``.
The reference has no such operator.

Per sequence and value head, with a state S of (dim_k, dim_v) in float32 and a_t = exp(g_t)::

    S_t = a_t S_{t-1} + k_t (beta_t (v_t - a_t S_{t-1}^T k_t))^T
    o_t = scale * S_t^T q_t

Value head h uses key head h // (heads_v // heads_k).  dim_k and dim_v are multiples of 8 up to 128.
"""
import torch
from torch import Tensor

from causal_conv1d_b200._ext import ext as _ext


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
    squeeze = q.dim() == 3
    if squeeze:
        q, k, v, g, beta = (t.unsqueeze(1) for t in (q, k, v, g, beta))
    out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    _ext.gated_delta_rule_update(q, k, v, g, beta, state, state_indices, out,
                                 q.shape[-1] ** -0.5 if scale is None else scale)
    return out.squeeze(1) if squeeze else out
