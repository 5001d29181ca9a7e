"""The other mixers of a hybrid layer: the gated delta rule and causal attention.

``gated_delta_scan`` and ``gated_delta_step`` are the decay scan's content-dependent
form in the same two modes: whole sequences with a backward, and one token
for a batch with the state of each head carried.  ``causal_attention`` is what
the recall heads beside them run over a prompt (/root/reference/src/kilat/arc/
attention.py:400-518 calls torch's scaled_dot_product_attention there).

As everywhere in this package only HIP tensors are accepted; the work is
enqueued on torch's current stream of q's device, with no synchronisation.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import triton_ops


def _native():
    return triton_ops._native


def _tensors(**ts) -> None:
    for name, t in ts.items():
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"kilat_amd: {name} must be a torch.Tensor")


def gated_delta_scan(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor,
    beta: torch.Tensor,
    *,
    scale: Optional[float] = None,
    initial_state: Optional[torch.Tensor] = None,
    return_final_state: bool = False,
    cu_seqlens: Optional[torch.Tensor] = None,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """The gated delta rule over whole sequences, per head with a state S of [Dk, Dv]:

        S_t = exp(g_t) (S_{t-1} - beta_t k_t (k_t' S_{t-1})) + beta_t k_t v_t'
        o_t = scale S_t' q_t

    q, k: [B,Hk,N,Dk]; v: [B,H,N,Dv], one of float32/bfloat16/float16, any strides (views
    of a projection are read as they are; channels that are not adjacent are
    copied).  H is a multiple of Hk: head h uses key head h // (H // Hk).  1 <= Dk <= 128,
    1 <= Dv <= 256.  Keys are used as given: normalise them before (a key longer
    than 1 / sqrt(beta) makes the state grow).
    g, beta: [B,H,N] log decays (up to 0; -inf forgets everything before) and write
    strengths, any float dtype, used as float32.
    scale: default Dk ** -0.5.  initial_state: [B,H,Dk,Dv], default zeros.
    cu_seqlens: int32/int64 [S+1] on the device, non-decreasing, for a packed
    batch (B=1): sequence s is the rows cu_seqlens[s]..cu_seqlens[s+1], and the
    states are [S,H,Dk,Dv].  Its values are never read on the host.  Rows of no
    sequence give zeros, in o and in the gradients.  (Its mean length decides into how
    many pieces the sequences are cut.)

    Returns o ([B,H,N,Dv], v's dtype, laid out like v), and with
    return_final_state also the final states (float32).  Arithmetic is float32
    whatever the dtype (what reaches only a 16-bit o: to 2^-16), and o is rounded
    once.  A value that is not finite reaches
    the tokens from its own on, in the columns and heads it reaches by the formula.

    With requires_grad on any input the result carries a backward (gradients of q,
    k, v, g, beta and initial_state, through both outputs), bit for bit
    reproducible.  It keeps the inputs, not copies.  In a chunk of 64 tokens that
    holds a value that is not finite, and before it in the same sequence, gradients
    are not finite either.
    """
    _tensors(q=q, k=k, v=v, g=g, beta=beta)
    return _native().gated_delta_scan(q, k, v, g, beta, scale, initial_state, bool(return_final_state), cu_seqlens)


def gated_delta_step(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor,
    beta: torch.Tensor,
    state: torch.Tensor,
    *,
    scale: Optional[float] = None,
    out: Optional[torch.Tensor] = None,
    new_state: Optional[torch.Tensor] = None,
    out_dtype: Optional[torch.dtype] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """One token of the gated delta rule for the whole batch, one launch.

    q, k: [B,Hk,Dk]; v: [B,H,Dv]; g, beta: [B,H]; state: [B,H,Dk,Dv] (used as
    float32, as the scan's final state is).  new_state may be the state itself
    (in place).  Returns (out [B,H,Dv], v's dtype or out_dtype, which may also be
    float32; new_state [B,H,Dk,Dv] float32).  Computes no gradient, as decay_step.
    """
    _tensors(q=q, k=k, v=v, g=g, beta=beta, state=state)
    return _native().gated_delta_step(q, k, v, g, beta, state, scale, out, new_state, out_dtype)


def causal_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    scale: Optional[float] = None,
    cu_seqlens: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """o_i = sum_{j<=i} softmax_j(scale q_i.k_j) v_j over whole prompts.

    q: [B,H,N,Dk]; k: [B,Hk,N,Dk]; v: [B,Hk,N,Dv], one of float32/bfloat16/float16, any
    strides.  H is a multiple of Hk: head h uses key head h // (H // Hk).  1 <= Dk,
    Dv <= 128.  scale: default Dk ** -0.5.  cu_seqlens: as in gated_delta_scan;
    rows of no sequence give zeros.

    Returns o [B,H,N,Dv] of q's dtype, laid out like q.  Softmax statistics and
    sums are float32; of 16-bit inputs the probabilities are rounded to the type, as the
    second product's operands.  No row sees a later one's values, finite or not.  A prefill's forward: inputs that require grad are refused.
    """
    _tensors(q=q, k=k, v=v)
    return _native().causal_attention(q, k, v, scale, cu_seqlens)


__all__ = ["gated_delta_scan", "gated_delta_step", "causal_attention"]
