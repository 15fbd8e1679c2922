"""Training operators: attention with its gradient, and rotary positions over several axes.

:func:`rotary_axes` turns queries and keys by their tokens' positions (time,
height, width, ...), :func:`sageattn_train` attends over them, and both have
backward passes of their own gfx950 kernels.  The reference has neither (its
``sageattn`` output carries no gradient).  Like ``sageattn``, every call is
asynchronous on the current stream of the tensors' device and allocates from
torch's caching allocator; gradients run on the stream of their forward call.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import torch

from . import core


def sageattn_train(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    tensor_layout: str = "HND",
    is_causal: bool = False,
    sm_scale: Optional[float] = None,
    return_lse: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Softmax attention that can be differentiated: the direct fp16/bf16 kernel of ``sageattn``
    forward (Q and K as they are, for any length), and a backward pass that recomputes the
    probabilities from the rows' log-sum-exp.

    Arguments, layouts, grouped heads and the causal mask (query i sees keys 0..i) are those of
    ``sageattn``; fp16 or bf16, head_dim 64 or 128.  Saved for the backward pass: q, k, v, the
    output and the LSE.  With ``return_lse`` the LSE ([B,Hq,Sq] fp32) is returned too, and its
    gradient is taken into account.  Gradients are deterministic (no atomics); dk and dv sum over
    the query heads that share a kv head.  They cannot be differentiated a second time, and there are
    no forward-mode derivatives (asking for either raises).

    A row without a live key (all its scores -inf) gets output 0, LSE -inf and zero gradients.  The
    backward pass takes exp(score - LSE) in fp32, which is off by about 2^-22 |LSE| of itself: scores
    beyond some 10^4 cost precision, and from 2^21 on it means nothing.  A row whose LSE is below
    -2^21 (all its keys masked by a large finite value; the output is their mean, or with key splits
    that of the splits' by LSEs of fp32) has zero gradients, scores above 2^21 are outside the range.  K and V have to be finite, masked or not, and bf16 V
    within fp16's range (65504), as the forward kernel takes it.
    """
    return core._host().sageattn_train(q, k, v, tensor_layout, is_causal, sm_scale, return_lse)


def sageattn_backward(
    dout: torch.Tensor,
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    out: torch.Tensor,
    lse: torch.Tensor,
    tensor_layout: str = "HND",
    is_causal: bool = False,
    sm_scale: Optional[float] = None,
    dlse: Optional[torch.Tensor] = None,
    smooth_k: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dq, dk, dv) of an attention call from its inputs, its output and its log-sum-exp, for
    programs that keep those themselves: ``out, lse = sageattn(..., return_lse=True)`` (of either
    path; the quantised path's rounding of Q and K is then taken as the identity, and a probability
    exp(score - lse) that comes out above 1 by it counts as 1), or attention over key ranges merged
    by their LSEs (pass the merged output and LSE with each range's k, v).

    dout and out have q's shape, layout and dtype; lse and dlse (the LSE's gradient, optional) are
    [B,Hq,Sq] fp32.

    ``smooth_k`` has to be what the forward call was given: with it the INT8 path attends over k minus
    its mean over the tokens, and its LSE is that of those scores.  (The output and the gradients do
    not depend on the shift; short calls, which take the direct kernel, have none.)  The LSEs of
    smoothed calls over several key ranges cannot be merged, each having its own shift, and dlse is
    refused with it."""
    if smooth_k and getattr(q, "ndim", 0) == getattr(k, "ndim", 0) == 4 and tensor_layout in ("HND", "NHD"):
        seq = 2 if tensor_layout == "HND" else 1
        smooth_k = not core.use_direct_path(q.shape[3], q.shape[seq], k.shape[seq], bool(is_causal), tensor_layout)
    return core._host().sageattn_backward(dout, q, k, v, out, lse, tensor_layout, is_causal, sm_scale, dlse,
                                          bool(smooth_k))


def rotary_axes(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    positions: torch.Tensor,
    axes_dim: Sequence[int],
    theta: Union[float, Sequence[float]] = 10000.0,
    tensor_layout: str = "HND",
    interleaved: bool = True,
    inverse: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Rotary positions with several axes (an image's height and width, a video's time, height and
    width, one axis for text), of queries and keys in one launch; differentiable, any number of
    times, in q and k (not in forward mode, which raises).

    q: [B,Hq,N,D] (HND) or [B,N,Hq,D] (NHD), fp16, bf16 or fp32, D 64 or 128; k likewise with its
    own head count, or None (then one tensor is returned).  positions: [N, A] or [B, N, A], int32,
    int64 or float32 (no gradient): a token's position on each of the A axes.  axes_dim: the A even
    widths, their sum R at most D.  Pair j of axis a turns by positions[a] * theta_a^(-2j/axes_dim[a]),
    (x, y) -> (x cos - y sin, x sin + y cos); theta is one number or one per axis.  The pairs, counted
    through the axes in order, are elements (2i, 2i+1) when ``interleaved``, else (i, i + R/2).
    Elements past R are copied.  ``inverse`` turns the other way.  Angles are reduced in 64 bits and off by
    about 2^-50 of themselves (int64 positions are taken to fp64); the rotation is fp32, rounded once.
    """
    return core._host().rotary_axes(q, k, positions, axes_dim, theta, tensor_layout, interleaved, inverse)
