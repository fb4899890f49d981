"""Sequence operators of the agents, as hand-written HIP kernels (csrc/sequence/, C ABI in include/pvder_sequence.h):

* :func:`decay_attention` -- linear attention whose memory decays by a factor per head, over whole windows, with its gradient;
* :func:`decay_attention_step` -- the same, one env step of every env, the state updated in place;
* :func:`gated_residual_norm` -- norm behind a block, gate, residual scale and norm before the next block in one pass, with its
  gradient.

An agent that has to infer what an observation does not show (the parameters of a randomised env, the grid's next moves) needs a
memory.  This one has a fixed size per env, so that 65 536 envs act in one launch, and the same function is trained on whole
windows in parallel.  ``agents/sequence.py`` holds the network and the agent that use them.

All calls are asynchronous on the current stream of the inputs' device, can be captured into a HIP graph, and refuse (``ValueError``,
``TypeError``) what the kernels do not take: forward-mode tangents, ``torch.func`` transforms, tracing (``torch.jit.trace``, ``make_fx``)
and tensors that wrap others among it.  There is no CPU fallback.  Checks, outputs and autograd nodes are in
csrc/sequence/torch_binding.cpp.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from .. import _native

MAX_HEAD, MAX_WIDTH = 128, 8192                      # include/pvder_sequence.h


def decay_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, *, scale: Optional[float] = None,
                    initial_state: Optional[torch.Tensor] = None, starts: Optional[torch.Tensor] = None,
                    lengths: Optional[torch.Tensor] = None,
                    output_final_state: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Linear attention with a decay for each head, over windows of T tokens.

    Per batch row and head, with g = exp(log_decay[h]) and a state S [DK, DV] in fp32::

        S_t = g S_{t-1} + k_t v_t^T            o_t = scale S_t^T q_t

    Args:
        q, k:  [B, T, H, DK] float32 or bfloat16; v: [B, T, H, DV] of the same type.  DK, DV in 1 .. 128.  Any strides, views of a
               packed projection for instance (a last dimension that is not dense is copied).
        log_decay: [H] float32, <= 0; a larger value or NaN counts as 0 (no decay), -inf remembers nothing.  A constant: it gets no
               gradient, and one that requires it is refused.
        scale: of the output, default DK ** -0.5.
        initial_state: [B, H, DK, DV] float32, S before the first token (default zeros).
        starts: [B, T] bool or uint8: an episode starts at this token, and nothing before it (nor ``initial_state``) counts from there on.
        lengths: [B] int32: tokens of each row (taken into 0 .. T).  Tokens behind them are not read; their output and gradients are 0.
        output_final_state: also return the state behind the last token of each row, [B, H, DK, DV] float32.

    Differentiable once in q, k, v and initial_state, through both outputs.  A value that is not finite reaches its own token and the
    later ones of its episode (in a gradient: the earlier ones), as in the recurrence above; an infinity may arrive as NaN.  A weight of
    zero, which a decay of -inf, one small enough or a start reaches, clears also what is not finite.

    States and all sums are held in float32.  With bfloat16 inputs the scores and the state are rounded to bfloat16 where they enter the
    products that make outputs and gradients of that type: an output is off by about 1.4 roundings of its own; float32 inputs have none of
    this.  A state that is returned (``output_final_state``, the gradient of ``initial_state``) is made of products of 24 bits, else of 16, so
    the last bits of bfloat16 results can depend on whether it is asked for.  Any call repeated gives the same bits.

    A capture into a HIP graph is refused (``RuntimeError``) where q, k, v or initial_state is a leaf, or a view of one, of a graph that lives
    on another stream: the backward pass would end the process.  Of few, long windows whose gradients are wanted the forward pass keeps up to
    33 MB of states besides its inputs.
    """
    return _native.sequence_torch().decay_attention(q, k, v, log_decay, scale, initial_state, starts, lengths, output_final_state)


def decay_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, state: torch.Tensor, *,
                         scale: Optional[float] = None, starts: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of :func:`decay_attention` for N rows (envs): returns o [N, H, DV] and updates ``state`` in place.

    Args:
        q, k: [N, H, DK], v: [N, H, DV], float32 or bfloat16, any strides; log_decay, scale: as for the window form.
        state: [N, H, DK, DV] float32, contiguous; must not overlap the other tensors.
        starts: [N] bool or uint8: an episode starts with this token; nothing of the row's state before it counts.

    As in the window form a weight of zero (a decay of -inf, a start) clears also a state that is not finite.

    For acting and evaluation: it has no gradient, and refuses tensors that would ask for one.
    """
    return _native.sequence_torch().decay_attention_step(q, k, v, log_decay, state, scale, starts)


def gated_residual_norm(residual: torch.Tensor, y: torch.Tensor, post_weight: torch.Tensor, pre_weight: torch.Tensor, *,
                        gate: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
                        eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """The residual stream between two blocks, in one pass::

        h = residual + scale * sigmoid(gate) * (y / rms(y)) * post_weight
        x = (h / rms(h)) * pre_weight                                             rms(z) = sqrt(mean(z ** 2) + eps)

    Args:
        residual, y, gate: [..., D] float32 or bfloat16, all alike, D in 1 .. 8192; ``gate`` None: no gate.
        post_weight (the norm behind the block), pre_weight (the norm before the next), scale (of the residual branch; None: 1):
               [D] float32, contiguous.
        eps: >= 0, inside the root.

    Returns (h, x), both contiguous and of the inputs' type; x is taken from h before its rounding.  Differentiable once in every
    tensor.  A row that is not finite stays alone in h, x and its own gradients, and reaches the gradients of the three weights.
    """
    return _native.sequence_torch().gated_residual_norm(residual, y, post_weight, pre_weight, gate, scale, eps)
