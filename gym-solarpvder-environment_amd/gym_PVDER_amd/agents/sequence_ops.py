"""Sequence operators of the agents, as hand-written HIP kernels (csrc/sequence/, C ABI in include/pvder_sequence.h):

* :func:`decay_attention` -- linear attention whose memory decays by a factor per head, over whole windows, with its gradient;
* :func:`decay_attention_step` -- the same, one env step of every env, the state updated in place;
* :func:`gated_residual_norm` -- norm behind a block, gate, residual scale and norm before the next block in one pass, with its
  gradient.

An agent that has to infer what an observation does not show (the parameters of a randomised env, the grid's next moves) needs a
memory.  This one has a fixed size per env, so that 65 536 envs act in one launch, and the same function is trained on whole
windows in parallel.  ``agents/sequence.py`` holds the network and the agent that use them.

All calls are asynchronous on the current stream of the inputs' device, can be captured into a HIP graph, and refuse (``ValueError``,
``TypeError``) what the kernels do not take.  There is no CPU fallback.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import math
import struct
from typing import Optional, Tuple, Union

import torch

from .. import _native

MAX_HEAD, MAX_WIDTH, MAX_TOKEN_STRIDE = 128, 8192, 1 << 26     # include/pvder_sequence.h
_DTYPES = {torch.float32: 0, torch.bfloat16: 1}

# struct pvder_seq_scan, pvder_seq_attn, pvder_seq_step, pvder_seq_norm
_SCAN = struct.Struct("@4Q12q2Q4q3f3i")
_ATTN_TAIL = struct.Struct("@4Q2q6i")
_STEP = struct.Struct("@4Q8q3Q1q5i1f")
_NORM = struct.Struct("@3Q3q6Q2Q2q5Q1q2i1f4x")
_MAX_SCANS = 3
_ATTN_BYTES = _MAX_SCANS * _SCAN.size + _ATTN_TAIL.size
_SEGMENTS_AT = _ATTN_BYTES - 4
_WORKSPACE_AT = _MAX_SCANS * _SCAN.size + 24


def _need(cond: bool, what: str) -> None:
    if not cond:
        raise ValueError(what)


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _gpu(name: str, t: torch.Tensor) -> None:
    _need(t.is_cuda, "%s is on %s: the kernels need a GPU, there is no CPU path" % (name, t.device))


def _on(device: torch.device):
    """The device of the call, made current if it is not, and its current stream."""
    ctx = contextlib.nullcontext() if torch.cuda.current_device() == device.index else torch.cuda.device(device)
    return ctx, torch.cuda.current_stream(device).cuda_stream


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with unit stride in its last dimension (a copy only where it has another)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _tokens(t: torch.Tensor) -> torch.Tensor:
    """``_rows`` of a [B, T, H, D] tensor whose tokens lie near enough for the kernels' 32-bit offsets within a chunk."""
    t = _rows(t)
    return t if t.stride(1) * t.element_size() <= MAX_TOKEN_STRIDE else t.contiguous()


def _tensors(device: Optional[torch.device], **tensors) -> torch.device:
    """Checks that all are tensors on one device (the first one's, or ``device``)."""
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor):
            raise TypeError("%s must be a tensor: got %s" % (name, type(t).__name__))
        if device is None:
            device = t.device
        _need(t.device == device, "%s is on %s, the call on %s" % (name, t.device, device))
    return device


def _given(**tensors) -> dict:
    return {n: t for n, t in tensors.items() if t is not None}


def _qkv(q, k, v, log_decay, dims: str):
    """Checks what the window form and the step form share; returns (H, DK, DV)."""
    _tensors(None, q=q, k=k, v=v, log_decay=log_decay)
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("q, k and v must be float32 or bfloat16, all three alike: got %s, %s, %s" % (q.dtype, k.dtype, v.dtype))
    _need(q.dim() == len(dims.split(",")) and k.dim() == q.dim() and v.dim() == q.dim(), "q, k and v must be [%s]" % dims)
    _need(k.shape == q.shape, "q and k differ in shape: %s, %s" % (tuple(q.shape), tuple(k.shape)))
    _need(v.shape[:-1] == q.shape[:-1], "v must be [%s] beside q: got %s, %s" % (dims, tuple(v.shape), tuple(q.shape)))
    H, DK, DV = q.shape[-2], q.shape[-1], v.shape[-1]
    _need(H >= 1 and 1 <= DK <= MAX_HEAD and 1 <= DV <= MAX_HEAD,
          "there must be a head, and heads must be 1 .. %d wide: got %d heads of %d and %d" % (MAX_HEAD, H, DK, DV))
    _need(q.numel() // max(1, H * DK) < 2 ** 31, "too many rows")
    if log_decay.dtype != torch.float32:
        raise TypeError("log_decay must be float32")
    _need(log_decay.shape == (H,) and log_decay.is_contiguous(), "log_decay must be a contiguous [%d], one for each head" % H)
    _need(not (log_decay.requires_grad and torch.is_grad_enabled()),
          "log_decay is a constant of the heads: the kernels give it no gradient; detach it")
    return H, DK, DV


def _scale(scale: Optional[float], dk: int) -> float:
    if scale is None:
        return dk ** -0.5
    if isinstance(scale, torch.Tensor) or not math.isfinite(scale):
        raise ValueError("scale must be a finite number")
    return float(scale)


def _flags(name: str, t: Optional[torch.Tensor], shape) -> None:
    if t is not None:
        if t.dtype not in (torch.bool, torch.uint8):
            raise TypeError("%s must be bool or uint8" % name)
        _need(tuple(t.shape) == tuple(shape), "%s must be %s: got %s" % (name, tuple(shape), tuple(t.shape)))


def _scan(q, k, v, o, s_in, s_out, s_strides, a_read, a_write, a_intra, reverse: bool) -> bytes:
    return _SCAN.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *o.stride()[:3],
                      _ptr(s_in), _ptr(s_out), *s_strides, a_read, a_write, a_intra, q.shape[3], v.shape[3], int(reverse))


def _run_scans(scans, shape, log_decay, starts, lengths, dtype) -> None:
    B, T, H = shape
    L = _native.sequence_lib()
    arg = bytearray(_ATTN_BYTES)
    for i, s in enumerate(scans):
        arg[i * _SCAN.size:(i + 1) * _SCAN.size] = s
    sb, st = starts.stride() if starts is not None else (0, 0)
    _ATTN_TAIL.pack_into(arg, _MAX_SCANS * _SCAN.size, log_decay.data_ptr(), _ptr(starts), _ptr(lengths), 0, sb, st, B, T, H, len(scans),
                         _DTYPES[dtype], 1)
    buf = (C.c_char * _ATTN_BYTES).from_buffer(arg)
    floats = L.pvder_seq_attn_plan(buf)
    if floats < 0:
        _native.check(int(floats), "pvder_seq_attn_plan")
    ctx, stream = _on(log_decay.device)
    with ctx:
        work = torch.empty(floats, dtype=torch.float32, device=log_decay.device) if floats else None
        struct.pack_into("@Q", arg, _WORKSPACE_AT, _ptr(work))
        rc = L.pvder_seq_attn_run(buf, stream)
    _native.check(rc, "pvder_seq_attn_run")


def _state_strides(t: Optional[torch.Tensor], H: int, DK: int, DV: int):
    return t.stride() if t is not None else (H * DK * DV, DK * DV, DV, 1)


def _attention_forward(q, k, v, log_decay, s_in, starts, lengths, scale, want_state):
    B, T, H, DK = q.shape
    DV = v.shape[3]
    out = torch.empty((B, T, H, DV), dtype=q.dtype, device=q.device)
    final = None
    if want_state:
        # (the state that goes out has the strides of the one that comes in: the kernel takes one set)
        final = torch.empty((B, H, DK, DV), dtype=torch.float32, device=q.device)
        if s_in is not None and not s_in.is_contiguous():
            s_in = s_in.contiguous()
    scan = _scan(q, k, v, out, s_in, final, _state_strides(s_in, H, DK, DV), scale, 1.0, scale, False)
    _run_scans([scan], (B, T, H), log_decay, starts, lengths, q.dtype)
    return out, final


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, s_in, starts, lengths, scale, want_state):
        ctx.set_materialize_grads(False)
        ctx.scale = scale
        ctx.save_for_backward(q, k, v, log_decay, s_in, starts, lengths)
        out, final = _attention_forward(q, k, v, log_decay, s_in, starts, lengths, scale, want_state)
        return (out, final) if want_state else out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dfinal=None):
        q, k, v, log_decay, s_in, starts, lengths = ctx.saved_tensors
        (B, T, H, DK), DV, scale = q.shape, v.shape[3], ctx.scale
        none = (None,) * 9
        if dout is None and dfinal is None:
            return none
        dev, dt = q.device, q.dtype
        dout = torch.zeros((B, T, H, DV), dtype=dt, device=dev) if dout is None else _tokens(dout)
        if dfinal is not None and not dfinal.is_contiguous():
            dfinal = dfinal.contiguous()
        need_q, need_k, need_v, _, need_s = ctx.needs_input_grad[:5]
        dq = dk = dv = ds = None
        scans = []
        if need_q:
            # dq_t = scale S_t do_t: the attention of do over (v, k), its state the transpose of S
            dq = torch.empty((B, T, H, DK), dtype=dt, device=dev)
            b, h, i, j = _state_strides(s_in, H, DK, DV)
            scans.append(_scan(dout, v, k, dq, s_in, None, (b, h, j, i), scale, 1.0, scale, False))
        plain = _state_strides(None, H, DK, DV)
        if need_k:
            dk = torch.empty((B, T, H, DK), dtype=dt, device=dev)
            scans.append(_scan(v, dout, q, dk, dfinal, None, (plain[0], plain[1], plain[3], plain[2]), 1.0, scale, scale, True))
        if need_v or need_s:
            dv = torch.empty((B, T, H, DV), dtype=dt, device=dev)
            ds = torch.empty((B, H, DK, DV), dtype=torch.float32, device=dev) if need_s else None
            scans.append(_scan(k, q, dout, dv, dfinal, ds, plain, 1.0, scale, scale, True))
        if scans:
            _run_scans(scans, (B, T, H), log_decay, starts, lengths, dt)
        return (dq, dk, dv if need_v else None, None, ds) + none[5:]


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
    later ones of its episode (in a gradient: the earlier ones), as in the recurrence above; an infinity may arrive as NaN.
    """
    H, DK, DV = _qkv(q, k, v, log_decay, "B, T, H, D")
    B, T = q.shape[:2]
    if not (initial_state is None and starts is None and lengths is None):
        _tensors(q.device, **_given(initial_state=initial_state, starts=starts, lengths=lengths))
        if initial_state is not None:
            if initial_state.dtype != torch.float32:
                raise TypeError("initial_state must be float32")
            _need(initial_state.shape == (B, H, DK, DV), "initial_state must be %s: got %s" % ((B, H, DK, DV), tuple(initial_state.shape)))
        _flags("starts", starts, (B, T))
        if lengths is not None:
            if lengths.dtype != torch.int32:
                raise TypeError("lengths must be int32")
            _need(lengths.shape == (B,) and lengths.is_contiguous(), "lengths must be a contiguous [%d]" % B)
    scale = _scale(scale, DK)
    _gpu("q", q)
    q, k, v = _tokens(q), _tokens(k), _tokens(v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or (initial_state is not None and initial_state.requires_grad)):
        return _DecayAttention.apply(q, k, v, log_decay, initial_state, starts, lengths, scale, bool(output_final_state))
    out, final = _attention_forward(q, k, v, log_decay, initial_state, starts, lengths, scale, output_final_state)
    return (out, final) if output_final_state else out


def decay_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, state: torch.Tensor, *,
                         scale: Optional[float] = None, starts: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of :func:`decay_attention` for N rows (envs): returns o [N, H, DV] and updates ``state`` in place.

    Args:
        q, k: [N, H, DK], v: [N, H, DV], float32 or bfloat16, any strides; log_decay, scale: as for the window form.
        state: [N, H, DK, DV] float32, contiguous; must not overlap the other tensors.
        starts: [N] bool or uint8: an episode starts with this token; the row's state is not read.

    For acting and evaluation: it has no gradient, and refuses tensors that would ask for one.
    """
    H, DK, DV = _qkv(q, k, v, log_decay, "N, H, D")
    N = q.shape[0]
    _tensors(q.device, state=state, **_given(starts=starts))
    if state.dtype != torch.float32:
        raise TypeError("state must be float32")
    _need(state.shape == (N, H, DK, DV) and state.is_contiguous(), "state must be a contiguous %s" % ((N, H, DK, DV),))
    _flags("starts", starts, (N,))
    _need(not (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad)),
          "the step form has no gradient: call it under torch.no_grad(), or train on windows with decay_attention")
    scale = _scale(scale, DK)
    _gpu("q", q)
    q, k, v = _rows(q), _rows(k), _rows(v)
    L = _native.sequence_lib()
    out = torch.empty((N, H, DV), dtype=q.dtype, device=q.device)
    arg = _STEP.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), *q.stride()[:2], *k.stride()[:2], *v.stride()[:2], *out.stride()[:2],
                     state.data_ptr(), log_decay.data_ptr(), _ptr(starts), starts.stride(0) if starts is not None else 0, N, H, DK, DV,
                     _DTYPES[q.dtype], scale)
    ctx, stream = _on(q.device)
    with ctx:
        rc = L.pvder_seq_step_run(arg, stream)
    _native.check(rc, "pvder_seq_step_run")
    torch.autograd.graph.increment_version(state)      # written behind autograd's back: a graph that saved it has to see that
    return out


# ---------------------------------------------------------------------------------------------------- gated residual norm
def _two(t: torch.Tensor, width: int) -> torch.Tensor:
    """``t`` as [rows, width] with dense rows (a view wherever its strides allow one)."""
    return _rows(t.reshape(-1, width))


def _norm_arg(h, y, gate, post, pre, scale, eps, h_out=None, x_out=None, stats=None, dh=None, dx=None, dh_out=None, dy_out=None,
              dgate_out=None, dparam=None, work=None) -> bytes:
    s = lambda t: 0 if t is None else t.stride(0)  # noqa: E731
    return _NORM.pack(_ptr(h), _ptr(y), _ptr(gate), s(h), s(y), s(gate), _ptr(post), _ptr(pre), _ptr(scale), _ptr(h_out), _ptr(x_out),
                      _ptr(stats), _ptr(dh), _ptr(dx), s(dh), s(dx), _ptr(dh_out), _ptr(dy_out), _ptr(dgate_out), _ptr(dparam), _ptr(work),
                      h.shape[0], h.shape[1], _DTYPES[h.dtype], eps)


def _norm_forward(h, y, post, pre, gate, scale, eps, want_stats):
    shape, D = h.shape, h.shape[-1]
    h2, y2, g2 = _two(h, D), _two(y, D), None if gate is None else _two(gate, D)
    R = h2.shape[0]
    h_out, x_out = torch.empty(shape, dtype=h.dtype, device=h.device), torch.empty(shape, dtype=h.dtype, device=h.device)
    stats = torch.empty((R, 2), dtype=torch.float32, device=h.device) if want_stats else None
    ctx, stream = _on(h.device)
    with ctx:
        rc = _native.sequence_lib().pvder_seq_norm_forward(_norm_arg(h2, y2, g2, post, pre, scale, eps, h_out, x_out, stats), stream)
    _native.check(rc, "pvder_seq_norm_forward")
    return h_out, x_out, stats


class _GatedResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, y, post, pre, gate, scale, eps):
        ctx.set_materialize_grads(False)
        h_out, x_out, stats = _norm_forward(h, y, post, pre, gate, scale, eps, True)
        ctx.eps = eps
        ctx.save_for_backward(h, y, post, pre, gate, scale, stats)
        return h_out, x_out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dx):
        h, y, post, pre, gate, scale, stats = ctx.saved_tensors
        if dh is None and dx is None:
            return (None,) * 7
        shape, D, dev = h.shape, h.shape[-1], h.device
        two = lambda t: None if t is None else _two(t, D)  # noqa: E731
        empty = lambda: torch.empty(shape, dtype=h.dtype, device=dev)  # noqa: E731
        need = ctx.needs_input_grad
        dh_out, dy_out, dgate_out = empty(), empty(), None if gate is None else empty()
        params = need[2] or need[3] or need[5]
        dparam = None
        if params:
            dparam = torch.empty((3, D), dtype=torch.float32, device=dev) if h.numel() else torch.zeros((3, D), dtype=torch.float32, device=dev)
        h2, y2, g2, dh, dx = two(h), two(y), two(gate), two(dh), two(dx)
        arg = lambda work: _norm_arg(h2, y2, g2, post, pre, scale, ctx.eps, None, None, stats, dh, dx, dh_out, dy_out, dgate_out, dparam, work)  # noqa: E731
        L = _native.sequence_lib()
        floats = L.pvder_seq_norm_workspace(arg(None)) if params else 0
        if floats < 0:
            _native.check(int(floats), "pvder_seq_norm_workspace")
        on, stream = _on(dev)
        with on:
            work = torch.empty(floats, dtype=torch.float32, device=dev) if floats else None
            rc = L.pvder_seq_norm_backward(arg(work), stream)
        _native.check(rc, "pvder_seq_norm_backward")
        return (dh_out if need[0] else None, dy_out if need[1] else None, dparam[0] if need[2] else None, dparam[1] if need[3] else None,
                dgate_out if need[4] else None, dparam[2] if need[5] else None, None)


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
    _tensors(None, residual=residual, y=y, post_weight=post_weight, pre_weight=pre_weight, **_given(gate=gate, scale=scale))
    if residual.dtype not in _DTYPES or any(t is not None and t.dtype != residual.dtype for t in (y, gate)):
        raise TypeError("residual, y and gate must be float32 or bfloat16, all alike")
    _need(residual.dim() >= 1 and 1 <= residual.shape[-1] <= MAX_WIDTH, "the last dimension must be 1 .. %d wide" % MAX_WIDTH)
    D = residual.shape[-1]
    for n, t in (("y", y), ("gate", gate)):
        _need(t is None or t.shape == residual.shape, "%s must have the shape of residual, %s" % (n, tuple(residual.shape)))
    for n, t in (("post_weight", post_weight), ("pre_weight", pre_weight), ("scale", scale)):
        if t is not None:
            if t.dtype != torch.float32:
                raise TypeError("%s must be float32" % n)
            _need(t.shape == (D,) and t.is_contiguous(), "%s must be a contiguous [%d]" % (n, D))
    if isinstance(eps, torch.Tensor) or not (math.isfinite(eps) and eps >= 0.0):
        raise ValueError("eps must be a finite number >= 0")
    _gpu("residual", residual)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (residual, y, post_weight, pre_weight, gate, scale)):
        return _GatedResidualNorm.apply(residual, y, post_weight, pre_weight, gate, scale, float(eps))
    return _norm_forward(residual, y, post_weight, pre_weight, gate, scale, float(eps), False)[:2]
