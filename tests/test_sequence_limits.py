"""Limits of the sequence operators' C entries and of what their Python side takes, without a GPU."""
import ctypes
import struct

import pytest
import torch

from test_sequence_ops import ATTN_TAIL, SCAN, STEP


def _attn(B=1, T=1, H=1, dk=8, dv=8, segments=1, work=0, states=(0, 0), state_strides=(0, 0, 0, 0)):
    row = max(dk, dv)
    one = SCAN.pack(*([64] * 4), *([0, row, 0] * 4), *states, *state_strides, 0, 1.0, 1.0, 1.0, dk, dv, 0, 0)
    return ctypes.create_string_buffer(one * 3 + ATTN_TAIL.pack(64, 0, 0, work, 0, 0, B, T, H, 1, 0, segments))


def test_launches_whose_threads_cannot_be_counted_are_refused():
    """A launch has fewer than 2^32 threads.  Batch rows are taken in parts, the heads of one row and the pieces of T are not."""
    from gym_PVDER_amd import _native
    _native.build_native()
    L = _native.sequence_lib()
    for bad in (dict(H=2 ** 26), dict(H=2 ** 25, dv=128), dict(B=3, H=2 ** 27), dict(H=2 ** 31 - 1), dict(B=2 ** 31 - 1, H=2 ** 31 - 1),
                dict(B=2 ** 20, H=64, T=512, segments=2, work=64), dict(B=1, H=2 ** 21, T=512, dk=128, dv=128, segments=2, work=64)):
        assert L.pvder_seq_attn_run(_attn(**bad), None) == _native.EINVAL, bad
    step = lambda N, H, d: STEP.pack(*([64] * 4), *([0] * 8), 64, 64, 0, 0, N, H, d, d, 0, 1.0)  # noqa: E731
    for N, H, d in ((1, 2 ** 26, 4), (5, 2 ** 24, 128), (2 ** 31 - 1, 2 ** 31 - 1, 1)):
        assert L.pvder_seq_step_run(step(N, H, d), None) == _native.EINVAL, (N, H, d)


def test_more_pieces_than_a_plan_makes_are_refused():
    """A piece is 64 tokens or more; the kernels count tokens in 32 bits."""
    from gym_PVDER_amd import _native
    L = _native.sequence_lib()
    for T, segments in ((2 ** 30, 2 ** 25), (512, 9), (63, 2), (0, 2)):
        assert L.pvder_seq_attn_run(_attn(T=T, segments=segments, work=64), None) == _native.EINVAL, (T, segments)


def test_states_whose_offsets_pass_32_bits_are_refused():
    """Also those of windows without a token, whose state goes through all the same."""
    from gym_PVDER_amd import _native
    L = _native.sequence_lib()
    for T in (0, 1):
        for states in ((64, 0), (0, 64)):
            for strides in ((0, 0, 2 ** 29, 1), (0, 0, 1, 2 ** 29), (0, 0, 2 ** 26, 1), (0, 0, -1, 1), (0, 0, 1, -8)):
                assert L.pvder_seq_attn_run(_attn(T=T, states=states, state_strides=strides), None) == _native.EINVAL, (T, states, strides)


def _calls():
    from gym_PVDER_amd.agents import sequence_ops as so
    q, g, w, state = torch.zeros(2, 5, 2, 8), torch.zeros(2), torch.ones(8), torch.zeros(5, 2, 8, 8)
    t, h = q[0], q[0, 0]
    return {"windows": (lambda x: so.decay_attention(x, q, q, g), q),
            "the state of windows": (lambda x: so.decay_attention(q, q, q, g, initial_state=x), torch.zeros(2, 2, 8, 8)),
            "steps": (lambda x: so.decay_attention_step(t, t, x, g, state), t),
            "the state of steps": (lambda x: so.decay_attention_step(t, t, t, g, x), state),
            "norm": (lambda x: so.gated_residual_norm(h, x, w, w)[0], h),
            "a weight of the norm": (lambda x: so.gated_residual_norm(h, h, w, w, scale=x)[0], w)}


@pytest.mark.parametrize("name", sorted(_calls()))
def test_what_the_kernels_would_silently_leave_out_is_refused(name):
    """A tangent would be dropped, a trace would record memory that nothing writes."""
    import torch.autograd.forward_ad as fwad
    from torch.fx.experimental.proxy_tensor import make_fx
    f, x = _calls()[name]
    with pytest.raises(ValueError, match="GPU"):
        f(x)
    with fwad.dual_level(), pytest.raises(ValueError, match="tangent"):
        f(fwad.make_dual(x, torch.ones_like(x)))
    with pytest.raises(ValueError, match="traced"):
        torch.jit.trace(f, (x,))
    for mode in ("real", "fake", "symbolic"):
        with pytest.raises(ValueError, match="traced"):
            make_fx(f, tracing_mode=mode)(x)
    for transform in (lambda: torch.func.jvp(f, (x,), (x,)), lambda: torch.func.vmap(f)(x[None]), lambda: torch.func.functionalize(f)(x),
                      lambda: torch.func.grad(lambda t: f(t).sum())(x)):
        with pytest.raises(ValueError, match="traced|wrappers"):
            transform()


class _Logged(torch.Tensor):
    """A tensor subclass that sees the operations on it."""
    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def test_tensors_that_stand_for_others_are_refused_and_parameters_are_not():
    f, x = _calls()["windows"]
    with pytest.raises(ValueError, match="wrappers"):
        f(torch.Tensor._make_subclass(_Logged, x))
    with pytest.raises(ValueError, match="GPU"):
        f(torch.nn.Parameter(x))
    from torch.utils.flop_counter import FlopCounterMode
    with FlopCounterMode(display=False), pytest.raises(ValueError, match="GPU"):     # (counts, and changes nothing)
        f(x)


def test_horizons_are_finite():
    """An infinite one made decays that are not numbers, which the kernels take as none."""
    from gym_PVDER_amd.agents import SequenceQNetwork
    for bad in ((4.0, float("inf")), (float("nan"), 5.0), (4.0, float("nan")), (1.0, 5.0), (4.0,)):
        with pytest.raises(ValueError, match="horizons"):
            SequenceQNetwork(horizons=bad, device="cpu")
    decay = SequenceQNetwork(horizons=(4.0, 1e9), device="cpu").log_decay
    assert torch.isfinite(decay).all() and (decay < 0).all() and bool((decay[1:] > decay[:-1]).all())
