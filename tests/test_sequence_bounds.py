"""What the tight bounds of tests/test_gpu_sequence_precision.py tell apart, by arithmetic on the CPU."""
import pytest
import torch

import test_gpu_sequence_precision as precision


def _summands(x, parts):
    """x as a sum of bf16 numbers, each the rounding of what the ones before left."""
    got, left = torch.zeros_like(x), x
    for _ in range(parts):
        part = left.to(torch.bfloat16).float()
        got, left = got + part, left - part
    return got


@pytest.mark.parametrize("seed", range(3))
@pytest.mark.parametrize("which", ["state", "ds0"])
def test_the_bound_of_states_tells_two_summands_from_three(which, seed):
    """States from weighted values of two bf16 summands (2^-16 of a term) fall outside, those of three (2^-24) inside."""
    c = precision.case(1, 7, 2, 16, 24, torch.bfloat16, "cpu", seed)
    val, mag = precision.reference(c)
    g = torch.exp(c["log_decay"]).view(1, 2, 1)
    tol = precision.bounds(c, mag)[which]
    left, scale = c["left"], 16 ** -0.5
    for parts, inside in ((3, True), (2, False), (1, False)):
        S = torch.zeros_like(val[which], dtype=torch.float32)
        for t in (range(7 - left, 7) if which == "state" else range(left)):
            x, y = (c["k"], c["v"]) if which == "state" else (c["q"], c["do"])
            w = g ** (6 - t) if which == "state" else scale * g ** (t + 1)
            S = S + x[:, t].float()[..., None] * _summands(w * y[:, t].float(), parts)[:, :, None]
        assert bool(((S.double() - val[which]).abs() <= tol).all()) == inside, parts
        assert (float((S.double() - val[which]).norm()) <= 2.0 ** -20 * float(mag[which].norm())) == inside, parts     # and by the norm of the whole


def test_a_result_that_is_not_there_fails():
    r = {"out": torch.ones(2).double()}
    precision.check({"out": torch.ones(2)}, r, {"out": torch.zeros(2)})
    for got in ({}, {"out": None}, {"out": torch.ones(2), "dq": torch.ones(2)}):
        with pytest.raises(AssertionError):
            precision.check(got, r, {"out": torch.zeros(2)})
