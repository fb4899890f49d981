"""States, and float32 results, to the last few roundings: windows in which few tokens count, so that few roundings are made.

An episode starts `left` tokens before the end and one `left` tokens behind the beginning, so that the state behind the window and the
gradient of the state before it are sums of `left` terms, whatever the window's length and the pieces that it is cut into.  u = 2^-24.
"""
import pytest
import torch

import sequence_reference as ref

U = 2.0 ** -24


def case(B, T, H, DK, DV, dtype, dev, seed=0, left=3):
    g = torch.Generator(device="cpu")
    g.manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    c = {n_: n(B, T, H, d).to(dtype).to(dev) for n_, d in (("q", DK), ("k", DK), ("v", DV), ("do", DV))}
    c["log_decay"] = torch.linspace(-0.03, -0.1, H).to(dev)
    c["starts"] = torch.zeros(B, T, dtype=torch.bool, device=dev)
    c["starts"][:, T - left] = c["starts"][:, left] = True
    c["left"] = left
    return c


def reference(c):
    """The values in 64 bits, and the sums of their terms' magnitudes."""
    def one(f):
        zero = torch.zeros(c["q"].shape[0], c["q"].shape[2], c["q"].shape[3], c["v"].shape[3])
        return ref.attention(f(c["q"]), f(c["k"]), f(c["v"]), c["log_decay"], c["q"].shape[3] ** -0.5, zero, c["starts"], None, f(c["do"]), zero)
    return one(lambda x: x), one(torch.abs)


def bounds(c, mag):
    """Roundings of a term, for log_decay >= -0.1 and weights g^n with n <= 7 (the tokens that count are few).

    A weight: log_decay times log2(e) (2 u: constant and product), times n (1 u), changes the exponent by 3 u x 0.7 in natural units, 2.1 u;
    the exponential itself 2 u (one unit in the last place); times the scale, itself rounded, 2 u: at most 7 u; for the states' n <= 3
    at most 5 u, and once more 3 u where a chunk's border lies between.
    A state: these, the product with the value (1 u), bf16: what three summands leave of it (1 u; each takes 8 bits), the product at a
    chunk's border (1 u), and the sum of `left` terms of three summands (2 u each, where the matrix cores cut off instead of rounding):
    12 + 6 left.
    float32 outputs: a product over DK or DV (2 u a term) in the scores or with the state, two weights, the products with them, the sum over
    the tokens of an episode, at most `most`: 2 (DK + DV) + 20 + 2 most."""
    T, left = c["q"].shape[1], c["left"]
    most = max(left, T - 2 * left)
    state = (12 + 6 * left) * U
    other = (2 * (c["q"].shape[3] + c["v"].shape[3]) + 20 + 2 * most) * U
    return {n: (state if n in ("state", "ds0") else other) * m for n, m in mag.items()}


def check(got, want, tol):
    """Each of `want` is there, nothing else is, and every element is within its bound."""
    assert set(got) == set(want), (sorted(got), sorted(want))
    for n, r in want.items():
        assert got[n] is not None, n
        x = got[n].detach().double().cpu()
        assert x.shape == r.shape, (n, x.shape, r.shape)
        off = (x - r).abs()
        assert bool((off <= tol[n]).all()), "%s: off by %.3g of its bound" % (n, float((off / tol[n].clamp(min=1e-300)).max()))


@pytest.fixture(scope="module")
def ops(gpu_device):
    from gym_PVDER_amd.agents import sequence_ops
    return sequence_ops


def _run(ops, c):
    leaf = {n: c[n].detach().requires_grad_() for n in ("q", "k", "v")}
    leaf["s0"] = torch.zeros(c["q"].shape[0], c["q"].shape[2], c["q"].shape[3], c["v"].shape[3], device=c["q"].device, requires_grad=True)
    out, end = ops.decay_attention(leaf["q"], leaf["k"], leaf["v"], c["log_decay"], initial_state=leaf["s0"], starts=c["starts"], output_final_state=True)
    dq, dk, dv, ds0 = torch.autograd.grad([out, end], list(leaf.values()), [c["do"], torch.zeros_like(end)])
    return {"out": out, "state": end, "dq": dq, "dk": dk, "dv": dv, "ds0": ds0}


# whole and ragged heads of every padded size, short windows and ones cut into pieces, ends inside a chunk and at its border
SHAPES = [(1, 6, 2, 16, 24), (2, 6, 3, 8, 8), (2, 40, 2, 64, 64), (1, 64, 2, 33, 20), (3, 99, 2, 128, 128), (1, 600, 2, 64, 64), (1, 515, 1, 128, 40),
          (1, 450, 3, 20, 100)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_states_are_sums_of_fp32_products(ops, gpu_device, shape, dtype):
    """Both states, the one behind the window and the gradient of the one before it, in both types.

    The norm of the whole: the error of a weight is common to many terms, at most 10 u; the other 20 roundings have both signs and come to
    the root of 20 times u / sqrt(3), 3 u: below 16 u = 2^-20."""
    c = case(*shape, dtype, gpu_device)
    val, mag = reference(c)
    got, tol = _run(ops, c), bounds(c, mag)
    assert all(x is not None for x in got.values())
    for n in ("state", "ds0"):
        check({n: got[n]}, {n: val[n]}, tol)
        assert float((got[n].detach().double().cpu() - val[n]).norm()) <= 2.0 ** -20 * float(mag[n].norm()), n


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 6, 1, 4, 4), (2, 6, 3, 8, 8), (2, 7, 2, 16, 24), (2, 6, 1, 33, 20), (1, 6, 2, 64, 64), (1, 6, 1, 128, 128)])
def test_float32_results_to_the_last_roundings(ops, gpu_device, shape):
    c = case(*shape, torch.float32, gpu_device)
    val, mag = reference(c)
    check(_run(ops, c), val, bounds(c, mag))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gate,scale", [(True, True), (False, False), (True, False), (False, True)])
@pytest.mark.parametrize("R,D", [(1, 4), (7, 16), (33, 100), (300, 17), (5, 2500), (3, 8192)])
def test_every_gradient_of_the_norm_is_there(ops, gpu_device, R, D, gate, scale, dtype):
    """Each tensor that was given has its gradient: none is missing, none is None."""
    g = torch.Generator(device="cpu")
    g.manual_seed(R + D)
    n = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    c = {"h": n(R, D).to(dtype), "y": n(R, D).to(dtype), "gate": n(R, D).to(dtype) if gate else None, "post": 1 + 0.2 * n(D), "pre": 1 + 0.2 * n(D),
         "scale": 0.5 + 0.2 * n(D) if scale else None}
    dh, dx = n(R, D).to(dtype), n(R, D).to(dtype)
    leaf = {m: None if x is None else x.to(gpu_device).requires_grad_() for m, x in c.items()}
    h, x = ops.gated_residual_norm(leaf["h"], leaf["y"], leaf["post"], leaf["pre"], gate=leaf["gate"], scale=leaf["scale"])
    names = [m for m in leaf if leaf[m] is not None]
    grads = torch.autograd.grad([h, x], [leaf[m] for m in names], [dh.to(gpu_device), dx.to(gpu_device)])
    val, mag = ref.norm(c["h"], c["y"], c["post"], c["pre"], c["gate"], c["scale"], 1e-6, dh, dx)
    absent = {"d" + m for m in c if c[m] is None}
    want = {m: r for m, r in val.items() if m not in absent}
    check({"h": h, "x": x, **{"d" + m: t for m, t in zip(names, grads)}}, want, ref.norm_bounds(dtype, R, D, val, mag))
