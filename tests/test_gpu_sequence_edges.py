"""Values that are not finite at the borders of episodes, weights of zero, and grids past their limits, on the GPU."""
import pytest
import torch

import sequence_reference as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
BAD = [float("nan"), float("inf"), -float("inf")]


@pytest.fixture(scope="module")
def ops(gpu_device):
    from gym_PVDER_amd.agents import sequence_ops
    return sequence_ops


def _inputs(B, T, H, DK, DV, dtype, dev, seed=0):
    g = torch.Generator(device="cpu")
    g.manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    return {"q": n(B, T, H, DK).to(dtype).to(dev), "k": n(B, T, H, DK).to(dtype).to(dev), "v": n(B, T, H, DV).to(dtype).to(dev),
            "log_decay": torch.linspace(-0.02, -0.3, H).to(dev), "do": n(B, T, H, DV).to(dtype).to(dev),
            "s0": n(B, H, DK, DV).to(dev), "ds": n(B, H, DK, DV).to(dev), "starts": torch.zeros(B, T, dtype=torch.bool, device=dev)}


def _gradients(ops, c, **kw):
    leaf = {n: c[n].detach().requires_grad_() for n in ("q", "k", "v", "s0")}
    out, end = ops.decay_attention(leaf["q"], leaf["k"], leaf["v"], c["log_decay"], initial_state=leaf["s0"], starts=c["starts"], output_final_state=True, **kw)
    got = torch.autograd.grad([out, end], list(leaf.values()), [c["do"], c["ds"]])
    return {"out": out.detach(), "state": end.detach(), **dict(zip(("dq", "dk", "dv", "ds0"), got))}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,at,DK,DV", [(3, 1, 8, 8), (70, 0, 32, 40), (70, 31, 32, 40), (70, 32, 64, 64), (70, 69, 128, 33), (600, 320, 64, 64), (600, 333, 20, 128)])
def test_the_first_token_of_an_episode_reaches_no_earlier_one(ops, gpu_device, T, at, DK, DV, dtype):
    """A gradient goes back to the start of its episode and not behind it, whatever the start's own token holds."""
    c = _inputs(2, T, 2, DK, DV, dtype, gpu_device)
    c["starts"][:, at] = True
    clean = ref.attention(c["q"], c["k"], c["v"], c["log_decay"], DK ** -0.5, c["s0"], c["starts"], None, c["do"], c["ds"])
    mag = ref.attention(c["q"].abs(), c["k"].abs(), c["v"].abs(), c["log_decay"], DK ** -0.5, c["s0"].abs(), c["starts"], None, c["do"].abs(), c["ds"].abs())
    tol = ref.attention_bounds(dtype, T, DK, DV, clean, mag)
    for n in ("q", "k", "v", "do"):
        for bad in BAD:
            d = dict(c, **{n: c[n].clone()})
            d[n][0, at, 0, 3] = bad
            got = _gradients(ops, d)
            earlier = {m: (got[m][:, :at], clean[m][:, :at], tol[m][:, :at]) for m in ("out", "dq", "dk", "dv")}
            earlier["ds0"] = got["ds0"], clean["ds0"], tol["ds0"]
            for m, (x, r, t) in earlier.items():
                over = (x.double().cpu() - r).abs() > t
                assert x.shape == r.shape and not bool(over.any() | torch.isnan(x).any()), (n, bad, m)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 40, 600])
def test_a_head_that_remembers_nothing_passes_nothing_on(ops, gpu_device, T, dtype):
    """A decay of -inf is a weight of zero between any two tokens: values that are not finite stay in their own token, in both directions."""
    c = _inputs(1, T, 2, 32, 24, dtype, gpu_device)
    c["log_decay"] = torch.tensor([-float("inf"), -1000.0], device=gpu_device)
    at = T // 2
    clean = _gradients(ops, c)
    others = torch.arange(T, device=gpu_device) != at
    for n in ("q", "k", "v", "do"):
        for bad in BAD:
            d = dict(c, **{n: c[n].clone()})
            d[n][0, at, :, 3] = bad
            got = _gradients(ops, d)
            for m in ("out", "dq", "dk", "dv"):
                assert torch.isfinite(got[m][:, others].float()).all(), (n, bad, m)
            assert torch.equal(got["ds0"], torch.zeros_like(got["ds0"])) and torch.equal(clean["ds0"], got["ds0"])
            if at < T - 1:
                assert torch.isfinite(got["state"]).all(), (n, bad)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("DK,DV", [(8, 8), (5, 3), (100, 66)])
def test_steps_clear_with_a_weight_of_zero_as_windows_do(ops, gpu_device, DK, DV, dtype):
    """A head that remembers nothing takes no state, finite or not: steps behind a window are the window."""
    c = _inputs(2, 6, 3, DK, DV, dtype, gpu_device)
    c["log_decay"] = torch.tensor([-float("inf"), -0.1, -1000.0], device=gpu_device)
    for bad in BAD:
        k = c["k"].clone()
        k[0, 1, (0, 2), 2] = bad                                      # (the head with a memory stays finite)
        out, end = ops.decay_attention(c["q"], k, c["v"], c["log_decay"], output_final_state=True)
        state = torch.zeros_like(end)
        state[:, (0, 2)] = bad
        steps = torch.stack([ops.decay_attention_step(c["q"][:, t], k[:, t], c["v"][:, t], c["log_decay"], state) for t in range(6)], 1)
        others = torch.arange(6, device=gpu_device) != 1
        assert torch.isfinite(state).all() and torch.isfinite(steps[:, others].float()).all() and torch.isfinite(out[:, others].float()).all(), bad
        # heads without a memory: one product a token, the same in both forms but for the order of a sum over DK and the rounding
        # of its terms to the inputs' type
        size = (c["q"].float().abs() * k.float().abs()).sum(-1, keepdim=True) * c["v"].float().abs() * DK ** -0.5
        tol = ((2 * DK + 8) * ref.U32 + (4 * ref.U16 if dtype == torch.bfloat16 else 0.0)) * size
        assert ((steps.float() - out.float()).abs() <= tol)[:, others][:, :, (0, 2)].all(), bad


def _far_rows(n, dev):
    """The first rows, the last ones, and those around the borders of any two or three equal parts."""
    at = [0, n - 1] + [n * i // p + d for p in (2, 3, 4) for i in range(1, p) for d in range(-40, 40)]
    return torch.tensor(sorted({min(max(i, 0), n - 1) for i in at}), device=dev)


def test_more_cells_than_the_threads_of_a_launch(ops, gpu_device):
    """Steps of over 2^26 cells, whose launch would have over 2^32 threads."""
    N = 2 ** 26 + 9
    g = torch.Generator(device=gpu_device)
    g.manual_seed(1)
    q, k, v = (torch.randn(N, 1, 1, generator=g, device=gpu_device) for _ in range(3))
    state = torch.randn(N, 1, 1, 1, generator=g, device=gpu_device)
    starts = torch.rand(N, generator=g, device=gpu_device) < 0.25
    decay = torch.full((1,), -0.25, device=gpu_device)
    want = (state * torch.exp(decay)).masked_fill(starts[:, None, None, None], 0.0) + k[..., None] * v[..., None]
    size = state.abs() + (k * v).abs()[..., None]
    out = ops.decay_attention_step(q, k, v, decay, state, starts=starts)
    # the weight's exponent and exponential, three products and a sum, on either side
    assert bool(((state - want).abs() <= 12 * ref.U32 * size).all())
    assert bool(((out - q * want[..., 0]).abs() <= 14 * ref.U32 * q.abs() * size[..., 0]).all())


def test_more_rows_than_the_threads_of_a_launch(ops, gpu_device):
    """Windows of over 2^26 rows, whose launch would have over 2^32 threads: every tensor of the rows behind the first part."""
    B, D = 2 ** 26 + 40, 4
    g = torch.Generator(device=gpu_device)
    g.manual_seed(2)
    q, k, v = (torch.randn(B, 1, 1, D, generator=g, device=gpu_device) for _ in range(3))
    s0 = torch.randn(B, 1, D, D, generator=g, device=gpu_device)
    starts = torch.rand(B, 1, generator=g, device=gpu_device) < 0.25
    lengths = (torch.rand(B, generator=g, device=gpu_device) < 0.75).to(torch.int32)
    decay = torch.full((1,), -0.25, device=gpu_device)
    out, end = ops.decay_attention(q, k, v, decay, initial_state=s0, starts=starts, lengths=lengths, output_final_state=True)
    assert torch.isfinite(out).all() and torch.isfinite(end).all()
    assert not out[lengths == 0].any() and torch.equal(end[lengths == 0], s0[lengths == 0])
    at = _far_rows(B, gpu_device)
    few, few_end = ops.decay_attention(q[at], k[at], v[at], decay, initial_state=s0[at], starts=starts[at], lengths=lengths[at], output_final_state=True)
    assert torch.equal(out[at], few) and torch.equal(end[at], few_end)


def _inputs_of_a_capture(ops, which, dev):
    """(the leaf, its operator's outputs as a function of it): a packed leaf's views, heads that are padded, a state."""
    g = torch.Generator(device="cpu")
    g.manual_seed(3)
    n = lambda *s: torch.randn(s, generator=g).to(dev)  # noqa: E731
    decay = torch.full((2,), -0.1, device=dev)
    if which == "views of a packed leaf":
        leaf = n(1, 9, 48).requires_grad_()
        return leaf, lambda: ops.decay_attention(*(leaf[..., i:i + 16].unflatten(-1, (2, 8)) for i in (0, 16, 32)), decay)
    if which == "small heads":
        leaf, k, v = n(1, 9, 2, 3).requires_grad_(), n(1, 9, 2, 3), n(1, 9, 2, 5)
        return leaf, lambda: ops.decay_attention(leaf, k, v, decay)
    if which == "small heads, the state":
        leaf, q, v = n(1, 2, 8, 3).requires_grad_(), n(1, 9, 2, 8), n(1, 9, 2, 3)
        return leaf, lambda: ops.decay_attention(q, q, v, decay, initial_state=leaf)
    leaf, y, w = n(4, 3, 8).requires_grad_(), n(12, 8), torch.ones(8, device=dev)
    return leaf, lambda: ops.gated_residual_norm(y, leaf.view(12, 8), w, w)[1]


@pytest.mark.parametrize("which", ["views of a packed leaf", "small heads", "small heads, the state", "a view in the norm"])
def test_a_capture_beside_a_living_graph_is_refused_behind_views_and_padding(ops, gpu_device, which):
    """Only forward passes are captured beside the living graph; behind its end forward and backward are, and replay right."""
    leaf, f = _inputs_of_a_capture(ops, which, gpu_device)
    out = f()
    do = torch.randn(out.shape, generator=torch.Generator().manual_seed(4)).to(gpu_device)
    torch.cuda.synchronize()
    g, t = torch.cuda.CUDAGraph(), torch.ones(4, device=gpu_device)
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="another stream"):
            f()
        with torch.no_grad():
            quiet = f()                                               # (asks for no gradient)
        t.mul_(2)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(quiet, out.detach())
    want = torch.autograd.grad(out, leaf, do)[0].clone()
    del out
    g2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g2):
        got = torch.autograd.grad(f(), leaf, do)[0]
    for _ in range(3):
        g2.replay()
        t.add_(1)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_tangents_are_refused_and_checkpoints_are_not(ops, gpu_device):
    import torch.autograd.forward_ad as fwad
    from torch.utils.checkpoint import checkpoint
    from torch.utils.flop_counter import FlopCounterMode
    c = _inputs(2, 600, 2, 16, 16, torch.float32, gpu_device)
    f = lambda q: ops.decay_attention(q, c["k"], c["v"], c["log_decay"], starts=c["starts"])  # noqa: E731
    with fwad.dual_level(), pytest.raises(ValueError, match="tangent"):
        f(fwad.make_dual(c["q"], torch.ones_like(c["q"])))
    q = c["q"].detach().requires_grad_()
    want, = torch.autograd.grad(f(q), q, c["do"])
    with FlopCounterMode(display=False):
        again, = torch.autograd.grad(f(q), q, c["do"])
    assert torch.equal(again, want)
    for reentrant in (False, True):
        q.grad = None
        checkpoint(f, q, use_reentrant=reentrant).backward(c["do"])
        assert torch.equal(q.grad, want), reentrant
    with torch.autograd.graph.save_on_cpu():
        out = f(q)
    assert torch.equal(torch.autograd.grad(out, q, c["do"])[0], want)
