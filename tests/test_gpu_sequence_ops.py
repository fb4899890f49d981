"""The sequence operators on the GPU against their formulas in 64 bits (tests/sequence_reference.py, which derives the bounds)."""
import pytest
import torch

import sequence_reference as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def ops(gpu_device):
    from gym_PVDER_amd.agents import sequence_ops
    return sequence_ops


def _gen(seed):
    g = torch.Generator(device="cpu")
    g.manual_seed(seed)
    return g


def _case(B, T, H, DK, DV, dtype, dev, episodes=False, state=False, seed=0):
    g = _gen(seed + 1000 * T + DK)
    n = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    packed = n(B, T, H * (2 * DK + DV)).to(dtype).to(dev)
    c = {"q": packed[..., :H * DK].unflatten(-1, (H, DK)), "k": packed[..., H * DK:2 * H * DK].unflatten(-1, (H, DK)),
         "v": packed[..., 2 * H * DK:].unflatten(-1, (H, DV)), "log_decay": torch.log1p(-torch.rand(H, generator=g) * 0.5).to(dev),
         "s0": n(B, H, DK, DV).to(dev) if state else None, "starts": None, "lengths": None,
         "do": n(B, T, H, DV).to(dtype).to(dev), "ds": n(B, H, DK, DV).to(dev) if state else None}
    if H > 1:
        c["log_decay"][0] = -1e-3
    if episodes:
        c["starts"] = (torch.rand(B, T, generator=g) < 0.06).to(dev)
        c["lengths"] = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32).to(dev)
        c["lengths"][-1] = T
    return c


def _both(c, scale):
    a = [c["q"], c["k"], c["v"], c["log_decay"], scale, c["s0"], c["starts"], c["lengths"], c["do"], c["ds"]]
    absolute = [None if x is None else (x.abs() if torch.is_tensor(x) and x.dtype.is_floating_point and i not in (3,) else x) for i, x in enumerate(a)]
    return ref.attention(*a), ref.attention(*absolute)


def _run(ops, c, scale=None, train=True):
    leaf = {n: None if c[n] is None else c[n].detach().requires_grad_(train) for n in ("q", "k", "v", "s0")}
    r = ops.decay_attention(leaf["q"], leaf["k"], leaf["v"], c["log_decay"], scale=scale, initial_state=leaf["s0"], starts=c["starts"],
                            lengths=c["lengths"], output_final_state=c["s0"] is not None)
    out, fin = r if c["s0"] is not None else (r, None)
    got = {"out": out, "state": fin}
    if train:
        names = [n for n in leaf if leaf[n] is not None]
        outs, gs = ([out, fin], [c["do"], c["ds"]]) if fin is not None else ([out], [c["do"]])
        for n, x in zip(names, torch.autograd.grad(outs, [leaf[n] for n in names], gs)):
            got["ds0" if n == "s0" else "d" + n] = x
    return got


# one token, one partial chunk, whole chunks, one token over, head sizes that fill no tile, every padded size, several pieces of T
SHAPES = [(1, 1, 1, 1, 1), (2, 1, 3, 16, 32), (2, 5, 3, 16, 16), (1, 16, 1, 32, 32), (1, 32, 2, 32, 64), (3, 33, 2, 24, 40), (1, 65, 1, 64, 64),
          (2, 160, 4, 64, 64), (2, 70, 1, 65, 128), (1, 131, 2, 128, 33), (1, 255, 1, 128, 128), (1, 256, 1, 7, 3), (2, 300, 1, 100, 20),
          (1, 1000, 2, 20, 64), (1, 700, 1, 128, 127), (1, 600, 1, 7, 3), (1, 450, 3, 64, 64), (3, 400, 2, 36, 65)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("episodes,state", [(False, False), (True, True), (True, False), (False, True)])
@pytest.mark.parametrize("shape", SHAPES)
def test_windows_and_gradients(ops, gpu_device, shape, episodes, state, dtype):
    B, T, H, DK, DV = shape
    c = _case(*shape, dtype, gpu_device, episodes, state)
    r, mag = _both(c, DK ** -0.5)
    tol = ref.attention_bounds(dtype, T, DK, DV, r, mag)
    ref.check(_run(ops, c), r, tol, str(shape))
    ref.check(_run(ops, c, train=False), {"out": r["out"], "state": r["state"]}, tol, "no grad")
    if dtype == torch.bfloat16 and r["out"].numel() > 4000:
        # many independent roundings of both signs: the whole is off by less than one rounding at its worst
        got = _run(ops, c)
        for n in ("out", "dq", "dk", "dv"):
            assert float((got[n].detach().double().cpu() - r[n]).norm() / r[n].norm()) < ref.U16, n


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_rows(ops, gpu_device, dtype):
    """More rows than the card takes at once, each of them checked."""
    c = _case(700, 20, 3, 32, 32, dtype, gpu_device, True, True)
    r, mag = _both(c, 32 ** -0.5)
    ref.check(_run(ops, c), r, ref.attention_bounds(dtype, 20, 32, 32, r, mag))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1000, 2, 20, 64), (2, 520, 3, 64, 33), (1, 450, 1, 128, 48), (6, 390, 48, 8, 8)])
def test_gradients_of_some_inputs_over_pieces(ops, gpu_device, shape, dtype):
    """Long windows of few rows: every choice of the inputs that want a gradient, and the same graph walked twice.  (The last shape is cut
    into pieces on the way forward only.)"""
    B, T, H, DK, DV = shape
    c = _case(*shape, dtype, gpu_device, True, True)
    r, mag = _both(c, DK ** -0.5)
    tol = ref.attention_bounds(dtype, T, DK, DV, r, mag)
    r0, mag0 = _both({**c, "ds": None}, DK ** -0.5)
    tol0 = ref.attention_bounds(dtype, T, DK, DV, r0, mag0)
    leaf = {n: c[n].detach().requires_grad_() for n in ("q", "k", "v", "s0")}
    outs = ops.decay_attention(leaf["q"], leaf["k"], leaf["v"], c["log_decay"], initial_state=leaf["s0"], starts=c["starts"], lengths=c["lengths"],
                               output_final_state=True)
    for choice in range(1, 16):
        names = [n for i, n in enumerate(leaf) if choice >> i & 1]
        first, again = (torch.autograd.grad(outs, [leaf[n] for n in names], [c["do"], c["ds"]], retain_graph=True) for _ in range(2))
        assert all(torch.equal(x, y) for x, y in zip(first, again)), names
        ref.check({"ds0" if n == "s0" else "d" + n: x for n, x in zip(names, first)}, r, tol, str(names))
        own = {n: leaf[n].detach().requires_grad_(n in names) for n in leaf}
        o = ops.decay_attention(own["q"], own["k"], own["v"], c["log_decay"], initial_state=own["s0"], starts=c["starts"], lengths=c["lengths"])
        alone = torch.autograd.grad(o, [own[n] for n in names], c["do"])
        ref.check({"ds0" if n == "s0" else "d" + n: x for n, x in zip(names, alone)}, r0, tol0, "alone %s" % names)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(ops, gpu_device, dtype):
    """Time-major tensors, one window seen by every row (stride 0), a head dimension that is not dense, states that are views."""
    B, T, H, DK, DV = 3, 40, 2, 16, 24
    c = _case(B, T, H, DK, DV, dtype, gpu_device, True, True)
    plain = _run(ops, c)
    tm = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    last = lambda x: x.transpose(1, 3).contiguous().transpose(1, 3)  # noqa: E731
    for lay in (tm, last):
        d = dict(c, q=lay(c["q"]), k=lay(c["k"]), v=lay(c["v"]), do=lay(c["do"]), starts=tm(c["starts"]), s0=c["s0"].transpose(2, 3).contiguous().transpose(2, 3),
                 ds=c["ds"].transpose(1, 2).contiguous().transpose(1, 2))
        got = _run(ops, d)
        for n in plain:
            assert torch.equal(got[n], plain[n]), n
    d = dict(c, k=c["k"][:1].expand(B, T, H, DK), v=c["v"][:1].expand(B, T, H, DV))
    e = dict(c, k=d["k"].contiguous(), v=d["v"].contiguous())
    a, b = _run(ops, d), _run(ops, e)
    for n in a:
        assert torch.equal(a[n], b[n]), n
    leaf = c["k"][:1, :, :1].detach().requires_grad_()                # shared over rows and heads: its gradient is the sum
    out = ops.decay_attention(c["q"], leaf.expand(B, T, H, DK), c["v"], c["log_decay"], starts=c["starts"], lengths=c["lengths"])
    got, = torch.autograd.grad([out], [leaf], [c["do"]])
    f = dict(c, k=leaf.detach().expand(B, T, H, DK), s0=None, ds=None)
    whole = _run(ops, f)["dk"].double().sum((0, 2), keepdim=True)
    assert float((got.double() - whole).norm() / whole.norm()) < 4 * torch.finfo(dtype).eps


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty(ops, gpu_device, dtype):
    z = lambda *s: torch.zeros(s, dtype=dtype, device=gpu_device)  # noqa: E731
    g = torch.full((2,), -0.1, device=gpu_device)
    for B, T in ((0, 4), (3, 0), (0, 0)):
        s0 = torch.randn(B, 2, 8, 4, device=gpu_device).requires_grad_()
        q = z(B, T, 2, 8).requires_grad_()
        out, fin = ops.decay_attention(q, z(B, T, 2, 8), z(B, T, 2, 4), g, initial_state=s0, output_final_state=True)
        assert out.shape == (B, T, 2, 4) and torch.equal(fin, s0)
        dq, ds = torch.autograd.grad([out, fin], [q, s0], [out, torch.ones_like(fin)])
        assert dq.shape == q.shape and torch.equal(ds, torch.ones_like(ds))
    # every row empty: zeros out, whatever stands behind the lengths, and the state as it was
    nan = torch.full((2, 50, 2, 8), float("nan"), dtype=dtype, device=gpu_device)
    s0 = torch.randn(2, 2, 8, 8, device=gpu_device).requires_grad_()
    q = nan.clone().requires_grad_()
    out, fin = ops.decay_attention(q, nan, nan, g, initial_state=s0, lengths=torch.tensor([0, -3], dtype=torch.int32, device=gpu_device),
                                   output_final_state=True)
    assert not out.any() and torch.equal(fin, s0)
    dq, ds = torch.autograd.grad([out, fin], [q, s0], [nan, torch.ones_like(fin)])
    assert not dq.any() and torch.equal(ds, torch.ones_like(ds))
    assert ops.decay_attention_step(z(0, 2, 8), z(0, 2, 8), z(0, 2, 8), g, torch.zeros(0, 2, 8, 8, device=gpu_device)).shape == (0, 2, 8)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [70, 600])
def test_values_that_are_not_finite_stay_where_they_belong(ops, gpu_device, dtype, T):
    """NaN and infinities behind the lengths and in finished episodes touch nothing; in a running one only what comes after it
    (in a gradient: before it)."""
    B, H, DK, DV = 2, 2, 32, 40
    c = _case(B, T, H, DK, DV, dtype, gpu_device, False, True)
    c["lengths"] = torch.tensor([T, T - 9], dtype=torch.int32, device=gpu_device)
    c["starts"] = torch.zeros(B, T, dtype=torch.bool, device=gpu_device)
    c["starts"][:, 50] = True
    for n in ("q", "k", "v"):
        c[n] = c[n].clone()
    clean = _run(ops, c)
    for n in ("q", "k", "v", "do"):
        d = dict(c, **{n: c[n].clone()})
        d[n][1, T - 9:] = float("nan")                                # behind the length
        got = _run(ops, d)
        for m in clean:
            assert torch.equal(got[m], clean[m]), (n, m)
    at = 41                                                           # the episode of tokens .. 49
    r, mag = _both(c, DK ** -0.5)
    tol = ref.attention_bounds(dtype, T, DK, DV, r, mag)["out"]
    for n, bad in (("k", float("nan")), ("v", float("inf")), ("v", float("nan")), ("k", -float("inf"))):
        d = dict(c, **{n: c[n].clone()})
        d[n][0, at, 0, 5] = bad
        got = _run(ops, d)
        out = got["out"].float()
        assert torch.equal(got["out"][1], clean["out"][1])                                   # the other row
        assert torch.equal(got["out"][0, :, 1], clean["out"][0, :, 1])                       # the other head
        assert not torch.isfinite(out[0, at:50, 0]).all(1).any()
        for part in (slice(0, at), slice(50, T)):                     # (token by token near it: other sums, within the same bound)
            assert bool(((out[0, part, 0].detach().double().cpu() - r["out"][0, part, 0]).abs() <= tol[0, part, 0]).all()), (n, bad, part)
        assert torch.isfinite(got["state"]).all()
        for m in ("dq", "dk", "dv"):
            assert torch.isfinite(got[m].float()[0, 50:]).all() and torch.isfinite(got[m].float()[1]).all() and torch.isfinite(got[m].float()[0, :, 1]).all()
        assert torch.isfinite(got["dq"].float()[0, :at]).all()
    d = dict(c, do=c["do"].clone())
    d["do"][0, at, 0, 3] = float("nan")
    got = _run(ops, d)
    assert torch.isfinite(got["dk"].float()[0, at + 1:]).all() and torch.isfinite(got["dv"].float()[0, at + 1:]).all()
    assert not torch.isfinite(got["dk"].float()[0, :at + 1, 0]).all(1).any()
    # a state that is not finite ends with the episode it came into
    d = dict(c, s0=c["s0"] * float("nan"))
    got = _run(ops, d)
    assert torch.isnan(got["out"][:, :50].float()).all() and torch.isfinite(got["out"][:, 50:].float()).all() and torch.isfinite(got["state"]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_decays_at_the_border(ops, gpu_device, dtype):
    """No decay at all, none given by NaN and growth, and heads that remember nothing."""
    B, T, DK, DV = 1, 90, 16, 16
    c = _case(B, T, 5, DK, DV, dtype, gpu_device, True, True)
    c["log_decay"] = torch.tensor([0.0, float("nan"), 3.0, -float("inf"), -200.0], device=gpu_device)
    got = _run(ops, c)
    c["log_decay"] = torch.tensor([0.0, 0.0, 0.0, -1e30, -200.0], device=gpu_device)
    r, mag = _both(c, DK ** -0.5)
    ref.check(got, r, ref.attention_bounds(dtype, T, DK, DV, r, mag))


def test_scale_and_differences(ops, gpu_device):
    """The window form is linear in each of its tensors: a difference quotient of any width is the derivative, up to rounding."""
    c = _case(2, 77, 2, 24, 20, torch.float32, gpu_device, True, True)
    got = _run(ops, c, scale=-0.7)

    def loss(**kw):
        d = dict(c, **kw)
        o, s = ops.decay_attention(d["q"], d["k"], d["v"], d["log_decay"], scale=-0.7, initial_state=d["s0"], starts=d["starts"],
                                   lengths=d["lengths"], output_final_state=True)
        return float((o.double() * c["do"].double()).sum() + (s.double() * c["ds"].double()).sum())

    g = _gen(5)
    for n, dn in (("q", "dq"), ("k", "dk"), ("v", "dv"), ("s0", "ds0")):
        x = c[n].detach()
        e = torch.randn(x.shape, generator=g).to(gpu_device)
        num = (loss(**{n: x + e}) - loss(**{n: x - e})) / 2
        ana = float((got[dn].double() * e.double()).sum())
        size = float((got[dn].double() * e.double()).abs().sum())
        assert abs(num - ana) < 2e-5 * size + 1e-6, n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (5, 2, 16, 16), (7, 3, 33, 20), (64, 4, 32, 32), (3, 2, 128, 128), (9, 1, 100, 7), (1, 4, 64, 64),
                                   (2, 2, 17, 68), (4, 1, 128, 65), (300, 3, 48, 80)])
def test_steps(ops, gpu_device, shape, dtype):
    N, H, DK, DV = shape
    c = _case(N, 6, H, DK, DV, dtype, gpu_device, False, True)
    c["starts"] = (torch.rand(N, 6, generator=_gen(3)) < 0.3).to(gpu_device)
    r, mag = _both(dict(c, lengths=None), DK ** -0.5)
    tol = ref.attention_bounds(dtype, 6, DK, DV, r, mag)
    state, outs = c["s0"].clone(), []
    for t in range(6):
        ver = state._version
        outs.append(ops.decay_attention_step(c["q"][:, t], c["k"][:, t], c["v"][:, t], c["log_decay"], state, starts=c["starts"][:, t]))
        assert state._version > ver
    ref.check({"out": torch.stack(outs, 1), "state": state}, {"out": r["out"], "state": r["state"]}, tol, str(shape))


def test_steps_leave_finished_rows_clean(ops, gpu_device):
    c = _case(4, 1, 2, 32, 32, torch.float32, gpu_device, False, True)
    state = c["s0"].clone()
    state[2] = float("nan")
    ops.decay_attention_step(c["q"][:, 0], c["k"][:, 0], c["v"][:, 0], c["log_decay"], state, starts=torch.tensor([0, 0, 1, 0], dtype=torch.uint8, device=gpu_device))
    assert torch.isfinite(state).all()
    assert torch.equal(state[2], (c["k"][2, 0, :, :, None] * c["v"][2, 0, :, None, :]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_window_then_window_then_steps(ops, gpu_device, dtype):
    """A stream cut anywhere gives what the whole gives: state out, state in, steps."""
    T, cuts = 170, (0, 61, 150)
    c = _case(2, T, 2, 32, 48, dtype, gpu_device, True, True)
    c["lengths"] = None
    r, mag = _both(c, 32 ** -0.5)
    tol = ref.attention_bounds(dtype, T, 32, 48, r, mag)
    state, outs = c["s0"], []
    for a, b in zip(cuts, cuts[1:]):
        o, state = ops.decay_attention(c["q"][:, a:b], c["k"][:, a:b], c["v"][:, a:b], c["log_decay"], initial_state=state, starts=c["starts"][:, a:b],
                                       output_final_state=True)
        outs.append(o)
    for t in range(cuts[-1], T):
        outs.append(ops.decay_attention_step(c["q"][:, t], c["k"][:, t], c["v"][:, t], c["log_decay"], state, starts=c["starts"][:, t])[:, None])
    ref.check({"out": torch.cat(outs, 1), "state": state}, {"out": r["out"], "state": r["state"]}, tol)


# ------------------------------------------------------------------------------------------------------------------- norm
def _norm_case(R, D, dtype, dev, gate=True, scale=True):
    g = _gen(R + 7 * D)
    n = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    return {"h": (2 * n(R, D)).to(dtype).to(dev), "y": n(R, D).to(dtype).to(dev), "gate": (3 * n(R, D)).to(dtype).to(dev) if gate else None,
            "post": (1 + 0.2 * n(D)).to(dev), "pre": (1 + 0.2 * n(D)).to(dev), "scale": (0.5 + 0.2 * n(D)).to(dev) if scale else None,
            "dh": n(R, D).to(dtype).to(dev), "dx": n(R, D).to(dtype).to(dev)}


def _norm_run(ops, c, eps=1e-6, which=("dh", "dx")):
    leaf = {n: None if c[n] is None else c[n].detach().requires_grad_() for n in ("h", "y", "gate", "post", "pre", "scale")}
    h, x = ops.gated_residual_norm(leaf["h"], leaf["y"], leaf["post"], leaf["pre"], gate=leaf["gate"], scale=leaf["scale"], eps=eps)
    names = [n for n in leaf if leaf[n] is not None]
    outs, gs = zip(*[(o, c[w]) for o, w in ((h, "dh"), (x, "dx")) if w in which])
    got = torch.autograd.grad(outs, [leaf[n] for n in names], gs, allow_unused=True)
    return {"h": h, "x": x, **{"d" + n: t for n, t in zip(names, got)}}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gate,scale", [(True, True), (False, False), (True, False), (False, True)])
@pytest.mark.parametrize("R,D", [(1, 1), (600, 5000), (1100, 2500), (1, 128), (3, 3), (5, 16), (300, 17), (1025, 100), (64, 128), (7, 513), (33, 1024), (2100, 64), (10, 2048),
                                 (3, 4100), (5, 8192), (2, 8191)])
def test_norm(ops, gpu_device, R, D, gate, scale, dtype):
    c = _norm_case(R, D, dtype, gpu_device, gate, scale)
    v, m = ref.norm(c["h"], c["y"], c["post"], c["pre"], c["gate"], c["scale"], 1e-6, c["dh"], c["dx"])
    tol = ref.norm_bounds(dtype, R, D, v, m)
    ref.check(_norm_run(ops, c), {n: x for n, x in v.items() if gate or n != "dgate"}, tol, "%d x %d" % (R, D))
    with torch.no_grad():
        h, x = ops.gated_residual_norm(c["h"], c["y"], c["post"], c["pre"], gate=c["gate"], scale=c["scale"])
    ref.check({"h": h, "x": x}, {"h": v["h"], "x": v["x"]}, tol, "no grad")


@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_layouts_and_parts(ops, gpu_device, dtype):
    """Rows of a wider tensor, more dimensions, one gradient of two, an eps that matters, rows that are all zeros, no rows."""
    c = _norm_case(60, 48, dtype, gpu_device)
    plain = _norm_run(ops, c)
    wide = torch.cat([c["y"], c["gate"], c["h"]], 1)
    d = dict(c, y=wide[:, :48], gate=wide[:, 48:96], h=wide[:, 96:])
    got = _norm_run(ops, d)
    for n in plain:
        assert torch.equal(got[n], plain[n]), n
    d = {n: x.view(3, 20, 48).transpose(0, 1) if n in ("h", "y", "gate", "dh", "dx") else x for n, x in c.items()}
    got = _norm_run(ops, d)
    for n in plain:
        if n in ("dpost", "dpre", "dscale"):                          # (the rows come in another order)
            assert float((got[n] - plain[n]).abs().max()) <= 60 * 2 * ref.U32 * 60 * float(plain[n].abs().max()) + 1e-6
        else:
            assert torch.equal(got[n].transpose(0, 1).reshape(60, 48), plain[n]), n
    for which in ("dh", "dx"):
        v, m = ref.norm(c["h"], c["y"], c["post"], c["pre"], c["gate"], c["scale"], 0.3, c["dh"] if which == "dh" else None, c["dx"] if which == "dx" else None)
        ref.check(_norm_run(ops, c, 0.3, (which,)), v, ref.norm_bounds(dtype, 60, 48, v, m), which)
    z = {n: torch.zeros_like(x) if n in ("h", "y") else x for n, x in c.items()}
    for n, x in _norm_run(ops, z).items():
        assert torch.isfinite(x).all(), n
    e = {n: x[:0] if n in ("h", "y", "gate", "dh", "dx") else x for n, x in c.items()}
    got = _norm_run(ops, e)
    assert got["h"].shape == (0, 48) and not got["dpost"].any() and got["dgate"].shape == (0, 48)


def test_each_gradient_by_itself(ops, gpu_device):
    """Any one tensor may be the only one that asks for a gradient."""
    for gate, scale in ((True, True), (False, True), (True, False)):
        c = _norm_case(30, 40, torch.float32, gpu_device, gate, scale)
        whole = _norm_run(ops, c)
        for n in ("h", "y", "gate", "post", "pre", "scale"):
            if c[n] is not None:
                d = dict(c, **{n: c[n].detach().requires_grad_()})
                h, x = ops.gated_residual_norm(d["h"], d["y"], d["post"], d["pre"], gate=d["gate"], scale=d["scale"])
                assert torch.equal(torch.autograd.grad([h, x], [d[n]], [c["dh"], c["dx"]])[0], whole["d" + n]), n
    for state in (True, False):
        c = _case(2, 40, 2, 16, 24, torch.float32, gpu_device, True, state)
        whole = _run(ops, c)
        for n in ("q", "k", "v", "s0"):
            if c[n] is not None:
                d = dict(c, **{n: c[n].detach().requires_grad_()})
                r = ops.decay_attention(d["q"], d["k"], d["v"], d["log_decay"], initial_state=d["s0"], starts=d["starts"], lengths=d["lengths"],
                                        output_final_state=state)
                got, = torch.autograd.grad(r, [d[n]], [c["do"], c["ds"]] if state else [c["do"]])
                assert torch.equal(got, whole["d" + n]), n


def test_norm_differences(ops, gpu_device):
    """The gradients against central differences of the formula in 64 bits, along random directions."""
    c = _norm_case(11, 20, torch.float32, gpu_device)
    got = _norm_run(ops, c)

    def loss(**kw):
        d = dict(c, **kw)
        v, _ = ref.norm(d["h"], d["y"], d["post"], d["pre"], d["gate"], d["scale"], 1e-6)
        return float((v["h"] * c["dh"].double().cpu()).sum() + (v["x"] * c["dx"].double().cpu()).sum())

    g, w = _gen(9), 1e-4
    for n in ("h", "y", "gate", "post", "pre", "scale"):
        e = torch.randn(c[n].shape, generator=g).double()
        x = c[n].double().cpu()
        num = (loss(**{n: x + w * e}) - loss(**{n: x - w * e})) / (2 * w)
        ana = got["d" + n].double().cpu() * e
        assert abs(num - float(ana.sum())) < 1e-5 * float(ana.abs().sum()), n      # w^2 = 1e-8 of third derivatives of size 1, fp32 gradients


def test_norm_row_that_is_not_finite_stays_alone(ops, gpu_device):
    c = _norm_case(70, 96, torch.float32, gpu_device)
    clean = _norm_run(ops, c)
    d = dict(c, y=c["y"].clone())
    d["y"][31, 4] = float("nan")
    got = _norm_run(ops, d)
    keep = torch.arange(70, device=gpu_device) != 31
    for n in ("h", "x", "dh", "dy", "dgate"):
        assert torch.equal(got[n][keep], clean[n][keep]), n
    for z in (float("inf"), -float("inf"), 1e30, -1e30):              # a gate that is open or shut for good
        d = dict(c, gate=torch.full_like(c["gate"], z))
        for n, x in _norm_run(ops, d).items():
            assert torch.isfinite(x).all(), n


# -------------------------------------------------------------------------------------------- streams, graphs, repetition
def _everything(ops, c, nc, step_state):
    got = _run(ops, c)
    got.update({"n" + n: x for n, x in _norm_run(ops, nc).items()})
    step_state.copy_(c["s0"])
    got["step"] = ops.decay_attention_step(c["q"][:, 0].detach(), c["k"][:, 0].detach(), c["v"][:, 0].detach(), c["log_decay"], step_state, starts=c["starts"][:, 0])
    return got


@pytest.mark.parametrize("dtype", DTYPES)
def test_repeated_on_other_streams_and_in_graphs(ops, gpu_device, dtype):
    """The same bits every time; two captured graphs that run in turn, with eager work between their replays and new inputs."""
    cs = [_case(2, 600, 2, 64, 64, dtype, gpu_device, True, True, seed=s) for s in (1, 2)]
    ncs = [_norm_case(1500, 100, dtype, gpu_device), _norm_case(900, 100, dtype, gpu_device)]
    states = [torch.empty_like(c["s0"]) for c in cs]
    want = [{n: x.detach().clone() for n, x in _everything(ops, c, nc, s).items()} for c, nc, s in zip(cs, ncs, states)]
    for i in range(2):
        again = _everything(ops, cs[i], ncs[i], states[i])
        assert all(torch.equal(again[n], want[i][n]) for n in want[i])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _everything(ops, cs[0], ncs[0], states[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(other[n], want[0][n]) for n in want[0])
    del again, other
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append({n: x.detach() for n, x in _everything(ops, cs[i], ncs[i], states[i]).items()})
        graphs.append(g)
    for turn in range(3):
        for i in (0, 1):
            graphs[i].replay()
            _everything(ops, cs[1 - i], ncs[1 - i], torch.empty_like(states[0]))
            torch.cuda.synchronize()
            for n in want[i]:
                assert torch.equal(outs[i][n], want[i][n]), (turn, i, n)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(outs[i][n], want[i][n]) for i in (0, 1) for n in want[i])
    keep = cs[0]["q"].clone()
    cs[0]["q"].copy_(cs[1]["q"])                                      # new values in the captured inputs
    fresh = {n: x.detach().clone() for n, x in _everything(ops, cs[0], ncs[0], torch.empty_like(states[0])).items()}
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(outs[0][n], fresh[n]) for n in fresh)
    cs[0]["q"].copy_(keep)


def test_a_long_cache_of_offsets(ops, gpu_device):
    """Rows that lie over 2^31 elements into their tensor."""
    T, H, D, B = 64, 1, 32, 3
    stride = 1_200_000_000
    big = torch.empty(2 * stride + T * H * D, dtype=torch.bfloat16, device=gpu_device)
    rows = big.as_strided((B, T, H, D), (stride, H * D, D, 1))
    c = _case(B, T, H, D, D, torch.bfloat16, gpu_device)
    rows.copy_(c["v"])
    want = _run(ops, c, train=False)["out"]
    assert torch.equal(ops.decay_attention(c["q"], c["k"], rows, c["log_decay"]), want)
    rows.copy_(c["q"])
    assert torch.equal(ops.decay_attention(rows, c["k"], c["v"], c["log_decay"]), want)
    tokens = big.as_strided((1, 5, H, D), (0, 40_000_000, D, 1))       # tokens 80 MB apart
    tokens.copy_(c["v"][:1, :5])
    assert torch.equal(ops.decay_attention(c["q"][:1, :5], c["k"][:1, :5], tokens, c["log_decay"]), want[:1, :5])


def test_many_rows_of_offsets(ops, gpu_device):
    """Norm rows and states over 2^31 elements into their tensors: the last of them as if they were alone."""
    R, D = 270_000, 8192
    y = torch.empty(R, D, dtype=torch.bfloat16, device=gpu_device)
    y[:-300] = 1.0
    y[-300:] = torch.randn(300, D, generator=_gen(5)).to(torch.bfloat16).to(gpu_device)
    post, pre = torch.rand(D, generator=_gen(6)).to(gpu_device), torch.rand(D, generator=_gen(7)).to(gpu_device)
    h, x = ops.gated_residual_norm(y, y, post, pre, gate=y)
    h1, x1 = ops.gated_residual_norm(y[-300:], y[-300:], post, pre, gate=y[-300:])
    assert torch.equal(h[-300:], h1) and torch.equal(x[-300:], x1)
    del h, x
    leaf, last = y.detach().requires_grad_(), y[-300:].detach().requires_grad_()
    g = torch.autograd.grad(ops.gated_residual_norm(leaf, leaf, post, pre), [leaf], [y, y])[0]
    assert torch.equal(g[-300:], torch.autograd.grad(ops.gated_residual_norm(last, last, post, pre), [last], [y[-300:], y[-300:]])[0])
    del y, leaf, last, g
    N, H, K = 140_000, 1, 128
    state = torch.zeros(N, H, K, K, device=gpu_device)
    q, k, v = (torch.randn(N, H, K, generator=_gen(s)).to(gpu_device) for s in (1, 2, 3))
    state[-9:] = torch.randn(9, H, K, K, generator=_gen(4)).to(gpu_device)
    few, decay = state[-9:].clone(), torch.full((H,), -0.1, device=gpu_device)
    out = ops.decay_attention_step(q, k, v, decay, state)
    assert torch.equal(out[-9:], ops.decay_attention_step(q[-9:], k[-9:], v[-9:], decay, few)) and torch.equal(state[-9:], few)


@pytest.mark.parametrize("dtype", DTYPES)
def test_small_heads_go_on_in_steps(ops, gpu_device, dtype):
    """Heads of less than 16 bytes: the window's state is one that the step form takes."""
    c = _case(2, 9, 2, 3, 1, dtype, gpu_device, False, True)
    whole, end = ops.decay_attention(c["q"], c["k"], c["v"], c["log_decay"], initial_state=c["s0"], output_final_state=True)
    out, state = ops.decay_attention(c["q"][:, :8], c["k"][:, :8], c["v"][:, :8], c["log_decay"], initial_state=c["s0"], output_final_state=True)
    last = ops.decay_attention_step(c["q"][:, 8], c["k"][:, 8], c["v"][:, 8], c["log_decay"], state)
    r, mag = _both({**c, "do": torch.zeros_like(c["do"]), "ds": torch.zeros_like(c["ds"])}, 3 ** -0.5)
    tol = ref.attention_bounds(dtype, 9, 3, 1, r, mag)
    ref.check({"out": torch.cat([out, last[:, None]], 1), "state": state}, {"out": r["out"], "state": r["state"]}, tol)
    ref.check({"out": whole, "state": end}, {"out": r["out"], "state": r["state"]}, tol)


def test_a_second_derivative_is_refused(ops, gpu_device):
    c, nc = _case(1, 9, 1, 8, 8, torch.float32, gpu_device), _norm_case(4, 8, torch.float32, gpu_device)
    q = c["q"].detach().requires_grad_()
    out = ops.decay_attention(q, c["k"], c["v"], c["log_decay"])
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad([out], [q], [c["do"]], create_graph=True)
    y = nc["y"].detach().requires_grad_()
    h, _ = ops.gated_residual_norm(nc["h"], y, nc["post"], nc["pre"])
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad([h], [y], [nc["dh"]], create_graph=True)


def test_inputs_changed_before_the_backward_pass_are_noticed(ops, gpu_device):
    c = _case(1, 9, 1, 8, 8, torch.float32, gpu_device)
    q, k = c["q"].detach().clone().requires_grad_(), c["k"].clone()
    out = ops.decay_attention(q, k, c["v"], c["log_decay"])
    k.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    state = torch.zeros(1, 1, 8, 8, device=gpu_device)
    loss = (state * torch.ones(1, device=gpu_device, requires_grad=True)).sum()
    ops.decay_attention_step(c["q"][:, 0], c["k"][:, 0], c["v"][:, 0], c["log_decay"], state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_a_capture_beside_a_living_graph_of_its_leaves_is_refused(ops, gpu_device):
    """Its backward pass would wait, within a capture, for the other graph's stream: refused in the forward pass, before anything."""
    c, nc = _case(1, 9, 1, 8, 8, torch.float32, gpu_device), _norm_case(4, 8, torch.float32, gpu_device)
    q, w = c["q"].detach().requires_grad_(), nc["post"].detach().requires_grad_()
    out = ops.decay_attention(q, c["k"], c["v"], c["log_decay"])
    h, x = ops.gated_residual_norm(nc["h"], nc["y"], w, nc["pre"])
    torch.cuda.synchronize()
    g, t = torch.cuda.CUDAGraph(), torch.ones(4, device=gpu_device)
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="another stream"):
            ops.decay_attention(q, c["k"], c["v"], c["log_decay"])
        with pytest.raises(RuntimeError, match="another stream"):
            ops.gated_residual_norm(nc["h"], nc["y"], w, nc["pre"])
        t.mul_(2)
    want = torch.autograd.grad(out, q, c["do"])[0].clone(), torch.autograd.grad([h, x], w, [nc["dh"], nc["dx"]])[0].clone()
    del out, h, x
    g2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g2):
        out = ops.decay_attention(q, c["k"], c["v"], c["log_decay"])
        h, x = ops.gated_residual_norm(nc["h"], nc["y"], w, nc["pre"])
        got = torch.autograd.grad(out, q, c["do"])[0], torch.autograd.grad([h, x], w, [nc["dh"], nc["dx"]])[0]
    for _ in range(3):
        g2.replay()
        t.add_(1)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
