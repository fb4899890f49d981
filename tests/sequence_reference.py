"""The sequence operators by their formulas, in 64 bits on the CPU, and what their kernels may be off.

Every bound counts roundings: a sum of n fp32 products is off by at most n 2^-24 of the sum of the products' magnitudes, which is
what the same formula gives for the magnitudes of its inputs.  A bf16 value is off by 2^-8 of itself at most.
"""
import torch

U32, U16 = 2.0 ** -24, 2.0 ** -8


def attention(q, k, v, log_decay, scale, s0=None, starts=None, lengths=None, do=None, ds=None):
    """The recurrence, token by token: {"out", "state"} and, with ``do`` / ``ds``, {"dq", "dk", "dv", "ds0"}."""
    q, k, v = (x.double().cpu() for x in (q, k, v))
    B, T, H, DK = q.shape
    DV = v.shape[3]
    g = torch.exp(log_decay.double().cpu()).view(1, H, 1, 1)
    S = torch.zeros(B, H, DK, DV, dtype=torch.float64) if s0 is None else s0.double().cpu().clone()
    starts = torch.zeros(B, T, dtype=torch.bool) if starts is None else starts.cpu().bool()
    lengths = torch.full((B,), T) if lengths is None else lengths.cpu().long().clamp(0, T)
    out, states = torch.zeros(B, T, H, DV, dtype=torch.float64), []
    for t in range(T):
        on, fresh = (t < lengths).view(B, 1, 1, 1), starts[:, t].view(B, 1, 1, 1)
        S = torch.where(on, torch.where(fresh, torch.zeros_like(S), g * S) + k[:, t, :, :, None] * v[:, t, :, None, :], S)
        states.append(S)
        out[:, t] = torch.where(on[..., 0], torch.einsum("bhi,bhij->bhj", q[:, t], S) * scale, torch.zeros(()).double())
    res = {"out": out, "state": S}
    if do is None and ds is None:
        return res
    do = torch.zeros_like(out) if do is None else do.double().cpu()
    G = torch.zeros_like(S) if ds is None else ds.double().cpu().clone()
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    zero = torch.zeros(()).double()
    for t in range(T - 1, -1, -1):
        on, fresh = (t < lengths).view(B, 1, 1, 1), starts[:, t].view(B, 1, 1, 1)
        dq[:, t] = torch.where(on[..., 0], torch.einsum("bhij,bhj->bhi", states[t], do[:, t]) * scale, zero)
        X = G + q[:, t, :, :, None] * do[:, t, :, None, :] * scale
        dk[:, t] = torch.where(on[..., 0], torch.einsum("bhij,bhj->bhi", X, v[:, t]), zero)
        dv[:, t] = torch.where(on[..., 0], torch.einsum("bhij,bhi->bhj", X, k[:, t]), zero)
        G = torch.where(on, torch.where(fresh, torch.zeros_like(X), g * X), G)
    res.update(dq=dq, dk=dk, dv=dv, ds0=G)
    return res


def attention_bounds(dtype, T, DK, DV, ref, magnitudes):
    """What each output may be off.  Roundings of a term, in fp32: a dot product over a head (DK or DV), a sum over tokens (T, each of
    them scaled once), and the weight g^n, whose exponent is off by 2 2^-24 relative to a number below 150 where the weight is not
    zero; 400 covers it and the few single products.  With bf16 inputs each term is rounded once more as an operand of the matrix
    cores, in the weighted scores or in the state that it passes through, and the output once.  A weight below 2^-126 is zero in fp32,
    so what it multiplies is lost: less than 2^-126 times the sum of the other factors' products, which stays below 2^23 for the
    normal deviates, lengths and head sizes used here (2^10 tokens, 2^7 columns, products of three below 2^6 on average)."""
    n = 2 * T + DK + DV + 400
    tol = {}
    for name, m in magnitudes.items():
        tol[name] = n * U32 * m + 2.0 ** (23 - 126)
        if dtype == torch.bfloat16 and name not in ("state", "ds0"):
            tol[name] = tol[name] + (1 + U16) * U16 * (m + ref[name].abs())
    return tol


def norm(h, y, post, pre, gate, scale, eps, dh=None, dx=None):
    """gated_residual_norm and its gradients: ({name: value}, {name: magnitude of its terms})."""
    f = lambda t: None if t is None else t.double().cpu()  # noqa: E731
    h, y, post, pre, gate, scale, dh, dx = (f(t) for t in (h, y, post, pre, gate, scale, dh, dx))
    sg = torch.ones_like(y) if gate is None else torch.sigmoid(gate)
    cs = torch.zeros_like(y) if gate is None else torch.sigmoid(-gate)
    sc = torch.ones_like(post) if scale is None else scale
    ry = ((y * y).mean(1, keepdim=True) + eps) ** -0.5
    n0 = y * ry
    u = n0 * post * sg
    hn = h + sc * u
    rh = ((hn * hn).mean(1, keepdim=True) + eps) ** -0.5
    val = {"h": hn, "x": hn * rh * pre}
    hm = h.abs() + (sc * u).abs()
    mag = {"h": hm, "x": (hm * rh * pre).abs() + (hn * rh * pre).abs() * (hm * hn.abs()).mean(1, keepdim=True) * rh * rh}
    if dh is None and dx is None:
        return val, mag
    dh = torch.zeros_like(h) if dh is None else dh
    dx = torch.zeros_like(h) if dx is None else dx
    w = dx * pre
    a = (w * hn).mean(1, keepdim=True)
    d = dh + rh * (w - hn * rh * rh * a)
    am = (w.abs() * hm).mean(1, keepdim=True)
    rm = 1 + (hm * hn.abs()).mean(1, keepdim=True) * rh * rh      # how much of its own size an error of h' adds to rh
    dm = dh.abs() + rh * (w.abs() + hm * rh * rh * am) * rm
    dn = d * sc * sg * post
    dnm = dm * (sc * sg * post).abs()
    b = (dn * y).mean(1, keepdim=True)
    val.update(dh=d, dy=ry * (dn - y * ry * ry * b), dgate=d * sc * n0 * post * sg * cs, dpost=(d * sc * sg * n0).sum(0),
               dpre=(dx * hn * rh).sum(0), dscale=(d * u).sum(0))
    mag.update(dh=dm, dy=ry * (dnm + y.abs() * ry * ry * (dnm * y.abs()).mean(1, keepdim=True)), dgate=dm * (sc * n0 * post * sg * cs).abs(),
               dpost=(dm * (sc * sg * n0).abs()).sum(0), dpre=(dx.abs() * hm * rh * rm).sum(0), dscale=(dm * u.abs()).sum(0))
    return val, mag


def norm_bounds(dtype, R, D, ref, magnitudes):
    """Roundings of a term: a mean over the row twice over (2 D), the few single products, the sigmoid's exponent (its argument is off
    by 2^-24 of a number below 100 where the result is not zero) and, for the weights, a sum over the rows (R)."""
    tol = {}
    for name, m in magnitudes.items():
        weight = name in ("dpost", "dpre", "dscale")
        tol[name] = (2 * D + 200 + (R if weight else 0)) * U32 * m
        if dtype == torch.bfloat16 and not weight:
            tol[name] = tol[name] + (1 + U16) * U16 * ref[name].abs()
    return tol


def check(got, ref, tol, what=""):
    for name, r in ref.items():
        if name not in got or got[name] is None:
            continue
        x = got[name].detach().double().cpu()
        assert x.shape == r.shape, (what, name, x.shape, r.shape)
        over = (x - r).abs() - tol[name]
        assert bool((over <= 0).all()), "%s %s: off by %.3g where %.3g is allowed" % (
            what, name, float((x - r).abs().flatten()[over.argmax()]) if x.numel() else 0.0, float(tol[name].flatten()[over.argmax()]))
