"""The sequence-policy operators in 64 bits, each value with a bound on a float32 kernel's error.

E = 2^-24 is half a float32 step. The kernels' exp and reciprocal are good to one unit in the last place
(2 E) and exp's argument is rounded twice (2 E |x| relative in the result), so a sigmoid of x is off by at
most (6 + 2 |x|) E relative: one addition, one reciprocal, and an exponential whose error counts at most once.
Outputs in a type of half step u = finfo(type).eps / 2 are off by u |value| more, and by half the smallest
subnormal.
"""

import torch

E = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounding(ref, dtype):
    """Bound of rounding `ref` to dtype once."""
    if dtype == torch.float64:
        return torch.zeros_like(ref)
    return half_step(dtype) * ref.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def check(got, ref, bound, what):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, f"{what}: shape {tuple(got.shape)}, not {tuple(ref.shape)}"
    nan = ref.isnan()
    assert torch.equal(got.isnan(), nan), f"{what}: NaN at other places"
    off = torch.where(nan, torch.zeros_like(ref), (got - ref).abs())
    over = (off - bound).masked_fill(nan, -1.0)
    if over.numel() and float(over.max()) > 0:
        at = int(over.argmax())
        raise AssertionError(f"{what}: off by {float(off.reshape(-1)[at]):.3g}, allowed {float(bound.reshape(-1)[at]):.3g}, "
                             f"value {float(ref.reshape(-1)[at]):.6g} at {at} of {ref.numel()}")


def recurrence(gates, state, keep, lengths, d_h=None, d_last=None):
    """{name: (value, bound)} of h, last, d_gates, d_state, step by step."""
    dtype = gates.dtype
    gates = gates.detach().double().cpu()
    n, T, U3 = gates.shape
    U = U3 // 3
    xf, z, xo = gates.split(U, 2)
    f, b, o, ob = torch.sigmoid(xf), torch.sigmoid(-xf), torch.sigmoid(xo), torch.sigmoid(-xo)
    sf, so = (8 + 2 * xf.abs()) * E, (8 + 2 * xo.abs()) * E      # a gate, with the product it enters
    c = torch.zeros(n, U, dtype=torch.float64) if state is None else state.detach().double().cpu()
    keep = torch.ones(n, T, dtype=torch.float64) if keep is None else keep.double().cpu()
    lengths = torch.full((n,), T) if lengths is None else lengths.long().cpu()
    live = (torch.arange(T)[None] < lengths[:, None])[..., None]
    err = torch.zeros_like(c)
    P, PE, Cs, CE = (torch.zeros(n, T, U, dtype=torch.float64) for _ in range(4))
    for t in range(T):
        k = torch.ones(n, 1, dtype=torch.float64) if t == 0 else keep[:, t - 1:t]
        on = live[:, t]
        p, pe = c * k, (err + E * c.abs()) * k.abs()
        now = f[:, t] * p + b[:, t] * z[:, t]
        # one more step's products and sums, whatever the order in which steps are joined
        ne = f[:, t] * pe + sf[:, t] * ((f[:, t] * p).abs() + (b[:, t] * z[:, t]).abs()) + 2 * E * now.abs()
        c, err = torch.where(on, now, c), torch.where(on, ne, err)
        P[:, t], PE[:, t], Cs[:, t], CE[:, t] = p, pe, c, err
    zero = torch.zeros((), dtype=torch.float64)
    h = torch.where(live, o * Cs, zero)
    out = {"h": (h, torch.where(live, o * CE + so * h.abs(), zero) + rounding(h, dtype)),
           "last": (c, err + E * c.abs())}
    if d_h is None and d_last is None:
        return out
    d_h = torch.zeros(n, T, U, dtype=torch.float64) if d_h is None else d_h.double().cpu()
    d_h = torch.where(live, d_h, zero)
    back = torch.zeros(n, U, dtype=torch.float64) if d_last is None else d_last.double().cpu()
    berr = torch.zeros_like(back)
    dg, ge = torch.zeros_like(gates), torch.zeros_like(gates)
    for t in range(T - 1, -1, -1):
        on = live[:, t]
        k = torch.ones(n, 1, dtype=torch.float64) if t == 0 else keep[:, t - 1:t]
        ft, bt, zt, pt, dh = f[:, t], b[:, t], z[:, t], P[:, t], d_h[:, t]
        od = o[:, t] * dh
        D = back + od
        De = berr + so[:, t] * od.abs() + E * D.abs()
        w = ft * bt
        we = w * (12 + 4 * xf[:, t].abs()) * E
        dxf, dxz, dxo = D * (pt - zt) * w, D * bt, dh * Cs[:, t] * o[:, t] * ob[:, t]
        dxfe = De * (pt - zt).abs() * w + D.abs() * (PE[:, t] + E * (pt - zt).abs()) * w + (D * (pt - zt)).abs() * we
        dxze = De * bt + D.abs() * bt * sf[:, t]
        dxoe = (dh * o[:, t] * ob[:, t]).abs() * CE[:, t] + dxo.abs() * (12 + 4 * xo[:, t].abs()) * E
        for j, (v, e) in enumerate(((dxf, dxfe), (dxz, dxze), (dxo, dxoe))):
            dg[:, t, j * U:(j + 1) * U] = torch.where(on, v, zero)
            ge[:, t, j * U:(j + 1) * U] = torch.where(on, e, zero)
        nb, nbe = ft * k * D, (ft * k).abs() * De + sf[:, t] * (ft * k * D).abs()
        back, berr = torch.where(on, nb, back), torch.where(on, nbe, berr)
    out["d_gates"] = (dg, ge + rounding(dg, dtype))
    out["d_state"] = (back, berr + E * back.abs())
    return out


def norm(x, residual, weight, eps, d_y=None, d_stream=None):
    """{name: (value, bound)} of y, stream, dx, dw. A sum of D terms in any order that adds at most D / 64 of
    them one after another, then joins 64 and the waves, is off by (D / 64 + 16) E of the sum of magnitudes."""
    dtype = x.dtype
    x, D = x.detach().double().cpu(), x.shape[-1]
    s = x if residual is None else x + residual.detach().double().cpu()
    w = torch.ones(D, dtype=torch.float64) if weight is None else weight.detach().double().cpu()
    long = (D / 64 + 16) * E
    inv = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    n = s * inv
    rel = long + 8 * E                         # of inv: half the sum's error, root, quotient, and the sum's own rounding
    out = {"y": (n * w, (rel + 4 * E) * (n * w).abs() + rounding(n * w, dtype)),
           "stream": (s, rounding(s, dtype) + E * s.abs())}
    if d_y is None:
        return out
    u = E if residual is not None else 0.0      # the sum's rounding
    dy = d_y.double().cpu()
    ds = torch.zeros_like(s) if d_stream is None else d_stream.double().cpu()
    g = dy * w
    mean, size = (g * n).mean(-1, keepdim=True), (g * n).abs().mean(-1, keepdim=True)
    dx = inv * (g - n * mean) + ds
    me = (u + rel + long + 4 * E) * size
    bound = inv * (n.abs() * me + (u + rel + 4 * E) * (n * mean).abs() + 4 * E * (g.abs() + (n * mean).abs()))
    bound = bound + (rel + 4 * E) * (inv * (g - n * mean)).abs() + 2 * E * ds.abs()
    out["dx"] = (dx, bound + rounding(dx, dtype))
    rows = dy.reshape(-1, D).shape[0]
    terms = (dy * n).reshape(-1, D)
    dw = terms.sum(0)
    out["dw"] = (dw, (u + rel + (rows + 16) * E) * terms.abs().sum(0) + rounding(dw, dtype))
    return out


def rows_of(logits, actions):
    """(log-probability, its bound, entropy, its bound, log-probabilities, p) per row. With d = z - max and p the
    probabilities: an exponential is off by (4 + 2 |d|) E, the sums of K by (K / 64 + 16) E."""
    z = logits.detach().double().cpu()
    K = z.shape[1]
    m = z.max(1, keepdim=True).values
    d = z - m
    log_p = torch.log_softmax(z, 1)
    p = log_p.exp()
    dd = torch.where(p > 0, d, torch.zeros_like(d)).abs()
    mean_d, mean_d2 = (p * dd).sum(1), (p * dd * dd).sum(1)
    long = (K / 64 + 20) * E
    a = actions.cpu().long()
    ok = (a >= 0) & (a < K)
    at = a.clamp(0, K - 1)[:, None]
    l = torch.where(ok, log_p.gather(1, at)[:, 0], torch.nan)
    da = dd.gather(1, at)[:, 0]
    log_s = (torch.logsumexp(z, 1) - m[:, 0]).abs()
    l_err = long + 2 * E * mean_d + 2 * E * (da + log_s) + 2 * E * l.abs().nan_to_num(0.0, 0.0, 0.0)
    H = -(p * torch.where(p > 0, log_p, torch.zeros_like(log_p))).sum(1)
    H = torch.where(torch.isnan(l) & ok, torch.nan, H)
    H_err = long * (1 + 2 * mean_d) + 2 * E * (mean_d + mean_d2) + 4 * E * (log_s + mean_d)
    return l, l_err, H, H_err, log_p, p


def policy_loss(logits, actions, old, adv, ref, mask, denom, lo, hi, kl_coef, entropy_coef, g=1.0):
    """{name: (value, bound)} of loss, terms, d_logits (for the incoming gradient g)."""
    dtype = logits.dtype
    M, K = logits.shape
    live = torch.ones(M, dtype=torch.bool) if mask is None else mask.cpu()
    z = torch.where(live[:, None], logits.detach().double().cpu(), torch.zeros(1, dtype=torch.float64))
    a = torch.where(live, actions.cpu().long(), torch.zeros(1, dtype=torch.long))
    l, le, H, He, log_p, p = rows_of(z, a)
    zero = torch.zeros((), dtype=torch.float64)
    n = float(denom) if denom is not None else max(1, int(live.sum()))
    A, x = adv.double().cpu(), l - old.double().cpu()
    xe = le + E * x.abs()
    xb = x.clamp(-20, 20)
    r = xb.exp()
    re = r * (xe + 6 * E + 2 * E * xb.abs())
    u, v = r * A, r.clamp(lo, hi) * A
    pg, pge = -torch.minimum(u, v), A.abs() * re + 4 * E * u.abs()
    inside = (x >= -20) & (x <= 20)
    gl, gle = torch.where((u <= v) & inside, -u, zero), pge
    kl, kle = torch.zeros_like(pg), torch.zeros_like(pg)
    if ref is not None:
        y = ref.double().cpu() - l
        d = y.clamp(-20, 20)
        e = d.exp()
        ye = le + E * y.abs()
        kl, kle = e - d - 1, (e - 1).abs() * ye + e * (8 * E + 2 * E * d.abs()) + 4 * E * (d.abs() + 1)
        gin = (y >= -20) & (y <= 20)
        gl = gl + torch.where(gin, kl_coef * (1 - e), zero)
        gle = gle + abs(kl_coef) * e * (ye + 8 * E + 2 * E * d.abs())
    out = ((r < lo) | (r > hi)).double()
    row = pg + kl_coef * kl - entropy_coef * H
    rowe = pge + abs(kl_coef) * kle + abs(entropy_coef) * He + 4 * E * (pg.abs() + abs(kl_coef) * kl + abs(entropy_coef) * H.abs())
    w = live.double()

    def total(v, e):
        v, e = torch.where(live, v, zero), torch.where(live, e, zero)
        return v.sum() / n, (e.sum() + (M / 64 + 8) * E * v.abs().sum()) / abs(n) + 2 * E * (v.sum() / n).abs()

    cols = [total(v, e) for v, e in ((pg, pge), (kl, kle), (H, He), (out, 0 * out))]
    res = {"loss": total(row, rowe), "terms": (torch.stack([c[0] for c in cols]), torch.stack([c[1] for c in cols]))}
    one = torch.zeros(M, K, dtype=torch.float64)
    one[torch.arange(M), a.clamp(0, K - 1)] = 1.0
    lp = torch.where(p > 0, log_p, zero)
    pe = p * (le[:, None] + (6 + 2 * lp.abs()) * E)
    s = (g / n * w)[:, None]
    dz = gl[:, None] * (one - p) + entropy_coef * p * (lp + H[:, None])
    de = gle[:, None] * (one - p).abs() + gl.abs()[:, None] * pe
    de = de + abs(entropy_coef) * (pe * (lp + H[:, None]).abs() + p * (He + le)[:, None] + 4 * E * p * (lp.abs() + H.abs()[:, None]))
    de = de + 6 * E * (gl[:, None] * (one + p)).abs()
    dz, de = torch.where(live[:, None], dz * s, zero), torch.where(live[:, None], de * s.abs(), zero)
    res["d_logits"] = (dz, de + 4 * E * dz.abs() + rounding(dz, dtype))
    return res
