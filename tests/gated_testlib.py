"""The gated linear recurrence and the group norm by their definitions in 64 bits, with their gradients, and bounds of the error that
the kernels' arithmetic may leave (u = 2^-24 is half a step of fp32; the rounding to the output's type comes on top in `assert_within`).

Gates.  For 16-bit tokens a sigmoid is an approximate exponential (2 steps of fp32, and its argument's rounding, |argument| u) and an
approximate reciprocal (1 step); for 32-bit ones both are good to 2 steps.  `gate_error` counts (8 + 4 |argument|) u for either, which
holds for the sigmoid and for 1 minus it, relatively."""
import torch

from serving_testlib import U


def gate_error(v):
    return (8 + 4 * v.abs()) * U


def gates64(x, r, i, rate, r_bias, i_bias, scale=8.0):
    """Decay, gain, term u of each token, and bounds of the relative errors of f (against |log f|), and of gain."""
    x, r = x.double(), r.double() + (r_bias.double() if r_bias is not None else 0.0)
    s, n = torch.sigmoid(r), torch.sigmoid(-r)
    if rate is not None:
        soft = torch.nn.functional.softplus(rate.double(), threshold=200.0)
        log = -scale * soft * s
        f, gain = log.exp(), (-(2.0 * log).expm1()).sqrt()
        # log f: the gate's error, 4 steps of softplus and products; f: that times |log f|, and the exponential; gain^2 = 1 - f^2: the error
        # of log f as long as it is small (d gain / gain <= half of it), else that of f; 2^-22 for the polynomial, the difference and the root
        log_e = gate_error(r) + 12 * U
        f_e = log.abs() * log_e + 8 * U
        gain_e = log_e + 2.0 ** -21
    else:
        log, f, gain = None, s, n
        f_e = gain_e = gate_error(r)
    g = torch.ones_like(x)
    g_e = torch.zeros_like(x)
    if i is not None:
        v = i.double() + (i_bias.double() if i_bias is not None else 0.0)
        g, g_e = torch.sigmoid(v), gate_error(v)
    u = gain * g * x
    return f, f_e, u, (gain_e + g_e + 4 * U) * u.abs()


def scan64(f, f_e, u, u_e, h0):
    """One sequence: f, u [L, C], h0 [C].  Returns the states and bounds of their errors.  The kernel joins maps instead of going token by
    token: each join is a product and a sum of what the formula has, off by u of the magnitudes, over 64 tokens 8 times, and once a tile:
    counted as 2 u a token on the running sum of the magnitudes."""
    h, e, mag = h0.double(), torch.zeros_like(h0, dtype=torch.float64), h0.double().abs()
    hs, es = torch.empty_like(u), torch.empty_like(u)
    for t in range(u.shape[0]):
        e = f[t] * (e + (f_e[t] + 2 * U) * mag) + u_e[t]
        h, mag = f[t] * h + u[t], f[t] * mag + u[t].abs()
        e = e + 2 * U * mag
        hs[t], es[t] = h, e
    return hs, es


def spans(lens):
    at = 0
    for n in lens:
        yield at, at + n
        at += n


def forward64(lens, x, r, i, rate, r_bias, i_bias, states, scale=8.0):
    """x, r, i [T, C], states [N, C].  Returns y, its bound, final states, their bound."""
    f, f_e, u, u_e = gates64(x, r, i, rate, r_bias, i_bias, scale)
    y, e = torch.zeros_like(u), torch.zeros_like(u)
    final, final_e = states.double().clone(), torch.zeros_like(states, dtype=torch.float64)
    for k, (a, b) in enumerate(spans(lens)):
        if b > a:
            y[a:b], e[a:b] = scan64(f[a:b], f_e[a:b], u[a:b], u_e[a:b], states[k])
            final[k], final_e[k] = y[b - 1], e[b - 1]
    return y, e, final, final_e


def autograd64(lens, tensors, states, dy, dfinal, scale=8.0):
    """Gradients by differentiating the definition, token by token.  tensors: x, r, i, rate, r_bias, i_bias (None where absent);
    returns a list like tensors + [states]."""
    v = [None if t is None else t.detach().double().requires_grad_() for t in tensors]
    h0 = states.detach().double().requires_grad_()
    x, r, i, rate, r_bias, i_bias = v
    rr = r + (r_bias if r_bias is not None else 0.0)
    if rate is not None:
        log = -scale * torch.nn.functional.softplus(rate, threshold=200.0) * torch.sigmoid(rr)
        f, gain = log.exp(), (-(2.0 * log).expm1()).sqrt()
    else:
        f, gain = torch.sigmoid(rr), torch.sigmoid(-rr)
    u = gain * x
    if i is not None:
        u = u * torch.sigmoid(i + (i_bias if i_bias is not None else 0.0))
    total = 0.0
    for k, (a, b) in enumerate(spans(lens)):
        h = h0[k]
        for t in range(a, b):
            h = f[t] * h + u[t]
            total = total + (h * dy[t].double()).sum()
        total = total + (h * dfinal[k].double()).sum()
    leaves = [t for t in (*v, h0) if t is not None]
    grads = iter(torch.autograd.grad(total, leaves))
    return [None if t is None else next(grads) for t in (*v, h0)]


def gradients64(lens, tensors, states, dy, dfinal, scale=8.0):
    """The same by the formulas, [(gradient, bound)] in the same order.  Each factor of a term carries its relative error as in
    `gates64`, the two terms of a difference their own bounds, the sums over T tokens T u of the sum of the magnitudes."""
    x, r, i, rate, r_bias, i_bias = tensors
    T = x.shape[0]
    rr = r.double() + (r_bias.double() if r_bias is not None else 0.0)
    f, f_e, u, u_e = gates64(x, r, i, rate, r_bias, i_bias, scale)
    s, n, s_e = torch.sigmoid(rr), torch.sigmoid(-rr), gate_error(rr)
    X = x.double()
    if i is not None:
        v = i.double() + (i_bias.double() if i_bias is not None else 0.0)
        g, ng, g_e = torch.sigmoid(v), torch.sigmoid(-v), gate_error(v)
    else:
        g, ng, g_e = torch.ones_like(X), torch.zeros_like(X), torch.zeros_like(X)
    if rate is not None:
        soft = torch.nn.functional.softplus(rate.double(), threshold=200.0)
        l = -scale * soft * s
        gain, l_e = (-(2.0 * l).expm1()).sqrt(), s_e + 12 * U
        gain_e = l_e + 2.0 ** -21
    else:
        gain, gain_e = n, s_e
    dh, dhE, before, beforeE = (torch.zeros_like(X) for _ in range(4))
    dstate, dstateE = dfinal.double().clone(), torch.zeros_like(dfinal, dtype=torch.float64)
    for k, (a, b) in enumerate(spans(lens)):
        if b == a:
            continue
        h, hE = scan64(f[a:b], f_e[a:b], u[a:b], u_e[a:b], states[k])
        before[a], before[a + 1:b], beforeE[a + 1:b] = states[k].double(), h[:-1], hE[:-1]
        back = torch.cat([torch.ones_like(f[:1]), f[a + 1:b].flip(0)])                 # dh[t] = f[t + 1] dh[t + 1] + dy[t]
        back_e = torch.cat([torch.zeros_like(f[:1]), f_e[a + 1:b].flip(0)])
        d, dE = scan64(back, back_e, dy[a:b].double().flip(0), torch.zeros_like(back), dfinal[k])
        dh[a:b], dhE[a:b] = d.flip(0), dE.flip(0) + 2 * U * d.flip(0).abs()
        dstate[k] = f[a] * dh[a]
        dstateE[k] = f[a] * dhE[a] + (f_e[a] + 2 * U) * dstate[k].abs()
    out = []
    dx = dh * gain * g
    out.append((dx, dhE * gain * g + (gain_e + g_e + 4 * U) * dx.abs()))
    if rate is not None:
        one, two = f * dh * before * l, dh * g * X * f * f * l / gain.clamp(min=1e-300)
        two = torch.where(l == 0, torch.zeros_like(two), two)
        m = one - two
        mE = (f * l).abs() * (dhE * before.abs() + dh.abs() * beforeE) + (f_e + l_e + 8 * U) * one.abs()
        mE = mE + dhE * (g * X * f * f * l / gain.clamp(min=1e-300)).abs() + (2 * f_e + l_e + g_e + gain_e + 2.0 ** -21 + 8 * U) * two.abs()
        dr, drE = m * n, mE * n + (s_e + 4 * U) * (m * n).abs()
        out.append((dr, drE))
    else:
        one, two = dh * before, dh * g * X
        dE = dhE * before.abs() + dh.abs() * beforeE + 4 * U * one.abs() + dhE * (g * X).abs() + (g_e + 4 * U) * two.abs()
        dr = (one - two) * s * n
        drE = dE * s * n + (2 * s_e + 4 * U) * dr.abs()
        out.append((dr, drE))
        m, mE = dr, drE
    total = lambda t, e: (t.sum(0), e.sum(0) + (T + 8) * U * t.abs().sum(0))  # noqa: E731
    di = dh * gain * X * g * ng
    diE = dhE * (gain * X * g * ng).abs() + (gain_e + 2 * g_e + 6 * U) * di.abs()
    out.append((di, diE) if i is not None else None)
    if rate is not None:
        ratio = torch.where(soft > 0, torch.sigmoid(rate.double()) / soft.clamp(min=1e-300), torch.ones_like(soft))
        t, e = total(m, mE)
        out.append((t * ratio, e * ratio + 16 * U * (t * ratio).abs()))
    else:
        out.append(None)
    out.append(total(dr, drE) if r_bias is not None else None)
    out.append(total(di, diE) if i_bias is not None else None)
    out.append((dstate, dstateE))
    return out


def act64(v, name):
    return {"silu": torch.nn.functional.silu, "sigmoid": torch.sigmoid, None: lambda t: t}[name](v)


def norm_bounds(x, G, weight, bias, z, act, eps, center, dy=None):
    """Bounds of the errors of y and, with dy, of dx, dweight, dbias, dz (64-bit values, a list).  S: a sum over the group's D values in
    registers and lanes, off by (D / 32 + 10) u of the magnitudes; xh is off by what the mean is, and by half of what the variance is."""
    T, C = x.shape
    D = C // G
    S = (D / 32 + 10) * U
    x = x.double().view(T, G, D)
    m = x.mean(-1, keepdim=True) if center else torch.zeros_like(x[..., :1])
    mE = S * x.abs().mean(-1, keepdim=True) if center else m
    d = x - m
    var = d.square().mean(-1, keepdim=True)
    rstd = 1.0 / (var + eps).sqrt()
    xh = d * rstd
    dE = mE + U * (x.abs() + m.abs())
    varE = S * var + 2.0 * (d.abs() * dE).mean(-1, keepdim=True) + dE.square().mean(-1, keepdim=True)
    rE = 0.5 * varE / (var + eps) + 4 * U                                          # relative
    xhE = dE * rstd + (rE + U) * xh.abs()
    w = weight.double().reshape(-1, D) if weight is not None else torch.ones_like(xh[:1])
    b = bias.double().reshape(-1, D) if bias is not None else torch.zeros_like(w)
    n = xh * w + b
    nE = xhE * w.abs() + 2 * U * ((xh * w).abs() + b.abs())
    zz = z.double().view_as(x) if z is not None else n
    p = torch.sigmoid(zz)
    a = {"silu": zz * p, "sigmoid": p, None: zz}[act]
    slope = {"silu": p * (1 + zz * (1 - p)), "sigmoid": p * (1 - p), None: torch.ones_like(p)}[act]
    aE = 0.0 if act is None else (gate_error(zz) + 2 * U) * a.abs()
    sE = 0.0 if act is None else (2 * gate_error(zz) + 4 * U) * p * (1 + (zz * (1 - p)).abs())
    if z is None:
        aE, sE = aE + 1.1 * nE, sE + 1.1 * nE
        yE = aE
    else:
        yE = nE * a.abs() + n.abs() * aE + U * (n * a).abs()
    out = [yE.reshape(T, C)]
    if dy is None:
        return out
    g = dy.double().view_as(x)
    dn, dnE = g * (slope if z is None else a), g.abs() * ((sE if z is None else aE) + 2 * U * (slope if z is None else a).abs())
    k, kE = dn * w, dnE * w.abs() + U * (dn * w).abs()
    m0 = k.mean(-1, keepdim=True) if center else torch.zeros_like(m)
    m0E = kE.mean(-1, keepdim=True) + S * k.abs().mean(-1, keepdim=True) if center else m0
    m1 = (k * xh).mean(-1, keepdim=True)
    m1E = (kE * xh.abs() + k.abs() * xhE).mean(-1, keepdim=True) + S * (k * xh).abs().mean(-1, keepdim=True)
    mag = k.abs() + m0.abs() + (xh * m1).abs()
    dxE = (kE + m0E + xhE * m1.abs() + xh.abs() * m1E + 4 * U * mag) * rstd + rE * mag * rstd
    out.append(dxE.reshape(T, C))
    sums = lambda e, t: (e.sum(0) + (T + 16) * U * t.abs().sum(0))  # noqa: E731
    for e, t, p_ in ((dnE * xh.abs() + dn.abs() * xhE, dn * xh, weight), (dnE, dn, bias)):
        if p_ is not None:
            v = sums(e, t)
            out.append((v if p_.numel() == C else v.sum(0) + G * U * t.abs().sum((0, 1))).reshape(p_.shape))
    if z is not None:
        out.append(((g.abs() * (nE * slope.abs() + n.abs() * (sE + 2 * U * slope.abs())))).reshape(T, C))
    return out


def norm64(x, G, weight, bias, z, act, eps, center):
    """x [T, C].  Differentiable in 64 bits."""
    T, C = x.shape
    x = x.view(T, G, C // G)
    if center:
        x = x - x.mean(-1, keepdim=True)
    n = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    if weight is not None:
        n = n * weight.reshape(-1, C // G)
    if bias is not None:
        n = n + bias.reshape(-1, C // G)
    return (act64(n, act) if z is None else n * act64(z.view_as(n), act)).reshape(T, C)
