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


def gradients64(lens, tensors, states, dy, dfinal, scale=8.0):
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


def act64(v, name):
    return {"silu": torch.nn.functional.silu, "sigmoid": torch.sigmoid, None: lambda t: t}[name](v)


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
