"""The definitions of the operators around the prefill, token by token in 64 bits, each with a bound of the error that fp32
arithmetic may leave (u = 2^-24 is half a step of fp32, rounding to the output's type comes on top in `assert_within`)."""
import torch

DEV = "cuda:0"
U = 2.0 ** -24


def assert_within(got, want, bound, what):
    """|got - want| <= bound + half a step of got's type, element by element."""
    info = torch.finfo(got.dtype)
    got, want, bound = got.double().cpu(), want.double().cpu(), bound.double().cpu()
    half = info.eps / 2 * want.abs() + info.tiny * info.eps
    if info.bits == 32:
        half = torch.zeros_like(half)                       # the bounds count fp32's own roundings
    worst = ((got - want).abs() / (bound + half).clamp(min=1e-300)).nan_to_num(nan=float("inf"))
    assert got.shape == want.shape and (worst.numel() == 0 or worst.max() <= 1.0), f"{what}: {worst.max():.3g} times the allowed error"


def silu64(x):
    return x * torch.sigmoid(x)


def conv64(x, weight, bias, history, activation):
    """One sequence: x [L, C], history [W - 1, C].  Returns y, bound, new history (fp64).  W products and sums, each off by u of the
    sum of the magnitudes; |silu'| <= 1.1; the exponential and quotient of the activation to 2^-18 in its range of arguments."""
    x, weight, history = x.double(), weight.double(), history.double()
    W, full = weight.shape[1], torch.cat([history, x])
    taps = [full[j:j + x.shape[0]] * weight[:, j] for j in range(W)]
    y = sum(taps) + (bias.double() if bias is not None else 0.0)
    bound = (W + 2) * U * (sum(t.abs() for t in taps) + (bias.double().abs() if bias is not None else 0.0))
    if activation == "silu":
        y, bound = silu64(y), 1.1 * bound + 2.0 ** -18 * silu64(y).abs()
    return y, bound, full[full.shape[0] - (W - 1):]


def scan64(u, dt, A, B, C, D, z, dt_bias, h, softplus):
    """One sequence: u, dt, z [L, Dm], B, C [L, G, Ns], h [Dm, Ns].  Returns y, bound, h, bound of h.  The running bound: the decay
    exp(s A) is off by 2^-21 + |s A| eps_s relatively (eps_s: the error of s, the sum x = dt + bias rounded, then the softplus), the
    term s u B by eps_s + 4 u, each sum by u."""
    u, dt, A, B, C, h = (t.double() for t in (u, dt, A, B, C, h))
    L, Dm = u.shape
    per = Dm // B.shape[1]
    x = dt + (dt_bias.double() if dt_bias is not None else 0.0)
    s = torch.nn.functional.softplus(x, threshold=200.0) if softplus else x
    eps = (8 + x.abs() + (dt_bias.double().abs() if dt_bias is not None else 0.0)) * 2 * U
    y, bound, E = torch.empty_like(u), torch.empty_like(u), torch.zeros_like(h)
    mag = h.abs()
    for t in range(L):
        Bt, Ct = B[t].repeat_interleave(per, 0), C[t].repeat_interleave(per, 0)
        a = torch.exp(s[t][:, None] * A)
        off = 2.0 ** -21 + (s[t][:, None] * A).abs() * (eps[t][:, None] + 3 * U)
        b = (s[t] * u[t])[:, None] * Bt
        E = a * (E + off * mag) + b.abs() * (eps[t][:, None] + 4 * U)
        h, mag = a * h + b, a * mag + b.abs()
        E = E + 2 * U * mag
        skip = D.double() * u[t] if D is not None else 0.0
        y[t] = (Ct * h).sum(-1) + skip
        bound[t] = (Ct.abs() * E).sum(-1) + (A.shape[1] + 2) * U * ((Ct.abs() * mag).sum(-1) + (skip.abs() if D is not None else 0.0))
    if z is not None:
        gate = silu64(z.double())
        y, bound = y * gate, bound * gate.abs() + 2.0 ** -18 * (y * gate).abs()
    return y, bound, h, E


def kda_step64(q, k, v, g, beta, A_log, dt_bias, scale, S, raw):
    """One token of one sequence, all heads: S [H, K, V].  Returns o, bound, S, bound of S.  Dots over 128 keys: 128 u of the sum of
    the magnitudes; decay and normalised operands to 2^-19 (a chain of an exponential, a sigmoid and an exponential, |log a| <= 5 raw)."""
    q, k, v, g, beta, S = (t.double() for t in (q, k, v, g, beta, S))
    if raw:
        q, k = (torch.nn.functional.normalize(t, dim=-1, eps=1e-6) for t in (q, k))
        g = -5.0 * torch.sigmoid(A_log.double().exp()[:, None] * (g + dt_bias.double().view(g.shape)))
        beta = torch.sigmoid(beta)
    S = S * g.exp()[:, :, None]
    e = 2.0 ** -19 + (g.abs() * 4 * U).amax()
    kS, kM = torch.einsum("hk,hkv->hv", k, S), torch.einsum("hk,hkv->hv", k.abs(), S.abs())
    r = beta[:, None] * (v - kS)
    rE = beta[:, None] * ((128 * U + 2 * e) * kM + 4 * U * v.abs()) + 4 * e * r.abs()
    new = S + torch.einsum("hk,hv->hkv", k, r)
    E = (e + 2 * U) * S.abs() + k.abs()[:, :, None] * (rE + (2 * e) * r.abs())[:, None, :] + 2 * U * new.abs()
    o = scale * torch.einsum("hk,hkv->hv", q, new)
    qM = torch.einsum("hk,hkv->hv", q.abs(), S.abs()) + (q.abs() * k.abs()).sum(-1)[:, None] * r.abs()
    oE = abs(scale) * ((130 * U + 3 * e) * qM + torch.einsum("hk,hkv->hv", q.abs(), E))
    return o, oE, new, E


def cu_of(lens, dtype=torch.int64):
    return torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=dtype, device=DEV)


def randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dtype)


def generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)
