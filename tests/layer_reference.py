"""Plain 64-bit forms of the layer operators, and the bound their kernels are held to.

A result is off by the rounding of its own type, u |y|, and by the fp32 arithmetic in front of it, c 2^-24 times the sum of
the magnitudes of the terms that were added (``mag``): every reference returns both."""

import torch

UNIT = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 0.0, torch.float32: 0.0}  # half the distance of subnormals


def check(got, want, mag, f32):
    """|got - want| <= u |want| + f32 mag, element by element; ``f32``: the relative error of the fp32 arithmetic."""
    got, dt = got.double().cpu(), got.dtype
    want, mag = want.double().cpu(), mag.double().cpu()
    assert got.shape == want.shape
    bound = UNIT[dt] * (want.abs() + f32 * mag) + f32 * mag + TINY[dt]
    over = (got - want).abs() - bound
    assert not torch.isnan(got).any()
    assert float(over.max()) <= 0 if over.numel() else True, f"{float(over.max()):.3e} over the bound, |error| up to {float((got - want).abs().max()):.3e}"


def silu(x):
    return x * torch.sigmoid(x)


def conv(x, w, bias, initial, lengths, act):
    x, w = x.double().cpu(), w.double().cpu()
    B, T, D = x.shape
    W = w.shape[1]
    bias = torch.zeros(D, dtype=torch.float64) if bias is None else bias.double().cpu()
    y, mag, state = torch.zeros_like(x), torch.zeros_like(x), torch.zeros(B, W - 1, D, dtype=torch.float64)
    for b in range(B):
        n = T if lengths is None else min(max(int(lengths[b]), 0), T)
        line = torch.zeros(W - 1 + n, D, dtype=torch.float64)
        if initial is not None:
            line[:W - 1] = initial[b].double().cpu()
        line[W - 1:] = x[b, :n]
        for t in range(n):
            s = bias + (line[t:t + W].t() * w).sum(1)
            m = bias.abs() + (line[t:t + W].t() * w).abs().sum(1)
            y[b, t] = silu(s) if act else s
            mag[b, t] = m * 1.1 if act else m  # |silu'| <= 1.1
        state[b] = line[n:]
    return y, mag, state


def softplus(x):
    return torch.logaddexp(x, torch.zeros_like(x))


def scan(u, dt, A, B, C, D, z, bias, soft, limit, initial, lengths):
    u, dt, A, B, C = (t.double().cpu() for t in (u, dt, A, B, C))
    b, T, d = u.shape
    G, N = B.shape[2:]
    dt = dt + (0 if bias is None else bias.double().cpu())
    dt = (softplus(dt) if soft else dt).clamp(*limit)
    B, C = B.repeat_interleave(d // G, 2), C.repeat_interleave(d // G, 2)
    h = torch.zeros(b, d, N, dtype=torch.float64) if initial is None else initial.double().cpu()
    hm = h.abs()
    y, mag = torch.zeros_like(u), torch.zeros_like(u)
    n = torch.full((b,), T) if lengths is None else lengths.cpu().clamp(0, T)
    for t in range(T):
        on = (n > t)[:, None, None]
        a = torch.exp(dt[:, t, :, None] * A)
        x = (dt[:, t] * u[:, t])[..., None] * B[:, t]
        h, hm = torch.where(on, a * h + x, h), torch.where(on, a * hm + x.abs(), hm)
        yt, mt = (C[:, t] * h).sum(-1), (C[:, t].abs() * hm).sum(-1)
        if D is not None:
            yt, mt = yt + D.double().cpu() * u[:, t], mt + (D.double().cpu() * u[:, t]).abs()
        if z is not None:
            g = silu(z[:, t].double().cpu())
            yt, mt = yt * g, mt * g.abs()
        y[:, t], mag[:, t] = torch.where(on[..., 0], yt, 0.0), torch.where(on[..., 0], mt, 0.0)
    return y, mag, h, hm


def scan_step(state, u, dt, A, B, C, D, z, bias, soft, limit):
    """state [b, .., N]: the rows of the sequences. Channel form, or head form with u [b, H, P]."""
    state, u, dt, A, B, C = (t.double().cpu() for t in (state, u, dt, A, B, C))
    heads = u.dim() == 3
    dt = dt + (0 if bias is None else bias.double().cpu())
    dt = (softplus(dt) if soft else dt).clamp(*limit)
    rep = u.shape[1] // B.shape[1]
    B, C = B.repeat_interleave(rep, 1), C.repeat_interleave(rep, 1)
    if heads:
        dt, A, B, C = dt[..., None], A[:, None, None], B[:, :, None], C[:, :, None]
        D = None if D is None else D.double().cpu() if D.dim() == 2 else D.double().cpu()[:, None]
    elif D is not None:
        D = D.double().cpu()
    x = (dt * u)[..., None] * B
    a = torch.exp(dt[..., None] * A)
    h, hm = a * state + x, a * state.abs() + x.abs()
    y, mag = (h * C).sum(-1), (hm * C.abs()).sum(-1)
    if D is not None:
        y, mag = y + D * u, mag + (D * u).abs()
    if z is not None:
        g = silu(z.double().cpu())
        y, mag = y * g, mag * g.abs()
    return y, mag, h, hm


def norm(v, eps):
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)


def codes(v):
    """Codes before they are rounded, and their scale."""
    scale = v.abs().amax(-1, keepdim=True) / 127
    return torch.where(scale > 0, v / torch.where(scale > 0, scale, 1.0), 0.0), scale[..., 0]


def check_codes(got, scale, want):
    """Every code is the value over its scale, rounded to nearest: at most half a step off, and as much more as fp32 values
    and scales carry (a value of 127 steps times 16 roundings)."""
    y, s = codes(want)
    assert (got.double().cpu() - y).abs().max() <= 0.5 + 127 * 16 * 2.0**-24
    assert ((scale.double().cpu() - s).abs() <= 16 * 2.0**-24 * s).all()
