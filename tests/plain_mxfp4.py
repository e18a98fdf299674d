"""MXFP4 and the products with it in 64 bits, from the format's definition, with bounds on what 32-bit sums of bfloat16 rows may be off.

A product of k terms whose sums are 32-bit is off by at most k * 2^-23 of the sum of the terms' sizes (half of a step a rounding, twice that
where an addition cuts instead of rounding); a result rounded to bfloat16 by 2^-8 of itself more."""

import torch

LEVELS = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def rounded(w):
    """The values (64-bit, on the CPU) that the blocks of 32 along the last dimension are rounded to."""
    w = w.detach().cpu().double()
    out = torch.zeros_like(w)
    for k in range(0, w.shape[-1], 32):
        v = w[..., k:k + 32]
        top = v.abs().amax(-1, keepdim=True)
        bad = ~torch.isfinite(v).all(-1, keepdim=True)
        exponent = torch.frexp(torch.where(bad | (top == 0), torch.ones_like(top), top))[1] - 3
        scale = torch.ldexp(torch.ones_like(top), exponent.clamp_min(-127))
        d = (v.abs() / scale)[..., None] - LEVELS
        near = d.abs().amin(-1, keepdim=True)
        even = torch.where(d.abs() == near, torch.tensor([0, 9, 1, 10, 2, 11, 3, 12]), 99).argmin(-1)       # of two, the even code
        out[..., k:k + 32] = torch.where(bad, torch.nan, torch.sign(v) * LEVELS[even] * scale)
    return out


def product(x, w):
    """(x w^T, the bound on a 32-bit sum) in 64 bits."""
    x, w = x.cpu().double(), w.cpu().double()
    return x @ w.T, x.shape[-1] * 2.0 ** -23 * (x.abs() @ w.abs().T)


def activation(z, act):
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z / 2 ** 0.5))
    return {"relu2": lambda: torch.relu(z) ** 2, "identity": lambda: z,
            "gelu_tanh": lambda: 0.5 * z * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3)))}[act]()


def activated(z, off, act):
    """(act(z), its bound): the slope is at most 1.13 (relu2: 2 (|z| + off)), and the function itself is 32-bit."""
    a = activation(z, act)
    slope = 2 * (z.abs() + off) if act == "relu2" else 1.13
    return a, slope * off + 2.0 ** -20 * a.abs() + 1e-30


def gated(x, gate, up, act, bias=None):
    g, g_off = product(x, gate)
    u, u_off = product(x, up)
    if bias is not None:
        b = bias.cpu().double()
        g, u = g + b[:len(b) // 2], u + b[len(b) // 2:]
        g_off, u_off = g_off + 2.0 ** -24 * g.abs(), u_off + 2.0 ** -24 * u.abs()
    a, off = activated(g, g_off, act)
    return a * u, off * u.abs() + (a.abs() + off) * u_off + 2.0 ** -23 * (a * u).abs()


def experts(x, ids, wts, first, down, act, weigh="output"):
    """(out, bound): `first` [E, 1 or 2, inter, hidden], `down` [E, hidden, inter], both 64-bit values."""
    rows, top = ids.shape
    out = torch.zeros(rows, down.shape[1], dtype=torch.float64)
    off = torch.zeros_like(out)
    for r in range(rows):
        for s in range(top):
            e, w = int(ids[r, s]), float(wts[r, s])
            if not 0 <= e < down.shape[0]:
                continue
            xr = x[r:r + 1].cpu().double()
            before = w if weigh == "input" else 1.0
            if first.shape[1] == 2:
                a, a_off = gated(xr * before, first[e, 0], first[e, 1], act)
            else:
                z, z_off = product(xr * before, first[e, 0])
                a, a_off = activated(z, z_off, act)
            after = 1.0 if weigh == "input" else w
            a, a_off = a * after, a_off * abs(after)
            a_off = a_off + 2.0 ** -8 * (a.abs() + a_off)                      # rounded to bfloat16 on the way
            y, y_off = product(a, down[e])
            out[r] += y[0]
            off[r] += (top * y_off + a_off @ down[e].abs().T)[0]                 # (one sum over all of the row's experts)
    return out, off


def hold(got, want, off):
    """got (bfloat16 or 32-bit) within `off` of want and one rounding to its own type."""
    got, limit = got.detach().cpu().double(), off * (1 + ROUND[got.dtype]) + ROUND[got.dtype] * want.abs() + 1e-30
    over = (got - want).abs() > limit
    assert torch.isfinite(got).all() and not over.any(), \
        f"{int(over.sum())} of {over.numel()} off, the worst by {float(((got - want).abs() / limit).max()):.3g} of the bound"
