"""The token operators' definitions in 64 bits on the CPU, with bounds of the fp32 kernels' rounding errors beside them."""
import math

import torch

U = 2.0 ** -24                              # half a step of fp32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def frequencies(sections, base, shared):
    pairs = sum(sections)
    if shared:
        return [base ** (-(j / pairs)) for j in range(pairs)]
    return [base ** (-(i / n)) for n in sections for i in range(n)]


def pair_index(pairs, interleaved):
    j = torch.arange(pairs)
    return (2 * j, 2 * j + 1) if interleaved else (j, j + pairs)


def rotate(x, positions, sections, base, interleaved, shared, back=False):
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)])
    ang = positions.double()[:, axis] * torch.tensor(frequencies(sections, base, shared), dtype=torch.float64)
    c, s = ang.cos()[:, None], ang.sin()[:, None] * (-1 if back else 1)
    ia, ib = pair_index(sum(sections), interleaved)
    y = x.clone()
    y[..., ia] = x[..., ia] * c - x[..., ib] * s
    y[..., ib] = x[..., ia] * s + x[..., ib] * c
    return y


def qk_norm_rope(x, w, g, positions, sections, base, interleaved, shared, eps):
    """(y, dx, dw) and their error bounds of one of queries / keys; x, g [tokens, heads, dim] of any type, w None: no norm."""
    step = half_step(x.dtype)
    x, g = x.double(), g.double()
    rot = dict(positions=positions, sections=sections, base=base, interleaved=interleaved, shared=shared)
    gr = rotate(g, back=True, **rot)
    top = lambda t: t.abs().amax(dim=-1, keepdim=True)
    if w is None:
        y, dx, dw = rotate(x, **rot), gr, None
        # sine and cosine are off by at most 2 U, a product of them by 3 U, two of them are added: 8 U of |a| + |b|
        return (y, 8 * U * 2 * top(x) + 2 * step * y.abs()), (dx, 8 * U * 2 * top(g) + 2 * step * dx.abs()), None
    w = w.double()
    r = (x.square().mean(dim=-1, keepdim=True) + eps).rsqrt()
    xhat = x * r
    y = rotate(xhat * w, **rot)
    m = (gr * w * xhat).mean(dim=-1, keepdim=True)
    dx = r * (gr * w - xhat * m)
    dw = (gr * xhat).sum(dim=(0, 1))
    # sum of squares: at most 32 additions in a lane and 6 across lanes, halved by the root; root, quotient and the products
    # with r and w: 5 more; rotation 8 -> below 32 U of |a| + |b| <= 2 max
    ey = 32 * U * 2 * top(xhat * w) + 2 * step * y.abs()
    am = (gr * w * xhat).abs().mean(dim=-1, keepdim=True)
    ed = r * (2 * 32 * U * 2 * top(g) * top(w[None, None]) + 2 * 64 * U * top(xhat) * (am + 2 * top(g) * top(w[None, None]) / 2)) + \
        2 * step * dx.abs()
    # a term of dw is off by 32 U of 2 max|g| |xhat|, the sums by U of the absolute sum for each of at most 160 additions
    # in a row (rows of a lane, lanes, waves, workgroups)
    tw = (2 * top(g) * xhat.abs()).sum(dim=(0, 1))
    return (y, ey), (dx, ed), (dw, 192 * U * tw + 2 * step * dw.abs())


def philox4x32(counter, key, rounds=10):
    """Salmon et al. 2011, on Python integers."""
    c, (k0, k1) = list(counter), key
    for _ in range(rounds):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(p1 >> 32) ^ c[1] ^ k0, p1 & 0xFFFFFFFF, (p0 >> 32) ^ c[3] ^ k1, p0 & 0xFFFFFFFF]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def dropout_gain(n, p, seed, offset):
    """The factor of each of n elements: 0 or 65536 / threshold."""
    t = int(math.floor((1.0 - p) * 65536.0 + 0.5))
    m = 0xFFFFFFFF
    fields = []
    for b in range((n + 7) // 8):
        for word in philox4x32((b & m, b >> 32, offset & m, (offset >> 32) & m), (seed & m, (seed >> 32) & m)):
            fields += [word & 0xFFFF, word >> 16]
    f = torch.tensor(fields[:n], dtype=torch.int64)
    return (f < t).double() * (65536.0 / t if t else 0.0)
