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


def attention(q, k, v, g, seqs, causal, scale):
    """(o, dq, dk, dv), each with its error bound, of packed sequences; seqs: (first query, queries, first key, keys).

    u = U, h = half a step of the type.  A score is a sum of dim products: off by dim u sum|q||k|; the exponent's fma, the row
    maximum and the exponential add a few u of its size, so a probability is off by eps_p relative, and by h once it is rounded
    for the second product (fp16: by 2^-25 absolute where it is subnormal).  Sums over n terms add n u of the absolute sum."""
    h = half_step(q.dtype)
    sub = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    if q.dtype == torch.float32:
        h = U
    group = q.shape[1] // k.shape[1]
    dim = q.shape[2]
    q, k, v, g = (t.double() for t in (q, k, v, g))
    out = [torch.zeros_like(t) for t in (q, q, k, v)]
    err = [torch.zeros_like(t) for t in (q, q, k, v)]
    for q0, lq, k0, lk in seqs:
        if lq == 0 or lk == 0:
            continue
        for hd in range(q.shape[1]):
            kh = hd // group
            Q, G, K, V = q[q0:q0 + lq, hd], g[q0:q0 + lq, hd], k[k0:k0 + lk, kh], v[k0:k0 + lk, kh]
            S = scale * Q @ K.t()
            seen = torch.ones(lq, lk, dtype=torch.bool)
            if causal:
                seen = torch.arange(lk)[None] <= torch.arange(lq)[:, None] + (lk - lq)
            S = S.masked_fill(~seen, float("-inf"))
            P = torch.softmax(S, dim=-1).nan_to_num(0.0)
            P = torch.where(seen, P, torch.zeros_like(P))
            size = torch.where(seen, S, torch.zeros_like(S)).abs().amax(dim=-1, keepdim=True)
            eps_p = scale * dim * U * (Q.abs() @ K.abs().t()).amax(dim=-1, keepdim=True) + 8 * U * (1 + 1.5 * size)
            n = lk + lk // 16 + 16
            o = P @ V
            PV = P @ V.abs()
            eo = (2 * eps_p + h + 2 * n * U) * PV + (2 * n * U + 2 * h) * o.abs() + sub * V.abs().sum(dim=0)
            dP = G @ V.t()
            delta = (G * o).sum(dim=-1, keepdim=True)
            dS = P * (dP - delta)
            e_dp = dim * U * (G.abs() @ V.abs().t())
            e_de = (G.abs() * eo).sum(dim=-1, keepdim=True) + dim * U * (G * o).abs().sum(dim=-1, keepdim=True)
            e_p = 2 * eps_p + 2 * n * U
            e_ds = P * (e_dp + e_de) + dS.abs() * (e_p + 4 * U + h) + sub * seen
            e_pv = P * (e_p + h) + sub * seen
            m = lq * group + 16
            out[0][q0:q0 + lq, hd] = o
            err[0][q0:q0 + lq, hd] = eo
            out[1][q0:q0 + lq, hd] = scale * dS @ K
            err[1][q0:q0 + lq, hd] = scale * (e_ds @ K.abs() + n * U * dS.abs() @ K.abs()) + 2 * h * out[1][q0:q0 + lq, hd].abs()
            out[2][k0:k0 + lk, kh] += scale * dS.t() @ Q
            err[2][k0:k0 + lk, kh] += scale * (e_ds.t() @ Q.abs() + m * U * dS.t().abs() @ Q.abs())
            out[3][k0:k0 + lk, kh] += P.t() @ G
            err[3][k0:k0 + lk, kh] += e_pv.t() @ G.abs() + m * U * P.t() @ G.abs()
    err[2] += 2 * h * out[2].abs()
    err[3] += 2 * h * out[3].abs()
    # what no formula covers: results next to the smallest numbers of the type
    return [(o, e + 1e-37 + sub) for o, e in zip(out, err)]
