"""Attention's fp16 backward pass where gradients are far from 1: dS may pass the type's range, or lie below it, where the results do
not.

Tolerance.  The kernels round every P and dS to fp16, relative 2^-11 at most (normalised, so that the type's range does not count),
independently of each other: in the mean square the error of a sum of terms dS_j k_j is 2^-11 / sqrt(3) of the root T of its terms'
squared norms (of their sum only where they do not cancel).  Then the result is rounded once, which is counted by rounding the exact
one.  With a factor of two, and another 1.8 where single rows are compared, whose errors scatter:
    |got - want| <= 2 |fp16(want) - want| + 2 2^-11 T     (L2 norms)"""
import pytest
import torch

from test_attention_gpu import spans, table

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from semantic_pyramid_for_image_generation_amd import ops
    return ops


def gradients(q, k, v, g, seqs, causal):
    """(gradient, T row by row) of q, k and v, and the largest |dS|, in 64 bits; seqs: (first query, queries, first key, keys)."""
    group, scale = q.shape[1] // k.shape[1], q.shape[2] ** -0.5
    q, k, v, g = (t.double() for t in (q, k, v, g))
    out, terms, worst = [torch.zeros_like(t) for t in (q, k, v)], [torch.zeros_like(t[..., 0]) for t in (q, k, v)], 0.0
    for q0, lq, k0, lk in seqs:
        for h in range(q.shape[1]):
            rows, keys, kh = slice(q0, q0 + lq), slice(k0, k0 + lk), h // group
            Q, G, K, V = q[rows, h], g[rows, h], k[keys, kh], v[keys, kh]
            S = scale * Q @ K.t()
            if causal:
                S = S.masked_fill(torch.arange(lk)[None] > torch.arange(lq)[:, None] + lk - lq, float("-inf"))
            P = torch.softmax(S, dim=-1)
            dP = G @ V.t()
            dS = P * (dP - (P * dP).sum(-1, keepdim=True))
            worst = max(worst, float(dS.abs().max()))
            dS, square = scale * dS, lambda t: t.square().sum(-1)
            out[0][rows, h], terms[0][rows, h] = dS @ K, dS.square() @ square(K)
            out[1][keys, kh] += dS.t() @ Q
            out[2][keys, kh] += P.t() @ G
            terms[1][keys, kh] += dS.square().t() @ square(Q)
            terms[2][keys, kh] += P.square().t() @ square(G)
    return [(o, t.sqrt()) for o, t in zip(out, terms)], worst


def close(got, want, what):
    (want, terms), got = want, got.double().cpu()
    err, allowed = float((got - want).norm()), 2 * float((want.half().double() - want).norm()) + 2 * 2.0 ** -11 * float(terms.norm())
    assert err <= allowed, f"{what}: {err / float(want.norm()):.3g} of the norm, {err / allowed:.3g} of the bound"       # (NaN: false)


def rows_close(got, want, what):
    (want, terms), got = want, got.double().cpu()
    err, rnd = ((t.square().sum(-1).sqrt()) for t in (got - want, want.half().double() - want))
    worst = float((err / (2 * rnd + 1.8 * 2 * 2.0 ** -11 * terms + 1e-30)).max())
    assert worst <= 1.0, f"{what}: {worst:.3g} of the bound"


def run(ops, dev, lens_q, lens_k, q, k, v, g, causal):
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v)]
    o = ops.attention(*leaves, table(lens_q, dev), table(lens_k, dev), causal=causal)
    return torch.autograd.grad(o, leaves, g.to(dev)), *gradients(q, k, v, g, spans(lens_q, lens_k, lens_k), causal)


# queries, keys, heads_q, heads_k, dim: results of 32 keys a workgroup; with at most 8192 rows of keys, and with more
@pytest.mark.parametrize("lens_q,lens_k,heads_q,heads_k,dim", [([256], [4096], 2, 2, 64), ([256], [4096], 8, 4, 64), ([130], [4096], 4, 4, 128),
                                                               ([200], [4096], 4, 4, 32)])
@pytest.mark.parametrize("power", [0, -8, -11, -14])
def test_small_gradients(ops, dev, lens_q, lens_k, heads_q, heads_k, dim, power):
    """dS is some 2^-17 of the type's numbers below g = 2^-8: its subnormals."""
    gen = torch.Generator().manual_seed(dim + heads_k)
    rand = lambda *s: torch.randn(*s, generator=gen)
    q, k, v = (rand(n, h, dim).half() for n, h in ((sum(lens_q), heads_q), (sum(lens_k), heads_k), (sum(lens_k), heads_k)))
    g = (rand(sum(lens_q), heads_q, dim) * 2.0 ** power).half()
    got, want, _ = run(ops, dev, lens_q, lens_k, q, k, v, g, False)
    for what, a, b in zip(("dq", "dk", "dv"), got, want):
        close(a, b, what)


@pytest.mark.parametrize("count,heads", [(1, 1), (1, 2), (40, 4)])          # the last: more than 8192 rows of keys
@pytest.mark.parametrize("dim", [128, 64])
def test_large_gradients(ops, dev, count, heads, dim):
    """|dS| beyond 65504 where every gradient fits: it carries no softmax scale yet, and the sums cancel."""
    gen = torch.Generator().manual_seed(5)
    rand = lambda *s: torch.randn(*s, generator=gen)
    lens = [64] * count
    T = sum(lens)
    q, k, v = (rand(T, heads, dim) for _ in range(3))
    q, k, v, g = (0.5 * q).half(), (0.5 * k).half(), (4 * v).half(), (rand(T, heads, dim) * (5000 if dim == 128 else 7000)).half()
    got, want, worst = run(ops, dev, lens, lens, q, k, v, g, True)
    assert worst > 65504 and all(float(w.abs().max()) < 65000 for w, _ in want)
    for what, a, b in zip(("dq", "dk", "dv"), got, want):
        close(a, b, what)


@pytest.mark.parametrize("heads_k", [1, 16])                                # with at most 8192 rows of keys, and with more
@pytest.mark.parametrize("dim", [16, 64, 128])
@pytest.mark.parametrize("rising", [True, False])
def test_gradients_of_many_sizes(ops, dev, heads_k, dim, rising):
    """Rows whose gradients run from 2^-20 to 2^10, and keys whose probabilities run over e^24: the normalisation moves on the way,
    in either direction.  dq is compared row by row, dk and dv key by key."""
    gen = torch.Generator().manual_seed(dim + heads_k)
    rand = lambda *s: torch.randn(*s, generator=gen)
    lens = [600, 70]
    T = sum(lens)
    ramp = torch.cat([torch.linspace(0, 1, n) if rising else torch.linspace(1, 0, n) for n in lens])[:, None, None]
    q, k, v = (rand(T, h, dim) for h in (heads_k, heads_k, heads_k))
    q, k = 0.3 * q, 0.3 * k
    q[..., 0], k[..., 0] = 4.0, (ramp[..., 0] * 24 - 12) * dim ** 0.5 / 4       # score 24 ramp - 12
    g = rand(T, heads_k, dim) * 2.0 ** (30 * ramp - 20)
    q, k, v, g = (t.half() for t in (q, k, v, g))
    got, want, _ = run(ops, dev, lens, lens, q, k, v, g, False)
    for what, a, b in zip(("dq", "dk", "dv"), got, want):
        rows_close(a, b, what)


def test_probabilities_below_the_type(ops, dev):
    """50000 keys of equal weight: P = 2 10^-5, among fp16's subnormals."""
    gen = torch.Generator().manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=gen).half()
    q, k, v, g = torch.zeros(48, 1, 64, dtype=torch.half), rand(50000, 1, 64), rand(50000, 1, 64), 1000 * rand(48, 1, 64)
    got, want, _ = run(ops, dev, [48], [50000], q, k, v, g, False)
    close(got[0], want[0], "dq")
    close(got[2], want[2], "dv")


def test_zero_and_infinite_gradients(ops, dev):
    """Rows without a gradient give zeros; an infinite one stays in its row of dq."""
    gen = torch.Generator().manual_seed(2)
    rand = lambda *s: torch.randn(*s, generator=gen).half()
    T = 300
    q, k, v, g = rand(T, 2, 64), rand(T, 2, 64), rand(T, 2, 64), rand(T, 2, 64)
    g[100:200] = 0
    g[250, 1, 3] = float("inf")
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v)]
    dq, = torch.autograd.grad(ops.attention(*leaves, table([T], dev)), leaves[:1], g.to(dev))
    assert not dq[100:200].any() and not torch.isfinite(dq[250, 1]).any()
    dq[250, 1] = 0
    assert torch.isfinite(dq).all()
    none = torch.autograd.grad(ops.attention(*leaves, table([T], dev)), leaves, torch.zeros_like(g).to(dev))
    assert not any(t.any() for t in none)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("below", [8.0, 12.0, 17.0])
@pytest.mark.parametrize("queries,heads", [(1, 2), (600, 64)])          # keys split; one pass
def test_outputs_of_the_tail(ops, dev, queries, heads, below, dtype):
    """One key takes nearly all of the weight and has no value; the output is what 20000 keys `below` it (by e^-below each) add up to.
    Their probabilities, 1 / e^17 = 4e-8, are far below fp16's normal numbers.

    The scores are exact (0 and -below, one product), so is the exponential but for the fp32 rounding of its argument (2^-24 of 25)
    and the unit's own (2^-22); a probability is rounded by half a step h of the type, all of them alike, and the result once.  The
    terms of both sums, of probabilities and of products, are alike, too, and may all be rounded the same way: 2^-24 for every
    addition in a row, a tile's 64 keys and then the tiles, for products of 16 bits all keys."""
    keys = 20000
    q = torch.zeros(queries, heads, 32)
    k, v = torch.zeros(keys + 1, 1, 32), torch.rand(keys + 1, 1, 32, generator=torch.Generator().manual_seed(0)) + 0.5
    q[..., 0], k[1:, :, 0], v[0] = 1.0, -below, 0.0
    q, k, v = (t.to(dtype) for t in (q, k, v))
    o = ops.attention(q.to(dev), k.to(dev), v.to(dev), table([queries], dev), table([keys + 1], dev), scale=1.0)
    w = torch.exp(torch.tensor(-below, dtype=torch.float64))
    want = (v[1:, 0].double().sum(dim=0) * w / (1 + keys * w)).expand(queries, heads, 32)
    h = torch.finfo(dtype).eps / 2
    row = keys / 64 + 64
    bound = (2 * h + 2.0 ** -24 * (25 + 4 + row + (row if dtype == torch.float32 else keys))) * want
    worst = float(((o.double().cpu() - want).abs() / bound).max())
    assert worst <= 1.0, worst


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("queries,heads", [(8, 1), (600, 64)])          # keys split; one pass
def test_rows_beside_a_rising_one(ops, dev, queries, heads, dtype):
    """Rows whose scores are all 12800 next to rows whose scores rise from tile to tile: the former's sums must not move with the
    latter's reference.  V is 0 in the first half of the keys and 1 in the second: the outputs are 1/2 and 1.  Scores are exact.  In
    16 bits the reference is a rounded product, so that all probabilities of a row are off from a power of two alike, rounded alike
    by at most half a step h for the second product, and added unrounded; the result is rounded once.  In fp32 they are 1 (and 0)
    and the sums exact."""
    keys = 16384
    q, k, v = torch.zeros(queries, heads, 32), torch.zeros(keys, 1, 32), torch.zeros(keys, 1, 32)
    q[0::2, :, 0], q[1::2, :, 1] = 128.0, 1.0
    k[:, 0, 0], k[:, 0, 1] = 100.0, (torch.arange(keys) // 64 * 8).float()
    v[keys // 2:] = 1.0
    o = ops.attention(*(t.to(dtype).to(dev) for t in (q, k, v)), table([queries], dev), table([keys], dev), scale=0.7)
    h = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    for got, want in ((o[0::2], 0.5), (o[1::2], 1.0)):
        worst = float((got.double() - want).abs().max())
        assert worst <= 2 * h * want, (want, worst)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("run", [32, 64])                               # other maxima in the waves of a workgroup; in its splits
@pytest.mark.parametrize("scale", [1.051, 0.985, 1.03])
def test_large_scores_joined_over_splits(ops, dev, run, scale, dtype):
    """One query, scores of 100000 and 99999 (times scale) by turns of `run` keys: parts whose maxima differ are joined by the powers
    of two that their probabilities were taken with.  Of those a rounded product of 2^17 is off by 2^-8 of a power, alike in all
    parts.  V is 1 at the larger scores: the output is 1 / (1 + e^-scale); rounded are P and the result (h each), and scale log2(e),
    2^-23 of it, and the unit's exponential, 2^-22."""
    keys = 2048
    q, k, v = torch.zeros(1, 1, 32), torch.zeros(keys, 1, 32), torch.zeros(keys, 1, 32)
    low = torch.arange(keys) // run % 2
    q[..., 0], q[..., 1], k[..., 0], k[:, 0, 1] = 250.0, 1.0, 400.0, -low.float()
    v[low == 0] = 1.0
    o = ops.attention(*(t.to(dtype).to(dev) for t in (q, k, v)), table([1], dev), table([keys], dev), scale=scale)
    want, h = 1 / (1 + torch.exp(torch.tensor(-scale, dtype=torch.float64)).item()), torch.finfo(dtype).eps / 2
    worst = float((o.double() - want).abs().max())
    assert worst <= (2 * h + 2.0 ** -20) * want, (worst / want, h)
