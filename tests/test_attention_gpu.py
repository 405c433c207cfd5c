"""Packed attention on the GPU against its definition in 64 bits (token_oracle.py derives the tolerances)."""
import pytest
import torch

import token_oracle as oracle
from test_token_ops_gpu import TYPES, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from semantic_pyramid_for_image_generation_amd import ops
    return ops


def table(ns, dev):
    return torch.tensor([0] + list(ns), dtype=torch.int64).cumsum(0).to(torch.int32).to(dev)


def spans(lens_q, slots, lens_k):
    out, a, b = [], 0, 0
    for lq, cap, lk in zip(lens_q, slots, lens_k):
        out.append((a, lq, b, lk))
        a, b = a + lq, b + cap
    return out


# queries, key slots, keys in use, rows behind the last sequence, heads_q, heads_k, dim, causal
CASES = {
    "one": ([1], [1], [1], 0, 1, 1, 8, False),
    "one_row": ([1], [70], [70], 0, 4, 2, 32, True),
    "tile": ([128], [128], [128], 0, 2, 1, 64, False),
    "odd_causal": ([65, 1, 0, 130], [65, 1, 0, 130], [65, 1, 0, 130], 0, 4, 4, 64, True),
    "odd_full": ([33, 129, 2], [33, 129, 2], [33, 129, 2], 3, 3, 1, 80, False),
    "wide": ([200], [200], [200], 0, 2, 2, 128, True),
    "prefix": ([5, 40, 3], [300, 64, 3], [300, 64, 3], 0, 8, 2, 128, True),          # queries behind cached keys
    "empty_rows": ([50, 7, 90], [20, 0, 200], [20, 0, 61], 9, 2, 1, 32, True),       # more queries than keys: rows see none
    "slots": ([1, 1, 3], [96, 96, 96], [17, 0, 96], 0, 10, 2, 64, True),             # cache slots, partly used
    "no_keys": ([4, 5], [0, 0], [0, 0], 0, 2, 2, 16, False),
    "group": ([70], [190], [190], 0, 40, 1, 16, True),
    "token": ([1, 1, 1, 1], [700, 700, 700, 700], [700, 1, 0, 333], 0, 8, 1, 128, True),     # new tokens, split keys
    "tokens_many_heads": ([2, 1], [150, 40], [150, 33], 2, 70, 1, 48, True),                 # a group wider than a tile
    "many": ([140] * 10 + [3], [140] * 10 + [3], [140] * 10 + [3], 0, 28, 4, 32, True),      # enough tiles for the one-pass kernel
    "many_full": ([300, 290, 1], [300, 290, 77], [300, 290, 70], 5, 64, 64, 16, False),
    "heads8": ([150, 20], [150, 20], [150, 20], 0, 16, 8, 24, True),
}


def make(case, dtype, seed=0):
    lq, slots, lk, behind, hq, hk, dim, causal = case
    gen = torch.Generator().manual_seed(seed + sum(lq) * 7 + dim)
    tq, tk = sum(lq) + behind, sum(slots) + behind
    rand = lambda *s: torch.randn(*s, generator=gen).to(dtype)
    return rand(tq, hq, dim), rand(tk, hk, dim), rand(tk, hk, dim), rand(tq, hq, dim)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", list(CASES))
def test_attention(ops, dev, name, dtype):
    case = CASES[name]
    lq, slots, lk, behind, hq, hk, dim, causal = case
    q, k, v, g = make(case, dtype)
    scale = 0.3 if name == "wide" else dim ** -0.5
    want = oracle.attention(q, k, v, g, spans(lq, slots, lk), causal, scale)
    k2, v2 = k.clone(), v.clone()                    # what no sequence uses holds NaN: it must not be read
    used = torch.zeros(k.shape[0], dtype=torch.bool)
    for _, _, k0, n in spans(lq, slots, lk):
        used[k0:k0 + n] = True
    k2[~used], v2[~used] = float("nan"), float("nan")
    q2, g2 = q.clone(), g.clone()
    q2[sum(lq):] = float("nan")
    g2[sum(lq):] = float("nan")
    qd, kd, vd = (t.to(dev).requires_grad_() for t in (q2, k2, v2))
    len_k = None if lk == slots else torch.tensor(lk, dtype=torch.int32, device=dev)
    kw = dict(causal=causal, scale=None if name != "wide" else scale)
    o = ops.attention(qd, kd, vd, table(lq, dev), table(slots, dev), len_k, **kw)
    grads = torch.autograd.grad(o, [qd, kd, vd], g2.to(dev))
    for what, got, (w, e) in zip(("o", "dq", "dk", "dv"), [o.detach(), *grads], want):
        assert got.dtype == dtype and got.is_contiguous()
        within(got, w, e, what)
    assert not o[sum(lq):].any() and not grads[0][sum(lq):].any() and not grads[1].cpu()[~used].any() and not grads[2].cpu()[~used].any()
    with torch.no_grad():                             # without the statistics for a backward pass, and once more: the same bits
        assert torch.equal(o, ops.attention(qd, kd, vd, table(lq, dev), table(slots, dev), len_k, **kw))
    again = torch.autograd.grad(ops.attention(qd, kd, vd, table(lq, dev), table(slots, dev), len_k, **kw), [qd, kd, vd], g2.to(dev))
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_views(ops, dev, dtype):
    """Views of one projection, heads-first memory, unaligned and expanded tensors: the bits of dense copies."""
    gen = torch.Generator().manual_seed(1)
    T, dim = 77, 32
    cu = table([30, 47], dev)
    big = torch.randn(T, 6, 3 * dim + 8, generator=gen).to(dtype).to(dev)
    views = [big[:, :, :dim], big[:, :, 1:dim + 1], big[:, :, 0:2 * dim:2], big[:, :, :dim].transpose(0, 1).contiguous().transpose(0, 1),
             big[:1, :, :dim].expand(T, 6, dim), big[:, :1, :dim].expand(T, 6, dim)]
    for x in views:
        q, k, v = x, x[:, 2:4], x[:, 4:6]
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        dense = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_() for t in (q, k, v)]
        a = ops.attention(*leaves, cu, causal=True)
        b = ops.attention(*dense, cu, causal=True)
        assert torch.equal(a, b)
        g = torch.randn(T, 12, dim, generator=gen).to(dtype).to(dev)[:, ::2]           # a strided gradient
        for s, t in zip(torch.autograd.grad(a, leaves, g), torch.autograd.grad(b, dense, g)):
            assert torch.equal(s, t)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_dimensions_of_size_one(ops, dev, dtype):
    """Their strides mean nothing: one row, one head, from views whose strides there are odd or zero."""
    x = torch.randn(5, 3, 33, device=dev).to(dtype)
    cu1, cu5 = table([1], dev), table([5], dev)
    one_row = torch.as_strided(x.contiguous()[:1, :, :32].clone(), (1, 3, 32), (3, 32, 1))
    one_head = torch.as_strided(x[:, :1, :32].contiguous(), (5, 1, 32), (32, 5, 1))
    for q, cu in ((one_row, cu1), (one_head, cu5)):
        o = ops.attention(q, q, q, cu, causal=True)
        assert torch.equal(o, ops.attention(*[q.clone(memory_format=torch.contiguous_format)] * 3, cu, causal=True))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_large_scores(ops, dev, dtype):
    """Scores in the hundreds: the running maximum keeps every exponential in range."""
    gen = torch.Generator().manual_seed(2)
    q = (20 * torch.randn(70, 2, 64, generator=gen)).to(dtype)
    k = (20 * torch.randn(200, 2, 64, generator=gen)).to(dtype)
    v = torch.randn(200, 2, 64, generator=gen).to(dtype)
    g = torch.randn(70, 2, 64, generator=gen).to(dtype)
    (w, e), *_ = oracle.attention(q, k, v, g, [(0, 70, 0, 200)], True, 0.125)
    o = ops.attention(q.to(dev), k.to(dev), v.to(dev), table([70], dev), table([200], dev), causal=True)
    within(o, w, e, "o")


def test_attention_bad_tables(ops, dev):
    """Entries outside the tensors and falling ones are clamped: nothing outside is touched and the call ends."""
    q = torch.randn(40, 2, 16, device=dev)
    for bad in ([0, 1000, 2000], [0, -5, 40], [7, 20, 10], [0, 40, 40], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1]):
        t = torch.tensor(bad, dtype=torch.int32, device=dev)
        o = ops.attention(q, q, q, t, causal=True)
        assert o.shape == q.shape
    o = ops.attention(q, q, q, table([40], dev), len_k=torch.tensor([-3], dtype=torch.int32, device=dev))
    assert not o.any()
    full = ops.attention(q, q, q, table([40], dev))
    assert torch.equal(full, ops.attention(q, q, q, table([40], dev), len_k=torch.tensor([10 ** 9], dtype=torch.int32, device=dev)))


def test_attention_empty(ops, dev):
    q, e = torch.randn(3, 2, 16, device=dev), torch.zeros(0, 2, 16, device=dev)
    cu0, cu3 = table([0], dev), table([3], dev)
    assert not ops.attention(q, e, e, cu3, cu0).any()
    assert ops.attention(e, q, q, cu0, cu3).shape == (0, 2, 16)
    assert not ops.attention(q, q, q, torch.zeros(1, dtype=torch.int32, device=dev)).any()        # no sequence at all
    leaves = [t.clone().requires_grad_() for t in (e, q, q)]
    grads = torch.autograd.grad(ops.attention(*leaves, cu0, cu3).sum(), leaves)
    assert not grads[1].any() and not grads[2].any()
    leaves = [t.clone().requires_grad_() for t in (q, e, e)]
    grads = torch.autograd.grad(ops.attention(*leaves, cu3, cu0).sum(), leaves)
    assert not grads[0].any()


def test_attention_differences(ops, dev):
    """Gradients against differences of the forward: fp32, step d along a random direction; the quotient is off by the third
    derivative's d^2 (below 1e-4 here) and by the forward's rounding over d."""
    gen = torch.Generator().manual_seed(4)
    lens = [37, 5]
    x = [torch.randn(42, h, 32, generator=gen).to(dev) for h in (4, 2, 2)]
    g = torch.randn(42, 4, 32, generator=gen).to(dev)
    leaves = [t.clone().requires_grad_() for t in x]
    grads = torch.autograd.grad(ops.attention(*leaves, table(lens, dev), causal=True), leaves, g)
    d = 2.0 ** -6
    for i in range(3):
        way = torch.randn(x[i].shape, generator=gen).to(dev)
        way /= way.norm()
        f = [(ops.attention(*[t + (s * d * way if j == i else 0) for j, t in enumerate(x)], table(lens, dev), causal=True).double()
              * g.double()).sum() for s in (1, -1)]
        quotient, exact = float((f[0] - f[1]) / (2 * d)), float((grads[i].double() * way.double()).sum())
        assert abs(quotient - exact) <= 1e-3 * float(grads[i].norm()), (i, quotient, exact)


def test_attention_second_order_refused(ops, dev):
    q = torch.randn(5, 1, 16, device=dev, requires_grad=True)
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(ops.attention(q, q, q, table([5], dev)).square().sum(), q, create_graph=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,heads", [([100], 2), ([130] * 9, 64)])          # split over keys; one pass
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_attention_hidden_nan(ops, dev, lens, heads, dtype, bad):
    """A NaN or an infinity in a key or value that the causal mask hides leaves the queries before it alone, to the bit where no
    tile has to be redone, and within the tolerance where it has; queries that see it get what the definition gives."""
    gen = torch.Generator().manual_seed(9)
    T = sum(lens)
    q, k, v = (torch.randn(T, h, 32, generator=gen).to(dtype) for h in (heads, heads // 2, heads // 2))
    spans_ = spans(lens, lens, lens)
    (w, e), *_ = oracle.attention(q, k, v, torch.zeros_like(q), spans_[:1], True, 32 ** -0.5)
    at = 40                                                                   # of the first sequence
    clean = ops.attention(q.to(dev), k.to(dev), v.to(dev), table(lens, dev), causal=True)
    for which in (0, 1):
        kb, vb = k.clone(), v.clone()
        (kb if which == 0 else vb)[at, 0, 3] = bad
        o = ops.attention(q.to(dev), kb.to(dev), vb.to(dev), table(lens, dev), causal=True)
        within(o[:at], w[:at], e[:at], f"before {which}")
        assert torch.equal(o[lens[0]:], clean[lens[0]:]) and torch.equal(o[:, 2:], clean[:, 2:])
        seen = o[at:lens[0], :2].float().cpu()
        if which == 1:
            col = seen[:, :, 3]
            assert not torch.isfinite(col).any()
            if bad != bad or dtype == torch.float32:
                assert torch.isnan(col).all() if bad != bad else (col == bad).all()
            within(o[at:lens[0], :2, 4:], w[at:lens[0], :2, 4:], e[at:lens[0], :2, 4:], "other columns")
        elif bad != bad:
            assert torch.isnan(seen).all()
