"""Token operators on the GPU against their definitions in 64 bits (token_oracle.py derives the tolerances)."""
import pytest
import torch

import token_oracle as oracle

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ops():
    from semantic_pyramid_for_image_generation_amd import ops
    return ops


def within(got, want, bound, what):
    err = (got.double().cpu() - want).abs()
    worst = (err / bound.clamp_min(1e-300)).max() if err.numel() else torch.zeros(())
    assert torch.isfinite(got).all() and float(worst) <= 1.0, f"{what}: {float(worst):.3g} of the bound, error {float(err.max()):.3g}"


# tokens, heads_q, heads_k, dim, sections, interleaved, shared
ROPE = [
    (1, 1, 1, 2, (1,), False, False),
    (3, 2, 1, 16, (8,), True, False),
    (7, 4, 2, 32, (8, 8), False, False),
    (65, 5, 1, 64, (10, 11, 11), False, True),
    (33, 3, 3, 80, (20,), False, False),             # rotated part that is no whole vector
    (33, 3, 3, 80, (10, 10), True, False),
    (19, 8, 2, 96, (16, 16), True, True),
    (130, 16, 2, 128, (16, 24, 24), False, True),
    (9, 2, 2, 34, (3, 5, 2), False, False),          # odd halves
    (5, 2, 1, 512, (64, 64, 64, 64), False, False),
    (4, 1, 1, 6, (1, 0, 1), True, False),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", ROPE)
@pytest.mark.parametrize("norm", [True, False])
def test_qk_norm_rope(ops, dev, case, dtype, norm):
    T, hq, hk, dim, sections, inter, shared = case
    gen = torch.Generator().manual_seed(T * 1000 + dim)
    rand = lambda *s: torch.randn(*s, generator=gen).to(dtype)
    qkv = rand(T, hq + 2 * hk, dim)
    gq, gk = rand(T, hq, dim), rand(T, hk, dim)
    w = [1 + 0.25 * rand(dim), 1 + 0.25 * rand(dim)] if norm else [None, None]
    pos = torch.randint(-50000, 2 ** 20, (T, len(sections)), generator=gen, dtype=torch.int32)
    rope = ops.AxialRope(sections, interleaved=inter, shared=shared)
    d = qkv.to(dev)
    q, k = d[:, :hq].requires_grad_(), d[:, hq:hq + hk].requires_grad_()
    wd = [None if t is None else t.to(dev).requires_grad_() for t in w]
    yq, yk = ops.qk_norm_rope(q, k, pos.to(dev), rope, *wd, eps=1e-6)
    leaves = [q, k] + ([wd[0], wd[1]] if norm else [])
    grads = torch.autograd.grad([yq, yk], leaves, [gq.to(dev), gk.to(dev)])
    for i, (x, g, y) in enumerate(((qkv[:, :hq], gq, yq), (qkv[:, hq:hq + hk], gk, yk))):
        wy, wx, ww = oracle.qk_norm_rope(x, w[i], g, pos, sections, 10000.0, inter, shared, 1e-6)
        assert y.dtype == dtype and y.is_contiguous()
        within(y.detach(), *wy, f"y[{i}]")
        within(grads[i], *wx, f"dx[{i}]")
        if norm:
            within(grads[2 + i], *ww, f"dw[{i}]")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [24, 40, 48, 80, 96, 112, 144, 160, 192, 224, 288, 384])
@pytest.mark.parametrize("tokens", [1, 11, 257])
def test_qk_norm_rope_group_sizes(ops, dev, dim, tokens, dtype):
    """Heads whose vectors are no power of two: groups of 3, 5, 6, 7, .. lanes, the last lanes of a wave without one."""
    test_qk_norm_rope(ops, dev, (tokens, 3, 2, dim, (dim // 2,), False, False), dtype, True)
    test_qk_norm_rope(ops, dev, (tokens, 1, 1, dim, (dim // 4, dim // 4), True, False), dtype, False)


@pytest.mark.parametrize("dtype", TYPES)
def test_qk_norm_rope_strides(ops, dev, dtype):
    """Views that are not 16-byte aligned, heads before tokens, a last dimension that is not dense: equal to dense copies."""
    gen = torch.Generator().manual_seed(3)
    base = torch.randn(4, 40, 133, generator=gen).to(dtype).to(dev)
    pos = torch.arange(40, dtype=torch.int32, device=dev)
    rope = ops.AxialRope((32,))
    w = torch.ones(64, dtype=dtype, device=dev)
    for view in (base[:, :, 1:65], base[:, :, 2:130:2], base[:, :, 64:128]):
        q = view.transpose(0, 1)                                # [tokens, heads, dim] of heads-first memory
        a = ops.qk_norm_rope(q, q[:, :2], pos, rope, w, w)
        b = ops.qk_norm_rope(q.contiguous(), q[:, :2].contiguous(), pos, rope, w, w)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_qk_norm_rope_edges(ops, dev):
    rope = ops.AxialRope((4,))
    w = torch.full((8,), 2.0, device=dev, requires_grad=True)
    e = torch.zeros(0, 2, 8, device=dev, requires_grad=True)
    y = ops.qk_norm_rope(e, e, torch.zeros(0, dtype=torch.int32, device=dev), rope, w, w)
    g = torch.autograd.grad([y[0].sum() + y[1].sum()], [e, w])
    assert y[0].shape == (0, 2, 8) and g[0].shape == (0, 2, 8) and torch.equal(g[1], torch.zeros_like(w))
    z = torch.zeros(3, 1, 8, device=dev)                                # a row of zeros stays zero, with eps and without a NaN
    y, _ = ops.qk_norm_rope(z, z, torch.full((3,), 2 ** 31 - 1, dtype=torch.int32, device=dev), rope, w, w)
    assert torch.equal(y, z)
    with pytest.raises(NotImplementedError):                             # second derivatives are refused
        x = torch.randn(3, 1, 8, device=dev, requires_grad=True)
        y, _ = ops.qk_norm_rope(x, x, torch.arange(3, dtype=torch.int32, device=dev), rope, w, w)
        gx, = torch.autograd.grad(y.square().sum(), x, create_graph=True)


def test_qk_norm_rope_far_positions(ops, dev):
    """The angle's reduction is exact: positions 2^31 - 1 and -2^31 rotate as precisely as position 1."""
    pos = torch.tensor([2 ** 31 - 1, -2 ** 31, 2 ** 30 + 1, 1], dtype=torch.int32)
    x = torch.randn(4, 2, 64, generator=torch.Generator().manual_seed(0))
    rope = ops.AxialRope((32,))
    y, _ = ops.qk_norm_rope(x.to(dev), x.to(dev), pos.to(dev), rope)
    two_pi = 6.283185307179586476925286766559
    ang = torch.tensor([[((f * int(p)) % 2 ** 64) / 2 ** 64 * two_pi for f in rope.fractions()] for p in pos], dtype=torch.float64)
    a, b = x[..., :32].double(), x[..., 32:].double()
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    want = torch.cat([a * c - b * s, a * s + b * c], dim=-1)
    within(y, want, 8 * oracle.U * 2 * x.abs().amax(dim=-1, keepdim=True).double() + 2 * oracle.U * want.abs(), "y")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 2047, 2048, 2050, 6001])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout_add(ops, dev, n, p, dtype):
    gen = torch.Generator().manual_seed(n)
    x, res, g = (torch.randn(n, generator=gen).to(dtype) for _ in range(3))
    seed, offset = 0x123456789ABCDEF, -3 + n
    gain = oracle.dropout_gain(n, p, seed, offset)
    rng = torch.tensor([seed, offset], dtype=torch.int64, device=dev)
    step = oracle.half_step(dtype)
    for with_res in (True, False):
        xd, rd = x.to(dev).requires_grad_(), res.to(dev).requires_grad_()
        y = ops.dropout_add(xd, rd if with_res else None, p, rng)
        want = gain * x.double() + (res.double() if with_res else 0)
        # the scale is rounded once, the multiply-add once, the result once
        bound = 2 * oracle.U * (gain * x.double()).abs() + (step + 2 * oracle.U) * want.abs() * 1.01
        within(y.detach(), want, bound, "y")
        assert torch.equal(y.detach().cpu()[gain == 0], res[gain == 0] if with_res else torch.zeros_like(res)[gain == 0])
        grads = torch.autograd.grad(y, [xd, rd] if with_res else [xd], g.to(dev))
        want = gain * g.double()
        within(grads[0], want, (2 * oracle.U + step) * 1.01 * want.abs(), "dx")
        if with_res:
            assert torch.equal(grads[1].cpu(), g)


def test_dropout_add_views_and_specials(ops, dev):
    rng = torch.tensor([5, 6], dtype=torch.int64, device=dev)
    x = torch.randn(33, 70, device=dev)
    a = ops.dropout_add(x[:, 1:65], x[:, 2:66], 0.3, rng)                # unaligned, strided: as dense copies
    assert torch.equal(a, ops.dropout_add(x[:, 1:65].contiguous(), x[:, 2:66].contiguous(), 0.3, rng))
    inf = torch.full((4096,), float("inf"), device=dev)
    y = ops.dropout_add(inf, None, 0.5, rng)                             # a dropped infinity is zero, not NaN
    assert torch.equal(torch.isinf(y).cpu(), oracle.dropout_gain(4096, 0.5, 5, 6) != 0) and not torch.isnan(y).any()
    assert ops.dropout_add(x[:0], x[:0], 0.3, rng).shape == (0, 70)
    b = ops.dropout_add(x, None, 0.3, rng.clone().add_(1))
    assert not torch.equal(b, ops.dropout_add(x, None, 0.3, rng))       # another key, other decisions
