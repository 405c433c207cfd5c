"""Attention's long sums in fp32: terms of one sign, so that what a running sum rounds away adds up.

Adding n equal parts into a running fp32 sum rounds every partial sum to its binade's step: the error's mean square is a twelfth of the
steps' squares.  With the whole at the top of a binade that is n 2^-48 / 12 (1/2 + 1/4 1/4 + 1/8 1/16 + ..), 0.22 2^-24 sqrt(n) of
the whole; right above a power of two the last steps are twice as large, 0.44 2^-24 sqrt(n).  n is what a kernel adds one after the
other: its tiles, each summed by itself before (at most 32 products).  The larger number is allowed, and four roundings (2^-22) for
the exponential, the reciprocal and the factors, and a tenth for the scatter of an L2 norm of some hundred elements."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    from semantic_pyramid_for_image_generation_amd import ops
    return ops


def allowed(parts):
    return 1.1 * U * (0.44 * (parts ** 0.5 + 32 ** 0.5) + 4)


@pytest.mark.parametrize("dim", [32, 64, 128])
def test_gradients_of_keys(ops, dev, dim):
    """32 keys of equal weight seen by 16384 queries of eight heads: dV = sum g / 32, dK = scale sum dS q with dS of the key's sign."""
    T, group, keys = 16384, 8, 32
    gen = torch.Generator(device=dev).manual_seed(dim)
    rand = lambda *s: torch.rand(*s, generator=gen, device=dev) + 1
    q, g = rand(T, group, dim), rand(T, group, dim)
    k = torch.zeros(keys, 1, dim, device=dev)
    sign = torch.tensor([1.0, -1.0], device=dev).repeat(keys // 2)
    v = sign[:, None, None].expand(keys, 1, dim).contiguous()                 # rows' delta is 0
    leaves = [t.requires_grad_() for t in (q, k, v)]
    cu = lambda n: torch.tensor([0, n], dtype=torch.int32, device=dev)
    o = ops.attention(*leaves, cu(T), cu(keys))
    dk, dv = torch.autograd.grad(o, leaves[1:], g)
    want_v = (g.double().sum(dim=(0, 1)) / keys).expand(keys, dim)
    want_k = sign.double()[:, None] * (g.double().sum(-1, keepdim=True) / keys * q.detach().double()).sum(dim=(0, 1)) * dim ** -0.5
    parts = T * group / 32 / 2                                                # tiles of 32 queries, in two groups of waves
    for what, a, b in (("dv", dv, want_v), ("dk", dk, want_k)):
        err = float((a[:, 0].double() - b).norm() / b.norm())
        assert err <= allowed(parts), (what, err, allowed(parts))


def test_long_cache(ops, dev):
    """One query against 262144 keys of equal weight, so many heads that the keys are not split: o = the mean of V."""
    heads, keys, dim = 1024, 262144, 4
    gen = torch.Generator(device=dev).manual_seed(0)
    v = torch.rand(keys, heads, dim, generator=gen, device=dev) + 1
    q, k = torch.zeros(1, heads, dim, device=dev), torch.ones(keys, heads, dim, device=dev)
    cu = lambda n: torch.tensor([0, n], dtype=torch.int32, device=dev)
    o = ops.attention(q, k, v, cu(1), cu(keys))
    want = v.double().mean(dim=0)
    err = float((o[0].double() - want).norm() / want.norm())
    assert err <= allowed(keys / 32 / 2), (err, allowed(keys / 32 / 2))
