"""Token operators under the parts of autograd that change what a backward pass is given."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from semantic_pyramid_for_image_generation_amd import ops
    return ops


def fused(ops, qkv, cu, pos, rope, w):
    """Queries, keys and values as slices of one projection, normalised and attended."""
    q, k = ops.qk_norm_rope(qkv[:, :4], qkv[:, 4:6], pos, rope, w, w)
    return torch.cat([ops.attention(q, k, qkv[:, 6:], cu, causal=True), ops.attention(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], cu)], dim=1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("pin", [False, True])
def test_saved_on_the_host(ops, dev, dtype, pin):
    """save_on_cpu() returns slices of a projection as dense tensors: the same gradients to the bit."""
    gen = torch.Generator().manual_seed(0)
    T = 150
    qkv, g, w = (torch.randn(*s, generator=gen).to(dtype).to(dev) for s in ((T, 8, 64), (T, 8, 64), (64,)))
    cu, pos = torch.tensor([0, 40, T], dtype=torch.int32, device=dev), torch.arange(T, dtype=torch.int32, device=dev)
    rope = ops.AxialRope((32,))
    grads = []
    for host in (False, True):
        leaves = [qkv.clone().requires_grad_(), w.clone().requires_grad_()]
        if host:
            with torch.autograd.graph.save_on_cpu(pin_memory=pin):
                y = fused(ops, leaves[0], cu, pos, rope, leaves[1])
        else:
            y = fused(ops, leaves[0], cu, pos, rope, leaves[1])
        torch.empty(64 * qkv.numel(), dtype=dtype, device=dev).fill_(float("nan"))       # what freed memory would hold
        grads.append(torch.autograd.grad(y, leaves, g))
    assert all(torch.equal(a, b) for a, b in zip(*grads)) and torch.isfinite(grads[0][0]).all()


def test_second_derivatives_are_refused(ops, dev):
    """Also with a cotangent that needs no gradient: a penalty on such a gradient must not vanish silently."""
    x, w = torch.randn(6, 4, 64, device=dev).requires_grad_(), torch.ones(64, device=dev, requires_grad=True)
    cu, pos = torch.tensor([0, 6], dtype=torch.int32, device=dev), torch.arange(6, dtype=torch.int32, device=dev)
    for y in (ops.attention(x, x, x, cu), ops.qk_norm_rope(x, x, pos, ops.AxialRope((32,)), w, w)[0]):
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(y.sum(), x, create_graph=True)
    y = ops.dropout_add(x, None, 0.5, torch.tensor([1, 2], device=dev))
    gx, = torch.autograd.grad(y.sum(), x, create_graph=True)               # linear: the gradient is a constant
    assert torch.equal(gx, torch.where(y == 0, 0.0, 2.0))


def test_block_in_inference_mode_then_in_training(dev):
    from semantic_pyramid_for_image_generation_amd.attention import SelfAttention2d
    block, x = SelfAttention2d(64).to(dev), torch.randn(2, 64, 6, 5, device=dev)
    with torch.inference_mode():
        y = block.eval()(x)
    z = block.train()(x)
    assert torch.equal(y, z)
    z.square().mean().backward()
    assert all(torch.isfinite(p.grad).all() for p in block.parameters())
