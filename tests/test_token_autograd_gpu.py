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


def test_captured_backward_beside_another_operators_graph(ops, dev):
    """The leaf's node was made by another operator: refused where that was on the default stream, whatever stream these operators
    met the leaf on; fine where it was on a side stream, though they met the leaf on the default one."""
    cu = torch.tensor([0, 5], dtype=torch.int32, device=dev)
    value, grad = torch.randn(5, 1, 64, device=dev), torch.randn(5, 1, 64, device=dev)
    side = torch.cuda.Stream(dev)
    for stream in (torch.cuda.default_stream(dev), side):
        x = value.clone().requires_grad_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            kept = x * 2                                               # lives on
        torch.cuda.synchronize()
        eager = None
        if stream is side:
            eager = ops.attention(x, x, x, cu)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops.attention(x, x, x, cu)
            if stream is side:
                gx, = torch.autograd.grad(y, x, grad)
            else:
                with pytest.raises(ops._lib.SempyrError, match="capture"):
                    torch.autograd.grad(y, x, grad)
        fresh = value.clone().requires_grad_()
        z = ops.attention(fresh, fresh, fresh, cu)
        want, = torch.autograd.grad(z, fresh, grad)
        for _ in range(3):
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, z) and (stream is not side or torch.equal(gx, want))
        assert kept.requires_grad and (eager is None or torch.equal(eager, z))
