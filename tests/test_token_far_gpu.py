"""Token operators on tensors of more than 2^31 elements: rows at the far end give the bits of a small tensor's rows."""
import pytest
import torch

import token_oracle as oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from semantic_pyramid_for_image_generation_amd import ops
    return ops


def test_attention_far_cache(ops, dev):
    """The second of two cache slots begins behind 2^31 elements (K and V are 4.5 GB each)."""
    slot, gen = 2 ** 21 + 100_000, torch.Generator(device=dev).manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=gen, device=dev).bfloat16()
    k, v = (torch.empty(slot + 1000, 8, 128, dtype=torch.bfloat16, device=dev) for _ in range(2))
    near_k, near_v, q = rand(1000, 8, 128), rand(1000, 8, 128), rand(700, 16, 128)
    k[slot:], v[slot:] = near_k, near_v
    k[:1] = v[:1] = 0
    cu_k = torch.tensor([0, slot, slot + 1000], dtype=torch.int32, device=dev)
    len_k = torch.tensor([1, 900], dtype=torch.int32, device=dev)
    for queries in (1, 700):                                   # keys split, one pass
        cu_q = torch.tensor([0, 0, queries], dtype=torch.int32, device=dev)
        far = ops.attention(q[:queries], k, v, cu_q, cu_k, len_k, causal=True)
        near = ops.attention(q[:queries], near_k, near_v, cu_q[1:].contiguous(), torch.tensor([0, 1000], dtype=torch.int32, device=dev),
                             len_k[1:].contiguous(), causal=True)
        # (another number of splits may be taken: the sums' order differs, not more)
        assert float((far.float() - near.float()).norm()) <= 2 ** -8 * float(near.float().norm())
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.attention(*leaves, torch.tensor([0, 0, 700], dtype=torch.int32, device=dev), cu_k, len_k, causal=True),
                                leaves, torch.ones_like(q))
    small = [t.detach().requires_grad_() for t in (q, near_k, near_v)]
    want = torch.autograd.grad(ops.attention(*small, torch.tensor([0, 700], dtype=torch.int32, device=dev),
                                             torch.tensor([0, 1000], dtype=torch.int32, device=dev), len_k[1:].contiguous(), causal=True),
                               small, torch.ones_like(q))
    for a, b in ((grads[0], want[0]), (grads[1][slot:], want[1]), (grads[2][slot:], want[2])):
        assert float((a.float() - b.float()).norm()) <= 2 ** -7 * float(b.float().norm())
    assert not grads[1][1:slot].any() and not grads[2][1:slot].any()


def test_qk_norm_rope_far_rows(ops, dev):
    T, gen = 270_000, torch.Generator(device=dev).manual_seed(2)
    q = torch.zeros(T, 64, 128, dtype=torch.bfloat16, device=dev)
    k = torch.randn(T, 1, 128, generator=gen, device=dev).bfloat16()
    q[-500:] = torch.randn(500, 64, 128, generator=gen, device=dev).bfloat16()
    pos = torch.arange(T, dtype=torch.int32, device=dev)
    w = torch.ones(128, dtype=torch.bfloat16, device=dev)
    rope = ops.AxialRope((64,))
    y, _ = ops.qk_norm_rope(q, k, pos, rope, w, w)
    z, _ = ops.qk_norm_rope(q[-500:].clone(), k[-500:], pos[-500:], rope, w, w)
    assert torch.equal(y[-500:], z) and not y[:1000].any()


def test_dropout_far_elements(ops, dev):
    n, tail = 2 ** 32 + 24 + 5, 29
    x = torch.ones(n, dtype=torch.bfloat16, device=dev)
    rng = torch.tensor([12, 34], device=dev)
    y = ops.dropout_add(x, None, 0.5, rng)
    fields = []
    for b in range((n - tail) // 8, (n + 7) // 8):
        for word in oracle.philox4x32((b & 0xFFFFFFFF, b >> 32, 34, 0), (12, 0)):
            fields += [word & 0xFFFF, word >> 16]
    want = torch.tensor([2.0 if f < 32768 else 0.0 for f in fields[:tail]])
    assert torch.equal(y[-tail:].float().cpu(), want)
