"""Token operators without a GPU: refusals, the frequency table, the generator's published test vectors, C entry checks."""
import ctypes
import math

import pytest
import torch

from token_oracle import dropout_gain, frequencies, philox4x32


@pytest.fixture(scope="module")
def ops():
    from semantic_pyramid_for_image_generation_amd import ops
    return ops


def test_philox_known_answers():
    """The generator's published vectors (counter, key -> words) hold for the oracle the GPU results are compared with."""
    assert philox4x32((0, 0, 0, 0), (0, 0)) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    m = 0xFFFFFFFF
    assert philox4x32((m, m, m, m), (m, m)) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    g = dropout_gain(4096, 0.25, 5, 7)
    assert abs(float(g.mean()) - 1.0) < 5 * math.sqrt(0.25 / 0.75 / 4096)


@pytest.mark.parametrize("sections,shared", [((8,), False), ((16, 24, 24), True), ((5, 0, 3), False), ((13, 14), False)])
def test_rope_fractions(ops, sections, shared):
    rope = ops.AxialRope(sections, 10000.0, shared=shared)
    want = frequencies(sections, 10000.0, shared)
    assert rope.frequencies() == want
    for f, turn in zip(want, rope.fractions()):
        assert abs(turn / 2 ** 64 - f / (2 * math.pi)) <= 2.0 ** -52
        for pos in (0, 1, -1, 123456, -(2 ** 31), 2 ** 31 - 1):         # the wrapping product is the angle modulo one turn
            wrapped = (turn * pos) % 2 ** 64 / 2 ** 64
            assert abs(math.cos(2 * math.pi * wrapped) - math.cos(pos * f)) <= 2.0 ** -52 * max(1, abs(pos)) * 8


def test_rope_table_on_the_host(ops):
    rope = ops.AxialRope((5, 0, 3))
    t = rope.table("cpu")
    assert t.dtype == torch.int64 and [int(v) % 2 ** 64 for v in t] == rope.fractions() and rope.table(torch.device("cpu")) is t


def test_rope_refusals(ops):
    E = ops._lib.SempyrError
    for bad in ((), (0,), (-1, 4), (1,) * 5):
        with pytest.raises(E):
            ops.AxialRope(bad)
    for base in (0.5, float("inf"), float("nan")):
        with pytest.raises(E):
            ops.AxialRope((4,), base)
    rope = ops.AxialRope((4, 4))
    q, k = torch.zeros(3, 2, 16), torch.zeros(3, 1, 16)
    pos = torch.zeros(3, 2, dtype=torch.int32)
    w = torch.ones(16)
    for args in ((q[0], k, pos, rope), (q, k[:2], pos, rope), (q, k[..., :8], pos, rope), (q[:, :0], k, pos, rope),
                 (q, k, pos[:2], rope), (q, k, pos.long(), rope), (q, k, pos[:, :1], rope), (q, k, pos[:, 0], rope),
                 (q[..., :15], k[..., :15], pos, rope), (q[..., :14], k[..., :14], pos, rope),
                 (q, k, pos, rope, w), (q, k, pos, rope, w[:8], w), (q, k, pos, rope, w, w, -1.0),
                 (q, k, pos, rope, w, w, float("nan")), (q, k.half(), pos, rope), (q.double(), k.double(), pos, rope),
                 (q, k, pos, rope, w.half(), w.half())):
        with pytest.raises(E):
            ops.qk_norm_rope(*args)
    with pytest.raises(E, match="GPU only"):
        ops.qk_norm_rope(q, k, pos, rope, w, w)


def test_dropout_refusals(ops):
    E = ops._lib.SempyrError
    x, rng = torch.zeros(4, 4), torch.zeros(2, dtype=torch.int64)
    for args in ((x, x[:2], 0.1, rng), (x, None, -0.1, rng), (x, None, 1.1, rng), (x, None, float("nan"), rng),
                 (x, None, 0.1, rng[:1]), (x, None, 0.1, rng.int()), (x, x.half(), 0.1, rng), (x.double(), None, 0.1, rng)):
        with pytest.raises(E):
            ops.dropout_add(*args)
    with pytest.raises(E, match="GPU only"):
        ops.dropout_add(x, None, 0.1, rng)


def test_attention_refusals(ops):
    E = ops._lib.SempyrError
    q, k = torch.zeros(6, 4, 16), torch.zeros(6, 2, 16)
    cu = torch.tensor([0, 2, 6], dtype=torch.int32)
    for args in ((q[0], k, k, cu), (q, k, k[:5], cu), (q, k[..., :8], k[..., :8], cu), (q[:, :3], k, k, cu), (q[:, :0], k, k, cu),
                 (q, k.half(), k, cu), (q.double(), k.double(), k.double(), cu), (q[..., :6], k[..., :6], k[..., :6], cu),
                 (torch.zeros(6, 1, 132),) * 3 + (cu,), (torch.zeros(6, 1, 12, dtype=torch.half),) * 3 + (cu,), (q[:5], k, k, cu),
                 (q, k, k, cu.long()), (q, k, k, cu[None]), (q, k, k, cu[:0]), (q, k, k, cu, cu[:2]), (q, k, k, cu, cu, cu),
                 (q, k, k, cu, cu, None, True, 0.0), (q, k, k, cu, cu, None, True, -1.0), (q, k, k, cu, cu, None, True, float("inf")),
                 (q, k, k, cu, cu, None, True, float("nan"))):
        with pytest.raises(E):
            ops.attention(*args)
    with pytest.raises(E, match="GPU only"):
        ops.attention(q, k, k, cu, causal=True)


def test_attention_oracle_gradients():
    """The oracle's gradients are those of differentiating its definition."""
    import token_oracle
    gen = torch.Generator().manual_seed(0)
    q, k, v, g = (torch.randn(n, h, 8, generator=gen, dtype=torch.float64).float() for n, h in ((11, 4), (15, 2), (15, 2), (11, 4)))
    seqs = [(0, 4, 0, 3), (4, 7, 3, 9)]
    got = token_oracle.attention(q, k, v, g, seqs, True, 0.4)
    leaves = [t.double().requires_grad_() for t in (q, k, v)]
    out = torch.zeros(11, 4, 8, dtype=torch.float64)
    for q0, lq, k0, lk in seqs:
        for h in range(4):
            s = 0.4 * leaves[0][q0:q0 + lq, h] @ leaves[1][k0:k0 + lk, h // 2].t()
            hide = torch.arange(lk)[None] > torch.arange(lq)[:, None] + lk - lq
            e = torch.where(hide, torch.zeros_like(s), s.exp())
            out[q0:q0 + lq, h] = e @ leaves[2][k0:k0 + lk, h // 2] / e.sum(-1, keepdim=True).clamp_min(1e-30)
    grads = torch.autograd.grad(out, leaves, g.double())
    for (w, e), t in zip(got, [out.detach(), *grads]):
        assert torch.allclose(w, t, rtol=0, atol=1e-12)


def test_c_entries_refuse_bad_descriptors():
    """Every refusal happens on the host, before a launch."""
    from semantic_pyramid_for_image_generation_amd import _lib
    L = _lib.lib
    sec = lambda *s: (ctypes.c_int32 * 4)(*s)
    good = dict(tokens=4, q_stride_token=32, q_stride_head=16, k_stride_token=16, k_stride_head=16, dtype=_lib.F32, heads_q=2,
                heads_k=1, dim=16, axes=1, sections=sec(8), interleaved=0, eps=1e-6)
    for change in (dict(dim=15), dict(dim=514), dict(dtype=3), dict(heads_q=0), dict(axes=0), dict(axes=5), dict(sections=sec(9)),
                   dict(sections=sec(0)), dict(sections=sec(-1)), dict(tokens=-1), dict(eps=-1.0), dict(eps=float("nan"))):
        d = _lib.RopeDesc(**{**good, **change})
        assert L.sempyr_qk_norm_rope_fwd(ctypes.byref(d), 16, 16, 16, 16, 16, 16, 16, 16, 0) < 0, change
        assert L.sempyr_last_error_string()
        assert L.sempyr_qk_norm_rope_bwd(ctypes.byref(d), *[16] * 13, 0) < 0, change
    d = _lib.RopeDesc(**good)
    assert L.sempyr_qk_norm_rope_fwd(ctypes.byref(d), 0, 16, 16, 16, 16, 16, 16, 16, 0) < 0        # null queries
    assert L.sempyr_qk_norm_rope_fwd(ctypes.byref(d), 16, 16, 16, 16, 16, 0, 16, 16, 0) < 0        # one weight only
    assert L.sempyr_qk_norm_rope_fwd(None, 16, 16, 16, 16, 16, 16, 16, 16, 0) < 0
    n = ctypes.c_int64()
    assert L.sempyr_qk_norm_rope_bwd_scratch(ctypes.byref(d), ctypes.byref(n)) == 0 and n.value >= 2 * 16
    for args in ((7, 16, 0, 16, 8, 0.1, 16), (0, 16, 0, 16, -1, 0.1, 16), (0, 16, 0, 16, 8, 1.5, 16), (0, 16, 0, 16, 8, -0.5, 16),
                 (0, 0, 0, 16, 8, 0.1, 16), (0, 16, 0, 16, 8, 0.1, 0), (0, 16, 0, 16, 8, float("nan"), 16),
                 (0, 16, 0, 16, 2 ** 34 + 1, 0.1, 16)):
        assert L.sempyr_dropout_add(*args, 0) < 0, args
    assert L.sempyr_dropout_add(0, 0, 0, 0, 0, 0.1, 0, 0) == 0             # nothing to do


def test_attention_c_entries_refuse():
    from semantic_pyramid_for_image_generation_amd import _lib
    L = _lib.lib
    good = dict(total_q=8, total_k=8, q_stride_token=64, q_stride_head=16, k_stride_token=32, k_stride_head=16, v_stride_token=32,
                v_stride_head=16, dtype=_lib.F32, heads_q=4, heads_k=2, dim=16, nseq=1, causal=1, scale=0.25)
    for change in (dict(dim=0), dict(dim=6), dict(dim=132), dict(dtype=-1), dict(heads_q=3), dict(heads_k=0), dict(nseq=-1),
                   dict(scale=0.0), dict(scale=float("nan")), dict(scale=3e38), dict(total_q=-1), dict(total_k=2 ** 31), dict(k_stride_token=33),
                   dict(k_stride_token=8), dict(v_stride_token=2 ** 24), dict(q_stride_head=-16)):
        d = _lib.AttentionDesc(**{**good, **change})
        n = ctypes.c_int64()
        assert L.sempyr_attention_workspace(ctypes.byref(d), ctypes.byref(n)) < 0, change
        assert L.sempyr_attention_fwd(ctypes.byref(d), *[16] * 10, 0, 16) < 0, change
        assert L.sempyr_attention_bwd(ctypes.byref(d), *[16] * 15) < 0, change
    d = _lib.AttentionDesc(**good)
    for hole in (0, 1, 2, 3, 4, 6):                     # (5: len_k may be absent)
        args = [16] * 10 + [0, 16]
        args[hole] = 0
        assert L.sempyr_attention_fwd(ctypes.byref(d), *args) < 0, hole
    args = [16] * 10 + [0, 16]
    args[1] = 20                                        # keys that are not 16-byte aligned
    assert L.sempyr_attention_fwd(ctypes.byref(d), *args) < 0
    n = ctypes.c_int64()
    d = _lib.AttentionDesc(**{**good, "total_q": 1, "total_k": 4096})
    assert L.sempyr_attention_workspace(ctypes.byref(d), ctypes.byref(n)) == 0 and n.value > 0
    assert L.sempyr_attention_fwd(ctypes.byref(d), *[16] * 10, n.value - 1, 16) < 0 and b"workspace" in L.sempyr_last_error_string()
    assert L.sempyr_attention_fwd(ctypes.byref(d), *[16] * 9, 0, n.value, 16) < 0


def test_launches_beyond_the_grid_are_refused():
    """More than 2^32 threads in a launch (none of these tensors would fit into memory)."""
    from semantic_pyramid_for_image_generation_amd import _lib
    L = _lib.lib
    d = _lib.RopeDesc(2 ** 31, 32, 16, 16, 16, _lib.F32, 4096, 4096, 16, 1, (ctypes.c_int32 * 4)(8), 0, 1e-6)
    assert L.sempyr_qk_norm_rope_fwd(ctypes.byref(d), *[16] * 8, 0) < 0 and b"rows" in L.sempyr_last_error_string()
    row = 65536 * 16
    for q, k in ((2 ** 30, 2 ** 30), (2 ** 24, 2 ** 24)):         # the one-pass kernel; the split one
        d = _lib.AttentionDesc(q, k, row, 16, row, 16, row, 16, _lib.F32, 65536, 65536, 16, 1 if q > 2 ** 24 else 2 ** 24, 1, 0.25)
        assert L.sempyr_attention_fwd(ctypes.byref(d), *[16] * 10, 2 ** 62, 16) < 0 and b"tiles" in L.sempyr_last_error_string()
        assert L.sempyr_attention_bwd(ctypes.byref(d), *[16] * 15) < 0 and b"tiles" in L.sempyr_last_error_string()


def test_captured_backward_of_leaves_that_another_graph_holds(ops, monkeypatch):
    """The check, with a plain function on the CPU and the streams played by numbers."""
    now = {'stream': 0, 'capturing': False}
    monkeypatch.setattr(ops, '_stream', lambda: now['stream'])
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: now['capturing'])

    class Product(torch.autograd.Function):
        @staticmethod
        def forward(ctx, a, b):
            ops._mark_leaves(ctx)
            ctx.save_for_backward(a, b)
            return a * b

        @staticmethod
        def backward(ctx, g):
            ops._check_backward("product", ctx, g)
            a, b = ctx.saved_tensors
            return g * b, g * a

    w, x = torch.ones(3, requires_grad=True), torch.ones(3)
    eager = Product.apply(w, x)
    now.update(stream=2, capturing=True)
    captured = Product.apply(w, x)
    with pytest.raises(ops._lib.SempyrError, match="capture"):
        torch.autograd.grad(captured.sum(), w)
    with pytest.raises(ops._lib.SempyrError, match="capture"):
        captured.sum().backward()
    fresh = w.detach().requires_grad_()                            # a leaf of its own
    assert torch.equal(torch.autograd.grad(Product.apply(fresh, x).sum(), fresh)[0], x)
    inner = Product.apply(fresh, x)                                # no leaf of the other graph takes this gradient
    assert torch.equal(torch.autograd.grad(Product.apply(inner, x).sum(), inner)[0], x)
    del eager, captured                                            # nothing of the other graph lives
    now.update(stream=1, capturing=False)
    side = Product.apply(w, x)                                     # made on a stream that can join a capture
    now.update(stream=2, capturing=True)
    assert torch.equal(torch.autograd.grad(Product.apply(w, x).sum(), w)[0], x)
    del side
    assert torch.equal(torch.autograd.grad(Product.apply(w, x).sum(), w)[0], x)
    now.update(stream=0, capturing=False)
    kept = Product.apply(w, x)
    now.update(stream=1)
    assert torch.equal(torch.autograd.grad(Product.apply(w, x).sum(), w)[0], x) and kept is not None      # eager: any stream
