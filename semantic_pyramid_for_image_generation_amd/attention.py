"""Self-attention over a feature map, the optional block of the generator (`Generator(gen_type, attention_size=S)`).  It has no
counterpart in the reference, whose generator is convolutional throughout (generator.py:97-134); left out, the generator is
the reference's."""
import torch
import torch.nn as nn

from . import ops, parallel
from .blocks import init_weights, run_conv, run_norm


class SelfAttention2d(nn.Module):
    """x + dropout(proj(attention(norm(x)))): every place of a map attends to every place of the same map.  Heads of 64 channels
    (fewer where the map has less), queries and keys normalised per head, positions rotated by row and column."""

    def __init__(self, channels, head_dim=64, dropout=0.0):
        super().__init__()
        head_dim = min(head_dim, channels)
        if channels % head_dim or head_dim % 8 or head_dim > 128:
            raise ValueError(f"SelfAttention2d: {channels} channels do not divide into heads of {head_dim}")
        if not 0.0 <= dropout < 1.0:
            raise ValueError(f"SelfAttention2d: dropout must lie in [0, 1), got {dropout}")
        self.heads, self.head_dim, self.dropout = channels // head_dim, head_dim, float(dropout)
        self.norm = nn.GroupNorm(1, channels)
        self.qkv = nn.Conv2d(channels, 3 * channels, kernel_size=1, bias=False)
        self.proj = nn.Conv2d(channels, channels, kernel_size=1)
        self.q_weight = nn.Parameter(torch.ones(head_dim))
        self.k_weight = nn.Parameter(torch.ones(head_dim))
        self.rope = ops.AxialRope((head_dim // 4, head_dim // 4))
        # {seed, offset} of the dropout's generator; the offset counts the training passes.  The seed is what torch's generator
        # would give next (a copy of it is asked: other layers' seeded values stay what they are), another one for every block.
        # Like that generator's state it is no part of the state_dict: a training that goes on exactly saves and restores it.
        state = torch.Generator().set_state(torch.get_rng_state())
        self.register_buffer('rng', torch.tensor([int(torch.randint(0, 2 ** 62, (), generator=state, device='cpu')), 0]), persistent=False)
        self._places = {}

    def init_weights(self):
        self.qkv.apply(init_weights)
        self.proj.apply(init_weights)
        nn.init.zeros_(self.proj.bias)

    def _grid(self, B, H, W, device):
        """(positions, sequence table) of B maps; kept per shape, except under a graph capture, whose memory is the graph's."""
        capturing = device.type == 'cuda' and torch.cuda.is_current_stream_capturing()
        key = (B, H, W, device)
        hit = self._places.get(key)
        if hit is None:
            # kept ones are made on the host: their copy has ended when it returns, so any stream may use them next.  (Not as
            # inference tensors, whatever the mode of the first pass: a later one saves them for its backward pass.)
            where = device if capturing else torch.device('cpu')
            with torch.inference_mode(False):
                i = torch.arange(B * H * W, device=where, dtype=torch.int32)
                hit = (torch.stack([i // W % H, i % W], dim=1).to(device, torch.int32),
                       torch.arange(0, (B + 1) * H * W, H * W, device=where, dtype=torch.int32).to(device))
            if not capturing:
                self._places[key] = hit
        return hit

    def __getstate__(self):
        return dict(self.__dict__, _places={})

    def forward(self, x):
        B, C, H, W = x.shape
        positions, table = self._grid(B, H, W, x.device)
        y = run_conv(self.qkv, run_norm(self.norm, x))
        # channels-last tokens: [B * H * W, 3, heads, head_dim]
        tokens = y.flatten(2).transpose(1, 2).reshape(B * H * W, 3, self.heads, self.head_dim)
        q, k, v = tokens.unbind(1)
        q, k = ops.qk_norm_rope(q, k, positions, self.rope, self.q_weight, self.k_weight)
        o = ops.attention(q, k, v, table)
        o = run_conv(self.proj, o.view(B, H * W, C).transpose(1, 2).reshape(B, C, H, W))
        if self.dropout == 0.0 or not self.training:
            return ops.add_act(x, o)
        # The backward pass needs this pass's offset (an addition and no copy: the loop's graph replay takes kernels only).
        # Ranks hold equal state and other samples: their decisions differ, too.
        now = self.rng + parallel.rank()
        self.rng[1].add_(1)
        return ops.dropout_add(o, x, self.dropout, now)
