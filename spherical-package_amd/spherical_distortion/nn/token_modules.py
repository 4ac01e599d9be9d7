"""nn.Module front-ends of the operators on token sequences."""
import torch
import torch.nn as nn

from .. import functional as F


class BucketAttention(nn.Module):
    """Self- or cross-attention of tokens [B, tokens, width] with a learned bias for each bucket of relative
    positions.  num_key_heads (a divisor of num_heads): heads that share keys and values.  The bias starts at
    zero; projections have no additive bias."""

    def __init__(self, width, num_heads, num_buckets, num_key_heads=None):
        super().__init__()
        num_key_heads = num_heads if num_key_heads is None else num_key_heads
        if width % num_heads or num_heads % num_key_heads:
            raise ValueError("width %d must divide into %d heads, and those into %d key heads"
                             % (width, num_heads, num_key_heads))
        if width // num_heads % 8 or not 8 <= width // num_heads <= 128:
            raise ValueError("width %d in %d heads: a head's values must be a multiple of 8 up to 128"
                             % (width, num_heads))
        if not 1 <= num_buckets <= 256:
            raise ValueError("num_buckets must be between 1 and 256, got %s" % num_buckets)
        self.num_heads, self.num_key_heads, self.dim = num_heads, num_key_heads, width // num_heads
        self.query = nn.Linear(width, width, bias=False)
        self.key_value = nn.Linear(width, 2 * num_key_heads * self.dim, bias=False)
        self.out = nn.Linear(width, width, bias=False)
        self.bias_table = nn.Parameter(torch.zeros(num_heads, num_buckets))

    def keys_and_values(self, x):
        """Keys and values [B, key heads, tokens, dim] of x: made once for a picture that many tokens ask."""
        B, L, _ = x.shape
        kv = self.key_value(x).view(B, L, 2, self.num_key_heads, self.dim)
        return kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)

    def forward(self, x, bucket_map, key_lengths=None, causal=False, keys_and_values=None):
        """x asks itself, or the keys and values handed in."""
        B, L, width = x.shape
        q = self.query(x).view(B, L, self.num_heads, self.dim).transpose(1, 2)
        k, v = self.keys_and_values(x) if keys_and_values is None else keys_and_values
        out = F.bucket_attention(q, k, v, self.bias_table, bucket_map, key_lengths, causal)
        return self.out(out.transpose(1, 2).reshape(B, L, width))


class AddRMSNorm(nn.Module):
    """(norm of x + residual, x + residual); a residual of None adds nothing."""

    def __init__(self, width, eps=1e-6):
        super().__init__()
        if not 1 <= width <= 16384:
            raise ValueError("width must be between 1 and 16384, got %s" % width)
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(width))

    def forward(self, x, residual=None):
        return F.add_rms_norm(x, residual, self.weight, self.eps)

    def quantized(self, x, residual=None, dtype=torch.int8):
        """(codes, scales, x + residual): the norm's rows in 8 bits, without gradients."""
        return F.add_rms_norm_quantized(x, residual, self.weight, self.eps, dtype)


class AddLayerNorm(nn.Module):
    """(layer norm of x + residual, x + residual); a residual of None adds nothing."""

    def __init__(self, width, eps=1e-5, bias=True):
        super().__init__()
        if not 1 <= width <= 16384:
            raise ValueError("width must be between 1 and 16384, got %s" % width)
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(width))
        self.bias = nn.Parameter(torch.zeros(width)) if bias else None

    def forward(self, x, residual=None):
        return F.add_layer_norm(x, residual, self.weight, self.bias, self.eps)


class GatedScan(nn.Module):
    """Tokens [B, tokens, width] mixed along the sequence by a gated linear recurrence of `channels` (None: width)
    channels, whose output is gated and projected back: linear in the number of tokens where attention is quadratic.
    both_ways: the second half of the channels runs from the last token to the first, so that every token sees all.
    The channels' gates begin with memories of two to about 400 tokens."""

    def __init__(self, width, channels=None, both_ways=False):
        super().__init__()
        channels = width if channels is None else channels
        if width < 1 or not 1 <= channels <= 1 << 20 or (both_ways and channels % 2):
            raise ValueError("width %s and channels %s must be positive, channels at most 2^20 and even both ways"
                             % (width, channels))
        self.channels, self.both_ways = channels, both_ways
        self.inputs = nn.Linear(width, 3 * channels)
        self.out = nn.Linear(channels, width, bias=False)
        with torch.no_grad():
            ways = 2 if both_ways else 1
            self.inputs.bias.zero_()
            self.inputs.bias[channels:2 * channels] = torch.linspace(0, 6, channels // ways).repeat(ways)

    def _out(self, h, z):
        return self.out(h * nn.functional.silu(z))

    def forward(self, x, state=None, lengths=None):
        """(tokens like x, last state [B, channels] float32); the state goes in front of the next call's tokens.  Both
        ways there is none: a state is refused, and None returned."""
        x, gate, z = self.inputs(x).chunk(3, -1)
        if not self.both_ways:
            h, last = F.gated_scan(x, gate, state, lengths)
            return self._out(h, z), last
        if state is not None:
            raise ValueError("a scan both ways begins with no state")
        half = self.channels // 2
        ahead, _ = F.gated_scan(x[..., :half], gate[..., :half], None, lengths)
        back, _ = F.gated_scan(x[..., half:], gate[..., half:], None, lengths, reverse=True)
        return self._out(torch.cat([ahead, back], -1), z), None

    @torch.no_grad()
    def step(self, x, state):
        """One token [B, width] of each sequence; state (float32 [B, channels]) is updated in place."""
        if self.both_ways:
            raise ValueError("a scan both ways has no single tokens")
        x, gate, z = self.inputs(x).chunk(3, -1)
        return self._out(F.gated_scan_step(x, gate, state), z)
