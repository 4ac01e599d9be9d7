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
