"""A small network over the tokens of a panorama: trained for a few steps, then asked at single directions.

    python examples/panorama_tokens.py [--steps 20]

A MappedConvolution turns an equirectangular picture into features on a coarse grid; its pixels are the tokens of
two blocks (norm with residual, attention whose bias goes by great-circle distance, norm, two linear layers).  The
task is synthetic: the mean colour of the hemisphere about each token's direction.  Training runs in bfloat16 with
AdamW whose moments lie in 8 bits.  Serving keeps a picture's keys and values and asks with one token for a
direction at a time; its last norm leaves rows in 8 bits.
"""
import argparse
import math
import os
import sys

sys.path.insert(1, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "spherical-package_amd"))

import torch  # noqa: E402
import torch.nn as nn  # noqa: E402

import spherical_distortion.functional as F  # noqa: E402
import spherical_distortion.nn as snn  # noqa: E402
import spherical_distortion.util as util  # noqa: E402
from spherical_distortion.optim import AdamW  # noqa: E402


class Block(nn.Module):
    def __init__(self, width, heads, buckets):
        super().__init__()
        self.norm1 = snn.AddRMSNorm(width)
        self.attention = snn.BucketAttention(width, heads, buckets, num_key_heads=heads // 2)
        self.norm2 = snn.AddRMSNorm(width)
        self.up, self.down = nn.Linear(width, 4 * width), nn.Linear(4 * width, width)

    def forward(self, x, residual, bucket_map, keys_and_values=None):
        y, residual = self.norm1(x, residual)
        y = self.attention(y, bucket_map, keys_and_values=keys_and_values)
        y, residual = self.norm2(y, residual)
        return self.down(nn.functional.gelu(self.up(y))), residual


class PanoramaTokens(nn.Module):
    """Pictures [B, 3, H, W] to one colour a token of the H / stride x W / stride grid."""

    def __init__(self, height, width, stride=8, channels=128, heads=4, buckets=24, device="cuda"):
        super().__init__()
        self.stem = snn.MappedConvolution(3, channels, kernel_size=9)
        self.blocks = nn.ModuleList([Block(channels, heads, buckets) for _ in range(2)])
        self.norm = snn.AddRMSNorm(channels)
        self.head = nn.Linear(channels, 3)
        self.register_buffer("sample_map", util.inverse_equirectangular_projection_map(
            (height, width), (3, 3), stride=stride, dilation=stride // 2, device=device))
        rows, columns = self.sample_map.shape[:2]
        lat = math.pi * (torch.arange(rows, device=device) / max(1, rows - 1) - 0.5)
        lon = 2 * math.pi * (torch.arange(columns, device=device) / columns - 0.5)
        self.register_buffer("lonlat", torch.stack([lon.expand(rows, columns), lat[:, None].expand(rows, columns)],
                                                   -1).reshape(-1, 2))
        self.register_buffer("bucket_map", util.great_circle_bucket_map(self.lonlat, num_buckets=buckets))
        self.buckets = buckets
        self.to(device)

    def tokens(self, picture):
        # the mapped operators compute on float32 tensors; the blocks in the type of their weights
        x = self.stem(picture, self.sample_map.to(picture.dtype))
        return x.flatten(2).transpose(1, 2).to(self.head.weight.dtype).contiguous()

    def forward(self, picture):
        x, residual = self.tokens(picture), None
        for block in self.blocks:
            x, residual = block(x, residual, self.bucket_map)
        return self.head(self.norm(x, residual)[0])

    @torch.no_grad()
    def keep(self, picture):
        """What serving keeps of a picture: the last block's input and its keys and values."""
        x, residual = self.tokens(picture), None
        for block in self.blocks[:-1]:
            x, residual = block(x, residual, self.bucket_map)
        last = self.blocks[-1]
        y, residual = last.norm1(x, residual)
        return y, residual, tuple(t.contiguous() for t in last.attention.keys_and_values(y))

    @torch.no_grad()
    def ask(self, kept, token):
        """Colour at one token of the grid: a single query against the picture's keys."""
        y, residual, keys_and_values = kept
        last = self.blocks[-1]
        y = last.attention(y[:, token:token + 1], self.bucket_map[token:token + 1], keys_and_values=keys_and_values)
        y, residual = last.norm2(y, residual[:, token:token + 1].contiguous())
        y = last.down(nn.functional.gelu(last.up(y)))
        codes, scales, _ = self.norm.quantized(y, residual)
        return self.head(F.dequantize_rows(codes, scales, dtype=y.dtype))


def main(steps=20, height=64, width=128, device="cuda:0", seed=0):
    torch.manual_seed(seed)
    net = PanoramaTokens(height, width, device=device)
    for module in (net.blocks, net.norm, net.head):
        module.to(torch.bfloat16)
    optimizer = AdamW(net.parameters(), lr=2e-3, moment_bits=8)
    near = net.lonlat
    directions = torch.stack([near[:, 1].cos() * near[:, 0].cos(), near[:, 1].cos() * near[:, 0].sin(),
                              near[:, 1].sin()], -1)
    hemisphere = ((directions @ directions.T) > 0).float() * near[:, 1].cos()[None]
    hemisphere /= hemisphere.sum(1, keepdim=True)
    losses = []
    for step in range(steps):
        coarse = torch.rand(4, 3, 8, 16, device=device)
        picture = nn.functional.interpolate(coarse, (height, width), mode="bilinear")
        pooled = nn.functional.adaptive_avg_pool2d(picture, net.sample_map.shape[:2]).flatten(2)
        want = (hemisphere @ pooled.transpose(1, 2).contiguous())
        loss = nn.functional.mse_loss(net(picture).float(), want)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    losses = [float(x) for x in losses]
    kept = net.keep(picture)
    token = net.lonlat.shape[0] // 2 + 3
    with torch.no_grad():
        full = net(picture)[:, token].float()
    off = float((net.ask(kept, token)[:, 0].float() - full).abs().max())
    print("loss %.4f -> %.4f in %d steps; one token asked alone differs by %.4f from the whole grid's"
          % (losses[0], losses[-1], steps, off))
    return losses, off


if __name__ == "__main__":
    parser = argparse.ArgumentParser()
    parser.add_argument("--steps", type=int, default=20)
    main(parser.parse_args().steps)
