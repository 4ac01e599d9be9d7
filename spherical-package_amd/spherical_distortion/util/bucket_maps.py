"""Bucket maps of relative positions, for functional.bucket_attention.

A map is made once for a pair of token grids and kept, as a sample map is: uint8 [queries, keys], the bucket of
each pair; 255 (never a bucket here) leaves a pair out.
"""
import math

import torch

OUTSIDE = 255


def _check(num_buckets):
    if not 1 <= num_buckets <= 255:
        raise ValueError("num_buckets must be between 1 and 255, got %s" % num_buckets)


def _directions(lonlat):
    lon, lat = lonlat.double().unbind(-1)
    return torch.stack([lat.cos() * lon.cos(), lat.cos() * lon.sin(), lat.sin()], -1)


def great_circle_bucket_map(lonlat, lonlat_keys=None, num_buckets=32, reach=None):
    """Buckets of the great-circle distance between tokens at `lonlat` [queries, 2] (longitude, latitude in
    radians) and `lonlat_keys` [keys, 2] (None: the same tokens).  Bucket floor(num_buckets sqrt(angle / pi)):
    narrow ones near the token, wide ones far away.  reach: pairs further apart (radians) are left out."""
    _check(num_buckets)
    a = _directions(lonlat)
    b = a if lonlat_keys is None else _directions(lonlat_keys)
    out = torch.empty(a.shape[0], b.shape[0], dtype=torch.uint8, device=lonlat.device)
    rows = max(1, (1 << 24) // max(1, b.shape[0]))   # float64 of 128 MB at a time
    for i in range(0, a.shape[0], rows):
        # the chord's half is the sine of half the angle: exact where tokens are close
        chord = torch.cdist(a[i:i + rows], b, compute_mode="donot_use_mm_for_euclid_dist")
        angle = 2 * torch.asin((chord / 2).clamp(max=1))
        bucket = (num_buckets * (angle / math.pi).sqrt()).long().clamp(max=num_buckets - 1)
        if reach is not None:
            bucket[angle > reach] = OUTSIDE
        out[i:i + rows] = bucket.to(torch.uint8)
    return out


def sequence_bucket_map(queries, keys, num_buckets=32, farthest=1024, device="cuda"):
    """Buckets of the distance |i - j| in a sequence of `keys` tokens whose last `queries` ones ask: half of the
    buckets for one distance each, the others for ranges that grow up to `farthest`."""
    _check(num_buckets)
    at = torch.arange(keys - queries, keys, device=device)
    far = (at[:, None] - torch.arange(keys, device=device)[None]).abs()
    near = max(1, num_buckets // 2)
    wide = max(1, num_buckets - near)
    ratio = math.log(max(2.0, farthest / near))
    grown = near + (far.clamp(min=near).double() / near).log() * (wide / ratio)
    return torch.where(far < near, far, grown.long()).clamp(max=num_buckets - 1).to(torch.uint8)
