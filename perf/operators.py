"""The work that the operators for token sequences on the sphere are measured on.

`listed()` gives the fixed cases, `draw()` further ones of the same ranges, `prepare()` what a
program has in hand before a pass (on the GPU), `run()` one pass through one operator, `work()` the
bytes and operations that the pass cannot do without, `exact()` the pass's outputs in 64 bits.
A case is a dict of plain values; its "path" names the operator and the direction:

  attend       attention with a learned bias for each bucket of relative positions, no gradients
  attend_train the same with the gradients of queries, keys, values and bias table
  attend_token the same for a few queries a sequence against a long cache of keys and values
  norm_train   addition of the residual and root-mean-square norm, with their gradients
  norm_codes   the same for serving: the norm's rows in 8 bits with a scale each, read back
  adamw        one AdamW step over all tensors of a model, moments in 32 bits
  adamw8       the same step with both moments held in 8 bits, a scale for each 256 values
"""
import math
import os
import sys

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
OUTSIDE = 255                 # the bucket of pairs that do not attend
BLOCK = 256                   # values that share a scale of an 8-bit moment
SMALLEST = 2.0 ** -126        # a block whose largest value is smaller holds zeros
SMALLEST_ROW = 2.0 ** -100    # the same for a row in 8 bits
MAX_PAIRS = 16 * 8192 * 8192  # scores of a drawn case
MAX_FLOPS = 14 * 64 * MAX_PAIRS
RATE, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01


def listed():
    return [
        # The smallest attention: the 7 x 7 tokens of 24 tangent patches, each patch by itself,
        # one bucket for each offset; launches and host time count.
        dict(name="attend_patches_f16", path="attend", dtype="f16", batch=24, heads=4, groups=1,
             queries=49, keys=49, dim=32, buckets=169, map="sphere", reach=0, causal=False,
             ragged=False),
        # Features of two pictures on a 48 x 96 grid, buckets of great-circle distance.
        dict(name="attend_grid_48x96_bf16", path="attend", dtype="bf16", batch=2, heads=16,
             groups=1, queries=4608, keys=4608, dim=64, buckets=32, map="sphere", reach=0,
             causal=False, ragged=False),
        # A training step on a 64 x 128 grid, four query heads to a key head: the largest pass.
        dict(name="train_grid_64x128_bf16", path="attend_train", dtype="bf16", batch=1, heads=16,
             groups=4, queries=8192, keys=8192, dim=64, buckets=48, map="sphere", reach=0,
             causal=False, ragged=False),
        # Full precision, sizes that fill no tile, pairs out of reach, queries that see nothing,
        # pictures of different numbers of valid tokens.
        dict(name="train_ragged_f32", path="attend_train", dtype="f32", batch=3, heads=6,
             groups=3, queries=1237, keys=1931, dim=40, buckets=33, map="sphere", reach=120,
             causal=False, ragged=True),
        # Tokens generated in order, wide heads: a causal training step.
        dict(name="train_causal_f16", path="attend_train", dtype="f16", batch=4, heads=8,
             groups=2, queries=2048, keys=2048, dim=128, buckets=32, map="line", reach=0,
             causal=True, ragged=False),
        # Serving: one new token for each of 16 sequences of different lengths.
        dict(name="token_16x16384_bf16", path="attend_token", dtype="bf16", batch=16, heads=32,
             groups=4, queries=1, keys=16384, dim=128, buckets=32, map="line", reach=0,
             causal=True, ragged=True),
        # A block's norm while training: eight pictures of 64 x 128 tokens.
        dict(name="norm_train_65536x1024_bf16", path="norm_train", dtype="bf16", rows=65536,
             width=1024),
        # The smallest norm: one token for each of 16 sequences, rows in int8.
        dict(name="norm_token_16x4096_int8", path="norm_codes", dtype="bf16", rows=16, width=4096,
             codes="int8"),
        # Odd sizes in full precision, rows in 8-bit floating point.
        dict(name="norm_odd_9001x1003_fp8", path="norm_codes", dtype="f32", rows=9001, width=1003,
             codes="fp8"),
        # The step of three small convolution layers: six tensors, launches and host time count.
        dict(name="adamw_small_net", path="adamw", dtype="f32", model="convs", width=16, depth=3),
        # The step of a model of 12 blocks, 86 million parameters in 121 tensors.
        dict(name="adamw_86m", path="adamw", dtype="f32", model="blocks", width=768, depth=12),
        # The same model's step with moments in 8 bits.
        dict(name="adamw8_86m", path="adamw8", dtype="f32", model="blocks", width=768, depth=12),
    ]


# ----------------------------------------------------------------------------- drawn cases
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_attention(rng):
    path = rng.choice(["attend", "attend_train", "attend_token"])
    groups = rng.choice([1, 1, 2, 3, 4, 8])
    case = dict(path=path, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                batch=_log(rng, 1, 24), heads=groups * _log(rng, 1, 8), groups=groups,
                queries=_log(rng, 1, 8192), keys=_log(rng, 1, 8192),
                dim=rng.choice([32, 64, 64, 128, 8 * rng.randint(1, 16)]),
                buckets=_log(rng, 2, 250), map=rng.choice(["sphere", "line"]),
                reach=rng.choice([0, 0, 120]), causal=False, ragged=rng.random() < 0.4)
    if rng.random() < 0.5:
        case["keys"] = case["queries"]
    if path == "attend_token":
        case |= dict(queries=rng.choice([1, 1, 1, 2, 5]), keys=_log(rng, 16, 16384), map="line",
                     causal=True, reach=0)
    elif case["map"] == "line":
        case |= dict(causal=rng.random() < 0.5, reach=0)
    return case


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "norm", "norm", "adamw", "adamw8"])
    if kind == "attention":
        while True:
            case = _draw_attention(rng)
            pairs = case["batch"] * case["heads"] * case["queries"] * case["keys"]
            cells = case["queries"] * case["keys"] * case["buckets"]
            if (pairs <= MAX_PAIRS and work(case)["flops"] <= MAX_FLOPS
                    and (case["path"] != "attend_train" or cells <= 48 * 8192 * 8192)):
                return case
    if kind == "norm":
        width = _log(rng, 16, 16384)
        width = max(16, width // 8 * 8) if rng.random() < 0.7 else width
        rows = _log(rng, 1, min(65536, 65536 * 1024 // width))
        case = dict(path=rng.choice(["norm_train", "norm_codes"]),
                    dtype=rng.choice(["bf16", "f16", "f32"]), rows=rows, width=width)
        if case["path"] == "norm_codes":
            case["codes"] = rng.choice(["int8", "fp8"])
        return case
    return dict(path=kind, dtype=rng.choice(["f32", "f32", "bf16"]), model="blocks",
                width=_log(rng, 17, 768), depth=rng.randint(1, 12))


# ----------------------------------------------------------------------------- sizes and work
def _lengths(case):
    """Valid keys of each sequence, largest first."""
    n, batch = case["keys"], case["batch"]
    return [n - b * n // (2 * batch) for b in range(batch)] if case["ragged"] else [n] * batch


def _pairs(case):
    total = 0
    for n in _lengths(case):
        queries = case["queries"]
        if case["causal"]:          # the last query sees all n keys, each one before it one less
            most = min(queries, n)
            total += most * n - most * (most - 1) // 2
        else:
            total += queries * n
    return total * case["heads"]


def _shapes(case):
    width, depth = case["width"], case["depth"]
    if case["model"] == "convs":
        sizes = []
        for i in range(depth):
            sizes += [(width << i, width << (i - 1) if i else 3, 9), (width << i,)]
        return sizes
    sizes = [(width, 48)]
    for _ in range(depth):
        sizes += [(width,), (3 * width, width), (width, width), (width,), (4 * width, width),
                  (4 * width,), (width, 4 * width), (width,), (12, 33), (width,)]
    return sizes


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    path = case["path"]
    if path.startswith("attend"):
        batch, heads, dim = case["batch"], case["heads"], case["dim"]
        keys = sum(_lengths(case)) * heads // case["groups"]
        queries = batch * heads * case["queries"]
        pairs = _pairs(case)
        maps = (sum(_lengths(case)) if path == "attend_token" else case["keys"]) * case["queries"]
        passed = 2 * queries * dim + 2 * keys * dim          # queries, output; keys, values
        if path != "attend_train":
            return {"bytes": passed * size + maps, "flops": 4 * dim * pairs}
        return {"bytes": 2 * passed * size + maps, "flops": 14 * dim * pairs}
    if path == "norm_train":
        n = case["rows"] * case["width"]
        return {"bytes": 8 * n * size, "flops": 16 * n}
    if path == "norm_codes":
        n = case["rows"] * case["width"]
        return {"bytes": 3 * n * size + 2 * n + 4 * case["rows"], "flops": 8 * n}
    n = sum(math.prod(s) for s in _shapes(case))
    if path == "adamw":
        return {"bytes": n * (3 * size + 16), "flops": 15 * n}
    return {"bytes": n * (3 * size + 4 + 4), "flops": 40 * n}


# ----------------------------------------------------------------------------- inputs
def _points(count):
    """`count` directions spread over the sphere, from pole to pole."""
    i = torch.arange(count, device=DEVICE, dtype=torch.float64) + 0.5
    z = 1 - 2 * i / count
    turn = i * (math.pi * (3 - math.sqrt(5)))
    r = (1 - z * z).clamp(min=0).sqrt()
    return torch.stack([r * turn.cos(), r * turn.sin(), z], 1).float()


def _sphere_map(case):
    angle = (_points(case["queries"]) @ _points(case["keys"]).T).clamp(-1, 1).acos() / math.pi
    buckets = (angle.sqrt() * case["buckets"]).long().clamp(max=case["buckets"] - 1)
    if case["reach"]:
        buckets[angle * 180 > case["reach"]] = OUTSIDE
        buckets[3::97] = OUTSIDE                          # queries that see nothing
    return buckets.to(torch.uint8)


def _line_map(case, first):
    """Buckets of the distance between query positions first, first + 1, .. and key positions:
    half of them for one distance each, the others for ranges that grow."""
    at = first[..., None, None] + torch.arange(case["queries"], device=DEVICE)[:, None]
    far = (at - torch.arange(case["keys"], device=DEVICE)).abs()
    near = max(1, case["buckets"] // 2)
    grown = near + (far.clamp(min=near).double() / near).log2() * max(1, near // 7)
    return torch.where(far < near, far, grown.long()).clamp(max=case["buckets"] - 1).to(torch.uint8)


def _normal(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEVICE) * scale).to(dtype)


def _prepare_attention(case, g):
    batch, heads, dim, dtype = case["batch"], case["heads"], case["dim"], TYPES[case["dtype"]]
    shared = heads // case["groups"]
    state = dict(case=case)
    # as projections leave them, [batch, tokens, heads, dim]; a cache has its heads outside
    state["query"] = _normal(g, batch, case["queries"], heads, dim, dtype=dtype).transpose(1, 2)
    for name in ("key", "value"):
        if case["path"] == "attend_token":
            state[name] = _normal(g, batch, shared, case["keys"], dim, dtype=dtype)
        else:
            state[name] = _normal(g, batch, case["keys"], shared, dim, dtype=dtype).transpose(1, 2)
    state["table"] = _normal(g, heads, case["buckets"], dtype=dtype, scale=0.7)
    lengths = torch.tensor(_lengths(case), device=DEVICE)
    lengths = lengths[torch.randperm(batch, generator=g, device=DEVICE)]
    state["lengths"] = lengths.to(torch.int32) if case["ragged"] else None
    if case["map"] == "sphere":
        state["map"] = _sphere_map(case)
    elif case["path"] == "attend_token":
        state["map"] = _line_map(case, lengths - case["queries"])
    else:
        state["map"] = _line_map(case, torch.tensor(case["keys"] - case["queries"], device=DEVICE))
    if case["path"] == "attend_train":
        state["grad"] = _normal(g, batch, heads, case["queries"], dim, dtype=dtype)
        for name in ("query", "key", "value", "table"):
            state[name].requires_grad_()
    return state


def _prepare_norm(case, g):
    shape, dtype = (case["rows"], case["width"]), TYPES[case["dtype"]]
    state = dict(case=case, x=_normal(g, *shape, dtype=dtype), residual=_normal(g, *shape, dtype=dtype, scale=3.0),
                 weight=(1 + _normal(g, case["width"], scale=0.2)).to(dtype))
    if case["path"] == "norm_train":
        state["grad"] = _normal(g, *shape, dtype=dtype)
        state["grad_sum"] = _normal(g, *shape, dtype=dtype)
        for name in ("x", "residual", "weight"):
            state[name].requires_grad_()
    return state


def _prepare_step(case, g):
    """Parameters, gradients and moments: views of flat tensors in which each begins a block."""
    shapes, dtype = _shapes(case), TYPES[case["dtype"]]
    starts, total = [], 0
    for s in shapes:
        starts.append(total)
        total += -(-math.prod(s) // BLOCK) * BLOCK
    used = torch.zeros(total, device=DEVICE, dtype=torch.bool)
    for a, s in zip(starts, shapes):
        used[a:a + math.prod(s)] = True

    def parts(flat, each=1):
        return [flat[a // each:a // each + math.prod(s)].view(s) if each == 1
                else flat[a // each:(a + math.prod(s) + each - 1) // each]
                for a, s in zip(starts, shapes)]

    def filled(scale):
        return torch.where(used, torch.randn(total, generator=g, device=DEVICE) * scale, 0.0)

    state = dict(case=case, step=1000, params=filled(0.02).to(dtype),
                 grads=(filled(1e-3) * filled(1.0).exp()).to(dtype))
    avg, sq = filled(3e-4), (filled(1e-3) * filled(1.0).exp()).square()
    if case["path"] == "adamw":
        state |= dict(avg=avg, sq=sq, lists=[parts(state["params"]), parts(state["grads"]),
                                             parts(avg), parts(sq)])
    else:
        (ac, a_s), (sc, s_s) = _avg_codes(avg), _sq_codes(sq)
        state |= dict(avg_codes=ac, avg_scales=a_s, sq_codes=sc, sq_scales=s_s,
                      lists=[parts(state["params"]), parts(state["grads"]), parts(ac),
                             parts(a_s, BLOCK), parts(sc), parts(s_s, BLOCK)])
    return state


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    if case["path"].startswith("attend"):
        return _prepare_attention(case, g)
    return _prepare_norm(case, g) if case["path"].startswith("norm") else _prepare_step(case, g)


# ----------------------------------------------------------------------------- plain forms
def _scores(state):
    """Scores [batch, key heads, group, queries, keys], which of them count, and the float32
    operands with an axis for the group."""
    case = state["case"]
    batch, heads, groups = case["batch"], case["heads"], case["groups"]
    q = state["query"].detach().float().reshape(batch, heads // groups, groups, case["queries"], -1)
    k, v = (state[n].detach().float().unsqueeze(2) for n in ("key", "value"))
    buckets = state["map"].long()
    seen = buckets < case["buckets"]
    bias = state["table"].detach().float()[:, buckets.clamp(max=case["buckets"] - 1)]
    if buckets.dim() == 3:
        bias = bias.transpose(0, 1)
    else:
        bias, seen = bias.unsqueeze(0), seen.unsqueeze(0)
    at = torch.arange(case["keys"], device=DEVICE)
    end = torch.full((batch,), case["keys"], device=DEVICE) if state["lengths"] is None else state["lengths"].long()
    seen = seen & (at < end[:, None, None])
    if case["causal"]:
        last = end[:, None] - case["queries"] + torch.arange(case["queries"], device=DEVICE)
        seen = seen & (at <= last[:, :, None])
    seen = seen[:, None, None]
    s = (q @ k.transpose(-1, -2)).mul_(1 / math.sqrt(case["dim"]))
    s += bias.reshape(-1, heads // groups, groups, case["queries"], case["keys"])
    return s.masked_fill_(~seen, -math.inf), q, k, v


def _plain_attention(state):
    case, dtype = state["case"], state["query"].dtype
    s, q, k, v = _scores(state)
    most = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(most.isinf(), 0.0, most)).exp_()
    p /= p.sum(-1, keepdim=True).clamp(min=1e-30)
    out = p @ v
    shape = state["query"].shape
    if case["path"] != "attend_train":
        return out.reshape(shape).to(dtype)
    g = state["grad"].float().reshape(q.shape)
    dv = p.transpose(-1, -2) @ g
    ds = p * ((g @ v.transpose(-1, -2)) - (g * out).sum(-1, keepdim=True))
    scale = 1 / math.sqrt(case["dim"])
    dq, dk = (ds @ k) * scale, (ds.transpose(-1, -2) @ q) * scale
    # the gradient of the table: for each query, the row's sums by bucket
    rows = ds.reshape(shape[0], shape[1], shape[2], -1).sum(0).transpose(0, 1).contiguous()
    one = (state["map"][:, :, None] == torch.arange(case["buckets"], device=DEVICE, dtype=torch.uint8)).float()
    dt = (rows @ one).sum(0)
    return [out.reshape(shape).to(dtype), dq.reshape(shape).to(dtype), dk.sum(2).to(dtype),
            dv.sum(2).to(dtype), dt.to(state["table"].dtype)]


def _plain_norm(state):
    x, residual, weight = (state[n].detach().float() for n in ("x", "residual", "weight"))
    dtype, h = state["x"].dtype, x + residual
    inverse = (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    y = h * inverse * weight
    if state["case"]["path"] == "norm_train":
        g = state["grad"].float()
        gw = g * weight
        dh = inverse * (gw - h * inverse.square() * (gw * h).mean(-1, keepdim=True))
        dh = (dh + state["grad_sum"].float()).to(dtype)
        return [y.to(dtype), h.to(dtype), dh, dh, (g * h * inverse).sum(0).to(state["weight"].dtype)]
    most = 127.0 if state["case"]["codes"] == "int8" else 448.0
    largest = y.abs().amax(-1, keepdim=True)
    live = largest >= SMALLEST_ROW
    scaled = y * torch.where(live, most / largest, 0.0)
    codes = scaled.round() if state["case"]["codes"] == "int8" else scaled.to(torch.float8_e4m3fn).float()
    scales = torch.where(live, largest * (1 / most), 0.0)
    return [(codes * scales).to(torch.bfloat16), scales.squeeze(-1), h.to(dtype)]


def _avg_codes(x):
    blocks = x.view(-1, BLOCK)
    scale = blocks.abs().amax(1)
    scale = torch.where(scale >= SMALLEST, scale, 0.0)
    inverse = torch.where(scale > 0, 1 / scale, 0.0)[:, None]
    codes = ((blocks.abs() * inverse).sqrt() * 127.0).round() * blocks.sign()
    return codes.to(torch.int8).view(-1), scale


def _sq_codes(x):
    blocks = x.view(-1, BLOCK)
    scale = blocks.amax(1)
    scale = torch.where(scale >= SMALLEST, scale, 0.0)
    inverse = torch.where(scale > 0, 1 / scale, 0.0)[:, None]
    codes = ((blocks * inverse).sqrt().sqrt() * 255.0).round()
    codes = codes.maximum(((blocks > 0) & (inverse > 0)).float())
    return codes.to(torch.uint8).view(-1), scale


def _avg_values(codes, scale):
    a = codes.view(-1, BLOCK).float() * (1 / 127.0)
    return ((a * a.abs()) * scale[:, None]).view(-1)


def _sq_values(codes, scale):
    a = codes.view(-1, BLOCK).float() * (1 / 255.0)
    a = a * a
    return ((a * a) * scale[:, None]).view(-1)


def _plain_update(state, avg, sq):
    """Moments and parameters of one step, in float32, in the flat tensors' order."""
    state["step"] += 1
    g = state["grads"].float()
    avg = avg * BETA1 + g * (1 - BETA1)
    sq = sq * BETA2 + (g * g) * (1 - BETA2)
    below = sq.sqrt() * (1 / math.sqrt(1 - BETA2 ** state["step"])) + EPS
    p = state["params"].float() * (1 - RATE * DECAY)
    state["params"].copy_(p - (avg / below) * (RATE / (1 - BETA1 ** state["step"])))
    return avg, sq


def _plain_step(state):
    if state["case"]["path"] == "adamw":
        avg, sq = _plain_update(state, state["avg"], state["sq"])
        state["avg"].copy_(avg)
        state["sq"].copy_(sq)
        return [state["params"], state["avg"], state["sq"]]
    avg, sq = _plain_update(state, _avg_values(state["avg_codes"], state["avg_scales"]),
                            _sq_values(state["sq_codes"], state["sq_scales"]))
    (ac, a_s), (sc, s_s) = _avg_codes(avg), _sq_codes(sq)
    state["avg_codes"].copy_(ac)
    state["avg_scales"].copy_(a_s)
    state["sq_codes"].copy_(sc)
    state["sq_scales"].copy_(s_s)
    return [state["params"], _avg_values(ac, a_s).to(torch.bfloat16), _sq_values(sc, s_s).to(torch.bfloat16)]


# ----------------------------------------------------------------------------- the framework's calls
def _functional():
    package = os.path.join(os.getcwd(), "spherical-package_amd")
    if package not in sys.path:
        sys.path.insert(1, package)
    import spherical_distortion.functional as F
    return F


def _own_attention(state):
    F, case = _functional(), state["case"]
    out = F.bucket_attention(state["query"], state["key"], state["value"], state["table"],
                             state["map"], key_lengths=state["lengths"], causal=case["causal"])
    if case["path"] != "attend_train":
        return out
    return [out.detach(), *torch.autograd.grad(out, [state[n] for n in ("query", "key", "value", "table")],
                                               state["grad"])]


def _own_norm(state):
    F, case = _functional(), state["case"]
    if case["path"] == "norm_train":
        y, total = F.add_rms_norm(state["x"], state["residual"], state["weight"], eps=1e-6)
        grads = torch.autograd.grad([y, total], [state["x"], state["residual"], state["weight"]],
                                    [state["grad"], state["grad_sum"]])
        return [y.detach(), total.detach(), *grads]
    codes, scales, total = F.add_rms_norm_quantized(state["x"], state["residual"], state["weight"],
                                                    eps=1e-6, dtype=CODES[case["codes"]])
    return [F.dequantize_rows(codes, scales, dtype=torch.bfloat16), scales, total]


def _own_step(state):
    F = _functional()
    state["step"] += 1
    settings = dict(step=state["step"], lr=RATE, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY)
    if state["case"]["path"] == "adamw":
        F.adamw_step(*state["lists"], **settings)
        return [state["params"], state["avg"], state["sq"]]
    F.adamw_step_8bit(*state["lists"], **settings)
    return [state["params"],
            F.adamw_moment_values(state["avg_codes"], state["avg_scales"], dtype=torch.bfloat16),
            F.adamw_moment_values(state["sq_codes"], state["sq_scales"], dtype=torch.bfloat16)]


def run(state):
    path = state["case"]["path"]
    if path.startswith("attend"):
        return _own_attention(state) if own else _plain_attention(state)
    if path.startswith("norm"):
        return _own_norm(state) if own else _plain_norm(state)
    return _own_step(state) if own else _plain_step(state)


# ----------------------------------------------------------------------------- in 64 bits
def _exact_attention(state):
    """Head by head, from the definition: softmax of scale q k + bias[bucket] over the pairs that
    count, and the derivative of the output's product with the given gradient."""
    case = state["case"]
    batch, heads, groups, train = case["batch"], case["heads"], case["groups"], "grad" in state
    q, k, v, table = (state[n].detach().double() for n in ("query", "key", "value", "table"))
    out = torch.zeros_like(q)
    dq, dk, dv, dt = (torch.zeros_like(t) for t in (q, k, v, table))
    order = torch.arange(case["queries"], device=DEVICE)[:, None]
    for b in range(batch):
        buckets = (state["map"][b] if state["map"].dim() == 3 else state["map"]).long()
        end = case["keys"] if state["lengths"] is None else int(state["lengths"][b])
        buckets = buckets[:, :end]
        counts = buckets < case["buckets"]
        if case["causal"]:
            counts = counts & (torch.arange(end, device=DEVICE)[None] <= order + (end - case["queries"]))
        some = counts.any(1, keepdim=True)
        if train:   # the pairs in the order of their buckets, and where each bucket ends
            sorted_buckets, by_bucket = buckets.reshape(-1).sort(stable=True)
            ends = torch.searchsorted(sorted_buckets, torch.arange(case["buckets"], device=DEVICE), right=True)
        for h in range(heads):
            kh, vh = k[b, h // groups, :end], v[b, h // groups, :end]
            logits = (q[b, h] @ kh.T) / math.sqrt(case["dim"])
            logits = logits + table[h][buckets.clamp(max=case["buckets"] - 1)]
            logits = logits.where(counts, torch.tensor(-math.inf, device=DEVICE, dtype=torch.float64))
            weights = torch.where(some, logits, 0.0).softmax(1) * some
            out[b, h] = weights @ vh
            if train:
                g = state["grad"][b, h].double()
                dv[b, h // groups, :end] += weights.T @ g
                toward = g @ vh.T
                slope = weights * (toward - (weights * toward).sum(1, keepdim=True))
                dq[b, h] = slope @ kh / math.sqrt(case["dim"])
                dk[b, h // groups, :end] += slope.T @ q[b, h] / math.sqrt(case["dim"])
                upto = torch.zeros(end * case["queries"] + 1, device=DEVICE, dtype=torch.float64)
                torch.cumsum(slope.reshape(-1)[by_bucket], 0, out=upto[1:])
                dt[h] += upto[ends].diff(prepend=upto[:1])
    return [out, dq, dk, dv, dt] if train else out


def _exact_norm(state):
    case = state["case"]
    h = state["x"].detach().double() + state["residual"].detach().double()
    weight = state["weight"].detach().double()
    length = torch.sqrt(torch.sum(h * h, 1) / case["width"] + 1e-6)[:, None]
    unit = h / length
    y = unit * weight
    if case["path"] == "norm_train":
        g = state["grad"].double()
        along = torch.sum(g * weight * unit, 1)[:, None] / case["width"]
        dh = (g * weight - unit * along) / length + state["grad_sum"].double()
        return [y, h, dh, dh, torch.sum(g * unit, 0)]
    # the codes are roundings: only the scales and the sums have a value of their own
    return [None, y.abs().max(1).values / (127 if case["codes"] == "int8" else 448), h]


def _exact_step(state):
    g, p = state["grads"].double(), state["params"].double()
    if state["case"]["path"] == "adamw":
        m, v = state["avg"].double(), state["sq"].double()
    else:
        m = state["avg_codes"].double().view(-1, BLOCK) / 127
        m = (m.sign() * m ** 2 * state["avg_scales"].double()[:, None]).view(-1)
        v = (state["sq_codes"].double().view(-1, BLOCK) / 255) ** 4
        v = (v * state["sq_scales"].double()[:, None]).view(-1)
    m, v, t = BETA1 * m + (1 - BETA1) * g, BETA2 * v + (1 - BETA2) * g ** 2, state["step"] + 1
    p = p - RATE * DECAY * p - RATE * (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + EPS)
    return [p, m, v] if state["case"]["path"] == "adamw" else [p, None, None]


def exact(case, seed):
    state = prepare(case, seed)
    if case["path"].startswith("attend"):
        return _exact_attention(state)
    return _exact_norm(state) if case["path"].startswith("norm") else _exact_step(state)
