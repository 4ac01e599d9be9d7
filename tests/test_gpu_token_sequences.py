"""Layer norm, the gated scan, Newton-Schulz and Muon as their users have them: the compiled and the Python implementation
of each against each other, derivatives that raise, streams, graphs, sizes beyond 2^31, and a run of them together."""
import copy

import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NS = (3.4445, -4.7750, 2.0315)


def _randn(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed + sum(shape))
    return torch.randn(*shape, generator=g).to(dtype).to(DEV)


def _both(name, *args):
    from _spherical_distortion_ext import _token_ops
    assert name in _token_ops.NATIVE_OPS
    a, b = getattr(_token_ops.ops, name)(*args), _token_ops.PYTHON_IMPL[name](*args)
    one = not isinstance(a, (tuple, list))
    for x, y in zip([a] if one else a, [b] if one else b):
        assert x.shape == y.shape and x.dtype == y.dtype and x.stride() == y.stride()
        assert torch.equal(x, y)
    return a


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_compiled_and_python_operators_agree(dtype):
    from _spherical_distortion_ext import _token_ops
    x, r, dy, ds = (_randn(20, 100, seed=i, dtype=dtype) for i in range(4))
    w, b = _randn(100, seed=4), _randn(100, seed=5)
    for residual in (r, None):
        for bias in (b, None):
            y, s, mean, inverse = _both("add_layer_norm", x, residual, w, bias, 1e-5)
        _both("layer_norm_pair", x, residual, w, b, 1e-5)
        for needs in ((True, True, True), (True, False, False), (False, True, False), (False, False, True)):
            for grad_sum in (ds, None):
                _both("add_layer_norm_backward", dy, grad_sum, x, residual, w, mean, inverse, *needs)
    for shape in ((2, 700, 40), (3, 6, 8), (2, 0, 8)):
        B, L, D = shape
        wide = _randn(B, L, 3 * D, dtype=dtype)
        x, gate, dy = wide.chunk(3, -1)
        state, dl = _randn(B, D, seed=1), _randn(B, D, seed=2)
        n = torch.tensor([L, L // 2, 0][:B], dtype=torch.int32, device=DEV)
        for args in ((state, n, False), (None, None, True), (state, None, False)):
            out, last = _both("gated_scan_forward", x, gate, *args)
            _both("gated_scan", x, gate, *args)
            for grads in ((dy, dl), (dy, None), (None, dl)):
                for needs in ((True, True, True), (True, False, False), (False, True, False), (False, False, True)):
                    _both("gated_scan_backward", *grads, x, gate, args[0], args[1], out, args[2], *needs)
    x, gate, state = _randn(5, 24, dtype=dtype), _randn(5, 24, seed=1, dtype=dtype), _randn(5, 24, seed=2)
    other = state.clone()
    assert torch.equal(_token_ops.ops.gated_scan_step(x, gate, state), _token_ops.PYTHON_IMPL["gated_scan_step"](x, gate, other))
    assert torch.equal(state, other)
    _both("orthogonalize", _randn(3, 70, 40, dtype=dtype), 5, list(NS), 1e-7)
    lists = [[_randn(*s, seed=i, dtype=d) for s in ((130, 20), (6, 3, 9))] for i, d in ((0, dtype), (1, dtype), (2, torch.float32))]
    twins = copy.deepcopy(lists)
    settings = (0.1, 0.9, True, 0.01, 5, list(NS), 1e-7)
    _token_ops.ops.muon_step(*lists, *settings)
    _token_ops.PYTHON_IMPL["muon_step"](*twins, *settings)
    assert all(torch.equal(a, b) for x, y in zip(lists, twins) for a, b in zip(x, y))


def test_python_operators_refuse_what_the_compiled_ones_refuse():
    from _spherical_distortion_ext import _token_ops
    x, w, s = torch.randn(3, 8, device=DEV), torch.ones(8, device=DEV), torch.zeros(3, 8, device=DEV)
    t = x[:, None]
    ns = (5, list(NS), 1e-7)
    bad = [("add_layer_norm", (x, x[:2], w, None, 1e-5)), ("add_layer_norm", (x, None, w[:4], None, 1e-5)),
           ("add_layer_norm", (x, None, w, w.half(), 1e-5)), ("add_layer_norm", (x, None, w, w, -1.0)),
           ("add_layer_norm", (x.double(), None, w, w, 1e-5)),
           ("add_layer_norm_backward", (x, None, x[:2], None, w, s[:, 0].contiguous(), s[:, 0].contiguous(), True, True, True)),
           ("add_layer_norm_backward", (x.half(), None, x, None, w, s[:, 0].contiguous(), s[:, 0].contiguous(), True, True, True)),
           ("gated_scan_forward", (t, t[:2], None, None, False)), ("gated_scan_forward", (t, t, s[:2], None, False)),
           ("gated_scan_forward", (t, t, s.half(), None, False)), ("gated_scan_forward", (x, x, None, None, False)),
           ("gated_scan_backward", (t, s.half(), t, t, None, None, t, False, True, True, True)),
           ("gated_scan_backward", (t[:2], s, t, t, None, None, t, False, True, True, True)),
           ("gated_scan_step", (x, x, s[:2])), ("gated_scan_step", (x, x.half(), s)), ("gated_scan_step", (x, x, s.half())),
           ("orthogonalize", (w, *ns)), ("orthogonalize", (x.double(), *ns)), ("orthogonalize", (x, 0, list(NS), 1e-7)),
           ("orthogonalize", (x, 5, [1.0, 2.0], 1e-7)), ("orthogonalize", (x, 5, [20.0, 0.0, 0.0], 1e-7)),
           ("muon_step", ([x], [x.half()], [s], 0.1, 0.9, True, 0.0, *ns)),
           ("muon_step", ([w], [w], [w], 0.1, 0.9, True, 0.0, *ns)), ("muon_step", ([], [x], [], 0.1, 0.9, True, 0.0, *ns)),
           ("muon_step", ([x, x], [s, s], [s.clone(), s.clone()], 0.1, 0.9, True, 0.0, *ns)),
           ("muon_step", ([x], [s], [s], 0.1, 0.9, True, 0.0, *ns))]
    before = x.clone()
    for name, args in bad:
        for fn in (getattr(_token_ops.ops, name), _token_ops.PYTHON_IMPL[name]):
            with pytest.raises(RuntimeError):
                fn(*args)
    assert torch.equal(x, before) and not bool(s.any())


def _forms():
    """name -> (differentiable inputs, function of them that returns a list of outputs)."""
    from _spherical_distortion_ext import _token_ops
    from spherical_distortion import functional as F
    x, r, w, b = _randn(4, 16), _randn(4, 16, seed=1), _randn(16, seed=2), _randn(16, seed=3)
    t, gate, state = _randn(2, 40, 16), _randn(2, 40, 16, seed=1), _randn(2, 16)
    n = torch.tensor([40, 13], dtype=torch.int32, device=DEV)
    forms = {}
    for kind, norm, scan in (("public", F.add_layer_norm, F.gated_scan),
                             ("operator", _token_ops.ops.layer_norm_pair, _token_ops.ops.gated_scan),
                             ("python", F.AddLayerNormFunction.apply, F.GatedScanFunction.apply)):
        forms[kind + " norm"] = [x, r, w, b], lambda a, c, u, v, norm=norm: list(norm(a, c, u, v, 1e-5))
        forms[kind + " norm alone"] = [x, w], lambda a, u, norm=norm: list(norm(a, None, u, None, 1e-5))[:1]
        forms[kind + " sum alone"] = [x, r, w, b], lambda a, c, u, v, norm=norm: [norm(a, c, u, v, 1e-5)[1]]
        forms[kind + " scan"] = [t, gate, state], lambda a, c, s, scan=scan: list(scan(a, c, s, n, True))
        forms[kind + " scan alone"] = [t, gate], lambda a, c, scan=scan: [scan(a, c, None, None, False)[0]]
    return forms


PARTS = (" norm", " norm alone", " sum alone", " scan", " scan alone")
NAMES = [kind + what for kind in ("public", "operator", "python") for what in PARTS]


@pytest.mark.parametrize("what", PARTS)
def test_all_forms_have_the_same_gradients(what):
    """Compiled and Python autograd functions: the same bits, and gradients only where wanted."""
    forms = _forms()
    inputs = forms["public" + what][0]
    for wanted in [[True] * len(inputs)] + [[i == j for j in range(len(inputs))] for i in range(len(inputs))]:
        results = []
        for kind in ("public", "operator", "python"):
            leaves = [t.clone().requires_grad_(want) for t, want in zip(inputs, wanted)]
            outs = forms[kind + what][1](*leaves)
            sum((o * (i + 1)).square().sum() for i, o in enumerate(outs)).backward()
            assert all(t.grad is None for t, want in zip(leaves, wanted) if not want)
            results.append([o.detach() for o in outs] + [t.grad for t in leaves if t.grad is not None])
        for other in results[1:]:
            assert len(other) == len(results[0]) and all(torch.equal(a, b) for a, b in zip(results[0], other))


@pytest.mark.parametrize("name", NAMES)
def test_second_derivatives_raise_beside_terms_that_have_one(name):
    inputs, fn = _forms()[name]
    leaves = [t.clone().requires_grad_() for t in inputs]
    outs = fn(*leaves)
    grads = torch.autograd.grad(sum(o.sum() for o in outs), leaves, create_graph=True, allow_unused=True)
    for g in grads:
        if g is not None:
            assert g.requires_grad
            with pytest.raises(RuntimeError):
                (g.square().sum() + sum(o.sum() for o in outs) + leaves[0].sum()).backward(retain_graph=True)


@pytest.mark.parametrize("name", [n for n in NAMES if not n.startswith("python")])
def test_forward_mode_raises(name):
    inputs, fn = _forms()[name]
    for i in range(len(inputs)):
        for grad_mode in (True, False):
            with fwd.dual_level(), torch.set_grad_enabled(grad_mode):
                dual = [fwd.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(inputs)]
                with pytest.raises((RuntimeError, NotImplementedError)):
                    fn(*dual)


def test_one_tensor_in_several_places():
    """A row added to itself, and a gate that is its own input: the gradient is the sum of both places'."""
    from spherical_distortion import functional as F
    x, w, dy = _randn(6, 40), _randn(40), _randn(6, 40, seed=1)
    pair = [x.clone().requires_grad_() for _ in range(2)]
    want = torch.autograd.grad(F.add_layer_norm(*pair, w)[0], pair, dy)
    leaf = x.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(F.add_layer_norm(leaf, leaf, w)[0], leaf, dy)[0], want[0] + want[1])
    t, dt = _randn(2, 50, 8), _randn(2, 50, 8, seed=1)
    pair = [t.clone().requires_grad_() for _ in range(2)]
    want = torch.autograd.grad(F.gated_scan(*pair)[0], pair, dt)
    leaf = t.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(F.gated_scan(leaf, leaf)[0], leaf, dt)[0], want[0] + want[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_parameters_in_one_buffer(dtype):
    """Muon on views at any address of flat buffers: what copies give, and nothing beside them changes.  Tiles, lines and sums
    are the same, so the bits are too."""
    from spherical_distortion import functional as F
    shapes = [(7, 9), (64, 31), (100, 201), (130, 129), (5, 3, 9)]
    sizes = [torch.Size(s).numel() for s in shapes]
    flat = [torch.full((sum(sizes) + 2 * len(sizes) + 1,), 7.0, dtype=d, device=DEV) for d in (dtype, dtype, torch.float32)]
    lists, at = [[], [], []], 1
    for i, (shape, n) in enumerate(zip(shapes, sizes)):
        for to, buffer in zip(lists, flat):
            to.append(buffer[at:at + n].view(shape))
            to[-1].copy_(_randn(*shape, seed=len(to)))
        at += n + 2
    twins = [[t.clone() for t in ts] for ts in lists]
    F.muon_step(*lists, lr=0.1, weight_decay=0.1)
    F.muon_step(*twins, lr=0.1, weight_decay=0.1)
    for ts, us in zip(lists, twins):
        assert all(torch.equal(t, u) for t, u in zip(ts, us))
    for buffer in flat:
        at = 0
        for n in sizes:
            assert float(buffer[at]) == 7
            at += n + 1
            assert float(buffer[at]) == 7
            at += 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_what_a_backward_reads_must_not_change_before_it(dtype):
    from spherical_distortion import functional as F
    x, r = (_randn(4, 16, seed=i, dtype=dtype) for i in range(2))
    w = _randn(16).requires_grad_()
    y, h = F.add_layer_norm(x, r, w)
    (h if dtype == torch.float32 else r).add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    x, state = _randn(2, 5, 16, dtype=dtype).requires_grad_(), _randn(2, 16)
    out, _ = F.gated_scan(x, x.detach(), state)
    F.gated_scan_step(x[:, 0].detach(), x[:, 0].detach(), state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_inference_tensors():
    from spherical_distortion import functional as F
    from spherical_distortion.optim import Muon
    with torch.inference_mode():
        x, w = _randn(2, 9, 16), torch.ones(16, device=DEV)
        y, h = F.add_layer_norm(x, x, w)
        out, last = F.gated_scan(y, h)
        F.gated_scan_step(y[:, 0], h[:, 0], last)
        p = _randn(6, 5)
        F.muon_step([p], [_randn(6, 5, seed=1)], [torch.zeros(6, 5, device=DEV)])
        assert bool(torch.stack([t.isfinite().all() for t in (out, last, p, F.orthogonalize(p))]).all())
    q = torch.nn.Parameter(_randn(6, 5))
    q.grad = _randn(6, 5, seed=1)
    with torch.inference_mode():
        Muon([q]).step()


# --------------------------------------------------------------------------- streams and graphs
def _work(dtype):
    """name -> (tensors that may be given new values, function that returns fresh tensors or the changed ones)."""
    from spherical_distortion import functional as F
    x, r, dy, ds = (_randn(300, 104, seed=i, dtype=dtype) for i in range(4))
    w, b = _randn(104, seed=4), _randn(104, seed=5)
    t, gate, dt = (_randn(2, 3000, 40, seed=i, dtype=dtype) for i in range(3))
    state, dl = _randn(2, 40, seed=7), _randn(2, 40, seed=8)
    n = torch.tensor([3000, 1234], dtype=torch.int32, device=DEV)
    one, one_gate = _randn(30, 40, dtype=dtype), _randn(30, 40, seed=1, dtype=dtype)
    held = _randn(30, 40, seed=2)
    shapes = ((16, 3, 9), (40, 30), (130, 200), (300, 70))
    params, grads = ([_randn(*s, seed=i, dtype=dtype) for s in shapes] for i in range(2))
    momenta = [_randn(*s, seed=2) for s in shapes]
    stack = _randn(3, 100, 150, dtype=dtype)

    def norm():
        leaves = [u.detach().requires_grad_() for u in (x, r, w, b)]
        y, h = F.add_layer_norm(*leaves)
        return [y.detach(), h.detach(), *torch.autograd.grad([y, h], leaves, [dy, ds])]

    def scan():
        leaves = [u.detach().requires_grad_() for u in (t, gate, state)]
        out, last = F.gated_scan(*leaves, n)
        return [out.detach(), last.detach(), *torch.autograd.grad([out, last], leaves, [dt, dl])]

    def step():
        return [F.gated_scan_step(one, one_gate, held), held]

    def muon():
        F.muon_step(params, grads, momenta, lr=0.01, weight_decay=0.1)
        return params + momenta

    def orthogonal():
        return [F.orthogonalize(stack)]
    return {"norm": ([x, r, w, b, dy, ds], norm), "scan": ([t, gate, state, dt, dl], scan),
            "step": ([one, one_gate, held], step), "muon": (params + grads + momenta, muon),
            "orthogonal": ([stack], orthogonal)}


WORK = ["norm", "scan", "step", "muon", "orthogonal"]


def _fresh(tensors, seed):
    with torch.no_grad():
        for i, t in enumerate(tensors):
            t.copy_(_randn(*t.shape, seed=seed + i))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", WORK)
def test_another_stream(name, dtype):
    tensors, run = _work(dtype)[name]
    _fresh(tensors, 1)
    want = [t.clone() for t in run()]
    _fresh(tensors, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [t.clone() for t in run()]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams_at_once():
    """Scans whose tiles wait for each other, norms and steps on two streams at the same time: the bits of one after another."""
    works = [_work(torch.bfloat16), _work(torch.bfloat16)]
    want = {name: [t.clone() for t in works[0][name][1]()] for name in ("norm", "scan", "orthogonal")}
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in works], [[], []]
    for _ in range(5):
        for work, stream, result in zip(works, streams, results):
            with torch.cuda.stream(stream):
                result.append({name: work[name][1]() for name in want})
    torch.cuda.synchronize()
    for result in results:
        for got in result:
            for name in want:
                assert all(torch.equal(a, b) for a, b in zip(got[name], want[name])), name


def test_a_backward_may_run_twice():
    from spherical_distortion import functional as F
    x, gate, w = _randn(2, 700, 16).requires_grad_(), _randn(2, 700, 16, seed=1).requires_grad_(), _randn(16).requires_grad_()
    y, h = F.add_layer_norm(x, gate, w)
    out, last = F.gated_scan(y, h)
    first, second = (torch.autograd.grad([out.sum(), last.sum()], [x, gate, w], retain_graph=keep) for keep in (True, False))
    assert all(torch.equal(a, c) for a, c in zip(first, second))


def test_one_row():
    """A vector is a row; float32 weights get float32 gradients beside 16-bit rows."""
    from spherical_distortion import functional as F
    for dtype in (torch.float32, torch.float16):
        x, w, b, dy = _randn(40, dtype=dtype), _randn(40, seed=1), _randn(40, seed=2), _randn(40, seed=3, dtype=dtype)
        results = []
        for shape in ((40,), (1, 40), (1, 1, 1, 40)):
            leaves = [x.view(shape).clone().requires_grad_(), w.clone().requires_grad_(), b.clone().requires_grad_()]
            y, h = F.add_layer_norm(leaves[0], None, *leaves[1:])
            assert y.shape == shape and h is leaves[0]
            grads = torch.autograd.grad(y, leaves, dy.view(shape))
            assert grads[1].dtype == grads[2].dtype == torch.float32
            results.append([t.flatten() for t in (y, *grads)])
        for other in results[1:]:
            assert all(torch.equal(a, c) for a, c in zip(results[0], other))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", WORK)
def test_two_graphs(name, dtype):
    """Two captures of the same work on tensors of their own, replayed in turn with new values and eager calls between: the
    bits of the eager calls each time."""
    works = [_work(dtype)[name] for _ in range(2)]
    eager = _work(dtype)[name]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager[1]()
    torch.cuda.current_stream().wait_stream(side)
    graphs, captured = [], []
    for tensors, run in works:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured.append(run())
        graphs.append(graph)
    for seed in (30, 60, 90):
        for which in (0, 1):
            _fresh(works[which][0], seed + which)
        torch.cuda.synchronize()
        for which in (0, 1):
            graphs[which].replay()
        for which in (1, 0):
            _fresh(eager[0], seed + which)
            want = eager[1]()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(captured[which], want))


# --------------------------------------------------------------------------- sizes
def _room(gib):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip("needs %d GiB of free GPU memory" % gib)


def test_norm_rows_beyond_a_launch():
    """More rows of one vector than a launch takes: the bits of calls on parts."""
    from spherical_distortion import functional as F
    _room(60)
    rows, width, cut = (1 << 30) + 1000, 8, ((1 << 32) - 1) // 256 * 64
    assert cut < rows
    x = _randn(1 << 16, width, dtype=torch.bfloat16).repeat(-(-rows // (1 << 16)), 1)[:rows]
    w = _randn(width)
    with torch.no_grad():
        y, _ = F.add_layer_norm(x, None, w)
        for part in (slice(0, 70), slice(cut - 70, cut + 70), slice(rows - 70, rows)):
            assert torch.equal(y[part], F.add_layer_norm(x[part], None, w)[0])


def test_norm_offsets_beyond_2_to_31():
    """Values at offsets beyond 2^31, forward and backward, of a width that fits no vector."""
    from spherical_distortion import functional as F
    _room(40)
    rows, width = (1 << 19) + 9, 4099
    x = torch.randn(1 << 12, width, device=DEV).half().repeat(129, 1)[:rows]
    assert x.shape[0] == rows and x.numel() > 1 << 31
    w, part = _randn(width), slice(rows - 5, rows)
    leaf = x.detach().requires_grad_()
    y, _ = F.add_layer_norm(leaf, None, w)
    dx, = torch.autograd.grad(y, leaf, x)
    few = x[part].clone().requires_grad_()
    z, _ = F.add_layer_norm(few, None, w)
    dz, = torch.autograd.grad(z, few, x[part])
    assert torch.equal(y[part], z) and torch.equal(dx[part], dz)


def test_scan_strides_beyond_2_to_31():
    """Tokens that lie 2^26 values from each other: the bits of the same tokens laid out."""
    from spherical_distortion import functional as F
    _room(24)
    big = torch.zeros(50 << 26, dtype=torch.bfloat16, device=DEV)
    views = [big.as_strided((2, 49, 24), (200, 1 << 26, 1), at) for at in (8, 1000)]
    dense = [_randn(2, 49, 24, seed=i, dtype=torch.bfloat16) for i in range(2)]
    for v, d in zip(views, dense):
        v.copy_(d)
    dy = dense[1]
    results = []
    for x, gate in (views, dense):
        leaves = [x.detach().requires_grad_(), gate.detach().requires_grad_()]
        out, last = F.gated_scan(*leaves)
        results.append([out, last, *torch.autograd.grad(out, leaves, dy)])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_scans_of_more_sequences_than_a_launch():
    """More sequences than a launch has workgroups; and more tiles, which then go one after the other."""
    from spherical_distortion import functional as F
    _room(60)
    batch, each = (1 << 24) + 2100, ((1 << 32) - 1) // 256
    x = _randn(1 << 12, 33, 1, dtype=torch.bfloat16).repeat(4098, 1, 1)[:batch].contiguous()
    assert x.shape[0] == batch > each
    leaf = x.detach().requires_grad_()
    out, last = F.gated_scan(leaf, x)
    dx, = torch.autograd.grad(out, leaf, x)
    for part in (slice(0, 2000), slice(each - 1000, each + 1000), slice(batch - 2000, batch)):
        few = x[part].clone().requires_grad_()
        a, b = F.gated_scan(few, x[part])
        c, = torch.autograd.grad(a, few, x[part])
        assert torch.equal(out[part], a) and torch.equal(last[part], b) and torch.equal(dx[part], c)
    del out, last, dx, leaf, x
    x = _randn(1000, 9000, 1, dtype=torch.bfloat16).repeat(1, 1000, 1)
    gate = torch.full((1, 1, 1), 1.5, dtype=torch.bfloat16, device=DEV).expand_as(x)
    out, _ = F.gated_scan(x, gate)
    for part in (slice(0, 1), slice(998, 1000)):
        a, _ = F.gated_scan(x[part], gate[part])
        # the same states by sums in another order, 5 tokens' memory: 32 roundings in 32 bits, and each rounded to bfloat16
        d = (out[part].float() - a.float()).abs()
        assert bool((d <= 2.0 ** -7 * a.float().abs() + 32 * 2.0 ** -24 * 6).all())


def test_a_matrix_of_gigabytes():
    """Buffers beyond 2^32 bytes.  The matrix has rank 4, so that its result is known: each singular value by itself.  The
    matrix itself is rounded: 2^-24 of each value; pieces of 22 bits, 3 roundings of a step: 4e-6 in all."""
    from spherical_distortion import functional as F
    _room(40)
    k, l = 12001, 100003
    g = torch.Generator(device=DEV).manual_seed(1)
    u, v = (torch.linalg.qr(torch.randn(n, 4, generator=g, device=DEV, dtype=torch.float64))[0] for n in (k, l))
    s = torch.tensor([4.0, 3.0, 2.0, 1.0], device=DEV, dtype=torch.float64)
    x = (u * s).float() @ v.t().float()
    got = F.orthogonalize(x, steps=1, coefficients=(1.5, -0.5, 0.0))
    del x
    n = s / s.norm()
    n = 1.5 * n - 0.5 * n ** 3
    for rows in (slice(0, 500), slice(k - 500, k)):
        want = (u[rows] * n) @ v.t()
        # the rows of u and v in 32 bits and their product's sum of four: 6 roundings of 2^-24 more
        assert float((got[rows].double() - want).norm()) <= 5e-6 * float(want.norm())


@pytest.mark.parametrize("shape", [(3, 240), (3, 428), (412, 4), (34, 1855), (40, 1834), (64, 300), (400, 4000)])
def test_bfloat16_matrices_of_few_long_rows(shape):
    """Rows that are nearly orthogonal to each other: S and P are nearly diagonal, and their roundings weigh whole rows.

    The result's own rounding is 2^-8 / sqrt(3) = 2.3e-3 at most in the root of the mean square.  X is rounded to 11 bits in
    each step, 2^-11 / sqrt(3), which a step multiplies by 1.3 at most where singular values have arrived (0.68 to 1.14):
    sqrt(1 + 1.3^2 + .. + 1.3^8) = 4.3 of them, 1.2e-3.  Together 2.6e-3; 2^-8 leaves half as much again."""
    from spherical_distortion import functional as F
    x = _randn(*shape, dtype=torch.bfloat16)
    y = x.double()
    y = y.t() if shape[0] > shape[1] else y
    y = y / (y.norm() + 1e-7)
    for _ in range(5):
        s = y @ y.t()
        y = NS[0] * y + (NS[1] * s + NS[2] * (s @ s)) @ y
    y = y.t() if shape[0] > shape[1] else y
    assert float((F.orthogonalize(x).double() - y).norm()) <= 2.0 ** -8 * float(y.norm())


@pytest.mark.parametrize("shape", [(1, 1), (1, 700), (16, 16), (17, 5), (3, 1000), (2050, 16), (16, 4096), (11, 4097), (9, 20000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_matrices_of_few_rows(shape, dtype):
    """Up to 16 rows or columns.  The steps are 64 bits where they go by S alone: the result's rounding, half a step of each value.
    Longer ones in bfloat16 (4097 and 20000) go through products of 11 bits: 2^-8 again."""
    from spherical_distortion import functional as F
    x = _randn(2, *shape, dtype=dtype)
    x[1] *= 1e-2
    got = F.orthogonalize(x)
    for i in range(2):
        y = x[i].double()
        y = y.t() if shape[0] > shape[1] else y
        y = y / (y.norm() + 1e-7)
        for _ in range(5):
            s = y @ y.t()
            y = NS[0] * y + (NS[1] * s + NS[2] * (s @ s)) @ y
        y = y.t() if shape[0] > shape[1] else y
        off = (got[i].double() - y).abs()
        if dtype == torch.bfloat16 and max(shape) > 4096:
            assert float(off.norm()) <= 2.0 ** -8 * float(y.norm())
        else:
            # eps is rounded to 32 bits, beside norms of 1e-2 and more: 1e-12; float16 values below 2^-14 by halves of 2^-24
            u = torch.finfo(dtype).eps / 2
            assert bool((off <= u * (1 + 1e-3) * y.abs() + 1e-9 + (2.0 ** -25 if dtype == torch.float16 else 0)).all())


def test_singular_values_far_apart():
    """Of 1 to 1e-4 of the largest, in few rows: squares of 1e-8 keep eight digits of 64 bits.  The matrix's own rounding to 32
    bits (2^-24 of the largest beside 1e-4 of it) is in the oracle's input too; 2^-24 of the result is its rounding."""
    from spherical_distortion import functional as F
    g = torch.Generator().manual_seed(5)
    u, v = (torch.linalg.qr(torch.randn(n, 8, generator=g, dtype=torch.float64))[0] for n in (8, 500))
    x = ((u * torch.logspace(0, -4, 8, dtype=torch.float64)) @ v.t()).float().to(DEV)
    y = x.double()
    y = y / (y.norm() + 1e-7)
    for _ in range(5):
        s = y @ y.t()
        y = NS[0] * y + (NS[1] * s + NS[2] * (s @ s)) @ y
    assert float((F.orthogonalize(x).double() - y).norm()) <= 2.0 ** -24 * float(y.norm()) * 1.001


# --------------------------------------------------------------------------- together
class _Block(torch.nn.Module):
    """Norm with residual, gated scan, norm with residual, two linear layers."""

    def __init__(self, width):
        super().__init__()
        from spherical_distortion import nn as snn
        self.norm1, self.norm2 = snn.AddLayerNorm(width), snn.AddLayerNorm(width)
        self.scan = snn.GatedScan(width, 2 * width)
        self.up, self.down = torch.nn.Linear(width, 3 * width), torch.nn.Linear(3 * width, width)

    def forward(self, x, residual, state, lengths=None, one=False):
        y, residual = self.norm1(x, residual)
        y, state = (self.scan.step(y, state), state) if one else self.scan(y, state, lengths)
        y, residual = self.norm2(y, residual)
        return self.down(torch.nn.functional.gelu(self.up(y))), residual, state


class _Net(torch.nn.Module):
    def __init__(self, width=24, outputs=5):
        super().__init__()
        from spherical_distortion import nn as snn
        self.blocks = torch.nn.ModuleList(_Block(width) for _ in range(2))
        self.norm, self.head = snn.AddLayerNorm(width, bias=False), torch.nn.Linear(width, outputs)

    def forward(self, x, states=None, lengths=None, one=False):
        residual, kept = None, []
        for i, block in enumerate(self.blocks):
            x, residual, state = block(x, residual, None if states is None else states[i], lengths, one)
            kept.append(state)
        return self.head(self.norm(x, residual)[0]), kept


def _plain(net, x):
    """The network in the types of its parameters by torch's own operations, on the CPU."""
    f = torch.nn.functional
    norm = lambda m, t: f.layer_norm(t, t.shape[-1:], m.weight, m.bias, m.eps)  # noqa: E731
    total = torch.zeros_like(x)
    for block in net.blocks:
        total = total + x
        u, gate, z = block.scan.inputs(norm(block.norm1, total)).chunk(3, -1)
        keep, h, hs = torch.sigmoid(gate), torch.zeros_like(u[:, 0]), []
        for t in range(x.shape[1]):
            h = keep[:, t] * h + (1 - keep[:, t]) * u[:, t]
            hs.append(h)
        total = total + block.scan.out(torch.stack(hs, 1) * f.silu(z))
        x = block.down(f.gelu(block.up(norm(block.norm2, total))))
    return net.head(norm(net.norm, total + x))


def test_a_network_trains_and_serves():
    """Two blocks: gradients against float64; steps by Muon (matrices) and AdamW (the rest); then served token by token.

    Float32 throughout: about a dozen operators in a row, whose sums of up to 72 values are off by at most 72 * 2^-24 of
    their terms: 5e-5 of sizes of order one, twice that for gradients, which pass them again."""
    from spherical_distortion.optim import AdamW, Muon
    torch.manual_seed(0)
    net = _Net().to(DEV)
    x, goal = _randn(3, 70, 24), _randn(3, 70, 5, seed=1)
    exact = copy.deepcopy(net).double().cpu()
    loss = (net(x)[0] - goal).square().mean()
    loss.backward()
    want = (_plain(exact, x.double().cpu()) - goal.double().cpu()).square().mean()
    want.backward()
    assert abs(loss.item() - want.item()) <= 5e-5 * want.item()
    for (name, p), q in zip(net.named_parameters(), exact.parameters()):
        off = (p.grad.double().cpu() - q.grad).norm()
        assert float(off) <= 1e-4 * float(q.grad.norm()) + 1e-7, name
    matrices = [p for p in net.parameters() if p.dim() > 1]
    others = [p for p in net.parameters() if p.dim() < 2]
    optimizers = [Muon(matrices, lr=0.02, weight_decay=0.01), AdamW(others, lr=1e-3)]
    before = [p.detach().clone() for p in net.parameters()]
    for _ in range(3):
        for o in optimizers:
            o.step()
            o.zero_grad()
        (net(x)[0] - goal).square().mean().backward()
    for p, q in zip(net.parameters(), before):
        assert bool(p.isfinite().all()) and not torch.equal(p, q)
    net.eval()
    with torch.no_grad():
        whole, last = net(x)
        out, states = net(x[:, :30].contiguous())
        assert float((out - whole[:, :30]).abs().max()) <= 5e-5 * max(1.0, float(whole.abs().max()))
        for t in range(30, 70):
            one, states = net(x[:, t].contiguous(), states, one=True)
            assert float((one - whole[:, t]).abs().max()) <= 5e-5 * max(1.0, float(whole.abs().max()))
        for a, b in zip(states, last):
            assert float((a - b).abs().max()) <= 5e-5 * max(1.0, float(b.abs().max()))
        # a padded batch: what counts is as without padding
        n = torch.tensor([70, 20, 0], dtype=torch.int32, device=DEV)
        ragged, _ = net(x, lengths=n)
        for b in range(3):
            off = (ragged[b, :int(n[b])] - whole[b, :int(n[b])]).abs()
            assert bool((off <= 5e-5 * max(1.0, float(whole.abs().max()))).all())


def test_scans_both_ways_see_every_token():
    """A change of the last token reaches the first, and of the first the last; in bfloat16 as well."""
    from spherical_distortion import nn as snn
    for dtype in (torch.float32, torch.bfloat16):
        torch.manual_seed(1)
        layer = snn.GatedScan(16, 32, both_ways=True).to(DEV).to(dtype)
        x = _randn(1, 12, 16, dtype=dtype).requires_grad_()
        out, last = layer(x)
        assert out.shape == x.shape and out.dtype == dtype and last is None
        for at, seen in ((0, 11), (11, 0)):
            g, = torch.autograd.grad(out[0, at].float().sum(), x, retain_graph=True)
            assert bool(g[0, seen].any())
        out.float().sum().backward()
        assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in layer.parameters())
