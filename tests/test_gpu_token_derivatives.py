"""What the operators on token sequences do not differentiate raises, and is never left out: second derivatives, beside
terms that have one too, and forward mode."""
import warnings

import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _attention_inputs():
    torch.manual_seed(3)
    q, k, v = (torch.randn(1, 2, 5, 8, device=DEV) for _ in range(3))
    return [q, k, v, torch.randn(2, 3, device=DEV)], torch.randint(0, 4, (5, 5), device=DEV).to(torch.uint8)


def _forms():
    """name -> (differentiable inputs, function of them that returns a list of outputs)."""
    from _spherical_distortion_ext import _token_ops
    from spherical_distortion import functional as F
    inputs, bmap = _attention_inputs()
    x, r, w = torch.randn(4, 16, device=DEV), torch.randn(4, 16, device=DEV), torch.rand(16, device=DEV) + 0.5
    forms = {}
    for kind, attend, norm in (("public", F.bucket_attention, F.add_rms_norm),
                               ("operator", _token_ops.ops.bucket_attention, _token_ops.ops.rms_norm_pair),
                               ("python", F.BucketAttentionFunction.apply, F.AddRMSNormFunction.apply)):
        forms[kind + " attention"] = inputs, lambda *t, attend=attend: [attend(*t, bmap, None, False, 0.4)]
        forms[kind + " norm"] = [x, r, w], lambda a, b, c, norm=norm: list(norm(a, b, c, 1e-6))
        forms[kind + " norm alone"] = [x, w], lambda a, c, norm=norm: list(norm(a, None, c, 1e-6))[:1]
        forms[kind + " sum alone"] = [x, r, w], lambda a, b, c, norm=norm: [norm(a, b, c, 1e-6)[1]]
    return forms


NAMES = [kind + what for kind in ("public", "operator", "python")
         for what in (" attention", " norm", " norm alone", " sum alone")]


@pytest.mark.parametrize("name", NAMES)
def test_second_derivatives_raise_beside_terms_that_have_one(name):
    inputs, fn = _forms()[name]
    plain = [t.clone().requires_grad_() for t in inputs]
    want = torch.autograd.grad(sum(o.sum() for o in fn(*plain)), plain, allow_unused=True)
    leaves = [t.clone().requires_grad_() for t in inputs]
    outs = fn(*leaves)
    grads = torch.autograd.grad(sum(o.sum() for o in outs), leaves, create_graph=True, allow_unused=True)
    for a, b in zip(grads, want):   # the first derivative is what it is without a graph
        assert (a is None) == (b is None) and (a is None or torch.equal(a, b))
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
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(lambda t: fn(*(t if j == i else u for j, u in enumerate(inputs)))[0], (inputs[i],),
                           (torch.ones_like(inputs[i]),))


@pytest.mark.parametrize("name", NAMES)
def test_a_recorded_backward_may_go_unused(name):
    """create_graph without a second derivative: gradients gather in .grad and are stepped on as ever."""
    inputs, fn = _forms()[name]
    leaves = [t.clone().requires_grad_() for t in inputs]
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")   # torch warns of the reference cycle that create_graph makes
        sum(o.sum() for o in fn(*leaves)).backward(create_graph=True)
    with torch.no_grad():
        for t in leaves:
            if t.grad is not None:
                t -= 0.1 * t.grad
                t.grad = None
