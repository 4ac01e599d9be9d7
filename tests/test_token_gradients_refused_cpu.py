"""Functions without gradients raise where one would be wanted, before anything touches a device."""
import pytest
import torch


def test_orthogonalize_refuses_to_drop_a_gradient():
    from spherical_distortion import functional as F
    x = torch.randn(4, 5)
    for leaf in (torch.nn.Parameter(x), x.clone().requires_grad_() * 2):
        with pytest.raises(RuntimeError, match="no gradients"):
            F.orthogonalize(leaf)
        for fine in (leaf.detach(), leaf):
            with torch.no_grad(), pytest.raises((NotImplementedError, RuntimeError)) as e:
                F.orthogonalize(fine)   # as far as the check of the device
            assert "no gradients" not in str(e.value)
