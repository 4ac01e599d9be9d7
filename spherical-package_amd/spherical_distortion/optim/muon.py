"""Muon over the framework's kernels: the update of each matrix made orthogonal, all matrices of a step in few launches."""
import torch

from _spherical_distortion_ext import _token_ops

from .. import functional as F
from . import adamw


class Muon(torch.optim.Optimizer):
    """Muon, on the GPU only: momentum, the update made orthogonal by `steps` products, decoupled weight decay.

    params: float32, bfloat16 or float16, contiguous, two axes at least; [out, ..] counts as a matrix of `out` rows.  Others
    (biases, norms' weights, tables looked up by row) belong to another optimizer.  Momenta are float32.  One without a
    gradient is left as it is.  A step checks every parameter before it changes one."""

    def __init__(self, params, lr=2e-2, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5,
                 coefficients=F.NEWTON_SCHULZ, eps=1e-7):
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coefficients=tuple(coefficients), eps=eps))

    @staticmethod
    def _check(group):
        if not group["lr"] >= 0 or not group["weight_decay"] >= 0:
            raise ValueError("lr and weight_decay must not be negative")
        if not 0 <= group["momentum"] < 1:
            raise ValueError("momentum must be in [0, 1), got %s" % group["momentum"])
        try:
            _token_ops.check_newton_schulz(group["steps"], group["coefficients"], group["eps"])
        except RuntimeError as e:
            raise ValueError(str(e)) from None
        for p in group["params"]:
            if p.dim() < 2:
                raise ValueError("Muon takes parameters of two axes at least, got one of shape %s" % (tuple(p.shape),))

    def add_param_group(self, group):
        super().add_param_group(group)
        try:
            self._check(self.param_groups[-1])
        except ValueError:
            self.param_groups.pop()
            raise

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is not None:
                    adamw.check_parameter("Muon", p)
        for group in self.param_groups:
            settings = {k: group[k] for k in ("lr", "momentum", "nesterov", "weight_decay", "steps", "coefficients", "eps")}
            calls = {}   # (type, device) -> lists of tensors
            for p in group["params"]:
                if p.grad is None:
                    continue
                m = self.state[p]["momentum"] if p in self.state else torch.zeros(p.shape, device=p.device)
                for to, t in zip(calls.setdefault((p.dtype, p.device), ([], [], [])), (p, p.grad.contiguous(), m)):
                    to.append(t)
            for lists in calls.values():
                F.muon_step(*lists, **settings)
                for p, _, m in zip(*lists):
                    self.state[p]["momentum"] = m
        return loss

    def load_state_dict(self, state_dict):
        """As torch.optim.Optimizer's, but momenta stay float32 (the base class casts them to the parameter's type)."""
        super().load_state_dict(state_dict)
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        held = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(saved, held):
            if "momentum" in state_dict["state"].get(i, {}):
                self.state[p]["momentum"] = state_dict["state"][i]["momentum"].detach().clone().to(p.device)
