"""Muon over the framework's kernels: the update of each matrix made orthogonal, all matrices of a step in few launches."""
import torch

from _spherical_distortion_ext import _token_ops

from .. import functional as F
from . import adamw


class Muon(torch.optim.Optimizer):
    """Muon, on the GPU only: momentum, the update made orthogonal by `steps` products, decoupled weight decay.

    params: float32, bfloat16 or float16, contiguous, two axes at least; [out, ..] counts as a matrix of `out` rows.  Others
    (biases, norms' weights, tables looked up by row) belong to another optimizer.  Momenta are float32.  One without a
    gradient is left as it is.  A step checks every group and parameter before it changes one.  In a graph a
    step keeps the settings of its capture; a parameter's first step, which makes its momentum, is refused there."""

    def __init__(self, params, lr=2e-2, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5,
                 coefficients=F.NEWTON_SCHULZ, eps=1e-7):
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coefficients=tuple(coefficients), eps=eps))

    @staticmethod
    def _check_settings(group):
        if not 0 <= group["lr"] <= 1e30 or not 0 <= group["weight_decay"] <= 1e30:
            raise ValueError("lr and weight_decay must not be negative (or beyond 1e30)")
        if not 0 <= group["momentum"] < 1:
            raise ValueError("momentum must be in [0, 1), got %s" % group["momentum"])
        try:
            _token_ops.check_newton_schulz(group["steps"], group["coefficients"], group["eps"])
        except RuntimeError as e:
            raise ValueError(str(e)) from None

    @staticmethod
    def _check_sides(p):
        rows = p.shape[0]
        if max(rows, p.numel() // rows if rows else 0) > 1 << 17 or p.numel() > 1 << 31:
            raise RuntimeError("Muon takes matrices with sides up to 131072 and 2^31 values, got a parameter of shape %s"
                             % (tuple(p.shape),))

    def _momentum(self, p):
        return self.state.get(p, {}).get("momentum")   # looking it up by [] would make an entry

    def _check_step(self):
        """All that a call would refuse, of every group that is stepped before one is."""
        stepped = [p for g in self.param_groups for p in g["params"] if p.grad is not None]
        for group in self.param_groups:
            if any(p.grad is not None for p in group["params"]):
                self._check_settings(group)
        for p in stepped:
            adamw.check_parameter("Muon", p)
            self._check_sides(p)
            m = self._momentum(p)
            if m is not None and not (m.shape == p.shape and m.dtype == torch.float32 and m.device == p.device
                                      and m.is_contiguous()):
                raise RuntimeError("a momentum must be float32, contiguous and beside its parameter of shape %s, got %s %s on %s"
                                   % (tuple(p.shape), m.dtype, tuple(m.shape), m.device))
        if any(p.is_cuda and self._momentum(p) is None for p in stepped) and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a parameter's first step cannot be captured: its momentum would begin as zeros in every replay")
        written = [p.data_ptr() for p in stepped if p.numel()]
        addresses = set(written)
        if len(addresses) < len(written):
            raise RuntimeError("a parameter is listed twice")
        if any(p.grad.data_ptr() in addresses for p in stepped if p.numel()):
            raise RuntimeError("a gradient is a parameter too")

    def add_param_group(self, group):
        super().add_param_group(group)
        try:
            self._check_settings(self.param_groups[-1])
            for p in self.param_groups[-1]["params"]:
                if p.dim() < 2:
                    raise ValueError("Muon takes parameters of two axes at least, got one of shape %s" % (tuple(p.shape),))
        except ValueError:
            self.param_groups.pop()
            raise

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._check_step()
        for group in self.param_groups:
            settings = {k: group[k] for k in ("lr", "momentum", "nesterov", "weight_decay", "steps", "coefficients", "eps")}
            calls = {}   # (type, device) -> lists of tensors
            for p in group["params"]:
                if p.grad is None:
                    continue
                m = self._momentum(p)
                if m is None:
                    m = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
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
