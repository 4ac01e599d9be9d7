"""AdamW over the framework's kernels: all tensors of a step in few launches, moments in 32 or 8 bits."""
import torch

from .. import functional as F

_BLOCK = 256   # values that share a scale in 8 bits
_TYPES = (torch.float32, torch.bfloat16, torch.float16)
_MOMENTS = {32: ("exp_avg", "exp_avg_sq"), 8: ("avg_codes", "avg_scales", "sq_codes", "sq_scales")}


def _on_gpu(p):
    return p.is_cuda


def _check(p):
    """What the step refuses of a parameter with a gradient."""
    if p.grad.is_sparse:
        raise RuntimeError("AdamW does not take sparse gradients")
    if not _on_gpu(p):
        raise RuntimeError("this backend runs on the GPU only: parameters must be CUDA/HIP tensors")
    if p.dtype not in _TYPES or p.grad.dtype != p.dtype:
        raise RuntimeError("parameters must be float32, bfloat16 or float16 and their gradients alike, got %s and %s"
                           % (p.dtype, p.grad.dtype))
    if not p.is_contiguous():
        raise RuntimeError("parameters must be contiguous, got strides %s of shape %s" % (p.stride(), tuple(p.shape)))


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay), on the GPU only.

    params: float32, bfloat16 or float16 and contiguous.  moment_bits: 32, or 8 for moments held as codes
    with a scale for each 256 values (2 bytes a value instead of 8; functional.adamw_step_8bit says which
    values they stand for); parameters of fewer than `smallest_8bit` values keep 32 bits.  Each parameter
    counts its own steps: one without a gradient is left as it is.  A step checks every parameter before it
    changes one, and counts for those whose call returned."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, moment_bits=32,
                 smallest_8bit=4096):
        if not lr >= 0 or not eps >= 0 or not weight_decay >= 0:
            raise ValueError("lr, eps and weight_decay must not be negative")
        if not all(0 <= b < 1 for b in betas):
            raise ValueError("betas must be in [0, 1), got %s" % (betas,))
        if moment_bits not in _MOMENTS:
            raise ValueError("moment_bits must be 32 or 8, got %s" % moment_bits)
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, moment_bits=moment_bits,
                                      smallest_8bit=smallest_8bit))

    @staticmethod
    def _begin(p, bits):
        state = {"step": 0}
        if bits == 32:
            for name in _MOMENTS[32]:
                state[name] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            return state
        blocks = -(-p.numel() // _BLOCK)
        for kind, dtype in (("avg", torch.int8), ("sq", torch.uint8)):
            state[kind + "_codes"] = torch.zeros(p.shape, dtype=dtype, device=p.device)
            state[kind + "_scales"] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
        return state

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is not None:
                    _check(p)
        for group in self.param_groups:
            settings = {k: group[k] for k in ("lr", "betas", "eps", "weight_decay")}
            calls = {}   # (type, device, step, bits) -> lists of tensors, states
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state.get(p)
                if not state:
                    eight = group["moment_bits"] == 8 and p.numel() >= group["smallest_8bit"]
                    state = self._begin(p, 8 if eight else 32)
                bits = 32 if "exp_avg" in state else 8
                names = _MOMENTS[bits]
                lists, states = calls.setdefault((p.dtype, p.device, state["step"] + 1, bits),
                                                 ([[] for _ in range(2 + len(names))], []))
                lists[0].append(p)
                lists[1].append(p.grad.contiguous())
                for i, name in enumerate(names):
                    lists[2 + i].append(state[name])
                states.append(state)
            for (_, _, step, bits), (lists, states) in calls.items():
                run = F.adamw_step if bits == 32 else F.adamw_step_8bit
                run(*lists, step=step, **settings)
                for p, state in zip(lists[0], states):
                    state["step"] = step
                    self.state[p] = state
        return loss

    def load_state_dict(self, state_dict):
        """As torch.optim.Optimizer's, but moments keep their types (the base class casts them to the
        parameter's, which codes and 32-bit moments of 16-bit parameters must not be)."""
        super().load_state_dict(state_dict)
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        held = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(saved, held):
            for name, value in state_dict["state"].get(i, {}).items():
                if torch.is_tensor(value) and name in _MOMENTS[32] + _MOMENTS[8]:
                    self.state[p][name] = value.detach().clone().to(p.device)
