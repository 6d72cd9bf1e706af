"""``AdamW`` over this library's kernel: a ``torch.optim.Optimizer`` (parameter groups, schedulers, ``state_dict``) whose step is one launch
for all tensors of a group (``ops.adamw_step``), with states in 32 or 8 bits and fp32 copies of 16-bit weights on request."""
import torch

from . import ops

BLOCK = 256              # values that share a scale of 8-bit states


class AdamW(torch.optim.Optimizer):
    """``p = p (1 - lr wd) - lr m^ / (sqrt(v^) + eps)``.  ``state_bits=8`` keeps the states of tensors with at least ``min_8bit_size`` values as
    e4m3 codes with a scale per 256 values (biases and norm weights are few, and steps there are sensitive: they stay in 32 bits).
    ``master_weights`` steps an fp32 copy of every 16-bit parameter, so that updates smaller than half a unit of the 16-bit type add up."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, master_weights=False, min_8bit_size=4096):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32; got {state_bits}")
        if not (lr >= 0 and eps >= 0 and weight_decay >= 0 and all(0 <= b < 1 for b in betas)):
            raise ValueError("lr, eps and weight_decay must not be negative, betas must be in [0, 1)")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits, master_weights=master_weights,
                                      min_8bit_size=min_8bit_size))

    @staticmethod
    def _init_state(p, group, state):
        state["step"] = 0
        if group["state_bits"] == 8 and p.numel() >= group["min_8bit_size"]:
            for name in ("exp_avg", "exp_avg_sq"):
                state[name] = torch.zeros_like(p, dtype=torch.uint8).view(torch.float8_e4m3fn)
                state[name + "_scale"] = torch.zeros((p.numel() + BLOCK - 1) // BLOCK, dtype=torch.float32, device=p.device)
        else:
            state["exp_avg"], state["exp_avg_sq"] = (torch.zeros_like(p, dtype=torch.float32) for _ in range(2))
        if group["master_weights"] and p.dtype != torch.float32:
            state["master"] = p.detach().to(torch.float32)

    @torch.no_grad()
    def step(self, closure=None):
        """Steps every parameter that has a gradient."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            calls = {}                      # parameters by the number of their step and their device: one call each, nearly always one in all
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if not state:
                    self._init_state(p, group, state)
                calls.setdefault((state["step"] + 1, p.device), []).append((p, state))
            for (step, _), items in calls.items():
                states = [s for _, s in items]
                column = lambda name: [s.get(name) for s in states]  # noqa: E731
                ops.adamw_step([p for p, _ in items], [p.grad for p, _ in items], column("exp_avg"), column("exp_avg_sq"), step, float(group["lr"]),
                               group["betas"], group["eps"], group["weight_decay"], masters=column("master"), exp_avg_scales=column("exp_avg_scale"),
                               exp_avg_sq_scales=column("exp_avg_sq_scale"))
                for s in states:
                    s["step"] = step
        return loss

    def load_state_dict(self, state_dict):
        """As in the base class, but states keep their own dtypes (the base class casts them to the parameters')."""
        super().load_state_dict(state_dict)
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        params = [p for group in self.param_groups for p in group["params"]]
        for i, p in zip(ids, params):
            for name, value in state_dict["state"].get(i, {}).items():
                if torch.is_tensor(value):
                    self.state[p][name] = value.detach().to(p.device, copy=True)
