"""AdamW over many tensors at once, its moments in 32 or in 8 bits: the optimizer step behind a backward pass (and, with
several ranks, behind the gradient exchange of `sphmap.parallel.GradReducer`).

`adamw_step` is the step itself on lists of tensors, `AdamW` the torch optimizer that keeps the lists."""
import torch

import _spherical_distortion_ext._C as _C

BLOCK = 256   # values of an 8-bit moment behind one scale


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, step, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, masters=None,
               exp_avg_scales=None, exp_avg_sq_scales=None, grad_scale=1.0):
    """One step over all tensors, in place, in one kernel launch for each kind of tensor (and each 440 of them):

        m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2  (g = grad * grad_scale)
        w = w (1 - lr weight_decay) - lr m / (1 - b1^step) / (sqrt(v / (1 - b2^step)) + eps)

    params float32, bfloat16 or float16, CUDA and contiguous like everything else here; grads of their params' dtype or
    float32.  masters: float32 copies of 16-bit params (None for any other), which are then what is updated, the param being
    its rounding.  exp_avgs and exp_avg_sqs (m, v): float32, or, with scales, float8_e4m3fn with a float32 scale for each 256
    values, ceil(numel / 256) for a tensor; v is then held as its square root.  What is written must not overlap anything else.
    step: the number of this step, from 1, or a float32 CUDA tensor that holds it, for CUDA graphs; lr may be a tensor too then."""
    on_device = isinstance(step, torch.Tensor)
    lr_at = lr if isinstance(lr, torch.Tensor) else None
    _C.adamw_step(params, grads, exp_avgs, exp_avg_sqs, masters, exp_avg_scales, exp_avg_sq_scales, 0.0 if on_device else float(step),
                  0.0 if lr_at is not None else float(lr), float(betas[0]), float(betas[1]), float(eps), float(weight_decay),
                  float(grad_scale), step if on_device else None, lr_at)


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update through `adamw_step`.

    state_bits 8 keeps both moments in 8 bits (2 bytes and 1/32 a value instead of 8).  master_weights keeps float32 copies of
    16-bit params.  capturable keeps the step's number on the device, one for each param group, so that a CUDA graph that holds
    `step()` counts on as it is replayed; lr may be a CUDA tensor then.  Such a graph reads the gradients where they were at its
    capture (zero_grad(set_to_none=False), or a backward pass in the same graph), and one step has to run before the capture,
    which makes the moments."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32, master_weights=False,
                 capturable=False):
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32, got %r" % (state_bits,))
        if isinstance(lr, torch.Tensor) and not capturable:
            raise ValueError("lr as a tensor needs capturable=True")
        if not isinstance(lr, torch.Tensor) and not lr >= 0:
            raise ValueError("lr must not be negative, got %r" % (lr,))
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError("betas must be in [0, 1), got %r" % (betas,))
        if not eps >= 0 or not weight_decay >= 0:
            raise ValueError("eps and weight_decay must not be negative")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      master_weights=master_weights, capturable=capturable))

    def _state_of(self, p, group, capturing):
        s = self.state[p]
        if not s:
            if capturing:
                raise RuntimeError("AdamW: a step has to run before one is captured in a graph")
            if not p.is_contiguous():
                raise RuntimeError("param must be contiguous")
            if not group["capturable"]:
                s["step"] = 0
            eight = group["state_bits"] == 8
            for name in ("exp_avg", "exp_avg_sq"):
                s[name] = torch.zeros_like(p, dtype=torch.float8_e4m3fn if eight else torch.float32,
                                           memory_format=torch.contiguous_format)
                if eight:
                    s[name + "_scale"] = torch.zeros(-(-p.numel() // BLOCK), dtype=torch.float32, device=p.device)
            if group["master_weights"] and p.dtype != torch.float32:
                s["master"] = p.detach().float()
        return s

    def _keep_count(self, group, capturing):
        """The step's number where `capturable` wants it, the group or its params' states, and on from where it was if that has
        changed since the last step."""
        if isinstance(group.get("step"), torch.Tensor) if group["capturable"] else "step" not in group:
            return
        states = [self.state[p] for p in group["params"] if self.state.get(p)]
        if not group["capturable"]:
            n = int(group.pop("step"))
            for s in states:
                s["step"] = n
        else:       # (a number until the device is known)
            counts = {s["step"] for s in states if "step" in s}
            if len(counts) > 1:
                raise RuntimeError("AdamW: params at different step numbers cannot become capturable together")
            if capturing and states:
                raise RuntimeError("AdamW: a step has to run before one is captured in a graph")
            group["step"] = counts.pop() if counts else group.get("step", 0)
            for s in states:
                s.pop("step", None)

    def load_state_dict(self, state_dict):
        """Moments and masters keep their own types (the base class would cast them to their param's)."""
        super().load_state_dict(state_dict)
        params = [p for g in self.param_groups for p in g["params"]]
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        for p, i in zip(params, saved):
            for k, v in state_dict["state"].get(i, {}).items():
                if isinstance(v, torch.Tensor):
                    self.state[p][k] = v.detach().to(device=p.device, copy=True)
        for g in self.param_groups:
            for k in ("step", "lr"):
                if isinstance(g.get(k), torch.Tensor) and g["params"]:
                    g[k] = g[k].detach().to(device=g["params"][0].device, copy=True)

    @torch.no_grad()
    def step(self, closure=None, grad_scale=1.0):
        """grad_scale multiplies the gradients (1 / ranks after a sum over them, a clipping factor)."""
        loss, self._grad_scale = None, grad_scale
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        capturing = torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()
        for group in self.param_groups:
            if capturing and not group["capturable"]:
                raise RuntimeError("AdamW: a captured step needs capturable=True (its number would stay what it was)")
            self._keep_count(group, capturing)
            together = {}   # params at one step number: all, unless some had no gradient in an earlier step
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.layout != torch.strided:
                    raise RuntimeError("gradients must be dense")
                s = self._state_of(p, group, capturing)
                together.setdefault((p.device, s.get("step")), []).append((p, s))
            if group["capturable"] and together:
                if len(together) > 1:
                    raise RuntimeError("a capturable param group must be on one device")
                if not isinstance(group["step"], torch.Tensor):
                    group["step"] = torch.tensor(float(group["step"]), device=next(iter(together))[0])
                group["step"] += 1
            for some in together.values():
                self._step(group, some)
        return loss

    def _step(self, group, some):
        states = [s for _, s in some]
        eight = group["state_bits"] == 8
        adamw_step([p for p, _ in some], [p.grad.contiguous() for p, _ in some], [s["exp_avg"] for s in states],
                   [s["exp_avg_sq"] for s in states], step=group["step"] if group["capturable"] else states[0]["step"] + 1, lr=group["lr"],
                   betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"],
                   masters=[s.get("master") for s in states] if group["master_weights"] else None,
                   exp_avg_scales=[s["exp_avg_scale"] for s in states] if eight else None,
                   exp_avg_sq_scales=[s["exp_avg_sq_scale"] for s in states] if eight else None, grad_scale=self._grad_scale)
        if not group["capturable"]:
            for s in states:
                s["step"] += 1
