"""The optimizer step on the device: entry points of the operators `sv3d::grad_square_sums`, `sv3d::adamw_step` and
`sv3d::moment_values` (csrc/torch_train_ops.cpp over the functions of the same names in include/sv3d_hip.h), and
the optimizer over them.  It does in two passes over the gradients what the reference's step does in five or more
(nnutils/train_utils.py:201-214: unscale, clip_grad_norm_, Adam).  GPU tensors only.
"""
import torch

from .ops import _ops, call

STATE_BLOCK = 128           # elements that share the scales of their 8-bit moments


def grad_square_sums(grads):
    """Sums of squares of the listed gradients in float64, as several numbers (`.sum().sqrt()` is their norm)."""
    return call("grad_square_sums", grads)


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, steps, *, scales=None, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
               weight_decay=0.0, max_norm=0.0, square_sums=None, grad_scale=None, found_inf=None, maximize=False, seed=0):
    """One AdamW step of all `params` (float32, float16 or bfloat16, each with its gradient, moments and step count),
    in place.  Gradients are first divided by `grad_scale` and, where `max_norm` is above 0, scaled to a common norm of
    at most `max_norm` as `torch.nn.utils.clip_grad_norm_` would; they themselves are left as they are.  Returns that
    common norm (before clipping) as a tensor, None without `max_norm`.

    The moments have their weight's sizes and strides.  They are float32, or uint8 with `scales` (uint8
    [ceil(numel/128), 2] per tensor, contiguous; ignored for float32 moments): 8 bits per value and a power of two per
    block of 128, rounded up or down with the probability of what is cut off, by a hash of element, step and `seed`
    (see `moment_values`).  `steps` are one-element float32 tensors on the device.

    Where the second moment is zero an `eps` below 2^-63 counts as 2^-63: a weight that never had a gradient stays.

    `lr` may be a one-element float32 tensor on the device; `grad_scale` and `found_inf` are such tensors or None, and
    with a `found_inf` that is not 0 nothing changes.  `square_sums` (of `grad_square_sums`) says whose norm is meant
    where that is not the norm of `grads` alone."""
    if len(params) == 0:
        return None
    clip = max_norm is not None and max_norm != 0
    if clip and not max_norm > 0:
        raise ValueError("max_norm must not be negative or NaN, got %r" % (max_norm,))
    with torch.no_grad():
        tensor_lr = lr if torch.is_tensor(lr) else None
        norm = call("adamw_step", params, grads, exp_avgs, exp_avg_sqs, scales if scales is not None else [], steps, tensor_lr,
                               grad_scale, found_inf, square_sums if clip else None, 0.0 if tensor_lr is not None else lr,
                               betas[0], betas[1], eps, weight_decay, max_norm if clip else 0.0, maximize, seed)
    return norm if clip else None


def moment_values(exp_avg, exp_avg_sq, scales):
    """The values of 8-bit moments as two bfloat16 tensors, which hold every one of them exactly."""
    return _ops.moment_values(exp_avg, exp_avg_sq, scales)


class AdamW(torch.optim.Optimizer):
    """AdamW with the whole step fused: unscaling and clipping included, many tensors per launch.

    lr, betas, eps, weight_decay, maximize: as `torch.optim.AdamW` (with weight_decay 0 the update of
    `torch.optim.Adam`).  `max_norm` > 0 clips the norm of all gradients of all groups together.  `state_bits` 8 holds
    the moments of every tensor of at least `min_8bit_size` elements in 8 bits, a quarter of the memory and less than
    two thirds of the step's traffic; `seed` picks how they are rounded.  `total_norm` is the norm of the last step's
    unscaled gradients (a tensor on the device) where `max_norm` is set.

    Works with `torch.amp.GradScaler` (call `scaler.step(optimizer)` alone: unscaling happens inside) and inside a HIP
    graph once the first step or `make_state` has made the state; a learning rate that changes under a captured step is a
    tensor."""

    _step_supports_amp_scaling = True       # GradScaler hands over grad_scale and found_inf instead of unscaling

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, maximize=False, max_norm=0.0,
                 state_bits=32, min_8bit_size=4096, seed=0):
        if not (torch.is_tensor(lr) or lr >= 0.0):
            raise ValueError("lr must not be negative, got %r" % (lr,))
        if torch.is_tensor(lr) and (lr.numel() != 1 or lr.dtype != torch.float32):
            raise ValueError("lr as a tensor must hold one float32")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError("betas must lie in [0, 1), got %r" % (betas,))
        if not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError("eps and weight_decay must not be negative, got %r and %r" % (eps, weight_decay))
        if not max_norm >= 0.0:
            raise ValueError("max_norm must not be negative, got %r" % (max_norm,))
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32, got %r" % (state_bits,))
        self.max_norm, self.state_bits, self.min_8bit_size, self.seed = max_norm, state_bits, min_8bit_size, seed
        self.total_norm = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, maximize=maximize))

    _own = ("max_norm", "state_bits", "min_8bit_size", "seed", "total_norm")

    def __getstate__(self):
        return {**super().__getstate__(), **{name: getattr(self, name) for name in self._own}}

    def _new_state(self, p):
        if p.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("sv3d.optim.AdamW makes a weight's state on its first step or in make_state(), one of which must come "
                               "before the capture")
        state = {"step": torch.zeros((), dtype=torch.float32, device=p.device)}
        if self.state_bits == 8 and p.numel() >= self.min_8bit_size:
            for name in ("exp_avg", "exp_avg_sq"):
                state[name] = torch.zeros_like(p, dtype=torch.uint8, memory_format=torch.preserve_format)
            blocks = -(-p.numel() // STATE_BLOCK)
            state["scales"] = torch.zeros(blocks, 2, dtype=torch.uint8, device=p.device)
        else:
            for name in ("exp_avg", "exp_avg_sq"):
                state[name] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
        return state

    @torch.no_grad()
    def make_state(self):
        """Makes the state of every weight that has a gradient and no state yet, as its first step would: ahead of the capture
        of that step in a HIP graph."""
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is not None and not self.state[p]:
                    self.state[p].update(self._new_state(p))

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        grad_scale, found_inf = getattr(self, "grad_scale", None), getattr(self, "found_inf", None)
        work, none = [], None
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            if not params:
                continue
            states = []
            for p in params:
                state = self.state[p]
                if not state:
                    state.update(self._new_state(p))
                states.append(state)
            scales = None
            if any("scales" in s for s in states):
                if none is None:
                    none = params[0].new_empty(0, dtype=torch.uint8)
                scales = [s.get("scales", none) for s in states]
            work.append((group, params, [p.grad for p in params], states, scales))
        sums = None
        if self.max_norm > 0 and len(work) > 1:         # one norm over all groups
            sums = grad_square_sums([g for w in work for g in w[2]])
        for group, params, grads, states, scales in work:
            norm = adamw_step(params, grads, [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states],
                              [s["step"] for s in states], scales=scales, lr=group["lr"], betas=group["betas"],
                              eps=group["eps"], weight_decay=group["weight_decay"], max_norm=self.max_norm,
                              square_sums=sums, grad_scale=grad_scale, found_inf=found_inf,
                              maximize=group["maximize"], seed=self.seed)
            if norm is not None:
                self.total_norm = norm
        return loss

    def load_state_dict(self, state_dict):
        """As every optimizer's, also from `torch.optim.Adam`'s and `AdamW`'s.  8-bit codes stay what they are, moments of
        any other type become float32 in their weight's strides, whatever the weight's type; step counts and a
        learning rate that is a tensor go to the weights' device.  A dict of another update is refused: one with
        `amsgrad`, or of an `Adam` whose `weight_decay` is part of the gradient."""
        found = {}

        def take(_, d):
            for group in d["param_groups"]:
                if group.get("amsgrad"):
                    raise ValueError("the saved optimizer has amsgrad=True, which this AdamW does not have")
                if group.get("weight_decay", 0) != 0 and not group.get("decoupled_weight_decay", True):
                    raise ValueError("the saved optimizer adds weight_decay=%r to the gradients (Adam), this AdamW takes it off "
                                     "the weights" % (group["weight_decay"],))
            found.update(d)

        # Hooks that the caller registered before loading may change or replace the dict, those after it the state: the dict
        # is looked at behind the former, what it holds is converted ahead of the latter.
        hooks = (self.register_load_state_dict_pre_hook(take),
                 self.register_load_state_dict_post_hook(lambda _: self._take_over(found), prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _take_over(self, state_dict):
        """The dict's state in place of what the base class made of it, which is of the weights' types."""
        kept = state_dict["state"]
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, params):
            for name, value in kept.get(i, {}).items():
                if name == "step":
                    value = torch.as_tensor(value, dtype=torch.float32).detach().to(device=p.device, copy=True)
                elif name in ("exp_avg", "exp_avg_sq") and value.dtype != torch.uint8 and value.shape == p.shape:
                    value = torch.empty_like(p, dtype=torch.float32, requires_grad=False).copy_(value.detach())
                elif torch.is_tensor(value):
                    value = value.detach().to(device=p.device, copy=True)
                self.state[p][name] = value
        for group in self.param_groups:
            for name, value in self.defaults.items():       # what older versions of torch did not save
                group.setdefault(name, value)
            if torch.is_tensor(group["lr"]) and group["params"]:
                group["lr"] = group["lr"].detach().to(device=group["params"][0].device, dtype=torch.float32, copy=True)
