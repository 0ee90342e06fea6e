"""AdamW on the library's kernels: every parameter of a group updated in a few launches, the clipping by the global gradient norm
folded into the update, moments in 32 or 8 bits.  The reference leaves optimizer and clipping to the HuggingFace Trainer
(slim/fine_tune.py:197-219)."""
import torch

from . import ops

# tensors with fewer elements keep 32-bit moments when state_bits is 8 (norm weights and biases: nothing to save there)
MIN_8BIT_NUMEL = 4096
_STATE_TENSORS = ("exp_avg", "exp_avg_sq", "scales", "master")
# what torch's Adam and AdamW record where their update is not this one (an Adam without weight decay is)
_OTHER_UPDATES = {"amsgrad": True, "maximize": True, "decoupled_weight_decay": False}


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update for dense fp32, bf16 and fp16 parameters on one GPU.

    state_bits: 32, or 8: first moments as e4m3 and second as e5m2 numbers with a pair of scales per 512 elements, rounded
    stochastically (an exponential average that moves by 0.1 % a step would stand still under rounding to nearest); the random
    bits are a function of `seed`, the step and the position, so a run can be repeated exactly; `seed` is an option of the groups
    and so part of state_dict(): a run that is loaded goes on with its own.  Tensors below MIN_8BIT_NUMEL elements keep
    32-bit moments.
    master_weights: 16-bit parameters keep an fp32 copy that is what is updated.
    max_grad_norm: gradients are multiplied by min(1, max_grad_norm / (norm + 1e-6)) as they are read, norm over all parameters
    of all groups; the gradients themselves stay as they were.  `last_norm` is that norm after a step (a 0-d tensor on the GPU).  It is not part
    of state_dict(): a run that is loaded needs it passed again.

    step() cannot be captured into a graph: it counts on the host.  (ops.grad_norm and ops.adamw_step can.)"""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, master_weights=False,
                 max_grad_norm=None, seed=0):
        self._check_options(dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits))
        if max_grad_norm is not None and not max_grad_norm > 0:
            raise ValueError(f"max_grad_norm must be positive, got {max_grad_norm}")
        self.max_grad_norm = max_grad_norm
        self.last_norm = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits, master_weights=master_weights, seed=int(seed)))

    @staticmethod
    def _check_options(group):
        lr, eps, weight_decay, betas, state_bits = (group[k] for k in ("lr", "eps", "weight_decay", "betas", "state_bits"))
        if not lr >= 0 or not eps >= 0 or not weight_decay >= 0:
            raise ValueError(f"lr, eps and weight_decay must not be negative, got {lr}, {eps}, {weight_decay}")
        if 0 < eps < 2.0 ** -126:
            raise ValueError(f"eps must be 0 or at least 2^-126, got {eps}")
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError(f"betas must lie in [0, 1), got {betas}")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")

    def add_param_group(self, param_group):
        """torch's, with the checks of the constructor on a group's own options."""
        self._check_options({**self.defaults, **param_group})
        super().add_param_group(param_group)

    @property
    def seed(self):
        return self.param_groups[0]["seed"]

    def _new_state(self, p, group):
        state = dict(step=0)
        if group["state_bits"] == 8 and p.numel() >= MIN_8BIT_NUMEL:
            state["exp_avg"] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn)
            state["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device).view(torch.float8_e5m2)
            state["scales"] = torch.zeros(-(-p.numel() // ops.ADAMW_BLOCK), 2, dtype=torch.float32, device=p.device)
        else:
            state["exp_avg"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            state["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        if group["master_weights"] and p.dtype != torch.float32:
            state["master"] = p.detach().float().contiguous()
        return state

    @staticmethod
    def _check(p):
        g = p.grad
        if not p.is_cuda:
            raise RuntimeError(f"parameters must be on the GPU: slim_amd has no CPU path (got device {p.device})")
        if p.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise TypeError(f"parameters must be float32, bfloat16 or float16, got {p.dtype}")
        if g.layout != torch.strided:
            raise RuntimeError("AdamW does not take sparse gradients")
        if not p.is_contiguous():
            raise ValueError(f"parameters must be contiguous, got strides {p.stride()} for {tuple(p.shape)}")

    def _norm(self, items):
        """The norm of all gradients, one value per element type combined."""
        by_type = {}
        for _, _, g in items:
            by_type.setdefault(g.dtype, []).append(g)
        norms = [ops.grad_norm(gs) for gs in by_type.values()]
        return norms[0] if len(norms) == 1 else torch.stack(norms).double().square().sum().sqrt().float()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        items = [(p, group, p.grad) for group in self.param_groups for p in group["params"] if p.grad is not None]
        for p, _, _ in items:
            self._check(p)
        items = [(p, group, g if g.is_contiguous() else g.contiguous()) for p, group, g in items if p.numel()]
        if not items:
            return loss
        if len({p.device for p, _, _ in items}) > 1:
            raise ValueError("AdamW updates parameters of one GPU")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW.step counts steps on the host and cannot be captured; ops.grad_norm and ops.adamw_step can")
        norm = None if self.max_grad_norm is None else self._norm(items)
        calls = {}
        for p, group, g in items:
            state = self.state.get(p) or self._new_state(p, group)       # (a new one is kept once nothing can be refused any more)
            key = (id(group), p.dtype, "scales" in state, "master" in state, state["step"] + 1)
            calls.setdefault(key, (group, []))[1].append((p, g, state))
        plans, first = [], 0
        for (_, _, eight, master, step), (group, members) in calls.items():
            states = [s for _, _, s in members]
            plans.append(ops._adamw_plan([p for p, _, _ in members], [g for _, g, _ in members], [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states],
                                        step=step, lr=float(group["lr"]), beta1=group["betas"][0], beta2=group["betas"][1], eps=group["eps"],
                                        weight_decay=group["weight_decay"], scales=[s["scales"] for s in states] if eight else None,
                                        masters=[s["master"] for s in states] if master else None, seed=group["seed"] + step * 0x9e3779b1, norm=norm,
                                        max_norm=self.max_grad_norm, first_index=first))
            first += len(members)
        self.last_norm = norm
        for plan, ((*_, step), (_, members)) in zip(plans, calls.items()):
            ops._adamw_run(plan)
            for p, _, state in members:
                state["step"] = step
                self.state[p] = state
        return loss

    def __getstate__(self):
        return dict(super().__getstate__(), max_grad_norm=self.max_grad_norm, last_norm=self.last_norm)

    def load_state_dict(self, state_dict):
        """torch's, with the state's own element types (which it would change to the parameters').  What torch.optim.AdamW saved over
        fp32 parameters loads too (its moments continue in 32 bits), but for amsgrad and maximize.  Registered pre-hooks decide what is loaded, post-hooks see the
        state as it stays."""
        seen = {}

        def take(_, final):                              # behind every other pre-hook: the dictionary that is loaded
            for group in final["param_groups"]:
                for name, value in _OTHER_UPDATES.items():
                    if group.get(name) == value and (name != "decoupled_weight_decay" or group.get("weight_decay")):
                        raise ValueError(f"AdamW cannot continue a state of another update: {name}={value}")
            seen.update(final)

        def repair(_):                                   # in front of every other post-hook
            for group in self.param_groups:
                for name in ("state_bits", "master_weights", "seed"):
                    group.setdefault(name, self.defaults[name])
            ids = [i for group in seen["param_groups"] for i in group["params"]]
            params = [p for group in self.param_groups for p in group["params"]]
            for i, p in zip(ids, params):
                saved = seen["state"].get(i)
                if saved is None:
                    continue
                self.state[p]["step"] = int(saved["step"])
                for name in _STATE_TENSORS:
                    if saved.get(name) is not None:
                        self.state[p][name] = saved[name].detach().to(p.device, copy=True).contiguous()
        handles = self.register_load_state_dict_pre_hook(take), self.register_load_state_dict_post_hook(repair, prepend=True)
        try:
            super().load_state_dict(state_dict)
        finally:
            for handle in handles:
                handle.remove()
