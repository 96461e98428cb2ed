"""AdamW for the drop-in modules (layers.DC_Generator_*, layers.DC_Discriminator) and any other parameters on the GPU: the
reference's loop (src/train_wgan_v2.py:489-490,612,634) with

    from pgan_optim import AdamW
    disc_optimizer = AdamW(discriminator.parameters(), lr=5e-5, betas=(0.5, 0.999), weight_decay=0.01)

All tensors of a group are stepped in one launch per forty tensors (HipOps.adamw_plan).  state_bits=8 holds both states in
8 bits with a power-of-two scale for every 256 elements (2 bytes an element instead of 8), rounded stochastically from
`seed`; state_bits=32 is torch.optim.AdamW's arithmetic.
"""
from __future__ import annotations

import torch

from pgan_hip import ADAMW_BLOCK, ADAMW_LEAST_EPS, PganError

_STATE = {32: ("exp_avg", "exp_avg_sq"), 8: ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")}


def _honoured(group) -> None:
    """Refuses a group's options (torch's names) that step() would have to pass over."""
    for name in ("maximize", "amsgrad", "differentiable"):
        if group.get(name):
            raise ValueError(f"AdamW: {name} is not supported")
    if group.get("decoupled_weight_decay") is False and group.get("weight_decay"):
        raise ValueError("AdamW: the weight decay of these groups is part of the gradient (torch.optim.Adam's), here it is decoupled")


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW on the GPU.  Parameters are contiguous float32, bfloat16 or float16 tensors of one device (gradients
    of any of the three types); a parameter without a gradient is left alone in that step.

    state: per parameter `step`, `exp_avg` and `exp_avg_sq` -- float32, or with state_bits=8 float8_e4m3fn codes of the first
    moment and of the root of the second, with their scales in `exp_avg_scale` and `exp_avg_sq_scale`.
    torch's amsgrad, maximize, differentiable and a decay that is part of the gradient are refused, in groups and loaded states.
    capturable: the steps are counted on the device, so that a captured graph counts on every replay; every parameter of a
    group then needs a gradient in every step; rates, decay, betas and eps are those of the capture.  Without it a step refuses
    to be captured."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, seed=0, capturable=False):
        if not lr >= 0 or not eps >= 0 or not weight_decay >= 0:
            raise ValueError(f"lr, eps and weight_decay must not be negative, got {lr}, {eps} and {weight_decay}")
        if not (eps == 0 or eps >= ADAMW_LEAST_EPS):
            raise ValueError(f"eps must be 0 or at least {ADAMW_LEAST_EPS}, got {eps}")
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError(f"betas must lie in [0, 1), got {betas}")
        if state_bits not in _STATE:
            raise ValueError(f"states are held in 32 or in 8 bits, got {state_bits}")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      seed=seed, capturable=capturable))
        self._plans = {}                # (group, steps made): plan and what it was made of
        self._recorded = []             # plans and counters of captured steps: their graphs write to this memory

    def __setstate__(self, state):
        super().__setstate__(state)
        self._plans, self._recorded = {}, getattr(self, "_recorded", [])

    def add_param_group(self, param_group):
        _honoured(param_group)
        super().add_param_group(param_group)

    @staticmethod
    def _layout(p, bits):
        """Names of a parameter's states with their types and elements."""
        n, blocks = p.numel(), -(-p.numel() // ADAMW_BLOCK)
        kinds = [(torch.float32, n)] * 2 if bits == 32 else [(torch.float8_e4m3fn, n)] * 2 + [(torch.float32, blocks)] * 2
        return dict(zip(_STATE[bits], kinds))

    def _fresh(self, p, bits):
        zeros = lambda dtype, n: torch.zeros(n * dtype.itemsize, dtype=torch.uint8, device=p.device).view(dtype)
        return {name: zeros(*kind) for name, kind in self._layout(p, bits).items()}

    def _plan(self, key, ps, bits):
        """The plan of these parameters, made anew where a parameter or a state is no longer the memory it was made for."""
        names = _STATE[bits]
        held = [[self.state[p][name] for p in ps] for name in names]
        made_of = [(p.data_ptr(), p.dtype, p.is_contiguous()) for p in ps] + [t.data_ptr() for ts in held for t in ts]
        old = self._plans.get(key)
        if old is not None and old[1] == made_of:
            return old[0]
        from layers import _ops
        plan = _ops(ps[0].device).adamw_plan([p.detach() for p in ps], held[0], held[1], scales=None if bits == 32 else held[2:])
        self._plans[key] = (plan, made_of)
        return plan

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for gi, group in enumerate(self.param_groups):
            ps = [p for p in group["params"] if p.grad is not None]
            if not ps:
                continue
            capturing = ps[0].is_cuda and torch.cuda.is_current_stream_capturing()
            if capturing and not group["capturable"]:
                raise RuntimeError("AdamW: a captured step needs capturable=True (the step's number would be recorded)")
            if group["capturable"] and len(ps) != len(group["params"]):
                raise RuntimeError("AdamW: with capturable=True every parameter of a group needs a gradient in every step")
            if group.get("counter") is not None and not group["capturable"]:
                self._read_counters()   # numbered steps from here on
                group.pop("counter")
            by_step = {}                # parameters that have been stepped equally often
            for p in ps:
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW: sparse gradients are not supported")
                st = self.state[p]
                if not st:
                    if not p.is_cuda:
                        raise RuntimeError(f"AdamW: this optimizer runs on the GPU only (got a parameter on {p.device})")
                    if capturing:
                        raise RuntimeError("AdamW: the first step makes the states; make it before the capture")
                    st["step"] = 0
                    st.update(self._fresh(p, group["state_bits"]))
                by_step.setdefault(st["step"], []).append(p)
            counter = None
            if group["capturable"]:
                if len(by_step) != 1:
                    raise RuntimeError("AdamW: with capturable=True all parameters of a group are stepped together")
                counter = group.get("counter")
                if counter is None:
                    if capturing:
                        raise RuntimeError("AdamW: make a step before the capture (it makes the counter on the device)")
                    counter = group["counter"] = torch.tensor([next(iter(by_step)), 0, 0, 0], dtype=torch.int32, device=ps[0].device)
            for k, (made, members) in enumerate(sorted(by_step.items(), key=lambda kv: kv[0])):
                plan = self._plan((gi, k), members, group["state_bits"])
                if capturing:
                    self._recorded.append((plan, counter))
                grads = [p.grad if p.grad.is_contiguous() else p.grad.contiguous() for p in members]
                with torch.cuda.device(members[0].device):
                    plan.step(grads, made + 1, float(group["lr"]), group["betas"][0], group["betas"][1], group["eps"],
                              group["weight_decay"], seed=group["seed"] + gi, step_dev=counter)
                torch.autograd.graph.increment_version(members)      # a backward pass that saved them says so
                if counter is None:
                    for p in members:
                        self.state[p]["step"] = made + 1
        return loss

    def state_dict(self):
        """As torch's, with the steps counted on the device written into each `step`."""
        self._read_counters()
        sd = super().state_dict()
        for g in sd["param_groups"]:
            g.pop("counter", None)
        return sd

    def _read_counters(self):
        for group in self.param_groups:
            if group.get("counter") is not None:
                made = int(group["counter"][0])
                for p in group["params"]:
                    if self.state[p]:
                        self.state[p]["step"] = made

    def load_state_dict(self, state_dict):
        """States keep the types they are held in (torch's own loading would cast codes and scales to the parameter's) and, where
        they are there already, their memory: a captured step goes on from what was loaded."""
        had = {}

        def take(_, state_dict):        # the last of the hooks before: torch loads the groups alone
            had.update(saved=self._checked(state_dict), held=dict(self.state), counters=[g.get("counter") for g in self.param_groups],
                       own=[{k: g[k] for k in self.defaults} for g in self.param_groups],
                       ids=[i for g in state_dict["param_groups"] for i in g["params"]])
            return {**state_dict, "state": {}}

        def give(_):                    # the first of those after
            self._take_over(**had)
        hooks = [self.register_load_state_dict_pre_hook(take), self.register_load_state_dict_post_hook(give, prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _checked(self, state_dict):
        """The saved states, refused before anything is changed if they do not fit."""
        saved = state_dict["state"]
        for own, g in zip(self.param_groups, state_dict["param_groups"]):
            _honoured(g)
            for i, p in zip(g["params"], own["params"]):
                b = g.get("state_bits", own["state_bits"])
                for name, (dtype, n) in self._layout(p, b).items() if i in saved else ():
                    t = saved[i].get(name)
                    if t is None or t.dtype != dtype or t.numel() != n:
                        raise ValueError(f"AdamW: the saved state holds no {name} of {n} elements in {dtype}")
        return saved

    def _take_over(self, saved, held, counters, own, ids):
        for g, options in zip(self.param_groups, own):      # those that another AdamW's groups do not have stay
            for k, v in options.items():
                g.setdefault(k, v)
            if "decoupled_weight_decay" in g:
                g["decoupled_weight_decay"] = True
        ps = [p for g in self.param_groups for p in g["params"]]
        bits = [g["state_bits"] for g in self.param_groups for _ in g["params"]]
        loaded = {}
        for i, p, b in zip(ids, ps, bits):
            if i not in saved:
                continue
            st, had = saved[i], held.get(p, {})
            new = {"step": int(st["step"])}
            for name, like in self._fresh(p, b).items():
                there = had.get(name)
                new[name] = there if there is not None and there.dtype == like.dtype and there.numel() == like.numel() else like
                loaded[p, name] = st[name].detach().reshape(-1)
            self.state[p] = new
        for (p, name), t in loaded.items():
            self.state[p][name].view(torch.uint8).copy_(t.contiguous().view(torch.uint8))
        for group, counter in zip(self.param_groups, counters):
            steps = {self.state[p]["step"] for p in group["params"] if p in self.state}
            group.pop("counter", None)
            if counter is not None and len(steps) == 1:         # a captured step reads it, whatever these groups say
                counter.copy_(torch.tensor([steps.pop(), 0, 0, 0], dtype=torch.int32))
                if group["capturable"]:
                    group["counter"] = counter
        self._plans = {}


__all__ = ["AdamW", "PganError"]
