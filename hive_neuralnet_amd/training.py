"""Training HiveFNN on the device operators.

The step that the reference's trainer takes with torch's operators
(hive_fnn/fnn_trainer.py:531-600 over fnn_network.py:175-253): a sampled
FNNTrainingBatch -> features of the roots and of every legal successor
(build_forward_batch) -> the network, its layer norms with the sigmoid in
front of them in one kernel -> the policy and value loss over the ragged
legal lists, with its gradient -> one AdamW launch for all weights.

    optimizer = AdamW(net.parameters(), lr=1e-3)           # moments in 32 bits; state_bits=8 in 8
    losses = train_batch(net, optimizer, buffer.sample_batch(2048))   # [total, policy, value], on the device

    python -m hive_neuralnet_amd.training --steps 50 --batch 2048     # the same on synthetic targets

layer_norm and policy_value_loss are autograd functions over the entry points
of training_ops.py, differentiable once, without rules for vmap, forward mode
or tensors that hold no memory; AdamW is a torch.optim.Optimizer of contiguous
parameters.
"""
from __future__ import annotations

import torch

from . import hive_gpu
from .fnn import HiveFNN
from .replay import FNNTrainingBatch, build_forward_batch


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, activation):
        y, mean, rstd = hive_gpu.load_extension().layer_norm_forward(x, weight, bias, eps, activation)
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        ctx.activation = activation
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, mean, rstd = ctx.saved_tensors
        dx, dw, db = hive_gpu.load_extension().layer_norm_backward(
            dy.contiguous(), x, mean, rstd, weight, bias, ctx.activation, need_dx=ctx.needs_input_grad[0])
        return dx, dw, db, None, None


def layer_norm(x: torch.Tensor, weight=None, bias=None, eps: float = 1e-5, activation=None) -> torch.Tensor:
    """Layer norm over the last dimension of x (activation="sigmoid": of
    sigmoid(x)), differentiable once in x, weight and bias."""
    return _LayerNorm.apply(x, weight, bias, eps, activation)


class _PolicyValueLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, values, num_actions, targets, pw, vt, vw, value_coef, loss_scale):
        # the gradient is held in 32 bits, so that what comes in (a scaler's factor) meets it before it is rounded
        ctx.types = logits.dtype, values.dtype
        logits, values = (t.float() if t.dtype in (torch.float16, torch.bfloat16) else t for t in (logits, values))
        losses, dlogits, dvalues = hive_gpu.load_extension().policy_value_loss(
            logits, values, num_actions, targets, pw, vt, vw, value_coef, loss_scale)
        ctx.save_for_backward(dlogits, dvalues)
        total, policy, value = losses.unbind(0)
        ctx.mark_non_differentiable(policy, value)
        return total.clone(), policy, value

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _policy, _value):
        dlogits, dvalues = ctx.saved_tensors
        return (dlogits * grad).to(ctx.types[0]), (dvalues * grad).to(ctx.types[1]), *([None] * 7)


def policy_value_loss(logits, values, num_actions, policy_targets, policy_weights, value_targets, value_weights,
                      value_coef: float = 1.0, loss_scale: float = 1.0):
    """(total, policy, value) of HiveGpuExtension.policy_value_loss; total is
    differentiable in logits and values (its gradients times loss_scale, which
    total itself is not multiplied by; rounded to 16 bits once, after the
    incoming gradient, so that a scaled total needs no loss_scale)."""
    return _PolicyValueLoss.apply(logits, values, num_actions, policy_targets, policy_weights, value_targets,
                                  value_weights, value_coef, loss_scale)


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay, all parameters of a group and type
    in one launch, the moments in 32 bits or, with state_bits=8, in 8
    (AdamWPlan).  A parameter without a gradient is left as it is, and the
    bias correction is that of the steps it has taken itself (parameters of
    one group and type that have taken different numbers of them take a
    launch each number).  `seed` seeds the rounding of 8-bit moments; each
    step takes the next one."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
                 state_bits: int = 32, seed: int = 0):
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self._ext = hive_gpu.load_extension()
        self.state_bits, self.seed, self.steps = state_bits, int(seed), 0
        self._plans: list = []  # (group, plan, the steps that each of its parameters has taken)
        self._make_plans(None)

    def _make_plans(self, states, taken=None) -> None:
        plans = []
        for group in self.param_groups:
            by_type: dict = {}
            for p in group["params"]:
                by_type.setdefault(p.dtype, []).append(p)
            for members in by_type.values():
                state = None
                if states is not None:
                    if len(plans) >= len(states):
                        raise ValueError("the saved state has fewer parameter lists than the optimizer")
                    state = {k: v.to(members[0].device, copy=True) for k, v in states[len(plans)].items()}
                plan = self._ext.prepare_adamw(members, self.state_bits, state)
                plans.append((group, plan, [0] * len(members) if taken is None else list(taken[len(plans)])))
        if states is not None and len(states) != len(plans):
            raise ValueError(f"the saved state has {len(states)} parameter lists, the optimizer {len(plans)}")
        self._plans = plans

    def add_param_group(self, param_group) -> None:
        if getattr(self, "_plans", None):
            raise ValueError("AdamW's parameters are fixed when it is made")
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        for key in ("lr", "eps", "weight_decay"):
            if not group[key] >= 0.0:
                raise ValueError(f"{key} must not be negative, got {group[key]}")
        if not all(0.0 <= beta < 1.0 for beta in group["betas"]):
            raise ValueError(f"betas must be in [0, 1), got {group['betas']}")

    @torch.no_grad()
    def step(self, closure=None, grad_scale: torch.Tensor | None = None):
        """One step from the parameters' gradients, times grad_scale[0] (a
        float32 tensor on the device) where given."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        seed = self.seed + self.steps + 1
        for group, plan, taken in self._plans:
            grads = [None if p.grad is None else p.grad.contiguous() for p in plan.params]
            for number in sorted({n for n, g in zip(taken, grads) if g is not None}, reverse=True):
                now = [g if n == number else None for n, g in zip(taken, grads)]
                plan.step(now, number + 1, lr=group["lr"], betas=group["betas"], eps=group["eps"],
                          weight_decay=group["weight_decay"], grad_scale=grad_scale, seed=seed)
                taken[:] = [n if g is None else n + 1 for n, g in zip(taken, now)]
        self.steps += 1
        return loss

    def __getstate__(self):
        """For copies and pickles: what the base class has and the moments (codes as bytes: a plain pickle knows no
        float8), from which a copy lays out its own plans."""
        return {**super().__getstate__(), "adamw": {
            "state_bits": self.state_bits, "seed": self.seed, "steps": self.steps,
            "states": [{k: t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for k, t in plan.state.items()}
                       for _, plan, _ in self._plans],
            "taken": [list(taken) for _, _, taken in self._plans]}}

    def __setstate__(self, state) -> None:
        own = state["adamw"]
        super().__setstate__({k: v for k, v in state.items() if k != "adamw"})
        self._ext = hive_gpu.load_extension()
        self.state_bits, self.seed, self.steps = own["state_bits"], own["seed"], own["steps"]
        self._make_plans([{k: t.view(torch.float8_e4m3fn) if t.dtype == torch.uint8 else t for k, t in held.items()}
                          for held in own["states"]], own["taken"])

    def state_dict(self):
        """The moments as they are held, the numbers of steps, the groups' settings."""
        for hook in self._optimizer_state_dict_pre_hooks.values():
            hook(self)
        groups = [{k: v for k, v in g.items() if k != "params"} for g in self.param_groups]
        saved = {"state_bits": self.state_bits, "seed": self.seed, "steps": self.steps,
                 "states": [dict(plan.state) for _, plan, _ in self._plans],
                 "taken": [list(taken) for _, _, taken in self._plans], "sizes": self._sizes(), "param_groups": groups}
        for hook in self._optimizer_state_dict_post_hooks.values():
            changed = hook(self, saved)
            saved = saved if changed is None else changed
        return saved

    def _sizes(self) -> list:
        return [[p.numel() for p in plan.params] for _, plan, _ in self._plans]

    def load_state_dict(self, state_dict) -> None:
        state_dict = dict(state_dict)  # a hook may change its entries
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            changed = hook(self, state_dict)
            state_dict = state_dict if changed is None else changed
        if state_dict["state_bits"] != self.state_bits:
            raise ValueError(f"the saved moments are in {state_dict['state_bits']} bits, these in {self.state_bits}")
        if len(state_dict["param_groups"]) != len(self.param_groups):
            raise ValueError(f"{len(state_dict['param_groups'])} saved groups, {len(self.param_groups)} here")
        if state_dict.get("sizes", self._sizes()) != self._sizes():
            raise ValueError("the saved state is of parameters of other sizes")
        taken = state_dict.get("taken")  # None: saved when one number served all
        if taken is None:
            taken = [[state_dict["steps"]] * len(plan.params) for _, plan, _ in self._plans]
        self._make_plans(state_dict["states"], taken)
        for group, saved in zip(self.param_groups, state_dict["param_groups"]):
            group.update(saved)
        self.seed, self.steps = state_dict["seed"], state_dict["steps"]
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)


def encode(net: HiveFNN, features: torch.Tensor) -> torch.Tensor:
    """HiveFNN.encode, the sigmoid and the layer norm in one kernel (where ln1
    is another module, or has hooks, as the module has it)."""
    h, norm = net.fc1(features), net.ln1
    if type(norm) is not torch.nn.LayerNorm or norm.normalized_shape != h.shape[-1:] or norm._forward_hooks or \
            norm._forward_pre_hooks or norm._backward_hooks or norm._backward_pre_hooks:
        return net.fc2(norm(torch.sigmoid(h)))
    return net.fc2(layer_norm(h, norm.weight, norm.bias, norm.eps, "sigmoid"))


def forward(net: HiveFNN, root_features, successor_features, action_to_root):
    """HiveFNN.forward on the training operators: (action_logits [N],
    root_values [B, 1]).  Hooks of the layers run, those of net itself do not."""
    root = encode(net, root_features)
    values = net.value_head(root)
    if action_to_root.shape[0] == 0:
        return values.new_zeros((0,)), values
    return net.score_actions(root[action_to_root], encode(net, successor_features)), values


def train_batch(net: HiveFNN, optimizer, batch: FNNTrainingBatch, value_coef: float = 1.0) -> torch.Tensor:
    """One training step on a sampled batch; returns [total, policy, value]
    (float32, on the device: reading them waits for the step)."""
    ext = hive_gpu.load_extension()
    B = int(batch.num_actions.shape[0])
    root, succ, action_to_root, num_actions = build_forward_batch(
        ext, batch.state_bytes, B, batch.num_actions, batch.root_features, batch.legal_moves)
    logits, values = forward(net, root, succ, action_to_root)
    losses, dlogits, dvalues = ext.policy_value_loss(
        logits.detach(), values.detach(), num_actions, batch.policy_targets, batch.policy_mask, batch.value_targets,
        batch.value_mask * batch.value_weights, value_coef)
    optimizer.zero_grad(set_to_none=True)
    trained = [(head, grad) for head, grad in ((logits, dlogits), (values, dvalues)) if head.requires_grad]
    if not trained:
        raise RuntimeError("nothing of the network requires a gradient")
    torch.autograd.backward([head for head, _ in trained], [grad for _, grad in trained])
    optimizer.step()
    return losses


def synthetic_batch(batch_size: int, expansion_mask: int = 0, max_ply: int = 120, seed: int = 0) -> FNNTrainingBatch:
    """Seeded random-play positions with random searched policies and results."""
    ext = hive_gpu.load_extension()
    B = int(batch_size)
    states, _ = hive_gpu.random_positions(B, expansion_mask, max_ply, seed)
    legal, n, features = ext.generate_legal_moves_and_fnn_features_batch(states, B)
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    live = torch.arange(legal.shape[1], device="cuda") < n.unsqueeze(1)
    policy = torch.rand(live.shape, generator=g, device="cuda").pow(6) * live
    ones = torch.ones((B, 1), device="cuda")
    return FNNTrainingBatch(states, policy / policy.sum(1, keepdim=True).clamp(min=1e-30), n.to(torch.int64),
                            torch.randint(-1, 2, (B, 1), generator=g, device="cuda").float(), ones, ones, ones,
                            features, legal)


def main() -> None:
    import argparse
    import time

    from .fnn import FNNConfig
    ap = argparse.ArgumentParser(description="train HiveFNN on synthetic targets")
    ap.add_argument("--steps", type=int, default=50)
    ap.add_argument("--batch", type=int, default=2048)
    ap.add_argument("--lr", type=float, default=1e-2)
    ap.add_argument("--state-bits", type=int, default=32, choices=(32, 8))
    a = ap.parse_args()
    torch.manual_seed(0)
    net = HiveFNN(FNNConfig.large()).cuda()
    optimizer = AdamW(net.parameters(), lr=a.lr, state_bits=a.state_bits)
    batch = synthetic_batch(a.batch)
    for i in range(a.steps):
        t = time.perf_counter()
        total, policy, value = train_batch(net, optimizer, batch).tolist()
        if i % max(1, a.steps // 10) == 0 or i == a.steps - 1:
            print(f"step {i:4d}  total {total:.4f}  policy {policy:.4f}  value {value:.4f}  "
                  f"{(time.perf_counter() - t) * 1e3:.2f} ms", flush=True)


if __name__ == "__main__":
    main()
