"""AdamW over flat buffers with the clip folded in, and Muon for the blocks' matrices.

``FusedAdamW`` presents the ``torch.optim.AdamW`` interface (``param_groups``,
``state``, ``state_dict`` / ``load_state_dict`` with the same keys and layout) so
checkpoints stay interchangeable with the reference (src/llmlab/train.py:169-170,
265-275), but on a B200 with a fused model it performs the whole update - gradient
clipping coefficient, AdamW on fp32 master weights and moments, and the bf16
shadow refresh - as one pass over HBM instead of the reference's clip + foreach
sequence.  Everywhere else it falls back to ``torch.optim.AdamW`` math on the
same state tensors.

``clip_and_step(max_norm)`` is the fused entry point: it returns the global
gradient norm as a device scalar without a host synchronisation.

``FusedMuon`` replaces AdamW's update of the blocks' weight matrices by their momentum with its
singular values moved next to one (ops/newton_schulz.py); embeddings, head and norms keep AdamW.
The reference has no counterpart.
"""

from __future__ import annotations

import torch

from .ops import functional as K
from .ops import lib as _lib
from .ops import newton_schulz as NS


class FusedAdamW(torch.optim.AdamW):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
                 engine=None):
        super().__init__(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                         foreach=False, fused=False)
        self.engine = engine
        self._flat_state = None
        self._step_count = 0

    # -------------------------------------------------------------- fused path --
    def _fused_ready(self) -> bool:
        engine = self.engine
        if engine is None or not _lib.available() or engine.flat_grad is None:
            return False
        if len(self.param_groups) != 1:
            return False
        params = self.param_groups[0]["params"]
        if len(params) != len(engine.params) or {id(p) for p in params} != set(engine.offsets):
            return False
        # Every gradient must already live in the flat buffer.
        for p in engine.params:
            if p.grad is None or p.grad.data_ptr() != engine.grad_view(p).data_ptr():
                return False
        return True

    def _ensure_flat_state(self) -> None:
        if self._flat_state is not None:
            return
        engine = self.engine
        exp_avg = torch.zeros_like(engine.flat_param)
        exp_avg_sq = torch.zeros_like(engine.flat_param)
        steps = torch.zeros(len(engine.params), dtype=torch.float32, device="cpu")
        for i, p in enumerate(engine.params):
            existing = self.state.get(p, {})
            m, v = engine._slice(exp_avg, p), engine._slice(exp_avg_sq, p)
            if "exp_avg" in existing:
                m.copy_(existing["exp_avg"])
                v.copy_(existing["exp_avg_sq"])
                steps[i] = float(existing["step"])
            # 0-d CPU step counters, as torch.optim.AdamW keeps them.
            self.state[p] = {"step": steps[i], "exp_avg": m, "exp_avg_sq": v}
        self._flat_state = (exp_avg, exp_avg_sq, steps)
        self._step_count = int(steps.max().item()) if len(steps) else 0

    @torch.no_grad()
    def clip_and_step(self, max_norm: float, error_if_nonfinite: bool = True) -> torch.Tensor:
        """Clip by global norm and update.  Returns the pre-clip norm (device scalar).

        On the fused path a non-finite norm skips the update on the device and the
        caller finds out when it reads the returned norm; the portable path raises
        like ``clip_grad_norm_(error_if_nonfinite=True)``.
        """
        if not self._fused_ready():
            params = [p for g in self.param_groups for p in g["params"]]
            norm = torch.nn.utils.clip_grad_norm_(params, max_norm,
                                                  error_if_nonfinite=error_if_nonfinite)
            self.step()
            return norm
        engine = self.engine
        self._ensure_flat_state()
        exp_avg, exp_avg_sq, steps = self._flat_state
        group = self.param_groups[0]
        stats = K.grad_norm_and_coef(engine.flat_grad[:engine.total], max_norm)
        self._step_count = int(steps[0].item()) + 1
        steps += 1
        beta1, beta2 = group["betas"]
        K.adamw_step(engine.flat_param, engine.flat_grad, exp_avg, exp_avg_sq, engine.flat_shadow,
                     step=self._step_count, lr=group["lr"], beta1=beta1, beta2=beta2,
                     eps=group["eps"], weight_decay=group["weight_decay"], coef=stats[1:2],
                     ok_flag=stats[2:3])
        engine.mark_shadow_current()
        return stats[0]

    @torch.no_grad()
    def step_with_stats(self, stats: torch.Tensor) -> torch.Tensor:
        """Update with a clip coefficient that is already on the device.

        ``stats`` is ``[norm, coefficient, finite flag]`` as produced by the fused
        gradient reduction (``BucketedDDP.finish``); returns the norm.
        """
        if not self._fused_ready():
            raise RuntimeError("step_with_stats needs gradients in the engine's flat buffer")
        engine = self.engine
        self._ensure_flat_state()
        exp_avg, exp_avg_sq, steps = self._flat_state
        group = self.param_groups[0]
        self._step_count = int(steps[0].item()) + 1
        steps += 1
        beta1, beta2 = group["betas"]
        K.adamw_step(engine.flat_param, engine.flat_grad, exp_avg, exp_avg_sq, engine.flat_shadow,
                     step=self._step_count, lr=group["lr"], beta1=beta1, beta2=beta2,
                     eps=group["eps"], weight_decay=group["weight_decay"], coef=stats[1:2],
                     ok_flag=stats[2:3])
        engine.mark_shadow_current()
        return stats[0]

    @torch.no_grad()
    def step(self, closure=None):
        if self._flat_state is not None and self._fused_ready():
            # Gradients were clipped (or not) by the caller; plain update.
            engine = self.engine
            exp_avg, exp_avg_sq, steps = self._flat_state
            group = self.param_groups[0]
            self._step_count = int(steps[0].item()) + 1
            steps += 1
            beta1, beta2 = group["betas"]
            K.adamw_step(engine.flat_param, engine.flat_grad, exp_avg, exp_avg_sq,
                         engine.flat_shadow, step=self._step_count, lr=group["lr"], beta1=beta1,
                         beta2=beta2, eps=group["eps"], weight_decay=group["weight_decay"])
            engine.mark_shadow_current()
            return None
        return super().step(closure)

    def load_state_dict(self, state_dict) -> None:
        super().load_state_dict(state_dict)
        # Loaded tensors are fresh copies; re-home them in the flat buffers lazily.
        self._flat_state = None


class FusedMuon(torch.optim.Optimizer):
    """Muon for weight matrices, AdamW for everything else.

    Matrices:  ``v <- momentum v + g``, ``u = g + momentum v``,
    ``W <- (1 - lr weight_decay) W - lr 0.2 sqrt(max(m, n)) NewtonSchulz(u)``.  The factor gives the
    update the root mean square of a typical AdamW update, so both parts share one learning rate
    and schedule.  Others: AdamW as in ``FusedAdamW``.

    On a B200 with a fused model the matrices of one kind of all layers are one stack inside the
    engine's flat buffers: one momentum kernel, one Newton-Schulz call and one update kernel (which
    also writes the bf16 shadow) per kind and step.  Elsewhere the same is done in PyTorch operators.
    """

    def __init__(self, matrices, others, lr=1e-3, momentum=0.95, nesterov=True, steps=5,
                 betas=(0.9, 0.95), eps=1e-8, weight_decay=0.0, engine=None):
        matrices, others = list(matrices), list(others)
        if any(p.dim() != 2 for p in matrices):
            raise ValueError("Muon updates matrices only")
        if not 0 <= momentum < 1:
            raise ValueError("momentum must be in [0, 1)")
        if not isinstance(steps, int) or not 1 <= steps <= NS.MAX_STEPS:
            raise ValueError(f"steps must be an integer in [1, {NS.MAX_STEPS}]")
        if lr < 0 or weight_decay < 0:
            raise ValueError("lr and weight_decay must be nonnegative")
        shared = dict(lr=lr, weight_decay=weight_decay)
        groups = [dict(params=matrices, kind="muon", momentum=momentum, nesterov=nesterov,
                       steps=steps, **shared),
                  dict(params=others, kind="adamw", betas=tuple(betas), eps=eps, **shared)]
        super().__init__([g for g in groups if g["params"]], shared)
        self.engine = engine
        self._flat_state = None

    @classmethod
    def from_model(cls, model, **kwargs):
        """Matrices of the blocks to Muon; embeddings, head and norms to AdamW."""
        matrices = [p for layer in model.layers for p in layer.parameters() if p.dim() == 2]
        chosen = {id(p) for p in matrices}
        return cls(matrices, [p for p in model.parameters() if id(p) not in chosen], **kwargs)

    # -------------------------------------------------------------- fused path --
    def _fused_ready(self) -> bool:
        engine = self.engine
        if engine is None or not _lib.available() or engine.flat_grad is None:
            return False
        params = [p for g in self.param_groups for p in g["params"]]
        if len(params) != len(engine.params) or {id(p) for p in params} != set(engine.offsets):
            return False
        return all(p.grad is not None and p.grad.data_ptr() == engine.grad_view(p).data_ptr()
                   for p in engine.params)

    def _stacks(self) -> list:
        """``(first parameter, layers, matrices per layer)`` of each stack: adjacent matrices of one
        shape in a layer (q|k|v|output, w1|w3), repeated at one distance from layer to layer."""
        engine = self.engine
        muon = {id(p) for g in self.param_groups if g["kind"] == "muon" for p in g["params"]}
        runs_of_layers = []
        for begin, end in engine.layer_ranges:
            inside = [p for p in engine.params
                      if id(p) in muon and begin <= engine.offsets[id(p)] < end]
            inside.sort(key=lambda p: engine.offsets[id(p)])
            runs = []
            for p in inside:
                last = runs[-1][-1] if runs else None
                if (last is not None and last.shape == p.shape
                        and engine.offsets[id(last)] + last.numel() == engine.offsets[id(p)]):
                    runs[-1].append(p)
                else:
                    runs.append([p])
            runs_of_layers.append(runs)
        stacks = []
        for same in zip(*runs_of_layers):
            offsets = [engine.offsets[id(run[0])] for run in same]
            step = offsets[1] - offsets[0] if len(offsets) > 1 else 0
            even = (all(b - a == step for a, b in zip(offsets, offsets[1:]))
                    and len({(len(run), run[0].shape) for run in same}) == 1)
            if even:
                stacks.append((offsets[0], len(same), step, len(same[0]), *same[0][0].shape))
            else:
                stacks += [(offset, 1, 0, len(run), *run[0].shape)
                           for offset, run in zip(offsets, same)]
        covered = sum(layers * per * m * n for _, layers, _, per, m, n in stacks)
        if covered != sum(p.numel() for g in self.param_groups if g["kind"] == "muon"
                          for p in g["params"]):
            raise RuntimeError("a Muon matrix lies outside the blocks")
        return stacks

    def _ranges(self, params) -> list:
        """Maximal runs ``(begin, end)`` of the AdamW parameters in the flat buffers."""
        engine = self.engine
        runs = []
        for p in sorted(params, key=lambda p: engine.offsets[id(p)]):
            begin = engine.offsets[id(p)]
            end = begin + p.numel()
            if runs and runs[-1][1] == begin:
                runs[-1][1] = end
            else:
                runs.append([begin, end])
        return runs

    def _ensure_flat_state(self) -> None:
        if self._flat_state is not None:
            return
        engine = self.engine
        # One buffer in the engine's layout: momentum of the matrices, first moment of the others.
        first = torch.zeros_like(engine.flat_param)
        others = [p for g in self.param_groups if g["kind"] == "adamw" for p in g["params"]]
        ranges, cursor = [], 0
        for begin, end in self._ranges(others):
            ranges.append((begin, end, cursor))
            cursor += -(-(end - begin) // 64) * 64
        second = torch.zeros(max(cursor, 1), dtype=torch.float32, device=first.device)
        self._step_count = 0
        for group in self.param_groups:
            for p in group["params"]:
                existing = self.state.get(p, {})
                held = {"step": torch.tensor(float(existing.get("step", 0.0)))}
                begin = engine.offsets[id(p)]
                if group["kind"] == "muon":
                    held["momentum_buffer"] = engine._slice(first, p)
                else:
                    held["exp_avg"] = engine._slice(first, p)
                    base = next(at + begin - lo for lo, hi, at in ranges if lo <= begin < hi)
                    held["exp_avg_sq"] = second[base:base + p.numel()].view(p.shape)
                for name, tensor in held.items():
                    if name != "step" and name in existing:
                        tensor.copy_(existing[name])
                self._step_count = max(self._step_count, int(held["step"].item()))
                self.state[p] = held
        self._flat_state = (first, second, ranges, self._stacks())

    @torch.no_grad()
    def _fused_update(self, coef, ok_flag) -> None:
        self._ensure_flat_state()
        engine = self.engine
        first, second, ranges, stacks = self._flat_state
        groups = {g["kind"]: g for g in self.param_groups}
        self._step_count += 1
        for held in self.state.values():
            held["step"] += 1
        muon = groups.get("muon")
        for offset, layers, step, per, m, n in stacks:
            length = per * m * n
            rows = lambda flat: flat.as_strided((layers, length), (max(step, length), 1),
                                                flat.storage_offset() + offset)
            update = torch.empty(layers, per, m, n, dtype=torch.float32, device=first.device)
            NS.muon_momentum(rows(engine.flat_grad), rows(first), update,
                             momentum=muon["momentum"], nesterov=muon["nesterov"], coef=coef,
                             ok_flag=ok_flag)
            direction = NS.newton_schulz(update, steps=muon["steps"])
            NS.muon_apply(rows(engine.flat_param), rows(engine.flat_shadow), direction,
                          decay=1.0 - muon["lr"] * muon["weight_decay"],
                          rate=muon["lr"] * 0.2 * max(m, n) ** 0.5, ok_flag=ok_flag)
        adamw = groups.get("adamw")
        if adamw is not None:
            beta1, beta2 = adamw["betas"]
            for begin, end, at in ranges:
                K.adamw_step(engine.flat_param[begin:end], engine.flat_grad[begin:end],
                             first[begin:end], second[at:at + end - begin],
                             engine.flat_shadow[begin:end], step=self._step_count, lr=adamw["lr"],
                             beta1=beta1, beta2=beta2, eps=adamw["eps"],
                             weight_decay=adamw["weight_decay"], coef=coef, ok_flag=ok_flag)
        engine.mark_shadow_current()

    # ------------------------------------------------------------ entry points --
    @torch.no_grad()
    def clip_and_step(self, max_norm: float, error_if_nonfinite: bool = True) -> torch.Tensor:
        """As ``FusedAdamW.clip_and_step``: clip by global norm, update, return the norm."""
        if not self._fused_ready():
            params = [p for g in self.param_groups for p in g["params"]]
            norm = torch.nn.utils.clip_grad_norm_(params, max_norm,
                                                  error_if_nonfinite=error_if_nonfinite)
            self.step()
            return norm
        stats = K.grad_norm_and_coef(self.engine.flat_grad[:self.engine.total], max_norm)
        return self.step_with_stats(stats)

    @torch.no_grad()
    def step_with_stats(self, stats: torch.Tensor) -> torch.Tensor:
        """As ``FusedAdamW.step_with_stats``."""
        if not self._fused_ready():
            raise RuntimeError("step_with_stats needs gradients in the engine's flat buffer")
        self._fused_update(stats[1:2], stats[2:3])
        return stats[0]

    @torch.no_grad()
    def step(self, closure=None):
        if self._flat_state is not None and self._fused_ready():
            self._fused_update(None, None)      # gradients were clipped (or not) by the caller
            return None
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                state["step"] = state.get("step", torch.tensor(0.0)) + 1
                p.mul_(1.0 - group["lr"] * group["weight_decay"])
                if group["kind"] == "muon":
                    v = state.setdefault("momentum_buffer", torch.zeros_like(p))
                    v.mul_(group["momentum"]).add_(p.grad)
                    u = p.grad + group["momentum"] * v if group["nesterov"] else v
                    direction = NS.newton_schulz_portable(u, steps=group["steps"])
                    p.add_(direction, alpha=-group["lr"] * 0.2 * max(p.shape) ** 0.5)
                    continue
                m = state.setdefault("exp_avg", torch.zeros_like(p))
                v = state.setdefault("exp_avg_sq", torch.zeros_like(p))
                beta1, beta2 = group["betas"]
                count = float(state["step"])
                m.lerp_(p.grad, 1 - beta1)
                v.mul_(beta2).addcmul_(p.grad, p.grad, value=1 - beta2)
                scale = (v.sqrt() / (1 - beta2 ** count) ** 0.5).add_(group["eps"])
                p.addcdiv_(m, scale, value=-group["lr"] / (1 - beta1 ** count))
        return loss

    def load_state_dict(self, state_dict) -> None:
        super().load_state_dict(state_dict)
        # Loaded tensors are fresh copies; re-home them in the flat buffers lazily.
        self._flat_state = None
