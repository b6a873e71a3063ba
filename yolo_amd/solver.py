"""Optimizer and learning-rate schedule of the training entry point, with detectron2's defaults for the keys the
reference's configs set (tools/train_net.py builds both through detectron2's DefaultTrainer: SGD with momentum,
no weight decay on normalisation parameters, WarmupMultiStepLR).  The update is one kernel over the training
engine's flat arenas when every parameter lives there, torch's own step otherwise.  SOLVER.CLIP_GRADIENTS (detectron2's key)
clips the gradients in front of the update: by value, by the norm of each tensor, or by the norm of all of them."""
from __future__ import annotations

from bisect import bisect_right
from typing import List, Optional, Sequence, Tuple

import torch

from . import ops

CLIP_TYPES = ("value", "norm", "full_model")


def _check_clip(clip_type: str, clip_value: float, norm_type: float) -> Tuple[str, float, float]:
    if clip_type not in CLIP_TYPES:
        raise ValueError(f"gradient clipping by {clip_type!r}: one of {', '.join(CLIP_TYPES)}")
    clip_value, norm_type = float(clip_value), float(norm_type)
    if not clip_value >= 0.0:
        raise ValueError(f"gradient clipping: CLIP_VALUE {clip_value} has to be 0 or more")
    if clip_type != "value" and norm_type not in (1.0, 2.0, float("inf")):
        raise ValueError(f"gradient clipping: NORM_TYPE {norm_type} (1, 2 and inf are built)")
    return clip_type, clip_value, norm_type


class GradientClipper:
    """Clips a fixed set of gradient tensors, call after call: ``clip_type`` "value" (each element to [-clip_value,
    clip_value]), "norm" (each tensor to norm clip_value) or "full_model" (all tensors together to norm clip_value), as
    detectron2's SOLVER.CLIP_GRADIENTS.CLIP_TYPE.  The tensors (f32 or bf16, one device) must stay in place: it holds them
    and a device table of their addresses, built once.  Its buffers belong to one call at a time (one stream)."""

    def __init__(self, grads: Sequence[torch.Tensor], clip_type: str, clip_value: float, norm_type: float = 2.0):
        self.clip_type, self.clip_value, self.norm_type = _check_clip(clip_type, clip_value, norm_type)
        grads = list(grads)
        self.per_tensor = clip_type == "norm"
        self.norms = self.coefs = self._ws = None
        if clip_type != "value" and grads:   # filled by the time the table's synchronous copy is done: any stream may come next
            n = len(grads) if self.per_tensor else 1
            self.norms, self.coefs = torch.ones(2, n, device=grads[0].device)
        self.table = ops.grad_table(grads)
        self.device = self.table.blocks.device
        if self.norms is not None:
            self._ws = torch.empty(ops.grad_norm_workspace_bytes(self.table), dtype=torch.uint8, device=self.device)

    @ops.on_own_device
    def measure(self) -> Optional[torch.Tensor]:
        """The norms the clipping goes by ([1] or [n_tensors], overwritten by the next call; ``coefs`` has the factors);
        None for "value".  The gradients are only read."""
        if self.clip_type == "value":
            return None
        ops.grad_norm(self.table, self.norms, self._ws, norm_type=self.norm_type, per_tensor=self.per_tensor,
                      max_norm=self.clip_value, coefs=self.coefs)
        return self.norms

    @ops.on_own_device
    def clip_(self) -> Optional[torch.Tensor]:
        """measure(), and the gradients clipped in place."""
        if self.clip_type == "value":
            ops.grad_clamp(self.table, self.clip_value)
            return None
        ops.grad_clip(self.table, self.norms, self.coefs, self._ws, max_norm=self.clip_value, norm_type=self.norm_type,
                      per_tensor=self.per_tensor)
        return self.norms


def _grads(parameters) -> List[torch.Tensor]:
    ps = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    seen, out = set(), []
    for p in ps:   # a parameter listed twice is clipped once
        if p.grad is not None and id(p) not in seen:
            seen.add(id(p))
            out.append(p.grad)
    return out


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0) -> torch.Tensor:
    """torch.nn.utils.clip_grad_norm_ for gradients on the GPU: scales them in place so that their common norm (1, 2 or inf)
    is at most ``max_norm`` and returns the norm it was, as a 0-d tensor that nothing has read back.  Each call builds the
    table of the gradients and copies it synchronously (the host waits for what is queued before it; not in a captured
    graph): a training loop that keeps its gradient tensors saves that with a GradientClipper."""
    grads = _grads(parameters)
    if not grads:
        return torch.zeros(())
    return GradientClipper(grads, "full_model", max_norm, norm_type).clip_()[0]


@torch.no_grad()
def clip_grad_value_(parameters, clip_value: float) -> None:
    """torch.nn.utils.clip_grad_value_ for gradients on the GPU: each element to [-clip_value, clip_value], in place."""
    grads = _grads(parameters)
    if grads:
        GradientClipper(grads, "value", clip_value).clip_()


class ArenaSGD(torch.optim.SGD):
    """torch.optim.SGD whose step is ONE kernel launch when every parameter it updates lives in the training
    engine's flat arenas (parameters, gradients; the momentum buffers then live in a third arena and the per-parameter
    ``momentum_buffer`` entries of the state are views of it, so ``state_dict()`` / ``load_state_dict()`` are torch's).
    Anything else -- parameters outside the arenas, Nesterov, dampening, a closure -- takes torch's own step.

    ``clip`` = (type, value, norm type) clips the gradients in front of the update (GradientClipper's types).  In the
    one-launch step the update reads them through the clip factors and leaves ``.grad`` as backward wrote it; in torch's own
    step they are clipped in place first, as detectron2 does, by a clipper built in each step (its table's copy waits for the
    work queued before it)."""

    def __init__(self, params, model=None, clip: Optional[Tuple[str, float, float]] = None, **kw):
        super().__init__(params, **kw)
        self._model = model
        self._clip = None if clip is None else _check_clip(*clip)
        self._clipper = None  # (GradientClipper over the gradient arena, SgdClipTable) of the one-launch step
        self._fused = None  # (engine, mom arena, block table, n blocks, [(param, mom view)], the two groups)
        self._fused_off = None  # (engine, reason): the one-launch step is not possible with this engine; not retried

    def _engine(self):
        bb = getattr(self._model, "backbone", None)
        return getattr(bb, "_train_engine", None)

    def _prepare(self, eng):
        """The one-launch step's state, or a string saying why it cannot be used (empty hyper-parameter groups --
        e.g. the norm group of a model built with MODEL.DARKNET.NORM "" -- do not count)."""
        groups = [g for g in self.param_groups if g["params"]]
        if not 1 <= len(groups) <= 2:
            return f"{len(groups)} non-empty parameter groups (the kernel takes one or two)"
        if any(g["nesterov"] or g["dampening"] != 0 or g["maximize"] for g in groups):
            return "nesterov / dampening / maximize"
        if groups[0]["momentum"] != groups[-1]["momentum"] or groups[0]["momentum"] == 0:
            return "momentum is zero or differs between the groups"
        arena, garena = eng.param_arena, eng.grad_arena
        base, gbase, n = arena.data_ptr(), garena.data_ptr(), arena.numel()
        segments, views, covered = [], [], 0
        mom = torch.zeros_like(arena)
        for gi, g in enumerate(groups):
            for prm in g["params"]:
                off = (prm.data_ptr() - base) // 4
                if prm.dtype != torch.float32 or off < 0 or off + prm.numel() > n or prm.grad is None or \
                        prm.grad.data_ptr() != gbase + 4 * off:
                    return "a parameter (or its .grad) lives outside the training engine's arenas"
                # a parameter is one contiguous run of the arena, possibly permuted (conv weights are channels_last)
                mview = torch.as_strided(mom, prm.shape, prm.stride(), off)
                st = self.state[prm]
                if st.get("momentum_buffer") is not None:
                    mview.copy_(st["momentum_buffer"])
                st["momentum_buffer"] = mview
                segments.append((off, prm.numel(), gi))
                views.append((prm, mview))
                covered += prm.numel()
        if covered != n:
            return "the optimizer's parameters do not cover the arena"
        segments.sort()
        table, nb = ops.sgd_block_table(segments, arena.device)
        self._clipper = None
        if self._clip is not None:
            runs = [garena[o:o + c] for o, c, _ in segments] if self._clip[0] == "norm" else [garena]
            self._clipper = GradientClipper(runs, *self._clip), ops.sgd_clip_table(segments, arena.device)
        return eng, mom, table, nb, views, (groups[0], groups[-1])

    @torch.no_grad()
    def step(self, closure=None):
        import os
        eng = self._engine()
        usable = closure is None and eng is not None and eng.param_arena is not None and \
            os.environ.get("YOLO_FUSED_SGD", "1") != "0"
        if usable and self._fused_off is not None and self._fused_off[0] is eng:
            usable = False  # already found impossible with this engine: torch's step, without preparing again
        if usable and (self._fused is None or self._fused[0] is not eng or
                       any(self.state[p].get("momentum_buffer") is not m for p, m in self._fused[4])):
            res = self._prepare(eng)
            if isinstance(res, str):
                import logging
                logging.getLogger(__name__).warning("ArenaSGD: one-launch step disabled (%s); using torch's step", res)
                self._fused, self._fused_off = None, (eng, res)
            else:
                self._fused = res
        if not usable or self._fused is None:
            self._fused = None
            return self._torch_step(closure)
        eng, mom, table, nb, views, (g0, g1) = self._fused
        if any(p.grad is None for p, _ in views):
            self._fused = None
            return self._torch_step(closure)
        hyper = (g0["lr"], g0["weight_decay"], g1["lr"], g1["weight_decay"], g0["momentum"])
        if self._clipper is None:
            ops.sgd_step(eng.param_arena, eng.grad_arena, mom, table, nb, *hyper)
        else:
            clipper, clip_table = self._clipper
            clipper.measure()
            by_value = clipper.clip_type == "value"
            ops.sgd_step_clipped(eng.param_arena, eng.grad_arena, mom, clip_table, *hyper, coefs=clipper.coefs,
                                 per_tensor=clipper.per_tensor, clip_value=clipper.clip_value if by_value else None)
        # in-place update outside autograd's sight: move the version counters ourselves (the engines key their
        # packed / folded weights on them)
        ps = [p for p, _ in views]
        torch._C._autograd._unsafe_set_version_counter(ps, [p._version + 1 for p in ps])
        return None

    def _torch_step(self, closure):
        if self._clip is not None:
            if closure is not None:
                raise RuntimeError("ArenaSGD: a closure computes the gradients inside the step, where they cannot be clipped "
                                   "first; call backward() and step() without one")
            grads = _grads(p for g in self.param_groups for p in g["params"])
            if grads:
                GradientClipper(grads, *self._clip).clip_()
        return super().step(closure)


def build_optimizer(cfg, model: torch.nn.Module) -> torch.optim.Optimizer:
    norm_params, other = [], []
    for name, p in model.named_parameters():
        if not p.requires_grad:
            continue
        (norm_params if ".norm." in name else other).append(p)
    groups = [dict(params=other, weight_decay=cfg.SOLVER.WEIGHT_DECAY),
              dict(params=norm_params, weight_decay=cfg.SOLVER.WEIGHT_DECAY_NORM)]
    c = cfg.SOLVER.get("CLIP_GRADIENTS", None)
    clip = (c.CLIP_TYPE, c.CLIP_VALUE, c.NORM_TYPE) if c is not None and c.ENABLED else None
    return ArenaSGD(groups, model=model, clip=clip, lr=cfg.SOLVER.BASE_LR, momentum=cfg.SOLVER.MOMENTUM,
                    nesterov=cfg.SOLVER.NESTEROV)


class WarmupMultiStepLR(torch.optim.lr_scheduler.LRScheduler):
    """lr = base * gamma^(number of milestones passed), ramped linearly from warmup_factor over warmup_iters."""

    def __init__(self, optimizer, milestones: List[int], gamma: float = 0.1, warmup_factor: float = 0.001,
                 warmup_iters: int = 1000, warmup_method: str = "linear", last_epoch: int = -1):
        assert list(milestones) == sorted(milestones), milestones
        self.milestones, self.gamma = list(milestones), gamma
        self.warmup_factor, self.warmup_iters, self.warmup_method = warmup_factor, warmup_iters, warmup_method
        super().__init__(optimizer, last_epoch)

    def _warmup(self) -> float:
        it = self.last_epoch
        if it >= self.warmup_iters:
            return 1.0
        if self.warmup_method == "constant":
            return self.warmup_factor
        alpha = it / self.warmup_iters
        return self.warmup_factor * (1 - alpha) + alpha

    def get_lr(self) -> List[float]:
        w = self._warmup()
        return [b * w * self.gamma ** bisect_right(self.milestones, self.last_epoch) for b in self.base_lrs]


def build_lr_scheduler(cfg, optimizer):
    if cfg.SOLVER.LR_SCHEDULER_NAME != "WarmupMultiStepLR":
        raise ValueError(f"unsupported LR scheduler {cfg.SOLVER.LR_SCHEDULER_NAME}")
    steps = [int(s) for s in cfg.SOLVER.STEPS]
    return WarmupMultiStepLR(optimizer, steps, cfg.SOLVER.GAMMA, cfg.SOLVER.WARMUP_FACTOR, cfg.SOLVER.WARMUP_ITERS,
                             cfg.SOLVER.WARMUP_METHOD)
