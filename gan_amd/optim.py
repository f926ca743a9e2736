"""Optimizers for the train step (reference: `getattr(torch.optim, cfg.optimizer)(model.parameters(), cfg.lr,
**cfg.optimizer_kwargs)`, train_celeba.py:75-77).

`make_optimizer` keeps that contract -- any torch.optim class by name -- and serves the README recipes' choice, Adam
(README.md:55,60; AdamW too), with `FlatAdam`: the same update rule as torch.optim.Adam run by ONE kernel over the
module's flat parameter / gradient arenas (gan_amd/utils.py: FlatArena) with the step count on the device, so the
whole optimizer step is two launches and can be captured in a HIP graph.  torch's own Adam needs capturable=True
for that, which costs a launch per parameter tensor for each bias-correction scalar (~600 launches per iteration
for the two StyleGAN2 networks).

`muon_step` / `FlatMuon` take matrices by their orthogonalised momentum instead (functional.orthogonalize), all of a
network's in shared launches; optimizer="Muon" in the train step."""
from __future__ import annotations

import ctypes
import math
from typing import Dict, List, Optional, Sequence, Tuple

import torch
from torch import Tensor, nn

from . import _lib
from . import functional as GF
from ._lib import check, ptr, require_gpu, stream_of
from .utils import FlatArena, arena_of

_FLAT_KEYS = {"betas", "eps", "weight_decay"}
_MUON_KEYS = {"weight_decay", "momentum", "nesterov", "ns_coefficients", "eps", "ns_steps", "adjust_lr_fn", "adam_lr", "betas", "adam_eps"}


class FlatAdam(torch.optim.Optimizer):
    """torch.optim.Adam / AdamW (amsgrad = False, maximize = False) over a FlatArena.

    * one `param_group` holding the arena's parameters; `lr`, `betas`, `eps`, `weight_decay` are read from it at every
      step (schedulers that edit param_groups work; under HIP-graph capture the values at capture time are baked in);
    * `state[p]` exposes `step` / `exp_avg` / `exp_avg_sq` like torch's Adam -- the moments are views into two flat
      buffers, `step` is ONE device scalar shared by the arena (torch keeps one per tensor: the same number unless a
      parameter skips updates);
    * parameters whose `.grad` is None are skipped, as torch does."""

    def __init__(self, arena: FlatArena, lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.0, decoupled: bool = False):
        if arena.grad is None:
            raise ValueError("FlatAdam needs an arena with a gradient buffer (arena_of(module, with_grad=True))")
        defaults = dict(lr=float(lr), betas=(float(betas[0]), float(betas[1])), eps=float(eps), weight_decay=float(weight_decay))
        super().__init__(arena.params, defaults)
        self.arena = arena
        self.decoupled = decoupled
        dev = arena.data.device
        self.exp_avg = torch.zeros_like(arena.data)
        self.exp_avg_sq = torch.zeros_like(arena.data)
        self.step_t = torch.zeros(4, dtype=torch.float32, device=dev)  # [0] = updates done so far
        self._point_state()

    def _point_state(self) -> None:
        step = self.step_t[0]
        for p, o in zip(self.arena.params, self.arena.offsets):
            n = p.numel()
            self.state[p] = {"step": step, "exp_avg": self.exp_avg[o:o + n].view(p.shape), "exp_avg_sq": self.exp_avg_sq[o:o + n].view(p.shape)}

    def _runs(self) -> List[Tuple[int, int]]:
        """(offset, numel) ranges of the arena to update: everything when every parameter has a gradient in its arena
        slice (the train step's case); otherwise the gradients are gathered into the arena first and the parameters
        without one are left out."""
        arena = self.arena
        base = arena.grad.data_ptr()
        missing, stray = False, False
        for p, o in zip(arena.params, arena.offsets):
            if p.grad is None:
                missing = True
            elif p.grad.data_ptr() != base + 4 * o:
                stray = True
        if not missing and not stray:
            return [(0, arena.numel)]
        present = [p.grad is not None for p in arena.params]
        if stray:
            arena.gather_grads()  # re-attaches every slice; `present` remembers who really had a gradient
        runs: List[Tuple[int, int]] = []
        align = arena.ALIGN
        for p, o, ok in zip(arena.params, arena.offsets, present):
            if not ok:
                continue
            n = (p.numel() + align - 1) // align * align
            if runs and runs[-1][0] + runs[-1][1] == o:
                runs[-1] = (runs[-1][0], runs[-1][1] + n)
            else:
                runs.append((o, n))
        return runs

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        arena = self.arena
        if not arena.intact():
            raise RuntimeError("FlatAdam: parameters were moved after flattening (model.to(...) / .half()); rebuild the optimizer")
        group = self.param_groups[0]
        lr, (b1, b2), eps, wd = group["lr"], group["betas"], group["eps"], group["weight_decay"]
        lib = _lib.load()
        st = stream_of(arena.data)
        advance = 1
        for off, n in self._runs():
            check(lib.gan_adam_step(arena.data.data_ptr() + 4 * off, arena.grad.data_ptr() + 4 * off, self.exp_avg.data_ptr() + 4 * off,
                                    self.exp_avg_sq.data_ptr() + 4 * off, n, ptr(self.step_t), advance, float(lr), float(b1), float(b2),
                                    float(eps), float(wd), int(self.decoupled), st), "gan_adam_step")
            advance = 0
        # the kernel wrote through raw pointers: no parameter's version moved, so cached GEMM images of the old values
        # would still match their keys
        GF.invalidate_packed(arena.params)
        return loss

    def zero_grad(self, set_to_none: bool = False) -> None:
        """The gradients live in the arena: zero it in one launch and keep the slices attached."""
        self.arena.grad.zero_()
        self.arena.attach_grads()

    def load_state_dict(self, state_dict) -> None:
        """Accepts a torch.optim.Adam state_dict of the same parameters: the per-tensor moments are copied into the flat
        buffers (which stay the storage), the step count is taken from the first entry."""
        super().load_state_dict(state_dict)
        with torch.no_grad():
            first = True
            for p, o in zip(self.arena.params, self.arena.offsets):
                s = self.state.get(p)
                if not s:
                    continue
                n = p.numel()
                self.exp_avg[o:o + n].copy_(s["exp_avg"].reshape(-1))
                self.exp_avg_sq[o:o + n].copy_(s["exp_avg_sq"].reshape(-1))
                if first:
                    self.step_t[0] = float(s["step"])
                    first = False
        self._point_state()


_SCALINGS = {None: 1, "original": 1, "match_rms_adamw": 2, "none": 0}


def _as_matrix(shape) -> Tuple[int, int]:
    rows = int(shape[0])
    return rows, math.prod(shape[1:])


@torch.no_grad()
def muon_step(params: Sequence[Tensor], grads: Sequence[Tensor], momentum_buffers: Sequence[Tensor], *, lr: float, momentum: float = 0.95,
              nesterov: bool = True, weight_decay: float = 0.0, adjust_lr_fn: Optional[str] = None, steps: int = 5,
              coefficients=GF.NS_COEFFICIENTS, eps: float = 1e-7) -> None:
    """One update of every parameter by its orthogonalised momentum, in place:
        buf <- momentum * buf + (1 - momentum) * grad
        u    = momentum * buf + (1 - momentum) * grad if nesterov else buf
        p   <- (1 - lr * weight_decay) * p - lr * s * orthogonalize(u)
    A parameter of two or more dimensions counts as the matrix (shape[0], everything else), a convolution as (out, in kh kw).
    s = sqrt(max(1, rows / cols)) for adjust_lr_fn None or "original", 0.2 sqrt(max(rows, cols)) for "match_rms_adamw", 1 for
    "none".  float32, contiguous, on one device; nothing may overlap.  All parameters share the launches; a gradient that is
    not finite makes its own parameter NaN and no other."""
    if not len(params) == len(grads) == len(momentum_buffers):
        raise _lib.GanAmdError(f"muon_step: {len(params)} parameters, {len(grads)} gradients, {len(momentum_buffers)} momentum buffers")
    if adjust_lr_fn not in _SCALINGS:
        raise _lib.GanAmdError(f"muon_step: adjust_lr_fn must be None, 'original', 'match_rms_adamw' or 'none', got {adjust_lr_fn!r}")
    if GF.has_tangent(*params, *grads, *momentum_buffers):
        raise _lib.GanAmdError("muon_step has no derivative: a tensor carries a tangent of forward-mode AD, pass its primal")
    held, mats, spans = [], [], []
    for p, g, m in zip(params, grads, momentum_buffers):
        if p.dim() < 2:
            raise _lib.GanAmdError(f"muon_step: parameters of two or more dimensions, got shape {tuple(p.shape)}")
        if p.shape != g.shape or p.shape != m.shape:
            raise _lib.GanAmdError(f"muon_step: parameter {tuple(p.shape)}, gradient {tuple(g.shape)}, momentum {tuple(m.shape)}")
        if not p.dtype == g.dtype == m.dtype == torch.float32:
            raise _lib.GanAmdError(f"muon_step takes float32, got {p.dtype}, {g.dtype}, {m.dtype}")
        if not p.device == g.device == m.device == params[0].device:
            raise _lib.GanAmdError("muon_step: parameters, gradients and momentum buffers must be on one device")
        if not (p.is_contiguous() and m.is_contiguous()):
            raise _lib.GanAmdError("muon_step: parameters and momentum buffers must be contiguous")
        if p.numel() == 0:
            continue
        g = g.contiguous()
        held.append(g)
        spans += [(t.data_ptr(), t.data_ptr() + t.numel() * 4, written) for t, written in ((p, True), (m, True), (g, False))]
        mats.append((g.data_ptr(), m.data_ptr(), p.data_ptr(), *_as_matrix(p.shape), 1))
    reads, writes = 0, 0  # where what lies below ends
    for start, end, written in sorted(spans):
        if start < writes or (written and start < reads):
            raise _lib.GanAmdError("muon_step: a parameter or momentum buffer is given twice, or overlaps another or a gradient")
        if written:
            writes = max(writes, end)
        else:
            reads = max(reads, end)
    require_gpu(*params[:1])
    if not mats:
        return
    _muon_launch((_lib.Matrix * len(mats))(*mats), params[0], lr, momentum, nesterov, weight_decay, adjust_lr_fn, steps, coefficients, eps)
    # written through raw pointers: cached GEMM images of the old values would still match their keys, and a backward that has saved
    # one of these tensors has to see that it changed
    GF.invalidate_packed(params)
    torch.autograd.graph.increment_version([*params, *momentum_buffers])


def _muon_launch(mats, like: Tensor, lr, momentum, nesterov, weight_decay, adjust_lr_fn, steps, coefficients, eps) -> None:
    a, b, c = (float(v) for v in coefficients)
    ws, nbytes = GF.matrix_workspace(mats, like.device)
    with _lib.on_device(like):
        check(GF._run("muon_step", sum(GF.ortho_flops(t.rows, t.cols, steps) for t in mats) if GF._PROFILE is not None else 0,
                      20 * sum(t.rows * t.cols for t in mats) if GF._PROFILE is not None else 0,
                      lambda: _lib.load().gan_muon_step(ctypes.addressof(mats), len(mats), float(lr), float(momentum), int(bool(nesterov)),
                                                        float(weight_decay), _SCALINGS[adjust_lr_fn], int(steps), a, b, c, float(eps), ptr(ws),
                                                        nbytes, stream_of(like))), "gan_muon_step")


class FlatMuon(torch.optim.Optimizer):
    """muon_step over a FlatArena for the matrices of a network, Adam for the rest of it (biases, norm scales, and whatever is a
    vector in a matrix's shape: one row or one column), in place on the arenas.  Where every parameter is two-dimensional, which
    is what torch.optim.Muon takes, all of them are matrices, as there, those of one row or column too.

    * two `param_groups`: the matrices (`lr`, `weight_decay`, `momentum`, `nesterov`, `ns_coefficients`, `eps`, `ns_steps`,
      `adjust_lr_fn`: torch.optim.Muon's names and update rule, its products in 22 bits instead of bfloat16's 8) and the rest
      (`lr` = `adam_lr`, by default the matrices' lr; `betas`, `eps` = `adam_eps`, `weight_decay` 0), read at every step
      (under HIP-graph capture the values at capture time are baked in);
    * `state[p]` is `momentum_buffer` for a matrix, `step` / `exp_avg` / `exp_avg_sq` for the rest (FlatAdam's: one shared step);
    * parameters whose `.grad` is None, and frozen ones, are skipped.

    torch.optim.Muon itself takes two-dimensional parameters only; here a convolution counts as the matrix (out, in kh kw)."""

    def __init__(self, arena: FlatArena, lr: float = 1e-3, weight_decay: float = 0.1, momentum: float = 0.95, nesterov: bool = True,
                 ns_coefficients=GF.NS_COEFFICIENTS, eps: float = 1e-7, ns_steps: int = 5, adjust_lr_fn: Optional[str] = None, *,
                 adam_lr: Optional[float] = None, betas: Tuple[float, float] = (0.9, 0.999), adam_eps: float = 1e-8):
        if arena.grad is None:
            raise ValueError("FlatMuon needs an arena with a gradient buffer (arena_of(module, with_grad=True))")
        if adjust_lr_fn not in _SCALINGS:
            raise ValueError(f"FlatMuon: adjust_lr_fn must be None, 'original', 'match_rms_adamw' or 'none', got {adjust_lr_fn!r}")
        self.arena = arena
        least = 1 if all(p.dim() == 2 for p in arena.params) else 2  # (what torch.optim.Muon takes goes all the same way, as there)
        self._matrix = [p.dim() >= 2 and min(_as_matrix(p.shape)) >= least for p in arena.params]
        matrices = [p for p, m in zip(arena.params, self._matrix) if m]
        rest = [p for p, m in zip(arena.params, self._matrix) if not m]
        groups = []
        if matrices:
            groups.append(dict(params=matrices, lr=float(lr), weight_decay=float(weight_decay), momentum=float(momentum), nesterov=bool(nesterov),
                               ns_coefficients=tuple(float(c) for c in ns_coefficients), eps=float(eps), ns_steps=int(ns_steps),
                               adjust_lr_fn=adjust_lr_fn))
        if rest:
            groups.append(dict(params=rest, lr=float(lr if adam_lr is None else adam_lr), betas=(float(betas[0]), float(betas[1])),
                               eps=float(adam_eps), weight_decay=0.0))
        super().__init__(groups, {})
        dev = arena.data.device
        self.exp_avg = torch.zeros_like(arena.data)  # the matrices' momentum too
        self.exp_avg_sq = torch.zeros_like(arena.data)
        self.step_t = torch.zeros(4, dtype=torch.float32, device=dev)  # [0] = updates done so far
        self._mats: Dict[Tuple[bool, ...], object] = {}
        self._point_state()

    def _point_state(self) -> None:
        step = self.step_t[0]
        for p, o, m in zip(self.arena.params, self.arena.offsets, self._matrix):
            n = p.numel()
            avg = self.exp_avg[o:o + n].view(p.shape)
            self.state[p] = {"momentum_buffer": avg} if m else {"step": step, "exp_avg": avg, "exp_avg_sq": self.exp_avg_sq[o:o + n].view(p.shape)}

    def _matrices(self, present: Tuple[bool, ...]):
        """The library's list of the matrices that take part (addresses in the arenas: they stay where they are)."""
        if present not in self._mats:
            a = self.arena
            rows = [(a.grad.data_ptr() + 4 * o, self.exp_avg.data_ptr() + 4 * o, a.data.data_ptr() + 4 * o, *_as_matrix(p.shape), 1)
                    for p, o, m, ok in zip(a.params, a.offsets, self._matrix, present) if m and ok]
            vecs = [v for p, o, m, ok in zip(a.params, a.offsets, self._matrix, present) if ok and not m for v in (o, p.numel())]
            self._mats[present] = ((_lib.Matrix * len(rows))(*rows), (ctypes.c_int64 * len(vecs))(*vecs))
        return self._mats[present]

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        arena = self.arena
        if not arena.intact():
            raise RuntimeError("FlatMuon: parameters were moved after flattening (model.to(...) / .half()); rebuild the optimizer")
        require_gpu(arena.data)
        base = arena.grad.data_ptr()
        present = tuple(p.grad is not None and p.requires_grad for p in arena.params)
        if any(p.grad is not None and p.grad.data_ptr() != base + 4 * o for p, o in zip(arena.params, arena.offsets)):
            absent = [p for p in arena.params if p.grad is None]
            arena.gather_grads()  # re-attaches every slice; `present` remembers who really had a gradient
            for p in absent:  # (a slice of zeros would count as a gradient from the next step on)
                p.grad = None
        mats, ranges = self._matrices(present)
        groups = {("momentum" in g): g for g in self.param_groups}
        if len(mats):
            g = groups[True]
            _muon_launch(mats, arena.data, g["lr"], g["momentum"], g["nesterov"], g["weight_decay"], g["adjust_lr_fn"], g["ns_steps"],
                         g["ns_coefficients"], g["eps"])
        if len(ranges):
            g = groups[False]
            with _lib.on_device(arena.data):
                check(_lib.load().gan_adam_step_ranges(ptr(arena.data), ptr(arena.grad), ptr(self.exp_avg), ptr(self.exp_avg_sq),
                                                       ctypes.addressof(ranges), len(ranges) // 2, ptr(self.step_t), 1, float(g["lr"]),
                                                       float(g["betas"][0]), float(g["betas"][1]), float(g["eps"]), float(g["weight_decay"]), 0,
                                                       stream_of(arena.data)), "gan_adam_step_ranges")
        # the kernels wrote through raw pointers (see FlatAdam.step)
        GF.invalidate_packed(arena.params)
        return loss

    zero_grad = FlatAdam.zero_grad

    def load_state_dict(self, state_dict) -> None:
        """The per-tensor entries are copied into the flat buffers, which stay the storage."""
        super().load_state_dict(state_dict)
        with torch.no_grad():
            for p, o, m in zip(self.arena.params, self.arena.offsets, self._matrix):
                s, n = self.state.get(p), p.numel()
                if not s:
                    continue
                if m:
                    self.exp_avg[o:o + n].copy_(s["momentum_buffer"].reshape(-1))
                else:
                    self.exp_avg[o:o + n].copy_(s["exp_avg"].reshape(-1))
                    self.exp_avg_sq[o:o + n].copy_(s["exp_avg_sq"].reshape(-1))
                    self.step_t[0] = float(s["step"])
        self._point_state()


def make_optimizer(name: str, module: nn.Module, lr: float, kwargs: Dict, *, capturable: bool = False) -> torch.optim.Optimizer:
    """The optimizer `name` (a torch.optim class name, train_celeba.py:75) for `module`'s parameters.  Adam / AdamW with
    only betas / eps / weight_decay set run as FlatAdam on a ROCm device, Muon as FlatMuon (matrices, convolutions among them, by their
    orthogonalised momentum; biases, norm scales and, beside such, matrices of one row or column by Adam at `adam_lr`, which is the
    matrices' `lr` unless given, ten times and more of what Adam usually gets); everything else is torch's own class
    (with capturable=True where it exists and the step is going to be captured in a HIP graph)."""
    params = list(module.parameters())
    on_gpu = bool(params) and all(p.is_cuda and p.dtype == torch.float32 for p in params)
    if name in ("Adam", "AdamW") and on_gpu and set(kwargs) <= _FLAT_KEYS:
        arena = arena_of(module, with_grad=True)
        kw = dict(kwargs)
        if name == "AdamW":
            kw.setdefault("weight_decay", 1e-2)  # torch.optim.AdamW's default
        return FlatAdam(arena, lr, decoupled=name == "AdamW", **kw)
    if name == "Muon" and on_gpu and set(kwargs) <= _MUON_KEYS:
        return FlatMuon(arena_of(module, with_grad=True), lr, **kwargs)
    cls = getattr(torch.optim, name)
    kw = dict(kwargs)
    if capturable and name in ("Adam", "AdamW", "NAdam", "RAdam", "Adamax", "Adadelta", "Adagrad", "ASGD", "RMSprop", "Rprop"):
        kw.setdefault("capturable", True)
    return cls(params, lr, **kw)
