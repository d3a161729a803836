"""AdamW over lists of tensors on csrc/adamw.hip: moments in 32 or in 8 bits, gradients clipped by their global norm in the same step.

``adamw_step`` is one step on tensors that the caller holds; ``AdamW`` is the torch.optim.Optimizer around it that
``train.RescaleTrainer`` uses for ``train_opt["optimizer"] == "AdamW"``."""
from __future__ import annotations

from typing import List, Optional, Sequence

import numpy as np
import torch

from . import _lib, runtime as rt
from .pointwise import _stream, on_device

#: values that share a scale of the 8-bit moments; every tensor's moments start at a multiple of it
BLOCK = 256
_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _need(cond, what):
    if not cond:
        raise RuntimeError("selfc_amd: " + (what if isinstance(what, str) else what()))


def state_size(numels: Sequence[int]) -> int:
    """Values of the moments' buffers for tensors of these sizes."""
    return sum(-(-n // BLOCK) * BLOCK for n in numels)


def _dense(t: torch.Tensor) -> bool:
    """Does the tensor fill one stretch of memory, in some order of its axes?"""
    want = 1
    for st, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if st != want:
            return False
        want *= n
    return True


def _order(t: torch.Tensor):
    """The order of the tensor's axes in memory: the strides of those that have one."""
    return tuple(st for st, n in zip(t.stride(), t.shape) if n != 1)


def _table(params, grads, steps):
    """(the C table of (parameter, gradient, step, size) per tensor, tensors it points to beyond the caller's own, the first tensor, blocks
    of the moments)."""
    tab = np.empty((len(grads), 4), dtype=np.uint64)
    got = _lib.host().table(params, grads, steps, tab.__array_interface__["data"][0])
    if got is not None:
        live, blocks = got
        first = params[0] if params else next((g for g in grads if g is not None), None) if live else None
        if first is not None:
            _lib.require_gpu(first)
            _need(first.dtype in _DTYPE, lambda: f"{first.dtype} tensors; expected float32, bfloat16 or float16")
        return tab, (), first, blocks
    keep = _look_closer(params, grads, steps)
    got = _lib.host().table([_as_flat(p) for p in params] if params is not None else None, [None if g is None else _as_flat(g) for g in grads], steps,
                        tab.__array_interface__["data"][0])
    _need(got is not None, "the tensors cannot be read")
    return tab, keep, params[0] if params else next(g for g in grads if g is not None), got[1]


def _as_flat(t):
    """the memory of a dense tensor, in its own order"""
    return t.detach().as_strided((t.numel(),), (1,))


def _look_closer(params, grads, steps):
    """Not everything is of one kind and contiguous: say what is refused; bring gradients into their tensors' order."""
    keep = []
    _need(params is None or len(params) == len(grads), lambda: f"{len(params)} tensors and {len(grads)} gradients")
    every = [(f"tensor {i}", t) for i, t in enumerate(params or [])] + [(f"gradient {i}", t) for i, t in enumerate(grads) if t is not None]
    _need(all(torch.is_tensor(t) for _, t in every), "expected tensors")
    first = every[0][1]
    _lib.require_gpu(first)
    _need(first.dtype in _DTYPE, lambda: f"{first.dtype} tensors; expected float32, bfloat16 or float16")
    for name, t in every:
        if t.dtype is not first.dtype or t.device != first.device or t.layout is not torch.strided:
            raise RuntimeError(f"selfc_amd: {name} is {t.dtype} on {t.device} ({t.layout}), expected {first.dtype} on {first.device}: one call takes one type on one GPU")
    for i, g in enumerate(grads):
        if g is None:
            continue
        if params is None:
            if not _dense(g):
                grads[i] = g.contiguous()
                keep.append(grads[i])
            continue
        p = params[i]
        _need(p.shape == g.shape, lambda: f"gradient {i} has shape {tuple(g.shape)}, its tensor {tuple(p.shape)}")
        _need(_dense(p), lambda: f"tensor {i} does not fill one stretch of memory (strides {p.stride()})")
        if g.stride() != p.stride():
            grads[i] = torch.empty_strided(p.shape, p.stride(), dtype=p.dtype, device=p.device).copy_(g)
            keep.append(grads[i])
    for i, p in enumerate(params or []):
        _need(_dense(p), lambda: f"tensor {i} does not fill one stretch of memory (strides {p.stride()})")
    _need(steps is None or (len(steps) == len(grads) and all(torch.is_tensor(s) and s.dtype is torch.float32 and s.device == first.device and s.numel() == 1 for s in steps)),
          "step: expected a float32 scalar on the tensors' GPU for each tensor")
    return keep


def grad_norm(grads: Sequence[Optional[torch.Tensor]]) -> torch.Tensor:
    """2-norm of all gradients (None entries are skipped) of one type on one GPU, as a device scalar; squares are summed in 64 bits."""
    grads = list(grads)
    tab, keep, first, _ = _table(None, grads, None)
    _need(first is not None, "grad_norm needs a gradient")
    with on_device(first):
        out = torch.empty((), dtype=torch.float32, device=first.device)
        part = torch.empty(_lib.lib().selfc_grad_norm_partials(len(grads)), dtype=torch.float64, device=first.device)
        rt.call("selfc_grad_norm", tab.__array_interface__["data"][0], len(grads), _DTYPE[first.dtype], part.data_ptr(), out.data_ptr(), _stream(first))
    return out


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[Optional[torch.Tensor]], exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor,
               exp_avg_scale: Optional[torch.Tensor] = None, exp_avg_sq_scale: Optional[torch.Tensor] = None, *, step, lr,
               beta1: float = 0.9, beta2: float = 0.999, eps: float = 1e-8, weight_decay: float = 0.01, seed: int = 0,
               max_norm: Optional[float] = None, norm: Optional[torch.Tensor] = None) -> None:
    """One AdamW step of `params` in place (decoupled weight decay; a tensor whose gradient is None is left as it is, with its moments).

    All tensors have one type (fp32, bf16 or f16; gradients the same), lie on one GPU and share no memory; arithmetic is in fp32.  The moments of all
    of them are held in two buffers of ``state_size`` values, tensor i behind the others at multiples of BLOCK values: fp32, or
    float8_e4m3fn (exp_avg) and float8_e5m2 (exp_avg_sq) with fp32 scales, one per BLOCK values.  In 8 bits the moments are rounded
    with a dither that is a function of (seed, step, the tensor's place in the list, the value's place in it): the same inputs give
    the same bits, on every rank of a data-parallel run.

    step: the number of this step (from 1 on), or a list of device scalars, one per tensor, that hold it (captured steps).
    lr: a float or a device scalar.  norm, max_norm: gradients count as scaled by min(1, max_norm / (norm + 1e-6)); norm is a device
    scalar (grad_norm); without it, it is computed here.  The gradients themselves are not changed.  A norm that is not finite acts as in
    the formula: infinite, the finite gradients count as 0; not a number, no parameter that has a gradient stays one."""
    _launch(_ready(params, grads, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, step, lr, beta1, beta2, eps, weight_decay, seed, max_norm, norm))


def _ready(params, grads, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, step, lr, beta1, beta2, eps, weight_decay, seed, max_norm, norm):
    """Everything that adamw_step refuses, and what _launch then takes: nothing is changed yet."""
    _need(0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0, lambda: f"betas are ({beta1}, {beta2})")
    grads = list(grads)
    steps = step if isinstance(step, (list, tuple)) else None
    tab, keep, first, blocks = _table(params, grads, steps)
    if first is None:
        return None
    bits8 = exp_avg.dtype is torch.float8_e4m3fn
    if bits8:
        _need(exp_avg_sq.dtype is torch.float8_e5m2, lambda: f"exp_avg is float8_e4m3fn, exp_avg_sq {exp_avg_sq.dtype}: expected float8_e5m2")
        _need(exp_avg_scale is not None and exp_avg_sq_scale is not None, "8-bit moments need their scales")
    else:
        _need(exp_avg.dtype is torch.float32 and exp_avg_sq.dtype is torch.float32, lambda: f"moments are {exp_avg.dtype} and {exp_avg_sq.dtype}: expected float32, or float8_e4m3fn and float8_e5m2")
    size, dev = blocks * BLOCK, first.device
    for name, t, n in (("exp_avg", exp_avg, size), ("exp_avg_sq", exp_avg_sq, size)) + ((("exp_avg_scale", exp_avg_scale, blocks), ("exp_avg_sq_scale", exp_avg_sq_scale, blocks)) if bits8 else ()):
        if t.device != dev or not t.is_contiguous() or t.numel() < n:
            raise RuntimeError(f"selfc_amd: {name}: expected {n} contiguous values on {dev}, got {tuple(t.shape)} on {t.device}")
    at, at_sq, n = exp_avg.data_ptr(), exp_avg_sq.data_ptr(), size if bits8 else 4 * size
    _need(at + n <= at_sq or at_sq + n <= at, "exp_avg and exp_avg_sq are the same memory, or share some")
    if bits8:
        used = sorted(((at, at + n), (at_sq, at_sq + n), *((t.data_ptr(), t.data_ptr() + 4 * blocks) for t in (exp_avg_scale, exp_avg_sq_scale))))
        _need(all(x[1] <= y[0] for x, y in zip(used, used[1:])), "the moments and their scales share memory")
    _need(not bits8 or (exp_avg_scale.dtype is torch.float32 and exp_avg_sq_scale.dtype is torch.float32), "the scales are float32")
    if steps is not None:
        host_step = 1.0
    else:
        host_step = float(step)
        _need(host_step >= 1 and host_step == int(host_step), lambda: f"step is {step}: steps are counted from 1")
        _need(not torch.cuda.is_current_stream_capturing(), "a captured step needs its number on the device (AdamW(..., capturable=True))")
    lr_dev = lr if torch.is_tensor(lr) and lr.is_cuda else None
    if lr_dev is not None:
        _need(lr.dtype is torch.float32 and lr.numel() == 1 and lr.device == first.device, "lr: expected a float32 scalar on the tensors' GPU")
    if max_norm is not None and norm is None and any(g is not None for g in grads):
        norm = grad_norm(grads)
    if max_norm is None:
        norm = None
    if norm is not None:
        _need(norm.dtype is torch.float32 and norm.numel() == 1 and norm.device == first.device, "norm: expected a float32 scalar on the tensors' GPU")
    args = (tab.__array_interface__["data"][0], len(grads), _DTYPE[first.dtype], 8 if bits8 else 32, at, at_sq,
            rt._ptr(exp_avg_scale) if bits8 else None, rt._ptr(exp_avg_sq_scale) if bits8 else None, 0.0 if lr_dev is not None else float(lr), rt._ptr(lr_dev),
            float(beta1), float(beta2), float(eps), float(weight_decay), host_step, int(seed) & 0xFFFFFFFF, rt._ptr(norm), float(max_norm or 0.0))
    return first, args, (tab, keep, norm), params, grads


def _launch(ready) -> None:
    """The launches of a step that _ready has checked."""
    if ready is None:
        return
    first, args, _, params, grads = ready          # (the third: what the arguments' addresses point to beyond the caller's own)
    with on_device(first):
        rt.call("selfc_adamw_step", *args, _stream(first))
    # the kernel wrote through raw pointers: autograd's saved-tensor checks and the packed-weight caches go by version
    _lib.host().written(params, grads)


class _Bucket:
    """The moments of one parameter group's tensors of one type on one GPU: two buffers (and two of scales), and every tensor's step."""

    def __init__(self, params: List[torch.Tensor], bits: int, capturable: bool, opt: torch.optim.Optimizer):
        self.params = params
        self.strides = None if all(map(torch.Tensor.is_contiguous, params)) else [p.stride() for p in params]
        dev, size = params[0].device, state_size([p.numel() for p in params])
        kinds = (torch.float8_e4m3fn, torch.float8_e5m2) if bits == 8 else (torch.float32, torch.float32)
        self.m, self.v = (torch.zeros(size, dtype=torch.uint8 if bits == 8 else torch.float32, device=dev).view(k) for k in kinds)
        self.scales = [torch.ones(size // BLOCK, dtype=torch.float32, device=dev) for _ in range(2)] if bits == 8 else [None, None]
        self.steps = torch.zeros(len(params), dtype=torch.float32, device=dev if capturable else "cpu")
        self.step_list = list(self.steps.unbind())
        at = 0
        for p, step in zip(params, self.step_list):
            n, blocks = p.numel(), -(-p.numel() // BLOCK)
            st = opt.state[p] = {"step": step}
            for name, buf in (("exp_avg", self.m), ("exp_avg_sq", self.v)):
                st[name] = buf[at:at + n].as_strided(p.shape, p.stride(), at) if _dense(p) else buf[at:at + n].view(p.shape)
            if bits == 8:
                for name, buf in zip(("exp_avg_scale", "exp_avg_sq_scale"), self.scales):
                    st[name] = buf[at // BLOCK:at // BLOCK + blocks]
            at += blocks * BLOCK


    def check_layout(self):
        """Moments lie in the order of their tensors' memory: that must not change under them."""
        if self.strides is None:
            same = all(map(torch.Tensor.is_contiguous, self.params))
        else:
            same = all(p.stride() == s for p, s in zip(self.params, self.strides))
        _need(same, "a parameter's memory format changed after its moments were allocated - convert the model before the first step")


class AdamW(torch.optim.Optimizer):
    """AdamW with the moments in 32 or 8 bits, all tensors of a group in one step (``adamw_step``), as a torch optimizer: parameter groups,
    ``lr`` that a scheduler may change, ``state_dict`` with one entry per parameter.

    state_bits: 32 (8 bytes of moments a value), or 8 (2 bytes, and 8 per BLOCK values for their scales).  max_norm: the gradients of all
    groups count as clipped to this global norm; ``grad_norm`` then holds the norm before clipping (a device scalar).  The ``.grad``
    tensors themselves are left as they are.  capturable: step numbers (and ``lr``, if it is a tensor) live on the GPU, so that a
    captured step keeps counting.  seed: of the dither of 8-bit moments (one of the groups' values, so ``state_dict`` holds it and a resumed run repeats
    the bits).  A parameter without a gradient is skipped, with its moments and its step.  Ranks that hold equal
    parameters and gradients stay equal bit for bit."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01, *, state_bits: int = 32,
                 max_norm: Optional[float] = None, capturable: bool = False, seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits is {state_bits}, expected 8 or 32")
        if not torch.is_tensor(lr) and not lr >= 0:
            raise ValueError(f"lr is {lr}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0) or not eps >= 0 or not weight_decay >= 0:
            raise ValueError(f"betas {betas}, eps {eps}, weight_decay {weight_decay}")
        if max_norm is not None and not max_norm > 0:
            raise ValueError(f"max_norm is {max_norm}")
        self.state_bits, self.max_norm, self.capturable = state_bits, max_norm, bool(capturable)
        self.grad_norm: Optional[torch.Tensor] = None
        self._buckets: dict = {}
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, seed=int(seed)))

    def __getstate__(self):
        raise TypeError("selfc_amd.AdamW is saved through state_dict(): its moments are views of shared buffers")

    def _group_buckets(self, gi: int) -> List[_Bucket]:
        group = self.param_groups[gi]
        have = self._buckets.get(gi)
        if have is None or sum(len(b.params) for b in have) != len(group["params"]) or any(p not in self.state for p in group["params"]):
            if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("selfc_amd: run a step, or ensure_state(), before the capture: a replay would clear the moments again")
            kinds: dict = {}
            for p in group["params"]:
                kinds.setdefault((p.dtype, p.device), []).append(p)
            have = self._buckets[gi] = [_Bucket(ps, self.state_bits, self.capturable, self) for ps in kinds.values()]
        return have

    def ensure_state(self):
        """Allocate the moments now (zeros) instead of at the first step: to load into, or before a capture."""
        for gi in range(len(self.param_groups)):
            self._group_buckets(gi)

    @torch.no_grad()
    def reset_state(self):
        """Moments and step numbers back to zero, in place: a captured step goes on from there."""
        for buckets in self._buckets.values():
            for b in buckets:
                for t in (b.m, b.v):
                    (t.view(torch.uint8) if t.element_size() == 1 else t).zero_()
                for t in b.scales:
                    if t is not None:
                        t.fill_(1.0)
                b.steps.zero_()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if not self.capturable and torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("selfc_amd: construct AdamW(..., capturable=True) to capture its step")
        work = [(gi, bi, b, [p.grad for p in b.params]) for gi in range(len(self.param_groups)) for bi, b in enumerate(self._group_buckets(gi))]
        work = [w for w in work if any(g is not None for g in w[3])]
        for _, _, b, _ in work:
            b.check_layout()
        norm = self.grad_norm
        if self.max_norm is not None and work:
            norms = [grad_norm(w[3]) for w in work]
            home = norms[0].device
            norm = norms[0] if len(norms) == 1 else torch.stack([n.to(home) for n in norms]).double().square().sum().sqrt().float()
        # every group's arguments are checked before anything is counted or launched: a refused step leaves all as it was
        ready = []
        for gi, bi, b, grads in work:
            group = self.param_groups[gi]
            kw = dict(lr=group["lr"], beta1=group["betas"][0], beta2=group["betas"][1], eps=group["eps"], weight_decay=group["weight_decay"],
                      seed=group["seed"] + 0x10001 * gi + bi, max_norm=self.max_norm, norm=None if self.max_norm is None else norm.to(b.params[0].device))
            args = (b.m, b.v, *b.scales)
            if self.capturable:
                ready.append(_ready(b.params, grads, *args, step=b.step_list, **kw))
                continue
            steps = b.steps.numpy() + 1
            active = [i for i, g in enumerate(grads) if g is not None]
            for t in sorted(set(steps[active].tolist())):          # usually one: parameters that were skipped before are behind
                ready.append(_ready(b.params, [g if g is not None and steps[i] == t else None for i, g in enumerate(grads)], *args, step=t, **kw))
        self.grad_norm = norm
        for _, _, b, grads in work:
            active = [i for i, g in enumerate(grads) if g is not None]
            if not self.capturable:
                b.steps.numpy()[active] += 1
            elif len(active) == len(grads):
                with on_device(b.params[0]):
                    b.steps.add_(1)
            else:
                with on_device(b.params[0]):
                    torch._foreach_add_([b.step_list[i] for i in active], 1)
        for r in ready:
            _launch(r)
        return loss

    def load_state_dict(self, state_dict):
        """Adopts the groups' hyper-parameters and copies the moments into the existing buffers (a captured step keeps its tensors).
        The saved state has to be of the same state_bits; a plain Adam / AdamW state file loads with state_bits=32.  In 8 bits it also has to be
        in the parameters' memory format: the values that share a scale are neighbours in memory, so another order has other blocks."""
        saved, groups = state_dict["state"], state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("selfc_amd: the saved state has other parameter groups than this optimizer")
        self.ensure_state()
        want = {"step", "exp_avg", "exp_avg_sq"} | ({"exp_avg_scale", "exp_avg_sq_scale"} if self.state_bits == 8 else set())
        pairs = [(saved.get(i), p) for g, own in zip(groups, self.param_groups) for i, p in zip(g["params"], own["params"])]
        for st, p in pairs:                                        # refuse before anything is changed
            if st is not None and st and set(st) != want:
                raise ValueError(f"selfc_amd: saved state has {sorted(st)}, expected {sorted(want)} (state_bits={self.state_bits})")
            for k in want - {"step"}:
                if st and (st[k].shape != self.state[p][k].shape or st[k].dtype != self.state[p][k].dtype):
                    raise ValueError(f"selfc_amd: saved {k} is {st[k].dtype} {tuple(st[k].shape)}, expected {self.state[p][k].dtype} {tuple(self.state[p][k].shape)}")
                if st and self.state_bits == 8 and _order(st[k]) != _order(self.state[p][k]):
                    raise ValueError(f"selfc_amd: saved {k} has strides {st[k].stride()}, its parameter {self.state[p][k].stride()}: 8-bit moments load into the memory "
                                     "format they were saved in only - convert the model before the optimizer's first step")
        with torch.no_grad():
            for st, p in pairs:
                for k, own in self.state[p].items():
                    if not st:
                        own.fill_(1.0) if k.endswith("scale") else own.view(torch.uint8).zero_() if own.element_size() == 1 else own.zero_()
                    elif k == "step":
                        own.fill_(float(st[k]))
                    else:
                        own.copy_(st[k])
        for g, own in zip(groups, self.param_groups):
            for k, v in g.items():
                if k == "lr" and torch.is_tensor(own.get("lr")):
                    own["lr"].fill_(float(v))
                elif k in own and k != "params" or k == "initial_lr":
                    own[k] = tuple(v) if isinstance(v, list) else v.clone() if torch.is_tensor(v) else v          # (the saved tensors stay the other's)
