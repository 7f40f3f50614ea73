"""AdamW over many tensors in one launch, on MI355X, with the moments in 32 bits or in 8.

``AdamW`` takes the place of the ``torch.optim.AdamW`` that the reference's loops construct (models/clavaddpm/trainer.py:44,
models/clavaddpm/train.py:384) for parameters that live as tensors: the guidance classifier, TabSyn's denoiser, ``LowRankEnsemble``.
(``ClavaDDPMTrainer`` keeps its own fused step over the training image.)  ``adamw_step`` is the step itself on lists of tensors.  The
update runs in libmtk_hip.so (mtk_adamw_step); there is no CPU path.

8-bit moments: e4m3 codes of the mean and of the root mean square with one fp32 power-of-two scale per 256 values, a quarter of the
memory of 32-bit ones; rounded up or down by a dither that depends on a value's place and the step, so slow averages keep moving.
"""
from __future__ import annotations

from array import array
from bisect import bisect_left
from operator import attrgetter
from typing import Sequence

import torch
from torch import Tensor

from . import _lib
from ._lib import launch, native
from .routing import DTYPES

SCALE_BLOCK = 256  # values per scale of the 8-bit moments


_dtype, _numel, _device, _dense, _address = attrgetter("dtype"), Tensor.numel, Tensor.get_device, Tensor.is_contiguous, Tensor.data_ptr


def _addresses(ts: Sequence[Tensor]):
    a = array("Q", map(_address, ts))
    return a, a.buffer_info()[0]


def _check_list(what: str, ts: Sequence[Tensor], dtype: torch.dtype, device: int, sizes: list[int]) -> None:
    # whole-list passes in C: a step over hundreds of tensors is otherwise bound by these checks
    if len(ts) != len(sizes):
        raise ValueError(f"adamw_step: {len(ts)} {what} for {len(sizes)} params")
    if list(map(_numel, ts)) == sizes and set(map(_dtype, ts)) == {dtype} and set(map(_device, ts)) == {device} and all(map(_dense, ts)):
        return
    for t, n in zip(ts, sizes):
        if t.dtype != dtype or t.get_device() != device or t.numel() != n or not t.is_contiguous():
            raise ValueError(f"adamw_step: {what}: expected contiguous {dtype} tensors of the params' sizes on cuda:{device}, got {tuple(t.shape)} {t.dtype} on "
                             f"{t.device}" + ("" if t.is_contiguous() else ", not contiguous"))


def _check_apart(params: Sequence[Tensor], grads: Sequence[Tensor], written: Sequence[Tensor]) -> None:
    span = lambda t: (t.data_ptr(), t.data_ptr() + t.nbytes)  # noqa: E731
    spans = sorted(span(t) for t in written if t.numel())
    if any(b[0] < a[1] for a, b in zip(spans, spans[1:])):
        raise ValueError("adamw_step: the same tensor twice, or tensors that share memory, among params and moments")
    starts = [a for a, _ in spans]
    for p, g in zip(params, grads):
        at, end = span(g)
        i = bisect_left(starts, end)
        if g.numel() and span(p) != (at, end) and i and spans[i - 1][1] > at:
            raise ValueError("adamw_step: a gradient shares memory with what the step writes")


def adamw_step(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avgs: Sequence[Tensor], exp_avg_sqs: Sequence[Tensor], step: int, *, lr: float,
               betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, exp_avg_scales: Sequence[Tensor] | None = None,
               exp_avg_sq_scales: Sequence[Tensor] | None = None, _hyper: Tensor | None = None) -> None:
    """One step, in place, over tensors of one type (float32, bfloat16, float16) on one device; ``step`` counts from 1.

    32-bit moments: ``exp_avgs`` / ``exp_avg_sqs`` are float32.  8-bit moments: they are float8_e4m3fn codes of the mean and of the ROOT mean
    square, and ``exp_avg_scales`` / ``exp_avg_sq_scales`` hold float32 [ceil(numel / 256)] scales.  A moment that is not finite becomes NaN.
    What is written (params, moments, scales) may not share memory, nor may a gradient with any of it (its own whole parameter excepted)."""
    if len(params) == 0:
        return
    q8 = exp_avg_scales is not None
    if q8 != (exp_avg_sq_scales is not None):
        raise ValueError("adamw_step: 8-bit moments need both exp_avg_scales and exp_avg_sq_scales")
    p0 = params[0]
    if not p0.is_cuda:
        raise RuntimeError("adamw_step: midst_toolkit_amd has no CPU path; move the params to the MI355X")
    if native().adamw(params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, step, lr, betas[0], betas[1], eps, weight_decay, _hyper):
        return
    if p0.dtype not in DTYPES:
        raise ValueError(f"adamw_step: params are {p0.dtype} (float32, bfloat16 or float16)")
    sizes, at = list(map(_numel, params)), p0.get_device()
    state = torch.float8_e4m3fn if q8 else torch.float32
    _check_list("params", params, p0.dtype, at, sizes)
    _check_list("grads", grads, p0.dtype, at, sizes)
    _check_list("exp_avgs", exp_avgs, state, at, sizes)
    _check_list("exp_avg_sqs", exp_avg_sqs, state, at, sizes)
    lists = [params, grads, exp_avgs, exp_avg_sqs]
    if q8:
        blocks = [-(-n // SCALE_BLOCK) for n in sizes]
        _check_list("exp_avg_scales", exp_avg_scales, torch.float32, at, blocks)
        _check_list("exp_avg_sq_scales", exp_avg_sq_scales, torch.float32, at, blocks)
        lists += [exp_avg_scales, exp_avg_sq_scales]
    _check_apart(params, grads, [t for i, ts in enumerate(lists) if i != 1 for t in ts])
    keep = [_addresses(ts) for ts in lists]
    addr = [a for _, a in keep] + ([] if q8 else [None, None])
    numel = array("q", sizes)
    args = [len(params), *addr, numel.buffer_info()[0], DTYPES[p0.dtype], 8 if q8 else 32]
    if _hyper is not None:
        launch(p0.device, _lib.lib().mtk_adamw_step_each, *args, _hyper.data_ptr())
    else:
        launch(p0.device, _lib.lib().mtk_adamw_step, *args, lr, betas[0], betas[1], eps, weight_decay, step, None)
    torch.autograd.graph.increment_version(params)  # written through raw pointers: autograd and the modules' caches have to see it


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW``'s update and arguments, plus ``state_bits`` (32 or 8: the moments' width).

    ``capturable=True`` keeps every parameter's step count (and, given as a float32 device tensor, the learning rate) on the device, so a step
    captured into a HIP graph counts its own replays; take one step before the capture, which creates the state.  Without it a step under capture is
    refused.  Parameters have to be contiguous, dense tensors of float32, bfloat16 or float16.  ``amsgrad``, ``maximize`` and ``differentiable``
    are refused unless False; ``foreach`` and ``fused`` choose between torch's own ways and say nothing here."""

    def __init__(self, params, lr: float | Tensor = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, amsgrad: bool = False, *,
                 maximize: bool = False, foreach: bool | None = None, capturable: bool = False, differentiable: bool = False, fused: bool | None = None, state_bits: int = 32):
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, amsgrad=amsgrad, maximize=maximize, foreach=foreach, capturable=capturable,
                                      differentiable=differentiable, fused=fused, state_bits=state_bits))

    @staticmethod
    def _check_group(group: dict) -> None:
        if group["state_bits"] not in (8, 32):
            raise ValueError(f"AdamW: state_bits {group['state_bits']} (8 or 32)")
        lr = group["lr"]
        if isinstance(lr, Tensor):
            if not group["capturable"] or lr.numel() != 1 or lr.dtype != torch.float32 or not lr.is_cuda:
                raise ValueError("AdamW: a tensor lr is one float32 number on the device, with capturable=True")
        elif not lr >= 0:
            raise ValueError(f"AdamW: lr {lr}")
        if not group["eps"] >= 0 or not group["weight_decay"] >= 0 or not all(0 <= b < 1 for b in group["betas"]):
            raise ValueError(f"AdamW: betas {group['betas']}, eps {group['eps']}, weight_decay {group['weight_decay']}")
        for name in ("amsgrad", "maximize", "differentiable"):
            if group.get(name):
                raise NotImplementedError(f"AdamW: {name} is not offered")

    def add_param_group(self, param_group: dict) -> None:
        self._check_group({**self.defaults, **param_group})
        super().add_param_group(param_group)

    def _init_state(self, p: Tensor, group: dict) -> dict:
        st = self.state[p]
        st["step"] = torch.zeros((), dtype=torch.int64, device=p.device) if group["capturable"] else 0
        if group["state_bits"] == 8:
            n = -(-p.numel() // SCALE_BLOCK)
            for name in ("exp_avg", "exp_avg_sq"):
                st[name] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn)
                st[name + "_scale"] = torch.ones(n, dtype=torch.float32, device=p.device)
        else:
            for name in ("exp_avg", "exp_avg_sq"):
                st[name] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        return st

    def __setstate__(self, state: dict) -> None:
        super().__setstate__(state)
        for group in self.param_groups:  # torch.optim.AdamW's groups have no width of the moments
            group.setdefault("state_bits", 32)
            group.setdefault("capturable", False)

    def load_state_dict(self, state_dict) -> None:
        """Of an ``AdamW`` or a ``torch.optim.AdamW``.  torch casts a loaded state to its parameter's type; here the moments are float32, or the codes
        they were, and every parameter has its step count: a number, or with ``capturable`` int64 on the device."""
        for saved in state_dict["param_groups"]:
            self._check_group({"state_bits": 32, "capturable": False, **saved})
        super().load_state_dict(state_dict)
        for group, saved in zip(self.param_groups, state_dict["param_groups"]):
            for i, p in zip(saved["params"], group["params"]):
                for name, v in state_dict["state"].get(i, {}).items():
                    if name == "step":
                        v = torch.tensor(int(v), dtype=torch.int64, device=p.device) if group["capturable"] else int(v)
                    elif isinstance(v, Tensor):
                        v = v.detach().to(device=p.device, dtype=torch.float32 if group["state_bits"] == 32 else v.dtype, copy=True).contiguous()
                    self.state[p][name] = v

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            sets: dict = {}  # one call per (device, type, step count); counts on the device are each parameter's own
            for p in group["params"]:
                if p.grad is None:
                    continue
                if not p.is_cuda:
                    raise RuntimeError("AdamW: midst_toolkit_amd has no CPU path; move the parameters to the MI355X")
                if p.grad.is_sparse:
                    raise ValueError("AdamW: sparse gradients are not supported")
                if not p.is_contiguous():
                    raise ValueError(f"AdamW: a parameter of shape {tuple(p.shape)} is not contiguous")
                capturing = torch.cuda.is_current_stream_capturing()
                if capturing and (not group["capturable"] or p not in self.state):
                    raise RuntimeError("AdamW: a captured step needs capturable=True and one step before the capture")
                st = self.state[p] if p in self.state and self.state[p] else self._init_state(p, group)
                g = p.grad if p.grad.dtype == p.dtype else p.grad.to(p.dtype)
                if not group["capturable"]:
                    st["step"] += 1
                key = (p.device, p.dtype, 1 if group["capturable"] else st["step"])
                sets.setdefault(key, []).append((p, g if g.is_contiguous() else g.contiguous(), st))
            for (dev, _, step), items in sets.items():
                self._run(group, dev, step, items)
        return loss

    def _run(self, group: dict, dev, step, items) -> None:
        col = lambda name: [st[name] for _, _, st in items]  # noqa: E731
        scales = {"exp_avg_scales": col("exp_avg_scale"), "exp_avg_sq_scales": col("exp_avg_sq_scale")} if group["state_bits"] == 8 else {}
        lr, hyper = group["lr"], None
        b1, b2 = group["betas"]
        if group["capturable"]:
            l = _lib.lib()
            hyper = torch.empty(len(items) * l.mtk_adamw_hyper_bytes(), dtype=torch.uint8, device=dev)
            lr_dev = lr if isinstance(lr, Tensor) else None
            if lr_dev is not None and lr_dev.device != dev:
                raise ValueError(f"AdamW: lr on {lr_dev.device}, parameters on {dev}")
            steps, at = _addresses(col("step"))
            launch(dev, l.mtk_adamw_count_each, len(steps), at, None if lr_dev is None else lr_dev.data_ptr(), 0.0 if lr_dev is not None else lr, b1, b2, group["eps"],
                   group["weight_decay"], hyper.data_ptr())
            lr = 0.0
        adamw_step([p for p, _, _ in items], [g for _, g, _ in items], col("exp_avg"), col("exp_avg_sq"), step, lr=lr, betas=(b1, b2), eps=group["eps"],
                   weight_decay=group["weight_decay"], _hyper=hyper, **scales)
