"""Low-rank fine-tunes of one denoiser, many at once, on MI355X.

The reference's ensemble attack fine-tunes whole copies of one base model, one after the other
(attacks/ensemble/clavaddpm_fine_tuning.py:45, attacks/ensemble/rmia/shadow_model_training.py:308).  Here the base is shared and frozen, a
model is a low-rank update of every linear layer, and the rows of all models run through each layer as one product:

  ``adapter_linear``   y = act(x W^T + b + s_e (x A_e^T) B_e^T) on rows sorted by model, with the gradients of x and of all A_e, B_e
  ``LowRankEnsemble``  an ``MLPDiffusion`` denoiser with E such fine-tunes: ``forward(x, timesteps, index, weights)``

Everything runs in libmtk_hip.so (mtk_adapter_forward / mtk_adapter_backward, mtk_route_rows ...).  There is no CPU path.
"""
from __future__ import annotations

import math

import torch
from torch import Tensor, nn
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import launch, native, raw_stream
from .model import MLPDiffusion, timestep_frequencies
from .routing import DTYPES, MAX_GROUPS, RowPlan, combine_rows, dispatch_rows, dtype_code, route_rows, rows_of

MAX_RANK, MAX_WIDTH, MAX_ROWS = 256, 8192, 16777216  # MTK_ADAPTER_MAX_* of include/mtk.h
ACTIVATIONS = {"none": 0, "relu": 1}  # enum mtk_activation


def _forward(x, weight, bias, down, up, offsets, scales, scale, act, keep):
    """mtk_adapter_forward: (y, what the backward reads of it)"""
    got = native().adapter_forward(x, weight, bias, down, up, offsets, scale if scales is None else scales, act, 1, raw_stream(x.get_device())) if keep else None
    if got is not None:
        return got
    dev, (M, din), (E, r, _), dout = x.device, x.shape, down.shape, weight.shape[0]
    l, dt = _lib.lib(), DTYPES[x.dtype]
    y = torch.empty((M, dout), dtype=x.dtype, device=dev)
    saved = torch.empty(l.mtk_adapter_saved_bytes(M, r, dt), dtype=torch.uint8, device=dev)
    if M:
        need = l.mtk_adapter_work_bytes(M, din, dout, r, E, dt, act, 0)
        work = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        launch(dev, l.mtk_adapter_forward, M, din, dout, r, E, dt, x.data_ptr(), x.stride(0), weight.data_ptr(), None if bias is None else bias.data_ptr(),
               down.data_ptr(), up.data_ptr(), offsets.data_ptr(), None if scales is None else scales.data_ptr(), scale, act, int(keep), y.data_ptr(),
               saved.data_ptr(), saved.numel(), None if work is None else work.data_ptr(), need)
    return y, saved


class _AdapterLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, down, up, offsets, scales, scale, act):
        xr = rows_of(x)
        y, saved = _forward(xr, weight, bias, down, up, offsets, scales, scale, act, True)
        ctx.save_for_backward(xr, weight, down, up, offsets, scales, y if act else None, saved)
        ctx.scale, ctx.act = scale, act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        x, weight, down, up, offsets, scales, y, saved = ctx.saved_tensors
        dev, (M, din), (E, r, _), dout = x.device, x.shape, down.shape, weight.shape[0]
        l, dt = _lib.lib(), DTYPES[x.dtype]
        want = ctx.needs_input_grad
        g = g.contiguous()
        got = native().adapter_backward(x, weight, down, up, offsets, ctx.scale if scales is None else scales, ctx.act, y, g, saved,
                                        want[0] + 2 * want[3] + 4 * want[4], raw_stream(x.get_device()))
        if got is not None:
            return got[0], None, None, got[1], got[2], None, None, None, None
        dx = torch.empty((M, din), dtype=x.dtype, device=dev) if want[0] else None
        if M == 0:
            return dx, None, None, torch.zeros_like(down) if want[3] else None, torch.zeros_like(up) if want[4] else None, None, None, None, None
        ddown = torch.empty_like(down) if want[3] else None
        dup = torch.empty_like(up) if want[4] else None
        work = torch.empty(l.mtk_adapter_work_bytes(M, din, dout, r, E, dt, ctx.act, 1), dtype=torch.uint8, device=dev)
        p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        launch(dev, l.mtk_adapter_backward, M, din, dout, r, E, dt, x.data_ptr(), x.stride(0), weight.data_ptr(), down.data_ptr(), up.data_ptr(),
               offsets.data_ptr(), p(scales), ctx.scale, ctx.act, p(y), g.data_ptr(), saved.data_ptr(), p(dx), p(ddown), p(dup), work.data_ptr(), work.numel())
        return dx, None, None, ddown, dup, None, None, None, None


def adapter_linear(x: Tensor, weight: Tensor, bias: Tensor | None, down: Tensor, up: Tensor, offsets: Tensor | RowPlan, scale: float | Tensor = 1.0,
                   activation: str = "none") -> Tensor:
    """``act(x W^T + b + s_e (x down_e^T) up_e^T)`` for rows sorted by model.

    ``x`` [M, din]; ``weight`` [dout, din] and ``bias`` [dout] (or None): the shared layer, frozen; ``down`` [E, r, din], ``up`` [E, dout, r]: one
    update per model; all of one type (float32, bfloat16, float16).  ``offsets``: int32 [E + 1], model e owns rows ``offsets[e]`` to
    ``offsets[e + 1] - 1`` (a ``RowPlan`` stands for its offsets); rows behind the last model's have the shared layer alone.  ``scale``: one
    number, or float32 [E] on the device.  ``activation``: "none" or "relu".  Differentiable in ``x``, ``down`` and ``up``."""
    if isinstance(offsets, RowPlan):
        offsets = offsets.offsets
    if not x.is_cuda:
        raise RuntimeError("adapter_linear: midst_toolkit_amd has no CPU path; move the rows to the MI355X")
    if activation in ACTIVATIONS:
        got = native().adapter_forward(x, weight, bias, down, up, offsets, scale, ACTIVATIONS[activation], 0, raw_stream(x.get_device()))
        if got is not None:
            return got
    dtype_code(x, "adapter_linear")
    if x.dim() != 2 or weight.dim() != 2 or down.dim() != 3 or up.dim() != 3:
        raise ValueError("adapter_linear: x [M, din], weight [dout, din], down [E, r, din], up [E, dout, r]")
    (M, din), (E, r, _), dout = x.shape, down.shape, weight.shape[0]
    if weight.shape[1] != din or down.shape[2] != din or tuple(up.shape) != (E, dout, r) or (bias is not None and tuple(bias.shape) != (dout,)):
        raise ValueError(f"adapter_linear: shapes do not fit: x {tuple(x.shape)}, weight {tuple(weight.shape)}, down {tuple(down.shape)}, up {tuple(up.shape)}"
                         + ("" if bias is None else f", bias {tuple(bias.shape)}"))
    if min(din, dout, r, E) < 1 or r > MAX_RANK or max(din, dout) > MAX_WIDTH or E > MAX_GROUPS or M > MAX_ROWS:
        raise ValueError(f"adapter_linear: {M} rows, {din} -> {dout} features, rank {r}, {E} models (up to {MAX_ROWS} rows, {MAX_WIDTH} features, rank "
                         f"{MAX_RANK}, {MAX_GROUPS} models, and none of them 0 but the rows)")
    if offsets.dtype != torch.int32 or tuple(offsets.shape) != (E + 1,):
        raise ValueError(f"adapter_linear: offsets are int32 [{E + 1}], got {offsets.dtype} {tuple(offsets.shape)}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"adapter_linear: activation {activation!r} (none or relu)")
    scales = None
    if isinstance(scale, Tensor):
        if scale.dtype != torch.float32 or tuple(scale.shape) != (E,):
            raise ValueError(f"adapter_linear: scale is a number or float32 [{E}], got {scale.dtype} {tuple(scale.shape)}")
        scales, scale = scale.detach().contiguous(), 1.0
    at, dt = x.get_device(), x.dtype
    for t, name in ((weight, "weight"), (bias, "bias"), (down, "down"), (up, "up")):
        if t is not None and (t.get_device() != at or t.dtype != dt):
            raise ValueError(f"adapter_linear: x is {dt} on {x.device}, {name} {t.dtype} on {t.device}")
    if offsets.get_device() != at or (scales is not None and scales.get_device() != at):
        raise ValueError(f"adapter_linear: x on {x.device}, offsets on {offsets.device}" + ("" if scales is None else f", scale on {scales.device}"))
    c = lambda t: t if t is None or t.is_contiguous() else t.contiguous()  # noqa: E731
    args = (c(weight), c(bias), c(down), c(up), c(offsets), scales, float(scale), ACTIVATIONS[activation])
    if torch.is_grad_enabled():
        if weight.requires_grad or (bias is not None and bias.requires_grad):
            raise NotImplementedError("adapter_linear: the shared layer is frozen; detach weight and bias")
        if x.requires_grad or down.requires_grad or up.requires_grad:
            return _AdapterLinear.apply(x, *args)
    return _forward(rows_of(x), *args, False)[0]


class LowRankEnsemble(nn.Module):
    """``n_models`` low-rank fine-tunes of a trained ``MLPDiffusion`` (the denoiser's ``proj``, blocks and head, MODEL:596-615; the
    time-embedding MLP is shared as it is).  The base weights are copied and frozen; the parameters are ``down[i]`` [E, r, in] and
    ``up[i]`` [E, out, r] of layer i.  ``up`` starts at zero, so every model starts as the base."""

    def __init__(self, denoiser: MLPDiffusion, n_models: int, rank: int = 16, alpha: float | None = None, num_timesteps: int | None = None):
        super().__init__()
        if getattr(denoiser, "label_conditioned", False):
            raise NotImplementedError("LowRankEnsemble: label-conditioned denoisers (IsTargetConditioned.EMBEDDING) are not supported")
        if not 1 <= n_models <= MAX_GROUPS or not 1 <= rank <= MAX_RANK:
            raise ValueError(f"LowRankEnsemble: {n_models} models of rank {rank} (up to {MAX_GROUPS} of rank {MAX_RANK})")
        if denoiser.training_dropout() != 0.0:
            raise NotImplementedError("LowRankEnsemble: the layers carry no dropout masks; call denoiser.eval() first")
        self.n_models, self.rank = n_models, rank
        self.scale = float(alpha if alpha is not None else rank) / rank
        self.num_timesteps = int(num_timesteps if num_timesteps is not None else denoiser.num_timesteps)
        layers = [denoiser.proj] + [b.linear for b in denoiser.mlp.blocks] + [denoiser.mlp.head]
        self.down, self.up = nn.ParameterList(), nn.ParameterList()
        for i, m in enumerate(layers):
            W = m.weight.detach()
            self.register_buffer(f"weight{i}", W.clone())
            self.register_buffer(f"bias{i}", m.bias.detach().clone())
            self.down.append(nn.Parameter(torch.randn(n_models, rank, W.shape[1], dtype=W.dtype, device=W.device) / math.sqrt(W.shape[1])))
            self.up.append(nn.Parameter(torch.zeros(n_models, W.shape[0], rank, dtype=W.dtype, device=W.device)))
        # MODEL:608: the time embedding depends on the timestep only: one table, evaluated once in 64 bits (frozen like the base)
        first, second = denoiser.timestep_embedding[0], denoiser.timestep_embedding[2]
        f = timestep_frequencies(denoiser.timestep_dimension).to(first.weight.device)
        arg = torch.arange(self.num_timesteps, device=f.device, dtype=torch.float32)[:, None] * f[None]
        table = torch.cat([torch.cos(arg), torch.sin(arg)], 1)
        if denoiser.timestep_dimension % 2:
            table = torch.cat([table, torch.zeros_like(table[:, :1])], 1)
        d = lambda t: t.detach().double()  # noqa: E731
        h = nn.functional.silu(table.double() @ d(first.weight).t() + d(first.bias))
        emb = h @ d(second.weight).t() + d(second.bias)
        self.register_buffer("time_table", emb.to(first.weight.dtype))

    def forward(self, x: Tensor, timesteps: Tensor, index: Tensor, weights: Tensor | None = None) -> Tensor:
        """``x`` [N, D], ``timesteps`` [N], ``index`` [N] or [N, k]: the models of record n (-1: the base).  -> [N, D]: the models' outputs for a
        record added up with ``weights`` (float32, ``index``'s shape; None: their mean).  Differentiable in the parameters and ``x``.
        Rows of a timestep or index out of range are NaN."""
        if not x.is_cuda:
            raise RuntimeError("LowRankEnsemble.forward: midst_toolkit_amd has no CPU path; move the module and inputs to the MI355X")
        if x.dim() != 2 or x.shape[1] != self.weight0.shape[1]:
            raise ValueError(f"LowRankEnsemble: x is [N, {self.weight0.shape[1]}], got {tuple(x.shape)}")
        if timesteps.shape != x.shape[:1] or index.shape[:1] != x.shape[:1]:
            raise ValueError(f"LowRankEnsemble: {x.shape[0]} records, timesteps {tuple(timesteps.shape)}, index {tuple(index.shape)}")
        plan = route_rows(index, self.n_models)
        t = timesteps.to(device=x.device, dtype=torch.int64)
        emb = self.time_table[t.clamp(0, self.num_timesteps - 1)]
        emb = torch.where(((t < 0) | (t >= self.num_timesteps))[:, None], float("nan"), emb)
        h = adapter_linear(dispatch_rows(x, plan), self.weight0, self.bias0, self.down[0], self.up[0], plan, self.scale)
        h = h + dispatch_rows(emb, plan)
        last = len(self.down) - 1
        for i in range(1, last + 1):
            h = adapter_linear(h, getattr(self, f"weight{i}"), getattr(self, f"bias{i}"), self.down[i], self.up[i], plan, self.scale,
                               "relu" if i < last else "none")
        if weights is None and plan.copies > 1:
            weights = torch.full((plan.n_rows, plan.copies), 1.0 / plan.copies, dtype=torch.float32, device=x.device)
        return combine_rows(h, plan, weights)
