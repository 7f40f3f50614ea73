"""Low-rank fine-tunes of one denoiser, many at once, on MI355X.

The reference's ensemble attack fine-tunes whole copies of one base model, one after the other
(attacks/ensemble/clavaddpm_fine_tuning.py:45, attacks/ensemble/rmia/shadow_model_training.py:308).  Here the base is shared and frozen, a
model is a low-rank update of every linear layer, and the rows of all models run through each layer as one product:

  ``adapter_linear``   y = act(x W^T + b + s_e (x A_e^T) B_e^T) on rows sorted by model, with the gradients of x and of all A_e, B_e
  ``LowRankEnsemble``  an ``MLPDiffusion`` denoiser with E such fine-tunes: ``forward(x, timesteps, index, weights)``

Everything runs in libmtk_hip.so (mtk_adapter_forward / mtk_adapter_backward, mtk_route_rows ...), the autograd nodes in csrc/mtk_torch.cpp.  There is no CPU path.
"""
from __future__ import annotations

import math

import torch
from torch import Tensor, nn

from ._lib import native, no_tangents, ordinary
from .model import MLPDiffusion, timestep_frequencies
from .routing import MAX_GROUPS, RowPlan, combine_rows, dispatch_rows, dtype_code, route_rows, rows_of

MAX_RANK, MAX_WIDTH, MAX_ROWS = 256, 8192, 16777216  # MTK_ADAPTER_MAX_* of include/mtk.h
ACTIVATIONS = {"none": 0, "relu": 1}  # enum mtk_activation


def adapter_linear(x: Tensor, weight: Tensor, bias: Tensor | None, down: Tensor, up: Tensor, offsets: Tensor | RowPlan, scale: float | Tensor = 1.0,
                   activation: str = "none") -> Tensor:
    """``act(x W^T + b + s_e (x down_e^T) up_e^T)`` for rows sorted by model.

    ``x`` [M, din]; ``weight`` [dout, din] and ``bias`` [dout] (or None): the shared layer, frozen; ``down`` [E, r, din], ``up`` [E, dout, r]: one
    update per model; all of one type (float32, bfloat16, float16).  ``offsets``: int32 [E + 1], model e owns rows ``offsets[e]`` to
    ``offsets[e + 1] - 1`` (a ``RowPlan`` stands for its offsets); rows behind the last model's have the shared layer alone.  ``scale``: one
    number, or float32 [E] on the device, a constant.  ``activation``: "none" or "relu".  Differentiable in ``x``, ``down`` and ``up``, backward and once."""
    if isinstance(offsets, RowPlan):
        offsets = offsets.offsets
    if not x.is_cuda:
        raise RuntimeError("adapter_linear: midst_toolkit_amd has no CPU path; move the rows to the MI355X")
    if activation in ACTIVATIONS:
        got = native().adapter(x, weight, bias, down, up, offsets, scale, ACTIVATIONS[activation])
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
    scales = scale if isinstance(scale, Tensor) else None
    if scales is not None and (scales.dtype != torch.float32 or tuple(scales.shape) != (E,)):
        raise ValueError(f"adapter_linear: scale is a number or float32 [{E}], got {scales.dtype} {tuple(scales.shape)}")
    at, dt = x.get_device(), x.dtype
    for t, name in ((weight, "weight"), (bias, "bias"), (down, "down"), (up, "up")):
        if t is not None and (t.get_device() != at or t.dtype != dt):
            raise ValueError(f"adapter_linear: x is {dt} on {x.device}, {name} {t.dtype} on {t.device}")
    if offsets.get_device() != at or (scales is not None and scales.get_device() != at):
        raise ValueError(f"adapter_linear: x on {x.device}, offsets on {offsets.device}" + ("" if scales is None else f", scale on {scales.device}"))
    if torch.is_grad_enabled() and (weight.requires_grad or (bias is not None and bias.requires_grad)):
        raise NotImplementedError("adapter_linear: the shared layer is frozen; detach weight and bias")
    if torch.is_grad_enabled() and scales is not None and scales.requires_grad:
        raise NotImplementedError("adapter_linear: scale gets no gradient; detach it")
    no_tangents("adapter_linear", x, weight, bias, down, up, scale)
    c = lambda t: t if t is None else t.contiguous()  # noqa: E731
    return ordinary("adapter_linear", x.device, native().adapter, rows_of(x), c(weight), c(bias), c(down), c(up), c(offsets),
                    float(scale) if scales is None else c(scales), ACTIVATIONS[activation])


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
        plan = route_rows(index.to(x.device), self.n_models)
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
