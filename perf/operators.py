"""The measured cases of three operators around ensembles of fine-tuned denoisers and their training.

rows     pairs (record, model) sorted by model and back: the plan from the model indices, the records' rows copied into the plan's
         order, the models' outputs brought back and added with weights; training: the gradients of both copies and of the weights
adapter  a linear layer shared by all models with one low-rank update per model, on rows sorted by model; training: the gradients
         of the rows and of the low-rank factors (the shared weights are frozen)
adamw    one AdamW step over many tensors, the moments held in 32 bits or in 8 (e4m3 codes with a power-of-two scale per 256 values)
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
BLOCK = 256  # values that share a scale of the 8-bit moments


# ------------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # a handful of records scored under two shadow models each, one request: launches count
        {"name": "rows serve 24", "op": "rows", "rows": 24, "copies": 2, "groups": 8, "width": 120, "dtype": "fp32", "train": False},
        # a training batch of the denoiser's size, ragged width, four models a record
        {"name": "rows train 4099", "op": "rows", "rows": 4099, "copies": 4, "groups": 17, "width": 1021, "dtype": "fp32", "train": True},
        # a whole table's hidden rows under two of sixteen models
        {"name": "rows train 100000", "op": "rows", "rows": 100000, "copies": 2, "groups": 16, "width": 1024, "dtype": "bf16", "train": True},
        # one record through one hidden layer
        {"name": "adapter serve 1", "op": "adapter", "rows": 1, "din": 1024, "dout": 1024, "rank": 8, "groups": 16, "dtype": "bf16", "relu": True, "train": False},
        # a small mixed request: a few rows of each of sixteen models
        {"name": "adapter serve 61", "op": "adapter", "rows": 61, "din": 512, "dout": 1024, "rank": 16, "groups": 16, "dtype": "fp32", "relu": True, "train": False},
        # one rank's training batch, in the denoiser's default precision
        {"name": "adapter train 2048", "op": "adapter", "rows": 2048, "din": 1024, "dout": 1024, "rank": 16, "groups": 16, "dtype": "fp32", "relu": False, "train": True},
        # scoring with odd sizes: nothing divides a tile, rows are not aligned
        {"name": "adapter serve 20011", "op": "adapter", "rows": 20011, "din": 517, "dout": 1021, "rank": 12, "groups": 33, "dtype": "fp16", "relu": True, "train": False},
        # a large training batch over sixteen models
        {"name": "adapter train 65536", "op": "adapter", "rows": 65536, "din": 1024, "dout": 1024, "rank": 16, "groups": 16, "dtype": "bf16", "relu": False, "train": True},
        # the low-rank factors of sixteen models of a six-layer denoiser: many small tensors
        {"name": "adamw adapters 32 bit", "op": "adamw", "tensors": 12, "values": 2200000, "dtype": "fp32", "bits": 32},
        # the same with the moments in 8 bits
        {"name": "adamw adapters 8 bit", "op": "adamw", "tensors": 12, "values": 2200000, "dtype": "fp32", "bits": 8},
        # sixteen whole denoisers in one step
        {"name": "adamw models 32 bit", "op": "adamw", "tensors": 192, "values": 55000000, "dtype": "fp32", "bits": 32},
        {"name": "adamw models 8 bit", "op": "adamw", "tensors": 192, "values": 220000000, "dtype": "bf16", "bits": 8},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rows", "adapter", "adamw"))
    if op == "rows":
        while True:
            c = {"op": op, "rows": _log(rng, 1, 100000), "copies": rng.randint(1, 8), "groups": _log(rng, 1, 300), "width": _log(rng, 1, 2048),
                 "dtype": rng.choice(list(TYPES)), "train": rng.random() < 0.5}
            if c["rows"] * c["copies"] * c["width"] * SIZE[c["dtype"]] <= 100000 * 2 * 1024 * 2:
                return c
    if op == "adapter":
        while True:
            c = {"op": op, "rows": _log(rng, 1, 65536), "din": _log(rng, 16, 2048), "dout": _log(rng, 16, 2048), "rank": _log(rng, 1, 64),
                 "groups": _log(rng, 1, 64), "dtype": rng.choice(list(TYPES)), "relu": False, "train": rng.random() < 0.5}
            c["relu"] = not c["train"] and rng.random() < 0.5
            cost = c["rows"] * (c["din"] * c["dout"] + c["groups"] * c["rank"] * (c["din"] + c["dout"])) * (4 if c["dtype"] == "fp32" else 1)
            if cost <= 65536 * 1024 * 1024:
                return c
    return {"op": op, "tensors": _log(rng, 1, 300), "values": _log(rng, 3000, 100000000), "dtype": rng.choice(list(TYPES)), "bits": rng.choice((8, 32))}


# ------------------------------------------------------------------------------------------------------------------ inputs
def _popular(g, n, groups):
    """Model indices as they meet a service: a few models take most rows, some none; about one row in twenty has the base alone (-1)."""
    p = 1.0 / torch.arange(1, groups + 1, device=DEV, dtype=torch.float32)
    p = p[torch.randperm(groups, generator=g, device=DEV)]
    cdf = torch.cumsum(p / p.sum(), 0)
    index = torch.searchsorted(cdf, torch.rand(n, generator=g, device=DEV)).clamp_(max=groups - 1)
    return torch.where(torch.rand(n, generator=g, device=DEV) < 0.05, -1, index)


def _tensor_sizes(tensors, values):
    """Layer sizes of a model: widths and biases in turn, whole and odd."""
    r = np.random.RandomState(tensors * 7 + values % 1000)
    w = np.where(np.arange(tensors) % 2 == 0, r.uniform(0.5, 1.5, tensors), r.uniform(0.0005, 0.02, tensors))
    return [max(1, int(v)) for v in w / w.sum() * values]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case)
    dt = TYPES[case["dtype"]]
    randn = lambda *shape: torch.randn(shape, generator=g, device=DEV)  # noqa: E731
    if case["op"] == "rows":
        n, k, d = case["rows"], case["copies"], case["width"]
        s["index"] = _popular(g, n * k, case["groups"]).reshape(n, k)
        s["x"] = randn(n, d).to(dt).requires_grad_(case["train"])
        s["y"] = randn(n * k, d).to(dt).requires_grad_(case["train"])
        s["weights"] = torch.softmax(randn(n, k), 1).requires_grad_(case["train"])
        if case["train"]:
            s["gx"], s["gout"] = randn(n * k, d).to(dt), randn(n, d).to(dt)
    elif case["op"] == "adapter":
        n, din, dout, r, e = (case[q] for q in ("rows", "din", "dout", "rank", "groups"))
        index = _popular(g, n, e)
        index = torch.where(index < 0, e, index)
        s["offsets"] = torch.searchsorted(index.sort().values, torch.arange(e + 1, device=DEV)).to(torch.int32)
        s["x"] = torch.relu(randn(n, din) + 0.2).to(dt).requires_grad_(case["train"])
        s["weight"] = (randn(dout, din) / math.sqrt(din)).to(dt)
        s["bias"] = (randn(dout) * 0.1).to(dt)
        s["down"] = (randn(e, r, din) / math.sqrt(din)).to(dt).requires_grad_(case["train"])
        s["up"] = (randn(e, dout, r) * 0.1).to(dt).requires_grad_(case["train"])
        s["scale"] = torch.rand(e, generator=g, device=DEV) + 0.5
        if case["train"]:
            s["gy"] = randn(n, dout).to(dt)
    else:
        sizes = _tensor_sizes(case["tensors"], case["values"])
        starts = np.cumsum([0] + [-(-v // BLOCK) * BLOCK for v in sizes])
        total = int(starts[-1])
        cut = lambda flat: [flat[a:a + v] for a, v in zip(starts.tolist(), sizes)]  # noqa: E731
        used = torch.zeros(total, device=DEV)
        for v in cut(used):
            v.fill_(1)
        # gradients whose size differs from value to value by some orders, as layers' do; moments of a run some steps old
        spread = torch.exp(2 * randn(total))
        s["flat_p"] = (randn(total) * 0.05 * used).to(dt)
        s["flat_g"] = (randn(total) * 1e-3 * spread * used).to(dt)
        m, v = randn(total) * 3e-4 * spread * used, (1e-3 * spread * used * (0.5 + torch.rand(total, generator=g, device=DEV))) ** 2
        if case["bits"] == 8:
            m, r = m.view(-1, BLOCK), v.sqrt().view(-1, BLOCK)
            ms, rs = (torch.exp2(torch.ceil(torch.log2(q.abs().amax(1).clamp(min=1e-30) / 448))) for q in (m, r))
            s["flat_m"] = (m / ms[:, None]).to(torch.float8_e4m3fn).view(-1)
            s["flat_v"] = (r / rs[:, None]).to(torch.float8_e4m3fn).view(-1)
            s["flat_ms"], s["flat_vs"] = ms, rs
            first = torch.from_numpy(starts).to(DEV)
            at = torch.arange(total, device=DEV)
            s["place"] = (at - first[torch.searchsorted(first, at, right=True) - 1]).int()  # each value's place in its own tensor
            blocks = [-(-q // BLOCK) for q in sizes]
            s["ms"], s["vs"] = list(ms.split(blocks)), list(rs.split(blocks))
        else:
            s["flat_m"], s["flat_v"] = m, v
        s["p"], s["g"], s["m"], s["v"] = (cut(s[q]) for q in ("flat_p", "flat_g", "flat_m", "flat_v"))
        s["step"] = 40
    return s


# ------------------------------------------------------------------------------------------------------------- plain forms
def _plain_rows(s):
    n, k, e = s["rows"], s["copies"], s["groups"]
    key = s["index"].reshape(-1)
    key = torch.where(key < 0, e, key)
    order = torch.sort(key, stable=True).indices
    slot = torch.empty_like(order)
    slot[order] = torch.arange(n * k, device=DEV)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), torch.cumsum(torch.bincount(key, minlength=e + 1)[:e], 0)])
    xs = s["x"][order // k]
    out = (s["y"][slot].float().view(n, k, -1) * s["weights"][:, :, None]).sum(1).to(s["y"].dtype)
    got = {"order": order.int(), "slot": slot.int().view(n, k), "offsets": offsets.int(), "xs": xs.detach(), "out": out.detach()}
    if s["train"]:
        got["dx"] = s["gx"][slot].float().view(n, k, -1).sum(1).to(s["x"].dtype)
        go = s["gout"].float()
        got["dy"] = (go[order // k] * s["weights"].detach().reshape(-1)[order][:, None]).to(s["y"].dtype)
        got["dweights"] = (s["y"].detach()[slot].float().view(n, k, -1) * go[:, None, :]).sum(2)
    return got


def _plain_adapter(s):
    e, r, din = s["down"].shape
    dout = s["up"].shape[1]
    x, w, down, up = (s[q].float() for q in ("x", "weight", "down", "up"))
    group = torch.searchsorted(s["offsets"][1:], torch.arange(x.shape[0], device=DEV, dtype=torch.int32), right=True)
    pick = (group[:, None] == torch.arange(e, device=DEV)) * s["scale"]
    low = (x @ down.reshape(e * r, din).t()).view(-1, e, r) * pick[:, :, None]
    y = x @ w.t() + s["bias"].float() + low.reshape(-1, e * r) @ up.permute(0, 2, 1).reshape(e * r, dout)
    if s["relu"]:
        y = torch.relu(y)
    return y.to(s["x"].dtype)


def _wrap(v):
    """`v` modulo 2^32 as a signed 32-bit number."""
    return (v + 2**31) % 2**32 - 2**31


def _dithered(value, u24, lowest):
    """e4m3 codes of value's blocks of 256 under a power-of-two scale: each value goes to one of its two neighbours by u24 (24 bits of
    a Weyl sequence); non-zero values go to `lowest` at least."""
    value = value.view(-1, BLOCK)
    mant, ex = torch.frexp(value.abs().amax(1))
    scale = torch.where(mant > 0, torch.ldexp(torch.ones_like(mant), (ex - 9 + (mant > 0.875).int()).clamp(min=-126)), 1.0)
    y = (value / scale[:, None]).abs()
    step = torch.exp2(torch.frexp(y).exponent.clamp(min=-5).float() - 4)  # spacing of the codes around y
    y = (torch.floor(y / step + (u24.view(-1, BLOCK) >> 4).float() * 2.0**-20) * step).clamp(max=448.0)
    y = torch.where(value != 0, y.clamp(min=lowest), y) * torch.sign(value)
    return y.to(torch.float8_e4m3fn).view(-1), scale


def _plain_adamw(s, lr=1e-4, b1=0.9, b2=0.999, eps=1e-8, wd=1e-2):
    step = s["step"]
    p, g = s["flat_p"].float(), s["flat_g"].float()
    m, v = s["flat_m"].float(), s["flat_v"].float()
    if s["bits"] == 8:
        m = (m.view(-1, BLOCK) * s["flat_ms"][:, None]).view(-1)
        v = (v.view(-1, BLOCK) * s["flat_vs"][:, None]).view(-1)
        v = v * v
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * (g * g)
    root = v.sqrt()
    p = p * (1 - lr * wd) - (lr / (1 - b1**step)) * (m / (root / math.sqrt(1 - b2**step) + eps))
    s["flat_p"].copy_(p)
    if s["bits"] == 8:
        phase = _wrap(step * 0x9E3779B1)
        um = (s["place"] * _wrap(0x6A09E667) + phase) >> 8 & 0xFFFFFF
        uv = (s["place"] * _wrap(0xBB67AE85) + phase) >> 8 & 0xFFFFFF
        m8, ms = _dithered(m, um, 0.0)
        v8, vs = _dithered(root, uv, 2.0**-9)
        s["flat_m"].copy_(m8), s["flat_v"].copy_(v8), s["flat_ms"].copy_(ms), s["flat_vs"].copy_(vs)
    else:
        s["flat_m"].copy_(m), s["flat_v"].copy_(v)


# ------------------------------------------------------------------------------------------------------------------ passes
def _adamw_state(s):
    got = {"params": s["flat_p"], "exp_avg": s["flat_m"], "exp_avg_sq": s["flat_v"]}
    if s["bits"] == 8:
        got |= {"exp_avg_scale": s["flat_ms"], "exp_avg_sq_scale": s["flat_vs"]}
    return got


def run(s):
    if own:
        import midst_toolkit_amd as mtk
    if s["op"] == "rows":
        if not own:
            return _plain_rows(s)
        plan = mtk.route_rows(s["index"], s["groups"])
        xs = mtk.dispatch_rows(s["x"], plan)
        out = mtk.combine_rows(s["y"], plan, s["weights"])
        got = {"order": plan.order, "slot": plan.slot, "offsets": plan.offsets, "xs": xs.detach(), "out": out.detach()}
        if s["train"]:
            got["dx"], got["dy"], got["dweights"] = torch.autograd.grad((xs, out), (s["x"], s["y"], s["weights"]), (s["gx"], s["gout"]))
        return got
    if s["op"] == "adapter":
        if own:
            y = mtk.adapter_linear(s["x"], s["weight"], s["bias"], s["down"], s["up"], s["offsets"], scale=s["scale"], activation="relu" if s["relu"] else "none")
        else:
            y = _plain_adapter(s)
        if not s["train"]:
            return {"y": y}
        dx, ddown, dup = torch.autograd.grad(y, (s["x"], s["down"], s["up"]), s["gy"])
        return {"y": y.detach(), "dx": dx, "ddown": ddown, "dup": dup}
    s["step"] += 1
    if own:
        scales = {"exp_avg_scales": s["ms"], "exp_avg_sq_scales": s["vs"]} if s["bits"] == 8 else {}
        mtk.adamw_step(s["p"], s["g"], s["m"], s["v"], s["step"], lr=1e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, **scales)
    else:
        _plain_adamw(s)
    return _adamw_state(s)


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "rows":
        n, p = case["rows"], case["rows"] * case["copies"]
        forth = (n + p) * case["width"] * size  # a copy out, or back
        plan = p * (8 + 4 + 4 + 4)
        both = 2 * forth + plan
        if case["train"]:
            both += forth + (n + 2 * p) * case["width"] * size + 8 * p
        return {"bytes": both, "flops": (4 if case["train"] else 2) * p * case["width"]}
    if case["op"] == "adapter":
        n, i, o, r, e = (case[q] for q in ("rows", "din", "dout", "rank", "groups"))
        e = min(e, n)
        low = 2 * n * r * (i + o)
        if not case["train"]:
            return {"bytes": (n * (i + o) + i * o + o + e * r * (i + o)) * size, "flops": 2 * n * i * o + low}
        return {"bytes": (2 * n * (i + o) + i * o + o + 2 * e * r * (i + o)) * size, "flops": 4 * n * i * o + 3 * low}
    each = 3 * size + (16 if case["bits"] == 32 else 4 + 16 / BLOCK)
    return {"bytes": case["values"] * each, "flops": 16 * case["values"]}


# ------------------------------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rows":
        n, k = case["rows"], case["copies"]
        flat = s["index"].reshape(-1).cpu().numpy().copy()
        flat[flat < 0] = case["groups"]
        order = torch.from_numpy(np.argsort(flat, kind="stable")).to(DEV)
        slot = torch.argsort(order).view(n, k)
        w = s["weights"].detach().double()
        y, out = s["y"].detach(), torch.zeros(n, case["width"], dtype=torch.float64, device=DEV)
        for j in range(k):
            out += w[:, j, None] * y[slot[:, j]].double()
        got = {"order": None, "slot": None, "offsets": None, "xs": s["x"].detach()[order // k].double(), "out": out}
        if case["train"]:
            got["dx"] = torch.zeros_like(out)
            got["dy"] = torch.empty(n * k, case["width"], dtype=torch.float64, device=DEV)
            got["dweights"] = torch.empty_like(w)
            go = s["gout"].double()
            for j in range(k):
                got["dx"] += s["gx"][slot[:, j]].double()
                got["dy"][slot[:, j]] = w[:, j, None] * go
                got["dweights"][:, j] = (go * y[slot[:, j]].double()).sum(1)
        return got
    if case["op"] == "adapter":
        x, w, down, up, scale = (s[q].detach().double() for q in ("x", "weight", "down", "up", "scale"))
        ends = s["offsets"].tolist()
        y = x @ w.t() + s["bias"].double()
        got = {"y": y}
        if case["train"]:
            gy = s["gy"].double()
            got |= {"dx": gy @ w, "ddown": torch.zeros_like(down), "dup": torch.zeros_like(up)}
        for q, (a, b) in enumerate(zip(ends[:-1], ends[1:])):
            if a == b:
                continue
            low = x[a:b] @ down[q].t()
            y[a:b] += scale[q] * (low @ up[q].t())
            if case["train"]:
                back = gy[a:b] @ up[q]
                got["dx"][a:b] += scale[q] * (back @ down[q])
                got["ddown"][q] = scale[q] * (back.t() @ x[a:b])
                got["dup"][q] = scale[q] * (gy[a:b].t() @ low)
        if case["relu"]:
            y.clamp_(min=0)
        return got
    t = s["step"] + 1
    g, m, v = s["flat_g"].double(), s["flat_m"].double(), s["flat_v"].double()
    if case["bits"] == 8:
        m = m * s["flat_ms"].double().repeat_interleave(BLOCK)
        v = (v * s["flat_vs"].double().repeat_interleave(BLOCK)) ** 2
    m = m + (1 - 0.9) * (g - m)
    v = v + (1 - 0.999) * (g * g - v)
    p = s["flat_p"].double() * (1 - 1e-4 * 1e-2)
    p -= 1e-4 * (m / (1 - 0.9**t)) / (torch.sqrt(v / (1 - 0.999**t)) + 1e-8)
    whole = case["bits"] == 32
    got = {"params": p, "exp_avg": m if whole else None, "exp_avg_sq": v if whole else None}
    return got if whole else got | {"exp_avg_scale": None, "exp_avg_sq_scale": None}
