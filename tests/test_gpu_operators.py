"""GPU: rows sorted by model and back, low-rank adapted linear layers, AdamW over many tensors - each against 64 bits (tests/operator_refs.py).

Tolerances count roundings.  A sum of K fp32 products is off by at most (K + 2) 2^-24 of the sum of its terms' magnitudes (each product
and each addition rounds by half a step); TWICE is allowed for the matrix instructions, whose inner additions may be in any order and
truncate (a whole step).  A stored 16-bit value is off by half a step of its type, eps / 2 of its magnitude; subnormal fp16 results by
half the smallest step, 2^-25."""
import math

import numpy as np
import pytest
import torch

import midst_toolkit_amd as mtk
from tests.operator_refs import adamw8_reference, adapter_reference, route_reference

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U32, TWICE = 2.0**-24, 2.0


def half(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    return 2.0**-25 if dt == torch.float16 else 2.0**-133 if dt == torch.bfloat16 else 2.0**-149


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dt=torch.float32):
    return torch.randn(shape, generator=g).to(dt).to(DEV)


def within(got, want, tol):
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), (float(((got - want).abs() - tol).max()), bad.nonzero()[:4].tolist())


# ------------------------------------------------------------------------------------------------------------------- rows
def make_index(g, N, k, E, kind):
    if kind == "one":
        return torch.full((N, k), E - 1, dtype=torch.int64)
    if kind == "none":
        return torch.full((N, k), -1, dtype=torch.int64)
    idx = torch.randint(-1, E, (N, k), generator=g)
    if kind == "few":  # most models without a pair
        idx = torch.where(idx < 0, idx, idx // max(1, E // 2) * max(1, E // 2))
    if kind == "bad" and N:
        idx[N // 2, 0], idx[N - 1, k - 1] = E, -7
    return idx


@pytest.mark.parametrize("N,k,E,kind", [(1, 1, 1, "any"), (1, 1, 1, "none"), (5, 3, 4, "bad"), (63, 1, 2, "any"), (64, 2, 1024, "any"), (777, 3, 31, "few"), (4096, 2, 16, "one"),
                                        (4097, 2, 17, "any"), (9000, 1, 3, "bad"), (30011, 4, 300, "any"), (70000, 3, 1024, "few"), (300000, 4, 5, "any")])
def test_plan_is_the_stable_sort(N, k, E, kind):
    idx = make_index(gen(N + k + E), N, k, E, kind)
    plan = mtk.route_rows(idx.to(DEV), E)
    order, slot, offsets = route_reference(idx.numpy(), E)
    assert np.array_equal(plan.order.cpu().numpy(), order)
    assert np.array_equal(plan.slot.cpu().numpy(), slot)
    assert np.array_equal(plan.offsets.cpu().numpy(), offsets)


def test_plan_shapes_and_types():
    for idx in (torch.tensor([2, 0, -1, 2]), torch.tensor([2, 0, -1, 2], dtype=torch.int32), torch.tensor([[2, 0, -1, 2]]).t(), torch.tensor([2, 0, -1, 2])[:0]):
        plan = mtk.route_rows(idx.to(DEV), 3)
        order, slot, offsets = route_reference(idx.numpy(), 3)
        assert np.array_equal(plan.order.cpu().numpy(), order) and np.array_equal(plan.slot.cpu().numpy(), slot) and np.array_equal(plan.offsets.cpu().numpy(), offsets)
    for bad in (torch.zeros(3), torch.zeros(3, dtype=torch.bool), torch.zeros(2, 2, 2, dtype=torch.int64), torch.zeros(3, 0, dtype=torch.int64)):
        with pytest.raises(ValueError):
            mtk.route_rows(bad.to(DEV), 3)
    for e in (0, 1025):
        with pytest.raises(ValueError):
            mtk.route_rows(torch.zeros(3, dtype=torch.int64, device=DEV), e)


def test_plans_and_weights_that_are_not_what_they_say():
    """A number of models that is not whole is not cut, weights without dimensions are not a record's"""
    idx = torch.zeros(1, dtype=torch.int64, device=DEV)
    for bad in (2.5, 2.0, "2", None):
        with pytest.raises(ValueError, match="whole number"):
            mtk.route_rows(idx, bad)
    assert mtk.route_rows(idx, np.int64(2)).n_groups == 2
    plan = mtk.route_rows(idx, 2)
    with pytest.raises(ValueError, match="weights"):
        mtk.combine_rows(torch.ones(1, 3, device=DEV), plan, torch.tensor(1.0, device=DEV))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,k,E,D", [(0, 2, 3, 5), (1, 1, 1, 1), (3, 8, 2, 2), (33, 2, 5, 7), (100, 4, 9, 33), (257, 3, 16, 120), (1000, 2, 7, 257), (70, 5, 1000, 1021), (50, 2, 4, 2050)])
def test_rows_forth_and_back(N, k, E, D, dt):
    g = gen(N * 31 + D)
    idx = make_index(g, N, k, E, "any").reshape(N, k)
    x, y, w = randn(g, N, D, dt=dt), randn(g, N * k, D, dt=dt), randn(g, N, k)
    gx, go = randn(g, N * k, D, dt=dt), randn(g, N, D, dt=dt)
    for t in (x, y, w):
        t.requires_grad_()
    plan = mtk.route_rows(idx.to(DEV), E)
    xs, out = mtk.dispatch_rows(x, plan), mtk.combine_rows(y, plan, w)
    dx, dy, dw = torch.autograd.grad((xs, out), (x, y, w), (gx, go))
    order, slot, _ = route_reference(idx.numpy(), E)
    order, slot = torch.from_numpy(order), torch.from_numpy(slot)
    c = lambda t: t.detach().cpu()  # noqa: E731
    assert torch.equal(c(xs), c(x)[order // k])
    terms = c(y).double()[slot.reshape(-1)].view(N, k, D) * c(w).double()[:, :, None]
    want, mag = terms.sum(1), terms.abs().sum(1)
    within(out, want, (k + 2) * U32 * mag + half(dt) * want.abs() * 1.001 + tiny(dt))
    terms = c(gx).double()[slot.reshape(-1)].view(N, k, D)
    want, mag = terms.sum(1), terms.abs().sum(1)
    within(dx, want, (k + 2) * U32 * mag + half(dt) * want.abs() * 1.001 + tiny(dt))
    want = c(go).double()[order // k] * c(w).double().reshape(-1)[order][:, None]
    within(dy, want, (half(dt) + 2 * U32) * want.abs() * 1.001 + tiny(dt))
    terms = c(y).double()[slot.reshape(-1)].view(N, k, D) * c(go).double()[:, None, :]
    within(dw, terms.sum(2), (D + 2) * U32 * terms.abs().sum(2))
    again = torch.autograd.grad((mtk.dispatch_rows(x, plan), mtk.combine_rows(y, plan, w)), (x, y, w), (gx, go))
    assert all(torch.equal(a, b) for a, b in zip(again, (dx, dy, dw)))  # the same bits
    # without weights, and with a gradient for one side only
    want = c(y).double()[slot.reshape(-1)].view(N, k, D)
    within(mtk.combine_rows(y.detach(), plan), want.sum(1), (k + 2) * U32 * want.abs().sum(1) + half(dt) * want.sum(1).abs() * 1.001 + tiny(dt))
    assert torch.equal(torch.autograd.grad(mtk.combine_rows(y.detach(), plan, w), w, go)[0], dw)
    assert torch.equal(torch.autograd.grad(mtk.combine_rows(y, plan, w.detach()), y, go)[0], dy)


def test_rows_gradients_against_differences():
    """<gradient, direction> against the change of the loss along it: every map is linear in each argument, so the difference is exact but
    for rounding - the fp32 sums behind both sides, (D k + 4) 2^-24 of the sum of magnitudes, times 4 for the two losses and the product."""
    g = gen(5)
    N, k, E, D = 40, 3, 6, 29
    plan = mtk.route_rows(make_index(g, N, k, E, "any").to(DEV), E)
    x, y, w = randn(g, N, D), randn(g, N * k, D), randn(g, N, k)
    gx, go = randn(g, N * k, D), randn(g, N, D)
    f = {"x": (x, lambda t: (mtk.dispatch_rows(t, plan).double() * gx.double())), "y": (y, lambda t: mtk.combine_rows(t, plan, w).double() * go.double()),
         "w": (w, lambda t: mtk.combine_rows(y, plan, t).double() * go.double())}
    for name, (t, loss) in f.items():
        d = randn(g, *t.shape)
        leaf = t.clone().requires_grad_()
        grad = torch.autograd.grad(loss(leaf).sum(), leaf)[0]
        up, down = loss(t + d), loss(t - d)
        tol = 4 * (D * k + 4) * U32 * float(up.abs().sum() + down.abs().sum() + (grad * d).abs().sum())
        assert abs(float((up.sum() - down.sum()) / 2 - (grad.double() * d.double()).sum())) <= tol, name


@pytest.mark.parametrize("dt", DTYPES)
def test_rows_keep_bad_values_to_themselves(dt):
    """An index out of range gives a NaN row and touches no other; infinities and NaN stay in their records."""
    g = gen(2)
    N, k, E, D = 50, 2, 4, 19
    idx = make_index(g, N, k, E, "bad")
    x = randn(g, N, D, dt=dt)
    x[7], x[9, 3] = float("nan"), float("inf")
    plan = mtk.route_rows(idx.to(DEV), E)
    xs = mtk.dispatch_rows(x, plan).cpu()
    order, slot, _ = route_reference(idx.numpy(), E)
    bad = torch.from_numpy(order < 0)
    assert int(bad.sum()) == 2 and bool(torch.isnan(xs[bad]).all())
    src = torch.from_numpy(np.where(order < 0, ~order, order)) // k
    assert torch.equal(torch.nan_to_num(xs[~bad].float()), torch.nan_to_num(x.cpu()[src[~bad]].float()))
    y = randn(g, N * k, D, dt=dt)
    clean = mtk.combine_rows(y, plan)
    lost = torch.zeros(N, dtype=torch.bool)  # a record with a pair out of range is NaN on the way back, and in its gradient, too
    lost[[N // 2, N - 1]] = True
    assert bool(torch.isnan(clean.cpu()[lost]).all()) and bool(torch.isfinite(clean.cpu()[~lost]).all())
    leaf = torch.zeros(N, D, dtype=dt, device=DEV, requires_grad=True)
    mtk.dispatch_rows(leaf, plan).backward(y)
    assert bool(torch.isnan(leaf.grad.cpu()[lost]).all()) and torch.equal(leaf.grad.cpu()[~lost], clean.cpu()[~lost])
    s = int(slot[11, 1])
    y[s] = float("nan")
    got = mtk.combine_rows(y, plan)
    assert bool(torch.isnan(got[11]).all())
    rest = (torch.arange(N) != 11) & ~lost
    assert torch.equal(got.cpu()[rest], clean.cpu()[rest])


def test_rows_past_the_caches():
    """A result larger than 256 MB is stored another way: the same values."""
    N, k, D = 70000, 2, 512
    x = torch.arange(N * D, device=DEV, dtype=torch.int32).remainder(8191).float().view(N, D)
    idx = torch.randint(-1, 7, (N, k), generator=gen(1)).to(DEV)
    plan = mtk.route_rows(idx, 7)
    xs = mtk.dispatch_rows(x, plan)
    assert xs.numel() * 4 > 256 << 20
    assert torch.equal(xs, x[plan.order.long() // k])
    big = torch.cat([xs, xs], 1)
    assert torch.equal(mtk.combine_rows(big, plan), torch.cat([2 * x, 2 * x], 1))


@pytest.mark.parametrize("dt,D", [(torch.float32, 509), (torch.bfloat16, 1021), (torch.float16, 8)])
def test_rows_past_the_caches_are_the_same_rows(dt, D):
    """Odd rows, weights and gradients of a call that goes past the caches, against the same records in two calls that do not"""
    size = torch.finfo(dt).bits // 8
    N, k = (400 << 20) // (3 * D * size), 2  # x and its two copies: 400 MB
    g = torch.Generator(device=DEV).manual_seed(3)
    x, y = (torch.randn(n, D, device=DEV, generator=g).to(dt) for n in (N, N * k))
    w = torch.randn(N, k, device=DEV, generator=g)
    idx = torch.randint(-1, 5, (N, k), device=DEV, generator=g)
    plan = mtk.route_rows(idx, 5)
    ys = y[plan.slot.long().view(-1)]  # a pair's row, in pair order
    leaves = [t.clone().requires_grad_() for t in (y, w)]
    out = mtk.combine_rows(leaves[0], plan, leaves[1])
    dy, dw = torch.autograd.grad(out, leaves, x)
    xs = mtk.dispatch_rows(x, plan)
    assert min(t.numel() * size for t in (xs, y)) + x.numel() * size > 256 << 20
    for part in (slice(0, N // 2), slice(N // 2, N)):
        p = mtk.route_rows(idx[part], 5)
        rows = ys.view(N, k, D)[part].reshape(-1, D)[p.order.long()].contiguous()
        small = [rows.requires_grad_(), w[part].clone().requires_grad_()]
        o = mtk.combine_rows(small[0], p, small[1])
        sy, sw = torch.autograd.grad(o, small, x[part])
        pairs = plan.slot[part].long().view(-1)
        assert torch.equal(o, out[part]) and torch.equal(sw, dw[part])
        assert torch.equal(sy[p.slot.long().view(-1)], dy[pairs])
        assert torch.equal(mtk.dispatch_rows(x[part], p)[p.slot.long().view(-1)], xs[pairs])


def test_rows_strides_and_shapes():
    g = gen(3)
    N, k, E, D = 40, 2, 5, 24
    idx = make_index(g, N, k, E, "any")
    plan = mtk.route_rows(idx.to(DEV), E)
    wide, yw = randn(g, N, 3 * D), randn(g, N * k, D + 3)
    for x in (wide[:, D:2 * D], wide[:, :D].t().contiguous().t(), wide[:1, :D].expand(N, D), wide[:, ::3], wide.flip(0)[:, 1:D + 1]):
        assert torch.equal(mtk.dispatch_rows(x, plan), mtk.dispatch_rows(x.contiguous(), plan))
    for y in (yw[:, 3:], yw[:, 1:2], yw[:, :D].t().contiguous().t(), yw[:1].expand(N * k, D + 3)):
        assert torch.equal(mtk.combine_rows(y, plan), mtk.combine_rows(y.contiguous(), plan))
    w = randn(g, k, N).t()
    assert torch.equal(mtk.combine_rows(yw, plan, w), mtk.combine_rows(yw, plan, w.contiguous()))
    x = wide.clone().requires_grad_()
    mtk.dispatch_rows(x, plan).sum().backward()  # an expanded gradient
    assert torch.equal(x.grad, torch.full_like(x, float(k)))
    for bad in (wide[:N - 1], wide.double(), wide[:, :0], wide[0]):
        with pytest.raises(ValueError):
            mtk.dispatch_rows(bad, plan)
    for bad in (w.double(), w[:, :1], w.reshape(-1), w.half()):
        with pytest.raises(ValueError):
            mtk.combine_rows(yw, plan, bad)


# ---------------------------------------------------------------------------------------------------------------- adapters
def make_offsets(g, M, E, kind):
    if kind == "base":  # no row has a model
        return torch.zeros(E + 1, dtype=torch.int32)
    if kind == "last":  # the last model owns everything
        return torch.tensor([0] * E + [M], dtype=torch.int32)
    idx = torch.randint(0, E + 1, (M,), generator=g)
    if kind == "few":
        idx = torch.where(idx == E, idx, idx // max(1, E // 3) * max(1, E // 3))
    return torch.searchsorted(idx.sort().values, torch.arange(E + 1)).to(torch.int32)


def adapter_inputs(g, M, din, dout, r, E, dt, kind="any"):
    return dict(x=randn(g, M, din, dt=dt), weight=(randn(g, dout, din) / math.sqrt(din)).to(dt), bias=randn(g, dout, dt=dt), down=(randn(g, E, r, din) / math.sqrt(din)).to(dt),
                up=(randn(g, E, dout, r) / math.sqrt(r)).to(dt), offsets=make_offsets(g, M, E, kind).to(DEV), scale=(torch.rand(E, generator=g) + 0.5).to(DEV))


def call(a, **kw):
    a = {**a, **kw}
    return mtk.adapter_linear(a["x"], a["weight"], a["bias"], a["down"], a["up"], a["offsets"], a["scale"], kw.get("activation", "none"))


def inner(dt):
    """The low-rank rows between their two products: a 16-bit type keeps them as hi + lo, and lo, at most half a step of the value, is rounded to
    half a step of its own."""
    return 0.0 if dt == torch.float32 else half(dt) ** 2 * 1.05


def tol(terms, low, K, r, want, dt, factor):
    """Sums of K products over `terms`; the low-rank part sums K, then r, with its inner value rounded (by half the smallest step at least, times
    the second factor).  The stored value rounds once more."""
    return (TWICE * (K + 2) * U32 * terms + (TWICE * (K + r + 8) * U32 + inner(dt)) * low + tiny(dt) * r * float(factor.detach().abs().max()) * 1.5
            + half(dt) * want.abs() * 1.01 + tiny(dt) * 4)


def tol_factor(mag, K, rows, want, dt, other):
    """A factor's gradient: sums over K features, then over a model's rows."""
    return (TWICE * (K + rows + 8) * U32 + inner(dt)) * mag + tiny(dt) * rows * float(other.detach().abs().max()) * 1.5 + half(dt) * want.abs() * 1.01 + tiny(dt) * 4


SHAPES = [(1, 1, 1, 1, 1, "any"), (1, 64, 64, 8, 4, "any"), (2, 7, 5, 3, 2, "any"), (31, 130, 67, 12, 5, "any"), (33, 64, 128, 16, 3, "last"), (64, 33, 130, 17, 64, "any"),
          (127, 257, 129, 33, 7, "few"), (130, 96, 200, 64, 4, "any"), (300, 70, 66, 100, 2, "any"), (700, 128, 192, 40, 2, "last"), (1100, 100, 130, 70, 3, "any"), (129, 40, 24, 256, 3, "any"), (513, 128, 256, 8, 1, "any"),
          (200, 120, 128, 4, 1024, "few"), (1000, 512, 48, 16, 16, "any"), (77, 64, 64, 8, 3, "base"), (2049, 64, 72, 16, 9, "few"), (16, 2050, 40, 8, 4, "any"),
          (700, 256, 1024, 16, 5, "any"), (9, 300, 1000, 9, 3, "any"), (300, 1030, 1030, 5, 9, "any"), (65, 40, 4100, 6, 7, "any"), (1, 1030, 40, 32, 3, "any"), (4, 513, 33, 8, 70, "any"), (16, 40, 50, 2, 3, "any"), (3, 20, 9, 10, 2, "base")]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,din,dout,r,E,kind", SHAPES)
def test_adapter_forward_and_gradients(M, din, dout, r, E, kind, dt):
    g = gen(M * 13 + din)
    a = adapter_inputs(g, M, din, dout, r, E, dt, kind)
    gy = randn(g, M, dout, dt=dt)
    for n in ("x", "down", "up"):
        a[n].requires_grad_()
    y = call(a)
    ref = adapter_reference(**{**a, "relu": False, "gy": gy})
    dx, ddown, dup = torch.autograd.grad(y, (a["x"], a["down"], a["up"]), gy)
    within(y, ref["y"], tol(ref["y_terms"], ref["y_low"], din, r, ref["y"], dt, a["up"]))
    within(dx, ref["dx"], tol(ref["dx_terms"], ref["dx_low"], dout, r, ref["dx"], dt, a["down"]))
    rows = int((a["offsets"][1:] - a["offsets"][:-1]).max())
    for name, got, K, other in (("ddown", ddown, dout, a["x"]), ("dup", dup, din, gy)):
        within(got, ref[name], tol_factor(ref[name + "_terms"], K, rows, ref[name], dt, other))
    # the same bits again, and alone
    y2 = call(a)
    assert torch.equal(y, y2)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y2, (a["x"], a["down"], a["up"]), gy), (dx, ddown, dup)))
    for i, n in enumerate(("x", "down", "up")):
        b = {**a, **{m: a[m].detach() for m in ("x", "down", "up") if m != n}}
        assert torch.equal(torch.autograd.grad(call(b), b[n], gy)[0], (dx, ddown, dup)[i]), n
    # without gradients the layer is the same, and so it is without a bias
    b = {n: t.detach() for n, t in a.items()}
    assert torch.equal(call(b), y)
    ref0 = adapter_reference(**{**b, "bias": None, "relu": True})
    within(call(b, bias=None, activation="relu"), ref0["y"], tol(ref0["y_terms"], ref0["y_low"], din, r, ref0["y"], dt, b["up"]))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,din,dout,r,E", [(1, 16, 8, 2, 1), (100, 33, 65, 8, 3), (300, 128, 128, 16, 4)])
def test_adapter_relu_gradient(M, din, dout, r, E, dt):
    """The mask: rows of x are scaled so that the layer's values stay clear of 0 by more than their tolerance; where one would not, its dy is 0
    (which adds nothing on either side)."""
    g = gen(M + din)
    a = adapter_inputs(g, M, din, dout, r, E, dt)
    gy = randn(g, M, dout, dt=dt)
    pre = adapter_reference(**{**a, "relu": False})
    near = pre["y"].abs() <= tol(pre["y_terms"], pre["y_low"], din, r, pre["y"], dt, a["up"])
    gy[near.to(DEV)] = 0
    for n in ("x", "down", "up"):
        a[n].requires_grad_()
    ref = adapter_reference(**{**a, "relu": True, "gy": gy})
    y = call(a, activation="relu")
    within(y, ref["y"], tol(pre["y_terms"], pre["y_low"], din, r, pre["y"], dt, a["up"]))
    dx, ddown, dup = torch.autograd.grad(y, (a["x"], a["down"], a["up"]), gy)
    within(dx, ref["dx"], tol(ref["dx_terms"], ref["dx_low"], dout, r, ref["dx"], dt, a["down"]))
    for name, got, K, other in (("ddown", ddown, dout, a["x"]), ("dup", dup, din, gy)):
        within(got, ref[name], tol_factor(ref[name + "_terms"], K, M, ref[name], dt, other))


def test_adapter_gradients_against_differences():
    """The layer is linear in x, down and up each, so a central difference is exact but for rounding: half of each loss's error bound
    (the forward tolerance times |gy|, summed), twice, and the gradients' own."""
    g = gen(8)
    M, din, dout, r, E = 90, 48, 40, 8, 4
    a = adapter_inputs(g, M, din, dout, r, E, torch.float32)
    gy = randn(g, M, dout)
    for n in ("x", "down", "up"):
        leaf = a[n].clone().requires_grad_()
        d = randn(g, *leaf.shape) * 0.3
        grad = torch.autograd.grad(call(a, **{n: leaf}), leaf, gy)[0]
        loss, err = [], 0.0
        for sign in (1, -1):
            b = {**a, n: a[n] + sign * d}
            ref = adapter_reference(**{**b, "relu": False})
            err += float((tol(ref["y_terms"], ref["y_low"], din, r, ref["y"], torch.float32, b["up"]) * gy.cpu().double().abs()).sum()) + 4 * U32 * float(
                ((ref["y_terms"] + ref["y_low"]) * gy.cpu().double().abs()).sum())  # a +- d is rounded too
            loss.append(float((call(b).double() * gy.double()).sum()))
        own = TWICE * (din + dout + M + r + 16) * U32 * float((grad.double().abs() * d.double().abs()).sum()) * 8
        assert abs((loss[0] - loss[1]) / 2 - float((grad.double() * d.double()).sum())) <= err + own, n


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M", [3, 200])
def test_a_diverged_model_leaves_the_others_alone(M, dt):
    """Infinite and NaN factors, rows and gradients of one model: every other model's rows and gradients keep their bits."""
    g = gen(17)
    din, dout, r, E = 72, 80, 8, 3
    a = adapter_inputs(g, M, din, dout, r, E, dt)
    a["offsets"] = torch.tensor([0, M // 3, 2 * M // 3, M], dtype=torch.int32, device=DEV)
    gy = randn(g, M, dout, dt=dt)

    def run(b, gy):
        b = {n: t.clone() for n, t in b.items()}
        for n in ("x", "down", "up"):
            b[n].requires_grad_()
        y = call(b)
        return (y.detach(),) + torch.autograd.grad(y, (b["x"], b["down"], b["up"]), gy)

    clean = run(a, gy)
    rows = slice(M // 3, 2 * M // 3)
    rest = torch.ones(M, dtype=torch.bool)
    rest[rows] = False
    for what in ("down", "up", "x", "gy"):
        for value in (float("inf"), float("nan")):
            b, gz = {n: t.clone() for n, t in a.items()}, gy.clone()
            if what == "gy":
                gz[rows] = value
            elif what == "x":
                b["x"][rows] = value
            else:
                b[what][1] = value
            y, dx, dd, du = run(b, gz)
            assert torch.equal(y.cpu()[rest], clean[0].cpu()[rest]) and torch.equal(dx.cpu()[rest], clean[1].cpu()[rest]), (what, value)
            for got, want in ((dd, clean[2]), (du, clean[3])):
                assert torch.equal(got[[0, 2]], want[[0, 2]]), (what, value)
            if what != "gy":
                assert not bool(torch.isfinite(y[rows]).any()), what


def shared_offsets(M, E, tile, apart=0):
    """Offsets whose borders fall inside tiles: no model has the first `apart` rows nor the last, two models have no rows, one has a single
    row, and the borders of three lie in one tile"""
    off = [apart + (M - 2 * apart) * e // E for e in range(E + 1)]
    off[2] = off[1]
    off[E - 1] = off[E]
    off[4], off[5] = off[3] + 1, off[3] + tile // 4
    return torch.tensor(off, dtype=torch.int32, device=DEV)


# rows, widths: each tile of the product (64, 128, 256 rows) with whole and with ragged feature tiles, both products of a step alike
SHARED = [(1500, 72, 80, 7, 64), (33 * 128 + 5, 1030, 1030, 7, 128), (52 * 256 + 77, 1000, 1000, 9, 256)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,din,dout,E,tile", SHARED)
def test_tiles_that_models_share(M, din, dout, E, tile, dt):
    g = gen(M)
    a = adapter_inputs(g, M, din, dout, 12, E, dt)
    a["offsets"] = shared_offsets(M, E, tile, 37)
    gy = randn(g, M, dout, dt=dt)
    for n in ("x", "down", "up"):
        a[n].requires_grad_()
    y = call(a)
    dx, dd, du = torch.autograd.grad(y, (a["x"], a["down"], a["up"]), gy)
    ref = adapter_reference(**{**a, "relu": False, "gy": gy})
    within(y, ref["y"], tol(ref["y_terms"], ref["y_low"], din, 12, ref["y"], dt, a["up"]))
    within(dx, ref["dx"], tol(ref["dx_terms"], ref["dx_low"], dout, 12, ref["dx"], dt, a["down"]))
    # a row is the same whatever the other models' factors hold: finite ones ..
    b = {n: t.detach().clone() for n, t in a.items()}
    off = a["offsets"].tolist()
    rest = torch.ones(M, dtype=torch.bool)
    for e in (0, 5):
        rest[off[e]:off[e + 1]] = False
    with torch.no_grad():
        for value in (2.0, float("inf"), float("nan")):
            for n, t in (("up", b["up"]), ("down", b["down"])):
                keep = t.clone()
                t[0, 0, 0], t[5] = value, value
                again = call(b)
                assert torch.equal(again.cpu()[rest], y.detach().cpu()[rest]), (n, value)
                if value != 2.0 and n == "up":
                    assert not bool(torch.isfinite(again[off[5]:off[6]]).any()) and not bool(torch.isfinite(again[off[0]:off[1], 0]).any())
                    assert torch.equal(again[off[0]:off[1], 1:], y.detach()[off[0]:off[1], 1:])  # what the value does not reach
                t.copy_(keep)
    for value in (float("inf"), float("nan")):  # .. and so its gradient
        c = {n: t.detach().clone() for n, t in a.items()}
        c["down"][5] = value
        c["x"].requires_grad_()
        again = torch.autograd.grad(call(c), c["x"], gy)[0]
        mine = torch.zeros(M, dtype=torch.bool)
        mine[off[5]:off[6]] = True
        assert torch.equal(again.cpu()[~mine], dx.cpu()[~mine]) and not bool(torch.isfinite(again.cpu()[mine]).any()), value


@pytest.mark.parametrize("M,din,dout,dt", [(1500, 72, 80, torch.bfloat16), (33 * 128 + 5, 1030, 1030, torch.float16), (700, 64, 96, torch.float32)])
def test_a_captured_layer_follows_its_offsets(M, din, dout, dt):
    """The models' borders are on the device: a replay takes those that its offsets hold, and what the last replay left in the workspace (rows of
    tiles that other models shared, a model that diverged) is not seen"""
    g = gen(M + 1)
    E = 7
    a = adapter_inputs(g, M, din, dout, 12, E, dt)
    gy = randn(g, M, dout, dt=dt)
    borders = [shared_offsets(M, E, 64), torch.tensor([0] * E + [M], dtype=torch.int32, device=DEV), shared_offsets(M, E, 128, 19), torch.zeros(E + 1, dtype=torch.int32, device=DEV),
               shared_offsets(M, E, 32, 5)]
    for n in ("x", "down", "up"):
        a[n].requires_grad_()
    off = borders[0].clone()

    def work():
        y = call(a, offsets=off)
        return (y.detach(),) + torch.autograd.grad(y, (a["x"], a["down"], a["up"]), gy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    finite = a["up"].detach().clone()
    for turn, border in enumerate(borders + borders):
        off.copy_(border)
        with torch.no_grad():
            a["up"].copy_(finite)
            if turn == 4:
                a["up"][5] = float("nan")
        want = work()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(got, want):
            assert torch.equal(torch.nan_to_num(p.float(), nan=7e4), torch.nan_to_num(q.float(), nan=7e4)), turn


@pytest.mark.parametrize("dt", DTYPES)
def test_more_models_in_a_tile_than_it_streams(dt):
    """Twelve models inside one tile of 64 rows beside eight long ones, and two dozen of three rows each"""
    g = gen(31)
    M, din, dout, r = 1600, 72, 80, 5
    for off in ([0, 200, 400, 600, 800] + [801 + 3 * i for i in range(12)] + [1000, 1200, 1400, 1600], [0, 1390] + [1390 + 3 * i for i in range(1, 24)] + [1590]):
        E = len(off) - 1
        a = adapter_inputs(g, M, din, dout, r, E, dt)
        a["offsets"] = torch.tensor(off, dtype=torch.int32, device=DEV)
        gy = randn(g, M, dout, dt=dt)
        a["x"].requires_grad_()
        y = call(a)
        dx = torch.autograd.grad(y, a["x"], gy)[0]
        ref = adapter_reference(**{**a, "relu": False, "gy": gy})
        within(y, ref["y"], tol(ref["y_terms"], ref["y_low"], din, r, ref["y"], dt, a["up"]))
        within(dx, ref["dx"], tol(ref["dx_terms"], ref["dx_low"], dout, r, ref["dx"], dt, a["down"]))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("r", [4, 8, 5])
def test_a_layer_of_one_feature_with_many_models(r, dt):
    """Fewer rows a model than a tile has, and factors of one piece: the last model's is the end of its tensor"""
    g = gen(r)
    M, din, E = 1000, 40, 32
    a = adapter_inputs(g, M, din, 1, r, E, dt)
    gy = randn(g, M, 1, dt=dt)
    for n in ("x", "down", "up"):
        a[n].requires_grad_()
    y = call(a)
    ref = adapter_reference(**{**a, "relu": False, "gy": gy})
    dx, ddown, dup = torch.autograd.grad(y, (a["x"], a["down"], a["up"]), gy)
    within(y, ref["y"], tol(ref["y_terms"], ref["y_low"], din, r, ref["y"], dt, a["up"]))
    within(dx, ref["dx"], tol(ref["dx_terms"], ref["dx_low"], 1, r, ref["dx"], dt, a["down"]))
    rows = int((a["offsets"][1:] - a["offsets"][:-1]).max())
    within(ddown, ref["ddown"], tol_factor(ref["ddown_terms"], 1, rows, ref["ddown"], dt, a["x"]))
    within(dup, ref["dup"], tol_factor(ref["dup_terms"], din, rows, ref["dup"], dt, gy))


def test_adapter_strides_scales_and_plans():
    g = gen(4)
    M, din, dout, r, E = 60, 40, 24, 4, 3
    a = adapter_inputs(g, M, din, dout, r, E, torch.float32)
    wide = randn(g, M, 2 * din + 3)
    for x in (wide[:, 3:3 + din], wide[:, ::2][:, :din], wide[:1, :din].expand(M, din), randn(g, din, M).t()):
        assert torch.equal(call(a, x=x), call(a, x=x.contiguous()))
    b = {**a, "weight": a["weight"].t().contiguous().t(), "up": a["up"].transpose(1, 2).contiguous().transpose(1, 2)}
    assert torch.equal(call(b), call(a))
    assert torch.equal(call(a, scale=2.5), call(a, scale=torch.full((E,), 2.5, device=DEV)))
    idx = torch.randint(-1, E, (M,), generator=g).to(DEV)
    plan = mtk.route_rows(idx, E)
    assert torch.equal(mtk.adapter_linear(a["x"], a["weight"], a["bias"], a["down"], a["up"], plan), call(a, offsets=plan.offsets, scale=1.0))
    x = wide[:, :din].clone().requires_grad_()
    call(a, x=x).sum().backward()  # an expanded gradient
    y = a["x"].clone().requires_grad_()
    xe = wide[:1, :din].clone().requires_grad_()
    call(a, x=xe.expand(M, din)).sum().backward()  # a broadcast input: its gradient is the rows' sum
    full = wide[:1, :din].expand(M, din).clone().requires_grad_()
    call(a, x=full).sum().backward()
    assert torch.equal(xe.grad, full.grad.sum(0, keepdim=True)) and y.grad is None


def test_adapter_without_rows():
    g = gen(6)
    a = adapter_inputs(g, 0, 8, 6, 2, 3, torch.float32)
    for n in ("x", "down", "up"):
        a[n].requires_grad_()
    y = call(a)
    assert y.shape == (0, 6)
    dx, dd, du = torch.autograd.grad(y, (a["x"], a["down"], a["up"]), torch.zeros(0, 6, device=DEV))
    assert dx.shape == (0, 8) and not bool(dd.any()) and not bool(du.any())


def test_adapter_refusals():
    g = gen(7)
    a = adapter_inputs(g, 6, 8, 6, 2, 3, torch.float32)
    bad = [dict(x=a["x"][0]), dict(x=a["x"][:, :7]), dict(weight=a["weight"].half()), dict(up=a["up"][:2]), dict(bias=a["bias"][:5]), dict(offsets=a["offsets"].long()),
           dict(offsets=a["offsets"][:3]), dict(scale=torch.ones(2, device=DEV)), dict(scale=torch.ones(3)), dict(activation="gelu"), dict(x=a["x"].double()),
           dict(weight=a["weight"].cpu()), dict(down=a["down"][:, :0], up=a["up"][:, :, :0])]
    for kw in bad:
        with pytest.raises(ValueError):
            call(a, **kw)
    with pytest.raises(NotImplementedError, match="frozen"):
        call(a, weight=a["weight"].clone().requires_grad_())


# a row, few rows in both tiles, each tile of the product as one run of lines and (many models) apart from it; ranks of a line and of several
HALVES = [(1, 72, 40, 8, 1), (2, 40, 72, 20, 2), (61, 130, 67, 12, 5), (300, 40, 72, 33, 4), (700, 72, 80, 12, 3), (700, 80, 72, 20, 40), (4229, 1030, 1030, 16, 7), (2048, 130, 1030, 64, 3),
          (16500, 1000, 131, 8, 40), (16384, 64, 1024, 100, 2)]


def strictly(mag, K, want):
    """Sums of K terms of magnitude `mag`, the low-rank rows off by 2^-22 of their own magnitude whatever that is, and the result's own rounding: of
    its magnitude, or half the smallest step."""
    return (TWICE * (K + 8) * U32 + 2.0**-22) * mag + half(torch.float16) * want.abs() * 1.01 + 2.0**-25 * 1.01


@pytest.mark.parametrize("M,din,dout,r,E", HALVES)
def test_half_precision_keeps_small_low_rank_values(M, din, dout, r, E):
    """Gradients of 1e-3 against factors that have just left zero: t = s g B_e is far below fp16's normal numbers (and u in the forward direction),
    the results are not.  The shared weights are zero, or they would drown the low-rank part."""
    g = gen(M + r)
    dt = torch.float16
    a = adapter_inputs(g, M, din, dout, r, E, dt)
    a["weight"].zero_(), a["bias"].zero_()
    rows = int((a["offsets"][1:] - a["offsets"][:-1]).max())

    def run(gy):
        leaves = {n: a[n].detach().clone().requires_grad_() for n in ("x", "down", "up")}
        y = call(a, **leaves)
        grads = torch.autograd.grad(y, list(leaves.values()), gy)
        return y, grads, adapter_reference(**{**a, "relu": False, "gy": gy})

    a["up"] = randn(g, E, dout, r, dt=dt) * 2e-4
    a["down"] = randn(g, E, r, din, dt=dt) * 16
    gy = randn(g, M, dout, dt=dt) * 1e-3
    _, (dx, ddown, _), ref = run(gy)
    assert float((a["scale"].max() * (gy.double() @ a["up"][0].double())).abs().max()) < 2.0**-12
    within(dx, ref["dx"], strictly(ref["dx_low"], dout + r, ref["dx"]))
    within(ddown, ref["ddown"], strictly(ref["ddown_terms"], dout + rows, ref["ddown"]))
    a["x"] = randn(g, M, din, dt=dt) * 1e-3
    a["down"] = randn(g, E, r, din, dt=dt) * 2e-4
    a["up"] = randn(g, E, dout, r, dt=dt) * 64
    y, (_, _, dup), ref = run(randn(g, M, dout, dt=dt) * 64)
    within(y, ref["y"], strictly(ref["y_low"], din + r, ref["y"]))
    within(dup, ref["dup"], strictly(ref["dup_terms"], din + rows, ref["dup"]))


@pytest.mark.parametrize("M,din,dout,r,E", HALVES)
def test_half_precision_keeps_large_low_rank_values(M, din, dout, r, E):
    """u beyond fp16's largest number where y, dx and the factors' gradients are well inside"""
    g = gen(M + r + 1)
    dt = torch.float16
    a = adapter_inputs(g, M, din, dout, r, E, dt)
    a["x"], a["down"] = randn(g, M, din, dt=dt) * 2048, randn(g, E, r, din, dt=dt) * 128
    a["up"], gy = randn(g, E, dout, r, dt=dt) * 2.0**-20, randn(g, M, dout, dt=dt) * 2.0**-12
    for n in ("x", "down", "up"):
        a[n].requires_grad_()
    a["weight"] *= 2.0**-9
    y = call(a)
    dx, ddown, dup = torch.autograd.grad(y, (a["x"], a["down"], a["up"]), gy)
    ref = adapter_reference(**{**a, "relu": False, "gy": gy})
    rows = int((a["offsets"][1:] - a["offsets"][:-1]).max())
    assert rows == 0 or float((a["x"].detach().double() @ a["down"][0].detach().double().t()).abs().max()) > 65504
    within(y, ref["y"], strictly(ref["y_terms"] + ref["y_low"], din + r, ref["y"]))
    within(dx, ref["dx"], strictly(ref["dx_terms"] + ref["dx_low"], dout + r, ref["dx"]))
    within(ddown, ref["ddown"], strictly(ref["ddown_terms"], dout + rows, ref["ddown"]))
    inside = ref["dup"].abs() < 65000
    assert bool(inside.any())
    within(torch.where(inside.to(DEV), dup, 0), torch.where(inside, ref["dup"], 0), strictly(ref["dup_terms"], din + rows, torch.where(inside, ref["dup"], 0)))


def test_a_scale_that_requires_grad_is_refused():
    """It would get none: refused whether or not anything else of the layer is trained"""
    g = gen(93)
    a = adapter_inputs(g, 30, 8, 6, 2, 3, torch.float32)
    want = call(a)
    scale = a["scale"].clone().requires_grad_()
    for kw in ({}, {n: a[n].clone().requires_grad_() for n in ("x", "down", "up")}, {"x": a["x"].t().contiguous().t()}):
        with pytest.raises(NotImplementedError, match="scale"):
            call(a, scale=scale, **kw)
    with torch.no_grad():
        assert torch.equal(call(a, scale=scale), want)
    x = a["x"].clone().requires_grad_()
    y = call(a, scale=scale.detach(), x=x)
    assert torch.equal(y, want) and torch.equal(torch.autograd.grad(y.sum(), x)[0], torch.autograd.grad(call(a, x=x).sum(), x)[0])


@pytest.mark.parametrize("off", [[0, 90, 10, 40], [50, 60, 70, 80], [-5, 20, 1000, 2000], [100, 60, 30, 0], [-9, -8, -7, -6], [2**31 - 1] * 4])
@pytest.mark.parametrize("M", [64, 700])
def test_offsets_that_make_no_sense_stay_inside_the_tensors(M, off):
    """Offsets live on the device, so the host cannot check them: whatever they hold, no row outside the tensors is touched and the call ends.
    Rows before the first offset have the shared layer alone."""
    g = gen(12)
    din, dout, r, E = 32, 48, 4, 3
    a = adapter_inputs(g, M, din, dout, r, E, torch.float32)
    a["offsets"] = torch.tensor(off, dtype=torch.int32, device=DEV)
    for n in ("x", "down", "up"):
        a[n].requires_grad_()
    y = call(a)
    y.sum().backward()
    assert bool(torch.isfinite(y).all())
    if off == [50, 60, 70, 80]:
        fine = a["offsets"].cpu().clamp(max=M)
        ref = adapter_reference(**{**a, "offsets": fine, "relu": False})
        within(y, ref["y"], tol(ref["y_terms"], ref["y_low"], din, r, ref["y"], torch.float32, a["up"]))


@pytest.mark.parametrize("off", [[0, 3000, 10, 40], [3, 2, 1, 0], [-5, 20, 5000, 9000], [4229, 60, 30, 0], [2**31 - 1] * 4])
@pytest.mark.parametrize("M,r,dt", [(4, 4, torch.bfloat16), (13, 2, torch.float32), (4229, 12, torch.float16)])
def test_such_offsets_in_the_fused_call_and_the_larger_tiles(M, r, dt, off):
    g = gen(M)
    wide = 1030 if M > 512 else 40
    a = adapter_inputs(g, M, wide, wide, r, 3, dt)
    a["offsets"] = torch.tensor(off, dtype=torch.int32, device=DEV)
    a["x"].requires_grad_()
    y = call(a)
    dx = torch.autograd.grad(y, a["x"], torch.ones_like(y))[0]
    assert bool(torch.isfinite(y).all()) and bool(torch.isfinite(dx).all())


def test_operators_in_inference_mode():
    g = gen(2)
    a = adapter_inputs(g, 33, 40, 24, 4, 3, torch.float32)
    idx = torch.randint(-1, 3, (33, 2), generator=g).to(DEV)
    want = mtk.route_rows(idx, 3)
    w = torch.rand(33, 2, generator=g).to(DEV)
    base = mtk.combine_rows(mtk.adapter_linear(mtk.dispatch_rows(a["x"], want), a["weight"], a["bias"], a["down"], a["up"], want), want, w)
    with torch.inference_mode():
        plan = mtk.route_rows(idx, 3)
        got = mtk.combine_rows(mtk.adapter_linear(mtk.dispatch_rows(a["x"], plan), a["weight"], a["bias"], a["down"], a["up"], plan), plan, w)
        assert torch.equal(got, base) and got.is_inference()
        p, q, m, v = (torch.ones(300, device=DEV) for _ in range(4))
        mtk.adamw_step([p], [q], [m], [v], 1, lr=0.1)
        assert not bool((p == 1).any())


# one shape for each tile of the products: 256 x 256 and 128 x 128 with 16 bits, 128 x 128 with fp32, both directions; 32 rows a wave in the shrink
BIG = [(16384, 64, 1024, 8, 3), (16384, 1024, 64, 20, 2), (20011, 131, 1000, 12, 33), (16500, 1000, 131, 33, 40), (16384, 96, 1024, 40, 70)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,din,dout,r,E", BIG)
def test_adapter_with_many_rows(M, din, dout, r, E, dt):
    g = gen(M + din + r)
    a = adapter_inputs(g, M, din, dout, r, E, dt)
    gy = randn(g, M, dout, dt=dt)
    for n in ("x", "down", "up"):
        a[n].requires_grad_()
    y = call(a)
    ref = adapter_reference(**{**a, "relu": False, "gy": gy})
    dx, ddown, dup = torch.autograd.grad(y, (a["x"], a["down"], a["up"]), gy)
    within(y, ref["y"], tol(ref["y_terms"], ref["y_low"], din, r, ref["y"], dt, a["up"]))
    within(dx, ref["dx"], tol(ref["dx_terms"], ref["dx_low"], dout, r, ref["dx"], dt, a["down"]))
    rows = int((a["offsets"][1:] - a["offsets"][:-1]).max())
    for name, got, K, other in (("ddown", ddown, dout, a["x"]), ("dup", dup, din, gy)):
        within(got, ref[name], tol_factor(ref[name + "_terms"], K, rows, ref[name], dt, other))
    y2 = call(a)
    assert torch.equal(y, y2)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y2, (a["x"], a["down"], a["up"]), gy), (dx, ddown, dup)))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M", [40, 700])
def test_adapter_operands_that_start_anywhere(M, dt):
    """Views at odd offsets, odd distances between rows, an expanded row: the values of aligned copies, bit for bit."""
    g = gen(M)
    din, dout, r, E = 128, 192, 8, 3
    a = adapter_inputs(g, M, din, dout, r, E, dt)
    gy = randn(g, M, dout, dt=dt)

    def moved(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)

    def run(b, gy):
        b = {n: t.detach() for n, t in b.items()}
        for n in ("x", "down", "up"):
            b[n].requires_grad_()
        y = call(b)
        return (y,) + torch.autograd.grad(y, (b["x"], b["down"], b["up"]), gy)

    want = run(a, gy)
    for names in (("x",), ("weight",), ("down", "up", "bias"), ("x", "weight", "down", "up", "bias")):
        assert all(torch.equal(p, q) for p, q in zip(run({**a, **{n: moved(a[n]) for n in names}}, gy), want)), names
    assert all(torch.equal(p, q) for p, q in zip(run(a, moved(gy)), want))
    wide = torch.empty(M, din + 1, dtype=dt, device=DEV)
    wide[:, 1:] = a["x"]
    assert all(torch.equal(p, q) for p, q in zip(run({**a, "x": wide[:, 1:]}, gy), want))
    row = a["x"][:1]
    assert torch.equal(call(a, x=row.expand(M, din)), call(a, x=row.expand(M, din).contiguous()))


def test_nodes_differentiate_once():
    g = gen(90)
    a = adapter_inputs(g, 20, 8, 6, 2, 3, torch.float32)
    plan = mtk.route_rows(torch.randint(0, 3, (10, 2), generator=g).to(DEV), 3)
    w = randn(g, 10, 2)
    for f, leaf in ((lambda t: call(a, x=t), randn(g, 20, 8)), (lambda t: mtk.dispatch_rows(t, plan), randn(g, 10, 5)), (lambda t: mtk.combine_rows(t, plan, w), randn(g, 20, 5))):
        leaf.requires_grad_()
        first = torch.autograd.grad((f(leaf) ** 2).sum(), leaf, create_graph=True)[0]
        with pytest.raises(RuntimeError, match="differentiates once only"):
            first.sum().backward()
        plain = torch.autograd.grad((f(leaf) ** 2).sum(), leaf)[0]
        assert torch.equal(plain, first.detach())


def test_forward_mode_is_refused():
    """A result without the tangent would be a wrong derivative: with and without requires_grad, for every differentiable argument and the frozen
    ones; in a dual level without tangents all is as ever."""
    g = gen(91)
    a = adapter_inputs(g, 20, 8, 6, 2, 3, torch.float32)
    plan = mtk.route_rows(torch.randint(0, 3, (10, 2), generator=g).to(DEV), 3)
    x, y, w = randn(g, 10, 5), randn(g, 20, 5), randn(g, 10, 2)
    want = (call(a), mtk.dispatch_rows(x, plan), mtk.combine_rows(y, plan, w))
    fw = torch.autograd.forward_ad
    with fw.dual_level():
        dual = lambda t, grad: fw.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t))  # noqa: E731
        for grad in (False, True):
            calls = [lambda n=n: call(a, **{n: dual(a[n], grad)}) for n in ("x", "weight", "bias", "down", "up", "scale")]
            calls += [lambda: mtk.dispatch_rows(dual(x, grad), plan), lambda: mtk.combine_rows(dual(y, grad), plan, w), lambda: mtk.combine_rows(y, plan, dual(w, grad))]
            calls += [lambda: call(a, x=dual(a["x"], grad)[:, :8].t().contiguous().t())]  # strides to copy
            for f in calls:
                with pytest.raises(NotImplementedError):
                    f()
        assert all(torch.equal(p, q) for p, q in zip((call(a), mtk.dispatch_rows(x, plan), mtk.combine_rows(y, plan, w)), want))


def test_batched_gradients_are_refused():
    g = gen(97)
    a = adapter_inputs(g, 20, 8, 6, 2, 3, torch.float32)
    plan = mtk.route_rows(torch.randint(0, 3, (10, 2), generator=g).to(DEV), 3)
    w = randn(g, 10, 2)
    for f, leaf in ((lambda t: call(a, x=t), randn(g, 20, 8)), (lambda t: mtk.dispatch_rows(t, plan), randn(g, 10, 5)), (lambda t: mtk.combine_rows(t, plan, w), randn(g, 20, 5))):
        leaf.requires_grad_()
        y = f(leaf)
        with pytest.raises(RuntimeError, match="batched|vmap"):
            torch.autograd.grad(y, leaf, torch.ones(3, *y.shape, device=DEV), is_grads_batched=True)
        y = f(leaf)
        assert torch.isfinite(torch.autograd.grad(y, leaf, torch.ones_like(y))[0]).all()


def test_torchs_errors_keep_their_type():
    """Out of memory is torch's exception, and so is what a saved-tensor hook raises"""
    g = gen(94)
    a = adapter_inputs(g, 4, 8, 8192, 2, 1, torch.float32)
    free, total = torch.cuda.mem_get_info()
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (64 << 20)) / total)
    try:
        with pytest.raises(torch.cuda.OutOfMemoryError):
            call(a, x=a["x"][:1].expand(1 << 20, 8))  # 32 GiB of results
        plan = mtk.route_rows(torch.zeros(1 << 21, dtype=torch.int64, device=DEV), 1)
        with pytest.raises(torch.cuda.OutOfMemoryError):
            mtk.dispatch_rows(a["up"].view(-1)[:4096].view(1, 4096).expand(1 << 21, 4096), plan)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)

    class Stop(Exception):
        pass

    def pack(t):
        raise Stop

    a["x"].requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        with pytest.raises(Stop):
            call(a)
    assert torch.isfinite(call(a)).all()


def test_functional_transforms_are_refused_by_name():
    """Whatever the library said last: the message is about this call"""
    g = gen(92)
    a = adapter_inputs(g, 20, 8, 6, 2, 3, torch.float32)
    plan = mtk.route_rows(torch.randint(0, 3, (10, 2), generator=g).to(DEV), 3)
    x, y = randn(g, 2, 10, 5), randn(g, 20, 5)
    with pytest.raises(AssertionError):  # the library refuses something else
        mtk.adamw_step([y], [y], [y.clone()], [y.clone()], 0, lr=1e-3)
    for f in (lambda: torch.vmap(lambda t: mtk.dispatch_rows(t, plan))(x), lambda: torch.vmap(lambda t: mtk.combine_rows(y, plan, t))(randn(g, 3, 10, 2)),
              lambda: torch.vmap(lambda t: call(a, scale=t))(torch.ones(4, 3, device=DEV)), lambda: torch.func.grad(lambda t: call(a, up=t).sum())(a["up"]),
              lambda: torch.func.jvp(lambda t: call(a, x=t), (a["x"],), (a["x"],)), lambda: torch.vmap(lambda t: mtk.route_rows(t, 3).slot)(torch.zeros(2, 4, dtype=torch.int64, device=DEV))):
        with pytest.raises(NotImplementedError, match="torch.func|forward-mode"):
            f()


# ------------------------------------------------------------------------------------------------------------------- AdamW
SIZES = [1, 2, 3, 5, 255, 256, 257, 1000, 1024, 4099]


def adamw_lists(g, sizes, dt, odd):
    """tensors of their own, or (odd) views that start anywhere in one buffer"""
    def cut(scale):
        if not odd:
            return [(randn(g, n) * scale).to(dt) for n in sizes]
        flat = (randn(g, sum(sizes) + len(sizes)) * scale).to(dt)
        at, out = 1, []
        for n in sizes:
            out.append(flat[at:at + n])
            at += n + 1
        return out
    return cut(0.1), cut(0.01)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("odd", [False, True])
def test_adamw_32_bit(dt, odd):
    """Six fp32 roundings lie between the moments and their 64-bit values, some sixteen between p and its own (the moments', a square root, two
    divisions, four products and sums); p rounds to its type at the end.  The reference continues from the step's own outputs."""
    g = gen(21)
    p, _ = adamw_lists(g, SIZES, dt, odd)
    m = [torch.zeros(n, device=DEV) for n in SIZES]
    v = [torch.zeros(n, device=DEV) for n in SIZES]
    lr, b1, b2, eps, wd = 3e-3, 0.9, 0.99, 1e-8, 0.05
    for t in range(1, 5):
        _, gr = adamw_lists(g, SIZES, dt, odd)
        P, M, V = ([q.cpu().double() for q in z] for z in (p, m, v))
        mtk.adamw_step(p, gr, m, v, t, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd)
        for i in range(len(SIZES)):
            G = gr[i].cpu().double()
            wm, wv = b1 * M[i] + (1 - b1) * G, b2 * V[i] + (1 - b2) * G * G
            within(m[i], wm, 6 * U32 * (M[i].abs() + G.abs()))
            within(v[i], wv, 6 * U32 * (V[i] + G * G) + 2.0**-140)
            upd = lr / (1 - b1**t) * wm / (torch.sqrt(wv) / math.sqrt(1 - b2**t) + eps)
            mag = lr / (1 - b1**t) * (M[i].abs() + G.abs()) / (torch.sqrt(wv) / math.sqrt(1 - b2**t) + eps)
            want = P[i] * (1 - lr * wd) - upd
            within(p[i], want, 4 * U32 * P[i].abs() + 16 * U32 * mag + half(dt) * (want.abs() + 1e-6) * 1.01 + tiny(dt))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("odd", [False, True])
def test_adamw_8_bit_codes(dt, odd):
    """Against the operator's own fp32 operations in numpy, step after step: codes and scales are equal.  The parameters' quotient goes by a
    reciprocal of one unit in the last place (2^-23) and a product: three half steps of the update more than an exact quotient, one half
    step on each side for the sum, and the type's own."""
    g = gen(22)
    p, _ = adamw_lists(g, SIZES, dt, odd)
    code = lambda n: torch.zeros(n, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)  # noqa: E731
    m, v = [code(n) for n in SIZES], [code(n) for n in SIZES]
    ms, vs = ([torch.ones(-(-n // 256), device=DEV) for n in SIZES] for _ in range(2))
    for t in range(1, 6):
        _, gr = adamw_lists(g, SIZES, dt, odd)
        for q in gr:
            q *= 10 ** (t - 3)
            q[::7] *= 1e-3
            q[3::11] = 0
        n = lambda z: [q.cpu().float().numpy() for q in z]  # noqa: E731
        P, M, V, MS, VS = n(p), n(m), n(v), n(ms), n(vs)
        mtk.adamw_step(p, gr, m, v, t, lr=1e-3, exp_avg_scales=ms, exp_avg_sq_scales=vs)
        for i in range(len(SIZES)):
            wp, wm, wms, wv, wvs = adamw8_reference(P[i], gr[i].cpu().float().numpy(), M[i], MS[i], V[i], VS[i], t)
            assert np.array_equal(ms[i].cpu().numpy(), wms.astype(np.float32)) and np.array_equal(vs[i].cpu().numpy(), wvs.astype(np.float32)), (t, i)
            assert np.array_equal(m[i].cpu().float().numpy(), wm.astype(np.float32)) and np.array_equal(v[i].cpu().float().numpy(), wv.astype(np.float32)), (t, i)
            want = torch.from_numpy(wp.astype(np.float64))
            upd = (want - torch.from_numpy(P[i]).double() * (1 - 1e-5)).abs()
            within(p[i], want, 4 * U32 * (upd + want.abs() + 1e-6) + half(dt) * 1.01 * want.abs() * (dt != torch.float32) + tiny(dt))


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_keeps_bad_gradients_to_themselves(bits):
    n = 700
    g = gen(9)
    p0, g0 = randn(g, n), randn(g, n)

    def run(grad):
        p = torch.nn.Parameter(p0.clone())
        opt = mtk.AdamW([p], lr=1e-2, state_bits=bits)
        for _ in range(3):
            p.grad = grad.clone()
            opt.step()
        return p.detach().cpu(), opt.state[p]["exp_avg"].float().cpu(), opt.state[p]["exp_avg_sq"].float().cpu()

    bad = g0.clone()
    bad[5], bad[300], bad[699] = float("nan"), float("inf"), -float("inf")
    keep = torch.ones(n, dtype=torch.bool)
    keep[[5, 300, 699]] = False
    zeroed = torch.where(keep.to(DEV), g0, torch.zeros_like(g0))
    a, b = run(bad), run(zeroed)
    for x, y in zip(a, b):
        assert torch.equal(x[keep], y[keep])
    assert bool(torch.isnan(a[0][~keep]).all())


def test_adamw_extremes():
    """Largest and smallest gradients: nothing overflows on the way that the formula does not overflow, and tiny averages keep a code."""
    for value in (1e-38, 1e-30, 1e-22, 1e18):
        for bits in (8, 32):
            p = torch.nn.Parameter(torch.ones(300, device=DEV))
            opt = mtk.AdamW([p], lr=1e-3, eps=0.0 if value > 1e-20 else 1e-8, weight_decay=0.0, state_bits=bits)
            for _ in range(4):
                p.grad = torch.full_like(p, value)
                opt.step()
            assert bool(torch.isfinite(p).all()), (value, bits)
            assert bool((p <= 1).all())


def test_adamw_refuses_tensors_that_share_memory():
    """Two of a launch's tensors in one place would be a race: the same one twice, or views that overlap, among all that is written; a gradient may be
    shared between parameters, or be its whole parameter."""
    z = lambda n=300: torch.ones(n, device=DEV)  # noqa: E731
    flat, m, g = z(1000), z(600), z()
    f8 = lambda: torch.zeros(300, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)  # noqa: E731
    ok = dict(params=[flat[:300], flat[300:600]], grads=[g, g], exp_avgs=[m[:300], m[300:]], exp_avg_sqs=[z(), z()])
    bad = [dict(exp_avgs=[m[:300]] * 2), dict(exp_avg_sqs=[m[100:400], z()]), dict(params=[flat[:300], flat[299:599]]), dict(exp_avgs=[flat[600:900], flat[700:]]),
           dict(grads=[flat[1:301], g]), dict(grads=[g, flat[:300]]), dict(grads=[g, m[:300]])]
    e8 = dict(params=ok["params"], grads=ok["grads"], exp_avgs=[f8(), f8()], exp_avg_sqs=[f8(), f8()], exp_avg_scales=[m[:2], m[2:4]], exp_avg_sq_scales=[m[4:6], m[6:8]])
    same = f8()
    bad8 = [dict(exp_avg_sq_scales=[m[1:3], m[6:8]]), dict(exp_avgs=[same, f8()], exp_avg_sqs=[f8(), same]), dict(exp_avg_scales=[flat[:2], m[2:4]])]
    for base, cases in ((ok, bad), (e8, bad8)):
        for kw in cases:
            before = [t.clone() for t in (flat, m)]
            with pytest.raises(ValueError, match="memory"):
                mtk.adamw_step(**{**base, **kw}, step=1, lr=1e-2)
            assert torch.equal(flat, before[0]) and torch.equal(m, before[1])
        mtk.adamw_step(**base, step=1, lr=1e-2)
        mtk.adamw_step(**{**base, "grads": [base["params"][0], g]}, step=2, lr=1e-2)
    p = torch.nn.Parameter(z())
    q = torch.nn.Parameter(z())
    p.grad = q.grad = torch.ones(300, device=DEV)
    mtk.AdamW([p, q]).step()
    assert torch.equal(p, q) and not bool((p == 1).any())


def test_adamw_where_a_squared_gradient_overflows():
    """The mean square is infinite, the quotient 0: parameters decay and no more, in both forms alike.  Gradients beside them go on as ever."""
    g = gen(35)
    n = 600
    grad = randn(g, n)
    far = torch.zeros(n, dtype=torch.bool)
    far[[0, 7, 300, 599]] = True
    grad[[0, 7, 300, 599]] = torch.tensor([1e20, -3e19, 2e38, 6e21], device=DEV)
    start, sides = randn(g, n), []
    for bits in (32, 8):
        p = torch.nn.Parameter(start.clone())
        opt = mtk.AdamW([p], lr=1e-2, weight_decay=0.5, state_bits=bits)
        p.grad = grad.clone()
        opt.step()
        sides.append(p.detach().cpu())
    decayed = start.cpu() * float(np.float32(1 - 1e-2 * 0.5))
    assert torch.equal(sides[0][far], decayed[far]) and torch.equal(sides[1][far], decayed[far])
    # elsewhere: the quotient by a reciprocal of one unit in its last place and a product, a root that may round the other way
    assert bool(((sides[0] - sides[1]).abs()[~far] <= 1e-2 * 8 * U32 + 2 * U32 * sides[0].abs()[~far]).all())


def test_adamw_roots_of_the_smallest_normal_numbers():
    """v = (1 - b2) g^2 from 2^-126 to 2^-118: the codes and scales of its root are those of the exact one"""
    b2 = 0.75  # (1 - b2) g^2 is exact for these g
    grad = torch.cat([torch.full((256,), 2.0 ** (k / 2) if k % 2 == 0 else 1.5 * 2.0 ** ((k - 1) // 2)) for k in range(-124, -115)]).to(DEV)
    n = grad.numel()
    code = lambda: torch.zeros(n, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)  # noqa: E731
    m, v = code(), code()
    ms, vs = (torch.ones(n // 256, device=DEV) for _ in range(2))
    p = torch.ones(n, device=DEV)
    z = np.zeros(n, np.float32)
    mtk.adamw_step([p], [grad], [m], [v], 1, lr=1e-3, betas=(0.9, b2), exp_avg_scales=[ms], exp_avg_sq_scales=[vs])
    _, wm, wms, wv, wvs = adamw8_reference(np.ones(n, np.float32), grad.cpu().numpy(), z, np.ones(n // 256), z, np.ones(n // 256), 1, b2=b2)
    assert np.array_equal(vs.cpu().numpy(), wvs.astype(np.float32)) and np.array_equal(v.cpu().float().numpy(), wv.astype(np.float32))
    assert np.array_equal(ms.cpu().numpy(), wms.astype(np.float32)) and np.array_equal(m.cpu().float().numpy(), wm.astype(np.float32))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dt", DTYPES)
def test_a_step_past_the_caches_is_the_same_step(dt, bits):
    """Tensors that together exceed what the caches hold take another way through memory; one by one they do not"""
    per = 3 * torch.finfo(dt).bits // 8 + (16 if bits == 32 else 4)
    n = (300 << 20) // per // 3
    g = torch.Generator(device=DEV).manual_seed(5)
    sides = []
    for odd in (0, 1, 3):  # a start inside a tensor: rows of 16 bytes begin anywhere
        p, q = (torch.randn(n + odd, device=DEV, generator=g).to(dt)[odd:] for _ in range(2))
        sides.append((p, q))
    assert sum(p.numel() for p, _ in sides) * per > 256 << 20
    blocks = -(-n // 256)

    def state():
        if bits == 8:
            return [torch.zeros(n, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2)] + [torch.ones(blocks, device=DEV) for _ in range(2)]
        return [torch.zeros(n, device=DEV) for _ in range(2)]

    def run(ps, qs, states, t):
        kw = dict(exp_avg_scales=[s[2] for s in states], exp_avg_sq_scales=[s[3] for s in states]) if bits == 8 else {}
        mtk.adamw_step(ps, qs, [s[0] for s in states], [s[1] for s in states], t, lr=1e-2, **kw)

    whole, single = ([(p.clone(), q, state()) for p, q in sides] for _ in range(2))
    for t in (1, 2):
        run(*zip(*whole), t)
        for one in single:
            run(*zip(one), t)
    for (p, _, s), (q, _, z) in zip(whole, single):
        assert torch.equal(p, q) and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(s, z))


def test_adamw_many_tensors_and_empty_ones():
    g = gen(30)
    sizes = [int(v) for v in torch.randint(0, 600, (200,), generator=g)] + [0, 0]
    ps = [torch.nn.Parameter(randn(g, n)) for n in sizes]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    ours, theirs = mtk.AdamW(ps, lr=1e-2, weight_decay=0.1), torch.optim.AdamW(qs, lr=1e-2, weight_decay=0.1, foreach=False)
    for _ in range(3):
        for p, q in zip(ps, qs):
            p.grad = randn(g, *p.shape)
            q.grad = p.grad.clone()
        ours.step()
        theirs.step()
    for p, q in zip(ps, qs):  # three steps of 1e-2, each off by some 16 half steps of fp32 at most, and p's own roundings
        assert torch.allclose(p, q, rtol=3 * 8 * U32, atol=3 * 1e-2 * 32 * U32)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_adamw_state_round_trip(bits, dt):
    """A saved and loaded state continues with the same bits, in the moments' own types."""
    g = gen(31)
    grads = [randn(g, 33, 17).to(dt) for _ in range(6)]
    p0 = randn(g, 33, 17).to(dt)

    def steps(p, opt, gs):
        for q in gs:
            p.grad = q.clone()
            opt.step()

    for capturable in (False, True):
        kw = dict(lr=1e-2, state_bits=bits, capturable=capturable)
        p = torch.nn.Parameter(p0.clone())
        opt = mtk.AdamW([p], **kw)
        steps(p, opt, grads)
        q = torch.nn.Parameter(p0.clone())
        first = mtk.AdamW([q], **kw)
        steps(q, first, grads[:3])
        second = mtk.AdamW([q], **kw)
        second.load_state_dict(first.state_dict())
        steps(q, second, grads[3:])
        assert torch.equal(p, q)
        for name in ("exp_avg", "exp_avg_sq"):
            a, b = opt.state[p][name], second.state[q][name]
            assert a.dtype == b.dtype == (torch.float8_e4m3fn if bits == 8 else torch.float32) and torch.equal(a.float(), b.float())
        assert int(second.state[q]["step"]) == 6


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("theirs", [dict(foreach=False), dict(capturable=True)])
def test_adamw_goes_on_from_torchs_state(theirs, dt):
    """A state that torch.optim.AdamW saved (its steps are float tensors, its moments of the parameters' type): the next step is that of the formula from
    those moments and that count, with a gradient for every parameter and for some."""
    g = gen(36)
    ps = [torch.nn.Parameter(randn(g, *shape).to(dt)) for shape in ((40, 3), (257,), (0,))]
    first = torch.optim.AdamW(ps, lr=1e-2, weight_decay=0.1, **theirs)
    for t in range(3):
        for i, p in enumerate(ps):
            p.grad = randn(g, *p.shape).to(dt) if i == 0 or t != 1 else None
        first.step()
    opt = mtk.AdamW(ps, lr=5.0)
    opt.load_state_dict(first.state_dict())
    assert opt.param_groups[0]["lr"] == 1e-2 and opt.param_groups[0]["state_bits"] == 32
    before = [p.detach().clone() for p in ps]
    moments = [[first.state[p][k].detach().double() for k in ("exp_avg", "exp_avg_sq")] for p in ps]
    grads = [randn(g, *p.shape).to(dt) for p in ps]
    for p, q in zip(ps, grads):
        p.grad = q.clone()
    opt.step()
    for p, p0, (m, v), q, t in zip(ps, before, moments, grads, (4, 3, 3)):
        st = opt.state[p]
        assert int(st["step"]) == t and st["exp_avg"].dtype == st["exp_avg_sq"].dtype == torch.float32
        q, p0 = q.double(), p0.double()
        wm, wv = 0.9 * m + 0.1 * q, 0.999 * v + 0.001 * q * q
        within(st["exp_avg"], wm.cpu(), (6 * U32 * (m.abs() + q.abs())).cpu())
        within(st["exp_avg_sq"], wv.cpu(), (6 * U32 * (v + q * q)).cpu() + 2.0**-140)
        den = torch.sqrt(wv) / math.sqrt(1 - 0.999**t) + 1e-8
        want = p0 * (1 - 1e-3) - 1e-2 / (1 - 0.9**t) * wm / den
        mag = 1e-2 / (1 - 0.9**t) * (m.abs() + q.abs()) / den
        within(p, want.cpu(), (4 * U32 * p0.abs() + 16 * U32 * mag + half(dt) * (want.abs() + 1e-6) * 1.01).cpu() + tiny(dt))
    assert (first.state[ps[0]]["exp_avg"].dtype == dt) and int(first.state[ps[0]]["step"]) == 3  # the other's state is its own
    bad = torch.optim.AdamW(ps, amsgrad=True)
    with pytest.raises(NotImplementedError, match="amsgrad"):
        opt.load_state_dict(bad.state_dict())
    assert opt.param_groups[0]["lr"] == 1e-2 and int(opt.state[ps[0]]["step"]) == 4  # as it was


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_counts_every_parameters_own_steps(bits):
    """Counts on the device are those on the host: parameters of two types, an empty one, some that go without a gradient now and then, from the
    first step on or later, more than a launch holds, and through a saved state.  The same bits."""
    g = gen(33)
    kinds = [(3 + i % 300, (torch.float32, torch.bfloat16, torch.float16)[i % 3]) for i in range(600)] + [(0, torch.float32), (40, torch.bfloat16)]
    start = [randn(g, n).to(dt) for n, dt in kinds]
    sides = []
    for capturable in (False, True):
        ps = [torch.nn.Parameter(t.clone()) for t in start]
        groups = [{"params": ps[:250]}, {"params": ps[250:], "weight_decay": 0.1}]
        sides.append([ps, mtk.AdamW(groups, lr=1e-2, state_bits=bits, capturable=capturable)])
    taken = [0] * len(kinds)
    for t in range(5):
        for i, (n, dt) in enumerate(kinds):
            grad = None if (i % 5 == 1 and t in (1, 2)) or (i % 7 == 3 and t == 0) or (i == 4 and t > 0) else randn(g, n).to(dt)
            taken[i] += grad is not None
            for ps, _ in sides:
                ps[i].grad = None if grad is None else grad.clone()
        for _, opt in sides:
            opt.step()
        if t == 2:  # go on from a saved state
            for side in sides:
                state = side[1].state_dict()
                side[1] = mtk.AdamW([{"params": side[0][:250]}, {"params": side[0][250:]}], capturable=side[1].defaults["capturable"])
                side[1].load_state_dict(state)
        for (p, q) in zip(*(ps for ps, _ in sides)):
            assert torch.equal(p, q), t
    for i, (p, q) in enumerate(zip(*(ps for ps, _ in sides))):
        a, b = (opt.state[w] for (_, opt), w in zip(sides, (p, q)))
        assert int(a["step"]) == int(b["step"]) == taken[i], i
        assert all(torch.equal(a[k].view(torch.uint8) if bits == 8 else a[k], b[k].view(torch.uint8) if bits == 8 else b[k]) for k in ("exp_avg", "exp_avg_sq"))


def test_one_count_on_the_device_for_all_tensors():
    """The C entries with a single count (mtk_adamw_count, then mtk_adamw_step with its numbers), over more tensors than a launch takes"""
    import ctypes as C

    from midst_toolkit_amd import _lib

    l, g = _lib.lib(), gen(37)
    sizes = [1 + 37 * i % 500 for i in range(70)]
    sizes[3] = sizes[69] = 0
    lists = [[randn(g, n) for n in sizes], None, [torch.zeros(n, device=DEV) for n in sizes], [torch.zeros(n, device=DEV) for n in sizes]]
    want = [[t.clone() for t in lists[i]] for i in (0, 2, 3)]
    step = torch.zeros((), dtype=torch.int64, device=DEV)
    hyper = torch.empty(l.mtk_adamw_hyper_bytes(), dtype=torch.uint8, device=DEV)
    numel = (C.c_int64 * len(sizes))(*sizes)
    stream = torch.cuda.current_stream().cuda_stream
    at = lambda ts: (C.c_void_p * len(ts))(*[t.data_ptr() for t in ts])  # noqa: E731
    for t in (1, 2, 3):
        lists[1] = [randn(g, n) for n in sizes]
        assert l.mtk_adamw_count(step.data_ptr(), None, 1e-2, 0.9, 0.99, 1e-8, 0.1, hyper.data_ptr(), stream) == 0
        assert l.mtk_adamw_step(len(sizes), *[at(ts) for ts in lists], None, None, numel, 0, 32, 0.0, 0.0, 0.0, 0.0, 0.0, 1, hyper.data_ptr(), stream) == 0
        mtk.adamw_step(want[0], lists[1], want[1], want[2], t, lr=1e-2, betas=(0.9, 0.99), weight_decay=0.1)
    assert int(step) == 3
    assert all(torch.equal(a, b) for got, ref in zip((lists[0], lists[2], lists[3]), want) for a, b in zip(got, ref))


def test_a_captured_step_counts_what_it_steps():
    """A graph that steps two of three parameters, of two types, with eager steps of all three in between"""
    g = gen(34)
    start = [randn(g, 300), randn(g, 300).bfloat16(), randn(g, 300)]
    sides = []
    for capturable in (False, True):
        ps = [torch.nn.Parameter(t.clone()) for t in start]
        sides.append((ps, mtk.AdamW(ps, lr=1e-2, capturable=capturable)))
    grads = [torch.zeros_like(t) for t in start]

    def step(ps, opt, which):
        for i, p in enumerate(ps):
            p.grad = grads[i] if i in which else None
        opt.step()

    def fill():
        for t in grads:
            t.copy_(randn(g, *t.shape))

    fill()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*sides[1], (0, 1, 2))
    torch.cuda.current_stream().wait_stream(side)
    step(*sides[0], (0, 1, 2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*sides[1], (0, 1))
    for t in range(5):
        fill()
        if t in (1, 2):
            for s in sides:
                step(*s, (1, 2))
        step(*sides[0], (0, 1))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(sides[0][0], sides[1][0])), t
    assert [int(sides[1][1].state[p]["step"]) for p in sides[1][0]] == [6, 8, 3]


def test_adamw_groups_closures_and_refusals():
    g = gen(32)
    a, b, c = (torch.nn.Parameter(randn(g, 4, 5)) for _ in range(3))
    frozen = c.detach().clone()
    opt = mtk.AdamW([{"params": [a], "lr": 1e-1, "state_bits": 8}, {"params": [b, c], "weight_decay": 0.0}], lr=1e-3)

    def closure():
        opt.zero_grad()
        loss = (a.sum() + (2 * b).sum()) ** 2
        loss.backward()
        return loss

    before = (a.detach().clone(), b.detach().clone())
    v = a._version
    loss = opt.step(closure)
    assert loss.requires_grad and a._version > v and torch.equal(c, frozen) and c not in opt.state
    # a first step is lr * sign(g) but for eps: within a thousandth
    assert torch.allclose((before[0] * (1 - 1e-1 * 1e-2) - a).abs(), torch.full_like(a, 1e-1), rtol=1e-3) and torch.allclose((before[1] - b).abs(), torch.full_like(b, 1e-3), rtol=1e-3)
    a.grad = torch.zeros(5, 4, device=DEV).t()  # a gradient of other strides is copied
    opt.step()
    t = torch.nn.Parameter(randn(g, 4, 5).t())
    t.grad = torch.ones_like(t)
    with pytest.raises(ValueError, match="not contiguous"):
        mtk.AdamW([t]).step()
    s = torch.nn.Parameter(randn(g, 4))
    s.grad = torch.ones(4, device=DEV).to_sparse()
    with pytest.raises(ValueError, match="sparse"):
        mtk.AdamW([s]).step()
    d = torch.nn.Parameter(randn(g, 4).double())
    d.grad = torch.ones_like(d)
    with pytest.raises(ValueError):
        mtk.AdamW([d]).step()
    x = [torch.zeros(4, device=DEV)]
    for bad in (dict(grads=[]), dict(grads=[torch.zeros(5, device=DEV)]), dict(grads=[torch.zeros(4, device=DEV).half()]), dict(exp_avgs=[torch.zeros(8, device=DEV)[::2]]),
                dict(exp_avg_scales=x), dict(exp_avg_sqs=[torch.zeros(4)]), dict(params=x * 2, grads=x * 2, exp_avgs=x * 2, exp_avg_sqs=x * 2)):
        kw = {**dict(params=x, grads=x, exp_avgs=x, exp_avg_sqs=x, step=1, lr=1e-3), **bad}
        with pytest.raises(ValueError):
            mtk.adamw_step(**kw)
    with pytest.raises(AssertionError):
        mtk.adamw_step(x, x, [torch.zeros(4, device=DEV)], [torch.zeros(4, device=DEV)], 0, lr=1e-3)


# --------------------------------------------------------------------------------------------------- streams, graphs, together
def test_operators_follow_the_current_stream():
    """Inputs written on a side stream behind a long product, the operators called there: the results are those of the default stream."""
    g = gen(40)
    M, din, dout, r, E = 256, 64, 64, 8, 4
    a = adapter_inputs(g, M, din, dout, r, E, torch.float32)
    idx = torch.randint(-1, E, (M, 2), generator=g).to(DEV)
    p0, g0 = randn(g, 1000), randn(g, 1000)

    def work():
        x = a["x"] * 2.0
        plan = mtk.route_rows(idx, E)
        h = mtk.combine_rows(mtk.dispatch_rows(call(a, x=x), plan), plan)
        p = p0.clone()
        mtk.adamw_step([p], [g0 * 2.0], [torch.zeros_like(p)], [torch.zeros_like(p)], 1, lr=1e-2)
        return h, p

    want = work()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    big = torch.randn(4096, 4096, device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(8):
            big = big @ big / 64
        got = work()
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def ensemble(g, D=24, layers=(64, 48), E=3, rank=4):
    torch.manual_seed(11)
    net = mtk.MLPDiffusion(D, 0, mtk.IsTargetConditioned.NONE, mtk.DiffusionParameters(list(layers), 0.0)).to(DEV)
    net.num_timesteps = 50
    for p in net.parameters():
        p.requires_grad_(False)
    ens = mtk.LowRankEnsemble(net, E, rank=rank, alpha=2 * rank)
    return net, ens


def ensemble_reference(net, ens, x, t, idx, w):
    """The ensemble in 64 bits, record by record's model: autograd's own graph on the CPU."""
    d = lambda q: q.detach().cpu().double()  # noqa: E731
    down = [d(p).requires_grad_() for p in ens.down]
    up = [d(p).requires_grad_() for p in ens.up]
    lin = [net.proj] + [b.linear for b in net.mlp.blocks] + [net.mlp.head]
    f = mtk.timestep_frequencies(net.timestep_dimension)
    arg = t.cpu().float()[:, None] * f[None]
    e = torch.cat([torch.cos(arg), torch.sin(arg)], 1).double()
    e = torch.nn.functional.silu(e @ d(net.timestep_embedding[0].weight).t() + d(net.timestep_embedding[0].bias))
    e = e @ d(net.timestep_embedding[2].weight).t() + d(net.timestep_embedding[2].bias)
    xd = d(x).requires_grad_()
    out = 0
    for j in range(idx.shape[1]):
        h = xd
        for i, m in enumerate(lin):
            m_idx = idx[:, j].cpu()
            on = (m_idx >= 0).double()[:, None] * ens.scale
            A, B = down[i][m_idx.clamp(min=0)], up[i][m_idx.clamp(min=0)]
            low = torch.bmm(torch.bmm(h[:, None], A.transpose(1, 2).contiguous()), B.transpose(1, 2).contiguous())[:, 0]
            h = h @ d(m.weight).t() + d(m.bias) + on * low
            if i == 0:
                h = h + e
            elif i < len(lin) - 1:
                h = torch.relu(h)
        out = out + w[:, j].cpu().double()[:, None] * h
    return out, xd, down, up


def close(got, want, rel=2e-4):
    """Chains of four layers in fp32: some 4 (K + 4) 2^-24 of the magnitudes, against their cancelled sums; 2e-4 of the largest."""
    got, want = got.detach().cpu().double(), want.detach()
    assert float((got - want).abs().max()) <= rel * float(want.abs().max()), float((got - want).abs().max() / want.abs().max())


def test_ensemble_starts_as_the_base_and_matches_64_bits():
    g = gen(50)
    net, ens = ensemble(g)
    N, D, E = 150, 24, 3
    x, t = randn(g, N, D), torch.randint(0, 50, (N,), generator=g).to(DEV)
    idx = torch.randint(-1, E, (N, 2), generator=g).to(DEV)
    with torch.no_grad():
        close(ens(x, t, idx[:, 0]), net(x, t).cpu().double())
        for p in ens.up:
            p.copy_(randn(g, *p.shape) * 0.1)
    w = torch.softmax(randn(g, N, 2), 1)
    xg = x.clone().requires_grad_()
    y = ens(xg, t, idx, w)
    gy = randn(g, N, D)
    grads = torch.autograd.grad(y, [xg, *ens.down, *ens.up], gy)
    want, xd, down, up = ensemble_reference(net, ens, x, t, idx, w)
    close(y, want)
    wants = torch.autograd.grad(want, [xd, *down, *up], gy.cpu().double())
    for a, b in zip(grads, wants):
        close(a, b, 1e-3)  # ReLU borders: a record whose value is within rounding of 0 may take the other side
    # one model per record and the mean of two equal ones agree; bad indices and timesteps are NaN in their records alone
    one = ens(x, t, idx[:, 0])
    two = ens(x, t, idx[:, :1].expand(N, 2))
    assert torch.allclose(one, two, rtol=1e-6, atol=1e-6)
    t2, idx2 = t.clone(), idx.clone()
    t2[3], t2[4], idx2[5, 1] = 50, -1, E
    bad = ens(x, t2, idx2, w)
    rest = torch.ones(N, dtype=torch.bool)
    rest[[3, 4, 5]] = False
    assert bool(torch.isnan(bad[[3, 4, 5]]).all()) and torch.allclose(bad.cpu()[rest], y.detach().cpu()[rest], rtol=1e-5, atol=1e-5)


def train(ens, opt, x, t, idx, noise, steps):
    for _ in range(steps):
        opt.zero_grad(set_to_none=False)
        loss = ((ens(x, t, idx) - noise) ** 2).mean()
        loss.backward()
        opt.step()
    return [p.detach().clone() for p in ens.parameters()]


def test_training_the_ensemble_with_our_step_and_torchs():
    """The operators as they are used: routed rows, adapted layers, their gradients, the step.  All optimizers see gradients of the same bits at
    the first step; eps = 1 keeps the update proportional to them.  The update, at most lr |g|, is then off by some 16 half steps of
    fp32 on either side, p by 4 of its own."""
    g = gen(51)
    N, D, E, kw = 120, 24, 3, dict(lr=1e-1, eps=1.0)
    x, noise = randn(g, N, D), randn(g, N, D)
    t, idx = torch.randint(0, 50, (N,), generator=g).to(DEV), torch.randint(0, E, (N,), generator=g).to(DEV)
    results = []
    for make in (lambda p: mtk.AdamW(p, **kw), lambda p: torch.optim.AdamW(p, **kw), lambda p: mtk.AdamW(p, **kw, capturable=True)):
        _, ens = ensemble(gen(1))
        start = [p.detach().clone() for p in ens.parameters()]
        results.append(train(ens, make(ens.parameters()), x, t, idx, noise, 1))
        grads = [p.grad for p in ens.parameters()]
    for a, b, c, s, gr in zip(*results, start, grads):
        assert torch.equal(a, c)
        assert bool(((a - b).abs() <= 32 * U32 * 1e-1 * gr.abs() + 8 * U32 * s.abs() + 2.0**-149).all())
    assert any(bool(gr.any()) for gr in grads)


@pytest.mark.parametrize("bits", [8, 32])
def test_a_captured_training_step_replays_like_the_eager_one(bits):
    g = gen(52)
    N, D, E = 100, 24, 3
    x, noise = randn(g, N, D), randn(g, N, D)
    t, idx = torch.randint(0, 50, (N,), generator=g).to(DEV), torch.randint(0, E, (N,), generator=g).to(DEV)

    def one(ens, opt):
        grads = torch.autograd.grad(((ens(x, t, idx) - noise) ** 2).sum() / N, list(ens.parameters()))
        for p, q in zip(ens.parameters(), grads):
            p.grad = q
        opt.step()

    _, eager = ensemble(gen(1))
    _, graph = ensemble(gen(1))
    with torch.no_grad():
        for a, b in zip(eager.parameters(), graph.parameters()):
            b.copy_(a)
    lr = torch.tensor(1e-3, device=DEV)
    oe, og = (mtk.AdamW(m.parameters(), lr=lr, state_bits=bits, capturable=True) for m in (eager, graph))
    plain = mtk.AdamW(graph.parameters(), lr=1e-3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one(graph, og)
    torch.cuda.current_stream().wait_stream(side)
    one(eager, oe)
    cg = torch.cuda.CUDAGraph()
    with torch.cuda.graph(cg):
        one(graph, og)
    for i in range(4):
        lr.fill_(1e-3 / (i + 1))
        x.copy_(randn(gen(60 + i), N, D))
        idx.copy_(torch.randint(-1, E, (N,), generator=gen(70 + i)))
        one(eager, oe)
        cg.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager.parameters(), graph.parameters()):
            assert torch.equal(a, b), i
        assert int(og.state[next(graph.parameters())]["step"]) == i + 2
    refused = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captur"):
        with torch.cuda.graph(refused):
            plain.step()


def test_gradients_that_a_captured_backward_may_not_take():
    """What a captured backward pass refuses, seen without a capture: a leaf whose accumulator an eager graph of the default stream keeps alive, and an
    eager graph's own nodes.  (The refused pass itself is not run: before, it ended the process.)"""
    from midst_toolkit_amd import _lib

    g = gen(95)
    a = adapter_inputs(g, 20, 8, 6, 2, 3, torch.float32)
    down = a["down"].requires_grad_()
    held = _lib.native().accumulates_on_default
    assert not held(down)  # no graph
    y = call(a)
    assert held(down) and held(y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = call(a)
    assert held(down)  # still the first graph's
    del y, z
    assert not held(down)
    with torch.cuda.stream(side):
        z = call(a)
        assert not held(down) and not held(z)
        z.sum().backward()
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.parametrize("bits", [8, 32])
def test_a_captured_backward_accumulates(bits):
    """backward() itself inside the capture, with no eager graph of the parameters alive: gradients and step are the eager ones at every replay"""
    g = gen(96)
    N, D, E = 80, 24, 3
    x, noise = randn(g, N, D), randn(g, N, D)
    t, idx = torch.randint(0, 50, (N,), generator=g).to(DEV), torch.randint(0, E, (N,), generator=g).to(DEV)

    def one(ens, opt):
        opt.zero_grad(set_to_none=True)
        ((ens(x, t, idx) - noise) ** 2).sum().backward()
        opt.step()

    _, eager = ensemble(gen(1))
    _, graph = ensemble(gen(1))
    with torch.no_grad():
        for p, q in zip(eager.parameters(), graph.parameters()):
            q.copy_(p)
    oe, og = (mtk.AdamW(m.parameters(), lr=1e-3, state_bits=bits, capturable=True) for m in (eager, graph))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one(graph, og)
    torch.cuda.current_stream().wait_stream(side)
    one(eager, oe)
    og.zero_grad(set_to_none=True)
    from midst_toolkit_amd import _lib

    assert not any(_lib.native().accumulates_on_default(p) for p in graph.parameters())
    cg = torch.cuda.CUDAGraph()
    with torch.cuda.graph(cg):
        one(graph, og)
    for i in range(4):
        x.copy_(randn(gen(60 + i), N, D))
        one(eager, oe)
        cg.replay()
        torch.cuda.synchronize()
        for p, q in zip(eager.parameters(), graph.parameters()):
            assert torch.equal(p, q) and torch.equal(p.grad, q.grad), i


def test_our_step_refreshes_the_modules_that_cache_their_weights():
    """TabSyn's denoiser keeps a packed copy keyed by its parameters' versions: after our step its loss is that of the new weights."""
    torch.manual_seed(0)
    model = mtk.tabsyn.Model(mtk.tabsyn.MLPDiffusion(12, dim_t=64)).to(DEV)
    twin = mtk.tabsyn.Model(mtk.tabsyn.MLPDiffusion(12, dim_t=64)).to(DEV)
    twin.load_state_dict(model.state_dict())
    g = gen(61)
    data, inj = randn(g, 40, 12), (randn(g, 40), randn(g, 40, 12))
    opt = mtk.AdamW(model.parameters(), lr=1e-2)
    losses = []
    for _ in range(3):
        loss = model(data, inj)
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    twin.load_state_dict(model.state_dict())
    with torch.no_grad():
        assert torch.equal(model(data, inj), twin(data, inj))
    assert len(set(losses)) == 3
