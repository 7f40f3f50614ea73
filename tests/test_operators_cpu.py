"""CPU: refusals of the row routing, low-rank adapter and AdamW entry points, and the arithmetic of the 8-bit moments' rounding."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

import midst_toolkit_amd as mtk
from midst_toolkit_amd import _lib
from tests.operator_refs import adamw8_reference, dither_codes


def test_no_cpu_path():
    plan = mtk.RowPlan(*(torch.zeros(2, dtype=torch.int32) for _ in range(3)), 1, 2, 1)
    with pytest.raises(RuntimeError, match="no CPU path"):
        mtk.route_rows(torch.zeros(2, dtype=torch.int64), 1)
    with pytest.raises(RuntimeError, match="no CPU path"):
        mtk.dispatch_rows(torch.zeros(2, 3), plan)
    with pytest.raises(RuntimeError, match="no CPU path"):
        mtk.combine_rows(torch.zeros(2, 3), plan)
    with pytest.raises(RuntimeError, match="no CPU path"):
        mtk.adapter_linear(torch.zeros(2, 3), torch.zeros(4, 3), None, torch.zeros(1, 2, 3), torch.zeros(1, 4, 2), torch.zeros(2, dtype=torch.int32))
    p = torch.nn.Parameter(torch.zeros(3))
    with pytest.raises(RuntimeError, match="no CPU path"):
        mtk.adamw_step([p], [p], [p], [p], 1, lr=1e-3)
    opt = mtk.AdamW([p])
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="no CPU path"):
        opt.step()


@pytest.mark.parametrize("bad", [dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8), dict(weight_decay=-1.0), dict(state_bits=16),
                                 dict(lr=torch.tensor(1e-3)), dict(lr=torch.tensor(1e-3), capturable=True), dict(lr=float("nan"))])
def test_adamw_arguments(bad):
    with pytest.raises(ValueError):
        mtk.AdamW([torch.nn.Parameter(torch.zeros(2))], **bad)


def test_adamw_takes_torchs_arguments():
    """The constructor calls that torch.optim.AdamW's users make, and what is refused: for all parameters, a group, one that is added"""
    p = lambda: torch.nn.Parameter(torch.zeros(2))  # noqa: E731
    kw = dict(amsgrad=False, maximize=False, foreach=None, capturable=False, differentiable=False, fused=None)
    torch.optim.AdamW([p()], 1e-3, (0.9, 0.99), 1e-8, 0.1, False, **{k: v for k, v in kw.items() if k != "amsgrad"})
    mtk.AdamW([p()], 1e-3, (0.9, 0.99), 1e-8, 0.1, False, **{k: v for k, v in kw.items() if k != "amsgrad"})
    opt = mtk.AdamW([{"params": [p()], "lr": 1e-2}], **{**kw, "foreach": True, "fused": True}, state_bits=8)
    assert opt.defaults["weight_decay"] == 1e-2 and opt.param_groups[0]["state_bits"] == 8
    for name in ("amsgrad", "maximize", "differentiable"):
        for make in (lambda n: mtk.AdamW([p()], **{n: True}), lambda n: mtk.AdamW([{"params": [p()], n: True}]), lambda n: opt.add_param_group({"params": [p()], n: True})):
            with pytest.raises(NotImplementedError, match=name):
                make(name)
    for bad in (dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=float("nan")), dict(state_bits=4), dict(lr=torch.tensor(1e-3))):
        with pytest.raises(ValueError):
            mtk.AdamW([{"params": [p()], **bad}], capturable=True)
        with pytest.raises(ValueError):
            opt.add_param_group({"params": [p()], **bad})
    assert len(opt.param_groups) == 1


def test_the_module_on_torchs_side_loads():
    """Its symbols resolve and it takes the library's functions, GPU or not"""
    assert _lib.native().declined() == ""


def test_adamw_lists_are_optional():
    mtk.adamw_step([], [], [], [], 1, lr=1e-3)


def test_c_entries_refuse_before_any_launch():
    """Every refusal comes from the host checks: nothing here reaches a GPU (there is none on this machine)."""
    l = _lib.lib()
    one = C.c_void_p(256)  # never dereferenced: the calls below are refused
    ARG, UNS = _lib.MTK_ERR_ARG, _lib.MTK_ERR_UNSUPPORTED
    assert l.mtk_route_rows(5, None, 3, one, one, one, None, 0, None) == ARG
    assert l.mtk_route_rows(-1, one, 3, one, one, one, None, 0, None) == ARG
    assert l.mtk_route_rows(5, one, 0, one, one, one, None, 0, None) == UNS
    assert l.mtk_route_rows(5, one, 1025, one, one, one, None, 0, None) == UNS
    assert l.mtk_route_rows(1 << 31, one, 3, one, one, one, one, 1 << 40, None) == UNS
    big = 1 << 20
    need = l.mtk_route_rows_work(big, 1024)
    assert need > 0 and l.mtk_route_rows(big, one, 1024, one, one, one, one, need - 1, None) == ARG
    assert l.mtk_rows_dispatch(4, 2, 0, 0, one, 8, one, None, one, None, None, None) == ARG
    assert l.mtk_rows_dispatch(4, 0, 8, 0, one, 8, one, None, one, None, None, None) == ARG
    assert l.mtk_rows_dispatch(4, 2, 8, 3, one, 8, one, None, one, None, None, None) == UNS
    assert l.mtk_rows_dispatch(1 << 30, 2, 8, 0, one, 8, one, None, one, None, None, None) == UNS
    assert l.mtk_rows_dispatch(4, 2, 8, 0, one, 8, one, None, None, None, None, None) == ARG
    assert l.mtk_rows_dispatch(4, 2, 8, 0, one, 8, one, None, one, one, None, None) == ARG
    assert l.mtk_rows_combine(4, 2, 8, 0, one, -1, one, None, one, None) == ARG
    assert l.mtk_rows_combine(4, 2, 8, 0, None, 8, one, None, one, None) == ARG
    fwd = lambda M=4, din=8, dout=8, r=2, E=2, dt=0, act=0, saved=1 << 30, x=one: l.mtk_adapter_forward(  # noqa: E731
        M, din, dout, r, E, dt, x, din, one, None, one, one, one, None, 1.0, act, 0, one, one, saved, None, 0, None)
    for kw in (dict(M=-1), dict(din=0), dict(dout=0), dict(r=0), dict(E=0), dict(saved=8), dict(x=None)):
        assert fwd(**kw) == ARG, kw
    for kw in (dict(r=257), dict(E=1025), dict(din=8193), dict(dout=8193), dict(M=(1 << 24) + 1), dict(dt=3), dict(act=2)):
        assert fwd(**kw) == UNS, kw
    assert fwd(M=5000, din=64, dout=64) == ARG  # no workspace
    assert l.mtk_adapter_backward(4, 8, 8, 2, 2, 0, one, 8, one, one, one, one, None, 1.0, 0, None, one, one, one, one, one, one, 16, None) == ARG
    assert l.mtk_adapter_backward(4, 8, 8, 2, 2, 0, one, 8, one, one, one, one, None, 1.0, 1, None, one, one, one, one, one, one, 1 << 30, None) == ARG
    for saved, work in ((264, 256), (256, 272)):  # 256-byte alignment is part of the layout
        assert l.mtk_adapter_forward(600, 8, 8, 2, 2, 0, one, 8, one, one, one, one, one, None, 1.0, 0, 0, one, saved, 1 << 30, work, 1 << 30, None) == ARG
        assert l.mtk_adapter_backward(600, 8, 8, 2, 2, 0, one, 8, one, one, one, one, None, 1.0, 0, None, one, saved, one, one, one, work, 1 << 30, None) == ARG
    ptrs, n = (C.c_void_p * 1)(256), (C.c_int64 * 1)(5)
    step = lambda dt=0, bits=32, lr=1e-3, b1=0.9, t=1, sc=ptrs, size=n, p=ptrs: l.mtk_adamw_step(  # noqa: E731
        1, p, ptrs, ptrs, ptrs, sc, sc, size, dt, bits, lr, b1, 0.999, 1e-8, 0.01, t, None, None)
    assert step(dt=7) == UNS and step(bits=4) == UNS and step(lr=-1.0) == ARG and step(lr=float("nan")) == ARG and step(b1=1.0) == ARG and step(t=0) == ARG
    assert step(bits=8, sc=None) == ARG and step(size=(C.c_int64 * 1)(-1)) == ARG and step(p=(C.c_void_p * 1)(None)) == ARG
    assert step(size=(C.c_int64 * 1)(1 << 40)) == UNS
    assert l.mtk_adamw_count(None, None, 1e-3, 0.9, 0.999, 1e-8, 0.0, one, None) == ARG
    assert l.mtk_adamw_count_each(2, None, None, 1e-3, 0.9, 0.999, 1e-8, 0.0, one, None) == ARG
    assert l.mtk_adamw_count_each(-1, ptrs, None, 1e-3, 0.9, 0.999, 1e-8, 0.0, one, None) == ARG
    assert l.mtk_adamw_count_each(1, (C.c_void_p * 1)(None), None, 1e-3, 0.9, 0.999, 1e-8, 0.0, one, None) == ARG
    for bad in ((-1e-3, 0.9, 0.999, 1e-8, 0.0), (float("nan"), 0.9, 0.999, 1e-8, 0.0), (1e-3, 1.0, 0.999, 1e-8, 0.0), (1e-3, 0.9, -0.1, 1e-8, 0.0), (1e-3, 0.9, 0.999, -1.0, 0.0),
                (1e-3, 0.9, 0.999, 1e-8, -0.1)):  # what the step refuses, whose numbers these become
        assert l.mtk_adamw_count_each(1, ptrs, None, *bad, one, None) == ARG and l.mtk_adamw_count(one, None, *bad, one, None) == ARG, bad
    assert l.mtk_adamw_step_each(1, ptrs, ptrs, ptrs, ptrs, None, None, n, 0, 32, None, None) == ARG
    assert l.mtk_adamw_step_each(1, ptrs, ptrs, ptrs, ptrs, None, None, n, 7, 32, one, None) == UNS
    assert l.mtk_adamw_scales(0) == 0 and l.mtk_adamw_scales(256) == 1 and l.mtk_adamw_scales(257) == 2


def test_workspace_sizes_are_monotonic_and_empty_for_nonsense():
    l = _lib.lib()
    assert l.mtk_adapter_saved_bytes(0, 8, 0) == 0 and l.mtk_adapter_saved_bytes(8, 8, 9) == 0
    assert 0 < l.mtk_adapter_saved_bytes(100, 8, 1) <= l.mtk_adapter_saved_bytes(1000, 8, 1)
    assert 0 < l.mtk_adapter_work_bytes(100, 64, 64, 8, 4, 1, 0, 1, 1, 1) < l.mtk_adapter_work_bytes(100, 64, 64, 8, 4, 1, 1, 1, 1, 1)
    assert l.mtk_adapter_work_bytes(100, 64, 64, 8, 4, 1, 0, 0, 0, 0) == 0  # few rows: nothing is laid out
    assert l.mtk_adapter_work_bytes(5000, 64, 64, 8, 4, 1, 0, 0, 1, 1) + 5000 * 64 * 2 <= l.mtk_adapter_work_bytes(5000, 64, 64, 8, 4, 1, 0, 0, 0, 1)
    ok = lambda p, ld, K, dt: l.mtk_adapter_streams(C.c_void_p(p), ld, K, dt)  # noqa: E731
    assert ok(256, 64, 64, 1) and ok(256, 0, 64, 1) and ok(256, 72, 64, 1) and ok(256, 32, 32, 0)
    assert not ok(258, 64, 64, 1) and not ok(256, 65, 64, 1) and not ok(256, 64, 32, 1) and not ok(256, 1 << 21, 64, 1) and not ok(256, 64, 64, 5)


def test_dither_rounds_to_neighbours_and_is_unbiased_over_the_steps():
    """The oracle of the 8-bit moments by itself: each value goes to one of its two neighbouring codes, codes stay where they are, and over
    n steps the mean is within the discrepancy of a Weyl sequence (below 4 log2(n) / n of a code step; n = 4096: 0.012) of the value."""
    codes = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy().astype(np.float64)
    x = np.concatenate([codes, np.exp(np.linspace(np.log(1e-4), np.log(448.0), 129))])[:256]
    x[-1] = 448.0
    place = np.arange(256)
    got = np.stack([dither_codes(x.astype(np.float32), 1.0, place, t, 0x6A09E667, 0.0) for t in range(1, 4097)])
    at = np.searchsorted(codes, x.astype(np.float32), side="right") - 1
    lo, hi = codes[at], codes[np.minimum(at + 1, len(codes) - 1)]
    assert np.all((got == lo) | (got == hi))
    exact = lo == x.astype(np.float32)
    assert np.all(got[:, exact] == lo[exact])
    step = np.where(hi > lo, hi - lo, 1.0)
    assert np.max(np.abs(got.mean(0) - x.astype(np.float32)) / step) < 0.012


def test_eight_bit_moments_follow_a_change_of_scale():
    """A gradient that drops tenfold: the root mean square has to come down with the average (a rounding to nearest would keep it).  From v = 1,
    g = 0.1: after n steps v = 0.01 + 0.99 * 0.999^n.  A value sits within one code step (1/8) of the average it follows, and the
    average of such values is off by no more than that: r within 25 %."""
    p, g = np.zeros(256, np.float32), np.full(256, 0.1, np.float32)
    m, ms, r, rs = np.zeros(256), 1.0, np.ones(256) * 256, 1.0 / 256
    for t in range(1, 3001):
        p, m, ms, r, rs = adamw8_reference(p, g, m, np.array([ms]), r, np.array([rs]), t, lr=0.0)
        ms, rs = float(ms[0]), float(rs[0])
    want = np.sqrt(0.01 + 0.99 * 0.999**3000)
    assert np.all(np.abs(r * rs / want - 1) < 0.25), (r * rs).min()


def test_pieces_of_a_factor_lie_inside_it(tmp_path):
    """The adapter kernels' lanes without a piece of their own load one all the same (and clear it): for every width from one feature on and
    every rank, each lane's piece has to lie inside its model's factor, the last model's with nothing behind it."""
    main = tmp_path / "pieces.cpp"
    main.write_text(r'''
#include <cstdio>
#include <initializer_list>
#include "mtk_low_piece.h"
int main() {
    for (int V : {4, 8})                                     // values of a 16-byte piece
        for (int N : {1, 2, 31, 33})
            for (int r = 1; r <= 256; ++r) {
                const int ld = (r + V - 1) / V * V;
                for (int n = 0; n < 64; ++n)                     // features of a tile, behind the last too
                    for (int j = 0; j < (r + 31) / 32 * 32; j += V) {  // the pieces of 32 values of the rank at a time
                        const int64_t at = mtk_low_piece(n, N, ld, ld, j);
                        if (at < 0 || at + V > (int64_t)N * ld || (j < r && at != (int64_t)(n < N ? n : N - 1) * ld + j)) {
                            std::printf("V %d N %d r %d feature %d value %d: offset %lld\n", V, N, r, n, j, (long long)at);
                            return 1;
                        }
                    }
            }
}
''')
    exe = tmp_path / "pieces"
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "midst-toolkit_amd", "csrc")
    subprocess.run(["g++", "-std=c++17", "-I", csrc, str(main), "-o", str(exe)], check=True)
    got = subprocess.run([str(exe)], capture_output=True, text=True)
    assert got.returncode == 0, got.stdout
