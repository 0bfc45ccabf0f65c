"""Layer norm over so many rows that a workgroup takes several turns: the next row's loads on their way, sums that share
their LDS with the turn before, a last turn that is partly empty, the weights' gradients over all turns; outputs that go past
the caches; rows behind 2^31 elements.  Against the float64 oracle with its bounds (tests/test_norm_gpu.py)."""
import pytest
import torch

import sv3d
from oracle import train_oracle as to
from test_norm_gpu import BF16, F16, F32, assert_near, check, make

pytestmark = pytest.mark.gpu

# Workgroups are at most 2048 of 256 threads (forward; as many threads in larger ones) and 512 (backward).  Turns of the
# forward and the backward for fp32, whether the row's end cuts a pack:
TURNS = [(66000, 24),       # 2 and 3, whole packs of fp32 and 16 bits
         (66000, 27),       # the same, cut
         (8300, 520),       # 5 and 5, whole
         (2500, 1337),      # 3 and 5, cut
         (2500, 4096),      # 3 and 5, whole, as many threads as packs
         (700, 8191)]       # 3 and 2, cut


@pytest.mark.parametrize("rows, cols", TURNS)
@pytest.mark.parametrize("x_type, param", [(F32, F32), (F16, F32), (BF16, BF16)])
def test_several_turns(rows, cols, x_type, param):
    x, w, b, dy = make(rows, cols, x_type, param, seed=rows + cols)
    check(x.cuda(), w.cuda(), b.cuda(), dy.cuda())


@pytest.mark.parametrize("rows, cols", [(66000, 27), (2500, 1337)])
def test_several_turns_of_half_precision_with_float32_results(rows, cols):
    x, w, b, dy = make(rows, cols, F16, F32, seed=rows)
    with torch.autocast("cuda", dtype=F16):
        check(x.cuda(), w.cuda(), b.cuda(), dy.cuda(), y_type=F32)


def on_device(rows, cols, x_type, seed):
    """Inputs of many elements, made and checked on the device."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return (rand(rows, cols) + 0.5).to(x_type), 1 + 0.3 * rand(cols), 0.3 * rand(cols), rand(rows, cols).to(x_type)


def assert_near_there(got, want, bound):
    """`assert_near` without the way to the host."""
    half, tiny = {F32: (2.0 ** -24, 2.0 ** -149), F16: (2.0 ** -11, 2.0 ** -24), BF16: (2.0 ** -8, 2.0 ** -133)}[got.dtype]
    room = bound + half * (want.abs() + bound) + tiny
    off = (got.double() - want).abs() / room
    assert bool(torch.isfinite(got).all()) and float(off.max()) <= 1.0, "off by %.3g of the room at worst" % float(off.max())


@pytest.mark.parametrize("rows, cols, x_type", [(16400, 4096, BF16), (16400, 4097, BF16), (9000, 7501, BF16), (70000, 1337, F16),
                                                (1500000, 27, F32), (70000, 512, F32), (40000, 1001, F32)])
def test_outputs_past_the_caches(rows, cols, x_type):
    """The forward moves more than 256 MB, the backward more again: rows on 16-byte alignment and off it."""
    assert rows * cols * 2 * x_type.itemsize >= 1 << 28 and cols <= 8192
    x, w, b, dy = on_device(rows, cols, x_type, rows + cols)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = sv3d.layer_norm(x, cols, w, b)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        wide = w.double()
        f = to.layer_norm(x.double(), wide, b.double(), 1e-5)
        assert_near_there(y, f["y"], f["e_y"])
        back = to.layer_norm_backward(f, dy.double(), wide)
        assert_near_there(dx, back["dx"], back["e_dx"])
        assert_near_there(dw, back["dw"], back["e_dw"])
        assert_near_there(db, back["db"], back["e_db"])


@pytest.mark.parametrize("cols", [8192, 8191])
def test_rows_behind_2_to_the_31_elements(cols):
    rows, some = 270000, torch.tensor([0, 1, 131071, 262144, 262150, 269998, 269999])
    assert rows * cols > 1 << 31
    g = torch.Generator().manual_seed(cols)
    values = (torch.randn(len(some), cols, generator=g) + 0.5).to(BF16)
    x = torch.zeros(rows, cols, dtype=BF16, device="cuda")
    x[some.cuda()] = values.cuda()
    y = sv3d.layer_norm(x, cols)
    f = to.layer_norm(values.double(), None, None, 1e-5)
    assert_near(y[some.cuda()], f["y"], f["e_y"])
    live = torch.zeros(rows, dtype=torch.bool, device="cuda")
    live[some.cuda()] = True
    assert torch.equal(y.abs().amax(1) > 0, live)
    del y
    _, mean, rstd = torch.ops.sv3d.layer_norm_stats(x, [cols], None, None, 1e-5, False)
    dx, dw, db = torch.ops.sv3d.layer_norm_backward(x, x, [cols], None, None, mean, rstd, True, True, True)
    back = to.layer_norm_backward(f, values.double(), None)
    assert_near(dx[some.cuda()], back["dx"], back["e_dx"])
    assert torch.equal(dx.abs().amax(1) > 0, live)
    # the other rows add zeros; their chain of additions is the bound's as well
    more = 2.0 ** -24 * rows / 64
    assert_near(dw, back["dw"], back["e_dw"] + more * (values.double() * f["h"]).abs().sum(0))
    assert_near(db, back["db"], back["e_db"] + more * values.double().abs().sum(0))
