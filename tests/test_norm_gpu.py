"""Layer norm on the GPU against the float64 oracle: sizes from one element to rows of many thousand, every type
combination, strides, rows that are not numbers, gradients, streams and graphs.  The tolerances are the oracle's bounds
of a float32 evaluation plus half a step of the type that is stored."""
import pytest
import torch

import sv3d
from oracle import train_oracle as to

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}      # steps near zero
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def make(rows, cols, x_type=F32, param=F32, seed=0, weight=True, bias=True, level=0.5):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = (rand(rows, cols) + level).to(x_type)
    w = (1 + 0.3 * rand(cols)).to(param) if weight else None
    b = (0.3 * rand(cols)).to(param) if bias else None
    return x, w, b, rand(rows, cols)


def wide(t):
    return None if t is None else t.detach().cpu().double()


def assert_near(got, want, bound, kind=None):
    """|got - want| within the bound plus half a step of got's type."""
    t = kind or got.dtype
    got = wide(got).reshape(want.shape)
    assert torch.equal(torch.isfinite(got), torch.isfinite(want))
    ok = torch.isfinite(want)
    room = (bound + HALF_STEP[t] * (want.abs() + bound) + TINY[t])[ok]
    off = (got - want)[ok].abs()
    assert bool((off <= room).all()), "off by %.3g of the room at worst" % float((off / room).max())


def check(x, w, b, dy, eps=1e-5, y_type=None, cols=None):
    """Forward and backward through autograd, against the oracle."""
    cols = cols or x.shape[-1]
    xg = x.detach().requires_grad_()
    wg, bg = (None if t is None else t.detach().requires_grad_() for t in (w, b))
    shape = x.shape[x.dim() - 1:] if w is None else w.shape
    y = sv3d.layer_norm(xg, shape, wg, bg, eps)
    assert y.dtype == (y_type or x.dtype) and y.shape == x.shape and y.is_contiguous()
    dy = dy.to(y.dtype)
    leaves = [t for t in (xg, wg, bg) if t is not None]
    grads = list(torch.autograd.grad(y, leaves, dy))
    flat = lambda t: wide(t).reshape(-1, cols)  # noqa: E731
    vec = lambda t: None if t is None else wide(t).reshape(-1)  # noqa: E731
    f = to.layer_norm(flat(x), vec(w), vec(b), eps)
    back = to.layer_norm_backward(f, flat(dy), vec(w))
    assert_near(y, f["y"].reshape(y.shape), f["e_y"].reshape(y.shape))
    dx = grads.pop(0)
    assert dx.dtype == x.dtype and dx.shape == x.shape
    assert_near(dx, back["dx"].reshape(dx.shape), back["e_dx"].reshape(dx.shape))
    for name, t in (("dw", w), ("db", b)):
        if t is None:
            continue
        got = grads.pop(0)
        assert got.dtype == t.dtype and got.shape == t.shape
        assert_near(got, back[name].reshape(got.shape), back["e_" + name].reshape(got.shape))
    with torch.no_grad():
        assert torch.equal(sv3d.layer_norm(x, shape, w, b, eps), y)
    return y


SIZES = [(1, 1), (3, 1), (1, 2), (2, 7), (5, 63), (4, 64), (7, 65), (6, 127), (128, 200), (33, 512), (9, 1000), (300, 24),
         (3, 1337), (5, 2048), (3, 2049), (2, 4097), (3, 8192), (2, 16384), (2, 20000), (1, 70001), (5003, 24), (2000, 513)]


@pytest.mark.parametrize("rows, cols", SIZES)
@pytest.mark.parametrize("x_type, param", [(F32, F32), (F16, F32), (BF16, BF16)])
def test_sizes_and_types(rows, cols, x_type, param):
    x, w, b, dy = make(rows, cols, x_type, param, seed=rows * 31 + cols)
    check(x.cuda(), w.cuda(), b.cuda(), dy.cuda())


@pytest.mark.parametrize("cols", [40, 200, 333, 4096])
@pytest.mark.parametrize("x_type", [F32, F16, BF16])
@pytest.mark.parametrize("weight, bias", [(None, None), (F32, None), (None, F32), ("x", "x"), (F32, "x"), ("x", F32)])
def test_weights_that_are_there_or_not_and_of_either_type(cols, x_type, weight, bias):
    x, w, b, dy = make(17, cols, x_type, F32, seed=cols, weight=weight is not None, bias=bias is not None)
    as_type = lambda t, kind: None if t is None else t.to(x_type if kind == "x" else F32).cuda()  # noqa: E731
    check(x.cuda(), as_type(w, weight), as_type(b, bias), dy.cuda())


@pytest.mark.parametrize("x_type, param", [(F32, F16), (F32, BF16), (F16, BF16)])
def test_weights_of_a_third_type_are_read_as_float32(x_type, param):
    x, w, b, dy = make(9, 72, x_type, param)
    check(x.cuda(), w.cuda(), b.cuda(), dy.cuda())


def test_rows_may_lie_anywhere():
    x, w, b, dy = make(24, 96, seed=5)
    w, b = w.cuda(), b.cuda()
    big = torch.randn(24, 200).cuda()
    big[:, 50:146] = x.cuda()
    check(big[:, 50:146], w, b, dy.cuda())                              # a slice of wider rows
    check(big[:, 51:147], w, b, dy.cuda())                              # that starts off any alignment
    check(x.cuda().view(2, 3, 4, 96), w, b, dy.cuda().view(2, 3, 4, 96))
    check(x.cuda().t().contiguous().t(), w, b, dy.cuda())               # rows that are not contiguous
    check(x.cuda()[::3], w, b, dy.cuda()[::3])                          # every third row
    check(x.cuda().view(4, 6, 96).transpose(0, 1), w, b, dy.cuda().view(6, 4, 96))
    check(x[:1].cuda().expand(24, 96), w, b, dy.cuda())                 # one row many times
    check(x.cuda(), w, b, dy[:1].cuda().expand(24, 96))                 # a gradient that is broadcast over rows
    check(x.cuda(), w, b, torch.ones((), device="cuda").expand(24, 96))  # and over everything
    odd = torch.randn(24 * 96 + 1).cuda()[1:]
    odd.copy_(x.cuda().view(-1))
    check(odd.view(24, 96), w, b, dy.cuda())                            # rows off 16-byte alignment
    half = torch.empty(24 * 96 + 1, dtype=F16).cuda()[1:]
    half.copy_(x.cuda().view(-1))
    wo = torch.empty(97).cuda()[1:]
    wo.copy_(w)
    check(half.view(24, 96), wo, b, dy.cuda())


def test_several_dimensions_are_normalised_together():
    g = torch.Generator().manual_seed(1)
    x, w, b, dy = (torch.randn(*s, generator=g).cuda() for s in ((6, 5, 4, 3), (5, 4, 3), (5, 4, 3), (6, 5, 4, 3)))
    check(x, w, b, dy, cols=60)
    check(x.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1), w, b, dy, cols=60)


@pytest.mark.parametrize("cols", [64, 300, 5000, 30000])
def test_constant_rows_large_levels_and_wide_ranges(cols):
    x, w, b, dy = make(8, cols, seed=cols)
    x[0] = 0.0
    x[1] = 3.25
    x[2] = 1e4 + x[2]                   # variance far below the mean's square
    x[3] *= 1e-6                        # variance far below eps
    x[4] *= 1e8
    x[5, : cols // 2] *= 1e-3
    check(x.cuda(), w.cuda(), b.cuda(), dy.cuda())


@pytest.mark.parametrize("cols", [48, 200, 3000, 30000])
@pytest.mark.parametrize("x_type", [F32, F16])
def test_a_row_that_is_no_number_spoils_no_other(cols, x_type):
    x, w, b, dy = make(6, cols, x_type, seed=2)
    x[1, cols // 3], x[4, 0] = float("nan"), float("inf")
    x[2, 1] = torch.finfo(x_type).min if x_type is F16 else -1e15
    y = sv3d.layer_norm(x.cuda(), cols, w.cuda(), b.cuda()).cpu()
    assert bool(y[[1, 4]].isnan().all())
    f = to.layer_norm(wide(x[[0, 2, 3, 5]]), wide(w), wide(b), 1e-5)
    assert_near(y[[0, 2, 3, 5]], f["y"], f["e_y"])
    xg = x.cuda().requires_grad_()
    dx, = torch.autograd.grad(sv3d.layer_norm(xg, cols, w.cuda(), b.cuda()), xg, dy.cuda().to(x_type))
    back = to.layer_norm_backward(f, wide(dy.to(x_type))[[0, 2, 3, 5]], wide(w))
    assert_near(dx[[0, 2, 3, 5]], back["dx"], back["e_dx"])


def test_empty_input_and_zero_gradients_of_the_weights():
    x = torch.empty(0, 16).cuda().requires_grad_()
    w, b = torch.ones(16).cuda().requires_grad_(), torch.zeros(16).cuda().requires_grad_()
    y = sv3d.layer_norm(x, 16, w, b)
    assert y.shape == (0, 16)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty(0, 16).cuda())
    assert dx.shape == (0, 16) and not dw.any() and not db.any()


@pytest.mark.parametrize("need", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1)])
@pytest.mark.parametrize("cols", [64, 3000])
def test_only_what_is_asked_for(need, cols):
    x, w, b, dy = (t.cuda() for t in make(10, cols))
    whole = [t.detach().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(sv3d.layer_norm(whole[0], cols, whole[1], whole[2]), whole, dy)
    some = [t.detach().requires_grad_(bool(n)) for t, n in zip((x, w, b), need)]
    leaves = [t for t in some if t.requires_grad]
    got = torch.autograd.grad(sv3d.layer_norm(some[0], cols, some[1], some[2]), leaves, dy)
    for a, e in zip(got, [t for t, n in zip(want, need) if n]):
        assert torch.equal(a, e)


def test_gradient_against_differences_of_the_definition():
    x, w, b, dy = make(5, 37, seed=9)
    g = torch.Generator().manual_seed(4)
    xg, wg, bg = (t.cuda().requires_grad_() for t in (x, w, b))
    grads = torch.autograd.grad(sv3d.layer_norm(xg, 37, wg, bg), (xg, wg, bg), dy.cuda())
    args = [t.double() for t in (x, w, b)]
    loss = lambda a: float((to.layer_norm(*a, 1e-5)["y"] * dy.double()).sum())  # noqa: E731
    for k, got in enumerate(grads):
        d = torch.randn(got.shape, generator=g).double()
        h = 1e-5
        move = lambda s: [t + s * h * d if i == k else t for i, t in enumerate(args)]  # noqa: E731
        quotient = (loss(move(1)) - loss(move(-1))) / (2 * h)
        along = float((wide(got) * d).sum())
        # roundings of the kernel's gradient (some 40 per entry here) and of the float64 difference
        room = 64 * 2.0 ** -24 * float((wide(got) * d).abs().sum()) + 1e-8 * abs(quotient) + 1e-8
        assert abs(along - quotient) < room, (k, along, quotient)


def test_same_bits_every_time_on_any_stream_and_with_calls_in_flight_together():
    x, w, b, dy = (t.cuda() for t in make(3000, 520, BF16))
    dy = dy.to(BF16)

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = sv3d.layer_norm(leaves[0], 520, leaves[1], leaves[2])
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = step()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(3):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(step())
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, e) for a, e in zip(r, want))


@pytest.mark.parametrize("cols", [200, 2500, 20000])
def test_captured_and_replayed(cols):
    x, w, b, dy = (t.cuda() for t in make(40, cols, F16))
    dy = dy.to(F16)

    def step(x, w, b):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = sv3d.layer_norm(leaves[0], cols, leaves[1], leaves[2])
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, w, b)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, w, b)
    for k in range(4):
        x.mul_(-0.75).add_(0.125 * k)
        w.add_(0.25)
        want = step(x, w, b)                   # eager work between the replays
        for t in out:
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(out, want)), k


def test_autocast_returns_float32_as_torch_does():
    x, w, b, dy = make(20, 300, F16, F32)
    with torch.autocast("cuda", dtype=F16):
        check_y = check(x.cuda(), w.cuda(), b.cuda(), dy.cuda(), y_type=F32)
        ref = torch.nn.functional.layer_norm(x.cuda(), (300,), w.cuda(), b.cuda())
    assert ref.dtype == check_y.dtype == F32


def test_module_stands_in_for_torchs():
    net = torch.nn.TransformerEncoderLayer(64, 4, 128, batch_first=True, dropout=0.0).cuda()
    x = torch.randn(6, 9, 64, device="cuda")
    want = net(x)
    want.square().sum().backward()
    grads = {k: p.grad.clone() for k, p in net.named_parameters()}
    net.zero_grad(set_to_none=True)
    assert sv3d.convert_layer_norm(net) == 2
    got = net(x)
    got.square().sum().backward()
    # both are float32 evaluations; products of 64 to 128 terms amplify a rounding about tenfold
    assert float((got - want).detach().abs().max()) < 1e-4 * float(want.detach().abs().max())
    # The sum of squares of a normalised row hardly depends on the row: with u = 2h the last norm's
    # dx = r (u - mean u - h mean(u h)) = 2 r h (1 - mean h^2) = 2 r h eps / (var + eps), so what goes further back is
    # eps / (var + eps) <= 1e-5 of terms (var is about 1, the norm's input being a sum of a norm's output and a small
    # one) that each carry roundings of 2^-24.  32 of them: 32 * 2^-24 / 1e-5 of the largest entry.
    for k, p in net.named_parameters():
        assert float((p.grad - grads[k]).abs().max()) < 32 * 2.0 ** -24 / 1e-5 * float(grads[k].abs().max()), k


def test_gradients_through_a_block_with_the_module():
    """A loss without that cancellation: a fixed random combination of the outputs.  Some fifty roundings on the way of
    each term (four products of 64 to 128 terms, two norms, a softmax) stay below 1e-4 of the largest entry."""
    torch.manual_seed(0)
    net = torch.nn.TransformerEncoderLayer(64, 4, 128, batch_first=True, dropout=0.0).cuda()
    x, c = torch.randn(6, 9, 64, device="cuda"), torch.randn(6, 9, 64, device="cuda")
    (net(x) * c).sum().backward()
    grads = {k: p.grad.clone() for k, p in net.named_parameters()}
    net.zero_grad(set_to_none=True)
    sv3d.convert_layer_norm(net)
    (net(x) * c).sum().backward()
    for k, p in net.named_parameters():
        assert float((p.grad - grads[k]).abs().max()) < 1e-4 * float(grads[k].abs().max()), k


def test_no_second_derivative_and_no_change_after_the_forward():
    x, w, b, dy = (t.cuda() for t in make(4, 32))
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(sv3d.layer_norm(x, 32, w, b), x, dy, create_graph=True)
    z = x * 1
    y = sv3d.layer_norm(z, 32, w, b)
    z.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, x, dy)


def test_the_graph_can_be_kept_used_in_part_and_only_once():
    x, w, b, dy = (t.cuda() for t in make(6, 40))
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    y = sv3d.layer_norm(leaves[0], 40, leaves[1], leaves[2])
    assert y.requires_grad and "LayerNormBackward" in y.grad_fn.name()
    first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    only_w, = torch.autograd.grad(y, leaves[1:2], dy, retain_graph=True)
    again = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(only_w, first[1]) and all(torch.equal(a, e) for a, e in zip(again, first))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, leaves, dy)
    # through checkpointing, whose hooks take the saved tensors away and recompute them
    from torch.utils.checkpoint import checkpoint
    y = checkpoint(lambda a: sv3d.layer_norm(a * 1, 40, leaves[1], leaves[2]), leaves[0], use_reentrant=False)
    assert all(torch.equal(a, e) for a, e in zip(torch.autograd.grad(y, leaves, dy), first))
    for t in leaves:
        t.grad = None
    (sv3d.layer_norm(leaves[0], 40, leaves[1], leaves[2]) * dy).sum().backward()
    (sv3d.layer_norm(leaves[0], 40, leaves[1], leaves[2]) * dy).sum().backward()
    assert all(torch.equal(t.grad, 2 * e) for t, e in zip(leaves, first))       # accumulated: twice the same bits


def test_operator_registration():
    tests = ("test_schema", "test_autograd_registration", "test_faketensor")
    x, w, b, dy = (t.cuda() for t in make(4, 32))
    for a in (x, w, b):
        a.requires_grad_()
    torch.library.opcheck(torch.ops.sv3d.layer_norm.default, (x, [32], w, b, 1e-5, False), test_utils=tests)
    _, mean, rstd = torch.ops.sv3d.layer_norm_stats(x.detach(), [32], None, None, 1e-5, False)
    torch.library.opcheck(torch.ops.sv3d.layer_norm_backward.default,
                          (dy, x.detach(), [32], None, None, mean, rstd, True, True, True), test_utils=("test_schema", "test_faketensor"))


def test_more_elements_than_32_bits_count():
    rows, cols = 70000, 32768                       # 2.3e9 elements of two bytes
    x = torch.empty(rows, cols, dtype=BF16, device="cuda")
    x[-3:] = torch.randn(3, cols, device="cuda").to(BF16)
    x[:3] = x[-3:]
    x[3:-3] = 0
    y = sv3d.layer_norm(x, cols)
    assert torch.equal(y[:3], y[-3:]) and not y[3].any()
    f = to.layer_norm(wide(x[-3:]), None, None, 1e-5)
    assert_near(y[-3:], f["y"], f["e_y"])
    del y
    _, mean, rstd = torch.ops.sv3d.layer_norm_stats(x, [cols], None, None, 1e-5, False)
    dx, _, _ = torch.ops.sv3d.layer_norm_backward(x, x, [cols], None, None, mean, rstd, True, False, False)
    assert torch.equal(dx[:3], dx[-3:])
    back = to.layer_norm_backward(f, wide(x[-3:]), None)
    assert_near(dx[-3:], back["dx"], back["e_dx"])
