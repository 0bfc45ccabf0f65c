"""The optimizer step on the GPU against the float64 oracle: many tensors, odd sizes, types, layouts, 32-bit and 8-bit
moments, clipping, loss scales, gradients that are no numbers, streams and graphs.  Tolerances are the oracle's bounds of
a float32 evaluation plus half a step of the type that is stored; an 8-bit moment has to be one of the two codes next to
its value, and the right one unless the value is within its bound of the border between them."""
import math

import pytest
import torch

from oracle import train_oracle as to
from sv3d import optim

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HYPER = dict(lr=2e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.02)


def wide(t):
    return t.detach().cpu().double().reshape(-1)


class Set:
    """Lists of tensors as `adamw_step` takes them, each inside a larger buffer whose rest must not change."""

    def __init__(self, sizes, types=F32, bits=32, seed=0, step=3.0, spread=1.0, offset=0):
        g = torch.Generator().manual_seed(seed)
        n = len(sizes)
        types = types if isinstance(types, (list, tuple)) else [types] * n
        bits = bits if isinstance(bits, (list, tuple)) else [bits] * n
        self.around, self.offset = [], offset
        self.p, self.g, self.m, self.v, self.e, self.steps = [], [], [], [], [], []
        for size, t, b in zip(sizes, types, bits):
            rand = lambda: torch.randn(size, generator=g)  # noqa: E731
            scale = 10.0 ** (spread * torch.randn(-(-size // 32) if size else 0, generator=g)).repeat_interleave(32)[:size] * 1e-2
            scale[: size // 7] = 0.0            # some never had a gradient
            p, grad, m = rand() * 0.3, rand() * scale, 0.3 * rand() * scale
            v = (0.3 + torch.rand(size, generator=g)) * scale ** 2
            self.p.append(self.put(p, t))
            self.g.append(self.put(grad, t))
            if b == 8:
                blocks = -(-size // 128)
                e = torch.stack([to.scale_bytes_of(m.double(), to.FIRST), to.scale_bytes_of(v.double(), to.SECOND)], 1)
                e = e.reshape(blocks, 2)
                self.m.append(self.put(self.codes(m, e[:, 0], to.FIRST), torch.uint8))
                self.v.append(self.put(self.codes(v, e[:, 1], to.SECOND), torch.uint8))
                self.e.append(self.put(e.reshape(-1), torch.uint8).view(blocks, 2))
            else:
                self.m.append(self.put(m, F32))
                self.v.append(self.put(v, F32))
                self.e.append(torch.empty(0, dtype=torch.uint8).cuda())
            self.steps.append(torch.tensor(step).cuda())
        self.bits = bits

    @staticmethod
    def codes(x, e, kind):
        low, high, _, _ = to.rounded(x.double(), e, kind, torch.zeros(len(x)))
        near = torch.where((x - low).abs() <= (high - x).abs(), low, high)
        unit = (2.0 ** (e.double() - kind["bias"])).repeat_interleave(128)[: len(x)]
        c = torch.searchsorted(to.code_values(kind), (near.abs() / unit).contiguous())
        return c + 128 * (x < 0) * (kind is to.FIRST)

    def put(self, values, t):
        """`values` in the middle of a buffer of a sentinel."""
        pad = 64
        buf = torch.full((len(values) + 2 * pad,), 77, dtype=t).cuda()
        at = pad + self.offset
        view = buf[at: at + len(values)]
        view.copy_(values.to(t))
        self.around.append((buf, at, len(values)))
        return view

    def values(self):
        """Everything in float64 on the host: [(p, g, m, v, bytes)]."""
        got = []
        for p, g, m, v, e, b in zip(self.p, self.g, self.m, self.v, self.e, self.bits):
            if b == 8:
                e = e.cpu().view(-1, 2)
                got.append((wide(p), wide(g), to.decode(m.cpu(), e[:, 0], to.FIRST), to.decode(v.cpu(), e[:, 1], to.SECOND), e))
            else:
                got.append((wide(p), wide(g), wide(m), wide(v), None))
        return got

    def step(self, **kw):
        args = {**HYPER, **kw}
        return optim.adamw_step(self.p, self.g, self.m, self.v, self.steps, scales=self.e if 8 in self.bits else None, **args)

    def assert_untouched_around(self):
        for buf, at, n in self.around:
            assert bool((buf[:at] == 77).all()) and bool((buf[at + n:] == 77).all())


def assert_near(got, want, bound, t, what):
    same = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    off = (got - want)[same].abs()
    room = (bound + HALF_STEP[t] * (want.abs() + bound) + TINY[t])[same]
    assert bool((off <= room).all()), "%s off by %.3g of the room" % (what, float((off / room).max()))


def assert_codes(got, want, bound, e, kind, part, what):
    """8-bit moments: rounding is monotonic, so a value within the bound of `want` has a byte and a code between those
    of the bound's two ends.  The move of values below the smallest normal one costs up to 2^-21 of a code's step."""
    ok = torch.isfinite(want)
    assert bool(got[~ok].isnan().all()), what
    least, most = (want.abs() - bound).clamp(min=0), torch.where(ok, want.abs() + bound, math.nan)
    assert bool(((e >= to.scale_bytes_of(least, kind)) & (e <= to.scale_bytes_of(most, kind))).all()), what
    gap = to.rounded(want, e, kind, part)[3]

    def code(x):
        low, high, over, _ = to.rounded(x, e, kind, part)
        return torch.where(over >= 0, high, low)

    room = bound + gap * 2.0 ** -20
    low, high = want - room, want + room
    if kind is to.SECOND:
        low = low.clamp(min=0)
    assert bool(((got >= code(low)) & (got <= code(high)))[ok].all()), what


def check_step(s, max_norm=0.0, scale=None, found_inf=None, maximize=False, seed=0, **kw):
    hyper = {**HYPER, **kw}
    before = s.values()
    steps = [float(t) for t in s.steps]
    call = dict(max_norm=max_norm, maximize=maximize, seed=seed, **kw)
    if scale is not None:
        call["grad_scale"] = torch.tensor(scale).cuda()
    if found_inf is not None:
        call["found_inf"] = torch.tensor(found_inf).cuda()
    norm = s.step(**call)
    clip, total = 1.0, None
    if max_norm:
        total = math.sqrt(sum(float((b[1] ** 2).sum()) for b in before)) / (scale or 1.0)
        if math.isfinite(total):
            assert abs(float(norm) - total) <= 2.0 ** -23 * total
        clip = to.clip_factor(total, max_norm)
    else:
        assert norm is None
    for k, ((p, g, m, v, _), (p1, g1, m1, v1, e1)) in enumerate(zip(before, s.values())):
        what = "tensor %d of %d elements" % (k, len(p))
        assert torch.equal(g1.nan_to_num(nan=1e30), g.nan_to_num(nan=1e30)), what
        assert float(s.steps[k]) == steps[k] + 1
        want = to.adamw(p, g, m, v, steps[k], scale=scale or 1.0, clip=clip, maximize=maximize, **hyper)
        assert_near(p1, want["p"], want["e_p"], s.p[k].dtype, what + " p")
        if s.bits[k] == 8:
            part = to.dither(len(p), int(steps[k]) + 1, seed)
            assert_codes(m1, want["m"], want["e_m"], e1[:, 0], to.FIRST, part // 65536, what + " exp_avg")
            assert_codes(v1, want["v"], want["e_v"], e1[:, 1], to.SECOND, part % 65536, what + " exp_avg_sq")
        else:
            assert_near(m1, want["m"], want["e_m"], F32, what + " exp_avg")
            assert_near(v1, want["v"], want["e_v"], F32, what + " exp_avg_sq")
    s.assert_untouched_around()
    return total


SIZES = [1, 2, 3, 5, 127, 128, 129, 255, 256, 257, 1000, 2047, 2048, 2049, 4095, 8193, 70001]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_sizes_types_and_alignments(bits, t, offset):
    s = Set(SIZES, t, bits, seed=offset, offset=offset)
    for _ in range(3):
        check_step(s, seed=5)


@pytest.mark.parametrize("n", [1, 63, 64, 65, 130, 450])
def test_numbers_of_tensors_of_every_kind_in_one_call(n):
    g = torch.Generator().manual_seed(n)
    pick = lambda options: [options[i] for i in torch.randint(len(options), (n,), generator=g).tolist()]  # noqa: E731
    sizes = [int(x) for x in torch.randint(0, 700, (n,), generator=g)]
    s = Set(sizes, pick([F32, F16, BF16]), pick([8, 32]), seed=n)
    check_step(s, max_norm=0.5)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("max_norm, scale, maximize", [(0.05, None, False), (1e6, None, True), (0.05, 1024.0, False),
                                                       (0.0, 65536.0, True), (float("inf"), 2.0, False)])
def test_clipping_scaling_and_direction(bits, max_norm, scale, maximize):
    s = Set([9000, 1, 300], bits=bits, seed=1)
    check_step(s, max_norm=max_norm, scale=scale, maximize=maximize, found_inf=0.0)


def test_norm_of_gradients_whose_squares_leave_float32():
    for size in (1e-30, 1e30):
        s = Set([5000, 17], seed=3)
        for g in s.g:
            g.mul_(size)
        check_step(s, max_norm=1.0)


@pytest.mark.parametrize("bits", [32, 8])
def test_found_inf_changes_nothing(bits):
    s = Set([5000, 17], bits=bits, seed=3)
    before = [b[0].clone() for b in s.around]
    s.g[0][7] = float("inf")
    before = [b[0].clone() for b in s.around]
    norm = s.step(max_norm=0.1, found_inf=torch.tensor(1.0).cuda(), grad_scale=torch.tensor(8.0).cuda())
    assert math.isinf(float(norm))
    assert all(torch.equal(b[0].nan_to_num(), k.nan_to_num()) for b, k in zip(s.around, before))
    assert all(float(t) == 3.0 for t in s.steps)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("max_norm", [0.0, 0.1])
def test_gradients_that_are_no_numbers(bits, max_norm):
    """Without clipping they spoil their own elements and no others; with it, as with clip_grad_norm_, a NaN norm is in
    every element and an infinite one leaves infinite elements NaN and the rest without a gradient."""
    s = Set([1000, 300], bits=bits, seed=2)
    s.g[0][5], s.g[0][200], s.g[0][201] = float("nan"), float("inf"), -float("inf")
    check_step(s, max_norm=max_norm)
    s = Set([1000, 300], bits=bits, seed=2)
    s.g[0][200] = float("inf")
    check_step(s, max_norm=max_norm)


def test_moments_at_both_ends_of_the_range():
    s = Set([512, 512, 512, 300], bits=8, seed=4, spread=4.0)
    s.g[1].zero_()
    s.g[1][3] = 1e-25                   # squares below float32's normal numbers
    s.g[2].mul_(1e6)
    s.g[3].mul_(1e-12)
    for _ in range(4):
        check_step(s)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_steps_from_a_fresh_state(bits):
    s = Set([1000, 129, 4], BF16, bits, seed=6, step=0.0)
    for group in (s.m, s.v, s.e):
        for x in group:
            x.zero_()
    g = torch.Generator().manual_seed(8)
    for _ in range(12):
        for x in s.g:
            x.copy_(torch.randn(x.shape, generator=g) * 0.01)
        check_step(s, max_norm=1.0)


@pytest.mark.parametrize("hyper", [dict(betas=(0.0, 0.0)), dict(lr=0.0), dict(eps=0.0), dict(weight_decay=0.0),
                                   dict(betas=(0.5, 0.99), eps=1e-3, lr=1.0)])
def test_hyperparameters(hyper):
    s = Set([700, 3], seed=7)
    if hyper.get("eps") == 0.0:         # 0/0 where there never was a gradient
        for x in (s.p, s.g, s.m, s.v):
            x[0][:100] = torch.tensor(1.0)
    check_step(s, **hyper)


def test_learning_rate_on_the_device():
    a, b = Set([700, 3], seed=7), Set([700, 3], seed=7)
    a.step(lr=0.25)
    b.step(lr=torch.tensor(0.25).cuda())
    assert all(torch.equal(x, y) for x, y in zip(a.p, b.p))


@pytest.mark.parametrize("bits", [32, 8])
def test_bits_do_not_depend_on_the_alignment_the_order_or_the_call(bits):
    """The same tensor gives the same bits alone, among others and off any alignment."""
    alone, among, off = Set([3001], bits=bits, seed=1), Set([3001, 77, 129], bits=bits, seed=1), Set([3001], bits=bits, seed=1, offset=1)
    for _ in range(2):
        for s in (alone, among, off):
            s.step()
    for s in (among, off):
        for x, y in ((alone.p, s.p), (alone.m, s.m), (alone.v, s.v), (alone.e, s.e)):
            assert torch.equal(x[0], y[0])


def test_layouts_follow_the_weight():
    w = torch.randn(8, 6, 3, 3).cuda().to(memory_format=torch.channels_last)
    g = torch.randn(8, 6, 3, 3).cuda()
    m, v, s = torch.zeros_like(w), torch.zeros_like(w), torch.zeros(()).cuda()
    flat = [x.clone(memory_format=torch.contiguous_format) for x in (w, m, v)]
    optim.adamw_step([w], [g], [m], [v], [s], **HYPER)                  # the gradient lies otherwise than its weight
    optim.adamw_step([flat[0]], [g], [flat[1]], [flat[2]], [torch.zeros(()).cuda()], **HYPER)
    assert w.is_contiguous(memory_format=torch.channels_last)
    assert torch.equal(w, flat[0]) and torch.equal(m, flat[1]) and torch.equal(v, flat[2])


def test_the_same_memory_twice_is_refused():
    s = Set([300, 300])
    bad = [
        ([s.p[0], s.p[0]], s.m, s.v, s.steps),
        (s.p, [s.m[0], s.m[0]], s.v, s.steps),
        (s.p, s.m, s.v, [s.steps[0], s.steps[0]]),
        (s.p, s.m, s.m, s.steps),
        ([s.p[0], s.around[0][0][65:365]], s.m, s.v, s.steps),
    ]
    for p, m, v, steps in bad:
        with pytest.raises(ValueError):
            optim.adamw_step(p, s.g, m, v, steps, **HYPER)
    with pytest.raises(RuntimeError):
        optim.adamw_step(s.p, [s.g[0], s.g[1].cpu()], s.m, s.v, s.steps, **HYPER)


def test_gradients_may_be_shared_but_lie_nowhere_else():
    s = Set([300, 300])
    before = [[x.clone() for x in list_] for list_ in (s.p, s.m, s.v, s.steps)]
    for g in ([s.p[0], s.g[1]], [s.g[0], s.m[0]], [s.g[0], s.around[0][0][65:365]]):
        with pytest.raises(ValueError):
            optim.adamw_step(s.p, g, s.m, s.v, s.steps, **HYPER)
    for list_, kept in zip((s.p, s.m, s.v, s.steps), before):
        assert all(torch.equal(x, y) for x, y in zip(list_, kept))
    twice = Set([300, 300])
    twice.g[1].copy_(twice.g[0])
    optim.adamw_step(s.p, [twice.g[0], twice.g[0]], s.m, s.v, s.steps, **HYPER)
    again = Set([300, 300])
    optim.adamw_step(again.p, twice.g, again.m, again.v, again.steps, **HYPER)
    for x, y in zip(s.p + s.m + s.v, again.p + again.m + again.v):
        assert torch.equal(x, y)


def test_square_sums():
    g = torch.Generator().manual_seed(0)
    xs = [torch.randn(n, generator=g).to(t).cuda() for n, t in ((0, F32), (1, F16), (70001, F32), (4097, BF16), (9, F32))]
    xs.append(torch.randn(40, 30, generator=g).cuda()[:, ::2])
    want = sum(float((wide(x) ** 2).sum()) for x in xs)
    got = optim.grad_square_sums(xs)
    assert got.dtype == torch.float64 and abs(float(got.sum()) - want) < 1e-12 * want
    assert torch.equal(got, optim.grad_square_sums(xs))


def test_moment_values():
    g = torch.Generator().manual_seed(0)
    for n in (1, 127, 128, 300, 70000):
        m, v = (torch.randint(0, 256, (n,), generator=g, dtype=torch.int32).to(torch.uint8) for _ in range(2))
        e = torch.randint(0, 248, (-(-n // 128), 2), generator=g, dtype=torch.int32).to(torch.uint8)
        a, b = optim.moment_values(m.cuda(), v.cuda(), e.cuda())
        assert a.dtype == b.dtype == BF16
        assert torch.equal(wide(a).nan_to_num(nan=-7), to.decode(m, e[:, 0], to.FIRST).nan_to_num(nan=-7))
        assert torch.equal(wide(b).nan_to_num(nan=-7), to.decode(v, e[:, 1], to.SECOND).nan_to_num(nan=-7))
    assert optim.moment_values(*(torch.empty(0, dtype=torch.uint8).cuda() for _ in range(3)))[0].numel() == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_and_replayed(bits):
    """Two captured steps on sets of their own and eager ones between the replays: the bits of eager steps."""
    mine, theirs = [Set([9000, 70, 300], bits=bits, seed=k) for k in (1, 2)], [Set([9000, 70, 300], bits=bits, seed=k) for k in (1, 2)]
    inf = torch.zeros(()).cuda()
    call = dict(max_norm=0.05, found_inf=inf, grad_scale=torch.tensor(4.0).cuda())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in mine + theirs:
            s.step(**call)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, norms = [], []
    for s in mine:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norms.append(s.step(**call))
        graphs.append(graph)
    for k in range(5):
        inf.fill_(1.0 if k == 2 else 0.0)
        for s in mine + theirs:
            for x in s.g:
                x.mul_(-0.5).add_(0.001 * k)
        want = [s.step(**call) for s in theirs]
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for a, b, na, nb in zip(mine, theirs, norms, want):
            assert torch.equal(na, nb)
            for x, y in zip(a.p + a.m + a.v + a.e + a.steps, b.p + b.m + b.v + b.e + b.steps):
                assert torch.equal(x, y), k


def test_on_streams_of_their_own():
    sets, want = [Set([40000, 300], bits=8, seed=k) for k in range(4)], [Set([40000, 300], bits=8, seed=k) for k in range(4)]
    for s in want:
        for _ in range(3):
            s.step(max_norm=0.1)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for s, stream in zip(sets, streams):
        stream.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                s.step(max_norm=0.1)
    torch.cuda.synchronize()
    for a, b in zip(sets, want):
        assert all(torch.equal(x, y) for x, y in zip(a.p + a.m + a.v + a.e, b.p + b.m + b.v + b.e))


# ---- the optimizer -----------------------------------------------------------------------------------------
def network(seed=0):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(40, 300), torch.nn.Tanh(), torch.nn.Linear(300, 7)).cuda()


def run(net, opt, steps, clip=None, seed=1):
    g = torch.Generator().manual_seed(seed)
    for _ in range(steps):
        x = torch.randn(16, 40, generator=g).cuda()
        opt.zero_grad(set_to_none=True)
        net(x).square().mean().backward()
        if clip is not None:
            torch.nn.utils.clip_grad_norm_(net.parameters(), clip)
        opt.step()


@pytest.mark.parametrize("kw", [dict(weight_decay=0.1), dict(weight_decay=0.0, maximize=True), dict(betas=(0.5, 0.9), eps=1e-4)])
def test_optimizer_takes_torchs_steps(kw):
    a, b = network(), network()
    run(a, torch.optim.AdamW(a.parameters(), lr=1e-2, **kw), 5, clip=0.02)
    ours = optim.AdamW(b.parameters(), lr=1e-2, max_norm=0.02, **kw)
    run(b, ours, 5)
    for x, y in zip(a.parameters(), b.parameters()):
        # five float32 steps of up to 1e-2 each; where a gradient is near zero its sign's size is what rounding decides
        assert float((x - y).abs().max()) < 1e-4
    assert ours.total_norm is not None and float(ours.total_norm) > 0


def test_optimizer_groups_share_one_norm_and_skip_weights_without_gradients():
    net = network()
    opt = optim.AdamW([{"params": [net[0].weight]}, {"params": [net[0].bias, net[2].weight, net[2].bias], "lr": 0.0}], lr=1e-2, max_norm=0.1)
    net(torch.randn(4, 40).cuda()).square().sum().backward()
    net[2].bias.grad = None
    want = torch.nn.utils.get_total_norm([p.grad for p in net.parameters() if p.grad is not None])
    before = [p.detach().clone() for p in net.parameters()]
    opt.step()
    assert abs(float(opt.total_norm) - float(want)) < 1e-5 * float(want)
    moved = [not torch.equal(p, q) for p, q in zip(net.parameters(), before)]
    assert moved == [True, False, False, False]
    assert net[2].bias not in opt.state or not opt.state[net[2].bias]


def test_optimizer_with_a_grad_scaler_skips_overflows_and_unscales():
    a, b = network(), network()
    oa, ob = torch.optim.AdamW(a.parameters(), lr=1e-2), optim.AdamW(b.parameters(), lr=1e-2, max_norm=0.02)
    sa, sb = (torch.amp.GradScaler("cuda", init_scale=2.0 ** 10) for _ in range(2))
    g = torch.Generator().manual_seed(1)
    for k in range(6):
        x = torch.randn(16, 40, generator=g).cuda() * (1e30 if k == 2 else 1.0)
        for net, opt, s in ((a, oa, sa), (b, ob, sb)):
            opt.zero_grad(set_to_none=True)
            s.scale(net[2](net[0](x)).square().mean()).backward()
        sa.unscale_(oa)
        torch.nn.utils.clip_grad_norm_(a.parameters(), 0.02)
        sa.step(oa)
        sa.update()
        sb.step(ob)
        sb.update()
        assert sa.get_scale() == sb.get_scale()
    for x, y in zip(a.parameters(), b.parameters()):
        assert float((x - y).abs().max()) < 1e-4
    assert all(float(s["step"]) == 5.0 for s in ob.state.values())


def test_optimizer_state_survives_saving_and_memory_formats():
    def make():
        net = network(3)
        return net, optim.AdamW(net.parameters(), lr=1e-2, state_bits=8, min_8bit_size=1000, max_norm=1.0, seed=9)
    a, oa = make()
    run(a, oa, 3)
    assert [s["exp_avg"].dtype for s in oa.state.values()] == [torch.uint8, F32, torch.uint8, F32]
    b, ob = make()
    b.load_state_dict(a.state_dict())
    ob.load_state_dict(oa.state_dict())
    run(a, oa, 3, seed=5)
    run(b, ob, 3, seed=5)
    for x, y in zip(a.parameters(), b.parameters()):
        assert torch.equal(x, y)


def test_optimizer_in_a_graph_and_its_state_made_before():
    net = network()
    rate = torch.tensor(1e-2).cuda()
    opt = optim.AdamW(net.parameters(), lr=rate, max_norm=0.1, state_bits=8, min_8bit_size=1000)
    for p in net.parameters():
        p.grad = torch.randn(p.shape).cuda()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(graph):
            opt.step()
    torch.cuda.synchronize()
    opt.step()
    twin = network()
    twin.load_state_dict(net.state_dict())
    other = optim.AdamW(twin.parameters(), lr=1e-2, max_norm=0.1, state_bits=8, min_8bit_size=1000)
    other.load_state_dict(opt.state_dict())
    for q, p in zip(twin.parameters(), net.parameters()):
        q.grad = p.grad
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(4):
        value = 1e-2 / (k + 1)
        rate.fill_(value)
        for group in other.param_groups:
            group["lr"] = float(rate)
        for p in net.parameters():
            p.grad.mul_(-0.7)
        other.step()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(net.parameters(), twin.parameters()):
            assert torch.equal(p, q), k


def test_a_step_between_forward_and_backward_is_noticed():
    net = network()
    opt = optim.AdamW(net.parameters())
    run(net, opt, 1)
    loss = net(torch.randn(4, 40).cuda()).square().sum()
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_operator_registration():
    s = Set([300, 20], bits=[8, 32])
    torch.library.opcheck(torch.ops.sv3d.adamw_step.default,
                          (s.p, s.g, s.m, s.v, s.e, s.steps, None, None, None, None, 1e-3, 0.9, 0.99, 1e-8, 0.0, 0.0, False, 0),
                          test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(torch.ops.sv3d.moment_values.default, (s.m[0], s.v[0], s.e[0]), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(torch.ops.sv3d.grad_square_sums.default, (s.g,), test_utils=("test_schema", "test_faketensor"))


def test_more_elements_than_32_bits_count():
    """2^32 + 300 elements: a tensor's pieces start at multiples of 2^31, elements 2^32 apart share their dither."""
    n, far, mid = 2 ** 32 + 300, 2 ** 32, 2 ** 31
    small = Set([300], BF16, 8, seed=1)
    p, g = (torch.zeros(n, dtype=BF16, device="cuda") for _ in range(2))
    m, v = (torch.zeros(n, dtype=torch.uint8, device="cuda") for _ in range(2))
    e, step = torch.zeros(-(-n // 128), 2, dtype=torch.uint8, device="cuda"), small.steps[0].clone()
    for at in (0, mid, far):
        for big, little in ((p, small.p[0]), (g, small.g[0]), (m, small.m[0]), (v, small.v[0])):
            big[at: at + 300] = little
        e[at // 128: at // 128 + 3] = small.e[0]
    sums = optim.grad_square_sums([g])
    assert abs(float(sums.sum()) - 3 * float((wide(small.g[0]) ** 2).sum())) < 1e-9
    before = small.values()[0]
    optim.adamw_step([p], [g], [m], [v], [step], scales=[e], **HYPER)
    small.step()
    for at in (0, far):
        for big, little in ((p, small.p[0]), (m, small.m[0]), (v, small.v[0])):
            assert torch.equal(big[at: at + 300], little)
        assert torch.equal(e[at // 128: at // 128 + 3], small.e[0])
    assert torch.equal(p[mid: mid + 300], small.p[0])
    want = to.adamw(*before[:4], 3.0, **HYPER)
    x = (torch.arange(300) + mid + 4 * 0x9E3779B1) % 2 ** 32
    x = (x ^ (x >> 16)) * 0x6A09E667 % 2 ** 32
    x = (x ^ (x >> 15)) * 0xBB67AE85 % 2 ** 32
    x = x ^ (x >> 16)
    bytes_mid = e[mid // 128: mid // 128 + 3].cpu()
    assert_codes(to.decode(m[mid: mid + 300].cpu(), bytes_mid[:, 0], to.FIRST), want["m"], want["e_m"], bytes_mid[:, 0], to.FIRST,
                 x // 65536, "exp_avg")
    assert not p[300:1000].any() and not p[mid + 300: mid + 1000].any() and not m[far - 1000: far].any()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_small_calls_give_the_bits_of_large_ones(bits, t):
    """A few thousand elements take one workgroup and one launch; among many others they take the general way."""
    few = [1, 2048, 130, 3001, 0, 2049]
    small, large = Set(few, t, bits, seed=1, offset=1), Set(few + [60000], t, bits, seed=1, offset=1)
    for k in range(3):
        a = small.step(max_norm=1e9, grad_scale=torch.tensor(2.0).cuda(), found_inf=torch.tensor(float(k == 1)).cuda())
        b = large.step(max_norm=1e9, grad_scale=torch.tensor(2.0).cuda(), found_inf=torch.tensor(float(k == 1)).cuda())
        assert float(a) <= float(b)
        for x, y in ((small.p, large.p), (small.m, large.m), (small.v, large.v), (small.e, large.e), (small.steps, large.steps)):
            assert all(torch.equal(i, j) for i, j in zip(x, y)), k
    small.assert_untouched_around()


def test_empty_tensors_and_a_norm_of_nothing():
    s = Set([0, 0])
    assert float(s.step(max_norm=1.0)) == 0.0 and all(float(t) == 4.0 for t in s.steps)
    sums = optim.grad_square_sums(s.g)
    assert sums.numel() == 0 and float(s.step(max_norm=1.0, square_sums=sums)) == 0.0
    s = Set([0, 5, 0])
    check_step(s, max_norm=0.1)
