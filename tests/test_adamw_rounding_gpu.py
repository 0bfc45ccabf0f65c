"""What the optimizer step rounds, and where: the root and the quotient of the update, second moments below float32's normal
numbers, decays far below a weight's last bit."""
import math

import pytest
import torch

from oracle import train_oracle as to
from sv3d import optim
from test_adamw_gpu import BF16, F16

pytestmark = pytest.mark.gpu


def one(values, bits=32, step=0.0):
    """Lists of one tensor: zero weights with the gradients `values` and no moments yet."""
    g = values.cuda()
    p = torch.zeros_like(g)
    if bits == 32:
        m, v, e = torch.zeros_like(g), torch.zeros_like(g), None
    else:
        m, v = (torch.zeros(g.shape, dtype=torch.uint8, device="cuda") for _ in range(2))
        e = [torch.zeros(-(-g.numel() // 128), 2, dtype=torch.uint8, device="cuda")]
    return p, g, m, v, torch.tensor(step).cuda(), e


def run(p, g, m, v, s, e, **kw):
    optim.adamw_step([p], [g], [m], [v], [s], scales=e, **{"weight_decay": 0.0, **kw})


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [3000, 100000])         # in one workgroup, and in many
def test_root_and_quotient_are_rounded_to_nearest(bits, n):
    """Without memory (both betas 0) the step of a gradient g is g / sqrt(g^2).  The root of a rounded square is |g| again
    (no overflow, no underflow) and a number divided by itself is 1: the step is lr exactly, whatever g is."""
    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, generator=g) * 10.0 ** (3 * torch.randn(n, generator=g))
    t = one(x, bits)
    run(*t, lr=0.5, betas=(0.0, 0.0), eps=0.0)
    assert torch.equal(t[0].cpu(), -0.5 * x.sign())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [3000, 100000])
@pytest.mark.parametrize("eps", [0.0, 1e-22])
def test_first_steps_of_gradients_whose_squares_are_not_normal(bits, n, eps):
    """g from 1e-19 to 1e-17 at the first step: v = 1e-3 g^2 lies below 2^-126 in steps of 2^-149, half a step of which is
    up to 2^-150 / 1e-41 of it, 7e-5, and half as much of the root.  A tenth of g's size is far outside."""
    g = torch.Generator().manual_seed(n)
    x = 10.0 ** (-19 + 2 * torch.rand(n, generator=g)) * (torch.randint(0, 2, (n,), generator=g) * 2 - 1)
    p, gr, m, v, s, e = one(x, bits)
    run(p, gr, m, v, s, e, lr=1.0, eps=eps)
    w = x.double()
    want = to.adamw(torch.zeros(n, dtype=torch.float64), w, 0 * w, 0 * w, 0.0, lr=1.0, betas=(0.9, 0.999), eps=eps, weight_decay=0.0)
    v1 = 1e-3 * w * w
    # the product (1 - beta2) g and the square are each rounded; 4 covers the double rounding of both near the border
    room = 4 * 2.0 ** -150 / v1 + 16 * 2.0 ** -24
    assert bool(((p.cpu().double() - want["p"]).abs() <= room).all()), float(((p.cpu().double() - want["p"]).abs() / room).max())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [3000, 100000])
@pytest.mark.parametrize("t", [F16, BF16])
def test_the_same_for_16_bit_weights(bits, n, t):
    """The root's and the quotient's errors, a few 2^-23, are far below half a step of the weight: the step without memory is lr
    again, and first steps of gradients whose squares are not normal are +-1 (bf16, whose numbers go that far down; what the
    squares lose, 3e-4 at most, is below half a step as well)."""
    g = torch.Generator().manual_seed(n)
    x = (torch.randn(n, generator=g) * 10.0 ** torch.randn(n, generator=g)).to(t)
    x[x == 0] = 1.0
    a = one(x, bits)
    a = (*a[:2], *(s if s.dtype == torch.uint8 else s.float() for s in a[2:4]), *a[4:])
    run(*a, lr=0.5, betas=(0.0, 0.0), eps=0.0)
    assert torch.equal(a[0].cpu(), (-0.5 * x.sign()).to(t))
    if t is BF16:
        x = (10.0 ** (-19 + 2 * torch.rand(n, generator=g)) * x.sign().float()).to(t)
        a = one(x, bits)
        a = (*a[:2], *(s if s.dtype == torch.uint8 else s.float() for s in a[2:4]), *a[4:])
        run(*a, lr=1.0, eps=0.0)
        assert torch.equal(a[0].cpu(), -x.sign())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [3000, 100000])
@pytest.mark.parametrize("eps", [1e-17, 5.7e-11, 5.9e-11, 1e-8])
def test_first_steps_of_16_bit_weights_on_both_sides_of_what_eps_hides(bits, n, eps):
    """From 5.8e-11 (2^-39 / sqrt(1 - beta2)) an eps is so large that roots of squares below 2^-126 do not show next to it.
    A weight is lr u rounded once to bf16 (half a step: 2^-8); the squares' loss is at most 3e-4 of the root."""
    g = torch.Generator().manual_seed(n)
    x = (10.0 ** (-19 + 2 * torch.rand(n, generator=g)) * (torch.randint(0, 2, (n,), generator=g) * 2 - 1)).to(BF16)
    a = one(x, bits)
    a = (*a[:2], *(s if s.dtype == torch.uint8 else s.float() for s in a[2:4]), *a[4:])
    run(*a, lr=1.0, eps=eps)
    w = x.double()
    want = to.adamw(0 * w, w, 0 * w, 0 * w, 0.0, lr=1.0, betas=(0.9, 0.999), eps=eps, weight_decay=0.0)["p"]
    off = (a[0].cpu().double() - want).abs() / want.abs()
    assert float(off.max()) <= 2.0 ** -8 + 4e-4


@pytest.mark.parametrize("n", [300, 40000])
@pytest.mark.parametrize("bits", [32, 8])
def test_weights_that_never_had_a_gradient_stay_without_eps(bits, n):
    t = one(torch.zeros(n), bits)
    t[0].fill_(0.25)
    run(*t, lr=1.0, eps=0.0)
    assert bool((t[0] == 0.25).all())


@pytest.mark.parametrize("n, bits", [(65536, 32), (65536, 8), (8192, 32)])
@pytest.mark.parametrize("lr, weight_decay", [(1e-5, 0.01), (2e-6, 0.01), (1e-4, 0.01)])
def test_small_decays_add_up(n, bits, lr, weight_decay):
    """Decays of 1e-7, 2e-8 and 1e-6 of weights in [0.5, 1), whose last bit is 2^-24: each step rounds a weight by half of
    that at most, at random (the update's size, 1e-5 of many digits, decides), so the mean over n weights of what
    T steps add up to is off by 2^-24 / sqrt(12) * sqrt(T / n) or so.  8 of those, and the decay's own size by 1e-3.
    The first step is not at random: without a memory of others every update is lr or -lr.  With lr = 33.55 last bits and a
    decay of 0.17 to 0.33 of one, 33.72 to 33.88 become 34 and -33.38 to -33.22 become -33, 0.25 too much on average of both
    for all weights at once: up to half a last bit, 2^-25, for an lr in general."""
    steps = 200
    g = torch.Generator().manual_seed(5)
    start = 0.5 + 0.5 * torch.rand(n, generator=g)
    start = start.clamp(0.51, 0.99)
    p, gr, m, v, s, e = one(torch.zeros(n), bits)
    q, gq, mq, vq, sq, eq = one(torch.zeros(n), bits)
    p.copy_(start)
    q.copy_(start)
    moved = torch.zeros(n, dtype=torch.float64, device="cuda")       # what the updates without decay add up to
    for _ in range(steps):
        x = torch.randn(n, generator=g).cuda()
        gr.copy_(x)
        gq.copy_(x)
        run(p, gr, m, v, s, e, lr=lr, weight_decay=weight_decay, seed=3)
        q.zero_()
        run(q, gq, mq, vq, sq, eq, lr=lr, seed=3)
        moved += q.double()
    got = float((start.double() - p.cpu().double() + moved.cpu()).mean())
    # the sum over the steps of lr wd p, with p as it was: it moves by 200 lr at most
    want = steps * lr * weight_decay * float(start.double().mean())
    room = 2.0 ** -25 + 8 * 2.0 ** -24 / math.sqrt(12) * math.sqrt(steps / n) + want * (1e-3 + steps * lr)
    assert abs(got - want) <= room, (got, want, room)


@pytest.mark.parametrize("weight_decay", [0.0, 0.1])
@pytest.mark.parametrize("n", [300, 40000])
def test_infinite_weights_stay_what_they_are(weight_decay, n):
    """As a mask that is held as a weight: an infinity less its decay is that infinity."""
    p, g, m, v, s, e = one(torch.zeros(n))
    p[::3], p[1::3] = math.inf, -math.inf
    want = p.clone()
    run(p, g, m, v, s, e, lr=0.01, weight_decay=weight_decay)
    assert torch.equal(p, want)
    half = want.to(BF16)
    gh = torch.zeros_like(half)
    run(half, gh, m, v, s, e, lr=0.01, weight_decay=weight_decay)
    assert torch.equal(half, want.to(BF16))
