"""The common norm of many gradients: more tensors of one type than a launch takes, and norms that are taken ahead of the
step."""
import pytest
import torch

from sv3d import optim
from test_adamw_gpu import BF16, F16, F32, Set, check_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [251, 600])
@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_norms_of_more_tensors_of_one_type_than_a_launch_takes(n, t):
    """A launch sums up 250 tensors.  Some are empty; the last one has most of the norm, so that a launch that is left out
    or written over shows."""
    g = torch.Generator().manual_seed(n)
    sizes = [int(x) for x in torch.randint(1, 9000, (n,), generator=g)]
    for k in range(5, n, 17):
        sizes[k] = 0
    s = Set(sizes, t, seed=n)
    s.g[-1].mul_(64.0)
    s.g[251 if n > 251 else 0].mul_(16.0)
    want = sum(float((x.double() ** 2).sum()) for x in s.g)
    got = optim.grad_square_sums(s.g)
    assert abs(float(got.sum()) - want) <= 1e-12 * want
    check_step(s, max_norm=0.05)


def kernels_of(f):
    """Names of the optimizer's kernels that f launches."""
    from torch.profiler import ProfilerActivity, profile
    f()
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        f()
        torch.cuda.synchronize()
    return [e.name for e in p.events() if "adamw" in e.name]


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_are_read_out_of_the_caches_wherever_a_norm_was_taken_of_them(bits):
    """In one call, or ahead of it for several groups; past them where there is no norm."""
    s = Set([60000, 300], bits=bits, seed=1)
    name = "adamw8_kernel" if bits == 8 else "adamw_kernel"
    taken = lambda f, past: any("%s<float, %s>(" % (name, past) in k for k in kernels_of(f))  # noqa: E731
    assert taken(lambda: s.step(max_norm=0.1), "false")
    assert taken(lambda: s.step(max_norm=0.1, square_sums=optim.grad_square_sums(s.g)), "false")
    assert taken(lambda: s.step(), "true")
