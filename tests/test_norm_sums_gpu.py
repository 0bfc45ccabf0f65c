"""The sums over rows of the layer norm's weight gradients."""
import pytest
import torch

import sv3d

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [24, 512, 1337, 8192, 20000])
@pytest.mark.parametrize("t", [torch.float32, torch.float16, torch.bfloat16])
def test_what_the_workgroups_add_up_loses_nothing_where_it_is_joined(cols, t):
    """db is a sum of rows 65 apart, which lie in workgroups of their own: 2^15, then 62 numbers that are small against it (2^-10,
    exact in every type) and -2^15.  A sum in float32 (last bit of 2^15: 2^-8) would lose the small ones; one that holds
    43 bits or more is exact, and so is its result."""
    rows, n = 65 * 64, 64
    x = torch.randn(rows, cols, device="cuda").to(t)
    w, b = (torch.ones(cols, device="cuda").requires_grad_() for _ in range(2))
    dy = torch.zeros(rows, cols, dtype=t, device="cuda")
    dy[::65] = 2.0 ** -10
    dy[0], dy[65 * (n - 1)] = 2.0 ** 15, -2.0 ** 15
    dw, db = torch.autograd.grad(sv3d.layer_norm(x, cols, w, b), (w, b), dy)
    assert db.dtype == torch.float32 and bool((db == (n - 2) * 2.0 ** -10).all())
