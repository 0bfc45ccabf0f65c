"""Layer norm and the optimizer step without a GPU: the oracle's formulas against differences and known values, the
refusals of the operators (shape-only kernels) and of the C ABI (argument checks come before any launch)."""
import ctypes
import math

import pytest
import torch

from oracle import train_oracle as to
from sv3d import _lib as L
from sv3d import norm, optim

F64 = torch.float64


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- the oracle ---------------------------------------------------------------------------------------------
def test_layer_norm_gradient_formulas_against_differences():
    g = gen(0)
    x, dy = torch.randn(3, 7, generator=g, dtype=F64), torch.randn(3, 7, generator=g, dtype=F64)
    w, b = torch.randn(7, generator=g, dtype=F64), torch.randn(7, generator=g, dtype=F64)
    eps, h = 1e-3, 1e-5
    got = to.layer_norm_backward(to.layer_norm(x, w, b, eps), dy, w)
    loss = lambda x, w, b: float((to.layer_norm(x, w, b, eps)["y"] * dy).sum())  # noqa: E731
    for name, k, t in (("dx", 0, x), ("dw", 1, w), ("db", 2, b)):
        for i in range(t.numel()):
            d = torch.zeros_like(t).view(-1)
            d[i] = h
            d = d.view(t.shape)
            args = [x, w, b]
            up, down = list(args), list(args)
            up[k], down[k] = t + d, t - d
            quotient = (loss(*up) - loss(*down)) / (2 * h)
            # third derivatives of order 1/eps^1.5 at most here; h^2 of them
            assert abs(quotient - float(got[name].reshape(-1)[i])) < 1e-6, (name, i)


def test_codes_are_ascending_exact_in_bf16_and_rounded_without_bias():
    for kind in (to.FIRST, to.SECOND):
        values = to.code_values(kind)
        assert bool((values[1:] > values[:-1]).all()) and float(values[8]) == 2.0 ** kind["lowest"]
        for byte in (kind["floor"], 127, 254):
            exact = values * 2.0 ** (byte - kind["bias"])
            exact = exact[exact < 2.0 ** 128]           # at byte 254 the topmost codes lie beyond float32
            assert torch.equal(exact.to(torch.bfloat16).double(), exact)
    # a value a quarter of the way between two codes goes up a quarter of the time: 4 sigma of 2^16 draws
    n = 1 << 16
    part = to.dither(n, 3, 5)
    for bits in (part // 65536, part % 65536):
        x = torch.full((n,), 1.0 + 1 / 32, dtype=F64)
        _, _, over, _ = to.rounded(x, torch.full((n // 128,), 127), to.FIRST, bits)
        up = float((over >= 0).double().mean())
        assert abs(up - 0.25) < 4 * math.sqrt(0.25 * 0.75 / n), up


def test_dither_bits_are_even_over_elements_and_over_steps():
    n = 1 << 16
    over_steps = torch.cat([to.dither(64, t, 0)[:64] for t in range(1024)])
    for x in (to.dither(n, 1, 0), over_steps):
        for half in (x // 65536, x % 65536):
            counts = torch.bincount(half >> 12, minlength=16).double()
            expect = n / 16
            chi2 = float(((counts - expect) ** 2 / expect).sum())
            assert chi2 < 50.0, chi2            # 15 degrees of freedom: above 50 once in 10^5
        assert abs(float(torch.corrcoef(torch.stack([x // 65536, x % 65536]).double())[0, 1])) < 5 / math.sqrt(n)


# ---- refusals of the operators --------------------------------------------------------------------------------
def meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("x, shape, weight, bias, eps", [
    (meta(4, 8), (7,), None, None, 1e-5),
    (meta(4, 8), (4, 4, 8), None, None, 1e-5),
    (meta(4, 8), (), None, None, 1e-5),
    (meta(4, 0), (0,), None, None, 1e-5),
    (meta(4, 8), (8,), meta(7), None, 1e-5),
    (meta(4, 8), (8,), meta(8), meta(2, 4), 1e-5),
    (meta(4, 8, dtype=torch.float64), (8,), None, None, 1e-5),
    (meta(4, 8, dtype=torch.int32), (8,), None, None, 1e-5),
    (meta(4, 8), (8,), meta(8, dtype=torch.float64), None, 1e-5),
    (meta(1, (1 << 24) + 1), ((1 << 24) + 1,), None, None, 1e-5),
])
def test_layer_norm_refuses(x, shape, weight, bias, eps):
    with pytest.raises(ValueError):
        norm.layer_norm(x, shape, weight, bias, eps)


def test_layer_norm_shapes_and_types_without_a_gpu():
    y, mean, rstd = torch.ops.sv3d.layer_norm_stats(meta(2, 3, 8, dtype=torch.bfloat16), [3, 8], None, None, 1e-5, False)
    assert y.shape == (2, 3, 8) and y.dtype == torch.bfloat16 and mean.shape == rstd.shape == (2,)
    y = torch.ops.sv3d.layer_norm(meta(2, 8, dtype=torch.float16), [8], meta(8), None, 1e-5, True)
    assert y.dtype == torch.float32 and y.shape == (2, 8)
    with pytest.raises(NotImplementedError):
        norm.layer_norm(torch.zeros(2, 8), 8)
    with pytest.raises(ValueError):             # statistics of another call
        torch.ops.sv3d.layer_norm_backward(meta(2, 8), meta(2, 8), [8], None, None, meta(3), meta(2), True, False, False)
    with pytest.raises(ValueError):
        torch.ops.sv3d.layer_norm_backward(meta(2, 4), meta(2, 8), [8], None, None, meta(2), meta(2), True, False, False)


def lists(n=100, dtype=torch.float32, bits=32, **changes):
    blocks = -(-n // 128)
    state = torch.float32 if bits == 32 else torch.uint8
    a = dict(params=[meta(n, dtype=dtype)], grads=[meta(n, dtype=dtype)], exp_avgs=[meta(n, dtype=state)],
             exp_avg_sqs=[meta(n, dtype=state)], steps=[meta()], scales=[meta(blocks, 2, dtype=torch.uint8)] if bits == 8 else None)
    a.update(changes)
    return a


def test_adamw_step_accepts_what_it_says():
    for a in (lists(), lists(bits=8), lists(0), lists(dtype=torch.bfloat16, bits=8), lists(129, bits=8)):
        assert optim.adamw_step(a.pop("params"), a.pop("grads"), a.pop("exp_avgs"), a.pop("exp_avg_sqs"), a.pop("steps"), **a) is None
    assert optim.adamw_step([], [], [], [], []) is None


@pytest.mark.parametrize("a", [
    lists(grads=[meta(99)]),
    lists(grads=[]),
    lists(grads=[meta(100, dtype=torch.bfloat16)]),
    lists(exp_avgs=[meta(100, dtype=torch.float16)]),
    lists(exp_avgs=[meta(100, dtype=torch.uint8)]),
    lists(exp_avg_sqs=[meta(100, 1)]),
    lists(steps=[meta(2)]),
    lists(steps=[meta(dtype=torch.int64)]),
    lists(dtype=torch.float64),
    lists(bits=8, scales=None),
    lists(bits=8, scales=[meta(2, 2, dtype=torch.uint8)]),
    lists(bits=8, scales=[meta(1, 2)]),
    lists(params=[meta(100, 2)[:, 0]]),                                     # gaps between its elements
    lists(params=[meta(1).expand(100)]),                                    # one element a hundred times
    lists(params=[meta(10, 10).t()], grads=[meta(10, 10)], exp_avgs=[meta(10, 10)], exp_avg_sqs=[meta(10, 10)]),
    lists(max_norm=-1.0),
    lists(max_norm=float("nan")),
])
def test_adamw_step_refuses(a):
    with pytest.raises(ValueError):
        optim.adamw_step(a.pop("params"), a.pop("grads"), a.pop("exp_avgs"), a.pop("exp_avg_sqs"), a.pop("steps"), **a)


@pytest.mark.parametrize("kw", [dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1.0),
                                dict(weight_decay=-1.0), dict(max_norm=-1.0), dict(state_bits=16),
                                dict(lr=torch.zeros(2)), dict(lr=torch.zeros((), dtype=F64))])
def test_optimizer_refuses(kw):
    with pytest.raises(ValueError):
        optim.AdamW([torch.nn.Parameter(torch.zeros(3))], **kw)


def test_optimizer_on_the_host_fails_loudly_and_moment_values_refuses():
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    with pytest.raises(NotImplementedError):
        optim.AdamW([p]).step()
    with pytest.raises(ValueError):
        optim.moment_values(meta(5), meta(5), meta(1, 2))
    with pytest.raises(ValueError):
        optim.moment_values(meta(300, dtype=torch.uint8), meta(300, dtype=torch.uint8), meta(2, 2, dtype=torch.uint8))


def test_state_dict_of_8_bit_moments_survives_loading_into_a_16_bit_model():
    def make():
        p = torch.nn.Parameter(torch.zeros(300, dtype=torch.bfloat16))
        return p, optim.AdamW([p], state_bits=8, min_8bit_size=1)
    p, a = make()
    a.state[p] = {"step": torch.tensor(7.0), "exp_avg": torch.arange(300).to(torch.uint8),
                  "exp_avg_sq": torch.arange(300).to(torch.uint8), "scales": torch.full((3, 2), 99, dtype=torch.uint8)}
    q, b = make()
    b.load_state_dict(a.state_dict())
    for name, value in a.state[p].items():
        assert b.state[q][name].dtype == value.dtype and torch.equal(b.state[q][name], value), name
        assert b.state[q][name].data_ptr() != value.data_ptr()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_state_dict_of_torchs_adam_is_taken_over_in_the_weights_layout(dtype):
    def make():
        torch.manual_seed(0)
        return [torch.nn.Parameter(torch.randn(4, 6, 3, 3).to(dtype)), torch.nn.Parameter(torch.randn(()).to(dtype))]
    params = make()
    a = torch.optim.Adam(params, lr=0.5, betas=(0.5, 0.75))
    for p in params:
        p.grad = torch.randn_like(p)
    a.step()
    saved = a.state_dict()
    saved["state"][1]["step"] = 1                               # as old files have it
    mine = make()
    mine[0].data = mine[0].data.to(memory_format=torch.channels_last)
    b = optim.AdamW(mine, lr=torch.tensor(0.1))
    b.load_state_dict(saved)
    assert b.param_groups[0]["lr"] == 0.5 and b.param_groups[0]["betas"] == (0.5, 0.75)
    for p, q in zip(params, mine):
        state = b.state[q]
        assert state["step"].dtype == torch.float32 and state["step"].numel() == 1 and state["step"] == 1
        for name in ("exp_avg", "exp_avg_sq"):
            assert state[name].dtype == torch.float32 and state[name].stride() == q.stride() and not state[name].requires_grad
            assert torch.equal(state[name], a.state[p][name].float())


def test_optimizer_can_be_copied_and_pickled():
    import copy
    import pickle
    a = optim.AdamW([torch.nn.Parameter(torch.zeros(3))], lr=0.5, max_norm=0.25, state_bits=8, min_8bit_size=7, seed=11)
    for b in (copy.deepcopy(a), pickle.loads(pickle.dumps(a))):
        assert (b.max_norm, b.state_bits, b.min_8bit_size, b.seed, b.param_groups[0]["lr"]) == (0.25, 8, 7, 11, 0.5)


def test_layer_norm_refuses_forward_mode_derivatives():
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            norm.layer_norm(fwd.make_dual(meta(2, 8), meta(2, 8)), 8)


def test_convert_layer_norm_keeps_parameters_and_leaves_subclasses_alone():
    class Own(torch.nn.LayerNorm):
        pass
    m = torch.nn.Sequential(torch.nn.LayerNorm(4), torch.nn.Sequential(Own(4), torch.nn.LayerNorm((2, 4), bias=False)))
    keys, weight = list(m.state_dict()), m[0].weight
    assert norm.convert_layer_norm(m) == 2
    assert type(m[0]) is norm.LayerNorm and type(m[1][0]) is Own and type(m[1][1]) is norm.LayerNorm
    assert m[0].weight is weight and list(m.state_dict()) == keys
    assert norm.convert_layer_norm(m) == 0


# ---- refusals of the C ABI: every one is decided before anything is launched ------------------------------------
INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -3
SOME = 1 << 20          # an aligned address that nothing ever reads: each call below is refused first


def norm_params(**kw):
    d = dict(rows=4, cols=8, x_stride=8, dy_stride=8, x_type=L.SV3D_F32, y_type=L.SV3D_F32, param_type=L.SV3D_F32, eps=1e-5)
    d.update(kw)
    return L.LayerNormParams(**d)


@pytest.mark.parametrize("kw, x, status", [
    (dict(rows=-1), SOME, INVALID), (dict(cols=0), SOME, INVALID), (dict(x_stride=-1), SOME, INVALID),
    (dict(x_type=3), SOME, INVALID), (dict(x_type=L.SV3D_F16, y_type=L.SV3D_BF16), SOME, INVALID),
    (dict(param_type=L.SV3D_F16), SOME, INVALID), (dict(eps=-1.0), SOME, INVALID), (dict(eps=math.nan), SOME, INVALID),
    (dict(cols=(1 << 24) + 1), SOME, UNSUPPORTED), (dict(), None, INVALID),
])
def test_abi_layer_norm_refuses(kw, x, status):
    lib = L.lib()
    p = norm_params(**kw)
    assert lib.sv3d_layer_norm_forward(ctypes.byref(p), x, None, None, SOME, None, None, None) == status
    assert lib.sv3d_layer_norm_backward(ctypes.byref(p), x, SOME, None, SOME, SOME, SOME, None, None, None, 0, None) == status


def test_abi_layer_norm_workspace_and_empty_calls():
    lib = L.lib()
    p = norm_params()
    for odd in range(5):                                # addresses off their element's size
        a = [SOME + 1 if i == odd else SOME for i in range(5)]
        assert lib.sv3d_layer_norm_forward(ctypes.byref(p), a[0], a[1], a[2], a[3], a[4], SOME, None) == INVALID
        assert lib.sv3d_layer_norm_backward(ctypes.byref(p), a[0], a[1], a[2], SOME, SOME, a[3], a[4], None, SOME, 1 << 30, None) == INVALID
    assert lib.sv3d_layer_norm_forward(None, SOME, None, None, SOME, None, None, None) == INVALID
    p, n = norm_params(), ctypes.c_size_t()
    assert lib.sv3d_layer_norm_workspace(ctypes.byref(p), None) == INVALID
    assert lib.sv3d_layer_norm_workspace(ctypes.byref(p), ctypes.byref(n)) == 0 and n.value > 0
    back = lambda ws, size: lib.sv3d_layer_norm_backward(ctypes.byref(p), SOME, SOME, None, SOME, SOME, None, SOME, None, ws,  # noqa: E731
                                                        size, None)
    assert back(SOME, n.value - 1) == WORKSPACE
    assert back(SOME + 4, n.value) == INVALID and back(None, n.value) == INVALID
    p = norm_params(rows=0)
    assert lib.sv3d_layer_norm_forward(ctypes.byref(p), None, None, None, None, None, None, None) == 0
    p = norm_params(dy_stride=-8)
    assert lib.sv3d_layer_norm_backward(ctypes.byref(p), SOME, SOME, None, SOME, SOME, SOME, None, None, None, 0, None) == INVALID


def tensor(**kw):
    d = dict(param=SOME, grad=SOME, exp_avg=SOME, exp_avg_sq=SOME, scales=None, step=SOME, numel=10, type=L.SV3D_F32, state_bits=32)
    d.update(kw)
    return L.AdamWTensor(**d)


@pytest.mark.parametrize("kw, status", [
    (dict(param=None), INVALID), (dict(grad=None), INVALID), (dict(exp_avg=None), INVALID), (dict(exp_avg_sq=None), INVALID),
    (dict(step=None), INVALID), (dict(numel=-1), INVALID), (dict(type=7), INVALID), (dict(state_bits=16), INVALID),
    (dict(state_bits=8), INVALID), (dict(param=SOME + 2), INVALID), (dict(exp_avg=SOME + 1), INVALID),
    (dict(numel=(1 << 40) + 1), UNSUPPORTED),
])
def test_abi_adamw_refuses_a_tensor(kw, status):
    p = L.AdamWParams(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8)
    arr = (L.AdamWTensor * 2)(tensor(), tensor(**kw))
    assert L.lib().sv3d_adamw_step(ctypes.byref(p), arr, 2, SOME, 1 << 16, None) == status


@pytest.mark.parametrize("kw, ws, size, status", [
    (dict(beta1=1.0), SOME, 1 << 16, INVALID), (dict(beta2=-0.1), SOME, 1 << 16, INVALID), (dict(eps=-1.0), SOME, 1 << 16, INVALID),
    (dict(eps=math.nan), SOME, 1 << 16, INVALID), (dict(square_sums=SOME, max_norm=-1.0), SOME, 1 << 16, INVALID),
    (dict(), None, 1 << 16, INVALID), (dict(), SOME, 8, WORKSPACE),
])
def test_abi_adamw_refuses_a_call(kw, ws, size, status):
    d = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8)
    d.update(kw)
    p = L.AdamWParams(**d)
    assert L.lib().sv3d_adamw_step(ctypes.byref(p), (L.AdamWTensor * 1)(tensor()), 1, ws, size, None) == status


def test_abi_square_sums_and_moment_values_refuse():
    lib, n = L.lib(), ctypes.c_int32()
    arr = (L.AdamWTensor * 2)(tensor(numel=100000), tensor(numel=0, grad=None))
    assert lib.sv3d_grad_square_sums_count(arr, 2, ctypes.byref(n)) == 0 and n.value > 0
    assert lib.sv3d_grad_square_sums_count(arr, 2, None) == INVALID
    assert lib.sv3d_grad_square_sums_count(None, 2, ctypes.byref(n)) == INVALID
    assert lib.sv3d_grad_square_sums(arr, 2, SOME, n.value + 1, None) == INVALID
    assert lib.sv3d_grad_square_sums(arr, 2, None, n.value, None) == INVALID
    assert lib.sv3d_moment_values(SOME, SOME, SOME, -1, SOME, SOME, None) == INVALID
    assert lib.sv3d_moment_values(SOME, None, SOME, 5, SOME, SOME, None) == INVALID
    assert lib.sv3d_moment_values(None, None, None, 0, None, None, None) == 0
    count, p = ctypes.c_size_t(), L.AdamWParams(beta1=0.9, beta2=0.9, max_norm=1.0)
    assert lib.sv3d_adamw_workspace(ctypes.byref(p), arr, -1, ctypes.byref(count)) == INVALID
    assert lib.sv3d_adamw_workspace(ctypes.byref(p), None, 2, ctypes.byref(count)) == INVALID
    assert lib.sv3d_adamw_workspace(ctypes.byref(p), arr, 2, ctypes.byref(count)) == 0
    clipped = count.value
    p.max_norm = 0.0
    assert lib.sv3d_adamw_workspace(ctypes.byref(p), arr, 2, ctypes.byref(count)) == 0 and clipped - count.value == 8 * n.value
    assert lib.sv3d_adamw_step(ctypes.byref(L.AdamWParams(beta1=0.9, beta2=0.9)), None, 0, None, 0, None) == 0


# ---- the trainer ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("argv, error", [(["--optim", "adamw"], RuntimeError), (["--optim", "adamw8"], RuntimeError),
                                         (["--hip_layer_norm", "1"], RuntimeError), (["--optim", "adamw", "--use_sgd"], ValueError)])
def test_trainer_on_the_host_refuses_what_needs_a_gpu(tmp_path, argv, error):
    from nnutils import train_utils

    class T(train_utils.Trainer):
        def init_dataset(self):
            self.dataloader = []

        def define_model(self):
            self.model = torch.nn.Linear(2, 2)

        def define_criterion(self):
            pass

    o = train_utils.add_training_flags().parse_args(["--checkpoint_dir", str(tmp_path), *argv])
    with pytest.raises(error):
        T(o, env=train_utils.DistEnv()).init_training()


def test_operators_see_the_same_through_torch_ops_and_directly():
    """What `sv3d._call` hands back to torch.ops (a mode that wants to see every function) and what it takes itself."""
    from torch.overrides import TorchFunctionMode
    from sv3d import ops

    class Watch(TorchFunctionMode):
        seen = 0

        def __torch_function__(self, func, types, args=(), kwargs=None):
            Watch.seen += 1
            return func(*args, **(kwargs or {}))

    x = meta(2, 8)
    with Watch():
        y = norm.layer_norm(x, 8)
    assert Watch.seen > 0 and y.shape == x.shape
    args = (x, (8,), None, None, 1e-5, False)
    assert ops._call.layer_norm(*args).shape == (2, 8)
    assert ops._call.layer_norm(*args[:-1]) is NotImplemented
    assert ops._call.layer_norm([x], *args[1:]) is NotImplemented
    assert ops._call.layer_norm(x, 8, *args[2:]) is NotImplemented
    assert ops._call.grad_square_sums((x, None)) is NotImplemented
    assert ops._call.grad_square_sums((x, x)).dtype == torch.float64
    p = torch.nn.Parameter(meta(5))
    with pytest.raises(RuntimeError, match="no_grad"):
        torch.ops.sv3d.adamw_step([p], [meta(5)], [meta(5)], [meta(5)], [], [meta()], None, None, None, None, 1e-3, 0.9, 0.9,
                                  1e-8, 0.0, 0.0, False, 0)
    assert optim.adamw_step([p], [meta(5)], [meta(5)], [meta(5)], [meta()]) is None
