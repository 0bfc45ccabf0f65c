"""Layer norm and the AdamW step in float64 on the CPU, from their definitions: what the training-step kernels are
checked against.  Test infrastructure only.

Each function also returns bounds on what a float32 evaluation may be off by.  They count roundings (half a step of
float32 is 2**-24 of the value) and are derived for any order of summation whose longest chain of additions is `depth`.
"""
import math

import torch

F32 = 2.0 ** -24


# ---- layer norm -----------------------------------------------------------------------------------------
def layer_norm(x, weight, bias, eps):
    """x [rows, cols] (float64).  Returns y, mean, rstd, h and the bounds of a float32 evaluation: of h, of y before
    it is stored, and of the statistics."""
    cols = x.shape[1]
    depth = 40 + cols / 512             # at most 32 per lane or cols/1024 per thread, then a tree; doubled
    mu = x.mean(1, keepdim=True)
    c = x - mu
    var = (c * c).mean(1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    h = c * r
    w = torch.ones(cols, dtype=x.dtype) if weight is None else weight
    b = torch.zeros(cols, dtype=x.dtype) if bias is None else bias
    y = h * w + b
    e_mu = depth * F32 * x.abs().mean(1, keepdim=True)
    # the mean's error enters the variance squared, a rounding of c twice
    e_r = r * (0.5 * ((depth + 6) * F32 * var + e_mu * e_mu + 2 * F32 * eps) * r * r + 3 * F32)
    e_h = r * (e_mu + F32 * c.abs()) + c.abs() * e_r + F32 * h.abs()
    e_y = w.abs() * e_h + 2 * F32 * (h * w).abs() + F32 * (b.abs() + y.abs())
    return {"y": y, "mean": mu[:, 0], "rstd": r[:, 0], "h": h, "e_h": e_h, "e_y": e_y, "e_mean": e_mu[:, 0],
            "e_rstd": e_r[:, 0]}


def layer_norm_backward(f, dy, weight):
    """Gradients for `f` = layer_norm(...) and their bounds (before they are stored)."""
    h, e_h = f["h"], f["e_h"]
    r, e_r = f["rstd"][:, None], f["e_rstd"][:, None]
    rows, cols = h.shape
    depth, down = 40 + cols / 512, 80 + rows / 64
    u = dy if weight is None else dy * weight
    mu_u, mu_uh = u.mean(1, keepdim=True), (u * h).mean(1, keepdim=True)
    dx = r * (u - mu_u - h * mu_uh)
    e_uh = depth * F32 * (u * h).abs().mean(1, keepdim=True) + (u.abs() * e_h).mean(1, keepdim=True)
    e_in = (F32 * (4 * u.abs() + 2 * mu_u.abs()) + depth * F32 * u.abs().mean(1, keepdim=True)
            + e_h * mu_uh.abs() + h.abs() * e_uh + 3 * F32 * (h * mu_uh).abs())
    e_dx = r * e_in + (dx / r).abs() * e_r + 2 * F32 * dx.abs()
    dw, db = (dy * h).sum(0), dy.sum(0)
    e_dw = (dy.abs() * e_h).sum(0) + down * F32 * (dy * h).abs().sum(0)
    e_db = down * F32 * dy.abs().sum(0)
    return {"dx": dx, "dw": dw, "db": db, "e_dx": e_dx, "e_dw": e_dw, "e_db": e_db}


# ---- 8-bit moments ----------------------------------------------------------------------------------------
BLOCK = 128
#: smallest normal exponent, largest code, what a scale byte is away from the exponent of the unit, lowest scale byte
FIRST = {"lowest": -6, "nan": 0x7f, "bias": 134, "floor": 20}
SECOND = {"lowest": -14, "nan": 0xff, "bias": 142, "floor": 34}


def code_values(kind):
    """What the codes 0 .. nan-1 stand for, ascending, in units of the block's power of two."""
    low = kind["lowest"]
    return torch.tensor([(c & 7) / 8 * 2.0 ** low if c < 8 else (1 + (c & 7) / 8) * 2.0 ** ((c >> 3) - 1 + low)
                         for c in range(kind["nan"])], dtype=torch.float64)


def _units(scale_bytes, n, kind):
    e = scale_bytes.double().clamp(min=kind["floor"])
    return (2.0 ** (e - kind["bias"])).repeat_interleave(BLOCK)[:n]


def decode(codes, scale_bytes, kind):
    """codes uint8 [n], scale_bytes uint8 [ceil(n/128)] -> float64 [n]."""
    c = codes.long()
    sign = torch.ones(len(c), dtype=torch.float64)
    if kind is FIRST:
        sign = torch.where(c >= 128, -1.0, 1.0).double()
        c = c & 127
    values = torch.cat([code_values(kind), torch.tensor([math.nan], dtype=torch.float64)])
    return sign * values[c.clamp(max=kind["nan"])] * _units(scale_bytes, len(codes), kind)


def dither(n, step, seed):
    """The 32-bit hash of (element, step, seed) as int64 [n]; its upper half rounds the first moment, its lower one
    the second."""
    wrap = 2 ** 32
    x = (torch.arange(n) + step * 0x9E3779B1 + seed * 0x6A09E667) % wrap
    x = (x ^ (x >> 16)) * 0x6A09E667 % wrap
    x = (x ^ (x >> 15)) * 0xBB67AE85 % wrap
    return x ^ (x >> 16)


def scale_bytes_of(x, kind):
    """The byte of each block: the exponent of its largest finite magnitude."""
    a = torch.where(torch.isfinite(x), x.abs(), 0.0)
    a = torch.nn.functional.pad(a, (0, -len(a) % BLOCK)).view(-1, BLOCK).amax(1)
    return torch.where(a > 0, torch.frexp(a)[1] + 126, 0).clamp(min=kind["floor"])


def rounded(x, scale_bytes, kind, part):
    """The values between which x (float64 [n]) is rounded and how far the way up plus the dither is from the border
    (below 0: down), given the blocks' bytes; `part` [n]: the 16 dither bits."""
    values, unit = code_values(kind), _units(scale_bytes, len(x), kind)
    a = (x.abs() / unit).contiguous()
    at = (torch.searchsorted(values, a, right=True) - 1).clamp(0, len(values) - 2)
    low, high = values[at], values[at + 1]
    over = (a - low) / (high - low) + (part.double() + 0.5) / 65536 - 1
    if kind is SECOND:
        low = torch.where(a > 0, low.clamp(min=float(values[1])), low)
        high = torch.maximum(high, low)
    return low * unit * x.sign(), high * unit * x.sign(), over, (values[at + 1] - values[at]) * unit


# ---- AdamW --------------------------------------------------------------------------------------------------
def adamw(p, g, m, v, step, *, lr, betas, eps, weight_decay, scale=1.0, clip=1.0, maximize=False):
    """One step in float64 from moments `m`, `v`; `step` counts the steps before this one.  `scale`, `clip`: what the
    gradients are divided and multiplied by.  Returns the new values and the bounds of a float32 evaluation."""
    b1, b2 = betas
    t = step + 1
    g = g / scale * clip * (-1 if maximize else 1)
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    rate, root = lr / (1 - b1 ** t), 1 / math.sqrt(1 - b2 ** t)
    den = torch.sqrt(v1) * root + eps
    u = rate * m1 / den
    p1 = p * (1 - lr * weight_decay) - u
    # per product: the factor's own rounding, g's factor, the product's, the sum's
    e_m = 4 * F32 * ((b1 * m).abs() + ((1 - b1) * g).abs())
    e_v = 6 * F32 * v1 + 2.0 ** -140        # squares below the smallest normal number lose digits
    e_den = torch.sqrt(v1) * root * 6 * F32 + root * torch.minimum(torch.sqrt(e_v), e_v / torch.sqrt(v1).clamp(min=1e-300)) + 2 * F32 * den
    e_u = rate * e_m / den + u.abs() * (e_den / den + 6 * F32)
    e_p = e_u + 3 * F32 * p.abs() + F32 * p1.abs()
    return {"p": p1, "m": m1, "v": v1, "e_p": e_p, "e_m": e_m, "e_v": e_v}


def clip_factor(norm, max_norm):
    c = max_norm / (norm + 1e-6)
    return 1.0 if c > 1.0 else c
