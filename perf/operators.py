"""The training-step operators on their own: layer norm (forward, and forward with backward) and the AdamW
step over many tensors with 32-bit or 8-bit states, unscaling and clipping included.

`own = False` computes them in plain torch operations, `own = True` through `sv3d`.  Sizes come from the
networks this repository trains (examples/cmr_synthetic.py: encoder, code of 200, heads, part basis) and from the
transformer camera head of the reference's network (256 image tokens and 8 queries per image, width 512), plus
generic wide and large ones.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LR, BETA1, BETA2, ADAM_EPS, DECAY = 1e-4, 0.9, 0.999, 1e-8, 0.01
NORM_EPS = 1e-5
ALIGN = 256                 # every tensor of a list starts at a multiple of this many elements
BLOCK = 128                 # elements that share the scales of their 8-bit states
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _sv3d():
    pkg = os.path.join(ROOT, "single-view-3d-reconstruction_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import sv3d
    return sv3d


# ---- cases ------------------------------------------------------------------------------------
def listed():
    norm = lambda name, rows, cols, dtype, train: {  # noqa: E731
        "name": name, "op": "layer_norm", "rows": rows, "cols": cols, "dtype": dtype, "train": train}
    adam = lambda name, layout, width, bits, dtype, clip, scaled: {  # noqa: E731
        "name": name, "op": "adamw", "layout": layout, "width": width, "bits": bits, "dtype": dtype,
        "clip": clip, "scaled": scaled}
    return [
        # the eight camera queries of one image: a call that is all latency
        norm("norm_queries", 8, 512, "float32", False),
        # the 200-wide image code of 64 images and their mirror images
        norm("norm_code_train", 128, 200, "float32", True),
        # 256 tokens + 8 queries of 16 images (batch 8 and mirror images), full precision
        norm("norm_tokens_train", 4224, 512, "float32", True),
        # odd rows and an odd width, half precision
        norm("norm_odd_train", 5003, 1337, "float16", True),
        # the tokens of 128 images at inference
        norm("norm_tokens_infer", 32768, 512, "bfloat16", False),
        # a wide network's activations
        norm("norm_wide_train", 16384, 4096, "bfloat16", True),
        # the part basis: one small tensor with its own optimizer
        adam("adamw_parts", "parts", 642, 32, "float32", 0.1, False),
        # encoder of the synthetic network (ResNet-18 trunk and code layers), clipped, fp16 loss scale
        adam("adamw_encoder", "encoder", 64, 32, "float32", 0.1, True),
        # the whole synthetic network: encoder and heads, 62 M weights
        adam("adamw_model", "model", 64, 32, "float32", 0.1, True),
        # the rehearsal encoder (an eighth of the channels) with 8-bit states
        adam("adamw8_small_encoder", "encoder", 8, 8, "float32", 0.1, True),
        # the whole synthetic network with 8-bit states
        adam("adamw8_model", "model", 64, 8, "float32", 0.1, True),
        # 16-bit weights of two 8192 x 8192 layers and what is around them, not clipped
        adam("adamw8_large", "large", 8192, 8, "bfloat16", 0.0, False),
    ]


def draw(rng):
    log = lambda a, b: int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))  # noqa: E731
    if rng.random() < 0.5:
        cols = log(8, 8192)
        return {"op": "layer_norm", "rows": log(1, min(65536, (1 << 26) // cols)), "cols": cols,
                "dtype": rng.choice(sorted(TYPES)), "train": rng.random() < 0.7}
    tensors = log(1, 200)
    return {"op": "adamw", "layout": "spread", "width": log(max(1000, 8 * tensors), 60_000_000), "tensors": tensors,
            "bits": rng.choice([8, 32]), "dtype": rng.choice(["float32", "float32", "bfloat16"]),
            "clip": rng.choice([0.0, 0.1, 1.0]), "scaled": rng.random() < 0.5}


def sizes(case):
    """Elements of each tensor of an AdamW case."""
    w, layout = case["width"], case["layout"]
    if layout == "parts":
        return [w * 8]
    if layout == "large":
        return [w * w, w, w * w, w, 4099, 1]
    if layout == "spread":          # sizes fall geometrically, as a network's do from heads to norms; most are odd
        n = case["tensors"]
        share = [0.5 ** (12 * k / n) for k in range(n)]
        return [max(1, int(w * s / sum(share))) | (k % 3 != 0) for k, s in enumerate(share)]
    stages = [(w, w, 1), (w, 2 * w, 2), (2 * w, 4 * w, 2), (4 * w, 8 * w, 2)]
    block = lambda a, b, down: [9 * a * b, b, b, 9 * b * b, b, b] + ([a * b, b, b] if down else [])  # noqa: E731
    encoder = [3 * 49 * w, w, w] + sum([block(a, b, s > 1) + block(b, b, False) for a, b, s in stages], [])
    encoder += [8 * w * 4 * w * 16, 4 * w, 4 * w, 4 * w, 64 * w * 200, 200, 200, 200, 200 * 200, 200, 200, 200]
    if layout == "encoder":
        return encoder
    heads = [(1926, 200), (56, 200), (8, 200), (512, 200), (1280 * 36 * 2, 512)]
    return encoder + sum([[o * i, o] for o, i in heads], [])


# ---- inputs -----------------------------------------------------------------------------------
def prepare(case, seed):
    dev = _device()
    g = torch.Generator(device=dev).manual_seed(int(seed))
    normal = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    t = TYPES[case["dtype"]]
    if case["op"] == "layer_norm":
        rows, cols = case["rows"], case["cols"]
        # activations whose channels have their own level and spread, weights near one
        x = (normal(rows, cols) * (0.5 + normal(cols).abs()) + 0.5 * normal(cols)).to(t)
        w, b = 1 + 0.1 * normal(cols), 0.1 * normal(cols)
        s = {"x": x, "w": w, "b": b}
        if case["train"]:
            s = {k: v.requires_grad_() for k, v in s.items()}
            s["dy"] = normal(rows, cols).to(t)
        return s
    ns = sizes(case)
    at, total = [], 0
    for n in ns:
        at.append(total)
        total += -(-n // ALIGN) * ALIGN
    # one flat buffer of each kind; the lists that the operator gets are views of them.  What lies between two
    # tensors is zero everywhere and stays so
    live = torch.zeros(total, dtype=torch.bool, device=dev)
    index = torch.zeros(total, dtype=torch.int64, device=dev)
    for a, n in zip(at, ns):
        live[a:a + n] = True
        index[a:a + n] = torch.arange(n, device=dev)
    scale = 1024.0 if case["scaled"] else 1.0
    # gradients of very different size from one group of elements to the next, about one in all (a logarithm spread
    # like this has a root mean square of 14); in one part in 64 none at all (what a mask leaves out).  The moments
    # are those of earlier gradients of that size, after clipping.
    size = 10.0 ** normal((total + 63) // 64).repeat_interleave(64)[:total] * live / (14.2 * math.sqrt(sum(ns)))
    size = size * (torch.rand((total + 31) // 32, generator=g, device=dev) > 1 / 64).repeat_interleave(32)[:total]
    past = size * min(1.0, case["clip"] or 1.0)
    p = 0.05 * normal(total) * live
    m = 0.3 * normal(total) * past
    v = (0.5 + torch.rand(total, generator=g, device=dev)) * past * past
    s = {"p": p.to(t), "g": (normal(total) * size * scale).to(t), "index": index, "steps": torch.full((len(ns),), 100.0, device=dev),
         "clip": case["clip"], "seed": int(seed) & 0xFFFF, "bits": case["bits"],
         "scale": torch.full((), scale, device=dev) if case["scaled"] else None,
         "found_inf": torch.zeros((), device=dev) if case["scaled"] else None}
    if case["bits"] == 8:
        half = torch.full((total,), 32768, dtype=torch.int32, device=dev)
        cm, em = _encode_first(m, half)
        cv, ev = _encode_second(v, half)
        s["m"], s["v"], s["e"] = cm, cv, torch.stack([em, ev], 1).contiguous()
    else:
        s["m"], s["v"] = m, v
    cut = lambda x: [x[a:a + n] for a, n in zip(at, ns)]  # noqa: E731
    s["lists"] = {k: cut(s[k]) for k in "pgmv"}
    s["lists"]["steps"] = [s["steps"][k] for k in range(len(ns))]
    s["lists"]["e"] = [s["e"][a // BLOCK:a // BLOCK + -(-n // BLOCK)] for a, n in zip(at, ns)] if case["bits"] == 8 else None
    return s


# ---- 8-bit states in torch operations -----------------------------------------------------------
# Blocks of 128 elements.  The first moment is held as sign, 4 exponent and 3 mantissa bits, the second as 5 exponent
# and 3 mantissa bits, both times a power of two of the block's own (one byte: the exponent of its largest value).
def _dither(index, step, seed):
    """16 + 16 bits of a hash of (element, step, seed): what is added below the last kept bit before cutting."""
    mask = 0xFFFFFFFF
    key = (step * 0x9E3779B1 + seed * 0x6A09E667) & mask
    x = (index + key) & mask
    x = (x ^ (x >> 16)) * 0x6A09E667 & mask
    x = (x ^ (x >> 15)) * 0xBB67AE85 & mask
    x = x ^ (x >> 16)
    return (x >> 16).to(torch.int32), (x & 0xFFFF).to(torch.int32)


def _power(e):
    return ((e + 127) << 23).view(torch.float32)


def _block_exponent(a, lowest):
    top = a.view(-1, BLOCK).amax(1)
    return (top.view(torch.int32) >> 23).clamp(min=lowest)


def _cut(t, dither, lowest):
    """Magnitudes -> codes: 2**lowest is the smallest normal value, three mantissa bits stay."""
    small = t < 2.0 ** lowest
    t = torch.where(small, t + 2.0 ** lowest, t)
    return ((t.view(torch.int32) + (dither << 4) + 8) >> 20) - ((126 + lowest) << 3) - 8 * small.to(torch.int32)


def _encode_first(m, dither):
    a = torch.where(m.isfinite(), m.abs(), 0.0)
    e = _block_exponent(a, 20)
    code = _cut((a.view(-1, BLOCK) * _power(134 - e)[:, None]).view(-1), dither, -6)
    code = torch.where(m.isfinite(), code, 127) | (m.signbit().to(torch.int32) << 7)
    return code.to(torch.uint8), e.to(torch.uint8)


def _encode_second(v, dither):
    a = torch.where(v.isfinite(), v, 0.0)
    e = _block_exponent(a, 34)
    code = _cut((a.view(-1, BLOCK) * _power(142 - e)[:, None]).view(-1), dither, -14)
    code = torch.where(a > 0, code.clamp(min=1), code)
    return torch.where(v.isfinite(), code, 255).to(torch.uint8), e.to(torch.uint8)


def _decode_first(code, e):
    value = code.view(torch.float8_e4m3fn).to(torch.float32)
    return (value.view(-1, BLOCK) * _power(e.to(torch.int32) - 134)[:, None]).view(-1)


def _decode_second(code, e):
    c = code.to(torch.int32)
    small = c < 8
    value = ((c + 8 * (112 + small.to(torch.int32))) << 20).view(torch.float32)
    value = torch.where(small, value - 2.0 ** -14, value)
    value = torch.where(c == 255, math.nan, value)
    return (value.view(-1, BLOCK) * _power(e.to(torch.int32) - 142)[:, None]).view(-1)


# ---- the operators ------------------------------------------------------------------------------
def run(state):
    if "x" in state:
        return _norm(state)
    return _adamw_own(state) if own else _adamw(state)


def _norm(s):
    x, w, b, dy = s["x"], s["w"], s["b"], s.get("dy")
    if own:
        sv3d = _sv3d()
        y = sv3d.layer_norm(x, (x.shape[-1],), w, b, NORM_EPS)
        if dy is None:
            return y
        dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    with torch.no_grad():
        f = x.float()
        c = f - f.mean(1, keepdim=True)
        r = (c.square().mean(1, keepdim=True) + NORM_EPS).rsqrt()
        h = c * r
        y = (h * w + b).to(x.dtype)
        if dy is None:
            return y
        d = dy.float()
        u = d * w
        dx = (u - u.mean(1, keepdim=True) - h * (u * h).mean(1, keepdim=True)) * r
        # rows are summed in 64 bits: there are thousands of them, and their signs differ
        return {"y": y, "dx": dx.to(x.dtype), "dw": (d * h).sum(0, dtype=torch.float64).float(),
                "db": d.sum(0, dtype=torch.float64).float()}


def _adamw(s):
    """All tensors at once: the flat buffers, with zeros between the tensors."""
    p, g, steps = s["p"], s["g"].float(), s["steps"]
    unscale = 1.0 / s["scale"].double() if s["scale"] is not None else torch.ones((), dtype=torch.float64, device=p.device)
    go = s["found_inf"] == 0 if s["found_inf"] is not None else True
    kept = (lambda new, old: torch.where(go, new, old)) if s["found_inf"] is not None else lambda new, old: new
    out = {}
    if s["clip"] > 0:
        norm = g.double().square().sum().sqrt() * unscale
        out["norm"] = norm.float()
        unscale = unscale * (s["clip"] / (norm + 1e-6)).clamp(max=1.0)
    g = g * unscale.float()
    steps.add_(go)
    t = steps[0].double()
    rate, root = (LR / (1 - BETA1 ** t)).float(), (1 / (1 - BETA2 ** t).sqrt()).float()
    if s["bits"] == 8:
        m, v = _decode_first(s["m"], s["e"][:, 0]), _decode_second(s["v"], s["e"][:, 1])
    else:
        m, v = s["m"], s["v"]
    m1 = BETA1 * m + (1 - BETA1) * g
    v1 = BETA2 * v + (1 - BETA2) * (g * g)
    p1 = p.float()
    p1 = p1 * (1 - LR * DECAY) - rate * (m1 / (v1.sqrt() * root + ADAM_EPS))
    p.copy_(kept(p1.to(p.dtype), p))
    if s["bits"] == 8:
        du, dv = _dither(s["index"], steps[0].long(), s["seed"])
        cm, em = _encode_first(m1, du)
        cv, ev = _encode_second(v1, dv)
        s["m"].copy_(kept(cm, s["m"]))
        s["v"].copy_(kept(cv, s["v"]))
        s["e"].copy_(kept(torch.stack([em, ev], 1), s["e"]))
        m1, v1 = (_decode_first(s["m"], s["e"][:, 0]).bfloat16(), _decode_second(s["v"], s["e"][:, 1]).bfloat16())
    else:
        m1, v1 = m.copy_(kept(m1, m)), v.copy_(kept(v1, v))
    return {**out, "p": p, "m": m1, "v": v1, "steps": steps}


def _adamw_own(s):
    optim = _sv3d().optim
    a = s["lists"]
    norm = optim.adamw_step(a["p"], a["g"], a["m"], a["v"], a["steps"], scales=a["e"], lr=LR, betas=(BETA1, BETA2),
                            eps=ADAM_EPS, weight_decay=DECAY, max_norm=s["clip"], grad_scale=s["scale"],
                            found_inf=s["found_inf"], seed=s["seed"])
    m, v = s["m"], s["v"]
    if s["bits"] == 8:      # both moments as the values that their codes stand for
        m, v = optim.moment_values(m, v, s["e"])
    return {**({"norm": norm} if s["clip"] > 0 else {}), "p": s["p"], "m": m, "v": v, "steps": s["steps"]}


# ---- what a pass cannot do without ----------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "layer_norm":
        n, c = case["rows"] * case["cols"], case["cols"]
        return {"bytes": n * size * (4 if case["train"] else 2) + 4 * c * (4 if case["train"] else 2),
                "flops": n * (22 if case["train"] else 8)}
    n = sum(sizes(case))
    # weights and moments read and written, gradients read; 8-bit states also come back as 16-bit values
    states = 16 if case["bits"] == 32 else 4 + 4 / BLOCK + 4
    return {"bytes": n * (3 * size + states), "flops": n * 20}


# ---- from the definitions, in 64 bits -------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_norm(case, s) if case["op"] == "layer_norm" else _exact_adamw(case, s)


def _exact_norm(case, s):
    x, w, b = s["x"].detach().double(), s["w"].detach().double(), s["b"].detach().double()
    var, mu = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
    sd = (var + NORM_EPS).sqrt()
    hat = (x - mu) / sd
    y = hat * w + b
    if not case["train"]:
        return y
    dy = s["dy"].double()
    dhat = dy * w
    n = case["cols"]
    # d hat_j / d x_i = (delta_ij - 1/n - hat_i hat_j / n) / sd
    along = (dhat * hat).sum(1, keepdim=True) / n
    dx = (dhat - dhat.sum(1, keepdim=True) / n - hat * along) / sd
    return {"y": y, "dx": dx, "dw": (dy * hat).sum(0), "db": dy.sum(0)}


def _exact_adamw(case, s):
    g = s["g"].double()
    if s["scale"] is not None:
        g = g / s["scale"].double()
    out = {}
    if case["clip"] > 0:
        out["norm"] = torch.linalg.vector_norm(g)
        g = g * min(1.0, case["clip"] / (float(out["norm"]) + 1e-6))
    t = 101
    codes = case["bits"] == 8
    m, v = s["m"], s["v"]
    if codes:
        # what each of the 256 codes stands for, looked up
        first = [(-1) ** (c >> 7) * (((c & 7) / 8 + 1) * 2.0 ** ((c >> 3 & 15) - 7) if c & 0x78 else (c & 7) / 8 * 2.0 ** -6)
                 for c in range(256)]
        second = [((c & 7) / 8 + 1) * 2.0 ** ((c >> 3) - 15) if c >> 3 else (c & 7) / 8 * 2.0 ** -14 for c in range(256)]
        table = lambda x: torch.tensor(x, dtype=torch.float64, device=g.device)  # noqa: E731
        first, second = table(first), table(second)
        wide = lambda e, bias: (2.0 ** (e.double() - bias)).repeat_interleave(BLOCK)  # noqa: E731
        m = first[m.long()] * wide(s["e"][:, 0], 134)
        v = second[v.long()] * wide(s["e"][:, 1], 142)
    m = BETA1 * m.double() + (1 - BETA1) * g
    v = BETA2 * v.double() + (1 - BETA2) * g * g
    p = s["p"].double() * (1 - LR * DECAY) - LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + ADAM_EPS)
    if codes:
        key = (t * 0x9E3779B1 + s["seed"] * 0x6A09E667) % 2 ** 32
        h = (s["index"] + key) % 2 ** 32
        h = (h ^ (h >> 16)) * 0x6A09E667 % 2 ** 32
        h = (h ^ (h >> 15)) * 0xBB67AE85 % 2 ** 32
        h = h ^ (h >> 16)
        m = _exact_round(m, first[:0x79], h // 65536, 134, 20, 7.0)
        v = _exact_round(v, second[:0xf9], h % 65536, 142, 34, 15.0)
    return {**out, "p": p, "m": m, "v": v, "steps": s["steps"].double() + 1}


def _exact_round(x, values, dither, bias, lowest, top):
    """Up to the next value where the part of the way to it that x has gone and the dither's part add up to one."""
    a = x.abs().view(-1, BLOCK)
    big = a.amax(1)
    exponent = torch.where(big > 0, torch.frexp(big)[1] - 1 + 127, lowest).clamp(min=lowest).double()
    unit = 2.0 ** (exponent - bias)
    a = (a / unit[:, None]).view(-1).contiguous()
    at = (torch.searchsorted(values, a, right=True) - 1).clamp(0, values.numel() - 2)
    low, high = values[at], values[at + 1]
    up = (a - low) / (high - low) + (dither.double() + 0.5) / 65536 >= 1
    got = torch.where(up, high, low)
    if top == 15.0:         # the second moment: nothing above zero becomes zero
        got = torch.where((x > 0) & (got == 0), values[1], got)
    return (got.view(-1, BLOCK) * unit[:, None]).view(-1) * x.sign()
