"""Cases of a normalised, clipped training step: group norm with an activation, the
global gradient norm, clipping by it, and the AdamW step that clips.

Each case runs in two forms on the same inputs: elementary torch operations
(``own`` false), and the calls a user makes of matrixman_b200 (``own`` true).
Everything is float32, the framework's compute type; optimiser states are held
in 32 or in 8 bits.  Feature maps are channels last.
"""

import math

import torch

own = False

EPS = 1e-5                      # group norm
CLIP_EPS = 1e-6                 # added to the norm that gradients are divided by
LR, BETA1, BETA2, ADAM_EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
STEPS_DONE = 20                 # optimiser steps before the measured one
BLOCK = 256                     # elements that share a scale of the 8-bit states
SMOOTH = ["none", "silu", "sigmoid", "gelu", "gelu_tanh"]
ACTS = SMOOTH + ["relu"]  # forward only: ReLU's slope jumps at 0, so a value one rounding from it has two answers


def listed():
    return [
        # The coarsest level of a detector, one image: the call's latency.
        {"name": "group norm 1x64x20x20", "op": "group_norm", "n": 1, "c": 64, "h": 20, "w": 20, "groups": 16,
         "act": "silu", "train": False},
        # The detector's 80 x 80 level at the batch that the framework's benchmark runs.
        {"name": "group norm 64x64x80x80", "op": "group_norm", "n": 64, "c": 64, "h": 80, "w": 80, "groups": 16,
         "act": "silu", "train": False},
        # Full-resolution features of an image decoder: a group is larger than an SM's memory.
        {"name": "group norm 2x128x512x512", "op": "group_norm", "n": 2, "c": 128, "h": 512, "w": 512, "groups": 32,
         "act": "silu", "train": False},
        # A training batch of odd feature maps, groups that do not divide into 16 bytes.
        {"name": "group norm train 5x130x37x41", "op": "group_norm", "n": 5, "c": 130, "h": 37, "w": 41, "groups": 13,
         "act": "gelu_tanh", "train": True},
        # Features of a linear layer, no pixels: a training batch of rows.
        {"name": "group norm train 4096x512", "op": "group_norm", "n": 4096, "c": 512, "h": 1, "w": 1, "groups": 8,
         "act": "gelu", "train": True},
        # A training batch at the resolution of the detector's second stage: the largest norm.
        {"name": "group norm train 16x128x160x160", "op": "group_norm", "n": 16, "c": 128, "h": 160, "w": 160,
         "groups": 32, "act": "silu", "train": True},
        # Watching the gradients of the framework's MLP: six small tensors, latency.
        {"name": "gradient norm mlp", "op": "norm", "p": "2", "layers": 0, "width": 0, "packed": False},
        # The same of six blocks of odd width, gradients packed one after the other (not 16-byte aligned).
        {"name": "gradient norm packed 6x1001", "op": "norm", "p": "2", "layers": 6, "width": 1001, "packed": True},
        # Clipping before the step of the framework's MLP.
        {"name": "clip mlp", "op": "clip", "p": "2", "layers": 0, "width": 0, "packed": False},
        # Clipping the gradients of twelve blocks: 72 tensors, 101 M values.
        {"name": "clip 12x1024", "op": "clip", "p": "2", "layers": 12, "width": 1024, "packed": False},
        # The clipped optimiser step of twelve blocks.
        {"name": "clipped adamw 32-bit 12x1024", "op": "adamw", "bits": 32, "layers": 12, "width": 1024,
         "packed": False},
        # The same of the framework's MLP with states in 8 bits.
        {"name": "clipped adamw 8-bit mlp", "op": "adamw", "bits": 8, "layers": 0, "width": 0, "packed": False},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["group_norm", "group_norm", "norm", "clip", "adamw"])
    if op == "group_norm":
        train = rng.random() < 0.6
        groups = _spread(rng, 1, 64)
        c = groups * _spread(rng, 1, max(1, 1024 // groups))
        most = (1 << 25) // c
        h = _spread(rng, 1, min(512, most))
        w = _spread(rng, max(1, h // 2), min(2 * h, max(1, most // h)))
        return {"op": op, "n": _spread(rng, 1, max(1, min(8192, most // (h * w)))), "c": c, "h": h, "w": w,
                "groups": groups, "act": rng.choice(SMOOTH if train else ACTS), "train": train}
    case = {"op": op, "layers": rng.randint(1, 12), "width": _spread(rng, 20, 1024), "packed": rng.random() < 0.5}
    if op == "adamw":
        case["bits"] = rng.choice([32, 8])
    else:
        case["p"] = rng.choice(["2", "2", "1", "inf"])
    return case


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

class _Span:
    """A dense device buffer of the framework, as torch sees it."""

    def __init__(self, t, shape=None):
        kind = {torch.float32: "<f4", torch.int64: "<i8"}[t.dtype]
        self.owner = t
        self.__cuda_array_interface__ = {"shape": tuple(t.shape) if shape is None else shape, "typestr": kind,
                                         "data": (t.element_ptr, False), "version": 3, "strides": None, "stream": None}


def _torch_view(t, shape=None):
    return torch.as_tensor(_Span(t, shape), device="cuda")


def _framework(t):
    """The framework's tensor with the values of a CUDA tensor."""
    import matrixman_b200 as matrixman
    matrixman.init()
    got = torch.empty(t.shape, dtype=t.dtype, device="matrixman")
    matrixman.synchronize()
    torch.cuda.synchronize()
    _torch_view(got).copy_(t)
    torch.cuda.synchronize()
    return got


def _shapes(case):
    """The tensors that are clipped or stepped: the framework's MLP, or blocks of
    two linear layers (width -> 4 width -> width) and a norm."""
    w = case["width"]
    if not case["layers"]:
        return [(512, 784), (512,), (256, 512), (256,), (10, 256), (10,)]
    return [(4 * w, w), (4 * w,), (w, 4 * w), (w,), (w,), (w,)] * case["layers"]


def _layout(case):
    """(shape, start, elements) of each tensor in a flat buffer, and the buffer's
    length: one right after the other where they are packed, else each at a
    multiple of BLOCK."""
    got, at = [], 0
    for shape in _shapes(case):
        n = math.prod(shape)
        got.append((shape, at, n))
        at += n if case["packed"] and not case.get("bits") == 8 else -(-n // BLOCK) * BLOCK
    return got, at


def _group_norm_inputs(case, g):
    """Feature maps as [n, pixels, c], in the order of channels-last memory."""
    n, c, s = case["n"], case["c"], case["h"] * case["w"]
    # Outputs of a convolution: channels of different scale and offset, a few outliers, bright and dark images.
    x = torch.randn(n, s, c, device="cuda", generator=g)
    x *= (0.3 + torch.rand(c, device="cuda", generator=g)) * (1 + 9 * (torch.rand(c, device="cuda", generator=g) < 0.01))
    x += torch.randn(c, device="cuda", generator=g) + 0.5 * torch.randn(n, 1, 1, device="cuda", generator=g)
    t = {"x": x, "weight": 1 + 0.1 * torch.randn(c, device="cuda", generator=g),
         "bias": 0.1 * torch.randn(c, device="cuda", generator=g)}
    if case["train"]:
        t["grad"] = 1e-2 * torch.randn(n, s, c, device="cuda", generator=g)
    return t


def _tensor_inputs(case, g):
    layout, total = _layout(case)
    names = ("p", "grad", "exp_avg", "exp_avg_sq") if case["op"] == "adamw" else ("grad",)
    t = {k: torch.zeros(total, device="cuda") for k in names}
    for shape, at, n in layout:
        scale = 1e-3 * math.exp(torch.randn((), device="cuda", generator=g).item())
        r = torch.randn(len(names), n, device="cuda", generator=g)
        t["grad"][at:at + n] = scale * r[0]
        if case["op"] == "adamw":
            t["p"][at:at + n] = 0.02 * r[1]
            t["exp_avg"][at:at + n] = 0.2 * scale * r[2]
            t["exp_avg_sq"][at:at + n] = (scale * (0.05 + r[3].abs())) ** 2
    return t


def _limit(case):
    """A limit that these gradients exceed, as in the steep steps that clipping is for."""
    n = sum(math.prod(shape) for shape in _shapes(case))
    return {"2": 2e-4 * math.sqrt(n), "1": 2e-4 * n, "inf": 2e-3}[case.get("p", "2")]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = (_group_norm_inputs if case["op"] == "group_norm" else _tensor_inputs)(case, g)
    s["case"] = dict(case)
    if case["op"] != "group_norm":
        s["layout"], s["limit"] = _layout(case)[0], _limit(case)
    if case["op"] == "adamw":
        s["step"] = STEPS_DONE
        if not own and case["bits"] == 8:
            s["exp_avg_code"], s["exp_avg_scale"] = _encode(s.pop("exp_avg"), 20, 127, 0)
            s["rms_code"], s["rms_scale"] = _encode(s.pop("exp_avg_sq").sqrt(), 19, 255, 1)
    if own:
        for k in [k for k, t in s.items() if isinstance(t, torch.Tensor)]:
            s[k] = _framework(s[k])
        if case["op"] == "group_norm":
            for k in ("x", "grad"):  # [n, c, h, w] over channels-last memory
                if k in s:
                    s[k] = s[k].view(case["n"], case["h"], case["w"], case["c"]).permute(0, 3, 1, 2)
            if case["train"]:
                for k in ("x", "weight", "bias"):
                    s[k].requires_grad_(True)
        else:
            _framework_parameters(s)
    return s


def _framework_parameters(s):
    """The program's parameters, gradients and optimiser over the flat buffers."""
    import matrixman_b200 as matrixman
    case = s["case"]
    part = {k: [s[k][at:at + n].view(shape) for shape, at, n in s["layout"]]
            for k in ("p", "grad", "exp_avg", "exp_avg_sq") if k in s}
    s["params"] = [torch.nn.Parameter(p) for p in part.get("p", part["grad"])]
    for p, grad in zip(s["params"], part["grad"]):
        p.grad = grad
    s["out"] = [_torch_view(s[k]) for k in (("grad",) if case["op"] != "adamw" else ("p", "exp_avg", "exp_avg_sq"))]
    if case["op"] == "adamw":
        bits = case["bits"]
        s["optimizer"] = opt = matrixman.optim.AdamW(s["params"], lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS,
                                                     weight_decay=DECAY, state_bits=bits, max_grad_norm=s["limit"])
        for p, m, v in zip(s["params"], part["exp_avg"], part["exp_avg_sq"]):
            if bits == 8:
                opt.set_state_values(p, m, v, step=s["step"])
            else:
                opt.state[p] = {"step": matrixman.to_device(torch.tensor(float(s["step"]))), "exp_avg": m,
                                "exp_avg_sq": v}
        if bits == 8:
            del s["exp_avg"], s["exp_avg_sq"], s["out"][1:]
    matrixman.synchronize()


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------

def _act(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "sigmoid":
        return torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * torch.special.erfc(-z * math.sqrt(0.5))
    if act == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if act == "sigmoid":
        s = torch.sigmoid(z)
        return s * (1 - s)
    if act == "gelu":
        return 0.5 * torch.special.erfc(-z * math.sqrt(0.5)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        c = 2 * math.sqrt(2 / math.pi)
        s = torch.sigmoid(c * (z + 0.044715 * z * z * z))
        return s + z * s * (1 - s) * c * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def _group_norm_plain(s):
    case = s["case"]
    n, c, px, groups = case["n"], case["c"], case["h"] * case["w"], case["groups"]
    x = s["x"].view(n, px, groups, c // groups)
    w, b = s["weight"].view(groups, -1), s["bias"].view(groups, -1)
    d = x - x.mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt((d * d).mean((1, 3), keepdim=True) + EPS)
    xh = d * rstd
    z = xh * w + b
    y = _act(z, case["act"]).view(n, px, c)
    if not case["train"]:
        return y
    dz = s["grad"].view(x.shape) * _act_slope(z, case["act"])
    g = dz * w
    dx = rstd * (g - g.mean((1, 3), keepdim=True) - xh * (g * xh).mean((1, 3), keepdim=True))
    return [y, dx.view(n, px, c), (dz * xh).sum((0, 1)).view(c), dz.sum((0, 1)).view(c)]


def _total(grad, p):
    """The norm of all gradients together (the gaps of the buffer are zero)."""
    if p == "inf":
        return grad.abs().amax()
    if p == "1":
        return grad.abs().sum(dtype=torch.float64).float()
    return (grad * grad).sum(dtype=torch.float64).sqrt().float()


def _clip_plain(s):
    total = _total(s["grad"], s["case"]["p"])
    s["grad"].mul_((s["limit"] / (total + CLIP_EPS)).clamp(max=1.0))
    s["limit"] *= 0.998
    return [total, s["grad"]]


def _encode(a, shift, top, least):
    """Codes and block scales of the log-linear 8-bit code of optimiser states:
    the magnitude's share of its block's largest, rounded (to even) to the bits
    of a float32 above `shift`, counted down from `top` (1.0)."""
    a = a.view(-1, BLOCK)
    size = a.abs()
    scale = size.amax(1, keepdim=True)
    scale = torch.where(scale < 2.0 ** -126, 0.0, scale)
    bits = (size * (1 / scale)).view(torch.int32)
    code = ((bits + ((1 << (shift - 1)) - 1) + ((bits >> shift) & 1)) >> shift) - (0x3F800000 >> shift) + top
    code = torch.where(size > 0, code.clamp(least, top), 0)
    return torch.where(a < 0, -code, code), scale


def _decode(code, scale, shift, top):
    size = ((code.abs() + (0x3F800000 >> shift) - top) << shift).view(torch.float32)
    value = torch.where(code != 0, size, 0.0) * scale
    return torch.where(code < 0, -value, value)


def _adamw_plain(s):
    total = _total(s["grad"], "2")
    s["step"] += 1
    step_size = LR / (1 - BETA1 ** s["step"])
    root = 1 / math.sqrt(1 - BETA2 ** s["step"])
    p, g = s["p"], s["grad"] * (s["limit"] / (total + CLIP_EPS)).clamp(max=1.0)
    if s["case"]["bits"] == 32:
        m, v = s["exp_avg"], s["exp_avg_sq"]
        m.mul_(BETA1).add_(g * (1 - BETA1))
        v.mul_(BETA2).add_(g * g * (1 - BETA2))
        p.copy_(p * (1 - LR * DECAY) - m / (v.sqrt() * root + ADAM_EPS) * step_size)
        return [total, p, m, v]
    r = _decode(s["rms_code"], s["rms_scale"], 19, 255).view(-1)
    m = _decode(s["exp_avg_code"], s["exp_avg_scale"], 20, 127).view(-1) * BETA1 + g * (1 - BETA1)
    r = torch.sqrt(r * r * BETA2 + g * g * (1 - BETA2))
    p.copy_(p * (1 - LR * DECAY) - m / (r * root + ADAM_EPS) * step_size)
    s["exp_avg_code"], s["exp_avg_scale"] = _encode(m, 20, 127, 0)
    s["rms_code"], s["rms_scale"] = _encode(r, 19, 255, 1)
    return [total, p]


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------

def _group_norm_own(s):
    import matrixman_b200 as matrixman
    case = s["case"]
    shape = (case["n"], case["h"] * case["w"], case["c"])
    if not case["train"]:
        with torch.no_grad():
            y = matrixman.group_norm(s["x"], case["groups"], s["weight"], s["bias"], EPS, activation=case["act"])
        return _torch_view(y, shape)
    y = matrixman.group_norm(s["x"], case["groups"], s["weight"], s["bias"], EPS, activation=case["act"])
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["grad"])
    return [_torch_view(y, shape), _torch_view(dx, shape), _torch_view(dw), _torch_view(db)]


def _norm_own(s):
    import matrixman_b200 as matrixman
    return _torch_view(matrixman.optim.grad_norm(s["params"], float(s["case"]["p"])))


def _clip_own(s):
    import matrixman_b200 as matrixman
    total = matrixman.optim.clip_grad_norm_(s["params"], s["limit"], float(s["case"]["p"]))
    s["limit"] *= 0.998  # the buffers come back clipped: the next pass has to clip again
    return [_torch_view(total), *s["out"]]


def _adamw_own(s):
    s["optimizer"].step()
    return [_torch_view(s["optimizer"].grad_norm), *s["out"]]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"group_norm": _group_norm_own, "norm": _norm_own, "clip": _clip_own, "adamw": _adamw_own}[op](state)
    if op == "norm":
        return _total(state["grad"], state["case"]["p"])
    return {"group_norm": _group_norm_plain, "clip": _clip_plain, "adamw": _adamw_plain}[op](state)


def work(case):
    if case["op"] == "group_norm":
        n = case["n"] * case["c"] * case["h"] * case["w"]
        # forward: x in, y out; backward: x and the gradient in, x's gradient out
        return {"bytes": 4 * n * (5 if case["train"] else 2) + 8 * case["c"], "flops": n * (30 if case["train"] else 10)}
    n = sum(math.prod(shape) for shape in _shapes(case))
    if case["op"] == "norm":
        return {"bytes": 4 * n, "flops": 2 * n}
    if case["op"] == "clip":
        return {"bytes": 8 * n, "flops": 3 * n}  # the gradients in and out
    # p, g and the states in, p and the states out
    return {"bytes": n * (28 if case["bits"] == 32 else 16), "flops": 18 * n}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_group_norm(case, g):
    t = {k: v.double() for k, v in _group_norm_inputs(case, g).items()}
    n, c, groups = case["n"], case["c"], case["groups"]
    x = t["x"].transpose(1, 2).reshape(n, groups, -1)  # a group's channels and pixels in one row
    var, mean = torch.var_mean(x, 2, unbiased=False, keepdim=True)
    sigma = torch.sqrt(var + EPS)
    w, b = (t[k].view(1, c, 1) for k in ("weight", "bias"))
    xc = (x - mean).reshape(n, c, -1)
    sc = sigma.expand(n, groups, c // groups).reshape(n, c, 1)
    f = {"none": lambda v: v * 1, "relu": lambda v: torch.maximum(v, torch.zeros_like(v)),
         "silu": lambda v: v / (1 + torch.exp(-v)), "sigmoid": lambda v: 1 / (1 + torch.exp(-v)),
         "gelu": lambda v: v * 0.5 * torch.special.erfc(-v / math.sqrt(2)),
         "gelu_tanh": lambda v: 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))),
         }[case["act"]]
    with torch.enable_grad():
        z = (xc / sc * w + b).requires_grad_(True)
        y = f(z)
        if case["train"]:
            dz, = torch.autograd.grad(y, z, t["grad"].transpose(1, 2))
    y = y.detach().transpose(1, 2)
    if not case["train"]:
        return y
    # d/dx of (x - mean) / sigma, term by term: through x, the mean and the variance
    gw, m = (dz * w).reshape(n, groups, -1), x.shape[2]
    dvar = (gw * (x - mean)).sum(2, keepdim=True) * -0.5 / sigma ** 3
    dx = gw / sigma + dvar * 2 * (x - mean) / m - (gw / sigma).sum(2, keepdim=True) / m
    return [y, dx.reshape(n, c, -1).transpose(1, 2), (dz * xc / sc).sum((0, 2)), dz.sum((0, 2))]


def exact(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    if case["op"] == "group_norm":
        return _exact_group_norm(case, g)
    s, layout = _tensor_inputs(case, g), _layout(case)[0]
    grads = [s["grad"][at:at + n].double() for _, at, n in layout]
    p = float(case.get("p", 2))
    total = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(v, p) for v in grads]), p)
    if case["op"] == "norm":
        return total
    clipped = s["grad"].double() * min(1.0, _limit(case) / (total.item() + CLIP_EPS))
    if case["op"] == "clip":
        return [total, clipped]
    m, r = s["exp_avg"], s["exp_avg_sq"].sqrt()
    if case["bits"] == 8:  # the state's values are what its codes stand for
        m, r = _decode(*_encode(m, 20, 127, 0), 20, 127).view(-1), _decode(*_encode(r, 19, 255, 1), 19, 255).view(-1)
        v = r.double() ** 2
    else:
        v = s["exp_avg_sq"].double()
    p, m, t = s["p"].double(), m.double(), STEPS_DONE + 1
    m = m + (1 - BETA1) * (clipped - m)
    v = v + (1 - BETA2) * (clipped ** 2 - v)
    p = p - LR * DECAY * p - LR * (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + ADAM_EPS)
    return [total, p, m, v] if case["bits"] == 32 else [total, p]
