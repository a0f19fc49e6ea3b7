"""Cases of the training-block operators: layer norm, linear with a fused epilogue, AdamW.

Each case runs in two forms on the same inputs: elementary torch operations
(``own`` false), and the calls a user makes of matrixman_b200 (``own`` true).
Everything is float32, the framework's compute type; optimiser states are held
in 32 or in 8 bits.
"""

import math

import torch

own = False

EPS = 1e-5                      # layer norm
LR, BETA1, BETA2, ADAM_EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
STEPS_DONE = 20                 # optimiser steps before the measured one
BLOCK = 256                     # elements that share a scale of the 8-bit states
ONE_BITS = 0x3F800000           # 1.0f


def listed():
    return [
        # The norm of a decoding step: a few tokens, where the call's latency is all of the time.
        {"name": "norm forward 16x1024", "op": "norm", "rows": 16, "width": 1024, "train": False},
        # The norm of a long prompt or an evaluation batch.
        {"name": "norm forward 32768x2048", "op": "norm", "rows": 32768, "width": 2048, "train": False},
        # A training batch whose ragged documents and odd width leave rows that are not 16-byte aligned.
        {"name": "norm train 5003x1250", "op": "norm", "rows": 5003, "width": 1250, "train": True},
        # A training batch of a wide model: the largest norm.
        {"name": "norm train 16384x4096", "op": "norm", "rows": 16384, "width": 4096, "train": True},
        # One token through a block's down projection, added to the residual stream.
        {"name": "linear token 1x4096x4096", "op": "linear", "rows": 1, "inner": 4096, "outer": 4096,
         "act": "none", "residual": True, "train": False},
        # The first layer of the framework's MLP (batch 256, 784 -> 512, ReLU).
        {"name": "linear 256x784x512", "op": "linear", "rows": 256, "inner": 784, "outer": 512, "act": "relu",
         "residual": False, "train": False},
        # An evaluation batch through a layer of odd sizes.
        {"name": "linear 1111x1502x2501", "op": "linear", "rows": 1111, "inner": 1502, "outer": 2501, "act": "silu",
         "residual": True, "train": False},
        # Fine-tuning on a ragged batch: forward and all gradients.
        {"name": "linear train 2000x1280x1000", "op": "linear", "rows": 2000, "inner": 1280, "outer": 1000,
         "act": "gelu_tanh", "residual": True, "train": True},
        # A training batch through a block's up projection: the largest product.
        {"name": "linear train 8192x2048x4096", "op": "linear", "rows": 8192, "inner": 2048, "outer": 4096,
         "act": "gelu", "residual": False, "train": True},
        # The optimiser step of the framework's MLP: six small tensors, launches and latency.
        {"name": "adamw 32-bit mlp", "op": "adamw", "bits": 32, "layers": 0, "width": 0},
        # The optimiser step of twelve blocks: 72 tensors, 101 M parameters.
        {"name": "adamw 32-bit 12x1024", "op": "adamw", "bits": 32, "layers": 12, "width": 1024},
        # States in 8 bits, where memory for two more copies of the parameters is missing.
        {"name": "adamw 8-bit 3x1500", "op": "adamw", "bits": 8, "layers": 3, "width": 1500},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "linear", "adamw"])
    if op == "norm":
        width = _spread(rng, 64, 8192)
        return {"op": op, "rows": _spread(rng, 1, min(65536, (1 << 26) // width)), "width": width,
                "train": rng.random() < 0.6}
    if op == "linear":
        inner, outer = _spread(rng, 32, 4096), _spread(rng, 32, 4096)
        rows = _spread(rng, 1, min(16384, (1 << 35) // (inner * outer)))
        return {"op": op, "rows": rows, "inner": inner, "outer": outer,
                "act": rng.choice(["none", "relu", "silu", "sigmoid", "gelu", "gelu_tanh"]),
                "residual": rng.random() < 0.5, "train": rng.random() < 0.5}
    bits = rng.choice([32, 8])
    return {"op": op, "bits": bits, "layers": rng.randint(1, 12 if bits == 32 else 3), "width": _spread(rng, 40, 1024)}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

class _Span:
    """A dense device buffer of the framework, as torch sees it."""

    def __init__(self, t):
        kind = {torch.float32: "<f4", torch.int64: "<i8"}[t.dtype]
        self.owner = t
        self.__cuda_array_interface__ = {"shape": tuple(t.shape), "typestr": kind, "data": (t.element_ptr, False),
                                         "version": 3, "strides": None, "stream": None}


def _torch_view(t):
    return torch.as_tensor(_Span(t), device="cuda")


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
    """The tensors of the optimiser's cases: the framework's MLP, or blocks of
    two linear layers (width -> 4 width -> width) and a norm."""
    w = case["width"]
    if not case["layers"]:
        return [(512, 784), (512,), (256, 512), (256,), (10, 256), (10,)]
    return [(4 * w, w), (4 * w,), (w, 4 * w), (w,), (w,), (w,)] * case["layers"]


def _layout(case):
    """(shape, start, elements) of each tensor in a flat buffer where each
    starts at a multiple of BLOCK, and the buffer's length."""
    got, at = [], 0
    for shape in _shapes(case):
        n = math.prod(shape)
        got.append((shape, at, n))
        at += -(-n // BLOCK) * BLOCK
    return got, at


def _norm_inputs(case, g):
    rows, width = case["rows"], case["width"]
    # Hidden states: rows of different scale and offset, a few outlier channels.
    x = torch.randn(rows, width, device="cuda", generator=g)
    x *= 1 + 9 * (torch.rand(width, device="cuda", generator=g) < 0.01)
    x *= 0.2 + 2 * torch.rand(rows, 1, device="cuda", generator=g)
    x += 0.5 * torch.randn(rows, 1, device="cuda", generator=g)
    s = {"x": x, "weight": 1 + 0.1 * torch.randn(width, device="cuda", generator=g),
         "bias": 0.1 * torch.randn(width, device="cuda", generator=g)}
    if case["train"]:
        s["grad"] = 1e-2 * torch.randn(rows, width, device="cuda", generator=g)
    return s


def _linear_inputs(case, g):
    rows, inner, outer = case["rows"], case["inner"], case["outer"]
    s = {"x": torch.randn(rows, inner, device="cuda", generator=g),
         "weight": torch.randn(outer, inner, device="cuda", generator=g) / math.sqrt(inner),
         "bias": 0.1 * torch.randn(outer, device="cuda", generator=g)}
    if case["residual"]:
        s["residual"] = torch.randn(rows, outer, device="cuda", generator=g)
    if case["train"]:
        # Gradients of a loss averaged over the batch; the padding's rows are zero.
        s["grad"] = 1e-3 * torch.randn(rows, outer, device="cuda", generator=g)
        s["grad"] *= (torch.rand(rows, 1, device="cuda", generator=g) < 0.95)
    return s


def _adamw_inputs(case, g):
    layout, total = _layout(case)
    p, grad, m, v = (torch.zeros(total, device="cuda") for _ in range(4))
    for shape, at, n in layout:
        scale = 1e-3 * math.exp(torch.randn((), device="cuda", generator=g).item())
        r = torch.randn(4, n, device="cuda", generator=g)
        p[at:at + n] = 0.02 * r[0]
        grad[at:at + n] = scale * r[1]
        m[at:at + n] = 0.2 * scale * r[2]
        v[at:at + n] = (scale * (0.05 + r[3].abs())) ** 2
    return {"p": p, "grad": grad, "exp_avg": m, "exp_avg_sq": v, "step": STEPS_DONE}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = {"norm": _norm_inputs, "linear": _linear_inputs, "adamw": _adamw_inputs}[case["op"]](case, g)
    s["case"] = dict(case)
    if case["op"] == "adamw":
        s["layout"] = _layout(case)[0]
        if not own and case["bits"] == 8:
            s["exp_avg_code"], s["exp_avg_scale"] = _encode(s.pop("exp_avg"), 20, 127, 0)
            s["rms_code"], s["rms_scale"] = _encode(s.pop("exp_avg_sq").sqrt(), 19, 255, 1)
    if own:
        for k in [k for k, t in s.items() if isinstance(t, torch.Tensor)]:
            s[k] = _framework(s[k])
            if case.get("train") and k != "grad":
                s[k].requires_grad_(True)
        if case["op"] == "adamw":
            _framework_optimizer(s)
    return s


def _framework_optimizer(s):
    """The program's parameters, gradients and optimiser over the flat buffers."""
    import matrixman_b200 as matrixman
    bits, params = s["case"]["bits"], []
    part = {k: [s[k][at:at + n].view(shape) for shape, at, n in s["layout"]]
            for k in ("p", "grad", "exp_avg", "exp_avg_sq")}
    for p, grad in zip(part["p"], part["grad"]):
        params.append(torch.nn.Parameter(p))
        params[-1].grad = grad
    s["optimizer"] = opt = matrixman.optim.AdamW(params, lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS,
                                                 weight_decay=DECAY, state_bits=bits)
    for p, m, v in zip(params, part["exp_avg"], part["exp_avg_sq"]):
        if bits == 8:
            opt.set_state_values(p, m, v, step=s["step"])
        else:
            opt.state[p] = {"step": matrixman.to_device(torch.tensor(float(s["step"]))), "exp_avg": m, "exp_avg_sq": v}
    s["params"] = params
    s["out"] = [_torch_view(s[k]) for k in ("p", "exp_avg", "exp_avg_sq")]
    if bits == 8:
        del s["exp_avg"], s["exp_avg_sq"], s["out"][1:]
    matrixman.synchronize()


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------

def _norm_plain(s):
    x, w = s["x"], s["weight"]
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    xh = d * rstd
    y = xh * w + s["bias"]
    if not s["case"]["train"]:
        return y
    dy = s["grad"]
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return [y, dx, (dy * xh).sum(0), dy.sum(0)]


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


def _linear_plain(s):
    case = s["case"]
    z = s["x"] @ s["weight"].t() + s["bias"]
    y = _act(z, case["act"])
    if case["residual"]:
        y = y + s["residual"]
    if not case["train"]:
        return y
    dz = s["grad"] * _act_slope(z, case["act"])
    return [y, dz @ s["weight"], dz.t() @ s["x"], dz.sum(0)]


def _encode(a, shift, top, least):
    """Codes and block scales of the log-linear 8-bit code: the magnitude's
    share of its block's largest, rounded (to even) to the bits of a float32
    above `shift`, counted down from `top` (1.0).  A block whose largest is
    below the smallest normal number is stored as zero."""
    a = a.view(-1, BLOCK)
    size = a.abs()
    scale = size.amax(1, keepdim=True)
    scale = torch.where(scale < 2.0 ** -126, 0.0, scale)
    bits = (size * (1 / scale)).view(torch.int32)
    code = ((bits + ((1 << (shift - 1)) - 1) + ((bits >> shift) & 1)) >> shift) - (ONE_BITS >> shift) + top
    code = torch.where(size > 0, code.clamp(least, top), 0)
    return torch.where(a < 0, -code, code), scale


def _decode(code, scale, shift, top):
    size = ((code.abs() + (ONE_BITS >> shift) - top) << shift).view(torch.float32)
    value = torch.where(code != 0, size, 0.0) * scale
    return torch.where(code < 0, -value, value)


def _adamw_plain(s):
    s["step"] += 1
    step_size = LR / (1 - BETA1 ** s["step"])
    root = 1 / math.sqrt(1 - BETA2 ** s["step"])
    p, g = s["p"], s["grad"]
    if s["case"]["bits"] == 32:
        m, v = s["exp_avg"], s["exp_avg_sq"]
        m.mul_(BETA1).add_(g * (1 - BETA1))
        v.mul_(BETA2).add_(g * g * (1 - BETA2))
        p.copy_(p * (1 - LR * DECAY) - m / (v.sqrt() * root + ADAM_EPS) * step_size)
        return [p, m, v]
    r = _decode(s["rms_code"], s["rms_scale"], 19, 255).view(-1)
    m = _decode(s["exp_avg_code"], s["exp_avg_scale"], 20, 127).view(-1) * BETA1 + g * (1 - BETA1)
    r = torch.sqrt(r * r * BETA2 + g * g * (1 - BETA2))
    p.copy_(p * (1 - LR * DECAY) - m / (r * root + ADAM_EPS) * step_size)
    s["exp_avg_code"], s["exp_avg_scale"] = _encode(m, 20, 127, 0)
    s["rms_code"], s["rms_scale"] = _encode(r, 19, 255, 1)
    m = _decode(s["exp_avg_code"], s["exp_avg_scale"], 20, 127).view(-1)
    r = _decode(s["rms_code"], s["rms_scale"], 19, 255).view(-1)
    v = r * r
    return [p, [(m[at:at + n].view(shape), v[at:at + n].view(shape)) for shape, at, n in s["layout"]]]


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------

def _norm_own(s):
    if not s["case"]["train"]:
        with torch.no_grad():
            return _torch_view(torch.nn.functional.layer_norm(s["x"], s["weight"].shape, s["weight"], s["bias"], EPS))
    y = torch.nn.functional.layer_norm(s["x"], s["weight"].shape, s["weight"], s["bias"], EPS)
    grads = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["grad"])
    return [_torch_view(t) for t in (y, *grads)]


def _linear_own(s):
    import matrixman_b200 as matrixman
    case = s["case"]
    if not case["train"]:
        with torch.no_grad():
            return _torch_view(matrixman.linear(s["x"], s["weight"], s["bias"], activation=case["act"],
                                                residual=s.get("residual")))
    y = matrixman.linear(s["x"], s["weight"], s["bias"], activation=case["act"], residual=s.get("residual"))
    grads = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["grad"])
    return [_torch_view(t) for t in (y, *grads)]


def _adamw_own(s):
    s["optimizer"].step()
    if s["case"]["bits"] == 32:
        return s["out"]
    values = [s["optimizer"].state_values(p) for p in s["params"]]
    return [s["out"][0], [(_torch_view(m), _torch_view(v)) for m, v in values]]


def run(state):
    if own:
        return {"norm": _norm_own, "linear": _linear_own, "adamw": _adamw_own}[state["case"]["op"]](state)
    return {"norm": _norm_plain, "linear": _linear_plain, "adamw": _adamw_plain}[state["case"]["op"]](state)


def work(case):
    if case["op"] == "norm":
        n = case["rows"] * case["width"]
        # forward: x in, y out; backward: x and the gradient in, x's gradient out
        return {"bytes": 4 * n * (5 if case["train"] else 2) + 8 * case["width"], "flops": n * (22 if case["train"] else 8)}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["inner"], case["outer"]
        moved = m * k + k * n + n + m * n * (2 if case["residual"] else 1)
        if case["train"]:
            moved += 2 * (m * k + k * n) + m * n + n  # x, weight and their gradients; the output's gradient
        return {"bytes": 4 * moved, "flops": 2 * m * n * k * (3 if case["train"] else 1)}
    n = sum(math.prod(shape) for shape in _shapes(case))
    # 32 bits: p, g, m, v in, p, m, v out; 8 bits: codes in and out, and the states' values out
    return {"bytes": n * (28 if case["bits"] == 32 else 24), "flops": 15 * n}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    if case["op"] == "norm":
        s = {k: t.double() for k, t in _norm_inputs(case, g).items()}
        x, w, b = s["x"], s["weight"], s["bias"]
        var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
        sigma = torch.sqrt(var + EPS)
        y = (x - mean) / sigma * w + b
        if not case["train"]:
            return y
        dy, n = s["grad"], case["width"]
        gw, d = dy * w, x - mean
        # d/dx of (x - mean) / sigma, term by term: through x, the mean and the variance
        dvar = (gw * d).sum(1, keepdim=True) * -0.5 / sigma ** 3
        dmean = -(gw / sigma).sum(1, keepdim=True)
        dx = gw / sigma + dvar * 2 * d / n + dmean / n
        return [y, dx, (dy * d / sigma).sum(0), dy.sum(0)]
    if case["op"] == "linear":
        s = {k: t.double() for k, t in _linear_inputs(case, g).items()}
        with torch.enable_grad():
            z = (torch.einsum("mk,nk->mn", s["x"], s["weight"]) + s["bias"]).requires_grad_(True)
            f = {"none": lambda v: v * 1, "relu": lambda v: torch.maximum(v, torch.zeros_like(v)),
                 "silu": lambda v: v / (1 + torch.exp(-v)), "sigmoid": lambda v: 1 / (1 + torch.exp(-v)),
                 "gelu": lambda v: v * 0.5 * torch.special.erfc(-v / math.sqrt(2)),
                 "gelu_tanh": lambda v: 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))),
                 }[case["act"]]
            a = f(z)
            y = (a + s["residual"] if case["residual"] else a).detach()
            if not case["train"]:
                return y
            dz, = torch.autograd.grad(a, z, s["grad"])
        return [y, torch.einsum("mn,nk->mk", dz, s["weight"]), torch.einsum("mn,mk->nk", dz, s["x"]), dz.sum(0)]
    s = _adamw_inputs(case, g)
    layout = _layout(case)[0]
    if case["bits"] == 8:  # the state's values are what its codes stand for
        m, r = s["exp_avg"], s["exp_avg_sq"].sqrt()
        s["exp_avg"] = _decode(*_encode(m, 20, 127, 0), 20, 127).view(-1)
        s["exp_avg_sq"] = _decode(*_encode(r, 19, 255, 1), 19, 255).view(-1).double() ** 2
    p, grad, m, v = (s[k].double() for k in ("p", "grad", "exp_avg", "exp_avg_sq"))
    t = s["step"] + 1
    m = m + (1 - BETA1) * (grad - m)
    v = v + (1 - BETA2) * (grad ** 2 - v)
    p = p - LR * DECAY * p - LR * (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + ADAM_EPS)
    if case["bits"] == 32:
        return [p, m, v]
    # Which code a value next to a border takes has no answer in 64 bits.
    return [p, [(None, None) for _ in layout]]
