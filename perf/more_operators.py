"""Dense layers in 8-bit integers and the norm before them: cases to time and compare.

Each case runs one operator either in its plain form (elementary torch
operations in 32 bits, ``own = False``) or through the framework's public
entry points (``own = True``).  Both get the same inputs from ``prepare``.

Definitions.  *Norm*: ``h = x + residual`` rounded to the tensors' type, ``y =
h * w / sqrt(mean(h^2) + eps)`` rounded once; its gradient is that of ``x``,
``residual`` (the same) and ``w`` from those of ``y`` and ``h``.  *8 bits*: a
row ``v`` is held as whole numbers ``n`` and a scale ``s = max|v| / 127``, each
``n`` the whole number nearest to ``v / s`` (of two, the even one).  *Products*: ``sum_k
a[m, k] * b[n, k]`` of whole numbers, times the row's scale and the channel's,
plus a bias, rounded once; the gated one, ``silu(gate) * up``, has blocks of
128 gate channels each followed by the 128 up channels that they gate.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_EPS = 1e-6
_framework = None


def _fw():
    """The framework's package (only where ``own`` is true)."""
    global _framework
    if _framework is None:
        import __graft_entry__

        _framework = __graft_entry__.load_package()
    return _framework


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # the residual stream of four sequences' one new token each: latency
        {"name": "norm_token", "op": "norm", "rows": 4, "width": 3584, "dtype": "bf16", "grad": False, "add": True},
        # a training step's norm and its gradient over a batch of tokens
        {"name": "norm_train", "op": "norm", "rows": 16384, "width": 3584, "dtype": "bf16", "grad": True, "add": True},
        # the same in 32 bits, rows of an odd width
        {"name": "norm_train_odd", "op": "norm", "rows": 4095, "width": 2561, "dtype": "fp32", "grad": True, "add": True},
        # one token on its way into a layer held in 8 bits
        {"name": "norm8_token", "op": "norm8", "rows": 1, "width": 3584, "dtype": "bf16", "add": True},
        # a prompt's tokens on theirs
        {"name": "norm8_prompt", "op": "norm8", "rows": 32768, "width": 3584, "dtype": "bf16", "add": True},
        # the MLP's activations of eight sequences' blocks of 32 tokens
        {"name": "quantize_block", "op": "quantize", "rows": 256, "width": 18944, "dtype": "bf16"},
        # those of a long prompt
        {"name": "quantize_prompt", "op": "quantize", "rows": 16384, "width": 18944, "dtype": "bf16"},
        # q, k and v of one token: the weights are read for a single row
        {"name": "linear_token", "op": "linear", "rows": 1, "out": 4608, "width": 3584, "bias": True, "dtype": "bf16"},
        # the down projection of eight sequences' blocks of 32 tokens: a long sum for few outputs
        {"name": "linear_block", "op": "linear", "rows": 256, "out": 3584, "width": 18944, "bias": False, "dtype": "bf16"},
        # q, k and v of a prompt of odd length
        {"name": "linear_prompt", "op": "linear", "rows": 8191, "out": 4608, "width": 3584, "bias": True, "dtype": "bf16"},
        # the MLP's gated product for one sequence's block of 32 tokens
        {"name": "swiglu_block", "op": "swiglu", "rows": 32, "out": 37888, "width": 3584, "dtype": "bf16"},
        # and for a prompt
        {"name": "swiglu_prompt", "op": "swiglu", "rows": 16384, "out": 37888, "width": 3584, "dtype": "bf16"},
    ]


def _between(rng, lo, hi):
    """A whole number spread evenly over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm8", "quantize", "linear", "linear", "linear", "swiglu", "swiglu"])
    if op in ("norm", "norm8", "quantize"):
        width = rng.choice([896, 3584, 18944, _between(rng, 16, 20000), 8 * _between(rng, 2, 2500)])
        rows = _between(rng, 1, min(32768, 110_000_000 // width))
        c = {"op": op, "rows": rows, "width": width, "dtype": rng.choice(["bf16", "bf16", "fp16"])}
        if op == "norm":
            c |= {"grad": rng.random() < 0.6, "dtype": rng.choice(["bf16", "fp16", "fp32"])}
        if op != "quantize":
            c["add"] = rng.random() < 0.8
        return c
    width = rng.choice([896, 3584, 18944, _between(rng, 16, 20000), 16 * _between(rng, 1, 1250)])
    if op == "swiglu":
        out = 256 * _between(rng, 1, 148)
        c = {"bias": False}
    else:
        out = rng.choice([512, 3584, 4608, _between(rng, 1, 40000), 8 * _between(rng, 1, 5000)])
        c = {"bias": rng.random() < 0.5}
    rows = _between(rng, 1, max(1, min(16384, 400_000_000_000 // (out * width))))
    c |= {"op": op, "rows": rows, "out": out, "width": width, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if op == "swiglu":
        del c["bias"]
    return c


# ------------------------------------------------------------------ inputs
def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g, dtype=dtype)


def _whole(g, rows, width):
    """Rows of 8-bit whole numbers as a normal row gives them (its largest near four deviations), and a scale of
    about one for each."""
    q = torch.empty(rows, width, dtype=torch.int8, device="cuda")
    q.copy_((_randn(g, rows, width, dtype=torch.float16) * 31.0).round_().clamp_(-127, 127))
    return q, torch.rand(rows, device="cuda", generator=g) + 0.5


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[c["dtype"]]
    s = {"case": c}
    if c["op"] in ("norm", "norm8", "quantize"):
        rows, width = c["rows"], c["width"]
        # some tokens' features stand out, as in a trained model's residual stream
        loud = torch.where(torch.rand(width, device="cuda", generator=g) < 0.01, 8.0, 1.0).to(dtype)
        s["x"] = _randn(g, rows, width, dtype=dtype) * loud
        if c["op"] == "quantize":
            return s
        s["residual"] = _randn(g, rows, width, dtype=dtype) * 2 * loud if c["add"] else None
        s["w"] = (1 + 0.2 * _randn(g, width)).to(dtype)
        if c["op"] == "norm" and c["grad"]:
            s["gy"] = _randn(g, rows, width, dtype=dtype)
            s["gh"] = _randn(g, rows, width, dtype=dtype) if c["add"] else None
            s["leaves"] = [t for t in (s["x"], s["residual"], s["w"]) if t is not None]
            for t in s["leaves"]:
                t.requires_grad_()
        return s
    s["q"], scale = _whole(g, c["rows"], c["width"])
    s["scale"] = scale * (3.0 / 127)
    s["wq"], scale = _whole(g, c["out"], c["width"])
    s["w_scale"] = scale * (3.0 / 127 / math.sqrt(c["width"]))
    s["bias"] = _randn(g, c["out"], dtype=dtype) if c.get("bias") else None
    return s


# ------------------------------------------------------------------ plain forms
def _plain_norm(s):
    c = s["case"]
    dtype = _DTYPES[c["dtype"]]
    x, w = s["x"].detach().to(torch.float32), s["w"].detach().to(torch.float32)
    h = x if s["residual"] is None else (x + s["residual"].detach().to(torch.float32)).to(dtype).to(torch.float32)
    rstd = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + _EPS)
    unit = h * rstd
    outs = ((unit * w).to(dtype),) + ((h.to(dtype),) if c["add"] else ())
    if not c["grad"]:
        return outs
    gy = s["gy"].to(torch.float32)
    g = gy * w
    dx = rstd * (g - unit * (g * unit).mean(-1, keepdim=True))
    if c["add"]:
        dx = dx + s["gh"].to(torch.float32)
    dx = dx.to(dtype)
    return outs + ((dx, dx) if c["add"] else (dx,)) + ((gy * unit).sum(0).to(dtype),)


def _plain_whole(v):
    """Rows of 64-bit values as whole numbers and scales (values next to a border decide in 64 bits)."""
    top = v.abs().amax(-1, keepdim=True)
    return torch.round(v * (127.0 / top)), top / 127.0


def _plain_norm8(s):
    c = s["case"]
    dtype = _DTYPES[c["dtype"]]
    h = s["x"] if s["residual"] is None else (s["x"].to(torch.float32) + s["residual"].to(torch.float32)).to(dtype)
    f = h.to(torch.float64)
    rstd = 1.0 / torch.sqrt((f * f).mean(-1, keepdim=True) + _EPS)
    n, scale = _plain_whole(f * s["w"].to(torch.float64))
    scale = (scale * rstd).to(torch.float32)
    return ((n * scale).to(dtype), scale[..., 0]) + ((h,) if c["add"] else ())


def _plain_quantize(s):
    n, scale = _plain_whole(s["x"].to(torch.float64))
    scale = scale.to(torch.float32)
    return (n * scale).to(s["x"].dtype), scale[..., 0]


def _plain_product(s):
    y = s["q"].to(torch.float32) @ s["wq"].to(torch.float32).T
    return y.mul_(s["scale"][:, None]).mul_(s["w_scale"])


def _plain_linear(s):
    y = _plain_product(s)
    if s["bias"] is not None:
        y = y + s["bias"].to(torch.float32)
    return y.to(_DTYPES[s["case"]["dtype"]])


def _plain_swiglu(s):
    y = _plain_product(s).view(s["q"].shape[0], -1, 2, 128)
    gate, up = y[:, :, 0], y[:, :, 1]
    y = gate / (1.0 + torch.exp(-gate)) * up
    return y.flatten(1).to(_DTYPES[s["case"]["dtype"]])


_PLAIN = {"norm": _plain_norm, "norm8": _plain_norm8, "quantize": _plain_quantize, "linear": _plain_linear,
          "swiglu": _plain_swiglu}


# ------------------------------------------------------------------ the framework's calls
def _own_norm(s):
    c = s["case"]
    y, h = _fw().add_rms_norm(s["x"], s["residual"], s["w"], _EPS)
    if not c["grad"]:
        return (y, h) if c["add"] else (y,)
    if not c["add"]:
        return (y,) + torch.autograd.grad(y, s["leaves"], s["gy"])
    return (y, h) + torch.autograd.grad((y, h), s["leaves"], (s["gy"], s["gh"]))


def _values(q, scale, dtype):
    """The values that whole numbers and their scales stand for: one product, rounded once."""
    return torch.mul(q, scale[..., None], out=torch.empty(q.shape, dtype=dtype, device=q.device))


def _own_norm8(s):
    c = s["case"]
    q, scale, h = _fw().add_rms_norm_int8(s["x"], s["residual"], s["w"], _EPS)
    return (_values(q, scale, s["x"].dtype), scale) + ((h,) if c["add"] else ())


def _own_quantize(s):
    q, scale = _fw().quantize_int8(s["x"])
    return _values(q, scale, s["x"].dtype), scale


def _own_linear(s):
    return _fw().linear_int8(s["q"], s["scale"], s["wq"], s["w_scale"], s["bias"], dtype=_DTYPES[s["case"]["dtype"]])


def _own_swiglu(s):
    return _fw().swiglu_int8(s["q"], s["scale"], s["wq"], s["w_scale"], dtype=_DTYPES[s["case"]["dtype"]])


_OWN = {"norm": _own_norm, "norm8": _own_norm8, "quantize": _own_quantize, "linear": _own_linear,
        "swiglu": _own_swiglu}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


# ------------------------------------------------------------------ work
def work(case):
    c = case
    n = c["rows"] * c["width"]
    if c["op"] in ("norm", "norm8", "quantize"):
        e = _BYTES[c["dtype"]]
        if c["op"] == "quantize":
            return {"bytes": n * (e + 1) + 4 * c["rows"], "flops": 3 * n}
        add = 2 if c["add"] else 0           # the residual in, the sum out
        if c["op"] == "norm8":
            return {"bytes": n * (e * (1 + add) + 1) + 4 * c["rows"] + e * c["width"], "flops": 6 * n}
        # backward: the gradient of y (and of h) in, the row's h and the gradient of x out; w in and its gradient out
        passes = 2 + add + ((3 + (1 if c["add"] else 0)) if c["grad"] else 0)
        return {"bytes": n * e * passes + e * c["width"] * (3 if c["grad"] else 1), "flops": (20 if c["grad"] else 5) * n}
    e = _BYTES[c["dtype"]]
    out = c["out"] // 2 if c["op"] == "swiglu" else c["out"]
    return {"bytes": n + c["out"] * c["width"] + 4 * (c["rows"] + c["out"]) + c["rows"] * out * e
            + (c["out"] * e if c.get("bias") else 0),
            "flops": 2 * c["rows"] * c["out"] * c["width"]}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_norm(c, s):
    x, w = s["x"].detach().double(), s["w"].detach().double().requires_grad_()
    h = x if s["residual"] is None else (x + s["residual"].detach().double()).to(s["x"].dtype).double()
    h.requires_grad_()
    with torch.enable_grad():
        y = w * h * torch.rsqrt(h.square().sum(-1, keepdim=True) / h.shape[-1] + _EPS)
        if c["grad"]:
            dh, dw = torch.autograd.grad(y, (h, w), s["gy"].double())
    outs = (y.detach(), h.detach()) if c["add"] else (y.detach(),)
    if not c["grad"]:
        return outs
    if c["add"]:
        dh = dh + s["gh"].double()
    return outs + ((dh, dh) if c["add"] else (dh,)) + (dw,)


def _exact_whole(v):
    scale = torch.linalg.vector_norm(v, ord=math.inf, dim=-1) / 127
    return (v / scale[..., None]).round() * scale[..., None], scale


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "norm":
        return _exact_norm(c, s)
    if c["op"] == "norm8":
        h = s["x"].double()
        if c["add"]:
            h = (h + s["residual"].double()).to(s["x"].dtype).double()
        v = h * s["w"].double() * torch.rsqrt(h.square().sum(-1, keepdim=True) / c["width"] + _EPS)
        return _exact_whole(v) + ((h,) if c["add"] else ())
    if c["op"] == "quantize":
        return _exact_whole(s["x"].double())
    y = torch.nn.functional.linear(s["q"].double() * s["scale"].double()[:, None],
                                   s["wq"].double() * s["w_scale"].double()[:, None],
                                   None if s["bias"] is None else s["bias"].double())
    if c["op"] == "linear":
        return y
    gate, up = y.unflatten(1, (-1, 256)).chunk(2, -1)
    return (torch.sigmoid(gate) * gate * up).flatten(1)
