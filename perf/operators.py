"""The training and serving operators around the quantizers, as cases that can be timed: norms, linear layers with a fused
epilogue, and the 8-bit copies of activations that both keep for their backward pass.

With `own` false `run` computes an operator in its plain form, elementary torch operations in 32 bits; with `own` true it
makes the calls that a user makes.  `exact` is the definition again, in 64 bits.  Shapes are those of the repository's
benchmark configurations and tests, or generic.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
GROUP = 32                       # elements that share a scale in an 8-bit copy


def listed():
    return [
        # One generated token's hidden state (Qwen3-4B) in front of its projections: launch and host cost.
        {"name": "norm_token", "op": "norm", "kind": "rms", "rows": 1, "cols": 2560, "dtype": "bf16", "train": False, "kept8": False},
        # The norms of a packed training batch, an odd number of tokens, input kept as it is.
        {"name": "norm_train", "op": "norm", "kind": "layer", "rows": 8191, "cols": 4096, "dtype": "fp16", "train": True, "kept8": False},
        # The same at the width of DeepSeek-V3, normalized values kept in 8 bits for the backward pass.
        {"name": "norm_train_8bit", "op": "norm", "kind": "rms", "rows": 16384, "cols": 7168, "dtype": "bf16", "train": True, "kept8": True},
        # fp32 rows of a width that is no multiple of anything.
        {"name": "norm_ragged", "op": "norm", "kind": "layer", "rows": 1777, "cols": 2563, "dtype": "fp32", "train": True, "kept8": False},
        # One generated token through the wide projection of Qwen3-4B: the weight is read once and nothing else counts.
        {"name": "linear_token", "op": "linear", "rows": 1, "inner": 2560, "outer": 9728, "act": "gelu", "bias": True, "residual": False,
         "dtype": "bf16", "train": False, "kept8": False},
        # A decode batch through the narrow projection back onto the residual stream.
        {"name": "linear_batch", "op": "linear", "rows": 48, "inner": 9728, "outer": 2560, "act": "none", "bias": True, "residual": True,
         "dtype": "bf16", "train": False, "kept8": False},
        # A long prompt through a projection of a DeepSeek-V3-shaped expert.
        {"name": "linear_prompt", "op": "linear", "rows": 16384, "inner": 7168, "outer": 2048, "act": "silu", "bias": False, "residual": False,
         "dtype": "fp16", "train": False, "kept8": False},
        # Training step of the wide projection of Qwen3-4B, input and pre-activation kept in 8 bits: the largest case.
        {"name": "linear_train_8bit", "op": "linear", "rows": 8192, "inner": 2560, "outer": 9728, "act": "gelu", "bias": True,
         "residual": False, "dtype": "bf16", "train": True, "kept8": True},
        # Training step of the projection back onto the residual stream, an odd number of tokens, input kept as it is.
        {"name": "linear_train", "op": "linear", "rows": 4099, "inner": 4096, "outer": 2560, "act": "none", "bias": True, "residual": True,
         "dtype": "bf16", "train": True, "kept8": False},
        # A small layer whose sides are no multiple of anything.
        {"name": "linear_ragged", "op": "linear", "rows": 777, "inner": 1545, "outer": 1003, "act": "gelu", "bias": True, "residual": True,
         "dtype": "fp16", "train": True, "kept8": False},
        # What a recomputation-free backward pass keeps of one layer's hidden states, and gets back.
        {"name": "keep_8bit", "op": "keep", "rows": 4099, "cols": 2560, "dtype": "bf16"},
        # The same over a long batch at the width of DeepSeek-V3, kept in fp32 by the program.
        {"name": "keep_8bit_fp32", "op": "keep", "rows": 16384, "cols": 7168, "dtype": "fp32"},
    ]


# ---- drawn cases ---------------------------------------------------------------------------------------------------
MAX_PRODUCTS = 8192 * 2560 * 9728     # of a linear layer: the largest listed
MAX_ELEMENTS = 1 << 27                # of a norm or a kept activation


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "linear", "linear", "linear", "keep"])
    dtype = rng.choice(["bf16", "bf16", "fp16"] if op == "linear" else ["bf16", "bf16", "fp16", "fp32"])
    if op == "keep":
        cols = max(1, _log(rng, 32, 16384) // GROUP) * GROUP
        return {"op": op, "rows": min(_log(rng, 1, 32768), MAX_ELEMENTS // cols), "cols": cols, "dtype": dtype}
    train = rng.random() < 0.6
    kept8 = train and dtype != "fp32" and rng.random() < 0.5       # (a program that saves memory holds 16-bit activations)
    if op == "norm":
        cols = _log(rng, 48, 12288)
        if kept8 or rng.random() < 0.6:
            cols = max(64, cols // 64 * 64)
        return {"op": op, "kind": rng.choice(["rms", "layer"]), "rows": min(_log(rng, 1, 32768), MAX_ELEMENTS // cols), "cols": cols,
                "dtype": dtype, "train": train, "kept8": kept8}
    inner, outer, rows = _log(rng, 96, 9728), _log(rng, 96, 9728), _log(rng, 1, 16384)
    if kept8 or rng.random() < 0.75:
        inner, outer = max(64, inner // 64 * 64), max(64, outer // 64 * 64)
    rows = min(rows, MAX_PRODUCTS // (inner * outer * (1 if train else 2)))
    return {"op": op, "rows": rows, "inner": inner, "outer": outer, "act": rng.choice(["none", "relu", "silu", "gelu"]),
            "bias": rng.random() < 0.6, "residual": rng.random() < 0.4, "dtype": dtype, "train": train, "kept8": kept8}


# ---- inputs --------------------------------------------------------------------------------------------------------
def _activation(g, shape, dtype):
    """Tokens of different magnitude, with a few columns ten times as large as the others."""
    x = torch.randn(shape, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn((shape[0], 1), generator=g, device="cuda"))
    x *= torch.where(torch.rand((1, shape[1]), generator=g, device="cuda") < 0.003, 10.0, 1.0)
    return x.to(dtype)


def _vector(g, n, dtype, mean):
    return (mean + 0.1 * torch.randn(n, generator=g, device="cuda")).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s, dtype = dict(case), DTYPES[case["dtype"]]
    if case["op"] == "linear":
        s["x"] = _activation(g, (case["rows"], case["inner"]), dtype)
        s["w"] = (torch.randn((case["outer"], case["inner"]), generator=g, device="cuda") / math.sqrt(case["inner"])).to(dtype)
        s["b"] = _vector(g, case["outer"], dtype, 0.0) if case["bias"] else None
        s["r"] = _activation(g, (case["rows"], case["outer"]), dtype) if case["residual"] else None
        out = (case["rows"], case["outer"])
    else:
        s["x"] = _activation(g, (case["rows"], case["cols"]), dtype)
        out = (case["rows"], case["cols"])
    if case["op"] == "norm":
        s["x"] += 0.25
        s["w"] = _vector(g, case["cols"], dtype, 1.0)
        s["b"] = _vector(g, case["cols"], dtype, 0.0) if case["kind"] == "layer" else None
    if case.get("train"):
        s["dy"] = torch.randn(out, generator=g, device="cuda").to(dtype)
        s["leaves"] = [s[k].requires_grad_(True) for k in ("x", "w", "b", "r") if s.get(k) is not None]
    return s


# ---- the plain forms, in 32 bits --------------------------------------------------------------------------------------
EPS = 1e-5
INV_SQRT2, INV_SQRT_2PI = 0.7071067811865476, 0.3989422804014327


def _act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * INV_SQRT2))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    return 0.5 * (1 + torch.erf(z * INV_SQRT2)) + z * INV_SQRT_2PI * torch.exp(-0.5 * z * z)


def _power(e):
    """2^e, made of its bits (a pow on the GPU is off by a rounding here and there)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _keep8(x):
    """(e4m3 codes as float8, exponent byte of each group of 32, the values they stand for in x's precision).  The exponent is that of the
    smallest power of two not below fl32(max|x| fl32(1/448)); codes are x over that power, rounded to nearest even."""
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    top = g.abs().amax(-1, keepdim=True).float() * torch.tensor(1 / 448, dtype=torch.float32, device=x.device)
    m, e = torch.frexp(top)
    e = torch.where(m == 0.5, e - 1, e)
    e = torch.where(top == 0, torch.zeros_like(e), (e + 127).clamp(0, 254))
    up = torch.where(e == 0, torch.ones_like(e), _power(127 - e)).to(x.dtype)
    codes = (g * up).clamp(-448, 448).to(torch.float8_e4m3fn)
    values = (codes.to(x.dtype) * _power(e - 127).to(x.dtype)).reshape(x.shape)
    return codes.reshape(x.shape), e.squeeze(-1).to(torch.uint8), values


def _norm_plain(s, wide):
    x, w, b = s["x"].detach().to(wide), s["w"].detach().to(wide), s["b"]
    mean = x.mean(-1, keepdim=True) if s["kind"] == "layer" else 0.0
    rstd = 1 / torch.sqrt((x - mean).square().mean(-1, keepdim=True) + EPS)
    xhat = (x - mean) * rstd
    y = xhat * w
    if b is not None:
        y = y + b.detach().to(wide)
    if not s["train"]:
        return [y]
    if s["kept8"]:
        xhat = _keep8(xhat)[2]
    dy = s["dy"].to(wide)
    g = dy * w
    dx = g - xhat * (g * xhat).mean(-1, keepdim=True)
    if s["kind"] == "layer":
        dx = dx - g.mean(-1, keepdim=True)
    grads = [dx * rstd, (dy * xhat).sum(0)]
    return [y] + grads + ([dy.sum(0)] if b is not None else [])


def _linear_plain(s, wide):
    x, w, act = s["x"].detach().to(wide), s["w"].detach().to(wide), s["act"]
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].detach().to(wide)
    y = _act(z, act)
    if s["r"] is not None:
        y = y + s["r"].detach().to(wide)
    if not s["train"]:
        return [y]
    dz = s["dy"].to(wide)
    if act != "none":                                   # what is kept of z: 8 bits, or the input's type
        dz = dz * _act_slope(_keep8(z)[2] if s["kept8"] else z.to(s["x"].dtype).to(wide), act)
    if s["kept8"]:
        x = _keep8(x)[2]
    grads = [dz @ w, dz.t() @ x]
    if s["b"] is not None:
        grads.append(dz.sum(0))
    return [y] + grads + ([s["dy"]] if s["r"] is not None else [])


def _plain(s):
    if s["op"] == "keep":
        codes, exponents, values = _keep8(s["x"].float())
        return [codes, exponents, values.to(s["x"].dtype)]
    out = _norm_plain(s, torch.float32) if s["op"] == "norm" else _linear_plain(s, torch.float32)
    return [v.to(s["x"].dtype) for v in out]


# ---- the framework's calls ----------------------------------------------------------------------------------------------
def _own(s):
    if s["op"] == "keep":
        from miles_amd.kernels.quant.act_checkpoint import checkpoint_activation

        kept = checkpoint_activation(s["x"])
        return [kept.codes, kept.scales, kept.restore()]
    if s["op"] == "norm":
        from miles_amd.kernels.norm import layer_norm, rms_norm

        if s["kind"] == "rms":
            y = rms_norm(s["x"], s["w"], EPS, checkpoint=s["kept8"])
        else:
            y = layer_norm(s["x"], s["w"], s["b"], EPS, checkpoint=s["kept8"])
    else:
        from miles_amd.kernels.linear import linear

        y = linear(s["x"], s["w"], s["b"], activation=None if s["act"] == "none" else s["act"], residual=s["r"], checkpoint=s["kept8"])
    if not s["train"]:
        return [y]
    return [y, *torch.autograd.grad(y, s["leaves"], s["dy"])]


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definition in 64 bits, written apart from the plain forms ---------------------------------------------------------
def _exact_keep8(x):
    """The codes of an 8-bit copy of x (64 bits), its exponent bytes, and what they stand for."""
    powers = torch.tensor([2.0**k for k in range(-400, 401)], dtype=torch.float64, device=x.device)
    power = lambda e: powers[(e + 400).long()]  # noqa: E731
    rows = x.reshape(-1, GROUP)
    bound = (rows.abs().max(dim=1).values.to(torch.float32) * torch.full((), 1 / 448, dtype=torch.float32, device=x.device)).double()
    some = bound > 0
    e = torch.floor(torch.log2(torch.where(some, bound, torch.ones_like(bound))))
    for _ in range(2):                                  # log2 may be off by a rounding next to a power of two
        e = torch.where(power(e) < bound, e + 1, e)
    e = torch.where(power(e - 1) >= bound, e - 1, e)
    byte = torch.where(some, torch.clamp(e + 127, 0, 254), torch.zeros_like(e))
    scale = power(byte - 127)[:, None]
    v = torch.where(byte[:, None] > 0, rows / scale, rows).clamp(-448.0, 448.0)
    # e4m3: steps of 2^(floor(log2|v|) - 3), at least 2^-9
    step = power(torch.clamp(torch.floor(torch.log2(v.abs().clamp_min(2.0**-20))), min=-6.0) - 3)
    code = torch.round(v / step) * step                 # (round: to the even neighbour)
    return code.reshape(x.shape), byte.reshape(*x.shape[:-1], -1), (code * scale).reshape(x.shape)


def _exact_linear(s):
    f = lambda t: t.detach().double()  # noqa: E731
    x, w, dtype = f(s["x"]), f(s["w"]), s["x"].dtype
    z = torch.addmm(f(s["b"]), x, w.t()) if s["b"] is not None else x.mm(w.t())
    cdf = lambda t: torch.special.ndtr(t)  # noqa: E731
    h = {"none": lambda: z, "relu": lambda: torch.maximum(z, torch.zeros_like(z)), "silu": lambda: z * torch.sigmoid(z),
         "gelu": lambda: z * cdf(z)}[s["act"]]()
    outs = [h + f(s["r"]) if s["r"] is not None else h]
    if not s["train"]:
        return outs
    dy = f(s["dy"])
    if s["act"] == "none":
        dz = dy
    else:
        kept = _exact_keep8(z)[2] if s["kept8"] else z.to(dtype).double()
        if s["act"] == "relu":
            dz = torch.where(kept > 0, dy, torch.zeros_like(dy))
        elif s["act"] == "silu":
            p = torch.sigmoid(kept)
            dz = dy * (p + kept * p * torch.sigmoid(-kept))
        else:
            dz = dy * (cdf(kept) + kept * torch.exp(kept.square() / -2) / math.sqrt(2 * math.pi))
    outs.append(dz.mm(w))
    outs.append(dz.t().mm(_exact_keep8(x)[2] if s["kept8"] else x))
    if s["b"] is not None:
        outs.append(dz.sum(dim=0))
    if s["r"] is not None:
        outs.append(dy)
    return outs


def _exact_norm(s):
    f = lambda t: t.detach().double()  # noqa: E731
    x, w, n, layer = f(s["x"]), f(s["w"]), s["cols"], s["kind"] == "layer"
    centred = x - x.sum(dim=1, keepdim=True) / n if layer else x
    sigma = torch.sqrt(centred.pow(2).sum(dim=1, keepdim=True) / n + EPS)
    unit = centred / sigma
    outs = [torch.addcmul(f(s["b"]), unit, w) if layer else unit * w]
    if not s["train"]:
        return outs
    if s["kept8"]:
        unit = _exact_keep8(unit)[2]
    dy = f(s["dy"])
    g = dy * w
    along = (g * unit).sum(dim=1, keepdim=True) / n
    flat = g.sum(dim=1, keepdim=True) / n if layer else 0.0
    outs += [(g - flat - unit * along) / sigma, (unit * dy).sum(dim=0)]
    return outs + ([dy.sum(dim=0)] if layer else [])


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "keep":
        codes, byte, values = _exact_keep8(s["x"].double())
        return [codes, byte, values]
    return _exact_norm(s) if case["op"] == "norm" else _exact_linear(s)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
KEPT = 1 + 1 / GROUP


def work(case):
    """Every input byte read once and every output byte written once; what is kept between the passes is written once and read once.
    Two operations for each product of a matrix product, a handful for each element elsewhere."""
    size = BYTES[case["dtype"]]
    if case["op"] == "keep":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (2 * size + 2 * KEPT), "flops": 4 * n}
    if case["op"] == "norm":
        n = case["rows"] * case["cols"]
        if not case["train"]:
            return {"bytes": n * 2 * size + 2 * case["cols"] * size, "flops": 6 * n}
        again = 2 * KEPT if case["kept8"] else size
        return {"bytes": n * (4 * size + again), "flops": 20 * n}
    m, k, n = case["rows"], case["inner"], case["outer"]
    forward = (m * k + n * k + m * n * (2 if case["residual"] else 1)) * size
    if not case["train"]:
        return {"bytes": forward, "flops": 2 * m * n * k}
    per = KEPT if case["kept8"] else size
    kept = (2 * m * n * per if case["act"] != "none" else 0) + (m * k * KEPT * 2 if case["kept8"] else m * k * size)
    backward = (m * n + 2 * n * k + m * k) * size
    return {"bytes": forward + kept + backward, "flops": 6 * m * n * k}
