"""The operators between a serving program's projections, as cases that can be timed: positions rotated into queries and keys
(forward and backward), keys and values appended to a paged cache, and the attention of one new token a sequence over that cache.

With `own` false `run` computes an operator in its plain form, elementary torch operations in 32 bits (angles in 64); with `own`
true it makes the calls that a user makes.  `exact` is the definition again, in 64 bits.  Heads and widths are those of the
repository's benchmark configuration (32 query heads, 8 key heads of 128) or generic.

A cache holds `keys` [pages, key heads, key width / x, page size, x], x the elements of 16 bytes, and `values` [pages, key heads, page
size, value width]; in 8 bits both are e4m3 codes, with an exponent byte for 32 elements of a token's vector in [pages, key heads, width /
32, page size].  Slot s of a token is place s % (page size) of page s // (page size).
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
GROUP = 32                       # elements of a vector that share a scale in 8 bits
KEPT = 1 + 1 / GROUP


def listed():
    return [
        # The queries and keys of one generated token: launch and host cost.
        {"name": "rotary_token", "op": "rotary", "batch": 1, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "turned": 128, "interleaved": False,
         "far": 32768, "stretch": 1.0, "dtype": "bf16", "train": False},
        # A training batch of four sequences, queries and keys as views of a fused projection's output.
        {"name": "rotary_train", "op": "rotary", "batch": 4, "tokens": 4096, "heads": 32, "kv_heads": 8, "dim": 128, "turned": 128, "interleaved": False,
         "far": 4096, "stretch": 1.0, "dtype": "bf16", "train": True},
        # A stretched context with positions up to a million, pairs side by side, a third of the head turned, an odd number of tokens.
        {"name": "rotary_far", "op": "rotary", "batch": 1, "tokens": 5003, "heads": 16, "kv_heads": 4, "dim": 192, "turned": 64, "interleaved": True,
         "far": 1 << 20, "stretch": 32.0, "dtype": "fp16", "train": True},
        # A decode batch: every sequence's new token rotated and appended, its queries rotated with it.
        {"name": "append_batch", "op": "append", "tokens": 64, "heads": 32, "kv_heads": 8, "key_dim": 128, "value_dim": 128, "page": 16, "turned": 128,
         "interleaved": False, "far": 32768, "kept8": False, "queries": True, "prompts": 64, "dtype": "bf16"},
        # The tokens of five prompts of different lengths at once.
        {"name": "append_prompts", "op": "append", "tokens": 8191, "heads": 32, "kv_heads": 8, "key_dim": 128, "value_dim": 128, "page": 16, "turned": 128,
         "interleaved": False, "far": 32768, "kept8": False, "queries": True, "prompts": 5, "dtype": "bf16"},
        # Long prompts into a cache of 8 bits, keys wider than values, half of a key turned.
        {"name": "append_prompts_8bit", "op": "append", "tokens": 16384, "heads": 32, "kv_heads": 4, "key_dim": 192, "value_dim": 128, "page": 64, "turned": 64,
         "interleaved": False, "far": 1 << 18, "kept8": True, "queries": False, "prompts": 3, "dtype": "bf16"},
        # One sequence that has just begun: launch and host cost.
        {"name": "attend_one", "op": "attend", "batch": 1, "shortest": 515, "longest": 515, "idle": 0, "heads": 32, "kv_heads": 8, "key_dim": 128, "value_dim": 128,
         "page": 16, "window": 0, "sinks": False, "kept8": False, "dtype": "bf16"},
        # A decode batch of sequences of every length, two places of it idle.
        {"name": "attend_batch", "op": "attend", "batch": 64, "shortest": 1, "longest": 8192, "idle": 2, "heads": 32, "kv_heads": 8, "key_dim": 128, "value_dim": 128,
         "page": 16, "window": 0, "sinks": False, "kept8": False, "dtype": "bf16"},
        # The same over twice as long contexts kept in 8 bits: the most that is read.
        {"name": "attend_batch_8bit", "op": "attend", "batch": 64, "shortest": 1, "longest": 16384, "idle": 2, "heads": 32, "kv_heads": 8, "key_dim": 128,
         "value_dim": 128, "page": 64, "window": 0, "sinks": False, "kept8": True, "dtype": "bf16"},
        # One very long context, whose length is all there is to split.
        {"name": "attend_long", "op": "attend", "batch": 1, "shortest": 131071, "longest": 131071, "idle": 0, "heads": 32, "kv_heads": 8, "key_dim": 128,
         "value_dim": 128, "page": 32, "window": 0, "sinks": False, "kept8": False, "dtype": "fp16"},
        # A layer that sees the last thousand tokens, with a sink for each head, keys wider than values.
        {"name": "attend_window", "op": "attend", "batch": 96, "shortest": 100, "longest": 12000, "idle": 0, "heads": 64, "kv_heads": 4, "key_dim": 192, "value_dim": 128,
         "page": 64, "window": 1000, "sinks": True, "kept8": False, "dtype": "bf16"},
        # Many query heads over one wide key head, an odd number of sequences.
        {"name": "attend_wide", "op": "attend", "batch": 33, "shortest": 7, "longest": 9001, "idle": 0, "heads": 40, "kv_heads": 1, "key_dim": 256, "value_dim": 256,
         "page": 128, "window": 0, "sinks": False, "kept8": False, "dtype": "fp16"},
    ]


# ---- drawn cases ---------------------------------------------------------------------------------------------------
MAX_TURNED = 4 * 4096 * 40 * 128      # elements of queries and keys in 16 bits: the largest listed
MAX_APPENDED = 8191 * 48 * 128
MAX_READ = 64 * 8192 * 8 * 256 // 3   # elements of keys and values that are attended to


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _heads(rng):
    kv_heads = rng.choice([1, 2, 4, 5, 8, 16])
    return kv_heads * rng.choice([n for n in (1, 2, 3, 4, 6, 8, 16, 20, 40, 128) if n * kv_heads <= 128]), kv_heads


def draw(rng):
    op = rng.choice(["rotary", "append", "attend", "attend"])
    heads, kv_heads = _heads(rng)
    if op == "rotary":
        dim = rng.choice([32, 64, 80, 96, 128, 160, 192, 256])
        batch = rng.choice([1, 1, 2, 3, 8])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        tokens = max(1, min(_log(rng, 1, 16384), MAX_TURNED * 2 // ((heads + kv_heads) * dim * batch * BYTES[dtype])))
        return {"op": op, "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "turned": rng.choice([dim, dim, dim // 2, rng.randrange(2, dim + 1, 2)]), "interleaved": rng.random() < 0.4, "far": _log(rng, 2048, 1 << 21),
                "stretch": rng.choice([1.0, 4.0, 40.0]), "dtype": dtype, "train": rng.random() < 0.6}
    kept8 = rng.random() < 0.4
    key_dim = rng.choice([32, 64, 96, 128, 128, 192, 256])
    value_dim = rng.choice([key_dim, key_dim, 64, 128])
    if not kept8 and rng.random() < 0.2:
        key_dim = value_dim = rng.choice([72, 80, 112])
    page, dtype = rng.choice([16, 32, 64, 128, 256]), rng.choice(["bf16", "bf16", "fp16"])
    if op == "append":
        queries = rng.random() < 0.6
        wide = kv_heads * (key_dim + value_dim) + (heads * key_dim if queries else 0)
        tokens = max(1, min(_log(rng, 1, 16384), MAX_APPENDED // wide))
        return {"op": op, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "key_dim": key_dim, "value_dim": value_dim, "page": page,
                "turned": rng.choice([key_dim // 16 * 16, max(16, key_dim // 32 * 16)]), "interleaved": rng.random() < 0.3, "far": _log(rng, 2048, 1 << 20), "kept8": kept8,
                "queries": queries, "prompts": min(tokens, _log(rng, 1, 256)), "dtype": dtype}
    batch = _log(rng, 1, 256)
    wide = kv_heads * (key_dim + value_dim)
    longest = max(1, min(_log(rng, 1, 131072), MAX_READ // (batch * wide)))
    return {"op": op, "batch": batch, "shortest": _log(rng, 1, longest) if longest > 1 else 1, "longest": longest, "idle": rng.choice([0, 0, batch // 8]), "heads": heads,
            "kv_heads": kv_heads, "key_dim": key_dim, "value_dim": value_dim, "page": page, "window": _log(rng, 1, 8192) if rng.random() < 0.3 else 0,
            "sinks": rng.random() < 0.3, "kept8": kept8, "dtype": dtype}


# ---- inputs --------------------------------------------------------------------------------------------------------
def _frequencies(turned, stretch):
    """Radians a position for every pair; stretched contexts slow down the pairs that turn less than once in 4096 positions, those
    that turn more than 32 times keep their speed, between the two runs a ramp."""
    f = 1.0 / 1e6 ** (torch.arange(0, turned, 2, dtype=torch.float64) / turned)
    turns = 4096 * f / (2 * math.pi)
    keep = ((turns - 1) / 31).clamp(0, 1)
    return (f * keep + f / stretch * (1 - keep)).cuda()


def _lengths(case):
    """From the shortest to the longest, more short ones than long ones; idle places have no token."""
    n = case["batch"]
    part = (torch.arange(n, dtype=torch.float64) / max(1, n - 1)) ** 2
    lengths = (case["shortest"] + part * (case["longest"] - case["shortest"])).round().long()
    if n == 1:
        lengths[:] = case["longest"]
    lengths[:case["idle"]] = 0
    return lengths


def _cache(g, pages, case):
    """Keys and values of every place of every page; a few channels of the keys are several times as large as the others."""
    dtype, kv, kd, vd, page = DTYPES[case["dtype"]], case["kv_heads"], case["key_dim"], case["value_dim"], case["page"]
    k = torch.randn((pages, kv, page, kd), generator=g, device="cuda")
    k *= torch.where(torch.rand((kv, 1, kd), generator=g, device="cuda") < 0.03, 4.0, 1.0)
    v = torch.randn((pages, kv, page, vd), generator=g, device="cuda").to(dtype)
    k = k.to(dtype)
    if not case["kept8"]:
        return {"keys": k.view(pages, kv, page, kd // 8, 8).transpose(2, 3).contiguous(), "values": v, "key_scales": None, "value_scales": None}
    (k, ks), (v, vs) = _keep8(k.float())[:2], _keep8(v.float())[:2]
    return {"keys": k.view(torch.uint8).view(pages, kv, page, kd // 16, 16).transpose(2, 3).contiguous().view(torch.float8_e4m3fn), "values": v,
            "key_scales": ks.transpose(2, 3).contiguous(), "value_scales": vs.transpose(2, 3).contiguous()}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s, dtype = dict(case), DTYPES[case["dtype"]]
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    if case["op"] == "rotary":
        b, t, h, kv, d = case["batch"], case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        fused = randn(b, t, (h + 2 * kv) * d).to(dtype)              # queries, keys and values of a fused projection
        s["q"], s["k"] = fused[..., :h * d].view(b, t, h, d), fused[..., h * d:(h + kv) * d].view(b, t, kv, d)
        first = torch.randint(0, max(1, case["far"] - t), (b, 1), generator=g, device="cuda")
        s["positions"] = first + torch.arange(t, device="cuda")
        s["inv_freq"], s["magnitude"] = _frequencies(case["turned"], case["stretch"]), 0.1 * math.log(case["stretch"]) + 1.0
        if case["train"]:
            s["leaves"] = [s[n].detach().requires_grad_(True) for n in ("q", "k")]
            s["q"], s["k"] = s["leaves"]
            s["dq"], s["dk"] = randn(b, t, h, d).to(dtype), randn(b, t, kv, d).to(dtype)
        return s
    if case["op"] == "append":
        t, h, kv, kd, page = case["tokens"], case["heads"], case["kv_heads"], case["key_dim"], case["page"]
        # sequences of about equal shares of the tokens, each at its own place of its own pages; one token of 29 is padding
        of = (torch.arange(t) * case["prompts"]) // t
        nth = torch.arange(t) - torch.searchsorted(of, of)
        start = torch.randint(0, case["far"], (case["prompts"],), generator=g, device="cuda").cpu()
        places = -(-(int(nth.max()) + 1 + page) // page)
        row = torch.randperm(case["prompts"] * places, generator=g, device="cuda").cpu().view(case["prompts"], places)
        at = start[of] % page + nth
        s["slots"] = torch.where(torch.arange(t) % 29 == 28, -1, row[of, at // page] * page + at % page).cuda()
        s["positions"] = (start[of] + nth).cuda()
        s |= _cache(g, case["prompts"] * places, case)
        wide = (h + kv) * kd + kv * case["value_dim"]
        fused = randn(t, wide).to(dtype)
        s["q"] = fused[:, :h * kd].view(t, h, kd) if case["queries"] else None
        s["k"], s["v"] = fused[:, h * kd:(h + kv) * kd].view(t, kv, kd), fused[:, (h + kv) * kd:].view(t, kv, case["value_dim"])
        s["inv_freq"] = _frequencies(case["turned"], 1.0)
        return s
    lengths, page = _lengths(case), case["page"]
    lengths = lengths[torch.randperm(case["batch"], generator=g, device="cuda").cpu()]
    wide = max(1, -(-case["longest"] // page))
    used = torch.arange(wide)[None] < (lengths[:, None] + page - 1) // page
    total = int(used.sum()) + 3
    table = torch.zeros((case["batch"], wide), dtype=torch.int32)
    table[used] = torch.randperm(total, generator=g, device="cuda").cpu()[:total - 3].int()
    s |= _cache(g, total, case)
    s["pages"], s["lengths"] = table.cuda(), lengths.int().cuda()
    s["q"] = (1.5 * randn(case["batch"], case["heads"], case["key_dim"])).to(dtype)
    s["sink"] = randn(case["heads"]) if case["sinks"] else None
    return s


# ---- the plain forms, in 32 bits --------------------------------------------------------------------------------------
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


def _turned(x, positions, inv_freq, magnitude, interleaved, back=False):
    """Every pair of the first 2 n elements of x [..., heads, d] turned by its angle and stretched, the rest as it is."""
    angle = positions[..., None, None].double() * inv_freq
    c, s = (torch.cos(angle) * magnitude).float(), (torch.sin(angle) * magnitude).float()
    if back:
        s = -s
    n = inv_freq.numel()
    x = x.float()
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    u, w = a * c - b * s, b * c + a * s
    both = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((both, x[..., 2 * n:]), -1)


def _rotary_plain(s):
    dtype = DTYPES[s["dtype"]]
    args = s["positions"], s["inv_freq"], s["magnitude"], s["interleaved"]
    outs = [_turned(s["q"].detach(), *args), _turned(s["k"].detach(), *args)]
    if s["train"]:
        outs += [_turned(s["dq"], *args, back=True), _turned(s["dk"], *args, back=True)]
    return [o.to(dtype) for o in outs]


def _append_plain(s):
    dtype, page = DTYPES[s["dtype"]], s["page"]
    args = s["positions"], s["inv_freq"], 1.0, s["interleaved"]
    real = s["slots"] >= 0
    slots = s["slots"][real]
    at = slots // page, slots % page
    k, v = _turned(s["k"], *args)[real], s["v"][real]
    if s["kept8"]:
        (k, ks), (v, vs) = _keep8(k)[:2], _keep8(v.float())[:2]
        s["key_scales"][at[0], :, :, at[1]] = ks
        s["value_scales"][at[0], :, :, at[1]] = vs
        s["keys"].view(torch.uint8)[at[0], :, :, at[1]] = k.view(torch.uint8).view(*k.shape[:2], -1, 16)
        s["values"].view(torch.uint8)[at[0], :, at[1]] = v.view(torch.uint8)
    else:
        s["keys"][at[0], :, :, at[1]] = k.to(dtype).view(*k.shape[:2], -1, 8)
        s["values"][at[0], :, at[1]] = v
    return _appended(s, _turned(s["q"], *args).to(dtype) if s["queries"] else None)


def _appended(s, q):
    """The cache, and the queries where there are any."""
    outs = [s["keys"], s["values"]] + ([s["key_scales"], s["value_scales"]] if s["kept8"] else [])
    return outs + ([q] if q is not None else [])


def _restored(codes, exponents, dtype):
    """What codes [..., n] with exponents [..., n / 32] stand for, as a program with tensors of `dtype` reads them."""
    e = exponents.int()[..., None]
    groups = codes.float().reshape(*codes.shape[:-1], -1, GROUP) * _power(e - 127).float()
    if dtype == torch.float16:
        groups = groups.clamp(-65504, 65504)
    return groups.reshape(codes.shape).to(dtype).float()


def _attend_plain(s):
    dtype, b, h, kv, page = DTYPES[s["dtype"]], s["batch"], s["heads"], s["kv_heads"], s["page"]
    kd, vd = s["key_dim"], s["value_dim"]
    pages = s["pages"].long()
    n = pages.shape[1] * page
    bytes_of = lambda t: t.view(torch.uint8) if s["kept8"] else t  # noqa: E731     (float8 tensors have no indexing)
    k = bytes_of(s["keys"])[pages].view(s["keys"].dtype).permute(0, 2, 1, 4, 3, 5).reshape(b, kv, n, kd)
    v = bytes_of(s["values"])[pages].view(s["values"].dtype).transpose(1, 2).reshape(b, kv, n, vd)
    if s["kept8"]:
        k = _restored(k, s["key_scales"][pages].permute(0, 2, 1, 4, 3).reshape(b, kv, n, kd // GROUP), dtype)
        v = _restored(v, s["value_scales"][pages].permute(0, 2, 1, 4, 3).reshape(b, kv, n, vd // GROUP), dtype)
    k, v = k.float(), v.float()
    at, lengths = torch.arange(n, device=k.device), s["lengths"][:, None].long()
    seen = at < lengths
    if s["window"]:
        seen = seen & (at >= lengths - s["window"])
    seen = seen[:, None, None]
    scores = s["q"].float().view(b, kv, h // kv, kd) @ k.transpose(2, 3) / math.sqrt(kd)
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    if s["sinks"]:
        sink = s["sink"].view(1, kv, h // kv, 1)
        top = torch.maximum(top, sink)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    if s["sinks"]:
        total = total + torch.exp(sink - top)
    out = p @ torch.where(seen.transpose(2, 3), v, 0.0) / torch.where(total == 0, 1.0, total)
    return out.reshape(b, h, vd).to(dtype)


def _plain(s):
    return {"rotary": _rotary_plain, "append": _append_plain, "attend": _attend_plain}[s["op"]](s)


# ---- the framework's calls ----------------------------------------------------------------------------------------------
def _own(s):
    if s["op"] == "rotary":
        from miles_amd.kernels.rotary import rotary

        q, k = rotary(s["q"], s["k"], s["positions"], s["inv_freq"], interleaved=s["interleaved"], scale=s["magnitude"])
        if not s["train"]:
            return [q, k]
        return [q, k, *torch.autograd.grad((q, k), s["leaves"], (s["dq"], s["dk"]))]
    from miles_amd.kernels.paged_cache import PagedCache, append_tokens

    cache = PagedCache(s["keys"], s["values"], s["key_scales"], s["value_scales"])
    if s["op"] == "append":
        q = append_tokens(cache, s["k"], s["v"], s["slots"], positions=s["positions"], inv_freq=s["inv_freq"], interleaved=s["interleaved"], q=s["q"])
        return _appended(s, q)
    from miles_amd.kernels.paged_attention import paged_attention

    return paged_attention(s["q"], cache, s["pages"], s["lengths"], window=s["window"] or None, sinks=s["sink"])


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definition in 64 bits, written apart from the plain forms ---------------------------------------------------------
def _exact_turned(x, positions, inv_freq, magnitude, interleaved, sign=1.0):
    """Pairs as complex numbers, times magnitude e^(i angle)."""
    n = inv_freq.numel()
    x = x.detach().double()
    wheel = torch.polar(torch.full((), magnitude, dtype=torch.float64, device=x.device), sign * torch.outer(positions.reshape(-1).double(), inv_freq))
    wheel = wheel.view(*positions.shape, 1, n)
    head, tail = x[..., :2 * n], x[..., 2 * n:]
    if interleaved:
        z = torch.view_as_complex(head.reshape(*head.shape[:-1], n, 2).contiguous()) * wheel
        return torch.cat((torch.view_as_real(z).reshape(head.shape), tail), dim=-1)
    z = torch.complex(*head.split(n, dim=-1)) * wheel
    return torch.cat((z.real, z.imag, tail), dim=-1)


def _exact_keep8(x):
    """The codes of an 8-bit copy of x (64 bits) and its exponent bytes."""
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
    v = torch.where(byte[:, None] > 0, rows / power(byte - 127)[:, None], rows).clamp(-448.0, 448.0)
    # e4m3: steps of 2^(floor(log2|v|) - 3), at least 2^-9
    step = power(torch.clamp(torch.floor(torch.log2(v.abs().clamp_min(2.0**-20))), min=-6.0) - 3)
    code = torch.round(v / step) * step                 # (round: to the even neighbour)
    return code.reshape(x.shape), byte.reshape(*x.shape[:-1], -1)


def _exact_append(s):
    page = s["page"]
    args = s["positions"], s["inv_freq"], 1.0, s["interleaved"]
    token = torch.nonzero(s["slots"] >= 0).squeeze(1)
    where, place = torch.div(s["slots"][token], page, rounding_mode="floor"), s["slots"][token].remainder(page)
    k, v = _exact_turned(s["k"], *args)[token], s["v"].double()[token]
    pages, kv = s["values"].shape[:2]
    keys = s["keys"].double().transpose(3, 4).reshape(pages, kv, s["key_dim"], page).permute(0, 3, 1, 2).contiguous()
    values = s["values"].double().permute(0, 2, 1, 3).contiguous()
    back = lambda t: t.permute(0, 2, 1, 3)  # noqa: E731                                        [pages, heads, places, width]
    outs = []
    if s["kept8"]:
        (k, ks), (v, vs) = _exact_keep8(k), _exact_keep8(v)
        for scales, new in ((s["key_scales"], ks), (s["value_scales"], vs)):
            scales = scales.double().permute(0, 3, 1, 2).contiguous()
            scales[where, place] = new
            outs.append(back(scales).transpose(2, 3))
    keys[where, place], values[where, place] = k, v
    x = s["keys"].shape[-1]
    outs = [back(keys).reshape(pages, kv, page, -1, x).transpose(2, 3), back(values)] + outs
    return outs + ([_exact_turned(s["q"], *args)] if s["queries"] else [])


def _exact_attend(s):
    """One sequence after the other, the tokens it sees alone."""
    dtype, kv, page, group = DTYPES[s["dtype"]], s["kv_heads"], s["page"], s["heads"] // s["kv_heads"]
    out = torch.zeros((s["batch"], s["heads"], s["value_dim"]), dtype=torch.float64, device="cuda")
    raw = (lambda t: t.view(torch.uint8)) if s["kept8"] else (lambda t: t)

    def vectors(stored, exponents, ids, first, last, keys):
        t = raw(stored)[ids].view(stored.dtype).double()
        t = t.transpose(2, 3).reshape(len(ids), kv, page, -1) if keys else t
        if exponents is not None:
            scale = torch.exp2(exponents[ids].double() - 127).transpose(2, 3)
            t = (t.view(*t.shape[:-1], -1, GROUP) * scale[..., None]).view(t.shape)
            if dtype == torch.float16:
                t = t.clamp(-65504.0, 65504.0)
            t = t.to(dtype).double()
        return t.transpose(0, 1).reshape(kv, len(ids) * page, -1)[:, first:last]

    for i, n in enumerate(s["lengths"].tolist()):
        if n == 0:
            continue
        low = max(0, n - s["window"]) if s["window"] else 0
        ids = s["pages"][i, low // page:-(-n // page)].long()
        span = ids, low % page, low % page + n - low
        k, v = vectors(s["keys"], s["key_scales"], *span, True), vectors(s["values"], s["value_scales"], *span, False)
        scores = torch.matmul(s["q"][i].double().view(kv, group, -1), k.transpose(1, 2)) * s["key_dim"] ** -0.5
        if s["sinks"]:                                  # one more score, of a token without a value
            scores = torch.cat((scores, s["sink"].double().view(kv, group, 1)), dim=2)
        weights = torch.softmax(scores, dim=2)[:, :, :n - low]
        out[i] = torch.matmul(weights, v).view(s["heads"], -1)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "attend":
        return _exact_attend(s)
    args = s["positions"], s["inv_freq"], s["magnitude"], s["interleaved"]
    outs = [_exact_turned(s["q"], *args), _exact_turned(s["k"], *args)]
    return outs + ([_exact_turned(s["dq"], *args, sign=-1.0), _exact_turned(s["dk"], *args, sign=-1.0)] if s["train"] else [])


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    """Every input byte read once and every output byte written once; of a cache the vectors that are written, or those that are seen.
    Two operations for each product of an attention's sums, a handful for each element elsewhere."""
    size = BYTES[case["dtype"]]
    if case["op"] == "rotary":
        n = case["batch"] * case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (2 * n * size + 8 * case["batch"] * case["tokens"]), "flops": passes * 3 * n}
    stored = KEPT if case["kept8"] else size
    if case["op"] == "append":
        n = case["tokens"] * case["kv_heads"] * (case["key_dim"] + case["value_dim"])
        q = case["tokens"] * case["heads"] * case["key_dim"] if case["queries"] else 0
        return {"bytes": n * (size + stored) + 2 * q * size + 16 * case["tokens"], "flops": 3 * (n + q)}
    lengths = _lengths(case)
    seen = int((lengths.clamp(max=case["window"]) if case["window"] else lengths).sum())
    wide = case["key_dim"] + case["value_dim"]
    return {"bytes": seen * case["kv_heads"] * wide * stored + case["batch"] * case["heads"] * wide * size + 4 * case["batch"],
            "flops": 2 * seen * case["heads"] * wide}
