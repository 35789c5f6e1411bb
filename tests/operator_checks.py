"""Plain forms of the training operators in 64 bits, and how far a result may be from them."""

import torch

HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}


def f64(t):
    return t.detach().double()


def within(got, want, slack, what=""):
    """Every value of `got` within half a step of its type of `want`, plus `slack` (a bound on what came before the rounding)."""
    got64 = f64(got)
    assert got64.shape == want.shape, (what, got64.shape, want.shape)
    same = torch.equal(torch.isnan(got64), torch.isnan(want))
    assert same, f"{what}: NaNs elsewhere"
    smallest = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    allowed = HALF_STEP[got.dtype] * (want.abs() + slack) + slack + smallest / 2
    off = torch.where(torch.isnan(want) | (got64 == want), torch.zeros_like(want), (got64 - want).abs())
    worst = (off - allowed).max().item() if off.numel() else 0.0
    assert worst <= 0, f"{what}: {worst:.3g} over the bound, at most {off.max().item():.3g} off values of {want.abs().max().item():.3g}"


def phi(z):
    return torch.special.ndtr(z)


def act64(z, name):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * phi(z)
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (z + 0.044715 * z**3)))
    return z


def slope64(z, name):
    if name is None:
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).double()
    z = z.clone().requires_grad_(True)
    with torch.enable_grad():
        return torch.autograd.grad(act64(z, name).sum(), z)[0]


def restored64(codes, scales):
    """What an 8-bit copy stands for."""
    powers = torch.tensor([2.0 ** (e - 127) for e in range(255)], dtype=torch.float64, device=codes.device)
    groups = codes.double().reshape(*codes.shape[:-1], codes.shape[-1] // 32, 32) * powers[scales.long()].unsqueeze(-1)
    return groups.reshape(codes.shape)
