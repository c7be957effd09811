"""Inputs and 64-bit definitions for the tests of the 4-bit operators (CPU and GPU)."""
import torch


def offsets_of(counts, head=0, device="cpu"):
    off = torch.tensor([0] + list(counts)).cumsum(0) + head
    return off.to(torch.int32).to(device)


def e2m1_round64(y):
    """Nearest e2m1 value, ties to the even code, saturating at 6."""
    a = y.abs()
    unit = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).to(torch.float64)
    return (torch.round(a / unit) * unit).clamp(max=6.0) * torch.sign(y)


def e4m3_round64(t):
    t = t.clamp(max=448.0)
    ulp = torch.exp2(torch.floor(torch.log2(t.clamp(min=2.0 ** -6))) - 3)
    return torch.round(t / ulp) * ulp


def quantise64(x, block, g=None):
    """(values q, scales s) of the definition: x ~ q s g."""
    v = x.double().unflatten(-1, (-1, block))
    amax = v.abs().amax(-1)
    if block == 16:
        gg = 1.0 if g is None else g.double().reshape(-1, *([1] * (amax.dim() - 1)))
        s = e4m3_round64(amax / (6 * gg))
        d = s * gg
    else:
        s = torch.where(amax > 0, torch.exp2(torch.ceil(torch.log2((amax / 6).clamp(min=2.0 ** -126)))), torch.full_like(amax, 2.0 ** -127))
        d = s
    q = torch.where((d > 0)[..., None], e2m1_round64(v / torch.where(d > 0, d, torch.ones_like(d))[..., None]), torch.zeros_like(v))
    return q.flatten(-2), s


def values64(q, s, g=None):
    """Packed codes and scales to values, without the library."""
    c = torch.stack([q & 15, q >> 4], -1).flatten(-2).long()
    mag = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=q.device)[c & 7]
    v = torch.where(c >= 8, -mag, mag)
    d = s.double() if s.dtype == torch.float8_e4m3fn else torch.exp2(s.view(torch.uint8).double() - 127)
    if g is not None:
        d = d * g.double().reshape(-1, *([1] * (d.dim() - 1)))
    return v * d.repeat_interleave(v.shape[-1] // d.shape[-1], -1)


def random_fp4(shape, fmt, gen, device="cpu"):
    """Random codes (all sixteen) and scales over a few octaves, straight from bits."""
    *lead, k = shape
    q = torch.randint(0, 256, (*lead, k // 2), generator=gen, dtype=torch.uint8)
    if fmt == "nvfp4":
        s = torch.exp2(torch.rand(*lead, k // 16, generator=gen) * 6 - 2).to(torch.float8_e4m3fn)
    else:
        s = torch.randint(120, 131, (*lead, k // 32), generator=gen, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    return q.to(device), s.to(device)
