"""The 4-bit cache's format in plain torch, on the CPU in 64 bits."""
import torch

LEVELS = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def encode(x):
    """x [..., hd] as (codes [..., hd / 2], scales [..., hd / 32]), by search over the levels."""
    shape = x.shape
    x = x.double().reshape(-1, 32)
    odd = ~torch.isfinite(x).all(-1)
    top = torch.where(odd[:, None], 1.0, x).abs().amax(-1)
    e = torch.full_like(top, -40)
    for k in range(-40, 130):   # the largest power of two that is not above the maximum
        e = torch.where(top >= 2.0 ** k, float(k), e)
    e = torch.where(top > 1.75 * 2.0 ** e, e + 1, e) - 2
    e = e.clamp(-23, 13)
    y = (x.abs() / 2.0 ** e[:, None]).clamp(max=6.0)
    off = (y[..., None] - LEVELS).abs()
    near = off.amin(-1, keepdim=True)
    # of two equally near levels the even code
    rank = torch.where(off == near, torch.tensor([0, 1, 0, 1, 0, 1, 0, 1]), 2)
    code = rank.argmin(-1) + 8 * torch.signbit(x)
    code = torch.where(odd[:, None], 0, code).view(*shape[:-1], shape[-1] // 2, 2)
    scale = torch.where(odd, 255, e + 127).view(*shape[:-1], shape[-1] // 32)
    return (code[..., 0] + 16 * code[..., 1]).to(torch.uint8), scale.to(torch.uint8)


def decode(codes, scales):
    """The values of such bytes."""
    signed = torch.cat([LEVELS, -LEVELS])
    c = codes.long()
    x = torch.stack([signed[c & 15], signed[c >> 4]], -1).flatten(-2)
    s = 2.0 ** (scales.double() - 127)
    s = torch.where(scales > 140, torch.nan, s)
    return (x * s.repeat_interleave(32, -1)).half().double()   # exact for scales of 104 to 140


def random_cache(gen, rows, kvh, hd, lo=122, hi=129):
    """Codes and scale bytes of lo .. hi - 1."""
    return (torch.randint(0, 256, (rows, kvh, hd // 2), generator=gen, dtype=torch.uint8),
            torch.randint(lo, hi, (rows, kvh, hd // 32), generator=gen, dtype=torch.uint8))
