"""4-bit codes of a cache in 64 bits on the CPU, straight from their definition.  Test infrastructure only."""
import torch

GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
MOST = {torch.bfloat16: 1.5 * 2.0 ** 127, torch.float16: 49152.0}


def scale_bytes(x, dtype):
    """Bytes of the scales of rows x (float64, dim a multiple of 32): the smallest power of two from 2^-100 on with max|x| <= 6 times it."""
    top = x.reshape(*x.shape[:-1], -1, 32).abs().amax(-1)
    lost = ~torch.isfinite(top)
    top = torch.where(lost, 0.0, top).clamp(max=MOST[dtype])
    e = torch.full(top.shape, -100, dtype=torch.int64)
    for _ in range(230):  # one power of two at a time
        e = torch.where(top > 6.0 * 2.0 ** e.double(), e + 1, e)
    return torch.where(lost, 255, e + 127).to(torch.uint8)


def nearest(x, scales):
    """The value of the grid times the scale that is nearest to each element, ties to the code of even number; NaN where the scale is."""
    s = (2.0 ** (scales.double() - 127)).repeat_interleave(32, -1)
    y = x.nan_to_num(0.0, 0.0, 0.0) / s
    a = y.abs().clamp(max=6.0)
    off = (a[..., None] - GRID).abs()
    order = off * 16 + torch.tensor([0.0, 1e-9] * 4, dtype=torch.float64)  # an odd code loses a tie
    v = GRID[order.argmin(-1)] * torch.where(y < 0, -1.0, 1.0) * s
    return torch.where((scales == 255).repeat_interleave(32, -1), torch.nan, v)


def values(codes, scales):
    """What bytes of two codes and their scales stand for."""
    codes = codes.cpu().long()
    c = torch.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    s = (2.0 ** (scales.cpu().double() - 127)).repeat_interleave(32, -1)
    v = GRID[c & 7] * torch.where(c >= 8, -1.0, 1.0) * s
    return torch.where((scales.cpu() == 255).repeat_interleave(32, -1), torch.nan, v)


def pack(x, dtype=torch.bfloat16):
    """Bytes of codes and scales of rows."""
    x = x.cpu().double()
    scales = scale_bytes(x, dtype)
    v = nearest(x, scales) / (2.0 ** (scales.double() - 127)).repeat_interleave(32, -1)
    c = (v.abs()[..., None] == GRID).int().argmax(-1) + 8 * (v < 0)
    c = c.to(torch.uint8)
    return c[..., ::2] | c[..., 1::2] << 4, scales
