"""AdamW in 64 bits, from its definition, on the CPU (for tests/test_gpu_adamw.py): one step from a
given state, the 8-bit codes included."""
import math

import torch

BLOCK = 256
GRID = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()   # 0 ... 448


def mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x6a09e667) & 0xffffffff
    x = x ^ (x >> 15)
    x = (x * 0xbb67ae85) & 0xffffffff
    return x ^ (x >> 16)


def random_words(index, seed, step):
    """32 random bits for the elements `index` (int64) of the state."""
    key = mix((mix(torch.tensor(seed & 0xffffffff)) + step) & 0xffffffff)
    return mix(mix((key + (index >> 32)) & 0xffffffff) ^ (index & 0xffffffff))


def to_codes(x, random16, positive):
    """(values of e4m3, scales) of `x` [blocks, 256] float64."""
    finite = torch.isfinite(x)
    mag = torch.where(finite, x.abs(), 0.0)
    scale = mag.amax(1, keepdim=True).float() * torch.tensor(1 / 448, dtype=torch.float32)
    scale = torch.where(scale >= 2.0 ** -100, scale, torch.zeros_like(scale))
    y = torch.where(scale > 0, mag / scale.double(), 0.0).clamp(max=448.0)
    at = torch.searchsorted(GRID, y.contiguous(), right=True) - 1
    above = torch.cat([GRID[1:], GRID[-1:]])
    gap = (above[at] - GRID[at]).clamp(min=1e-300)
    q = torch.where((y - GRID[at]) / gap + (random16.double() + 0.5) / 65536 >= 1, above[at], GRID[at])
    if positive:
        q = torch.where((mag.float() > 0) & (q == 0), GRID[1], q)
    return torch.where(finite, torch.copysign(q, x), math.nan), scale


def step(p, g, m, v, t, lr, b1, b2, eps, decay, coef):
    """(p, m, v, size of the change) after step t, everything float64."""
    g = g * coef
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    change = lr / (1 - b1 ** t) * m / (v.sqrt() / math.sqrt(1 - b2 ** t) + eps)
    return p * (1 - lr * decay) - change, m, v, change
