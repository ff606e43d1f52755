"""Plain CPU restatements, in 64 bits, of the feature-image operators (``dr.group_norm``,
``dr.dropout``) and of the random bits their masks come from."""

import torch

U = 2.0**-24  # half a unit in the last place of float32


def philox4x32_10(counter, key):
    """Four 32-bit words (ints) for a counter of four words and a key of two: Salmon, Moraes, Dror
    and Shaw, "Parallel random numbers: as easy as 1, 2, 3" (2011)."""
    c, k = list(counter), list(key)
    for _ in range(10):
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & 0xFFFFFFFF, (p0 >> 32) ^ c[3] ^ k[1], p0 & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def threshold(p: float) -> int:
    return min(65535, int(p * 65536 + 0.5))


def keep_mask(count: int, p: float, seed: int, layer: int = 0, first: int = 0) -> torch.Tensor:
    """Which of the elements ``first .. first + count - 1`` are kept."""
    seed &= (1 << 64) - 1
    key = (seed & 0xFFFFFFFF, seed >> 32)
    bits = []
    for block in range(first // 8, (first + count + 7) // 8):
        for word in philox4x32_10((block & 0xFFFFFFFF, block >> 32, layer, 0), key):
            bits += [word & 0xFFFF, word >> 16]
    skip = first % 8
    return torch.tensor(bits[skip:skip + count]) >= threshold(p)


def keep_scale(p: float) -> float:
    return 65536 / (65536 - threshold(p))


def activate(z, activation: str):
    if activation == "silu":
        return z * torch.sigmoid(z)
    return torch.relu(z) if activation == "relu" else z


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, activation="none", factor=None):
    """Group norm of ``[batch, ..., channels]`` with 64-bit arithmetic and autograd; ``factor`` is
    the dropout's mask times its scale."""
    batch, channels = x.shape[0], x.shape[-1]
    v = x.double().reshape(batch, -1, groups, channels // groups)
    mean = v.mean((1, 3), keepdim=True)
    d = v - mean
    h = (d / (d.square().mean((1, 3), keepdim=True) + eps).sqrt()).reshape(batch, -1, channels)
    if weight is not None:
        h = h * weight.double().reshape(-1, 1, channels)
    if bias is not None:
        h = h + bias.double().reshape(-1, 1, channels)
    y = activate(h, activation).reshape(x.shape)
    return y if factor is None else y * factor
