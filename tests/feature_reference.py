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
    """Which of the elements ``first .. first + count - 1`` are kept: the generator again, for all
    counters at once."""
    seed &= (1 << 64) - 1
    block = torch.arange(first // 8, (first + count + 7) // 8)
    word = 0xFFFFFFFF
    c = [block & word, block >> 32, torch.full_like(block, layer), torch.zeros_like(block)]
    k = [seed & word, seed >> 32]
    for _ in range(10):
        # Products wrap in signed 64 bits, which keeps all their bits.
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [((p1 >> 32) & word) ^ c[1] ^ k[0], p1 & word, ((p0 >> 32) & word) ^ c[3] ^ k[1], p0 & word]
        k = [(k[0] + 0x9E3779B9) & word, (k[1] + 0xBB67AE85) & word]
    bits = torch.stack([half for w in c for half in (w & 0xFFFF, w >> 16)], 1).reshape(-1)
    return bits[first % 8:first % 8 + count] >= threshold(p)


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
