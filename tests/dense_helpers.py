"""Helpers of the dense products' tests: random 4-bit GGUF rows, their values in 64 bits by the C oracle (the reference's
dequant), activations and their slopes in 64 bits."""

import numpy as np

from oracle import lib as olib

TYPES = {"Q4_0": (32, 18), "Q4_1": (32, 20), "Q4_K": (256, 144), "IQ4_NL": (32, 18)}  # values, bytes a block
EPS = {"bf16": 2.0 ** -7, "f16": 2.0 ** -10, "f32": 2.0 ** -23}


def random_rows(rng, qtype: str, n: int, k: int, scale: float = 0.02) -> np.ndarray:
    """(n, row bytes) random blocks: any codes and 6-bit scales, fp16 scales around ``scale``."""
    per, size = TYPES[qtype]
    b = rng.integers(0, 256, (n, k // per, size), dtype=np.uint8)

    def half(lo, hi):
        return rng.uniform(lo, hi, (n, k // per, 1)).astype(np.float16).view(np.uint8)

    if qtype == "Q4_K":
        b[..., 0:2], b[..., 2:4] = half(scale / 64, scale / 16), half(scale / 16, scale / 8)
    else:
        b[..., 0:2] = half(-scale, scale) if qtype != "IQ4_NL" else half(-scale / 16, scale / 16)
        if qtype == "Q4_1":
            b[..., 2:4] = half(-8 * scale, 0)
    return b.reshape(n, -1)


def values(qtype: str, raw: np.ndarray, k: int) -> np.ndarray:
    """The rows' values in float64 (the oracle's fp32 values: each exact or rounded once, 2^-24)."""
    return olib.oracle().dequant_rows(qtype, raw, k).astype(np.float64)


def parts(qtype: str, raw: np.ndarray, k: int) -> np.ndarray:
    """|code x scale| + |minimum| of every value: the magnitudes whose roundings a product can carry."""
    w = np.abs(values(qtype, raw, k))
    if qtype not in ("Q4_1", "Q4_K"):
        return w
    # the value with its code zeroed is the minimum alone
    per, size = TYPES[qtype]
    z = raw.reshape(raw.shape[0], k // per, size).copy()
    z[..., 4 if qtype == "Q4_1" else 16:] = 0
    m = np.abs(values(qtype, z.reshape(raw.shape), k))
    return w + 2 * m


def act(name: str, z):
    import torch
    if name == "silu":
        return z * torch.sigmoid(z)
    return 0.5 * z * (1 + torch.tanh((2 / np.pi) ** 0.5 * (z + 0.044715 * z ** 3)))


def slope(name: str, z):
    import torch
    if name == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    c = (2 / np.pi) ** 0.5
    r = torch.tanh(c * (z + 0.044715 * z ** 3))
    return 0.5 * (1 + r) + 0.5 * z * (1 - r * r) * c * (1 + 3 * 0.044715 * z * z)


def torch_dtype(name: str):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]
