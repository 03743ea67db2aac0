"""The latent cache of the MLA models in 4 and 8 bits: sizes, and what a row stands for, in plain PyTorch.

A token's row holds its normed latent (width L) in codes with a scale per group and its rotated key part (width R) in 16 bits:

* 4 bits: groups of 16, the scale their largest magnitude / 7 to four significant bits (2^-20 to 1.875 * 2^10), codes the nearest of -7 to 7;
* 8 bits: groups of 32, the scale the smallest power of two (2^-15 to 2^7) that brings their largest magnitude to 448 or less, codes e4m3.

A group with a value that is no finite number reads back as NaN. Values are exact in bf16. On the GPU a row is bytes (`csrc/mla_cache.cuh` has their order);
the CPU engine keeps the values themselves in its float cache, as it does for the other quantised caches.
"""
from __future__ import annotations

import torch

BITS = {"int4": 4, "fp8": 8}             # kv_dtype -> bits of a latent; every other kv_dtype keeps latents in the compute dtype
GROUP = {4: 16, 8: 32}
ATTENDED = (64, 128, 256, 512)           # latent widths that the attention kernel takes; rows are written and read back at every width that fits


def latent_bits(kv_dtype: str) -> int:
    return BITS.get(kv_dtype, 16)


def fits(L: int, R: int, bits: int) -> bool:
    return bits in GROUP and R == 64 and 64 <= L <= 512 and L % 64 == 0


def row_bytes(L: int, R: int, bits: int) -> int:
    """Bytes of a token's row (16 bits: the plain row)."""
    if bits == 16:
        return 2 * (L + R)
    if not fits(L, R, bits):
        raise ValueError(f"latents of width {L} beside {R} in {bits} bits: the cache takes multiples of 64 up to 512, beside 64, in 4 or 8 bits")
    return (L * bits // 8 + 2 * R + L // GROUP[bits] + 15) // 16 * 16


def quantised(y: torch.Tensor, bits: int) -> torch.Tensor:
    """The values that rows [.., L] (64 bits) read back as, in 64 bits."""
    g = y.double().reshape(*y.shape[:-1], -1, GROUP[bits])
    bad = ~torch.isfinite(g).all(-1, keepdim=True)
    top = torch.where(bad, 0.0, g).abs().amax(-1, keepdim=True)
    if bits == 4:
        m, e = torch.frexp(top / 7)
        s = torch.ldexp(torch.round(m * 16), e - 4).clamp(2.0 ** -20, 1.875 * 2.0 ** 10)
        v = torch.round(g / s).clamp(-7, 7) * s
    else:
        m, e = torch.frexp(top / 448)
        s = torch.ldexp(torch.ones_like(top), torch.where(top > 0, torch.where(m > 0.5, e, e - 1), -15).clamp(-15, 7))
        x = g / s
        step = torch.ldexp(torch.ones_like(x), (torch.frexp(x).exponent - 1).clamp(-6, 8) - 3)
        v = (torch.round(x / step) * step).clamp(-448, 448) * s
    return torch.where(bad, float("nan"), v).reshape(y.shape)
