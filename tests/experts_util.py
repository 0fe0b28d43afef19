"""Inputs and error bounds of the tests of 4-bit products and routed experts."""
import torch

from cache_util import UNIT
from oracle import cache as oc


def sums(K):
    """Error of an fp32 sum of K exact products, of its sum of magnitudes: a rounding for every eight products that an MFMA
    takes together, and some for joining waves and parts."""
    return (K / 8 + 64) * 2.0 ** -24


def four_bit(g, *shape, std=1.0, pad=0, shift=0):
    """Codes and scales of normal values [..., K] on the CPU; scales with rows `pad` bytes longer, `shift` bytes behind an
    allocation's start."""
    x = torch.randn(*shape, generator=g) * std * torch.exp(0.5 * torch.randn(*shape[:-1], 1, generator=g))
    codes, scales = oc.fp4_encode(x)
    return codes, lay_scales(scales, pad, shift)


def lay_scales(scales, pad, shift):
    rows = scales.numel() // scales.shape[-1]
    width = scales.shape[-1] + pad
    flat = torch.full((rows * width + shift,), 255, dtype=torch.uint8)
    flat[shift:].view(rows, width)[:, :scales.shape[-1]] = scales.reshape(rows, -1)
    strides = [1]
    for i, n in enumerate(reversed(scales.shape[1:])):
        strides.insert(0, strides[0] * (n if i else width))
    return flat.as_strided(scales.shape, strides, shift)


def to_dev(t, dev):
    """The same values at the same strides and offset on the device (Tensor.to would close the gaps)."""
    if t is None:
        return None
    n = t.storage_offset() + sum((s - 1) * st for s, st in zip(t.shape, t.stride())) + 1
    whole = t.as_strided((n,), (1,), 0).to(dev)
    return whole.as_strided(t.shape, t.stride(), t.storage_offset())


def product_tolerance(out, mag, K, dtype):
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
    return UNIT[dtype] * out.abs() + 1.01 * sums(K) * mag + tiny
