"""Shared inputs and tolerances of the 4-bit cache's tests."""
from __future__ import annotations

import numpy as np
import torch

from conftest import bits
from oracle import fp4


def random_rows(seed: int, *shape, spread: float = 0.7):
    """bf16 rows whose channels differ in size, some by several times, as keys' do."""
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * torch.exp(spread * torch.randn(*shape[-2:], generator=g))).bfloat16()


class Cache:
    """A 4-bit cache full of quantized rows: tensors for the device, and its values in 64 bits."""

    def __init__(self, seed: int, pages: int, page_size: int, heads: int, dim: int, layout: str):
        self.layout, self.page_size = layout, page_size
        data, scale, values = [], [], []
        for i in range(2):
            codes, powers = fp4.quantize(bits(random_rows(seed + i, pages, page_size, heads, dim)))
            d, s = fp4.pack(codes), powers.transpose(0, 2, 3, 1)
            data.append(torch.from_numpy(d if layout == "NHD" else np.ascontiguousarray(d.transpose(0, 2, 1, 3))))
            scale.append(torch.from_numpy(np.ascontiguousarray(s)))
            values.append(fp4.dequantize(codes, powers))
        self.tensors = data + scale
        self.k, self.v = values

    def on(self, mas, dev):
        return mas.page.Fp4KVCache(*(t.to(dev) for t in self.tensors))


def tolerance(out, size, reach: float, positions: int, p_round: float):
    """What a kernel's bf16 output may be off by, elementwise.

    out: the exact outputs; size: the same sums over |v|; reach: the largest sum of a score's absolute terms.
    The products of bf16 queries and decoded keys are exact in fp32; the sum of up to 256 of them, the scale and the
    distance to the reference add up to 260 roundings of 2^-24 of reach. That moves a weight by as much, relatively, and
    the sum of weights that it is divided by: twice. Each weight is rounded by p_round and enters sums of `positions`
    fp32 terms above and below the fraction (2^-24 each). The output is rounded once to bf16, 2^-8 of itself.
    """
    score = reach * 260 * 2.0 ** -24
    weights = 2 * score * (1 + score) + p_round + 2 * positions * 2.0 ** -24 + 2.0 ** -20
    return np.abs(out) * 2.0 ** -8 + size * weights * (1 + 2.0 ** -8) + 1e-30


P_TWO_TERMS = 2.0 ** -16   # a weight as two bf16 terms: half a step of a half step
P_BF16 = 2.0 ** -8         # a weight rounded to bf16


def check(got: torch.Tensor, exact, positions: int, p_round: float):
    out, size, reach = exact
    y = got.detach().float().cpu().numpy().astype(np.float64)
    off = np.abs(y - out)
    allowed = tolerance(out, size, reach, positions, p_round)
    assert np.isfinite(y).all()
    assert (off <= allowed).all(), f"off by up to {(off / allowed).max():.3f} of what is allowed"
