"""The operators around the 4-bit KV cache, restated in 64 bits - test infrastructure (see oracle/__init__.py).

Written from the definitions, not from any kernel source: a block of 32 elements is 32 e2m1 codes under one power of
two; the codes are found by a search over their eight magnitudes, the power by a search over the powers; attention is
the softmax formula row by row; the step plan a loop over rows and tokens. Arrays are numpy: bf16 as uint16 bit
patterns (oracle.numerics), codes and powers as uint8.

Pinned by tests/test_oracle_fp4.py: closed-form blocks (ties, the power's borders, zeros, NaN), every e2m1 code
through both directions, the half-step bound on random rows; attention against torch's scaled_dot_product_attention in
64 bits; the plan against hand-written steps.
"""
from __future__ import annotations

import numpy as np

from .numerics import bf16_to_f32

BLOCK = 32
MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(bits: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """bf16 bits [..., dim] -> codes [..., dim] (one a byte, 0..15) and powers [..., dim / 32]."""
    x = bf16_to_f32(bits).astype(np.float64).reshape(bits.shape[:-1] + (bits.shape[-1] // BLOCK, BLOCK))
    with np.errstate(invalid="ignore"):
        top = np.abs(x).max(-1)
    finite = np.isfinite(top)
    top = np.where(finite, top, 1.0)
    powers = np.zeros(top.shape, dtype=np.int64)
    for s in range(254, -1, -1):                       # the smallest s with top < 7 * 2^(s - 127)
        powers = np.where(top < 7.0 * 2.0 ** (s - 127), s, powers)
    y = np.abs(np.where(finite[..., None], x, 0.0)) / 2.0 ** (powers[..., None] - 127.0)
    dist = np.abs(y[..., None] - MAGNITUDES)
    best = dist.min(-1, keepdims=True)
    tied = dist == best                                # a tie lies between neighbours: the even code
    code = np.where(tied.sum(-1) > 1, np.where(tied[..., ::2].any(-1), 2 * np.argmax(tied[..., ::2], -1), 0),
                    np.argmax(tied, -1)).astype(np.uint8)
    code |= (np.signbit(x).astype(np.uint8) << 3)
    code = np.where(finite[..., None], code, 0).astype(np.uint8)
    return code.reshape(bits.shape), np.where(finite, powers, 255).astype(np.uint8)


def pack(codes: np.ndarray) -> np.ndarray:
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).astype(np.uint8)


def unpack(packed: np.ndarray) -> np.ndarray:
    return np.stack((packed & 15, packed >> 4), -1).reshape(packed.shape[:-1] + (-1,))


def dequantize(codes: np.ndarray, powers: np.ndarray) -> np.ndarray:
    """Codes [..., dim] and powers [..., dim / 32] -> float64 values (infinite where bf16 has no number so large)."""
    v = MAGNITUDES[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    p = np.where(powers == 255, np.nan, 2.0 ** (powers.astype(np.float64) - 127))
    return (v.reshape(powers.shape + (BLOCK,)) * p[..., None]).reshape(codes.shape)


def cache_rows(data: np.ndarray, scale: np.ndarray, layout: str) -> np.ndarray:
    """A cache's values as float64 [pages, page_size, heads, dim]."""
    d = data if layout == "NHD" else data.transpose(0, 2, 1, 3)
    return dequantize(unpack(d), scale.transpose(0, 3, 1, 2))


def _attend(q, k, v, scale, last):
    """softmax attention of q [n, dim] over k, v [L, dim], row i over positions 0..last[i]; also the same sum over
    |v| (the size of what was added up) and the largest sum of a score's |q k| terms (the size of its terms)."""
    out, size = np.zeros_like(q), np.zeros_like(q)
    reach = 0.0
    for i in range(q.shape[0]):
        m = int(last[i]) + 1
        if m <= 0:
            continue
        s = k[:m] @ q[i] * scale
        with np.errstate(invalid="ignore"):
            w = np.exp(s - s.max())
        w /= w.sum()
        out[i], size[i] = w @ v[:m], w @ np.abs(v[:m])
        reach = max(reach, float((np.abs(k[:m]) @ np.abs(q[i])).max()) * abs(scale))
    return out, size, reach


def decode_attention(q_bits, k, v, tables, seq_lens, scale, scale2=1.0):
    """k, v float64 [pages, page_size, Hk, dim]. Returns float64 (out, size, reach), out [B, Hq, dim]; see _attend."""
    return context_attention(q_bits, k, v, tables, seq_lens, np.arange(len(seq_lens) + 1), scale, scale2)


def context_attention(q_bits, k, v, tables, seq_lens, cu, scale, scale2=1.0):
    q = bf16_to_f32(q_bits).astype(np.float64)
    page_size, hk = k.shape[1], k.shape[2]
    group = q.shape[1] // hk
    out, size, reach = np.zeros_like(q), np.zeros_like(q), 0.0
    for r in range(len(cu) - 1):
        a, b, n = int(cu[r]), int(cu[r + 1]), int(seq_lens[r])
        if b <= a or n <= 0:
            continue
        pos = np.arange(n)
        pages = np.asarray(tables[r], dtype=np.int64)[pos // page_size]
        kr, vr = k[pages, pos % page_size], v[pages, pos % page_size]
        last = np.arange(a, b) - b + n
        for h in range(q.shape[1]):
            o, z, t = _attend(q[a:b, h], kr[:, h // group], vr[:, h // group], scale, last)
            out[a:b, h], size[a:b, h], reach = o * scale2, z * abs(scale2), max(reach, t)
    return out, size, reach


def plan_step(new, cached, tables, free_pages, free_range, page_size, num_tokens):
    """Rows and tokens in turn. Returns a dict of the outputs, `tables` a grown copy, and the error bits."""
    tables = np.array(tables)
    head, tail = int(free_range[0]), int(free_range[1])
    n_free = min(max(0, tail - head), len(free_pages)) if head >= 0 else 0
    taken, bits, full = 0, 0, False
    positions, rows, slots, cu, lens = [], [], [], [0], []
    for r in range(len(new)):
        n, c = int(new[r]), int(cached[r])
        lens.append(c)
        if n < 0 or c < 0 or c + n > tables.shape[1] * page_size:
            bits |= 2
            n = 0
        else:
            need = -(-(c + n) // page_size) - -(-c // page_size)
            if full or len(positions) + n > num_tokens or taken + need > n_free:
                full = True
                if n > 0:
                    bits |= 64
                n = 0
        for p in range(c, c + n):
            block = p // page_size
            if block >= -(-c // page_size) and p % page_size == 0:
                tables[r, block] = free_pages[(head + taken) % len(free_pages)]
                taken += 1
            page = int(tables[r, block])
            if page < 0:
                bits |= 8
            positions.append(p)
            rows.append(r)
            slots.append(page * page_size + p % page_size if page >= 0 else -1)
        lens[-1] = c + n
        cu.append(len(positions))
    pad = num_tokens - len(positions)
    return {"positions": positions + [0] * pad, "batch_indices": rows + [-1] * pad, "slot_mapping": slots + [-1] * pad,
            "cu_seqlens_q": cu, "seq_lens": lens, "free_range": [head + taken, tail], "tables": tables, "bits": bits}
