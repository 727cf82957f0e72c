"""The 4-bit cache's oracle (oracle/fp4.py) pinned to closed forms and to torch in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import bits
from oracle import fp4
from oracle.numerics import bf16_to_f32


def _block(*values):
    return bits(torch.tensor(list(values) + [0.0] * (32 - len(values))).bfloat16())


@pytest.mark.parametrize("power", [1, 100, 127, 200, 250])
def test_every_code_survives_both_directions(power):
    """A block of the sixteen values under a power, its largest 6 of it, quantizes to itself."""
    values = np.concatenate((fp4.MAGNITUDES, -fp4.MAGNITUDES)) * 2.0 ** (power - 127)
    codes, powers = fp4.quantize(_block(*values))
    assert powers.tolist() == [power]
    assert codes[:16].tolist() == list(range(16))
    assert np.array_equal(fp4.dequantize(codes, powers)[:16], values)


@pytest.mark.parametrize("x,code", [(0.25, 0), (0.75, 2), (1.25, 2), (1.75, 4), (2.5, 4), (3.5, 6), (5.0, 6),
                                    (0.26, 1), (0.24, 0), (5.03125, 7), (4.96875, 6), (-0.75, 10), (-0.25, 8)])
def test_ties_go_to_the_even_code(x, code):
    codes, powers = fp4.quantize(_block(6.0, x))
    assert powers.tolist() == [127] and codes[:2].tolist() == [7, code]


@pytest.mark.parametrize("top,power", [(6.96875, 127), (7.0, 128), (3.484375, 126), (3.5, 127), (0.0, 0), (2.0 ** -126, 0),
                                       (6.9375 * 2.0 ** -127, 0), (7.0 * 2.0 ** -127, 1)])
def test_the_power_is_the_smallest_under_which_nothing_is_cut_off(top, power):
    assert fp4.quantize(_block(top))[1].tolist() == [power]


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_block_with_a_non_number_is_nan(bad):
    codes, powers = fp4.quantize(_block(1.0, bad))
    assert powers.tolist() == [255] and not codes.any() and np.isnan(fp4.dequantize(codes, powers)).all()


@pytest.mark.parametrize("scale", [2.0 ** -130, 1e-20, 1.0, 3e5, 1e30])
def test_elements_are_off_by_at_most_half_a_step(scale):
    """Steps are 1/2 below 2, 1 below 4 and 2 below 6 (and 6 to 7 rounds to 6), in units of the power."""
    x = bits((torch.randn(64, 128, generator=torch.Generator().manual_seed(1)) * scale).bfloat16())
    codes, powers = fp4.quantize(x)
    unit = np.repeat(2.0 ** (powers.astype(np.float64) - 127), 32, -1)
    want, got = bf16_to_f32(x).astype(np.float64) / unit, fp4.dequantize(codes, powers) / unit
    half = np.where(np.abs(want) <= 2, 0.25, np.where(np.abs(want) <= 4, 0.5, 1.0))
    assert np.abs(want).max() < 7 and (np.abs(got - want) <= half).all()
    assert np.array_equal(fp4.unpack(fp4.pack(codes)), codes)


def test_attention_is_torchs():
    g = torch.Generator().manual_seed(2)
    q = torch.randn(7, 4, 64, generator=g).bfloat16()
    k, v = torch.randn(6, 16, 2, 64, generator=g).double(), torch.randn(6, 16, 2, 64, generator=g).double()
    tables, lens, cu = np.array([[4, 0], [3, 1], [5, 2]]), [20, 9, 31], [0, 3, 3, 7]
    out, size, *_ = fp4.context_attention(bits(q), k.numpy(), v.numpy(), tables, lens, cu, 0.2, 1.5)
    for r in (0, 2):
        rows = lambda c: c[torch.tensor(tables[r])].flatten(0, 1)[:lens[r]].transpose(0, 1).repeat_interleave(2, 0)
        n = cu[r + 1] - cu[r]
        mask = torch.ones(n, lens[r], dtype=torch.bool).tril(lens[r] - n)
        want = torch.nn.functional.scaled_dot_product_attention(q[cu[r]:cu[r + 1]].double().transpose(0, 1), rows(k),
                                                                rows(v), attn_mask=mask, scale=0.2)
        np.testing.assert_allclose(out[cu[r]:cu[r + 1]], 1.5 * want.transpose(0, 1).numpy(), rtol=1e-12, atol=1e-12)
    assert (size >= np.abs(out)).all()


def test_plan_of_a_step_by_hand():
    tables = np.full((4, 3), 99)
    tables[0, 0], tables[1, 0] = 7, 8
    got = fp4.plan_step([1, 3, 0, 5], [4, 3, 0, 0], tables, [50, 51, 52, 53, 54], [9, 13], 4, 12)
    # row 0 opens a block at position 4, row 1 fills its first and opens its second, row 3 opens two
    assert got["positions"] == [4, 3, 4, 5, 0, 1, 2, 3, 4, 0, 0, 0]
    assert got["batch_indices"] == [0, 1, 1, 1, 3, 3, 3, 3, 3, -1, -1, -1]
    assert got["slot_mapping"] == [54 * 4, 8 * 4 + 3, 200, 201, 204, 205, 206, 207, 208, -1, -1, -1]
    assert got["cu_seqlens_q"] == [0, 1, 4, 4, 9] and got["seq_lens"] == [5, 6, 0, 5] and got["free_range"] == [13, 13]
    assert got["tables"].tolist() == [[7, 54, 99], [8, 50, 99], [99, 99, 99], [51, 52, 99]] and got["bits"] == 0


def test_plan_stops_at_the_first_row_that_does_not_fit():
    t = np.zeros((4, 2), dtype=np.int64)
    got = fp4.plan_step([2, 9, 1, 1], [0, 0, 3, 3], t, [5, 6], [0, 1], 4, 8)       # row 1 is past its table
    assert got["cu_seqlens_q"] == [0, 2, 2, 3, 4] and got["bits"] == 2 and got["seq_lens"] == [2, 0, 4, 4]
    got = fp4.plan_step([2, 5, 1, 1], [0, 0, 3, 3], t, [5, 6], [0, 1], 4, 8)       # row 1 wants two pages
    assert got["cu_seqlens_q"] == [0, 2, 2, 2, 2] and got["bits"] == 64 and got["seq_lens"] == [2, 0, 3, 3]
