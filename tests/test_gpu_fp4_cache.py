"""The 4-bit cache's store, append and load on the GPU against the 64-bit oracle: bit for bit."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import bits, from_bits
from fp4_common import random_rows
from oracle import fp4

pytestmark = pytest.mark.gpu
FILL = 0xA5


def _empty(mas, dev, pages, ps, heads, dim, layout):
    c = mas.page.fp4_kv_cache(pages, ps, heads, dim, dev, layout)
    for t in c:
        t.fill_(FILL)
    return c


def _expect(cache, layout, slots, rows, ps):
    """The cache's tensors after rows (keys, values) were put into slots, the rest untouched."""
    want = [np.full(tuple(t.shape), FILL, dtype=np.uint8) for t in cache]
    for i, x in enumerate(rows):
        codes, powers = fp4.quantize(x)
        packed = fp4.pack(codes)
        for t, slot in enumerate(slots):
            if slot >= 0:
                page, entry = slot // ps, slot % ps
                if layout == "NHD":
                    want[i][page, entry] = packed[t]
                else:
                    want[i][page, :, entry] = packed[t]
                want[2 + i][page, :, :, entry] = powers[t]
    return want


def _same(cache, want):
    for name, t, w in zip(("k", "v", "k_scale", "v_scale"), cache, want):
        assert np.array_equal(t.cpu().numpy(), w), name


SHAPES = [  # heads, dim, page_size, tokens, layout
    (8, 128, 16, 64, "HND"), (8, 128, 256, 37, "NHD"), (1, 64, 16, 1, "HND"), (3, 32, 32, 5, "NHD"),
    (2, 256, 64, 19, "HND"), (5, 96, 16, 23, "NHD"), (17, 128, 16, 9, "HND"), (1, 32, 16, 3, "NHD"),
]


@pytest.mark.parametrize("heads,dim,ps,n,layout", SHAPES)
def test_slots_there_and_back(mas, dev, heads, dim, ps, n, layout):
    """Rows taken from column views of one projection's output go to their slots; -1 is skipped; the rows read back are
    exactly the values that the codes stand for."""
    pages = 2 + -(-n // ps)
    qkv = torch.cat((random_rows(1, n, heads, dim).flatten(1), random_rows(2, n, heads, dim).flatten(1),
                     random_rows(3, n, 1, 8).flatten(1)), -1).to(dev)
    key, value = qkv[:, :heads * dim], qkv[:, heads * dim:2 * heads * dim].unflatten(-1, (heads, dim))
    slots = torch.randperm(pages * ps, generator=torch.Generator().manual_seed(4))[:n]
    slots[n // 2] = -1
    cache, flags = _empty(mas, dev, pages, ps, heads, dim, layout), torch.zeros(1, dtype=torch.int32, device=dev)
    mas.store_kv_slots_fp4(key, value, cache, slots.to(dev), layout, error_flags=flags)
    rows = [bits(key).reshape(n, heads, dim), bits(value)]
    _same(cache, _expect(cache, layout, slots.tolist(), rows, ps))
    back = mas.load_kv_slots_fp4(cache, slots.to(dev), layout, error_flags=flags)
    for x, y in zip(rows, back):
        want = fp4.dequantize(*fp4.quantize(x))
        want[n // 2] = 0.0
        assert np.array_equal(y.float().cpu().numpy().astype(np.float64), want)
    assert int(flags) == 0


@pytest.mark.parametrize("ps,layout", [(16, "HND"), (64, "NHD")])
def test_block_table_form(mas, dev, ps, layout):
    """Three rows of odd lengths through block tables; errors are reported and skipped, nothing else is touched."""
    heads, dim, new, cached = 2, 128, [5, 1, 40], [ps - 2, 0, 3]
    n, width = sum(new), 4
    tables = torch.randperm(3 * width, generator=torch.Generator().manual_seed(5)).to(torch.int32).reshape(3, width)
    tables[1, 0] = 99                                               # a page outside the cache
    batch = torch.repeat_interleave(torch.arange(3), torch.tensor(new)).to(torch.int32)
    pos = torch.cat([torch.arange(c, c + m) for c, m in zip(cached, new)]).to(torch.int32)
    batch[-1], pos[-2], pos[-3] = 7, -4, width * ps                  # no such row; below the row; past its table
    key, value = random_rows(6, n, heads, dim), random_rows(7, n, heads, dim)
    slots = []
    for b, p in zip(batch.tolist(), pos.tolist()):
        ok = b < 3 and 0 <= p < width * ps and int(tables[b, p // ps]) < 12
        slots.append(int(tables[b, p // ps]) * ps + p % ps if ok else -1)
    cache, flags = _empty(mas, dev, 12, ps, heads, dim, layout), torch.zeros(1, dtype=torch.int32, device=dev)
    indptr = (torch.arange(4) * width).to(torch.int32)
    mas.append_paged_kv_cache_fp4(key.to(dev), value.to(dev), batch.to(dev), pos.to(dev), cache, tables.flatten().to(dev),
                                  indptr.to(dev), None, layout, error_flags=flags)
    _same(cache, _expect(cache, layout, slots, [bits(key), bits(value)], ps))
    assert int(flags) == 2 | 4 | 8


def test_every_bf16_value(mas, dev):
    """All 65536 bf16 bit patterns, each beside a largest element at several distances above it, and in order."""
    every = np.arange(65536, dtype=np.uint16).reshape(-1, 16)
    tops = np.empty_like(every)
    for i, up in enumerate((0, 0x80, 0x100, 0x17f, 0x180, 0x200, 0x2a0, 0x320) * 2):
        tops[:, i] = np.minimum((every[:, i] & 0x7fff).astype(np.int64) + up, 0x7f7f)
    rows = np.concatenate((every.reshape(-1, 32), np.concatenate((every[:, :8], tops[:, :8], every[:, :8], tops[:, 8:]), 1),
                           np.concatenate((every[:, 8:], tops[:, 8:], every[:, 8:], tops[:, :8]), 1)))
    x = from_bits(rows.reshape(-1, 4, 32))
    n = x.shape[0]
    cache = _empty(mas, dev, -(-n // 16), 16, 4, 32, "HND")
    slots = torch.arange(n, device=dev)
    mas.store_kv_slots_fp4(x.to(dev), x.flip(0).to(dev), cache, slots, "HND")
    _same(cache, _expect(cache, "HND", range(n), [bits(x), bits(x.flip(0))], 16))
    got = mas.load_kv_slots_fp4(cache, slots, "HND")[0].float().cpu().numpy()
    codes, powers = fp4.quantize(bits(x))
    want = fp4.dequantize(codes, powers)
    nan, large = np.isnan(want), np.abs(want) >= 2.0 ** 128       # (rounded past bf16's numbers: infinite, as a cast gives)
    assert np.isnan(got[nan]).all() and np.isinf(got[large]).all()
    rest = ~(nan | large)
    assert np.array_equal(got[rest].astype(np.float64), want[rest])


def test_slots_past_the_cache(mas, dev):
    cache = _empty(mas, dev, 2, 16, 2, 64, "NHD")
    x = random_rows(8, 3, 2, 64).to(dev)
    slots = torch.tensor([3, 32, 1 << 40], device=dev)
    flags = torch.zeros(1, dtype=torch.int32, device=dev)
    mas.store_kv_slots_fp4(x, x, cache, slots, error_flags=flags)
    _same(cache, _expect(cache, "NHD", [3, -1, -1], [bits(x)] * 2, 16))
    assert int(flags) == 16
    flags.zero_()
    key, value = mas.load_kv_slots_fp4(cache, slots, error_flags=flags)
    assert int(flags) == 16 and not key[1:].any() and not value[1:].any() and key[0].any()


def test_nothing_to_do(mas, dev):
    cache = _empty(mas, dev, 2, 16, 2, 64, "NHD")
    none = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=dev)
    mas.store_kv_slots_fp4(none, none, cache, torch.empty(0, dtype=torch.int64, device=dev))
    key, _ = mas.load_kv_slots_fp4(cache, torch.empty(0, dtype=torch.int64, device=dev))
    assert key.shape == (0, 2, 64) and all(bool((t == FILL).all()) for t in cache)


def test_views_of_a_larger_allocation(mas, dev):
    """Caches of one layer out of a pool of layers, with strides of their own; destinations wider than the rows."""
    heads, dim, ps, n = 2, 128, 16, 21
    big = [torch.full((3, 4, heads, ps, 96), FILL, dtype=torch.uint8, device=dev)[1, :, :, :, 16:16 + dim // 2] for _ in range(2)]
    big += [torch.full((4, 3, heads, dim // 32, ps), FILL, dtype=torch.uint8, device=dev)[:, 2] for _ in range(2)]
    cache = mas.page.Fp4KVCache(*big)
    key, value = random_rows(9, n, heads, dim), random_rows(10, n, heads, dim)
    slots = torch.randperm(4 * ps, generator=torch.Generator().manual_seed(11))[:n]
    mas.store_kv_slots_fp4(key.to(dev), value.to(dev), cache, slots.to(dev), "HND")
    _same(cache, _expect(cache, "HND", slots.tolist(), [bits(key), bits(value)], ps))
    assert all(bool((t._base[0] == FILL).all()) for t in big[:2])
    wide = torch.full((n, heads * dim + 64), 7.0, dtype=torch.bfloat16, device=dev)
    out = torch.empty(n, heads, dim, dtype=torch.bfloat16, device=dev)
    mas.load_kv_slots_fp4(cache, slots.to(dev), "HND", key=wide[:, :heads * dim], value=out)
    assert np.array_equal(wide[:, :heads * dim].reshape(n, heads, dim).float().cpu().numpy(),
                          fp4.dequantize(*fp4.quantize(bits(key))).astype(np.float32))
    assert bool((wide[:, heads * dim:] == 7.0).all())


@pytest.mark.parametrize("heads,dim,ps,layout", [(2, 128, 16, "HND"), (9, 64, 32, "NHD"), (1, 64, 256, "HND")])
def test_prompts(mas, dev, heads, dim, ps, layout):
    """Prompts long enough for four tokens per wavefront: rows that start and end inside a group of four, at odd entries,
    whose pages are not in order; some destinations outside the cache. Then the same rows by their slots, and back."""
    new, cached = [1030, 1, 701, 2050, 3], [5, 17, 0, 31, ps - 1]
    n, width = sum(new), max(-(-(c + m) // ps) for c, m in zip(cached, new))
    pages = len(new) * width
    tables = torch.randperm(pages, generator=torch.Generator().manual_seed(12)).to(torch.int32).reshape(len(new), width)
    tables[2, 3] = -1
    batch = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).to(torch.int32)
    pos = torch.cat([torch.arange(c, c + m) for c, m in zip(cached, new)]).to(torch.int32)
    batch[40] = -1
    slots = [int(tables[b, p // ps]) * ps + p % ps if b >= 0 and int(tables[b, p // ps]) >= 0 else -1
             for b, p in zip(batch.tolist(), pos.tolist())]
    key, value = random_rows(13, n, heads, dim), random_rows(14, n, heads, dim)
    cache, flags = _empty(mas, dev, pages, ps, heads, dim, layout), torch.zeros(1, dtype=torch.int32, device=dev)
    indptr = (torch.arange(len(new) + 1) * width).to(torch.int32)
    mas.append_paged_kv_cache_fp4(key.to(dev), value.to(dev), batch.to(dev), pos.to(dev), cache, tables.flatten().to(dev),
                                  indptr.to(dev), None, layout, error_flags=flags)
    want = _expect(cache, layout, slots, [bits(key), bits(value)], ps)
    _same(cache, want)
    lost = any(int(tables[b, p // ps]) < 0 for b, p in zip(batch.tolist(), pos.tolist()) if b >= 0)   # a row that long
    assert int(flags) == (4 | 8 if lost else 4)
    again, s = _empty(mas, dev, pages, ps, heads, dim, layout), torch.tensor(slots, device=dev)
    flags.zero_()
    mas.store_kv_slots_fp4(key.to(dev), value.to(dev), again, s, layout, error_flags=flags)
    _same(again, want)
    for x, y in zip((key, value), mas.load_kv_slots_fp4(again, s, layout, error_flags=flags)):
        back = fp4.dequantize(*fp4.quantize(bits(x)))
        back[torch.tensor(slots) < 0] = 0.0
        assert np.array_equal(y.float().cpu().numpy().astype(np.float64), back)
    assert int(flags) == 0
