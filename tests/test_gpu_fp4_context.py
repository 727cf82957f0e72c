"""Context attention over the 4-bit cache on the GPU against the formula in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import bits
from fp4_common import P_BF16, Cache, check, random_rows, tolerance
from oracle import fp4

pytestmark = pytest.mark.gpu


def _case(seed, hq, hk, dim, ps, layout, rows, extra=1, pages=None):
    """rows: (new tokens, positions) of each."""
    width = max(1, max(-(-n // ps) for _, n in rows)) + extra
    pages = pages or len(rows) * width + 1
    g = torch.Generator().manual_seed(seed)
    tables = (torch.randperm(pages, generator=g)[:len(rows) * width] if pages > len(rows) * width
              else torch.randint(0, pages, (len(rows) * width,), generator=g)).reshape(len(rows), width).to(torch.int32)
    cu = [0]
    for n, _ in rows:
        cu.append(cu[-1] + n)
    return (Cache(seed, pages, ps, hk, dim, layout), random_rows(seed + 7, cu[-1], hq, dim), tables,
            [n for _, n in rows], cu)


def _run(mas, dev, cache, q, tables, lens, cu, scale, scale2=1.0, ws_bytes=64 << 20, max_q=None, max_kv=0, **other):
    ws = torch.full((ws_bytes,), 255, dtype=torch.uint8, device=dev) if ws_bytes else None
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    return mas.attention.batch_context_with_fp4_kv_cache(
        q.to(dev), cache.on(mas, dev), ws, tables.to(dev), i32(lens), max_q or max(b - a for a, b in zip(cu, cu[1:])), max_kv, scale,
        scale2, len(lens), i32(cu), kv_layout=cache.layout, **other)


CASES = [  # q heads, kv heads, head_dim, page size, layout, (new tokens, positions) of each row
    (4, 1, 128, 16, "HND", [(1, 1), (2, 2), (33, 33), (64, 64)]),
    (4, 1, 128, 16, "NHD", [(65, 65), (130, 200), (7, 129)]),
    (12, 1, 128, 64, "HND", [(40, 40), (3, 90), (70, 71)]),      # eight wavefronts
    (32, 8, 128, 256, "NHD", [(20, 300), (1, 257)]),
    (8, 8, 128, 16, "HND", [(129, 150), (16, 16)]),              # one head per kv head: 128-token tiles
    (6, 3, 128, 32, "NHD", [(66, 100), (1, 31)]),                # two
    (7, 1, 128, 16, "HND", [(35, 70)]),                          # seven: a head group with a gap
    (4, 1, 64, 16, "HND", [(1, 1), (65, 65), (33, 150)]),
    (16, 1, 64, 128, "NHD", [(50, 60), (10, 200)]),              # eight wavefronts, half of them staging
    (3, 3, 64, 16, "NHD", [(130, 260)]),
    (4, 1, 128, 16, "HND", [(16, 1500)]),                        # split key ranges
    (12, 1, 128, 16, "NHD", [(30, 2000), (30, 700)]),
    (8, 2, 64, 32, "HND", [(5, 1100)]),
]


@pytest.mark.parametrize("hq,hk,dim,ps,layout,rows", CASES)
@pytest.mark.parametrize("ws_bytes", [64 << 20, 0])
def test_against_the_formula(mas, dev, hq, hk, dim, ps, layout, rows, ws_bytes):
    cache, q, tables, lens, cu = _case(hq * 5 + dim, hq, hk, dim, ps, layout, rows)
    flags = torch.zeros(1, dtype=torch.int32, device=dev)
    out = _run(mas, dev, cache, q, tables, lens, cu, dim ** -0.5, ws_bytes=ws_bytes, error_flags=flags)
    check(out, fp4.context_attention(bits(q), cache.k, cache.v, tables.numpy(), lens, cu, dim ** -0.5), max(lens), P_BF16)
    assert int(flags) == 0
    assert torch.equal(out, _run(mas, dev, cache, q, tables, lens, cu, dim ** -0.5, ws_bytes=ws_bytes))


@pytest.mark.parametrize("prompts", [[(100, 1100)], [(20, 40), (70, 900), (1, 64)], [(120, 120)]])
@pytest.mark.parametrize("hq,hk,graph_rows", [(32, 8, 17), (12, 1, 17), (8, 2, 70)])
def test_padded_rows_of_a_captured_graph(mas, dev, prompts, hq, hk, graph_rows):
    """The prompts first, then a padding row on a sink page and empty rows: planned on the device, by each workgroup
    (up to 64 rows) or by a planner launch."""
    tokens = sum(n for n, _ in prompts)
    total = -(-tokens // 64) * 64
    pad = total - tokens
    rows = prompts + ([(pad, pad)] if pad else [(0, 1)]) + [(0, 1)] * (graph_rows - len(prompts) - 1)
    cache, q, tables, lens, cu = _case(hq + len(prompts), hq, hk, 128, 16, "HND", rows, pages=80)
    wide = torch.full((graph_rows, 512), 79, dtype=torch.int32)
    wide[:len(prompts), :tables.shape[1]] = tables[:len(prompts)]
    out = _run(mas, dev, cache, q, wide, lens, cu, 0.1, max_q=total, max_kv=8192)
    check(out, fp4.context_attention(bits(q), cache.k, cache.v, wide.numpy(), lens, cu, 0.1), max(lens), P_BF16)


@pytest.mark.parametrize("layout", ["HND", "NHD"])
def test_what_lies_past_a_row_does_not_matter(mas, dev, layout):
    rows = [(5, 21), (40, 40), (17, 99)]
    cache, q, tables, lens, cu = _case(21, 4, 1, 128, 16, layout, rows)
    for r, m in enumerate(lens):
        page = int(tables[r, m // 16])
        for t in cache.tensors[2:]:
            t[page, :, :, m % 16:] = 255
        tables[r, m // 16 + 1:] = -1
    flags = torch.zeros(1, dtype=torch.int32, device=dev)
    out = _run(mas, dev, cache, q, tables, lens, cu, 0.1, error_flags=flags)
    want = fp4.context_attention(bits(q), cache.k, cache.v, np.maximum(tables.numpy(), 0), lens, cu, 0.1)
    check(out, want, 99, P_BF16)
    assert int(flags) == 0


@pytest.mark.parametrize("dim", [64, 128])
def test_bad_pages_and_lengths(mas, dev, dim):
    """A page outside the cache leaves its positions out (they count as zeros' weight nowhere); tokens before position
    0 get zeros; both are reported."""
    rows = [(4, 60), (6, 6)]
    cache, q, tables, lens, cu = _case(22, 4, 1, dim, 16, "HND", rows)
    flags = torch.zeros(1, dtype=torch.int32, device=dev)
    out = _run(mas, dev, cache, q, tables, [60, 3], cu, 0.1, error_flags=flags)
    assert int(flags) == 2 and not out[4:7].any()
    want = fp4.context_attention(bits(q[7:]), cache.k, cache.v, tables.numpy()[1:], [3], [0, 3], 0.1)
    check(out[7:], want, 3, P_BF16)
    flags.zero_()
    out = _run(mas, dev, cache, q, tables, [60, tables.shape[1] * 16 + 1], cu, 0.1, error_flags=flags)
    assert int(flags) == 2
    check(out[:4], fp4.context_attention(bits(q[:4]), cache.k, cache.v, tables.numpy()[:1], [60], [0, 4], 0.1), 60, P_BF16)


def test_a_bad_page_is_reported_and_its_rows_read_nothing(mas, dev):
    """As over the bf16 cache: positions on a page id outside the cache enter as zero keys and values."""
    rows = [(4, 60)]
    cache, q, tables, lens, cu = _case(23, 4, 1, 128, 16, "HND", rows)
    lost = int(tables[0, 1])
    tables[0, 1] = 1 << 30
    flags = torch.zeros(1, dtype=torch.int32, device=dev)
    out = _run(mas, dev, cache, q, tables, lens, cu, 0.1, error_flags=flags)
    assert int(flags) == 8
    cache.k[lost], cache.v[lost] = 0.0, 0.0
    tables[0, 1] = lost
    check(out, fp4.context_attention(bits(q), cache.k, cache.v, tables.numpy(), lens, cu, 0.1), 60, P_BF16)


def test_a_nan_that_counts_shows(mas, dev):
    """A NaN key block at position 40 makes the tokens that reach it NaN, and only those."""
    rows = [(64, 64)]
    cache, q, tables, lens, cu = _case(24, 4, 1, 128, 16, "HND", rows)
    cache.tensors[2][int(tables[0, 2]), 0, 1, 8] = 255
    out = _run(mas, dev, cache, q, tables, lens, cu, 0.1).cpu()
    assert bool(out[:40].isfinite().all()) and bool(out[40:].isnan().all())


@pytest.mark.parametrize("hq,hk,dim,ws_bytes", [(4, 1, 128, 0), (8, 1, 128, 0), (4, 1, 64, 0), (12, 1, 64, 0), (4, 1, 128, 8 << 20)])
def test_values_that_are_no_numbers_reach_only_the_tokens_after_them(mas, dev, hq, hk, dim, ws_bytes):
    """NaN value blocks, and values past bf16's largest number, at positions inside the prompt: the tokens before them,
    whose weight there is none, are as if they were not there; the tokens from them on are NaN in those elements."""
    rows = [(150, 900 if ws_bytes else 300), (40, 40)]
    cache, q, tables, lens, cu = _case(27, hq, hk, dim, 16, "HND", rows)
    first, large = {}, {}                            # (row, element): its first position that is no number

    def spoil(r, p, element, power, code):
        page, slot = int(tables[r, p // 16]), p % 16
        cache.tensors[3][page, 0, element // 32, slot] = power
        row = cache.tensors[1][page, 0, slot]
        row[16 * (element // 32):16 * (element // 32) + 16] = 0x11     # 1/2: finite at any power below 255
        row[element // 2] = code | code << 4
        cols = range(element // 32 * 32, element // 32 * 32 + 32) if power == 255 else (element & ~1, element | 1)
        for c in cols:
            first[r, c] = min(p, first.get((r, c), p))
        large[r, p, element // 32] = power

    n = lens[0]
    spoil(0, n - 150 + 33, 5, 255, 0)
    spoil(0, n - 150 + 97, 7, 255, 0)
    spoil(0, n - 2, 40, 254, 4)                      # 2 * 2^127
    spoil(0, n - 70, 62, 253, 14)                    # -4 * 2^126
    spoil(1, 39, 33, 254, 7)
    out = _run(mas, dev, cache, q, tables, lens, cu, 2.0 ** -10, ws_bytes=ws_bytes).float().cpu().numpy()
    values = cache.v.copy()
    spoiled = np.zeros_like(out, dtype=bool)
    for (r, p, block), power in large.items():
        page, slot = int(tables[r, p // 16]), p % 16
        values[page, slot, 0, 32 * block:32 * block + 32] = 0.0
        t = int(cu[r]) + p - (lens[r] - rows[r][0])
        spoiled[t:int(cu[r + 1]), :, 32 * block:32 * block + 32] = True
    want = fp4.context_attention(bits(q), cache.k, values, tables.numpy(), lens, cu, 2.0 ** -10)
    ok = ~spoiled
    allowed = tolerance(*want, max(lens), P_BF16)
    assert np.isfinite(out[ok]).all() and (np.abs(out - want[0])[ok] <= allowed[ok]).all()
    no_number = np.zeros_like(spoiled)
    for (r, c), p in first.items():
        no_number[int(cu[r]) + p - (lens[r] - rows[r][0]):int(cu[r + 1]), :, c] = True
    assert np.isnan(out[no_number]).all() and np.isfinite(out[~no_number]).all()


@pytest.mark.parametrize("scale,size", [(0.1, 2.0 ** 50), (0.1, 2.0 ** -50), (3.0, 4.0)])
def test_scales_and_sizes(mas, dev, scale, size):
    cache, q, tables, lens, cu = _case(25, 8, 2, 128, 16, "HND", [(50, 170), (3, 3)])
    q = (q.float() * size).bfloat16()
    out = _run(mas, dev, cache, q, tables, lens, cu, scale / size, 2.0)
    check(out, fp4.context_attention(bits(q), cache.k, cache.v, tables.numpy(), lens, cu, scale / size, 2.0), 170, P_BF16)


def test_fp8_output_and_rows_behind_the_last(mas, dev):
    """The fp8 form is the quantize of the bf16 one; tokens past the last row's, and columns around the heads, stay."""
    cache, q, tables, lens, cu = _case(26, 8, 2, 128, 16, "NHD", [(50, 170), (3, 3)])
    room = torch.full((60, 8, 160), 3.0, dtype=torch.bfloat16, device=dev)
    wide = torch.zeros(60, 8, 128, dtype=torch.bfloat16)
    wide[:53] = q
    out = _run(mas, dev, cache, wide, tables, lens, cu, 0.1, out=room[:, :, 16:144])
    check(out[:53], fp4.context_attention(bits(q), cache.k, cache.v, tables.numpy(), lens, cu, 0.1), 170, P_BF16)
    assert bool((room[53:] == 3).all()) and bool((room[:, :, :16] == 3).all()) and bool((room[:, :, 144:] == 3).all())
    quant = _run(mas, dev, cache, q, tables, lens, cu, 0.1, out_quant_scale=0.03)
    want = (out[:53].float().cpu() / torch.tensor(0.03)).clamp(-448, 448).to(torch.float8_e4m3fn)
    assert torch.equal(quant.cpu().view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("dim,pages,layout", [(128, 5 << 20, "HND"), (64, 9 << 20, "NHD")])
def test_prompts_far_into_a_large_cache(mas, dev, dim, pages, layout):
    """Byte offsets past 2^32 in the codes: rows stored by slots into the last pages, read back, and attended."""
    ps, n = 16, 150
    kv = mas.page.fp4_kv_cache(pages, ps, 1, dim, dev, layout)
    k, v, q = random_rows(31, n, 1, dim), random_rows(32, n, 1, dim), random_rows(33, 40, 4, dim)
    order = torch.randperm(12, generator=torch.Generator().manual_seed(4))[:-(-n // ps)]
    table = (pages - 12 + order)[None].to(torch.int32)
    p = torch.arange(n)
    slots = table[0, p // ps].long() * ps + p % ps
    mas.page.store_kv_slots_fp4(k.to(dev), v.to(dev), kv, slots.to(dev), layout)
    values = [fp4.dequantize(*fp4.quantize(bits(x))) for x in (k, v)]
    for got, want in zip(mas.page.load_kv_slots_fp4(kv, slots.to(dev), layout), values):
        assert np.array_equal(got.float().cpu().numpy(), want)
    held = []
    for x in values:
        few = np.zeros((12, ps, 1, dim))
        few[order[p // ps].numpy(), (p % ps).numpy()] = x
        held.append(few)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    out = mas.attention.batch_context_with_fp4_kv_cache(q.to(dev), kv, None, table.to(dev), i32(n), 40, 0, 0.1, 1.0, 1, i32(0, 40),
                                                        kv_layout=layout)
    check(out, fp4.context_attention(bits(q), *held, order[None].numpy(), [n], [0, 40], 0.1), n, P_BF16)


def test_calls_without_rows(mas, dev):
    kv = mas.page.fp4_kv_cache(4, 16, 2, 128, dev, "HND")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    none = torch.empty(0, 8, 128, dtype=torch.bfloat16, device=dev)
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=dev)
    out = mas.attention.batch_context_with_fp4_kv_cache(none, kv, ws, torch.zeros(0, 3, dtype=torch.int32, device=dev), i32(), 1, 0,
                                                        0.1, 1.0, 0, i32(0), kv_layout="HND")
    assert out.shape == none.shape
    out = mas.attention.batch_decode_with_fp4_kv_cache(none, kv, ws, torch.zeros(0, 3, dtype=torch.int32, device=dev), i32(), 0, 0.1,
                                                       1.0, kv_layout="HND")
    assert out.shape == none.shape
    # rows, but tables of no width: nothing to attend
    q, flags = random_rows(34, 3, 8, 128).to(dev), torch.zeros(1, dtype=torch.int32, device=dev)
    out = mas.attention.batch_decode_with_fp4_kv_cache(q, kv, ws, torch.zeros(3, 0, dtype=torch.int32, device=dev), i32(0, 0, 0), 0,
                                                       0.1, 1.0, out=torch.ones_like(q), kv_layout="HND", error_flags=flags)
    assert not out.any() and int(flags) == 0


@pytest.mark.parametrize("rows,ws_bytes", [([(8, 3000)], 64 << 20), ([(8, 3000)], 0), ([(8, 3000)] + [(3, 40)] * 16, 64 << 20)])
def test_a_nan_query_shows(mas, dev, rows, ws_bytes):
    """In a call that splits its key range, one that does not, and one laid out on the device."""
    cache, q, tables, lens, cu = _case(35, 8, 2, 128, 16, "HND", rows)
    q[3, 5, 17] = float("nan")
    out = _run(mas, dev, cache, q, tables, lens, cu, 0.1, ws_bytes=ws_bytes, max_q=512 if len(rows) > 1 else None).cpu()
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[3, 5] = True
    assert bool(out[bad].isnan().all()) and bool(out[~bad].isfinite().all())


def test_more_tokens_than_max_q_len(mas, dev):
    """A row of more tokens than the call says, its key range split: reported, and the tokens past max_q_len stay."""
    cache, q, tables, lens, cu = _case(36, 8, 2, 128, 16, "HND", [(8, 3000), (5, 2000)])
    flags = torch.zeros(1, dtype=torch.int32, device=dev)
    out = torch.full(q.shape, 3.0, dtype=torch.bfloat16, device=dev)
    _run(mas, dev, cache, q, tables, lens, cu, 0.1, max_q=5, out=out, error_flags=flags)
    assert int(flags) == 2 and bool((out[5:8] == 3).all())
    kept = list(range(5)) + list(range(8, 13))
    want = fp4.context_attention(bits(q), cache.k, cache.v, tables.numpy(), lens, cu, 0.1)
    check(out[kept], (want[0][kept], want[1][kept], want[2]), 3000, P_BF16)
