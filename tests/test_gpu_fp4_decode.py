"""Decode attention over the 4-bit cache on the GPU against the formula in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import bits
from fp4_common import P_TWO_TERMS, Cache, check, random_rows
from oracle import fp4

pytestmark = pytest.mark.gpu


def _tables(seed, rows, width, pages):
    return torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[:rows * width].reshape(rows, width).to(torch.int32)


def _run(mas, dev, cache, q, tables, lens, scale, scale2=1.0, ws_bytes=128 << 20, **other):
    ws = torch.full((ws_bytes,), 255, dtype=torch.uint8, device=dev)
    return mas.attention.batch_decode_with_fp4_kv_cache(q.to(dev), cache.on(mas, dev), ws, tables.to(dev), lens.to(dev), 0, scale,
                                                        scale2, kv_layout=cache.layout, **other)


def _case(seed, hq, hk, dim, ps, layout, lens, extra=2):
    rows, width = len(lens), max(1, max(-(-n // ps) for n in lens)) + extra
    cache = Cache(seed, rows * width + 1, ps, hk, dim, layout)
    return cache, random_rows(seed + 7, rows, hq, dim), _tables(seed, rows, width, rows * width + 1), torch.tensor(lens, dtype=torch.int32)


CASES = [  # q heads, kv heads, head_dim, page size, layout, lengths
    (32, 8, 128, 16, "HND", [1, 15, 16, 17, 700]),
    (12, 1, 128, 256, "NHD", [255, 256, 257, 33]),
    (32, 8, 128, 16, "NHD", [31, 32, 0, 2300]),          # an empty row; a row of several splits
    (8, 8, 128, 32, "HND", [100, 47, 1]),                # one query head per kv head
    (16, 1, 128, 64, "NHD", [64, 65, 500]),              # a full tile of query heads
    (14, 2, 64, 16, "HND", [1, 16, 33, 1000]),           # 7 per kv head, head_dim 64
    (4, 4, 64, 128, "NHD", [129, 5]),
    (12, 3, 256, 16, "HND", [40, 300, 2]),
    (5, 1, 256, 64, "NHD", [70, 600]),
    (8, 2, 128, 16, "HND", [9000]),                      # one row in many short splits
]


@pytest.mark.parametrize("hq,hk,dim,ps,layout,lens", CASES)
def test_against_the_formula(mas, dev, hq, hk, dim, ps, layout, lens):
    cache, q, tables, n = _case(hq * 3 + dim, hq, hk, dim, ps, layout, lens)
    flags = torch.zeros(1, dtype=torch.int32, device=dev)
    out = _run(mas, dev, cache, q, tables, n, dim ** -0.5, error_flags=flags)
    check(out, fp4.decode_attention(bits(q), cache.k, cache.v, tables.numpy(), lens, dim ** -0.5), max(lens), P_TWO_TERMS)
    assert int(flags) == 0
    again = _run(mas, dev, cache, q, tables, n, dim ** -0.5)
    assert torch.equal(out, again)
    if 0 in lens:
        assert not out[lens.index(0)].any()


@pytest.mark.parametrize("rows", [40, 300])
def test_large_grids(mas, dev, rows):
    """Many rows of mixed lengths under a table that reaches further: 256-position splits and longer."""
    lens = [int(x) for x in torch.randint(0, 400, (rows,), generator=torch.Generator().manual_seed(rows))]
    lens[3] = 3000
    cache = Cache(rows, 64, 16, 2, 128, "HND")
    tables = torch.randint(0, 64, (rows, 512), generator=torch.Generator().manual_seed(1)).to(torch.int32)
    q = random_rows(2, rows, 8, 128)
    out = _run(mas, dev, cache, q, tables, torch.tensor(lens, dtype=torch.int32), 0.09)
    check(out, fp4.decode_attention(bits(q), cache.k, cache.v, tables.numpy(), lens, 0.09), 3000, P_TWO_TERMS)


def test_a_small_workspace_makes_longer_splits(mas, dev):
    lens = [5000, 40, 1025]
    cache, q, tables, n = _case(5, 8, 2, 128, 16, "HND", lens)
    need = mas.attention.decode_workspace_bytes(3, 8, 128, tables.shape[1], 16, 4)
    out = _run(mas, dev, cache, q, tables, n, 0.1, 0.5, ws_bytes=need)
    check(out, fp4.decode_attention(bits(q), cache.k, cache.v, tables.numpy(), lens, 0.1, 0.5), 5000, P_TWO_TERMS)
    with pytest.raises(mas._lib.KernelError):
        _run(mas, dev, cache, q, tables, n, 0.1, ws_bytes=64)


def test_what_lies_past_a_row_does_not_matter(mas, dev):
    """NaN blocks behind the rows' ends, in the same pages, and page ids outside the cache past them."""
    lens = [5, 16, 35, 300]
    cache, q, tables, n = _case(6, 8, 2, 128, 16, "HND", lens)
    for r, m in enumerate(lens):
        if m % 16:
            page = int(tables[r, m // 16])
            for t in cache.tensors[2:]:
                t[page, :, :, m % 16:] = 255
        tables[r, -(-m // 16):] = torch.tensor([-1, 1 << 30] * 20)[:tables.shape[1] - -(-m // 16)].to(torch.int32)
    flags = torch.zeros(1, dtype=torch.int32, device=dev)
    out = _run(mas, dev, cache, q, tables, n, 0.1, error_flags=flags)
    check(out, fp4.decode_attention(bits(q), cache.k, cache.v, np.clip(tables.numpy(), 0, cache.k.shape[0] - 1), lens, 0.1), 300,
          P_TWO_TERMS)
    assert int(flags) == 0


def test_bad_pages_are_skipped_and_lengths_clamped(mas, dev):
    """A page id outside the cache leaves its positions out; a length past the table is the table's reach; a negative
    one is an empty row."""
    lens = [100, 90, 33]
    cache, q, tables, n = _case(7, 8, 2, 128, 16, "HND", lens, extra=0)
    good = tables.clone()
    tables[0, 2], tables[2, 0] = -5, 1 << 20
    flags = torch.zeros(1, dtype=torch.int32, device=dev)
    out = _run(mas, dev, cache, q, tables, n, 0.1, error_flags=flags)
    assert int(flags) == 8
    for r, (lost, m) in {0: (2, 100), 2: (0, 33)}.items():
        pages = [p for i, p in enumerate(good[r, :-(-m // 16)].tolist()) if i != lost]
        want = fp4.decode_attention(bits(q[r:r + 1]), cache.k, cache.v, np.array([pages]), [m - 16], 0.1)
        check(out[r:r + 1], want, m, P_TWO_TERMS)
    tables[2, :3] = -1                                             # nothing left
    out = _run(mas, dev, cache, q, tables, n, 0.1)
    assert not out[2].any()
    flags.zero_()
    width = good.shape[1]
    out = _run(mas, dev, cache, q, good, torch.tensor([width * 16 + 1, -3, 33], dtype=torch.int32), 0.1, error_flags=flags)
    assert int(flags) == 2 and not out[1].any()
    want = fp4.decode_attention(bits(q), cache.k, cache.v, good.numpy(), [width * 16, 0, 33], 0.1)
    check(out, want, width * 16, P_TWO_TERMS)


@pytest.mark.parametrize("where", ["key", "value", "query"])
def test_a_nan_that_counts_shows(mas, dev, where):
    """A NaN block at an attended position makes the heads that read it NaN (a value block: its 32 elements), no other."""
    cache, q, tables, n = _case(8, 8, 2, 128, 16, "HND", [50, 60])
    page = int(tables[1, 2])
    if where == "query":
        q[1, 5, 17] = float("nan")
    else:
        cache.tensors[2 if where == "key" else 3][page, 1, 2, 4] = 255
    out = _run(mas, dev, cache, q, tables, n, 0.1).cpu()
    bad = torch.zeros_like(out, dtype=torch.bool)
    if where == "query":
        bad[1, 5] = True
    elif where == "key":
        bad[1, 4:] = True
    else:
        bad[1, 4:, 64:96] = True
    assert bool(out[bad].isnan().all()) and bool(out[~bad].isfinite().all())


@pytest.mark.parametrize("scale,size", [(0.0, 1.0), (-0.2, 1.0), (0.1, 2.0 ** 60), (0.1, 2.0 ** -60), (3.0, 4.0), (0.1, 2.0 ** -125)])
def test_scales_and_sizes(mas, dev, scale, size):
    """A zero, a negative and a large score scale; queries far from 1, the keys' product brought back by the scale."""
    cache, q, tables, n = _case(9, 8, 2, 128, 16, "HND", [70, 600])
    q = (q.float() * size).bfloat16()
    s = scale / size if size >= 2.0 ** -60 else scale
    out = _run(mas, dev, cache, q, tables, n, s)
    check(out, fp4.decode_attention(bits(q), cache.k, cache.v, tables.numpy(), [70, 600], s), 600, P_TWO_TERMS)


def test_queries_with_an_outlier(mas, dev):
    """One element far above the head's others: the others still count for what they are."""
    cache, q, tables, n = _case(10, 8, 2, 128, 16, "HND", [200, 33])
    q[:, :, 3] = 300.0
    q[:, ::2, 3] = 2.0 ** 14
    scale = 2.0 ** -10
    out = _run(mas, dev, cache, q, tables, n, scale)
    check(out, fp4.decode_attention(bits(q), cache.k, cache.v, tables.numpy(), [200, 33], scale), 200, P_TWO_TERMS)


@pytest.mark.parametrize("host", [True, False])
def test_fp8_output(mas, dev, host):
    lens, scale = [17, 900], 0.02
    cache, q, tables, n = _case(11, 32, 8, 128, 16, "HND", lens)
    quant = scale if host else torch.tensor(scale, device=dev)
    out = _run(mas, dev, cache, q, tables, n, 0.088, out_quant_scale=quant)
    plain = _run(mas, dev, cache, q, tables, n, 0.088)
    assert out.dtype == torch.float8_e4m3fn
    want = (plain.float().cpu() / torch.tensor(scale)).clamp(-448, 448).to(torch.float8_e4m3fn)
    assert torch.equal(out.cpu().view(torch.uint8), want.view(torch.uint8))


def test_strided_queries_and_outputs(mas, dev):
    """Queries as column views, an output with room around its rows, which stays as it was; another stream."""
    lens = [20, 1, 64]
    cache, q, tables, n = _case(12, 8, 2, 128, 16, "NHD", lens)
    wide = torch.zeros(3, 12 * 128, dtype=torch.bfloat16)
    wide[:, :8 * 128] = q.flatten(1)
    wide = wide.to(dev)
    room = torch.full((5, 8, 160), 3.0, dtype=torch.bfloat16, device=dev)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    c, t, m, ws = cache.on(mas, dev), tables.to(dev), n.to(dev), torch.empty(1 << 20, dtype=torch.uint8, device=dev)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        mas.attention.batch_decode_with_fp4_kv_cache(wide[:, :1024].unflatten(-1, (8, 128)), c, ws, t, m, 0, 0.1, 1.0,
                                                     out=room[1:4, :, 16:144], kv_layout="NHD")
    torch.cuda.current_stream().wait_stream(stream)
    check(room[1:4, :, 16:144], fp4.decode_attention(bits(q), cache.k, cache.v, tables.numpy(), lens, 0.1), 64, P_TWO_TERMS)
    assert bool((room[0] == 3).all()) and bool((room[4] == 3).all()) and bool((room[:, :, :16] == 3).all())
    assert bool((room[:, :, 144:] == 3).all())


def test_pages_far_into_a_large_cache(mas, dev):
    """Page offsets past 2^32 bytes (a 5 GiB codes tensor; the last pages hold the row)."""
    pages, ps, hk, dim = 5 << 20, 16, 1, 128
    few = Cache(13, 4, ps, hk, dim, "HND")
    c = mas.page.fp4_kv_cache(pages, ps, hk, dim, dev)
    for t, s in zip(c, few.tensors):
        t[-4:] = s.to(dev)
    q, lens = random_rows(14, 2, 4, dim), [60, 33]
    tables = torch.tensor([[3, 1, 0, 2], [2, 3, 1, 0]])
    out = mas.attention.batch_decode_with_fp4_kv_cache(
        q.to(dev), c, torch.empty(1 << 20, dtype=torch.uint8, device=dev), (tables + pages - 4).to(torch.int32).to(dev),
        torch.tensor(lens, dtype=torch.int32, device=dev), 0, 0.1, 1.0, kv_layout="HND")
    check(out, fp4.decode_attention(bits(q), few.k, few.v, tables.numpy(), lens, 0.1), 60, P_TWO_TERMS)


@pytest.mark.parametrize("dim,pages,layout", [(64, 5 << 20, "NHD"), (256, 2 << 20, "HND")])
def test_other_head_dims_in_a_large_cache(mas, dev, dim, pages, layout):
    few = Cache(15, 16, 16, 1, dim, layout)
    c = mas.page.fp4_kv_cache(pages, 16, 1, dim, dev, layout)
    for t, s in zip(c, few.tensors):
        t[-16:] = s.to(dev)
    q, lens = random_rows(16, 2, 5, dim), [250, 128]
    tables = torch.stack([torch.randperm(16, generator=torch.Generator().manual_seed(i)) for i in range(2)])
    out = mas.attention.batch_decode_with_fp4_kv_cache(
        q.to(dev), c, torch.empty(1 << 20, dtype=torch.uint8, device=dev), (tables + pages - 16).to(torch.int32).to(dev),
        torch.tensor(lens, dtype=torch.int32, device=dev), 0, 0.1, 1.0, kv_layout=layout)
    check(out, fp4.decode_attention(bits(q), few.k, few.v, tables.numpy(), lens, 0.1), 250, P_TWO_TERMS)


def test_as_many_rows_as_a_call_takes(mas, dev):
    """65535 rows of 8 kv heads under a table of 40 pages of 1024: more (row, head, 1024 positions) than a grid holds, so
    the splits get longer; rows of all lengths, some as long as the table."""
    rows, ps, width, dim = 65535, 1024, 40, 64
    cache = Cache(17, 2, ps, 8, dim, "HND")
    g = torch.Generator().manual_seed(18)
    lens = torch.randint(0, 50, (rows,), generator=g).to(torch.int32)
    tables = torch.randint(0, 2, (rows, width), generator=g).to(torch.int32)
    some = [0, 1, 777, 32768, 65533, 65534]
    for r, n in zip(some, (width * ps, 1, 5000, 20481, 0, 16 * ps + 1)):
        lens[r] = n
    q = random_rows(19, rows, 8, dim)
    out = _run(mas, dev, cache, q, tables, lens, 0.1, ws_bytes=6 << 30)
    some += list(range(2000, 2040))
    want = fp4.decode_attention(bits(q[some]), cache.k, cache.v, tables[some].numpy(), lens[some].tolist(), 0.1)
    check(out[some], want, width * ps, P_TWO_TERMS)
    assert bool(out.isfinite().all())


@pytest.mark.parametrize("rows,lens", [(64, [131072, 1, 16385, 300]), (1100, [40000, 20])])
def test_tables_far_wider_than_the_rows(mas, dev, rows, lens):
    """A launch holds fewer splits than the table has 1024 positions: a long row's get longer."""
    ps, width = 256, 512
    cache = Cache(20, 8, ps, 8, 64, "HND")
    g = torch.Generator().manual_seed(21)
    n = torch.randint(0, 300, (rows,), generator=g).to(torch.int32)
    n[:len(lens)] = torch.tensor(lens, dtype=torch.int32)
    tables = torch.randint(0, 8, (rows, width), generator=g).to(torch.int32)
    q = random_rows(22, rows, 8, 64)
    out = _run(mas, dev, cache, q, tables, n, 0.1, ws_bytes=1 << 30)
    some = list(range(40))
    want = fp4.decode_attention(bits(q[some]), cache.k, cache.v, tables[some].numpy(), n[some].tolist(), 0.1)
    check(out[some], want, max(lens), P_TWO_TERMS)


@pytest.mark.parametrize("where", ["key", "value", "query"])
def test_a_nan_shows_through_the_merge(mas, dev, where):
    """As above, in rows of several splits; a NaN query makes every split's scores NaN."""
    cache, q, tables, n = _case(23, 8, 2, 128, 16, "HND", [3000, 2500])
    page = int(tables[1, 60])
    if where == "query":
        q[1, 5, 17] = float("nan")
    else:
        cache.tensors[2 if where == "key" else 3][page, 1, 2, 4] = 255
    out = _run(mas, dev, cache, q, tables, n, 0.1).cpu()
    bad = torch.zeros_like(out, dtype=torch.bool)
    if where == "query":
        bad[1, 5] = True
    elif where == "key":
        bad[1, 4:] = True
    else:
        bad[1, 4:, 64:96] = True
    assert bool(out[bad].isnan().all()) and bool(out[~bad].isfinite().all())
