"""Refusals of the 4-bit cache's operators and of the step plan, on the CPU: the wrappers' (with fake GPU tensors,
nothing launches) and the C entry points' (nothing is dereferenced before they return)."""
from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

BF16, I32, I64, U8 = torch.bfloat16, torch.int32, torch.int64, torch.uint8
P = 4096          # any 16-byte aligned address


def _gpu(*shape, dtype=BF16):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def _cache(mas, pages=4, ps=16, heads=2, dim=64, layout="NHD", **other):
    shape = (pages, ps, heads, dim // 2) if layout == "NHD" else (pages, heads, ps, dim // 2)
    parts = {"k": _gpu(*shape, dtype=U8), "v": _gpu(*shape, dtype=U8),
             "k_scale": _gpu(pages, heads, dim // 32, ps, dtype=U8), "v_scale": _gpu(pages, heads, dim // 32, ps, dtype=U8)}
    return mas.page.Fp4KVCache(**{**parts, **other})


def test_a_zeroed_cache(mas):
    c = mas.page.fp4_kv_cache(3, 16, 2, 128, "cpu")
    assert c.k.shape == c.v.shape == (3, 2, 16, 64) and c.k_scale.shape == c.v_scale.shape == (3, 2, 4, 16)
    assert mas.fp4_kv_cache(3, 32, 2, 64, "cpu", "NHD").k.shape == (3, 32, 2, 32)
    assert not any(t.any() for t in c) and all(t.dtype == U8 for t in c)
    for bad in ((3, 8, 2, 128, "cpu"), (3, 24, 2, 128, "cpu"), (3, 16, 2, 48, "cpu"), (3, 16, 2, 128, "cpu", "HDN")):
        with pytest.raises(ValueError):
            mas.page.fp4_kv_cache(*bad)


def test_cpu_tensors_are_refused(mas):
    c = mas.page.fp4_kv_cache(3, 16, 2, 64, "cpu")
    x, i = torch.zeros(1, 2, 64, dtype=BF16), torch.zeros(1, dtype=I64)
    with pytest.raises(ValueError, match="GPU"):
        mas.store_kv_slots_fp4(x, x, c, i, "HND")
    with pytest.raises(ValueError, match="GPU"):
        mas.load_kv_slots_fp4(c, i, "HND")
    with pytest.raises(ValueError, match="GPU"):
        mas.plan_step(i.int(), i.int(), torch.zeros(1, 1, dtype=I32), i.int(), torch.zeros(2, dtype=I64), 16, 4)


@pytest.mark.parametrize("what,match", [
    ("layout", "kv_layout"), ("pair", "Fp4KVCache"), ("dtype", "uint8"), ("scale_shape", "k_scale and v_scale must be"),
    ("page", "power of two"), ("strides", "same shape and strides"), ("scale_strides", "last two dimensions"),
    ("dims", "4-D"), ("head_dim", "multiple of 32"), ("last", "contiguous in its last")])
def test_caches_that_are_none(mas, what, match):
    with FakeTensorMode():
        x, slots = _gpu(3, 2, 64), _gpu(3, dtype=I64)
        layout, c = "NHD", _cache(mas)
        if what == "layout":
            layout = "NDH"
        elif what == "pair":
            c = c[:2]
        elif what == "dtype":
            c = _cache(mas, k=_gpu(4, 16, 2, 32))
        elif what == "scale_shape":
            c = _cache(mas, k_scale=_gpu(4, 2, 16, 2, dtype=U8), v_scale=_gpu(4, 2, 16, 2, dtype=U8))
        elif what == "page":
            c = _cache(mas, ps=8)
        elif what == "strides":
            c = _cache(mas, v=_gpu(4, 2, 16, 32, dtype=U8).transpose(1, 2))
        elif what == "scale_strides":
            s = _gpu(4, 2, 4, 16, dtype=U8)[:, :, ::2]
            c = _cache(mas, k_scale=s, v_scale=s)
        elif what == "dims":
            c = _cache(mas, k=_gpu(4, 16, 64, dtype=U8))
        elif what == "head_dim":
            c = mas.page.Fp4KVCache(*[_gpu(4, 16, 2, 24, dtype=U8)] * 2, *[_gpu(4, 2, 1, 16, dtype=U8)] * 2)
        elif what == "last":
            c = _cache(mas, k=_gpu(4, 16, 32, 2, dtype=U8).transpose(2, 3))
        with pytest.raises((ValueError, TypeError), match=match):
            mas.store_kv_slots_fp4(x, x, c, slots, layout)


def test_rows_that_do_not_fit_the_cache(mas):
    with FakeTensorMode():
        c, slots, i = _cache(mas), _gpu(3, dtype=I64), _gpu(3, dtype=I32)
        good = _gpu(3, 2, 64)
        for key, value, s, error in ((_gpu(3, 3, 64), good, slots, ValueError), (good, _gpu(2, 2, 64), slots, ValueError),
                                     (good.float(), good, slots, TypeError), (good, good, i, TypeError),
                                     (good, good, _gpu(4, dtype=I64), ValueError), (good, _gpu(3, 120), slots, ValueError)):
            with pytest.raises(error):
                mas.store_kv_slots_fp4(key, value, c, s)
            with pytest.raises(error):
                mas.load_kv_slots_fp4(c, s, key=key, value=value)
        with pytest.raises(TypeError, match="positions must be torch.int32"):
            mas.append_paged_kv_cache_fp4(good, good, i, slots, c, i, i)
        with pytest.raises(ValueError, match="same length"):
            mas.append_paged_kv_cache_fp4(good, good, i, _gpu(2, dtype=I32), c, i, i)
        with pytest.raises(ValueError, match="error_flags"):
            mas.store_kv_slots_fp4(good, good, c, slots, error_flags=torch.zeros(1, dtype=I32, device="cpu"))


def test_attention_refusals(mas):
    att = mas.attention
    with FakeTensorMode():
        c, q, t, n = _cache(mas, dim=128), _gpu(3, 8, 128), _gpu(3, 4, dtype=I32), _gpu(3, dtype=I32)
        ws, cu = _gpu(1 << 20, dtype=U8), _gpu(4, dtype=I32)
        decode, context = att.batch_decode_with_fp4_kv_cache, att.batch_context_with_fp4_kv_cache
        bad = [
            (dict(q=_gpu(3, 8, 64)), ValueError, "query must be"), (dict(q=_gpu(3, 8, 128).float()), TypeError, "bfloat16"),
            (dict(q=_gpu(3, 7, 128)), ValueError, "multiple of num_kv_heads"), (dict(t=_gpu(2, 4, dtype=I32)), ValueError, "block_tables"),
            (dict(n=_gpu(2, dtype=I32)), ValueError, "seq_lens"), (dict(t=_gpu(3, 4, dtype=I64)), TypeError, "int32"),
            (dict(out=_gpu(3, 8, 64)), ValueError, "out must be"), (dict(s=torch.ones(1)), TypeError, "Python floats"),
            (dict(quant=-1.0), ValueError, "positive"), (dict(out_dtype=torch.float16), ValueError, "out_dtype"),
            (dict(c=c[:2]), ValueError, "Fp4KVCache"), (dict(ws=torch.empty(16, dtype=U8)), ValueError, "GPU"),
            (dict(c=_cache(mas, dim=96), q=_gpu(3, 8, 96)), ValueError, "head_dim"),
        ]
        for change, error, match in bad:
            a = dict(q=q, c=c, ws=ws, t=t, n=n, s=0.1, out=None, quant=None, out_dtype=None)
            a.update(change)
            common = dict(out=a["out"], out_dtype=a["out_dtype"], out_quant_scale=a["quant"])
            with pytest.raises(error, match=match):
                decode(a["q"], a["c"], a["ws"], a["t"], a["n"], 64, a["s"], 1.0, **common)
            with pytest.raises(error, match=match):
                context(a["q"], a["c"], a["ws"], a["t"], a["n"], 1, 64, a["s"], 1.0, 3, cu, **common)
        with pytest.raises(ValueError, match="at most 16"):
            decode(_gpu(3, 34, 128), c, ws, t, n, 64)
        with pytest.raises(ValueError, match="needs a workspace"):
            decode(q, c, None, t, n, 64)
        with pytest.raises(ValueError, match="expected batch_size"):
            context(q, c, ws, t, n, 1, 64, 0.1, 1.0, 2, cu)
        with pytest.raises(TypeError, match="cum_seq_lens_q"):
            context(q, c, ws, t, n, 1, 64, 0.1, 1.0, 3, _gpu(4, dtype=I64))
        with pytest.raises(ValueError, match="64 or 128"):
            context(_gpu(3, 8, 256), _cache(mas, dim=256), ws, t, n, 1, 64, 0.1, 1.0, 3, cu)


def test_plan_refusals(mas):
    # real tensors of the right kind are needed for the memory checks: the meta device has no addresses, so only the
    # checks before them run here
    with FakeTensorMode():
        new, tables, pages, rng = _gpu(3, dtype=I32), _gpu(3, 4, dtype=I32), _gpu(9, dtype=I32), _gpu(2, dtype=I64)
        out = mas.step.step_tables(3, 8, "cuda")
        good = dict(new=new, cached=_gpu(3, dtype=I32), tables=tables, pages=pages, rng=rng, ps=16, n=8, out=out)
        for change, error, match in (
                (dict(new=_gpu(3, dtype=I64)), TypeError, "new_lens"), (dict(cached=_gpu(2, dtype=I32)), ValueError, "cached_lens"),
                (dict(tables=_gpu(2, 4, dtype=I32)), ValueError, "block_tables"), (dict(tables=_gpu(4, 3, dtype=I32).t()), ValueError, "block_tables"),
                (dict(tables=_gpu(1, 4, dtype=I32).expand(3, 4)), ValueError, "overlap"),
                (dict(pages=_gpu(9, 1, dtype=I32)), ValueError, "free_pages"), (dict(rng=_gpu(3, dtype=I64)), ValueError, "free_range"),
                (dict(n=9), ValueError, "StepTables of 9"), (dict(n=-1), ValueError, "negative"), (dict(ps=0), ValueError, "page_size"),
                (dict(out=mas.step.step_tables(2, 8, "cuda")), ValueError, "cu_seqlens_q"),
                (dict(out=out._replace(slot_mapping=_gpu(8, dtype=I32))), TypeError, "slot_mapping")):
            a = {**good, **change}
            with pytest.raises(error, match=match):
                mas.plan_step(a["new"], a["cached"], a["tables"], a["pages"], a["rng"], a["ps"], a["n"], out=a["out"])


def test_shared_memory_is_found(mas):
    buf = torch.zeros(16, dtype=I32)
    f = mas.step._overlap
    assert f(buf[:8], buf[7:]) and f(buf, buf[3:4]) and not f(buf[:8], buf[8:]) and not f(buf[:0], buf)


def test_c_entry_points_refuse(mas):
    lib = mas.load_library()

    def store(ps=16, dim=64, k=P, stride=16 * 2 * 32, scale=P, key=P, rows=3, slots=P, pages=4):
        return lib.mas_store_kv_slots_fp4(k, P, stride, 64, 32, scale, P, 64, 32, pages, ps, key, 128, 64, P, 128, 64, slots,
                                          rows, 2, dim, None, None)
    assert store(rows=0) == 0
    for change, status in ((dict(ps=8), -2), (dict(ps=24), -2), (dict(ps=0), -1), (dict(dim=48), -2), (dict(k=None), -1),
                           (dict(k=P + 8), -3), (dict(stride=40), -3), (dict(scale=P + 2), -3), (dict(key=P + 4), -3),
                           (dict(key=None), -1), (dict(slots=None), -1), (dict(rows=-1), -1), (dict(pages=-1), -1),
                           (dict(rows=1 << 40), -2), (dict(rows=1 << 27), -2)):
        assert store(**change) == status, change

    def decode(ps=16, dim=128, hq=8, hk=2, out=P, ws=P, ws_bytes=1 << 20, blocks=4, pages=4, tables=P, entry=128, fp8=0, quant=0.0, batch=3):
        return lib.mas_paged_decode_attention_fp4(out, 1024, 128, P, 1024, 128, P, P, 4096, entry, 64, P, P, 128, 64, pages,
                                                  ps, tables, 4, blocks, P, batch, hq, hk, dim, 0.1, 1.0, fp8, None, quant, ws,
                                                  ws_bytes, None, None)
    for change, status in ((dict(ps=8), -2), (dict(dim=96), -2), (dict(hq=34), -2), (dict(hq=7), -1), (dict(hk=0), -1),
                           (dict(out=None), -1), (dict(out=P + 2), -3), (dict(ws=None), -1), (dict(ws=P + 4), -3),
                           (dict(pages=0), -1), (dict(tables=None), -1), (dict(entry=1 << 30), -2), (dict(fp8=1), -1),
                           (dict(blocks=1 << 40), -2), (dict(batch=65536), -2), (dict(batch=65535, hq=200, hk=200), -2)):
        assert decode(**change) == status, change
    assert decode(hq=0) == 0 and decode(ws_bytes=16) in (-1, -4)   # (-4: no GPU to ask for its size)

    def context(ps=16, dim=128, hq=8, scale=0.1, k=P, entry=128, pages=4, rows=3):
        return lib.mas_paged_context_attention_fp4(P, 1024, 128, P, 1024, 128, k, P, 4096, entry, 64, P, P, 128, 64, pages, ps,
                                                   P, 4, 4, P, P, rows, 5, 0, hq, 2, dim, scale, 1.0, 0, None, 0.0, None, 0,
                                                   None, None)
    assert context(rows=0) == 0
    for change, status in ((dict(ps=8), -2), (dict(dim=256), -2), (dict(hq=7), -1), (dict(scale=0.0), -1), (dict(k=None), -1),
                           (dict(entry=1 << 30), -2), (dict(entry=24), -3), (dict(pages=0), -1)):
        assert context(**change) == status, change

    def plan(pos=P, rows=3, seq=P + 64, rng=P, out=P + 128, ps=16, n=8, blocks=4, ring=9, pages=P):
        return lib.mas_plan_step(pos, P, P, P, seq, out, P, 4, blocks, P, P, rows, pages, ring, rng, ps, n, None, None)
    for change, status in ((dict(pos=None), -1), (dict(rows=-1), -1), (dict(seq=P), -1), (dict(out=P), -1), (dict(rng=None), -1),
                           (dict(ps=0), -1), (dict(n=-1), -1), (dict(blocks=1 << 40), -2), (dict(n=1 << 31), -2),
                           (dict(pages=None), -1), (dict(ring=1 << 31), -2)):
        assert plan(**change) == status, change


def test_ops_are_registered(mas):
    names = {n for n in dir(torch.ops.mas) if not n.startswith("_")}
    assert {"append_paged_kv_cache_fp4", "store_kv_slots_fp4", "load_kv_slots_fp4", "paged_decode_attention_fp4",
            "paged_context_attention_fp4", "plan_step"} <= names


def test_direct_calls_leave_other_forms_to_the_wrappers(mas):
    """On the CPU no form is taken, whatever the arguments are, and a refusal costs little."""
    import timeit
    mas.load_library()
    d = mas._lib.direct
    if d is None:
        pytest.skip("direct_calls.so not built")
    c = mas.page.fp4_kv_cache(3, 16, 2, 64, "cpu")
    x, i = torch.zeros(1, 2, 64, dtype=BF16), torch.zeros(1, dtype=I64)
    calls = [lambda: d.store_slots_fp4(x, x, c, i, "HND", None), lambda: d.load_slots_fp4(x, x, c, i, "HND", None),
             lambda: d.append_fp4(*[None] * 9), lambda: d.decode_attention_fp4(*[None] * 11),
             lambda: d.context_attention_fp4(*[None] * 14), lambda: d.plan_step(*[None] * 8),
             lambda: d.plan_step(i.int(), i.int(), i.int().view(1, 1), i.int(), i, 16, mas.step.step_tables(1, 1, "cpu"), None),
             lambda: d.plan_step(), lambda: d.append_fp4(x, x, i, i, c[:2], i, i, "HND", None)]
    for call in calls:
        assert call() is None
        assert min(timeit.repeat(call, number=200, repeat=10)) / 200 < 2e-5
