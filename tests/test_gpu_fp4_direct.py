"""The native calls of the 4-bit cache's operators and of the step plan against the wrappers' general way."""
from __future__ import annotations

import pytest
import torch

from fp4_common import Cache, random_rows

pytestmark = pytest.mark.gpu


def _both(mas, monkeypatch, call):
    """call's results by the native way, checked to have been taken, and by the general one."""
    mas.load_library()
    assert mas._lib.direct is not None
    taken = []

    class Watch:
        def __getattr__(self, name):
            fn = getattr(direct, name)

            def run(*args):
                st = fn(*args)
                taken.append((name, st))
                return st
            return run

    direct = mas._lib.direct
    with monkeypatch.context() as m:
        m.setattr(mas._lib, "direct", Watch())
        a = [t.clone() for t in call()]
        m.setattr(mas._lib, "direct", None)
        b = [t.clone() for t in call()]
    assert taken and all(st == 0 for _, st in taken), taken
    for x, y in zip(a, b):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("hk", [1, 2])
def test_store_load_append(mas, dev, monkeypatch, layout, hk):
    qkv = random_rows(1, 9, 2 * hk, 128).flatten(1).to(dev)
    key, value = qkv[:, :hk * 128], qkv[:, hk * 128:].unflatten(-1, (hk, 128))
    slots = torch.tensor([5, 33, 7, -1, 0, 60, 61, 16, 31], device=dev)
    tables = torch.tensor([[2, 0, 1, 3]], dtype=torch.int32, device=dev)
    indptr = torch.tensor([0, 4], dtype=torch.int32, device=dev)
    batch, pos = torch.zeros(9, dtype=torch.int32, device=dev), torch.arange(30, 39, dtype=torch.int32, device=dev)
    for flags in (None, torch.zeros(1, dtype=torch.int32, device=dev)):
        def stores():
            c = mas.page.fp4_kv_cache(4, 16, hk, 128, dev, layout)
            mas.store_kv_slots_fp4(key, value, c, slots, layout, error_flags=flags)
            mas.append_paged_kv_cache_fp4(key, value, batch, pos, c, tables.flatten(), indptr, None, layout, error_flags=flags)
            return [*c, *mas.load_kv_slots_fp4(c, slots, layout, error_flags=flags)]
        _both(mas, monkeypatch, stores)


@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("quant", [None, 0.05, "device"])
def test_attention(mas, dev, monkeypatch, layout, quant):
    cache = Cache(2, 24, 16, 2, 128, layout).on(mas, dev)
    quant = torch.tensor(0.05, device=dev) if quant == "device" else quant
    q = random_rows(3, 40, 8, 128).to(dev)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    tables, ws = torch.arange(24, device=dev).to(torch.int32).view(2, 12), torch.empty(1 << 20, dtype=torch.uint8, device=dev)
    _both(mas, monkeypatch, lambda: [mas.attention.batch_decode_with_fp4_kv_cache(
        q[:2], cache, ws, tables, i32(180, 33), 0, 0.1, 1.0, kv_layout=layout, out_quant_scale=quant)])
    for w in (ws, None):
        _both(mas, monkeypatch, lambda: [mas.attention.batch_context_with_fp4_kv_cache(
            q, cache, w, tables, i32(180, 40), 30, 0, 0.1, 1.0, 2, i32(0, 30, 40), kv_layout=layout, out_quant_scale=quant)])


def test_plan(mas, dev, monkeypatch):
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    new, cached, rng = i32(3, 1, 20), i32(15, 16, 0), torch.tensor([7, 12], device=dev)
    for out in (None, mas.step.step_tables(3, 30, dev)):
        def plan():
            tables = torch.arange(12, device=dev).to(torch.int32).view(3, 4)
            return [*mas.plan_step(new, cached, tables, i32(50, 51, 52, 53, 54), rng, 16, 30, out=out), tables]
        _both(mas, monkeypatch, plan)


def test_what_the_native_calls_leave_is_refused(mas, dev):
    """Forms that do not check out come back to the wrappers, which raise."""
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    c = mas.page.fp4_kv_cache(4, 16, 2, 64, dev, "NHD")
    x, slots = random_rows(4, 3, 2, 64).to(dev), torch.arange(3, device=dev)
    mas.store_kv_slots_fp4(x, x, c, slots)
    for bad in ((x.float(), x, c, slots), (x, x[:2], c, slots), (x, x, c[:2], slots), (x, x, c, slots.int())):
        with pytest.raises((ValueError, TypeError)):
            mas.store_kv_slots_fp4(*bad)
    with pytest.raises(ValueError, match="shares memory"):
        t = mas.step.step_tables(2, 2, dev)
        mas.plan_step(i32(1, 1), t.seq_lens, torch.zeros(2, 2, dtype=torch.int32, device=dev), i32(1, 2),
                      torch.tensor([0, 2], device=dev), 16, 2, out=t)
