"""plan_step on the GPU against the oracle's loop, and a run of steps through the 4-bit cache."""
from __future__ import annotations

import random

import numpy as np
import pytest
import torch

from conftest import bits
from fp4_common import P_BF16, P_TWO_TERMS, check, random_rows
from oracle import fp4

pytestmark = pytest.mark.gpu


def _plan(mas, dev, new, cached, tables, pages, rng, ps, tokens, out=None):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    flags = torch.zeros(1, dtype=torch.int32, device=dev)
    t = tables.to(dev)
    got = mas.plan_step(i32(new), i32(cached), t, i32(pages), torch.tensor(rng, device=dev), ps, tokens, out=out, error_flags=flags)
    return got, t, int(flags)


def _same(got, tables, flags, want):
    for name in ("positions", "batch_indices", "slot_mapping", "cu_seqlens_q", "seq_lens", "free_range"):
        assert getattr(got, name).tolist() == want[name], name
    assert np.array_equal(tables.cpu().numpy(), want["tables"]) and flags == want["bits"]


@pytest.mark.parametrize("seed", range(24))
def test_against_the_loop(mas, dev, seed):
    """Random steps: decode rows, prompts, idle rows, any page size, full and scarce pools and token counts, bad lengths."""
    r = random.Random(seed)
    rows, ps = r.choice((1, 2, 7, 64, 255, 256, 257, 700)), r.choice((1, 3, 16, 16, 64, 256))
    width = r.randint(1, 40)
    cached = [r.randint(0, width * ps) for _ in range(rows)]
    new = [min(r.choice((0, 1, 1, 1, r.randint(0, 300))), width * ps - c) for c in cached]
    if seed % 3 == 2:
        for _ in range(3):
            i = r.randrange(rows)
            cached[i], new[i] = r.choice(((-1, 3), (5, -2), (width * ps, 1), (2 ** 31 - 1, 2 ** 31 - 1), (0, 2 ** 31 - 1)))
    ring = r.randint(1, 4000)
    head = r.randint(0, 10 ** 12)
    free = r.choice((ring, ring, r.randint(0, ring), 0))
    total = sum(max(0, n) for n in new if n < 2 ** 30)
    tokens = r.choice((total, total + 63, max(0, total - r.randint(1, 40)), 0)) if seed % 4 else total
    pages = [r.randint(0, 10 ** 6) for _ in range(ring)]
    tables = torch.randint(0, 10 ** 6, (rows, width), generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    if seed % 5 == 4:
        tables[tables % 7 == 0] = -1
    want = fp4.plan_step(new, cached, tables.numpy(), pages, (head, head + free), ps, tokens)
    _same(*_plan(mas, dev, new, cached, tables, pages, (head, head + free), ps, tokens), want)


def test_edges(mas, dev):
    t = torch.zeros(0, 3, dtype=torch.int32)
    got, _, flags = _plan(mas, dev, [], [], t, [4], (0, 1), 16, 5)                 # no rows: padding
    assert got.slot_mapping.tolist() == [-1] * 5 and got.cu_seqlens_q.tolist() == [0] and flags == 0
    t = torch.zeros(2, 2, dtype=torch.int32)
    for rng, free in (((0, 0), []), ((5, 3), [1, 2]), ((-4, 3), [1, 2])):            # no pages, a range that is none
        got, _, flags = _plan(mas, dev, [1, 1], [0, 16], t, free, rng, 16, 4)
        assert flags == 64 and got.seq_lens.tolist() == [0, 16] and got.free_range.tolist() == list(rng)
    got, _, flags = _plan(mas, dev, [16, 16], [0, 0], t, [8, 9], (1, 3), 16, 32)     # the ring wraps
    assert got.slot_mapping.tolist() == list(range(144, 160)) + list(range(128, 144)) and flags == 0


def test_a_long_prompt_and_many_rows(mas, dev):
    new, cached = [20000] + [1] * 3000 + [777], [5] + [17] * 3000 + [0]
    tables = torch.arange(3002 * 1251).reshape(3002, 1251).to(torch.int32)
    pages = list(range(10 ** 7, 10 ** 7 + 6000))
    want = fp4.plan_step(new, cached, tables.numpy(), pages, (123456, 123456 + 6000), 16, 23800)
    _same(*_plan(mas, dev, new, cached, tables, pages, (123456, 123456 + 6000), 16, 23800), want)


def test_outputs_need_memory_of_their_own(mas, dev):
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    new, cached, tables, rng = i(1, 1), i(0, 0), torch.zeros(2, 2, dtype=torch.int32, device=dev), torch.tensor([0, 4], device=dev)
    out = mas.step.step_tables(2, 4, dev)
    for bad in (out._replace(seq_lens=cached), out._replace(free_range=rng), out._replace(seq_lens=new)):
        with pytest.raises(ValueError, match="shares memory"):
            mas.plan_step(new, cached, tables, i(5, 6, 7, 8), rng, 16, 4, out=bad)


class _Conversation:
    """Rows of one layer served by the operators, and what they hold on the host: the values their 4-bit cache stands
    for."""

    def __init__(self, mas, dev, rows, hq, hk, dim, ps, width, pages):
        self.mas, self.dev, self.shape, self.ps = mas, dev, (hq, hk, dim), ps
        self.cache = mas.page.fp4_kv_cache(pages, ps, hk, dim, dev)
        self.tables = torch.full((rows, width), -1, dtype=torch.int32, device=dev)
        self.ring = torch.randperm(pages, generator=torch.Generator().manual_seed(3)).to(torch.int32).to(dev)
        self.flags = torch.zeros(1, dtype=torch.int32, device=dev)
        self.workspace = torch.empty(32 << 20, dtype=torch.uint8, device=dev)
        self.held = [[np.zeros((0, hk, dim)), np.zeros((0, hk, dim))] for _ in range(rows)]

    def store(self, t, key, value):
        self.mas.store_kv_slots_fp4(key, value, self.cache, t.slot_mapping, "HND", error_flags=self.flags)

    def decode(self, t, q, out):
        return self.mas.attention.batch_decode_with_fp4_kv_cache(q, self.cache, self.workspace, self.tables, t.seq_lens, 0, 0.09,
                                                                 1.0, out=out, kv_layout="HND", error_flags=self.flags)

    def context(self, t, q, max_q):
        return self.mas.attention.batch_context_with_fp4_kv_cache(
            q, self.cache, self.workspace, self.tables, t.seq_lens, max_q, 0, 0.09, 1.0, self.tables.shape[0], t.cu_seqlens_q,
            kv_layout="HND", error_flags=self.flags)

    def hold(self, new, key, value):
        at = 0
        for r, n in enumerate(new):
            for i, x in enumerate((key, value)):
                y = fp4.dequantize(*fp4.quantize(bits(x[at:at + n])))
                self.held[r][i] = np.concatenate((self.held[r][i], y))
            at += n

    def exact(self, new, q):
        """What attention over the held rows gives each new token."""
        hq, hk, dim = self.shape
        outs = []
        cu = 0
        for r, n in enumerate(new):
            k, v = (np.concatenate((x, np.zeros(((-len(x)) % self.ps, hk, dim)))).reshape(-1, self.ps, hk, dim) for x in self.held[r])
            outs.append(fp4.context_attention(bits(q[cu:cu + n]), k, v, [np.arange(len(k))], [len(self.held[r][0])], [0, n], 0.09))
            cu += n
        return np.concatenate([o[0] for o in outs]), np.concatenate([o[1] for o in outs]), max(o[2] for o in outs)


@pytest.mark.parametrize("hq,hk,dim,ps", [(8, 2, 128, 16), (12, 1, 64, 32)])
def test_a_conversation(mas, dev, hq, hk, dim, ps):
    """Plan, store, attend: prompts of odd lengths in two chunks, then decode steps captured in one graph and replayed, the
    graph's own outputs feeding its next replay; every step's outputs against the formula over what was stored."""
    rows = 5
    c = _Conversation(mas, dev, rows, hq, hk, dim, ps, 20, 80)
    lens, rng = torch.zeros(rows, dtype=torch.int32, device=dev), torch.tensor([0, 80], device=dev)
    for step, new in enumerate(([33, 1, 70, 16, 5], [20, 90, 0, 1, 17])):
        n = sum(new)
        key, value, q = (random_rows(50 + 10 * step + i, n, h, dim) for i, h in enumerate((hk, hk, hq)))
        t = mas.plan_step(torch.tensor(new, dtype=torch.int32, device=dev), lens, c.tables, c.ring, rng, ps, n, error_flags=c.flags)
        c.store(t, key.to(dev), value.to(dev))
        out = c.context(t, q.to(dev), max(new))
        c.hold(new, key, value)
        check(out, c.exact(new, q), max(len(h[0]) for h in c.held), P_BF16)
        lens, rng = t.seq_lens, t.free_range
    # decode steps, in a graph
    one = torch.ones(rows, dtype=torch.int32, device=dev)
    t = mas.step.step_tables(rows, rows, dev)
    key, value = (torch.empty(rows, hk, dim, dtype=torch.bfloat16, device=dev) for _ in range(2))
    q, out = torch.empty(rows, hq, dim, dtype=torch.bfloat16, device=dev), torch.empty(rows, hq, dim, dtype=torch.bfloat16, device=dev)
    lens, rng = lens.clone(), rng.clone()
    saved = [x.clone() for x in (lens, rng, c.tables)]

    def step():
        mas.plan_step(one, lens, c.tables, c.ring, rng, ps, rows, out=t, error_flags=c.flags)
        c.store(t, key, value)
        c.decode(t, q, out)
        lens.copy_(t.seq_lens)
        rng.copy_(t.free_range)

    key.zero_(), value.zero_(), q.zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for x, y in zip((lens, rng, c.tables), saved):
        x.copy_(y)
    for i in range(2 * ps + 3):
        rows_now = [random_rows(200 + 3 * i + j, rows, h, dim) for j, h in enumerate((hk, hk, hq))]
        for x, y in zip((key, value, q), rows_now):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        c.hold([1] * rows, *rows_now[:2])
        if i % 5 == 0 or i > 2 * ps:
            check(out, c.exact([1] * rows, rows_now[2]), max(len(h[0]) for h in c.held), P_TWO_TERMS)
    assert lens.tolist() == [len(h[0]) for h in c.held] and int(c.flags) == 0


def test_two_graphs_with_workspaces_of_their_own(mas, dev):
    """Two captured decode steps, each with its own workspace, replayed in turn and on two streams at once."""
    g = torch.Generator().manual_seed(9)
    from fp4_common import Cache
    runs = []
    for i in range(2):
        cache = Cache(60 + i, 64, 16, 2, 128, "HND")
        q = random_rows(70 + i, 6, 8, 128)
        lens = torch.randint(1, 1000, (6,), generator=g).to(torch.int32)
        tables = torch.randint(0, 64, (6, 64), generator=g).to(torch.int32)
        args = (q.to(dev), cache.on(mas, dev), torch.empty(8 << 20, dtype=torch.uint8, device=dev), tables.to(dev), lens.to(dev))
        out = torch.empty(6, 8, 128, dtype=torch.bfloat16, device=dev)
        call = lambda a=args, o=out: mas.attention.batch_decode_with_fp4_kv_cache(*a, 0, 0.1, 1.0, out=o, kv_layout="HND")
        call()
        torch.cuda.synchronize()
        want = out.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        runs.append((graph, out, want, args))             # (a graph's tensors live as long as it is replayed)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for _, out, _, _ in runs:
            out.zero_()
        torch.cuda.synchronize()
        for s, (graph, _, _, _) in zip(streams, runs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for _, out, want, _ in runs:
            assert torch.equal(out, want)
