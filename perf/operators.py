"""Timed cases of the operators around a KV cache held in 4 bits, each in its plain form (elementary torch) and as a
call of this package's kernels.

The cache holds keys and values as microscaling fp4: a head's row of ``head_dim`` elements is cut into blocks of 32, a
block stored as 32 e2m1 codes (two a byte, the even element in the low half) and one power of two (a byte, exponent +
127). The block's power of two is the smallest one, of at least 2^-127, under which its largest element lies below 7,
so that no element is cut off by more than half a step; a block that holds a NaN or an infinity stands for NaN. Codes lie
as ``[pages, page_size, kv_heads, head_dim / 2]`` ("NHD") or ``[pages, kv_heads, page_size, head_dim / 2]`` ("HND"),
the powers as ``[pages, kv_heads, head_dim / 32, page_size]``.

- ``plan``: block tables, slots, positions and row lengths of a step, from its requests' lengths and the free pages.
- ``store``: a step's keys and values put into the cache and read back from their slots.
- ``decode``: attention of one query token per row over the cache.
- ``context``: causal attention of prompt rows over the cache.

Head shapes and lengths are those of ``mini-agent-serve_amd/workloads.py`` and ragged ones around them. Lengths come from
the case alone (its ``lens`` seed), so that a pass's work does not depend on the values' seed; the seed draws the values
and the pages' order.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BLOCK = 32                 # elements that share a power of two
WORKSPACE = 128 << 20      # the engine's attention workspace
NEVER = -1                 # the slot and row of a padding token


def listed():
    return [
        # The step plan of a decode batch: 256 conversations, one token each, some of which open a page. All latency.
        {"name": "plan_decode_256", "op": "plan", "decodes": 256, "max_len": 8192, "prompts": 0, "new": 0, "cached": 0,
         "page_size": 16, "tokens": 256, "lens": 1},
        # The step plan of a mixed step: 64 decode rows and chunked prompts, the token count padded to a multiple of 64.
        {"name": "plan_mixed_8384", "op": "plan", "decodes": 64, "max_len": 8192, "prompts": 8, "new": 2900,
         "cached": 4000, "page_size": 16, "tokens": 8384, "lens": 2},
        # A decode batch's new keys and values, one layer: 64 tokens into 64 pages.
        {"name": "store_64", "op": "store", "seqs": 64, "new": 1, "cached": 3001, "kv_heads": 8, "head_dim": 128,
         "page_size": 16, "layout": "HND"},
        # A prefill step's: 4 prompts of 2048 tokens.
        {"name": "store_8192", "op": "store", "seqs": 4, "new": 2048, "cached": 0, "kv_heads": 8, "head_dim": 128,
         "page_size": 16, "layout": "HND"},
        # One conversation being decoded: the smallest attention call, all latency.
        {"name": "decode_1x4096", "op": "decode", "rows": 1, "max_len": 4096, "reach": 8192, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "page_size": 16, "layout": "HND", "lens": 9},
        # A full decode batch: 64 rows of 1..8192 positions. Most of a decode step's time.
        {"name": "decode_64x8192", "op": "decode", "rows": 64, "max_len": 8192, "reach": 8192, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "page_size": 16, "layout": "HND", "lens": 0},
        # A middling batch of the larger model's heads, 256-slot pages in the other layout, odd lengths under a table
        # that reaches further.
        {"name": "decode_24x3000_group12", "op": "decode", "rows": 24, "max_len": 3000, "reach": 8192, "q_heads": 96,
         "kv_heads": 8, "head_dim": 128, "page_size": 256, "layout": "NHD", "lens": 2},
        # Many short rows of a shard's heads, head_dim 64.
        {"name": "decode_200x1000_dim64", "op": "decode", "rows": 200, "max_len": 1000, "reach": 1024, "q_heads": 16,
         "kv_heads": 4, "head_dim": 64, "page_size": 16, "layout": "HND", "lens": 4},
        # An agent's turn: a few new tokens after a long cached prefix.
        {"name": "context_turn_128_after4096", "op": "context", "rows": 1, "new": 128, "cached": 4096, "ragged": False,
         "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page_size": 16, "layout": "HND", "lens": 0},
        # Chunked prefill as it arrives: prompts of odd lengths after odd cached prefixes.
        {"name": "context_ragged_6x1500", "op": "context", "rows": 6, "new": 1500, "cached": 3000, "ragged": True,
         "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page_size": 16, "layout": "HND", "lens": 3},
        # Fresh prompts: the attention of an 8192-token prefill step.
        {"name": "context_4x2048", "op": "context", "rows": 4, "new": 2048, "cached": 0, "ragged": False,
         "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page_size": 16, "layout": "HND", "lens": 0},
        # Fresh prompts, the larger model's heads: the largest call.
        {"name": "context_4x4096_group12", "op": "context", "rows": 4, "new": 4096, "cached": 0, "ragged": False,
         "q_heads": 96, "kv_heads": 8, "head_dim": 128, "page_size": 256, "layout": "NHD", "lens": 0},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


#: No drawn case costs more than the largest listed one (context_4x4096_group12's operations, decode_64x8192's bytes).
_MOST_FLOPS, _MOST_BYTES = 1.6e12, 2.8e8


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w["flops"] <= _MOST_FLOPS and w["bytes"] <= _MOST_BYTES:
            return case


def _draw(rng):
    op = rng.choice(("plan", "store", "decode", "decode", "decode", "context", "context", "context"))
    page_size = rng.choice((16, 16, 64, 256))
    if op == "plan":
        case = {"op": op, "decodes": _spread(rng, 1, 1000), "max_len": _spread(rng, 16, 16000), "prompts": 0, "new": 0,
                "cached": 0, "page_size": page_size, "tokens": 0, "lens": rng.randint(0, 999)}
        if rng.random() < 0.6:
            case.update(prompts=rng.randint(1, 16), new=_spread(rng, 1, 2000), cached=rng.randint(0, 5000))
        n = sum(new for new, _ in _plan_lens(case))
        case["tokens"] = n if rng.random() < 0.3 else -(-n // 64) * 64
        return case
    kv = rng.choice((8, 8, 8, 4, 1))                      # whole, or a shard's kv heads
    heads = {"kv_heads": kv, "head_dim": rng.choice((128, 128, 128, 64)), "page_size": page_size,
             "layout": rng.choice(("HND", "HND", "NHD"))}
    if op == "store":
        return {"op": op, "seqs": _spread(rng, 1, 200), "new": _spread(rng, 1, 3000), "cached": rng.randint(0, 4000),
                **heads}
    q_heads = kv * rng.choice((4, 4, 12, 1, 7))
    if op == "decode":
        most = _spread(rng, 32, 20000)
        return {"op": op, "rows": _spread(rng, 1, 200), "max_len": most,
                "reach": most if rng.random() < 0.5 else max(8192, most), "q_heads": q_heads, **heads,
                "lens": rng.randint(0, 999)}
    return {"op": op, "rows": _spread(rng, 1, 12), "new": _spread(rng, 2, 5000),
            "cached": 0 if rng.random() < 0.4 else _spread(rng, 1, 9000), "ragged": rng.random() < 0.6,
            "q_heads": q_heads, **heads, "lens": rng.randint(0, 999)}


# ---- lengths -----------------------------------------------------------------------------------------

def _plan_lens(case):
    """(new tokens, cached positions) of each row: decode rows, then prompts."""
    r = random.Random(case["lens"])
    rows = [(1, r.randint(0, case["max_len"] - 1)) for _ in range(case["decodes"])]
    return rows + [(r.randint(1, case["new"]), r.randint(0, case["cached"])) for _ in range(case["prompts"])]


def _decode_lens(case):
    r = random.Random(case["lens"])
    return [r.randint(1, case["max_len"]) for _ in range(case["rows"])]


def _context_lens(case):
    """(new tokens, cached positions) of each row."""
    if not case["ragged"]:
        return [(case["new"], case["cached"])] * case["rows"]
    r = random.Random(case["lens"])
    return [(r.randint(1, case["new"]), r.randint(0, case["cached"])) for _ in range(case["rows"])]


# ---- what a pass cannot do without ---------------------------------------------------------------------

def _attended(n, c):
    """(query, key) pairs of n new tokens after c cached positions, causal."""
    return n * c + n * (n + 1) // 2


def work(case):
    op, ps = case["op"], case["page_size"]
    if op == "plan":
        # lengths read and written, positions, rows and slots of every token written, a page read and written each
        lens = _plan_lens(case)
        opened = sum(-(-(n + c) // ps) - -(-c // ps) for n, c in lens)
        return {"bytes": 16 * len(lens) + 16 * case["tokens"] + 8 * opened, "flops": 8 * case["tokens"]}
    hk, d = case["kv_heads"], case["head_dim"]
    row = hk * (d // 2 + d // BLOCK)                      # one position's keys (or values) in the cache, bytes
    if op == "store":
        n = case["seqs"] * case["new"]
        return {"bytes": n * (2 * (4 * hk * d + 2 * row) + 16), "flops": 8 * n * hk * d}
    hq = case["q_heads"]
    if op == "decode":
        lens = _decode_lens(case)
        pages = sum(-(-n // ps) for n in lens)
        return {"bytes": sum(lens) * 2 * row + len(lens) * (hq * d * 4 + 4) + 4 * pages, "flops": 4 * sum(lens) * hq * d}
    lens = _context_lens(case)
    pages = sum(-(-(n + c) // ps) for n, c in lens)
    return {"bytes": sum(n + c for n, c in lens) * 2 * row + sum(n for n, _ in lens) * hq * d * 4 + 4 * pages,
            "flops": 4 * sum(_attended(n, c) for n, c in lens) * hq * d}


# ---- inputs --------------------------------------------------------------------------------------------

class _Values:
    """Seeded values drawn on the GPU, and seeded choices on the host."""

    def __init__(self, seed):
        self.dev = torch.device("cuda", torch.cuda.current_device())
        self.gen = torch.Generator(device=self.dev).manual_seed(seed)
        self.rng = random.Random(seed)
        self.host = torch.Generator().manual_seed(seed)

    def normal(self, *size):
        return torch.randn(*size, generator=self.gen, device=self.dev, dtype=torch.bfloat16)

    def channels(self, heads, dim):
        """Sizes of a head's channels: most near 1, a few several times larger, as rotated keys have them."""
        return torch.exp(0.7 * torch.randn(heads, dim, generator=self.gen, device=self.dev))

    def ints(self, values, dtype=torch.int32):
        return torch.tensor(values, dtype=dtype, device=self.dev)

    def tables(self, lens, page_size, reach):
        """Block tables of rows of `lens` positions over a pool that just holds them, pages in random order;
        columns past a row's pages point at the pool's last page."""
        need = [-(-n // page_size) for n in lens]
        pages = sum(need) + 1
        width = max(max(need), -(-reach // page_size))
        perm = torch.randperm(pages - 1, generator=self.host).to(torch.int32)
        tables = torch.full((len(lens), width), pages - 1, dtype=torch.int32)
        at = 0
        for row, k in enumerate(need):
            tables[row, :k] = perm[at:at + k]
            at += k
        return tables.to(self.dev), pages


def _quantize(x):
    """bf16 [..., dim] -> codes uint8 [..., dim / 2] and powers uint8 [..., dim / 32]."""
    b = x.float().unflatten(-1, (-1, BLOCK))
    most = b.abs().amax(-1)
    finite = torch.isfinite(most)
    frac, exp = torch.frexp(torch.where(finite, most, torch.ones_like(most)))   # most = frac 2^exp, 1/2 <= frac < 1
    power = torch.where(most > 0, exp - 3 + (frac >= 0.875).int(), torch.full_like(exp, -127)).clamp(min=-127)
    y = torch.ldexp(b.abs(), -power[..., None])
    code = ((y > 0.25).to(torch.uint8) + (y >= 0.75).to(torch.uint8) + (y > 1.25).to(torch.uint8)
            + (y >= 1.75).to(torch.uint8) + (y > 2.5).to(torch.uint8) + (y >= 3.5).to(torch.uint8)
            + (y > 5.0).to(torch.uint8))
    code = (code | (torch.signbit(b).to(torch.uint8) << 3)) * finite[..., None].to(torch.uint8)
    code = code.flatten(-2)
    powers = torch.where(finite, power + 127, torch.full_like(power, 255)).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), powers


def _cache(v, pages, case):
    """The keys' and values' codes and powers of a cache full of quantized rows."""
    ps, hk, d = case["page_size"], case["kv_heads"], case["head_dim"]
    parts = []
    for scaled in (True, False):
        sizes = v.channels(hk, d) if scaled else torch.ones(hk, d, device=v.dev)
        codes = torch.empty(pages, hk, ps, d // 2, dtype=torch.uint8, device=v.dev)
        powers = torch.empty(pages, hk, d // BLOCK, ps, dtype=torch.uint8, device=v.dev)
        step = max(1, (1 << 24) // (hk * ps * d))
        for p in range(0, pages, step):
            n = min(step, pages - p)
            c, s = _quantize((v.normal(n, hk, ps, d).float() * sizes[:, None]).bfloat16())
            codes[p:p + n], powers[p:p + n] = c, s.transpose(-1, -2)
        parts.append((codes if case["layout"] == "HND" else codes.transpose(1, 2).contiguous(), powers))
    return [parts[0][0], parts[1][0], parts[0][1], parts[1][1]]


def prepare(case, seed):
    v, op, ps = _Values(seed), case["op"], case["page_size"]
    s = {"case": case}
    if op == "plan":
        lens = _plan_lens(case)
        cached = [c for _, c in lens]
        width = max(-(-(n + c) // ps) for n, c in lens)
        tables, pages = v.tables(cached, ps, width * ps)
        opened = sum(-(-(n + c) // ps) - -(-c // ps) for n, c in lens)
        # the free pages: a ring, the first of them somewhere in it
        spare = opened + v.rng.randint(1, 64)
        ring = torch.randperm(spare, generator=v.host).to(torch.int32) + pages
        first = v.rng.randint(0, spare - 1)
        s.update(new=v.ints([n for n, _ in lens]), cached=v.ints(cached), tables=tables, ring=ring.to(v.dev),
                 range=v.ints([first, first + spare], torch.int64),
                 out=[torch.empty(n, dtype=t, device=v.dev) for n, t in (
                     (case["tokens"], torch.int32), (case["tokens"], torch.int32), (case["tokens"], torch.int64),
                     (len(lens) + 1, torch.int32), (len(lens), torch.int32), (2, torch.int64))])
        return s
    hk, d = case["kv_heads"], case["head_dim"]
    if op == "store":
        new, cached, seqs = case["new"], case["cached"], case["seqs"]
        n = seqs * new
        tables, pages = v.tables([cached + new] * seqs, ps, 0)
        qkv = torch.cat([(v.normal(n, hk, d).float() * v.channels(hk, d)).bfloat16().flatten(1),
                         v.normal(n, hk * d)], -1)       # keys and values as the projection leaves them: one row each
        shape = (pages, hk, ps, d // 2) if case["layout"] == "HND" else (pages, ps, hk, d // 2)
        cache = [torch.zeros(shape, dtype=torch.uint8, device=v.dev) for _ in range(2)]
        cache += [torch.zeros(pages, hk, d // BLOCK, ps, dtype=torch.uint8, device=v.dev) for _ in range(2)]
        positions = torch.arange(cached, cached + new, dtype=torch.int32, device=v.dev).repeat(seqs)
        batch = torch.arange(seqs, dtype=torch.int32, device=v.dev).repeat_interleave(new)
        page = tables[batch.long(), positions.long() // ps].long()
        s.update(key=qkv[:, :hk * d].unflatten(-1, (hk, d)), value=qkv[:, hk * d:].unflatten(-1, (hk, d)), cache=cache,
                 positions=positions, batch=batch, tables=tables, kv_indices=tables.flatten(),
                 kv_indptr=v.ints([r * tables.shape[1] for r in range(seqs + 1)]), slots=page * ps + positions.long() % ps,
                 out=[torch.empty(n, hk, d, dtype=torch.bfloat16, device=v.dev) for _ in range(2)])
        return s
    hq = case["q_heads"]
    if op == "decode":
        kv_lens = _decode_lens(case)
        v.rng.shuffle(kv_lens)
        tokens, reach = len(kv_lens), case["reach"]
    else:
        lens = _context_lens(case)
        v.rng.shuffle(lens)
        kv_lens, tokens, reach = [n + c for n, c in lens], sum(n for n, _ in lens), 0
        cu = [0]
        for n, _ in lens:
            cu.append(cu[-1] + n)
        s.update(cu=v.ints(cu), max_q=max(n for n, _ in lens), max_kv=max(kv_lens), cu_host=cu)
    tables, pages = v.tables(kv_lens, ps, reach)
    s.update(q=v.normal(tokens, hq, d), cache=_cache(v, pages, case), tables=tables, seq_lens=v.ints(kv_lens),
             lens_host=kv_lens, workspace=torch.zeros(WORKSPACE, dtype=torch.uint8, device=v.dev),
             out=torch.empty(tokens, hq, d, dtype=torch.bfloat16, device=v.dev))
    return s


# ---- a pass --------------------------------------------------------------------------------------------

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _package():
    from __graft_entry__ import load_package
    return load_package()


def _run_own(s):
    mas, case = _package(), s["case"]
    op = case["op"]
    if op == "plan":
        t = mas.step.plan_step(s["new"], s["cached"], s["tables"], s["ring"], s["range"], case["page_size"],
                               case["tokens"], out=mas.step.StepTables(*s["out"]))
        return {"positions": t.positions, "batch": t.batch_indices, "slots": t.slot_mapping, "cu": t.cu_seqlens_q,
                "seq_lens": t.seq_lens, "range": t.free_range, "tables": s["tables"]}
    cache = mas.page.Fp4KVCache(*s["cache"])
    if op == "store":
        mas.page.append_paged_kv_cache_fp4(s["key"], s["value"], s["batch"], s["positions"], cache, s["kv_indices"],
                                           s["kv_indptr"], None, case["layout"])
        key, value = mas.page.load_kv_slots_fp4(cache, s["slots"], case["layout"], key=s["out"][0], value=s["out"][1])
        return {"key": key, "value": value}
    scale = case["head_dim"] ** -0.5
    if op == "decode":
        return {"out": mas.attention.batch_decode_with_fp4_kv_cache(
            s["q"], cache, s["workspace"], s["tables"], s["seq_lens"], case["reach"], scale, 1.0, out=s["out"],
            kv_layout=case["layout"])}
    return {"out": mas.attention.batch_context_with_fp4_kv_cache(
        s["q"], cache, s["workspace"], s["tables"], s["seq_lens"], s["max_q"], s["max_kv"], scale, 1.0, case["rows"],
        s["cu"], out=s["out"], kv_layout=case["layout"])}


def _run_plain(s):
    op = s["case"]["op"]
    if op == "plan":
        return _plan(s)
    if op == "store":
        return _store(s)
    return _attention(s)


def _plan(s):
    case = s["case"]
    ps, tokens = case["page_size"], case["tokens"]
    dev = s["new"].device
    new, cached, width = s["new"].long(), s["cached"].long(), s["tables"].shape[1]
    fits = (new >= 0) & (cached >= 0) & (cached + new <= width * ps)
    new = torch.where(fits, new, torch.zeros_like(new))
    have = (cached + ps - 1) // ps
    need = torch.where(fits, (cached + new + ps - 1) // ps - have, torch.zeros_like(new))
    head, tail = s["range"][0], s["range"][1]
    # rows in order, as long as the pages and the tokens reach
    taken = (torch.cumsum(need, 0) <= tail - head) & (torch.cumsum(new, 0) <= tokens)
    new, need = new * taken, need * taken
    cu = torch.cat((torch.zeros(1, dtype=torch.int64, device=dev), torch.cumsum(new, 0)))
    first = torch.cumsum(need, 0) - need
    t = torch.arange(tokens, device=dev)
    row = torch.searchsorted(cu[1:], t, right=True)
    real = row < new.shape[0]
    row = torch.where(real, row, torch.zeros_like(row))
    pos = torch.where(real, cached[row] + t - cu[row], torch.zeros_like(t))
    block = pos // ps
    fresh = real & (block >= have[row])
    page = torch.where(fresh, s["ring"][(head + first[row] + block - have[row]) % s["ring"].shape[0]].long(),
                       s["tables"][row, block].long())
    # a page opened by a token of its first slot enters the row's table
    opens = fresh & (pos % ps == 0)
    flat = torch.where(opens, row * width + block, torch.full_like(row, s["tables"].numel()))
    grown = torch.cat((s["tables"].flatten(), torch.zeros(1, dtype=torch.int32, device=dev)))
    grown[flat] = page.int()
    s["tables"].copy_(grown[:-1].view_as(s["tables"]))
    slots = torch.where(real, page * ps + pos % ps, torch.full_like(pos, NEVER))
    return {"positions": pos.int(), "batch": torch.where(real, row, torch.full_like(row, NEVER)).int(), "slots": slots,
            "cu": cu.int(), "seq_lens": (s["cached"].long() + new).int(),
            "range": torch.stack((head + need.sum(), tail)), "tables": s["tables"]}


def _heads_last(codes, layout):
    """Codes with a page's slots before its heads."""
    return codes if layout == "NHD" else codes.transpose(1, 2)


def _decode_rows(codes, powers):
    """Codes [n, heads, dim / 2] and powers [n, heads, dim / 32] -> fp32 [n, heads, dim]."""
    steps = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0],
                         device=codes.device)
    x = torch.stack((steps[(codes & 15).long()], steps[(codes >> 4).long()]), -1).flatten(-2)
    power = torch.ldexp(torch.ones_like(powers, dtype=torch.float32), powers.int() - 127)
    power = torch.where(powers == 255, torch.full_like(power, math.nan), power)
    return (x.unflatten(-1, (-1, BLOCK)) * power[..., None]).flatten(-2)


def _store(s):
    case, ps = s["case"], s["case"]["page_size"]
    b, pos = s["batch"].long(), s["positions"].long()
    page = s["kv_indices"][s["kv_indptr"][b].long() + pos // ps].long()
    out = []
    for i, x in enumerate((s["key"], s["value"])):
        codes, powers = _quantize(x)
        _heads_last(s["cache"][i], case["layout"])[page, pos % ps] = codes
        s["cache"][2 + i].permute(0, 3, 1, 2)[page, pos % ps] = powers
        at, entry = s["slots"] // ps, s["slots"] % ps
        y = _decode_rows(_heads_last(s["cache"][i], case["layout"])[at, entry],
                         s["cache"][2 + i].permute(0, 3, 1, 2)[at, entry])
        s["out"][i].copy_(y)
        out.append(s["out"][i])
    return {"key": out[0], "value": out[1]}


def _row_of(s, i, table, length):
    """fp32 keys (i = 0) or values (i = 1) of a row's positions, [length, heads, dim]."""
    ps = s["case"]["page_size"]
    pages = table[: -(-length // ps)].long()
    codes = _heads_last(s["cache"][i][pages], s["case"]["layout"]).flatten(0, 1)[:length]
    return _decode_rows(codes, s["cache"][2 + i][pages].permute(0, 3, 1, 2).flatten(0, 1)[:length])


def _attention(s):
    """Both attentions: row r's tokens are its last positions, each attending to the ones up to its own."""
    case, q = s["case"], s["q"]
    hk, d = case["kv_heads"], case["head_dim"]
    g = case["q_heads"] // hk
    first = s["cu_host"] if case["op"] == "context" else list(range(case["rows"] + 1))
    for r, length in enumerate(s["lens_host"]):
        a, b = first[r], first[r + 1]
        n = b - a
        key, value = (_row_of(s, i, s["tables"][r], length) for i in (0, 1))
        at = torch.arange(length, device=q.device)
        hidden = at[None, :] > at[length - n:, None] if n > 1 else None
        # [kv heads, query heads of each, tokens, dim], as many kv heads at once as 2^29 scores allow
        x = q[a:b].float().view(n, hk, g, d).permute(1, 2, 0, 3)
        kt, vh = key.permute(1, 2, 0).contiguous(), value.transpose(0, 1).contiguous()
        many = max(1, min(hk, (1 << 29) // (g * n * length)))
        for h in range(0, hk, many):
            part = x[h:h + many].reshape(-1, g * n, d)
            scores = torch.matmul(part, kt[h:h + many]).view(-1, g, n, length) * d ** -0.5
            if hidden is not None:
                scores.masked_fill_(hidden, -math.inf)
            p = torch.exp(scores - scores.amax(-1, keepdim=True))
            o = torch.matmul(p.view(-1, g * n, length), vh[h:h + many]).view(-1, g, n, d) / p.sum(-1, keepdim=True)
            s["out"][a:b].view(n, hk, g, d)[:, h:h + many] = o.permute(2, 0, 1, 3).to(torch.bfloat16)
    return {"out": s["out"]}


# ---- the same in 64 bits -------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "plan":
        return None                                     # whole numbers throughout
    if op == "store":
        return {"key": _nearest64(s["key"]), "value": _nearest64(s["value"])}
    hk, ps, d = case["kv_heads"], case["page_size"], case["head_dim"]
    g = case["q_heads"] // hk
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    first = list(range(case["rows"] + 1)) if op == "decode" else s["cu_host"]
    for r, length in enumerate(s["lens_host"]):
        a, b = first[r], first[r + 1]
        pages = s["tables"][r, : -(-length // ps)].long()
        kv = []
        for i in (0, 1):
            x = _values64(s["cache"][i][pages], s["cache"][2 + i][pages], case["layout"])
            kv.append(x.transpose(0, 1).flatten(1, 2)[:, :length])       # [heads, length, dim]
        last = torch.arange(length - (b - a), length, device=out.device)[:, None]
        over = torch.arange(length, device=out.device)[None, :] > last
        for e in range(hk * g):
            scores = torch.mm(s["q"][a:b, e].double(), kv[0][e // g].t().contiguous()) / math.sqrt(d)
            out[a:b, e] = torch.mm(torch.softmax(scores.masked_fill_(over, -math.inf), -1), kv[1][e // g].contiguous())
    return {"out": out}


def _values64(codes, powers, layout):
    """Whole pages' values, [pages, heads, page_size, dim]: an e2m1 code is (1 + m / 2) 2^(e - 1), or m / 2 for e = 0."""
    if layout == "NHD":
        codes = codes.transpose(1, 2)
    both = torch.stack((codes % 16, codes // 16), -1).flatten(-2)
    e, m = (both // 2 % 4).double(), (both % 2).double()
    size = torch.where(e == 0, m / 2, (1 + m / 2) * torch.exp2(e - 1))
    size = torch.where(both >= 8, -size, size)
    power = torch.exp2(powers.double() - 127).transpose(-1, -2).repeat_interleave(BLOCK, -1)
    return size * power


def _nearest64(x):
    """Each element's nearest step of its block, ties to the even code."""
    b = x.double().unflatten(-1, (-1, BLOCK))
    top = b.abs().amax(-1, keepdim=True)
    power = torch.full_like(top, 2.0 ** -127)
    exps = torch.arange(-126, 128, device=x.device, dtype=torch.float64)
    # the smallest power of two p with top < 7 p
    count = torch.searchsorted(7 * torch.exp2(exps), top.flatten(), right=True).view(top.shape)
    power = torch.where(top >= 7 * 2.0 ** -127, torch.exp2(exps[count.clamp(max=len(exps) - 1)]), power)
    steps = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    best = torch.zeros_like(b)
    gap = torch.full_like(b, math.inf)
    for code in (0, 2, 4, 6, 1, 3, 5, 7):               # even codes first: a tie keeps them
        dist = (b.abs() / power - steps[code]).abs()
        nearer = dist < gap
        best, gap = torch.where(nearer, steps[code], best), torch.where(nearer, dist, gap)
    return (torch.copysign(best, b) * power).flatten(-2)
