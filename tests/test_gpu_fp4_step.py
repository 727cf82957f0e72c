"""A whole step over the 4-bit cache (layer_pass.ForwardStep, kv_format="fp4"), and the 4-bit operators in a compiled
step. The step over the bf16 cache, made from the same seed, is the measure of all that the cache does not touch."""
from __future__ import annotations

import dataclasses

import numpy as np
import pytest
import torch

from conftest import bits, fp8_codes
from fp4_common import P_BF16, P_TWO_TERMS, random_rows, tolerance
from oracle import fp4
from oracle import numerics as on

pytestmark = pytest.mark.gpu


def _shape(mas, prompts, decode_rows=5, max_len=300, page_size=16, reach=512):
    wl = mas.workloads
    layer = dataclasses.replace(wl.SHAPES["decode64_24b"], vocab=4096)
    return wl.StepShape("test_step", decode_rows=decode_rows, max_len=max_len, prompts=prompts, layers=2,
                        page_size=page_size, reach=reach, layer=layer)


def _check_fp8(codes, exact, positions, p_round, scale):
    """e4m3 codes of a bf16 output over scale: off by the bf16 output's tolerance and half an e4m3 step (2^-4 of the
    value, 2^-10 below 2^-6), and by the division's own 2^-24."""
    out, size, reach = exact
    z = np.clip(out / scale, -448, 448)
    moved = tolerance(out, size, reach, positions, p_round) / scale
    allowed = moved + np.maximum((np.abs(z) + moved) * (2.0 ** -4 + 2.0 ** -20), 2.0 ** -10)
    assert (np.abs(on.fp8_to_f32(codes).astype(np.float64) - z) <= allowed).all()


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("case", [dict(prompts=()), dict(prompts=((20, 50),)),
                                  dict(prompts=((60, 0), (1, 400), (33, 127)), decode_rows=9, page_size=64),
                                  dict(prompts=((17, 255),), decode_rows=1, max_len=40, page_size=256, reach=1024)])
def test_forward_step(mas, dev, case, graph):
    shape = _shape(mas, **case)
    plain = mas.layer_pass.ForwardStep(shape, dev, seed=11)
    plain.run()
    fs = mas.layer_pass.ForwardStep(shape, dev, seed=11, kv_format="fp4")
    if graph:
        before = [fs.residual.clone(), fs.final_in.clone()] + [layer["qkv"].clone() for layer in fs.layers]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            fs.run()
            with torch.cuda.graph(g, stream=side):
                fs.run()
        torch.cuda.synchronize()
        for _ in range(3):                           # the step in place: from the same inputs again each time
            for t, was in zip([fs.residual, fs.final_in] + [layer["qkv"] for layer in fs.layers], before):
                t.copy_(was)
            g.replay()
            torch.cuda.synchronize()
    else:
        fs.run()
    torch.cuda.synchronize()
    lay, ls, ps = fs.layout, shape.layer, shape.page_size
    n, d = fs.num_tokens, fs.num_decodes
    real = d + sum(q for q, _ in shape.prompts)
    # what the cache does not touch
    assert torch.equal(fs.residual, plain.residual) and torch.equal(fs.final_in, plain.final_in)
    assert torch.equal(fs.silu_out.view(torch.uint8), plain.silu_out.view(torch.uint8))
    # the plan is the host's layout; padding comes last and has no slot
    used = d + len(shape.prompts)
    assert torch.equal(fs.plan.positions[:real].cpu(), lay.positions[:real])
    assert torch.equal(fs.plan.batch_indices[:real].cpu(), lay.batch_indices[:real])
    assert torch.equal(fs.plan.seq_lens[:used].cpu(), lay.seq_lens[:used])
    assert fs.plan.slot_mapping[real:].tolist() == [-1] * (n - real)
    slots = fs.plan.slot_mapping[:real].cpu()
    rows, pos = lay.batch_indices[:real].long(), lay.positions[:real].long()
    assert torch.equal(slots, lay.block_tables[rows, pos // ps].long() * ps + pos % ps)
    # the last layer's cache holds every real token's rotated key and its value, quantized
    last = fs.layers[-1]
    q, k, v = fs.views(last)
    assert torch.equal(q[:real], plain.views(plain.layers[-1])[0][:real])
    kv = [t.cpu().numpy() for t in last["kv"]]
    held = [fp4.cache_rows(kv[i], kv[2 + i], "HND") for i in range(2)]
    for rows_, have in ((k, held[0]), (v, held[1])):
        want = fp4.dequantize(*fp4.quantize(bits(rows_[:real].reshape(real, ls.kv_heads, ls.head_dim))))
        assert np.array_equal(have[slots.numpy() // ps, slots.numpy() % ps], want)
    # and the attention reads it
    qb = bits(q).reshape(n, ls.q_heads, ls.head_dim)
    tables, lens = lay.block_tables.numpy(), lay.seq_lens.numpy()
    got, scale = fp8_codes(fs.attn_out), float(fs.act_scale)
    exact = fp4.decode_attention(qb[:d], *held, tables[:d], lens[:d], fs.scale)
    _check_fp8(got[:d], exact, int(lens.max()), P_TWO_TERMS, scale)
    if shape.prompts:
        cu = np.cumsum([0] + [x for x, _ in shape.prompts])
        exact = fp4.context_attention(qb[d:real], *held, tables[d:used], lens[d:used], cu, fs.scale)
        _check_fp8(got[d:real], exact, int(lens.max()), P_BF16, scale)


def test_forward_step_refuses(mas, dev):
    with pytest.raises(ValueError, match="kv_format"):
        mas.layer_pass.ForwardStep(_shape(mas, ()), dev, kv_format="int4")
    with pytest.raises(ValueError, match="query scale"):
        mas.layer_pass.ForwardStep(_shape(mas, (), reach=16384), dev, kv_format="fp4")


def test_compiled_step(mas, dev):
    """Plan, store, both attentions and the load, compiled and captured, over views of one buffer: as the eager step."""
    rows, tokens, hq, hk, dim, ps, pages = 3, 24, 8, 2, 128, 16, 40

    def fresh():
        cache = mas.page.fp4_kv_cache(pages, ps, hk, dim, dev, "HND")
        for t in cache:
            t.zero_()
        return (cache, torch.zeros(rows, 8, dtype=torch.int32, device=dev),
                torch.zeros(tokens, hq, dim, dtype=torch.bfloat16, device=dev),
                torch.zeros(8 << 20, dtype=torch.uint8, device=dev))

    qkv = random_rows(5, tokens, hq + 2 * hk, dim).flatten(1).to(dev)
    new = torch.tensor([1, 1, 17], dtype=torch.int32, device=dev)
    cached = torch.tensor([3, 40, 5], dtype=torch.int32, device=dev)
    free = torch.arange(pages, dtype=torch.int32, device=dev).flip(0).contiguous()
    span = torch.tensor([0, pages], device=dev)
    old = random_rows(6, pages * ps, hk, dim).to(dev)

    def step(qkv, kv, tables, out, workspace):
        plan = mas.plan_step(new, cached, tables, free, span, ps, qkv.shape[0])
        q = qkv[:, :hq * dim].unflatten(-1, (hq, dim))
        k = qkv[:, hq * dim:(hq + hk) * dim]
        v = qkv[:, (hq + hk) * dim:].unflatten(-1, (hk, dim))
        mas.page.store_kv_slots_fp4(k, v, kv, plan.slot_mapping, "HND")
        mas.attention.batch_decode_with_fp4_kv_cache(q[:2], kv, workspace, tables[:2], plan.seq_lens[:2], 128, 0.1, 1.0,
                                                     out=out[:2], kv_layout="HND")
        mas.attention.batch_context_with_fp4_kv_cache(q, kv, workspace, tables[2:], plan.seq_lens[2:], 17, 128, 0.1, 1.0,
                                                      1, plan.cu_seqlens_q[2:], None, out=out, kv_layout="HND")
        back = mas.page.load_kv_slots_fp4(kv, plan.slot_mapping[:2], "HND")
        return out * 2, back[0] + back[1], plan.positions + 1

    def prepared():
        kv, tables, out, workspace = fresh()
        mas.page.store_kv_slots_fp4(old, old.flip(0).contiguous(), kv, torch.arange(pages * ps, device=dev), "HND")
        tables[1, :3] = torch.tensor([1, 2, 3])
        tables[0, 0], tables[2, 0] = 4, 5
        return kv, tables, out, workspace

    eager = prepared()
    want = step(qkv, *eager)
    torch._dynamo.reset()
    compiled = torch.compile(step, dynamic=True)
    args = prepared()
    got = compiled(qkv, *args)
    for a, b in zip(got + tuple(args[0]) + args[1:3], want + tuple(eager[0]) + eager[1:3]):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        compiled(qkv, *args)
        with torch.cuda.graph(g, stream=side):
            captured = compiled(qkv, *args)
    for _ in range(3):
        for t in captured:
            t.zero_()
        args[2].zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured + tuple(args[0]) + args[1:3], want + tuple(eager[0]) + eager[1:3]):
            assert torch.equal(a, b)
