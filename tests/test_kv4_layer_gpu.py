"""KV4Attention and the decode harness on it: a prompt, then tokens one by one, against 64 bits; the harness's step with
the 4-bit cache against its step with the fp16 one; a captured step."""
import os
import sys

import pytest
import torch

from oracle import serving_oracle as orc

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def test_layer_prompt_then_tokens(cuda):
    from vllm_quick_amd.layers.kv4_attention import KV4Attention, KV4Metadata, rope_table, slots_of
    heads, kv, d, p = 6, 2, 64, 16
    attn = KV4Attention(heads, d, kv)
    cache = attn.make_cache(9, p, cuda)
    cos_sin = rope_table(64, d, device=cuda)
    tables = torch.tensor([[3, 7, 1], [8, 0, 5]], dtype=torch.int32, device=cuda)
    g = torch.Generator().manual_seed(0)
    lens = [0, 0]
    for counts in ([20, 33], [1, 1], [3, 0], [1, 1]):
        t = sum(counts)
        qkv = torch.randn(t, (heads + 2 * kv) * d, generator=g).half().to(cuda)
        q, k, v = qkv.split([heads * d, kv * d, kv * d], 1)
        pos = torch.cat([torch.arange(n, n + m) for n, m in zip(lens, counts)]).to(cuda)
        seq = torch.repeat_interleave(torch.arange(2), torch.tensor(counts)).to(cuda)
        lens = [n + m for n, m in zip(lens, counts)]
        start = torch.tensor([0, counts[0], t], dtype=torch.int32, device=cuda)
        seq_lens = torch.tensor(lens, dtype=torch.int32, device=cuda)
        single = counts == [1, 1]
        meta = KV4Metadata(pos, slots_of(tables, pos, p, seq), tables, seq_lens, max(lens), None if single else start,
                           1 if single else max(counts))
        out = attn(q, k, v, cache, cos_sin, meta).view(t, heads, d)
        turned = orc.rotate64(q.cpu().view(t, heads, d), cos_sin.cpu(), pos.cpu(), False)[0].half()
        want, tol = orc.attend(turned, cache.cpu(), tables.cpu(), seq_lens.cpu(), start.cpu(), d**-0.5, 0, True)
        # the layer's queries are rotated in 32 bits before their rounding: a step of fp16 where that tips over
        tol = tol + 2.0**-10 * 2 * 4 * 8
        assert ((out.cpu().double() - want).abs() <= tol).all()


def test_slots_and_table(cuda):
    from vllm_quick_amd.layers.kv4_attention import rope_table, slots_of
    tables = torch.tensor([[4, 2], [0, 9]], dtype=torch.int32)
    assert slots_of(tables, torch.tensor([17, 3]), 16).tolist() == [2 * 16 + 1, 3]
    assert slots_of(tables, torch.tensor([0, 15, 16]), 16, torch.tensor([1, 1, 1])).tolist() == [0, 15, 9 * 16]
    t = rope_table(100001, 64)
    assert t.shape == (100001, 64) and t.dtype == torch.float32
    import math
    assert abs(float(t[100000, 3]) - math.cos(100000 * 10000.0**(-6 / 64))) < 2.0**-23
    assert abs(float(t[100000, 32])) == abs(float(torch.tensor(math.sin(100000.0), dtype=torch.float32)))
    assert rope_table(5, 0).shape == (5, 0)


def test_layer_refuses_heads_that_cannot_be_shared():
    from vllm_quick_amd.layers.kv4_attention import KV4Attention
    with pytest.raises(ValueError, match="cannot share"):
        KV4Attention(6, 64, 4)


@pytest.mark.parametrize("model", ["7b", "70b"])
def test_harness_step_on_the_4_bit_cache(cuda, model):
    """One layer's attention with the 4-bit cache against the fp16 cache's on the same keys and values: they differ by what
    4 bits keep of a value (half a step of 15 of a head's range, averaged over the context)."""
    from benchmarks.llama_decode import SHAPES, Model, rope_tables
    cfg = dict(SHAPES[model], hidden=512, inter=1024, heads=4, kv_heads=2 if model == "70b" else 4)
    bs, n = 3, 40
    with torch.inference_mode():
        plain = Model(cfg, 1, bs, n + 8, cuda, seed=1)
        four = Model(cfg, 1, bs, n + 8, cuda, seed=1, kv4=True)
        got = []
        for m in (plain, four):
            g = torch.Generator(device=cuda).manual_seed(3)
            outs = []
            layer = m.layers[0]
            layer.behind_attention = lambda x, att: att  # the attention itself
            for pos in range(n):
                x = torch.randn(bs, cfg["hidden"], generator=g, device=cuda).half()
                if m.kv4:
                    outs.append(layer(x, pos, m.cos_sin, None, pos + 1, m.kv4_metadata(bs, pos, pos + 1)))
                else:
                    outs.append(layer(x, pos, *rope_tables(m.cos[pos], m.sin[pos]), pos + 1))
            got.append(torch.stack(outs).float())
    rel = ((got[1] - got[0]).norm() / got[0].norm()).item()
    # a normal head of 128 values spans about 5.3 of its deviations: half a step rms is 5.3 / 15 / sqrt(12) = 0.10 of one
    # value; keys add as much through the scores
    assert 0.01 < rel < 0.3


def test_harness_runs(cuda):
    from benchmarks.llama_decode import run
    out = run("7b", (1, 4), n_layers=1, ctx_len=100, device=cuda, kv4=True, logprobs=3)
    assert out["kv_cache"].startswith("4 bits") and "3 alternative" in out["logprobs"]
    assert all(out["by_batch"][b]["tokens_per_s"] > 0 for b in ("1", "4"))
    plain = run("7b", (1, ), n_layers=1, ctx_len=100, device=cuda)
    assert "kv_cache" not in plain and "logprobs" not in plain


def test_captured_harness_step_chooses_what_the_eager_one_does(cuda):
    from benchmarks.llama_decode import SHAPES, Model
    cfg = dict(SHAPES["7b"], hidden=512, inter=1024, heads=4, kv_heads=4, vocab=1000)
    with torch.inference_mode():
        m = Model(cfg, 2, 4, 64, cuda, seed=2, kv4=True, logprobs=5)
        tokens = torch.randint(0, 1000, (4, ), device=cuda)
        meta = m.kv4_metadata(4, 0, 1)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            m.step(tokens, 0, 1, meta)
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = m.step(tokens, 0, 1, meta)
        from vllm_quick_amd.layers.kv4_attention import slots_of
        for pos in range(20):
            meta.positions.fill_(pos)
            meta.slots.copy_(slots_of(meta.block_tables, meta.positions, 16))
            meta.seq_lens.fill_(pos + 1)
            before = [layer.kv4_cache.clone() for layer in m.layers]
            want = [t.clone() for t in m.step(tokens, pos, pos + 1, meta)]
            for layer, c in zip(m.layers, before):
                layer.kv4_cache.copy_(c)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)
            assert torch.equal(want[0], want[2][:, 0]) and (want[1][:, :-1] >= want[1][:, 1:]).all()
            tokens.copy_(want[0])


@pytest.mark.parametrize("window,interleaved", [(0, False), (25, True)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_layer_against_the_oracle_with_nothing_to_spare(cuda, dtype, window, interleaved):
    """Prompts and tokens through the layer, the oracle given the queries as the operator rotates them (which has tests of
    its own), so that attention's counted roundings are all that is allowed."""
    from vllm_quick_amd import ops
    from vllm_quick_amd.layers.kv4_attention import KV4Attention, KV4Metadata, rope_table, slots_of
    heads, kv, d, p = 6, 2, 64, 16
    attn = KV4Attention(heads, d, kv, window=window, interleaved=interleaved)
    cache = attn.make_cache(9, p, cuda)
    cos_sin = rope_table(64, d, device=cuda)
    tables = torch.tensor([[3, 7, 1], [8, 0, 5]], dtype=torch.int32, device=cuda)
    g = torch.Generator().manual_seed(4)
    lens = [0, 0]
    for counts in ([20, 33], [1, 1], [3, 0], [1, 1], [20, 9]):
        t = sum(counts)
        qkv = torch.randn(t, (heads + 2 * kv) * d, generator=g).to(dtype).to(cuda)
        q, k, v = qkv.split([heads * d, kv * d, kv * d], 1)
        pos = torch.cat([torch.arange(n, n + m) for n, m in zip(lens, counts)]).to(cuda)
        seq = torch.repeat_interleave(torch.arange(2), torch.tensor(counts)).to(cuda)
        lens = [n + m for n, m in zip(lens, counts)]
        start = torch.tensor([0, counts[0], t], dtype=torch.int32, device=cuda)
        seq_lens = torch.tensor(lens, dtype=torch.int32, device=cuda)
        single = counts == [1, 1]
        slots = slots_of(tables, pos, p, seq)
        meta = KV4Metadata(pos, slots, tables, seq_lens, max(lens), None if single else start, 1 if single else max(counts))
        beside = cache.clone()
        turned = ops.rope_append_kv4(pos, q.view(t, heads, d), k.view(t, kv, d), v.view(t, kv, d), cos_sin, beside, slots, interleaved)
        out = attn(q, k, v, cache, cos_sin, meta).view(t, heads, d)
        assert torch.equal(cache, beside)
        want, tol = orc.attend(turned.cpu(), cache.cpu(), tables.cpu(), seq_lens.cpu(), start.cpu(), d**-0.5, window, dtype == torch.float16)
        assert ((out.cpu().double() - want).abs() <= tol).all()
