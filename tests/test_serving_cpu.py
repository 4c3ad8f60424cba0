"""libserving_ops.so without a GPU: symbols, sizes, refusals of the C entries and of the operators (nothing is launched),
and the oracle's own pieces against each other."""
import ctypes
import os
import re
import subprocess
import sys

import pytest
import torch

from oracle import serving_oracle as orc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "serving_ops.h")


@pytest.fixture(scope="module")
def lib():
    import vllm_quick_amd  # noqa: F401  (torch's HIP runtime first)
    raw = ctypes.CDLL(os.path.join(ROOT, "vllm_quick_amd", "csrc", "libserving_ops.so"))
    raw.serving_strerror.restype = ctypes.c_char_p
    for name in ("serving_kv4_cache_bytes", "serving_attend_kv4_workspace_bytes", "serving_token_logprobs_workspace_bytes"):
        getattr(raw, name).restype = ctypes.c_size_t
    return raw


@pytest.fixture(scope="module")
def ops():
    from vllm_quick_amd import ops
    return ops


P = ctypes.c_void_p(4096)  # never dereferenced: every call below is refused first
LL = ctypes.c_longlong


def test_every_declared_symbol_is_there(lib):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(serving_[a-z0-9_]+)\s*\(", text)))
    assert len(names) >= 9
    for n in names:
        assert hasattr(lib, n), n
    assert lib.serving_abi_version() == 1
    assert lib.serving_strerror(0) == b"ok" and lib.serving_strerror(-99) == b"unknown serving error"
    texts = [lib.serving_strerror(-i) for i in range(1, 10)]
    assert len(set(texts)) == 9 and b"unknown serving error" not in texts


def test_sizes(lib):
    assert lib.serving_kv4_cache_bytes(LL(10), 16, 8, 128) == 10 * 8 * 16 * 136
    assert lib.serving_kv4_cache_bytes(LL(10), 24, 8, 128) == 0 and lib.serving_kv4_cache_bytes(LL(10), 16, 8, 96) == 0
    assert lib.serving_kv4_cache_bytes(LL(1 << 30), 4096, 8, 128) == (1 << 30) * 8 * 4096 * 136
    assert lib.serving_token_logprobs_workspace_bytes(4, 1000, 5, 0) == 0
    assert lib.serving_token_logprobs_workspace_bytes(4, 0, 0, 0) == 0
    assert lib.serving_token_logprobs_workspace_bytes(4, 500000, 5, 0) > 0
    assert lib.serving_attend_kv4_workspace_bytes(1, 1, 7, 2, 128, 1, 100, 0) == 0  # refused sizes
    one = lib.serving_attend_kv4_workspace_bytes(1, 1, 8, 2, 128, 1, 65536, 0)
    assert one > 0 and one % ((128 + 2) * 4 * 8) == 0


def append(lib, q=P, k=P, v=P, cs=P, pos=P, slots=P, out=P, cache=P, stride=1024, cstride=128, tokens=3, heads=8, kv=2, d=128,
           rotary=128, positions=64, blocks=4, block=16):
    s = [LL(stride), LL(128)]
    return lib.serving_rope_append_kv4(q, *s, k, *s, v, *s, cs, LL(cstride), pos, slots, out, cache, tokens, heads, kv, d, rotary, 0,
                                       LL(positions), LL(blocks), block, 0, None)


def test_append_refusals(lib):
    for name in ("q", "k", "v", "cs", "pos", "slots", "out", "cache"):
        assert append(lib, **{name: None}) == -1, name
    odd = ctypes.c_void_p(4104)
    for name in ("q", "k", "v", "cs", "out", "cache"):
        assert append(lib, **{name: odd}) == -6, name
    assert append(lib, stride=1020) == -6 and append(lib, cstride=127) == -6
    for name in ("tokens", "heads", "kv", "blocks"):
        assert append(lib, **{name: 0}) == -2 and append(lib, **{name: -1}) == -2, name
    assert append(lib, positions=-1) == -2 and append(lib, heads=70000) == -2
    assert append(lib, d=96) == -3 and append(lib, block=8) == -4 and append(lib, block=8192) == -4
    assert append(lib, rotary=24) == -5 and append(lib, rotary=144) == -5 and append(lib, rotary=-16) == -5
    assert append(lib, tokens=(1 << 30) + 1) == -8


def test_read_refusals(lib):
    def read(cache=P, slots=P, k=P, v=P, rows=3, kv=2, d=128, blocks=4, block=16):
        return lib.serving_read_kv4(cache, slots, k, v, LL(rows), kv, d, LL(blocks), block, 0, None)

    for name in ("cache", "slots", "k", "v"):
        assert read(**{name: None}) == -1, name
    for name in ("cache", "k", "v"):
        assert read(**{name: ctypes.c_void_p(4098)}) == -6, name
    assert read(rows=0) == -2 and read(kv=0) == -2 and read(blocks=0) == -2 and read(blocks=1 << 31) == -2
    assert read(d=32) == -3 and read(block=0) == -4 and read(rows=1 << 39) == -8


def attend(lib, q=P, cache=P, tables=P, lens=P, start=P, out=P, ws=P, stride=1024, width=4, tokens=3, seqs=2, heads=8, kv=2, d=128,
           blocks=4, block=16, scale=1.0, window=0, most_q=2, most=100, ws_bytes=1 << 30):
    return lib.serving_attend_kv4(q, LL(stride), LL(128), cache, tables, LL(width), width, lens, start, out, tokens, seqs, heads, kv, d,
                                  LL(blocks), block, ctypes.c_float(scale), window, most_q, most, 0, ws, ctypes.c_size_t(ws_bytes), None)


def test_attend_refusals(lib):
    for name in ("q", "cache", "tables", "lens", "out"):
        assert attend(lib, **{name: None}) == -1, name
    for name in ("q", "cache", "out"):
        assert attend(lib, **{name: ctypes.c_void_p(4100)}) == -6, name
    assert attend(lib, stride=12) == -6
    assert attend(lib, start=None) == -2  # one query a sequence: tokens has to be seqs
    assert attend(lib, start=None, tokens=2) == -2  # and max_query_len 1
    for name in ("tokens", "seqs", "heads", "kv", "width", "blocks", "most_q", "most"):
        assert attend(lib, **{name: 0}) == -2, name
    assert attend(lib, heads=7) == -2 and attend(lib, window=-1) == -2 and attend(lib, most=(1 << 27) + 1) == -2
    assert attend(lib, scale=float("nan")) == -2 and attend(lib, scale=float("inf")) == -2
    assert attend(lib, d=80) == -3 and attend(lib, block=20) == -4
    assert attend(lib, width=1 << 24) == -8
    assert attend(lib, most=100000, ws=None) == -9 and attend(lib, most=100000, ws_bytes=16) == -9
    assert attend(lib, most=100000, ws=ctypes.c_void_p(4100)) == -6


def test_logprobs_refusals(lib):
    def score(x=P, ids=P, lp=P, ent=P, tid=P, tlp=P, rows=2, vocab=100, top=3, kind=0, ws=P, ws_bytes=1 << 30):
        return lib.serving_token_logprobs(x, LL(vocab), ids, lp, ent, tid, tlp, rows, vocab, top, kind, ws, ctypes.c_size_t(ws_bytes), None)

    for name in ("x", "ids", "lp", "ent", "tid", "tlp"):
        assert score(**{name: None}) == -1, name
    assert score(rows=0) == -2 and score(vocab=0) == -2 and score(top=65) == -2 and score(top=-1) == -2 and score(vocab=2) == -2
    assert score(kind=3) == -2 and score(kind=-1) == -2
    assert score(x=ctypes.c_void_p(4097)) == -6 and score(x=ctypes.c_void_p(4098), kind=2) == -6
    assert score(vocab=500000, ws=None) == -9 and score(vocab=500000, ws_bytes=8) == -9
    assert score(vocab=2096641) == -2 and score(vocab=20000, rows=1 << 30) == -8


# ---------------------------------------------------------------------------------------------------------------
# the operators: shapes and types are refused before devices, and CPU tensors at last
# ---------------------------------------------------------------------------------------------------------------
def append_args(**change):
    a = dict(positions=torch.zeros(3, dtype=torch.int64), query=torch.zeros(3, 8, 128, dtype=torch.float16),
             key=torch.zeros(3, 2, 128, dtype=torch.float16), value=torch.zeros(3, 2, 128, dtype=torch.float16),
             cos_sin=torch.zeros(10, 128), cache=torch.zeros(4, 2, 16 * 136, dtype=torch.uint8), slots=torch.zeros(3, dtype=torch.int64))
    a.update(change)
    return a


@pytest.mark.parametrize("change,error,text", [
    (dict(query=torch.zeros(3, 8, 128)), RuntimeError, "Half or BFloat16"),
    (dict(key=torch.zeros(3, 2, 128, dtype=torch.bfloat16)), RuntimeError, "key"),
    (dict(value=torch.zeros(3, 2, 128)), RuntimeError, "value"),
    (dict(cos_sin=torch.zeros(10, 128, dtype=torch.float16)), RuntimeError, "cos_sin"),
    (dict(positions=torch.zeros(3, dtype=torch.int32)), RuntimeError, "positions"),
    (dict(slots=torch.zeros(3, dtype=torch.int32)), RuntimeError, "slots"),
    (dict(cache=torch.zeros(4, 2, 16 * 136)), RuntimeError, "cache"),
    (dict(query=torch.zeros(3, 1024, dtype=torch.float16)), ValueError, "query must be"),
    (dict(query=torch.zeros(3, 8, 96, dtype=torch.float16)), ValueError, "64 or 128"),
    (dict(cache=torch.zeros(4, 2, 24 * 136, dtype=torch.uint8)), ValueError, "multiple of 16"),
    (dict(cache=torch.zeros(4, 2, 16 * 72, dtype=torch.uint8)), ValueError, "cache must be"),
    (dict(cache=torch.zeros(4, 2, 2 * 16 * 136, dtype=torch.uint8)[:, :, ::2]), ValueError, "contiguous"),
    (dict(key=torch.zeros(3, 4, 128, dtype=torch.float16)), ValueError, "key must be"),
    (dict(value=torch.zeros(2, 2, 128, dtype=torch.float16)), ValueError, "value must be"),
    (dict(positions=torch.zeros(4, dtype=torch.int64)), ValueError, "positions"),
    (dict(slots=torch.zeros(3, 1, dtype=torch.int64)), ValueError, "slots"),
    (dict(cos_sin=torch.zeros(10, 40)), ValueError, "multiple of 16"),
    (dict(cos_sin=torch.zeros(10, 256)), ValueError, "no larger than a head"),
    (dict(cos_sin=torch.zeros(128)), ValueError, "cos_sin must be"),
    (dict(), RuntimeError, "GPU tensor"),
])
def test_append_operator_refusals(ops, change, error, text):
    with pytest.raises(error, match=text):
        ops.rope_append_kv4(**append_args(**change))


def attend_args(**change):
    a = dict(query=torch.zeros(2, 8, 128, dtype=torch.float16), cache=torch.zeros(4, 2, 16 * 136, dtype=torch.uint8),
             block_tables=torch.zeros(2, 3, dtype=torch.int32), seq_lens=torch.zeros(2, dtype=torch.int32), scale=1.0, max_seq_len=40)
    a.update(change)
    return a


@pytest.mark.parametrize("change,error,text", [
    (dict(query=torch.zeros(2, 8, 128)), RuntimeError, "Half or BFloat16"),
    (dict(block_tables=torch.zeros(2, 3, dtype=torch.int64)), RuntimeError, "block_tables"),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int64)), RuntimeError, "seq_lens"),
    (dict(query=torch.zeros(2, 7, 128, dtype=torch.float16)), ValueError, "cannot share"),
    (dict(query=torch.zeros(2, 0, 128, dtype=torch.float16)), ValueError, "cannot share"),
    (dict(query=torch.zeros(3, 8, 128, dtype=torch.float16)), ValueError, "one query for each"),
    (dict(max_query_len=2), ValueError, "max_query_len is 1"),
    (dict(max_query_len=0), ValueError, "max_query_len"),
    (dict(block_tables=torch.zeros(3, 3, dtype=torch.int32)), ValueError, "block_tables"),
    (dict(seq_lens=torch.zeros(2, 1, dtype=torch.int32)), ValueError, "seq_lens"),
    (dict(max_seq_len=0), ValueError, "2\\^27"),
    (dict(max_seq_len=1 << 28), ValueError, "2\\^27"),
    (dict(window=-1), ValueError, "window"),
    (dict(scale=float("nan")), ValueError, "finite"),
    (dict(scale=1e300), ValueError, "finite"),
    (dict(query_start=torch.zeros(2, dtype=torch.int32)), ValueError, "query_start"),
    (dict(query_start=torch.zeros(3, dtype=torch.int64)), RuntimeError, "query_start"),
    (dict(), RuntimeError, "GPU tensor"),
])
def test_attend_operator_refusals(ops, change, error, text):
    with pytest.raises(error, match=text):
        ops.paged_attention_kv4(**attend_args(**change))


@pytest.mark.parametrize("args,error,text", [
    ((torch.zeros(2, 5, dtype=torch.float64), torch.zeros(2, dtype=torch.int64), 1), RuntimeError, "Float"),
    ((torch.zeros(2, 5), torch.zeros(2, dtype=torch.int32), 1), RuntimeError, "token_ids"),
    ((torch.zeros(5), torch.zeros(1, dtype=torch.int64), 1), ValueError, "logits must be"),
    ((torch.zeros(2, 0), torch.zeros(2, dtype=torch.int64), 0), ValueError, "logits must be"),
    ((torch.zeros(2, 5), torch.zeros(3, dtype=torch.int64), 1), ValueError, "token_ids"),
    ((torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64), 6), ValueError, "top_n"),
    ((torch.zeros(2, 500), torch.zeros(2, dtype=torch.int64), 65), ValueError, "top_n"),
    ((torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64), -1), ValueError, "top_n"),
    ((torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64), 1), RuntimeError, "GPU tensor"),
])
def test_logprobs_operator_refusals(ops, args, error, text):
    with pytest.raises(error, match=text):
        ops.token_logprobs(*args)


def test_other_operator_refusals(ops):
    with pytest.raises(ValueError, match="64 or 128"):
        ops.kv4_cache(2, 16, 2, 80, torch.device("cpu"))
    with pytest.raises(ValueError, match="multiple of 16"):
        ops.kv4_cache(2, 8, 2, 64, torch.device("cpu"))
    with pytest.raises(ValueError, match="blocks and heads"):
        ops.kv4_cache(0, 16, 2, 64, torch.device("cpu"))
    cache = ops.kv4_cache(2, 16, 2, 64, torch.device("cpu"))
    with pytest.raises(RuntimeError, match="dtype"):
        ops.kv4_read(cache, torch.zeros(1, dtype=torch.int64), 64, torch.float32)
    with pytest.raises(RuntimeError, match="slots"):
        ops.kv4_read(cache, torch.zeros(1), 64, torch.float16)
    with pytest.raises(ValueError, match="slots"):
        ops.kv4_read(cache, torch.zeros(1, 1, dtype=torch.int64), 64, torch.float16)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        ops.kv4_read(cache, torch.zeros(1, dtype=torch.int64), 64, torch.float16)


def test_oracle_reads_what_it_stores():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 20, 3, 64, generator=g)
    cache = torch.zeros(3, 3, 16 * 72, dtype=torch.uint8)
    slots = torch.randperm(48, generator=g)[:20]
    orc.store(cache, 64, slots, x[0], x[1])
    for got, want in zip(orc.values(cache, 64, slots), x):
        codes, scale, least = orc.quantise(want)
        assert torch.equal(got, least.double()[..., None] + codes.double() * scale.double()[..., None])


def test_oracle_attention_is_torchs():
    g = torch.Generator().manual_seed(1)
    n, d = 37, 64
    cache = torch.zeros(3, 1, 16 * 72, dtype=torch.uint8)
    tables = torch.tensor([[2, 0, 1]], dtype=torch.int32)
    j = torch.arange(n)
    slots = tables[0].long()[j // 16] * 16 + j % 16
    orc.store(cache, d, slots, torch.randn(n, 1, d, generator=g), torch.randn(n, 1, d, generator=g))
    q = torch.randn(n, 2, d, generator=g).half()
    got, _ = orc.attend(q, cache, tables, torch.tensor([n]), torch.tensor([0, n]), 0.1, 0, True)
    k, v, _ = orc.values(cache, d, slots)
    want = torch.nn.functional.scaled_dot_product_attention(q.double().transpose(0, 1), k.transpose(0, 1).expand(2, n, d),
                                                            v.transpose(0, 1).expand(2, n, d), is_causal=True, scale=0.1)
    assert torch.allclose(got, want.transpose(0, 1), rtol=1e-12, atol=1e-12)


def test_more_than_a_grid_holds_is_refused(lib):
    assert append(lib, tokens=1 << 26) == -8
    assert attend(lib, tokens=1 << 28, heads=16) == -8


@pytest.mark.parametrize("change,text", [
    (dict(query=torch.zeros(3, 0, 128, dtype=torch.float16)), "0 heads"),  # (its keys would not be stored)
    (dict(cos_sin=torch.zeros(0, 128)), "no positions"),
])
def test_append_operator_refuses_nothing_to_rotate_by(ops, change, text):
    with pytest.raises(ValueError, match=text):
        ops.rope_append_kv4(**append_args(**change))


def test_slots_of_positions():
    """Rows of a padded batch (position -1), positions past the table and pages without a block have no slot."""
    from vllm_quick_amd.layers.kv4_attention import slots_of
    tables = torch.tensor([[5, 2], [7, -1], [0, 0]], dtype=torch.int32)
    got = slots_of(tables, torch.tensor([17, 3, -1]), 16)
    assert got.tolist() == [2 * 16 + 1, 7 * 16 + 3, -1]
    got = slots_of(tables, torch.tensor([0, 31, 32, 15, 16, 10**9]), 16, torch.tensor([0, 0, 0, 1, 1, 2]))
    assert got.tolist() == [80, 47, -1, 127, -1, -1]
    assert slots_of(tables[:, :0], torch.tensor([0, 1, -1]), 16).tolist() == [-1, -1, -1]


def test_a_promise_of_more_rows_than_there_are(lib):
    """max_query_len is an upper bound: one far above the rows of the batch asks for what the rows themselves do."""
    for tokens, seqs, heads, kv, most in ((4, 2, 128, 1, 65536), (600, 1, 128, 1, 65536), (5, 2, 64, 1, 100000), (7, 3, 65535, 1, 3000)):
        want = lib.serving_attend_kv4_workspace_bytes(tokens, seqs, heads, kv, 128, tokens, most, 0)
        for rows in (tokens + 1, 32768, 1 << 30, (1 << 30) + 1, 0x7fffffff):
            assert lib.serving_attend_kv4_workspace_bytes(tokens, seqs, heads, kv, 128, rows, most, 0) == want, (tokens, rows)
            if want:  # (refused for that alone)
                assert attend(lib, tokens=tokens, seqs=seqs, heads=heads, kv=kv, most=most, most_q=rows, ws=None) == -9
    assert lib.serving_attend_kv4_workspace_bytes(0x7fffffff, 0x7fffffff, 65535, 1, 128, 0x7fffffff, 1 << 27, 0) == 0
    assert attend(lib, tokens=0x7fffffff, seqs=0x7fffffff, heads=65535, kv=1, most_q=0x7fffffff, most=1 << 27) == -8


def test_awq_operators_do_without_the_torch_extension():
    """Where only libw4a16.so is built the AWQ operators import as they are, and the others say what is missing."""
    code = """
import sys
sys.modules["vllm_quick_amd._C_native"] = None  # its import fails
import torch
from vllm_quick_amd import ops
from vllm_quick_amd.layers.linear import ColumnParallelLinear
assert callable(ops.awq_gemm) and callable(ops.awq_dequantize)
cache = ops.kv4_cache(2, 16, 2, 64, torch.device("cpu"))
try:
    ops.kv4_read(cache, torch.zeros(1, dtype=torch.int64), 64, torch.float16)
except ImportError as e:
    assert "_C_native" in str(e)
else:
    raise AssertionError
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-1500:]
