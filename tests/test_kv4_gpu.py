"""The 4-bit paged cache on the GPU: rotation and appending, reading back, attention, alone and one after the other,
against the oracle (fp32 by the format's definition for stored bytes, 64 bits for everything else).  Tolerances come
from the oracle, which counts the roundings (oracle/serving_oracle.py)."""
import pytest
import torch

from oracle import serving_oracle as orc

pytestmark = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops():
    from vllm_quick_amd import ops
    return ops


def table(positions, rotary):
    inv = 10000.0**(-torch.arange(0, rotary, 2, dtype=torch.float64) / max(rotary, 1))
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * inv
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def inputs(t, heads, kv, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(t, heads + 2 * kv, d, generator=g) * torch.exp(0.7 * torch.randn(heads + 2 * kv, d, generator=g))
    return [x.to(dtype) for x in qkv.split([heads, kv, kv], 1)]


def append_case(t, heads, kv, d, p, rotary, interleaved, dtype, seed, blocks=None, positions=257):
    q, k, v = inputs(t, heads, kv, d, dtype, seed)
    g = torch.Generator().manual_seed(seed + 1)
    blocks = blocks or (t + p - 1) // p + 3
    pos = torch.randint(0, positions, (t, ), generator=g)
    slots = torch.randperm(blocks * p, generator=g)[:t]
    cache = torch.randint(0, 256, (blocks, kv, p * (d + 8)), generator=g, dtype=torch.uint8)  # what was there stays
    return q, k, v, pos, slots, cache, table(positions, rotary)


def check_append(ops, cuda, case, interleaved, d):
    q, k, v, pos, slots, cache, cs = case
    got_cache = cache.to(cuda)
    out = ops.rope_append_kv4(pos.to(cuda), q.to(cuda), k.to(cuda), v.to(cuda), cs.to(cuda), got_cache, slots.to(cuda), interleaved)
    want_cache = cache.clone()
    orc.store(want_cache, d, slots, orc.rotate32(k, cs, pos, interleaved), v.float())
    got, want = got_cache.cpu(), want_cache
    nan = lambda c: torch.isnan(c.view(torch.float16))  # noqa: E731  (a NaN's bits are not defined)
    pairs = nan(got) & nan(want)
    assert torch.equal(torch.where(pairs, 0, got.view(torch.int16)), torch.where(pairs, 0, want.view(torch.int16)))
    x, size = orc.rotate64(q, cs, pos, interleaved)
    tol = torch.finfo(q.dtype).eps / 2 * x.abs() + 2.0**-22 * size + 2.0**-25  # one rounding; three in fp32 before it
    assert out.dtype == q.dtype and out.shape == q.shape
    assert ((out.cpu().double() - x).abs() <= tol).all()
    return got_cache


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("t,heads,kv,d,p,rotary,interleaved", [
    (1, 1, 1, 128, 16, 128, False),
    (1, 32, 32, 128, 16, 128, False),
    (3, 7, 1, 64, 16, 64, False),
    (5, 12, 4, 64, 32, 32, True),
    (17, 8, 2, 128, 48, 96, False),
    (33, 4, 4, 128, 64, 16, True),
    (65, 3, 3, 64, 4096, 48, False),
    (19, 5, 5, 128, 16, 0, False),
    (511, 4, 2, 128, 16, 128, False),
    (512, 4, 2, 128, 16, 128, True),
    (77, 1, 1, 64, 16, 64, False),  # sixteen tokens a workgroup
    (13, 70, 7, 64, 16, 64, True),  # several passes over a token's heads
    (1000, 6, 3, 64, 32, 64, False),
])
def test_append(ops, cuda, t, heads, kv, d, p, rotary, interleaved, dtype):
    check_append(ops, cuda, append_case(t, heads, kv, d, p, rotary, interleaved, TYPES[dtype], seed=t), interleaved, d)


def test_append_values_stand_where_they_should(ops, cuda):
    """In 64 bits: a stored element is within half a step of what it was, but for the roundings of the two parameters."""
    case = append_case(40, 4, 2, 128, 16, 128, False, torch.bfloat16, 3)
    q, k, v, pos, slots, cache, cs = case
    dev = cache.to(cuda)
    ops.rope_append_kv4(pos.to(cuda), q.to(cuda), k.to(cuda), v.to(cuda), cs.to(cuda), dev, slots.to(cuda))
    kk, vv, _ = orc.values(dev.cpu(), 128, slots)
    for got, x in ((kk, orc.rotate64(k, cs, pos, False)[0]), (vv, v.double())):
        least, most = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
        step = (most - least) / 15
        # scale off by half a step of fp16 (and by least's): 15 of it at the top; least off by half a step of fp16
        bound = step * 0.5 + (16 * step + 2 * least.abs()) * 2.0**-11 + 2.0**-20 * x.abs()
        assert ((got - x).abs() <= bound).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_append_values_that_no_scale_holds(ops, cuda, dtype):
    """Constant heads, heads of tiny values, infinities, NaN, and what passes fp16's range."""
    d, p = 64, 16
    case = list(append_case(12, 2, 2, d, p, 0, False, TYPES[dtype], 5))
    k, v = case[1], case[2]
    k[0], v[0] = 0.0, -1.25
    k[1] *= 2.0**-20
    v[1] *= 2.0**-14
    k[2, 0, 5], v[2, 1, 63] = float("nan"), float("nan")
    k[3, 1, 0], v[3, 0, 7] = float("inf"), -float("inf")
    k[4, 0, 9], v[4, 1, 9] = 60000.0, -60000.0
    if dtype == "bf16":
        k[5, 0, 1], v[5, 1, 2], v[5, 0, 3] = -1e20, 1e20, 1e5
    case[6] = torch.zeros(3, 0)
    dev = check_append(ops, cuda, case, False, d)
    kk, vv, _ = orc.values(dev.cpu(), d, case[4])
    assert (kk[0] == 0).all() and (vv[0] == -1.25).all()
    assert torch.isnan(kk[2, 0]).all() and not torch.isnan(kk[2, 1]).any() and torch.isnan(vv[3, 0]).all()
    got_k, got_v = ops.kv4_read(dev, case[4].to(cuda), d, TYPES[dtype])
    assert torch.equal(torch.isnan(got_k.cpu()), torch.isnan(kk.to(TYPES[dtype])))


def test_append_leaves_padded_rows_and_every_other_slot_alone(ops, cuda):
    d, p, t = 128, 16, 20
    case = list(append_case(t, 4, 2, d, p, 128, False, torch.float16, 9))
    case[4] = case[4].clone()
    case[4][[3, 7, 19]] = torch.tensor([-1, 10**12, case[5].shape[0] * p])
    check_append(ops, cuda, case, False, d)
    k, v = ops.kv4_read(case[5].to(cuda), case[4].to(cuda), d, torch.float16)
    assert (k[[3, 7, 19]] == 0).all() and (v[[3, 7, 19]] == 0).all()


def test_append_position_outside_the_table_is_nan(ops, cuda):
    d = 128
    q, k, v, pos, slots, cache, cs = append_case(4, 2, 2, d, 16, 64, False, torch.float16, 11)
    pos = torch.tensor([0, -1, 257, 256])
    dev = cache.to(cuda)
    out = ops.rope_append_kv4(pos.to(cuda), q.to(cuda), k.to(cuda), v.to(cuda), cs.to(cuda), dev, slots.to(cuda)).cpu()
    assert torch.isnan(out[1:3, :, :64]).all() and torch.equal(out[1:3, :, 64:], q[1:3, :, 64:])
    assert not torch.isnan(out[[0, 3]]).any()
    kk, vv, _ = orc.values(dev.cpu(), d, slots)
    assert torch.isnan(kk[1:3]).all() and not torch.isnan(kk[[0, 3]]).any() and not torch.isnan(vv).any()


def test_append_strides(ops, cuda):
    """Views of one qkv tensor, transposed heads, addresses off the 16-byte grid, a table that is a view."""
    d, p, t, heads, kv = 64, 16, 21, 6, 2
    q, k, v, pos, slots, cache, cs = append_case(t, heads, kv, d, p, 32, False, torch.bfloat16, 13)
    qkv = torch.cat([q.reshape(t, -1), k.reshape(t, -1), v.reshape(t, -1)], 1).to(cuda)
    a, b, c = (x.view(t, -1, d) for x in qkv.split([heads * d, kv * d, kv * d], 1))
    odd = torch.empty(t * heads * d + 1, dtype=q.dtype, device=cuda)[1:].view(t, heads, d)
    odd.copy_(q)
    turned = torch.empty(kv, t, d, dtype=q.dtype, device=cuda).transpose(0, 1)
    turned.copy_(k)
    wide = torch.empty(t, kv, 2 * d, dtype=q.dtype, device=cuda)
    wide[..., ::2] = v.to(cuda)
    tab = torch.empty(cs.shape[0], 37, device=cuda)[:, 5:37]
    tab.copy_(cs)
    pos2 = torch.stack([pos, pos], 1).to(cuda)[:, 0]
    results = []
    for args in ((a, b, c, cs.to(cuda), pos.to(cuda)), (odd, turned, wide[..., ::2], tab, pos2)):
        dev = cache.to(cuda)
        out = ops.rope_append_kv4(args[4], args[0], args[1], args[2], args[3], dev, slots.to(cuda))
        results.append((out, dev))
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    check_append(ops, cuda, (q, k, v, pos, slots, cache, cs), False, d)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("d,p,kv,rows", [(64, 16, 3, 1), (128, 32, 2, 77), (128, 16, 1, 1000)])
def test_read(ops, cuda, d, p, kv, rows, dtype):
    case = append_case(50, kv, kv, d, p, 0, False, TYPES[dtype], 17)
    dev = check_append(ops, cuda, case[:6] + (torch.zeros(1, 0), ), False, d)
    g = torch.Generator().manual_seed(1)
    slots = case[4][torch.randint(0, 50, (rows, ), generator=g)]  # the same slot as often as you like
    k, v = ops.kv4_read(dev, slots.to(cuda), d, TYPES[dtype])
    kk, vv, _ = orc.values(dev.cpu(), d, slots)
    for got, want in ((k, kk), (v, vv)):
        # fp32 product and sum, one rounding each, then the type's
        tol = torch.finfo(TYPES[dtype]).eps / 2 * want.abs() * (1 + 2.0**-20) + 2.0**-23 * 16 * want.abs().amax(-1, keepdim=True) + 2.0**-25
        assert ((got.cpu().double() - want).abs() <= tol).all()


# ---------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------
def filled_cache(lens, kv, d, p, seed, gain=1.0, spare=2):
    """A cache with random values in every slot of the sequences and rubbish (NaN parameters too) everywhere else."""
    g = torch.Generator().manual_seed(seed)
    used = [max(1, -(-max(n, 1) // p)) for n in lens]
    blocks = sum(used) + spare
    cache = torch.randint(0, 256, (blocks, kv, p * (d + 8)), generator=g, dtype=torch.uint8)
    cache.view(torch.float16)[:, :, p * d // 2:] = float("nan")
    order = torch.randperm(blocks, generator=g).to(torch.int32)
    wide = max(used)
    tables = torch.full((len(lens), wide), -7, dtype=torch.int32)  # behind a sequence's blocks stands no block
    at = 0
    for b, u in enumerate(used):
        tables[b, :u] = order[at:at + u]
        at += u
    for b, n in enumerate(lens):
        if n:
            j = torch.arange(n)
            slots = tables[b].long()[j // p] * p + j % p
            x = torch.randn(2, n, kv, d, generator=g) * torch.exp(0.7 * torch.randn(2, 1, kv, d, generator=g)) * gain
            x[1] += 0.3 * torch.randn(1, kv, d, generator=g)
            orc.store(cache, d, slots, x[0], x[1])
    return cache, tables


def attend_case(lens, counts, heads, kv, d, p, dtype, seed, gain=1.0):
    cache, tables = filled_cache(lens, kv, d, p, seed, gain)
    g = torch.Generator().manual_seed(seed + 1)
    start = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
    query = (torch.randn(int(start[-1]), heads, d, generator=g) * 1.2).to(dtype)
    return query, cache, tables, torch.tensor(lens, dtype=torch.int32), start


def check_attend(ops, cuda, case, window=0, scale=None, max_seq_len=None, ragged=True, out=None):
    query, cache, tables, lens, start = case
    scale = query.shape[2]**-0.5 if scale is None else scale
    counts = (start[1:] - start[:-1]).tolist()
    got = ops.paged_attention_kv4(query.to(cuda), cache.to(cuda), tables.to(cuda), lens.to(cuda), scale,
                                  max_seq_len or max(1, int(lens.max())), query_start=start.to(cuda) if ragged else None,
                                  max_query_len=max(1, max(counts)) if ragged else 1, window=window, out=out)
    want, tol = orc.attend(query, cache, tables, lens, start, scale, window, query.dtype == torch.float16)
    assert got.dtype == query.dtype and got.shape == query.shape
    mine = ~torch.isnan(want)
    bad = (got.cpu().double() - want).abs()[mine] > tol[mine]
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((got.cpu().double() - want).abs() / tol)[mine].max())} of what is allowed"
    assert not torch.isnan(got.cpu()[mine]).any()
    return got


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("lens,heads,kv,d,p", [
    ([1], 1, 1, 128, 16),
    ([1, 2, 15, 16, 17, 31, 32, 33], 2, 2, 64, 16),
    ([129], 4, 4, 128, 16),
    ([0, 5, 0, 64, 100], 6, 2, 128, 32),     # sequences without a token
    ([700, 3, 511], 7, 1, 64, 48),           # blocks whose tokens are no power of two
    ([300, 1], 16, 1, 128, 64),
    ([40, 77], 34, 2, 64, 16),               # more heads to a kv head than a tile's columns
    ([70, 20], 80, 1, 128, 16),
    ([2100], 8, 2, 128, 128),                # several pieces a sequence
    ([1025, 4, 600], 5, 5, 64, 4096),
])
def test_attend_one_token(ops, cuda, lens, heads, kv, d, p, dtype):
    check_attend(ops, cuda, attend_case(lens, [1] * len(lens), heads, kv, d, p, TYPES[dtype], seed=len(lens) + d), ragged=False)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("lens,counts,heads,kv,d,p", [
    ([5, 130, 64], [5, 3, 1], 4, 2, 128, 16),
    ([20, 200], [0, 7], 8, 1, 64, 32),                  # a sequence without a query
    ([3, 90], [8, 2], 2, 2, 128, 16),                   # more queries than tokens: rows that see nothing
    ([1300, 90], [5, 5], 14, 2, 64, 16),
    ([100, 37], [100, 37], 2, 2, 128, 16),              # whole prompts
    ([333], [129], 6, 2, 64, 48),
    ([400, 1, 257], [130, 1, 257], 8, 1, 128, 32),
    ([65], [65], 3, 3, 64, 16),
])
@pytest.mark.parametrize("window", [0, 1, 40])
def test_attend_several_tokens(ops, cuda, lens, counts, heads, kv, d, p, dtype, window):
    check_attend(ops, cuda, attend_case(lens, counts, heads, kv, d, p, TYPES[dtype], seed=sum(lens)), window=window)


@pytest.mark.parametrize("window", [1, 16, 33, 500, 5000])
def test_attend_window_of_one_token(ops, cuda, window):
    check_attend(ops, cuda, attend_case([1, 33, 700, 1400], [1] * 4, 6, 2, 128, 16, torch.float16, 3), window=window, ragged=False)


@pytest.mark.parametrize("gain", [2.0**-12, 2.0**-5, 300.0])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_attend_sizes_of_values(ops, cuda, gain, dtype):
    """Values far from 1 (their scales subnormal in fp16 at the small end); the queries keep the scores in range."""
    case = attend_case([400, 31], [1, 1], 4, 2, 128, 16, TYPES[dtype], 7, gain)
    check_attend(ops, cuda, case, scale=128**-0.5 / gain, ragged=False)


@pytest.mark.parametrize("scale", [0.0, -0.1, 2.0, 30.0])
@pytest.mark.parametrize("counts", [[1, 1], [9, 40]])
def test_attend_scales(ops, cuda, scale, counts):
    check_attend(ops, cuda, attend_case([500, 60], counts, 4, 2, 64, 16, torch.float16, 21), scale=scale)


@pytest.mark.parametrize("size", [2.0**-20, 1e-3, 500.0])
def test_attend_sizes_of_queries(ops, cuda, size):
    query, *rest = attend_case([90, 300], [2, 50], 4, 2, 128, 16, torch.float16, 23)
    query = query * size
    query[:, 0, ::3] = 0
    query[1] = 0
    check_attend(ops, cuda, (query, *rest), scale=128**-0.5 / size)


def test_attend_does_not_see_what_stands_behind(ops, cuda):
    """Stored NaN and values of 6e4 at tokens that a row must not see change nothing of that row, bit for bit."""
    d, p = 128, 16
    for counts in ([1, 4], [40, 70]):
        query, cache, tables, lens, start = attend_case([100, 90], counts, 4, 2, d, p, torch.float16, 31)
        args = lambda c, l: (query.to(cuda), c.to(cuda), tables.to(cuda), l.to(cuda), 0.1, 128)  # noqa: E731
        kw = dict(query_start=start.to(cuda), max_query_len=max(counts))
        base = ops.paged_attention_kv4(*args(cache, lens), **kw).cpu()
        n = int(lens[1])
        slot = (tables[1].long()[(n - 1) // p] * p + (n - 1) % p).view(1)
        for x in (float("nan"), 60000.0):
            other = cache.clone()
            orc.store(other, d, slot, torch.full((1, 2, d), x), torch.full((1, 2, d), x))
            got = ops.paged_attention_kv4(*args(other, lens), **kw).cpu()
            last = int(start[2]) - 1
            assert torch.equal(got[:last], base[:last])
            assert torch.isnan(got[last]).all() or x == x


def test_attend_blocks_that_do_not_exist_are_nan(ops, cuda):
    query, cache, tables, lens, start = attend_case([100, 90], [1, 1], 4, 2, 128, 16, torch.float16, 37)
    for bad in (-1, cache.shape[0], 2**31 - 1):
        wrong = tables.clone()
        wrong[1, 2] = bad
        got = ops.paged_attention_kv4(query.to(cuda), cache.to(cuda), wrong.to(cuda), lens.to(cuda), 0.1, 128).cpu()
        assert torch.isnan(got[1]).all() and not torch.isnan(got[0]).any()


def test_attend_rows_of_no_sequence_and_rows_past_the_promise(ops, cuda):
    query, cache, tables, lens, start = attend_case([700, 90], [3, 2], 4, 2, 64, 16, torch.bfloat16, 41)
    more = torch.cat([query, query[:2]])
    out = torch.full(more.shape, 7.0, dtype=more.dtype, device=cuda)
    for most in (3, 2):
        out.fill_(7.0)
        got = ops.paged_attention_kv4(more.to(cuda), cache.to(cuda), tables.to(cuda), lens.to(cuda), 0.125, 700,
                                      query_start=start.to(cuda), max_query_len=most, out=out)
        assert got.data_ptr() == out.data_ptr()
        assert (out[5:] == 7.0).all()
        want, tol = orc.attend(query, cache, tables, lens, start, 0.125, 0, False)
        off = (out[:5].cpu().double() - want).abs() <= tol
        assert off[[0, 1, 3, 4]].all()
        assert off[2].all() if most == 3 else torch.isnan(out[2]).all()


def test_attend_lengths_that_the_launch_was_not_sized_for(ops, cuda):
    """max_seq_len sizes the launch alone: longer sequences are read whole, as a captured step's are later on."""
    case = attend_case([1500, 40], [1, 1], 4, 2, 128, 16, torch.float16, 43)
    for most in (1, 64, 600, 1 << 20):
        check_attend(ops, cuda, case, max_seq_len=most, ragged=False)


def test_attend_strides(ops, cuda):
    query, cache, tables, lens, start = attend_case([300, 45], [1, 1], 6, 2, 64, 16, torch.float16, 47)
    args = (cache.to(cuda), tables.to(cuda), lens.to(cuda), 0.125, 300)
    base = ops.paged_attention_kv4(query.to(cuda), *args)
    odd = torch.empty(query.numel() + 1, dtype=query.dtype, device=cuda)[1:].view(query.shape)
    odd.copy_(query)
    turned = torch.empty(6, 2, 64, dtype=query.dtype, device=cuda).transpose(0, 1)
    turned.copy_(query)
    wide = torch.full((2, tables.shape[1] + 5), 99, dtype=torch.int32, device=cuda)
    wide[:, :tables.shape[1]] = tables.to(cuda)
    for q, t in ((odd, wide[:, :tables.shape[1]]), (turned, tables.to(cuda).t().contiguous().t())):
        assert torch.equal(ops.paged_attention_kv4(q, args[0], t, *args[2:]), base)


def test_attend_same_call_same_bits(ops, cuda):
    query, cache, tables, lens, start = attend_case([2600, 900], [1, 1], 8, 2, 128, 16, torch.float16, 53)
    args = [x.to(cuda) for x in (query, cache, tables, lens)]
    first = ops.paged_attention_kv4(*args, 0.1, 2600)
    for _ in range(3):
        assert torch.equal(ops.paged_attention_kv4(*args, 0.1, 2600), first)


def test_long_cache_passes_32_bits(ops, cuda):
    """Blocks whose bytes lie beyond 4 GiB of the cache's start are appended to, read and attended to."""
    d, p, kv = 128, 64, 8
    blocks = (9 << 29) // (kv * p * (d + 8)) + 1  # 4.5 GiB
    cache = torch.empty(blocks, kv, p * (d + 8), dtype=torch.uint8, device=cuda)
    n = 100
    tables = torch.tensor([[blocks - 1, 0]], dtype=torch.int32)
    j = torch.arange(n)
    slots = tables[0].long()[j // p] * p + j % p
    q, k, v = inputs(n, kv, kv, d, torch.float16, 3)
    cs = table(n, 128)
    rotated = ops.rope_append_kv4(j.to(cuda), q.to(cuda), k.to(cuda), v.to(cuda), cs.to(cuda), cache, slots.to(cuda))
    small = torch.zeros(2, kv, p * (d + 8), dtype=torch.uint8)
    orc.store(small, d, j, orc.rotate32(k, cs, j, False), v.float())
    got = ops.kv4_read(cache, slots.to(cuda), d, torch.float16)
    want = ops.kv4_read(small.to(cuda), j.to(cuda), d, torch.float16)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    lens = torch.tensor([n], dtype=torch.int32, device=cuda)
    a = ops.paged_attention_kv4(rotated[-1:], cache, tables.to(cuda), lens, 0.09, n)
    b = ops.paged_attention_kv4(rotated[-1:], small.to(cuda), torch.tensor([[0, 1]], dtype=torch.int32, device=cuda), lens, 0.09, n)
    assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------------------------
def test_a_prompt_then_tokens_one_by_one(ops, cuda):
    """A prompt in two chunks, then single tokens, two sequences at once: every step against the oracle on what the
    cache holds; the same tokens in one chunk leave the same cache."""
    d, p, heads, kv, dtype = 128, 16, 8, 2, torch.bfloat16
    total = [45, 23]
    q, k, v = inputs(sum(total), heads, kv, d, dtype, 61)
    cs = table(64, 128)
    tables = torch.tensor([[5, 1, 4], [2, 0, 0]], dtype=torch.int32)
    base = [0, total[0]]

    def slots_of(b, lo, hi):
        j = torch.arange(lo, hi)
        return tables[b].long()[j // p] * p + j % p

    cache = torch.zeros(6, kv, p * (d + 8), dtype=torch.uint8, device=cuda)
    done = [0, 0]
    for step in [(20, 9), (20, 10), (1, 1), (1, 1), (1, 1), (1, 1), (1, 0)]:
        rows, pos, slots, start = [], [], [], [0]
        for b, m in enumerate(step):
            rows.append(torch.arange(base[b] + done[b], base[b] + done[b] + m))
            pos.append(torch.arange(done[b], done[b] + m))
            slots.append(slots_of(b, done[b], done[b] + m))
            done[b] += m
            start.append(start[-1] + m)
        rows, pos, slots = torch.cat(rows), torch.cat(pos), torch.cat(slots)
        turned = ops.rope_append_kv4(pos.to(cuda), q[rows].to(cuda), k[rows].to(cuda), v[rows].to(cuda), cs.to(cuda), cache, slots.to(cuda))
        lens = torch.tensor(done, dtype=torch.int32)
        check_attend(ops, cuda, (turned.cpu(), cache.cpu(), tables, lens, torch.tensor(start, dtype=torch.int32)))
    whole = torch.zeros_like(cache)
    pos = torch.cat([torch.arange(n) for n in done])
    slots = torch.cat([slots_of(b, 0, n) for b, n in enumerate(done)])
    rows = torch.cat([torch.arange(base[b], base[b] + n) for b, n in enumerate(done)])
    ops.rope_append_kv4(pos.to(cuda), q[rows].to(cuda), k[rows].to(cuda), v[rows].to(cuda), cs.to(cuda), whole, slots.to(cuda))
    assert torch.equal(whole, cache)


def test_captured_steps_replay(ops, cuda):
    """A captured decode step (append, attention over pieces, scoring) replayed with new tokens and lengths, eager work
    between; a second graph of the same calls lives beside it."""
    d, p, heads, kv, b, vocab = 128, 16, 8, 2, 3, 1500
    g = torch.Generator(device=cuda).manual_seed(5)
    lens0 = [600, 37, 1000]
    cache_cpu, tables = filled_cache([n + 8 for n in lens0], kv, d, p, 71)
    fresh = cache_cpu.to(cuda)
    cs = table(2048, 128).to(cuda)
    tables = tables.to(cuda)
    w = torch.randn(heads * d, vocab, generator=g, device=cuda, dtype=torch.float16) * 0.02

    def make():
        st = dict(cache=fresh.clone(), qkv=torch.zeros(b, heads + 2 * kv, d, dtype=torch.float16, device=cuda),
                  lens=torch.tensor(lens0, dtype=torch.int32, device=cuda), tok=torch.zeros(b, dtype=torch.int64, device=cuda))
        return st

    def step(st):
        at = st["lens"].long() - 1
        slots = tables.long().gather(1, (at // p)[:, None])[:, 0] * p + at % p
        q, k, v = st["qkv"].split([heads, kv, kv], 1)
        q = ops.rope_append_kv4(at, q, k, v, cs, st["cache"], slots)
        o = ops.paged_attention_kv4(q, st["cache"], tables, st["lens"], 0.09, 1024)
        return o, ops.token_logprobs(o.view(b, -1) @ w, st["tok"], 4)

    graphs = []
    side = torch.cuda.Stream()
    for _ in range(2):
        st = make()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(st)
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = step(st)
        graphs.append((graph, st, out))
    eager = make()
    for _, st, _ in graphs:
        st["cache"].copy_(fresh)
    for i in range(5):
        x = torch.randn(b, heads + 2 * kv, d, generator=g, device=cuda).half()
        tok = torch.randint(0, vocab, (b, ), generator=g, device=cuda)
        for st in [eager] + [s for _, s, _ in graphs]:
            st["qkv"].copy_(x)
            st["tok"].copy_(tok)
            st["lens"].copy_(torch.tensor([n + 1 + i for n in lens0], dtype=torch.int32))
        want = step(eager)
        torch.cuda.synchronize()
        for graph, st, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, st, out in graphs:
            assert torch.equal(out[0], want[0]) and torch.equal(st["cache"], eager["cache"])
            for x1, y1 in zip(out[1], want[1]):
                assert torch.equal(x1, y1)


def test_two_streams_at_once(ops, cuda):
    cases = [attend_case([1500, 40], [1, 1], 4, 2, 128, 16, torch.float16, 80 + i) for i in range(2)]
    args = [[x.to(cuda) for x in c[:4]] for c in cases]
    want = [ops.paged_attention_kv4(*a, 0.09, 1500) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.paged_attention_kv4(*args[i], 0.09, 1500))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_empty_calls(ops, cuda):
    d, p = 64, 16
    cache = ops.kv4_cache(2, p, 2, d, cuda)
    assert (cache == 0).all() and cache.shape == (2, 2, p * (d + 8))
    none = torch.zeros(0, dtype=torch.int64, device=cuda)
    out = ops.rope_append_kv4(none, torch.zeros(0, 4, d, dtype=torch.float16, device=cuda), torch.zeros(0, 2, d, dtype=torch.float16, device=cuda),
                              torch.zeros(0, 2, d, dtype=torch.float16, device=cuda), torch.zeros(3, 32, device=cuda), cache, none)
    assert out.shape == (0, 4, d)
    k, v = ops.kv4_read(cache, none, d, torch.bfloat16)
    assert k.shape == (0, 2, d) and v.dtype == torch.bfloat16
    out = ops.paged_attention_kv4(torch.zeros(0, 4, d, dtype=torch.float16, device=cuda), cache,
                                  torch.zeros(0, 3, dtype=torch.int32, device=cuda), torch.zeros(0, dtype=torch.int32, device=cuda), 1.0, 5)
    assert out.shape == (0, 4, d)
