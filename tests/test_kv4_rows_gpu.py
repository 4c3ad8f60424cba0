"""Attention over the 4-bit cache where a sequence has many columns (queries x heads of a kv head): batches large enough
that each wave takes columns of its own, and those of few or uneven rows, where waves share the keys."""
import pytest
import torch

from oracle import serving_oracle as orc
from test_kv4_gpu import TYPES, attend_case, check_attend

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from vllm_quick_amd import ops
    return ops


def in_a_large_batch(case, tiles):
    """The case with rows of no sequence behind it, so many that the batch counts as one that fills the chip."""
    query, *rest = case
    rows = max(0, -(-tiles * 32 // query.shape[1]) - query.shape[0])
    return torch.cat([query, torch.ones(rows, *query.shape[1:], dtype=query.dtype)]), *rest


def check_in_a_large_batch(ops, cuda, case, tiles=2048, **kw):
    case = in_a_large_batch(case, tiles)
    out = torch.full(case[0].shape, 7.0, dtype=case[0].dtype, device=cuda)
    got = check_attend(ops, cuda, case, out=out, **kw)
    assert (got[int(case[4][-1]):] == 7.0).all()
    return got


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("lens,counts,heads,kv,d,p", [
    ([65], [65], 3, 3, 64, 16),
    ([100, 37], [100, 37], 2, 2, 128, 16),
    ([333], [129], 6, 2, 64, 48),                       # 387 columns: a workgroup's last wave has a few
    ([400, 1, 257], [130, 1, 257], 8, 1, 128, 32),
    ([3, 90], [40, 9], 8, 4, 128, 16),                  # more queries than tokens: rows that see nothing
    ([0, 200, 50], [33, 40, 0], 4, 2, 64, 16),
    ([90, 17], [1, 1], 130, 2, 128, 16),                # single tokens of many heads
    ([1500], [70], 2, 2, 64, 16),                       # set aside in between
])
@pytest.mark.parametrize("window", [0, 1, 40])
def test_columns_of_their_own(ops, cuda, lens, counts, heads, kv, d, p, dtype, window):
    check_in_a_large_batch(ops, cuda, attend_case(lens, counts, heads, kv, d, p, TYPES[dtype], seed=sum(lens)), window=window)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("window", [0, 1300])
def test_columns_of_their_own_over_long_sequences(ops, cuda, dtype, window):
    check_in_a_large_batch(ops, cuda, attend_case([2500, 2200], [40, 33], 4, 2, 128, 64, TYPES[dtype], 61), 4096, window=window)


def test_columns_of_their_own_of_many_sequences(ops, cuda):
    """More sequences than are ordered by their length, and as many as are."""
    g = torch.Generator().manual_seed(5)
    for seqs in (64, 70):
        counts = torch.randint(0, 34, (seqs, ), generator=g).tolist()
        lens = [c + int(x) for c, x in zip(counts, torch.randint(0, 50, (seqs, ), generator=g))]
        counts[3] = 33
        check_in_a_large_batch(ops, cuda, attend_case(lens, counts, 2, 1, 64, 16, torch.float16, seqs))


def test_columns_of_their_own_do_not_see_what_stands_behind(ops, cuda):
    d, p = 128, 16
    query, cache, tables, lens, start = in_a_large_batch(attend_case([100, 90], [40, 70], 4, 2, d, p, torch.float16, 31), 2048)
    run = lambda c, t: ops.paged_attention_kv4(query.to(cuda), c.to(cuda), t.to(cuda), lens.to(cuda), 0.1, 128,  # noqa: E731
                                               query_start=start.to(cuda), max_query_len=70).cpu()[:110]
    base = run(cache, tables)
    slot = (tables[1].long()[89 // p] * p + 89 % p).view(1)
    for x in (float("nan"), 60000.0):
        other = cache.clone()
        orc.store(other, d, slot, torch.full((1, 2, d), x), torch.full((1, 2, d), x))
        got = run(other, tables)
        assert torch.equal(got[:109], base[:109]) and not torch.isnan(base[:109]).any()
        assert torch.isnan(got[109]).all() or x == x
    for bad in (-1, cache.shape[0], 2**31 - 1):  # a block of its last 26 tokens that does not exist
        wrong = tables.clone()
        wrong[1, 4] = bad
        got = run(cache, wrong)
        seen = 40 + 70 - 26
        assert torch.equal(got[:seen], base[:seen]) and torch.isnan(got[seen:]).all()


@pytest.mark.parametrize("large", [False, True])
def test_rows_past_the_promise_among_many(ops, cuda, large):
    case = attend_case([300, 90], [43, 20], 4, 1, 64, 16, torch.bfloat16, 41)
    query, cache, tables, lens, start = in_a_large_batch(case, 2048) if large else case
    out = torch.full(query.shape, 7.0, dtype=query.dtype, device=cuda)
    ops.paged_attention_kv4(query.to(cuda), cache.to(cuda), tables.to(cuda), lens.to(cuda), 0.125, 300,
                            query_start=start.to(cuda), max_query_len=30, out=out)
    want, tol = orc.attend(query, cache, tables, lens, start, 0.125, 0, False)
    got = out.cpu().double()
    kept = list(range(30)) + list(range(43, 63))
    assert ((got - want).abs() <= tol)[kept].all() and torch.isnan(got[30:43]).all() and (got[63:] == 7.0).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("lens,counts,heads,kv,d,p,window", [
    ([5000], [1], 128, 1, 128, 64, 0),                  # one token of many heads, in pieces
    ([3000, 700], [50, 40], 4, 2, 64, 16, 0),           # rows of a prompt, in pieces
    ([3000, 700], [50, 40], 4, 2, 64, 16, 900),
    ([600, 900, 33, 0, 700], [200, 1, 1, 0, 1], 8, 2, 128, 32, 0),  # one prompt with single tokens
    ([600, 900, 33, 0, 700], [200, 1, 1, 0, 1], 8, 2, 128, 32, 100),
    ([1, 50, 2], [1, 50, 1], 66, 33, 64, 16, 0),
])
def test_few_rows_share_the_keys(ops, cuda, lens, counts, heads, kv, d, p, window, dtype):
    check_attend(ops, cuda, attend_case(lens, counts, heads, kv, d, p, TYPES[dtype], seed=sum(lens)), window=window)


def test_both_ways_agree(ops, cuda):
    """The same rows alone and in a large batch: within what either may be off."""
    case = attend_case([700, 300], [90, 80], 4, 2, 128, 16, torch.bfloat16, 71)
    alone = check_attend(ops, cuda, case)
    among = check_in_a_large_batch(ops, cuda, case)[:170]
    _, tol = orc.attend(*case, 128**-0.5, 0, False)
    assert ((alone.cpu().double() - among.cpu().double()).abs() <= 2 * tol).all()


def test_out_may_be_the_query(ops, cuda):
    for lens, counts, tiles in (([300, 40], [1, 1], 0), ([5000], [1], 0), ([300], [90], 0), ([300], [90], 2048)):
        query, cache, tables, lens_, start = in_a_large_batch(attend_case(lens, counts, 4, 2, 64, 16, torch.float16, 73), tiles)
        q, args = query.to(cuda), [x.to(cuda) for x in (cache, tables, lens_)]
        kw = dict(query_start=start.to(cuda), max_query_len=max(counts))
        rows = int(start[-1])
        want = ops.paged_attention_kv4(q, *args, 0.1, max(lens), **kw)[:rows]
        assert ops.paged_attention_kv4(q, *args, 0.1, max(lens), out=q, **kw).data_ptr() == q.data_ptr()
        assert torch.equal(q[:rows], want) and torch.equal(q[rows:].cpu(), query[rows:])
    both = torch.zeros(3, 4, 64, dtype=torch.float16, device=cuda)
    with pytest.raises(RuntimeError, match="single memory location"):
        ops.paged_attention_kv4(both[:2], *args[:1], torch.zeros(2, 1, dtype=torch.int32, device=cuda),
                                torch.ones(2, dtype=torch.int32, device=cuda), 0.1, 1, out=both[1:])


def test_outs_that_are_refused(ops, cuda):
    query, cache, tables, lens, start = [x.to(cuda) for x in attend_case([30, 4], [1, 1], 4, 2, 64, 16, torch.float16, 79)]
    args = (query, cache, tables, lens, 0.1, 30)
    for out, error, text in ((query[:1].clone(), ValueError, "out must be"), (query.float(), RuntimeError, "out"),
                             (torch.empty(2, 64, 4, dtype=query.dtype, device=cuda).transpose(1, 2), ValueError, "contiguous"),
                             (torch.empty(513, dtype=query.dtype, device=cuda)[1:].view(2, 4, 64), RuntimeError, "aligned"),
                             (query.cpu(), RuntimeError, "GPU tensor")):
        with pytest.raises(error, match=text):
            ops.paged_attention_kv4(*args, out=out)


def test_gradients_are_refused(ops, cuda):
    query, cache, tables, lens, start = [x.to(cuda) for x in attend_case([30, 4], [1, 1], 4, 2, 64, 16, torch.float16, 83)]
    slots = torch.zeros(2, dtype=torch.int64, device=cuda)
    slots[1] = 40
    kv = torch.zeros(2, 2, 64, dtype=torch.float16, device=cuda)
    cs = torch.zeros(1, 64, device=cuda)
    calls = [lambda q: ops.paged_attention_kv4(q, cache, tables, lens, 0.1, 30),
             lambda q: ops.rope_append_kv4(slots, q, kv, kv, cs, cache, slots),
             lambda q: ops.token_logprobs(q.view(2, -1), slots, 1)]
    for call in calls:
        leaf = query.clone().requires_grad_()
        with pytest.raises(RuntimeError, match="requires a gradient"):
            call(leaf)
        with torch.no_grad():
            call(leaf)


def test_tables_without_a_block(ops, cuda):
    """No sequence has a block: every row of single tokens sees nothing; of other batches nobody knows where rows are."""
    query, cache, tables, lens, start = [x.to(cuda) for x in attend_case([30, 4], [1, 1], 4, 2, 64, 16, torch.float16, 89)]
    assert (ops.paged_attention_kv4(query, cache, tables[:, :0], lens, 0.1, 30) == 0).all()
    with pytest.raises(ValueError, match="no columns"):
        ops.paged_attention_kv4(query, cache, tables[:, :0], lens, 0.1, 30, query_start=start)


def test_one_cache_serves_both_types(ops, cuda):
    """What an fp16 caller appended a bf16 caller attends to, to the same values."""
    query, cache, tables, lens, start = attend_case([200, 70], [1, 1], 4, 2, 128, 16, torch.bfloat16, 97)
    small = torch.round(query.float() * 8) / 8  # (of few enough digits for either type)
    for dtype in TYPES.values():
        check_attend(ops, cuda, (small.to(dtype), cache, tables, lens, start), ragged=False)


@pytest.mark.parametrize("seqs,kv,longest,window", [
    (200, 1, 3000, 0), (200, 1, 3000, 700),  # more sequences than lanes
    (70, 4, 700, 0), (64, 4, 5000, 0), (130, 1, 2500, 0),
    (300, 4, 900, 0),                        # too many to be cut
])
def test_one_long_sequence_among_short_ones(ops, cuda, seqs, kv, longest, window):
    """It comes in pieces wherever it stands, the others in one, those without a token in none that count."""
    for at in (0, seqs // 2, seqs - 1):
        lens = [(7 * i) % 40 for i in range(seqs)]
        lens[at] = longest
        case = attend_case(lens, [1] * seqs, 2 * kv, kv, 64, 16, torch.float16, seqs + at)
        check_attend(ops, cuda, case, window=window, ragged=False)


def test_a_prompt_among_tokens_in_pieces(ops, cuda):
    lens, counts = [40] * 36, [1] * 36
    lens[5], counts[5], lens[20], counts[20], counts[30] = 3000, 90, 1300, 3, 0
    for window in (0, 1000):
        check_attend(ops, cuda, attend_case(lens, counts, 16, 8, 64, 16, torch.bfloat16, 101), window=window)


def test_a_captured_step_of_sequences_that_grow(ops, cuda):
    """Captured for the longest sequence there may be: each replay cuts what it finds into pieces anew."""
    case = attend_case([6000, 1, 300, 40], [1] * 4, 8, 2, 128, 16, torch.float16, 103)
    query, cache, tables, _, start = [x.to(cuda) for x in case]
    lens = torch.ones(4, dtype=torch.int32, device=cuda)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.paged_attention_kv4(query, cache, tables, lens, 0.1, 6000)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.paged_attention_kv4(query, cache, tables, lens, 0.1, 6000)
    for now in ([1, 1, 1, 1], [6000, 1, 300, 40], [900, 0, 5, 40], [4097, 1, 299, 0]):
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want, tol = orc.attend(case[0], case[1], case[2], torch.tensor(now), case[4], 0.1, 0, True)
        assert ((got.cpu().double() - want).abs() <= tol).all()
        assert torch.equal(got, ops.paged_attention_kv4(query, cache, tables, lens, 0.1, 6000))


def test_what_is_written_counts_as_changed(ops, cuda):
    """A tensor saved for a backward pass and then written to here is found out, as after torch's own writes in place."""
    query, cache, tables, lens, start = [x.to(cuda) for x in attend_case([30, 4], [1, 1], 4, 2, 64, 16, torch.float16, 107)]
    slots = torch.tensor([-1, -1], device=cuda)
    new = torch.zeros(2, 2, 64, dtype=torch.float16, device=cuda)
    before = cache._version
    ops.rope_append_kv4(slots, query, new, new, torch.zeros(1, 64, device=cuda), cache, slots)
    assert cache._version > before
    leaf = torch.ones(2, 4, 64, dtype=torch.float16, device=cuda, requires_grad=True)
    out = torch.zeros_like(query)
    loss = (leaf * out).sum()
    ops.paged_attention_kv4(query, cache, tables, lens, 0.1, 30, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        inner = torch.zeros_like(query)
    ops.paged_attention_kv4(query, cache, tables, lens, 0.1, 30, out=inner)
    assert torch.equal(inner, out)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("counts,large", [([1, 1], False), ([3, 40], False), ([20, 40], True)])
def test_blocks_that_a_window_has_left_behind_may_hold_anything(ops, cuda, counts, large, dtype):
    """Freed blocks in front of a window: parameters of infinity or NaN, and ids that no cache has, change nothing."""
    window, p, d = 40, 16, 64
    query, cache, tables, lens, start = attend_case([100, 333], counts, 4, 2, d, p, TYPES[dtype], 109, gain=1500.0)
    if large:
        query, cache, tables, lens, start = in_a_large_batch((query, cache, tables, lens, start), 2048)
    run = lambda c, t: ops.paged_attention_kv4(query.to(cuda), c.to(cuda), t.to(cuda), lens.to(cuda), 0.125 / 1500, 333,  # noqa: E731
                                               query_start=start.to(cuda), max_query_len=max(counts), window=window).cpu()
    rows = sum(counts)
    want, tol = orc.attend(query, cache, tables, lens, start, 0.125 / 1500, window, dtype == "fp16")
    assert bool(torch.isfinite(want[:rows]).all())
    for bits in (0x7c00, 0x7e00, 0xfc00):
        wrong, left = cache.clone(), tables.clone()
        for b in range(2):
            first = int(lens[b]) - counts[b] + 1 - window  # the first key that the first row sees
            for page in range(first // p):
                wrong[tables[b, page].long()].view(torch.int16)[:, p * d // 2:] = bits - (1 << 16 if bits > 0x7fff else 0)
        for gone in (False, True):
            if gone:
                wrong[0] = 0
                spare = [i for i in range(cache.shape[0]) if i not in tables.flatten().tolist()]
                if 0 not in spare:  # block 0 is one of a sequence's: leave it to the others to be read in its place
                    wrong[0] = cache[0]
                else:
                    wrong[0].view(torch.int16)[:, p * d // 2:] = bits - (1 << 16 if bits > 0x7fff else 0)
                for b in range(2):
                    left[b, :(int(lens[b]) - counts[b] + 1 - window) // p] = -1
            got = run(wrong, left)[:rows].double()
            off = int((~((got - want[:rows]).abs() <= tol[:rows])).sum())
            assert off == 0, (hex(bits), gone, off)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("seqs,kv,d,window", [
    (200, 4, 128, 0), (200, 4, 128, 30),    # two waves a workgroup
    (260, 4, 64, 0), (400, 4, 128, 0),      # one and two
    (530, 4, 64, 0), (530, 4, 64, 7),       # one
    (1600, 1, 128, 0),
])
def test_many_short_sequences(ops, cuda, seqs, kv, d, window, dtype):
    lens = [(11 * i) % 140 for i in range(seqs)]
    case = attend_case(lens, [1] * seqs, kv, kv, d, 16, TYPES[dtype], seqs)
    check_attend(ops, cuda, case, window=window, ragged=False)
    check_attend(ops, cuda, case, window=window, ragged=False, max_seq_len=1)  # (the rest of them is read all the same)


@pytest.mark.parametrize("heads,kv,longest,window", [(8, 2, 300, 0), (8, 2, 300, 50), (4, 4, 300, 0), (8, 1, 2600, 0), (8, 1, 2600, 1500)])
def test_prompts_among_more_sequences_than_lanes(ops, cuda, heads, kv, longest, window):
    """Prompts before, at and behind the 64th sequence, sequences without rows, rows past the promise."""
    seqs = 140
    counts, lens = [1] * seqs, [(13 * i) % 60 + 1 for i in range(seqs)]
    for at, rows in ((0, 70), (63, 41), (64, 90), (139, 33)):
        counts[at], lens[at] = rows, longest
    for at in (7, 62, 65, 128):
        counts[at] = 0
    query, cache, tables, lens, start = attend_case(lens, counts, heads, kv, 64, 16, torch.float16, longest)
    check_attend(ops, cuda, (query, cache, tables, lens, start), window=window)
    out = torch.full(query.shape, 7.0, dtype=query.dtype, device=cuda)
    ops.paged_attention_kv4(query.to(cuda), cache.to(cuda), tables.to(cuda), lens.to(cuda), 0.125, longest,
                            query_start=start.to(cuda), max_query_len=50, window=window, out=out)
    want, tol = orc.attend(query, cache, tables, lens, start, 0.125, window, True)
    late = torch.zeros(len(query), dtype=torch.bool)
    for at in (0, 64):
        late[int(start[at]) + 50:int(start[at + 1])] = True
    got = out.cpu().double()
    assert torch.isnan(got[late]).all()
    off = int((~((got - want).abs() <= tol))[~late].sum())
    assert off == 0, off


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("seqs,rows,heads,kv,window", [(90, 7, 32, 8, 0), (90, 7, 32, 8, 20), (40, 20, 32, 8, 0), (70, 9, 24, 8, 0), (33, 5, 160, 16, 0)])
def test_many_short_sequences_of_several_rows(ops, cuda, seqs, rows, heads, kv, window, dtype):
    """One and two waves for tiles of 32 columns; evenly spread rows and uneven ones."""
    counts = [max(1, rows - i % 3) for i in range(seqs)]
    lens = [c + (7 * i) % 50 for i, c in enumerate(counts)]
    check_attend(ops, cuda, attend_case(lens, counts, heads, kv, 64, 16, TYPES[dtype], seqs), window=window)
    counts[1], lens[1] = 3 * rows, 4 * rows
    check_attend(ops, cuda, attend_case(lens, counts, heads, kv, 64, 16, TYPES[dtype], seqs), window=window)


@pytest.mark.parametrize("lens,counts,heads,kv", [([700], [600], 128, 1), ([900, 40], [3, 2], 64, 1), ([2600], [5], 8, 2)])
def test_more_rows_promised_than_there_are(ops, cuda, lens, counts, heads, kv):
    """An upper bound that is far too high, beyond 32 bits of columns too, changes no bit."""
    query, cache, tables, lens_, start = [x.to(cuda) for x in attend_case(lens, counts, heads, kv, 64, 16, torch.float16, 113)]
    run = lambda rows: ops.paged_attention_kv4(query, cache, tables, lens_, 0.125, max(lens), query_start=start, max_query_len=rows)  # noqa: E731
    want = run(sum(counts))
    for rows in (32768, 10**6, (1 << 30) + 1, 0x7fffffff):
        assert torch.equal(run(rows), want)


def test_more_sequences_than_a_grid_has_in_one_direction(ops, cuda):
    """70 000 sequences of three drafted tokens and 24 heads, which are columns enough for waves of their own."""
    seqs, rows, heads, d, p = 70000, 3, 24, 64, 16
    few = attend_case([9, 3, 16, 5], [rows] * 4, heads, 1, d, p, torch.float16, 127)
    query, cache, tables, lens, _ = [x.to(cuda) for x in few]
    again = lambda t: t.repeat(seqs // 4, *[1] * (t.dim() - 1))  # noqa: E731
    start = torch.arange(seqs + 1, dtype=torch.int32, device=cuda) * rows
    got = ops.paged_attention_kv4(again(query), cache, again(tables), again(lens), 0.125, 16, query_start=start, max_query_len=rows)
    want, tol = orc.attend(*few, 0.125, 0, True)
    for at in (0, 65532 * rows, (seqs - 4) * rows):
        assert ((got[at:at + 4 * rows].cpu().double() - want).abs() <= tol).all()
    assert torch.equal(got.view(seqs // 4, -1), got[:4 * rows].view(1, -1).expand(seqs // 4, -1))


def test_tangents_are_refused(ops, cuda):
    """Forward-mode differentiation: no result that silently lacks its tangent."""
    import torch.autograd.forward_ad as fwad
    query, cache, tables, lens, start = [x.to(cuda) for x in attend_case([30, 4], [1, 1], 4, 2, 64, 16, torch.float16, 83)]
    slots = torch.tensor([0, 40], device=cuda)
    kv = torch.zeros(2, 2, 64, dtype=torch.float16, device=cuda)
    cs = torch.zeros(41, 64, device=cuda)
    calls = [(query, lambda x: ops.paged_attention_kv4(x, cache, tables, lens, 0.1, 30)),
             (query, lambda x: ops.paged_attention_kv4(query, cache, tables, lens, 0.1, 30, out=x)),
             (query, lambda x: ops.rope_append_kv4(slots, x, kv, kv, cs, cache, slots)),
             (kv, lambda x: ops.rope_append_kv4(slots, query, x, kv, cs, cache, slots)),
             (kv, lambda x: ops.rope_append_kv4(slots, query, kv, x, cs, cache, slots)),
             (cs, lambda x: ops.rope_append_kv4(slots, query, kv, kv, x, cache, slots)),
             (query.view(2, -1), lambda x: ops.token_logprobs(x, slots, 1))]
    for of, call in calls:
        with fwad.dual_level():
            dual = fwad.make_dual(of.clone(), torch.ones_like(of))
            with pytest.raises(RuntimeError, match="tangent"):
                call(dual)
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):
                call(dual)
            call(fwad.unpack_dual(dual).primal)
        call(of.clone())
