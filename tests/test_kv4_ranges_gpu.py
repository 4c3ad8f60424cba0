"""Attention over the 4-bit cache where the values of a sequence's tokens, or the queries of a tile, are of very different
sizes: one token's values 10^3 to 10^9 times the others', attended to or not, first, in between, last or behind what a
row sees, in every form of the kernels; against 64 bits, within what the kernel's roundings come to key by key."""
import math

import pytest
import torch

from oracle import serving_oracle as orc
from test_kv4_gpu import TYPES
from test_kv4_rows_gpu import in_a_large_batch

pytestmark = pytest.mark.gpu

# sequences, rows of each, heads, kv heads, head size, tokens of a sequence, whether rows of no sequence fill the chip
FORMS = {
    "8 waves": (2, 1, 4, 2, 128, 70, False),
    "4 waves": (300, 1, 1, 1, 64, 40, False),
    "2 waves": (200, 1, 4, 4, 128, 40, False),
    "1 wave": (530, 1, 4, 4, 64, 40, False),
    "pieces": (1, 1, 8, 2, 128, 2600, False),
    "8 waves, 32 columns": (150, 9, 3, 1, 128, 40, False),
    "4 waves, 32 columns": (70, 9, 12, 4, 64, 40, False),
    "2 waves, 32 columns": (90, 7, 32, 8, 64, 40, False),
    "1 wave, 32 columns": (33, 5, 320, 32, 64, 30, False),
    "columns of their own": (2, 40, 4, 2, 128, 90, True),
}


@pytest.fixture(scope="module")
def ops():
    from vllm_quick_amd import ops
    return ops


def stored(seqs, kv, d, n, heads_of):
    """A cache of pages of 16 tokens and its tables: heads_of(length) -> keys and values [2, length, kv, D] of five
    sequences (of fewer, where there are fewer), which the others repeat; rubbish behind each."""
    g = torch.Generator().manual_seed(seqs + n)
    pages = -(-n // 16)
    lens = [n - i % 5 for i in range(seqs)]
    cache = torch.randint(0, 256, (seqs * pages + 2, kv, 16 * (d + 8)), generator=g, dtype=torch.uint8)
    cache.view(torch.float16)[:, :, 8 * d:] = float("nan")
    tables = torch.randperm(seqs * pages + 2, generator=g)[:seqs * pages].view(seqs, pages).to(torch.int32)
    for b in range(min(seqs, 5)):
        j = torch.arange(lens[b])
        orc.store(cache, d, tables[b].long()[j // 16] * 16 + j % 16, *heads_of(lens[b], g))
    for b in range(5, seqs):
        cache[tables[b].long()] = cache[tables[b % 5].long()]
    return cache, tables, torch.tensor(lens, dtype=torch.int32)


def case_of(form, dtype, large, small, share, where):
    """One token of values of deviation `large` at `where` of each sequence, all others of `small`; its score is share ln 2
    above what the others' are around."""
    seqs, rows, heads, kv, d, n, many = FORMS[form]
    g = torch.Generator().manual_seed(n)
    way = (torch.randint(0, 2, (d, ), generator=g) * 2 - 1).float()

    def heads_of(length, g):
        x = torch.randn(2, length, kv, d, generator=g)
        at = {"first": 0, "between": length // 2, "last": length - 1}[where]
        x[0] *= 0.3
        x[0, at] = way * (share * math.log(2) / d**0.5)
        x[1] *= small
        x[1, at] *= large / small
        return x

    cache, tables, lens = stored(seqs, kv, d, n, heads_of)
    query = (way + 0.3 * torch.randn(seqs * rows, heads, d, generator=g)).to(dtype)
    case = query, cache, tables, lens, torch.arange(seqs + 1, dtype=torch.int32) * rows
    return in_a_large_batch(case, 2048) if many else case


def run(ops, cuda, case, rows, scale, window=0):
    query, cache, tables, lens, start = case
    return ops.paged_attention_kv4(query.to(cuda), cache.to(cuda), tables.to(cuda), lens.to(cuda), scale, int(lens.max()),
                                   query_start=start.to(cuda) if rows > 1 else None, max_query_len=rows, window=window).cpu()


def some_of(case):
    """The first three and the last two sequences, or all that there are."""
    query, cache, tables, lens, start = case
    if len(lens) <= 5:
        return [(slice(0, int(start[-1])), (query[:int(start[-1])], cache, tables, lens, start))]
    rows = int(start[1])
    parts = []
    for b in (0, 1, 2, len(lens) - 2, len(lens) - 1):
        at = slice(b * rows, (b + 1) * rows)
        parts.append((at, (query[at], cache, tables[b:b + 1], lens[b:b + 1], torch.tensor([0, rows]))))
    return parts


def check(ops, cuda, form, case, scale=None, window=0):
    scale = FORMS[form][4]**-0.5 if scale is None else scale
    got = run(ops, cuda, case, FORMS[form][1], scale, window).double()
    for at, part in some_of(case):
        want, tol = orc.attend_counted(*part, scale, window)
        off = (got[at] - want).abs() / tol
        assert not (off > 1).any() and not torch.isnan(off).any(), f"{float((off > 1).double().mean()):.3f} of the results off, worst {float(off.max()):.3g} of what is allowed"


@pytest.mark.parametrize("where", ["first", "between", "last"])
@pytest.mark.parametrize("large,small,share", [
    (1500.0, 1e-6, 0),
    (30.0, 1e-4, 12),
    (30.0, 1e-5, 12),
    (10.0, 1e-2, 20),
    (3000.0, 3.0, 8),
])
@pytest.mark.parametrize("form", FORMS)
def test_a_large_token_that_is_attended_to(ops, cuda, form, large, small, share, where):
    for dtype in TYPES.values():
        check(ops, cuda, form, case_of(form, dtype, large, small, share, where))


def test_a_large_token_among_many(ops, cuda):
    """What each of 20 000 others loses adds up."""
    FORMS["many"] = (1, 1, 2, 1, 128, 20000, False)
    try:
        for large, small, share in ((30.0, 1e-4, 12), (50.0, 1e-3, 16), (10.0, 1e-2, 20)):
            for dtype in TYPES.values():
                check(ops, cuda, "many", case_of("many", dtype, large, small, share, "first"))
    finally:
        del FORMS["many"]


@pytest.mark.parametrize("where", ["first", "between", "last"])
@pytest.mark.parametrize("large,small,share", [
    (6000.0, 1e-4, -24),
    (15000.0, 1e-3, -30),
    (15000.0, 1e-6, -45),
    (100.0, 1e-4, -13),
])
@pytest.mark.parametrize("form", FORMS)
def test_a_large_token_that_is_hardly_attended_to(ops, cuda, form, large, small, share, where):
    for dtype in TYPES.values():
        check(ops, cuda, form, case_of(form, dtype, large, small, share, where))


@pytest.mark.parametrize("large,small,share", [(15000.0, 1e-3, 0), (6000.0, 1e-4, 6)])
@pytest.mark.parametrize("form", [f for f in FORMS if FORMS[f][1] > 1])
def test_a_large_token_that_a_window_leaves_behind(ops, cuda, form, large, small, share):
    """The first rows of a sequence see it, the last ones do not."""
    _, rows, _, _, _, n, _ = FORMS[form]
    for dtype in TYPES.values():
        check(ops, cuda, form, case_of(form, dtype, large, small, share, "first"), window=n - rows // 2 - 4)


@pytest.mark.parametrize("size", [1.0, 2.0**-10])
@pytest.mark.parametrize("form", [f for f in FORMS if FORMS[f][1] > 1])
def test_what_rows_do_not_see_changes_no_bit_of_them(ops, cuda, form, size):
    """Heads of the largest scale that fp16 holds, or of NaN, in the last token of each sequence, which its last row alone
    sees, or in the first one, which a window hides from it."""
    _, rows, _, kv, d, n, _ = FORMS[form]
    wide = torch.full((1, kv, d), 6e4)
    wide[..., ::2] = -6e4
    for dtype in TYPES.values():
        case = case_of(form, dtype, size, size, 0, "first")
        query, cache, tables, lens, start = case
        last = start[1:].long() - 1
        others = torch.ones(int(start[-1]), dtype=torch.bool)
        others[last] = False
        for at, window, kept in (("last", 0, others), ("first", n - 4, ~others)):
            # (lengths differ: the shortest sequences' last rows see their first token through this window)
            kept = kept.clone()
            if at == "first":
                kept[last[lens <= n - 4]] = False
            base = run(ops, cuda, case, rows, d**-0.5, window)[:int(start[-1])]
            for x in (wide, torch.full((1, kv, d), float("nan"))):
                other = cache.clone()
                for b, length in enumerate(lens.tolist()):
                    j = length - 1 if at == "last" else 0
                    orc.store(other, d, tables[b, j // 16].long().view(1) * 16 + j % 16, x, x)
                got = run(ops, cuda, (query, other, tables, lens, start), rows, d**-0.5, window)[:int(start[-1])]
                assert torch.equal(got[kept], base[kept]) and not torch.isnan(base).any()
                assert not torch.equal(got[~kept], base[~kept])


@pytest.mark.parametrize("size", [1e4, 1e6, 1e8, 1e10, 1e20, 1e31, -1e9, -1e31])
@pytest.mark.parametrize("form", FORMS)
def test_scores_of_any_size(ops, cuda, form, size):
    """Scores so far apart that one token of each row has all the weight (to what 64 bits say); bf16 queries, whose type
    has the range."""
    query, *rest = case_of(form, torch.float32, 1.0, 1.0, 0, "first")
    query = (query * (abs(size) if abs(size) > 1e10 else 1.0)).bfloat16()
    check(ops, cuda, form, (query, *rest), scale=math.copysign(1.0, size) if abs(size) > 1e10 else size)


@pytest.mark.parametrize("large", [0, 1, -1])
@pytest.mark.parametrize("form", [f for f in FORMS if FORMS[f][2] * FORMS[f][1] > FORMS[f][3]])
def test_a_query_that_is_far_larger_than_its_neighbours(ops, cuda, form, large):
    """One head of one row (of each sequence) 10^9, 10^12 or 10^30 times, in fp16 10^6 times the others, which share its tile."""
    seqs, rows, heads, _, d, _, _ = FORMS[form]
    for dtype, low, high in (("bf16", 1.0, 1e9), ("bf16", 1.0, 1e12), ("bf16", 1e-6, 1e24), ("fp16", 1e-2, 1e4)):
        query, *rest = case_of(form, torch.float32, 1.0, 1.0, 0, "first")
        query = query * low
        head = heads - 1 if large < 0 else large
        at = torch.arange(seqs) * rows + (rows - 1 if large else 0)
        query[at, head] *= high / low
        assert torch.isfinite(query.to(TYPES[dtype])).all()
        check(ops, cuda, form, (query.to(TYPES[dtype]), *rest), scale=d**-0.5 / low)
