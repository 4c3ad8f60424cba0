"""Log probabilities of given tokens, entropy and the most likely tokens on the GPU, against 64 bits.

Tolerances: Z - 1 is a sum of fp32 exponentials, each off by at most |d| 2^-23 (its argument's rounding; below d = -40 it
weighs nothing) and the steps of 32 additions a lane and 22 between lanes: relatively 2^-23 (40 + 54) of the sum without
the maximum.  log Z moves by that times (Z - 1) / Z; the differences x - m are rounded once (2^-24) and so is the result.
The entropy is a sum of two positive terms with the same relative errors."""
import pytest
import torch

from oracle import serving_oracle as orc

pytestmark = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SUM = 2.0**-23 * 94


@pytest.fixture(scope="module")
def ops():
    from vllm_quick_amd import ops
    return ops


def near(got, want, tol):
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    fine = torch.isfinite(want)
    assert ((got - want).abs()[fine] <= tol[fine]).all(), float(((got - want).abs() / tol)[fine].max())


def check(ops, cuda, logits, tokens, top, dev_logits=None):
    got = ops.token_logprobs(logits.to(cuda) if dev_logits is None else dev_logits, tokens.to(cuda), top)
    given, entropy, at, best = orc.logprobs(logits, tokens, top)
    x = logits.double()
    most = x.amax(1)
    rest = 1 - (x == most[:, None]).sum(1) * torch.exp(most - torch.logsumexp(x, 1))  # (Z - 1) / Z, or what is not a maximum's
    moved = SUM * rest.clamp(min=0).nan_to_num(0.0) + 2.0**-40
    near(got[0], given, 2.0**-23 * given.abs() + moved)
    near(got[1], entropy, 4 * SUM * entropy.abs() + 2.0**-40)
    assert got[2].dtype == torch.int64 and torch.equal(got[2].cpu(), at)
    near(got[3], best, 2.0**-23 * best.abs() + moved[:, None])
    return got


def random_logits(rows, vocab, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * 2.5
    x[torch.arange(rows), torch.randint(0, vocab, (rows, ), generator=g)] += torch.rand(rows, generator=g) * 20
    return x.to(dtype), torch.randint(0, vocab, (rows, ), generator=g)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 0), (1, 1, 1), (3, 2, 2), (2, 7, 3), (5, 64, 64), (4, 65, 20), (3, 513, 64), (2, 1000, 20), (7, 4099, 5),
    (2, 8185, 1), (3, 8186, 20), (2, 8192, 3), (2, 8193, 64), (3, 32000, 5), (2, 32761, 2), (2, 32762, 2), (2, 32765, 2),
    (2, 32768, 1), (3, 32769, 64), (2, 65536, 20), (3, 128011, 5), (1, 262145, 64), (300, 1001, 3),
])
def test_logprobs(ops, cuda, rows, vocab, top, dtype):
    check(ops, cuda, *random_logits(rows, vocab, TYPES[dtype], rows * 7 + vocab), top)


@pytest.mark.parametrize("vocab", [900, 32000, 70001])
@pytest.mark.parametrize("top", [1, 20, 64])
def test_rows_of_equals(ops, cuda, vocab, top):
    """The lowest index first: rows of one value, of two, of both zeros, and ties at the border."""
    x = torch.zeros(6, vocab)
    x[1, ::2] = -0.0
    x[2, 1::3] = 1.0
    x[3] = torch.arange(vocab).float().div(400, rounding_mode="floor")
    x[4] = -x[3]
    x[5, vocab // 2:vocab // 2 + 30] = 2.0
    for dtype in TYPES.values():
        check(ops, cuda, x.to(dtype), torch.full((6, ), vocab - 1), top)


@pytest.mark.parametrize("vocab", [50, 5000, 40000])
def test_rows_with_tokens_shut_out(ops, cuda, vocab):
    """-inf throughout, but for one token, but for fewer than are asked for; infinities; NaN."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn(8, vocab, generator=g)
    x[0] = -float("inf")
    x[1] = -float("inf")
    x[1, vocab - 3] = -4.0
    x[2, 3:] = -float("inf")
    x[3, 11] = float("inf")
    x[4, 17] = float("nan")
    x[5, ::2] = -float("inf")
    x[6, 0] = -float("nan")
    x[6, 30:32] = float("inf")
    x[7] = torch.finfo(torch.float16).min
    x[7, 4] = 3.0
    tokens = torch.tensor([0, vocab - 3, 40, 11, 3, 0, 1, 4])
    for dtype in TYPES.values():
        check(ops, cuda, x.to(dtype), tokens, 9)


def test_tokens_outside_the_vocabulary(ops, cuda):
    x, _ = random_logits(4, 40000, torch.float16, 3)
    check(ops, cuda, x, torch.tensor([-1, 40000, 2**40, 39999]), 2)
    x, _ = random_logits(4, 400, torch.float16, 3)
    check(ops, cuda, x, torch.tensor([-100, 400, -2**40, 0]), 2)


def test_one_token_has_nearly_everything(ops, cuda):
    """The log probability of the likely token, and the entropy, keep their digits where they are tiny."""
    x = torch.full((5, 3000), -3.0)
    for i, lift in enumerate((5, 15, 25, 40, 80)):
        x[i, 100 + i] = lift
    check(ops, cuda, x, torch.arange(100, 105), 3)


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
def test_strides(ops, cuda, dtype):
    x, tokens = random_logits(5, 777, TYPES[dtype], 4)
    wide = torch.full((5, 900), 50.0, dtype=x.dtype, device=cuda)
    for at in (0, 1, 3, 8, 123):
        view = wide[:, at:at + 777]
        wide.fill_(50.0)
        view.copy_(x)
        check(ops, cuda, x, tokens, 4, dev_logits=view)
    across = x.t().contiguous().to(cuda).t()
    check(ops, cuda, x, tokens, 4, dev_logits=across)
    same = x[:1].to(cuda).expand(5, 777)
    check(ops, cuda, x[:1].expand(5, 777), tokens, 4, dev_logits=same)
    every = torch.stack([tokens, tokens], 1).to(cuda)[:, 0]
    assert torch.equal(ops.token_logprobs(x.to(cuda), every)[0], ops.token_logprobs(x.to(cuda), tokens.to(cuda))[0])


def test_more_than_2_31_logits(ops, cuda):
    rows, vocab = 70000, 32000
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device=cuda)
    x[-1, 7] = 5.0
    tokens = torch.full((rows, ), 7, dtype=torch.int64, device=cuda)
    given, entropy, at, best = ops.token_logprobs(x, tokens, 2)
    assert at[-1].tolist() == [7, 0] and at[0].tolist() == [0, 1]
    few, fe, _, fb = ops.token_logprobs(x[-2:].clone(), tokens[-2:], 2)
    assert torch.equal(given[-2:], few) and torch.equal(entropy[-2:], fe) and torch.equal(best[-2:], fb)


def test_empty(ops, cuda):
    out = ops.token_logprobs(torch.zeros(0, 10, device=cuda), torch.zeros(0, dtype=torch.int64, device=cuda), 3)
    assert [tuple(t.shape) for t in out] == [(0, ), (0, ), (0, 3), (0, 3)]


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("rows,vocab,top", [
    (2, 12000, 64), (3, 16377, 5), (2, 16378, 20), (2, 16381, 3), (2, 16382, 1), (2, 16384, 2), (2, 16385, 64), (300, 9000, 4),
    (1030, 8500, 2),  # too many rows for one workgroup each
])
def test_logprobs_of_middling_vocabularies(ops, cuda, rows, vocab, top, dtype):
    check(ops, cuda, *random_logits(rows, vocab, TYPES[dtype], rows * 3 + vocab), top)


@pytest.mark.parametrize("top", [1, 64])
def test_rows_of_equals_of_a_middling_vocabulary(ops, cuda, top):
    x = torch.zeros(4, 14001)
    x[1, 1::3] = 1.0
    x[2] = torch.arange(14001).float().div(400, rounding_mode="floor")
    x[3, 17] = float("nan")
    for dtype in TYPES.values():
        check(ops, cuda, x.to(dtype), torch.full((4, ), 14000), top)
