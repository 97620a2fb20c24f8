"""Token log probabilities (WarpPipeEngine.token_logprobs) against the 64-bit
oracle (oracle/attention.py).

Bounds. Ranks and alternatives are compared exactly. Log probabilities and
entropies are fp32: x - M is exact to one rounding (2^-24 of it), the sum of up
to 2^17 positive terms in per-thread chains of at most a few hundred and a tree
above them is within about 2^-17 relative (2^-24 times the longest chain, plus
2^-22 of each exponential), its logarithm within 2^-17; the entropy adds the
second sum's own 2^-17 of at most 30. Bound: 2^-20 |value| + 2^-14 for the
entropy, 2^-20 |value| + 2^-16 for log probabilities."""

import math

import pytest
import torch

from adapterslotsplusplus_b200 import WarpPipeConfig, WarpPipeEngine
from oracle.attention import token_logprobs

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def eng(cuda):
    return WarpPipeEngine(WarpPipeConfig(max_tokens=1024))


def logits(rows, vocab, dtype, seed=0, sharp=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g) * sharp).to(dtype)


def close(got, want, slack):
    got, want = got.double().cpu(), want.double()
    same = (got == want) | (got.isnan() & want.isnan())
    fin = torch.isfinite(want) & torch.isfinite(got)
    assert bool((same | fin).all()), (got[~(same | fin)], want[~(same | fin)])
    err = ((got - want).abs() - 2.0 ** -20 * want.abs())[fin]
    assert not err.numel() or float(err.max()) <= slack, float(err.max())


def check(eng, x, tokens, top):
    got = eng.token_logprobs(x.cuda() if not x.is_cuda else x, tokens.cuda(), top)
    lp, rank, ent, ids, top_lp = token_logprobs(x, tokens, top)
    close(got.logprob, lp, 2.0 ** -16)
    close(got.entropy, ent, 2.0 ** -14)
    close(got.top_logprobs, top_lp, 2.0 ** -16)
    assert torch.equal(got.rank.cpu().long(), rank)
    assert torch.equal(got.top_ids.cpu().long(), ids)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 7, 3), (3, 33, 32), (2, 1000, 5), (5, 4096, 20),
                                            (4, 32000, 5), (1, 50021, 32), (300, 2003, 1), (700, 1024, 0),
                                            (3, 131075, 20)])
def test_sizes(eng, dtype, rows, vocab, top):
    g = torch.Generator().manual_seed(1)
    x = logits(rows, vocab, dtype)
    check(eng, x, torch.randint(0, vocab, (rows,), generator=g), top)


@pytest.mark.parametrize("dtype", DTYPES)
def test_likely_tokens_and_sharp_rows(eng, dtype):
    """The given token is the maximum, or one logit has nearly all the mass."""
    x = logits(6, 30000, dtype)
    x[0, 17] = 60
    x[1, 29999] = 30
    x[2, 0] = 12
    check(eng, x, x.float().argmax(1), 4)
    check(eng, x * 0, torch.arange(6), 6)  # uniform: every logit ties


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_go_to_the_lowest_index(eng, dtype):
    g = torch.Generator().manual_seed(3)
    x = torch.randint(-3, 4, (40, 9000), generator=g).to(dtype)  # thousands of equal maxima: more than any list holds
    check(eng, x, torch.randint(0, 9000, (40,), generator=g), 32)
    y = torch.zeros(2, 70000, dtype=dtype)
    y[0, 5000:] = -0.0  # both zeros are equal
    check(eng, y, torch.tensor([3, 69999]), 32)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_logits(eng, dtype):
    low = torch.finfo(dtype).min
    x = logits(8, 5000, dtype)
    x[0, 10:] = -math.inf
    x[1, 4990:] = low
    x[2] = -math.inf  # an empty row
    x[3] = low  # uniform over the type's lowest value
    x[4] = -math.inf
    x[4, 4321] = -5  # one token left
    x[5, ::2] = low
    x[6, 1::2] = -math.inf
    x[7] = -math.inf
    x[7, 100:200] = low
    check(eng, x, torch.tensor([3, 4, 5, 6, 4321, 0, 1, 150]), 12)


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_and_infinity(eng, dtype):
    x = logits(3, 3000, dtype)
    x[0, 77] = math.nan
    x[1, 2999] = math.inf
    got = eng.token_logprobs(x.cuda(), torch.tensor([1, 2, 3]).cuda(), 3)
    assert bool(got.logprob[:2].isnan().all()) and bool(got.entropy[:2].isnan().all())
    assert int(got.top_ids[0, 0]) == 77 and int(got.top_ids[1, 0]) == 2999
    check(eng, x[2:], torch.tensor([3]), 3)


def test_large_offsets_and_ranges(eng):
    x = logits(4, 20000, torch.float32)
    check(eng, x + 3e4, torch.arange(4), 5)
    check(eng, x * 1e4, torch.arange(4), 5)
    check(eng, x * 1e-6, torch.arange(4), 5)


@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
def test_tokens_outside_the_vocabulary(eng, idx):
    x = logits(4, 1000, torch.bfloat16)
    t = torch.tensor([-1, 1000, 5, -100], dtype=idx)
    check(eng, x, t, 2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_strided_and_unaligned_rows(eng, dtype, offset):
    wide = logits(5, 3011, dtype).cuda()
    view = wide[:, offset:offset + 2999]
    check(eng, view, torch.arange(5), 7)
    check(eng, wide.t().contiguous().t()[:, :2000], torch.arange(5), 7)  # columns apart: copied


def test_no_rows_and_repeats(eng):
    got = eng.token_logprobs(torch.empty(0, 100, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"), 4)
    assert got.logprob.shape == (0,) and got.top_ids.shape == (0, 4)
    x, t = logits(9, 40000, torch.bfloat16).cuda(), torch.arange(9).cuda()
    a = eng.token_logprobs(x, t, 8)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(a, eng.token_logprobs(x, t, 8)))


def test_refusals(eng):
    x, t = logits(2, 100, torch.bfloat16).cuda(), torch.zeros(2, dtype=torch.int64, device="cuda")
    for f in (lambda: eng.token_logprobs(x, t, 33), lambda: eng.token_logprobs(x, t, -1),
              lambda: eng.token_logprobs(x[:, :3], t, 4), lambda: eng.token_logprobs(x.double(), t),
              lambda: eng.token_logprobs(x, t.float()), lambda: eng.token_logprobs(x, t[:1]),
              lambda: eng.token_logprobs(x.cpu(), t), lambda: eng.token_logprobs(x[0], t)):
        with pytest.raises(RuntimeError):
            f()
    p = x.data_ptr()
    assert eng._lib.wp_token_logprobs(eng.handle, p, None, None, None, None, p, 10, p, 4, 2, 100, 0, 1, None) == -1
    assert eng._lib.wp_token_logprobs(None, p, None, None, None, None, p, 100, p, 4, 2, 100, 0, 1, None) == -1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mask", [-1e4, -6e4, -1e6, -1e9, -1e10, -1e12, -1e15, -1e20, -1e30, -1e36, -1e38, -3e38])
def test_mask_constants(eng, dtype, mask):
    """Masked logits that hold some large negative number (minus infinity in
    fp16 where it has no such number): a thread's first vectors, alternate
    logits, whole parts of a row, all but one, all."""
    x = logits(7, 40000, dtype)
    x[0, :64] = mask
    x[1, 5:] = mask
    x[2, ::2] = mask
    x[3, 1000:39000] = mask
    x[4] = mask
    x[4, 31234] = 1.5
    x[5] = mask
    x[6, 20000:] = mask
    x[6, :10000] = mask / 3
    check(eng, x, torch.tensor([100, 3, 1, 39500, 31234, 7, 5]), 8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", [1e5, 1e6, 2e6, 1e8, 3e9, 1e10, 1e15, 1e30, 1e37, 1e38])
def test_rows_of_enormous_logits(eng, dtype, size):
    x = logits(6, 9000, torch.float64)
    x[0] += size
    x[1] -= size
    x[2] *= size / 16
    x[3, 77] = size
    x[4, ::3] = size
    x[4, 1::3] = -size
    x[5] = size
    check(eng, x.to(dtype), torch.tensor([100, 3, 1, 77, 1, 7]), 8)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rest", [-math.inf, -1e10, 2.0, 3e9, 1e37])
@pytest.mark.parametrize("odd", [math.nan, math.inf])
def test_nan_and_infinity_among_any_logits(eng, dtype, rest, odd):
    """One NaN or plus infinity anywhere makes the row NaN, whatever the other
    logits are; the row beside it is not touched."""
    x = logits(4, 20000, dtype)
    want = eng.token_logprobs(x[3:].cuda(), torch.tensor([5]).cuda(), 2)
    for i, at in enumerate((0, 9999, 19999)):
        x[i] = rest
        x[i, at] = odd
    got = eng.token_logprobs(x.cuda(), torch.tensor([3, 9999, 1, 5]).cuda(), 2)
    assert bool(got.logprob[:3].isnan().all()) and bool(got.entropy[:3].isnan().all())
    assert bool(got.top_logprobs[:3].isnan().all())
    check(eng, x[3:], torch.tensor([5]), 2)
    assert float(want.logprob[0]) == pytest.approx(float(got.logprob[3]), rel=1e-5)


def test_tensors_of_another_device_are_refused(eng):
    x, t = logits(2, 100, torch.bfloat16).cuda(), torch.zeros(2, dtype=torch.int64, device="cuda")
    here, eng.device = eng.device, torch.device("cuda", 1)
    try:
        with pytest.raises(RuntimeError, match="cuda:1"):
            eng.token_logprobs(x, t)
    finally:
        eng.device = here
    eng.token_logprobs(x, t)
