"""Attention over packed prompts (WarpPipeEngine.prompt_attention) against the
64-bit oracle (oracle/attention.py).

Bounds. A weight p <= 1 is rounded once to the inputs' type (u / 2 relative, u
= 2^-8 in bf16, 2^-11 in fp16), so the weighted mean moves by at most u / 2 of
sum p |v| / sum p <= max |v|, and the result is rounded by u / 2 of itself.
Scores are fp32 sums of exact products within 2^-17 of |score| <= 64, which
moves weights by under 2^-10 relative. Bound: u / 2 |ref| + (u / 2 + 2^-10)
max |v|; lse: 2^-10."""

import math

import pytest
import torch

from adapterslotsplusplus_b200 import WarpPipeConfig, WarpPipeEngine
from oracle.attention import attend

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng(cuda):
    return WarpPipeEngine(WarpPipeConfig(max_tokens=1024))


def starts(n):
    return torch.tensor([0] + list(n)).cumsum(0).to(torch.int32).cuda()


def oracle(q, k, v, nq, nk, scale):
    """attend() for every sequence, on the GPU in 64 bits where it is long."""
    outs, lses, a, b = [], [], 0, 0
    for n, t in zip(nq, nk):
        qs, ks, vs = q[a:a + n], k[b:b + t], v[b:b + t]
        a, b = a + n, b + t
        if n * t <= 3000 or not bool(torch.isfinite(vs.float()).all()):
            o, l = attend(qs, ks, vs, scale)
        else:
            g = q.shape[1] // k.shape[1]
            kk, vv = ks.cuda().double().repeat_interleave(g, 1), vs.cuda().double().repeat_interleave(g, 1)
            s = torch.einsum("ihd,jhd->hij", qs.cuda().double(), kk) * scale
            i, j = torch.arange(n, device="cuda")[:, None], torch.arange(t, device="cuda")
            s = s.masked_fill(j > i + t - n, -math.inf)
            l = torch.logsumexp(s, 2)
            p = torch.where((l == -math.inf)[..., None], 0.0, (s - torch.where(l == -math.inf, 0.0, l)[..., None]).exp())
            o, l = torch.einsum("hij,jhd->ihd", p, vv).cpu(), l.t().cpu()
        outs.append(o)
        lses.append(l)
    return torch.cat(outs), torch.cat(lses)


def check(eng, nq, nk, heads, kv_heads, dim, dtype, max_q=None, scale=None, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(sum(nq), heads, dim, generator=g).to(dtype)
    k = (torch.randn(sum(nk), kv_heads, dim, generator=g) * spread).to(dtype)
    v = torch.randn(sum(nk), kv_heads, dim, generator=g).to(dtype)
    same = nq is nk
    out, lse = eng.prompt_attention(q.cuda(), k.cuda(), v.cuda(), starts(nq), None if same else starts(nk), max_q, scale, True)
    ref, rl = oracle(q, k, v, nq, nk, dim ** -0.5 if scale is None else scale)
    u = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    big = float(v.float().abs().max()) if v.numel() else 0.0
    err = (out.double().cpu() - ref).abs() - u / 2 * ref.abs()
    assert float(err.max()) <= (u / 2 + 2.0 ** -10) * big, (float(err.max()), int(err.flatten(1).amax(1).argmax()))
    seen = torch.isfinite(rl)
    assert torch.equal(seen, torch.isfinite(lse.cpu()))
    assert float((lse.double().cpu() - rl)[seen].abs().max()) <= 2.0 ** -10
    assert eng.device_error(clear=True) == 0


DTYPES = [torch.bfloat16, torch.float16]
HEADS = [(4, 4, 64), (8, 2, 128), (6, 1, 64), (7, 1, 128), (24, 2, 128)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("lens", [[1], [4] * 9, [1, 2, 3, 15, 16, 17], [63, 64, 65], [127, 128, 129, 1], [300, 7, 255, 256, 257]])
def test_prompts(eng, dtype, heads, kv_heads, dim, lens):
    check(eng, lens, lens, heads, kv_heads, dim, dtype, max(lens))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
def test_chunks_behind_their_context(eng, dtype, heads, kv_heads, dim):
    nq, nk = [1, 5, 64, 130, 33], [200, 5, 65, 400, 161]
    check(eng, nq, nk, heads, kv_heads, dim, dtype, max(nq))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("max_q", [1, 17, 200, 10 ** 6, None])
def test_any_max_q_is_correct(eng, dtype, max_q):
    lens = [40, 1, 0, 201, 3]
    check(eng, lens, lens, 8, 2, 128, dtype, max_q)


@pytest.mark.parametrize("dim", [8, 16, 40, 72, 80, 96, 120])
@pytest.mark.parametrize("max_q", [4, 200])
def test_other_head_dims(eng, dim, max_q):
    lens = [4, 150, 33]
    check(eng, lens, lens, 6, 2, dim, torch.bfloat16, max_q)


@pytest.mark.parametrize("max_q", [1, 300])
def test_rows_that_see_nothing(eng, max_q):
    """More queries than keys, no keys at all, no queries."""
    check(eng, [5, 3, 0, 300, 20], [2, 0, 7, 170, 20], 4, 2, 64, torch.bfloat16, max_q)
    q = torch.ones(3, 2, 64, dtype=torch.float16, device="cuda")
    out, lse = eng.prompt_attention(q, q[:0], q[:0], starts([3]), starts([0]), max_q, return_lse=True)
    assert not out.any() and bool((lse == -math.inf).all())
    assert eng.prompt_attention(q[:0], q, q, starts([0]), starts([3])).shape == (0, 2, 64)
    assert eng.prompt_attention(q[:0], q[:0], q[:0], starts([])).shape == (0, 2, 64)


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_prompts(eng, dtype):
    check(eng, [2000, 1], [2000, 1], 4, 1, 128, dtype, 2000)
    check(eng, [700], [2500], 2, 2, 64, dtype, 700)


@pytest.mark.parametrize("max_q", [1, 400])
def test_growing_scores(eng, max_q):
    """Keys that grow along the sequence: the running maximum moves in every
    tile; and scores that are all the same."""
    n = 400
    q = torch.ones(n, 2, 64).bfloat16()
    k = (torch.arange(n)[:, None, None] / n * 6 * torch.ones(1, 2, 64)).bfloat16()
    v = torch.randn(n, 2, 64).bfloat16()
    for key in (k, k.flip(0), k * 0):
        out = eng.prompt_attention(q.cuda(), key.cuda(), v.cuda(), starts([n]), max_q=max_q).double().cpu()
        ref, _ = oracle(q, key, v, [n], [n], 64 ** -0.5)
        err = (out - ref).abs() - 2.0 ** -9 * ref.abs()
        assert float(err.max()) <= (2.0 ** -9 + 2.0 ** -10) * float(v.abs().max())


@pytest.mark.parametrize("max_q", [1, 300])
@pytest.mark.parametrize("dtype", DTYPES)
def test_unseen_keys_do_not_reach_a_row(eng, dtype, max_q):
    """Infinities and NaN in K and V of later tokens and of other sequences."""
    lens = [100, 37, 290]
    q, k, v = (torch.randn(sum(lens), 2, 64).to(dtype) for _ in range(3))
    clean = eng.prompt_attention(q.cuda(), k.cuda(), v.cuda(), starts(lens), max_q=max_q)
    k2, v2 = k.clone(), v.clone()
    v2[60, :, 3] = math.inf
    k2[61] = math.nan
    v2[62] = math.nan
    v2[100:137] = math.inf  # the whole second sequence
    v2[137 + 200, 1, 0] = math.nan
    got = eng.prompt_attention(q.cuda(), k2.cuda(), v2.cuda(), starts(lens), max_q=max_q)
    # rows that see none of these: equal but for the fp32 order of sums
    big = float(v.abs().max())
    tol = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -10
    for a, b, h in ((0, 60, slice(None)), (137, 337, slice(None)), (337, 427, slice(0, 1))):
        assert float((got[a:b, h].float() - clean[a:b, h].float()).abs().max()) <= 2 * tol * big
    ref, _ = oracle(q, k2, v2, lens, lens, 64 ** -0.5)
    assert torch.equal(got.cpu().isnan(), ref.isnan())
    assert torch.equal(got.cpu().isinf(), ref.isinf())


def test_strided_and_unaligned(eng):
    lens = [30, 140]
    T = sum(lens)
    fused = torch.randn(T, 8 + 2 + 2, 64, device="cuda").bfloat16()  # one qkv projection's output
    q, k, v = fused[:, :8], fused[:, 8:10], fused[:, 10:]
    want = eng.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), starts(lens), max_q=140)
    assert torch.equal(eng.prompt_attention(q, k, v, starts(lens), max_q=140), want)
    swapped = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]  # heads outermost
    assert torch.equal(eng.prompt_attention(*swapped, starts(lens), max_q=140), want)
    odd = [torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t) for t in (q, k, v)]
    assert torch.equal(eng.prompt_attention(*odd, starts(lens), max_q=140), want)


def test_other_stream_and_graph(eng):
    lens = [30, 140, 5]
    q, k, v = (torch.randn(sum(lens), 4, 128, device="cuda").half() for _ in range(3))
    cu = starts(lens)
    want = eng.prompt_attention(q, k, v, cu, max_q=140)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = eng.prompt_attention(q, k, v, cu, max_q=140)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = eng.prompt_attention(q, k, v, cu, max_q=140)
    for n in ([30, 140, 5], [175, 0, 0], [1, 2, 100]):
        cu.copy_(starts(n))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[:sum(n)], eng.prompt_attention(q, k, v, cu, max_q=140)[:sum(n)])


def test_bad_offsets_are_not_followed(eng):
    q = torch.randn(20, 2, 64, device="cuda").bfloat16()
    assert eng.device_error(clear=True) == 0
    eng.prompt_attention(q, q, q, torch.tensor([0, 10, 10 ** 6], dtype=torch.int32, device="cuda"))
    assert eng.device_error(clear=True) == 2
    eng.prompt_attention(q, q, q, torch.tensor([0, -7, 20], dtype=torch.int32, device="cuda"))
    assert eng.device_error(clear=True) == 2


def test_refusals(eng):
    q = torch.randn(10, 4, 64, device="cuda").bfloat16()
    cu = starts([10])
    for i, f in enumerate((
            lambda: eng.prompt_attention(q, q.half(), q.half(), cu),
            lambda: eng.prompt_attention(q.float(), q.float(), q.float(), cu),
            lambda: eng.prompt_attention(q, q[:, :3], q[:, :3], cu),
            lambda: eng.prompt_attention(q, q, q[:5], cu),
            lambda: eng.prompt_attention(q[0], q, q, cu),
            lambda: eng.prompt_attention(q, q[..., :32], q[..., :32], cu),
            lambda: eng.prompt_attention(q[..., :12], q[..., :12], q[..., :12], cu),
            lambda: eng.prompt_attention(*[torch.zeros(4, 2, 136, device="cuda").half()] * 3, starts([4])),
            lambda: eng.prompt_attention(q, q, q, cu.long()),
            lambda: eng.prompt_attention(q, q, q, cu.cpu()),
            lambda: eng.prompt_attention(q, q, q, cu, starts([5, 5])),
            lambda: eng.prompt_attention(q.cpu(), q.cpu(), q.cpu(), cu))):
        with pytest.raises(RuntimeError):
            f()
            pytest.fail(f"call {i} was accepted")
    assert eng._lib.wp_prompt_attention(None, *[None] * 3, 0, 0, None, 0, 0, None, 0, 0, None, None, 1, 1, 1, 1, 1, 1, 64,
                                        0.1, 1, None) == -1


@pytest.mark.parametrize("nq", [[0] * 700 + [300] + [0] * 700, [1, 0, 2] * 300 + [700], [260] * 90, [1500] + [30] * 200])
def test_far_fewer_and_far_more_items_than_sms(eng, nq):
    check(eng, nq, nq, 8, 8, 64, torch.bfloat16, max_q=max(nq))
    check(eng, nq, [n + 3 if n else 0 for n in nq], 12, 4, 128, torch.float16, max_q=max(nq))


def test_which_cta_takes_an_item_does_not_change_results(eng):
    nq = [900, 1, 400, 650, 33, 1200]
    q, k, v = (torch.randn(sum(nq), h, 128, device="cuda", dtype=torch.bfloat16) for h in (16, 4, 4))
    first = eng.prompt_attention(q, k, v, starts(nq), max_q=max(nq))
    for _ in range(10):
        assert torch.equal(eng.prompt_attention(q, k, v, starts(nq), max_q=max(nq)), first)


@pytest.mark.parametrize("max_q", [1, 300])
@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 3e38), (torch.bfloat16, -1e36), (torch.float16, 65504.0)])
def test_unseen_values_of_any_size_do_not_reach_a_row(eng, dtype, size, max_q):
    """The largest finite numbers in V of later tokens, of another sequence and
    of rows that belong to none: the weight of a key that a row must not see is
    exactly 0, so every bit of the row stays."""
    lens = [100, 37, 290]
    T = sum(lens)
    q, k, v = (torch.randn(T + 20, 2, 64).to(dtype) for _ in range(3))
    clean = eng.prompt_attention(q.cuda(), k.cuda(), v.cuda(), starts(lens), max_q=max_q)
    v[61] = size
    v[110] = size
    v[137 + 200, 1] = size
    v[T:] = size
    got = eng.prompt_attention(q.cuda(), k.cuda(), v.cuda(), starts(lens), max_q=max_q)
    for a, b, h in ((0, 61, slice(None)), (100, 110, slice(None)), (137, 337, slice(None)), (337, T, slice(0, 1))):
        assert torch.equal(got[a:b, h], clean[a:b, h])
    assert bool(torch.isfinite(got[:T]).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("empty", [0, 70])
def test_many_small_weights_beside_a_large_one(eng, dtype, empty):
    """60000 keys of weight e^-18 (2^-26 of the first key's, below what fp16
    holds) whose sum counts: out = n e^-18 / (1 + n e^-18). All V are of one
    sign, so a weight's relative error moves the result by as much: u / 2 for
    the weights, u / 2 for the result, 2^-10 for the scores (see the top); and
    half a step of the smallest 16-bit weight, 2^-33 of the largest, per key.
    (With 70 empty sequences beside it the call takes the warp-level kernel.)"""
    n = 60000
    q = torch.ones(3, 1, 64, dtype=dtype)
    k = torch.zeros(n, 1, 64, dtype=dtype)
    k[0] = 1
    v = torch.ones(n, 1, 64, dtype=dtype)
    v[0] = 0
    out, lse = eng.prompt_attention(q.cuda(), k.cuda(), v.cuda(), starts([3] + [0] * empty), starts([n] + [0] * empty), 3,
                                    18 / 64, True)
    tail = torch.tensor([n - 3, n - 2, n - 1], dtype=torch.float64) * math.exp(-18)
    ref = (tail / (1 + tail))[:, None, None]
    u = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    err = (out.double().cpu() - ref).abs()
    assert float((err - (u + 2.0 ** -10) * ref).max()) <= n * 2.0 ** -33, float(err.max())
    assert float((lse.double().cpu() - (18 + torch.log1p(tail))[:, None]).abs().max()) <= 2.0 ** -10


def test_rows_computed_again_hold_nobody_up(eng):
    """An infinity near the start of 400000 keys sends every row of the long
    sequence to the kernel's exact path, over a second of it in each warp, while
    other items of the same CTA wait. All of them come out: the rows that see
    the infinity, their other dimensions, and the sequence beside it, whose bits
    stay. Bound: at the top, once for each side."""
    nq, nk = [10240, 300], [400000, 300]
    q, k, v = (torch.randn(n, 4, 64, device="cuda", dtype=torch.bfloat16) for n in (sum(nq), sum(nk), sum(nk)))
    clean = eng.prompt_attention(q, k, v, starts(nq), starts(nk), 10240)
    v[5, :, 3] = math.inf
    got = eng.prompt_attention(q, k, v, starts(nq), starts(nk), 10240)
    assert eng.device_error(clear=True) == 0
    assert torch.equal(got[10240:], clean[10240:])
    assert bool((got[:10240, :, 3] == math.inf).all())
    rest = [d for d in range(64) if d != 3]
    a, b = got[:10240, :, rest].float(), clean[:10240, :, rest].float()
    u = 2.0 ** -8
    big = float(v[:, :, rest].float().abs().max())
    assert bool(((a - b).abs() <= 2 * (u / 2 * b.abs() + (u / 2 + 2.0 ** -10) * big)).all())


def test_tensors_of_another_device_are_refused(eng):
    q, cu = torch.randn(10, 4, 64, device="cuda").bfloat16(), starts([10])
    here, eng.device = eng.device, torch.device("cuda", 1)
    try:
        with pytest.raises(RuntimeError, match="cuda:1"):
            eng.prompt_attention(q, q, q, cu)
    finally:
        eng.device = here
    eng.prompt_attention(q, q, q, cu)
