"""The 4-bit key/value cache (KvCache4): bytes written by append, values read
back, and attention, against the 64-bit oracle (oracle/attention.py).

Bounds. append and read are exact: the format's fp32 steps are single IEEE
operations, so bytes and values have to be equal. attention rounds twice: each
weight times V's scale to fp16 (relative 2^-12, so at most 2^-12 * 15 * scale =
2^-12 of V's range in the weighted mean), and the result to 16 bits (2^-9 in
bf16, 2^-12 in fp16, of the result). Scores are fp32 sums of exact products: at
the tested sizes (|score| below 64, 128 terms) they are within 64 * 2^-17, which
moves a weight by under 2^-10 relative in the worst case and the mean by that
times V's range. Bound: u |ref| + (2^-11 + 2^-10) range(V), u = 2^-8 or 2^-11."""

import math

import pytest
import torch

from adapterslotsplusplus_b200 import KvCache4, WarpPipeConfig, WarpPipeEngine
from adapterslotsplusplus_b200._lib import WarpPipeError
from oracle.attention import attend, kv4_tile, kv4_values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng(cuda):
    return WarpPipeEngine(WarpPipeConfig(max_tokens=1024))


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Batch:
    """Sequences with their tokens in a cache whose pages are handed out in no
    order, from the host's own copy of K and V."""

    def __init__(self, eng, total, kv_heads, dim, dtype, page_size=64, seed=0, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.total, self.dtype = total, dtype
        self.k = [(torch.randn(t, kv_heads, dim, generator=g) * spread + 0.5).to(dtype) for t in total]
        self.v = [(torch.randn(t, kv_heads, dim, generator=g) * spread).to(dtype) for t in total]
        need = [-(-t // page_size) for t in total]
        order = torch.randperm(sum(need) + 3, generator=g).tolist()
        self.table = torch.full((len(total), max(max(need), 1) + 1), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            for j in range(n):
                self.table[b, j] = order.pop()
        self.cache = KvCache4(eng, sum(need) + 3, kv_heads, dim, page_size, dtype)
        self.cache.pages.fill_(0xFF)  # every scale and zero outside is NaN
        self.table = self.table.cuda()
        self.lens = i32(total)

    def append_all(self):
        T = sum(self.total)
        if T:
            cu = i32([0] + self.total).cumsum(0).to(torch.int32)
            self.cache.append(torch.cat(self.k).cuda(), torch.cat(self.v).cuda(), self.table, self.lens, cu)
        return self


def starts(n):
    return torch.tensor([0] + n).cumsum(0).to(torch.int32).cuda()


def check_attention(batch, new, heads, max_q=None, seed=1, scale=None):
    g = torch.Generator().manual_seed(seed)
    kvh, dim, dtype = batch.cache.kv_heads, batch.cache.head_dim, batch.dtype
    q = torch.randn(sum(new), heads, dim, generator=g).to(dtype)
    out, lse = batch.cache.attention(q.cuda(), batch.table, batch.lens, starts(new), max(new) if max_q is None else max_q,
                                     scale=scale, return_lse=True)
    out, lse = out.double().cpu(), lse.double().cpu()
    u = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    at = 0
    for b, n in enumerate(new):
        if n == 0:
            continue
        k, v = kv4_values(batch.k[b]), kv4_values(batch.v[b])
        ref, rl = attend(q[at:at + n], k, v, 1 / math.sqrt(dim) if scale is None else scale)
        span = float((v.amax(-1) - v.amin(-1)).max()) if v.numel() else 0.0
        err = (out[at:at + n] - ref).abs() - u * ref.abs()
        assert float(err.max()) <= (2.0 ** -11 + 2.0 ** -10) * span, (b, float(err.max()), span)
        seen = torch.isfinite(rl)
        assert torch.equal(seen, torch.isfinite(lse[at:at + n]))
        # scores within 64 * 2^-17, and the sum's own fp32 rounding
        assert float((lse[at:at + n] - rl)[seen].abs().max() if seen.any() else 0) <= 2.0 ** -10
        at += n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page_size", [16, 64, 80])
def test_append_writes_the_declared_bytes(eng, dtype, dim, page_size):
    total = [1, 16, 17, 37, 64, 100]
    b = Batch(eng, total, 2, dim, dtype, page_size).append_all()
    pages = b.cache.pages.cpu()
    table = b.table.cpu()
    for s, t in enumerate(total):
        pad = -(-t // 16) * 16
        for h in range(2):
            for i in range(pad // 16):
                k, v = (torch.zeros(16, dim, dtype=dtype) for _ in range(2))
                n = min(16, t - 16 * i)
                k[:n], v[:n] = b.k[s][16 * i:16 * i + n, h], b.v[s][16 * i:16 * i + n, h]
                got = pages[table[s, 16 * i // page_size], h, i % (page_size // 16)]
                want = kv4_tile(k, v)
                mask = torch.ones(16 * dim + 128, dtype=torch.bool)
                for tok in range(n, 16):  # bytes of tokens that were never written stay as they were
                    mask[tok * dim // 2:(tok + 1) * dim // 2] = False
                    one = (8 * dim + torch.arange(8 * dim).view(dim // 64, 8, 4, 4, 4)[:, :, tok % 8 // 2, :,
                                                                                    tok % 2 * 2 + tok // 8].reshape(-1))
                    mask[one] = False
                    for o in (16 * dim, 16 * dim + 64):
                        mask[o + 4 * tok:o + 4 * tok + 4] = False
                assert torch.equal(got[mask], want[mask]), (s, h, i)
                assert bool((got[~mask] == 0xFF).all()), (s, h, i)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
def test_append_in_pieces_and_read(eng, dtype, dim):
    """Tokens that arrive one, a few or many at a time end in the same cache,
    and a read of any number of last tokens gives their values."""
    total = [1, 5, 33, 130]
    b = Batch(eng, total, 3, dim, dtype)
    have = [0] * 4
    while have != total:
        n = [min(t - x, step) for t, x, step in zip(total, have, (1, 2, 7, 50))]
        k = torch.cat([b.k[s][have[s]:have[s] + n[s]] for s in range(4)])
        v = torch.cat([b.v[s][have[s]:have[s] + n[s]] for s in range(4)])
        have = [x + y for x, y in zip(have, n)]
        # k and v as column slices of one fused tensor: strided rows
        both = torch.cat([k, v], 1).cuda()
        b.cache.append(both[:, :3], both[:, 3:], b.table, i32(have), starts(n))
    whole = Batch(eng, total, 3, dim, dtype).append_all()
    for n in (total, [1, 0, 20, 129], [0, 5, 1, 17]):
        k, v = b.cache.read(b.table, b.lens, starts(n), sum(n))
        k2, v2 = whole.cache.read(whole.table, whole.lens, starts(n), sum(n))
        want_k = torch.cat([kv4_values(b.k[s])[total[s] - n[s]:] for s in range(4)]).to(dtype)
        want_v = torch.cat([kv4_values(b.v[s])[total[s] - n[s]:] for s in range(4)]).to(dtype)
        for got, want in ((k, want_k), (v, want_v), (k2, want_k), (v2, want_v)):
            assert torch.equal(got.cpu(), want)
    assert eng.device_error(clear=True) == 0


def test_one_token_without_offsets(eng):
    b = Batch(eng, [4, 16, 18, 65], 2, 128, torch.bfloat16).append_all()
    k, v = b.cache.read(b.table, b.lens)
    assert torch.equal(k.cpu(), torch.cat([kv4_values(x)[-1:] for x in b.k]).to(torch.bfloat16))
    new_k, new_v = torch.randn(4, 2, 128).bfloat16(), torch.randn(4, 2, 128).bfloat16()
    b.cache.append(new_k.cuda(), new_v.cuda(), b.table, b.lens)  # overwrites the last tokens
    k, v = b.cache.read(b.table, b.lens)
    assert torch.equal(k.cpu(), kv4_values(new_k).bfloat16()) and torch.equal(v.cpu(), kv4_values(new_v).bfloat16())


def test_constant_and_extreme_rows(eng):
    """A constant row has scale 0; rows of the type's largest values and of its
    subnormals keep their own."""
    for dtype in (torch.bfloat16, torch.float16):
        b = Batch(eng, [6], 1, 64, dtype)
        top = 3e4 if dtype == torch.float16 else 1e38
        b.k[0][0] = 1.25
        b.k[0][1] = 0
        b.k[0][2] = torch.linspace(-top, top, 64).to(dtype)
        b.k[0][3] = (torch.linspace(0, 1, 64) * (1e-7 if dtype == torch.float16 else 1e-39)).to(dtype)
        b.append_all()
        k, _ = b.cache.read(b.table, b.lens, starts([6]), 6)
        assert torch.equal(k.cpu(), kv4_values(b.k[0]).to(dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,kv_heads,group", [(64, 3, 1), (128, 2, 4), (128, 1, 8), (64, 2, 7), (128, 1, 12)])
def test_decode(eng, dtype, dim, kv_heads, group):
    total = [1, 2, 15, 16, 17, 63, 64, 65, 200, 700]
    b = Batch(eng, total, kv_heads, dim, dtype).append_all()
    check_attention(b, [1] * len(total), kv_heads * group)
    assert eng.device_error(clear=True) == 0


@pytest.mark.parametrize("page_size", [16, 48, 128])
def test_page_sizes(eng, page_size):
    b = Batch(eng, [3, 47, 49, 300], 2, 128, torch.bfloat16, page_size).append_all()
    check_attention(b, [1] * 4, 8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [1, 3, 8])
def test_several_queries(eng, dtype, group):
    """Ragged numbers of query tokens, none among them, and any max_q."""
    total = [5, 40, 64, 130, 257, 1]
    b = Batch(eng, total, 2, 128, dtype).append_all()
    for new in ([1, 5, 0, 3, 9, 1], [5, 4, 3, 2, 1, 0], [5, 40, 17, 33, 20, 1]):
        for max_q in (max(new), 1):
            check_attention(b, new, 2 * group, max_q)


def test_rows_that_see_nothing(eng):
    """More queries than tokens, and empty sequences: zeros, lse -inf."""
    b = Batch(eng, [0, 2, 0, 20], 2, 64, torch.bfloat16).append_all()
    check_attention(b, [1, 5, 3, 1], 4)
    empty = Batch(eng, [0, 0], 2, 64, torch.bfloat16)
    out, lse = empty.cache.attention(torch.ones(2, 2, 64, dtype=torch.bfloat16, device="cuda"), empty.table, empty.lens,
                                     return_lse=True)
    assert not out.any() and bool((lse == -math.inf).all())
    none = empty.cache.attention(torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda"), empty.table[:0], empty.lens[:0])
    assert none.shape == (0, 2, 64)


def test_long_context_is_split_and_joined(eng):
    """One sequence over every warp of the GPU; the same twice, bit for bit."""
    b = Batch(eng, [9001, 33], 1, 128, torch.bfloat16).append_all()
    check_attention(b, [1, 1], 2)
    q = torch.randn(2, 2, 128, device="cuda").bfloat16()
    outs = [b.cache.attention(q, b.table, b.lens) for _ in range(3)]
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_unseen_tokens_do_not_reach_a_row(eng):
    """Infinities in tokens after a query, NaN past the end of the page."""
    b = Batch(eng, [70], 1, 128, torch.bfloat16)
    clean = Batch(eng, [70], 1, 128, torch.bfloat16).append_all()
    b.k[0][67:, :, 3] = math.inf
    b.v[0][67:, :, 5] = -math.inf
    b.append_all()
    q = torch.randn(6, 4, 128, device="cuda").bfloat16()
    got = b.cache.attention(q, b.table, b.lens, starts([6]), 6)
    want = clean.cache.attention(q, clean.table, clean.lens, starts([6]), 6)
    assert torch.equal(got[:3], want[:3])
    assert bool(got[3:].isnan().any())


def test_uneven_magnitudes(eng):
    """V's scales over many orders of magnitude, a dominating first token, and
    queries of large and tiny norm."""
    for dtype in (torch.bfloat16, torch.float16):
        b = Batch(eng, [150], 1, 64, dtype)
        b.v[0] *= (10.0 ** torch.linspace(-3, 2, 150)).to(dtype)[:, None, None]
        b.k[0][0] *= 4
        b.append_all()
        check_attention(b, [4], 4)
        check_attention(b, [4], 4, scale=1e-4)
        check_attention(b, [1], 4, scale=0.0)


def test_strided_queries(eng):
    b = Batch(eng, [40, 90], 2, 64, torch.bfloat16).append_all()
    wide = torch.randn(2, 8, 64, device="cuda").bfloat16()
    views = [wide[:, :4], wide[:, 1::2], wide.transpose(0, 1).contiguous().transpose(0, 1)[:, :4]]
    odd = torch.randn(2 * 4 * 64 + 3, device="cuda").bfloat16()[3:].view(2, 4, 64)  # not 16-byte aligned
    for q in views + [odd]:
        want = b.cache.attention(q.contiguous().clone(), b.table, b.lens)
        assert torch.equal(b.cache.attention(q, b.table, b.lens), want)


def test_streams_and_graph(eng):
    """Calls on two streams at once do not share scratch; a captured step
    follows lengths that change between replays."""
    b = Batch(eng, [500, 900], 2, 128, torch.bfloat16).append_all()
    q = torch.randn(2, 8, 128, device="cuda").bfloat16()
    want = b.cache.attention(q, b.table, b.lens)
    other = Batch(eng, [900, 40], 2, 128, torch.bfloat16, seed=5).append_all()
    want2 = other.cache.attention(q, other.table, other.lens)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        with torch.cuda.stream(s1):
            x = b.cache.attention(q, b.table, b.lens)
        with torch.cuda.stream(s2):
            y = other.cache.attention(q, other.table, other.lens)
        torch.cuda.synchronize()
        assert torch.equal(x, want) and torch.equal(y, want2)
    k = torch.randn(2, 2, 128, device="cuda").bfloat16()
    v = torch.randn(2, 2, 128, device="cuda").bfloat16()
    lens = b.lens.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.cache.append(k, v, b.table, lens)
        out = b.cache.attention(q, b.table, lens)
    for n in ([500, 900], [17, 64], [1, 333]):
        lens.copy_(i32(n))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, b.cache.attention(q, b.table, lens))


def test_bad_pages_and_lengths_are_not_followed(eng):
    b = Batch(eng, [40, 90], 2, 64, torch.bfloat16).append_all()
    q = torch.randn(2, 4, 64, device="cuda").bfloat16()
    assert eng.device_error(clear=True) == 0
    bad = b.table.clone()
    bad[1, 0] = 10 ** 6
    b.cache.attention(q, bad, b.lens)
    assert eng.device_error(clear=True) == 2
    b.cache.read(bad, b.lens)
    assert eng.device_error(clear=True) == 0  # the last token's page is a good one
    before = b.cache.pages.clone()
    bad[:, 0] = -5
    b.cache.append(q[:, :2], q[:, 2:], bad, i32([40, 50]))
    assert eng.device_error(clear=True) == 2
    assert torch.equal(before, b.cache.pages)
    b.cache.attention(q, b.table, i32([40, 10 ** 7]))
    assert eng.device_error(clear=True) == 2
    b.cache.append(q[:, :2], q[:, 2:], b.table, i32([0, 0]))  # more new tokens than the sequences have
    assert eng.device_error(clear=True) == 2
    assert torch.equal(before, b.cache.pages)


def test_refusals(eng):
    b = Batch(eng, [40], 2, 64, torch.bfloat16).append_all()
    c = b.cache
    q = torch.randn(1, 4, 64, device="cuda").bfloat16()
    bad = [
        lambda: KvCache4(eng, 4, 2, 96),
        lambda: KvCache4(eng, 4, 2, 64, page_size=24),
        lambda: KvCache4(eng, 4, 2, 64, dtype=torch.float32),
        lambda: KvCache4(eng, pages=torch.zeros(4, 2, 4, 1000, dtype=torch.uint8, device="cuda")),
        lambda: c.attention(q.half(), b.table, b.lens),
        lambda: c.attention(q[..., :32], b.table, b.lens),
        lambda: c.attention(q[:, :3], b.table, b.lens),
        lambda: c.attention(q, b.table.long(), b.lens),
        lambda: c.attention(q, b.table, b.lens.cpu()),
        lambda: c.attention(q, b.table[:0], b.lens),
        lambda: c.attention(torch.cat([q, q]), b.table, b.lens),
        lambda: c.attention(q, b.table, b.lens, starts([1, 1])),
        lambda: c.append(q, q, b.table, b.lens),
        lambda: c.append(q[:, :2], q[:0, :2], b.table, b.lens),
        lambda: c.read(b.table, b.lens, starts([1])),
        lambda: c.attention(q.cpu(), b.table, b.lens),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(RuntimeError):
            f()
            pytest.fail(f"call {i} was accepted")
    lib, h = eng._lib, eng.handle
    args = [q.data_ptr(), None, q.data_ptr(), 256, 64, c.pages.data_ptr(), c.num_pages, 64, b.table.data_ptr(), 2,
            b.lens.data_ptr(), None, 1, 1, 1, 4, 2, 64, 0.1, 1, None, 0, None]
    assert lib.wp_kv4_attention(h, *args) == -1 and b"workspace" in lib.wp_last_error(h)
    assert lib.wp_kv4_attention(None, *args) == -1
    with pytest.raises(WarpPipeError):
        eng._check(lib.wp_kv4_append(h, c.pages.data_ptr(), 1, 24, q.data_ptr(), 8, 8, q.data_ptr(), 8, 8,
                                     b.table.data_ptr(), 2, b.lens.data_ptr(), None, 1, 1, 2, 64, 1, None))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
def test_nan_and_infinity_stay_in_the_cache(eng, dtype, dim):
    """A NaN or an infinity in a row of K or V makes that row NaN (its scale or
    zero is none or infinite), for read and for the queries that see it, and
    nothing else."""
    clean = Batch(eng, [70, 20], 2, dim, dtype).append_all()
    b = Batch(eng, [70, 20], 2, dim, dtype)
    b.k[0][66, 0, 3] = math.nan
    b.v[0][67, 1, dim - 1] = math.nan
    b.k[1][19, 0, 9] = -math.nan
    b.v[1][3, 1, 0] = math.inf
    b.append_all()
    k, v = b.cache.read(b.table, b.lens, starts([70, 20]), 90)
    for got, x in ((k, b.k), (v, b.v)):
        want = torch.cat([kv4_values(y) for y in x]).to(dtype)
        assert torch.equal(got.cpu().isnan(), want.isnan())
        assert torch.equal(got.cpu().nan_to_num(7.0), want.nan_to_num(7.0))
    assert bool(k[66, 0].isnan().all()) and bool(v[67, 1].isnan().all()) and bool(k[89, 0].isnan().all())
    q = torch.randn(9, 4, dim, device="cuda").to(dtype)
    got = b.cache.attention(q, b.table, b.lens, starts([6, 3]), 6)
    want = clean.cache.attention(q, clean.table, clean.lens, starts([6, 3]), 6)
    bad = torch.zeros(9, 4, dtype=torch.bool)
    bad[2:6, :2] = True  # token 66 and later see K's NaN of the first kv head
    bad[3:6, 2:] = True  # token 67 and later V's of the second
    bad[8, :2] = True
    bad[6:, 2:] = True
    assert torch.equal(got.cpu().isnan(), bad[..., None].expand_as(got))
    assert torch.equal(got.cpu()[~bad], want.cpu()[~bad])


def test_tensors_of_another_device_are_refused(eng):
    """The engine's device is the cache's: everything else is refused before a
    kernel could follow its address."""
    b = Batch(eng, [40], 2, 64, torch.bfloat16).append_all()
    c = b.cache
    q = torch.randn(1, 4, 64, device="cuda").bfloat16()
    here, eng.device = eng.device, torch.device("cuda", 1)
    try:
        for f in (lambda: KvCache4(eng, pages=c.pages), lambda: c.attention(q, b.table, b.lens),
                  lambda: c.append(q[:, :2], q[:, 2:], b.table, b.lens), lambda: c.read(b.table, b.lens)):
            with pytest.raises(RuntimeError, match="cuda:1"):
                f()
    finally:
        eng.device = here
    c.attention(q, b.table, b.lens)
