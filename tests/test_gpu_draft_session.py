"""DraftSession (adapterslotsplusplus_b200/draft.py): prompts, drafted tokens
over the 4-bit caches and their log probabilities, with the LoRA of an adapter
pool, against the same decoder with its attention in plain torch.

Bounds as in tests/test_gpu_draft.py: both sides round every projection and
attention output to bf16 once, independently, so two layers differ by rounding
noise (DRAFT_TOL of the output's rms). The plain side attends to the values
that the caches stand for, so quantisation is on both sides."""

import math

import pytest
import torch

from adapterslotsplusplus_b200 import AdapterPool, WarpPipeConfig, WarpPipeEngine
from adapterslotsplusplus_b200.draft import DraftDecoder, DraftSession
from oracle.attention import attend

pytestmark = pytest.mark.gpu
DRAFT_TOL = 6e-2
VOCAB = 1003


@pytest.fixture()
def setup(cuda):
    eng = WarpPipeEngine(WarpPipeConfig(max_tokens=1024))
    model = DraftDecoder(layers=2, hidden=256, heads=4, inter=512, vocab=VOCAB, device=cuda)
    dims = model.dims()
    pool = AdapterPool(eng, num_slots=4, dims=dims, rank=16, max_adapters=8)
    g = torch.Generator().manual_seed(1)
    for t in range(4):
        pool.register_host(t, pool.pack([((torch.randn(16, d, generator=g) * 0.05).bfloat16(),
                                          (torch.randn(o, 16, generator=g) * 0.05).bfloat16()) for d, o in dims]))
    session = DraftSession(model, eng, num_pages=40, page_size=16)
    return eng, model, pool, session


def starts(n):
    return torch.tensor([0] + list(n)).cumsum(0).to(torch.int32).cuda()


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def adapters(pool, n, ids):
    """The step's segment table: sequence b's n[b] tokens use adapter ids[b]."""
    tokens = torch.tensor([a for a, k in zip(ids, n) for _ in range(k)], dtype=torch.int64, device="cuda")
    pool.prepare(ids)
    assert pool.build_seg_bounds(tokens)
    return dict(lora="pool", pool=pool, scale=2.0)


def close(a, b):
    a, b = a.float(), b.float()
    assert float((a - b).abs().max()) <= DRAFT_TOL * float(b.pow(2).mean().sqrt())


def plain(session, table, lens, n, whole):
    """attention(layer, q, k, v) in 64 bits over the call's own K and V (whole)
    or what the session's caches, already appended to, stand for."""
    total = lens.tolist()

    def f(layer, q, k, v):
        if not whole:
            k, v = session.caches[layer].read(table, lens, starts(total), sum(total))
        out, a, b = [], 0, 0
        for i, t in zip(n, n if whole else total):
            out.append(attend(q[a:a + i], k[b:b + t], v[b:b + t], 1 / math.sqrt(64))[0])
            a, b = a + i, b + t
        return torch.cat(out).to(q).contiguous()

    return f


def test_prompts_drafts_and_scores(setup):
    eng, model, pool, session = setup
    ids, n = [0, 0, 2], [5, 37, 1]
    table = torch.randperm(40)[:36].view(3, 12).to(torch.int32).cuda()
    g = torch.Generator(device="cuda").manual_seed(3)

    def tokens(k):
        return (torch.randn(sum(k), 256, device="cuda", generator=g) * 0.5).bfloat16()

    head = model.lm_head
    # prompts
    x, lens = tokens(n), i32(n)
    lora = adapters(pool, n, ids)
    h = session.prefill(x, starts(n), table, lens, max(n), **lora)
    model.lm_head = None
    close(h, model.forward(x, 0, attention=plain(session, table, lens, n, True), **lora))
    # a second chunk behind the first, over what the cache stands for
    more = [20, 3, 7]
    total = [a + b for a, b in zip(n, more)]
    x, lens = tokens(more), i32(total)
    lora = adapters(pool, more, ids)
    model.lm_head = head
    h = session.prefill(x, starts(more), table, lens, 20, context=(starts(total), sum(total)), **lora)
    assert model.lm_head is head
    model.lm_head = None
    close(h, model.forward(x, 0, attention=plain(session, table, lens, more, False), **lora))
    # drafted tokens: 1, 4 and 2
    draft = [1, 4, 2]
    total = [a + b for a, b in zip(total, draft)]
    x, lens = tokens(draft), i32(total)
    lora = adapters(pool, draft, ids)
    h = session.decode(x, table, lens, starts(draft), 4, **lora)
    ref = model.forward(x, 0, attention=plain(session, table, lens, draft, False), **lora)
    close(h, ref)
    # one token each, without offsets
    total = [t + 1 for t in total]
    x, lens = tokens([1, 1, 1]), i32(total)
    lora = adapters(pool, [1, 1, 1], ids)
    h = session.decode(x, table, lens, **lora)
    close(h, model.forward(x, 0, attention=plain(session, table, lens, [1, 1, 1], False), **lora))
    # scores
    model.lm_head = head
    given = torch.tensor([3, VOCAB - 1, 500], device="cuda")
    lp = session.score(h, given, top=4)
    ref = torch.log_softmax(torch.nn.functional.linear(h, head).double(), 1)
    best = ref.sort(dim=1, descending=True, stable=True)
    assert torch.equal(lp.top_ids.long(), best.indices[:, :4])
    assert float((lp.top_logprobs - best.values[:, :4]).abs().max()) < 1e-4
    assert float((lp.logprob - ref[torch.arange(3), given]).abs().max()) < 1e-4
    assert eng.device_error(clear=True) == 0


def test_decode_step_in_a_graph(setup):
    """One captured step serves growing sequences and changing adapters."""
    eng, model, pool, session = setup
    n, ids = [9, 30], [1, 3]
    table = torch.arange(40, device="cuda", dtype=torch.int32).view(2, 20)
    lens = i32(n)
    lora = adapters(pool, n, ids)
    session.prefill((torch.randn(39, 256, device="cuda") * 0.5).bfloat16(), starts(n), table, lens, 30, **lora)
    x = (torch.randn(2, 256, device="cuda") * 0.5).bfloat16()
    given = torch.tensor([1, 2], device="cuda")
    lens.add_(1)
    lora = adapters(pool, [1, 1], ids)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        session.score(session.decode(x, table, lens, **lora), given, 2)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h = session.decode(x, table, lens, **lora)
        lp = session.score(h, given, 2)
    for ids in ([1, 3], [0, 2], [3, 3]):
        adapters(pool, [1, 1], ids)
        x.normal_(0, 0.5)
        graph.replay()
        again = session.decode(x, table, lens, **lora)
        assert torch.equal(h, again)
        assert torch.equal(lp.top_ids, session.score(again, given, 2).top_ids)
        lens.add_(1)


def test_refusals(setup):
    eng, model, pool, session = setup
    model.lm_head = None
    with pytest.raises(RuntimeError):
        session.score(torch.zeros(1, 256, device="cuda", dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int64, device="cuda"))
    with pytest.raises(RuntimeError):
        DraftSession(DraftDecoder(layers=1, hidden=256, heads=8, inter=256, device="cuda"), eng, 4)  # head_dim 32
