"""Timed cases of the operators around the LoRA projections of a serving step.

    prompt    WarpPipeEngine.prompt_attention: causal attention over packed prompts, grouped heads, each sequence
              optionally behind a context (a later chunk of a prompt)
    cache     KvCache4.attention: one or a few query tokens per sequence over a paged cache held in 4 bits
    append    KvCache4.append and KvCache4.read: new tokens into that cache, and a range of it back in 16 bits
    score     WarpPipeEngine.token_logprobs: log probability, rank and entropy of given tokens, and the top alternatives

`own` chooses between the plain form (elementary torch operations in 32 bits) and the framework's kernels.

Layout of the 4-bit cache: uint8 pages [num_pages, kv_heads, page_size / 16, 16 D + 128]. A tile of 16 tokens holds the
codes of K ([16 tokens][D / 2 bytes], dimension 2b in the low and 2b + 1 in the high half of byte b), the codes of V
([D / 64][8 g][4 c][4 m][4 j] bytes: token 2c + (j >> 1) + 8 (j & 1), dimension 64 h + 16 m + g in the low half and
8 further in the high half), then (scale, zero) in 16 bits for each token of K and of V.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
PAGE = 64


# ---- the cases -------------------------------------------------------------------------------------------------------


def _prompt(dtype, seqs, lo, hi, past, heads, kv_heads, dim, **name):
    return dict(op="prompt", dtype=dtype, seqs=seqs, lo=lo, hi=hi, past=past, heads=heads, kv_heads=kv_heads, dim=dim, **name)


def _cache(dtype, seqs, lo, hi, queries, heads, kv_heads, dim, **name):
    return dict(op="cache", dtype=dtype, seqs=seqs, lo=lo, hi=hi, queries=queries, heads=heads, kv_heads=kv_heads, dim=dim,
                **name)


def _append(dtype, seqs, lo, hi, new, read_all, kv_heads, dim, **name):
    return dict(op="append", dtype=dtype, seqs=seqs, lo=lo, hi=hi, new=new, read_all=read_all, kv_heads=kv_heads, dim=dim,
                **name)


def _score(dtype, rows, vocab, top, **name):
    return dict(op="score", dtype=dtype, rows=rows, vocab=vocab, top=top, **name)


def listed():
    return [
        # the small decoder's own step: 64 sequences of 4 drafted tokens, 12 heads of 64
        _prompt("bf16", 64, 4, 4, 0, 12, 12, 64, name="prompt_drafts"),
        # chunks of prompts of mixed lengths (one token to many) behind contexts of up to 600 tokens, grouped heads
        _prompt("fp16", 16, 1, 1500, 600, 32, 8, 128, name="prompt_ragged"),
        # one long prompt
        _prompt("bf16", 1, 8192, 8192, 0, 32, 8, 128, name="prompt_long"),
        # one user, one token: latency
        _cache("bf16", 1, 2000, 2000, 1, 32, 8, 128, name="cache_one"),
        # the small decoder: many short contexts, every head its own K and V
        _cache("bf16", 256, 1, 512, 1, 12, 12, 64, name="cache_drafts"),
        # verification of up to 5 drafted tokens per sequence, 40 heads of 128
        _cache("fp16", 16, 300, 4000, 5, 40, 40, 128, name="cache_verify"),
        # a full batch of long contexts, grouped heads
        _cache("bf16", 32, 4096, 32768, 1, 32, 8, 128, name="cache_long"),
        # a decode step's new tokens, each read back
        _append("bf16", 256, 1, 2000, 1, False, 8, 128, name="append_step"),
        # a chunk of each prompt goes in, the whole context comes back for the chunk's attention
        _append("fp16", 8, 700, 4096, 512, True, 8, 128, name="append_chunk"),
        # a few sequences' next tokens with 5 alternatives
        _score("bf16", 4, 32000, 5, name="score_step"),
        # verification of a batch's drafted tokens, a large vocabulary, 20 alternatives
        _score("bf16", 256, 128000, 20, name="score_verify"),
        # the log probabilities of a prompt's own tokens, logits in 32 bits, an odd vocabulary
        _score("fp32", 2048, 32003, 1, name="score_prompt"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "cache", "cache", "append", "score", "score"])
    dtype = rng.choice(["bf16", "fp16"])
    dim = rng.choice([64, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8])
    if op == "prompt":
        hi = _log(rng, 1, 6000)
        most = max(1, int(1.2e9 / (heads * (hi + 1.0) ** 2)))  # the plain form's padded scores
        return _prompt(dtype, _log(rng, 1, min(96, most)), _log(rng, 1, hi), hi, rng.choice([0, 0, _log(rng, 1, 1000)]), heads,
                       kv_heads, dim)
    if op == "cache":
        hi = _log(rng, 16, 30000)
        most = max(1, int(6e8 / (hi * kv_heads * dim)))
        return _cache(dtype, _log(rng, 1, min(300, most)), _log(rng, 1, hi), hi, rng.choice([1, 1, 1, 3, 8]), heads, kv_heads,
                      dim)
    if op == "append":
        hi = _log(rng, 4, 4000)
        new = rng.choice([1, _log(rng, 1, hi)])
        most = max(1, int(4e7 / (hi * kv_heads * dim)))
        return _append(dtype, _log(rng, 1, min(300, most)), _log(rng, 1, hi), hi, new, rng.random() < 0.5, kv_heads, dim)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    vocab = _log(rng, 1000, 150000)
    return _score(dtype, _log(rng, 1, min(3000, int(3.4e7 / vocab))), vocab, rng.choice([0, 1, 5, 20]))


def _lens(case):
    """Lengths of the case's sequences, spread over their logarithm: (tokens of this call, all tokens)."""
    rng = random.Random(7)
    long = [_log(rng, case["lo"], case["hi"]) for _ in range(case["seqs"])]
    if long:
        long[-1] = case["hi"]
    if case["op"] == "prompt":
        return long, [n + (_log(rng, 1, case["past"]) if case["past"] else 0) for n in long]
    if case["op"] == "cache":
        return [min(n, rng.randint(1, case["queries"])) for n in long], long
    return [min(n, case["new"]) for n in long], long


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "score":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (20 + 8 * case["top"]), "flops": 6 * n}
    new, total = _lens(case)
    dim, kv = case["dim"], case["kv_heads"]
    if case["op"] == "append":
        read = sum(total if case["read_all"] else new)
        return {"bytes": (sum(new) + read) * kv * (5 * dim + 8), "flops": (4 * sum(new) + 2 * read) * kv * 2 * dim}
    pairs = sum(n * t - n * (n - 1) // 2 for n, t in zip(new, total))
    flops = 4 * dim * case["heads"] * pairs
    queries = 2 * 2 * sum(new) * case["heads"] * dim
    if case["op"] == "prompt":
        return {"bytes": queries + 2 * 2 * sum(total) * kv * dim, "flops": flops}
    return {"bytes": queries + sum(total) * kv * (dim + 8), "flops": flops}


# ---- inputs ----------------------------------------------------------------------------------------------------------


def _starts(lens):
    return torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()


def _keys_values(g, n, kv, dim, dtype):
    """K with a few strong channels, V without; the values of the attention paths."""
    k = torch.randn(n, kv, dim, device="cuda", generator=g)
    k = k * (1 + 3 * (torch.rand(kv, dim, device="cuda", generator=g) > 0.95))
    v = torch.randn(n, kv, dim, device="cuda", generator=g)
    return k.to(dtype), v.to(dtype)


def _codes(x):
    """4-bit codes of x's last axis, and the axis' scale and zero in x's own type."""
    zero = x.amin(-1)
    f, z = x.float(), zero.float()
    scale = ((f.amax(-1) - z) * (1.0 / 15.0)).to(x.dtype)
    step = scale.float().unsqueeze(-1)
    code = torch.where(step > 0, torch.round((f - z.unsqueeze(-1)) / step), 0.0).clamp(0, 15)
    return code.to(torch.uint8), scale, zero


def _tile_bytes(code_k, code_v, scales):
    """Codes [N, 16, D] and scales [N, 2, 16, 2] of whole tiles -> [N, 16 D + 128] bytes."""
    n, _, dim = code_k.shape
    k = code_k[..., 0::2] | code_k[..., 1::2] << 4
    v = code_v.view(n, 2, 4, 2, dim // 64, 4, 2, 8).permute(0, 4, 7, 2, 5, 3, 1, 6)  # h g c m j1 j0 half
    v = v[..., 0] | v[..., 1] << 4
    return torch.cat([k.reshape(n, -1), v.reshape(n, -1), scales.reshape(n, -1).view(torch.uint8)], 1)


def _cache_content(case, seed):
    """All tokens of the case's sequences, their codes, and where each goes."""
    new, total = _lens(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, dim, kv, dtype = sum(total), case["dim"], case["kv_heads"], DTYPES[case["dtype"]]
    k, v = _keys_values(g, n, kv, dim, dtype)
    return g, new, total, k, v


def _pages(total, k, v, g):
    """The pages with every token of k and v in them, and the table of each sequence's pages (in no order)."""
    kv, dim = k.shape[1], k.shape[2]
    count = torch.tensor([-(-t // PAGE) for t in total])
    num = int(count.sum())
    order = torch.randperm(num, device="cuda", generator=g)
    table = torch.zeros(len(total), int(count.max()), dtype=torch.int32, device="cuda")
    table[torch.arange(table.shape[1]) < count.unsqueeze(1)] = order.to(torch.int32)
    seq = torch.repeat_interleave(torch.arange(len(total), device="cuda"), torch.tensor(total, device="cuda"))
    pos = torch.arange(sum(total), device="cuda") - _starts(total)[seq]
    row = table[seq, pos // PAGE].long() * PAGE + pos % PAGE
    tiles = num * PAGE // 16

    def place(x):
        y = torch.zeros(num * PAGE, *x.shape[1:], dtype=x.dtype, device="cuda")
        y[row] = x
        return y.view(tiles, 16, kv, -1).permute(0, 2, 1, 3).reshape(tiles * kv, 16, -1)

    (ck, sk, zk), (cv, sv, zv) = _codes(k), _codes(v)
    scales = torch.stack([place(torch.stack(p, -1)) for p in ((sk, zk), (sv, zv))], 1)
    pages = _tile_bytes(place(ck), place(cv), scales)
    pages = pages.view(num, PAGE // 16, kv, -1).permute(0, 2, 1, 3).contiguous()
    return pages, table


_engines = []


def _engine():
    from adapterslotsplusplus_b200 import WarpPipeEngine

    if not _engines:
        _engines.append(WarpPipeEngine())
    return _engines[0]


def prepare(case, seed):
    if case["op"] == "score":
        return _prepare_score(case, seed)
    new, total = _lens(case)
    heads, dim, dtype = case.get("heads"), case["dim"], DTYPES[case["dtype"]]
    if case["op"] == "prompt":
        g = torch.Generator(device="cuda").manual_seed(seed)
        k, v = _keys_values(g, sum(total), case["kv_heads"], dim, dtype)
        q = torch.randn(sum(new), heads, dim, device="cuda", generator=g).to(dtype)
        s = dict(q=q, k=k, v=v, cu=_starts(new), cu_k=_starts(total), longest=max(new), longest_k=max(total))
    else:
        g, new, total, k, v = _cache_content(case, seed)
        pages, table = _pages(total, k, v, g)
        s = dict(table=table, lens=torch.tensor(total, dtype=torch.int32, device="cuda"), cu=_starts(new), dtype=dtype)
        if case["op"] == "cache":
            s.update(pages=pages, q=torch.randn(sum(new), heads, dim, device="cuda", generator=g).to(dtype), longest=max(new))
        else:
            read = total if case["read_all"] else new
            s.update(pages=pages, cu_read=_starts(read), tokens=sum(read))
            s["k"], s["v"] = _keys_values(g, sum(new), case["kv_heads"], dim, dtype)
    s.update(op=case["op"])
    if own:
        from adapterslotsplusplus_b200 import KvCache4

        s["engine"] = _engine()
        if "pages" in s:
            s["cache"] = KvCache4(s["engine"], pages=s["pages"], dtype=dtype)
    return s


def _rows_of(total, new):
    """Rows of the last new[b] tokens of each sequence among all of them."""
    ends = torch.tensor(total).cumsum(0).tolist()
    return torch.cat([torch.arange(e - n, e) for e, n in zip(ends, new)]).cuda()


def _prepare_score(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, vocab = case["rows"], case["vocab"]
    logits = torch.randn(rows, vocab, device="cuda", generator=g) * 2
    likely = torch.randint(0, vocab, (rows, 16), device="cuda", generator=g)
    logits.scatter_(1, likely, torch.rand(rows, 16, device="cuda", generator=g) * 8 + 6)
    some = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    tokens = torch.where(torch.arange(rows, device="cuda") % 4 == 3, some, likely[:, 0])
    s = dict(op="score", logits=logits.to(DTYPES[case["dtype"]]), tokens=tokens, top=case["top"])
    if own:
        s["engine"] = _engine()
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------


def run(s):
    if own:
        if s["op"] == "prompt":
            return s["engine"].prompt_attention(s["q"], s["k"], s["v"], s["cu"], s["cu_k"], max_q=s["longest"])
        if s["op"] == "cache":
            return s["cache"].attention(s["q"], s["table"], s["lens"], s["cu"], max_q=s["longest"])
        if s["op"] == "append":
            s["cache"].append(s["k"], s["v"], s["table"], s["lens"], s["cu"])
            return s["cache"].read(s["table"], s["lens"], s["cu_read"], s["tokens"])
        return tuple(s["engine"].token_logprobs(s["logits"], s["tokens"], s["top"]))
    return {"prompt": _plain_prompt, "cache": _plain_cache, "append": _plain_append, "score": _plain_score}[s["op"]](s)


def _seq_of(cu, n):
    """(sequence, place in it) of each of n packed tokens."""
    each = cu[1:] - cu[:-1]
    seq = torch.repeat_interleave(torch.arange(each.numel(), device=cu.device), each, output_size=n)
    return seq, torch.arange(n, device=cu.device) - cu[seq]


def _padded(x, cu, longest):
    """Packed [T, ...] -> [B, longest, ...], in 32 bits, zero past each sequence's end."""
    at = cu[:-1, None] + torch.arange(longest, device=x.device)
    inside = at < cu[1:, None]
    y = x[at.clamp(max=x.shape[0] - 1)].float()
    return torch.where(inside.view(*inside.shape, *[1] * (x.dim() - 1)), y, 0.0)


def _attend(q, k, v, n, t):
    """q [B, n, Hq, D], k and v [B, t, Hkv, D] padded to the longest; n, t: lengths of each sequence."""
    B, N, H, D = q.shape
    T, K = k.shape[1], k.shape[2]
    i, j = torch.arange(N, device=q.device), torch.arange(T, device=q.device)
    seen = (j <= i[:, None] + (t - n).view(B, 1, 1)) & (j < t.view(B, 1, 1)) & (i[:, None] < n.view(B, 1, 1))
    seen = seen.view(B, 1, 1, N, T)
    q = q.view(B, N, K, H // K, D).permute(0, 2, 3, 1, 4).reshape(B, K, -1, D) * (1.0 / math.sqrt(D))
    w = (q @ k.permute(0, 2, 3, 1)).view(B, K, H // K, N, T).masked_fill_(~seen, -math.inf)
    top = w.amax(-1, keepdim=True)
    w = w.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = w.sum(-1, keepdim=True)
    out = (w.view(B, K, -1, T) @ v.transpose(1, 2)).view(B, K, H // K, N, D) / torch.where(total == 0, 1.0, total)
    return out.permute(0, 3, 1, 2, 4).reshape(B, N, H, D)


def _plain_prompt(s):
    q, k, v = _padded(s["q"], s["cu"], s["longest"]), *(_padded(s[x], s["cu_k"], s["longest_k"]) for x in "kv")
    out = _attend(q, k, v, s["cu"][1:] - s["cu"][:-1], s["cu_k"][1:] - s["cu_k"][:-1])
    return out[_seq_of(s["cu"], s["q"].shape[0])].to(s["q"].dtype)


def _plain_cache(s):
    dim, dtype = s["q"].shape[2], s["dtype"]
    tiles = s["pages"][s["table"].long()].transpose(2, 3).flatten(1, 2)  # [B, tiles, Hkv, bytes]
    B, N, K, _ = tiles.shape
    codes = tiles[..., : 16 * dim]
    codes = torch.stack([codes & 15, codes >> 4], -1)
    ck = codes[..., : 8 * dim, :].reshape(B, N, K, 16, dim)
    cv = codes[..., 8 * dim :, :].reshape(B, N, K, dim // 64, 8, 4, 4, 2, 2, 2)  # h g c m j1 j0 half
    cv = cv.permute(0, 1, 2, 8, 5, 7, 3, 6, 9, 4).reshape(B, N, K, 16, dim)
    scales = tiles[..., 16 * dim :].contiguous().view(dtype).float().view(B, N, K, 2, 16, 2)
    k, v = (scales[..., x, :, 1:] + scales[..., x, :, :1] * c for x, c in ((0, ck), (1, cv)))
    k, v = (x.transpose(2, 3).reshape(B, N * 16, K, dim) for x in (k, v))
    held = (torch.arange(N * 16, device=k.device) < s["lens"][:, None]).view(B, -1, 1, 1)
    out = _attend(_padded(s["q"], s["cu"], s["longest"]), k, torch.where(held, v, 0.0), s["cu"][1:] - s["cu"][:-1], s["lens"])
    return out[_seq_of(s["cu"], s["q"].shape[0])].to(dtype)


def _places(s, cu, n):
    """Byte offsets in the flat pages of the last tokens of each sequence: of K's codes, V's codes, both's scales."""
    _, kv, tiles, size = s["pages"].shape
    dim = (size - 128) // 16
    seq, i = _seq_of(cu, n)
    pos = s["lens"][seq] - (cu[1:] - cu[:-1])[seq] + i
    page = s["table"][seq, pos // (16 * tiles)].long()
    tile = (page[:, None] * kv + torch.arange(kv, device=pos.device)) * tiles + (pos // 16 % tiles)[:, None]
    t, base = (pos % 16)[:, None, None], (tile * size)[..., None]
    b = torch.arange(dim // 2, device=pos.device)  # (h, g, m) of V's bytes
    h, g, m = b // 32, b // 4 % 8, b % 4
    at_v = (((h * 8 + g) * 4 + t % 8 // 2) * 4 + m) * 4 + t % 2 * 2 + t // 8
    four = torch.arange(4, device=pos.device) + 4 * t
    return base + t * (dim // 2) + b, base + 8 * dim + at_v, base + 16 * dim + four, base + 16 * dim + 64 + four


def _plain_append(s):
    flat, dtype, dim = s["pages"].view(-1), s["dtype"], s["k"].shape[2]
    at_k, at_v, at_sk, at_sv = _places(s, s["cu"], s["k"].shape[0])
    (ck, sk, zk), (cv, sv, zv) = _codes(s["k"]), _codes(s["v"])
    flat[at_k] = ck[..., 0::2] | ck[..., 1::2] << 4
    pair = cv.view(*cv.shape[:2], dim // 64, 4, 2, 8).transpose(3, 5)  # h g half m
    flat[at_v] = (pair[..., 0, :] | pair[..., 1, :] << 4).flatten(2)
    flat[at_sk] = torch.stack([sk, zk], -1).view(torch.uint8)
    flat[at_sv] = torch.stack([sv, zv], -1).view(torch.uint8)
    at_k, at_v, at_sk, at_sv = _places(s, s["cu_read"], s["tokens"])
    k = torch.stack([flat[at_k] & 15, flat[at_k] >> 4], -1).flatten(2).float()
    v = flat[at_v]
    v = torch.stack([v & 15, v >> 4], -1).view(v.shape[0], v.shape[1], dim // 64, 8, 4, 2)  # h g m half
    v = v.permute(0, 1, 2, 4, 5, 3).reshape(k.shape).float()
    sk, sv = (flat[a].view(dtype).float() for a in (at_sk, at_sv))
    return (sk[..., 1:] + sk[..., :1] * k).to(dtype), (sv[..., 1:] + sv[..., :1] * v).to(dtype)


def _plain_score(s):
    x = s["logits"].float()
    vocab = x.shape[1]
    top = x.amax(1, keepdim=True)
    e = (x - top).exp()
    total = e.sum(1, keepdim=True)
    log = total.log()
    given = x.gather(1, s["tokens"][:, None])
    entropy = (log - (torch.where(e > 0, x - top, 0.0) * e).sum(1, keepdim=True) / total)[:, 0]
    rank = ((x > given).sum(1) + 1).to(torch.int32)
    bits = (x + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -1 - (bits & 0x7FFFFFFF), bits)  # as the values are ordered
    order = order * 2**32 + (vocab - 1 - torch.arange(vocab, device=x.device))  # of equal values the first
    ids = vocab - 1 - (order.topk(s["top"], 1).values & 0xFFFFFFFF)
    return (given - top - log)[:, 0], rank, entropy, ids.to(torch.int32), x.gather(1, ids) - top - log


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "score":
        x = state["logits"].double()
        lp = x - torch.logsumexp(x, 1, keepdim=True)
        p = lp.exp()
        entropy = -(p * lp).sum(1)
        best = lp.sort(dim=1, descending=True, stable=True)
        return (lp[torch.arange(x.shape[0]), state["tokens"]], None, entropy, None, best.values[:, : case["top"]])
    new, total = _lens(case)
    if case["op"] == "append":
        _, _, _, k, v = _cache_content(case, seed)
        at = _rows_of(total, new)
        k[at], v[at] = state["k"], state["v"]
        if not case["read_all"]:
            k, v = k[at], v[at]
        return _stand_for(k), _stand_for(v)
    if case["op"] == "cache":
        _, _, _, k, v = _cache_content(case, seed)
        k, v = _stand_for(k), _stand_for(v)
    else:
        k, v = state["k"].double(), state["v"].double()
    q, out = state["q"].double(), []
    group = case["heads"] // case["kv_heads"]
    a = b = 0
    for n, t in zip(new, total):
        qs, ks, vs = q[a : a + n].transpose(0, 1), k[b : b + t].transpose(0, 1), v[b : b + t].transpose(0, 1)
        late = torch.ones(n, t, dtype=torch.bool, device="cuda").triu(t - n + 1)
        rows = []
        for h in range(case["heads"]):
            score = qs[h] @ ks[h // group].T / math.sqrt(case["dim"])
            rows.append(torch.softmax(score.masked_fill(late, -math.inf), 1) @ vs[h // group])
        out.append(torch.stack(rows, 1))
        a, b = a + n, b + t
    return torch.cat(out)


def _stand_for(x):
    """The values that 4-bit codes of x stand for, in 64 bits: the scale is the range's fifteenth in x's own type."""
    low, high = x.double().aminmax(dim=-1, keepdim=True)
    scale = ((high - low) / 15).to(x.dtype).double()
    return low + scale * torch.round((x.double() - low) / scale.clamp(min=1e-300)).clamp(0, 15)
