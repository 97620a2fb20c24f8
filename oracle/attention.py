"""CPU oracles, in 64 bits, of the operators around the LoRA projections:
the 4-bit cache's format, attention, and token log probabilities. Plain loops
over the formulas; nothing here is shared with the kernels."""

from __future__ import annotations

import math

import torch


def kv4_codes(x: torch.Tensor):
    """Codes [.., D] uint8, scale and zero [..] of x [.., D] (fp16 / bf16):
    the stated fp32 steps, each a single IEEE operation."""
    f = x.float()
    zero, high = f.amin(-1), f.amax(-1)
    scale = ((high - zero) * torch.tensor(1.0 / 15.0, dtype=torch.float32)).to(x.dtype)
    step = scale.float()[..., None]
    code = torch.where(step > 0, torch.round((f - zero[..., None]) / step), torch.zeros_like(f)).clamp(0, 15)
    return code.to(torch.uint8), scale, zero.to(x.dtype)


def kv4_values(x: torch.Tensor) -> torch.Tensor:
    """The values the codes of x stand for, in 64 bits."""
    code, scale, zero = kv4_codes(x)
    return zero.double()[..., None] + scale.double()[..., None] * code.double()


def kv4_tile(k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """The bytes of one tile: k and v [16, D]."""
    D = k.shape[1]
    out = torch.zeros(16 * D + 128, dtype=torch.uint8)
    (ck, sk, zk), (cv, sv, zv) = kv4_codes(k), kv4_codes(v)
    for t in range(16):
        for b in range(D // 2):
            out[t * (D // 2) + b] = int(ck[t, 2 * b]) | int(ck[t, 2 * b + 1]) << 4
        for d in range(D):
            if d % 16 < 8:
                h, m, g = d // 64, d // 16 % 4, d % 8
                c, j = t % 8 // 2, t % 2 * 2 + t // 8
                out[8 * D + (((h * 8 + g) * 4 + c) * 4 + m) * 4 + j] = int(cv[t, d]) | int(cv[t, d + 8]) << 4
    for i, (s, z) in enumerate(((sk, zk), (sv, zv))):
        out[16 * D + 64 * i:16 * D + 64 * (i + 1)] = torch.stack([s, z], 1).contiguous().view(torch.uint8).view(-1)
    return out


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float):
    """Causal attention of one sequence: q [n, H, D], k and v [t, K, D]; query
    i sees the keys j <= i + t - n. Returns (out [n, H, D], lse [n, H]) in 64
    bits; a row that sees nothing is 0 with lse -inf. Sums run over the
    visible keys only."""
    n, H, D = q.shape
    t, K = k.shape[0], k.shape[1]
    out = torch.zeros(n, H, D, dtype=torch.float64)
    lse = torch.full((n, H), -math.inf, dtype=torch.float64)
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    for i in range(n):
        m = i + t - n + 1
        if m <= 0:
            continue
        for h in range(H):
            s = k[:m, h * K // H] @ q[i, h] * scale
            lse[i, h] = torch.logsumexp(s, 0)
            out[i, h] = (s - lse[i, h]).exp() @ v[:m, h * K // H]
    return out, lse


def token_logprobs(x: torch.Tensor, tokens: torch.Tensor, top: int):
    """(logprob, rank, entropy, ids, top logprobs) of x [rows, vocab], in 64
    bits; rows that are all -inf: -inf, entropy 0."""
    x, tokens = x.double().cpu(), tokens.cpu().long()
    rows, vocab = x.shape
    empty = (x == -math.inf).all(1)
    below = x - x.amax(1, keepdim=True)  # first: log l would vanish beside a maximum of 1e38
    lp = below - below.exp().sum(1, keepdim=True).log()
    lp[empty] = -math.inf
    p = lp.exp()
    ent = -torch.where(p == 0, 0.0, p * lp).sum(1)
    ent[x.isnan().any(1) | (x == math.inf).any(1)] = math.nan
    inside = (tokens >= 0) & (tokens < vocab)
    at = tokens.clamp(0, vocab - 1)
    given = torch.where(inside, x[torch.arange(rows), at], -math.inf)
    got = torch.where(inside, lp[torch.arange(rows), at], torch.where(lp.isnan().any(1), math.nan, -math.inf))
    rank = (x > given[:, None]).sum(1) + 1
    order = torch.where(x.isnan(), math.inf, x)  # NaN above +inf: only used where no +inf is in the row
    ids = torch.sort(order, dim=1, descending=True, stable=True).indices[:, :top]
    return got, rank, ent, ids, torch.gather(lp, 1, ids)
