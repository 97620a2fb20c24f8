"""Multi-tenant draft step: a small decoder whose LoRA projections run the
grouped apply over an AdapterPool.

The reference's draft-side integration wraps a draft model's linears so that
every tenant's draft-LoRA is applied to the whole batch in one pass per layer
(BGMVLoRALinear / wrap_draft, benchmarks/e2e/serve_multitenant.py:56-120)
and captures the draft step in a CUDA graph (benchmarks/kernel/
bench_graph_capture.py:47-103). Here the base linears are plain GEMMs and
each projection's LoRA is one add_lora call of this library on the pool's
stacked slots; the step's segment table (tokens sorted by tenant) is built
once per step and shared by all 7 x layers calls.

DraftDecoder is random-init (no checkpoint): RMSNorm, multi-head attention
over each sequence's lookahead tokens (causal), SwiGLU MLP, an optional LM
head. `lora="pool"` uses the library, `lora="torch"` a plain-torch per-token
gather of the same adapters (the stock path the grouped apply replaces, for
comparison and tests), `lora="none"` the base model alone.

DraftSession serves a batch with it: prompts of different lengths (packed
attention), their K and V in 4-bit paged caches, drafted tokens over those
caches, and the log probabilities by which they are verified.
"""

from __future__ import annotations

import math
from typing import Callable, List, Optional

import torch
import torch.nn.functional as F

from .engine import TokenLogprobs, WarpPipeEngine
from .kvcache import KvCache4

PROJ_NAMES = ("q", "k", "v", "o", "gate", "up", "down")


class DraftDecoder:
    def __init__(self, layers: int = 12, hidden: int = 768, heads: int = 12, inter: int = 3072, vocab: int = 0,
                 device="cuda", dtype=torch.bfloat16, seed: int = 0):
        self.layers, self.hidden, self.heads, self.inter, self.vocab = layers, hidden, heads, inter, vocab
        self.dtype = dtype
        g = torch.Generator(device=device).manual_seed(seed)

        def w(o, i):
            return (torch.randn(o, i, device=device, generator=g) * (1.0 / math.sqrt(i))).to(dtype)

        self.w = []
        for _ in range(layers):
            self.w.append({"q": w(hidden, hidden), "k": w(hidden, hidden), "v": w(hidden, hidden),
                           "o": w(hidden, hidden), "gate": w(inter, hidden), "up": w(inter, hidden),
                           "down": w(hidden, inter)})
        self.lm_head = w(vocab, hidden) if vocab else None

    def dims(self) -> List[tuple]:
        """(d_in, d_out) of the LoRA projections, in call order (layer-major)."""
        h, i = self.hidden, self.inter
        per = [(h, h), (h, h), (h, h), (h, h), (h, i), (h, i), (i, h)]
        return [p for _ in range(self.layers) for p in per]

    @staticmethod
    def _rms(x):
        xf = x.float()
        return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + 1e-6)).to(x.dtype)

    def forward(self, x: torch.Tensor, seq_len: int, lora: str = "none", pool=None, scale: float = 1.0,
                torch_lora: Optional[dict] = None, attention: Optional[Callable] = None,
                head: bool = True) -> torch.Tensor:
        """x [T, hidden] (T = sequences x seq_len, sequences adapter-sorted).
        lora "pool": pool.add_lora per projection (the segment table must be
        built for this step); "torch": torch_lora = {"ids": [T] adapter ids,
        "A": [p] -> [n_adapters, r, d], "B": [p] -> [n_adapters, o, r]}.
        attention(layer, q, k, v) -> [T, heads, head_dim] on packed q, k, v of
        that shape takes the place of the attention over each sequence's own
        seq_len tokens (seq_len is then not used). Logits where the decoder has
        an LM head; hidden states where it has none, or without `head`."""
        T, H = x.shape
        nh, hd = self.heads, H // self.heads

        def proj(p, name, inp, W):
            out = F.linear(inp, W)
            if lora == "pool":
                pool.add_lora(p, out, inp, scale)
            elif lora == "torch":
                ids = torch_lora["ids"]
                valid = (ids >= 0)
                A = torch_lora["A"][p][ids.clamp(min=0)]  # [T, r, d]
                B = torch_lora["B"][p][ids.clamp(min=0)]  # [T, o, r]
                h = torch.einsum("td,trd->tr", inp.float(), A.float()) * scale
                # H enters the expand in the weights' 16-bit type, as the
                # stock bgmv_expand and this library's kernels take it
                h = h.to(inp.dtype).float()
                d = torch.einsum("tr,tor->to", h, B.float()) * valid.unsqueeze(1)
                out = (out.float() + d).to(out.dtype)
            return out

        for li, L in enumerate(self.w):
            base = li * len(PROJ_NAMES)
            h = self._rms(x)
            q = proj(base + 0, "q", h, L["q"])
            k = proj(base + 1, "k", h, L["k"])
            v = proj(base + 2, "v", h, L["v"])
            if attention is not None:
                a = attention(li, q.view(T, nh, hd), k.view(T, nh, hd), v.view(T, nh, hd)).view(T, H)
            else:
                q = q.view(-1, seq_len, nh, hd).transpose(1, 2)
                k = k.view(-1, seq_len, nh, hd).transpose(1, 2)
                v = v.view(-1, seq_len, nh, hd).transpose(1, 2)
                a = F.scaled_dot_product_attention(q, k, v, is_causal=True)
                a = a.transpose(1, 2).reshape(T, H).contiguous()
            x = x + proj(base + 3, "o", a, L["o"])
            h2 = self._rms(x)
            g = proj(base + 4, "gate", h2, L["gate"])
            u = proj(base + 5, "up", h2, L["up"])
            m = (F.silu(g.float()) * u.float()).to(x.dtype).contiguous()
            x = x + proj(base + 6, "down", m, L["down"])
        x = self._rms(x)
        if head and self.lm_head is not None:
            return F.linear(x, self.lm_head)
        return x


class DraftSession:
    """A batch of sequences on a DraftDecoder, every layer's K and V in a 4-bit
    paged cache (KvCache4, one per layer over the same page table).

    Page tables, lengths and offsets are int32 CUDA tensors that the caller
    keeps (KvCache4 says what they hold); a decode step is graph-capturable.
    The LoRA arguments are DraftDecoder.forward's.

        h = session.prefill(x, cu, table, lens, max_q)        # the prompts
        h = session.decode(x, table, lens, cu, max_q)         # drafted tokens
        lp = session.score(h, tokens, top=5)                  # their log probabilities
    """

    def __init__(self, model: DraftDecoder, engine: WarpPipeEngine, num_pages: int, page_size: int = 64):
        self.model, self.engine = model, engine
        dim = model.hidden // model.heads
        device = model.w[0]["q"].device
        if device != engine.device:
            raise RuntimeError(f"DraftSession: the model is on {device}, the engine on {engine.device}")
        self.caches = [KvCache4(engine, num_pages, model.heads, dim, page_size, model.dtype) for _ in range(model.layers)]

    def prefill(self, x: torch.Tensor, cu, table, lens, max_q: int, context=None, **lora) -> torch.Tensor:
        """Prompts, or chunks of them: x [tokens, hidden] packed, cu their
        offsets, lens the lengths with these tokens included. Without context
        (whole prompts) a token attends to its prompt's K and V as computed;
        with context = (cu_all, tokens_all), the offsets and the total of the
        full lengths, to those that the cache stands for."""

        def attention(layer, q, k, v):
            cache = self.caches[layer]
            cache.append(k, v, table, lens, cu)
            if context is None:
                return self.engine.prompt_attention(q, k, v, cu, max_q=max_q)
            cu_all, total = context
            k_all, v_all = cache.read(table, lens, cu_all, total)
            return self.engine.prompt_attention(q, k_all, v_all, cu, cu_all, max_q=max_q)

        return self._hidden(x, attention, lora)

    def decode(self, x: torch.Tensor, table, lens, cu=None, max_q: int = 1, **lora) -> torch.Tensor:
        """The next tokens of every sequence (one each without cu; the drafted
        ones of a verification with it)."""

        def attention(layer, q, k, v):
            cache = self.caches[layer]
            cache.append(k, v, table, lens, cu)
            return cache.attention(q, table, lens, cu, max_q)

        return self._hidden(x, attention, lora)

    def _hidden(self, x, attention, lora):
        # hidden states: score() takes the logits it needs
        return self.model.forward(x, 0, attention=attention, head=False, **lora)

    def score(self, hidden: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogprobs:
        """Log probability, rank and entropy of a given token per hidden state,
        and the `top` alternatives."""
        if self.model.lm_head is None:
            raise RuntimeError("DraftSession.score: the model has no LM head (vocab=0)")
        return self.engine.token_logprobs(F.linear(hidden, self.model.lm_head), tokens, top)
