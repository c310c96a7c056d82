"""A Llama-shaped decoder stack around the LRQK cache, for end-to-end tokens/s.

Only the call pattern matters here: every layer calls ``cache.update(q, k, v, layer)`` exactly
as the reference's patched attention does (lrqk_attention.py:2254-2290, 2326-2344) -- raw K/V
and ordinary causal attention over the prompt, the active set ``[b,Hq,k+L,d]`` and exact
single-query attention per decoded token.  Projections, norms, rotary embedding, SwiGLU and the
prompt attention are plain PyTorch-ROCm library calls on random-initialised weights (rotary positions
that are scaled, interleaved or over caches in 8 bits: the HIP library's); the cache path (factorisation, selection, fetch, decode attention) is the HIP library.

``new_byte_caches`` gives a dense K/V cache in 8 bits instead, which ``generate`` takes as any other and
``generate_drafted`` decodes several looked-up tokens at once over (rotary positions, attention, verification and the
cache are the HIP library's there).

``cache=None`` runs the same module with a dense K/V cache; with ``k + lite`` at least as long as
the whole sequence the LRQK run returns every cached token (the growing-prefix branch,
lrqk_attention.py:1526-1545) and must produce the same tokens.
"""
from __future__ import annotations

import math
import time
from dataclasses import dataclass
from typing import List, Optional, Tuple

import torch
import torch.nn.functional as F

from . import ops
from .cache import DynamicLRQKCache


@dataclass
class DecoderConfig:
    layers: int = 32
    hidden: int = 4096
    heads: int = 32
    kv_heads: int = 8
    head_dim: int = 128
    intermediate: int = 14336
    vocab: int = 128256
    rope_theta: float = 5e5
    rms_eps: float = 1e-5
    rope_interleaved: bool = False           # pairs of neighbours; else halves
    rope_scaling: Optional[dict] = None      # as ops.RotaryPlan takes it


LLAMA3_8B = DecoderConfig()


def _rms(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    v = x.float()
    v = v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + eps)
    return (v * w.float()).to(x.dtype)


class ByteCaches:
    """A dense K/V cache in 8 bits: an ``ops.ByteCache`` a layer, and the lengths that they share (int32 [b])."""

    def __init__(self, cfg: DecoderConfig, batch: int, capacity: int, dtype, kind: str, device):
        self.layers = [ops.ByteCache(batch, cfg.kv_heads, capacity, cfg.head_dim, dtype, kind, device) for _ in range(cfg.layers)]
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)

    @property
    def capacity(self) -> int:
        return self.layers[0].capacity


class LookedUp:
    """A sequence's tokens, and where every ``ngram`` of them ended the last time."""

    def __init__(self, tokens: List[int], ngram: int):
        self.tokens, self.ngram, self._ends, self._done = list(tokens), ngram, {}, ngram

    def drafts(self, n: int) -> List[int]:
        """n tokens: those that followed the last ``ngram`` where they stood before, the last time that they did; -1: nothing."""
        for end in range(self._done, len(self.tokens)):
            self._ends[tuple(self.tokens[end - self.ngram:end])] = end
        self._done = max(self._done, len(self.tokens))
        end = self._ends.get(tuple(self.tokens[-self.ngram:]), len(self.tokens))
        found = self.tokens[end:end + n]
        return found + [-1] * (n - len(found))


class LlamaShapeDecoder:
    def __init__(self, cfg: DecoderConfig = LLAMA3_8B, dtype=torch.bfloat16, device="cuda:0", seed: int = 0,
                 mlp_chunk: int = 16384, context_scale: float = 0.0):
        """``context_scale`` > 0 adds a fixed direction of that length (in units of an embedding's length) to every
        token embedding.  With random weights and random ids the hidden states of successive positions are
        unrelated, so every decode step selects a fresh set of tokens; a shared component makes successive
        queries (and all keys) correlated, as the residual stream of a trained model does, and the selection then
        drifts slowly from step to step -- the regime the cache is built for."""
        self.cfg, self.dtype, self.device = cfg, dtype, torch.device(device)
        self.mlp_chunk = mlp_chunk
        self.context_scale = context_scale
        g = torch.Generator(device=self.device).manual_seed(seed)

        def w(*shape, std=0.02):
            return (torch.randn(shape, generator=g, device=self.device, dtype=torch.float32) * std).to(dtype)

        c = cfg
        self.embed = w(c.vocab, c.hidden)
        ctx = torch.randn((c.hidden,), generator=g, device=self.device, dtype=torch.float32)
        self.context = (ctx / ctx.norm() * (0.02 * math.sqrt(c.hidden)) * context_scale).to(dtype)
        self.lm_head = w(c.hidden, c.vocab)
        self.final_norm = torch.ones(c.hidden, dtype=dtype, device=self.device)
        self.layers = []
        for _ in range(c.layers):
            self.layers.append(dict(
                n1=torch.ones(c.hidden, dtype=dtype, device=self.device),
                n2=torch.ones(c.hidden, dtype=dtype, device=self.device),
                wq=w(c.hidden, c.heads * c.head_dim), wk=w(c.hidden, c.kv_heads * c.head_dim),
                wv=w(c.hidden, c.kv_heads * c.head_dim), wo=w(c.heads * c.head_dim, c.hidden),
                wg=w(c.hidden, c.intermediate), wu=w(c.hidden, c.intermediate), wd=w(c.intermediate, c.hidden)))
        half = c.head_dim // 2
        self.inv_freq = 1.0 / (c.rope_theta ** (torch.arange(0, half, device=self.device, dtype=torch.float32) / half))
        self.rope = None   # (else the library turns q and k, in one launch)
        if c.rope_interleaved or c.rope_scaling is not None:
            self.rope = ops.RotaryPlan(c.head_dim, c.rope_theta, c.rope_interleaved, c.rope_scaling, self.device)
        self._byte_plan = self.rope   # over caches in 8 bits, whose sequences have positions of their own
        self.ws = ops.Workspace()
        self.dense: Optional[List[Tuple[torch.Tensor, torch.Tensor]]] = None
        self.progress = None   # optional callable(str), called once per layer while the prompt is processed
        self.path_events = None  # a list: decode steps append an event pair around each layer's cache path

    # ------------------------------------------------------------------ pieces
    def _rope(self, x: torch.Tensor, pos0: int) -> torch.Tensor:
        """x [b,H,s,d]; rotate-half convention, positions pos0 .. pos0+s-1."""
        s, d = x.shape[2], x.shape[3]
        ang = torch.arange(pos0, pos0 + s, device=x.device, dtype=torch.float32)[:, None] * self.inv_freq[None, :]
        cos, sin = torch.cos(ang), torch.sin(ang)
        x1, x2 = x[..., :d // 2].float(), x[..., d // 2:].float()
        return torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], dim=-1).to(x.dtype)

    def _rotary_plan(self) -> ops.RotaryPlan:
        """Of prompts, tokens and drafts over caches in 8 bits alike (at 100K ``_rope``'s angles in fp32 are off by up to 4e-3)."""
        if self._byte_plan is None:
            self._byte_plan = ops.RotaryPlan(self.cfg.head_dim, self.cfg.rope_theta, device=self.device)
        return self._byte_plan

    def _mlp(self, L, x: torch.Tensor) -> torch.Tensor:
        out = torch.empty_like(x)
        flat, oflat = x.view(-1, x.shape[-1]), out.view(-1, x.shape[-1])
        for i in range(0, flat.shape[0], self.mlp_chunk):
            t = flat[i:i + self.mlp_chunk]
            oflat[i:i + self.mlp_chunk] = (F.silu(t @ L["wg"]) * (t @ L["wu"])) @ L["wd"]
        return out

    def new_cache(self, r=32, num_active_tokens=2048, lite_tokens=64, max_iter=(2, 2), tol=(1e-2, 1e-2),
                  max_sequence_length=4096) -> DynamicLRQKCache:
        return DynamicLRQKCache(r=r, num_active_tokens=num_active_tokens, lite_tokens=lite_tokens, max_iter=max_iter,
                                tol=tol, max_sequence_length=max_sequence_length,
                                num_key_value_groups=self.cfg.heads // self.cfg.kv_heads)

    def new_byte_caches(self, batch: int, capacity: int, kind: str = "int8") -> ByteCaches:
        """``kind`` as ``ops.ByteCache`` takes it; ``capacity``: tokens of a sequence, the generated ones among them."""
        return ByteCaches(self.cfg, batch, capacity, self.dtype, kind, self.device)

    # ------------------------------------------------------------------ one forward over s new positions
    @torch.inference_mode()
    def forward(self, ids: torch.Tensor, pos0: int, cache: Optional[DynamicLRQKCache]) -> torch.Tensor:
        """ids [b,s] -> logits of the last position [b,vocab].  pos0: the first one's position (0 begins anew; over caches in 8 bits
        a token stands behind what its sequence has, which ``generate_drafted`` may leave different: then that of the longest)."""
        c = self.cfg
        b, s = ids.shape
        rope, where = self.rope, pos0
        x = self.embed[ids]
        if self.context_scale:
            x = x + self.context
        if cache is None and self.dense is None:
            self.dense = [None] * c.layers
        if isinstance(cache, ByteCaches):
            if pos0 + s > cache.capacity or (s > 1 and pos0 > 0):
                raise ValueError(f"tokens {pos0} .. {pos0 + s - 1}: the cache has room for {cache.capacity}, and a prompt comes at once")
            rope = self._rotary_plan()
            if pos0 == 0:
                cache.lengths = torch.zeros_like(cache.lengths)
            else:
                where = cache.lengths[:, None]
        for li, L in enumerate(self.layers):
            hcur = _rms(x, L["n1"], c.rms_eps)
            q = (hcur @ L["wq"]).view(b, s, c.heads, c.head_dim).transpose(1, 2)
            k = (hcur @ L["wk"]).view(b, s, c.kv_heads, c.head_dim).transpose(1, 2)
            v = (hcur @ L["wv"]).view(b, s, c.kv_heads, c.head_dim).transpose(1, 2).contiguous()
            if rope is None:
                q, k = self._rope(q, pos0).contiguous(), self._rope(k, pos0).contiguous()
            else:
                q, k = ops.rotary(rope, q, k, where)
            if cache is None:
                if self.dense[li] is None:
                    self.dense[li] = (k, v)
                else:
                    self.dense[li] = (torch.cat([self.dense[li][0], k], 2), torch.cat([self.dense[li][1], v], 2))
                K, V = self.dense[li]
                o = F.scaled_dot_product_attention(q, K, V, is_causal=s > 1, enable_gqa=True)
            elif isinstance(cache, ByteCaches):
                seen = ops.byte_append(cache.layers[li], k, v, cache.lengths)
                if s > 1:
                    o = F.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=True)
                else:
                    o = ops.byte_attention(q, cache.layers[li], seen)
                if li == c.layers - 1:
                    cache.lengths = seen
            elif s > 1:
                cache.update(q, k, v, li)   # factorises the prompt; the prompt itself attends densely
                o = F.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=True)
            else:
                eng = cache.lwattn[li]
                eng.attn_in_step = True
                eng.last_attn = None
                if self.path_events is not None:
                    e0 = torch.cuda.Event(enable_timing=True)
                    e0.record()
                K, V = cache.update(q, k, v, li)
                if eng.last_attn is not None:
                    o = eng.last_attn
                else:   # prefix / edge branches return a view of the first n slots of the persistent buffers
                    o = ops.attention(self.ws, q, eng.Kgpu, eng.Vgpu, n_valid=K.shape[2])
                if self.path_events is not None:
                    e1 = torch.cuda.Event(enable_timing=True)
                    e1.record()
                    self.path_events.append((e0, e1))
            x = x + o.transpose(1, 2).reshape(b, s, c.heads * c.head_dim) @ L["wo"]
            x = x + self._mlp(L, _rms(x, L["n2"], c.rms_eps))
            if s > 1 and self.progress is not None:
                self.progress(f"prompt: layer {li + 1}/{c.layers}")
        last = _rms(x[:, -1], self.final_norm, c.rms_eps)
        return (last @ self.lm_head).float()

    @torch.inference_mode()
    def generate(self, ids: torch.Tensor, new_tokens: int, cache: Optional[DynamicLRQKCache]):
        """Greedy decoding.  Returns (tokens [b,new_tokens], prefill seconds, decode seconds, per-step seconds)."""
        self.dense = None
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        tok = self.forward(ids, 0, cache).argmax(-1)
        torch.cuda.synchronize()
        t_prefill = time.perf_counter() - t0
        out = [tok]
        steps = []
        pos = ids.shape[1]
        t0 = time.perf_counter()
        for _ in range(new_tokens - 1):
            t1 = time.perf_counter()
            tok = self.forward(tok[:, None], pos, cache).argmax(-1)
            out.append(tok)
            pos += 1
            steps.append(time.perf_counter() - t1)
        torch.cuda.synchronize()
        t_decode = time.perf_counter() - t0
        return torch.stack(out, 1), t_prefill, t_decode, steps

    # ------------------------------------------------------------------ several drafted tokens at once
    @torch.inference_mode()
    def _draft_logits(self, ids: torch.Tensor, mask: torch.Tensor, positions: torch.Tensor, caches: ByteCaches):
        """ids [b,s] of which token i sees the cached ones and those of mask [s,s] -> logits of every position [b,s,vocab], and k, v
        of every layer, which go into the cache once it is known which tokens stay."""
        c = self.cfg
        b, s = ids.shape
        plan = self._rotary_plan()
        x = self.embed[ids]
        if self.context_scale:
            x = x + self.context
        rows = []
        for L, layer in zip(self.layers, caches.layers):
            hcur = _rms(x, L["n1"], c.rms_eps)
            q = (hcur @ L["wq"]).view(b, s, c.heads, c.head_dim).transpose(1, 2)
            k = (hcur @ L["wk"]).view(b, s, c.kv_heads, c.head_dim).transpose(1, 2)
            v = (hcur @ L["wv"]).view(b, s, c.kv_heads, c.head_dim).transpose(1, 2)
            q, k = ops.rotary(plan, q, k, positions)
            o = ops.byte_attention(q, layer, caches.lengths, k, v, mask)
            rows.append((k, v))
            x = x + o.transpose(1, 2).reshape(b, s, c.heads * c.head_dim) @ L["wo"]
            x = x + self._mlp(L, _rms(x, L["n2"], c.rms_eps))
        return (_rms(x, self.final_norm, c.rms_eps) @ self.lm_head).float(), rows

    @torch.inference_mode()
    def generate_drafted(self, ids: torch.Tensor, new_tokens: int, caches: ByteCaches, drafts: int = 7, ngram: int = 2,
                         temperature: float = 0.0, generator: Optional[torch.Generator] = None):
        """Decoding with drafts that are looked up in the sequence itself: a round attends with a sequence's last token and up to
        ``drafts`` that followed its last ``ngram`` tokens before, verifies them against the model's probabilities (of
        ``temperature``; 0: its most probable token) and keeps those that stand.  A round's tokens have the distribution that its own
        logits give, token after token as without drafts.  Those of ``generate``, which is greedy, are not the same to the last
        bit: products are rounded otherwise, and a block that a round completes is read as it came until the round is over, where
        ``generate`` reads it in 8 bits from its last token on.  ids [b,l] -> (tokens [b,new_tokens], rounds)."""
        b, l = ids.shape
        if drafts < 1 or ngram < 1 or new_tokens < 1 or temperature < 0:
            raise ValueError(f"drafts={drafts}, ngram={ngram}, new_tokens={new_tokens}, temperature={temperature}")
        if l + new_tokens + drafts > caches.capacity:
            raise ValueError(f"{l} + {new_tokens} tokens and {drafts} drafts beyond the cache's {caches.capacity}")

        def chances(logits):
            if temperature == 0.0:
                return torch.zeros_like(logits).scatter_(-1, logits.argmax(-1, keepdim=True), 1.0)
            return torch.softmax(logits / temperature, -1)

        def drawn(s):
            return torch.rand((b, s), generator=generator, device=self.device)
        first = chances(self.forward(ids, 0, caches))[:, None]
        _, _, token = ops.verify_drafts(torch.zeros((b, 1), dtype=torch.int32, device=self.device), first, drawn(1))
        told = [LookedUp(row + [t], ngram) for row, t in zip(ids.tolist(), token.tolist())]
        s = drafts + 1
        mask = torch.ones((s, s), dtype=torch.bool, device=self.device).tril()
        steps = torch.arange(s, dtype=torch.int32, device=self.device)
        rounds = 0
        while min(len(row.tokens) for row in told) < l + new_tokens:
            # (a sequence that has all its tokens goes along and keeps none)
            full = [len(row.tokens) >= l + new_tokens for row in told]
            asked = [row.tokens[-1:] + row.drafts(drafts) for row in told]
            nodes = torch.tensor(asked, dtype=torch.int32, device=self.device)
            logits, rows = self._draft_logits(nodes.clamp(min=0).long(), mask, caches.lengths[:, None] + steps, caches)
            path, counts, token = ops.verify_drafts(nodes, chances(logits), drawn(s))
            counts = torch.where(torch.tensor(full, device=self.device), torch.zeros_like(counts), counts)
            for layer, (k, v) in zip(caches.layers, rows):
                seen = ops.byte_append(layer, k, v, caches.lengths, counts, path)
            caches.lengths = seen
            for row, kept, n, t in zip(told, asked, counts.tolist(), token.tolist()):
                if n:
                    row.tokens += kept[1:n] + [t]
            rounds += 1
        return torch.tensor([row.tokens[l:l + new_tokens] for row in told], device=self.device), rounds
