"""Llama-style decoder (RMSNorm, rotary positions, SwiGLU FFN, no biases), optionally tensor-parallel with
sequence parallelism.

Shapes of the 7B configuration named by the benchmark set: 32 layers, d_model 4096, 32 heads, FFN 11008,
vocab 32000, RoPE θ = 1e4, RMSNorm eps 1e-6. The building blocks follow the reference layers
(``RMSNorm``: ``crates/torsh-nn/src/layers/normalization/layer_group/mod.rs:491-514``; ``SwiGLU`` with the gate in
the second half: ``layers/activation/gated.rs:536-608``; ``RotaryPositionalEmbedding``: ``layers/embedding.rs:372-430``).
With a :class:`~torsh_b200.parallel.tensor_parallel.TPContext` the projections are Column/RowParallelLinear
(fused all-gather→GEMM and GEMM→reduce-scatter) and activations between blocks stay sharded along tokens.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from .. import nn
from ..ops import attention as attn_ops
from ..ops import elementwise as ew
from ..ops import kv_cache as kv_ops
from ..ops import linear as lin_ops
from ..ops import norm as norm_ops
from ..ops import rotary as rot_ops
from ..ops import softmax as sm_ops
from ..ops import speculative as spec_ops


@dataclass
class LlamaConfig:
    vocab_size: int = 32000
    hidden_size: int = 4096
    intermediate_size: int = 11008
    num_layers: int = 32
    num_heads: int = 32
    max_seq_len: int = 4096
    rope_theta: float = 10000.0
    rms_eps: float = 1e-6
    initializer_range: float = 0.02

    @classmethod
    def llama_7b(cls, **kw):
        return cls(**kw)

    @classmethod
    def tiny(cls, **kw):
        base = dict(vocab_size=1024, hidden_size=256, intermediate_size=768, num_layers=2, num_heads=4, max_seq_len=256)
        base.update(kw)
        return cls(**base)

    @property
    def head_dim(self):
        return self.hidden_size // self.num_heads

    @property
    def padded_vocab(self):
        return (self.vocab_size + 63) // 64 * 64


class _W(nn.Module):
    def __init__(self, n_out, n_in, std):
        super().__init__()
        self.weight = nn.Parameter(torch.empty(n_out, n_in).normal_(0.0, std))

    def forward(self, x, residual=None):
        return lin_ops.linear(x, self.weight, None, residual=residual)


class LlamaBlock(nn.Module):
    def __init__(self, cfg: LlamaConfig, tp=None):
        super().__init__()
        self.cfg, self.tp = cfg, tp
        E, F, std = cfg.hidden_size, cfg.intermediate_size, cfg.initializer_range
        self.world = tp.world if tp is not None else 1
        self.local_heads = cfg.num_heads // self.world
        self.input_norm = nn.RMSNorm(E, cfg.rms_eps)
        self.post_attn_norm = nn.RMSNorm(E, cfg.rms_eps)
        if tp is None:
            self.qkv, self.o = _W(3 * E, E, std), _W(E, E, std / math.sqrt(2 * cfg.num_layers))
            self.gate_up, self.down = _W(2 * F, E, std), _W(E, F, std / math.sqrt(2 * cfg.num_layers))
        else:
            from ..parallel.tensor_parallel import ColumnParallelLinear, RowParallelLinear
            # column-parallel outputs are laid out per rank as [q | k | v] of the local heads and [up | gate] of the
            # local FFN slice, so no re-shuffle is needed after the GEMM
            self.qkv = ColumnParallelLinear(E, 3 * E, bias=False, tp=tp, init_std=std)
            self.o = RowParallelLinear(E, E, bias=False, tp=tp, init_std=std / math.sqrt(2 * cfg.num_layers))
            self.gate_up = ColumnParallelLinear(E, 2 * F, bias=False, tp=tp, init_std=std)
            self.down = RowParallelLinear(F, E, bias=False, tp=tp, init_std=std / math.sqrt(2 * cfg.num_layers))

    def forward(self, x, B: int, S: int):
        """``x``: ``[B*S, E]`` (or this rank's ``[B*S/tp, E]`` token shard under TP+SP)."""
        cfg, H, D = self.cfg, self.local_heads, self.cfg.head_dim
        h, x = norm_ops.rms_norm_fork(x, self.input_norm.weight, cfg.rms_eps)
        qkv = self.qkv(h)                                        # [B*S, 3*H*D] (all tokens, local heads)
        ctx = attn_ops.rope_flash_attention_qkvpacked(qkv, B, S, H, D, cfg.rope_theta)
        x = self.o(ctx, residual=x)
        h, x = norm_ops.rms_norm_fork(x, self.post_attn_norm.weight, cfg.rms_eps)
        return self.down(ew.swiglu(self.gate_up(h)), residual=x)

    def step(self, x, B: int, T: int, cache, layer: int, positions, freqs, tree_mask=None, counts=None):
        """``T`` new tokens per sequence on top of ``cache`` (:class:`~torsh_b200.ops.kv_cache.PagedKVCache`), which gets their keys and values."""
        cfg, H, D = self.cfg, self.local_heads, self.cfg.head_dim
        h = norm_ops.rms_norm(x, self.input_norm.weight, cfg.rms_eps)
        qkv = self.qkv(h).view(B, T, 3, H, D)
        q, k = rot_ops.rotary(qkv[:, :, 0], qkv[:, :, 1], positions, freqs)
        cache.write(layer, k, qkv[:, :, 2], counts)
        x = self.o(cache.attend(layer, q, tree_mask, counts).reshape(B * T, H * D), residual=x)
        h = norm_ops.rms_norm(x, self.post_attn_norm.weight, cfg.rms_eps)
        return self.down(ew.swiglu(self.gate_up(h)), residual=x)


class LlamaModel(nn.Module):
    """Whole model, or one pipeline stage of it (``layer_range``; first stage owns the embedding, last stage the
    final norm and the LM head)."""

    def __init__(self, cfg: LlamaConfig, tp=None, layer_range: range | None = None, first_stage: bool = True,
                 last_stage: bool = True, vocab_parallel: bool = False):
        super().__init__()
        self.cfg, self.tp, self.first_stage, self.last_stage = cfg, tp, first_stage, last_stage
        # vocab_parallel: the LM head is split over the tensor-parallel ranks by vocabulary rows (column-parallel
        # linear fed by the token shards) and the loss is computed without gathering the logits; otherwise every
        # rank computes all logits from the gathered hidden states
        self.vocab_parallel = bool(vocab_parallel and tp is not None and tp.world > 1)
        layers = layer_range if layer_range is not None else range(cfg.num_layers)
        if first_stage:
            w = torch.zeros(cfg.padded_vocab, cfg.hidden_size)
            w[: cfg.vocab_size].normal_(0.0, cfg.initializer_range)
            self.embed = nn.Parameter(w)
        self.layers = nn.ModuleList([LlamaBlock(cfg, tp) for _ in layers])
        if last_stage:
            self.norm = nn.RMSNorm(cfg.hidden_size, cfg.rms_eps)
            if self.vocab_parallel:
                from ..parallel.tensor_parallel import ColumnParallelLinear
                vp = (cfg.vocab_size + 128 * tp.world - 1) // (128 * tp.world) * (128 * tp.world)
                self.lm_head_tp = ColumnParallelLinear(cfg.hidden_size, vp, bias=False, tp=tp, init_std=cfg.initializer_range)
            else:
                w = torch.zeros(cfg.padded_vocab, cfg.hidden_size)
                w[: cfg.vocab_size].normal_(0.0, cfg.initializer_range)
                self.lm_head = nn.Parameter(w)

    def replicated_parameters(self):
        """Parameters every tensor-parallel rank holds in full but feeds with its own token shard (norm weights, the
        embedding): their gradients are partial sums and must be all-reduced over the TP group."""
        out = [p for n, p in self.named_parameters() if "norm" in n]
        if self.first_stage:
            out.append(self.embed)
        return out

    def _shard_tokens(self, x):
        if self.tp is None or self.tp.world == 1:
            return x
        rows = x.shape[0] // self.tp.world
        return x[self.tp.rank * rows:(self.tp.rank + 1) * rows].contiguous()

    def forward(self, inp: torch.Tensor, B: int | None = None, S: int | None = None, targets: torch.Tensor | None = None):
        """First stage: ``inp`` = token ids ``[B, S]``. Later stages: hidden states from the previous stage."""
        if self.first_stage:
            B, S = inp.shape
            x = self._shard_tokens(ew.embedding(inp, self.embed).reshape(B * S, -1))
        else:
            x = inp
        for blk in self.layers:
            x = blk(x, B, S)
        if not self.last_stage:
            return x
        return self.head(x, B, S, targets)

    def head(self, x, B: int, S: int, targets: torch.Tensor | None = None):
        """Final norm + LM head (+ fused cross-entropy when ``targets`` is given) on the last stage's hidden states."""
        h = norm_ops.rms_norm(x, self.norm.weight, self.cfg.rms_eps)
        if self.vocab_parallel:
            from ..parallel.tensor_parallel import _gather_cols, vocab_parallel_cross_entropy
            logits_local = self.lm_head_tp(h)                       # [B*S, V/tp]: all tokens, this rank's vocabulary rows
            if targets is None:
                full = torch.cat(_gather_cols(logits_local, self.tp.group), -1)
                return full.view(B, S, -1)[..., : self.cfg.vocab_size]
            return vocab_parallel_cross_entropy(logits_local, targets, self.tp.group, self.cfg.vocab_size)
        if self.tp is not None and self.tp.world > 1:
            from ..parallel.tensor_parallel import _AllGatherRowsReplicated
            h = _AllGatherRowsReplicated.apply(h, self.tp.group)
        logits = lin_ops.linear(h, self.lm_head, None)
        if targets is None:
            return logits.view(B, S, -1)[..., : self.cfg.vocab_size]
        return sm_ops.cross_entropy(logits, targets.reshape(-1), num_classes=self.cfg.vocab_size)

    # ------------------------------------------------------------------------------------------------ generation
    def make_cache(self, batch: int, max_len: int, dtype: torch.dtype | None = None, page: int = 64):
        """A cache for ``batch`` sequences of up to ``max_len`` tokens; ``dtype`` is the weights' unless given (int8 and float8_e4m3fn hold half)."""
        cfg = self.cfg
        return kv_ops.PagedKVCache(len(self.layers), cfg.num_heads, cfg.head_dim, batch, max_len, dtype or self.embed.dtype, page, device=self.embed.device)

    @torch.no_grad()
    def decode(self, tokens: torch.Tensor, cache, tree_mask: torch.Tensor | None = None, counts: torch.Tensor | None = None):
        """Hidden states ``[B * T, E]`` (after the final norm) of ``T`` new tokens per sequence on top of the cache, which gets their keys
        and values; its lengths stay (:meth:`~torsh_b200.ops.kv_cache.PagedKVCache.advance` keeps them). With ``tree_mask`` a token's
        position is its depth in the tree."""
        if not (self.first_stage and self.last_stage) or self.tp is not None:
            raise NotImplementedError("LlamaModel.decode: the whole model on one device")
        B, T = tokens.shape
        if not hasattr(self, "_rotary_freqs") or self._rotary_freqs.device != tokens.device:
            self._rotary_freqs = rot_ops.rotary_frequencies(self.cfg.head_dim, self.cfg.rope_theta, device=tokens.device)[0]
        depth = torch.arange(T, device=tokens.device) if tree_mask is None else tree_mask.sum(-1) - 1
        positions = cache.lengths.long()[:, None] + depth
        x = ew.embedding(tokens, self.embed).reshape(B * T, -1)
        for i, blk in enumerate(self.layers):
            x = blk.step(x, B, T, cache, i, positions, self._rotary_freqs, tree_mask, counts)
        return norm_ops.rms_norm(x, self.norm.weight, self.cfg.rms_eps)

    def _probs(self, h, temperature: float):
        """fp32 probabilities ``[rows, V]`` of the next token; all on the likeliest one at temperature 0."""
        logits = lin_ops.linear(h, self.lm_head, None)[:, : self.cfg.vocab_size].float()
        if temperature == 0:
            return torch.zeros_like(logits).scatter_(1, logits.argmax(-1, keepdim=True), 1.0)
        warm = logits / temperature
        # where that is out of range, from the largest on: infinity less infinity is no number
        cold = (logits - logits.amax(-1, keepdim=True)) / max(temperature, torch.finfo(torch.float32).tiny)
        return torch.softmax(torch.where(warm.amax(-1, keepdim=True).isfinite(), warm, cold), -1)

    @torch.no_grad()
    def generate(self, input_ids: torch.Tensor, max_new_tokens: int, temperature: float = 0.0, draft: "LlamaModel | None" = None, drafted: int = 4,
                 cache_dtype: torch.dtype | None = None, generator: torch.Generator | None = None) -> torch.Tensor:
        """``input_ids [B, S]`` and ``max_new_tokens`` more tokens each, from a cache of keys and values instead of running the context again.

        With ``draft`` (a smaller model over the same vocabulary) each round drafts ``drafted`` tokens and verifies them in one pass of this
        model (:func:`~torsh_b200.ops.speculative.verify_draft`): the tokens are distributed as without it, and the same at temperature 0
        up to the rounding of sums over different numbers of rows. Raises where this model's probabilities are no numbers; a draft's that are none
        are never accepted."""
        if not temperature >= 0:
            raise ValueError("generate: temperature is not negative")
        if draft is not None and (draft.cfg.vocab_size != self.cfg.vocab_size or drafted < 1):
            raise ValueError("generate: the draft model has the same vocabulary, and drafts at least one token")
        B, S = input_ids.shape
        if B == 0 or S == 0 or max_new_tokens <= 0:
            return input_ids
        dev = input_ids.device
        room = S + max_new_tokens + (drafted if draft is not None else 0)
        rand = lambda *s: torch.rand(*s, device=dev, generator=generator)   # noqa: E731
        models = [self] if draft is None else [self, draft]
        caches = [m.make_cache(B, room + 1, cache_dtype) for m in models]
        for m, c in zip(models, caches):            # all of the prompt but its last token, which the first step feeds
            if S > 1:
                c.reserve(S - 1)
                m.decode(input_ids[:, :-1], c)
                c.advance(S - 1)
        done = [input_ids[b].tolist() for b in range(B)]
        last = input_ids[:, -1:]
        while min(len(d) for d in done) < S + max_new_tokens:
            T = 1 if draft is None else drafted + 1
            tokens, q = last, []
            if draft is not None:
                c = caches[1]
                c.reserve(T)
                for _ in range(drafted):            # one token more than is drafted: its keys are needed where all are accepted
                    p = draft._probs(draft.decode(tokens[:, -1:], c), temperature)
                    c.advance(1)
                    nxt = spec_ops.verify_draft(p[:, None], tokens[:, -1:], rand(B, 1))[2].clamp(min=0)   # none: a token that is refused below
                    tokens, q = torch.cat([tokens, nxt[:, None]], 1), q + [p]
                draft.decode(tokens[:, -1:], c)
                c.advance(1)
            caches[0].reserve(T)
            probs = self._probs(self.decode(tokens, caches[0]), temperature).view(B, T, -1)
            taken, _, nxt = spec_ops.verify_draft(probs, tokens, rand(B, T), torch.stack(q, 1) if q else None)
            took, follow = taken.tolist(), nxt.tolist()
            if min(follow) < 0:
                raise RuntimeError("generate: the model's probabilities are no numbers")
            caches[0].advance([n + 1 for n in took])
            for b, (n, more) in enumerate(zip(took, torch.cat([tokens[:, 1:], nxt[:, None]], 1).tolist())):
                done[b] += more[:n] + more[-1:]
            if draft is not None:
                caches[1].truncate(caches[0].host_lengths)
            last = nxt[:, None]
            full = [b for b in range(B) if len(done[b]) >= S + max_new_tokens]
            for b in full:                          # sequences that are done stay where they are: no room beyond is asked for
                keep = min(caches[0].host_lengths[b], S + max_new_tokens - 1)
                for c in caches:
                    c.truncate([keep if i == b else n for i, n in enumerate(c.host_lengths)])
        return torch.tensor([d[: S + max_new_tokens] for d in done], dtype=input_ids.dtype, device=dev)


LlamaForCausalLM = LlamaModel
