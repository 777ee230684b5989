"""Verification of drafted tokens against the target's probabilities (speculative decoding).

Kernel: ``csrc/kernels/verify_draft.cu``; CPU tensors run the same rules in PyTorch. The reference samples one token at a time
(``crates/torsh-text/src/generation.rs``: ``TextSampler``); the tokens accepted here, and the one that follows, are distributed as
if they had been drawn that way.
"""
from __future__ import annotations

import torch

from .. import _native as nv

_MAX_NODES = 1024


def _check(probs, tokens, uniforms, draft_probs, parents, counts):
    if probs.dim() != 3 or probs.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("verify_draft: probs is [B, T, V] in fp32 or bf16")
    B, T, V = probs.shape
    if not 1 <= T <= _MAX_NODES or V < 1:
        raise ValueError(f"verify_draft: 1 to {_MAX_NODES} nodes a sequence and a vocabulary, got {T} and {V}")
    if V > 1 << 22:
        raise ValueError("verify_draft: at most 2^22 tokens in the vocabulary")
    if tokens.shape != (B, T) or uniforms.shape != (B, T):
        raise ValueError(f"verify_draft: tokens and uniforms are [{B}, {T}]")
    if tokens.is_floating_point() or not uniforms.is_floating_point():
        raise TypeError("verify_draft: tokens are integers, uniforms floating-point numbers in [0, 1)")
    if draft_probs is not None:
        if parents is not None:
            raise ValueError("verify_draft: a tree's candidates are fixed tokens: give parents or draft_probs, not both")
        if draft_probs.shape != (B, T - 1, V) or draft_probs.dtype != probs.dtype:
            raise ValueError(f"verify_draft: draft_probs is [{B}, {T - 1}, {V}] in the type of probs")
    if parents is not None and (parents.shape not in ((T,), (B, T)) or parents.is_floating_point()):
        raise ValueError(f"verify_draft: parents are integers, [{T}] or [{B}, {T}]")
    if counts is not None and (counts.shape != (B,) or counts.is_floating_point()):
        raise ValueError(f"verify_draft: counts are integers, [{B}]")
    at = probs.get_device()
    for t in (tokens, uniforms, draft_probs, parents, counts):
        if t is not None and t.get_device() != at:
            raise ValueError("verify_draft: all tensors are on one device")


def verify_draft(probs: torch.Tensor, tokens: torch.Tensor, uniforms: torch.Tensor, draft_probs: torch.Tensor | None = None,
                 parents: torch.Tensor | None = None, counts: torch.Tensor | None = None):
    """Which drafted tokens the target accepts, and the token that follows: ``(accepted [B], path [B, T], next_token [B])``, int64.

    Node 0 of a sequence is its last confirmed token, nodes ``1 .. T-1`` are drafted; ``probs[b, i]`` is the target's distribution
    after node ``i``, ``tokens[b, i]`` the node's token (``tokens[:, 0]`` is not looked at). ``uniforms`` are the random numbers.

    * with ``draft_probs`` (``[B, T-1, V]``, what each token of a chain was drawn from) node ``i + 1`` is accepted while
      ``uniforms[b, i] * q < p``; after a refusal the next token is drawn from ``max(p - q, 0)``
    * without, the candidates are fixed: a chain, or the tree that ``parents`` gives (``[T]`` or ``[B, T]``, ``parents[i] < i``).
      The children of node ``i`` share ``uniforms[b, i]`` and take, in index order, intervals of their probabilities; where the number
      falls into none, the next token is drawn from the other tokens

    ``accepted`` counts the drafted tokens on the accepted path, ``path`` holds its nodes from node 0 on, padded with -1. The next
    token inverts the cumulative sum at ``uniforms[b, T-1]``, in 64 bits. ``counts`` (``[B]``, at least 1) says how many nodes of
    a sequence there are. Tokens outside the vocabulary and parents that do not come before their node are never accepted;
    a NaN or a negative number counts as no probability; where nothing has any, ``next_token`` is -1.
    """
    if probs.is_cuda:
        out = (nv._decode or nv.decode_calls()).verify(probs, tokens, uniforms, draft_probs, parents, counts)
        if out is not None:
            return out
    # not as the kernel takes it: refused, converted, or computed here
    _check(probs, tokens, uniforms, draft_probs, parents, counts)
    if probs.is_cuda:
        rows = lambda x: x if x is None or x.stride(2) == 1 else x.contiguous()   # noqa: E731
        as_ = lambda x, t: x if x is None else x.to(t).contiguous()   # noqa: E731
        with torch.cuda.device(probs.device):
            out = nv.decode_calls().verify(rows(probs), as_(tokens, torch.int64), as_(uniforms, torch.float32), rows(draft_probs), as_(parents, torch.int64),
                                           None if counts is None else counts.clamp(1, probs.shape[1]).to(torch.int32).contiguous())
        if out is not None:
            return out
    return _verify_plain(probs, tokens, uniforms, draft_probs, parents, counts)


def _verify_plain(probs, tokens, uniforms, draft_probs=None, parents=None, counts=None):
    """One sequence after the other in fp64; the CPU path and the test oracle."""
    B, T, V = probs.shape
    took, paths, nexts = [], [], []
    clean = lambda row: torch.where(row > 0, row, torch.zeros_like(row))   # noqa: E731  negative and NaN: no probability
    for b in range(B):
        n = T if counts is None else min(max(int(counts[b]), 1), T)
        par = list(range(-1, T - 1)) if parents is None else (parents if parents.dim() == 1 else parents[b]).tolist()
        tok, u = tokens[b].tolist(), uniforms[b].float().double().tolist()
        children: dict = {}
        for i in range(1, n):
            if 0 <= par[i] < i and 0 <= tok[i] < V:
                children.setdefault(par[i], []).append(i)
        at, path = 0, [0]
        while True:
            row = probs[b, at].double()
            rest, low, step = clean(row), 0.0, None
            if draft_probs is not None and at + 1 < n:
                q = draft_probs[b, at].double()
                c = children.get(at, [None])[0]
                if c is not None and u[at] * float(q[tok[c]]) < float(row[tok[c]]):
                    step = c
                rest = clean(row - q)
            elif draft_probs is None:
                for c in children.get(at, []):
                    mass = float(rest[tok[c]])
                    if step is None and low <= u[at] < low + mass:
                        step = c
                    low += mass
                    rest[tok[c]] = 0
            if step is None:
                break
            at = step
            path.append(at)
        if not float(rest.sum()) > 0:
            rest = clean(row)
        held = rest.nonzero()
        if held.numel() == 0:
            nexts.append(-1)
        else:
            sums = rest.cumsum(0)
            nexts.append(min(int((~(sums > u[T - 1] * float(sums[-1]))).sum()), int(held.max())))
        took.append(len(path) - 1)
        paths.append(path + [-1] * (T - len(path)))
    mk = lambda x, *s: torch.tensor(x, dtype=torch.int64, device=probs.device).reshape(*s)   # noqa: E731
    return mk(took, B), mk(paths, B, T), mk(nexts, B)
