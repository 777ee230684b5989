"""Operators of decoding with a cache: rotary positions, a paged and quantised cache of keys and values, attention over it for
single tokens and for trees of drafted tokens, and the verification of drafted tokens.

Where ``own`` is false, ``run`` computes each operator in elementary torch operations, in 32 bits (64 where that loses what
matters); where it is true, it makes the calls that a program makes of ``torsh_b200``.

Kinds:

* ``rotary``     queries and keys turned by their positions; ``train``: forward and backward
* ``cache``      keys and values quantised into their pages, and the same positions read back
* ``attention``  queries of the newest tokens (one, or a tree of drafted ones) over the cache
* ``verify``     drafted tokens accepted or refused from given uniform numbers, and the token that follows
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
BITS = {"bf16": torch.int16, "int8": torch.int8, "e4m3": torch.int8}   # what is moved about
SIZE = {"bf16": 2, "fp32": 4, "int8": 1, "e4m3": 1}
TINY = 2.0 ** -100   # rows whose largest magnitude is below are held as zeros


def listed():
    return [
        # one decoding step of 16 sequences deep in their contexts: latency
        dict(name="rotary_step", kind="rotary", batch=16, tokens=1, heads=32, kv_heads=8, dim=128, rot=128, interleaved=False, scaling="wavelength", far=60000, dtype="bf16", train=False),
        # q and k of a Llama-7B layer in long-context training
        dict(name="rotary_train", kind="rotary", batch=2, tokens=4096, heads=32, kv_heads=32, dim=128, rot=128, interleaved=True, scaling="none", far=0, dtype="bf16", train=True),
        # full precision, half of each head turned, positions beyond 100000, an odd length
        dict(name="rotary_partial_fp32", kind="rotary", batch=3, tokens=1531, heads=16, kv_heads=4, dim=64, rot=32, interleaved=False, scaling="yarn", far=120000, dtype="fp32", train=True),
        # the newest token of 13 sequences enters an int8 cache
        dict(name="cache_step_int8", kind="cache", batch=13, tokens=1, heads=8, dim=128, page=16, store="int8", far=5000, ragged=False),
        # prompts of 8 sequences enter an e4m3 cache with Llama-7B's heads, padded to the longest
        dict(name="cache_prompt_e4m3", kind="cache", batch=8, tokens=2048, heads=32, dim=128, page=64, store="e4m3", far=0, ragged=True),
        # the first tokens of a short answer, GPT-2-medium's heads: latency
        dict(name="attn_token_short", kind="attention", batch=1, tokens=1, heads=16, kv_heads=16, dim=64, context=77, page=16, store="bf16", ragged=False),
        # one sequence with a very long context: all of the GPU works on eight heads
        dict(name="attn_token_long", kind="attention", batch=1, tokens=1, heads=32, kv_heads=8, dim=128, context=131071, page=64, store="int8", ragged=False),
        # a decoding step of a full server, contexts of very different lengths
        dict(name="attn_batch_ragged", kind="attention", batch=64, tokens=1, heads=32, kv_heads=8, dim=128, context=8192, page=16, store="e4m3", ragged=True),
        # trees of 48 drafted tokens, Llama-7B's heads
        dict(name="attn_tree", kind="attention", batch=8, tokens=48, heads=32, kv_heads=32, dim=128, context=4096, page=32, store="bf16", ragged=False),
        # trees of up to 27 drafted tokens, four query heads to a head of the cache
        dict(name="attn_tree_grouped", kind="attention", batch=12, tokens=27, heads=32, kv_heads=8, dim=128, context=6000, page=16, store="int8", ragged=True),
        # chains of 5 drafted tokens of a full server, drawn from a smaller model's distribution
        dict(name="verify_chain", kind="verify", batch=64, tokens=6, vocab=128000, draft=True, dtype="fp32"),
        # one sequence's tree of candidates over GPT-2's vocabulary
        dict(name="verify_tree", kind="verify", batch=1, tokens=26, vocab=50257, draft=False, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    """An integer spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _two(k):
    """2^k in 64 bits, from its bits: pow() need not be exact."""
    return ((k.long() + 1023) << 52).view(torch.float64)


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 250)


def draw(rng):
    kind = rng.choice(["rotary", "rotary", "cache", "cache", "attention", "attention", "attention", "verify"])
    most = max(_cost(c) for c in listed() if c["kind"] == kind)
    while True:
        case = _draw(rng, kind)
        if _cost(case) <= most:
            return case


def _draw(rng, kind):
    if kind == "rotary":
        dim = rng.choice([64, 64, 80, 96, 128, 128])
        train = rng.random() < 0.6
        tokens = _log(rng, 16, 4096) if train else _log(rng, 1, 4096)
        kv = rng.choice([1, 2, 4, 8, 16])
        return dict(kind=kind, batch=_log(rng, 1, 64), tokens=tokens, heads=kv * rng.choice([1, 2, 4]), kv_heads=kv, dim=dim, rot=rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)]),
                    interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "ntk", "yarn", "wavelength"]), far=rng.choice([0, 0, _log(rng, 10, 1000000)]), dtype=rng.choice(["bf16", "bf16", "fp32"]), train=train)
    if kind == "cache":
        return dict(kind=kind, batch=_log(rng, 1, 64), tokens=_log(rng, 1, 4096), heads=rng.choice([1, 2, 4, 8, 12, 16, 32]), dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]),
                    store=rng.choice(["bf16", "int8", "int8", "e4m3", "e4m3"]), far=rng.choice([0, _log(rng, 1, 8000)]), ragged=rng.random() < 0.5)
    if kind == "attention":
        kv = rng.choice([1, 2, 4, 8, 8, 16, 32])
        heads = kv * rng.choice([1, 2, 4, 8]) if kv < 16 else kv
        return dict(kind=kind, batch=_log(rng, 1, 64), tokens=1 if rng.random() < 0.5 else _log(rng, 2, 64), heads=heads, kv_heads=kv, dim=rng.choice([64, 128, 128]),
                    context=_log(rng, 1, 131072), page=rng.choice([16, 32, 64, 128]), store=rng.choice(["bf16", "int8", "e4m3"]), ragged=rng.random() < 0.5)
    return dict(kind=kind, batch=_log(rng, 1, 64), tokens=_log(rng, 2, 48), vocab=_log(rng, 1000, 128000), draft=rng.random() < 0.5, dtype=rng.choice(["fp32", "fp32", "bf16"]))


# ------------------------------------------------------------------------------------------------ sizes
def _starts(case, limit):
    """Lengths of the sequences: all the same, or spread evenly over a tenth to the whole of `limit`."""
    b = case["batch"]
    return [int(limit * (0.1 + 0.9 * (i + 1) / b)) if case["ragged"] else limit for i in range(b)]


def _counts(case):
    """New tokens of the sequences: the full number, or spread evenly over half to the whole of it."""
    b, t = case["batch"], case["tokens"]
    return [max(1, int(t * (0.5 + 0.5 * (i + 1) / b))) if case["ragged"] else t for i in range(b)]


def work(case):
    if case["kind"] == "rotary":
        rows = case["batch"] * case["tokens"]
        n = rows * (case["heads"] + case["kv_heads"]) * case["dim"]
        passes = 2 if case["train"] else 1
        return {"bytes": passes * 2 * n * SIZE[case["dtype"]] + rows * 8, "flops": passes * 3 * n}
    if case["kind"] == "cache":
        rows = sum(_counts(case)) * case["heads"] * 2
        held = rows * (case["dim"] * SIZE[case["store"]] + (0 if case["store"] == "bf16" else 4))
        out = case["batch"] * case["tokens"] * case["heads"] * 2 * case["dim"] * 2   # the padding comes back as zeros
        return {"bytes": rows * case["dim"] * 2 + 2 * held + out, "flops": 4 * rows * case["dim"]}
    if case["kind"] == "attention":
        length = [s + c for s, c in zip(_starts(case, case["context"]), _counts(case))]
        held = sum(length) * case["kv_heads"] * 2 * (case["dim"] * SIZE[case["store"]] + (0 if case["store"] == "bf16" else 4))
        rows = case["batch"] * case["tokens"] * case["heads"] * case["dim"]
        flops = sum(4 * case["dim"] * case["heads"] * c * n for c, n in zip(_counts(case), length))
        return {"bytes": held + rows * 4, "flops": flops}
    rows = case["batch"] * (2 if case["draft"] else 1)
    return {"bytes": rows * case["vocab"] * SIZE[case["dtype"]] + case["batch"] * case["tokens"] * 24, "flops": 2 * rows * case["vocab"]}


# ------------------------------------------------------------------------------------------------ inputs
def _frequencies(case):
    """Radians per position of each pair, in 64 bits, and the factor on the turned columns: as the scaling rules for long contexts have them."""
    rot, base, factor, trained = case["rot"], 10000.0, 8.0, 4096.0
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    if case["scaling"] == "ntk":
        base = base * factor ** (rot / max(rot - 2, 1))
    f = base ** (-i / rot)
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] == "yarn":   # pairs that turn often keep their rate, slow ones are stretched, a ramp between
        at = lambda turns: rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))   # noqa: E731
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    if case["scaling"] == "wavelength":   # by the wavelength against the trained length
        turns = trained * f / (2 * math.pi)
        mix = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        f = f / factor * (1 - mix) + f * mix
    return f, 1.0


def _tree(tokens, gen):
    """A random tree: parents [tokens] (the root has -1), and which token is itself or an ancestor of which."""
    at = torch.arange(tokens)
    parents = (torch.rand(tokens, generator=gen) * at.clamp(max=8)).long() + (at - 8).clamp(min=0)
    parents = torch.minimum(parents, at - 1)
    seen = torch.eye(tokens, dtype=torch.bool)
    for t in range(1, tokens):
        seen[t] |= seen[parents[t]]
    return parents, seen


def _pages(case, gen, lengths):
    """Page table of sequences of `lengths` tokens whose pages lie anywhere in the pool, and the pool's size (its last page is nobody's)."""
    need = [max(1, -(-n // case["page"])) for n in lengths]
    pages = sum(need) + case["batch"] + 1
    order = torch.randperm(pages - 1, generator=gen)
    table = torch.zeros(len(need), max(need), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table.to(DEV), pages


def _pool(case, pages, heads, gen, filled):
    """Pages of keys and values with their scales. Places that nothing was written to hold what memory holds: in bf16 and e4m3 also NaN."""
    shape = (pages, heads, case["page"], case["dim"])
    made = []
    for _ in range(2):
        scales = None
        if case["store"] == "bf16":
            p = torch.randn(shape, device=DEV, generator=gen, dtype=torch.bfloat16) if filled else torch.full(shape, math.nan, device=DEV, dtype=torch.bfloat16)
        else:
            if case["store"] == "int8":
                p = torch.randint(-127, 128, shape, device=DEV, generator=gen, dtype=torch.int8) if filled else torch.full(shape, 55, device=DEV, dtype=torch.int8)
                unit = 2.5 / 127
            else:
                p = (torch.randn(shape, device=DEV, generator=gen, dtype=torch.bfloat16) * 100).clamp(-448, 448).to(torch.float8_e4m3fn) if filled else torch.full(shape, 0x7F, device=DEV, dtype=torch.int8).view(torch.float8_e4m3fn)
                unit = 2.0 ** -7
            scales = torch.rand(shape[:3], device=DEV, generator=gen) * unit + 0.5 * unit
            if case["store"] == "e4m3":   # powers of two, as they are written
                scales = _two(torch.frexp(scales)[1] - 1).float()
        made += [p, scales]
    return made


def prepare(case, seed):
    gen, host = torch.Generator(DEV).manual_seed(seed), torch.Generator().manual_seed(seed)
    randn = lambda *s, dtype=torch.bfloat16: torch.randn(*s, device=DEV, generator=gen).to(dtype)   # noqa: E731
    s = dict(case=case)
    b, t = case["batch"], case["tokens"]
    if case["kind"] == "rotary":
        dt = DTYPES[case["dtype"]]
        s["q"], s["k"] = (randn(b, t, h, case["dim"], dtype=dt) for h in (case["heads"], case["kv_heads"]))
        first = torch.randint(0, case["far"] + 1, (b, 1), generator=host) + (case["far"] if t == 1 else 0)
        s["positions"] = (first + torch.arange(t)).to(DEV)
        f, s["magnitude"] = _frequencies(case)
        s["freqs"] = f.to(DEV)
        if case["train"]:
            s["dq"], s["dk"] = randn(*s["q"].shape, dtype=dt), randn(*s["k"].shape, dtype=dt)
            s["q"].requires_grad_(), s["k"].requires_grad_()
    elif case["kind"] == "cache":
        far = torch.randint(0, case["far"] + 1, (b,), generator=host)
        s["start"] = far.to(DEV, torch.int32)
        s["counts"] = torch.tensor(_counts(case))[torch.randperm(b, generator=host)].to(DEV, torch.int32)
        s["k"], s["v"] = randn(b, t, case["heads"], case["dim"]), randn(b, t, case["heads"], case["dim"])
        s["k"] *= torch.exp(torch.randn(case["heads"], 1, device=DEV, generator=gen)).to(torch.bfloat16)   # heads differ in their range
        s["table"], pages = _pages(case, host, [int(n) + t for n in far])
        s["kp"], s["ks"], s["vp"], s["vs"] = _pool(case, pages, case["heads"], gen, False)
    elif case["kind"] == "attention":
        order = torch.randperm(b, generator=host)
        start, counts = torch.tensor(_starts(case, case["context"]))[order], torch.tensor(_counts(case))[order]
        s["start"], s["counts"] = start.to(DEV, torch.int32), counts.to(DEV, torch.int32)
        s["q"] = randn(b, t, case["heads"], case["dim"])
        s["table"], pages = _pages(case, host, [int(n) + t for n in start])
        s["kp"], s["ks"], s["vp"], s["vs"] = _pool(case, pages, case["kv_heads"], gen, True)
        s["mask"] = _tree(t, host)[1].to(DEV) if t > 1 else None
        s["longest"] = int((start + t).max())
        if case["store"] != "int8":   # what lies behind the last token of each sequence, in its page, was never written
            at = start + counts
            ends = torch.nonzero(at % case["page"])[:, 0]
            last = s["table"].cpu()[ends, at[ends] // case["page"]].long().to(DEV)
            wild = (torch.arange(case["page"]) >= (at[ends] % case["page"])[:, None]).to(DEV)
            for p in (s["kp"], s["vp"]):
                bits = p.view(torch.int16 if case["store"] == "bf16" else torch.int8)
                bits[last] = torch.where(wild[:, None, :, None], 0x7FFF if case["store"] == "bf16" else 0x7F, bits[last])   # NaN
    else:
        v, dt = case["vocab"], DTYPES[case["dtype"]]
        parents, seen = _tree(t, host)
        if case["draft"]:
            parents = torch.arange(t) - 1
            seen = torch.ones(t, t, dtype=torch.bool).tril()
        logits = (3 if case["draft"] else 5) * torch.randn(b, t, v, device=DEV, generator=gen)
        s["probs"] = torch.softmax(logits, -1).to(dt)
        s["uniforms"] = torch.rand(b, t, device=DEV, generator=gen)
        s["counts"] = torch.tensor([max(1, t - i % 3) for i in range(b)], dtype=torch.int32, device=DEV)
        if case["draft"]:
            d = torch.softmax(logits[:, :-1] + 0.4 * torch.randn(b, t - 1, v, device=DEV, generator=gen), -1).to(dt)
            drawn = torch.multinomial(d.float().view(-1, v), 1, generator=gen).view(b, t - 1)
            s["draft_probs"] = d
        else:   # each child is one of its parent's likeliest tokens, so that paths are followed
            s["draft_probs"] = None
            best = logits.topk(16, -1).indices
            pick = torch.arange(1, t, device=DEV) % 8
            drawn = best[:, parents[1:].to(DEV)].gather(-1, pick.expand(b, -1)[..., None])[..., 0]
            s["uniforms"] *= 0.7
        s["tokens"] = torch.cat([torch.zeros(b, 1, dtype=torch.long, device=DEV), drawn], 1)
        s["parents"], s["seen"] = parents.to(DEV), seen.to(DEV)
        del logits
    return s


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(s):
    case = s["case"]
    if case["kind"] == "rotary":
        from torsh_b200.ops.rotary import rotary
        q, k = rotary(s["q"], s["k"], s["positions"], s["freqs"], interleaved=case["interleaved"], magnitude=s["magnitude"])
        if not case["train"]:
            return q, k
        return (q, k, *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"])))
    if case["kind"] == "cache":
        from torsh_b200.ops.kv_cache import kv_cache_read, kv_cache_write
        kv_cache_write(s["k"], s["v"], s["kp"], s["vp"], s["table"], s["start"], counts=s["counts"], k_scales=s["ks"], v_scales=s["vs"])
        return kv_cache_read(s["kp"], s["vp"], s["table"], s["counts"], case["tokens"], begin=s["start"], k_scales=s["ks"], v_scales=s["vs"], dtype=torch.bfloat16)
    if case["kind"] == "attention":
        from torsh_b200.ops.kv_cache import kv_cache_attention
        return kv_cache_attention(s["q"], s["kp"], s["vp"], s["table"], s["start"], tree_mask=s["mask"], counts=s["counts"], k_scales=s["ks"], v_scales=s["vs"], max_len=s["longest"])
    from torsh_b200.ops.speculative import verify_draft
    return verify_draft(s["probs"], s["tokens"], s["uniforms"], draft_probs=s["draft_probs"], parents=None if case["draft"] else s["parents"], counts=s["counts"])


# ------------------------------------------------------------------------------------------------ the plain forms
def _turn(x, cos, sin, rot, interleaved, dtype):
    x = x.float()
    r, rest = x[..., :rot], x[..., rot:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :rot // 2], r[..., rot // 2:])
    u, w = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    return torch.cat([turned, rest], -1).to(dtype)


def _run_rotary(s):
    case = s["case"]
    angle = s["positions"].double()[..., None, None] * s["freqs"]
    cos, sin = (torch.cos(angle) * s["magnitude"]).float(), (torch.sin(angle) * s["magnitude"]).float()
    turn = lambda x, back: _turn(x, cos, -sin if back else sin, case["rot"], case["interleaved"], x.dtype)   # noqa: E731
    out = turn(s["q"].detach(), False), turn(s["k"].detach(), False)
    return (*out, turn(s["dq"], True), turn(s["dk"], True)) if case["train"] else out


def _quantised(x, store):
    """Codes and scales of rows: what is stored, and one number a row."""
    if store == "bf16":
        return x.to(torch.bfloat16), None
    big = x.float().abs().amax(-1)
    if store == "int8":
        scale = big / 127
    else:
        f, e = torch.frexp(big)
        scale = _two(e - 9 + (f > 0.875)).float()
    scale = torch.where(big < TINY, 0, scale)
    r = x.double() / torch.where(scale > 0, scale, 1).double()[..., None]   # 64 bits: a quotient next to a half must not be rounded onto it
    r = torch.where(scale[..., None] > 0, r, 0)
    return (torch.round(r).to(torch.int8) if store == "int8" else r.float().to(torch.float8_e4m3fn)), scale


def _run_cache(s):
    case = s["case"]
    t, page = case["tokens"], case["page"]
    at = s["start"].long()[:, None] + torch.arange(t, device=DEV)
    held = torch.arange(t, device=DEV)[None] < s["counts"][:, None]
    slot = torch.where(held, s["table"].long().gather(1, at // page), s["kp"].shape[0] - 1)   # rows that do not count go to nobody's page
    out = []
    for x, pages, scales in ((s["k"], s["kp"], s["ks"]), (s["v"], s["vp"], s["vs"])):
        codes, scale = _quantised(x, case["store"])
        bits = pages.view(BITS[case["store"]])
        bits[slot, :, at % page] = codes.view(bits.dtype)
        back = bits[slot, :, at % page].view(pages.dtype).float()
        if scales is not None:
            scales[slot, :, at % page] = scale
            back = back * scales[slot, :, at % page][..., None]
        out.append(torch.where(held[..., None, None], back, 0).to(torch.bfloat16))
    return tuple(out)


def _run_attention(s):
    case = s["case"]
    b, t, h, g, d = case["batch"], case["tokens"], case["kv_heads"], case["heads"] // case["kv_heads"], case["dim"]
    n = s["longest"]
    table = s["table"].long()

    def rows(pages, scales):
        x = pages.view(BITS[case["store"]])[table].view(pages.dtype).float()   # [B, pages, H, page, D]
        if scales is not None:
            x = x * scales[table][..., None]
        return x.transpose(1, 2).reshape(b, h, -1, d)[:, :, :n]

    at = torch.arange(n, device=DEV)
    start, counts = s["start"].long()[:, None], s["counts"].long()[:, None]
    new = (at - start).clamp(0, t - 1)                                  # [B, n]: which of the new tokens, if any
    mask = s["mask"] if s["mask"] is not None else torch.ones(1, 1, dtype=torch.bool, device=DEV)
    seen = (at < start)[:, None] | (((at >= start) & (at < start + counts))[:, None] & mask[:, new].transpose(0, 1))   # [B, T, n]
    live = torch.arange(t, device=DEV) < counts                         # [B, T]
    seen = seen & live[..., None]
    written = (at < start + counts)[:, None, :, None]
    k, v = rows(s["kp"], s["ks"]), torch.where(written, rows(s["vp"], s["vs"]), 0)
    q = s["q"].float().view(b, t, h, g, d).permute(0, 2, 3, 1, 4).reshape(b, h, g * t, d)
    score = torch.matmul(q, k.transpose(-1, -2)).view(b, h, g, t, n) / math.sqrt(d)
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(torch.isfinite(top), top, 0))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.view(b, h, g * t, n), v).view(b, h, g, t, d) / torch.where(total > 0, total, 1)
    return o.permute(0, 3, 1, 2, 4).reshape(b, t, h * g, d).to(torch.bfloat16)


def _run_verify(s):
    case = s["case"]
    b, t, v = case["batch"], case["tokens"], case["vocab"]
    p, tokens, u = s["probs"], s["tokens"], s["uniforms"].double()
    node = torch.arange(t, device=DEV)
    live = node < s["counts"].long()[:, None]                           # [B, T]
    parents = s["parents"][1:]
    mass = p[:, parents].gather(-1, tokens[:, 1:, None])[..., 0].double()   # [B, T-1]: each token's probability after its parent
    if case["draft"]:
        ok = u[:, :-1] * s["draft_probs"].gather(-1, tokens[:, 1:, None])[..., 0].double() < mass
    else:   # siblings share the parent's number: each takes the interval behind the ones before it; a token that comes twice has none the second time
        before = (parents[:, None] == parents[None]) & (node[1:, None] > node[None, 1:])
        twice = (before & (tokens[:, 1:, None] == tokens[:, None, 1:]) & live[:, None, 1:]).any(-1)
        mass = torch.where(twice | ~live[:, 1:], 0, mass)
        low = torch.matmul(before.double(), mass[..., None])[..., 0]
        ok = (u[:, parents] >= low) & (u[:, parents] < low + mass)
    ok = torch.cat([torch.ones(b, 1, dtype=torch.bool, device=DEV), ok], 1) & live
    on = ~(s["seen"] & ~ok[:, None]).any(-1)                            # accepted, and so are all its ancestors
    accepted = on.sum(-1) - 1
    path = torch.where(on, node, t).sort(-1).values
    path = torch.where(path < t, path, -1)
    last = torch.where(on, node, 0).amax(-1)
    one = torch.arange(b, device=DEV)
    row = p[one, last].double()
    if case["draft"]:
        refused = last + 1 < s["counts"]
        q = s["draft_probs"][one, last.clamp(max=t - 2)].double()
        rest = torch.where(refused[:, None], (row - q).clamp(min=0), row)
    else:
        child = (s["parents"] == last[:, None]) & live                  # [B, T]
        taken = torch.zeros(b, v, device=DEV, dtype=torch.double).scatter_add_(1, tokens, child.double())
        rest = torch.where(taken > 0, 0, row)
    total = rest.sum(-1, keepdim=True)
    rest = torch.where(total > 0, rest, row)
    sums = rest.cumsum(-1)
    token = (sums <= u[:, -1:] * sums[:, -1:]).sum(-1)
    token = torch.minimum(token, torch.where(rest > 0, torch.arange(v, device=DEV), 0).amax(-1))
    return accepted, path, token


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind == "rotary":
        return _run_rotary(state)
    if kind == "cache":
        return _run_cache(state)
    if kind == "attention":
        return _run_attention(state)
    return _run_verify(state)


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        z = torch.polar(torch.full((), s["magnitude"], dtype=torch.double, device=DEV), torch.einsum("bt,f->btf", s["positions"].double(), s["freqs"]))[:, :, None]
        half = case["rot"] // 2

        def turned(x, by):
            x = x.detach().double()
            i = torch.arange(half, device=DEV)
            a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
            w = torch.complex(x[..., a], x[..., b]) * by
            y = x.clone()
            y[..., a], y[..., b] = w.real, w.imag
            return y

        out = [turned(s["q"], z), turned(s["k"], z)]
        return tuple(out + [turned(s["dq"], z.conj()), turned(s["dk"], z.conj())] if case["train"] else out)
    if case["kind"] == "cache":
        out = []
        for x in (s["k"].double(), s["v"].double()):
            if case["store"] != "bf16":
                big = x.abs().amax(-1, keepdim=True)
                if case["store"] == "int8":
                    unit = (big / 127).float().double()
                    x = torch.round(x / unit) * unit
                else:   # the least power of two that brings the row to 448; three bits behind the leading one, the smallest step 2^-9
                    k = torch.arange(-100, 101, device=DEV)
                    unit = _two(torch.where(448 * _two(k) >= big, k, 101).amin(-1, keepdim=True))
                    step = _two((torch.frexp(x / unit)[1] - 1).clamp(min=-6) - 3)
                    x = torch.round(x / unit / step) * step * unit
            for b, n in enumerate(s["counts"].tolist()):
                x[b, n:] = 0
            out.append(x)
        return tuple(out)
    if case["kind"] == "attention":
        g, n_heads = case["heads"] // case["kv_heads"], case["kv_heads"]
        out = torch.zeros(s["q"].shape, dtype=torch.double, device=DEV)
        for b in range(case["batch"]):
            first, n = int(s["start"][b]), int(s["counts"][b])
            at = torch.arange(first + n, device=DEV)
            page, row = s["table"][b].long()[at // case["page"]], at % case["page"]
            for h in range(n_heads):
                k, v = (x.view(BITS[case["store"]])[page, h, row].view(x.dtype).double() for x in (s["kp"], s["vp"]))
                if s["ks"] is not None:
                    k, v = k * s["ks"][page, h, row].double()[:, None], v * s["vs"][page, h, row].double()[:, None]
                q = s["q"][b, :n, h * g:(h + 1) * g].double()
                score = torch.einsum("tgd,nd->tgn", q, k) * case["dim"] ** -0.5
                if s["mask"] is not None:
                    score[..., first:].masked_fill_(~s["mask"][:n, None, :n], -math.inf)
                out[b, :n, h * g:(h + 1) * g] = torch.einsum("tgn,nd->tgd", torch.softmax(score, -1), v)
        return out
    # verification, one sequence after the other
    took, paths, nexts = [], [], []
    parents = s["parents"].tolist()
    for b in range(case["batch"]):
        n, tokens, u = int(s["counts"][b]), s["tokens"][b].tolist(), s["uniforms"][b].double().tolist()
        at, path = 0, [0]
        while True:
            children = [c for c in range(1, n) if parents[c] == at]
            row = s["probs"][b, at].double()
            rest, low, step = row.clone(), 0.0, None
            if case["draft"] and children:
                q = s["draft_probs"][b, at].double()
                if u[at] * float(q[tokens[children[0]]]) < float(row[tokens[children[0]]]):
                    step = children[0]
                rest = (row - q).clamp(min=0)
            for c in children if not case["draft"] else []:
                mass = float(rest[tokens[c]])
                if step is None and low <= u[at] < low + mass:
                    step = c
                low += mass
                rest[tokens[c]] = 0
            if step is None:
                break
            at = step
            path.append(at)
        if not float(rest.sum()) > 0:
            rest = row
        sums = rest.cumsum(0)
        token = min(int((sums <= u[-1] * float(sums[-1])).sum()), int(rest.nonzero().max()))
        took.append(len(path) - 1)
        paths.append(path + [-1] * (case["tokens"] - len(path)))
        nexts.append(token)
    return tuple(torch.tensor(x, device=DEV) for x in (took, paths, nexts))
