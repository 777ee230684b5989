"""Rotary positions, the paged cache, attention over it and the verification of drafted tokens against 64-bit references.

Tolerances count roundings: one to a type with unit u = eps / 2 is off by at most u times the value (bf16 2^-8, fp16 2^-11, fp32 2^-24).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16
E4M3 = torch.float8_e4m3fn
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


# ------------------------------------------------------------------------------------------------ rotary
def _turn64(x, positions, freqs, interleaved, magnitude, inverse=False):
    z = torch.polar(torch.ones((), device=DEV, dtype=torch.float64), positions.double()[..., None] * freqs)[..., None, :] * magnitude
    z = z.conj() if inverse else z
    h = freqs.numel()
    i = torch.arange(h, device=DEV)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + h)
    y = x.double().clone()
    w = torch.complex(y[..., a], y[..., b]) * z
    y[..., a], y[..., b] = w.real, w.imag
    return y


def _rotary_close(got, x, ref, magnitude):
    # cos and sin to 4 units of fp32, two products and a sum in fp32 (3 units of |a| + |b|), one rounding to the type
    norm = magnitude * (x.double().abs().amax() * 2)
    assert got.dtype == x.dtype
    assert ((got.double() - ref).abs() <= HALF[x.dtype] * ref.abs() + 8 * 2.0 ** -24 * norm).all()


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("B,T,Hq,Hk,D,R", [(1, 1, 1, 1, 64, 64), (3, 5, 8, 2, 128, 128), (2, 37, 6, 3, 128, 64), (5, 1, 4, 4, 80, 80),
                                           (2, 3, 5, 1, 96, 34), (1, 700, 3, 2, 64, 32), (4, 9, 2, 2, 100, 50), (2, 2, 3, 1, 7, 4), (1, 3, 2, 1, 64, 0)])
def test_rotary(dtype, interleaved, B, T, Hq, Hk, D, R):
    from torsh_b200.ops.rotary import rotary, rotary_frequencies
    g = _gen(B * T + D)
    q, k = (torch.randn(B, T, h, D, device=DEV, generator=g).to(dtype).requires_grad_() for h in (Hq, Hk))
    pos = torch.randint(0, 1_000_000, (B, T), device=DEV, generator=g)
    freqs, m = rotary_frequencies(R, scaling="yarn" if R else "none", factor=4.0, device=DEV)
    yq, yk = rotary(q, k, pos, freqs, interleaved, m)
    dq, dk = torch.randn_like(yq), torch.randn_like(yk)
    gq, gk = torch.autograd.grad((yq, yk), (q, k), (dq, dk))
    for got, x, inv in ((yq, q, False), (yk, k, False), (gq, dq, True), (gk, dk, True)):
        _rotary_close(got, x.detach(), _turn64(x.detach(), pos, freqs, interleaved, m, inv), m)
    # the gradient is that of differences too: the map is linear, so <dy, f(x)> = <f'(dy), x>
    lhs = (dq.double() * _turn64(q.detach(), pos, freqs, interleaved, m)).sum()
    assert abs(lhs - (gq.double() * q.detach().double()).sum()) <= HALF[dtype] * 2 * (dq.double().abs() * q.detach().double().abs()).sum() * m * 2
    # alone
    only, none = rotary(q.detach(), None, pos, freqs, interleaved, m)
    assert none is None and torch.equal(only, yq.detach())


def test_rotary_gradient_of_a_gradient_and_of_one_output():
    from torsh_b200.ops.rotary import rotary, rotary_frequencies
    g = _gen(3)
    q, k = (torch.randn(2, 3, 2, 64, device=DEV, generator=g).requires_grad_() for _ in range(2))
    pos = torch.arange(3, device=DEV).expand(2, 3).contiguous()
    freqs, _ = rotary_frequencies(64, device=DEV)
    yq, yk = rotary(q, k, pos, freqs)
    gq, gk = torch.autograd.grad(yq.sum(), (q, k), allow_unused=True)      # nothing comes back through k but zeros
    _rotary_close(gq, torch.ones_like(yq), _turn64(torch.ones_like(yq), pos, freqs, True, 1.0, True), 1.0)
    assert gk is None or not gk.any()
    dy = torch.randn_like(q).requires_grad_()
    yq, _ = rotary(q, None, pos, freqs)
    (gq,) = torch.autograd.grad(yq, q, dy, create_graph=True)
    w = torch.randn_like(q)
    (gd,) = torch.autograd.grad((gq * w).sum(), dy)                        # the rotation of w
    _rotary_close(gd, w, _turn64(w, pos, freqs, True, 1.0), 1.0)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("D,R", [(96, 34), (64, 36), (64, 32), (80, 70), (12, 6)])
def test_rotary_leaves_the_other_columns_as_they_are(dtype, interleaved, D, R):
    from torsh_b200.ops.rotary import rotary, rotary_frequencies
    x = torch.randn(2, 5, 3, D, device=DEV, generator=_gen(D)).to(dtype)
    x[..., R::3], x[..., R + 1::5] = math.inf, math.nan
    pos = torch.arange(5, device=DEV) + 7
    freqs, _ = rotary_frequencies(R, device=DEV)
    y, _ = rotary(x, None, pos, freqs, interleaved, 1.25)
    bits = torch.int16 if dtype == BF16 else torch.int32
    assert torch.equal(y[..., R:].contiguous().view(bits), x[..., R:].contiguous().view(bits))
    ref = _turn64(x, pos.expand(2, 5), freqs, interleaved, 1.25)
    _rotary_close(y[..., :R], x[..., :R], ref[..., :R], 1.25)


def test_rotary_strides_beyond_32_bits_and_heads_between_tokens():
    """Rows so far apart that their strides do not fit 32 bits, and blocks whose rows are of several tokens and of both tensors."""
    from torsh_b200.ops.rotary import rotary, rotary_frequencies
    freqs, _ = rotary_frequencies(64, device=DEV)
    store = torch.empty((1 << 31) + 4096, dtype=BF16, device=DEV)
    q = store.as_strided((2, 3, 64), ((1 << 31) + 8, 64, 1))
    q.copy_(torch.randn(2, 3, 64, device=DEV, generator=_gen(4)))
    pos = torch.tensor([3, 1000], device=DEV)
    y, _ = rotary(q, None, pos, freqs)
    _rotary_close(y, q, _turn64(q, pos, freqs, True, 1.0), 1.0)
    del store, q
    for N, hq, hk in ((3000, 3, 1), (40000, 5, 2), (5000, 70, 1)):
        q, k = (torch.randn(N, h, 64, device=DEV, generator=_gen(N + h)).to(BF16) for h in (hq, hk))
        pos = torch.randint(0, 5000, (N,), device=DEV, generator=_gen(2))
        for interleaved in (True, False):
            for x, y in zip((q, k), rotary(q, k, pos, freqs, interleaved)):
                _rotary_close(y, x, _turn64(x, pos, freqs, interleaved, 1.0), 1.0)


def test_rotary_strides_and_shared_positions():
    from torsh_b200.ops.rotary import rotary, rotary_frequencies
    B, T, H, D = 3, 11, 4, 64
    packed = torch.randn(B * T, 3 * H * D, device=DEV, generator=_gen(1)).to(BF16)
    q, k = (packed[:, i * H * D:(i + 1) * H * D].view(B, T, H, D) for i in range(2))
    freqs, _ = rotary_frequencies(D, device=DEV)
    pos = torch.arange(T, device=DEV, dtype=torch.int32)
    yq, yk = rotary(q, k, pos, freqs, False)
    _rotary_close(yq, q, _turn64(q, pos.expand(B, T), freqs, False, 1.0), 1.0)
    _rotary_close(yk, k, _turn64(k, pos.expand(B, T), freqs, False, 1.0), 1.0)
    # heads in front of tokens, a row that starts off a 16-byte boundary, and packed tokens without a batch
    qt = torch.randn(B, H, T, D, device=DEV, generator=_gen(2)).to(BF16).transpose(1, 2)
    odd = torch.randn(B * T * H * D + 1, device=DEV, generator=_gen(3)).to(BF16)[1:].view(B, T, H, D)
    for x in (qt, odd):
        y, _ = rotary(x, None, pos, freqs, True)
        _rotary_close(y, x, _turn64(x, pos.expand(B, T), freqs, True, 1.0), 1.0)
    flat, _ = rotary(q.reshape(B * T, H, D), None, pos.repeat(B), freqs, False)
    assert torch.equal(flat.view(B, T, H, D), yq)
    dy = torch.randn(B, H, T, D, device=DEV, generator=_gen(4)).to(BF16).transpose(1, 2)
    x = q.detach().clone().requires_grad_()
    (gx,) = torch.autograd.grad(rotary(x, None, pos, freqs, False)[0], x, dy)
    _rotary_close(gx, dy, _turn64(dy, pos.expand(B, T), freqs, False, 1.0, True), 1.0)
    empty, _ = rotary(torch.empty(0, 4, 2, 64, device=DEV, dtype=BF16), None, torch.arange(4, device=DEV), freqs)
    assert empty.shape == (0, 4, 2, 64)


# ------------------------------------------------------------------------------------------------ cache
def _codes64(x, dtype):
    """Codes as numbers, and scales: the definition in 64 bits, row by row."""
    big = x.double().abs().amax(-1, keepdim=True)
    if dtype == torch.int8:
        unit = (big / 127).float().double()
        return torch.where(big < 2.0 ** -100, 0.0, torch.round(x.double() / unit)).nan_to_num(0.0), torch.where(big < 2.0 ** -100, 0.0, unit)
    k = torch.arange(-120, 130, device=x.device).double()
    two = torch.tensor([2.0 ** i for i in range(-120, 130)], device=x.device, dtype=torch.float64)
    unit = torch.where(448 * two >= big, two, math.inf).amin(-1, keepdim=True)
    r = x.double() / unit
    e = (torch.frexp(r)[1] - 1).clamp(min=-6) - 3
    step = two[e.long() + 120]
    del k
    return torch.where(big < 2.0 ** -100, 0.0, torch.round(r / step) * step), torch.where(big < 2.0 ** -100, 0.0, unit)


def _cache(pages, H, page, D, dtype, fill=0x55):
    mk = lambda: torch.full((pages, H, page, D * (2 if dtype == BF16 else 1)), fill, dtype=torch.int8, device=DEV).view(dtype)   # noqa: E731
    sc = lambda: torch.full((pages, H, page), 7.0, device=DEV) if dtype != BF16 else None   # noqa: E731
    return mk(), mk(), sc(), sc()


@pytest.mark.parametrize("dtype", [BF16, torch.int8, E4M3])
@pytest.mark.parametrize("xdtype", [BF16, torch.float32])
@pytest.mark.parametrize("B,T,H,D,page", [(1, 1, 1, 64, 16), (3, 21, 2, 128, 16), (2, 130, 5, 64, 48), (9, 4, 3, 128, 32)])
def test_cache_write_and_read(dtype, xdtype, B, T, H, D, page):
    from torsh_b200.ops.kv_cache import kv_cache_read, kv_cache_write
    g = _gen(T)
    x = torch.randn(B, T, H, 2 * D, device=DEV, generator=g) * torch.exp(3 * torch.randn(B, T, H, 1, device=DEV, generator=g))
    x = x.to(xdtype)
    k, v = x[..., :D], x[..., D:]                      # strided rows
    k[0, 0, 0] = 0
    v[-1, -1, -1] = 2.0 ** -110 if xdtype == torch.float32 else 0
    if D == 128:
        k[-1, 0, 0, 5] = 448.0 * 4                     # a largest value that meets 448 to the bit
        v[0, 0, 0] = torch.arange(D, device=DEV).to(xdtype) - 64   # halves: multiples of max / 127 that meet k + 1/2
    start = torch.randint(0, 2 * page, (B,), device=DEV, generator=g).int()
    counts = torch.randint(0, T + 1, (B,), device=DEV, generator=g).int()
    counts[0] = T
    per = -(-(2 * page + T) // page)
    table = torch.randperm(B * per + 2, device=DEV, generator=g)[:B * per].view(B, per).int()
    kp, vp, ks, vs = _cache(B * per + 2, H, page, D, dtype)
    before = [None if t is None else t.clone() for t in (kp, vp, ks, vs)]
    kv_cache_write(k, v, kp, vp, table, start, counts, ks, vs)
    touched = torch.zeros(B * per + 2, page, dtype=torch.bool, device=DEV)
    for src, pages, scales in ((k, kp, ks), (v, vp, vs)):
        for b in range(B):
            n = int(counts[b])
            if not n:
                continue
            at = torch.arange(n, device=DEV) + start[b]
            slot, row = table[b][at // page].long(), at % page
            touched[slot, row] = True
            bits = pages.view(torch.int8) if dtype == E4M3 else pages
            got = bits[slot, :, row].view(dtype)
            if dtype == BF16:
                assert torch.equal(got, src[b, :n].to(BF16))
            else:
                codes, unit = _codes64(src[b, :n], dtype)
                assert torch.equal(got.double(), codes)
                assert torch.equal(scales[slot, :, row].double(), unit[..., 0])
    for t, was in zip((kp, vp, ks, vs), before):       # nothing else was written
        if t is not None:
            t, was = (u.view(torch.int8) if u.dtype == E4M3 else u for u in (t, was))
            same = (t == was) if t.dim() == 3 else (t.view(torch.int16 if t.dtype == BF16 else t.dtype) == was.view(torch.int16 if t.dtype == BF16 else t.dtype)).all(-1)
            assert same.transpose(1, 2)[~touched].all()
    for out in (BF16, torch.float32):
        rk, rv = kv_cache_read(kp, vp, table, counts, T + 3, start, ks, vs, out)
        for got, src in ((rk, k), (rv, v)):
            assert got.shape == (B, T + 3, H, D) and got.dtype == out
            for b in range(B):
                n = int(counts[b])
                assert not got[b, n:].any()
                codes, unit = (src[b, :n].to(BF16).double(), 1.0) if dtype == BF16 else _codes64(src[b, :n], dtype)
                assert torch.equal(got[b, :n], (codes * unit).float().to(out))   # code times scale is exact in 32 bits


@pytest.mark.parametrize("dtype", [torch.int8, E4M3])
def test_rows_are_quantised_alike_on_every_device(dtype):
    from torsh_b200.ops.kv_cache import kv_cache_write, quantize_rows
    x = torch.randn(3000, 96, device=DEV, generator=_gen(2)) * torch.exp(4 * torch.randn(3000, 1, device=DEV, generator=_gen(3)))
    here, there = quantize_rows(x, dtype), quantize_rows(x.cpu(), dtype)
    for a, b in zip(here, there):
        assert torch.equal(a.cpu().view(torch.int8), b.view(torch.int8))
    rows = x[:48, :64].contiguous()                                         # and as the kernel does it
    kp, vp, ks, vs = _cache(1, 3, 16, 64, dtype, 0)
    kv_cache_write(rows.view(1, 16, 3, 64), rows.view(1, 16, 3, 64), kp, vp, torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV),
                   None, ks, vs)
    codes, scale = quantize_rows(rows, dtype)
    assert torch.equal(kp.transpose(1, 2).reshape(48, 64).view(torch.int8), codes.view(torch.int8)) and torch.equal(ks.transpose(1, 2).reshape(48), scale)


def test_cache_rows_that_are_not_numbers():
    from torsh_b200.ops.kv_cache import kv_cache_read, kv_cache_write
    k = torch.randn(1, 4, 2, 64, device=DEV, generator=_gen(5)).to(BF16)
    k[0, 1, 0, 3], k[0, 2, 1, 7] = math.nan, -math.inf
    table, start, n = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV), torch.full((1,), 4, device=DEV, dtype=torch.int32)
    for dtype in (torch.int8, E4M3):
        kp, vp, ks, vs = _cache(1, 2, 16, 64, dtype)
        kv_cache_write(k, k, kp, vp, table, start, None, ks, vs)
        rk, _ = kv_cache_read(kp, vp, table, n, 4, None, ks, vs)
        nan = torch.zeros(4, 2, dtype=torch.bool, device=DEV)
        nan[1, 0] = nan[2, 1] = True
        assert torch.equal(rk[0].isnan().all(-1), nan) and torch.equal(rk[0].isnan().any(-1), nan)


def test_cache_positions_without_a_page():
    """Positions behind the table, negative starts and pages outside the pool are skipped, and read as zeros."""
    from torsh_b200.ops.kv_cache import kv_cache_read, kv_cache_write
    kp, vp, _, _ = _cache(2, 1, 16, 64, BF16, 0)
    k = torch.ones(4, 3, 1, 64, device=DEV, dtype=BF16)
    table = torch.tensor([[0], [7], [-1], [1]], dtype=torch.int32, device=DEV)
    start = torch.tensor([14, 0, 0, -2], dtype=torch.int32, device=DEV)
    kv_cache_write(k, k, kp, vp, table, start)
    assert kp[0, 0, 14:].eq(1).all() and kp.float().sum() == 2 * 64
    rk, rv = kv_cache_read(kp, vp, table, torch.full((4,), 3, device=DEV), 3, start)
    assert rk[0, :2].eq(1).all() and rk.float().sum() == 2 * 64 and torch.equal(rk, rv)


def test_cache_rows_more_than_32_bits_apart():
    from torsh_b200.ops.kv_cache import kv_cache_attention, kv_cache_write
    store = torch.empty((1 << 31) + 4096, dtype=BF16, device=DEV)
    for strides in ((4096, 1 << 31, 64, 1), (4096, 128, 1 << 31, 1)):
        x = store.as_strided((1, 2, 2, 64), strides)
        x.copy_(torch.randn(1, 2, 2, 64, device=DEV, generator=_gen(1)))
        y = x.contiguous()
        table, start = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
        pools = [_cache(1, 2, 16, 64, BF16, 0) for _ in range(2)]
        for z, (kp, vp, _, _) in zip((x, y), pools):
            kv_cache_write(z, z, kp, vp, table, start)
        assert torch.equal(pools[0][0], pools[1][0]) and torch.equal(pools[0][0][0, :, :2], y[0].transpose(0, 1))
        assert torch.equal(*(kv_cache_attention(z, *pools[0][:2], table, start) for z in (x, y)))


# ------------------------------------------------------------------------------------------------ attention
def _filled(pages, H, page, D, dtype, g):
    if dtype == BF16:
        return torch.randn(pages, H, page, D, device=DEV, generator=g).to(BF16), None
    if dtype == torch.int8:
        return torch.randint(-127, 128, (pages, H, page, D), device=DEV, generator=g, dtype=torch.int8), torch.rand(pages, H, page, device=DEV, generator=g) * 0.02 + 0.002
    p = (torch.randn(pages, H, page, D, device=DEV, generator=g) * 60).clamp(-448, 448).to(E4M3)
    return p, 2.0 ** torch.randint(-9, -3, (pages, H, page), device=DEV, generator=g).float()


def _attend64(q, kp, vp, ks, vs, table, start, mask, counts, scale, limit=1 << 30):
    """``(output, sum of p |v|)`` in 64 bits, one sequence and head after the other; what a row does not see is left out of its sums."""
    B, T, Hq, D = q.shape
    H, page = kp.shape[1:3]
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    mass = torch.zeros_like(out)
    for b in range(B):
        s0, n = int(start[b]), (T if counts is None else int(counts[b]))
        total = min(s0 + n, limit, table.shape[1] * page)
        if n == 0 or total == 0:
            continue
        at = torch.arange(total, device=DEV)
        slot, row = table[b].long()[at // page], at % page
        there = (slot >= 0) & (slot < kp.shape[0])
        slot = torch.where(there, slot, 0)
        seen = torch.ones(T, total, dtype=torch.bool, device=DEV)
        if total > s0:
            m = torch.ones(T, T, dtype=torch.bool, device=DEV).tril() if mask is None else mask if mask.dim() == 2 else mask[b]
            seen[:, s0:] = m[:, :total - s0]
        for h in range(Hq):
            hk = h // (Hq // H)
            k, v = (torch.where(there[:, None], (x.view(torch.int8) if x.dtype == E4M3 else x)[slot, hk, row].view(x.dtype).double(), 0) for x in (kp, vp))
            if ks is not None:
                k, v = k * torch.where(there, ks[slot, hk, row].double(), 0)[:, None], v * torch.where(there, vs[slot, hk, row].double(), 0)[:, None]
            s = torch.where(seen[:n], (q[b, :n, h].double() @ k.T) * scale, -math.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0)
            out[b, :n, h], mass[b, :n, h] = p @ v, p @ v.abs()
    return out, mass


def _attention_close(got, ref, mass, dtype):
    # P rounded to bf16 or fp16 and the output to bf16; scores are sums of at most 128 products in fp32, off by at most 130 units of
    # sum |q k| scale, which stays below 8 here: 130 * 8 * 2^-24 < 2^-13 relative in p
    p = 2.0 ** -8 if dtype == BF16 else 2.0 ** -11
    assert torch.isfinite(got).all()
    assert ((got.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + (p + 2.0 ** -13) * 1.01 * mass).all()


def _case(B, T, Hq, H, D, page, contexts, dtype, seed=0, extra=3):
    g = _gen(seed + T + B)
    start = torch.tensor((list(contexts) * B)[:B], dtype=torch.int32, device=DEV)
    need = [-(-(int(s) + T) // page) for s in start.tolist()]
    pages = sum(need) + extra
    order = torch.randperm(pages, device=DEV, generator=g).int()
    table = torch.full((B, max(need)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    kp, ks = _filled(pages, H, page, D, dtype, g)
    vp, vs = _filled(pages, H, page, D, dtype, g)
    q = torch.randn(B, T, Hq, D, device=DEV, generator=g).to(BF16)
    return q, kp, vp, ks, vs, table, start


def _random_tree(T, seed):
    from torsh_b200.ops.kv_cache import tree_mask_of
    g = torch.Generator().manual_seed(seed)
    parents = torch.tensor([-1] + [int(torch.randint(max(0, i - 6), i, (1,), generator=g)) for i in range(1, T)])
    return tree_mask_of(parents).to(DEV)


SHAPES = [(1, 1, 1, 1, 64, 16, [0]), (2, 1, 4, 4, 128, 16, [15, 16]), (3, 1, 8, 2, 128, 32, [17, 1, 700]), (5, 1, 12, 12, 64, 64, [100, 0, 63, 64, 65]),
          (1, 1, 8, 1, 128, 16, [9001]), (2, 7, 8, 2, 128, 16, [333, 5]), (3, 13, 2, 2, 64, 48, [40, 0, 95]), (2, 48, 4, 4, 128, 32, [500, 31]),
          (2, 27, 16, 4, 128, 16, [129, 1000]), (1, 64, 8, 1, 64, 128, [2000]), (2, 33, 3, 1, 64, 16, [16, 250]), (150, 1, 2, 1, 64, 16, [3, 200, 31, 0]),
          # many tiles and units to a CTA, ends anywhere in them
          (4, 8, 32, 8, 128, 64, [5000, 3001, 8064, 127]), (6, 40, 16, 16, 64, 16, [2900, 4096, 77, 5003, 640, 3333]), (1, 150, 4, 2, 128, 32, [3100])]


@pytest.mark.parametrize("dtype", [BF16, torch.int8, E4M3])
@pytest.mark.parametrize("shape", SHAPES)
def test_cache_attention(dtype, shape):
    from torsh_b200.ops.kv_cache import kv_cache_attention
    q, kp, vp, ks, vs, table, start = _case(*shape, dtype)
    B, T, _, _, D = shape[:5]
    for mask in (None, _random_tree(T, 3)):
        got = kv_cache_attention(q, kp, vp, table, start, mask, None, ks, vs)
        _attention_close(got, *_attend64(q, kp, vp, ks, vs, table, start, mask, None, D ** -0.5), dtype)
    counts = torch.randint(0, T + 1, (B,), device=DEV, generator=_gen(8)).int()
    counts[-1] = T
    mask = torch.rand(B, T, T, device=DEV, generator=_gen(9)) < 0.5        # any mask, one per sequence: rows may see nothing new
    got = kv_cache_attention(q, kp, vp, table, start, mask, counts, ks, vs, scale=0.05)
    _attention_close(got, *_attend64(q, kp, vp, ks, vs, table, start, mask, counts, 0.05), dtype)
    assert all(not got[b, int(n):].any() for b, n in enumerate(counts.tolist()))


@pytest.mark.parametrize("dtype", [BF16, torch.int8, E4M3])
@pytest.mark.parametrize("G", [1, 4, 16, 32])
def test_cache_attention_rows_that_see_nothing(dtype, G):
    from torsh_b200.ops.kv_cache import kv_cache_attention
    q, kp, vp, ks, vs, table, start = _case(3, 5, 2 * G, 2, 64, 16, [0, 0, 20], dtype)
    mask = torch.zeros(5, 5, dtype=torch.bool, device=DEV)
    mask[2, 1] = True
    got = kv_cache_attention(q, kp, vp, table, start, mask, None, ks, vs)
    _attention_close(got, *_attend64(q, kp, vp, ks, vs, table, start, mask, None, 0.125), dtype)
    assert not got[:2, [0, 1, 3, 4]].any()


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("G", [1, 8, 32])
@pytest.mark.parametrize("contexts", [[37, 12], [30037, 20012]])
def test_cache_attention_what_is_not_seen_does_not_reach_a_row(dtype, G, contexts):
    """NaN behind the end of a sequence, and infinities and NaN in new tokens that only some rows see."""
    from torsh_b200.ops.kv_cache import kv_cache_attention
    T, D = 6, 128
    q, kp, vp, ks, vs, table, start = _case(2, T, G, 1, D, 16, contexts, dtype)
    clean = kp.clone(), vp.clone()
    for b in range(2):
        for pos in range(int(start[b]) + T, table.shape[1] * 16):           # never written
            if int(table[b, pos // 16]) >= 0:
                for x in (kp, vp):
                    x.view(torch.int8 if dtype == E4M3 else torch.int16)[int(table[b, pos // 16]), 0, pos % 16] = 0x7F if dtype == E4M3 else 0x7FFF
                if ks is not None:
                    ks[int(table[b, pos // 16]), 0, pos % 16] = math.nan
                    vs[int(table[b, pos // 16]), 0, pos % 16] = math.inf
    mask = torch.eye(T, dtype=torch.bool, device=DEV)
    mask[:, 0] = True
    ref, mass = _attend64(q, *clean, None if ks is None else ks.nan_to_num(1.0), None if vs is None else vs.clamp(max=1.0), table, start, mask, None, D ** -0.5)
    _attention_close(kv_cache_attention(q, kp, vp, table, start, mask, None, ks, vs), ref, mass, dtype)
    pos = int(start[0]) + 3                                                 # new token 3 of sequence 0: only row 3 sees it
    p, r = int(table[0, pos // 16]), pos % 16
    for x in (kp, vp):
        if dtype == BF16:
            x[p, 0, r, 5], x[p, 0, r, 70] = math.inf, math.nan
        else:
            x.view(torch.int8)[p, 0, r, 5] = 0x7F
    if ks is not None:
        ks[p, 0, r] = math.nan
    got = kv_cache_attention(q, kp, vp, table, start, mask, None, ks, vs)
    assert got[0, 3].isnan().any()
    got[0, 3] = ref[0, 3].to(BF16)
    _attention_close(got, ref, mass, dtype)


@pytest.mark.parametrize("dtype", [BF16, torch.int8, E4M3])
def test_cache_attention_scales_of_all_sizes(dtype):
    """Values whose scales differ by 2^80 between tokens, queries from tiny to huge, and scores that underflow against each other."""
    from torsh_b200.ops.kv_cache import kv_cache_attention
    q, kp, vp, ks, vs, table, start = _case(2, 3, 4, 2, 64, 16, [90, 200], dtype)
    q[0, 0] *= 2.0 ** -60
    q[0, 1] *= 8
    q[1, 2, 0, 0], q[1, 2, 1] = 2.0 ** 20, 0
    size = 2.0 ** torch.randint(-40, 40, vp.shape[:3], device=DEV, generator=_gen(4)).float()
    if vs is None:
        vp = (vp.float() * size[..., None]).to(BF16)
    else:
        vs = vs * size
    got = kv_cache_attention(q, kp, vp, table, start, None, None, ks, vs, scale=0.125)
    ref, mass = _attend64(q, kp, vp, ks, vs, table, start, None, None, 0.125)
    # the queries of 2^20 and of 8 times the size: scores up to 2^20, whose error of 130 units of fp32 is up to 2^3: those rows are
    # only compared where one key decides
    hard = torch.zeros(2, 3, 4, 1, dtype=torch.bool, device=DEV)
    hard[1, 2, 0] = True
    hard[0, 1] = True
    p = 2.0 ** -8 if dtype == BF16 else 2.0 ** -11
    off = (got.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + (p + 2.0 ** -13) * 1.01 * mass
    assert (off | hard).all() and torch.isfinite(got).all()
    assert (got.double() - ref)[0, 1].abs().amax() <= (2.0 ** -7 + 2.0 ** -9) * mass[0, 1].amax()


@pytest.mark.parametrize("dtype", [BF16, torch.int8])
def test_cache_attention_of_bad_tables_and_limits(dtype):
    """Pages outside the pool read as zeros; a context longer than its table, or than max_len, is what there is of it."""
    from torsh_b200.ops.kv_cache import kv_cache_attention
    q, kp, vp, ks, vs, table, start = _case(3, 2, 4, 2, 64, 16, [60, 100, 130], dtype)
    table[0, 1], table[1, 0] = 10 ** 6, -5
    got = kv_cache_attention(q, kp, vp, table, start, None, None, ks, vs)
    _attention_close(got, *_attend64(q, kp, vp, ks, vs, table, start, None, None, 0.125), dtype)
    for limit in (0, 1, 50, 61, 96, 131):
        got = kv_cache_attention(q, kp, vp, table, start, None, None, ks, vs, max_len=limit)
        _attention_close(got, *_attend64(q, kp, vp, ks, vs, table, start, None, None, 0.125, limit), dtype)
    long = start + 500
    got = kv_cache_attention(q, kp, vp, table, long, None, None, ks, vs)
    _attention_close(got, *_attend64(q, kp, vp, ks, vs, table, long, None, None, 0.125), dtype)


def test_cache_attention_strides_streams_and_repeats():
    """q out of a packed projection, another stream, a captured call, and the same bits every time."""
    from torsh_b200.ops.kv_cache import kv_cache_attention
    B, T, H, D = 4, 3, 8, 64
    q, kp, vp, ks, vs, table, start = _case(B, T, H, H, D, 16, [1000, 3, 77, 500], E4M3)
    packed = torch.zeros(B, T, 3, H, D, device=DEV, dtype=BF16)
    packed[:, :, 1] = q
    want = kv_cache_attention(q, kp, vp, table, start, None, None, ks, vs)
    assert torch.equal(want, kv_cache_attention(packed[:, :, 1], kp, vp, table, start, None, None, ks, vs))
    assert torch.equal(want, kv_cache_attention(q.transpose(1, 2).contiguous().transpose(1, 2), kp, vp, table.long(), start.long(), None, None, ks, vs))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [kv_cache_attention(q, kp, vp, table, start, None, None, ks, vs) for _ in range(20)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(want, o) for o in outs)
    graphs = []
    for _ in range(2):                                                      # two graphs of the same call do not share a workspace
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            y = kv_cache_attention(q, kp, vp, table, start, None, None, ks, vs)
        graphs.append((gr, y))
    for gr, y in graphs:
        y.zero_()
        gr.replay()
    start += 1
    want = kv_cache_attention(q, kp, vp, table, start, None, None, ks, vs)
    for gr, _ in graphs:
        gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(want, y) for _, y in graphs)


@pytest.mark.parametrize("dtype", [BF16, torch.int8])
def test_cache_offsets_beyond_32_bits(dtype):
    from torsh_b200.ops.kv_cache import kv_cache_attention, kv_cache_read, kv_cache_write
    H, page, D, T = 32, 128, 128, 5
    pages = (1 << 32) // (H * page * D) + 40                               # more than 2^32 elements in a pool
    kp, vp = (torch.empty(pages, H, page, D, dtype=dtype, device=DEV) for _ in range(2))
    ks, vs = (None, None) if dtype == BF16 else (torch.zeros(pages, H, page, device=DEV) for _ in range(2))
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device=DEV)
    g = _gen(11)
    start = torch.zeros(1, dtype=torch.int32, device=DEV)
    k, v = (torch.randn(1, 300, H, D, device=DEV, generator=g).to(BF16) for _ in range(2))
    kv_cache_write(k, v, kp, vp, table, start, None, ks, vs)
    rk, rv = kv_cache_read(kp, vp, table, torch.full((1,), 300, device=DEV), 300, None, ks, vs, torch.float32)
    if dtype == BF16:
        assert torch.equal(rk, k.float()) and torch.equal(rv, v.float())
    else:
        codes, unit = _codes64(v, dtype)
        assert torch.equal(rv, (codes * unit).float())
    q = torch.randn(1, T, H, D, device=DEV, generator=g).to(BF16)
    start.fill_(300 - T)
    got = kv_cache_attention(q, kp, vp, table, start, None, None, ks, vs)
    _attention_close(got, *_attend64(q, kp, vp, ks, vs, table, start, None, None, D ** -0.5), dtype)


# ------------------------------------------------------------------------------------------------ verification
def _verify_inputs(B, T, V, dtype, seed, sharp=4.0):
    g = _gen(seed)
    logits = sharp * torch.randn(B, T, V, device=DEV, generator=g)
    probs = torch.softmax(logits, -1).to(dtype)
    draft = torch.softmax(logits[:, :-1] + 0.5 * torch.randn(B, T - 1, V, device=DEV, generator=g), -1).to(dtype)
    tokens = torch.zeros(B, T, dtype=torch.int64, device=DEV)
    if T > 1:
        tokens[:, 1:] = torch.multinomial(draft.float().view(-1, V), 1, generator=g).view(B, T - 1)
    return probs, draft, tokens, torch.rand(B, T, device=DEV, generator=g)


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
@pytest.mark.parametrize("B,T,V", [(1, 1, 5), (40, 4, 17), (7, 9, 1000), (33, 5, 4097), (3, 33, 50257), (2, 3, 300001)])
def test_verify_draft(dtype, B, T, V):
    from torsh_b200.ops.speculative import _verify_plain, verify_draft
    probs, draft, tokens, u = _verify_inputs(B, T, V, dtype, T + V)
    counts = torch.tensor([max(1, T - i % 4) for i in range(B)], device=DEV, dtype=torch.int32)
    g = torch.Generator().manual_seed(T)
    parents = torch.tensor([-1] + [int(torch.randint(0, i, (1,), generator=g)) for i in range(1, T)], device=DEV)
    best = probs.float().topk(min(4, V), -1).indices
    cand = tokens.clone()
    for i in range(1, T):
        cand[:, i] = best[:, int(parents[i]), i % min(4, V)]
    per_seq = parents.expand(B, T).clone()
    if T > 2:
        per_seq[0, 2] = 1
    calls = [(tokens, draft, None, None), (tokens, draft, None, counts), (tokens, None, None, counts), (cand, None, parents, None), (cand, None, parents, counts), (cand, None, per_seq, counts)]
    for tok, d, par, n in calls:
        got = verify_draft(probs, tok, u, d, par, n)
        want = _verify_plain(probs, tok, u, d, par, n)
        for x, y in zip(got, want):
            assert x.dtype == torch.int64 and torch.equal(x, y)
    if T > 1 and V > 16:
        assert int(verify_draft(probs, tokens, u, draft)[0].max()) > 0


def test_verify_draft_edges():
    """Numbers at the borders, no mass, NaN, tokens and parents outside their range, the same token twice, rows that are views."""
    from torsh_b200.ops.speculative import _verify_plain, verify_draft
    V = 100
    p = torch.zeros(6, 4, 2 * V, device=DEV)[..., :V]                      # strided rows
    p[:, :, 3], p[:, :, 7], p[:, :, 99] = 0.5, 0.25, 0.25
    p[1] = 0
    p[2, :, 3] = math.nan
    p[3, :, 7] = -1.0
    tokens = torch.tensor([[0, 3, 3, 7], [0, 3, 7, 9], [0, 7, 3, 99], [0, 99, 7, 3], [0, -1, 200, 3], [0, 99, 99, 99]], device=DEV)
    parents = torch.tensor([[-1, 0, 0, 0], [-1, 0, 1, 1], [-1, 0, 1, 2], [-1, 0, 0, 1], [-1, 0, 0, 0], [-1, 3, -7, 0]], device=DEV)
    for x in (0.0, 0.25, 0.5, 0.499999, 0.75, 0.999999, 1.0):
        u = torch.full((6, 4), x, device=DEV)
        for d, par in ((None, None), (None, parents), (p[:, :-1].flip(0).contiguous(), None), (p[:, :-1], None)):
            for a, b in zip(verify_draft(p, tokens, u, d, par), _verify_plain(p, tokens, u, d, par)):
                assert torch.equal(a, b)
    assert verify_draft(p, tokens, u)[2][1] == -1


@pytest.mark.parametrize("form", ["draft", "chain", "tree"])
def test_verify_draft_keeps_the_targets_distribution(form):
    """The first token that comes out (accepted or drawn) has the target's distribution: counts of 40000 independent sequences, each within
    six standard deviations of a binomial."""
    from torsh_b200.ops.speculative import verify_draft
    B, T, V = 40000, 3, 11
    g = _gen(21)
    p1 = torch.softmax(torch.randn(1, T, V, device=DEV, generator=g), -1)
    q1 = torch.softmax(torch.randn(1, T - 1, V, device=DEV, generator=g), -1)
    probs, u = p1.expand(B, T, V), torch.rand(B, T, device=DEV, generator=g)
    tokens = torch.zeros(B, T, dtype=torch.int64, device=DEV)
    if form == "draft":
        tokens[:, 1] = torch.multinomial(q1[0, 0], B, True, generator=g)
        tokens[:, 2] = torch.multinomial(q1[0, 1], B, True, generator=g)
        acc, path, nxt = verify_draft(probs, tokens, u, q1.expand(B, T - 1, V))
    else:
        tokens[:, 1], tokens[:, 2] = 4, 8
        acc, path, nxt = verify_draft(probs, tokens, u, None, torch.tensor([-1, 0, 0], device=DEV) if form == "tree" else None)
    first = torch.where(acc > 0, tokens.gather(1, path[:, 1:2].clamp(min=0))[:, 0], nxt)
    want = p1[0, 0].double()
    got = torch.bincount(first, minlength=V).double() / B
    assert ((got - want).abs() <= 6 * (want * (1 - want) / B).sqrt()).all()


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("dtype", [BF16, torch.int8, E4M3])
def test_a_tree_step_through_the_cache(dtype):
    """Rotary, write, attention of a tree, verification and keeping the accepted path, against the same tokens fed one by one."""
    from torsh_b200.ops.kv_cache import PagedKVCache, tree_mask_of
    from torsh_b200.ops.rotary import rotary, rotary_frequencies
    from torsh_b200.ops.speculative import verify_draft
    B, H, Hk, D, T, V = 3, 8, 2, 64, 7, 50
    g = _gen(31)
    freqs, m = rotary_frequencies(D, scaling="wavelength", factor=8.0, device=DEV)
    parents = torch.tensor([-1, 0, 0, 1, 2, 4, 4], device=DEV)
    mask = tree_mask_of(parents)
    depth = mask.sum(-1) - 1
    cache = PagedKVCache(1, Hk, D, B, 300, dtype=dtype, page=16)
    chain = PagedKVCache(1, Hk, D, B, 300, dtype=dtype, page=48)
    n0 = torch.tensor([5, 130, 64], device=DEV)
    kv = torch.randn(2, B, 140, Hk, D, device=DEV, generator=g).to(BF16)
    for c in (cache, chain):
        c.reserve([140] * B)
        c.write(0, kv[0], kv[1], counts=n0)
        c.advance(n0.tolist())
    q, k, v = (torch.randn(B, T, h, D, device=DEV, generator=g).to(BF16) for h in (H, Hk, Hk))
    pos = n0[:, None] + depth
    qr, kr = rotary(q, k, pos, freqs, False, m)
    cache.reserve(T)
    cache.write(0, kr, v)
    out = cache.attend(0, qr, mask)
    probs = torch.softmax(4 * torch.randn(B, T, V, device=DEV, generator=g), -1)
    tokens = torch.zeros(B, T, dtype=torch.int64, device=DEV)
    top = probs.topk(2, -1).indices
    tokens[:, 1:] = top[:, parents[1:], torch.tensor([0, 1, 0, 0, 0, 1], device=DEV)]
    u = torch.rand(B, T, device=DEV, generator=g) * 0.8
    acc, path, nxt = verify_draft(probs, tokens, u, None, parents)
    cache.keep(path, acc)
    cache.advance(acc + 1)
    # one by one along the accepted path
    for i in range(int(acc.max()) + 1):
        at = path[:, i].clamp(min=0)
        pick = lambda x: x[torch.arange(B, device=DEV), at][:, None]   # noqa: E731
        live = (i <= acc).int()
        chain.reserve(1)
        chain.write(0, pick(kr), pick(v), counts=live)
        one = chain.attend(0, pick(qr), counts=live)
        chain.advance(live.tolist())
        for b in range(B):
            if live[b]:
                torch.testing.assert_close(one[b, 0].float(), out[b, at[b]].float(), rtol=2.0 ** -6, atol=2.0 ** -6)   # two bf16 roundings of P and O each
    assert cache.host_lengths == chain.host_lengths
    for x, y in zip(cache.read(0), chain.read(0)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("cache_dtype", [BF16, E4M3])
def test_llama_decodes_from_the_cache(cache_dtype):
    """Hidden states of the last tokens, prompt and steps through the cache, are as near to fp32 as those of the whole context run at once
    (twice as far at most; an e4m3 cache rounds keys and values by 2^-4 where bf16 does by 2^-8: sixteen times)."""
    from torsh_b200.models.llama import LlamaConfig, LlamaModel
    torch.manual_seed(0)
    cfg = LlamaConfig.tiny(num_layers=3, initializer_range=0.05)
    m = LlamaModel(cfg).to(DEV, BF16).eval()
    ref = LlamaModel(cfg).double().eval()
    ref.load_state_dict({k: v.double().cpu() for k, v in m.state_dict().items()})
    ids = torch.randint(0, cfg.vocab_size, (3, 70), device=DEV)
    with torch.no_grad():
        want = ref.decode(ids.cpu(), ref.make_cache(3, 80)).view(3, 70, -1)
        whole = m.decode(ids, _primed(m, 3, 80, BF16, 70)).view(3, 70, -1)
        c = _primed(m, 3, 80, cache_dtype, 60)
        got = [m.decode(ids[:, :60], c).view(3, 60, -1)]
        c.advance(60)
        for i in range(60, 70):
            c.reserve(1)
            got.append(m.decode(ids[:, i:i + 1], c).view(3, 1, -1))
            c.advance(1)
    got = torch.cat(got, 1)
    off = lambda x: (x.double().cpu() - want).norm()   # noqa: E731
    assert off(got) <= (2 if cache_dtype == BF16 else 16) * off(whole)
    out = m.generate(ids[:, :9], 12, draft=m, drafted=3, cache_dtype=cache_dtype)
    assert out.shape == (3, 21) and torch.equal(out[:, :9], ids[:, :9])


def _primed(m, batch, most, dtype, n):
    c = m.make_cache(batch, most, dtype, page=16)
    c.reserve(n)
    return c


# ------------------------------------------------------------------------------------------------ at the edges of the documentation
@pytest.mark.parametrize("G", [2, 24])
@pytest.mark.parametrize("dtype", [torch.int8, E4M3])
def test_cache_attention_scales_below_zero(dtype, G):
    """Scales of a caller's own may have any sign."""
    from torsh_b200.ops.kv_cache import kv_cache_attention
    q, kp, vp, ks, vs, table, start = _case(2, 3, 2 * G, 2, 128, 16, [300, 41], dtype)
    ks, vs = (x * torch.where(torch.rand(x.shape, device=DEV, generator=_gen(i)) < 0.5, -1, 1) for i, x in enumerate((ks, vs)))
    got = kv_cache_attention(q, kp, vp, table, start, None, None, ks, vs)
    _attention_close(got, *_attend64(q, kp, vp, ks, vs, table, start, None, None, 128 ** -0.5), dtype)


@pytest.mark.parametrize("dtype", [BF16, torch.int8])
@pytest.mark.parametrize("shape", [(2, 1500, 4, 2, 64, 48, [0, 70]), (1, 700, 2, 1, 128, 80, [0]), (4, 20, 3, 3, 64, 16, [5, 0, 33, 1])])
def test_cache_attention_of_a_prompt(dtype, shape):
    """Prompts: many row tiles that begin in the middle of a key tile, most of them without a context, with pages of no power of two."""
    from torsh_b200.ops.kv_cache import kv_cache_attention
    q, kp, vp, ks, vs, table, start = _case(*shape, dtype)
    B, T, _, _, D = shape[:5]
    got = kv_cache_attention(q, kp, vp, table, start, None, None, ks, vs)
    _attention_close(got, *_attend64(q, kp, vp, ks, vs, table, start, None, None, D ** -0.5), dtype)
    # a mask that is a view of a larger one, off any boundary and with rows of odd length
    big = torch.rand(T + 3, T + 5, device=DEV, generator=_gen(T)) < 0.3
    mask = big[1:T + 1, 3:T + 3]
    got = kv_cache_attention(q, kp, vp, table, start, mask, None, ks, vs)
    _attention_close(got, *_attend64(q, kp, vp, ks, vs, table, start, mask, None, D ** -0.5), dtype)
    assert torch.equal(got, kv_cache_attention(q, kp, vp, table, start, mask.contiguous(), None, ks, vs))


def test_cache_calls_on_many_sequences_and_on_none():
    from torsh_b200.ops.kv_cache import kv_cache_attention, kv_cache_read, kv_cache_write
    B = 70000
    kp, vp, ks, vs = _cache(300, 1, 16, 64, torch.int8, 1)
    table = (torch.arange(B, device=DEV) % 300).int()[:, None]
    start = (torch.arange(B, device=DEV) % 17 - 1).int()                    # a negative start is no context
    q = torch.randn(B, 1, 2, 64, device=DEV, generator=_gen(0)).to(BF16)
    got = kv_cache_attention(q, kp, vp, table, start, None, None, ks, vs)
    want = torch.where((start >= 16)[:, None, None, None], 7.0, 7.0)        # every value is code 1 times scale 7
    assert ((got.float() - want).abs() <= 7 * 2.0 ** -8).all()
    for n in (0, 1):
        e, t = q[:n], table[:n]
        assert kv_cache_attention(e, kp, vp, t, start[:n], None, None, ks, vs).shape == e.shape
        assert kv_cache_attention(e[:, :0], kp, vp, t, start[:n], None, None, ks, vs).shape == (n, 0, 2, 64)
        assert kv_cache_read(kp, vp, t, start[:n], 0, None, ks, vs)[0].shape == (n, 0, 1, 64)
    kv_cache_write(q[:0, :, :1], q[:0, :, :1], kp, vp, table[:0], start[:0], None, ks, vs)
    for pool, wide in ((0, 1), (300, 0)):                                   # an empty pool, a table without columns
        args = kp[:pool], vp[:pool], table[:3, :wide]
        kv_cache_write(q[:3, :, :1], q[:3, :, :1], *args, start[:3], None, ks[:pool], vs[:pool])
        assert not kv_cache_read(*args, start[3:6], 4, None, ks[:pool], vs[:pool])[0].any()
        assert not kv_cache_attention(q[:3], *args, start[3:6], None, None, ks[:pool], vs[:pool]).any()


def test_cache_integers_beyond_32_bits_are_not_wrapped():
    from torsh_b200.ops.kv_cache import kv_cache_attention, kv_cache_read, kv_cache_write
    kp, vp, _, _ = _cache(2, 1, 16, 64, BF16, 0)
    table = torch.tensor([[0], [1]], device=DEV)
    k = torch.ones(2, 4, 1, 64, device=DEV, dtype=BF16)
    for tab, start in ((table, [1 << 32, -(1 << 32)]), (table, [-1, 1 << 31]), (table + (1 << 32), [0, 0])):
        kv_cache_write(k, k, kp, vp, tab, torch.tensor(start, device=DEV))
        kv_cache_write(k, k, kp, vp, tab.clamp(max=2 ** 31 - 1).int(), torch.tensor(start, device=DEV).clamp(-2 ** 31, 2 ** 31 - 1).int())
    assert not kp.any()
    kv_cache_write(k, k, kp, vp, table, torch.tensor([0, 12], device=DEV))
    big = torch.tensor([2 ** 31 - 1, 1 << 40], device=DEV)
    rk, _ = kv_cache_read(kp, vp, table, big, 16)
    assert torch.equal(rk[:, :, 0], kp[:, 0])
    assert not kv_cache_read(kp, vp, table, big, 16, big)[0].any()
    got = kv_cache_attention(k, kp, vp, table, big, scale=0.0)              # all that the tables reach, alike: a quarter is ones
    assert got.eq(0.25).all()


def test_bad_pages_are_reported_where_the_checks_are_on():
    from torsh_b200 import _native as nv
    from torsh_b200.ops.kv_cache import kv_cache_attention, kv_cache_read, kv_cache_write
    q, kp, vp, ks, vs, table, start = _case(2, 20, 2, 1, 64, 16, [60, 3], E4M3)
    bad = table.clone()
    bad[0, 2] = kp.shape[0]
    calls = [lambda t: kv_cache_write(q[:, :, :1], q[:, :, :1], kp, vp, t, start - 28, None, ks, vs), lambda t: kv_cache_read(kp, vp, t, start, 60, None, ks, vs),
             lambda t: kv_cache_attention(q[:, :1], kp, vp, t, start, None, None, ks, vs), lambda t: kv_cache_attention(q, kp, vp, t, start, None, None, ks, vs)]
    nv.check_status()
    nv.enable_kernel_checks(True)
    try:
        for call in calls:
            call(table.clamp(min=0))
            if call is not calls[0]:
                nv.check_status()
            else:                                                           # the second sequence begins in front of position 0
                with pytest.raises(nv.KernelCheckFailed):
                    nv.check_status()
            call(bad.clamp(min=0))
            with pytest.raises(nv.KernelCheckFailed):
                nv.check_status()
        nv.check_status()
    finally:
        nv.enable_kernel_checks(False)
    kv_cache_attention(q, kp, vp, bad, start, None, None, ks, vs)
    nv.check_status()


def test_rotary_offsets_beyond_32_bits():
    from torsh_b200.ops.rotary import rotary, rotary_frequencies
    N, H, D = 600_000, 32, 128                                              # 2.5e9 elements
    q = torch.empty(N, H, D, device=DEV, dtype=BF16)
    for i in range(0, N, 100_000):
        q[i:i + 100_000].normal_()
    freqs, _ = rotary_frequencies(64, device=DEV)
    pos = torch.arange(N, device=DEV)
    y, _ = rotary(q, None, pos, freqs, False)
    for i in (0, 262_000, 524_280, N - 40):
        s = slice(i, i + 40)
        _rotary_close(y[s], q[s], _turn64(q[s], pos[s], freqs, False, 1.0), 1.0)


def test_captured_calls_and_calls_on_two_streams():
    """Each operator captured and replayed over new contents, and run on two streams at once from two threads."""
    import threading
    from torsh_b200.ops.kv_cache import kv_cache_attention, kv_cache_read, kv_cache_write
    from torsh_b200.ops.rotary import rotary, rotary_frequencies
    from torsh_b200.ops.speculative import verify_draft
    B, T, H, D, V = 3, 24, 4, 64, 500
    freqs, _ = rotary_frequencies(D, device=DEV)
    table = torch.arange(B * 8, device=DEV).int().view(B, 8)

    def make(seed):
        g = _gen(seed)
        q, k, v = (torch.randn(B, T, H, D, device=DEV, generator=g).to(BF16) for _ in range(3))
        start = torch.randint(0, 90, (B,), device=DEV, generator=g).int()
        return [q, k, v, start, *_verify_inputs(B, T, V, torch.float32, seed)]

    def step(x, pages):
        q, k, v, start, probs, draft, tokens, u = x
        pos = start.long()[:, None] + torch.arange(T, device=DEV)
        q, k = rotary(q, k, pos, freqs)
        kv_cache_write(k, v, *pages[:2], table, start, None, *pages[2:])
        out = kv_cache_attention(q, *pages[:2], table, start, None, None, *pages[2:])
        back = kv_cache_read(*pages[:2], table, start + T, 128, None, *pages[2:])
        return [out, *back, *verify_draft(probs, tokens, u, draft), *verify_draft(probs, tokens, u)]

    def pool():
        return _cache(B * 8, H, 16, D, torch.int8, 0)

    inputs = [make(i) for i in range(4)]
    want = [step(x, pool()) for x in inputs]
    held, pages = [t.clone() for t in inputs[0]], pool()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(held, pages)
    for x, w in zip(inputs, want):
        for p in pages:
            p.zero_()
        for a, b in zip(held, x):
            a.copy_(b)
        clean = pool()
        for p, c in zip(pages, clean):
            p.copy_(c)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(outs, w))
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            pages = pool()
            for _ in range(20):
                for p, c in zip(pages, pool()):
                    p.copy_(c)
                got[i] = step(inputs[i], pages)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))


def test_rotary_backward_in_a_graph():
    from torsh_b200.ops.rotary import rotary, rotary_frequencies
    freqs, _ = rotary_frequencies(64, device=DEV)
    pos = torch.arange(9, device=DEV).expand(2, 9).contiguous()
    x = torch.randn(2, 9, 4, 64, device=DEV, generator=_gen(6)).requires_grad_()
    dy = torch.randn_like(x)

    def both():
        yq, yk = rotary(x, x * 2, pos, freqs, False)
        return torch.autograd.grad((yq, yk), x, (dy, dy))[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dx = both()
    dx.zero_()
    graph.replay()
    assert torch.equal(dx, want)
    _rotary_close(dx, dy, 3 * _turn64(dy, pos, freqs, False, 1.0, True), 3.0)


def test_verify_draft_of_what_is_no_probability():
    """Infinities, and numbers outside [0, 1): whatever comes out is in range."""
    from torsh_b200.ops.speculative import verify_draft
    B, T, V = 6, 5, 3001
    probs, draft, tokens, u = _verify_inputs(B, T, V, torch.float32, 3)
    probs[0, :, 5], probs[1], draft[2] = math.inf, math.inf, math.inf
    probs[3] = 3e38
    u[4], u[5] = math.nan, -2.0
    u[:2, T - 1] = 0
    for d in (draft, None):
        acc, path, nxt = verify_draft(probs, tokens, u, d)
        assert ((acc >= 0) & (acc < T)).all() and ((path >= -1) & (path < T)).all() and ((nxt >= -1) & (nxt < V)).all()
        assert torch.equal((path >= 0).sum(1), acc + 1)


def test_a_captured_step_of_a_paged_cache_goes_on():
    """A tree step - write, attend, verify, keep, advance - captured once and replayed while the sequences grow, beside a place without one."""
    from torsh_b200.ops.kv_cache import PagedKVCache, tree_mask_of
    from torsh_b200.ops.speculative import verify_draft
    B, T, H, D, V = 3, 5, 2, 64, 40
    parents = torch.tensor([-1, 0, 0, 1, 2], device=DEV)
    mask = tree_mask_of(parents)
    g = _gen(9)
    steps = [[torch.randn(B, T, H, D, device=DEV, generator=g).to(BF16) for _ in range(3)]
             + [torch.softmax(3 * torch.randn(B, T, V, device=DEV, generator=g), -1), torch.randint(0, V, (B, T), device=DEV, generator=g), torch.rand(B, T, device=DEV, generator=g)]
             for _ in range(12)]

    def make():
        c = PagedKVCache(1, H, D, batch=B, max_len=96, dtype=torch.int8, page=16, num_pages=12, device=DEV)
        c.reserve([96, 0, 70])
        return c

    def step(c, x):
        q, k, v, probs, tokens, u = x
        c.write(0, k, v)
        out = c.attend(0, q, mask)
        acc, path, nxt = verify_draft(probs, tokens, u, None, parents)
        c.keep(path, acc)
        c.advance(acc + 1, most=T)
        return out, acc, nxt

    eager = make()
    want = [[y.clone() for y in step(eager, x)] for x in steps]
    assert int(eager.lengths.max()) > 2 * T                                # beyond what there was at the capture
    held, c = [x.clone() for x in steps[0]], make()
    table = c.page_table.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(c, held)
    for x, w in zip(steps, want):
        for a, b in zip(held, x):
            a.copy_(b)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(outs, w))
        assert not outs[0][1].any()
    assert torch.equal(c.lengths, eager.lengths) and torch.equal(c.page_table, table)
    for (a, b), (sa, sb) in ((c.layers[0], c.scales[0]),):
        (ea, eb), (esa, esb) = eager.layers[0], eager.scales[0]
        assert torch.equal(a, ea) and torch.equal(b, eb) and torch.equal(sa, esa) and torch.equal(sb, esb)


@pytest.mark.parametrize("dtype", [BF16, torch.int8, E4M3])
@pytest.mark.parametrize("wide", [0, 5000])
@pytest.mark.parametrize("shape", [(3, 5, 64, 2, 64, 16, [0, 0, 20]), (2, 3, 48, 2, 128, 16, [300, 41]), (2, 33, 3, 1, 64, 16, [16, 250]), (2, 6, 32, 1, 128, 16, [37, 12]),
                                   (4, 20, 3, 3, 64, 16, [5, 0, 33, 1]), (5, 17, 4, 2, 128, 48, [127, 128, 0, 129, 1]), (1, 1, 20, 1, 64, 16, [0])])
def test_cache_attention_of_short_sequences_in_short_and_wide_tables(dtype, wide, shape):
    """The width of the table decides which kernel takes many rows over little: both, with rows that see nothing, counts, scales below zero,
    and infinities and NaN in new tokens that other rows do not see."""
    from torsh_b200.ops.kv_cache import kv_cache_attention
    q, kp, vp, ks, vs, table, start = _case(*shape, dtype)
    B, T, _, H, D = shape[:5]
    table = torch.nn.functional.pad(table, (0, wide), value=-1)
    if ks is not None:
        ks, vs = (x * torch.where(torch.rand(x.shape, device=DEV, generator=_gen(i)) < 0.5, -1, 1) for i, x in enumerate((ks, vs)))
    g = _gen(T)
    counts = torch.randint(0, T + 1, (B,), device=DEV, generator=g).int()
    counts[0] = T
    for mask, n in ((None, None), (torch.rand(T, T, device=DEV, generator=g) < 0.3, None), (torch.rand(B, T, T, device=DEV, generator=g) < 0.5, counts)):
        got = kv_cache_attention(q, kp, vp, table, start, mask, n, ks, vs)
        _attention_close(got, *_attend64(q, kp, vp, ks, vs, table, start, mask, n, D ** -0.5), dtype)
    mask = torch.eye(T, dtype=torch.bool, device=DEV)
    ref, mass = _attend64(q, kp, vp, ks, vs, table, start, mask, None, D ** -0.5)
    pos = int(start[0]) + T // 2                                            # only row T // 2 of sequence 0 sees it
    p, r = int(table[0, pos // shape[5]]), pos % shape[5]
    if dtype == BF16:
        vp[p, :, r, 3], vp[p, :, r, D - 1], kp[p, :, r, 5] = math.inf, math.nan, math.nan
    else:
        vs[p, :, r], ks[p, :, r] = math.inf, math.nan
    got = kv_cache_attention(q, kp, vp, table, start, mask, None, ks, vs)
    assert got[0, T // 2].isnan().any()
    got[0, T // 2] = ref[0, T // 2].to(BF16)
    _attention_close(got, ref, mass, dtype)


@pytest.mark.parametrize("dtype", [BF16, torch.int8])
@pytest.mark.parametrize("wide", [0, 5000])
def test_cache_attention_of_queries_that_are_no_numbers(dtype, wide):
    """A query with an infinity or a NaN spoils its own row."""
    from torsh_b200.ops.kv_cache import kv_cache_attention
    q, kp, vp, ks, vs, table, start = _case(2, 9, 8, 2, 64, 16, [200, 3], dtype)
    table = torch.nn.functional.pad(table, (0, wide), value=-1)
    ref, mass = _attend64(q, kp, vp, ks, vs, table, start, None, None, 0.125)
    bad = q.clone()
    bad[0, 4, 3, 5], bad[1, 0, 0, 0], bad[1, 8, 7] = math.nan, math.inf, math.nan
    got = kv_cache_attention(bad, kp, vp, table, start, None, None, ks, vs)
    for at in ((0, 4, 3), (1, 0, 0), (1, 8, 7)):
        assert got[at].isnan().any()
        got[at] = ref[at].to(BF16)
    _attention_close(got, ref, mass, dtype)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_cache_attention_of_many_rows_captured_and_on_several_streams(dtype):
    import threading
    from torsh_b200.ops.kv_cache import kv_cache_attention
    q, kp, vp, ks, vs, table, start = _case(6, 30, 8, 4, 64, 16, [900, 3, 77, 500, 0, 1300], dtype)
    table = torch.nn.functional.pad(table, (0, 2000), value=-1)
    starts = [start, start // 2, start // 3, torch.zeros_like(start)]
    want = [kv_cache_attention(q, kp, vp, table, s, None, None, ks, vs) for s in starts]
    held, graphs = start.clone(), []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = kv_cache_attention(q, kp, vp, table, held, None, None, ks, vs)
        graphs.append((graph, out))
    for s, w in zip(starts, want):
        held.copy_(s)
        for graph, out in graphs:
            out.zero_()
            graph.replay()
        assert all(torch.equal(out, w) for _, out in graphs)
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            outs = [kv_cache_attention(q, kp, vp, table, starts[i], None, None, ks, vs) for _ in range(25)]
            torch.cuda.current_stream().synchronize()
            got[i] = outs

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(o, w) for outs, w in zip(got, want) for o in outs)
