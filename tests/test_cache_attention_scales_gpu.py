"""8-bit values whose scales differ by any factor: every row is as exact as its own values allow, whatever the scales of tokens that it does not
see or hardly attends to."""
import math

import pytest
import torch

from test_decoding_gpu import DEV, E4M3, _attend64, _case, _gen, _random_tree

pytestmark = pytest.mark.gpu


def _close(got, ref, mass, weight, n):
    """P (times a scale) is rounded to halves (2^-11) and the output to bf16 (2^-8); scores as in the operators' tests, 2^-13. Halves below
    2^-14 are off by 2^-25 at most; the largest of a row is 2^8 at least, so that is 2^-33 of the row's largest product `weight` of a probability and a
    scale, for each of n tokens, times a code of 448 at most."""
    assert torch.isfinite(got).all()
    off = (got.double() - ref).abs() - 2.0 ** -8 * ref.abs() - (2.0 ** -11 + 2.0 ** -13) * 1.01 * mass - n * 448 * 2.0 ** -33 * weight[..., None]
    assert (off <= 0).all(), float(off.max())


def _weight(q, kp, ks, vs, table, start, mask, scale, H, page):
    """The largest p * |scale| of each row, and the number of tokens."""
    B, T, Hq, D = q.shape
    out = torch.zeros(B, T, Hq, dtype=torch.float64, device=DEV)
    most = 0
    for b in range(B):
        s0 = int(start[b])
        at = torch.arange(s0 + T, device=DEV)
        most = max(most, s0 + T)
        slot, row = table[b].long()[at // page], at % page
        seen = torch.ones(T, s0 + T, dtype=torch.bool, device=DEV)
        seen[:, s0:] = mask
        for h in range(Hq):
            hk = h // (Hq // H)
            k = (kp.view(torch.int8) if kp.dtype == E4M3 else kp)[slot, hk, row].view(kp.dtype).double() * ks[slot, hk, row].double()[:, None]
            p = torch.softmax(torch.where(seen, (q[b, :, h].double() @ k.T) * scale, -math.inf), -1)
            out[b, :, h] = (p * vs[slot, hk, row].double().abs()).amax(-1)
    return out, most


# few rows whole and cut, many rows in short tables (few rows' kernel) and wide ones (tcgen05), whole and cut, several row tiles
SHAPES = [((2, 6, 2, 1, 128, 16, [37, 120]), 0), ((1, 3, 8, 2, 64, 16, [30037]), 0), ((2, 40, 2, 1, 64, 16, [21, 300]), 0), ((2, 40, 2, 1, 64, 16, [21, 300]), 5000),
          ((1, 30, 4, 2, 128, 16, [20037]), 0), ((2, 150, 2, 1, 128, 48, [7, 260]), 5000)]


@pytest.mark.parametrize("dtype", [torch.int8, E4M3])
@pytest.mark.parametrize("up", [20, 45, 90])
@pytest.mark.parametrize("shape,wide", SHAPES)
def test_a_large_scale_does_not_reach_rows_that_do_not_see_it(dtype, up, shape, wide):
    from torsh_b200.ops.kv_cache import kv_cache_attention
    q, kp, vp, ks, vs, table, start = _case(*shape, dtype)
    B, T, Hq, H, D, page = shape[:6]
    table = torch.nn.functional.pad(table, (0, wide), value=-1)
    mask = _random_tree(T, 5)
    for b in range(B):                                                      # token 1 of the new ones: its branch sees it, others do not
        pos = int(start[b]) + 1
        vs[int(table[b, pos // page]), :, pos % page] *= 2.0 ** up
    assert not mask[:, 1].all()
    got = kv_cache_attention(q, kp, vp, table, start, mask, None, ks, vs)
    ref, mass = _attend64(q, kp, vp, ks, vs, table, start, mask, None, D ** -0.5)
    _close(got, ref, mass, *_weight(q, kp, ks, vs, table, start, mask, D ** -0.5, H, page))


@pytest.mark.parametrize("dtype", [torch.int8, E4M3])
@pytest.mark.parametrize("shape,wide", SHAPES)
def test_a_large_scale_that_no_row_attends_to(dtype, shape, wide):
    """In the context, 2^40 times the others, under keys with e^-60 of their probability: the others decide."""
    from torsh_b200.ops.kv_cache import kv_cache_attention
    q, kp, vp, ks, vs, table, start = _case(*shape, dtype)
    B, T, Hq, H, D, page = shape[:6]
    table = torch.nn.functional.pad(table, (0, wide), value=-1)
    mask = _random_tree(T, 5)
    q = q.abs() + 0.5                                                       # so that one key is far from all queries
    k8 = kp.view(torch.int8) if dtype == E4M3 else kp
    for b in range(B):
        pos = int(start[b]) // 2
        p, r = int(table[b, pos // page]), pos % page
        k8[p, :, r] = torch.full((D,), -100.0, device=DEV).to(dtype).view(torch.int8)
        ks[p, :, r] = 60 * math.sqrt(D) / (100 * 0.5 * D)                    # q . k / sqrt(D) <= -60
        vs[p, :, r] *= 2.0 ** 40
    got = kv_cache_attention(q, kp, vp, table, start, mask, None, ks, vs)
    ref, mass = _attend64(q, kp, vp, ks, vs, table, start, mask, None, D ** -0.5)
    # larger queries: scores up to sum |q k| / sqrt(D), off by at most 130 units of it
    big = float((q.double().abs().sum(-1).amax() * (kp.double().abs().amax(-1) * ks.double()).amax()) / math.sqrt(D))
    weight, n = _weight(q, kp, ks, vs, table, start, mask, D ** -0.5, H, page)
    assert torch.isfinite(got).all()
    off = (got.double() - ref).abs() - 2.0 ** -8 * ref.abs() - (2.0 ** -11 + 2 * 130 * 2.0 ** -24 * big) * 1.01 * mass - n * 448 * 2.0 ** -33 * weight[..., None]
    assert (off <= 0).all(), float(off.max())


@pytest.mark.parametrize("dtype", [torch.int8, E4M3])
@pytest.mark.parametrize("spread", [10, 30, 50])
@pytest.mark.parametrize("shape,wide", SHAPES)
def test_scales_of_any_size_and_sign(dtype, spread, shape, wide):
    """Each token's scale 2^-spread to 2^spread times as large, some zero, of either sign, under any mask."""
    from torsh_b200.ops.kv_cache import kv_cache_attention
    q, kp, vp, ks, vs, table, start = _case(*shape, dtype)
    B, T, Hq, H, D, page = shape[:6]
    g = _gen(spread)
    table = torch.nn.functional.pad(table, (0, wide), value=-1)
    vs = vs * 2.0 ** ((2 * torch.rand(vs.shape, device=DEV, generator=g) - 1) * spread)
    vs = torch.where(torch.rand(vs.shape, device=DEV, generator=g) < 0.1, 0.0, vs) * torch.where(torch.rand(vs.shape, device=DEV, generator=g) < 0.5, -1, 1)
    mask = torch.rand(T, T, device=DEV, generator=g) < 0.4
    mask |= torch.eye(T, dtype=torch.bool, device=DEV)
    got = kv_cache_attention(q, kp, vp, table, start, mask, None, ks, vs)
    ref, mass = _attend64(q, kp, vp, ks, vs, table, start, mask, None, D ** -0.5)
    _close(got, ref, mass, *_weight(q, kp, ks, vs, table, start, mask, D ** -0.5, H, page))


@pytest.mark.parametrize("dtype", [torch.int8, E4M3])
@pytest.mark.parametrize("size", [2.0 ** -91, 2.0 ** -50, 2.0 ** 30, 2.0 ** 105])
@pytest.mark.parametrize("shape,wide", SHAPES)
def test_scales_at_the_ends_of_what_pages_hold(dtype, size, shape, wide):
    """All values tiny or huge; and values of nothing but zeros, which still share in the softmax."""
    from torsh_b200.ops.kv_cache import kv_cache_attention
    q, kp, vp, ks, _, table, start = _case(*shape, dtype)
    B, T, Hq, H, D, page = shape[:6]
    g = _gen(1)
    table = torch.nn.functional.pad(table, (0, wide), value=-1)
    vs = size * (1 + torch.rand(ks.shape, device=DEV, generator=g))
    if 2.0 ** -61 < size < 2.0 ** 61:
        vs = torch.where(torch.rand(vs.shape, device=DEV, generator=g) < 0.3, 0.0, vs)
    mask = _random_tree(T, 5)
    got = kv_cache_attention(q, kp, vp, table, start, mask, None, ks, vs)
    ref, mass = _attend64(q, kp, vp, ks, vs, table, start, mask, None, D ** -0.5)
    _close(got, ref, mass, *_weight(q, kp, ks, vs, table, start, mask, D ** -0.5, H, page))
    assert not kv_cache_attention(q, kp, vp, table, start, mask, None, ks, torch.zeros_like(vs)).any()


@pytest.mark.parametrize("dtype", [torch.int8, E4M3])
@pytest.mark.parametrize("shape,wide", SHAPES)
def test_scales_beyond_the_ends_are_none_and_infinite(dtype, shape, wide):
    """As documented: 2^122 and more is no finite number to the rows that see it, and nothing to the others; less than 2^-92 is zero."""
    from torsh_b200.ops.kv_cache import kv_cache_attention
    q, kp, vp, ks, vs, table, start = _case(*shape, dtype)
    B, T, Hq, H, D, page = shape[:6]
    table = torch.nn.functional.pad(table, (0, wide), value=-1)
    mask = _random_tree(T, 5)
    call = lambda: kv_cache_attention(q, kp, vp, table, start, mask, None, ks, vs)   # noqa: E731
    at = [(int(table[b, (int(start[b]) + 1) // page]), (int(start[b]) + 1) % page) for b in range(B)]   # token 1 of the new ones
    for p, r in at:
        vs[p, :, r] = 2.0 ** -93
    small = call()
    for p, r in at:
        vs[p, :, r] = 0
    assert torch.equal(small, call())
    ref, mass = _attend64(q, kp, vp, ks, vs, table, start, mask, None, D ** -0.5)
    for scale in (2.0 ** 122, -2.0 ** 127):
        for p, r in at:
            vs[p, :, r] = scale
        got = call()
        seen = mask[:, 1]
        assert not torch.isfinite(got[:, seen]).any()
        got[:, seen] = ref[:, seen].to(got.dtype)
        _close(got, ref, mass, *_weight(q, kp, ks, torch.where(vs.abs() >= 2.0 ** 122, 0.0, vs), table, start, mask, D ** -0.5, H, page))
