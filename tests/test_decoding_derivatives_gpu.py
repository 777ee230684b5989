"""Derivatives of the decoding operators on a GPU that the kernels do not compute themselves: forward mode, learned frequencies, batched
gradients. Each against the formula in 64 bits.

Tolerances: fp32 inputs. Sines and cosines, two products and a sum in fp32 are off by at most 8 units of 2^-24 of magnitude * 2 max|x|, as in the
tests of the operators.
"""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = 2.0 ** -24


def _gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def _setup(interleaved, D=64, R=32, B=2, T=3):
    from torsh_b200.ops.rotary import rotary_frequencies
    g = _gen(D + R)
    q, k, dq, dk = (torch.randn(B, T, h, D, device=DEV, generator=g) for h in (4, 2, 4, 2))
    pos = torch.randint(0, 5000, (B, T), device=DEV, generator=g)
    return q, k, dq, dk, pos, rotary_frequencies(R, device=DEV)[0]


def _turn64(x, pos, freqs, interleaved, magnitude=1.0, inverse=False):
    h, R = freqs.numel(), 2 * freqs.numel()
    w = pos.double()[..., None, None] * freqs
    c, s = w.cos() * magnitude, (-w if inverse else w).sin() * magnitude
    y = x.double().clone()
    a, b = (x[..., 0:R:2].double(), x[..., 1:R:2].double()) if interleaved else (x[..., :h].double(), x[..., h:R].double())
    u, v = a * c - b * s, a * s + b * c
    if interleaved:
        y[..., 0:R:2], y[..., 1:R:2] = u, v
    else:
        y[..., :h], y[..., h:R] = u, v
    return y


def _close(got, ref, x, magnitude=1.0):
    assert ((got.double() - ref).abs() <= UNIT * ref.abs() + 8 * UNIT * magnitude * 2 * float(x.abs().max())).all()


# ------------------------------------------------------------------------------------------------ forward mode
@pytest.mark.parametrize("interleaved", [True, False])
def test_rotary_carries_tangents(interleaved):
    from torsh_b200.ops.rotary import rotary
    q, k, dq, dk, pos, freqs = _setup(interleaved)
    for which in ("q", "k", "both"):
        with fwd.dual_level():
            a = fwd.make_dual(q, dq) if which != "k" else q
            b = fwd.make_dual(k, dk) if which != "q" else k
            outs = [fwd.unpack_dual(y) for y in rotary(a, b, pos, freqs, interleaved, 1.25)]
        for x, dx, y, on in ((q, dq, outs[0], which != "k"), (k, dk, outs[1], which != "q")):
            _close(y.primal, _turn64(x, pos, freqs, interleaved, 1.25), x, 1.25)
            assert (y.tangent is not None) or not on
            if on:
                _close(y.tangent, _turn64(dx, pos, freqs, interleaved, 1.25), dx, 1.25)
    assert fwd.unpack_dual(rotary(q, None, pos, freqs)[0]).tangent is None


def test_jacobians_of_rotary_are_its_matrix():
    """The framework's forward-mode Jacobian, whose columns are the turned unit vectors."""
    from torsh_b200.autograd import transforms
    from torsh_b200.ops.rotary import rotary, rotary_frequencies
    freqs, _ = rotary_frequencies(4, device=DEV)
    x, pos = torch.randn(2, 1, 6, device=DEV, generator=_gen(1)), torch.tensor([3, 900], device=DEV)
    eye = torch.eye(12, device=DEV).view(12, 2, 1, 6)
    want = torch.stack([_turn64(e, pos, freqs, True) for e in eye], -1).view(2, 1, 6, 2, 1, 6)
    _close(transforms.jacfwd(lambda a: rotary(a, None, pos, freqs)[0])(x), want, torch.ones(1))
    y, dy = transforms.jvp(lambda a: rotary(a, None, pos, freqs)[0], (x,), (torch.ones_like(x),))
    _close(dy, _turn64(torch.ones_like(x), pos, freqs, True), torch.ones(1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("T", [1, 20])
def test_cache_attention_carries_tangents(dtype, T):
    """The derivative in q, against that of the formula in 64 bits. The primal's roundings reach it: keys and values are exact in fp32, the
    query and its tangent are bf16 already, and only the output is rounded (2^-8), after sums in fp32 of at most 200 products."""
    from torsh_b200.ops.kv_cache import kv_cache_attention, kv_cache_read, kv_cache_write
    g = _gen(T)
    H, G, D, n = 2, 2, 64, 40
    eight = dtype != torch.bfloat16
    kp, vp = (torch.zeros(5, H, 16, D, dtype=torch.int8 if eight else dtype, device=DEV).view(dtype) for _ in range(2))
    ks, vs = (torch.zeros(5, H, 16, device=DEV) if eight else None for _ in range(2))
    table, start = torch.tensor([[4, 0, 2, 3]], dtype=torch.int32, device=DEV), torch.tensor([n], dtype=torch.int32, device=DEV)
    k, v = (torch.randn(1, n + T, H, D, device=DEV, generator=g).bfloat16() for _ in range(2))
    kv_cache_write(k, v, kp, vp, table, start * 0, None, ks, vs)
    q, dq = (torch.randn(1, T, H * G, D, device=DEV, generator=g).bfloat16() for _ in range(2))
    with fwd.dual_level():
        out = fwd.unpack_dual(kv_cache_attention(fwd.make_dual(q, dq), kp, vp, table, start, None, None, ks, vs))
    assert out.tangent is not None
    rk, rv = (x[0].double() for x in kv_cache_read(kp, vp, table, start + T, n + T, None, ks, vs, torch.float32))
    for t in range(T):
        for h in range(H * G):
            kk, vv = rk[:n + t + 1, h // G], rv[:n + t + 1, h // G]
            p = torch.softmax(kk @ q[0, t, h].double() / 8, 0)
            ds = kk @ dq[0, t, h].double() / 8
            dp = p * (ds - (p * ds).sum())
            for got, want, mass in ((out.primal, p @ vv, p @ vv.abs()), (out.tangent, dp @ vv, (p * (ds.abs() + (p * ds.abs()).sum())) @ vv.abs())):
                assert ((got[0, t, h].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -13 * mass).all()


def test_cache_writes_refuse_tangents():
    from torsh_b200.ops.kv_cache import kv_cache_write
    kp, vp = (torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    table, start = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    k = torch.ones(1, 3, 1, 64, dtype=torch.bfloat16, device=DEV)
    with fwd.dual_level():
        d = fwd.make_dual(k, k)
        for a, b in ((d, k), (k, d)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                kv_cache_write(a, b, kp, vp, table, start)
    assert not kp.any() and not vp.any()
    kv_cache_write(k, k, kp, vp, table, start)
    assert kp[0, 0, :3].eq(1).all() and not math.isnan(float(kp.sum()))


# ------------------------------------------------------------------------------------------------ learned frequencies
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("which", ["freqs", "all"])
def test_rotary_gives_frequencies_their_gradient(interleaved, which):
    """dL/df_i = sum over tokens and heads of p (dy_b y_a - dy_a y_b), against 64 bits and differences. A pair's term is two products of
    fp32 numbers, each off by a few units; their sum over tokens in fp32 or more: 64 units of the sum of magnitudes. Freqs are fp64 and so is the last sum."""
    from torsh_b200.ops.rotary import rotary
    q, k, dq, dk, pos, freqs = _setup(interleaved)
    pos = pos % 50
    f = freqs.clone().requires_grad_()
    a, b = (x.clone().requires_grad_(which == "all") for x in (q, k))
    outs = rotary(a, b, pos, f, interleaved)
    wrt = (f, a, b) if which == "all" else (f,)
    grads = torch.autograd.grad(outs, wrt, (dq, dk))
    want, size = torch.zeros_like(freqs), torch.zeros_like(freqs)
    h = freqs.numel()
    i = torch.arange(h, device=DEV)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + h)
    for x, dy in ((q, dq), (k, dk)):
        y = _turn64(x, pos, freqs, interleaved)
        p = pos.double()[..., None, None]
        terms = p * dy.double()[..., ib] * y[..., ia], -p * dy.double()[..., ia] * y[..., ib]
        want += sum(t.sum((0, 1, 2)) for t in terms)
        size += sum(t.abs().sum((0, 1, 2)) for t in terms)
    assert grads[0].dtype == torch.float64 and ((grads[0] - want).abs() <= 64 * UNIT * size).all()

    def loss(fr):
        return sum((d.double() * _turn64(x, pos, fr, interleaved)).sum() for x, d in ((q, dq), (k, dk)))
    e = torch.zeros_like(freqs)
    e[3] = 1e-6
    assert abs((loss(freqs + e) - loss(freqs - e)) / 2e-6 - want[3]) <= 1e-6 * size[3] + 1e-4   # the formula itself
    if which == "all":
        for g, d in zip(grads[1:], (dq, dk)):
            _close(g, _turn64(d, pos, freqs, interleaved, 1.0, True), d)


# ------------------------------------------------------------------------------------------------ batched gradients, tangents of gradients
@pytest.mark.parametrize("interleaved", [True, False])
def test_batched_gradients_of_rotary(interleaved):
    """The framework's reverse-mode Jacobian: one batched backward pass."""
    from torsh_b200.autograd import transforms
    from torsh_b200.ops.rotary import rotary, rotary_frequencies
    freqs, _ = rotary_frequencies(4, device=DEV)
    x, k, pos = torch.randn(2, 1, 6, device=DEV, generator=_gen(1)), torch.randn(2, 2, 6, device=DEV, generator=_gen(2)), torch.tensor([3, 900], device=DEV)
    eye = torch.eye(12, device=DEV).view(12, 2, 1, 6)
    want = torch.stack([_turn64(e, pos, freqs, interleaved) for e in eye], -1).view(2, 1, 6, 2, 1, 6)
    for other in (None, k):                                                 # alone, and as one of two
        _close(transforms.jacrev(lambda a: rotary(a, other, pos, freqs, interleaved)[0])(x), want, torch.ones(1))
        with torch.no_grad():
            _close(transforms.jacrev(lambda a: torch.enable_grad()(rotary)(a, other, pos, freqs, interleaved)[0])(x), want, torch.ones(1))
    # both outputs, several gradients at once, differentiated again in those gradients
    a, b = x.clone().requires_grad_(), k.clone().requires_grad_()
    outs = rotary(a, b, pos, freqs, interleaved, 1.25)
    da, db = (torch.randn(3, *y.shape, device=DEV, generator=_gen(4)).requires_grad_() for y in outs)
    ga, gb = torch.autograd.grad(outs, (a, b), (da, db), is_grads_batched=True, create_graph=True)
    for i in range(3):
        for g, d in ((ga, da), (gb, db)):
            _close(g[i].detach(), _turn64(d[i].detach(), pos, freqs, interleaved, 1.25, True), d.detach(), 1.25)
    w = torch.randn_like(ga)
    (gg,) = torch.autograd.grad((ga * w).sum(), da)
    for i in range(3):
        _close(gg[i], _turn64(w[i], pos, freqs, interleaved, 1.25), w, 1.25)


def test_gradients_that_carry_tangents():
    """Reverse mode first, forward mode through its backward pass."""
    from torsh_b200.ops.rotary import rotary
    q, k, dq, dk, pos, freqs = _setup(True)
    a, b = q.clone().requires_grad_(), k.clone().requires_grad_()
    outs = rotary(a, b, pos, freqs)
    t = torch.randn_like(dq)
    with fwd.dual_level():
        ga, gb = torch.autograd.grad(outs, (a, b), (fwd.make_dual(dq, t), dk))
        ga = fwd.unpack_dual(ga)
    _close(ga.primal, _turn64(dq, pos, freqs, True, 1.0, True), dq)
    _close(ga.tangent, _turn64(t, pos, freqs, True, 1.0, True), t)
    _close(gb, _turn64(dk, pos, freqs, True, 1.0, True), dk)
