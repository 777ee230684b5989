"""Decoding operators without a GPU: their formulas against plain loops, and the calls that they refuse."""
import math

import pytest
import torch

from torsh_b200.ops.kv_cache import PagedKVCache, kv_cache_attention, kv_cache_read, kv_cache_write, quantize_rows, tree_mask_of
from torsh_b200.ops.rotary import rotary, rotary_frequencies
from torsh_b200.ops.speculative import verify_draft

E4M3 = torch.float8_e4m3fn


# ------------------------------------------------------------------------------------------------ rotary
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("D,R", [(8, 8), (10, 4), (6, 0)])
def test_rotary_formula_and_gradient(interleaved, D, R):
    torch.manual_seed(0)
    q, k = torch.randn(2, 3, 2, D, dtype=torch.float64, requires_grad=True), torch.randn(2, 3, 1, D, dtype=torch.float64, requires_grad=True)
    pos = torch.tensor([[0, 7, 100000], [3, 2, 1]])
    freqs, m = rotary_frequencies(R, scaling="yarn" if R else "none", factor=4.0)
    yq, yk = rotary(q, k, pos, freqs, interleaved, m)
    for x, y in ((q, yq), (k, yk)):
        for b in range(2):
            for t in range(3):
                want = x[b, t].detach().clone()
                for i in range(R // 2):
                    a, c = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
                    w = float(pos[b, t]) * float(freqs[i])
                    want[:, a] = m * (x[b, t, :, a] * math.cos(w) - x[b, t, :, c] * math.sin(w)).detach()
                    want[:, c] = m * (x[b, t, :, a] * math.sin(w) + x[b, t, :, c] * math.cos(w)).detach()
                torch.testing.assert_close(y[b, t].detach(), want, rtol=1e-12, atol=1e-12)
    assert torch.autograd.gradcheck(lambda a, b: rotary(a, b, pos, freqs, interleaved, m), (q, k))


def test_rotary_matches_the_fixed_form():
    from torsh_b200.ops.elementwise import rope
    x = torch.randn(2, 5, 3, 16)
    torch.testing.assert_close(rotary(x, None, torch.arange(5), rotary_frequencies(16)[0])[0], rope(x), rtol=1e-5, atol=1e-5)


def test_rotary_frequencies():
    plain, one = rotary_frequencies(64)
    assert one == 1.0 and plain.dtype == torch.float64 and plain[0] == 1.0
    assert torch.equal(rotary_frequencies(64, scaling="linear", factor=4.0)[0], plain / 4)
    ntk, _ = rotary_frequencies(64, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], plain[-1] / 4, rel_tol=1e-12)
    for name in ("yarn", "wavelength"):
        f, m = rotary_frequencies(64, scaling=name, factor=4.0, trained_len=4096)
        assert f[0] == plain[0] and math.isclose(f[-1], plain[-1] / 4, rel_tol=1e-12)
        assert ((f <= plain) & (f >= plain / 4 * (1 - 1e-12))).all() and (f.diff() < 0).all()
        assert math.isclose(m, 0.1 * math.log(4.0) + 1 if name == "yarn" else 1.0)
    turns = 4096 * plain / (2 * math.pi)
    f, _ = rotary_frequencies(64, scaling="wavelength", factor=8.0, low=1.0, high=4.0)
    assert torch.equal(f[turns >= 4], plain[turns >= 4]) and torch.allclose(f[turns <= 1], plain[turns <= 1] / 8, rtol=1e-12)
    for bad in (dict(dim=3), dict(dim=4, scaling="other"), dict(dim=4, factor=0.5), dict(dim=4, base=1.0), dict(dim=4, scaling="wavelength", low=4.0, high=2.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


@pytest.mark.parametrize("bad,exc", [
    (dict(k=torch.zeros(2, 4, 1, 8)), ValueError), (dict(k=torch.zeros(2, 3, 1, 6)), ValueError), (dict(k=torch.zeros(2, 3, 1, 8).half()), ValueError),
    (dict(positions=torch.zeros(2, 3)), TypeError), (dict(positions=torch.zeros(3, 3, dtype=torch.long)), ValueError),
    (dict(positions=torch.zeros(2, dtype=torch.long)), ValueError), (dict(freqs=torch.ones(5, dtype=torch.float64)), ValueError)])
def test_rotary_refusals(bad, exc):
    kw = dict(q=torch.zeros(2, 3, 2, 8), k=None, positions=torch.zeros(2, 3, dtype=torch.long), freqs=torch.ones(4, dtype=torch.float64))
    rotary(**kw)
    with pytest.raises(exc):
        rotary(**{**kw, **bad})


# ------------------------------------------------------------------------------------------------ cache
def test_quantised_rows():
    torch.manual_seed(1)
    x = torch.randn(50, 64).bfloat16()
    x[0], x[1, 3], x[2, 5] = 0, math.nan, math.inf
    x[3] = torch.arange(64) - 32                       # -32 is the largest: 16 / (32 / 127) = 63.5 is a tie
    codes, s = quantize_rows(x, torch.int8)
    assert s[0] == 0 and not codes[0].any() and s[1].isnan() and s[2].isnan()
    r = x[3:].double() / s[3:, None].double()
    assert torch.equal(codes[3:].double(), r.round()) and int(codes[3].min()) == -127
    codes, s = quantize_rows(x, E4M3)
    big = x[3:].float().abs().amax(-1)
    assert ((big / s[3:] <= 448) & (big / s[3:] > 224)).all() and (torch.frexp(s[3:])[0] == 0.5).all()
    back = codes[3:].double() * s[3:, None].double()
    step = torch.maximum(x[3:].double().abs() * 2.0 ** -4, s[3:, None].double() * 2.0 ** -10)   # half of a step of e4m3, half of its smallest
    assert ((back - x[3:].double()).abs() <= step).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8, E4M3, torch.float32])
def test_cache_write_read_and_attend_on_the_cpu(dtype):
    torch.manual_seed(2)
    B, T, H, G, D, page = 2, 5, 2, 3, 8, 16
    kp, vp = (torch.zeros(6, H, page, D).to(dtype) for _ in range(2))
    ks, vs = (torch.zeros(6, H, page), torch.zeros(6, H, page)) if dtype in (torch.int8, E4M3) else (None, None)
    table = torch.tensor([[4, 1], [0, 3]], dtype=torch.int32)
    lens = [20, 9]
    k, v = torch.randn(B, 30, H, D), torch.randn(B, 30, H, D)
    kv_cache_write(k, v, kp, vp, table, torch.zeros(B, dtype=torch.int32), torch.tensor(lens), ks, vs)
    rk, rv = kv_cache_read(kp, vp, table, torch.tensor(lens), 22, None, ks, vs, torch.float32)
    for got, src in ((rk, k), (rv, v)):
        for b in range(B):
            codes, s = quantize_rows(src[b, :lens[b]], dtype)
            assert torch.equal(got[b, :lens[b]], codes.float() * (1 if s is None else s[..., None])) and not got[b, lens[b]:].any()
    q = torch.randn(B, T, H * G, D)
    start, counts = torch.tensor([15, 6]), torch.tensor([5, 3])
    mask = tree_mask_of(torch.tensor([-1, 0, 0, 1, 2]))
    got = kv_cache_attention(q, kp, vp, table, start, mask, counts, ks, vs)
    for b in range(B):
        for t in range(T):
            for h in range(H * G):
                if t >= counts[b]:
                    assert not got[b, t, h].any()
                    continue
                keys = list(range(int(start[b]))) + [int(start[b]) + j for j in range(int(counts[b])) if mask[t, j]]
                kk, vv = rk[b, keys, h // G].double(), rv[b, keys, h // G].double()
                w = torch.softmax(kk @ q[b, t, h].double() / math.sqrt(D), 0)
                torch.testing.assert_close(got[b, t, h].double(), w @ vv, rtol=1e-5, atol=1e-5)


def test_cpu_attention_keeps_what_is_not_seen_apart():
    kp, vp = torch.randn(2, 1, 16, 8), torch.randn(2, 1, 16, 8)
    vp[0, 0, 4, 2], kp[0, 0, 4, 1] = math.inf, math.nan
    q = torch.randn(1, 3, 2, 8)
    table, start = torch.tensor([[0, 1]]), torch.tensor([3])
    mask = torch.eye(3, dtype=torch.bool)
    got = kv_cache_attention(q, kp, vp, table, start, mask)
    assert got[0, 1].isnan().any() and torch.isfinite(got[0, [0, 2]]).all()
    none = kv_cache_attention(q, kp, vp, table, torch.tensor([0]), torch.zeros(3, 3, dtype=torch.bool))
    assert not none.any()


@pytest.mark.parametrize("B,T", [(0, 3), (2, 0)])
def test_attention_over_nothing(B, T):
    kp, vp = torch.randn(2, 1, 16, 8), torch.randn(2, 1, 16, 8)
    table, start = torch.zeros(B, 1, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
    assert kv_cache_attention(torch.randn(B, T, 2, 8), kp, vp, table, start).shape == (B, T, 2, 8)
    kv_cache_write(torch.randn(B, T, 1, 8), torch.randn(B, T, 1, 8), kp, vp, table, start)
    assert kv_cache_read(kp, vp, table, start, 4)[0].shape == (B, 4, 1, 8)


def test_an_empty_pool_or_table_holds_nothing():
    k = torch.randn(2, 3, 1, 8)
    for pages, width in ((0, 2), (2, 0)):
        kp, vp = torch.zeros(pages, 1, 16, 8), torch.zeros(pages, 1, 16, 8)
        table, start = torch.zeros(2, width, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
        kv_cache_write(k, k, kp, vp, table, start)
        assert not kp.any() and not kv_cache_read(kp, vp, table, start + 3, 3)[0].any()
        assert not kv_cache_attention(k, kp, vp, table, start).any()


def test_negative_starts_and_integers_beyond_32_bits():
    kp, vp = torch.zeros(2, 1, 16, 8), torch.zeros(2, 1, 16, 8)
    table = torch.tensor([[0], [1]])
    k = torch.ones(2, 4, 1, 8)
    kv_cache_write(k, k, kp, vp, table, torch.tensor([-2, -1]))             # these sequences are left out
    kv_cache_write(k, k, kp, vp, table, torch.tensor([1 << 32, -(1 << 32)]))
    kv_cache_write(k, k, kp, vp, table + (1 << 32), torch.tensor([0, 0]))   # no pages of the pool
    assert not kp.any()
    kv_cache_write(k, k, kp, vp, table, torch.tensor([0, 2]), torch.tensor([1 << 32, 1]))
    assert kp[0, 0, :4].eq(1).all() and kp[1, 0, 2].eq(1).all() and kp.sum() == 5 * 8
    rk, _ = kv_cache_read(kp, vp, table, torch.tensor([1 << 33, 3]), 4)
    assert rk[0].eq(1).all() and rk[1, 2].eq(1).all() and rk.float().sum() == 5 * 8


def test_tree_masks():
    parents = torch.tensor([-1, 0, 1, 1, 0, 4, -1])
    m = tree_mask_of(parents)
    for i in range(7):
        up, j = {i}, i
        while int(parents[j]) >= 0:
            j = int(parents[j])
            up.add(j)
        assert set(m[i].nonzero().flatten().tolist()) == up
    deep = torch.arange(-1, 99)
    assert torch.equal(tree_mask_of(deep), torch.ones(100, 100, dtype=torch.bool).tril())
    assert tree_mask_of(parents.expand(3, 7)).shape == (3, 7, 7)
    with pytest.raises(ValueError):
        tree_mask_of(torch.tensor([-1, 1]))
    with pytest.raises(TypeError):
        tree_mask_of(torch.tensor([-1.0, 0.0]))


def _attention_args():
    return dict(q=torch.zeros(2, 3, 4, 64), k_pages=torch.zeros(5, 2, 16, 64, dtype=torch.int8), v_pages=torch.zeros(5, 2, 16, 64, dtype=torch.int8),
                page_table=torch.zeros(2, 2, dtype=torch.int32), start=torch.zeros(2, dtype=torch.int32), k_scales=torch.ones(5, 2, 16), v_scales=torch.ones(5, 2, 16))


@pytest.mark.parametrize("bad,exc", [
    (dict(q=torch.zeros(2, 3, 3, 64)), ValueError), (dict(q=torch.zeros(2, 3, 4, 32)), ValueError), (dict(q=torch.zeros(3, 4, 64)), ValueError),
    (dict(v_pages=torch.zeros(5, 2, 16, 64)), ValueError), (dict(v_pages=torch.zeros(4, 2, 16, 64, dtype=torch.int8)), ValueError),
    (dict(k_scales=None), ValueError), (dict(v_scales=torch.ones(5, 2, 8)), ValueError), (dict(k_scales=torch.ones(5, 2, 16).double()), ValueError),
    (dict(page_table=torch.zeros(3, 2, dtype=torch.int32)), ValueError), (dict(page_table=torch.zeros(2, 2)), ValueError),
    (dict(start=torch.zeros(3, dtype=torch.int32)), ValueError), (dict(start=torch.zeros(2)), ValueError), (dict(counts=torch.zeros(1, dtype=torch.int32)), ValueError),
    (dict(tree_mask=torch.ones(3, 3)), ValueError), (dict(tree_mask=torch.ones(2, 2, dtype=torch.bool)), ValueError), (dict(max_len=-1), ValueError), (dict(scale=-1.0), ValueError), (dict(scale=math.nan), ValueError),
    (dict(q=torch.zeros(2, 3, 4, 64, requires_grad=True)), RuntimeError),
    (dict(k_pages=torch.zeros(5, 2, 16, 64).to(torch.uint8), v_pages=torch.zeros(5, 2, 16, 64).to(torch.uint8)), TypeError),
    (dict(k_pages=torch.zeros(5, 2, 16, 64).bfloat16(), v_pages=torch.zeros(5, 2, 16, 64).bfloat16()), ValueError),
    (dict(k_pages=torch.zeros(5, 16, 2, 64, dtype=torch.int8).transpose(1, 2)), ValueError)])
def test_attention_refusals(bad, exc):
    kv_cache_attention(**_attention_args())
    with pytest.raises(exc):
        kv_cache_attention(**{**_attention_args(), **bad})


@pytest.mark.parametrize("bad,exc", [
    (dict(v=torch.zeros(2, 3, 2, 32)), ValueError), (dict(k=torch.zeros(2, 3, 1, 64), v=torch.zeros(2, 3, 1, 64)), ValueError),
    (dict(k=torch.zeros(2, 3, 2, 64).int(), v=torch.zeros(2, 3, 2, 64).int()), ValueError), (dict(start=torch.zeros(1, dtype=torch.int32)), ValueError),
    (dict(k=torch.zeros(2, 3, 2, 64, requires_grad=True)), RuntimeError), (dict(k_scales=None), ValueError), (dict(counts=torch.ones(2)), ValueError)])
def test_write_refusals(bad, exc):
    kw = {**_attention_args(), "k": torch.zeros(2, 3, 2, 64), "v": torch.zeros(2, 3, 2, 64)}
    del kw["q"]
    kv_cache_write(**kw)
    with pytest.raises(exc):
        kv_cache_write(**{**kw, **bad})


@pytest.mark.parametrize("bad,exc", [(dict(max_len=-1), ValueError), (dict(dtype=torch.int32), TypeError), (dict(dtype=E4M3), TypeError), (dict(lengths=torch.ones(3, dtype=torch.int32)), ValueError),
                                     (dict(begin=torch.ones(2)), ValueError), (dict(page_table=torch.zeros(2, dtype=torch.int32)), ValueError)])
def test_read_refusals(bad, exc):
    kw = {**_attention_args(), "lengths": torch.ones(2, dtype=torch.int32), "max_len": 4}
    del kw["q"], kw["start"]
    kv_cache_read(**kw)
    with pytest.raises(exc):
        kv_cache_read(**{**kw, **bad})


def test_paged_cache_keeps_its_pages():
    c = PagedKVCache(2, 1, 8, batch=2, max_len=64, dtype=torch.int8, page=16, num_pages=5, device="cpu")
    c.reserve([20, 3])
    assert c.page_table[0, :2].tolist() == [0, 1] and c.page_table[1, 0] == 2
    c.advance([20, 3])
    c.reserve(12)
    assert len(c._free) == 2
    with pytest.raises(ValueError):
        c.reserve([45, 0])
    c.reserve([44, 0])
    with pytest.raises(RuntimeError):
        c.reserve([44, 40])
    c.release(0)
    assert len(c._free) == 4 and c.lengths.tolist() == [0, 3] and c.host_lengths == [0, 3]
    c.advance(torch.tensor([0, 2]), most=4)
    assert c.lengths.tolist() == [0, 5] and c.host_lengths == [4, 7]
    for bad in (dict(page=8), dict(page=0), dict(dtype=torch.int32)):
        with pytest.raises((ValueError, TypeError)):
            PagedKVCache(**{**dict(num_layers=1, num_heads=1, head_dim=8, batch=1, max_len=16, page=16, device="cpu"), **bad})


def _fed(c, tokens, seed):
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(c.batch, tokens, 1, 8, generator=g) for _ in range(2))
    c.write(0, k, v)
    return k, v


def test_a_place_without_a_sequence_reaches_no_other_sequence():
    """Batched steps go on over places that were never used, and places whose sequence was released: their rows belong nowhere."""
    c = PagedKVCache(1, 1, 8, batch=3, max_len=64, dtype=torch.float32, page=16, num_pages=4, device="cpu")
    c.reserve([16, 16, 0])
    _fed(c, 16, 0)
    c.advance([16, 16, 0])
    c.release(0)
    c.reserve([0, 32, 0])                                   # gets the released page
    k, v = _fed(c, 32, 1)
    c.advance([0, 32, 0])
    for got, want in zip(c.read(0, torch.float32), (k, v)):
        assert torch.equal(got[1, 16:48], want[1]) and not got[[0, 2]].any()
    q = torch.randn(3, 1, 2, 8)
    assert not c.attend(0, q)[[0, 2]].any()


@pytest.mark.parametrize("owner", [0, 1, 2])
def test_keeping_a_path_leaves_other_places_alone(owner):
    """The sequence that owns page 0 keeps its path whichever place it has, beside places that have no page."""
    c = PagedKVCache(1, 1, 8, batch=3, max_len=32, dtype=torch.float32, page=16, num_pages=2, device="cpu")
    c.reserve([20 if b == owner else 0 for b in range(3)])
    assert c.page_table[owner, 0] == 0
    k, v = _fed(c, 5, 2)
    path = torch.tensor([[0, 2, 4, -1, -1]] * 3)
    c.keep(path, torch.tensor([2, 2, 2]))
    c.advance([3 if b == owner else 0 for b in range(3)])
    for got, want in zip(c.read(0, torch.float32), (k, v)):
        assert torch.equal(got[owner, :3], want[owner, [0, 2, 4]])
    assert torch.equal(c.layers[0][0][0, 0, 3:5], k[owner, 3:5, 0])            # what is not on the path stays
    none = PagedKVCache(1, 1, 8, batch=2, max_len=32, dtype=torch.float32, page=16, device="cpu")
    none.keep(path[:2], torch.tensor([2, 2]))
    assert not none.layers[0][0].any()


# ------------------------------------------------------------------------------------------------ verification
def test_verify_by_hand():
    p = torch.tensor([[[0.5, 0.25, 0.25, 0.0], [0.0, 0.5, 0.5, 0.0], [0.25, 0.25, 0.25, 0.25]]])
    q = torch.tensor([[[0.25, 0.75, 0.0, 0.0], [0.0, 1.0, 0.0, 0.0]]])
    tok = torch.tensor([[0, 0, 1]])
    call = lambda u, **kw: [x.tolist() for x in verify_draft(p, tok, torch.tensor([u]), **kw)]   # noqa: E731
    assert call([0.99, 0.49, 0.6], draft_probs=q) == [[2], [[0, 1, 2]], [2]]             # both accepted: the bonus token from p_2
    assert call([0.99, 0.5, 0.0], draft_probs=q) == [[1], [[0, 1, -1]], [2]]             # 0.5 * 1 < 0.5 fails: max(p - q, 0) is all at 2
    # fixed chain: token 0 needs u < 0.5, token 1 after it u < 0.5
    assert call([0.4, 0.49, 0.0]) == [[2], [[0, 1, 2]], [0]]
    assert call([0.5, 0.0, 0.6]) == [[0], [[0, -1, -1]], [2]]                            # the rest of p_0 without token 0: 1 and 2 alike
    # a tree: both nodes are children of the root, tokens 0 and 1: [0, 0.5) and [0.5, 0.75)
    par = torch.tensor([-1, 0, 0])
    assert call([0.6, 0.0, 0.6], parents=par) == [[1], [[0, 2, -1]], [2]]
    assert call([0.8, 0.0, 0.6], parents=par) == [[0], [[0, -1, -1]], [2]]
    assert call([0.6, 0.0, 0.6], parents=par, counts=torch.tensor([2])) == [[0], [[0, -1, -1]], [2]]


@pytest.mark.parametrize("bad,exc", [
    (dict(probs=torch.zeros(2, 3, 8).double()), ValueError), (dict(probs=torch.zeros(3, 8)), ValueError), (dict(tokens=torch.zeros(2, 2, dtype=torch.long)), ValueError),
    (dict(tokens=torch.zeros(2, 3)), TypeError), (dict(uniforms=torch.zeros(2, 3, dtype=torch.long)), TypeError), (dict(uniforms=torch.zeros(2, 2)), ValueError),
    (dict(draft_probs=torch.zeros(2, 3, 8)), ValueError), (dict(draft_probs=torch.zeros(2, 2, 8).bfloat16()), ValueError),
    (dict(parents=torch.zeros(2, dtype=torch.long)), ValueError), (dict(parents=torch.zeros(3)), ValueError),
    (dict(parents=torch.tensor([-1, 0, 0]), draft_probs=torch.zeros(2, 2, 8)), ValueError), (dict(counts=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(probs=torch.zeros(2, 1025, 2), tokens=torch.zeros(2, 1025, dtype=torch.long), uniforms=torch.zeros(2, 1025)), ValueError)])
def test_verify_refusals(bad, exc):
    kw = dict(probs=torch.ones(2, 3, 8) / 8, tokens=torch.zeros(2, 3, dtype=torch.long), uniforms=torch.zeros(2, 3))
    verify_draft(**kw)
    with pytest.raises(exc):
        verify_draft(**{**kw, **bad})


# ------------------------------------------------------------------------------------------------ together
def _llama(layers=2, seed=0, hidden=32, heads=2):
    from torsh_b200.models.llama import LlamaConfig, LlamaModel
    torch.manual_seed(seed)
    m = LlamaModel(LlamaConfig(vocab_size=50, hidden_size=hidden, intermediate_size=64, num_layers=layers, num_heads=heads, max_seq_len=256, initializer_range=0.3))
    return m.eval()


def _greedy(m, ids, n):
    with torch.no_grad():
        for _ in range(n):
            ids = torch.cat([ids, m(ids)[:, -1].argmax(-1, keepdim=True)], 1)
    return ids


@pytest.mark.parametrize("S", [1, 5])
def test_generate_from_a_cache_is_the_whole_context_run_again(S):
    m, small = _llama(), _llama(1, 7)
    ids = torch.randint(0, 50, (3, S))
    want = _greedy(m, ids, 20)
    assert torch.equal(m.generate(ids, 20), want)
    for draft, k in ((small, 1), (small, 3), (m, 4)):      # the model itself as the draft: everything is accepted
        assert torch.equal(m.generate(ids, 20, draft=draft, drafted=k), want)
    assert m.generate(ids, 0) is ids
    assert m.generate(ids, 7, cache_dtype=torch.int8).shape == (3, S + 7)


def test_generate_samples_and_refuses():
    m, small = _llama(), _llama(1, 7)
    ids = torch.randint(0, 50, (2, 4))
    g = lambda: torch.Generator().manual_seed(3)   # noqa: E731
    assert torch.equal(m.generate(ids, 9, 1.0, generator=g()), m.generate(ids, 9, 1.0, generator=g()))
    assert m.generate(ids, 9, 1.0, draft=small, generator=g()).shape == (2, 13)
    for bad in (dict(temperature=-1.0), dict(draft=small, drafted=0)):
        with pytest.raises(ValueError):
            m.generate(ids, 2, **bad)


def test_generate_for_nobody_and_nothing():
    m = _llama()
    for ids, n in ((torch.zeros(0, 4, dtype=torch.int64), 3), (torch.zeros(2, 0, dtype=torch.int64), 3), (torch.ones(2, 4, dtype=torch.int64), 0)):
        assert torch.equal(m.generate(ids, n), ids)


def test_decode_of_a_tree_gives_each_path_its_own_states():
    m = _llama()
    ids = torch.randint(0, 50, (2, 6))
    c = m.make_cache(2, 40, page=16)
    c.reserve(6)
    m.decode(ids, c)
    c.advance(6)
    parents = torch.tensor([-1, 0, 0, 1, 2])
    tokens = torch.randint(0, 50, (2, 5))
    mask = tree_mask_of(parents)
    c.reserve(5)
    h = m.decode(tokens, c, mask).view(2, 5, -1)
    for i in range(5):
        path = mask[i].nonzero().flatten()
        flat = m.make_cache(2, 40, page=16)
        flat.reserve(6 + len(path))
        want = m.decode(torch.cat([ids, tokens[:, path]], 1), flat).view(2, 6 + len(path), -1)[:, -1]
        torch.testing.assert_close(h[:, i], want, rtol=1e-4, atol=1e-4)
