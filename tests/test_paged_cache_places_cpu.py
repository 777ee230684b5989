"""A paged cache whose batch has places without a sequence, and lengths that the host knows only as upper bounds."""
import pytest
import torch

from torsh_b200.ops.kv_cache import PagedKVCache


def _cache(batch=2, max_len=64, num_pages=None, **kw):
    return PagedKVCache(1, 1, 8, batch=batch, max_len=max_len, dtype=torch.float32, page=16, num_pages=num_pages, device="cpu", **kw)


def _rows(batch, T, seed):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randn(batch, T, h, 8, generator=g) for h in (2, 1, 1))


@pytest.mark.parametrize("form", ["tensor", "bounded", "int", "list"])
@pytest.mark.parametrize("used", [False, True])
def test_a_place_without_a_sequence_stays_empty(form, used):
    """Steps of a batch advance every place; those without a sequence (never used, or released) neither grow, nor get pages, nor stop the
    others, and the sequence that comes to such a place begins at position 0."""
    c = _cache(num_pages=5)
    if used:
        c.reserve([4, 20])
        c.write(0, *_rows(2, 20, 9)[1:])
        c.advance([0, 20])
        c.release(1)
    free, steps = len(c._free), 60
    for i in range(steps):
        c.reserve([1, 0])
        q, k, v = _rows(2, 1, i)
        c.write(0, k, v)
        assert not c.attend(0, q)[1].any()
        one = torch.ones(2, dtype=torch.int64)
        if form == "bounded":
            c.advance(one, most=1)
        else:
            c.advance({"tensor": one, "int": 1, "list": [1, 1]}[form])
    assert c.lengths.tolist() == [steps, 0] and not (c.page_table[1] >= 0).any()
    assert len(c._free) + 4 == 5 >= free and c.read(0, torch.float32)[0].shape[1] == steps
    # a sequence comes
    fresh = _cache(batch=1)
    c.reserve([0, 3])
    fresh.reserve(3)
    q, k, v = _rows(2, 3, 77)
    c.write(0, k, v)
    fresh.write(0, k[1:], v[1:])
    # the batch is as wide as its longest sequence: sums of 8 and 3 products (and zeros) below 8, perhaps in another order, 16 units of 2^-24 * 8
    torch.testing.assert_close(c.attend(0, q)[1:], fresh.attend(0, q[1:]), rtol=0, atol=2.0 ** -17)
    assert torch.equal(c.attend(0, q)[1, 0], v[1, 0].expand(2, 8))          # the first token sees itself alone
    c.advance(torch.tensor([0, 3]))
    assert c.lengths.tolist() == [steps, 3] and c.host_lengths == [steps, 3]
    assert torch.equal(c.read(0, torch.float32)[0][1, :3], k[1])


def test_truncating_never_lengthens():
    """After a bounded advance the host has upper bounds: a length between what a sequence has and that bound leaves it as it is."""
    c = _cache()
    c.reserve([20, 20])
    q, k, v = _rows(2, 5, 1)
    c.write(0, k, v)
    c.advance(torch.tensor([1, 4]), most=5)
    c.truncate([5, 3])
    assert c.lengths.tolist() == [1, 3] and all(n >= m for n, m in zip(c.host_lengths, [1, 3]))
    # the next token sees what was accepted, and itself
    q, k2, v2 = _rows(2, 1, 2)
    c.write(0, k2, v2)
    got = c.attend(0, q)
    for b, n in enumerate((1, 3)):
        kk, vv = torch.cat([k[b, :n, 0], k2[b, :, 0]]), torch.cat([v[b, :n, 0], v2[b, :, 0]])
        torch.testing.assert_close(got[b, 0], torch.softmax(q[b, 0] @ kk.T / 8 ** 0.5, -1) @ vv)
    for bad in ([6, 0], [-1, 0], [1], [1, 1, 1]):
        with pytest.raises(ValueError):
            c.truncate(bad)
    c.truncate([0, 2])
    assert c.lengths.tolist() == [0, 2]


def test_upper_bounds_refuse_nothing_that_there_is_room_for():
    """Steps that keep one token of five: the bounds pass max_len, and what the pool has, long before the sequences do."""
    c = _cache(batch=1, num_pages=4)
    for i in range(59):
        c.reserve(5)
        q, k, v = _rows(1, 5, i)
        c.write(0, k, v)
        c.advance(torch.tensor([1]), most=5)
    assert c.lengths.tolist() == [59] and 59 <= c.host_lengths[0] <= 64
    for i in range(59):
        assert torch.equal(c.read(0, torch.float32)[0][0, i], _rows(1, 5, i)[1][0, 0])
    c.reserve(5)
    for n in (6, 1000):
        with pytest.raises(ValueError):
            c.reserve(n)
    two = _cache(num_pages=4)
    two.reserve(30)
    two.advance(torch.tensor([1, 1]), most=30)
    two.reserve(30)
    with pytest.raises(RuntimeError):
        two.reserve([40, 0])
    two.reserve([0, 31])
    assert len(two._free) == 0 and two.lengths.tolist() == [1, 1]


@pytest.mark.parametrize("bad", [[1], [1, 1, 1], []])
def test_tokens_of_other_batches_are_refused(bad):
    """A list that is too short reserved for the places that it had, and said nothing of the others."""
    c = _cache()
    c.reserve([5, 5])
    for call in (c.reserve, c.advance):
        with pytest.raises(ValueError):
            call(bad)
    assert c.lengths.tolist() == [0, 0] == c.host_lengths and len(c._free) == 6


def test_a_place_whose_table_names_others_pages_has_a_length():
    """A caller's own table (here a prefix that two places share) counts as a sequence."""
    c = _cache()
    c.reserve([20, 0])
    c.page_table[1] = c.page_table[0]
    q, k, v = _rows(2, 20, 3)
    c.write(0, k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1))
    for tokens in (5, [5, 5], torch.tensor([5, 5])):
        c.advance(tokens)
    c.advance(torch.tensor([5, 5]), most=5)
    assert c.lengths.tolist() == [20, 20] == c.host_lengths
    rk, rv = c.read(0, torch.float32)
    assert torch.equal(rk, k[:1].expand(2, -1, -1, -1)) and torch.equal(rv, v[:1].expand(2, -1, -1, -1))
    c.truncate([20, 7])
    assert c.lengths.tolist() == [20, 7]
