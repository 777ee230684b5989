"""A paged cache whose steps are captured once and replayed, and that is given more room in between."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _make():
    from torsh_b200.ops.kv_cache import PagedKVCache
    return PagedKVCache(1, 2, 64, batch=2, max_len=320, dtype=torch.bfloat16, page=16, num_pages=40, device=DEV)


def test_room_is_counted_from_what_replays_have_kept():
    """reserve() between replays: the host has seen one step, the device many."""
    g = torch.Generator(DEV).manual_seed(0)
    steps = [tuple(torch.randn(2, 3, 2, 64, device=DEV, generator=g).bfloat16() for _ in range(3)) + (torch.randint(1, 4, (2,), device=DEV, generator=g),) for _ in range(60)]

    def step(c, x):
        q, k, v, n = x
        c.write(0, k, v)
        out = c.attend(0, q)
        c.advance(n, most=3)
        return out

    eager, c = _make(), _make()
    held = [x.clone() for x in steps[0]]
    c.reserve(30)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(c, held)
    assert c.lengths.tolist() == [0, 0]                                     # captured, not run
    for i, x in enumerate(steps):
        if i % 10 == 0:
            c.reserve(30)                                                   # ten steps of at most three
        eager.reserve(3)
        want = step(eager, x)
        for a, b in zip(held, x):
            a.copy_(b)
        graph.replay()
        assert torch.equal(out, want), i
    assert torch.equal(c.lengths, eager.lengths) and int(c.lengths.min()) > 60
    for a, b in zip(c.read(0), eager.read(0)):
        n = int(c.lengths.max())
        assert a.shape[1] == n and torch.equal(a, b[:, :n]) and not b[:, n:].any()
    c.truncate([50, int(c.lengths[1])])
    assert int(c.lengths[0]) == 50
    with pytest.raises(ValueError):
        c.truncate([51, 0])
