"""What the device-side index checks say about a batch that has places without a sequence."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture
def checks():
    from torsh_b200 import _native as nv
    nv.check_status()
    nv.enable_kernel_checks(True)
    yield nv
    nv.enable_kernel_checks(False)
    try:
        nv.check_status()
    except nv.KernelCheckFailed:
        pass


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("T,G", [(1, 1), (5, 2), (40, 4)])
@pytest.mark.parametrize("max_len", [128, 4096])
def test_places_without_a_sequence_are_no_bad_index(checks, dtype, T, G, max_len):
    """Every call of a step (few and many rows, short and wide tables) over a place that was never used and one that was released; a sequence that
    outgrows its pages is reported as before."""
    from torsh_b200.ops.kv_cache import PagedKVCache, kv_cache_read
    c = PagedKVCache(1, 2, 64, batch=3, max_len=max_len, dtype=dtype, page=16, device=DEV)
    g = torch.Generator(DEV).manual_seed(T)
    rows = lambda h: torch.randn(3, T, h, 64, device=DEV, generator=g).bfloat16()   # noqa: E731
    c.reserve([T, 0, T])
    c.write(0, rows(2), rows(2))
    c.advance(T)
    c.release(2)
    for _ in range(2):
        c.reserve([T, 0, 0])
        c.write(0, rows(2), rows(2))
        assert not c.attend(0, rows(2 * G))[1:].any()
        c.advance(torch.full((3,), T, device=DEV), most=T)
        assert not c.read(0)[0][1:].any()
    kv_cache_read(*c.layers[0], c.page_table, torch.full((3,), T, dtype=torch.int32, device=DEV), T, None, *c.scales[0])
    torch.cuda.synchronize()
    checks.check_status()
    for call in (lambda: c.write(0, rows(2), rows(2)), lambda: c.attend(0, rows(2 * G)))[:2 if len(c._owned[0]) * 16 < max_len else 1]:   # attention ends with the table
        while int(c.lengths[0]) + T <= len(c._owned[0]) * 16:               # up to the end of what the sequence has
            c.lengths[0] += T
        call()
        torch.cuda.synchronize()
        with pytest.raises(checks.KernelCheckFailed):
            checks.check_status()


def test_other_pages_of_an_empty_place_are_reported(checks):
    """Only -1 means no page, and only where the first page says so."""
    from torsh_b200.ops.kv_cache import kv_cache_write
    kp, vp = (torch.zeros(4, 1, 16, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    k = torch.ones(1, 3, 1, 64, dtype=torch.bfloat16, device=DEV)
    for table, start, bad in (([-1, -1], 0, False), ([-1, -1], 15, False), ([-2, -1], 0, True), ([-1, 9], 16, True), ([2, -1], 16, True), ([2, -1], 0, False), ([-1, -1], 31, True)):
        kv_cache_write(k, k, kp, vp, torch.tensor([table], dtype=torch.int32, device=DEV), torch.tensor([start], dtype=torch.int32, device=DEV))
        torch.cuda.synchronize()
        if bad:
            with pytest.raises(checks.KernelCheckFailed):
                checks.check_status()
        else:
            checks.check_status()
