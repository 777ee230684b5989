"""Values that are infinite or no numbers, under finite keys: the rows that see them get exactly them, the others nothing of them."""
import math

import pytest
import torch

from test_decoding_gpu import BF16, DEV, E4M3, _attend64, _attention_close, _case, _gen

pytestmark = pytest.mark.gpu

# (B, T, query heads, heads, D, page, contexts), columns that the table has beyond the sequences. Few rows, whole and cut units; many rows in
# short tables (few rows' kernel) and wide ones (tcgen05), new tokens in one key tile and in several, cut units, several row tiles
SHAPES = [((2, 6, 2, 1, 128, 16, [37, 12]), 0), ((2, 6, 2, 1, 128, 16, [30037, 20012]), 0), ((1, 40, 2, 1, 64, 16, [21]), 0), ((1, 40, 2, 1, 64, 16, [21]), 5000),
          ((3, 150, 2, 1, 64, 16, [100, 333, 0]), 5000), ((1, 30, 4, 2, 128, 16, [30037]), 0), ((2, 200, 1, 1, 128, 48, [7, 60]), 5000), ((2, 130, 3, 1, 64, 16, [8000, 127]), 0)]


@pytest.mark.parametrize("dtype,what", [(BF16, "values"), (E4M3, "values"), (E4M3, "scales"), (torch.int8, "scales")])
@pytest.mark.parametrize("where", ["new", "context"])
@pytest.mark.parametrize("shape,wide", SHAPES)
def test_rows_get_the_odd_values_that_they_see(dtype, what, where, shape, wide):
    from torsh_b200.ops.kv_cache import kv_cache_attention
    q, kp, vp, ks, vs, table, start = _case(*shape, dtype)
    B, T, Hq, H, D, page = shape[:6]
    table = torch.nn.functional.pad(table, (0, wide), value=-1)
    mask = (torch.rand(B, T, T, device=DEV, generator=_gen(T)) < 0.4) | torch.eye(T, dtype=torch.bool, device=DEV)
    ref, mass = _attend64(q, kp, vp, ks, vs, table, start, mask, None, D ** -0.5)
    # per sequence two tokens: an early and a late one, of the new tokens or of the context
    plus, minus, nan = (torch.zeros(B, T, D, dtype=torch.bool, device=DEV) for _ in range(3))
    for b in range(B):
        s = int(start[b])
        places = [(1, s + 1), (T - 1, s + T - 1)] if where == "new" else [(None, s // 3), (None, s - 1)]
        for i, (j, pos) in enumerate(places):
            if pos < 0 or (where == "context" and s == 0):
                continue
            p, r = int(table[b, pos // page]), pos % page
            seen = mask[b, :, j] if j is not None else torch.ones(T, dtype=torch.bool, device=DEV)
            if what == "scales":
                vs[p, :, r] = (math.inf, math.nan)[i]
                nan[b, seen] = True
            elif dtype == BF16:
                vp[p, :, r, 3], vp[p, :, r, (D - 1, 40)[i]] = (math.inf, -math.inf)[i], (math.nan, math.inf)[i]
                (plus, minus)[i][b, seen, 3] = True
                (nan, plus)[i][b, seen, (D - 1, 40)[i]] = True
            else:
                vp.view(torch.int8)[p, :, r, (3, 40)[i]] = (0x7F, -1)[i]
                nan[b, seen, (3, 40)[i]] = True
    nan, plus, minus = nan | (plus & minus), plus & ~minus, minus & ~plus
    assert (nan | plus | minus).any()
    got = kv_cache_attention(q, kp, vp, table, start, mask, None, ks, vs)
    heads = lambda x: x[:, :, None].expand(B, T, Hq, D)   # noqa: E731
    if what == "scales":                                                    # infinity times a code is infinite or no number
        assert not torch.isfinite(got[heads(nan)]).any()
    else:
        assert got[heads(nan)].isnan().all()
        assert (got[heads(plus)] == math.inf).all() and (got[heads(minus)] == -math.inf).all()
    got = torch.where(heads(nan | plus | minus), ref.to(BF16), got)
    _attention_close(got, ref, mass, dtype)                                 # the reference has the tokens' old values, which these rows do not see
