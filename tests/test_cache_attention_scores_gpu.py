"""How exact the scores of attention over an int8 cache are, where sums of queries are large and sums of products are small."""
import pytest
import torch

from test_decoding_gpu import BF16, DEV, _gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("G,wide", [(1, 0), (12, 0), (20, 5000)])
def test_scores_of_queries_of_one_sign(G, wide):
    """Two tokens whose codes differ everywhere and whose scores are within 1 of each other, values 1 and -1: the output is tanh(difference / 2).

    A score is a sum of 128 products of a bf16 query in [1, 2) and a code, in steps of 16 that are added up in fp32: eight roundings (or
    truncations) of at most 2^-23 of the partial sum; whichever columns a step takes, they are alike. The two probabilities are rounded to halves
    (2^-11 each, 2^-10 of the difference of the scores), the output to bf16: 2^-8 of it, times the slope 2 / (1 - out^2). The root of the mean square of a
    sum is at most the sum of the roots of the mean squares."""
    from torsh_b200.ops.kv_cache import kv_cache_attention
    B, H, D = 64, 4, 128
    g = _gen(G)
    q = (1 + torch.rand(B, 1, H, 1, D, device=DEV, generator=g)).to(BF16)
    codes = torch.randint(-120, 121, (B, H, 2, D), device=DEV, generator=g).double()
    w = q[:, 0, :, 0].double()
    for c in range(D):                                                      # token 1 comes as near to token 0 as a code can bring it
        gap = ((codes[:, :, 0] - codes[:, :, 1]) * w).sum(-1)
        codes[:, :, 1, c] = (codes[:, :, 1, c] + (gap / w[..., c]).round()).clamp(-127, 127)
    gap = ((codes[:, :, 0] - codes[:, :, 1]) * w).sum(-1)
    assert gap.abs().max() <= 1 and int(codes.abs().max()) <= 127
    partial = (codes * w[:, :, None]).cumsum(-1)[..., 15::16].square().mean((0, 1, 2)).sqrt().sum()
    kp, vp = (torch.zeros(B, H, 16, D, dtype=torch.int8, device=DEV) for _ in range(2))
    kp[:, :, :2] = codes.to(torch.int8)
    vp[:, :, 0], vp[:, :, 1] = 1, -1
    ones = torch.ones(B, H, 16, device=DEV)
    table = torch.nn.functional.pad(torch.arange(B, device=DEV).int()[:, None], (0, wide), value=-1)
    qq = q.expand(B, 1, H, G, D).reshape(B, 1, H * G, D)
    out = kv_cache_attention(qq, kp, vp, table, torch.ones(B, dtype=torch.int32, device=DEV), None, None, ones, ones, scale=1.0)
    y = out.double().view(B, H, G, D)[..., 0]
    rms = lambda x: float(x.square().mean().sqrt())   # noqa: E731
    off = rms(2 * torch.atanh(y) - gap[..., None])
    bound = 2 * 2.0 ** -23 * float(partial) + 2.0 ** -10 + 2.0 ** -8 * rms(2 * y / (1 - y * y))
    assert off <= bound < 0.007, (off, bound)
