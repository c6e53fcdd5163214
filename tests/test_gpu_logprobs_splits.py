"""Log probabilities under every split of a row over blocks and warps, and walks of many steps, against a vectorised evaluation in 64 bits.
Each case names the split that it is there for, so that a change of the rule shows."""
import re

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from berth_b200.kernels import ops   # noqa: E402
from tests.strict import wrong   # noqa: E402

INF, NAN = float("inf"), float("nan")


def _logits(seed, R, V, f32, pad):
    """Rows between undecided and certain; among them (from the first on, and one the last) rows that are masked but for a few, masked
    altogether, equal, rising, falling, of few values, with a NaN or an infinity."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(R, V + pad, device="cuda", generator=g) * 2.5
    likely = torch.randint(0, V, (R, 4), device="cuda", generator=g)
    x.scatter_(1, likely, torch.rand(R, 4, device="cuda", generator=g) * 18.0)
    token = torch.where(torch.rand(R, device="cuda", generator=g) < 0.5, likely[:, 0], torch.randint(0, V, (R,), device="cuda", generator=g))
    i = torch.arange(V + pad, device="cuda").float()
    few = torch.full_like(i, -INF)
    few[[0, V // 3, V // 2, V - 1]] = torch.tensor([1.0, 3.0, 1.0, 2.0], device="cuda")
    nan, inf = x[0].clone(), x[0].clone()
    nan[V // 2], inf[V - 2] = NAN, INF
    half = torch.where(i.long() % 2 == 1, x[0], torch.tensor(-INF, device="cuda"))
    kinds = [few, half, torch.zeros_like(i), -i / V * 9, i / V * 9, torch.floor(i / 7) % 5, torch.full_like(i, -INF), nan, inf,
             torch.where(i == V // 3, 30.0, -30.0)]
    at = seed % len(kinds)
    for r in {*range(min(R - 1, len(kinds))), R - 1}:
        if R > 2 or r == R - 1:
            x[r] = kinds[(at + r) % len(kinds)]
    token[0], token[R - 1] = V // 3, V - 1
    x[:, V:] = NAN
    return (x if f32 else x.half()), token.int()


def _reference(x, token, n, inv_temp):
    """(logprob, rank, entropy, top, top_logprob, ln z - max) of some rows, in 64 bits and whole numbers."""
    V = x.shape[1]
    bits = (x.float() + 0.0).view(torch.int32).long()
    value = torch.where(torch.isnan(x), -(1 << 31), torch.where(bits < 0, -(bits & 0x7fffffff), bits))
    order = (value << 24) + ((1 << 24) - 1 - torch.arange(V, device=x.device))
    t = token.long()[:, None]
    rank = (order > order.gather(1, t)).sum(1)
    rank[torch.isnan(x.gather(1, t)[:, 0])] = -1
    top = (1 << 24) - 1 - (torch.topk(order, n, 1)[0] & ((1 << 24) - 1))
    del order, value, bits
    z = x.double() * inv_temp
    most = z.amax(1, keepdim=True)                      # NaN where there is one
    z -= torch.where(torch.isinf(most), 0.0, most)
    lse = torch.log(torch.exp(z).sum(1, keepdim=True))
    lp = z - lse
    h = -torch.where(z > -INF, torch.exp(lp) * lp, 0.0).sum(1)
    none, bad = (most == -INF)[:, 0], (torch.isnan(most) | (most == INF))[:, 0]
    lp[none], h[none] = -INF, 0.0
    lp[bad], h[bad] = NAN, NAN
    return [v.cpu().numpy() for v in (lp.gather(1, t)[:, 0], rank, h, top, lp.gather(1, top), torch.where(none | bad, 0.0, lse[:, 0]))]


# rows, vocabulary, fp32, blocks of a row, warps of a block
CASES = [(1, 2314, True, 1, 8), (700, 5003, True, 1, 4), (600, 98301, False, 1, 8), (421, 60000, False, 1, 8), (1200, 248320, True, 1, 8),
         (421, 248320, False, 1, 16), (300, 120011, False, 1, 16), (600, 300007, True, 1, 16), (160, 38881, True, 4, 4), (1, 9001, False, 4, 4),
         (77, 100003, True, 8, 4), (150, 250000, False, 8, 4), (149, 700001, False, 8, 4), (40, 248320, True, 8, 8), (37, 1200007, False, 8, 8),
         (16, 248320, True, 16, 8), (2, 5000003, False, 16, 8), (1, 3000001, True, 16, 8)]


@pytest.mark.parametrize("R,V,f32,ctas,warps", CASES)
def test_every_split(R, V, f32, ctas, warps):
    for seed, n, inv_temp, pad in ((R, 5, 1.0, 0), (R + 1, 32, 1.25, 3), (R + 4, 0, 0.75, 0)):
        x, token = _logits(seed, R, V, f32, pad)
        f, i = dict(dtype=torch.float32, device="cuda"), dict(dtype=torch.int32, device="cuda")
        lp, rank, h, top, top_lp = torch.full((R,), NAN, **f), torch.full((R,), -7, **i), torch.full((R,), NAN, **f), torch.full((R, n), -7, **i), torch.full((R, n), NAN, **f)
        torch.cuda.synchronize()
        ops.logprobs(x, token, lp, rank, h, top, top_lp, V, inv_temp)
        ran = re.search(r"block=(\d+) .* cluster=(\d+)", ops.last_launch())
        assert (int(ran[1]), int(ran[2])) == (warps * 32, ctas), ops.last_launch()
        torch.cuda.synchronize()
        # in units of 2^-24: a term's exponent, four roundings of (x - max) * inv_temp * log2 e, 2.8 for each binary order that a likely
        # term lies below the largest (20 of them: 56), 2^y itself 4, trees, joins and logarithm below 36; a step of the walk adds its sum
        # and may move the maximum: three roundings
        steps = -(-V // ((4 if f32 else 8) * warps * 32 * ctas * 4))
        run = (3 * steps + 96) * 2.0 ** -24
        got = [v.cpu().numpy() for v in (lp, rank, h, top, top_lp)]
        some = max(1, (1 << 28) // (8 * V))
        for a in range(0, R, some):
            b = min(R, a + some)
            w_lp, w_rank, w_h, w_top, w_top_lp, spread = _reference(x[a:b, :V], token[a:b], n, inv_temp)
            assert (got[1][a:b] == w_rank).all(), (a, np.argwhere(got[1][a:b] != w_rank)[:4])
            assert (got[3][a:b] == w_top).all(), (a, np.argwhere(got[3][a:b] != w_top)[:4])
            size = lambda v: np.where(np.isfinite(v), np.abs(v), 0.0)
            for name, g, w, tol in (("logprob", got[0][a:b], w_lp, run + size(w_lp) * 6 * 2.0 ** -24), ("top", got[4][a:b], w_top_lp, run + size(w_top_lp) * 6 * 2.0 ** -24),
                                    ("entropy", got[2][a:b], w_h, 2 * run * (1 + size(w_h) + np.abs(spread)))):
                bad = wrong(g, w, tol)
                assert not bad.any(), (name, a, np.argwhere(bad)[:4], g[bad][:4], w[bad][:4])
