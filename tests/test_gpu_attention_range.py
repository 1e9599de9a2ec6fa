"""GPU: the cache's attentions at the ends of their range: large scores, values of very different sizes, unseen rows, sizes
near 2^31."""
import math

import numpy as np
import pytest

from test_gpu_window import Case, kx, sp  # noqa: F401 (kx: fixture)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def one_hot_rows(c, ctx, samples=None):
    """Large scores: a row whose largest score leads by more than both scores' errors is its key's value. A score is off by
    2^-19 of sum |q||k| (Case.check), so the lead has to be twice that and 40 (e^-40: no other weight shows); the value keeps 2^-18.
    Every row is finite and inside its values' range. Returns how many rows were decided."""
    B, Rq, S, H, Hkv, dk, dv = c.dims
    got = ctx[:, : H * dv].double().view(B, Rq, H, dv)
    decided = 0
    for b in range(B):
        ql, kl = c.q_len[b], c.k_len[b]
        seen = c.seen(b).cuda()
        for h in range(H):
            q, k, v = (x.cuda().double() for x in (c.q[b, :ql, h], c.k[b, :kl, h // (H // Hkv)], c.v[b, :kl, h // (H // Hkv)]))
            k, v = (torch.where(torch.isfinite(x), x, torch.zeros_like(x)) for x in (k, v))
            some = seen.any(1)
            s = (q @ k.T / math.sqrt(dk)).masked_fill(~seen, -math.inf)
            size = (q.abs() @ k.abs().T / math.sqrt(dk)).masked_fill(~seen, 0).amax(1)
            top = s.topk(min(2, kl), 1)
            lead = top.values[:, 0] - top.values[:, -1] if kl > 1 else torch.full((ql,), math.inf, device="cuda")
            sure = some & ((lead > 2 * size * 2.0**-19 + 40) | (seen.sum(1) == 1))
            out = got[b, :ql, h]
            assert bool(out.isfinite().all()), (b, h)
            assert bool((out.abs() <= v.abs().max() * (1 + 2.0**-18)).all()), (b, h)
            want = v[top.indices[:, 0]]
            assert bool(((out - want).abs()[sure] <= 2.0**-18 * v.abs().max()).all()), (b, h)
            decided += int(sure.sum())
    return decided


@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("Rq,S", [(300, 300), (9, 1500)])
@pytest.mark.parametrize("big", [1e3, 3e3, 1e4, 3e4, 1e5, 1e8])
def test_large_scores_of_a_prompt(kx, dk, Rq, S, big):  # noqa: F811
    """q and k of one size, so that no tile goes the plain way: scores up to 1e17, unsplit and split over CTAs"""
    c = Case(1, Rq, S, 4, 2, dk, 64, big=big, seed=21)
    assert one_hot_rows(c, c.run(kx)) > 3 * Rq
    assert int(c.status) == 0


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("score", [2.0**18, 2.0**21, 2.0**24, 2.0**26, 1.4 * 2.0**26, 2.0**27, 1.7 * 2.0**27, 2.0**30])
def test_large_scores_of_one_sign(kx, sign, score):  # noqa: F811
    """all scores near one another and far from zero: largest ones that are 2^-10 apart"""
    c = Case(1, 200, 200, 2, 1, 32, 48, window=150, sinks=3, seed=5)
    g = torch.Generator().manual_seed(3)
    a = 1 + torch.randperm(200, generator=g) / 1024.0
    c.k[:] = 0
    c.q[:] = 0
    c.k[0, :, 0, :4] = a[:, None] * 2.0**8
    c.q[0, :, :, :4] = sign * score / 4 / 2.0**8 * math.sqrt(32)
    assert one_hot_rows(c, c.run(kx)) == 2 * 200
    assert int(c.status) == 0
