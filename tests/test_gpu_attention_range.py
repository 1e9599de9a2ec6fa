"""GPU: the cache's attentions at the ends of their range: large scores, values of very different sizes, unseen rows, sizes
near 2^31."""
import math

import numpy as np
import pytest

from kv_model import ref
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


def scored(dtype, scores, v, heads=1, group=2, page=16, q0=1.0):
    """A cache (test_gpu_paged.Case) of rows whose keys have the given scores: key j is scores[j] / (4 q0) four times, q is
    q0 four times, the scale 1. scores: (rows, keys), v: (rows, keys, dv)."""
    import test_gpu_paged as tp
    rows, keys = scores.shape
    c = tp.Case([keys] * rows, heads, group, 64, v.shape[2], page, dtype)
    c.host = []
    k = torch.zeros(rows, keys, heads, 64, dtype=torch.float64)
    k[..., :4] = (scores.double() / (4 * q0))[:, :, None, None]
    stored = k.to(tp.DTYPES[dtype])
    assert bool((stored.double() == k).all())  # the scores are what was asked for
    values = v[:, :, None].expand(-1, -1, heads, -1).to(tp.DTYPES[dtype])
    j = torch.arange(keys)
    for r in range(rows):
        p = c.table[r, j.cuda() // page].long()
        c.k[0][p, :, j.cuda() % page] = stored[r].cuda()
        c.v[0][p, :, j.cuda() % page] = values[r].cuda()
        c.host.append((stored[r].double().numpy(), values[r].double().numpy()))
    c.q = torch.zeros(rows, heads * group, 64)
    c.q[..., :4] = q0
    c.q = c.q.view(rows, -1)
    return c


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("keys", [90, 4000])
def test_large_scores_over_the_cache(kx, dtype, sign, keys):  # noqa: F811
    """The largest base-2 scores from 2^18 to 2^40, by both launches: one key leads by 1/8 of its score, every other weight is 0;
    the value keeps 2^-18 (its weight's parts and the division)."""
    tops = [2.0**18, 2.0**24, 2.0**25, 1.25 * 2.0**25, 2.0**26, 1.25 * 2.0**26, 1.5 * 2.0**26, 2.0**27, 1.75 * 2.0**27, 2.0**28, 2.0**40]
    g = torch.Generator().manual_seed(keys)
    near = torch.randint(5, 8, (len(tops), keys), generator=g).double()  # eighths; negative scores: the least of them leads
    lead = torch.randint(0, keys, (len(tops),), generator=g)
    near[torch.arange(len(tops)), lead] = 8 if sign > 0 else 4
    scores = sign * near / 8 * torch.tensor(tops, dtype=torch.float64)[:, None]
    v = torch.randn(len(tops), keys, 72, generator=g)
    if sign < 0:
        scores *= 2
    # the keys' part of a score is below 2^12, so that every cache holds it; q takes the rest
    got = []
    for r, top in enumerate(tops):
        q0 = top / 2.0**12
        c = scored(dtype, scores[r:r + 1], v[r:r + 1], q0=q0)
        got.append(c.run(kx, scale=1 / math.log2(math.e)).view(2, 72).cpu().double())
        want = torch.from_numpy(c.host[0][1][lead[r], 0])
        assert bool(got[-1].isfinite().all()), top
        assert float((got[-1] - want).abs().max()) <= 2.0**-18 * float(v.abs().max()), top
        assert int(c.status) == 0


@pytest.mark.parametrize("Rq,S,window,sinks,dk", [(150, 700, 100, 5, 64), (150, 700, 90, 0, 128), (9, 3000, 1500, 70, 64),
                                                   (20, 2500, 1111, 3, 128), (64, 70, 3, 2, 32)])
def test_unseen_rows_leave_no_trace(kx, Rq, S, window, sinks, dk):  # noqa: F811
    """the same bits whatever lies in rows that no query sees, behind the last key or in the rows behind the queries"""
    k_len, q_len = [S, S - 30, S], [Rq, Rq - 3, 1]
    out = []
    for fill in (0.0, float("nan"), float("inf"), 1e6, 1e-30, -3e38):
        c = Case(3, Rq, S, 4, 2, dk, 64, window, sinks, q_len=q_len, k_len=k_len, seed=6)
        for b in range(3):
            unseen = torch.ones(S, dtype=torch.bool)
            unseen[: k_len[b]] = ~c.seen(b).any(0)
            assert b or bool(unseen.any())
            c.k[b][unseen] = fill
            c.v[b][unseen] = fill
            c.q[b, q_len[b]:] = fill
        out.append(c.run(kx).clone())
        assert int(c.status) == 0
    c.check(out[0])
    for o in out[1:]:
        assert torch.equal(o, out[0])


@pytest.mark.parametrize("dk,dv", [(64, 64), (32, 128)])
@pytest.mark.parametrize("Rq,S", [(512, 512), (5, 2000)])
@pytest.mark.parametrize("far,drop", [(2.0**18, -17.375), (2.0**25, -20.75), (2.0**30, -20.75), (2.0**38, -26.375), (2.0**39, -20)])
def test_tiles_of_far_values_under_small_weights(kx, Rq, S, dk, dv, far, drop):  # noqa: F811
    """Every other pair of 64-key tiles holds values `far` times the others' under weights of about e^drop: the output keeps
    its bits relative to sum p|v|, whichever comes first. Scores are single exact products; the exponential's argument is
    off by three roundings of at most 40 (2^-24 each) and a weight twice by that; p's and the values' parts, the
    exponential and the sums: 2^-18, as everywhere."""
    for first in (0, 1):
        c = Case(1, Rq, S, 2, 1, dk, dv, seed=17)
        j = torch.arange(S)
        high = (j // 128) % 2 == first
        g = torch.Generator().manual_seed(4)
        score = torch.randint(-16, 1, (S,), generator=g) / 8 + torch.where(high, drop, 0.0)
        c.k[:] = 0
        c.k[0, :, 0, 1] = score
        c.q[:] = 0
        c.q[..., 1] = 1
        c.v = c.v.sign() * (1 + torch.rand(c.v.shape, generator=g))
        c.v[0, high] *= far
        got = c.run(kx, scale=1.0).double().view(Rq, 2, dv)
        seen, v = c.seen(0).cuda(), c.v[0, :, 0].double().cuda()
        p = torch.exp(score.double().cuda())[None] * seen
        p = p / p.sum(1, keepdim=True)
        size = p @ v.abs().amax(1)
        tol = math.expm1(2 * 3 * 40 * 2.0**-24) + 2.0**-18
        assert float(((got - (p @ v)[:, None]).abs() / size[:, None, None]).max()) <= tol
        assert int(c.status) == 0


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("keys", [90, 6001])
@pytest.mark.parametrize("small,drop", [(2.0**-14, -20.75), (2.0**-20, -24.25), (2.0**-2, -17.375), (2.0**-10, -24.25), (2.0**-14, -27.75)])
def test_steps_of_far_values_under_small_weights_over_the_cache(kx, dtype, keys, small, drop):  # noqa: F811
    """Pairs of 16-key steps with values of 2^15 under weights of about e^drop, in turn with pairs of small values under
    large weights: the output keeps its bits relative to sum p|v|. Tolerance as for the prompt's tiles."""
    for first in (0, 1):
        g = torch.Generator().manual_seed(keys)
        high = (torch.arange(keys) // 32) % 2 == first
        scores = torch.randint(-16, 1, (2, keys), generator=g) / 8 + torch.where(high, drop, 0.0)
        v = (1 + torch.rand(2, keys, 72, generator=g)) * torch.randn(2, keys, 72, generator=g).sign()
        v = (v * torch.where(high, 2.0**15, small)[:, None]).half().float().clamp(-65504, 65504)  # 65536 is not an f16 number
        c = scored(dtype, scores, v, group=3)
        got = c.run(kx, scale=1.0).view(2, 3, 72).cpu().double()
        p = torch.softmax(scores.double(), 1)
        tol = math.expm1(2 * 3 * 40 * 2.0**-24) + 2.0**-18
        for r in range(2):
            stored = torch.from_numpy(c.host[r][1][:, 0])
            size = p[r] @ stored.abs().amax(1)
            assert float((got[r] - p[r] @ stored).abs().max() / size) <= tol
        assert int(c.status) == 0


def test_a_timeout_keeps_the_status_bits(kx):  # noqa: F811
    """one status word for a step's calls: a wait that gives up adds its bit to those that are there"""
    status = torch.full((1,), 2 | 4, dtype=torch.int32, device="cuda")
    waited = torch.zeros(1, dtype=torch.int64, device="cuda")
    kx.call("kx_probe_bounded_wait", 0, 5_000_000, status.data_ptr(), waited.data_ptr(), None)
    torch.cuda.synchronize()
    assert int(status) == 1 | 2 | 4


@pytest.mark.parametrize("window", [0, 40])
def test_the_most_query_rows(kx, window):  # noqa: F811
    """Rq of 2^31 - 1, of which the sample has a few: the rows behind them are not there"""
    c = Case(1, 150, 200, 2, 1, 32, 32, window=window, sinks=1, q_len=[150], k_len=[200])
    want = c.run(kx).clone()
    c.args(kx)
    dims, c.dims = c.dims, (1, 2**31 - 1) + c.dims[2:]
    c.launch(kx, sp())
    torch.cuda.synchronize()
    c.dims = dims
    c.check(c.ctx)
    assert torch.equal(c.ctx, want) and int(c.status) == 0


@pytest.mark.parametrize("rows", [2**31 - 1, 2**31 - 65535, 65535 * 16 + 1])
def test_append_with_the_most_rows(kx, rows):  # noqa: F811
    """room for up to 2^31 - 1 rows per slot, of which the first slot has 13: the others are not there"""
    from test_gpu_kv import Pair
    out = []
    for r in (13, rows):
        p = Pair(kx, 2, 4, 12, 8, heads=2, dk=16, dv=24, dtype="f32")
        p.extend([13, 0])
        x, count = torch.randn(13, 48, generator=torch.Generator().manual_seed(2)).cuda(), p.ints([13, 0])
        kx.call("kx_kv_append", ref(p.c), 0, x.data_ptr(), 48, x.data_ptr(), 48, count.data_ptr(), r, p.status.data_ptr(), sp())
        torch.cuda.synchronize()
        assert int(p.status) == 0
        out.append((p.bits(p.k), p.bits(p.v)))
    assert np.array_equal(out[0][0], out[1][0]) and np.array_equal(out[0][1], out[1][1])


@pytest.mark.parametrize("dtype,page,max_pages", [("f16", 8, 2**28 - 1), ("f16", 16, 2**27 - 1), ("f32", 1, 2**31 - 1025), ("bf16", 1, 2**31 - 1025)])
def test_sequences_of_almost_2_to_31_tokens(kx, dtype, page, max_pages):  # noqa: F811
    """A table that names few pages again and again: 0 for the first half, 1 for the second, 2 for the last 16 tokens, 3 for
    the first 16. A lane adds up to 2^19 terms (2^31 over 1184 warps of four lanes): an fp32 sum is off by 2^19 2^-24 of itself at most,
    the output by twice that."""
    import test_gpu_paged as tp
    length, d, n = max_pages * page, 8, 16 // page if page < 16 else 1
    g = torch.Generator().manual_seed(1)
    k = torch.randn(4 * n, page, d, generator=g).to(tp.DTYPES[dtype])
    v = (torch.randn(4 * n, page, d, generator=g) / 8 + torch.tensor([1.0, 3.0, 7.0, -5.0]).repeat_interleave(n)[:, None, None]).to(tp.DTYPES[dtype])
    table = torch.empty(1, max_pages, dtype=torch.int32, device="cuda")
    for at, which in ((0, 0), (max_pages // 2, 1)):
        table[0, at:] = which * n
    table[0, -n:] = torch.arange(2 * n, 3 * n, dtype=torch.int32, device="cuda")
    table[0, :n] = torch.arange(3 * n, 4 * n, dtype=torch.int32, device="cuda")
    lens = torch.tensor([length], dtype=torch.int32, device="cuda")
    c = tp.Case.__new__(tp.Case)
    c.lens, c.heads, c.G, c.dk, c.dv, c.page, c.layer, c.dtype = [length], 1, 2, d, d, page, 0, dtype
    c.k, c.v = k.cuda()[None, :, None].contiguous(), v.cuda()[None, :, None].contiguous()
    c.q, c.table, c.d_lens = torch.randn(1, 2 * d, generator=g) / 4, table, lens
    c.refs, c.status = torch.ones(4 * n, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    q = c.q.double().view(2, d)
    rows = lambda ids: [x.double()[ids].reshape(-1, d) for x in (k, v)]  # noqa: E731
    (k0, v0), (k2, v2), (k3, v3) = (rows(list(range(i * n, i * n + n))) for i in (0, 2, 3))
    # the first tokens and the window's
    c.window, c.sinks = 5, 3
    got = c.run(kx).view(2, d).double().cpu()
    want, tol = tp.exact(q.numpy(), torch.cat([k3[:3], k2[-5:]]).numpy(), torch.cat([v3[:3], v2[-5:]]).numpy(), 1 / math.sqrt(d))
    assert np.all(np.abs(got.numpy() - want) <= tol)
    # all of them: page 0 and page n half each, the 32 others do not show
    c.window, c.sinks = 0, 0
    got = c.run(kx).view(2, d).double().cpu()
    kk, vv = (torch.cat([x.double()[0], x.double()[n]]) for x in (k, v))
    want = torch.softmax(q @ kk.T / math.sqrt(d), 1) @ vv
    assert float((got - want).abs().max()) <= 2 * (2.0**19 * 2.0**-24) * 3.5, (got, want)
    assert int(c.status) == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("keys", [1, 2, 15, 90, 4000])
def test_the_largest_values_over_the_cache(kx, dtype, keys):  # noqa: F811
    """nearly equal weights over values just below 2^127: the output is one of them, not the overflow of their sum"""
    g = torch.Generator().manual_seed(keys)
    scores = torch.randint(-4, 1, (2, keys), generator=g) / 8
    v = 2.0**126 * (1.5 + torch.rand(2, keys, 40, generator=g, dtype=torch.float64) / 4)
    v[1] *= torch.randn(keys, 40, generator=g).sign()
    c = scored(dtype, scores, v)
    got = c.run(kx, scale=1.0).view(2, 2, 40).cpu().double()
    for r in range(2):
        want = torch.softmax(scores[r].double(), 0) @ torch.from_numpy(c.host[r][1][:, 0])
        assert float((got[r] - want).abs().max()) <= 2.0**-17 * 2.0**127
    assert int(c.status) == 0


@pytest.mark.parametrize("S", [2, 130, 1000])
def test_the_largest_values_of_a_prompt(kx, S):  # noqa: F811
    """the plain way"""
    c = Case(1, S, S, 2, 1, 32, 32, window=700, sinks=2, seed=8)
    g = torch.Generator().manual_seed(S)
    c.v = 2.0**127 * (1.5 + torch.rand(c.v.shape, generator=g, dtype=torch.float64) / 4).float()
    c.v[0, ::3] *= -1
    got = c.run(kx).double().view(S, 2, 32)
    seen = c.seen(0).cuda()
    for h in range(2):
        s = (c.q[0, :, h].double().cuda() @ c.k[0, :, 0].double().cuda().T / math.sqrt(32)).masked_fill(~seen, -math.inf)
        want = torch.softmax(s, 1) @ c.v[0, :, 0].double().cuda()
        assert float((got[:, h] - want).abs().max()) <= 2.0**-17 * 2.0**128


@pytest.mark.parametrize("B,S", [(1, 3000), (40, 90)])
def test_queries_without_keys(kx, B, S):  # noqa: F811
    """samples of no keys: rows of zeros, split launches and others; the rows behind the queries are left alone"""
    c = Case(B, 20, S, 2, 1, 64, 40, q_len=[17] * B, k_len=[0] * B)
    ctx = c.run(kx).view(B, 20, 80)
    assert not ctx[:, :17].any() and bool((ctx[:, 17:] == 7).all()) and int(c.status) == 0
