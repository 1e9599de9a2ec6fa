"""GPU: attention of prompts with a sliding window and visible first tokens against the definition in 64 bits."""
import math

import numpy as np
import pytest

from kv_model import BAD_REQUEST

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kx(libkx):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from kernix_b200 import kx_abi
    return kx_abi


def sp():
    return torch.cuda.current_stream().cuda_stream


class Case:
    """Rows of B samples; what no query sees (and the columns behind the rows) is NaN."""

    def __init__(self, B, Rq, S, H, Hkv, dk, dv, window=0, sinks=0, q_len=None, k_len=None, big=1.0, pad=0, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.dims, self.window, self.sinks = (B, Rq, S, H, Hkv, dk, dv), window, sinks
        self.q_len = q_len if q_len is not None else [Rq] * B
        self.k_len = k_len if k_len is not None else [S] * B
        self.lens_given = q_len is not None or k_len is not None
        self.ld = [H * dk + pad, Hkv * dk + pad, Hkv * dv + pad, H * dv + pad]
        rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float32)  # noqa: E731
        self.q, self.k, self.v = rnd(B, Rq, H, dk) * big, rnd(B, S, Hkv, dk) * big, rnd(B, S, Hkv, dv)
        for b in range(B):
            self.q[b, self.q_len[b]:] = float("nan")
            seen = self.seen(b).any(0)
            self.k[b, : self.k_len[b]][~seen] = float("nan")
            self.v[b, : self.k_len[b]][~seen] = float("inf")
            self.k[b, self.k_len[b]:] = float("nan")
            self.v[b, self.k_len[b]:] = float("-inf")

    def seen(self, b):
        t = np.arange(self.k_len[b] - self.q_len[b], self.k_len[b])[:, None]
        j = np.arange(self.k_len[b])[None, :]
        return torch.from_numpy((j <= t) & ((self.window <= 0) | (j > t - self.window) | (j < self.sinks)))

    def padded(self, x, ld):
        rows = x.reshape(-1, x.shape[2] * x.shape[3])
        out = torch.full((rows.shape[0], ld), float("nan"))
        out[:, : rows.shape[1]] = rows
        return out.cuda()

    def args(self, kx):
        B, Rq, S, H, Hkv, dk, dv = self.dims
        self.d = [self.padded(x, ld) for x, ld in zip((self.q, self.k, self.v), self.ld)]
        self.ctx = torch.full((B * Rq, self.ld[3]), 7.0, device="cuda")
        self.lens = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (self.q_len, self.k_len)]
        self.ws = torch.empty(kx.lib().kx_attention_window_ws(B, S, Hkv, dk, dv), dtype=torch.uint8, device="cuda")
        self.ws.fill_(255)
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def launch(self, kx, stream, scale=0.0):
        B, Rq, S, H, Hkv, dk, dv = self.dims
        ql, kl = [x.data_ptr() if self.lens_given else None for x in self.lens]
        kx.call("kx_attention_window", self.d[0].data_ptr(), self.ld[0], self.d[1].data_ptr(), self.ld[1], self.d[2].data_ptr(),
                self.ld[2], self.ctx.data_ptr(), self.ld[3], B, Rq, S, H, Hkv, dk, dv, ql, kl, self.window, self.sinks, scale,
                self.ws.data_ptr(), self.ws.numel(), self.status.data_ptr(), stream)

    def run(self, kx, scale=0.0):
        self.args(kx)
        self.launch(kx, sp(), scale)
        torch.cuda.synchronize()
        return self.ctx

    def check(self, ctx, scale=0.0, samples=None):
        """Scores: products of operands kept to 2^-21 (two parts, both sides) summed in at most 24 tensor-core steps that may
        truncate (24 x 2^-24): under 2^-19 of sum |q||k|; a weight is off by exp(+-that), twice. Weights' and values'
        parts (2^-22 each, of the largest value in 64 keys where that is more), the exponential, a tile's 12 steps and
        the fp32 sums over the tiles: under 2^-18 of the largest value seen."""
        B, Rq, S, H, Hkv, dk, dv = self.dims
        scale = scale or 1 / math.sqrt(dk)
        G = H // Hkv
        got = ctx[:, : H * dv].double().view(B, Rq, H, dv)
        for b in samples if samples is not None else range(B):
            ql, kl = self.q_len[b], self.k_len[b]
            if ql == 0:
                continue
            seen = self.seen(b).cuda()
            for h in range(H):
                q, k, v = (x.cuda().double() for x in (self.q[b, :ql, h], self.k[b, :kl, h // G], self.v[b, :kl, h // G]))
                k, v = (torch.where(torch.isfinite(x), x, torch.zeros_like(x)) for x in (k, v))
                s = (scale * q @ k.T).masked_fill(~seen, -math.inf)
                top = s.amax(1, keepdim=True)
                p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
                den = p.sum(1, keepdim=True)
                want = p @ v / torch.where(den == 0, torch.ones_like(den), den)
                size = (abs(scale) * q.abs() @ k.abs().T).masked_fill(~seen, 0).amax(1, keepdim=True)
                tol = (torch.expm1(2 * size * 2.0**-19) + 2.0**-18) * v.abs().max()
                err = (got[b, :ql, h] - want).abs()
                assert bool((err <= tol).all()), (b, h, float(err.max()), float(tol.max()), int(torch.argmax(err.amax(1))))
        for b in range(B):
            assert bool((got[b, self.q_len[b]:] == 7).all())
        if self.ld[3] > H * dv:
            assert bool((ctx[:, H * dv:] == 7).all())


@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (32, 16), (80, 72), (1, 1), (50, 33), (128, 64), (16, 128)])
@pytest.mark.parametrize("S", [1, 63, 64, 65, 129, 400])
def test_head_dims_and_lengths(kx, dk, dv, S):
    c = Case(2, S, S, 4, 2, dk, dv, window=0, seed=S)
    c.check(c.run(kx))
    assert int(c.status) == 0


@pytest.mark.parametrize("G", [1, 3, 8, 130])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (64, 64), (65, 100), (200, 0), (100000, 5), (0, 9), (130, 700)])
def test_windows_and_shared_heads(kx, G, window, sinks):
    c = Case(1, 300, 300, G, 1, 64, 64, window, sinks, seed=G)
    c.check(c.run(kx))


@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4), (300, 70)])
def test_ragged_samples_and_chunks(kx, window, sinks):
    """chunks of longer sequences, samples without queries or keys, more queries than keys"""
    c = Case(8, 150, 700, 6, 2, 72, 80, window, sinks, q_len=[150, 0, 1, 149, 64, 30, 0, 150], k_len=[700, 400, 700, 149, 65, 7, 0, 1])
    ctx = c.run(kx)
    c.check(ctx)
    assert not ctx[5 * 150:5 * 150 + 23].any() and not ctx[7 * 150:7 * 150 + 149].any() and int(c.status) == 0


@pytest.mark.parametrize("window,sinks,Rq", [(0, 0, 3000), (700, 4, 3000), (2000, 0, 5)])
def test_long(kx, window, sinks, Rq):
    c = Case(1, Rq, 3000, 8, 2, 128, 128, window, sinks, seed=5)
    c.check(c.run(kx))
    again = c.ctx.clone()
    c.launch(kx, sp())
    torch.cuda.synchronize()
    assert torch.equal(again, c.ctx)


@pytest.mark.parametrize("B,Rq,S,H,Hkv,dk,dv,window,sinks", [
    (1, 1, 5000, 1, 1, 64, 64, 0, 0), (1, 1, 3000, 8, 2, 128, 128, 0, 0), (2, 129, 4000, 2, 2, 64, 50, 0, 0),
    (1, 100, 4000, 3, 1, 128, 33, 1500, 7), (3, 300, 1100, 6, 2, 80, 72, 0, 0), (1, 40, 2500, 140, 1, 32, 32, 0, 0)])
def test_few_rows_over_many_keys(kx, B, Rq, S, H, Hkv, dk, dv, window, sinks):
    """blocks of rows whose keys are split over several CTAs"""
    c = Case(B, Rq, S, H, Hkv, dk, dv, window, sinks, seed=S)
    ctx = c.run(kx).clone()
    c.check(ctx)
    c.launch(kx, sp())
    torch.cuda.synchronize()
    assert torch.equal(ctx, c.ctx)


def test_split_blocks_of_all_kinds(kx):
    """some with a few keys, some without any, a bad sample, one with values that parts cannot hold"""
    c = Case(5, 60, 2000, 2, 1, 64, 64, q_len=[60, 60, 30, 0, 60], k_len=[2000, 70, 7, 5, 1900], pad=3)
    c.k[4, 1000, 0, 3] = float("nan")
    c.args(kx)
    c.launch(kx, sp())
    torch.cuda.synchronize()
    ctx = c.ctx[:, :128]
    c.k[4, 1000, 0, 3] = 0
    assert bool(ctx[240:300].isnan().all())
    c.ctx[240:300, :128] = float("nan")
    c.check(c.ctx, samples=[0, 1, 2, 3])
    c.lens[1][0] = 2001
    c.launch(kx, sp())
    torch.cuda.synchronize()
    assert bool(c.ctx[:60, :128].isnan().all()) and int(c.status) == BAD_REQUEST
    c.ctx[:60, :128] = 0
    c.check(c.ctx, samples=[1, 2, 3])


@pytest.mark.parametrize("pad", [1, 3, 4])
def test_row_pitches(kx, pad):
    c = Case(2, 70, 130, 4, 2, 64, 48, 50, 2, pad=pad)
    c.check(c.run(kx))


@pytest.mark.parametrize("scale", [-0.2, 1e-8, 3.0])
def test_scales(kx, scale):
    c = Case(1, 100, 100, 2, 1, 32, 32)
    c.check(c.run(kx, scale), scale)


@pytest.mark.parametrize("big", [1e-15, 1e-6, 40.0])
def test_small_and_large_values(kx, big):
    c = Case(1, 200, 200, 4, 2, 64, 64, 90, 3, big=big)
    c.check(c.run(kx))


@pytest.mark.parametrize("big", [1e-8, 1e-13, 1e-20, 1e-32, 1e10, 1e15])
@pytest.mark.parametrize("Rq", [9, 300])
def test_small_and_large_v(kx, big, Rq):
    """outputs as exact relative to their own values, whatever their size"""
    c = Case(2, Rq, 300, 4, 2, 64, 80, window=90, sinks=3, seed=12)
    c.v *= big
    c.check(c.run(kx))
    assert int(c.status) == 0


def test_one_large_value_among_small_ones(kx):
    """a key and a value 2^12 times the others in their tile: the others keep their accuracy"""
    c = Case(1, 200, 200, 2, 2, 64, 64)
    c.k[0, 70, :, 5] *= 4096 / 8
    c.v[0, 70, :, 7] *= 4096
    ctx = c.run(kx)
    c.check(ctx)
    first = Case(1, 200, 200, 2, 2, 64, 64)  # rows before it: as if it were not there, to fp32's accuracy
    want = first.run(kx)
    assert float((ctx[:70] - want[:70]).abs().max()) <= 2.0**-18 * float(first.v.abs().max())


@pytest.mark.parametrize("what", ["k_nan", "v_nan", "v_inf", "k_huge", "q_huge", "q_nan"])
def test_values_that_parts_cannot_hold(kx, what):
    """rows that do not see them are as exact as ever, rows that do follow the formula"""
    c = Case(1, 300, 300, 4, 2, 64, 64, window=120, sinks=2)
    kv = {"k_nan": (c.k, float("nan")), "v_nan": (c.v, float("nan")), "v_inf": (c.v, float("inf")), "k_huge": (c.k, 1e25)}
    if what in kv:
        t, value = kv[what]
        t[0, 100, 0, 9] = value
        bad, heads = range(100, 220), [0, 1]
    else:
        c.q[0, 30, 1, 9] = 1e25 if what == "q_huge" else float("nan")
        bad, heads = [30], [1]
    ctx = c.run(kx).view(300, 4, 64).clone()
    for i in bad:
        for h in heads:
            row = ctx[i, h]
            if what == "v_nan":
                assert bool(row[9].isnan()) and bool(row[:9].isfinite().all()) and bool(row[10:].isfinite().all())
            elif what == "v_inf":
                assert float(row[9]) == math.inf and bool(row[:9].isfinite().all())
            elif what in ("k_nan", "q_nan"):
                assert bool(row.isnan().all())
            else:
                assert bool(row.isfinite().all())
    clean = Case(1, 300, 300, 4, 2, 64, 64, window=120, sinks=2)
    if what not in kv:
        clean.q[0, 30, 1, 9] = 0
    want = clean.run(kx).view(300, 4, 64)
    keep = torch.ones(300, 4, dtype=torch.bool)
    for i in bad:
        for h in heads:
            keep[i, h] = False
    diff = (ctx - want)[keep.cuda()].abs().max()
    assert float(diff) <= 2.0**-17 * float(clean.v[:, :, :].abs().max())
    if what.endswith("huge"):  # one weight takes the row, or none of the others'
        q, k, v = (x.double() for x in (c.q, c.k, c.v))
        i, h = list(bad)[0], heads[0]
        seen = c.seen(0)[i]
        s = (k[0, :, h // 2] @ q[0, i, h]) / 8
        p = torch.softmax(s.masked_fill(~seen, -math.inf), 0)
        assert float((ctx[i, h].cpu().double() - p @ v[0, :, h // 2]).abs().max()) <= 2.0**-17 * float(v.abs().max())


@pytest.mark.parametrize("far", [1e6, 3e8, 1e11, -1e9])
@pytest.mark.parametrize("what", ["k", "v", "both"])
def test_one_row_far_above_its_neighbours(kx, what, far):
    """finite, but so far above the rest of its tile that common scales would cost the others their bits: rows that do not see
    it are as exact as ever, rows that do follow the formula, whether it takes all of the weight or none"""
    def make(value):
        c = Case(1, 300, 300, 4, 2, 64, 64, window=120, sinks=2, seed=3)
        if what != "v":
            c.k[0, 100, 0, 9] = value
        if what != "k":
            c.v[0, 100, 0, 7] = value
        return c
    c, clean = make(far), make(1.0)
    got, want = c.run(kx).view(300, 4, 64).clone(), clean.run(kx).view(300, 4, 64)
    top = float(clean.v.abs().max())
    unseen = torch.ones(300, 4, dtype=torch.bool)
    unseen[100:220, :2] = False
    unseen = unseen.cuda()
    assert float((got - want)[unseen].abs().max()) <= 2.0**-17 * top
    q, k, v = (x.double().cuda() for x in (c.q, c.k, c.v))
    seen = c.seen(0).cuda()
    for h in range(2):
        s = (q[0, :, h] @ torch.where(torch.isfinite(k[0, :, 0]), k[0, :, 0], 0.0).T / 8).masked_fill(~seen, -math.inf)
        p = torch.softmax(s, 1)
        v0 = torch.where(torch.isfinite(v[0, :, 0]), v[0, :, 0], 0.0)
        # against the weights' share of the far value, and of the others
        tol = 2.0**-15 * (p @ v0.abs())[100:220] + 2.0**-17 * top
        err = (got[100:220, h].double() - (p @ v0)[100:220]).abs()
        if what != "v":  # scores of 1e6 and more are only good to 2^-24 of themselves in fp32: rows where two keys tie are left out
            err, tol = err[(s[100:220].topk(2).values.diff(dim=1).abs() > 1).squeeze(1)], tol[(s[100:220].topk(2).values.diff(dim=1).abs() > 1).squeeze(1)]
        assert bool((err <= tol).all()), float((err / tol).max())


def test_bad_lengths(kx):
    for ql, kl in (([5, -1], [9, 9]), ([11, 3], [9, 9]), ([5, 5], [10, 9]), ([5, 5], [9, -2])):
        c = Case(2, 10, 9, 2, 1, 32, 32, q_len=[5, 5], k_len=[9, 9])
        c.args(kx)
        c.lens = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (ql, kl)]
        c.launch(kx, sp())
        torch.cuda.synchronize()
        bad = [b for b in range(2) if not (0 <= ql[b] <= 10 and 0 <= kl[b] <= 9)][0]
        assert int(c.status) == BAD_REQUEST and bool(c.ctx[bad * 10:bad * 10 + 10].isnan().all())
        good = c.ctx[(1 - bad) * 10:(1 - bad) * 10 + ql[1 - bad]]
        assert bool(good.isfinite().all())


@pytest.mark.parametrize("window,sinks", [(2**31 - 1, 2**31 - 1), (2**31 - 1, 0), (70, 2**31 - 1), (69, 2**31 - 1)])
def test_largest_windows(kx, window, sinks):
    """the largest numbers, with queries before the first key"""
    c = Case(2, 90, 70, 3, 1, 32, 32, window, sinks, q_len=[90, 70], k_len=[70, 70])
    ctx = c.run(kx)
    c.check(ctx)
    assert not ctx[:20].any()


def test_as_kx_attention(kx):
    """without a window the causal case of the library's attention"""
    c = Case(3, 128, 128, 8, 8, 64, 64)
    ctx = c.run(kx)
    out = torch.zeros_like(ctx)
    kx.call("kx_attention", c.d[0].data_ptr(), 512, c.d[1].data_ptr(), 512, c.d[2].data_ptr(), 512, out.data_ptr(), 512, 3, 128, 128, 8,
            64, 64, 1, c.status.data_ptr(), sp())
    torch.cuda.synchronize()
    c.check(ctx)
    c.check(out)


def test_captured_and_on_two_streams(kx):
    cases = [Case(2, 200, 300, 4, 2, 64, 64, 100, 3, seed=i) for i in range(2)]
    want = [c.run(kx).clone() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    graphs = [torch.cuda.CUDAGraph() for _ in cases]
    for c, g, s in zip(cases, graphs, streams):
        c.args(kx)
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            c.launch(kx, torch.cuda.current_stream().cuda_stream)
    for _ in range(5):
        for c, g, s in zip(cases, graphs, streams):
            with torch.cuda.stream(s):
                c.ctx.fill_(0)
                g.replay()
    torch.cuda.synchronize()
    for c, w in zip(cases, want):
        assert torch.equal(c.ctx, w)
    cases[0].ctx.fill_(7)
    torch.cuda.synchronize()
    cases[0].launch(kx, None)      # the default stream
    torch.cuda.synchronize()
    assert torch.equal(cases[0].ctx, want[0])


def test_prompt_then_tokens_agree(kx):
    """a prompt's last row is what the token attention computes from a cache that holds its keys and values"""
    from kv_model import describe, ref
    B, S, H, Hkv, d, page, window, sinks = 3, 333, 8, 2, 64, 16, 100, 4
    k_len = [333, 7, 120]
    c = Case(B, S, S, H, Hkv, d, d, window, sinks, q_len=k_len, k_len=k_len, seed=9)
    ctx = c.run(kx)
    pages = 21
    table = torch.arange(B * pages, dtype=torch.int32, device="cuda").view(B, pages).flip(1).contiguous()
    kp, vp = (torch.zeros(1, B * pages, Hkv, page, d, device="cuda") for _ in range(2))
    lens = torch.tensor(k_len, dtype=torch.int32, device="cuda")
    refs = torch.ones(B * pages, dtype=torch.int32, device="cuda")
    cache = describe(kx, kp, vp, table, lens, refs, "f32")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    kx.call("kx_kv_append", ref(cache), 0, c.d[1].data_ptr(), c.ld[1], c.d[2].data_ptr(), c.ld[2], lens.data_ptr(), S, st.data_ptr(), sp())
    q = torch.stack([c.d[0][b * S + k_len[b] - 1] for b in range(B)])
    out = torch.zeros(B, H * d, device="cuda")
    ws = torch.empty(kx.lib().kx_attention_paged_ws(ref(cache), H, B), dtype=torch.uint8, device="cuda")
    kx.call("kx_attention_paged", ref(cache), 0, q.data_ptr(), H * d, H, None, B, window, sinks, 0.0, out.data_ptr(), H * d,
            ws.data_ptr(), ws.numel(), st.data_ptr(), sp())
    torch.cuda.synchronize()
    for b in range(B):
        assert float((out[b] - ctx[b * S + k_len[b] - 1]).abs().max()) <= 2.0**-17 * 6
    assert int(st) == 0
