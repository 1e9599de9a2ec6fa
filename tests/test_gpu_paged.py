"""GPU: attention of one new token over the paged cache against the definition in 64 bits, and the cache's operators
used together as a decoder uses them."""
import math

import numpy as np
import pytest

from kv_model import BAD_REQUEST, describe, ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def kx(libkx):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from kernix_b200 import kx_abi
    return kx_abi


def sp():
    return torch.cuda.current_stream().cuda_stream


def visible(length, window, sinks):
    j = np.arange(length)
    return (window <= 0) | (j > length - 1 - window) | (j < sinks)


def exact(q, k, v, scale):
    """q (group, dk), k (keys, dk), v (keys, dv), all visible, in 64 bits -> (group, dv) and its tolerance.

    The scores come from products of operands that keep at least 21 bits (2^-21 of sum |q||k| each side of a product's
    two rounded parts) summed in at most 24 tensor-core steps that may truncate (24 x 2^-24): under 2^-19 of
    sum |q||k| in all. A weight p is off by the factor exp(+-that), twice (weight and sum). Weights and their parts
    (2^-22), the exponential (2^-22), the fp32 sums over a warp's steps and the joins add less than 2^-18 of max |v|."""
    if k.shape[0] == 0:
        return np.zeros((q.shape[0], v.shape[1])), np.zeros((q.shape[0], 1))
    s = scale * q @ k.T
    p = np.exp(s - s.max(1, keepdims=True))
    size = abs(scale) * (np.abs(q) @ np.abs(k).T).max(1, keepdims=True)
    tol = (np.expm1(2 * size * 2.0**-19) + 2.0**-18) * np.abs(v).max() + 1e-30
    return p @ v / p.sum(1, keepdims=True), tol


class Case:
    """A cache whose pools are NaN everywhere but at the keys that the tokens see (or `fill` where they do not)."""

    def __init__(self, lens, heads, group, dk, dv, page, dtype, window=0, sinks=0, layers=1, layer=0, fill=float("nan"), seed=0,
                 big=1.0, spare=2):
        rng = np.random.default_rng(seed)
        self.lens, self.heads, self.G, self.dk, self.dv, self.page = lens, heads, group, dk, dv, page
        self.window, self.sinks, self.layer, self.dtype = window, sinks, layer, dtype
        n = len(lens)
        need = [-(-x // page) for x in lens]
        n_pages, max_pages = sum(need) + spare, max(1, max(need))
        g = torch.Generator().manual_seed(seed)
        self.k = torch.full((layers, n_pages, heads, page, dk), fill, dtype=DTYPES[dtype])
        self.v = torch.full((layers, n_pages, heads, page, dv), fill, dtype=DTYPES[dtype])
        ids = rng.permutation(n_pages).astype(np.int32)
        table = np.full((n, max_pages), -1, np.int32)
        self.host = []
        at = 0
        for s, length in enumerate(lens):
            table[s, : need[s]] = ids[at:at + need[s]]
            at += need[s]
            j = np.flatnonzero(visible(length, window, sinks))
            kk = (torch.randn(len(j), heads, dk, generator=g) * big).to(DTYPES[dtype])
            vv = torch.randn(len(j), heads, dv, generator=g).to(DTYPES[dtype])
            p = torch.from_numpy(table[s, j // page].astype(np.int64)) if len(j) else torch.zeros(0, dtype=torch.int64)
            slot = torch.from_numpy(j % page)
            self.k[layer][p, :, slot] = kk
            self.v[layer][p, :, slot] = vv
            self.host.append((kk.double().numpy(), vv.double().numpy()))
        self.q = torch.randn(n, heads * group * dk, generator=g) * big
        self.table, self.d_lens = torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.refs = torch.ones(n_pages, dtype=torch.int32, device="cuda")
        self.k, self.v = self.k.cuda(), self.v.cuda()
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def cache(self, kx):
        return describe(kx, self.k, self.v, self.table, self.d_lens, self.refs, self.dtype)

    def run(self, kx, q=None, seqs=None, scale=0.0, ctx=None, ws=None):
        c, H = self.cache(kx), self.heads * self.G
        q = (self.q if q is None else q).cuda()
        n = q.shape[0]
        if ctx is None:
            ctx = torch.full((n, H * self.dv), 7.0, device="cuda")
        self.ws = torch.empty(kx.lib().kx_attention_paged_ws(ref(c), H, n), dtype=torch.uint8, device="cuda") if ws is None else ws
        kx.call("kx_attention_paged", ref(c), self.layer, q.data_ptr(), q.stride(0), H, None if seqs is None else seqs.data_ptr(), n,
                self.window, self.sinks, scale, ctx.data_ptr(), ctx.stride(0), self.ws.data_ptr(), self.ws.numel(),
                self.status.data_ptr(), sp())
        torch.cuda.synchronize()
        return ctx

    def want(self, row, slot, q=None, scale=0.0):
        q = (self.q if q is None else q)[row].double().numpy().reshape(self.heads, self.G, self.dk)
        k, v = self.host[slot]
        outs = [exact(q[h], k[:, h], v[:, h], scale or 1 / math.sqrt(self.dk)) for h in range(self.heads)]
        return np.concatenate([o for o, _ in outs]), np.concatenate([np.broadcast_to(t, o.shape) for o, t in outs])

    def check(self, ctx, rows=None, q=None, scale=0.0):
        got = ctx.double().cpu().numpy()
        for row, slot in rows or [(i, i) for i in range(len(self.lens))]:
            want, tol = self.want(row, slot, q, scale)
            g = got[row, : self.heads * self.G * self.dv].reshape(want.shape)
            err = np.abs(g - want)
            assert np.all(err <= tol), (row, slot, float(err.max()), float(np.max(tol)))


SHAPES = [  # heads, group, dk, dv, page, window, sinks
    (1, 1, 64, 64, 16, 0, 0), (2, 4, 128, 128, 16, 0, 0), (3, 3, 72, 80, 8, 37, 4), (1, 8, 8, 8, 1, 5, 0),
    (2, 9, 128, 64, 32, 0, 3), (4, 2, 96, 128, 64, 100, 30), (1, 20, 40, 120, 128, 1, 1), (8, 1, 64, 64, 4, 129, 200)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_ragged_rows(kx, dtype, shape):
    heads, group, dk, dv, page, window, sinks = shape
    c = Case([1, 0, 2, 7, 8, 9, 15, 16, 17, 63, 64, 65, 127, 128, 131, 500, 1000, 0, 3], heads, group, dk, dv, page, dtype, window, sinks)
    ctx = c.run(kx)
    c.check(ctx)
    assert int(c.status) == 0 and not ctx[1].any() and not ctx[17].any()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens,window,sinks", [([20000], 0, 0), ([1, 30011, 5], 0, 0), ([40000, 39999], 20001, 9), ([257] * 300, 0, 0),
                                               ([30, 0] * 100 + [9000, 1], 0, 0)])
def test_long_and_many_rows(kx, dtype, lens, window, sinks):
    """heads split over many CTAs and joined; ranges that cover several rows"""
    c = Case(lens, 2, 4, 128, 128, 32, dtype, window, sinks, seed=3)
    first = c.run(kx)
    c.check(first)
    again = c.run(kx)
    assert torch.equal(first, again)


@pytest.mark.parametrize("window,sinks", [(2**31 - 1, 2**31 - 1), (2**31 - 1, 0), (3, 2**31 - 1)])
def test_largest_windows(kx, window, sinks):
    c = Case([700, 1, 0, 16], 2, 2, 64, 64, 16, "bf16", window, sinks)
    c.check(c.run(kx))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_infinities_in_masked_places_and_layers(kx, dtype):
    c = Case([100, 31, 64], 2, 2, 64, 64, 16, dtype, window=10, sinks=2, layers=3, layer=2, fill=float("inf"))
    c.check(c.run(kx))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("big", [1e-6, 30.0])
def test_small_and_large_values(kx, dtype, big):
    """nearly equal weights, and weights that one key takes almost whole"""
    c = Case([300, 17], 2, 4, 64, 128, 16, dtype, big=big, seed=4)
    c.check(c.run(kx))


def test_scale_and_row_strides(kx):
    c = Case([50, 3, 200], 2, 3, 64, 72, 8, "f16")
    q = torch.full((3, 2 * 3 * 64 + 5), float("nan"))
    q[:, :384] = c.q
    ctx = torch.full((3, 2 * 3 * 72 + 3), 7.0, device="cuda")
    c.run(kx, q=q, ctx=ctx, scale=-0.3)
    c.check(ctx, scale=-0.3, q=c.q)
    assert bool((ctx[:, 432:] == 7).all())


def test_rows_name_their_slots(kx):
    """several rows of one slot, rows that are left alone, slots out of range"""
    c = Case([50, 0, 200], 2, 3, 64, 64, 8, "bf16")
    seqs = torch.tensor([2, -1, 0, 2, 1, 3, -5, 2**31 - 1], dtype=torch.int32, device="cuda")
    q = torch.randn(8, 384, generator=torch.Generator().manual_seed(8))
    ctx = c.run(kx, q=q, seqs=seqs)
    c.check(ctx, rows=[(0, 2), (2, 0), (3, 2), (4, 1)], q=q)
    assert bool((ctx[[1, 6]] == 7).all()) and bool(ctx[[5, 7]].isnan().all()) and int(c.status) == BAD_REQUEST


def test_rows_name_their_slots_in_a_split_launch(kx):
    c = Case([3000, 0, 700], 2, 3, 64, 64, 8, "bf16")
    seqs = torch.tensor([-1, 2, -1, 0, 5, 1, 2, -9, -1], dtype=torch.int32, device="cuda")
    q = torch.randn(9, 384, generator=torch.Generator().manual_seed(8))
    ctx = c.run(kx, q=q, seqs=seqs)
    c.check(ctx, rows=[(1, 2), (3, 0), (5, 1), (6, 2)], q=q)
    assert bool((ctx[[0, 2, 7, 8]] == 7).all()) and bool(ctx[4].isnan().all()) and int(c.status) == BAD_REQUEST
    ctx = c.run(kx, q=q, seqs=torch.full_like(seqs, -1))
    assert bool((ctx == 7).all())


@pytest.mark.parametrize("page", [2, 1024])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_smallest_and_largest_pages(kx, page, dtype):
    c = Case([1, 1500, 1024, 1025, 2], 2, 2, 32, 40, page, dtype, window=300, sinks=5)
    c.check(c.run(kx))


def test_layers_inside_a_page(kx):
    c = Case([90, 33], 2, 4, 64, 48, 16, "f16", layers=3, layer=1)
    for x in ("k", "v"):
        setattr(c, x, getattr(c, x).transpose(0, 1).contiguous().transpose(0, 1))
    c.check(c.run(kx))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_split_launch_captured(kx, dtype):
    """replays follow the lengths, which are device memory"""
    c = Case([6000, 100, 2000], 2, 4, 64, 64, 16, dtype, seed=6)
    c.run(kx)
    cc, qd, ctx = c.cache(kx), c.q.cuda(), torch.zeros(3, 512, device="cuda")
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        kx.call("kx_attention_paged", ref(cc), 0, qd.data_ptr(), 512, 8, None, 3, 0, 0, 0.0, ctx.data_ptr(), 512, c.ws.data_ptr(),
                c.ws.numel(), None, torch.cuda.current_stream().cuda_stream)
    for lens in ([6000, 100, 2000], [5, 99, 1999], [0, 0, 1], [5999, 1, 0]):
        c.d_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        short = Case.__new__(Case)
        short.__dict__.update(c.__dict__)
        short.lens, short.host = lens, [(k[:n], v[:n]) for (k, v), n in zip(c.host, lens)]
        short.check(ctx)


@pytest.mark.parametrize("long", [False, True])
def test_bad_pages_and_lengths_give_nan_rows(kx, long):
    n = 5000 if long else 60
    c = Case([n, n, n, n], 2, 2, 64, 64, 16, "f16", window=40 if not long else 3000)
    c.table[0, n // 16] = -1                    # the page of the last tokens
    c.table[1, 0] = 10**9 if long else -1       # behind the window: not read
    if not long:
        c.table[1, 0] = 10**9
    c.d_lens[2] = -3
    c.d_lens[3] = c.table.shape[1] * 16 + 1
    ctx = c.run(kx)
    assert bool(ctx[[0, 2, 3]].isnan().all()) and int(c.status) == BAD_REQUEST
    c.check(ctx, rows=[(1, 1)])


def test_nan_in_a_seen_place_shows(kx):
    c = Case([70, 70], 1, 2, 64, 64, 16, "bf16")
    p = int(c.table[1, 69 // 16])
    c.v[0, p, 0, 69 % 16, 3] = float("nan")
    ctx = c.run(kx)
    c.check(ctx, rows=[(0, 0)])
    bad = ctx[1].view(2, 64).isnan()
    assert bool(bad[:, 3].all())


def test_offsets_past_32_bits(kx):
    """pages two gigabytes apart"""
    gap, page, d = 1 << 30, 16, 64
    pool = torch.empty(4 * gap, dtype=torch.bfloat16, device="cuda")
    c = Case([60], 1, 4, d, d, page, "bf16")
    for x, off in (("k", 0), ("v", 1024)):
        far = torch.as_strided(pool, (1, 4, 1, page, d), (8, gap, page * d, d, 1), off)
        far.copy_(getattr(c, x)[:, :4])
        setattr(c, x, far)
    c.table = c.table.clone()
    keep = c.table[0].tolist()
    if max(keep) > 3:                           # the pages in use, renumbered
        src = Case([60], 1, 4, d, d, page, "bf16")
        for new, old in enumerate(keep):
            c.k[0, new].copy_(src.k[0, old])
            c.v[0, new].copy_(src.v[0, old])
        c.table = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    c.check(c.run(kx))


def test_two_streams_with_workspaces_of_their_own(kx):
    cases = [Case([9000, 100], 2, 4, 64, 64, 16, "f16", seed=i) for i in range(2)]
    want = [c.run(kx).clone() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for c, s in zip(cases, streams):
        qd, ctx, ws = c.q.cuda(), torch.zeros_like(want[0]), torch.empty_like(c.ws)
        got.append((qd, ctx, ws))
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s, (qd, ctx, ws) in zip(cases, streams, got):
            cc = c.cache(kx)
            kx.call("kx_attention_paged", ref(cc), 0, qd.data_ptr(), qd.stride(0), 8, None, 2, 0, 0, 0.0, ctx.data_ptr(), ctx.stride(0),
                    ws.data_ptr(), ws.numel(), None, s.cuda_stream)
    torch.cuda.synchronize()
    for w, (_, ctx, _) in zip(want, got):
        assert torch.equal(w, ctx)


def test_default_stream(kx):
    c = Case([3000, 5], 2, 4, 64, 64, 16, "f16", seed=2)
    cc, qd, ctx = c.cache(kx), c.q.cuda(), torch.zeros(2, 512, device="cuda")
    ws = torch.empty(kx.lib().kx_attention_paged_ws(ref(cc), 8, 2), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    kx.call("kx_attention_paged", ref(cc), 0, qd.data_ptr(), qd.stride(0), 8, None, 2, 0, 0, 0.0, ctx.data_ptr(), ctx.stride(0),
            ws.data_ptr(), ws.numel(), None, None)
    torch.cuda.synchronize()
    c.check(ctx)


@pytest.mark.parametrize("dtype,window,sinks", [("f32", 0, 0), ("f16", 24, 3), ("bf16", 0, 0)])
def test_a_decoder_over_the_cache(kx, dtype, window, sinks):
    """Prompts, token steps captured in a graph, forks, releases and compaction in between: every step's attention
    against the definition over each sequence's own history."""
    rng = np.random.default_rng(7)
    n, page, heads, G, dk, dv, layers, dt = 6, 8, 2, 3, 32, 40, 2, DTYPES[dtype]
    n_pages, max_pages = 90, 16
    k = torch.full((layers, n_pages, heads, page, dk), float("nan"), dtype=dt, device="cuda")
    v = torch.full((layers, n_pages, heads, page, dv), float("nan"), dtype=dt, device="cuda")
    table = torch.full((n, max_pages), -1, dtype=torch.int32, device="cuda")
    lens, refs = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    c = describe(kx, k, v, table, lens, refs, dtype)
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    status, granted = ints([0]), ints([0] * n)
    ws = torch.empty(max(kx.lib().kx_kv_ws(ref(c)), kx.lib().kx_attention_paged_ws(ref(c), heads * G, n)), dtype=torch.uint8, device="cuda")
    w, st = (ws.data_ptr(), ws.numel()), status.data_ptr()
    history = [[([], []) for _ in range(layers)] for _ in range(n)]

    def stored(rows, d):
        return rows.to(dt).double().view(-1, heads, d).numpy()

    def prompt(want, rows):
        kx.call("kx_kv_extend", ref(c), ints(want).data_ptr(), granted.data_ptr(), *w, st, sp())
        for layer in range(layers):
            kr, vr = (torch.randn(n * rows, heads * d, generator=g) for d in (dk, dv))
            kd, vd = kr.cuda(), vr.cuda()
            kx.call("kx_kv_append", ref(c), layer, kd.data_ptr(), heads * dk, vd.data_ptr(), heads * dv, granted.data_ptr(), rows, st, sp())
            for s, cnt in enumerate(want):
                history[s][layer][0].extend(stored(kr, dk)[s * rows:s * rows + cnt])
                history[s][layer][1].extend(stored(vr, dv)[s * rows:s * rows + cnt])

    g = torch.Generator().manual_seed(11)
    prompt([13, 40, 1, 8, 0, 0], 40)
    a, b = ints([0, 1]), ints([4, 5])
    kx.call("kx_kv_fork", ref(c), a.data_ptr(), b.data_ptr(), 2, *w, st, sp())
    for s, t in ((0, 4), (1, 5)):
        history[t] = [([*x], [*y]) for x, y in history[s]]

    one = ints([1] * n)
    qd, kd, vd = (torch.zeros(layers, n, heads * d, device="cuda") for d in (G * dk, dk, dv))
    ctx = torch.zeros(layers, n, heads * G * dv, device="cuda")

    def step(stream):
        kx.call("kx_kv_extend", ref(c), one.data_ptr(), granted.data_ptr(), *w, st, stream)
        for layer in range(layers):
            kx.call("kx_kv_append", ref(c), layer, kd[layer].data_ptr(), heads * dk, vd[layer].data_ptr(), heads * dv,
                    granted.data_ptr(), 1, st, stream)
            kx.call("kx_attention_paged", ref(c), layer, qd[layer].data_ptr(), heads * G * dk, heads * G, None, n, window, sinks, 0.0,
                    ctx[layer].data_ptr(), heads * G * dv, *w, st, stream)

    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        step(torch.cuda.current_stream().cuda_stream)
    live = ints([0])
    for i in range(25):
        qr, kr, vr = (torch.randn(layers, n, heads * d, generator=g) for d in (G * dk, dk, dv))
        qd.copy_(qr), kd.copy_(kr), vd.copy_(vr)
        graph.replay()
        torch.cuda.synchronize()
        for layer in range(layers):
            ks, vs = stored(kr[layer], dk), stored(vr[layer], dv)
            for s in range(n):
                history[s][layer][0].append(ks[s])
                history[s][layer][1].append(vs[s])
                seen = visible(len(history[s][layer][0]), window, sinks)
                kk, vv = np.array(history[s][layer][0])[seen], np.array(history[s][layer][1])[seen]
                qs = qr[layer, s].double().numpy().reshape(heads, G, dk)
                got = ctx[layer, s].double().cpu().numpy().reshape(heads, G, dv)
                for h in range(heads):
                    want, tol = exact(qs[h], kk[:, h], vv[:, h], 1 / math.sqrt(dk))
                    assert np.all(np.abs(got[h] - want) <= tol), (i, layer, s, h)
        if i % 6 == 5:              # a sequence ends, another one's copy takes its slot, the pool is compacted
            s, t = rng.permutation(n)[:2].tolist()
            a, b = ints([s]), ints([t])
            kx.call("kx_kv_free", ref(c), a.data_ptr(), 1, st, sp())
            kx.call("kx_kv_fork", ref(c), b.data_ptr(), a.data_ptr(), 1, *w, st, sp())
            history[s] = [([*x], [*y]) for x, y in history[t]]
            kx.call("kx_kv_compact", ref(c), live.data_ptr(), *w, sp())
            assert int(live) == int((refs > 0).sum()) == int((refs[: int(live)] > 0).sum())
    assert int(status) == 0
