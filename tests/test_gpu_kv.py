"""GPU: the pages of a key-value cache against a sequential model, bit for bit (tests/kv_model.py)."""
import numpy as np
import pytest

from kv_model import BAD_REQUEST, NO_PAGES, Pages, describe, ref

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


class Pair:
    """A cache on the device and its model, checked against each other after every operation."""

    def __init__(self, kx, n_seqs, max_pages, n_pages, page, heads=2, dk=8, dv=16, dtype="f16", layers=1, inner=False, seed=0):
        self.kx, self.page, self.heads, self.dk, self.dv, self.layers, self.dt = kx, page, heads, dk, dv, layers, DTYPES[dtype]
        self.m = Pages(n_seqs, max_pages, n_pages, page)
        g = torch.Generator().manual_seed(seed)
        pools = []
        for d in (dk, dv):
            # inner: the layers of a page lie one after another, with a gap behind them
            shape = (n_pages, layers + 1, heads, page, d) if inner else (layers, n_pages + 1, heads, page, d)
            t = torch.randn(shape, generator=g).to(self.dt).cuda()
            pools.append(t[:, :layers].transpose(0, 1) if inner else t[:, :n_pages])
        self.k, self.v = pools
        self.m.pools = [self.bits(t) for t in pools]
        self.table, self.lens, self.refs = (torch.from_numpy(a.copy()).cuda() for a in (self.m.table, self.m.lens, self.m.refs))
        self.c = describe(kx, self.k, self.v, self.table, self.lens, self.refs, dtype)
        self.ws = torch.randint(0, 255, (kx.lib().kx_kv_ws(ref(self.c)),), dtype=torch.uint8, device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    @staticmethod
    def bits(t):
        return t.contiguous().view(torch.int32 if t.dtype == torch.float32 else torch.int16).cpu().numpy()

    def w(self):
        return self.ws.data_ptr(), self.ws.numel()

    def ints(self, a):
        return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()

    def extend(self, want, in_place=False):
        want = np.pad(np.asarray(want, np.int32), (0, len(self.m.lens) - len(want)))  # a word for every slot
        d = self.ints(want)
        granted = d if in_place else torch.full_like(d, 77)
        self.kx.call("kx_kv_extend", ref(self.c), d.data_ptr(), granted.data_ptr(), *self.w(), self.status.data_ptr(), sp())
        assert np.array_equal(granted.cpu().numpy(), self.m.extend(want))
        return granted

    def free(self, seqs):
        d = self.ints(seqs)
        self.kx.call("kx_kv_free", ref(self.c), d.data_ptr(), len(seqs), self.status.data_ptr(), sp())
        self.m.free(seqs)

    def fork(self, src, dst):
        a, b = self.ints(src), self.ints(dst)
        self.kx.call("kx_kv_fork", ref(self.c), a.data_ptr(), b.data_ptr(), len(src), *self.w(), self.status.data_ptr(), sp())
        self.m.fork(np.asarray(src), np.asarray(dst))

    def compact(self):
        n = torch.full((1,), -1, dtype=torch.int32, device="cuda")
        self.kx.call("kx_kv_compact", ref(self.c), n.data_ptr(), *self.w(), sp())
        assert int(n) == self.m.compact()

    def append(self, layer, counts, rows, seed=0, ldk=None, ldv=None, shift=0):
        """the model takes torch's rounding to the cache's type"""
        n = len(counts)
        assert n == len(self.m.lens)
        g = torch.Generator().manual_seed(seed)
        src = []
        for d, ld in ((self.dk, ldk), (self.dv, ldv)):
            w = self.heads * d
            ld = ld or w
            t = torch.full((n * rows * ld + shift,), float("nan"))
            view = t[shift:].view(n * rows, ld)
            view[:, :w] = torch.randn(n * rows, w, generator=g) * 3
            src.append((view, t.cuda(), ld))
        d = self.ints(counts)
        (kh, kd, lk), (vh, vd, lv) = src
        self.kx.call("kx_kv_append", ref(self.c), layer, kd.data_ptr() + 4 * shift, lk, vd.data_ptr() + 4 * shift, lv,
                     d.data_ptr(), rows, self.status.data_ptr(), sp())
        for pool, host, dim in zip(self.m.pools, (kh, vh), (self.dk, self.dv)):
            as_stored = self.bits(host[:, : self.heads * dim].to(self.dt)).reshape(n, rows, self.heads, dim)
            for s, c in enumerate(np.asarray(counts).tolist()):
                if c <= 0:
                    continue
                if c > rows or c > self.m.lens[s]:
                    self.m.status |= BAD_REQUEST
                    continue
                for i in range(c):
                    pos = int(self.m.lens[s]) - c + i
                    pool[layer, self.m.table[s, pos // self.page], :, pos % self.page] = as_stored[s, i]

    def check(self):
        torch.cuda.synchronize()
        assert np.array_equal(self.table.cpu().numpy(), self.m.table)
        assert np.array_equal(self.lens.cpu().numpy(), self.m.lens)
        assert np.array_equal(self.refs.cpu().numpy(), self.m.refs)
        assert int(self.status) == self.m.status
        for t, want in zip((self.k, self.v), self.m.pools):
            wrong = np.argwhere(self.bits(t) != want)
            assert len(wrong) == 0, wrong[:4].tolist()


@pytest.mark.parametrize("n_seqs,max_pages,n_pages,page", [(1, 1, 1, 1), (3, 7, 12, 4), (40, 9, 130, 8), (1100, 5, 2600, 2),
                                                           (70, 80, 4099, 16)])
def test_extend_takes_the_lowest_free_pages_in_order(kx, n_seqs, max_pages, n_pages, page):
    rng = np.random.default_rng(n_seqs)
    p = Pair(kx, n_seqs, max_pages, n_pages, page)
    for i in range(4):
        p.extend(rng.integers(-2, max_pages * page // 2 + 2, n_seqs), in_place=i == 2)
        p.check()
        p.free(rng.integers(0, n_seqs, n_seqs // 2).tolist())
        p.check()


def test_extend_refuses_what_does_not_fit(kx):
    p = Pair(kx, 4, 4, 6, 8)
    p.extend([8, 33, 9, 0])        # the second is longer than a table row: left out, the others served
    p.check()
    assert p.m.status == NO_PAGES
    p.extend([1, 32, 7, 5])        # 1 + 4 pages where 3 are free: the second and the fourth are refused, not the third
    assert p.m.lens.tolist() == [9, 0, 16, 0]
    p.check()
    p.extend([2**31 - 1] * 4)      # sums past 32 bits
    p.check()


def test_bad_lengths_are_left_alone(kx):
    p = Pair(kx, 3, 4, 12, 4)
    p.extend([4, 4, 4])
    for bad in (-1, 17, 2**31 - 1):
        p.lens[1] = bad
        want, granted = p.ints([3, 3, 3]), p.ints([9, 9, 9])
        p.status.zero_()
        p.kx.call("kx_kv_extend", ref(p.c), want.data_ptr(), granted.data_ptr(), *p.w(), p.status.data_ptr(), sp())
        assert granted.tolist()[1] == 0 and int(p.lens[1]) == bad and int(p.status) & BAD_REQUEST
        src, dst = p.ints([1]), p.ints([2])
        p.kx.call("kx_kv_fork", ref(p.c), src.data_ptr(), dst.data_ptr(), 1, *p.w(), p.status.data_ptr(), sp())
        before = p.bits(p.k)
        rows = torch.ones(3, 64, device="cuda")
        p.status.zero_()
        p.kx.call("kx_kv_append", ref(p.c), 0, rows.data_ptr(), 64, rows.data_ptr(), 64, p.ints([0, 1, 0]).data_ptr(), 1,
                  p.status.data_ptr(), sp())
        assert int(p.status) == BAD_REQUEST and np.array_equal(before, p.bits(p.k))


def test_free_twice_and_out_of_range(kx):
    p = Pair(kx, 5, 600, 700, 1)
    p.extend([600, 10, 20, 5, 1])
    p.fork([1, 1], [0, 0])         # slot 0 is not empty: both refused
    p.free([3, -1, 3, 5, 0, 0, -7])
    p.check()
    assert p.m.status == BAD_REQUEST and int(p.m.refs.sum()) == 31


@pytest.mark.parametrize("dtype,layers,inner", [("f16", 1, False), ("bf16", 3, True), ("f32", 2, False), ("f32", 2, True)])
@pytest.mark.parametrize("rows,counts", [(1, [1, 0, 1, 1]), (5, [5, 0, -3, 3]), (37, [37, 1, 20, 0])])
def test_append(kx, dtype, layers, inner, rows, counts):
    p = Pair(kx, 4, 9, 30, 8, heads=3, dk=24, dv=8, dtype=dtype, layers=layers, inner=inner)
    p.extend([13, 7, 8, 1])
    p.extend(counts)
    for layer in range(layers):
        p.append(layer, counts, rows, seed=layer)
        p.append(layer, counts, rows, seed=9 + layer, ldk=75, ldv=30, shift=1)  # rows of odd pitch and alignment
    p.check()
    assert p.m.status == 0


def test_append_refuses_counts_and_pages_out_of_range(kx):
    p = Pair(kx, 3, 4, 12, 4)
    p.extend([6, 6, 6])
    p.append(0, [2, 3, 7], 2)      # more rows than given; more than the slot holds
    p.check()
    assert p.m.status == BAD_REQUEST
    for bad in (-1, 12, 2**31 - 1):
        p.table[0, 1] = bad
        before = p.bits(p.k)
        p.status.zero_()
        rows = torch.ones(3, 64, device="cuda")
        p.kx.call("kx_kv_append", ref(p.c), 0, rows.data_ptr(), 64, rows.data_ptr(), 64, p.ints([1, 0, 0]).data_ptr(), 1,
                  p.status.data_ptr(), sp())
        assert int(p.status) == BAD_REQUEST and np.array_equal(before, p.bits(p.k))


@pytest.mark.parametrize("dtype,layers,inner,page", [("f16", 1, False, 4), ("bf16", 3, True, 64), ("f32", 2, False, 16)])
def test_fork_shares_full_pages_and_copies_the_tail(kx, dtype, layers, inner, page):
    p = Pair(kx, 12, 6, 40, page, heads=3, dk=40, dv=136, dtype=dtype, layers=layers, inner=inner)
    p.extend([2 * page, 3 * page + 1, 1, 0, page - 1])
    p.fork([0, 1, 1, 4, 3, 2], [5, 6, 11, 7, 8, -1])
    p.check()
    p.extend([1] * 12)             # children and parents grow apart
    p.append(layers - 1, [1 if s else 0 for s in p.m.lens.tolist()], 1)
    p.check()
    p.free([0, 1])
    p.check()
    p.fork([5, 6, 6, 6], [0, 1, 1, 6])     # a slot named twice, a slot onto itself
    p.check()
    assert p.m.status & BAD_REQUEST


def test_fork_without_pages(kx):
    p = Pair(kx, 8, 4, 6, 4)
    p.extend([5, 4, 3])
    p.fork([0, 2, 1, 0, 2], [3, 4, 5, 6, 7])   # two free pages: the third and fourth copies are refused, the shared one is not
    p.check()
    assert p.m.lens.tolist() == [5, 4, 3, 5, 3, 4, 0, 0] and p.m.status == NO_PAGES
    p.fork([9, -1, 0], [6, 7, 8])              # slots out of range
    p.check()


@pytest.mark.parametrize("n_pages,layers,inner,dtype", [(1, 1, False, "f16"), (130, 2, True, "bf16"), (5000, 1, False, "f32"),
                                                        (4096, 2, False, "f16")])
def test_compact(kx, n_pages, layers, inner, dtype):
    rng = np.random.default_rng(n_pages)
    p = Pair(kx, 50, 64, n_pages, 4, heads=1, dk=16, dv=8, dtype=dtype, layers=layers, inner=inner)
    p.compact()
    p.check()                      # an empty pool
    for _ in range(3):
        p.extend(rng.integers(0, max(2, n_pages // 5), 50))
        p.fork([0, 1, 2], [47, 48, 49])
        p.free(rng.integers(0, 50, 30).tolist())
        p.compact()
        p.check()
        p.compact()                # nothing left to move
        p.check()


def test_more_pages_slots_and_pairs_than_one_pass_takes(kx):
    rng = np.random.default_rng(8)
    p = Pair(kx, 2600, 40, 70001, 4, heads=1, dk=8, dv=8)
    p.extend(rng.integers(0, 120, 2600))
    p.check()
    ended = rng.permutation(2600)[:1250]
    p.free(ended.tolist())
    p.check()
    parents = np.setdiff1d(np.arange(2600), ended)
    p.fork(rng.choice(parents, 1200), ended[:1200])
    p.check()
    p.free(rng.permutation(2600)[:900].tolist())
    p.compact()
    p.check()
    p.extend(rng.integers(0, 20, 2600))
    p.check()


def test_without_a_status_word_and_on_the_default_stream(kx):
    p = Pair(kx, 4, 3, 5, 4)
    want, granted = p.ints([9, 9, 9, 1]), p.ints([0] * 4)
    seqs, src, dst = p.ints([0, 9, 0]), p.ints([1, 1]), p.ints([0, 1])
    torch.cuda.synchronize()
    kx.call("kx_kv_extend", ref(p.c), want.data_ptr(), granted.data_ptr(), *p.w(), None, None)
    kx.call("kx_kv_free", ref(p.c), seqs.data_ptr(), 3, None, None)
    kx.call("kx_kv_fork", ref(p.c), src.data_ptr(), dst.data_ptr(), 2, *p.w(), None, None)
    assert np.array_equal(p.m.extend(want.cpu().numpy()), granted.cpu().numpy())
    p.m.free([0, 9, 0])
    p.m.fork(np.array([1, 1]), np.array([0, 1]))
    p.m.status = 0
    p.check()


def test_turnover_captured_in_a_graph(kx):
    """a step of free, extend, append and fork, captured once and replayed on changing requests"""
    p = Pair(kx, 16, 8, 90, 4, heads=2, dk=16, dv=16, dtype="bf16")
    rng = np.random.default_rng(5)
    p.extend(rng.integers(1, 20, 16))
    seqs, want, src, dst = p.ints([0] * 4), p.ints([0] * 16), p.ints([0] * 2), p.ints([0] * 2)
    granted, rows = torch.zeros_like(want), torch.zeros(16 * 9, 32, device="cuda")

    def step(stream):
        st = p.status.data_ptr()
        kx.call("kx_kv_free", ref(p.c), seqs.data_ptr(), 4, st, stream)
        kx.call("kx_kv_extend", ref(p.c), want.data_ptr(), granted.data_ptr(), *p.w(), st, stream)
        kx.call("kx_kv_append", ref(p.c), 0, rows.data_ptr(), 32, rows.data_ptr(), 32, granted.data_ptr(), 9, st, stream)
        kx.call("kx_kv_fork", ref(p.c), src.data_ptr(), dst.data_ptr(), 2, *p.w(), st, stream)

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        step(torch.cuda.current_stream().cuda_stream)
    for i in range(6):
        ended = rng.permutation(16)[:4]
        w = rng.integers(0, 10, 16)
        w[ended[2:]] = 0           # two of the ended slots take children instead
        rest = np.setdiff1d(np.arange(16), ended)
        seqs.copy_(p.ints(ended)), want.copy_(p.ints(w)), src.copy_(p.ints(rest[:2])), dst.copy_(p.ints(ended[2:]))
        x = torch.randn(16 * 9, 32, generator=torch.Generator().manual_seed(i))
        rows.copy_(x)
        graph.replay()
        p.m.free(ended.tolist())
        got = p.m.extend(w.astype(np.int32))
        assert np.array_equal(granted.cpu().numpy(), got)
        stored = Pair.bits(x.to(torch.bfloat16)).reshape(16, 9, 2, 16)
        for s in range(16):
            for j in range(got[s]):
                pos = int(p.m.lens[s]) - int(got[s]) + j
                for pool in p.m.pools:
                    pool[0, p.m.table[s, pos // 4], :, pos % 4] = stored[s, j]
        p.m.fork(rest[:2], ended[2:])
        p.check()
