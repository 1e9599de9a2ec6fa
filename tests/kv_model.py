"""The pages of a key-value cache as a plain sequential model (numpy), and a device copy of one for the tests."""
import ctypes

import numpy as np

NO_PAGES, BAD_REQUEST = 2, 4
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
TYPE_IDS = {"f32": 0, "f16": 1, "bf16": 2}


class Pages:
    """table, lens, refs and per-layer page contents (any numpy arrays whose first axis is the page)."""

    def __init__(self, n_seqs, max_pages, n_pages, page):
        self.page, self.n_pages, self.max_pages = page, n_pages, max_pages
        self.table = np.full((n_seqs, max_pages), -1, np.int32)
        self.lens, self.refs = np.zeros(n_seqs, np.int32), np.zeros(n_pages, np.int32)
        self.pools = []  # arrays (layers, n_pages, ...)
        self.status = 0

    def pages(self, tokens):
        return -(-int(tokens) // self.page)

    def free_ids(self):
        return np.flatnonzero(self.refs == 0).tolist()

    def extend(self, want):
        ids, granted, asked, n_free = self.free_ids(), np.zeros_like(want), 0, int((self.refs == 0).sum())
        for s, w in enumerate(want.tolist()):
            if w <= 0:
                continue
            if int(self.lens[s]) + w > self.max_pages * self.page:
                self.status |= NO_PAGES
                continue
            have, need = self.pages(self.lens[s]), self.pages(self.lens[s] + w) - self.pages(self.lens[s])
            asked += need
            if need and asked > n_free:
                self.status |= NO_PAGES
                continue
            got, ids = ids[:need], ids[need:]
            self.table[s, have:have + need] = got
            self.refs[got] = 1
            self.lens[s] += w
            granted[s] = w
        return granted

    def free(self, seqs):
        for s in seqs:
            if s < 0:
                continue
            if s >= len(self.lens):
                self.status |= BAD_REQUEST
                continue
            for p in self.table[s]:
                if 0 <= p < self.n_pages:
                    self.refs[p] -= 1
            self.table[s], self.lens[s] = -1, 0

    def fork(self, src, dst):
        lens0, ids, n_free, asked, seen = self.lens.copy(), self.free_ids(), int((self.refs == 0).sum()), 0, set()
        n = len(lens0)
        for a, b in zip(src.tolist(), dst.tolist()):
            if b < 0:
                continue
            first = b not in seen
            seen.add(b)
            if not (0 <= a < n and b < n and a != b and first and lens0[b] == 0):
                self.status |= BAD_REQUEST
                continue
            full, part = lens0[a] // self.page, lens0[a] % self.page != 0
            asked += part
            if part and asked > n_free:
                self.status |= NO_PAGES
                continue
            row = np.full(self.max_pages, -1, np.int32)
            row[:full] = self.table[a, :full]
            np.add.at(self.refs, row[:full], 1)
            if part:
                row[full] = ids.pop(0)
                self.refs[row[full]] = 1
                for pool in self.pools:
                    pool[:, row[full]] = pool[:, self.table[a, full]]
            self.table[b], self.lens[b] = row, lens0[a]

    def compact(self):
        n_live = int((self.refs > 0).sum())
        holes, late = np.flatnonzero(self.refs[:n_live] == 0), n_live + np.flatnonzero(self.refs[n_live:] > 0)
        to = np.arange(self.n_pages, dtype=np.int32)
        to[late] = holes
        for pool in self.pools:
            pool[:, holes] = pool[:, late]
        self.table = np.where(self.table >= 0, to[np.maximum(self.table, 0)], -1).astype(np.int32)
        self.refs[holes], self.refs[late] = self.refs[late], 0
        return n_live


def describe(kx, k, v, table, lens, refs, dtype):
    """A kx_kv over torch tensors: k, v (layers, n_pages, heads, page, d), any strides of the first two axes."""
    c = kx.KvCache()
    c.type, c.layers, c.n_pages, c.heads, c.page, c.dk = TYPE_IDS[dtype], *k.shape
    c.dv, (c.n_seqs, c.max_pages) = v.shape[4], table.shape
    c.k, c.v, c.table, c.lens, c.refs = (t.data_ptr() for t in (k, v, table, lens, refs))
    c.k_layer, c.k_page, c.v_layer, c.v_page = k.stride(0), k.stride(1), v.stride(0), v.stride(1)
    return c


def fake(kx, **kw):
    """A valid description over made-up addresses, for calls that are refused before anything runs."""
    c = kx.KvCache()
    c.type, c.layers, c.n_pages, c.page, c.heads, c.dk, c.dv, c.n_seqs, c.max_pages = 1, 2, 10, 16, 2, 64, 64, 4, 5
    c.k, c.v, c.table, c.lens, c.refs = 0x10000, 0x20000, 0x30000, 0x40000, 0x50000
    c.k_page = c.v_page = 2 * 16 * 64
    c.k_layer = c.v_layer = 10 * 2 * 16 * 64
    for name, value in kw.items():
        setattr(c, name, value)
    return c


def ref(c):
    return ctypes.byref(c)
