"""Measured cases of the key-value cache operators: the pages of a cache (extend, append, fork, free, compact), the
attention of one new token over the paged cache, and the attention of a prompt with a sliding window whose first tokens
stay visible. `run` computes an operator in its plain form (elementary torch operations), or, where `own` is true, with
the calls a user makes of the library (kernix_b200.kx_abi, include/kx_kernels.h).

Conventions of the operators, as both forms compute them:

* a cache holds `layers` x `n_pages` pages of `page` tokens x `heads` key-value heads; sequence slot s owns the pages
  table[s][0 .. ceil(lens[s] / page)), -1 behind them; refs[p] counts the table entries that name page p, 0 = free;
* a token at position t sees key j when j <= t and (window <= 0 or j > t - window or j < sinks);
* free pages are handed out lowest id first, in the order of the sequences.
"""
import ctypes
import math
import zlib

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE_IDS = {"f32": 0, "f16": 1, "bf16": 2}
NO_PAGES = 2  # status bit: a request was refused for want of free pages


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one chat, one new token: the encoder configuration's heads (8 x 64) over a cache of its 128 tokens; latency
        dict(name="token_one_f32", op="token", n=1, H=8, heads=8, dk=64, dv=64, page=16, type="f32", lmin=128, lmax=128,
             window=0, sinks=0),
        # a serving batch in mid-stream: ragged lengths, grouped heads, 16-bit cache
        dict(name="token_batch_bf16", op="token", n=32, H=32, heads=8, dk=128, dv=128, page=16, type="bf16", lmin=1,
             lmax=4096, window=0, sinks=0),
        # a few very long documents: the cache's length has to be split to fill the GPU
        dict(name="token_long_f16", op="token", n=3, H=16, heads=4, dk=128, dv=128, page=64, type="f16", lmin=60000,
             lmax=131001, window=0, sinks=0),
        # streaming sessions: far past the window, which moves; the first tokens stay; odd head dims, fp32 cache
        dict(name="token_window_f32", op="token", n=48, H=12, heads=4, dk=72, dv=80, page=32, type="f32", lmin=900,
             lmax=9001, window=1000, sinks=4),
        # the page bookkeeping of one scheduler step: half of the slots end and take new prompts
        dict(name="pages_turnover", op="turnover", slots=256, page=16, max_pages=256, n_pages=24576),
        # one decode step of one layer: a token of each sequence into its page
        dict(name="append_step_bf16", op="append", n=64, rows=1, heads=8, dk=128, dv=128, page=16, type="bf16", lmax=2048),
        # prompts into the cache, one layer: ragged rows of a padded batch
        dict(name="append_prompts_f16", op="append", n=12, rows=1999, heads=8, dk=128, dv=128, page=16, type="f16", lmax=0),
        # parallel samples of a prompt: full pages shared, the half-filled last page copied, 4 layers
        dict(name="fork_samples", op="fork", parents=8, children=6, heads=8, dk=64, dv=64, page=32, type="bf16", layers=4,
             lmax=1500, n_pages=4096),
        # a pool after hours of turnover: live pages moved to its low end, tables rewritten, 2 layers
        dict(name="compact_pool", op="compact", slots=96, heads=4, dk=128, dv=128, page=16, type="bf16", layers=2,
             lmax=1024, n_pages=8192),
        # the encoder configuration's layer (8 samples x 128 rows, 8 heads of 64) read as a causal prompt with a window
        dict(name="prompt_short", op="prompt", B=8, Rq=128, S=128, H=8, heads=8, dk=64, dv=64, window=48, sinks=4, full=True),
        # a long prompt through a windowed layer, grouped heads
        dict(name="prompt_long", op="prompt", B=1, Rq=16384, S=16384, H=16, heads=4, dk=128, dv=128, window=2048, sinks=4,
             full=True),
        # the next chunk of prompts that are partly cached, padded batch, odd sizes, no window
        dict(name="prompt_chunk_odd", op="prompt", B=3, Rq=700, S=2501, H=6, heads=2, dk=80, dv=72, window=0, sinks=0,
             full=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["token", "token", "token", "turnover", "append", "fork", "compact", "prompt", "prompt", "prompt"])
    heads = rng.choice([1, 2, 3, 4, 6, 8])
    page = rng.choice([8, 16, 32, 64, 128])
    dt = rng.choice(["f32", "f16", "bf16"])
    if op == "token":
        dk, dv = rng.choice([(64, 64), (128, 128), (32, 32), (80, 80), (96, 64), (72, 128), (112, 120)])
        group = rng.choice([1, 2, 3, 4, 6, 8, 12])
        lmax = _log(rng, 1, 100000)
        lmax = min(lmax, int(400e6 / (heads * (dk + dv) * DTYPES[dt].itemsize)))
        n = max(1, min(_log(rng, 1, 200), int(400e6 / (lmax * heads * (dk + dv) * DTYPES[dt].itemsize))))
        window = rng.choice([0, 0, _log(rng, 1, 8192)])
        return dict(op=op, n=n, H=heads * group, heads=heads, dk=dk, dv=dv, page=page, type=dt, lmin=rng.choice([1, lmax]),
                    lmax=lmax, window=window, sinks=rng.choice([0, 1, 4, 16, 100]))
    if op == "turnover":
        slots, max_pages = _log(rng, 1, 512), _log(rng, 1, 300)
        return dict(op=op, slots=slots, page=page, max_pages=max_pages,
                    n_pages=min(60000, max(1, int(slots * max_pages * rng.choice([0.3, 0.6, 1.0])))))
    dk, dv = rng.choice([(64, 64), (128, 128), (32, 32), (80, 80), (96, 64), (72, 128), (112, 120)])
    if op == "append":
        n, rows = _log(rng, 1, 64), rng.choice([1, 1, 2, _log(rng, 1, 2000)])
        return dict(op=op, n=n, rows=rows, heads=heads, dk=dk, dv=dv, page=page, type=dt, lmax=rng.choice([0, _log(rng, 1, 3000)]))
    if op == "fork":
        parents, children = _log(rng, 1, 16), _log(rng, 1, 8)
        return dict(op=op, parents=parents, children=children, heads=heads, dk=dk, dv=dv, page=page, type=dt,
                    layers=rng.choice([1, 2, 3]), lmax=_log(rng, 1, 1500), n_pages=rng.choice([1024, 2500]))
    if op == "compact":
        slots = _log(rng, 1, 96)
        n_pages = _log(rng, 64, 4096)
        return dict(op=op, slots=slots, heads=rng.choice([1, 2, 4]), dk=dk, dv=dv, page=rng.choice([8, 16, 32]), type=dt,
                    layers=rng.choice([1, 2]), lmax=max(1, min(2000, n_pages * 8 // slots)), n_pages=n_pages)
    S = _log(rng, 1, 9000)
    H = heads * rng.choice([1, 2, 3, 4, 8])
    dk, dv = rng.choice([(dk, dv), (50, 33), (24, 100)])
    while S * S * H * (dk + dv) > 2.5e11:
        S //= 2
    B = max(1, min(_log(rng, 1, 12), int(2.5e11 / (S * S * H * (dk + dv)))))
    Rq = rng.choice([S, S, max(1, S // 3), min(S, 129)])
    return dict(op="prompt", B=B, Rq=Rq, S=S, H=H, heads=heads, dk=dk, dv=dv,
                window=rng.choice([0, _log(rng, 1, 3000), _log(rng, 1, 3000)]), sinks=rng.choice([0, 1, 4, 33]),
                full=rng.choice([True, False]))


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(rs, n, lo, hi):
    """n lengths in [lo, hi], spread over their logarithm; the longest is there."""
    ls = np.exp(rs.uniform(math.log(max(1, lo)), math.log(max(1, hi)), n)).round().astype(np.int64).clip(lo, hi)
    ls[rs.randint(n)] = hi
    return ls


def _shapes(case):
    """Everything about a case that the seed alone decides on the host: lengths, tables, references."""
    op, page = case["op"], case.get("page", 1)
    # lengths go by the case alone (so that work() is exact), pages and values by the seed
    rs = np.random.RandomState(zlib.crc32(repr(sorted((x, y) for x, y in case.items() if x not in ("name", "_seed"))).encode()))
    if op == "token":
        lens = _lengths(rs, case["n"], case["lmin"], case["lmax"])
    elif op == "append":
        old = rs.randint(0, case["lmax"] + 1, case["n"])
        count = np.full(case["n"], 1) if case["rows"] == 1 else rs.randint(0, case["rows"] + 1, case["n"])
        count[rs.randint(case["n"])] = case["rows"]
        lens = old + count
    elif op == "turnover":
        lens = rs.randint(0, case["max_pages"] * page + 1, case["slots"])
    elif op == "fork":
        lens = np.concatenate([_lengths(rs, case["parents"], 1, case["lmax"]), np.zeros(case["parents"] * case["children"], np.int64)])
    elif op == "compact":
        lens = rs.randint(0, case["lmax"] + 1, case["slots"])
    else:  # prompt
        k_len = np.full(case["B"], case["S"]) if case["full"] else rs.randint(1, case["S"] + 1, case["B"])
        k_len[0] = case["S"]
        q_len = np.minimum(k_len, np.full(case["B"], case["Rq"]) if case["full"] else rs.randint(1, case["Rq"] + 1, case["B"]))
        q_len[0] = case["Rq"]
        return dict(k_len=k_len, q_len=q_len, rs=rs)
    need = -(-lens // page)
    n_pages = case.get("n_pages", int(need.sum() * 1.1) + 3)
    # a sequence whose pages the pool no longer holds is not there
    for s in range(len(lens)):
        if need[: s + 1].sum() > n_pages * 0.95 + 1 or need[: s + 1].sum() > n_pages:
            lens[s] = need[s] = 0
    max_pages = case.get("max_pages", int(max(1, need.max())) + 1)
    table = np.full((len(lens), max_pages), -1, np.int32)
    ids = np.random.RandomState(case["_seed"] % (1 << 31)).permutation(n_pages).astype(np.int32)
    at = 0
    for s, c in enumerate(need):
        table[s, :c] = ids[at:at + c]
        at += c
    refs = np.zeros(n_pages, np.int32)
    refs[table[table >= 0]] = 1
    out = dict(lens=lens.astype(np.int32), table=table, refs=refs, n_pages=n_pages, max_pages=max_pages, need=need, rs=rs)
    if op == "append":
        out["count"] = count.astype(np.int32)
    if op == "turnover":
        slots = case["slots"]
        out["ended"] = rs.permutation(slots)[: (slots + 1) // 2].astype(np.int32)
        want = np.zeros(slots, np.int32)
        want[out["ended"]] = rs.randint(1, case["max_pages"] * page + 1, len(out["ended"]))
        out["want"] = want
    if op == "fork":
        out["src"] = np.repeat(np.arange(case["parents"], dtype=np.int32), case["children"])
        out["dst"] = (case["parents"] + rs.permutation(case["parents"] * case["children"])).astype(np.int32)
    return out


def prepare(case, seed):
    case = dict(case, _seed=seed)
    sh = _shapes(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    cuda = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    st = dict(case=case, host=sh)
    if case["op"] == "prompt":
        B, Rq, S, H, heads, dk, dv = (case[x] for x in ("B", "Rq", "S", "H", "heads", "dk", "dv"))
        st["q"] = torch.randn(B * Rq, H * dk, device="cuda", generator=g)
        st["k"] = torch.randn(B * S, heads * dk, device="cuda", generator=g)
        st["v"] = torch.randn(B * S, heads * dv, device="cuda", generator=g)
        st["ctx"] = torch.zeros(B * Rq, H * dv, device="cuda")
        st["q_len"], st["k_len"] = cuda(sh["q_len"].astype(np.int32)), cuda(sh["k_len"].astype(np.int32))
        if own:
            from kernix_b200 import kx_abi
            st["ws"] = torch.empty(kx_abi.lib().kx_attention_window_ws(B, S, heads, dk, dv), dtype=torch.uint8, device="cuda")
            st["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        return st
    for x in ("lens", "table", "refs"):
        st[x] = cuda(sh[x])
    layers, dt = case.get("layers", 1), DTYPES[case.get("type", "f16")]
    heads, dk, dv = case.get("heads", 1), case.get("dk", 8), case.get("dv", 8)
    if case["op"] != "turnover":
        for x, d in (("kc", dk), ("vc", dv)):
            st[x] = torch.empty(layers, sh["n_pages"], heads, case["page"], d, dtype=dt, device="cuda")
            for pool in st[x]:
                pool.copy_(torch.randn(pool.shape, device="cuda", generator=g, dtype=dt if dt != torch.float32 else None))
    if case["op"] == "token":
        st["q"] = torch.randn(case["n"], case["H"] * dk, device="cuda", generator=g)
        st["ctx"] = torch.zeros(case["n"], case["H"] * dv, device="cuda")
    elif case["op"] == "append":
        st["count"] = cuda(sh["count"])
        st["k"] = torch.randn(case["n"] * case["rows"], heads * dk, device="cuda", generator=g)
        st["v"] = torch.randn(case["n"] * case["rows"], heads * dv, device="cuda", generator=g)
    elif case["op"] == "turnover":
        st["ended"], st["want"] = cuda(sh["ended"]), cuda(sh["want"])
        st["granted"] = torch.zeros_like(st["want"])
        # the pool itself is not touched by the bookkeeping; the handle needs one
        st["kc"] = torch.zeros(1, sh["n_pages"], 1, case["page"], 8, dtype=dt, device="cuda")
        st["vc"] = torch.zeros(1, sh["n_pages"], 1, case["page"], 8, dtype=dt, device="cuda")
    elif case["op"] == "fork":
        st["src"], st["dst"] = cuda(sh["src"]), cuda(sh["dst"])
    elif case["op"] == "compact":
        # the bookkeeping before the call, so that a pass can be repeated (the pages it moved from keep their contents)
        st["lens0"], st["table0"], st["refs0"] = st["lens"].clone(), st["table"].clone(), st["refs"].clone()
        st["n_live"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    st["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    if own:
        from kernix_b200 import kx_abi
        c = kx_abi.KvCache()
        c.type, c.layers, c.n_pages, c.page, c.heads = TYPE_IDS[case.get("type", "f16")], layers, sh["n_pages"], case["page"], heads
        c.dk, c.dv, c.n_seqs, c.max_pages = dk, dv, len(sh["lens"]), sh["max_pages"]
        c.k, c.v = st["kc"].data_ptr(), st["vc"].data_ptr()
        c.k_page, c.v_page = st["kc"].stride(1), st["vc"].stride(1)
        c.k_layer, c.v_layer = st["kc"].stride(0), st["vc"].stride(0)
        c.table, c.lens, c.refs = st["table"].data_ptr(), st["lens"].data_ptr(), st["refs"].data_ptr()
        st["cache"], st["handle"] = c, ctypes.byref(c)
        if case["op"] == "token":
            nbytes = kx_abi.lib().kx_attention_paged_ws(st["handle"], case["H"], case["n"])
        else:
            nbytes = kx_abi.lib().kx_kv_ws(st["handle"])
        st["ws"] = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _softmax_pv(s, vis, v):
    """Softmax over the last axis of s where vis, 0 in rows that see nothing; times v."""
    s = s.masked_fill(~vis, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    den = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(den == 0, torch.ones_like(den), den)


def _plain_token(st):
    c = st["case"]
    n, H, heads, dk, dv, page = (c[x] for x in ("n", "H", "heads", "dk", "dv", "page"))
    P = max(1, int(st["host"]["need"].max()))
    pages = st["table"][:, :P].clamp(min=0).long()
    k = st["kc"][0][pages].float().transpose(1, 2).reshape(n, heads, P * page, dk)
    v = st["vc"][0][pages].float().transpose(1, 2).reshape(n, heads, P * page, dv)
    j = torch.arange(P * page, device="cuda")
    t = (st["lens"].long() - 1)[:, None]
    vis = j <= t
    if c["window"] > 0:
        vis &= (j > t - c["window"]) | (j < c["sinks"])
    v = torch.where(vis[:, None, :, None], v, torch.zeros((), device="cuda"))
    s = torch.matmul(st["q"].view(n, heads, H // heads, dk) * (1.0 / math.sqrt(dk)), k.transpose(2, 3))
    st["ctx"].copy_(_softmax_pv(s, vis[:, None, None, :], v).reshape(n, H * dv))
    return st["ctx"]


def _plain_prompt(st):
    c = st["case"]
    B, Rq, S, H, heads, dk, dv = (c[x] for x in ("B", "Rq", "S", "H", "heads", "dk", "dv"))
    G = H // heads
    j = torch.arange(S, device="cuda")
    for b in range(B):
        ql, kl = int(st["host"]["q_len"][b]), int(st["host"]["k_len"][b])
        k = st["k"][b * S:b * S + kl].view(kl, heads, dk).permute(1, 2, 0)[:, None]
        v = st["v"][b * S:b * S + kl].view(kl, heads, dv).transpose(0, 1)[:, None]
        for i0 in range(0, ql, 512):
            i1 = min(ql, i0 + 512)
            hi = kl - ql + i1  # keys behind the last row's position are seen by none
            q = st["q"][b * Rq + i0:b * Rq + i1].view(i1 - i0, heads, G, dk).permute(1, 2, 0, 3) * (1.0 / math.sqrt(dk))
            t = torch.arange(kl - ql + i0, kl - ql + i1, device="cuda")[:, None]
            vis = j[:hi] <= t
            if c["window"] > 0:
                vis &= (j[:hi] > t - c["window"]) | (j[:hi] < c["sinks"])
            o = _softmax_pv(torch.matmul(q, k[..., :hi]), vis, v[:, :, :hi])
            st["ctx"][b * Rq + i0:b * Rq + i1] = o.permute(2, 0, 1, 3).reshape(i1 - i0, H * dv)
    return st["ctx"]


def _free_list(refs):
    """ids of the free pages, lowest first (as long as refs; the rest is -1), and how many there are"""
    n = refs.numel()
    free = refs == 0
    rank = torch.where(free, torch.cumsum(free, 0) - 1, torch.full_like(refs, n, dtype=torch.int64))
    ids = torch.full((n + 1,), -1, dtype=torch.int32, device="cuda")
    ids[rank] = torch.arange(n, dtype=torch.int32, device="cuda")
    return ids[:n], free.sum()


def _plain_free(st, seqs):
    rows = st["table"][seqs.long()].long()
    st["refs"].scatter_add_(0, rows.clamp(min=0).view(-1), -(rows >= 0).view(-1).int())
    st["table"][seqs.long()] = -1
    st["lens"][seqs.long()] = 0


def _plain_turnover(st):
    c, table, lens = st["case"], st["table"], st["lens"].long()
    page, (slots, width) = c["page"], table.shape
    _plain_free(st, st["ended"])
    lens, want = st["lens"].long(), st["want"].long()
    have = (lens + page - 1) // page
    fits = lens + want <= width * page
    need = torch.where(fits, (lens + want + page - 1) // page - have, 0)
    ids, n_free = _free_list(st["refs"])
    upto = torch.cumsum(need, 0)
    ok = fits & ((need == 0) | (upto <= n_free))
    col = torch.arange(width, device="cuda")[None, :]
    new = ok[:, None] & (col >= have[:, None]) & (col < (have + need)[:, None])
    which = ((upto - need)[:, None] + col - have[:, None]).clamp(0, ids.numel() - 1)
    table.copy_(torch.where(new, ids[which], table))
    st["refs"].scatter_add_(0, ids[which].clamp(min=0).long().view(-1), new.view(-1).int())
    st["granted"].copy_(torch.where(ok, want, 0))
    st["lens"].copy_(lens + st["granted"])
    st["status"].copy_((fits & ~ok).any() * NO_PAGES)
    return [st["table"], st["lens"], st["refs"], st["granted"], st["status"]]


def _plain_append(st):
    c = st["case"]
    n, rows, heads, dk, dv, page = (c[x] for x in ("n", "rows", "heads", "dk", "dv", "page"))
    kc, vc = st["kc"][0], st["vc"][0]
    i = torch.arange(rows, device="cuda")[None, :]
    count = st["count"].long()[:, None]
    pos = (st["lens"].long()[:, None] - count + i).clamp(min=0)
    ids = torch.gather(st["table"].long(), 1, (pos // page).clamp(max=st["table"].shape[1] - 1))
    live = (i < count).view(-1)
    # rows behind a sequence's count write the value of the first live row of the batch to that row's own place
    first = torch.argmax(live.int())
    at = torch.where(live, torch.arange(n * rows, device="cuda"), first)
    p, s = ids.reshape(-1)[at], (pos % page).reshape(-1)[at]
    kc[p, :, s] = st["k"].view(n * rows, heads, dk)[at].to(kc.dtype)
    vc[p, :, s] = st["v"].view(n * rows, heads, dv)[at].to(vc.dtype)
    return [st["kc"], st["vc"]]


def _plain_fork(st):
    c, table = st["case"], st["table"]
    page, width = c["page"], table.shape[1]
    _plain_free(st, st["dst"])
    src, dst = st["src"].long(), st["dst"].long()
    lens = st["lens"].long()[src]
    part = lens % page != 0
    ids, n_free = _free_list(st["refs"])
    upto = torch.cumsum(part, 0)
    ok = ~part | (upto <= n_free)
    fresh = ids[(upto - 1).clamp(0, ids.numel() - 1)].long()
    col = torch.arange(width, device="cuda")[None, :]
    rows = table[src].long()
    last = (part[:, None]) & (col == (lens // page)[:, None])
    rows = torch.where(last, fresh[:, None], rows)
    rows = torch.where(ok[:, None], rows, -1)
    tail = table[src, (lens // page).clamp(max=width - 1)].long()
    take = ok & part
    to = torch.where(take, fresh, tail.clamp(min=0))  # a child without a partial page copies a page onto itself
    for pool in (st["kc"], st["vc"]):
        pool[:, to] = pool[:, tail.clamp(min=0)]
    table[dst] = rows.int()
    st["refs"].scatter_add_(0, rows.clamp(min=0).view(-1), (rows >= 0).view(-1).int())
    st["lens"][dst] = torch.where(ok, lens, 0).int()
    st["status"].copy_((~ok).any() * NO_PAGES)
    return [st["kc"], st["vc"], st["table"], st["lens"], st["refs"], st["status"]]


def _restore(st):
    st["table"].copy_(st["table0"])
    st["refs"].copy_(st["refs0"])


def _plain_compact(st):
    _restore(st)
    refs, n = st["refs"], st["refs"].numel()
    live = refs > 0
    st["n_live"].copy_(live.sum())
    p = torch.arange(n, device="cuda")
    hole, late = ~live & (p < st["n_live"]), live & (p >= st["n_live"])
    # the r-th hole takes the r-th late page
    lists = torch.full((2, n + 1), 0, dtype=torch.int64, device="cuda")
    for row, mask in zip(lists, (hole, late)):
        row[torch.where(mask, torch.cumsum(mask, 0) - 1, n)] = p
    to = torch.where(late, lists[0][(torch.cumsum(late, 0) - 1).clamp(min=0)], p)
    frm = torch.where(hole, lists[1][(torch.cumsum(hole, 0) - 1).clamp(min=0)], p)
    for pool in (st["kc"], st["vc"]):
        for layer in pool:
            layer.copy_(layer[frm])
    st["table"].copy_(torch.where(st["table"] >= 0, to[st["table"].clamp(min=0).long()].int(), st["table"]))
    moved = refs[frm]
    refs.copy_(torch.where(late, torch.zeros_like(refs), moved))
    return [st["kc"], st["vc"], st["table"], st["lens"], st["refs"], st["n_live"]]


# ------------------------------------------------------------------------------------------------ one pass
def run(st):
    c = st["case"]
    op = c["op"]
    if not own:
        return {"token": _plain_token, "prompt": _plain_prompt, "turnover": _plain_turnover, "append": _plain_append,
                "fork": _plain_fork, "compact": _plain_compact}[op](st)
    from kernix_b200 import kx_abi
    stream = torch.cuda.current_stream().cuda_stream
    if op == "prompt":
        kx_abi.call("kx_attention_window", st["q"].data_ptr(), c["H"] * c["dk"], st["k"].data_ptr(), c["heads"] * c["dk"],
                    st["v"].data_ptr(), c["heads"] * c["dv"], st["ctx"].data_ptr(), c["H"] * c["dv"], c["B"], c["Rq"], c["S"],
                    c["H"], c["heads"], c["dk"], c["dv"], st["q_len"].data_ptr(), st["k_len"].data_ptr(), c["window"], c["sinks"],
                    0.0, st["ws"].data_ptr(), st["ws"].numel(), st["status"].data_ptr(), stream)
        return st["ctx"]
    h, ws, status = st["handle"], st["ws"].data_ptr(), st["status"].data_ptr()
    if op == "token":
        kx_abi.call("kx_attention_paged", h, 0, st["q"].data_ptr(), c["H"] * c["dk"], c["H"], None, c["n"], c["window"], c["sinks"],
                    0.0, st["ctx"].data_ptr(), c["H"] * c["dv"], ws, st["ws"].numel(), status, stream)
        return st["ctx"]
    if op == "append":
        kx_abi.call("kx_kv_append", h, 0, st["k"].data_ptr(), c["heads"] * c["dk"], st["v"].data_ptr(), c["heads"] * c["dv"],
                    st["count"].data_ptr(), c["rows"], status, stream)
        return [st["kc"], st["vc"]]
    if op == "turnover":
        kx_abi.call("kx_kv_free", h, st["ended"].data_ptr(), st["ended"].numel(), status, stream)
        kx_abi.call("kx_kv_extend", h, st["want"].data_ptr(), st["granted"].data_ptr(), ws, st["ws"].numel(), status, stream)
        return [st["table"], st["lens"], st["refs"], st["granted"], st["status"]]
    if op == "fork":
        kx_abi.call("kx_kv_free", h, st["dst"].data_ptr(), st["dst"].numel(), status, stream)
        kx_abi.call("kx_kv_fork", h, st["src"].data_ptr(), st["dst"].data_ptr(), st["src"].numel(), ws, st["ws"].numel(), status, stream)
        return [st["kc"], st["vc"], st["table"], st["lens"], st["refs"], st["status"]]
    _restore(st)
    kx_abi.call("kx_kv_compact", h, st["n_live"].data_ptr(), ws, st["ws"].numel(), stream)
    return [st["kc"], st["vc"], st["table"], st["lens"], st["refs"], st["n_live"]]


# ------------------------------------------------------------------------------------------------ work
def _pairs(pos, window, sinks):
    """keys that tokens at the positions `pos` (int array) see"""
    seen = np.maximum(pos + 1, 0)
    if window > 0:
        first = np.maximum(pos - window + 1, 0)
        seen = np.maximum(pos - first + 1, 0) + np.minimum(np.minimum(sinks, first), np.maximum(pos + 1, 0))
    return seen


def work(case):
    c, op = case, case["op"]
    size = DTYPES[c.get("type", "f16")].itemsize
    sh = _shapes(dict(c, _seed=1))
    if op == "prompt":
        flops = rows = 0
        for ql, kl in zip(sh["q_len"].tolist(), sh["k_len"].tolist()):
            flops += int(_pairs(np.arange(kl - ql, kl), c["window"], c["sinks"]).sum()) * 2 * (c["dk"] + c["dv"]) * c["H"]
            rows += ql * c["H"] + kl * c["heads"]
        return dict(bytes=rows * (c["dk"] + c["dv"]) * 4, flops=flops)
    need = sh["need"]
    if op == "token":
        seen = int(_pairs(sh["lens"].astype(np.int64) - 1, c["window"], c["sinks"]).sum())
        per = c["dk"] + c["dv"]
        return dict(bytes=seen * c["heads"] * per * size + c["n"] * c["H"] * per * 4, flops=seen * c["H"] * 2 * per)
    if op == "append":
        return dict(bytes=int(sh["count"].sum()) * c["heads"] * (c["dk"] + c["dv"]) * (4 + size), flops=0)
    if op == "turnover":
        # the table rows of the slots that turn over are read and written, every reference count read, those of the pages written
        moved = int(need[sh["ended"]].sum()) + int(-(-sh["want"] // c["page"]).sum())
        return dict(bytes=4 * (sh["n_pages"] + 2 * moved + 4 * c["slots"]), flops=0)
    token = c["heads"] * (c["dk"] + c["dv"]) * size * c["layers"]
    if op == "fork":
        lens = sh["lens"][sh["src"]].astype(np.int64)
        return dict(bytes=int((lens % c["page"]).sum()) * token * 2 + 4 * (sh["n_pages"] + 2 * int(need[sh["src"]].sum())), flops=0)
    live = int((sh["refs"] > 0).sum())
    late = int((sh["refs"][live:] > 0).sum())
    return dict(bytes=late * c["page"] * token * 2 + 4 * (2 * sh["n_pages"] + 2 * int(need.sum())), flops=0)


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_rows(q, k, v, pos, window, sinks):
    """Attention of the rows q (rows x group x dk) at the positions pos over k, v (keys x d), by the definition."""
    out = torch.zeros(q.shape[0], q.shape[1], v.shape[1], dtype=torch.float64, device=q.device)
    j = torch.arange(k.shape[0], device=q.device)
    for r0 in range(0, q.shape[0], 256):
        t = pos[r0:r0 + 256, None]
        vis = (j <= t) & ((window <= 0) | (j > t - window) | (j < sinks))
        s = torch.einsum("rgd,jd->rgj", q[r0:r0 + 256], k) / math.sqrt(q.shape[2])
        w = torch.where(vis[:, None], s, torch.tensor(-math.inf, dtype=torch.float64, device=q.device))
        top = w.max(dim=2, keepdim=True).values.clamp(min=-1e300)
        e = torch.exp(w - top) * vis[:, None]
        out[r0:r0 + 256] = torch.einsum("rgj,jd->rgd", e, v) / e.sum(2, keepdim=True).clamp(min=1e-300)
    return out


def exact(case, seed):
    c, op = case, case["op"]
    if op == "turnover":
        return None  # whole numbers only
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    sh = st["host"]
    if op == "prompt":
        B, Rq, S, H, heads, dk, dv = (c[x] for x in ("B", "Rq", "S", "H", "heads", "dk", "dv"))
        if float(B) * Rq * S * H * (dk + dv) > 4e12:
            return None
        q, k, v = (st[x].double() for x in "qkv")
        out = torch.zeros(B, Rq, heads, H // heads, dv, dtype=torch.float64, device="cuda")
        for b in range(B):
            ql, kl = int(sh["q_len"][b]), int(sh["k_len"][b])
            pos = torch.arange(kl - ql, kl, device="cuda")
            for h in range(heads):
                qh = q.view(B, Rq, heads, H // heads, dk)[b, :ql, h]
                out[b, :ql, h] = _exact_rows(qh, k.view(B, S, heads, dk)[b, :kl, h], v.view(B, S, heads, dv)[b, :kl, h], pos,
                                             c["window"], c["sinks"])
        return out.view(B * Rq, H * dv)
    if op == "token":
        n, H, heads, dk, dv, page = (c[x] for x in ("n", "H", "heads", "dk", "dv", "page"))
        out = torch.zeros(n, heads, H // heads, dv, dtype=torch.float64, device="cuda")
        for s in range(n):
            length = int(sh["lens"][s])
            if length == 0:
                continue
            ids = torch.from_numpy(sh["table"][s, : sh["need"][s]].astype(np.int64)).cuda()
            pos = torch.tensor([length - 1], device="cuda")
            for h in range(heads):
                k, v = (st[x][0][ids, h].double().reshape(-1, d)[:length] for x, d in (("kc", dk), ("vc", dv)))
                out[s, h] = _exact_rows(st["q"].double().view(n, heads, H // heads, dk)[s, h][None], k, v, pos, c["window"], c["sinks"])[0]
        return out.view(n, H * dv)
    # pages that are copied or moved: their values in 64 bits; whole numbers have no other value than the plain form's
    kc, vc = st["kc"].double(), st["vc"].double()
    if op == "append":
        for s in range(c["n"]):
            count, length = int(sh["count"][s]), int(sh["lens"][s])
            if count == 0:
                continue
            pos = np.arange(length - count, length)
            ids = torch.from_numpy(sh["table"][s, pos // c["page"]].astype(np.int64)).cuda()
            slot = torch.from_numpy(pos % c["page"]).cuda()
            rows = slice(s * c["rows"], s * c["rows"] + count)
            kc[0, ids, :, slot] = st["k"][rows].double().view(count, c["heads"], c["dk"])
            vc[0, ids, :, slot] = st["v"][rows].double().view(count, c["heads"], c["dv"])
        return [kc, vc]
    refs = sh["refs"].copy()
    if op == "fork":
        free = np.flatnonzero(refs == 0).tolist()
        for s in sh["src"]:
            length = int(sh["lens"][s])
            if length % c["page"] and free:
                for pool in (kc, vc):
                    pool[:, free[0]] = pool[:, int(sh["table"][s, length // c["page"]])]
                free.pop(0)
            elif length % c["page"]:
                break  # a child that finds no page is left out, and so is each one after it that needs one
        return [kc, vc, None, None, None, None]
    live = int((refs > 0).sum())
    holes, late = np.flatnonzero(refs[:live] == 0), live + np.flatnonzero(refs[live:] > 0)
    for pool in (kc, vc):
        pool[:, torch.from_numpy(holes).cuda()] = pool[:, torch.from_numpy(late).cuda()]
    return [kc, vc, None, None, None, None]
