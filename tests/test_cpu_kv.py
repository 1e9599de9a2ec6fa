"""CPU: the cache entry points refuse bad descriptions and arguments before anything reaches a device."""
import pytest

from kv_model import fake, ref

BAD = [dict(type=3), dict(type=-1), dict(layers=0), dict(n_pages=0), dict(page=0), dict(page=24), dict(page=2048), dict(heads=0),
       dict(dk=0), dict(dk=60), dict(dv=4), dict(dk=2048), dict(n_seqs=0), dict(max_pages=0), dict(max_pages=1 << 30),
       dict(k=None), dict(v=None), dict(table=None), dict(lens=None), dict(refs=None), dict(k=0x10008), dict(v=0x20002),
       dict(k_page=2 * 16 * 64 - 8), dict(v_page=2 * 16 * 64 + 4), dict(k_layer=2 * 16 * 64), dict(v_layer=0),
       dict(k_layer=-4096), dict(heads=1 << 15, page=1024)]


@pytest.fixture(scope="module")
def kx(libkx):
    from kernix_b200 import kx_abi
    return kx_abi


def test_workspace_covers_every_list(kx):
    c = fake(kx)
    assert kx.lib().kx_kv_ws(ref(c)) >= 4 * (3 * 10 + 4 * 4 + 1)
    assert kx.lib().kx_kv_ws(None) == 0


@pytest.mark.parametrize("kw", BAD, ids=lambda kw: "-".join(f"{a}={b}" for a, b in kw.items()))
def test_bad_descriptions_are_refused(kx, kw):
    c, L = fake(kx, **kw), kx.lib()
    assert L.kx_kv_ws(ref(c)) == 0
    p, n = 0x60000, 1 << 20
    assert L.kx_kv_extend(ref(c), p, p, p, n, None, None) == -1
    assert L.kx_kv_append(ref(c), 0, p, 1 << 12, p, 1 << 12, p, 1, None, None) == -1
    assert L.kx_kv_fork(ref(c), p, p, 1, p, n, None, None) == -1
    assert L.kx_kv_free(ref(c), p, 1, None, None) == -1
    assert L.kx_kv_compact(ref(c), p, p, n, None) == -1


def test_layouts_that_are_not_refused(kx):
    """layers inside a page, and a pool of one layer whose layer stride is not looked at"""
    L, per = kx.lib(), 2 * 16 * 64
    assert L.kx_kv_ws(ref(fake(kx, k_page=2 * per, k_layer=per, v_page=3 * per, v_layer=per))) > 0
    assert L.kx_kv_ws(ref(fake(kx, layers=1, k_layer=0, v_layer=-1))) > 0
    assert L.kx_kv_ws(ref(fake(kx, page=1, k_page=128, v_page=128, k_layer=1280, v_layer=1280))) > 0


def test_bad_arguments_are_refused(kx):
    c, L = fake(kx), kx.lib()
    p, n = 0x60000, kx.lib().kx_kv_ws(ref(c))
    for args in [(None, p, p, n), (p, None, p, n), (p, p, None, n), (p, p, p, n - 1), (p, p, p + 8, n)]:
        assert L.kx_kv_extend(ref(c), *args, None, None) == -1
    for args in [(2, p, 128, p, 128, p, 1), (-1, p, 128, p, 128, p, 1), (0, None, 128, p, 128, p, 1), (0, p, 127, p, 128, p, 1),
                 (0, p, 128, p, 127, p, 1), (0, p, 128, None, 128, p, 1), (0, p, 128, p, 128, None, 1), (0, p, 128, p, 128, p, -1)]:
        assert L.kx_kv_append(ref(c), *args, None, None) == -1
    for args in [(p, p, 5, p, n), (p, p, -1, p, n), (None, p, 1, p, n), (p, None, 1, p, n), (p, p, 1, p, n - 1)]:
        assert L.kx_kv_fork(ref(c), *args, None, None) == -1
    assert L.kx_kv_free(ref(c), None, 1, None, None) == -1 and L.kx_kv_free(ref(c), p, -1, None, None) == -1
    assert L.kx_kv_compact(ref(c), None, p, n, None) == -1 and L.kx_kv_compact(ref(c), p, p, n - 1, None) == -1


def test_nothing_to_do_launches_nothing(kx):
    c, L = fake(kx), kx.lib()
    p, n = 0x60000, kx.lib().kx_kv_ws(ref(c))
    assert L.kx_kv_free(ref(c), None, 0, None, None) == 0
    assert L.kx_kv_fork(ref(c), None, None, 0, p, n, None, None) == 0
    assert L.kx_kv_append(ref(c), 0, None, 0, None, 0, None, 0, None, None) == 0


def test_paged_attention_refuses_bad_arguments(kx):
    c, L = fake(kx), kx.lib()
    p, n = 0x60000, kx.lib().kx_attention_paged_ws(ref(c), 4, 2)
    assert n > 0

    def call(c=c, layer=0, q=p, ldq=256, H=4, seqs=None, n_rows=2, window=0, sinks=0, scale=0.0, ctx=p, ldc=256, ws=p, nbytes=n):
        return L.kx_attention_paged(ref(c), layer, q, ldq, H, seqs, n_rows, window, sinks, scale, ctx, ldc, ws, nbytes, None, None)

    for kw in [dict(layer=2), dict(layer=-1), dict(q=None), dict(ldq=255), dict(H=3), dict(H=0), dict(n_rows=5), dict(n_rows=-1),
               dict(sinks=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(ctx=None), dict(ldc=255), dict(ws=None),
               dict(ws=p + 4), dict(nbytes=n - 1)]:
        assert call(**kw) == -1, kw
    for kw in BAD + [dict(dk=136, k_page=2 * 16 * 136, k_layer=10 * 2 * 16 * 136)]:
        bad = fake(kx, **kw)
        assert L.kx_attention_paged_ws(ref(bad), 4, 2) == 0 and call(c=bad) == -1, kw
    assert call(n_rows=0) == 0


def test_window_attention_refuses_bad_arguments(kx):
    L, p = kx.lib(), 0x60000
    n = L.kx_attention_window_ws(2, 100, 2, 64, 48)
    assert n > 0
    names = ["q", "ldq", "k", "ldk", "v", "ldv", "ctx", "ldc", "B", "Rq", "S", "H", "Hkv", "dk", "dv", "q_len", "k_len", "window",
             "sinks", "scale", "ws", "nbytes", "status", "stream"]
    good = dict(q=p, ldq=256, k=p, ldk=128, v=p, ldv=96, ctx=p, ldc=192, B=2, Rq=5, S=100, H=4, Hkv=2, dk=64, dv=48, q_len=None,
                k_len=None, window=0, sinks=0, scale=0.0, ws=p, nbytes=n, status=None, stream=None)

    def call(**kw):
        a = dict(good, **kw)
        return L.kx_attention_window(*[a[x] for x in names])

    for kw in [dict(q=None), dict(k=None), dict(v=None), dict(ctx=None), dict(ldq=255), dict(ldk=127), dict(ldv=95), dict(ldc=191),
               dict(B=-1), dict(Rq=-1), dict(S=0), dict(H=3), dict(H=0), dict(Hkv=0), dict(dk=0), dict(dk=129), dict(dv=0), dict(dv=129),
               dict(sinks=-1), dict(scale=float("nan")), dict(ws=None), dict(ws=p + 64), dict(nbytes=n - 1)]:
        assert call(**kw) == -1, kw
    assert call(B=0) == 0 and call(Rq=0) == 0
    for args in [(-1, 100, 2, 64, 48), (2, 0, 2, 64, 48), (2, 100, 0, 64, 48), (2, 100, 2, 129, 48), (2, 100, 2, 64, 0)]:
        assert L.kx_attention_window_ws(*args) == 0
