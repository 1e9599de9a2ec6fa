"""CPU: descriptions and arguments at the ends of their ranges, refused or taken before anything reaches a device."""
import pytest

from kv_model import fake, ref


@pytest.fixture(scope="module")
def kx(libkx):
    from kernix_b200 import kx_abi
    return kx_abi


@pytest.mark.parametrize("scale,ok", [(2.3e38, True), (-2.3e38, True), (2.4e38, False), (-3e38, False), (float("inf"), False)])
def test_scales_whose_base_2_form_is_finite(kx, scale, ok):
    """calls of no rows return 0 where the arguments are taken, -1 where they are refused"""
    c, L, p = fake(kx), kx.lib(), 0x60000
    n = L.kx_attention_paged_ws(ref(c), 4, 0)
    assert L.kx_attention_paged(ref(c), 0, p, 256, 4, None, 0, 0, 0, scale, p, 256, p, n, None, None) == (0 if ok else -1)
    n = L.kx_attention_window_ws(0, 100, 2, 64, 48)
    assert L.kx_attention_window(p, 256, p, 128, p, 96, p, 192, 0, 5, 100, 4, 2, 64, 48, None, None, 0, 0, scale, p, n, None,
                                 None) == (0 if ok else -1)


PER = 2 * 16 * 64


@pytest.mark.parametrize("kw", [
    dict(n_pages=1 << 30, k_page=1 << 40, v_page=1 << 40, k_layer=PER, v_layer=PER, layers=1 << 30),  # products of 2^70
    dict(n_pages=1 << 30, k_page=1 << 40), dict(layers=2**31 - 1, k_layer=1 << 56), dict(layers=2**31 - 1, v_layer=1 << 56),
    dict(n_seqs=(1 << 30) + 1), dict(n_seqs=2**31 - 1), dict(page=1, max_pages=2**31 - 1), dict(page=1, max_pages=2**31 - 1024)],
    ids=lambda kw: "-".join(f"{a}={b}" for a, b in kw.items()))
def test_layouts_past_the_ranges_are_refused(kx, kw):
    assert kx.lib().kx_kv_ws(ref(fake(kx, **kw))) == 0


@pytest.mark.parametrize("kw", [
    dict(n_seqs=1 << 30), dict(page=1, max_pages=2**31 - 1025), dict(n_pages=1 << 30, k_layer=PER << 30, v_layer=PER << 30),
    dict(k_layer=10 * PER, v_layer=9 * PER + PER), dict(k_page=2 * PER, k_layer=PER, v_page=3 * PER - 8, v_layer=2 * PER - 8),
    dict(layers=1 << 20, k_page=PER << 20, k_layer=PER, v_page=PER << 20, v_layer=PER),
    dict(layers=1 << 20, n_pages=1 << 20, k_layer=PER << 20, v_layer=PER << 20)],
    ids=lambda kw: "-".join(f"{a}={b}" for a, b in kw.items()))
def test_layouts_at_the_ends_of_the_ranges(kx, kw):
    assert kx.lib().kx_kv_ws(ref(fake(kx, **kw))) > 0
