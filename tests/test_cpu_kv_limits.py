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
