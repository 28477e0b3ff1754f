"""Addresses that the mixture-of-experts entries could not read or write are refused on the host (no GPU needed)."""
import pytest

P, ODD = 32, 34                                           # stand for addresses, one of them off by half a word
ALIGN = -5


def _calls(lib):
    """name -> (call, which arguments are 4-byte addresses)"""
    tables = (P,) * 6                                     # offsets, tiles, wide tiles, rows, slots, source
    return {
        "plan": (lambda a: lib.nvfp4_moe_plan(a[0], 4, 4, 2, *a[1:7], a[7], None), (P,) + tables + (P,)),
        "route": (lambda a: lib.nvfp4_moe_route(a[0], 0, 8, None, 4, 8, 2, 1, *a[1:], None), (P, P, P) + tables + (P,)),
        "route_backward": (lambda a: lib.nvfp4_moe_route_backward(a[0], a[1], 0, 8, a[2], a[3], 4, 8, 2, 1, P, None), (P,) * 4),
        "dispatch": (lambda a: lib.nvfp4_moe_dispatch(a[0], 0, 8, a[1], a[2], 4, 8, 2, 8, a[3], None), (P,) * 4),
        "combine": (lambda a: lib.nvfp4_moe_combine(a[0], 0, 8, a[1], a[2], 4, 2, 8, a[3], 0, None), (P,) * 4),
        "combine_backward": (lambda a: lib.nvfp4_moe_combine_backward(a[0], 0, 8, a[1], 0, 8, a[2], a[3], a[4], 4, 8, 2, 8, a[5], a[6], None), (P,) * 7),
        "dispatch_nvfp4": (lambda a: lib.nvfp4_moe_dispatch_nvfp4(P, 0, 64, *a, 4, 8, 2, 64, P, P, None, None), (P,) * 5),
        "gemm": (lambda a: lib.nvfp4_moe_gemm(P, P, P, P, *a, P, 8, 4, 128, 256, 1.0, None), (P,) * 4),
    }


@pytest.mark.parametrize("name", ["plan", "route", "route_backward", "dispatch", "combine", "combine_backward", "dispatch_nvfp4", "gemm"])
def test_misaligned_addresses_are_refused(lib, name):
    call, good = _calls(lib)[name]
    for i in range(len(good)):
        args = good[:i] + (ODD,) + good[i + 1:]
        assert call(args) == ALIGN, (name, i)


@pytest.mark.parametrize("kind", [1, 2])
def test_16_bit_elements_need_even_addresses(lib, kind):
    assert lib.nvfp4_moe_route(33, kind, 8, None, 4, 8, 2, 1, *(P,) * 9, None) == ALIGN
    assert lib.nvfp4_moe_route_backward(P, 33, kind, 8, P, P, 4, 8, 2, 1, P, None) == ALIGN
    assert lib.nvfp4_moe_dispatch(33, kind, 8, P, P, 4, 8, 2, 8, P, None) == ALIGN
