"""Refusals of the KV-cache operators at the limits of their arguments; nothing here touches a device."""
import ctypes as C

import pytest

from test_kv_args import ARG, P, view

CUDA = 3            # what an accepted call returns where there is no device, or where its memory is nobody's


@pytest.mark.parametrize("scale,want", [(1.5e38, True), (-3.4e38, True), (1.0001e38, True), (1e38, False), (-1e38, False), (0.0, False)])
def test_scales_whose_powers_of_two_leave_single_precision(brrr, scale, want):
    """log2(e) x 3e38 is infinite, and a score of zero times that no number."""
    L, v = brrr.lib(), view(brrr)
    r = C.byref(v)
    calls = [L.brrr_attn_tree(r, 1, 1, None, P, None, None, 0, P, 4, scale, 0, None, P, None, None), L.brrr_kv_weigh(r, 1, 1, None, P, None, None, None, 0, P, 4, scale, 0, P, None),
             L.brrr_attn_blocks(r, 1, None, P, 16, P, 4, 1, 1, 0, P, 4, scale, None, P, P, None, None)]
    if want:
        assert calls == [ARG] * 3
    elif not __import__("torch").cuda.is_available():
        assert calls == [CUDA] * 3
