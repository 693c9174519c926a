"""CPU: mea_clip_grad_norm refuses what it could not scale, before any device work."""
import ctypes

import pytest

from memory_efficient_attn_layer_b200 import _lib


def _call(spans, max_norm=1.0, kind=0):
    L, k = _lib.lib(), len(spans)
    at, n, dt = zip(*spans)
    need = L.mea_grad_norm_workspace_size(k)
    return L.mea_clip_grad_norm(k, (ctypes.c_void_p * k)(*at), (ctypes.c_longlong * k)(*n), (ctypes.c_int * k)(*dt), kind,
                                max_norm, 0x7000000, 0x7100000, need, None)


@pytest.mark.parametrize("spans,text", [
    ([(0x1000, 100, 2), (0x1000 + 396, 10, 2)], b"overlap"),  # the last fp32 of the first is the first of the second
    ([(0x1000 + 198, 10, 0), (0x1000, 100, 1)], b"overlap"),  # 16-bit elements, out of order
    ([(0x9000, 5, 2), (0x1000, 1000, 2), (0x8000, 1, 2), (0x1800, 1, 0)], b"overlap"),
    ([(0x1000, 3, 7)], b"dtype 7"), ([(0x1001, 3, 0)], b"not aligned"), ([(0x1002, 3, 2)], b"not aligned"),
    ([(0x1000, -1, 2)], b"-1 elements"), ([(None, 3, 2)], b"NULL"),
])
def test_lists_are_refused(spans, text):
    assert _call(spans) in (1, 3)
    assert text in _lib.lib().mea_last_error_string()


def test_thresholds_and_kinds_are_refused():
    for bad in (-1.0, float("nan")):
        assert _call([(0x1000, 3, 2)], max_norm=bad) == 1
    assert _call([(0x1000, 3, 2)], kind=3) == 1
