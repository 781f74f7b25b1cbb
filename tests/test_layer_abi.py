"""Calls of the layers' C ABI that are refused before anything runs."""
import ctypes

import pytest


def _gated(rows, bg, bu, *, kept=None, ws=256, hidden=6, dim=8, t=0):
    """Return codes of the forward and the backward, with addresses that are never read."""
    from gsr import _lib
    L = _lib.lib()
    n = 1 << 30
    fwd = L.gsr_gated_fwd(256, rows, dim, dim, t, 256, 256, hidden, bg, bu, 0, 256, kept, ws, n, None)
    a = L.gsr_last_error()
    bwd = L.gsr_gated_bwd(256, rows, dim, dim, t, 256, 256, hidden, bg, bu, 0, 256, hidden, kept, 256, 256, 256, None, None, ws, n,
                          None)
    return (fwd, a), (bwd, L.gsr_last_error())


@pytest.mark.parametrize("rows", [1, 64, 65, 5000])
@pytest.mark.parametrize("bg,bu", [(256, None), (None, 256)])
def test_biases_go_together(rows, bg, bu):
    """One bias without the other is refused whatever kernel the sizes take."""
    for code, error in _gated(rows, ctypes.c_void_p(bg), ctypes.c_void_p(bu)):
        assert code == -1 and b"bg and bu" in error


@pytest.mark.parametrize("rows", [1, 64, 5000])
def test_buffers_are_aligned(rows):
    """workspace and kept start at multiples of 256 bytes, as their parts' offsets assume."""
    for kw in (dict(ws=256 + 16), dict(kept=256 + 128), dict(ws=255, kept=512)):
        for code, error in _gated(rows, None, None, hidden=600, dim=300, **kw):
            assert code == -1 and b"256 bytes" in error
