"""The 8-bit cache and shared-prefix entries on the host: calls at the edges of
what their documentation allows."""

import ctypes

from b200ops.runtime import lib as L


def test_prefix_workspace_alignment():
    """Piece rows of the prefix are stored 32 bytes at a time: a workspace at 16
    modulo 32 is refused before any launch (a decode's may be there)."""
    lib = L.load()
    p = ctypes.c_void_p(1 << 20)  # an address that is never read
    for code in (L.BF16, L.I8, L.F8E4M3):
        scale = None if code == L.BF16 else p
        need = lib.b200_paged_attention_prefix_workspace_size(2, 8, 2, 128, 16, 16, 8, 4, code, None)
        assert need > 0
        for off in (8, 16, 48):
            assert lib.b200_paged_attention_prefix(
                p, p, p, scale, scale, p, p, p, p, p, 2, 8, 2, 128, 16, 16, 8, 4, 0.0, L.BF16, code, L.I32,
                ctypes.c_void_p((1 << 20) + off), need, None, None) == L.ERR_ALIGNMENT
