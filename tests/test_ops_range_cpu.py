"""Size queries of the operators' C entries at the ends of their ranges (no GPU)."""
import ctypes as C

from test_ops_cpu import attn, refuse

from tossctr import _lib


def test_rows_beyond_32_bits_ask_for_no_workspace():
    """2^29 positions of eight heads over one are 2^32 rows: refused, and not before a workspace of terabytes is asked for."""
    for heads in (4, 8, 24):
        a = attn(T=1 << 29, H=heads, Hkv=1, S=4096)
        assert _lib.query("ctr_diffattn_fwd_ws_size", C.byref(a)) == 0
        refuse("sizes", "ctr_diffattn_fwd", C.byref(a), None, 0, None)
    assert _lib.query("ctr_diffattn_fwd_ws_size", C.byref(attn(T=1, S=4096))) > 0
