"""CPU test: an adapter set remembers the workspace sizes of a bounded number of token counts, however
many a server's batches have."""
import ctypes as C

import hymoe


def test_bounded():
    ad = object.__new__(hymoe.Adapters)
    ad.L, ad.spec, ad._bytes = hymoe.lib(), hymoe.AdapterSpec(4, 16, 256, 256, hymoe.TYPE_BF16, None, None, None), {}
    for T in range(5000):
        n = ad._workspace_bytes(T, T % 2 == 1)
        assert len(ad._bytes) <= 256 and n == ad._workspace_bytes(T, T % 2 == 1)
        want = C.c_size_t()
        assert ad.L.hymoe_adapt_workspace(C.byref(ad.spec), T, T % 2, C.byref(want)) == 0 and want.value == n
