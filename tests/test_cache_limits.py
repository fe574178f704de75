"""Calls of the cache that no single launch covers are refused on the host, before any device call."""
import ctypes

from if_i_could_turn_back_time_amd import _capi as C
from test_cache_abi import P, SHAPE, _cache, _seqs


def test_more_threads_than_a_launch_has():
    L, r = C.lib(), ctypes.byref
    wide = _cache(heads=4096, head_dim=256)
    one = _seqs(seqs=65535, tokens=65535)
    assert L.fb_cache_append(r(wide), r(one), P, 1 << 20, 256, P, 1 << 20, 256, 0, None) == SHAPE
    many = _seqs(cu=P, seqs=65535, tokens=500000, max_new=20)
    for w in (None, P):
        assert L.fb_cache_attention(r(wide), r(many), P, 1 << 20, 256, 4096, 0, 1.0, P, P, w, 128, 128,
                                    128, P, 1 << 60, None) == SHAPE
    cut = _cache(page=1 << 24)
    assert L.fb_cache_evict(r(cut), r(_seqs()), P, 200, 100, 100, 0x7FFFFFFF, 2, P, 128, 128, P, P, P,
                            None) == SHAPE
