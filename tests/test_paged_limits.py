"""The largest calls of the paged K/V cache's C ABI, by its host checks (no GPU)."""
import ctypes

from test_paged_cache import L, OK, P, SHAPE  # noqa: F401  (L: the fixture)


def test_more_workgroups_than_a_launch_holds(L):
    """2^24 workgroups of 256 threads, or more, are refused before any launch."""
    def append(N, H, D):
        return L.od_page_append(P, H * D, D, P, H * D, D, P, P, P, P, 4, 16, P, 3, 3, P, P, 2, N, H, D, None)
    assert append(2 ** 29, 2, 64) == append(2 ** 28, 1, 256) == append(2 ** 27, 2, 128) == SHAPE

    def read(T, H, D, form):
        return L.od_page_read(P, P, P, P, 4, 16, P, 3, 3, P, 2, T, H, D, form, P, P, P, P, None)
    assert read(2 ** 28, 2, 64, 0) == read(2 ** 27, 1, 256, 0) == read(2 ** 26, 1, 128, 1) == read(2 ** 28, 2, 64, 2) == SHAPE


def test_no_splits_where_the_merge_does_not_fit(L):
    """The merge of key splits has a workgroup a token: a call of 2^24 tokens or more is not split, whatever its bounds say (bf16
    pages: no image)."""
    n = ctypes.c_int64(-1)
    for new in (1, 1000):
        assert L.od_paged_attn_ws_of(1, 2 ** 24, 4, 4, 64, new, 100000, 0, ctypes.byref(n)) == OK and n.value == 0
        assert L.od_paged_attn_ws_of(1, 2 ** 24 - 1, 4, 4, 64, new, 100000, 0, ctypes.byref(n)) == OK and n.value > 0
