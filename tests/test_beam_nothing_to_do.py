"""A cache reorder without work is a call that does nothing, not an error (and needs no device)."""
import ctypes as C

import pytest

import axon_hip as H


@pytest.mark.parametrize("field", ["n_groups", "n_regions", "max_len"])
def test_a_reorder_without_work(field):
    """Each size 0 alone, the others as in a call that has work, and no memory to touch."""
    a = H.CacheReorderArgs()
    a.n_groups, a.n_beams, a.n_regions, a.region_stride, a.unit_positions, a.unit_bytes, a.max_len = 1, 4, 2, 640, 1, 64, 10
    with pytest.raises(H.HipError, match="null"):  # (with work the memory is asked for)
        H.call("cache_reorder", C.c_void_p(C.addressof(a)))
    setattr(a, field, 0)
    H.call("cache_reorder", C.c_void_p(C.addressof(a)))
