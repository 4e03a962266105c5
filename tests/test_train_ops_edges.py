"""Further calls that the training operators refuse, on the CPU: every check comes before anything is enqueued."""
import ctypes as C

import pytest

from litnicelm_b200 import plugin, training

BASE = 1 << 20  # an address that nothing dereferences
EINVAL, ECUDA = -1, -2


def view(shape, dtype=0, strides=None, ptr=BASE):
    size = 2 if dtype == 2 else 4
    if strides is None:
        strides, at = [], size
        for d in reversed(shape):
            strides.insert(0, at)
            at *= d
    return plugin.DevTensor(ptr, tuple(shape), tuple(strides), dtype, 1).view()


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(plugin.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    return training._library()


def text(lib):
    return lib.litnice_b200_last_error(None).decode()


def ref(t):
    return None if t is None else C.addressof(t)


@pytest.mark.parametrize("shape,turned", [((5, 5, 20, 30), (2400, 12000, 120, 4)), ((4, 40, 40), (6400, 4, 160)),
                                          ((2, 3, 7, 80, 80), (591360, 197120, 28160, 352, 4))], ids=str)
def test_orthogonalise_in_place_wants_the_same_strides(lib, shape, turned):
    """One matrix of a call is written while another may still be read."""
    x, out = view(shape), view(shape, strides=turned)
    need = lib.litnice_b200_orthogonalise_workspace(ref(x))
    assert lib.litnice_b200_orthogonalise(ref(x), ref(out), 5, 64 * BASE, need, None) == EINVAL
    assert "out lies on x with another stride" in text(lib)
