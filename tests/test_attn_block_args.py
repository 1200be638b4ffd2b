"""Host-side arguments of the attention block's wrappers that need no GPU: stand-ins for CUDA
tensors carry shapes and types, nothing is launched."""
import ctypes
import gc

import pytest
import torch

from gdn_18646_b200 import ops


class Stand:
    """What the checks ask of a contiguous CUDA tensor."""

    def __init__(self, shape, dtype):
        self.t = torch.empty(shape, dtype=dtype)
        self.is_cuda, self.dtype, self.shape = True, dtype, self.t.shape

    def __getattr__(self, name):
        return getattr(self.t, name)


def _spec(positions=(3, 10), pairs=32, sections=(16, 8, 8), T=10):
    return ops._rope_spec(Stand(positions, torch.int32), Stand((pairs,), torch.float32), sections, "half", T)


def test_the_sections_live_as_long_as_the_spec():
    spec = _spec()
    for i in range(200):                                        # other specs push the array out of the cache
        ops._int_array((i, 32 - i, 7))
    gc.collect()
    junk = [(ctypes.c_int * 3)(-7, -7, -7) for _ in range(2000)]
    assert list((ctypes.c_int * 3).from_address(spec.sections)) == [16, 8, 8], len(junk)


@pytest.mark.parametrize("shape,sections,T", [((10, 3), (16, 8, 8), 10), ((30,), (16, 8, 8), 10), ((2, 3), (10, 11, 11), 2),
                                              ((3, 11), (16, 8, 8), 10), ((2, 10), (32,), 10), ((4, 5, 2), (16, 16), 20)])
def test_positions_of_another_order_are_refused(shape, sections, T):
    with pytest.raises(RuntimeError, match="positions"):
        _spec(shape, sections=sections, T=T)


@pytest.mark.parametrize("shape,sections,T", [((3, 10), (16, 8, 8), 10), ((3, 2, 5), (16, 8, 8), 10), ((10,), (32,), 10),
                                              ((1, 10), (32,), 10), ((2, 5), (32,), 10), ((2, 0), (16, 16), 0)])
def test_positions_by_axis_are_taken(shape, sections, T):
    spec = _spec(shape, sections=sections, T=T)
    assert (spec.positions_ld, spec.axes, spec.rot) == (T, len(sections), 64)
