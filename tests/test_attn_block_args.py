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


def _attention_args(monkeypatch, **kw):
    """The C arguments of a call of one token over 100 positions."""
    taken = []
    monkeypatch.setattr(ops._lib, "call", lambda *a: taken.append(a))
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    q = Stand((1, 4, 64), torch.bfloat16)
    cache = [Stand((8, 16, 2, 64), torch.bfloat16) for _ in range(2)]
    ops.paged_attention(q, *cache, Stand((1, 8), torch.int32), Stand((2,), torch.int32), Stand((1,), torch.int32), out=q,
                        **dict(dict(max_q=1, max_kv=100), **kw))
    (name, *args), = taken
    return dict(zip("q q_ld cache cu kv out lse B T Hq max_q max_kv causal window".split(), args))


@pytest.mark.parametrize("name", ["max_q", "max_kv", "window"])
@pytest.mark.parametrize("value,taken", [(2 ** 32 + 1, 2 ** 31 - 1), (2 ** 31, 2 ** 31 - 1), (2 ** 40, 2 ** 31 - 1), (-2 ** 32 + 1, -1),
                                         (-1, -1), (7, 7), (0, 0)])
def test_sizes_past_32_bits_keep_their_order(monkeypatch, name, value, taken):
    """Not their low 32 bits: 2^32 + 1 would be a bound of one position."""
    assert _attention_args(monkeypatch, **{name: value})[name] == taken
    assert ops.paged_attention_workspace(1, 1, 4, 2, 64, **{"max_q": 1, "max_kv": 100, name: value}) == \
        ops.paged_attention_workspace(1, 1, 4, 2, 64, **{"max_q": 1, "max_kv": 100, name: taken})


@pytest.mark.parametrize("rows", [2 ** 31, 2 ** 32 + 1])
def test_more_rows_than_an_int_are_refused(rows):
    y = type("Rows", (), dict(dtype=torch.bfloat16, is_cuda=True, shape=torch.Size((rows, 8)), is_contiguous=lambda s: True,
                              numel=lambda s: rows * 8, dim=lambda s: 2))()
    with pytest.raises(RuntimeError, match="rows"):
        ops.block_norm(y, y)
    with pytest.raises(RuntimeError, match="rows"):
        ops.block_norm_backward(y, y, y)
