"""How the states of a reordering are cut into pieces, for tensors whose dimensions do not lie in memory in their
order (no GPU needed)."""
import itertools

import numpy as np
import pytest
import torch

from radx_amd.beam import _pieces


def cut(t, row_dim=0, length_dim=None, d=None):
    d = t if d is None else d
    return _pieces(t.shape, t.stride(), d.stride(), t.element_size(), row_dim, length_dim)


def bytes_of(origin_row, outer_strides, outer, unit, units):
    """The bytes of a row, by their distance from its first."""
    places = [o * outer_strides[0] + p * outer_strides[1] for o in range(outer[0]) for p in range(outer[1])]
    return np.add.outer(np.array(places), np.arange(unit * units)).reshape(-1) + origin_row


def elements_of(shape, strides, size, row_dim):
    """The same, from the tensor's own strides."""
    at = np.zeros(1, np.int64)
    for i, (n, s) in enumerate(zip(shape, strides)):
        if i != row_dim:
            at = np.add.outer(at, np.arange(n) * s * size).reshape(-1)
    return np.add.outer(at, np.arange(size)).reshape(-1)


@pytest.mark.parametrize("shape,order,row_dim,length_dim,want", [
    # images whose channels are innermost: a row is one block
    ((8, 16, 16, 4), (0, 3, 1, 2), 0, None, ((1, 1), 2048, 1)),
    # a matrix for each head, transposed
    ((8, 4, 32, 64), (0, 1, 3, 2), 0, None, ((1, 1), 16384, 1)),
    # [rows, positions, heads, width] seen as [rows, heads, positions, width]: a position is heads x width elements
    ((8, 40, 3, 16), (0, 2, 1, 3), 0, 2, ((1, 1), 96, 40)),
    # [rows, heads, positions, width] seen as [rows, positions, heads, width]: a piece for each head
    ((8, 3, 40, 16), (0, 2, 1, 3), 0, 1, ((1, 3), 32, 40)),
    # one position: all of the row
    ((8, 3, 1, 16), (0, 1, 2, 3), 0, 2, ((1, 1), 96, 1)),
])
def test_dimensions_are_taken_as_they_lie_in_memory(shape, order, row_dim, length_dim, want):
    t = torch.zeros(shape, dtype=torch.bfloat16).permute(order)
    _, _, src_outer, dst_outer, outer, unit, units = cut(t, row_dim, length_dim)
    assert (outer, unit, units) == want and src_outer == dst_outer


@pytest.mark.parametrize("order", list(itertools.permutations(range(4))))
@pytest.mark.parametrize("view", [lambda t: t, lambda t: t[:, :, 1:5], lambda t: t[:, :, :, 2:], lambda t: t[:, 1:3, ::2]])
def test_a_row_s_bytes_are_its_own(order, view):
    """Whatever the order, the pieces are the bytes that the tensor's strides name, each once, in source and target alike.  In
    place no such row is scattered over more than two strided dimensions; between two orders it may be, which is refused."""
    t = view(torch.zeros(6, 3, 7, 5)).permute(order)
    row_dim = order.index(0)
    into = torch.zeros(t.shape)
    for d in (t, into):
        try:
            _, _, src_outer, dst_outer, outer, unit, units = cut(t, row_dim, None, d)
        except ValueError as e:
            assert d is into and "scattered" in str(e)
            continue
        src, dst = bytes_of(0, src_outer, outer, unit, units), bytes_of(0, dst_outer, outer, unit, units)
        want = np.stack([elements_of(t.shape, t.stride(), 4, row_dim), elements_of(d.shape, d.stride(), 4, row_dim)])
        got = np.stack([src, dst])
        assert np.array_equal(got[:, np.argsort(dst)], want[:, np.argsort(want[1])])


def test_a_position_s_bytes_have_to_lie_together():
    t = torch.zeros(8, 40, 3, 16)
    with pytest.raises(ValueError, match="contiguous"):
        cut(t[:, :, :2].transpose(1, 2), 0, 2)
    with pytest.raises(ValueError, match="contiguous"):  # positions outermost
        cut(torch.zeros(40, 8, 16), 1, 0)
