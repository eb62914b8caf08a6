"""Reordering of tensors whose dimensions do not lie in memory in their order."""
import numpy as np
import pytest

from test_gpu_beam import bits, fill, on, plain_reorder

pytestmark = pytest.mark.gpu

# the tensor in memory, the order in which its dimensions are seen, which of the seen ones are the rows and the positions
VIEWS = {"channels innermost": ((12, 7, 6, 5), (0, 3, 1, 2), 0, None), "a matrix transposed": ((12, 3, 17, 9), (0, 1, 3, 2), 0, None),
         "heads before positions": ((12, 40, 3, 17), (0, 2, 1, 3), 0, 2), "positions before heads": ((12, 3, 40, 16), (0, 2, 1, 3), 0, 1),
         "rows last": ((2, 12, 40, 5), (0, 2, 3, 1), 3, 1), "one position": ((12, 3, 1, 16), (0, 2, 1, 3), 0, 1)}


@pytest.mark.parametrize("name", VIEWS)
@pytest.mark.parametrize("into", [None, "alike", "contiguous"])
def test_reorder_views(device, name, into):
    import torch
    import radx_amd
    shape, order, row_dim, length_dim = VIEWS[name]
    parents = np.array([[0, 0, 1, 3], [3, 2, 1, 0], [2, 2, 2, -1]], np.int32)
    src = fill(shape, torch.float16, 5).permute(order)
    dst = fill(shape, torch.float16, 6).permute(order)
    dst = dst.contiguous() if into == "contiguous" else dst
    for lengths in ((None,) if length_dim is None or into == "contiguous" else (None, [0, 1, 40], [17, -3, 1000])):
        n = None if lengths is None else np.array(lengths, np.int32)
        dim = None if lengths is None else length_dim
        want = plain_reorder(src, (src if into is None else dst).clone(), parents, 4, n, dim, row_dim)
        got, out = src.to(device), dst.to(device)
        if name == "a matrix transposed" and into == "contiguous":  # three dimensions that follow each other differently
            with pytest.raises(ValueError, match="scattered"):
                radx_amd.beam_reorder(got, on(parents, device), into=out)
            continue
        assert got.stride() == src.stride() and out.stride() == dst.stride()
        radx_amd.beam_reorder(got, on(parents, device), into=None if into is None else out, lengths=None if n is None else on(n, device),
                              length_dim=dim, row_dim=row_dim)
        assert torch.equal(bits(got if into is None else out), bits(want)), lengths
        assert into is None or torch.equal(bits(got), bits(src))
