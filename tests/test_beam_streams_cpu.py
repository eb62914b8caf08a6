"""Streams that the Python driver takes (no GPU needed)."""
import pytest
import torch  # noqa: F401  before the library

from radx_amd.beam import _stream


class Stream:
    """What is looked at of a torch.cuda.Stream."""

    def __init__(self, cuda_stream, device_index):
        self.cuda_stream, self.device_index = cuda_stream, device_index


def test_a_stream_of_the_tensors_device():
    assert _stream(Stream(4096, 1), 1) == 4096
    assert _stream(4096, 1) == 4096  # a handle alone
    assert _stream(0, 1) == 0


def test_a_stream_of_another_device_is_refused():
    with pytest.raises(ValueError, match="cuda:1, expected cuda:0"):
        _stream(Stream(4096, 1), 0)
