"""Beam search calls at the ends of what they take."""
import pytest

pytestmark = pytest.mark.gpu


def test_streams_of_another_device_are_refused(device):
    """A stream of another device: nothing is made or launched."""
    import torch
    import radx_amd
    from test_beam_streams_cpu import Stream
    other = Stream(0, 1)
    sel = radx_amd.BeamSelector(1, 4, 100, 4)
    steps = torch.zeros(3, 1, 4, dtype=torch.int32, device=device)
    for call in (lambda: sel.select(torch.zeros(4, 100, device=device), torch.zeros(1, 4, device=device), 4, stream=other),
                 lambda: radx_amd.beam_reorder(torch.zeros(4, 3, device=device), steps[0], stream=other),
                 lambda: radx_amd.beam_backtrace(steps, steps, stream=other)):
        with pytest.raises(ValueError, match="the stream is of"):
            call()
    sel.close()
