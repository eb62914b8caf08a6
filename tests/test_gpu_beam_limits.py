"""Beam search calls at the ends of what they take."""
import numpy as np
import pytest

from test_gpu_beam import on

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


def test_select_of_the_most_items(device):
    """2^20 items of four beams, which share a row of logits.  Numbers are small multiples of 1/64, so that scores are
    exact, and tie between beams."""
    import torch
    import radx_amd
    batch, beams, vocab, k = 1 << 20, 4, 10, 3
    g = torch.Generator(device=device).manual_seed(1)
    row = torch.randperm(vocab, generator=g, device=device).float().reshape(1, vocab) / 64
    cum = -torch.randint(0, 30, (batch, beams), generator=g, device=device).float() / 64
    sel = radx_amd.BeamSelector(batch, beams, vocab, k)
    scores, parents, tokens = sel.select(row.expand(batch * beams, vocab), cum, k, normalize=False)
    best, at = (cum.unsqueeze(2) + row).reshape(batch, beams * vocab).sort(dim=1, descending=True, stable=True)
    assert torch.equal(scores, best[:, :k])
    assert torch.equal(parents, (at[:, :k] // vocab).int()) and torch.equal(tokens, (at[:, :k] % vocab).int())
    sel.close()


def test_reorder_of_the_most_items(device):
    import torch
    import radx_amd
    batch, beams, width = 65535, 3, 5
    g = torch.Generator(device=device).manual_seed(2)
    state = torch.randint(0, 1 << 30, (batch * beams, width), generator=g, device=device, dtype=torch.int32)
    parents = torch.randint(-1, beams + 1, (batch, beams), generator=g, device=device, dtype=torch.int32)
    place = torch.arange(beams, device=device)
    source = torch.where((parents >= 0) & (parents < beams), parents.long(), place) + torch.arange(batch, device=device).unsqueeze(1) * beams
    want = state[source.reshape(-1)]
    radx_amd.beam_reorder(state, parents)
    assert torch.equal(state, want)


def test_backtrace_of_the_most_items(device):
    import torch
    import radx_amd
    total, batch, k = 7, 65535, 4
    g = torch.Generator(device=device).manual_seed(3)
    tokens = torch.randint(0, 1 << 30, (total, batch, k), generator=g, device=device, dtype=torch.int32)
    parents = torch.randint(0, k, (total, batch, k), generator=g, device=device, dtype=torch.int32)
    steps = torch.randint(0, total + 1, (batch,), generator=g, device=device, dtype=torch.int32)
    got = radx_amd.beam_backtrace(tokens, parents, steps=steps)
    place = torch.arange(k, device=device).expand(batch, k)
    for t in range(total - 1, -1, -1):
        live = (t < steps).unsqueeze(1)
        assert torch.equal(got[:, :, t], torch.where(live, tokens[t].gather(1, place), -1))
        place = torch.where(live, parents[t].gather(1, place).long(), place)


@pytest.mark.parametrize("ends", [None, (1 << 24) - 70000])
def test_backtrace_of_the_most_steps(device, ends):
    """Two beams whose places a step keeps or exchanges: the place at a step is the sum of the exchanges behind it."""
    import radx_amd
    total = (1 << 24) - 1
    last = total if ends is None else ends
    rng = np.random.default_rng(4)
    change = rng.integers(0, 2, total, dtype=np.int32)
    tokens = rng.integers(0, 1 << 30, (total, 1, 2), dtype=np.int32)
    parents = np.stack([change, 1 - change], 1).reshape(total, 1, 2)
    steps = None if ends is None else on(np.array([ends], np.int32), device)
    got = radx_amd.beam_backtrace(on(tokens, device), on(parents, device), steps=steps).cpu().numpy()
    behind = np.concatenate([np.bitwise_xor.accumulate(change[1:last][::-1])[::-1], [0]])
    for j in range(2):
        assert np.array_equal(got[0, j, :last], tokens[np.arange(last), 0, behind ^ j])
        assert (got[0, j, last:] == -1).all()


def test_captured_reorder_and_backtrace(device):
    """More states than one launch takes, with lengths, and the sequences with and without an output of the caller's, replayed
    with other inputs and eager work in between."""
    import torch
    import radx_amd
    batch, beams, total = 3, 4, 50
    g = torch.Generator(device=device).manual_seed(5)
    make = [lambda i=i: torch.randn(batch * beams, 2, 9 + i % 5, 8, generator=g, device=device) for i in range(30)]
    states, eager = [m() for m in make], None
    parents = torch.zeros(batch, beams, dtype=torch.int32, device=device)
    lengths = torch.zeros(batch, dtype=torch.int32, device=device)
    tokens, ways = (torch.zeros(total, batch, beams, dtype=torch.int32, device=device) for _ in range(2))
    steps = torch.zeros(batch, dtype=torch.int32, device=device)
    record = torch.full((batch, beams, total), -5, dtype=torch.int32, device=device)

    def calls(states, record):
        radx_amd.beam_reorder(states, parents, lengths=lengths, length_dim=2)
        return radx_amd.beam_backtrace(tokens, ways, steps=steps), radx_amd.beam_backtrace(tokens, ways, steps=steps, out=record)

    calls([s.clone() for s in states], record.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made, _ = calls(states, record)
    for _ in range(4):
        for t, low, high in ((parents, -1, beams + 1), (lengths, -1, 15), (tokens, 0, 1000), (ways, -1, beams + 1), (steps, -1, total + 3)):
            t.copy_(torch.randint(low, high, t.shape, generator=g, device=device, dtype=torch.int32))
        eager, again = [s.clone() for s in states], record.clone()
        want, _ = calls(eager, again)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(s, e) for s, e in zip(states, eager))
        assert torch.equal(made, want) and torch.equal(record, again)
        torch.ones(100000, device=device).sum().item()


def test_calls_that_overlapped_leave_the_handle_as_it_was(device):
    """Two selections of one handle on two streams, in no order: their results are nobody's, as documented, but later calls are
    right again, whichever of the handle's counters they take."""
    import torch
    import radx_amd
    from test_gpu_beam import check_best, make_logits, plain_scores, run_select
    sel = radx_amd.BeamSelector(8, 4, 131072, 8)
    streams = [torch.cuda.Stream() for _ in range(2)]
    calls = []
    for batch, beams, vocab, k, dtype in ((4, 4, 131072, 8, "bf16"), (8, 4, 32000, 8, "bf16")):
        logits, x = make_logits(batch, beams, vocab, dtype, device, seed=vocab)
        cum = (-np.random.default_rng(k).random((batch, beams))).astype(np.float32)
        calls.append((logits, x, cum, on(cum, device), k))
    torch.cuda.synchronize()
    outs = [sel.select(logits, dev_cum, k) for logits, _, _, dev_cum, k in calls]
    work = torch.zeros(1 << 26, device=device)
    for _ in range(25):
        for _ in range(4):
            work.add_(1.0)  # both streams wait for this, so that their calls start together
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for _ in range(3):  # fewer in flight than the handle has sets of counters
            for s, (logits, _, _, dev_cum, k), out in zip(streams, calls, outs):
                sel.select(logits, dev_cum, k, out=out, stream=s)
        torch.cuda.synchronize()
    want = []
    for turn in range(40):
        logits, x, cum, dev_cum, k = calls[turn % 2]
        got = run_select(sel, logits, dev_cum, k)
        if turn < 2:
            check_best(got, plain_scores(x, cum), x, k, x.shape[2])
            want.append(got)
        assert all(np.array_equal(g, w) for g, w in zip(got, want[turn % 2])), turn
    sel.close()
