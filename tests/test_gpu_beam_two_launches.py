"""Selections whose join is a launch of its own (many rows, many lists or many places), and joins with more equal
scores than are ranked at once: beams that have ended, rows that offer nothing, handles with an earlier call's entries.
Within a beam the order is exact by contract, and here it is asked for exactly."""
import numpy as np
import pytest

from test_gpu_beam import DTYPES, check_best, make_logits, on, plain_best, plain_scores, run_select, torch_dtype, words_of

pytestmark = pytest.mark.gpu

# batch, beams, vocab, k.  One launch takes at most 1024 slices (of 4096 or 8192 elements), 128 lists and 4096 entries an
# item, and k <= 64; in the other form a thread holds the join's entries in registers where there are few.
CALLS = [(4, 5, 6007, 10), (3, 4, 5003, 100), (2, 64, 3001, 128), (300, 4, 2003, 8), (1, 64, 9001, 64), (1, 9, 120007, 70)]


def check_within_beams(got, x, scores, vocab):
    """The places of one beam hold its best tokens, without a gap: logit down, token up.  (A finished beam has one.)"""
    _, p, t = got[:3]
    for b in range(p.shape[0]):
        for i in np.unique(p[b][p[b] >= 0]):
            tokens = t[b][p[b] == i]
            offered = np.flatnonzero(scores[b, i] > -np.inf)
            first = offered[np.argsort(-x[b, i, offered], kind="stable")[:len(tokens)]]
            assert np.array_equal(tokens, first), (b, i)


def full_handle(radx_amd, batch, beams, vocab, k, dtype, device):
    """A selector whose scratch holds the entries of a call with far better logits."""
    sel = radx_amd.BeamSelector(batch, beams, vocab, k)
    logits, _ = make_logits(batch, beams, vocab, dtype, device, seed=99)
    run_select(sel, logits + 1000.0, on(np.zeros((batch, beams), np.float32), device), k, normalize=False)
    return sel


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("call", CALLS, ids=str)
def test_order_within_a_beam_is_exact(device, call, dtype):
    import radx_amd
    batch, beams, vocab, k = call
    logits, x = make_logits(batch, beams, vocab, dtype, device, seed=vocab)
    cum = (-np.random.default_rng(k).random((batch, beams))).astype(np.float32)
    sel = full_handle(radx_amd, batch, beams, vocab, k, dtype, device)
    got = run_select(sel, logits, on(cum, device), k)
    scores = plain_scores(x, cum)
    check_best(got, scores, x, k, vocab)
    check_within_beams(got, x, scores, vocab)
    sel.close()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("call", CALLS, ids=str)
def test_finished_beams(device, call, dtype):
    import torch
    import radx_amd
    batch, beams, vocab, k = call
    end = 17
    logits, x = make_logits(batch, beams, vocab, dtype, device, seed=8, spread=1.0)
    rng = np.random.default_rng(2)
    cum = (-8.0 * rng.random((batch, beams))).astype(np.float32)
    cum[rng.random((batch, beams)) < 0.1] = -np.inf
    ended = rng.random((batch, beams)) < 0.5
    if batch > 2:
        ended[0], ended[1] = False, True
    logits[torch.from_numpy(ended.reshape(-1)).to(device)] = float("nan")
    x[ended] = 0.0
    live = np.argwhere(~ended & np.isfinite(cum))[0]
    logits[live[0] * beams + live[1], end] = x[live[0], live[1], end] = 30.0
    sel = full_handle(radx_amd, batch, beams, vocab, k, dtype, device)
    got = run_select(sel, logits, on(cum, device), k, finished=on(ended, device), end_token=end)
    scores = plain_scores(x, cum, finished=ended, end_token=end)
    check_best(got, scores, x, k, vocab)
    check_within_beams(got, x, scores, vocab)
    flags = np.take_along_axis(ended, np.maximum(got[1], 0), 1) | (got[2] == end)
    assert np.array_equal(got[3], flags & (got[1] >= 0))
    sel.close()


@pytest.mark.parametrize("call", CALLS, ids=str)
def test_rows_that_offer_nothing(device, call):
    """A NaN or +inf in a row, nothing but -inf, a mask that leaves nothing, a cum score that is no number."""
    import radx_amd
    batch, beams, vocab, k = call
    for dtype in DTYPES:
        logits, x = make_logits(batch, beams, vocab, dtype, device, seed=3)
        rng = np.random.default_rng(4)
        cum = (-rng.random((batch, beams))).astype(np.float32)
        allowed = rng.random((batch * beams, vocab)) < 0.5
        kinds = rng.integers(0, 9, batch * beams)
        for row, kind in enumerate(kinds):
            at = int(rng.integers(vocab))
            if kind < 2:
                allowed[row, at] = True
                value = (np.nan, np.inf)[kind]
                logits[row, at] = value
                x[row // beams, row % beams, at] = value
            elif kind == 2:
                logits[row] = -np.inf
                x[row // beams, row % beams] = -np.inf
            elif kind == 3:
                allowed[row] = False
            elif kind < 7:
                cum[row // beams, row % beams] = (np.nan, np.inf, -np.inf)[kind - 4]
        sel = full_handle(radx_amd, batch, beams, vocab, k, dtype, device)
        full = allowed.reshape(batch, beams, vocab)
        for normalize in (True, False):
            got = run_select(sel, logits, on(cum, device), k, allowed=on(words_of(allowed), device), normalize=normalize)
            scores = plain_scores(x, cum, allowed=full, normalize=normalize)
            check_best(got, scores, np.nan_to_num(x, nan=0.0), k, vocab, normalize)
            check_within_beams(got, x, scores, vocab)
        cum[:] = -np.inf
        got = run_select(sel, logits, on(cum, device), k)
        assert np.all(got[0] == -np.inf) and np.all(got[1] == -1) and np.all(got[2] == -1)
        sel.close()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,beams,vocab,k", [(2, 60, 1001, 64), (2, 64, 1001, 128), (1, 20, 30011, 64), (1, 40, 30011, 100)])
@pytest.mark.parametrize("share", [0.0, 0.3, 1.0])
def test_more_equal_scores_than_are_ranked_at_once(device, batch, beams, vocab, k, share, dtype):
    """Every entry of every list, and every finished beam, at one of two scores: the lists are joined a few at a time.  Scores
    are given, so every one is exact."""
    import torch
    import radx_amd
    rng = np.random.default_rng(beams)
    ended = rng.random((batch, beams)) < share
    cum = (-1.0 * rng.integers(0, 2, (batch, beams))).astype(np.float32)
    logits = torch.zeros(batch * beams, vocab, device=device, dtype=torch_dtype(dtype))
    x = np.zeros((batch, beams, vocab))
    sel = full_handle(radx_amd, batch, beams, vocab, k, dtype, device)
    end = vocab - 1
    got = run_select(sel, logits, on(cum, device), k, normalize=False, finished=on(ended, device), end_token=end)
    want = plain_best(plain_scores(x, cum, finished=ended, end_token=end, normalize=False), x, k)
    assert np.array_equal(got[0], want[0].astype(np.float32)) and np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
    flags = np.take_along_axis(ended, np.maximum(got[1], 0), 1) | (got[2] == end)
    assert np.array_equal(got[3], flags & (got[1] >= 0))
    sel.close()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [4, 64, 128])
def test_what_is_not_finite_in_a_long_slice(device, dtype, k):
    """A workgroup takes a whole row of ten tiles; NaN and +inf in the first tile, in a later one and in the last, alone and
    many, with candidates counted by their distance from the first tile's largest value."""
    import torch
    import radx_amd
    batch, beams, tile = 256, 4, 4096 if dtype == "f32" else 8192
    vocab = 9 * tile + 77
    g = torch.Generator(device=device).manual_seed(k)
    x = torch.randn((batch * beams, vocab), generator=g, device=device).to(torch_dtype(dtype))
    nan, inf = float("nan"), float("inf")
    x[0, 5] = nan
    x[1, 4 * tile + 9] = inf
    x[2, vocab - 1] = nan
    x[3, :3 * tile] = -inf
    x[4, 3 * tile:4 * tile] = nan
    x[5, :] = inf
    x[6, ::3] = -nan
    x[7, 8 * tile:8 * tile + 600] = inf
    x[8, 0] = inf
    x[9, tile:] = -inf
    x[10, :] = nan
    x[11, :] = torch.finfo(x.dtype).min
    cum = -torch.rand((batch, beams), generator=g, device=device)
    sel = full_handle(radx_amd, batch, beams, vocab, k, dtype, device)
    for normalize in (True, False):
        got = run_select(sel, x, cum, k, normalize=normalize)
        items = [0, 1, 2, 3]
        xv = x.view(batch, beams, vocab)[items].double().cpu().numpy()
        scores = plain_scores(xv, cum.cpu().numpy()[items], normalize=normalize)
        check_best([part[items] for part in got], scores, np.nan_to_num(xv, nan=0.0), k, vocab, normalize)
        check_within_beams([part[items] for part in got], xv, scores, vocab)
    sel.close()
