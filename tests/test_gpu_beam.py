"""Beam search on the GPU against plain implementations in 64 bits (numpy), written from the definitions
in include/radx_hip.h."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

DTYPES = ["f32", "bf16", "f16"]


def torch_dtype(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


# ---------------------------------------------------------------------------------------------
# selection
# ---------------------------------------------------------------------------------------------
def plain_scores(x, cum, allowed=None, finished=None, end_token=None, normalize=True):
    """[batch, beams, vocab] scores in 64 bits, -inf where nothing is offered."""
    x = np.array(x, dtype=np.float64)
    if allowed is not None:
        x[~allowed] = -np.inf
    out = np.full(x.shape, -np.inf)
    for b, i in np.ndindex(cum.shape):
        if not np.isfinite(cum[b, i]):
            continue
        if finished is not None and finished[b, i]:
            out[b, i, end_token] = cum[b, i]
            continue
        row = x[b, i]
        if np.isnan(row).any() or (row == np.inf).any() or not (row > -np.inf).any():
            continue
        out[b, i] = row + float(cum[b, i])
        if normalize:
            top = row.max()
            with np.errstate(over="ignore", invalid="ignore"):
                out[b, i] = float(cum[b, i]) + ((row - top) - math.log(math.fsum(np.exp(row - top))))
            out[b, i][row == -np.inf] = -np.inf
    return out


def plain_best(scores, x, k):
    """(scores, parents, tokens) of the k best: score down, beam up, logit down, token up."""
    batch, beams, vocab = scores.shape
    s = np.full((batch, k), -np.inf)
    p = np.full((batch, k), -1)
    t = np.full((batch, k), -1)
    for b in range(batch):
        flat = scores[b].reshape(-1)
        order = np.lexsort((np.arange(flat.size), -np.nan_to_num(x[b].reshape(-1).astype(np.float64), nan=0.0),
                            np.arange(flat.size) // vocab, -flat))[:k]
        order = order[flat[order] > -np.inf]
        s[b, :len(order)], p[b, :len(order)], t[b, :len(order)] = flat[order], order // vocab, order % vocab
    return s, p, t


def lse_bound(vocab):
    """What the kernel's log of the sum may be off by.  A term 2^(d log2 e) is the hardware's exponential, within an ulp
    (2^-23) of 2^t, of a t off by three roundings: d's, a product's and the joining fma's, 3 * 2^-24 |d| of the
    term in all; eight terms are added in three rounded additions (3 * 2^-24) and go on in 64 bits.  Over the terms,
    weighted by their size, |d| has a mean of at most log n (entropy of the softmax = log S + mean |d| <= log n, S >= 1)."""
    return (3.0 * math.log(max(vocab, 2)) + 5.0) * 2.0 ** -24


def words_of(allowed):
    """[rows, vocab] truth values as int32 words, bit v & 31 of word v >> 5."""
    rows, vocab = allowed.shape
    bits = np.zeros((rows, (vocab + 31) // 32 * 32), np.uint8)
    bits[:, :vocab] = allowed
    return np.packbits(bits, axis=1, bitorder="little").view(np.int32)


def on(a, device):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to(device)


def make_logits(batch, beams, vocab, dtype, device, seed, spread=3.0, pad=0):
    """(device tensor [rows, vocab], the values it holds as float64 [batch, beams, vocab])"""
    import torch
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((batch * beams, vocab + pad)) * spread).astype(np.float32)
    t = torch.from_numpy(x).to(torch_dtype(dtype)).to(device)
    t = t[:, :vocab] if pad else t
    return t, t.float().cpu().numpy().astype(np.float64).reshape(batch, beams, vocab)


def run_select(selector, *args, **kw):
    import torch
    out = selector.select(*args, **kw)
    torch.cuda.synchronize()
    return [o.cpu().numpy() for o in out]


def check_best(got, scores, x, k, vocab, normalize=True):
    """The places are the plain form's.  A score is rounded once (half an ulp, 2^-24 of it); two candidates may
    change places only where their scores are within twice the sum's bound of each other."""
    s, p, t = got[:3]
    want_s, want_p, want_t = plain_best(scores, x, k)
    off = lse_bound(vocab) if normalize else 0.0
    none = want_s == -np.inf
    assert np.array_equal(s == -np.inf, none) and np.array_equal(p == -1, none) and np.array_equal(t == -1, none)
    ok = ~none
    assert np.all(np.abs(s[ok] - want_s[ok]) <= np.abs(want_s[ok]) * 2.0 ** -24 + off + 1e-12)
    for b in range(s.shape[0]):
        live = ok[b]
        places = p[b][live].astype(np.int64) * vocab + t[b][live]
        assert len(set(places.tolist())) == len(places)
        true = scores[b].reshape(-1)[places]
        same = (p[b][live] == want_p[b][live]) & (t[b][live] == want_t[b][live])
        assert np.all(same | ((np.abs(true - want_s[b][live]) <= 2 * off) & (true != want_s[b][live])))


SHAPES = [(1, 1, 1, 1), (1, 1, 5, 8), (2, 3, 7, 4), (1, 4, 31, 8), (3, 2, 32, 4), (2, 5, 33, 10), (1, 2, 255, 16), (1, 64, 100, 128),
          (2, 4, 1023, 8), (1, 4, 4096, 8), (1, 3, 4097, 6), (2, 2, 8192, 4), (2, 2, 8193, 33), (1, 5, 20011, 10), (3, 8, 50001, 16),
          (1, 4, 131072, 64), (5, 1, 70001, 1), (1, 7, 40003, 128), (300, 3, 2001, 4), (4, 16, 33000, 40)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_select(device, shape, dtype):
    import radx_amd
    batch, beams, vocab, k = shape
    logits, x = make_logits(batch, beams, vocab, dtype, device, seed=vocab + k)
    cum = (-5.0 - 4.0 * np.random.default_rng(k).random((batch, beams))).astype(np.float32)
    sel = radx_amd.BeamSelector(batch, beams, vocab, k)
    for normalize in (True, False):
        got = run_select(sel, logits, on(cum, device), k, normalize=normalize)
        check_best(got, plain_scores(x, cum, normalize=normalize), x, k, vocab, normalize)
    sel.close()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,beams,vocab,k,pad", [(2, 3, 1000, 6, 1), (1, 4, 9001, 8, 7), (4, 2, 12345, 16, 55)])
def test_select_rows_of_any_pitch(device, dtype, batch, beams, vocab, k, pad):
    """Rows that begin at every alignment, with values behind them that would win."""
    import torch
    import radx_amd
    rng = np.random.default_rng(pad)
    whole = torch.full((batch * beams, vocab + pad), 1000.0)
    whole[:, :vocab] = torch.from_numpy(rng.standard_normal((batch * beams, vocab)).astype(np.float32))
    whole = whole.to(torch_dtype(dtype)).to(device)
    sel = radx_amd.BeamSelector(batch, beams, vocab + pad, k)
    cum = (-rng.random((batch, beams))).astype(np.float32)
    for start in (0, pad):
        logits = whole[:, start:vocab + start] if start == 0 else whole.flip(1)[:, start:vocab + start]
        x = logits.float().cpu().numpy().astype(np.float64).reshape(batch, beams, vocab)
        got = run_select(sel, logits, on(cum, device), k)
        check_best(got, plain_scores(x, cum), x, k, vocab)
        got3 = run_select(sel, logits.unflatten(0, (batch, beams)), on(cum, device), k)
        assert all(np.array_equal(u, v) for u, v in zip(got, got3))
    sel.close()


def test_select_one_row_for_all_beams(device):
    """The first step: one distribution behind every beam, all but the first beam at -inf; and all alike."""
    import radx_amd
    batch, beams, vocab, k = 3, 4, 5003, 9
    row, x1 = make_logits(1, 1, vocab, "bf16", device, seed=1)
    x = np.broadcast_to(x1, (batch, beams, vocab)).copy()
    cum = np.full((batch, beams), -np.inf, np.float32)
    cum[:, 0] = 0.0
    sel = radx_amd.BeamSelector(batch, beams, vocab, k)
    logits = row.expand(batch * beams, vocab)
    got = run_select(sel, logits, on(cum, device), k)
    check_best(got, plain_scores(x, cum), x, k, vocab)
    assert np.all(got[1] == 0)
    cum[:] = -1.0
    got = run_select(sel, logits, on(cum, device), k)
    # equal rows have equal sums: the four beams tie, the lower beam first
    assert np.array_equal(got[1], np.broadcast_to(np.arange(k) % beams, (batch, k)))
    check_best(got, plain_scores(x, cum), x, k, vocab)
    sel.close()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("share", [0.5, 0.02, "single", "empty rows", "nothing"])
@pytest.mark.parametrize("shared", [False, True])
def test_select_under_a_mask(device, dtype, share, shared):
    """What is masked counts for nothing, whatever it holds."""
    import torch
    import radx_amd
    batch, beams, vocab, k = 3, 4, 9005, 8
    rng = np.random.default_rng(5)
    rows = 1 if shared else batch * beams
    if share == "single":
        allowed = np.zeros((rows, vocab), bool)
        allowed[np.arange(rows), rng.integers(0, vocab, rows)] = True
    elif share == "nothing":
        allowed = np.zeros((rows, vocab), bool)
    else:
        allowed = rng.random((rows, vocab)) < (0.3 if share == "empty rows" else share)
        if share == "empty rows" and not shared:
            allowed[::2] = False
    logits, x = make_logits(batch, beams, vocab, dtype, device, seed=6)
    full = np.broadcast_to(allowed, (batch * beams, vocab)).reshape(batch, beams, vocab)
    bad = torch.from_numpy(~full.reshape(batch * beams, vocab)).to(device)
    junk = torch.tensor([float("nan"), float("inf"), float("-inf"), 500.0, torch.finfo(logits.dtype).min], device=device).to(logits.dtype)
    logits = torch.where(bad, junk[torch.arange(vocab, device=device) % 5], logits)
    cum = (-rng.random((batch, beams))).astype(np.float32)
    sel = radx_amd.BeamSelector(batch, beams, vocab, k)
    words = on(words_of(allowed), device)
    assert words.shape == (rows, (vocab + 31) // 32)
    got = run_select(sel, logits, on(cum, device), k, allowed=words)
    check_best(got, plain_scores(x, cum, allowed=full), x, k, vocab)
    sel.close()


def test_select_mask_words_with_a_pitch(device):
    import torch
    import radx_amd
    batch, beams, vocab, k = 2, 3, 4000, 6
    rng = np.random.default_rng(9)
    allowed = rng.random((batch * beams, vocab)) < 0.1
    logits, x = make_logits(batch, beams, vocab, "f16", device, seed=10)
    wide = torch.full((batch * beams, 125 + 3), -1, dtype=torch.int32, device=device)
    wide[:, :125] = on(words_of(allowed), device)
    cum = np.zeros((batch, beams), np.float32)
    sel = radx_amd.BeamSelector(batch, beams, vocab, k)
    got = run_select(sel, logits, on(cum, device), k, allowed=wide[:, :125])
    check_best(got, plain_scores(x, cum, allowed=allowed.reshape(batch, beams, vocab)), x, k, vocab)
    sel.close()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [3, 300, 20000, 70001])
@pytest.mark.parametrize("fill", ["zero", "lowest", "-inf", "lowest but few", "-inf but few", "small numbers", "falling", "rising"])
def test_select_many_ties(device, dtype, vocab, fill):
    """Rows whose values are all or mostly alike, or few different ones: ties go to the lower beam, then the lower token.
    Scores are given, so every one is exact."""
    import torch
    import radx_amd
    batch, beams, k = 2, 3, 40
    rng = np.random.default_rng(vocab)
    info = torch.finfo(torch_dtype(dtype))
    base = {"zero": 0.0, "lowest": info.min, "-inf": -np.inf, "lowest but few": info.min, "-inf but few": -np.inf}.get(fill, 0.0)
    x = np.full((batch * beams, vocab), base)
    if fill.endswith("few"):
        for r in range(batch * beams):
            x[r, rng.integers(0, vocab, 5)] = rng.integers(-4, 4, 5) * 0.5
    elif fill == "small numbers":
        x = rng.integers(-3, 4, x.shape) * 0.25
    elif fill == "falling":
        x = np.broadcast_to(-(np.arange(vocab) // 7 % 256) * 0.25, x.shape).copy()
    elif fill == "rising":
        x = np.broadcast_to((np.arange(vocab) * 256 // vocab) * 0.25, x.shape).copy()
    logits = on(x, device).to(torch_dtype(dtype))
    x = logits.double().cpu().numpy().reshape(batch, beams, vocab)
    cum = (rng.integers(-4, 0, (batch, beams)) * 0.5).astype(np.float32)
    sel = radx_amd.BeamSelector(batch, beams, vocab, k)
    got = run_select(sel, logits, on(cum, device), k, normalize=False)
    scores = plain_scores(x, cum, normalize=False)
    want = plain_best(scores, x, k)
    with np.errstate(over="ignore"):
        assert np.array_equal(got[0], want[0].astype(np.float32))
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
    # normalised: the same order within each beam, and the scores of a flat row
    got = run_select(sel, logits, on(cum, device), k)
    with np.errstate(over="ignore", invalid="ignore"):
        check_best(got, plain_scores(x, cum), x, k, vocab)
    sel.close()


@pytest.mark.parametrize("k", [1, 32, 64, 128])
def test_select_best_in_one_place(device, k):
    """All of the best values at one thread's places of a tile, and more of them than a threshold by threads expects."""
    import torch
    import radx_amd
    vocab = 40000
    x = np.random.default_rng(k).standard_normal((2, vocab)).astype(np.float32)
    # a thread's elements of a 16-bit tile of 8192: 8 adjacent ones in each quarter
    for first in (0, 8192 * 3):
        for lane in range(100, 100 + 2 * k + 3):
            for j in range(4):
                at = first + j * 2048 + (lane % 256) * 8
                x[:, at:at + 8] = 20.0 + np.random.default_rng(at).permutation(8) + (lane % 5)
    logits = torch.from_numpy(x).to(device).to(torch.bfloat16)
    xv = logits.double().cpu().numpy().reshape(1, 2, vocab)
    cum = np.array([[-1.0, -1.25]], np.float32)
    sel = radx_amd.BeamSelector(1, 2, vocab, k)
    got = run_select(sel, logits, on(cum, device), k, normalize=False)
    want = plain_best(plain_scores(xv, cum, normalize=False), xv, k)
    assert np.array_equal(got[0], want[0].astype(np.float32)) and np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
    sel.close()


def test_select_leaves_out_what_is_not_finite(device):
    """A NaN or +inf in a row, a cum score that is no number: that beam offers nothing, the others are as before."""
    import torch
    import radx_amd
    batch, beams, vocab, k = 1, 6, 17000, 12
    logits, x = make_logits(batch, beams, vocab, "f32", device, seed=3)
    cum = np.linspace(-2, -1, beams, dtype=np.float32)[None].copy()
    for row, at, value in ((0, 5, np.nan), (1, 16999, np.inf), (2, 0, -np.inf), (3, 9000, np.nan)):
        logits[row, at] = value
        x[0, row, at] = value
    cum[0, 4] = np.nan
    sel = radx_amd.BeamSelector(batch, beams, vocab, k)
    for normalize in (True, False):
        got = run_select(sel, logits, on(cum, device), k, normalize=normalize)
        assert set(got[1].reshape(-1).tolist()) <= {2, 5}
        check_best(got, plain_scores(x, cum, normalize=normalize), np.nan_to_num(x, nan=0.0), k, vocab, normalize)
    cum[:] = np.inf
    got = run_select(sel, logits, on(cum, device), k)
    assert np.all(got[0] == -np.inf) and np.all(got[1] == -1) and np.all(got[2] == -1)
    sel.close()


@pytest.mark.parametrize("flag", ["bool", "uint8"])
def test_select_finished_beams(device, flag):
    import torch
    import radx_amd
    batch, beams, vocab, k, end = 4, 5, 6007, 10, 17
    logits, x = make_logits(batch, beams, vocab, "bf16", device, seed=8, spread=1.0)
    rng = np.random.default_rng(2)
    cum = (-8.0 * rng.random((batch, beams))).astype(np.float32)
    ended = rng.random((batch, beams)) < 0.5
    ended[0], ended[1] = False, True
    logits[torch.from_numpy(ended.reshape(-1)).to(device)] = float("nan")  # a finished beam's logits are not looked at
    x[ended] = 0.0
    logits[0, end] = x[0, 0, end] = 30.0  # somebody ends now
    sel = radx_amd.BeamSelector(batch, beams, vocab, k)
    flags = on(ended if flag == "bool" else ended.astype(np.uint8) * 7, device)
    got = run_select(sel, logits, on(cum, device), k, finished=flags, end_token=end)
    assert got[3].dtype == (np.bool_ if flag == "bool" else np.uint8)
    check_best(got, plain_scores(x, cum, finished=ended, end_token=end), x, k, vocab)
    want = np.zeros((batch, k), bool)
    for b, j in np.ndindex(batch, k):
        want[b, j] = got[1][b, j] >= 0 and (ended[b, got[1][b, j]] or got[2][b, j] == end)
    assert np.array_equal(got[3].astype(bool), want) and want[0].any() and not want[0].all()
    assert np.array_equal(got[1][1] >= 0, np.arange(k) < beams)  # five candidates, ten places
    sel.close()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [300, 40001])
def test_select_subnormal_logits(device, dtype, vocab):
    """Numbers below the type's normal ones, and zeros of both signs, which are one value.  Scores are given and cum is
    0, so every one is exact."""
    import torch
    import radx_amd
    k = 20
    rng = np.random.default_rng(vocab)
    step = float(torch.finfo(torch_dtype(dtype)).smallest_normal) * 2.0 ** -7  # a number of all three types
    n = rng.integers(-100, 5, (2, vocab)).astype(np.float64)
    n[1] = np.minimum(n[1], -0.0)  # the second beam has zeros of both signs at the top
    n[1, ::3][n[1, ::3] == 0] = 0.0
    logits = torch.from_numpy(n * step).to(torch_dtype(dtype))
    x = logits.double().numpy().reshape(1, 2, vocab)
    assert np.array_equal(x.reshape(2, vocab), n * step)
    sel = radx_amd.BeamSelector(1, 2, vocab, k)
    cum = np.zeros((1, 2), np.float32)
    got = run_select(sel, logits.to(device), on(cum, device), k, normalize=False)
    want = plain_best(plain_scores(x, cum, normalize=False) + 0.0, x, k)
    assert np.array_equal(got[0], want[0].astype(np.float32))
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
    sel.close()


def test_select_extreme_logits(device):
    """Float32 logits over the type's whole range, and cum scores far apart."""
    import torch
    import radx_amd
    vocab, k = 3001, 8
    rng = np.random.default_rng(12)
    x = rng.standard_normal((4, vocab)).astype(np.float32)
    x[0] *= 5e37
    x[1] *= 1e-30
    x[2, :] = np.finfo(np.float32).min
    x[3, :7] = np.finfo(np.float32).max
    cum = np.array([[-1.0, -2.0, -3.0, -1e6]], np.float32)
    sel = radx_amd.BeamSelector(1, 4, vocab, k)
    xv = x.astype(np.float64).reshape(1, 4, vocab)
    got = run_select(sel, on(x, device), on(cum, device), k)
    check_best(got, plain_scores(xv, cum), xv, k, vocab)
    sel.close()


@pytest.mark.parametrize("kind", ["clustered", "falling", "rising", "few allowed in one place", "sixteen equal rows"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [3, 16, 100])
def test_select_lists_and_queues(device, kind, dtype, k):
    """Rows of many tiles whose best values come all at once, ever better, or in few threads' hands: the lists' and
    queues' limits.  Scores are given, so every one is exact."""
    import torch
    import radx_amd
    batch, beams, vocab = 1, 16, 150001
    rng = np.random.default_rng(k)
    x = rng.standard_normal((beams, vocab)).astype(np.float32)
    if kind == "clustered":
        for at in (0, 8190, 65536, vocab - 700):
            x[:, at:at + 700] += 6.0
    elif kind == "falling":
        x = np.broadcast_to(-np.arange(vocab, dtype=np.float32) / 1000, x.shape) + x * 1e-3
    elif kind == "rising":
        x = np.broadcast_to(np.arange(vocab, dtype=np.float32) / 5000, x.shape) + x * 1e-3
    elif kind == "sixteen equal rows":
        x[:] = x[0]
    allowed = None
    if kind == "few allowed in one place":
        allowed = np.zeros((beams, vocab), bool)
        allowed[:, 99000:99000 + 3000] = True
    logits = torch.from_numpy(np.ascontiguousarray(x)).to(device).to(torch_dtype(dtype))
    xv = logits.double().cpu().numpy().reshape(batch, beams, vocab)
    cum = (-np.arange(beams) % 4 * 0.25).astype(np.float32)[None].copy()
    sel = radx_amd.BeamSelector(batch, beams, vocab, k)
    words = None if allowed is None else on(words_of(allowed), device)
    got = run_select(sel, logits, on(cum, device), k, allowed=words, normalize=False)
    full = None if allowed is None else allowed[None]
    want = plain_best(plain_scores(xv, cum, allowed=full, normalize=False), xv, k)
    assert np.array_equal(got[0], want[0].astype(np.float32)) and np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
    got = run_select(sel, logits, on(cum, device), k, allowed=words)
    check_best(got, plain_scores(xv, cum, allowed=full), xv, k, vocab)
    sel.close()


@pytest.mark.parametrize("kind", ["normal", "rising", "falling", "few values", "late", "first tile empty", "under a mask"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [4, 64, 128])
def test_select_long_slices(device, kind, dtype, k):
    """So many rows that one workgroup takes a whole one of ten tiles (of 4096 elements, 8192 of the 16-bit types), whose
    threshold rises on the way.  Three items are compared."""
    import torch
    import radx_amd
    batch, beams, tile = 256, 4, 4096 if dtype == "f32" else 8192
    vocab = 9 * tile + 77
    g = torch.Generator(device=device).manual_seed(k)
    x = torch.randn((batch * beams, vocab), generator=g, device=device)
    token = torch.arange(vocab, device=device)
    allowed = None
    if kind == "rising":
        x = x * 1e-2 + token / vocab * 30.0
    elif kind == "falling":
        x = x * 1e-2 - token / vocab * 30.0
    elif kind == "few values":
        x = (x * 2).round() * 0.5
    elif kind == "late":
        x[:, 7 * tile:8 * tile:5] += 8.0
    elif kind == "first tile empty":
        x[:, :tile] = -math.inf
    elif kind == "under a mask":
        allowed = np.random.default_rng(k).random((1, vocab)) < 0.02
    x = x.to(torch_dtype(dtype))
    cum = -torch.rand((batch, beams), generator=g, device=device)
    sel = radx_amd.BeamSelector(batch, beams, vocab, k)
    got = run_select(sel, x, cum, k, allowed=None if allowed is None else on(words_of(allowed), device))
    items = [0, 100, 255]
    xv = x.view(batch, beams, vocab)[items].double().cpu().numpy()
    full = None if allowed is None else np.broadcast_to(allowed, xv.shape)
    check_best([part[items] for part in got], plain_scores(xv, cum.cpu().numpy()[items], allowed=full), xv, k, vocab)
    sel.close()


def test_select_past_32_bits(device):
    """Rows that begin more than 4 GiB into the logits."""
    import torch
    import radx_amd
    batch, beams, vocab, k = 9000, 2, 131072, 4
    logits = torch.zeros(batch * beams, vocab, dtype=torch.bfloat16, device=device)
    cum = torch.zeros(batch, beams, device=device)
    at = torch.arange(batch, device=device) * 7 % vocab
    logits[torch.arange(batch, device=device) * 2 + 1, at] = 30.0
    sel = radx_amd.BeamSelector(batch, beams, vocab, k)
    scores, parents, tokens = sel.select(logits, cum, k, normalize=False)
    assert bool((tokens[:, 0] == at).all()) and bool((parents[:, 0] == 1).all()) and bool((scores[:, 0] == 30.0).all())
    assert bool((scores[:, 1:] == 0.0).all()) and bool((parents[:, 1:] == 0).all())
    assert bool((tokens[:, 1:] == torch.arange(k - 1, device=device)).all())
    sel.close()
    del logits
    torch.cuda.empty_cache()


def test_select_very_many_rows(device):
    """More rows than slices are wanted, each of several tiles, all of them one row in memory."""
    import torch
    import radx_amd
    batch, beams, vocab, k = 40000, 64, 20000, 1
    row = torch.zeros(1, vocab, dtype=torch.bfloat16, device=device)
    row[0, 19999] = 4.0
    cum = torch.zeros(batch, beams, device=device)
    cum[:, 63] = 1.0
    sel = radx_amd.BeamSelector(batch, beams, vocab, k)
    scores, parents, tokens = sel.select(row.expand(batch * beams, vocab), cum, k, normalize=False)
    assert bool((tokens == 19999).all()) and bool((parents == 63).all()) and bool((scores == 5.0).all())
    sel.close()


def test_select_two_graphs_one_handle(device):
    """Two captured graphs of one handle, replayed in turn on one stream with eager calls between them."""
    import torch
    import radx_amd
    batch, beams, k = 2, 4, 8
    sel = radx_amd.BeamSelector(batch, beams, 60000, k)
    graphs = []
    for vocab in (9001, 60000):
        logits, x = make_logits(batch, beams, vocab, "bf16", device, seed=vocab)
        cum = (-np.random.default_rng(vocab).random((batch, beams))).astype(np.float32)
        dev_cum = on(cum, device)
        sel.select(logits, dev_cum, k)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = sel.select(logits, dev_cum, k)
        graphs.append((g, out, logits, x, cum, dev_cum, vocab))
    for turn in range(6):
        g, out, logits, x, cum, dev_cum, vocab = graphs[turn % 2]
        for o in out:
            o.zero_()
        eager = sel.select(logits, dev_cum, k)
        g.replay()
        again = sel.select(logits, dev_cum, k)
        torch.cuda.synchronize()
        for o, e, f in zip(out, eager, again):
            assert torch.equal(o, e) and torch.equal(o, f)
        check_best([o.cpu().numpy() for o in out], plain_scores(x, cum), x, k, vocab)
    del graphs
    sel.close()


def test_select_is_the_same_every_time(device):
    """No result hangs on the order in which workgroups or atomics come."""
    import radx_amd
    batch, beams, vocab, k = 16, 8, 100003, 16
    logits, x = make_logits(batch, beams, vocab, "bf16", device, seed=4)
    cum = on((-np.random.default_rng(1).random((batch, beams))).astype(np.float32), device)
    sel = radx_amd.BeamSelector(batch, beams, vocab, k)
    first = run_select(sel, logits, cum, k)
    for _ in range(5):
        again = run_select(sel, logits, cum, k)
        assert all(np.array_equal(u, v) for u, v in zip(first, again))
    sel.close()


def test_select_one_handle_for_smaller_calls(device):
    """A handle serves every call within its limits; nothing carries over."""
    import radx_amd
    sel = radx_amd.BeamSelector(8, 16, 60000, 64)
    for batch, beams, vocab, k, dtype in ((8, 16, 60000, 64, "f32"), (1, 1, 10, 2, "bf16"), (3, 16, 59999, 5, "f16"), (8, 2, 60000, 64, "bf16"), (1, 16, 4, 64, "f32")):
        logits, x = make_logits(batch, beams, vocab, dtype, device, seed=vocab)
        cum = (-np.random.default_rng(beams).random((batch, beams))).astype(np.float32)
        got = run_select(sel, logits, on(cum, device), k)
        check_best(got, plain_scores(x, cum), x, k, vocab)
    for bad in ((9, 16, 100, 4), (1, 17, 100, 4), (1, 1, 60001, 4), (1, 1, 100, 65)):
        batch, beams, vocab, k = bad
        logits, _ = make_logits(batch, beams, vocab, "f32", device, seed=1)
        with pytest.raises(radx_amd.RadxError, match="limits"):
            sel.select(logits, on(np.zeros((batch, beams), np.float32), device), k)
    sel.close()


def test_select_refuses_tensors(device):
    import torch
    import radx_amd
    sel = radx_amd.BeamSelector(2, 4, 100, 8)
    x = torch.zeros(8, 100, device=device)
    cum = torch.zeros(2, 4, device=device)
    flags = torch.zeros(2, 4, dtype=torch.bool, device=device)
    for args, kw in (((x.double(), cum, 8), {}), ((x[:7], cum, 8), {}), ((x, cum.double(), 8), {}), ((x, cum.t(), 8), {}), ((x.t().contiguous().t(), cum, 8), {}),
                     ((x.cpu(), cum, 8), {}), ((x, cum, 8), dict(finished=flags)), ((x, cum, 8), dict(end_token=3)),
                     ((x, cum, 8), dict(finished=flags.float(), end_token=3)), ((x, cum, 8), dict(finished=flags[:1], end_token=3)),
                     ((x, cum, 8), dict(allowed=torch.zeros(8, 3, dtype=torch.int32, device=device))),
                     ((x, cum, 8), dict(allowed=torch.zeros(2, 4, dtype=torch.int32, device=device))),
                     ((x, cum, 8), dict(allowed=torch.zeros(8, 4, dtype=torch.int64, device=device))),
                     ((x, cum, 8), dict(out=(cum, cum)))):
        with pytest.raises(ValueError):
            sel.select(*args, **kw)
    with pytest.raises(ValueError, match="end_token"):
        sel.select(x, cum, 8, finished=flags, end_token=100)
    for k in (0, -1, 129):
        with pytest.raises(ValueError, match="k must"):
            sel.select(x, cum, k)
    both = torch.zeros(2, 4, dtype=torch.int32, device=device)
    with pytest.raises(radx_amd.RadxError, match="overlap"):
        sel.select(x, cum, 4, out=(cum, both, torch.zeros_like(both)))
    with pytest.raises(radx_amd.RadxError, match="overlap"):
        sel.select(x, cum, 4, out=(torch.zeros_like(cum), both, both))
    sel.close()


# ---------------------------------------------------------------------------------------------
# reordering
# ---------------------------------------------------------------------------------------------
def plain_reorder(src, dst, parents, beams_to, lengths=None, length_dim=None, row_dim=0):
    """On the host: rows moved one by one, from a copy of the source."""
    import torch
    src = src.clone()
    batch, k = parents.shape
    beams = src.shape[row_dim] // batch
    s, d = src.movedim(row_dim, 0), dst.movedim(row_dim, 0)
    if length_dim is not None:
        ld = length_dim if length_dim > row_dim else length_dim + 1
    for b in range(batch):
        for j in range(k):
            p = int(parents[b, j])
            if not 0 <= p < beams:
                continue
            u, v = s[b * beams + p], d[b * beams_to + j]
            if lengths is not None:
                n = max(0, min(int(lengths[b]), u.shape[ld - 1]))
                u, v = u.narrow(ld - 1, 0, n), v.narrow(ld - 1, 0, n)
            v.copy_(u)
    return dst


def fill(shape, dtype, seed):
    import torch
    g = torch.Generator()
    g.manual_seed(seed)
    if dtype.is_floating_point:
        return torch.randn(shape, generator=g).to(dtype)
    return torch.randint(-100, 100, shape, generator=g).to(dtype)


def bits(t):
    import torch
    return t.contiguous().view(torch.uint8).cpu()


@pytest.mark.parametrize("beams,k", [(1, 1), (2, 2), (3, 3), (4, 4), (5, 5), (8, 8), (8, 3), (13, 13), (16, 16), (17, 17), (32, 32), (33, 20), (64, 64)])
@pytest.mark.parametrize("inner", [(1,), (7,), (64,), (3, 5, 16), (2, 129, 3), (4001,)])
def test_reorder_in_place(device, beams, k, inner):
    import torch
    import radx_amd
    batch = 3
    rng = np.random.default_rng(beams * 100 + len(inner))
    for dtype in (torch.bfloat16, torch.float32, torch.int8):
        host = fill((batch * beams,) + inner, dtype, beams)
        parents = rng.integers(0, beams, (batch, k)).astype(np.int32)
        if k > 2:
            parents[0, 1] = -1          # left as it was
            parents[1, 2] = beams       # so is this
            parents[2] = np.arange(k)   # nothing moves
        want = plain_reorder(host, host.clone(), parents, beams)
        got = host.to(device)
        radx_amd.beam_reorder(got, on(parents, device))
        assert torch.equal(bits(got), bits(want))


@pytest.mark.parametrize("beams,k", [(4, 4), (3, 6), (6, 3), (1, 5), (16, 64)])
def test_reorder_into_other_tensors(device, beams, k):
    import torch
    import radx_amd
    batch = 4
    parents = np.random.default_rng(k).integers(-1, beams, (batch, k)).astype(np.int32)
    states = [fill((batch * beams, 5, 33), torch.float32, 1), fill((batch * beams, 7), torch.bfloat16, 2), fill((batch * beams, 2, 3, 1), torch.int64, 3)]
    into = [fill((batch * k,) + s.shape[1:], s.dtype, 9) for s in states]
    want = [plain_reorder(s, d.clone(), parents, k) for s, d in zip(states, into)]
    src, dst = [s.to(device) for s in states], [d.to(device) for d in into]
    radx_amd.beam_reorder(src, on(parents, device), into=dst)
    for s, d, w, u in zip(src, dst, want, states):
        assert torch.equal(bits(d), bits(w)) and torch.equal(bits(s), bits(u))


@pytest.mark.parametrize("layout", ["rows heads positions", "rows positions heads", "layers rows positions", "positions rows"])
@pytest.mark.parametrize("in_place", [True, False])
def test_reorder_layouts_and_lengths(device, layout, in_place):
    """Caches longer than the sequences: what lies behind a length, and around a view, stays."""
    import torch
    import radx_amd
    batch, beams = 3, 4
    rows = batch * beams
    parents = np.array([[0, 0, 1, 3], [3, 2, 1, 0], [2, 2, 2, -1]], np.int32)
    shape, row_dim, length_dim = {"rows heads positions": ((rows, 3, 40, 16), 0, 2), "rows positions heads": ((rows, 40, 3, 17), 0, 1),
                                  "layers rows positions": ((2, rows, 40, 5), 1, 2), "positions rows": ((40, rows, 9), 1, None)}[layout]
    host = fill(shape, torch.float16, 5)
    other = fill(shape, torch.float16, 6)
    for lengths in ([0, 1, 40], [40, 40, 40], [17, -3, 1000]) if length_dim is not None else (None,):
        n = None if lengths is None else np.array(lengths, np.int32)
        got, into = host.to(device), other.to(device)
        want = plain_reorder(host, host.clone() if in_place else other.clone(), parents, beams, n, length_dim, row_dim)
        radx_amd.beam_reorder(got, on(parents, device), into=None if in_place else into, lengths=None if n is None else on(n, device),
                              length_dim=length_dim, row_dim=row_dim)
        assert torch.equal(bits(got if in_place else into), bits(want)), lengths
    if length_dim is not None:  # a view of the first positions
        got, want = host.to(device), host.clone()
        plain_reorder(want.narrow(length_dim, 0, 11), want.narrow(length_dim, 0, 11), parents, beams, row_dim=row_dim)
        radx_amd.beam_reorder(got.narrow(length_dim, 0, 11), on(parents, device), row_dim=row_dim)
        assert torch.equal(bits(got), bits(want))


def test_reorder_many_states_in_one_call(device):
    import torch
    import radx_amd
    batch, beams = 2, 3
    parents = np.array([[1, 1, 0], [2, 0, 2]], np.int32)
    hosts = [fill((batch * beams, 1 + i % 7, 4 + 31 * (i % 3)), (torch.float32, torch.bfloat16, torch.uint8)[i % 3], i) for i in range(61)]
    hosts.insert(10, torch.zeros(batch * beams, 0, 4))
    got = [h.to(device) for h in hosts]
    radx_amd.beam_reorder(got, on(parents, device))
    for h, g in zip(hosts, got):
        assert torch.equal(bits(g), bits(plain_reorder(h, h.clone(), parents, beams)))


def test_reorder_odd_addresses(device):
    """States that begin at every byte, with neighbours on both sides that have to stay."""
    import torch
    import radx_amd
    beams, width = 5, 37
    parents = np.array([[4, 0, 0, 2, 1]], np.int32)
    for start in range(16):
        host = fill((beams * width + 64,), torch.uint8, start)
        got = host.to(device)
        want = host.clone()
        view = want[start:start + beams * width].view(beams, width)
        plain_reorder(view, view, parents, beams)
        radx_amd.beam_reorder(got[start:start + beams * width].view(beams, width), on(parents, device))
        assert torch.equal(got.cpu(), want), start


def test_reorder_past_32_bits(device):
    """Offsets of more than 4 GiB, within a row and between rows."""
    import torch
    import radx_amd
    beams, width = 4, (1 << 31) // 2 + 24
    state = torch.empty(beams, width, dtype=torch.bfloat16, device=device)
    for r in range(beams):
        state[r].fill_(r + 1)
    state[:, -1] = torch.arange(10, 10 + beams, device=device)
    radx_amd.beam_reorder(state, on(np.array([[3, 3, 1, 2]], np.int32), device))
    torch.cuda.synchronize()
    for r, p in enumerate((3, 3, 1, 2)):
        assert float(state[r, -1]) == 10 + p and bool((state[r, :-1] == p + 1).all())
    del state
    torch.cuda.empty_cache()


def test_reorder_refuses_tensors(device):
    import torch
    import radx_amd
    s = torch.zeros(8, 16, device=device)
    p = torch.zeros(2, 4, dtype=torch.int32, device=device)
    for args, kw in (((s, p.long()), {}), ((s, p[0]), {}), ((s, p.t()), {}), ((s[:7], p), {}), ((s, p), dict(row_dim=2)), ((s, p), dict(lengths=p[:, 0])),
                     ((s, p), dict(lengths=p[:, 0].contiguous())), ((s, p), dict(lengths=p[:, 0].contiguous(), length_dim=0)),
                     ((s, p), dict(into=s.double())), ((s, p), dict(into=torch.zeros(8, 17, device=device))), ((s, p), dict(into=[s, s])),
                     (([s, torch.zeros(4, 2, device=device)], p), {}), ((s.cpu(), p), {})):
        with pytest.raises(ValueError):
            radx_amd.beam_reorder(*args, **kw)
    wide = torch.zeros(9, 16, device=device)
    with pytest.raises(radx_amd.RadxError, match="overlap"):
        radx_amd.beam_reorder(wide[:8], p, into=wide[1:])
    with pytest.raises(radx_amd.RadxError, match="written twice"):
        radx_amd.beam_reorder([s, s], p)
    line = torch.zeros(100, device=device)
    with pytest.raises(radx_amd.RadxError, match="rows and pieces overlap"):
        radx_amd.beam_reorder(line.as_strided((8, 3, 2), (4, 4, 1)), p)


# ---------------------------------------------------------------------------------------------
# backtrace
# ---------------------------------------------------------------------------------------------
def plain_backtrace(tokens, parents, steps, out):
    total, batch, k = tokens.shape
    for b in range(batch):
        ends = total if steps is None else max(0, min(total, int(steps[b])))
        place = np.arange(k)
        for t in range(ends - 1, -1, -1):
            out[b, :, t] = tokens[t, b, place]
            up = parents[t, b, place]
            place = np.where((up >= 0) & (up < k), up, place)
    return out


@pytest.mark.parametrize("k", [1, 2, 3, 4, 8, 13, 31, 64, 100, 128])
@pytest.mark.parametrize("total", [1, 2, 17, 64, 65, 1000, 4097])
def test_backtrace(device, k, total):
    import radx_amd
    batch = 3
    rng = np.random.default_rng(total * 200 + k)
    tokens = rng.integers(0, 1 << 24, (total, batch, k)).astype(np.int32)
    parents = rng.integers(-1, k + 1, (total, batch, k)).astype(np.int32)
    got = radx_amd.beam_backtrace(on(tokens, device), on(parents, device)).cpu().numpy()
    assert np.array_equal(got, plain_backtrace(tokens, parents, None, np.empty((batch, k, total), np.int32)))
    # permutations keep all places alive to the first step; ragged lengths, and an output with a pitch
    parents = np.argsort(rng.random((total, batch, k)), axis=2).astype(np.int32)
    steps = np.array([total, max(0, total // 2), total + 5 if k % 2 else -2], np.int32)
    out = np.full((batch, k, total + 3), -7, np.int32)
    dev_out = on(out, device)
    radx_amd.beam_backtrace(on(tokens, device), on(parents, device), steps=on(steps, device), out=dev_out[:, :, :total])
    plain_backtrace(tokens, parents, steps, out[:, :, :total])
    assert np.array_equal(dev_out.cpu().numpy(), out)


def test_backtrace_long(device):
    """More steps than one workgroup's memory holds at once."""
    import radx_amd
    total, batch, k = 30011, 2, 16
    rng = np.random.default_rng(0)
    tokens = rng.integers(0, 1000, (total, batch, k)).astype(np.int32)
    parents = np.argsort(rng.random((total, batch, k)), axis=2).astype(np.int32)
    got = radx_amd.beam_backtrace(on(tokens, device), on(parents, device)).cpu().numpy()
    assert np.array_equal(got, plain_backtrace(tokens, parents, None, np.empty((batch, k, total), np.int32)))


def test_backtrace_refuses_tensors(device):
    import torch
    import radx_amd
    t = torch.zeros(5, 2, 3, dtype=torch.int32, device=device)
    for args, kw in (((t.long(), t), {}), ((t, t.long()), {}), ((t[0], t[0]), {}), ((t, t[:4]), {}), ((t.transpose(0, 1), t.transpose(0, 1)), {}),
                     ((t, t), dict(steps=torch.zeros(3, dtype=torch.int32, device=device))), ((t, t), dict(out=torch.zeros(2, 3, 4, dtype=torch.int32, device=device))),
                     ((t, t), dict(out=torch.zeros(2, 5, 3, dtype=torch.int32, device=device).transpose(1, 2)))):
        with pytest.raises(ValueError):
            radx_amd.beam_backtrace(*args, **kw)
    assert radx_amd.beam_backtrace(t[:0], t[:0]).shape == (2, 3, 0)


# ---------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------
class Decoder:
    """A toy model whose next logits are a function of its state: state <- M[token] + 0.5 state, logits = state W.
    Values are multiples of 1/8 in small ranges, so that every product and sum below is exact in float32."""

    def __init__(self, vocab, width, seed):
        rng = np.random.default_rng(seed)
        self.m = rng.integers(-8, 9, (vocab, width)).astype(np.float64) / 8
        self.w = rng.integers(-8, 9, (width, vocab)).astype(np.float64) / 8
        self.vocab, self.width = vocab, width


@pytest.mark.parametrize("captured", [False, True])
def test_a_decoding_loop(device, captured):
    """select, reorder and backtrace over some steps, against a search on the host that copies whole hypotheses.
    Captured: one graph of a step, replayed, with eager work in between."""
    import torch
    import radx_amd
    batch, beams, vocab, width, steps, end = 3, 4, 701, 24, 12, 5
    model = Decoder(vocab, width, 1)
    m, w = on(model.m.astype(np.float32), device), on(model.w.astype(np.float32), device)
    rng = np.random.default_rng(3)
    start = rng.integers(-8, 9, (batch, width)).astype(np.float64) / 8

    # on the host: hypotheses are (score, tokens, state, ended)
    hyps = [[(0.0, (), start[b], False)] for b in range(batch)]
    for _ in range(steps):
        for b in range(batch):
            found = []
            for i, (score, toks, state, ended) in enumerate(hyps[b]):
                if ended:
                    found.append((score, i, end))
                    continue
                x = (state @ model.w)
                logp = x - x.max() - math.log(math.fsum(np.exp(x - x.max())))
                found += [(score + lp, i, v) for v, lp in enumerate(logp)]
            found.sort(key=lambda c: (-c[0], c[1], c[2]))
            hyps[b] = [(np.float32(s), hyps[b][i][1] + (v,), np.round((model.m[v] + 0.5 * hyps[b][i][2]) * 8) / 8, hyps[b][i][3] or v == end)
                       for s, i, v in found[:beams]]

    sel = radx_amd.BeamSelector(batch, beams, vocab, beams)
    state = on(np.repeat(start, beams, 0).astype(np.float32), device)
    cum = torch.full((batch, beams), float("-inf"), device=device)
    cum[:, 0] = 0.0
    finished = torch.zeros((batch, beams), dtype=torch.bool, device=device)
    tokens = torch.zeros((steps, batch, beams), dtype=torch.int32, device=device)
    parents = torch.zeros_like(tokens)
    at = torch.zeros(1, dtype=torch.int64, device=device)
    new = (torch.empty_like(cum), torch.empty((batch, beams), dtype=torch.int32, device=device),
           torch.empty((batch, beams), dtype=torch.int32, device=device), torch.empty_like(finished))

    def step():
        logits = (state.unsqueeze(2) * w).sum(1)
        sel.select(logits, cum, beams, finished=finished, end_token=end, out=new)
        radx_amd.beam_reorder(state, new[1])
        moved = m[new[2].reshape(-1).long().clamp(min=0)] + 0.5 * state
        state.copy_((moved * 8).round() / 8)
        cum.copy_(new[0])
        finished.copy_(new[3])
        tokens.index_copy_(0, at, new[2].unsqueeze(0))
        parents.index_copy_(0, at, new[1].unsqueeze(0))
        at.add_(1)

    if captured:
        keep = [t.clone() for t in (state, cum, finished, at)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        for t, k in zip((state, cum, finished, at), keep):
            t.copy_(k)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for t, k in zip((state, cum, finished, at), keep):
            t.copy_(k)
    for _ in range(steps):
        if captured:
            graph.replay()
            torch.cuda.synchronize()
            torch.ones(1000, device=device).sum().item()
        else:
            step()
    sequences = radx_amd.beam_backtrace(tokens, parents).cpu().numpy()
    for b in range(batch):
        for j, (score, toks, _, ended) in enumerate(hyps[b]):
            assert tuple(sequences[b, j]) == toks, (b, j)
            # a step's score is rounded once and its sum has its bound; the steps add up
            bound = steps * (abs(float(score)) * 2.0 ** -24 + lse_bound(vocab))
            assert abs(float(cum[b, j]) - float(score)) <= bound
            assert bool(finished[b, j]) == ended
    sel.close()


def test_calls_on_streams_of_their_own(device):
    """Two handles on two streams, and states moved on a third, all at once."""
    import torch
    import radx_amd
    streams = [torch.cuda.Stream() for _ in range(3)]
    cases = []
    for i in range(2):
        logits, x = make_logits(4, 4, 30000 + i, "bf16", device, seed=i)
        cum = (-np.random.default_rng(i).random((4, 4))).astype(np.float32)
        cases.append((radx_amd.BeamSelector(4, 4, 40000, 8), logits, x, cum, on(cum, device)))
    host = fill((16, 3, 1000), torch.float32, 3)
    state = host.to(device)
    parents = np.random.default_rng(7).integers(0, 4, (4, 4)).astype(np.int32)
    dev_parents = on(parents, device)
    torch.cuda.synchronize()
    for _ in range(4):
        outs = [sel.select(logits, dev_cum, 8, stream=s) for (sel, logits, _, _, dev_cum), s in zip(cases, streams)]
        radx_amd.beam_reorder(state, dev_parents, stream=streams[2])
        torch.cuda.synchronize()
        host = plain_reorder(host, host.clone(), parents, 4)
        assert torch.equal(state.cpu(), host)
        for (sel, _, x, cum, _), out in zip(cases, outs):
            check_best([o.cpu().numpy() for o in out], plain_scores(x, cum), x, 8, x.shape[2])
    for c in cases:
        c[0].close()


def test_c_plus_plus_layer(device):
    """The C++ layer's search over made-up logits equals the host's, token by token (harness/beam_test.cpp)."""
    import os
    import subprocess
    exe = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "harness", "beam_test")
    for args in ([], ["--batch", "1", "--beams", "1", "--vocab", "7", "--steps", "3", "--width", "1"], ["--batch", "2", "--beams", "17", "--vocab", "3001", "--steps", "5"]):
        out = subprocess.run([exe] + args, capture_output=True, text=True, timeout=100)
        assert out.returncode == 0 and "PASS" in out.stdout, out.stdout + out.stderr
